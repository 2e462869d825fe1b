"""A speculating server's decode step over tensors of the caller's own, whole: twenty sequences behind one prompt, their verify blocks appended to an e4m3 cache, attended with the prompt's pages read once for all, the target's
head, and the drafted tokens tested on the device. Against a plain 64-bit forward, against batches without groups, and captured into a graph."""
import numpy as np
import pytest
import torch

import splosh_b200 as S
from helpers import observed
from more_reference import verify
from splosh_b200.paged import debug_paged_plan_shared
from test_gpu_own_pass import DIM, HEADS, KV, LAYERS, ROT, THETA, TOLERANCE, Model

pytestmark = pytest.mark.gpu

PAGE, PAGES, PROMPT, SEQUENCES, BLOCK = 32, 168, 3328, 20, 3
# Keys and values are rounded to e4m3: independent relative errors of at most 2^-4 / sqrt(3) = 3.6e-2 (root mean square) of each, in two layers: 2 x 3.6e-2 of what the attention adds, which is at most all of the logits;
# beside what the 16-bit roundings do.
QUANTISED = 7.2e-2 + TOLERANCE


class Spec(Model):
    def __init__(self):
        super().__init__(7)
        self.k, self.v = ([torch.full((PAGES, KV, PAGE, DIM), 0x7f, device="cuda", dtype=torch.uint8) for _ in range(LAYERS)] for _ in range(2))
        self.ks, self.vs = ([torch.full((PAGES, KV, PAGE), float("nan"), device="cuda") for _ in range(LAYERS)] for _ in range(2))

    def paged(self, sequences, rows):
        return S.PagedAttention(self.engine, HEADS, KV, DIM, PAGES, page_tokens=PAGE, dtype="e4m3", rotary_dim=ROT, rope_theta=THETA, max_sequences=sequences, max_rows=rows, max_context=PAGE * PAGES)

    def layers_of_a_pass(self, paged, b, n, stream=None):
        e, p = self.engine, {k: v.data_ptr() for k, v in b.items()}
        ld = (HEADS + 2 * KV) * DIM
        for layer, w in enumerate(self.layers):
            scales = {"k_scale": self.ks[layer].data_ptr(), "v_scale": self.vs[layer].data_ptr()}
            e.pass_norm(p["h"], w["norm"][0], n, self.g.hidden, p["x"])
            e.pass_gemm(w["qkv"][0], p["x"], n, p["qkv"])
            paged.append(p["qkv"], p["qkv"] + 4 * HEADS * DIM, p["qkv"] + 4 * (HEADS + KV) * DIM, p["q"], self.k[layer].data_ptr(), self.v[layer].data_ptr(), ld=ld, q_norm=w["qn"][0], k_norm=w["kn"][0],
                         stream=stream, **scales)
            paged.attend(p["q"], self.k[layer].data_ptr(), self.v[layer].data_ptr(), p["a"], out_dtype="f32", stream=stream, **scales)
            e.pass_gemm(w["o"][0], p["a"], n, p["h"], p["h"])
            e.pass_norm(p["h"], w["post"][0], n, self.g.hidden, p["x"])
            e.pass_mlp_in(w["gate"][0], w["up"][0], p["x"], n, p["act"], p["scratch"])
            e.pass_gemm(w["down"][0], p["act"], n, p["h"], p["h"])
        e.pass_norm(p["h"], self.final[0], n, self.g.hidden, p["x"])
        e.pass_gemm_head(p["x"], n, p["logits"])

    def verify_step(self, paged, tokens, rows, lengths, table, groups, drafts, candidates, uniform, **settings):
        """tokens: the rows' tokens; drafts: the token drafted to follow each (negative: none)."""
        n = len(tokens)
        b = self.buffers(n)
        def device(x, t):
            return torch.from_numpy(np.ascontiguousarray(x, t)).cuda()
        dt, first = device(tokens, np.uint32), device(np.concatenate([[0], np.cumsum(rows)]), np.int32)
        dd, ci, cp, du = device(drafts, np.int32), device(candidates[0], np.int32), device(candidates[1], np.float32), device(uniform, np.float32)
        arrays = {k: torch.full((n,), v, device="cuda", dtype=torch.int32 if k == "top_k" else torch.float32) for k, v in settings.items()}
        accepted, following = (torch.full((len(rows),), -9, device="cuda", dtype=torch.int32) for _ in range(2))
        torch.cuda.synchronize()
        self.engine.pass_begin()
        paged.batch(rows, lengths, table, groups=groups)
        self.engine.pass_embed(dt.data_ptr(), n, b["h"].data_ptr())
        self.layers_of_a_pass(paged, b, n)
        self.engine.pass_verify(b["logits"].data_ptr(), len(rows), n, self.g.vocab, self.g.vocab - 7, first.data_ptr(), dd.data_ptr(), du.data_ptr(), b["ids"].data_ptr(), accepted.data_ptr(), following.data_ptr(),
                                candidates=ci.shape[1], candidate_ids=ci.data_ptr(), probabilities=cp.data_ptr(), **{k: v.data_ptr() for k, v in arrays.items()})
        self.engine.pass_wait()
        return b["logits"].cpu().numpy(), b["ids"].cpu().numpy(), accepted.cpu().numpy(), following.cpu().numpy()


@pytest.fixture(scope="module")
def model():
    m = Spec()
    yield m
    m.engine.close()


def off(a, b):
    return float((np.linalg.norm(a - b, axis=-1) / np.linalg.norm(b, axis=-1)).max())


def test_a_decode_step_of_a_speculating_server(model):
    rng = np.random.default_rng(3)
    order = rng.permutation(PAGES).astype(np.int32)
    prompt = rng.integers(0, model.g.vocab, PROMPT)
    shared = order[:PROMPT // PAGE]
    table = np.stack([np.concatenate([shared, order[len(shared) + 3 * s:len(shared) + 3 * (s + 1)]]) for s in range(SEQUENCES)])
    paged = model.paged(SEQUENCES, 64)
    for a in range(0, PROMPT, 64):                              # the prompt once, in the first sequence's pages
        model.step(paged, prompt[a:a + 64], [64], [a + 64], table[:1])
    own = [rng.integers(0, model.g.vocab, 5 + 2 * s) for s in range(SEQUENCES)]
    for s in range(1, SEQUENCES):                               # what each has added since
        held = len(own[s]) - 1
        model.step(paged, own[s][:held], [held], [PROMPT + held], table[s:s + 1])
    held = len(own[0]) - 1
    model.step(paged, own[0][:held], [held], [PROMPT + held], table[:1])
    # A block: the last token and two drafted ones.
    drafts = rng.integers(0, model.g.vocab, (SEQUENCES, BLOCK - 1))
    blocks = [np.concatenate([own[s][-1:], drafts[s]]) for s in range(SEQUENCES)]
    rows, lengths = [BLOCK] * SEQUENCES, [PROMPT + len(own[s]) - 1 + BLOCK for s in range(SEQUENCES)]
    drafted = np.concatenate([np.concatenate([drafts[s], [-1]]) for s in range(SEQUENCES)])
    u = rng.random((len(drafted), 2)).astype(np.float32)
    groups = [(SEQUENCES, PROMPT)]
    assert debug_paged_plan_shared(rows, lengths, groups, heads=HEADS, kv_heads=KV, head_dim=DIM, dtype="e4m3", pages=1, page_tokens=PAGE, max_sequences=SEQUENCES, max_rows=64, max_context=PAGE * PAGES)[4]
    # First with candidates that mean nothing, to see the logits; then as a drafter that knows them would have it.
    some = (np.tile(np.arange(8), (len(drafted), 1)), np.full((len(drafted), 8), 0.125, np.float32))
    logits, *_ = model.verify_step(paged, np.concatenate(blocks), rows, lengths, table, groups, drafted, some, u)
    near = np.argsort(-logits, axis=1, kind="stable")[:, :8]
    drafted = np.where(drafted >= 0, near[np.arange(len(drafted)), rng.integers(0, 3, len(drafted))], -1)
    q = rng.dirichlet(np.ones(8), len(drafted)).astype(np.float32)
    settings = dict(temperature=0.9, top_k=500, top_p=0.95)
    again, ids, accepted, following = model.verify_step(paged, np.concatenate(blocks), rows, lengths, table, groups, drafted, (near, q), u, **settings)
    assert np.array_equal(again, logits)
    f = np.float32
    want = np.array([verify(logits[r, :model.g.vocab - 7], f(0.9), 500, f(0.95), f(0.0), int(drafted[r]), list(zip(near[r].tolist(), q[r].tolist())), u[r]) for r in range(len(drafted))])
    assert np.array_equal(ids, want) and (ids < 0).any() and (ids >= 0).any()
    for s in range(SEQUENCES):
        mine = want[s * BLOCK:(s + 1) * BLOCK]
        stop = next((i for i in range(BLOCK) if mine[i] >= 0), BLOCK)
        assert accepted[s] == stop and following[s] == (mine[stop] if stop < BLOCK else -1)
    # The same rows without groups: the sums of the joint prefix differ in their order alone.
    plain, *_ = model.verify_step(paged, np.concatenate(blocks), rows, lengths, table, [], drafted, (near, q), u, **settings)
    assert off(logits, plain) <= TOLERANCE
    # And from the definition.
    for s in (0, 5):
        tokens = np.concatenate([prompt, own[s][:-1], blocks[s]])
        worst = off(logits[s * BLOCK:(s + 1) * BLOCK], model.plain(tokens)[-BLOCK:])
        observed(f"a speculating server's step, sequence {s}: {worst:.2e} of the logits' norm")
        assert worst <= QUANTISED


def test_append_attention_and_the_drafts_test_in_a_graph(model):
    """The three calls on a stream of the caller's, captured once and replayed while the sequences grow behind their common pages: the same bits as calls made one by one."""
    rng = np.random.default_rng(4)
    order = rng.permutation(PAGES).astype(np.int32)
    shared = PROMPT // PAGE
    table = np.stack([np.concatenate([order[:shared], order[shared + 3 * s:shared + 3 * (s + 1)]]) for s in range(SEQUENCES)])
    width, n = (HEADS + 2 * KV) * DIM, BLOCK * SEQUENCES
    start = torch.randn((2, PAGES, KV, PAGE, DIM), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.float8_e4m3fn).view(torch.uint8)
    states = []
    for graph_form in (False, True):
        paged = model.paged(SEQUENCES, n)
        g = torch.Generator(device="cuda").manual_seed(5)
        k, v = start[0].clone(), start[1].clone()
        ks, vs = (torch.full((PAGES, KV, PAGE), 0.02, device="cuda") for _ in range(2))
        qkv, q, out = torch.zeros((n, width), device="cuda"), torch.zeros((n, HEADS, DIM), device="cuda", dtype=torch.bfloat16), torch.zeros((n, HEADS * DIM), device="cuda")
        first, drafts = torch.arange(0, n + 1, BLOCK, device="cuda", dtype=torch.int32), torch.zeros(n, device="cuda", dtype=torch.int32)
        u, ids = torch.zeros((n, 2), device="cuda"), torch.zeros(n + 2 * SEQUENCES, device="cuda", dtype=torch.int32)
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()

        def calls():
            b, scales = qkv.data_ptr(), {"k_scale": ks.data_ptr(), "v_scale": vs.data_ptr()}
            paged.append(b, b + 4 * HEADS * DIM, b + 4 * (HEADS + KV) * DIM, q.data_ptr(), k.data_ptr(), v.data_ptr(), ld=width, stream=stream.cuda_stream, **scales)
            paged.attend(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), out_dtype="f32", stream=stream.cuda_stream, **scales)
            model.engine.pass_verify(out.data_ptr(), SEQUENCES, n, HEADS * DIM, HEADS * DIM, first.data_ptr(), drafts.data_ptr(), u.data_ptr(), ids.data_ptr(), ids[n:].data_ptr(), ids[n + SEQUENCES:].data_ptr(),
                                     stream=stream.cuda_stream)
        def batch(t):
            paged.batch([BLOCK] * SEQUENCES, [PROMPT + BLOCK * (t + 1) + s for s in range(SEQUENCES)], table, groups=[(SEQUENCES, PROMPT)], stream=stream.cuda_stream)
        batch(0)
        graph = torch.cuda.CUDAGraph()
        if graph_form:
            with torch.cuda.graph(graph, stream=stream):
                calls()
        results = []
        for t in range(16):
            with torch.cuda.stream(stream):
                qkv.normal_(generator=g); u.uniform_(generator=g); drafts.random_(0, HEADS * DIM, generator=g)
                batch(t)
                if graph_form:
                    graph.replay()
                else:
                    calls()
                results.append((out.clone(), ids.clone()))
        stream.synchronize()
        states.append((results, k.clone(), v.clone(), ks.clone(), vs.clone()))
    (a, *ca), (b, *cb) = states
    assert all(torch.equal(x[0], y[0]) and torch.equal(x[1], y[1]) for x, y in zip(a, b)) and all(torch.equal(x, y) for x, y in zip(ca, cb))
