"""A whole pass over the caller's own tensors, built from the engine's primitives as a program would use them: embedding, norm, q|k|v GEMM, append with norms and rotation, attention over the
paged cache, output GEMM, norm, MLP, the target's head, sampling. Against a plain 64-bit forward of the same quantised weights, and in the forms a server runs it in: the prompt at once, in chunks, and
token by token; several sequences in one batch; a decode step captured into a graph."""
import numpy as np
import pytest
import torch

import splosh_b200 as S
from helpers import observed
from oracle import oracle as O
from paged_reference import sample

pytestmark = pytest.mark.gpu

LAYERS, HEADS, KV, DIM, ROT, THETA, PAGE, PAGES = 2, 8, 2, 128, 32, 1e6, 32, 24


def bits_to_float(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


class Model:
    """Two layers of the tiny shape's width on tensors of the caller's own."""

    def __init__(self, seed=0):
        self.g = S.tiny_geometry()
        self.engine = S.Engine(self.g, S.EngineConfig(max_slots=1, max_rows=64, kv_pages=4, max_context=512))
        self.target = O.Model(O.tiny_geometry())
        self.engine.load_model(self.target)
        rng = np.random.default_rng(seed)
        H, I = self.g.hidden, self.g.inter

        def q4(n, k):
            t = O.quantize_mlx4((rng.standard_normal((n, k)) * 0.03).astype(np.float32))
            dense = O.dequant_mlx4(t[0], bits_to_float(t[1]), bits_to_float(t[2]), k).astype(np.float64)
            return self.engine.tensor_q4(*t), dense

        def vec(n):
            b = (O.bf16_round((1.0 + 0.1 * rng.standard_normal(n)).astype(np.float32)).view(np.uint32) >> 16).astype(np.uint16)
            return self.engine.tensor_vector(b), bits_to_float(b).astype(np.float64)
        self.layers = [dict(norm=vec(H), qkv=q4((HEADS + 2 * KV) * DIM, H), qn=vec(DIM), kn=vec(DIM), o=q4(H, HEADS * DIM), post=vec(H), gate=q4(I, H), up=q4(I, H), down=q4(H, I))
                       for _ in range(LAYERS)]
        self.final = vec(H)
        self.k = [torch.full((PAGES, KV, PAGE, DIM), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(LAYERS)]
        self.v = [torch.full_like(self.k[0], float("nan")) for _ in range(LAYERS)]

    def paged(self, sequences, rows):
        return S.PagedAttention(self.engine, HEADS, KV, DIM, PAGES, page_tokens=PAGE, rotary_dim=ROT, rope_theta=THETA, max_sequences=sequences, max_rows=rows, max_context=PAGE * PAGES)

    def buffers(self, n):
        def new(*shape, dtype=torch.float32):
            return torch.zeros(shape, device="cuda", dtype=dtype)
        g = self.g
        return dict(h=new(n, g.hidden), x=new(n, g.hidden), qkv=new(n, (HEADS + 2 * KV) * DIM), q=new(n, HEADS, DIM, dtype=torch.bfloat16), a=new(n, HEADS, DIM), act=new(n, g.inter),
                    scratch=new(n, g.inter), logits=new(n, g.vocab), ids=new(n, dtype=torch.int32), u=new(n))

    def layers_of_a_pass(self, paged, b, n, stream=None):
        e, p = self.engine, {k: v.data_ptr() for k, v in b.items()}
        ld = (HEADS + 2 * KV) * DIM
        for layer, w in enumerate(self.layers):
            e.pass_norm(p["h"], w["norm"][0], n, self.g.hidden, p["x"])
            e.pass_gemm(w["qkv"][0], p["x"], n, p["qkv"])
            paged.append(p["qkv"], p["qkv"] + 4 * HEADS * DIM, p["qkv"] + 4 * (HEADS + KV) * DIM, p["q"], self.k[layer].data_ptr(), self.v[layer].data_ptr(), ld=ld, q_norm=w["qn"][0], k_norm=w["kn"][0],
                         stream=stream)
            paged.attend(p["q"], self.k[layer].data_ptr(), self.v[layer].data_ptr(), p["a"], out_dtype="f32", stream=stream)
            e.pass_gemm(w["o"][0], p["a"], n, p["h"], p["h"])
            e.pass_norm(p["h"], w["post"][0], n, self.g.hidden, p["x"])
            e.pass_mlp_in(w["gate"][0], w["up"][0], p["x"], n, p["act"], p["scratch"])
            e.pass_gemm(w["down"][0], p["act"], n, p["h"], p["h"])
        e.pass_norm(p["h"], self.final[0], n, self.g.hidden, p["x"])
        e.pass_gemm_head(p["x"], n, p["logits"])

    def step(self, paged, tokens, rows, lengths, table, uniform=None, **settings):
        n = len(tokens)
        b = self.buffers(n)
        dt = torch.from_numpy(np.asarray(tokens, np.uint32)).cuda()
        if uniform is not None:
            b["u"].copy_(torch.from_numpy(np.asarray(uniform, np.float32)))
        arrays = {k: torch.full((n,), v, device="cuda", dtype=torch.int32 if k == "top_k" else torch.float32) for k, v in settings.items()}
        torch.cuda.synchronize()
        self.engine.pass_begin()
        paged.batch(rows, lengths, table)
        self.engine.pass_embed(dt.data_ptr(), n, b["h"].data_ptr())
        self.layers_of_a_pass(paged, b, n)
        if uniform is not None:
            self.engine.pass_sample(b["logits"].data_ptr(), n, self.g.vocab, self.g.vocab - 7, b["ids"].data_ptr(), b["u"].data_ptr(), **{k: v.data_ptr() for k, v in arrays.items()})
        self.engine.pass_wait()
        return b["logits"].cpu().numpy(), b["ids"].cpu().numpy()

    def plain(self, tokens):
        """The same in 64 bits without any rounding of activations: [tokens][vocab]."""
        packed, scales, biases = self.target.q4(-1, "embed")
        h = O.dequant_mlx4(packed[tokens], bits_to_float(scales[tokens]), bits_to_float(biases[tokens]), self.g.hidden).astype(np.float64)
        n, position = len(tokens), np.arange(len(tokens))

        def norm(x, w):
            return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.g.eps) * w

        def turn(x):
            y = x.copy()
            for i in range(ROT // 2):
                a = (position * THETA ** (-2.0 * i / ROT))[:, None]
                y[..., i], y[..., i + ROT // 2] = x[..., i] * np.cos(a) - x[..., i + ROT // 2] * np.sin(a), x[..., i + ROT // 2] * np.cos(a) + x[..., i] * np.sin(a)
            return y
        for w in self.layers:
            qkv = norm(h, w["norm"][1]) @ w["qkv"][1].T
            q, k, v = (t.reshape(n, -1, DIM) for t in np.split(qkv, [HEADS * DIM, (HEADS + KV) * DIM], axis=1))
            q, k = turn(norm(q, w["qn"][1])), turn(norm(k, w["kn"][1]))
            out = np.zeros((n, HEADS, DIM))
            for head in range(HEADS):
                s = q[:, head] @ k[:, head * KV // HEADS].T / np.sqrt(DIM)
                s[np.triu_indices(n, 1)] = -np.inf
                s = np.exp(s - s.max(1, keepdims=True))
                out[:, head] = s @ v[:, head * KV // HEADS] / s.sum(1, keepdims=True)
            h = h + out.reshape(n, -1) @ w["o"][1].T
            x = norm(h, w["post"][1])
            gate, up = x @ w["gate"][1].T, x @ w["up"][1].T
            h = h + (gate / (1.0 + np.exp(-gate)) * up) @ w["down"][1].T
        packed, scales, biases = self.target.q4(-1, "head")
        return norm(h, self.final[1]) @ O.dequant_mlx4(packed, bits_to_float(scales), bits_to_float(biases), self.g.hidden).astype(np.float64).T


@pytest.fixture(scope="module")
def model():
    m = Model()
    yield m
    m.engine.close()


# GEMM inputs are rounded to bf16 (2^-9 each, ten roundings deep), keys, values and probabilities too: independent relative errors of 2^-9 through two layers of four GEMMs and an attention come to
# about sqrt(14) 2^-9 = 7e-3 of the logits' norm; twice that is allowed.
TOLERANCE = 1.5e-2


def close(a, b):
    worst = np.linalg.norm(a - b, axis=-1) / np.linalg.norm(b, axis=-1)
    assert worst.max() <= TOLERANCE, worst.max()
    return float(worst.max())


def test_a_prompt_at_once_in_chunks_and_token_by_token(model):
    rng = np.random.default_rng(1)
    tokens = rng.integers(0, model.g.vocab, 45)
    want = model.plain(tokens)
    order = rng.permutation(PAGES).astype(np.int32)
    paged = model.paged(1, 64)
    whole, _ = model.step(paged, tokens, [45], [45], order[None, :2])
    observed(f"a pass over the caller's tensors, 45 rows: {close(whole, want):.2e} of the logits' norm")
    chunked = []
    for a, b in ((0, 1), (1, 33), (33, 44), (44, 45)):
        chunked.append(model.step(paged, tokens[a:b], [b - a], [b], order[None, 4:6])[0])
    close(np.concatenate(chunked), want)
    single = [model.step(paged, tokens[i:i + 1], [1], [i + 1], order[None, 8:10])[0] for i in range(45)]
    close(np.concatenate(single), want)


def test_several_sequences_sampled_on_the_device(model):
    """A prompt beside decoding sequences in one batch; the ids are the definition's on the logits of the pass."""
    rng = np.random.default_rng(2)
    order = rng.permutation(PAGES).astype(np.int32)
    table = np.stack([order[:3], order[3:6], order[6:9]])
    tokens = [rng.integers(0, model.g.vocab, n) for n in (34, 20, 60)]
    paged = model.paged(3, 64)
    for s in (0, 1):
        held = len(tokens[s]) - 1
        model.step(paged, tokens[s][:held], [held], [held], table[s:s + 1])
    rows = np.concatenate([tokens[0][-1:], tokens[1][-1:], tokens[2]])
    u = rng.random(len(rows)).astype(np.float32)
    logits, ids = model.step(paged, rows, [1, 1, 60], [34, 20, 60], table, uniform=u, temperature=0.8, top_k=200, top_p=0.95, min_p=0.001)
    close(logits, np.concatenate([model.plain(tokens[0])[-1:], model.plain(tokens[1])[-1:], model.plain(tokens[2])]))
    f = np.float32
    assert np.array_equal(ids, [sample(logits[r, :model.g.vocab - 7], f(0.8), 200, f(0.95), f(0.001), u[r]) for r in range(len(rows))])


def test_append_attention_and_sampling_of_a_decode_step_in_a_graph(model):
    """The three calls on a stream of the caller's, captured once and replayed while the sequences grow: the same bits as calls made one by one."""
    rng = np.random.default_rng(3)
    table = rng.permutation(PAGES).astype(np.int32)[:6].reshape(2, 3)
    width = (HEADS + 2 * KV) * DIM
    states = []
    for graph_form in (False, True):
        paged = model.paged(2, 2)
        g = torch.Generator(device="cuda").manual_seed(5)
        k, v = torch.zeros_like(model.k[0]), torch.zeros_like(model.v[0])
        qkv, q, out = torch.zeros((2, width), device="cuda"), torch.zeros((2, HEADS, DIM), device="cuda", dtype=torch.bfloat16), torch.zeros((2, HEADS * DIM), device="cuda")
        u, ids = torch.zeros(2, device="cuda"), torch.zeros(2, device="cuda", dtype=torch.int32)
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()

        def calls():
            b = qkv.data_ptr()
            paged.append(b, b + 4 * HEADS * DIM, b + 4 * (HEADS + KV) * DIM, q.data_ptr(), k.data_ptr(), v.data_ptr(), ld=width, stream=stream.cuda_stream)
            paged.attend(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), out_dtype="f32", stream=stream.cuda_stream)
            model.engine.pass_sample(out.data_ptr(), 2, HEADS * DIM, HEADS * DIM, ids.data_ptr(), u.data_ptr(), stream=stream.cuda_stream)
        paged.batch([1, 1], [1, 1], table, stream=stream.cuda_stream)
        graph = torch.cuda.CUDAGraph()
        if graph_form:
            with torch.cuda.graph(graph, stream=stream):
                calls()
        results = []
        for t in range(70):
            with torch.cuda.stream(stream):
                qkv.normal_(generator=g); u.uniform_(generator=g)
                paged.batch([1, 1], [t + 1, t // 2 + 1], table, stream=stream.cuda_stream)
                if graph_form:
                    graph.replay()
                else:
                    calls()
                results.append((out.clone(), ids.clone()))
        stream.synchronize()
        states.append((results, k.clone(), v.clone()))
    (a, ka, va), (b, kb, vb) = states
    assert all(torch.equal(x[0], y[0]) and torch.equal(x[1], y[1]) for x, y in zip(a, b)) and torch.equal(ka, kb) and torch.equal(va, vb)


def test_the_callers_device_stays_current_and_a_closed_engine_is_refused():
    e = S.Engine(S.tiny_geometry(), S.EngineConfig(max_slots=1, max_rows=8, kv_pages=1, max_context=256))
    before = torch.cuda.current_device()
    paged = S.PagedAttention(e, 4, 2, 64, 2, page_tokens=16, max_sequences=1, max_rows=1, max_context=32)
    paged.batch([1], [1], np.zeros((1, 1), np.int32))
    assert torch.cuda.current_device() == before
    e.pass_wait()
    e.close()
    with pytest.raises(S.EngineError):
        paged.batch([1], [1], np.zeros((1, 1), np.int32))
    paged.close()


def test_an_object_closed_behind_its_engine_gives_its_memory_back():
    def once():
        e = S.Engine(S.tiny_geometry(), S.EngineConfig(max_slots=1, max_rows=8, kv_pages=1, max_context=256))
        paged = S.PagedAttention(e, 24, 4, 256, 2, page_tokens=16, max_sequences=8, max_rows=64, max_context=32)      # 39 MB of partial sums
        e.close()
        paged.close()
    once()
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    for _ in range(3):
        once()
    torch.cuda.synchronize()
    assert before - torch.cuda.mem_get_info()[0] < 20e6
