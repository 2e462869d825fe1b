"""Drafted tokens tested on the device against the definition in 64 bits: what stays, and the tokens in the place of what does not, have to be the same ones."""
import numpy as np
import pytest
import torch

import splosh_b200 as S
from more_reference import verify
from test_gpu_sampling import logits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    e = S.Engine(S.tiny_geometry(), S.EngineConfig(max_slots=1, max_rows=64, kv_pages=4, max_context=512))
    yield e
    e.close()


def device(engine, x, limit, blocks, drafts, candidates, settings, uniform, stream=None, ld=None):
    """`blocks`: the sequences' rows. candidates: (ids, probabilities) [rows][c] or None. Returns (ids, accepted, next)."""
    rows = x.shape[0]
    first = torch.from_numpy(np.concatenate([[0], np.cumsum(blocks)]).astype(np.int32)).cuda()
    dx, du, dd = torch.from_numpy(x).cuda(), torch.from_numpy(np.ascontiguousarray(uniform, np.float32)).cuda(), torch.from_numpy(np.ascontiguousarray(drafts, np.int32)).cuda()
    arrays = [None if s is None else torch.from_numpy(np.ascontiguousarray(np.broadcast_to(s, rows), t)).cuda() for s, t in zip(settings, (np.float32, np.int32, np.float32, np.float32))]
    more = {}
    if candidates is not None:
        ci, cp = torch.from_numpy(np.ascontiguousarray(candidates[0], np.int32)).cuda(), torch.from_numpy(np.ascontiguousarray(candidates[1], np.float32)).cuda()
        more = dict(candidates=ci.shape[1], candidate_ids=ci.data_ptr(), probabilities=cp.data_ptr())
    ids = torch.full((rows + 1,), -5, dtype=torch.int32, device="cuda")
    accepted, following = (torch.full((len(blocks) + 1,), -5, dtype=torch.int32, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    t, k, p, m = (None if b is None else b.data_ptr() for b in arrays)
    engine.pass_verify(dx.data_ptr(), len(blocks), rows, ld or x.shape[1], limit, first.data_ptr(), dd.data_ptr(), du.data_ptr(), ids.data_ptr(), accepted.data_ptr(), following.data_ptr(), temperature=t, top_k=k,
                       top_p=p, min_p=m, stream=stream, **more)
    engine.pass_wait()
    torch.cuda.synchronize()
    assert ids[rows].item() == -5 and accepted[-1].item() == -5 and following[-1].item() == -5
    return ids[:rows].cpu().numpy(), accepted[:-1].cpu().numpy(), following[:-1].cpu().numpy()


def expected(x, limit, blocks, drafts, candidates, settings, uniform):
    full = [np.broadcast_to(o if s is None else s, x.shape[0]) for s, o in zip(settings, (1.0, 0, 1.0, 0.0))]
    f32 = np.float32
    ids = np.array([verify(x[r, :limit], f32(full[0][r]), int(full[1][r]), f32(full[2][r]), f32(full[3][r]), int(drafts[r]),
                           None if candidates is None else list(zip(candidates[0][r].tolist(), np.asarray(candidates[1][r], f32).tolist())), np.asarray(uniform[r], f32)) for r in range(x.shape[0])])
    accepted, following, at = [], [], 0
    for n in blocks:
        stop = next((i for i in range(n) if ids[at + i] >= 0), n)
        accepted.append(stop); following.append(ids[at + stop] if stop < n else -1)
        at += n
    return ids, np.array(accepted), np.array(following)


def drafter(rng, x, limit, count, noise=1.0):
    """Candidates of a drafter that sees nearly the same logits, their probabilities, and the one it took."""
    y = np.where(x[:, :limit] > -np.inf, np.nan_to_num(x[:, :limit], nan=-9.0), -2.0) + noise * rng.standard_normal((x.shape[0], limit))
    ids = np.argsort(-y, axis=1, kind="stable")[:, :count]
    value = np.take_along_axis(y, ids, 1)
    p = np.exp(value - value.max(1, keepdims=True))
    p = (p / p.sum(1, keepdims=True)).astype(np.float32)
    taken = np.minimum((np.cumsum(p, 1) < rng.random((x.shape[0], 1))).sum(1), count - 1)
    return ids[np.arange(x.shape[0]), taken], (ids, p)


def blocks_of(rng, rows):
    blocks = []
    while sum(blocks) < rows:
        blocks.append(int(min(rng.integers(0, 9), rows - sum(blocks))))
    return blocks


def agree(engine, x, limit, blocks, drafts, candidates, settings, uniform, **more):
    got, want = device(engine, x, limit, blocks, drafts, candidates, settings, uniform, **more), expected(x, limit, blocks, drafts, candidates, settings, uniform)
    for g, w in zip(got, want):
        assert np.array_equal(g, w), (settings, g.tolist(), w.tolist())
    return got


SETTINGS = [(None, None, None, None), (0.8, 20, 0.95, None), (0.7, None, 0.9, None), (1.3, None, None, 0.05), (0.9, 500, 0.98, 0.001), (0.0, 5, 0.5, 0.5), (1.0, 1, None, None), (1.0, None, 0.0, None),
            (1.0, 7, 1.0, 0.0), (5.0, None, 0.999, None), (0.05, 100000, 0.99, 1e-6), (1.0, 9000, 0.99, 0.001), (0.9, None, 0.95, 0.02)]


@pytest.mark.parametrize("width,limit", [(1, 1), (2, 2), (31, 30), (1000, 1000), (1025, 1023), (32000, 32000), (65537, 65536), (248320, 248077)])
@pytest.mark.parametrize("settings", SETTINGS)
def test_the_definitions_answers(engine, width, limit, settings):
    rng = np.random.default_rng(width + sum(int(100 * (s or 0)) for s in settings))
    rows = 12
    x, u = logits(rng, rows, width), rng.random((rows, 2)).astype(np.float32)
    drafts, candidates = drafter(rng, x, limit, min(limit, 16))
    drafts[[3, 11]] = -1
    agree(engine, x, limit, [4, 0, 5, 3], drafts, candidates, settings, u)
    agree(engine, x, limit, [4, 0, 5, 3], drafts, None, settings, u)


def test_settings_of_their_own_for_every_row(engine):
    rng = np.random.default_rng(4)
    rows, width = 96, 5003
    x, u = logits(rng, rows, width), rng.random((rows, 2)).astype(np.float32)
    settings = (rng.choice([0.0, 0.5, 1.0, 2.0], rows), rng.choice([0, 1, 40, 6000], rows), rng.choice([0.3, 0.95, 1.0], rows), rng.choice([0.0, 0.1, 1.0, 2.0], rows))
    for count, noise in ((1, 0.5), (16, 0.0), (64, 3.0)):
        drafts, candidates = drafter(rng, x, width, count, noise)
        ids, accepted, _ = agree(engine, x, width, blocks_of(rng, rows), drafts, candidates, settings, u)
        assert (ids < 0).any() and (ids >= 0).any()


def test_a_drafter_of_other_tokens_and_odd_lists(engine):
    """Drafts that are no token of the vocabulary, or not among the candidates; candidates out of range, listed twice, of probability zero, or masked."""
    rng = np.random.default_rng(5)
    rows, width = 24, 3000
    x, u = logits(rng, rows, width), rng.random((rows, 2)).astype(np.float32)
    x[:, rng.random(width) < 0.3] = -np.inf
    x[:, rng.random(width) < 0.1] = np.nan
    drafts, (ids, p) = drafter(rng, x, width, 8)
    ids, p = ids.copy(), p.copy()
    ids[0, 3], ids[1, 0], ids[2, 5] = width + 7, -4, 2147483647
    ids[3, 1] = ids[3, 0]; ids[4, 4] = ids[4, 2]; ids[4, 5] = ids[4, 2]
    p[5] = 0.0; p[6, 0] = 0.0
    drafts[7], drafts[8], drafts[9], drafts[10] = width, 2147483647, -1, -2147483648
    drafts[11] = int(np.nanargmax(x[11])); ids[11] = (ids[11] + 1) % width          # perhaps not listed
    masked = np.flatnonzero(x[12] == -np.inf)
    drafts[12], ids[12, 0] = masked[0], masked[0]
    x[13] = -np.inf
    x[14] = np.nan
    x[15] = -np.inf; x[15, 77] = 1.0; drafts[15] = 77; ids[15, 0] = 77; p[15] = 0.0; p[15, 0] = 1.0
    x[16, [5, 900]] = np.inf; drafts[16] = 900
    for settings in ((None, None, None, None), (0.7, 50, 0.9, 0.01), (0.0, None, None, None), (1.0, 2, None, None), (1.0, None, 0.8, None), (1.0, None, None, 0.1)):
        agree(engine, x, width, [8, 1, 0, 6, 9], drafts, (ids, p), settings, u)
        agree(engine, x, width, [8, 1, 0, 6, 9], drafts, None, settings, u)


def test_ties_and_flat_rows(engine):
    """Equal logits: every cut, every draw and every candidate falls inside a group of ties, at places that both sides compute exactly (weights of one, probabilities of whole powers of two)."""
    width, rows = 32768, 12
    rng = np.random.default_rng(9)
    for base in (np.full(width, -1.0, np.float32), np.where(np.arange(width) % 4 == 0, 2.0, -0.0).astype(np.float32), np.where(np.arange(width) % 2 == 0, 2.0, -40.0).astype(np.float32)):
        x = np.repeat(base[None], rows, 0)
        ids = np.stack([rng.choice(np.flatnonzero(base == base.max()), 8, replace=False) for _ in range(rows)])
        p = np.repeat(np.float32([0.5, 0.25, 0.125, 0.0625, 2.0 ** -15, 2.0 ** -16, 2.0 ** -20, 0.0])[None], rows, 0)
        drafts = ids[np.arange(rows), np.arange(rows) % 8].copy()
        drafts[5] = -1
        u = np.stack([np.full(rows, 0.5), (np.arange(rows) + 0.5) / rows], 1).astype(np.float32)
        for settings in ((None, None, None, None), (None, 1024, None, None), (None, 8192, None, None), (None, 5, 0.5, None), (None, None, 0.25, None), (1e-3, None, 0.5, None), (None, 16384, 0.5, 1.0)):
            agree(engine, x, width, [5, 7], drafts, (ids, p), settings, u)
            agree(engine, x, width, [5, 7], drafts, None, settings, u)


@pytest.mark.parametrize("temperature", [1e-3, 0.3, 3.0, 20.0, 1e4])
def test_bins_of_few_and_of_very_many_values(engine, temperature):
    rng = np.random.default_rng(6)
    for width in (9000, 100003):
        x, u = logits(rng, 7, width), rng.random((7, 2)).astype(np.float32)
        drafts, candidates = drafter(rng, x, width, 16)
        drafts[6] = -1
        for k, p, m in ((0, 1.0, 0.0), (0, 0.9, 0.0), (5000, 0.99, 0.0), (8000, 1.0, 0.3), (0, 0.5, 0.7), (30, 0.9, 0.2)):
            agree(engine, x, width, [7], drafts, candidates, (temperature, k, p, m), u)


@pytest.mark.parametrize("width", [262144, 262145, 524288])
def test_vocabularies_at_and_past_what_a_cluster_holds(engine, width):
    rng = np.random.default_rng(width)
    x, u = logits(rng, 3, width), rng.random((3, 2)).astype(np.float32)
    drafts, candidates = drafter(rng, x, width, 16)
    for settings in ((None, None, None, None), (0.8, 50, 0.9, 0.01), (1.0, 9000, 0.95, 0.0), (0.0, None, None, None)):
        agree(engine, x, width, [3], drafts, candidates, settings, u)


def test_infinite_and_tiny_temperatures(engine):
    rng = np.random.default_rng(22)
    x, u = logits(rng, 9, 3000), rng.random((9, 2)).astype(np.float32)
    drafts, candidates = drafter(rng, x, 3000, 4)
    for settings in ((np.inf, None, None, None), (np.inf, 30, None, None), (np.inf, None, 0.25, None), (1e-37, None, None, None), (1e-37, None, 0.9, None), (1e30, None, 0.999, None)):
        agree(engine, x, 3000, [9], drafts, candidates, settings, u)


def test_uniform_numbers_at_their_ends(engine):
    """0 keeps whatever has a probability; 1 and just below it refuse what the target likes less than the drafter."""
    rng = np.random.default_rng(2)
    x = logits(rng, 8, 2000)
    drafts, candidates = drafter(rng, x, 2000, 8, 0.2)
    below = np.float32(1.0) - np.float32(2.0 ** -24)
    u = np.array([[0, 0], [0, below], [below, 0.5], [below, below], [1, 1], [1, 0.3], [1e-30, 1e-30], [0.5, 1e-30]], np.float32)
    for settings in ((None, None, None, None), (0.8, 10, None, None), (1.0, None, 0.9, None)):
        agree(engine, x, 2000, [8], drafts, candidates, settings, u)
        agree(engine, x, 2000, [8], drafts, None, settings, u)


def test_what_comes_out_is_distributed_as_the_target(engine):
    """A drafter far from the target: over 20,000 blocks of one draft the first token that comes out has the target's distribution (each share within five deviations of a binomial's)."""
    rng = np.random.default_rng(11)
    rows, width = 20000, 8
    row = rng.normal(0, 1.5, width).astype(np.float32)
    x = np.repeat(row[None], rows, 0)
    q = rng.dirichlet(np.ones(4)).astype(np.float32)
    ids = np.repeat(rng.permutation(width)[None, :4], rows, 0)
    drafts = ids[0][np.minimum((np.cumsum(q) < rng.random((rows, 1))).sum(1), 3)]
    got, _, _ = device(engine, x, width, [rows], drafts, (ids, np.repeat(q[None], rows, 0)), (0.9, None, None, None), rng.random((rows, 2)))
    token = np.where(got < 0, drafts, got)
    p = np.exp((row - row.max()).astype(np.float64) / 0.9); p /= p.sum()
    share = np.bincount(token, minlength=width) / rows
    assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / rows) + 1e-9).all()


def test_strides_streams_and_a_captured_graph(engine):
    rng = np.random.default_rng(12)
    rows = 16
    x, u = logits(rng, rows, 6001), rng.random((rows, 2)).astype(np.float32)
    drafts, candidates = drafter(rng, x, 5000, 16)
    settings = (0.9, 40, 0.9, 0.02)
    want = expected(x, 5000, [9, 7], drafts, candidates, settings, u)
    for stream in (None, 0, torch.cuda.Stream().cuda_stream):
        agree(engine, x, 5000, [9, 7], drafts, candidates, settings, u, stream=stream)
    # Captured once, replayed on other logits.
    cuda = [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (x, u, drafts.astype(np.int32), candidates[0].astype(np.int32), candidates[1], np.array([0, 9, 16], np.int32))]
    out = torch.zeros(rows + 4, dtype=torch.int32, device="cuda")
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        engine.pass_verify(cuda[0].data_ptr(), 2, rows, 6001, 5000, cuda[5].data_ptr(), cuda[2].data_ptr(), cuda[1].data_ptr(), out.data_ptr(), out[rows:].data_ptr(), out[rows + 2:].data_ptr(), candidates=16,
                           candidate_ids=cuda[3].data_ptr(), probabilities=cuda[4].data_ptr(), stream=stream.cuda_stream)
    for seed in (1, 2):
        other = logits(np.random.default_rng(seed), rows, 6001)
        cuda[0].copy_(torch.from_numpy(other))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ids, accepted, following = expected(other, 5000, [9, 7], drafts, candidates, (None,) * 4, u)
        assert np.array_equal(out.cpu().numpy(), np.concatenate([ids, accepted, following]))
    assert len(want[1]) == 2


def test_it_agrees_with_the_host_sampler(engine):
    """With a top-k of 20, what spl_speculative_resolve answers for the same uniform numbers (its sums are 32-bit: these rows lie away from its boundaries)."""
    rng = np.random.default_rng(31)
    rows, width = 40, 4000
    x = logits(rng, rows, width)
    drafts, (ids, p) = drafter(rng, x, width, 16)
    sampler = S.Sampler(temperature=0.9, top_p=0.9, top_k=20, seed=5)
    u, host = np.zeros((rows, 2), np.float32), []
    for r in range(rows):
        order = np.argsort(-x[r], kind="stable")[:20]
        kept, target = sampler.distribution(order.astype(np.int32), x[r, order])
        state = sampler.state.value
        u[r, 0], u[r, 1] = sampler.uniform01(), sampler.uniform01()
        sampler.state.value = state
        answer = sampler.resolve(int(drafts[r]), ids[r].astype(np.int32), p[r], kept, target)
        host.append(-1 if answer is None else answer)
    got, _, _ = device(engine, x, width, [rows], drafts, (ids, p), (0.9, 20, 0.9, None), u)
    assert np.array_equal(got, host)


def test_refusals(engine):
    a = torch.zeros(4096, device="cuda").data_ptr()
    good = dict(device_logits=a, sequences=1, rows=2, ld=100, vocab_limit=100, device_first=a, device_drafts=a, device_uniform=a, device_ids=a, device_accepted=a, device_next=a)
    for bad in (dict(device_logits=None), dict(sequences=0), dict(sequences=65536), dict(rows=0), dict(rows=65536), dict(vocab_limit=0), dict(vocab_limit=101), dict(ld=1 << 20, vocab_limit=(1 << 19) + 1),
                dict(device_first=None), dict(device_drafts=None), dict(device_uniform=None), dict(device_ids=None), dict(device_accepted=None), dict(device_next=None), dict(candidates=-1),
                dict(candidates=65, candidate_ids=a, probabilities=a), dict(candidates=4), dict(candidates=4, candidate_ids=a), dict(candidates=4, probabilities=a)):
        with pytest.raises(S.EngineError):
            engine.pass_verify(**{**good, **bad})


def test_ends_of_sequences_that_are_out_of_range_are_cut(engine):
    """device_first is the caller's: numbers past the rows, or that fall, count no row that is not there."""
    rng = np.random.default_rng(1)
    x, u = logits(rng, 4, 100), rng.random((4, 2)).astype(np.float32)
    cuda = [torch.from_numpy(a).cuda() for a in (x, u, np.full(4, -1, np.int32), np.array([-5, 2, 1, 9], np.int32))]
    out = torch.zeros(10, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    engine.pass_verify(cuda[0].data_ptr(), 3, 4, 100, 100, cuda[3].data_ptr(), cuda[2].data_ptr(), cuda[1].data_ptr(), out.data_ptr(), out[4:].data_ptr(), out[7:].data_ptr())
    engine.pass_wait()
    ids = out[:4].tolist()
    assert out[4:7].tolist() == [0, 0, 0] and out[7:].tolist() == [ids[0], -1, ids[1]]
