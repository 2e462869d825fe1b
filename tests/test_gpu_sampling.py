"""Sampling on the device against the definition in 64 bits: the token has to be the same one."""
import ctypes as C

import numpy as np
import pytest
import torch

import splosh_b200 as S
from oracle import oracle as O
from paged_reference import sample

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    g = S.tiny_geometry()
    e = S.Engine(g, S.EngineConfig(max_slots=2, max_rows=64, kv_pages=8, max_context=512))
    e.load_model(O.Model(O.tiny_geometry()))
    yield e
    e.close()


def device_sample(engine, x, limit, settings, uniform, ld=None, stream=None):
    """x [rows][width]; settings (temperature, top_k, top_p, min_p): arrays or None."""
    rows = x.shape[0]
    dx = torch.from_numpy(x).cuda()
    types = (np.float32, np.int32, np.float32, np.float32)
    buffers = [None if s is None else torch.from_numpy(np.ascontiguousarray(np.broadcast_to(s, rows), t)).cuda() for s, t in zip(settings, types)]
    du = torch.from_numpy(np.ascontiguousarray(uniform, np.float32)).cuda()
    ids = torch.full((rows + 1,), -5, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    t, k, p, m = (None if b is None else b.data_ptr() for b in buffers)
    engine.pass_sample(dx.data_ptr(), rows, ld or x.shape[1], limit, ids.data_ptr(), du.data_ptr(), temperature=t, top_k=k, top_p=p, min_p=m, stream=stream)
    engine.pass_wait()
    torch.cuda.synchronize()
    assert ids[rows].item() == -5
    return ids[:rows].cpu().numpy()


def expected(x, limit, settings, uniform):
    off = (1.0, 0, 1.0, 0.0)
    full = [np.broadcast_to(o if s is None else s, x.shape[0]) for s, o in zip(settings, off)]
    f32 = np.float32
    return np.array([sample(x[r, :limit], f32(full[0][r]), int(full[1][r]), f32(full[2][r]), f32(full[3][r]), f32(uniform[r])) for r in range(x.shape[0])])


def logits(rng, rows, width, deviation=2.0):
    x = rng.normal(0, deviation, (rows, width)).astype(np.float32)
    for r in range(rows):
        x[r, rng.integers(0, width, 20)] += rng.uniform(4, 9, 20).astype(np.float32)
    return x


@pytest.mark.parametrize("width,limit", [(1, 1), (2, 2), (31, 30), (1000, 1000), (1025, 1023), (32000, 32000), (65537, 65536), (248320, 248077)])
@pytest.mark.parametrize("settings", [(None, None, None, None), (0.8, 20, 0.95, None), (0.7, None, 0.9, None), (1.3, None, None, 0.05), (0.9, 500, 0.98, 0.001), (0.0, 5, 0.5, 0.5), (1.0, 1, None, None),
                                      (1.0, None, 0.0, None), (1.0, 7, 1.0, 0.0), (5.0, None, 0.999, None), (0.05, 100000, 0.99, 1e-6)])
def test_the_definitions_token(engine, width, limit, settings):
    rng = np.random.default_rng(width + sum(int(100 * (s or 0)) for s in settings))
    rows = 6
    x, u = logits(rng, rows, width), rng.random(rows).astype(np.float32)
    assert np.array_equal(device_sample(engine, x, limit, settings, u), expected(x, limit, settings, u))


def test_settings_of_their_own_for_every_row(engine):
    rng = np.random.default_rng(4)
    rows, width = 64, 5003
    x, u = logits(rng, rows, width), rng.random(rows).astype(np.float32)
    settings = (rng.choice([0.0, 0.5, 1.0, 2.0], rows), rng.choice([0, 1, 40, 6000], rows), rng.choice([0.3, 0.95, 1.0], rows), rng.choice([0.0, 0.1, 1.0, 2.0], rows))
    assert np.array_equal(device_sample(engine, x, width, settings, u), expected(x, width, settings, u))


def test_ties_go_to_the_lowest_index(engine):
    """Equal logits: every cut and every draw falls inside a group of ties, at places that both sides compute exactly (weights of one)."""
    width = 40000
    x = np.full((16, width), -1.0, np.float32)
    u = np.array([0.0, 0.25, 0.5, 0.75, 0.999, 0.5, 0.5, 0.5] * 2, np.float32)
    k = np.array([0] * 8 + [1, 10, 1000, 39999, 40000, 50000, 3, 1024], np.int32)
    p = np.array([1.0, 0.5, 0.25, 0.125, 1.0, 0.0, 0.75, 0.5] * 2, np.float32)
    settings = (None, k, p, np.array([0.0, 1.0] * 8, np.float32))
    assert np.array_equal(device_sample(engine, x, width, settings, u), expected(x, width, settings, u))
    x[:, ::3] = 2.0
    x[:, 1::3] = -0.0
    x[:, 4::6] = 0.0                                          # the same value as minus zero
    for settings in ((None, k, None, None), (None, k, p, None), (1e-3, None, p, None), (None, k, None, np.float32(0.5))):
        assert np.array_equal(device_sample(engine, x, width, settings, u), expected(x, width, settings, u))


@pytest.mark.parametrize("temperature", [1e-3, 0.3, 3.0, 20.0, 1e4])
def test_bins_of_few_and_of_very_many_values(engine, temperature):
    """At low temperatures nearly everything lies in the last bin, at high ones everything in the first, which no list holds."""
    rng = np.random.default_rng(6)
    for width in (9000, 100003):
        x, u = logits(rng, 7, width), rng.random(7).astype(np.float32)
        for k, p, m in ((0, 1.0, 0.0), (0, 0.9, 0.0), (5000, 0.99, 0.0), (8000, 1.0, 0.3), (0, 0.5, 0.7), (30, 0.9, 0.2)):
            assert np.array_equal(device_sample(engine, x, width, (temperature, k, p, m), u), expected(x, width, (temperature, k, p, m), u)), (k, p, m)


@pytest.mark.parametrize("k", [2000, 4096, 4097, 6000, 20000, 70000])
def test_a_large_top_k_and_the_other_filters_on_what_it_leaves(engine, k):
    rng = np.random.default_rng(k)
    x, u = logits(rng, 8, 80000), rng.random(8).astype(np.float32)
    for settings in ((1.0, k, 1.0, 0.0), (1.0, k, 0.999, 0.0), (0.8, k, 0.7, 0.01), (2.0, k, 1.0, 0.02)):
        assert np.array_equal(device_sample(engine, x, 80000, settings, u), expected(x, 80000, settings, u)), settings


@pytest.mark.parametrize("width", [262144, 262145, 400001, 524288])
def test_vocabularies_at_and_past_what_a_cluster_holds(engine, width):
    rng = np.random.default_rng(width)
    x, u = logits(rng, 3, width), rng.random(3).astype(np.float32)
    for settings in ((None, None, None, None), (0.8, 50, 0.9, 0.01), (1.0, 9000, 0.95, 0.0), (0.0, None, None, None)):
        assert np.array_equal(device_sample(engine, x, width, settings, u), expected(x, width, settings, u)), settings


def test_values_that_are_never_picked(engine):
    rng = np.random.default_rng(8)
    width = 3000
    x, u = logits(rng, 12, width), rng.random(12).astype(np.float32)
    x[:, rng.random(width) < 0.4] = -np.inf
    x[:, rng.random(width) < 0.2] = np.nan
    x[0] = -np.inf                                           # nothing left: id 0
    x[1] = np.nan
    x[2, 5:] = -np.inf
    x[3, :] = -np.inf; x[3, 1234] = -3.4e38                   # one value, the type's lowest
    x[4, [7, 90, 2000]] = np.inf                             # the largest values share the weight
    x[5] = np.where(np.isnan(x[5]), x[5], np.float32(-3.4028235e38))      # all at the lowest value
    x[6, 17] = 3.4028235e38
    for settings in ((None, None, None, None), (0.7, 50, 0.9, 0.01), (0.0, None, None, None), (1.0, 2, None, None), (1e-30, None, 0.5, None), (1e30, None, 0.999, None)):
        assert np.array_equal(device_sample(engine, x, width, settings, u), expected(x, width, settings, u)), settings


def test_uniform_numbers_at_their_ends(engine):
    rng = np.random.default_rng(2)
    x = logits(rng, 4, 2000)
    u = np.array([0.0, np.float32(1.0) - np.float32(2.0 ** -24), 1.0, 1e-30], np.float32)
    for settings in ((None, None, None, None), (0.8, 10, None, None), (1.0, None, 0.9, None)):
        assert np.array_equal(device_sample(engine, x, 2000, settings, u), expected(x, 2000, settings, u))


def test_draws_follow_the_distribution(engine):
    """A flat vocabulary and uniform numbers in equal steps: token i has to come back for every u inside its share, whatever the index (weights of one: both sides are exact)."""
    width = 4096
    x = np.zeros((512, width), np.float32)
    u = ((np.arange(512) + 0.5) / 512).astype(np.float32)
    assert np.array_equal(device_sample(engine, x, width, (None, None, None, None), u), np.ceil(u.astype(np.float64) * width).astype(int) - 1)


def test_rows_with_a_stride_and_streams(engine):
    rng = np.random.default_rng(12)
    x, u = logits(rng, 8, 6001), rng.random(8).astype(np.float32)
    want = expected(x, 5000, (0.9, 40, 0.9, 0.02), u)
    for stream in (None, 0, torch.cuda.Stream().cuda_stream):
        assert np.array_equal(device_sample(engine, x, 5000, (0.9, 40, 0.9, 0.02), u, stream=stream), want)


def test_a_step_sampled_on_the_device_is_the_host_samplers_token(engine):
    """The last step's logits: spl_sample against the definition on them, and, with top-k and top-p, against the host sampler given the same uniform numbers
    (its sums are 32-bit: these draws lie away from its boundaries)."""
    rng = np.random.default_rng(3)
    engine.reset_slot(0)
    engine.step([S.EngineRow(0, int(t), i, i >= 8) for i, t in enumerate(rng.integers(0, engine.g.vocab, 24))])
    x = engine.all_logits()
    sampler = S.Sampler(temperature=0.9, top_p=0.9, top_k=20, seed=77)
    ids, values = engine.topk(20, 31000)
    state = sampler.state.value
    host = [sampler.sample(i, v) for i, v in zip(ids, values)]
    sampler.state.value = state
    u = np.array([sampler.uniform01() for _ in host], np.float32)
    got = engine.sample(u, temperature=0.9, top_k=20, top_p=0.9, vocab_limit=31000)
    assert np.array_equal(got, host)
    assert np.array_equal(got, expected(x, 31000, (0.9, 20, 0.9, None), u))
    assert np.array_equal(engine.sample(u, temperature=0.0), engine.argmax())
    per_row = np.linspace(0.5, 2.0, 16).astype(np.float32)
    assert np.array_equal(engine.sample(u, temperature=per_row, min_p=0.02), expected(x, engine.g.vocab, (per_row, None, None, 0.02), u))


def test_refusals(engine):
    d = torch.zeros(4096, device="cuda")
    a = d.data_ptr()
    for args in ((a, 0, 100, 100), (a, 1, 100, 101), (a, 1, 100, 0), (a, 1, 1 << 20, (1 << 19) + 1), (a, 65536, 1, 1), (None, 1, 100, 100)):
        with pytest.raises(S.EngineError):
            engine.pass_sample(*args, a, a)
    with pytest.raises(S.EngineError):
        engine.pass_sample(a, 1, 100, 100, a, None)
    engine.reset_slot(0)
    engine.step([S.EngineRow(0, 5, 0, True)])
    with pytest.raises(S.EngineError):
        engine.sample([0.5, 0.5])
    with pytest.raises(S.EngineError):
        engine.sample([0.5], vocab_limit=engine.g.vocab + 1)


def test_infinite_values_share_the_weight_under_min_p(engine):
    """Several infinite logits with min-p and nothing else that ends what stays, at every share of theirs: on rows of few values, on rows that hold fewer values than top-k, and behind a cut."""
    rng = np.random.default_rng(21)
    u = np.array([0.0, 0.1, 0.33, 0.34, 0.5, 0.66, 0.67, 0.9, 0.999], np.float32)
    for width, at, settings in ((3000, [7, 90, 2000], (None, None, None, 0.05)), (3000, [7, 90, 2000], (0.7, None, None, 0.5)), (3000, [7, 90, 2000], (None, None, None, 1e-6)), (9500, [4, 5, 9000], (None, 9000, None, 0.05)),
                                (20000, [0, 900, 19999], (1.0, 9000, 1.0, 0.05)), (248077, [1, 100000, 248000], (None, None, None, 0.9)), (3000, [17], (None, None, None, 0.05)), (3000, [7, 90], (None, 2, None, 0.05))):
        x = logits(rng, len(u), width)
        if width == 9500:
            x[:, rng.random(width) < 0.5] = -np.inf
        x[:, at] = np.inf
        want = expected(x, width, settings, u)
        assert set(want) <= set(at)
        assert np.array_equal(device_sample(engine, x, width, settings, u), want), (width, settings)


def test_an_infinite_temperature_weighs_all_alike(engine):
    """Every value's weight is one, but for -inf and NaN; beside infinite values the finite ones have none."""
    rng = np.random.default_rng(22)
    u = np.array([0.0, 0.1, 0.33, 0.34, 0.5, 0.66, 0.67, 0.9, 0.999], np.float32)
    for width in (40, 3000, 9000):
        x = logits(rng, len(u), width)
        x[:, rng.random(width) < 0.3] = -np.inf
        x[:, rng.random(width) < 0.1] = np.nan
        x[0, 3:9] = [3.4e38, -3.4e38, 1e-40, -1e-40, 0.0, -0.0]
        for settings in ((np.inf, None, None, None), (np.inf, 30, None, None), (np.inf, None, 0.25, None), (np.inf, None, None, 0.5), (np.inf, 20, 0.5, 1.0), (np.inf, 6000, 0.75, 0.1)):
            assert np.array_equal(device_sample(engine, x, width, settings, u), expected(x, width, settings, u)), (width, settings)
        x[:, [5, 20, 31]] = np.inf
        for k, p, m, stay in ((None, None, None, 3), (None, None, 0.5, 3), (2, None, None, 2), (20, 0.5, 1.0, 2), (None, 0.25, None, 1), (6000, None, 0.1, 3), (None, None, 1.0, 3)):
            want = [(5, 20, 31)[max(int(np.ceil(np.float64(v) * stay)) - 1, 0)] for v in u]
            assert np.array_equal(device_sample(engine, x, width, (np.inf, k, p, m), u), want), (width, k, p, m)


@pytest.mark.parametrize("temperature", [1e-35, 8e-37, 1e-37, 3e-38, 1e-38, 1e-40, 1e-44])
def test_temperatures_near_the_types_smallest(engine, temperature):
    """Logits of the temperature's size, and some up to thousands of it below the maximum."""
    rng = np.random.default_rng(23)
    t = np.float32(temperature)
    for width in (2000, 50000):
        x = (rng.normal(0, 2, (9, width)) * np.float64(t)).astype(np.float32)
        x[:, rng.integers(0, width, 20)] += (rng.uniform(4, 9, 20) * np.float64(t)).astype(np.float32)
        x[:, ::3] = (-rng.uniform(20, 4000, x[:, ::3].shape) * np.float64(t)).astype(np.float32)
        x[:, 1:300:9] = (x.max(1, keepdims=True).astype(np.float64) - np.linspace(1380.0, 1425.0, len(range(1, 300, 9))) * np.float64(t)).astype(np.float32)
        u = rng.random(9).astype(np.float32)
        for settings in ((t, None, None, None), (t, None, 0.9, None), (t, None, None, 0.05), (t, None, 0.95, 0.01), (t, 40, None, None), (t, 40, 0.9, 0.02), (t, 9000, 0.98, 0.001), (t, None, None, 1e-6)):
            assert np.array_equal(device_sample(engine, x, width, settings, u), expected(x, width, settings, u)), (width, settings)


def fastest(engine, x, limit, settings, u, runs=8):
    """The token of every row, and the shortest of some runs on the device, in us."""
    rows = x.shape[0]
    types = (np.float32, np.int32, np.float32, np.float32)
    dx, du = torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda()
    buffers = [None if s is None else torch.from_numpy(np.ascontiguousarray(np.broadcast_to(s, rows), t)).cuda() for s, t in zip(settings, types)]
    t, k, p, m = (None if b is None else b.data_ptr() for b in buffers)
    ids, least = torch.zeros(rows, dtype=torch.int32, device="cuda"), float("inf")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(runs):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        with torch.cuda.stream(stream):
            begin.record()
            engine.pass_sample(dx.data_ptr(), rows, x.shape[1], limit, ids.data_ptr(), du.data_ptr(), temperature=t, top_k=k, top_p=p, min_p=m, stream=stream.cuda_stream)
            end.record()
        end.synchronize()
        least = min(least, begin.elapsed_time(end) * 1e3)
    return ids.cpu().numpy(), least


@pytest.fixture(scope="module")
def large(engine):
    """Twelve rows of 248,077 logits, and what sampling them takes where nothing is in the way."""
    rng = np.random.default_rng(31)
    x, u = logits(rng, 12, 248077), rng.random(12).astype(np.float32)
    ids, ordinary = fastest(engine, x, 248077, (1.0, None, 0.95, None), u)
    assert np.array_equal(ids, expected(x, 248077, (1.0, None, 0.95, None), u))
    return x, u, ordinary


@pytest.mark.parametrize("settings", [(0.1, 20, None, None), (0.2, 1000, None, None), (0.1, 50, 0.9, None), (0.1, None, None, 1e-14), (0.05, 100, None, 0.01), (0.1, None, 0.99, 1e-20)])
def test_values_without_a_weight_do_not_slow_a_row_down(engine, large, settings):
    x, u, ordinary = large
    ids, took = fastest(engine, x, 248077, settings, u)
    assert np.array_equal(ids, expected(x, 248077, settings, u))
    assert took < 4 * ordinary


@pytest.mark.parametrize("settings", [(3.0, None, 0.95, 0.02), (3.0, None, None, 0.05), (2.5, None, 0.95, 0.02)])
def test_the_draws_bins_do_not_crowd_out_the_end(engine, large, settings):
    x, u, ordinary = large
    ids, took = fastest(engine, x, 248077, settings, u)
    assert np.array_equal(ids, expected(x, 248077, settings, u))
    assert took < 4 * ordinary
