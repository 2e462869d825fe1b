"""The paged cache of the caller's own: append and attention against plain 64-bit implementations, over types, head layouts, page sizes, lengths from one
token on, windows, padding, streams and graphs. What may not be read is NaN."""
import numpy as np
import pytest
import torch

import splosh_b200 as S
from helpers import observed
from paged_reference import Scene, TYPES, check_attention, half_step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    e = S.Engine(S.tiny_geometry(), S.EngineConfig(max_slots=1, max_rows=64, kv_pages=4, max_context=512))
    yield e
    e.close()


def bf16_bits(x):
    return x.to(torch.bfloat16).view(torch.int16).numpy().view(np.uint16)


# ---- attention -----------------------------------------------------------------------------------
def attend(engine, scene, out_dtype=None, stream=None, paged=None):
    paged = paged or scene.paged(engine, S.PagedAttention)
    out = torch.full((scene.total + 1, scene.heads, scene.head_dim), 7.0, device="cuda", dtype=TYPES[out_dtype or scene.dtype])
    torch.cuda.synchronize()
    paged.batch(scene.rows, scene.lengths, scene.table, stream=stream)
    paged.attend(scene.dq.data_ptr(), scene.k.data_ptr(), scene.v.data_ptr(), out.data_ptr(), out_dtype=out_dtype, stream=stream)
    engine.pass_wait()
    torch.cuda.synchronize()
    assert (out[scene.total:] == 7.0).all()              # rows behind the last sequence stay
    return out[:scene.total]


SHAPES = [(8, 2, 128), (24, 4, 256), (6, 6, 64), (16, 1, 128), (5, 1, 64), (12, 2, 256), (32, 1, 64)]


@pytest.mark.parametrize("heads,kv_heads,head_dim", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("out_dtype", ["same", "f32"])
def test_head_shapes_and_types(engine, heads, kv_heads, head_dim, dtype, out_dtype):
    scene = Scene(heads + head_dim, heads, kv_heads, head_dim, [1, 0, 7, 3], [1, 40, 150, 301], dtype=dtype)
    out = dtype if out_dtype == "same" else "f32"
    worst = check_attention(scene, attend(engine, scene, out), out)
    observed(f"paged attention {heads}/{kv_heads}/{head_dim} {dtype} -> {out}: {worst:.2f} of the bound")


@pytest.mark.parametrize("page_tokens", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_page_sizes_and_layouts(engine, page_tokens, layout, head_dim):
    scene = Scene(page_tokens + head_dim, 4, 2, head_dim, [2, 1, 5], [page_tokens, page_tokens + 1, 3 * page_tokens - 1], page_tokens=page_tokens, layout=layout)
    check_attention(scene, attend(engine, scene, "f32"), "f32")


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 511, 640, 1000])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_lengths_around_tiles_and_pages(engine, length, head_dim):
    scene = Scene(length, 4, 1, head_dim, [min(length, 3), 1], [length, length], page_tokens=64)
    check_attention(scene, attend(engine, scene), "bf16")


@pytest.mark.parametrize("rows,lengths", [([130], [130]), ([301, 1, 1], [301, 77, 500]), ([97], [700]), ([33, 34, 35], [33, 99, 290]), ([16] * 9, [16 + 37 * i for i in range(9)])])
@pytest.mark.parametrize("heads,kv_heads,head_dim,dtype", [(6, 1, 256, "bf16"), (8, 2, 128, "fp16"), (3, 1, 64, "bf16")])
def test_prompts_chunks_and_mixed_batches(engine, rows, lengths, heads, kv_heads, head_dim, dtype):
    scene = Scene(sum(lengths), heads, kv_heads, head_dim, rows, lengths, page_tokens=16, dtype=dtype, layout="token")
    check_attention(scene, attend(engine, scene), dtype)


@pytest.mark.parametrize("head_dim,dtype", [(64, "bf16"), (64, "fp16"), (128, "bf16"), (128, "fp16"), (256, "bf16"), (256, "fp16")])
@pytest.mark.parametrize("count,around", [(149, 256), (200, 300), (40, 1000), (300, 20)])
def test_blocks_of_several_tiles_and_pieces(engine, head_dim, dtype, count, around):
    """More tiles than blocks: a block takes several tiles of one sequence and pieces of several sequences, one after the other."""
    lengths = [around] * count if around == 256 else [around + (37 * i) % around for i in range(count)]
    scene = Scene(count, 2, 1, head_dim, [1 + i % 2 for i in range(count)], lengths, page_tokens=64, dtype=dtype)
    check_attention(scene, attend(engine, scene, "f32"), "f32")
    again = attend(engine, scene, "f32")
    for _ in range(5):
        assert torch.equal(attend(engine, scene, "f32"), again)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 129, 300])
@pytest.mark.parametrize("causal", [True, False])
def test_windows_and_blocks_that_see_themselves(engine, window, causal):
    scene = Scene(window, 8, 2, 128, [16, 1, 40], [300, 150, 40], page_tokens=32, causal=causal, window=window)
    check_attention(scene, attend(engine, scene, "f32"), "f32")


@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_long_contexts_of_few_rows(engine, head_dim):
    scene = Scene(9, 4, 1, head_dim, [1, 4], [9001, 5000], page_tokens=128)
    check_attention(scene, attend(engine, scene), "bf16")


def test_scores_far_apart_and_a_maximum_that_keeps_rising(engine):
    """Keys that grow with the position raise a row's maximum tile after tile; large queries make most probabilities vanish."""
    for dtype in ("bf16", "fp16"):
        scene = Scene(3, 4, 2, 128, [4, 200], [900, 700], page_tokens=64, dtype=dtype)
        for s, (keys, _) in enumerate(scene.tokens):
            factor = torch.linspace(0.1, 12.0, keys.shape[0]).to(TYPES[dtype]).double()[:, None, None]
            keys.copy_((keys * factor).to(TYPES[dtype]).double())
            for i in range(-(-keys.shape[0] // 64)):
                part = keys[i * 64:(i + 1) * 64]
                scene.k[scene.table[s, i], :, :part.shape[0]] = part.transpose(0, 1).to(TYPES[dtype]).cuda()
        check_attention(scene, attend(engine, scene, "f32"), "f32")


def test_what_the_mask_hides_may_be_anything(engine):
    """Infinities in tokens that a row does not see: behind the last token, in front of the window."""
    scene = Scene(5, 4, 1, 128, [1, 1], [200, 77], page_tokens=64, window=50)
    want, _ = scene.expected()
    for s, length in enumerate(scene.lengths):
        for cache in (scene.k, scene.v):
            for token in range(length - 50):
                cache[scene.table[s, token // 64], :, token % 64] = float("inf") if token % 2 else float("nan")
    check_attention(scene, attend(engine, scene, "f32"), "f32")


def test_what_is_no_number_in_a_token_that_is_seen_shows(engine):
    """A NaN in one key or value reaches exactly the rows that see it, in any place of a tile."""
    for place in (0, 1, 2, 3, 67, 130):
        for which in ("k", "v"):
            scene = Scene(place, 2, 1, 128, [140], [140], page_tokens=64)
            getattr(scene, which)[scene.table[0, place // 64], 0, place % 64, 5] = float("nan")
            out = attend(engine, scene, "f32")
            assert out[place:].isnan().any(-1).all()
            if which == "k":
                assert not out[:place].isnan().any()


def test_a_masked_tokens_values_do_not_count_however_large(engine):
    """Later tokens of a chunk with values near the type's end: a weight of nothing, not of next to nothing."""
    scene = Scene(17, 2, 1, 128, [100], [100], page_tokens=64)
    keys, values = scene.tokens[0]
    values[50:] = 3e38
    for token in range(50, 100):
        scene.v[scene.table[0, token // 64], :, token % 64] = 3e38
    out = attend(engine, scene, "f32")[:50].double().cpu()
    want, bound = scene.expected()
    assert ((out - want[:50]).abs() <= bound[:50]).all()


def test_strides_of_a_cache_that_holds_keys_and_values_side_by_side(engine):
    """K and V of a page next to each other, and the layers' pages interleaved: every stride larger than the data."""
    scene = Scene(11, 4, 2, 128, [3, 1], [90, 33], page_tokens=32)
    wide = torch.full((scene.pages, 3, 2, 32, 128 + 64), float("nan"), device="cuda", dtype=torch.bfloat16)
    wide[:, 1, :, :, :128], wide[:, 2, :, :, :128] = scene.k, scene.v
    paged = S.PagedAttention(engine, 4, 2, 128, scene.pages, page_tokens=32, strides=(wide.stride(0), wide.stride(2), wide.stride(3)), max_sequences=2, max_rows=4, max_context=96)
    scene.k, scene.v = wide[:, 1], wide[:, 2]
    check_attention(scene, attend(engine, scene, paged=paged), "bf16")


def test_pages_shared_by_sequences(engine):
    """Two sequences that begin with the same pages read the same tokens."""
    scene = Scene(21, 4, 2, 128, [1, 1], [64, 70], page_tokens=32)
    table = scene.table.copy()
    table[0, :2] = table[1, :2]
    scene.table = table
    scene.tokens[0] = tuple(x[:64] for x in scene.tokens[1])
    check_attention(scene, attend(engine, scene), "bf16")


def test_runs_are_equal_to_the_bit_and_streams_do_not_matter(engine):
    scene = Scene(2, 24, 4, 256, [1, 8, 50], [3000, 777, 50], page_tokens=256)
    first = attend(engine, scene)
    again = attend(engine, scene)
    side = torch.cuda.Stream()
    other = attend(engine, scene, stream=side.cuda_stream)
    legacy = attend(engine, scene, stream=0)
    assert torch.equal(first, again) and torch.equal(first, other) and torch.equal(first, legacy)


def test_a_captured_graph_follows_the_batch(engine):
    """The graph of a decode step, replayed with longer sequences in other pages."""
    scenes = [Scene(30 + i, 8, 2, 128, [1, 2], lengths, page_tokens=32, spare_pages=40 - sum(-(-n // 32) for n in lengths)) for i, lengths in enumerate(([40, 33], [41, 600], [1, 2]))]
    paged = S.PagedAttention(engine, 8, 2, 128, 40, page_tokens=32, scale=scenes[0].scale, max_sequences=2, max_rows=3, max_context=700)
    q, k, v = (torch.empty_like(x) for x in (scenes[0].dq, scenes[0].k, scenes[0].v))
    out = torch.zeros((3, 8, 128), device="cuda", dtype=torch.bfloat16)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    paged.batch(scenes[0].rows, scenes[0].lengths, scenes[0].table, stream=stream.cuda_stream)
    with torch.cuda.graph(graph, stream=stream):
        paged.attend(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), stream=stream.cuda_stream)
        with pytest.raises(S.EngineError) as caught:
            paged.batch(scenes[0].rows, scenes[0].lengths, scenes[0].table, stream=stream.cuda_stream)
        assert caught.value.case == "invalidArgument" and "capture" in str(caught.value)
    for scene in scenes:
        with torch.cuda.stream(stream):
            q.copy_(scene.dq); k.copy_(scene.k); v.copy_(scene.v)
            paged.batch(scene.rows, scene.lengths, scene.table, stream=stream.cuda_stream)
            graph.replay()
        stream.synchronize()
        check_attention(scene, out, "bf16")


@pytest.mark.parametrize("page_tokens", [16, 256])
def test_steps_without_a_wait_between_them(engine, page_tokens):
    """Batch, append and attend queued one after the other, several sequences growing and leaving: what a step without waits reads is what the step before wrote, to the bit."""
    heads, kv_heads, dim, steps, pages = 8, 2, 128, 24, 3 * (-(-400 // page_tokens))
    g = torch.Generator().manual_seed(page_tokens)
    x = torch.randn((steps, 2, 3, heads + 2 * kv_heads, dim), generator=g).cuda()
    table = torch.randperm(pages, generator=g).numpy().astype(np.int32).reshape(3, -1)
    start = torch.randn((2, pages, kv_heads, page_tokens, dim), generator=g).to(torch.bfloat16).cuda()

    def run(wait):
        paged = S.PagedAttention(engine, heads, kv_heads, dim, pages, page_tokens=page_tokens, rotary_dim=64, rope_theta=1e4, max_sequences=3, max_rows=3, max_context=400)
        k, v = start[0].clone(), start[1].clone()
        q, out = (torch.zeros((steps, 2, 3, heads, dim), device="cuda", dtype=torch.bfloat16) for _ in range(2))
        torch.cuda.synchronize()
        for step in range(steps):
            lengths = [1 + step, 120 + step, (300 if step % 2 else 5) + step]
            paged.batch([1, 1, 1], lengths, table)
            for layer in range(2):                        # of one cache: the second writes what the first has read
                row = x[step, layer].data_ptr()
                paged.append(row, row + 4 * heads * dim, row + 4 * (heads + kv_heads) * dim, q[step, layer].data_ptr(), k.data_ptr(), v.data_ptr(), ld=(heads + 2 * kv_heads) * dim)
                paged.attend(q[step, layer].data_ptr(), k.data_ptr(), v.data_ptr(), out[step, layer].data_ptr())
                if wait:
                    engine.pass_wait()
        engine.pass_wait()
        torch.cuda.synchronize()
        return out, k, v

    for a, b in zip(run(True), run(False)):
        assert torch.equal(a, b)


# ---- append --------------------------------------------------------------------------------------
def expected_append(x, position, rotary, theta, weight, eps):
    """[rows][heads][head_dim] in 64 bits, and the bound on the 32-bit arithmetic in front of the rounding."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    z, wide = y.clone(), y.abs().clone()
    half = rotary // 2
    for i in range(half):
        angle = position.double() * float(theta) ** (-2.0 * i / rotary)
        c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        z[..., i], z[..., i + half] = y[..., i] * c - y[..., i + half] * s, y[..., i + half] * c + y[..., i] * s
        wide[..., i] = wide[..., i + half] = y[..., i].abs() + y[..., i + half].abs()
    # Norm: the sum's relative error is below 16 steps of 2^-24 for 256 terms in eight serial and five tree additions, root, quotient and two products
    # five more; turn: angle within 2^-23 turns (2^-20 of the values), sine and cosine and three operations a few steps.
    return z, wide * 2.0 ** -19


@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 128), (24, 4, 256), (3, 3, 64), (1, 1, 64), (40, 8, 128)])
@pytest.mark.parametrize("rotary", [0, 2, 6, "quarter", "whole"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("source,norm,layout", [("f32", True, "head"), ("f32", False, "token"), ("fp16", False, "head"), ("bf16", True, "token")])
def test_append(engine, heads, kv_heads, head_dim, rotary, dtype, source, norm, layout):
    rotary = {"quarter": head_dim // 4, "whole": head_dim}.get(rotary, rotary)
    rows, lengths, page = [1, 0, 5, 20], [200001, 9, 5, 60], 32
    theta = 1e6
    seed = heads + head_dim + rotary
    g = torch.Generator().manual_seed(seed)
    total, pages = sum(rows), 8
    table = np.full((4, -(-200001 // page)), 0, np.int32)      # a long sequence whose earlier tokens lie in one page (they are not touched)
    table[0, 200000 // page] = 5
    table[1, 0], table[2, 0], table[3, :2] = 6, 1, (4, 2)
    width = heads + 2 * kv_heads
    x = torch.randn((total, width + 1, head_dim), generator=g).to(TYPES[source])
    wq, wk = (1.0 + 0.2 * torch.randn(head_dim, generator=g)).to(torch.bfloat16), (1.0 + 0.2 * torch.randn(head_dim, generator=g)).to(torch.bfloat16)
    shape = (pages, kv_heads, page, head_dim) if layout == "head" else (pages, page, kv_heads, head_dim)
    k, v = torch.full(shape, 3.0, device="cuda", dtype=TYPES[dtype]), torch.full(shape, 3.0, device="cuda", dtype=TYPES[dtype])
    q = torch.full((total + 1, heads, head_dim), 3.0, device="cuda", dtype=TYPES[dtype])
    dx = x.cuda()
    paged = S.PagedAttention(engine, heads, kv_heads, head_dim, pages, page_tokens=page, dtype=dtype, layout=layout, rotary_dim=rotary, rope_theta=theta, max_sequences=4, max_rows=total,
                             max_context=200001)
    norms = [engine.tensor_vector(bf16_bits(w)) for w in (wq, wk)] if norm else [None, None]
    torch.cuda.synchronize()
    paged.batch(rows, lengths, table)
    size, base = x.element_size(), dx.data_ptr()
    paged.append(base, base + size * heads * head_dim, base + size * (heads + kv_heads) * head_dim, q.data_ptr(), k.data_ptr(), v.data_ptr(), dtype=source, ld=(width + 1) * head_dim,
                 q_norm=norms[0], k_norm=norms[1])
    engine.pass_wait()
    for t in norms:
        if t:
            engine.tensor_destroy(t)
    sequence = np.repeat(np.arange(4), rows)
    position = np.concatenate([np.arange(n - r, n) for r, n in zip(rows, lengths)])
    eps = engine.g.eps
    want = [expected_append(x[:, a:b], torch.from_numpy(position), r, theta, w if norm and w is not None else None, eps)
            for a, b, r, w in ((0, heads, rotary, wq), (heads, heads + kv_heads, rotary, wk), (heads + kv_heads, width, 0, None))]
    kk, vv = (c.cpu() if layout == "head" else c.cpu().transpose(1, 2) for c in (k, v))
    touched = torch.zeros((pages, page), dtype=torch.bool)
    page_of, slot_of = table[sequence, position // page], position % page
    touched[page_of, slot_of] = True
    got = [q[:total].cpu(), kk[page_of, :, slot_of], vv[page_of, :, slot_of]]
    for name, g_, (w_, e_) in zip("qkv", got, want):
        bound = e_ + half_step(dtype) * (w_.abs() + e_) + 2.0 ** -25
        worst = ((g_.double() - w_).abs() / bound).max().item()
        assert worst <= 1.0, (name, worst)
    assert (q[total:] == 3.0).all() and (kk.transpose(1, 2)[~touched] == 3.0).all() and (vv.transpose(1, 2)[~touched] == 3.0).all()


def test_refusals(engine):
    def make(**more):
        args = dict(heads=4, kv_heads=2, head_dim=128, pages=8, page_tokens=32, max_sequences=2, max_rows=4, max_context=128)
        args.update(more)
        return S.PagedAttention(engine, **args)
    for bad in (dict(head_dim=96), dict(heads=5), dict(heads=130, kv_heads=2), dict(page_tokens=48), dict(page_tokens=512), dict(pages=0), dict(rotary_dim=130), dict(rotary_dim=3), dict(window=-1),
                dict(dtype="f32"), dict(max_rows=0), dict(max_sequences=0), dict(max_context=0), dict(scale=-1.0), dict(scale=float("nan")), dict(rotary_dim=64, rope_theta=0.0),
                dict(strides=(8192, 4096, 64)), dict(strides=(8192, 4100, 128)), dict(strides=(4096, 4096, 128)), dict(layout="channel"), dict(dtype="int8")):
        with pytest.raises(S.EngineError) as caught:
            make(**bad)
        assert caught.value.case == "invalidArgument", bad
    paged = make()
    buffer = torch.zeros(1 << 16, device="cuda")
    a = buffer.data_ptr()
    with pytest.raises(S.EngineError) as caught:
        paged.attend(a, a, a, a)
    assert "no batch" in str(caught.value)
    good = ([1, 1], [33, 20], np.array([[0, 1], [2, 3]], np.int32))
    paged.batch(*good)
    for case, rows, lengths, table in (("invalidRows", [2, 1], [1, 20], good[2]), ("invalidRows", [-1, 1], [33, 20], good[2]), ("contextExceeded", [1, 1], [129, 20], np.zeros((2, 5), np.int32)),
                                       ("invalidRows", [1, 1], [33, 20], np.array([[0, 8], [2, 3]], np.int32)), ("invalidRows", [1, 1], [33, 20], np.array([[0, -1], [2, 3]], np.int32)),
                                       ("invalidRows", [1, 1], [33, 20], np.array([[0], [2]], np.int32)), ("invalidRows", [0, 0], [33, 20], good[2]), ("invalidRows", [3, 2], [33, 20], good[2]),
                                       ("invalidRows", [1, 1, 1], [1, 1, 1], np.array([[0], [1], [2]], np.int32))):
        with pytest.raises(S.EngineError) as caught:
            paged.batch(rows, lengths, table)
        assert caught.value.case == case, (rows, lengths)
    for call in (lambda: paged.attend(a + 8, a, a, a), lambda: paged.attend(a, a + 2, a, a), lambda: paged.attend(a, a, a, a + 4), lambda: paged.attend(a, a, a, a, out_dtype="fp16"),
                 lambda: paged.append(a + 4, a, a, a, a, a), lambda: paged.append(a, a, a, a, a, a, ld=100), lambda: paged.append(a, a, a, a, a, a, ld=1025), lambda: paged.attend(None, a, a, a)):
        with pytest.raises(S.EngineError) as caught:
            call()
        assert caught.value.case == "invalidArgument"
    vector = engine.tensor_vector(np.zeros(64, np.uint16))
    with pytest.raises(S.EngineError):
        paged.append(a, a, a, a, a, a, q_norm=vector)
    engine.tensor_destroy(vector)
    # One page that two sequences would write to: attention may read it, append refuses.
    paged.batch([1, 1], [33, 20], np.array([[0, 1], [1, 3]], np.int32))
    with pytest.raises(S.EngineError) as caught:
        paged.append(a, a, a, a, a, a)
    assert "one page" in str(caught.value)
    paged.close()


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("page_tokens", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("window", [64, 65, 96, 100, 128, 200])
def test_windows_that_begin_anywhere_in_a_tile(engine, head_dim, page_tokens, window):
    """The first chunks of a piece's first tile are left out, and its first product begins in the middle of a chunk or at its start; everything in front is NaN."""
    lengths = [256, 300, 129, 192]
    scene = Scene(window + page_tokens, 2, 1, head_dim, [1] * 4, lengths, page_tokens=page_tokens, window=window)
    for cache in (scene.k, scene.v):
        for s, length in enumerate(lengths):
            for token in range(length - window):
                cache[scene.table[s, token // page_tokens], :, token % page_tokens] = float("nan")
    check_attention(scene, attend(engine, scene, "f32"), "f32")


def test_a_new_object_rotates_by_its_own_table_at_once(engine):
    """Append on a stream that waits for nobody, right behind the object's making: the table of angles is there. (Every object has another base, and often the memory of the one before.)"""
    heads, kv_heads, dim, rows = 2, 1, 128, 4
    g = torch.Generator().manual_seed(40)
    x = torch.randn((rows, heads + 2 * kv_heads, dim), generator=g).cuda()
    k, v = (torch.zeros((1, kv_heads, 16, dim), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    stream, base = torch.cuda.Stream(), x.data_ptr()
    for i in range(40):
        q = torch.zeros((2, rows, heads, dim), device="cuda", dtype=torch.bfloat16)
        torch.cuda.synchronize()
        paged = S.PagedAttention(engine, heads, kv_heads, dim, 1, page_tokens=16, rotary_dim=dim, rope_theta=10.0 ** (1 + i % 7), max_sequences=1, max_rows=rows, max_context=16)
        for n in range(2):
            paged.batch([rows], [16], np.zeros((1, 1), np.int32), stream=stream.cuda_stream)
            paged.append(base, base + 4 * heads * dim, base + 4 * (heads + kv_heads) * dim, q[n].data_ptr(), k.data_ptr(), v.data_ptr(), ld=(heads + 2 * kv_heads) * dim, stream=stream.cuda_stream)
            torch.cuda.synchronize()
        want, e = expected_append(x[:, :heads].cpu(), torch.arange(12, 16), dim, 10.0 ** (1 + i % 7), None, 0.0)
        for got in q:
            assert ((got.double().cpu() - want).abs() <= e + half_step("bf16") * (want.abs() + e)).all()
        paged.close()


def test_a_new_norm_weight_is_there_at_once(engine):
    """Append on a stream that waits for nobody, right behind the weight's making."""
    heads, dim = 1, 256
    g = torch.Generator().manual_seed(41)
    x = torch.randn((1, heads + 2, dim), generator=g).cuda()
    k, v = (torch.zeros((1, 1, 16, dim), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    stream, base = torch.cuda.Stream(), x.data_ptr()
    paged = S.PagedAttention(engine, heads, 1, dim, 1, page_tokens=16, max_sequences=1, max_rows=1, max_context=16)
    paged.batch([1], [1], np.zeros((1, 1), np.int32), stream=stream.cuda_stream)
    for i in range(40):
        weight = (1.0 + 0.2 * torch.randn(dim, generator=g)).to(torch.bfloat16)
        q = torch.zeros((1, heads, dim), device="cuda", dtype=torch.bfloat16)
        torch.cuda.synchronize()
        norm = engine.tensor_vector(bf16_bits(weight))
        paged.append(base, base + 4 * dim, base + 8 * dim, q.data_ptr(), k.data_ptr(), v.data_ptr(), ld=(heads + 2) * dim, q_norm=norm, k_norm=norm, stream=stream.cuda_stream)
        torch.cuda.synchronize()
        engine.tensor_destroy(norm)
        want, e = expected_append(x[:, :heads].cpu(), torch.zeros(1), 0, 1.0, weight, engine.g.eps)
        assert ((q.double().cpu() - want).abs() <= e + half_step("bf16") * (want.abs() + e)).all()
    paged.close()


@pytest.mark.parametrize("behind", ["attention", "sampling", "torch", "nothing"])
def test_a_batch_set_on_another_stream_with_events_between(engine, behind):
    """The batch's copies lie behind a long wait on a stream of their own; attention on another stream, behind an event and behind a kernel of that stream, goes by the new batch: its blocks read
    their range, pages and first tiles ahead of the kernel in front of them, never ahead of the event."""
    heads, kv_heads, dim, pages = 8, 2, 128, 48
    scenes = [Scene(60 + i, heads, kv_heads, dim, [1, 2, 1], lengths, page_tokens=32, spare_pages=pages - sum(-(-n // 32) for n in lengths)) for i, lengths in enumerate(([300, 33, 500], [41, 600, 2]))]
    def new():
        return S.PagedAttention(engine, heads, kv_heads, dim, pages, page_tokens=32, scale=scenes[0].scale, max_sequences=3, max_rows=4, max_context=700)
    paged, other = new(), new()
    want = [attend(engine, scene, "f32", paged=paged) for scene in scenes]      # (both batches have been set once: all tables hold valid numbers)
    other.batch(scenes[0].rows, scenes[0].lengths, scenes[0].table)
    out, side = torch.zeros((20, 4, heads, dim), device="cuda"), torch.zeros((4, heads, dim), device="cuda")
    uniform, ids = torch.full((4,), 0.5, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    engine.pass_wait()
    setting, running = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for n in range(20):
        scene = scenes[n % 2]
        with torch.cuda.stream(setting):
            torch.cuda._sleep(400_000)
        paged.batch(scene.rows, scene.lengths, scene.table, stream=setting.cuda_stream)
        if behind == "attention":
            other.attend(scenes[0].dq.data_ptr(), scenes[0].k.data_ptr(), scenes[0].v.data_ptr(), side.data_ptr(), out_dtype="f32", stream=running.cuda_stream)
        elif behind == "sampling":
            engine.pass_sample(side.data_ptr(), 4, heads * dim, heads * dim, ids.data_ptr(), uniform.data_ptr(), stream=running.cuda_stream)
        elif behind == "torch":
            with torch.cuda.stream(running):
                side.add_(1.0)
        running.wait_stream(setting)
        paged.attend(scene.dq.data_ptr(), scene.k.data_ptr(), scene.v.data_ptr(), out[n].data_ptr(), out_dtype="f32", stream=running.cuda_stream)
        setting.wait_stream(running)
    torch.cuda.synchronize()
    engine.pass_wait()
    for n in range(20):
        assert torch.equal(out[n], want[n % 2]), n
