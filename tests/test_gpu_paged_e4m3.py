"""The paged cache of e4m3: append and attention against plain 64-bit implementations, over head layouts, page sizes, lengths from one token on, windows, prompts and chunks, graphs and streams.
What may not be read is NaN, codes and scales."""
import numpy as np
import pytest
import torch

import splosh_b200 as S
from helpers import observed
from more_reference import E4M3, LARGEST, SCALE_MIN, Scene, check
from paged_reference import TYPES, half_step
from test_gpu_paged import bf16_bits, expected_append

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    e = S.Engine(S.tiny_geometry(), S.EngineConfig(max_slots=1, max_rows=64, kv_pages=4, max_context=512))
    yield e
    e.close()


def attend(engine, scene, out_dtype=None, stream=None, paged=None):
    paged = paged or scene.paged(engine, S.PagedAttention)
    out = torch.full((scene.total + 1, scene.heads, scene.head_dim), 7.0, device="cuda", dtype=TYPES[out_dtype or scene.q_type])
    torch.cuda.synchronize()
    paged.batch(scene.rows, scene.lengths, scene.table, stream=stream, groups=scene.groups)
    paged.attend(scene.dq.data_ptr(), scene.k.data_ptr(), scene.v.data_ptr(), out.data_ptr(), out_dtype=out_dtype, stream=stream, **scene.scales())
    engine.pass_wait()
    torch.cuda.synchronize()
    assert (out[scene.total:] == 7.0).all()              # rows behind the last sequence stay
    return out[:scene.total]


@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 128), (24, 4, 256), (6, 6, 64), (16, 1, 128), (5, 1, 64), (12, 2, 256), (32, 1, 64), (64, 1, 128)])
@pytest.mark.parametrize("out_dtype", ["bf16", "f32"])
def test_head_shapes(engine, heads, kv_heads, head_dim, out_dtype):
    scene = Scene(heads + head_dim, heads, kv_heads, head_dim, [1, 0, 7, 3], [1, 40, 150, 301])
    worst = check(scene, attend(engine, scene, out_dtype), out_dtype)
    observed(f"e4m3 attention {heads}/{kv_heads}/{head_dim} -> {out_dtype}: {worst:.2f} of the bound")


@pytest.mark.parametrize("page_tokens", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_page_sizes_and_layouts(engine, page_tokens, layout, head_dim):
    scene = Scene(page_tokens + head_dim, 4, 2, head_dim, [2, 1, 5], [page_tokens, page_tokens + 1, 3 * page_tokens - 1], page_tokens=page_tokens, layout=layout)
    check(scene, attend(engine, scene, "f32"), "f32")


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 511, 640, 1000])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_lengths_around_tiles_and_pages(engine, length, head_dim):
    scene = Scene(length, 4, 1, head_dim, [min(length, 3), 1], [length, length], page_tokens=64)
    check(scene, attend(engine, scene, "f32"), "f32")


@pytest.mark.parametrize("rows,lengths", [([130], [130]), ([301, 1, 1], [301, 77, 500]), ([97], [700]), ([33, 34, 35], [33, 99, 290]), ([16] * 9, [16 + 37 * i for i in range(9)])])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(6, 1, 256), (8, 2, 128), (3, 1, 64)])
def test_prompts_chunks_and_mixed_batches(engine, rows, lengths, heads, kv_heads, head_dim):
    scene = Scene(sum(lengths), heads, kv_heads, head_dim, rows, lengths, page_tokens=16, layout="token")
    check(scene, attend(engine, scene, "f32"), "f32")


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("count,around", [(149, 256), (200, 300), (40, 1000), (300, 20)])
def test_blocks_of_several_tiles_and_pieces(engine, head_dim, count, around):
    lengths = [around] * count if around == 256 else [around + (37 * i) % around for i in range(count)]
    scene = Scene(count, 2, 1, head_dim, [1 + i % 2 for i in range(count)], lengths, page_tokens=64)
    check(scene, attend(engine, scene, "f32"), "f32")
    again = attend(engine, scene, "f32")
    for _ in range(5):
        assert torch.equal(attend(engine, scene, "f32"), again)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 129, 300])
@pytest.mark.parametrize("causal", [True, False])
def test_windows_and_blocks_that_see_themselves(engine, window, causal):
    scene = Scene(window, 8, 2, 128, [16, 1, 40], [300, 150, 40], page_tokens=32, causal=causal, window=window)
    check(scene, attend(engine, scene, "f32"), "f32")


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("page_tokens", [16, 64, 256])
@pytest.mark.parametrize("window", [64, 65, 96, 128, 200])
def test_windows_that_begin_anywhere_in_a_tile(engine, head_dim, page_tokens, window):
    """Everything in front of the window is NaN, codes and scales."""
    lengths = [256, 300, 129, 192]
    scene = Scene(window + page_tokens, 2, 1, head_dim, [1] * 4, lengths, page_tokens=page_tokens, window=window)
    for s, length in enumerate(lengths):
        for token in range(length - window):
            at = (int(scene.table[s, token // page_tokens]), slice(None), token % page_tokens)
            for codes, scales in ((scene.k, scene.ks), (scene.v, scene.vs)):
                codes.view(torch.uint8)[at] = 0x7f; scales[at] = float("nan") if token % 2 else float("inf")
    check(scene, attend(engine, scene, "f32"), "f32")


@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_long_contexts_of_few_rows(engine, head_dim):
    scene = Scene(9, 4, 1, head_dim, [1, 4], [9001, 5000], page_tokens=128)
    check(scene, attend(engine, scene, "f32"), "f32")


def test_scores_far_apart_and_a_maximum_that_keeps_rising(engine):
    """Keys that grow with the position raise a row's maximum tile after tile; most probabilities vanish."""
    scene = Scene(3, 4, 2, 128, [4, 200], [900, 700], page_tokens=64)
    for s, (_, k_scale, _, _) in enumerate(scene.tokens):
        factor = torch.linspace(0.1, 12.0, k_scale.shape[0]).double()
        k_scale.copy_((k_scale * factor[:, None]).float().double())
        for i in range(-(-k_scale.shape[0] // 64)):
            part = k_scale[i * 64:(i + 1) * 64]
            scene.ks[scene.table[s, i], :, :part.shape[0]] = part.transpose(0, 1).float().cuda()
    check(scene, attend(engine, scene, "f32"), "f32")


def test_values_of_very_different_sizes(engine):
    """Scales of values that span many powers of two, scales of zero among them: every row's own largest products count, whatever others' are."""
    scene = Scene(8, 4, 2, 128, [3, 60, 1], [300, 200, 1000], page_tokens=32)
    g = torch.Generator().manual_seed(5)
    for s, (_, _, _, v_scale) in enumerate(scene.tokens):
        v_scale.copy_((v_scale * torch.exp2(8.0 * torch.randn(v_scale.shape, generator=g, dtype=torch.float64))).float().double())
        v_scale[::7] = 0.0
        for i in range(-(-v_scale.shape[0] // 32)):
            part = v_scale[i * 32:(i + 1) * 32]
            scene.vs[scene.table[s, i], :, :part.shape[0]] = part.transpose(0, 1).float().cuda()
    check(scene, attend(engine, scene, "f32"), "f32")


def test_value_scales_out_of_range(engine):
    """Negative ones and those above 2^40 are no numbers for whoever sees their token; at 2^40 and beside zeros all is as defined, and the smallest count as 2^-60."""
    scene = Scene(9, 4, 2, 128, [140], [140], page_tokens=64)
    good = attend(engine, scene, "f32")
    for value in (-1.0, -1e-30, 1.1e12, float("inf")):
        scene.vs[scene.table[0, 1], 0, 6] = value               # token 70 of the first kv head
        out = attend(engine, scene, "f32")
        assert out[70:, :2].isnan().all() and torch.equal(out[:, 2:], good[:, 2:])
    for value, as_if in ((2.0 ** 40, 2.0 ** 40), (0.0, 2.0 ** -60), (1e-38, 2.0 ** -60), (2.0 ** -61, 2.0 ** -60)):
        scene.vs[scene.table[0, 1], 0, 6] = value
        scene.tokens[0][3][70, 0] = as_if
        check(scene, attend(engine, scene, "f32"), "f32")
    scene.vs[scene.vs.isfinite()] = 0.0
    scene.tokens[0][3][:] = 2.0 ** -60
    check(scene, attend(engine, scene, "f32"), "f32")


def test_queries_of_very_different_sizes(engine):
    """Rows of tiny, of large and of no queries at all; a channel far above the others."""
    scene = Scene(8, 4, 2, 256, [8, 8], [200, 150], page_tokens=32)
    factor = torch.tensor([1e-30, 1e-10, 1e-3, 0.0, 1.0, 3.0, 1e-38, 1e-20] * 2)[:, None, None]
    scene.q = (scene.q.float() * factor).to(torch.bfloat16)
    scene.q[4, 1, 17], scene.q[5, 0, 3] = 30.0, -50.0
    scene.dq.copy_(scene.q)
    check(scene, attend(engine, scene, "f32"), "f32")


def test_what_is_no_number_in_a_token_that_is_seen_shows(engine):
    """A NaN in one key, value or scale reaches the rows that see it, in any place of a tile; in a query its row alone."""
    for place in (0, 1, 2, 3, 67, 130):
        for which in ("k", "v", "ks", "vs"):
            scene = Scene(place, 2, 1, 128, [140], [140], page_tokens=64)
            at = (int(scene.table[0, place // 64]), 0, place % 64)
            if which in "kv":
                getattr(scene, which).view(torch.uint8)[at + (5,)] = 0x7f
            else:
                getattr(scene, which)[at] = float("nan")
            out = attend(engine, scene, "f32")
            assert out[place:].isnan().any(-1).all(), which
            if which in ("k", "ks"):
                assert not out[:place].isnan().any(), which
    scene = Scene(1, 2, 1, 128, [4], [300], page_tokens=64)
    scene.dq[1, 0, 9] = float("nan"); scene.dq[2, 1, 100] = float("inf")
    out = attend(engine, scene, "f32")
    assert out[1, 0].isnan().all() and out[2, 1].isnan().all()
    scene.q[1, 0], scene.q[2, 1] = 0.0, 0.0
    scene.dq.copy_(scene.q)
    good = attend(engine, scene, "f32")
    rest = torch.ones((4, 2), dtype=torch.bool); rest[1, 0] = rest[2, 1] = False
    assert torch.equal(out[rest], good[rest])


def test_strides_of_a_cache_that_holds_keys_and_values_side_by_side(engine):
    scene = Scene(11, 4, 2, 128, [3, 1], [90, 33], page_tokens=32)
    wide = torch.full((scene.pages, 3, 2, 32, 128 + 16), 0x7f, device="cuda", dtype=torch.uint8)
    wide[:, 1, :, :, :128], wide[:, 2, :, :, :128] = scene.k.view(torch.uint8), scene.v.view(torch.uint8)
    paged = S.PagedAttention(engine, 4, 2, 128, scene.pages, page_tokens=32, dtype="e4m3", strides=(wide.stride(0), wide.stride(2), wide.stride(3)), max_sequences=2, max_rows=4, max_context=96)
    scene.k, scene.v = wide[:, 1], wide[:, 2]
    check(scene, attend(engine, scene, paged=paged), "bf16")


def test_a_cache_past_two_to_the_31_bytes(engine):
    """Pages whose codes lie beyond what 32 bits of offset reach."""
    scene = Scene(13, 8, 2, 256, [2, 1], [300, 200], page_tokens=256)
    pages, token, head = 5000, 256, 256 * 256
    page = 2 * head + (1 << 19)                              # 655,360 bytes apart
    assert (pages - 1) * page > 2 ** 31
    move = np.linspace(pages - 1, pages - 2 - scene.pages, scene.pages).astype(np.int64)
    big = [torch.zeros(pages * page, device="cuda", dtype=torch.uint8) for _ in range(2)]
    scales = [torch.full((pages, 2, 256), float("nan"), device="cuda") for _ in range(2)]
    for cache, wide in ((scene.k, big[0]), (scene.v, big[1])):
        wide.view(pages, page)[torch.from_numpy(move).cuda(), :2 * head] = cache.view(torch.uint8).reshape(scene.pages, -1)
    for one, wide in ((scene.ks, scales[0]), (scene.vs, scales[1])):
        wide[torch.from_numpy(move).cuda()] = one
    scene.table = np.where(scene.table >= 0, move[np.maximum(scene.table, 0)], -1).astype(np.int32)
    scene.k, scene.v, scene.ks, scene.vs = *big, *scales
    paged = S.PagedAttention(engine, 8, 2, 256, pages, page_tokens=256, dtype="e4m3", strides=(page, head, token), max_sequences=2, max_rows=3, max_context=300)
    check(scene, attend(engine, scene, "f32", paged=paged), "f32")


def test_runs_are_equal_to_the_bit_and_streams_do_not_matter(engine):
    scene = Scene(2, 24, 4, 256, [1, 8, 50], [3000, 777, 50], page_tokens=256)
    first = attend(engine, scene)
    side = torch.cuda.Stream()
    for stream in (None, side.cuda_stream, 0):
        assert torch.equal(first, attend(engine, scene, stream=stream))


def test_a_captured_graph_follows_the_batch(engine):
    """The graph of a decode step, append and attention, replayed with longer sequences in other pages."""
    scenes = [Scene(30 + i, 8, 2, 128, [1, 2], lengths, page_tokens=32, spare_pages=40 - sum(-(-n // 32) for n in lengths)) for i, lengths in enumerate(([40, 33], [41, 600], [1, 2]))]
    paged = S.PagedAttention(engine, 8, 2, 128, 40, page_tokens=32, dtype="e4m3", scale=scenes[0].scale, max_sequences=2, max_rows=3, max_context=700)
    q, k, v, ks, vs = (torch.empty_like(x) for x in (scenes[0].dq, scenes[0].k, scenes[0].v, scenes[0].ks, scenes[0].vs))
    out = torch.zeros((3, 8, 128), device="cuda", dtype=torch.bfloat16)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    paged.batch(scenes[0].rows, scenes[0].lengths, scenes[0].table, stream=stream.cuda_stream)
    with torch.cuda.graph(graph, stream=stream):
        paged.attend(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), stream=stream.cuda_stream, k_scale=ks.data_ptr(), v_scale=vs.data_ptr())
    for scene in scenes:
        with torch.cuda.stream(stream):
            q.copy_(scene.dq); k.view(torch.uint8).copy_(scene.k.view(torch.uint8)); v.view(torch.uint8).copy_(scene.v.view(torch.uint8)); ks.copy_(scene.ks); vs.copy_(scene.vs)
            paged.batch(scene.rows, scene.lengths, scene.table, stream=stream.cuda_stream)
            graph.replay()
        stream.synchronize()
        check(scene, out, "bf16")


@pytest.mark.parametrize("page_tokens", [16, 256])
def test_steps_without_a_wait_between_them(engine, page_tokens):
    """Batch, append and attend queued one after the other, several sequences growing and leaving: what a step without waits reads is what the step before wrote, to the bit."""
    heads, kv_heads, dim, steps, pages = 8, 2, 128, 24, 3 * (-(-400 // page_tokens))
    g = torch.Generator().manual_seed(page_tokens)
    x = torch.randn((steps, 2, 3, heads + 2 * kv_heads, dim), generator=g).cuda()
    table = torch.randperm(pages, generator=g).numpy().astype(np.int32).reshape(3, -1)
    start = torch.randn((2, pages, kv_heads, page_tokens, dim), generator=g).to(E4M3).cuda()

    def run(wait):
        paged = S.PagedAttention(engine, heads, kv_heads, dim, pages, page_tokens=page_tokens, dtype="e4m3", rotary_dim=64, rope_theta=1e4, max_sequences=3, max_rows=3, max_context=400)
        k, v = start[0].view(torch.uint8).clone(), start[1].view(torch.uint8).clone()
        ks, vs = (torch.full((pages, kv_heads, page_tokens), 0.01, device="cuda") for _ in range(2))
        q, out = (torch.zeros((steps, 2, 3, heads, dim), device="cuda", dtype=torch.bfloat16) for _ in range(2))
        torch.cuda.synchronize()
        scales = {"k_scale": ks.data_ptr(), "v_scale": vs.data_ptr()}
        for step in range(steps):
            lengths = [1 + step, 120 + step, (300 if step % 2 else 5) + step]
            paged.batch([1, 1, 1], lengths, table)
            for layer in range(2):                        # of one cache: the second writes what the first has read
                row = x[step, layer].data_ptr()
                paged.append(row, row + 4 * heads * dim, row + 4 * (heads + kv_heads) * dim, q[step, layer].data_ptr(), k.data_ptr(), v.data_ptr(), ld=(heads + 2 * kv_heads) * dim, **scales)
                paged.attend(q[step, layer].data_ptr(), k.data_ptr(), v.data_ptr(), out[step, layer].data_ptr(), **scales)
                if wait:
                    engine.pass_wait()
        engine.pass_wait()
        torch.cuda.synchronize()
        return out, k, v, ks, vs

    for a, b in zip(run(True), run(False)):
        assert torch.equal(a, b)


# ---- append --------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 128), (24, 4, 256), (3, 3, 64), (1, 1, 64), (40, 8, 128)])
@pytest.mark.parametrize("rotary", [0, 6, "quarter", "whole"])
@pytest.mark.parametrize("source,norm,layout", [("f32", True, "head"), ("f32", False, "token"), ("fp16", False, "head"), ("bf16", True, "token")])
def test_append(engine, heads, kv_heads, head_dim, rotary, source, norm, layout):
    """Queries as in a 16-bit cache. Of keys and values y: the scale is max |y| / 448 to the arithmetic's error and two roundings; a code times its scale is within half a step of e4m3 (2^-4 of the value, or 2^-10 of the
    scale below the smallest normal code) of y, and the arithmetic's error."""
    rotary = {"quarter": head_dim // 4, "whole": head_dim}.get(rotary, rotary)
    rows, lengths, page, theta = [1, 0, 5, 20], [200001, 9, 5, 60], 32, 1e6
    g = torch.Generator().manual_seed(heads + head_dim + rotary)
    total, pages = sum(rows), 8
    table = np.full((4, -(-200001 // page)), 0, np.int32)
    table[0, 200000 // page] = 5
    table[1, 0], table[2, 0], table[3, :2] = 6, 1, (4, 2)
    width = heads + 2 * kv_heads
    x = torch.randn((total, width + 1, head_dim), generator=g)
    x[3, heads:] *= 1e-6                                       # a small token, and one of nothing
    x[4, heads:] = 0.0
    x = x.to(TYPES[source])
    wq, wk = ((1.0 + 0.2 * torch.randn(head_dim, generator=g)).to(torch.bfloat16) for _ in range(2))
    shape = (pages, kv_heads, page, head_dim) if layout == "head" else (pages, page, kv_heads, head_dim)
    k, v = (torch.full(shape, 0x41, device="cuda", dtype=torch.uint8) for _ in range(2))
    ks, vs = (torch.full((pages, kv_heads, page), 3.0, device="cuda") for _ in range(2))
    q = torch.full((total + 1, heads, head_dim), 3.0, device="cuda", dtype=torch.bfloat16)
    dx = x.cuda()
    paged = S.PagedAttention(engine, heads, kv_heads, head_dim, pages, page_tokens=page, dtype="e4m3", layout=layout, rotary_dim=rotary, rope_theta=theta, max_sequences=4, max_rows=total, max_context=200001)
    norms = [engine.tensor_vector(bf16_bits(w)) for w in (wq, wk)] if norm else [None, None]
    torch.cuda.synchronize()
    paged.batch(rows, lengths, table)
    size, base = x.element_size(), dx.data_ptr()
    paged.append(base, base + size * heads * head_dim, base + size * (heads + kv_heads) * head_dim, q.data_ptr(), k.data_ptr(), v.data_ptr(), dtype=source, ld=(width + 1) * head_dim,
                 q_norm=norms[0], k_norm=norms[1], k_scale=ks.data_ptr(), v_scale=vs.data_ptr())
    engine.pass_wait()
    for t in norms:
        if t:
            engine.tensor_destroy(t)
    sequence = np.repeat(np.arange(4), rows)
    position = np.concatenate([np.arange(n - r, n) for r, n in zip(rows, lengths)])
    want = [expected_append(x[:, a:b], torch.from_numpy(position), r, theta, w if norm and w is not None else None, engine.g.eps)
            for a, b, r, w in ((0, heads, rotary, wq), (heads, heads + kv_heads, rotary, wk), (heads + kv_heads, width, 0, None))]
    page_of, slot_of = table[sequence, position // page], position % page
    touched = torch.zeros((pages, page), dtype=torch.bool)
    touched[page_of, slot_of] = True
    w, e = want[0]
    assert ((q[:total].cpu().double() - w).abs() <= e + half_step("bf16") * (w.abs() + e) + 2.0 ** -25).all() and (q[total:] == 3.0).all()
    for codes, scales, (w, e) in ((k, ks, want[1]), (v, vs, want[2])):
        codes, scales = (codes.cpu() if layout == "head" else codes.cpu().transpose(1, 2)), scales.cpu()
        assert (codes.transpose(1, 2)[~touched] == 0x41).all() and (scales.transpose(1, 2)[~touched] == 3.0).all()
        code, scale = codes[page_of, :, slot_of].view(E4M3).double(), scales[page_of, :, slot_of].double()
        exact = (w.abs().amax(-1) / LARGEST).clamp(min=SCALE_MIN)
        assert ((scale - exact).abs() <= e.amax(-1) / LARGEST + 2.0 ** -23 * exact).all()
        y, s = code * scale[..., None], scale[..., None]
        # (The quotient y / scale has two roundings of its own in front of the code's.)
        bound = e + 2.0 ** -23 * w.abs()
        assert ((y - w).abs() <= bound + torch.maximum(2.0 ** -4 * (w.abs() + bound), 2.0 ** -10 * s)).all()


def test_append_keeps_what_is_no_number(engine):
    """An infinity makes its head's codes or scale no number; a NaN stays one; the token's other heads do not notice."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn((2, 4, 128), generator=g)
    x[0, 1, 7], x[1, 3, 9] = float("inf"), float("nan")     # token 0's key, token 1's second value head
    dx = x.cuda()
    paged = S.PagedAttention(engine, 0 + 1, 1, 128, 1, page_tokens=16, dtype="e4m3", max_sequences=1, max_rows=2, max_context=16)
    k, v = (torch.zeros((1, 1, 16, 128), device="cuda", dtype=torch.uint8) for _ in range(2))
    ks, vs = (torch.zeros((1, 1, 16), device="cuda") for _ in range(2))
    q = torch.zeros((2, 1, 128), device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    paged.batch([2], [2], np.zeros((1, 1), np.int32))
    base = dx.data_ptr()
    paged.append(base, base + 512, base + 3 * 512, q.data_ptr(), k.data_ptr(), v.data_ptr(), ld=512, k_scale=ks.data_ptr(), v_scale=vs.data_ptr())
    engine.pass_wait()
    key = k.view(E4M3).float()[0, 0] * ks[0, 0, :, None]
    value = v.view(E4M3).float()[0, 0] * vs[0, 0, :, None]
    assert key[0].isnan().all() and not key[1].isnan().any()
    assert value[1, 9].isnan() and not value[0].isnan().any() and not value[1, :9].isnan().any()


def test_refusals(engine):
    def make(**more):
        args = dict(heads=4, kv_heads=2, head_dim=128, pages=8, page_tokens=32, dtype="e4m3", max_sequences=2, max_rows=4, max_context=128)
        return S.PagedAttention(engine, **{**args, **more})
    for bad in (dict(head_dim=96), dict(strides=(2 * 32 * 136, 32 * 136, 136)), dict(dtype="e5m2")):
        with pytest.raises(S.EngineError) as caught:
            make(**bad)
        assert caught.value.case == "invalidArgument", bad
    a = torch.zeros(1 << 16, device="cuda").data_ptr()
    paged, plain = make(), make(dtype="bf16")
    scales = {"k_scale": a, "v_scale": a}
    with pytest.raises(S.EngineError) as caught:
        paged.attend(a, a, a, a, **scales)
    assert "no batch" in str(caught.value)
    table = np.array([[0, 1], [2, 3]], np.int32)
    paged.batch([1, 1], [33, 20], table)
    plain.batch([1, 1], [33, 20], table)
    for call, word in ((lambda: paged.attend(a, a, a, a), "has scales"), (lambda: paged.append(a, a, a, a, a, a), "has scales"), (lambda: plain.attend(a, a, a, a, **scales), "no scales"),
                       (lambda: plain.append(a, a, a, a, a, a, **scales), "no scales"), (lambda: paged.attend(a, a, a, a, k_scale=a), ""), (lambda: paged.append(a, a, a, a, a, a, v_scale=a), ""),
                       (lambda: paged.attend(a, a, a, a, k_scale=a + 4, v_scale=a), "16-byte"), (lambda: paged.append(a, a, a, a, a, a, k_scale=a, v_scale=a + 8), "16-byte"),
                       (lambda: paged.attend(a, a + 8, a, a, **scales), "16-byte"), (lambda: paged.attend(a, a, a, a, out_dtype="fp16", **scales), "queries' type"),
                       (lambda: paged.attend(a, a, a, a, out_dtype="e4m3", **scales), "queries' type"), (lambda: paged.append(a, a, a, a, a, a, dtype="e4m3", **scales), "rows are")):
        with pytest.raises(S.EngineError) as caught:
            call()
        assert caught.value.case == "invalidArgument" and word in str(caught.value)
    paged.batch([1, 1], [33, 20], np.array([[0, 1], [1, 3]], np.int32))
    with pytest.raises(S.EngineError) as caught:
        paged.append(a, a, a, a, a, a, **scales)
    assert "one page" in str(caught.value)
    paged.close()
    with pytest.raises(S.EngineError):
        paged.attend(a, a, a, a, **scales)
