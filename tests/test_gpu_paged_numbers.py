"""Attention over a paged cache where numbers end: what is no number in tokens whose pieces are joined, and scores near the ends of fp32. Wherever a sequence is cut, a row answers as in one piece."""
import pytest
import torch

from more_reference import Scene
from splosh_b200.paged import debug_paged_plan
from test_gpu_paged_e4m3 import attend, engine      # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


def spoil(scene, sequence, tokens, which, kv_head=0, channel=5):
    """NaN in keys or values (one channel of a code or number) or scales of these tokens of a sequence."""
    for token in tokens:
        at = (int(scene.table[sequence, token // scene.page_tokens]), kv_head, token % scene.page_tokens)
        if which in ("ks", "vs"):
            getattr(scene, which)[at] = float("nan")
        elif scene.dtype == "e4m3":
            getattr(scene, which).view(torch.uint8)[at + (channel,)] = 0x7f
        else:
            getattr(scene, which)[at + (channel,)] = float("nan")


def last_pieces(scene):
    """The first token of each (kv head, tile of rows)'s last piece of the first sequence, and how many it is cut into."""
    items = debug_paged_plan(scene.rows, scene.lengths, heads=scene.heads, kv_heads=scene.kv_heads, head_dim=scene.head_dim, pages=1, page_tokens=256, dtype=scene.dtype, max_sequences=len(scene.rows),
                             max_rows=scene.total, max_context=1 << 20)[1]
    items = items[items[:, 0] == 0]
    count = {}
    for it in items:
        key = tuple(it[2:4])
        count[key] = (max(count.get(key, (0, 0))[0], int(it[5])), count.get(key, (0, 0))[1] + 1)
    return count


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "e4m3"])
@pytest.mark.parametrize("heads,kv_heads,head_dim,rows,length", [
    (4, 1, 128, 1, 129), (4, 1, 128, 1, 257), (8, 2, 128, 1, 385), (24, 4, 256, 1, 1025), (2, 1, 64, 1, 129), (8, 1, 256, 1, 2177),        # up to eight packed rows: the newest token alone in the last piece
    (8, 2, 64, 2, 9001), (2, 1, 128, 4, 20000),
    (12, 2, 256, 3, 1300), (16, 1, 128, 4, 1300), (16, 1, 64, 1, 4097), (24, 4, 256, 8, 4000),                                              # nine to 128
    (6, 1, 256, 30, 8000), (8, 1, 128, 40, 3000), (4, 1, 64, 200, 5000)])                                                                  # more
def test_a_piece_of_tokens_that_are_no_numbers_is_not_lost(engine, dtype, heads, kv_heads, head_dim, rows, length):
    """All that a row sees in its last piece is NaN: the row is, and no other sequence or kv head."""
    scene = Scene(length + rows, heads, kv_heads, head_dim, [rows, 1], [length, 200], page_tokens=64, dtype=dtype)
    good = attend(engine, scene, "f32")
    pieces = last_pieces(scene)
    assert max(n for _, n in pieces.values()) > 1
    start = min(128 * tile for tile, _ in pieces.values())
    group = heads // kv_heads
    keep = {w: getattr(scene, w).view(torch.uint8).clone() for w in ("k", "v")}, scene.ks.clone(), scene.vs.clone()
    for which in ("k", "v") + (("ks", "vs") if dtype == "e4m3" else ()):
        for w in ("k", "v"):
            getattr(scene, w).view(torch.uint8).copy_(keep[0][w])
        scene.ks.copy_(keep[1]); scene.vs.copy_(keep[2])
        spoil(scene, 0, range(start, length), which)
        out = attend(engine, scene, "f32")
        sees = torch.arange(rows) + length - rows >= start
        assert sees.any()
        wrong = out[:rows][sees.cuda()][:, :group]
        assert (wrong[..., 5] if which == "v" else wrong).isnan().all(), which
        assert torch.equal(out[:rows, group:], good[:rows, group:]) and torch.equal(out[rows:], good[rows:])


@pytest.mark.parametrize("dtype,heads,kv_heads,head_dim,rows,length,shared", [
    ("e4m3", 8, 1, 128, 2, 2000, 0), ("e4m3", 24, 4, 256, 8, 8000, 0), ("e4m3", 16, 2, 64, 8, 8000, 0), ("e4m3", 24, 4, 256, 1, 4400, 4096), ("bf16", 24, 4, 256, 1, 4400, 4096), ("fp16", 16, 2, 64, 1, 4400, 4096),
    ("bf16", 4, 1, 128, 1, 2000, 0), ("bf16", 6, 1, 256, 30, 8000, 0)])
def test_a_value_that_is_no_number_in_a_piece_of_vanishing_weight(engine, dtype, heads, kv_heads, head_dim, rows, length, shared):
    """Scores of the first tile in hundreds: the other pieces' factors are 0, and 0 times NaN is none."""
    n = 12 if shared else 1
    scene = Scene(rows + length, heads, kv_heads, head_dim, [rows] * n, [length + 3 * i for i in range(n)], page_tokens=64, dtype=dtype, groups=[(n, shared)] if shared else ())
    pages = scene.table[0, :2].tolist()
    if dtype == "e4m3":
        scene.ks[pages] *= 400.0
    else:
        scene.k[pages] *= 400.0
    good = attend(engine, scene, "f32")
    assert good.isfinite().all()
    spoil(scene, 0, [length - rows], "v")
    out = attend(engine, scene, "f32")
    group = heads // kv_heads
    assert out[:rows, :group, 5].isnan().all()
    out[:rows, :group, 5] = good[:rows, :group, 5]
    assert torch.equal(out, good)


def aligned(scene, scale_of, query):
    """Every key of the first sequence is the same vector, every query that vector times `query`; the keys' scales are scale_of(token)."""
    heads, kv_heads, dim = scene.heads, scene.kv_heads, scene.head_dim
    g = torch.Generator().manual_seed(9)
    direction = torch.where(torch.rand(dim, generator=g) < 0.5, -1.0, 1.0)
    scene.q[:] = (query * direction).to(torch.bfloat16)
    scene.dq.copy_(scene.q)
    scene.k.view(torch.uint8).copy_(direction.to(torch.float8_e4m3fn).view(torch.uint8).cuda().expand(scene.k.shape))
    for token in range(scene.lengths[0]):
        scene.ks[int(scene.table[0, token // scene.page_tokens]), :, token % scene.page_tokens] = scale_of(token)


SHAPES = [(4, 1, 128, 1), (24, 4, 256, 1), (8, 2, 256, 4), (12, 1, 128, 4), (8, 1, 64, 1), (32, 2, 128, 5), (8, 1, 256, 40)]


def one_weight(engine, heads, kv_heads, head_dim, rows, length, best, query, least):
    """All scores far below zero (or above), one of them the largest by far: its token's value comes out, however the sequence is cut. The weight is exactly one, so the value is off by the roundings of its scale's
    reciprocal, of that one's and of the product with it: 2^-21 is more than these."""
    rows = min(rows, length)
    best = min(best, length - rows)
    scene = Scene(length, heads, kv_heads, head_dim, [rows], [length], page_tokens=64)
    # (Negative scores: the smallest scale's is the largest.)
    aligned(scene, lambda token: least if token == best else 4.0 * least if query < 0 else 0.25 * least, query)
    assert 1e30 < abs(query) * head_dim ** 0.5 * 1.44 * least and abs(query) * head_dim * 4.0 * least < 3.0e38
    out = attend(engine, scene, "f32").double().cpu()
    _, _, values, v_scale = scene.tokens[0]
    want = (values[best] * v_scale[best, :, None]).repeat_interleave(heads // kv_heads, 0)[None]
    assert ((out - want).abs() <= 2.0 ** -21 * want.abs()).all()


@pytest.mark.parametrize("heads,kv_heads,head_dim,rows", SHAPES)
@pytest.mark.parametrize("length,best", [(40, 0), (129, 128), (300, 130), (2000, 7), (2000, 1500)])
@pytest.mark.parametrize("query,least", [(-1.0, 1e30), (-1.0, 1e32), (1.0, 1e31)])
def test_scores_far_below_zero(engine, heads, kv_heads, head_dim, rows, length, best, query, least):
    one_weight(engine, heads, kv_heads, head_dim, rows, length, best, query, least)


@pytest.mark.parametrize("heads,kv_heads,head_dim,rows", SHAPES)
@pytest.mark.parametrize("length,best", [(40, 0), (300, 130), (2000, 1500)])
@pytest.mark.parametrize("query,least", [(-2.0 ** -20, 1e36), (2.0 ** -10, 1e36), (2.0 ** -20, 1e37)])
def test_scales_of_keys_near_the_end_of_fp32(engine, heads, kv_heads, head_dim, rows, length, best, query, least):
    """Keys whose scores with these queries are ordinary fp32 numbers, although their products with the queries' codes would not be."""
    one_weight(engine, heads, kv_heads, head_dim, rows, length, best, query, least)
