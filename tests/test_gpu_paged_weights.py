"""Attention over a cache of e4m3 where few tokens, or very many small ones, make a row: a weight counts with all of fp16's bits, in every form."""
import pytest
import torch

from more_reference import E4M3, Scene
from test_gpu_paged_e4m3 import attend, engine      # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu

SHAPES = [(4, 1, 128, 1), (24, 4, 256, 1), (6, 1, 64, 1), (12, 2, 256, 5), (16, 2, 128, 2), (56, 8, 256, 5), (40, 8, 128, 2), (8, 1, 128, 30)]


def within(scene, got):
    want, bound = scene.expected()
    error, bound = (got.double().cpu() - want).abs(), bound + 2.0 ** -24 * want.abs()
    assert (error <= bound).all(), f"{(error / bound).nan_to_num(0.0).max().item():.2f} of the bound"      # (a code of zero seen alone: none of none)


@pytest.mark.parametrize("heads,kv_heads,head_dim,rows", SHAPES)
@pytest.mark.parametrize("window", [0, 1, 2, 3])
def test_rows_that_see_few_tokens(engine, heads, kv_heads, head_dim, rows, window):
    """No sum of many roundings hides what one weight's is."""
    for seed in range(4):
        lengths = [rows + i for i in range(12)] if not window else [rows + 37 * i for i in range(12)]
        scene = Scene(100 * seed + rows + window, heads, kv_heads, head_dim, [rows] * 12, lengths, page_tokens=64, window=window, causal=seed % 2 == 0)
        within(scene, attend(engine, scene, "f32"))


@pytest.mark.parametrize("heads,kv_heads,head_dim,rows", SHAPES)
@pytest.mark.parametrize("below", [20.0, 23.3, 24.5, 26.5])
def test_many_tokens_of_small_weight_beside_a_large_one(engine, heads, kv_heads, head_dim, rows, below):
    """One token has 2^below times the weight of each of the others, and nothing in its values: what comes out is the others'."""
    length = 4000
    scene = Scene(rows, heads, kv_heads, head_dim, [rows], [length], page_tokens=64)
    g = torch.Generator().manual_seed(9)
    direction = torch.where(torch.rand(head_dim, generator=g) < 0.5, -1.0, 1.0)
    keys, k_scale, values, v_scale = scene.tokens[0]
    scene.q[:] = direction.to(torch.bfloat16)
    keys[:] = direction.double()
    v_scale[:] = 0.5
    values.abs_()
    values[1000] = 0.0
    # Scores are head_dim^0.5 times the keys' scales.
    k_scale[:] = 1.0
    k_scale[1000] = float(torch.tensor(1.0 + below * 0.6931471805599453 / head_dim ** 0.5))      # (an fp32 number, as the cache holds)
    scene.dq.copy_(scene.q)
    for page in range(-(-length // 64)):
        part, at = slice(64 * page, min(length, 64 * page + 64)), int(scene.table[0, page])
        count = part.stop - part.start
        scene.k[at, :, :count] = keys[part].transpose(0, 1).to(E4M3).cuda()
        scene.v[at, :, :count] = values[part].transpose(0, 1).to(E4M3).cuda()
        scene.ks[at, :, :count] = k_scale[part].transpose(0, 1).float().cuda()
        scene.vs[at, :, :count] = v_scale[part].transpose(0, 1).float().cuda()
    within(scene, attend(engine, scene, "f32"))
