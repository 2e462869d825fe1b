"""Attention of sequences that begin with the same pages: against plain 64-bit implementations, and against batches without groups."""
import numpy as np
import pytest
import torch

import splosh_b200 as S
from more_reference import Scene, check
from paged_reference import TYPES
from splosh_b200.paged import debug_paged_plan_shared
from test_gpu_paged_e4m3 import attend, engine      # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


def joint(scene):
    return debug_paged_plan_shared(scene.rows, scene.lengths, scene.groups, heads=scene.heads, kv_heads=scene.kv_heads, head_dim=scene.head_dim, pages=1, page_tokens=256, window=scene.window,
                                   causal=scene.causal, dtype=scene.dtype, max_sequences=len(scene.rows), max_rows=scene.total, max_context=1 << 20)[4]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "e4m3"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(24, 4, 256), (8, 8, 128), (16, 2, 64), (64, 1, 128)])
@pytest.mark.parametrize("out_dtype", ["same", "f32"])
def test_types_and_head_shapes(engine, dtype, heads, kv_heads, head_dim, out_dtype):
    shared = 8192 if kv_heads == 1 else 2560
    scene = Scene(heads + head_dim, heads, kv_heads, head_dim, [1, 2, 1, 0, 1, 1, 2, 1, 1, 1, 1, 2], [shared + 1 + 37 * i + 2 for i in range(12)], page_tokens=64, dtype=dtype, groups=[(12, shared)])
    assert joint(scene)
    out = scene.q_type if out_dtype == "same" else "f32"
    check(scene, attend(engine, scene, out), out)


@pytest.mark.parametrize("rows", [1, 3, 6, 16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_blocks_of_rows_that_straddle_two_units(engine, rows, causal, dtype):
    shared = {1: 4096, 3: 8192, 6: 20480, 16: 8192}[rows]
    scene = Scene(rows, 12, 2, 128, [rows] * 20, [shared + rows + 11 * i for i in range(20)], page_tokens=128, dtype=dtype, causal=causal, groups=[(20, shared)])
    assert joint(scene)
    check(scene, attend(engine, scene, "f32"), "f32")


@pytest.mark.parametrize("dtype", ["fp16", "e4m3"])
def test_several_groups_prompts_among_them_and_sequences_of_their_own(engine, dtype):
    """Two groups that are worth it, one of a single sequence, one whose prefix is too short, a group with a prompt in its middle, and two sequences without one."""
    rows = [1] * 10 + [2] * 6 + [1] + [1, 1] + [1, 1, 1, 1, 1, 40, 1, 1, 1, 1, 1] + [1, 30]
    groups = [(10, 1600), (6, 1280), (1, 640), (2, 64), (11, 1920)]
    shared = sum(([t] * n for n, t in groups), []) + [0, 0]
    lengths = [t + r + (53 * i) % 400 for i, (t, r) in enumerate(zip(shared, rows))]
    scene = Scene(77, 24, 4, 128, rows, lengths, page_tokens=64, dtype=dtype, layout="token", groups=groups)
    assert joint(scene)
    check(scene, attend(engine, scene, "f32"), "f32")


@pytest.mark.parametrize("rows,heads,kv_heads,shared", [(1, 8, 2, 8192), (1, 12, 2, 8192), (2, 8, 8, 4096), (4, 24, 4, 8192), (6, 24, 4, 20480), (5, 8, 2, 20480), (8, 32, 4, 8192)])
@pytest.mark.parametrize("head_dim", [128, 256])
def test_both_forms_over_a_cache_of_e4m3(engine, rows, heads, kv_heads, shared, head_dim):
    """Four to 64 packed rows a sequence, two to nine sequences: joint rows of 16, 32, 48 and 128 a block, full and not."""
    for n in (2, 5, 9):
        scene = Scene(rows + n, heads, kv_heads, head_dim, [rows] * n, [shared + rows + 77 * i for i in range(n)], page_tokens=64, dtype="e4m3", groups=[(n, shared)])
        if joint(scene):
            check(scene, attend(engine, scene, "f32"), "f32")
    assert joint(scene)


def test_a_window_leaves_a_prefix_to_each_sequence(engine):
    scene = Scene(4, 8, 2, 128, [1] * 12, [1024 + 1 + 9 * i for i in range(12)], page_tokens=64, dtype="bf16", window=1000, groups=[(12, 1024)])
    assert not joint(scene)
    check(scene, attend(engine, scene, "f32"), "f32")


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_rows_whose_weight_lies_on_one_side(engine, dtype):
    """Rows whose prefix has all the weight and rows whose own tokens have: the joining goes by the largest score of both."""
    scene = Scene(6, 8, 2, 128, [2] * 16, [4096 + 2 + 17 * i for i in range(16)], page_tokens=128, dtype=dtype, groups=[(16, 4096)])
    assert joint(scene)
    scene.q = (scene.q.float() * torch.tensor([20.0, 0.01, 5.0, 1.0] * 8)[:, None, None]).to(TYPES[scene.q_type])
    scene.dq.copy_(scene.q)
    check(scene, attend(engine, scene, "f32"), "f32")


def test_runs_are_equal_to_the_bit(engine):
    for dtype in ("bf16", "e4m3"):
        scene = Scene(2, 24, 4, 256, [1] * 9 + [8] * 3, [4608 + 8 + 100 * i for i in range(12)], page_tokens=256, dtype=dtype, groups=[(12, 4608)])
        assert joint(scene)
        first = attend(engine, scene)
        paged = scene.paged(engine, S.PagedAttention)
        for stream in (None, torch.cuda.Stream().cuda_stream, 0):
            assert torch.equal(first, attend(engine, scene, stream=stream)) and torch.equal(first, attend(engine, scene, stream=stream, paged=paged))


@pytest.mark.parametrize("dtype,each,long,longer", [("bf16", 1, 2048, 2944), ("e4m3", 1, 2048, 2944), ("e4m3", 8, 6144, 8192), ("e4m3", 30, 6528, 8192)])
def test_graphs_captured_with_groups_and_without_follow_any_batch(engine, dtype, each, long, longer):
    """One object, a graph captured before any group, one captured with a prefix met together: both replayed behind batches of either kind."""
    rows, pages = [each] * 12, 290
    def make(i, shared, groups):
        own = [shared + each + (31 * (n + i)) % 300 for n in range(12)]
        held = sum(-(-n // 64) for n in own) - (shared // 64 * 11 if groups else 0)
        return Scene(40 + i, 12, 4, 128, rows, own, page_tokens=64, dtype=dtype, groups=[(12, shared)] if groups else [], spare_pages=pages - held)
    scenes = [make(0, 256, False), make(1, long, True), make(2, 256, False), make(3, longer, True), make(4, 64, True)]
    assert [joint(s) for s in scenes] == [False, True, False, True, False]
    paged = scenes[0].paged(engine, S.PagedAttention, max_context=longer + 512)
    q, k, v, ks, vs = (torch.empty_like(x) for x in (scenes[0].dq, scenes[0].k, scenes[0].v, scenes[0].ks, scenes[0].vs))
    out = torch.zeros((2, 12 * each, 12, 128), device="cuda")
    scales = {"k_scale": ks.data_ptr(), "v_scale": vs.data_ptr()} if dtype == "e4m3" else {}
    stream = torch.cuda.Stream()
    graphs = []
    for n in range(2):
        paged.batch(rows, scenes[n].lengths, scenes[n].table, stream=stream.cuda_stream, groups=scenes[n].groups)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            paged.attend(q.data_ptr(), k.data_ptr(), v.data_ptr(), out[n].data_ptr(), out_dtype="f32", stream=stream.cuda_stream, **scales)
        graphs.append(graph)
    for scene in scenes:
        with torch.cuda.stream(stream):
            q.copy_(scene.dq); ks.copy_(scene.ks); vs.copy_(scene.vs)
            k.view(torch.uint8).copy_(scene.k.view(torch.uint8)); v.view(torch.uint8).copy_(scene.v.view(torch.uint8))
            paged.batch(rows, scene.lengths, scene.table, stream=stream.cuda_stream, groups=scene.groups)
            for graph in graphs:
                graph.replay()
        stream.synchronize()
        for n in range(2):
            check(scene, out[n], "f32")


def test_batches_of_either_kind_one_after_the_other_without_waits(engine):
    scenes = [Scene(50 + i, 8, 2, 128, [1] * 16, [shared + 1 + (13 * n) % 200 for n in range(16)], page_tokens=32, dtype="bf16", groups=[(16, shared)] if shared else [], spare_pages=900)
              for i, shared in enumerate((2048, 0, 1536))]
    paged = scenes[0].paged(engine, S.PagedAttention, max_context=4096, page_tokens=32)
    big = max(s.pages for s in scenes)
    paged = S.PagedAttention(engine, 8, 2, 128, big, page_tokens=32, scale=scenes[0].scale, max_sequences=16, max_rows=16, max_context=4096)
    out = torch.zeros((12, 16, 8, 128), device="cuda")
    torch.cuda.synchronize()
    for n in range(12):
        s = scenes[n % 3]
        paged.batch(s.rows, s.lengths, s.table, groups=s.groups)
        paged.attend(s.dq.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), out[n].data_ptr(), out_dtype="f32")
    engine.pass_wait()
    for n in range(12):
        check(scenes[n % 3], out[n], "f32")


def test_a_group_that_is_refused_leaves_the_batch(engine):
    scene = Scene(3, 4, 2, 128, [1] * 8, [256 + 10 + i for i in range(8)], page_tokens=64, dtype="bf16", groups=[(8, 256)])
    paged = scene.paged(engine, S.PagedAttention)
    want = attend(engine, scene, "f32", paged=paged)
    table = scene.table.copy()
    table[3, 1] = scene.table[0, 2]
    for bad, t in (([(8, 100)], scene.table), ([(9, 256)], scene.table), ([(8, 320)], scene.table), ([(8, 256)], table), ([(-1, 256)], scene.table), ([(8, -64)], scene.table)):
        with pytest.raises(S.EngineError) as caught:
            paged.batch(scene.rows, scene.lengths, t, groups=bad)
        assert caught.value.case == "invalidRows"
    out = torch.zeros_like(want)
    paged.attend(scene.dq.data_ptr(), scene.k.data_ptr(), scene.v.data_ptr(), out.data_ptr(), out_dtype="f32")
    engine.pass_wait()
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("each,shared", [(1, 8192), (8, 12288), (30, 8192)])
def test_a_key_that_is_no_number_in_a_prefix_reaches_who_sees_it(engine, dtype, each, shared):
    """Keys of the first kv head of one token, and of all tokens: the rows' heads on it are NaN, those on the second are not."""
    scene = Scene(9, 6, 2, 128, [each] * 12, [shared + each + 19 * i for i in range(12)], page_tokens=64, dtype=dtype, groups=[(12, shared)])
    assert joint(scene)
    k = scene.k.view(torch.uint8) if dtype == "e4m3" else scene.k
    for pages in (scene.table[0, 3:4], scene.table[:, :]):
        pages = torch.from_numpy(np.unique(pages[pages >= 0])).cuda().long()
        k[pages, 0, 5 if len(pages) == 1 else slice(None), 7] = 0x7f if dtype == "e4m3" else float("nan")
        out = attend(engine, scene, "f32")
        assert torch.isnan(out[:, :3]).all() and torch.isfinite(out[:, 3:]).all()
