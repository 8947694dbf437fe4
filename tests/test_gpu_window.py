"""Attention under a window with sinks against 64 bits: every kind of cache and
kernel, windows and sinks at the edges of blocks and stages, rows outside the
window that hold NaN and blocks outside it that are missing."""

import numpy as np
import pytest
import torch

from helpers import pkg
from span_oracle import CODE, Case

pytestmark = pytest.mark.gpu

ops = pkg("paged_ops")

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
STARTS = [0, 16, 63, 299, 1000, 1, 0, 5, 130, 500, 2100, 0]
COUNTS = [1, 1, 1, 1, 1, 1, 2, 33, 70, 200, 1, 90]
SHAPES = [(8, 2, 128, BF16, BF16), (8, 8, 64, FP16, FP16), (6, 2, 80, BF16, BF16), (6, 2, 96, FP16, FP16),
          (24, 1, 128, BF16, BF16), (9, 3, 64, BF16, BF16), (4, 2, 256, BF16, BF16), (4, 2, 64, FP32, FP32),
          (8, 2, 128, FP32, FP32), (8, 2, 128, BF16, CODE), (16, 16, 64, FP16, CODE), (6, 2, 80, BF16, CODE),
          (4, 1, 128, FP32, CODE), (3, 1, 40, FP16, FP16), (3, 1, 40, BF16, CODE)]
WINDOWS = [(1, 0), (5, 4), (16, 16), (33, 1), (64, 70), (100, 17), (256, 4), (1 << 40, 3)]


def run(case, device, **kw):
    q, k, v, scales, step = case.place(device)
    return ops.attention(q, k, v, case.layers - 1, step, case.scaling, window=case.window, sinks=case.sinks, **scales,
                         **kw), step


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache_dtype", SHAPES)
def test_window_matches_64_bits(device, heads, kv_heads, dim, dtype, cache_dtype, window, sinks):
    case = Case(STARTS, COUNTS, heads, kv_heads, dim, dtype, cache_dtype, window=window, sinks=sinks, seed=window % 97)
    out, _ = run(case, device)
    case.check(out)


@pytest.mark.parametrize("bs", [1, 4, 8, 12, 32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache_dtype",
                         [(8, 2, 128, BF16, BF16), (4, 4, 64, FP32, FP32), (8, 2, 64, FP16, CODE)])
def test_window_of_other_block_sizes(device, bs, heads, kv_heads, dim, dtype, cache_dtype):
    for window, sinks in [(48, 5), (200, 0), (77, 130)]:
        case = Case(STARTS, COUNTS, heads, kv_heads, dim, dtype, cache_dtype, bs=bs, window=window, sinks=sinks, seed=bs)
        out, _ = run(case, device)
        case.check(out)


@pytest.mark.parametrize("kind", ["decodes", "prompts"])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(8, 2, 128, BF16), (2, 2, 64, FP32), (8, 2, 256, FP16)])
def test_window_steps_of_one_kind(device, kind, heads, kv_heads, dim, dtype):
    starts, counts = ([700, 20, 5000, 63], [1] * 4) if kind == "decodes" else ([700, 0, 64], [130, 257, 64])
    case = Case(starts, counts, heads, kv_heads, dim, dtype, window=150, sinks=4, seed=3)
    out, _ = run(case, device)
    case.check(out)


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 8, 64), (6, 2, 64), (16, 16, 128), (32, 8, 128)])
def test_window_of_few_and_many_fp32_tiles(device, heads, kv_heads, dim):
    """Tiles that two workgroups take, and as many as the chip's workgroups or more."""
    for starts, counts in [([0, 40, 300], [70, 129, 64]), ([40 + i for i in range(18)], [130 + i for i in range(18)])]:
        case = Case(starts, counts, heads, kv_heads, dim, FP32, window=90, sinks=5, seed=dim)
        out, _ = run(case, device)
        case.check(out)


@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache_dtype", [
    (8, 2, 128, BF16, BF16), (8, 8, 64, FP16, FP16), (6, 2, 80, BF16, BF16), (4, 2, 256, BF16, BF16),
    (4, 2, 64, FP32, FP32), (8, 2, 128, BF16, CODE), (3, 1, 40, FP16, FP16)])
@pytest.mark.parametrize("starts,counts", [([40, 300, 1000, 0], [1] * 4), ([40, 300, 7], [1, 70, 33])])
def test_new_rows_are_written_and_seen(device, heads, kv_heads, dim, dtype, cache_dtype, starts, counts):
    case = Case(starts, counts, heads, kv_heads, dim, dtype, cache_dtype, window=50, sinks=3, seed=5)
    q, k, v, scales, step = case.place(device)
    gen = torch.Generator().manual_seed(9)
    rows = [torch.randn((sum(counts), kv_heads, dim), generator=gen).to(dtype).to(device) for _ in range(2)]
    k2, v2, s2 = k.clone(), v.clone(), {n: x.clone() for n, x in scales.items()}
    layer = case.layers - 1
    ops.reshape_and_cache(*rows, k2, v2, step.scatter_slots, layer, **s2)
    want = ops.attention(q, k2, v2, layer, step, case.scaling, window=50, sinks=3, **s2)
    padded = [torch.cat([r, r], dim=2)[:, :, :dim] for r in rows]  # strides of their own
    for new in (rows, padded):
        k1, v1, s1 = k.clone(), v.clone(), {n: x.clone() for n, x in scales.items()}
        got = ops.attention(q, k1, v1, layer, step, case.scaling, new_key=new[0], new_value=new[1], window=50, sinks=3,
                            **s1)
        assert torch.equal(got, want)
        for a, b in ((k1, k2), (v1, v2)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_a_window_past_every_context_is_plain_attention(device):
    for heads, kv_heads, dim, dtype in [(8, 2, 128, BF16), (4, 4, 64, FP32), (4, 2, 256, FP16)]:
        case = Case(STARTS, COUNTS, heads, kv_heads, dim, dtype, window=5000, sinks=2)
        q, k, v, _, step = case.place(device)
        plain = ops.attention(q, k, v, 1, step, case.scaling)
        case.check(plain)
        case.check(ops.attention(q, k, v, 1, step, case.scaling, window=5000, sinks=2))


def test_pooled_tables_query_layouts_and_out(device):
    case = Case(STARTS, COUNTS, 8, 2, 128, BF16, window=60, sinks=4, seed=8)
    q, k, v, _, step = case.place(device)
    want = ops.attention(q, k, v, 1, step, case.scaling, window=60, sinks=4)
    pool = torch.full((40, case.table.shape[1]), -1, dtype=torch.int32, device=device)
    rows = np.random.Generator(np.random.PCG64(1)).permutation(40)[:len(STARTS)].astype(np.int32)
    pool[torch.from_numpy(rows).long().to(device)] = torch.from_numpy(case.table).to(device)
    pooled = ops.pack_step(pool, STARTS, COUNTS, 16, num_kv_heads=2, num_query_heads=8, head_dim=128, dtype=BF16,
                           rows=rows)
    assert torch.equal(ops.attention(q, k, v, 1, pooled, case.scaling, window=60, sinks=4), want)
    head_major = q.transpose(0, 1).contiguous()[None]
    guard = torch.full((q.shape[0] + 2, 8, 128), 7.0, dtype=BF16, device=device)
    ops.attention(head_major, k, v, 1, step, case.scaling, out=guard[1:-1], window=60, sinks=4)
    assert torch.equal(guard[1:-1], want) and bool((guard[0] == 7).all()) and bool((guard[-1] == 7).all())


def test_missing_blocks_inside_the_window(device):
    """A row whose window has no block gives zeros; one with some is attention over the others."""
    for heads, kv_heads, dim, dtype, cache in [(8, 2, 128, BF16, BF16), (4, 2, 64, FP32, FP32), (8, 2, 128, BF16, CODE),
                                               (4, 2, 256, BF16, BF16)]:
        case = Case([400, 400, 64], [1, 40, 30], heads, kv_heads, dim, dtype, cache, window=40, sinks=0, seed=4)
        case.table[0, :] = -1
        case.table[1, 23] = 10 ** 6
        case.table[2, :] = -7
        case.seen[0][:] = False
        case.seen[1][:, 23 * 16:24 * 16] = False
        case.seen[2][:] = False
        case._reference()
        out, _ = run(case, device)
        case.check(out)
        assert bool((out[0] == 0).all()) and bool((out[-30:] == 0).all())


def test_repack_and_rerun_of_a_graph(device):
    """A captured layer serves contexts that grow from inside the window past it."""
    starts, counts, window, sinks = [40, 90, 130, 20], [1, 1, 1, 1], 64, 5
    for heads, kv_heads, dim, dtype in [(8, 2, 128, BF16), (4, 4, 64, FP32)]:
        cases = [Case([s + n for s in starts], counts, heads, kv_heads, dim, dtype, window=window, sinks=sinks, seed=2,
                      drop=False, poison=False) for n in (0, 30, 60, 100)]
        width = cases[-1].full_table.shape[1]
        table = torch.zeros((4, width), dtype=torch.int32, device=device)
        shape = max((c.keys.shape for c in cases), key=lambda s: s[0])
        k, v = (torch.zeros((2, *shape), dtype=dtype, device=device) for _ in range(2))
        q = torch.zeros((4, heads, dim), dtype=dtype, device=device)

        def fill(c):
            table.zero_()
            table[:, :c.full_table.shape[1]] = torch.from_numpy(c.full_table).to(device)
            k[1, :c.keys.shape[0]], v[1, :c.vals.shape[0]] = c.keys.to(device), c.vals.to(device)
            q.copy_(c.query)

        fill(cases[0])
        step = ops.pack_step(table, cases[0].starts, counts, 16, num_kv_heads=kv_heads, num_query_heads=heads,
                             head_dim=dim, dtype=dtype, partition_size=4096)
        out = torch.zeros_like(q)
        ops.attention(q, k, v, 1, step, cases[0].scaling, out=out, window=window, sinks=sinks)
        stream = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            step.rerun()
            ops.attention(q, k, v, 1, step, cases[0].scaling, out=out, window=window, sinks=sinks)
        for c in cases + cases[::-1]:
            fill(c)
            step.repack(c.starts, counts)
            out.zero_()
            graph.replay()
            c.check(out)
            c.check(ops.attention(q, k, v, 1, step, c.scaling, window=window, sinks=sinks))


def test_other_streams_and_two_steps(device):
    case = Case(STARTS, COUNTS, 8, 2, 128, BF16, window=60, sinks=4, seed=8, drop=False, poison=False)
    q, k, v, _, step = case.place(device)
    want = ops.attention(q, k, v, 1, step, case.scaling, window=60, sinks=4)
    wide = ops.attention(q, k, v, 1, step, case.scaling, window=200, sinks=4)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        q2, k2, v2, _, step2 = case.place(device)
        got = [ops.attention(q2, k2, v2, 1, step2, case.scaling, window=60, sinks=4) for _ in range(3)]
    for _ in range(3):
        assert torch.equal(ops.attention(q, k, v, 1, step, case.scaling, window=60, sinks=4), want)
        assert torch.equal(ops.attention(q, k, v, 1, step, case.scaling, window=200, sinks=4), wide)
    side.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_empty_steps(device):
    table = torch.full((2, 4), -1, dtype=torch.int32, device=device)
    cache = torch.zeros((1, 4, 16, 2, 64), dtype=BF16, device=device)
    step = ops.pack_step(table, [0, 0], [0, 0], 16, num_kv_heads=2, num_query_heads=4, head_dim=64, dtype=BF16)
    out = ops.attention(torch.zeros((0, 4, 64), dtype=BF16, device=device), cache, cache, 0, step, 1.0, window=4)
    assert out.shape == (0, 4, 64)


@pytest.mark.parametrize("scaling", [0.0, -0.3])
def test_scalings_of_zero_and_below(device, scaling):
    case = Case(STARTS, COUNTS, 8, 2, 128, BF16, window=60, sinks=4, seed=8)
    case.scaling = scaling
    case._reference()
    out, _ = run(case, device)
    case.check(out)


def test_refusals(device):
    case = Case([40], [1], 8, 2, 128, BF16, window=60)
    q, k, v, _, step = case.place(device)
    for bad in (0, -1, 1.5):
        with pytest.raises(ValueError, match="window must be"):
            ops.attention(q, k, v, 1, step, 1.0, window=bad)
    with pytest.raises(ValueError, match="sinks must be"):
        ops.attention(q, k, v, 1, step, 1.0, window=4, sinks=-1)
    with pytest.raises(ValueError, match="sinks go with a window"):
        ops.attention(q, k, v, 1, step, 1.0, sinks=4)
    with pytest.raises(ValueError, match="scales go with"):
        ops.attention(q, k, v, 1, step, 1.0, window=4, key_scales=q, value_scales=q)
    with pytest.raises(ValueError, match="dtype"):
        ops.attention(q.half(), k, v, 1, step, 1.0, window=4)
    with pytest.raises(RuntimeError, match="Layer index"):
        ops.attention(q, k, v, 2, step, 1.0, window=4)
