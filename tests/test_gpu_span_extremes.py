"""Windows and trees at the ends of their ranges: rows past 4 GiB of a cache, more
work items than a grid's second dimension holds, the largest trees, two trees of a
step at once."""

import numpy as np
import pytest
import torch

from helpers import pkg
from span_oracle import CODE, Case, random_tree

pytestmark = pytest.mark.gpu

ops = pkg("paged_ops")

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def flat(parents):
    return torch.tensor([p for up in parents for p in up], dtype=torch.int32)


def trees(counts, seed=0):
    rng = np.random.Generator(np.random.PCG64(seed))
    return [random_tree(rng, n) for n in counts]


def attend(case, device, k, v, scales, table, **kw):
    step = ops.pack_step(table.to(device), case.starts, case.counts, case.bs, num_kv_heads=case.kv_heads,
                         num_query_heads=case.heads, head_dim=case.dim, dtype=case.cache_dtype)
    q = case.query.to(device)
    if case.parents is None:
        return step, ops.attention(q, k, v, 0, step, case.scaling, window=case.window, sinks=case.sinks, **scales)
    tree = ops.pack_tree(step, flat(case.parents).to(device), window=case.window, sinks=case.sinks)
    return step, ops.tree_attention(q, k, v, 0, step, tree, case.scaling, **scales)


@pytest.mark.parametrize("kind", ["window", "tree"])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache_dtype,blocks", [
    (16, 8, 128, BF16, BF16, 140000), (8, 8, 256, FP16, FP16, 70000), (8, 8, 128, FP32, FP32, 70000),
    (8, 8, 128, BF16, CODE, 280000), (8, 8, 40, FP16, FP16, 430000)])
def test_rows_past_4_gib(device, kind, heads, kv_heads, dim, dtype, cache_dtype, blocks):
    """The same rows in the last blocks of a cache of more than 2^32 bytes."""
    if kind == "window":
        case = Case([0, 300, 1, 700], [1, 1, 40, 33], heads, kv_heads, dim, dtype, cache_dtype, window=90, sinks=5,
                    layers=1)
    else:
        case = Case([0, 300, 70], [3, 20, 40], heads, kv_heads, dim, dtype, cache_dtype, parents=trees([3, 20, 40]),
                    layers=1)
    near = len(case.keys)
    assert blocks * 16 * kv_heads * dim * case.keys.element_size() > 2 ** 32
    k, v = (torch.empty((1, blocks, 16, kv_heads, dim), dtype=cache_dtype, device=device) for _ in range(2))
    scales = {name: torch.ones((1, blocks, kv_heads), device=device) for name in case.scales}
    for cache, rows in ((k, case.keys), (v, case.vals)):
        cache[0, blocks - near:].copy_(rows.to(device))
    for name, s in case.scales.items():
        scales[name][0, blocks - near:] = s.to(device)
    table = torch.from_numpy(case.table)
    far = torch.where((table >= 0) & (table < near), table + (blocks - near), table).to(torch.int32)
    step, out = attend(case, device, k, v, scales, far)
    case.check(out)
    if kind == "tree":  # and the rows of a path of each tree
        nodes = torch.full((63,), -1, dtype=torch.int32)
        nodes[0], nodes[3:6], nodes[23:25] = 2, torch.tensor([0, 7, 19]), torch.tensor([5, 39])
        slots = step.scatter_slots.clone()
        def rows(cache):
            cache = cache.view(torch.uint8) if cache_dtype == CODE else cache
            return cache.view(-1, kv_heads, dim)[slots].clone()
        before = [rows(x) for x in (k, v)]
        ops.keep_rows(k, v, step, nodes.to(device), torch.tensor([1, 3, 2], dtype=torch.int32, device=device), **scales)
        if cache_dtype != CODE:
            for was, now in zip(before, (rows(x) for x in (k, v))):
                want = was.clone()
                want[0], want[3:6], want[23:25] = was[2], was[[3, 10, 22]], was[[28, 62]]
                assert torch.equal(now, want)


def test_more_items_than_65535(device):
    """70000 decodes under a window and 70000 trees: copies of seven sequences."""
    copies = 10000
    starts = [0, 3, 40, 150, 299, 310, 77]
    case = Case(starts, [1] * 7, 8, 2, 64, BF16, window=120, sinks=4, layers=1)
    k, v = case.keys[None].to(device), case.vals[None].to(device)
    table = torch.from_numpy(case.table).repeat(copies, 1).to(device)
    q = case.query.repeat(copies, 1, 1).to(device)
    step = ops.pack_step(table, starts * copies, [1] * 7 * copies, 16, partition_size=32, num_kv_heads=2,
                         num_query_heads=8, head_dim=64, dtype=BF16)
    out = ops.attention(q, k, v, 0, step, case.scaling, window=120, sinks=4).view(copies, 7, 8, 64)
    assert list(step._windows.values())[0].num_decode_items > 2 * 65535
    assert bool((out == out[:1]).all())
    case.check(out[-1])

    counts = [1, 2, 3, 1, 2, 1, 3]
    case = Case(starts, counts, 8, 2, 64, BF16, parents=trees(counts), layers=1)
    k, v = case.keys[None].to(device), case.vals[None].to(device)
    table = torch.from_numpy(case.table).repeat(copies, 1).to(device)
    step = ops.pack_step(table, starts * copies, counts * copies, 16, num_kv_heads=2, num_query_heads=8, head_dim=64,
                         dtype=BF16)
    tree = ops.pack_tree(step, flat(case.parents).repeat(copies).to(device))
    out = ops.tree_attention(case.query.repeat(copies, 1, 1).to(device), k, v, 0, step, tree,
                             case.scaling).view(copies, 13, 8, 64)
    assert bool((out == out[:1]).all())
    case.check(out[-1])


@pytest.mark.parametrize("window", [None, 1024])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache_dtype", [(8, 2, 128, BF16, BF16), (2, 2, 64, FP32, FP32),
                                                                  (4, 2, 256, FP16, FP16), (4, 2, 128, BF16, CODE),
                                                                  (3, 1, 40, FP16, FP16)])
def test_the_largest_trees(device, heads, kv_heads, dim, dtype, cache_dtype, window):
    """1024 nodes behind a context of any length, beside trees of one node."""
    counts = [1024, 1, 1024]
    parents = trees(counts, seed=9)
    parents[2] = list(range(-1, 1023))  # a chain
    case = Case([0, 2000, 1100], counts, heads, kv_heads, dim, dtype, cache_dtype, parents=parents, window=window,
                sinks=3 if window else 0, seed=4)
    q, k, v, scales, step = case.place(device)
    tree = ops.pack_tree(step, flat(parents).to(device), window=window, sinks=case.sinks)
    assert tree.masks.shape == (2049, 32)
    assert tree.position_ids[1025:].tolist() == list(range(1100, 2124))
    case.check(ops.tree_attention(q, k, v, 1, step, tree, case.scaling, **scales))


def test_two_trees_of_a_step_at_once(device):
    """Each has its own work lists and workspace: calls on two streams in turn and
    together give the same bits."""
    counts = [30, 9, 60, 17]
    parents = trees(counts, seed=2)
    case = Case([3000, 200, 900, 5000], counts, 16, 4, 128, BF16, parents=parents, drop=False, poison=False)
    q, k, v, _, step = case.place(device)
    on = flat(parents).to(device)
    full, windowed = ops.pack_tree(step, on), ops.pack_tree(step, on, window=700, sinks=4)
    alone = [ops.tree_attention(q, k, v, 1, step, t, case.scaling) for t in (full, windowed)]
    case.check(alone[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        a = ops.tree_attention(q, k, v, 1, step, full, case.scaling)
        with torch.cuda.stream(side):
            b = ops.tree_attention(q, k, v, 1, step, windowed, case.scaling)
        torch.cuda.synchronize()
        assert torch.equal(a, alone[0]) and torch.equal(b, alone[1])
