"""Attention under windows and over trees where scores climb along the context, so that
a row's running maximum outgrows the one its sums are kept at and these are rescaled,
with something in them.  That the scores do so is shown here, on the host."""

import math

import numpy as np
import pytest
import torch

import cache8_oracle
from helpers import pkg
from span_oracle import CODE, Case, random_tree

pytestmark = pytest.mark.gpu

ops = pkg("paged_ops")

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
SHAPES = [(8, 2, 128, BF16, BF16), (8, 8, 64, FP16, FP16), (6, 2, 80, BF16, BF16), (6, 2, 96, FP16, FP16),
          (24, 1, 128, BF16, BF16), (4, 2, 256, BF16, BF16), (4, 2, 256, FP16, FP16), (4, 2, 64, FP32, FP32),
          (8, 2, 128, FP32, FP32), (8, 2, 128, BF16, CODE), (16, 16, 64, FP16, CODE), (6, 2, 80, BF16, CODE),
          (3, 1, 40, FP16, FP16)]
STAIR = 6.5   # how much the scores rise (natural units; 9.4 to the base 2) ...
EVERY = 160   # ... every so many positions
HEADROOM = 8 / math.log2(math.e)


class Climbing(Case):
    """Queries share a direction per KV head, along which the keys grow with their
    position in steps."""

    def __init__(self, starts, counts, heads, kv_heads, dim, dtype, cache_dtype=None, seed=0, **kw):
        super().__init__(starts, counts, heads, kv_heads, dim, dtype, cache_dtype, seed=seed, poison=False, **kw)
        gen = torch.Generator().manual_seed(seed + 5)
        along = torch.randint(0, 2, (kv_heads, dim), generator=gen).float() * 2 - 1
        query = along.repeat_interleave(heads // kv_heads, dim=0) + 0.3 * torch.randn((sum(counts), heads, dim),
                                                                                      generator=gen)
        self.query = query.to(dtype)
        keys = 0.5 * torch.randn(self.k64.shape, generator=gen)
        flat = keys.view(-1, kv_heads, dim)
        for i, (s, c) in enumerate(zip(starts, counts)):
            pos = np.arange(s + c)
            slot = torch.from_numpy(self.full_table[i, pos // self.bs].astype(np.int64) * self.bs + pos % self.bs)
            height = torch.from_numpy(pos // EVERY).float() * STAIR / math.sqrt(dim)
            flat[slot] += height[:, None, None] * along
        if self.cache_dtype == CODE:
            codes, scales = torch.zeros(keys.shape, dtype=torch.uint8).view(CODE), torch.zeros(keys.shape[:1] + (kv_heads,))
            cache8_oracle.write(codes, scales, keys.to(dtype).float().reshape(-1, kv_heads, dim),
                                list(range(keys.shape[0] * self.bs)))
            self.keys, self.scales["key_scales"] = codes, scales
            self.k64 = cache8_oracle.values(codes, scales).double().clone()
        else:
            self.keys = keys.to(self.cache_dtype)
            self.k64 = self.keys.double()
        self._reference()

    def rises(self, i, waves, tile, run):
        """The least number of times that a row of sequence i (of the first heads of the
        first four KV heads: those of one share a direction) outgrows its kept maximum by
        more than the headroom, after its first seen tile, in any wave's tiles of any run
        that spans three steps."""
        start, count = self.starts[i], self.counts[i]
        first, group = sum(self.counts[:i]), self.heads // self.kv_heads
        pos = np.arange(start + count)
        slot = torch.from_numpy(self.full_table[i, pos // self.bs].astype(np.int64) * self.bs + pos % self.bs)
        k = self.k64.reshape(-1, self.kv_heads, self.dim)[slot][:, :4].transpose(0, 1)
        q = self.query[first:first + count, ::group][:, :4].double().transpose(0, 1)
        s = (q @ k.transpose(1, 2) * self.scaling).masked_fill(~torch.from_numpy(self.seen[i]), -math.inf)
        pad = -s.shape[-1] % tile
        top = torch.nn.functional.pad(s, (0, pad), value=-math.inf).unflatten(-1, (-1, tile)).amax(-1)
        seen = torch.isfinite(top).any(0).any(0).nonzero()[:, 0]  # tiles that some row sees
        top = top[..., seen]
        least = None
        for r0 in range(0, top.shape[-1], run):
            for w in range(waves):
                mine = top[..., r0:r0 + run][..., w::waves]
                if mine.shape[-1] * waves * tile < 3 * EVERY + waves * tile:
                    continue
                kept = torch.full(mine.shape[:2], -math.inf, dtype=torch.float64)
                n = torch.zeros(mine.shape[:2])
                for t in range(mine.shape[-1]):
                    grow = mine[..., t] - kept > HEADROOM
                    n += grow & torch.isfinite(kept)
                    kept = torch.where(grow, mine[..., t], kept)
                n = n.min()
                least = n if least is None else min(least, n)
        return least


def climbs(case, run=10 ** 6):
    found = [case.rises(i, waves, 32, run) for i in range(len(case.starts)) for waves in (1, 2, 4)]
    found = [n for n in found if n is not None]
    assert found and min(found) >= 1


STARTS, COUNTS = [1500, 40, 900, 2700, 700], [1, 1, 40, 1, 200]


@pytest.mark.parametrize("window,sinks", [(10 ** 6, 0), (800, 4)])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache_dtype", SHAPES)
def test_windows(device, heads, kv_heads, dim, dtype, cache_dtype, window, sinks):
    case = Climbing(STARTS, COUNTS, heads, kv_heads, dim, dtype, cache_dtype, window=window, sinks=sinks, seed=dim)
    climbs(case)
    q, k, v, scales, step = case.place(device)
    case.check(ops.attention(q, k, v, 1, step, case.scaling, window=window, sinks=sinks, **scales))


@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache_dtype", SHAPES)
def test_windows_of_whole_partitions(device, heads, kv_heads, dim, dtype, cache_dtype):
    """Decodes that one workgroup walks whole."""
    case = Climbing([2300, 1900], [1, 1], heads, kv_heads, dim, dtype, cache_dtype, window=1700, sinks=4, seed=dim)
    climbs(case)
    q, k, v, scales, _ = case.place(device)
    step = ops.pack_step(torch.from_numpy(case.table).to(device), case.starts, case.counts, case.bs,
                         num_kv_heads=kv_heads, num_query_heads=heads, head_dim=dim, dtype=case.cache_dtype,
                         partition_size=4096)
    case.check(ops.attention(q, k, v, 1, step, case.scaling, window=1700, sinks=4, **scales))


@pytest.mark.parametrize("window,sinks", [(None, 0), (900, 4)])
@pytest.mark.parametrize("split", [0, 12, 800])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache_dtype", SHAPES)
def test_trees(device, heads, kv_heads, dim, dtype, cache_dtype, split, window, sinks, monkeypatch):
    """Split by the planner's choice, in runs of 12 stages, and not at all."""
    rng = np.random.Generator(np.random.PCG64(dim))
    starts, counts = [1500, 2200, 900], [26, 9, 40]
    parents = [random_tree(rng, n) for n in counts]
    case = Climbing(starts, counts, heads, kv_heads, dim, dtype, cache_dtype, window=window, sinks=sinks,
                    parents=parents, seed=dim)
    q, k, v, scales, step = case.place(device)
    if split:
        plan = ops._plan_tree
        monkeypatch.setattr(ops, "_plan_tree", lambda s, d, n: plan(s, d, n or split))
    tree = ops.pack_tree(step, torch.tensor([p for t in parents for p in t], dtype=torch.int32), window=window,
                         sinks=sinks)
    if split:
        climbs(case, run=2 * split)
        assert dim == 40 or tree._plan.split_stages == split
    case.check(ops.tree_attention(q, k, v, 1, step, tree, case.scaling, **scales))


@pytest.mark.parametrize("dim,dtype", [(64, FP16), (80, BF16), (128, BF16), (256, BF16)])
def test_trees_of_more_units_than_compute_units(device, dim, dtype):
    """Workgroups of two waves."""
    rng = np.random.Generator(np.random.PCG64(2))
    starts, counts = [1000 + 40 * i for i in range(12)], [12] * 12
    parents = [random_tree(rng, n) for n in counts]
    case = Climbing(starts, counts, 32, 32, dim, dtype, parents=parents, seed=dim)
    climbs(case)
    q, k, v, _, step = case.place(device)
    tree = ops.pack_tree(step, torch.tensor([p for t in parents for p in t], dtype=torch.int32))
    assert tree._plan.num_items * 32 > 256
    case.check(ops.tree_attention(q, k, v, 1, step, tree, case.scaling))
