"""Trees of drafted tokens round a result once: probabilities enter the product with V
as two terms of the 16-bit type, so that a verified row is off 64 bits by what the
decode of the same token is."""

import numpy as np
import pytest
import torch

from helpers import pkg
from span_oracle import CODE, Case, random_tree

pytestmark = pytest.mark.gpu

ops = pkg("paged_ops")

BF16, FP16 = torch.bfloat16, torch.float16
SHAPES = [(8, 2, 128, BF16, BF16), (8, 8, 64, FP16, FP16), (6, 2, 80, BF16, BF16), (6, 2, 96, FP16, FP16),
          (4, 2, 256, BF16, BF16), (4, 2, 256, FP16, FP16), (64, 32, 128, BF16, BF16), (8, 2, 128, BF16, CODE),
          (16, 16, 64, FP16, CODE), (6, 2, 80, BF16, CODE)]


class TwoTerms(Case):
    """A weight is off by h^2 of itself where ``Case`` allows h (half a step, h =
    eps / 2, of the 16-bit type): a term is rounded by h of its value at most, the
    second one is what the first left.  That holds for the numerator and for the sum.
    Scores are kept below 1, so that the fp32 terms of the bound, which grow with
    them, stay below what a single rounding of the weights leaves."""

    def __init__(self, *args, **kw):
        self.small = False
        super().__init__(*args, **kw)
        self.scaling *= 0.1
        self.small = True
        self._reference()

    def _reference(self):
        super()._reference()
        if not self.small:
            return
        first, bounds = 0, []
        u, eps = 2.0 ** -24, torch.finfo(self.dtype).eps
        group = self.heads // self.kv_heads
        for i, (start, count) in enumerate(zip(self.starts, self.counts)):
            pos = np.arange(start + count)
            slot = torch.from_numpy(self.full_table[i, pos // self.bs].astype(np.int64) * self.bs + pos % self.bs)
            k, v = (x.reshape(-1, self.kv_heads, self.dim)[slot].repeat_interleave(group, dim=1).transpose(0, 1)
                    for x in (self.k64, self.v64))
            q = self.query[first:first + count].double().transpose(0, 1)
            mask = torch.from_numpy(self.seen[i])
            s = (q @ k.transpose(1, 2) * self.scaling).masked_fill(~mask, -float("inf"))
            a = torch.softmax(s, dim=-1) @ v.abs()
            mag = (q.abs() @ k.abs().transpose(1, 2) * self.scaling).masked_fill(~mask, 0).amax(dim=-1, keepdim=True)
            n = mask.sum(dim=-1)[None, :, None]
            rel = 2 * ((self.dim + 10) * mag.clamp(min=1.0) + n + 16) * u + 2 * (eps / 2) ** 2
            ref = self.ref[first:first + count].transpose(0, 1)
            least = 2.0 ** -24 * n * float(v.abs().max()) if self.dtype == FP16 else 0.0
            bounds.append((eps / 2 * ref.abs() * (1 + rel) + rel * a * (1 + eps / 2) + least).transpose(0, 1) + 1e-30)
            first += count
        self.bound = torch.cat(bounds)


@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3)])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache_dtype", SHAPES)
def test_trees_round_a_result_once(device, heads, kv_heads, dim, dtype, cache_dtype, window, sinks):
    rng = np.random.Generator(np.random.PCG64(3))
    starts, counts = [20, 45, 0, 33, 61, 30, 5, 50], [16, 9, 20, 33, 1, 12, 40, 25]
    parents = [random_tree(rng, n) for n in counts]
    case = TwoTerms(starts, counts, heads, kv_heads, dim, dtype, cache_dtype, parents=parents, window=window,
                    sinks=sinks, seed=dim + heads)
    q, k, v, scales, step = case.place(device)
    tree = ops.pack_tree(step, torch.tensor([p for t in parents for p in t], dtype=torch.int32), window=window,
                         sinks=sinks)
    case.check(ops.tree_attention(q, k, v, 1, step, tree, case.scaling, **scales))
