"""Attention over part of a paged context in 64 bits, from its definition, with
an error bound that is derived from the arithmetic the kernels document.

A row's result is sum_j w_j v_j with softmax weights w of scores s_j.  With
u = 2^-24 (fp32 accumulation) and h = eps / 2 of the 16-bit type (a rounding is
off by at most half a step):
  * a score is off by at most (D + 2) u sum_d |q_d k_d| scaling, and taking it to
    the exponent's base and through exp2 adds a few u of its magnitude, so each
    weight is off by a factor of 1 +- (D + 10) u S with S = max_j sum_d |q_d k_d|
    scaling (at least 1); twice, numerator and sum;
  * summing N terms in fp32, in any order, is off by N u of the sum of
    magnitudes, in the numerator and in the denominator;
  * 16-bit kernels round each probability once before the product (h), and the
    sum counts the rounded ones (h again);
  * in fp16 one below its smallest normal is off by up to 2^-25 of the largest
    (twice, for N of them, of max |v|);
  * the result is rounded once (h |result|).
All but the last two are relative to A = sum_j w_j |v_j|."""

import math

import numpy as np
import torch

import cache8_oracle
from helpers import pkg

ops = pkg("paged_ops")
CODE = ops.CODE_DTYPE


def depths(parents):
    out = []
    for i, p in enumerate(parents):
        out.append(out[p] + 1 if 0 <= p < i else 0)
    return out


def ancestors(parents):
    """[n, n] bool: column j is row i or an ancestor of it."""
    n = len(parents)
    m = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        m[i, i] = True
        if 0 <= p < i:
            m[i] |= m[p]
    return m


def seen_mask(start, count, window=None, sinks=0, parents=None):
    """[count, start + count] bool: what each new token sees."""
    depth = np.arange(count) if parents is None else np.asarray(depths(parents))
    p = start + depth[:, None]
    q = np.arange(start + count)[None]
    seen = q <= p
    if window is not None:
        seen &= (p - q < window) | (q < sinks)
    if parents is not None:
        seen[:, start:] = ancestors(parents)
    return seen


def random_tree(rng, n):
    return [-1] + [int(rng.integers(max(0, i - 12), i)) for i in range(1, n)]


class Case:
    """A step with its caches and 64-bit reference; ``parents`` per sequence for
    trees.  Rows that no query sees are NaN, blocks without a seen row are missing
    from the table (``drop``)."""

    def __init__(self, starts, counts, heads, kv_heads, dim, dtype, cache_dtype=None, bs=16, window=None, sinks=0,
                 parents=None, seed=0, drop=True, poison=True, spread=1.0, layers=2):
        self.starts, self.counts, self.bs, self.dim = list(starts), list(counts), bs, dim
        self.heads, self.kv_heads, self.dtype = heads, kv_heads, dtype
        self.cache_dtype = cache_dtype = cache_dtype or dtype
        self.window, self.sinks, self.parents, self.layers = window, sinks, parents, layers
        gen = torch.Generator().manual_seed(seed)
        rng = np.random.Generator(np.random.PCG64(seed + 1))
        ends = [s + c for s, c in zip(starts, counts)]
        need = [-(-e // bs) for e in ends]
        blocks = sum(need) + 3
        order = rng.permutation(blocks)
        self.table = np.full((len(ends), max(need + [1])), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.seen = [seen_mask(s, c, window, sinks, None if parents is None else parents[i])
                     for i, (s, c) in enumerate(zip(starts, counts))]
        shape = (blocks, bs, kv_heads, dim)
        keys, vals = (torch.randn(shape, generator=gen) * spread for _ in range(2))
        self.scales = {}
        if cache_dtype == CODE:
            held = []
            for x in (keys, vals):
                codes, scales = torch.zeros(shape, dtype=torch.uint8).view(CODE), torch.zeros((blocks, kv_heads))
                cache8_oracle.write(codes, scales, x.to(dtype).float().reshape(-1, kv_heads, dim),
                                    list(range(blocks * bs)))
                held.append((codes, scales))
            k64, v64 = (cache8_oracle.values(c, s) for c, s in held)
            keys, vals = held[0][0], held[1][0]
            self.scales = {"key_scales": held[0][1], "value_scales": held[1][1]}
        else:
            keys, vals = keys.to(cache_dtype), vals.to(cache_dtype)
            k64, v64 = keys.double(), vals.double()
        self.query = torch.randn((sum(counts), heads, dim), generator=gen).to(dtype)
        self.scaling = 1.0 / math.sqrt(dim)
        self.k64, self.v64 = k64.double().clone(), v64.double().clone()
        if poison:
            flat_k, flat_v = (x.view(-1, kv_heads, dim) for x in (keys.view(torch.uint8) if cache_dtype == CODE else
                                                                  keys, vals.view(torch.uint8) if cache_dtype == CODE
                                                                  else vals))
            bad = 0x7f if cache_dtype == CODE else float("nan")
            unseen = np.ones(blocks * bs, bool)
            for i, m in enumerate(self.seen):
                pos = np.flatnonzero(m.any(axis=0))
                unseen[self.table[i, pos // bs].astype(np.int64) * bs + pos % bs] = False
            flat_k[torch.from_numpy(unseen)] = bad
            flat_v[torch.from_numpy(unseen)] = bad
        self.full_table = self.table.copy()
        if drop:
            for i, m in enumerate(self.seen):
                cols = np.zeros(self.table.shape[1], bool)
                cols[np.flatnonzero(m.any(axis=0)) // bs] = True
                gone = np.flatnonzero(~cols)
                self.table[i, gone] = np.where(gone % 3 == 0, 10 ** 6, -1 - gone % 2)
        self.keys, self.vals = keys, vals
        self._reference()

    def _reference(self):
        out, bound = [], []
        first = 0
        eps = torch.finfo(self.dtype).eps if self.dtype != torch.float32 else 0.0
        u, group = 2.0 ** -24, self.heads // self.kv_heads
        for i, (start, count) in enumerate(zip(self.starts, self.counts)):
            if count == 0:
                continue
            pos = np.arange(start + count)
            slot = torch.from_numpy(self.full_table[i, pos // self.bs].astype(np.int64) * self.bs + pos % self.bs)
            k, v = (x.reshape(-1, self.kv_heads, self.dim)[slot].repeat_interleave(group, dim=1).transpose(0, 1)
                    for x in (self.k64, self.v64))
            q = self.query[first:first + count].double().transpose(0, 1)
            mask = torch.from_numpy(self.seen[i])
            s = (q @ k.transpose(1, 2) * self.scaling).masked_fill(~mask, -math.inf)
            w = torch.nan_to_num(torch.softmax(s, dim=-1))
            mag = (q.abs() @ k.abs().transpose(1, 2) * abs(self.scaling)).masked_fill(~mask, 0).amax(dim=-1, keepdim=True)
            n = mask.sum(dim=-1)[None, :, None]
            ref, a = w @ v, w @ v.abs()
            rel = 2 * ((self.dim + 10) * mag.clamp(min=1.0) + n + 16) * u + eps
            half = max(eps, 2 * u) / 2
            least = 2.0 ** -24 * n * float(v.abs().max()) if self.dtype == torch.float16 and v.numel() else 0.0
            out.append(ref.transpose(0, 1))
            bound.append((half * ref.abs() * (1 + rel) + rel * a * (1 + half) + least).transpose(0, 1) + 1e-30)
            first += count
        self.ref = torch.cat(out) if out else torch.zeros(0, self.heads, self.dim)
        self.bound = torch.cat(bound) if bound else self.ref

    def place(self, device):
        """(query, key_cache, value_cache, scales, step) on the device: the rows in
        the last layer, the others NaN."""
        def cache(x):
            full = torch.full((self.layers, *x.shape), float("nan"), dtype=torch.float32).to(x.dtype) \
                if x.dtype != CODE else torch.full((self.layers, *x.shape), 0x7f, dtype=torch.uint8).view(CODE)
            (full.view(torch.uint8) if x.dtype == CODE else full)[-1] = x.view(torch.uint8) if x.dtype == CODE else x
            return full.to(device)

        scales = {}
        for name, s in self.scales.items():
            full = torch.ones((self.layers, *s.shape))
            full[-1] = s
            scales[name] = full.to(device)
        step = ops.pack_step(torch.from_numpy(self.table).to(device), self.starts, self.counts, self.bs,
                             num_kv_heads=self.kv_heads, num_query_heads=self.heads, head_dim=self.dim,
                             dtype=self.cache_dtype)
        return self.query.to(device), cache(self.keys), cache(self.vals), scales, step

    def check(self, out):
        got = out.double().cpu()
        assert torch.isfinite(got).all(), f"not finite at {torch.nonzero(~torch.isfinite(got))[:4].tolist()}"
        off = (got - self.ref).abs() / self.bound
        worst = int(off.reshape(-1).argmax()) if off.numel() else 0
        at = np.unravel_index(worst, tuple(off.shape)) if off.numel() else None
        assert off.numel() == 0 or float(off.max()) <= 1.0, \
            f"{float(off.max()):.2f} of the bound at {at}: {got[at]:.6g}, {self.ref[at]:.6g}"
