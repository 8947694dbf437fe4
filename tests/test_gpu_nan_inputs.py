"""A NaN in a query row or in an attended K row makes the results that depend on
it NaN, in every decode and prefill kernel, and leaves the others alone."""

import numpy as np
import pytest
import torch

import cache8_oracle as oracle
from helpers import pkg

pytestmark = pytest.mark.gpu

ops = pkg("paged_ops")
CODE = oracle.CODE

STARTS, COUNTS = [9, 499, 299, 63, 20, 100, 0], [1, 1, 1, 1, 1, 40, 70]
BAD_QUERIES = [1, 3, 5]  # sequences; a multi-token one's second token
BAD_KEYS = {2: 250, 4: 7, 6: 30}  # sequence -> position of its NaN in KV head 0


@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache_dtype", [
    (8, 2, 128, torch.bfloat16, CODE), (16, 16, 64, torch.float16, CODE), (6, 2, 80, torch.bfloat16, CODE),
    (3, 1, 40, torch.float16, CODE), (4, 2, 64, torch.float32, CODE),
    (8, 2, 128, torch.bfloat16, torch.bfloat16), (4, 4, 64, torch.float16, torch.float16),
    (6, 2, 96, torch.float16, torch.float16), (24, 1, 128, torch.bfloat16, torch.bfloat16),
    (4, 2, 256, torch.bfloat16, torch.bfloat16), (8, 2, 128, torch.float32, torch.float32),
    (24, 2, 64, torch.float32, torch.float32), (3, 1, 40, torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("phases", [None, "split"])
def test_nan_inputs_reach_their_results(device, heads, kv_heads, dim, dtype, cache_dtype, phases):
    bs, gen = 16, torch.Generator().manual_seed(dim)
    ends = [s + c for s, c in zip(STARTS, COUNTS)]
    need = [-(-e // bs) for e in ends]
    table = np.full((len(ends), max(need)), -1, dtype=np.int32)
    table[np.arange(max(need)) < np.asarray(need)[:, None]] = np.arange(sum(need))
    first = np.cumsum([0] + need[:-1]) * bs
    slots = torch.cat([torch.arange(a, a + e) for a, e in zip(first.tolist(), ends)]).to(device)
    q = torch.randn((sum(COUNTS), heads, dim), generator=gen).to(dtype).to(device)
    k, v = (torch.randn((sum(ends), kv_heads, dim), generator=gen).to(dtype).to(device) for _ in range(2))
    step = ops.pack_step(torch.from_numpy(table).to(device), STARTS, COUNTS, bs, num_kv_heads=kv_heads,
                         num_query_heads=heads, head_dim=dim, dtype=cache_dtype, partition_size=64,
                         prefill_tile=ops.prefill_tile_for(heads, kv_heads))

    def run(q, k):
        caches = [torch.zeros((1, sum(need), bs, kv_heads, dim), dtype=cache_dtype, device=device) for _ in range(2)]
        scales = {}
        if cache_dtype == CODE:
            scales = {n: torch.zeros((1, sum(need), kv_heads), device=device) for n in ("key_scales", "value_scales")}
        ops.reshape_and_cache(k, v, *caches, slots, 0, **scales)
        if phases is None:
            return ops.attention(q, *caches, 0, step, dim**-0.5, **scales)
        out = torch.empty_like(q)
        ops.decode(q, *caches, 0, step, dim**-0.5, out=out, phases=1, **scales)
        ops.decode(q, *caches, 0, step, dim**-0.5, out=out, phases=2, **scales)
        return ops.prefill(q, *caches, 0, step, dim**-0.5, out=out, **scales)

    want = run(q, k)
    assert torch.isfinite(want).all()
    bad = torch.zeros(want.shape[:2], dtype=torch.bool)
    at = np.cumsum([0] + COUNTS[:-1])
    q2, k2 = q.clone(), k.clone()
    for i in BAD_QUERIES:
        t = int(at[i]) + (COUNTS[i] > 1)
        q2[t, :, dim // 2] = float("nan")
        bad[t] = True
    offset = np.cumsum([0] + ends[:-1])
    for i, p in BAD_KEYS.items():
        k2[int(offset[i]) + p, 0, 1] = float("nan")
        seen = max(p - STARTS[i], 0)  # the tokens at or behind the NaN's position
        bad[at[i] + seen:at[i] + COUNTS[i], :heads // kv_heads] = True
    got = run(q2, k2)
    assert torch.equal(torch.isnan(got).all(-1).cpu(), bad)
    if cache_dtype == CODE:
        # (a NaN counts for no scale: the largest value of its block's head may
        # have been the one it replaced, so the NaN's own sequences are not compared)
        for i in BAD_KEYS:
            bad[at[i]:at[i] + COUNTS[i]] = True
    assert torch.equal(got[~bad.to(device)], want[~bad.to(device)])
