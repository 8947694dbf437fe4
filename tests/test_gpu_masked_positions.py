"""Positions that a step's table leaves out (block ids outside the pool) among
valid ones whose scores lie far below them, or next to a pool whose block 0
holds anything: they count for nothing, in the softmax's maximum as in its
products, in prefill and decode over every cache type, against fp64."""

import numpy as np
import pytest
import torch

import cache8_oracle as oracle
from helpers import pkg

pytestmark = pytest.mark.gpu

ops = pkg("paged_ops")
CODE = oracle.CODE

STARTS, COUNTS = [100, 0, 37, 200, 3, 0], [70, 30, 150, 1, 1, 200]
# (sequence, column) of blocks of 16 that are missing: the first, some in
# mid-context, a chunk's own, a half of a stage, the last.
MISSING = {(0, 0): -1, (0, 3): 10**6, (0, 8): -5, (1, 1): -1, (2, 2): -1, (2, 3): -1, (2, 11): 2**31 - 1, (3, 0): -1,
           (3, 7): -1, (5, 0): -1, (5, 1): -1, (5, 6): -1}


def case(heads, kv_heads, dim, dtype, cache_dtype, depth, block0, bs=16, seed=0):
    """Query rows along -u and keys along u for one direction u, so that every
    score is about -depth; block 0, in no sequence, holds ``block0`` in K and V."""
    gen = torch.Generator().manual_seed(seed)
    ends = [s + c for s, c in zip(STARTS, COUNTS)]
    need = [-(-e // bs) for e in ends]
    blocks = sum(need) + 2
    order = 1 + np.random.Generator(np.random.PCG64(seed)).permutation(blocks - 1)
    table = np.full((len(ends), max(need)), -1, dtype=np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    u = torch.sign(torch.randn(dim, generator=gen))
    shape = (blocks, bs, kv_heads, dim)
    keys = u + 0.3 * torch.randn(shape, generator=gen)
    vals = torch.randn(shape, generator=gen) + 1.0
    q = -(depth / np.sqrt(dim)) * u * (1 + 0.1 * torch.randn((sum(COUNTS), heads, 1), generator=gen))
    keys[0], vals[0] = block0, block0
    if cache_dtype == CODE:
        held = []
        for x in (keys, vals):
            codes, scales = torch.zeros(shape, dtype=torch.uint8).view(CODE), torch.zeros((blocks, kv_heads))
            oracle.write(codes, scales, x.to(dtype).float().reshape(-1, kv_heads, dim), list(range(blocks * bs)))
            held += [codes, scales]
        pools = [oracle.values(torch.nan_to_num(c.float()), s) for c, s in (held[:2], held[2:])]
    else:
        held = [keys.to(cache_dtype), None, vals.to(cache_dtype), None]
        pools = [torch.nan_to_num(held[0].double()), torch.nan_to_num(held[2].double())]
    for (i, c), b in MISSING.items():
        c = c * 16 // bs
        for j in range(c, c + max(16 // bs, 1)):
            table[i, j] = b
    return q.to(dtype), held, pools, table


def check(out, q, pools, table, dtype, depth):
    dim = q.shape[2]
    ref, size, peak = oracle.attention(q, *pools, table, STARTS, COUNTS, dim**-0.5)
    out = out.cpu().double()
    assert torch.isfinite(out).all()
    # One rounding of the result, a probability rounded to the query's type in
    # the sum or the product (2 u in all); a score is a chain of dim products
    # of one sign (the noise beside them is below 2 in all) in fp32, scaled and
    # shifted by the maximum: (dim + 4) 2^-24 of at most 1.5 depth + 2, twice
    # (its own and the maximum's), of a probability.  fp16's probabilities have
    # steps of 2^-24 of the row's largest, its results too.
    u = oracle.ROW_EPS[dtype]
    each = 2 * u + 2 * (dim + 4) * 2.0**-24 * (1.5 * depth + 2) + 1.5e-5
    bound = (1 + 2 * u) * u * ref.abs() + each * size
    if dtype == torch.float16:
        bound = bound + 2.0**-24 + 2.0**-25 * peak
    excess = ((out - ref).abs() - bound).max().item()
    assert excess <= 0, f"{excess:.3e} over the bound"


def run(heads, kv_heads, dim, dtype, cache_dtype, depth, block0, device, bs=16):
    q, held, pools, table = case(heads, kv_heads, dim, dtype, cache_dtype, depth, block0, bs)
    kc, ks, vc, vs = (None if t is None else t[None].to(device) for t in held)
    step = ops.pack_step(torch.from_numpy(table).to(device), STARTS, COUNTS, bs, num_kv_heads=kv_heads,
                         num_query_heads=heads, head_dim=dim, dtype=cache_dtype,
                         prefill_tile=ops.prefill_tile_for(heads, kv_heads))
    out = ops.attention(q.to(device), kc, vc, 0, step, dim**-0.5, key_scales=ks, value_scales=vs)
    check(out, q, pools, table, dtype, depth)


# e^-30 is among fp16's zeros, e^-130 below fp32's least number
DEPTHS = {torch.float16: 30.0, torch.bfloat16: 130.0, torch.float32: 130.0}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,dim,bs", [
    (8, 2, 128, 16), (4, 4, 64, 16), (6, 2, 80, 16), (4, 2, 96, 16), (4, 2, 128, 8), (4, 2, 64, 1), (2, 1, 256, 16)])
def test_scores_far_below_a_missing_blocks_over_8_bits(device, heads, kv_heads, dim, bs, dtype):
    run(heads, kv_heads, dim, dtype, CODE, DEPTHS[dtype], 0.0, device, bs)


SHAPES = [(8, 2, 128, 16, torch.float16), (8, 2, 128, 16, torch.bfloat16), (4, 4, 64, 16, torch.float16),
          (4, 4, 64, 16, torch.bfloat16), (6, 2, 80, 16, torch.float16), (4, 2, 96, 16, torch.bfloat16),
          (4, 2, 128, 8, torch.bfloat16), (4, 2, 128, 1, torch.float16), (4, 1, 256, 16, torch.float16),
          (2, 1, 256, 16, torch.bfloat16), (2, 1, 256, 4, torch.bfloat16), (4, 2, 64, 16, torch.float32),
          (4, 2, 128, 16, torch.float32), (3, 1, 40, 16, torch.bfloat16)]


@pytest.mark.parametrize("heads,kv_heads,dim,bs,dtype", SHAPES)
def test_scores_far_below_a_missing_blocks(device, heads, kv_heads, dim, bs, dtype):
    run(heads, kv_heads, dim, dtype, dtype, DEPTHS[dtype], 0.0, device, bs)


@pytest.mark.parametrize("heads,kv_heads,dim,bs,dtype", SHAPES[::3])
def test_far_below_a_block_of_the_other_sign(device, heads, kv_heads, dim, bs, dtype):
    # block 0 along -u: a score of +depth in a place that counts for nothing
    run(heads, kv_heads, dim, dtype, dtype, DEPTHS[dtype], -1.0, device, bs)


@pytest.mark.parametrize("block0", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("heads,kv_heads,dim,bs,dtype", SHAPES)
def test_block_0_of_no_sequence_holds_anything(device, heads, kv_heads, dim, bs, dtype, block0):
    run(heads, kv_heads, dim, dtype, dtype, 2.0, block0, device, bs)


@pytest.mark.parametrize("heads,kv_heads,dim,bs,dtype", [(8, 2, 128, 16, torch.float16), (4, 4, 64, 16, torch.bfloat16),
                                                         (6, 2, 80, 16, torch.bfloat16), (4, 2, 128, 4, torch.bfloat16),
                                                         (4, 2, 64, 16, torch.float32)])
@pytest.mark.parametrize("fused", [True, False])
def test_new_rows_without_a_block_hold_anything(device, heads, kv_heads, dim, bs, dtype, fused):
    # attention() writes the step's rows itself; those of missing blocks are NaN
    # and go nowhere
    q, held, pools, table = case(heads, kv_heads, dim, dtype, dtype, 2.0, float("nan"), bs)
    blocks = held[0].shape[0]
    rows = []
    for pool in held[::2]:
        flat = pool.reshape(-1, kv_heads, dim)
        new = torch.full((sum(COUNTS), kv_heads, dim), float("nan"), dtype=dtype)
        t = 0
        for i, (s, c) in enumerate(zip(STARTS, COUNTS)):
            for p in range(s, s + c):
                b = int(table[i, p // bs])
                if 0 <= b < blocks:
                    new[t] = flat[b * bs + p % bs]
                    flat[b * bs + p % bs] = 9.0  # (what the write replaces)
                t += 1
        rows.append(new)
    kc, vc = (held[i][None].to(device) for i in (0, 2))
    step = ops.pack_step(torch.from_numpy(table).to(device), STARTS, COUNTS, bs, num_kv_heads=kv_heads,
                         num_query_heads=heads, head_dim=dim, dtype=dtype,
                         prefill_tile=ops.prefill_tile_for(heads, kv_heads))
    out = ops.attention(q.to(device), kc, vc, 0, step, dim**-0.5, new_key=rows[0].to(device),
                        new_value=rows[1].to(device), fused_prefill_write=fused)
    check(out, q, pools, table, dtype, 2.0)
    for cache, pool in zip((kc, vc), pools):
        assert torch.equal(cache[0, 1:].cpu().double(), pool[1:])


@pytest.mark.parametrize("scaling", [0.0, -0.1])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache_dtype", [
    (8, 2, 128, torch.bfloat16, CODE), (4, 4, 64, torch.float16, CODE), (8, 2, 128, torch.bfloat16, torch.bfloat16),
    (4, 4, 64, torch.float16, torch.float16), (6, 2, 80, torch.bfloat16, torch.bfloat16),
    (2, 1, 256, torch.bfloat16, torch.bfloat16), (4, 2, 128, torch.float32, torch.float32),
    (3, 1, 40, torch.float16, torch.float16)])
@pytest.mark.parametrize("fused", [False, True])
def test_scaling_of_zero_and_below(device, heads, kv_heads, dim, dtype, cache_dtype, scaling, fused):
    # the softmax of -0.1 q.k, and (0) the mean of V, with missing blocks
    q, held, pools, table = case(heads, kv_heads, dim, dtype, cache_dtype, 3.0, 0.0)
    kc, ks, vc, vs = (None if t is None else t[None].to(device) for t in held)
    step = ops.pack_step(torch.from_numpy(table).to(device), STARTS, COUNTS, 16, num_kv_heads=kv_heads,
                         num_query_heads=heads, head_dim=dim, dtype=cache_dtype,
                         prefill_tile=ops.prefill_tile_for(heads, kv_heads))
    rows = {}
    if fused:  # the rows that are there already, written again
        if cache_dtype == CODE:
            pytest.skip("8-bit rows are coded afresh")
        at = [(int(table[i, p // 16]), p % 16) for i, (s, c) in enumerate(zip(STARTS, COUNTS)) for p in range(s, s + c)]
        for name, pool in (("new_key", held[0]), ("new_value", held[2])):
            rows[name] = torch.stack([pool[b, j] if 0 <= b < pool.shape[0] else torch.zeros_like(pool[0, 0])
                                      for b, j in at]).to(device)
        rows["fused_prefill_write"] = True
    out = ops.attention(q.to(device), kc, vc, 0, step, scaling, key_scales=ks, value_scales=vs, **rows)
    ref, size, peak = oracle.attention(q, *pools, table, STARTS, COUNTS, scaling)
    out = out.cpu().double()
    assert torch.isfinite(out).all()
    # scores are below 3 * 1.5 * dim / 10 + 2 (see check)
    u = oracle.ROW_EPS[dtype]
    bound = (1 + 2 * u) * u * ref.abs() + (2 * u + 2 * (dim + 4) * 2.0**-24 * (dim / 2 + 2) + 1.5e-5) * size
    if dtype == torch.float16:
        bound = bound + 2.0**-24 + 2.0**-25 * peak
    excess = ((out - ref).abs() - bound).max().item()
    assert excess <= 0, f"{excess:.3e} over the bound"
