"""The 8-bit cache: its write bit for bit against the rules one block at a
time, attention over it against fp64, and the two together as a server runs
them."""

import numpy as np
import pytest
import torch

import cache8_oracle as oracle
from helpers import pkg

pytestmark = pytest.mark.gpu

ops = pkg("paged_ops")
CODE = oracle.CODE


def empty(layers, blocks, bs, heads, dim, device, garbage=False):
    """Codes and scales of K and V; ``garbage``: codes and scales of every kind."""
    shape = (layers, blocks, bs, heads, dim)
    if not garbage:
        return [torch.zeros(shape, dtype=CODE, device=device) for _ in range(2)] + [
            torch.zeros((layers, blocks, heads), device=device) for _ in range(2)]
    gen = torch.Generator(device=device).manual_seed(9)
    codes = [torch.randint(0, 256, shape, generator=gen, device=device, dtype=torch.uint8) for _ in range(2)]
    scales = [2.0 ** torch.randint(-12, 3, (layers, blocks, heads), generator=gen, device=device).float()
              for _ in range(2)]
    return [c.view(CODE) for c in codes] + scales


def same(mine, want, layer):
    """Codes equal as bytes (but for the payload of NaN), scales equal."""
    (kc, vc, ks, vs), (wkc, wks, wvc, wvs) = mine, want
    for codes, scales, wc, ws in ((kc, ks, wkc, wks), (vc, vs, wvc, wvs)):
        assert torch.equal(scales[layer].cpu(), ws)
        a, b = codes[layer].cpu().view(torch.uint8), wc.view(torch.uint8)
        nan = ((a & 0x7F) == 0x7F) & ((b & 0x7F) == 0x7F)
        assert torch.equal(a[~nan], b[~nan])


def stored(x):
    """Rows as the write codes them, fp32 on the CPU."""
    y = x.float().cpu()
    most = 61440.0 if x.dtype == torch.float16 else 1.875 * 2.0**127
    return torch.where(torch.isfinite(y), y.clamp(-most, most), y)


def expect(mine, layer, k, v, slots):
    kc, vc, ks, vs = mine
    out = []
    for codes, scales, x in ((kc, ks, k), (vc, vs, v)):
        out += oracle.write(codes[layer].cpu().clone(), scales[layer].cpu().clone(), stored(x), slots.tolist())
    return out


WRITES = [  # kv_heads, dim, block, runs of (first slot, tokens)
    (8, 128, 16, [(0, 16), (16, 16), (32, 5)]),                   # whole blocks from their first row, a partial one
    (2, 64, 16, [(3, 1), (20, 1), (47, 1), (64, 1)]),             # decodes into the middle, end and start of blocks
    (3, 64, 32, [(5, 70), (100, 1), (133, 27)]),                  # chunks that start and end inside blocks
    (1, 96, 16, [(9, 40), (64, 3), (79, 2)]),                     # a run over a block's end into a fresh block
    (2, 80, 1, [(4, 9)]),                                         # blocks of one row
    (2, 128, 4, [(2, 13), (20, 4)]),
    (1, 256, 8, [(6, 19)]),
    (2, 36, 16, [(1, 20), (40, 1)]),                              # no vector path
    (3, 7, 5, [(0, 12), (13, 2)]),                                # odd everything
    (1, 64, 256, [(3, 300), (700, 68)]),                          # the largest block
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kv_heads,dim,bs,runs", WRITES)
def test_write(device, kv_heads, dim, bs, runs, dtype):
    slots = torch.cat([torch.arange(a, a + n) for a, n in runs])
    blocks = int(slots.max()) // bs + 2
    gen = torch.Generator().manual_seed(len(slots))
    mine = empty(2, blocks, bs, kv_heads, dim, device, garbage=True)
    for magnitude in (1.0, 0.01, 30.0):  # the second keeps the scales, the third makes them grow
        k, v = ((magnitude * torch.randn((len(slots), kv_heads, dim), generator=gen)).to(dtype).to(device)
                for _ in range(2))
        want = expect(mine, 1, k, v, slots)
        before = [t[0].clone() for t in mine]
        ops.reshape_and_cache(k, v, mine[0], mine[1], slots.to(device), 1, mine[2], mine[3])
        same(mine, want, 1)
        assert all(torch.equal(a.view(torch.uint8) if a.dtype == CODE else a,
                               b[0].view(torch.uint8) if b.dtype == CODE else b[0]) for a, b in zip(before, mine))


def test_write_of_extremes(device):
    # zeros, the scale's floor, powers of two around 448, infinities, NaN, the
    # ends of the types' ranges; one head each
    big = torch.finfo(torch.bfloat16).max
    cases = [[0.0, -0.0, 0.0], [1e-30, -1e-38, 2.0**-133], [448.0, 1.0, -447.0], [450.0, 0.001, 449.0],
             [float("inf"), 1.0, -2.0], [float("nan"), float("-inf"), 0.25], [big, -big, 1.0],
             [float("inf"), float("nan"), float("-inf")], [2.0**-55, 448 * 2.0**-64, 450 * 2.0**-64]]
    for dtype in (torch.bfloat16, torch.float32, torch.float16):
        x = torch.tensor(cases).unsqueeze(0).expand(3, -1, -1).repeat(1, 1, 8).to(dtype).to(device)
        mine = empty(1, 2, 4, len(cases), 24, device)
        slots = torch.tensor([0, 1, 2])
        want = expect(mine, 0, x, -x, slots)
        ops.reshape_and_cache(x, -x, mine[0], mine[1], slots.to(device), 0, mine[2], mine[3])
        same(mine, want, 0)
    # fp16's largest values come back finite
    x = torch.full((1, 1, 64), 65504.0, dtype=torch.float16, device=device)
    mine = empty(1, 1, 4, 1, 64, device)
    ops.reshape_and_cache(x, x, mine[0], mine[1], torch.zeros(1, dtype=torch.int64, device=device), 0, mine[2], mine[3])
    assert float(mine[0].float()[0, 0, 0, 0, 0] * mine[2][0, 0, 0]) == 61440.0


@pytest.mark.parametrize("dtype,rows,count", [
    (torch.bfloat16, 1, 1), (torch.float32, 1, 1), (torch.float16, 3, 1), (torch.float16, 3, 3)])
def test_the_lowest_values_stay_finite(device, dtype, rows, count):
    # V rows of a type's lowest value: a weighted mean of them, not an infinity
    # (one row where a sum of two is past fp32)
    mine = empty(1, 1, 16, 1, 64, device)
    x = torch.full((rows, 1, 64), torch.finfo(dtype).min, dtype=dtype, device=device)
    slots = torch.arange(rows, device=device)
    ops.reshape_and_cache(torch.zeros_like(x), x, mine[0], mine[1], slots, 0, mine[2], mine[3])
    table = torch.zeros((1, 1), dtype=torch.int32, device=device)
    step = ops.pack_step(table, [rows - count], [count], 16, num_kv_heads=1, num_query_heads=4, head_dim=64, dtype=CODE)
    out = ops.attention(torch.ones((count, 4, 64), dtype=dtype, device=device), mine[0], mine[1], 0, step, 0.1,
                        key_scales=mine[2], value_scales=mine[3])
    # equal weights of equal values: a weight's rounding and the result's, 2^-10 in fp16, on either side of the value
    most = 61440.0 if dtype == torch.float16 else 1.875 * 2.0**127
    assert ((out.double() / -most - 1).abs() <= 2.0**-9).all()


def test_slots_outside_the_pool_are_skipped(device):
    mine = empty(1, 4, 8, 2, 64, device, garbage=True)
    slots = torch.tensor([-1, 0, 1, -5, 31, 32, 10**12])
    k = torch.randn((7, 2, 64)).to(torch.bfloat16).to(device)
    want = expect(mine, 0, k, k, slots)
    ops.reshape_and_cache(k, k, mine[0], mine[1], slots.to(device), 0, mine[2], mine[3])
    same(mine, want, 0)


def test_positions_outside_the_table_leave_their_k_rows_out(device):
    # beside a block's other rows: those are re-coded as the block grows, the
    # skipped row's too; V rows are written all the same
    bs, kv, dim = 8, 2, 64
    gen = torch.Generator().manual_seed(8)
    mine = empty(1, 4, bs, kv, dim, device, garbage=True)
    slots = torch.tensor([3, 4, 5, 8, 9, 10, 31])
    bad = torch.tensor([False, True, False, False, True, True, True])
    x = 20 * torch.randn((7, 4, dim), generator=gen).to(torch.bfloat16)
    q, k, v = x.to(device).split([2, 1, 1], dim=1)
    k, v = k.expand(-1, kv, -1), v.expand(-1, kv, -1)
    table = ops.rope_table(10, dim, device=device)
    pos = torch.where(bad, torch.tensor(10), torch.arange(7)).to(device)
    turned = ops.rotate(q, k.contiguous(), pos, table)[1]
    want = []
    for i, rows, at in ((0, turned, torch.where(bad, torch.tensor(-1), slots)), (1, v, slots)):
        want += oracle.write(mine[i][0].cpu().clone(), mine[2 + i][0].cpu().clone(), stored(rows), at.tolist())
    want[1][3], want[0][3] = mine[2][0, 3].cpu(), mine[0][0, 3].cpu()  # (nothing of it is written)
    out = ops.rotate_and_cache(q, k, v, mine[0], mine[1], slots.to(device), 0, pos, table, key_scales=mine[2],
                               value_scales=mine[3])
    assert torch.equal(torch.isnan(out).all(-1).all(-1).cpu(), bad)
    same(mine, want, 0)


def test_token_by_token_keeps_the_values(device):
    # Appending one row at a time only ever re-codes by powers of two: the
    # values are those of the whole block at once, but for subnormal codes.
    gen = torch.Generator().manual_seed(4)
    x = (torch.randn((16, 2, 64), generator=gen) * torch.logspace(-1, 1.5, 16)[:, None, None]).to(torch.bfloat16)
    x = x.to(device)
    one, whole = empty(1, 1, 16, 2, 64, device), empty(1, 1, 16, 2, 64, device)
    for t in range(16):
        ops.reshape_and_cache(x[t:t + 1], x[t:t + 1], one[0], one[1], torch.tensor([t], device=device), 0, one[2], one[3])
    ops.reshape_and_cache(x, x, whole[0], whole[1], torch.arange(16, device=device), 0, whole[2], whole[3])
    assert torch.equal(one[2], whole[2])
    a, b = (oracle.values(c[0][0].cpu(), c[2][0].cpu()) for c in (one, whole))
    # Where a value is normal under the last scale S it was under every earlier
    # one: the same four bits.  Below that (2^-6 S) the first rounding is off by
    # 2^-4 of it, 2^-10 S, each growth by half a subnormal step of its scale,
    # 2^-10 (S + S/2 + ...), and the whole block's by 2^-10 S.
    assert ((a - b).abs() <= 2.0**-8 * one[2][0].cpu().double()[:, None, :, None]).all()
    normal = b.abs() >= 2.0**-5 * one[2][0].cpu().double()[:, None, :, None]
    assert torch.equal(a[normal], b[normal])


@pytest.mark.parametrize("kv_heads,dim,bs,runs", WRITES[:5] + WRITES[7:8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rotate_and_cache_is_the_two_calls(device, kv_heads, dim, bs, runs, dtype):
    slots = torch.cat([torch.arange(a, a + n) for a, n in runs]).to(device)
    tokens, heads = len(slots), 2 * kv_heads
    gen = torch.Generator().manual_seed(7)
    x = torch.randn((tokens, heads + 2 * kv_heads, dim), generator=gen).to(dtype).to(device)
    q, k, v = x.split([heads, kv_heads, kv_heads], dim=1)
    w = (1 + 0.1 * torch.randn(dim, generator=gen)).to(dtype).to(device)
    table = ops.rope_table(tokens, dim, device=device)
    pos = torch.arange(tokens, device=device)
    blocks = int(slots.max()) // bs + 2
    want, mine = (empty(1, blocks, bs, kv_heads, dim, device, garbage=True) for _ in range(2))
    rq, rk = ops.rotate(q, k, pos, table, query_weight=w, key_weight=w)
    ops.reshape_and_cache(rk, v, want[0], want[1], slots, 0, want[2], want[3])
    got = ops.rotate_and_cache(q, k, v, mine[0], mine[1], slots, 0, pos, table, query_weight=w, key_weight=w,
                               key_scales=mine[2], value_scales=mine[3])
    assert torch.equal(got, rq)
    for a, b in zip(mine, want):
        assert torch.equal(a.view(torch.uint8) if a.dtype == CODE else a, b.view(torch.uint8) if b.dtype == CODE else b)


# ---- attention ---------------------------------------------------------------


def build(heads, kv_heads, dim, bs, starts, counts, dtype, device, holes=False, seed=0, layers=1):
    """A cache whose rows past each context are NaN codes and whose unused
    blocks have NaN scales, and the step's query."""
    gen = torch.Generator().manual_seed(seed)
    ends = [s + c for s, c in zip(starts, counts)]
    need = [-(-e // bs) for e in ends]
    blocks = sum(need) + 3
    perm = np.random.Generator(np.random.PCG64(seed)).permutation(blocks)
    table = np.full((len(ends), max(max(need), 1)), -1, dtype=np.int32)
    codes = [torch.full((layers, blocks, bs, kv_heads, dim), 0x7F, dtype=torch.uint8).view(CODE) for _ in range(2)]
    scales = [torch.full((layers, blocks, kv_heads), float("nan")) for _ in range(2)]
    at = 0
    for i, (e, n) in enumerate(zip(ends, need)):
        table[i, :n] = perm[at:at + n]
        at += n
        if e == 0:
            continue
        pos = np.arange(e)
        slots = (table[i, pos // bs].astype(np.int64) * bs + pos % bs).tolist()
        x = torch.randn((2, e, kv_heads, dim), generator=gen) * torch.exp(torch.randn((2, 1, kv_heads, dim), generator=gen))
        x = x * torch.exp(0.5 * torch.randn((2, e, 1, 1), generator=gen))
        for c, s, y in zip(codes, scales, x):
            oracle.write(c[-1], s[-1], y.to(torch.bfloat16).float(), slots)
        if holes and n > 2:
            table[i, n // 2] = -1
            if n > 4:
                table[i, 1] = blocks
    q = torch.randn((sum(counts), heads, dim), generator=gen).to(dtype)
    return q, codes, scales, table


def attend(heads, kv_heads, dim, bs, starts, counts, dtype, device, partition=None, holes=False, seed=0):
    q, codes, scales, table = build(heads, kv_heads, dim, bs, starts, counts, dtype, device, holes, seed)
    scale = 1.0 / np.sqrt(dim)
    dev = [t.to(device) for t in (*codes, *scales)]
    step = ops.pack_step(torch.from_numpy(table).to(device), starts, counts, bs, num_kv_heads=kv_heads,
                         num_query_heads=heads, head_dim=dim, dtype=CODE, partition_size=partition)
    out = torch.full((q.shape[0], heads, dim), 77.0, dtype=dtype, device=device)
    ops.attention(q.to(device), dev[0], dev[1], 0, step, scale, out=out, key_scales=dev[2], value_scales=dev[3])
    vals = [oracle.values(c[0], torch.nan_to_num(s[0])) for c, s in zip(codes, scales)]
    ref, size, peak = oracle.attention(q, *vals, table, starts, counts, scale)
    out = out.cpu().double()
    assert torch.isfinite(out).all()
    # One rounding of the result (u); a probability enters its product rounded
    # to the query's type, by u of itself at most, in the sum as in the
    # product (prefill) or one of the two (2 u in all; the decode takes two
    # terms, u^2); scores and sums in fp32, 1.5e-5 of a probability.  fp16's
    # steps below 2^-14 are 2^-24: of V, of the result, and of probabilities,
    # which count there from 2^14 (decode) or 2^6 (prefill) at the row's largest,
    # so that one is off by 2^-25 / 2^6 of the largest at most.
    u = oracle.ROW_EPS[dtype]
    several = torch.from_numpy(np.repeat(np.asarray(counts) > 1, counts))[:, None, None]
    each = torch.where(several, torch.tensor(2 * u), torch.tensor(u * u)) + 1.5e-5
    bound = (1 + 2 * u) * u * ref.abs() + each * size
    if dtype == torch.float16:
        bound = bound + 2.0**-24 + 2.0**-31 * peak
    excess = ((out - ref).abs() - bound).max().item()
    assert excess <= 0, f"{excess:.3e} over the bound"


CONTEXTS = [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257, 500]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,dim,bs", [
    (32, 8, 128, 16), (8, 8, 128, 16), (4, 4, 64, 16), (9, 3, 64, 16), (16, 2, 128, 32), (14, 2, 64, 16),
    (12, 1, 128, 16), (32, 1, 64, 16), (40, 2, 128, 16), (4, 2, 96, 16), (6, 2, 80, 32), (4, 4, 128, 64),
    (4, 2, 128, 8), (4, 2, 64, 1), (3, 1, 256, 16), (6, 3, 112, 16), (2, 1, 40, 12), (3, 3, 7, 16)])
def test_decode(device, heads, kv_heads, dim, bs, dtype):
    attend(heads, kv_heads, dim, bs, [c - 1 for c in CONTEXTS], [1] * len(CONTEXTS), dtype, device, partition=128)


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (6, 3, 64), (4, 4, 96), (3, 1, 48)])
def test_decode_fp32_queries(device, heads, kv_heads, dim):
    attend(heads, kv_heads, dim, 16, [c - 1 for c in CONTEXTS], [1] * len(CONTEXTS), torch.float32, device)


@pytest.mark.parametrize("partition", [64, 256, 512, 2048])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 4, 64), (3, 1, 128), (16, 1, 96)])
def test_decode_partitions(device, heads, kv_heads, dim, partition):
    starts = [0, 511, 512, 513, 1500, 63, 4200]
    attend(heads, kv_heads, dim, 16, starts, [1] * len(starts), torch.bfloat16, device, partition=partition)


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [
    (32, 16, 64, torch.bfloat16), (16, 16, 128, torch.float16), (32, 8, 128, torch.bfloat16)])
def test_decode_of_many_sequences(device, heads, kv_heads, dim, dtype):
    # launches of more work than the chip holds at once, some of it to merge
    starts = [(7 * i) % 45 + (100 if i % 50 == 0 else 0) for i in range(540 * 8 // kv_heads)]
    attend(heads, kv_heads, dim, 16, starts, [1] * len(starts), dtype, device, partition=64)


@pytest.mark.parametrize("bs", [16, 4, 32])
def test_missing_blocks_and_empty_rows(device, bs):
    # holes in the tables, a sequence whose only block is missing
    starts, counts = [200, 300, 99, 0, 40, 120], [1, 1, 30, 1, 5, 70]
    attend(8, 2, 128, bs, starts, counts, torch.bfloat16, device, holes=True, partition=64)
    q, codes, scales, table = build(4, 2, 64, 16, [3, 20], [1, 4], torch.bfloat16, device)
    table[:] = -1
    step = ops.pack_step(torch.from_numpy(table).to(device), [3, 20], [1, 4], 16, num_kv_heads=2, num_query_heads=4,
                         head_dim=64, dtype=CODE)
    out = ops.attention(q.to(device), codes[0].to(device), codes[1].to(device), 0, step, 0.125,
                        key_scales=scales[0].to(device), value_scales=scales[1].to(device))
    assert torch.equal(out, torch.zeros_like(out))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,dim,bs", [
    (32, 8, 128, 16), (4, 4, 64, 16), (9, 3, 64, 32), (4, 2, 96, 16), (6, 2, 80, 32), (16, 1, 128, 16), (4, 2, 128, 8),
    (4, 2, 128, 64), (2, 1, 128, 1), (5, 1, 64, 128), (14, 2, 64, 16), (2, 1, 256, 16), (3, 1, 40, 12)])
def test_prefill(device, heads, kv_heads, dim, bs, dtype):
    starts, counts = [0, 0, 0, 17, 130, 64, 7, 250], [2, 16, 65, 30, 41, 64, 128, 3]
    attend(heads, kv_heads, dim, bs, starts, counts, dtype, device)


def test_prefill_long_and_mixed(device):
    attend(8, 2, 128, 16, [0, 700, 5, 999], [333, 129, 1, 1], torch.bfloat16, device)
    attend(4, 4, 64, 16, [1200, 0, 640, 3], [70, 1, 200, 1], torch.float16, device)


def test_prefill_fp32_queries(device):
    attend(4, 2, 64, 16, [0, 33], [40, 20], torch.float32, device)


@pytest.mark.parametrize("counts", [[1, 1], [20, 9]])
@pytest.mark.parametrize("heads,kv_heads,dim,bs", [(4, 2, 128, 16), (2, 2, 64, 4), (6, 2, 80, 16), (4, 2, 64, 1),
                                                   (2, 2, 40, 16), (2, 2, 256, 16)])
def test_fp16_queries_over_values_past_fp16(device, heads, kv_heads, dim, bs, counts):
    # bf16 rows with a value of 61440 and one of 65536: fp16 queries read the
    # first as it is and the second as an infinity, whatever kernel runs
    starts = [20 - counts[0], 21 - counts[1]]
    blocks = 2 * -(-21 // bs)
    gen = torch.Generator().manual_seed(dim)
    k = 0.1 * torch.randn((41, kv_heads, dim), generator=gen)
    v = torch.randn((41, kv_heads, dim), generator=gen)
    v[3, 0, 5], v[2, 0, 3], v[22, 1, 7] = 61440.0, 65536.0, -65536.0
    table = torch.arange(blocks, dtype=torch.int32).reshape(2, -1)
    slots = torch.cat([torch.arange(20), torch.arange(21) + blocks // 2 * bs])
    mine = empty(1, blocks, bs, kv_heads, dim, device)
    ops.reshape_and_cache(k.to(torch.bfloat16).to(device), v.to(torch.bfloat16).to(device), mine[0], mine[1],
                          slots.to(device), 0, mine[2], mine[3])
    vals = [oracle.values(c[0].cpu(), s[0].cpu()) for c, s in ((mine[0], mine[2]), (mine[1], mine[3]))]
    flat = vals[1].reshape(-1, kv_heads, dim)
    assert flat[slots[3], 0, 5] == 61440 and flat[slots[2], 0, 3] == 65536 and flat[slots[22], 1, 7] == -65536
    assert flat.abs()[slots].gt(60000).sum() == 3
    flat[flat.abs() > 65000] = 0.0
    q = torch.randn((sum(counts), heads, dim), generator=gen).to(torch.float16)
    step = ops.pack_step(table.to(device), starts, counts, bs, num_kv_heads=kv_heads, num_query_heads=heads, head_dim=dim,
                         dtype=CODE)
    out = ops.attention(q.to(device), mine[0], mine[1], 0, step, dim**-0.5, key_scales=mine[2], value_scales=mine[3])
    out = out.cpu().double()
    ref, size, peak = oracle.attention(q, *vals, table.numpy(), starts, counts, dim**-0.5)
    over = torch.zeros(out.shape, dtype=torch.bool)  # results that weigh an infinity
    group = heads // kv_heads
    over[:counts[0], :group, 3] = True
    over[counts[0]:, group:, 7] = True
    late = torch.cat([torch.arange(s, s + c) for s, c in zip(starts, counts)])
    sees = (late >= torch.tensor([2] * counts[0] + [2] * counts[1]))[:, None, None]  # (both are their third tokens)
    assert not torch.isfinite(out[over & sees]).any()
    # the others: as in attend() above, with one term of a probability
    u = 2.0**-11
    bound = (1 + 2 * u) * u * ref.abs() + (2 * u + 1.5e-5) * size + 2.0**-24 + 2.0**-31 * peak
    assert ((out - ref).abs() <= bound)[~over].all()


@pytest.mark.parametrize("dim,kv_heads,bs", [(128, 8, 16), (64, 8, 4), (40, 8, 16)])
def test_caches_past_32_bit_offsets(device, dim, kv_heads, bs):
    # a layer of more than 2^32 codes, its sequence in the last blocks: the same
    # rows, codes and results as in a small cache
    heads, need = 2 * kv_heads, 7
    blocks = 2**32 // (bs * kv_heads * dim) + 100
    small = [t.to(device) for t in empty(2, need, bs, kv_heads, dim, device)]
    large = [torch.empty((2, blocks, bs, kv_heads, dim), dtype=torch.uint8, device=device).view(CODE) for _ in range(2)]
    large += [torch.zeros((2, blocks, kv_heads), device=device) for _ in range(2)]
    total = need * bs - 3
    x = torch.randn((total, heads + 2 * kv_heads, dim), device=device).to(torch.bfloat16)
    q, k, v = x.split([heads, kv_heads, kv_heads], dim=1)
    rope = ops.rope_table(total, dim, device=device)
    tables = [torch.arange(n - need, n, dtype=torch.int32, device=device).reshape(1, -1) for n in (need, blocks)]
    for start, count in ((0, total - 1), (total - 1, 1)):
        outs = []
        for cache, table in zip((small, large), tables):
            step = ops.pack_step(table, [start], [count], bs, num_kv_heads=kv_heads, num_query_heads=heads, head_dim=dim,
                                 dtype=CODE)
            part = slice(start, start + count)
            rq = ops.rotate_and_cache(q[part], k[part], v[part], cache[0], cache[1], step.scatter_slots, 1,
                                      step.position_ids, rope, key_scales=cache[2], value_scales=cache[3])
            outs.append(ops.attention(rq, cache[0], cache[1], 1, step, dim**-0.5, key_scales=cache[2],
                                      value_scales=cache[3]))
        assert torch.equal(*outs) and torch.isfinite(outs[0]).all()
    for a, b in zip(small[:2], large[:2]):
        a, b = (t.view(torch.uint8)[1, -need:].reshape(need * bs, -1)[:total] for t in (a, b))
        assert torch.equal(a, b)
    for a, b in zip(small[2:], large[2:]):
        assert torch.equal(a[1], b[1, -need:])


# ---- together, as a server runs them ------------------------------------------


def test_steps_of_a_sequence(device):
    """Prompt chunks, then decodes, through rotate_and_cache and attention, and
    beside it the same in fp64 over the values the rules give."""
    heads, kv, dim, bs, dtype = 8, 2, 128, 16, torch.bfloat16
    gen = torch.Generator().manual_seed(0)
    mine = empty(2, 40, bs, kv, dim, device, garbage=True)
    table = np.random.Generator(np.random.PCG64(1)).permutation(40).astype(np.int32).reshape(2, 20)
    rope = ops.rope_table(320, dim, device=device)
    w = (1 + 0.1 * torch.randn(dim, generator=gen)).to(dtype).to(device)
    done = [0, 0]
    for counts in ([100, 1], [30, 17], [1, 1], [1, 1], [1, 150], [1, 1]):
        starts, done = done, [d + c for d, c in zip(done, counts)]
        t = sum(counts)
        x = (torch.randn((t, heads + 2 * kv, dim), generator=gen) * 2).to(dtype).to(device)
        q, k, v = x.split([heads, kv, kv], dim=1)
        step = ops.pack_step(torch.from_numpy(table).to(device), starts, counts, bs, num_kv_heads=kv,
                             num_query_heads=heads, head_dim=dim, dtype=CODE)
        rk = ops.rotate(q, k, step.position_ids, rope, query_weight=w, key_weight=w)[1]
        want = expect(mine, 1, rk, v, step.scatter_slots.cpu())
        rq = ops.rotate_and_cache(q, k, v, mine[0], mine[1], step.scatter_slots, 1, step.position_ids, rope,
                                  query_weight=w, key_weight=w, key_scales=mine[2], value_scales=mine[3])
        out = ops.attention(rq, mine[0], mine[1], 1, step, dim**-0.5, key_scales=mine[2], value_scales=mine[3])
        same(mine, want, 1)
        ref, size, _ = oracle.attention(rq.cpu(), oracle.values(want[0], want[1]), oracle.values(want[2], want[3]), table,
                                     starts, counts, dim**-0.5)
        u = 2.0**-8
        assert ((out.cpu().double() - ref).abs() <= 1.01 * u * ref.abs() + (2 * u + 1.5e-5) * size).all()
        # the same rows through attention()'s own write
        again = ops.attention(rq, mine[0], mine[1], 1, step, dim**-0.5, new_key=rk, new_value=v, key_scales=mine[2],
                              value_scales=mine[3])
        same(mine, want, 1)
        assert torch.equal(again, out)


def test_phases_streams_and_graphs(device):
    heads, kv, dim, bs, dtype = 8, 2, 128, 16, torch.bfloat16
    starts, counts = [900, 40, 2000, 300], [1, 1, 1, 20]
    q, codes, scales, table = build(heads, kv, dim, bs, starts, counts, dtype, device)
    q, kc, vc, ks, vs = (t.to(device) for t in (q, *codes, *scales))
    step = ops.pack_step(torch.from_numpy(table).to(device), starts, counts, bs, num_kv_heads=kv,
                         num_query_heads=heads, head_dim=dim, dtype=CODE, partition_size=256)
    args = dict(key_scales=ks, value_scales=vs)
    want = ops.attention(q, kc, vc, 0, step, 0.1, **args)
    out = torch.full_like(want, 7.0)
    ops.decode(q, kc, vc, 0, step, 0.1, out=out, **args)
    assert torch.equal(out[:3], want[:3]) and bool((out[3:] == 7).all())
    ops.decode(q, kc, vc, 0, step, 0.1, out=out, phases=1, **args)
    out[:3] = 5
    ops.decode(q, kc, vc, 0, step, 0.1, out=out, phases=2, **args)
    multi = [0, 2]  # one-partition rows belong to the first phase
    assert torch.equal(out[multi], want[multi])
    out = torch.full_like(want, 7.0)
    ops.prefill(q, kc, vc, 0, step, 0.1, out=out, **args)
    assert torch.equal(out[3:], want[3:]) and bool((out[:3] == 7).all())
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
    with torch.cuda.graph(graph):
        ops.attention(q, kc, vc, 0, step, 0.1, out=out, **args)
    for _ in range(3):
        q.copy_(torch.randn_like(q.float()).to(q.dtype))
        want = ops.attention(q, kc, vc, 0, step, 0.1, **args)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.attention(q, kc, vc, 0, step, 0.1, **args)
    side.synchronize()
    assert torch.equal(got, want)


def test_a_graph_of_two_layers_and_a_repacked_step(device):
    # two captured graphs of one step, two layers each, that share its workspace
    # and write their rows; the step moves on by a token between the replays
    heads, kv, dim, bs, dtype = 8, 2, 64, 16, torch.bfloat16
    starts, counts = [300, 40, 700], [1, 1, 1]
    table = torch.arange(3 * 60, dtype=torch.int32, device=device).reshape(3, 60).flip(1).contiguous()
    mine, want = (empty(2, 180, bs, kv, dim, device, garbage=True) for _ in range(2))
    for c in (*mine[:2], *want[:2]):  # no NaN codes in the contexts
        u = c.view(torch.uint8)
        u[(u & 0x7F) == 0x7F] = 0x30
    step = ops.pack_step(table, starts, counts, bs, num_kv_heads=kv, num_query_heads=heads, head_dim=dim, dtype=CODE,
                         partition_size=128)
    x = [torch.randn((3, heads + 2 * kv, dim), device=device).to(dtype) for _ in range(2)]
    outs = [torch.empty((3, heads, dim), dtype=dtype, device=device) for _ in range(2)]

    def layer(i, cache, step, out=None):
        q, k, v = x[i].split([heads, kv, kv], dim=1)
        return ops.attention(q, cache[0], cache[1], i, step, 0.125, out=out, new_key=k, new_value=v,
                             key_scales=cache[2], value_scales=cache[3])

    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    keep = [t.clone() for t in mine]
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph):
            layer(i, mine, step, outs[i])
    for t, k in zip(mine, keep):
        assert torch.equal(t.view(torch.uint8), k.view(torch.uint8))  # (a capture runs nothing)
    for move in range(4):
        now = [s + move for s in starts]
        if move:
            step.repack(now)
        fresh = ops.pack_step(table, now, counts, bs, num_kv_heads=kv, num_query_heads=heads, head_dim=dim, dtype=CODE,
                              partition_size=128)
        for t in x:
            t.copy_(torch.randn_like(t.float()).to(dtype) * 2**move)
        refs = [layer(i, want, fresh) for i in range(2)]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], refs[i]) and torch.isfinite(refs[i]).all()
        for a, b in zip(mine, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("heads,kv_heads,dim,bs,tokens", [
    (32, 8, 128, 16, 1100), (9, 3, 64, 16, 5000), (3, 1, 256, 16, 3500), (8, 8, 128, 16, 2101), (9, 3, 64, 32, 11111),
    (2, 2, 256, 8, 4203), (4, 2, 36, 4, 2100)])
def test_large_steps_are_their_parts(device, heads, kv_heads, dim, bs, tokens):
    # steps of more rows than the chip has lanes for, against calls of whole blocks
    gen = torch.Generator(device=device).manual_seed(2)
    x = torch.randn((tokens, heads + 2 * kv_heads, dim), generator=gen, device=device).to(torch.bfloat16)
    q, k, v = x.split([heads, kv_heads, kv_heads], dim=1)
    w = (1 + 0.1 * torch.randn(dim, generator=gen, device=device)).to(torch.bfloat16)
    rope, pos = ops.rope_table(tokens, dim, device=device), torch.arange(tokens, device=device)
    blocks = -(-tokens // bs) + 1
    slots = torch.arange(tokens, device=device)
    for codes in (False, True):
        if codes:
            mine, want = (empty(1, blocks, bs, kv_heads, dim, device) for _ in range(2))
        else:
            mine, want = ([torch.zeros((1, blocks, bs, kv_heads, dim), dtype=torch.bfloat16, device=device)
                           for _ in range(2)] + [None, None] for _ in range(2))

        def call(cache, lo, hi):
            return ops.rotate_and_cache(q[lo:hi], k[lo:hi], v[lo:hi], cache[0], cache[1], slots[lo:hi], 0, pos[lo:hi],
                                        rope, query_weight=w, key_scales=cache[2], value_scales=cache[3])

        got = call(mine, 0, tokens)
        parts = torch.cat([call(want, lo, min(lo + 160, tokens)) for lo in range(0, tokens, 160)])
        assert torch.equal(got, parts)
        for a, b in zip(mine, want):
            assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_a_store_behind_the_layers_hook(device):
    # a store of 8-bit codes as an engine runs it: prompts, a prompt in chunks,
    # decodes and a swap, every layer's result against fp64 over what the store holds
    heads, kv, dim, layers, dtype = 8, 2, 64, 2, torch.bfloat16
    hook = pkg("model.paged_attention")
    metrics = pkg("metrics")
    request = pkg("engine.request").Request
    store = pkg("memory.manager").PagedKVCacheManager(total_blocks=64, block_size=16, num_heads=kv, head_dim=dim,
                                                      dtype=CODE, num_layers=layers, device=device, total_cpu_blocks=16)
    store.num_query_heads = heads
    gen = torch.Generator(device=device).manual_seed(5)

    class Layer:
        scaling = dim**-0.5

    seqs = [request(i, list(range(n))) for i, n in enumerate((37, 120))]
    for seq in seqs:
        store.allocate_prefix_blocks(seq)
    recorder = metrics.enable()
    try:
        for starts, counts in (([0, 0], [37, 64]), ([37, 64], [1, 56]), ([38, 120], [1, 1]), ([39, 121], [1, 1])):
            for seq, start, count in zip(seqs, starts, counts):
                while seq.block_table.get_tokens_count() < start + count:
                    store.allocate_slot_for_next_token(seq)
            context = hook.PagedStepContext(store, seqs, starts, counts)
            t = sum(counts)
            for i in range(layers):
                x = 2 * torch.randn((1, heads + 2 * kv, t, dim), generator=gen, device=device).to(dtype)
                q, k, v = x.split([heads, kv, kv], dim=1)
                module = Layer()
                module.paged_context, module.layer_idx = context, i
                out = hook.paged_attention_forward(module, q, k, v)[0][0].cpu().double()
                rows = [store.gather_layer_keys(i, context.gather_slots), store.gather_layer_values(i, context.gather_slots)]
                new = torch.cat([torch.arange(c)[s:] + o for o, s, c in zip(
                    (0, starts[0] + counts[0]), starts, [a + b for a, b in zip(starts, counts)])]).to(device)
                # half a step of e4m3, or of its least numbers (values below 16 keep scales below 16 / 224)
                for got, given in zip(rows, (k, v)):
                    given = given[0].transpose(0, 1).float()
                    off = (got[new].float() - given).abs()
                    assert (off <= 2.0**-4 * given.abs() + 2.0**-10 * 16 / 224).all()
                n = [a + b for a, b in zip(starts, counts)]
                pool = [torch.zeros((2, 256, kv, dim), dtype=torch.float64) for _ in range(2)]
                for p, r in zip(pool, rows):
                    for j, part in enumerate(r.cpu().double().split(n)):
                        p[j, :n[j]] = part
                ref, size, _ = oracle.attention(q[0].transpose(0, 1).cpu(), *pool, [[0], [1]], starts, counts, dim**-0.5)
                u = 2.0**-8
                assert ((out - ref).abs() <= 1.01 * u * ref.abs() + (2 * u + 1.5e-5) * size).all()
            store.swap_out(seqs[0])
            store.swap_in(seqs[0])
        torch.cuda.synchronize()
        assert recorder.poll() > 0
    finally:
        metrics.disable()


def test_blocks_are_copied_and_swapped_with_their_scales(device):
    store_of = pkg("memory.manager").PagedKVCacheManager
    store = store_of(total_blocks=32, block_size=16, num_heads=2, head_dim=64, dtype=CODE, num_layers=2, device=device)
    request = pkg("engine.request").Request
    seq = request(1, list(range(50)))
    store.allocate_prefix_blocks(seq)
    gen = torch.Generator().manual_seed(3)
    k, v = (torch.randn((2, 50, 2, 64), generator=gen).to(torch.bfloat16).to(device) for _ in range(2))
    slots = store.write_prefix_kv(seq, k, v)
    before = store.gather_kv_cache(seq)
    for layer in range(2):
        got = before[layer][0][0].transpose(0, 1).float()
        # e4m3's half step is 2^-4 of a value, 2^-10 of the scale below its
        # least normal one; the scale is less than max / 224
        x = k[layer].float()
        assert ((got - x).abs() <= 2.0**-4 * x.abs() + 2.0**-10 * x.abs().max() / 224).all()
    store.swap_out(seq)
    other = request(2, list(range(500)))
    store.allocate_prefix_blocks(other)
    store.write_prefix_kv(other, 9 * torch.ones((2, 500, 2, 64), device=device), torch.ones((2, 500, 2, 64), device=device))
    store.free_sequence(other)
    store.swap_in(seq)
    after = store.gather_kv_cache(seq)
    for a, b in zip(before, after):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    copy = [torch.zeros_like(store.key_cache), torch.zeros_like(store.key_scales)]
    pairs = [(int(b), int(b)) for b in seq.block_table.get_physical_blocks()]
    ops.copy_blocks(store.key_cache, copy[0], pairs)
    ops.copy_blocks(ops.scales_as_blocks(store.key_scales), ops.scales_as_blocks(copy[1]), pairs)
    ids = [b for b, _ in pairs]
    assert torch.equal(copy[0].view(torch.uint8)[:, ids], store.key_cache.view(torch.uint8)[:, ids])
    assert torch.equal(copy[1][:, ids], store.key_scales[:, ids])
    assert slots.numel() == 50
