"""Rotation of Q and K rows (paged_ops.rotate) and its append to the paged
cache (paged_ops.rotate_and_cache) against the formulas in fp64."""

import numpy as np
import pytest
import torch

import cache8_oracle as oracle
from helpers import pkg

pytestmark = pytest.mark.gpu

ops = pkg("paged_ops")
EPS = 1e-6


def rows(tokens, heads, kv_heads, dim, dtype, seed=0, fused=True):
    """Q, K, V as views of one projection's output (or tensors of their own)."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((tokens, heads + 2 * kv_heads, dim), generator=gen) * torch.exp(torch.randn(dim, generator=gen))
    x = x.to(dtype).cuda()
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    return (q, k, v) if fused else (q.contiguous(), k.contiguous(), v.contiguous())


def weights(dim, dtype, seed=1):
    gen = torch.Generator().manual_seed(seed)
    return [(1 + 0.3 * torch.randn(dim, generator=gen)).to(dtype).cuda() for _ in range(2)]


def check(got, x, weight, positions, table, interleaved):
    ref, size = oracle.rotated(x.cpu(), None if weight is None else weight.cpu(), positions.cpu(), table.cpu(), EPS,
                               interleaved)
    got = got.cpu().double()
    u = oracle.ROW_EPS[x.dtype]
    # The norm's factor: a lane's 8 squares in a chain, 6 levels over the
    # lanes, a division, an addition and rsqrt (2 units): 12 half-units (2^-24)
    # and twice 2 for the products with it and the weight; a rotated element:
    # two products and a sum, 2 half-units of |a cos| + |b sin| <= |a| + |b|.
    # 20 half-units of |a| + |b| hold it all, 32 are allowed; then one rounding.
    bound = u * ref.abs() + 32 * 2.0**-24 * (1 + u) * size + (2.0**-25 if x.dtype == torch.float16 else 0)
    excess = ((got - ref).abs() - bound).max().item()
    assert excess <= 0, f"{excess:.3e} over the bound"


SHAPES = [  # heads, kv_heads, dim, rotary, interleaved
    (32, 8, 128, 128, False), (8, 8, 64, 64, False), (9, 3, 64, 32, True), (4, 1, 96, 96, False),
    (4, 4, 80, 80, True), (2, 1, 256, 256, False), (2, 2, 256, 64, True), (3, 3, 40, 24, False), (2, 1, 8, 8, False),
    (5, 5, 36, 20, False), (2, 1, 100, 100, True), (3, 1, 7, 6, False), (2, 1, 7, 2, True), (1, 1, 250, 126, False),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("norm", [None, "rows", "fp32"])
@pytest.mark.parametrize("heads,kv_heads,dim,rotary,interleaved", SHAPES)
def test_rotate(device, heads, kv_heads, dim, rotary, interleaved, norm, dtype):
    for tokens in (1, 19):
        q, k, _ = rows(tokens, heads, kv_heads, dim, dtype, seed=tokens)
        qw, kw = (None, None) if norm is None else weights(dim, torch.float32 if norm == "fp32" else dtype)
        table = ops.rope_table(500, rotary, device=device)
        pos = torch.randint(0, 500, (tokens,), generator=torch.Generator().manual_seed(5)).to(device)
        pos[0] = 499
        got_q, got_k = ops.rotate(q, k, pos, table, query_weight=qw, key_weight=kw, eps=EPS, interleaved=interleaved)
        check(got_q, q, qw, pos, table, interleaved)
        check(got_k, k, kw, pos, table, interleaved)


@pytest.mark.parametrize("dim", [64, 36])
def test_one_weight_and_in_place(device, dim):
    q, k, _ = rows(11, 6, 2, dim, torch.bfloat16)
    kw = weights(dim, torch.bfloat16)[1]
    table = ops.rope_table(64, 12 if dim == 36 else dim, device=device)
    pos = torch.arange(11, device=device) * 3
    want_q, want_k = ops.rotate(q, k, pos, table, key_weight=kw)
    check(want_q, q, None, pos, table, False)
    check(want_k, k, kw, pos, table, False)
    got = ops.rotate(q, k, pos, table, key_weight=kw, out_query=q, out_key=k)
    assert got[0] is q and got[1] is k
    assert torch.equal(q, want_q) and torch.equal(k, want_k)


def test_rows_of_zeros_and_strides(device):
    # The norm of a row of zeros is zeros (eps); rows through transposed and
    # sliced views, an odd element offset (no vector loads), a step over tokens.
    gen = torch.Generator().manual_seed(2)
    base = torch.randn((4, 21, 66), generator=gen).to(torch.bfloat16).to(device)
    q = base.transpose(0, 1)[::2, :, 1:65]
    k = torch.zeros((11, 2, 64), dtype=torch.bfloat16, device=device)
    w = weights(64, torch.bfloat16)
    table = ops.rope_table(32, 64, device=device)
    pos = torch.arange(11, device=device)
    got_q, got_k = ops.rotate(q, k, pos, table, query_weight=w[0], key_weight=w[1])
    check(got_q, q, w[0], pos, table, False)
    assert torch.equal(got_k, k)
    # columns with a stride are copied first
    got, _ = ops.rotate(base.transpose(1, 2)[..., :4].transpose(0, 1)[:11], k[:, :, :4].contiguous(), pos,
                        ops.rope_table(32, 4, device=device))
    check(got, base.transpose(1, 2)[..., :4].transpose(0, 1)[:11], None, pos, ops.rope_table(32, 4, device=device),
          False)


def test_positions_outside_the_table(device):
    q, k, v = rows(6, 4, 2, 64, torch.float32)
    table = ops.rope_table(10, 64, device=device)
    pos = torch.tensor([0, 10, 9, -1, 2**40, 3], device=device)
    bad = torch.tensor([False, True, False, True, True, False])
    got_q, got_k = ops.rotate(q, k, pos, table)
    assert torch.equal(torch.isnan(got_q).all(-1).all(-1).cpu(), bad)
    assert torch.equal(torch.isnan(got_k).any(-1).any(-1).cpu(), bad)
    caches = [torch.full((1, 2, 4, 2, 64), 7.0, device=device) for _ in range(2)]
    got = ops.rotate_and_cache(q, k, v, *caches, torch.arange(6, device=device), 0, pos, table)
    assert torch.equal(torch.isnan(got).all(-1).all(-1).cpu(), bad)
    flat = caches[0].view(-1, 2, 64)[:6].cpu()
    assert bool((flat[bad] == 7).all()) and not bool((flat[~bad] == 7).any())
    assert torch.equal(caches[1].view(-1, 2, 64)[:6], v)


def test_far_positions(device):
    # fp32 angles would be off by 2^-24 * 2^20 = 0.06 here
    table = ops.rope_table(1 << 20, 64, theta=500000.0, device=device)
    p = (1 << 20) - 1
    want = p * 500000.0 ** (-np.arange(0, 64, 2) / 64)
    # (the angle is one fp64 product: off by 2^20 * 2^-52 at most)
    assert np.abs(table[p, :32].double().cpu().numpy() - np.cos(want)).max() < 2.0**-24
    assert np.abs(table[p, 32:].double().cpu().numpy() - np.sin(want)).max() < 2.0**-24


def cache_of(shape, dtype, device, seed=3):
    gen = torch.Generator(device=device).manual_seed(seed)
    return [torch.randn(shape, generator=gen, device=device).to(dtype) for _ in range(2)]


@pytest.mark.parametrize("heads,kv_heads,dim,rotary,interleaved", SHAPES[:6] + SHAPES[9:12])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rotate_and_cache_is_the_two_calls(device, heads, kv_heads, dim, rotary, interleaved, dtype):
    tokens = 37
    q, k, v = rows(tokens, heads, kv_heads, dim, dtype)
    w = weights(dim, dtype)
    table = ops.rope_table(100, rotary, device=device)
    pos = torch.arange(tokens, device=device)
    slots = torch.randperm(2 * 5 * 8, generator=torch.Generator().manual_seed(1))[:tokens].to(device)
    slots[5], slots[7] = -1, 10 * 8  # skipped
    want, mine = cache_of((2, 10, 8, kv_heads, dim), dtype, device), cache_of((2, 10, 8, kv_heads, dim), dtype, device)
    rq, rk = ops.rotate(q, k, pos, table, query_weight=w[0], key_weight=w[1], interleaved=interleaved)
    ops.reshape_and_cache(rk, v, *want, slots, 1)
    out = torch.empty_like(rq)
    got = ops.rotate_and_cache(q, k, v, *mine, slots, 1, pos, table, query_weight=w[0], key_weight=w[1],
                               interleaved=interleaved, out=out)
    assert got is out and torch.equal(got, rq)
    assert torch.equal(mine[0], want[0]) and torch.equal(mine[1], want[1])


@pytest.mark.parametrize("dim", [64, 36])
def test_rows_that_do_not_turn(device, dim):
    # the library's call without a table: norms alone
    native = pkg("_native")
    q, k, _ = rows(21, 4, 2, dim, torch.bfloat16)
    w = weights(dim, torch.bfloat16)
    outs = [torch.empty((21, n, dim), dtype=torch.bfloat16, device=device) for n in (4, 2)]
    dims = native.PaRotateDims(
        num_tokens=21, num_query_heads=4, num_kv_heads=2, head_dim=dim, dtype=native.PA_DTYPE_BF16,
        weight_dtype=native.PA_DTYPE_BF16, eps=EPS, query_token_stride=q.stride(0), query_head_stride=dim,
        key_token_stride=k.stride(0), key_head_stride=dim, query_out_token_stride=4 * dim, query_out_head_stride=dim,
        key_out_token_stride=2 * dim, key_out_head_stride=dim)
    status = native.load_library().pa_rotate(
        dims, q.data_ptr(), k.data_ptr(), None, None, w[0].data_ptr(), w[1].data_ptr(), outs[0].data_ptr(),
        outs[1].data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert status == native.PA_OK
    still = torch.cat([torch.ones(1, dim // 2), torch.zeros(1, dim // 2)], 1)  # cosines, sines
    for got, x, weight in zip(outs, (q, k), w):
        check(got, x, weight, torch.zeros(21, dtype=torch.int64), still, False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (3, 3, 64), (2, 1, 256), (2, 1, 36), (3, 1, 7)])
def test_norms_alone(device, heads, kv_heads, dim, dtype):
    # positions and a table of None: rows are normalised and stay where they are
    q, k, v = rows(37, heads, kv_heads, dim, dtype)
    w = weights(dim, dtype)
    still = torch.cat([torch.ones(1, dim // 2), torch.zeros(1, dim // 2)], 1)  # cosines, sines
    got = ops.rotate(q, k, None, None, query_weight=w[0], key_weight=w[1], eps=EPS)
    for y, x, weight in zip(got, (q, k), w):
        check(y, x, weight, torch.zeros(37, dtype=torch.int64), still, False)
    same = ops.rotate(q, k, None, None)  # nothing to do: the rows
    assert torch.equal(same[0], q) and torch.equal(same[1], k)
    slots = torch.arange(37, device=device) + 3
    for code in (dtype, oracle.CODE):
        want, mine = ([t.to(code) for t in cache_of((2, 6, 8, kv_heads, dim), torch.float32, device)] for _ in range(2))
        scales = [[torch.ones((2, 6, kv_heads), device=device) for _ in range(2)] for _ in range(2)]
        if code is not oracle.CODE:
            scales = [[None, None], [None, None]]
        ops.reshape_and_cache(got[1], v, *want, slots, 1, *scales[0])
        out = ops.rotate_and_cache(q, k, v, *mine, slots, 1, None, None, query_weight=w[0], key_weight=w[1], eps=EPS,
                                   key_scales=scales[1][0], value_scales=scales[1][1])
        assert torch.equal(out, got[0])
        for a, b in zip(mine, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert code is not oracle.CODE or all(torch.equal(a, b) for a, b in zip(*scales))


def test_no_tokens(device):
    q, k, v = rows(0, 4, 2, 64, torch.bfloat16)
    table = ops.rope_table(4, 64, device=device)
    none = torch.empty(0, dtype=torch.int64, device=device)
    caches = cache_of((1, 2, 4, 2, 64), torch.bfloat16, device)
    assert ops.rotate_and_cache(q, k, v, *caches, none, 0, none, table).shape == (0, 4, 64)
    assert ops.rotate(q, k, none, table)[1].shape == (0, 2, 64)


def test_on_another_stream_and_in_a_graph(device):
    q, k, v = rows(33, 8, 2, 128, torch.bfloat16)
    table = ops.rope_table(100, 128, device=device)
    pos, slots = torch.arange(33, device=device), torch.arange(33, device=device) + 5
    want, mine = cache_of((1, 8, 16, 2, 128), torch.bfloat16, device), cache_of((1, 8, 16, 2, 128), torch.bfloat16, device)
    ref = ops.rotate_and_cache(q, k, v, *want, slots, 0, pos, table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.rotate_and_cache(q, k, v, *mine, slots, 0, pos, table)
    side.synchronize()
    assert torch.equal(got, ref) and torch.equal(mine[0], want[0])
    out = torch.empty_like(ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rotate_and_cache(q, k, v, *mine, slots, 0, pos, table, out=out)
    for i in range(3):
        q.copy_(torch.randn_like(q.float()).to(q.dtype))
        pos.add_(i)
        ref = ops.rotate_and_cache(q, k, v, *want, slots, 0, pos, table)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(mine[0], want[0]) and torch.equal(mine[1], want[1])
