"""What the rotation and the 8-bit cache refuse, without a GPU."""

import ctypes

import pytest
import torch

import cache8_oracle as oracle
from helpers import pkg

native = pkg("_native")
ops = pkg("paged_ops")

needs_library = pytest.mark.skipif(not native.library_built(), reason="the HIP library is not built")
CODE = torch.float8_e4m3fn


def caches(dtype=CODE, shape=(2, 4, 16, 2, 64)):
    return torch.zeros(shape, dtype=dtype), torch.zeros(shape, dtype=dtype)


def test_scales_go_with_their_cache():
    k, v = caches()
    good = torch.zeros((2, 4, 2))
    assert ops._cache_scales(k, v, good, good).key == good.data_ptr()
    assert ops._cache_scales(*caches(torch.bfloat16), None, None) is None
    for ks, vs in ((None, None), (good, None), (good.double(), good), (good[:1], good), (good, torch.zeros((2, 4, 3))),
                   (torch.zeros((2, 2, 4)).transpose(1, 2), good), (good, good.to("meta"))):
        with pytest.raises(ValueError):
            ops._cache_scales(k, v, ks, vs)
    with pytest.raises(ValueError):
        ops._cache_scales(*caches(torch.bfloat16), good, good)
    with pytest.raises(ValueError):
        ops._cache_scales(k, v.to(torch.bfloat16), good, good)


def test_cpu_tensors_are_refused():
    k, v = caches()
    s, rows, slots = torch.zeros((2, 4, 2)), torch.zeros((1, 2, 64)), torch.zeros(1, dtype=torch.int64)
    table = ops.rope_table(4, 64)
    with pytest.raises(RuntimeError, match="device tensors"):
        ops.reshape_and_cache(rows, rows, k, v, slots, 0, s, s)
    with pytest.raises(RuntimeError, match="device tensors"):
        ops.rotate(rows, rows, slots, table)
    with pytest.raises(RuntimeError, match="device tensors"):
        ops.rotate_and_cache(rows, rows, rows, k, v, slots, 0, slots, table, key_scales=s, value_scales=s)


def test_a_cpu_store_of_codes_is_refused():
    with pytest.raises(ValueError, match="device memory"):
        pkg("memory.manager").PagedKVCacheManager(4, 16, 2, 64, dtype=CODE, device="cpu")
    assert pkg("memory.strategies").resolve_dtype("fp8") is CODE


def test_bytes_of_a_step():
    # 17 and 32 tokens in blocks of 16: two blocks each; K and V codes of two
    # heads of 64, their scales, bf16 rows of 8 heads in and out, the table
    got = pkg("metrics").step_bytes([17, 32], 2, 8, 2, 64, 1, 16, 2)
    assert got == 49 * 2 * 2 * 64 + 4 * 2 * 2 * 4 + 2 * 8 * 64 * 2 * 2 + 4 * 4 + 2 * 4


def test_rope_table():
    t = ops.rope_table(5, 8, theta=100.0)
    assert t.shape == (5, 8) and t.dtype == torch.float32
    angle = 3 * 100.0 ** (-torch.arange(0, 8, 2, dtype=torch.float64) / 8)
    assert torch.equal(t[3], torch.cat([angle.cos(), angle.sin()]).float())
    for bad in ((5, 7), (5, 0), (0, 8), (5, -2)):
        with pytest.raises(ValueError):
            ops.rope_table(*bad)


def rotation_call(q=(3, 4, 64), k=(3, 2, 64), dtype=torch.bfloat16, kdtype=None, pos=None, table=None, **kw):
    return ops._rotate_dims(torch.zeros(q, dtype=dtype), torch.zeros(k, dtype=kdtype or dtype),
                              torch.zeros(3, dtype=torch.int64) if pos is None else pos,
                              ops.rope_table(8, 64) if table is None else table, kw.get("qw"), kw.get("kw"), 1e-6, False)


def test_rotation_arguments():
    assert rotation_call().rotary_dim == 64
    f32, bf16 = torch.ones(64), torch.ones(64, dtype=torch.bfloat16)
    assert rotation_call(qw=f32, kw=f32).weight_dtype == native.PA_DTYPE_F32
    assert rotation_call(kw=bf16).weight_dtype == native.PA_DTYPE_BF16
    bad = [dict(q=(3, 64)), dict(q=(2, 4, 64)), dict(k=(3, 2, 32)), dict(kdtype=torch.float32), dict(dtype=torch.float64),
           dict(pos=torch.zeros(3, dtype=torch.int32)), dict(pos=torch.zeros(4, dtype=torch.int64)),
           dict(table=ops.rope_table(8, 66)), dict(table=ops.rope_table(8, 64).double()),
           dict(table=torch.zeros((8, 33))), dict(table=torch.zeros((0, 64))), dict(table=torch.zeros((8, 0))),
           dict(table=torch.zeros((64, 8)).t()), dict(qw=torch.ones(32)), dict(qw=torch.ones(64, dtype=torch.float16)),
           dict(qw=f32, kw=bf16), dict(kw=torch.ones((64, 2))[:, 0])]
    for kw in bad:
        with pytest.raises(ValueError):
            rotation_call(**kw)


def test_rows_without_a_rotation():
    rows = [torch.zeros((3, n, 64), dtype=torch.bfloat16) for n in (4, 2)]
    dims = ops._rotate_dims(*rows, None, None, None, torch.ones(64), 1e-6, False)
    assert dims.rotary_dim == 0 and dims.num_positions == 0 and dims.weight_dtype == native.PA_DTYPE_F32
    for pos, table in ((None, ops.rope_table(8, 64)), (torch.zeros(3, dtype=torch.int64), None)):
        with pytest.raises(ValueError, match="together"):
            ops._rotate_dims(*rows, pos, table, None, None, 1e-6, False)


def test_outputs_of_rows():
    like = torch.zeros((3, 4, 64), dtype=torch.bfloat16)
    ops._check_rows_out(torch.zeros((4, 3, 64), dtype=torch.bfloat16).transpose(0, 1), like, "out")
    ops._check_rows_out(torch.zeros((3, 8, 64), dtype=torch.bfloat16)[:, 2:6], like, "out")
    for bad in (like.float(), like[:2], torch.zeros((1, 4, 64), dtype=torch.bfloat16).expand(3, 4, 64),
                torch.zeros((3, 64, 4), dtype=torch.bfloat16).transpose(1, 2), like.to("meta"),
                torch.zeros(1000, dtype=torch.bfloat16).as_strided((3, 4, 64), (64, 64, 1))):
        with pytest.raises(ValueError):
            ops._check_rows_out(bad, like, "out")


def test_the_least_scale():
    for amax, e in ((0.0, -64), (1e-30, -64), (448.0, 0), (448.5, 1), (224.0, -1), (1.0, -8), (1.75, -8), (1.76, -7)):
        assert oracle.scale_for(amax) == 2.0**e


FAKE = 1 << 20  # never read: the call is refused first


def dims_of(**kw):
    d = dict(num_tokens=3, num_query_heads=4, num_kv_heads=2, head_dim=64, block_size=16, total_blocks=4, num_layers=2,
             dtype=native.PA_DTYPE_BF16, cache_dtype=native.PA_DTYPE_BF16, weight_dtype=native.PA_DTYPE_BF16,
             num_positions=8, rotary_dim=64, eps=1e-6)
    d.update(kw)
    return ctypes.byref(native.PaRotateDims(**d))


POINTERS = dict(query=FAKE, key=FAKE, value=FAKE, positions=FAKE, cos_sin=FAKE, query_weight=None, key_weight=None,
                query_out=FAKE, key_cache=FAKE, value_cache=FAKE, key_scales=None, value_scales=None, slots=FAKE)


def rotate(dims, **kw):
    p = {**POINTERS, **kw}
    return native.load_library().pa_rotate(dims, p["query"], p["key"], p["positions"], p["cos_sin"], p["query_weight"],
                                           p["key_weight"], p["query_out"], p.get("key_out", FAKE), None)


def rotate_and_cache(dims, layer=0, **kw):
    return native.load_library().pa_rotate_and_cache(dims, *{**POINTERS, **kw}.values(), layer, None)


@needs_library
@pytest.mark.parametrize("dims,pointers,status", [
    (dict(dtype=9), {}, native.PA_ERR_INVALID_ARGUMENT),
    (dict(dtype=native.PA_DTYPE_E4M3, cache_dtype=native.PA_DTYPE_E4M3), {}, native.PA_ERR_INVALID_ARGUMENT),
    (dict(num_tokens=-1), {}, native.PA_ERR_INVALID_ARGUMENT),
    (dict(num_query_heads=0), {}, native.PA_ERR_INVALID_ARGUMENT),
    (dict(num_kv_heads=0), {}, native.PA_ERR_INVALID_ARGUMENT),
    (dict(head_dim=264), {}, native.PA_ERR_UNSUPPORTED),
    (dict(num_tokens=1 << 30), {}, native.PA_ERR_UNSUPPORTED),
    (dict(rotary_dim=63), {}, native.PA_ERR_INVALID_ARGUMENT),
    (dict(rotary_dim=66), {}, native.PA_ERR_INVALID_ARGUMENT),
    (dict(rotary_dim=-2), {}, native.PA_ERR_INVALID_ARGUMENT),
    (dict(num_positions=0), {}, native.PA_ERR_INVALID_ARGUMENT),
    ({}, dict(positions=None), native.PA_ERR_INVALID_ARGUMENT),
    ({}, dict(cos_sin=None), native.PA_ERR_INVALID_ARGUMENT),
    ({}, dict(query=None), native.PA_ERR_INVALID_ARGUMENT),
    ({}, dict(key=None), native.PA_ERR_INVALID_ARGUMENT),
    ({}, dict(query_out=None), native.PA_ERR_INVALID_ARGUMENT),
    (dict(weight_dtype=native.PA_DTYPE_F16), dict(query_weight=FAKE), native.PA_ERR_INVALID_ARGUMENT),
    (dict(num_tokens=0), {}, native.PA_OK),
])
def test_rotations_the_library_refuses(dims, pointers, status):
    assert rotate(dims_of(**dims), **pointers) == status
    assert rotate_and_cache(dims_of(**dims), **pointers) == status


@needs_library
def test_caches_the_library_refuses():
    lib = native.load_library()
    codes = dict(cache_dtype=native.PA_DTYPE_E4M3)
    bad = native.PA_ERR_INVALID_ARGUMENT
    assert rotate_and_cache(dims_of(**codes)) == bad
    assert b"scales" in lib.pa_last_error_message()
    assert rotate_and_cache(dims_of(**codes), key_scales=FAKE) == bad
    assert rotate_and_cache(dims_of(), key_scales=FAKE, value_scales=FAKE) == bad
    assert rotate_and_cache(dims_of(cache_dtype=native.PA_DTYPE_F16)) == bad
    assert rotate_and_cache(dims_of(block_size=0)) == bad
    assert rotate_and_cache(dims_of(), layer=2) == bad and rotate_and_cache(dims_of(), layer=-1) == bad
    for name in ("key_cache", "value_cache", "slots", "value"):
        assert rotate_and_cache(dims_of(), **{name: None}) == bad
    assert rotate_and_cache(dims_of(block_size=257, **codes), key_scales=FAKE,
                            value_scales=FAKE) == native.PA_ERR_UNSUPPORTED
    assert rotate(None) == bad and rotate_and_cache(None) == bad and rotate(dims_of(), key_out=None) == bad

    def write(dtype=native.PA_DTYPE_BF16, key=FAKE, scales=FAKE, layer=0, bs=16, tokens=1, dim=64):
        return lib.pa_reshape_and_cache_8bit(key, FAKE, 64, 64, 64, 64, FAKE, FAKE, scales, scales, FAKE, tokens, 2,
                                             dim, bs, 4, 1, layer, dtype, None)

    assert write(dtype=native.PA_DTYPE_E4M3) == bad and write(key=None) == bad and write(scales=None) == bad
    assert write(layer=1) == bad and write(bs=512) == native.PA_ERR_UNSUPPORTED and write(tokens=0) == native.PA_OK
    assert write(dim=257) == native.PA_ERR_UNSUPPORTED


@needs_library
def test_attention_the_library_refuses():
    lib = native.load_library()
    dims = native.PaStepDims(num_seqs=1, num_query_tokens=1, num_query_heads=4, num_kv_heads=2, head_dim=64,
                             block_size=16, total_blocks=4, num_layers=1, max_blocks_per_seq=1, partition_size=64,
                             dtype=native.PA_DTYPE_BF16)

    def decode(d=dims, key=FAKE, value=FAKE, layer=0, query=FAKE):
        return lib.pa_decode_8bit(3, query, FAKE, FAKE, native.PaCacheScales(key, value), layer, d, FAKE, FAKE, FAKE, FAKE,
                                  1, None, 0, 1.0, FAKE, None, 0, None)

    def prefill(d=dims, key=FAKE, value=FAKE, layer=0, query=FAKE):
        return lib.pa_prefill_8bit(query, FAKE, FAKE, native.PaCacheScales(key, value), layer, d, FAKE, FAKE, FAKE, FAKE,
                                   1, 128, 1.0, FAKE, None)

    bad = native.PA_ERR_INVALID_ARGUMENT
    for call in (decode, prefill):
        assert call(key=None) == bad and call(value=None) == bad and call(query=None) == bad
        assert call(layer=1) == bad
        wrong = native.PaStepDims()
        ctypes.pointer(wrong)[0] = dims
        wrong.dtype = native.PA_DTYPE_E4M3
        assert call(d=wrong) == bad

    def layer(call, scales=FAKE, rows=None):
        return lib.pa_attention_step_8bit(call, FAKE, FAKE, FAKE, scales, scales, 0, rows, 1.0, FAKE, None)

    one = native.PaStepCall(dims=dims, num_decode_items=1)
    assert layer(None) == bad and layer(ctypes.byref(one), scales=None) == bad
    assert layer(ctypes.byref(one), rows=ctypes.byref(native.PaNewRows())) == bad
    assert layer(ctypes.byref(native.PaStepCall(dims=dims))) == native.PA_OK  # no work items
