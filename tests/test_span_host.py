"""Host code of windows and trees: the longest shorter context of a window, the
plans of trees against lists counted here, struct layouts and the arguments that
the entry points refuse before any launch.  No GPU needed."""

import ctypes
import subprocess

import numpy as np
import pytest

from helpers import pkg
from test_abi import HEADER

native = pkg("_native")
STAGE = 64


@pytest.fixture(scope="module")
def lib():
    return native.load_library()


def test_struct_layouts(tmp_path):
    structs = {name: getattr(native, name) for name in ("PaWindow", "PaTreeDims", "PaTreePlan", "PaTreeCall")}
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "paged_attention_amd.h"', "int main(void) {"]
    for name, st in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        for field, _ in st._fields_:
            lines.append(f'printf("{name}.{field} %zu\\n", offsetof({name}, {field}));')
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", f"-I{HEADER.parent}", str(tmp_path / "layout.c"), "-o",
                    str(tmp_path / "layout")], check=True)
    got = dict(line.split() for line in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True,
                                                       check=True).stdout.splitlines())
    for name, st in structs.items():
        assert int(got[name]) == ctypes.sizeof(st), name
        for field, _ in st._fields_:
            assert int(got[f"{name}.{field}"]) == getattr(st, field).offset, f"{name}.{field}"


def shorter(ctx, window, sinks, bs):
    """Tokens of the blocks that hold a visible position of the last query, the last
    block cut at the context's end: what a decode under the window walks."""
    seen = [q for q in range(ctx) if ctx - 1 - q < window or q < sinks]
    blocks = {q // bs for q in seen}
    return sum(min(bs, ctx - b * bs) for b in blocks)


@pytest.mark.parametrize("block_size", [1, 4, 16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 0), (16, 4), (33, 17), (7, 200)])
def test_window_context_is_the_longest_of_all_shorter_ones(lib, block_size, window, sinks):
    longest = 0
    for ctx in range(0, 150):
        longest = max(longest, shorter(ctx, window, sinks, block_size))
        got = lib.pa_window_context(ctx, native.PaWindow(window, sinks), block_size)
        assert longest <= got <= max(ctx, 0)
        # (the sinks' whole blocks, and the window begun anywhere in one)
        assert got <= -(-sinks // block_size) * block_size + window + block_size - 1


def test_window_context_without_a_window(lib):
    big = 2 ** 31 - 1
    assert lib.pa_window_context(777, native.PaWindow(0, 9), 16) == 777
    assert lib.pa_window_context(big, native.PaWindow(big, big), 16) == big
    assert lib.pa_window_context(0, native.PaWindow(4, 4), 16) == 0


def plan_of(lib, starts, counts, *, heads=(32, 8), head_dim=128, dtype=native.PA_DTYPE_BF16, block_size=16,
            window=0, sinks=0, split=0, batch=None):
    s, n = np.array(starts, np.int64), np.array(counts, np.int64)
    dims = native.PaTreeDims(len(s) if batch is None else batch, int(n.sum()), heads[0], heads[1], head_dim, dtype,
                             block_size, 256, split, native.PaWindow(window, sinks))
    plan = native.PaTreePlan()
    rc = lib.pa_plan_tree(s.ctypes.data, n.ctypes.data, dims, ctypes.byref(plan))
    return rc, plan


def counted(starts, counts, tile, split, window, sinks):
    """Items, joined tiles and partial rows, by the stages that hold a position some
    node of the tile may see (or, for lack of sinks, lie in its first stage)."""
    items = merges = rows = 0
    for s, n in zip(starts, counts):
        for t0 in range(0, n, tile):
            m = min(tile, n - t0)
            lo = max(s - window + 1, 0) if window else 0
            seen = {q // STAGE for q in range(s + t0 + m) if q >= lo or q < sinks}
            runs = -(-len(seen) // split)
            items += runs
            if runs > 1:
                merges, rows = merges + 1, rows + runs * m
    return items, merges, rows


@pytest.mark.parametrize("heads,head_dim,dtype", [((32, 8), 128, "BF16"), ((32, 32), 64, "F16"), ((8, 4), 256, "BF16"),
                                                  ((16, 4), 128, "E4M3"), ((8, 8), 64, "F32")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 0), (300, 70)])
@pytest.mark.parametrize("split", [0, 1, 3, 100])
def test_plan_counts(lib, heads, head_dim, dtype, window, sinks, split):
    starts, counts = [0, 63, 64, 1000, 5, 2500], [1, 2, 64, 65, 0, 100]
    rc, plan = plan_of(lib, starts, counts, heads=heads, head_dim=head_dim, dtype=getattr(native, f"PA_DTYPE_{dtype}"),
                       window=window, sinks=sinks, split=split)
    assert rc == native.PA_OK and plan.bad_seq == -1
    assert plan.mask_words == 4 and plan.tile > 0
    assert plan.split_stages == split if split else 1 <= plan.split_stages <= 64
    want = counted(starts, counts, plan.tile, plan.split_stages, window, sinks)
    assert (plan.num_items, plan.num_merge_items, plan.num_partial_rows) == want


def test_plan_without_lists(lib):
    for kw in ({"heads": (0, 0)}, {"heads": (8, 8), "head_dim": 96, "dtype": native.PA_DTYPE_F32},
               {"heads": (8, 8), "head_dim": 40}, {"block_size": 24}):
        rc, plan = plan_of(lib, [10], [33], **kw)
        assert rc == native.PA_OK and plan.mask_words == 2
        assert (plan.tile, plan.num_items, plan.num_merge_items, plan.num_partial_rows) == (0, 0, 0, 0)
    rc, plan = plan_of(lib, [], [])
    assert rc == native.PA_OK and plan.num_items == 0 and plan.mask_words == 1
    rc, plan = plan_of(lib, [7, 0], [0, 0])
    assert rc == native.PA_OK and plan.num_items == 0


def test_plan_of_the_longest_contexts(lib):
    """Splits stay within what a workgroup keeps of the block table."""
    big = 2 ** 31 - 1 - 1024
    rc, plan = plan_of(lib, [big], [1024], block_size=16, split=2 ** 30)
    assert rc == native.PA_OK and plan.split_stages * STAGE // 16 <= 3584
    stages = -(-(big + 1024) // STAGE)
    assert plan.num_items >= stages // plan.split_stages
    rc, plan = plan_of(lib, [big + 1], [1024])
    assert rc == native.PA_ERR_INVALID_ARGUMENT and plan.bad_seq == 0


@pytest.mark.parametrize("starts,counts,kw,bad", [
    ([0, -1], [1, 1], {}, 1), ([0], [1025], {}, 0), ([4, 4, 4], [1, 9, 1], {"window": 8}, 1), ([0], [-1], {}, 0),
    ([0], [1], {"block_size": 0}, -1), ([0], [1], {"window": -1}, -1), ([0], [1], {"sinks": -1}, -1),
    ([0], [1], {"split": -1}, -1), ([0], [1], {"heads": (6, 4)}, -1), ([0], [1], {"heads": (6, 0)}, -1),
    ([0], [1], {"batch": -1}, -1)])
def test_plan_refusals(lib, starts, counts, kw, bad):
    rc, plan = plan_of(lib, starts, counts, **kw)
    assert rc == native.PA_ERR_INVALID_ARGUMENT
    if kw.get("batch") is None:
        assert plan.bad_seq == bad
    assert lib.pa_last_error_message()


def step_dims(**kw):
    d = dict(num_seqs=1, num_query_tokens=1, num_query_heads=8, num_kv_heads=4, head_dim=64, block_size=16,
             total_blocks=8, num_layers=1, max_blocks_per_seq=1, partition_size=512, dtype=native.PA_DTYPE_BF16,
             q_token_stride=512, q_head_stride=64)
    d.update(kw)
    return native.PaStepDims(**d)


def refused(lib, rc, text, code=None):
    assert rc == (native.PA_ERR_INVALID_ARGUMENT if code is None else code)
    assert text in lib.pa_last_error_message(), lib.pa_last_error_message()


def test_entry_points_refuse_before_any_launch(lib):
    P = 0x1000
    window = native.PaWindow(4, 0)

    def windowed(dims, w=window, layer=0, call=None, scales=None, rows=None):
        call = call or native.PaStepCall(dims=dims, decode_items=P, num_decode_items=1, block_tables=P, context_lens=P,
                                         cu_seqlens=P)
        return lib.pa_attention_window(ctypes.byref(call), w, P, P, P, scales, scales, layer, rows, 1.0, P, None)

    refused(lib, lib.pa_attention_window(None, window, P, P, P, None, None, 0, None, 1.0, P, None), b"")
    refused(lib, windowed(step_dims(), native.PaWindow(0, 0)), b"window")
    refused(lib, windowed(step_dims(), native.PaWindow(4, -1)), b"sinks")
    refused(lib, windowed(step_dims(num_query_heads=6)), b"multiple of num_kv_heads")
    refused(lib, windowed(step_dims(), layer=1), b"Layer index 1 out of range")

    def tree(dims=None, layer=0, scales=None, **kw):
        call = native.PaTreeCall(dims=dims or step_dims(), block_tables=P, context_lens=P, cu_seqlens=P,
                                 scatter_slots=P, masks=P, positions=P)
        call.plan.mask_words = 1
        for name, value in kw.items():
            setattr(call, name, value)
        return lib.pa_tree_attention(ctypes.byref(call), P, P, P, scales, scales, layer, None, 1.0, P, None)

    refused(lib, lib.pa_tree_attention(None, P, P, P, None, None, 0, None, 1.0, P, None), b"")
    refused(lib, tree(masks=None), b"masks")
    refused(lib, tree(layer=3), b"Layer index 3 out of range")
    refused(lib, tree(window=native.PaWindow(-1, 0)), b"window")
    refused(lib, tree(dims=step_dims(num_query_heads=6)), b"multiple of num_kv_heads")

    dims = native.PaTreeDims(1, 1, 0, 0, 64, native.PA_DTYPE_BF16, 16, 256, 0, native.PaWindow(0, 0))
    plan = native.PaTreePlan(mask_words=1)
    refused(lib, lib.pa_pack_tree(None, P, P, None, dims, plan, P, P, None, None, None), b"")
    refused(lib, lib.pa_accept_tree(P, P, P, P, -1, 1, P, P, P, None), b"")
    refused(lib, lib.pa_accept_tree(P, None, P, P, 1, 1, P, P, P, None), b"")
    refused(lib, lib.pa_keep_rows(None, P, None, None, step_dims(), P, P, P, P, P, None), b"")
    refused(lib, lib.pa_keep_rows(P, P, None, None, step_dims(head_dim=0), P, P, P, P, P, None), b"")


def test_nothing_to_do_is_no_launch(lib):
    P = 0x1000
    empty = step_dims(num_seqs=0, num_query_tokens=0)
    assert lib.pa_accept_tree(None, None, None, None, 0, 0, None, None, None, None) == native.PA_OK
    assert lib.pa_keep_rows(P, P, None, None, empty, None, None, None, None, None, None) == native.PA_OK
