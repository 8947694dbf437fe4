"""Host side of windows and trees between calls: what the entry points refuse, and in what
order.  No GPU needed: a call that reached a launch would report the missing device."""

import ctypes

import pytest

from helpers import pkg
from test_span_host import refused, step_dims

native = pkg("_native")


@pytest.fixture(scope="module")
def lib():
    return native.load_library()


@pytest.mark.parametrize("scales", [None, 0x1000])
def test_a_windowed_call_is_checked_whole_before_its_rows_are_written(lib, scales):
    P = 0x1000
    rows = native.PaNewRows(P, P, 512, 64, 512, 64)

    def call(dims=None, **kw):
        c = native.PaStepCall(dims=dims or step_dims(max_blocks_per_seq=64), block_tables=P, context_lens=P, cu_seqlens=P,
                              scatter_slots=P, prefill_tile=64, workspace=P, workspace_bytes=1 << 30)
        for name, value in {"decode_items": P, "num_decode_items": 3, "prefill_items": P, "num_prefill_items": 2,
                            **kw}.items():
            setattr(c, name, value)
        return lib.pa_attention_window(ctypes.byref(c), native.PaWindow(4, 0), P, P, P, scales, scales, 0,
                                       ctypes.byref(rows), 1.0, P, None)

    refused(lib, call(prefill_items=None), b"prefill_items")
    refused(lib, call(decode_items=None), b"decode_items")
    refused(lib, call(workspace_bytes=8), b"workspace of", native.PA_ERR_WORKSPACE)
    refused(lib, call(num_merge_items=1), b"merge_items")
    refused(lib, call(dims=step_dims(head_dim=300)), b"not supported", native.PA_ERR_UNSUPPORTED)
    # A step of single tokens whose launch would write the rows itself, if it could.
    single = {"num_prefill_items": 0}
    refused(lib, call(workspace_bytes=8, **single), b"workspace of", native.PA_ERR_WORKSPACE)
    refused(lib, call(dims=step_dims(head_dim=300), **single), b"not supported", native.PA_ERR_UNSUPPORTED)
