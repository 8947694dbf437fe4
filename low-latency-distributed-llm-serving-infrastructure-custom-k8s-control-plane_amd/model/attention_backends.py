"""Attention backends behind the per-layer hook.

Same API as the reference's app/model/attention_backends.py:
``AttentionBackend.supports / attend``, ``TorchSdpBackend``, the ``native``
backend, the ``_BACKENDS`` registry and ``select_backend`` driven by
``LLM_PAGED_BACKEND`` in {auto, torch, native, hip (= native)}.

``NativePagedBackend`` here is the MI355X path: decode, prefill and mixed
steps all run in the HIP kernels over the block tables, on the device, with
no dense mask and no host copies.  Unlike the reference's native backend
(decode-only, attention_backends.py:85-86) it therefore supports every step
shape of a GPU store; a CPU store is refused (supports -> False) so the hook
falls back to SDPA as the reference does for shapes its backend refuses.
"""

from __future__ import annotations

import os
from abc import ABC, abstractmethod
from typing import TYPE_CHECKING, Optional

import torch
import torch.nn.functional as F

from .. import _native, metrics, paged_ops

if TYPE_CHECKING:
    from ..memory.manager import PagedKVCacheManager
    from .paged_attention import PagedStepContext

BACKEND_ENV_VAR = "LLM_PAGED_BACKEND"
TORCH_BACKEND = "torch"
NATIVE_BACKEND = "native"


def native_kernel_available() -> bool:
    """The HIP library loads and a ROCm device is visible
    (attention_backends.py:19-24)."""
    if not torch.cuda.is_available():
        return False
    try:
        _native.load_library()
    except (RuntimeError, OSError):
        return False
    return True


class AttentionBackend(ABC):
    name: str = ""

    @abstractmethod
    def supports(self, context: "PagedStepContext", num_query_tokens: int) -> bool:
        ...

    @abstractmethod
    def attend(self, query: torch.Tensor, store: "PagedKVCacheManager", layer_idx: int,
               context: "PagedStepContext", scaling: float, dropout: float,
               window: Optional[int] = None) -> torch.Tensor:
        """``window``: given (by name) for a layer that sees less than its contexts, whose
        query at position p sees the positions q <= p with p - q < window or q <
        ``context.sinks``.  A backend without it serves the other layers alone: such a
        call is a TypeError."""


def dense_sdpa(query, store, layer_idx, context, scaling, dropout, window=None) -> torch.Tensor:
    """Gather the step's whole context of one layer into dense [1, H_kv, C, D]
    K/V and run torch SDPA under the context's mask (block-diagonal and causal, or
    of its window or trees); returns
    [1, T, H_q, D] (the computation of attention_backends.py:55-78 and of the
    inline path paged_attention.py:165-180)."""
    slots = context.gather_slots
    k = store.gather_layer_keys(layer_idx, slots).transpose(0, 1).unsqueeze(0)
    v = store.gather_layer_values(layer_idx, slots).transpose(0, 1).unsqueeze(0)
    out = F.scaled_dot_product_attention(
        query, k, v,
        attn_mask=context.attention_mask(query.device) if window is None else context.attention_mask(query.device,
                                                                                                    window),
        dropout_p=dropout,
        scale=scaling,
        enable_gqa=query.shape[1] != k.shape[1],
    )
    return out.transpose(1, 2).contiguous()


class TorchSdpBackend(AttentionBackend):
    """The reference's own fallback backend: dense gather + SDPA
    (attention_backends.py:48-78).  Not the MI355X path."""

    name = TORCH_BACKEND

    def supports(self, context: "PagedStepContext", num_query_tokens: int) -> bool:
        return True

    def attend(self, query, store, layer_idx, context, scaling, dropout, window=None):
        return dense_sdpa(query, store, layer_idx, context, scaling, dropout, window)


class NativePagedBackend(AttentionBackend):
    """HIP paged attention on the GPU (decode split-K + MFMA prefill)."""

    name = NATIVE_BACKEND

    def supports(self, context: "PagedStepContext", num_query_tokens: int) -> bool:
        return (
            num_query_tokens > 0
            and getattr(context, "packed", None) is not None
            and context.store.on_gpu
        )

    def attend(self, query, store, layer_idx, context, scaling, dropout, new_key=None, new_value=None, window=None):
        """``new_key`` / ``new_value`` ([T, H_kv, D] on the store's device, its
        dtype): the layer's new rows, written into the cache first
        (:func:`paged_ops.attention`); without them the caller has written
        them.  ``window``: of this layer, with the context's sinks."""
        if context.packed is None:
            if not native_kernel_available():
                raise RuntimeError(
                    "libpaged_attention_amd.so is not loaded or no ROCm device is visible; "
                    "build the HIP extension to enable the native backend"
                )
            raise RuntimeError("the native backend needs a step packed on the GPU store")
        step = context.packed_for(int(query.shape[1]))
        scales = {}
        if getattr(store, "key_scales", None) is not None:
            scales = {"key_scales": store.key_scales, "value_scales": store.value_scales}
        recorder = metrics.current()
        if recorder is None:
            return self._launch(query, store, layer_idx, context, step, scaling, new_key, new_value, window,
                                scales).unsqueeze(0)
        stream = torch.cuda.current_stream(query.device)
        start = recorder.begin(stream)
        out = self._launch(query, store, layer_idx, context, step, scaling, new_key, new_value, window, scales)
        known = context.__dict__.setdefault("_attention_bytes", {})
        nbytes = known.get(window)
        if nbytes is None:
            lens = context.context_lens
            if window is not None:  # what the window of the first new token and the sinks leave
                lens = [min(c, window + n - 1 + context.sinks) for c, n in zip(lens, context.new_token_counts)]
            nbytes = known[window] = metrics.step_bytes(
                lens, context.num_query_tokens, int(query.shape[1]), store.num_heads, store.head_dim,
                store.key_cache.element_size(), store.block_size, query.element_size() if scales else 0)
        recorder.end(start, nbytes, context.num_query_tokens, stream)
        return out.unsqueeze(0)

    @staticmethod
    def _launch(query, store, layer_idx, context, step, scaling, new_key, new_value, window, scales):
        # (a window that no context of the step reaches past is none, but in a
        # captured launch, which may serve longer contexts)
        if window is not None and step.max_context <= window and not torch.cuda.is_current_stream_capturing():
            window = None
        if getattr(context, "parents", None) is not None:
            tree = context.tree_for(int(query.shape[1]), window)
            return paged_ops.tree_attention(query, store.key_cache, store.value_cache, layer_idx, step, tree, scaling,
                                            new_key=new_key, new_value=new_value, **scales)
        limits = {} if window is None else {"window": window, "sinks": context.sinks}
        return paged_ops.attention(query, store.key_cache, store.value_cache, layer_idx, step, scaling,
                                   new_key=new_key, new_value=new_value, **scales, **limits)


_BACKENDS = {
    TORCH_BACKEND: TorchSdpBackend,
    NATIVE_BACKEND: NativePagedBackend,
}


_ALIASES = {"hip": NATIVE_BACKEND}


def select_backend(requested: Optional[str] = None) -> AttentionBackend:
    """Backend named by ``requested`` or $LLM_PAGED_BACKEND (default auto),
    as attention_backends.py:126-144: auto = native when the HIP library and a
    ROCm device are there, else torch; an unknown name is a ValueError and an
    explicit native request without the library a RuntimeError."""
    name = (requested or os.getenv(BACKEND_ENV_VAR) or "auto").strip().lower()
    name = _ALIASES.get(name, name)
    if name == "auto":
        name = NATIVE_BACKEND if native_kernel_available() else TORCH_BACKEND
    elif name not in _BACKENDS:
        raise ValueError(
            f"{BACKEND_ENV_VAR}={name!r} names no paged-attention backend "
            f"(choose auto, {TORCH_BACKEND} or {NATIVE_BACKEND}/hip)")
    elif name == NATIVE_BACKEND and not native_kernel_available():
        raise RuntimeError(
            f"{BACKEND_ENV_VAR}={NATIVE_BACKEND} needs libpaged_attention_amd.so and a ROCm device")
    return _BACKENDS[name]()
