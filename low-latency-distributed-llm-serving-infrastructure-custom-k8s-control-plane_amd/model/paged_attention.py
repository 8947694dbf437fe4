"""Paged attention on top of the paged KV cache: the per-step and per-layer glue.

The operator API is the reference's (app/model/paged_attention.py):
``PagedStepContext`` with the same constructor and attributes, the per-layer
hook ``paged_attention_forward`` registered in transformers'
ALL_ATTENTION_FUNCTIONS, ``register_paged_attention`` and
``run_paged_forward``.  The step runs flat: all sequences of a step are one
``[1, T]`` batch.

On a GPU store the context is packed once per step (``self.packed``: each
sequence's row of the device-resident block-table pool, cu_seqlens, slots,
positions and the attention work lists, from the step's host arrays handed
over in pinned memory and the packing kernels), and every layer then writes
its new K/V rows and runs the HIP attention kernels on the device without
host syncs (for a decode step the rows are written inside the decode
launches).  A GPU store always
takes the HIP path: with no backend installed the hook installs it, and the
reference's dense SDPA path is refused there (it would gather the whole
context and build a T x C mask on the device).
"""

from __future__ import annotations

from typing import List, Optional

import numpy as np
import torch

from .. import paged_ops

PAGED_ATTENTION_NAME = "paged"

# The backend every layer dispatches to (paged_attention.py:22-25).  None on a
# CPU store means the inline SDPA path; a GPU store installs the HIP backend.
_BACKEND = None
_FALLBACK_BACKEND = None


def _get_fallback_backend():
    global _FALLBACK_BACKEND
    if _FALLBACK_BACKEND is None:
        from .attention_backends import TorchSdpBackend

        _FALLBACK_BACKEND = TorchSdpBackend()
    return _FALLBACK_BACKEND


def set_backend(backend) -> None:
    """Install the backend every layer dispatches to (None = the default)."""
    global _BACKEND
    _BACKEND = backend


def _offsets(counts: np.ndarray) -> torch.Tensor:
    """int64 [n + 1]: 0 followed by the running totals of ``counts``."""
    out = np.zeros(counts.shape[0] + 1, dtype=np.int64)
    np.cumsum(counts, out=out[1:])
    return torch.from_numpy(out)


def _depths(parents: List[int]) -> np.ndarray:
    """int64 [n] depth of each node; a parent that is no earlier node is none."""
    depth = np.zeros(len(parents), dtype=np.int64)
    for i, p in enumerate(parents):
        if 0 <= p < i:
            depth[i] = depth[p] + 1
    return depth


def _ancestors(parents: List[int]) -> np.ndarray:
    """bool [n, n]: node j is node i or one of its ancestors."""
    over = np.eye(len(parents), dtype=bool)
    for i, p in enumerate(parents):
        if 0 <= p < i:
            over[i] |= over[p]
    return over


class PagedStepContext:
    """Slot bookkeeping and attention layout of one engine step
    (paged_attention.py:37-118).

    Attributes (the reference's): store, sequences, start_positions,
    new_token_counts, context_lens (lists), cu_seqlens, cu_context_offsets
    (CPU int64 tensors), scatter_slots, gather_slots (int64 on the store's
    device), num_query_tokens, num_context_tokens.  ``packed`` is the GPU
    description of the step (None on a CPU store).  The host-side lists and
    offsets are built on first use: a GPU step needs none of them.

    ``window`` / ``sinks``: every layer's queries see at most the last ``window``
    positions and the first ``sinks`` ones (a layer that passes a
    ``sliding_window`` of its own sees the smaller of the two, and those sinks).
    ``parents``: one list per sequence, for a step whose new tokens are trees of
    drafted ones (the index of each node's parent in its sequence's list, -1 for
    a root); a node's position is then its depth's, and it sees its sequence's
    context, its ancestors and itself.
    """

    def __init__(self, store, sequences: List, start_positions: List[int], new_token_counts: List[int],
                 prefill_tile: Optional[int] = None, *, window: Optional[int] = None, sinks: int = 0,
                 parents: Optional[List[List[int]]] = None) -> None:
        if not (len(sequences) == len(start_positions) == len(new_token_counts)):
            raise ValueError(
                f"sequences ({len(sequences)}), start_positions ({len(start_positions)}) "
                f"and new_token_counts ({len(new_token_counts)}) must have the same length"
            )
        self.store = store
        self.sequences = sequences if isinstance(sequences, list) else list(sequences)
        self.packed: Optional[paged_ops.PackedStep] = None
        self._gather_slots: Optional[torch.Tensor] = None
        self._masks: dict = {}
        if window is not None and window < 1:
            raise ValueError(f"window must be a positive number of tokens, got {window}")
        if sinks < 0:
            raise ValueError(f"sinks must be a number of tokens, got {sinks}")
        if parents is not None and [len(p) for p in parents] != [int(c) for c in new_token_counts]:
            raise ValueError("parents must have one list per sequence with one entry per new token")
        self.window = window
        self.sinks = int(sinks)
        self.parents = parents
        self._trees: dict = {}
        self._parents_on: Optional[torch.Tensor] = None  # the parents on the store's device
        self._rows, self._starts, self._counts = store.step_rows(self.sequences, start_positions, new_token_counts)
        if store.on_gpu:
            if self.sequences:
                self.packed = store.pack_rows(self._rows, self._starts, self._counts)
                self.scatter_slots = self.packed.scatter_slots
            else:
                self.scatter_slots = torch.empty((0,), dtype=torch.long, device=store.device)
        else:
            self.scatter_slots = torch.from_numpy(store._host_slots(self._rows, self._starts, self._counts))
            self._gather_slots = torch.from_numpy(
                store._host_slots(self._rows, np.zeros_like(self._starts), self._starts + self._counts))

    # -- host-side views of the step (built on first use) ------------------------------
    def _cached(self, name, build):
        value = self.__dict__.get(name)
        if value is None:
            value = self.__dict__[name] = build()
        return value

    @property
    def start_positions(self) -> List[int]:
        return self._cached("_start_list", self._starts.tolist)

    @property
    def new_token_counts(self) -> List[int]:
        return self._cached("_count_list", self._counts.tolist)

    @property
    def context_lens(self) -> List[int]:
        return self._cached("_ctx_list", lambda: (self._starts + self._counts).tolist())

    @property
    def cu_seqlens(self) -> torch.Tensor:
        return self._cached("_cu_q", lambda: _offsets(self._counts))

    @property
    def cu_context_offsets(self) -> torch.Tensor:
        return self._cached("_cu_c", lambda: _offsets(self._starts + self._counts))

    def packed_for(self, num_query_heads: int) -> paged_ops.PackedStep:
        """The packed step with prefill work items and decode workspace sized
        for ``num_query_heads`` (re-packs once if the store did not know the
        model's head count)."""
        if self.packed is None:
            raise RuntimeError("this step is not on a GPU store")
        tile = paged_ops.prefill_tile_for(num_query_heads, self.store.num_heads)
        if self.packed.prefill_tile != tile:
            first = self.packed
            self.packed = self.store.pack_rows(self._rows, self._starts, self._counts,
                                               num_query_heads=num_query_heads, partition_size=first.partition_size)
            # (the first one's choice, which is none of a caller's: windows choose their own)
            self.packed._partition_given = first._partition_given
        return self.packed

    def window_of(self, sliding_window: Optional[int]) -> Optional[int]:
        """The window of a layer that passes ``sliding_window`` (None: none)."""
        if sliding_window is None or self.window is None:
            return self.window if sliding_window is None else int(sliding_window)
        return min(int(sliding_window), self.window)

    def within(self, window: int) -> bool:
        """Whether no context of the step reaches past ``window``, so that it limits nothing
        (never in a launch that a graph captures, which may serve longer contexts)."""
        if self.packed is None:
            return max(self.context_lens, default=0) <= window
        return self.packed.max_context <= window and not torch.cuda.is_current_stream_capturing()

    def tree_for(self, num_query_heads: int, window: Optional[int] = None) -> paged_ops.TreeStep:
        """The step's packed trees for layers of ``num_query_heads`` under ``window``."""
        step = self.packed_for(num_query_heads)
        tree = self._trees.get((num_query_heads, window))
        if tree is None or tree.step is not step:
            if self._parents_on is None:
                flat = torch.tensor([p for parents in self.parents for p in parents], dtype=torch.int32)
                self._parents_on = flat.pin_memory().to(step.buffer.device, non_blocking=True)
            tree = paged_ops.pack_tree(step, self._parents_on, num_kv_heads=self.store.num_heads,
                                       num_query_heads=num_query_heads, head_dim=self.store.head_dim,
                                       dtype=self.store.dtype, window=window,
                                       sinks=self.sinks if window is not None else 0)
            self._trees[(num_query_heads, window)] = tree
        return tree

    @property
    def gather_slots(self) -> torch.Tensor:
        """int64 [C]: slots of every context token, sequence by sequence."""
        if self._gather_slots is None:
            if self.packed is not None:
                self._gather_slots = self.packed.gather_slots
            else:
                self._gather_slots = torch.empty((0,), dtype=torch.long, device=self.store.device)
        return self._gather_slots

    @property
    def num_query_tokens(self) -> int:
        return int(self._counts.sum()) if self.packed is None else self.packed.num_query_tokens

    @property
    def num_context_tokens(self) -> int:
        return int((self._starts + self._counts).sum())

    def position_ids(self, device: torch.device) -> torch.Tensor:
        """[1, T] positions, restarting at every sequence boundary."""
        if self.packed is not None and torch.device(device) == self.packed.buffer.device:
            if self.parents is not None:
                return self.tree_for(int(self.store.num_query_heads or self.store.num_heads)).position_ids.unsqueeze(0)
            return self.packed.position_ids.unsqueeze(0)
        counts = np.asarray(self.new_token_counts, dtype=np.int64)
        total = int(counts.sum()) if counts.size else 0
        owner = np.repeat(np.arange(counts.size), counts)
        first = self.cu_seqlens.numpy()[:-1]
        inside = np.arange(total, dtype=np.int64) - first[owner]
        if self.parents is not None and total:
            inside = np.concatenate([_depths(p) for p in self.parents])
        pos = inside + np.asarray(self.start_positions, np.int64)[owner]
        return torch.from_numpy(pos).to(device).unsqueeze(0)

    def attention_mask(self, device: torch.device, window: Optional[int] = None) -> torch.Tensor:
        """Block-diagonal causal mask, bool (1, 1, T, C), True = attended:
        query token i of sequence s (position start_s + i) sees context
        position j of the same sequence when j <= start_s + i.

        Under a window it sees those with position - j < window or j < sinks, and
        the nodes of a tree see, of the new tokens, their ancestors and themselves.

        Only the SDPA path materialises it; the HIP kernels evaluate the same
        rule from cu_seqlens and context_lens."""
        device = torch.device(device)
        mask = self._masks.get((device, window))
        if mask is not None:
            return mask
        q_seq = torch.repeat_interleave(torch.arange(len(self.new_token_counts)),
                                        torch.tensor(self.new_token_counts, dtype=torch.long))
        c_seq = torch.repeat_interleave(torch.arange(len(self.context_lens)),
                                        torch.tensor(self.context_lens, dtype=torch.long))
        q_pos = self.position_ids(torch.device("cpu"))[0]
        c_pos = torch.arange(self.num_context_tokens) - self.cu_context_offsets[c_seq]
        own = q_seq[:, None] == c_seq[None, :]
        mask = own & (c_pos[None, :] <= q_pos[:, None])
        if window is not None:
            mask &= (q_pos[:, None] - c_pos[None, :] < window) | (c_pos[None, :] < self.sinks)
        if self.parents is not None:
            first, end = self.cu_seqlens.tolist(), self.cu_context_offsets.tolist()
            for i, parents in enumerate(self.parents):
                mask[first[i]:first[i + 1], end[i + 1] - len(parents):end[i + 1]] = torch.from_numpy(_ancestors(parents))
        mask = self._masks[(device, window)] = mask[None, None].to(device)
        return mask


def _default_backend(store):
    """The backend a layer uses when none is installed: the HIP backend for a
    GPU store (installed for every later layer; raises when the library is
    missing), none (inline SDPA) for a CPU store."""
    global _BACKEND
    if not store.on_gpu:
        return None
    from .attention_backends import select_backend

    _BACKEND = select_backend("native")
    return _BACKEND


def paged_attention_forward(
    module: torch.nn.Module,
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    attention_mask: Optional[torch.Tensor] = None,
    dropout: float = 0.0,
    scaling: Optional[float] = None,
    **kwargs,
) -> tuple[torch.Tensor, None]:
    """Per-layer hook (paged_attention.py:138-180): write the layer's new K/V
    into the paged blocks, then attend through the installed backend.  A CPU
    store falls back to SDPA for shapes the backend refuses, or runs the
    inline SDPA path with none installed; a GPU store runs the HIP kernels.

    ``sliding_window``, which transformers hands over for layers that have one,
    limits the layer to that window (the context's ``window`` limits every layer,
    and its ``sinks`` stay visible in both).  A window that some context reaches past
    goes to the backend's ``attend`` as ``window``."""
    context: PagedStepContext = module.paged_context
    store = context.store
    layer_idx = module.layer_idx
    # [1, H_kv, T, D] projections -> [T, H_kv, D] views (no copy)
    new_key, new_value = key[0].transpose(0, 1), value[0].transpose(0, 1)
    scale = module.scaling if scaling is None else scaling
    window = context.window_of(kwargs.get("sliding_window"))
    limits = {} if window is None or context.within(window) else {"window": window}
    backend = _BACKEND if _BACKEND is not None else _default_backend(store)
    if store.on_gpu:
        from .attention_backends import NativePagedBackend

        if not isinstance(backend, NativePagedBackend):
            raise RuntimeError(
                f"a GPU store runs the HIP paged-attention backend, not {type(backend).__name__} "
                "(dense SDPA would gather every context and build a T x C mask on the device)")
        if query.shape[2] == 0:
            return query.new_empty((1, 0, query.shape[1], query.shape[3])), None
        # The backend writes the new rows (inside the decode launches for a
        # step of single-token sequences) before it attends.
        new_key, new_value = store.checked_layer_kv(layer_idx, new_key, new_value, context.num_query_tokens)
        return backend.attend(query, store, layer_idx, context, scale, dropout, new_key=new_key,
                              new_value=new_value, **limits), None
    store.scatter_layer_kv(layer_idx, new_key, new_value, context.scatter_slots)
    if backend is not None:
        if not backend.supports(context, query.shape[2]):
            backend = _get_fallback_backend()
        return backend.attend(query, store, layer_idx, context, scale, dropout, **limits), None
    from .attention_backends import dense_sdpa

    return dense_sdpa(query, store, layer_idx, context, scale, dropout, **limits), None


def _decoder(model) -> torch.nn.Module:
    """The module holding the decoder layers: the model's own decoder when it
    exposes one, else the first of its usual attributes that has ``layers``."""
    getter = getattr(model, "get_decoder", None)
    if callable(getter):
        try:
            decoder = getter()
        except (AttributeError, NotImplementedError):
            decoder = None
        if decoder is not None and hasattr(decoder, "layers"):
            return decoder
    for name in ("model", "transformer", "base_model"):
        inner = getattr(model, name, None)
        if inner is not None and hasattr(inner, "layers"):
            return inner
    return model


def register_paged_attention(model, backend=None) -> None:
    """Route every decoder layer of ``model`` through the paged hook
    (paged_attention.py:183-188) and install ``backend`` (by default the one
    select_backend names: the HIP backend when the library and a ROCm device
    are there)."""
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS

    from .attention_backends import select_backend

    ALL_ATTENTION_FUNCTIONS.register(PAGED_ATTENTION_NAME, paged_attention_forward)
    for layer in _decoder(model).layers:
        layer.self_attn.paged_context = None
    model.config._attn_implementation = PAGED_ATTENTION_NAME
    set_backend(backend if backend is not None else select_backend())


def run_paged_forward(model, context: PagedStepContext, input_ids: torch.Tensor, logits_to_keep=None
                      ) -> torch.Tensor:
    """One flat forward pass whose K/V lands in the paged blocks
    (paged_attention.py:191-207).  ``logits_to_keep`` (a device index tensor
    or a count) restricts the LM head to those rows, e.g. each sequence's
    last token."""
    for layer in _decoder(model).layers:
        layer.self_attn.paged_context = context
    extra = {} if logits_to_keep is None else {"logits_to_keep": logits_to_keep}
    out = model(input_ids, position_ids=context.position_ids(input_ids.device), use_cache=False, **extra)
    return out.logits
