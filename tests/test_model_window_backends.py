"""Backends of a user's own under models whose layers have a window: one that knows no
windows serves the contexts that no window limits, and is refused the others."""

import inspect

import pytest

pytest.importorskip("transformers")

import torch

from helpers import pkg
from test_model_span import Served, causal, dense_logits, tiny_model, tokens

paged_attention = pkg("model.paged_attention")
backends = pkg("model.attention_backends")


class WithoutWindows(backends.AttentionBackend):
    name = "without windows"

    def supports(self, context, num_query_tokens):
        return True

    def attend(self, query, store, layer_idx, context, scaling, dropout):
        return backends.dense_sdpa(query, store, layer_idx, context, scaling, dropout)


@pytest.fixture
def served(monkeypatch):
    model = tiny_model("qwen2", "cpu", window=24)
    served = Served(model, "cpu")
    monkeypatch.setattr(paged_attention, "_BACKEND", WithoutWindows())
    return served


def test_contexts_inside_the_window(served):
    ids = tokens(24, 1)
    seq = served.add(ids[:20])
    want = dense_logits(served.model, ids, causal(24, 24), list(range(24)), "cpu")
    _, first = served.step([(seq, 0, ids[:20])])
    rows = [first[0]]
    for i in range(20, 24):
        rows.append(served.step([(seq, i, ids[i:i + 1])])[1][0])
    assert float((torch.cat(rows) - want).abs().max()) <= 1e-3
    with pytest.raises(TypeError, match="window"):  # (its first context past the window)
        served.step([(seq, 24, tokens(1, 2))])


def test_the_interface_names_the_window():
    for backend in (backends.AttentionBackend, backends.TorchSdpBackend, backends.NativePagedBackend):
        assert inspect.signature(backend.attend).parameters["window"].default is None
