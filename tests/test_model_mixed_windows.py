"""Models of which some layers have a window and some none, through the paged hook: causal
steps and steps of trees against the model's own forward under a dense mask a kind."""

import numpy as np
import pytest
import torch

transformers = pytest.importorskip("transformers")

from helpers import pkg
from span_oracle import depths, random_tree, seen_mask
from test_model_span import Served, tokens

paged_attention = pkg("model.paged_attention")

WINDOW = 40


def mixed_model(device):
    cfg = transformers.Qwen2Config(
        vocab_size=256, hidden_size=512, intermediate_size=256, num_hidden_layers=3, num_attention_heads=8,
        num_key_value_heads=2, max_position_embeddings=2048, initializer_range=0.08, sliding_window=WINDOW,
        use_sliding_window=True, layer_types=["sliding_attention", "full_attention", "sliding_attention"])
    torch.manual_seed(0)
    return transformers.Qwen2ForCausalLM(cfg).to(device=device, dtype=torch.float32).eval()


def dense(model, ids, seen, positions, device):
    """``seen``: (of layers with the window, of the others) [n, n]."""
    was = model.config._attn_implementation
    model.config._attn_implementation = "eager"
    low = torch.finfo(model.dtype).min
    masks = {kind: torch.zeros(m.shape).masked_fill(~torch.from_numpy(m), low)[None, None].to(device)
             for kind, m in zip(("sliding_attention", "full_attention"), seen)}
    try:
        with torch.inference_mode():
            return model(torch.tensor([ids], device=device), attention_mask=masks,
                         position_ids=torch.tensor([positions], device=device), use_cache=False).logits[0].float()
    finally:
        model.config._attn_implementation = was


def check(device, window, sinks, tol):
    model = mixed_model(device)
    served = Served(model, device)
    limits = [min(w for w in (WINDOW, window) if w is not None), window]
    kw = {"window": window, "sinks": sinks}
    rng = np.random.Generator(np.random.PCG64(7))
    contexts, counts = [tokens(90, 1), tokens(12, 2), tokens(33, 3)], [18, 5, 30]
    seqs = [served.add(ids) for ids in contexts]
    worst = 0.0
    _, got = served.step([(s, 0, ids[:-1]) for s, ids in zip(seqs, contexts)], **kw)
    _, last = served.step([(s, len(ids) - 1, ids[-1:]) for s, ids in zip(seqs, contexts)], **kw)
    for ids, rows, row in zip(contexts, got, last):
        n = len(ids)
        want = dense(model, ids, [seen_mask(0, n, w, sinks) for w in limits], list(range(n)), device)
        worst = max(worst, float((torch.cat([rows, row]) - want).abs().max()))
    parents = [random_tree(rng, n) for n in counts]
    drafted = [tokens(n, 20 + n) for n in counts]
    _, got = served.step([(s, len(ids), d) for s, ids, d in zip(seqs, contexts, drafted)], parents=parents, **kw)
    for ids, up, new, rows in zip(contexts, parents, drafted, got):
        n, m = len(ids), len(new)
        seen = []
        for w in limits:
            mask = np.zeros((n + m, n + m), bool)
            mask[:n, :n] = seen_mask(0, n, w, sinks)
            mask[n:] = seen_mask(n, m, w, sinks, up)
            seen.append(mask)
        want = dense(model, ids + new, seen, list(range(n)) + [n + d for d in depths(up)], device)[n:]
        worst = max(worst, float((rows - want).abs().max()))
    assert worst <= tol, worst


@pytest.mark.parametrize("window,sinks", [(None, 0), (64, 3)])
def test_cpu(monkeypatch, window, sinks):
    monkeypatch.setattr(paged_attention, "_BACKEND", None)
    check("cpu", window, sinks, 1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(None, 0), (64, 3)])
def test_gpu(device, monkeypatch, window, sinks):
    monkeypatch.setattr(paged_attention, "_BACKEND", None)
    check("cuda", window, sinks, 2e-3)
