"""Models whose layers see a window, and steps of trees, through the paged hook:
logits against the model's own forward under a dense mask, on a CPU store (the SDPA
path) and on the GPU (the HIP kernels), in fp32 and for 8-bit stores in bf16."""

import numpy as np
import pytest
import torch

from helpers import pkg
from span_oracle import depths, random_tree, seen_mask

transformers = pytest.importorskip("transformers")

paged_attention = pkg("model.paged_attention")
backends = pkg("model.attention_backends")
manager_mod = pkg("memory.manager")
sequence_mod = pkg("engine.request")
ops = pkg("paged_ops")

BLOCK_SIZE = 16


def tiny_model(kind, device, dtype=torch.float32, window=None, layers=2, heads=8, kv_heads=2, head_dim=64):
    config = {"llama": transformers.LlamaConfig, "qwen2": transformers.Qwen2Config}[kind]
    extra = {"sliding_window": window, "use_sliding_window": True,
             "layer_types": ["sliding_attention"] * layers} if kind == "qwen2" else {"head_dim": head_dim}
    cfg = config(vocab_size=256, hidden_size=heads * head_dim, intermediate_size=256, num_hidden_layers=layers,
                 num_attention_heads=heads, num_key_value_heads=kv_heads,
                 max_position_embeddings=2048, initializer_range=0.08, **extra)
    torch.manual_seed(0)
    cls = {"llama": transformers.LlamaForCausalLM, "qwen2": transformers.Qwen2ForCausalLM}[kind]
    model = cls(cfg).to(device=device, dtype=dtype)
    return model.eval()


def dense_logits(model, ids, seen, positions, device):
    """The model's own forward under a dense mask."""
    was = model.config._attn_implementation
    model.config._attn_implementation = "eager"
    mask = torch.zeros(seen.shape, dtype=model.dtype).masked_fill(~torch.from_numpy(seen), torch.finfo(model.dtype).min)
    try:
        with torch.inference_mode():
            return model(torch.tensor([ids], device=device), attention_mask=mask[None, None].to(device),
                         position_ids=torch.tensor([positions], device=device), use_cache=False).logits[0].float()
    finally:
        model.config._attn_implementation = was


def causal(n, window=None, sinks=0):
    return seen_mask(0, n, window, sinks)


class Served:
    def __init__(self, model, device, dtype=None):
        self.model, self.device = model, device
        self.store = manager_mod.PagedKVCacheManager.from_model_config(
            model.config, total_blocks=200, block_size=BLOCK_SIZE, dtype=dtype or model.dtype, device=device)
        paged_attention.register_paged_attention(model)

    def add(self, prompt):
        seq = sequence_mod.Request(seq_id=len(prompt), prompt_token_ids=list(prompt))
        self.store.allocate_prefix_blocks(seq)
        return seq

    def step(self, entries, **kw):
        for seq, start, tokens in entries:
            while seq.block_table.get_tokens_count() < start + len(tokens):
                self.store.allocate_slot_for_next_token(seq)
        ctx = paged_attention.PagedStepContext(self.store, [e[0] for e in entries], [e[1] for e in entries],
                                               [len(e[2]) for e in entries], **kw)
        flat = torch.tensor([[t for e in entries for t in e[2]]], device=self.device)
        with torch.inference_mode():
            logits = paged_attention.run_paged_forward(self.model, ctx, flat)[0].float()
        return ctx, list(torch.split(logits, [len(e[2]) for e in entries]))


@pytest.fixture(autouse=True)
def restore_backend(monkeypatch):
    monkeypatch.setattr(paged_attention, "_BACKEND", paged_attention._BACKEND)


def tokens(n, seed):
    return np.random.Generator(np.random.PCG64(seed)).integers(0, 256, n).tolist()


def check_windows(device, kind, layer_window, window, sinks, tol):
    """Prompts in chunks, then decodes, of contexts inside and past the window."""
    model = tiny_model(kind, device, window=layer_window)
    both = [w for w in (layer_window, window) if w is not None]
    limit = min(both) if both else None
    streams = [tokens(90, 1), tokens(20, 2), tokens(150, 3)]
    want = [dense_logits(model, ids, causal(len(ids), limit, sinks), list(range(len(ids))), device) for ids in streams]
    served = Served(model, device)
    kw = {"window": window, "sinks": sinks}
    seqs = [served.add(ids[:n]) for ids, n in zip(streams, (40, 15, 100))]
    plan = [[(0, 0, 30), (1, 0, 15)], [(0, 30, 10), (2, 0, 100)]]
    plan += [[(0, 40 + i, 1), (1, 15 + i, 1), (2, 100 + i, 1)] for i in range(5)]
    plan += [[(0, 45, 40), (2, 105, 1)], [(0, 85, 1), (2, 106, 44)]]
    worst = 0.0
    for entries in plan:
        _, got = served.step([(seqs[i], start, streams[i][start:start + n]) for i, start, n in entries], **kw)
        for (i, start, n), rows in zip(entries, got):
            worst = max(worst, float((rows - want[i][start:start + n]).abs().max()))
    assert worst <= tol, worst


@pytest.mark.parametrize("kind,layer_window,window,sinks", [("qwen2", 24, None, 0), ("llama", None, 17, 5),
                                                           ("qwen2", 40, 64, 3)])
def test_cpu_windows_match_the_models_forward(monkeypatch, kind, layer_window, window, sinks):
    monkeypatch.setattr(paged_attention, "_BACKEND", None)
    check_windows("cpu", kind, layer_window, window, sinks, 1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,layer_window,window,sinks", [("qwen2", 24, None, 0), ("llama", None, 17, 5),
                                                           ("qwen2", 40, 64, 3), ("qwen2", 4096, None, 0)])
def test_gpu_windows_match_the_models_forward(device, kind, layer_window, window, sinks):
    check_windows("cuda", kind, layer_window, window, sinks, 2e-3)


def check_trees(device, window, sinks, tol):
    model = tiny_model("llama", device)
    served = Served(model, device)
    rng = np.random.Generator(np.random.PCG64(4))
    contexts, counts = [tokens(50, 1), tokens(7, 2), tokens(120, 3)], [20, 1, 33]
    seqs = [served.add(ids) for ids in contexts]
    served.step([(s, 0, ids) for s, ids in zip(seqs, contexts)], window=window, sinks=sinks)
    parents = [random_tree(rng, n) for n in counts]
    drafted = [tokens(n, 10 + n) for n in counts]
    ctx, got = served.step([(s, len(ids), d) for s, ids, d in zip(seqs, contexts, drafted)], parents=parents,
                           window=window, sinks=sinks)
    worst = 0.0
    for ids, up, new, rows in zip(contexts, parents, drafted, got):
        n, m = len(ids), len(new)
        seen = np.zeros((n + m, n + m), bool)
        seen[:n, :n] = causal(n, window, sinks)
        seen[n:] = seen_mask(n, m, window, sinks, up)
        at = list(range(n)) + [n + d for d in depths(up)]
        want = dense_logits(model, ids + new, seen, at, device)[n:]
        worst = max(worst, float((rows - want).abs().max()))
    assert worst <= tol, worst
    return model, served, contexts, seqs, parents, drafted, ctx, got


@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 4)])
def test_cpu_trees_match_the_models_forward(monkeypatch, window, sinks):
    monkeypatch.setattr(paged_attention, "_BACKEND", None)
    check_trees("cpu", window, sinks, 1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 4)])
def test_gpu_tree_step_then_decode(device, window, sinks):
    """Verify trees, keep the accepted rows, and go on from them."""
    model, served, contexts, seqs, parents, drafted, ctx, got = check_trees("cuda", window, sinks, 2e-3)
    predicted = torch.cat([rows.argmax(dim=-1) for rows in got])
    # Make some of the model's own choices drafted ones: a child takes its parent's.
    first = 0
    for up, new in zip(parents, drafted):
        for j in range(1, len(up)):
            if j % 2:
                new[j] = int(predicted[first + up[j]])
        first += len(up)
    ctx, got = served.step([(s, len(ids), d) for s, ids, d in zip(seqs, contexts, drafted)], parents=parents,
                           window=window, sinks=sinks)
    predicted = torch.cat([rows.argmax(dim=-1) for rows in got])
    flat = torch.tensor([t for d in drafted for t in d], device="cuda")
    path = ops.accept_tree(ctx.packed, ctx.tree_for(8, window if window and ctx.packed.max_context > window else None),
                           flat, predicted)
    kept = served.store.keep_accepted(ctx, path)
    assert max(kept) > 1
    entries, streams, first = [], [], 0
    for seq, ids, new, n, nxt in zip(seqs, contexts, drafted, kept, path.next_tokens.tolist()):
        nodes = path.nodes[first:first + n].tolist()
        first += len(new)
        streams.append(ids + [new[j] for j in nodes] + [nxt])
        assert seq.block_table.get_tokens_count() == len(ids) + n
        assert len(seq.block_table.get_physical_blocks()) == -(-(len(ids) + n) // BLOCK_SIZE)
        entries.append((seq, len(ids) + n, [nxt]))
    _, rows = served.step(entries, window=window, sinks=sinks)
    for ids, row in zip(streams, rows):
        want = dense_logits(model, ids, causal(len(ids), window, sinks), list(range(len(ids))), "cuda")[-1]
        assert float((row[0] - want).abs().max()) <= 2e-3


@pytest.mark.gpu
def test_gpu_tree_step_of_an_8bit_store(device):
    """A bf16 model over an 8-bit store: kept rows are the values the store held."""
    model = tiny_model("llama", "cuda", dtype=torch.bfloat16)
    served = Served(model, "cuda", dtype=torch.float8_e4m3fn)
    ids, up = tokens(30, 1), [-1, 0, 0, 1, 1, 2, 3, 5]
    seq = served.add(ids)
    served.step([(seq, 0, ids)])
    new = tokens(len(up), 5)
    ctx, _ = served.step([(seq, 30, new)], parents=[up])
    slots = ctx.packed.scatter_slots.clone()
    held = [[x(layer, slots).float() for layer in range(2)] for x in (served.store.gather_layer_keys,
                                                                     served.store.gather_layer_values)]
    nodes = torch.tensor([0, 2, 5, -1, -1, -1, -1, -1], dtype=torch.int32, device="cuda")
    path = ops.AcceptedPath(nodes, torch.tensor([3], dtype=torch.int32, device="cuda"),
                            torch.tensor([1], device="cuda"))
    assert served.store.keep_accepted(ctx, path) == [3]
    for x, was in zip((served.store.gather_layer_keys, served.store.gather_layer_values), held):
        for layer in range(2):
            got = x(layer, slots[:3]).float()
            want = was[layer][[0, 2, 5]]
            # (a block's scale may have grown: half a step of four significant bits, or of the least code)
            assert bool(((got - want).abs() <= want.abs() * 2.0 ** -4 + 2.0 ** -10 * 448 * 2.0 ** -6).all())


def test_contexts_refuse_bad_limits():
    model_store = manager_mod.PagedKVCacheManager(total_blocks=8, block_size=4, num_heads=1, head_dim=8, device="cpu")
    seq = sequence_mod.Request(seq_id=1, prompt_token_ids=[1, 2, 3])
    model_store.allocate_prefix_blocks(seq)
    make = paged_attention.PagedStepContext
    for kw in ({"window": 0}, {"sinks": -1}, {"parents": [[-1]]}, {"parents": []}):
        with pytest.raises(ValueError):
            make(model_store, [seq], [0], [3], **kw)
    assert make(model_store, [seq], [0], [3], window=5).window_of(3) == 3
    assert make(model_store, [seq], [0], [3], window=5).window_of(None) == 5
    assert make(model_store, [seq], [0], [3]).window_of(7) == 7
    with pytest.raises(RuntimeError, match="device memory"):
        model_store.keep_accepted(make(model_store, [seq], [0], [3]), None)


def test_block_tables_truncate():
    store = manager_mod.PagedKVCacheManager(total_blocks=8, block_size=4, num_heads=1, head_dim=8, device="cpu")
    seq = sequence_mod.Request(seq_id=1, prompt_token_ids=list(range(14)))
    store.allocate_prefix_blocks(seq)
    table = seq.block_table
    blocks, free = table.get_physical_blocks(), store.allocator.get_num_free_blocks()
    table.truncate(9)
    assert table.get_physical_blocks() == blocks[:3] and table.get_tokens_count() == 9
    assert store.allocator.get_num_free_blocks() == free + 1
    assert store.tables.host[table.row, :5].tolist() == blocks[:3] + [-1, -1] and store.tables.tokens[table.row] == 9
    table.truncate(8)
    assert table.get_physical_blocks() == blocks[:2]
    table.append_tokens(3)
    assert table.get_tokens_count() == 11 and len(table.get_physical_blocks()) == 3
    with pytest.raises(ValueError, match="cannot keep"):
        table.truncate(12)
    table.truncate(0)
    assert table.get_physical_blocks() == [] and store.allocator.get_num_free_blocks() == 8
