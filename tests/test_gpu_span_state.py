"""What a step under a window, or of trees, keeps from one call to the next, and what a
call leaves as it was."""

import gc
import weakref

import numpy as np
import pytest
import torch

from helpers import pkg
from span_oracle import CODE, Case, ancestors, random_tree
from test_gpu_tree import plain_accept

pytestmark = pytest.mark.gpu

ops = pkg("paged_ops")
manager_mod = pkg("memory.manager")
request_mod = pkg("engine.request")
paged_attention = pkg("model.paged_attention")

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def store_of(device, lengths, kv_heads=2, head_dim=64, query_heads=8, blocks=600):
    m = manager_mod.PagedKVCacheManager(total_blocks=blocks, block_size=16, num_heads=kv_heads, head_dim=head_dim,
                                        dtype=BF16, num_layers=1, device=device)
    m.num_query_heads = query_heads
    seqs = [request_mod.Request(i + 1, list(range(n))) for i, n in enumerate(lengths)]
    for seq in seqs:
        m.allocate_prefix_blocks(seq)
    return m, seqs


def slots_of(m, seqs, lengths):
    out = []
    for seq, n in zip(seqs, lengths):
        blocks = np.asarray(seq.block_table.get_physical_blocks(), np.int64)
        out.append(blocks[np.arange(n) // 16] * 16 + np.arange(n) % 16)
    return np.concatenate(out)


def attend(m, step, window, query_heads=8):
    q = torch.randn((step.num_query_tokens, query_heads, m.head_dim), dtype=BF16, device=m.device)
    return ops.attention(q, m.key_cache, m.value_cache, 0, step, 0.1, window=window, sinks=4)


def test_gather_slots_are_there_after_a_windowed_call(device):
    """The lists of a window are no later step on the pool: slots first read behind it
    (and behind a repack with it) are the step's, and it makes no other step stale."""
    lengths = [200, 330]
    m, seqs = store_of(device, lengths)
    want = slots_of(m, seqs, lengths)
    context = paged_attention.PagedStepContext(m, seqs, [n - 1 for n in lengths], [1, 1])
    attend(m, context.packed, 48)
    assert [s is not None for s in context.packed._windows.values()] == [True]
    assert np.array_equal(context.gather_slots.cpu().numpy(), want)
    older = m.pack_step(seqs, [n - 1 for n in lengths], [1, 1])
    newer = m.pack_step(seqs, [n - 1 for n in lengths], [1, 1])
    attend(m, older, 48)
    assert np.array_equal(newer.gather_slots.cpu().numpy(), want)
    attend(m, newer, 48)
    newer.repack([n - 2 for n in lengths], [1, 1])
    assert np.array_equal(newer.gather_slots.cpu().numpy(), slots_of(m, seqs, [n - 1 for n in lengths]))
    with pytest.raises(RuntimeError, match="earlier step"):
        older.gather_slots


@pytest.mark.parametrize("window", [48, 4096])
def test_a_step_goes_with_its_last_reference(device, window):
    """Under a window that its contexts reach past, and under one that they do not: its
    device memory does not wait for the garbage collector."""
    m, seqs = store_of(device, [200, 330])
    step = m.pack_step(seqs, [199, 329], [1, 1])
    attend(m, step, window)
    gone = weakref.ref(step)
    gc.disable()
    try:
        del step
        assert gone() is None
    finally:
        gc.enable()


def test_a_step_packed_again_for_its_heads_splits_a_window_as_a_new_one(device):
    """A store that does not know its model's heads packs a step again for them, with
    the partition that it had: which is none that a caller asked for."""
    lengths = [6000, 5000, 7000]
    m, seqs = store_of(device, lengths, query_heads=None, blocks=1200)
    starts = [n - 1 for n in lengths]
    context = paged_attention.PagedStepContext(m, seqs, starts, [1] * 3)
    first = context.packed
    step = context.packed_for(8)
    assert step is not first and step.partition_size == first.partition_size
    m.num_query_heads = 8
    fresh = m.pack_step(seqs, starts, [1] * 3)
    for window in (256, 1024, 3000):
        got, want = (ops._window_step(s, window, 4, 2, 8, 64, BF16).partition_size for s in (step, fresh))
        assert got == want
    given = m.pack_rows(context._rows, context._starts, context._counts, num_query_heads=8, partition_size=512)
    assert ops._window_step(given, 1024, 4, 2, 8, 64, BF16).partition_size == 512


def flat(parents, device):
    return torch.tensor([p for t in parents for p in t], dtype=torch.int32, device=device)


def check_tree(step, tree, parents, drafted, predicted):
    masks, first = tree.masks.cpu().numpy().view(np.uint32), 0
    for up in parents:
        n = len(up)
        bits = ((masks[first:first + n, :, None] >> np.arange(32, dtype=np.uint32)) & 1).reshape(n, -1)
        assert np.array_equal(bits[:, :n], ancestors(up))
        first += n
    path = ops.accept_tree(step, tree, drafted, predicted)
    nodes, kept, nexts = plain_accept(parents, drafted.tolist(), predicted.tolist())
    assert path.nodes.tolist() == nodes and path.counts.tolist() == kept and path.next_tokens.tolist() == nexts


def test_trees_of_one_tensor_of_parents(device):
    """A tree accepts the paths of the parents that its masks are of, whatever another
    tree of the same tensor, or its owner, has put there since."""
    counts = [30, 1, 45]
    rng = np.random.Generator(np.random.PCG64(3))
    old, new, last = ([random_tree(rng, n) for n in counts] for _ in range(3))
    case = Case([100, 7, 300], counts, 8, 2, 128, BF16, parents=old)
    q, k, v, _, step = case.place(device)
    drafted, predicted = (torch.from_numpy(rng.integers(0, 2, sum(counts))).to(device) for _ in range(2))
    shared = flat(old, device)
    one, two = ops.pack_tree(step, shared), ops.pack_tree(step, shared, window=64, sinks=3)
    paths = [plain_accept(p, drafted.tolist(), predicted.tolist()) for p in (old, new, last)]
    assert paths[0] != paths[1] and paths[1] != paths[2]
    one.repack(flat(new, device))
    check_tree(step, one, new, drafted, predicted)
    check_tree(step, two, old, drafted, predicted)
    two.repack()  # (reads the tensor as it is)
    check_tree(step, two, new, drafted, predicted)
    shared.copy_(flat(last, device))
    check_tree(step, one, new, drafted, predicted)
    one.rerun()
    check_tree(step, one, last, drafted, predicted)
    check_tree(step, two, new, drafted, predicted)


@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache_dtype", [
    (8, 2, 128, BF16, BF16), (9, 3, 64, FP16, FP16), (4, 2, 256, BF16, BF16), (4, 2, 64, FP32, FP32),
    (8, 2, 128, BF16, CODE)])
def test_a_graph_of_trees_whose_runs_change(device, heads, kv_heads, dim, dtype, cache_dtype):
    """A captured layer of trees whose contexts shrink and grow again, so that tiles are
    split in other runs, or in none, at other places of the lists."""
    counts = [20, 90, 9]
    rng = np.random.Generator(np.random.PCG64(dim))
    places = [[3000, 2500, 2900], [40, 2400, 700], [2900, 0, 130], [70, 64, 1], [2999, 2222, 1111]]
    cases = [Case(starts, counts, heads, kv_heads, dim, dtype, cache_dtype, poison=False, drop=False, seed=4,
                  parents=[random_tree(rng, n) for n in counts]) for starts in places]
    q, k, v, scales, _ = cases[0].place(device)
    table = torch.zeros(cases[0].table.shape, dtype=torch.int32, device=device)

    def fill(c):
        table.fill_(-1)
        table[:, :c.full_table.shape[1]] = torch.from_numpy(c.full_table).to(device)
        for cache, x in ((k, c.keys), (v, c.vals)):
            cache.view(torch.uint8)[1, :x.shape[0]] = x.view(torch.uint8).to(device)
        for name, s in c.scales.items():
            scales[name][1, :s.shape[0]] = s.to(device)
        q.copy_(c.query)

    fill(cases[0])
    step = ops.pack_step(table, cases[0].starts, counts, 16, num_kv_heads=kv_heads, num_query_heads=heads,
                         head_dim=dim, dtype=cache_dtype)
    tree = ops.pack_tree(step, flat(cases[0].parents, device))
    out = torch.zeros_like(q)

    def layer():
        step.rerun()
        tree.rerun()
        ops.tree_attention(q, k, v, 1, step, tree, cases[0].scaling, out=out, **scales)

    layer()
    cases[0].check(out)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        layer()
    sizes = set()
    for c in cases + cases[::-1]:
        fill(c)
        step.repack(c.starts, counts)
        tree.repack(flat(c.parents, device))
        plan = ops._plan_tree(step, tree._dims, tree._plan.split_stages)
        sizes.add((plan.num_items, plan.num_merge_items))
        out.zero_()
        graph.replay()
        c.check(out)
        c.check(ops.tree_attention(q, k, v, 1, step, tree, c.scaling, **scales))
    assert len(sizes) > 2


@pytest.mark.parametrize("starts,counts", [([40, 300, 700], [1, 33, 1]), ([40, 700], [1, 1])])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache_dtype", [
    (8, 2, 128, BF16, BF16), (4, 2, 64, FP32, FP32), (8, 2, 128, BF16, CODE)])
def test_a_refused_windowed_call_writes_no_rows(device, heads, kv_heads, dim, dtype, cache_dtype, starts, counts):
    case = Case(starts, counts, heads, kv_heads, dim, dtype, cache_dtype, window=50, sinks=3)
    q, k, v, scales, step = case.place(device)
    rows = torch.full((sum(counts), kv_heads, dim), 300.0, dtype=dtype, device=device)

    def call():
        ops.attention(q, k, v, 1, step, case.scaling, new_key=rows, new_value=rows, window=50, sinks=3, **scales)

    call()
    for cached in step._window_calls.values():
        cached[0]._obj.workspace_bytes = 8
    rows.mul_(1.5)
    was = [x.clone() for x in (k, v, *scales.values())]
    with pytest.raises(RuntimeError, match="workspace of"):
        call()
    for x, y in zip(was, (k, v, *scales.values())):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_a_windowed_step_refuses_a_write_inside_the_prefill(device):
    case = Case([40, 0], [1, 33], 8, 2, 128, BF16, window=50)
    q, k, v, _, step = case.place(device)
    rows = torch.zeros((34, 2, 128), dtype=BF16, device=device)
    with pytest.raises(ValueError, match="fused_prefill_write"):
        ops.attention(q, k, v, 1, step, 1.0, new_key=rows, new_value=rows, fused_prefill_write=True, window=50)
    ops.attention(q, k, v, 1, step, 1.0, new_key=rows, new_value=rows, fused_prefill_write=False, window=50)


def test_trees_of_other_sizes_after_a_repack(device):
    """The same number of nodes, dealt otherwise to the sequences."""
    starts, counts, others = [700, 90, 0], [40, 16, 8], [8, 16, 40]
    rng = np.random.Generator(np.random.PCG64(9))
    parents, drawn = ([random_tree(rng, n) for n in c] for c in (counts, others))
    ends = [s + max(a, b) for s, a, b in zip(starts, counts, others)]
    table, at = np.full((3, -(-max(ends) // 16)), -1, np.int32), 0
    cases = [Case(starts, c, 8, 2, 128, BF16, parents=p, seed=9, poison=False, drop=False)
             for c, p in ((counts, parents), (others, drawn))]
    blocks = sum(-(-e // 16) for e in ends)
    k, v = (torch.zeros((2, blocks, 16, 2, 128), dtype=BF16, device=device) for _ in range(2))
    for i, e in enumerate(ends):
        n = -(-e // 16)
        table[i, :n] = np.arange(at, at + n)
        at += n
    q = torch.zeros((64, 8, 128), dtype=BF16, device=device)

    def fill(c):
        for i, (s, n) in enumerate(zip(c.starts, c.counts)):
            pos = np.arange(s + n)
            mine, here = (torch.from_numpy(t[i, pos // 16].astype(np.int64) * 16 + pos % 16)
                          for t in (c.full_table, table))
            for cache, x in ((k, c.keys), (v, c.vals)):
                cache[1].view(-1, 2, 128)[here.to(device)] = x.view(-1, 2, 128)[mine].to(device)
        q.copy_(c.query)

    fill(cases[0])
    step = ops.pack_step(torch.from_numpy(table).to(device), starts, counts, 16, num_kv_heads=2, num_query_heads=8,
                         head_dim=128, dtype=BF16)
    tree = ops.pack_tree(step, flat(parents, device))
    for c in cases + cases[:1]:
        fill(c)
        step.repack(starts, c.counts)
        tree.repack(flat(c.parents, device))
        c.check(ops.tree_attention(q, k, v, 1, step, tree, c.scaling))


def test_refusals_of_trees_and_windows_that_outgrow_their_lists(device, monkeypatch):
    case = Case([3000], [26], 8, 2, 128, BF16, parents=[list(range(-1, 25))], drop=False)
    q, k, v, _, _ = case.place(device)
    step = ops.pack_step(torch.from_numpy(case.table).to(device), [40], [26], 16, num_kv_heads=2, num_query_heads=8,
                         head_dim=128, dtype=BF16)
    tree = ops.pack_tree(step, flat(case.parents, device))
    step.repack([3000], [26])
    with pytest.raises(ValueError, match="longer work lists"):
        tree.repack()
    with pytest.raises(RuntimeError, match="repack its tree"):
        ops.tree_attention(q, k, v, 1, step, tree, case.scaling)
    case.check(ops.tree_attention(q, k, v, 1, step, ops.pack_tree(step, tree.parents), case.scaling))
    decode = ops.pack_step(torch.from_numpy(case.table).to(device), [3000], [1], 16, num_kv_heads=2,
                           num_query_heads=8, head_dim=128, dtype=BF16)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="a graph cannot capture"):
        ops.attention(q[:1], k, v, 1, decode, 1.0, window=64)
