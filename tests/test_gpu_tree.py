"""Trees of drafted tokens: masks and positions from the parents, attention
against 64 bits, the accepted path, and the rows it keeps."""

import numpy as np
import pytest
import torch

import cache8_oracle
from helpers import pkg
from span_oracle import CODE, Case, ancestors, depths, random_tree

pytestmark = pytest.mark.gpu

ops = pkg("paged_ops")

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
STARTS = [0, 1, 17, 63, 64, 200, 1000, 330, 2500]
COUNTS = [1, 5, 16, 33, 64, 1, 26, 100, 40]
SHAPES = [(8, 2, 128, BF16, BF16), (8, 8, 64, FP16, FP16), (6, 2, 80, BF16, BF16), (6, 2, 96, FP16, FP16),
          (24, 1, 128, BF16, BF16), (9, 3, 64, BF16, BF16), (7, 1, 128, FP16, FP16), (4, 2, 256, BF16, BF16),
          (4, 2, 64, FP32, FP32), (8, 2, 128, FP32, FP32), (8, 2, 128, BF16, CODE), (16, 16, 64, FP16, CODE),
          (6, 2, 80, BF16, CODE), (4, 1, 128, FP32, CODE), (3, 1, 40, FP16, FP16), (3, 1, 40, BF16, CODE)]


def trees(counts, seed=0):
    rng = np.random.Generator(np.random.PCG64(seed))
    return [random_tree(rng, n) if n else [] for n in counts]


def flat(parents):
    return torch.tensor([p for t in parents for p in t], dtype=torch.int32)


@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 4), (128, 70), (1000, 0)])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache_dtype", SHAPES)
def test_tree_attention_matches_64_bits(device, heads, kv_heads, dim, dtype, cache_dtype, window, sinks):
    parents = trees(COUNTS, seed=heads)
    case = Case(STARTS, COUNTS, heads, kv_heads, dim, dtype, cache_dtype, window=window, sinks=sinks, parents=parents,
                seed=dim)
    q, k, v, scales, step = case.place(device)
    tree = ops.pack_tree(step, flat(parents).to(device), window=window, sinks=sinks)
    case.check(ops.tree_attention(q, k, v, 1, step, tree, case.scaling, **scales))


@pytest.mark.parametrize("bs", [1, 8, 12, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache_dtype",
                         [(8, 2, 128, BF16, BF16), (4, 4, 64, FP32, FP32), (8, 2, 64, FP16, CODE)])
def test_other_block_sizes(device, bs, heads, kv_heads, dim, dtype, cache_dtype):
    parents = trees(COUNTS, seed=bs)
    for window in (None, 120):
        case = Case(STARTS, COUNTS, heads, kv_heads, dim, dtype, cache_dtype, bs=bs, parents=parents, seed=bs,
                    window=window, sinks=9 if window else 0)
        q, k, v, scales, step = case.place(device)
        tree = ops.pack_tree(step, flat(parents), window=window, sinks=case.sinks)
        case.check(ops.tree_attention(q, k, v, 1, step, tree, case.scaling, **scales))


@pytest.mark.parametrize("starts,counts", [([9000], [30]), ([9000], [1]), ([0], [300]), ([5000, 3], [64, 1000]),
                                           ([100] * 40, [7] * 40), ([5, 0, 77], [4, 0, 4])])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(8, 2, 128, BF16), (4, 4, 64, FP32)])
def test_other_steps(device, starts, counts, heads, kv_heads, dim, dtype):
    parents = trees(counts, seed=1)
    case = Case(starts, counts, heads, kv_heads, dim, dtype, parents=parents, seed=1)
    q, k, v, _, step = case.place(device)
    tree = ops.pack_tree(step, flat(parents))
    case.check(ops.tree_attention(q, k, v, 1, step, tree, case.scaling))


@pytest.mark.parametrize("window,sinks", [(None, 0), (150, 5)])
@pytest.mark.parametrize("dim,dtype", [(64, FP16), (80, BF16), (96, FP16), (128, BF16), (256, BF16)])
def test_more_units_than_compute_units(device, dim, dtype, window, sinks):
    counts = [1 + (37 * i) % 90 for i in range(20)]
    case = Case([13 * i * i for i in range(20)], counts, 32, 16, dim, dtype, parents=trees(counts), window=window,
                sinks=sinks, seed=dim)
    q, k, v, _, step = case.place(device)
    tree = ops.pack_tree(step, flat(case.parents).to(device), window=window, sinks=sinks)
    assert tree._plan.num_items * 16 > 256
    case.check(ops.tree_attention(q, k, v, 1, step, tree, case.scaling))


def test_a_chain_is_causal_attention_and_roots_see_the_context_alone(device):
    starts, counts = [300, 20], [50, 9]
    chain = [list(range(-1, n - 1)) for n in counts]
    causal = Case(starts, counts, 8, 2, 128, BF16, seed=6)
    q, k, v, _, step = causal.place(device)
    causal.check(ops.tree_attention(q, k, v, 1, step, ops.pack_tree(step, flat(chain)), causal.scaling))
    roots = [[-1] * n for n in counts]
    case = Case(starts, counts, 8, 2, 128, BF16, parents=roots, seed=6)
    q, k, v, _, step = case.place(device)
    for bad in (-1, -5, 10 ** 6, 2 ** 31 - 1):  # (what is no earlier node reads as a root)
        tree = ops.pack_tree(step, torch.full((sum(counts),), bad, dtype=torch.int32, device=device))
        case.check(ops.tree_attention(q, k, v, 1, step, tree, case.scaling))
    own = torch.cat([torch.arange(n, dtype=torch.int32) for n in counts])  # (a node is not its own parent)
    case.check(ops.tree_attention(q, k, v, 1, step, ops.pack_tree(step, own.to(device)), case.scaling))


@pytest.mark.parametrize("counts", [[1, 5, 64, 0, 33], [1000, 2], [1024], [31, 32, 33, 65]])
def test_masks_and_positions(device, counts):
    parents = trees(counts, seed=7)
    starts = [11 * i for i in range(len(counts))]
    table = torch.zeros((len(counts), 200), dtype=torch.int32, device=device)
    step = ops.pack_step(table, starts, counts, 16)
    tree = ops.pack_tree(step, flat(parents).to(device))
    masks, positions = tree.masks.cpu().numpy().view(np.uint32), tree.position_ids.cpu().numpy()
    first = 0
    for start, up in zip(starts, parents):
        n = len(up)
        bits = (masks[first:first + n, :, None] >> np.arange(32, dtype=np.uint32)) & 1
        bits = bits.reshape(n, masks.shape[1] * 32)
        want = np.zeros((n, bits.shape[1]), np.uint32)
        want[:, :n] = ancestors(up)
        assert np.array_equal(bits, want)
        assert np.array_equal(positions[first:first + n], start + np.asarray(depths(up), np.int64))
        first += n


@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache_dtype",
                         [(8, 2, 128, BF16, BF16), (4, 2, 64, FP32, FP32), (8, 2, 128, BF16, CODE),
                          (3, 1, 40, FP16, FP16)])
def test_new_rows_queries_out_and_streams(device, heads, kv_heads, dim, dtype, cache_dtype):
    counts, starts = [16, 1, 30], [70, 500, 3]
    parents = trees(counts, seed=2)
    case = Case(starts, counts, heads, kv_heads, dim, dtype, cache_dtype, parents=parents, seed=2)
    q, k, v, scales, step = case.place(device)
    gen = torch.Generator().manual_seed(4)
    rows = [torch.randn((sum(counts), kv_heads, dim), generator=gen).to(dtype).to(device) for _ in range(2)]
    tree = ops.pack_tree(step, flat(parents))
    k2, v2, s2 = k.clone(), v.clone(), {n: x.clone() for n, x in scales.items()}
    ops.reshape_and_cache(*rows, k2, v2, step.scatter_slots, 1, **s2)
    want = ops.tree_attention(q, k2, v2, 1, step, tree, case.scaling, **s2)
    k1, v1, s1 = k.clone(), v.clone(), {n: x.clone() for n, x in scales.items()}
    guard = torch.full((q.shape[0] + 2, heads, dim), 7.0, dtype=dtype, device=device)
    ops.tree_attention(q.transpose(0, 1).contiguous()[None], k1, v1, 1, step, tree, case.scaling, out=guard[1:-1],
                       new_key=rows[0], new_value=rows[1], **s1)
    assert torch.equal(guard[1:-1], want) and bool((guard[0] == 7).all()) and bool((guard[-1] == 7).all())
    assert torch.equal(k1.view(torch.uint8), k2.view(torch.uint8))
    assert torch.equal(v1.view(torch.uint8), v2.view(torch.uint8))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = ops.pack_tree(step, flat(parents))
        got = [ops.tree_attention(q, k2, v2, 1, step, other, case.scaling, **s2) for _ in range(3)]
    same = [ops.tree_attention(q, k2, v2, 1, step, tree, case.scaling, **s2) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(x, want) for x in got + same)


def test_missing_blocks(device):
    for heads, kv_heads, dim, dtype, cache in [(8, 2, 128, BF16, BF16), (4, 2, 64, FP32, FP32), (8, 2, 64, BF16, CODE)]:
        parents = trees([20, 20], seed=3)
        case = Case([400, 64], [20, 20], heads, kv_heads, dim, dtype, cache, parents=parents, seed=4)
        case.table[0, 3] = -1
        case.table[0, 20] = 10 ** 6
        case.table[1, :] = -1
        case.seen[0][:, 48:64] = False
        case.seen[0][:, 320:336] = False
        case.seen[1][:] = False
        case._reference()
        q, k, v, scales, step = case.place(device)
        out = ops.tree_attention(q, k, v, 1, step, ops.pack_tree(step, flat(parents)), case.scaling, **scales)
        case.check(out)
        assert bool((out[20:] == 0).all())


def plain_accept(parents, drafted, predicted):
    nodes, counts, nexts, first = [], [], [], 0
    for up in parents:
        n, path = len(up), [0] if up else []
        while path:
            want = predicted[first + path[-1]]
            ahead = [j for j in range(path[-1] + 1, n) if up[j] == path[-1] and drafted[first + j] == want]
            if not ahead:
                break
            path.append(ahead[0])
        nodes += path + [-1] * (n - len(path))
        counts.append(len(path))
        nexts.append(int(predicted[first + path[-1]]) if path else -1)
        first += n
    return nodes, counts, nexts


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("vocabulary", [1, 3, 50])
def test_accepted_paths(device, seed, vocabulary):
    counts = [[1, 40, 0, 26], [200, 64, 3], [1024], [65] * 9][seed]
    rng = np.random.Generator(np.random.PCG64(seed))
    parents = trees(counts, seed)
    if seed == 2:
        parents = [list(range(-1, 1023))]
    drafted, predicted = (rng.integers(0, vocabulary, sum(counts)) for _ in range(2))
    table = torch.zeros((len(counts), 200), dtype=torch.int32, device=device)
    step = ops.pack_step(table, [5] * len(counts), counts, 16)
    tree = ops.pack_tree(step, flat(parents).to(device))
    path = ops.accept_tree(step, tree, torch.from_numpy(drafted).to(device), torch.from_numpy(predicted).to(device))
    nodes, kept, nexts = plain_accept(parents, drafted, predicted)
    assert path.nodes.tolist() == nodes and path.counts.tolist() == kept and path.next_tokens.tolist() == nexts


def kept_case(seed, bs, counts, starts):
    rng = np.random.Generator(np.random.PCG64(seed))
    need = [-(-(s + c) // bs) for s, c in zip(starts, counts)]
    blocks = sum(need) + 2
    order = rng.permutation(blocks)
    table = np.full((len(counts), max(need)), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    nodes, kept = [], []
    for c in counts:
        n = int(rng.integers(0, c + 1))
        nodes += sorted(rng.permutation(c)[:n].tolist()) + [-1] * (c - n)
        kept.append(n)
    return table, blocks, nodes, kept


def moves(table, bs, starts, counts, nodes, kept):
    out, first = [], 0
    for i, (s, c) in enumerate(zip(starts, counts)):
        for j in range(min(kept[i], c)):
            node = nodes[first + j]
            if not (j <= node < c) or (j > 0 and node <= nodes[first + j - 1]):
                break
            slots = []
            for p in (s + node, s + j):
                b = table[i, p // bs] if p // bs < table.shape[1] else -1
                slots.append(int(b) * bs + p % bs if b >= 0 else -1)
            if node != j and min(slots) >= 0:
                out.append(tuple(slots))
        first += c
    return out


@pytest.mark.parametrize("dtype,kv_heads,dim", [(BF16, 8, 128), (FP16, 1, 40), (FP32, 3, 64), (BF16, 1, 33),
                                                (BF16, 32, 128)])
@pytest.mark.parametrize("bs", [1, 12, 16])
def test_kept_rows(device, dtype, kv_heads, dim, bs):
    counts, starts = [26, 1, 64, 0, 300, 7], [5, 40, 0, 9, 77, 16]
    table, blocks, nodes, kept = kept_case(dim + bs, bs, counts, starts)
    gen = torch.Generator().manual_seed(1)
    caches = [torch.randn((3, blocks, bs, kv_heads, dim), generator=gen).to(dtype) for _ in range(2)]
    step = ops.pack_step(torch.from_numpy(table).to(device), starts, counts, bs)
    dev = [c.to(device) for c in caches]
    ops.keep_rows(*dev, step, torch.tensor(nodes, dtype=torch.int32, device=device),
                  torch.tensor(kept, dtype=torch.int32, device=device))
    for got, cache in zip(dev, caches):
        want = cache.clone()
        rows = want.view(3, blocks * bs, -1)
        for a, b in moves(table, bs, starts, counts, nodes, kept):
            rows[:, b] = rows[:, a]
        assert torch.equal(got.cpu().view(torch.uint8), want.view(torch.uint8))


def test_kept_rows_of_bad_paths_and_missing_blocks(device):
    counts, starts, bs = [8, 8, 8, 8, 40], [5, 40, 9, 16, 30], 16
    table, blocks, _, _ = kept_case(3, bs, counts, starts)
    table[4, 2] = -1
    table[4, 3] = 10 ** 6
    nodes = [0, 3, 3, 5, 6, 7, -1, -1] + [2, 1, 5, 6, -1, -1, -1, -1] + [1, 4, 99, 7, -1, -1, -1, -1] + \
        [-1] * 8 + [1, 2, 5, 20, 25, 39] + [-1] * 34
    kept = [6, 4, 10 ** 6, -4, 6]
    caches = [torch.randn((2, blocks, bs, 2, 64)).to(BF16) for _ in range(2)]
    step = ops.pack_step(torch.from_numpy(table).to(device), starts, counts, bs)
    dev = [c.to(device) for c in caches]
    ops.keep_rows(*dev, step, torch.tensor(nodes, dtype=torch.int32, device=device),
                  torch.tensor(kept, dtype=torch.int32, device=device))
    limited = np.where((table >= 0) & (table < blocks), table, -1)
    for got, cache in zip(dev, caches):
        want = cache.clone()
        rows = want.view(2, blocks * bs, -1)
        for a, b in moves(limited, bs, starts, counts, nodes, kept):
            rows[:, b] = rows[:, a]
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("kv_heads,dim,bs", [(2, 64, 16), (1, 40, 16), (3, 128, 8), (2, 256, 32)])
def test_kept_rows_of_an_8bit_cache(device, kv_heads, dim, bs):
    """Values stay, but for a rounding where a block's scale grew."""
    counts, starts = [26, 1, 64, 100], [5, 40, 0, 77]
    table, blocks, nodes, kept = kept_case(dim, bs, counts, starts)
    gen = torch.Generator().manual_seed(1)
    held = []
    for _ in range(2):
        codes = torch.zeros((2, blocks, bs, kv_heads, dim), dtype=torch.uint8).view(CODE)
        scales = torch.zeros((2, blocks, kv_heads))
        for layer in range(2):
            rows = torch.randn((blocks * bs, kv_heads, dim), generator=gen)
            rows *= torch.exp(2 * torch.randn((blocks, 1, kv_heads, 1), generator=gen)).expand(
                -1, bs, -1, -1).reshape(-1, kv_heads, 1)
            cache8_oracle.write(codes[layer], scales[layer], rows, list(range(blocks * bs)))
        held.append((codes, scales))
    step = ops.pack_step(torch.from_numpy(table).to(device), starts, counts, bs)
    dev = [(c.to(device), s.to(device)) for c, s in held]
    ops.keep_rows(dev[0][0], dev[1][0], step, torch.tensor(nodes, dtype=torch.int32, device=device),
                  torch.tensor(kept, dtype=torch.int32, device=device), dev[0][1], dev[1][1])
    todo = moves(table, bs, starts, counts, nodes, kept)
    for (codes, scales), (got, got_scales) in zip(held, dev):
        got, got_scales = got.cpu(), got_scales.cpu()
        for layer in range(2):
            value = cache8_oracle.values(codes[layer], scales[layer]).double()  # [blocks, bs, heads, dim]
            want_scale = scales[layer].clone()
            for a, b in todo:
                want_scale[b // bs] = torch.maximum(want_scale[b // bs], scales[layer, a // bs])
            assert torch.equal(got_scales[layer], want_scale)
            want = value.clone().view(blocks * bs, kv_heads, dim)
            for a, b in todo:  # (rows move down in order: each is read before it is written)
                want[b] = value.view(blocks * bs, kv_heads, dim)[a]
            factor = want_scale.double().repeat_interleave(bs, dim=0)[..., None]
            coded = (want / factor).float().to(CODE).double() * factor
            back = cache8_oracle.values(got[layer], got_scales[layer]).double().view(blocks * bs, kv_heads, dim)
            assert torch.equal(back, coded)


def test_a_step_together(device):
    """Pack, attend, accept and keep, eagerly and as a graph over changing trees:
    the kept rows then serve a causal step."""
    heads, kv_heads, dim, bs, starts, counts = 8, 2, 128, 16, [100, 260, 3], [20, 31, 9]
    parents = trees(counts, seed=11)
    case = Case(starts, counts, heads, kv_heads, dim, BF16, parents=parents, seed=11, poison=False, layers=3)
    q, k, v, _, step = case.place(device)
    rng = np.random.Generator(np.random.PCG64(5))
    drafted = torch.from_numpy(rng.integers(0, 3, sum(counts))).to(device)
    predicted = torch.from_numpy(rng.integers(0, 3, sum(counts))).to(device)
    tree = ops.pack_tree(step, flat(parents).to(device))
    out = torch.empty_like(q)

    def pass_():
        tree.rerun()
        ops.tree_attention(q, k, v, 2, step, tree, case.scaling, out=out)
        path = ops.accept_tree(step, tree, drafted, predicted)
        ops.keep_rows(k, v, step, path.nodes, path.counts)
        return path

    saved = k.clone(), v.clone()
    path = pass_()
    case.check(out)
    nodes, kept, nexts = plain_accept(parents, drafted.tolist(), predicted.tolist())
    assert path.nodes.tolist() == nodes and path.counts.tolist() == kept and path.next_tokens.tolist() == nexts
    assert sum(kept) > len(kept)
    after = k.clone(), v.clone()
    rows = [x.clone().view(3, -1, kv_heads * dim) for x in saved]
    for a, b in moves(case.table, bs, starts, counts, nodes, kept):
        for x in rows:
            x[:, b] = x[:, a]
    for got, want in zip(after, rows):
        assert torch.equal(got.view(torch.uint8), want.view_as(got).view(torch.uint8))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = pass_()
    for seed in (12, 13, 11):
        other = trees(counts, seed=seed)
        tree.repack(flat(other).to(device))
        k.copy_(saved[0]), v.copy_(saved[1])
        out.zero_()
        graph.replay()
        again = Case(starts, counts, heads, kv_heads, dim, BF16, parents=other, seed=11, poison=False, layers=3)
        again.check(out)
        nodes, kept, nexts = plain_accept(other, drafted.tolist(), predicted.tolist())
        assert captured.nodes.tolist() == nodes and captured.counts.tolist() == kept


def test_a_refused_call_writes_no_rows(device):
    case = Case([4000], [6], 8, 2, 128, BF16, parents=trees([6]))
    q, k, v, _, step = case.place(device)
    tree = ops.pack_tree(step, flat(case.parents).to(device))
    assert tree._plan.num_partial_rows > 0
    tree._workspace_bytes = 0
    was = k.clone(), v.clone()
    rows = torch.ones((6, 2, 128), dtype=BF16, device=device)
    with pytest.raises(RuntimeError, match="workspace of"):
        ops.tree_attention(q, k, v, 1, step, tree, 1.0, new_key=rows, new_value=rows)
    for x, y in zip(was, (k, v)):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))


def test_refusals(device):
    case = Case([40, 9], [6, 3], 8, 2, 128, BF16, parents=trees([6, 3]))
    q, k, v, _, step = case.place(device)
    parents = flat(case.parents).to(device)
    tree = ops.pack_tree(step, parents)
    for bad in (parents[:-1], parents.float()):
        with pytest.raises(ValueError, match="parents must be"):
            ops.pack_tree(step, bad)
    with pytest.raises(ValueError, match="than the window"):
        ops.pack_tree(step, parents, window=5)
    with pytest.raises(ValueError, match="sinks go with a window"):
        ops.pack_tree(step, parents, sinks=5)
    _, _, _, _, other = case.place(device)
    with pytest.raises(ValueError, match="another step"):
        ops.tree_attention(q, k, v, 1, other, tree, 1.0)
    with pytest.raises(ValueError, match="was packed for"):
        ops.tree_attention(q[:, :4], k, v, 1, step, tree, 1.0)
    with pytest.raises(ValueError, match="another dtype than the cache's"):
        ops.tree_attention(q, k, v, 1, step, ops.pack_tree(step, parents, dtype=FP16), 1.0)
    with pytest.raises(RuntimeError, match="Layer index"):
        ops.tree_attention(q, k, v, 2, step, tree, 1.0)
    with pytest.raises(ValueError, match="together"):
        ops.tree_attention(q, k, v, 1, step, tree, 1.0, new_key=q)
    step.repack([40, 9], [6, 3])
    with pytest.raises(RuntimeError, match="repack its tree"):
        ops.tree_attention(q, k, v, 1, step, tree, 1.0)
    tree.repack()
    ops.tree_attention(q, k, v, 1, step, tree, 1.0)
    tokens = torch.zeros(9, dtype=torch.int64, device=device)
    with pytest.raises(ValueError, match="drafted must be"):
        ops.accept_tree(step, tree, tokens.int(), tokens)
    with pytest.raises(ValueError, match="predicted must be"):
        ops.accept_tree(step, tree, tokens, tokens[:-1])
    nodes, counts = torch.zeros(9, dtype=torch.int32, device=device), torch.zeros(2, dtype=torch.int32, device=device)
    with pytest.raises(ValueError, match="nodes must be"):
        ops.keep_rows(k, v, step, nodes[:-1], counts)
    with pytest.raises(ValueError, match="counts must be"):
        ops.keep_rows(k, v, step, nodes, counts.long())
    with pytest.raises(ValueError, match="blocks of 16"):
        ops.keep_rows(k.view(2, -1, 8, 2, 128), v.view(2, -1, 8, 2, 128), step, nodes, counts)
    with pytest.raises(RuntimeError, match="device tensors"):
        ops.keep_rows(k, v, step, nodes.cpu(), counts)
    table = torch.zeros((1, 100), dtype=torch.int32, device=device)
    big = ops.pack_step(table, [0], [1025], 16)
    with pytest.raises(ValueError, match="1025 nodes"):
        ops.pack_tree(big, torch.zeros(1025, dtype=torch.int32))
