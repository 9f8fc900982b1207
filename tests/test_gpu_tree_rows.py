"""Tokens of a drafted-token step that no row has, and rows that got no pages (core/tree_decode.py): what the plan says of them, and that the
store, the attention and the acceptance behind it leave everything of other rows as it was."""
import numpy as np
import pytest
import torch

from oracle import ref_tree as ref
from tree_util import i32, random_parents, starts_of, tables

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    import micro_vllm_amd  # noqa: F401
    from micro_vllm_amd.core import tree_decode
    return tree_decode


def stale_plan(ops, rows, tokens, max_nodes, mask, slots):
    """A plan's buffers as an earlier step left them: `slots` are places that belong to someone else by now."""
    out = ops.TreePlan.empty(rows, tokens, max_nodes, DEV, mask=mask)
    for t in out:
        if t is not None:
            t.fill_(3)
    out.slots.copy_(slots)
    return out


@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("lead,counts,tail,max_nodes", [
    (0, [3], 1, None), (0, [1], 900, None), (0, [5, 0, 8], 9, None), (4, [5, 7], 0, None), (70, [64, 1], 700, None), (0, [40, 6], 3, 10),
    (0, [0, 0], 50, 4), (3, [200, 256], 5, 65), (0, [1] * 300, 1000, None)])
def test_tokens_that_no_row_has_name_no_place(ops, tree, lead, counts, tail, max_nodes):
    """Tokens in front of the first row, behind the last and past the bound of a row: their slots name no place whatever the buffer held, so
    the store writes the live tokens' keys and values and nothing else.  Their other values are left alone."""
    page, hkv, d, hq = 16, 2, 64, 4
    rng = np.random.default_rng(lead + sum(counts) + tail)
    bound = max(counts + [1]) if max_nodes is None else max_nodes
    live_counts = [min(n, bound) for n in counts]
    ctx = rng.integers(0, 50, len(counts)).tolist()
    table, pages = tables(ctx, live_counts, page, rng)
    starts = [lead + s for s in starts_of(counts)]
    T, first = starts[-1] + tail, pages
    pages += -(-T // page)                                        # a place of its own for every token of the earlier step
    stale = first * page + torch.arange(T, dtype=torch.int32)
    parents = torch.zeros(T, dtype=torch.int32)
    for b, n in enumerate(counts):
        parents[starts[b]:starts[b] + n] = random_parents([n], rng)
    out = stale_plan(ops, len(counts), T, bound, tree, stale)
    free = [p for b, c in enumerate(ctx) for p in table[b][-(-c // page):-(-(c + live_counts[b]) // page)]]
    ops.tree_plan(i32(ctx, DEV), i32(starts, DEV), i32(table, DEV), i32(free, DEV), bound, page, pages, parents=parents.to(DEV) if tree else None, out=out)
    live = {starts[b] + i: table[b][(c + i) // page] * page + (c + i) % page for b, c in enumerate(ctx) for i in range(live_counts[b])}
    got = out.slots.tolist()
    assert all(got[t] == s for t, s in live.items())
    assert all(got[t] < 0 for t in range(T) if t not in live)
    dead = torch.tensor([t not in live for t in range(T)])
    assert all((t[dead.to(DEV)] == 3).all() for t in (out.positions, out.rows, out.mask) if t is not None)

    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=g).to(BF16)
    k, v = (torch.randn(pages, page, hkv, d, generator=g).to(BF16) for _ in range(2))
    dk, dv = k.to(DEV), v.to(DEV)
    ops.qkv_norm_rotary_slots(qkv.to(DEV), out.positions, out.slots, dk, dv, hq)
    kv = qkv[:, hq * d:].view(T, 2, hkv, d)
    for t, s in live.items():
        k[s // page, s % page], v[s // page, s % page] = kv[t, 0], kv[t, 1]
    assert torch.equal(dk.cpu(), k) and torch.equal(dv.cpu(), v)


def test_a_step_without_rows_names_no_place(ops):
    out = stale_plan(ops, 0, 6, 8, True, torch.arange(6, dtype=torch.int32))
    none = i32([], DEV)
    ops.tree_plan(none, i32([0], DEV), torch.zeros(0, 4, dtype=torch.int32, device=DEV), none, 8, 16, 10, parents=torch.zeros(6, dtype=torch.int32, device=DEV),
                  out=out)
    assert (out.slots < 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_recorded_step_of_fewer_nodes_each_time(ops, dtype):
    """A step recorded for 40 tokens, replayed with fewer of them while the cached tokens grow over the places of the step before: each replay
    leaves the cache as its own nodes' keys and values make it."""
    rows, hq, hkv, d, page, T, bound, cols = 3, 4, 2, 64, 16, 40, 20, 8
    pages = rows * cols
    g = torch.Generator(device=DEV).manual_seed(2)
    rng = np.random.default_rng(2)
    table = [list(range(cols * b, cols * (b + 1))) for b in range(rows)]      # column j of row b is page 8 b + j, held or taken
    ctx, starts, bt, free = i32([0] * rows, DEV), i32([0] * (rows + 1), DEV), i32(table, DEV), i32([-1] * 6, DEV)
    parents = torch.zeros(T, dtype=torch.int32, device=DEV)
    qkv = torch.zeros(T, (hq + 2 * hkv) * d, dtype=dtype, device=DEV)
    k, v = (torch.zeros(pages, page, hkv, d, dtype=dtype, device=DEV) for _ in range(2))
    plan, q, o = ops.TreePlan.empty(rows, T, bound, DEV), torch.empty(T, hq, d, dtype=dtype, device=DEV), torch.zeros(T, hq, d, dtype=dtype, device=DEV)
    plan.slots.fill_(-1)

    def go():
        ops.tree_plan(ctx, starts, bt, free, bound, page, pages, parents=parents, out=plan)
        ops.qkv_norm_rotary_slots(qkv, plan.positions, plan.slots, k, v, hq, out=q)
        ops.tree_attn(q, k, v, ctx, starts, bt, plan.mask, bound, out=o)

    go()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    lens = [15, 0, 30]
    for counts in ([17, 20, 3], [9, 1, 11], [1, 0, 1], [0, 0, 0], [2, 16, 0]):
        at = starts_of(counts)
        take = [table[b][j] for b in range(rows) for j in range(-(-lens[b] // page), -(-(lens[b] + counts[b]) // page))]
        ctx.copy_(i32(lens, DEV))
        starts.copy_(i32(at, DEV))
        free.copy_(i32(take + [-1] * (6 - len(take)), DEV))
        parents[:at[-1]] = random_parents(counts, rng).to(DEV)
        qkv.normal_(generator=g)
        want_k, want_v, kv = k.clone(), v.clone(), qkv[:, hq * d:].view(T, 2, hkv, d)
        for b, (c, n) in enumerate(zip(lens, counts)):
            for i in range(n):
                p, s = table[b][(c + i) // page], (c + i) % page
                want_k[p, s], want_v[p, s] = kv[at[b] + i, 0], kv[at[b] + i, 1]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(s < 0 for s in plan.slots[at[-1]:].tolist()) and plan.taken.sum().item() == len(take)
        assert torch.equal(k, want_k) and torch.equal(v, want_v), counts
        lens = [c + (n + 1) // 2 for c, n in zip(lens, counts)]


# ------------------------------------------------------------------------------------------------------- rows without pages
@pytest.mark.parametrize("page", [1, 16, 64])
@pytest.mark.parametrize("tree", [True, False])
def test_a_refused_row_names_no_pages_behind_its_cached_tokens(ops, page, tree):
    """Columns that hold what earlier steps left: a row that gets pages has those, one that does not (none left, or no columns) has -1 where its nodes
    would lie, up to the table's end; columns behind the nodes and those of cached tokens stay."""
    ctx, counts, cols = [page, 3 * page, 2 * page, page, 6 * page], [2 * page, 2 * page, 0, 9 * page, page], 8
    old = [[100 * b + j for j in range(cols)] for b in range(5)]
    free = [301, 102, 7]
    for n_free in range(4):
        bt = i32(old, DEV)
        starts = starts_of(counts)
        parents = random_parents(counts, np.random.default_rng(page)) if tree and max(counts) <= 256 else None
        plan = ops.tree_plan(i32(ctx, DEV), i32(starts, DEV), bt, i32(free[:n_free], DEV), max(counts), page, 1000,
                             parents=None if parents is None else parents.to(DEV), tokens=starts[-1])
        slots, positions, _, _, taken, _ = ref.plan(ctx, starts, old, free[:n_free], page, 1000, parents)
        want = [list(r) for r in old]
        want[0][1:3] = free[:2] if n_free >= 2 else [-1, -1]
        want[1][3:5] = [-1, -1]
        want[3][1:8] = [-1] * 7                                    # wants ten columns
        want[4][6] = -1
        assert bt.tolist() == want and plan.taken.tolist() == taken == [2 if n_free >= 2 else -1, -1, 0, -1, -1]
        assert plan.slots.tolist() == slots and plan.positions.tolist() == positions


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_refused_row_reads_and_moves_nothing_of_other_rows(ops, dtype):
    """Row 1 is refused, and the pages its old columns name are row 0's nodes' now: its attention sees its cached tokens alone, and the acceptance leaves row
    0's nodes where row 0 has them."""
    page, hq, hkv, d, layers = 16, 4, 2, 64, 3
    g = torch.Generator().manual_seed(1)
    ctx, starts = [16, 32], [0, 20, 44]
    old = [[4, 0, 1, -1], [5, 6, 2, 3]]
    bt = i32(old, DEV)
    parents = torch.tensor([i - 1 for i in range(20)] + [-1, 0] + [i - 2 for i in range(2, 24)], dtype=torch.int32)
    plan = ops.tree_plan(i32(ctx, DEV), i32(starts, DEV), bt, i32([2, 3, 1], DEV), 24, page, 7, parents=parents.to(DEV))
    assert plan.taken.tolist() == [2, -1] and bt.tolist() == [[4, 2, 3, -1], [5, 6, -1, -1]]
    k, v = (torch.randn(layers, 7, page, hkv, d, generator=g).to(dtype).to(DEV) for _ in range(2))
    qkv = torch.randn(44, (hq + 2 * hkv) * d, generator=g).to(dtype).to(DEV)
    q = ops.qkv_norm_rotary_slots(qkv, plan.positions, plan.slots, k[0], v[0], hq)
    out = ops.tree_attn(q, k[0], v[0], i32(ctx, DEV), i32(starts, DEV), bt, plan.mask, 24)
    seen = [set(range(i + 1)) for i in range(20)] + [set() for _ in range(24)]
    o, mag, size, count = ref.attn(q.cpu(), k[0].cpu(), v[0].cpu(), ctx, starts, bt.tolist(), seen, d ** -0.5)
    assert ((out.double().cpu() - o).abs() <= ref.attn_bound(o, mag, size, count, d, dtype)).all()
    tokens = torch.arange(44, device=DEV)
    picks = torch.full((44,), -1, device=DEV)
    picks[20:44:2] = torch.arange(22, 46, 2, device=DEV)               # row 1: 0, 2, 4, ..: every node after the first would move
    picks[0] = 1
    before_k, before_v = k.clone(), v.clone()
    ops.tree_accept(tokens, picks, i32(starts, DEV), i32(ctx, DEV), 24, parents=parents.to(DEV), caches=ops.TreeCaches(k, v), block_table=bt)
    assert torch.equal(k, before_k) and torch.equal(v, before_v)


@pytest.mark.parametrize("layers", [0, 2, 70])
def test_acceptance_of_rows_that_got_no_pages(ops, layers):
    """A refused row has an empty path, its old length and nothing moved, in its own half-filled page neither; the rows beside it as without it."""
    ctx, counts, page, hkv, d = [20, 5, 30, 0], [12, 9, 40, 3], 16, 1, 16
    rng = np.random.default_rng(layers)
    starts = starts_of(counts)
    table, pages = tables(ctx, counts, page, rng)
    parents = torch.tensor([max(-1, i - 2) for n in counts for i in range(n)], dtype=torch.int32)
    tokens = torch.arange(starts[-1])
    picks = torch.cat([tokens[2:], torch.zeros(2, dtype=torch.int64)])             # node i's child is i + 2
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(max(1, layers), pages, page, hkv, d, generator=g).to(BF16) for _ in range(2))
    for taken in ([1, 0, 3, 1], [-1, 0, 3, 1], [1, -1, -1, 1], [-1, -1, -1, -1]):
        dk, dv = k.to(DEV), v.to(DEV)
        got = ops.tree_accept(tokens.to(DEV), picks.to(DEV), i32(starts, DEV), i32(ctx, DEV), 40, parents=parents.to(DEV),
                              caches=ops.TreeCaches(dk, dv) if layers else None, block_table=i32(table, DEV), taken=i32(taken, DEV))
        path, ids, n, lens = ref.accept(tokens.tolist(), picks.tolist(), starts, ctx, 40, parents)
        for b, t in enumerate(taken):
            if t < 0:
                path[b], ids[b], n[b], lens[b] = [-1] * 40, [-1] * 40, 0, ctx[b]
        assert n[3] == (2 if taken[3] >= 0 else 0)
        assert got.path.tolist() == path and got.ids.tolist() == ids and got.counts.tolist() == n and got.lens.tolist() == lens
        assert torch.equal(dk.cpu(), ref.move(k, ctx, table, path, n) if layers else k)
        assert torch.equal(dv.cpu(), ref.move(v, ctx, table, path, n) if layers else v)


def test_a_recorded_step_whose_row_is_refused_and_comes_again(ops):
    """Plan, store, attention and acceptance recorded once.  Replayed with no columns for the second row's nodes it keeps its length and the cache its content;
    replayed with some it goes on, and all of it is what the eager calls give."""
    page, hq, hkv, d, T, pages = 16, 4, 2, 64, 30, 12
    g = torch.Generator(device=DEV).manual_seed(4)
    starts, bt, free = i32([0, 12, 30], DEV), i32([[0, 3, 2], [1, 2, 3]], DEV), i32([-1, -1, -1, -1], DEV)
    ctx, parents = i32([10, 16], DEV), i32([max(-1, i - 2) for n in (12, 18) for i in range(n)], DEV)
    k, v = (torch.randn(1, pages, page, hkv, d, generator=g, device=DEV).to(BF16) for _ in range(2))
    tokens, qkv = torch.arange(T, device=DEV), torch.randn(T, (hq + 2 * hkv) * d, generator=g, device=DEV).to(BF16)
    picks = torch.cat([tokens[2:], tokens[:2] - 9])
    plan, got, caches = ops.TreePlan.empty(2, T, 18, DEV), ops.TreePath.empty(2, 18, DEV), ops.TreeCaches(k, v)
    q, o = torch.empty(T, hq, d, dtype=BF16, device=DEV), torch.empty(T, hq, d, dtype=BF16, device=DEV)

    def go():
        ops.tree_plan(ctx, starts, bt, free, 18, page, pages, parents=parents, out=plan)
        ops.qkv_norm_rotary_slots(qkv, plan.positions, plan.slots, k[0], v[0], hq, out=q)
        ops.tree_attn(q, k[0], v[0], ctx, starts, bt, plan.mask, 18, out=o)
        ops.tree_accept(tokens, picks, starts, ctx, 18, parents=parents, caches=caches, block_table=bt, out=got, taken=plan.taken)

    state = (bt, k, v)
    begin = [t.clone() for t in state]
    go()
    for t, b in zip(state, begin):
        t.copy_(b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for turn, cols in enumerate(([[0, 3, 2], [1, 2, 3]], [[0, 7, 2], [1, 8, 9]])):
        results = []
        for run in (graph.replay, go):
            for t, b in zip(state, begin):
                t.copy_(b)
            bt.copy_(i32(cols, DEV))
            free.copy_(i32([7, 8, 9, 10], DEV))
            ctx.copy_(i32([10, 16 if turn else 16 + 32], DEV))          # (a row without columns for its nodes, then the same row with them)
            torch.cuda.synchronize()
            run()
            torch.cuda.synchronize()
            results.append([t.clone() for t in (*plan, *got, bt, k, v)])
        assert all(torch.equal(a, b) for a, b in zip(*results)), turn
        assert plan.taken.tolist() == ([1, 2] if turn else [1, -1])
        assert got.counts.tolist() == ([6, 9] if turn else [6, 0]) and got.lens.tolist() == ([16, 25] if turn else [16, 48])
        if turn == 0:
            assert torch.equal(k[0, 1:7], begin[1][0, 1:7]) and torch.equal(k[0, 8:], begin[1][0, 8:])      # pages 0 and 7 are row 0's


def test_caches_that_layers_share_are_named_once(ops):
    """A path of 0, 2, 5 moved twice in one cache would leave node 5 where node 2 belongs: refused."""
    k, v = (torch.zeros(3, 4, 16, 2, 64, dtype=BF16, device=DEV) for _ in range(2))
    ops.TreeCaches(k, v)
    ops.TreeCaches([k[2], k[0]], [v[2], v[0]])
    flat = k.view(-1, 16, 2, 64)                                     # twelve pages: caches of four that overlap
    for a, b in (([k[0], k[0]], [v[0], v[1]]), ([k[0]], [k[0]]), ([k[0], k[1]], [v[0], k[0]]), ([flat[0:4], flat[2:6]], [v[0], v[1]])):
        with pytest.raises(AssertionError):
            ops.TreeCaches(a, b)
