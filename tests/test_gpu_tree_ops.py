"""The ops of a step that verifies drafted tokens (core/tree_decode.py), each against the 64-bit restatement in oracle/ref_tree.py, at the
sizes and masks where they can go wrong, and together with the one-token path they stand beside."""
import numpy as np
import pytest
import torch

from oracle import ref_tree as ref
from tree_util import AttnCase, i32, random_parents, starts_of, tables

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    import micro_vllm_amd  # noqa: F401
    from micro_vllm_amd.core import tree_decode
    return tree_decode


# ---------------------------------------------------------------------------------------------------------------- plan
def run_plan(ops, ctx, counts, page, parents, free, table, pages, tail=2, max_nodes=None, with_mask=None, stride_extra=0):
    starts = starts_of(counts)
    T = starts[-1]
    max_nodes = max(counts + [1]) if max_nodes is None else max_nodes
    cols = len(table[0]) if table else 1
    buf = torch.full((max(1, len(ctx)), cols + stride_extra), -77, dtype=torch.int32, device=DEV)
    bt = buf[:len(ctx), :cols]
    if ctx:
        bt.copy_(torch.tensor(table, dtype=torch.int32))
    with_mask = parents is not None if with_mask is None else with_mask
    out = ops.TreePlan.empty(len(ctx), T + tail, max_nodes, DEV, mask=with_mask)
    for t in out:
        if t is not None:
            t.fill_(-5)
    par = None if parents is None else torch.cat([parents, torch.zeros(tail, dtype=torch.int32)]).to(DEV)
    ops.tree_plan(i32(ctx, DEV), i32(starts, DEV), bt, i32(free, DEV), max_nodes, page, pages, parents=par, out=out)
    slots, positions, rows, seen, taken, want_table = ref.plan(ctx, starts, table, free, page, pages, parents)
    assert out.slots[:T].tolist() == slots
    assert out.positions[:T].tolist() == positions
    assert out.rows[:T].tolist() == rows
    assert out.taken.tolist() == taken
    assert bt.tolist() == want_table
    if with_mask:
        assert torch.equal(out.mask[:T].cpu(), ref.mask_words(seen, out.mask.shape[1]))
        assert (out.mask[T:] == -5).all()
    for t in (out.slots, out.positions, out.rows):      # tokens behind the last row
        assert (t[T:] == -5).all()
    if stride_extra:
        assert (buf[:, cols:] == -77).all()


def split_pool(ctx, counts, page, rng):
    """(table with the pages of cached tokens only, free pages in some order, pages)."""
    table, pages = tables(ctx, counts, page, rng)
    free = []
    for b, c in enumerate(ctx):
        held = -(-c // page)
        free += [p for p in table[b][held:] if p >= 0]
        table[b][held:] = [-1] * (len(table[b]) - held)
    return table, [free[i] for i in rng.permutation(len(free))], pages


@pytest.mark.parametrize("page", [1, 16, 48, 64, 256])
@pytest.mark.parametrize("counts,ctx", [
    ([1], [0]), ([1], [255]), ([7], [45]), ([64], [0]), ([65, 3], [10, 64]), ([256, 1, 0, 200], [63, 256, 17, 0]),
    ([0, 0], [0, 5]), ([5, 0, 64, 33, 17], [100, 7, 64, 15, 0])])
def test_plan_of_trees(ops, page, counts, ctx):
    rng = np.random.default_rng(page * 31 + sum(counts))
    table, free, pages = split_pool(ctx, counts, page, rng)
    parents = random_parents(counts, rng, forest=True)
    run_plan(ops, ctx, counts, page, parents, free, table, pages)


@pytest.mark.parametrize("rows", [3, 65, 300, 1100])
def test_plan_of_many_rows_and_a_strided_table(ops, rows):
    rng = np.random.default_rng(rows)
    counts, ctx = rng.integers(0, 9, rows).tolist(), rng.integers(0, 70, rows).tolist()
    table, free, pages = split_pool(ctx, counts, 16, rng)
    run_plan(ops, ctx, counts, 16, random_parents(counts, rng), free, table, pages, stride_extra=3)


def test_plan_of_chains_portions_and_odd_parents(ops):
    rng = np.random.default_rng(5)
    counts, ctx = [5000, 1, 700, 0, 257], [3, 0, 1000, 9, 255]
    table, free, pages = split_pool(ctx, counts, 64, rng)
    run_plan(ops, ctx, counts, 64, None, free, table, pages)                        # portions of prompts: no limit on their length
    counts = [200, 1, 64, 0]
    table, free, pages = split_pool(ctx[:4], counts, 64, rng)
    run_plan(ops, ctx[:4], counts, 64, None, free, table, pages, with_mask=True)      # a chain's mask
    # parents that are no earlier node: themselves, later ones, far out of range
    odd = torch.tensor([0, 0, 5, -9, 2 ** 31 - 1, 3, -2 ** 31, 6], dtype=torch.int32)
    table, free, pages = split_pool([20], [8], 16, rng)
    run_plan(ops, [20], [8], 16, odd, free, table, pages)


def test_plan_gives_rows_their_pages_first_come(ops):
    """Free pages that do not last: the row that finds too few and every later row that needs any get none, rows that need none
    are served; a table without columns for a row refuses it and takes nothing; pages outside the pool have no slots."""
    page, ctx, counts = 16, [16, 30, 5, 64, 0], [20, 10, 3, 1, 1]          # needs 2, 1, 0, 1, 1
    table = [[3, -1, -1, -1, -1], [5, 6, -1, -1, -1], [7, -1, -1, -1, -1], [1, 2, 8, 9, -1], [-1, -1, -1, -1, -1]]
    parents = random_parents(counts, np.random.default_rng(1))
    for free in ([], [20], [20, 21], [20, 21, 22], [20, 21, 22, 23], [20, 21, 22, 23, 24, 25]):
        run_plan(ops, ctx, counts, page, parents, free, table, 40)
    narrow = [r[:3] for r in table]
    narrow[3] = [1, 2, 8]                                                  # holds fewer than its cached tokens even
    run_plan(ops, ctx, counts, page, parents, [20, 21, 22, 23], narrow, 40)
    run_plan(ops, ctx, counts, page, parents, [-1, 500, 22, 23, 24], [[-4, -1, -1, -1, -1]] + table[1:], 40)


# --------------------------------------------------------------------------------------------------- norm, rotation, store
def rotary_freqs(half, base=10000.0):
    return torch.tensor([base ** (-i / half) for i in range(half)], dtype=torch.float64)


@pytest.mark.parametrize("src,dst", [(BF16, BF16), (F32, BF16), (F32, F32)])
@pytest.mark.parametrize("hq,hkv,d,rot,adjacent", [
    (32, 8, 128, 128, False), (32, 4, 64, 64, True), (4, 4, 64, 32, False), (5, 1, 128, 48, True), (3, 3, 80, 80, False),
    (6, 2, 96, 0, False), (7, 7, 20, 6, False), (1, 1, 256, 256, False), (2, 2, 33, 32, True), (9, 3, 512, 128, False)])
def test_norm_rotary_slots(ops, src, dst, hq, hkv, d, rot, adjacent):
    g = torch.Generator().manual_seed(hq * d + rot)
    for T, far in ((1, 5), (37, 4000), (300, 2 ** 31 - 1)):
        page, pages = 16, 40
        wide = torch.randn(T, (hq + 2 * hkv) * d + 24, generator=g).to(src) * 3
        wide[0, :d] = 0                                           # a head of zeros: eps alone under the root
        qkv = wide[:, 8:8 + (hq + 2 * hkv) * d]
        positions = torch.randint(0, far, (T,), generator=g, dtype=torch.int64).to(torch.int32)
        positions[-1] = far
        slots = torch.randperm(pages * page, generator=g)[:T].to(torch.int32)
        if T > 1:
            slots[1], slots[T // 2], slots[T - 2] = -1, pages * page, 2 ** 31 - 1
        qn, kn = (1 + 0.3 * torch.randn(d, generator=g) for _ in range(2))
        freqs = rotary_freqs(rot // 2) if rot else None
        kc, vc = (torch.randn(pages, page, hkv, d, generator=g).to(dst) for _ in range(2))
        for q_norm, k_norm in ((qn, kn), (None, kn), (None, None)):
            dk, dv = kc.to(DEV), vc.to(DEV)
            out = torch.full((T, hq * d + 8), 7.0, dtype=dst, device=DEV)
            dw = wide.to(DEV)
            ops.qkv_norm_rotary_slots(dw[:, 8:8 + (hq + 2 * hkv) * d], positions.to(DEV), slots.to(DEV), dk, dv, hq,
                                      None if q_norm is None else q_norm.to(DEV), None if k_norm is None else k_norm.to(DEV), 1e-5,
                                      None if freqs is None else freqs.to(DEV), adjacent, out=out[:, :hq * d].unflatten(1, (hq, d)))
            q, k, v, mq, mk = ref.norm_rotary(qkv, hq, hkv, d, positions, q_norm, k_norm, 1e-5, freqs, adjacent)
            # fp32: the mean of d squares (d / 2 + 4 half steps relatively), root, division and weight, sine and cosine (2^-22), two
            # products and a sum; the angle in fp64 (2^-51 of it, an absolute error of sine and cosine); then the output's rounding
            half = torch.finfo(dst).eps / 2
            rel = (d / 2 + 32) * 2.0 ** -24 + far * 2.0 ** -50
            for got, want, mag in ((out[:, :hq * d].view(T, hq, d), q, mq),):
                assert ((got.double().cpu() - want).abs() <= half * want.abs() + 1.01 * rel * mag + 1e-37).all()
            assert (out[:, hq * d:] == 7.0).all()
            live = [(t, int(s)) for t, s in enumerate(slots.tolist()) if 0 <= s < pages * page]
            want_k, want_v = kc.double().view(-1, hkv, d).clone(), vc.double().view(-1, hkv, d).clone()
            tol = torch.zeros_like(want_k)
            for t, s in live:
                want_k[s], want_v[s] = k[t], v[t].to(dst).double()
                tol[s] = half * k[t].abs() + 1.01 * rel * mk[t] + 1e-37
            assert ((dk.double().cpu().view(-1, hkv, d) - want_k).abs() <= tol).all()
            assert torch.equal(dv.double().cpu().view(-1, hkv, d), want_v)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d,rot,adjacent", [(128, 128, False), (64, 32, False), (64, 64, True), (80, 80, False)])
def test_norm_rotary_slots_in_place(ops, dtype, d, rot, adjacent):
    """q written over its own part of the rows: the same values as beside them; k and v of the rows stay."""
    g = torch.Generator(device=DEV).manual_seed(3)
    hq, hkv, T = 6, 2, 50
    qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=g, device=DEV).to(dtype)
    pos, slots = torch.arange(T, dtype=torch.int32, device=DEV) + 1000, torch.arange(T, dtype=torch.int32, device=DEV)
    w, freqs = torch.rand(d, generator=g, device=DEV) + 0.5, rotary_freqs(rot // 2).to(DEV)
    caches = [torch.zeros(4, 16, hkv, d, dtype=dtype, device=DEV) for _ in range(4)]
    beside = ops.qkv_norm_rotary_slots(qkv, pos, slots, caches[0], caches[1], hq, w, w, 1e-6, freqs, adjacent)
    over = qkv.clone()
    ops.qkv_norm_rotary_slots(over, pos, slots, caches[2], caches[3], hq, w, w, 1e-6, freqs, adjacent,
                              out=over[:, :hq * d].unflatten(1, (hq, d)))
    assert torch.equal(over[:, :hq * d].reshape(T, hq, d), beside) and torch.equal(over[:, hq * d:], qkv[:, hq * d:])
    assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("off,extra,out_off", [(1, 0, 0), (8, 1, 0), (0, 0, 3), (4, 4, 0)])
def test_norm_rotary_slots_of_rows_that_are_not_aligned(ops, dtype, off, extra, out_off):
    """Rows, strides and outputs off the 16-byte grid: the values of rows on it, up to a sum's order."""
    g = torch.Generator(device=DEV).manual_seed(9)
    hq, hkv, d, T = 5, 2, 128, 21
    width = (hq + 2 * hkv) * d
    buf = torch.randn(T, width + off + extra, generator=g, device=DEV).to(dtype)
    pos, slots = torch.arange(T, dtype=torch.int32, device=DEV) * 7, torch.arange(T, dtype=torch.int32, device=DEV)
    w, freqs = torch.rand(d, generator=g, device=DEV) + 0.5, rotary_freqs(d // 2).to(DEV)
    caches = [torch.zeros(2, 16, hkv, d, dtype=dtype, device=DEV) for _ in range(2)]
    out = torch.zeros(T, hq * d + 8, dtype=dtype, device=DEV)[:, out_off:out_off + hq * d].unflatten(1, (hq, d))
    ops.qkv_norm_rotary_slots(buf[:, off:off + width], pos, slots, *caches, hq, w, w, 1e-6, freqs, out=out)
    q, k, v, mq, mk = ref.norm_rotary(buf[:, off:off + width].cpu(), hq, hkv, d, pos.cpu(), w.cpu(), w.cpu(), 1e-6, freqs.cpu(), False)
    half, rel = torch.finfo(dtype).eps / 2, (d / 2 + 32) * 2.0 ** -24 + 140 * 2.0 ** -50       # (as in test_norm_rotary_slots)
    assert ((out.double().cpu() - q).abs() <= half * q.abs() + 1.01 * rel * mq).all()
    got = [c.view(-1, hkv, d)[:T].double().cpu() for c in caches]
    assert ((got[0] - k).abs() <= half * k.abs() + 1.01 * rel * mk).all() and torch.equal(got[1], v.to(dtype).double())


# ------------------------------------------------------------------------------------------------------------- attention
# Which kernel a launch takes goes by its rows and by the keys that its table has room for: behind this many columns more every launch takes the form
# for much work (bf16: 16, 32 or (heads of 64) 64 stacked rows a workgroup, past 64 (heads of 128: 32) keys shared by the waves; fp32: 32 rows).
MUCH = 26000


def run_attn(ops, case, splits=0, mask="case", max_nodes=None, hq_stride=0, cols=0):
    T, hq, d = case.q.shape
    buf = torch.full((T, hq * d + hq_stride), 7.0, dtype=case.dtype, device=DEV)
    out = buf[:, :hq * d].unflatten(1, (hq, d))
    if hq_stride:
        qb = torch.zeros(T, hq * d + hq_stride, dtype=case.dtype, device=DEV)
        qb[:, :hq * d] = case.q.reshape(T, hq * d).to(DEV)
        q = qb[:, :hq * d].unflatten(1, (hq, d))
    else:
        q = case.q.to(DEV)
    m = None if mask is None else case.mask().to(DEV)
    table = torch.nn.functional.pad(i32(case.table, DEV), (0, cols), value=-1)
    ops.tree_attn(q, case.k.to(DEV), case.v.to(DEV), i32(case.ctx, DEV), i32(case.starts, DEV), table, m, max_nodes or case.max_nodes, out=out,
                  num_splits=splits)
    assert (out[case.T:] == 7.0).all(), "tokens behind the last row"
    assert hq_stride == 0 or (buf[:, hq * d:] == 7.0).all()
    return out


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hkv,d,page", [(8, 2, 128, 64), (4, 4, 64, 16), (7, 1, 128, 256), (16, 2, 64, 64), (3, 1, 64, 32), (1, 1, 128, 16)])
@pytest.mark.parametrize("ctx,counts", [
    ([0], [1]), ([45], [7]), ([1, 16, 63, 64, 65], [1, 2, 17, 64, 3]), ([300, 0, 129, 1000], [64, 33, 0, 20]), ([500, 31], [65, 130])])
def test_attention_of_trees(ops, dtype, hq, hkv, d, page, ctx, counts):
    case = AttnCase(ctx, counts, hq, hkv, d, page, dtype, seed=hq * 1000 + d + page + sum(ctx), forest=True)
    want = case.reference()
    for splits in (0, 1, 3, 64):
        for cols in (0, MUCH):
            case.check(run_attn(ops, case, splits, cols=cols), f"splits {splits} columns {cols}", want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_of_the_largest_trees(ops, dtype):
    case = AttnCase([200, 3], [256, 250], 8, 1, 128 if dtype == BF16 else 64, 64, dtype, seed=9)
    want = case.reference()
    for splits in (0, 1, 2):
        for cols in (0, MUCH):
            case.check(run_attn(ops, case, splits, cols=cols), f"splits {splits} columns {cols}", want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq", [2, 4, 12])
def test_attention_of_a_chain_is_the_causal_one(ops, dtype, d, hq):
    case = AttnCase([100, 0, 37], [30, 64, 1], hq, 2, d, 16, dtype, seed=2)
    case.seen = [set(range(i + 1)) for n in case.counts for i in range(n)]
    want = case.reference()
    for cols in (0, MUCH):
        a, b = run_attn(ops, case, mask=None, cols=cols), run_attn(ops, case, cols=cols)
        assert torch.equal(a, b)
        case.check(a, "chain", want)


@pytest.mark.parametrize("hq,n,d", [(8, 8, 128), (8, 17, 128), (8, 17, 64), (8, 2, 64), (8, 4, 64), (8, 8, 64), (8, 4, 128)])
@pytest.mark.parametrize("ctx", [700, 1500, 3136])
def test_splits_that_keys_do_not_fill(ops, hq, n, d, ctx):
    """Numbers of splits that leave the last of them short, or without any key, and masks with bits of nodes that a row does not have."""
    case = AttnCase([ctx - n, 40], [n, 1], hq, 1, d, 64, BF16, seed=ctx + n)
    want, seen = case.reference(), case.seen
    case.seen = [s | set(range(n if t < n else 1, 64)) for t, s in enumerate(seen)]
    for splits in (2, 3, 4, 7, 8, 30):
        for cols in (0, MUCH):
            case.check(run_attn(ops, case, splits, cols=cols), f"splits {splits} columns {cols}", want)


@pytest.mark.parametrize("hq,n,d", [(8, 17, 64), (8, 17, 128), (8, 8, 128), (2, 3, 128), (8, 8, 64)])
@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_thousands_of_keys_in_one_piece(ops, hq, n, d, page, dtype):
    """More keys than the page numbers that a wave holds at a time (64 tiles of 64), with holes in the table on either side, and non-finite values there."""
    case = AttnCase([8500, 4100], [n, 2], hq, 1, d, page, dtype, seed=page + n)
    for key in (4090, 4200, 8300):
        case.table[0][key // page] = -1
    used = {p for row in case.table for p in row}
    for p in set(range(case.pages)) - used:
        case.v[p], case.k[p] = float("nan"), float("inf")
    want = case.reference()
    for splits in (1, 2, 0):
        case.check(run_attn(ops, case, splits, cols=MUCH), f"splits {splits}", want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_of_many_rows(ops, dtype):
    """More rows than a wave has lanes, more than the joining launch has workgroups for one each; some without nodes."""
    rng = np.random.default_rng(4)
    ctx, counts = rng.integers(0, 40, 700).tolist(), rng.integers(0, 3, 700).tolist()
    ctx[300], counts[300] = 2000, 5
    case = AttnCase(ctx, counts, 2, 1, 64, 16, dtype, seed=4)
    want = case.reference()
    for splits in (0, 1, 4):
        for cols in (0, MUCH):
            case.check(run_attn(ops, case, splits, cols=cols), f"splits {splits} columns {cols}", want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d,page", [(64, 16), (64, 64), (128, 64)])
def test_rows_of_up_to_32_heads_and_nodes_in_a_full_launch(ops, dtype, d, page):
    """Workgroups for half the chip and more with short rows (bf16, heads of 64: eight waves on 32 stacked rows); holes in the table, a node whose key and value are not
    finite."""
    rng = np.random.default_rng(page + d)
    ctx, counts = rng.integers(0, 700, 70).tolist(), rng.integers(0, 9, 70).tolist()
    counts[0], counts[5] = 8, 8
    case = AttnCase(ctx, counts, 8, 2, d, page, dtype, seed=page + d, forest=True)
    for b in (3, 9, 40):
        case.table[b][0] = -1
    t = case.starts[5]
    case.seen = [s - {2} if t <= i < t + 8 else s for i, s in enumerate(case.seen)]
    p, s = case.table[5][(ctx[5] + 2) // page], (ctx[5] + 2) % page
    case.k[p, s], case.v[p, s] = float("nan"), float("inf")
    want = case.reference()
    for splits in (0, 1, 2, 5):
        case.check(run_attn(ops, case, splits), f"splits {splits}", want)


@pytest.mark.parametrize("page", [16, 64])
def test_64_heads_and_nodes_in_one_workgroup_a_unit(ops, page):
    """26 rows on eight key/value heads of 128: workgroups of 64 stacked rows for most of the chip and no more than it has; rows that rise, a hole, a value
    that is not finite."""
    rng = np.random.default_rng(page)
    ctx, counts = rng.integers(0, 300, 26).tolist(), rng.integers(0, 17, 26).tolist()
    counts[0], ctx[7], counts[7] = 16, 900, 12
    case = AttnCase(ctx, counts, 32, 8, 128, page, BF16, seed=page, forest=True)
    case.table[3][0] = -1
    t = case.starts[7]
    case.seen = [s - {2} if t <= i < t + 12 else s for i, s in enumerate(case.seen)]
    p, s = case.table[7][902 // page], 902 % page
    case.k[p, s], case.v[p, s] = float("nan"), float("inf")
    case.q[t + 5] *= 40                                    # scores of hundreds: the second pass
    want = case.reference()
    for splits in (0, 1, 2):
        case.check(run_attn(ops, case, splits), f"splits {splits}", want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,d", [(1, 64), (2, 128), (8, 64), (8, 128)])
@pytest.mark.parametrize("cols", [0, MUCH])
def test_a_query_that_is_not_finite_is_its_own(ops, dtype, hq, d, cols):
    """NaN in one head of one node: NaN there, every other head and node as without it; a mask of more words than the nodes need."""
    case = AttnCase([200], [30], hq, 1, d, 16, dtype, seed=17)
    case.words = 4
    want = case.reference()
    case.q[11, hq - 1, 7] = float("nan")
    keep = torch.ones(30, hq, dtype=torch.bool)
    keep[11, hq - 1] = False
    for splits in (1, 3):
        out = run_attn(ops, case, splits, cols=cols)[:30].double().cpu()
        o, mag, size, count = want
        assert out[11, hq - 1].isnan().all() and ((out - o).abs() <= ref.attn_bound(o, mag, size, count, d, dtype))[keep].all()


def test_threads_with_streams_of_their_own(ops):
    """Four threads, a stream each, rows cut into splits: everyone's workspace is their own."""
    import threading
    cases = [AttnCase([900 + 40 * i, 30], [20, 7 + i], 8, 2, 64, 64, BF16, seed=30 + i) for i in range(4)]
    alone = [run_attn(ops, c, 6) for c in cases]
    torch.cuda.synchronize()
    got, wrong = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = run_attn(ops, cases[i], 6)
                torch.cuda.current_stream().synchronize()
        except Exception as e:      # (an assertion of a thread is the test's)
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and all(torch.equal(a, b) for a, b in zip(alone, got))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_nodes_past_the_bound_are_left_alone(ops, dtype):
    case = AttnCase([50, 20], [40, 6], 4, 1, 64, 16, dtype, seed=15)
    want = [t.clone() for t in case.reference()]
    for cols in (0, MUCH):
        for splits in (1, 2):
            out = run_attn(ops, case, splits, max_nodes=10, cols=cols)
            assert (out[10:40] == 7.0).all()
            keep = torch.ones(case.T, dtype=torch.bool)
            keep[10:40] = False
            o, mag, size, count = (t[keep] for t in want)
            err = (out[:case.T].double().cpu()[keep] - o).abs()
            assert (err <= ref.attn_bound(o, mag, size, count, 64, dtype)).all()
    plan = ops.TreePlan.empty(2, case.T, 10, DEV)
    for t in plan:
        t.fill_(-5)
    ops.tree_plan(i32(case.ctx, DEV), i32(case.starts, DEV), i32(case.table, DEV), i32(list(range(90)), DEV), 10, 16, 100, parents=case.parents.to(DEV),
                  out=plan)
    assert all((t[10:40] == -5).all() and (t[:10] != -5).all() and (t[40:] != -5).all() for t in (plan.slots, plan.positions, plan.rows))
    assert (plan.mask[10:40] == -5).all() and plan.taken.tolist() == [0, 0]
    tokens = torch.zeros(case.T, dtype=torch.int64, device=DEV)
    got = ops.tree_accept(tokens, tokens, i32(case.starts, DEV), i32(case.ctx, DEV), 10)
    assert got.counts.tolist() == [10, 6] and got.lens.tolist() == [60, 26]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [64, 128])
def test_masks_that_are_no_trees(ops, dtype, d):
    """Any bits: a node that does not see itself, one that sees a later node, nodes that see nothing (zeros, where nothing is cached)."""
    rng = np.random.default_rng(8)
    case = AttnCase([0, 70, 0], [40, 70, 1], 6, 2, d, 16, dtype, seed=4)
    for b, n in enumerate(case.counts):
        for i in range(n):
            case.seen[case.starts[b] + i] = set(np.nonzero(rng.random(n) < 0.3)[0].tolist())
    case.seen[5], case.seen[case.starts[1] + 3], case.seen[case.starts[2]] = set(), set(), set()
    want = case.reference()
    for splits in (0, 1, 5):
        for cols in (0, MUCH):
            out = run_attn(ops, case, splits, hq_stride=16, cols=cols)
            case.check(out, f"splits {splits} columns {cols}", want)
            assert (out[5] == 0).all() and (out[case.starts[2]] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d,hq,hkv", [(128, 4, 1), (64, 4, 4), (128, 16, 2), (64, 8, 1), (128, 1, 1), (64, 2, 1)])
@pytest.mark.parametrize("cols", [0, MUCH])
def test_what_is_masked_may_be_infinite_or_nan(ops, dtype, d, hq, hkv, cols):
    """Keys and values of nodes that are not seen, of places behind the last node and of pages that are nobody's hold NaN and infinities:
    nodes that see none of it get what they get without it; those that see an infinite value get it in that entry alone."""
    for n, ctx in ((20, 37), (64, 64), (33, 0)):
        case = AttnCase([ctx], [n], hq, hkv, d, 16, dtype, seed=n)
        bad = {i for i in range(n) if i % 3 == 1}
        where = lambda i: (case.table[0][(ctx + i) // 16], (ctx + i) % 16)      # noqa: E731
        case.seen = [s - bad | ({i} if i not in bad else set()) for i, s in enumerate(case.seen)]
        used = {p for p in case.table[0] if p >= 0}
        for p in range(case.pages):
            if p not in used:
                case.k[p], case.v[p] = float("nan"), float("nan")
        for at in range(ctx + n, len(used) * 16):
            p, s = case.table[0][at // 16], at % 16
            case.k[p, s], case.v[p, s] = float("nan"), float("inf")
        clean = case.reference()
        for i in bad:
            p, s = where(i)
            case.k[p, s], case.v[p, s] = [float("inf"), float("nan"), -float("inf")][i % 3], [float("nan"), float("inf")][i % 2]
        for splits in (0, 1, 2):
            out = run_attn(ops, case, splits, cols=cols)
            case.check(out, f"n {n} splits {splits}", clean)
        # one finite key with one infinite entry of its value: nodes that see it get the infinity there and nothing else changes
        p, s = where(2)
        case.v[p, s, :, 5] = float("inf")
        case.v[p, s, :, d - 1] = -float("inf")
        out = run_attn(ops, case, cols=cols).double().cpu()[:n]
        sees = torch.tensor([2 in z for z in case.seen])
        assert (out[sees][:, :, 5] == float("inf")).all() and (out[sees][:, :, d - 1] == -float("inf")).all()
        keep = torch.ones(d, dtype=torch.bool)
        keep[5] = keep[d - 1] = False
        o, mag, size, count = clean
        bound = ref.attn_bound(o, mag, size, count, d, dtype)
        assert ((out - o).abs() <= bound)[~sees].all() and ((out - o).abs() <= bound)[:, :, keep].all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (2, 2, 64), (8, 1, 64), (3, 3, 128), (4, 4, 128), (2, 1, 128), (8, 1, 128)])
@pytest.mark.parametrize("cols", [0, MUCH])
def test_places_without_a_page_do_not_count(ops, dtype, hq, hkv, d, cols):
    case = AttnCase([100, 90, 40], [20, 40, 8], hq, hkv, d, 16, dtype, seed=6)
    case.table[0][2] = -1                                  # among the cached tokens
    case.table[1][(90 + 16) // 16] = case.pages + 5         # among the nodes
    case.table[2] = [-1] * len(case.table[2])               # a row without any page: zeros
    want = case.reference()
    for splits in (0, 1, 4):
        out = run_attn(ops, case, splits, cols=cols)
        case.check(out, f"splits {splits}", want)
        assert (out[case.starts[2]:case.T] == 0).all()
    narrow = AttnCase([100], [20], hq, hkv, d, 16, dtype, seed=6)
    narrow.table = [narrow.table[0][:7]]                    # no column for the last nodes: their keys do not count
    narrow.check(run_attn(ops, narrow, cols=cols), "narrow table")


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scores_of_any_size(ops, dtype):
    """Scores of hundreds on either side of zero, and one key that outweighs all others wherever it lies."""
    for hq, hkv, d in ((4, 2, 64), (8, 1, 64), (2, 1, 128), (8, 1, 128)):
        case = AttnCase([130], [24], hq, hkv, d, 64, dtype, seed=11, scale_q=30.0)
        want = case.reference()
        for cols in (0, MUCH):
            case.check(run_attn(ops, case, cols=cols), f"large scores, columns {cols}", want)
        for at in (0, 15, 16, 63, 64, 129, 131):
            case = AttnCase([130], [24], hq, hkv, d, 64, dtype, seed=12)
            p, s = case.table[0][at // 64], at % 64
            case.k[p, s] = case.q[5, ::hq // hkv].to(F32).to(dtype) * 4
            want = case.reference()
            for splits in (1, 3):
                for cols in (0, MUCH):
                    case.check(run_attn(ops, case, splits, cols=cols), f"key {at} columns {cols}", want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq", [1, 2, 8])
@pytest.mark.parametrize("d", [64, 128])
def test_scores_of_minus_two_million(ops, dtype, hq, d):
    """Every key that a row sees has a score of -2^21, -2^22 or -2^23 (products of powers of two, exact in any order): those of -2^21 share the weight."""
    case = AttnCase([90], [24], hq, 1, d, 16, dtype, seed=16)
    case.q.zero_()
    case.q[:, :, 3] = 2.0 ** 10
    case.k.zero_()
    for j in range(114):
        case.k[case.table[0][j // 16], j % 16, :, 3] = -(2.0 ** (12 + j % 3))
    want = torch.zeros(24, hq, d, dtype=torch.float64)
    for t in range(24):
        best = [j for j in range(0, 114, 3) if j < 90 or j - 90 in case.seen[t]]
        want[t] = torch.stack([case.v[case.table[0][j // 16], j % 16, 0].double() for j in best]).mean(0)
    # equal weights: sums of up to 38 values and of as many weights, a division, a rounding of each; bf16: the weight's rounding and the output's
    tol = (100 * 2.0 ** -24 + (2.02 * 2.0 ** -8 if dtype == BF16 else 0)) * case.v.abs().max().item()
    for splits in (1, 3):
        for cols in (0, MUCH):
            table = torch.nn.functional.pad(i32(case.table, DEV), (0, cols), value=-1)
            out = ops.tree_attn(case.q.to(DEV), case.k.to(DEV), case.v.to(DEV), i32(case.ctx, DEV), i32(case.starts, DEV), table, case.mask().to(DEV), 24,
                                softmax_scale=0.5, num_splits=splits)
            assert ((out[:24].double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 2), (8, 1)])
@pytest.mark.parametrize("step", [-1.0, 1.0])
def test_scores_that_rise_or_fall_along_the_keys(ops, d, hq, hkv, step):
    """Scores that climb (fall) by one per key, over hundreds: no key of the first block says anything about the last ones', and nothing before
    them has a weight left.  The second half of the keys is out of reach of the first by more than fp32's range."""
    case = AttnCase([700, 0, 90], [20, 30, 24], hq, hkv, d, 64, BF16, seed=13)
    case.q.zero_()
    case.q[:, :, 0], case.q[:, :, 1] = d ** 0.5, 1.0
    for b, (c, n) in enumerate(zip(case.ctx, case.counts)):
        for j in range(c + n):
            p, s = case.table[b][j // 64], j % 64
            case.k[p, s, :, 0] = step * j
    want = case.reference()
    for splits in (0, 1, 2):
        for cols in (0, MUCH):
            case.check(run_attn(ops, case, splits, cols=cols), f"splits {splits} columns {cols}", want)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq", [1, 2, 8])
@pytest.mark.parametrize("cols", [0, MUCH])
def test_values_near_the_end_of_the_range(ops, d, hq, cols):
    """Values of 2^100 and scores 30 above those of the first keys: no sum may overflow on the way."""
    case = AttnCase([400], [24], hq, 1, d, 64, BF16, seed=14)
    case.v.mul_(2.0 ** 100)
    for j in (200, 390, 405):
        p, s = case.table[0][j // 64], j % 64
        case.k[p, s] = case.q[7, ::hq].to(F32).to(BF16) * 4
    want = case.reference()
    for splits in (0, 1, 2):
        out = run_attn(ops, case, splits, cols=cols)
        assert torch.isfinite(out[:case.T].float()).all()
        case.check(out, f"splits {splits}", want)


def test_a_long_cache_past_32_bit_offsets(ops):
    """Pages whose first value lies past 2^31 (and 2^32 bytes) from the pool's: 16 GiB of cache for two rows."""
    hkv, d, page = 8, 128, 64
    pages = (1 << 33) // (page * hkv * d * 2) + 8
    k = torch.zeros(pages, page, hkv, d, dtype=BF16, device=DEV)
    v = torch.zeros(pages, page, hkv, d, dtype=BF16, device=DEV)
    small = AttnCase([200, 70], [9, 40], 16, hkv, d, page, BF16, seed=3)
    far = [pages - 1 - i if i % 2 else pages // 2 + i for i in range(small.pages)]
    for i, p in enumerate(far):
        k[p], v[p] = small.k[i].to(DEV), small.v[i].to(DEV)
    table = [[far[p] if p >= 0 else -1 for p in row] for row in small.table]
    out = ops.tree_attn(small.q.to(DEV), k, v, i32(small.ctx, DEV), i32(small.starts, DEV), i32(table, DEV), small.mask().to(DEV), small.max_nodes)
    assert torch.equal(out[:small.T], run_attn(ops, small)[:small.T])
    small.check(out, "far pages")


def test_store_and_accept_past_32_bit_offsets(ops):
    """Slots whose first value lies past 2^32 bytes from the pool's: stored there, and moved there."""
    hkv, d, page, hq = 8, 128, 64, 8
    pages = (1 << 32) // (page * hkv * d * 2) + 4
    k = torch.zeros(pages, page, hkv, d, dtype=BF16, device=DEV)
    v = torch.zeros(pages, page, hkv, d, dtype=BF16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(6)
    qkv = torch.randn(6, (hq + 2 * hkv) * d, generator=g, device=DEV).to(BF16)
    table = i32([[pages - 1, pages - 2]], DEV)
    starts, ctx = i32([0, 6], DEV), i32([61], DEV)
    plan = ops.tree_plan(ctx, starts, table, i32([pages - 2], DEV), 6, page, pages, parents=i32([-1, 0, 0, 2, 3, 4], DEV))
    assert plan.slots.tolist() == [(pages - 1) * page + 61 + i for i in range(3)] + [(pages - 2) * page + i for i in range(3)]
    ops.qkv_norm_rotary_slots(qkv, plan.positions, plan.slots, k, v, hq)
    kv = qkv[:, hq * d:].view(6, 2, hkv, d)
    where = [(pages - 1, 61 + i) for i in range(3)] + [(pages - 2, i) for i in range(3)]
    assert all(torch.equal(k[p, s], kv[i, 0]) and torch.equal(v[p, s], kv[i, 1]) for i, (p, s) in enumerate(where))
    tokens = torch.arange(6, device=DEV)
    picks = torch.tensor([2, 9, 3, 4, 5, 9], device=DEV)      # 0, 2, 3, 4, 5
    got = ops.tree_accept(tokens, picks, starts, ctx, 6, parents=i32([-1, 0, 0, 2, 3, 4], DEV), caches=ops.TreeCaches([k], [v]), block_table=table)
    assert got.path.tolist() == [[0, 2, 3, 4, 5, -1]]
    for j, node in enumerate([0, 2, 3, 4, 5]):
        p, s = where[j]
        assert torch.equal(k[p, s], kv[node, 0]) and torch.equal(v[p, s], kv[node, 1])
    assert int((k != 0).any(-1).any(-1).sum()) == 6            # and nowhere else


# ---------------------------------------------------------------------------------------------------------------- accept
def accept_case(ctx, counts, page, layers, hkv, d, dtype, seed, vocab=5, forest=False):
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    starts = starts_of(counts)
    table, pages = tables(ctx, counts, page, rng)
    tokens, picks = torch.from_numpy(rng.integers(0, vocab, starts[-1])), torch.from_numpy(rng.integers(0, vocab, starts[-1]))
    shape = (layers, pages, page, hkv, d)
    return starts, table, tokens, picks, random_parents(counts, rng, forest), torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)


@pytest.mark.parametrize("layers,hkv,d,dtype", [(1, 1, 64, BF16), (3, 2, 128, BF16), (2, 8, 128, F32), (70, 1, 8, BF16), (130, 1, 4, F32)])
@pytest.mark.parametrize("ctx,counts,page", [([0], [1], 16), ([15, 16, 3], [40, 64, 1], 16), ([100, 0, 63, 64], [256, 0, 200, 65], 64)])
def test_accept_moves_the_path(ops, layers, hkv, d, dtype, ctx, counts, page):
    for seed, as_list, chain, max_path in ((1, False, False, None), (2, True, False, 3), (3, False, True, None), (4, True, False, 200)):
        starts, table, tokens, picks, parents, k, v = accept_case(ctx, counts, page, layers, hkv, d, dtype, seed, vocab=2, forest=seed == 4)
        par = None if chain else parents
        if chain:
            picks[:-1] = tokens[1:]                       # long paths: the target picks what was drafted, now and then not
            picks[7::9] += 1
        dk, dv = k.to(DEV), v.to(DEV)
        caches = ops.TreeCaches(list(dk) if as_list else dk, list(dv) if as_list else dv)
        got = ops.tree_accept(tokens.to(DEV), picks.to(DEV), i32(starts, DEV), i32(ctx, DEV), max(counts + [1]),
                              parents=None if par is None else par.to(DEV), max_path=max_path, caches=caches, block_table=i32(table, DEV))
        path, ids, counts_, lens = ref.accept(tokens.tolist(), picks.tolist(), starts, ctx, max_path or max(counts + [1]), par)
        assert got.path.tolist() == path and got.ids.tolist() == ids and got.counts.tolist() == counts_ and got.lens.tolist() == lens
        assert torch.equal(dk.cpu(), ref.move(k, ctx, table, path, counts_))
        assert torch.equal(dv.cpu(), ref.move(v, ctx, table, path, counts_))
        alone = ops.tree_accept(tokens.to(DEV), picks.to(DEV), i32(starts, DEV), i32(ctx, DEV), max(counts + [1]),
                                parents=None if par is None else par.to(DEV), max_path=max_path)
        assert all(torch.equal(a, b) for a, b in zip(alone, got))


def test_accept_takes_the_lowest_child_and_no_other_roots(ops):
    """Equal tokens among the children: the lowest; nodes without a parent are no children of node 0; a parent behind its child is none."""
    parents = torch.tensor([-1, -1, 0, 0, 0, 3, 2, 9, 2, 2], dtype=torch.int32)
    tokens = torch.tensor([7, 1, 2, 1, 1, 4, 9, 4, 5, 5])
    picks = torch.tensor([1, 1, 5, 4, 4, 4, 4, 4, 4, 4])
    path, ids, counts, lens = ref.accept(tokens.tolist(), picks.tolist(), [0, 10], [4], 10, parents)
    assert path[0][:counts[0]] == [0, 3, 5]
    got = ops.tree_accept(tokens.to(DEV), picks.to(DEV), i32([0, 10], DEV), i32([4], DEV), 10, parents=parents.to(DEV))
    assert got.path.tolist() == path and got.ids.tolist() == ids


def test_accept_leaves_places_without_a_page_alone(ops):
    starts, table, tokens, picks, parents, k, v = accept_case([14, 14], [20, 20], 16, 2, 1, 64, BF16, 5)
    picks[:-1] = tokens[1:]
    table[0][1] = -1
    table[1][0] = 10 ** 6
    dk, dv = k.to(DEV), v.to(DEV)
    sub = torch.arange(20, dtype=torch.int32).repeat(2) - 1
    got = ops.tree_accept(tokens.to(DEV), picks.to(DEV), i32(starts, DEV), i32([14, 14], DEV), 20, parents=sub.to(DEV),
                          caches=ops.TreeCaches(dk, dv), block_table=i32(table, DEV))
    assert torch.equal(dk.cpu(), ref.move(k, [14, 14], table, got.path.tolist(), got.counts.tolist()))


# ------------------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_verified_tree_is_the_chain_it_accepts(ops, dtype):
    """Plan, store, attention and acceptance over two layers, three steps in a row: every accepted node's attention is what the same tokens
    give when they come one by one as chains of one node, and afterwards both caches hold the same keys and values for the sequence."""
    rows, hq, hkv, d, page, layers, n = 3, 8, 2, 64, 16, 2, 24
    g = torch.Generator(device=DEV).manual_seed(1)
    rng = np.random.default_rng(1)
    table_w, pages = 12, 40
    vocab = torch.randn(50, layers, (hq + 2 * hkv) * d, generator=g, device=DEV).to(dtype)     # a token's q | k | v per layer
    w, freqs = torch.rand(d, generator=g, device=DEV) + 0.5, rotary_freqs(d // 2).to(DEV)

    def world():
        shape = (layers, pages, page, hkv, d)
        return {"k": torch.zeros(shape, dtype=dtype, device=DEV), "v": torch.zeros(shape, dtype=dtype, device=DEV),
                "bt": torch.full((rows, table_w), -1, dtype=torch.int32, device=DEV), "free": torch.arange(pages, dtype=torch.int32, device=DEV),
                "len": torch.zeros(rows, dtype=torch.int32, device=DEV)}

    def step(wd, tokens, counts, parents):
        starts = i32(starts_of(counts), DEV)
        par = None if parents is None else parents.to(DEV)
        plan = ops.tree_plan(wd["len"], starts, wd["bt"], wd["free"], max(counts), page, pages, parents=par, tokens=len(tokens))
        assert (plan.taken >= 0).all()
        wd["free"] = wd["free"][int(plan.taken.sum()):].contiguous()
        outs = []
        for i in range(layers):
            q = ops.qkv_norm_rotary_slots(vocab[tokens, i].contiguous(), plan.positions, plan.slots, wd["k"][i], wd["v"][i], hq, w, w, 1e-6, freqs)
            outs.append(ops.tree_attn(q, wd["k"][i], wd["v"][i], wd["len"], starts, wd["bt"], plan.mask, max(counts)))
        return starts, par, torch.stack(outs)

    tree, chain = world(), world()
    history = [[int(x)] for x in rng.integers(0, 50, rows)]
    for _ in range(3):
        counts = [n, 1, 9]
        parents = random_parents(counts, rng)
        tokens = torch.from_numpy(rng.integers(0, 50, sum(counts))).to(DEV)
        at = starts_of(counts)
        for b in range(rows):
            tokens[at[b]] = history[b][-1]
        starts, par, outs = step(tree, tokens, counts, parents)
        picks = torch.from_numpy(rng.integers(0, 50, sum(counts))).to(DEV)
        for b in range(rows):                                  # the target agrees down to some node
            way = ref.ancestors(parents, at[b], int(rng.integers(counts[b] // 2, counts[b])))[::-1]
            for a, c in zip(way, way[1:]):
                picks[at[b] + a] = tokens[at[b] + c]
        got = ops.tree_accept(tokens, picks, starts, tree["len"], max(counts), parents=par, caches=ops.TreeCaches(tree["k"], tree["v"]),
                              block_table=tree["bt"])
        taken = got.counts.tolist()
        for j in range(max(taken)):                            # the same tokens one by one
            live = [b for b in range(rows) if j < taken[b]]
            one = [1 if b in live else 0 for b in range(rows)]
            toks = torch.stack([tokens[at[b] + got.path[b, j]] for b in live])
            _, _, single = step(chain, toks, one, None)
            for i, b in enumerate(live):
                a, e = outs[:, at[b] + int(got.path[b, j])].double(), single[:, i].double()
                # (two results of the same sums in another order, bf16 with its own weights' and outputs' rounding)
                tol = 4 * torch.finfo(dtype).eps if dtype == BF16 else 2e-5
                assert ((a - e).abs() <= tol * (1 + e.abs())).all()
            chain["len"] += i32(one, DEV)
        # the tree keeps whole pages for nodes that were not accepted: give them back by hand, as a user's bookkeeping does
        assert got.lens.tolist() == chain["len"].tolist()
        tree["len"] = got.lens.clone()
        for b in range(rows):
            length, used = int(tree["len"][b]), -(-int(tree["len"][b]) // page)
            back = tree["bt"][b, used:][tree["bt"][b, used:] >= 0]
            tree["free"] = torch.cat([tree["free"], back])
            tree["bt"][b, used:] = -1
            for s in range(length):
                p, e = int(tree["bt"][b, s // page]), int(chain["bt"][b, s // page])
                assert torch.equal(tree["k"][:, p, s % page], chain["k"][:, e, s % page])
                assert torch.equal(tree["v"][:, p, s % page], chain["v"][:, e, s % page])
            history[b] += [int(x) for x in got.ids[b, :taken[b]]]


@pytest.mark.parametrize("d,hq,hkv", [(64, 8, 2), (128, 8, 1), (128, 4, 4)])
def test_one_node_is_the_decode_attention(ops, d, hq, hkv):
    """A row of one node against the one-token op beside it (core.paged_attention.paged_attn_decode, which appends the key itself)."""
    from micro_vllm_amd.core.paged_attention import paged_attn_decode
    case = AttnCase([5, 300, 64, 1000], [1, 1, 1, 1], hq, hkv, d, 64, BF16, seed=21, tail=0)
    k_new = torch.stack([case.k[case.table[b][c // 64], c % 64] for b, c in enumerate(case.ctx)]).to(DEV)
    v_new = torch.stack([case.v[case.table[b][c // 64], c % 64] for b, c in enumerate(case.ctx)]).to(DEV)
    want = paged_attn_decode(case.q.to(DEV), k_new, v_new, case.k.to(DEV), case.v.to(DEV), i32(case.ctx, DEV), i32(case.table, DEV))
    o, mag, size, count = case.reference()
    both = 2 * ref.attn_bound(o, mag, size, count, d, BF16)
    assert ((run_attn(ops, case).double().cpu() - want.double().cpu()).abs() <= both).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_recorded_steps_replay(ops, dtype):
    """Two recorded steps (plan, store, attention cut into splits, acceptance) replayed in turn on two streams, eager work and new inputs
    between them: every replay is what the eager calls give on the same inputs."""
    def make(seed):
        case = AttnCase([700, 30], [20, 33], 8, 2, 64, 64, dtype, seed=seed, tail=0)
        g = torch.Generator(device=DEV).manual_seed(seed)
        s = {"case": case, "ctx": i32(case.ctx, DEV), "starts": i32(case.starts, DEV), "bt": i32(case.table, DEV), "free": i32([0], DEV),
             "parents": case.parents.to(DEV), "k": case.k.to(DEV)[None].repeat(2, 1, 1, 1, 1), "v": case.v.to(DEV)[None].repeat(2, 1, 1, 1, 1),
             "qkv": torch.randn(case.T, 12 * 64, generator=g, device=DEV).to(dtype), "freqs": rotary_freqs(32).to(DEV),
             "w": torch.rand(64, generator=g, device=DEV) + 0.5, "tokens": torch.randint(0, 3, (case.T,), generator=g, device=DEV),
             "picks": torch.randint(0, 3, (case.T,), generator=g, device=DEV)}
        s["caches"] = ops.TreeCaches(s["k"], s["v"])
        s["plan"], s["path"] = ops.TreePlan.empty(2, case.T, case.max_nodes, DEV), ops.TreePath.empty(2, 16, DEV)
        s["q"], s["o"] = torch.empty(case.T, 8, 64, dtype=dtype, device=DEV), torch.empty(case.T, 8, 64, dtype=dtype, device=DEV)
        return s

    def go(s):
        n = s["case"].max_nodes
        plan = ops.tree_plan(s["ctx"], s["starts"], s["bt"], s["free"], n, 64, s["case"].pages, parents=s["parents"], out=s["plan"])
        for i in range(2):
            ops.qkv_norm_rotary_slots(s["qkv"], plan.positions, plan.slots, s["k"][i], s["v"][i], 8, s["w"], s["w"], 1e-6, s["freqs"], out=s["q"])
            ops.tree_attn(s["q"], s["k"][i], s["v"][i], s["ctx"], s["starts"], s["bt"], plan.mask, n, out=s["o"], num_splits=5)
        ops.tree_accept(s["tokens"], s["picks"], s["starts"], s["ctx"], n, parents=s["parents"], caches=s["caches"], block_table=s["bt"], out=s["path"])

    def results(s):
        return [t.clone() for t in (*s["plan"], s["bt"], s["q"], s["o"], *s["path"], s["k"], s["v"])]

    pair = [make(1), make(2)]
    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in pair:
        go(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            go(s)
        graphs.append(graph)
    for turn in range(4):
        start = []
        for s in pair:
            s["qkv"].add_(0.25)
            s["picks"].copy_((s["picks"] + 1) % 3)
            start.append((s["k"].clone(), s["v"].clone()))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        replayed = [results(s) for s in pair]
        for s, (k, v), got in zip(pair, start, replayed):
            s["k"].copy_(k)
            s["v"].copy_(v)
            for t in (*s["plan"], s["q"], s["o"], *s["path"]):
                t.fill_(0)
            go(s)
            torch.cuda.synchronize()
            for a, b in zip(got, results(s)):
                assert torch.equal(a, b), f"replay {turn}"
