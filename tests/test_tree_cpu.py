"""Host side of the ops of a step that verifies drafted tokens: what the C entry points and their Python shims refuse before anything is
launched, and the oracle of their GPU tests against other statements of the same things."""
import pytest
import torch

from oracle import ref_tree as ref
from tree_util import AttnCase

NULL, P = None, 1 << 20      # an address that is 16-byte aligned; nothing may follow it
FAR = 1 << 30                # another


@pytest.fixture(scope="module")
def nv():
    import micro_vllm_amd  # noqa: F401
    from micro_vllm_amd import _native
    return _native


def plan(nv, ctx=P, starts=P, parents=P, bt=P, stride=8, cols=8, free=P, n_free=4, rows=2, tokens=10, nodes=8, page=16, pages=10, slots=P, pos=P,
         row=P, mask=P, words=1, taken=P):
    return nv.lib().mv_tree_plan(ctx, starts, parents, bt, stride, cols, free, n_free, rows, tokens, nodes, page, pages, slots, pos, row, mask,
                                 words, taken, NULL)


def test_plan_refuses(nv):
    bad = [dict(ctx=NULL), dict(starts=NULL), dict(bt=NULL), dict(free=NULL), dict(slots=NULL), dict(pos=NULL), dict(row=NULL), dict(taken=NULL),
           dict(rows=-1), dict(tokens=-1), dict(nodes=-1), dict(page=0), dict(pages=0), dict(cols=-1), dict(stride=7), dict(n_free=-1),
           dict(words=0), dict(words=5), dict(nodes=65, words=1)]
    for b in bad:
        assert plan(nv, **b) == nv.MV_ERR_INVALID_ARG, b
    assert plan(nv, nodes=257, words=4) == nv.MV_ERR_UNSUPPORTED
    assert plan(nv, nodes=257, mask=NULL) == nv.MV_ERR_UNSUPPORTED           # parents alone
    assert plan(nv, page=1 << 16, pages=1 << 16) == nv.MV_ERR_UNSUPPORTED     # slots past 32 bits
    assert plan(nv, rows=0, ctx=NULL, bt=NULL) == nv.MV_OK


def store(nv, qkv=P, ld=1024, qn=P, kn=P, freq=P, rot=64, pos=P, slots=P, out=FAR, ldq=512, k=P, v=P, n=100, tokens=3, hq=8, hkv=4, d=64, src=0, dst=0):
    return nv.lib().mv_qkv_norm_rotary_slots(qkv, ld, qn, kn, 1e-6, freq, rot, 0, pos, slots, out, ldq, k, v, n, tokens, hq, hkv, d, src, dst, NULL)


def test_store_refuses(nv):
    bad = [dict(qkv=NULL), dict(pos=NULL), dict(slots=NULL), dict(out=NULL), dict(k=NULL), dict(v=NULL), dict(freq=NULL), dict(ld=1023), dict(ldq=511),
           dict(tokens=-1), dict(hq=0), dict(hkv=0), dict(d=0), dict(rot=-2), dict(rot=63), dict(rot=66), dict(n=0)]
    for b in bad:
        assert store(nv, **b) == nv.MV_ERR_INVALID_ARG, b
    assert store(nv, dst=1) == nv.MV_ERR_UNSUPPORTED
    # q over anything of the rows but its own part, or over that in another type or with another stride
    for b in (dict(out=P + 512 * 2, ldq=1024), dict(out=P + 16, ldq=1024), dict(out=P, ldq=512), dict(out=P, ldq=1024, src=1), dict(out=P - 16, ldq=1024),
              dict(out=P + 2 * 1024 * 2 + 1023 * 2, ldq=600), dict(out=P + 1000 * 2, ldq=1100, ld=1100), dict(tokens=1, out=P - 1022)):
        assert store(nv, **b) == nv.MV_ERR_INVALID_ARG, b
    assert store(nv, tokens=0, qkv=NULL) == nv.MV_OK


def attn(nv, q=P, ldq=512, k=P, v=P, ctx=P, starts=P, bt=P, stride=8, cols=8, mask=P, words=1, out=FAR, ldo=512, ws=NULL, ws_bytes=0, rows=2, tokens=9,
         nodes=8, hq=8, hkv=4, d=64, page=16, pages=20, scale=0.1, splits=1, f32=0):
    return nv.lib().mv_tree_attn(q, ldq, k, v, ctx, starts, bt, stride, cols, mask, words, out, ldo, ws, ws_bytes, rows, tokens, nodes, hq, hkv, d,
                                 page, pages, scale, splits, f32, NULL)


def test_attention_refuses(nv):
    bad = [dict(q=NULL), dict(k=NULL), dict(v=NULL), dict(ctx=NULL), dict(starts=NULL), dict(bt=NULL), dict(out=NULL), dict(q=P + 8), dict(k=P + 2),
           dict(out=P + 4), dict(ldq=508), dict(ldq=516), dict(ldo=500), dict(ldo=515), dict(rows=-1), dict(tokens=-1), dict(nodes=-1), dict(hq=6),
           dict(hkv=0), dict(cols=0), dict(stride=7), dict(page=0), dict(pages=0), dict(splits=0), dict(scale=0.0), dict(scale=-1.0),
           dict(scale=float("nan")), dict(scale=float("inf")), dict(words=0), dict(words=5), dict(nodes=65)]
    for b in bad:
        assert attn(nv, **b) == nv.MV_ERR_INVALID_ARG, b
    for b in (dict(d=96, hq=4, ldq=384, ldo=384), dict(hq=36, ldq=4096, ldo=4096), dict(page=48), dict(page=8), dict(nodes=257, words=4), dict(splits=65),
              dict(cols=(1 << 26) + 1, stride=1 << 27), dict(rows=1 << 16), dict(rows=60000, hq=36, hkv=36, ldq=4096, ldo=4096)):      # keys past 2^30, rows
        assert attn(nv, **b) == nv.MV_ERR_UNSUPPORTED, b
    for b in (dict(out=P), dict(out=P + 16), dict(out=P, ldo=1024), dict(out=P + 256, ldq=640, ldo=640), dict(tokens=1, out=P - 1008)):
        assert attn(nv, **b) == nv.MV_ERR_INVALID_ARG, b          # out over q
    assert attn(nv, splits=2) == nv.MV_ERR_WORKSPACE
    need = nv.lib().mv_tree_attn_workspace_bytes(9, 8, 64, 2)
    assert need >= 2 * 9 * 8 * 66 * 4
    assert attn(nv, splits=2, ws=P, ws_bytes=need - 1) == nv.MV_ERR_WORKSPACE
    assert attn(nv, splits=2, ws=P + 4, ws_bytes=need) == nv.MV_ERR_WORKSPACE
    for b in (dict(rows=0), dict(tokens=0), dict(nodes=0)):
        assert attn(nv, q=NULL, **b) == nv.MV_OK


def accept(nv, tokens=P, picks=P, parents=P, starts=P, ctx=P, bt=P, stride=8, cols=8, k=(P,), v=(P,), layers=1, row_bytes=256, page=16, pages=20, rows=2,
           n=9, nodes=8, max_path=8, path=FAR, ids=FAR, counts=FAR, lens=FAR):
    import ctypes
    arr = lambda t: None if t is None else (ctypes.c_void_p * len(t))(*t)      # noqa: E731
    return nv.lib().mv_tree_accept(tokens, picks, parents, starts, ctx, bt, stride, cols, arr(k), arr(v), layers, row_bytes, page, pages, rows, n,
                                   nodes, max_path, path, ids, counts, lens, NULL)


def test_accept_refuses(nv):
    bad = [dict(tokens=NULL), dict(picks=NULL), dict(starts=NULL), dict(ctx=NULL), dict(path=NULL), dict(ids=NULL), dict(counts=NULL), dict(bt=NULL),
           dict(k=None), dict(v=None), dict(k=(NULL,)), dict(v=(P + 8,)), dict(rows=-1), dict(n=-1), dict(nodes=-1), dict(max_path=0), dict(layers=-1),
           dict(page=0), dict(pages=0), dict(row_bytes=0), dict(stride=7), dict(lens=P), dict(ids=P)]
    for b in bad:
        assert accept(nv, **b) == nv.MV_ERR_INVALID_ARG, b
    for b in (dict(nodes=257), dict(max_path=257), dict(row_bytes=24)):
        assert accept(nv, **b) == nv.MV_ERR_UNSUPPORTED, b
    assert accept(nv, rows=0, tokens=NULL) == nv.MV_OK


def test_shims_refuse_tensors_off_the_device(nv):
    from micro_vllm_amd.core import tree_decode as ops
    z = torch.zeros(4, dtype=torch.int32)
    case = AttnCase([5], [3], 4, 2, 64, 16, torch.bfloat16)
    with pytest.raises(AssertionError):
        ops.tree_plan(z, z, torch.zeros(4, 4, dtype=torch.int32), z, 4, 16, 10, tokens=4)
    with pytest.raises(AssertionError):
        ops.tree_attn(case.q, case.k, case.v, z, z, torch.zeros(4, 4, dtype=torch.int32), None, 4)
    with pytest.raises(AssertionError):
        ops.qkv_norm_rotary_slots(torch.zeros(4, 8 * 64), z, z, case.k, case.v, 4)
    with pytest.raises(AssertionError):
        ops.TreeCaches([case.k], [case.v])
    with pytest.raises(AssertionError):
        ops.tree_accept(z.long(), z.long(), z, z, 4)


def test_pick_of_splits_stays_in_its_range(nv):
    L = nv.lib()
    for rows in (1, 3, 64, 5000):
        for nodes in (1, 16, 256):
            for keys in (1, 64, 5000, 1 << 20):
                assert all(1 <= L.mv_tree_attn_pick_splits(rows, nodes, 8, 2, 64, keys, f32) <= 64 for f32 in (0, 1))


def test_oracle_attention_is_a_dense_softmax():
    """A row's oracle output against scaled_dot_product_attention with the same mask laid out densely."""
    case = AttnCase([21], [13], 4, 2, 64, 16, torch.float32, seed=1)
    o, mag, _, count = case.reference()
    keys = [(case.table[0][j // 16], j % 16) for j in range(34)]
    k = torch.stack([case.k[p, s] for p, s in keys]).double().permute(1, 0, 2)
    v = torch.stack([case.v[p, s] for p, s in keys]).double().permute(1, 0, 2)
    see = torch.zeros(13, 34, dtype=torch.bool)
    see[:, :21] = True
    for i in range(13):
        for j in case.seen[i]:
            see[i, 21 + j] = True
    want = torch.nn.functional.scaled_dot_product_attention(case.q[:13].double().permute(1, 0, 2), k.repeat_interleave(2, 0), v.repeat_interleave(2, 0),
                                                            attn_mask=see[None])
    assert torch.allclose(o, want.permute(1, 0, 2), atol=1e-12) and count.tolist() == see.sum(1).tolist() and (mag >= o.abs() - 1e-12).all()


def test_oracle_plan_by_hand():
    parents = torch.tensor([-1, 0, 0, 1, -1, 4, 0])
    slots, pos, rows, seen, taken, table = ref.plan([5, 3], [0, 4, 7], [[2, -1], [7, -1]], [9, 4], 4, 20, parents)
    assert taken == [-1, 1] and slots[:4] == [-1] * 4 and slots[4:] == [7 * 4 + 3, 9 * 4, 9 * 4 + 1] and table == [[2, -1], [7, 9]]
    assert pos[:4] == [5, 6, 6, 7] and seen[3] == {0, 1, 3} and rows == [0] * 4 + [1] * 3


def test_acceptance_of_planned_rows_refuses(nv):
    """The form with what the plan took: the same checks, and shims that want the plan's tensor as it is."""
    import ctypes
    one = (ctypes.c_void_p * 1)(P)

    def planned(tokens=P, taken=P, rows=2, nodes=8, row_bytes=256, counts=FAR, layers=1):
        return nv.lib().mv_tree_accept_planned(tokens, P, P, P, P, taken, P, 8, 8, one, one, layers, row_bytes, 16, 20, rows, 9, nodes, 8, FAR, FAR + 4096,
                                               counts, FAR + 12288, NULL)

    for b in (dict(tokens=NULL), dict(counts=NULL), dict(rows=-1), dict(nodes=-1), dict(layers=-1), dict(row_bytes=0)):
        assert planned(**b) == nv.MV_ERR_INVALID_ARG, b
    assert planned(nodes=257) == nv.MV_ERR_UNSUPPORTED and planned(row_bytes=24) == nv.MV_ERR_UNSUPPORTED
    assert planned(rows=0, tokens=NULL, taken=NULL) == nv.MV_OK


def test_acceptance_refuses_outputs_over_what_it_reads_or_writes(nv):
    """Every output on every input and every other output, whole, by its last or its first value; next to them it is no refusal: the entry gets as far as
    the device, of which there is none here that takes these addresses."""
    import ctypes
    rows, n, path_len, cols, stride, K = 3, 9, 8, 5, 7, 1 << 12
    sizes = {"tokens": 8 * n, "picks": 8 * n, "parents": 4 * n, "starts": 4 * rows + 4, "ctx": 4 * rows, "taken": 4 * rows,
             "bt": 4 * ((rows - 1) * stride + cols), "path": 4 * rows * path_len, "ids": 8 * rows * path_len, "counts": 4 * rows, "lens": 4 * rows}
    apart = {name: P + K * i for i, name in enumerate(sizes)}
    outs = ("path", "ids", "counts", "lens")

    def call(entry=None, **at):
        a = {**apart, **at}
        caches = (ctypes.c_void_p * 1)(FAR)
        head = [a["tokens"], a["picks"], a["parents"], a["starts"], a["ctx"]]
        tail = [a["bt"], stride, cols, caches, caches, 1, 256, 16, 20, rows, n, 8, path_len, a["path"], a["ids"], a["counts"], a["lens"], NULL]
        L = nv.lib()
        return L.mv_tree_accept(*head, *tail) if entry == "plain" else L.mv_tree_accept_planned(*head, a["taken"], *tail)

    for o in outs:
        for other in sizes:
            if other == o:
                continue
            for at in (apart[other], apart[other] + sizes[other] - 4, apart[other] - sizes[o] + 4):
                assert call(**{o: at}) == nv.MV_ERR_INVALID_ARG, (o, other)
                if other != "taken":
                    assert call("plain", **{o: at}) == nv.MV_ERR_INVALID_ARG, (o, other)
    if torch.cuda.is_available():
        return
    assert call() not in (nv.MV_ERR_INVALID_ARG, nv.MV_OK)
    for o in outs:
        for other in sizes:
            if other != o:
                for at in (apart[other] + sizes[other], apart[other] - sizes[o]):
                    assert call(**{o: at}) not in (nv.MV_ERR_INVALID_ARG, nv.MV_OK), (o, other)
    assert call(counts=apart["bt"] + 4 * cols, lens=apart["bt"] + 4 * (stride + cols)) == nv.MV_ERR_INVALID_ARG       # 3 values between rows 2 apart
    assert call(lens=apart["bt"] + 4 * (stride * (rows - 1) + cols)) != nv.MV_ERR_INVALID_ARG


def test_plan_refuses_outputs_over_what_it_reads_or_writes(nv):
    rows, n, cols, stride, n_free, words, K = 3, 9, 5, 7, 6, 2, 1 << 12
    sizes = {"ctx": 4 * rows, "starts": 4 * rows + 4, "parents": 4 * n, "free": 4 * n_free, "bt": 4 * ((rows - 1) * stride + cols), "slots": 4 * n,
             "pos": 4 * n, "row": 4 * n, "mask": 8 * n * words, "taken": 4 * rows}
    apart = {name: P + K * i for i, name in enumerate(sizes)}
    ins = ("ctx", "starts", "parents", "free")
    call = lambda **at: plan(nv, stride=stride, cols=cols, n_free=n_free, rows=rows, tokens=n, words=words, **{**apart, **at})      # noqa: E731
    for o in sizes:
        for other in sizes:
            if other == o or (o in ins and other in ins):
                continue
            for at in (apart[other], apart[other] + sizes[other] - 4, apart[other] - sizes[o] + 4):
                assert call(**{o: at}) == nv.MV_ERR_INVALID_ARG, (o, other)
    if torch.cuda.is_available():
        return
    assert call() not in (nv.MV_ERR_INVALID_ARG, nv.MV_OK)
    for o in sizes:
        for other in sizes:
            if other != o:
                for at in (apart[other] + sizes[other], apart[other] - sizes[o]):
                    assert call(**{o: at}) not in (nv.MV_ERR_INVALID_ARG, nv.MV_OK), (o, other)


@pytest.mark.parametrize("f32", [0, 1])
def test_attention_refuses_out_and_workspace_over_what_it_reads(nv, f32):
    rows, n, hq, hkv, d, page, pages, cols, stride, words, splits, K = 3, 9, 8, 4, 64, 16, 5, 6, 9, 2, 3, 1 << 19
    size = 4 if f32 else 2
    need = nv.lib().mv_tree_attn_workspace_bytes(n, hq, d, splits)
    pool = pages * page * hkv * d * size
    ld = hq * d + 32                                         # rows of q and out with room behind each
    span = ((n - 1) * ld + hq * d) * size
    sizes = {"q": span, "k": pool, "v": pool, "ctx": 4 * rows, "starts": 4 * rows + 4, "bt": 4 * ((rows - 1) * stride + cols), "mask": 8 * n * words,
             "out": span, "ws": need}
    assert max(sizes.values()) < K // 2
    apart = {name: FAR + K * i + K // 2 for i, name in enumerate(sizes)}
    call = lambda **at: attn(nv, ldq=ld, ldo=ld, stride=stride, cols=cols, words=words, ws_bytes=need, rows=rows, tokens=n, hq=hq, hkv=hkv, d=d, page=page,      # noqa: E731
                             pages=pages, splits=splits, f32=f32, **{**apart, **at})
    even = lambda x: x // 16 * 16                            # noqa: E731  (out and workspace are 16-byte aligned)
    for o in ("out", "ws"):
        for other in sizes:
            if other != o:
                for at in (apart[other], even(apart[other] + sizes[other] - 1), even(apart[other] - sizes[o] + 16)):
                    assert call(**{o: at}) == nv.MV_ERR_INVALID_ARG, (o, other, at - apart[other])
    if torch.cuda.is_available():
        return
    assert call() not in (nv.MV_ERR_INVALID_ARG, nv.MV_OK)
    for o in ("out", "ws"):
        for other in sizes:
            if other != o:
                for at in (even(apart[other] + sizes[other] + 15), even(apart[other] - sizes[o])):
                    assert call(**{o: at}) not in (nv.MV_ERR_INVALID_ARG, nv.MV_OK), (o, other)
    # one cache for keys and values is read alone, and rows of out in the room behind those of q are no overlap
    assert call(v=apart["k"]) not in (nv.MV_ERR_INVALID_ARG, nv.MV_OK)
    wide = dict(ldq=2 * hq * d, ldo=2 * hq * d)
    assert attn(nv, q=FAR, out=FAR + hq * d * size, hq=hq, hkv=hkv, d=d, f32=f32, **wide) not in (nv.MV_ERR_INVALID_ARG, nv.MV_OK)


@pytest.mark.parametrize("src,dst", [(0, 0), (1, 0), (1, 1)])
def test_store_refuses_caches_and_q_over_what_it_reads_or_writes(nv, src, dst):
    n, hq, hkv, d, rot, slots, K = 9, 8, 4, 64, 32, 50, 1 << 19
    sb, db, ld, ldq = (4 if src else 2), (4 if dst else 2), (hq + 2 * hkv) * d + 16, hq * d + 16
    pool = slots * hkv * d * db
    sizes = {"qkv": ((n - 1) * ld + (hq + 2 * hkv) * d) * sb, "qn": 4 * d, "kn": 4 * d, "freq": 4 * rot, "pos": 4 * n, "slots": 4 * n,
             "out": ((n - 1) * ldq + hq * d) * db, "k": pool, "v": pool}
    apart = {name: FAR + K * i + K // 2 for i, name in enumerate(sizes)}
    outs = ("out", "k", "v")
    call = lambda ldq=ldq, **at: store(nv, ld=ld, ldq=ldq, rot=rot, n=slots, tokens=n, hq=hq, hkv=hkv, d=d, src=src, dst=dst, **{**apart, **at})      # noqa: E731
    for o in outs:
        for other in sizes:
            if other != o:
                for at in (apart[other], apart[other] + sizes[other] - 2, apart[other] - sizes[o] + 2):
                    assert call(**{o: at}) == nv.MV_ERR_INVALID_ARG, (o, other, at - apart[other])
    if torch.cuda.is_available():
        return
    assert call() not in (nv.MV_ERR_INVALID_ARG, nv.MV_OK)
    for o in outs:
        for other in sizes:
            if other != o:
                for at in (apart[other] + sizes[other], apart[other] - sizes[o]):
                    assert call(**{o: at}) not in (nv.MV_ERR_INVALID_ARG, nv.MV_OK), (o, other)
    if sb == db:                                              # q over its own part of the rows
        assert call(out=apart["qkv"], ldq=ld) not in (nv.MV_ERR_INVALID_ARG, nv.MV_OK)


def test_caches_are_named_once(nv):
    from micro_vllm_amd.core.tree_decode import _apart
    assert _apart([], 64) and _apart([128], 64) and _apart([256, 0, 64, 192, 128], 64)
    assert not _apart([64, 128, 64], 64) and not _apart([0, 100, 48], 64)
