"""A step that verifies drafted tokens over the paged cache: its plan, the store of its keys and values, its attention and the
acceptance (csrc/tree_ops.hip, tree_attn.hip).

Row b of a step is a sequence with ctx_lens[b] cached tokens; it brings the nodes row_start[b] .. row_start[b + 1] - 1 of the step's
tokens.  Node 0 is the last token that is known, every other node continues an earlier node of its row (parents: its index in the row,
-1 or anything that is not an earlier node: none).  Node i lies in the cache at index ctx_lens[b] + i of its sequence whatever its
depth, at position ctx_lens[b] + depth.  Per layer: `qkv_norm_rotary_slots`, then `tree_attn`; once a step: `tree_plan` in front,
`tree_accept` behind.  With parents=None and mask=None the nodes of a row are a chain, so the same calls verify a plain draft.

No counterpart in the reference, whose decode step is one token a row (core/engine.py:241-285).  The tensors a call reads and writes lie
on one device, which has to be the current one; every call goes to the current stream, allocates nothing when it is given `out` (and
`workspace`), and can be captured.  Rows must not share the pages that a step's nodes lie in.
"""
import ctypes
from functools import lru_cache
from typing import Optional

import torch

from .. import _native as nv

MAX_NODES = 256      # nodes of a row with a tree or a mask


_I32, _I64, _F32, _BF16 = torch.int32, torch.int64, torch.float32, torch.bfloat16
# hipStream_t of a device's current stream, for a device that tensors lie on (nv.stream_ptr also asks which device and whether there is one: 0.3 us of
# a small step's 8)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _vec(t: torch.Tensor, n: int, dev: int, dtype=_I32) -> int:
    """Address of a contiguous vector of n values on device `dev` (one call a tensor of a step's many: what it asks is what there is to ask)."""
    assert t.shape == (n,) and t.dtype is dtype and t.get_device() == dev and t.is_contiguous(), \
        f"contiguous {dtype} vector of {n} on cuda:{dev} expected, got {t.dtype} {tuple(t.shape)} on {t.device}"
    return t.data_ptr()


def _table(t: torch.Tensor, rows: int, dev: int):
    shape = t.shape
    assert len(shape) == 2 and shape[0] == rows and t.dtype is _I32 and t.get_device() == dev, "int32 block table [rows, columns] expected"
    stride, one = t.stride()
    assert one == 1 or shape[1] == 1, "block table rows must be contiguous"
    return t.data_ptr(), stride if rows > 1 else shape[1], shape[1]


def _current(t: torch.Tensor) -> int:
    """Device of a call: that of its first tensor, which has to be the current one."""
    dev = t.get_device()
    assert dev >= 0, "device tensors expected"
    assert dev == torch._C._cuda_getDevice(), "the tensors' device has to be the current one"
    return dev


def _mask(m: torch.Tensor, tokens: int, max_nodes: int, dev: int):
    shape = m.shape
    assert m.dtype is _I64 and len(shape) == 2 and shape[0] == tokens and m.is_contiguous() and m.get_device() == dev, \
        "int64 mask [tokens, words] expected"
    assert shape[1] * 64 >= max_nodes, f"{shape[1]} mask words for {max_nodes} nodes"
    return m.data_ptr(), shape[1]


class TreePlan:
    """What tree_plan leaves.  Per token: slots (page * page size + place in it, negative: none), positions, rows, mask [tokens, words] int64
    (bit i of word i // 64: node i of the row is the token itself or an ancestor; None where no mask was asked for); per row: taken, the
    pages taken off the free list, -1 for a row that did not get its pages.  The buffers are checked once, here."""
    __slots__ = ("_t", "_p", "tokens", "n_rows", "words", "device")

    def __init__(self, slots: torch.Tensor, positions: torch.Tensor, rows: torch.Tensor, mask: Optional[torch.Tensor], taken: torch.Tensor):
        self.tokens, self.n_rows, self.device = slots.shape[0], taken.shape[0], slots.get_device()
        assert self.device >= 0, "device tensors expected"
        self._t = (slots, positions, rows, mask, taken)
        m, self.words = (None, 0) if mask is None else _mask(mask, self.tokens, 1, self.device)
        self._p = (*[_vec(t, self.tokens, self.device) for t in (slots, positions, rows)], m, _vec(taken, self.n_rows, self.device))

    slots = property(lambda self: self._t[0])
    positions = property(lambda self: self._t[1])
    rows = property(lambda self: self._t[2])
    mask = property(lambda self: self._t[3])
    taken = property(lambda self: self._t[4])

    def __iter__(self):
        return iter(self._t)

    @classmethod
    def empty(cls, rows: int, tokens: int, max_nodes: int, device, mask: bool = True) -> "TreePlan":
        i32 = [torch.empty(n, dtype=_I32, device=device) for n in (tokens, tokens, tokens, rows)]
        m = torch.empty(tokens, max(1, (max_nodes + 63) // 64), dtype=_I64, device=device) if mask else None
        return cls(i32[0], i32[1], i32[2], m, i32[3])


def tree_plan(ctx_lens: torch.Tensor, row_start: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor, max_nodes: int,
              page: int, num_pages: int, parents: Optional[torch.Tensor] = None, out: Optional[TreePlan] = None,
              tokens: Optional[int] = None, mask: Optional[bool] = None) -> TreePlan:
    """The tables of a step from its rows' lengths, on the device: pages for the nodes, slots, positions, rows and ancestor masks.

    ctx_lens [rows] and row_start [rows + 1] int32; max_nodes bounds the nodes of a row (256 where there are parents or a mask, any
    number of them, as of a prompt's portion, otherwise; tokens past it are no nodes).  block_table [rows, columns] int32 in place: columns
    of the cached tokens are kept, the ones that the nodes open get pages of free_pages in row order, free_pages[0] first, whatever they
    held (pages of an earlier step's nodes that were not accepted are the caller's to give back first).  A row whose
    pages are not there any more, and every row behind it that needs some, or one that has no columns for them, gets none (taken -1, slots
    -1, and -1 in the columns that its nodes would open, which may hold pages that are another row's by now).  parents int32 [tokens], None: a chain.  `tokens` (default: those of parents or out) is the number of
    tokens that the outputs hold, which may be more than the rows have: the others' slots are negative afterwards (-1 in place of what an earlier
    step left), so that a store of all of them stores the nodes, and the rest of their values is left alone.  `mask` (default: with
    parents or out, what they have) says whether a mask is wanted.  Outputs and table may share no memory with each other or the inputs."""
    rows, dev = ctx_lens.shape[0], _current(ctx_lens)
    if out is None:
        if tokens is None:
            assert parents is not None, "how many tokens the step has is given by parents, out or tokens"
            tokens = parents.shape[0]
        out = TreePlan.empty(rows, tokens, max_nodes, ctx_lens.device, mask=parents is not None if mask is None else mask)
    else:
        assert (tokens is None or tokens == out.tokens) and out.n_rows == rows and out.device == dev, "out is of another step's sizes"
        assert mask is None or mask == (out.mask is not None)
        tokens = out.tokens
    if rows == 0 and tokens:
        out.slots.fill_(-1)      # (the entry point has nothing to launch)
    slots, positions, row_of, m, taken = out._p
    assert m is None or out.words * 64 >= max_nodes, f"{out.words} mask words for {max_nodes} nodes"
    assert max_nodes <= MAX_NODES or (m is None and parents is None), f"trees and masks go up to {MAX_NODES} nodes a row"
    bt, bt_stride, cols = _table(block_table, rows, dev)
    free = free_pages.shape[0]
    nv.check("mv_tree_plan", nv.lib().mv_tree_plan(
        _vec(ctx_lens, rows, dev), _vec(row_start, rows + 1, dev), None if parents is None else _vec(parents, tokens, dev), bt, bt_stride,
        cols, _vec(free_pages, free, dev), free, rows, tokens, max_nodes, page, num_pages, slots, positions, row_of, m, out.words, taken,
        _stream(dev)))
    return out


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor, dev: int):
    shape, dtype = k_cache.shape, k_cache.dtype
    assert len(shape) == 4 and v_cache.shape == shape and v_cache.dtype is dtype, "caches [pages, page, kv heads, d] of one type expected"
    assert dtype is _BF16 or dtype is _F32, f"bf16 or float32 caches, not {dtype}"
    assert k_cache.is_contiguous() and v_cache.is_contiguous() and k_cache.get_device() == dev and v_cache.get_device() == dev
    return shape


def _heads(t: torch.Tensor, shape, dtype, dev: int, what: str) -> int:
    """Row stride of [tokens, heads, d] whose heads lie side by side."""
    assert t.shape == shape and t.dtype is dtype and t.get_device() == dev, f"{what}: {dtype} {tuple(shape)} expected, got {t.dtype} {tuple(t.shape)}"
    row, head, one = t.stride()
    assert one == 1 and (head == shape[2] or shape[1] == 1), f"{what}: heads must lie side by side"
    return row if shape[0] > 1 else shape[1] * shape[2]


def qkv_norm_rotary_slots(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                          heads: int, q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
                          inv_freq: Optional[torch.Tensor] = None, adjacent: bool = False,
                          out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows of qkv [tokens, (heads + 2 kv_heads) * d] = q heads | k heads | v heads of one projection.  Every head of q and of k is divided
    by its root mean square and multiplied by q_norm / k_norm (float32 [d], shared by the heads; None: no norm), its first
    2 * inv_freq.numel() dimensions are turned by positions[t] * inv_freq (float64; None: no rotation; `adjacent` pairs (2i, 2i + 1), else i
    with i + half), all of it in fp32 and rounded once.  q goes to out [tokens, heads, d], k and v to k_cache / v_cache
    [pages, page, kv_heads, d] at slots[t] (negative or past the last page: not stored; no two tokens may name one slot).  qkv bf16 with bf16
    caches, float32 with either; out has the caches' type and may be q's own part of qkv where the types agree; apart from that out, k_cache and v_cache may share no
    memory with each other or an input."""
    dev = _current(qkv)
    pages, page, kv_heads, d = _cache(k_cache, v_cache, dev)
    (tokens, width), src, dst = qkv.shape, qkv.dtype, k_cache.dtype
    assert width == (heads + 2 * kv_heads) * d, f"rows of {width} values are not {heads} + 2 x {kv_heads} heads of {d}"
    assert (src is _BF16 and dst is _BF16) or src is _F32, "bf16 rows with bf16 caches, or float32 rows"
    ld, one = qkv.stride()
    assert one == 1 or width == 1
    if out is None:
        out = torch.empty(tokens, heads, d, dtype=dst, device=qkv.device)
    rot = 0 if inv_freq is None else 2 * inv_freq.shape[0]
    nv.check("mv_qkv_norm_rotary_slots", nv.lib().mv_qkv_norm_rotary_slots(
        qkv.data_ptr(), ld if tokens > 1 else width, None if q_norm is None else _vec(q_norm, d, dev, _F32),
        None if k_norm is None else _vec(k_norm, d, dev, _F32), eps, None if rot == 0 else _vec(inv_freq, rot // 2, dev, torch.float64), rot,
        adjacent, _vec(positions, tokens, dev), _vec(slots, tokens, dev), out.data_ptr(), _heads(out, (tokens, heads, d), dst, dev, "out"),
        k_cache.data_ptr(), v_cache.data_ptr(), pages * page, tokens, heads, kv_heads, d, src is _F32, dst is _F32, _stream(dev)))
    return out


@lru_cache(maxsize=1024)
def _pick_splits(dev: int, rows: int, max_nodes: int, heads: int, kv_heads: int, d: int, max_keys: int, f32: bool) -> int:
    """mv_tree_attn_pick_splits, a function of the sizes and of the current device (the argument `dev`)."""
    return nv.lib().mv_tree_attn_pick_splits(rows, max_nodes, heads, kv_heads, d, max_keys, f32)


def tree_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, ctx_lens: torch.Tensor, row_start: torch.Tensor,
              block_table: torch.Tensor, mask: Optional[torch.Tensor], max_nodes: int, softmax_scale: Optional[float] = None,
              out: Optional[torch.Tensor] = None, num_splits: int = 0, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of every node over its row's cached tokens and the nodes that its mask names (bit i of word i // 64: node i; it need not
    be a tree's; None: a chain), whose keys and values are in the cache already.  q [tokens, heads, d] bf16 or float32 as the caches
    [pages, page, kv_heads, d]; d 64 or 128, up to eight heads to a kv head, pages of a power of two of 16 tokens or more; max_nodes (at most
    256) bounds the nodes of a row.  A node that sees nothing gets zeros; places without a page (-1) and keys behind the table's last
    column do not count; tokens behind the last row, and nodes past max_nodes, keep what `out` held.  Scores (below 2^30 in size) and
    softmax in fp32; bf16: weights rounded to bf16 in front of the product with the values (2.0 to 2.3e-3 off in all, 1.65e-3 of it the output's rounding).
    What the table has room for picks the kernel and its splits: pass block_table[:, :cols] where the rows are known to be shorter (up to twice as quick for
    a short row).  `out` and `workspace` may share no memory with each other or an input; the table
    has room for 2^30 keys at most.  num_splits 0: picked; `workspace`: float32, at least
    tree_attn_workspace(...) bytes, of this call alone while it runs (default: allocated); out=None allocates zeros, a launch more."""
    dev = _current(q)
    pages, page, kv_heads, d = _cache(k_cache, v_cache, dev)
    shape, dtype = q.shape, q.dtype
    assert len(shape) == 3 and shape[2] == d and dtype is k_cache.dtype, "q [tokens, heads, head size] of the caches' type"
    tokens, heads, _ = shape
    assert heads % kv_heads == 0, f"{heads} heads on {kv_heads}"
    rows = ctx_lens.shape[0]
    m, words = (None, 0) if mask is None else _mask(mask, tokens, max_nodes, dev)
    if out is None:
        out = torch.zeros(shape, dtype=dtype, device=q.device)
    q_ptr, out_ptr = q.data_ptr(), out.data_ptr()
    assert out_ptr != q_ptr or tokens == 0, "out may not be q"
    bt, bt_stride, cols = _table(block_table, rows, dev)
    L, f32 = nv.lib(), dtype is _F32
    if num_splits <= 0:
        num_splits = _pick_splits(dev, rows, max_nodes, heads, kv_heads, d, cols * page, f32)
    ws = need = 0
    if num_splits > 1:
        need = L.mv_tree_attn_workspace_bytes(tokens, heads, d, num_splits)
        if workspace is None:
            workspace = torch.empty(need // 4, dtype=_F32, device=q.device)
        assert workspace.get_device() == dev and workspace.is_contiguous()
        ws, need = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    nv.check("mv_tree_attn", L.mv_tree_attn(
        q_ptr, _heads(q, shape, dtype, dev, "q"), k_cache.data_ptr(), v_cache.data_ptr(), _vec(ctx_lens, rows, dev),
        _vec(row_start, rows + 1, dev), bt, bt_stride, cols, m, words, out_ptr, _heads(out, shape, dtype, dev, "out"), ws or None, need, rows,
        tokens, max_nodes, heads, kv_heads, d, page, pages, d ** -0.5 if softmax_scale is None else softmax_scale, num_splits, f32,
        _stream(dev)))
    return out


def tree_attn_workspace(tokens: int, rows: int, max_nodes: int, heads: int, kv_heads: int, d: int, max_keys: int, num_splits: int = 0,
                        dtype: torch.dtype = torch.bfloat16) -> int:
    """Bytes of workspace of a tree_attn call (max_keys: its block table's columns times the page size); 0: none."""
    L = nv.lib()
    splits = num_splits if num_splits > 0 else L.mv_tree_attn_pick_splits(rows, max_nodes, heads, kv_heads, d, max_keys, int(dtype == torch.float32))
    return L.mv_tree_attn_workspace_bytes(tokens, heads, d, splits)


def _apart(addresses, nbytes: int) -> bool:
    """Whether pieces of nbytes at these addresses share nothing."""
    at = sorted(addresses)
    return all(b - a >= nbytes for a, b in zip(at, at[1:]))


class TreeCaches:
    """The key and value caches of a model's layers for `tree_accept`: [layers, pages, page, kv_heads, d] each, or lists of
    [pages, page, kv_heads, d] (KVCacheManager.k_caches / .v_caches), no two of which share memory (a cache that layers share is named once: named twice, its tokens would be
    moved twice).  Holds the tensors and their addresses."""

    def __init__(self, k_caches, v_caches):
        k, v = list(k_caches), list(v_caches)
        assert len(k) == len(v) and len(k) > 0
        self.device = k[0].get_device()
        assert self.device >= 0, "device tensors expected"
        self.pages, self.page, kv_heads, d = _cache(k[0], v[0], self.device)
        for a, b in zip(k, v):
            assert _cache(a, b, self.device) == k[0].shape and a.dtype is k[0].dtype, "the layers' caches are of one shape and type"
        self.row_bytes = kv_heads * d * k[0].element_size()
        assert self.row_bytes % 16 == 0 and all(t.data_ptr() % 16 == 0 for t in k + v), "a token's keys must be whole 16-byte pieces"
        assert _apart([t.data_ptr() for t in k + v], k[0].numel() * k[0].element_size()), "every cache is named once, and none lies in another"
        self.layers = len(k)
        self._tensors = (k, v)
        self.k = (ctypes.c_void_p * len(k))(*[t.data_ptr() for t in k])
        self.v = (ctypes.c_void_p * len(v))(*[t.data_ptr() for t in v])


class TreePath:
    """What tree_accept leaves, per row: path [max_path] (accepted nodes, node 0 first, -1 behind them), ids [max_path] int64 (the target's
    picks along it: the row's new tokens, the last of them not yet in the cache; -1 behind them), counts, lens (ctx_lens + counts).  The
    buffers are checked once, here."""
    __slots__ = ("_t", "_p", "n_rows", "max_path", "device")

    def __init__(self, path: torch.Tensor, ids: torch.Tensor, counts: torch.Tensor, lens: torch.Tensor):
        (self.n_rows, self.max_path), self.device = path.shape, path.get_device()
        assert self.device >= 0, "device tensors expected"
        assert path.dtype is _I32 and path.is_contiguous()
        assert ids.shape == path.shape and ids.dtype is _I64 and ids.is_contiguous() and ids.get_device() == self.device
        self._t = (path, ids, counts, lens)
        self._p = (path.data_ptr(), ids.data_ptr(), _vec(counts, self.n_rows, self.device), _vec(lens, self.n_rows, self.device))

    path = property(lambda self: self._t[0])
    ids = property(lambda self: self._t[1])
    counts = property(lambda self: self._t[2])
    lens = property(lambda self: self._t[3])

    def __iter__(self):
        return iter(self._t)

    @classmethod
    def empty(cls, rows: int, max_path: int, device) -> "TreePath":
        return cls(torch.empty(rows, max_path, dtype=_I32, device=device), torch.empty(rows, max_path, dtype=_I64, device=device),
                   torch.empty(rows, dtype=_I32, device=device), torch.empty(rows, dtype=_I32, device=device))


def tree_accept(tokens: torch.Tensor, picks: torch.Tensor, row_start: torch.Tensor, ctx_lens: torch.Tensor, max_nodes: int,
                parents: Optional[torch.Tensor] = None, max_path: Optional[int] = None, caches: Optional[TreeCaches] = None,
                block_table: Optional[torch.Tensor] = None, out: Optional[TreePath] = None, taken: Optional[torch.Tensor] = None) -> TreePath:
    """The part of every row's tree that the target model agrees with: from node 0 on to the lowest later node whose parent is the
    current one and whose token (int64 [tokens]) is the target's pick behind it (int64 [tokens]), until there is none or the path has
    max_path nodes (default: out's, else max_nodes).  With `caches` the keys and values of the path's j-th node are moved to index
    ctx_lens[b] + j of the sequence in every layer (places without a page: not moved), which is where a sequence of lens[b] tokens has
    them; all of it one launch for up to 64 layers.  A row without nodes has an empty path, and so has one that did not get its pages
    (`taken`, the plan's, is negative): its nodes are stored nowhere, its length stays.  Without `taken` every row counts as stored.  No output may share
    memory with another or with an input."""
    n_tokens, rows, dev = tokens.shape[0], ctx_lens.shape[0], _current(tokens)
    assert max_nodes <= MAX_NODES, f"trees go up to {MAX_NODES} nodes a row"
    if out is None:
        out = TreePath.empty(rows, max(1, max_nodes) if max_path is None else max_path, tokens.device)
    assert out.n_rows == rows and out.device == dev and (max_path is None or max_path == out.max_path), "out is of another step's sizes"
    path, ids, counts, lens = out._p
    ctx = _vec(ctx_lens, rows, dev)
    if caches is None:
        move = (None, 0, 0, None, None, 0, 0, 0, 0)
    else:
        assert block_table is not None and caches.device == dev, "moving keys and values takes the block table, on the caches' device"
        move = (*_table(block_table, rows, dev), caches.k, caches.v, caches.layers, caches.row_bytes, caches.page, caches.pages)
    nv.check("mv_tree_accept_planned", nv.lib().mv_tree_accept_planned(
        _vec(tokens, n_tokens, dev, _I64), _vec(picks, n_tokens, dev, _I64), None if parents is None else _vec(parents, n_tokens, dev),
        _vec(row_start, rows + 1, dev), ctx, None if taken is None else _vec(taken, rows, dev), *move, rows, n_tokens, max_nodes, out.max_path, path, ids, counts, lens, _stream(dev)))
    return out
