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
from typing import NamedTuple, Optional

import torch

from .. import _native as nv

MAX_NODES = 256      # nodes of a row with a tree or a mask


def _i32(t: torch.Tensor, n: Optional[int] = None) -> int:
    assert t.is_cuda and t.dtype == torch.int32 and t.dim() == 1 and t.is_contiguous(), "contiguous int32 device vector expected"
    assert n is None or t.shape[0] == n, f"{t.shape[0]} values where {n} are expected"
    return t.data_ptr()


def _table(t: torch.Tensor, rows: int):
    assert t.is_cuda and t.dtype == torch.int32 and t.dim() == 2 and t.shape[0] == rows and (t.stride(1) == 1 or t.shape[1] == 1), \
        "int32 block table [rows, columns] expected"
    return t.data_ptr(), t.stride(0) if rows > 1 else t.shape[1], t.shape[1]


def _same_device(first: torch.Tensor, *others):
    idx = first.get_device()
    assert idx == torch.cuda.current_device(), "the tensors' device has to be the current one"
    for t in others:
        assert t is None or t.get_device() == idx, "tensors on different devices"


class TreePlan(NamedTuple):
    """What tree_plan leaves.  Per token: slots (page * page size + place in it, -1: none), positions, rows, mask [tokens, words] int64
    (bit i of word i // 64: node i of the row is the token itself or an ancestor; None where no mask was asked for); per row: taken, the
    pages taken off the free list, -1 for a row that did not get its pages."""
    slots: torch.Tensor
    positions: torch.Tensor
    rows: torch.Tensor
    mask: Optional[torch.Tensor]
    taken: torch.Tensor

    @classmethod
    def empty(cls, rows: int, tokens: int, max_nodes: int, device, mask: bool = True) -> "TreePlan":
        i32 = [torch.empty(n, dtype=torch.int32, device=device) for n in (tokens, tokens, tokens, rows)]
        words = max(1, (max_nodes + 63) // 64)
        m = torch.empty(tokens, words, dtype=torch.int64, device=device) if mask else None
        return cls(i32[0], i32[1], i32[2], m, i32[3])


def tree_plan(ctx_lens: torch.Tensor, row_start: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor, max_nodes: int,
              page: int, num_pages: int, parents: Optional[torch.Tensor] = None, out: Optional[TreePlan] = None,
              tokens: Optional[int] = None, mask: Optional[bool] = None) -> TreePlan:
    """The tables of a step from its rows' lengths, on the device: pages for the nodes, slots, positions, rows and ancestor masks.

    ctx_lens [rows] and row_start [rows + 1] int32; max_nodes bounds the nodes of a row (256 where there are parents or a mask, any
    number of them, as of a prompt's portion, otherwise; nodes past it are left alone).  block_table [rows, columns] int32 in place: columns
    of the cached tokens are kept, the ones that the nodes open get pages of free_pages in row order, free_pages[0] first.  A row whose
    pages are not there any more, and every row behind it that needs some, or one that has no columns for them, gets none (taken -1, slots
    -1, its columns untouched).  parents int32 [tokens], None: a chain.  `tokens` (default: those of parents or out) is the number of
    tokens that the outputs hold; `mask` (default: with parents or out, what they have) says whether a mask is wanted."""
    rows = ctx_lens.shape[0]
    if tokens is None:
        assert out is not None or parents is not None, "how many tokens the step has is given by parents, out or tokens"
        tokens = (out.slots if out is not None else parents).shape[0]
    if out is None:
        out = TreePlan.empty(rows, tokens, max_nodes, ctx_lens.device, mask=parents is not None if mask is None else mask)
    else:
        assert mask is None or mask == (out.mask is not None)
    m, words = out.mask, 0
    if m is not None:
        assert m.is_cuda and m.dtype == torch.int64 and m.dim() == 2 and m.shape[0] == tokens and m.is_contiguous()
        words = m.shape[1]
        assert words * 64 >= max_nodes, f"{words} mask words for {max_nodes} nodes"
    assert (m is None and parents is None) or max_nodes <= MAX_NODES, f"trees and masks go up to {MAX_NODES} nodes a row"
    bt, bt_stride, cols = _table(block_table, rows)
    _same_device(ctx_lens, row_start, block_table, free_pages, parents, *out)
    nv.check("mv_tree_plan", nv.lib().mv_tree_plan(
        _i32(ctx_lens), _i32(row_start, rows + 1), None if parents is None else _i32(parents, tokens), bt, bt_stride, cols,
        _i32(free_pages), free_pages.shape[0], rows, tokens, int(max_nodes), int(page), int(num_pages), _i32(out.slots, tokens),
        _i32(out.positions, tokens), _i32(out.rows, tokens), None if m is None else m.data_ptr(), words, _i32(out.taken, rows),
        nv.stream_ptr()))
    return out


def _norm(w: Optional[torch.Tensor], d: int):
    if w is None:
        return None
    assert w.is_cuda and w.dtype == torch.float32 and w.numel() == d and w.is_contiguous(), "norm weight: float32 [head size]"
    return w.data_ptr()


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor):
    assert k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.dtype == v_cache.dtype, "caches [pages, page, kv heads, d]"
    assert k_cache.is_contiguous() and v_cache.is_contiguous() and k_cache.dtype in (torch.bfloat16, torch.float32)
    return k_cache.shape


def qkv_norm_rotary_slots(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                          heads: int, q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
                          inv_freq: Optional[torch.Tensor] = None, adjacent: bool = False,
                          out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows of qkv [tokens, (heads + 2 kv_heads) * d] = q heads | k heads | v heads of one projection.  Every head of q and of k is divided
    by its root mean square and multiplied by q_norm / k_norm (float32 [d], shared by the heads; None: no norm), its first
    2 * inv_freq.numel() dimensions are turned by positions[t] * inv_freq (float64; None: no rotation; `adjacent` pairs (2i, 2i + 1), else i
    with i + half), all of it in fp32 and rounded once.  q goes to out [tokens, heads, d], k and v to k_cache / v_cache
    [pages, page, kv_heads, d] at slots[t] (negative or past the last page: not stored; no two tokens may name one slot).  qkv bf16 with bf16
    caches, float32 with either; out has the caches' type and may be q's own part of qkv where the types agree."""
    pages, page, kv_heads, d = _cache(k_cache, v_cache)
    assert qkv.is_cuda and qkv.dim() == 2 and qkv.dtype in (torch.bfloat16, torch.float32) and (qkv.stride(1) == 1 or qkv.shape[1] == 1)
    tokens = qkv.shape[0]
    assert qkv.shape[1] == (heads + 2 * kv_heads) * d, f"rows of {qkv.shape[1]} values are not {heads} + 2 x {kv_heads} heads of {d}"
    src_f32, dst_f32 = qkv.dtype == torch.float32, k_cache.dtype == torch.float32
    assert src_f32 or not dst_f32, "float32 caches take float32 rows"
    if out is None:
        out = torch.empty(tokens, heads, d, dtype=k_cache.dtype, device=qkv.device)
    assert out.shape == (tokens, heads, d) and out.dtype == k_cache.dtype and out.stride(2) == 1 and (heads == 1 or out.stride(1) == d)
    rot = 0
    if inv_freq is not None:
        rot = 2 * inv_freq.numel()
        assert inv_freq.is_cuda and inv_freq.dtype == torch.float64 and inv_freq.is_contiguous() and rot <= d
    _same_device(qkv, positions, slots, k_cache, v_cache, q_norm, k_norm, inv_freq, out)
    ld = qkv.stride(0) if tokens > 1 else qkv.shape[1]
    ldq = out.stride(0) if tokens > 1 else heads * d
    nv.check("mv_qkv_norm_rotary_slots", nv.lib().mv_qkv_norm_rotary_slots(
        qkv.data_ptr(), ld, _norm(q_norm, d), _norm(k_norm, d), float(eps), nv.ptr(inv_freq), rot, int(adjacent), _i32(positions, tokens),
        _i32(slots, tokens), out.data_ptr(), ldq, k_cache.data_ptr(), v_cache.data_ptr(), pages * page, tokens, int(heads), kv_heads, d,
        int(src_f32), int(dst_f32), nv.stream_ptr()))
    return out


def tree_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, ctx_lens: torch.Tensor, row_start: torch.Tensor,
              block_table: torch.Tensor, mask: Optional[torch.Tensor], max_nodes: int, softmax_scale: Optional[float] = None,
              out: Optional[torch.Tensor] = None, num_splits: int = 0, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of every node over its row's cached tokens and the nodes that its mask names (bit i of word i // 64: node i; it need not
    be a tree's; None: a chain), whose keys and values are in the cache already.  q [tokens, heads, d] bf16 or float32 as the caches
    [pages, page, kv_heads, d]; d 64 or 128, up to eight heads to a kv head, pages of a power of two of 16 tokens or more; max_nodes (at most
    256) bounds the nodes of a row.  A node that sees nothing gets zeros; places without a page (-1) and keys behind the table's last
    column do not count; tokens behind the last row, and nodes past max_nodes, keep what `out` held.  Scores and softmax in fp32; bf16:
    weights rounded to bf16 in front of the product with the values.  num_splits 0: picked; `workspace`: float32, at least
    tree_attn_workspace(...) bytes, of this call alone while it runs (default: allocated)."""
    pages, page, kv_heads, d = _cache(k_cache, v_cache)
    assert q.is_cuda and q.dim() == 3 and q.dtype == k_cache.dtype and q.shape[2] == d, "q [tokens, heads, head size] of the caches' type"
    tokens, heads, _ = q.shape
    assert q.stride(2) == 1 and (heads == 1 or q.stride(1) == d), "q heads must be contiguous"
    assert heads % kv_heads == 0, f"{heads} heads on {kv_heads}"
    rows = ctx_lens.shape[0]
    words = 0
    if mask is not None:
        assert mask.is_cuda and mask.dtype == torch.int64 and mask.dim() == 2 and mask.shape[0] == tokens and mask.is_contiguous()
        words = mask.shape[1]
        assert words * 64 >= max_nodes, f"{words} mask words for {max_nodes} nodes"
    if out is None:
        out = torch.zeros(tokens, heads, d, dtype=q.dtype, device=q.device)
    assert out.shape == q.shape and out.dtype == q.dtype and out.stride(2) == 1 and (heads == 1 or out.stride(1) == d)
    assert out.data_ptr() != q.data_ptr() or q.numel() == 0, "out may not be q"
    bt, bt_stride, cols = _table(block_table, rows)
    _same_device(q, k_cache, v_cache, ctx_lens, row_start, block_table, mask, out, workspace)
    L = nv.lib()
    if num_splits <= 0:
        num_splits = L.mv_tree_attn_pick_splits(rows, int(max_nodes), heads, kv_heads, d, cols * page, int(q.dtype == torch.float32))
    need = L.mv_tree_attn_workspace_bytes(tokens, heads, d, num_splits)
    if need and workspace is None:
        workspace = torch.empty(need // 4, dtype=torch.float32, device=q.device)
    scale = d ** -0.5 if softmax_scale is None else float(softmax_scale)
    nv.check("mv_tree_attn", L.mv_tree_attn(
        q.data_ptr(), q.stride(0) if tokens > 1 else heads * d, k_cache.data_ptr(), v_cache.data_ptr(), _i32(ctx_lens),
        _i32(row_start, rows + 1), bt, bt_stride, cols, nv.ptr(mask), words, out.data_ptr(), out.stride(0) if tokens > 1 else heads * d,
        workspace.data_ptr() if need else None, workspace.numel() * workspace.element_size() if need else 0, rows, tokens, int(max_nodes),
        heads, kv_heads, d, page, pages, scale, int(num_splits), int(q.dtype == torch.float32), nv.stream_ptr()))
    return out


def tree_attn_workspace(tokens: int, rows: int, max_nodes: int, heads: int, kv_heads: int, d: int, max_keys: int, num_splits: int = 0,
                        dtype: torch.dtype = torch.bfloat16) -> int:
    """Bytes of workspace of a tree_attn call (max_keys: its block table's columns times the page size); 0: none."""
    L = nv.lib()
    splits = num_splits if num_splits > 0 else L.mv_tree_attn_pick_splits(rows, max_nodes, heads, kv_heads, d, max_keys, int(dtype == torch.float32))
    return L.mv_tree_attn_workspace_bytes(tokens, heads, d, splits)


class TreeCaches:
    """The key and value caches of a model's layers for `tree_accept`: [layers, pages, page, kv_heads, d] each, or lists of
    [pages, page, kv_heads, d] (KVCacheManager.k_caches / .v_caches).  Holds the tensors and their addresses."""

    def __init__(self, k_caches, v_caches):
        k, v = list(k_caches), list(v_caches)
        assert len(k) == len(v) and len(k) > 0
        self.pages, self.page, kv_heads, d = _cache(k[0], v[0])
        for a, b in zip(k, v):
            assert a.is_cuda and _cache(a, b) == k[0].shape and a.dtype == k[0].dtype
            assert a.get_device() == k[0].get_device() and b.get_device() == k[0].get_device(), "tensors on different devices"
        self.row_bytes = kv_heads * d * k[0].element_size()
        assert self.row_bytes % 16 == 0 and all(t.data_ptr() % 16 == 0 for t in k + v), "a token's keys must be whole 16-byte pieces"
        self.layers, self.first = len(k), k[0]
        self._tensors = (k, v)
        self.k = (ctypes.c_void_p * len(k))(*[t.data_ptr() for t in k])
        self.v = (ctypes.c_void_p * len(v))(*[t.data_ptr() for t in v])


class TreePath(NamedTuple):
    """What tree_accept leaves, per row: path [max_path] (accepted nodes, node 0 first, -1 behind them), ids [max_path] int64 (the target's
    picks along it: the row's new tokens, the last of them not yet in the cache; -1 behind them), counts, lens (ctx_lens + counts)."""
    path: torch.Tensor
    ids: torch.Tensor
    counts: torch.Tensor
    lens: torch.Tensor

    @classmethod
    def empty(cls, rows: int, max_path: int, device) -> "TreePath":
        return cls(torch.empty(rows, max_path, dtype=torch.int32, device=device), torch.empty(rows, max_path, dtype=torch.int64, device=device),
                   torch.empty(rows, dtype=torch.int32, device=device), torch.empty(rows, dtype=torch.int32, device=device))


def tree_accept(tokens: torch.Tensor, picks: torch.Tensor, row_start: torch.Tensor, ctx_lens: torch.Tensor, max_nodes: int,
                parents: Optional[torch.Tensor] = None, max_path: Optional[int] = None, caches: Optional[TreeCaches] = None,
                block_table: Optional[torch.Tensor] = None, out: Optional[TreePath] = None) -> TreePath:
    """The part of every row's tree that the target model agrees with: from node 0 on to the lowest later node whose parent is the
    current one and whose token (int64 [tokens]) is the target's pick behind it (int64 [tokens]), until there is none or the path has
    max_path nodes (default: out's, else max_nodes).  With `caches` the keys and values of the path's j-th node are moved to index
    ctx_lens[b] + j of the sequence in every layer (places without a page: not moved), which is where a sequence of lens[b] tokens has
    them; all of it one launch for up to 64 layers.  A row without nodes has an empty path."""
    n_tokens, rows = tokens.shape[0], ctx_lens.shape[0]
    assert tokens.is_cuda and tokens.dtype == torch.int64 and tokens.dim() == 1 and tokens.is_contiguous()
    assert picks.is_cuda and picks.dtype == torch.int64 and picks.shape == tokens.shape and picks.is_contiguous()
    assert max_nodes <= MAX_NODES, f"trees go up to {MAX_NODES} nodes a row"
    if max_path is None:
        max_path = out.path.shape[1] if out is not None else max(1, max_nodes)
    if out is None:
        out = TreePath.empty(rows, max_path, tokens.device)
    assert out.path.shape == (rows, max_path) and out.path.dtype == torch.int32 and out.path.is_contiguous()
    assert out.ids.shape == (rows, max_path) and out.ids.dtype == torch.int64 and out.ids.is_contiguous()
    assert rows == 0 or out.lens.data_ptr() != ctx_lens.data_ptr(), "the new lengths may not overwrite the old ones"
    bt = bt_stride = cols = layers = 0
    if caches is not None:
        assert block_table is not None, "moving keys and values takes the block table"
        bt, bt_stride, cols = _table(block_table, rows)
        layers = caches.layers
    _same_device(tokens, picks, parents, row_start, ctx_lens, *out, None if caches is None else caches.first,
                 None if caches is None else block_table)
    nv.check("mv_tree_accept", nv.lib().mv_tree_accept(
        tokens.data_ptr(), picks.data_ptr(), None if parents is None else _i32(parents, n_tokens), _i32(row_start, rows + 1),
        _i32(ctx_lens), bt or None, bt_stride, cols, caches.k if layers else None, caches.v if layers else None, layers,
        caches.row_bytes if layers else 0, caches.page if layers else 0, caches.pages if layers else 0, rows, n_tokens, int(max_nodes),
        int(max_path), out.path.data_ptr(), out.ids.data_ptr(), _i32(out.counts, rows), _i32(out.lens, rows), nv.stream_ptr()))
    return out
