"""The operators of a step that verifies drafted tokens, as they are measured: their inputs, their plain forms in elementary torch
operations, the calls a user makes of the framework's kernels, what a pass cannot do without, and what 64-bit arithmetic gives.

A row (sequence) with ctx cached tokens brings n drafted nodes: node 0 is the last token that is known, every other node continues an
earlier one (parents, -1: none).  Nodes of all rows lie back to back (row_start); node i lies in the cache at index ctx + i of its sequence.

  plan    block tables, slots, positions and ancestor masks from request lengths and parents (tree_plan)
  store   norm of every head of q and k, rotation by position, keys and values to their slots (qkv_norm_rotary_slots)
  attn    attention of every node over the cached tokens, its ancestors and itself (tree_attn)
  accept  the walk along the target's own picks, and the accepted nodes' keys and values moved behind the cached ones in every
          layer (tree_accept)
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one chat that drafts a few tokens: the smallest plan, a launch's latency
        {"name": "plan-chat", "op": "plan", "rows": 1, "ctx": 45, "spread": 0, "nodes": 8, "ragged": False, "page": 256, "tree": True},
        # a full server between two steps: 256 rows of any length, full trees, small pages
        {"name": "plan-256-rows", "op": "plan", "rows": 256, "ctx": 8191, "spread": 3, "nodes": 64, "ragged": True, "page": 64, "tree": True},
        # one row of an 8B model's heads, 16 drafted nodes, far into a long sequence
        {"name": "store-8b-16", "op": "store", "rows": 1, "ctx": 100000, "spread": 0, "nodes": 16, "ragged": False, "page": 256, "hq": 32, "hkv": 8, "d": 128, "rot": 128, "adjacent": False, "src": "bf16", "dst": "bf16"},
        # a batch of 32 such rows with trees of 64 nodes
        {"name": "store-8b-32x64", "op": "store", "rows": 32, "ctx": 4096, "spread": 3, "nodes": 64, "ragged": False, "page": 256, "hq": 32, "hkv": 8, "d": 128, "rot": 128, "adjacent": False, "src": "bf16", "dst": "bf16"},
        # a small model kept in 32 bits, heads of 64 of which half turns, neighbouring pairs, odd tree sizes
        {"name": "store-1b-f32", "op": "store", "rows": 16, "ctx": 700, "spread": 2, "nodes": 33, "ragged": True, "page": 64, "hq": 32, "hkv": 4, "d": 64, "rot": 32, "adjacent": True, "src": "f32", "dst": "f32"},
        # a chat of a few lines on a small model: the shortest attention, tiles mostly padding
        {"name": "attn-1b-chat", "op": "attn", "rows": 1, "ctx": 45, "spread": 0, "nodes": 7, "ragged": False, "page": 256, "hq": 32, "hkv": 4, "d": 64, "dtype": "bf16"},
        # one token's worth of an 8B model behind a long context, 16 nodes: the keys' stream, cut over the chip
        {"name": "attn-8b-bs1-4k", "op": "attn", "rows": 1, "ctx": 4096, "spread": 0, "nodes": 16, "ragged": False, "page": 256, "hq": 32, "hkv": 8, "d": 128, "dtype": "bf16"},
        # continuous batching with full trees: 32 requests at whatever length each has reached
        {"name": "attn-8b-bs32-uneven", "op": "attn", "rows": 32, "ctx": 8191, "spread": 3, "nodes": 64, "ragged": True, "page": 256, "hq": 32, "hkv": 8, "d": 128, "dtype": "bf16"},
        # one GPU's share of a 70B model over eight, eight long contexts, eight heads to a key, small pages
        {"name": "attn-70b-shard-bs8-8k", "op": "attn", "rows": 8, "ctx": 8191, "spread": 0, "nodes": 48, "ragged": False, "page": 64, "hq": 8, "hkv": 1, "d": 128, "dtype": "bf16"},
        # the same mechanism in 32 bits, one head to a key
        {"name": "attn-f32-bs4", "op": "attn", "rows": 4, "ctx": 1500, "spread": 2, "nodes": 24, "ragged": True, "page": 64, "hq": 16, "hkv": 16, "d": 64, "dtype": "f32"},
        # the chat's own: a walk of a few steps, a few rows of 22 layers
        {"name": "accept-1b-chat", "op": "accept", "rows": 1, "ctx": 45, "spread": 0, "nodes": 8, "ragged": False, "page": 256, "layers": 22, "hkv": 4, "d": 64, "dtype": "bf16"},
        # 64 rows of an 8B model's heads, half its layers (the caches' own size is what limits it here)
        {"name": "accept-8b-64x64", "op": "accept", "rows": 64, "ctx": 4090, "spread": 3, "nodes": 64, "ragged": True, "page": 64, "layers": 16, "hkv": 8, "d": 128, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["plan", "store", "store", "attn", "attn", "attn", "accept"])
    c = {"op": op, "spread": rng.choice([0, 0, 1, 2, 3]), "ragged": rng.random() < 0.5, "page": rng.choice([16, 64, 256])}
    if op == "plan":
        c.update(rows=_log(rng, 1, 160), ctx=_log(rng, 1, 8191), nodes=_log(rng, 1, 64), tree=rng.random() < 0.8)
        return c
    c["d"] = rng.choice([64, 128])
    c["hkv"] = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8])
    if op == "accept":
        c.update(rows=_log(rng, 1, 40), ctx=_log(rng, 1, 4090), nodes=_log(rng, 1, 64), layers=_log(rng, 1, 16), dtype=rng.choice(["bf16", "bf16", "f32"]))
        if c["dtype"] == "f32":
            c["rows"] = (c["rows"] + 1) // 2
        return c
    c["hq"] = c["hkv"] * group
    if op == "store":
        src = rng.choice(["bf16", "f32"])
        c.update(rows=_log(rng, 1, 32), ctx=_log(rng, 1, 100000), nodes=_log(rng, 1, 64), rot=rng.choice([c["d"], c["d"], c["d"] // 2]),
                 adjacent=rng.random() < 0.3, src=src, dst="bf16" if src == "bf16" or rng.random() < 0.5 else "f32")
        while c["rows"] * c["nodes"] * (c["hq"] + 2 * c["hkv"]) * c["d"] * (2 if c["src"] == "f32" else 1) > 32 * 64 * 48 * 128:
            c["rows"] = (c["rows"] + 1) // 2 if c["rows"] > 1 else 1
            c["nodes"] = c["nodes"] if c["rows"] > 1 else max(1, c["nodes"] // 2)
        return c
    c.update(rows=_log(rng, 1, 32), ctx=_log(rng, 1, 8191), nodes=_log(rng, 1, 64), dtype=rng.choice(["bf16", "bf16", "bf16", "f32"]))
    # (products in 32 bits take sixteen times as long)
    products, keys = 32 * 38 * 32 * 4096 * 128 // (16 if c["dtype"] == "f32" else 1), 32 * 4096 * 8 * 128 // (2 if c["dtype"] == "f32" else 1)

    def costly():
        return c["rows"] * c["nodes"] * c["hq"] * c["ctx"] * c["d"] > products or c["rows"] * c["ctx"] * c["hkv"] * c["d"] > keys

    while c["rows"] > 1 and costly():
        c["rows"] = (c["rows"] + 1) // 2
    while c["ctx"] > 1 and costly():
        c["ctx"] //= 2
    return c


# ---------------------------------------------------------------------------------------- inputs

def _ctx_lens(case):
    """Lengths of the rows: all alike, or scattered below the largest (the golden ratio's multiples: no two alike, no order)."""
    low = {0: 1.0, 1: 0.75, 2: 0.4, 3: 0.06}[case["spread"]]
    return [max(0, int(case["ctx"] * (low + (1 - low) * ((0.13 + 0.6180339887 * (i + 1)) % 1.0)))) if case["spread"] else case["ctx"]
            for i in range(case["rows"])]


def _node_counts(case):
    n = case["nodes"]
    return [max(1, int(n * (0.25 + 0.75 * ((0.71 + 0.7548776662 * (i + 1)) % 1.0)) + 0.5)) if case["ragged"] else n for i in range(case["rows"])]


def _parents(case, rng):
    """Up to eight continuations of node 0, each later node one of an earlier one: the trees that drafters of a few levels leave."""
    out = []
    for n in _node_counts(case):
        for i in range(n):
            if i == 0:
                out.append(-1)
            elif i <= 8:
                out.append(0)
            else:
                out.append(int(rng.integers(i // 8, i // 3 + 1)))
    return np.array(out, dtype=np.int32)


def _starts(case):
    return np.concatenate([[0], np.cumsum(_node_counts(case))]).astype(np.int32)


def _pool(case, rng):
    """(block table [rows, width] with every page a row needs, pages in the pool): shuffled pages."""
    page = case["page"]
    need = [-(-(c + n) // page) for c, n in zip(_ctx_lens(case), _node_counts(case))]
    pages = sum(need) + 3
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((case["rows"], max(need) + 1), -1, dtype=np.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    return table, pages


def _shared_pool(case, rng):
    """The same where only the pages that a step's nodes lie in are a row's own, and all before them one page that the rows share (a common
    prompt): what a step writes, without gigabytes of cache around it."""
    page = case["page"]
    table = np.full((case["rows"], max(-(-(c + n) // page) for c, n in zip(_ctx_lens(case), _node_counts(case))) + 1), -1, dtype=np.int32)
    own_pages = []
    for b, (c, n) in enumerate(zip(_ctx_lens(case), _node_counts(case))):
        first, last = c // page, (c + n - 1) // page
        table[b, :first] = 0
        own_pages += [(b, j) for j in range(first, last + 1)]
    for (b, j), p in zip(own_pages, rng.permutation(len(own_pages))):
        table[b, j] = 1 + int(p)
    return table, len(own_pages) + 2


def _slots_of(case, table):
    page, out = case["page"], []
    for b, (c, n) in enumerate(zip(_ctx_lens(case), _node_counts(case))):
        out += [int(table[b, (c + i) // page]) * page + (c + i) % page for i in range(n)]
    return np.array(out, dtype=np.int32)


def _depths(parents, starts):
    depth = np.zeros(len(parents), dtype=np.int64)
    for b in range(len(starts) - 1):
        for t in range(starts[b], starts[b + 1]):
            depth[t] = 0 if parents[t] < 0 else depth[starts[b] + parents[t]] + 1
    return depth


def _masks(parents, starts, words):
    mask = np.zeros((len(parents), words), dtype=np.uint64)
    for b in range(len(starts) - 1):
        for t in range(starts[b], starts[b + 1]):
            i = int(t - starts[b])
            if parents[t] >= 0:
                mask[t] = mask[starts[b] + parents[t]]
            mask[t, i // 64] |= np.uint64(1) << np.uint64(i % 64)
    return mask.view(np.int64)


def _accepted(parents, starts, rng):
    """For each row a path down its tree that a target took.  Its nodes lie behind the places that they are moved to, so that a pass run
    twice finds the same inputs."""
    paths = []
    for b in range(len(starts) - 1):
        par = parents[starts[b]:starts[b + 1]]
        fits = []
        for i in range(len(par)):
            path = [i]
            while par[path[0]] >= 0:
                path.insert(0, int(par[path[0]]))
            if len(path) == 1 or path[1] >= len(path):
                fits.append(path)
        longest = [p for p in fits if len(p) >= 3] or fits
        paths.append(longest[int(rng.integers(len(longest)))])
    return paths


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def _randn(gen, shape, dtype, scale=1.0):
    t = torch.empty(shape, dtype=dtype, device=DEV)
    flat = t.view(-1)
    for i in range(0, flat.numel(), 1 << 28):      # (in pieces: the 32-bit numbers behind a large cache are not kept)
        part = flat[i:i + (1 << 28)]
        part.copy_(torch.randn(part.numel(), generator=gen, device=DEV) * scale)
    return t


def _inv_freq(rot):
    return 500000.0 ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)


def _raw(case, seed):
    """The inputs, alike for both forms and for the 64-bit one."""
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    parents, starts = _parents(case, rng), _starts(case)
    words = (case["nodes"] + 63) // 64
    r = {"parents": _dev(parents), "row_start": _dev(starts), "ctx": _dev(np.array(_ctx_lens(case), dtype=np.int32)),
         "host": (parents, starts), "tokens": len(parents), "words": words}
    if case["op"] == "plan":
        page = case["page"]
        table, pages = _pool(case, rng)
        held = [-(-c // page) for c in _ctx_lens(case)]
        free = [int(table[b, j]) for b in range(case["rows"]) for j in range(held[b], table.shape[1]) if table[b, j] >= 0]
        for b in range(case["rows"]):
            table[b, held[b]:] = -1
        r.update(table=_dev(table), pages=pages, free=_dev(rng.permutation(np.array(free or [0], dtype=np.int32))))
    elif case["op"] == "store":
        table, pages = _shared_pool(case, rng)
        src, dst, d = DTYPES[case["src"]], DTYPES[case["dst"]], case["d"]
        r.update(qkv=_randn(gen, (len(parents), (case["hq"] + 2 * case["hkv"]) * d), src, 2.0),
                 q_norm=1 + 0.2 * torch.randn(d, generator=gen, device=DEV), k_norm=1 + 0.2 * torch.randn(d, generator=gen, device=DEV),
                 positions=_dev((np.repeat(_ctx_lens(case), np.diff(starts)) + _depths(parents, starts)).astype(np.int32)),
                 slots=_dev(_slots_of(case, table)), inv_freq=_dev(_inv_freq(case["rot"])),
                 k=_randn(gen, (pages, case["page"], case["hkv"], d), dst), v=_randn(gen, (pages, case["page"], case["hkv"], d), dst))
    elif case["op"] == "attn":
        table, pages = _pool(case, rng)
        dt, d = DTYPES[case["dtype"]], case["d"]
        r.update(table=_dev(table), mask=_dev(_masks(parents, starts, words)), q=_randn(gen, (len(parents), case["hq"], d), dt),
                 k=_randn(gen, (pages, case["page"], case["hkv"], d), dt), v=_randn(gen, (pages, case["page"], case["hkv"], d), dt))
    else:
        table, pages = _shared_pool(case, rng)
        dt = DTYPES[case["dtype"]]
        tokens, picks = rng.integers(0, 128256, len(parents)), rng.integers(0, 128256, len(parents))
        for b, path in enumerate(_accepted(parents, starts, rng)):
            for cur, nxt in zip(path, path[1:]):
                picks[starts[b] + cur] = tokens[starts[b] + nxt]
        shape = (case["layers"], pages, case["page"], case["hkv"], case["d"])
        r.update(table=_dev(table), ids=_dev(tokens), picks=_dev(picks), k=_randn(gen, shape, dt), v=_randn(gen, shape, dt))
    return r


def _tree_ops():
    import micro_vllm_amd  # noqa: F401
    from micro_vllm_amd.core import tree_decode
    return tree_decode


def prepare(case, seed):
    r = _raw(case, seed)
    r["case"] = case
    host_starts = r["host"][1]
    counts = np.diff(host_starts)
    r["row_of"] = _dev(np.repeat(np.arange(case["rows"]), counts).astype(np.int64))
    r["node_of"] = _dev(np.concatenate([np.arange(n) for n in counts]).astype(np.int64))
    r["max_path"] = case["nodes"] if case["nodes"] < 16 else 16
    r["max_keys"] = max(c + int(n) for c, n in zip(_ctx_lens(case), counts))
    if own:
        ops = _tree_ops()
        if case["op"] == "plan":
            r["out"] = ops.TreePlan.empty(case["rows"], r["tokens"], case["nodes"], DEV)
        elif case["op"] == "store":
            r["out"] = torch.empty(r["tokens"], case["hq"], case["d"], dtype=r["k"].dtype, device=DEV)
        elif case["op"] == "attn":
            r["out"] = torch.empty_like(r["q"])
        else:
            r["caches"] = ops.TreeCaches(r["k"], r["v"])
            r["out"] = ops.TreePath.empty(case["rows"], r["max_path"], DEV)
    return r


# ---------------------------------------------------------------------------------------- a pass

def run(state):
    case = state["case"]
    if own:
        return _own(case["op"], case, state)
    return {"plan": _plan_plain, "store": _store_plain, "attn": _attn_plain, "accept": _accept_plain}[case["op"]](case, state)


def _own(op, case, s):
    ops = _tree_ops()
    if op == "plan":
        p = ops.tree_plan(s["ctx"], s["row_start"], s["table"], s["free"], max_nodes=case["nodes"], page=case["page"], num_pages=s["pages"],
                          parents=s["parents"] if case["tree"] else None, out=s["out"])
        return p.slots, p.positions, p.rows, p.mask, p.taken, s["table"]
    if op == "store":
        q = ops.qkv_norm_rotary_slots(s["qkv"], s["positions"], s["slots"], s["k"], s["v"], heads=case["hq"], q_norm=s["q_norm"],
                                      k_norm=s["k_norm"], eps=1e-6, inv_freq=s["inv_freq"], adjacent=case["adjacent"], out=s["out"])
        return q, s["k"], s["v"]
    if op == "attn":
        return ops.tree_attn(s["q"], s["k"], s["v"], s["ctx"], s["row_start"], s["table"], s["mask"], max_nodes=case["nodes"], out=s["out"])
    p = ops.tree_accept(s["ids"], s["picks"], s["row_start"], s["ctx"], max_nodes=case["nodes"], parents=s["parents"], caches=s["caches"],
                        block_table=s["table"], out=s["out"])
    return p.path, p.ids, p.counts, p.lens, s["k"], s["v"]


def _padded(s, case, values, fill):
    """A value per node as [rows, nodes]."""
    out = torch.full((case["rows"], case["nodes"]), fill, dtype=values.dtype, device=DEV)
    out[s["row_of"], s["node_of"]] = values
    return out


def _plan_plain(case, s):
    page, n_max = case["page"], case["nodes"]
    ctx, start = s["ctx"].long(), s["row_start"].long()
    n = start[1:] - start[:-1]
    held, total = (ctx + page - 1) // page, (ctx + n + page - 1) // page
    need = torch.where(n > 0, total - held, torch.zeros_like(n))
    wide = total > s["table"].shape[1]
    need = torch.where(wide, torch.zeros_like(need), need)
    upto = torch.cumsum(need, 0)
    refused = wide | ((need > 0) & (upto > s["free"].numel()))
    before = upto - need
    col = torch.arange(s["table"].shape[1], device=DEV)[None, :]
    fresh = (col >= held[:, None]) & (col < total[:, None]) & ~refused[:, None]
    pick = (before[:, None] + col - held[:, None]).clamp(0, max(s["free"].numel() - 1, 0))
    s["table"].copy_(torch.where(fresh, s["free"][pick], s["table"]))
    row, node = s["row_of"], s["node_of"]
    at = ctx[row] + node
    pg = s["table"][row, (at // page).clamp(max=s["table"].shape[1] - 1)].long()
    ok = ~refused[row] & (pg >= 0) & (pg < s["pages"])
    slots = torch.where(ok, pg * page + at % page, torch.full_like(at, -1))
    # ancestors by doubling: bits of the node and its parent, then of those two steps up, and so on
    if case["tree"]:
        up = _padded(s, case, s["parents"].long(), -1)
    else:
        up = (torch.arange(n_max, device=DEV) - 1)[None, :].expand(case["rows"], n_max).contiguous()
    idx = torch.arange(n_max, device=DEV)
    sees = torch.zeros(case["rows"], n_max, n_max, dtype=torch.bool, device=DEV)
    sees[:, idx, idx] = True
    step = 1
    while step < n_max:
        far = up.clamp(min=0)
        sees = sees | (torch.gather(sees, 1, far[:, :, None].expand(-1, -1, n_max)) & (up >= 0)[:, :, None])
        up = torch.where(up >= 0, torch.gather(up, 1, far), up)
        step *= 2
    depth = sees.sum(2) - 1
    words = s["words"]
    bits = torch.zeros(case["rows"], n_max, words * 64, dtype=torch.int64, device=DEV)
    bits[:, :, :n_max] = sees
    mask = (bits.view(case["rows"], n_max, words, 64) << torch.arange(64, device=DEV)).sum(3)
    taken = torch.where(refused, torch.full_like(need, -1), need)
    return slots.int(), (ctx[row] + depth[row, node]).int(), row.int(), mask[row, node], taken.int(), s["table"]


def _store_plain(case, s):
    hq, hkv, d, rot = case["hq"], case["hkv"], case["d"], case["rot"]
    x = s["qkv"].float().view(-1, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    angle = s["positions"].double()[:, None] * s["inv_freq"][None, :]
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]

    def turned(t, w):
        t = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w
        out = t.clone()
        if case["adjacent"]:
            a, b = t[..., 0:rot:2], t[..., 1:rot:2]
            out[..., 0:rot:2], out[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
        else:
            a, b = t[..., :rot // 2], t[..., rot // 2:rot]
            out[..., :rot // 2], out[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
        return out

    dt = s["k"].dtype
    where = s["slots"].long()
    s["k"].view(-1, hkv, d)[where] = turned(k, s["k_norm"]).to(dt)
    s["v"].view(-1, hkv, d)[where] = v.to(dt)
    return turned(q, s["q_norm"]).to(dt), s["k"], s["v"]


def _attn_plain(case, s):
    rows, n_max, hq, hkv, d, page = case["rows"], case["nodes"], case["hq"], case["hkv"], case["d"], case["page"]
    g, keys = hq // hkv, s["max_keys"]
    at = torch.arange(keys, device=DEV)
    slot = s["table"].long().clamp(min=0)[:, at // page] * page + at % page
    k = s["k"].view(-1, hkv, d)[slot].float().permute(0, 2, 3, 1).contiguous()                 # [rows, hkv, d, keys]
    v = s["v"].view(-1, hkv, d)[slot].float().permute(0, 2, 1, 3).contiguous()                 # [rows, hkv, keys, d]
    q = torch.zeros(rows, n_max, hq, d, device=DEV)
    q[s["row_of"], s["node_of"]] = s["q"].float()
    q = q.view(rows, n_max, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(rows, hkv, n_max * g, d)
    word = torch.zeros(rows, n_max, s["words"], dtype=torch.int64, device=DEV)
    word[s["row_of"], s["node_of"]] = s["mask"]
    node = at[None, :] - s["ctx"].long()[:, None]                                               # [rows, keys]: which node a key is
    inside = (node >= 0) & (node < n_max)
    far = node.clamp(0, n_max - 1)
    bit = (torch.gather(word, 2, (far // 64)[:, None, :].expand(rows, n_max, keys)) >> (far % 64)[:, None, :]) & 1
    n = (s["row_start"][1:] - s["row_start"][:-1]).long()
    seen = (node < 0)[:, None, :] | ((bit == 1) & (inside & (node < n[:, None]))[:, None, :])     # [rows, n_max, keys]
    score = torch.matmul(q, k) * d ** -0.5
    score = score.view(rows, hkv, n_max, g, keys).masked_fill_(~seen[:, None, :, None, :], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = (score - top).exp_()
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total > 0, total, torch.ones_like(total))).view(rows, hkv, n_max * g, keys)
    o = torch.matmul(p, v).view(rows, hkv, n_max, g, d).permute(0, 2, 1, 3, 4).reshape(rows, n_max, hq, d)
    return o[s["row_of"], s["node_of"]].to(s["q"].dtype)


def _accept_plain(case, s):
    rows, n_max, page = case["rows"], case["nodes"], case["page"]
    start, ctx, node_at = s["row_start"].long(), s["ctx"].long(), torch.arange(n_max, device=DEV)
    ids, picks, parents = _padded(s, case, s["ids"], -1), _padded(s, case, s["picks"], -2), _padded(s, case, s["parents"].long(), -2)
    alive = (start[1:] - start[:-1]) > 0
    cur = torch.zeros(rows, dtype=torch.int64, device=DEV)
    path, out_ids = [], []
    for _ in range(s["max_path"]):
        pick = torch.gather(picks, 1, cur[:, None])[:, 0]
        path.append(torch.where(alive, cur, torch.full_like(cur, -1)))
        out_ids.append(torch.where(alive, pick, torch.full_like(pick, -1)))
        fits = (parents == cur[:, None]) & (ids == pick[:, None]) & (node_at[None, :] > cur[:, None])
        first = torch.where(fits, node_at[None, :], torch.full_like(fits, n_max, dtype=torch.int64)).amin(1)
        alive = alive & (first < n_max)
        cur = torch.where(first < n_max, first, cur)
    path, out_ids = torch.stack(path, 1), torch.stack(out_ids, 1)
    counts = (path >= 0).sum(1)

    def slots(index):
        pg = torch.gather(s["table"].long(), 1, (index // page).clamp(0, s["table"].shape[1] - 1))
        return pg.clamp(min=0) * page + index % page

    step = torch.arange(path.shape[1], device=DEV)[None, :].expand_as(path)
    dst = slots(ctx[:, None] + step).reshape(-1)
    src = slots(ctx[:, None] + torch.where(path >= 0, path, step)).reshape(-1)
    # (behind a path's end a row is copied from itself, which may be behind its last page: to page 0 of the pool, which nothing moves in)
    live = (path >= 0).reshape(-1)
    src, dst = torch.where(live, src, torch.zeros_like(src)), torch.where(live, dst, torch.zeros_like(dst))
    for cache in (s["k"], s["v"]):
        flat = cache.view(case["layers"], -1, case["hkv"], case["d"])
        flat[:, dst] = flat[:, src]
    return path.int(), out_ids, counts.int(), (ctx + counts).int(), s["k"], s["v"]


# ---------------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    rows, counts, ctx = case["rows"], _node_counts(case), _ctx_lens(case)
    tokens = sum(counts)
    if case["op"] == "plan":
        words = (case["nodes"] + 63) // 64
        return {"bytes": tokens * ((4 if case["tree"] else 0) + 12 + 8 * words) + rows * 20, "flops": tokens * 10}
    if case["op"] == "store":
        size = {"bf16": 2, "f32": 4}
        values = tokens * (case["hq"] + 2 * case["hkv"]) * case["d"]
        return {"bytes": values * (size[case["src"]] + size[case["dst"]]) + tokens * 8, "flops": values * 8}
    size = {"bf16": 2, "f32": 4}[case["dtype"]]
    if case["op"] == "attn":
        keys = sum(c + n for c, n in zip(ctx, counts))
        pairs = sum(n * (c + n) for c, n in zip(ctx, counts))
        return {"bytes": (2 * keys * case["hkv"] + 2 * tokens * case["hq"]) * case["d"] * size, "flops": 4 * pairs * case["hq"] * case["d"]}
    # about three nodes of a row move (each read and written), keys and values, in every layer
    moved = rows * 3 * case["layers"] * 2 * case["hkv"] * case["d"] * size * 2
    return {"bytes": moved + tokens * 20 + rows * 32, "flops": tokens * 4}


# ---------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    r = _raw(case, seed)
    parents, starts = r["host"]
    ctx = _ctx_lens(case)
    page = case["page"]
    if case["op"] == "plan":
        table, free = r["table"].cpu().numpy().copy(), r["free"].cpu().numpy()
        if not case["tree"]:
            parents = np.concatenate([np.arange(n) - 1 for n in np.diff(starts)])
        slots, rows, taken, used, full = [], [], [], 0, False
        for b in range(case["rows"]):
            n = int(starts[b + 1] - starts[b])
            held, total = -(-ctx[b] // page), -(-(ctx[b] + n) // page)
            need = total - held
            full = full or (need > 0 and used + need > len(free))
            ok = total <= table.shape[1] and not (full and need > 0)
            if ok:
                table[b, held:total] = free[used:used + need]
                used += need
            taken.append(need if ok else -1)
            slots += [int(table[b, (ctx[b] + i) // page]) * page + (ctx[b] + i) % page if ok else -1 for i in range(n)]
            rows += [b] * n
        positions = np.repeat(ctx, np.diff(starts)) + _depths(parents, starts)
        return (_dev(np.array(slots)), _dev(positions), _dev(np.array(rows)), _dev(_masks(parents, starts, r["words"])), _dev(np.array(taken)),
                _dev(table))
    if case["op"] == "store":
        hq, hkv, d, rot = case["hq"], case["hkv"], case["d"], case["rot"]
        x = r["qkv"].double().view(-1, hq + 2 * hkv, d)
        x[:, :hq + hkv] /= ((x[:, :hq + hkv] ** 2).sum(-1, keepdim=True) / d + 1e-6).sqrt()
        x[:, :hq] *= r["q_norm"].double()
        x[:, hq:hq + hkv] *= r["k_norm"].double()
        turn = torch.polar(torch.ones(len(parents), rot // 2, dtype=torch.float64, device=DEV), r["positions"].double()[:, None] * r["inv_freq"])
        head = x[:, :hq + hkv, :rot]
        z = torch.complex(head[..., 0::2].contiguous(), head[..., 1::2].contiguous()) if case["adjacent"] else \
            torch.complex(head[..., :rot // 2].contiguous(), head[..., rot // 2:].contiguous())
        z = z * turn[:, None, :]
        x[:, :hq + hkv, :rot] = torch.stack([z.real, z.imag], -1).flatten(-2) if case["adjacent"] else torch.cat([z.real, z.imag], -1)
        k, v = r["k"].double(), r["v"].double()
        k.view(-1, hkv, d)[r["slots"].long()] = x[:, hq:hq + hkv]
        v.view(-1, hkv, d)[r["slots"].long()] = x[:, hq + hkv:]
        return x[:, :hq].contiguous(), k, v
    if case["op"] == "attn":
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        table = r["table"].cpu().numpy()
        out = torch.zeros(len(parents), hq, d, dtype=torch.float64, device=DEV)
        for b in range(case["rows"]):
            lo, hi = int(starts[b]), int(starts[b + 1])
            n = hi - lo
            see = np.zeros((n, ctx[b] + n), dtype=bool)
            see[:, :ctx[b]] = True
            for i in range(n):
                j = i
                while j >= 0:
                    see[i, ctx[b] + j] = True
                    j = int(parents[lo + j])
            pages = _dev(table[b, :-(-(ctx[b] + n) // page)].astype(np.int64))
            k = r["k"][pages].reshape(-1, hkv, d)[:ctx[b] + n].double()
            v = r["v"][pages].reshape(-1, hkv, d)[:ctx[b] + n].double()
            hide = ~_dev(see)
            for h in range(hq):
                s = (r["q"][lo:hi, h].double() @ k[:, h * hkv // hq].t().contiguous()) / math.sqrt(d)
                out[lo:hi, h] = torch.softmax(s.masked_fill(hide, float("-inf")), -1) @ v[:, h * hkv // hq].contiguous()
        return out
    table, ids, picks = r["table"].cpu().numpy(), r["ids"].cpu().numpy(), r["picks"].cpu().numpy()
    length = case["nodes"] if case["nodes"] < 16 else 16
    path, got, counts = np.full((case["rows"], length), -1, dtype=np.int64), np.full((case["rows"], length), -1, dtype=np.int64), []
    k, v = r["k"].double(), r["v"].double()
    moves = []
    for b in range(case["rows"]):
        lo, hi = int(starts[b]), int(starts[b + 1])
        walk = [0]
        while len(walk) < length:
            after = [c for c in range(walk[-1] + 1, hi - lo) if parents[lo + c] == walk[-1] and ids[lo + c] == picks[lo + walk[-1]]]
            if not after:
                break
            walk.append(after[0])
        path[b, :len(walk)] = walk
        got[b, :len(walk)] = picks[lo + np.array(walk)]
        counts.append(len(walk))
        for j, node in enumerate(walk):
            a, e = ctx[b] + node, ctx[b] + j
            moves.append((int(table[b, a // page]) * page + a % page, int(table[b, e // page]) * page + e % page))
    src, dst = _dev(np.array([m[0] for m in moves])), _dev(np.array([m[1] for m in moves]))
    for cache in (k, v):
        flat = cache.view(case["layers"], -1, case["hkv"], case["d"])
        flat[:, dst] = flat[:, src]
    counts = np.array(counts)
    return _dev(path), _dev(got), _dev(counts), _dev(np.array(ctx) + counts), k, v
