"""Plain restatement, in 64 bits and row by row, of the ops of a step that verifies drafted tokens (micro_vllm_amd.core.tree_decode).
CPU only, written from the definitions; shares no code with the library."""
import math

import torch


def parent_of(parents, start, i):
    """Parent of node i of the row that begins at `start`: an earlier node, else -1."""
    p = i - 1 if parents is None else int(parents[start + i])
    return p if 0 <= p < i else -1


def ancestors(parents, start, i):
    """Node i and its ancestors, itself first."""
    out = []
    while i >= 0:
        out.append(i)
        i = parent_of(parents, start, i)
    return out


def plan(ctx, starts, table, free, page, num_pages, parents=None):
    """(slots, positions, rows, visible [sets of nodes], taken, table) of lists; the table is a copy."""
    table = [list(r) for r in table]
    slots, positions, rows, seen, taken = [], [], [], [], []
    used, empty = 0, False
    for b, c in enumerate(ctx):
        n = starts[b + 1] - starts[b]
        held, total = -(-c // page), -(-(c + n) // page)
        need, ok = total - held, total <= len(table[b])
        if ok and need > 0:
            empty = empty or used + need > len(free)
            ok = not empty
        if ok:
            table[b][held:total] = free[used:used + need]
            used += need
        else:
            end = min(total, len(table[b]))
            table[b][held:end] = [-1] * max(0, end - held)
        taken.append(need if ok else -1)
        for i in range(n):
            up = ancestors(parents, starts[b], i)
            pg = table[b][(c + i) // page] if ok else -1
            slots.append(pg * page + (c + i) % page if 0 <= pg < num_pages else -1)
            positions.append(c + len(up) - 1)
            rows.append(b)
            seen.append(set(up))
    return slots, positions, rows, seen, taken, table


def mask_words(seen, words):
    out = torch.zeros(len(seen), words, dtype=torch.int64)
    for t, s in enumerate(seen):
        for i in s:
            bit = 1 << (i % 64)
            out[t, i // 64] |= bit - (1 << 64) if bit >> 63 else bit
    return out


def norm_rotary(qkv, heads, kv_heads, d, positions, q_norm, k_norm, eps, inv_freq, adjacent):
    """(q [T, heads, d], k, v [T, kv_heads, d]) in fp64, and for each of q and k the sum of magnitudes that an entry is formed from."""
    x = qkv.double().view(qkv.shape[0], heads + 2 * kv_heads, d)
    out = []
    for part, w in ((x[:, :heads], q_norm), (x[:, heads:heads + kv_heads], k_norm)):
        y = part.clone()
        if w is not None:
            y = y / torch.sqrt((y ** 2).mean(-1, keepdim=True) + eps) * w.double()
        size = y.abs()
        if inv_freq is not None:
            half = inv_freq.numel()
            for i in range(half):
                e0, e1 = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
                ang = positions.double() * inv_freq[i]
                c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
                a, b = y[:, :, e0].clone(), y[:, :, e1].clone()
                y[:, :, e0], y[:, :, e1] = a * c - b * s, b * c + a * s
                size[:, :, e0] = size[:, :, e1] = a.abs() + b.abs()
        out += [y, size]
    return out[0], out[2], x[:, heads + kv_heads:], out[1], out[3]


def attn(q, k_cache, v_cache, ctx, starts, table, seen, scale):
    """(o, sum p |v|, largest sum |q k| scale over the keys seen, keys seen), each per token and head; `seen`: nodes that a token sees.
    Where a place has no page its key does not count."""
    T, heads, d = q.shape
    pages, page, kv_heads, _ = k_cache.shape
    o, mag = torch.zeros(T, heads, d, dtype=torch.float64), torch.zeros(T, heads, d, dtype=torch.float64)
    size, count = torch.zeros(T, heads, dtype=torch.float64), torch.zeros(T, dtype=torch.int64)
    for b, c in enumerate(ctx):
        for t in range(starts[b], starts[b + 1]):
            places = [j for j in range(c)] + [c + i for i in sorted(seen[t])]
            where = [(table[b][j // page], j % page) for j in places if j // page < len(table[b])]
            where = [(p, s) for p, s in where if 0 <= p < pages]
            if not where:
                continue
            p, s = torch.tensor([w[0] for w in where]), torch.tensor([w[1] for w in where])
            k, v = k_cache[p, s].double(), v_cache[p, s].double()
            count[t] = len(where)
            for h in range(heads):
                kh, vh = k[:, h * kv_heads // heads], v[:, h * kv_heads // heads]
                w = torch.softmax((kh @ q[t, h].double()) * scale, 0)
                o[t, h], mag[t, h] = w @ vh, w @ vh.abs()
                size[t, h] = ((kh.abs() @ q[t, h].double().abs()) * scale).max()
    return o, mag, size, count


def attn_bound(o, mag, size, count, d, dtype):
    """How far fp32 arithmetic (and, for bf16, weights rounded to bf16) may leave the result, per entry.  A score is a sum of d products:
    off by (d + 2) 2^-24 sum |q k| scale at most, a weight by twice that relatively (its own and the denominator's), by 2^-22 for the
    exponential's argument and value; sums over the keys add count 2^-24 each for numerator and denominator; then the weight's and the
    output's own rounding."""
    u = 2.0 ** -24
    rel = 2 * ((d + 2) * u * size + 8 * u * (1 + size)) + 2 * (count[:, None] + 8) * u
    half = torch.finfo(dtype).eps / 2
    return (rel[..., None] + (half if dtype == torch.bfloat16 else 0.0)) * mag * 1.01 + half * o.abs() * 1.01 + 1e-37


def accept(tokens, picks, starts, ctx, max_path, parents=None):
    """(path, ids, counts, lens) as lists."""
    path, ids, counts, lens = [], [], [], []
    for b, c in enumerate(ctx):
        lo, n = starts[b], starts[b + 1] - starts[b]
        walk = [0] if n else []
        while walk and len(walk) < max_path:
            nxt = [i for i in range(n) if parent_of(parents, lo, i) == walk[-1] and tokens[lo + i] == picks[lo + walk[-1]]]
            if not nxt:
                break
            walk.append(nxt[0])
        path.append(walk + [-1] * (max_path - len(walk)))
        ids.append([int(picks[lo + i]) for i in walk] + [-1] * (max_path - len(walk)))
        counts.append(len(walk))
        lens.append(c + len(walk))
    return path, ids, counts, lens


def move(cache, ctx, table, path, counts):
    """cache [layers, pages, page, ...] with the path's nodes behind the cached tokens; a copy."""
    out = cache.clone()
    pages, page = cache.shape[1], cache.shape[2]

    def place(b, at):
        col = at // page
        pg = table[b][col] if col < len(table[b]) else -1
        return (pg, at % page) if 0 <= pg < pages else None

    for b, c in enumerate(ctx):
        for j in range(counts[b]):
            src, dst = place(b, c + path[b][j]), place(b, c + j)
            if src is not None and dst is not None:
                out[:, dst[0], dst[1]] = cache[:, src[0], src[1]]
    return out


def scale_of(d):
    return 1.0 / math.sqrt(d)
