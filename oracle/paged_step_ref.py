"""Plain restatements at 64 bits of the operators around a paged context: norms and rotation of
q and k with their gradients, block tables, ancestor masks and attention of drafted trees.
Test infrastructure only."""

from __future__ import annotations

import numpy as np

PAGE = 64


def norm_rope(x, w, cos, sin, *, eps, norm=True, interleaved=False):
    """x [..., T, D] rows, w broadcastable gains or None, cos/sin [T, R/2] of the rows' positions (or
    None): (y, magnitude), all float64.  magnitude bounds what a result element is made of."""
    x = np.asarray(x, np.float64)
    n = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) if norm else x.copy()
    if w is not None:
        n = n * w
    return rotate(n, cos, sin, interleaved), rotate(np.abs(n), None if cos is None else np.abs(cos),
                                                    None if sin is None else np.abs(sin), interleaved, sign=1.0)


def _pairs(r, interleaved):
    i = np.arange(r // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)


def rotate(n, cos, sin, interleaved, sign=-1.0):
    if cos is None:
        return n.copy()
    y = n.copy()
    a, b = _pairs(2 * cos.shape[-1], interleaved)
    y[..., a] = n[..., a] * cos + sign * n[..., b] * sin
    y[..., b] = n[..., b] * cos + n[..., a] * sin
    return y


def norm_rope_grads(x, w, cos, sin, dy, *, eps, norm=True, interleaved=False):
    """(dx, magnitude of dx, terms of dw, magnitudes of dw's terms): dw is the sum of its terms over
    the rows that share a gain."""
    x, dy = np.asarray(x, np.float64), np.asarray(dy, np.float64)
    g = rotate(dy, cos, None if sin is None else -sin, interleaved)
    ga = rotate(np.abs(dy), None if cos is None else np.abs(cos), None if sin is None else np.abs(sin), interleaved, 1.0)
    if not norm:
        return g, ga, None, None
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    xh = x * r
    one = 1.0 if w is None else w
    u, ua = g * one, ga * np.abs(one)
    dx = r * (u - xh * (u * xh).mean(-1, keepdims=True))
    mag = r * (ua + np.abs(xh) * (ua * np.abs(xh)).mean(-1, keepdims=True))
    return dx, mag, g * xh, ga * np.abs(xh)


def block_table(old, lens, free, table, max_pages, keep=None):
    """Request by request: (table, slots, positions, new lengths, pages taken, pages lacking,
    requests out of range)."""
    out, slots, pos, new = [], [], [], []
    at = taken = lacking = bad = 0
    for b, n in enumerate(lens):
        cap_in = 0 if table is None else min(len(table[b]), max_pages) * PAGE
        o = min(max(old[b], 0), cap_in)
        mine = [t for t in range(n) if keep is None or keep[at + t]]
        room = max_pages * PAGE - o
        bad += o != old[b] or len(mine) > room
        want = min(len(mine), room)
        have, need = -(-o // PAGE), -(-(o + want) // PAGE) - (-(-o // PAGE))
        got = max(0, min(need, len(free) - taken))
        lacking += need - got
        if got < need:
            want = max(0, min(want, (have + got) * PAGE - o))
        row = [int(x) for x in (table[b][:have] if table is not None else [])] + [int(x) for x in free[taken:taken + got]]
        taken += need
        out.append(row + [-1] * (max_pages - len(row)))
        slot = [-1] * n
        for r, t in enumerate(mine[:want]):
            a = o + r
            slot[t] = row[a // PAGE] * PAGE + a % PAGE if row[a // PAGE] >= 0 else -1
        slots += slot
        pos += [o + t for t in range(n)]
        new.append(o + want)
        at += n
    return out, slots, pos, new, taken - lacking, lacking, int(bad)


def ancestors(parents, lens):
    """[T][set of seen tokens] of packed parents (bad ones are roots)."""
    out, at = [], 0
    for n in lens:
        mine = []
        for i in range(n):
            up = parents[at + i]
            mine.append((mine[up] if 0 <= up < i else set()) | {i})
        out += mine
        at += n
    return out


def mask_words(seen, words):
    rows = []
    for s in seen:
        w = [0] * words
        for j in s:
            w[j // 64] |= 1 << (j % 64)
        rows.append([x - 2**64 if x >= 2**63 else x for x in w])
    return np.array(rows, np.int64).reshape(len(seen), words)


def tree_attention(q, k, v, seen, scale, k_ctx, v_ctx):
    """One sequence and head: q, k, v [n, D], contexts [C, D], seen [n] sets of main keys.  Returns
    (o, weighted sum of |v|, |context's part of o|, max over keys of scale * sum |q k|)."""
    n, c = q.shape[0], k_ctx.shape[0]
    keys, vals = np.concatenate([k_ctx, k]), np.concatenate([v_ctx, v])
    vis = np.zeros((n, c + k.shape[0]), bool)
    vis[:, :c] = True
    for i, s in enumerate(seen):
        vis[i, [c + j for j in s]] = True
    with np.errstate(invalid="ignore"):
        z = np.where(vis, (q @ keys.T) * scale, -np.inf)
        m = np.abs(scale) * np.where(vis, np.abs(q) @ np.abs(keys).T, 0).max(-1)
    e = np.exp(z - z.max(-1, keepdims=True))
    w = e / e.sum(-1, keepdims=True)
    o, a = np.zeros_like(q), np.zeros_like(q)
    for i in range(n):  # only what the row sees
        o[i] = w[i, vis[i]] @ vals[vis[i]]
        a[i] = w[i, vis[i]] @ np.abs(vals[vis[i]])
    return o, a, np.abs(w[:, :c] @ v_ctx), m
