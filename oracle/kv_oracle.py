"""Plain 64-bit restatement of the paged key-value cache's operators (include/rans_kv.h), on the CPU: test
infrastructure only, never imported by the package."""
from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantise(x):
    """Rows [.., dim] -> (code value indices uint8 [.., dim] with the sign in bit 3, scale bytes [.., dim / 32]), by a
    search over the grid: the nearest value, of two equally near ones the even index."""
    x = np.asarray(x, np.float64)
    blocks = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    finite = np.isfinite(blocks).all(-1)
    top = np.where(finite, np.abs(np.where(np.isfinite(blocks), blocks, 0)).max(-1), 0.0)
    e = np.where(top > 0, np.frexp(np.where(top > 0, top, 1.0))[1] - 3, -63).clip(-63, 63)
    y = np.where(finite[..., None], np.where(np.isfinite(blocks), blocks, 0.0), 0.0) / np.exp2(e)[..., None]
    dist = np.abs(np.minimum(np.abs(y), 7.0)[..., None] - GRID)        # (7 and all above saturate)
    near = dist == dist.min(-1, keepdims=True)
    order = [0, 2, 4, 6, 1, 3, 5, 7]                       # even indices win a tie
    index = np.array(order)[near[..., order].argmax(-1)]
    sign = np.where(finite[..., None], np.signbit(y), False)
    return (index + 8 * sign).astype(np.uint8).reshape(x.shape), np.where(finite, e + 127, 255).astype(np.uint8)


def pack(index):
    """Code indices [.., dim] -> the stored bytes [.., dim / 2]."""
    dim = index.shape[-1]
    out = np.zeros((*index.shape[:-1], dim // 2), np.uint8)
    for d in range(dim):
        out[..., d % 32 // 8 * (dim // 8) + d // 32 * 4 + d % 8 // 2] |= index[..., d] << (4 * (d % 2))
    return out


def values(index, scale):
    """What code indices and scale bytes stand for."""
    v = np.where(index >= 8, -1.0, 1.0) * GRID[index & 7]
    f = np.where(scale == 255, np.nan, np.exp2(scale.astype(np.float64) - 127))
    return v * np.repeat(f, 32, axis=-1)


def attend(q, k, v, scale):
    """q [heads, dim]; k, v [kv_heads, n, dim] -> out, log_sum, share per token [kv_heads, n], and per output value
    sum p |v| (the size that rounding errors are measured by)."""
    heads, dim = q.shape
    kv, n, _ = k.shape
    if n == 0:
        return np.zeros((heads, dim)), np.full(heads, -np.inf), np.zeros((kv, 0)), np.zeros((heads, dim))
    qg = q.astype(np.float64).reshape(kv, heads // kv, dim)
    s = np.einsum("hgd,hnd->hgn", qg, k.astype(np.float64)) * scale
    top = s.max(-1, keepdims=True)
    p = np.exp(s - top)
    total = p.sum(-1, keepdims=True)
    p = p / total
    out = np.einsum("hgn,hnd->hgd", p, v.astype(np.float64))
    size = np.einsum("hgn,hnd->hgd", p, np.abs(v.astype(np.float64)))
    return (out.reshape(heads, dim), (top + np.log(total)).reshape(heads), p.sum(1), size.reshape(heads, dim))


def evict_moves(weight, position, seen, budget, recent):
    """One (sequence, kv head): weight, position [n] -> list of (to, from) places."""
    n = len(weight)
    if n <= budget:
        return []

    def rank(t):
        if position[t] >= seen - recent:
            return (0, 0.0, t)
        w = float(weight[t])
        return (1, 0.0, t) if np.isnan(w) else (2, -w, t)

    kept = set(sorted(range(n), key=rank)[:budget])
    holes = [t for t in range(budget) if t not in kept]
    movers = [t for t in range(budget, n) if t in kept]
    return list(zip(holes, movers))
