"""Plain numpy form of the 4-bit cache, attention over it and draft
verification, from their definitions: one element or one row at a time, sums in
64 bits."""
import numpy as np

F = np.float32
LIMIT = F(16384)
ORDER = (0, 4, 1, 5, 2, 6, 3, 7)


def rotate(x, cos, sin, split_half):
    """x [rows, heads, hd] at the rows' cos/sin [rows, hd/2]; every fp32 step rounded."""
    a, b = (x[..., :x.shape[-1] // 2], x[..., x.shape[-1] // 2:]) if split_half else (x[..., 0::2], x[..., 1::2])
    c, s = cos[:, None], sin[:, None]
    first, second = a * c - b * s, a * s + b * c
    return np.concatenate([first, second], -1) if split_half else np.stack([first, second], -1).reshape(x.shape)


def quantise(x):
    """(codes, D, M) of fp32 x [..., hd], as the definition's fp32 steps give them."""
    with np.errstate(all="ignore"):
        x = np.clip(np.where(np.isnan(x), F(0), x), -LIMIT, LIMIT).reshape(*x.shape[:-1], -1, 32)
        lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
        D = ((hi - lo) * F(16 / 15)).astype(np.float16)
        d = D.astype(F)
        M = (lo - d).astype(np.float16)
        inv = np.where(d > 0, F(16) / d, F(0)).astype(F)
        c = np.clip(np.rint(((x - M.astype(F)) - d) * inv), 0, 15).astype(np.int64)
    return c.reshape(*c.shape[:-2], -1), D[..., 0], M[..., 0]


def value(c, D, M):
    """What codes [..., hd] stand for (float64 holds the exact sum; one rounding to fp16)."""
    c = c.reshape(*c.shape[:-1], -1, 32)
    v = D.astype(np.float64)[..., None] * (1 + c / 16) + M.astype(np.float64)[..., None]
    return v.astype(np.float16).astype(np.float64).reshape(*v.shape[:-2], -1)


def stored(x):
    return value(*quantise(x))


def put(cache, keys, head, pos, c, D, M):
    """Writes one head vector's codes into a cache's bytes [head, tile, 20 hd]."""
    hd = c.size
    groups = hd // 32
    tile = cache[head, pos // 32]
    words, halves = tile[:16 * hd].view(np.uint32), tile[16 * hd:].view(np.float16)
    p = pos % 32
    for d in range(hd):
        g, r = d // 32, d % 32
        w, i = ((p * 4 + r // 8) * groups + g, r % 8) if keys else (((g * 8 + r % 8) * 4 + p // 8) * 4 + r // 8, p % 8)
        shift = (4 * i + 2) % 32
        both = (int(words[w]) << (32 - shift) | int(words[w]) >> shift) & 0xFFFFFFFF
        both = (both & ~15) | int(c[d])
        words[w] = (both << shift | both >> (32 - shift)) & 0xFFFFFFFF
    for g in range(groups):
        at = 2 * (p * groups + g) if keys else g * 64 + p // 8 * 8 + ORDER.index(p % 8)
        halves[at], halves[at + (1 if keys else 32)] = D[g], M[g]


def attend(q, k, v, pos, scale):
    """out [rows, H, hd] of rotated q [rows, H, hd] over k, v [len, KVH, hd]; row r sees positions up to pos + r.
    Also the largest sum of |q k| scale, by which rounding errors of a score are bounded."""
    rows, heads, hd = q.shape
    out, most = np.zeros(q.shape), 0.0
    q = q.astype(np.float64)
    for r in range(rows):
        for h in range(heads):
            g = h // (heads // k.shape[1])
            kk = k[:pos + r + 1, g]
            z = kk @ q[r, h] * scale
            most = max(most, float((np.abs(kk) @ np.abs(q[r, h])).max()) * scale)
            e = np.exp(z - z.max())
            out[r, h] = (e / e.sum()) @ v[:pos + r + 1, g]
    return out, most


def verify(logits, drafts, uniforms, temperature, probs, count):
    """(accepted, next token) of one sequence."""
    k = 0
    while True:
        x = logits[k].astype(np.float64)
        m = x.max()
        if np.isnan(x).any() or not np.isfinite(m):
            return k, -1
        d = int(drafts[k]) if k < count else -1
        first = int(np.argmax(logits[k]))
        if not temperature > 0:
            if k < count and d == first:
                k += 1
                continue
            return k, first
        e = np.exp((x - m) / np.float64(temperature))
        p = e / e.sum()
        inside = 0 <= d < x.size
        if k < count and inside:
            q = 1.0 if probs is None else np.float64(probs[k, d])
            if np.float64(uniforms[k]) * q < p[d]:
                k += 1
                continue
        if k < count:
            if probs is not None:
                p = np.maximum(p - probs[k].astype(np.float64), 0)
            elif inside:
                p[d] = 0
        c = np.cumsum(p)
        over = np.nonzero((c > np.float64(uniforms[-1]) * c[-1]) & (p > 0))[0]
        if over.size:
            return k, int(over[0])
        weight = np.nonzero(p > 0)[0]
        return k, int(weight[-1]) if weight.size else first
