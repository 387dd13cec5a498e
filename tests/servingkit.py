"""Sampling, adapters and the 8-bit cache in plain numpy, 64 bits, one row, token or sequence at a time; shares nothing with the product."""
import numpy as np

BLOCK = 64


def sample(row, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.0):
    """(token, log probability) of one row of float32 logits."""
    row = np.where(np.isnan(row), -np.inf, np.asarray(row, np.float32)).astype(np.float64)
    t = float(np.float32(temperature))
    top = row.max()
    if top == -np.inf:
        return -1, np.nan
    if not t > 0:
        return int(np.argmax(row)), 0.0
    order = np.lexsort((np.arange(row.size), -row))
    with np.errstate(invalid="ignore", over="ignore"):
        w = (row == top).astype(np.float64) if np.isinf(top) else np.exp(np.where(row == -np.inf, -np.inf, (row - top) / t))
    if np.isinf(t) and not np.isinf(top):
        w = np.where(row == -np.inf, 0.0, 1.0)
    if 0 < top_k < row.size:
        order = order[:top_k]
    p = float(np.float32(top_p))
    if p < 1:
        mass = np.cumsum(w[order].astype(np.longdouble))
        order = order[:int(np.searchsorted(mass, max(p, 0.0) * mass[-1], side="left")) + 1]
    least = float(np.float32(min_p))
    if least > 0:
        order = order[w[order] >= min(least, 1.0)]
    order = np.sort(order[w[order] > 0])
    mass = np.cumsum(w[order].astype(np.longdouble))
    at = min(int(np.searchsorted(mass, float(np.float32(u)) * mass[-1], side="right")), order.size - 1)
    return int(order[at]), float(np.log(w[order[at]] / mass[-1]))


def quantize(block):
    """A block [64, dim] of one head: codes and the largest value, by float64 quotient and product, halves away from zero."""
    top = np.abs(block).max()
    if not np.isfinite(top):
        return np.zeros(block.shape, np.int64), np.nan
    if top == 0:
        return np.zeros(block.shape, np.int64), top
    r = block.astype(np.float64) * (np.float64(127.0) / np.float64(top))
    return np.clip(np.sign(r) * np.floor(np.abs(r) + 0.5), -128, 127).astype(np.int64), top


def held(rows, exact=True):
    """Rows [positions, heads, dim] of one sequence as the cache holds them.  exact: codes times scale in 64 bits, else in float32."""
    kind = np.float64 if exact else np.float32
    out = rows.astype(kind)
    for b in range(0, rows.shape[0] - BLOCK + 1, BLOCK):
        for h in range(rows.shape[1]):
            codes, top = quantize(rows[b:b + BLOCK, h])
            out[b:b + BLOCK, h] = codes.astype(kind) * (kind(top) / kind(127))
    return out


def attend(q, k, v, first, scale=None):
    """q [rows, heads, dim] at positions first ..., k and v [positions, kv heads, dim] as they are held: result and what float32 arithmetic
    may be off by: scores by the query's rounding (2^-24 of its largest value against the row of keys), by three float32 roundings and the
    exponential's argument (2^-22 of the score), weights by 2^-23, the weighted sum by 2^-22 for every tile of 64."""
    rows, heads, dim = q.shape
    group = heads // k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    out, tol = np.empty(q.shape), np.empty(q.shape)
    for j in range(rows):
        n = first + j + 1
        for h in range(heads):
            kk, vv, qq = k[:n, h // group], v[:n, h // group], q[j, h].astype(np.float64)
            with np.errstate(invalid="ignore"):
                s = kk @ qq * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[j, h] = w @ vv
                off = 2.0 ** -24 * np.abs(qq).max() * np.abs(kk).sum(1).max() * scale + 2.0 ** -22 * (np.abs(s).max() + 1)
                tol[j, h] = (2 * off + 2.0 ** -22 * (n / 64 + 4)) * np.abs(vv).max()
    return out, tol


def adapter(x, down, up, scale, base):
    """One token: result, and what float32 sums of exact products may be off by: 2^-23 a link, for as many links as a CTA's warp may add up."""
    x, d, u = x.astype(np.float64), down.astype(np.float64), up.astype(np.float64)
    h = d @ x
    links = 6 * (-(-x.size // 128)) + 24
    off_h = links * 2.0 ** -23 * (np.abs(d) @ np.abs(x))
    links_u = 6 * (-(-d.shape[0] // 16)) + 4
    off = abs(scale) * (np.abs(u) @ off_h + links_u * 2.0 ** -23 * (np.abs(u) @ np.abs(h)))
    y = scale * (u @ h)
    y = y if base is None else y + base.astype(np.float64)
    return y, off + 2.0 ** -23 * np.abs(y) + 1e-30
