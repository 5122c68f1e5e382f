"""Long contexts over a paged cache restated on the CPU in numpy, 64 bits, one row at a time: what block_attention's operators compute.  Shares no
code with the product.  Tensors come as float64 arrays of the 16-bit values (`value`); a cache layer is [pages, 2, page, kv heads, dim]."""
import numpy as np


def rotate(x, table, pos, interleave):
    """x [rows, heads, dim] turned by table[pos] [.., 2] (cos, sin), positions clamped to the table; unrounded."""
    y = x.copy()
    half = table.shape[1]
    for n, p in enumerate(np.clip(pos, 0, table.shape[0] - 1)):
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if interleave else (i, i + half)
            c, s = (np.float64(t) for t in table[p, i])
            y[n, :, a], y[n, :, b] = x[n, :, a] * c - x[n, :, b] * s, x[n, :, b] * c + x[n, :, a] * s
    return y


def step_of(x):
    """The smallest power of two, 2^-100 at least, of which 127 reach the largest finite magnitude of x."""
    x = np.abs(x[np.isfinite(x)])
    e = -100
    while x.size and x.max() > 127 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def bounds(keys):
    """keys [block, dim] -> (largest, smallest in steps: int [2, dim], step)."""
    step = step_of(keys)
    out = np.zeros((2, keys.shape[1]), np.int64)
    for d in range(keys.shape[1]):
        col = keys[:, d][~np.isnan(keys[:, d])]
        if col.size:
            out[0, d] = np.clip(np.ceil(col.max() / step), -127, 127)
            out[1, d] = np.clip(np.floor(col.min() / step), -127, 127)
    return out, step


def score(q, bound, step):
    """q [group, dim] against one block: fp32 of the sum of whole numbers, times the step."""
    a = np.clip(np.rint(np.where(np.isnan(q), 0.0, q) / step_of(q)), -127, 127)
    return np.float32(np.maximum(a * bound[0], a * bound[1]).sum()) * np.float32(step)


def select(q, all_bounds, all_steps, pages, n, block, top, first, last):
    """q [heads, dim] of a row of n tokens whose request has `pages`; all_bounds [pages, kv heads, per, 2, dim], -> [kv heads, top]."""
    h, per = all_bounds.shape[1], all_bounds.shape[2]
    group, have = q.shape[0] // h, -(-n // block)
    out = np.full((h, top), -1, np.int64)
    for g in range(h):
        if have <= top:
            out[g, :have] = np.arange(have)
            continue
        ranked = []
        for j in range(first, have - last):
            s = np.float32(-np.inf)
            if j // per < len(pages) and 0 <= pages[j // per] < all_bounds.shape[0]:
                pg = pages[j // per]
                s = score(q[g * group:(g + 1) * group], all_bounds[pg, g, j % per].astype(np.float64), all_steps[pg, g, j % per])
            ranked.append((-s, j))
        chosen = [j for _, j in sorted(ranked)[:top - first - last]]
        out[g] = sorted(list(range(first)) + chosen + list(range(have - last, have)))
    return out


def attend(q, kv, blocks, pages, n, block, scale):
    """q [heads, dim], blocks [kv heads, top] -> (out [heads, dim], bound on |out| that fp32 work may be off by, before the output's rounding)."""
    h, page, d = kv.shape[3], kv.shape[2], kv.shape[4]
    group = q.shape[0] // h
    out, off = np.zeros((q.shape[0], d)), np.zeros((q.shape[0], d))
    for g in range(h):
        tokens, seen = [], -1
        for j in blocks[g]:
            if j <= seen:
                continue
            seen = j
            for t in range(j * block, min((j + 1) * block, n)):
                if t // page < len(pages) and 0 <= pages[t // page] < kv.shape[0]:
                    tokens.append((pages[t // page], t % page))
        if not tokens:
            continue
        k = np.stack([kv[p, 0, s, g] for p, s in tokens])
        v = np.stack([kv[p, 1, s, g] for p, s in tokens])
        for i in range(g * group, (g + 1) * group):
            z = scale * (k @ q[i])
            p = np.exp(z - z.max())
            p /= p.sum()
            out[i] = p @ v
            # a score in fp32: d products summed in any order, the scale (and log2 e) on top: (d + 4) 2^-24 of the terms' magnitudes; the weights take
            # twice the largest such error (numerator and sum), 2^-21 for the exponential and its argument's rounding (8 half steps), 2^-15 for a weight
            # in 16-bit terms (two of them, a half step of a half step each, and their sum), and the sums over the tokens (T + 64) 2^-23
            err = (d + 4) * 2.0 ** -24 * abs(scale) * (np.abs(k) @ np.abs(q[i])).max() + 2.0 ** -23 * np.abs(z - z.max()).max()
            off[i] = (2 * err + 2.0 ** -21 + 2.0 ** -15 + (len(tokens) + 64) * 2.0 ** -23) * (p @ np.abs(v))
    return out, off
