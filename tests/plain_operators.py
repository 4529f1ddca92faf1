"""The operators around a draft tree in 64 bits (numpy): what tests hold the kernels to, and how far rounding may take them."""
import numpy as np

import oracle as orc

LOG2E = 1.4426950408889634
F16_HALF = 2.0 ** -11                                    # half a step of fp16, relative


def head_values(fmt, rows, n, rs, hb, h, hd):
    """Head h of n row bytes as fp64 [n, hd]."""
    b = np.ascontiguousarray(rows.reshape(-1)[:n * rs].reshape(n, rs)[:, h * hb:h * hb + orc.head_bytes(fmt, hd)])
    if fmt == orc.F16:
        return b.view(np.float16).astype(np.float64).reshape(n, hd)
    return orc.dequantize(fmt, b.reshape(-1), n * hd).astype(np.float64).reshape(n, hd)


def scales(fmt, rows, n, rs, hb, h, hd):
    b = rows.reshape(-1)[:n * rs].reshape(n, rs)[:, h * hb:h * hb + orc.head_bytes(fmt, hd)]
    blk = 34 if fmt == orc.Q8_0 else 18
    return np.ascontiguousarray(b.reshape(n, hd // 32, blk)[:, :, :2]).view(np.float16).astype(np.float64)[..., 0]


def query(fmt, q, hd):
    """The call's query rounding, fp64 [rows, hd]: f16 over f16 keys, q8_0 over quantized ones."""
    if fmt == orc.F16:
        return q.astype(np.float16).astype(np.float64)
    return orc.dequantize(orc.Q8_0, orc.quantize(orc.Q8_0, q), q.size).astype(np.float64).reshape(q.shape)


def attn_tree(shape, K, V, n, Q, n_nodes, mask):
    """(O / l, lse, tolerance of O / l, tolerance of lse) of the rows [nkv * rows] over n keys, the last n_nodes the draft's.

    Tolerances. A score is a sum over 32-blocks of dot * dk * (dq * scale): dots are exact, the row's factor a pair of fp16 that
    keeps 22 bits or, below 2^-9, an absolute 2^-25; products, sums and the shift by the maximum are fp32. So it is off by at
    most eps = 2^-19 sum |terms| + 2^-25 sum |dot dk| (f16 keys: products of fp16 in fp32, the first alone), and e^score by that
    share. O: a value enters as d * q rounded to fp16 with its probability in full, or (f16 values, and calls of up to 8 rows) a
    value in full with its probability or probability * d rounded once: half a step of fp16 of sum p |v| / l either way
    (2^-25 where what is rounded is below 2^-14: at most that times sum |v|, or |q|, over l), then the result's own half step
    (2^-25 at most below 2^-14). lse: the maximum's share of eps, the sum of fp32 probabilities
    (2^-19 covers its rounding) and the result's fp32 steps."""
    nkv, rows, hd, fmt, rs, hb = shape.nkv, shape.rows, shape.hd, shape.fmt, shape.rs, shape.hb
    O, lse = np.zeros((nkv * rows, hd)), np.full(nkv * rows, -np.inf)
    tol_o, tol_l = np.zeros((nkv * rows, hd)), np.zeros(nkv * rows)
    see = np.ones((rows, n), bool)
    for r in range(rows):
        see[r, n - n_nodes:] = [(int(mask[r % n_nodes]) >> j) & 1 for j in range(n_nodes)]
    for h in range(nkv):
        q = query(fmt, Q[h * rows:(h + 1) * rows], hd)
        k, v = head_values(fmt, K, n, rs, hb, h, hd), head_values(fmt, V, n, rs, hb, h, hd)
        any_row = see.any(0)
        k, v = np.where(any_row[:, None], k, 0.0), np.where(any_row[:, None], v, 0.0)   # what no row sees never counts
        if fmt == orc.F16:
            terms = np.abs(q) @ np.abs(k).T * shape.scale
            eps = 2.0 ** -19 * terms
        else:
            qb, kb = q.reshape(rows, -1, 32), k.reshape(n, -1, 32)
            dk = np.abs(scales(fmt, K, n, rs, hb, h, hd))
            dq = np.maximum(np.abs(qb).max(2) / 127.0, 1e-30)
            eps = np.zeros((rows, n))
            for b in range(hd // 32):
                dot = np.abs(qb[:, b] @ kb[:, b].T)
                off = 8.0 * np.abs(qb[:, b].sum(1))[:, None] * dk[None, :, b] if fmt == orc.Q4_0 else 0.0   # the nibbles' offset
                eps += 2.0 ** -19 * (dot + off) * shape.scale + 2.0 ** -25 * (dot + off) / dq[:, b][:, None]
        s = np.where(see, q @ k.T * shape.scale, -np.inf)
        eps = np.where(see, eps, 0.0)
        m = s.max(1)
        live = m > -np.inf
        p = np.exp(s[live] - m[live][:, None])
        l = p.sum(1)
        at = np.flatnonzero(live) + h * rows
        O[at] = p @ v / l[:, None]
        lse[at] = m[live] + np.log(l)
        worst = eps[live].max(1)[:, None] + 2.0 ** -18
        spread = p @ np.abs(v) / l[:, None]
        units = np.abs(v)
        if fmt != orc.F16:
            d = scales(fmt, V, n, rs, hb, h, hd)
            units = np.maximum(units, units / np.where(d != 0, np.abs(d), 1.0).repeat(32, axis=1))
        tol_o[at] = F16_HALF * spread + 2.0 ** -25 * units.sum(0) / l[:, None] + 2 * worst * spread + np.maximum(F16_HALF * (np.abs(O[at]) + 2.0 ** -9 * spread), 2.0 ** -25)
        tol_l[at] = worst[:, 0] + 2.0 ** -19 + 2.0 ** -22 * np.abs(lse[at])
    return O, lse, tol_o, tol_l


def norm_rope(x, w, eps, freq, pos, n_rot, interleaved):
    """fp64 [n, heads, hd]."""
    x = x.astype(np.float64)
    y = x if w is None else x / np.sqrt((x * x).mean(2, keepdims=True) + np.float64(np.float32(eps))) * w.astype(np.float64)
    y = y.copy()
    half = n_rot // 2
    if half == 0:
        return y
    th = pos.astype(np.float64)[:, None, None] * freq.astype(np.float64)[None, None, :half]
    c, s = np.cos(th), np.sin(th)
    a, b = (slice(0, n_rot, 2), slice(1, n_rot, 2)) if interleaved else (slice(0, half), slice(half, n_rot))
    ya, yb = y[..., a].copy(), y[..., b].copy()
    y[..., a], y[..., b] = ya * c - yb * s, ya * s + yb * c
    return y


def logprobs(x, scale, given, n_top):
    """x fp32 [rows, vocab] -> logp, lse, entropy, top ids, top log probabilities (64 bits; ids int32)."""
    rows, vocab = x.shape
    y = x.astype(np.float64) * np.float64(np.float32(scale))
    with np.errstate(all="ignore"):
        m = y.max(1)
        ms = np.where(np.isfinite(m), m, 0.0)
        ln = np.log(np.exp(y - ms[:, None]).sum(1))
        lse = ms + ln
        bad = np.isnan(y).any(1) | (m == np.inf)
        none = m == -np.inf
        lse = np.where(bad, np.nan, np.where(none, -np.inf, lse))
        lp = np.where(none[:, None], -np.inf, (y - ms[:, None]) - ln[:, None])   # (of far values lse has lost ln)
        lp[bad] = np.nan
        ent = -np.where(lp > -np.inf, np.exp(lp) * np.where(lp > -np.inf, lp, 0.0), 0.0).sum(1)
        ent = np.where(bad, np.nan, np.where(none, 0.0, ent))
        logp = np.full(given.shape, np.nan)
        ok = (given >= 0) & (given < vocab)
        logp[ok] = np.take_along_axis(lp, np.clip(given, 0, vocab - 1), 1)[ok]
        key = np.where(np.isnan(x), np.inf, x.astype(np.float64))
        order = np.lexsort((np.broadcast_to(np.arange(vocab), x.shape), -key, ~np.isnan(x)), axis=1)[:, :n_top]
    top = np.full((rows, n_top), -1, np.int32)
    top_lp = np.full((rows, n_top), -np.inf)
    k = min(n_top, vocab)
    top[:, :k] = order[:, :k]
    top_lp[:, :k] = np.take_along_axis(lp, order[:, :k], 1)
    return logp, lse, ent, top, top_lp


def random_tree(rng, n, depth=None):
    """(parents, masks): node 0 the root, node i's parent before it."""
    parent, mask = [-1], [1]
    for i in range(1, n):
        p = int(rng.integers(max(0, i - (depth or i)), i))
        parent.append(p)
        mask.append(mask[p] | 1 << i)
    return parent, np.array(mask, np.uint64)
