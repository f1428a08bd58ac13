"""The paged 8-bit cache, attention over it and log probabilities in 64 bits, with numpy alone: what the tests compare with."""
import numpy as np

TOP = {0: 127.0, 1: 448.0}   # largest codes of int8, e4m3


def e4m3_values():
    """Values of the 256 codes: sign, four exponent bits (bias 7), three mantissa bits; no NaN."""
    u = np.arange(256)
    e, m = (u >> 3) & 15, u & 7
    mag = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    return np.where(u & 128, -mag, mag)


VALUES = {0: np.arange(256).astype(np.uint8).view(np.int8).astype(np.float64), 1: e4m3_values()}


def decode(fmt, codes, exps):
    """codes [..., block, dim], exps [...] -> values."""
    return VALUES[fmt][codes] * 2.0 ** (exps.astype(np.float64) - 127)[..., None, None]


def round_code(fmt, x):
    """The nearest value a code stands for (ties to even), of x divided by its scale."""
    x = np.clip(np.where(np.isnan(x), 0.0, x), -TOP[fmt], TOP[fmt])
    if fmt == 0:
        return np.rint(x)
    step = 2.0 ** (np.frexp(np.maximum(np.abs(x), 2.0 ** -6))[1] - 4.0)
    return np.rint(x / step) * step


def least_exponent(fmt, amax):
    """Exponent byte (at least 7) of the least power of two with amax <= top * 2^(e - 127)."""
    e = 7
    while amax > TOP[fmt] * 2.0 ** (e - 127):
        e += 1
    return min(e, 253)


def append(fmt, values, exps, rows, slots, block):
    """values [blocks, heads, block, dim] (decoded) and exps [blocks, heads], changed in place by rows [n, heads, dim]. The bytes behind a
    block's last token stay, and so stand for other values under another exponent."""
    i, n = 0, len(slots)
    while i < n:
        if slots[i] < 0:
            i += 1
            continue
        j = i + 1
        while j < n and slots[j] == slots[j - 1] + 1 and slots[j] % block:
            j += 1
        b, off = slots[i] // block, slots[i] % block
        for h in range(rows.shape[1]):
            x = rows[i:j, h].astype(np.float64)
            finite = np.abs(x[np.isfinite(x)])
            e = least_exponent(fmt, finite.max() if finite.size else 0.0)
            old = int(exps[b, h])
            e = max(e, old) if off else e
            s = 2.0 ** (e - 127.0)
            if e > old:
                values[b, h, :off] = round_code(fmt, values[b, h, :off] / s) * s
            values[b, h, off + j - i:] *= 2.0 ** (e - old)
            values[b, h, off:off + j - i] = round_code(fmt, x / s) * s
            exps[b, h] = e
        i = j


def attend(q, k, v, table, lengths, row_start, block, scale, window):
    """q [rows, heads, dim], decoded k / v [blocks, kv, block, dim] -> (y, sum p |v|, sum |q||k| scale at its largest), NaN rows where q is."""
    heads, kv = q.shape[1], k.shape[1]
    y, mag, top = np.full(q.shape, np.nan), np.zeros(q.shape), 0.0
    for r, total in enumerate(lengths):
        n = row_start[r + 1] - row_start[r]
        ids = np.array([table[r][p // block] for p in range(total)], dtype=np.int64)
        there = (ids >= 0) & (ids < k.shape[0])
        off = np.arange(total) % block
        kk, vv = k[np.where(there, ids, 0), :, off], v[np.where(there, ids, 0), :, off]   # [total, kv, dim]
        for i in range(n):
            at, p = row_start[r] + i, total - n + i
            see = there & (np.arange(total) <= p)
            if window:
                see &= p - np.arange(total) < window
            for h in range(heads):
                m = h // (heads // kv)
                if not see.any():
                    y[at, h] = 0.0
                    continue
                s = scale * (kk[see, m] @ q[at, h])
                w = np.exp(s - s.max())
                w /= w.sum()
                y[at, h] = w @ vv[see, m]
                mag[at, h] = w @ np.abs(vv[see, m])
                if np.isfinite(q[at, h]).all():
                    top = max(top, scale * (np.abs(kk[see, m]) @ np.abs(q[at, h])).max())
    return y, mag, top


def logprobs(x, tokens, top):
    x = x.astype(np.float64)
    m = x.max(1, keepdims=True)
    e = np.exp(x - m)
    l = e.sum(1, keepdims=True)
    lse = m + np.log(l)
    p = e / l
    ent = -(np.where(p > 0, p * np.where(p > 0, x - lse, 0.0), 0.0)).sum(1)
    order = np.argsort(-x, axis=1, kind="stable")[:, :top]
    return x[np.arange(len(x)), tokens] - lse[:, 0], ent, order, np.take_along_axis(x, order, 1) - lse
