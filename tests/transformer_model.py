"""The transformer operators in numpy, in 64 bits and from their definitions: what the tests of the launches compare with."""
import math

import numpy as np

BLOCK = 64
LEAST = 2.0 ** -100


def scale_of(x):
    """fl32(max / 127) over the finite values; a 64-bit quotient rounds to the same 32-bit number as the exact one."""
    a = np.abs(x[np.isfinite(x)]).astype(np.float64)
    s = np.float32(a.max() / 127) if a.size else np.float32(0)
    return np.float32(0) if s < LEAST else s


def nearest(q):
    """Half away from zero, at most 127. (Quotients of 31-bit by 24-bit numbers that are no tie are further from one than 2^-40.)"""
    return np.clip(np.sign(q) * np.floor(np.abs(q) + 0.5), -127, 127).astype(np.int64)


def codes_of(x, s):
    if s == 0:
        return np.zeros(x.shape, np.int64)
    with np.errstate(invalid="ignore"):
        q = np.clip(np.where(np.isnan(x), 0, x).astype(np.float64) / np.float64(s), -1000, 1000)
    return nearest(q)


class Cache:
    """Codes and scales by page: codes[part][page] [64, heads, dim], scales[part][page][head]."""

    def __init__(self, pages, heads, dim):
        self.pages, self.heads, self.dim = pages, heads, dim
        self.codes = np.zeros((2, pages, BLOCK, heads, dim), np.int64)
        self.scales = np.zeros((2, pages, heads), np.float32)

    def page(self, table, i, block):
        if block < 0 or block >= table.shape[1] or not 0 <= table[i, block] < self.pages:
            return None
        return int(table[i, block])

    def append(self, starts, lengths, table, keys, values):
        for i in range(len(lengths)):
            n = int(starts[i + 1] - starts[i])
            first = int(lengths[i]) - n
            for block in range(max(first, 0) // BLOCK, (int(lengths[i]) - 1) // BLOCK + 1):
                page = self.page(table, i, block)
                a, b = max(first, block * BLOCK), min(int(lengths[i]), (block + 1) * BLOCK)
                if page is None or a >= b:
                    continue
                old = a - block * BLOCK
                for part, x in enumerate((keys, values)):
                    for h in range(self.heads):
                        new = x[starts[i] + a - first:starts[i] + b - first, h]
                        was = self.scales[part, page, h] if old else np.float32(0)
                        s = max(was, scale_of(new))
                        c = self.codes[part, page, :, h]
                        if s > was:
                            c[:old] = nearest(c[:old] * np.float64(was) / np.float64(s))
                        c[old:old + b - a] = codes_of(new, s)
                        self.scales[part, page, h] = s

    def tokens(self, i, table, positions):
        """(keys, values, whether it is a token of the cache) of a sequence's positions, 32-bit products code * scale."""
        out = np.zeros((2, len(positions), self.heads, self.dim), np.float32)
        there = np.zeros(len(positions), bool)
        for at, p in enumerate(positions):
            page = self.page(table, i, p // BLOCK) if p >= 0 else None
            if page is not None:
                there[at] = True
                for part in range(2):
                    out[part, at] = self.codes[part, page, p % BLOCK].astype(np.float32) * self.scales[part, page][:, None]
        return out[0], out[1], there

    def read(self, starts, lengths, table, into):
        k, v = (t.copy() for t in into)
        for i in range(len(lengths)):
            n = int(starts[i + 1] - starts[i])
            k[starts[i]:starts[i + 1]], v[starts[i]:starts[i + 1]], _ = self.tokens(i, table, np.arange(lengths[i] - n, lengths[i]))
        return k, v

    def attend(self, starts, lengths, table, q, into, *, scale=None, cap=0.0, causal=True, window=0, slopes=None, only=None):
        """The result and a bound on how far the launch may be off, see the comment at the bound. only: the (row, head) to work out."""
        out, bound = into.astype(np.float64), np.zeros(into.shape)
        heads = q.shape[1]
        group = heads // self.heads
        scale = np.float64(np.float32(self.dim ** -0.5 if scale is None else scale))
        for i in range(len(lengths)):
            n, total = int(starts[i + 1] - starts[i]), int(lengths[i])
            k, v, there = self.tokens(i, table, np.arange(total))
            j = np.arange(total)
            for r in range(n):
                if only is not None and not any((int(starts[i]) + r, h) in only for h in range(heads)):
                    continue
                p = total - n + r
                sees = there & ((j <= p) if causal else True) & ((p - j < window) if window else True) & (p >= 0)
                for h in range(heads):
                    row = starts[i] + r
                    if only is not None and (int(row), h) not in only:
                        continue
                    out[row, h] = 0
                    x = q[row, h].astype(np.float64)
                    if not sees.any():
                        continue
                    if not np.isfinite(x).all():
                        out[row, h] = np.nan
                        continue
                    kk, vv = k[sees, h // group].astype(np.float64), v[sees, h // group].astype(np.float64)
                    t = scale * (kk @ x)
                    size = np.abs(t).max()
                    # q is off by 2^-22 of its row's largest element; a score goes through five roundings of 2^-24 and is used in
                    # units of log 2; tanh is off by 2^-22
                    off = 2.0 ** -22 * abs(scale) * np.abs(x).max() * np.abs(kk).sum(1).max() + 2.0 ** -21 * size
                    if cap:
                        t = cap * np.tanh(t / cap)
                        off += 2.0 ** -21 * cap
                    if slopes is not None:
                        far = np.float64(slopes[h]) * np.abs(p - j[sees])
                        t = t - far
                        off += 2.0 ** -22 * np.abs(far).max() + 2.0 ** -22 * np.abs(t).max()
                    w = np.exp(t - t.max())
                    out[row, h] = (w @ vv) / w.sum()
                    # weights are off by that and two exponentials of 2^-22, then rounded by 2^-23 of the page's largest: 64 tokens
                    # of a page together by 2^-17 of it. Numerator and denominator: twice. Sums of 32 bits: 2^-24 for each page.
                    bound[row, h] = np.abs(vv).max() * (2 * off + 2.0 ** -16 + 2.0 ** -23 * (total / BLOCK + 8))
        return out, bound



def activate(z, act, p0=0.0):
    if act == 1:
        return np.maximum(z, 0)
    if act == 2:
        return np.where(z > 0, z, z * np.float64(np.float32(p0)))
    if act == 3:
        return np.clip(z, 0, 6)
    if act == 4:
        return 1 / (1 + np.exp(-z))
    if act == 5:
        return z * np.tanh(np.log1p(np.exp(z)))
    return z


def linear(x, weight, scale, bias, into, *, starts=None, index=None, gated=False, act=0, act_p0=0.0):
    """The result of the grouped product and a bound on how far the launch may be off."""
    y, bound = into.astype(np.float64), np.zeros(into.shape)
    rows = len(into)
    s = np.array([scale_of(r) for r in x], np.float32) if len(x) else np.zeros(0, np.float32)
    c = np.stack([codes_of(r, t) for r, t in zip(x, s)]) if len(x) else np.zeros((0, weight.shape[2]), np.int64)
    starts = [0, rows] if starts is None else starts
    for e in range(len(weight)):
        for r in range(starts[e], starts[e + 1]):
            src = r if index is None else int(index[r])
            ok = 0 <= src < len(x)
            acc = (weight[e].astype(np.int64) @ c[src]) if ok else np.zeros(weight.shape[1], np.int64)
            unit = np.float64(s[src]) * scale[e].astype(np.float64) if ok else np.zeros(weight.shape[1])
            b = bias[e].astype(np.float64) if bias is not None else 0.0
            z = acc * unit + b
            off = 4 * 2.0 ** -24 * (np.abs(acc * unit) + np.abs(b))  # the sum as a float, two products, one addition
            if gated:
                n = len(z) // 2
                g, u = z[:n], z[n:]
                sig = 1 / (1 + np.exp(-g))
                y[r] = g * sig * u
                # silu moves by at most 1.1 of what its argument does; its exponential is off by 2^-23 |g| + 2^-22, its quotient by 2^-22
                bound[r] = np.abs(u) * 1.1 * off[:n] + np.abs(g * sig) * off[n:] + np.abs(y[r]) * (2.0 ** -23 * np.abs(g) + 2.0 ** -20) + 1e-37
            else:
                y[r] = activate(z, act, act_p0)
                # the steepest activation moves by 1.1 of its argument; those with an exponential are off by 2^-23 |z| + 2^-20 themselves
                own = np.abs(y[r]) * (2.0 ** -23 * np.abs(z) + 2.0 ** -20) if act in (4, 5) else np.abs(y[r]) * 2.0 ** -24
                bound[r] = 1.1 * off + own + 1e-37
    return y, bound
