"""The text operators (rotary positions, attention over a paged cache, linears
on 4-bit weights) in 64 bits, from their formulas, and the batches that their
tests share. No GPU and nothing of the library in here."""
import math

import numpy as np

D = 128
NONE = 0xFFFFFFFF  # no page
HALF_STEP = 2.0 ** -8  # bf16: half a step, relative


def bf16(x):
    """Bit patterns of x rounded to nearest even."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where((u & 0x7FFFFFFF) > 0x7F800000, np.uint16(0x7FC0), r).astype(np.uint16)


def f64(bits):
    return (np.asarray(bits, np.uint32) << 16).view(np.float32).astype(np.float64)


def normal(rng, *shape, std=1.0, mean=0.0):
    """bf16 bit patterns"""
    return bf16(rng.standard_normal(shape) * std + mean)


def close(got, want, tol):
    """Bit patterns against 64-bit values: infinities and NaN in the same
    places, the rest within tol (an array)."""
    g = f64(got)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(g), np.isnan(want))
    assert np.array_equal(g[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    off = np.abs(g - np.where(fine, want, 0.0))[fine]
    tol = np.broadcast_to(tol, want.shape)[fine]
    worst = np.argmax(off - tol) if off.size else 0
    assert (off <= tol).all(), (off[worst], tol[worst], want[fine][worst], (off > tol).sum(), off.size)


class Batch:
    """Sequences of past + new tokens in pages dealt in a shuffled order."""

    def __init__(self, rng, past, new, kv_heads, page=16, spare=2, pad_front=0, pad_back=0,
                 holes=(), head_dim=D, fill=None, shared=False):
        self.past, self.new, self.kv, self.page = list(past), list(new), kv_heads, page
        self.lengths = np.array([max(p + n, 0) for p, n in zip(past, new)], np.uint32)
        used = [-(-int(n) // page) for n in self.lengths]
        self.pages, self.ld = sum(used) + spare, max(max(used), 1) + 1
        order = rng.permutation(self.pages)
        self.table = np.full((len(used), self.ld), NONE, np.uint32)
        at = 0
        for i, n in enumerate(used):
            self.table[i, :n] = order[at:at + n]
            at += n
        for s, e in holes:
            self.table[s, e] = NONE if (s + e) % 2 else self.pages  # either is no page
        self.starts = (pad_front + np.concatenate([[0], np.cumsum(new)])).astype(np.uint32)
        self.rows = int(self.starts[-1]) + pad_back
        shape = (self.pages, page, kv_heads, head_dim)
        self.k, self.v = normal(rng, *shape), normal(rng, *shape)
        if fill is not None:  # what no token lies in
            free = np.ones((self.pages, page), bool)
            for i, n in enumerate(self.lengths):
                for t in range(int(n)):
                    if self.table[i, t // page] < self.pages:
                        free[self.table[i, t // page], t % page] = False
            self.k[free], self.v[free] = fill, fill

    def slots(self, s):
        """(token, page, slot) of each token of sequence s that is stored"""
        t = np.arange(int(self.lengths[s]))
        page = self.table[s, t // self.page]
        t = t[page < self.pages]
        return t, self.table[s, t // self.page], t % self.page


def attention(b, q, out, scale, window=0):
    """(the result in 64 bits over out's own values, a bound of the error):
    probabilities rounded to bf16 in numerator and denominator move a result by
    half a step of the mean distance from it; scores are sums of 128 products in
    fp32 and the exponential's argument is rounded to fp32, 1e-4 of that mean
    covers both at the tests' scores (below 100); the store rounds once."""
    rows, heads, _ = q.shape
    want, tol = f64(out), np.zeros(out.shape)
    G = heads // b.kv
    for s in range(len(b.new)):
        t, page, slot = b.slots(s)
        k, v = f64(b.k[page, slot]), f64(b.v[page, slot])
        for i in range(b.new[s]):
            r, p = int(b.starts[s]) + i, int(b.lengths[s]) - b.new[s] + i
            see = (t <= p) & ((t > p - window) if window else True)
            if not see.any():
                want[r] = 0.0
                continue
            for h in range(heads):
                kk, vv = k[see, h // G], v[see, h // G]
                score = kk @ f64(q[r, h]) * scale
                w = np.exp(score - score.max())
                w /= w.sum()
                with np.errstate(invalid="ignore"):
                    want[r, h] = w @ vv
                    off = w @ np.abs(vv - want[r, h])
                tol[r, h] = HALF_STEP * np.abs(want[r, h]) + (1.01 * HALF_STEP + 1e-4) * off + 1e-30
    return want, tol


def frequencies(n, base, scaling="plain", factor=1.0, original=0.0, low=0.0, high=0.0):
    """(radians a position of each pair, attention factor)"""
    f = []
    for i in range(n // 2):
        x = base ** (-2.0 * i / n)
        if scaling == "linear":
            x /= factor
        elif scaling == "ntk":
            x = (base * factor ** (n / (n - 2))) ** (-2.0 * i / n)
        elif scaling == "parts":
            keep = min(1.0, max(0.0, (original * x / (2 * math.pi) - low) / (high - low)))
            x = keep * x + (1 - keep) * x / factor
        elif scaling == "yarn":
            at = [n / 2 * math.log(original / (t * 2 * math.pi), base) for t in (high, low)]
            lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), n - 1)
            keep = 1 - min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            x = keep * x + (1 - keep) * x / factor
        f.append(x)
    return np.array(f), 0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0


def rotary(x, positions, freq, factor, layout, norm=None, eps=1e-6):
    """(x [rows, heads, dim] as bit patterns turned, a bound of the error). In
    fp32: the sines are 2e-7 off, a product and a sum round three times
    (2^-24), the norm's sum and reciprocal root take 1e-6: 2e-6 of the two
    values' magnitudes; the store rounds once."""
    x = f64(x)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * f64(norm)
    n = 2 * len(freq)
    angle = np.asarray(positions, np.float64)[:, None] * freq
    c, s = factor * np.cos(angle)[:, None], factor * np.sin(angle)[:, None]
    y, size = x.copy(), np.abs(x)
    a, b = (x[..., :n // 2], x[..., n // 2:n]) if layout == "half" else (x[..., 0:n:2], x[..., 1:n:2])
    u, v = a * c - b * s, a * s + b * c
    m = factor * (np.abs(a) + np.abs(b))
    if layout == "half":
        y[..., :n], size[..., :n] = np.concatenate([u, v], -1), np.concatenate([m, m], -1)
    else:
        y[..., 0:n:2], y[..., 1:n:2], size[..., 0:n:2], size[..., 1:n:2] = u, v, m, m
    return y, HALF_STEP * np.abs(y) + 2e-6 * size + 1e-38


def linear4(x, weight, scales, zeros, group, bias=None):
    """(x W^T + bias, a bound of the error). A group's sum of (128 + q) x goes
    through four or fewer MFMA of 32 products, 40 roundings of 2^-24 of at
    most sum 143 |x| s, and what it is reduced by through as many; a row's sum
    over its groups adds a rounding each of a partial sum below the same; the
    store rounds once."""
    q = np.stack([weight & 15, weight >> 4], -1).reshape(weight.shape[0], -1, group).astype(np.float64)
    z = f64(zeros)[..., None] if zeros is not None else 8.0
    s = f64(scales)[..., None]
    w = ((q - z) * s).reshape(weight.shape[0], -1)
    xv = f64(x)
    y = xv @ w.T + (f64(bias) if bias is not None else 0.0)
    size = np.abs(xv) @ np.repeat(f64(scales), group, 1).T * 143
    return y, HALF_STEP * np.abs(y) + 80 * 2.0 ** -24 * size + 1e-38
