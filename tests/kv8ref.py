"""Plain 64-bit forms of the 8-bit K/V cache, of attention over it, of eviction
and of the three-axis rotation, on the CPU (numpy), for the tests of oi_kv8_*
and oi_rope_axes_launch.  The cache is simulated byte for byte, in one buffer of
the layout of include/oi.h."""
import numpy as np

EMIN, EMAX = -24, 10


def exponent(amax):
    """The least e in [EMIN, EMAX] with amax <= 127 * 2^e, off a list of all."""
    for e in range(EMIN, EMAX):
        if amax <= 127.0 * 2.0 ** e:
            return e
    return EMAX


class Cache:
    """A cache buffer; fill: bytes that it holds before anything is stored."""

    def __init__(self, n_kv, hd, cap, block, fill=None):
        self.n_kv, self.hd, self.cap, self.block = n_kv, hd, cap, block
        n, m = n_kv * cap * hd, n_kv * cap // block
        size = (2 * n + 2 * m + 255) // 256 * 256
        self.buf = np.zeros(size, np.uint8) if fill is None else fill[:size].copy()
        b = self.buf.view(np.int8)
        self.kc = b[:n].reshape(n_kv, cap, hd)
        self.vc = b[n:2 * n].reshape(n_kv, cap // 64, hd, 64)
        self.ke = b[2 * n:2 * n + m].reshape(n_kv, cap // block)
        self.ve = b[2 * n + m:2 * n + 2 * m].reshape(n_kv, cap // block)

    def get(self, which, h, s):
        return self.kc[h, s] if which == "k" else self.vc[h, s // 64, :, s % 64]

    def put(self, which, h, s, codes):
        if which == "k":
            self.kc[h, s] = codes
        else:
            self.vc[h, s // 64, :, s % 64] = codes

    def exps(self, which):
        return self.ke if which == "k" else self.ve

    def exp(self, which, h, b):
        """A block's exponent; a byte outside the format's range counts as the nearest in it."""
        return min(max(int(self.exps(which)[h, b]), EMIN), EMAX)

    def values(self, which, n):
        """Slots 0..n-1 as float64 [n_kv][n][hd]."""
        codes = self.kc[:, :n] if which == "k" else \
            self.vc.transpose(0, 1, 3, 2).reshape(self.n_kv, self.cap, self.hd)[:, :n]
        e = np.repeat(self.exps(which).clip(EMIN, EMAX), self.block, 1)[:, :n, None]
        return codes.astype(np.float64) * 2.0 ** e.astype(np.float64)

    def append(self, k, v, past):
        """k, v [n][n_kv][hd] behind `past` slots."""
        n = k.shape[0]
        for which, x in (("k", k), ("v", v)):
            x = x.astype(np.float64)
            for h in range(self.n_kv):
                for b in range(past // self.block, (past + n - 1) // self.block + 1):
                    s0, s1 = b * self.block, (b + 1) * self.block
                    a, z = max(s0, past), min(s1, past + n)
                    rows = x[a - past:z - past, h]
                    finite = np.abs(rows[np.isfinite(rows)])
                    e = exponent(finite.max() if finite.size else 0.0)
                    if s0 < past:
                        old = self.exp(which, h, b)
                        e = max(e, old)
                        if e > old:
                            for s in range(s0, past):
                                c = self.get(which, h, s).astype(np.float64)
                                self.put(which, h, s, np.rint(c * 2.0 ** (old - e)))
                    self.exps(which)[h, b] = e
                    with np.errstate(invalid="ignore"):
                        c = np.clip(np.rint(rows * 2.0 ** -e), -127, 127)
                    c = np.where(np.isnan(rows), 0, c)
                    for s in range(a, z):
                        self.put(which, h, s, c[s - a])


def attend(c, q, scale, n, past, mass=None):
    """(out [n][n_heads][hd], mass after the call, A): A is the largest sum of
    |q_d k_d| * scale of a score, which error bounds go by."""
    n_heads, hd = q.shape[1], q.shape[2]
    g, end = n_heads // c.n_kv, past + n
    out = np.empty((n, n_heads, hd))
    m = None if mass is None else mass.astype(np.float64).copy()
    if m is not None:
        m[:, past:end] = 0
    seen = np.arange(end) <= past + np.arange(n)[:, None]
    K, V = c.values("k", end), c.values("v", end)
    A = 0.0
    for h in range(n_heads):
        kv = h // g
        x = np.float64(q[:, h])
        s = x @ K[kv].T * scale
        A = max(A, float(np.where(seen, np.abs(x) @ np.abs(K[kv]).T * abs(scale), 0).max()))
        s = np.where(seen, s, -np.inf)
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[:, h] = p @ V[kv]
        if m is not None:
            m[kv, :end] += p.sum(0)
    return out, m, A


def evict(c, mass, n, keep, first, last, dst):
    """Fills dst (a Cache); returns kept [n_kv][keep]."""
    kept = np.empty((c.n_kv, keep), np.int32)
    for h in range(c.n_kv):
        key = mass[h, :n].astype(np.float64)
        key = np.where(np.isnan(key), -np.inf, key)
        nan_last = np.isnan(mass[h, :n])
        middle = sorted(range(first, n - last), key=lambda s: (nan_last[s], -key[s], s))[:keep - first - last]
        kept[h] = sorted(list(range(first)) + middle + list(range(n - last, n)))
        for which in "kv":
            for b in range((keep + dst.block - 1) // dst.block):
                slots = kept[h, b * dst.block:(b + 1) * dst.block]
                x = [c.get(which, h, s).astype(np.float64) * 2.0 ** c.exp(which, h, s // c.block) for s in slots]
                e = exponent(np.abs(x).max())
                dst.exps(which)[h, b] = e
                for i, r in enumerate(x):
                    dst.put(which, h, b * dst.block + i, np.rint(r * 2.0 ** -e))
    return kept


def axis_of(i, sections, interleaved):
    if interleaved:
        return i % 3 if i < 3 * sections[i % 3] else 0
    return 0 if i < sections[0] else 1 if i < sections[0] + sections[1] else 2


def rope(x, w, pos, inv_freq, rotary, sections, interleaved, eps):
    """x [n][heads][hd] float64-able, w [hd] or None, pos [3][n]."""
    x = np.float64(x)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.float64(w)
    half = rotary // 2
    y = x.copy()
    for i in range(half):
        ang = pos[axis_of(i, sections, interleaved)].astype(np.float64) * float(inv_freq[i])
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
        y[..., i] = x[..., i] * c - x[..., i + half] * s
        y[..., i + half] = x[..., i] * s + x[..., i + half] * c
    return y
