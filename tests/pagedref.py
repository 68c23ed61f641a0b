"""Plain forms of the paged f16 cache's operators (include/oi.h) in numpy, request
after request, attention in 64 bits."""
import numpy as np

TOP = 65504.0


def pages_of(slots, page):
    return -(-slots // page)


def stored(x):
    """Rows as the cache holds them: rounded to nearest even, nothing infinite, no NaN."""
    x = np.nan_to_num(np.asarray(x, np.float32), nan=0.0, posinf=TOP, neginf=-TOP)
    return np.clip(x, -TOP, TOP).astype(np.float16)


class Pool:
    """A cache buffer in its parts: k [page][head][slot][dim], v [page][head][slot / 8][dim][8]."""

    def __init__(self, n_kv, hd, n_pages, page, fill):
        self.n_kv, self.hd, self.n_pages, self.page = n_kv, hd, n_pages, page
        one = n_pages * n_kv * page * hd
        self.buf = np.array(fill, np.uint8)
        f = self.buf.view(np.float16)
        self.k = f[:one].reshape(n_pages, n_kv, page, hd)
        self.v = f[one:2 * one].reshape(n_pages, n_kv, page // 8, hd, 8)

    def append(self, k, v, slots):
        k, v = stored(k), stored(v)
        for t, s in enumerate(np.asarray(slots).tolist()):
            if 0 <= s < self.n_pages * self.page:
                p, o = divmod(s, self.page)
                self.k[p, :, o] = k[t]
                self.v[p, :, o // 8, :, o % 8] = v[t]

    def request(self, row, end):
        """K and V [head][slot][dim] of slots 0 .. end - 1, float64."""
        p = np.asarray(row)[:pages_of(end, self.page)]
        k = self.k[p].transpose(1, 0, 2, 3).reshape(self.n_kv, -1, self.hd)
        v = self.v[p].transpose(1, 0, 2, 4, 3).reshape(self.n_kv, -1, self.hd)
        return k[:, :end].astype(np.float64), v[:, :end].astype(np.float64)


def plan(past, new, table, free, n_free, n_rows, page):
    """(table, n_free, lens, starts, slots, pos) after oi_paged_plan_launch."""
    table = np.array(table)
    lens, starts = [], [0]
    slots, pos = np.full(n_rows, -1, np.int32), np.zeros((3, n_rows), np.int32)
    n_free = min(max(n_free, 0), len(free))
    rows = wanted = taken = 0
    for i, (a, b) in enumerate(zip(past, new)):
        b = max(b, 0)
        r0, rows = rows, rows + b
        starts.append(min(rows, n_rows))
        held = 0
        if a >= 0 and rows <= n_rows and a + b <= table.shape[1] * page:
            have = pages_of(a, page)
            need = pages_of(a + b, page) - have
            wanted += need
            if need == 0 or wanted <= n_free:
                for k in range(need):
                    table[i, have + k] = free[n_free - 1 - taken - k]
                taken += need
                held = a + b
                for k in range(b):
                    p = table[i, (a + k) // page]
                    slots[r0 + k] = p * page + (a + k) % page if 0 <= p < len(free) else -1
                    pos[:, r0 + k] = a + k
        lens.append(held)
    return table, n_free - taken, np.array(lens, np.int32), np.array(starts, np.int32), slots, pos


def release(held, keep, table, free, n_free, page):
    """(free, n_free) after oi_paged_release_launch."""
    free = np.array(free)
    out = []
    for i, h in enumerate(held):
        h = min(max(h, 0), table.shape[1] * page)
        k = min(max(keep[i], 0), h) if keep is not None else 0
        out += [table[i, j] for j in range(pages_of(k, page), pages_of(h, page))]
    if n_free + len(out) > len(free):
        return free, n_free
    for j, p in enumerate(out):
        free[n_free + len(out) - 1 - j] = p
    return free, n_free + len(out)


def attention(q, k, v, scale):
    """q [n][heads][dim] of a request's newest tokens, k and v [kv head][slot][dim]: out in
    64 bits, the largest sum |q_d k_d| |scale| of a score, and max |v| per (head, dim)."""
    n, h, d = q.shape
    hk, end = k.shape[:2]
    g = h // hk
    out = np.zeros((n, h, d))
    size = 0.0
    top = np.abs(v).max(1) if end else np.zeros((hk, d))
    for head in range(h):
        x = q[:, head].astype(np.float64)
        s = x @ k[head // g].T * scale
        if end:
            size = max(size, float((np.abs(x) @ np.abs(k[head // g]).T).max()) * abs(scale))
        for t in range(n):
            seen = end - n + t + 1
            if seen > 0:
                p = np.exp(s[t, :seen] - s[t, :seen].max())
                out[t, head] = p @ v[head // g][:seen] / p.sum()
    return out, size, np.repeat(top, g, 0)
