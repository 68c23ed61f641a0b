"""What attention over the paged cache keeps of a weight, where an output's own rounding does not
hide it.  Through oi.paged, against 64 bits; names as in test_gpu_paged_attn.py.
"""
import numpy as np
import pytest

import pagedref
from oi import paged
from test_gpu_paged_attn import F16, F32, NP, Batch, dev, host, queries

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

LOG2E = 1.4426950408889634


def exponent_error(size, hd):
    """A weight's relative error by its score and exponent (test_gpu_paged_attn.py); size: the largest sum |q_d k_d| |scale|."""
    return (2.0 ** -22 + (hd / 8 + 4) * 2.0 ** -24) * size + 2.0 ** -21 * (1.45 * size + 40)


@pytest.mark.parametrize("n_kv,g,hd,n_q", [(2, 4, 128, 16), (2, 8, 128, 16), (1, 40, 128, 2), (2, 8, 256, 16), (1, 12, 256, 10)])
def test_tokens_weights_hold_22_bits_at_any_number_of_rows(n_kv, g, hd, n_q):
    """An F16 call of at most 64 rows of a kv head and of more: V is 1 or -1 and a row sees 1 to 40
    slots, so that many outputs are small and rounded finely.  Beside that rounding (2^-11 of the
    output) a value of size 1 is off by 2 E (exponents, above and below the line), the weights'
    2^-22 and the additions' 2^-22 (end / 4 + 60), 5e-5 together; weights of 11 bits are off by up
    to 1.2e-4 for two slots."""
    ends = [16, 19, 24, 40]
    b = Batch(n_kv + g + hd + n_q, n_kv, hd, 16, ends)
    for i, e in enumerate(ends):
        slots = [int(b.table[i, j // 16]) * 16 + j % 16 for j in range(e)]
        b.ref.append(b.rng.standard_normal((e, n_kv, hd)).astype(np.float32), b.rng.choice([-1.0, 1.0], (e, n_kv, hd)), slots)
    b.buf.copy_(dev(b.ref.buf))
    q = queries(b.rng, len(ends) * n_q, n_kv * g, hd, F16, 0.3)
    got = b.tokens(n_kv * g, F16, n_q, q)
    starts = [i * n_q for i in range(len(ends) + 1)]
    for i, lo, hi, (out, size, _) in b.want(q, starts, hd ** -0.5):
        tol = 2.0 ** -11 * np.abs(out) + 2 * exponent_error(size, hd) + 2.0 ** -22 * (ends[i] / 4 + 61) + 2.0 ** -25
        err = np.abs(got[lo:hi].astype(np.float64) - out)
        assert (err <= tol).all(), (i, float((err / tol).max()))


class Sink:
    """A sequence of n + 1 slots of one kv head, `times` in a call: slot `at` has K of 1 throughout, the others 0 in
    the first half of the dimensions and 1 in the second."""

    def __init__(self, n, at, hd, page, z, v, times):
        self.n, self.hd, self.times = n, hd, times
        pages = pagedref.pages_of(n + 1, page)
        self.plan = paged.Paged(1, hd, pages, page)
        self.buf = torch.zeros(self.plan.nbytes // 2, dtype=torch.float16, device="cuda")
        one = pages * page * hd
        k, vv = self.buf[:one].view(pages, page, hd), self.buf[one:2 * one].view(pages, page // 8, hd, 8)
        self.v, self.z = np.float16(v), np.float16(z)
        vv.copy_(dev(self.v).view(1, 1, hd, 1).expand_as(vv))
        k[:, :, hd // 2:] = 1.0
        k[at // page, at % page] = 1.0
        vv[at // page, at % page // 8, :, at % 8] = dev(self.z)
        self.pages = pages
        self.table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(times, 1)
        self.lens = torch.full((times,), n + 1, dtype=torch.int32, device="cuda")

    def run(self, which, t, q, heads, scale):
        rows, times = q.shape[0], self.times
        qd = dev(q.reshape(rows, -1)).repeat(times, 1)
        out = torch.full_like(qd, 7.0)
        p = lambda x: x.data_ptr()
        if which == "tokens":
            need = self.plan.tokens_workspace_bytes(heads, times, rows)
            ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
            self.plan.tokens(p(self.buf), heads, t, p(qd), times, rows, p(self.lens), p(self.table), self.pages, p(out), p(ws), need,
                             scale=scale)
        else:
            need = self.plan.prompts_workspace_bytes(heads, times, times * rows)
            ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
            starts = torch.arange(times + 1, dtype=torch.int32, device="cuda") * rows
            self.plan.prompts(p(self.buf), heads, t, p(qd), times, times * rows, p(starts), p(self.lens), p(self.table), self.pages,
                              p(out), p(ws), need, scale=scale)
        return host(out).reshape(times, rows, heads, self.hd).astype(np.float64)


@pytest.mark.parametrize("n,times", [(700, 1), (100000, 1), (20000, 600)])
@pytest.mark.parametrize("place", ["first", "middle", "last"])
@pytest.mark.parametrize("which,t,rows,heads,hd", [
    ("tokens", F32, 1, 14, 128), ("tokens", F16, 1, 14, 128), ("tokens", F16, 2, 14, 128), ("tokens", F32, 1, 14, 256),
    ("tokens", F16, 6, 14, 128), ("tokens", F32, 6, 14, 128), ("tokens", F16, 6, 14, 256),
    ("prompts", F16, 2, 14, 128), ("prompts", F16, 2, 14, 256), ("prompts", F32, 2, 14, 128), ("prompts", F32, 2, 14, 256),
])
def test_small_weights(which, t, rows, heads, hd, place, n, times):
    """N equal slots of V = v, each 2^-x of the largest weight w0, whose V is z (0, or of v's size):
    out = (z + N w v) / (1 + N w), w = 2^-x.  Above and below the line
    * a weight of the others is off by w (rel + 2 E), rel 2^-22 or, in F16 prompts, 2^-11, or by `least` of w0 beside 2 w E,
      but at most lost (w): f16 numbers end at a step of 2^-24, so half of it over w0, which is 2^(P - 1) or more;
      the large one is off by rel;
    * sums of numbers of one sign are off by their chain's roundings, 2^-24 each.  A long sequence by itself is
      cut in 128 parts or more, 4 units more each: (n / 128 + 256) / 16 products of 16 slots in a
      chain, each of at most 16 roundings, then 4 waves and up to 512 parts; one of many may be whole, n roundings.
    (Each part has a maximum of its own, so that of many parts only one has small weights.)
    An F16 output is rounded once."""
    rng = np.random.default_rng(n + hd)
    # the rows see all slots but the last few, which are of the others
    at = {"first": 0, "middle": n // 2 + 7, "last": n - rows}[place]
    scale = 1 / (hd // 2 * LOG2E)
    xs = np.array([0.0, 3, 7.3, 11, 14.5, 17, 17.6, 20.2, 24.4, 26.7, 28.6, 31.3, 33.4, 34.6])
    base = rng.uniform(-4, 4, heads)  # of all scores
    prompts = which == "prompts" or rows * heads > 64
    if t == F16 and which == "prompts":
        rel, least = 2.0 ** -11, 2.0 ** -25 / 2.0 ** (6 - 1)
    else:
        rel, least = 2.0 ** -22, 2.0 ** -25 / 2.0 ** ((15 if not prompts else 9 if t == F16 else 12) - 1)
    chain = ((n / 128 if times == 1 else n) + 256 + 4 + 512) * 2.0 ** -24
    q = np.concatenate([np.broadcast_to(x[None, :, None], (rows, heads, hd // 2)) for x in (xs, base)], 2).astype(NP[t])
    half = hd // 2 * float(np.float32(scale * LOG2E))
    x, y = (q.astype(np.float64)[0, :, i] * half for i in (0, hd - 1))
    e = exponent_error((np.abs(x) + np.abs(y)) / LOG2E, hd)[:, None]
    for z in (np.zeros(hd), rng.uniform(-2, 2, hd)):
        v = rng.uniform(1, 2, hd) * rng.choice([-1, 1], hd)
        s = Sink(n, at, hd, 64, z, v, times)
        zz, vv, w = np.abs(s.z.astype(np.float64)), np.abs(s.v.astype(np.float64)), 2.0 ** -x[:, None]
        got = s.run(which, t, q, heads, scale)
        for j in range(rows):
            others = n - rows + 1 + j
            below = 1 + others * w
            want = (s.z.astype(np.float64) + others * w * s.v.astype(np.float64)) / below
            off = others * (np.minimum(w, w * rel + least) + 2 * e * w)
            above = off * vv + rel * zz + chain * (zz + others * w * vv)
            tol = (above + np.abs(want) * (off + rel + chain * below)) / below * 1.01
            if t == F16:
                tol = tol + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
            err = np.abs(got[:, j] - want)
            assert (err <= tol).all(), (j, [(float(a), float(b)) for a, b in zip(x, (err / tol).max((0, 2)))])
