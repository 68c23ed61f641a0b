"""Attention over the paged cache (paged_attn.hip) against the plain 64-bit form of
pagedref.py, through oi.paged.

Let A be the largest sum of |q_d k_d| * |scale| of a score, which is in natural units.
* Score: an element of an f32 q is two halves, off by 2^-22 of itself, so a score by
  2^-22 A; the products' sum has at most hd / 8 + 4 roundings one after another, 2^-24 A
  each (K, and an f16 q, are exact).
* Exponent, of size at most X = 1.45 A + 40 (the running maximum and the offset 15 in it):
  the factor scale * log2(e), the multiply-add, two sums and exp2, each 2^-24 X, below
  2^-21 X together.
* So a weight is off by E = (2^-22 + (hd / 8 + 4) 2^-24) A + 2^-21 X of itself.
  out = sum p v / sum p is off by 2 E of the largest |V| of its dimension; p's two halves
  add 2^-22 and the f32 sums, at most end / 4 + 60 additions one after another above and
  below the line, 2^-23 each.
* An f16 output is rounded once (2^-11), and f16 prompts (with them tokens of more than 64
  rows of a kv head, which go the same way) round p once (2^-11 of each
  weight, above and below the line: 2^-10).  What f16 has no numbers for is below 2^-25 of
  p, which is 2^3 or more in f16 prompts for a weight of 1, while the largest is at least a
  half: 2^-27 of it, above and below the line 2^-26 a slot.  In f32 prompts p is 2^9 or
  more: 2^-32 a slot.
"""
import numpy as np
import pytest

import pagedref
from oi import paged

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, F16 = 0, 1
NP = {F32: np.float32, F16: np.float16}


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


def tolerance(size, top, end, hd, out_type, prompts):
    x = 1.45 * size + 40
    e = (2.0 ** -22 + (hd / 8 + 4) * 2.0 ** -24) * size + 2.0 ** -21 * x
    rel = 2 * e + 2.0 ** -22 + (end / 4 + 60) * 2.0 ** -22
    if out_type == F16:
        rel += 2.0 ** -11
        if prompts:
            rel += 2.0 ** -10 + end * 2.0 ** -26
    elif prompts:
        rel += end * 2.0 ** -32
    return rel * top + (2.0 ** -24 if out_type == F16 else 1e-38)


class Batch:
    """Sequences of given lengths over a pool whose other bytes are anything, NaN among them."""

    def __init__(self, seed, n_kv, hd, page, ends, spread=1.0, extra=3):
        rng = self.rng = np.random.default_rng(seed)
        counts = [pagedref.pages_of(max(e, 0), page) for e in ends]
        self.n_pages = sum(counts) + extra
        self.n_kv, self.hd, self.page, self.ends = n_kv, hd, page, ends
        self.plan = paged.Paged(n_kv, hd, self.n_pages, page)
        fill = rng.integers(0, 256, self.plan.nbytes).astype(np.uint8)
        self.ref = pagedref.Pool(n_kv, hd, self.n_pages, page, fill)
        self.ref.buf.view(np.float16)[rng.random(self.ref.buf.size // 2) < 0.3] = np.nan
        order = rng.permutation(self.n_pages)
        self.width = max(counts + [1]) + 1
        self.table = rng.integers(-100, 10 * self.n_pages, (len(ends), self.width)).astype(np.int32)
        at = 0
        for i, (e, c) in enumerate(zip(ends, counts)):
            self.table[i, :c] = order[at:at + c]
            at += c
            if e > 0:
                slots = [self.table[i, j // page] * page + j % page for j in range(e)]
                k, v = (self.rows(e, spread) for _ in range(2))
                self.ref.append(k, v, slots)
        self.buf, self.lens, self.table_d = dev(self.ref.buf), dev(np.int32(ends)), dev(self.table)

    def rows(self, n, spread):
        x = self.rng.standard_normal((n, self.n_kv, self.hd)) * np.exp(spread * 0.5 * self.rng.standard_normal((n, 1, 1)))
        return (x * np.where(self.rng.random(self.hd) < 0.04, 5.0, 1.0)).astype(np.float32)

    def want(self, q, starts, scale):
        """Per sequence: (out, size, top) of rows starts[i] .. starts[i + 1] - 1."""
        for i, e in enumerate(self.ends):
            a, b = starts[i], starts[i + 1]
            if b > a:
                k, v = self.ref.request(self.table[i], max(e, 0))
                yield i, a, b, pagedref.attention(q[a:b], k, v, scale)

    def check(self, got, q, starts, t, prompts, scale, what=""):
        worst = 0.0
        for i, a, b, (out, size, top) in self.want(q, starts, scale):
            tol = tolerance(size, top, max(self.ends[i], 0), self.hd, t, prompts)
            err = np.abs(got[a:b].astype(np.float64) - out)
            assert np.isfinite(got[a:b]).all(), (what, i)
            bad = err > tol
            assert not bad.any(), "%s sequence %d: %d values, worst %.3g of the tolerance, at %s" % (
                what, i, bad.sum(), (err / tol).max(), np.argwhere(bad)[:3].tolist())
            worst = max(worst, float((err / tol).max()) if err.size else 0.0)
        return worst

    def workspace(self, n):
        return torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")  # f32 NaN throughout

    def tokens(self, heads, t, n_q, q, scale=None, qs=None, in_place=False, stream=None, ws=None):
        """q [n_seqs * n_q][heads][hd] of type t (numpy); rows qs elements apart."""
        n = len(self.ends) * n_q
        row = heads * self.hd
        qs = row if qs is None else qs
        wide = self.rng.standard_normal((n, qs)).astype(NP[t])
        wide[:, :row] = q.reshape(n, row)
        qd = dev(wide)
        od = qd if in_place else dev(np.full((n + 2, qs), 7.0, NP[t]))
        need = self.plan.tokens_workspace_bytes(heads, len(self.ends), n_q)
        ws = self.workspace(need) if ws is None else ws
        self.plan.tokens(self.buf.data_ptr(), heads, t, qd.data_ptr(), len(self.ends), n_q, self.lens.data_ptr(),
                         self.table_d.data_ptr(), self.width, od.data_ptr(), ws.data_ptr(), need, scale=scale, q_stride=qs,
                         out_stride=qs, stream=stream)
        got = host(od)
        if not in_place:
            assert (got[n:] == 7).all() and (got[:, row:] == 7).all(), "other memory was written"
        else:
            assert (got[:, row:] == wide[:, row:]).all()
        return got[:n, :row].reshape(n, heads, self.hd)

    def prompts(self, heads, t, starts, n_rows, q, scale=None, qs=None, in_place=False):
        row = heads * self.hd
        qs = row if qs is None else qs
        wide = self.rng.standard_normal((n_rows, qs)).astype(NP[t])
        wide[:, :row] = q.reshape(n_rows, row)
        qd, sd = dev(wide), dev(np.int32(starts))
        od = qd if in_place else dev(np.full((n_rows + 2, qs), 7.0, NP[t]))
        need = self.plan.prompts_workspace_bytes(heads, len(self.ends), n_rows)
        ws = self.workspace(need)
        self.plan.prompts(self.buf.data_ptr(), heads, t, qd.data_ptr(), len(self.ends), n_rows, sd.data_ptr(),
                          self.lens.data_ptr(), self.table_d.data_ptr(), self.width, od.data_ptr(), ws.data_ptr(), need,
                          scale=scale, q_stride=qs, out_stride=qs)
        got = host(od)
        first, last = max(starts[0], 0), min(starts[-1], n_rows)
        if in_place:
            assert (got[:, row:] == wide[:, row:]).all() and (got[last:] == wide[last:]).all() and (got[:first] == wide[:first]).all()
        else:
            assert (got[last:] == 7).all() and (got[:first] == 7).all() and (got[:, row:] == 7).all(), "other memory was written"
        return got[:n_rows, :row].reshape(n_rows, heads, self.hd)


def queries(rng, n, heads, hd, t, size=1.5):
    return (size * rng.standard_normal((n, heads, hd))).astype(NP[t])


TOKENS = [  # kv heads, group, head_dim, page, tokens, lengths
    (1, 1, 128, 16, 1, [1]),
    (1, 1, 256, 64, 1, [0]),
    (8, 4, 128, 16, 1, [1031]),
    (2, 8, 256, 64, 1, [130, 4097]),
    (8, 4, 128, 64, 1, [17, 900, 31, 32, 33, 64, 65, 1, 2500, 0, 127, 128]),
    (4, 8, 128, 32, 5, [200, 5, 3, 777, 64, 0, 1, 2048]),
    (2, 3, 128, 16, 7, [100, 37, 16, 15]),
    (1, 16, 256, 32, 16, [300, 16, 1000]),
    (1, 24, 128, 64, 1, [650, 70]),
    (2, 40, 128, 16, 3, [90, 500]),
    (2, 2, 256, 16, 2, [1, 2, 3, 4, 5, 33]),
    (1, 1, 128, 64, 1, [20000, 3]),   # long beside short: split over workers
    (1, 4, 256, 64, 2, [9000]),
    (2, 4, 128, 16, 1, list(range(0, 300))),  # more sequences than threads
    (2, 8, 256, 64, 8, [333, 7]),     # 64 rows of a kv head
    (2, 13, 128, 16, 5, [90, 2, 200, 0, 64, 5, 4]),  # 65: from here on as packed prompts
    (4, 16, 128, 32, 16, [2048, 100, 16, 15, 1]),
    (1, 9, 256, 16, 16, [1500, 31]),
]


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("case", TOKENS, ids=[str(c)[:60] for c in TOKENS])
def test_tokens(case, t):
    n_kv, g, hd, page, n_q, ends = case
    b = Batch(hd + page + n_q + len(ends), n_kv, hd, page, ends)
    h = n_kv * g
    q = queries(b.rng, len(ends) * n_q, h, hd, t)
    starts = [i * n_q for i in range(len(ends) + 1)]
    got = b.tokens(h, t, n_q, q)
    b.check(got, q, starts, t, n_q * g > 64, hd ** -0.5)
    # strided rows, in place: the same bits
    again = b.tokens(h, t, n_q, q, qs=h * hd + 24, in_place=True)
    assert (again.view(np.uint8) == got.view(np.uint8)).all()


PROMPTS = [  # kv heads, group, head_dim, page, (tokens, length) of each sequence, rows behind the last
    (1, 1, 128, 16, [(1, 1)], 0),
    (1, 1, 256, 64, [(3, 3)], 2),
    (4, 8, 128, 16, [(301, 301), (5, 5), (17, 17), (64, 64), (128, 128), (0, 0), (129, 129), (33, 33)], 3),
    (8, 4, 128, 64, [(77, 5000), (19, 3000)], 0),
    (2, 8, 256, 32, [(250, 1300), (63, 63), (1, 700), (130, 131)], 1),
    (2, 3, 128, 32, [(100, 140), (43, 43), (44, 45)], 5),
    (1, 16, 256, 16, [(9, 200), (16, 16)], 0),
    (1, 130, 128, 64, [(2, 66), (1, 400)], 0),        # more query heads than rows of a tile
    (8, 1, 128, 64, [(1000, 1000), (513, 1200)], 7),
    (1, 2, 128, 16, [(600, 6000)], 0),                # few tiles, split over workers
    (2, 4, 128, 16, [(3, 0), (10, 4), (5, 5), (70, 40), (0, 90), (4, 1)], 2),  # lengths below the tokens: rows that see nothing
    (1, 4, 128, 16, [(i % 4, i) for i in range(300)], 0),
    (1, 1, 256, 64, [(400, 9000)], 0),
]


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("case", PROMPTS, ids=[str(c)[:60] for c in PROMPTS])
def test_prompts(case, t):
    n_kv, g, hd, page, seqs, pad = case
    ends = [e for _, e in seqs]
    b = Batch(hd + page + len(ends) + 7, n_kv, hd, page, ends)
    h = n_kv * g
    starts = np.cumsum([0] + [n for n, _ in seqs]).tolist()
    n_rows = starts[-1] + pad
    q = queries(b.rng, n_rows, h, hd, t)
    got = b.prompts(h, t, starts, n_rows, q)
    b.check(got, q, starts, t, True, hd ** -0.5)
    again = b.prompts(h, t, starts, n_rows, q, qs=h * hd + 40, in_place=True)
    assert (again[:starts[-1]].view(np.uint8) == got[:starts[-1]].view(np.uint8)).all()


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("which", ["tokens", "prompts"])
def test_scales_and_sizes(which, t):
    """Negative, zero and large scales; f32 rows from 2^-100 to 2^40; weights that one slot dominates."""
    for seed, (scale, size) in enumerate([(-0.1, 1.0), (0.0, 1.0), (0.5, 4.0), (1.0, 1e-30 if t == F32 else 1e-6),
                                          (2.0 ** -45, 2.0 ** 40) if t == F32 else (2e-3, 3000.0)]):
        b = Batch(50 + seed, 2, 128, 16, [150, 33, 700], spread=2.0)
        q = queries(b.rng, 9, 8, 128, t, size)
        starts = [0, 3, 6, 9]
        if which == "tokens":
            got = b.tokens(8, t, 3, q, scale=scale)
        else:
            got = b.prompts(8, t, starts, 9, q, scale=scale)
        b.check(got, q, starts, t, which == "prompts", scale, "scale %g" % scale)


def test_rows_of_nan_and_infinity_stay_by_themselves():
    """A row of q that is not finite gives rows that are not finite, and no others."""
    for which in ("tokens", "prompts"):
        for t in (F32, F16):
            b = Batch(70, 2, 128, 32, [200, 90, 40])
            q = queries(b.rng, 12, 8, 128, t)
            q[1, 3] = np.nan
            q[4, 0, 5] = np.inf
            q[7, 7, 0] = -np.inf
            starts = [0, 4, 8, 12]
            got = b.tokens(8, t, 4, q) if which == "tokens" else b.prompts(8, t, starts, 12, q)
            bad = ~np.isfinite(got).all(-1)
            assert np.argwhere(bad).tolist() == [[1, 3], [4, 0], [7, 7]], (which, t)
            clean = np.where(bad[..., None], 0, q).astype(NP[t])
            ref = b.tokens(8, t, 4, clean) if which == "tokens" else b.prompts(8, t, starts, 12, clean)
            assert (np.where(bad[..., None], 0, got) == np.where(bad[..., None], 0, ref)).all()


def test_numbers_that_the_host_does_not_see():
    """Lengths past the table, negative ones, page ids that the pool lacks, starts outside the rows: as stated."""
    b = Batch(90, 2, 128, 16, [64, 30, 48])
    q = queries(b.rng, 3, 4, 128, F32)
    good = b.tokens(4, F32, 1, q)
    b.table_d[1, 1] = -3              # counts as the pool's last page
    b.table[1, 1] = b.n_pages - 1
    last = b.ref.k[b.n_pages - 1], b.ref.v[b.n_pages - 1]
    for x in last:
        x[...] = np.float16(0.5)
    b.buf.copy_(dev(b.ref.buf))
    b.lens[2] = -7
    b.ends = [64, 30, 0]
    got = b.tokens(4, F32, 1, q)
    b.check(got, q, [0, 1, 2, 3], F32, False, 128 ** -0.5)
    assert (got[0] == good[0]).all() and (got[2] == 0).all()
    # a length past its table row: the row's slots
    b = Batch(91, 1, 128, 16, [80, 80])
    b.lens.fill_(10 ** 9)
    full = b.width * 16
    b.table[:, 5] = b.n_pages + 9
    b.table_d.copy_(dev(b.table))
    b.table[:, 5] = b.n_pages - 1
    for x in (b.ref.k[b.n_pages - 1], b.ref.v[b.n_pages - 1]):
        x[...] = np.float16(-1.25)
    b.buf.copy_(dev(b.ref.buf))
    b.ends = [full, full]
    q = queries(b.rng, 6, 4, 128, F16)
    b.check(b.tokens(4, F16, 3, q), q, [0, 3, 6], F16, False, 128 ** -0.5)
    b.check(b.prompts(4, F16, [0, 3, 6], 6, q), q, [0, 3, 6], F16, True, 128 ** -0.5)
    q = queries(b.rng, 6, 4, 128, F16)
    got = b.prompts(4, F16, [-4, 2, 99], 6, q)
    b.check(got, q, [0, 2, 6], F16, True, 128 ** -0.5)


@pytest.mark.parametrize("which", ["tokens", "prompts"])
def test_offsets_past_32_bits(which):
    """Pages beyond 4 GiB of K (and as much V before V's)."""
    n_kv, hd, page, n_pages = 8, 256, 64, 18000
    plan = paged.Paged(n_kv, hd, n_pages, page)
    buf = torch.zeros(plan.nbytes // 2, dtype=torch.float16, device="cuda")
    small = Batch(95, n_kv, hd, page, [100, 130])
    far = np.array([n_pages - 1, 3, 9000, n_pages - 2, 16384, 5, 8191, 12000], np.int32)[:small.n_pages]
    one, o1 = n_pages * n_kv * page * hd, small.n_pages * n_kv * page * hd
    src = small.buf.view(torch.float16)
    buf[:one].view(n_pages, -1)[far] = src[:o1].view(small.n_pages, -1)
    buf[one:2 * one].view(n_pages, -1)[far] = src[o1:2 * o1].view(small.n_pages, -1)
    q = queries(small.rng, 4, 16, hd, F16)
    starts = [0, 2, 4]
    small.check(small.tokens(16, F16, 2, q) if which == "tokens" else small.prompts(16, F16, starts, 4, q), q, starts, F16,
                which == "prompts", hd ** -0.5)
    small.plan, small.buf = plan, buf
    pages = np.where((small.table >= 0) & (small.table < small.n_pages), far[np.clip(small.table, 0, small.n_pages - 1)], -1)
    small.table_d.copy_(dev(np.int32(pages)))
    got = small.tokens(16, F16, 2, q) if which == "tokens" else small.prompts(16, F16, starts, 4, q)
    small.check(got, q, starts, F16, which == "prompts", hd ** -0.5)


def test_the_same_bits_every_time_and_on_any_stream():
    b = Batch(99, 2, 128, 32, [5000, 77, 1200, 9])
    q = queries(b.rng, 4, 16, 128, F32)
    one = b.tokens(16, F32, 1, q)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        assert (b.tokens(16, F32, 1, q, stream=st.cuda_stream) == one).all()
    qs = queries(b.rng, 160, 16, 128, F16)
    two = b.prompts(16, F16, [0, 100, 140, 155, 160], 160, qs)
    for _ in range(3):
        assert (b.prompts(16, F16, [0, 100, 140, 155, 160], 160, qs) == two).all()
