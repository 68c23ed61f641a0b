"""Whether attention over the paged cache counts every slot once, however a call's work is
shared out: q is 0, so all weights of a row are one power of two, and V is 0 but for a 1 in one
dimension of a slot, by a pattern of the slot's number.  A row's output is then, per
dimension, how many of its slots are marked there over how many it sees: sums of whole
numbers (below 2^24, exact in 32 bits, and at powers of two in the weights' 16) and one
division.  1 / l and its product with the sum are off by 2^-23 together (a reciprocal that is
not rounded correctly: 2^-22 allowed), an f16 output by 2^-11 more, and by 2^-25 below its
normal numbers.

The largest patterns mark a dimension in 1 of `hd` units of 32 slots: a unit lost or counted
twice at 120001 slots changes a dimension by 1 in 15; the tests without a GPU show that each
would be seen."""
import numpy as np
import pytest

import pagedref
from oi import paged

torch = pytest.importorskip("torch")

F32, F16 = 0, 1
NP = {F32: np.float32, F16: np.float16}
DT = {F32: torch.float32, F16: torch.float16}

PATTERNS = {  # the marked dimension of slot j, before the head's shift
    "unit": lambda j, hd: j // 32 % hd,
    "stretch": lambda j, hd: j // 32 // hd * 7 % hd,
    "slot": lambda j, hd: j % hd,
}


def marked(pattern, end, hd):
    return PATTERNS[pattern](np.arange(end), hd)


def counts(mark, hd, seen):
    """Per number of slots seen (rising): how many of them are marked in each dimension."""
    out, so_far, at = np.zeros((len(seen), hd)), np.zeros(hd), 0
    for i, n in enumerate(seen):
        n = max(n, 0)
        so_far = so_far + np.bincount(mark[at:n], minlength=hd)
        out[i], at = so_far, max(at, n)
    return out


def tolerance(want, t):
    return want * (2.0 ** -22 + (2.0 ** -11 if t == F16 else 0)) + (2.0 ** -25 if t == F16 else 0)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("end,hd", [(1031, 128), (9000, 256), (20000, 128), (120001, 256), (130000, 128)])
def test_a_unit_lost_or_counted_twice_is_seen(end, hd, t):
    """Mistakes planted in the plain form: each unit of 32 slots left out, and taken twice."""
    found = []
    for pattern in ("unit", "stretch"):
        mark = marked(pattern, end, hd)
        whole = counts(mark, hd, [end])[0]
        want = whole / end
        per = []
        for u in range(-(-end // 32)):
            some = np.bincount(mark[32 * u:32 * u + 32], minlength=hd)
            ok = True
            for wrong, n in ((whole - some, end - some.sum()), (whole + some, end + some.sum())):
                ok = ok and bool((np.abs(wrong / n - want) > tolerance(want, t) + 2.0 ** -11 * wrong / n * (t == F16)).any())
            per.append(ok)
        found.append(per)
    assert np.array(found).any(0).all()


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Marked:
    """Sequences whose V is a pattern, K anything finite; all other bytes NaN."""

    def __init__(self, seed, n_kv, hd, page, ends, pattern):
        rng = np.random.default_rng(seed)
        self.n_kv, self.hd, self.page, self.ends = n_kv, hd, page, ends
        each = [pagedref.pages_of(e, page) for e in ends]
        n_pages = sum(each) + 2
        self.plan = paged.Paged(n_kv, hd, n_pages, page)
        order = rng.permutation(n_pages)
        self.width = max(each) + 1
        table = rng.integers(-9, 2 * n_pages, (len(ends), self.width)).astype(np.int32)
        self.buf = torch.full((self.plan.nbytes // 2,), float("nan"), dtype=torch.float16, device="cuda")
        slots, dims, at = [], [], 0
        self.marks = []
        for i, (e, c) in enumerate(zip(ends, each)):
            table[i, :c] = order[at:at + c]
            at += c
            j = np.arange(e)
            slots.append(table[i, j // page] * page + j % page)
            self.marks.append((marked(pattern, e, hd) + 3 * i) % hd)
            dims.append(self.marks[-1])
        slots, dims = dev(np.concatenate(slots).astype(np.int64)), dev(np.concatenate(dims).astype(np.int64))
        one = n_pages * n_kv * page * hd
        k = self.buf[:one].view(n_pages, n_kv, page, hd)
        v = self.buf[one:2 * one].view(n_pages, n_kv, page // 8, hd, 8)
        for head in range(n_kv):
            p, o = slots // page, slots % page
            k[p, head, o] = 0.25 * (head + 1)
            v[p, head, o // 8, :, o % 8] = 0.0
            v[p, head, o // 8, (dims + 17 * head) % hd, o % 8] = 1.0
        self.table, self.lens = dev(table), dev(np.int32(ends))

    def check(self, which, t, heads, news):
        """news: tokens of each sequence (all alike for the tokens call)."""
        starts = np.cumsum([0] + news).tolist()
        n, row = starts[-1], heads * self.hd
        q = torch.zeros(n, row, dtype=DT[t], device="cuda")
        out = torch.full((n + 1, row), 7.0, dtype=DT[t], device="cuda")
        s = len(self.ends)
        p = lambda x: x.data_ptr()
        if which == "tokens":
            need = self.plan.tokens_workspace_bytes(heads, s, news[0])
            ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
            self.plan.tokens(p(self.buf), heads, t, p(q), s, news[0], p(self.lens), p(self.table), self.width, p(out), p(ws), need)
        else:
            need = self.plan.prompts_workspace_bytes(heads, s, n)
            ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
            sd = dev(np.int32(starts))
            self.plan.prompts(p(self.buf), heads, t, p(q), s, n, p(sd), p(self.lens), p(self.table), self.width, p(out), p(ws), need)
        torch.cuda.synchronize()
        got = out.cpu().numpy().astype(np.float64)
        assert (got[n] == 7).all()
        got = got[:n].reshape(n, heads, self.hd)
        g = heads // self.n_kv
        for i, e in enumerate(self.ends):
            a, b = starts[i], starts[i + 1]
            seen = [max(e - (b - a) + j + 1, 0) for j in range(b - a)]
            plain = counts(self.marks[i], self.hd, seen) / np.maximum(seen, 1)[:, None]
            for head in range(heads):
                want = np.roll(plain, 17 * (head // g), 1)
                err = np.abs(got[a:b, head] - want)
                bad = err > tolerance(want, t)
                assert not bad.any(), (i, head, np.argwhere(bad)[:4].tolist(), got[a:b, head][bad][:4], want[bad][:4])


TOKENS = [  # kv heads, group, head_dim, page, tokens, lengths
    (1, 1, 128, 16, 1, [20000]),
    (1, 4, 256, 64, 2, [9000]),
    (1, 1, 256, 64, 1, [120001]),
    (1, 2, 128, 64, 1, [130000, 5]),
    (2, 4, 256, 32, 1, [900, 120001, 1500]),            # a long one among short ones
    (8, 4, 128, 16, 1, [1031]),
    (1, 24, 128, 64, 1, [20000, 70]),                   # two tiles of rows a wave
    (1, 40, 128, 16, 1, [9000, 500]),                   # groups of waves
    (1, 64, 256, 32, 1, [5000]),
    (8, 2, 128, 32, 1, [17 + 41 * i for i in range(100)]),  # a border in many tiles
    (1, 1, 128, 16, 1, [(i * 37) % 700 for i in range(1500)]),
    (4, 5, 128, 64, 16, [4000, 20000, 64, 33]),         # more than 64 rows of a kv head
    (1, 8, 128, 64, 8, [130000] + [100] * 63),          # many rows of many parts
    (2, 8, 256, 32, 8, [60000] + [90] * 20),
    (1, 16, 128, 16, 2, [60000] + [40] * 600),
]


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("pattern", list(PATTERNS))
@pytest.mark.parametrize("case", TOKENS, ids=[str(c)[:60] for c in TOKENS])
def test_tokens_count_every_slot_once(case, pattern, t):
    n_kv, g, hd, page, n_q, ends = case
    Marked(len(ends) + hd, n_kv, hd, page, ends, pattern).check("tokens", t, n_kv * g, [n_q] * len(ends))


PROMPTS = [  # kv heads, group, head_dim, page, (tokens, length) of each sequence
    (1, 2, 128, 16, [(100, 20000)]),
    (1, 1, 256, 64, [(20, 120001)]),
    (2, 2, 256, 64, [(130, 9000), (1, 40), (5, 5)]),
    (1, 8, 128, 64, [(77, 20000), (19, 9000)]),
    (2, 8, 128, 16, [(301, 301), (5, 5), (17, 17), (64, 64), (128, 128), (129, 129), (33, 33), (90, 90), (250, 250)]),
    (4, 2, 128, 32, [(700, 900), (513, 1200), (1, 700), (64, 2000), (200, 200)]),  # about as many tiles as workers
    (8, 4, 128, 64, [(400, 2000), (300, 300)]),
    (1, 4, 256, 16, [(i % 5, 3 * i + i % 5) for i in range(400)]),
    (1, 3, 128, 64, [(1, 130000)]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("pattern", list(PATTERNS))
@pytest.mark.parametrize("case", PROMPTS, ids=[str(c)[:60] for c in PROMPTS])
def test_prompts_count_every_slot_once(case, pattern, t):
    n_kv, g, hd, page, seqs = case
    Marked(len(seqs) + hd, n_kv, hd, page, [e for _, e in seqs], pattern).check("prompts", t, n_kv * g, [n for n, _ in seqs])
