"""Pages given and taken back, slots of packed rows and the append to the paged cache
(paged.hip) against the plain forms of pagedref.py, through oi.paged.  All are exact
by definition: whole numbers, and values rounded once."""
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


class State:
    """The pool's state on the device, with borders of other numbers around every array."""

    def __init__(self, table, free, n_free, n_pages, page):
        self.plan = paged.Paged(2, 128, n_pages, page)
        self.page, self.width = page, table.shape[1]
        self.table, self.free, self.n_free = dev(np.int32(table)), dev(np.int32(free)), dev(np.int32([n_free, 77]))

    def step(self, past, new, n_rows, pos=True):
        n = len(past)
        self.past, self.new = dev(np.int32(past)), dev(np.int32(new))
        out = [torch.full((k + 3,), 12345, dtype=torch.int32, device="cuda") for k in (n, n + 1, n_rows, 3 * n_rows)]
        self.plan.plan(n, self.past.data_ptr(), self.new.data_ptr(), self.table.data_ptr(), self.width,
                       self.free.data_ptr(), self.n_free.data_ptr(), n_rows, *[x.data_ptr() for x in out[:3]],
                       out[3].data_ptr() if pos else None)
        got = [host(x) for x in out]
        for x, k in zip(got, (n, n + 1, n_rows, 3 * n_rows if pos else 0)):
            assert (x[k:] == 12345).all(), "numbers behind an array were written"
        return got[0][:n], got[1][:n + 1], got[2][:n_rows], got[3][:3 * n_rows].reshape(3, n_rows)


def pool(rng, past, page, width, n_pages):
    """Tables for sequences that hold past slots; the rest of the pages on the list."""
    order = rng.permutation(n_pages)
    table, at = rng.integers(-5, 5 * n_pages, (len(past), width)), 0
    for i, x in enumerate(past):
        k = pagedref.pages_of(max(x, 0), page)
        if k <= width:
            table[i, :k] = order[at:at + k]
            at += k
    free = np.concatenate([order[at:], rng.integers(0, n_pages, at)])
    return table, free, n_pages - at


CASES = [  # sequences, page, past up to, new up to, table entries, pages beyond those held, rows beyond those asked for
    (1, 16, 0, 1, 1, 1, 0),
    (1, 64, 1000, 3, 20, 2, 5),
    (5, 16, 40, 20, 6, 100, 3),
    (61, 32, 300, 1, 12, 61, 0),
    (64, 16, 64, 17, 8, 30, 7),        # the list runs out in the middle
    (200, 64, 500, 90, 10, 40, 100),   # and among many pages
    (1024, 16, 33, 2, 4, 1024, 0),
    (1025, 16, 33, 5, 4, 900, 11),     # more sequences than threads
    (2500, 32, 70, 3, 4, 700, -500),   # the rows run out
    (3, 16, 100, 6000, 400, 1200, 9),  # two launches
    (300, 64, 700, 180, 16, 500, 64),
    (2100, 16, 20, 9, 4, 5000, -900),
    (7, 32, 50, 0, 3, 5, 0),           # nothing to do
]


@pytest.mark.parametrize("case", CASES, ids=[str(c) for c in CASES])
def test_plan_and_release(case):
    n, page, past_hi, new_hi, width, spare, rows_more = case
    rng = np.random.default_rng(sum(case))
    past = rng.integers(0, past_hi + 1, n)
    new = rng.integers(0, new_hi + 1, n)
    new[rng.integers(0, n)] = new_hi
    if n > 50:  # numbers that the pool does not serve
        past[3], new[5], past[7] = -4, -9, width * page - 1 if new[7] > 1 else past[7]
    n_pages = int(sum(pagedref.pages_of(max(x, 0), page) for x in past)) + spare
    n_rows = max(0, int(np.maximum(new, 0).sum()) + rows_more)
    table, free, n_free = pool(rng, past, page, width, n_pages)
    # pages that a served sequence holds are the pool's, but for one
    if n > 2 and past[2] > page:
        table[2, 0] = n_pages
    s = State(table, free, n_free, n_pages, page)
    want = pagedref.plan(past, new, table, free, n_free, n_rows, page)
    got = s.step(past, new, n_rows, pos=n % 2 == 1)
    assert (host(s.table) == want[0]).all()
    assert host(s.n_free).tolist() == [want[1], 77]
    assert (got[0] == want[2]).all() and (got[1] == want[3]).all() and (got[2] == want[4]).all()
    if n % 2 == 1:
        assert (got[3] == want[5]).all()
    assert (host(s.free) == free).all()
    # what was taken goes back to where it was
    lens = dev(got[0])
    keep = dev(np.minimum(np.int32(past), got[0]))
    s.plan.release(n, lens.data_ptr(), keep.data_ptr(), s.table.data_ptr(), width, s.free.data_ptr(), s.n_free.data_ptr())
    assert host(s.n_free).tolist() == [n_free, 77] and (host(s.free) == free).all()
    # sequences end, each or in part
    for part in (False, True):
        held = got[0]
        k = rng.integers(-2, past_hi + 3, n).astype(np.int32) if part else None
        f0, c0 = host(s.free).copy(), int(host(s.n_free)[0])
        wf, wc = pagedref.release(held, k, want[0], f0, c0, page)
        kd = dev(k) if part else None
        s.plan.release(n, lens.data_ptr(), kd.data_ptr() if part else None, s.table.data_ptr(), width, s.free.data_ptr(),
                       s.n_free.data_ptr())
        assert host(s.n_free).tolist() == [wc, 77] and (host(s.free)[:wc] == wf[:wc]).all(), part
        s.free.copy_(dev(np.int32(free)))
        s.n_free[0] = n_free


def test_release_of_more_pages_than_the_pool_has():
    rng = np.random.default_rng(3)
    table = rng.integers(0, 20, (4, 8))
    free = np.arange(20)
    s = State(table, free, 5, 20, 16)
    held = dev(np.int32([64, 64, 64, 65]))  # 17 pages beside 5
    s.plan.release(4, held.data_ptr(), None, s.table.data_ptr(), 8, s.free.data_ptr(), s.n_free.data_ptr())
    assert host(s.n_free).tolist() == [5, 77] and (host(s.free) == free).all()
    held[3] = 40  # 15 of them
    s.plan.release(4, held.data_ptr(), None, s.table.data_ptr(), 8, s.free.data_ptr(), s.n_free.data_ptr())
    assert host(s.n_free).tolist() == [20, 77]
    wf, _ = pagedref.release([64, 64, 64, 40], None, table, free, 5, 16)
    assert (host(s.free) == wf).all()


def test_a_captured_step_goes_by_the_numbers_that_it_finds():
    """Decode steps replayed: lengths, tables and the list move on from replay to replay."""
    rng = np.random.default_rng(8)
    n, page, width, n_pages = 9, 16, 12, 80
    past = rng.integers(1, 60, n)
    table, free, n_free = pool(rng, past, page, width, n_pages)
    s = State(table, free, n_free, n_pages, page)
    past_d, new_d = dev(np.int32(past)), dev(np.ones(n, np.int32))
    lens, starts, slots = (torch.zeros(k, dtype=torch.int32, device="cuda") for k in (n, n + 1, n))
    pos = torch.zeros(3, n, dtype=torch.int32, device="cuda")
    st = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()

    def step():
        s.plan.plan(n, past_d.data_ptr(), new_d.data_ptr(), s.table.data_ptr(), width, s.free.data_ptr(),
                    s.n_free.data_ptr(), n, lens.data_ptr(), starts.data_ptr(), slots.data_ptr(), pos.data_ptr(),
                    stream=torch.cuda.current_stream().cuda_stream)
        past_d.copy_(lens)
    with torch.cuda.graph(g, stream=st):
        step()
    for i in range(40):
        table, n_free, want_lens, want_starts, want_slots, want_pos = pagedref.plan(past, [1] * n, table, free, n_free, n, page)
        g.replay()
        assert (host(s.table) == table).all() and host(s.n_free)[0] == n_free, i
        assert (host(lens) == want_lens).all() and (host(slots) == want_slots).all() and (host(pos) == want_pos).all()
        assert (host(starts) == want_starts).all()
        past = want_lens


# ----------------------------------------------------------------- append --

def rows(rng, n, n_kv, hd, t, special):
    x = (rng.standard_normal((n, n_kv, hd)) * np.exp(2 * rng.standard_normal((n, 1, 1)))).astype(np.float32)
    if special:
        flat = x.reshape(-1)
        at = rng.choice(flat.size, 12, replace=False)
        flat[at] = [np.nan, np.inf, -np.inf, 65504, 65519.9, 65520, -7e4, 1e30, 2.0 ** -25, 2.0 ** -24, 6e-8, -0.0]
    with np.errstate(over="ignore"):
        return x.astype(NP[t])


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("n_kv,hd,page,news", [
    (1, 128, 16, [1]),
    (8, 128, 64, [1] * 13),
    (2, 256, 32, [5, 1, 40, 0, 17, 8, 3]),
    (3, 128, 16, [100, 7, 9, 64]),
    (5, 256, 64, [33, 2]),
    (16, 128, 32, [20, 20, 1, 1, 1, 90]),
    (8, 128, 64, [300, 5, 1, 1, 40]),  # more rows than one a workgroup
    (2, 256, 16, [1] * 270),
    (1, 256, 32, [9, 400, 0, 7]),
])
def test_append(t, n_kv, hd, page, news):
    rng = np.random.default_rng(n_kv * hd + page + len(news) + t)
    past = rng.integers(0, 3 * page, len(news))
    n_pages = int(sum(pagedref.pages_of(a + b, page) for a, b in zip(past, news))) + 2
    width = max(pagedref.pages_of(a + b, page) for a, b in zip(past, news))
    table, free, n_free = pool(rng, past, page, width, n_pages)
    n = sum(news) + 5
    slots = pagedref.plan(past, news, table, free, n_free, n, page)[4]
    slots[-2:] = [n_pages * page, -7]  # numbers that the pool does not have
    plan = paged.Paged(n_kv, hd, n_pages, page)
    fill = rng.integers(0, 256, plan.nbytes).astype(np.uint8)
    ref = pagedref.Pool(n_kv, hd, n_pages, page, fill)
    k, v = rows(rng, n, n_kv, hd, t, True), rows(rng, n, n_kv, hd, t, True)
    ref.append(k, v, slots)
    buf, kd, vd, sd = dev(fill), dev(k), dev(v), dev(np.int32(slots))
    plan.append(buf.data_ptr(), t, kd.data_ptr(), vd.data_ptr(), n, sd.data_ptr())
    assert (host(buf) == ref.buf).all()
    # the same rows beside others in wider ones, in no order
    wide = rng.standard_normal((n, 24 + 2 * n_kv * hd)).astype(NP[t])
    order = rng.permutation(n)
    wide[:, 8:8 + n_kv * hd] = k.reshape(n, -1)[order]
    wide[:, 16 + n_kv * hd:16 + 2 * n_kv * hd] = v.reshape(n, -1)[order]
    buf, w, sd = dev(fill), dev(wide), dev(np.int32(slots[order]))
    size = NP[t]().itemsize
    plan.append(buf.data_ptr(), t, w.data_ptr() + 8 * size, w.data_ptr() + (16 + n_kv * hd) * size, n, sd.data_ptr(),
                k_stride=wide.shape[1], v_stride=wide.shape[1])
    assert (host(buf) == ref.buf).all()


def test_append_past_32_bits():
    """A pool of 9 GiB: bytes from slot to slot pass 2^32, elements of V 2^32 too."""
    n_kv, hd, page, n_pages = 8, 256, 64, 18000
    plan = paged.Paged(n_kv, hd, n_pages, page)
    assert plan.nbytes > 2 ** 33
    buf = torch.zeros(plan.nbytes // 2, dtype=torch.float16, device="cuda")
    one = n_pages * n_kv * page * hd
    rng = np.random.default_rng(1)
    slots = np.array([n_pages * page - 1] + list(range(n_pages * page // 2, n_pages * page // 2 + 16)) + [3], np.int32)
    n = len(slots)
    k, v = rows(rng, n, n_kv, hd, F32, False), rows(rng, n, n_kv, hd, F32, False)
    kd, vd, sd = dev(k), dev(v), dev(slots)
    plan.append(buf.data_ptr(), F32, kd.data_ptr(), vd.data_ptr(), n, sd.data_ptr())
    kp = buf[:one].view(n_pages, n_kv, page, hd)
    vp = buf[one:2 * one].view(n_pages, n_kv, page // 8, hd, 8)
    for t, s in enumerate(slots.tolist()):
        p, o = divmod(s, page)
        assert (host(kp[p, :, o]) == pagedref.stored(k[t])).all() and (host(vp[p, :, o // 8, :, o % 8]) == pagedref.stored(v[t])).all(), s
    used = sorted({s // page for s in slots.tolist()})
    assert int(torch.count_nonzero(kp).item()) == int(torch.count_nonzero(kp[used]).item()) == np.count_nonzero(pagedref.stored(k))
    assert int(torch.count_nonzero(vp).item()) == np.count_nonzero(pagedref.stored(v))
