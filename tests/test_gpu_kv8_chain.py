"""The operators of a layer over the 8-bit cache together, as a program uses
them, and the cases that single calls do not reach: a cache longer than 32-bit
offsets, calls in place, a prompt wide enough for the largest workgroups, an
eviction in the middle of a captured token loop.  Tolerances: those of
test_gpu_kv8.py and test_gpu_rope.py."""
import numpy as np
import pytest

import kv8ref
from oi import kv8, rope
from test_gpu_kv8 import DT, F16, F32, NP, attn, check, dev, filled, rows, same_bytes, weight_error

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [F32, F16])
def test_prompt_tokens_eviction_tokens(t):
    """Rotate, append and attend a prompt, then tokens; evict; go on at the
    positions that follow, in the slots that are left.  Every step against the
    plain forms, fed with the rotated values that the GPU made (the cache is
    compared byte for byte), the rotation with its own."""
    rng = np.random.default_rng(31 + t)
    heads, n_kv, hd, rot, sec, cap, block, keep = 8, 2, 128, 128, (24, 20, 20), 256, 32, 100
    half = rot // 2
    f = (1e6 ** (-np.arange(half) / half)).astype(np.float32)
    plan, turn = kv8.KV8(n_kv, hd, cap, block), rope.RopeAxes(heads, n_kv, hd, rot, sec, True, 1e-6)
    fill = rng.integers(0, 256, plan.nbytes).astype(np.uint8)
    ref, buf = kv8ref.Cache(n_kv, hd, cap, block, fill), dev(fill)
    spare_ref, spare = kv8ref.Cache(n_kv, hd, cap, block, fill), dev(fill)
    qn, kn = (1 + 0.1 * rng.standard_normal((2, hd))).astype(np.float32)
    wd = [dev(x) for x in (f, qn, kn)]
    mass_ref, mass = np.full((n_kv, cap), np.nan, np.float64), torch.full((n_kv, cap), float("nan"), device="cuda")
    spare_mass = torch.full((n_kv, cap), float("nan"), device="cuda")
    pos, spare_pos = (torch.zeros(n_kv, cap, dtype=torch.int32, device="cuda") for _ in "ab")
    past, at = 0, 0  # slots in use; the next position

    def step(n):
        nonlocal past, at, mass_ref
        q, k, v = (rng.standard_normal((n, h, hd)).astype(NP[t]) for h in (heads, n_kv, n_kv))
        p = np.repeat(np.arange(at, at + n, dtype=np.int32)[None], 3, 0)
        p[1:, n // 2:] += 7  # part of it is an image
        d = [dev(x) for x in (p, q, k, v)]
        turn.launch(n, d[0].data_ptr(), *(x.data_ptr() for x in wd), t, d[1].data_ptr(), d[2].data_ptr(), t,
                    d[1].data_ptr(), d[2].data_ptr())
        plan.append(buf.data_ptr(), t, d[2].data_ptr(), d[3].data_ptr(), n, past)
        out = torch.empty_like(d[1])
        ws = torch.empty(plan.attn_workspace_bytes(heads, n), dtype=torch.uint8, device="cuda")
        plan.attn(buf.data_ptr(), heads, t, d[1].data_ptr(), n, past, out.data_ptr(), ws.data_ptr(), ws.numel(),
                  mass=mass.data_ptr())
        pos[:, past:past + n] = d[0][0]
        torch.cuda.synchronize()
        gq, gk = d[1].cpu().numpy(), d[2].cpu().numpy()
        for got, x, w in ((gq, q, qn), (gk, k, kn)):
            want = kv8ref.rope(x, w, p, f, rot, sec, True, 1e-6)
            X = np.abs(want).max(-1, keepdims=True) * 2 ** 0.5
            assert np.all(np.abs(got - want) <= 2.0 ** -24 * 40 * X + (2.0 ** -11 * np.abs(want) + 2.0 ** -25) * t)
        ref.append(gk, v, past)
        same_bytes(ref, buf, "%d tokens at slot %d" % (n, past))
        want, mass_ref, A = kv8ref.attend(ref, gq, hd ** -0.5, n, past, mass_ref)
        check(out.cpu().numpy().astype(np.float64), want, A, np.abs(ref.values("v", past + n)).max(), t, past + n)
        m = mass.cpu().numpy()
        assert np.all(np.isnan(m[:, past + n:]))
        end = past + n
        tol = 2 * weight_error(A) + 2.0 ** -22 + 2.0 ** -24 * (n * heads / n_kv + 4)
        assert np.all(np.abs(m[:, :end] - mass_ref[:, :end]) <= 10 * tol * mass_ref[:, :end] + 1e-30)  # ten steps
        mass_ref = m.astype(np.float64)  # errors of one step each
        past, at = end, at + n

    step(90)
    for n in (1, 1, 5, 1):
        step(n)
    kept = torch.zeros(n_kv, keep, dtype=torch.int32, device="cuda")
    for _ in range(2):
        want = kv8ref.evict(ref, mass_ref.astype(np.float32), past, min(keep, past - 3), 4, 20, spare_ref)
        n_keep = want.shape[1]
        kept = torch.zeros(n_kv, n_keep, dtype=torch.int32, device="cuda")
        plan.evict(buf.data_ptr(), mass.data_ptr(), pos.data_ptr(), past, n_keep, 4, 20, plan, spare.data_ptr(),
                   spare_mass.data_ptr(), spare_pos.data_ptr(), kept.data_ptr())
        torch.cuda.synchronize()
        assert np.array_equal(kept.cpu().numpy(), want)
        same_bytes(spare_ref, spare, "after eviction")
        h = np.arange(n_kv)[:, None]
        assert torch.equal(spare_pos[:, :n_keep], pos[dev(h), kept.long()])
        m = np.full((n_kv, cap), np.nan)
        m[:, :n_keep] = mass_ref[h, want]
        assert np.array_equal(spare_mass.cpu().numpy()[:, :n_keep], m[:, :n_keep].astype(np.float32))
        # the caches change places; the spare's old content is what the next eviction overwrites
        ref, spare_ref, buf, spare, mass, spare_mass, pos, spare_pos = \
            spare_ref, ref, spare, buf, spare_mass, mass, spare_pos, pos
        mass[:, n_keep:] = float("nan")
        mass_ref, past = m, n_keep
        for n in (1, 30, 2):
            step(n)


def test_offsets_past_32_bits():
    """Two kv heads of 2^23 + 64 slots of 256 dimensions: K alone passes 2^32
    bytes.  All slots are zero (their scores 0) but a few at the far end."""
    n_kv, hd, cap, heads = 2, 256, (1 << 23) + 64, 2
    plan = kv8.KV8(n_kv, hd, cap, 64)
    assert plan.nbytes > 1 << 33
    buf = torch.zeros(plan.nbytes, dtype=torch.uint8, device="cuda")
    small = kv8ref.Cache(n_kv, hd, 128, 64)  # the last 128 slots
    rng = np.random.default_rng(41)
    past, n = cap - 70, 69
    k, v = rows(rng, n, n_kv, hd, F32), rows(rng, n, n_kv, hd, F32)
    small.append(k, v, 128 - 70)
    kd, vd = dev(k), dev(v)
    plan.append(buf.data_ptr(), F32, kd.data_ptr(), vd.data_ptr(), n, past)
    got = [torch.empty(n_kv, 127, hd, device="cuda") for _ in "kv"]
    plan.read(buf.data_ptr(), cap - 128, 127, F32, got[0].data_ptr(), got[1].data_ptr())
    torch.cuda.synchronize()
    for which, g in zip("kv", got):
        assert np.array_equal(g.cpu().numpy(), small.values(which, 127).astype(np.float32)), which
    end = past + n
    assert not bool(buf[:past // 64 * 64 * hd].any()) and not bool(buf[cap * hd:(cap + past // 64 * 64) * hd].any())
    # one token and a prompt: the zero slots add exp(0) each and nothing to the sum
    for m in (1, 66):
        q = (3 * rng.standard_normal((m, heads, hd))).astype(np.float32)
        mass = torch.zeros(n_kv, cap, device="cuda")
        want = np.empty((m, heads, hd))
        first = np.empty((m, heads))
        for i in range(m):
            seen = 58 + n - m + i + 1  # of the last 128
            for h in range(heads):
                s = small.values("k", seen)[h] @ np.float64(q[i, h]) / 16.0
                w = np.exp(s)
                total = w.sum() + (cap - 128)
                want[i, h] = w @ small.values("v", seen)[h] / total
                first[i, h] = 1 / total
        out = attn(plan, buf, q, m, end - m, F32, mass=mass)
        A = float(np.max([np.max(np.abs(np.float64(q[:, h])) @ np.abs(small.values("k", 127)[h]).T / 16.0)
                          for h in range(heads)]))
        err = np.abs(out - want).max() / np.abs(small.values("v", 127)).max()
        # sums over 2^17 units, spread over 64 waves or more; 2^-24 of the whole each, above and below the line
        assert err <= 2 * weight_error(A) + 2.0 ** -22 + 2.0 ** -23 * (end / 64 / 64 + 100), err
        got_first = mass[:, 0].cpu().numpy()
        assert np.allclose(got_first, first.sum(0), rtol=1e-3), (got_first, first.sum(0))
        assert abs(float(mass.double().sum()) - m * heads) < 1e-3 * m * heads
        assert not bool(mass[:, end:].any())
        del mass
    # eviction from it: the slots with a mass above the others', and the ends
    mass = torch.zeros(n_kv, cap, device="cuda")
    mass[0, cap - 100] = 2.0
    mass[1, 77] = 3.0
    dplan = kv8.KV8(n_kv, hd, 64, 64)
    dbuf, dmass = torch.zeros(dplan.nbytes, dtype=torch.uint8, device="cuda"), torch.zeros(n_kv, 64, device="cuda")
    kept = torch.zeros(n_kv, 40, dtype=torch.int32, device="cuda")
    plan.evict(buf.data_ptr(), mass.data_ptr(), None, end, 40, 2, 30, dplan, dbuf.data_ptr(), dmass.data_ptr(), None,
               kept.data_ptr())
    torch.cuda.synchronize()
    tail = list(range(end - 30, end))
    assert kept[0].tolist() == list(range(9)) + [cap - 100] + tail
    assert kept[1].tolist() == list(range(9)) + [77] + tail
    o = [torch.empty(n_kv, 40, hd, device="cuda") for _ in "kv"]
    dplan.read(dbuf.data_ptr(), 0, 40, F32, o[0].data_ptr(), o[1].data_ptr())
    for which, g in zip("kv", o):
        full = small.values(which, 127)
        x = np.concatenate([np.zeros((n_kv, 10, hd)), full[:, 97:]], 1)
        x[0, 9] = full[0, 28]
        step = [2.0 ** kv8ref.exponent(np.abs(x[h]).max()) for h in range(n_kv)]
        want = np.stack([np.rint(x[h] / step[h]) * step[h] for h in range(n_kv)])
        assert np.array_equal(g.cpu().numpy(), want.astype(np.float32)), which


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("hd,n,past", [(128, 1, 300), (256, 7, 40), (128, 150, 20), (256, 150, 700)])
def test_attn_in_place(t, hd, n, past):
    rng = np.random.default_rng(51 + n)
    plan, ref, buf = filled(rng, 2, hd, 1024, 32, past + n)
    q = rng.standard_normal((n, 8, hd)).astype(NP[t])
    want = attn(plan, buf, q, n, past, t)
    x = dev(q)
    ws = torch.empty(plan.attn_workspace_bytes(8, n), dtype=torch.uint8, device="cuda")
    plan.attn(buf.data_ptr(), 8, t, x.data_ptr(), n, past, x.data_ptr(), ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    assert np.array_equal(x.cpu().numpy().astype(np.float64), want)


@pytest.mark.parametrize("t", [F32, F16])
def test_wide_prompt(t):
    """8160 rows of each of 8 kv heads: the largest workgroups, one split."""
    rng = np.random.default_rng(61)
    n, past, heads, n_kv = 2040, 13, 32, 8
    plan, ref, buf = filled(rng, n_kv, 128, 2112, 64, past + n)
    q = rng.standard_normal((n, heads, 128)).astype(NP[t])
    mass0 = np.zeros((n_kv, 2112), np.float32)
    mass = dev(mass0)
    want, wmass, A = kv8ref.attend(ref, q, 128 ** -0.5, n, past, mass0)
    got = attn(plan, buf, q, n, past, t, mass=mass)
    check(got, want, A, np.abs(ref.values("v", past + n)).max(), t, past + n)
    tol = 2 * weight_error(A) + 2.0 ** -22 + 2.0 ** -24 * (n * 4 + 4)
    m = mass.cpu().numpy()
    assert np.all(np.abs(m - wmass) <= tol * wmass + 1e-30)


def test_mass_of_far_slots_is_not_rounded_away():
    """A token over 30000 equal slots adds 1 / 30000 to each, relative error of a
    weight's, whatever the row's maximum and sum are."""
    plan = kv8.KV8(1, 128, 30016, 64)
    ref = kv8ref.Cache(1, 128, 30016, 64)
    ref.ke[:] = 0
    ref.kc[:, :, 0] = 100
    q = np.zeros((1, 3, 128), np.float32)
    q[0, :, 0] = [0.5, -0.25, 0.0]  # scores of 50, -25 and 0
    mass = torch.full((1, 30016), float("nan"), device="cuda")
    attn(plan, dev(ref.buf), q, 1, 29999, F32, mass=mass, scale=1.0)
    m = mass.cpu().numpy()[0]
    assert np.isnan(m[30000:]).all() and np.isnan(m[:29999]).all() and abs(m[29999] * 30000 / 3 - 1) < 1e-5
    mass.zero_()
    attn(plan, dev(ref.buf), q, 1, 29999, F32, mass=mass, scale=1.0)
    m = mass.cpu().numpy()[0, :30000].astype(np.float64)
    assert np.all(np.abs(m * 30000 / 3 - 1) <= weight_error(50.0) + 2.0 ** -23 * (30000 / 64 + 40))


def test_captured_eviction():
    """Append, attend and evict in one captured graph, replayed with eager calls
    between: each replay equals the eager result."""
    rng = np.random.default_rng(71)
    plan, ref, buf = filled(rng, 2, 128, 256, 16, 200)
    dplan = kv8.KV8(2, 128, 128, 16)
    q, k, v = (dev(rng.standard_normal((1, h, 128)).astype(np.float32)) for h in (8, 2, 2))
    ws = torch.empty(plan.attn_workspace_bytes(8, 1), dtype=torch.uint8, device="cuda")
    start, mass0 = buf.clone(), torch.rand(2, 256, device="cuda")
    mass, out = mass0.clone(), torch.empty_like(q)
    dbuf = torch.zeros(dplan.nbytes, dtype=torch.uint8, device="cuda")
    dmass, kept = torch.zeros(2, 128, device="cuda"), torch.zeros(2, 128, dtype=torch.int32, device="cuda")

    def run():
        st = torch.cuda.current_stream().cuda_stream
        plan.append(buf.data_ptr(), F32, k.data_ptr(), v.data_ptr(), 1, 200, stream=st)
        plan.attn(buf.data_ptr(), 8, F32, q.data_ptr(), 1, 200, out.data_ptr(), ws.data_ptr(), ws.numel(),
                  mass=mass.data_ptr(), stream=st)
        plan.evict(buf.data_ptr(), mass.data_ptr(), None, 201, 128, 4, 32, dplan, dbuf.data_ptr(), dmass.data_ptr(),
                   None, kept.data_ptr(), stream=st)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run()
    for i in range(5):
        q.normal_()
        k.normal_()
        results = []
        for how in (g.replay, run):
            buf.copy_(start)
            mass.copy_(mass0)
            dbuf.zero_()
            how()
            torch.cuda.synchronize()
            results.append([x.clone() for x in (buf, mass, out, dbuf, dmass, kept)])
        assert all(torch.equal(a, b) for a, b in zip(*results)), i


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("n_heads,n_kv,hd,block,n,past", [
    (8, 1, 128, 16, 90, 37),      # 720 rows, five and a half workgroups' tiles
    (7, 1, 128, 64, 75, 0),       # 525 rows of groups of 7, nothing before them
    (16, 2, 128, 32, 65, 1000),   # splits that the first rows see whole and the last in part
    (8, 1, 256, 16, 66, 200),
    (12, 2, 256, 64, 100, 0),
    (16, 1, 256, 32, 40, 1500),
    (513, 1, 128, 64, 1, 100),    # one token of more heads than go by sixteen
    (6, 6, 128, 32, 530, 3),      # no sharing
])
def test_many_rows(t, n_heads, n_kv, hd, block, n, past):
    """More than 512 rows of a kv head: the prompt kernel in each of its forms,
    with the mass, host and device length (other splits)."""
    rng = np.random.default_rng(n_heads + n + past)
    end, cap = past + n, (past + n + 63) // 64 * 64 + 640
    plan, ref, buf = filled(rng, n_kv, hd, cap, block, end)
    q = (1.5 * rng.standard_normal((n, n_heads, hd))).astype(NP[t])
    mass0 = rng.random((n_kv, cap)).astype(np.float32)
    mass0[:, past:] = np.nan
    want, wmass, A = kv8ref.attend(ref, q, hd ** -0.5, n, past, mass0)
    vmax = np.abs(ref.values("v", end)).max()
    plain = attn(plan, buf, q, n, past, t)
    check(plain, want, A, vmax, t, end)
    pd = torch.tensor([past], dtype=torch.int32, device="cuda")
    for dev_past in (None, pd):
        mass = dev(mass0)
        got = attn(plan, buf, q, n, past if dev_past is None else -9, t, mass=mass, past_dev=dev_past, pad=8)
        check(got, want, A, vmax, t, end)
        m = mass.cpu().numpy().astype(np.float64)
        assert np.all(np.isnan(m[:, end:]))
        added = wmass[:, :end] - np.where(np.arange(end) < past, mass0[:, :end].astype(np.float64), 0)
        tol = 2 * weight_error(A) + 2.0 ** -22 + 2.0 ** -24 * (n * n_heads / n_kv + 4)
        assert np.all(np.abs(m[:, :end] - wmass[:, :end]) <= tol * added + 2.0 ** -23 * wmass[:, :end] + 1e-30)
    same_bytes(ref, buf)


@pytest.mark.parametrize("t", [F32, F16])
def test_many_rows_extremes(t):
    """Rows of zero, of infinity and of NaN, blocks of very different size, a
    negative scale: in the prompt kernel."""
    rng = np.random.default_rng(81)
    n, heads, past = 70, 8, 150
    plan, ref, _ = filled(rng, 1, 128, 256, 16, 220)
    ref.ve[0] = rng.integers(-14, 7, ref.ve.shape[1])
    ref.ke[0] = rng.integers(-12, -4, ref.ke.shape[1])
    buf = dev(ref.buf)
    q = rng.standard_normal((n, heads, 128)).astype(NP[t])
    q[0] = 0
    q[1] *= NP[t](1e-6)
    q[2] *= NP[t](100)
    clean = q.copy()
    q[3, 0, 7] = np.inf
    q[4, 1, 9] = np.nan
    want, _, A = kv8ref.attend(ref, clean, -0.1, n, past)
    got = attn(plan, buf, q, n, past, t, scale=-0.1)
    assert np.all(np.isnan(got[4, 1])) and not np.any(np.isfinite(got[3, 0]))
    ok = np.ones((n, heads), bool)
    ok[3, 0] = ok[4, 1] = False
    check(got[ok], want[ok], A, np.abs(ref.values("v", 220)).max(), t, 220)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("n", [1, 300])
def test_one_projection_in_place(t, n):
    """q, k and v in the rows of one projection: rotated where they lie, appended and
    attended from there, the result back over q.  Bit for bit as from buffers of
    their own."""
    rng = np.random.default_rng(71 + n)
    heads, n_kv, hd, past = 4, 2, 128, 40
    plan, turn = kv8.KV8(n_kv, hd, 384, 32), rope.RopeAxes(heads, n_kv, hd, 64, (12, 10, 10), False, 1e-6)
    a, b = heads * hd, (heads + n_kv) * hd
    row = b + n_kv * hd
    x = rng.standard_normal((n, row)).astype(NP[t])
    fill = rng.integers(0, 256, plan.nbytes).astype(np.uint8)
    kv0 = dev(rng.standard_normal((2, past, n_kv, hd)).astype(NP[t]))
    pos = dev(np.stack([np.arange(n), np.arange(n) // 7, np.arange(n) % 7]).astype(np.int32) + past)
    f, w = dev((1e4 ** (-np.arange(32) / 32)).astype(np.float32)), dev((1 + 0.1 * rng.standard_normal((2, hd))).astype(np.float32))
    ws = torch.empty(plan.attn_workspace_bytes(heads, n), dtype=torch.uint8, device="cuda")

    def run(q, k, v, qs, ks, vs, out):
        buf = dev(fill)
        plan.append(buf.data_ptr(), t, kv0[0].data_ptr(), kv0[1].data_ptr(), past, 0)
        turn.launch(n, pos.data_ptr(), f.data_ptr(), w[0].data_ptr(), w[1].data_ptr(), t, q, k, t, q, k, q_stride=qs,
                    k_stride=ks, q_out_stride=qs, k_out_stride=ks)
        plan.append(buf.data_ptr(), t, k, v, n, past, k_stride=ks, v_stride=vs)
        plan.attn(buf.data_ptr(), heads, t, q, n, past, out, ws.data_ptr(), ws.numel(), q_stride=qs, out_stride=qs)
        torch.cuda.synchronize()
        return buf.cpu().numpy()

    one = dev(x)
    p, es = one.data_ptr(), one.element_size()
    got = run(p, p + a * es, p + b * es, row, row, row, p)
    q, k, v = (dev(np.ascontiguousarray(x[:, i:j])) for i, j in ((0, a), (a, b), (b, row)))
    out = torch.empty_like(q)
    want = run(q.data_ptr(), k.data_ptr(), v.data_ptr(), a, b - a, b - a, out.data_ptr())
    assert np.array_equal(got, want)
    assert torch.equal(one[:, :a], out) and torch.equal(one[:, a:b], k) and torch.equal(one[:, b:], v)


@pytest.mark.parametrize("t", [F32, F16])
def test_stated_workspace_is_enough_where_rows_are_split(t):
    """A prompt whose mass splits its rows at this length and at the capacity does not."""
    rng = np.random.default_rng(81 + t)
    heads, n_kv, hd, cap, n, past = 8, 8, 128, 5632, 1664, 1024
    plan, ref, buf = filled(rng, n_kv, hd, cap, 64, past + n)
    q = rng.standard_normal((n, heads, hd)).astype(NP[t])
    mass0 = np.zeros((n_kv, cap), np.float32)
    mass = dev(mass0)
    want, wmass, A = kv8ref.attend(ref, q, hd ** -0.5, n, past, mass0)
    got = attn(plan, buf, q, n, past, t, mass=mass)
    check(got, want, A, np.abs(ref.values("v", past + n)).max(), t, past + n)
    tol = 2 * weight_error(A) + 2.0 ** -22 + 2.0 ** -24 * (n + 4)
    m = mass.cpu().numpy()
    assert np.all(np.abs(m - wmass) <= tol * wmass + 1e-30)
