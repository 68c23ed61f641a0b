"""The 8-bit K/V cache on the GPU (kv8.hip, kv8_attn.hip) against the plain
64-bit forms of kv8ref.py, through oi.kv8.

Append, read and evict are exact by definition (a power-of-two step, one
rounding half to even), so whole buffers are compared byte for byte, with
arbitrary bytes beforehand: what a call does not own has to stay.

Attention.  Let A be the largest sum of |q_d k_d| * |scale| of a score, which is
in natural units.
* Score: an element of an f32 q is two halves, off by 2^-22 of itself (2^-11 of
  a remainder of 2^-11), so a score by 2^-22 A; the products' sum has at most
  hd / 8 + 4 roundings one after another, 2^-24 A each (K's bytes, and an f16 q,
  are exact).
* Exponent, of size at most X = 1.45 A + 40 (the running maximum, V's exponent
  and the offset 15 in it): the factor scale * log2(e), the multiply-add, two
  sums and exp2, each 2^-24 X, below 2^-21 X together.
* So a weight is off by E = (2^-22 + (hd / 8 + 4) 2^-24) A + 2^-21 X of itself.
  out = sum p v / sum p is off by 2 E of the largest |V|; p's two halves add 2^-22
  and the f32 sums, at most end / 64 + 40 additions one after another above and
  below the line, 2^-23 each.
* An f16 call rounds p once (2^-11 of the largest |V|) and its output once (2^-11).
The mass of a slot is a sum of weights with two exponents' errors (the score's and
the row's log-sum's) and n * group additions of 2^-24.
"""
import numpy as np
import pytest

import kv8ref
from oi import _native, kv8

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, F16 = 0, 1
DT = {F32: torch.float32, F16: torch.float16}
NP = {F32: np.float32, F16: np.float16}


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def rows(rng, n, n_kv, hd, t):
    """Rows whose sizes differ from token to token, some dimensions larger."""
    x = rng.standard_normal((n, n_kv, hd)) * np.exp(rng.standard_normal((n, 1, 1)))
    x *= np.where(rng.random(hd) < 0.05, 6.0, 1.0)
    return x.astype(NP[t])


def noise(rng, plan):
    """A buffer's former content: any bytes."""
    return rng.integers(0, 256, plan.nbytes).astype(np.uint8)


def both(rng, n_kv, hd, cap, block):
    plan = kv8.KV8(n_kv, hd, cap, block)
    fill = noise(rng, plan)
    return plan, kv8ref.Cache(n_kv, hd, cap, block, fill), dev(fill)


def same_bytes(ref, buf, what=""):
    torch.cuda.synchronize()
    got = buf.cpu().numpy()
    bad = np.nonzero(got != ref.buf)[0]
    assert bad.size == 0, "%s: %d bytes differ, the first at %d of %d (K codes end at %d, V at %d)" % (
        what, bad.size, bad[0], got.size, ref.kc.size, 2 * ref.kc.size)


# ----------------------------------------------------------------- append --

@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("n_kv,hd,block,calls", [
    (1, 128, 16, [1, 1, 14, 1, 30, 17]),
    (2, 128, 32, [1, 31, 1, 64, 3, 90]),
    (3, 256, 64, [5, 58, 1, 1, 63, 65, 2]),
    (2, 256, 16, [130, 1, 7]),
    (8, 128, 64, [1] * 9 + [120]),
])
def test_append(t, n_kv, hd, block, calls):
    rng = np.random.default_rng(len(calls) * 100 + hd + block + t)
    cap = (sum(calls) + 63) // 64 * 64 + 64
    plan, ref, buf = both(rng, n_kv, hd, cap, block)
    past = 0
    for i, n in enumerate(calls):
        with np.errstate(over="ignore"):  # the last calls of an f16 case hold infinities
            k, v = rows(rng, n, n_kv, hd, t), rows(rng, n, n_kv, hd, t) * NP[t](0.1 * 3 ** i)
        ref.append(k, v, past)
        kd, vd = dev(k), dev(v)
        plan.append(buf.data_ptr(), t, kd.data_ptr(), vd.data_ptr(), n, past)
        past += n
        same_bytes(ref, buf, "call %d of %d tokens" % (i, n))


def test_append_overwrites_a_rejected_draft():
    rng = np.random.default_rng(5)
    plan, ref, buf = both(rng, 2, 128, 192, 32)
    for n, past in [(70, 0), (6, 70), (4, 72), (9, 60), (1, 64), (128, 64)]:
        k, v = rows(rng, n, 2, 128, F32), rows(rng, n, 2, 128, F32)
        ref.append(k, v, past)
        kd, vd = dev(k), dev(v)
        plan.append(buf.data_ptr(), F32, kd.data_ptr(), vd.data_ptr(), n, past)
        same_bytes(ref, buf, "%d at %d" % (n, past))


def test_append_strided_rows_of_a_fused_projection():
    rng = np.random.default_rng(6)
    n, n_kv, hd = 37, 2, 128
    for t in (F32, F16):
        plan, ref, buf = both(rng, n_kv, hd, 128, 64)
        wide = rng.standard_normal((n, 8 + 2 * n_kv * hd + 24)).astype(NP[t])
        k = wide[:, 8:8 + n_kv * hd].reshape(n, n_kv, hd)
        v = wide[:, 8 + n_kv * hd:8 + 2 * n_kv * hd].reshape(n, n_kv, hd)
        ref.append(k, v, 50)
        w, size = dev(wide), NP[t]().itemsize
        plan.append(buf.data_ptr(), t, w.data_ptr() + 8 * size, w.data_ptr() + (8 + n_kv * hd) * size, n, 50,
                    k_stride=wide.shape[1], v_stride=wide.shape[1])
        same_bytes(ref, buf)


def test_append_values_at_the_ends_of_the_format():
    """Zeros, the smallest and largest, ties, infinities, NaN; each block alone."""
    rng = np.random.default_rng(7)
    n_kv, hd = 1, 128
    k = np.zeros((96, n_kv, hd), np.float32)
    k[16:32, 0, 0] = 2.0 ** -30
    k[32:48] = (np.arange(16 * hd) % 255 - 127).reshape(16, 1, hd) / 2.0  # ties of a step of 1 (half-way codes)
    k[40, 0, 5] = 127.0
    k[48:64, 0, :4] = [np.inf, -np.inf, np.nan, 3.0]
    k[64:80, 0, :4] = [3e38, -1e6, 130048.0, np.nan]
    k[80:96] = np.nan
    for t in (F32, F16):
        with np.errstate(over="ignore"):
            x = k.astype(NP[t])
        plan, ref, buf = both(rng, n_kv, hd, 128, 16)
        with np.errstate(invalid="ignore", over="ignore"):
            ref.append(x, -x, 0)
        kd, vd = dev(x), dev(-x)
        plan.append(buf.data_ptr(), t, kd.data_ptr(), vd.data_ptr(), 96, 0)
        same_bytes(ref, buf)


def test_append_growth_past_many_steps():
    """One token 2^40 times larger than its block: the earlier codes go to 0."""
    rng = np.random.default_rng(8)
    plan, ref, buf = both(rng, 1, 256, 64, 64)
    for past, scale in [(0, 2.0 ** -24), (1, 2.0 ** -20), (2, 1.0), (3, 2.0 ** 16), (4, 1e-8)]:
        k = (rng.standard_normal((1, 1, 256)) * scale).astype(np.float32)
        ref.append(k, 3 * k, past)
        kd, vd = dev(k), dev(3 * k)
        plan.append(buf.data_ptr(), F32, kd.data_ptr(), vd.data_ptr(), 1, past)
        same_bytes(ref, buf, "at %d" % past)


# ------------------------------------------------------------------- read --

@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("n_kv,hd,block,slot0,n", [(1, 128, 16, 0, 1), (2, 256, 32, 63, 2), (3, 128, 64, 5, 200),
                                                   (2, 128, 32, 64, 128), (1, 256, 16, 191, 1)])
def test_read(t, n_kv, hd, block, slot0, n):
    rng = np.random.default_rng(slot0 + n)
    plan, ref, buf = both(rng, n_kv, hd, 256, block)
    k = rows(rng, 256, n_kv, hd, F32)
    ref.append(k, 0.3 * k, 0)
    buf = dev(ref.buf)
    out = [torch.full((n_kv * n * hd + 64,), -7.0, dtype=DT[t], device="cuda") for _ in "kv"]
    plan.read(buf.data_ptr(), slot0, n, t, out[0].data_ptr(), out[1].data_ptr())
    torch.cuda.synchronize()
    for which, o in zip("kv", out):
        got = o.cpu().numpy()
        want = ref.values(which, slot0 + n)[:, slot0:].astype(NP[t])  # at most 7 bits: exact in either type
        assert np.array_equal(got[:-64].reshape(n_kv, n, hd), want)
        assert np.all(got[-64:] == -7.0)
    same_bytes(ref, buf)


# -------------------------------------------------------------- attention --

def filled(rng, n_kv, hd, cap, block, n, scale_k=1.0, scale_v=1.0):
    """A cache with n slots stored, arbitrary bytes past them, and its copy on the GPU."""
    plan = kv8.KV8(n_kv, hd, cap, block)
    ref = kv8ref.Cache(n_kv, hd, cap, block, noise(rng, plan))
    ref.append(rows(rng, n, n_kv, hd, F32) * np.float32(scale_k), rows(rng, n, n_kv, hd, F32) * np.float32(scale_v), 0)
    return plan, ref, dev(ref.buf)


def weight_error(A, hd=256):
    return (2.0 ** -22 + (hd / 8 + 4) * 2.0 ** -24) * A + 2.0 ** -21 * (1.45 * A + 40)


def attn(plan, buf, q, n, past, t, mass=None, past_dev=None, scale=None, pad=0, stream=None):
    """One call with arbitrary bytes (NaN) in the workspace and the output, rows `pad` elements further apart."""
    n, heads, hd = q.shape
    wide = np.full((n, heads * hd + pad), np.nan, NP[t])
    wide[:, :heads * hd] = q.reshape(n, -1)
    qd = dev(wide)
    out = torch.full((n, heads * hd + pad), float("nan"), dtype=DT[t], device="cuda")
    ws = torch.full((plan.attn_workspace_bytes(heads, n) // 4,), float("nan"), device="cuda")
    torch.cuda.synchronize()
    plan.attn(buf.data_ptr(), heads, t, qd.data_ptr(), n, past, out.data_ptr(), ws.data_ptr(), ws.numel() * 4,
              scale=scale, mass=None if mass is None else mass.data_ptr(),
              n_past_dev=None if past_dev is None else past_dev.data_ptr(), q_stride=heads * hd + pad,
              out_stride=heads * hd + pad, stream=stream)
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    assert np.all(np.isnan(got[:, heads * hd:]))
    return got[:, :heads * hd].reshape(n, heads, hd).astype(np.float64)


def check(got, want, A, vmax, t, end):
    tol = 2 * weight_error(A) + 2.0 ** -22 + 2.0 ** -23 * (end / 64 + 40)
    if t == F16:
        tol += 2.0 ** -11 + 2.0 ** -11
    err = np.abs(got - want).max()
    print("error %.3g of %.3g allowed" % (err / vmax, tol))
    assert err <= tol * vmax, (err / vmax, tol)


ATTN = [  # n_heads, n_kv, hd, block, n, past
    (1, 1, 128, 16, 1, 0),      # a first token
    (4, 1, 128, 32, 1, 62),     # one slot short of a tile
    (4, 1, 128, 32, 1, 63),     # exactly a tile
    (8, 2, 128, 64, 1, 64),     # one over
    (32, 8, 128, 32, 1, 1030),
    (16, 2, 256, 64, 1, 700),
    (12, 2, 128, 16, 1, 300),   # a group of 6
    (7, 1, 256, 16, 3, 130),    # a group of 7
    (20, 1, 128, 64, 1, 500),   # a group of more than a tile of rows
    (16, 2, 256, 64, 6, 1000),  # a draft
    (8, 8, 128, 32, 5, 333),    # no sharing
    (4, 2, 128, 16, 17, 0),     # a short prompt from nothing
    (4, 1, 128, 64, 65, 31),
    (8, 2, 256, 32, 100, 0),
    (8, 2, 128, 64, 200, 77),
    (16, 4, 128, 32, 333, 500),
    (2, 1, 256, 16, 257, 190),
]


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("n_heads,n_kv,hd,block,n,past", ATTN)
def test_attn(t, n_heads, n_kv, hd, block, n, past):
    rng = np.random.default_rng(n_heads * 1000 + n + past)
    end = past + n
    plan, ref, buf = filled(rng, n_kv, hd, (end + 63) // 64 * 64 + 64, block, end)
    q = (1.5 * rng.standard_normal((n, n_heads, hd))).astype(NP[t])
    mass0 = rng.random((n_kv, plan.capacity)).astype(np.float32)
    mass0[:, past:] = np.nan  # what a new slot, or none, held before
    mass = dev(mass0)
    want, wmass, A = kv8ref.attend(ref, q, hd ** -0.5, n, past, mass0)
    vmax = np.abs(ref.values("v", end)).max()
    plain = attn(plan, buf, q, n, past, t, pad=8)
    check(plain, want, A, vmax, t, end)
    got = attn(plan, buf, q, n, past, t, mass=mass, pad=16)
    assert np.array_equal(got, plain)  # the mass does not change the output
    m = mass.cpu().numpy().astype(np.float64)
    assert np.all(np.isnan(m[:, end:]))
    # a weight's relative error is a score's; sums of at most n * group of them, and one addition
    tol = 2 * weight_error(A) + 2.0 ** -22 + 2.0 ** -24 * (n * n_heads / n_kv + 4)
    added = wmass[:, :end] - np.where(np.arange(end) < past, mass0[:, :end].astype(np.float64), 0)
    assert np.all(np.abs(m[:, :end] - wmass[:, :end]) <= tol * added + 2.0 ** -23 * wmass[:, :end] + 1e-30)
    # every row's weights sum to one
    assert abs(added.sum() - n * n_heads) <= 1e-9 * n * n_heads
    same_bytes(ref, buf)


def test_attn_long_split_context():
    """More slots than one round of the splits, and both sides of a unit's end."""
    rng = np.random.default_rng(11)
    plan, ref, buf = filled(rng, 1, 128, 20096, 64, 20050)
    for past in (12287, 20000):
        for n in (1, 5):
            q = (2 * rng.standard_normal((n, 4, 128))).astype(np.float32)
            want, _, A = kv8ref.attend(ref, q, 128 ** -0.5, n, past)
            check(attn(plan, buf, q, n, past, F32), want, A, np.abs(ref.values("v", past + n)).max(), F32, past + n)


@pytest.mark.parametrize("hd,heads", [(128, 8), (256, 3)])
def test_f16_token_keeps_its_weights(hd, heads):
    """Two slots of opposite values and nearly equal weights: what is left of them is
    the weights' difference, to an f32 call's error and the output's one rounding."""
    rng = np.random.default_rng(91 + hd)
    plan = kv8.KV8(1, hd, 64, 16)
    ref = kv8ref.Cache(1, hd, 64, 16, noise(rng, plan))
    u, x = 0.05 * rng.standard_normal((2, hd))
    ref.append(np.stack([u, -u])[:, None].astype(np.float32), np.stack([x, -x])[:, None].astype(np.float32), 0)
    q = rng.standard_normal((1, heads, hd)).astype(np.float16)
    want, _, A = kv8ref.attend(ref, q, hd ** -0.5, 1, 1, None)
    got = attn(plan, dev(ref.buf), q, 1, 1, F16)
    tol = 2 * weight_error(A) + 2.0 ** -22 + 2.0 ** -23 * 41
    err = np.abs(got - want) - 2.0 ** -11 * np.abs(want) - 2.0 ** -25
    assert err.max() <= tol * np.abs(ref.values("v", 2)).max()


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("n", [1, 40])
def test_attn_blocks_of_very_different_size(t, n):
    """V's blocks 2^20 apart in size, the larger ones less attended to: the
    weight of a small block's bytes stays a full f16 beside them."""
    rng = np.random.default_rng(12)
    past = 200
    plan, ref, _ = filled(rng, 1, 128, 256, 16, 256)
    ref.ve[0] = rng.integers(-14, 7, ref.ve.shape[1])
    ref.ke[0] = rng.integers(-12, -4, ref.ke.shape[1])
    q = (rng.standard_normal((n, 4, 128))).astype(NP[t])
    want, _, A = kv8ref.attend(ref, q, 128 ** -0.5, n, past)
    check(attn(plan, dev(ref.buf), q, n, past, t), want, A, np.abs(ref.values("v", past + n)).max(), t, past + n)


def test_attn_far_tail_of_small_weights():
    """One slot far above the rest in score: the 4000 others, each 2^-22 of it,
    together weigh 2^-10, and are not lost."""
    n_kv, hd, end = 1, 128, 4096
    plan = kv8.KV8(n_kv, hd, end, 64)
    ref = kv8ref.Cache(n_kv, hd, end, 64)
    k = np.zeros((end, 1, hd), np.float32)
    v = np.zeros((end, 1, hd), np.float32)
    k[:, 0, 0] = 1.0
    k[100, 0, 0] = 127 / 64
    v[:, 0, 1] = 1.0
    v[100, 0, 1] = 0.0
    ref.append(k, v, 0)
    q = np.zeros((1, 1, hd), np.float32)
    q[0, 0, 0] = 22 * np.log(2.0) / (63 / 64)
    want, _, A = kv8ref.attend(ref, q, 1.0, 1, end - 1)
    assert 2.0 ** -10.1 < want[0, 0, 1] < 2.0 ** -9.9
    got = attn(plan, dev(ref.buf), q, 1, end - 1, F32, scale=1.0)
    # relative to the small result itself: the scores' error and the sums'
    assert abs(got[0, 0, 1] / want[0, 0, 1] - 1) <= 2 * weight_error(A) + 2.0 ** -20
    got = attn(plan, dev(ref.buf), q.astype(np.float16), 1, end - 1, F16, scale=1.0)
    want, _, A = kv8ref.attend(ref, q.astype(np.float16), 1.0, 1, end - 1)
    assert abs(got[0, 0, 1] / want[0, 0, 1] - 1) <= 2.0 ** -11 + 2.0 ** -11 + 2 * weight_error(A)


@pytest.mark.parametrize("t", [F32, F16])
def test_attn_extremes_of_q(t):
    """A zero row, a tiny row, a large one, one of infinity and one of NaN: each
    row is its own."""
    rng = np.random.default_rng(13)
    plan, ref, buf = filled(rng, 1, 128, 192, 32, 150)
    n = 6
    q = rng.standard_normal((n, 2, 128)).astype(NP[t])
    q[0] = 0
    q[1] *= NP[t](1e-6)
    q[2] *= NP[t](300)
    q[3, 0, 7] = np.inf
    q[4, 1, 9] = np.nan
    want, _, _ = kv8ref.attend(ref, np.where(np.isfinite(q), q, 0), 128 ** -0.5, n, 144)
    got = attn(plan, buf, q, n, 144, t)
    vmax = np.abs(ref.values("v", 150)).max()
    assert np.all(np.isnan(got[4, 1])) and not np.any(np.isfinite(got[3, 0]))
    for i, h in [(i, h) for i in range(n) for h in range(2) if (i, h) not in ((3, 0), (4, 1))]:
        x = np.abs(np.float64(q[i, h])) @ np.abs(ref.values("k", 150)[0]).T * 128 ** -0.5
        check(got[i, h], want[i, h], x.max(), vmax, t, 150)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0])
def test_attn_any_scale(scale):
    rng = np.random.default_rng(14)
    plan, ref, buf = filled(rng, 2, 128, 192, 16, 130)
    q = (0.3 * rng.standard_normal((2, 4, 128))).astype(np.float32)
    want, _, A = kv8ref.attend(ref, q, scale, 2, 128)
    check(attn(plan, buf, q, 2, 128, F32, scale=scale), want, A, np.abs(ref.values("v", 130)).max(), F32, 130)


@pytest.mark.parametrize("n", [1, 3, 70])
def test_length_on_the_device(n):
    """The length in device memory: the same slots, clamped to what fits."""
    rng = np.random.default_rng(15)
    plan, ref, buf = filled(rng, 2, 128, 512, 32, 512)
    for given in (0, 5, 63, 64, 300, 512 - n, 511, 10 ** 9, -4):
        past = min(max(given, 0), 512 - n)
        pd = torch.tensor([given], dtype=torch.int32, device="cuda")
        q = rng.standard_normal((n, 4, 128)).astype(np.float32)
        mass0 = rng.random((2, 512)).astype(np.float32)
        mass = dev(mass0)
        want, wmass, A = kv8ref.attend(ref, q, 128 ** -0.5, n, past, mass0)
        got = attn(plan, buf, q, n, 99999, F32, mass=mass, past_dev=pd)
        check(got, want, A, np.abs(ref.values("v", past + n)).max(), F32, past + n)
        m = mass.cpu().numpy()
        assert np.array_equal(m[:, past + n:], mass0[:, past + n:])
        assert np.abs(m - wmass).max() <= 1e-4 * n
        k, v = rows(rng, n, 2, 128, F32), rows(rng, n, 2, 128, F32)
        ref.append(k, v, past)
        kd, vd = dev(k), dev(v)
        plan.append(buf.data_ptr(), F32, kd.data_ptr(), vd.data_ptr(), n, -1, n_past_dev=pd.data_ptr())
        same_bytes(ref, buf, "length %d" % given)


def test_replayed_step():
    """One captured graph of append and attend with the length on the device,
    replayed over 70 tokens with eager work between, equals the eager steps bit
    for bit."""
    rng = np.random.default_rng(16)
    n_kv, heads, hd, cap, past0 = 2, 8, 128, 256, 60
    plan, ref, buf = filled(rng, n_kv, hd, cap, 16, past0)
    eager = buf.clone()
    steps = 70
    k, v, q = (dev(rng.standard_normal((steps, h, hd)).astype(np.float32)) for h in (n_kv, n_kv, heads))
    kb, vb, qb = k[0].clone(), v[0].clone(), q[0].clone()
    out, ws = torch.empty_like(qb), torch.empty(plan.attn_workspace_bytes(heads, 1), dtype=torch.uint8, device="cuda")
    mass = torch.zeros(n_kv, cap, device="cuda")
    pd = torch.tensor([past0], dtype=torch.int32, device="cuda")

    def step(cache, m):
        st = torch.cuda.current_stream().cuda_stream
        plan.append(cache.data_ptr(), F32, kb.data_ptr(), vb.data_ptr(), 1, 0, n_past_dev=pd.data_ptr(), stream=st)
        plan.attn(cache.data_ptr(), heads, F32, qb.data_ptr(), 1, 0, out.data_ptr(), ws.data_ptr(), ws.numel(),
                  mass=m.data_ptr(), n_past_dev=pd.data_ptr(), stream=st)

    graph = torch.cuda.CUDAGraph()
    spare, spare_mass = buf.clone(), mass.clone()
    with torch.cuda.graph(graph):
        step(buf, mass)
    assert torch.equal(buf, spare) and torch.equal(mass, spare_mass)  # capturing ran nothing
    mass_e = mass.clone()
    for i in range(steps):
        kb.copy_(k[i])
        vb.copy_(v[i])
        qb.copy_(q[i])
        pd.fill_(past0 + i)
        graph.replay()
        got = out.clone()
        step(eager, mass_e)
        torch.cuda.synchronize()
        assert torch.equal(got, out) and torch.equal(buf, eager) and torch.equal(mass, mass_e), "step %d" % i
    host_past = attn(plan, eager, q[-1].cpu().numpy()[None], 1, past0 + steps - 1, F32)
    assert np.abs(host_past[0] - out.cpu().numpy()).max() <= 1e-4


def test_other_stream():
    rng = np.random.default_rng(17)
    plan, ref, buf = filled(rng, 2, 128, 640, 32, 600)
    q = rng.standard_normal((4, 4, 128)).astype(np.float32)
    want = attn(plan, buf, q, 4, 596, F32)
    s = torch.cuda.Stream()
    got = attn(plan, buf, q, 4, 596, F32, stream=s.cuda_stream)
    assert np.array_equal(got, want)


def test_same_call_twice_gives_the_same_bits():
    rng = np.random.default_rng(18)
    plan, ref, buf = filled(rng, 2, 256, 3200, 64, 3000)
    for n in (1, 130):
        q = rng.standard_normal((n, 8, 256)).astype(np.float32)
        m = [torch.zeros(2, plan.capacity, device="cuda") for _ in range(2)]
        a, b = (attn(plan, buf, q, n, 2800, F32, mass=x) for x in m)
        assert np.array_equal(a, b) and torch.equal(m[0], m[1])


# ---------------------------------------------------------------- eviction --

@pytest.mark.parametrize("hd,block,dst_block,n,keep,first,last", [
    (128, 32, 32, 200, 100, 4, 16), (128, 16, 64, 64, 1, 0, 0), (256, 64, 16, 130, 130, 0, 0),
    (128, 64, 64, 65, 64, 0, 64), (256, 32, 32, 300, 129, 7, 0), (128, 16, 16, 1, 1, 0, 1),
    (128, 64, 32, 2500, 77, 77, 0), (128, 32, 64, 2500, 1333, 3, 1000), (128, 32, 64, 1500, 1499, 0, 0),
])
@pytest.mark.parametrize("masses", ["spread", "ties"])
def test_evict(masses, hd, block, dst_block, n, keep, first, last):
    rng = np.random.default_rng(n + keep)
    n_kv = 2
    plan, ref, buf = filled(rng, n_kv, hd, (n + 63) // 64 * 64 + 64, block, n)
    dplan, dref, dbuf = both(rng, n_kv, hd, (keep + 63) // 64 * 64, dst_block)
    mass = rng.standard_normal((n_kv, plan.capacity)).astype(np.float32)
    if masses == "ties":
        mass = rng.integers(-2, 3, mass.shape).astype(np.float32)
        mass[rng.random(mass.shape) < 0.1] = np.nan
        mass[rng.random(mass.shape) < 0.1] = -0.0
        mass[rng.random(mass.shape) < 0.05] = -np.inf
        mass[rng.random(mass.shape) < 0.05] = np.inf
    pos = rng.integers(-10 ** 6, 10 ** 6, mass.shape).astype(np.int32)
    kept = kv8ref.evict(ref, mass, n, keep, first, last, dref)
    old_mass, old_pos = np.float32(rng.random((n_kv, dplan.capacity))), np.full((n_kv, dplan.capacity), 9, np.int32)
    md, pd, kd = dev(old_mass), dev(old_pos), torch.full((n_kv * keep + 16,), -5, dtype=torch.int32, device="cuda")
    sm, sp = dev(mass), dev(pos)
    plan.evict(buf.data_ptr(), sm.data_ptr(), sp.data_ptr(), n, keep, first, last, dplan, dbuf.data_ptr(),
               md.data_ptr(), pd.data_ptr(), kd.data_ptr())
    torch.cuda.synchronize()
    got = kd.cpu().numpy()
    assert np.array_equal(got[:n_kv * keep].reshape(n_kv, keep), kept) and np.all(got[n_kv * keep:] == -5)
    same_bytes(dref, dbuf, "the new cache")
    same_bytes(ref, buf, "the old cache")
    h = np.arange(n_kv)[:, None]
    old_mass[:, :keep] = mass[h, kept]
    old_pos[:, :keep] = pos[h, kept]
    assert np.array_equal(md.cpu().numpy().view(np.uint32), old_mass.view(np.uint32))
    assert np.array_equal(pd.cpu().numpy(), old_pos)
    assert np.array_equal(sm.cpu().numpy().view(np.uint32), mass.view(np.uint32))
    # without positions
    md2, kd2 = dev(old_mass), torch.zeros(n_kv, keep, dtype=torch.int32, device="cuda")
    plan.evict(buf.data_ptr(), sm.data_ptr(), None, n, keep, first, last, dplan, dbuf.data_ptr(), md2.data_ptr(), None,
               kd2.data_ptr())
    torch.cuda.synchronize()
    assert np.array_equal(kd2.cpu().numpy(), kept)
    same_bytes(dref, dbuf, "again")


def test_evict_many_slots():
    """More slots than threads of the selection, equal masses throughout and not."""
    rng = np.random.default_rng(21)
    n, keep = 70001, 30011
    plan = kv8.KV8(1, 128, 70016, 64)
    buf = dev(noise(rng, plan))
    dplan = kv8.KV8(1, 128, 30016, 64)
    dbuf = torch.zeros(dplan.nbytes, dtype=torch.uint8, device="cuda")
    for mass in (np.ones((1, 70016), np.float32), rng.random((1, 70016)).astype(np.float32),
                 rng.integers(0, 4, (1, 70016)).astype(np.float32)):
        order = np.argsort(-mass[0, 5:n - 100], kind="stable")[:keep - 105] + 5
        want = np.sort(np.concatenate([np.arange(5), order, np.arange(n - 100, n)]))
        sm, md = dev(mass), torch.zeros(1, 30016, device="cuda")
        kd = torch.zeros(keep, dtype=torch.int32, device="cuda")
        plan.evict(buf.data_ptr(), sm.data_ptr(), None, n, keep, 5, 100, dplan, dbuf.data_ptr(), md.data_ptr(), None,
                   kd.data_ptr())
        torch.cuda.synchronize()
        assert np.array_equal(kd.cpu().numpy(), want)
        assert np.array_equal(md.cpu().numpy()[0, :keep], mass[0, want])


@pytest.mark.parametrize("n", [4095, 4097, 24577, 65536, 65537])
@pytest.mark.parametrize("kind", ["spread", "levels", "equal"])
def test_evict_around_the_sizes_of_the_selection(n, kind):
    rng = np.random.default_rng(n)
    cap, keep = (n + 63) // 64 * 64, n // 3
    plan, dplan = kv8.KV8(2, 128, cap, 32), kv8.KV8(2, 128, (keep + 63) // 64 * 64, 32)
    buf = torch.zeros(plan.nbytes, dtype=torch.uint8, device="cuda")
    dbuf = torch.zeros(dplan.nbytes, dtype=torch.uint8, device="cuda")
    mass = {"spread": np.exp(3 * rng.standard_normal((2, cap))), "levels": rng.integers(0, 3, (2, cap)),
            "equal": np.full((2, cap), 0.25)}[kind].astype(np.float32)
    mass[:, n:] = np.inf  # behind the slots in use
    first, last = 4, 64
    sm, md = dev(mass), torch.zeros(2, dplan.capacity, device="cuda")
    kd = torch.zeros(2, keep, dtype=torch.int32, device="cuda")
    plan.evict(buf.data_ptr(), sm.data_ptr(), None, n, keep, first, last, dplan, dbuf.data_ptr(), md.data_ptr(), None,
               kd.data_ptr())
    torch.cuda.synchronize()
    for h in range(2):
        order = np.argsort(-mass[h, first:n - last], kind="stable")[:keep - first - last] + first
        want = np.sort(np.concatenate([np.arange(first), order, np.arange(n - last, n)]))
        assert np.array_equal(kd[h].cpu().numpy(), want), h
        assert np.array_equal(md[h].cpu().numpy()[:keep], mass[h, want])
