"""Attention over the 8-bit cache where V's blocks lie far apart in size: zero
blocks (exponent -24) beside one that is attended to, exponents over the whole
range of the format, the heavy slots in the small blocks.  Errors are bounded
element by element, by what that element's row sums up, not by the largest |V| of
the cache.

With w the softmax weights, S = sum w |V| of an element, and E a weight's relative
error (test_gpu_kv8.py):
* numerator and sum are off by E S each, and by 2^-23 S for each of end / 64 + 40
  additions one after another (both together);
* an f32 call's weights are two halves, 2^-22; an f16 call's are rounded once above
  the line and at most once below, 2^-11 of S each, and its output once, 2^-11 of
  the output (2^-25 in the subnormals);
* a weight that reaches f16 below its normal numbers is off by half a subnormal,
  2^-25, where the row's largest product w 2^e stands at 2^7 or more (in the f32 form
  at 2^14; 2^7 is the weaker): sum over the slots of 2^-32 |code| max(w 2^e) above the
  line.  Below the line weights of blocks at most 2^4 apart may be rounded so:
  2^-32 2^4 of the row's sum each, end 2^-28 in all.
"""
import numpy as np
import pytest

import kv8ref
from oi import kv8
from test_gpu_kv8 import F16, F32, NP, attn, dev, noise, weight_error

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def softmax(ref, q, scale, n, past):
    """Weights [n_heads][n][end] in 64 bits and the largest sum of |q_d k_d| |scale|."""
    heads, end, A = q.shape[1], past + n, 0.0
    seen = np.arange(end) <= past + np.arange(n)[:, None]
    K, w = ref.values("k", end), np.empty((heads, n, end))
    for h in range(heads):
        k = K[h // (heads // ref.n_kv)]
        s = np.where(seen, np.float64(q[:, h]) @ k.T * scale, -np.inf)
        A = max(A, float(np.where(seen, np.abs(np.float64(q[:, h])) @ np.abs(k).T * abs(scale), 0).max()))
        p = np.exp(s - s.max(1, keepdims=True))
        w[h] = p / p.sum(1, keepdims=True)
    return w, A


def check_rows(ref, q, scale, n, past, t, got, mass):
    """out and mass (which began at zero) against the weights, element by element."""
    heads, hd, end, g = q.shape[1], q.shape[2], past + n, q.shape[1] // ref.n_kv
    w, A = softmax(ref, q, scale, n, past)
    V = ref.values("v", end)
    step = 2.0 ** np.repeat(ref.ve.clip(kv8ref.EMIN, kv8ref.EMAX), ref.block, 1)[:, :end].astype(np.float64)
    E = weight_error(A, hd)
    worst = 0.0
    for h in range(heads):
        v, e = V[h // g], step[h // g]
        want, S = w[h] @ v, w[h] @ np.abs(v)
        top = (w[h] * e).max(1, keepdims=True)
        tol = (2 * E + 2.0 ** -22 + 2.0 ** -23 * (end / 64 + 40) + end * 2.0 ** -28) * S
        tol = tol + 2.0 ** -32 * top * (np.abs(v) / e[:, None]).sum(0) + 1e-30
        if t == F16:
            tol = tol + 2.0 ** -10 * S + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
        worst = max(worst, float((np.abs(got[:, h] - want) / tol).max()))
    print("error %.3g of the bound" % worst)
    assert worst <= 1
    if mass is not None:
        m = mass.cpu().numpy().astype(np.float64)
        sums = w.reshape(ref.n_kv, g, n, end).sum((1, 2))
        tol = 2 * E + 2.0 ** -22 + 2.0 ** -24 * (n * g + 4)
        assert np.all(np.abs(m[:, :end] - sums) <= tol * sums + 1e-30)
        assert abs(m[:, :end].sum() - n * heads) <= tol * n * heads  # every row's weights sum to one
        assert np.all(m[:, end:] == 0)


def both_ways(ref, q, scale, n, past, t):
    plan, buf = kv8.KV8(ref.n_kv, ref.hd, ref.cap, ref.block), dev(ref.buf)
    plain = attn(plan, buf, q, n, past, t, scale=scale)
    check_rows(ref, q, scale, n, past, t, plain, None)
    mass = torch.zeros(ref.n_kv, ref.cap, device="cuda")
    got = attn(plan, buf, q, n, past, t, mass=mass, scale=scale)
    assert np.array_equal(got, plain)
    check_rows(ref, q, scale, n, past, t, got, mass)


# rows of a kv head: the forms by 8 and by 16, several tiles of 16, the prompt's (128 and 256 a workgroup)
SHAPES = [  # n, group, n_kv, end
    (1, 8, 1, 8192), (1, 16, 1, 8192), (10, 4, 1, 8192), (70, 8, 1, 8192),  # split over the slots
    (1, 16, 1, 128), (10, 4, 1, 128), (35, 16, 1, 128),                     # not
    (1, 16, 2, 4100), (300, 2, 2, 1100),
]


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("n,group,n_kv,end", SHAPES)
@pytest.mark.parametrize("size,bits", [(1.0, 15.3), (16.0, 11.4), (256.0, 7.7), (4000.0, 11.2), (60000.0, 7.6),
                                       (60000.0, 3.5)])
def test_one_block_among_zeros(size, bits, n, group, n_kv, end, hd, t):
    """V is zero but for one block of 16 slots, one of which scores `bits` bits above all others: the
    zero slots' weight is what divides the output."""
    rng = np.random.default_rng(int(size) + end + n)
    past, cap = end - n, (end + 63) // 64 * 64 + 64
    ref = kv8ref.Cache(n_kv, hd, cap, 16, noise(rng, kv8.KV8(n_kv, hd, cap, 16)))
    k, v = np.zeros((2, end, n_kv, hd), np.float32)
    block = past // 32  # in the middle of what every row sees
    at = 16 * block + 5
    k[at, :, 0] = 1
    v[16 * block:16 * block + 16] = size * rng.standard_normal((16, n_kv, hd)).clip(-1.0, 1.0)
    ref.append(k, v, 0)
    assert np.sum(ref.ve[:, :(end + 15) // 16] != kv8ref.EMIN) == n_kv
    q = rng.standard_normal((n, n_kv * group, hd)).astype(NP[t])
    q[:, :, 0] = bits * np.log(2.0)
    both_ways(ref, q, 1.0, n, past, t)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("hd,block", [(128, 16), (128, 64), (256, 32)])
@pytest.mark.parametrize("n,group,n_kv,end", SHAPES)
@pytest.mark.parametrize("kind", ["any", "rising", "falling", "one large"])
def test_exponents_over_the_whole_range(kind, n, group, n_kv, end, hd, block, t):
    """Blocks of any exponent in any order, with scores that favour the small ones so
    that they hold most of the weight."""
    rng = np.random.default_rng(hd + block + end + n)
    past = end - n
    cap = (end + 63) // 64 * 64 + 64
    ref = kv8ref.Cache(n_kv, hd, cap, block, noise(rng, kv8.KV8(n_kv, hd, cap, block)))
    blocks = (end + block - 1) // block
    if kind == "any":
        ev = rng.integers(-24, 11, (n_kv, blocks))
    elif kind == "one large":
        ev = np.full((n_kv, blocks), -12)
        ev[:, blocks // 3] = 10
    else:
        ev = np.tile(np.linspace(-24, 10, blocks).round().astype(int), (n_kv, 1))
        ev = ev if kind == "rising" else ev[:, ::-1]
    # the score's bits against V's exponent: a tenth of it to most of it
    slope = rng.uniform(0.1, 0.6, (n_kv, blocks))
    slots = np.repeat(ev, block, 1)[:, :end]
    k = 0.3 * rng.standard_normal((end, n_kv, hd)).astype(np.float32)
    k[:, :, 0] = (-slots * np.repeat(slope, block, 1)[:, :end]).T / 8
    v = rng.integers(-127, 128, (end, n_kv, hd)).astype(np.float32)
    v[::block, :, 0] = 127
    ref.append(k, v * 2.0 ** slots.T[:, :, None].astype(np.float32), 0)
    assert np.array_equal(ref.ve[:, :blocks], ev)
    q = (0.05 * rng.standard_normal((n, n_kv * group, hd))).astype(NP[t])
    q[:, :, 0] = 8 * np.log(2.0)
    both_ways(ref, q, 1.0, n, past, t)


@pytest.mark.parametrize("n,group,hd", [(1, 16, 128), (40, 1, 128), (35, 16, 128), (600, 1, 128), (600, 1, 256)])
def test_bytes_behind_the_last_slot_change_nothing(n, group, hd):
    """The last unit's other slots, their blocks' exponents among them, hold anything: the same bits come out."""
    rng = np.random.default_rng(n + hd)
    end, got = n + 530, []
    cap = (end + 63) // 64 * 64 + 64
    k, v = rng.standard_normal((2, end, 1, hd)).astype(np.float32)
    v *= np.exp2(-rng.integers(0, 12, (end, 1, 1))).astype(np.float32)
    q = rng.standard_normal((n, group, hd)).astype(np.float16)
    for fill in (0, 10, 246, 127, 128):
        ref = kv8ref.Cache(1, hd, cap, 16, np.full(kv8.KV8(1, hd, cap, 16).nbytes, fill, np.uint8))
        ref.append(k, v, 0)
        mass = torch.zeros(1, cap, device="cuda")
        got.append((attn(kv8.KV8(1, hd, cap, 16), dev(ref.buf), q, n, end - n, F16, mass=mass), mass.cpu().numpy()))
        assert np.array_equal(got[-1][0], got[0][0]) and np.array_equal(got[-1][1], got[0][1]), fill
