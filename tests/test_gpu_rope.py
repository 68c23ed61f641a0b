"""The rotation of q and k by three axes (rope.hip) against its 64-bit form.

An output element is x c - y s (or x s + y c) of values up to X = max |x| of its
row after the norm.  The norm: the sum of hd squares in f32 (a tree, at most
log2(hd) + 2 roundings of 2^-24), a root and two products, together below
2^-24 (hd / 64 + 16) of the value.  Sine and cosine of an angle that is reduced
in 64 bits and rounded to f32 within pi/4: 2^-25 for the rounding and 2 units in
the last place.  Two products and a sum: 3 * 2^-24 of 2 X.  Together below
2^-24 * 40 X; an f16 output adds half a unit in its last place, 2^-11 of it.
"""
import numpy as np
import pytest

import kv8ref
from oi import rope

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

NP = {0: np.float32, 1: np.float16}
DT = {0: torch.float32, 1: torch.float16}


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def inv_freq(rotary, theta=1e6):
    half = rotary // 2
    return (theta ** (-np.arange(half) / max(half, 1))).astype(np.float32)


def close(got, want, t):
    X = np.abs(want).max(-1, keepdims=True) * 2 ** 0.5
    tol = 2.0 ** -24 * 40 * X + (2.0 ** -11 * np.abs(want) + 2.0 ** -25 if t else 0)
    err = np.abs(np.float64(got) - want)
    assert np.all(err <= tol), (err / tol).max()


CASES = [  # heads, kv, hd, rotary, sections, interleaved, n, in, out, norm, gate
    (4, 2, 128, 128, (24, 20, 20), True, 1, 0, 0, True, False),
    (16, 2, 256, 64, (11, 11, 10), True, 37, 0, 1, True, True),
    (16, 2, 256, 64, (11, 11, 10), False, 300, 0, 0, True, True),
    (3, 1, 128, 128, (16, 24, 24), False, 65, 1, 1, False, False),
    (5, 5, 128, 64, (32, 0, 0), False, 9, 1, 0, True, False),
    (2, 1, 256, 256, (44, 42, 42), True, 5, 0, 0, False, False),
    (1, 1, 128, 0, (0, 0, 0), False, 3, 0, 0, True, False),
    (8, 8, 128, 2, (0, 0, 1), False, 4, 0, 0, True, True),
    (4, 4, 128, 96, (0, 40, 8), True, 260, 1, 0, True, True),
]


@pytest.mark.parametrize("heads,kv,hd,rot,sec,il,n,ti,to,norm,gate", CASES)
def test_rope(heads, kv, hd, rot, sec, il, n, ti, to, norm, gate):
    rng = np.random.default_rng(hd + n + rot)
    hs, pad = (2 * hd if gate else hd), 8
    q = rng.standard_normal((n, heads * hs + pad)).astype(NP[ti])
    k = (5 * rng.standard_normal((n, kv * hd + 2 * pad))).astype(NP[ti])
    pos = rng.integers(-1000, 300000, (3, n)).astype(np.int32)
    w = [(1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) if norm else None for _ in "qk"]
    f = inv_freq(rot)
    plan = rope.RopeAxes(heads, kv, hd, rot, sec, il, 1e-6)
    qo = torch.full((n, heads * hd + pad), -3.0, dtype=DT[to], device="cuda")
    ko = torch.full((n, kv * hd + pad), -3.0, dtype=DT[to], device="cuda")
    d = [dev(pos), dev(f if rot else np.zeros(1, np.float32)), dev(q), dev(k)] + [None if x is None else dev(x) for x in w]
    plan.launch(n, d[0].data_ptr() if rot else None, d[1].data_ptr() if rot else None,
                *(None if x is None else x.data_ptr() for x in d[4:]), ti, d[2].data_ptr(), d[3].data_ptr(), to,
                qo.data_ptr(), ko.data_ptr(), q_stride=q.shape[1], q_head_stride=hs, k_stride=k.shape[1],
                q_out_stride=qo.shape[1], k_out_stride=ko.shape[1])
    torch.cuda.synchronize()
    for x, wx, o, h, s in ((q, w[0], qo, heads, hs), (k, w[1], ko, kv, hd)):
        rows = x[:, :h * s].reshape(n, h, s)[..., :hd]
        want = kv8ref.rope(rows, wx, pos, f, rot, sec, il, 1e-6)
        got = o.cpu().numpy()
        assert np.all(got[:, h * hd:] == -3.0)
        close(got[:, :h * hd].reshape(n, h, hd), want, to)


@pytest.mark.parametrize("t", [0, 1])
@pytest.mark.parametrize("n", [1, 400])
def test_in_place(t, n):
    rng = np.random.default_rng(3)
    q, k = rng.standard_normal((n, 4, 128)).astype(NP[t]), rng.standard_normal((n, 2, 128)).astype(NP[t])
    pos = np.repeat(np.arange(n, dtype=np.int32)[None], 3, 0) + 5
    f = inv_freq(64)
    plan = rope.RopeAxes(4, 2, 128, 64, (12, 10, 10), True, 1e-6)
    qd, kd, pd, fd = dev(q), dev(k), dev(pos), dev(f)
    w = torch.ones(128, device="cuda")
    plan.launch(n, pd.data_ptr(), fd.data_ptr(), w.data_ptr(), w.data_ptr(), t, qd.data_ptr(), kd.data_ptr(), t,
                qd.data_ptr(), kd.data_ptr())
    torch.cuda.synchronize()
    for x, o in ((q, qd), (k, kd)):
        close(o.cpu().numpy(), kv8ref.rope(x, np.ones(128), pos, f, 64, (12, 10, 10), True, 1e-6), t)


def test_far_positions_and_large_frequencies():
    """Angles of 10^9 and more keep their remainder: it is taken in 64 bits."""
    n = 64
    rng = np.random.default_rng(4)
    q, k = rng.standard_normal((n, 1, 128)).astype(np.float32), rng.standard_normal((n, 1, 128)).astype(np.float32)
    pos = rng.integers(-2 ** 31, 2 ** 31, (3, n)).astype(np.int32)
    pos[:, 0], pos[:, 1] = 2 ** 31 - 1, -2 ** 31
    f = np.concatenate([inv_freq(126), [7.25]]).astype(np.float32)
    plan = rope.RopeAxes(1, 1, 128, 128, (24, 20, 20), True, 1e-6)
    qd, kd, pd, fd = dev(q), dev(k), dev(pos), dev(f)
    plan.launch(n, pd.data_ptr(), fd.data_ptr(), None, None, 0, qd.data_ptr(), kd.data_ptr(), 0, qd.data_ptr(),
                kd.data_ptr())
    torch.cuda.synchronize()
    # the product pos * freq is exact in 64 bits (31 + 24 bits); the remainder's
    # error is 2^-53 of the angle, 2e-6 at most here
    for x, o in ((q, qd), (k, kd)):
        want = kv8ref.rope(x, None, pos, f, 128, (24, 20, 20), True, 1e-6)
        X = np.abs(want).max(-1, keepdims=True) * 2 ** 0.5
        assert np.all(np.abs(o.cpu().numpy() - want) <= (2.0 ** -24 * 40 + 2.0 ** -53 * 1.6e10 * 2) * X)
