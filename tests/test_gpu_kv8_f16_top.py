"""The top of f16's range: a block's largest values round to 65536 and beyond
(codes of a step of 1024), which f16 does not hold.  What is finite in the cache
comes out of the f16 forms finite: +-65504."""
import numpy as np
import pytest

import kv8ref
from oi import kv8
from test_gpu_kv8 import F16, F32, NP, attn, dev, noise

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TOP = 65504.0


def cache(values, hd, n_kv=1, block=16, slots=None):
    """V (and K / 2^20 of it) with values[i] in every dimension of block i."""
    end = block * len(values) if slots is None else slots
    cap = (end + 63) // 64 * 64
    plan = kv8.KV8(n_kv, hd, cap, block)
    ref = kv8ref.Cache(n_kv, hd, cap, block, noise(np.random.default_rng(3), plan))
    v = np.repeat(np.asarray(values, np.float32), block)[:end, None, None] * np.ones((1, n_kv, hd), np.float32)
    return plan, ref, v


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("hd", [128, 256])
def test_read_at_the_top_of_f16(hd, t):
    values = [65504.0, -65504.0, 65024.0, 65280.0, -65472.0, np.inf, -np.inf, 70000.0, -130048.0, 1.0, 0.0, 33000.0]
    plan, ref, v = cache(values, hd)
    n = v.shape[0]
    with np.errstate(invalid="ignore"):
        ref.append(v, -v, 0)
    buf = dev(ref.buf)
    out = [torch.empty(1, n, hd, dtype=torch.float16 if t == F16 else torch.float32, device="cuda") for _ in "kv"]
    plan.read(buf.data_ptr(), 0, n, t, out[0].data_ptr(), out[1].data_ptr())
    torch.cuda.synchronize()
    for which, o in zip("kv", out):
        want = ref.values(which, n)
        assert np.abs(want).max() == 130048
        if t == F16:
            want = want.clip(-TOP, TOP)
        assert np.array_equal(o.cpu().numpy(), want.astype(NP[t]))


@pytest.mark.parametrize("x", [65504.0, -65504.0, np.inf])
def test_an_f16_value_comes_back_finite(x):
    """f16 in, f16 out, through append and read: off by at most half a step of its block (2^9).
    Infinity is 127 steps of its block's finite values, of which there are none here: 127 * 2^-24."""
    plan, ref, _ = cache([0.0] * 4, 128)
    rows = torch.full((3, 1, 128), x, dtype=torch.float16, device="cuda")
    buf = dev(ref.buf)
    plan.append(buf.data_ptr(), F16, rows.data_ptr(), rows.data_ptr(), 3, 0)
    out = [torch.empty(1, 3, 128, dtype=torch.float16, device="cuda") for _ in "kv"]
    plan.read(buf.data_ptr(), 0, 3, F16, out[0].data_ptr(), out[1].data_ptr())
    torch.cuda.synchronize()
    want, tol = (x, 512) if np.isfinite(x) else (127 * 2.0 ** -24, 0)
    for o in out:
        got = o.cpu().numpy().astype(np.float64)
        assert np.all(np.isfinite(got)) and np.abs(got - want).max() <= tol


# one wave's rows and 16, merged splits (each of the merges), the prompt's tiles whole and split, masses beside them
CALLS = [  # n, group, n_kv, end, mass
    (1, 1, 1, 64, False), (1, 16, 1, 128, False), (1, 4, 1, 4096, False), (1, 16, 1, 4096, True), (40, 2, 1, 4096, False),
    (35, 16, 1, 128, False), (600, 1, 1, 4096, True), (257, 8, 8, 600, False), (300, 2, 2, 1100, False),
]


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("n,group,n_kv,end,with_mass", CALLS)
def test_attention_at_the_top_of_f16(n, group, n_kv, end, with_mass, hd, t):
    """Every V the same: the output is that value, whatever the weights."""
    rng = np.random.default_rng(end)
    for x, stored in ((65504.0, 65536.0), (-65504.0, -65536.0), (1e9, 130048.0), (1000.0, 1000.0)):
        plan, ref, v = cache([x] * ((end + 15) // 16), hd, n_kv, slots=end)
        ref.append(rng.standard_normal(v.shape).astype(np.float32), v, 0)
        assert np.all(ref.values("v", end) == stored)
        q = rng.standard_normal((n, n_kv * group, hd)).astype(NP[t])
        mass = torch.zeros(n_kv, plan.capacity, device="cuda") if with_mass else None
        got = attn(plan, dev(ref.buf), q, n, end - n, t, mass=mass)
        want = np.clip(stored, -TOP, TOP) if t == F16 else stored
        # the sums' roundings above and below the line, and of an f16 call the weights' and its output's
        tol = 2.0 ** -22 + 2.0 ** -23 * (end / 64 + 40) + (2.0 ** -10 + 2.0 ** -11 if t == F16 else 0)
        assert np.abs(got / want - 1).max() <= tol
        if t == F16:
            assert np.abs(got).max() <= TOP


@pytest.mark.parametrize("n,group,end", [(2, 2, 64), (2, 2, 4096), (40, 2, 300), (600, 1, 700), (600, 1, 4096)])
@pytest.mark.parametrize("t", [F32, F16])
def test_what_is_not_finite_stays_so(n, group, end, t):
    """A row of q that holds NaN gives NaN, not a number."""
    rng = np.random.default_rng(end)
    plan, ref, v = cache([65504.0] * ((end + 15) // 16), 128, slots=end)
    ref.append(rng.standard_normal(v.shape).astype(np.float32), v, 0)
    q = rng.standard_normal((n, group, 128)).astype(NP[t])
    q[n // 2, 0, 3] = np.nan
    got = attn(plan, dev(ref.buf), q, n, end - n, t)
    assert np.all(np.isnan(got[n // 2, 0]))
    got[n // 2, 0] = 0
    assert np.all(np.isfinite(got))
