"""A token whose q holds NaN or infinity gives its weight to no slot that it does
not see: the call's later slots get what the other rows give them."""
import numpy as np
import pytest

from test_gpu_kv8 import F16, F32, NP, attn, filled, weight_error
from test_gpu_kv8_range import softmax

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("n,group,hd,past", [(4, 2, 128, 130), (3, 4, 256, 0), (8, 2, 128, 60), (4, 1, 128, 20000),
                                             (5, 3, 256, 1500),        # at most 16 rows
                                             (20, 2, 128, 130), (130, 2, 128, 64), (600, 1, 128, 100), (40, 4, 256, 70)])
def test_masked_slots_of_a_bad_row(n, group, hd, past, bad, t):
    rng = np.random.default_rng(n + past)
    end, row = past + n, n // 3
    plan, ref, buf = filled(rng, 1, hd, (end + 63) // 64 * 64, 32, end)
    q = rng.standard_normal((n, group, hd)).astype(NP[t])
    w, A = softmax(ref, q, hd ** -0.5, n, past)
    w[0, row] = 0  # the row that gives nothing that can be compared
    want = w.sum((0, 1))
    q[row, 0, 5] = bad
    mass = torch.zeros(1, plan.capacity, device="cuda")
    got = attn(plan, buf, q, n, past, t, mass=mass)
    assert not np.any(np.isfinite(got[row, 0]))
    m = mass.cpu().numpy()[0].astype(np.float64)
    hidden = slice(past + row + 1, end)
    tol = 2 * weight_error(A, hd) + 2.0 ** -22 + 2.0 ** -24 * (n * group + 4)
    assert np.all(np.abs(m[hidden] - want[hidden]) <= tol * want[hidden] + 1e-30)
    assert np.all(np.isnan(m[:past + row + 1])) or bad == np.inf
