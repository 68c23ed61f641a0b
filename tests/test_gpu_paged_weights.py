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
