"""Attention over the paged cache where scores are far beyond what exponents hold: rows
whose largest score is 2^25 and more in base 2 (the append itself stores +-65504 for
infinities), where the rounded product of a score and its factor and the unrounded one
lie whole powers of two apart.  Through oi.paged, against the plain 64-bit form.

Every element of a slot's K is one number, every element of a row of q too, so scores of slots
with the same number are the same number in any arithmetic, and those of others lie thousands
apart: a row's weights are equal among the slots of its largest score and 0 elsewhere.  Then
only sums and an output's rounding remain: the tolerance of
test_gpu_paged_attn.py for scores of size 0.  Rows of small q beside them keep its tolerance
for their own size."""
import numpy as np
import pytest

from test_gpu_paged_attn import F16, F32, NP, Batch, dev, tolerance

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def batch(seed, n_kv, hd, page, ends, same, top):
    """K of a slot one number: `same` for all, or each its own below `top`, 2^-10 of it apart or more."""
    b = Batch(seed, n_kv, hd, page, ends)
    for i, e in enumerate(ends):
        if e == 0:
            continue
        slots = np.array([int(b.table[i, j // page]) * page + j % page for j in range(e)])
        if same:
            a = np.full(e, top)
        else:  # the largest again from time to time, every other at most 1023 / 1024 of it
            a = top * b.rng.integers(100, 1024, e) / 1024
            a[b.rng.random(e) < 0.02] = top
            a[0] = top / 128
        k = np.broadcast_to(a[:, None, None], (e, n_kv, hd)).astype(np.float32)
        v = b.rng.standard_normal((e, n_kv, hd)).astype(np.float32)
        b.ref.append(k, v, slots)
    b.buf.copy_(dev(b.ref.buf))
    return b


def run(b, which, t, heads, n_q, q, scale):
    n = len(b.ends)
    if which == "tokens":
        return b.tokens(heads, t, n_q, q, scale=scale)
    return b.prompts(heads, t, [n_q * i for i in range(n + 1)], n_q * n, q, scale=scale)


def check(b, got, q, n_q, t, prompts, scale, small):
    """small: which (token, head) rows of q have scores of ordinary size."""
    starts = [n_q * i for i in range(len(b.ends) + 1)]
    assert np.isfinite(got).all()
    for i, lo, hi, (out, size, top) in b.want(q, starts, scale):
        end = max(b.ends[i], 0)
        err = np.abs(got[lo:hi].astype(np.float64) - out)
        tol = np.broadcast_to(tolerance(0.0, top, end, b.hd, t, prompts), err.shape).copy()
        if small[lo:hi].any():
            k, v = b.ref.request(b.table[i], end)
            own = np.abs(np.where(small[lo:hi, :, None], q[lo:hi], 0)).max() * b.hd * np.abs(k).max() * abs(scale)
            tol[small[lo:hi]] = np.broadcast_to(tolerance(own, top, end, b.hd, t, prompts), err.shape)[small[lo:hi]]
        assert (err <= tol).all(), (i, float((err / tol).max()), np.argwhere(err > tol)[:3].tolist())


SIZES = [(40.0, 65504.0), (1000.0, 3000.0), (3000.0, 65504.0), (61440.0, 65504.0)]
WIDE = SIZES + [(2.0 ** 40, 65504.0), (2.0 ** 70, 65504.0)]  # f32 only


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("which", ["tokens", "prompts"])
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("same", [True, False])
def test_large_scores(same, hd, which, t):
    for n, (x, top) in enumerate(WIDE if t == F32 else SIZES):
        for sign in (1.0, -1.0):
            b = batch(10 * n + hd, 2, hd, 32, [300, 33, 0, 1, 1500], same, top)
            n_q = 3
            q = np.full((5 * n_q, 8, hd), x * sign, NP[t])
            got = run(b, which, t, 8, n_q, q, hd ** -0.5)
            check(b, got, q, n_q, t, which == "prompts", hd ** -0.5, np.zeros(q.shape[:2], bool))


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("which", ["tokens", "prompts"])
@pytest.mark.parametrize("hd,heads,n_q,ends", [
    (128, 2, 1, [20000]),          # parts of many workers joined
    (256, 4, 2, [9000, 40]),
    (128, 12, 16, [700, 90]),      # more than 64 rows of a kv head
    (128, 24, 2, [900, 64, 5]),    # groups of waves
])
def test_large_scores_beside_small_ones(hd, heads, n_q, ends, which, t):
    """Rows of every size in one wave."""
    for same in (True, False):
        b = batch(7 + len(ends) + heads, 1, hd, 16, ends, same, 65504.0)
        n = len(ends) * n_q
        q = np.broadcast_to(b.rng.choice([40.0, -3000.0, 2e-4, -1e-5, 0.0, 1000.0], (n, heads, 1)), (n, heads, hd)).astype(NP[t])
        small = np.abs(q[:, :, 0]) < 1
        got = run(b, which, t, heads, n_q, q, hd ** -0.5)
        check(b, got, q, n_q, t, which == "prompts" or n_q * heads > 64, hd ** -0.5, small)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("which", ["tokens", "prompts"])
def test_scores_around_the_size_where_products_round_to_whole_numbers(which, t):
    """Largest scores of 2^18 to 2^32: each row another."""
    hd = 128
    b = batch(77, 1, hd, 64, [500, 70], False, 1024.0)
    n_q, heads = 5, 12
    scale = 1 / 1024 / hd / 1.4426950408889634  # times log2(e), and a K of 1024: q itself in base 2
    rng = np.random.default_rng(3)
    size = (2.0 ** rng.uniform(18, 32, (2 * n_q, heads, 1))) if t == F32 else 2.0 ** rng.uniform(10, 15.9, (2 * n_q, heads, 1))
    if t == F16:
        scale *= 2.0 ** 14
    q = np.broadcast_to(np.rint(size), (2 * n_q, heads, hd)).astype(NP[t])
    got = run(b, which, t, heads, n_q, q, scale)
    check(b, got, q, n_q, t, which == "prompts", scale, np.zeros(q.shape[:2], bool))


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("which", ["tokens", "prompts"])
def test_rows_that_are_not_finite_stay_so_beside_large_scores(which, t):
    b = batch(5, 1, 128, 16, [200, 90], False, 65504.0)
    q = np.full((8, 4, 128), 40.0, NP[t])
    q[1, 2, 7], q[5, 0, 3], q[6, 3] = np.nan, np.inf, np.nan
    got = run(b, which, t, 4, 4, q, 128 ** -0.5)
    bad = np.zeros((8, 4), bool)
    bad[1, 2] = bad[5, 0] = bad[6, 3] = True
    assert (np.isfinite(got).all(-1) == ~bad).all()
    clean = np.where(bad[..., None], 0, q).astype(NP[t])
    ref = run(b, which, t, 4, 4, clean, 128 ** -0.5)
    assert (got[~bad] == ref[~bad]).all()
