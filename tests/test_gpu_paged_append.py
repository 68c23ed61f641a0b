"""The paged append on both sides of the number of elements where it goes over from a row a
workgroup to runs of neighbouring slots, at both head dims, against pagedref.py number for
number."""
import numpy as np
import pytest

import pagedref
from oi import paged
from test_gpu_paged import F16, F32, NP, dev, host, pool, rows

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("n_kv,hd,page,news", [
    (1, 256, 32, [1024]), (1, 256, 32, [1025]), (1, 256, 16, [9, 400, 0, 7, 700]), (1, 128, 64, [1] * 2048), (1, 128, 64, [1] * 2049),
    (2, 256, 16, [1] * 270 + [5, 300]), (2, 256, 64, [33, 2, 17, 600]), (8, 256, 32, [70, 1, 1, 1, 60]), (3, 128, 16, [1000, 1, 3]),
    (32, 256, 16, [20, 12]), (32, 256, 16, [20, 13]), (64, 128, 32, [1] * 40), (1024, 256, 16, [1]), (1024, 256, 16, [2]),
])
def test_append_by_rows_and_by_runs(n_kv, hd, page, news, t):
    rng = np.random.default_rng(n_kv * hd + page + len(news) + t)
    past = rng.integers(0, 2 * page, len(news))
    n_pages = int(sum(pagedref.pages_of(a + b, page) for a, b in zip(past, news))) + 2
    width = max(pagedref.pages_of(a + b, page) for a, b in zip(past, news))
    table, free, n_free = pool(rng, past, page, width, n_pages)
    n = sum(news)
    slots = pagedref.plan(past, news, table, free, n_free, n, page)[4]
    plan = paged.Paged(n_kv, hd, n_pages, page)
    fill = rng.integers(0, 256, plan.nbytes).astype(np.uint8)
    k, v = rows(rng, n, n_kv, hd, t, True), rows(rng, n, n_kv, hd, t, True)
    for order in (np.arange(n), rng.permutation(n)):
        ref = pagedref.Pool(n_kv, hd, n_pages, page, fill)
        ref.append(k[order], v[order], slots[order])
        buf, kd, vd, sd = dev(fill), dev(k[order]), dev(v[order]), dev(np.int32(slots[order]))
        plan.append(buf.data_ptr(), t, kd.data_ptr(), vd.data_ptr(), n, sd.data_ptr())
        assert (host(buf) == ref.buf).all()
