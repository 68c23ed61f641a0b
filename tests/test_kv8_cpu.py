"""The 8-bit K/V cache and the three-axis rotation without a GPU: sizes, what
the entries refuse (before anything reaches a device), and the properties of the
format that the header states, on the plain form that the GPU tests compare
with."""
import ctypes
import re

import numpy as np
import pytest

import kv8ref
from oi import _native, kv8

E_ARG, E_RANGE = -1, -6
P = 1 << 20  # an aligned address that is never read


def dims(n_kv=2, hd=128, cap=256, block=32):
    return _native.KV8Dims(n_kv, hd, cap, block)


def lib():
    return _native.hip()


@pytest.mark.parametrize("d", [(0, 128, 256, 32), (2, 96, 256, 32), (2, 128, 250, 32), (2, 128, 0, 32),
                               (2, 128, 256, 8), (2, 128, 256, 48), (2, 128, -64, 32), (-1, 128, 64, 32),
                               (2, 128, (1 << 28) + 64, 64), (1025, 128, 64, 64)])
def test_bad_dims(d):
    D = dims(*d)
    L, r = lib(), ctypes.byref(D)
    assert L.oi_kv8_bytes(r) == 0
    assert L.oi_kv8_attn_workspace_bytes(r, 2, 1) == 0
    assert L.oi_kv8_append_launch(r, P, 0, P, 256, P, 256, 1, 0, None, None) == E_ARG
    assert L.oi_kv8_read_launch(r, P, 0, 1, 0, P, P, None) == E_ARG
    assert L.oi_kv8_attn_launch(r, P, 2, 0, P, 256, 1.0, 1, 0, None, None, P, 256, P, 1 << 30, None) == E_ARG
    assert L.oi_kv8_evict_launch(r, P, P, None, 8, 4, 0, 0, r, 8 * P, 8 * P, None, P, None) == E_ARG
    with pytest.raises(_native.OIError):
        kv8.KV8(*d)


def test_sizes():
    for n_kv, hd, cap, block in [(1, 128, 64, 16), (2, 256, 192, 32), (8, 128, 4096, 64), (3, 128, 64, 64)]:
        n = kv8.KV8(n_kv, hd, cap, block).nbytes
        assert n == kv8ref.Cache(n_kv, hd, cap, block).buf.size
    # a whole layer of a long context: sizes past 32 bits
    assert kv8.KV8(8, 256, 1 << 24, 64).nbytes == 2 * 8 * (1 << 24) * 256 + 2 * 8 * (1 << 18)
    assert lib().oi_kv8_bytes(None) == 0


def test_append_refusals():
    L, r = lib(), ctypes.byref(dims())
    ok = [r, P, 0, P, 256, P, 256, 1, 0, None, None]
    for at, bad, code in [(1, None, E_ARG), (3, None, E_ARG), (5, None, E_ARG), (2, 2, E_ARG), (2, -1, E_ARG),
                          (1, P + 16, E_ARG), (3, P + 4, E_ARG), (5, P + 8, E_ARG), (4, 255, E_ARG), (4, 257, E_ARG),
                          (6, 128, E_ARG), (7, 0, E_RANGE), (7, 257, E_RANGE), (8, 256, E_RANGE), (8, -1, E_RANGE),
                          (7, -3, E_RANGE), (8, 2 ** 31 - 1, E_RANGE)]:
        a = list(ok)
        a[at] = bad
        assert L.oi_kv8_append_launch(*a) == code, (at, bad)
        assert b"kv8 append" in L.oi_last_error()
    a = list(ok)
    a[2], a[4] = 1, 260  # f16 rows 520 bytes apart
    assert L.oi_kv8_append_launch(*a) == E_ARG


def test_read_refusals():
    L, r = lib(), ctypes.byref(dims())
    ok = [r, P, 0, 1, 0, P, P, None]
    for at, bad, code in [(1, None, E_ARG), (5, None, E_ARG), (6, None, E_ARG), (4, 3, E_ARG), (5, P + 8, E_ARG),
                          (1, P + 128, E_ARG), (2, -1, E_RANGE), (2, 256, E_RANGE), (3, 0, E_RANGE), (3, 257, E_RANGE)]:
        a = list(ok)
        a[at] = bad
        assert L.oi_kv8_read_launch(*a) == code, (at, bad)


def test_attn_refusals():
    L, r = lib(), ctypes.byref(dims())
    need = L.oi_kv8_attn_workspace_bytes(r, 4, 3)
    assert need > 0
    ok = [r, P, 4, 0, P, 512, 0.1, 3, 5, None, P, P, 512, P, need, None]
    for at, bad, code in [(1, None, E_ARG), (4, None, E_ARG), (11, None, E_ARG), (13, None, E_ARG), (2, 3, E_ARG),
                          (2, 0, E_ARG), (2, 8192, E_ARG), (3, 8, E_ARG), (4, P + 4, E_ARG), (5, 511, E_ARG),
                          (6, float("nan"), E_ARG), (6, float("inf"), E_ARG), (7, 0, E_RANGE), (7, 300, E_RANGE),
                          (8, 254, E_RANGE), (8, -2, E_RANGE), (10, P + 2, E_ARG), (12, 500, E_ARG),
                          (13, P + 8, E_ARG), (14, 16, E_ARG), (14, -1, E_ARG)]:
        a = list(ok)
        a[at] = bad
        assert L.oi_kv8_attn_launch(*a) == code, (at, bad)
        assert b"kv8 attention" in L.oi_last_error()
    for out, stride, mass in [(P, 1024, None), (P, 512, 8 * P)]:  # in place: another stride, or with mass
        a = list(ok)
        a[10], a[11], a[12] = mass, out, stride
        assert L.oi_kv8_attn_launch(*a) == E_ARG
    a = list(ok)
    a[9] = P + 2  # the device length
    assert L.oi_kv8_attn_launch(*a) == E_ARG
    for heads, n in [(3, 1), (0, 1), (4, 0), (4, 257), (-4, 1)]:
        assert L.oi_kv8_attn_workspace_bytes(r, heads, n) == 0


@pytest.mark.parametrize("hd", [128, 256])
def test_workspace_covers_every_length(hd):
    """The stated workspace is enough at every length, type, and with or without mass
    (a call with none says what it needs)."""
    L = lib()

    def needed(r, heads, t, n, past, mass):
        assert L.oi_kv8_attn_launch(r, P, heads, t, 2 * P, heads * hd, 1.0, n, past, None, 4 * P if mass else None,
                                    8 * P, heads * hd, 16 * P, 0, None) == E_ARG
        return int(re.search(rb"bytes, (\d+) needed", L.oi_last_error()).group(1))

    for n_kv, group, cap, n in [(1, 3, 116032, 2078), (16, 16, 960, 298), (8, 2, 7488, 901), (1, 8, 27840, 195),
                                (1, 4, 10048, 1230), (8, 8, 40960, 3), (8, 4, 9600, 30), (2, 2, 64, 9),
                                (4, 1, 100032, 1), (16, 16, 960, 298), (8, 4, 33024, 2047)]:
        D = dims(n_kv, hd, cap, 64)
        r = ctypes.byref(D)
        most = L.oi_kv8_attn_workspace_bytes(r, n_kv * group, n)
        for past in sorted({*range(0, cap - n + 1, max(1, cap // 1500)), cap - n}):
            for t in (0, 1):
                for mass in (False, True):
                    assert needed(r, n_kv * group, t, n, past, mass) <= most, (n_kv, group, cap, n, past, t, mass)


def test_evict_refusals():
    L, r = lib(), ctypes.byref(dims())
    other = ctypes.byref(dims(cap=128, block=64))
    far = 64 * P
    ok = [r, P, 4 * P, 6 * P, 200, 100, 4, 8, other, far, far + 4 * P, far + 6 * P, far + 8 * P, None]
    for at, bad, code in [(1, None, E_ARG), (2, None, E_ARG), (3, None, E_ARG), (9, None, E_ARG), (10, None, E_ARG),
                          (11, None, E_ARG), (12, None, E_ARG), (1, P + 64, E_ARG), (9, far + 64, E_ARG),
                          (4, 0, E_RANGE), (4, 257, E_RANGE), (5, 0, E_RANGE), (5, 201, E_RANGE), (5, 129, E_RANGE),
                          (6, -1, E_RANGE), (7, -1, E_RANGE), (6, 93, E_RANGE), (7, 2 ** 31 - 1, E_RANGE),
                          (2, 4 * P + 4, E_ARG), (12, far + 8 * P + 2, E_ARG), (9, P, E_ARG), (9, P + 256, E_ARG), (10, 4 * P, E_ARG), (11, 6 * P + 512, E_ARG)]:
        a = list(ok)
        a[at] = bad
        assert L.oi_kv8_evict_launch(*a) == code, (at, bad)
    for d in (dims(n_kv=4, cap=128), dims(hd=256, cap=128)):
        a = list(ok)
        a[8] = ctypes.byref(d)
        assert L.oi_kv8_evict_launch(*a) == E_ARG


def test_rope_refusals():
    L = lib()

    def D(h=4, kv=2, hd=128, rot=128, s=(24, 20, 20), il=1, eps=1e-6):
        return _native.RopeAxesDims(h, kv, hd, rot, (ctypes.c_int32 * 3)(*s), il, eps)

    good = D()
    ok = [ctypes.byref(good), 3, P, P, P, P, 0, P, 512, 128, P, 256, 1, 4 * P, 512, 8 * P, 256, None]
    for at, bad, code in [(1, 0, E_RANGE), (1, -1, E_RANGE), (2, None, E_ARG), (3, None, E_ARG), (6, 2, E_ARG),
                          (12, 8, E_ARG), (7, None, E_ARG), (10, None, E_ARG), (13, None, E_ARG), (15, None, E_ARG),
                          (7, P + 4, E_ARG), (8, 508, E_ARG), (8, 514, E_ARG), (9, 64, E_ARG), (9, 130, E_ARG),
                          (9, 256, E_ARG), (11, 128, E_ARG), (14, 511, E_ARG), (14, 516, E_ARG), (16, 128, E_ARG),
                          (9, -128, E_ARG)]:
        a = list(ok)
        a[at] = bad
        assert L.oi_rope_axes_launch(*a) == code, (at, bad)
    for d in (D(hd=96), D(rot=130), D(rot=7), D(s=(24, 20, 21)), D(s=(-1, 45, 20)), D(h=0), D(kv=0), D(rot=-2),
              D(eps=float("nan")), D(eps=-1.0)):
        a = list(ok)
        a[0] = ctypes.byref(d)
        assert L.oi_rope_axes_launch(*a) == E_ARG
    a = list(ok)
    a[0] = None
    assert L.oi_rope_axes_launch(*a) == E_ARG
    # in place with another type, another row stride, a gate beside each head, another k stride
    for at, bad in [((13,), (P,)), ((12, 13, 14), (0, P, 1024)), ((8, 9, 12, 13, 14), (1024, 256, 0, P, 1024)),
                    ((12, 10, 15, 16), (0, 2 * P, 2 * P, 512))]:
        a = list(ok)
        for i, b in zip(at, bad):
            a[i] = b
        assert L.oi_rope_axes_launch(*a) == E_ARG, (at, bad)
    for at in (2, 3, 4, 5):
        a = list(ok)
        a[at] = P + 2
        assert L.oi_rope_axes_launch(*a) == E_ARG, at


def test_overlap_refusals():
    """An output that shares memory with another argument, whole or in part."""
    L, D = lib(), dims()
    r, size, M = ctypes.byref(D), kv8.KV8(2, 128, 256, 32).nbytes, 1 << 24
    c, row = M, 256 * 4  # the cache; a K or V row's bytes

    for k, v in [(c, 2 * M), (2 * M, c + size - 256), (c - row, 2 * M), (c - 9 * 2 * row + 16, 2 * M)]:
        assert L.oi_kv8_append_launch(r, c, 0, k, 512, v, 256, 10, 0, None, None) == E_ARG, (k, v)
        assert b"in the cache" in L.oi_last_error()
    for k, v in [(c, 2 * M), (2 * M, c + size - 256), (2 * M, 2 * M), (2 * M, 2 * M + 10 * row - 16)]:
        assert L.oi_kv8_read_launch(r, c, 0, 10, 0, k, v, None) == E_ARG, (k, v)
        assert b"overlap" in L.oi_last_error()

    need, row = L.oi_kv8_attn_workspace_bytes(r, 4, 3), 512 * 4
    q, out, ws, mass = 2 * M, 3 * M, 4 * M, 5 * M
    for a in [dict(out=q + 16), dict(out=q + 2 * row - 16), dict(out=c + size - 256), dict(out=ws + 16),
              dict(out=mass - 3 * row + 16), dict(ws=c), dict(ws=q + 2 * row), dict(ws=mass), dict(mass=c + 16),
              dict(mass=q + 4), dict(out=q + row, stride=1024), dict(out=q + 512, stride=1024, q_stride=1024),
              dict(out=q - 512 + 4096, stride=1024, q_stride=1024), dict(q=M >> 1, q_stride=1 << 40)]:
        b = dict(dict(q=q, out=out, ws=ws, mass=mass, stride=512, q_stride=512), **a)
        assert L.oi_kv8_attn_launch(r, c, 4, 0, b["q"], b["q_stride"], 0.1, 3, 5, None, b["mass"], b["out"],
                                    b["stride"], b["ws"], need, None) == E_ARG, a
        assert b"overlaps" in L.oi_last_error()

    other = ctypes.byref(dims(cap=128, block=64))
    for at, bad in [(9, 3 * M), (10, 2 * M + 512), (10, c), (11, 3 * M + 512), (11, 2 * M), (12, 3 * M), (12, 2 * M),
                    (12, 5 * M), (12, 6 * M + 1020), (12, 7 * M + 4), (10, 7 * M), (10, 5 * M), (11, 5 * M + 64)]:
        a = [r, c, 2 * M, 3 * M, 200, 100, 4, 8, other, 5 * M, 6 * M, 7 * M, 8 * M, None]
        a[at] = bad
        assert L.oi_kv8_evict_launch(*a) == E_ARG, (at, bad)
        assert b"overlap" in L.oi_last_error()

    D = _native.RopeAxesDims(4, 2, 128, 128, (ctypes.c_int32 * 3)(24, 20, 20), 1, 1e-6)
    # q and k of one projection's rows (q, k, v: 1024 elements), f32; then the outputs
    q, k, row = 2 * M, 2 * M + 512 * 4, 1024 * 4
    for qo, ko, qs, ks in [(q + 16, 3 * M, 1024, 256), (k, 3 * M, 1024, 256), (3 * M, q + 512, 256 * 4, 1024),
                           (3 * M, k + 512, 256 * 4, 1024), (3 * M, 3 * M, 512, 256), (3 * M, 3 * M + 2047, 512, 256),
                           (q, k - 16, 1024, 1024), (q, k + row - 16, 1024, 256), (q + 9 * row + 2048 - 16, 3 * M, 512, 256)]:
        a = [ctypes.byref(D), 10, M, M, None, None, 0, q, 1024, 128, k, 1024, 0, qo, qs, ko & ~15, ks, None]
        assert L.oi_rope_axes_launch(*a) == E_ARG, (qo, ko)
        assert b"overlaps" in L.oi_last_error(), (qo, ko)
    # in place in the projection's rows, or beside it: what is refused here is the positions' alignment
    for qo, ko, qs, ks in [(q, k, 1024, 1024), (q, 3 * M, 1024, 256), (3 * M, k, 512, 1024), (q, k + 1024, 1024, 1024)]:
        a = [ctypes.byref(D), 10, M + 2, M, None, None, 0, q, 1024, 128, k, 1024, 0, qo, qs, ko, ks, None]
        assert L.oi_rope_axes_launch(*a) == E_ARG, (qo, ko)
        assert b"misaligned" in L.oi_last_error(), (qo, ko)
    for n, code in [(1 << 24, E_RANGE), (2 ** 31 - 1, E_RANGE)]:
        a = [ctypes.byref(D), n, M, M, None, None, 0, q, 1024, 128, k, 1024, 0, q, 1024, k, 1024, None]
        assert L.oi_rope_axes_launch(*a) == code


def test_format_one_rounding():
    """A value stored once is off by at most half a step, and the step is the
    least power of two that holds the block."""
    rng = np.random.default_rng(1)
    k = (rng.standard_normal((64, 1, 128)) * np.exp(2 * rng.standard_normal((64, 1, 1)))).astype(np.float32)
    c = kv8ref.Cache(1, 128, 64, 16)
    c.append(k, k, 0)
    for b in range(4):
        x = np.float64(k[16 * b:16 * b + 16, 0])
        step = 2.0 ** int(c.ke[0, b])
        assert np.abs(x).max() <= 127 * step and np.abs(x).max() > 127 * step / 2
        assert np.abs(c.values("k", 64)[0, 16 * b:16 * b + 16] - x).max() <= step / 2
    assert np.array_equal(c.values("k", 64), c.values("v", 64))


def test_format_growing_block():
    """A block filled token by token while its range keeps growing ends less
    than one final step off (half a step for the last rounding, and the earlier
    ones, of halves of smaller steps, sum to less than another half)."""
    rng = np.random.default_rng(2)
    for trial in range(20):
        k = (rng.standard_normal((16, 1, 128)) * np.exp2(rng.uniform(0, 0.9) * np.arange(16))[:, None, None])
        k = k.astype(np.float32)
        c = kv8ref.Cache(1, 128, 64, 16)
        for i in range(16):
            c.append(k[i:i + 1], k[i:i + 1], i)
        step = 2.0 ** int(c.ke[0, 0])
        assert np.abs(c.values("k", 16)[0] - np.float64(k[:, 0])).max() < step


@pytest.mark.parametrize("amax,e", [(0.0, -24), (127.0, 0), (np.nextafter(np.float32(127), np.float32(128)), 1),
                                    (1.0, -6), (1.984375, -6), (2.0, -5), (65504.0, 10), (1e9, 10),
                                    (127 * 2.0 ** -24, -24), (1e-30, -24), (2.0 ** -17, -23)])
def test_exponent(amax, e):
    assert kv8ref.exponent(float(amax)) == e
