"""What the entries of the 8-bit cache and of the rotation refuse before anything
reaches a device: small inputs inside an output, a scale that f32 does not hold."""
import ctypes

import pytest

from oi import _native, kv8

E_ARG = -1
M = 1 << 24  # addresses that are never read


def lib():
    return _native.hip()


def dims(cap=256, block=32):
    return ctypes.byref(_native.KV8Dims(2, 128, cap, block))


def test_a_device_length_inside_an_output():
    """*n_past_dev is read again after outputs are written."""
    L, r, size = lib(), dims(), kv8.KV8(2, 128, 256, 32).nbytes
    for at in (M, M + 4, M + size - 4):
        assert L.oi_kv8_append_launch(r, M, 0, 2 * M, 256, 3 * M, 256, 10, 0, at, None) == E_ARG, at
        assert b"n_past_dev" in L.oi_last_error() and b"misaligned" not in L.oi_last_error()
    need = L.oi_kv8_attn_workspace_bytes(r, 4, 3)
    q, out, ws, mass = 2 * M, 3 * M, 4 * M, 5 * M
    for at in (out, out + 512 * 4 * 3 - 4, ws, ws + 64, mass, mass + 2 * 256 * 4 - 4):
        assert L.oi_kv8_attn_launch(r, M, 4, 0, q, 512, 0.1, 3, 0, at, mass, out, 512, ws, need, None) == E_ARG, at
        assert b"overlaps" in L.oi_last_error()
    # rows further apart than they are long, the length between them: an output's span is taken as a whole
    assert L.oi_kv8_attn_launch(r, M, 4, 0, q, 512, 0.1, 3, 0, out + 2048, mass, out, 1024, ws, need, None) == E_ARG


def rope_args(**over):
    D = _native.RopeAxesDims(4, 2, 128, 128, (ctypes.c_int32 * 3)(24, 20, 20), 1, 1e-6)
    a = dict(dict(pos=M, inv_freq=2 * M, q_norm=3 * M, k_norm=4 * M, qo=7 * M, ko=8 * M), **over)
    return [ctypes.byref(D), 10, a["pos"], a["inv_freq"], a["q_norm"], a["k_norm"], 0, 5 * M, 512, 128, 6 * M, 256, 0,
            a["qo"], 512, a["ko"], 256, None], D


@pytest.mark.parametrize("out,size", [("qo", 10 * 512 * 4), ("ko", 10 * 256 * 4)])
@pytest.mark.parametrize("what,length", [("pos", 3 * 10 * 4), ("inv_freq", 64 * 4), ("q_norm", 128 * 4),
                                         ("k_norm", 128 * 4)])
def test_rotation_inputs_inside_an_output(what, length, out, size):
    L, base = lib(), 7 * M if out == "qo" else 8 * M
    for at in (base, base + 1024, base + size - 4, base - length + 4):
        a, keep = rope_args(**{what: at})
        assert L.oi_rope_axes_launch(*a) == E_ARG, at
        assert b"overlaps" in L.oi_last_error()


def test_rotation_without_norm_or_turn_has_no_such_inputs():
    """What is not read is not compared: the call gets as far as the alignment of what is."""
    L = lib()
    a, keep = rope_args(q_norm=None, k_norm=3 * M + 2)
    assert L.oi_rope_axes_launch(*a) == E_ARG and b"misaligned" in L.oi_last_error()
    keep.rotary_dim, keep.sections = 0, (ctypes.c_int32 * 3)(0, 0, 0)
    a[2] = a[3] = 7 * M
    assert L.oi_rope_axes_launch(*a) == E_ARG and b"misaligned" in L.oi_last_error()


@pytest.mark.parametrize("scale", [3.4e38, -3.0e38, 2.5e38])
def test_scale_that_f32_does_not_hold_in_base_2(scale):
    """scale * log2(e) is what the kernels multiply by: infinite, every output would be NaN."""
    L, r = lib(), dims()
    need = L.oi_kv8_attn_workspace_bytes(r, 4, 3)
    rc = L.oi_kv8_attn_launch(r, M, 4, 0, 2 * M, 512, scale, 3, 5, None, None, 3 * M, 512, 4 * M, need, None)
    assert rc == E_ARG and b"scale" in L.oi_last_error()


def test_workspace_of_a_call_that_is_refused():
    """More rows than one call takes: no size, as for other arguments that the call refuses."""
    L, r = lib(), dims(cap=1 << 21)
    for heads, n in [(8, 262140), (4, 524280), (2, 1048560)]:
        assert L.oi_kv8_attn_workspace_bytes(r, heads, n) > 0
        assert L.oi_kv8_attn_workspace_bytes(r, heads, n + 1) == 0
        need = 1 << 60
        rc = L.oi_kv8_attn_launch(r, M, heads, 0, 1 << 50, 128 * heads, 0.1, n + 1, 0, None, None, 1 << 52, 128 * heads,
                                  1 << 54, need, None)
        assert rc == -6 and b"too many rows" in L.oi_last_error()
