"""RMSNorm and rotation of q and k by positions of three axes, on the device
(oi_rope_axes_launch).  Pointers are device addresses (integers)."""
import ctypes

from . import _native
from ._native import check


class RopeAxes:
    """The shape of a layer's q and k heads and how its rotary pairs belong to
    the axes (oi_rope_axes_dims)."""

    def __init__(self, n_heads, n_kv_heads, head_dim, rotary_dim, sections, interleaved, eps):
        self.dims = _native.RopeAxesDims(int(n_heads), int(n_kv_heads), int(head_dim), int(rotary_dim),
                                         (ctypes.c_int32 * 3)(*sections), int(bool(interleaved)), eps)
        self.n_heads, self.n_kv_heads, self.head_dim = n_heads, n_kv_heads, head_dim
        self._d = ctypes.addressof(self.dims)
        self._lib = _native.hip()

    def launch(self, n, pos, inv_freq, q_norm, k_norm, in_type, q, k, out_type, q_out, k_out, q_stride=None,
               q_head_stride=None, k_stride=None, q_out_stride=None, k_out_stride=None, stream=None):
        """pos [3][n] int32; q_norm / k_norm None: no norm.  Strides in elements;
        by default heads and tokens lie one after the other."""
        hd = self.head_dim
        qh = hd if q_head_stride is None else q_head_stride
        check(self._lib.oi_rope_axes_launch(
            self._d, n, pos, inv_freq, q_norm, k_norm, in_type, q, self.n_heads * qh if q_stride is None else q_stride,
            qh, k, self.n_kv_heads * hd if k_stride is None else k_stride, out_type, q_out,
            self.n_heads * hd if q_out_stride is None else q_out_stride, k_out,
            self.n_kv_heads * hd if k_out_stride is None else k_out_stride, stream))
