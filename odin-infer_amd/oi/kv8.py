"""The 8-bit K/V cache on the device (oi_kv8_*): append, read, attention,
eviction.  Pointers are device addresses (integers); nothing here allocates or
waits."""
import ctypes
import math

from . import _native
from ._native import check


class KV8:
    """The shape of a layer's cache: kv heads, head_dim, capacity (slots, a
    multiple of 64) and block (slots that share an exponent).  The buffer of
    `nbytes` is the caller's (oi.h has its layout)."""

    def __init__(self, n_kv_heads, head_dim, capacity, block=64):
        self.dims = _native.KV8Dims(int(n_kv_heads), int(head_dim), int(capacity), int(block))
        self.n_kv_heads, self.head_dim, self.capacity, self.block = n_kv_heads, head_dim, capacity, block
        self._d = ctypes.addressof(self.dims)
        self._lib = _native.hip()
        self.nbytes = int(self._lib.oi_kv8_bytes(self._d))
        if not self.nbytes:
            raise _native.OIError(-1, "kv8: bad dims (head_dim 128 or 256, capacity a multiple of 64, "
                                      "block 16, 32 or 64)")

    def append(self, cache, type, k, v, n, n_past, n_past_dev=None, k_stride=None, v_stride=None, stream=None):
        """K and V rows [n][n_kv_heads][head_dim] behind the n_past slots in use."""
        row = self.n_kv_heads * self.head_dim
        check(self._lib.oi_kv8_append_launch(self._d, cache, type, k, row if k_stride is None else k_stride, v,
                                             row if v_stride is None else v_stride, n, n_past, n_past_dev, stream))

    def read(self, cache, slot0, n, type, k, v, stream=None):
        """Slots slot0.. as values, k and v [n_kv_heads][n][head_dim]."""
        check(self._lib.oi_kv8_read_launch(self._d, cache, slot0, n, type, k, v, stream))

    def attn_workspace_bytes(self, n_heads, n):
        return int(self._lib.oi_kv8_attn_workspace_bytes(self._d, n_heads, n))

    def attn(self, cache, n_heads, type, q, n, n_past, out, workspace, workspace_bytes, scale=None, mass=None,
             n_past_dev=None, q_stride=None, out_stride=None, stream=None):
        """Causal attention of the last n tokens over the cache (scale: default
        1 / sqrt(head_dim)); mass: each slot's weight, accumulated."""
        row = n_heads * self.head_dim
        check(self._lib.oi_kv8_attn_launch(self._d, cache, n_heads, type, q, row if q_stride is None else q_stride,
                                           1.0 / math.sqrt(self.head_dim) if scale is None else scale, n, n_past,
                                           n_past_dev, mass, out, row if out_stride is None else out_stride,
                                           workspace, workspace_bytes, stream))

    def evict(self, cache, mass, pos, n, keep, n_first, n_last, dst, dst_cache, dst_mass, dst_pos, kept, stream=None):
        """The slots worth keeping, into another cache (dst: its KV8)."""
        check(self._lib.oi_kv8_evict_launch(self._d, cache, mass, pos, n, keep, n_first, n_last, dst._d, dst_cache,
                                            dst_mass, dst_pos, kept, stream))
