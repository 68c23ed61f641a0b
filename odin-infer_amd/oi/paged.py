"""The paged f16 K/V cache of many sequences on the device (oi_paged_*): pages
given and taken back, append, attention of the newest tokens and of packed
prompts.  Pointers are device addresses (integers); nothing here allocates or
waits."""
import ctypes
import math

from . import _native
from ._native import check


class Paged:
    """The shape of a layer's pool: kv heads, head_dim, pages and slots of a page
    (16, 32 or 64).  The buffer of `nbytes` is the caller's (oi.h has its layout)."""

    def __init__(self, n_kv_heads, head_dim, n_pages, page=64):
        self.dims = _native.PagedDims(int(n_kv_heads), int(head_dim), int(n_pages), int(page))
        self.n_kv_heads, self.head_dim, self.n_pages, self.page = n_kv_heads, head_dim, n_pages, page
        self._d = ctypes.addressof(self.dims)
        self._lib = _native.hip()
        self.nbytes = int(self._lib.oi_paged_bytes(self._d))
        if not self.nbytes:
            raise _native.OIError(-1, "paged: bad dims (head_dim 128 or 256, page 16, 32 or 64, n_pages * page at most "
                                      "2^28)")

    def plan(self, n_seqs, n_past, n_new, table, table_stride, free_pages, n_free, n_rows, lens, starts, slots, pos=None,
             stream=None):
        """Pages for n_new[i] more slots of each sequence; the lengths after, the
        packed rows' begins, slots and (pos [3][n_rows]) positions."""
        check(self._lib.oi_paged_plan_launch(self._d, n_seqs, n_past, n_new, table, table_stride, free_pages, n_free,
                                             n_rows, lens, starts, slots, pos, stream))

    def release(self, n_seqs, n_held, n_keep, table, table_stride, free_pages, n_free, stream=None):
        """Pages behind the first n_keep[i] (None: 0) of n_held[i] slots back to the list."""
        check(self._lib.oi_paged_release_launch(self._d, n_seqs, n_held, n_keep, table, table_stride, free_pages, n_free,
                                                stream))

    def append(self, cache, type, k, v, n, slots, k_stride=None, v_stride=None, stream=None):
        """K and V rows [n][n_kv_heads][head_dim] into their slots."""
        row = self.n_kv_heads * self.head_dim
        check(self._lib.oi_paged_append_launch(self._d, cache, type, k, row if k_stride is None else k_stride, v,
                                               row if v_stride is None else v_stride, n, slots, stream))

    def tokens_workspace_bytes(self, n_heads, n_seqs, n_q=1):
        return int(self._lib.oi_paged_tokens_workspace_bytes(self._d, n_heads, n_seqs, n_q))

    def tokens(self, cache, n_heads, type, q, n_seqs, n_q, lens, table, table_stride, out, workspace, workspace_bytes,
               scale=None, q_stride=None, out_stride=None, stream=None):
        """Causal attention of the newest n_q tokens of each sequence (scale: default
        1 / sqrt(head_dim))."""
        row = n_heads * self.head_dim
        check(self._lib.oi_paged_tokens_launch(self._d, cache, n_heads, type, q, row if q_stride is None else q_stride,
                                               1.0 / math.sqrt(self.head_dim) if scale is None else scale, n_seqs, n_q,
                                               lens, table, table_stride, out, row if out_stride is None else out_stride,
                                               workspace, workspace_bytes, stream))

    def prompts_workspace_bytes(self, n_heads, n_seqs, n_rows):
        return int(self._lib.oi_paged_prompts_workspace_bytes(self._d, n_heads, n_seqs, n_rows))

    def prompts(self, cache, n_heads, type, q, n_seqs, n_rows, starts, lens, table, table_stride, out, workspace,
                workspace_bytes, scale=None, q_stride=None, out_stride=None, stream=None):
        """The same for packed rows, sequence i's being starts[i] .. starts[i + 1] - 1."""
        row = n_heads * self.head_dim
        check(self._lib.oi_paged_prompts_launch(self._d, cache, n_heads, type, q, row if q_stride is None else q_stride,
                                                1.0 / math.sqrt(self.head_dim) if scale is None else scale, n_seqs,
                                                n_rows, starts, lens, table, table_stride, out,
                                                row if out_stride is None else out_stride, workspace, workspace_bytes,
                                                stream))
