"""A paged key-value cache for a token at a time: the pool of pages, the tables that say whose they are, and the operators of
`ops` on them. Everything that changes lives on the device (page tables, lengths, reference counts), nothing is read back, so that a
step that appends, attends, forks or frees can be captured in a CUDA Graph after one call of each kind has run. Calls on one cache
belong on one stream, or in an order that events give them.

The reference keeps the keys and values of its autoregressive prefix per layer in contiguous tensors
(thunderworld_fp4/cosmos/ar_cache.py:57-153); there is no paged cache in it.
"""
import torch
from . import ops
from ._lib import load


class PagedCache:
    """`sequences` slots of up to max_tokens tokens over a pool of `pages` pages of page_size tokens each, one layer.

    dtype torch.bfloat16, or torch.float8_e4m3fn with float32 [kv_heads] k_scale / v_scale (ones by default)."""

    def __init__(self, pages, page_size, kv_heads, head_dim=128, *, sequences, max_tokens, dtype=torch.bfloat16, device='cuda', k_scale=None,
                 v_scale=None):
        device = torch.device(device)
        if device.type == 'cuda' and device.index is None:
            device = torch.device('cuda', torch.cuda.current_device())
        ops.require_sm100(device)
        if min(pages, page_size, kv_heads, sequences, max_tokens) < 1:
            raise ValueError('pages, page_size, kv_heads, sequences and max_tokens must be positive')
        self.page_size = page_size
        if dtype not in (torch.bfloat16, torch.float8_e4m3fn):
            raise ValueError('pages must be bfloat16 or float8_e4m3fn')
        shape = pages, kv_heads, page_size, head_dim * dtype.itemsize
        self.k_pages, self.v_pages = (torch.zeros(shape, device=device, dtype=torch.uint8).view(dtype) for _ in range(2))
        self.table = torch.full((sequences, ops.cdiv(max_tokens, page_size)), -1, device=device, dtype=torch.int32)
        self.lengths = torch.zeros(sequences, device=device, dtype=torch.int32)
        self.refs = torch.zeros(pages, device=device, dtype=torch.int32)
        self.k_scale, self.v_scale = k_scale, v_scale
        ops._cache(self.k_pages, self.v_pages, self.table, self.lengths, self.refs)                    # its checks, before the first call
        ops._check_scales(device, kv_heads, k_scale, v_scale, dtype is torch.float8_e4m3fn)

    @property
    def _pools(self):
        return self.k_pages, self.v_pages

    @property
    def _tables(self):
        return self.table, self.lengths, self.refs

    def append(self, k, v, slots=None, cu=None):
        ops.cache_append_(k, v, *self._pools, *self._tables, slots=slots, cu=cu, k_scale=self.k_scale, v_scale=self.v_scale)

    def attend(self, q, slots=None, *, scale=None, return_lse=False, out=None):
        return ops.paged_attention(q, *self._pools, self.table, self.lengths, slots=slots, scale=scale, k_scale=self.k_scale, v_scale=self.v_scale,
                                   return_lse=return_lse, out=out)

    def fork(self, parents, children):
        ops.cache_fork_(*self._pools, *self._tables, parents, children)

    def free(self, slots):
        ops.cache_free_(*self._tables, slots, self.page_size)

    def compact(self):
        return ops.cache_compact_(*self._pools, *self._tables)

    def check(self):
        """Raise if any paged operator on this device, on whatever stream, left something out since the status was last reset (waits for it)."""
        status = ops.device_status(self.k_pages.device)
        if status:
            raise RuntimeError(load().tw_status(status).decode())
