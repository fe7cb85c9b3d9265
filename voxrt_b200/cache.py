"""Paged int8 key / value cache and the attention over it: KvCache.write, read and attend, each a thin call into
libvxg.so's C ABI on torch CUDA tensors. Batches are stacked along the token axis; lengths and offsets are device tensors,
so a decode step can be captured in a CUDA graph and replayed as the sequences grow."""
from __future__ import annotations

import ctypes as C
import math

import torch

from ._lib import lib
from .kernels import _DTYPES, _addr, _call, _dt, _empty, _need, _on


class _Desc(C.Structure):  # vxg_kv_cache
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scales", C.c_void_p), ("v_scales", C.c_void_p),
                ("n_pages", C.c_int), ("heads", C.c_int), ("page", C.c_int), ("head_dim", C.c_int)]


def _stacked(t: torch.Tensor, heads: int, hd: int, what: str) -> int:
    """Row stride of a stacked [rows, heads, head_dim] operand whose rows are contiguous."""
    _need(t.dim() == 3 and t.shape[1] == heads and t.shape[2] == hd,
          f"{what} has shape {tuple(t.shape)}, not (rows, {heads}, {hd})")
    _need(t.stride(2) == 1 and (heads == 1 or t.stride(1) == hd), f"{what}'s rows must be contiguous")
    return t.stride(0) if t.shape[0] > 1 else heads * hd


class KvCache:
    """A pool of n_pages pages: k, v int8 [n_pages, heads, page, head_dim] with one f32 scale per (page, head) in ks and
    vs. page 16, 32, 64 or 128; head_dim 64 or 128. The pool does not know which pages are whose: a page table
    [n_seq, max_pages] (int32) lists each sequence's pages in order, entries behind its last page are not read."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, ks: torch.Tensor, vs: torch.Tensor):
        _need(k.dim() == 4 and k.dtype == torch.int8 and k.is_contiguous() and k.is_cuda,
              "k must be a contiguous int8 CUDA tensor [n_pages, heads, page, head_dim]")
        _need(v.shape == k.shape and v.dtype == torch.int8 and v.is_contiguous() and v.device == k.device,
              "v must be like k")
        for t in (ks, vs):
            _need(t.shape == k.shape[:2] and t.dtype == torch.float32 and t.is_contiguous() and t.device == k.device,
                  "scales must be contiguous float32 [n_pages, heads] on the codes' device")
        self.k, self.v, self.ks, self.vs = k, v, ks, vs
        self.n_pages, self.heads, self.page, self.head_dim = k.shape
        self._desc = _Desc(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), *k.shape)
        self._ref = C.addressof(self._desc)

    @classmethod
    def empty(cls, n_pages: int, heads: int, head_dim: int, page: int = 64, device=None) -> "KvCache":
        dev = device if device is not None else torch.device("cuda", torch.cuda.current_device())
        codes = [torch.zeros((n_pages, heads, page, head_dim), dtype=torch.int8, device=dev) for _ in range(2)]
        scales = [torch.zeros((n_pages, heads), dtype=torch.float32, device=dev) for _ in range(2)]
        return cls(*codes, *scales)

    def _batch(self, table, a, cu, stream, *more):
        _on(self.k.device, stream, table, a, cu, *more)
        for t, what in ((table, "the page table"), (a, "lengths"), (cu, "offsets")):
            _need(t.dtype == torch.int32 and t.is_contiguous(), f"{what} must be contiguous int32")
        _need(table.dim() == 2 and a.shape == (table.shape[0],) and cu.shape == (table.shape[0] + 1,),
              f"page table {tuple(table.shape)}, lengths {tuple(a.shape)} and offsets {tuple(cu.shape)} do not belong "
              "to one batch")
        return table.shape

    def _mine(self):
        return (self.k, self.v, self.ks, self.vs)

    def write(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor, cu: torch.Tensor,
              stream=None) -> None:
        """Quantise and append k and v [rows, heads, head_dim] (f32, f16 or bf16, any row stride): rows cu[s] .. cu[s+1]
        go to positions start[s] .. of sequence s. A started page's scale grows when it has to, and its earlier codes
        with it. Pages that are written must belong to one sequence each."""
        n_seq, width = self._batch(table, start, cu, stream, k, v)
        _need(k.dtype == v.dtype and k.shape == v.shape, "k and v must be alike")
        ld_k, ld_v = _stacked(k, self.heads, self.head_dim, "k"), _stacked(v, self.heads, self.head_dim, "v")
        _call(lib().vxg_cache_write, self.k.device, stream, (k, v, table, start, cu) + self._mine(), self._ref, _addr(k),
              ld_k, _addr(v), ld_v, _dt(k), k.shape[0], _addr(table), n_seq, width, _addr(start), _addr(cu))

    def read(self, table: torch.Tensor, start: torch.Tensor, cu: torch.Tensor, total: int,
             dtype: torch.dtype = torch.float32, stream=None):
        """The values of cu[s+1] - cu[s] tokens from position start[s] of each sequence: k, v [total, heads, head_dim]."""
        n_seq, width = self._batch(table, start, cu, stream)
        _need(dtype in _DTYPES, f"element type {dtype} is none of float16, bfloat16, float32")
        dev = self.k.device
        k, v = (_empty((total, self.heads, self.head_dim), dtype, dev, stream) for _ in range(2))
        _call(lib().vxg_cache_read, dev, stream, (table, start, cu) + self._mine(), self._ref, _addr(table), n_seq, width,
              _addr(start), _addr(cu), total, _DTYPES[dtype], _addr(k), _addr(v))
        return k, v

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, cu: torch.Tensor,
               scale: float | None = None, causal: bool = True, window: int = 0, out: torch.Tensor | None = None,
               stream=None) -> torch.Tensor:
        """softmax(scale * q k^T) v of q [rows, heads, head_dim] over the cached tokens of each row's sequence:
        lengths[s] tokens, the rows' own included (write before attending). Query i of n sits at position
        lengths - n + i; it sees positions up to its own (causal) and, with window > 0, the last `window` of them. heads
        is a multiple of the cache's; neighbouring query heads share a cache head. scale defaults to head_dim ** -0.5."""
        heads = q.shape[1] if q.dim() == 3 else 0
        _need(heads > 0 and heads % self.heads == 0, f"{heads} query heads for {self.heads} key / value heads")
        n_seq, width = self._batch(table, lengths, cu, stream, q, out)
        dev = self.k.device
        ld_q = _stacked(q, heads, self.head_dim, "q")
        if out is None:
            out = _empty(tuple(q.shape), q.dtype, dev, stream)
        _need(out.dtype == q.dtype and out.shape == q.shape, "out must be like q")
        ld_out = _stacked(out, heads, self.head_dim, "out")
        total = q.shape[0]
        # the workspace is this call's own: captured graphs and streams never share one
        if torch.cuda.current_device() == dev.index:
            nb = lib().vxg_cache_attention_workspace_bytes(total, n_seq, heads, self.heads, self.head_dim)
        else:
            with torch.cuda.device(dev):
                nb = lib().vxg_cache_attention_workspace_bytes(total, n_seq, heads, self.heads, self.head_dim)
        ws = _empty((nb,), torch.uint8, dev, stream)
        _call(lib().vxg_cache_attention, dev, stream, (q, table, lengths, cu, out) + self._mine(), self._ref, _addr(q),
              ld_q, heads, _dt(q), total, _addr(table), n_seq, width, _addr(lengths), _addr(cu),
              float(scale) if scale is not None else 1.0 / math.sqrt(self.head_dim), int(causal), int(window),
              _addr(out), ld_out, _addr(ws), nb)
        return out
