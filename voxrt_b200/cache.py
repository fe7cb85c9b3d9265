"""Paged int8 key / value cache and the attention over it: KvCache.write, read and attend, each a thin call into
libvxg.so's C ABI on torch CUDA tensors. Batches are stacked along the token axis; lengths and offsets are device tensors,
so a decode step can be captured in a CUDA graph and replayed as the sequences grow."""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import lib
from .kernels import _DTYPES, _call, _dt, _fits, _gpu, _like


class _Desc(C.Structure):  # vxg_kv_cache
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scales", C.c_void_p), ("v_scales", C.c_void_p),
                ("n_pages", C.c_int), ("heads", C.c_int), ("page", C.c_int), ("head_dim", C.c_int)]


def _stacked(t: torch.Tensor, heads: int, hd: int, what: str) -> int:
    """Row stride of a stacked [rows, heads, head_dim] operand whose rows are contiguous."""
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != hd:
        raise ValueError(f"{what} has shape {tuple(shape)}, not (rows, {heads}, {hd})")
    _fits(shape[0])
    if t.is_contiguous():
        return heads * hd
    if t.stride(2) != 1 or (heads > 1 and t.stride(1) != hd):
        raise ValueError(f"{what}'s rows must be contiguous")
    return t.stride(0) if shape[0] > 1 else heads * hd


class KvCache:
    """A pool of n_pages pages: k, v int8 [n_pages, heads, page, head_dim] with one f32 scale per (page, head) in ks and
    vs. page 16, 32, 64 or 128; head_dim 64 or 128. The pool does not know which pages are whose: a page table
    [n_seq, max_pages] (int32) lists each sequence's pages in order, entries behind its last page are not read."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, ks: torch.Tensor, vs: torch.Tensor):
        if k.dim() != 4 or k.dtype != torch.int8 or not k.is_contiguous() or k.get_device() < 0:
            raise ValueError("k must be a contiguous int8 CUDA tensor [n_pages, heads, page, head_dim]")
        if v.shape != k.shape or v.dtype != torch.int8 or not v.is_contiguous() or v.device != k.device:
            raise ValueError("v must be like k")
        for t in (ks, vs):
            if t.shape != k.shape[:2] or t.dtype != torch.float32 or not t.is_contiguous() or t.device != k.device:
                raise ValueError("scales must be contiguous float32 [n_pages, heads] on the codes' device")
        self.k, self.v, self.ks, self.vs = k, v, ks, vs
        self.n_pages, self.heads, self.page, self.head_dim = k.shape
        self._desc = _Desc(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), *k.shape)
        self._ref = C.addressof(self._desc)
        self._ws_bytes = {}  # attend's workspace size by its shape

    @classmethod
    def empty(cls, n_pages: int, heads: int, head_dim: int, page: int = 64, device=None) -> "KvCache":
        dev = device if device is not None else torch.device("cuda", torch.cuda.current_device())
        codes = [torch.zeros((n_pages, heads, page, head_dim), dtype=torch.int8, device=dev) for _ in range(2)]
        scales = [torch.zeros((n_pages, heads), dtype=torch.float32, device=dev) for _ in range(2)]
        return cls(*codes, *scales)

    def _batch(self, table, a, cu, stream, *more):
        """(GPU, sequences, pages of a table row) of a batch whose lengths and offsets are a and cu."""
        idx = _gpu(stream, self.k, table, a, cu, *more)
        for t in (table, a, cu):
            if t.dtype != torch.int32 or not t.is_contiguous():
                raise ValueError("the page table, lengths and offsets must be contiguous int32")
        n_seq, width = table.shape if table.dim() == 2 else (-1, 0)
        if a.shape != (n_seq,) or cu.shape != (n_seq + 1,):
            raise ValueError(f"page table {tuple(table.shape)}, lengths {tuple(a.shape)} and offsets {tuple(cu.shape)} do "
                             "not belong to one batch")
        _fits(n_seq, width)
        return idx, n_seq, width

    def write(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor, cu: torch.Tensor,
              stream=None) -> None:
        """Quantise and append k and v [rows, heads, head_dim] (f32, f16 or bf16, any row stride): rows cu[s] .. cu[s+1]
        go to positions start[s] .. of sequence s. A started page's scale grows when it has to, and its earlier codes
        with it. Pages that are written must belong to one sequence each."""
        idx, n_seq, width = self._batch(table, start, cu, stream, k, v)
        if k.dtype != v.dtype or k.shape != v.shape:
            raise ValueError("k and v must be alike")
        heads, hd = self.heads, self.head_dim
        ld_k, ld_v = _stacked(k, heads, hd, "k"), _stacked(v, heads, hd, "v")
        _call(lib().vxg_cache_write, idx, stream, (k, v, table, start, cu, self.k, self.v, self.ks, self.vs), self._ref,
              k.data_ptr(), ld_k, v.data_ptr(), ld_v, _dt(k), k.shape[0], table.data_ptr(), n_seq, width,
              start.data_ptr(), cu.data_ptr())

    def read(self, table: torch.Tensor, start: torch.Tensor, cu: torch.Tensor, total: int,
             dtype: torch.dtype = torch.float32, stream=None):
        """The values of cu[s+1] - cu[s] tokens from position start[s] of each sequence: k, v [total, heads, head_dim]."""
        idx, n_seq, width = self._batch(table, start, cu, stream)
        if dtype not in _DTYPES:
            raise ValueError(f"element type {dtype} is none of float16, bfloat16, float32")
        _fits(total)
        shape = (total, self.heads, self.head_dim)
        k, v = _like(self.k, shape, dtype, stream), _like(self.k, shape, dtype, stream)
        _call(lib().vxg_cache_read, idx, stream, (table, start, cu, self.k, self.v, self.ks, self.vs), self._ref,
              table.data_ptr(), n_seq, width, start.data_ptr(), cu.data_ptr(), total, _DTYPES[dtype], k.data_ptr(),
              v.data_ptr())
        return k, v

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, cu: torch.Tensor,
               scale: float | None = None, causal: bool = True, window: int = 0, out: torch.Tensor | None = None,
               stream=None) -> torch.Tensor:
        """softmax(scale * q k^T) v of q [rows, heads, head_dim] over the cached tokens of each row's sequence:
        lengths[s] tokens, the rows' own included (write before attending). Query i of n sits at position
        lengths - n + i; it sees positions up to its own (causal) and, with window > 0, the last `window` of them. heads
        is a multiple of the cache's; neighbouring query heads share a cache head. scale defaults to head_dim ** -0.5."""
        idx, n_seq, width = self._batch(table, lengths, cu, stream, q, out)
        if torch._C._cuda_getDevice() != idx:  # the workspace's size is the current device's
            with torch.cuda.device(idx):
                return self.attend(q, table, lengths, cu, scale, causal, window, out, stream)
        heads, hd = q.shape[1] if q.dim() == 3 else 0, self.head_dim
        if heads == 0 or heads % self.heads != 0:
            raise ValueError(f"{heads} query heads for {self.heads} key / value heads")
        if window < 0:
            raise ValueError("window must not be negative")
        dt, ld_q = _dt(q), _stacked(q, heads, hd, "q")
        if out is None:
            out = _like(q, q.shape, q.dtype, stream)
        elif out.dtype != q.dtype or out.shape != q.shape:
            raise ValueError("out must be like q")
        ld_out = _stacked(out, heads, hd, "out")
        total = q.shape[0]
        # the workspace is this call's own: captured graphs and streams never share one
        nb = self._ws_bytes.get((total, n_seq, heads, dt))
        if nb is None:
            nb = lib().vxg_cache_attention_workspace_bytes(total, n_seq, heads, self.heads, hd, dt)
            if len(self._ws_bytes) < 4096:
                self._ws_bytes[total, n_seq, heads, dt] = nb
        ws = _like(q, (nb,), torch.uint8, stream)
        _call(lib().vxg_cache_attention, idx, stream, (q, table, lengths, cu, out, self.k, self.v, self.ks, self.vs),
              self._ref, q.data_ptr(), ld_q, heads, dt, total, table.data_ptr(), n_seq, width, lengths.data_ptr(),
              cu.data_ptr(), scale if scale is not None else hd ** -0.5, causal, min(window, 0x7FFFFFFF), out.data_ptr(), ld_out,
              ws.data_ptr(), nb)
        return out
