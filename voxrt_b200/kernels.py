"""Kernel-level API mirroring the reference's kernel trait (crates/voxrt/src/kernels/mod.rs, packed.rs): device
TernaryMatrix / QuantAct operands, the Epilogue enum and gemm_ep, each a thin call into libvxg.so's C ABI.

Device memory and streams are torch CUDA tensors / streams (plumbing only); the arithmetic runs in the library's
sm_100a kernels.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import numpy as np
import torch

from ._lib import check, lib

GROUP = 128


@dataclass(frozen=True)
class Epilogue:
    """kernels/mod.rs:14-21: Store, Silu, AddScaled(s)."""

    kind: int
    scale: float = 0.0

    @staticmethod
    def AddScaled(s: float) -> "Epilogue":
        return Epilogue(2, float(s))


Epilogue.Store = Epilogue(0)
Epilogue.Silu = Epilogue(1)


def _stream_ptr(stream=None):
    s = stream if stream is not None else torch.cuda.current_stream()
    return C.c_void_p(s.cuda_stream)


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}  # vxg_dtype


def _dt(t: torch.Tensor) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"element type {t.dtype} is none of float16, bfloat16, float32")
    return code


def _fits(*sizes: int) -> None:
    """Sizes go to the C entries as int, which ctypes would cut to 32 bits without a word."""
    if max(sizes) > 0x7FFFFFFF:
        raise ValueError(f"a size of {max(sizes)} is more than the entries take (2^31 - 1)")


def _rows(t: torch.Tensor, n: int, d: int, what: str) -> int:
    """Row stride in elements of an [n, d] operand whose rows are contiguous."""
    _fits(n, d)
    if t.shape != (n, d):
        raise ValueError(f"{what} has shape {tuple(t.shape)}, not {(n, d)}")
    if t.is_contiguous():
        return d
    if d > 1 and t.stride(1) != 1:
        raise ValueError(f"{what}'s rows must be contiguous")
    ld = t.stride(0) if n > 1 else d
    if ld < d:
        raise ValueError(f"{what}'s row stride {ld} is below its width {d}")
    return ld


def _gpu(stream, *tensors) -> int:
    """The index of the one GPU that every operand (None left out) and the stream are on."""
    idx = tensors[0].get_device()
    if idx < 0:
        raise ValueError("operands must be CUDA tensors")
    for t in tensors:
        if t is not None and t.get_device() != idx:
            raise ValueError(f"operands on {tensors[0].device} and {t.device}")
    if stream is not None and stream.device.index != idx:
        raise ValueError(f"the stream is not {tensors[0].device}'s")
    return idx


def _like(t: torch.Tensor, shape, dtype, stream) -> torch.Tensor:
    """Memory for an output on t's device: the allocator has to know the stream that writes it."""
    if stream is None:
        return t.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(stream):
        return t.new_empty(shape, dtype=dtype)


def _call(fn, idx: int, stream, used, *args):
    """A C entry on GPU `idx`. On a stream other than the current one, the allocator is told which operands are in use
    there, so that memory freed by the caller meanwhile is not handed out early."""
    if stream is None:
        raw = torch._C._cuda_getCurrentRawStream(idx)
    else:
        raw = stream.cuda_stream
        for t in used:
            if t is not None:
                t.record_stream(stream)
    if torch._C._cuda_getDevice() == idx:
        status = fn(*args, raw)
    else:
        with torch.cuda.device(idx):
            status = fn(*args, raw)
    if status:
        check(status)


def _addr(t):
    return None if t is None else t.data_ptr()


class TernaryMatrix:
    """Ternary weights [out, inp] resident on the GPU in one of the kernels' formats, chosen at load time like the
    reference's Layout (packed.rs:8-27): "2bit" = 2-bit codes tiled per 128 rows x 128 columns, unpacked to int8
    inside the SM; "int8" = int8 rows (4x the bytes, no unpack). f32 scales tile-major in both.
    TernaryMatrix::from_packed_layout (packed.rs:73-130)."""

    def __init__(self, out, inp, group, weights, scales_t, fmt="2bit"):
        self.out, self.inp, self.group, self.fmt = out, inp, group, fmt
        self.weights, self.scales_t = weights, scales_t

    @property
    def codes(self):
        return self.weights

    @classmethod
    def from_packed(cls, qweight, scales_f16, out, inp, group=GROUP, device=None, fmt="2bit"):
        L = lib()
        q = np.ascontiguousarray(qweight, np.uint8)
        s = np.ascontiguousarray(scales_f16).view(np.uint16)
        ns = L.vxg_ternary_scales_count(out, inp, group)
        st = np.empty(ns, np.float32)
        if fmt == "2bit":
            w = np.empty(L.vxg_ternary_codes_bytes(out, inp), np.uint8)
            check(L.vxg_ternary_repack(q.ctypes.data, s.ctypes.data, out, inp, group, w.ctypes.data, st.ctypes.data))
        elif fmt == "int8":
            w = np.empty(L.vxg_ternary_i8_bytes(out, inp), np.int8)
            check(L.vxg_ternary_repack_i8(q.ctypes.data, s.ctypes.data, out, inp, group, w.ctypes.data,
                                          st.ctypes.data))
        else:
            raise ValueError(f"unknown weight format {fmt!r}")
        dev = device if device is not None else torch.device("cuda", torch.cuda.current_device())
        return cls(out, inp, group, torch.from_numpy(w).to(dev), torch.from_numpy(st).to(dev), fmt)

    @classmethod
    def from_module(cls, m: dict, device=None, fmt="2bit"):
        """From a synthetic / model-file module dict {qweight, scales, out, in, group}."""
        return cls.from_packed(m["qweight"], m["scales"], m["out"], m["in"], m["group"], device, fmt)


class QuantAct:
    """int8 activations [n, inp] + f32 scales [n, inp/group] on the GPU (QuantAct, packed.rs:286-298)."""

    def __init__(self, x: torch.Tensor, scales: torch.Tensor, group: int = GROUP):
        assert x.dtype == torch.int8 and x.is_cuda and x.is_contiguous()
        assert scales.dtype == torch.float32 and scales.is_cuda and scales.is_contiguous()
        self.x, self.scales, self.group = x, scales, group
        self.n, self.inp = x.shape


def gemm_ep(w: TernaryMatrix, x: QuantAct, y: torch.Tensor, bias: torch.Tensor | None = None,
            ep: Epilogue = Epilogue.Store, group_sums: torch.Tensor | None = None, stream=None):
    """y[n, out] = epilogue(x x w^T) (+ bias): kernels::gemm_ep (kernels/mod.rs:324-362), on the tensor cores."""
    assert x.inp == w.inp and x.group == w.group, "input width / group mismatch"
    assert y.dtype == torch.float32 and y.is_contiguous() and tuple(y.shape) == (x.n, w.out)
    fn = lib().vxg_gemm_ternary_i8 if w.fmt == "2bit" else lib().vxg_gemm_ternary_i8w
    check(fn(_ptr(x.x), _ptr(x.scales), _ptr(w.weights), _ptr(w.scales_t), x.n, w.out, w.inp, w.group, ep.kind,
             ep.scale, _ptr(bias), _ptr(y), _ptr(group_sums), _stream_ptr(stream)))
    return y


def gemm_silu_quant(w: TernaryMatrix, x: QuantAct, stream=None) -> QuantAct:
    """FeedForward::forward_fused's linear1 (encoder.rs:79-94): Silu GEMM, then per-(row, 128) int8 for linear2,
    fused in one kernel; returns the int8 activations linear2 consumes."""
    assert x.inp == w.inp and x.group == w.group, "input width / group mismatch"
    q = torch.empty((x.n, w.out), dtype=torch.int8, device=x.x.device)
    s = torch.empty((x.n, w.out // GROUP), dtype=torch.float32, device=x.x.device)
    fn = lib().vxg_gemm_ternary_silu_q if w.fmt == "2bit" else lib().vxg_gemm_ternary_silu_q_w
    check(fn(_ptr(x.x), _ptr(x.scales), _ptr(w.weights), _ptr(w.scales_t), x.n, w.out, w.inp, w.group, _ptr(q),
             _ptr(s), _stream_ptr(stream)))
    return QuantAct(q, s, GROUP)


def gemm_qkv_quant(w: TernaryMatrix, x: QuantAct, heads: int, bias_u: torch.Tensor, bias_v: torch.Tensor,
                   stream=None):
    """The stacked q|k|v projection with the attention's per-head operands quantised in the epilogue (encoder.rs:
    138-187, :349-377). Returns (qu, squ, qv, sqv, k, sk, y): int8 [heads, n, 128] codes with f32 [heads, n] scales
    for q + bias_u, q + bias_v and k, and y [n, 3 * heads * 128] f32 whose v columns hold the v projection."""
    assert w.fmt == "2bit" and w.out == 3 * heads * 128 and x.inp == w.inp and x.group == w.group
    dev = x.x.device
    q8 = [torch.empty((heads, x.n, 128), dtype=torch.int8, device=dev) for _ in range(3)]
    sc = [torch.empty((heads, x.n), dtype=torch.float32, device=dev) for _ in range(3)]
    y = torch.empty((x.n, w.out), dtype=torch.float32, device=dev)
    check(lib().vxg_gemm_ternary_qkv_quant(_ptr(x.x), _ptr(x.scales), _ptr(w.weights), _ptr(w.scales_t), x.n, heads,
                                           w.inp, w.group, _ptr(bias_u), _ptr(bias_v), _ptr(q8[0]), _ptr(q8[1]),
                                           _ptr(q8[2]), _ptr(sc[0]), _ptr(sc[1]), _ptr(sc[2]), _ptr(y),
                                           _stream_ptr(stream)))
    return q8[0], sc[0], q8[1], sc[1], q8[2], sc[2], y


def glu_row_order(n: int) -> np.ndarray:
    """Source rows (the reference's [value; gate] order) of the rows of a GLU projection as its GEMM expects them."""
    L = lib()
    order = np.array([L.vxg_glu_source_row(r, n) for r in range(n)], np.int64)
    assert order.min() >= 0, f"GLU projection width {n} unsupported"
    return order


def gemm_glu(w: TernaryMatrix, x: QuantAct, stream=None) -> torch.Tensor:
    """pointwise_conv1 + glu_row (encoder.rs:594-596, tensor.rs:936-940) fused: `w` holds the projection's rows in
    glu_row_order; returns y [n, out / 2] f32."""
    assert w.fmt == "2bit" and x.inp == w.inp and x.group == w.group
    y = torch.empty((x.n, w.out // 2), dtype=torch.float32, device=x.x.device)
    check(lib().vxg_gemm_ternary_glu(_ptr(x.x), _ptr(x.scales), _ptr(w.weights), _ptr(w.scales_t), x.n, w.out, w.inp,
                                     w.group, _ptr(y), _stream_ptr(stream)))
    return y


def gemm(w: TernaryMatrix, x: QuantAct, y: torch.Tensor, bias: torch.Tensor | None = None, stream=None):
    """kernels::gemm (kernels/mod.rs:319-321)."""
    return gemm_ep(w, x, y, bias, Epilogue.Store, stream=stream)


def quantize(x: torch.Tensor, group: int = GROUP, stream=None) -> QuantAct:
    """QuantAct::quantize (packed.rs:302-312) on the GPU: per-(token, group) absmax/127 int8. f32, f16 or bf16 rows (any
    row stride); group = x.shape[1] gives the one scale a token that gemm_i8 reads."""
    idx = _gpu(stream, x)
    if x.dim() != 2 or x.shape[1] == 0 or group <= 0:
        raise ValueError("quantize takes rows")
    n, d = x.shape
    dt, ld = _dt(x), _rows(x, n, d, "x")
    q = _like(x, (n, d), torch.int8, stream)
    s = _like(x, (n, d // group), torch.float32, stream)
    if x.dtype == torch.float32 and x.is_contiguous() and d <= 8192:
        _call(lib().vxg_quantize_rows, idx, stream, (x,), x.data_ptr(), n, d, group, q.data_ptr(), s.data_ptr())
    else:
        _call(lib().vxg_quantize_tokens, idx, stream, (x,), x.data_ptr(), ld, dt, n, d, group, q.data_ptr(), s.data_ptr())
    return QuantAct(q, s, group)


def _scales_of(x: QuantAct) -> torch.Tensor:
    """x's scales, one for each of its groups: the kernels read that many."""
    _fits(x.n, x.inp, x.group)
    if x.group <= 0 or x.inp % x.group != 0 or x.scales.numel() != x.n * (x.inp // x.group):
        raise ValueError(f"{x.scales.numel()} scales for {x.n} rows of width {x.inp} in groups of {x.group}")
    return x.scales


def dequantize(x: QuantAct, dtype: torch.dtype = torch.float32, stream=None) -> torch.Tensor:
    """The values that the codes stand for, q * scale, rounded once to `dtype`."""
    q, s = x.x, _scales_of(x)
    idx = _gpu(stream, q, s)
    if dtype not in _DTYPES:
        raise ValueError(f"element type {dtype} is none of float16, bfloat16, float32")
    out = _like(q, q.shape, dtype, stream)
    _call(lib().vxg_dequantize_rows, idx, stream, (q, s), q.data_ptr(), s.data_ptr(), x.n, x.inp, x.group,
          _DTYPES[dtype], out.data_ptr())
    return out


def _rms(x, n, d, gamma, eps, v, vs, x_res, y, group, q, s, stream):
    idx = _gpu(stream, x, gamma, v, x_res, y)
    dt = _dt(x)
    if gamma.dtype != torch.float32 or not gamma.is_contiguous() or gamma.numel() != d:
        raise ValueError("gamma must be d contiguous float32 values")
    ld_v = ld_r = ld_y = 0
    if v is not None:
        ld_v = _rows(v, n, d, "v")
    if x_res is not None:
        ld_r = _rows(x_res, n, d, "x_res")
    if y is not None:
        ld_y = _rows(y, n, d, "y")
    for t in (v, x_res, y):
        if t is not None and t.dtype != x.dtype:
            raise ValueError("v, x_res and y must have x's element type")
    _call(lib().vxg_rms_quant, idx, stream, (x, gamma, v, x_res, y), x.data_ptr(), _rows(x, n, d, "x"), _addr(v), ld_v, vs,
          dt, n, d, gamma.data_ptr(), eps, _addr(x_res), ld_r, _addr(y), ld_y, group, _addr(q), _addr(s))


def rms_quant(x: torch.Tensor, gamma: torch.Tensor, group: int | None = None, eps: float = 1e-6,
              v: torch.Tensor | None = None, vs: float = 1.0, x_res: torch.Tensor | None = None,
              y: torch.Tensor | None = None, stream=None) -> QuantAct:
    """RMSNorm -> int8 with the residual add in front, in one pass: h = x + vs * v (stored to x_res, which may be x),
    h / sqrt(mean h^2 + eps) * gamma (stored to y, unquantised, when given), then int8 per token (group None or d: for
    gemm_i8) or per `group` columns (128: for the ternary GEMMs). f32, f16 or bf16 rows of any stride; gamma f32."""
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError("x must be [n, d]")
    n, d = x.shape
    _fits(n, d)
    group = d if group is None else int(group)
    if group <= 0 or d % group != 0:
        raise ValueError(f"group {group} does not divide the row width {d}")
    if x.get_device() < 0:
        raise ValueError("operands must be CUDA tensors")
    q = _like(x, (n, d), torch.int8, stream)
    s = _like(x, (n, d // group), torch.float32, stream)
    _rms(x, n, d, gamma, eps, v, vs, x_res, y, group, q, s, stream)
    return QuantAct(q, s, group)


def rms_norm(x: torch.Tensor, gamma: torch.Tensor, out: torch.Tensor, eps: float = 1e-6, v: torch.Tensor | None = None,
             vs: float = 1.0, x_res: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """rms_quant without the quantisation (the norm in front of an output head) -> out (may be x if x_res is not)."""
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError("x must be [n, d]")
    _rms(x, *x.shape, gamma, eps, v, vs, x_res, out, 1, None, None, stream)
    return out


class Int8Matrix:
    """int8 weights [out, inp] with one f32 scale per output row, resident on the GPU: gemm_i8's weights."""

    def __init__(self, w: torch.Tensor, scales: torch.Tensor):
        if w.dtype != torch.int8 or w.get_device() < 0 or w.dim() != 2 or not w.is_contiguous():
            raise ValueError("weights must be a contiguous int8 CUDA tensor [out, inp]")
        self.out, self.inp = w.shape
        if (scales.dtype != torch.float32 or scales.get_device() != w.get_device() or not scales.is_contiguous() or
                scales.numel() != self.out):
            raise ValueError("one float32 scale per output row, on the weights' device")
        self.w, self.scales = w, scales

    @classmethod
    def from_float(cls, w: torch.Tensor) -> "Int8Matrix":
        """Float weights [out, inp] on the GPU, each row quantised to its own absmax / 127."""
        a = quantize(w, w.shape[1])
        return cls(a.x, a.scales.view(-1))


def gemm_i8(w: Int8Matrix, x: QuantAct, y: torch.Tensor, bias: torch.Tensor | None = None,
            ep: Epilogue = Epilogue.Store, stream=None) -> torch.Tensor:
    """y[n, out] = epilogue(x w^T + bias) for int8 activations with one scale a token: exact int32 sums, then
    sum * (token scale * channel scale). y: f32, f16 or bf16 rows of any stride, read first for AddScaled."""
    wq, xq, sx = w.w, x.x, _scales_of(x)
    idx = _gpu(stream, wq, xq, sx, y, bias)
    n, out, inp = x.n, w.out, w.inp
    if x.inp != inp or x.group != inp:
        raise ValueError(f"activations of width {x.inp} and group {x.group} for weights of width {inp}: one scale a token "
                         "is wanted")
    if bias is not None and (bias.dtype != torch.float32 or not bias.is_contiguous() or bias.numel() != out):
        raise ValueError("bias must be `out` contiguous float32 values")
    _call(lib().vxg_gemm_i8, idx, stream, (xq, sx, wq, w.scales, y, bias), xq.data_ptr(), sx.data_ptr(), wq.data_ptr(),
          w.scales.data_ptr(), n, out, inp, ep.kind, ep.scale, _addr(bias), _dt(y), y.data_ptr(), _rows(y, n, out, "y"))
    return y


def ln_quant(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, group: int = GROUP, pre=None,
             x_out: torch.Tensor | None = None, stream=None) -> QuantAct:
    """TernaryLinear::prepare_normed (ternary_linear.rs:132-158): LayerNorm(x) -> int8, fused. `pre` = (g0, b0)
    applies a first LayerNorm whose f32 output goes to x_out (norm_out of the previous layer)."""
    n, d = x.shape
    q = torch.empty((n, d), dtype=torch.int8, device=x.device)
    s = torch.empty((n, d // group), dtype=torch.float32, device=x.device)
    g0, b0 = pre if pre is not None else (None, None)
    check(lib().vxg_ln_quant(_ptr(x), n, d, _ptr(g0), _ptr(b0), _ptr(x_out), _ptr(gamma), _ptr(beta), group,
                             _ptr(q), _ptr(s), _stream_ptr(stream)))
    return QuantAct(q, s, group)


def layer_norm(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, out: torch.Tensor, stream=None):
    """LayerNormP::forward (encoder.rs:60-62) -> out (may be x)."""
    n, d = x.shape
    check(lib().vxg_ln_quant(_ptr(x), n, d, _ptr(gamma), _ptr(beta), _ptr(out), None, None, GROUP, None, None,
                             _stream_ptr(stream)))
    return out


def attention_i8(qkv: torch.Tensor, rel_k: torch.Tensor, tmax: int, offsets, lengths, bias_u: torch.Tensor,
                 bias_v: torch.Tensor, heads: int = 8, scaling: float | None = None, want_f32: bool = True,
                 want_q: bool = True, workspace: torch.Tensor | None = None, stream=None):
    """attn_core_int8 (encoder.rs:317-534) for utterances stacked in qkv rows. Returns (ctx f32 | None,
    QuantAct of ctx per head | None)."""
    rows, ld = qkv.shape
    d = heads * 128
    if scaling is None:
        scaling = float(np.float32(1.0) / np.sqrt(np.float32(128.0), dtype=np.float32))
    off = np.ascontiguousarray(offsets, np.int32)
    ln = np.ascontiguousarray(lengths, np.int32)
    nb = lib().vxg_attention_workspace_bytes(rows, tmax, len(ln), heads)
    if workspace is None or workspace.numel() < nb:
        workspace = torch.empty(nb, dtype=torch.uint8, device=qkv.device)
    ctx = torch.zeros((rows, d), dtype=torch.float32, device=qkv.device) if want_f32 else None
    cq = torch.zeros((rows, d), dtype=torch.int8, device=qkv.device) if want_q else None
    cs = torch.zeros((rows, heads), dtype=torch.float32, device=qkv.device) if want_q else None
    check(lib().vxg_attention_i8(_ptr(qkv), ld, _ptr(rel_k), tmax, off.ctypes.data, ln.ctypes.data, len(ln),
                                 _ptr(bias_u), _ptr(bias_v), heads, 128, float(scaling), _ptr(ctx), _ptr(cq),
                                 _ptr(cs), _ptr(workspace), workspace.numel(), _stream_ptr(stream)))
    return ctx, (QuantAct(cq, cs, 128) if want_q else None)


def fold_bn(dw, gamma, beta, mean, var):
    """ConvModule::load (encoder.rs:546-579): BN(eval) folded into the depthwise conv -> (dw_t [k, d], bias [d])."""
    dw = np.ascontiguousarray(dw, np.float32)
    d, k = dw.shape[0], dw.shape[-1]
    dw_t = np.empty((k, d), np.float32)
    dw_b = np.empty(d, np.float32)
    args = [np.ascontiguousarray(a, np.float32) for a in (gamma, beta, mean, var)]
    check(lib().vxg_fold_bn(dw.ctypes.data, *[a.ctypes.data for a in args], d, k, dw_t.ctypes.data,
                            dw_b.ctypes.data))
    return dw_t, dw_b


def conv_glu_dw_silu(g: torch.Tensor, offsets, lengths, dw_t: torch.Tensor, dw_b: torch.Tensor, want_f32=True,
                     want_q=True, stream=None):
    """ConvModule middle (encoder.rs:596-626): GLU -> depthwise conv -> SiLU (-> int8 for pointwise_conv2)."""
    rows, ld = g.shape
    k, d = dw_t.shape
    off = np.ascontiguousarray(offsets, np.int32)
    ln = np.ascontiguousarray(lengths, np.int32)
    nb = lib().vxg_conv_workspace_bytes(rows, len(ln))
    ws = torch.empty(nb, dtype=torch.uint8, device=g.device)
    hb = torch.zeros((rows, d), dtype=torch.float32, device=g.device) if want_f32 else None
    q = torch.zeros((rows, d), dtype=torch.int8, device=g.device) if want_q else None
    s = torch.zeros((rows, d // 128), dtype=torch.float32, device=g.device) if want_q else None
    check(lib().vxg_conv_glu_dw_silu_quant(_ptr(g), ld, off.ctypes.data, ln.ctypes.data, len(ln), _ptr(dw_t),
                                           _ptr(dw_b), d, k, _ptr(hb), _ptr(q), _ptr(s), _ptr(ws), nb,
                                           _stream_ptr(stream)))
    return hb, (QuantAct(q, s, 128) if want_q else None)


class Subsampling:
    """Device weights of the dw-striding Conv2d x8 front end in the layouts Subsampling::load prepares
    (subsampling.rs:31-96): 3x3 kernels tap-major [9][C], pointwise [C][C], final linear with its columns permuted
    to channels-last (f*C + c)."""

    def __init__(self, sw: dict, device=None):
        dev = device if device is not None else torch.device("cuda", torch.cuda.current_device())
        c = sw["conv0_w"].shape[0]
        k = sw["conv0_w"].shape[-1]
        d = sw["lin_w"].shape[0]
        f3 = sw["lin_w"].shape[1] // c
        tap = lambda w: np.ascontiguousarray(np.asarray(w, np.float32).reshape(c, k * k).T)
        lw = np.asarray(sw["lin_w"], np.float32).reshape(d, c, f3).transpose(0, 2, 1).reshape(d, f3 * c)
        T = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(dev)
        self.t = [T(tap(sw["conv0_w"])), T(sw["conv0_b"]), T(tap(sw["dw1_w"])), T(sw["dw1_b"]),
                  T(np.asarray(sw["pw1_w"]).reshape(c, c)), T(sw["pw1_b"]), T(tap(sw["dw2_w"])), T(sw["dw2_b"]),
                  T(np.asarray(sw["pw2_w"]).reshape(c, c)), T(sw["pw2_b"]), T(lw), T(sw["lin_b"])]
        self.n_mels, self.d_model = int(sw["n_mels"]), d

    @staticmethod
    def out_frames(t_in: int) -> int:
        return lib().vxg_sub_out_frames(int(t_in))

    def forward(self, feats: torch.Tensor, t_in, stream=None) -> torch.Tensor:
        """Stacked feats [sum t_in, n_mels] -> stacked [sum out_frames, d_model] (Subsampling::forward)."""
        t_in = np.ascontiguousarray(t_in, np.int32)
        rows = sum(self.out_frames(t) for t in t_in)
        out = torch.empty((rows, self.d_model), dtype=torch.float32, device=feats.device)
        nb = lib().vxg_subsampling_workspace_bytes(t_in.ctypes.data, len(t_in), self.n_mels)
        ws = torch.empty(nb, dtype=torch.uint8, device=feats.device)
        check(lib().vxg_subsampling(_ptr(feats), t_in.ctypes.data, len(t_in), self.n_mels,
                                    *[_ptr(a) for a in self.t], self.d_model, _ptr(out), _ptr(ws), nb,
                                    _stream_ptr(stream)))
        return out
