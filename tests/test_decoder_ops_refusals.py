"""CPU: what the int8 decoder entries refuse, before anything reaches a GPU, and what they accept as empty."""
import ctypes as C
import os
import subprocess
import sys

import pytest
import torch

from voxrt_b200 import _lib
from voxrt_b200.cache import KvCache, _Desc
from voxrt_b200.kernels import Epilogue, Int8Matrix, dequantize, gemm_i8, quantize, rms_quant

P = 1 << 20  # stands for a device address: no refused or empty call follows it
ARG, UNSUP, OK = _lib.VXG_ERR_ARG, _lib.VXG_ERR_UNSUPPORTED, _lib.VXG_OK


def _rms(x=P, ld=64, v=None, dt=2, n=4, d=64, gamma=P, eps=1e-6, res=None, y=None, group=64, q=P, s=P, ldv=64, ldr=64):
    return _lib.lib().vxg_rms_quant(x, ld, v, ldv, 1.0, dt, n, d, gamma, eps, res, ldr, y, 64, group, q, s, None)


@pytest.mark.parametrize("kw,want", [
    (dict(x=None), ARG), (dict(gamma=None), ARG), (dict(q=None, s=None), ARG), (dict(s=None), ARG), (dict(dt=3), ARG),
    (dict(dt=-1), ARG), (dict(n=-1), ARG), (dict(d=0, group=1), ARG), (dict(ld=63), ARG), (dict(v=P, ldv=1), ARG),
    (dict(v=P, res=P, ldr=63), ARG), (dict(res=P), ARG), (dict(eps=-1.0), ARG), (dict(eps=float("nan")), ARG),
    (dict(group=0), ARG), (dict(group=48), ARG), (dict(group=4), UNSUP), (dict(d=32776, ld=32776, group=32776), UNSUP),
    (dict(n=0), OK), (dict(n=0, x=None, gamma=None, q=None, s=None), OK)])
def test_rms_quant(kw, want):
    assert _rms(**kw) == want
    assert want == OK or _lib.lib().vxg_last_error()


def test_quantize_and_dequantize():
    L = _lib.lib()
    for a, want in (((P, 64, 2, 4, 64, 64, None, P), ARG), ((None, 64, 2, 4, 64, 64, P, P), ARG),
                    ((P, 64, 9, 4, 64, 64, P, P), ARG), ((P, 60, 2, 4, 64, 64, P, P), ARG),
                    ((P, 64, 2, 4, 64, 2, P, P), UNSUP), ((P, 64, 2, 0, 64, 64, P, P), OK)):
        assert L.vxg_quantize_tokens(*a, None) == want
    for a, want in (((P, P, 4, 64, 64, 2, None), ARG), ((P, P, 4, 64, 48, 2, P), ARG), ((P, P, 4, 64, 64, 5, P), ARG),
                    ((P, P, -1, 64, 64, 2, P), ARG), ((P, P, 0, 64, 64, 2, P), OK)):
        assert L.vxg_dequantize_rows(*a, None) == want


@pytest.mark.parametrize("kw,want", [
    (dict(x=None), ARG), (dict(x=P + 8), ARG), (dict(w=P + 4), ARG), (dict(m=-1), ARG), (dict(n=0), ARG), (dict(ep=3), ARG),
    (dict(dt=4), ARG), (dict(ld=31), ARG), (dict(k=40), UNSUP), (dict(k=131072), UNSUP), (dict(m=0), OK)])
def test_gemm(kw, want):
    a = dict(x=P, sx=P, w=P, sw=P, m=4, n=32, k=64, ep=0, s=0.0, bias=None, dt=2, y=P, ld=32)
    a.update(kw)
    assert _lib.lib().vxg_gemm_i8(*a.values(), None) == want


def _cache(**kw):
    a = dict(k=P, v=P, k_scales=P, v_scales=P, n_pages=8, heads=2, page=16, head_dim=64)
    a.update(kw)
    return _Desc(**a)


BAD_CACHE = [(dict(k=None), ARG), (dict(k=P + 4), ARG), (dict(v_scales=None), ARG), (dict(n_pages=0), ARG),
             (dict(heads=0), ARG), (dict(page=8), UNSUP), (dict(page=48), UNSUP), (dict(head_dim=96), UNSUP),
             (dict(n_pages=1 << 27), UNSUP)]


def _write(c, k=P, ldk=128, v=P, ldv=128, dt=2, total=4, table=P, n_seq=1, width=4, start=P, cu=P):
    return _lib.lib().vxg_cache_write(C.addressof(c), k, ldk, v, ldv, dt, total, table, n_seq, width, start, cu, None)


def _attend(c, q=P, ld=256, heads=4, dt=2, total=4, table=P, n_seq=1, width=4, lens=P, cu=P, scale=0.1, causal=1, window=0,
            out=P, ldo=256, ws=P, nb=1 << 30):
    return _lib.lib().vxg_cache_attention(C.addressof(c), q, ld, heads, dt, total, table, n_seq, width, lens, cu, scale,
                                          causal, window, out, ldo, ws, nb, None)


def _read(c, table=P, n_seq=1, width=4, start=P, cu=P, total=4, dt=2, k=P, v=P):
    return _lib.lib().vxg_cache_read(C.addressof(c), table, n_seq, width, start, cu, total, dt, k, v, None)


@pytest.mark.parametrize("kw,want", BAD_CACHE)
def test_bad_cache(kw, want):
    c = _cache(**kw)
    assert _write(c) == want and _attend(c) == want and _read(c) == want
    assert _lib.lib().vxg_cache_write(None, P, 128, P, 128, 2, 4, P, 1, 4, P, P, None) == ARG


@pytest.mark.parametrize("kw,want", [
    (dict(table=None), ARG), (dict(cu=None), ARG), (dict(total=-1), ARG), (dict(n_seq=-1), ARG), (dict(width=0), ARG),
    (dict(dt=7), ARG), (dict(width=1 << 27), UNSUP), (dict(total=0), OK), (dict(n_seq=0), OK), (dict(n_seq=0, table=None, cu=None), OK)])
def test_bad_batch(kw, want):
    c = _cache()
    assert _write(c, **kw) == want and _attend(c, **kw) == want and _read(c, **kw) == want


def test_batches_of_too_many_sequences():
    for n_seq in ((1 << 30) + 1, 0x7FFFFFFF):
        for call in (_write, _attend, _read):
            assert call(_cache(), n_seq=n_seq) == UNSUP and b"sequences" in _lib.lib().vxg_last_error()


def test_write_read_attend():
    c = _cache()
    for kw in (dict(k=None), dict(v=None), dict(ldk=127), dict(ldv=1), dict(start=None)):
        assert _write(c, **kw) == ARG
    assert _read(c, k=None, v=None) == ARG and _read(c, k=P + 8) == ARG
    for kw in (dict(heads=3), dict(heads=0), dict(window=-1), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(q=None), dict(ws=None), dict(ld=255), dict(ldo=128), dict(ld=257), dict(q=P + 8), dict(ws=P + 8),
               dict(nb=16), dict(lens=None)):
        assert _attend(c, **kw) == ARG, kw
    L = _lib.lib()
    assert L.vxg_cache_attention_workspace_bytes(0, 1, 4, 2, 64, 2) == 0
    assert L.vxg_cache_attention_workspace_bytes(4, 1, 3, 2, 64, 2) == 0
    assert L.vxg_cache_attention_workspace_bytes(4, 1, 4, 2, 64, 2) > 0


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf"), 2.4e38, -3e38])
def test_scales_beyond_the_kernels_range(scale):
    """The kernels take the scale times log2(e), which an accepted 3e38 turned into infinity."""
    assert _attend(_cache(), scale=scale) == ARG and b"scale" in _lib.lib().vxg_last_error()
    if abs(scale) < 1e39:
        assert _attend(_cache(), scale=scale / 2, nb=16) == ARG and b"workspace" in _lib.lib().vxg_last_error()


def test_python_refusals():
    x = torch.zeros((2, 64))
    with pytest.raises(ValueError, match="CUDA"):
        rms_quant(x, torch.ones(64))
    with pytest.raises(ValueError, match="divide"):
        rms_quant(x, torch.ones(64), group=48)
    with pytest.raises(ValueError, match="CUDA"):
        quantize(x.half(), 64)
    with pytest.raises(ValueError, match="int8"):
        Int8Matrix(x, torch.ones(2))
    with pytest.raises(ValueError, match="int8"):
        KvCache(x, x, x, x)
    assert Epilogue.AddScaled(2.0).kind == 2


class _Act:
    """A QuantAct whose tensors may lie on the CPU."""

    def __init__(self, n, inp, scales, group):
        self.x, self.scales, self.group, self.n, self.inp = torch.zeros((n, inp), dtype=torch.int8), scales, group, n, inp


@pytest.mark.parametrize("kw", [dict(m=0x7FFFFFFF), dict(m=0x7FFFFF01), dict(n=0x7FFFFFFF, ld=0x7FFFFFFF),
                                dict(m=1, n=0x7FFFFF01, ld=0x7FFFFF01)])
def test_gemm_sizes_that_pass_31_bits_within_a_tile(kw):
    test_gemm(kw, UNSUP)


@pytest.mark.parametrize("shape,group", [((1, 1), 64), ((3, 1), 64), ((4, 3), 16), ((16,), 15), ((5, 1), 64), ((0, 1), 64), ((4, 1), 0)])
def test_scales_that_do_not_fit_the_codes(shape, group):
    """Too few scales (left over from a slice, or meant to be broadcast) would be read past their end."""
    a = _Act(4, 64, torch.ones(shape), group)
    with pytest.raises(ValueError, match="scales for 4 rows"):
        dequantize(a)
    w = _Act(8, 64, None, 64)
    w.w, w.scales, w.out = w.x, torch.ones(8), 8
    with pytest.raises(ValueError, match="scales for 4 rows"):
        gemm_i8(w, a, torch.zeros((4, 8)))
    for op in (lambda x: dequantize(x), lambda x: gemm_i8(w, x, torch.zeros((4, 8)))):  # the right count goes on
        with pytest.raises(ValueError, match="CUDA"):
            op(_Act(4, 64, torch.ones((4, 1)), 64))


def test_quantize_rows_of_an_empty_batch():
    L = _lib.lib()
    assert L.vxg_quantize_rows(None, 0, 64, 64, None, None, None) == OK
    for a in ((None, 4, 64, 64, P, P), (P, 4, 64, 64, None, P), (P, 4, 64, 64, P, None), (P, -1, 64, 64, P, P),
              (P, 4, 64, 48, P, P), (P, 4, 64, 0, P, P), (None, 0, 0, 1, None, None), (P, 4, 8200, 8200, P, P)):
        assert L.vxg_quantize_rows(*a, None) == ARG


@pytest.mark.parametrize("dtype,pad", [(torch.float32, 0), (torch.float32, 8), (torch.bfloat16, 0)])
def test_quantize_goes_to_the_operands_gpu(monkeypatch, dtype, pad):
    """Whatever the type and stride: the call is made on the operand's GPU and the given stream, with x in use there, and
    the outputs are allocated for that stream."""
    from voxrt_b200 import kernels as K

    seen = []
    monkeypatch.setattr(K, "_gpu", lambda stream, *t: 1)
    monkeypatch.setattr(K, "_like", lambda t, shape, dt, stream: seen.append(stream) or torch.empty(shape, dtype=dt))
    monkeypatch.setattr(K, "_call", lambda fn, idx, stream, used, *a: seen.append((idx, stream, used[0])))
    monkeypatch.setattr(K, "QuantAct", lambda *a: a)
    x = torch.zeros((4, 64 + pad), dtype=dtype)[:, :64]
    q, s, group = K.quantize(x, 32, stream="side")
    assert seen[:2] == ["side", "side"] and seen[2][:2] == (1, "side") and seen[2][2] is x
    assert q.shape == (4, 64) and s.shape == (4, 2) and group == 32


NO_GPU = """
from voxrt_b200 import _lib
from voxrt_b200.cache import _Desc
import ctypes as C
L, P = _lib.lib(), 1 << 20
c = _Desc(P, P, P, P, 8, 2, 16, 64)
for m in (1, 40, 65, 5000):
    assert L.vxg_gemm_i8(P, P, P, P, m, 32, 64, 0, 0.0, None, 2, P, 32, None) not in (0, 5) and L.vxg_last_error()
for n in (1, 5000):
    assert L.vxg_rms_quant(P, 64, None, 64, 1.0, 2, n, 64, P, 1e-6, None, 64, None, 64, 64, P, P, None) == 2
    assert L.vxg_quantize_tokens(P, 64, 2, n, 64, 64, P, P, None) == 2
    assert L.vxg_dequantize_rows(P, P, n, 64, 64, 2, P, None) == 2
    for dt in range(3):
        assert L.vxg_cache_attention(C.addressof(c), P, 256, 4, dt, n, P, 1, 4, P, P, 0.1, 1, 0, P, 256, P, 1 << 40, None) != 0
        assert L.vxg_cache_write(C.addressof(c), P, 128, P, 128, dt, n, P, 1, 4, P, P, None) != 0
        assert L.vxg_cache_read(C.addressof(c), P, 1, 4, P, P, n, dt, P, P, None) != 0
    assert L.vxg_cache_attention_workspace_bytes(n, 1, 4, 2, 64, 2) > 0
"""


def test_without_a_gpu():
    """A process that sees no GPU gets errors from every entry, and lives on."""
    env = {**os.environ, "CUDA_VISIBLE_DEVICES": ""}
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", NO_GPU], cwd=root, env=env, capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stderr[-800:])


def test_device_status_says_what_happened(monkeypatch):
    for code, status, text in ((0x302, ARG, "page id, length or offset"), (0x301, _lib.VXG_ERR_TIMEOUT, "bounded wait")):
        monkeypatch.setattr(_lib, "device_status", lambda: code)
        with pytest.raises(_lib.VxgError, match=text) as e:
            _lib.check_device()
        assert e.value.status == status
    monkeypatch.setattr(_lib, "device_status", lambda: 0)
    _lib.check_device()


def test_operands_across_an_element_boundary():
    """A pointer that is no multiple of its element would fault on the GPU."""
    L, c = _lib.lib(), _cache()

    def refused(status):
        return status == ARG and b"aligned" in L.vxg_last_error()

    for dt, off in ((0, 1), (1, 1), (2, 2)):
        for kw in (dict(x=P + off), dict(v=P + off), dict(v=P, res=P + off), dict(y=P + off), dict(gamma=P + 2), dict(s=P + 1)):
            assert refused(_rms(dt=dt, **kw)), kw
        assert refused(L.vxg_quantize_tokens(P + off, 64, dt, 4, 64, 64, P, P, None))
        assert refused(L.vxg_dequantize_rows(P, P, 4, 64, 64, dt, P + off, None))
        for sx, sw, bias, y in ((P + 2, P, None, P), (P, P + 1, None, P), (P, P, P + 2, P), (P, P, None, P + off)):
            assert refused(L.vxg_gemm_i8(P, sx, P, sw, 4, 32, 64, 0, 0.0, bias, dt, y, 32, None))
        assert refused(_write(c, dt=dt, k=P + off)) and refused(_write(c, dt=dt, v=P + off))
    assert refused(L.vxg_dequantize_rows(P, P + 2, 4, 64, 64, 2, P, None))
    for kw in (dict(table=P + 2), dict(cu=P + 1)):
        assert refused(_write(c, **kw)) and refused(_attend(c, **kw)) and refused(_read(c, **kw))
    assert refused(_write(c, start=P + 2)) and refused(_attend(c, lens=P + 2)) and refused(_read(c, start=P + 2))
    for kw in (dict(k_scales=P + 2), dict(v_scales=P + 1)):
        assert refused(_write(_cache(**kw))) and refused(_attend(_cache(**kw))) and refused(_read(_cache(**kw)))


def test_sizes_that_an_int_does_not_hold(monkeypatch):
    """ctypes cuts a size to 32 bits: 2^32 + 5 rows would become 5, and a window of 2^32 + 5 keys one of 5."""
    from voxrt_b200 import kernels as K

    most = (1 << 32) + 5
    wide = lambda *shape: torch.zeros((1,) * len(shape)).expand(shape)
    calls = []
    monkeypatch.setattr(KvCache.attend.__globals__["torch"]._C, "_cuda_getDevice", lambda: 0)
    for m in (K, sys.modules["voxrt_b200.cache"]):
        monkeypatch.setattr(m, "_call", lambda fn, idx, stream, used, *a: calls.append(a))
        monkeypatch.setattr(m, "_like", lambda t, shape, dt, stream: torch.empty(shape, dtype=dt))
        monkeypatch.setattr(m, "_gpu", lambda stream, *t: 0)
    monkeypatch.setattr(K, "QuantAct", lambda *a: a)
    a = _Act(1, 16, torch.ones((1, 1)), 16)
    a.n, a.scales = most, wide(most, 1)
    w = _Act(8, 16, None, 16)
    w.w, w.scales, w.out = w.x, torch.ones(8), 8
    for run in (lambda: K.quantize(wide(most, 16), 16), lambda: K.rms_quant(wide(most, 16), torch.ones(16)),
                lambda: K.rms_norm(wide(most, 16), torch.ones(16), wide(most, 16)), lambda: K.dequantize(a),
                lambda: K.gemm_i8(w, a, wide(most, 8))):
        with pytest.raises(ValueError, match="size of 4294967301"):
            run()
    c = KvCache.__new__(KvCache)
    c.k = c.v = c.ks = c.vs = torch.zeros(1)
    c.heads, c.head_dim, c.page, c.n_pages, c._ref, c._ws_bytes = 2, 64, 16, 8, None, {}
    ints = lambda *shape: torch.zeros((1,) * len(shape), dtype=torch.int32).expand(shape).contiguous()
    table, lens, cu = ints(1, 4), ints(1), ints(2)
    for run in (lambda: c.write(wide(most, 2, 64), wide(most, 2, 64), table, lens, cu), lambda: c.read(table, lens, cu, most),
                lambda: c.attend(wide(most, 2, 64), table, lens, cu)):
        with pytest.raises(ValueError, match="size of 4294967301"):
            run()
    assert not calls
    q = torch.zeros((1, 2, 64))
    for window, want in ((0, 0), (7, 7), (most, 0x7FFFFFFF)):
        c.attend(q, table, lens, cu, window=window)
        assert calls.pop()[13] == want
    for window in (-1, -most + 5):
        with pytest.raises(ValueError, match="negative"):
            c.attend(q, table, lens, cu, window=window)
