"""GPU: residual add + RMSNorm -> int8, the 16-bit quantiser and the reading back of codes, against 64-bit arithmetic.
Codes and scales are bit-equal: the library's sum of squares is a 64-bit one, so its order does not matter."""
import numpy as np
import pytest
import torch

from decoder_ops_ref import DTYPES, HALF, bits_equal, f32, quant, rms

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from voxrt_b200 import kernels

    return kernels


def _rows(rng, n, d, dtype, pad=0, scale=1.0):
    x = torch.from_numpy((rng.standard_normal((n, d + pad)) * scale).astype(np.float32)).to(dtype).cuda()
    return x[:, :d]


# one element; odd widths (scalar loads); one warp a row; several warps; 2, 4 and 8 vectors a thread
SHAPES = [(1, 1, 1), (3, 7, 7), (5, 64, 64), (9, 250, 250), (2, 256, 8), (4, 1000, 1000), (1, 1024, 1024),
          (33, 1024, 128), (17, 1152, 384), (3, 1029, 1029), (7, 4096, 16), (2, 4104, 4104), (3, 8192, 128),
          (2, 8200, 8200), (2, 20480, 2048), (1, 32768, 32768)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,group", SHAPES)
def test_rms_quant(K, n, d, group, dtype):
    rng = np.random.default_rng(d * 31 + n)
    x, v = _rows(rng, n, d, dtype), _rows(rng, n, d, dtype, scale=0.3)
    gamma = (1 + 0.3 * rng.standard_normal(d)).astype(np.float32)
    for vs in (None, 1.0, 0.5):
        res = torch.empty_like(x) if vs else None
        y = torch.empty_like(x)
        a = K.rms_quant(x, torch.from_numpy(gamma).cuda(), group, 1e-5, v=v if vs else None, vs=vs or 1.0, x_res=res, y=y)
        h, want = rms(f32(x), gamma, 1e-5, f32(v) if vs else None, vs or 1.0)
        q, s = quant(want, group)
        assert np.array_equal(a.x.cpu().numpy(), q) and bits_equal(f32(a.scales), s)
        assert torch.equal(y.cpu(), torch.from_numpy(want).to(dtype))
        if vs:
            assert torch.equal(res.cpu(), torch.from_numpy(h).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_in_place_and_norm_only(K, dtype):
    rng = np.random.default_rng(3)
    for n, d, pad in ((6, 1024, 3), (6, 1024, 64), (5, 96, 5)):
        x, v = _rows(rng, n, d, dtype, pad), _rows(rng, n, d, dtype, pad)
        gamma = (1 + 0.3 * rng.standard_normal(d)).astype(np.float32)
        g = torch.from_numpy(gamma).cuda()
        h, want = rms(f32(x), gamma, 1e-6, f32(v))
        q, s = quant(want, d)
        out = K.rms_norm(x, g, torch.empty((n, d), dtype=dtype, device="cuda"), v=v)
        assert torch.equal(out.cpu(), torch.from_numpy(want).to(dtype))
        a = K.rms_quant(x, g, v=v, x_res=x)  # the residual stream in place
        assert np.array_equal(a.x.cpu().numpy(), q) and bits_equal(f32(a.scales), s)
        assert torch.equal(x.cpu(), torch.from_numpy(h).to(dtype))


def test_zero_rows_and_non_finite(K):
    """A zero row gives codes 0 and scale 1; NaN and infinity stay visible in x_res and y, and give code 0."""
    x = torch.randn((4, 512), generator=torch.Generator().manual_seed(1)).cuda()
    x[0] = 0
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    v = torch.zeros_like(x)
    g = torch.ones(512, device="cuda")
    res, y = torch.empty_like(x), torch.empty_like(x)
    a = K.rms_quant(x, g, v=v, x_res=res, y=y)
    h, want = rms(f32(x), np.ones(512, np.float32), 1e-6)
    q, s = quant(want, 512)
    assert np.array_equal(a.x.cpu().numpy(), q) and bits_equal(f32(a.scales), s)
    assert not a.x[0].any() and float(a.scales[0]) == 1.0
    assert torch.isnan(y[1]).all() and torch.isnan(res[1, 3]) and torch.isinf(res[2, 5])
    e = K.rms_quant(x[:0], g)
    assert tuple(e.x.shape) == (0, 512)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,group", [(1, 16, 16), (37, 640, 128), (9, 1000, 1000), (4, 10240, 10240), (3, 20, 4 * 5)])
def test_quantize_and_back(K, n, d, group, dtype):
    rng = np.random.default_rng(n + d)
    x = _rows(rng, n, d, dtype, pad=5, scale=4.0)
    a = K.quantize(x, group)
    q, s = quant(f32(x), group)
    assert np.array_equal(a.x.cpu().numpy(), q) and bits_equal(f32(a.scales), s)
    for out in DTYPES:
        back = K.dequantize(a, out)
        want = torch.from_numpy((q.reshape(n, -1, group).astype(np.float32) * s[..., None]).reshape(n, d)).to(out)
        assert torch.equal(back.cpu(), want)
    # off by half a step of the group's scale at most, and the roundings of the reciprocal and of code x scale: each
    # within 127 x 1.5 half-steps of f32 of a scale
    err = np.abs(f32(K.dequantize(a)).astype(np.float64) - f32(x)).reshape(n, -1, group)
    assert (err <= s[..., None] * (0.5 + 127 * 3 * HALF[torch.float32])).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_non_finite_tiny_and_huge(K, dtype):
    """Per group: NaN gives code 0 and the others keep their scale; an infinity makes the group's scale infinite; values
    at either end of the type; all in one call, next to ordinary groups."""
    x = torch.randn((6, 1280), generator=torch.Generator().manual_seed(3)).to(dtype)
    x[0, ::7] = float("nan")
    x[1, 130] = float("inf")
    x[2, 256:384] *= torch.finfo(dtype).smallest_normal
    x[3, :128] = torch.finfo(dtype).max
    x[4, 128:256] = float("nan")
    x[5, 640:768] = 0
    wide = torch.empty((6, 1288), dtype=dtype, device="cuda")[:, :1280]
    wide.copy_(x)
    for group in (128, 1280, 320):
        q, s = quant(f32(x), group)
        a = K.quantize(wide, group)
        assert np.array_equal(a.x.cpu().numpy(), q) and bits_equal(f32(a.scales), s)


def test_existing_quantizer_agrees(K):
    x = torch.randn((33, 1024), generator=torch.Generator().manual_seed(7)).cuda()
    wide = torch.empty((33, 1030), device="cuda")[:, :1024]
    wide.copy_(x)
    for group in (128, 1024):
        a, b = K.quantize(x, group), K.quantize(wide, group)
        assert torch.equal(a.x, b.x) and torch.equal(a.scales, b.scales)


def test_feeds_the_ternary_product(K, oracle_lib):
    """group 128: the codes are the ternary GEMM's activations."""
    from voxrt_b200 import synth

    rng = np.random.default_rng(5)
    mod = synth.ternary_module(rng, 256, 512, 128)
    w_rows, sw = oracle_lib.unpack_matrix(mod["qweight"], mod["scales"], 256, 512, 128)
    x = _rows(rng, 19, 512, torch.bfloat16)
    gamma = (1 + 0.1 * rng.standard_normal(512)).astype(np.float32)
    a = K.rms_quant(x, torch.from_numpy(gamma).cuda(), 128)
    y = torch.empty((19, 256), device="cuda")
    K.gemm_ep(K.TernaryMatrix.from_module(mod), a, y)
    q, s = quant(rms(f32(x), gamma, 1e-6)[1], 128)
    assert bits_equal(f32(y), oracle_lib.gemm(w_rows, sw, q, s, 128))


@pytest.mark.parametrize("dtype,pad", [(torch.float32, 0), (torch.float32, 8), (torch.float16, 0)])
def test_quantize_empty_batch_and_side_stream(K, dtype, pad):
    """An empty batch gives empty codes; on a side stream, neither the input nor the outputs are handed out again while that
    stream still has the call in front of it."""
    wide = lambda n: torch.ones((n, 256 + pad), dtype=dtype, device="cuda")[:, :256]
    e = K.quantize(wide(0), 128)
    assert tuple(e.x.shape) == (0, 256) and tuple(e.scales.shape) == (0, 2)
    side = torch.cuda.Stream()
    x = wide(1 << 12)
    want = K.quantize(x, 128)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
    a = K.quantize(x, 128, stream=side)
    old = x.data_ptr()
    del x
    again = wide(1 << 12)
    assert again.data_ptr() != old  # still read by the side stream
    side.synchronize()
    assert torch.equal(a.x, want.x) and torch.equal(a.scales, want.scales)
    codes = a.x.data_ptr()
    del a
    assert torch.empty((1 << 12, 256), dtype=torch.int8, device="cuda").data_ptr() != codes  # the side stream's memory


@pytest.mark.parametrize("d", [1, 8])  # element by element, and with the next row's look-ahead
def test_most_rows(K, d):
    """2^31 - 1 rows: the row index plus a step of the grid passes 31 bits. Only a few runs of the input are written, and
    compared; the rest is whatever the memory holds."""
    n = 2 ** 31 - 1
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < n * (3 * d + 4) * 1.2:
        pytest.skip("not enough memory")
    x = torch.empty((n, d), dtype=torch.float16, device="cuda")
    runs = [slice(0, 1000), slice(2 ** 30 - 500, 2 ** 30 + 500), slice(n - 20000, n)]
    g = torch.Generator(device="cuda").manual_seed(d)
    for r in runs:
        x[r] = torch.randn((r.stop - r.start, d), generator=g, device="cuda").half()
    a = K.quantize(x, d)
    for r in runs:
        q, s = quant(f32(x[r]), d)
        assert np.array_equal(a.x[r].cpu().numpy(), q) and bits_equal(f32(a.scales[r]), s)
    del x, a
    torch.cuda.empty_cache()


def test_other_stream_and_graph(K):
    g = torch.rand(1024, device="cuda") + 0.5
    x = torch.randn((64, 1024), device="cuda", dtype=torch.float16)
    want = K.rms_quant(x, g)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    a = K.rms_quant(x, g, stream=side)
    side.synchronize()
    assert torch.equal(a.x, want.x) and torch.equal(a.scales, want.scales)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b = K.rms_quant(x, g)
    x.mul_(-1)
    graph.replay()
    assert torch.equal(b.x, -want.x) and torch.equal(b.scales, want.scales)
