"""GPU: the int8 product with token and channel scales against exact integer sums; the f32 steps behind them bit for bit."""
import numpy as np
import pytest
import torch

from decoder_ops_ref import DTYPES, HALF, bits_equal, f32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from voxrt_b200 import kernels

    return kernels


def _case(seed, m, n, k, lo=-127):
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(lo, 128, (m, k), generator=g, dtype=torch.int8)
    w = torch.randint(lo, 128, (n, k), generator=g, dtype=torch.int8)
    sx, sw = torch.rand((m, 1), generator=g) * 0.01 + 1e-3, torch.rand(n, generator=g) * 0.01 + 1e-3
    bias = torch.randn(n, generator=g)
    # sums of up to 2^31 are exact in f64
    s = (x.double().cuda() @ w.double().cuda().t()).cpu().numpy()
    v = s.astype(np.float32) * (sx.numpy() * sw.numpy()[None]).astype(np.float32)
    return x.cuda(), sx.cuda(), w.cuda(), sw.cuda(), bias.cuda(), v.astype(np.float32)


# one token, few, the edges of every kernel's tiles, odd channel counts, K of one piece / a short tail / long
SHAPES = [(1, 1, 16), (1, 17, 48), (2, 40, 16), (7, 33, 1040), (8, 128, 128), (9, 100, 144), (16, 1000, 4096),
          (17, 24, 272), (31, 640, 2048), (33, 129, 96), (64, 256, 1024), (65, 130, 176), (127, 257, 400),
          (128, 256, 256), (129, 255, 4112), (200, 1024, 640), (256, 512, 128), (257, 300, 2064), (600, 700, 336),
          (1000, 1031, 1024), (4, 2048, 16384), (300, 264, 16384), (100, 50, 16), (300, 17, 32),
          (20, 2080, 48), (44, 4100, 1040), (513, 2049, 272)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(K, m, n, k):
    x, sx, w, sw, bias, v = _case(m * 7 + n, m, n, k)
    W, X = K.Int8Matrix(w, sw), K.QuantAct(x, sx, k)
    for dtype in DTYPES:
        y = K.gemm_i8(W, X, torch.empty((m, n), dtype=dtype, device="cuda"))
        assert torch.equal(y.cpu(), torch.from_numpy(v).to(dtype))
        y = K.gemm_i8(W, X, torch.empty((m, n), dtype=dtype, device="cuda"), bias=bias)
        assert torch.equal(y.cpu(), torch.from_numpy(v + f32(bias)[None]).to(dtype))
    y0 = torch.randn((m, n), generator=torch.Generator().manual_seed(1)).cuda()
    y = K.gemm_i8(W, X, y0.clone(), ep=K.Epilogue.AddScaled(0.5))
    assert bits_equal(f32(y), (f32(y0).astype(np.float64) + 0.5 * v.astype(np.float64)).astype(np.float32))


@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_epilogues_and_strides(K, m):
    n, k = 200, 512
    x, sx, w, sw, bias, v = _case(m, m, n, k)
    sw = sw * 0.05
    v = (v * np.float64(0.05)).astype(np.float64)
    W, X = K.Int8Matrix(w, sw), K.QuantAct(x, sx, k)
    for dtype in DTYPES:
        wide = torch.full((m, n + 3), 7.0, dtype=dtype, device="cuda")
        K.gemm_i8(W, X, wide[:, :n], bias=bias, ep=K.Epilogue.Silu)
        t = v + f32(bias)[None]
        want = t / (1 + np.exp(-t))
        # f32 steps of v, +bias, exp, 1 + e, divide: under 16 half-steps of the larger operand; then the type's rounding
        tol = 16 * 2.0 ** -24 * (np.abs(v) + np.abs(f32(bias))[None] + np.abs(want)) * (1 + np.abs(t)) + HALF[dtype] * np.abs(want)
        assert (np.abs(f32(wide[:, :n]) - want) <= tol + 1e-30).all()
        assert (f32(wide[:, n:]) == 7.0).all()  # what lies beside the output stays


def test_extreme_codes(K):
    """-128 and 127 everywhere: the largest sums K allows stay exact."""
    for m, k in ((1, 131056), (40, 131056), (300, 131056)):
        x = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
        w = torch.full((130, k), -128, dtype=torch.int8, device="cuda")
        w[1::2] = 127
        one = torch.ones(130, device="cuda")
        y = K.gemm_i8(K.Int8Matrix(w, one), K.QuantAct(x, torch.ones((m, 1), device="cuda"), k),
                      torch.empty((m, 130), device="cuda"))
        want = torch.tensor([16384.0 * k, -16256.0 * k] * 65, dtype=torch.float64).float()
        assert torch.equal(y.cpu(), want.expand(m, 130))


def test_most_tokens(K):
    """As many tokens as the entry takes, 2^31 - 256. Only a few runs of the input are written, and compared."""
    m, k = 2 ** 31 - 256, 16
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < m * 22 * 1.2:
        pytest.skip("not enough memory")
    x = torch.empty((m, k), dtype=torch.int8, device="cuda")
    sx, y = torch.empty((m, 1), device="cuda"), torch.empty((m, 1), dtype=torch.float16, device="cuda")
    runs = [slice(0, 600), slice(2 ** 30 - 300, 2 ** 30 + 300), slice(m - 600, m)]
    parts = [_case(i, 600, 1, k) for i in range(len(runs))]
    _, _, w, sw, _, _ = parts[0]
    for r, p in zip(runs, parts):
        x[r], sx[r] = p[0], p[1]
    K.gemm_i8(K.Int8Matrix(w, sw), K.QuantAct(x, sx, k), y)
    for r, p in zip(runs, parts):
        s = (p[0].double() @ w.double().t()).float() * (p[1] * sw[None])
        assert torch.equal(y[r], s.half())
    del x, sx, y
    torch.cuda.empty_cache()


def test_rows_do_not_depend_on_the_batch(K):
    x, sx, w, sw, _, v = _case(11, 700, 384, 1024)
    W = K.Int8Matrix(w, sw)
    for m in (1, 3, 12, 30, 64, 100, 333, 700):
        y = K.gemm_i8(W, K.QuantAct(x[:m].contiguous(), sx[:m].contiguous(), 1024), torch.empty((m, 384), device="cuda"))
        assert bits_equal(f32(y), v[:m])


def test_from_float_and_empty(K):
    w = torch.randn((70, 96), generator=torch.Generator().manual_seed(2)).cuda()
    for dtype in DTYPES:
        W = K.Int8Matrix.from_float(w.to(dtype))
        back = W.w.float() * W.scales[:, None]
        assert ((back - w.to(dtype).float()).abs() <= 0.5001 * W.scales[:, None]).all()
    e = K.QuantAct(torch.empty((0, 96), dtype=torch.int8, device="cuda"), torch.empty((0, 1), device="cuda"), 96)
    assert tuple(K.gemm_i8(W, e, torch.empty((0, 70), device="cuda")).shape) == (0, 70)


def test_other_stream_and_graph(K):
    for m in (3, 300):
        x, sx, w, sw, _, v = _case(m, m, 256, 512)
        W, X = K.Int8Matrix(w, sw), K.QuantAct(x, sx, 512)
        side = torch.cuda.Stream()
        y = torch.empty((m, 256), device="cuda")
        torch.cuda.synchronize()
        K.gemm_i8(W, X, y, stream=side)
        side.synchronize()
        assert bits_equal(f32(y), v)
        out = torch.zeros((m, 256), device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            K.gemm_i8(W, X, out)
        x.neg_()
        graph.replay()
        assert bits_equal(f32(out), -v)
