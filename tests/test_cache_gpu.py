"""GPU: the paged int8 cache (written, appended to, read back) bit for bit against its formulas, the attention over it
within a bound derived from its arithmetic, and a whole decoder step of all operators together."""
import numpy as np
import pytest
import torch

from decoder_ops_ref import DTYPES, Cache, attend, bits_equal, f32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def KvCache():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from voxrt_b200.cache import KvCache as C

    return C


def _int(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _table(rng, lens, page, spare=2, extra=3):
    """Scattered pages; entries behind a sequence's last page are not valid ids."""
    need = [-(-n // page) for n in lens]
    ids = rng.permutation(sum(need) + extra)
    width = max(need) + spare
    t = np.full((len(lens), width), 1 << 30, np.int64)
    at = 0
    for s, n in enumerate(need):
        t[s, :n] = ids[at:at + n]
        at += n
    return t, sum(need) + extra


def _pair(KvCache, rng, n_pages, heads, page, hd):
    ref = Cache(n_pages, heads, page, hd, rng)
    T = lambda a: torch.from_numpy(a.copy()).cuda()
    return ref, KvCache(T(ref.codes[0]), T(ref.codes[1]), T(ref.scales[0]), T(ref.scales[1]))


def _same(ref, c):
    for w, (codes, scales) in enumerate(((c.k, c.ks), (c.v, c.vs))):
        assert np.array_equal(codes.cpu().numpy(), ref.codes[w])
        assert bits_equal(f32(scales), ref.scales[w])


def _ok():
    from voxrt_b200._lib import device_status

    assert device_status() == 0


def _kv(rng, rows, heads, hd, dtype, grow=1.0, pad=0):
    out = []
    for _ in range(2):
        x = rng.standard_normal((rows, heads * hd + pad)) * grow
        out.append(torch.from_numpy(x.astype(np.float32)).to(dtype).cuda()[:, :heads * hd].unflatten(1, (heads, hd)))
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,hd,heads", [(16, 64, 3), (32, 128, 2), (64, 128, 1), (128, 64, 2), (128, 128, 8)])
def test_write_append_read(KvCache, dtype, page, hd, heads):
    """A prefill of ragged runs (one empty), then appended runs and single tokens with growing and shrinking sizes."""
    rng = np.random.default_rng(page + hd + heads)
    steps = [[page + 5, 0, 1, 3 * page], [0, 2, 1, 1], [1, 1, 1, 1], [page - 1, 3, 2 * page + 1, 1], [1, 1, 1, 1]]
    total = np.sum(steps, axis=0)
    table, n_pages = _table(rng, total, page)
    ref, c = _pair(KvCache, rng, n_pages, heads, page, hd)
    start = np.zeros(4, np.int64)
    for i, new in enumerate(steps):
        cu = np.concatenate([[0], np.cumsum(new)])
        k, v = _kv(rng, int(cu[-1]) + 2, heads, hd, dtype, grow=[1.0, 0.01, 3.0, 0.5, 10.0][i], pad=0 if i % 2 else 3)
        c.write(k, v, _int(table), _int(start), _int(cu))
        ref.write([f32(k), f32(v)], table, start, cu)
        _same(ref, c)
        start = start + new
    rs, rn = np.array([3, 0, page - 1, page + 7]), np.minimum(total, [page, 2, 3, 2 * page - 8])
    rn = np.minimum(rn, total - rs)
    cu = np.concatenate([[0], np.cumsum(rn)])
    for out in DTYPES:
        got = c.read(_int(table), _int(rs), _int(cu), int(cu[-1]), out)
        for w in range(2):
            want = np.concatenate([ref.rows(w, table, s, rs[s], rs[s] + rn[s]) for s in range(4)])
            assert torch.equal(got[w].cpu(), torch.from_numpy(want).to(out))
    _ok()


def test_write_twice_is_the_same(KvCache):
    rng = np.random.default_rng(1)
    table, n_pages = _table(rng, [90, 40], 32)
    ref, c = _pair(KvCache, rng, n_pages, 2, 32, 64)
    start, cu = [70, 33], [0, 20, 27]
    k, v = _kv(rng, 27, 2, 64, torch.float32, grow=5.0)
    for _ in range(2):
        c.write(k, v, _int(table), _int(start), _int(cu))
        ref.write([f32(k), f32(v)], table, start, cu)
        _same(ref, c)


def test_zero_tiny_and_non_finite_values(KvCache):
    """All-zero pages have scale 0 and grow from it; the smallest values keep a finite reciprocal; NaN -> 0, inf -> +-127."""
    rng = np.random.default_rng(2)
    table, n_pages = _table(rng, [16, 16, 16, 16], 16)
    ref, c = _pair(KvCache, rng, n_pages, 1, 16, 64)
    k, v = _kv(rng, 32, 1, 64, torch.float32)
    k[0:8] = 0
    k[8:16] = 1e-44
    v[16:24] *= 1e-38
    k[16, 0, 3], k[17, 0, 5], k[18, 0, 7] = float("nan"), float("inf"), float("-inf")
    k[24:32] = float("nan")
    v[24:32] = float("inf")
    cu = [0, 8, 16, 24, 32]
    for start in ([0, 0, 0, 0], [8, 8, 8, 8]):
        c.write(k, v, _int(table), _int(start), _int(cu))
        ref.write([f32(k), f32(v)], table, start, cu)
        _same(ref, c)
        k = k.roll(8, 0).contiguous()  # each sequence goes on with another one's values
    assert float(c.ks[int(table[0][0]), 0]) >= 0.0
    _ok()


def test_bad_indices_are_skipped_and_reported(KvCache):
    from voxrt_b200._lib import device_status

    rng = np.random.default_rng(3)
    lens = [40, 40, 40]
    table, n_pages = _table(rng, lens, 16)
    good, c = _pair(KvCache, rng, n_pages, 2, 16, 64)
    k, v = _kv(rng, 120, 2, 64, torch.float16)
    cu, start = [0, 40, 80, 120], [0, 0, 0]
    bad = table.copy()
    bad[1, 1], bad[2, 0] = n_pages, -5
    c.write(k, v, _int(bad), _int(start), _int(cu))
    assert device_status() == 0x302 and device_status() == 0
    want = Cache(n_pages, 2, 16, 64)
    want.codes, want.scales = [a.copy() for a in good.codes], [a.copy() for a in good.scales]
    # sequence 0 whole, 1 without its second page, 2 without its first
    for s, lo, hi in ((0, 0, 40), (1, 0, 16), (1, 32, 40), (2, 16, 40)):
        want.write([f32(k[40 * s + lo:40 * s + hi]), f32(v[40 * s + lo:40 * s + hi])], [table[s]], [lo], [0, hi - lo])
    _same(want, c)
    # a start behind the table, a negative one, offsets that run past the rows or backwards
    for st, of in (([0, 16 * table.shape[1] - 39, -1], cu), ([0, 0, 0], [0, 40, 80, 121]), ([0, 0, 0], [0, 40, 20, 20])):
        c2 = KvCache(c.k.clone(), c.v.clone(), c.ks.clone(), c.vs.clone())
        c2.write(k, v, _int(table), _int(st), _int(of))
        assert device_status() == 0x302
    q = torch.randn((3, 4, 64), device="cuda", dtype=torch.float16)
    out = c.attend(q, _int(bad), _int(lens), _int([0, 1, 2, 3]))
    assert device_status() == 0x302
    w = Cache(n_pages, 2, 16, 64)
    w.codes, w.scales = [c.k.cpu().numpy(), c.v.cpu().numpy()], [f32(c.ks), f32(c.vs)]
    o, b = attend(w, f32(q)[:1], table, lens[:1], [0, 1], 0.125, True, 0, torch.float16)
    assert (np.abs(f32(out)[:1] - o) <= b).all()  # the sound sequence is not touched by the others' faults
    out = torch.full_like(q, 3.0)
    c.attend(q, _int(table), _int([40, 16 * table.shape[1] + 1, -1]), _int([0, 1, 2, 3]), out=out)
    assert device_status() == 0x302 and (out[1:] == 3.0).all()


def test_read_leaves_out_what_is_out_of_range(KvCache):
    """A sequence whose rows run past the output, or whose positions run past the table, is left out as a whole, as in a
    write, and reported; the others are read."""
    from voxrt_b200._lib import check, device_status, lib

    rng = np.random.default_rng(4)
    table, n_pages = _table(rng, [40, 40], 16)
    ref, c = _pair(KvCache, rng, n_pages, 2, 16, 64)
    most = 16 * table.shape[1]
    for start, cu, sound in (([0, 0], [0, 20, 41], [0]), ([0, most - 10], [0, 20, 40], [0]), ([-1, 3], [0, 20, 40], [1]),
                             ([5, 7], [0, 20, 40], [0, 1])):
        out = torch.full((2, 40, 2, 64), 5.0, device="cuda")
        t, a, o = _int(table), _int(start), _int(cu)
        check(lib().vxg_cache_read(c._ref, t.data_ptr(), 2, table.shape[1], a.data_ptr(), o.data_ptr(), 40, 2,
                                   out[0].data_ptr(), out[1].data_ptr(), torch.cuda.current_stream().cuda_stream))
        assert device_status() == (0 if len(sound) == 2 else 0x302)
        for w in range(2):
            for s in range(2):
                got = f32(out[w][cu[s]:min(cu[s + 1], 40)])
                want = ref.rows(w, table, s, start[s], start[s] + 20) if s in sound else np.full_like(got, 5.0)
                assert bits_equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("hd,heads,new", [(64, 2, 3), (128, 2, 7), (64, 2, 30), (128, 2, 30), (64, 2, 150), (128, 2, 150)])
def test_pages_out_of_range_are_masked(KvCache, hd, heads, new, page, dtype):
    """The keys of a page whose id is out of range take no part, in tiles of every size: first, middle and last pages, a
    sequence that has no other, and one that is sound."""
    from voxrt_b200._lib import device_status

    rng = np.random.default_rng(hd + new + page)
    lens = [5 * page + 7, 2 * page, page + 1, 700]
    table, n_pages = _table(rng, lens, page)
    ref, c = _pair(KvCache, rng, n_pages, 1, page, hd)
    ref.scales[0] *= np.float32(0.02)
    c.ks.copy_(torch.from_numpy(ref.scales[0]))
    hidden = [(0, 0), (0, 2), (0, 5), (1, 0), (1, 1), (2, 1)]
    bad = table.copy()
    for i, (s, pg) in enumerate(hidden):
        bad[s, pg] = [-1, n_pages, 1 << 30][i % 3]
    count = [min(new, 5 * page), min(new, page), 1, new]
    cu = np.concatenate([[0], np.cumsum(count)])
    q = torch.from_numpy(rng.standard_normal((int(cu[-1]), heads, hd)).astype(np.float32) * 1.5).to(dtype).cuda()
    for window in (0, page + 3):
        got = f32(c.attend(q, _int(bad), _int(lens), _int(cu), scale=0.11, window=window)).astype(np.float64)
        want, bound = attend(ref, f32(q), table, lens, cu, float(np.float32(0.11)), True, window, dtype, hidden)
        assert device_status() == 0x302
        assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,heads,new", [(64, 2, 3), (128, 2, 7), (64, 2, 30), (128, 2, 30), (64, 2, 150), (128, 2, 150)])
def test_pages_out_of_range_under_other_extremes(KvCache, hd, heads, new, dtype):
    """A negative scale beside such pages, scale 0, and NaN and infinite queries that see no other page, which give 0 like
    any query that sees no key."""
    from voxrt_b200._lib import device_status

    rng = np.random.default_rng(hd + new)
    lens = [200, 200]
    table, n_pages = _table(rng, lens, 32)
    ref, c = _pair(KvCache, rng, n_pages, 1, 32, hd)
    ref.scales[0] *= np.float32(0.02)
    c.ks.copy_(torch.from_numpy(ref.scales[0]))
    bad = table.copy()
    bad[0, [1, 4, 6]] = n_pages
    bad[1, :7] = -1
    hidden = [(0, 1), (0, 4), (0, 6)] + [(1, i) for i in range(7)]
    cu = [0, new, 2 * new]
    q = torch.from_numpy(rng.standard_normal((2 * new, heads, hd)).astype(np.float32) * 1.5).to(dtype).cuda()
    finite = f32(q)
    q[new:, 0, 5], q[new:, 1, 7] = float("nan"), float("inf")
    for scale in (-0.2, 0.0, 0.2):
        got = f32(c.attend(q, _int(bad), _int(lens), _int(cu), scale=scale)).astype(np.float64)
        want, bound = attend(ref, finite, table, lens, cu, float(np.float32(scale)), True, 0, dtype, hidden)
        assert device_status() == 0x302
        assert (np.abs(got - want) <= bound).all() and (got[new:] == 0).all()


CASES = [  # (page, hd, kv heads, query heads, lengths, new tokens, causal, window)
    (16, 64, 1, 1, [1], [1], True, 0),
    (16, 64, 2, 2, [1, 17, 64, 65, 200], [1, 1, 1, 1, 1], True, 0),
    (64, 128, 2, 8, [1, 63, 64, 129, 500], [1, 1, 1, 1, 1], True, 0),
    (32, 128, 1, 16, [300, 31], [1, 1], True, 0),
    (128, 128, 2, 6, [400, 0, 130], [1, 0, 1], True, 0),
    (64, 64, 3, 3, [700, 90], [2, 5], True, 0),
    (16, 128, 2, 2, [150, 16, 300], [150, 16, 7], True, 0),
    (32, 64, 1, 4, [129, 200], [129, 1], True, 0),
    (128, 64, 2, 4, [260, 70], [70, 70], True, 0),
    (64, 128, 1, 5, [100, 37], [37, 37], False, 0),
    (16, 64, 2, 2, [333, 50], [1, 1], True, 40),
    (16, 128, 1, 2, [200, 129], [100, 129], True, 33),
    (64, 64, 1, 3, [90, 20], [90, 3], False, 25),
    (32, 64, 2, 2, [5, 0, 64], [9, 4, 70], True, 0),      # more queries than cached tokens: rows without a key
    (128, 128, 1, 32, [1000], [1], True, 0),
    (16, 128, 2, 8, [300, 700, 90], [300, 130, 1], True, 0),   # tiles of many rows, with a single-token sequence among them
    (64, 64, 1, 4, [1000], [200], True, 130),
    (32, 128, 1, 2, [250, 0], [250, 3], False, 0),
    (128, 128, 2, 4, [50, 200], [200, 200], True, 0),          # most rows of the first sequence see no key
    (128, 64, 3, 3, [513, 129], [257, 128], True, 0),
    (64, 128, 1, 7, [700], [101], False, 300),
    (64, 128, 8, 8, [2500], [1], True, 0),                # one sequence over many shares
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,hd,kv,heads,lens,new,causal,window", CASES)
def test_attention(KvCache, page, hd, kv, heads, lens, new, causal, window, dtype):
    rng = np.random.default_rng(page + hd + heads + sum(lens))
    table, n_pages = _table(rng, lens, page)
    ref, c = _pair(KvCache, rng, n_pages, kv, page, hd)
    for w in range(2):
        ref.scales[w] *= np.float32(0.02) * np.exp(rng.standard_normal(ref.scales[w].shape)).astype(np.float32)
    c.ks.copy_(torch.from_numpy(ref.scales[0]))
    c.vs.copy_(torch.from_numpy(ref.scales[1]))
    cu = np.concatenate([[0], np.cumsum(new)])
    rows = int(cu[-1])
    # a page that no query sees may hold any scale
    unused = sorted(set(range(n_pages)) - set(table[table < n_pages].tolist()))
    c.ks[unused], c.vs[unused] = float("nan"), float("inf")
    wide = torch.from_numpy(rng.standard_normal((rows + 2, heads * hd + 8)).astype(np.float32) * 1.5).to(dtype).cuda()
    q = wide[:, :heads * hd].unflatten(1, (heads, hd))
    out = torch.full((rows + 2, heads, hd), 9.0, dtype=dtype, device="cuda")
    c.attend(q, _int(table), _int(lens), _int(cu), scale=0.11, causal=causal, window=window, out=out)
    want, bound = attend(ref, f32(q), table, lens, cu, float(np.float32(0.11)), causal, window, dtype)
    _ok()
    got = f32(out).astype(np.float64)
    assert (got[rows:] == 9.0).all()  # rows behind the last sequence stay
    bad = np.abs(got[:rows] - want[:rows]) > bound[:rows]
    assert not bad.any(), (bad.sum(), np.abs(got[:rows] - want[:rows]).max())


def test_masked_places_do_not_leak(KvCache):
    """Scales of pages that lie wholly outside a window, and codes behind a sequence's end, take no part."""
    rng = np.random.default_rng(8)
    lens, page = [200, 75], 16
    table, n_pages = _table(rng, lens, page)
    ref, c = _pair(KvCache, rng, n_pages, 2, page, 64)
    cu = [0, 1, 2]
    q = torch.randn((2, 2, 64), device="cuda")
    want, bound = attend(ref, f32(q), table, lens, cu, 0.125, True, 20, torch.float32)
    for s in range(2):
        for pg in range((lens[s] - 20) // page):
            c.ks[int(table[s, pg])], c.vs[int(table[s, pg])] = float("nan"), float("inf")
    got = f32(c.attend(q, _int(table), _int(lens), _int(cu), window=20))
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_queries(KvCache, dtype):
    """Very large, very small and zero queries keep their precision; a NaN or an infinity shows in its own row only."""
    rng = np.random.default_rng(9)
    table, n_pages = _table(rng, [100], 32)
    ref, c = _pair(KvCache, rng, n_pages, 1, 32, 128)
    big, small = (3e4, 1e-6) if dtype == torch.float16 else (1e30, 1e-30)
    q = torch.from_numpy(rng.standard_normal((1, 6, 128)).astype(np.float32)).cuda()
    q[0, 1] *= big / 4
    q[0, 2] *= small
    q[0, 3] = 0
    q = q.to(dtype)
    q[0, 4, 7], q[0, 5, 9] = float("nan"), float("inf")
    cu = [0, 1]
    got = f32(c.attend(q, _int(table), _int([100]), _int(cu), scale=1.0))
    # the first four heads one at a time, each with a scale that brings its scores to ordinary size
    assert np.isnan(got[0, 4:]).all() and np.isfinite(got[0, [0, 2, 3]]).all()
    for h, scale in ((0, 0.01), (1, 0.01 / big), (2, 0.01 / small), (3, 1.0)):
        got = f32(c.attend(q[:, h:h + 1].contiguous(), _int(table), _int([100]), _int(cu), scale=scale))
        want, bound = attend(ref, f32(q)[:, h:h + 1], table, [100], cu, float(np.float32(scale)), True, 0, dtype)
        assert (np.abs(got - want) <= bound).all(), h


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("length", ["one block", 300])  # whole tiles, tiles of several shares
@pytest.mark.parametrize("hd,heads,new", [(64, 2, 3), (128, 2, 7), (64, 2, 20), (128, 2, 20), (64, 2, 80), (128, 2, 80)])
def test_smallest_value_scales(KvCache, hd, heads, new, length, dtype):
    """Value scales from the smallest that a write leaves, 2^-126, on, in tiles of every size. Everything is compared times
    2^118, the oracle with scales that are larger by as much (exact). On top of its bound: results below 2^-126 are
    subnormal, off by half a step of 2^-149 (bf16: 2^-133), and so are up to 64 joined parts in f32."""
    length = (60 if new < 60 else 100) if length == "one block" else length
    rng = np.random.default_rng(hd + new)
    table, n_pages = _table(rng, [length], 32)
    ref, c = _pair(KvCache, rng, n_pages, 1, 32, hd)
    ref.scales[0] *= np.float32(0.02)
    ref.scales[1] = (2.0 ** -126 * rng.uniform(1, 4, ref.scales[1].shape)).astype(np.float32)
    ref.scales[1][table[0, 0]] = np.float32(2.0 ** -126)
    c.ks.copy_(torch.from_numpy(ref.scales[0]))
    c.vs.copy_(torch.from_numpy(ref.scales[1]))
    q = torch.from_numpy(rng.standard_normal((new, heads, hd)).astype(np.float32)).to(dtype).cuda()
    cu = [0, new]
    got = f32(c.attend(q, _int(table), _int([length]), _int(cu), scale=0.11)).astype(np.float64) * 2.0 ** 118
    ref.scales[1] = ref.scales[1] * np.float32(2.0 ** 118)
    want, bound = attend(ref, f32(q), table, [length], cu, float(np.float32(0.11)), True, 0, dtype)
    bound += 2.0 ** 118 * (64 * 2.0 ** -150 + (2.0 ** -134 if dtype == torch.bfloat16 else 2.0 ** -150))
    _ok()
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("scale", [-0.3, 0.0])
@pytest.mark.parametrize("hd,heads,new,dtype", [
    (64, 2, 3, torch.float32), (128, 4, 2, torch.bfloat16), (128, 2, 7, torch.float16), (64, 2, 20, torch.bfloat16),
    (64, 2, 80, torch.float32), (128, 2, 80, torch.float32), (128, 2, 20, torch.float16), (64, 4, 80, torch.float16),
    (128, 4, 80, torch.bfloat16)])
def test_scales_that_are_not_positive(KvCache, hd, heads, new, dtype, scale):
    """Peaked scores under a negative scale, whose softmax follows the smallest products, and scale 0, which weighs every
    key alike, in tiles of every size."""
    rng = np.random.default_rng(hd + new + heads)
    lens, count = [300, 150], [new, max(1, new - 3)]
    table, n_pages = _table(rng, lens, 32)
    ref, c = _pair(KvCache, rng, n_pages, 1, 32, hd)
    ref.scales[0] *= np.float32(0.02)
    c.ks.copy_(torch.from_numpy(ref.scales[0]))
    cu = np.concatenate([[0], np.cumsum(count)])
    q = torch.from_numpy(rng.standard_normal((int(cu[-1]), heads, hd)).astype(np.float32) * 1.5).to(dtype).cuda()
    got = f32(c.attend(q, _int(table), _int(lens), _int(cu), scale=scale)).astype(np.float64)
    want, bound = attend(ref, f32(q), table, lens, cu, float(np.float32(scale)), True, 0, dtype)
    _ok()
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length", [257, 300, 448, 1000])  # the last step of 64 keys: one key, a few, none, most
@pytest.mark.parametrize("hd,heads,new", [(64, 2, 3), (128, 2, 7), (64, 2, 30), (128, 2, 30), (64, 2, 150), (128, 2, 150)])
def test_scores_that_rise_all_along(KvCache, hd, heads, new, length, dtype):
    """Every 64 keys outweigh all before them by about e^7.6, so that the softmax's reference moves in every step, in
    tiles of every size."""
    rng = np.random.default_rng(hd + new + length)
    table, n_pages = _table(rng, [length], 16)
    ref, c = _pair(KvCache, rng, n_pages, 1, 16, hd)
    sign = np.where(rng.random(hd) < 0.5, -1, 1)
    for pg in range(-(-length // 16)):  # scores: about 1.9 a page on
        ref.codes[0][table[0, pg], 0] = sign[None] * rng.integers(112, 128, (16, 1))
        ref.scales[0][table[0, pg]] = np.float32((pg + 1) * 2.0 / 127 / hd)
    c.k.copy_(torch.from_numpy(ref.codes[0]))
    c.ks.copy_(torch.from_numpy(ref.scales[0]))
    q = torch.from_numpy(np.tile(sign, (new, heads, 1)).astype(np.float32)).to(dtype).cuda()
    cu = [0, new]
    got = f32(c.attend(q, _int(table), _int([length]), _int(cu), scale=1.0)).astype(np.float64)
    want, bound = attend(ref, f32(q), table, [length], cu, 1.0, True, 0, dtype)
    _ok()
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("dtype,hd,heads,new", [(torch.float32, 64, 2, 3), (torch.bfloat16, 128, 2, 7),
                                               (torch.float32, 128, 2, 30), (torch.float16, 64, 2, 30)])
def test_small_tiles_take_key_scales_of_either_sign(KvCache, dtype, hd, heads, new):
    """A write leaves no negative scale, but codes and scales may come from elsewhere; only an id out of range masks."""
    rng = np.random.default_rng(hd + new)
    table, n_pages = _table(rng, [200], 16)
    ref, c = _pair(KvCache, rng, n_pages, 1, 16, hd)
    ref.scales[0] *= (0.02 * np.where(rng.random(ref.scales[0].shape) < 0.5, -1, 1)).astype(np.float32)
    c.ks.copy_(torch.from_numpy(ref.scales[0]))
    q = torch.from_numpy(rng.standard_normal((new, heads, hd)).astype(np.float32)).to(dtype).cuda()
    got = f32(c.attend(q, _int(table), _int([200]), _int([0, new]), scale=0.11)).astype(np.float64)
    oracle = Cache(n_pages, 1, 16, hd)  # the same keys as codes of the other sign, for the bound's sake
    oracle.codes, oracle.scales = [a.copy() for a in ref.codes], [a.copy() for a in ref.scales]
    flip = (oracle.scales[0] < 0)[:, :, None, None]
    oracle.codes[0] = np.where(flip, -oracle.codes[0], oracle.codes[0])
    oracle.scales[0] = np.abs(oracle.scales[0])
    want, bound = attend(oracle, f32(q), table, [200], [0, new], float(np.float32(0.11)), True, 0, dtype)
    _ok()
    assert (np.abs(got - want) <= bound).all()


def test_shared_pages_other_stream_and_graph(KvCache):
    """Two sequences over the same prefix pages; a captured call replayed with other lengths; a side stream."""
    rng = np.random.default_rng(10)
    ref, c = _pair(KvCache, rng, 8, 2, 32, 128)
    table = np.array([[0, 1, 2, 3], [0, 1, 4, 5]])
    lens, cu = [100, 90], [0, 1, 2]
    q = torch.randn((2, 4, 128), device="cuda", dtype=torch.bfloat16)
    tt, ll, cc = _int(table), _int(lens), _int(cu)
    check = lambda got, L: (lambda o, b: (np.abs(f32(got) - o) <= b).all())(
        *attend(ref, f32(q), table, L, cu, 128 ** -0.5, True, 0, torch.bfloat16))
    assert check(c.attend(q, tt, ll, cc), lens)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    out = c.attend(q, tt, ll, cc, stream=side)
    side.synchronize()
    assert check(out, lens)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:  # two graphs, each with a workspace of its own
        with torch.cuda.graph(g):
            outs.append(c.attend(q, tt, ll, cc))
    for new in ([1, 128], [65, 2]):
        ll.copy_(_int(new))
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert check(outs[0], new) and check(outs[1], new)
    _ok()


def test_long_cache(KvCache):
    """60,000 cached tokens, one query: the keys are shared out over the whole GPU and joined."""
    L, page, hd = 60000, 128, 128
    g = torch.Generator(device="cuda").manual_seed(4)
    n = -(-L // page)
    codes = [torch.randint(-127, 128, (n, 2, page, hd), generator=g, device="cuda", dtype=torch.int8) for _ in range(2)]
    scales = [torch.rand((n, 2), generator=g, device="cuda") * 0.02 + 0.005 for _ in range(2)]
    c = KvCache(*codes, *scales)
    q = torch.randn((1, 6, hd), generator=g, device="cuda")
    got = c.attend(q, torch.arange(n, device="cuda", dtype=torch.int32)[None], _int([L]), _int([0, 1])).double()
    k, v = ((a.double() * s.double()[:, :, None, None]).transpose(0, 1).reshape(2, -1, hd)[:, :L]
            for a, s in zip(codes, scales))
    for h in range(6):
        e = (k[h // 3] @ q[0, h].double()) / hd ** 0.5
        p = torch.softmax(e, 0)
        off = (hd + 8) * 2.0 ** -23 * float((k[h // 3].abs() @ q[0, h].double().abs()).max()) / hd ** 0.5
        off += 2.0 ** -21 * float(e.abs().max())
        bound = (p @ v[h // 3].abs()) * (2.0 ** -22 + 2 * off + 2.0 ** -20 + (L / 8 + 32) * 2.0 ** -23)
        assert ((got[0, h] - p @ v[h // 3]).abs() <= bound).all()


def test_offsets_past_32_bits(KvCache):
    """A pool of more than 4 GiB of codes: pages at its far end are written, read and attended to."""
    heads, page, hd = 8, 128, 128
    n = (1 << 32) // (heads * page * hd) + 8
    ref, _ = _pair(KvCache, np.random.default_rng(0), 2, heads, page, hd)
    codes = [torch.empty((n, heads, page, hd), dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros((n, heads), device="cuda") for _ in range(2)]
    c = KvCache(*codes, *scales)
    rng = np.random.default_rng(6)
    k, v = _kv(rng, 200, heads, hd, torch.float16)
    far = np.array([[n - 1, n - 3]])
    c.write(k, v, _int(far), _int([0]), _int([0, 200]))
    ref.write([f32(k), f32(v)], [[1, 0]], [0], [0, 200])
    got = c.read(_int(far), _int([0]), _int([0, 200]), 200)
    for w in range(2):
        assert bits_equal(f32(got[w]), ref.rows(w, [[1, 0]], 0, 0, 200))
    q = torch.randn((1, heads, hd), device="cuda")
    want, bound = attend(ref, f32(q), [[1, 0]], [200], [0, 1], hd ** -0.5, True, 0, torch.float32)
    assert (np.abs(f32(c.attend(q, _int(far), _int([200]), _int([0, 1]))) - want) <= bound).all()
    _ok()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,heads,new", [(64, 2, 3), (128, 2, 7), (64, 2, 20), (128, 2, 100)])
def test_longest_sequence(KvCache, hd, heads, new, dtype):
    """A sequence at the longest length that a table may hold, 2^31 - 256: its last pages are written, read and, through a
    window, attended to by tiles of every size. The entries in front of those pages are no valid ids."""
    page, window, last = 128, 500, 8
    width = 0x7FFFFF00 // page
    L, near = width * page, last * page  # the same places of the same pages in a short sequence
    rng = np.random.default_rng(hd + new)
    ref, c = _pair(KvCache, rng, last, 1, page, hd)
    for w, s in ((0, c.ks), (1, c.vs)):
        ref.scales[w] *= np.float32(0.02)
        s.copy_(torch.from_numpy(ref.scales[w]))
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    table[0, -last:] = torch.arange(last, device="cuda", dtype=torch.int32)
    short, cu = np.arange(last)[None], [0, new]
    k, v = _kv(rng, new, 1, hd, dtype)
    c.write(k, v, table, _int([L - new]), _int(cu))
    ref.write([f32(k), f32(v)], short, [near - new], cu)
    _same(ref, c)
    got = c.read(table, _int([L - 300]), _int([0, 300]), 300)
    for w in range(2):
        assert bits_equal(f32(got[w]), ref.rows(w, short, 0, near - 300, near))
    q = torch.from_numpy(rng.standard_normal((new, heads, hd)).astype(np.float32) * 1.5).to(dtype).cuda()
    got = f32(c.attend(q, table, _int([L]), _int(cu), scale=0.11, window=window)).astype(np.float64)
    want, bound = attend(ref, f32(q), short, [near], cu, float(np.float32(0.11)), True, window, dtype)
    _ok()
    assert (np.abs(got - want) <= bound).all()


def test_a_decoder_step_of_all_operators(KvCache):
    """norm -> q|k|v product -> cache -> attention -> output product onto the residual -> norm -> feed-forward: a prefill
    of two ragged sequences and two captured single-token steps, each operator against its formula on the library's own
    inputs, so that no rounding piles up."""
    from decoder_ops_ref import quant, rms
    from voxrt_b200 import kernels as K

    d, heads, kv, hd, ff, page = 256, 4, 2, 64, 512, 16
    rng = np.random.default_rng(12)
    W = lambda o, i: K.Int8Matrix.from_float(torch.from_numpy(rng.standard_normal((o, i)).astype(np.float32)).cuda() / i ** 0.5)
    wqkv, wo, w1, w2 = W((heads + 2 * kv) * hd, d), W(d, heads * hd), W(ff, d), W(d, ff)
    g1, g2 = (torch.from_numpy((1 + 0.1 * rng.standard_normal(d)).astype(np.float32)).cuda() for _ in range(2))
    table, n_pages = _table(rng, [40, 25], page)
    ref, c = _pair(KvCache, rng, n_pages, kv, page, hd)
    tt = _int(table)

    def step(x, start, lens, cu):
        a = K.rms_quant(x, g1)
        qkv = K.gemm_i8(wqkv, a, torch.empty((x.shape[0], wqkv.out), dtype=x.dtype, device="cuda"))
        q, k, v = (t.unflatten(1, (-1, hd)) for t in qkv.split([heads * hd, kv * hd, kv * hd], 1))
        c.write(k, v, tt, start, cu)
        o = c.attend(q, tt, lens, cu)
        b = K.quantize(o.flatten(1), heads * hd)
        p = K.gemm_i8(wo, b, torch.empty_like(x))
        h = torch.empty_like(x)
        e = K.rms_quant(x, g2, v=p, x_res=h)
        u = K.gemm_i8(w1, e, torch.empty((x.shape[0], ff), dtype=x.dtype, device="cuda"), ep=K.Epilogue.Silu)
        f = K.quantize(u, ff)
        y = K.gemm_i8(w2, f, h.clone(), ep=K.Epilogue.AddScaled(1.0))
        return dict(a=a, qkv=qkv, q=q, k=k, v=v, o=o, b=b, p=p, h=h, e=e, u=u, f=f, y=y)

    def product(w, a):
        s = a.x.double() @ w.w.double().t()
        return s.float() * (a.scales.view(-1, 1) * w.scales[None])

    def check(x, r, start, lens, cu):
        dt = x.dtype
        for a, src in ((r["a"], rms(f32(x), f32(g1), 1e-6)[1]), (r["e"], rms(f32(x), f32(g2), 1e-6, f32(r["p"]))[1]),
                       (r["b"], f32(r["o"].flatten(1))), (r["f"], f32(r["u"]))):
            q, s = quant(src, src.shape[1])
            assert np.array_equal(a.x.cpu().numpy(), q) and bits_equal(f32(a.scales), s)
        assert torch.equal(r["qkv"], product(wqkv, r["a"]).to(dt)) and torch.equal(r["p"], product(wo, r["b"]).to(dt))
        t = product(w1, r["e"]).double()
        assert torch.allclose(r["u"].double(), t * torch.sigmoid(t), rtol=2.0 ** -8 + 1e-5, atol=1e-7)
        assert torch.equal(r["y"], (r["h"].double() + product(w2, r["f"]).double()).float().to(dt))
        ref.write([f32(r["k"]), f32(r["v"])], table, start, cu)
        _same(ref, c)
        want, bound = attend(ref, f32(r["q"]), table, lens, cu, hd ** -0.5, True, 0, dt)
        assert (np.abs(f32(r["o"]) - want) <= bound).all()

    x = torch.from_numpy(rng.standard_normal((52, d)).astype(np.float32)).to(torch.bfloat16).cuda()
    start, lens, cu = [0, 0], [33, 19], [0, 33, 52]
    check(x, step(x, _int(start), _int(lens), _int(cu)), start, lens, cu)
    x1 = torch.empty((2, d), dtype=torch.bfloat16, device="cuda")
    s1, l1, cu1 = _int([33, 19]), _int([34, 20]), _int([0, 1, 2])
    keep = [t.clone() for t in (c.k, c.v, c.ks, c.vs)]
    x1.copy_(x[:2])
    step(x1, s1, l1, cu1)  # warm up before the capture, then put the cache back
    for t, s in zip((c.k, c.v, c.ks, c.vs), keep):
        t.copy_(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = step(x1, s1, l1, cu1)
    for i in range(2):
        x1.copy_(torch.from_numpy(rng.standard_normal((2, d)).astype(np.float32) * (1 + 2 * i)))
        s1.copy_(_int([33 + i, 19 + i]))
        l1.copy_(_int([34 + i, 20 + i]))
        graph.replay()
        check(x1, r, [33 + i, 19 + i], [34 + i, 20 + i], [0, 1, 2])
    _ok()
