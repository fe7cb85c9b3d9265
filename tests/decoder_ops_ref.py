"""Plain 64-bit / exact restatements of the int8 decoder operators, for their tests."""
import numpy as np
import torch

F = np.float32
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a step, relative
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def f32(t):
    return t.detach().float().cpu().numpy()


def bits_equal(a, b):
    a, b = np.asarray(a, F), np.asarray(b, F)
    return a.shape == b.shape and np.array_equal(a.view(np.uint32), b.view(np.uint32))


def quant(y, group):
    """(codes, scales) of f32 rows: the library's quantiser (a NaN is skipped by the maximum and gets code 0)."""
    n, d = y.shape
    p = y.reshape(n, d // group, group)
    with np.errstate(all="ignore"):
        top = np.nanmax(np.where(np.isnan(p), F(0), np.abs(p)), axis=2)
        s = np.where(top == 0, F(1), top / F(127)).astype(F)
        t = p * (F(1) / s)[..., None]
        q = np.clip(np.rint(t), -127, 127)
    return np.where(np.isnan(q), 0, q).astype(np.int8).reshape(n, d), s


def rms(x, gamma, eps, v=None, vs=1.0):
    """(h, y) in f32: the residual sum and the normalised row, sums and root in 64 bits."""
    h = x if v is None else (x.astype(np.float64) + np.float64(F(vs)) * v.astype(np.float64)).astype(F)
    with np.errstate(all="ignore"):
        ms = np.square(h.astype(np.float64)).sum(1, keepdims=True) / h.shape[1]
        r = (1.0 / np.sqrt(ms + np.float64(F(eps)))).astype(F)
        return h, ((h * r).astype(F) * gamma).astype(F)


class Cache:
    """The paged cache on the host, written token run by token run."""

    def __init__(self, n_pages, heads, page, hd, rng=None):
        self.page, self.heads, self.hd = page, heads, hd
        self.codes = [np.zeros((n_pages, heads, page, hd), np.int8) for _ in range(2)]
        self.scales = [np.zeros((n_pages, heads), F) for _ in range(2)]
        if rng is not None:  # what an earlier owner of the pages left
            for c, s in zip(self.codes, self.scales):
                c[:] = rng.integers(-127, 128, c.shape)
                s[:] = rng.uniform(0.5, 2, s.shape)

    def write(self, kv, table, start, cu):
        """kv: two f32 arrays [rows, heads, hd]."""
        P = self.page
        with np.errstate(all="ignore"):
            for s in range(len(start)):
                a, n = int(start[s]), int(cu[s + 1] - cu[s])
                for pg in range(a // P, (a + n + P - 1) // P if n else 0):
                    lo, hi = max(a, pg * P), min(a + n, (pg + 1) * P)
                    held, pid = max(0, a - pg * P), table[s][pg]
                    for w in range(2):
                        x = kv[w][cu[s] + lo - a:cu[s] + hi - a]  # [tokens, heads, hd]
                        top = np.max(np.where(np.isfinite(x), np.abs(x), F(0)), axis=(0, 2))
                        new = np.where(top > 0, np.maximum(top / F(127), F(2.0 ** -126)), F(0)).astype(F)
                        old = self.scales[w][pid].copy() if held else np.zeros(self.heads, F)
                        sc = np.maximum(old, new)
                        for h in range(self.heads):
                            c = self.codes[w][pid, h]
                            if held and sc[h] != old[h]:
                                c[:held] = np.clip(np.rint(c[:held].astype(F) * (old[h] / sc[h])), -127, 127)
                            inv = F(1) / sc[h] if sc[h] > 0 else F(0)
                            q = np.clip(np.rint(x[:, h] * inv), -127, 127)
                            c[lo - pg * P:hi - pg * P] = np.where(np.isnan(q), 0, q)
                        self.scales[w][pid] = sc

    def rows(self, w, table, s, lo, hi):
        """f32 values of positions lo .. hi of sequence s: [tokens, heads, hd]."""
        out = np.zeros((hi - lo, self.heads, self.hd), F)
        for i, pos in enumerate(range(lo, hi)):
            pid = table[s][pos // self.page]
            out[i] = self.codes[w][pid, :, pos % self.page].astype(F) * self.scales[w][pid][:, None]
        return out


def attend(cache, q, table, lens, cu, scale, causal, window, dtype, hidden=()):
    """(out, bound) in 64 bits, without the keys of the pages hidden (sequence, place in its table); `bound` is how far the library's result may be off, element by element.

    Per probability: f16 rounding, 11 significant bits and so at most 2^-11 (f32 queries: two parts, 2^-22), and the error of
    its score, twice (numerator and denominator). Codes are exact, and the value scales enter in f32 before that rounding. A score is a sum of hd exact products in f32, in the tensor cores' order: at most (hd + 8) half-steps
    of truncation (2^-23) of sum |q k|, and for 16-bit queries, whose codes enter as 1152 + code against a start of -1152
    times the row's sum, of 16 partial sums of size 1152 sum |q| k_scale more; exp2 and the scale products add less than 2^-20 relative for the scores' size met
    here. A probability is rounded in units of 2^-7 (at the coarsest) of the largest value scale `ref`: f16's finest step
    2^-24 there puts an absolute 2^-25 * 2^-7 * ref * 127 on each key's term, whatever its size, against a sum of at
    least 1. The sums over L keys: (L / 8 + 32) * 2^-23. Then one rounding to the output type: f16 results below 2^-14 are
    subnormal with steps of 2^-24, so that rounding alone is up to 2^-25 there, whatever the value."""
    rows, heads, hd = q.shape
    share = heads // cache.heads
    out, bound = np.zeros((rows, heads, hd)), np.zeros((rows, heads, hd))
    prob = 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11
    for s in range(len(lens)):
        L, n = int(lens[s]), int(cu[s + 1] - cu[s])
        if n == 0 or L == 0:
            continue
        k, v = (cache.rows(w, table, s, 0, L).astype(np.float64) for w in range(2))
        ref = max(float(cache.scales[1][p].max()) for p in table[s][:-(-L // cache.page)])
        for i in range(n):
            pos = L - n + i
            seen = np.ones(L, bool)
            if causal:
                seen &= np.arange(L) <= pos
            if window:
                seen &= np.arange(L) > pos - window
            for hs, pg in hidden:
                if hs == s:
                    seen[pg * cache.page:(pg + 1) * cache.page] = False
            if not seen.any():
                continue
            biased = 0.0
            if dtype != torch.float32:
                biased = 16 * 2.0 ** -23 * 1152 * max(cache.scales[0][table[s][j // cache.page]].max() for j in np.flatnonzero(seen))
            for h in range(heads):
                qq = q[cu[s] + i, h].astype(np.float64)
                kk, vv = k[seen, h // share], v[seen, h // share]
                e = kk @ qq * scale
                p = np.exp(e - e.max())
                p /= p.sum()
                off = (hd + 8) * 2.0 ** -23 * (np.abs(kk) @ np.abs(qq) * abs(scale)).max() + 2.0 ** -21 * np.abs(e).max()
                off += biased * np.abs(qq).sum() * abs(scale)
                out[cu[s] + i, h] = p @ vv
                bound[cu[s] + i, h] = ((p @ np.abs(vv)) * (prob + 2 * off + 2.0 ** -20 + (L / 8 + 32) * 2.0 ** -23) +
                                       L * 127 * 2.0 ** -32 * ref)
    return out, bound + HALF[dtype] * (np.abs(out) + bound) + (2.0 ** -25 if dtype == torch.float16 else 1e-30)
