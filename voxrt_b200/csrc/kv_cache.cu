// Paged int8 key / value cache: one scale per (page, head), codes [n_pages][heads][page][head_dim].
//
// Writing n new tokens of a sequence behind its `start` cached ones, per touched (page, head):
//   A = max |new|, finite values only;  s0 = the stored scale if the page holds earlier tokens of the sequence, else 0;
//   s = max(s0, A / 127)  (A / 127 not below 2^-126, so that 1 / s is finite; 0 while everything is zero);
//   earlier codes: c -> round_ties_even(c * (s0 / s)) where s != s0;
//   new codes: clamp(round_ties_even(x * (1 / s)), +-127), a NaN is stored as 0, and 0 where s = 0.
// A scale only grows while a page fills, so a token written alone is off by at most half a step of the page's final
// scale plus half a step for each growth after it.
//
// Bound by memory for long runs, by the chain of dependent loads (offsets, page table, values) for single tokens: one
// block takes one page of K or V and a run of heads, finds its sequence with 32 probes a step, and holds a head's new values
// in registers between the maximum and the codes, with the next head's on their way. Measured: 64 sequences of one token
// 5.5 us; 8 ragged sequences of up to 2048 tokens, 8 heads of 128, 24.7 us (79 MB, 3.2 TB/s), read back 21.0 us (80 MB,
// 3.8 TB/s).
#include <cuda_runtime.h>

#include <algorithm>

#include "common.h"
#include "dtype.cuh"
#include "kv_cache.cuh"
#include "math.cuh"

namespace vxg {
namespace cache {

struct WriteParams {
  vxg_kv_cache c;
  const void* src[2];
  long long ld[2];
  const int* table;
  const int* start;
  const int* cu;
  int* status;
  int total, n_seq, max_pages, run;  // run: heads of a block
};

__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.402823466e38f ? a : 0.0f;  // NaN and infinity take no part in the scale
}

// code of v under inv = 1 / s: an infinity is the largest code (inv > 0), a NaN 0
__device__ __forceinline__ uint32_t code8(float v, float inv) { return (uint32_t)quant_code(v, inv) & 0xFFu; }

// Largest i < n with at(i) <= x, or 0; `at` does not decrease. Every lane of the warp asks for the same x.
template <class At>
__device__ __forceinline__ int find32(int n, long long x, At at) {
  const int lane = threadIdx.x & 31;
  int lo = 0;
  while (n > 1) {
    const int step = (n + 31) / 32, i = lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, i < n && at(lo + i) <= x);
    const int k = below ? 31 - __clz(below) : 0;
    lo += k * step;
    n = ::min(step, n - k * step);
  }
  return lo;
}

// Pages of sequence s in the launch's item order: at most (cu[s+1] - cu[s] - 2) / page + 2 of them are touched, and
// items base(s) .. base(s + 1) with base(s) = cu[s] / page + 2 s are as many or more, so that total / page + 2 n_seq
// items cover every batch without the host knowing its lengths. NV: vectors of eight values a thread holds; with fewer
// threads than that covers (LONG) the rest is read twice.
template <int DT, int THREADS, int NV, bool VEC, bool LONG>
__global__ void __launch_bounds__(THREADS) cache_write_kernel(const WriteParams p) {
  using T = typename Elem<DT>::type;
  __shared__ float wmax[2][THREADS / 32];
  const int P = p.c.page, H = p.c.heads, D = p.c.head_dim;
  const int item = blockIdx.x, which = blockIdx.z, h0 = blockIdx.y * p.run, h1 = ::min(H, h0 + p.run);
  auto base = [&](int s) { return (long long)(__ldg(p.cu + s) / P) + 2LL * s; };
  const int s = find32(p.n_seq, item, base);
  const int t0 = __ldg(p.cu + s), n = __ldg(p.cu + s + 1) - t0;
  if (n == 0) return;
  const long long a = __ldg(p.start + s);
  const bool good = t0 >= 0 && n >= 0 && (long long)t0 + n <= p.total && a >= 0 && a + n <= (long long)p.max_pages * P;
  if (!good) {
    if (threadIdx.x == 0) atomicCAS(p.status + 1, 0, VXG_DEV_CACHE_INDEX);
    return;
  }
  const int first = (int)a / P, pg = first + (int)(item - base(s));  // page of the sequence; a + n < 2^31
  if (pg < first || (long long)pg * P >= a + n) return;
  const int pid = __ldg(p.table + (size_t)s * p.max_pages + pg);
  const int held = pg == first ? (int)a - pg * P : 0;                   // earlier tokens of the sequence in this page
  const int end = (int)::min(a + n - (long long)pg * P, (long long)P);  // new tokens: slots held .. end
  const long long tok = t0 + ((long long)pg * P + held - a);            // stacked row of slot `held`
  const T* x = static_cast<const T*>(p.src[which]) + tok * p.ld[which];
  const long long ld = p.ld[which];
  const int shift = D == 128 ? 4 : 3, vpr = 1 << shift, vecs = (end - held) << shift;
  auto at = [&](int h, int i) { return x + (i >> shift) * ld + (size_t)h * D + (i & (vpr - 1)) * 8; };
  auto load = [&](int h, int i, float (&f)[8]) {
    const T* r = at(h, i);
    if (VEC) {
      load8<DT>(r, f);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) f[e] = Elem<DT>::widen(r[e]);
    }
  };
  // the thread's first HELD vectors stay in registers as they lie in memory
  constexpr int HELD = VEC ? NV : 0;
  Raw<DT> raw[NV], ahead[NV];
  auto fetch = [&](int h, Raw<DT> (&v)[NV]) {
#pragma unroll
    for (int j = 0; j < HELD; j++)
      if ((int)threadIdx.x + j * THREADS < vecs) {
        const uint4* r = reinterpret_cast<const uint4*>(at(h, (int)threadIdx.x + j * THREADS));
        v[j].w[0] = r[0];
        if constexpr (DT == VXG_DT_F32) v[j].w[1] = r[1];
      }
  };
  fetch(h0, raw);  // on their way before the page's id is here
  if (pid < 0 || pid >= p.c.n_pages) {
    if (threadIdx.x == 0) atomicCAS(p.status + 1, 0, VXG_DEV_CACHE_INDEX);
    return;
  }
  float* scales = (which ? p.c.v_scales : p.c.k_scales) + (size_t)pid * H;
  int8_t* pages = (which ? p.c.v : p.c.k) + (size_t)pid * H * P * D;
  float s0 = held ? scales[h0] : 0.0f;
  for (int h = h0; h < h1; h++) {
    float s0n = 0.0f;
    if (h + 1 < h1) {
      fetch(h + 1, ahead);
      if (held) s0n = scales[h + 1];
    }
    auto each = [&](auto&& f) {  // f(i, values) for the thread's vectors
#pragma unroll
      for (int j = 0; j < HELD; j++)
        if ((int)threadIdx.x + j * THREADS < vecs) {
          float v[8];
          unpack<DT>(raw[j], v);
          f((int)threadIdx.x + j * THREADS, v);
        }
      if (LONG || !VEC)
        for (int i = threadIdx.x + HELD * THREADS; i < vecs; i += THREADS) {
          float v[8];
          load(h, i, v);
          f(i, v);
        }
    };
    float m = 0.0f, seen = 0.0f;  // seen: NaN if one of the thread's values is
    each([&](int, const float (&v)[8]) {
#pragma unroll
      for (int e = 0; e < 8; e++) m = fmaxf(m, fabsf(v[e])), seen = max_nan(seen, v[e]);
    });
    const bool plain = seen == seen && m <= 3.402823466e38f;  // every value of the thread finite
    if (!plain) {
      m = 0.0f;
      each([&](int, const float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; e++) m = fmaxf(m, finite_abs(v[e]));
      });
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) wmax[h & 1][threadIdx.x >> 5] = m;
    __syncthreads();  // also: every thread has read the old scale before one of them writes the new one
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) m = fmaxf(m, wmax[h & 1][w]);
    const float s1 = fmaxf(s0, m > 0.0f ? fmaxf(__fdiv_rn(m, 127.0f), 1.17549435e-38f) : 0.0f);
    int8_t* codes = pages + (size_t)h * P * D;
    if (threadIdx.x == 0) scales[h] = s1;
    if (held && s1 != s0) {
      const float ratio = __fdiv_rn(s0, s1);
      for (int i = threadIdx.x; i < held * D / 4; i += THREADS) {
        const uint32_t w = reinterpret_cast<uint32_t*>(codes)[i];
        uint32_t r = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) r |= code8((float)(int8_t)(w >> (8 * e)), ratio) << (8 * e);
        reinterpret_cast<uint32_t*>(codes)[i] = r;
      }
    }
    const float inv = s1 > 0.0f ? __fdiv_rn(1.0f, s1) : 0.0f;  // finite: s1 >= 2^-126
    each([&](int i, const float (&v)[8]) {
      uint32_t w[2] = {0, 0};
      if (plain) {  // |value * inv| <= 127 (1 + 2^-23): the code is the rounding shifter's low byte
#pragma unroll
        for (int k = 0; k < 2; k++) w[k] = quant_word_fast(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3], inv);
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) w[e >> 2] |= code8(v[e], inv) << (8 * (e & 3));
      }
      *reinterpret_cast<uint2*>(codes + (size_t)held * D + (size_t)i * 8) = make_uint2(w[0], w[1]);
    });
    s0 = s0n;
#pragma unroll
    for (int j = 0; j < HELD; j++) raw[j] = ahead[j];
  }
}

template <int DT, int THREADS, int NV, bool LONG>
void write_launch(WriteParams p, int items, bool vec, cudaStream_t st) {
  // heads of a block: all of them once that leaves four blocks for every SM
  p.run = (int)std::max(1LL, std::min((long long)p.c.heads, 2LL * items * p.c.heads / (4LL * sm_count())));
  const dim3 grid((unsigned)items, (unsigned)((p.c.heads + p.run - 1) / p.run), 2);
  if (vec) cache_write_kernel<DT, THREADS, NV, true, LONG><<<grid, THREADS, 0, st>>>(p);
  else cache_write_kernel<DT, THREADS, NV, false, LONG><<<grid, THREADS, 0, st>>>(p);
}

struct ReadParams {
  vxg_kv_cache c;
  void* dst[2];
  const int* table;
  const int* start;
  const int* cu;
  int* status;
  int total, n_seq, max_pages;
};

// A thread reads 16 codes of one (token, head).
template <int DT>
__global__ void __launch_bounds__(256) cache_read_kernel(ReadParams p) {
  using T = typename Elem<DT>::type;
  const int P = p.c.page, H = p.c.heads, D = p.c.head_dim, vpt = H * D / 16;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  // the sequence of the warp's first token, then on to this thread's
  int lo = find32(p.n_seq, (i & ~31LL) / vpt, [&](int s) { return (long long)__ldg(p.cu + s); });
  const long long tok = i / vpt;
  if (tok >= p.total) return;
  while (lo + 1 < p.n_seq && __ldg(p.cu + lo + 1) <= tok) lo++;
  const long long a = __ldg(p.start + lo), t0 = __ldg(p.cu + lo), t1 = __ldg(p.cu + lo + 1), at = tok - t0;
  if (at < 0 || tok >= t1) return;  // rows behind the last sequence stay as they are
  const int e = (int)(i % vpt) * 16, h = e / D;
  const long long pos = a + at;
  int pid = -1;
  if (t0 >= 0 && t1 <= p.total && a >= 0 && a + (t1 - t0) <= (long long)p.max_pages * P) pid = __ldg(p.table + (size_t)lo * p.max_pages + pos / P);
  if (pid < 0 || pid >= p.c.n_pages) {
    atomicCAS(p.status + 1, 0, VXG_DEV_CACHE_INDEX);
    return;
  }
  const size_t ph = (size_t)pid * H + h, src = (ph * P + pos % P) * D + (e - h * D);
#pragma unroll
  for (int w = 0; w < 2; w++) {
    T* out = static_cast<T*>(p.dst[w]);
    if (!out) continue;
    const float s = __ldg((w ? p.c.v_scales : p.c.k_scales) + ph);
    const uint4 c4 = *reinterpret_cast<const uint4*>((w ? p.c.v : p.c.k) + src);
    const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
    for (int k = 0; k < 2; k++) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; j++) f[j] = __fmul_rn((float)(int8_t)(c[2 * k + (j >> 2)] >> (8 * (j & 3))), s);
      store8<DT>(out + tok * H * D + e + 8 * k, f);
    }
  }
}

}  // namespace cache

vxg_status cache_check(const vxg_kv_cache* c) {
  VXG_ARG(c, "NULL cache");
  VXG_ARG(c->n_pages > 0 && c->heads > 0, "bad cache shape: %d pages of %d heads", c->n_pages, c->heads);
  VXG_ARG(c->k && c->v && c->k_scales && c->v_scales, "NULL cache buffer");
  VXG_ARG(aligned(16, c->k, c->v) && aligned(4, c->k_scales, c->v_scales),
          "the cache's codes must be 16-byte aligned, its scales 4-byte aligned");
  if ((c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128) ||
      (c->head_dim != 64 && c->head_dim != 128) || c->heads > 65535 ||
      (long long)c->n_pages * c->heads * c->page > 0x7FFFFFFFLL) {
    set_error("cache of %d pages of %d tokens, %d heads of %d not supported (16, 32, 64 or 128 tokens; heads of 64 or "
              "128; fewer than 2^31 rows)", c->n_pages, c->page, c->heads, c->head_dim);
    return VXG_ERR_UNSUPPORTED;
  }
  return VXG_OK;
}

vxg_status cache_batch_check(const vxg_kv_cache* c, const int* table, int n_seq, int max_pages, const int* a,
                             const int* cu, int total) {
  VXG_ARG(n_seq >= 0 && max_pages >= 0 && total >= 0, "bad batch: %d sequences of %d pages, %d rows", n_seq, max_pages,
          total);
  VXG_ARG(n_seq == 0 || total == 0 || (table && a && cu && max_pages > 0), "NULL page table, lengths or offsets");
  VXG_ARG(aligned(4, table, a, cu), "page table, lengths and offsets must be 4-byte aligned");
  if ((long long)max_pages * c->page > 0x7FFFFF00LL || n_seq > (1 << 30)) {  // 32 probes a step pass 31 bits beyond
    set_error("%d sequences of %d pages of %d tokens not supported", n_seq, max_pages, c->page);
    return VXG_ERR_UNSUPPORTED;
  }
  return VXG_OK;
}

}  // namespace vxg

using namespace vxg;

extern "C" {

vxg_status vxg_cache_write(const vxg_kv_cache* c, const void* k, long long ld_k, const void* v, long long ld_v, int dtype,
                           int total, const int* table, int n_seq, int max_pages, const int* start, const int* cu,
                           void* stream) {
  clear_error();
  vxg_status r = cache_check(c);
  if (r == VXG_OK) r = cache_batch_check(c, table, n_seq, max_pages, start, cu, total);
  if (r != VXG_OK) return r;
  VXG_ARG(dtype_known(dtype), "unknown element type %d", dtype);
  if (total == 0 || n_seq == 0) return VXG_OK;
  VXG_ARG(k && v, "NULL input");
  VXG_ARG(aligned(dtype_bytes(dtype), k, v), "k and v are not aligned to their elements");
  const long long row = (long long)c->heads * c->head_dim;
  VXG_ARG(ld_k >= row && ld_v >= row, "a row stride is below heads * head_dim = %lld", row);
  const long long items = (long long)total / c->page + 2LL * n_seq;
  if (items > 0x7FFFFFFFLL) {
    set_error("%d sequences of %d rows are more than one launch covers", n_seq, total);
    return VXG_ERR_UNSUPPORTED;
  }
  int* status = device_status();
  VXG_ARG(status, "no CUDA device");
  const long long eb = (long long)dtype_bytes(dtype);
  const bool vec = (((uintptr_t)k | (uintptr_t)v | (uintptr_t)(ld_k * eb) | (uintptr_t)(ld_v * eb)) & 15) == 0;
  cache::WriteParams p = {*c, {k, v}, {ld_k, ld_v}, table, start, cu, status, total, n_seq, max_pages, 1};
  with_dtype(dtype, [&](auto tag) {
    constexpr int DT = decltype(tag)::value;
    cudaStream_t st = (cudaStream_t)stream;
    const int most = std::min(total, c->page) * c->head_dim / 8;  // vectors of a page and head
    // a few tokens a sequence: small blocks, which all fit the GPU at once (64 sequences of one token: 5.2 us, 9.1 us with
    // blocks of 256)
    if (total <= 4LL * n_seq) cache::write_launch<DT, 64, 1, true>(p, (int)items, vec, st);
    else if (most <= 512) cache::write_launch<DT, 256, 2, false>(p, (int)items, vec, st);
    else if (most <= 1024) cache::write_launch<DT, 256, 4, false>(p, (int)items, vec, st);
    else cache::write_launch<DT, 256, 8, false>(p, (int)items, vec, st);
  });
  note_launch();
  VXG_CUDA(cudaGetLastError());
  return VXG_OK;
}

vxg_status vxg_cache_read(const vxg_kv_cache* c, const int* table, int n_seq, int max_pages, const int* start,
                          const int* cu, int total, int dtype, void* k, void* v, void* stream) {
  clear_error();
  vxg_status r = cache_check(c);
  if (r == VXG_OK) r = cache_batch_check(c, table, n_seq, max_pages, start, cu, total);
  if (r != VXG_OK) return r;
  VXG_ARG(dtype_known(dtype), "unknown element type %d", dtype);
  if (total == 0 || n_seq == 0) return VXG_OK;
  VXG_ARG(k || v, "no output given");
  VXG_ARG((((uintptr_t)k | (uintptr_t)v) & 15) == 0, "outputs must be 16-byte aligned");
  const long long blocks = ((long long)total * (c->heads * c->head_dim / 16) + 255) / 256;
  if (blocks > 0x7FFFFFFFLL) {
    set_error("%d rows are more than one launch covers", total);
    return VXG_ERR_UNSUPPORTED;
  }
  int* status = device_status();
  VXG_ARG(status, "no CUDA device");
  cache::ReadParams p = {*c, {k, v}, table, start, cu, status, total, n_seq, max_pages};
  with_dtype(dtype, [&](auto tag) {
    constexpr int DT = decltype(tag)::value;
    cache::cache_read_kernel<DT><<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(p);
  });
  note_launch();
  VXG_CUDA(cudaGetLastError());
  return VXG_OK;
}

}  // extern "C"
