// Attention over the paged int8 cache for many queries: tiles of 256 (query, query head) rows on tcgen05.
//
// A CTA holds two halves of 128 rows. Per block of 128 keys, four warps turn the codes into f16 operands in shared memory
// (keys as they are, values times v_scale / ref * 2^8 with ref the largest value scale of the piece, rounding 2^-11),
// one thread issues S = Q K^T and O += P V for both halves in turn, and a warpgroup a half does the softmax: a thread
// owns a row, reads its 128 scores from TMEM twice (maximum, then exponentials) and writes the probabilities back over
// them as f16, which is the second product's operand. While one half is in its softmax the tensor cores work for the
// other. The row's reference maximum only moves when a score exceeds it by more than 8 (in powers of two): probabilities
// then are at most 2^8, times 2^7 for the sake of f16's small end, and O is rarely rescaled. Softmax sums, scores and O are
// f32. Query rows are scaled by a power of two like in the few-row kernels.
//
// TMEM (512 columns): S and P of the halves at 0 and 128, O at 256 and 256 + HD. A half's next S overwrites its P: the
// tensor cores run one thread's products in order, and the commit that reports S also reports the product before it.
#include <cuda_runtime.h>

#include "cached_attention.cuh"

namespace vxg {
namespace catt {
namespace tc {

constexpr int MT = 256, BK = 128;
constexpr int SOFT_WARPS = 8, CONV_WARPS = 4, MMA_WARP = SOFT_WARPS + CONV_WARPS;
constexpr int THREADS = (MMA_WARP + 1) * 32;
constexpr int RING = 4;  // blocks (scales) and pieces (ref) that the converting warps can be ahead, and one more

template <int HD>
struct Layout {
  static constexpr uint32_t HALF = 128 * 128;             // 128 rows of 64 f16
  static constexpr uint32_t OPER = HD / 64 * HALF;        // 128 rows of HD
  static constexpr uint32_t Q = 0;                        // [2]
  static constexpr uint32_t K = Q + 2 * OPER;             // [2]
  static constexpr uint32_t V = K + 2 * OPER;             // [2]
  static constexpr uint32_t KS = V + 2 * OPER;            // [RING][8] f32
  static constexpr uint32_t REF = KS + RING * 32;         // [RING] f32
  static constexpr uint32_t BARS = REF + RING * 4;
  static constexpr uint32_t BYTES = BARS + 20 * 8 + 1024;
  static_assert(BYTES <= 232448, "shared memory budget");
};

// The blocks of a share, one after the other; pieces without a key are passed over.
struct Blocks {
  Piece w;
  int b, nb, piece;  // block of the piece, blocks it has, pieces so far
  __device__ __forceinline__ Blocks(const Params& p, const Piece& first) : w(first), piece(0) { settle(p); }
  __device__ __forceinline__ bool done() const { return w.left <= 0; }
  __device__ __forceinline__ void settle(const Params& p) {
    while (w.left > 0 && w.t.nblk == 0) w.next(p, MT, BK);
    b = 0;
    nb = w.left > 0 ? w.take() : 0;
  }
  __device__ __forceinline__ void next(const Params& p) {
    if (++b == nb) {
      w.next(p, MT, BK);
      settle(p);
      piece++;
    }
  }
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <int HD, int DT>
__global__ void __launch_bounds__(THREADS, 1) attend_tc_kernel(const Params p) {
  using Lay = Layout<HD>;
  using T = typename Elem<DT>::type;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* ks_s = reinterpret_cast<float*>(smem + Lay::KS);
  float* ref_s = reinterpret_cast<float*>(smem + Lay::REF);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Lay::BARS);
  uint64_t *kfull = bars, *kempty = bars + 2, *vfull = bars + 4, *vempty = bars + 6;  // by stage
  uint64_t *qfull = bars + 8, *sfull = bars + 10, *pfull = bars + 12, *ofull = bars + 14;  // by half
  uint64_t* drain = bars + 16;
  __shared__ Piece first_s;
  __shared__ uint32_t holder;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int KV = p.c.heads, P = p.c.page;

  if (tid == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(kfull + i, CONV_WARPS);
      mbar_init(kempty + i, 1);
      mbar_init(vfull + i, CONV_WARPS);
      mbar_init(vempty + i, 1);
      mbar_init(qfull + i, 4);
      mbar_init(sfull + i, 1);
      mbar_init(pfull + i, 4);
      mbar_init(ofull + i, 1);
    }
    mbar_init(drain, 1);
    fence_mbar_init();
  }
  if (warp == MMA_WARP) {
    tmem_alloc(&holder, 512);
    tmem_relinquish();
  }
  __syncwarp();
  tc_fence_before();
  find_share<THREADS, MT, BK>(p, &first_s);  // ends with a block barrier
  tc_fence_after();
  const uint32_t tmem = holder;
  const Piece first = first_s;

  if (warp >= SOFT_WARPS && warp < MMA_WARP) {
    // ---------------------------------------------------------------------------------------- codes -> operands
    // Pass i of a block covers its keys 16 i .. 16 i + 15, which lie in one page: warp v takes four of them, eight lanes
    // (16 codes each) a key.
    constexpr int LPK = HD / 16, KPW = 32 / LPK;          // lanes a key, keys a warp and pass
    constexpr int PASSES = BK / (CONV_WARPS * KPW);        // 8 for 128 columns, 4 for 64
    constexpr int CHUNKS = BK / 16;
    const int cw = warp - SOFT_WARPS, kk = cw * KPW + lane / LPK, e0 = lane % LPK * 16;
    uint4 kr[PASSES], vr[PASSES];
    int pid = -1;           // page of the block's 16-key piece `lane` (lanes 0 .. 7)
    float ksl = 0.0f, vsl = 0.0f;
    float ref = 0.0f, vf_l = 0.0f;
    bool ok = true;
    auto pages = [&](const Blocks& x) {
      pid = -1, ksl = 0.0f, vsl = 0.0f;
      const Tile& t = x.w.t;
      const long long key = (long long)(t.blk0 + x.w.off + x.b) * BK + 16 * lane;
      const long long pg = key / P;
      if (lane < CHUNKS && pg * P < t.kmax && (pg + 1) * P > t.kmin) {
        pid = __ldg(p.table + (size_t)t.s * p.max_pages + pg);
        if (pid < 0 || pid >= p.c.n_pages) {
          atomicCAS(p.status + 1, 0, VXG_DEV_CACHE_INDEX);
          pid = -1;
        } else {
          ksl = __ldg(p.c.k_scales + (size_t)pid * KV + x.w.h);
          vsl = __ldg(p.c.v_scales + (size_t)pid * KV + x.w.h);
        }
      }
    };
    auto load = [&](const Blocks& x, const int8_t* codes, uint4 (&r)[PASSES]) {
      const long long key0 = (long long)(x.w.t.blk0 + x.w.off + x.b) * BK;
#pragma unroll
      for (int i = 0; i < PASSES; i++) {
        const int k = i * CONV_WARPS * KPW + kk;
        const int id = __shfl_sync(0xffffffffu, pid, k / 16);
        r[i] = make_uint4(0, 0, 0, 0);
        if (id >= 0 && key0 + k < x.w.t.kmax)
          r[i] = __ldg(reinterpret_cast<const uint4*>(codes + (((size_t)id * KV + x.w.h) * P + (size_t)((key0 + k) % P)) * HD + e0));
      }
    };
    auto largest = [&](const Blocks& x) {  // the piece's largest value scale
      const Tile& t = x.w.t;
      const long long k0 = ::max((long long)(t.blk0 + x.w.off) * BK, (long long)t.kmin);
      const long long k1 = ::min((long long)(t.blk0 + x.w.off + x.nb) * BK, (long long)t.kmax);
      float m = 0.0f;
      for (long long pg = k0 / P + lane; pg * P < k1; pg += 32) {
        const int id = __ldg(p.table + (size_t)t.s * p.max_pages + pg);
        if (id >= 0 && id < p.c.n_pages) m = fmaxf(m, __ldg(p.c.v_scales + (size_t)id * KV + x.w.h));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      return m;
    };
    // 16 codes -> two 16-byte chunks of the operand row; the upper half of the lanes of a key stores its odd chunk first,
    // so that the eight lanes of a store phase meet eight different chunks
    auto put = [&](uint8_t* dst, int k, uint4 x, bool scaled, __half2 f) {
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
      uint32_t h[8];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        h[2 * i] = codes_to_f16(__byte_perm(w[i], 0, 0x4140));
        h[2 * i + 1] = codes_to_f16(__byte_perm(w[i], 0, 0x4342));
      }
      if (scaled) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const __half2 v = __hmul2(*reinterpret_cast<__half2*>(&h[i]), f);
          h[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
      }
      uint8_t* base = dst + (e0 / 64) * Lay::HALF;
      const uint32_t c = (uint32_t)(e0 % 64) / 8;
      const bool odd = HD == 128 && e0 >= 64;
      const uint4 a = make_uint4(h[0], h[1], h[2], h[3]), b = make_uint4(h[4], h[5], h[6], h[7]);
      *reinterpret_cast<uint4*>(base + sw128_offset((uint32_t)k, c + (odd ? 1 : 0))) = odd ? b : a;
      *reinterpret_cast<uint4*>(base + sw128_offset((uint32_t)k, c + (odd ? 0 : 1))) = odd ? a : b;
    };
    Blocks x(p, first);
    if (!x.done()) {
      pages(x);
      ref = largest(x);
      load(x, p.c.k, kr);
      load(x, p.c.v, vr);
    }
    for (int it = 0; !x.done(); it++) {
      const int st = it & 1;
      if (it >= 2 && !wait_phase(kempty + st, ((it >> 1) - 1) & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (cw == 0) {
        if (lane < 8) ks_s[(it % RING) * 8 + lane] = ksl;
        if (lane == 8 && x.b == 0) ref_s[x.piece % RING] = ref;
      }
#pragma unroll
      for (int i = 0; i < PASSES; i++)
        put(smem + Lay::K + st * Lay::OPER, i * CONV_WARPS * KPW + kk, kr[i], false, __half2());
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(kfull + st);
      vf_l = ref > 0.0f ? vsl / ref * 256.0f : 0.0f;
      // the next block's page, scales and keys on their way before this block's values are written
      Blocks nx = x;
      nx.next(p);
      if (!nx.done()) {
        pages(nx);
        if (nx.b == 0) ref = largest(nx);
        load(nx, p.c.k, kr);
      }
      if (it >= 2 && !wait_phase(vempty + st, ((it >> 1) - 1) & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
#pragma unroll
      for (int i = 0; i < PASSES; i++) {
        const int k = i * CONV_WARPS * KPW + kk;
        put(smem + Lay::V + st * Lay::OPER, k, vr[i], true, __float2half2_rn(__shfl_sync(0xffffffffu, vf_l, k / 16)));
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(vfull + st);
      if (!nx.done()) load(nx, p.c.v, vr);
      x = nx;
    }
  } else if (warp == MMA_WARP) {
    // --------------------------------------------------------------------------------------------- MMA issuer
    if (lane == 0) {
      constexpr uint32_t QK = idesc_f16(128, BK, false), PV = idesc_f16(128, HD, true);
      bool ok = true;
      uint32_t nq = 0, np = 0;  // pieces begun, probabilities consumed (per half)
      int it = 0;
      auto wait = [&](uint64_t* b, uint32_t phase) {
        if (ok && !wait_phase(b, phase & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN)) ok = false;
        if (ok) tc_fence_after();
        return ok;
      };
      auto scores = [&](int half, int st) {
        const uint32_t q = smem_u32(smem + Lay::Q + half * Lay::OPER), k = smem_u32(smem + Lay::K + st * Lay::OPER);
#pragma unroll
        for (int c = 0; c < HD / 64; c++)
#pragma unroll
          for (int j = 0; j < 4; j++)
            mma_f16_ss(tmem + half * 128, umma_desc_sw128(q + c * Lay::HALF) + 2 * j, umma_desc_sw128(k + c * Lay::HALF) + 2 * j,
                       QK, (c | j) != 0 ? 1u : 0u);
        mma_commit(sfull + half);
      };
      auto values = [&](int half, int st, bool fresh) {
        const uint32_t v = smem_u32(smem + Lay::V + st * Lay::OPER);
#pragma unroll
        for (int j = 0; j < BK / 16; j++)
          mma_f16_ts(tmem + 256 + half * HD, tmem + half * 128 + 8 * j, umma_desc_sw128_mn(v + j * 2048, Lay::HALF), PV,
                     fresh && j == 0 ? 0u : 1u);
      };
      for (Blocks x(p, first); !x.done() && ok;) {
        for (int half = 0; half < 2 && ok; half++) {
          if (!wait(qfull + half, nq)) break;
          if (half == 0 && !wait(kfull + (it & 1), it >> 1)) break;
          scores(half, it & 1);
        }
        if (!ok) break;
        mma_commit(kempty + (it & 1));
        nq++;
        const int nb = x.nb;
        for (int b = 0; b < nb && ok; b++, it++, np++) {
          const bool more = b + 1 < nb;
          if (!wait(vfull + (it & 1), it >> 1)) break;
          for (int half = 0; half < 2 && ok; half++) {
            if (!wait(pfull + half, np)) break;
            values(half, it & 1, b == 0);
            if (!more) mma_commit(ofull + half);
            if (more && half == 0 && !wait(kfull + ((it + 1) & 1), (it + 1) >> 1)) break;
            if (more) scores(half, (it + 1) & 1);
          }
          if (!ok) break;
          mma_commit(vempty + (it & 1));
          if (more) mma_commit(kempty + ((it + 1) & 1));
          x.next(p);
        }
      }
      mma_commit(drain);  // nothing is in flight when the block ends
      wait_phase(drain, 0, p.status, VXG_DEV_TIMEOUT_DRAIN);
    }
  } else {
    // ------------------------------------------------------------------------------------------------ softmax
    const int half = warp >> 2, r = half * 128 + (warp & 3) * 32 + lane;  // the thread's row of the tile
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t S = tmem + lanes + half * 128, O = tmem + lanes + 256 + half * HD;
    bool ok = true;
    uint32_t it = 0, pieces = 0;
    for (Piece w = first; w.left > 0 && ok; w.next(p, MT, BK)) {
      const Tile& t = w.t;
      const int take = w.take(), nb = t.nblk > 0 ? take : 0;
      const bool live = r < t.rows;
      const int rr = t.r0 + (live ? r : 0), i = rr / p.share, head = w.h * p.share + rr % p.share;
      const long long pos = (long long)t.L - t.n + i;
      const int khi = p.causal ? (int)::max(0LL, ::min((long long)t.L, pos + 1)) : t.L;
      const int klo = p.window > 0 ? (int)::max(0LL, pos - p.window + 1) : 0;
      float m = -INFINITY, l = 0.0f, unit = 0.0f;
      if (nb > 0) {
        // ---- this row of Q: scaled by a power of two, f16, into the half's operand
        const T* q = static_cast<const T*>(p.q) + (long long)(t.q0 + i) * p.ld_q + (long long)head * HD;
        auto chunk = [&](int c) { return live ? reinterpret_cast<const uint4*>(q)[c] : make_uint4(0, 0, 0, 0); };
        float top = 0.0f;
#pragma unroll 4
        for (int c = 0; c < HD / 8; c++) {
          const uint4 raw = chunk(c);
          const uint32_t x[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const float2 f = widen2<DT>(x[k]);
            top = max3(top, fabsf(f.x), fabsf(f.y));
          }
        }
        int ex = 14 - ((int)(__float_as_uint(top) >> 23) - 127);
        ex = top == 0.0f || !(top <= 3.402823466e38f) ? 0 : ::min(ex, 126);
        const float up = __int_as_float((ex + 127) << 23);
        const float rowf = __int_as_float((127 - ex) << 23) * p.scale_log2;
        uint8_t* qs = smem + Lay::Q + half * Lay::OPER;
#pragma unroll 4
        for (int c = 0; c < HD / 8; c++) {  // a second time, from L1
          const uint4 raw = chunk(c);
          const uint32_t x[4] = {raw.x, raw.y, raw.z, raw.w};
          uint32_t h[4];
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const float2 f = widen2<DT>(x[k]);
            h[k] = pack_f16(f.x * up, f.y * up);
          }
          *reinterpret_cast<uint4*>(qs + (c / 8) * Lay::HALF + sw128_offset((uint32_t)(r & 127), (uint32_t)(c % 8))) =
              make_uint4(h[0], h[1], h[2], h[3]);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(qfull + half);
        // keys that every row of the warp sees: [all_lo, all_hi)
        const int all_hi = __reduce_min_sync(0xffffffffu, live ? khi : 0x7FFFFFFF);
        const int all_lo = __reduce_max_sync(0xffffffffu, live ? klo : 0);

        for (int b = 0; b < nb; b++, it++) {
          if (ok && !wait_phase(sfull + half, it & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN)) ok = false;
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const int key0 = (t.blk0 + w.off + b) * BK;
          const bool inside = key0 >= all_lo && key0 + BK <= all_hi;
          const float* ks = ks_s + (it % RING) * 8;
          if (b == 0) unit = ref_s[pieces % RING] * (1.0f / 256.0f);
          // ---- the block's maximum
          float mx = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < BK; c += 32) {
            uint32_t a[32];
            tmem_ld32(S + c, a);
            tmem_wait_ld();
            if (!inside) {
#pragma unroll
              for (int j = 0; j < 32; j++)
                if (key0 + c + j < klo || key0 + c + j >= khi) a[j] = 0xFF800000u;  // -inf
            }
#pragma unroll
            for (int g = 0; g < 2; g++) {
              float x = max3(__uint_as_float(a[16 * g]), __uint_as_float(a[16 * g + 1]), __uint_as_float(a[16 * g + 2]));
#pragma unroll
              for (int j = 3; j < 15; j += 2)
                x = max3(x, __uint_as_float(a[16 * g + j]), __uint_as_float(a[16 * g + j + 1]));
              x = fmaxf(x, __uint_as_float(a[16 * g + 15]));
              const float f = rowf * ks[c / 16 + g];
              // -inf x 0 would be NaN: a piece without a visible key has no maximum
              mx = fmaxf(mx, x == -INFINITY ? x : x * f);
            }
          }
          // ---- move the reference when the maximum has outgrown it
          const bool grow = mx > m + 8.0f;
          if (__any_sync(0xffffffffu, grow)) {
            const float alpha = grow ? ex2(m - mx) : 1.0f;
            if (grow) m = mx;
            l *= alpha;
            if (b > 0) {
#pragma unroll 1
              for (int c = 0; c < HD; c += 32) {
                uint32_t a[32];
                tmem_ld32(O + c, a);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 32; j++) a[j] = __float_as_uint(__uint_as_float(a[j]) * alpha);
                tmem_st32(O + c, a);
              }
            }
          }
          const float mm = m == -INFINITY ? 0.0f : m - 7.0f;  // probabilities times 2^7
          // ---- probabilities over the scores: chunk c's 32 scores are read before its 16 columns are written
          float l0 = 0.0f, l1 = 0.0f;
#pragma unroll 1
          for (int c = 0; c < BK; c += 32) {
            uint32_t a[32], o[16];
            tmem_ld32(S + c, a);
            tmem_wait_ld();
            const float f0 = rowf * ks[c / 16], f1 = rowf * ks[c / 16 + 1];
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float f = j < 16 ? f0 : f1;
              float x0 = fmaf(__uint_as_float(a[j]), f, -mm), x1 = fmaf(__uint_as_float(a[j + 1]), f, -mm);
              if (!inside) {
                if (key0 + c + j < klo || key0 + c + j >= khi) x0 = -INFINITY;
                if (key0 + c + j + 1 < klo || key0 + c + j + 1 >= khi) x1 = -INFINITY;
              }
              const float p0 = ex2(x0), p1 = ex2(x1);
              l0 += p0;
              l1 += p1;
              o[j / 2] = pack_f16(p0, p1);
            }
            tmem_st16(S + c / 2, o);
          }
          l += l0 + l1;
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(pfull + half);
        }
        if (ok && !wait_phase(ofull + half, pieces & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        pieces++;
      }
      // ---- the row's result, whole or for the join
      const bool whole = w.off == 0 && take == t.cost;
      float* part = p.part + ((size_t)blockIdx.x * MAX_PIECES + (w.first ? 0 : 1)) * MT * (HD + 2) + (size_t)r * (HD + 2);
      T* out = static_cast<T*>(p.out) + (long long)(t.q0 + i) * p.ld_out + (long long)head * HD;
      const float inv = l == 0.0f ? 0.0f : unit / l;
      if (live && !whole) part[0] = m - 7.0f, part[1] = l;
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t a[32];
        if (nb > 0) {
          tmem_ld32(O + c, a);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int j = 0; j < 32; j++) a[j] = 0;
        }
        if (live && whole) {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = l == 0.0f ? 0.0f : __uint_as_float(a[j + k]) * inv;
            store8<DT>(out + c + j, v);
          }
        } else if (live) {
#pragma unroll
          for (int j = 0; j < 32; j += 2)
            *reinterpret_cast<float2*>(part + 2 + c + j) =
                make_float2(__uint_as_float(a[j]) * unit, __uint_as_float(a[j + 1]) * unit);
        }
        __syncwarp();
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int HD, int DT>
vxg_status launch(const Params& p, const Plan& pl, cudaStream_t st) {
  constexpr int smem = (int)Layout<HD>::BYTES;
  const vxg_status r = smem_attr((const void*)attend_tc_kernel<HD, DT>, smem);
  if (r != VXG_OK) return r;
  attend_tc_kernel<HD, DT><<<pl.grid, THREADS, smem, st>>>(p);
  VXG_CUDA(cudaGetLastError());
  join_kernel<HD, DT, MT, BK><<<dim3(pl.grid - 1, MT / 4), 128, 0, st>>>(p);
  note_launch(2);
  VXG_CUDA(cudaGetLastError());
  return VXG_OK;
}

}  // namespace tc

vxg_status launch_tc(const Params& p, const Plan& pl, int head_dim, int dtype, cudaStream_t st) {
  if (head_dim == 128)
    return dtype == VXG_DT_BF16 ? tc::launch<128, VXG_DT_BF16>(p, pl, st) : tc::launch<128, VXG_DT_F16>(p, pl, st);
  return dtype == VXG_DT_BF16 ? tc::launch<64, VXG_DT_BF16>(p, pl, st) : tc::launch<64, VXG_DT_F16>(p, pl, st);
}

}  // namespace catt
}  // namespace vxg
