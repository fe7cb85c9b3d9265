// Attention over the paged int8 cache for many queries: tiles of 256 (query, query head) rows on tcgen05.
//
// A CTA holds two halves of 128 rows. Per block of 128 keys, one warp brings the codes by TMA and four turn them into f16
// operands in shared memory, which is exact. One warp issues S = Q K^T and O += P V for both halves in turn, in steps of 64
// keys, and a warpgroup a half does the softmax: a thread owns a row, reads its 64 scores of a step from TMEM twice
// (maximum, then exponentials) and writes the probabilities back over them as f16, the second product's operand, times
// v_scale / ref with ref the largest value scale of the piece. That is the one rounding of an operand (2^-11): with the
// values scaled before the product there were two more, and f16 results were off by 3.2e-4 of their norm instead of 2.7e-4,
// at the same speed. A half has two score buffers, so that the next step's scores are ready when a softmax ends. The row's
// reference only moves when a score exceeds it by more than 2^8: probabilities are at most that, times 2^7 for the sake of
// f16's small end, and O is rarely rescaled. Softmax sums, scores and O are f32. Query rows are scaled by a power of two
// like in the other kernels.
//
// TMEM (512 columns): scores of a half at 128 half and 64 columns on, O at 256 + HD half. A step's scores overwrite the
// probabilities of the step before last: the tensor cores run one thread's products in order.
//
// Bound by the softmax warps, of which registers and TMEM allow two a scheduler, and by the pieces' ends, which are serial
// (the last product, the result, the next Q, the first product): per 128 keys and 256 rows the tensor cores need 2048
// clocks (measured alone) and the exponentials as many (16 a clock). Measured, 4 sequences of 2048 queries, 32 heads over
// 8: behind 4096, 8192 and 16384 tokens 806, 1377 and 2742 us, 2.6 to 3.1 us for a further block of 128 keys of a CTA; behind
// none 507 us, where the CTAs with the first queries' tiles have some 36 pieces of one to three blocks each, by which a
// piece's end costs about 10 us (inferred). 4 ragged sequences of up to 2048 queries behind up to 2000: 404 us, 500
// TFLOP/s of what is visible. Slower: longer unrolled loops (instruction fetches of four roles), one pass over scores held in
// registers. No gain: sixteen softmax warps of half rows, a quarter of the exponentials by polynomial.
#include <cuda_runtime.h>

#include <cmath>

#include "cached_attention.cuh"

namespace vxg {
namespace catt {
namespace tc {

constexpr int MT = 256, BK = 128, SB = 64;  // rows, keys of an operand stage, keys of a step of the softmax
constexpr int SOFT_WARPS = 8, CONV_WARPS = 4, MMA_WARP = SOFT_WARPS + CONV_WARPS, LOAD_WARP = MMA_WARP + 1;
constexpr int THREADS = (LOAD_WARP + 1) * 32;
// Blocks' scales and pieces' refs in flight: the loading warp fills block j only after block j - 1 has found a free operand
// stage, so after the scores of j - 3 and the softmax of j - 4; half of these would do.
constexpr int RING = 8;

template <int HD>
struct Layout {
  static constexpr uint32_t HALF = 128 * 128;             // 128 rows of 64 f16
  static constexpr uint32_t OPER = HD / 64 * HALF;        // 128 rows of HD
  static constexpr uint32_t Q = 0;                        // [2]
  static constexpr uint32_t K = Q + 2 * OPER;             // [2]
  static constexpr uint32_t V = K + 2 * OPER;             // [2]
  static constexpr uint32_t RAW = 128 * HD;               // a block's codes
  static constexpr uint32_t RK = V + 2 * OPER, RV = RK + RAW;
  static constexpr uint32_t KS = RV + RAW;                // [RING][8] f32: key scales of the block's 16-key pieces
  static constexpr uint32_t VF = KS + RING * 32;          // [RING][8] f32: their value scales / ref
  static constexpr uint32_t REF = VF + RING * 32;         // [RING] f32, its sign bit set where one of the piece's page ids is out of range
  static constexpr uint32_t BARS = REF + RING * 4;
  static constexpr uint32_t BYTES = BARS + 27 * 8 + 1024;
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
__global__ void __launch_bounds__(THREADS, 1)
    attend_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params p) {
  using Lay = Layout<HD>;
  using T = typename Elem<DT>::type;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* ks_s = reinterpret_cast<float*>(smem + Lay::KS);
  float* vf_s = reinterpret_cast<float*>(smem + Lay::VF);
  float* ref_s = reinterpret_cast<float*>(smem + Lay::REF);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Lay::BARS);
  uint64_t *kfull = bars, *kempty = bars + 2, *vfull = bars + 4, *vempty = bars + 6;  // by stage
  uint64_t *qfull = bars + 8, *sfull = bars + 10, *pfull = bars + 14;  // by half; sfull, pfull: and buffer
  uint64_t* obut = bars + 18;  // by half: a piece's products but the last step's
  uint64_t* drain = bars + 20;
  uint64_t *rkfull = bars + 21, *rkempty = bars + 22, *rvfull = bars + 23, *rvempty = bars + 24;
  uint64_t* ofull = bars + 25;  // by half: the last product of a piece
  __shared__ Piece first_s;
  __shared__ uint32_t holder;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int KV = p.c.heads, PL = p.page_log2;  // pages are powers of two

  if (tid == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(kfull + i, CONV_WARPS);
      mbar_init(kempty + i, 1);
      mbar_init(vfull + i, CONV_WARPS);
      mbar_init(vempty + i, 1);
      mbar_init(qfull + i, 4);
      mbar_init(obut + i, 1);
      mbar_init(ofull + i, 1);
    }
    for (int i = 0; i < 4; i++) {
      mbar_init(sfull + i, 1);
      mbar_init(pfull + i, 4);
    }
    mbar_init(drain, 1);
    mbar_init(rkfull, 1);
    mbar_init(rkempty, CONV_WARPS);
    mbar_init(rvfull, 1);
    mbar_init(rvempty, CONV_WARPS);
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

  if (warp == LOAD_WARP) {
    // ------------------------------------------------------------------------------------------------- loader
    // Lane l holds the page and scales of the block's 16-key piece l; a page's first piece brings it.
    constexpr int CHUNKS = BK / 16;
    const int ppp = 1 << (PL - 4), box = ::min(128, 1 << PL);  // pieces of a page, rows of a copy
    bool ok = true, gone = false;
    float ref = 0.0f;
    int it = 0, ik = 0, iv = 0;  // blocks; copies of keys and of values begun
    for (Blocks x(p, first); !x.done() && ok; x.next(p), it++) {
      const Tile& t = x.w.t;
      const int key0 = (t.blk0 + x.w.off + x.b) * BK, h = x.w.h;
      int pid = -1;
      float ks = 0.0f, vs = 0.0f;
      auto page_id = [&](int pg) {
        int id = __ldg(p.table + (size_t)t.s * p.max_pages + pg);
        if (id < 0 || id >= p.c.n_pages) {
          atomicCAS(p.status + 1, 0, VXG_DEV_CACHE_INDEX);
          id = -1;
        }
        return id;
      };
      if (x.b == 0) {  // the piece's largest value scale
        const int k0 = ::max(key0, t.kmin), k1 = ::min(key0 + x.nb * BK, t.kmax);
        ref = 0.0f;
        gone = false;
        for (int pg = (k0 >> PL) + lane; pg <= (k1 - 1) >> PL; pg += 32) {  // in pages: k1 + 32 pages may pass 31 bits
          const int id = page_id(pg);
          if (id >= 0) ref = fmaxf(ref, __ldg(p.c.v_scales + (size_t)id * KV + h));
          else gone = true;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, o));
        gone = __any_sync(0xffffffffu, gone);
      }
      const int pg = (key0 + 16 * ::min(lane, CHUNKS - 1)) >> PL;
      if (lane < CHUNKS && pg << PL < t.kmax && (pg + 1) << PL > t.kmin) {  // a page that some row sees
        pid = page_id(pg);
        if (pid >= 0) {
          ks = __ldg(p.c.k_scales + (size_t)pid * KV + h);
          vs = __ldg(p.c.v_scales + (size_t)pid * KV + h);
        } else {
          ks = NO_PAGE;
        }
      }
      const bool bring = pid >= 0 && lane % ppp == 0;
      const uint32_t bytes = (uint32_t)__popc(__ballot_sync(0xffffffffu, bring)) * box * HD;
      const int row = (pid * KV + h) << PL;
      if (it > 0 && !wait_phase(rkempty, (it - 1) & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane < CHUNKS) {
        ks_s[(it % RING) * 8 + lane] = ks;
        vf_s[(it % RING) * 8 + lane] = ref > 0.0f ? vs / ref : 0.0f;
      }
      if (lane == 8 && x.b == 0) ref_s[x.piece % RING] = gone ? -ref : ref;
      __syncwarp();
      if (lane == 0) mbar_arrive_expect_tx(rkfull, bytes);
      __syncwarp();
      if (bring) tma_load_2d(smem + Lay::RK + lane * 16 * HD, &map_k, 0, row, rkfull);
      ik++;
      if (it > 0 && !wait_phase(rvempty, (it - 1) & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(rvfull, bytes);
      __syncwarp();
      if (bring) tma_load_2d(smem + Lay::RV + lane * 16 * HD, &map_v, 0, row, rvfull);
      iv++;
    }
    // every copy lands before the block may end, after a wait that ran out as well
    if (ik > 0) wait_phase(rkfull, (ik - 1) & 1, p.status, VXG_DEV_TIMEOUT_DRAIN);
    if (iv > 0) wait_phase(rvfull, (iv - 1) & 1, p.status, VXG_DEV_TIMEOUT_DRAIN);
  } else if (warp >= SOFT_WARPS && warp < MMA_WARP) {
    // ---------------------------------------------------------------------------------------- codes -> operands
    // Eight lanes (16 codes each; four for 64 columns) take a key, a warp four (eight) keys a pass, all in one 16-key piece.
    constexpr int LPK = HD / 16, KPW = 32 / LPK, PASSES = BK / (CONV_WARPS * KPW);
    const int kk = (warp - SOFT_WARPS) * KPW + lane / LPK, ch = lane % LPK, e0 = ch * 16;
    const uint32_t swap = HD == 128 && e0 >= 64;
    auto get = [&](const uint8_t* raw, int k) {  // the copies' swizzle: 128-byte rows by row % 8, 64-byte rows by row / 2 % 4
      return *reinterpret_cast<const uint4*>(raw + k * HD + ((HD == 128 ? ch ^ (k & 7) : ch ^ ((k >> 1) & 3)) << 4));
    };
    // 16 codes -> two 16-byte chunks of the operand row; the upper half of the lanes of a key stores its odd chunk first,
    // so that the eight lanes of a store phase meet eight different chunks
    auto put = [&](uint8_t* dst, int k, uint4 x) {
      const uint32_t w[4] = {swap ? x.z : x.x, swap ? x.w : x.y, swap ? x.x : x.z, swap ? x.y : x.w};
      uint32_t h[8];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        h[2 * i] = codes_to_f16(__byte_perm(w[i], 0, 0x4140));
        h[2 * i + 1] = codes_to_f16(__byte_perm(w[i], 0, 0x4342));
      }
      uint8_t* base = dst + (e0 / 64) * Lay::HALF;
      const uint32_t c = (uint32_t)(e0 % 64) / 8;
      *reinterpret_cast<uint4*>(base + sw128_offset((uint32_t)k, c + swap)) = make_uint4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<uint4*>(base + sw128_offset((uint32_t)k, c + 1 - swap)) = make_uint4(h[4], h[5], h[6], h[7]);
    };
    bool ok = true;
    auto wait = [&](uint64_t* b, int phase) {
      if (ok && !wait_phase(b, (uint32_t)phase & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      return ok;
    };
    int it = 0;
    for (Blocks x(p, first); !x.done(); x.next(p), it++) {
      const int st = it & 1;
      if (it >= 2 && !wait(kempty + st, (it >> 1) - 1)) break;
      if (!wait(rkfull, it)) break;
      uint8_t* dk = smem + Lay::K + st * Lay::OPER;
#pragma unroll 2  // more would cost more in instruction fetches than it hides
      for (int i = 0; i < PASSES; i++) {
        const int k = i * CONV_WARPS * KPW + kk;
        put(dk, k, get(smem + Lay::RK, k));
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(kfull + st);
        mbar_arrive(rkempty);
      }
      if (it >= 2 && !wait(vempty + st, (it >> 1) - 1)) break;
      if (!wait(rvfull, it)) break;
      uint8_t* dv = smem + Lay::V + st * Lay::OPER;
#pragma unroll 2
      for (int i = 0; i < PASSES; i++) {
        const int k = i * CONV_WARPS * KPW + kk;
        put(dv, k, get(smem + Lay::RV, k));
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(vfull + st);
        mbar_arrive(rvempty);
      }
    }
  } else if (warp == MMA_WARP) {
    // --------------------------------------------------------------------------------------------- MMA issuer
    // The whole warp walks and waits, so that the operand descriptors stay in uniform registers, and one lane issues.
    // With one lane doing all of it, the descriptors' arithmetic took longer than the products.
    // A negative `scale` negates Q here, so that the softmax's factors are positive: a step's maximum is taken of unscaled
    // scores. Free here; negating Q where it is loaded was slower (4 x 2048 causal, 16 heads of 64: 208 us against 198).
    constexpr uint32_t PV = idesc_f16(128, HD, true);
    const uint32_t QK = idesc_f16(128, SB, false) | (p.negate ? 1u << 13 : 0u);  // negate A
    const bool leader = elect_one();
    // descriptor = fixed upper word, lower word = address / 16 and the offset between 64-column halves
    const uint64_t desc_k = umma_desc_sw128(smem_u32(smem)), desc_mn = umma_desc_sw128_mn(smem_u32(smem), Lay::HALF);
    bool ok = true;
    uint32_t nq0 = 0, nq1 = 0, n0 = 0, n1 = 0;  // by half: pieces begun, steps whose values are under way
    int it = 0;
    auto wait = [&](uint64_t* b, uint32_t phase) {
      if (ok && !wait_phase(b, phase & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (ok) tc_fence_after();
      return ok;
    };
    // step n of a half: 64 keys (`sub` of the operand stage), scores in buffer n % 2
    auto scores = [&](int half, uint32_t n, int st, int sub) {
      const uint32_t buf = n & 1, d = tmem + half * 128 + buf * SB;
      const uint64_t q = desc_k + (Lay::Q + half * Lay::OPER) / 16, k = desc_k + (Lay::K + st * Lay::OPER + sub * SB * 128) / 16;
      if (leader) {
#pragma unroll
        for (int c = 0; c < HD / 64; c++)
#pragma unroll
          for (int j = 0; j < 4; j++)
            mma_f16_ss(d, q + c * (Lay::HALF / 16) + 2 * j, k + c * (Lay::HALF / 16) + 2 * j, QK, (c | j) != 0 ? 1u : 0u);
        mma_commit(sfull + 2 * half + buf);
      }
      __syncwarp();
    };
    auto values = [&](int half, uint32_t n, int st, int sub, bool fresh, int left) {  // left: steps of the piece behind this
      const uint64_t v = desc_mn + (Lay::V + st * Lay::OPER + sub * SB * 128) / 16;
      if (leader) {
#pragma unroll
        for (int j = 0; j < SB / 16; j++)
          mma_f16_ts(tmem + 256 + half * HD, tmem + half * 128 + (n & 1) * SB + 8 * j, v + j * 128, PV, fresh && j == 0 ? 0u : 1u);
        if (left <= 1) mma_commit((left == 1 ? obut : ofull) + half);
      }
      __syncwarp();
    };
    auto commit = [&](uint64_t* b) {
      if (leader) mma_commit(b);
      __syncwarp();
    };
    for (Blocks x(p, first); !x.done() && ok;) {
      const bool two = x.w.t.rows > 128;  // else the second half has no rows and stays out
      const int nb = x.nb, ns = 2 * nb;
      if (!wait(qfull, nq0) || !wait(kfull + (it & 1), it >> 1)) break;
      for (int i = 0; i < 2; i++) scores(0, n0 + i, it & 1, i);
      nq0++;
      if (two) {
        if (!wait(qfull + 1, nq1)) break;
        for (int i = 0; i < 2; i++) scores(1, n1 + i, it & 1, i);
        nq1++;
      }
      commit(kempty + (it & 1));
      for (int i = 0; i < ns; i++) {
        const int st = it & 1, sub = i & 1;
        const bool more = i + 2 < ns;
        if (sub == 0 && !wait(vfull + st, it >> 1)) break;
        if (!wait(pfull + (n0 & 1), n0 >> 1)) break;
        values(0, n0, st, sub, i == 0, ns - 1 - i);
        if (more) {  // the step after next, over the probabilities that these products read
          if (sub == 0 && !wait(kfull + (st ^ 1), (it + 1) >> 1)) break;
          scores(0, n0 + 2, st ^ 1, sub);
        }
        n0++;
        if (two) {
          if (!wait(pfull + 2 + (n1 & 1), n1 >> 1)) break;
          values(1, n1, st, sub, i == 0, ns - 1 - i);
          if (more) scores(1, n1 + 2, st ^ 1, sub);
          n1++;
        }
        if (sub == 1) {
          commit(vempty + st);
          if (more) commit(kempty + (st ^ 1));
          it++;
          x.next(p);
        }
      }
    }
    commit(drain);  // nothing is in flight when the block ends
    wait_phase(drain, 0, p.status, VXG_DEV_TIMEOUT_DRAIN);
  } else {
    // ------------------------------------------------------------------------------------------------ softmax
    const int half = warp >> 2, r = half * 128 + (warp & 3) * 32 + lane;  // the thread's row of the tile
    constexpr int LPR = HD / 8, RPI = 32 / LPR;  // lanes a row and rows an access where a warp moves rows as wholes
    const int wrow = (warp & 3) * 32;            // the warp's first row of its half
    const uint32_t lanes = (uint32_t)wrow << 16;
    const uint32_t S0 = tmem + lanes + half * 128, O = tmem + lanes + 256 + half * HD;
    bool ok = true;
    uint32_t it = 0, pieces = 0;         // steps and pieces of this half so far
    uint32_t ring = 0, ring_piece = 0;   // blocks and pieces with keys of the CTA so far
    for (Piece w = first; w.left > 0 && ok; w.next(p, MT, BK)) {
      const Tile& t = w.t;
      if (half * 128 >= t.rows) {
        if (t.nblk > 0) ring += w.take(), ring_piece++;
        continue;
      }
      const int take = w.take(), nb = t.nblk > 0 ? take : 0;
      const bool live = r < t.rows;
      const int rr = t.r0 + (live ? r : 0), i = rr / p.share, head = w.h * p.share + rr % p.share;
      const long long pos = (long long)t.L - t.n + i;
      const int khi = p.causal ? (int)::max(0LL, ::min((long long)t.L, pos + 1)) : t.L;
      const int klo = p.window > 0 ? (int)::max(0LL, pos - p.window + 1) : 0;
      float m = -INFINITY, l = 0.0f, ref = 0.0f;
      if (nb > 0) {
        // ---- the warp's rows of Q: each scaled by a power of two, f16, into the half's operand. LPR lanes read a row.
        const long long qoff = live ? (long long)(t.q0 + i) * p.ld_q + (long long)head * HD : -1;
        uint8_t* qs = smem + Lay::Q + half * Lay::OPER;
        int ex = 0;  // of this thread's own row
#pragma unroll 1
        for (int n0 = 0; n0 < LPR; n0 += 8) {
          uint4 raw[8];
#pragma unroll
          for (int n = 0; n < 8; n++) {
            const long long o = __shfl_sync(0xffffffffu, qoff, (n0 + n) * RPI + lane / LPR);
            raw[n] = make_uint4(0, 0, 0, 0);
            if (o >= 0) raw[n] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + o + lane % LPR * 8);
          }
#pragma unroll
          for (int n = 0; n < 8; n++) {
            const uint32_t x[4] = {raw[n].x, raw[n].y, raw[n].z, raw[n].w};
            float2 f[4];
            float top = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++) {
              f[k] = widen2<DT>(x[k]);
              top = max3(top, fabsf(f[k].x), fabsf(f[k].y));
            }
#pragma unroll
            for (int o = 1; o < LPR; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            int e = 14 - ((int)(__float_as_uint(top) >> 23) - 127);
            e = top == 0.0f || !(top <= 3.402823466e38f) ? 0 : ::min(e, 126);
            const int got = __shfl_sync(0xffffffffu, e, lane % RPI * LPR);
            if (lane / RPI == n0 + n) ex = got;
            const float up = __int_as_float((e + 127) << 23);
            uint32_t h[4];
#pragma unroll
            for (int k = 0; k < 4; k++) h[k] = pack_f16(f[k].x * up, f[k].y * up);
            const int c = lane % LPR;
            *reinterpret_cast<uint4*>(qs + (c / 8) * Lay::HALF +
                                      sw128_offset((uint32_t)(wrow + (n0 + n) * RPI + lane / LPR), (uint32_t)(c % 8))) =
                make_uint4(h[0], h[1], h[2], h[3]);
          }
        }
        // not 0, which NO_PAGE would turn into NaN; below f32's range the scores are alike in any case
        const float rowf = fmaxf(__int_as_float((127 - ex) << 23) * p.scale_log2, 1.4e-45f);
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(qfull + half);
        // keys that every row of the warp sees: [all_lo, all_hi)
        const int all_hi = __reduce_min_sync(0xffffffffu, live ? khi : 0x7FFFFFFF);
        const int all_lo = __reduce_max_sync(0xffffffffu, live ? klo : 0);

        for (int b = 0; b < 2 * nb; b++, it++) {
          const uint32_t buf = it & 1, S = S0 + buf * SB;
          if (ok && !wait_phase(sfull + 2 * half + buf, (it >> 1) & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN)) ok = false;
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const int key0 = (t.blk0 + w.off) * BK + b * SB;
          const bool inside = key0 >= all_lo && key0 + SB <= all_hi;
          const int scales = ((ring + b / 2) % RING) * 8 + (b & 1) * (SB / 16);
          const float *ks = ks_s + scales, *vf = vf_s + scales;
          if (b == 0) ref = ref_s[ring_piece % RING];
          if (__float_as_int(ref) < 0) {  // scores that NO_PAGE takes to -inf, whatever the query
#pragma unroll 1
            for (int g = 0; g < SB / 16; g++)
              if (ks[g] == NO_PAGE) tmem_st16_const(S + 16 * g, __float_as_uint(INFINITY));
            tmem_wait_st();
          }
          // ---- the step's maximum
          float mx = -INFINITY;
          auto maximum = [&](auto tag) {
            constexpr bool masked = decltype(tag)::value;
            uint32_t a[2][32];
            tmem_ld32(S, a[0]);
            tmem_ld32(S + 32, a[1]);
            tmem_wait_ld();
#pragma unroll
            for (int g = 0; g < 4; g++) {
              const uint32_t* v = a[g >> 1] + 16 * (g & 1);
              float y[16];
#pragma unroll
              for (int j = 0; j < 16; j++) {
                y[j] = __uint_as_float(v[j]);
                const int key = key0 + 16 * g + j;
                if (masked && (key < klo || key >= khi)) y[j] = -INFINITY;
              }
              float x = max3(y[0], y[1], y[2]), z = max3(y[3], y[4], y[5]);
              x = max3(x, y[6], y[7]), z = max3(z, y[8], y[9]);
              x = max3(x, y[10], y[11]), z = max3(z, y[12], y[13]);
              x = max3(x, y[14], y[15]), x = fmaxf(x, z);
              // -inf x 0 would be NaN: a piece without a visible key has no maximum
              const float f = rowf * ks[g];
              mx = fmaxf(mx, masked && x == -INFINITY ? x : x * f);
            }
          };
          if (inside) maximum(std::false_type());
          else maximum(std::true_type());
          // ---- move the reference when the maximum has outgrown it
          const bool grow = mx > m + 8.0f;
          if (__any_sync(0xffffffffu, grow)) {
            const float alpha = grow ? ex2(m - mx) : 1.0f;
            if (grow) m = mx;
            l *= alpha;
            if (b > 0) {  // once the products of the step before are in O: the next step's scores come behind them
              const bool more = b + 1 < 2 * nb;
              uint64_t* bar = more ? sfull + 2 * half + (buf ^ 1) : obut + half;
              if (!wait_phase(bar, (more ? (it + 1) >> 1 : pieces) & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN)) ok = false;
              ok = __all_sync(0xffffffffu, ok);
              if (!ok) break;
              tc_fence_after();
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
          // ---- probabilities over the scores: 32 scores are read before their 16 columns are written
          uint64_t sum[4] = {0, 0, 0, 0};  // eight partial sums of the step
          auto exponentials = [&](auto tag) {
            constexpr bool masked = decltype(tag)::value;
            const uint64_t mm2 = pk2(-mm, -mm);
            uint32_t a[32];
            tmem_ld32(S, a);
#pragma unroll 1
            for (int c = 0; c < SB; c += 32) {
              uint64_t x[16];
              const float f0 = rowf * ks[c / 16], f1 = rowf * ks[c / 16 + 1], g0 = vf[c / 16], g1 = vf[c / 16 + 1];
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; j++) {
                const float f = j < 8 ? f0 : f1;
                x[j] = ffma2(pk2(__uint_as_float(a[2 * j]), __uint_as_float(a[2 * j + 1])), pk2(f, f), mm2);
              }
              if (c + 32 < SB) tmem_ld32(S + c + 32, a);  // under this chunk's exponentials
              uint32_t o[16];
#pragma unroll
              for (int j = 0; j < 16; j++) {
                float x0, x1;
                upk2(x[j], x0, x1);
                if (masked) {
                  const int key = key0 + c + 2 * j;
                  if (key < klo || key >= khi) x0 = -INFINITY;
                  if (key + 1 < klo || key + 1 >= khi) x1 = -INFINITY;
                }
                const float p0 = ex2(x0), p1 = ex2(x1);
                sum[j & 3] = fadd2(sum[j & 3], pk2(p0, p1));
                float y0, y1;
                upk2(fmul2(pk2(p0, p1), j < 8 ? pk2(g0, g0) : pk2(g1, g1)), y0, y1);
                o[j] = pack_f16(y0, y1);
              }
              tmem_st16(S + c / 2, o);
            }
          };
          if (inside) exponentials(std::false_type());
          else exponentials(std::true_type());
          float l0, l1;
          upk2(fadd2(fadd2(sum[0], sum[1]), fadd2(sum[2], sum[3])), l0, l1);
          l += l0 + l1;
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(pfull + 2 * half + buf);
        }
        ring += nb;
        // Every phase of every barrier is met once and in turn, obut's too where no reference has moved in the last step: a
        // wait by parity is right only if the phase before was met, and commits to two barriers have no order that PTX states.
        if (ok && !wait_phase(obut + half, pieces & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN)) ok = false;
        if (ok && !wait_phase(ofull + half, pieces & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        ring_piece++, pieces++;
      }
      // ---- the row's result, whole or for the join
      const bool whole = w.off == 0 && take == t.cost;
      float* part = p.part + ((size_t)blockIdx.x * MAX_PIECES + (w.first ? 0 : 1)) * MT * (HD + 2) + (size_t)r * (HD + 2);
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // ref last: their product may be too small for f32's digits
      if (live && !whole) part[0] = m - 7.0f, part[1] = l;
      uint8_t* os = smem + Lay::Q + half * Lay::OPER;  // the half's products are done with Q
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
        if (whole) {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint32_t h[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
              const float v0 = __uint_as_float(a[j + 2 * k]) * inv * fabsf(ref), v1 = __uint_as_float(a[j + 2 * k + 1]) * inv * fabsf(ref);
              h[k] = narrow2<DT>(l == 0.0f ? 0.0f : v0, l == 0.0f ? 0.0f : v1);
            }
            *reinterpret_cast<uint4*>(os + (c / 64) * Lay::HALF +
                                      sw128_offset((uint32_t)(wrow + lane), (uint32_t)((c % 64 + j) / 8))) =
                make_uint4(h[0], h[1], h[2], h[3]);
          }
        } else if (live) {
#pragma unroll
          for (int j = 0; j < 32; j += 2)
            *reinterpret_cast<float2*>(part + 2 + c + j) =
                make_float2(__uint_as_float(a[j]) * fabsf(ref), __uint_as_float(a[j + 1]) * fabsf(ref));
        }
        __syncwarp();
      }
      if (whole) {
        const long long ooff = live ? (long long)(t.q0 + i) * p.ld_out + (long long)head * HD : -1;
#pragma unroll 4
        for (int n = 0; n < LPR; n++) {
          const int row = n * RPI + lane / LPR, c = lane % LPR;
          const long long o = __shfl_sync(0xffffffffu, ooff, row);
          const uint4 v = *reinterpret_cast<const uint4*>(os + (c / 8) * Lay::HALF +
                                                          sw128_offset((uint32_t)(wrow + row), (uint32_t)(c % 8)));
          if (o >= 0) *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + o + c * 8) = v;
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
  CUtensorMap mk, mv;
  vxg_status r = smem_attr((const void*)attend_tc_kernel<HD, DT>, smem);
  if (r == VXG_OK) r = cache_map(&mk, p.c, p.c.k, 128);
  if (r == VXG_OK) r = cache_map(&mv, p.c, p.c.v, 128);
  if (r != VXG_OK) return r;
  attend_tc_kernel<HD, DT><<<pl.grid, THREADS, smem, st>>>(mk, mv, p);
  VXG_CUDA(cudaGetLastError());
  return launch_join<HD, DT, MT, BK>(p, pl, st);
}

}  // namespace tc

vxg_status launch_tc(Params p, const Plan& pl, int head_dim, int dtype, cudaStream_t st) {
  p.negate = p.scale_log2 < 0.0f;
  p.scale_log2 = std::fabs(p.scale_log2);
  if (head_dim == 128)
    return dtype == VXG_DT_BF16 ? tc::launch<128, VXG_DT_BF16>(p, pl, st) : tc::launch<128, VXG_DT_F16>(p, pl, st);
  return dtype == VXG_DT_BF16 ? tc::launch<64, VXG_DT_BF16>(p, pl, st) : tc::launch<64, VXG_DT_F16>(p, pl, st);
}

}  // namespace catt
}  // namespace vxg
