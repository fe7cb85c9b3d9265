// Attention of new queries over the paged int8 cache:
//   out = sum_j softmax_j(scale * q . k_j) v_j,  k_j = code * k_scale[page], v_j = code * v_scale[page],
// for query i of n of a sequence of length L at position p = L - n + i: keys j < L, j <= p (causal), j > p - window.
// A query with no key gives 0.
//
// Arithmetic. Codes are exact in f16, so both products run on mma.m16n8k16 with f16 operands and f32 sums. A query row
// is scaled by a power of two so that its largest element lies in [2^14, 2^15): bf16 and f16 queries are then exact
// down to 2^-29 of that element; f32 queries are split into two f16 parts (22 bits). The page's key scale, the row's
// power of two, `scale` and log2(e) multiply the f32 sum. The softmax is kept in f32 with a running maximum and sum;
// a probability enters the second product as f16(p * 2^14 * v_scale / ref), ref being the largest value scale met so
// far (rounding 2^-11 of each term at most, 2^-39 absolute against the largest; two parts for f32), and ref and 2^-14 multiply
// the result. The sum of the row is taken from the unrounded p.
//
// Work split. A tile is MT consecutive (query, query head) rows of one sequence and KV head, so a key is read once for
// all the query heads that share it. The keys it sees, in blocks of 64, times all tiles and KV heads form one line of
// work units that is cut into equal shares, one a CTA: a CTA works off its share tile by tile, and a tile that spans
// shares leaves partial results (maximum, sum, unnormalised row) that a second small kernel joins. Lengths are read on
// the device, so the launch does not depend on them and can be captured; every CTA finds its share with one scan.
//   few rows  (MT = 16): the four consumer warps take 16 keys of each block and meet at the end of a tile's share;
//   many rows (MT = 64): each consumer warp takes 16 rows and all 64 keys.
// A fifth warp brings the codes by TMA (one box per page, 128- or 64-byte swizzle so that the operand reads below are
// free of bank conflicts) and the scales into a ring of stages. Operand layout: the k slots of a step are permuted so
// that a thread's operand words are consecutive codes (keys: of one key; values: one word of four keys, transposed by
// byte permutes), and the result's columns come out as consecutive runs a thread.
#include <cuda_runtime.h>

#include <algorithm>

#include "common.h"
#include "cached_attention.cuh"

namespace vxg {
namespace catt {

constexpr int BK = 64;       // keys per block
constexpr int CONS = 4;      // consumer warps
constexpr int THREADS = (CONS + 1) * 32;
template <int HD, int MT>
struct Layout {
  static constexpr uint32_t TILE = BK * HD;      // bytes of one block's keys or values
  static constexpr uint32_t STAGE = 2 * TILE;
  static constexpr int STAGES = HD == 128 ? (MT == 16 ? 4 : 5) : 8;
  static constexpr uint32_t SCALES = STAGES * STAGE;           // [stage][K 4, V 4] f32
  static constexpr uint32_t MERGE = SCALES + STAGES * 32;      // few rows: [CONS][16][HD + 4] f32 and (max, sum)
  static constexpr uint32_t MERGE_BYTES = MT == 16 ? CONS * 16 * (HD + 4) * 4 : 0;
  static constexpr uint32_t STAT = MERGE + MERGE_BYTES;        // [CONS][16][2] f32
  static constexpr uint32_t BARS = (STAT + (MT == 16 ? CONS * 16 * 8 : 0) + 15) / 16 * 16;
  static constexpr uint32_t BYTES = BARS + 2 * STAGES * 8 + 1024;  // + alignment
};

// Running softmax state of a warp's 16 rows: thread (g, c) holds rows g and g + 8.
template <int HD>
struct State {
  float o[HD / 8][4];
  float m[2], l[2];
  float ref;
};

template <int HD, int DT, int MT>
__global__ void __launch_bounds__(THREADS, 2)
    attend_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params p) {
  using Lay = Layout<HD, MT>;
  using T = typename Elem<DT>::type;
  constexpr bool SPLIT = DT == VXG_DT_F32;
  constexpr bool FEW = MT == 16;
  constexpr int TOK = FEW ? 16 : 64;  // keys of a block that one warp takes
  constexpr int KS = HD / 16;         // k steps of the first product
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* scales_s = reinterpret_cast<float*>(smem + Lay::SCALES);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Lay::BARS);
  uint64_t* empty = full + Lay::STAGES;
  __shared__ Piece first_s;  // the share's first piece
  __shared__ Piece piece_s;  // few rows: the consumers' next one
  __shared__ int fail;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int KV = p.c.heads, PL = p.page_log2, P = 1 << PL;  // pages are powers of two

  if (tid == 0) {
    for (int i = 0; i < Lay::STAGES; i++) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, CONS);
    }
    fence_mbar_init();
    fail = 0;
  }

  find_share<THREADS, MT, BK>(p, &first_s);
  Piece w = first_s;
  if (w.left == 0) return;

  if (warp == CONS) {
    // ------------------------------------------------------------------------------------------------ producer
    const int box = ::min(P, BK);
    int it = 0;
    bool ok = true;
    for (; w.left > 0 && ok; w.next(p, MT, BK)) {
      const Tile& t = w.t;
      const int take = w.take(), h = w.h, off = w.off;
      if (t.nblk > 0) {
        int have = -1;  // first page of the 32 that the lanes hold
        int pid = -1;
        float ks = 0.0f, vs = 0.0f;
        for (int b = t.blk0 + off; b < t.blk0 + off + take; b++, it++) {
          const int pg0 = (b * BK) >> PL, npg = BK > P ? BK >> PL : 1;
          if (have < 0 || pg0 + npg > have + 32) {
            have = pg0;
            const int pg = pg0 + lane;
            pid = -1, ks = 0.0f, vs = 0.0f;
            if ((long long)pg * P < t.kmax && (long long)(pg + 1) * P > t.kmin) {  // a page that some row sees
              pid = __ldg(p.table + (size_t)t.s * p.max_pages + pg);
              if (pid < 0 || pid >= p.c.n_pages) {
                atomicCAS(p.status + 1, 0, VXG_DEV_CACHE_INDEX);
                pid = -1;
              } else {
                ks = __ldg(p.c.k_scales + (size_t)pid * KV + h);
                vs = __ldg(p.c.v_scales + (size_t)pid * KV + h);
              }
            }
          }
          const int st = it % Lay::STAGES;
          if (it >= Lay::STAGES && !wait_phase(empty + st, ((it / Lay::STAGES) - 1) & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN))
            ok = false;
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const int src = pg0 - have + ((lane & 3) * 16 >> PL);  // page of the block's 16-key piece lane & 3
          const float a = __shfl_sync(0xffffffffu, ks, src & 31), v = __shfl_sync(0xffffffffu, vs, src & 31);
          if (lane < 8) scales_s[st * 8 + lane] = lane < 4 ? a : v;
          const unsigned valid = __ballot_sync(0xffffffffu, pid >= 0);
          const unsigned span = npg == 32 ? ~0u : ((1u << npg) - 1u);
          const unsigned bring = (valid >> (pg0 - have)) & span;
          __syncwarp();
          if (lane == 0) mbar_arrive_expect_tx(full + st, (uint32_t)__popc(bring) * box * HD * 2);
          __syncwarp();
          const int mypage = lane - (pg0 - have);
          if (mypage >= 0 && mypage < npg && pid >= 0) {
            const int row = (int)(((long long)pid * KV + h) * P) + ((b * BK) & (P - 1));
            uint8_t* dst = smem + st * Lay::STAGE + mypage * box * HD;
            tma_load_2d(dst, &map_k, 0, row, full + st);
            tma_load_2d(dst + Lay::TILE, &map_v, 0, row, full + st);
          }
        }
      }
    }
    // every copy that was issued lands before the block may end
    const int last = ::min(it, (int)Lay::STAGES);
    for (int i = it - last; i < it; i++)
      wait_phase(full + i % Lay::STAGES, (i / Lay::STAGES) & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN);
    return;
  }

  // -------------------------------------------------------------------------------------------------- consumers
  const int g = lane >> 2, c = lane & 3;
  int it = 0;
  bool ok = true;
  while (w.left > 0) {
    const Tile& t = w.t;
    const int take = w.take(), h = w.h, off = w.off;
    const int row0 = FEW ? 0 : warp * 16;  // this warp's rows of the tile
    // this thread's two rows: operand fragments, limits, power of two
    uint32_t qa[KS][4], qb[SPLIT ? KS : 1][4];
    float rowf[2];
    int klo[2], khi[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int r = row0 + g + 8 * e;
      const bool live = r < t.rows;
      const int rr = t.r0 + (live ? r : 0), i = rr / p.share, head = h * p.share + rr % p.share;
      const long long pos = (long long)t.L - t.n + i;
      khi[e] = !live ? 0 : p.causal ? (int)::max(0LL, ::min((long long)t.L, pos + 1)) : t.L;
      klo[e] = p.window > 0 ? (int)::max(0LL, pos - p.window + 1) : 0;
      const T* q = static_cast<const T*>(p.q) + (long long)(t.q0 + i) * p.ld_q + (long long)head * HD + c * (HD / 4);
      float f[HD / 4];
      float top = 0.0f;
#pragma unroll
      for (int d = 0; d < HD / 4; d += 8) {
        float v8[8];
        if (live) {
          load8<DT>(q + d, v8);
        } else {
#pragma unroll
          for (int k = 0; k < 8; k++) v8[k] = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < 8; k++) f[d + k] = v8[k], top = fmaxf(top, fabsf(v8[k]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^(14 - exponent of the largest), within f32's range; 1 for a row that is zero or holds an infinity
      int ex = 14 - ((int)(__float_as_uint(top) >> 23) - 127);
      ex = top == 0.0f || !(top <= 3.402823466e38f) ? 0 : ::min(ex, 126);
      const float up = __int_as_float((ex + 127) << 23);
      rowf[e] = __int_as_float((127 - ex) << 23) * p.scale_log2;
#pragma unroll
      for (int w = 0; w < KS; w++) {
        const float x0 = f[4 * w] * up, x1 = f[4 * w + 1] * up, x2 = f[4 * w + 2] * up, x3 = f[4 * w + 3] * up;
        qa[w][e] = pack_f16(x0, x1);
        qa[w][2 + e] = pack_f16(x2, x3);
        if (SPLIT) {
          qb[w][e] = pack_rest(x0, x1, qa[w][e]);
          qb[w][2 + e] = pack_rest(x2, x3, qa[w][2 + e]);
        }
      }
    }
    // keys that every live row of the tile sees: [all_lo, all_hi)
    const int last_i = (t.r0 + t.rows - 1) / p.share, first_i = t.r0 / p.share;
    const long long all_hi = p.causal ? (long long)t.L - t.n + first_i + 1 : t.L;
    const long long all_lo = p.window > 0 ? (long long)t.L - t.n + last_i - p.window + 1 : 0;

    State<HD> S;
#pragma unroll
    for (int j = 0; j < HD / 8; j++)
#pragma unroll
      for (int k = 0; k < 4; k++) S.o[j][k] = 0.0f;
    S.m[0] = S.m[1] = -INFINITY;
    S.l[0] = S.l[1] = 0.0f;
    S.ref = 0.0f;

    const int nb = t.nblk > 0 ? take : 0;
    for (int b = 0; b < nb; b++, it++) {
      const int st = it % Lay::STAGES;
      if (ok && !wait_phase(full + st, (it / Lay::STAGES) & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const uint8_t* kt = smem + st * Lay::STAGE;
      const uint8_t* vt = kt + Lay::TILE;
      const int key0 = (t.blk0 + off + b) * BK;
      const int tok0 = FEW ? warp * 16 : 0;  // this warp's keys of the block
      // ---- scores
      float s[TOK / 8][4];
#pragma unroll
      for (int j = 0; j < TOK / 8; j++) {
#pragma unroll
        for (int k = 0; k < 4; k++) s[j][k] = 0.0f;
        const int r = tok0 + 8 * j + g;
        uint32_t w[HD / 16];
        if (HD == 128) {
#pragma unroll
          for (int k = 0; k < 2; k++) {
            const uint4 x = *reinterpret_cast<const uint4*>(kt + r * 128 + (((2 * c + k) ^ (r & 7)) << 4));
            w[4 * k] = x.x, w[4 * k + 1] = x.y, w[4 * k + 2] = x.z, w[4 * k + 3] = x.w;
          }
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(kt + r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
          w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
        }
#pragma unroll
        for (int k = 0; k < KS; k++) {
          const uint32_t b0 = codes_to_f16(__byte_perm(w[k], 0, 0x4140)), b1 = codes_to_f16(__byte_perm(w[k], 0, 0x4342));
          mma_f16(s[j], qa[k], b0, b1);
          if (SPLIT) mma_f16(s[j], qb[k], b0, b1);
        }
      }
      // ---- scale, mask, running maximum
      const bool inside = key0 >= all_lo && key0 + BK <= all_hi;
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < TOK / 8; j++) {
        const float ks = scales_s[st * 8 + (tok0 + 8 * j) / 16];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          float x = s[j][k] * (rowf[k >> 1] * ks);
          if (!inside) {
            const int key = key0 + tok0 + 8 * j + 2 * c + (k & 1);
            if (key < klo[k >> 1] || key >= khi[k >> 1]) x = -INFINITY;
          }
          s[j][k] = x;
          mx[k >> 1] = fmaxf(mx[k >> 1], x);
        }
      }
      float vsm = 0.0f;
#pragma unroll
      for (int j = 0; j < TOK / 16; j++) vsm = fmaxf(vsm, scales_s[st * 8 + 4 + tok0 / 16 + j]);
      const float ref = fmaxf(S.ref, vsm);
      const float reff = S.ref == ref ? 1.0f : S.ref / ref;
      float alpha[2], mu[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
        const float m = fmaxf(S.m[e], mx[e]);
        mu[e] = m == -INFINITY ? 0.0f : m;
        alpha[e] = ex2(S.m[e] - mu[e]);
        S.m[e] = m;
        S.l[e] *= alpha[e];
        alpha[e] *= reff;
      }
      S.ref = ref;
      if (!__all_sync(0xffffffffu, alpha[0] == 1.0f && alpha[1] == 1.0f)) {
#pragma unroll
        for (int j = 0; j < HD / 8; j++)
#pragma unroll
          for (int k = 0; k < 4; k++) S.o[j][k] *= alpha[k >> 1];
      }
      // ---- probabilities and the second product, 16 keys a step
#pragma unroll
      for (int kk = 0; kk < TOK / 16; kk++) {
        const float vf = ref > 0.0f ? scales_s[st * 8 + 4 + tok0 / 16 + kk] / ref * 16384.0f : 0.0f;
        uint32_t pa[4], pb[4];
#pragma unroll
        for (int e = 0; e < 2; e++)  // key group 2 kk + e
#pragma unroll
          for (int r = 0; r < 2; r++) {
            const float p0 = ex2(s[2 * kk + e][2 * r] - mu[r]), p1 = ex2(s[2 * kk + e][2 * r + 1] - mu[r]);
            S.l[r] += p0 + p1;
            pa[2 * e + r] = pack_f16(p0 * vf, p1 * vf);
            if (SPLIT) pb[2 * e + r] = pack_rest(p0 * vf, p1 * vf, pa[2 * e + r]);
          }
        const int r0 = tok0 + 16 * kk + 2 * c;
        constexpr int W = HD / 32;  // words of a key that a thread takes
        uint32_t x[4][W];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int r = r0 + (k & 1) + 8 * (k >> 1);
          if (HD == 128) {
            const uint4 y = *reinterpret_cast<const uint4*>(vt + r * 128 + ((g ^ (r & 7)) << 4));
            x[k][0] = y.x, x[k][1] = y.y, x[k][W - 2] = y.z, x[k][W - 1] = y.w;
          } else {
            const uint2 y = *reinterpret_cast<const uint2*>(vt + r * 64 + (((g >> 1) ^ ((r >> 1) & 3)) << 4) + (g & 1) * 8);
            x[k][0] = y.x, x[k][1] = y.y;
          }
        }
#pragma unroll
        for (int w = 0; w < W; w++)
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const uint32_t sel = k | (k << 4) | ((4 + k) << 8) | ((4 + k) << 12);
            const uint32_t b0 = codes_to_f16(__byte_perm(x[0][w], x[1][w], sel));
            const uint32_t b1 = codes_to_f16(__byte_perm(x[2][w], x[3][w], sel));
            mma_f16(S.o[4 * w + k], pa, b0, b1);
            if (SPLIT) mma_f16(S.o[4 * w + k], pb, b0, b1);
          }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + st);
    }
    if (!ok) {
      // give up together: no block barrier is left hanging
      if (lane == 0) fail = 1;
    }
#pragma unroll
    for (int e = 0; e < 2; e++) {
      S.l[e] += __shfl_xor_sync(0xffffffffu, S.l[e], 1);
      S.l[e] += __shfl_xor_sync(0xffffffffu, S.l[e], 2);
    }
    const float unit = S.ref * (1.0f / 16384.0f);
    const bool whole = off == 0 && take == t.cost;
    float* part = p.part + ((size_t)blockIdx.x * MAX_PIECES + (w.first ? 0 : 1)) * MT * (HD + 2);
    // thread (g, c)'s columns: HD / 4 consecutive ones, the first HD / 8 in o[.][0 or 2], the rest in o[.][1 or 3]
    if (FEW) {
      float* mo = reinterpret_cast<float*>(smem + Lay::MERGE);
      float* ms = reinterpret_cast<float*>(smem + Lay::STAT);
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float* row = mo + (warp * 16 + g + 8 * e) * (HD + 4) + c * (HD / 4);
#pragma unroll
        for (int j = 0; j < HD / 8; j++) {
          row[j] = S.o[j][2 * e] * unit;
          row[HD / 8 + j] = S.o[j][2 * e + 1] * unit;
        }
        if (c == 0) {
          ms[(warp * 16 + g + 8 * e) * 2] = S.m[e];
          ms[(warp * 16 + g + 8 * e) * 2 + 1] = S.l[e];
        }
      }
      named_bar_sync(1, CONS * 32);
      if (tid == 0) {  // one thread walks on for all of them, so that they always agree on the barriers to come
        Piece n = w;
        n.next(p, MT, BK);
        piece_s = n;
      }
      for (int r = warp; r < t.rows; r += CONS) {
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < CONS; w++) m = fmaxf(m, ms[(w * 16 + r) * 2]);
        const float mu = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, acc[HD / 32] = {};
#pragma unroll
        for (int w = 0; w < CONS; w++) {
          const float f = ex2(ms[(w * 16 + r) * 2] - mu);
          l += f * ms[(w * 16 + r) * 2 + 1];
#pragma unroll
          for (int k = 0; k < HD / 32; k++) acc[k] += f * mo[(w * 16 + r) * (HD + 4) + 32 * k + lane];
        }
        if (whole) {
          const int rr = t.r0 + r;
          T* o = static_cast<T*>(p.out) + (long long)(t.q0 + rr / p.share) * p.ld_out +
                 (long long)(h * p.share + rr % p.share) * HD;
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
          for (int k = 0; k < HD / 32; k++) o[32 * k + lane] = Elem<DT>::narrow(acc[k] * inv);
        } else {
          float* o = part + r * (HD + 2);
          if (lane == 0) o[0] = m, o[1] = l;
#pragma unroll
          for (int k = 0; k < HD / 32; k++) o[2 + 32 * k + lane] = acc[k];
        }
      }
      named_bar_sync(1, CONS * 32);  // the buffers are free for the next piece
    } else {
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int r = row0 + g + 8 * e;
        if (r >= t.rows) continue;
        if (whole) {
          const int rr = t.r0 + r;
          T* o = static_cast<T*>(p.out) + (long long)(t.q0 + rr / p.share) * p.ld_out +
                 (long long)(h * p.share + rr % p.share) * HD + c * (HD / 4);
          const float inv = S.l[e] == 0.0f ? 0.0f : unit / S.l[e];
#pragma unroll
          for (int j = 0; j < HD / 8; j += 8) {
            float a[8], b2[8];
#pragma unroll
            for (int k = 0; k < 8; k++) a[k] = S.o[j + k][2 * e] * inv, b2[k] = S.o[j + k][2 * e + 1] * inv;
            store8<DT>(o + j, a);
            store8<DT>(o + HD / 8 + j, b2);
          }
        } else {
          float* o = part + r * (HD + 2);
          if (c == 0) o[0] = S.m[e], o[1] = S.l[e];
          o += 2 + c * (HD / 4);
#pragma unroll
          for (int j = 0; j < HD / 8; j++) {
            o[j] = S.o[j][2 * e] * unit;
            o[HD / 8 + j] = S.o[j][2 * e + 1] * unit;
          }
        }
      }
    }
    if (FEW) {
      if (fail) return;  // set before the first of the two barriers above
      w = piece_s;
    } else {
      if (!ok) return;
      w.next(p, MT, BK);
    }
  }
}

constexpr int CTAS_PER_SM = 2;

// The three kernels by the average number of (query, query head) rows a sequence and KV head has: up to 16 rows, tiles of
// 16; up to 96, tiles of 64; beyond, tiles of 256 on tcgen05 (16-bit queries).
static vxg_status plan(int total, int n_seq, int heads, int kv, int hd, int dtype, Plan* pl) {
  const long long share = heads / kv, rows = (long long)total * share;
  pl->mt = rows <= 16LL * n_seq ? 16 : rows <= 96LL * n_seq || dtype == VXG_DT_F32 ? 64 : 256;
  const long long slots = rows / pl->mt + n_seq;
  if (slots > 0x3FFFFFFF) {
    set_error("%d rows of %d heads are more than one launch covers", total, heads);
    return VXG_ERR_UNSUPPORTED;
  }
  pl->slots = (int)slots;
  pl->grid = sm_count() * (pl->mt == 256 ? 1 : CTAS_PER_SM);
  pl->rec_bytes = (size_t)pl->grid * 8 * sizeof(long long);
  pl->part_bytes = (size_t)pl->grid * MAX_PIECES * pl->mt * (hd + 2) * sizeof(float);
  return VXG_OK;
}

template <int HD, int DT, int MT>
vxg_status launch(const Params& p, const Plan& pl, cudaStream_t st) {
  CUtensorMap mk, mv;
  vxg_status r = cache_map(&mk, p.c, p.c.k, BK);
  if (r == VXG_OK) r = cache_map(&mv, p.c, p.c.v, BK);
  if (r != VXG_OK) return r;
  constexpr int smem = (int)Layout<HD, MT>::BYTES;
  static_assert((smem + 1024) * CTAS_PER_SM <= 228 * 1024, "two blocks share an SM");
  if ((r = smem_attr((const void*)attend_kernel<HD, DT, MT>, smem)) != VXG_OK) return r;
  attend_kernel<HD, DT, MT><<<pl.grid, THREADS, smem, st>>>(mk, mv, p);
  VXG_CUDA(cudaGetLastError());
  join_kernel<HD, DT, MT, BK><<<dim3(pl.grid - 1, MT / 4), 128, 0, st>>>(p);
  note_launch(2);
  VXG_CUDA(cudaGetLastError());
  return VXG_OK;
}

}  // namespace catt
}  // namespace vxg

using namespace vxg;

extern "C" {

size_t vxg_cache_attention_workspace_bytes(int total, int n_seq, int heads, int kv_heads, int head_dim, int dtype) {
  catt::Plan pl;
  if (total <= 0 || n_seq <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || head_dim <= 0 || !dtype_known(dtype))
    return 0;
  if (catt::plan(total, n_seq, heads, kv_heads, head_dim, dtype, &pl) != VXG_OK) return 0;
  return pl.rec_bytes + pl.part_bytes;
}

vxg_status vxg_cache_attention(const vxg_kv_cache* c, const void* q, long long ld_q, int heads, int dtype, int total,
                               const int* table, int n_seq, int max_pages, const int* len, const int* cu, float scale,
                               int causal, int window, void* out, long long ld_out, void* workspace, size_t ws_bytes,
                               void* stream) {
  clear_error();
  vxg_status r = cache_check(c);
  if (r == VXG_OK) r = cache_batch_check(c, table, n_seq, max_pages, len, cu, total);
  if (r != VXG_OK) return r;
  VXG_ARG(dtype_known(dtype), "unknown element type %d", dtype);
  VXG_ARG(heads > 0 && heads % c->heads == 0, "%d query heads for %d key / value heads", heads, c->heads);
  VXG_ARG(window >= 0, "window must not be negative");
  VXG_ARG(scale == scale && scale - scale == 0.0f, "scale must be finite");
  if (total == 0 || n_seq == 0) return VXG_OK;
  VXG_ARG(q && out && workspace, "NULL pointer");
  const long long row = (long long)heads * c->head_dim, eb = (long long)dtype_bytes(dtype);
  VXG_ARG(ld_q >= row && ld_out >= row, "a row stride is below heads * head_dim = %lld", row);
  VXG_ARG((((uintptr_t)q | (uintptr_t)out | (uintptr_t)(ld_q * eb) | (uintptr_t)(ld_out * eb) | (uintptr_t)workspace) & 15) == 0,
          "q, out, their rows and the workspace must be 16-byte aligned");
  catt::Plan pl;
  if ((r = catt::plan(total, n_seq, heads, c->heads, c->head_dim, dtype, &pl)) != VXG_OK) return r;
  VXG_ARG(ws_bytes >= pl.rec_bytes + pl.part_bytes, "workspace of %zu bytes, %zu needed", ws_bytes,
          pl.rec_bytes + pl.part_bytes);
  int* status = device_status();
  VXG_ARG(status, "no CUDA device");
  catt::Params p = {};
  p.c = *c, p.q = q, p.out = out, p.ld_q = ld_q, p.ld_out = ld_out, p.table = table, p.len = len, p.cu = cu;
  p.rec = static_cast<long long*>(workspace);
  p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + pl.rec_bytes);
  p.status = status, p.n_seq = n_seq, p.max_pages = max_pages, p.total = total, p.heads = heads;
  p.share = heads / c->heads, p.window = window, p.causal = causal != 0, p.slots = pl.slots, p.grid = pl.grid;
  for (p.page_log2 = 4; 1 << p.page_log2 < c->page;) p.page_log2++;
  p.scale_log2 = scale * 1.44269504088896340736f;
  cudaStream_t st = (cudaStream_t)stream;
  if (pl.mt == 256) return catt::launch_tc(p, pl, c->head_dim, dtype, st);
  with_dtype(dtype, [&](auto tag) {
    constexpr int DT = decltype(tag)::value;
    if (c->head_dim == 128) r = pl.mt == 16 ? catt::launch<128, DT, 16>(p, pl, st) : catt::launch<128, DT, 64>(p, pl, st);
    else r = pl.mt == 16 ? catt::launch<64, DT, 16>(p, pl, st) : catt::launch<64, DT, 64>(p, pl, st);
  });
  return r;
}

}  // extern "C"
