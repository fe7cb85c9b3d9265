// Attention of new queries over the paged int8 cache:
//   out = sum_j softmax_j(scale * q . k_j) v_j,  k_j = code * k_scale[page], v_j = code * v_scale[page],
// for query i of n of a sequence of length L at position p = L - n + i: keys j < L, j <= p (causal), j > p - window.
// A query with no key gives 0.
//
// Arithmetic. Codes are exact in f16, so both products run on mma.m16n8k16 with f16 operands and f32 sums. A query row
// is scaled by a power of two so that its largest element lies in [2^14, 2^15): bf16 and f16 queries are then exact
// down to 2^-29 of that element; f32 queries are split into two f16 parts (22 bits). The page's key scale, the row's
// power of two, `scale` and log2(e) multiply the f32 sum. The softmax is kept in f32 with a running sum and a reference
// that may lag behind the maximum by up to 2^8, so that it seldom moves; a probability enters the second product as
// f16(p * 2^7 * v_scale / ref), ref being the largest value scale met so far (rounding 2^-11 of each term at most, 2^-32
// absolute against the largest; two parts for f32, 2^-22), which costs digits where p * v_scale falls below 2^-21 of ref
// (f32: 2^-10), as in a page whose scale is that much smaller than another's; ref and 2^-7 multiply the result. The sum of
// the row is taken from the unrounded p.
//
// Work split. A tile is MT consecutive (query, query head) rows of one sequence and KV head, so a key is read once for
// all the query heads that share it. The keys it sees, in blocks of 64, times all tiles and KV heads form one line of
// work units that is cut into equal shares, one a CTA: a CTA works off its share tile by tile, and a tile that spans
// shares leaves partial results (maximum, sum, unnormalised row) that a second small kernel joins. Lengths are read on
// the device, so the launch does not depend on them and can be captured; every CTA finds its share with one scan.
// This file: tiles of 64 rows, a consumer warp takes 16 rows and all 64 keys of a block (f32 queries, heads of 64).
// cached_attention_few.cu: up to 16 rows. cached_attention_tc.cu: 256 rows.
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
constexpr int MT = 64;       // rows per tile, 16 a consumer warp
constexpr int CONS = 4;      // consumer warps
constexpr int THREADS = (CONS + 1) * 32;
template <int HD>
struct Layout {
  static constexpr uint32_t TILE = BK * HD;      // bytes of one block's keys or values
  static constexpr uint32_t STAGE = 2 * TILE;
  static constexpr int STAGES = HD == 128 ? 5 : 8;
  static constexpr uint32_t SCALES = STAGES * STAGE;  // [stage][K 4, V 4] f32
  static constexpr uint32_t BARS = SCALES + STAGES * 32;
  static constexpr uint32_t BYTES = BARS + 2 * STAGES * 8 + 1024;  // + alignment
};

// Running softmax state of a warp's 16 rows: thread (g, c) holds rows g and g + 8.
template <int HD>
struct State {
  float o[HD / 8][4];
  float m[2], l[2];
  float ref;
};

template <int HD, int DT>
__global__ void __launch_bounds__(THREADS, 2)
    attend_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params p) {
  using Lay = Layout<HD>;
  using T = typename Elem<DT>::type;
  constexpr bool SPLIT = DT == VXG_DT_F32;
  constexpr int TOK = 32;  // keys a warp takes at a time
  constexpr bool BIASED = !SPLIT;
  constexpr int KS = HD / 16;         // k steps of the first product
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* scales_s = reinterpret_cast<float*>(smem + Lay::SCALES);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Lay::BARS);
  uint64_t* empty = full + Lay::STAGES;
  __shared__ Piece first_s;  // the share's first piece
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < Lay::STAGES; i++) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, CONS);
    }
    fence_mbar_init();
  }

  find_share<THREADS, MT, BK>(p, &first_s);
  Piece w = first_s;
  if (w.left == 0) return;

  if (warp == CONS) {
    produce<HD, MT, BK, Lay::STAGES>(p, w, map_k, map_v, smem, scales_s, full, empty);
    return;
  }

  // -------------------------------------------------------------------------------------------------- consumers
  const int g = lane >> 2, c = lane & 3;
  int st = 0;
  uint32_t phase = 0;
  bool ok = true;
  while (w.left > 0) {
    const Tile& t = w.t;
    const int take = w.take(), h = w.h, off = w.off;
    const int row0 = warp * 16;  // this warp's rows of the tile
    // this thread's two rows: operand fragments, limits, power of two
    uint32_t qa[KS][4], qb[SPLIT ? KS : 1][4];
    float rowf[2], bias[2];
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
      float top = 0.0f, sum = 0.0f;
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
        // a word of four codes gives the pairs (0, 2) and (1, 3) with a mask and a shift
        qa[w][e] = pack_f16(x0, x2);
        qa[w][2 + e] = pack_f16(x1, x3);
        if (SPLIT) {
          qb[w][e] = pack_rest(x0, x2, qa[w][e]);
          qb[w][2 + e] = pack_rest(x1, x3, qa[w][2 + e]);
        }
        if (BIASED) sum = add_f16(add_f16(sum, qa[w][e]), qa[w][2 + e]);
      }
      if (BIASED) {
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        bias[e] = -1152.0f * sum;
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
    float inv_ref = 0.0f;
    // 32 keys of a block: what fits the registers beside O and Q for heads of 64. f32 queries over heads of 128 spill some
    // 850 bytes a thread here (4 x 1024 queries over 1000, 16 heads: 553 us).
    auto keys32 = [&](auto tag, const uint8_t* kt, const uint8_t* vt, const float* scales, int key0) {
      constexpr bool masked = decltype(tag)::value;
      // ---- scores. 16-bit queries: the codes enter as 1152 + code, and the sums begin at -1152 times the row's sum
      float s[TOK / 8][4];
#pragma unroll
      for (int j = 0; j < TOK / 8; j++) {
#pragma unroll
        for (int k = 0; k < 4; k++) s[j][k] = BIASED ? bias[k >> 1] : 0.0f;
        const int r = 8 * j + g;  // rows of 32 keys begin on a swizzle period
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
          const uint32_t b0 = BIASED ? codes_biased(w[k]) : codes_to_f16(w[k]);
          const uint32_t b1 = BIASED ? codes_biased(w[k] >> 8) : codes_to_f16(w[k] >> 8);
          mma_f16(s[j], qa[k], b0, b1);
          if (SPLIT) mma_f16(s[j], qb[k], b0, b1);
        }
      }
      // ---- scale, mask
      float mx[2] = {-INFINITY, -INFINITY}, vsm = 0.0f;
#pragma unroll
      for (int j = 0; j < TOK / 8; j++) {
        const float ks = scales[j / 2];
        vsm = fmaxf(vsm, scales[4 + j / 2]);
#pragma unroll
        for (int k = 0; k < 4; k++) {
          float x = ks == NO_PAGE ? -INFINITY : s[j][k] * (rowf[k >> 1] * ks);
          if (masked) {
            const int key = key0 + 8 * j + 2 * c + (k & 1);
            if (key < klo[k >> 1] || key >= khi[k >> 1]) x = -INFINITY;
          }
          s[j][k] = x;
          mx[k >> 1] = fmaxf(mx[k >> 1], x);
        }
      }
      // ---- the rows' references move when a score has outgrown one by 2^8, ref when a value scale is larger than all before
      const bool wider = vsm > S.ref;
      if (__any_sync(0xffffffffu, wider || mx[0] > S.m[0] + 8.0f || mx[1] > S.m[1] + 8.0f)) {
        float reff = 1.0f;
        if (wider) {  // the same in the whole warp
          const float old = S.ref;
          S.ref = fmaxf(vsm, 1.17549435e-38f);  // what a written page has at least, so that the reciprocal is finite
          inv_ref = 1.0f / S.ref;
          reff = old / S.ref;
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
          const float m = fmaxf(S.m[e], mx[e]), alpha = ex2(S.m[e] - (m == -INFINITY ? 0.0f : m));
          S.m[e] = m;
          S.l[e] *= alpha;
#pragma unroll
          for (int j = 0; j < HD / 8; j++) S.o[j][2 * e] *= alpha * reff, S.o[j][2 * e + 1] *= alpha * reff;
        }
      }
      const float mu[2] = {S.m[0] == -INFINITY ? 0.0f : S.m[0], S.m[1] == -INFINITY ? 0.0f : S.m[1]};
      // ---- probabilities, times 2^7 and the value scale, and the second product, 16 keys a step
#pragma unroll
      for (int kk = 0; kk < TOK / 16; kk++) {
        const float vf = scales[4 + kk] * inv_ref * 128.0f;
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
        constexpr int W = HD / 32;  // words of a key that a thread takes
        uint32_t x[4][W];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int r = 16 * kk + 2 * c + (k & 1) + 8 * (k >> 1);
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
    };
    for (int b = 0; b < nb; b++) {
      ok = __all_sync(0xffffffffu, wait_phase(full + st, phase, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN));
      if (!ok) break;
      const uint8_t* kt = smem + st * Lay::STAGE;
      const int key0 = (t.blk0 + off + b) * BK;
      const bool inside = key0 >= all_lo && key0 + BK <= all_hi;
#pragma unroll 1
      for (int k = 0; k < BK; k += TOK) {
        const float* sc = scales_s + st * 8 + k / 16;
        if (inside) keys32(std::false_type(), kt + k * HD, kt + Lay::TILE + k * HD, sc, key0 + k);
        else keys32(std::true_type(), kt + k * HD, kt + Lay::TILE + k * HD, sc, key0 + k);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + st);
      if (++st == Lay::STAGES) st = 0, phase ^= 1;
    }
    if (!ok) return;
#pragma unroll
    for (int e = 0; e < 2; e++) {
      S.l[e] += __shfl_xor_sync(0xffffffffu, S.l[e], 1);
      S.l[e] += __shfl_xor_sync(0xffffffffu, S.l[e], 2);
    }
    const float unit = 1.0f / 128.0f;  // and S.ref last: their product may be too small for f32's digits
    const bool whole = off == 0 && take == t.cost;
    float* part = p.part + ((size_t)blockIdx.x * MAX_PIECES + (w.first ? 0 : 1)) * MT * (HD + 2);
    // thread (g, c)'s columns: HD / 4 consecutive ones, the first HD / 8 in o[.][0 or 2], the rest in o[.][1 or 3]
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
          for (int k = 0; k < 8; k++) a[k] = S.o[j + k][2 * e] * inv * S.ref, b2[k] = S.o[j + k][2 * e + 1] * inv * S.ref;
          store8<DT>(o + j, a);
          store8<DT>(o + HD / 8 + j, b2);
        }
      } else {
        float* o = part + r * (HD + 2);
        if (c == 0) o[0] = S.m[e], o[1] = S.l[e];
        o += 2 + c * (HD / 4);
#pragma unroll
        for (int j = 0; j < HD / 8; j++) {
          o[j] = S.o[j][2 * e] * unit * S.ref;
          o[HD / 8 + j] = S.o[j][2 * e + 1] * unit * S.ref;
        }
      }
    }
    w.next(p, MT, BK);
  }
}

constexpr int CTAS_PER_SM = 2;

// The kernels by the average number of (query, query head) rows a sequence and KV head has. Up to 8 and 16 rows: tiles of
// as many. More: tiles of 256 on tcgen05, which pay from a handful of rows on although most of a tile is empty then
// (measured, 16 sequences over 4000 tokens, heads of 128: 20 rows 97 us against 124 with tiles of 64, 96 rows 110 against
// 232); but tiles of 64 for f32 queries, whose two parts would not fit a 256-row tile, and for up to 64 rows of heads of
// 64, where they are the faster ones (8 sequences over 1000, 32 rows: 30 us against 34).
static vxg_status plan(int total, int n_seq, int heads, int kv, int hd, int dtype, Plan* pl) {
  const long long share = heads / kv, rows = (long long)total * share;
  const bool tiles64 = dtype == VXG_DT_F32 || (hd == 64 && rows <= 64LL * n_seq);
  pl->mt = rows <= 8LL * n_seq ? 8 : rows <= 16LL * n_seq ? 16 : tiles64 ? 64 : 256;
  const long long slots = rows / pl->mt + n_seq;
  if (slots > 0x3FFFFFFF) {
    set_error("%d rows of %d heads are more than one launch covers", total, heads);
    return VXG_ERR_UNSUPPORTED;
  }
  pl->slots = (int)slots;
  pl->grid = sm_count() * (pl->mt == 256 ? 1 : pl->mt == 8 ? FEW_CTAS_8 : CTAS_PER_SM);
  pl->rec_bytes = (size_t)pl->grid * 8 * sizeof(long long);
  pl->part_bytes = (size_t)pl->grid * MAX_PIECES * pl->mt * (hd + 2) * sizeof(float);
  return VXG_OK;
}

template <int HD, int DT>
vxg_status launch(const Params& p, const Plan& pl, cudaStream_t st) {
  CUtensorMap mk, mv;
  vxg_status r = cache_map(&mk, p.c, p.c.k, BK);
  if (r == VXG_OK) r = cache_map(&mv, p.c, p.c.v, BK);
  if (r != VXG_OK) return r;
  constexpr int smem = (int)Layout<HD>::BYTES;
  static_assert((smem + 1024) * CTAS_PER_SM <= 228 * 1024, "two blocks share an SM");
  if ((r = smem_attr((const void*)attend_kernel<HD, DT>, smem)) != VXG_OK) return r;
  attend_kernel<HD, DT><<<pl.grid, THREADS, smem, st>>>(mk, mv, p);
  VXG_CUDA(cudaGetLastError());
  return launch_join<HD, DT, MT, BK>(p, pl, st);
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
  const float scale_log2 = scale * 1.44269504088896340736f;
  VXG_ARG(scale_log2 - scale_log2 == 0.0f, "scale, and its product with log2(e), must be finite");
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
  p.status = status, p.n_seq = n_seq, p.max_pages = max_pages, p.total = total;
  p.share = heads / c->heads, p.window = window, p.causal = causal != 0, p.slots = pl.slots;
  for (p.page_log2 = 4; 1 << p.page_log2 < c->page;) p.page_log2++;
  p.scale_log2 = scale_log2;
  cudaStream_t st = (cudaStream_t)stream;
  if (pl.mt == 256) return catt::launch_tc(p, pl, c->head_dim, dtype, st);
  if (pl.mt <= 16) return catt::launch_few(p, pl, c->head_dim, dtype, st);
  with_dtype(dtype, [&](auto tag) {
    constexpr int DT = decltype(tag)::value;
    if constexpr (DT == VXG_DT_F32) {
      r = c->head_dim == 128 ? catt::launch<128, DT>(p, pl, st) : catt::launch<64, DT>(p, pl, st);
    } else {
      r = catt::launch<64, DT>(p, pl, st);
    }
  });
  return r;
}

}  // extern "C"
