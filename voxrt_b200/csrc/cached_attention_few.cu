// Attention over the paged int8 cache for few rows: tiles of up to 8 or 16 (query, query head) rows of a sequence and KV
// head, as in decoding one token, bound by the cache's bytes.
//
// Keys are the rows of the products (S^T = K Q^T, O^T = V^T P^T), so that up to eight query rows fill the narrow side of
// mma.m16n8k16 and a warp's state is small enough for twelve consumer warps an SM. Four consumer warps take 16 keys each of
// a block of 64; codes go from shared memory to operand registers with a mask, a shift and (values) a byte permute per
// word. Keys enter as 1152 + code, an f16 that needs no subtraction, and the sums begin at -1152 times the query row's sum
// (f32 queries, which need more than 16 bits of it, subtract). P^T comes out of S^T by an 8 x 8 transpose within the warp.
// The warps' states meet in shared memory at the end of a piece. Measured: 64 ragged sequences over up to 16000 tokens, 8
// cache heads of 128 for 32 query heads, 241 us (1.28 GB, 5.3 TB/s); f32 queries 312 us (4.1 TB/s); 16 heads of 64 without
// sharing 289 us (4.4 TB/s); 16-row tiles, 16 x 4 queries over 4000, 63 us (2.1 TB/s); one sequence over 1500 tokens, 16
// heads of 64, 12 us, the chain of dependent loads of the two kernels for the most part.
#include <cuda_runtime.h>

#include "cached_attention.cuh"

namespace vxg {
namespace catt {
namespace few {

constexpr int BK = 64, CONS = 4, THREADS = (CONS + 1) * 32;

template <int HD, int NQ>
struct Layout {
  static constexpr int MT = 8 * NQ;
  static constexpr uint32_t STAGE = 2 * BK * HD;
  static constexpr int STAGES = (NQ == 1 ? 3 : 4) * 128 / HD;
  static constexpr int LD = HD + 4;
  static constexpr uint32_t SCALES = STAGES * STAGE;                // [stage][K 4, V 4] f32
  static constexpr uint32_t MERGE = SCALES + STAGES * 32;           // [CONS][MT][LD] f32
  static constexpr uint32_t STAT = MERGE + CONS * MT * LD * 4;      // [CONS][MT][2] f32: maximum, sum
  static constexpr uint32_t BARS = STAT + CONS * MT * 8;
  static constexpr uint32_t BYTES = BARS + 2 * STAGES * 8 + 1024;   // + alignment
};

// d[i][j] of an 8 x 8 matrix of f16 (row lane / 4, columns 2 (lane % 4) ..) -> its transpose, laid out alike
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <int HD, int DT, int NQ>
__global__ void __launch_bounds__(THREADS, NQ == 1 ? FEW_CTAS_8 : 2)
    attend_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params p) {
  using Lay = Layout<HD, NQ>;
  using T = typename Elem<DT>::type;
  constexpr int MT = Lay::MT, LD = Lay::LD;
  constexpr bool SPLIT = DT == VXG_DT_F32;
  constexpr int KS = HD / 16;  // k steps of the first product, row tiles of the second
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* scales_s = reinterpret_cast<float*>(smem + Lay::SCALES);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Lay::BARS);
  uint64_t* empty = full + Lay::STAGES;
  __shared__ Piece first_s;  // the share's first piece
  __shared__ Piece piece_s;  // the consumers' next one
  __shared__ int fail;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < Lay::STAGES; i++) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, CONS);
    }
    fence_mbar_init();
    fail = 0;
  }
  find_share<THREADS, MT, BK>(p, &first_s);  // ends with a block barrier
  Piece w = first_s;
  if (w.left == 0) return;
  if (warp == CONS) {
    produce<HD, MT, BK, Lay::STAGES>(p, w, map_k, map_v, smem, scales_s, full, empty);
    return;
  }

  const int g = lane >> 2, c = lane & 3;
  int st = 0;
  uint32_t phase = 0;
  bool ok = true;
  while (w.left > 0) {
    const Tile& t = w.t;
    const int take = w.take(), h = w.h, off = w.off;
    // ---- operand B of the first product: row 8 n + g, this thread's quarter of it, in the order of the codes' pairs
    uint32_t qa[NQ][KS][2], qr[SPLIT ? NQ : 1][KS][2];
    // of rows 8 n + 2 c + e, which this thread's scores belong to
    float rowf[NQ][2], bias[NQ][2];
    int klo[NQ][2], khi[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
      const int r = 8 * n + g;
      const bool live = r < t.rows;
      const int rr = t.r0 + (live ? r : 0), i = rr / p.share, head = h * p.share + rr % p.share;
      const long long pos = (long long)t.L - t.n + i;
      const int hi = !live ? 0 : p.causal ? (int)::max(0LL, ::min((long long)t.L, pos + 1)) : t.L;
      const int lo = p.window > 0 ? (int)::max(0LL, pos - p.window + 1) : 0;
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
#pragma unroll
      for (int k = 0; k < KS; k++) {
        const float x0 = f[4 * k] * up, x1 = f[4 * k + 1] * up, x2 = f[4 * k + 2] * up, x3 = f[4 * k + 3] * up;
        qa[n][k][0] = pack_f16(x0, x2);
        qa[n][k][1] = pack_f16(x1, x3);
        if (SPLIT) {
          qr[n][k][0] = pack_rest(x0, x2, qa[n][k][0]);
          qr[n][k][1] = pack_rest(x1, x3, qa[n][k][1]);
        } else {
          sum = add_f16(add_f16(sum, qa[n][k][0]), qa[n][k][1]);
        }
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const float rf = __int_as_float((127 - ex) << 23) * p.scale_log2, bi = SPLIT ? 0.0f : -1152.0f * sum;
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int src = (2 * c + e) * 4;
        rowf[n][e] = __shfl_sync(0xffffffffu, rf, src);
        bias[n][e] = __shfl_sync(0xffffffffu, bi, src);
        khi[n][e] = __shfl_sync(0xffffffffu, hi, src);
        klo[n][e] = __shfl_sync(0xffffffffu, lo, src);
      }
    }
    const int nb = t.nblk > 0 ? take : 0, blk = t.blk0 + off;
    // blocks [in0, in1) of the piece: every live row of the tile sees all of their keys
    const int last_i = (t.r0 + t.rows - 1) / p.share, first_i = t.r0 / p.share;
    const long long all_hi = p.causal ? (long long)t.L - t.n + first_i + 1 : t.L;
    const long long all_lo = p.window > 0 ? (long long)t.L - t.n + last_i - p.window + 1 : 0;
    const int in0 = (int)::min((long long)nb, ::max(0LL, (all_lo + BK - 1) / BK - blk));
    const int in1 = (int)::min((long long)nb, ::max((long long)in0, all_hi > 0 ? all_hi / BK - blk : 0LL));

    float o[NQ][KS][4], m[NQ][2], l[NQ][2];  // o[n][i]: columns HD/8 g + 2 i (0, 1) and the next (2, 3), rows 2 c and 2 c + 1
    float ref = 0.0f, inv_ref = 0.0f;
#pragma unroll
    for (int n = 0; n < NQ; n++) {
#pragma unroll
      for (int i = 0; i < KS; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) o[n][i][k] = 0.0f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.0f;
    }

    auto block = [&](auto tag, int b) {
      constexpr bool masked = decltype(tag)::value;
      const uint8_t* kt = smem + st * Lay::STAGE;
      const uint8_t* vt = kt + BK * HD;
      const int tok0 = warp * 16, key0 = (blk + b) * BK + tok0 + g;
      const float ks = scales_s[st * 8 + warp], vs = scales_s[st * 8 + 4 + warp];
      // ---- scores of keys tok0 + g and tok0 + g + 8
      float s[NQ][4];
#pragma unroll
      for (int n = 0; n < NQ; n++)
#pragma unroll
        for (int k = 0; k < 4; k++) s[n][k] = bias[n][k & 1];
      uint32_t x0[HD / 16], x1[HD / 16];
      auto key = [&](int r, uint32_t (&x)[HD / 16]) {
        if (HD == 128) {
#pragma unroll
          for (int k = 0; k < 2; k++) {
            const uint4 y = *reinterpret_cast<const uint4*>(kt + r * 128 + (((2 * c + k) ^ (r & 7)) << 4));
            x[4 * k] = y.x, x[4 * k + 1] = y.y, x[4 * k + 2] = y.z, x[4 * k + 3] = y.w;
          }
        } else {
          const uint4 y = *reinterpret_cast<const uint4*>(kt + r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
          x[0] = y.x, x[1] = y.y, x[2] = y.z, x[3] = y.w;
        }
      };
      key(tok0 + g, x0);
      key(tok0 + g + 8, x1);
      float s2[NQ][4] = {};  // a second chain of sums
#pragma unroll
      for (int k = 0; k < KS; k++) {
        uint32_t a[4];
        if (SPLIT) a[0] = codes_to_f16(x0[k]), a[1] = codes_to_f16(x1[k]), a[2] = codes_to_f16(x0[k] >> 8), a[3] = codes_to_f16(x1[k] >> 8);
        else a[0] = codes_biased(x0[k]), a[1] = codes_biased(x1[k]), a[2] = codes_biased(x0[k] >> 8), a[3] = codes_biased(x1[k] >> 8);
#pragma unroll
        for (int n = 0; n < NQ; n++) {
          mma_f16(k & 1 ? s2[n] : s[n], a, qa[n][k][0], qa[n][k][1]);
          if (SPLIT) mma_f16(k & 1 ? s2[n] : s[n], a, qr[n][k][0], qr[n][k][1]);
        }
      }
      // the values' codes on their way under the softmax
      constexpr int W = HD / 32;  // words of a key that a thread takes
      uint32_t v[4][W];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int r = tok0 + 2 * c + (k & 1) + 8 * (k >> 1);
        if (HD == 128) {
          const uint4 y = *reinterpret_cast<const uint4*>(vt + r * 128 + ((g ^ (r & 7)) << 4));
          v[k][0] = y.x, v[k][1] = y.y, v[k][W - 2] = y.z, v[k][W - 1] = y.w;
        } else {
          const uint2 y = *reinterpret_cast<const uint2*>(vt + r * 64 + (((g >> 1) ^ ((r >> 1) & 3)) << 4) + (g & 1) * 8);
          v[k][0] = y.x, v[k][1] = y.y;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + st);
      // ---- scale, mask
      bool over = false;
#pragma unroll
      for (int n = 0; n < NQ; n++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int e = k & 1;
          s[n][k] = (s[n][k] + s2[n][k]) * (rowf[n][e] * ks);
          if (ks == NO_PAGE) s[n][k] = -INFINITY;
          if (masked) {
            const int key = key0 + (k >> 1) * 8;
            if (key < klo[n][e] || key >= khi[n][e]) s[n][k] = -INFINITY;
          }
          over = over || s[n][k] > m[n][e] + 8.0f;
        }
      // ---- the rows' references move when a score has outgrown one by 2^8, ref when a value scale is larger than all before
      const bool wider = vs > ref;
      if (__any_sync(0xffffffffu, over || wider)) {
        float reff = 1.0f;
        if (wider) {  // the same in the whole warp
          const float old = ref;
          ref = fmaxf(vs, 1.17549435e-38f);  // what a written page has at least, so that the reciprocal is finite
          inv_ref = 1.0f / ref;
          reff = old / ref;
        }
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float mx = fmaxf(s[n][e], s[n][2 + e]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            mx = fmaxf(mx, m[n][e]);
            const float a = ex2(m[n][e] - (mx == -INFINITY ? 0.0f : mx));
            m[n][e] = mx;
            l[n][e] *= a;
#pragma unroll
            for (int i = 0; i < KS; i++) o[n][i][e] *= a * reff, o[n][i][2 + e] *= a * reff;
          }
      }
      // ---- probabilities, times 2^7 and the value scale for the second product
      const float vf = vs * inv_ref * 128.0f;
      uint32_t pb[NQ][2], pr[SPLIT ? NQ : 1][2];
#pragma unroll
      for (int n = 0; n < NQ; n++) {
        float pv[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float mu = m[n][k & 1] == -INFINITY ? 0.0f : m[n][k & 1];
          pv[k] = ex2(s[n][k] - mu);
        }
        l[n][0] += pv[0] + pv[2];
        l[n][1] += pv[1] + pv[3];
#pragma unroll
        for (int k = 0; k < 4; k++) pv[k] *= vf;
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const uint32_t hi = pack_f16(pv[2 * k], pv[2 * k + 1]);
          pb[n][k] = transpose8(hi);
          if (SPLIT) pr[n][k] = transpose8(pack_rest(pv[2 * k], pv[2 * k + 1], hi));
        }
      }
      // ---- the second product: row tile i holds columns 2 i and 2 i + 1 of every g's run
#pragma unroll
      for (int i = 0; i < KS; i++) {
        const uint32_t sel = i & 1 ? 0x7632 : 0x5410;  // two columns of two keys: (key 0, key 0, key 1, key 1)
        const uint32_t y0 = __byte_perm(v[0][i >> 1], v[1][i >> 1], sel), y1 = __byte_perm(v[2][i >> 1], v[3][i >> 1], sel);
        const uint32_t a[4] = {codes_to_f16(y0), codes_to_f16(y0 >> 8), codes_to_f16(y1), codes_to_f16(y1 >> 8)};
#pragma unroll
        for (int n = 0; n < NQ; n++) {
          mma_f16(o[n][i], a, pb[n][0], pb[n][1]);
          if (SPLIT) mma_f16(o[n][i], a, pr[n][0], pr[n][1]);
        }
      }
    };
    for (int b = 0; b < nb; b++) {
      ok = __all_sync(0xffffffffu, wait_phase(full + st, phase, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN));
      if (!ok) break;
      if (b >= in0 && b < in1) block(std::false_type(), b);
      else block(std::true_type(), b);
      if (++st == Lay::STAGES) st = 0, phase ^= 1;
    }
    if (!ok && lane == 0) fail = 1;  // read behind the second barrier below: all give up together
    // ---- the warps' states meet
    auto result = [&](float x) { return x * (1.0f / 128.0f) * ref; };  // ref / 128 alone may be too small for f32's digits
    const bool whole = off == 0 && take == t.cost;
    float* part = p.part + ((size_t)blockIdx.x * MAX_PIECES + (w.first ? 0 : 1)) * MT * (HD + 2);
    float* mo = reinterpret_cast<float*>(smem + Lay::MERGE);
    float* ms = reinterpret_cast<float*>(smem + Lay::STAT);
#pragma unroll
    for (int n = 0; n < NQ; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
        const int r = warp * MT + 8 * n + 2 * c + e;
        float* row = mo + r * LD + (HD / 8) * g;
#pragma unroll
        for (int i = 0; i < KS; i += 2)
          *reinterpret_cast<float4*>(row + 2 * i) = make_float4(result(o[n][i][e]), result(o[n][i][2 + e]), result(o[n][i + 1][e]), result(o[n][i + 1][2 + e]));
        if (g == 0) ms[2 * r] = m[n][e], ms[2 * r + 1] = l[n][e];
      }
    named_bar_sync(1, CONS * 32);
    if (tid == 0) {  // one thread walks on for all of them, so that they always agree on the barriers to come
      Piece n = w;
      n.next(p, MT, BK);
      piece_s = n;
    }
    for (int r = warp; r < t.rows; r += CONS) {
      float mx = -INFINITY;
#pragma unroll
      for (int k = 0; k < CONS; k++) mx = fmaxf(mx, ms[(k * MT + r) * 2]);
      const float mu = mx == -INFINITY ? 0.0f : mx;
      float sum = 0.0f, acc[HD / 32] = {};
#pragma unroll
      for (int k = 0; k < CONS; k++) {
        const float f = ex2(ms[(k * MT + r) * 2] - mu);
        sum += f * ms[(k * MT + r) * 2 + 1];
#pragma unroll
        for (int j = 0; j < HD / 32; j++) acc[j] += f * mo[(k * MT + r) * LD + 32 * j + lane];
      }
      if (whole) {
        const int rr = t.r0 + r;
        T* out = static_cast<T*>(p.out) + (long long)(t.q0 + rr / p.share) * p.ld_out +
                 (long long)(h * p.share + rr % p.share) * HD;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int j = 0; j < HD / 32; j++) out[32 * j + lane] = Elem<DT>::narrow(acc[j] * inv);
      } else {
        float* x = part + r * (HD + 2);
        if (lane == 0) x[0] = mx, x[1] = sum;
#pragma unroll
        for (int j = 0; j < HD / 32; j++) x[2 + 32 * j + lane] = acc[j];
      }
    }
    named_bar_sync(1, CONS * 32);  // the buffers are free for the next piece
    if (fail) return;
    w = piece_s;
  }
}

template <int HD, int DT, int NQ>
vxg_status launch(const Params& p, const Plan& pl, cudaStream_t st) {
  CUtensorMap mk, mv;
  vxg_status r = cache_map(&mk, p.c, p.c.k, BK);
  if (r == VXG_OK) r = cache_map(&mv, p.c, p.c.v, BK);
  if (r != VXG_OK) return r;
  constexpr int smem = (int)Layout<HD, NQ>::BYTES;
  static_assert((smem + 1024) * (NQ == 1 ? FEW_CTAS_8 : 2) <= 228 * 1024, "the blocks share an SM");
  if ((r = smem_attr((const void*)attend_few_kernel<HD, DT, NQ>, smem)) != VXG_OK) return r;
  attend_few_kernel<HD, DT, NQ><<<pl.grid, THREADS, smem, st>>>(mk, mv, p);
  VXG_CUDA(cudaGetLastError());
  return launch_join<HD, DT, 8 * NQ, BK>(p, pl, st);
}

}  // namespace few

vxg_status launch_few(const Params& p, const Plan& pl, int head_dim, int dtype, cudaStream_t st) {
  vxg_status r = VXG_OK;
  with_dtype(dtype, [&](auto tag) {
    constexpr int DT = decltype(tag)::value;
    if (head_dim == 128) r = pl.mt == 8 ? few::launch<128, DT, 1>(p, pl, st) : few::launch<128, DT, 2>(p, pl, st);
    else r = pl.mt == 8 ? few::launch<64, DT, 1>(p, pl, st) : few::launch<64, DT, 2>(p, pl, st);
  });
  return r;
}

}  // namespace catt
}  // namespace vxg
