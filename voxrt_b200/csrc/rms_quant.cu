// Residual add + RMSNorm + int8, the plain int8 quantiser for 16-bit activations, and the reading back of codes.
//
//   h = fma(vs, v, x);  r = f32(1 / sqrt(sum(h^2) / d + eps));  y = (h * r) * gamma;
//   per group: a = max|y|, s = a / 127 (1 if a = 0), code = clamp(round_ties_even(y * (1/s)), +-127)
//
// The sum of squares and 1/sqrt run in 64 bits and are rounded once. A 24-bit square is exact there and the sum's own
// error is below 2^-45, so that how a row is split over threads (by the number of rows, among others) shows in its root
// only where that lies within 2^-45 of the middle between two f32 values: in fewer than one row in a million by this
// bound. Scale and code are the quantiser's of the other entries (quant_scale,
// quant_code: a NaN gives code 0 and is skipped by the maximum).
//
// Bound by memory: x and v are read once, the sum, the codes and the normalised row written once, and a row stays in
// registers (eight elements a thread and vector) between the two reductions: all of it with up to four vectors a thread.
// With eight, beside the next row's, 330 (16-bit) to 1030 bytes (f32) a thread spill: 4096 x 16384 f32 takes 346 us,
// 2.5 TB/s. A row of up to 256 elements belongs to one warp, a longer one to a block. Measured: 16384 x 4096 bf16 with
// residual 100 us (470 MB, 4.7 TB/s), 16384 x 1024 f16 31 us (3.8 TB/s), 8192 x 4096 f32 86 us (5.1 TB/s), one row of 1024
// 2.8 us. Without the codes and the residual 16384 x 4096 takes 58 us, the quantiser alone 41. 16-bit rows are held below the copy rate by issue (68 % of the slots busy):
// with the squares summed in f32 the first would take 5 % less, f32 rows the same.
#include <cuda_runtime.h>

#include <algorithm>

#include "common.h"
#include "dtype.cuh"
#include "math.cuh"

namespace vxg {
namespace rms {

constexpr int MAX_D = 32768;
constexpr int MAX_THREADS = 512;   // per row, with up to 8 vectors a thread
constexpr int WARP_ROWS = 4;       // rows of a block when a row is one warp's

struct Params {
  const void* x;
  const void* v;
  const float* gamma;
  void* x_res;
  void* y;
  int8_t* q;
  float* scales;
  long long ld_x, ld_v, ld_res, ld_y;
  double eps, inv_d;
  float vs;
  int n, d, group;
  int lanes;  // group < d, a power-of-two number of 8-element vectors, at most 32: its maximum by shuffles; else 0
  int vec;    // every row of every operand starts on a 16-byte boundary (q: 8) and d % 8 == 0
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// 1 / sqrt(v) in 64 bits, rounded to 32, by one step of Householder's third-order method: from a 32-bit root y, with
// e = 1 - v y^2 below 2^-21, the series y (1 + e / 2 + 3 e^2 / 8) leaves 5 e^3 / 16, less than a 64-bit rounding. Outside f32's range the library's operations.
__device__ __forceinline__ float inv_root(double v) {
  if (!(v > 1e-36 && v < 1e37)) return (float)__ddiv_rn(1.0, __dsqrt_rn(v));
  const double y = (double)rsqrtf((float)v);
  const double e = fma(-v * y, y, 1.0);
  return (float)fma(y * e, fma(e, 0.375, 0.5), y);
}

// NV vectors a thread, vector j of thread t covers elements 8 (t + j * threads) .. + 8. NORM: with the norm; else the
// row is quantised as it is. A block works off rows blockIdx, blockIdx + gridDim, .. and asks for the next row's vectors
// before the current one's reductions, whose barriers would else leave the memory idle. One element at a time (VEC
// false) there is no such look-ahead.
template <int DT, int NV, bool NORM, bool VEC>
__global__ void __launch_bounds__(MAX_THREADS) rms_quant_kernel(const Params p) {
  using T = typename Elem<DT>::type;
  extern __shared__ float gmax[];  // maxima of the groups that no shuffle covers
  __shared__ double wsum[2][MAX_THREADS / 32];
  __shared__ float wmax[2][MAX_THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool one_warp = blockDim.y > 1;  // a row per warp, blockDim = (32, WARP_ROWS)
  const int threads = blockDim.x, nwarps = threads >> 5, ng = p.d / p.group;
  const unsigned step = gridDim.x * blockDim.y, n = p.n;  // rows of up to 2^31 - 1 plus a step pass 31 bits, not 32
  const bool res = NORM && p.v != nullptr;
  Raw<DT> xr[NV], vr[NORM ? NV : 1];
  auto fetch = [&](unsigned row) {
    const T* x = static_cast<const T*>(p.x) + (long long)row * p.ld_x;
    const T* v = static_cast<const T*>(p.v) + (long long)row * p.ld_v;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const int c = 8 * ((int)threadIdx.x + j * threads);
#pragma unroll
      for (int i = 0; i < (DT == VXG_DT_F32 ? 2 : 1); i++) {
        xr[j].w[i] = c < p.d ? reinterpret_cast<const uint4*>(x + c)[i] : make_uint4(0, 0, 0, 0);
        if (NORM && res && c < p.d) vr[j].w[i] = reinterpret_cast<const uint4*>(v + c)[i];
      }
    }
  };
  unsigned row = blockIdx.x * blockDim.y + threadIdx.y;
  if (VEC && row < n) fetch(row);
  // a whole warp, or the whole block where barriers follow, leaves the loop together
  for (int turn = 0; row < n; row += step, turn ^= 1) {
    float h[NV][8];
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const int c = 8 * ((int)threadIdx.x + j * threads);
      float b[8];
      if (VEC) {
        unpack<DT>(xr[j], h[j]);
        if (NORM && res) unpack<DT>(vr[j], b);
      } else {
        const T* x = static_cast<const T*>(p.x) + (long long)row * p.ld_x;
        const T* v = static_cast<const T*>(p.v) + (long long)row * p.ld_v;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          h[j][i] = c + i < p.d ? Elem<DT>::widen(x[c + i]) : 0.0f;
          if (NORM && res) b[i] = c + i < p.d ? Elem<DT>::widen(v[c + i]) : 0.0f;
        }
      }
      if (NORM && res && c < p.d) {
#pragma unroll
        for (int i = 0; i < 8; i++) h[j][i] = __fmaf_rn(p.vs, b[i], h[j][i]);
        if (p.x_res) {
          T* r = static_cast<T*>(p.x_res) + (long long)row * p.ld_res;
          if (VEC) {
            store8<DT>(r + c, h[j]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
              if (c + i < p.d) r[c + i] = Elem<DT>::narrow(h[j][i]);
          }
        }
      }
    }
    if (VEC && row + step < n) fetch(row + step);
    if (NORM) {
      double sum = 0.0;
#pragma unroll
      for (int j = 0; j < NV; j++)
#pragma unroll
        for (int i = 0; i < 8; i++) sum = fma((double)h[j][i], (double)h[j][i], sum);
      sum = warp_sum(sum);
      if (!one_warp) {  // two buffers: a fast warp may be at the next row's sum while a slow one still reads
        if (lane == 0) wsum[turn][warp] = sum;
        __syncthreads();
        sum = warp_sum(lane < nwarps ? wsum[turn][lane] : 0.0);
      }
      const float rstd = inv_root(sum * p.inv_d + p.eps);
#pragma unroll
      for (int j = 0; j < NV; j++) {
        const int c = 8 * ((int)threadIdx.x + j * threads);
        if (c >= p.d) continue;
        float g[8];
        if (VEC) {
          load8<VXG_DT_F32>(p.gamma + c, g);
        } else {
#pragma unroll
          for (int i = 0; i < 8; i++) g[i] = c + i < p.d ? __ldg(p.gamma + c + i) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) h[j][i] = __fmul_rn(__fmul_rn(h[j][i], rstd), g[i]);
        if (p.y) {
          T* y = static_cast<T*>(p.y) + (long long)row * p.ld_y;
          if (VEC) {
            store8<DT>(y + c, h[j]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
              if (c + i < p.d) y[c + i] = Elem<DT>::narrow(h[j][i]);
          }
        }
      }
    }
    if (!p.q) continue;

    // the groups' maxima, then one scale and reciprocal per vector
    float amax[NV], seen = 0.0f;  // seen: NaN if one of the thread's values is
#pragma unroll
    for (int j = 0; j < NV; j++) {
      amax[j] = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; i++) amax[j] = fmaxf(amax[j], fabsf(h[j][i])), seen = max_nan(seen, h[j][i]);
    }
    if (ng == 1) {
      float m = amax[0];
#pragma unroll
      for (int j = 1; j < NV; j++) m = fmaxf(m, amax[j]);
      m = warp_max(m);
      if (!one_warp) {  // two buffers: a fast warp may be at the next row's maximum while a slow one still reads
        if (lane == 0) wmax[turn][warp] = m;
        __syncthreads();
        m = warp_max(lane < nwarps ? wmax[turn][lane] : 0.0f);
      }
#pragma unroll
      for (int j = 0; j < NV; j++) amax[j] = m;
    } else if (p.lanes) {
      for (int o = 1; o < p.lanes; o <<= 1) {
#pragma unroll
        for (int j = 0; j < NV; j++) amax[j] = fmaxf(amax[j], __shfl_xor_sync(0xffffffffu, amax[j], o));
      }
    } else {  // group % 8 == 0, so a vector lies in one group; maxima of non-negative floats order like their bits
      float* gm = gmax + threadIdx.y * ng;
      auto meet = [&]() {
        if (one_warp) __syncwarp();
        else __syncthreads();
      };
      meet();  // the last row's maxima have been read
      for (int g = threadIdx.x; g < ng; g += threads) gm[g] = 0.0f;
      meet();
#pragma unroll
      for (int j = 0; j < NV; j++) {
        const int c = 8 * ((int)threadIdx.x + j * threads);
        if (c < p.d) atomicMax(reinterpret_cast<int*>(gm + c / p.group), __float_as_int(amax[j]));
      }
      meet();
#pragma unroll
      for (int j = 0; j < NV; j++) {
        const int c = 8 * ((int)threadIdx.x + j * threads);
        if (c < p.d) amax[j] = gm[c / p.group];
      }
    }
    int8_t* q = p.q + (size_t)row * p.d;
    float* sc = p.scales + (size_t)row * ng;
    float s = 0.0f, inv = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const int c = 8 * ((int)threadIdx.x + j * threads);
      if (c >= p.d) continue;
      if (j == 0 || ng > 1) {
        s = quant_scale(amax[j]);
        inv = __fdiv_rn(1.0f, s);
      }
      if (ng == 1 ? c == 0 : c % p.group == 0) sc[ng == 1 ? 0 : c / p.group] = s;
      uint32_t w[2];
      if (seen == seen && amax[j] > 1e-35f && amax[j] < 1e38f) {  // the code is the rounding shifter's low byte
#pragma unroll
        for (int k = 0; k < 2; k++) w[k] = quant_word_fast(h[j][4 * k], h[j][4 * k + 1], h[j][4 * k + 2], h[j][4 * k + 3], inv);
      } else {
#pragma unroll
        for (int k = 0; k < 2; k++)
          w[k] = ((uint32_t)quant_code(h[j][4 * k], inv) & 0xFFu) | (((uint32_t)quant_code(h[j][4 * k + 1], inv) & 0xFFu) << 8) |
                 (((uint32_t)quant_code(h[j][4 * k + 2], inv) & 0xFFu) << 16) |
                 (((uint32_t)quant_code(h[j][4 * k + 3], inv) & 0xFFu) << 24);
      }
      if (VEC) {
        *reinterpret_cast<uint2*>(q + c) = make_uint2(w[0], w[1]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (c + i < p.d) q[c + i] = (int8_t)(w[i >> 2] >> (8 * (i & 3)));
      }
    }
  }
}

// value = code * scale, rounded once to the output type; groups are consecutive in memory, so element i is in group
// i / group. 16 codes a thread where a group holds whole vectors, one otherwise.
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) dequantize_kernel(const int8_t* __restrict__ q, const float* __restrict__ s,
                                                         unsigned long long total, unsigned group,
                                                         typename Elem<DT>::type* __restrict__ out) {
  constexpr int E = VEC ? 16 : 1;
  const unsigned long long step = (unsigned long long)gridDim.x * blockDim.x * E;
  for (unsigned long long i = ((unsigned long long)blockIdx.x * blockDim.x + threadIdx.x) * E; i < total; i += step) {
    const float sc = __ldg(s + ((i >> 32) ? i / group : (unsigned)i / group));
    if (VEC) {
      const uint4 w4 = *reinterpret_cast<const uint4*>(q + i);
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int k = 0; k < 2; k++) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = __fmul_rn((float)(int8_t)(w[2 * k + (e >> 2)] >> (8 * (e & 3))), sc);
        store8<DT>(out + i + 8 * k, v);
      }
    } else {
      out[i] = Elem<DT>::narrow(__fmul_rn((float)q[i], sc));
    }
  }
}

// As many blocks as the GPU holds at once, or as there are rows.
template <class Kernel>
void start(Kernel k, const Params& p, dim3 grid, dim3 block, size_t smem, cudaStream_t st) {
  int per_sm = 1;
  if (grid.x > (unsigned)sm_count() &&
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k, (int)(block.x * block.y), smem) != cudaSuccess || per_sm < 1)
    per_sm = 1;
  grid.x = std::min(grid.x, (unsigned)(sm_count() * per_sm));
  k<<<grid, block, smem, st>>>(p);
}

template <int DT, int NV, bool NORM>
void launch(const Params& p, dim3 grid, dim3 block, size_t smem, cudaStream_t st) {
  if (p.vec) start(rms_quant_kernel<DT, NV, NORM, true>, p, grid, block, smem, st);
  else start(rms_quant_kernel<DT, NV, NORM, false>, p, grid, block, smem, st);
}

template <int DT, bool NORM>
void launch_nv(int nv, const Params& p, dim3 grid, dim3 block, size_t smem, cudaStream_t st) {
  switch (nv) {
    case 1: launch<DT, 1, NORM>(p, grid, block, smem, st); break;
    case 2: launch<DT, 2, NORM>(p, grid, block, smem, st); break;
    case 4: launch<DT, 4, NORM>(p, grid, block, smem, st); break;
    default: launch<DT, 8, NORM>(p, grid, block, smem, st); break;
  }
}

static vxg_status run(Params p, int dtype, bool norm, cudaStream_t st) {
  VXG_ARG(dtype_known(dtype), "unknown element type %d", dtype);
  VXG_ARG(p.n >= 0 && p.d > 0, "bad shape n=%d d=%d", p.n, p.d);
  if (p.n > 0) VXG_ARG(p.x && (!norm || p.gamma) && (p.q || p.y || p.x_res), "NULL input, or no output given");
  VXG_ARG(!p.q || p.scales, "codes without scales");
  VXG_ARG(aligned(dtype_bytes(dtype), p.x, p.v, p.x_res, p.y) &&
              aligned(4, p.gamma, p.scales), "an operand is not aligned to its elements");
  VXG_ARG(!p.q || (p.group > 0 && p.d % p.group == 0), "group %d does not divide the row width %d", p.group, p.d);
  if (!p.q) p.group = p.d;
  VXG_ARG(p.ld_x >= p.d && (!p.v || p.ld_v >= p.d) && (!p.x_res || p.ld_res >= p.d) && (!p.y || p.ld_y >= p.d),
          "a row stride is below the row width %d", p.d);
  if (p.d > MAX_D || (p.group != p.d && p.group % 8 != 0)) {
    set_error("row width %d (max %d) or group %d (the row or a multiple of 8) not supported", p.d, MAX_D, p.group);
    return VXG_ERR_UNSUPPORTED;
  }
  if (p.n == 0) return VXG_OK;
  const size_t eb = dtype_bytes(dtype);
  auto rows16 = [&](const void* a, long long ld) { return !a || (((uintptr_t)a | (uintptr_t)(ld * (long long)eb)) & 15) == 0; };
  p.vec = p.d % 8 == 0 && rows16(p.x, p.ld_x) && rows16(p.v, p.ld_v) && rows16(p.x_res, p.ld_res) && rows16(p.y, p.ld_y) &&
          ((uintptr_t)p.q & 7) == 0 && ((uintptr_t)p.gamma & 15) == 0;
  const int vecs = (p.d + 7) / 8, lanes = p.group / 8;
  p.lanes = p.group < p.d && lanes <= 32 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
  // Many rows: 256 threads a row, whose barriers are cheaper; few (fewer than four an SM): 512, which shortens a row's
  // own time. Measured, 4096 columns, bf16: 16384 rows 114 against 132 us, one row 4.0 against 3.7 us
  // (both sides before the codes' fast rounding, which brought the first to 102).
  const int most = p.n < 4 * sm_count() ? 512 : 256;
  int nv = 1;
  while (nv < 8 && (vecs + nv - 1) / nv > most) nv *= 2;
  const int threads = ((vecs + nv - 1) / nv + 31) / 32 * 32;
  dim3 block(threads), grid(p.n);
  if (threads == 32) {
    block.y = WARP_ROWS;
    grid.x = ((unsigned)p.n + WARP_ROWS - 1) / WARP_ROWS;
  }
  const size_t smem = p.group < p.d && !p.lanes ? (size_t)block.y * (p.d / p.group) * sizeof(float) : 0;  // <= 16 KB
  with_dtype(dtype, [&](auto tag) {
    constexpr int DT = decltype(tag)::value;
    if (norm) launch_nv<DT, true>(nv, p, grid, block, smem, st);
    else launch_nv<DT, false>(nv, p, grid, block, smem, st);
  });
  note_launch();
  VXG_CUDA(cudaGetLastError());
  return VXG_OK;
}

}  // namespace rms
}  // namespace vxg

using namespace vxg;

extern "C" {

vxg_status vxg_rms_quant(const void* x, long long ld_x, const void* v, long long ld_v, float vs, int dtype, int n, int d,
                         const float* gamma, float eps, void* x_res, long long ld_res, void* y, long long ld_y,
                         int group, int8_t* q, float* scales, void* stream) {
  clear_error();
  VXG_ARG(eps >= 0.0f, "eps must not be negative");
  VXG_ARG(n <= 0 || !x_res || v, "x_res needs the residual input");
  rms::Params p = {};
  p.x = x, p.v = v, p.gamma = gamma, p.x_res = x_res, p.y = y, p.q = q, p.scales = scales;
  p.ld_x = ld_x, p.ld_v = ld_v, p.ld_res = ld_res, p.ld_y = ld_y;
  p.eps = eps, p.inv_d = 1.0 / d, p.vs = vs, p.n = n, p.d = d, p.group = group;
  return rms::run(p, dtype, true, (cudaStream_t)stream);
}

vxg_status vxg_quantize_tokens(const void* x, long long ld_x, int dtype, int n, int d, int group, int8_t* q,
                               float* scales, void* stream) {
  clear_error();
  VXG_ARG(n <= 0 || (q && scales), "NULL output");
  rms::Params p = {};
  p.x = x, p.q = q, p.scales = scales, p.ld_x = ld_x, p.n = n, p.d = d, p.group = group;
  return rms::run(p, dtype, false, (cudaStream_t)stream);
}

vxg_status vxg_dequantize_rows(const int8_t* q, const float* scales, int n, int inp, int group, int dtype, void* out,
                               void* stream) {
  clear_error();
  VXG_ARG(n <= 0 || (q && scales && out), "NULL pointer");
  VXG_ARG(dtype_known(dtype), "unknown element type %d", dtype);
  VXG_ARG(n >= 0 && inp > 0 && group > 0 && inp % group == 0, "bad shape n=%d inp=%d group=%d", n, inp, group);
  VXG_ARG(aligned(dtype_bytes(dtype), out) && aligned(4, scales), "an operand is not aligned to its elements");
  if (n == 0) return VXG_OK;
  const unsigned long long total = (unsigned long long)n * (unsigned)inp;
  const bool vec = group % 16 == 0 && (((uintptr_t)q | (uintptr_t)out) & 15) == 0;
  const unsigned long long per_block = 256ull * (vec ? 16 : 1);
  const unsigned blocks = (unsigned)std::min<unsigned long long>((total + per_block - 1) / per_block, 1u << 20);
  with_dtype(dtype, [&](auto tag) {
    constexpr int DT = decltype(tag)::value;
    using T = typename Elem<DT>::type;
    if (vec)
      rms::dequantize_kernel<DT, true><<<blocks, 256, 0, (cudaStream_t)stream>>>(q, scales, total, (unsigned)group, (T*)out);
    else
      rms::dequantize_kernel<DT, false><<<blocks, 256, 0, (cudaStream_t)stream>>>(q, scales, total, (unsigned)group, (T*)out);
  });
  note_launch();
  VXG_CUDA(cudaGetLastError());
  return VXG_OK;
}

}  // extern "C"
