// int8 x int8 matrix product with a scale per token and per output channel:
//   S[t, o] = sum_k x[t, k] w[o, k]  (exact int32),  v = f32(S) * (sx[t] * sw[o]) (+ bias[o]),  y = ep(v).
// K < 131072 keeps every sum inside int32 (|x|, |w| <= 128), so sums may be split and joined in any order and every
// kernel shape gives the same bits.
//
// Few tokens: the weights' bytes bound the product, so a block takes 16 output channels and all of K, its warps share
// the K axis, and the weights go from memory straight into the operand registers of mma.m16n8k32: a thread's four
// 16-byte loads of a channel are k slots 4c..4c+3 of four steps, and as the token operand is loaded in the same order the
// permutation of k cancels. The warps' partial sums meet in shared memory.
#include <cuda_runtime.h>

#include <algorithm>

#include "common.h"
#include "dtype.cuh"
#include "math.cuh"

namespace vxg {
namespace i8 {

struct Params {
  const int8_t* x;
  const float* sx;
  const int8_t* w;
  const float* sw;
  const float* bias;
  void* y;
  long long ld_y;
  int M, N, K;
  int ep;
  float ep_scale;
};

__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// y = ep(f32(S) * (sx * sw) + bias); `old` is read for ADD_SCALED only.
__device__ __forceinline__ float finish(const Params& p, int s, float sx, float sw, float bias, float old) {
  float v = __fmul_rn((float)s, __fmul_rn(sx, sw));
  if (p.bias) v = __fadd_rn(v, bias);
  if (p.ep == VXG_EP_SILU) return silu_fast(v);
  if (p.ep == VXG_EP_ADD_SCALED) return __fmaf_rn(p.ep_scale, v, old);
  return v;
}

constexpr int FEW_WARPS = 8;
constexpr int SEG = 64;  // bytes of K per thread quad and step

// NT tiles of eight tokens, 16 output channels per block.
template <int DT, int NT>
__global__ void __launch_bounds__(FEW_WARPS * 32) gemm_few_kernel(Params p) {
  using T = typename Elem<DT>::type;
  __shared__ int part[FEW_WARPS][NT * 8][17];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int mt = (p.M + 8 * NT - 1) / (8 * NT);
  const int n0 = (int)(blockIdx.x / mt) * 16, m0 = (int)(blockIdx.x % mt) * 8 * NT;
  const int8_t* w0 = p.w + (size_t)::min(n0 + g, p.N - 1) * p.K;
  const int8_t* w1 = p.w + (size_t)::min(n0 + g + 8, p.N - 1) * p.K;
  const int8_t* xr[NT];
#pragma unroll
  for (int j = 0; j < NT; j++) xr[j] = p.x + (size_t)::min(m0 + 8 * j + g, p.M - 1) * p.K;
  int acc[NT][4] = {};
  const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll 4
  for (int k = warp * SEG + 16 * c; k < p.K + 16 * c; k += FEW_WARPS * SEG) {
    const bool in = k < p.K;  // K % 16 == 0: a 16-byte piece is inside or outside
    const uint4 a0 = in ? __ldcs(reinterpret_cast<const uint4*>(w0 + k)) : zero;
    const uint4 a1 = in ? __ldcs(reinterpret_cast<const uint4*>(w1 + k)) : zero;
    const uint32_t f0[4] = {a0.x, a1.x, a0.y, a1.y}, f1[4] = {a0.z, a1.z, a0.w, a1.w};
#pragma unroll
    for (int j = 0; j < NT; j++) {
      const uint4 b = in ? __ldg(reinterpret_cast<const uint4*>(xr[j] + k)) : zero;
      mma_s8(acc[j], f0, b.x, b.y);
      mma_s8(acc[j], f1, b.z, b.w);
    }
  }
#pragma unroll
  for (int j = 0; j < NT; j++)
#pragma unroll
    for (int i = 0; i < 4; i++) part[warp][8 * j + 2 * c + (i & 1)][g + 8 * (i >> 1)] = acc[j][i];
  __syncthreads();
  T* y = static_cast<T*>(p.y);
  for (int i = threadIdx.x; i < NT * 8 * 16; i += FEW_WARPS * 32) {
    const int t = i >> 4, o = i & 15;
    int s = 0;
#pragma unroll
    for (int k = 0; k < FEW_WARPS; k++) s += part[k][t][o];
    const int m = m0 + t, n = n0 + o;
    if (m < p.M && n < p.N) {
      T* yo = y + (size_t)m * p.ld_y + n;
      *yo = Elem<DT>::narrow(finish(p, s, __ldg(p.sx + m), __ldg(p.sw + n), p.bias ? __ldg(p.bias + n) : 0.0f,
                                    p.ep == VXG_EP_ADD_SCALED ? Elem<DT>::widen(*yo) : 0.0f));
    }
  }
}

template <int DT, int NT>
vxg_status launch_few(const Params& p, cudaStream_t st) {
  const long long blocks = (long long)((p.M + 8 * NT - 1) / (8 * NT)) * ((p.N + 15) / 16);
  if (blocks > 0x7FFFFFFFLL) {
    set_error("M = %d x N = %d is more than one launch covers", p.M, p.N);
    return VXG_ERR_UNSUPPORTED;
  }
  gemm_few_kernel<DT, NT><<<(unsigned)blocks, FEW_WARPS * 32, 0, st>>>(p);
  note_launch();
  VXG_CUDA(cudaGetLastError());
  return VXG_OK;
}

}  // namespace i8
}  // namespace vxg

using namespace vxg;

extern "C" vxg_status vxg_gemm_i8(const int8_t* x, const float* sx, const int8_t* w, const float* sw, int M, int N, int K,
                                  vxg_epilogue ep, float ep_scale, const float* bias, int dtype, void* y,
                                  long long ld_y, void* stream) {
  clear_error();
  VXG_ARG(M <= 0 || (x && sx && w && sw && y), "NULL pointer");
  VXG_ARG(M >= 0 && N > 0 && K > 0, "bad shape M=%d N=%d K=%d", M, N, K);
  VXG_ARG(dtype_known(dtype), "unknown element type %d", dtype);
  VXG_ARG(ep == VXG_EP_STORE || ep == VXG_EP_SILU || ep == VXG_EP_ADD_SCALED, "bad epilogue %d", (int)ep);
  VXG_ARG(ld_y >= N, "output row stride %lld is below N = %d", ld_y, N);
  VXG_ARG((((uintptr_t)x | (uintptr_t)w) & 15) == 0, "x and w must be 16-byte aligned");
  if (K % 16 != 0 || K >= 131072) {
    set_error("K = %d not supported (a multiple of 16 below 131072)", K);
    return VXG_ERR_UNSUPPORTED;
  }
  if (M == 0) return VXG_OK;
  i8::Params p = {x, sx, w, sw, bias, y, ld_y, M, N, K, (int)ep, ep_scale};
  vxg_status r = VXG_OK;
  with_dtype(dtype, [&](auto tag) {
    constexpr int DT = decltype(tag)::value;
    cudaStream_t st = (cudaStream_t)stream;
    r = M <= 8 ? i8::launch_few<DT, 1>(p, st)
        : M <= 16 ? i8::launch_few<DT, 2>(p, st)
        : M <= 32 ? i8::launch_few<DT, 4>(p, st) : i8::launch_few<DT, 8>(p, st);
  });
  return r;
}
