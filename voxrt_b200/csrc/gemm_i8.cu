// int8 x int8 matrix product with a scale per token and per output channel:
//   S[t, o] = sum_k x[t, k] w[o, k]  (exact int32),  v = f32(S) * (sx[t] * sw[o]) (+ bias[o]),  y = ep(v).
// K < 131072 keeps every sum inside int32 (|x|, |w| <= 128), so sums may be split and joined in any order and every
// kernel shape gives the same bits.
//
// Few tokens (up to 64): the weights' bytes bound the product, so a block takes 16 or 32 output channels and all of K, its
// warps share the K axis, and the weights go from memory straight into the operand registers of mma.m16n8k32: the words of a
// thread's 16-byte load of a channel are its k slots of two steps, and as the token operand is loaded in the same order the
// permutation of k cancels. The warps' partial sums meet in shared memory. Measured: one token, 16384 x 8192 weights
// (larger than L2) 24 to 27 us, 5.0 to 5.7 TB/s; 37 tokens, 16384 x 8192 41 us (3.3 TB/s); 8192 x 2048 with three and four
// sets of operands in turn (50 and 67 MB, in L2 for a part) 7.1 and 9.0 us.
#include <cuda_runtime.h>

#include <algorithm>

#include "common.h"
#include "dtype.cuh"
#include "math.cuh"
#include "ptx.cuh"
#include "wait.cuh"

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

// NT tiles of eight tokens, MT tiles of 16 output channels per block.
template <int DT, int NT, int MT>
__global__ void __launch_bounds__(FEW_WARPS * 32) gemm_few_kernel(Params p) {
  using T = typename Elem<DT>::type;
  constexpr int CH = 16 * MT, LD = CH + 1;
  extern __shared__ int part[];  // [FEW_WARPS][NT * 8][LD]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int mt = (p.M + 8 * NT - 1) / (8 * NT);
  const int n0 = (int)(blockIdx.x / mt) * CH, m0 = (int)(blockIdx.x % mt) * 8 * NT;
  const int8_t* wr[2 * MT];
#pragma unroll
  for (int j = 0; j < 2 * MT; j++) wr[j] = p.w + (size_t)::min(n0 + 8 * j + g, p.N - 1) * p.K;
  const int8_t* xr[NT];
#pragma unroll
  for (int j = 0; j < NT; j++) xr[j] = p.x + (size_t)::min(m0 + 8 * j + g, p.M - 1) * p.K;
  int acc[MT][NT][4] = {};
  const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll NT * MT <= 2 ? 4 : 2
  for (int k = warp * SEG + 16 * c; k < p.K + 16 * c; k += FEW_WARPS * SEG) {
    const bool in = k < p.K;  // K % 16 == 0: a 16-byte piece is inside or outside
    uint4 a[2 * MT], b[NT];
#pragma unroll
    for (int j = 0; j < 2 * MT; j++) a[j] = in ? __ldcs(reinterpret_cast<const uint4*>(wr[j] + k)) : zero;
#pragma unroll
    for (int j = 0; j < NT; j++) b[j] = in ? __ldg(reinterpret_cast<const uint4*>(xr[j] + k)) : zero;
#pragma unroll
    for (int i = 0; i < MT; i++) {
      const uint4 a0 = a[2 * i], a1 = a[2 * i + 1];
      const uint32_t f0[4] = {a0.x, a1.x, a0.y, a1.y}, f1[4] = {a0.z, a1.z, a0.w, a1.w};
#pragma unroll
      for (int j = 0; j < NT; j++) {
        mma_s8(acc[i][j], f0, b[j].x, b[j].y);
        mma_s8(acc[i][j], f1, b[j].z, b[j].w);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
      for (int e = 0; e < 4; e++)
        part[(warp * NT * 8 + 8 * j + 2 * c + (e & 1)) * LD + 16 * i + g + 8 * (e >> 1)] = acc[i][j][e];
  __syncthreads();
  T* y = static_cast<T*>(p.y);
  for (int i = threadIdx.x; i < NT * 8 * CH; i += FEW_WARPS * 32) {
    const int t = i / CH, o = i % CH, m = m0 + t, n = n0 + o;
    if (m >= p.M || n >= p.N) continue;
    int s = 0;
#pragma unroll
    for (int k = 0; k < FEW_WARPS; k++) s += part[(k * NT * 8 + t) * LD + o];
    T* yo = y + (size_t)m * p.ld_y + n;
    *yo = Elem<DT>::narrow(finish(p, s, __ldg(p.sx + m), __ldg(p.sw + n), p.bias ? __ldg(p.bias + n) : 0.0f,
                                  p.ep == VXG_EP_ADD_SCALED ? Elem<DT>::widen(*yo) : 0.0f));
  }
}

template <int DT, int NT, int MT>
vxg_status launch_few_mt(const Params& p, cudaStream_t st) {
  const long long blocks = (long long)((p.M + 8 * NT - 1) / (8 * NT)) * ((p.N + 16 * MT - 1) / (16 * MT));
  if (blocks > 0x7FFFFFFFLL) {
    set_error("M = %d x N = %d is more than one launch covers", p.M, p.N);
    return VXG_ERR_UNSUPPORTED;
  }
  constexpr int smem = FEW_WARPS * NT * 8 * (16 * MT + 1) * (int)sizeof(int);
  const vxg_status r = smem_attr((const void*)gemm_few_kernel<DT, NT, MT>, smem);
  if (r != VXG_OK) return r;
  gemm_few_kernel<DT, NT, MT><<<(unsigned)blocks, FEW_WARPS * 32, smem, st>>>(p);
  note_launch();
  VXG_CUDA(cudaGetLastError());
  return VXG_OK;
}

// Every block reads all the tokens' bytes, from L2: from 17 tokens on that is as much as the weights, and a block takes
// 32 channels to halve it, as long as that leaves a block for about every second SM.
template <int DT, int NT>
vxg_status launch_few(const Params& p, cudaStream_t st) {
  if (NT >= 3 && p.N >= 2048) return launch_few_mt<DT, NT, 2>(p, st);
  return launch_few_mt<DT, NT, 1>(p, st);
}

// ------------------------------------------------------------------------------------------------ many tokens
// A pair of CTAs (cta_group::2) owns a tile of 256 tokens x BN channels: each brings 128 rows of x and BN / 2 rows of w
// into its shared memory, the leader issues M = 256 products over both, and each CTA's TMEM receives its 128 tokens'
// int32 sums. Sharing w this way halves the operand bytes an SM reads per product, which is what limits a single CTA's
// 128 x 256 tile. Persistent over tiles, two TMEM buffers, so a tile's epilogue runs under the next one's products.
// Roles: warps 0-7 epilogue (TMEM lanes 32 (w % 4).., column half w / 4), warp 8 TMA producer, warp 9 MMA issuer (leader).
// Measured, 8192 x 16384 x 4096: 346 .. 356 us, 3.1 .. 3.2 POP/s, 90 .. 93 % of twice the bf16 library product's rate (8192 x
// 8192 x 4096 alone: tensor pipe 88 % busy); 1500 x 1024 x 4096: 11.1 us, of which a tile's 16 stages are 6 and the rest is
// launch, fill and epilogue. Stages of 128 k, with a wait and a commit each, were slower at small tiles, where issuing is the
// bound (256 x 512 x 16384: 32.8 against 23.5 us).
namespace tc {

constexpr int BM = 256, BK = 256, SUB = 128, EPI_WARPS = 8, THREADS = (EPI_WARPS + 2) * 32;
constexpr int GROUP_M = 8;  // token tiles that share a run of weight tiles while both stay in L2

template <int BN>
struct Cfg {
  static constexpr uint32_t A_BYTES = 128 * BK, B_BYTES = BN / 2 * BK, STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = BN == 256 ? 3 : 4;       // of two swizzled runs of 128 k: a wait and a commit for 8 products
  static constexpr uint32_t A_SUB = 128 * SUB, B_SUB = BN / 2 * SUB;
  static constexpr uint32_t COLS = 2 * BN;             // two accumulators
  static constexpr uint32_t XCH = STAGES * STAGE;      // [8][32][17] int32: rows that cannot be stored as vectors
  static constexpr uint32_t SCALE = XCH + EPI_WARPS * 32 * 17 * 4;  // [2][BN] channel scales, [2][BN] bias
  static constexpr uint32_t BARS = SCALE + 4 * BN * 4;
  static constexpr uint32_t BYTES = BARS + (2 * STAGES + 4) * 8 + 16 + 1024;
  static_assert(BYTES <= 232448, "shared memory budget");
};

// Tile t of the launch: runs of GROUP_M token tiles, weight tile by weight tile.
__device__ __forceinline__ void tile_of(int t, int mt, int nt, int& m, int& n) {
  const int per = GROUP_M * nt, g = t / per, in = t % per, rows = ::min(GROUP_M, mt - g * GROUP_M);
  m = g * GROUP_M + in % rows;
  n = in / rows;
}

__device__ __forceinline__ void stg32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// VEC: every 32-byte run of an output row is aligned and inside or outside the row as a whole.
template <int DT, int BN, bool VEC>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    gemm_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const Params p,
                   int* status) {
  using C = Cfg<BN>;
  using T = typename Elem<DT>::type;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BARS);  // leader: both CTAs' bytes of a stage have landed
  uint64_t* empty = full + C::STAGES;                            // a stage's products are done
  uint64_t* tfull = empty + C::STAGES;                           // an accumulator is complete
  uint64_t* tempty = tfull + 2;                                  // leader: both CTAs have read an accumulator
  uint32_t* holder = reinterpret_cast<uint32_t*>(tempty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; i++) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(tfull + i, 1);
      mbar_init(tempty + i, 2 * EPI_WARPS);
    }
    fence_mbar_init();
  }
  if (warp == EPI_WARPS + 1) {
    tmem_alloc_pair(holder, C::COLS);
    tmem_relinquish_pair();
  }
  if (warp == EPI_WARPS && lane == 0) {
    prefetch_tmap(&map_x);
    prefetch_tmap(&map_w);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *holder;

  const int mt = (p.M + BM - 1) / BM, nt = (p.N + BN - 1) / BN, tiles = mt * nt;
  const int chunks = (p.K + BK - 1) / BK, pairs = gridDim.x / 2, pair = blockIdx.x / 2;

  if (warp == EPI_WARPS) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs) {
        int m, n;
        tile_of(t, mt, nt, m, n);
        for (int c = 0; c < chunks; c++, it++) {
          const int s = it % C::STAGES;
          if (it >= C::STAGES && !wait_phase(empty + s, ((it / C::STAGES) - 1) & 1, status, VXG_DEV_TIMEOUT_PRODUCER)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(full + s, 2 * C::STAGE);
          const uint32_t bar = map_cluster(full + s, 0);
          uint8_t* a = smem + s * C::STAGE;
#pragma unroll
          for (int h = 0; h < BK / SUB; h++) {
            tma_load_2d_pair(a + h * C::A_SUB, &map_x, c * BK + h * SUB, m * BM + (int)rank * 128, bar);
            tma_load_2d_pair(a + C::A_BYTES + h * C::B_SUB, &map_w, c * BK + h * SUB, n * BN + (int)rank * (BN / 2), bar);
          }
        }
      }
      // The copies land before the block ends: their products' commits say so; after a timeout, wait for longer than a
      // copy can take.
      const int last = ::min(it, (int)C::STAGES);
      for (int i = it - last; i < it && ok; i++)
        ok = wait_phase(empty + i % C::STAGES, (i / C::STAGES) & 1, status, VXG_DEV_TIMEOUT_DRAIN);
      if (!ok)
        for (const uint64_t t0 = globaltimer(); globaltimer() - t0 < 10000000ull;) __nanosleep(10000);
    }
  } else if (warp == EPI_WARPS + 1) {
    // the whole warp walks and waits, which keeps the descriptors in uniform registers; one lane issues
    if (rank == 0) {
      const bool leader = elect_one();
      const uint64_t da = umma_desc_sw128(smem_u32(smem)), db = umma_desc_sw128(smem_u32(smem + C::A_BYTES));
      int it = 0, k = 0, s = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs, k++) {
        const int b = k & 1;
        ok = k < 2 || wait_phase(tempty + b, ((k >> 1) - 1) & 1, status, VXG_DEV_TIMEOUT_MMA);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + b * BN;
        for (int c = 0; c < chunks; c++, it++) {
          ok = __all_sync(0xffffffffu, wait_phase(full + s, phase, status, VXG_DEV_TIMEOUT_MMA));
          if (!ok) break;
          tc_fence_after();
          const uint64_t ad = da + (uint32_t)s * (C::STAGE / 16), bd = db + (uint32_t)s * (C::STAGE / 16);
          if (leader) {
#pragma unroll
            for (int j = 0; j < BK / 32; j++)
              mma_i8_pair(d, ad + (j / 4) * (C::A_SUB / 16) + 2 * (j % 4), bd + (j / 4) * (C::B_SUB / 16) + 2 * (j % 4),
                          idesc_i8(BM, BN), j != 0 || c != 0 ? 1u : 0u);
            mma_commit_pair(empty + s);
          }
          __syncwarp();
          if (++s == C::STAGES) s = 0, phase ^= 1;
        }
        if (ok && leader) mma_commit_pair(tfull + b);
        __syncwarp();
      }
    }
  } else {
    const int q = warp & 3, half = warp >> 2, tid = threadIdx.x;
    float* sw_s = reinterpret_cast<float*>(smem + C::SCALE);
    int* xch = reinterpret_cast<int*>(smem + C::XCH) + warp * 32 * 17;
    T* y = static_cast<T*>(p.y);
    int k = 0;
    bool ok = true;
    for (int t = pair; t < tiles; t += pairs, k++) {
      const int b = k & 1;
      int m, n;
      tile_of(t, mt, nt, m, n);
      const int n0 = n * BN;
      float* sw = sw_s + b * BN;
      float* bs = sw_s + (2 + b) * BN;
      for (int i = tid; i < BN; i += EPI_WARPS * 32) {
        sw[i] = n0 + i < p.N ? __ldg(p.sw + n0 + i) : 0.0f;
        bs[i] = p.bias && n0 + i < p.N ? __ldg(p.bias + n0 + i) : 0.0f;
      }
      named_bar_sync(1, EPI_WARPS * 32);  // also: nobody is still at the tile that used this half two tiles ago
      const int row0 = m * BM + (int)rank * 128 + q * 32, row = row0 + lane;
      const float sx = row < p.M ? __ldg(p.sx + row) : 0.0f;
      // a warp that gave up goes on to meet the others' barriers, without reading or writing anything more
      ok = ok && wait_phase(tfull + b, (k >> 1) & 1, status, VXG_DEV_TIMEOUT_EPILOGUE);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) continue;
      tc_fence_after();
#pragma unroll 1
      for (int c0 = half * (BN / 2); c0 < (half + 1) * (BN / 2); c0 += 32) {
        uint32_t r[32];
        tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * BN + c0), r);
        tmem_wait_ld();
        if (c0 + 32 == (half + 1) * (BN / 2)) {  // the warp's last read of this accumulator
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(map_cluster(tempty + b, 0));
        }
        if (VEC) {
          constexpr int E = DT == VXG_DT_F32 ? 8 : 16;  // elements of 32 bytes
          if (row < p.M) {
            T* yo = y + (size_t)row * p.ld_y + n0 + c0;
#pragma unroll
            for (int j = 0; j < 32; j += E) {
              if (n0 + c0 + j < p.N) {
                float v[E];
                if (p.ep == VXG_EP_ADD_SCALED) {
#pragma unroll
                  for (int e = 0; e < E; e += 8) {
                    float o8[8];
                    load8<DT>(yo + j + e, o8);
#pragma unroll
                    for (int i = 0; i < 8; i++) v[e + i] = o8[i];
                  }
                }
#pragma unroll
                for (int e = 0; e < E; e++)
                  v[e] = finish(p, (int)r[j + e], sx, sw[c0 + j + e], bs[c0 + j + e], p.ep == VXG_EP_ADD_SCALED ? v[e] : 0.0f);
                uint32_t o[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                  if constexpr (DT == VXG_DT_F32) o[e] = __float_as_uint(v[e]);
                  else o[e] = narrow2<DT>(v[2 * e], v[2 * e + 1]);
                }
                stg32(yo + j, o);
              }
            }
          }
        } else {
          // rows of any alignment: through shared memory, so that a store covers consecutive columns of one row
          const int o = lane & 15;
#pragma unroll
          for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int j = 0; j < 16; j++) xch[lane * 17 + j] = (int)r[16 * h + j];
            __syncwarp();
            const int cc = c0 + 16 * h + o, col = n0 + cc;
            const float swc = sw[cc], bsc = bs[cc];
#pragma unroll 4
            for (int i = 0; i < 32; i += 2) {
              const int rr = i + (lane >> 4);
              const float sxi = __shfl_sync(0xffffffffu, sx, rr);
              if (row0 + rr < p.M && col < p.N) {
                T* yo = y + (size_t)(row0 + rr) * p.ld_y + col;
                *yo = Elem<DT>::narrow(finish(p, xch[rr * 17 + o], sxi, swc, bsc,
                                              p.ep == VXG_EP_ADD_SCALED ? Elem<DT>::widen(*yo) : 0.0f));
              }
            }
            __syncwarp();
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // neither CTA leaves while the other may still signal its barriers
  if (warp == EPI_WARPS + 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, C::COLS);
  }
}

template <int DT, int BN>
vxg_status launch(const Params& p, cudaStream_t st) {
  int* status = device_status();
  VXG_ARG(status, "no CUDA device");
  CUtensorMap mx, mw;
  vxg_status r = make_tmap_2d_u8(&mx, p.x, (uint64_t)p.M, (uint64_t)p.K, (uint64_t)p.K, 128, SUB);
  if (r == VXG_OK) r = make_tmap_2d_u8(&mw, p.w, (uint64_t)p.N, (uint64_t)p.K, (uint64_t)p.K, BN / 2, SUB);
  if (r != VXG_OK) return r;
  const long long tiles = (long long)((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN);
  if (tiles > 0x3FFFFFFF) {
    set_error("M = %d x N = %d is more than one launch covers", p.M, p.N);
    return VXG_ERR_UNSUPPORTED;
  }
  const int e = DT == VXG_DT_F32 ? 8 : 16;
  const bool vec = p.N % e == 0 && (((uintptr_t)p.y | (uintptr_t)(p.ld_y * (long long)dtype_bytes(DT))) & 31) == 0;
  const void* k = vec ? (const void*)gemm_tc_kernel<DT, BN, true> : (const void*)gemm_tc_kernel<DT, BN, false>;
  if ((r = smem_attr(k, (int)Cfg<BN>::BYTES)) != VXG_OK) return r;
  const int grid = 2 * (int)std::min<long long>(tiles, sm_count() / 2);
  void* args[] = {&mx, &mw, const_cast<Params*>(&p), &status};
  VXG_CUDA(cudaLaunchKernel(k, dim3(grid), dim3(THREADS), args, Cfg<BN>::BYTES, st));
  note_launch();
  VXG_CUDA(cudaGetLastError());
  return VXG_OK;
}

}  // namespace tc

// Channels of a tile: rounds of tiles over the pairs of SMs times a stage's time, which was measured as 0.29, 0.39 and 0.72 us
// per 256 k for 64, 128 and 256 channels: near bn + 64.
static int pick_bn(const Params& p, int pairs) {  // pairs > 0
  int best = 256;
  long long cost = 0;
  for (int bn = 256; bn >= 64; bn /= 2) {
    const long long tiles = (long long)((p.M + tc::BM - 1) / tc::BM) * ((p.N + bn - 1) / bn);
    const long long c = (tiles + pairs - 1) / pairs * (bn + 64);
    if (bn == 256 || c < cost) best = bn, cost = c;
  }
  return best;
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
  VXG_ARG(aligned(16, x, w), "x and w must be 16-byte aligned");
  VXG_ARG(aligned(4, sx, sw, bias) && aligned(dtype_bytes(dtype), y), "an operand is not aligned to its elements");
  if (K % 16 != 0 || K >= 131072) {
    set_error("K = %d not supported (a multiple of 16 below 131072)", K);
    return VXG_ERR_UNSUPPORTED;
  }
  if (M > 0x7FFFFF00 || N > 0x7FFFFF00) {  // rows and channels of the last tile are counted in 31 bits
    set_error("M = %d x N = %d not supported (up to 2^31 - 256 each)", M, N);
    return VXG_ERR_UNSUPPORTED;
  }
  if (M == 0) return VXG_OK;
  i8::Params p = {x, sx, w, sw, bias, y, ld_y, M, N, K, (int)ep, ep_scale};
  vxg_status r = VXG_OK;
  with_dtype(dtype, [&](auto tag) {
    constexpr int DT = decltype(tag)::value;
    cudaStream_t st = (cudaStream_t)stream;
    if (M <= 64) {
      switch ((M + 7) / 8) {
        case 1: r = i8::launch_few<DT, 1>(p, st); break;
        case 2: r = i8::launch_few<DT, 2>(p, st); break;
        case 3: r = i8::launch_few<DT, 3>(p, st); break;
        case 4: r = i8::launch_few<DT, 4>(p, st); break;
        case 5: r = i8::launch_few<DT, 5>(p, st); break;
        case 6: r = i8::launch_few<DT, 6>(p, st); break;
        default: r = i8::launch_few<DT, 8>(p, st); break;
      }
    } else {
      const int bn = i8::pick_bn(p, std::max(1, sm_count() / 2));  // no GPU: the launch says so
      r = bn == 256 ? i8::tc::launch<DT, 256>(p, st)
          : bn == 128 ? i8::tc::launch<DT, 128>(p, st) : i8::tc::launch<DT, 64>(p, st);
    }
  });
  return r;
}
