// What the attention kernels over the paged cache share: tiles, the cut of all tiles' keys into equal shares, a share's
// walk from piece to piece, the join of the pieces, and the operand conversions.
#pragma once
#include <cuda_runtime.h>

#include <limits>

#include "common.h"
#include "dtype.cuh"
#include "kv_cache.cuh"
#include "ptx.cuh"
#include "wait.cuh"

namespace vxg {
namespace catt {

constexpr int MAX_PIECES = 2;  // partial results a CTA can leave: its first and its last

struct Params {
  vxg_kv_cache c;
  const void* q;
  void* out;
  long long ld_q, ld_out;
  const int* table;
  const int* len;
  const int* cu;
  float* part;      // [grid][2][MT][HD + 2]
  long long* rec;   // [grid][8]: begin, first unit and end of the tile it lies in, slot of the batch, KV head, all units, shares
  int* status;
  // in this order 16-row tiles spill 300 bytes and not 332 (heads of 128): 62 us against 73 for 16 x 4 queries over 4000
  int n_seq, max_pages, slots, total, share, causal, window, page_log2;
  float scale_log2;
  int negate;  // tcgen05: scale_log2 is positive and the queries are negated
};

struct Plan {
  int mt, grid, slots;
  size_t rec_bytes, part_bytes;
};

// Stands for the key scale of a page whose id is out of range: its keys take no part.
constexpr float NO_PAGE = -std::numeric_limits<float>::infinity();

constexpr int FEW_CTAS_8 = 3;  // CTAs an SM, tiles of up to 8 rows
// Tiles of up to 16 rows (cached_attention_few.cu).
vxg_status launch_few(const Params& p, const Plan& pl, int head_dim, int dtype, cudaStream_t st);
// 256-row tiles on tcgen05, f16 and bf16 queries (cached_attention_tc.cu).
vxg_status launch_tc(Params p, const Plan& pl, int head_dim, int dtype, cudaStream_t st);

// Rows of codes [n_pages * heads * page][head_dim], copied in boxes of a page or `most` rows.
inline vxg_status cache_map(CUtensorMap* map, const vxg_kv_cache& c, const int8_t* base, int most) {
  return make_tmap_2d_u8(map, base, (uint64_t)c.n_pages * c.heads * c.page, (uint64_t)c.head_dim, (uint64_t)c.head_dim,
                         (uint32_t)(c.page < most ? c.page : most), (uint32_t)c.head_dim);
}

// One tile: MT rows of sequence s; `cost` units per KV head (0: no such tile, 1 where no key is visible).
struct Tile {
  int s, n, L, q0;       // sequence, its queries, its length, its first stacked row
  int r0, rows;          // first (query, head) row and their number
  int kmin, kmax;        // keys [kmin, kmax) that any of its rows sees
  int blk0, nblk, cost;
};

__device__ __forceinline__ long long slot_base(const Params& p, int s, int MT) {
  return (long long)__ldg(p.cu + s) * p.share / MT + s;
}

__device__ __forceinline__ int find_seq(const Params& p, long long slot, int MT) {
  int lo = 0, hi = p.n_seq;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (slot_base(p, mid, MT) <= slot) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The tile of a slot; s is a lower bound of its sequence and moves up to it.
__device__ __forceinline__ Tile tile_at(const Params& p, long long slot, int& s, int MT, int BK) {
  while (s + 1 < p.n_seq && slot_base(p, s + 1, MT) <= slot) s++;
  Tile t;
  t.s = s;
  t.q0 = __ldg(p.cu + s);
  const long long n = (long long)__ldg(p.cu + s + 1) - t.q0;
  t.n = (int)n;
  t.L = __ldg(p.len + s);
  t.cost = 0;
  t.nblk = 0;
  const long long k = slot - slot_base(p, s, MT);
  if (n == 0 || k < 0) return t;
  if (n < 0 || t.q0 < 0 || t.q0 + n > p.total || t.L < 0 || t.L > (long long)p.max_pages * p.c.page) {
    atomicCAS(p.status + 1, 0, VXG_DEV_CACHE_INDEX);
    return t;
  }
  const long long r0 = k * MT, all = n * p.share;
  if (r0 >= all) return t;
  t.r0 = (int)r0;
  t.rows = (int)(all - r0 < MT ? all - r0 : MT);
  const int i0 = t.r0 / p.share, i1 = (t.r0 + t.rows - 1) / p.share;
  t.kmax = p.causal ? ::max(0, ::min(t.L, t.L - t.n + i1 + 1)) : t.L;
  t.kmin = 0;
  if (p.window > 0) t.kmin = (int)::max(0LL, (long long)t.L - t.n + i0 - p.window + 1);
  t.blk0 = t.kmin / BK;
  t.nblk = t.kmax > t.kmin ? (t.kmax + BK - 1) / BK - t.blk0 : 0;
  t.cost = ::max(1, t.nblk);
  return t;
}

// What a CTA works on: keys blk0 + off .. of tile t for KV head h, `left` units of its share to go (0: done).
struct Piece {
  Tile t;
  long long slot, left;
  int h, off, first;
  __device__ __forceinline__ int take() const { return (int)::min((long long)(t.cost - off), left); }
  // Moves on to the next piece. Ends the share where no tile is left, whatever the lengths have become meanwhile.
  __device__ __forceinline__ void next(const Params& p, int MT, int BK) {
    left -= take();
    off = 0;
    first = 0;
    if (left > 0 && ++h == p.c.heads) {
      h = 0;
      int s = t.s;
      do {
        if (++slot >= p.slots) {
          left = 0;
          return;
        }
        t = tile_at(p, slot, s, MT, BK);
      } while (t.cost == 0);
    }
  }
};

// The CTA's share of the line of all work units, as its first piece (left = 0: none): every thread of the block sums the
// costs of a run of slots, one scan over the block, then the thread in whose run the share begins walks it again.
template <int THREADS, int MT, int BK>
__device__ __forceinline__ void find_share(const Params& p, Piece* first_s) {
  constexpr int WARPS = THREADS / 32;
  __shared__ long long warp_tot[WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int KV = p.c.heads;
  if (tid == 0) first_s->left = 0;
  grid_launch_dependents();  // the join, which waits for this kernel's end
  const int per = (p.slots + THREADS - 1) / THREADS;
  const int sl0 = ::min(p.slots, tid * per), sl1 = ::min(p.slots, sl0 + per);
  const int first_seq = sl0 < sl1 ? find_seq(p, sl0, MT) : 0;
  long long mine = 0;
  {
    int s = first_seq;
    for (int i = sl0; i < sl1; i++) mine += tile_at(p, i, s, MT, BK).cost;
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_tot[warp] = incl;
  __syncthreads();
  long long before = 0, units = 0;
#pragma unroll
  for (int i = 0; i < WARPS; i++) {
    if (i < warp) before += warp_tot[i];
    units += warp_tot[i];
  }
  before += incl - mine;
  units *= KV;
  const long long parts = ::min((long long)gridDim.x, units);  // at least one unit a CTA
  if (blockIdx.x < parts) {
    const long long begin = units * blockIdx.x / parts, end = units * (blockIdx.x + 1) / parts;
    if (begin >= before * KV && begin < (before + mine) * KV) {
      long long at = before;
      int s = first_seq;
      for (int i = sl0; i < sl1; i++) {
        const Tile t = tile_at(p, i, s, MT, BK);
        if (begin < (at + t.cost) * KV) {
          const long long in = begin - at * KV;
          first_s->t = t;
          first_s->slot = i;
          first_s->h = (int)(in / t.cost);
          first_s->off = (int)(in % t.cost);
          first_s->left = end - begin;
          first_s->first = 1;
          long long* r = p.rec + blockIdx.x * 8;
          r[0] = begin, r[1] = begin - first_s->off, r[2] = r[1] + t.cost, r[3] = i, r[4] = first_s->h, r[5] = units, r[6] = parts;
          break;
        }
        at += t.cost;
      }
    }
  }
  __syncthreads();
  if (tid == 0 && first_s->left == 0) p.rec[blockIdx.x * 8] = -1;  // more CTAs than units
}

// One warp brings the share's blocks of BK keys: codes [K BK x HD][V BK x HD] by TMA, one box per page, into a ring of
// STAGES stages, and the scales of a block's 16-key pieces (four of K, four of V) beside it. Pages and scales are looked
// up 32 pages at a time. Pages that no row of the tile sees are not brought and have scale 0; a page whose id is out of range
// is not brought either, and has key scale NO_PAGE.
template <int HD, int MT, int BK, int STAGES>
__device__ __forceinline__ void produce(const Params& p, Piece w, const CUtensorMap& map_k, const CUtensorMap& map_v,
                                        uint8_t* smem, float* scales_s, uint64_t* full, uint64_t* empty) {
  const int lane = threadIdx.x & 31, KV = p.c.heads, PL = p.page_log2, P = 1 << PL;
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
              ks = NO_PAGE;
            } else {
              ks = __ldg(p.c.k_scales + (size_t)pid * KV + h);
              vs = __ldg(p.c.v_scales + (size_t)pid * KV + h);
            }
          }
        }
        const int st = it % STAGES;
        if (it >= STAGES && !wait_phase(empty + st, ((it / STAGES) - 1) & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN))
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
          uint8_t* dst = smem + st * (2 * BK * HD) + mypage * box * HD;
          tma_load_2d(dst, &map_k, 0, row, full + st);
          tma_load_2d(dst + BK * HD, &map_v, 0, row, full + st);
        }
      }
    }
  }
  // every copy that was issued lands before the block may end
  const int last = ::min(it, (int)STAGES);
  for (int i = it - last; i < it; i++)
    wait_phase(full + i % STAGES, (i / STAGES) & 1, p.status, VXG_DEV_TIMEOUT_CACHE_ATTN);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two int8 codes in bytes 0 and 2 of w -> two f16. Flipping a code's sign bit adds 128, and 0x64 above it makes the
// f16 1024 + 128 + code, exactly.
__device__ __forceinline__ uint32_t codes_biased(uint32_t w) { return (w & 0x00FF00FFu) ^ 0x64806480u; }
__device__ __forceinline__ uint32_t codes_to_f16(uint32_t w) {
  const uint32_t biased = codes_biased(w);
  const uint32_t off = 0x64806480u;  // 1152, 1152
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&biased), *reinterpret_cast<const __half2*>(&off));
  return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// sum plus the two f16 of h
__device__ __forceinline__ float add_f16(float sum, uint32_t h) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return sum + f.x + f.y;
}
// the part of (a, b) that pack_f16 leaves out
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return pack_f16(a - f.x, b - f.y);
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Joins the partial results of the tiles that span shares: block b looks at the tile in which share b begins, unless an
// earlier share begins inside it too; a warp takes a row.
template <int HD, int DT, int MT, int BK>
__global__ void __launch_bounds__(128) join_kernel(const Params p) {
  using T = typename Elem<DT>::type;
  constexpr int N = HD / 32;
  const int b = blockIdx.x + 1, lane = threadIdx.x & 31, r = blockIdx.y * 4 + (threadIdx.x >> 5);
  grid_wait();  // launched while the kernel in front still runs
  const long long* rec = p.rec + (size_t)b * 8;
  const long long begin = rec[0];
  if (begin < 0) return;
  const long long u0 = rec[1], u1 = rec[2], prev = rec[-8];
  if (u0 == begin || prev > u0) return;  // the share begins with its tile, or an earlier one joins it
  int s = 0;
  s = find_seq(p, rec[3], MT);
  const Tile t = tile_at(p, rec[3], s, MT, BK);
  if (r >= t.rows) return;
  const int h = (int)rec[4];
  auto at = [&](int j) {  // the part that share j left of this tile
    const int k = j == b - 1 && prev != u0 ? 1 : 0;
    return p.part + ((size_t)j * MAX_PIECES + k) * MT * (HD + 2) + (size_t)r * (HD + 2);
  };
  // shares b - 1 .. last hold parts of the tile: share j begins at floor(units j / parts), and last is the one of unit u1 - 1
  const int last = (int)((u1 * rec[6] + rec[5] - 1) / rec[5]) - 1;
  float m = -INFINITY;
  for (int j = b - 1 + lane; j <= last; j += 32) m = fmaxf(m, at(j)[0]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float mu = m == -INFINITY ? 0.0f : m;
  float l = 0.0f, acc[N] = {};
#pragma unroll 4
  for (int j = b - 1; j <= last; j++) {
    const float* x = at(j);
    const float f = ex2(x[0] - mu);
    l += f * x[1];
#pragma unroll
    for (int k = 0; k < N; k++) acc[k] += f * x[2 + 32 * k + lane];
  }
  const int rr = t.r0 + r;
  T* o = static_cast<T*>(p.out) + (long long)(t.q0 + rr / p.share) * p.ld_out +
         (long long)(h * p.share + rr % p.share) * HD;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int k = 0; k < N; k++) o[32 * k + lane] = Elem<DT>::narrow(acc[k] * inv);
}

// The join is put behind its kernel with the launch's latency hidden under it (its blocks wait for the kernel's end).
template <int HD, int DT, int MT, int BK>
vxg_status launch_join(const Params& p, const Plan& pl, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(pl.grid - 1, MT / 4);
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  VXG_CUDA(cudaLaunchKernelEx(&cfg, join_kernel<HD, DT, MT, BK>, p));
  note_launch(2);
  VXG_CUDA(cudaGetLastError());
  return VXG_OK;
}

}  // namespace catt
}  // namespace vxg
