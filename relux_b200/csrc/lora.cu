// A shared projection with low-rank adapters of many requests beside it: C[m] = x[m] W + f_s (x[m] A_s^T) B_s^T, s the adapter of the
// request that row m belongs to, or none.  A_s [rank][K], B_s [N][rank] in slots of two arrays, as checkpoints hold them (lora_A, lora_B).
//
// Two launches: lora_down_kernel, or lora_rows_kernel (lora_rows.cu) for tiles of one request's rows, takes t = x A_s^T, and rounds a float32 x to bf16 while it holds the
// rows; lora_gemm_kernel (lora_gemm.cu) is the projection, whose epilogue or last steps add t B_s^T.  (Of a row or two in one.)  Three where the rows are many and of so many requests that tiles of one request's rows would be mostly
// empty, or where the projection is not this call's: lora_down_kernel, the projection's GEMM (skinny_gemm_sm100_kernel, which may take t itself), and lora_up_kernel, which adds up
// the GEMM's pieces and, on the way out, t B_s^T.
// No tile of a product holds rows of one request and another's adapter: a product with that by zeros would carry its infinities and NaN over.
// In lora_down_kernel and lora_up_kernel rows are taken in groups of 16 of one adapter, wherever in the batch they lie: the host sorts the requests by adapter,
// so that an adapter is read once for 16 of its rows.  Bound: HBM, W and the adapters in use once, for few rows; for prompts the GEMM.
#include <algorithm>
#include <type_traits>
#include <vector>

#include "common.cuh"
#include "internal.h"
#include "lora.cuh"
#include "projection.cuh"
#include "tile_gemm.cuh"

namespace relux {

namespace {

constexpr int kLoraThreads = 256, kLoraWarps = kLoraThreads / 32;
constexpr int kUpCols = 32 * kLoraWarps;   // columns of a block of lora_up_kernel, 32 a warp
constexpr int kGroupRows = 16;
constexpr int kMostParts = 4;              // of K, of lora_down_kernel
constexpr int kMost = 1 << 30;                       // rows, k, n: counted in 32 bits, a tile past the last
constexpr int kMostGridY = 65535;
constexpr int kFewRows = 128, kSomeRows = 512;       // of up to so many rows a list names each
constexpr int kSmallList = 128, kLargeList = 1024;   // pieces of a list that travels as an argument of the launch

// The rows of a call (or of a part of it), in the order of their adapters, cut into groups of one adapter.
// Of few rows: every group and its rows.
template <int kCap>
struct RowList {
  static constexpr bool kNamesRows = true;
  struct Group {
    int32_t slot;        // adapter, or -1
    int16_t first, n;    // its rows' places
    int32_t used;        // which of the call's adapters, in order
  };
  Group group[kCap];
  int16_t row[kCap];
};
// Of many: a piece is a range of neighbouring rows of one adapter, a run all the pieces of one; groups are cut within runs, all but a run's last of full size.
template <int kCap>
struct RunList {
  static constexpr bool kNamesRows = false;
  int32_t n_pieces, n_runs;
  int32_t at[kCap + 1];      // first place, in this order, of a piece
  int32_t row[kCap];         // its first row
  int32_t slot[kCap];        // of a run: adapter, or -1
  int32_t run_at[kCap + 1];  // first place of a run
  int32_t group[kCap + 1];   // first group of a run
};
// The last of n ascending entries that is no more than v.
__host__ __device__ __forceinline__ int last_up_to(const int32_t* a, int n, int v) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a[mid] <= v) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// Rows of a group to shared memory (-1: none), and its adapter.  By all threads; a barrier follows.
template <int kCap>
__device__ __forceinline__ int used_of(const RowList<kCap>& list, int group) { return list.group[group].used; }
template <int kCap>
__device__ __forceinline__ int group_rows(const RowList<kCap>& list, int group, int32_t* rows) {
  const auto g = list.group[group];
  if (threadIdx.x < kGroupRows) rows[threadIdx.x] = (int)threadIdx.x < g.n ? list.row[g.first + threadIdx.x] : -1;
  return g.slot;
}
template <int kCap>
__device__ __forceinline__ int group_rows(const RunList<kCap>& list, int group, int32_t* rows) {
  const int run = last_up_to(list.group, list.n_runs, group);
  const int first = list.run_at[run] + (group - list.group[run]) * kGroupRows, end = list.run_at[run + 1];
  if (threadIdx.x < kGroupRows) {
    const int v = first + threadIdx.x;
    int r = -1;
    if (v < end) {
      const int piece = last_up_to(list.at, list.n_pieces, v);
      r = list.row[piece] + v - list.at[piece];
    }
    rows[threadIdx.x] = r;
  }
  return list.slot[run];
}

struct DownParams {
  const void* x;
  uint16_t* x_bf16;       // float32 x: the projection's operand [M][K], in halves [2][M][K]; or nullptr: there is no projection
  const uint16_t* a;      // [slots][rank][K]
  float* t;               // [M][rank], without factors
  int32_t M, K, rank;
};

// t[row][r] = sum over k of x[row][k] A_s[r][k].  grid (groups, parts of K, kSlice-th parts of the rank), the parts of K a cluster, 8 warps that take 32 k each in turn.  mma.sync: a group is a
// handful of rows, and the bound is reading A_s and x.  A thread's eight neighbouring k of a row are the pairs of two k-slices, in the same order for x and A_s.
enum Rows { kBf16, kRounded, kSplit };   // x: bf16; float32, rounded; float32, in two halves; each for the projection too where there is one
template <int kSlice, Rows kX, class List>
__global__ void __launch_bounds__(kLoraThreads, 2) lora_down_kernel(const DownParams p, const __grid_constant__ List list) {
  constexpr int kTiles = kSlice / 8;
  constexpr int kSlab = kGroupRows * kSlice;
  extern __shared__ __align__(16) float slabs[];   // [warp][16][kSlice], then what the other parts send to the first one
  __shared__ int32_t rows[kGroupRows];
  const int slot = group_rows(list, blockIdx.x, rows);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int steps = (p.K + 31) / 32, s0 = (int)((int64_t)steps * blockIdx.y / gridDim.y), s1 = (int)((int64_t)steps * (blockIdx.y + 1) / gridDim.y);
  const int r0 = blockIdx.z * kSlice;
  const uint16_t* const a = p.a + ((size_t)max(slot, 0) * p.rank + r0) * p.K;
  const bool rounds = kX != kBf16 && p.x_bf16 && r0 == 0;
  if (slot >= 0)   // the adapter's first pieces to L2, while the launch before this one ends (a prefetch returns no data, so it may be early)
    for (int s = s0 + warp; s < min(s1, s0 + 4 * kLoraWarps); s += kLoraWarps) {
      const int k = s * 32 + 8 * t;
      if (t == 0 && k < p.K)
#pragma unroll
        for (int j = 0; j < kTiles; j++) asm volatile("prefetch.global.L2 [%0];" ::"l"(a + (size_t)(8 * j + g) * p.K + k));
    }
  // waits before it releases: the projection behind it may read its weights early (launch_chained, head of a chain)
  chain_wait();
  chain_release();
  if (slot < 0 && !rounds) return;   // (the same in all parts)
  if (slot >= 0 && gridDim.y > 1) cluster_arrive();
  __syncthreads();
  const int32_t r[2] = {rows[g], rows[8 + g]};
  float acc[kTiles][4];
#pragma unroll
  for (int j = 0; j < kTiles; j++)
#pragma unroll
    for (int i = 0; i < 4; i++) acc[j][i] = 0.f;
  const uint4 none = make_uint4(0u, 0u, 0u, 0u);

#pragma unroll(kSlice <= 32 ? 4 : 1)
  for (int s = s0 + warp; s < s1; s += kLoraWarps) {
    const int k = s * 32 + 8 * t;
    const bool in = k < p.K;   // K is a multiple of 8
    uint4 x[2], low[2], w[kTiles];   // low: of float32 rows that are not rounded for a projection what bf16 leaves
    if (slot >= 0)
#pragma unroll
      for (int j = 0; j < kTiles; j++) w[j] = in ? load_chained(reinterpret_cast<const uint4*>(a + (size_t)(8 * j + g) * p.K + k)) : none;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const size_t at = (size_t)max(r[h], 0) * p.K + k;
      const bool there = in && r[h] >= 0;
      if constexpr (kX == kBf16) {
        x[h] = there ? load_chained(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.x) + at)) : none;
      } else {
        const float4* src = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.x) + at);
        const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f), u = there ? load_chained(src) : zero, v = there ? load_chained(src + 1) : zero;
        if constexpr (kX == kRounded) {
          x[h] = make_uint4(round_bf16x2(u.x, u.y), round_bf16x2(u.z, u.w), round_bf16x2(v.x, v.y), round_bf16x2(v.z, v.w));
        } else {
          uint2 hi[2], lo[2];
          split_halves(u, 1.f, hi[0], lo[0]);
          split_halves(v, 1.f, hi[1], lo[1]);
          x[h] = make_uint4(hi[0].x, hi[0].y, hi[1].x, hi[1].y);
          low[h] = make_uint4(lo[0].x, lo[0].y, lo[1].x, lo[1].y);
        }
        if (there && rounds) {
          *reinterpret_cast<uint4*>(p.x_bf16 + at) = x[h];
          if constexpr (kX == kSplit) *reinterpret_cast<uint4*>(p.x_bf16 + (size_t)p.M * p.K + at) = low[h];
        }
      }
    }
    if (slot >= 0) {
      auto multiply = [&](const uint4 (&y)[2]) {
        const uint32_t a0[4] = {y[0].x, y[1].x, y[0].y, y[1].y}, a1[4] = {y[0].z, y[1].z, y[0].w, y[1].w};
#pragma unroll
        for (int j = 0; j < kTiles; j++) {
          mma_bf16_16816(acc[j], a0, w[j].x, w[j].y);
          mma_bf16_16816(acc[j], a1, w[j].z, w[j].w);
        }
      };
      multiply(x);
      if constexpr (kX == kSplit) multiply(low);
    }
  }
  if constexpr (kX != kBf16) fence_chained_writes();
  if (slot < 0) return;
  // the warps' sums, then the parts', in their order
  const int parts = gridDim.y, part = blockIdx.y;
  float* const mine = slabs + warp * kSlab;
#pragma unroll
  for (int j = 0; j < kTiles; j++) {
    *reinterpret_cast<float2*>(mine + g * kSlice + 8 * j + 2 * t) = make_float2(acc[j][0], acc[j][1]);
    *reinterpret_cast<float2*>(mine + (8 + g) * kSlice + 8 * j + 2 * t) = make_float2(acc[j][2], acc[j][3]);
  }
  __syncthreads();
  constexpr int kEach = (kSlab / 4 + kLoraThreads - 1) / kLoraThreads;
  float4 sum[kEach];
#pragma unroll
  for (int e = 0; e < kEach; e++) {
    const int i = threadIdx.x + e * kLoraThreads;
    if (i >= kSlab / 4) continue;
    sum[e] = reinterpret_cast<const float4*>(slabs)[i];
#pragma unroll
    for (int w = 1; w < kLoraWarps; w++) {
      const float4 v = reinterpret_cast<const float4*>(slabs + w * kSlab)[i];
      sum[e].x += v.x; sum[e].y += v.y; sum[e].z += v.z; sum[e].w += v.w;
    }
  }
  if (parts > 1) {
    float4* const inbox = reinterpret_cast<float4*>(slabs + kLoraWarps * kSlab);
    cluster_wait();   // the first part has begun
    if (part > 0)
#pragma unroll
      for (int e = 0; e < kEach; e++) {
        const int i = threadIdx.x + e * kLoraThreads;
        if (i >= kSlab / 4) continue;
        const uint32_t to = mapa_u32(smem_u32(inbox + (part - 1) * (kSlab / 4) + i), 0u);
        store_cluster(to, __float_as_uint(sum[e].x));
        store_cluster(to + 4, __float_as_uint(sum[e].y));
        store_cluster(to + 8, __float_as_uint(sum[e].z));
        store_cluster(to + 12, __float_as_uint(sum[e].w));
      }
    cluster_arrive();
    cluster_wait();
    if (part > 0) return;
#pragma unroll
    for (int e = 0; e < kEach; e++) {
      const int i = threadIdx.x + e * kLoraThreads;
      if (i >= kSlab / 4) continue;
      for (int k = 0; k < parts - 1; k++) {
        const float4 v = inbox[k * (kSlab / 4) + i];
        sum[e].x += v.x; sum[e].y += v.y; sum[e].z += v.z; sum[e].w += v.w;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < kEach; e++) {
    const int i = threadIdx.x + e * kLoraThreads;
    if (i >= kSlab / 4) continue;
    const int row = rows[4 * i / kSlice];
    if (row < 0) continue;
    const size_t to = (size_t)row * p.rank + r0 + 4 * i % kSlice;
    *reinterpret_cast<float4*>(p.t + to) = sum[e];
  }
}

// The GEMM's blocks of rows come in turns; t comes in pieces, from the GEMM; any of these, every row may be two of the GEMM's, M apart, and the columns those of a further launch (of its own: one sum more
// for the first column took six registers, and 64 rows x 4096 x 6144, rank 16, 23.7 us for 22.4).
enum Up { kPlain, kInTurns, kTInPieces, kAny };
struct UpParams {
  const float* part;      // the GEMM's pieces [piece][M][N]; nullptr: no shared projection
  int32_t halves, first_block;   // kAny: the GEMM's rows of a row less one; block of 256 columns that this launch begins with
  GemmRanges rg;
  const float* t;         // [M][rank], or (t_parts) in as many pieces [M][t_cols], of every adapter in use for every row
  int32_t t_parts, t_cols;
  const uint16_t* b;      // [slots][N][rank]
  const float* factors;   // [slots], or nullptr: ones
  void* out;
  int32_t M, N, out_bf16, adds;   // adds: to what out holds
};

// out[row][n] = sum of the GEMM's pieces (+ what out holds) + f_s sum over r of t[row][r] B_s[n][r].  grid (groups, blocks of 256 columns), 32 columns a warp: its four
// tiles of the MMA take columns 8 (n / 2) + 2 tile + n % 2, so that a thread's results of a row are eight neighbours.  t is split into two bf16 halves, hi and lo:
// 16 bits of it, where the projection's x has eight.
template <int kRank, Up kUp, class List>
__global__ void __launch_bounds__(kLoraThreads) lora_up_kernel(const UpParams p, const __grid_constant__ List list) {
  constexpr int kStride = kRank + 8, kSlices = (kRank + 31) / 32;   // k slices of 32 (one, of 8 or 16, for small ranks)
  __shared__ __align__(16) uint16_t t_hi[kGroupRows * kStride], t_lo[kGroupRows * kStride];
  __shared__ int32_t rows[kGroupRows];
  constexpr bool kTurns = kUp == kInTurns || kUp == kAny, kFew = kUp == kTInPieces || kUp == kAny;
  chain_release();
  const int slot = group_rows(list, blockIdx.x, rows);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = ((kUp == kAny ? p.first_block : 0) + (int)blockIdx.y) * kUpCols + warp * 32, n = n0 + 8 * t;
  // adapters were complete before the chain's head began: read ahead of the launches before this one
  uint4 w[kSlices][4];
  float factor = 1.f;
  if (slot >= 0) {
    const uint16_t* const b = p.b + (size_t)slot * p.N * kRank;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int col = n0 + 8 * (g >> 1) + 2 * j + (g & 1);
      const uint16_t* src = b + (size_t)min(col, p.N - 1) * kRank;
#pragma unroll
      for (int s = 0; s < kSlices; s++) {
        w[s][j] = make_uint4(0u, 0u, 0u, 0u);
        if constexpr (kRank >= 32) {
          w[s][j] = load_chained(reinterpret_cast<const uint4*>(src + 32 * s + 8 * t));
        } else if constexpr (kRank == 16) {
          const uint2 v = load_chained(reinterpret_cast<const uint2*>(src + 4 * t));
          w[s][j].x = v.x;
          w[s][j].y = v.y;
        } else {
          w[s][j].x = load_chained(reinterpret_cast<const uint32_t*>(src + 2 * t));
        }
      }
    }
    if (p.factors) factor = load_chained(p.factors + slot);
  }
  __syncthreads();
  chain_wait();
  // the shared projection's sums, and what out holds, are where the adapter's begin
  const int col_tile = n / kGemmTileCols;
  const int same = kTurns || !p.part ? 1 : p.rg.pieces(col_tile);
  float acc[4][4];
  auto add = [&](int h, const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      acc[j][2 * h] += v[2 * j];
      acc[j][2 * h + 1] += v[2 * j + 1];
    }
  };
  auto add_f32 = [&](int h, const float* src) {
    const float4 a = load_chained(reinterpret_cast<const float4*>(src)), b = load_chained(reinterpret_cast<const float4*>(src) + 1);
    const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    add(h, v);
  };
#pragma unroll
  for (int j = 0; j < 4; j++)
#pragma unroll
    for (int i = 0; i < 4; i++) acc[j][i] = 0.f;
#pragma unroll
  for (int h = 0; h < 2; h++) {   // (the first pieces of both rows are on their way together)
    const int row = rows[8 * h + g];
    if (p.part && row >= 0 && n < p.N) add_f32(h, p.part + (size_t)row * p.N + n);
  }
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int row = rows[8 * h + g];
    if (row < 0 || n >= p.N) continue;
    const size_t at = (size_t)row * p.N + n;
    if constexpr (kUp == kAny) {
      for (int o = 0; o <= p.halves; o++) {
        const int pieces = p.part ? p.rg.pieces(p.rg.tile_of(col_tile, row + o * p.M)) : 1;
        for (int s = o ? 0 : 1; s < pieces; s++) add_f32(h, p.part + ((size_t)s * (1 + p.halves) + o) * p.M * p.N + at);
      }
    } else {
      const int pieces = !p.part ? 1 : kTurns ? p.rg.pieces(p.rg.tile_of(col_tile, row)) : same;
#pragma unroll 2
      for (int s = 1; s < pieces; s++) add_f32(h, p.part + (size_t)s * p.M * p.N + at);
    }
    if (p.adds) {
      if (p.out_bf16) {
        const uint4 a = load_chained(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.out) + at));
        const float v[8] = {bf16_lo(a.x), bf16_hi(a.x), bf16_lo(a.y), bf16_hi(a.y), bf16_lo(a.z), bf16_hi(a.z), bf16_lo(a.w), bf16_hi(a.w)};
        add(h, v);
      } else {
        add_f32(h, reinterpret_cast<const float*>(p.out) + at);
      }
    }
  }
  if (slot >= 0) {
    for (int i = threadIdx.x; i < kGroupRows * kRank / 4; i += kLoraThreads) {
      const int at = 4 * i / kRank, r = 4 * i % kRank, row = rows[at];
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      bool whole = true;
      if constexpr (List::kNamesRows && kFew) {
        whole = kUp == kAny && !p.t_parts;
        if (row >= 0 && !whole) {
          const float* src = p.t + (size_t)row * p.t_cols + used_of(list, blockIdx.x) * kRank + r;
#pragma unroll 8
          for (int s = 0; s < p.t_parts; s++) {
            const float4 u = load_chained(reinterpret_cast<const float4*>(src + (size_t)s * p.M * p.t_cols));
            v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
          }
        }
      }
      if (row >= 0 && whole) v = load_chained(reinterpret_cast<const float4*>(p.t + (size_t)row * kRank + r));
      uint2 hi, lo;
      split_halves(v, factor, hi, lo);
      *reinterpret_cast<uint2*>(t_hi + at * kStride + r) = hi;
      *reinterpret_cast<uint2*>(t_lo + at * kStride + r) = lo;
    }
    __syncthreads();
#pragma unroll
    for (int half = 0; half < 2; half++) {
      const uint16_t* const src = half ? t_lo : t_hi;
#pragma unroll
      for (int s = 0; s < kSlices; s++) {
        const uint16_t* const row0 = src + g * kStride;
        const uint16_t* const row1 = row0 + 8 * kStride;
        if constexpr (kRank >= 32) {
          const uint4 u = *reinterpret_cast<const uint4*>(row0 + 32 * s + 8 * t), v = *reinterpret_cast<const uint4*>(row1 + 32 * s + 8 * t);
          const uint32_t a0[4] = {u.x, v.x, u.y, v.y}, a1[4] = {u.z, v.z, u.w, v.w};
#pragma unroll
          for (int j = 0; j < 4; j++) {
            mma_bf16_16816(acc[j], a0, w[s][j].x, w[s][j].y);
            mma_bf16_16816(acc[j], a1, w[s][j].z, w[s][j].w);
          }
        } else {
          uint32_t a0[4];
          if constexpr (kRank == 16) {
            const uint2 u = *reinterpret_cast<const uint2*>(row0 + 4 * t), v = *reinterpret_cast<const uint2*>(row1 + 4 * t);
            a0[0] = u.x; a0[1] = v.x; a0[2] = u.y; a0[3] = v.y;
          } else {
            a0[0] = *reinterpret_cast<const uint32_t*>(row0 + 2 * t);
            a0[1] = *reinterpret_cast<const uint32_t*>(row1 + 2 * t);
            a0[2] = a0[3] = 0u;
          }
#pragma unroll
          for (int j = 0; j < 4; j++) mma_bf16_16816(acc[j], a0, w[s][j].x, w[s][j].y);
        }
      }
    }
  }
  if (n >= p.N) return;   // N is a multiple of 8
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int row = rows[8 * h + g];
    if (row < 0) continue;
    const size_t at = (size_t)row * p.N + n;
    if (p.out_bf16) {
      *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.out) + at) =
          make_uint4(round_bf16x2(acc[0][2 * h], acc[0][2 * h + 1]), round_bf16x2(acc[1][2 * h], acc[1][2 * h + 1]), round_bf16x2(acc[2][2 * h], acc[2][2 * h + 1]),
                     round_bf16x2(acc[3][2 * h], acc[3][2 * h + 1]));
    } else {
      float4* dst = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at);
      dst[0] = make_float4(acc[0][2 * h], acc[0][2 * h + 1], acc[1][2 * h], acc[1][2 * h + 1]);
      dst[1] = make_float4(acc[2][2 * h], acc[2][2 * h + 1], acc[3][2 * h], acc[3][2 * h + 1]);
    }
  }
  fence_chained_writes();
}

// ---- the host's half ----
struct Request {
  int32_t row, n, slot;
};
// Neighbouring requests of one adapter as one, in row order.
std::vector<Request> merged_requests(int n_seqs, const int32_t* n_rows, const int32_t* adapter) {
  std::vector<Request> v;
  int row = 0;
  for (int i = 0; i < n_seqs; i++) {
    const int n = n_rows ? n_rows[i] : 1;
    if (!n) continue;
    if (!v.empty() && v.back().slot == adapter[i]) v.back().n += n;
    else v.push_back(Request{row, n, adapter[i]});
    row += n;
  }
  return v;
}
bool by_slot(const Request& a, const Request& b) { return a.slot < b.slot; }
// The list of all of them, or of some; returns the groups.
template <int kCap>
int make_list(std::vector<Request> r, RowList<kCap>* list) {
  std::stable_sort(r.begin(), r.end(), by_slot);
  int groups = 0, at = 0, used = -1;
  for (const Request& q : r)
    for (int i = 0; i < q.n; i++, at++) {
      if (!groups || list->group[groups - 1].slot != q.slot || list->group[groups - 1].n == kGroupRows) {
        used += q.slot >= 0 && (!groups || list->group[groups - 1].slot != q.slot);
        list->group[groups++] = {q.slot, (int16_t)at, 0, used};
      }
      list->group[groups - 1].n++;
      list->row[at] = (int16_t)(q.row + i);
    }
  return groups;
}
template <int kCap>
int make_list(std::vector<Request> r, RunList<kCap>* list) {
  std::stable_sort(r.begin(), r.end(), by_slot);
  list->n_pieces = (int)r.size();
  list->n_runs = 0;
  int at = 0, groups = 0;
  for (size_t i = 0; i < r.size(); i++) {
    if (i == 0 || r[i].slot != r[i - 1].slot) {
      if (i) groups += (at - list->run_at[list->n_runs - 1] + kGroupRows - 1) / kGroupRows;
      list->slot[list->n_runs] = r[i].slot;
      list->run_at[list->n_runs] = at;
      list->group[list->n_runs++] = groups;
    }
    list->at[i] = at;
    list->row[i] = r[i].row;
    at += r[i].n;
  }
  groups += (at - list->run_at[list->n_runs - 1] + kGroupRows - 1) / kGroupRows;
  list->at[r.size()] = list->run_at[list->n_runs] = at;
  list->group[list->n_runs] = groups;
  return groups;
}

template <int kSlice, class List>
int32_t launch_down(Pool* p, const DownParams& prm, const List& list, int groups, int parts, Rows kind) {
  const size_t smem = (size_t)(kLoraWarps + parts - 1) * kGroupRows * kSlice * sizeof(float);
  static_assert((kLoraWarps + kMostParts - 1) * kGroupRows * kSlice * sizeof(float) <= 48 << 10, "more shared memory than a launch has without asking");
  auto go = [&](auto kernel) -> int32_t {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)groups, (unsigned)parts, (unsigned)(prm.rank / kSlice));
    cfg.blockDim = dim3(kLoraThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = p->dev->stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = at[0].val.clusterDim.z = 1;
    at[0].val.clusterDim.y = (unsigned)parts;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = p->tune.get(RELUX_TUNE_CHAINED_LAUNCHES) != 0 ? 2 : 1;
    RELUX_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, prm, list));
    count_launch(p->dev);
    return RELUX_OK;
  };
  return kind == kBf16 ? go(lora_down_kernel<kSlice, kBf16, List>) : kind == kRounded ? go(lora_down_kernel<kSlice, kRounded, List>) : go(lora_down_kernel<kSlice, kSplit, List>);
}
template <int kRank, class List>
int32_t launch_up(Pool* p, UpParams prm, const List& list, int groups) {
  const bool chained = p->tune.get(RELUX_TUNE_CHAINED_LAUNCHES) != 0;
  const int blocks = (prm.N + kUpCols - 1) / kUpCols;
  for (prm.first_block = 0; prm.first_block < blocks; prm.first_block += kMostGridY) {
    const dim3 grid((unsigned)groups, (unsigned)std::min(blocks - prm.first_block, kMostGridY));
    auto go = [&](auto kernel) -> int32_t {
      RELUX_CUDA_TRY(launch_chained(chained, kernel, grid, dim3(kLoraThreads), 0, p->dev->stream, prm, list));
      return RELUX_OK;
    };
    int32_t rc;
    if (prm.halves || blocks > kMostGridY)
      rc = go(lora_up_kernel<kRank, kAny, List>);
    else if constexpr (std::is_same_v<List, RowList<kFewRows>>)   // one block of rows
      rc = prm.t_parts ? go(lora_up_kernel<kRank, kTInPieces, List>) : go(lora_up_kernel<kRank, kPlain, List>);
    else
      rc = prm.part && prm.rg.in_turns() ? go(lora_up_kernel<kRank, kInTurns, List>) : go(lora_up_kernel<kRank, kPlain, List>);
    if (rc) return rc;
    count_launch(p->dev);
  }
  return RELUX_OK;
}

// A call's lists, one launch each: of every row, or by parts of up to kLargeList requests.
template <class Launch>
int32_t for_lists(int M, const std::vector<Request>& requests, Launch launch) {
  if (M <= kFewRows) {
    RowList<kFewRows> list;
    return launch(list, make_list(requests, &list));
  }
  if (M <= kSomeRows) {
    RowList<kSomeRows> list;
    return launch(list, make_list(requests, &list));
  }
  for (size_t i = 0; i < requests.size(); i += kLargeList) {
    std::vector<Request> part(requests.begin() + i, requests.begin() + std::min(requests.size(), i + kLargeList));
    int32_t rc;
    if (part.size() <= kSmallList) {
      RunList<kSmallList> list;
      rc = launch(list, make_list(part, &list));
    } else {
      RunList<kLargeList> list;
      rc = launch(list, make_list(part, &list));
    }
    if (rc) return rc;
  }
  return RELUX_OK;
}
// Calls f with the rank as a constant.
template <class F>
int32_t with_rank(int rank, F f) {
  switch (rank) {
    case 8: return f(std::integral_constant<int, 8>());
    case 16: return f(std::integral_constant<int, 16>());
    case 32: return f(std::integral_constant<int, 32>());
    case 64: return f(std::integral_constant<int, 64>());
    default: return f(std::integral_constant<int, 128>());
  }
}
// beside: the launch behind it streams W meanwhile.
int32_t run_down(Pool* p, Rows kind, const DownParams& prm, const std::vector<Request>& requests, bool beside) {
  return for_lists(prm.M, requests, [&](const auto& list, int groups) {
    using List = std::decay_t<decltype(list)>;
    // parts of K: two blocks an SM where groups are full, of 1024 k at least, four at most and beside another launch two: larger clusters start late (64 bf16 rows x 4096 x 6144, rank
    // 16: 23.3 us in one part, 19.5 in four, 20.7 in eight; 300 rows x 4096: 29.5 in four, 35.0 in eight; beside lora_gemm_kernel, 12 rows x 4096: 12.0 in two, 13.2 in four, 13.8 in eight).
    // By the call's sizes alone: a row's sums do not depend on the adapters of the others.
    const int parts = std::max(1, std::min({beside ? 2 : kMostParts, 2 * p->dev->sm_count / ((prm.M + kGroupRows - 1) / kGroupRows), prm.K / 1024}));
    // slices of the rank: of few rows 16, so that more SMs read an adapter (one row of rank 128 x 4096 x 4096: 23 us with the whole rank a block); of many 64, since
    // every slice reads x again
    if (prm.rank == 8) return launch_down<8>(p, prm, list, groups, parts, kind);
    if constexpr (List::kNamesRows) {
      return launch_down<16>(p, prm, list, groups, parts, kind);
    } else {
      if (prm.rank == 16) return launch_down<16>(p, prm, list, groups, parts, kind);
      if (prm.rank == 32) return launch_down<32>(p, prm, list, groups, parts, kind);
      return launch_down<64>(p, prm, list, groups, parts, kind);
    }
  });
}

// Tiles of rows of one adapter for lora_rows_kernel and lora_gemm_kernel; false where they are too many, or less than seven tenths full (16 requests of 80 rows, rank 16,
// 4096 x 4096, 62 % full: 58.1 us in tiles, 54.2 without; of 100 rows, 78 %: 61.1 and 67.8; one request of 1024 rows, rank 64: 38.0 and 53.3).
bool make_tiles(int M, const std::vector<Request>& requests, LoraTiles* tiles) {
  int64_t n = 0;
  for (const Request& r : requests) n += (r.n + 127) / 128;
  if (M <= 128 || n > kMaxLoraTiles || 7 * 128 * n > 10 * (int64_t)M) return false;
  tiles->n = 0;
  for (const Request& r : requests)
    for (int i = 0; i < r.n; i += 128) {
      tiles->row[tiles->n] = r.row + i;
      tiles->rows[tiles->n] = (int16_t)std::min(128, r.n - i);
      tiles->slot[tiles->n++] = r.slot;
    }
  return true;
}

// The form of a call, by its sizes (and, for tiles, by how its rows are spread over requests), and what it takes of the layers' scratch.
enum class Form { kOneLaunch, kFewRows, kTiles, kColumns, kGroups };
struct LoraPlan {
  Form form;
  bool halves;      // kGroups: the projection is of rows in two halves, one behind the others
  std::vector<Request> requests;
  LoraTiles tiles;
  int t_parts;      // kColumns
  size_t t_bytes, bytes;
};
void plan_lora(const Pool* p, const relux_matmul_lora_args* a, LoraPlan* plan) {
  const bool x_bf16 = a->x_dtype == RELUX_DTYPE_BF16;
  const int sms = p->dev->sm_count;
  plan->requests = merged_requests(a->n_seqs, a->n_rows, a->adapter);
  plan->t_bytes = (size_t)a->m * a->rank * sizeof(float);   // or two halves of two bytes
  plan->halves = false;
  // few rows of small rank: what the epilogue's warps can do while W streams (bf16 rows x 4096 x 4096, rank 16, with lora_down_kernel in eight parts of K both: one row 11.6 us so and
  // 13.3 with lora_up_kernel, 16 rows 13.1 and 15.5; rank 64, 16 rows: 22.4 and 19.5).  float32 rows are split there, by every CTA for itself: one row 13.2 and 13.2, with most of
  // their rounding less; 16 rows x 4096 x 14336 31.4 and 26.0.
  if (a->w && a->m <= (x_bf16 ? kNarrowRows : 8) && a->m * a->rank <= (x_bf16 ? kNarrowSums : kNarrowSums / 2)) {
    // In one launch, every CTA of which takes t over its part of K: of so few sums, and so few tiles that read the same pieces of an adapter at once (one row, rank 16, x 4096 x 1024
    // 6.6 us so, 7.9 in two; x 256 x 4096 4.4 and 5.6; x 4096 x 4096 10.3 and 10.5; rank 32 10.9 and 10.75; rank 16 x 4096 x 14336 27.9 and 21.9).
    const bool one = a->m * a->rank <= kOneT && (a->n - 1) / kRowsOp + 1 <= sms / 4;
    plan->form = one ? Form::kOneLaunch : Form::kFewRows;
    plan->bytes = one ? 0 : plan->t_bytes;
    return;
  }
  // float32 rows in two halves, as twice as many rows of the projection: what it is for is the bits (bf16 results, against 64 bits: 1.65e-3 off, rounded rows 2.4e-3).  No form of its own:
  // rank 16, 9 rows x 4096 x 4096 22.8 us (rounded 17.7), 64 x 4096 x 6144 34.0 (25.4), 700 x 4096 x 4096 64 (43); 8192 rows, rank 8, 565 (239).
  if (a->w && !x_bf16 && a->x_halves) {
    plan->form = Form::kGroups;
    plan->halves = true;
    plan->bytes = layer_scratch_bytes(2 * a->m, a->k, a->n, plan->t_bytes, true);
    return;
  }
  if (a->w && (int64_t)a->n_slots * std::max(a->n, a->rank) < (int64_t)1 << 31 && make_tiles(a->m, plan->requests, &plan->tiles)) {
    plan->form = Form::kTiles;
    plan->bytes = (x_bf16 ? 0 : pad256((size_t)a->m * a->k * 2)) + plan->t_bytes;
    return;
  }
  // Of up to 128 rows t may be further columns of the projection, all rows with every adapter in use (AdapterColumns): their bytes are the adapters', read once, and a launch less.  It
  // pays where they are few, or large: of small rank a step of adapters is more boxes than a step of W (bf16 rows x 4096 x 4096: 64 rows, 16 slots of rank 16 15.6 us so, 18.1 by
  // lora_down_kernel; 32 rows, rank 128 29.9 and 36.3; 64 float32 rows, 48 slots of rank 64 29.2 and 31.2; 20, rank 16, 20 slots 15.2 and 15.7; 64 rows x 6144, 48 slots, rank 16 24.6
  // and 19.5, rank 32 25.3 and 22.7; 40 rows x 1024 x 1024, 8 slots of rank 8 13.4 and 9.7).  Parts of K by the call's sizes alone, so that a row's sums do not depend on the
  // adapters of the others.
  const int most = std::min(a->m, a->n_slots);
  const bool columns = a->w && a->m <= kFewRows && a->k >= 2048 && (most * a->rank <= 320 || (a->rank >= 64 && most * a->rank >= 2048));
  const int tiles_of_t = (std::min(most, kFewRows) * a->rank + 127) / 128;
  plan->form = columns ? Form::kColumns : Form::kGroups;
  plan->t_parts = std::min({8, 2 * sms / tiles_of_t, (a->k + 63) / 64 / 4});
  plan->t_bytes *= columns ? (size_t)most * plan->t_parts : 1;
  plan->bytes = layer_scratch_bytes(a->m, a->k, a->w ? a->n : 0, plan->t_bytes, true);
}

}  // namespace

int32_t do_matmul_lora(Pool* p, const relux_matmul_lora_args* a) {
  if (!a || !a->x || !a->lora_a || !a->lora_b || !a->adapter || !a->out) { set_error("nil argument"); return RELUX_ERR_INVALID_ARG; }
  if (a->m <= 0 || a->k <= 0 || a->n <= 0 || a->n_seqs <= 0 || a->n_slots <= 0) {
    set_error("matmul_lora: M=%d K=%d N=%d, %d requests and %d slots must be positive", a->m, a->k, a->n, a->n_seqs, a->n_slots);
    return RELUX_ERR_INVALID_ARG;
  }
  auto dtype_ok = [](int32_t t) { return t == RELUX_DTYPE_F32 || t == RELUX_DTYPE_BF16; };
  if (!dtype_ok(a->x_dtype) || !dtype_ok(a->out_dtype)) { set_error("bad dtype flag"); return RELUX_ERR_INVALID_ARG; }
  for (int i = 0; i < 2; i++)
    if (a->reserved[i]) { set_error("reserved fields must be zero"); return RELUX_ERR_INVALID_ARG; }
  if (a->x_halves != 0 && a->x_halves != 1) { set_error("matmul_lora: x_halves=%d must be 0 or 1", a->x_halves); return RELUX_ERR_INVALID_ARG; }
  int64_t rows = 0;
  for (int i = 0; i < a->n_seqs; i++) {
    const int n = a->n_rows ? a->n_rows[i] : 1;
    if (n < 0) { set_error("matmul_lora: negative row count of request %d", i); return RELUX_ERR_INVALID_ARG; }
    if (a->adapter[i] < -1 || a->adapter[i] >= a->n_slots) {
      set_error("matmul_lora: adapter %d of request %d outside [-1, %d)", a->adapter[i], i, a->n_slots);
      return RELUX_ERR_INVALID_ARG;
    }
    rows += n;
  }
  if (a->m > kMost || a->k > kMost || a->n > kMost) { set_error("matmul_lora: M=%d K=%d N=%d, up to %d each", a->m, a->k, a->n, kMost); return RELUX_ERR_UNSUPPORTED; }
  if (a->x_halves && a->x_dtype == RELUX_DTYPE_F32 && a->m > kMost / 2) { set_error("matmul_lora: M=%d above %d with x_halves", a->m, kMost / 2); return RELUX_ERR_UNSUPPORTED; }
  if (rows != a->m) { set_error("matmul_lora: the requests have %lld rows, M=%d", (long long)rows, a->m); return RELUX_ERR_INVALID_ARG; }
  int32_t rc;
  if ((rc = check_dev_align(a->x, "x")) || (rc = check_dev_align(a->w, "w")) || (rc = check_dev_align(a->lora_a, "lora_a")) || (rc = check_dev_align(a->lora_b, "lora_b")) ||
      (rc = check_dev_align(a->factors, "factors")) || (rc = check_dev_align(a->out, "out")))
    return rc;
  if (a->k % 8 != 0 || a->n % 8 != 0 || (a->rank != 8 && a->rank != 16 && a->rank != 32 && a->rank != 64 && a->rank != 128)) {
    set_error("matmul_lora: K=%d and N=%d must be multiples of 8, rank=%d one of 8, 16, 32, 64, 128", a->k, a->n, a->rank);
    return RELUX_ERR_UNSUPPORTED;
  }
  LoraPlan plan;
  plan_lora(p, a, &plan);
  const std::vector<Request>& requests = plan.requests;
  const bool x_bf16 = a->x_dtype == RELUX_DTYPE_BF16;
  DownParams down{};
  down.x = a->x;
  down.a = (const uint16_t*)a->lora_a;
  down.M = a->m;
  down.K = a->k;
  down.rank = a->rank;
  if (plan.form == Form::kTiles) {
    if ((rc = grow(p->dev, p->layer_buf, plan.bytes))) return rc;
    uint16_t* const rounded = x_bf16 ? nullptr : (uint16_t*)p->layer_buf.p;
    uint16_t* const t_hi = (uint16_t*)((char*)p->layer_buf.p + plan.bytes - plan.t_bytes);
    uint16_t* const t_lo = t_hi + (size_t)a->m * a->rank;
    const uint16_t* x = (const uint16_t*)(x_bf16 ? a->x : nullptr);   // nullptr: lora_rows_kernel rounds
    // so few tiles that even in eight parts of K they leave half of the SMs idle: float32 rows are rounded by a launch of their own, but for short K (rank 16, 4096 x 4096: 256
    // rows 28.1 us so and 32.9 without, 1024 rows 45.5 and 46.8, 1536 66.3 and 64.4; 1024 rows of K 8192 48 to 62 and 62, of K 1024 22.6 and 21.3)
    if (!x_bf16 && plan.tiles.n * 16 <= p->dev->sm_count && a->k >= 2048) {
      if ((rc = launch_cast(p, (const float*)a->x, rounded, (size_t)a->m * a->k))) return rc;
      x = rounded;
    }
    if ((rc = launch_lora_rows(p, a, plan.tiles, x, rounded, t_hi, t_lo))) return rc;
    return launch_lora_gemm(p, a, x_bf16 ? x : rounded, nullptr, &plan.tiles, nullptr, t_hi, t_lo);
  }
  if (plan.form == Form::kOneLaunch || plan.form == Form::kFewRows) {
    if (plan.form == Form::kFewRows) {
      if ((rc = grow(p->dev, p->layer_buf, plan.bytes))) return rc;
      down.t = (float*)p->layer_buf.p;
      if ((rc = run_down(p, x_bf16 ? kBf16 : kSplit, down, requests, true))) return rc;
    }
    int32_t row_slots[kNarrowRows];
    for (const Request& r : requests) std::fill(row_slots + r.row, row_slots + r.row + r.n, r.slot);
    return launch_lora_gemm(p, a, x_bf16 ? (const uint16_t*)a->x : nullptr, row_slots, nullptr, down.t, nullptr, nullptr);
  }
  LayerScratch sc;
  const int gemm_rows = plan.halves ? 2 * a->m : a->m;
  if ((rc = layer_scratch(p, gemm_rows, a->k, a->w ? a->n : 0, plan.t_bytes, &sc, true))) return rc;
  UpParams up{};
  if (plan.form == Form::kColumns) {
    AdapterColumns cols{a->lora_a, a->n_slots, a->rank, 0, plan.t_parts, (float*)sc.rest, {}};
    std::vector<int32_t> ids;
    for (const Request& r : requests)
      if (r.slot >= 0) ids.push_back(r.slot);
    std::sort(ids.begin(), ids.end());
    cols.n_used = (int)(std::unique_copy(ids.begin(), ids.end(), cols.slot) - cols.slot);
    if (!x_bf16 && (rc = launch_cast(p, (const float*)a->x, sc.a_bf16, (size_t)a->m * a->k))) return rc;
    const WeightRef w{a->w, a->n};
    if ((rc = launch_skinny_gemm(p, x_bf16 ? (const uint16_t*)a->x : sc.a_bf16, a->m, a->k, &w, 1, sc.part, sc.part_cap, &up.rg, TimeStamp{nullptr, nullptr}, &cols, x_bf16)))
      return rc;
    up.part = sc.part;
    up.t_parts = plan.t_parts;
    up.t_cols = cols.n_used * a->rank;
    up.t = cols.t;
  } else {
    if (a->w && !x_bf16) down.x_bf16 = sc.a_bf16;
    down.t = (float*)sc.rest;
    if ((rc = run_down(p, x_bf16 ? kBf16 : a->w && !plan.halves ? kRounded : kSplit, down, requests, false))) return rc;
    if (a->w) {
      const WeightRef w{a->w, a->n};
      if ((rc = launch_skinny_gemm(p, x_bf16 ? (const uint16_t*)a->x : sc.a_bf16, gemm_rows, a->k, &w, 1, sc.part, sc.part_cap, &up.rg))) return rc;
      up.part = sc.part;
    }
    up.t = down.t;
  }
  up.b = (const uint16_t*)a->lora_b;
  up.factors = a->factors;
  up.out = a->out;
  up.halves = plan.halves;
  up.M = a->m;
  up.N = a->n;
  up.out_bf16 = a->out_dtype == RELUX_DTYPE_BF16;
  up.adds = a->accumulate != 0;
  return with_rank(a->rank, [&](auto r) {
    return for_lists(a->m, requests, [&](const auto& list, int groups) { return launch_up<decltype(r)::value>(p, up, list, groups); });
  });
}

size_t matmul_lora_scratch(const Pool* p, const relux_matmul_lora_args* a) {
  LoraPlan plan;
  plan_lora(p, a, &plan);
  return plan.bytes;
}

}  // namespace relux
