// Rows between two projections: the root-mean-square norm with the residual's addition (RMSNorm.Forward, rmsnorm.go:69-97, and the
// additions of Block.Forward, transformer_block.go:119-142), and rows in 8 bits for relux_matmul_int8.
//
//   h = x + residual,  y = h * (1 / sqrt(mean(h^2) + eps)) * weight
//   8 bits: a = max |y|,  scale = a / 127,  code = y * (127 / a) to the nearest whole number, even on a tie: the rule of the 8-bit cache
//
// Everything is float32 from the inputs to the one rounding of each result (h is normalised before it is rounded for residual_out); sums of
// squares are taken by thread, then by tree.  Bound: HBM, x and the residual read once, the results written once; up to some hundred KB the
// latency of one load, two reductions and a store.
#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "tile_gemm.cuh"

namespace relux {

namespace {

constexpr int kMaxRowThreads = 1024, kMaxNV = 4, kMaxParts = 4;
// Of a row's traffic, from which on a part of it has a block of its own while there are idle SMs (float32 rows of 16384: 60 of them 5.0 us in one block each, 4.65 in two; 30 of them 5.1 and, in four, 4.0).
constexpr int64_t kPartBytes = 128 << 10;
constexpr int kMaxNormDim = 8 * kMaxRowThreads * kMaxNV;
constexpr float kTiny = 1e-36f;   // rows without a value this large have no finite 127 / a: zeros

struct NormParams {
  const void* x;
  const void* residual;      // nullptr: h = x
  const void* weight;        // nullptr: ones
  void* residual_out;        // type of the residual
  void* out;
  int8_t* codes;
  float* scales;
  int32_t n_rows, d;
  int32_t weight_bf16, out_bf16;
  float eps, inv_d;
};

__device__ __forceinline__ float top_of(float a, float b) {   // a NaN stays one
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Eight values of a thread: a chunk of eight neighbours, or (kApart, where a type is float32) two quads that lie a team's width apart, so that a warp's load is of whole
// 32-byte sectors: halves of them, 16 bytes a thread of 32, ask L2 for everything twice.
struct alignas(16) Raw8 {   // as they lie in memory
  uint4 lo, hi;             // hi: float32 only
};
template <bool kBf16, bool kApart>
__device__ __forceinline__ Raw8 load_raw(const void* p, size_t lo, size_t hi) {
  Raw8 r;
  if constexpr (kBf16 && kApart) {
    const uint2 a = load_chained(reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + lo)),
                b = load_chained(reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + hi));
    r.lo = make_uint4(a.x, a.y, b.x, b.y);
  } else if constexpr (kBf16) {
    r.lo = load_chained(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + lo));
  } else {
    r.lo = load_chained(reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p) + lo));
    r.hi = load_chained(reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p) + hi));
  }
  return r;
}
template <bool kBf16>
__device__ __forceinline__ void widen(const Raw8& r, float (&v)[8]) {
  if constexpr (kBf16) {
    v[0] = bf16_lo(r.lo.x); v[1] = bf16_hi(r.lo.x); v[2] = bf16_lo(r.lo.y); v[3] = bf16_hi(r.lo.y);
    v[4] = bf16_lo(r.lo.z); v[5] = bf16_hi(r.lo.z); v[6] = bf16_lo(r.lo.w); v[7] = bf16_hi(r.lo.w);
  } else {
    v[0] = __uint_as_float(r.lo.x); v[1] = __uint_as_float(r.lo.y); v[2] = __uint_as_float(r.lo.z); v[3] = __uint_as_float(r.lo.w);
    v[4] = __uint_as_float(r.hi.x); v[5] = __uint_as_float(r.hi.y); v[6] = __uint_as_float(r.hi.z); v[7] = __uint_as_float(r.hi.w);
  }
}
template <bool kApart>
__device__ __forceinline__ void store8(void* p, size_t lo, size_t hi, const float (&v)[8], bool bf16) {
  if (bf16) {
    const uint4 u = make_uint4(round_bf16x2(v[0], v[1]), round_bf16x2(v[2], v[3]), round_bf16x2(v[4], v[5]), round_bf16x2(v[6], v[7]));
    uint16_t* const q = reinterpret_cast<uint16_t*>(p);
    if constexpr (kApart) {
      *reinterpret_cast<uint2*>(q + lo) = make_uint2(u.x, u.y);
      *reinterpret_cast<uint2*>(q + hi) = make_uint2(u.z, u.w);
    } else {
      *reinterpret_cast<uint4*>(q + lo) = u;
    }
  } else {
    float* const q = reinterpret_cast<float*>(p);
    *reinterpret_cast<float4*>(q + lo) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(q + hi) = make_float4(v[4], v[5], v[6], v[7]);
  }
}

__device__ __forceinline__ void store4(void* p, size_t at, const float (&v)[8], bool bf16) {   // the first four of them
  if (bf16) *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p) + at) = make_uint2(round_bf16x2(v[0], v[1]), round_bf16x2(v[2], v[3]));
  else *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + at) = make_float4(v[0], v[1], v[2], v[3]);
}

// One team a row: kLanes: `blockDim.x` lanes of a warp, a power of two, with kNV rows to a team; kBlock; kCluster: a cluster of blocks, a part of the row each.
// A thread holds kNV times eight values: of its part of the row the chunks threadIdx.x + i * blockDim.x, or chunk threadIdx.x of row i.  kNorm = false: only the
// 8-bit form of x.
enum Team { kLanes, kBlock, kCluster };
template <bool kXBf16, bool kRBf16, int kNV, Team kTeam, bool kNorm>
__global__ void __launch_bounds__(kTeam == kLanes ? 256 : kMaxRowThreads) norm_rows_kernel(const NormParams p) {
  constexpr bool kWarp = kTeam == kLanes, kParts = kTeam == kCluster, kApart = !kXBf16 || !kRBf16;
  __shared__ float sums[32], tops[32], part_sums[kMaxParts], part_tops[kMaxParts];
  constexpr int kRows = kWarp ? kNV : 1, kEach = kWarp ? 1 : kNV;   // rows, and chunks of each
  const int parts = kParts ? (int)cluster_size() : 1, part = kParts ? (int)cluster_ctarank() : 0;
  if constexpr (kParts) cluster_arrive();   // this block has begun: its shared memory may be written from the others
  // waits before it releases: a launch behind this one may rely on everything older (launch_chained, head of a chain)
  chain_wait();
  chain_release();
  const uint32_t row0 = kWarp ? (blockIdx.x * blockDim.y + threadIdx.y) * kNV : blockIdx.x / parts;   // past 2^31 in the last block of that many rows
  const int chunks = p.d >> 3, lanes = blockDim.x, per = (chunks + parts - 1) / parts, first = part * per, end = min(chunks, first + per);
  const bool adds = kNorm && p.residual;
  Raw8 rx[kNV], rr[kNV];
  float v[kNV][8], sum[kRows];
  auto row_of = [&](int i) { return kWarp ? row0 + i : row0; };
  auto quad_of = [&](int i, int h) {   // half h of the eight values
    const int j = kWarp ? 0 : i;
    return 2 * first + (kApart ? (int)threadIdx.x + (2 * j + h) * lanes : 2 * ((int)threadIdx.x + j * lanes) + h);
  };
  auto there = [&](int i, int h) { return quad_of(i, h) < 2 * end; };   // (not apart: both halves or none)
  auto mine = [&](int i, int h) { return row_of(i) < (uint32_t)p.n_rows && there(i, h); };
  auto at = [&](int i, int h) { return (size_t)row_of(i) * p.d + 4 * quad_of(i, h); };
  auto load = [&](auto bf16, const void* from, int i) { return load_raw<decltype(bf16)::value, kApart>(from, at(i, 0), mine(i, 1) ? at(i, 1) : at(i, 0)); };
  auto store = [&](void* to, int i, bool bf16) {
    if (mine(i, 1)) store8<kApart>(to, at(i, 0), at(i, 1), v[i], bf16);
    else if (mine(i, 0)) store4(to, at(i, 0), v[i], bf16);
  };

#pragma unroll
  for (int i = 0; i < kNV; i++)
    if (mine(i, 0)) rx[i] = load(std::bool_constant<kXBf16>(), p.x, i);
  if (adds)
#pragma unroll
    for (int i = 0; i < kNV; i++)
      if (mine(i, 0)) rr[i] = load(std::bool_constant<kRBf16>(), p.residual, i);

#pragma unroll
  for (int i = 0; i < kRows; i++) sum[i] = 0.f;
#pragma unroll
  for (int i = 0; i < kNV; i++) {
    widen<kXBf16>(rx[i], v[i]);
    if (adds) {
      float r[8];
      widen<kRBf16>(rr[i], r);
#pragma unroll
      for (int k = 0; k < 8; k++) v[i][k] += r[k];
      if (p.residual_out) store(p.residual_out, i, kRBf16);
    }
#pragma unroll
    for (int k = 0; k < 8; k++) {
      if (!mine(i, k / 4)) v[i][k] = 0.f;
      if constexpr (kNorm) sum[i / kEach] = fmaf(v[i][k], v[i][k], sum[i / kEach]);
    }
  }
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  if constexpr (kNorm) {
#pragma unroll
    for (int i = 0; i < kRows; i++)
      for (int o = kWarp ? lanes >> 1 : 16; o > 0; o >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
    if constexpr (!kWarp) {
      if (lane == 0) sums[warp] = sum[0];
      __syncthreads();
      sum[0] = warp_sum(lane < warps ? sums[lane] : 0.f);
      if constexpr (kParts) {   // to all parts, which add them up in their order
        cluster_wait();
        if (threadIdx.x < parts) store_cluster(mapa_u32(smem_u32(part_sums + part), threadIdx.x), __float_as_uint(sum[0]));
        cluster_arrive();
        cluster_wait();
        sum[0] = 0.f;
        for (int k = 0; k < parts; k++) sum[0] += part_sums[k];
      }
    }
#pragma unroll
    for (int i = 0; i < kRows; i++) sum[i] = rsqrtf(fmaf(sum[i], p.inv_d, p.eps));
    float w[8];
#pragma unroll
    for (int i = 0; i < kNV; i++) {
      const float r = sum[i / kEach];
      if (p.weight && there(i, 0) && (!kWarp || i == 0)) {
        const size_t lo = 4 * quad_of(i, 0), hi = there(i, 1) ? 4 * quad_of(i, 1) : lo;
        if (p.weight_bf16) widen<true>(load_raw<true, kApart>(p.weight, lo, hi), w);
        else widen<false>(load_raw<false, kApart>(p.weight, lo, hi), w);
      }
#pragma unroll
      for (int k = 0; k < 8; k++) {
        v[i][k] *= r;
        if (p.weight && there(i, 0)) v[i][k] *= w[k];
      }
      if (p.out) store(p.out, i, p.out_bf16);
    }
  }
  if (p.codes) {
    float top[kRows];
#pragma unroll
    for (int i = 0; i < kRows; i++) top[i] = 0.f;
#pragma unroll
    for (int i = 0; i < kNV; i++)
#pragma unroll
      for (int k = 0; k < 8; k++) top[i / kEach] = top_of(top[i / kEach], mine(i, k / 4) ? fabsf(v[i][k]) : 0.f);
#pragma unroll
    for (int i = 0; i < kRows; i++)
      for (int o = kWarp ? lanes >> 1 : 16; o > 0; o >>= 1) top[i] = top_of(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
    if constexpr (!kWarp) {
      if (lane == 0) tops[warp] = top[0];
      __syncthreads();
      top[0] = lane < warps ? tops[lane] : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top[0] = top_of(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
      if constexpr (kParts) {
        if constexpr (!kNorm) cluster_wait();
        if (threadIdx.x < parts) store_cluster(mapa_u32(smem_u32(part_tops + part), threadIdx.x), __float_as_uint(top[0]));
        cluster_arrive();
        cluster_wait();
        for (int k = 0; k < parts; k++) top[0] = top_of(top[0], part_tops[k]);
      }
    }
#pragma unroll
    for (int i = 0; i < kNV; i++) {
      // an infinity or a NaN: the scale is NaN and the codes are zeros, so that the row, and nothing else, comes out as NaN
      const float t = top[i / kEach];
      const bool finite = __float_as_uint(t) < 0x7F800000u, some = finite && t >= kTiny;
      const float up = some ? __fdiv_rn(127.f, t) : 0.f;
      if (mine(i, 0) && quad_of(i, 0) == 0) p.scales[row_of(i)] = some ? __fdiv_rn(t, 127.f) : finite ? 0.f : __uint_as_float(0x7FC00000u);
      uint32_t q[8], w[2];
#pragma unroll
      for (int k = 0; k < 8; k++) q[k] = some ? (uint32_t)__float2int_rn(__fmul_rn(v[i][k], up)) : 0u;
#pragma unroll
      for (int k = 0; k < 2; k++) w[k] = __byte_perm(__byte_perm(q[4 * k], q[4 * k + 1], 0x0040), __byte_perm(q[4 * k + 2], q[4 * k + 3], 0x0040), 0x5410);
      if constexpr (kApart) {
#pragma unroll
        for (int h = 0; h < 2; h++)
          if (mine(i, h)) *reinterpret_cast<uint32_t*>(p.codes + at(i, h)) = w[h];
      } else {
        if (mine(i, 0)) *reinterpret_cast<uint2*>(p.codes + at(i, 0)) = make_uint2(w[0], w[1]);
      }
    }
  }
  fence_chained_writes();   // codes, and bf16 rows, are a projection's operands
}

template <bool kXBf16, bool kRBf16, int kNV, Team kTeam, bool kNorm>
int32_t launch_one(Pool* p, const NormParams& prm, dim3 grid, dim3 block, int parts = 1) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = p->dev->stream;
  cudaLaunchAttribute at[2];
  cfg.attrs = at;
  if (p->tune.get(RELUX_TUNE_CHAINED_LAUNCHES) != 0) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (kTeam == kCluster) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs].val.clusterDim.x = (unsigned)parts;
    at[cfg.numAttrs].val.clusterDim.y = at[cfg.numAttrs].val.clusterDim.z = 1;
    cfg.numAttrs++;
  }
  RELUX_CUDA_TRY(cudaLaunchKernelEx(&cfg, norm_rows_kernel<kXBf16, kRBf16, kNV, kTeam, kNorm>, prm));
  count_launch(p->dev);
  return RELUX_OK;
}
template <bool kXBf16, bool kRBf16, bool kNorm>
int32_t launch_typed(Pool* p, const NormParams& prm) {
  const int chunks = prm.d / 8;
  if (chunks <= 32) {
    int lanes = 1;
    while (lanes < chunks) lanes *= 2;
    const dim3 block(lanes, 256 / lanes);
    auto grid = [&](int rows) { return dim3((unsigned)((prm.n_rows + (int64_t)block.y * rows - 1) / ((int64_t)block.y * rows))); };
    // four rows a team once the SMs are full of teams of one (20440 rows of 128, bf16: 6.1 us with one, 4.1 with four)
    if ((int64_t)prm.n_rows * lanes > (int64_t)p->dev->sm_count * 2048) return launch_one<kXBf16, kRBf16, 4, kLanes, kNorm>(p, prm, grid(4), block);
    return launch_one<kXBf16, kRBf16, 1, kLanes, kNorm>(p, prm, grid(1), block);
  }
  int parts = 1;
  const int64_t bytes = (int64_t)prm.d * ((kXBf16 ? 2 : 4) + (prm.residual ? (kRBf16 ? 4 : 8) : 0) + (prm.out ? (prm.out_bf16 ? 2 : 4) : 0));
  while (parts < kMaxParts && bytes / parts >= kPartBytes && prm.n_rows <= p->dev->sm_count / (2 * parts)) parts *= 2;
  // As few chunks a thread as the block's limit lets.  Of more bf16 rows than are resident at once as many as keep blocks at 256 threads, so that more rows are on their
  // way (8192 rows of 8192: 91 us in blocks of 1024 threads, 84 in blocks of 256); of float32 that gives nothing (5000 rows of 4096: 30.7 us with two chunks a thread,
  // 29.4 with one; 400 of 16384 23.7 with four and 22.1 with two).
  const int each = (chunks + parts - 1) / parts;
  int nv = each <= kMaxRowThreads ? 1 : each <= 2 * kMaxRowThreads ? 2 : 4;
  if (kXBf16 && kRBf16 && prm.n_rows > 2 * p->dev->sm_count)
    while (nv < 4 && each > 256 * nv) nv *= 2;
  const int threads = ((each + nv - 1) / nv + 31) / 32 * 32;
  const dim3 grid((unsigned)prm.n_rows * (unsigned)parts), block((unsigned)threads);
  static_assert(kMaxNormDim / 8 / 2 <= 2 * kMaxRowThreads, "half of a row takes more than two chunks a thread");
  if (parts > 1)
    return nv == 1 ? launch_one<kXBf16, kRBf16, 1, kCluster, kNorm>(p, prm, grid, block, parts) : launch_one<kXBf16, kRBf16, 2, kCluster, kNorm>(p, prm, grid, block, parts);
  return nv == 1 ? launch_one<kXBf16, kRBf16, 1, kBlock, kNorm>(p, prm, grid, block)
       : nv == 2 ? launch_one<kXBf16, kRBf16, 2, kBlock, kNorm>(p, prm, grid, block)
                 : launch_one<kXBf16, kRBf16, 4, kBlock, kNorm>(p, prm, grid, block);
}

// w [k][n] -> codes [n][k] and a scale per column.  One block per 64 columns: their largest magnitudes, then the codes through shared memory, so
// that reads and writes are coalesced.  Once per model.
constexpr int kImpCols = 64, kImpRows = 64;
template <bool kBf16>
__global__ void __launch_bounds__(256) int8_weights_kernel(const void* w, int k, int n, int8_t* codes, float* scales) {
  __shared__ float top[4][kImpCols], ups[kImpCols];
  __shared__ int8_t tile[kImpRows][kImpCols + 4];
  const int col = threadIdx.x & (kImpCols - 1), part = threadIdx.x / kImpCols, n0 = blockIdx.x * kImpCols;
  const bool mine = n0 + col < n;
  auto value = [&](int r) -> float {
    const size_t at = (size_t)r * n + n0 + col;
    return kBf16 ? f32_from_bf16_bits(reinterpret_cast<const uint16_t*>(w)[at]) : reinterpret_cast<const float*>(w)[at];
  };
  float t = 0.f;
  if (mine)
#pragma unroll 8
    for (int r = part; r < k; r += 4) t = top_of(t, fabsf(value(r)));
  top[part][col] = t;
  __syncthreads();
  if (part == 0) {
    t = top_of(top_of(top[0][col], top[1][col]), top_of(top[2][col], top[3][col]));
    const bool finite = __float_as_uint(t) < 0x7F800000u, some = finite && t >= kTiny;
    ups[col] = some ? __fdiv_rn(127.f, t) : 0.f;
    if (mine) scales[n0 + col] = some ? __fdiv_rn(t, 127.f) : finite ? 0.f : __uint_as_float(0x7FC00000u);
  }
  __syncthreads();
  const float up = ups[col];
  for (int r0 = 0; r0 < k; r0 += kImpRows) {
#pragma unroll 4
    for (int r = part; r < kImpRows; r += 4) tile[r][col] = mine && up != 0.f && r0 + r < k ? (int8_t)__float2int_rn(__fmul_rn(value(r0 + r), up)) : (int8_t)0;
    __syncthreads();
    for (int i = threadIdx.x; i < kImpCols * (kImpRows / 4); i += 256) {
      const int c = i / (kImpRows / 4), r = i % (kImpRows / 4) * 4;   // four codes of one column; k is a multiple of 16
      if (n0 + c < n && r0 + r < k) {
        const uint32_t v = (uint8_t)tile[r][c] | (uint32_t)(uint8_t)tile[r + 1][c] << 8 | (uint32_t)(uint8_t)tile[r + 2][c] << 16 | (uint32_t)(uint8_t)tile[r + 3][c] << 24;
        *reinterpret_cast<uint32_t*>(codes + (size_t)(n0 + c) * k + r0 + r) = v;
      }
    }
    __syncthreads();
  }
}

bool dtype_ok(int32_t t) { return t == RELUX_DTYPE_F32 || t == RELUX_DTYPE_BF16; }

template <bool kNorm>
int32_t launch_rows(Pool* p, const NormParams& prm, bool x_bf16, bool r_bf16) {
  if constexpr (kNorm)
    return x_bf16 ? (r_bf16 ? launch_typed<true, true, true>(p, prm) : launch_typed<true, false, true>(p, prm))
                  : (r_bf16 ? launch_typed<false, true, true>(p, prm) : launch_typed<false, false, true>(p, prm));
  else
    return x_bf16 ? launch_typed<true, true, false>(p, prm) : launch_typed<false, false, false>(p, prm);
}

int32_t check_codes(const int8_t* codes, const float* scales, int d) {
  if (!codes || !scales) { set_error("8-bit rows need codes and scales"); return RELUX_ERR_INVALID_ARG; }
  if (d % 16 != 0) { set_error("8-bit rows of %d numbers: must be a multiple of 16", d); return RELUX_ERR_UNSUPPORTED; }
  int32_t rc = check_dev_align(codes, "codes");
  return rc ? rc : check_dev_align(scales, "scales");
}

}  // namespace

// Checks of a norm's arguments, before anything is launched.
int32_t check_rmsnorm(const relux_rmsnorm_args* a) {
  if (!a || !a->x) { set_error("nil argument"); return RELUX_ERR_INVALID_ARG; }
  if (a->n_rows <= 0 || a->d <= 0) { set_error("RMSNorm: rows=%d d=%d must be positive", a->n_rows, a->d); return RELUX_ERR_INVALID_ARG; }
  if (a->d % 8 != 0 || a->d > kMaxNormDim) {
    set_error("RMSNorm: d=%d must be a multiple of 8, up to %d", a->d, kMaxNormDim);
    return RELUX_ERR_UNSUPPORTED;
  }
  if (!dtype_ok(a->x_dtype) || !dtype_ok(a->residual_dtype) || !dtype_ok(a->weight_dtype) || !dtype_ok(a->out_dtype)) { set_error("bad dtype flag"); return RELUX_ERR_INVALID_ARG; }
  if (!(a->eps >= 0.f)) { set_error("RMSNorm: eps=%g must not be negative", (double)a->eps); return RELUX_ERR_INVALID_ARG; }
  for (int i = 0; i < 5; i++)
    if (a->reserved[i]) { set_error("reserved fields must be zero"); return RELUX_ERR_INVALID_ARG; }
  if (a->residual_out && !a->residual) { set_error("RMSNorm: residual_out without a residual"); return RELUX_ERR_INVALID_ARG; }
  if (!a->out && !a->codes) { set_error("RMSNorm: no output given"); return RELUX_ERR_INVALID_ARG; }
  int32_t rc;
  if (a->codes || a->scales)
    if ((rc = check_codes(a->codes, a->scales, a->d))) return rc;
  if ((rc = check_dev_align(a->x, "x")) || (rc = check_dev_align(a->residual, "residual")) || (rc = check_dev_align(a->residual_out, "residual_out")) ||
      (rc = check_dev_align(a->weight, "weight")) || (rc = check_dev_align(a->out, "out")))
    return rc;
  return RELUX_OK;
}

int32_t do_rmsnorm(Pool* p, const relux_rmsnorm_args* a) {
  if (int32_t rc = check_rmsnorm(a)) return rc;
  NormParams prm{};
  prm.x = a->x;
  prm.residual = a->residual;
  prm.weight = a->weight;
  prm.residual_out = a->residual_out;
  prm.out = a->out;
  prm.codes = a->codes;
  prm.scales = a->scales;
  prm.n_rows = a->n_rows;
  prm.d = a->d;
  prm.weight_bf16 = a->weight_dtype == RELUX_DTYPE_BF16;
  prm.out_bf16 = a->out_dtype == RELUX_DTYPE_BF16;
  prm.eps = a->eps;
  prm.inv_d = 1.f / (float)a->d;
  return launch_rows<true>(p, prm, a->x_dtype == RELUX_DTYPE_BF16, a->residual_dtype == RELUX_DTYPE_BF16);
}

int32_t do_int8_rows(Pool* p, const relux_int8_rows_args* a) {
  if (!a || !a->x) { set_error("nil argument"); return RELUX_ERR_INVALID_ARG; }
  if (a->n_rows <= 0 || a->d <= 0) { set_error("int8_rows: rows=%d d=%d must be positive", a->n_rows, a->d); return RELUX_ERR_INVALID_ARG; }
  if (!dtype_ok(a->x_dtype)) { set_error("bad dtype flag"); return RELUX_ERR_INVALID_ARG; }
  if (a->reserved) { set_error("reserved fields must be zero"); return RELUX_ERR_INVALID_ARG; }
  int32_t rc = check_codes(a->codes, a->scales, a->d);
  if (rc || (rc = check_dev_align(a->x, "x"))) return rc;
  if (a->d > kMaxNormDim) { set_error("int8_rows: d=%d above %d", a->d, kMaxNormDim); return RELUX_ERR_UNSUPPORTED; }
  NormParams prm{};
  prm.x = a->x;
  prm.codes = a->codes;
  prm.scales = a->scales;
  prm.n_rows = a->n_rows;
  prm.d = a->d;
  const bool bf16 = a->x_dtype == RELUX_DTYPE_BF16;
  return launch_rows<false>(p, prm, bf16, bf16);
}

int32_t do_int8_weights(Pool* p, const relux_int8_weights_args* a) {
  if (!a || !a->w) { set_error("nil argument"); return RELUX_ERR_INVALID_ARG; }
  if (a->k <= 0 || a->n <= 0) { set_error("int8_weights: K=%d N=%d must be positive", a->k, a->n); return RELUX_ERR_INVALID_ARG; }
  if (!dtype_ok(a->w_dtype)) { set_error("bad dtype flag"); return RELUX_ERR_INVALID_ARG; }
  if (a->reserved) { set_error("reserved fields must be zero"); return RELUX_ERR_INVALID_ARG; }
  int32_t rc = check_codes(a->codes, a->scales, a->k);
  if (rc || (rc = check_dev_align(a->w, "w"))) return rc;
  if (a->n % 8 != 0) { set_error("int8_weights: N=%d must be a multiple of 8", a->n); return RELUX_ERR_UNSUPPORTED; }
  const dim3 grid((unsigned)((a->n - 1) / kImpCols + 1));
  if (a->w_dtype == RELUX_DTYPE_BF16) int8_weights_kernel<true><<<grid, 256, 0, p->dev->stream>>>(a->w, a->k, a->n, a->codes, a->scales);
  else int8_weights_kernel<false><<<grid, 256, 0, p->dev->stream>>>(a->w, a->k, a->n, a->codes, a->scales);
  RELUX_CUDA_TRY(cudaGetLastError());
  count_launch(p->dev);
  return RELUX_OK;
}

}  // namespace relux
