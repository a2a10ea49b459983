// Whole attention layer steps on the device: the work of MLA.forwardCached (internal/transformer/mla.go:272-397) and
// MHA.forwardCached (mha.go:245-369) either side of the cached attention, so that a caller hands over the layer
// input x and gets the layer output back.  For MLA:
//   1. projections  q^C = x W_Q, q^R = x W_QR, c^KV = x W_DKV, k^R = x W_KR          mla.go:285-288
//   2. decoupled RoPE on q^R and k^R at position cacheLen + s                          mla.go:297-307, rope.go:130-180
//   3. append (c^KV, k^R) to the paged latent cache                                    mla.go:309-314
//   4. absorbed attention over the cache (the kernels of mla_decode.cu)                mla.go:317-377
//   5. output projection  out = o W_O                                                  mla.go:380-389
// and for GQA: q, k, v = x Wq, x Wk, x Wv (mha.go:251-258), RoPE on q and k (mha.go:272-282), append k / v
// (mha.go:284-289), attention (mha.go:292-348), Wo (mha.go:351-355).
// The projections are skinny GEMMs (M = sequences x new tokens, at most a few hundred rows) against bf16 weight
// matrices of up to 16384 x 16384: they are bound by streaming the weights from HBM once.  FAST mode runs them on
// tcgen05 (activations rounded to bf16, f32 accumulation in tensor memory, split along K so that every SM streams an
// equal share of the weights); REFERENCE mode runs them in the reference's own float32 operation order
// (matmulBatched3D, matmul.go: k ascending, multiply then add, never fused), bit for bit.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <type_traits>
#include <vector>
#include "common.cuh"
#include "internal.h"
#include "projection.cuh"
#include "umma.cuh"

namespace relux {

int32_t stage_in(Pool* p, GrowBuf& buf, const void* src, size_t bytes, int mem, const void** dptr);

namespace {

constexpr int kTileN = kGemmTileCols, kTileK = 64;
constexpr int kStageW = kTileK * kTileN * 2;   // 16 KB of weights: two [64 k][64 n] blocks, 128-byte swizzle, MN-major
constexpr int kMaxTok = 256;                   // activation rows of one block

struct GemmMaps {
  CUtensorMap a;                 // activations [M][K] bf16, box: 64 k x NT rows
  CUtensorMap w[kMaxWeights];    // weights [K][N_j] bf16
};
struct GemmParams {
  int32_t n_weights;
  int32_t tile_first[kMaxWeights + 1];   // first 128-column tile of every weight
  int32_t n_cols[kMaxWeights];           // N_j
  int32_t col_first[kMaxWeights];        // first output column of weight j in the concatenated result
  int32_t M, n_total;
  GemmRanges rg;
  float* part;                           // [piece][M][n_total] f32
  // With one block of rows every weight is read once; of more than 16 MB of them, they are loaded to be evicted first, and push out each
  // other and not the activations, partials and cached rows around them: MLA layer of 16 x 4096, 1.36 GB, 266.3 -> 258.4 us, GQA layers of
  // 84 MB, with the cached rows loaded so too, 66.6 -> 65.1 (24 x 2048), 76.4 -> 73.3 (128 x 300), 35.2 -> 34.3 (2 x 400).  Fewer may stay
  // in L2 from call to call.
  int32_t streams;
  // The result of more than 32 rows, in all its pieces no more than half of L2, is stored to stay there until it is summed (layer steps:
  // 100 x 1000 of d_model 4096 113 -> 107.6 us, 60 x 1000 of 16384 281 -> 278; up to 32 rows 1 % slower so).  More cannot stay, and would
  // push out what can (layer prompts of 2 x 2048 and 4 x 2048 tokens, 100 and 201 MB: 523 and 1013 us so, 521 and 1007 without).
  int32_t keeps;
  int32_t* status;
  TimeStamp time;                        // input projections only
};

// NT: activation rows of a block (the N of the MMA).  As many stages as shared memory holds.
template <int NT>
struct GemmShape {
  static constexpr int kStageX = NT * kTileK * 2;   // [NT rows][64 k] bf16, 128-byte swizzle, K-major
  static constexpr int kStage = kStageW + kStageX;
  static constexpr int kStages = (232448 - 1024) / kStage;
  static constexpr int kSmem = kStages * kStage + 1024;
  static constexpr int kAcc = NT < 32 ? 32 : NT;    // columns of one of the two accumulators
};

// A launch's part in AdapterColumns, or nothing.
struct NoItems {};
struct AdapterItems {
  CUtensorMap a;                         // [n_slots * rank][K], box: 64 k x an adapter
  int32_t items, parts, steps, rank, n_used, shift;   // shift: log2 of the adapters of a tile
  float* t;
  int32_t slot[kMaxUsed];
};
// GemmWalk, then the worker's items; first to those who have the fewest steps.
template <bool kBlocks>
struct ItemWalk : GemmWalk<kBlocks> {
  const AdapterItems& it;
  int item, mine;   // item: the current one, or -1
  __device__ ItemWalk(const GemmRanges& rg, int id, const AdapterItems& items) : GemmWalk<kBlocks>(rg, id), it(items), item(-1), mine(gridDim.x - 1 - id) {}
  __device__ int total() const {
    int n = GemmWalk<kBlocks>::total();
    for (int i = mine; i < it.items; i += gridDim.x) n += (i % it.parts + 1) * it.steps / it.parts - i % it.parts * it.steps / it.parts;
    return n;
  }
  __device__ bool next() {
    if (item < 0) {
      if (GemmWalk<kBlocks>::next()) return true;
      item = mine;
    } else {
      item += gridDim.x;
    }
    if (item >= it.items) return false;
    const int p = item % it.parts;
    this->col = 0;
    this->k0 = p * it.steps / it.parts;
    this->k1 = (p + 1) * it.steps / it.parts;
    return true;
  }
  __device__ int tile() const { return item / it.parts; }
  __device__ int adapters() const { return min(1 << it.shift, it.n_used - (tile() << it.shift)); }   // of the item's tile
};

struct GemmBars {
  uint64_t full[12], empty[12], acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  volatile int32_t abort_flag;
};
static_assert(GemmShape<16>::kStages <= 12 && sizeof(GemmBars) <= 1024, "barrier block too small");

__device__ __noinline__ void gemm_wait_slow(uint64_t* bar, uint32_t parity, GemmBars* b, int32_t* status) {
  for (uint32_t i = 0; i < kSpinLimit; i++) {
    if (mbar_try_wait(bar, parity)) return;
    if ((i & 255) == 255 && b->abort_flag) return;
    if (i > 512) __nanosleep(20);
  }
  b->abort_flag = 1;
  set_status(status, RELUX_ERR_TIMEOUT);
}
// Bounded wait: a wait that runs out records RELUX_ERR_TIMEOUT and raises the CTA's abort flag; nobody leaves a loop early.
__device__ __forceinline__ void gemm_wait(uint64_t* bar, uint32_t parity, GemmBars* b, int32_t* status) {
  if (!mbar_try_wait(bar, parity)) gemm_wait_slow(bar, parity, b, status);
}

// part[piece][m][n] = x [M][K] x [W_0 | W_1 | ...] over the piece's K steps.  Bound: HBM, every weight is read once.
// grid (workers), 192 threads: warps 0-3 epilogue, warp 4 TMA producer, warp 5 MMA issuer.
//   * The WEIGHTS are the M = 128 operand (MN-major: the row-major rows as they lie in HBM) and the activations, 16 to 256
//     rows, the N operand, so that a stage is 16 KB of weights and no more activations than there are: with the
//     activations as the M = 128 operand a stage of 16 rows was half padding, read from L2 for every step.
//   * One CTA per SM walks its pieces (GemmRanges) without draining its pipeline in between (two accumulators: a piece is
//     written out while the next one's MMAs run).
//   * The weights do not depend on the launches before this one, whose tail and launch gap they hide: the producer
//     fills its stages with them before chain_wait().  The first kernel of a layer step (cast_bf16_kernel) releases its
//     successors only when everything before the step is complete, so that weights written earlier in the stream are there.
// Measured with the chained launches around it (a layer step, before -> now): 16 rows of d_model 16384, 1.36 GB of weights,
// 308 -> 272 us; 24 rows of d_model 4096, 84 MB, 82.8 -> 67.0 us.
template <int NT, class Items>
__global__ void __launch_bounds__(192, 1) skinny_gemm_sm100_kernel(const __grid_constant__ GemmMaps maps, const __grid_constant__ GemmParams prm, const __grid_constant__ Items items) {
  constexpr bool kItems = std::is_same_v<Items, AdapterItems>;
  using SH = GemmShape<NT>;
  constexpr int kStages = SH::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  GemmBars* bars = reinterpret_cast<GemmBars*>(smem + kStages * SH::kStage);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr bool kBlocks = NT >= 128;   // smaller blocks hold all rows
  auto walk = [&] {
    if constexpr (kItems) return ItemWalk<kBlocks>(prm.rg, blockIdx.x, items);
    else return GemmWalk<kBlocks>(prm.rg, blockIdx.x);
  }();
  auto in_items = [&](const auto& w) {
    if constexpr (kItems) return w.item >= 0;
    else return false;
  };
  auto weight_of = [&](int tile) -> int {
    int j = 0;
    while (j + 1 < prm.n_weights && tile >= prm.tile_first[j + 1]) j++;
    return j;
  };
  chain_release();
  if ((smem_u32(smem) & 1023u) != 0) {
    chain_wait();
    if (threadIdx.x == 0) set_status(prm.status, RELUX_ERR_UNSUPPORTED);
    return;
  }
  if (threadIdx.x == 0) {
    stamp_begin(prm.time);   // the launch that cleared the slot is complete: see cast_bf16_kernel
    for (int s = 0; s < kStages; s++) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
    for (int b = 0; b < 2; b++) { mbar_init(&bars->acc_full[b], 1); mbar_init(&bars->acc_empty[b], 4); }
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc<1>(&bars->tmem_base, 2 * SH::kAcc);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  if (warp == 4) {
    const bool el = elect_one();
    const uint64_t policy = prm.streams ? make_evict_first_policy() : make_evict_normal_policy();   // (a branch around the loads cost 3 %)
    if (el) tma_prefetch_desc(&maps.a);
    const int n = walk.total(), ahead = min(n, kStages);
    auto wx = walk;   // the activations' place, up to kStages steps behind
    walk.next();
    wx.next();
    int k = walk.k0, kx = wx.k0, j = weight_of(walk.col);
    auto load_w = [&](int g) {   // the weights of step g of this worker; arms the stage for both operands
      const int s = g % kStages;
      if (el) {
        uint8_t* sw = smem + s * SH::kStage;
        if constexpr (kItems)
          if (in_items(walk)) {
            const int some = walk.adapters();
            mbar_expect_tx(&bars->full[s], some * items.rank * 128 + SH::kStageX);
            for (int q = 0; q < some; q++)
              tma_load_2d(sw + q * items.rank * 128, &items.a, k * kTileK, items.slot[(walk.tile() << items.shift) + q] * items.rank, &bars->full[s]);
          }
        const int n0 = (walk.col - prm.tile_first[j]) * kTileN;
        if (!in_items(walk)) {
          mbar_expect_tx(&bars->full[s], SH::kStage);   // out-of-range parts of a box are zero-filled and still counted
          tma_load_2d_hint(sw, &maps.w[j], n0, k * kTileK, &bars->full[s], policy);
          tma_load_2d_hint(sw + kStageW / 2, &maps.w[j], n0 + 64, k * kTileK, &bars->full[s], policy);
        }
      }
      __syncwarp();
      if (++k == walk.k1 && walk.next()) {
        k = walk.k0;
        j = weight_of(walk.col);
      }
    };
    auto load_x = [&](int g) {
      const int s = g % kStages;
      if (el) tma_load_2d(smem + s * SH::kStage + kStageW, &maps.a, kx * kTileK, kBlocks ? wx.block * NT : 0, &bars->full[s]);
      __syncwarp();
      if (++kx == wx.k1 && wx.next()) kx = wx.k0;
    };
    for (int g = 0; g < ahead; g++) load_w(g);
    chain_wait();
    for (int g = 0; g < n; g++) {
      if (g >= ahead) {
        gemm_wait(&bars->empty[g % kStages], (g / kStages - 1) & 1, bars, prm.status);
        load_w(g);
      }
      load_x(g);
    }
  } else if (warp == 5) {
    chain_wait();
    const bool el = elect_one();
    const uint32_t idesc = make_idesc_bf16(kTileN, NT, true, false), idesc_items = make_idesc_bf16(kTileN, NT, false, false);
    int g = 0;
    for (int piece = 0; walk.next(); piece++) {
      const uint32_t d = tmem + (piece & 1) * SH::kAcc;
      if (piece >= 2) gemm_wait(&bars->acc_empty[piece & 1], ((piece >> 1) - 1) & 1, bars, prm.status);
      tc_fence_after();
      for (int k = walk.k0; k < walk.k1; k++, g++) {
        const int s = g % kStages;
        gemm_wait(&bars->full[s], (g / kStages) & 1, bars, prm.status);
        tc_fence_after();
        if (el) {
          const uint32_t sw = smem_u32(smem + s * SH::kStage);
          const uint64_t dW = make_desc_mnmajor_sw128(sw, kStageW / 2);
          const uint64_t dX = make_desc_kmajor_sw128(sw + kStageW);
          if (!in_items(walk)) {
#pragma unroll
            for (int kk = 0; kk < kTileK / 16; kk++)
              umma_ss<1>(d, dW + ((uint32_t)(kk * 2048) >> 4), dX + ((uint32_t)(kk * 32) >> 4), idesc, k != walk.k0 || kk != 0);
          } else {
            const uint64_t dA = make_desc_kmajor_sw128(sw);   // adapters lie K-major; rows of the tile behind the last one hold anything
#pragma unroll
            for (int kk = 0; kk < kTileK / 16; kk++)
              umma_ss<1>(d, dA + ((uint32_t)(kk * 32) >> 4), dX + ((uint32_t)(kk * 32) >> 4), idesc_items, k != walk.k0 || kk != 0);
          }
          umma_commit<1>(&bars->empty[s]);
        }
        __syncwarp();
      }
      if (el) umma_commit<1>(&bars->acc_full[piece & 1]);
      __syncwarp();
    }
  } else {
    // epilogue: thread = weight column, accumulator column = activation row; a warp writes 128 bytes of a row at once
    constexpr bool kKeep = NT >= 64;
    const uint64_t stay = !kKeep ? 0 : prm.keeps ? make_evict_last_policy() : make_evict_normal_policy();
    chain_wait();
    for (int piece = 0; walk.next(); piece++) {
      const int j = weight_of(walk.col), m0 = kBlocks ? walk.block * NT : 0;
      int n = (walk.col - prm.tile_first[j]) * kTileN + warp * 32 + lane, n_cols = prm.n_cols[j], row_stride = prm.n_total;
      const int m_end = min(NT, prm.M - m0);
      float* dst = prm.part + ((size_t)walk.split * prm.M + m0) * prm.n_total + prm.col_first[j] + n;
      if constexpr (kItems)
        if (in_items(walk)) {
          n = walk.tile() * kTileN + warp * 32 + lane;
          n_cols = row_stride = items.n_used * items.rank;
          dst = items.t + (size_t)(walk.item % items.parts) * prm.M * row_stride + n;
        }
      gemm_wait(&bars->acc_full[piece & 1], (piece >> 1) & 1, bars, prm.status);
      tc_fence_after();
      const bool ok = !bars->abort_flag, mine = n < n_cols;
#pragma unroll 1
      for (int c = 0; c < m_end; c += 32) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(tmem + ((uint32_t)(warp * 32) << 16) + (piece & 1) * SH::kAcc + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int q = 0; q < 32; q++)
          if (mine && c + q < m_end) {
            float* to = dst + (size_t)(c + q) * row_stride;
            const float x = ok ? __uint_as_float(v[q]) : 0.f;
            if constexpr (kKeep) store_hint(to, x, stay);
            else *to = x;
          }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->acc_empty[piece & 1]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) stamp_end(prm.time);
  if (warp == 0) tmem_dealloc<1>(tmem, 2 * SH::kAcc);
}

// The reference's matmulBatched3D in its own operation order: out[m][n] = sum over k ascending of x[m][k] * w[k][n],
// float32, multiply then add, never fused.  One thread per output element; threads of a warp read consecutive n.
__global__ void gemm_reference_kernel(const float* __restrict__ x, const uint16_t* __restrict__ w, float* __restrict__ out, int M, int K,
                                      int N, int out_stride, int col_first) {
  const int n = blockIdx.x * blockDim.x + threadIdx.x, m = blockIdx.y;
  if (n >= N || m >= M) return;
  const float* xr = x + (size_t)m * K;
  float acc = 0.f;
  for (int k = 0; k < K; k++) acc = __fadd_rn(acc, __fmul_rn(xr[k], f32_from_bf16_bits(w[(size_t)k * N + n])));
  out[(size_t)m * out_stride + col_first + n] = acc;
}

// The first kernel of a layer step.  It waits before it releases the launch after it, which may therefore rely on
// everything that was queued before the step without a wait of its own.
__global__ void cast_bf16_kernel(const float* __restrict__ src, uint16_t* __restrict__ dst, size_t n8) {
  chain_wait();
  chain_release();
  const size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n8) return;
  const float4 a = load_chained(reinterpret_cast<const float4*>(src) + 2 * i), b = load_chained(reinterpret_cast<const float4*>(src) + 2 * i + 1);
  reinterpret_cast<uint4*>(dst)[i] = make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y), pack_bf16x2(b.z, b.w));
  fence_chained_writes();
}

// Sums the K splits of the projection result (fixed order, so the result does not depend on scheduling), applies
// RoPE (rope.go:168-176: pairs (2i, 2i+1) of a head, out0 = x0 c - x1 s, out1 = x1 c + x0 s, unfused) at position
// len[seq] + s to the segments that ask for it, and scatters every segment to its own buffer.
// One thread per pair of adjacent columns of the concatenated result.
struct ProjSeg {
  int32_t n;          // columns of this segment (= of its weight matrix)
  int32_t rope_dim;   // 0: no rotation; else the per-head width the rotation works on
  void* dst;          // [M][n], f32 or bf16
  int32_t bf16;
  int32_t by_tma;     // the next launch reads it by TMA
  const float* src;   // [M][n] where its projection is whole, a call of its own; nullptr: the pieces of the joint one
};
struct FinishParams {
  const float* part;
  GemmRanges rg;
  int32_t tile_first[kMaxWeights];   // first 128-column tile of every segment
  int32_t M, n_total, S, n_segs;
  int32_t row0;                    // first row of this launch
  ProjSeg seg[kMaxWeights];
  const int32_t* len;              // this layer's lengths BEFORE the append
  const int32_t* seq_ids;
  const float* rope_cos;           // [positions][rope_dim / 2]
  const float* rope_sin;
  int32_t rope_positions;
  int32_t same_pos;                // the reference's own rule (rope.go:151-158): on a non-empty cache every new row takes position len
  int32_t* status;
};
template <bool kTurns>   // the row blocks come in turns (GemmRanges): a tile is a column and a row
__global__ void proj_finish_kernel(const FinishParams p) {
  const int pair = blockIdx.x * blockDim.x + threadIdx.x, m = p.row0 + blockIdx.y;
  const int col = 2 * pair;
  chain_release();
  chain_wait();
  if (col >= p.n_total || m >= p.M) return;
  int c = col, j = 0;
  while (j + 1 < p.n_segs && c >= p.seg[j].n) {
    c -= p.seg[j].n;
    j++;
  }
  const ProjSeg sg = p.seg[j];
  float v0 = 0.f, v1 = 0.f;
  if (sg.src) {
    const float2 t = load_chained(reinterpret_cast<const float2*>(sg.src + (size_t)m * sg.n + c));
    v0 = t.x;
    v1 = t.y;
  } else {
    const int col_tile = p.tile_first[j] + c / kTileN;
    const int pieces = p.rg.pieces(kTurns ? p.rg.tile_of(col_tile, m) : col_tile);
#pragma unroll 4
    for (int s = 0; s < pieces; s++) {
      const float2 t = load_chained(reinterpret_cast<const float2*>(p.part + ((size_t)s * p.M + m) * p.n_total + col));
      v0 += t.x;
      v1 += t.y;
    }
  }
  if (sg.rope_dim > 0) {
    const int i = m / p.S, s = m % p.S;
    const int seq = p.seq_ids ? p.seq_ids[i] : i;
    const int len0 = load_chained(p.len + seq);
    const int pos = (p.same_pos && len0 > 0) ? len0 : len0 + s;
    if (pos >= p.rope_positions) {
      set_status(p.status, RELUX_ERR_OVERFLOW);   // the reference panics: position >= maxSeqLen (rope.go:160-162)
    } else {
      const int half = sg.rope_dim / 2, idx = (c % sg.rope_dim) >> 1;
      const float cs = p.rope_cos[(size_t)pos * half + idx], sn = p.rope_sin[(size_t)pos * half + idx];
      const float r0 = __fsub_rn(__fmul_rn(v0, cs), __fmul_rn(v1, sn));
      const float r1 = __fadd_rn(__fmul_rn(v1, cs), __fmul_rn(v0, sn));
      v0 = r0;
      v1 = r1;
    }
  }
  if (sg.bf16) {
    reinterpret_cast<uint32_t*>(sg.dst)[((size_t)m * sg.n + c) >> 1] = pack_bf16x2(v0, v1);
    if (sg.by_tma) fence_chained_writes();
  } else {
    *reinterpret_cast<float2*>(reinterpret_cast<float*>(sg.dst) + (size_t)m * sg.n + c) = make_float2(v0, v1);
  }
}

// out [M][N] = sum over the pieces of one weight's tiles; a thread sums four adjacent columns.
template <bool kTurns>
__global__ void sum_splits_kernel(const float* __restrict__ part, GemmRanges rg, int N, size_t n4, float* __restrict__ out) {
  chain_release();
  chain_wait();
  const size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n4) return;
  const int col_tile = (int)(4 * i % (unsigned)N) / kTileN;
  const int pieces = rg.pieces(kTurns ? rg.tile_of(col_tile, (int)(4 * i / (unsigned)N)) : col_tile);
  float4 acc = load_chained(reinterpret_cast<const float4*>(part) + i);
#pragma unroll 4
  for (int s = 1; s < pieces; s++) {
    const float4 t = load_chained(reinterpret_cast<const float4*>(part) + (size_t)s * n4 + i);
    acc.x += t.x; acc.y += t.y; acc.z += t.z; acc.w += t.w;
  }
  reinterpret_cast<float4*>(out)[i] = acc;
}

template <int NT, class Items>
int32_t launch_skinny_gemm_rows(Pool* p, const GemmMaps& maps, const GemmParams& g, int workers, const Items& items, bool chained) {
  if (int32_t rc = allow_smem(p->dev, skinny_gemm_sm100_kernel<NT, Items>, GemmShape<NT>::kSmem)) return rc;
  RELUX_CUDA_TRY(launch_chained(chained && p->tune.get(RELUX_TUNE_CHAINED_LAUNCHES) != 0, skinny_gemm_sm100_kernel<NT, Items>, dim3(workers), dim3(192),
                                (size_t)GemmShape<NT>::kSmem, p->dev->stream, maps, g, items));
  count_launch(p->dev);
  return RELUX_OK;
}

// Deals the tiles to one worker per SM, `beside` blocks of `block_rows` rows beside each other.  max_pieces: pieces of a tile that
// the scratch holds.  *cost_us: what this takes beyond what every dealing takes, from measured parts (4 to 25600 rows against
// weights of 1024 x 1024 to 16384 x 16384): a step takes an SM 0.28 us whatever the rows of its block, and a tenth more where the
// workers don't walk in step; the weights come at 7 TB/s, again for every turn of blocks when they exceed L2; the last piece of
// a worker is written at 16 ns per row with nothing to hide it; pieces are written and read at 3 TB/s.
GemmRanges deal_tiles(int sms, int col_tiles, int M, int block_rows, int beside, int K, int cols, int max_pieces, int split_knob, double* cost_us) {
  GemmRanges r{};
  r.steps = (K + kTileK - 1) / kTileK;
  r.col_tiles = col_tiles;
  r.row_blocks = (M + block_rows - 1) / block_rows;
  r.block_rows = block_rows;
  r.beside = beside;
  const int turns = (r.row_blocks + beside - 1) / beside, tiles = col_tiles * turns, units = tiles * r.steps;
  r.workers = std::max(1, std::min(std::max(1, sms / beside), units / 4));   // pieces of fewer than four steps do not pay for their share of the result
  if (split_knob) r.workers = std::max(1, (int)std::min<int64_t>(units, (int64_t)tiles * split_knob));
  r.full = tiles / r.workers;
  r.rest = tiles % r.workers;
  r.range = r.rest * r.steps / r.workers;
  r.more = r.rest * r.steps % r.workers;
  const double step = 0.28, write = 0.016 * std::min(block_rows, M), per_piece = (double)M * cols * 4 / tiles / 3e6, bytes = (double)K * cols * 2;
  const double weights = bytes * (bytes > 60e6 ? turns : 1) / 7e6;
  auto cost = [&](double steps, double pieces) { return std::max((r.full * r.steps + steps) * step, weights) + write + pieces * per_piece; };
  if (!r.rest) {
    *cost_us = cost(0, tiles);
    return r;
  }
  const int fits = std::max(1, std::min(r.workers / r.rest, max_pieces)), most_split = std::max(1, r.steps / 4);
  const bool even = r.range > 0 && (r.steps - 2) / r.range + 2 <= max_pieces;   // may the ranges be even?
  const double even_cost = cost(1.1 * r.rest * r.steps / r.workers, tiles + r.workers) + std::max(0.0, write - r.range * step / 2);
  auto split_cost = [&](int s) { return cost((r.steps + s - 1) / s, tiles + (double)r.rest * (s - 1)); };
  if (block_rows <= 64) {
    // few rows: results are small, and what counts is that no SM idles
    if (fits >= most_split) r.split = most_split;
    else if (!even || 6 * fits * r.rest >= 5 * r.workers) r.split = fits;
  } else {
    r.split = 1;
    for (int s = 2; s <= std::min(fits, most_split); s++)
      if (split_cost(s) < split_cost(r.split)) r.split = s;
    if (even && even_cost < split_cost(r.split)) r.split = 0;
  }
  *cost_us = r.split ? split_cost(r.split) : even_cost;
  return r;
}

}  // namespace

int32_t launch_skinny_gemm(Pool* p, const uint16_t* a_bf16, int M, int K, const WeightRef* ws, int nw, float* part, size_t part_cap_bytes,
                           GemmRanges* ranges, TimeStamp time, const AdapterColumns* adapters, bool head) {
  GemmMaps maps;
  GemmParams g;
  memset(&g, 0, sizeof(g));
  int tiles = 0, cols = 0;
  for (int j = 0; j < nw; j++) {
    if (!make_tmap_2d(&maps.w[j], (void*)ws[j].w, (uint64_t)K, (uint64_t)ws[j].n, 64, kTileK)) {
      set_error("tensor map for a weight matrix could not be encoded");
      return RELUX_ERR_CUDA;
    }
    g.tile_first[j] = tiles;
    g.n_cols[j] = ws[j].n;
    g.col_first[j] = cols;
    tiles += (ws[j].n + kTileN - 1) / kTileN;
    cols += ws[j].n;
  }
  for (int j = nw; j < kMaxWeights; j++) maps.w[j] = maps.w[0];
  g.tile_first[nw] = tiles;
  g.n_weights = nw;
  g.M = M;
  g.n_total = cols;
  const int steps = (K + kTileK - 1) / kTileK;
  if ((int64_t)tiles * ((M + 127) / 128) * steps >= (int64_t)1 << 31) { set_error("a projection of more than 2^31 steps"); return RELUX_ERR_UNSUPPORTED; }
  // Rows of a block: the smallest tile that holds them all (padding costs L2 reads and shared memory), up to 256; more than 128
  // rows also as blocks of 128 where that keeps more SMs busy or leaves less padding (256 rows of 4096 x 1024: 14.8 us, one block
  // of 256 20.2).  Up to 16 blocks beside each other, whichever number leaves the fewest SMs idle: with all of them beside
  // each other 19200 rows had 75 workers (4096 x 4096: 1.28 ms, now 0.71).
  int nt = 16;
  while (nt < M && nt < kMaxTok) nt *= 2;
  const int max_pieces = (int)std::min<size_t>(std::max<size_t>(1, part_cap_bytes / ((size_t)M * cols * 4)), 1 << 20);
  double best = 0;
  for (int rows = nt; rows >= std::min(nt, 128); rows /= 2)
    for (int beside = std::min(16, (M + rows - 1) / rows); beside >= 1; beside--) {
      double cost = 0;
      const GemmRanges r = deal_tiles(p->dev->sm_count, tiles, M, rows, beside, K, cols, max_pieces, p->tune.get(RELUX_TUNE_GEMM_SPLIT), &cost);
      if (!g.rg.workers || cost < best) {
        g.rg = r;
        best = cost;
      }
    }
  nt = g.rg.block_rows;
  if (!make_tmap_2d(&maps.a, (void*)a_bf16, (uint64_t)M, (uint64_t)K, kTileK, nt)) {
    set_error("tensor map for the activations could not be encoded");
    return RELUX_ERR_CUDA;
  }
  const int workers = g.rg.workers * g.rg.beside;
  g.part = part;
  g.streams = g.rg.row_blocks == 1 && (int64_t)K * cols * 2 > ((int64_t)16 << 20);
  const int tiles_of_block = g.rg.full * g.rg.workers + g.rg.rest;
  const int pieces_of_block = g.rg.full * g.rg.workers + (g.rg.split ? g.rg.rest * g.rg.split : g.rg.rest ? g.rg.rest + g.rg.workers : 0);
  g.keeps = (int64_t)M * cols * 4 * pieces_of_block / tiles_of_block <= kResidentBytes;
  g.status = p->d_status;
  g.time = time;
  *ranges = g.rg;
  if (adapters) {   // of up to 128 rows, in one block
    AdapterItems items;
    if (!make_tmap_2d(&items.a, (void*)adapters->lora_a, (uint64_t)adapters->n_slots * adapters->rank, (uint64_t)K, kTileK, adapters->rank)) {
      set_error("tensor map for adapters could not be encoded");
      return RELUX_ERR_CUDA;
    }
    items.shift = 0;
    while (adapters->rank << (items.shift + 1) <= kTileN) items.shift++;
    items.parts = adapters->parts;
    items.items = ((adapters->n_used - 1 >> items.shift) + 1) * items.parts;
    items.steps = steps;
    items.rank = adapters->rank;
    items.n_used = adapters->n_used;
    items.t = adapters->t;
    std::copy(adapters->slot, adapters->slot + adapters->n_used, items.slot);
    switch (nt) {
      case 16: return launch_skinny_gemm_rows<16>(p, maps, g, workers, items, !head);
      case 32: return launch_skinny_gemm_rows<32>(p, maps, g, workers, items, !head);
      case 64: return launch_skinny_gemm_rows<64>(p, maps, g, workers, items, !head);
      default: return launch_skinny_gemm_rows<128>(p, maps, g, workers, items, !head);
    }
  }
  switch (nt) {
    case 16: return launch_skinny_gemm_rows<16>(p, maps, g, workers, NoItems{}, !head);
    case 32: return launch_skinny_gemm_rows<32>(p, maps, g, workers, NoItems{}, !head);
    case 64: return launch_skinny_gemm_rows<64>(p, maps, g, workers, NoItems{}, !head);
    case 128: return launch_skinny_gemm_rows<128>(p, maps, g, workers, NoItems{}, !head);
    default: return launch_skinny_gemm_rows<kMaxTok>(p, maps, g, workers, NoItems{}, !head);
  }
}

bool gemm_sm100_eligible(int K, const WeightRef* ws, int nw) {
  if (K % 8 != 0 || nw > kMaxWeights) return false;
  for (int j = 0; j < nw; j++)
    if (ws[j].n % 8 != 0 || ((uintptr_t)ws[j].w & 15) != 0) return false;
  return true;
}

namespace {

int32_t launch_gemm_reference(Pool* p, const float* x, int M, int K, const WeightRef* ws, int nw, float* out, int out_stride) {
  int col = 0;
  for (int j = 0; j < nw; j++) {
    dim3 grid((ws[j].n + 127) / 128, M);
    gemm_reference_kernel<<<grid, 128, 0, p->dev->stream>>>(x, (const uint16_t*)ws[j].w, out, M, K, ws[j].n, out_stride, col);
    RELUX_CUDA_TRY(cudaGetLastError());
    count_launch(p->dev);
    col += ws[j].n;
  }
  return RELUX_OK;
}

// cos / sin tables of the decoupled RoPE exactly as NewRotaryEmbedding builds them (rope.go:59-68):
// theta = float32(1) / float32(pow(base, 2i / headDim)), angle = float32(pos * theta), cos / sin in float64, rounded.
int32_t ensure_rope_table(Pool* p, int dHR, float base, int positions) {
  if (p->rope_dim == dHR && p->rope_base == base && p->rope_positions >= positions) return RELUX_OK;
  const int half = dHR / 2;
  std::vector<float> tab((size_t)2 * positions * half);
  for (int pos = 0; pos < positions; pos++)
    for (int i = 0; i < half; i++) {
      const float theta = 1.0f / (float)std::pow((double)base, (double)(2 * i) / (double)dHR);
      const float angle = (float)((double)pos * (double)theta);
      tab[(size_t)pos * half + i] = (float)std::cos((double)angle);
      tab[(size_t)positions * half + (size_t)pos * half + i] = (float)std::sin((double)angle);
    }
  int32_t rc = grow(p->dev, p->rope_tab, tab.size() * 4);
  if (rc) return rc;
  RELUX_CUDA_TRY(cudaMemcpyAsync(p->rope_tab.p, tab.data(), tab.size() * 4, cudaMemcpyHostToDevice, p->dev->stream));
  RELUX_CUDA_TRY(cudaStreamSynchronize(p->dev->stream));   // `tab` goes out of scope
  p->rope_dim = dHR;
  p->rope_base = base;
  p->rope_positions = positions;
  return RELUX_OK;
}

}  // namespace

int32_t launch_cast(Pool* p, const float* src, uint16_t* dst, size_t n) {
  RELUX_CUDA_TRY(launch_chained(p->tune.get(RELUX_TUNE_CHAINED_LAUNCHES) != 0, cast_bf16_kernel, dim3((unsigned)((n / 8 + 255) / 256)), dim3(256), 0,
                                p->dev->stream, src, dst, n / 8));
  count_launch(p->dev);
  return RELUX_OK;
}

namespace {

// The finish kernel behind the projections of a layer.
int32_t finish_projections(Pool* p, const SeqBatch& sb, int layer, int M, int S, const ProjSeg* segs, int nw, const float* part, const GemmRanges& ranges, bool same_pos) {
  FinishParams f;
  memset(&f, 0, sizeof(f));
  f.part = part;
  f.rg = ranges;
  for (int j = 1; j < nw; j++) f.tile_first[j] = f.tile_first[j - 1] + (segs[j - 1].n + kTileN - 1) / kTileN;
  f.M = M;
  f.S = S;
  f.n_segs = nw;
  int rope_dim = 0;
  for (int j = 0; j < nw; j++) {
    f.seg[j] = segs[j];
    f.n_total += segs[j].n;
    if (segs[j].rope_dim) rope_dim = segs[j].rope_dim;
  }
  f.len = p->d_len + (size_t)layer * p->prm.max_seqs;
  f.seq_ids = sb.d_seq_ids;
  f.rope_cos = (const float*)p->rope_tab.p;
  f.rope_sin = f.rope_cos ? f.rope_cos + (size_t)p->rope_positions * (rope_dim / 2) : nullptr;
  f.rope_positions = p->rope_positions;
  f.same_pos = same_pos ? 1 : 0;
  f.status = p->d_status;
  constexpr int kMostGridY = 65535;
  for (f.row0 = 0; f.row0 < M; f.row0 += kMostGridY) {
    const dim3 grid((f.n_total / 2 + 255) / 256, std::min(M - f.row0, kMostGridY));
    RELUX_CUDA_TRY(launch_chained(p->tune.get(RELUX_TUNE_CHAINED_LAUNCHES) != 0, ranges.in_turns() ? proj_finish_kernel<true> : proj_finish_kernel<false>, grid, dim3(256),
                                  0, p->dev->stream, f));
    count_launch(p->dev);
  }
  return RELUX_OK;
}

// x [M][K] f32 -> every segment's buffer: cast (or the norm that a block begins with) + split-K tensor-core GEMM (or the reference-order GEMM), then the
// finish kernel.  The GEMM's device time goes to the pool's projection ring.
int32_t project_and_finish(Pool* p, const SeqBatch& sb, int layer, const float* dx, int M, int K, int S, const WeightRef* ws,
                           const ProjSeg* segs, int nw, bool mma, uint16_t* a_bf16, float* part, size_t part_cap, bool same_pos = false,
                           const relux_rmsnorm_args* norm = nullptr) {
  int n_total = 0;
  for (int j = 0; j < nw; j++) n_total += ws[j].n;
  GemmRanges ranges{};
  if (mma) {
    int32_t rc = norm ? do_rmsnorm(p, norm) : launch_cast(p, dx, a_bf16, (size_t)M * K);
    if (rc) return rc;
    const TimeStamp time = time_stamp_next(p, p->proj_times);
    rc = launch_skinny_gemm(p, a_bf16, M, K, ws, nw, part, part_cap, &ranges, time);
    if (rc) return rc;
    time_stamp_done(p->proj_times, time);
  } else {
    int32_t rc = time_events_begin(p, p->proj_times);
    if (rc) return rc;
    rc = launch_gemm_reference(p, dx, M, K, ws, nw, part, n_total);
    if (rc) return rc;
    if ((rc = time_events_end(p, p->proj_times))) return rc;
  }
  return finish_projections(p, sb, layer, M, S, segs, nw, part, ranges, same_pos);
}

// out [M][N] f32 = attn [M][K] x W_O [K][N]; `out` is the caller's buffer (host or device).  d_attn: float32, or nullptr when
// the rows are in a_bf16 already (mma).
int32_t output_projection(Pool* p, const float* d_attn, int M, int K, const void* w_o, int N, bool mma, uint16_t* a_bf16, float* part,
                          size_t part_cap, void* out, int out_mem) {
  cudaStream_t st = p->dev->stream;
  const bool direct = out_mem == RELUX_MEM_DEVICE;
  float* d_out = direct ? (float*)out : nullptr;
  if (!direct) {
    int32_t rc = grow(p->dev, p->out_buf, (size_t)M * N * 4);
    if (rc) return rc;
    d_out = (float*)p->out_buf.p;
  }
  const WeightRef outp[1] = {{w_o, N}};
  if (mma) {
    GemmRanges ranges{};
    int32_t rc = d_attn ? launch_cast(p, d_attn, a_bf16, (size_t)M * K) : RELUX_OK;
    if (!rc) rc = launch_skinny_gemm(p, a_bf16, M, K, outp, 1, part, part_cap, &ranges);
    if (rc) return rc;
    const size_t n4 = (size_t)M * N / 4;
    RELUX_CUDA_TRY(launch_chained(p->tune.get(RELUX_TUNE_CHAINED_LAUNCHES) != 0, ranges.in_turns() ? sum_splits_kernel<true> : sum_splits_kernel<false>,
                                  dim3((unsigned)((n4 + 255) / 256)), dim3(256), 0, st, (const float*)part, ranges, N, n4, d_out));
    count_launch(p->dev);
  } else {
    int32_t rc = launch_gemm_reference(p, d_attn, M, K, outp, 1, d_out, N);
    if (rc) return rc;
  }
  if (!direct) {
    RELUX_CUDA_TRY(cudaMemcpyAsync(out, d_out, (size_t)M * N * 4, cudaMemcpyDeviceToHost, st));
    RELUX_CUDA_TRY(cudaStreamSynchronize(st));
  }
  return RELUX_OK;
}

// Validation shared by the two layer entry points; fills the batch with S rows per sequence.
int32_t layer_batch(Pool* p, int layer, int n_seqs, const int32_t* seq_ids, int S, const char* what, SeqBatch* sb) {
  const relux_pool_params& prm = p->prm;
  if (layer < 0 || layer >= prm.num_layers) {
    set_error("layerIdx=%d out of range [0, %d)", layer, prm.num_layers);
    return RELUX_ERR_INVALID_ARG;
  }
  if (n_seqs <= 0 || n_seqs > prm.max_seqs) {
    set_error("n_seqs=%d outside [1, max_seqs=%d]", n_seqs, prm.max_seqs);
    return RELUX_ERR_INVALID_ARG;
  }
  int32_t rc = stage_batch(p, n_seqs, seq_ids, nullptr, S, sb);
  if (rc) return rc;
  for (int i = 0; i < sb->n_seqs; i++) {   // the reference panics on overflow (kvcache.go:282-285, mla_cache.go:160-164)
    const int s = sb->seq[i];
    const int len = p->h_len[(size_t)layer * prm.max_seqs + s], cap = p->seq_pages[s] * prm.page_tokens;
    if (len + S > cap) {
      set_error("%s: layer %d overflow: total=%d + newLen=%d > capacity=%d (sequence %d)", what, layer, len, S, cap, s);
      return RELUX_ERR_OVERFLOW;
    }
  }
  return RELUX_OK;
}

size_t part_bytes(int M, int max_n, bool few_pieces) {
  const size_t piece = (size_t)M * max_n * 4, most = (size_t)64 << 20;
  return pad256(std::max<size_t>(few_pieces ? std::min(most, 8 * piece) : most, piece * 4));
}

}  // namespace

size_t layer_scratch_bytes(int M, int max_k, int max_n, size_t rest_bytes, bool few_pieces) {
  return pad256((size_t)M * max_k * 2) + part_bytes(M, max_n, few_pieces) + rest_bytes;
}
int32_t layer_scratch(Pool* p, int M, int max_k, int max_n, size_t rest_bytes, LayerScratch* out, bool few_pieces) {
  int32_t rc = grow(p->dev, p->layer_buf, layer_scratch_bytes(M, max_k, max_n, rest_bytes, few_pieces));
  if (rc) return rc;
  out->part_cap = part_bytes(M, max_n, few_pieces);
  char* base = (char*)p->layer_buf.p;
  out->a_bf16 = (uint16_t*)base;
  out->part = (float*)(base + pad256((size_t)M * max_k * 2));
  out->rest = (char*)out->part + out->part_cap;
  return RELUX_OK;
}

int32_t do_mla_layer(Pool* p, const relux_mla_layer_args* a) {
  if (!a || !a->w) { set_error("nil argument struct"); return RELUX_ERR_INVALID_ARG; }
  const relux_pool_params& prm = p->prm;
  if (prm.kind != RELUX_POOL_MLA) { set_error("pool kind does not match this call (MLA pool needed)"); return RELUX_ERR_INVALID_ARG; }
  const relux_mla_layer_weights& w = *a->w;
  if (!a->x || !a->out || !w.w_q || !w.w_qr || !w.w_dkv || !w.w_kr || !w.w_uk || !w.w_uv || !w.w_o) {
    set_error("nil input, output or weight pointer");
    return RELUX_ERR_INVALID_ARG;
  }
  const int H = a->num_heads, D = a->d_model, S = a->q_tokens, dC = prm.mla_dc, dHR = prm.mla_dhr;
  if (H <= 0 || D <= 0 || S <= 0 || D % H != 0) {   // NewMLA, mla.go:69-74
    set_error("NewMLA: dModel=%d not divisible by numHeads=%d (or non-positive sizes)", D, H);
    return RELUX_ERR_INVALID_ARG;
  }
  if (dHR % 2 != 0) { set_error("NewMLA: dHR=%d must be even for paired RoPE rotation", dHR); return RELUX_ERR_INVALID_ARG; }
  if (a->mode != RELUX_ATTN_FAST && a->mode != RELUX_ATTN_REFERENCE && a->mode != RELUX_ATTN_REFERENCE_FAITHFUL) { set_error("bad mode"); return RELUX_ERR_INVALID_ARG; }
  const bool faithful = a->mode == RELUX_ATTN_REFERENCE_FAITHFUL;
  if (faithful && !p->compat) { set_error("RELUX_ATTN_REFERENCE_FAITHFUL needs a pool created with RELUX_POOL_FLAG_REFERENCE_COMPAT"); return RELUX_ERR_INVALID_ARG; }
  if (a->x_dtype != RELUX_DTYPE_F32) { set_error("x must be float32"); return RELUX_ERR_UNSUPPORTED; }
  const int Dh = D / H;
  const float rope_base = a->rope_base == 0.f ? 10000.f : a->rope_base;   // NewMLA, mla.go:78-80
  SeqBatch sb;
  int32_t rc = layer_batch(p, a->layer, a->n_seqs, a->seq_ids, S, "MLACache.Append", &sb);
  if (rc) return rc;
  const int M = sb.n_seqs * S;
  rc = ensure_rope_table(p, dHR, rope_base, prm.max_pages_per_seq * prm.page_tokens);
  if (rc) return rc;
  const void* dx = nullptr;
  rc = stage_in(p, p->in_a, a->x, (size_t)M * D * 4, a->x_mem, &dx);
  if (rc) return rc;

  const WeightRef proj[4] = {{w.w_q, H * Dh}, {w.w_qr, H * dHR}, {w.w_dkv, dC}, {w.w_kr, dHR}};
  const WeightRef outp[1] = {{w.w_o, D}};
  const int n_total = H * Dh + H * dHR + dC + dHR;
  const bool fast = a->mode == RELUX_ATTN_FAST;
  const bool mma = fast && !p->tune.get(RELUX_TUNE_GEMM_GENERIC) && gemm_sm100_eligible(D, proj, 4) && gemm_sm100_eligible(H * Dh, outp, 1);
  const size_t q_es = fast ? 2 : 4;
  const size_t b_qc = pad256((size_t)M * H * Dh * q_es), b_qr = pad256((size_t)M * H * dHR * q_es), b_c = pad256((size_t)M * dC * 4),
               b_kr = pad256((size_t)M * dHR * 4);
  LayerScratch sc;
  rc = layer_scratch(p, M, std::max(D, H * Dh), std::max(n_total, D), b_qc + b_qr + b_c + b_kr + (size_t)M * H * Dh * 4, &sc);
  if (rc) return rc;
  void* d_qc = sc.rest;
  void* d_qr = sc.rest + b_qc;
  float* d_c = (float*)(sc.rest + b_qc + b_qr);
  float* d_kr = (float*)(sc.rest + b_qc + b_qr + b_c);
  float* d_attn = (float*)(sc.rest + b_qc + b_qr + b_c + b_kr);
  // 1 + 2. projections, RoPE on q^R and k^R
  const ProjSeg segs[4] = {{H * Dh, 0, d_qc, fast ? 1 : 0, 1}, {H * dHR, dHR, d_qr, fast ? 1 : 0, S > 1}, {dC, 0, d_c, 0, 0}, {dHR, dHR, d_kr, 0, 0}};
  rc = project_and_finish(p, sb, a->layer, (const float*)dx, M, D, S, proj, segs, 4, mma, sc.a_bf16, sc.part, sc.part_cap, faithful);
  if (rc) return rc;
  // 3. append (advances the cursors).  A one-token step on the tensor-core path leaves the append to the attention's
  //    preparation launch (absorb + append + stream partition in one kernel, as relux_mla_step does).
  relux_attn_args probe;
  memset(&probe, 0, sizeof(probe));
  probe.mode = a->mode;
  probe.num_heads = H;
  probe.head_dim = Dh;
  probe.q_tokens = S;
  const bool fused_append = fast && S == 1 && mla_step_fusable(p, probe);
  if (!fused_append) {
    rc = launch_mla_append(p, sb, a->layer, d_c, d_kr, RELUX_DTYPE_F32, 1);
    if (rc) return rc;
  }
  for (int i = 0; i < sb.n_seqs; i++) {
    int32_t& len = p->h_len[(size_t)a->layer * prm.max_seqs + sb.seq[i]];
    note_append(p, a->layer, sb.seq[i], len, S);
    len += S;
  }
  // 4. attention over the cache, the S new rows included
  relux_attn_args aa;
  memset(&aa, 0, sizeof(aa));
  aa.layer = a->layer;
  aa.n_seqs = sb.n_seqs;
  aa.seq_ids = a->seq_ids;
  aa.q_tokens = S;
  aa.extra_tokens = 0;
  aa.causal = a->causal;
  aa.num_heads = H;
  aa.head_dim = Dh;
  aa.scale = (float)(1.0 / std::sqrt((double)(Dh + dHR)));   // mla.go:344-345
  aa.q_dtype = fast ? RELUX_DTYPE_BF16 : RELUX_DTYPE_F32;
  aa.q_layout = RELUX_LAYOUT_TOKEN_MAJOR;
  aa.w_uk = w.w_uk;
  aa.w_uv = w.w_uv;
  aa.mode = a->mode;
  const StepAppend step{d_c, d_kr, RELUX_DTYPE_F32, nullptr, 1, 1, mma};   // one row per sequence
  const bool o_bf16 = mma && mla_writes_bf16(p, sb, aa);   // the output projection's operand, rounded by the kernel that makes it
  rc = fast ? launch_mla_decode_fast(p, sb, aa, d_qc, d_qr, o_bf16 ? (void*)sc.a_bf16 : d_attn, o_bf16, fused_append ? &step : nullptr)
            : launch_attn_reference_mla(p, sb, aa, (const float*)d_qc, (const float*)d_qr, d_attn);
  // 5. output projection
  if (!rc) rc = output_projection(p, o_bf16 ? nullptr : d_attn, M, H * Dh, w.w_o, D, mma, sc.a_bf16, sc.part, sc.part_cap, a->out, a->out_mem);
  if (rc) take_rows_back(p, sb, a->layer);   // a call that fails leaves the lengths as they were
  return rc;
}

// ---- the attention half of a block: what relux_gqa_block_cached adds to a layer step ----
namespace {

struct BlockScratch {
  uint16_t* y;        // the norm's rows, then attention's, as bf16 [M][D]
  int8_t* codes;      // and in 8 bits
  float* scales;
  float* projected;   // [M][n_q + n_k + n_v], a projection behind the other
  char* rest;
};
int32_t block_scratch(Pool* p, int M, int D, int n_total, size_t rest_bytes, BlockScratch* out) {
  const size_t off_codes = pad256((size_t)M * D * 2), off_scales = off_codes + pad256((size_t)M * D), off_proj = off_scales + pad256((size_t)M * 4),
               off_rest = off_proj + pad256((size_t)M * n_total * 4);
  if (int32_t rc = grow(p->dev, p->block_buf, off_rest + rest_bytes)) return rc;
  char* base = (char*)p->block_buf.p;
  *out = BlockScratch{(uint16_t*)base, (int8_t*)(base + off_codes), (float*)(base + off_scales), (float*)(base + off_proj), base + off_rest};
  return RELUX_OK;
}

relux_rmsnorm_args block_norm(const relux_gqa_layer_args* a, const relux_gqa_block_args* b, const void* x, int M) {
  relux_rmsnorm_args n;
  memset(&n, 0, sizeof(n));
  n.n_rows = M;
  n.d = a->d_model;
  n.eps = b->eps;
  n.x_dtype = a->x_dtype;
  n.residual_dtype = b->residual_dtype;
  n.weight_dtype = b->norm_dtype;
  n.x = x;
  n.residual = b->residual;
  n.weight = b->norm_weight;
  n.residual_out = b->residual_out;
  return n;
}

// Before anything is launched or written to the cache.
int32_t check_block(Pool* p, const relux_gqa_layer_args* a, const relux_gqa_block_args* b) {
  if (a->mode != RELUX_ATTN_FAST) { set_error("a block runs in RELUX_ATTN_FAST only"); return RELUX_ERR_UNSUPPORTED; }
  for (int i = 0; i < 3; i++)
    if (b->reserved[i]) { set_error("reserved fields must be zero"); return RELUX_ERR_INVALID_ARG; }
  int32_t rc;
  bool lora = false;
  for (const relux_block_projection* q : {&b->q, &b->k, &b->v, &b->o}) {
    if ((q->codes == nullptr) != (q->scales == nullptr) || (q->lora_a == nullptr) != (q->lora_b == nullptr)) {
      set_error("a block's projection: codes need scales, and lora_a lora_b");
      return RELUX_ERR_INVALID_ARG;
    }
    if ((rc = check_dev_align(q->codes, "codes")) || (rc = check_dev_align(q->scales, "scales")) || (rc = check_dev_align(q->lora_a, "lora_a")) ||
        (rc = check_dev_align(q->lora_b, "lora_b")) || (rc = check_dev_align(q->factors, "factors")))
      return rc;
    lora = lora || q->lora_a;
  }
  if (a->out_mem == RELUX_MEM_DEVICE && (rc = check_dev_align(a->out, "out"))) return rc;
  relux_rmsnorm_args n = block_norm(a, b, a->x, 1);
  n.out = (void*)16;   // an output is given later
  if (a->x_mem == RELUX_MEM_HOST) n.x = n.out;
  if ((rc = check_rmsnorm(&n))) return rc;
  if (!lora) return RELUX_OK;
  if (!b->adapter || b->n_slots <= 0) { set_error("a block's adapters need the requests' slots"); return RELUX_ERR_INVALID_ARG; }
  if (b->rank != 8 && b->rank != 16 && b->rank != 32 && b->rank != 64 && b->rank != 128) { set_error("rank=%d must be one of 8, 16, 32, 64, 128", b->rank); return RELUX_ERR_UNSUPPORTED; }
  for (int i = 0; i < a->n_seqs && a->n_seqs <= p->prm.max_seqs; i++)
    if (b->adapter[i] < -1 || b->adapter[i] >= b->n_slots) {
      set_error("adapter %d of request %d outside [-1, %d)", b->adapter[i], i, b->n_slots);
      return RELUX_ERR_INVALID_ARG;
    }
  return RELUX_OK;
}

relux_matmul_lora_args block_adapters(int M, int K, int N, const relux_gqa_block_args* b, const relux_block_projection& q, const void* w, const void* y, bool y_f32, int n_seqs,
                                      const int32_t* rows_each, float* dst) {
  relux_matmul_lora_args l;
  memset(&l, 0, sizeof(l));
  l.m = M;
  l.k = K;
  l.n = N;
  l.rank = b->rank;
  l.n_slots = b->n_slots;
  l.n_seqs = n_seqs;
  l.x_dtype = y_f32 ? RELUX_DTYPE_F32 : RELUX_DTYPE_BF16;
  l.out_dtype = RELUX_DTYPE_F32;
  l.accumulate = q.codes != nullptr;
  l.x = y;
  l.w = q.codes ? nullptr : w;
  l.lora_a = q.lora_a;
  l.lora_b = q.lora_b;
  l.factors = q.factors;
  l.adapter = b->adapter;
  l.n_rows = rows_each;
  l.out = dst;
  return l;
}

// Room for all that a block's projections ask for, before anything of the call is launched: none of them allocates on its way.  attn_f32: attention's rows come as float32.
int32_t reserve_projections(Pool* p, const relux_gqa_layer_args* a, const relux_gqa_block_args* b, int M, const WeightRef* proj, const WeightRef& outp, int n_total, bool attn_f32,
                            int n_seqs, const int32_t* rows_each) {
  const int D = a->d_model;
  const relux_block_projection* q[4] = {&b->q, &b->k, &b->v, &b->o};
  const WeightRef w[4] = {proj[0], proj[1], proj[2], outp};
  bool joint = true;
  for (int j = 0; j < 3; j++) joint = joint && !q[j]->codes && !q[j]->lora_a;
  size_t most = joint ? layer_scratch_bytes(M, D, n_total, 0) : 0;
  for (int j = joint ? 3 : 0; j < 4; j++) {
    if (q[j]->lora_a) {
      const relux_matmul_lora_args l = block_adapters(M, D, w[j].n, b, *q[j], w[j].w, nullptr, j == 3 && attn_f32, n_seqs, rows_each, nullptr);
      most = std::max(most, matmul_lora_scratch(p, &l));
    } else if (!q[j]->codes) {
      most = std::max(most, layer_scratch_bytes(M, D, w[j].n, 0));
    }
  }
  int32_t rc = grow(p->dev, p->layer_buf, most);
  if (!rc && a->out_mem != RELUX_MEM_DEVICE) rc = grow(p->dev, p->out_buf, (size_t)M * D * 4);
  return rc;
}

// dst [M][N] f32 = rows x one projection of a block: its 8-bit or bf16 weights, and its adapters.  y: the rows as bf16 or (y_f32) float32, codes: in 8 bits, each
// where it is needed.
int32_t project_one(Pool* p, int M, int K, int N, const relux_gqa_block_args* b, const relux_block_projection& q, const void* w, const void* y, bool y_f32,
                    const BlockScratch& bs, int n_seqs, const int32_t* rows_each, float* dst) {
  int32_t rc;
  if (q.codes)
    if ((rc = launch_matmul_int8(p, M, K, N, bs.codes, bs.scales, q.codes, q.scales, dst, false))) return rc;
  if (q.lora_a) {
    const relux_matmul_lora_args l = block_adapters(M, K, N, b, q, w, y, y_f32, n_seqs, rows_each, dst);
    return do_matmul_lora(p, &l);
  }
  if (q.codes) return RELUX_OK;
  LayerScratch sc;
  if ((rc = layer_scratch(p, M, K, N, 0, &sc))) return rc;
  return output_projection(p, y_f32 ? (const float*)y : nullptr, M, K, w, N, true, y_f32 ? sc.a_bf16 : (uint16_t*)y, sc.part, sc.part_cap, dst, RELUX_MEM_DEVICE);
}

// h = x + residual, its norm, and q, k, v in their buffers.
int32_t block_projections(Pool* p, const SeqBatch& sb, const relux_gqa_layer_args* a, const relux_gqa_block_args* b, const void* dx, int M, const WeightRef* proj,
                          ProjSeg* segs, const BlockScratch& bs, const int32_t* rows_each) {
  const relux_block_projection* q[3] = {&b->q, &b->k, &b->v};
  bool wants_bf16 = false, wants_codes = false, joint = true;
  for (const relux_block_projection* r : q) {
    wants_bf16 = wants_bf16 || !r->codes || r->lora_a;
    wants_codes = wants_codes || r->codes;
    joint = joint && !r->codes && !r->lora_a;
  }
  relux_rmsnorm_args n = block_norm(a, b, dx, M);
  n.out_dtype = RELUX_DTYPE_BF16;
  n.out = wants_bf16 ? bs.y : nullptr;
  n.codes = wants_codes ? bs.codes : nullptr;
  n.scales = wants_codes ? bs.scales : nullptr;
  int32_t rc;
  if (joint) {
    int n_total = 0;
    for (int j = 0; j < 3; j++) n_total += proj[j].n;
    LayerScratch sc;
    if ((rc = layer_scratch(p, M, a->d_model, n_total, 0, &sc))) return rc;
    return project_and_finish(p, sb, a->layer, nullptr, M, a->d_model, a->q_tokens, proj, segs, 3, true, bs.y, sc.part, sc.part_cap, false, &n);
  }
  if ((rc = do_rmsnorm(p, &n))) return rc;
  float* dst = bs.projected;
  for (int j = 0; j < 3; j++) {
    if ((rc = project_one(p, M, a->d_model, proj[j].n, b, *q[j], proj[j].w, bs.y, false, bs, sb.n_seqs, rows_each, dst))) return rc;
    segs[j].src = dst;
    dst += (size_t)M * proj[j].n;
  }
  time_none(p->proj_times);
  return finish_projections(p, sb, a->layer, M, a->q_tokens, segs, 3, nullptr, GemmRanges{}, false);
}

// out [M][d_model] = attention's rows x W_O.
int32_t block_output(Pool* p, const relux_gqa_layer_args* a, const relux_gqa_block_args* b, const void* attn, bool attn_bf16, int M, int K, const BlockScratch& bs,
                     const int32_t* rows_each) {
  const int N = a->d_model;
  const bool direct = a->out_mem == RELUX_MEM_DEVICE;
  int32_t rc;
  if (!direct && (rc = grow(p->dev, p->out_buf, (size_t)M * N * 4))) return rc;
  float* dst = direct ? (float*)a->out : (float*)p->out_buf.p;
  if (b->o.codes) {
    const relux_int8_rows_args r{M, K, attn_bf16 ? RELUX_DTYPE_BF16 : RELUX_DTYPE_F32, 0, attn, bs.codes, bs.scales};
    if ((rc = do_int8_rows(p, &r))) return rc;
  }
  if ((rc = project_one(p, M, K, N, b, b->o, a->w->w_o, attn, !attn_bf16, bs, M / a->q_tokens, rows_each, dst))) return rc;
  if (!direct) {
    RELUX_CUDA_TRY(cudaMemcpyAsync(a->out, dst, (size_t)M * N * 4, cudaMemcpyDeviceToHost, p->dev->stream));
    RELUX_CUDA_TRY(cudaStreamSynchronize(p->dev->stream));
  }
  return RELUX_OK;
}

}  // namespace

// MHA.forwardCached (mha.go:245-369) for a batch of independent sequences: projections with Wq / Wk / Wv, RoPE on q
// and k at position cacheLen + s (when the layer has a rotary embedding), append of k / v, GQA attention, Wo.  With b the attention half of a
// block around it: the residual's addition and the norm first, and projections with adapters or 8-bit weights.
static int32_t gqa_layer(Pool* p, const relux_gqa_layer_args* a, const relux_gqa_block_args* b) {
  if (!a || !a->w) { set_error("nil argument struct"); return RELUX_ERR_INVALID_ARG; }
  const relux_pool_params& prm = p->prm;
  if (prm.kind != RELUX_POOL_GQA) { set_error("pool kind does not match this call (GQA pool needed)"); return RELUX_ERR_INVALID_ARG; }
  const relux_gqa_layer_weights& w = *a->w;
  const relux_block_projection none{}, bq = b ? b->q : none, bk = b ? b->k : none, bv = b ? b->v : none, bo = b ? b->o : none;
  if (!a->x || !a->out || (!w.w_q && !bq.codes) || (!w.w_k && !bk.codes) || (!w.w_v && !bv.codes) || (!w.w_o && !bo.codes)) {
    set_error("nil input, output or weight pointer");
    return RELUX_ERR_INVALID_ARG;
  }
  const int H = a->num_heads, D = a->d_model, S = a->q_tokens, Hkv = prm.gqa_num_kv_heads, hd = prm.gqa_head_dim;
  if (H <= 0 || D <= 0 || S <= 0 || D % H != 0 || D / H != hd || H % Hkv != 0) {   // NewMHAGQA, mha.go
    set_error("dModel=%d / numHeads=%d must equal the pool's head_dim=%d, numHeads a multiple of numKVHeads=%d", D, H, hd, Hkv);
    return RELUX_ERR_INVALID_ARG;
  }
  if (a->rope && hd % 2 != 0) { set_error("NewRotaryEmbedding: headDim=%d, must be even and > 0", hd); return RELUX_ERR_INVALID_ARG; }
  if (a->mode != RELUX_ATTN_FAST && a->mode != RELUX_ATTN_REFERENCE && a->mode != RELUX_ATTN_REFERENCE_FAITHFUL) { set_error("bad mode"); return RELUX_ERR_INVALID_ARG; }
  const bool faithful = a->mode == RELUX_ATTN_REFERENCE_FAITHFUL;
  if (faithful && (!p->compat || !a->advance)) { set_error("RELUX_ATTN_REFERENCE_FAITHFUL needs a pool created with RELUX_POOL_FLAG_REFERENCE_COMPAT and advance != 0"); return RELUX_ERR_INVALID_ARG; }
  const bool x_bf16 = b && a->x_dtype == RELUX_DTYPE_BF16;
  if (a->x_dtype != RELUX_DTYPE_F32 && !x_bf16) { set_error("x must be float32"); return RELUX_ERR_UNSUPPORTED; }
  if (p->int8 && a->mode != RELUX_ATTN_FAST) { set_error("a pool of 8-bit rows takes RELUX_ATTN_FAST only"); return RELUX_ERR_UNSUPPORTED; }
  if (a->mode == RELUX_ATTN_FAST && (!p->has_tmap || prm.page_tokens != 64 || hd != 128 || H / Hkv > 32)) {
    // checked before anything is written to the cache
    set_error("GQA FAST kernels need page_tokens=64, head_dim=128 and num_heads/num_kv_heads <= 32 "
              "(got page_tokens=%d head_dim=%d group=%d); use RELUX_ATTN_REFERENCE for other shapes", prm.page_tokens, hd, H / Hkv);
    return RELUX_ERR_UNSUPPORTED;
  }
  if (b)
    if (int32_t rc = check_block(p, a, b)) return rc;
  const float rope_base = a->rope_base == 0.f ? 10000.f : a->rope_base;
  SeqBatch sb;
  int32_t rc = layer_batch(p, a->layer, a->n_seqs, a->seq_ids, S, "Append", &sb);
  if (rc) return rc;
  const int M = sb.n_seqs * S;
  if (a->rope) {
    rc = ensure_rope_table(p, hd, rope_base, prm.max_pages_per_seq * prm.page_tokens);
    if (rc) return rc;
  }
  const void* dx = nullptr;
  rc = stage_in(p, p->in_a, a->x, (size_t)M * D * (x_bf16 ? 2 : 4), a->x_mem, &dx);
  if (rc) return rc;
  const WeightRef proj[3] = {{w.w_q, H * hd}, {w.w_k, Hkv * hd}, {w.w_v, Hkv * hd}};
  const WeightRef outp[1] = {{w.w_o, D}};
  const int n_total = (H + 2 * Hkv) * hd;
  const bool fast = a->mode == RELUX_ATTN_FAST;
  const bool mma = fast && !p->tune.get(RELUX_TUNE_GEMM_GENERIC) && gemm_sm100_eligible(D, proj, 3) && gemm_sm100_eligible(H * hd, outp, 1);
  if (b && !mma) { set_error("a block needs the tensor-core projections: knob RELUX_TUNE_GEMM_GENERIC is set, or a weight is not 16-byte aligned"); return RELUX_ERR_UNSUPPORTED; }
  const size_t q_es = fast ? 2 : 4;
  const size_t b_q = pad256((size_t)M * H * hd * q_es), b_kv = pad256((size_t)M * Hkv * hd * 4);
  LayerScratch sc{};
  BlockScratch bs{};
  if (b) {   // in a block of its own: projections with adapters use the layers' scratch themselves
    rc = block_scratch(p, M, D, n_total, b_q + 2 * b_kv + (size_t)M * H * hd * 4, &bs);
    sc.rest = bs.rest;
    sc.a_bf16 = bs.y;
  } else {
    rc = layer_scratch(p, M, std::max(D, H * hd), std::max(n_total, D), b_q + 2 * b_kv + (size_t)M * H * hd * 4, &sc);
  }
  if (rc) return rc;
  void* d_q = sc.rest;
  float* d_k = (float*)(sc.rest + b_q);
  float* d_v = (float*)(sc.rest + b_q + b_kv);
  float* d_attn = (float*)(sc.rest + b_q + 2 * b_kv);
  relux_attn_args aa;
  memset(&aa, 0, sizeof(aa));
  aa.mode = a->mode;
  aa.num_heads = H;
  aa.q_tokens = S;
  aa.extra_tokens = a->advance ? 0 : S;
  const bool fused_append = fast && gqa_append_fusable(p, aa, S, a->advance != 0);
  const bool o_bf16 = mma && fused_append;   // the output projection's operand, rounded by the kernel that makes it
  const int rd = a->rope ? hd : 0;
  ProjSeg segs[3] = {{H * hd, rd, d_q, fast ? 1 : 0, S > 1}, {Hkv * hd, rd, d_k, 0, 0}, {Hkv * hd, 0, d_v, 0, 0}};
  std::vector<int32_t> rows_each;
  if (b) {
    rows_each.assign((size_t)sb.n_seqs, S);
    rc = reserve_projections(p, a, b, M, proj, outp[0], n_total, !o_bf16, sb.n_seqs, rows_each.data());
    if (!rc) rc = block_projections(p, sb, a, b, dx, M, proj, segs, bs, rows_each.data());
  } else {
    rc = project_and_finish(p, sb, a->layer, (const float*)dx, M, D, S, proj, segs, 3, mma, sc.a_bf16, sc.part, sc.part_cap, faithful);
  }
  if (rc) return rc;
  // append: the GEMM rows are token-major [row][Hkv][hd]; advance = 0 leaves the rows past the cursor (verify).  A short
  // step leaves the append to the attention launch.
  if (!fused_append) {
    rc = launch_gqa_append(p, sb, a->layer, d_k, d_v, RELUX_DTYPE_F32, RELUX_LAYOUT_TOKEN_MAJOR, a->advance);
    if (rc) return rc;
  }
  if (a->advance)
    for (int i = 0; i < sb.n_seqs; i++) {
      int32_t& len = p->h_len[(size_t)a->layer * prm.max_seqs + sb.seq[i]];
      note_append(p, a->layer, sb.seq[i], len, S);
      len += S;
    }
  aa.layer = a->layer;
  aa.n_seqs = sb.n_seqs;
  aa.seq_ids = a->seq_ids;
  aa.causal = a->causal;
  aa.head_dim = hd;
  aa.scale = (float)(1.0 / std::sqrt((double)hd));   // mha.go:319
  aa.q_dtype = fast ? RELUX_DTYPE_BF16 : RELUX_DTYPE_F32;
  aa.q_layout = RELUX_LAYOUT_TOKEN_MAJOR;
  const GqaAppend app{d_k, d_v, RELUX_DTYPE_F32, RELUX_LAYOUT_TOKEN_MAJOR, a->advance ? 1 : 0, sb.rows.data()};
  rc = fused_append ? launch_gqa_stream(p, sb, aa, d_q, o_bf16 ? (void*)sc.a_bf16 : d_attn, o_bf16, &app)
       : fast       ? launch_gqa_decode_fast(p, sb, aa, d_q, d_attn)
                    : launch_attn_reference_gqa(p, sb, aa, (const float*)d_q, d_attn);
  if (!rc)
    rc = b ? block_output(p, a, b, o_bf16 ? (const void*)sc.a_bf16 : d_attn, o_bf16, M, H * hd, bs, rows_each.data())
           : output_projection(p, o_bf16 ? nullptr : d_attn, M, H * hd, w.w_o, D, mma, sc.a_bf16, sc.part, sc.part_cap, a->out, a->out_mem);
  if (rc && a->advance) take_rows_back(p, sb, a->layer);   // a call that fails leaves the lengths as they were
  return rc;
}
int32_t do_gqa_layer(Pool* p, const relux_gqa_layer_args* a) { return gqa_layer(p, a, nullptr); }
int32_t do_gqa_block(Pool* p, const relux_gqa_layer_args* a, const relux_gqa_block_args* b) {
  if (!b) { set_error("nil argument struct"); return RELUX_ERR_INVALID_ARG; }
  return gqa_layer(p, a, b);
}


// ComputeBackend.MatMulFloat32 as matmulBatched3D uses it (interface.go:25-29, mha.go:759-785): C = A x B with A, C float32
// and B a bf16 weight matrix [K][N] on the device.
int32_t do_matmul(Pool* p, const relux_matmul_args* a) {
  if (!a || !a->a || !a->b || !a->c) { set_error("nil argument"); return RELUX_ERR_INVALID_ARG; }
  const int M = a->m, K = a->k, N = a->n;
  if (M <= 0 || K <= 0 || N <= 0) { set_error("MatMulFloat32: M=%d K=%d N=%d must be positive", M, K, N); return RELUX_ERR_INVALID_ARG; }
  if (a->mode != RELUX_ATTN_FAST && a->mode != RELUX_ATTN_REFERENCE) { set_error("bad mode"); return RELUX_ERR_INVALID_ARG; }
  for (int i = 0; i < 4; i++)
    if (a->reserved[i]) { set_error("reserved fields must be zero"); return RELUX_ERR_INVALID_ARG; }
  int32_t rc;
  if ((rc = check_dev_align(a->b, "B"))) return rc;
  if (a->a_mem == RELUX_MEM_DEVICE && (rc = check_dev_align(a->a, "A"))) return rc;
  if (a->c_mem == RELUX_MEM_DEVICE && (rc = check_dev_align(a->c, "C"))) return rc;
  const WeightRef w[1] = {{a->b, N}};
  const bool fast = a->mode == RELUX_ATTN_FAST;
  if (fast && (p->tune.get(RELUX_TUNE_GEMM_GENERIC) || !gemm_sm100_eligible(K, w, 1) || N % 4 != 0)) {
    set_error("MatMulFloat32 FAST needs K and N multiples of 8 (got K=%d N=%d); use RELUX_ATTN_REFERENCE", K, N);
    return RELUX_ERR_UNSUPPORTED;
  }
  const void* dA = nullptr;
  rc = stage_in(p, p->in_a, a->a, (size_t)M * K * 4, a->a_mem, &dA);
  if (rc) return rc;
  LayerScratch sc;
  rc = layer_scratch(p, M, K, N, 0, &sc);
  if (rc) return rc;
  return output_projection(p, (const float*)dA, M, K, a->b, N, fast, sc.a_bf16, sc.part, sc.part_cap, a->c, a->c_mem);
}

}  // namespace relux
