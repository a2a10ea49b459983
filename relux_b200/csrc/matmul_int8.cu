// Product of 8-bit rows with 8-bit weights on the tensor cores: C[m][n] = sa[m] * sw[n] * sum_k a[m][k] * w[n][k], the sum in 32-bit whole
// numbers, exact for every K that the call takes, whatever the order of its parts.
//
// Bound: HBM up to some hundred rows (a weight is one byte, read once), the tensor cores above.  The layout is that of the bf16 projections
// (skinny_gemm_sm100_kernel): the weights are the M = 128 operand, 16 to 256 activation rows the N operand, a stage is 128 bytes of K of both, and
// one CTA per SM walks its share of the tiles (GemmRanges) without draining its pipeline.  What differs:
//   * both operands lie K-major, as the quantiser and the import write them;
//   * a tile that one CTA does alone leaves it as the result, scaled and rounded; a tile that is cut along K is joined by the CTA whose piece is done
//     last: whole numbers add up to the same sum in any order, so the join needs no order and no launch of its own;
//   * the weights of a worker's first steps are brought into L2, not into shared memory, while the launch before this one ends: a prefetch
//     returns no data, so it may be early whatever that launch writes.
#include <algorithm>

#include "common.cuh"
#include "internal.h"
#include "projection.cuh"
#include "umma.cuh"

namespace relux {

namespace {

constexpr int kStepK = 128;                        // bytes of K of a step
constexpr int kStageWeights = kGemmTileCols * kStepK;
constexpr int kMaxBlockRows = 256;
constexpr int kPrefetchSteps = 16;

template <int NT>
struct Int8Shape {
  static constexpr int kStage = kStageWeights + NT * kStepK;
  static constexpr int kStages = (232448 - 1024) / kStage;
  static constexpr int kSmem = kStages * kStage + 1024;
  static constexpr int kAcc = NT < 32 ? 32 : NT;
};
struct Int8Bars {
  uint64_t full[12], empty[12], acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  volatile int32_t abort_flag, last;
};
static_assert(Int8Shape<16>::kStages <= 12 && sizeof(Int8Bars) <= 1024, "barrier block too small");

struct Int8Maps {
  CUtensorMap a, w;   // rows of K bytes, seen as rows of K / 2 elements of two bytes
};
struct Int8Params {
  GemmRanges rg;
  int32_t M, N, max_pieces, out_bf16;
  const float* a_scale;
  const float* w_scale;
  void* out;
  int32_t* part;      // [slot][piece][row of the block][128]
  int32_t* arrived;   // [slot], zero between launches
  int32_t* status;
};

__device__ __noinline__ void int8_wait_slow(uint64_t* bar, uint32_t parity, Int8Bars* b, int32_t* status) {
  for (uint32_t i = 0; i < kSpinLimit; i++) {
    if (mbar_try_wait(bar, parity)) return;
    if ((i & 255) == 255 && b->abort_flag) return;
    if (i > 512) __nanosleep(20);
  }
  b->abort_flag = 1;
  set_status(status, RELUX_ERR_TIMEOUT);
}
// Bounded: a wait that runs out records RELUX_ERR_TIMEOUT and raises the CTA's abort flag; nobody leaves a loop early.
__device__ __forceinline__ void int8_wait(uint64_t* bar, uint32_t parity, Int8Bars* b, int32_t* status) {
  if (!mbar_try_wait(bar, parity)) int8_wait_slow(bar, parity, b, status);
}
__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// grid (workers), 192 threads: warps 0-3 epilogue, warp 4 TMA producer, warp 5 MMA issuer.
template <int NT>
__global__ void __launch_bounds__(192, 1) matmul_int8_kernel(const __grid_constant__ Int8Maps maps, const __grid_constant__ Int8Params prm) {
  using SH = Int8Shape<NT>;
  constexpr int kStages = SH::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  Int8Bars* bars = reinterpret_cast<Int8Bars*>(smem + kStages * SH::kStage);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr bool kBlocks = NT >= 128;   // smaller blocks hold all rows
  GemmWalk<kBlocks> walk(prm.rg, blockIdx.x);
  chain_release();
  if ((smem_u32(smem) & 1023u) != 0) {
    chain_wait();
    if (threadIdx.x == 0) set_status(prm.status, RELUX_ERR_UNSUPPORTED);
    return;
  }
  if (threadIdx.x == 0) {
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
    if (el) {
      tma_prefetch_desc(&maps.a);
      tma_prefetch_desc(&maps.w);
    }
    auto ahead = walk;
    for (int g = 0; g < kPrefetchSteps && ahead.next();)
      for (int k = ahead.k0; k < ahead.k1 && g < kPrefetchSteps; k++, g++)
        if (el) tma_prefetch_2d(&maps.w, k * (kStepK / 2), ahead.col * kGemmTileCols);
    chain_wait();
    int g = 0;
    while (walk.next())
      for (int k = walk.k0; k < walk.k1; k++, g++) {
        const int s = g % kStages;
        if (g >= kStages) int8_wait(&bars->empty[s], (g / kStages - 1) & 1, bars, prm.status);
        if (el) {
          uint8_t* st = smem + s * SH::kStage;
          mbar_expect_tx(&bars->full[s], SH::kStage);   // out-of-range parts of a box are zero-filled and still counted
          tma_load_2d(st, &maps.w, k * (kStepK / 2), walk.col * kGemmTileCols, &bars->full[s]);
          tma_load_2d(st + kStageWeights, &maps.a, k * (kStepK / 2), kBlocks ? walk.block * NT : 0, &bars->full[s]);
        }
        __syncwarp();
      }
  } else if (warp == 5) {
    const bool el = elect_one();
    const uint32_t idesc = make_idesc_s8(kGemmTileCols, NT);
    int g = 0;
    for (int piece = 0; walk.next(); piece++) {
      const uint32_t d = tmem + (piece & 1) * SH::kAcc;
      if (piece >= 2) int8_wait(&bars->acc_empty[piece & 1], ((piece >> 1) - 1) & 1, bars, prm.status);
      tc_fence_after();
      for (int k = walk.k0; k < walk.k1; k++, g++) {
        const int s = g % kStages;
        int8_wait(&bars->full[s], (g / kStages) & 1, bars, prm.status);
        tc_fence_after();
        if (el) {
          const uint32_t st = smem_u32(smem + s * SH::kStage);
          const uint64_t dW = make_desc_kmajor_sw128(st), dX = make_desc_kmajor_sw128(st + kStageWeights);
#pragma unroll
          for (int kk = 0; kk < kStepK / 32; kk++)
            umma_ss_i8(d, dW + ((uint32_t)(kk * 32) >> 4), dX + ((uint32_t)(kk * 32) >> 4), idesc, k != walk.k0 || kk != 0);
          umma_commit<1>(&bars->empty[s]);
        }
        __syncwarp();
      }
      if (el) umma_commit<1>(&bars->acc_full[piece & 1]);
      __syncwarp();
    }
  } else {
    // thread = weight column, accumulator column = activation row
    chain_wait();
    for (int piece = 0; walk.next(); piece++) {
      const int block = kBlocks ? walk.block : 0, m0 = block * NT, n = walk.col * kGemmTileCols + warp * 32 + lane;
      const int m_end = min(NT, prm.M - m0);
      const int tile = prm.rg.tile_of(walk.col, m0), pieces = prm.rg.pieces(tile);
      const bool mine = n < prm.N;
      const float sw = mine ? load_chained(prm.w_scale + n) : 0.f;
      int8_wait(&bars->acc_full[piece & 1], (piece >> 1) & 1, bars, prm.status);
      tc_fence_after();
      const bool ok = !bars->abort_flag;
      const uint32_t acc = tmem + ((uint32_t)(warp * 32) << 16) + (piece & 1) * SH::kAcc;
      const int slot = (tile - prm.rg.full * prm.rg.workers) * prm.rg.beside + (kBlocks ? block % prm.rg.beside : 0);
      int32_t* const parts = prm.part + (size_t)slot * prm.max_pieces * NT * kGemmTileCols + warp * 32 + lane;
      bool finish = m_end > 0;   // (blocks beside each other may reach past the last row)
      if (pieces > 1 && m_end > 0) {
        int32_t* dst = parts + (size_t)walk.split * NT * kGemmTileCols;
#pragma unroll 1
        for (int c = 0; c < m_end; c += 32) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(acc + c, v);
          tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 32; q++)
            if (c + q < m_end) dst[(c + q) * kGemmTileCols] = (int32_t)v[q];
        }
        __threadfence();
        epilogue_sync();
        if (threadIdx.x == 0) {
          const bool last = atomicAdd(prm.arrived + slot, 1) == pieces - 1;
          if (last) prm.arrived[slot] = 0;
          bars->last = last;
          __threadfence();
        }
        epilogue_sync();
        finish = bars->last != 0;
      }
      if (finish)
#pragma unroll 1
        for (int c = 0; c < m_end; c += 32) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(acc + c, v);
          const float sa_mine = c + lane < m_end ? load_chained(prm.a_scale + m0 + c + lane) : 0.f;
          tmem_ld_wait();
          if (pieces > 1)
            for (int s = 0; s < pieces; s++)
              if (s != walk.split) {
                const int32_t* src = parts + ((size_t)s * NT + c) * kGemmTileCols;
#pragma unroll
                for (int q = 0; q < 32; q++)
                  if (c + q < m_end) v[q] += (uint32_t)load_chained(src + q * kGemmTileCols);
              }
          const size_t at = (size_t)(m0 + c) * prm.N + n;
#pragma unroll
          for (int q = 0; q < 32; q++) {
            const float sa = __shfl_sync(0xffffffffu, sa_mine, q);
            const float x = ok ? __fmul_rn(__fmul_rn((float)(int32_t)v[q], sa), sw) : 0.f;
            if (mine && c + q < m_end) {
              if (prm.out_bf16) reinterpret_cast<__nv_bfloat16*>(prm.out)[at + (size_t)q * prm.N] = __float2bfloat16_rn(x);
              else reinterpret_cast<float*>(prm.out)[at + (size_t)q * prm.N] = x;
            }
          }
        }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->acc_empty[piece & 1]);
    }
    fence_chained_writes();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc<1>(tmem, 2 * SH::kAcc);
}

template <int NT>
int32_t launch_rows(Pool* p, const Int8Maps& maps, const Int8Params& prm, int workers) {
  if (int32_t rc = allow_smem(p->dev, matmul_int8_kernel<NT>, Int8Shape<NT>::kSmem)) return rc;
  RELUX_CUDA_TRY(launch_chained(p->tune.get(RELUX_TUNE_CHAINED_LAUNCHES) != 0, matmul_int8_kernel<NT>, dim3(workers), dim3(192),
                                (size_t)Int8Shape<NT>::kSmem, p->dev->stream, maps, prm));
  count_launch(p->dev);
  return RELUX_OK;
}

}  // namespace

int32_t launch_matmul_int8(Pool* p, int M, int K, int N, const int8_t* a, const float* a_scale, const int8_t* w, const float* w_scale, void* out,
                           bool out_bf16) {
  Int8Params prm{};
  const int tiles = (N + kGemmTileCols - 1) / kGemmTileCols, steps = (K + kStepK - 1) / kStepK;
  if ((int64_t)tiles * ((M + 127) / 128) * steps >= (int64_t)1 << 31) { set_error("a product of more than 2^31 steps"); return RELUX_ERR_UNSUPPORTED; }
  // blocks of rows and how many beside each other: as launch_skinny_gemm, whose steps move the same bytes in the same time
  int nt = 16;
  while (nt < M && nt < kMaxBlockRows) nt *= 2;
  double best = 0;
  for (int rows = nt; rows >= std::min(nt, 128); rows /= 2)
    for (int beside = std::min(16, (M + rows - 1) / rows); beside >= 1; beside--) {
      double cost = 0;
      const GemmRanges r = deal_tiles(p->dev->sm_count, tiles, M, rows, beside, steps, N, (double)K * N, 64, 0, &cost);
      if (!prm.rg.workers || cost < best) {
        prm.rg = r;
        best = cost;
      }
    }
  const GemmRanges& rg = prm.rg;
  nt = rg.block_rows;
  int slots = rg.rest * rg.beside;
  prm.max_pieces = 1;
  for (int t = 0; t < rg.rest; t++) prm.max_pieces = std::max(prm.max_pieces, rg.pieces(rg.full * rg.workers + t));
  if (prm.max_pieces == 1) slots = 0;
  if (slots > Pool::kArrived) {   // (tiles that are cut are fewer than the workers)
    set_error("matmul_int8: %d tiles in pieces", slots);
    return RELUX_ERR_UNSUPPORTED;
  }
  const size_t part_bytes = (size_t)slots * prm.max_pieces * nt * kGemmTileCols * sizeof(int32_t);
  if (part_bytes)
    if (int32_t rc = grow(p->dev, p->int8_part, part_bytes)) return rc;
  Int8Maps maps;
  if (!make_tmap_2d(&maps.w, (void*)w, (uint64_t)N, (uint64_t)K / 2, kStepK / 2, kGemmTileCols) ||
      !make_tmap_2d(&maps.a, (void*)a, (uint64_t)M, (uint64_t)K / 2, kStepK / 2, nt)) {
    set_error("tensor map for 8-bit rows could not be encoded");
    return RELUX_ERR_CUDA;
  }
  prm.M = M;
  prm.N = N;
  prm.out_bf16 = out_bf16;
  prm.a_scale = a_scale;
  prm.w_scale = w_scale;
  prm.out = out;
  prm.part = (int32_t*)p->int8_part.p;
  prm.arrived = p->int8_arrived;
  prm.status = p->d_status;
  const int workers = rg.workers * rg.beside;
  switch (nt) {
    case 16: return launch_rows<16>(p, maps, prm, workers);
    case 32: return launch_rows<32>(p, maps, prm, workers);
    case 64: return launch_rows<64>(p, maps, prm, workers);
    case 128: return launch_rows<128>(p, maps, prm, workers);
    default: return launch_rows<256>(p, maps, prm, workers);
  }
}

// |code| <= 128 whatever the bytes are: 2^14 K stays below 2^31
constexpr int kMaxInt8K = 131056;

int32_t do_matmul_int8(Pool* p, const relux_matmul_int8_args* a) {
  if (!a || !a->a || !a->a_scales || !a->w || !a->w_scales || !a->out) { set_error("nil argument"); return RELUX_ERR_INVALID_ARG; }
  if (a->m <= 0 || a->k <= 0 || a->n <= 0) { set_error("matmul_int8: M=%d K=%d N=%d must be positive", a->m, a->k, a->n); return RELUX_ERR_INVALID_ARG; }
  if (a->out_dtype != RELUX_DTYPE_F32 && a->out_dtype != RELUX_DTYPE_BF16) { set_error("bad dtype flag"); return RELUX_ERR_INVALID_ARG; }
  for (int i = 0; i < 4; i++)
    if (a->reserved[i]) { set_error("reserved fields must be zero"); return RELUX_ERR_INVALID_ARG; }
  int32_t rc;
  if ((rc = check_dev_align(a->a, "a")) || (rc = check_dev_align(a->a_scales, "a_scales")) || (rc = check_dev_align(a->w, "w")) ||
      (rc = check_dev_align(a->w_scales, "w_scales")) || (rc = check_dev_align(a->out, "out")))
    return rc;
  if (a->k % 16 != 0 || a->n % 8 != 0 || a->k > kMaxInt8K) {
    set_error("matmul_int8: K=%d must be a multiple of 16, up to %d, and N=%d a multiple of 8", a->k, kMaxInt8K, a->n);
    return RELUX_ERR_UNSUPPORTED;
  }
  return launch_matmul_int8(p, a->m, a->k, a->n, a->a, a->a_scales, a->w, a->w_scales, a->out, a->out_dtype == RELUX_DTYPE_BF16);
}

}  // namespace relux
