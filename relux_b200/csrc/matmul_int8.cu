// Product of 8-bit rows with 8-bit weights on the tensor cores: C[m][n] = sa[m] * sw[n] * sum_k a[m][k] * w[n][k], the sum in 32-bit whole
// numbers, exact for every K that the call takes, whatever the order of its parts.
//
// Bound: HBM up to some hundred rows (a weight is one byte, read once), the tensor cores above.  Both operands lie K-major, as the quantiser and the
// import write them; a step is 128 bytes of K of both.  Two shapes of a tile:
//   * up to 128 rows: 128 weight columns are the M operand of the MMA and the rows, padded to 16 .. 128, its N operand, so that a stage
//     is 16 KB of weights and no more rows than there are;
//   * more: 128 rows are the M operand and 256 columns the N operand, so that a thread of the epilogue holds a row, and results leave by TMA in
//     pieces of 128 bytes.  (With columns as the M operand a thread held a column, and stored two bytes at a time: 644 us for 8192 x 4096 x 16384
//     where the loads and MMAs alone take 320.)
// Tiles that would leave SMs idle are cut along K among the CTAs of a cluster, which hand each other slices of their sums through distributed shared
// memory; every CTA finishes one slice.  Whole numbers add up to the same in any order, so a result does not depend on the cut.  (The pieces
// through L2, joined by the last of them, took 35 us more at 300 x 8192 x 4096.)
// The weights of a CTA's first steps are brought into L2, not into shared memory, while the launch before this one ends: a prefetch returns no data,
// so it may be early whatever that launch writes.
#include <algorithm>

#include "common.cuh"
#include "internal.h"
#include "umma.cuh"

namespace relux {

namespace {

constexpr int kStepK = 128;                 // bytes of K of a step
constexpr int kRowsOp = 128;                // rows of the M operand
constexpr int kStageRows = kRowsOp * kStepK;
constexpr int kPrefetchBytes = 256 << 10;   // of weights, by CTA
constexpr int kGroup = 16;                  // row blocks that share the columns they are multiplied with, wide tiles
constexpr int kOutRow = 128;                // bytes of a row of the staging tiles of the epilogue

// NC: rows of the N operand.  Wide tiles have 256.
template <int NC>
struct Int8Shape {
  static constexpr bool kWide = NC == 256;
  static constexpr int kMaxCluster = kWide ? 4 : 8;
  static constexpr int kStage = kStageRows + NC * kStepK;
  static constexpr int kBars = 1024;
  static constexpr int kScales = kWide ? 2 * NC * 4 : 0;                        // the columns' scales, by accumulator
  static constexpr int kOut = kWide ? 4 * 2 * 32 * kOutRow : 0;                 // two staging tiles of 32 rows a warp
  static constexpr int kSlices = kWide ? 0 : (NC < 32 ? 32 : NC) * kRowsOp * 4;  // the slices from the cluster (wide: in the stages, which are free then)
  static constexpr int kStages = (232448 - kBars - kScales - kOut - kSlices) / kStage < 12 ? (232448 - kBars - kScales - kOut - kSlices) / kStage : 12;
  static constexpr int kSmem = kStages * kStage + kOut + kSlices + kScales + kBars;
  static constexpr int kAcc = NC < 32 ? 32 : NC;
};
// The slices that a CTA receives, one from each of the others, fit: columns of a slice are counted by the kernel's rule.
constexpr bool slices_fit(int cols, int grain, int most, int room) {
  for (int size = 2; size <= most; size++)
    for (int i = 0, units = (cols + grain - 1) / grain; i < size; i++)
      if ((size - 1) * (((i + 1) * units / size - i * units / size) * grain) * kRowsOp * 4 > room) return false;
  return true;
}
constexpr bool slices_fit_up_to(int cols, int grain, int most, int room) {
  for (int c = 1; c <= cols; c++)
    if (!slices_fit(c, grain, most, room)) return false;
  return true;
}
static_assert(slices_fit_up_to(16, 1, 8, Int8Shape<16>::kSlices) && slices_fit_up_to(32, 1, 8, Int8Shape<32>::kSlices) &&
              slices_fit_up_to(64, 1, 8, Int8Shape<64>::kSlices) && slices_fit_up_to(128, 1, 8, Int8Shape<128>::kSlices) &&
              slices_fit_up_to(256, 32, 4, Int8Shape<256>::kStages * Int8Shape<256>::kStage) &&
              slices_fit_up_to(256, 64, 4, Int8Shape<256>::kStages * Int8Shape<256>::kStage), "no room for the slices");
struct Int8Bars {
  uint64_t full[12], empty[12], acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  volatile int32_t abort_flag;
};
static_assert(sizeof(Int8Bars) <= 1024, "barrier block too small");

struct Int8Maps {
  CUtensorMap r, c;   // M and N operand: rows of K bytes, seen as rows of K / 2 elements of two bytes
  CUtensorMap out;    // wide tiles: rows of two-byte elements, two for a float32
};
struct Int8Params {
  int32_t M, N, steps, tiles, row_blocks, col_tiles, out_bf16;
  const float* a_scale;
  const float* w_scale;
  void* out;
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
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void store_cluster(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ float int8_scaled(uint32_t sum, float sa, float sw) { return __fmul_rn(__fmul_rn((float)(int32_t)sum, sa), sw); }

// A tile's place.  Wide tiles: kGroup row blocks walk the columns together, so that what the SMs read at a time is few rows and few columns.
template <bool kWide>
__device__ __forceinline__ void tile_place(const Int8Params& p, int tile, int& r, int& c) {
  if constexpr (!kWide) {
    r = tile;
    c = 0;
  } else {
    const int per = kGroup * p.col_tiles, group = tile / per, rest = tile - group * per, rows = min(kGroup, p.row_blocks - group * kGroup);
    c = rest / rows;
    r = group * kGroup + rest - c * rows;
  }
}

// grid (clusters x size), 192 threads: warps 0-3 epilogue, warp 4 TMA producer, warp 5 MMA issuer.  The CTAs of a cluster have the same tiles and a part
// of K each; a cluster of more than one CTA has one tile.
template <int NC>
__global__ void __launch_bounds__(192, 1) matmul_int8_kernel(const __grid_constant__ Int8Maps maps, const __grid_constant__ Int8Params prm) {
  using SH = Int8Shape<NC>;
  constexpr int kStages = SH::kStages;
  constexpr bool kWide = SH::kWide;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* const out_tiles = smem + kStages * SH::kStage;
  uint8_t* const slices = kWide ? smem : out_tiles + SH::kOut;
  float* const scales = reinterpret_cast<float*>(out_tiles + SH::kOut + SH::kSlices);
  Int8Bars* bars = reinterpret_cast<Int8Bars*>(out_tiles + SH::kOut + SH::kSlices + SH::kScales);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int size = (int)cluster_size(), rank = (int)cluster_ctarank();
  const int first = blockIdx.x / size, stride = gridDim.x / size;
  const int k0 = rank * prm.steps / size, k1 = (rank + 1) * prm.steps / size;
  chain_release();
  if ((smem_u32(smem) & 1023u) != 0) {   // (the same in every CTA)
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
  if (size > 1) cluster_arrive();   // this CTA has begun: its shared memory may be written from the others
  const uint32_t tmem = bars->tmem_base;

  if (warp == 4) {
    const bool el = elect_one();
    if (el) {
      tma_prefetch_desc(&maps.r);
      tma_prefetch_desc(&maps.c);
      constexpr int kWeightBytes = kWide ? NC * kStepK : kStageRows;
      int left = kPrefetchBytes / kWeightBytes;
      for (int tile = first; tile < prm.tiles && left > 0; tile += stride) {
        int r, c;
        tile_place<kWide>(prm, tile, r, c);
        for (int k = k0; k < k1 && left > 0; k++, left--) {
          if constexpr (kWide) tma_prefetch_2d(&maps.c, k * (kStepK / 2), c * NC);
          else tma_prefetch_2d(&maps.r, k * (kStepK / 2), r * kRowsOp);
        }
      }
    }
    __syncwarp();
    chain_wait();
    int g = 0;
    for (int tile = first; tile < prm.tiles; tile += stride) {
      int r, c;
      tile_place<kWide>(prm, tile, r, c);
      for (int k = k0; k < k1; k++, g++) {
        const int s = g % kStages;
        if (g >= kStages) int8_wait(&bars->empty[s], (g / kStages - 1) & 1, bars, prm.status);
        if (el) {
          uint8_t* st = smem + s * SH::kStage;
          mbar_expect_tx(&bars->full[s], SH::kStage);   // out-of-range parts of a box are zero-filled and still counted
          tma_load_2d(st, &maps.r, k * (kStepK / 2), r * kRowsOp, &bars->full[s]);
          tma_load_2d(st + kStageRows, &maps.c, k * (kStepK / 2), c * NC, &bars->full[s]);
        }
        __syncwarp();
      }
    }
  } else if (warp == 5) {
    const bool el = elect_one();
    const uint32_t idesc = make_idesc_s8(kRowsOp, NC);
    int g = 0, piece = 0;
    for (int tile = first; tile < prm.tiles; tile += stride, piece++) {
      const uint32_t d = tmem + (piece & 1) * SH::kAcc;
      if (piece >= 2) int8_wait(&bars->acc_empty[piece & 1], ((piece >> 1) - 1) & 1, bars, prm.status);
      tc_fence_after();
      for (int k = k0; k < k1; k++, g++) {
        const int s = g % kStages;
        int8_wait(&bars->full[s], (g / kStages) & 1, bars, prm.status);
        tc_fence_after();
        if (el) {
          const uint32_t st = smem_u32(smem + s * SH::kStage);
          const uint64_t dR = make_desc_kmajor_sw128(st), dC = make_desc_kmajor_sw128(st + kStageRows);
#pragma unroll
          for (int kk = 0; kk < kStepK / 32; kk++)
            umma_ss_i8(d, dR + ((uint32_t)(kk * 32) >> 4), dC + ((uint32_t)(kk * 32) >> 4), idesc, k != k0 || kk != 0);
          umma_commit<1>(&bars->empty[s]);
        }
        __syncwarp();
      }
      if (el) umma_commit<1>(&bars->acc_full[piece & 1]);
      __syncwarp();
    }
  } else {
    chain_wait();
    int piece = 0, staged = 0;
    for (int tile = first; tile < prm.tiles; tile += stride, piece++) {
      int r, c;
      tile_place<kWide>(prm, tile, r, c);
      const int buf = piece & 1, at_row = r * kRowsOp + warp * 32 + lane;   // this thread's column (wide: row)
      const uint32_t acc = tmem + ((uint32_t)(warp * 32) << 16) + buf * SH::kAcc;
      const int cols = kWide ? min(NC, prm.N - c * NC) : prm.M;             // of the N operand that exist
      const bool mine = at_row < (kWide ? prm.M : prm.N);
      float sa_of[kWide ? 1 : (NC + 31) / 32];   // this lane's rows' scales: lane, lane + 32, ...
      if constexpr (!kWide)
#pragma unroll
        for (int i = 0; i < (NC + 31) / 32; i++) sa_of[i] = i * 32 + lane < prm.M ? load_chained(prm.a_scale + i * 32 + lane) : 0.f;
      const float own = mine ? load_chained((kWide ? prm.a_scale : prm.w_scale) + at_row) : 0.f;
      if constexpr (kWide) {   // (a warp that is here has passed the barrier of the tile before, and with it every warp the end of the one before that)
#pragma unroll
        for (int i = 0; i < NC / 128; i++) {
          const int q = threadIdx.x + i * 128;
          scales[buf * NC + q] = q < cols ? load_chained(prm.w_scale + c * NC + q) : 0.f;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }
      int8_wait(&bars->acc_full[buf], (piece >> 1) & 1, bars, prm.status);
      tc_fence_after();
      const bool ok = !bars->abort_flag;
      // the columns that this CTA finishes
      int q0 = 0, q1 = cols;
      if (size > 1) {
        const int grain = !kWide ? 1 : prm.out_bf16 ? 64 : 32, units = (cols + grain - 1) / grain;
        auto begin = [&](int i) { return min(cols, i * units / size * grain); };
        q0 = begin(rank);
        q1 = begin(rank + 1);
        // slices to the others: [from][column of the slice][128 rows]
        cluster_wait();
        if constexpr (kWide) {   // the others' stages: they are free once their MMAs are done
          cluster_arrive();
          cluster_wait();
        }
        const uint32_t here = smem_u32(slices) + (uint32_t)(warp * 32 + lane) * 4;
#pragma unroll 1
        for (int to = 0; to < size; to++) {
          if (to == rank) continue;
          const int b = begin(to), e = begin(to + 1);
          const uint32_t there = mapa_u32(here, (uint32_t)to) + (uint32_t)((rank < to ? rank : rank - 1) * (e - b)) * (kRowsOp * 4);
#pragma unroll 1
          for (int q = b; q < e; q += 8) {
            uint32_t v[8];
            tmem_ld_32x32b_x8(acc + q, v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; i++)
              if (q + i < e) store_cluster(there + (uint32_t)(q - b + i) * (kRowsOp * 4), v[i]);
          }
        }
        cluster_arrive();
        cluster_wait();
      }
      const int32_t* const got = reinterpret_cast<const int32_t*>(slices) + warp * 32 + lane;
      if constexpr (!kWide) {
        // thread = column; a warp writes 64 or 128 bytes of a row at once
#pragma unroll 1
        for (int q = q0; q < q1; q += 8) {
          uint32_t v[8];
          tmem_ld_32x32b_x8(acc + q, v);
          tmem_ld_wait();
#pragma unroll 1
          for (int s = 0; s < size - 1; s++)
#pragma unroll
            for (int i = 0; i < 8; i++)
              if (q + i < q1) v[i] += (uint32_t)got[(s * (q1 - q0) + q - q0 + i) * kRowsOp];
          // (all eight before the first store: one by one each waited for the one before, 180 clocks a row)
          float x[8];
#pragma unroll
          for (int i = 0; i < 8; i++) {
            float sa = sa_of[0];
#pragma unroll
            for (int j = 1; j < (NC + 31) / 32; j++)
              if ((q + i) / 32 == j) sa = sa_of[j];
            x[i] = int8_scaled(ok ? v[i] : 0u, __shfl_sync(0xffffffffu, sa, (q + i) & 31), own);
          }
          const size_t at = (size_t)q * prm.N + at_row;
          if (prm.out_bf16) {
            uint16_t* const to = reinterpret_cast<uint16_t*>(prm.out) + at;
#pragma unroll
            for (int i = 0; i < 8; i++) store_if(to + (size_t)i * prm.N, __bfloat16_as_ushort(__float2bfloat16_rn(x[i])), mine && q + i < q1);
          } else {
            float* const to = reinterpret_cast<float*>(prm.out) + at;
#pragma unroll
            for (int i = 0; i < 8; i++) store_if(to + (size_t)i * prm.N, x[i], mine && q + i < q1);
          }
        }
      } else {
        // thread = row: 32 (bf16: 64) columns at a time to a staging tile of the warp, 128-byte swizzle, and out by TMA, which leaves out what
        // lies past the last row or column
        uint8_t* const tiles = out_tiles + warp * 2 * 32 * kOutRow;
        const int wide = prm.out_bf16 ? 64 : 32;
#pragma unroll 1
        for (int q = q0; q < q1; q += wide, staged++) {
          uint8_t* const tile_smem = tiles + (staged & 1) * 32 * kOutRow;
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");   // the store before the last has read its tile
          __syncwarp();
#pragma unroll 1
          for (int h = 0; h < wide && q + h < q1; h += 32) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(acc + q + h, v);
            tmem_ld_wait();
#pragma unroll 1
            for (int s = 0; s < size - 1; s++)
#pragma unroll
              for (int i = 0; i < 32; i++)
                if (q + h + i < q1) v[i] += (uint32_t)got[(s * (q1 - q0) + q + h - q0 + i) * kRowsOp];
            const float4* sw = reinterpret_cast<const float4*>(scales + buf * NC + q + h);
            float x[32];
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const float4 s4 = sw[i];
              x[4 * i] = int8_scaled(ok ? v[4 * i] : 0u, own, s4.x);
              x[4 * i + 1] = int8_scaled(ok ? v[4 * i + 1] : 0u, own, s4.y);
              x[4 * i + 2] = int8_scaled(ok ? v[4 * i + 2] : 0u, own, s4.z);
              x[4 * i + 3] = int8_scaled(ok ? v[4 * i + 3] : 0u, own, s4.w);
            }
            if (prm.out_bf16) {
#pragma unroll
              for (int i = 0; i < 4; i++)
                *reinterpret_cast<uint4*>(tile_smem + swz128(lane, h / 8 + i)) =
                    make_uint4(round_bf16x2(x[8 * i], x[8 * i + 1]), round_bf16x2(x[8 * i + 2], x[8 * i + 3]), round_bf16x2(x[8 * i + 4], x[8 * i + 5]),
                               round_bf16x2(x[8 * i + 6], x[8 * i + 7]));
            } else {
#pragma unroll
              for (int i = 0; i < 8; i++) *reinterpret_cast<float4*>(tile_smem + swz128(lane, i)) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
            }
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&maps.out, (c * NC + q) * (prm.out_bf16 ? 1 : 2), r * kRowsOp + warp * 32, tile_smem);
            tma_store_commit();
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->acc_empty[buf]);
    }
    if constexpr (kWide) {
      if (lane == 0) tma_store_wait_all();
      __syncwarp();
    } else {
      fence_chained_writes();
    }
  }
  if (size > 1 && warp >= 4) {   // the epilogue's barriers count every thread
    cluster_wait();
    if constexpr (kWide) {
      cluster_arrive();
      cluster_wait();
    }
    cluster_arrive();
    cluster_wait();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc<1>(tmem, 2 * SH::kAcc);
}

template <int NC>
int32_t launch_shape(Pool* p, const Int8Maps& maps, const Int8Params& prm) {
  using SH = Int8Shape<NC>;
  if (int32_t rc = allow_smem(p->dev, matmul_int8_kernel<NC>, SH::kSmem)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(192);
  cfg.dynamicSmemBytes = SH::kSmem;
  cfg.stream = p->dev->stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  // As many CTAs to a tile as leave every tile a cluster that is resident at once.  A cluster lies within one of the GPU's groups of SMs, so there are
  // fewer of them than SMs / size: 74 of two, 45 of three, 33 of four.
  int size = 1;
  for (int s = 2; s <= SH::kMaxCluster && 2 * s <= prm.steps && prm.tiles * s <= p->dev->sm_count; s++) {
    int& most = p->dev->int8_clusters[s];
    if (!most) {
      at[0].val.clusterDim.x = (unsigned)s;
      cfg.gridDim = dim3((unsigned)(s * p->dev->sm_count));
      RELUX_CUDA_TRY(cudaOccupancyMaxActiveClusters(&most, matmul_int8_kernel<NC>, &cfg));
    }
    if (prm.tiles <= most) size = s;
  }
  cfg.gridDim = dim3((unsigned)(size > 1 ? prm.tiles * size : std::min(prm.tiles, p->dev->sm_count)));
  at[0].val.clusterDim.x = (unsigned)size;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = p->tune.get(RELUX_TUNE_CHAINED_LAUNCHES) != 0 ? 2 : 1;
  RELUX_CUDA_TRY(cudaLaunchKernelEx(&cfg, matmul_int8_kernel<NC>, maps, prm));
  count_launch(p->dev);
  return RELUX_OK;
}

}  // namespace

int32_t launch_matmul_int8(Pool* p, int M, int K, int N, const int8_t* a, const float* a_scale, const int8_t* w, const float* w_scale, void* out,
                           bool out_bf16) {
  Int8Params prm{};
  Int8Maps maps{};
  const bool wide = M > 128;
  int nc = 16;
  while (!wide && nc < M) nc *= 2;
  if (wide) nc = 256;
  prm.M = M;
  prm.N = N;
  prm.steps = (K + kStepK - 1) / kStepK;
  prm.row_blocks = (M + kRowsOp - 1) / kRowsOp;
  prm.col_tiles = (N + (wide ? nc : kRowsOp) - 1) / (wide ? nc : kRowsOp);
  const int64_t tiles = wide ? (int64_t)prm.row_blocks * prm.col_tiles : prm.col_tiles;
  if (tiles * prm.steps >= (int64_t)1 << 31) { set_error("a product of more than 2^31 steps"); return RELUX_ERR_UNSUPPORTED; }
  prm.tiles = (int)tiles;
  prm.out_bf16 = out_bf16;
  prm.a_scale = a_scale;
  prm.w_scale = w_scale;
  prm.out = out;
  prm.status = p->d_status;
  const int8_t* rows = wide ? a : w;
  const int8_t* cols = wide ? w : a;
  bool made = make_tmap_2d(&maps.r, (void*)rows, (uint64_t)(wide ? M : N), (uint64_t)K / 2, kStepK / 2, kRowsOp) &&
              make_tmap_2d(&maps.c, (void*)cols, (uint64_t)(wide ? N : M), (uint64_t)K / 2, kStepK / 2, nc);
  if (wide) made = made && make_tmap_2d(&maps.out, out, (uint64_t)M, (uint64_t)N * (out_bf16 ? 1 : 2), kOutRow / 2, 32);
  if (!made) {
    set_error("tensor map for 8-bit rows could not be encoded");
    return RELUX_ERR_CUDA;
  }
  switch (nc) {
    case 16: return launch_shape<16>(p, maps, prm);
    case 32: return launch_shape<32>(p, maps, prm);
    case 64: return launch_shape<64>(p, maps, prm);
    case 128: return launch_shape<128>(p, maps, prm);
    default: return launch_shape<256>(p, maps, prm);
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
