// What the products of matmul_int8.cu and lora_gemm.cu share: tiles, stages, the hand-over of a cluster's parts.
//
// A step is 128 bytes of K of both operands.  Two shapes of a tile:
//   * up to 128 rows: 128 weight columns are the M operand of the MMA and the rows, padded to 16 .. 128, its N operand, so that a stage
//     is 16 KB of weights and no more rows than there are;
//   * more ("wide"): 128 rows are the M operand and 256 columns the N operand, so that a thread of the epilogue holds a row, and results leave by
//     TMA in pieces of 128 bytes.
// One CTA per SM walks its tiles without draining its pipeline in between (two accumulators).  Tiles that would leave SMs idle are cut along K among
// the CTAs of a cluster, one tile a cluster: each CTA hands the others their slices of its sums through distributed shared memory, and finishes
// one slice.
#pragma once

#include <algorithm>

#include "common.cuh"
#include "internal.h"
#include "umma.cuh"

namespace relux {

constexpr int kStepBytes = 128;             // of K, of a step
constexpr int kRowsOp = 128;                // rows of the M operand
constexpr int kStageRows = kRowsOp * kStepBytes;
constexpr int kGroup = 16;                  // row blocks that share the columns they are multiplied with, wide tiles
constexpr int kOutRow = 128;                // bytes of a row of the epilogue's staging tiles

// NC: rows of the N operand; wide tiles have 256.  kMore: bytes that the epilogue needs beside.  kSliceRows: columns of slices that there is room for.
// kHalves: N operands of a step, where rows are two halves.  kMost: stages.
template <int NC, int kMoreBytes, int kSliceRows = NC < 32 ? 32 : NC, int kHalves = 1, int kMost = 12>
struct TileShape {
  static constexpr bool kWide = NC == 256;
  static constexpr int kMaxCluster = kWide ? 4 : 8;
  static constexpr int kStage = kStageRows + kHalves * NC * kStepBytes;
  static constexpr int kBars = 1024;
  static constexpr int kMore = kMoreBytes;
  static constexpr int kOut = kWide ? 4 * 2 * 32 * kOutRow : 0;                              // two staging tiles of 32 rows a warp
  static constexpr int kSlices = kWide ? 0 : kSliceRows * kRowsOp * 4;                      // the slices from the cluster (wide: in the stages, which are free then)
  static constexpr int kRoom = 232448 - kBars - kMore - kOut - kSlices;
  static constexpr int kStages = kRoom / kStage < kMost ? kRoom / kStage : kMost;
  static constexpr int kSmem = kStages * kStage + kOut + kSlices + kMore + kBars;
  static constexpr int kAcc = NC < 32 ? 32 : NC;
};
// Columns of the N operand that CTA i of a cluster finishes: [slice_begin(i), slice_begin(i + 1)), in units of `grain`.
__host__ __device__ constexpr int slice_begin(int i, int cols, int grain, int size) {
  const int b = i * ((cols + grain - 1) / grain) / size * grain;
  return b < cols ? b : cols;
}
// Whether the slices that a CTA receives fit in `room` bytes, `more` further ones of its own among them.
constexpr bool slices_fit(int cols, int grain, int most, int more, int room) {
  for (int c = 1; c <= cols; c++)
    for (int size = 2; size <= most; size++)
      for (int i = 0; i < size; i++)
        if ((size - 1 + more) * (slice_begin(i + 1, c, grain, size) - slice_begin(i, c, grain, size)) * kRowsOp * 4 > room) return false;
  return true;
}

struct TileBars {
  uint64_t full[12], empty[12], acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  volatile int32_t abort_flag;
};
static_assert(sizeof(TileBars) <= 1024, "barrier block too small");

__device__ __noinline__ inline void tile_wait_slow(uint64_t* bar, uint32_t parity, TileBars* b, int32_t* status) {
  for (uint32_t i = 0; i < kSpinLimit; i++) {
    if (mbar_try_wait(bar, parity)) return;
    if ((i & 255) == 255 && b->abort_flag) return;
    if (i > 512) __nanosleep(20);
  }
  b->abort_flag = 1;
  set_status(status, RELUX_ERR_TIMEOUT);
}
// Bounded: a wait that runs out records RELUX_ERR_TIMEOUT and raises the CTA's abort flag; nobody leaves a loop early.
__device__ __forceinline__ void tile_wait(uint64_t* bar, uint32_t parity, TileBars* b, int32_t* status) {
  if (!mbar_try_wait(bar, parity)) tile_wait_slow(bar, parity, b, status);
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
__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// Barriers and tensor memory of a CTA (warp 0 allocates); returns the base of tensor memory.  fills: arrivals that fill a stage, TMA's among them.
template <class SH>
__device__ __forceinline__ uint32_t tile_setup(TileBars* bars, int size, int fills = 1) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < SH::kStages; s++) { mbar_init(&bars->full[s], fills); mbar_init(&bars->empty[s], 1); }
    for (int b = 0; b < 2; b++) { mbar_init(&bars->acc_full[b], 1); mbar_init(&bars->acc_empty[b], 4); }
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (threadIdx.x < 32) {
    tmem_alloc<1>(&bars->tmem_base, 2 * SH::kAcc);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (size > 1) cluster_arrive();   // this CTA has begun: its shared memory may be written from the others
  return bars->tmem_base;
}
// The epilogue's warps, a tile that is cut along K: slices to the others, [from][column of the slice][128 rows], and back when all have arrived.
// (A warp's store is 128 neighbouring bytes; 16 bytes a thread to rows that lie apart took 3 us longer for 200 x 4096 x 4096.)
// part i of K is CTA i of the cluster, or (kPer 2) the CTA of this one's side in pair i.
// also(): sends more with them, by all of these warps.
struct NothingMore {
  __device__ __forceinline__ void operator()() const {}
};
template <class SH, int kPer = 1, class Also = NothingMore>
__device__ __forceinline__ void swap_slices(uint32_t acc, int cols, int grain, int size, int rank, const uint8_t* slices, Also also = Also()) {
  cluster_wait();
  also();
  if constexpr (SH::kWide) {   // the others' stages: they are free once their MMAs are done
    cluster_arrive();
    cluster_wait();
  }
  const uint32_t side = kPer == 2 ? cluster_ctarank() & 1u : 0u;
  constexpr int kAtOnce = SH::kWide ? 16 : 8;
#pragma unroll 1
  for (int to = 0; to < size; to++) {
    if (to == rank) continue;
    const int b = slice_begin(to, cols, grain, size), e = slice_begin(to + 1, cols, grain, size);
    const uint32_t there = mapa_u32(smem_u32(slices) + threadIdx.x * 4, (uint32_t)to * kPer + side) + (uint32_t)((rank < to ? rank : rank - 1) * (e - b)) * (kRowsOp * 4);
#pragma unroll 1
    for (int q = b; q < e; q += kAtOnce) {
      uint32_t v[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; i += 8) tmem_ld_32x32b_x8(acc + q + i, *reinterpret_cast<uint32_t(*)[8]>(v + i));
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < kAtOnce; i++)
        if (q + i < e) store_cluster(there + (uint32_t)(q - b + i) * (kRowsOp * 4), v[i]);
    }
  }
  cluster_arrive();
  cluster_wait();
}
// The other warps' part in it, and the end of a CTA.
template <class SH>
__device__ __forceinline__ void tile_end(uint32_t tmem, int size) {
  if (size > 1 && threadIdx.x >= 128) {   // the barriers count every thread
    cluster_wait();
    if constexpr (SH::kWide) {
      cluster_arrive();
      cluster_wait();
    }
    cluster_arrive();
    cluster_wait();
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x < 32) tmem_dealloc<1>(tmem, 2 * SH::kAcc);
}

// Wide tiles: what the others have sent of columns c .. c + 15 of this CTA's slice of n columns, for this thread's row: add(i, v) for column c + i.
template <class Add>
__device__ __forceinline__ void add_slices(const uint8_t* slices, int size, int n, int c, Add add) {
#pragma unroll 1
  for (int s = 0; s < size - 1; s++) {
    const uint32_t* const got = reinterpret_cast<const uint32_t*>(slices) + (s * n + c) * kRowsOp + threadIdx.x;
#pragma unroll
    for (int i = 0; i < 16; i++)
      if (c + i < n) add(i, got[i * kRowsOp]);
  }
}

// Wide tiles: kGroup row blocks walk the columns together, so that what the SMs read at a time is few rows and few columns.
__device__ __forceinline__ void wide_place(int tile, int row_blocks, int col_tiles, int& r, int& c) {
  const int per = kGroup * col_tiles, group = tile / per, rest = tile - group * per, rows = min(kGroup, row_blocks - group * kGroup);
  c = rest / rows;
  r = group * kGroup + rest - c * rows;
}

// Launches `kernel` over `tiles` tiles of kPer CTAs each, in as many parts of K as leave every tile a cluster that is resident at once: a cluster lies within
// one of the GPU's groups of SMs, so there are fewer of them than SMs / size (74 of two, 45 of three, 33 of four CTAs).
template <class SH, int kThreads = 192, int kPer = 1, typename... KArgs, typename... Args>
int32_t launch_tiles(Pool* p, void (*kernel)(KArgs...), int tiles, int steps, const Args&... args) {
  if (int32_t rc = allow_smem(p->dev, kernel, SH::kSmem)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = SH::kSmem;
  cfg.stream = p->dev->stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  auto resident = [&](int size, int* most) -> int32_t {
    int& known = p->dev->tile_clusters[size];
    if (!known) {
      at[0].val.clusterDim.x = (unsigned)size;
      cfg.gridDim = dim3((unsigned)(size * p->dev->sm_count));
      RELUX_CUDA_TRY(cudaOccupancyMaxActiveClusters(&known, kernel, &cfg));
    }
    *most = known;
    return RELUX_OK;
  };
  int parts = 1, most = p->dev->sm_count;
  for (int s = 2; s <= SH::kMaxCluster && 2 * s <= steps && tiles <= p->dev->sm_count / (s * kPer); s++) {
    if (int32_t rc = resident(s * kPer, &most)) return rc;
    if (tiles <= most) parts = s;
  }
  if (parts == 1 && kPer > 1)
    if (int32_t rc = resident(kPer, &most)) return rc;
  cfg.gridDim = dim3((unsigned)((parts > 1 ? tiles * parts : std::min(tiles, kPer > 1 ? most : p->dev->sm_count)) * kPer));
  at[0].val.clusterDim.x = (unsigned)(parts * kPer);
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = p->tune.get(RELUX_TUNE_CHAINED_LAUNCHES) != 0 ? 2 : 1;
  RELUX_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
  count_launch(p->dev);
  return RELUX_OK;
}

}  // namespace relux
