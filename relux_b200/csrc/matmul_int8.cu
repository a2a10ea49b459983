// Product of 8-bit rows with 8-bit weights on the tensor cores: C[m][n] = sa[m] * sw[n] * sum_k a[m][k] * w[n][k], the sum in 32-bit whole
// numbers, exact for every K that the call takes, whatever the order of its parts.
//
// Bound: HBM up to some hundred rows (a weight is one byte, read once), the tensor cores above.  Both operands lie K-major, as the quantiser and the
// import write them.  Tiles as in tile_gemm.cuh, wide ones by pairs of CTAs, 256 rows x 256 columns.  Whole numbers add up to the same in any order, so a result does not depend on the cut along K.
// The weights of a CTA's first steps are brought into L2, not into shared memory, while the launch before this one ends: a prefetch returns no data,
// so it may be early whatever that launch writes.
// What did not do: columns as the M operand throughout, whose epilogue stored two bytes a thread (644 us for 8192 x 4096 x 16384, the loads and MMAs
// alone 320); parts of tiles joined through L2 by the last of them (35 us more at 300 x 8192 x 4096).
#include "tile_gemm.cuh"

namespace relux {

namespace {

constexpr int kPrefetchBytes = 256 << 10;   // of weights, by CTA

template <int NC>
using Int8Shape = TileShape<NC, 0>;
static_assert(slices_fit(16, 1, 8, 0, Int8Shape<16>::kSlices) && slices_fit(32, 1, 8, 0, Int8Shape<32>::kSlices) && slices_fit(64, 1, 8, 0, Int8Shape<64>::kSlices) &&
              slices_fit(128, 1, 8, 0, Int8Shape<128>::kSlices), "no room for the slices");
// Pairs of CTAs: a tile of 256 rows x 256 columns, each CTA with 128 of both in its stages and its rows' sums.
struct PairShape {
  static constexpr bool kWide = true;
  static constexpr int kMaxCluster = 4;   // parts of K
  static constexpr int kTile = 256, kStage = 2 * kStageRows, kStages = 6, kAcc = kTile;
  static constexpr int kOut = 4 * 2 * 32 * kOutRow, kScales = 2 * kTile * 4, kBars = 1024;
  static constexpr int kSmem = kStages * kStage + kOut + kScales + kBars;
};
static_assert(PairShape::kSmem <= 232448 && slices_fit(256, 32, 4, 0, PairShape::kStages * PairShape::kStage) &&
              slices_fit(256, 64, 4, 0, PairShape::kStages * PairShape::kStage), "no room for the slices");

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

__device__ __forceinline__ float int8_scaled(uint32_t sum, float sa, float sw) { return __fmul_rn(__fmul_rn((float)(int32_t)sum, sa), sw); }

// Up to 128 rows.  grid (tiles x parts of K), 192 threads: warps 0-3 epilogue, warp 4 TMA producer, warp 5 MMA issuer.
template <int NC>
__global__ void __launch_bounds__(192, 1) matmul_int8_kernel(const __grid_constant__ Int8Maps maps, const __grid_constant__ Int8Params prm) {
  using SH = Int8Shape<NC>;
  constexpr int kStages = SH::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* const slices = smem + kStages * SH::kStage;
  TileBars* bars = reinterpret_cast<TileBars*>(slices + SH::kSlices);
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
  const uint32_t tmem = tile_setup<SH>(bars, size);

  if (warp == 4) {
    const bool el = elect_one();
    if (el) {
      tma_prefetch_desc(&maps.r);
      tma_prefetch_desc(&maps.c);
      int left = kPrefetchBytes / kStageRows;
      for (int tile = first; tile < prm.tiles && left > 0; tile += stride)
        for (int k = k0; k < k1 && left > 0; k++, left--) tma_prefetch_2d(&maps.r, k * (kStepBytes / 2), tile * kRowsOp);
    }
    __syncwarp();
    chain_wait();
    int g = 0;
    for (int tile = first; tile < prm.tiles; tile += stride)
      for (int k = k0; k < k1; k++, g++) {
        const int s = g % kStages;
        if (g >= kStages) tile_wait(&bars->empty[s], (g / kStages - 1) & 1, bars, prm.status);
        if (el) {
          uint8_t* st = smem + s * SH::kStage;
          mbar_expect_tx(&bars->full[s], SH::kStage);   // out-of-range parts of a box are zero-filled and still counted
          tma_load_2d(st, &maps.r, k * (kStepBytes / 2), tile * kRowsOp, &bars->full[s]);
          tma_load_2d(st + kStageRows, &maps.c, k * (kStepBytes / 2), 0, &bars->full[s]);
        }
        __syncwarp();
      }
  } else if (warp == 5) {
    const bool el = elect_one();
    const uint32_t idesc = make_idesc_s8(kRowsOp, NC);
    int g = 0, piece = 0;
    for (int tile = first; tile < prm.tiles; tile += stride, piece++) {
      const uint32_t d = tmem + (piece & 1) * SH::kAcc;
      if (piece >= 2) tile_wait(&bars->acc_empty[piece & 1], ((piece >> 1) - 1) & 1, bars, prm.status);
      tc_fence_after();
      for (int k = k0; k < k1; k++, g++) {
        const int s = g % kStages;
        tile_wait(&bars->full[s], (g / kStages) & 1, bars, prm.status);
        tc_fence_after();
        if (el) {
          const uint32_t st = smem_u32(smem + s * SH::kStage);
          const uint64_t dR = make_desc_kmajor_sw128(st), dC = make_desc_kmajor_sw128(st + kStageRows);
#pragma unroll
          for (int kk = 0; kk < kStepBytes / 32; kk++)
            umma_ss_i8<1>(d, dR + ((uint32_t)(kk * 32) >> 4), dC + ((uint32_t)(kk * 32) >> 4), idesc, k != k0 || kk != 0);
          umma_commit<1>(&bars->empty[s]);
        }
        __syncwarp();
      }
      if (el) umma_commit<1>(&bars->acc_full[piece & 1]);
      __syncwarp();
    }
  } else {
    chain_wait();
    int piece = 0;
    for (int tile = first; tile < prm.tiles; tile += stride, piece++) {
      const int buf = piece & 1, n = tile * kRowsOp + warp * 32 + lane;   // this thread's column
      const uint32_t acc = tmem + ((uint32_t)(warp * 32) << 16) + buf * SH::kAcc;
      const bool mine = n < prm.N;
      float sa_of[(NC + 31) / 32];   // this lane's rows' scales: lane, lane + 32, ...
#pragma unroll
      for (int i = 0; i < (NC + 31) / 32; i++) sa_of[i] = i * 32 + lane < prm.M ? load_chained(prm.a_scale + i * 32 + lane) : 0.f;
      const float sw = mine ? load_chained(prm.w_scale + n) : 0.f;
      tile_wait(&bars->acc_full[buf], (piece >> 1) & 1, bars, prm.status);
      tc_fence_after();
      const bool ok = !bars->abort_flag;
      // the rows that this CTA finishes
      int q0 = 0, q1 = prm.M;
      if (size > 1) {
        q0 = slice_begin(rank, prm.M, 1, size);
        q1 = slice_begin(rank + 1, prm.M, 1, size);
        swap_slices<SH>(acc, prm.M, 1, size, rank, slices);
      }
      const int32_t* const got = reinterpret_cast<const int32_t*>(slices) + warp * 32 + lane;
      constexpr int kAtOnce = NC <= 32 ? 8 : 16;   // a warp writes 64 or 128 bytes of a row at once
#pragma unroll 1
      for (int q = q0; q < q1; q += kAtOnce) {
        uint32_t v[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; i += 8) tmem_ld_32x32b_x8(acc + q + i, *reinterpret_cast<uint32_t(*)[8]>(v + i));
        tmem_ld_wait();
#pragma unroll 1
        for (int s = 0; s < size - 1; s++)
#pragma unroll
          for (int i = 0; i < kAtOnce; i++)
            if (q + i < q1) v[i] += (uint32_t)got[(s * (q1 - q0) + q - q0 + i) * kRowsOp];
        // (all before the first store: one by one each waited for the one before, 180 clocks a row)
        float x[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) {
          float sa = sa_of[0];
#pragma unroll
          for (int j = 1; j < (NC + 31) / 32; j++)
            if ((q + i) / 32 == j) sa = sa_of[j];
          x[i] = int8_scaled(ok ? v[i] : 0u, __shfl_sync(0xffffffffu, sa, (q + i) & 31), sw);
        }
        const size_t at = (size_t)q * prm.N + n;
        if (prm.out_bf16) {
          uint16_t* const to = reinterpret_cast<uint16_t*>(prm.out) + at;
#pragma unroll
          for (int i = 0; i < kAtOnce; i++) store_if(to + (size_t)i * prm.N, __bfloat16_as_ushort(__float2bfloat16_rn(x[i])), mine && q + i < q1);
        } else {
          float* const to = reinterpret_cast<float*>(prm.out) + at;
#pragma unroll
          for (int i = 0; i < kAtOnce; i++) store_if(to + (size_t)i * prm.N, x[i], mine && q + i < q1);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->acc_empty[buf]);
    }
    fence_chained_writes();
  }
  tile_end<SH>(tmem, size);
}

struct PairBars {
  uint64_t full[PairShape::kStages], empty[PairShape::kStages], acc_full[2], acc_empty[2], drain;
  uint32_t tmem_base;
  volatile int32_t abort_flag;
};
__device__ __noinline__ void pair_wait_slow(uint64_t* bar, uint32_t parity, PairBars* b, int32_t* status) {
  for (uint32_t i = 0; i < kSpinLimit; i++) {
    if (mbar_try_wait(bar, parity)) return;
    if ((i & 255) == 255 && b->abort_flag) return;
    if (i > 512) __nanosleep(20);
  }
  b->abort_flag = 1;
  set_status(status, RELUX_ERR_TIMEOUT);
}
__device__ __forceinline__ void pair_wait(uint64_t* bar, uint32_t parity, PairBars* b, int32_t* status) {
  if (!mbar_try_wait(bar, parity)) pair_wait_slow(bar, parity, b, status);
}

// More rows.  grid (tiles x parts of K x 2), 192 threads, the roles as above; a pair's MMAs are issued by its first CTA.  A CTA loads half of the columns that it multiplies
// with: 32 KB a step where a CTA by itself loaded 48 for 128 x 256, which L2 did not deliver at the rate of the MMAs (78 of 96 bytes a clock and SM).
__global__ void __launch_bounds__(192, 1) matmul_int8_pair_kernel(const __grid_constant__ Int8Maps maps, const __grid_constant__ Int8Params prm) {
  using SH = PairShape;
  constexpr int kStages = SH::kStages, kTile = SH::kTile;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* const out_tiles = smem + kStages * SH::kStage;
  float* const scales = reinterpret_cast<float*>(out_tiles + SH::kOut);
  PairBars* bars = reinterpret_cast<PairBars*>(out_tiles + SH::kOut + SH::kScales);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int size = (int)cluster_size() / 2, rank = (int)cluster_ctarank(), part = rank >> 1, side = rank & 1;
  const int first = blockIdx.x / (2 * size), stride = gridDim.x / (2 * size);
  const int k0 = part * prm.steps / size, k1 = (part + 1) * prm.steps / size;
  const uint16_t both = (uint16_t)(3u << (2 * part));
  chain_release();
  if ((smem_u32(smem) & 1023u) != 0) {   // (the same in every CTA)
    chain_wait();
    if (threadIdx.x == 0) set_status(prm.status, RELUX_ERR_UNSUPPORTED);
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; s++) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
    for (int b = 0; b < 2; b++) { mbar_init(&bars->acc_full[b], 1); mbar_init(&bars->acc_empty[b], 8); }
    mbar_init(&bars->drain, 1);
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc<2>(&bars->tmem_base, 2 * SH::kAcc);
    tmem_relinquish<2>();
  }
  tc_fence_before();
  cluster_sync();   // barriers and tensor memory of all
  tc_fence_after();
  if (size > 1) cluster_arrive();   // (for swap_slices: this CTA has begun)
  const uint32_t tmem = bars->tmem_base;

  if (warp == 4) {
    const bool el = elect_one();
    if (el) {
      tma_prefetch_desc(&maps.r);
      tma_prefetch_desc(&maps.c);
      int left = kPrefetchBytes / kStageRows;
      for (int tile = first; tile < prm.tiles && left > 0; tile += stride) {
        int r, c;
        wide_place(tile, prm.row_blocks, prm.col_tiles, r, c);
        for (int k = k0; k < k1 && left > 0; k++, left--) tma_prefetch_2d(&maps.c, k * (kStepBytes / 2), c * kTile + side * 128);
      }
    }
    __syncwarp();
    chain_wait();
    int g = 0;
    for (int tile = first; tile < prm.tiles; tile += stride) {
      int r, c;
      wide_place(tile, prm.row_blocks, prm.col_tiles, r, c);
      for (int k = k0; k < k1; k++, g++) {
        const int s = g % kStages;
        if (g >= kStages) pair_wait(&bars->empty[s], (g / kStages - 1) & 1, bars, prm.status);
        if (el) {
          uint8_t* st = smem + s * SH::kStage;
          const uint32_t full = mapa_u32(smem_u32(&bars->full[s]), (uint32_t)rank & ~1u);
          if (side == 0) mbar_expect_tx(&bars->full[s], 2 * SH::kStage);   // of both CTAs; out-of-range parts of a box are zero-filled and still counted
          tma_load_2d_2sm(st, &maps.r, k * (kStepBytes / 2), r * kTile + side * 128, full);
          tma_load_2d_2sm(st + kStageRows, &maps.c, k * (kStepBytes / 2), c * kTile + side * 128, full);
        }
        __syncwarp();
      }
    }
  } else if (warp == 5) {
    if (side == 0) {
      const bool el = elect_one();
      const uint32_t idesc = make_idesc_s8(kTile, kTile);
      int g = 0, piece = 0;
      for (int tile = first; tile < prm.tiles; tile += stride, piece++) {
        const uint32_t d = tmem + (piece & 1) * SH::kAcc;
        if (piece >= 2) pair_wait(&bars->acc_empty[piece & 1], ((piece >> 1) - 1) & 1, bars, prm.status);
        tc_fence_after();
        for (int k = k0; k < k1; k++, g++) {
          const int s = g % kStages;
          pair_wait(&bars->full[s], (g / kStages) & 1, bars, prm.status);
          tc_fence_after();
          if (el) {
            const uint32_t st = smem_u32(smem + s * SH::kStage);
            const uint64_t dR = make_desc_kmajor_sw128(st), dC = make_desc_kmajor_sw128(st + kStageRows);
#pragma unroll
            for (int kk = 0; kk < kStepBytes / 32; kk++)
              umma_ss_i8<2>(d, dR + ((uint32_t)(kk * 32) >> 4), dC + ((uint32_t)(kk * 32) >> 4), idesc, k != k0 || kk != 0);
            umma_commit_mc<2>(&bars->empty[s], both);
          }
          __syncwarp();
        }
        if (el) umma_commit_mc<2>(&bars->acc_full[piece & 1], both);
        __syncwarp();
      }
      // nothing of this pair is freed while an MMA is in flight, after a wait that gave up either
      if (el) umma_commit<2>(&bars->drain);
      __syncwarp();
      mbar_wait(&bars->drain, 0);
    }
  } else {
    chain_wait();
    const uint32_t lead_empty[2] = {mapa_u32(smem_u32(&bars->acc_empty[0]), (uint32_t)rank & ~1u), mapa_u32(smem_u32(&bars->acc_empty[1]), (uint32_t)rank & ~1u)};
    int piece = 0, staged = 0;
    for (int tile = first; tile < prm.tiles; tile += stride, piece++) {
      int r, c;
      wide_place(tile, prm.row_blocks, prm.col_tiles, r, c);
      const int buf = piece & 1, row0 = r * kTile + side * 128 + warp * 32;
      const uint32_t acc = tmem + ((uint32_t)(warp * 32) << 16) + buf * SH::kAcc;
      const int cols = min(kTile, prm.N - c * kTile);
      const float sa = row0 + lane < prm.M ? load_chained(prm.a_scale + row0 + lane) : 0.f;
      // (a warp that is here has passed the barrier of the tile before, and with it every warp the end of the one before that)
#pragma unroll
      for (int i = 0; i < kTile / 128; i++) {
        const int q = threadIdx.x + i * 128;
        scales[buf * kTile + q] = q < cols ? load_chained(prm.w_scale + c * kTile + q) : 0.f;
      }
      epilogue_sync();
      pair_wait(&bars->acc_full[buf], (piece >> 1) & 1, bars, prm.status);
      tc_fence_after();
      const bool ok = !bars->abort_flag;
      const int wide = prm.out_bf16 ? 64 : 32;   // columns of a store
      int q0 = 0, q1 = cols;   // the columns that this CTA finishes
      if (size > 1) {
        q0 = slice_begin(part, cols, wide, size);
        q1 = slice_begin(part + 1, cols, wide, size);
        swap_slices<SH, 2>(acc, cols, wide, size, part, smem);
      }
      // thread = row: 32 (bf16: 64) columns at a time to a staging tile of the warp, 128-byte swizzle, and out by TMA, which leaves out what lies past the last row or column
      uint8_t* const tiles = out_tiles + warp * 2 * 32 * kOutRow;
#pragma unroll 1
      for (int q = q0; q < q1; q += wide, staged++) {
        uint8_t* const tile_smem = tiles + (staged & 1) * 32 * kOutRow;
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");   // the store before the last has read its tile
        __syncwarp();
#pragma unroll 1
        for (int h = 0; h < wide && q + h < q1; h += 16) {   // (sixteen: code that runs once is fetched as it goes)
          uint32_t v[16];
          tmem_ld_32x32b_x8(acc + q + h, *reinterpret_cast<uint32_t(*)[8]>(v));
          tmem_ld_32x32b_x8(acc + q + h + 8, *reinterpret_cast<uint32_t(*)[8]>(v + 8));
          tmem_ld_wait();
          add_slices(smem, size, q1 - q0, q + h - q0, [&](int i, uint32_t u) { v[i] += u; });
          const float4* sw = reinterpret_cast<const float4*>(scales + buf * kTile + q + h);
          float x[16];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float4 s4 = sw[i];
            x[4 * i] = int8_scaled(ok ? v[4 * i] : 0u, sa, s4.x);
            x[4 * i + 1] = int8_scaled(ok ? v[4 * i + 1] : 0u, sa, s4.y);
            x[4 * i + 2] = int8_scaled(ok ? v[4 * i + 2] : 0u, sa, s4.z);
            x[4 * i + 3] = int8_scaled(ok ? v[4 * i + 3] : 0u, sa, s4.w);
          }
          if (prm.out_bf16) {
#pragma unroll
            for (int i = 0; i < 2; i++)
              *reinterpret_cast<uint4*>(tile_smem + swz128(lane, h / 8 + i)) =
                  make_uint4(round_bf16x2(x[8 * i], x[8 * i + 1]), round_bf16x2(x[8 * i + 2], x[8 * i + 3]), round_bf16x2(x[8 * i + 4], x[8 * i + 5]),
                             round_bf16x2(x[8 * i + 6], x[8 * i + 7]));
          } else {
#pragma unroll
            for (int i = 0; i < 4; i++) *reinterpret_cast<float4*>(tile_smem + swz128(lane, h / 4 + i)) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&maps.out, (c * kTile + q) * (prm.out_bf16 ? 1 : 2), row0, tile_smem);
          tma_store_commit();
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(lead_empty[buf]);   // the accumulator is free again
    }
    if (lane == 0) tma_store_wait_all();
    __syncwarp();
  }
  if (size > 1 && warp >= 4) {   // the epilogue's barriers count every thread
    cluster_wait();
    cluster_arrive();
    cluster_wait();
    cluster_arrive();
    cluster_wait();
  }
  tc_fence_before();
  cluster_sync();
  if (warp == 0) tmem_dealloc<2>(tmem, 2 * SH::kAcc);
}

}  // namespace

int32_t launch_matmul_int8(Pool* p, int M, int K, int N, const int8_t* a, const float* a_scale, const int8_t* w, const float* w_scale, void* out,
                           bool out_bf16) {
  Int8Params prm{};
  Int8Maps maps{};
  const bool wide = M > 128;
  int nc = 16;
  while (nc < M && nc < 128) nc *= 2;
  prm.M = M;
  prm.N = N;
  prm.steps = (K + kStepBytes - 1) / kStepBytes;
  prm.row_blocks = (M - 1) / PairShape::kTile + 1;
  prm.col_tiles = (N - 1) / (wide ? PairShape::kTile : kRowsOp) + 1;
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
  bool made = make_tmap_2d(&maps.r, (void*)rows, (uint64_t)(wide ? M : N), (uint64_t)K / 2, kStepBytes / 2, kRowsOp) &&
              make_tmap_2d(&maps.c, (void*)cols, (uint64_t)(wide ? N : M), (uint64_t)K / 2, kStepBytes / 2, wide ? 128 : nc);
  if (wide) made = made && make_tmap_2d(&maps.out, out, (uint64_t)M, (uint64_t)N * (out_bf16 ? 1 : 2), kOutRow / 2, 32);
  if (!made) {
    set_error("tensor map for 8-bit rows could not be encoded");
    return RELUX_ERR_CUDA;
  }
  if (wide) return launch_tiles<PairShape, 192, 2>(p, matmul_int8_pair_kernel, prm.tiles, prm.steps, maps, prm);
  switch (nc) {
    case 16: return launch_tiles<Int8Shape<16>>(p, matmul_int8_kernel<16>, prm.tiles, prm.steps, maps, prm);
    case 32: return launch_tiles<Int8Shape<32>>(p, matmul_int8_kernel<32>, prm.tiles, prm.steps, maps, prm);
    case 64: return launch_tiles<Int8Shape<64>>(p, matmul_int8_kernel<64>, prm.tiles, prm.steps, maps, prm);
    default: return launch_tiles<Int8Shape<128>>(p, matmul_int8_kernel<128>, prm.tiles, prm.steps, maps, prm);
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
