// Product of 8-bit rows with 8-bit weights on the tensor cores: C[m][n] = sa[m] * sw[n] * sum_k a[m][k] * w[n][k], the sum in 32-bit whole
// numbers, exact for every K that the call takes, whatever the order of its parts.
//
// Bound: HBM up to some hundred rows (a weight is one byte, read once), the tensor cores above.  Both operands lie K-major, as the quantiser and the
// import write them.  Tiles as in tile_gemm.cuh.  Whole numbers add up to the same in any order, so a result does not depend on the cut along K.
// The weights of a CTA's first steps are brought into L2, not into shared memory, while the launch before this one ends: a prefetch returns no data,
// so it may be early whatever that launch writes.
// What did not do: columns as the M operand throughout, whose epilogue stored two bytes a thread (644 us for 8192 x 4096 x 16384, the loads and MMAs
// alone 320); parts of tiles joined through L2 by the last of them (35 us more at 300 x 8192 x 4096).
#include "tile_gemm.cuh"

namespace relux {

namespace {

constexpr int kPrefetchBytes = 256 << 10;   // of weights, by CTA

template <int NC>
using Int8Shape = TileShape<NC, NC == 256 ? 2 * NC * 4 : 0>;   // wide: the columns' scales, by accumulator
static_assert(slices_fit(16, 1, 8, 0, Int8Shape<16>::kSlices) && slices_fit(32, 1, 8, 0, Int8Shape<32>::kSlices) && slices_fit(64, 1, 8, 0, Int8Shape<64>::kSlices) &&
              slices_fit(128, 1, 8, 0, Int8Shape<128>::kSlices) && slices_fit(256, 32, 4, 0, Int8Shape<256>::kStages * Int8Shape<256>::kStage) &&
              slices_fit(256, 64, 4, 0, Int8Shape<256>::kStages * Int8Shape<256>::kStage), "no room for the slices");

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

template <bool kWide>
__device__ __forceinline__ void tile_place(const Int8Params& p, int tile, int& r, int& c) {
  r = tile;
  c = 0;
  if constexpr (kWide) wide_place(tile, p.row_blocks, p.col_tiles, r, c);
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
  TileBars* bars = reinterpret_cast<TileBars*>(out_tiles + SH::kOut + SH::kSlices + SH::kMore);
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
      constexpr int kWeightBytes = kWide ? NC * kStepBytes : kStageRows;
      int left = kPrefetchBytes / kWeightBytes;
      for (int tile = first; tile < prm.tiles && left > 0; tile += stride) {
        int r, c;
        tile_place<kWide>(prm, tile, r, c);
        for (int k = k0; k < k1 && left > 0; k++, left--) {
          if constexpr (kWide) tma_prefetch_2d(&maps.c, k * (kStepBytes / 2), c * NC);
          else tma_prefetch_2d(&maps.r, k * (kStepBytes / 2), r * kRowsOp);
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
        if (g >= kStages) tile_wait(&bars->empty[s], (g / kStages - 1) & 1, bars, prm.status);
        if (el) {
          uint8_t* st = smem + s * SH::kStage;
          mbar_expect_tx(&bars->full[s], SH::kStage);   // out-of-range parts of a box are zero-filled and still counted
          tma_load_2d(st, &maps.r, k * (kStepBytes / 2), r * kRowsOp, &bars->full[s]);
          tma_load_2d(st + kStageRows, &maps.c, k * (kStepBytes / 2), c * NC, &bars->full[s]);
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
        epilogue_sync();
      }
      tile_wait(&bars->acc_full[buf], (piece >> 1) & 1, bars, prm.status);
      tc_fence_after();
      const bool ok = !bars->abort_flag;
      // the columns that this CTA finishes
      int q0 = 0, q1 = cols;
      if (size > 1) {
        const int grain = !kWide ? 1 : prm.out_bf16 ? 64 : 32;   // (wide: one store's columns)
        q0 = slice_begin(rank, cols, grain, size);
        q1 = slice_begin(rank + 1, cols, grain, size);
        swap_slices<SH>(acc, cols, grain, size, rank, slices);
      }
      if constexpr (!kWide) {
        const int32_t* const got = reinterpret_cast<const int32_t*>(slices) + warp * 32 + lane;
        // thread = column; a warp writes 64 or 128 bytes of a row at once
        constexpr int kAtOnce = NC <= 32 ? 8 : 16;
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
            x[i] = int8_scaled(ok ? v[i] : 0u, __shfl_sync(0xffffffffu, sa, (q + i) & 31), own);
          }
          const size_t at = (size_t)q * prm.N + at_row;
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
          for (int h = 0; h < wide && q + h < q1; h += 16) {   // (sixteen: code that runs once is fetched as it goes)
            uint32_t v[16];
            tmem_ld_32x32b_x8(acc + q + h, *reinterpret_cast<uint32_t(*)[8]>(v));
            tmem_ld_32x32b_x8(acc + q + h + 8, *reinterpret_cast<uint32_t(*)[8]>(v + 8));
            tmem_ld_wait();
            add_slices(slices, size, q1 - q0, q + h - q0, [&](int i, uint32_t u) { v[i] += u; });
            const float4* sw = reinterpret_cast<const float4*>(scales + buf * NC + q + h);
            float x[16];
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const float4 s4 = sw[i];
              x[4 * i] = int8_scaled(ok ? v[4 * i] : 0u, own, s4.x);
              x[4 * i + 1] = int8_scaled(ok ? v[4 * i + 1] : 0u, own, s4.y);
              x[4 * i + 2] = int8_scaled(ok ? v[4 * i + 2] : 0u, own, s4.z);
              x[4 * i + 3] = int8_scaled(ok ? v[4 * i + 3] : 0u, own, s4.w);
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
  tile_end<SH>(tmem, size);
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
  prm.steps = (K + kStepBytes - 1) / kStepBytes;
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
  bool made = make_tmap_2d(&maps.r, (void*)rows, (uint64_t)(wide ? M : N), (uint64_t)K / 2, kStepBytes / 2, kRowsOp) &&
              make_tmap_2d(&maps.c, (void*)cols, (uint64_t)(wide ? N : M), (uint64_t)K / 2, kStepBytes / 2, nc);
  if (wide) made = made && make_tmap_2d(&maps.out, out, (uint64_t)M, (uint64_t)N * (out_bf16 ? 1 : 2), kOutRow / 2, 32);
  if (!made) {
    set_error("tensor map for 8-bit rows could not be encoded");
    return RELUX_ERR_CUDA;
  }
  switch (nc) {
    case 16: return launch_tiles<Int8Shape<16>>(p, matmul_int8_kernel<16>, prm.tiles, prm.steps, maps, prm);
    case 32: return launch_tiles<Int8Shape<32>>(p, matmul_int8_kernel<32>, prm.tiles, prm.steps, maps, prm);
    case 64: return launch_tiles<Int8Shape<64>>(p, matmul_int8_kernel<64>, prm.tiles, prm.steps, maps, prm);
    case 128: return launch_tiles<Int8Shape<128>>(p, matmul_int8_kernel<128>, prm.tiles, prm.steps, maps, prm);
    default: return launch_tiles<Int8Shape<256>>(p, matmul_int8_kernel<256>, prm.tiles, prm.steps, maps, prm);
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
