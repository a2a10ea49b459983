// t = f_s x A_s^T for calls whose rows fill tiles of one request (LoraTiles): the rows are the M operand of the MMA and the adapter's rank its N operand, both K-major.
// What lora_down_kernel does for rows wherever they lie; here an adapter is read once for 128 rows and not for 16.
//
// bf16 rows come by TMA.  float32 rows are rounded on their way into the stages by eight warps, which write the projection's operand as well.  Bound: HBM, x once (and
// its rounded form).  A tile's rows past the request's end meet the wrong adapter and are not stored.  Tiles as in tile_gemm.cuh, cut along K among a cluster while
// there are idle SMs.
#include "lora.cuh"
#include "tile_gemm.cuh"

namespace relux {

namespace {

constexpr int kRoundWarps = 16;
template <int NC>
using DownShape = TileShape<NC, 0, NC <= 32 ? 64 : NC == 64 ? 96 : 160>;
template <int NC>
constexpr bool fits = slices_fit(NC, 8, DownShape<NC>::kMaxCluster, 0, DownShape<NC>::kSlices);
static_assert(fits<16> && fits<32> && fits<64> && fits<128>, "no room for the slices");

struct DownMaps {
  CUtensorMap x;   // bf16 rows [M][K], box 64 k x 128 rows
  CUtensorMap a;   // [slots * rank][K], box 64 k x NC rows (rank 8: another adapter's rows behind it, whose sums are not read)
};
struct DownTileParams {
  int32_t rank, steps, tiles, K;
  const float* x_f32;      // or nullptr: bf16 rows
  uint16_t* x_bf16;
  const float* factors;    // [slots], or nullptr: ones
  uint16_t* t_hi;          // [M][rank]
  uint16_t* t_lo;
  int32_t* status;
};

// grid (tiles x parts of K): warps 0-3 epilogue, warp 4 TMA producer, warp 5 MMA issuer, then the warps that round.
template <int NC, bool kRounds>
__global__ void __launch_bounds__(kRounds ? 192 + 32 * kRoundWarps : 192, 1)
lora_rows_kernel(const __grid_constant__ DownMaps maps, const __grid_constant__ DownTileParams prm, const __grid_constant__ LoraTiles list) {
  using SH = DownShape<NC>;
  constexpr int kStages = SH::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* const slices = smem + kStages * SH::kStage;
  TileBars* bars = reinterpret_cast<TileBars*>(slices + SH::kSlices);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int size = (int)cluster_size(), part = (int)cluster_ctarank();
  const int first = blockIdx.x / size, stride = gridDim.x / size;
  const int k0 = part * prm.steps / size, k1 = (part + 1) * prm.steps / size;
  // waits before it releases: the projection behind it reads its weights early (launch_chained, head of a chain)
  if ((smem_u32(smem) & 1023u) != 0) {   // (the same in every CTA)
    chain_wait();
    if (threadIdx.x == 0) set_status(prm.status, RELUX_ERR_UNSUPPORTED);
    return;
  }
  const uint32_t tmem = tile_setup<SH>(bars, size, kRounds ? 1 + kRoundWarps : 1);
  chain_wait();
  chain_release();

  if (warp == 4) {
    const bool el = elect_one();
    int g = 0;
    for (int tile = first; tile < prm.tiles; tile += stride) {
      const int slot = list.slot[tile];
      if (slot < 0) continue;
      for (int k = k0; k < k1; k++, g++) {
        const int s = g % kStages;
        if (g >= kStages) tile_wait(&bars->empty[s], (g / kStages - 1) & 1, bars, prm.status);
        if (el) {
          uint8_t* st = smem + s * SH::kStage;
          mbar_expect_tx(&bars->full[s], kRounds ? NC * kStepBytes : SH::kStage);   // out-of-range parts of a box are zero-filled and still counted
          if (!kRounds) tma_load_2d(st, &maps.x, k * 64, list.row[tile], &bars->full[s]);
          tma_load_2d(st + kStageRows, &maps.a, k * 64, slot * prm.rank, &bars->full[s]);
        }
        __syncwarp();
      }
    }
  } else if (warp == 5) {
    const bool el = elect_one();
    const uint32_t idesc = make_idesc_bf16(kRowsOp, NC, false, false);
    int g = 0, piece = 0;
    for (int tile = first; tile < prm.tiles; tile += stride) {
      if (list.slot[tile] < 0) continue;
      const uint32_t d = tmem + (piece & 1) * SH::kAcc;
      if (piece >= 2) tile_wait(&bars->acc_empty[piece & 1], ((piece >> 1) - 1) & 1, bars, prm.status);
      tc_fence_after();
      for (int k = k0; k < k1; k++, g++) {
        const int s = g % kStages;
        tile_wait(&bars->full[s], (g / kStages) & 1, bars, prm.status);
        tc_fence_after();
        if (el) {
          const uint32_t st = smem_u32(smem + s * SH::kStage);
          const uint64_t dX = make_desc_kmajor_sw128(st), dA = make_desc_kmajor_sw128(st + kStageRows);
#pragma unroll
          for (int kk = 0; kk < 4; kk++) umma_ss<1>(d, dX + ((uint32_t)(kk * 32) >> 4), dA + ((uint32_t)(kk * 32) >> 4), idesc, k != k0 || kk != 0);
          umma_commit<1>(&bars->empty[s]);
        }
        __syncwarp();
      }
      if (el) umma_commit<1>(&bars->acc_full[piece & 1]);
      __syncwarp();
      piece++;
    }
  } else if (kRounds && warp >= 6) {
    // thread: four pieces of four k of a step, the next step's on their way while they are rounded.  (A warp loads 256 neighbouring bytes of two rows at once;
    // pieces of eight k, half of each 32 bytes a load, asked L2 for everything twice: 3300 rows of
    // 8192, rank 16, N 1024, 125 us so and 99.  Two or three steps on their way are no faster for long K, and slower for short.)
    const int id = threadIdx.x - 192, quad = id & 15;
    constexpr int kRowsAtOnce = 2 * kRoundWarps, kPieces = 128 / kRowsAtOnce;
    int g = 0;
    for (int tile = first; tile < prm.tiles; tile += stride) {
      const int slot = list.slot[tile], rows = list.rows[tile];
      const size_t base = (size_t)list.row[tile] * prm.K;
      float4 next[kPieces];
      auto fetch = [&](int k) {
        const int col = k * 64 + 4 * quad;
#pragma unroll
        for (int i = 0; i < kPieces; i++) {
          const int row = i * kRowsAtOnce + (id >> 4);
          const bool in = k < k1 && row < rows && col < prm.K;   // K is a multiple of 8
          next[i] = in ? load_chained(reinterpret_cast<const float4*>(prm.x_f32 + base + (size_t)row * prm.K + col)) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      };
      fetch(k0);
      for (int k = k0; k < k1; k++) {
        uint2 y[kPieces];
#pragma unroll
        for (int i = 0; i < kPieces; i++) y[i] = make_uint2(round_bf16x2(next[i].x, next[i].y), round_bf16x2(next[i].z, next[i].w));
        fetch(k + 1);
        const int col = k * 64 + 4 * quad;
#pragma unroll
        for (int i = 0; i < kPieces; i++) {
          const int row = i * kRowsAtOnce + (id >> 4);
          if (row < rows && col < prm.K) *reinterpret_cast<uint2*>(prm.x_bf16 + base + (size_t)row * prm.K + col) = y[i];
        }
        if (slot >= 0) {
          const int s = g % kStages;
          if (g >= kStages) tile_wait(&bars->empty[s], (g / kStages - 1) & 1, bars, prm.status);
#pragma unroll
          for (int i = 0; i < kPieces; i++) *reinterpret_cast<uint2*>(smem + s * SH::kStage + swz128(i * kRowsAtOnce + (id >> 4), quad >> 1) + (quad & 1) * 8) = y[i];
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->full[s]);
          g++;
        }
      }
    }
    fence_chained_writes();   // the projection reads them by TMA
  } else {
    int piece = 0;
    for (int tile = first; tile < prm.tiles; tile += stride) {
      const int slot = list.slot[tile];
      if (slot < 0) {
        if (size > 1) {   // (the cluster's only tile: swap_slices' barriers)
          cluster_wait();
          cluster_arrive();
          cluster_wait();
        }
        continue;
      }
      const int buf = piece & 1, m = warp * 32 + lane;
      const uint32_t acc = tmem + ((uint32_t)(warp * 32) << 16) + buf * SH::kAcc;
      const float factor = prm.factors ? load_chained(prm.factors + slot) : 1.f;
      tile_wait(&bars->acc_full[buf], (piece >> 1) & 1, bars, prm.status);
      tc_fence_after();
      const bool ok = !bars->abort_flag, mine = m < list.rows[tile];
      int q0 = 0, q1 = prm.rank;   // what this CTA finishes of the rank
      if (size > 1) {
        q0 = slice_begin(part, prm.rank, 8, size);
        q1 = slice_begin(part + 1, prm.rank, 8, size);
        swap_slices<SH>(acc, prm.rank, 8, size, part, slices);
      }
      const float* const got = reinterpret_cast<const float*>(slices) + threadIdx.x;
      const size_t to = (size_t)(list.row[tile] + m) * prm.rank;
#pragma unroll 1
      for (int q = q0; q < q1; q += 8) {
        uint32_t v[8];
        tmem_ld_32x32b_x8(acc + q, v);
        tmem_ld_wait();
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = ok ? __uint_as_float(v[i]) : 0.f;
#pragma unroll 1
        for (int s = 0; s < size - 1; s++)
#pragma unroll
          for (int i = 0; i < 8; i++) x[i] += got[(s * (q1 - q0) + q - q0 + i) * kRowsOp];
        uint2 hi[2], lo[2];
        split_halves(make_float4(x[0], x[1], x[2], x[3]), factor, hi[0], lo[0]);
        split_halves(make_float4(x[4], x[5], x[6], x[7]), factor, hi[1], lo[1]);
        if (mine) {
          *reinterpret_cast<uint4*>(prm.t_hi + to + q) = make_uint4(hi[0].x, hi[0].y, hi[1].x, hi[1].y);
          *reinterpret_cast<uint4*>(prm.t_lo + to + q) = make_uint4(lo[0].x, lo[0].y, lo[1].x, lo[1].y);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->acc_empty[buf]);
      piece++;
    }
    fence_chained_writes();
  }
  tile_end<SH>(tmem, size);
}

template <int NC>
int32_t launch_nc(Pool* p, const DownMaps& maps, const DownTileParams& prm, const LoraTiles& tiles) {
  return prm.x_f32 ? launch_tiles<DownShape<NC>, 192 + 32 * kRoundWarps>(p, lora_rows_kernel<NC, true>, prm.tiles, prm.steps, maps, prm, tiles)
                   : launch_tiles<DownShape<NC>>(p, lora_rows_kernel<NC, false>, prm.tiles, prm.steps, maps, prm, tiles);
}

}  // namespace

int32_t launch_lora_rows(Pool* p, const relux_matmul_lora_args* a, const LoraTiles& tiles, const uint16_t* x, uint16_t* rounded, uint16_t* t_hi, uint16_t* t_lo) {
  DownTileParams prm{};
  DownMaps maps{};
  prm.rank = a->rank;
  prm.steps = (a->k + 63) / 64;
  prm.tiles = tiles.n;
  prm.K = a->k;
  if (!x) prm.x_f32 = (const float*)a->x;
  prm.x_bf16 = rounded;
  prm.factors = a->factors;
  prm.t_hi = t_hi;
  prm.t_lo = t_lo;
  prm.status = p->d_status;
  const int nc = std::max(16, a->rank);
  if ((x && !make_tmap_2d(&maps.x, (void*)x, (uint64_t)a->m, (uint64_t)a->k, 64, kRowsOp)) ||
      !make_tmap_2d(&maps.a, (void*)a->lora_a, (uint64_t)a->n_slots * a->rank, (uint64_t)a->k, 64, nc)) {
    set_error("tensor map for rows with adapters could not be encoded");
    return RELUX_ERR_CUDA;
  }
  switch (nc) {
    case 16: return launch_nc<16>(p, maps, prm, tiles);
    case 32: return launch_nc<32>(p, maps, prm, tiles);
    case 64: return launch_nc<64>(p, maps, prm, tiles);
    default: return launch_nc<128>(p, maps, prm, tiles);
  }
}

}  // namespace relux
