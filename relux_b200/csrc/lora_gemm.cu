// The shared projection of a call with low-rank adapters, C[m] = x[m] W + t[m] B_s^T, s the adapter of row m, in one launch behind lora_down_kernel
// (lora.cu) or lora_rows_kernel (lora_rows.cu), which take t = x A_s^T.  x and W are bf16, W as the layers hold it ([K][N]: MN-major in the MMA), B_s [N][rank].  Tiles as in tile_gemm.cuh.
//
//   * Up to 16 rows (bound: HBM, W and the adapters in use): the epilogue's warps and as many helpers, idle while W streams, take t B_s^T on the CUDA cores
//     in float32, a thread a column, and add it to the sums when they come: a row meets its own adapter only.  float32 rows are split in two bf16 halves on
//     their way into the stages: W is multiplied with both, which costs MMAs and no bytes.  (Of 17 to 128 rows that takes longer than W: 64 rows of
//     rank 16 x 4096 x 6144 24 us so, 21 by lora_up_kernel behind a GEMM of its own.)
//   * Wide tiles (bound: the tensor cores): every tile holds rows of one request, so that t B_s^T is further K steps of the same accumulator, t as two
//     bf16 halves, hi and lo.  Rows of the tile past the request's end are computed with the wrong adapter and not stored.
//     A row never meets another request's adapter by way of a zero: zero times an infinity in that adapter would be NaN in this row.
//   * Of a row or two every CTA takes t over its part of K itself, and the parts of t go to the others with the slices of the sums: no launch before this one.
// Behind another launch of the call W is read ahead of it, and bf16 x too: that one is a chain's head (launch_chained).
#include "lora.cuh"
#include "tile_gemm.cuh"

namespace relux {

namespace {

constexpr int kPrefetchSteps = 32;
constexpr int kRowsT = kNarrowSums * 4;   // bytes of t
constexpr int kRing = 8;           // pieces of adapters, eight of a row's rank for a column, that are on their way for each of 256 threads
template <int NC>
using LoraShape = TileShape<NC, NC == 256 ? 0 : kRowsT + kRing * 256 * 16, NC + 8, NC == 256 ? 1 : 2, 8>;   // the adapter's part of a slice lies with the others'; nine stages: 12 rows 0.3 us more
static_assert(slices_fit(16, 1, 8, 1, LoraShape<16>::kSlices) && slices_fit(256, 32, 4, 0, LoraShape<256>::kStages * LoraShape<256>::kStage) &&
              slices_fit(256, 64, 4, 0, LoraShape<256>::kStages * LoraShape<256>::kStage), "no room for the slices");

template <int NC, bool kOne>
constexpr int kLoraGemmThreads = NC == 256 ? 192 : kOne ? 448 : 320;

struct LoraMaps {
  CUtensorMap x;      // [M][K], box 64 k x the rows of an operand
  CUtensorMap w;      // [K][N], box 64 n x 64 k
  CUtensorMap t[2];   // wide: hi and lo [M][rank], box 64 x 128 rows, zeros past the rank
  CUtensorMap b;      // wide: [slots * N][rank], box 64 x 256 rows
  CUtensorMap out;    // wide: rows of two-byte elements, two for a float32
};
struct LoraGemmParams {
  int32_t M, N, rank, steps, tiles, col_tiles, out_bf16, adds;
  int32_t x_early;           // x was complete before the chain's head began
  const float* x_f32;        // up to kNarrowRows rows of float32 [M][K]: split here, into the stages
  int32_t K;
  const float* t;            // narrow: [M][rank], without factors
  const uint16_t* b;         // narrow: [slots][N][rank]
  const float* factors;      // narrow: [slots], or nullptr
  const uint16_t* a;         // in one launch: [slots][rank][K]
  const void* x_rows;        // in one launch: the caller's rows, bf16 or (x_f32) float32
  void* out;
  int32_t* status;
};
static_assert(LoraShape<kNarrowRows>::kMaxCluster * kOneT * 4 <= kRowsT && LoraShape<kNarrowRows>::kMaxCluster * kOneT <= 128, "no room for the parts of t, or no thread");
struct NarrowRows {
  int32_t slot[kNarrowRows];   // of every row, or -1
};

template <int NC, class Rows, bool kOne>
__global__ void __launch_bounds__(kLoraGemmThreads<NC, kOne>, 1) lora_gemm_kernel(const __grid_constant__ LoraMaps maps, const __grid_constant__ LoraGemmParams prm, const __grid_constant__ Rows list) {
  using SH = LoraShape<NC>;
  constexpr int kStages = SH::kStages;
  constexpr bool kWide = SH::kWide;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* const out_tiles = smem + kStages * SH::kStage;
  uint8_t* const slices = kWide ? smem : out_tiles + SH::kOut;
  float* const t_rows = reinterpret_cast<float*>(out_tiles + SH::kOut + SH::kSlices);
  TileBars* bars = reinterpret_cast<TileBars*>(out_tiles + SH::kOut + SH::kSlices + SH::kMore);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int size = (int)cluster_size(), rank = (int)cluster_ctarank();
  const int first = blockIdx.x / size, stride = gridDim.x / size;
  const int t_steps = (prm.rank + 63) / 64;   // of one half of t
  // place of a tile, its rows and its steps of K
  struct Place {
    int c, row0, rows, slot, k0, k1;
  };
  auto place = [&](int tile) {
    Place at;
    if constexpr (kWide) {
      int r;
      wide_place(tile, list.n, prm.col_tiles, r, at.c);
      at.row0 = list.row[r];
      at.rows = list.rows[r];
      at.slot = list.slot[r];
    } else {
      at.c = tile;
      at.row0 = 0;
      at.rows = prm.M;
      at.slot = -1;
    }
    const int steps = prm.steps + (at.slot >= 0 ? 2 * t_steps : 0);
    at.k0 = rank * steps / size;
    at.k1 = (rank + 1) * steps / size;
    return at;
  };
  chain_release();
  if ((smem_u32(smem) & 1023u) != 0) {   // (the same in every CTA)
    chain_wait();
    if (threadIdx.x == 0) set_status(prm.status, RELUX_ERR_UNSUPPORTED);
    return;
  }
  const bool rounds_x = NC == kNarrowRows && prm.x_f32;
  const uint32_t tmem = tile_setup<SH>(bars, size, rounds_x ? 5 : 1);

  bool has_t = false;
  auto low_sync = [] { asm volatile("bar.sync 2, 256;" ::: "memory"); };
  auto low_wait = [&] {
    if (!has_t) chain_wait();
    has_t = true;
    low_sync();   // the tile before is done with t
  };
  // Up to 16 rows: t B_s^T of a tile and this CTA's rows, behind the slices of the others.  By the epilogue's warps (half 0) and the helpers (half 1), a thread a
  // column, rows in turn.  What a thread reads of B_s goes through a ring of its own in shared memory, the first pieces ahead of t.  (Through registers, by
  // unrolled loops, 32 rows of rank 16 took 11000 clocks: code that runs once is fetched as it goes.)
  auto low_half = [&](const Place& at, int half) {
    const int id = half ? threadIdx.x - 192 : threadIdx.x, n = at.c * kRowsOp + id;
    const int q0 = size > 1 ? slice_begin(rank, prm.M, 1, size) : 0, q1 = size > 1 ? slice_begin(rank + 1, prm.M, 1, size) : prm.M;
    const bool mine = n < prm.N;
    float* const low = reinterpret_cast<float*>(slices) + (size - 1) * (q1 - q0) * kRowsOp + id;
    const int shift = 31 - __clz(prm.rank >> 3), chunks = 1 << shift;   // ranks are powers of two
    uint8_t* const ring = reinterpret_cast<uint8_t*>(t_rows) + kRowsT + (half * 128 + id) * 16;
    const int count = ((q1 - q0 + 1 - half) >> 1) << shift;
    constexpr int kFetch = kRing / 2;
    auto fetch = [&](int first_piece) {   // half a ring: piece i is chunk i % chunks of row i / chunks of this half
#pragma unroll 1
      for (int i = first_piece; i < min(first_piece + kFetch, count); i++) {
        const int slot = list.slot[q0 + 2 * (i >> shift) + half];
        const bool some = slot >= 0 && mine;
        const uint16_t* src = prm.b + ((size_t)(some ? slot : 0) * prm.N + (some ? n : 0)) * prm.rank + (i & (chunks - 1)) * 8;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(ring + (i & (kRing - 1)) * (256 * 16))), "l"(src), "r"(some ? 16 : 0) : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(0);   // adapters were complete before the chain's head began
    fetch(kFetch);
    low_wait();
    for (int i = threadIdx.x - (half ? 64 : 0); i < (q1 - q0) * prm.rank / 4; i += 256) {
      const int slot = list.slot[q0 + 4 * i / prm.rank];
      float4 u = make_float4(0.f, 0.f, 0.f, 0.f);   // (what t holds of a row without an adapter is nobody's)
      if (slot >= 0) {
        u = load_chained(reinterpret_cast<const float4*>(prm.t + (size_t)q0 * prm.rank) + i);
        const float f = prm.factors ? load_chained(prm.factors + slot) : 1.f;
        u.x *= f; u.y *= f; u.z *= f; u.w *= f;
      }
      reinterpret_cast<float4*>(t_rows)[i] = u;
    }
    low_sync();
    float sum = 0.f;
#pragma unroll 1
    for (int g = 0; g < count; g += kFetch) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
#pragma unroll 1
      for (int i = g; i < min(g + kFetch, count); i++) {
        const int c = i & (chunks - 1), q = 2 * (i >> shift) + half;
        const uint4 w = *reinterpret_cast<const uint4*>(ring + (i & (kRing - 1)) * (256 * 16));
        const float4* t = reinterpret_cast<const float4*>(t_rows + q * prm.rank + c * 8);
        const float4 t0 = t[0], t1 = t[1];
        if (c == 0) sum = 0.f;
        sum = fmaf(t0.x, bf16_lo(w.x), sum); sum = fmaf(t0.y, bf16_hi(w.x), sum); sum = fmaf(t0.z, bf16_lo(w.y), sum); sum = fmaf(t0.w, bf16_hi(w.y), sum);
        sum = fmaf(t1.x, bf16_lo(w.z), sum); sum = fmaf(t1.y, bf16_hi(w.z), sum); sum = fmaf(t1.z, bf16_lo(w.w), sum); sum = fmaf(t1.w, bf16_hi(w.w), sum);
        if (c == chunks - 1) low[q * kRowsOp] = sum;
      }
      fetch(g + 2 * kFetch);
    }
    low_sync();
  };

  // In one launch: the part of t that comes from this CTA's part of K, [row][rank] with factors, by the epilogue's warps and the last four, four sums of a row a warp at a time.  The
  // cluster's parts lie side by side, kOneT values each.
  auto down_part = [&] {
    const int c0 = rank * prm.steps / size * 64, c1 = min((rank + 1) * prm.steps / size * 64, prm.K);
    for (int d = 4 * (warp < 4 ? warp : warp - 6); d < prm.M * prm.rank; d += 32) {   // (a rank is a multiple of eight)
      const int row = d / prm.rank, slot = list.slot[row];
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      if (slot >= 0) {
        const uint16_t* const a = prm.a + ((size_t)slot * prm.rank + d % prm.rank) * prm.K;
#pragma unroll 4
        for (int k = c0 + 8 * lane; k < c1; k += 256) {
          uint4 w[4];
#pragma unroll
          for (int i = 0; i < 4; i++) w[i] = load_chained(reinterpret_cast<const uint4*>(a + (size_t)i * prm.K + k));
          float x[8];
          if (prm.x_f32) {
            const float4* src = reinterpret_cast<const float4*>(prm.x_f32 + (size_t)row * prm.K + k);
            const float4 u = load_chained(src), v = load_chained(src + 1);
            x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
          } else {
            const uint4 u = load_chained(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(prm.x_rows) + (size_t)row * prm.K + k));
            x[0] = bf16_lo(u.x); x[1] = bf16_hi(u.x); x[2] = bf16_lo(u.y); x[3] = bf16_hi(u.y); x[4] = bf16_lo(u.z); x[5] = bf16_hi(u.z); x[6] = bf16_lo(u.w); x[7] = bf16_hi(u.w);
          }
#pragma unroll
          for (int i = 0; i < 4; i++) {
            sum[i] = fmaf(x[0], bf16_lo(w[i].x), sum[i]); sum[i] = fmaf(x[1], bf16_hi(w[i].x), sum[i]);
            sum[i] = fmaf(x[2], bf16_lo(w[i].y), sum[i]); sum[i] = fmaf(x[3], bf16_hi(w[i].y), sum[i]);
            sum[i] = fmaf(x[4], bf16_lo(w[i].z), sum[i]); sum[i] = fmaf(x[5], bf16_hi(w[i].z), sum[i]);
            sum[i] = fmaf(x[6], bf16_lo(w[i].w), sum[i]); sum[i] = fmaf(x[7], bf16_hi(w[i].w), sum[i]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; i++) sum[i] = warp_sum(sum[i]);
      const float f = slot >= 0 && prm.factors ? load_chained(prm.factors + slot) : 1.f;
      if (lane < 4) t_rows[rank * kOneT + d + lane] = f * (lane == 0 ? sum[0] : lane == 1 ? sum[1] : lane == 2 ? sum[2] : sum[3]);
    }
  };
  // The parts to the others, with the slices: a thread a value and a CTA.
  auto send_parts = [&] {
    const int i = threadIdx.x % kOneT, to = threadIdx.x / kOneT;
    if (to < size && to != rank && i < prm.M * prm.rank)
      store_cluster(mapa_u32(smem_u32(t_rows + rank * kOneT + i), (uint32_t)to), __float_as_uint(t_rows[rank * kOneT + i]));
  };
  // t B_s^T of a tile, a thread a column, for each of up to kOneT / 8 rows: of all of t, since parts of it that an infinity in B_s is multiplied with may differ in sign.
  uint4 b_own[kOneT / 8];
  const int one_shift = 31 - __clz(prm.rank >> 3), one_last = (prm.rank >> 3) - 1;   // ranks are powers of two
  auto load_b = [&](const Place& at) {
    const int n = at.c * kRowsOp + threadIdx.x;
#pragma unroll
    for (int i = 0; i < kOneT / 8; i++) {
      const int row = i >> one_shift, slot = row < prm.M ? list.slot[row] : -1;
      b_own[i] = make_uint4(0u, 0u, 0u, 0u);
      if (slot >= 0 && n < prm.N) b_own[i] = load_chained(reinterpret_cast<const uint4*>(prm.b + ((size_t)slot * prm.N + n) * prm.rank) + (i & one_last));
    }
  };
  auto low_of = [&](float (&low)[kOneT / 8]) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kOneT / 8; i++) {
      if (8 * i >= prm.M * prm.rank) continue;
      float4 t0 = make_float4(0.f, 0.f, 0.f, 0.f), t1 = t0;
#pragma unroll 1
      for (int s = 0; s < size; s++) {
        const float4* t = reinterpret_cast<const float4*>(t_rows + s * kOneT + 8 * i);
        const float4 u = t[0], v = t[1];
        t0.x += u.x; t0.y += u.y; t0.z += u.z; t0.w += u.w;
        t1.x += v.x; t1.y += v.y; t1.z += v.z; t1.w += v.w;
      }
      const uint4 w = b_own[i];
      if ((i & one_last) == 0) sum = 0.f;
      sum = fmaf(t0.x, bf16_lo(w.x), sum); sum = fmaf(t0.y, bf16_hi(w.x), sum); sum = fmaf(t0.z, bf16_lo(w.y), sum); sum = fmaf(t0.w, bf16_hi(w.y), sum);
      sum = fmaf(t1.x, bf16_lo(w.z), sum); sum = fmaf(t1.y, bf16_hi(w.z), sum); sum = fmaf(t1.z, bf16_lo(w.w), sum); sum = fmaf(t1.w, bf16_hi(w.w), sum);
#pragma unroll
      for (int r = 0; r < kOneT / 8; r++)
        if (r == i >> one_shift) low[r] = sum;   // the last of a row's chunks stays
    }
  };

  if (warp == 4) {
    const bool el = elect_one();
    if (el) {
      if (!rounds_x) tma_prefetch_desc(&maps.x);
      tma_prefetch_desc(&maps.w);
    }
    if constexpr (kOne) {   // no launch of this call before this one: nothing is read early, but brought into L2
      if (el) {
        int left = kPrefetchSteps;
        for (int tile = first; tile < prm.tiles && left > 0; tile += stride) {
          const Place at = place(tile);
          for (int k = at.k0; k < at.k1 && left > 0; k++, left--)
#pragma unroll
            for (int i = 0; i < 2; i++) tma_prefetch_2d(&maps.w, at.c * kRowsOp + 64 * i, k * 64);
        }
      }
      __syncwarp();
      chain_wait();
    }
    const int w_at = kWide ? kStageRows : 0, x_at = kWide ? 0 : kStageRows;   // the M operand comes first
    auto load_w = [&](const Place& at, int k, int s) {   // W of one step; arms the stage for both operands (out-of-range parts of a box are zero-filled and still counted)
      uint8_t* st = smem + s * SH::kStage + w_at;
      mbar_expect_tx(&bars->full[s], rounds_x ? kStageRows : kStageRows + NC * kStepBytes);
#pragma unroll
      for (int i = 0; i < (kWide ? 4 : 2); i++) tma_load_2d(st + i * 8192, &maps.w, at.c * (kWide ? 256 : kRowsOp) + 64 * i, k * 64, &bars->full[s]);
    };
    auto load_x = [&](const Place& at, int k, int s) { tma_load_2d(smem + s * SH::kStage + x_at, &maps.x, k * 64, at.row0, &bars->full[s]); };
    // W of the first steps ahead of the launch before this one, and x where it may be
    bool waited = false;
    auto wait_once = [&] {
      if (!waited) chain_wait();
      waited = true;
    };
    int g = 0, early = 0;
    if (!prm.x_early && first < prm.tiles) {
      const Place at = place(first);
      int k = at.k0;
      for (; k < min(at.k1, prm.steps) && early < kStages; k++, early++)
        if (el) load_w(at, k, early);
      // and to L2 what there are no stages for (a prefetch returns no data, so it could be early anyway)
      for (int ahead = 0; k < min(at.k1, prm.steps) && ahead < kPrefetchSteps; k++, ahead++)
        if (el)
#pragma unroll
          for (int i = 0; i < (kWide ? 4 : 2); i++) tma_prefetch_2d(&maps.w, at.c * (kWide ? 256 : kRowsOp) + 64 * i, k * 64);
      __syncwarp();
      wait_once();
    }
    for (int tile = first; tile < prm.tiles; tile += stride) {
      const Place at = place(tile);
      for (int k = at.k0; k < at.k1; k++, g++) {
        const int s = g % kStages;
        if (g >= kStages) tile_wait(&bars->empty[s], (g / kStages - 1) & 1, bars, prm.status);
        if (k < prm.steps) {
          if (el) {
            if (g >= early) load_w(at, k, s);
            if (!rounds_x) load_x(at, k, s);
          }
        } else if constexpr (kWide) {
          wait_once();   // t is the launch's before this one
          if (el) {
            const int e = k - prm.steps, half = e / t_steps, r = (e - half * t_steps) * 64;
            uint8_t* st = smem + s * SH::kStage;
            mbar_expect_tx(&bars->full[s], SH::kStage);
            tma_load_2d(st, &maps.t[half], r, at.row0, &bars->full[s]);
            tma_load_2d(st + kStageRows, &maps.b, r, at.slot * prm.N + at.c * 256, &bars->full[s]);
          }
        }
        __syncwarp();
      }
    }
  } else if (warp == 5) {
    const bool el = elect_one();
    const uint32_t idesc = make_idesc_bf16(kRowsOp, NC, !kWide, kWide), idesc_t = make_idesc_bf16(kRowsOp, NC, false, false);
    int g = 0, piece = 0;
    for (int tile = first; tile < prm.tiles; tile += stride, piece++) {
      const Place at = place(tile);
      const uint32_t d = tmem + (piece & 1) * SH::kAcc;
      if (piece >= 2) tile_wait(&bars->acc_empty[piece & 1], ((piece >> 1) - 1) & 1, bars, prm.status);
      tc_fence_after();
      for (int k = at.k0; k < at.k1; k++, g++) {
        const int s = g % kStages;
        tile_wait(&bars->full[s], (g / kStages) & 1, bars, prm.status);
        tc_fence_after();
        if (el) {
          const uint32_t st = smem_u32(smem + s * SH::kStage);
          if (k < prm.steps) {
            const uint64_t dW = make_desc_mnmajor_sw128(st + (kWide ? kStageRows : 0), 8192), dX = make_desc_kmajor_sw128(st + (kWide ? 0 : kStageRows));
#pragma unroll
            for (int kk = 0; kk < 4; kk++) {
              const uint64_t w = dW + ((uint32_t)(kk * 2048) >> 4), x = dX + ((uint32_t)(kk * 32) >> 4);
              umma_ss<1>(d, kWide ? x : w, kWide ? w : x, idesc, k != at.k0 || kk != 0);
              if (rounds_x) umma_ss<1>(d, w, x + ((uint32_t)(NC * kStepBytes) >> 4), idesc, true);   // the rows' second half
            }
          } else if constexpr (kWide) {
            const uint64_t dT = make_desc_kmajor_sw128(st), dB = make_desc_kmajor_sw128(st + kStageRows);
            const int e = k - prm.steps, left = prm.rank - e % t_steps * 64;   // (of rank 8 the second half of the slice is zeros)
            for (int kk = 0; kk < 4 && 16 * kk < left; kk++)
              umma_ss<1>(d, dT + ((uint32_t)(kk * 32) >> 4), dB + ((uint32_t)(kk * 32) >> 4), idesc_t, k != at.k0 || kk != 0);
          }
          umma_commit<1>(&bars->empty[s]);
        }
        __syncwarp();
      }
      if (el) umma_commit<1>(&bars->acc_full[piece & 1]);
      __syncwarp();
    }
  } else if (kOne && warp >= 10) {
    chain_wait();
    if (first < prm.tiles) {
      down_part();
      low_sync();
    }
  } else if (!kWide && warp >= 6) {
    // helpers: few float32 rows as two bf16 halves, and half of t B_s^T
    const int id = threadIdx.x - 192;
    if constexpr (kOne) chain_wait();
    int g = 0;
    for (int tile = first; tile < prm.tiles; tile += stride) {
      const Place at = place(tile);
      if (rounds_x) {   // thread: eight k of a row, four steps' loads on their way together (of rows that do not exist the stages hold anything: no one reads their sums)
        const int row = id >> 3, chunk = id & 7;
        const bool there = row < prm.M;
        for (int k = at.k0; k < at.k1; k += 4) {
          float4 u[4], v[4];
          if (there)
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const int col = (k + i) * 64 + 8 * chunk;
              const bool in = k + i < at.k1 && col < prm.K;   // K is a multiple of 8
              const float4* src = reinterpret_cast<const float4*>(prm.x_f32 + (size_t)row * prm.K + (in ? col : 0));
              u[i] = in ? load_chained(src) : make_float4(0.f, 0.f, 0.f, 0.f);
              v[i] = in ? load_chained(src + 1) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (k + i < at.k1) {
              const int s = g % kStages;
              if (g >= kStages) tile_wait(&bars->empty[s], (g / kStages - 1) & 1, bars, prm.status);
              if (there) {
                uint2 hi[2], lo[2];
                split_halves(u[i], 1.f, hi[0], lo[0]);
                split_halves(v[i], 1.f, hi[1], lo[1]);
                uint8_t* const to = smem + s * SH::kStage + kStageRows + swz128(row, chunk);
                *reinterpret_cast<uint4*>(to) = make_uint4(hi[0].x, hi[0].y, hi[1].x, hi[1].y);
                *reinterpret_cast<uint4*>(to + NC * kStepBytes) = make_uint4(lo[0].x, lo[0].y, lo[1].x, lo[1].y);
                fence_proxy_async();
              }
              __syncwarp();
              if (lane == 0) mbar_arrive(&bars->full[s]);
              g++;
            }
        }
      }
      if constexpr (!kOne) low_half(at, 1);
    }
  } else {
    if constexpr (kWide || kOne) chain_wait();
    int piece = 0, staged = 0;
    for (int tile = first; tile < prm.tiles; tile += stride, piece++) {
      const Place at = place(tile);
      const int buf = piece & 1;
      const uint32_t acc = tmem + ((uint32_t)(warp * 32) << 16) + buf * SH::kAcc;
      const int cols = kWide ? min(256, prm.N - at.c * 256) : prm.M;   // of the N operand that exist
      const int grain = !kWide ? 1 : prm.out_bf16 ? 64 : 32;
      const int q0 = size > 1 ? slice_begin(rank, cols, grain, size) : 0, q1 = size > 1 ? slice_begin(rank + 1, cols, grain, size) : cols;
      const float* const got = reinterpret_cast<const float*>(slices) + threadIdx.x;
      if constexpr (kOne) {
        load_b(at);
        if (tile == first) {
          down_part();
          low_sync();
        }
      } else if constexpr (!kWide) {
        low_half(at, 0);
      }
      tile_wait(&bars->acc_full[buf], (piece >> 1) & 1, bars, prm.status);
      tc_fence_after();
      const bool ok = !bars->abort_flag;
      if (size > 1) {
        if constexpr (kOne) swap_slices<SH>(acc, cols, grain, size, rank, slices, send_parts);
        else swap_slices<SH>(acc, cols, grain, size, rank, slices);
      }
      if constexpr (!kWide) {
        // thread = column; a warp writes 64 or 128 bytes of a row at once
        const int n = at.c * kRowsOp + warp * 32 + lane;
        const bool mine = n < prm.N;
        float low[kOneT / 8] = {};
        if constexpr (kOne) low_of(low);
#pragma unroll 1
        for (int q = q0; q < q1; q += 8) {
          uint32_t v[8];
          tmem_ld_32x32b_x8(acc + q, v);
          const size_t to = (size_t)q * prm.N + n;
          float before[8];
#pragma unroll
          for (int i = 0; i < 8; i++) before[i] = 0.f;
          if (prm.adds)
#pragma unroll
            for (int i = 0; i < 8; i++)
              if (mine && q + i < q1)
                before[i] = prm.out_bf16 ? f32_from_bf16_bits(load_chained(reinterpret_cast<const uint16_t*>(prm.out) + to + (size_t)i * prm.N))
                                         : load_chained(reinterpret_cast<const float*>(prm.out) + to + (size_t)i * prm.N);
          tmem_ld_wait();
          float x[8];
#pragma unroll
          for (int i = 0; i < 8; i++) x[i] = ok ? __uint_as_float(v[i]) : 0.f;
#pragma unroll 1
          for (int s = 0; s < (kOne ? size - 1 : size); s++)   // the others' parts, then the adapter's
#pragma unroll
            for (int i = 0; i < 8; i++)
              if (q + i < q1) x[i] += got[(s * (q1 - q0) + q - q0 + i) * kRowsOp];
          if constexpr (kOne)
#pragma unroll
            for (int r = 0; r < kOneT / 8; r++)
#pragma unroll
              for (int i = 0; i < 8; i++)
                if (q + i == r) x[i] += low[r];
#pragma unroll
          for (int i = 0; i < 8; i++) x[i] += before[i];
          if (prm.out_bf16) {
            uint16_t* const dst = reinterpret_cast<uint16_t*>(prm.out) + to;
#pragma unroll
            for (int i = 0; i < 8; i++) store_if(dst + (size_t)i * prm.N, __bfloat16_as_ushort(__float2bfloat16_rn(x[i])), mine && q + i < q1);
          } else {
            float* const dst = reinterpret_cast<float*>(prm.out) + to;
#pragma unroll
            for (int i = 0; i < 8; i++) store_if(dst + (size_t)i * prm.N, x[i], mine && q + i < q1);
          }
        }
      } else {
        // thread = row: 32 (bf16: 64) columns at a time to a staging tile of the warp, 128-byte swizzle, and out by TMA, which leaves out what lies past the last
        // column; of warps with rows past the request's end straight to the rows
        uint8_t* const tiles = out_tiles + warp * 2 * 32 * kOutRow;
        const int wide = prm.out_bf16 ? 64 : 32, m = warp * 32 + lane;
        const bool whole = warp * 32 + 32 <= at.rows, mine = m < at.rows;
#pragma unroll 1
        for (int q = q0; q < q1; q += wide, staged += whole) {
          uint8_t* const tile_smem = tiles + (staged & 1) * 32 * kOutRow;
          if (whole) {
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");   // the store before the last has read its tile
            __syncwarp();
          }
#pragma unroll 1
          for (int h = 0; h < wide && q + h < q1; h += 16) {
            uint32_t v[16];
            tmem_ld_32x32b_x8(acc + q + h, *reinterpret_cast<uint32_t(*)[8]>(v));
            tmem_ld_32x32b_x8(acc + q + h + 8, *reinterpret_cast<uint32_t(*)[8]>(v + 8));
            tmem_ld_wait();
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = ok ? __uint_as_float(v[i]) : 0.f;
            add_slices(slices, size, q1 - q0, q + h - q0, [&](int i, uint32_t u) { x[i] += __uint_as_float(u); });
            const int col = at.c * 256 + q + h;
            const size_t to = (size_t)(at.row0 + m) * prm.N + col;
            if (prm.adds && mine)
#pragma unroll
              for (int i = 0; i < 2; i++)
                if (col + 8 * i < prm.N) {   // N is a multiple of 8
                  if (prm.out_bf16) {
                    const uint4 a = load_chained(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(prm.out) + to) + i);
                    x[8 * i] += bf16_lo(a.x); x[8 * i + 1] += bf16_hi(a.x); x[8 * i + 2] += bf16_lo(a.y); x[8 * i + 3] += bf16_hi(a.y);
                    x[8 * i + 4] += bf16_lo(a.z); x[8 * i + 5] += bf16_hi(a.z); x[8 * i + 6] += bf16_lo(a.w); x[8 * i + 7] += bf16_hi(a.w);
                  } else {
                    const float4* src = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(prm.out) + to) + 2 * i;
                    const float4 a = load_chained(src), b = load_chained(src + 1);
                    x[8 * i] += a.x; x[8 * i + 1] += a.y; x[8 * i + 2] += a.z; x[8 * i + 3] += a.w;
                    x[8 * i + 4] += b.x; x[8 * i + 5] += b.y; x[8 * i + 6] += b.z; x[8 * i + 7] += b.w;
                  }
                }
            if (prm.out_bf16) {
#pragma unroll
              for (int i = 0; i < 2; i++) {
                const uint4 y = make_uint4(round_bf16x2(x[8 * i], x[8 * i + 1]), round_bf16x2(x[8 * i + 2], x[8 * i + 3]), round_bf16x2(x[8 * i + 4], x[8 * i + 5]),
                                           round_bf16x2(x[8 * i + 6], x[8 * i + 7]));
                if (whole) *reinterpret_cast<uint4*>(tile_smem + swz128(lane, h / 8 + i)) = y;
                else if (mine && col + 8 * i < prm.N) reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(prm.out) + to)[i] = y;
              }
            } else {
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const float4 y = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                if (whole) *reinterpret_cast<float4*>(tile_smem + swz128(lane, h / 4 + i)) = y;
                else if (mine && col + 4 * i < prm.N) reinterpret_cast<float4*>(reinterpret_cast<float*>(prm.out) + to)[i] = y;
              }
            }
          }
          if (whole) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&maps.out, (at.c * 256 + q) * (prm.out_bf16 ? 1 : 2), at.row0 + warp * 32, tile_smem);
              tma_store_commit();
            }
            __syncwarp();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->acc_empty[buf]);
    }
    if constexpr (kWide) {
      if (lane == 0) tma_store_wait_all();
      __syncwarp();
    }
    fence_chained_writes();
  }
  tile_end<SH>(tmem, size);
}

template <int NC, bool kOne, class Rows>
int32_t launch_rows(Pool* p, const LoraMaps& maps, const LoraGemmParams& prm, const Rows& rows) {
  return launch_tiles<LoraShape<NC>, kLoraGemmThreads<NC, kOne>>(p, lora_gemm_kernel<NC, Rows, kOne>, prm.tiles, prm.steps, maps, prm, rows);
}

}  // namespace

int32_t launch_lora_gemm(Pool* p, const relux_matmul_lora_args* a, const uint16_t* x, const int32_t* row_slots, const LoraTiles* tiles, const float* t,
                         const uint16_t* t_hi, const uint16_t* t_lo) {
  LoraGemmParams prm{};
  LoraMaps maps{};
  const int M = a->m, K = a->k, N = a->n;
  const int nc = tiles ? 256 : kNarrowRows;
  prm.M = M;
  prm.N = N;
  prm.rank = a->rank;
  prm.steps = (K + 63) / 64;
  prm.col_tiles = (N + (tiles ? nc : kRowsOp) - 1) / (tiles ? nc : kRowsOp);
  const int64_t count = (int64_t)prm.col_tiles * (tiles ? tiles->n : 1);
  if (count * (prm.steps + 4) >= (int64_t)1 << 31) { set_error("a product of more than 2^31 steps"); return RELUX_ERR_UNSUPPORTED; }
  prm.tiles = (int)count;
  prm.out_bf16 = a->out_dtype == RELUX_DTYPE_BF16;
  prm.adds = a->accumulate != 0;
  prm.x_early = a->x_dtype == RELUX_DTYPE_BF16 || !x;
  prm.x_f32 = x ? nullptr : (const float*)a->x;
  prm.K = K;
  prm.t = t;
  prm.a = (const uint16_t*)a->lora_a;
  prm.x_rows = a->x;
  prm.b = (const uint16_t*)a->lora_b;
  prm.factors = a->factors;
  prm.out = a->out;
  prm.status = p->d_status;
  bool made = (!x || make_tmap_2d(&maps.x, (void*)x, (uint64_t)M, (uint64_t)K, 64, tiles ? kRowsOp : nc)) && make_tmap_2d(&maps.w, (void*)a->w, (uint64_t)K, (uint64_t)N, 64, 64);
  if (tiles)
    made = made && make_tmap_2d(&maps.t[0], (void*)t_hi, (uint64_t)M, (uint64_t)a->rank, 64, kRowsOp) &&
           make_tmap_2d(&maps.t[1], (void*)t_lo, (uint64_t)M, (uint64_t)a->rank, 64, kRowsOp) &&
           make_tmap_2d(&maps.b, (void*)a->lora_b, (uint64_t)a->n_slots * N, (uint64_t)a->rank, 64, 256) &&
           make_tmap_2d(&maps.out, a->out, (uint64_t)M, (uint64_t)N * (prm.out_bf16 ? 1 : 2), kOutRow / 2, 32);
  if (!made) {
    set_error("tensor map for a projection with adapters could not be encoded");
    return RELUX_ERR_CUDA;
  }
  if (tiles) return launch_rows<256, false>(p, maps, prm, *tiles);
  NarrowRows rows;
  std::copy(row_slots, row_slots + M, rows.slot);
  std::fill(rows.slot + M, rows.slot + kNarrowRows, -1);
  return t ? launch_rows<kNarrowRows, false>(p, maps, prm, rows) : launch_rows<kNarrowRows, true>(p, maps, prm, rows);
}

}  // namespace relux
