// The projections' shared parts: how tiles of weights are dealt to the SMs, and the calls of layer_step.cu that other files make.
#pragma once

#include "internal.h"

namespace relux {

constexpr int kMaxWeights = 4;      // weight matrices that share one activation matrix in a launch
constexpr int kGemmTileCols = 128;  // weight columns of a tile

// How a launch's tiles (128 weight columns x one block of rows) are dealt out.  `full` rounds of whole tiles, neighbouring tiles
// side by side: the workers then walk K in step and together read whole weight rows, which DRAM serves faster than 256-byte
// pieces of rows that lie far apart (0.54 GB: 86.8 us so, 90.1 us with every worker somewhere else in K; 0.82 GB: 128.5 against
// 130.8 us).  The tiles that are left are cut along K, `split` equal parts each (also in step), or (split = 0) their K steps,
// laid end to end, are cut into ranges that differ by at most one step.  A PIECE is the part of a tile that one worker does;
// piece j of a tile (in K order) is split j of the result.
// With more rows than a block holds, `beside` blocks have workers of their own that walk the same columns of weights in step, so
// that a column is read once for all of them; the blocks after those are further tiles of the same workers.
struct GemmRanges {
  int32_t workers, steps, full, split;   // of one of the blocks beside each other.  steps: K steps per tile (0: one piece per tile)
  int32_t range, more;                   // split = 0: steps per worker, one more for the first `more` of them
  int32_t rest;                          // tiles that are left after the full rounds
  int32_t beside, row_blocks, block_rows, col_tiles;
  bool in_turns() const { return row_blocks != beside; }
  __host__ __device__ int tile_of(int col, int row) const { return row / block_rows / beside * col_tiles + col; }
  __host__ __device__ int begin(int w) const {   // in steps of the tiles that are left
    if (!split) return w * range + (w < more ? w : more);
    return w < rest * split ? w / split * steps + w % split * steps / split : rest * steps;
  }
  __host__ __device__ int worker_of(int u) const {   // split = 0
    const int big = more * (range + 1);
    return u < big ? (int)((unsigned)u / (unsigned)(range + 1)) : more + (int)((unsigned)(u - big) / (unsigned)range);
  }
  __host__ __device__ int pieces(int tile) const {
    const int t = tile - full * workers;
    if (!steps || t < 0) return 1;
    return split ? split : worker_of((t + 1) * steps - 1) - worker_of(t * steps) + 1;
  }
};
// The pieces of one worker: GemmWalk walk(rg, w); while (walk.next()) ... walk.col, walk.block, steps [k0, k1), split.
// kBlocks: there may be more than one row block.
template <bool kBlocks>
struct GemmWalk {
  const GemmRanges& g;
  int w, n, u, u1, col, block, block0, k0, k1, split;
  __device__ GemmWalk(const GemmRanges& rg, int id)
      : g(rg), w(kBlocks ? id / rg.beside : id), n(0), u(rg.begin(w)), u1(rg.begin(w + 1)), col(0), block(0), block0(kBlocks ? id - w * rg.beside : 0),
        k0(0), k1(0), split(0) {}
  __device__ int total() const { return g.full * g.steps + g.begin(w + 1) - g.begin(w); }
  __device__ bool next() {
    int tile;
    split = 0;
    if (n < g.full) {
      tile = n++ * g.workers + w;
      k0 = 0;
      k1 = g.steps;
    } else {
      if (u >= u1) return false;
      const int t = u / g.steps;
      tile = g.full * g.workers + t;
      k0 = u - t * g.steps;
      u = min(u1, (t + 1) * g.steps);
      k1 = u - t * g.steps;
      split = g.split ? w - t * g.split : w - g.worker_of(t * g.steps);
    }
    col = tile;
    if constexpr (kBlocks) {
      block = block0;
      if (g.row_blocks != g.beside) {
        const int turn = tile / g.col_tiles;
        col = tile - turn * g.col_tiles;
        block += turn * g.beside;
      }
    }
    return true;
  }
};

// Further columns of a projection of up to 128 rows: x A_s^T of every adapter in use, for every row (a row's own are what is read of them).  A tile is 128 / rank adapters, cut into
// `parts` equal parts of K, which are dealt to the workers behind their pieces: cuts that do not depend on which adapters they are.
constexpr int kMaxUsed = 128;
struct AdapterColumns {
  const void* lora_a;        // [n_slots][rank][K]
  int32_t n_slots, rank, n_used, parts;
  float* t;                  // [part][M][n_used * rank]
  int32_t slot[kMaxUsed];
};
struct WeightRef {
  const void* w;
  int n;
};
struct LayerScratch {
  uint16_t* a_bf16;
  float* part;
  size_t part_cap;
  char* rest;
};
// [activations as bf16 (M x max_k) | split partials | caller's buffers (rest_bytes)].  few_pieces: room for eight pieces of the result, or four where that is over 64 MB,
// and not for 64 MB of them.
int32_t layer_scratch(Pool* p, int M, int max_k, int max_n, size_t rest_bytes, LayerScratch* out, bool few_pieces = false);
size_t layer_scratch_bytes(int M, int max_k, int max_n, size_t rest_bytes, bool few_pieces = false);   // what it makes room for
inline size_t pad256(size_t b) { return (b + 255) & ~(size_t)255; }
// n float32 values, a multiple of 8, rounded to bf16 by the reference's rule.
int32_t launch_cast(Pool* p, const float* src, uint16_t* dst, size_t n);
bool gemm_sm100_eligible(int K, const WeightRef* ws, int nw);
// part[piece][M][n_total] = A[M][K] x [W_0 | W_1 | ...]; returns the ranges, which say how many pieces every tile has.  head: nothing of the call is before it.
int32_t launch_skinny_gemm(Pool* p, const uint16_t* a_bf16, int M, int K, const WeightRef* ws, int nw, float* part, size_t part_cap_bytes,
                           GemmRanges* ranges, TimeStamp time = TimeStamp{nullptr, nullptr}, const AdapterColumns* adapters = nullptr, bool head = false);

}  // namespace relux
