// Attention of more than 32 query rows per kv head, on the 5th-generation tensor cores (tcgen05 + TMEM): drafted trees over the bf16 and the 8-bit
// grouped-query cache, and prompts (or long verifies) over the 8-bit one.
//
// o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - max),  where query token i sees every cached row and, of the drafted ones, itself
// and its ancestors; of a prompt, every row up to its own.  The g query heads of a kv head times the S nodes are R rows that read the same keys: R * 4 * 128
// operations for the 512 (264) bytes of a token and kv head, so the cache's bytes bound trees of up to some 200 rows (100 on the 8-bit cache) and the tensor
// cores and the softmax larger ones.  Measured, join of the parts included, on a card that was idle before (1965 MHz): 64 x 8192 tokens, 64 rows 337 us on bf16 (6.4
// TB/s), 396 on 8 bits (2.8 TB/s); 8 x 32768 tokens, 512 rows 546 us (1.0 PFLOP/s), 667 on 8 bits.  After a second of such calls, under the power cap (990 W, 1360
// to 1480 MHz on bf16, 1770 on 8 bits): 385, 440, 645 and 750.  Times further down are of this kernel alone, from idle.
//
// A STREAM is the tiles of 128 keys that up to 256 of a kv head's rows (one or two blocks of 128, M of both contractions) see.  All streams of the
// call, each its tiles and kFixUnits units of fixed cost, laid end to end, are cut into a range per SM (make_ranges); a PIECE is the part of a stream inside a
// range.
// A piece that is a whole stream writes its output; others leave float32 partials that merge_tree_kernel joins.
//
// Roles of a CTA:
//   producer   a tile's K and V by TMA, 32 KB each, into a ring; on the 8-bit cache page by page, 8 KB each, and the scales, into rings of their own
//   scales     (8-bit cache) a warp: the keys' scales of a tile to where the softmax reads them, the values' over their unit to the converters
//   converters (8-bit cache, four warps for K, four for V) codes -> binary16 operands in the ring's swizzled layout.  K as whole numbers: a row's scale multiplies its column of
//              scores, in float32.  V times its scale over a power of two that all of the piece's rows share so far (11 bits, as P has then; 2^21 between
//              the largest row and one that may not be exact to 11 bits); where a row comes that is too large for it, the power grows and O is rescaled.
//   MMA        step k = (tile, block): S = Q K^T (S buffer k & 1), O[block] += P V with P read from tensor memory over the scores it came from
//   softmax    eight warps of 16 rows of a block each, four lanes to a row: scores from TMEM, running max (updated lazily), P back to TMEM.  Up to
//              64 rows, four warps take the even steps and four the odd ones, each with an O of its own,
//              which meet at the piece's end.
// What bounds it.  bf16, up to 64 rows: HBM.  More rows: the softmax warps, for whom a step of 128 rows takes 1550 clocks (2570 beside converters), most of it
// the latency of their instructions (512 of exponentials a warp), against 1020 of MMAs.  8 bits, up to 64 rows: converters and softmax share issue slots and
// shared memory, through which a tile's operands, codes and queries come to 1760 clocks, and each alone adds a fourth to what the rest takes: 408 us of 64 x 8192
// tokens, a build before the last, were 300 without the converters' work, 332 without the softmax's, 234 without either.
// Order of issue: QK(k + 1), PV(k): the tensor pipe executes in issue order, so QK(k + 2) finds its S buffer read.
// A product with P = 0 does not hide an infinity or a NaN among the values: those of drafted rows and of what lies behind are set to zero in the tile, and
// the rows that see one become NaN at the end.  (8-bit rows have them in their scale alone; a code is always a number.)
// Every wait is bounded (RELUX_ERR_TIMEOUT, an abort flag that ends the other waits; all warps reach the end and TMEM is freed).
#include <algorithm>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <new>

#include "common.cuh"
#include "gqa_int8_parts.cuh"
#include "internal.h"
#include "softmax_parts.cuh"
#include "umma.cuh"

namespace relux {

namespace {

constexpr int kTile = 128, kD = kGqaD, kPage = kGqaPageTok;
constexpr int kHalf = 16384;                   // [128 rows][64 16-bit columns], 128-byte swizzle
constexpr int kSlot = 2 * kHalf;               // K or V of a tile, or 128 query rows
constexpr int kRawSlot = kPage * kD;           // codes of K or V of a page
constexpr int kTilesAhead = 4;                 // (8-bit cache) of a tile in L2 before its loads
// Tiles: what a piece costs beyond its own (queries in, results out).  With 1, 2 and 4: 100 x 700 tokens, 64 rows, 8 bits 101, 99.5, 96 us; 4 x 500 tokens behind
// 1500 122, 123, 119; 40 x 1500, 64 rows, bf16 53.5, 51.6, 51.2; long ones the same.
constexpr int kFixUnits = 4;
constexpr int kSoftmaxWarps = 8, kConvWarps = 4;   // of K, and of V
constexpr int kWarpScale = kSoftmaxWarps + 2 * kConvWarps + 2;
constexpr uint32_t kTmemCols = 512, kTmemO = 256;
constexpr float kRescaleThreshold = 8.0f;      // log2: P reaches 2^8 before the running max follows
// (8-bit cache) log2: what P and its sum are larger by.  Binary16 has 11 bits down to 2^-14, and P reaches 2^(8 + 7): probabilities keep 11 bits down to 2^-21
// of the row's largest, and below are off by at most 2^-32 of it.
constexpr float kPUp = 7.0f;
constexpr int kInlineSmall = 32, kInlineLarge = 256;
constexpr int kMaxWorkers = 160;

// A group of rows of a sequence: rows [row0, row0 + rows_rb) of every kv head.
struct TreeSeq {
  int32_t seq, i;              // sequence of the pool, and of the call
  int32_t len0, end;           // tokens that all of its rows see, and that any does; a tree's nodes are those from len0 on
  int32_t row0;
  int32_t unit0;               // first unit, one kv head counted
};
struct TreeCommon {
  const TreeSeq* seqs;         // device copy, or nullptr: inline
  const int8_t* parents;       // of a device copy
  int32_t one_tree, tree;      // tree = 0: query token s sees tokens below row_end + s (causal), or below row_end
  int32_t causal;
  const int32_t* table;
  int32_t table_stride, num_pages, n_seqs, Hkv, H, g, S, R;
  uint32_t over_g;             // 2^31 / g, rounded up: a row below 2^31 / g over g is a product (a division by g a row was half of a piece's fixed cost)
  int32_t n_rb, rows_rb;       // groups of a sequence, rows of each (the last may have fewer)
  int32_t krow0, vrow0;
  const float* scales;         // 8-bit cache: of the layer
  const uint8_t* codes;        // and the pool's rows
  float scale_log2;
  const uint16_t* q;           // bf16
  int32_t out_bf16;
  void* out;
  float* part_o;               // [2 * workers][rows_rb][128]
  float* part_ml;              // [2 * workers][rows_rb][2]
  int32_t* status;
  TimeStamp time;
};
template <int N>
struct TreeParams {
  TreeCommon c;
  TreeSeq seqs[N + 1];
  alignas(2) int8_t parents[N][kTreeNodes];
  int32_t cuts[kMaxWorkers + 1];   // ranges: units cuts[w] to cuts[w + 1]
};

__device__ __forceinline__ int token_of(const TreeCommon& c, int row) { return (int)__umulhi(2u * (uint32_t)row, c.over_g); }

// The streams as every role walks them: pieces of this range, in order.  Sequence by sequence, kv head by kv head, group by group: the groups of a kv head
// read the same tiles.
struct Piece {
  int32_t e, kvh, us, tb, te, tiles;   // group (of all), kv head, first unit of the stream, tiles [tb, te) of `tiles`
};
template <int N>
struct Streams {
  const TreeParams<N>& prm;
  int32_t u_begin, u_end;
  __device__ __forceinline__ Streams(const TreeParams<N>& p, int worker) : prm(p), u_begin(p.cuts[worker]), u_end(p.cuts[worker + 1]) {}
  __device__ __forceinline__ int unit0(int e) const { return prm.c.seqs ? prm.c.seqs[e].unit0 : prm.seqs[e].unit0; }
  __device__ __forceinline__ TreeSeq seq(int e) const { return prm.c.seqs ? prm.c.seqs[e] : prm.seqs[e]; }
  __device__ __forceinline__ void cut(Piece& p) const {
    if (p.us >= u_end) return;
    p.tiles = unit0(p.e + 1) - unit0(p.e) - kFixUnits;
    p.te = min(p.tiles, u_end - p.us);
  }
  // The stream that unit u belongs to, from its tile at u on.
  __device__ __forceinline__ Piece at(int u) const {
    const int n_rb = prm.c.n_rb, Hkv = prm.c.Hkv;
    int lo = 0, hi = prm.c.n_seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (unit0(mid * n_rb) * Hkv <= u) lo = mid;
      else hi = mid;
    }
    const int e0 = lo * n_rb, n0 = unit0(e0), head = unit0(e0 + n_rb) - n0;
    Piece p;
    p.kvh = (u - n0 * Hkv) / head;
    const int base = n0 * Hkv + p.kvh * head;
    lo = e0;
    hi = e0 + n_rb;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (base + unit0(mid) - n0 <= u) lo = mid;
      else hi = mid;
    }
    p.e = lo;
    p.us = base + unit0(lo) - n0;
    p.tb = u - p.us;
    p.te = p.tiles = 0;
    cut(p);
    return p;
  }
  __device__ __forceinline__ bool valid(const Piece& p) const { return p.us < u_end; }
  __device__ __forceinline__ Piece next(const Piece& q) const {
    Piece p = q;
    p.us += p.tiles + kFixUnits;
    p.tb = 0;
    if ((++p.e) % prm.c.n_rb == 0) {
      if (++p.kvh < prm.c.Hkv) p.e -= prm.c.n_rb;
      else p.kvh = 0;
    }
    cut(p);
    return p;
  }
  __device__ __forceinline__ Piece first() const {
    const Piece p = at(u_begin);
    return p.tb < p.tiles ? p : next(p);   // a range may begin in the fixed-cost units of a stream
  }
};

struct Bars {
  uint64_t full[6], empty[6], s_full[2], p_full[2], q_full, pv, fin, drain;
  uint32_t tmem_base;
  volatile int32_t abort_flag;
  int32_t first[4];            // piece of this range: its e, kvh, us, tb
  // (bf16) Of a piece: nodes with an infinity or a NaN among their values.  The MMA warp writes it once a piece, before `fin`; of the next piece it does so
  // behind that one's q_full, at which every softmax warp arrives when it has read this.
  uint64_t bad_nodes;
  float v_unit[4];             // (8-bit cache) of a tile: what O is to be multiplied by
  union {
    uint64_t see[256];         // what a row sees: of the nodes (a bit each), or how many tokens from len0 on
    struct {
      uint64_t of_two[64];     // (two: up to 64 rows)
      float halves[2][3][64];  // a row's max, sum and unit of O, of either half of the warps
    };
  };
  alignas(16) uint32_t v_scale[4][kTile];   // (8-bit cache) of a tile's values, over their unit, binary16 twice
  alignas(16) float k_scale[4][kTile];   // (8-bit cache) of a tile's keys
  // (8-bit cache) Of piece n, in place n & 7: nodes with an infinity or a NaN among their values, and whether a cached row has one.  The warp of the scales
  // writes a piece's once, before it hands over the piece's last tile, and nobody clears them.  It may be four tiles ahead of the softmax warps, of pieces of
  // one tile four pieces, one of which has not been read out.  Place n & 7 is written again for piece n + 8: the last tile of that is handed over only when
  // the softmax warps have left a tile of piece n + 4 or a later one, behind their reading of piece n's flags.
  struct {
    uint64_t nodes;
    uint32_t all;
  } bad[8];
  uint64_t raw_full[9], raw_empty[9], scale_full[4], scale_empty[4], info[4], info_empty[4];
  // Without an 8-bit cache there is no room for these from v_scale on.
};

template <bool kI8, int kNB>
struct Plan {
  // Rings.  bf16: of 32 KB slots, K and V of a tile in turn.  8-bit cache: of operands, two slots of 32 KB for K and three of a page, 16 KB, for V; of codes,
  // slots of 8 KB, K and V apart: what is being converted is no prefetch, and HBM wants some 50 KB an SM on their way.  (K and V must have slots of their own: a
  // warp that waits for some of a slot's phases only cannot tell them apart.)
  static constexpr int kSlots = kI8 ? 2 : kNB == 2 ? 5 : 6, kSlotsV = kI8 ? 3 : 0;
  static constexpr int kRawK = kI8 ? (kNB == 2 ? 3 : 4) : 0, kRawV = kI8 ? (kNB == 2 ? 2 : 5) : 0, kRaw = kRawK + kRawV;
  static constexpr int kScaleSlots = kI8 ? 4 : 0;                 // scales as they come, of a tile, 1 KB
  static constexpr int kQ = 0;
  static constexpr int kRing = kNB * kSlot;
  static constexpr int kRingV = kRing + kSlots * kSlot;
  static constexpr int kRawAt = kRingV + kSlotsV * kHalf;
  static constexpr int kScaleAt = kRawAt + kRaw * kRawSlot;
  static constexpr int kBars = kScaleAt + kScaleSlots * 1024;
  static constexpr int kTotal = kBars + (int)(kI8 ? sizeof(Bars) : kNB == 1 ? offsetof(Bars, v_scale) : offsetof(Bars, see) + sizeof(Bars::see));
  static_assert(kTotal <= 232448, "more shared memory than a CTA may use");
  static constexpr int kWarpLoad = kSoftmaxWarps + (kI8 ? 2 * kConvWarps : 0), kWarpMma = kWarpLoad + 1;
  // Four more warps where registers are dealt out anew, of the 96 of the launch, which warps do by fours.  Two blocks: with 152, 64 and 48 the warp that issues the
  // MMAs kept a pointer in local memory, and 8 x 32768 tokens, 64 nodes, 64 heads took 934 us where it was 770 with these.  One block: 64 x 8192 tokens of 64 rows 392
  // us with 144, 64 and 64, 397 with 144, 72 and 48, 384 with 128, 80 and 64, 378 with these.
  static constexpr int kThreads = 32 * (kI8 ? kWarpLoad + 4 : kWarpMma + 1);
  static constexpr int kRegsSoftmax = kNB == 1 ? 136 : 144, kRegsConv = kNB == 1 ? 72 : 64, kRegsOther = 64;
  static_assert(!kI8 || 256 * kRegsSoftmax + 256 * kRegsConv + 128 * kRegsOther <= 640 * 96, "more registers than the block is launched with");
};
// The wait that gives up raises the flag, which ends all others; the kernel's end reports it.  Short, and not a function of its own: a call takes registers that
// a role may have given back, and the roles of a block share one instruction cache.  (With the report and a pause in every wait, and all loops of the
// converters unrolled, the 8-bit kernel waited 5.3 cycles for an instruction per one issued, now 0.6 to 1.4; 16 x 8192 tokens, 64 rows, took 149 us, now 113.)
__device__ __forceinline__ void wait_bar(uint64_t* bar, uint32_t parity, Bars* b) {
  for (uint32_t i = 0; !mbar_try_wait(bar, parity); i++)
    if (i >= kSpinLimit || b->abort_flag) {
      b->abort_flag = 1;
      break;
    }
}

// Registers from or to the block's pool, by all warps of a warpgroup.
template <int kRegs, bool kOn>
__device__ __forceinline__ void regs_up() {
  if constexpr (kOn) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs, bool kOn>
__device__ __forceinline__ void regs_down() {
  if constexpr (kOn) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// Instruction descriptor of binary16 operands: make_idesc_bf16 with formats 0.
constexpr uint32_t idesc_of(bool f16, bool b_mn_major) { return make_idesc_bf16(128, 128, false, b_mn_major) & (f16 ? ~((7u << 7) | (7u << 10)) : ~0u); }

template <bool kI8>
__device__ __forceinline__ uint32_t pack_p(float lo, float hi) {
  if constexpr (kI8) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return round_bf16x2(lo, hi);
  }
}
// exp2(score * factor - max) of a lane's 2 x 32 scores (tmem_ld_16x256b_x16), packed in the order of tmem_st_16x128b_x16; row sums are added to ps2.
// (All of them on the special-function unit: a fourth on the FMA pipe, by a polynomial, changed nothing with bf16 rows, and with converters beside it
// 8 x 32768 tokens, 64 nodes, 64 heads took 721 us for 658.)
template <bool kI8>
__device__ __forceinline__ void exp_scores(const uint32_t (&sv)[64], const uint64_t (&factor2)[2], const uint64_t (&neg_m2)[2], uint32_t (&pw)[32], uint64_t (&ps2)[2]) {
#pragma unroll
  for (int i = 0; i < 32; i++) {   // pair i: row i & 1
    const uint64_t x2 = fma2(pack2(__uint_as_float(sv[2 * i]), __uint_as_float(sv[2 * i + 1])), factor2[i & 1], neg_m2[i & 1]);
    float p0, p1;
    unpack2(x2, p0, p1);
    p0 = ex2_approx(p0);
    p1 = ex2_approx(p1);
    ps2[i & 1] = add2(ps2[i & 1], pack2(p0, p1));
    pw[i] = pack_p<kI8>(p0, p1);
  }
}

template <bool kI8, int kNB, int N>
__global__ void __launch_bounds__(Plan<kI8, kNB>::kThreads, 1)
    tree_sm100_kernel(const __grid_constant__ CUtensorMap tmap, const __grid_constant__ TreeParams<N> prm) {
  using PL = Plan<kI8, kNB>;
  const TreeCommon& c = prm.c;
  extern __shared__ __align__(1024) uint8_t smem[];
  Bars* bars = reinterpret_cast<Bars*>(smem + PL::kBars);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool two = kNB == 1 && c.rows_rb <= 64;   // two halves of the softmax warps on steps in turn
  if ((smem_u32(smem) & 1023u) != 0) {            // the swizzled layouts need it
    chain_wait();
    if (threadIdx.x == 0) set_status(c.status, RELUX_ERR_UNSUPPORTED);
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < 6; s++) {
      mbar_init(&bars->full[s], kI8 ? kConvWarps : 1);
      mbar_init(&bars->empty[s], 1);
    }
    if constexpr (kI8) {
      for (int s = 0; s < 9; s++) {
        mbar_init(&bars->raw_full[s], 1);
        mbar_init(&bars->raw_empty[s], kConvWarps);
      }
      for (int s = 0; s < 4; s++) {
        mbar_init(&bars->scale_full[s], 1);
        mbar_init(&bars->scale_empty[s], 1);
        mbar_init(&bars->info[s], 1);
        mbar_init(&bars->info_empty[s], (two ? kSoftmaxWarps / 2 : kSoftmaxWarps) + kConvWarps);
      }
    }
    for (int s = 0; s < 2; s++) {
      mbar_init(&bars->s_full[s], 1);
      mbar_init(&bars->p_full[s], two ? kSoftmaxWarps / 2 : kSoftmaxWarps);
    }
    mbar_init(&bars->q_full, kSoftmaxWarps);
    mbar_init(&bars->pv, 1);
    mbar_init(&bars->fin, 2);
    mbar_init(&bars->drain, 1);
    bars->abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap);
  }
  const Streams<N> streams(prm, blockIdx.x);
  // (One block) the first piece, of every role, is searched for by one thread, before the wait for the launch ahead: the search in every role was a good
  // part of the roles' code, which share one instruction cache (64 x 8192 tokens, 64 rows, 8 bits: 424 us, 390 so; 100 x 700 97 and 94).  With two blocks the steps
  // come out of the compiler slower for it, whatever its reason: 8 x 32768 tokens of 512 rows 648 us and 807.
  if (kNB == 1 && threadIdx.x == 32) {
    if (c.seqs) chain_wait();   // the list is a copy that was queued just before this launch
    const Piece p = streams.first();
    bars->first[0] = p.e;
    bars->first[1] = p.kvh;
    bars->first[2] = p.us;
    bars->first[3] = p.tb;
  }
  if (warp == 0) {
    tmem_alloc<1>(&bars->tmem_base, kTmemCols);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  chain_release();
  chain_wait();
  if (threadIdx.x == 0) stamp_begin(c.time);
  auto first_piece = [&]() -> Piece {
    if constexpr (kNB == 2) return streams.first();
    Piece p{bars->first[0], bars->first[1], bars->first[2], bars->first[3], 0, 0};
    streams.cut(p);
    return p;
  };
  auto rows_of = [&](const TreeSeq& sq) -> int { return min(c.rows_rb, c.R - sq.row0); };
  auto blocks_of = [&](const TreeSeq& sq) -> int { return kNB == 1 ? 1 : (rows_of(sq) + 127) / 128; };

  if (warp == PL::kWarpLoad) {
    regs_down<PL::kRegsOther, kI8>();
    // =============================== producer ===============================
    const bool el = elect_one();
    int h = 0;   // half tiles so far: K of tile n is 2 n, V 2 n + 1
    for (Piece p = first_piece(); streams.valid(p); p = streams.next(p)) {
      const TreeSeq sq = streams.seq(p.e);
      const int kvh = p.kvh;
      const int last_slot = max(0, (sq.end + kPage - 1) / kPage - 1);   // a tile's second page may lie past the rows: nobody sees those keys
      const int32_t* row = c.table + (size_t)sq.seq * c.table_stride;
      // page ids of sixteen tiles, a page a lane, and of the next sixteen
      auto window = [&](int t) -> int32_t {
        int32_t pg = __ldg(row + min(2 * t + lane, last_slot));
        if (pg < 0 || pg >= c.num_pages) {   // reported, and replaced by page 0 so that no load leaves the pool
          set_status(c.status, RELUX_ERR_BAD_PAGE);
          pg = 0;
        }
        return pg;
      };
      int32_t ids = 0, ids2 = window(p.tb);
      for (int t = p.tb; t < p.te; t++) {
        const int j = (t - p.tb) & 15;
        if (j == 0) {
          ids = ids2;
          ids2 = window(t + 16);
        }
        int32_t pg[2];
#pragma unroll
        for (int k = 0; k < 2; k++) pg[k] = __shfl_sync(0xffffffffu, ids, 2 * j + k);
        if constexpr (kI8) {
          // The tile kTilesAhead on is asked for now, by six lanes: K, V and scales of its two pages.
          const int a = 2 * (j + kTilesAhead) + (lane & 1);
          const int32_t near = __shfl_sync(0xffffffffu, ids, a & 31), far = __shfl_sync(0xffffffffu, ids2, a & 31), pa = a < 32 ? near : far;
          if (t + kTilesAhead < p.te && lane < 6) {
            const size_t head = (size_t)pa * c.Hkv + kvh;
            if (lane < 2) prefetch_l2(c.scales + head * (2 * kPage), kInt8ScaleBytes);
            else prefetch_l2(c.codes + ((size_t)(lane < 4 ? c.krow0 : c.vrow0) + head * kPage) * kD, kRawSlot);
          }
          __syncwarp();
        }
#pragma unroll
        for (int kv = 0; kv < 2; kv++, h++) {
          const int32_t row0 = kv ? c.vrow0 : c.krow0;
          if constexpr (kI8) {
            if (kv == 0) {   // the scales of both, [page][K, V][64]
              const int st = (h >> 1) & 3, use = h >> 3;
              if (use > 0) wait_bar(&bars->scale_empty[st], (use - 1) & 1, bars);
              if (el) {
                mbar_expect_tx(&bars->scale_full[st], 2 * kInt8ScaleBytes);
                for (int k = 0; k < 2; k++)
                  bulk_load(smem + PL::kScaleAt + st * 1024 + k * kInt8ScaleBytes, c.scales + ((size_t)pg[k] * c.Hkv + kvh) * (2 * kPage), kInt8ScaleBytes,
                            &bars->scale_full[st]);
              }
              __syncwarp();
            }
#pragma unroll
            for (int k = 0; k < 2; k++) {
              const int at = 2 * (h >> 1) + k;   // page of its kind
              const int st = kv ? PL::kRawK + at % PL::kRawV : at % PL::kRawK, use = kv ? at / PL::kRawV : at / PL::kRawK;
              if (use > 0) wait_bar(&bars->raw_empty[st], (use - 1) & 1, bars);
              if (el) {
                mbar_expect_tx(&bars->raw_full[st], kRawSlot);
                tma_load_2d(smem + PL::kRawAt + st * kRawSlot, &tmap, 0, row0 + (pg[k] * c.Hkv + kvh) * kPage, &bars->raw_full[st]);
              }
              __syncwarp();
            }
          } else {
            const int st = h % PL::kSlots, use = h / PL::kSlots;
            if (use > 0) wait_bar(&bars->empty[st], (use - 1) & 1, bars);
            if (el) {
              uint8_t* dst = smem + PL::kRing + st * kSlot;
              mbar_expect_tx(&bars->full[st], kSlot);
              for (int k = 0; k < 2; k++) {
                const int32_t y = row0 + (pg[k] * c.Hkv + kvh) * kPage;
                tma_load_2d(dst + k * 8192, &tmap, 0, y, &bars->full[st]);
                tma_load_2d(dst + kHalf + k * 8192, &tmap, 64, y, &bars->full[st]);
              }
            }
          }
          __syncwarp();
        }
      }
    }
  } else if (warp == PL::kWarpMma) {
    regs_down<PL::kRegsOther, kI8>();
    // =============================== MMA issuer ===============================
    const bool el = elect_one();
    constexpr uint32_t idesc_qk = idesc_of(kI8, false), idesc_pv = idesc_of(kI8, true);
    const uint64_t dQ = make_desc_kmajor_sw128(smem_u32(smem + PL::kQ));
    int k = 0, tt = 0, n = 0;   // steps, tiles, pieces so far
    for (Piece p = first_piece(); streams.valid(p); p = streams.next(p), n++) {
      const TreeSeq sq = streams.seq(p.e);
      const int nb = blocks_of(sq), tiles = p.te - p.tb;
      uint64_t bad_nodes = 0;                 // (bf16) this lane's of the piece
      wait_bar(&bars->q_full, n & 1, bars);   // the queries are there, and O and the flags of the piece before have been read
      auto issue_qk = [&](int t, int b, int step) {
        const int h = kI8 ? tt + t : 2 * (tt + t), st = h % PL::kSlots;
        if (b == 0) wait_bar(&bars->full[st], (h / PL::kSlots) & 1, bars);
        tc_fence_after();
        if (el) {
          const uint64_t dK = make_desc_kmajor_sw128(smem_u32(smem + PL::kRing + st * kSlot));
          const uint64_t dQb = dQ + ((uint32_t)(b * kSlot) >> 4);
#pragma unroll
          for (int ks = 0; ks < 8; ks++) {
            const uint32_t off = (uint32_t)((ks >> 2) * kHalf + (ks & 3) * 32) >> 4;
            umma_ss<1>(tmem + (step & 1) * 128, dQb + off, dK + off, idesc_qk, ks != 0);
          }
          if (b == nb - 1) umma_commit<1>(&bars->empty[st]);
          umma_commit<1>(&bars->s_full[step & 1]);
        }
        __syncwarp();
      };
      auto issue_pv = [&](int t, int b, int step) {
        const int o = two ? step & 1 : b;
        const bool more = t > (two ? 1 : 0);   // O holds something already
        if constexpr (kI8) {   // V page by page
          wait_bar(&bars->p_full[step & 1], (step >> 1) & 1, bars);
#pragma unroll 1
          for (int k = 0; k < 2; k++) {
            const int at = 2 * (tt + t) + k, st = at % PL::kSlotsV;
            if (b == 0) wait_bar(&bars->full[PL::kSlots + st], (at / PL::kSlotsV) & 1, bars);
            tc_fence_after();   // P, and a rescaled O
            if (el) {
              const uint64_t dV = make_desc_mnmajor_sw128(smem_u32(smem + PL::kRingV + st * kHalf), kHalf / 2);
#pragma unroll
              for (int ks = 0; ks < 4; ks++)
                umma_ts<1>(tmem + kTmemO + o * 128, tmem + (step & 1) * 128 + k * 32 + ks * 8, dV + ((uint32_t)(ks * 2048) >> 4), idesc_pv, more || (k | ks) != 0);
              if (b == nb - 1) umma_commit<1>(&bars->empty[PL::kSlots + st]);
              if (k == 1) umma_commit<1>(&bars->pv);
            }
            __syncwarp();
          }
        } else {
          const int h = 2 * (tt + t) + 1, st = h % PL::kSlots;
          if (b == 0) {
            wait_bar(&bars->full[st], (h / PL::kSlots) & 1, bars);
            {   // infinities and NaN among drafted values, and behind them
              const int from = sq.len0 - (p.tb + t) * kTile;   // first drafted row of the tile
              if (from < kTile) {
                uint8_t* v = smem + PL::kRing + st * kSlot;
                bool any = false;
                auto at = [&](int r) { return reinterpret_cast<uint4*>(v + ((lane >> 3) & 1) * kHalf + swz128(r, lane & 7)); };
                for (int r0 = max(from, 0) + (lane >> 4); r0 < kTile; r0 += 16) {   // 16 lanes a row, eight of them on their way
                  uint32_t bad = 0;
#pragma unroll
                  for (int q = 0; q < 8; q++)
                    if (r0 + 2 * q < kTile) {
                      const uint4 w = *at(r0 + 2 * q);
                      if (bf16x2_not_finite(w.x) | bf16x2_not_finite(w.y) | bf16x2_not_finite(w.z) | bf16x2_not_finite(w.w)) bad |= 1u << q;
                    }
                  any |= bad != 0;
                  for (; bad; bad &= bad - 1) {
                    const int r = r0 + 2 * (__ffs(bad) - 1);
                    const uint4 w = *at(r);
                    *at(r) = make_uint4(bf16x2_finite(w.x), bf16x2_finite(w.y), bf16x2_finite(w.z), bf16x2_finite(w.w));
                    if (r - from < kTreeNodes) bad_nodes |= 1ull << (r - from);
                  }
                }
                if (any) fence_proxy_async();
                __syncwarp();
              }
            }
          }
          wait_bar(&bars->p_full[step & 1], (step >> 1) & 1, bars);
          tc_fence_after();   // P, and a rescaled O
          if (el) {
            const uint64_t dV = make_desc_mnmajor_sw128(smem_u32(smem + PL::kRing + st * kSlot), kHalf);
#pragma unroll
            for (int ks = 0; ks < 8; ks++)
              umma_ts<1>(tmem + kTmemO + o * 128, tmem + (step & 1) * 128 + ks * 8, dV + ((uint32_t)(ks * 2048) >> 4), idesc_pv, more || ks != 0);
            if (b == nb - 1) umma_commit<1>(&bars->empty[st]);
            umma_commit<1>(&bars->pv);
          }
          __syncwarp();
        }
      };
      const int steps = tiles * nb;
#pragma unroll 1
      for (int s = -1; s < steps; s++) {   // one place for each, for the sake of the registers
        if (s + 1 < steps) issue_qk(nb == 2 ? (s + 1) >> 1 : s + 1, nb == 2 ? (s + 1) & 1 : 0, k + s + 1);
        if (s >= 0) issue_pv(nb == 2 ? s >> 1 : s, nb == 2 ? s & 1 : 0, k + s);
      }
      k += steps;
      tt += tiles;
      if constexpr (!kI8) {
        const uint32_t lo = __reduce_or_sync(0xffffffffu, (uint32_t)bad_nodes), hi = __reduce_or_sync(0xffffffffu, (uint32_t)(bad_nodes >> 32));
        if (lane == 0) bars->bad_nodes = (uint64_t)hi << 32 | lo;
      }
      if (el) umma_commit<1>(&bars->fin);         // the piece's products are complete
      if (lane == 0) mbar_arrive(&bars->fin);     // and what this warp, or the converters before they handed over the values, wrote beside them
      __syncwarp();
    }
    // nothing may be freed while an MMA is in flight: the read-out's waits say so, unless one gave up
    if (el) umma_commit<1>(&bars->drain);
    __syncwarp();
    mbar_wait(&bars->drain, 0);
  } else if (warp < kSoftmaxWarps) {
    // =============================== softmax ===============================
    // Warp w reads TMEM lanes 32 (w & 3) .. +31 (the hardware's rule), of which warps w and w + 4 take 16 each: rows 16 w .. 16 w + 15 of a block.
    // Few rows then keep all four schedulers busy.  (two: both take the same 16.)
    // A lane works on two rows of a block, row_in and row_in + 8.  With two blocks their states change places after every step, so that the code is there once.
    regs_up<PL::kRegsSoftmax, kI8>();
    const int set = two ? warp >> 2 : 0, row_warp = two ? warp & 3 : warp;
    const int r16 = (warp & 3) * 32 + (two ? 0 : (warp >> 2) * 16), row_in = 16 * row_warp + (lane >> 2);
    const uint32_t lane_addr = (uint32_t)r16 << 16;
    int k0 = 0, tt0 = 0, n = 0;   // steps, tiles and pieces before this one
    for (Piece p = first_piece(); streams.valid(p); p = streams.next(p), n++) {
      const TreeSeq sq = streams.seq(p.e);
      const int nb = blocks_of(sq), rows = rows_of(sq), tiles = p.te - p.tb;
      struct State {
        float m[2], l[2], f[2];   // running max, sum, what a score is multiplied by
      } st, other;
      auto next_block = [&] {
        if (kNB == 2 && nb == 2) {
          const State t = st;
          st = other;
          other = t;
        }
      };
      // ---- queries in: copies straight to the matrix operand's place ----
      const int i0 = 4 * set;
#pragma unroll 4
      for (int i = i0; i < (two ? i0 + 4 : 8 * nb); i++) {   // 16 lanes a row; two: half of the rows each
        const int b = kNB == 2 ? i >> 3 : 0, j = (2 * i + (lane >> 4)) & 15, row = 128 * b + 16 * row_warp + j, ch = lane & 15;
        const bool there = row < rows;
        const int s = token_of(c, sq.row0 + row), hq = sq.row0 + row - s * c.g;
        const uint16_t* src = c.q + (there ? (((size_t)sq.i * c.S + s) * c.H + (size_t)p.kvh * c.g + hq) * kD + ch * 8 : 0);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem + PL::kQ + b * kSlot + (ch >> 3) * kHalf + swz128(r16 + j, ch & 7))),
                     "l"(__cvta_generic_to_global(src)), "r"(there ? 16 : 0)
                     : "memory");
      }
#pragma unroll
      for (int hf = 0; hf < 2; hf++) {
        st.m[hf] = -INFINITY;
        st.l[hf] = 0.f;
        st.f[hf] = c.scale_log2;
      }
      other = st;
      asm volatile("cp.async.wait_all;" ::: "memory");
      if constexpr (kI8) {   // in place to binary16, by a power of two a row
#pragma unroll 1
        for (int b = 0; b < nb; b++, next_block())
#pragma unroll 2
          for (int i = i0; i < (two ? i0 + 4 : 8); i++) {
            const int j = 2 * i + (lane >> 4), ch = lane & 15;
            uint4* at = reinterpret_cast<uint4*>(smem + PL::kQ + b * kSlot + (ch >> 3) * kHalf + swz128(r16 + j, ch & 7));
            float x[8], up, down;
            load8(x, reinterpret_cast<const uint16_t*>(at));
            query_factor(row_top(x), up, down);
            *at = make_uint4(pack_p<true>(x[0] * up, x[1] * up), pack_p<true>(x[2] * up, x[3] * up), pack_p<true>(x[4] * up, x[5] * up), pack_p<true>(x[6] * up, x[7] * up));
            if (two) {
              if (ch == 0) bars->halves[0][0][16 * row_warp + j] = score_factor(c.scale_log2, down);
            } else {
              const float f = __shfl_sync(0xffffffffu, down, ((lane >> 2) & 1) * 16);
#pragma unroll
              for (int hf = 0; hf < 2; hf++)
                if (((lane >> 2) + 8 * hf) >> 1 == i) st.f[hf] = score_factor(c.scale_log2, f);
            }
          }
        if (two) {   // to the other warp of these rows
          asm volatile("bar.sync %0, 64;" ::"r"(1 + row_warp) : "memory");
#pragma unroll
          for (int hf = 0; hf < 2; hf++) st.f[hf] = bars->halves[0][0][row_in + 8 * hf];
        }
      }
      fence_proxy_async();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->q_full);
      // What the rows see, a row a lane (16), while the first scores are on their way, and only of a piece that has tiles in which rows differ.  A tree's
      // parents two a lane, so that a node's way up is one of shuffles.
      if (p.te * kTile > sq.len0) {
        uint32_t up2 = 0xffffu;
        if (c.tree && 2 * lane < c.S) up2 = reinterpret_cast<const uint16_t*>(c.seqs ? c.parents + (c.one_tree ? 0 : sq.i) * kTreeNodes : prm.parents[c.one_tree ? 0 : sq.i])[lane];
#pragma unroll 1
        for (int b = 0; b < nb; b++) {
          const int row = 128 * b + 16 * row_warp + (lane & 15), s = token_of(c, sq.row0 + row);
          uint64_t see = 0;
          if (c.tree) {
            int j = row < rows && s < sq.end - sq.len0 ? s : -1;
            while (__any_sync(0xffffffffu, j >= 0)) {
              const uint32_t pair = __shfl_sync(0xffffffffu, up2, (j & 63) >> 1);
              if (j >= 0) {
                see |= 1ull << j;
                j = (int8_t)(pair >> (8 * (j & 1)));
              }
            }
          } else if (c.causal) {
            see = s - token_of(c, sq.row0);
          }
          if (lane < 16) bars->see[row] = see;
        }
        __syncwarp();
      }
      // ---- tiles ----
      const int first = two && (k0 & 1) != set ? p.tb + 1 : p.tb;
      float v_unit = 1.f, shrink = 1.f;   // O's unit, and what it has grown by
#pragma unroll 1
      for (int t = first, b = 0; t < p.te;) {
        const int tile = tt0 + t - p.tb, step = k0 + (t - p.tb) * nb + b;
        const int from = sq.len0 - t * kTile;   // first drafted row of the tile
        if (kI8 && b == 0) {
          wait_bar(&bars->info[tile & 3], (tile >> 2) & 1, bars);
          const float unit = bars->v_unit[tile & 3];
          shrink = t > first ? v_unit / unit : 1.f;
          v_unit = unit;
        }
        const uint32_t tmem_s = tmem + lane_addr + (step & 1) * 128, tmem_o = tmem + lane_addr + kTmemO + (two ? set : b) * 128;
        wait_bar(&bars->s_full[step & 1], (step >> 1) & 1, bars);
        if (128 * b + 16 * row_warp < rows) {   // else the whole warp's rows are none
          tc_fence_after();
          uint32_t sv[64];
          tmem_ld_16x256b_x16(tmem_s, sv);
          tmem_ld_wait();
          if constexpr (kI8) {
            const float* k_scale = bars->k_scale[tile & 3];
#pragma unroll
            for (int i = 0; i < 16; i++) {
              const float2 s = *reinterpret_cast<const float2*>(k_scale + 8 * i + 2 * (lane & 3));
              const uint64_t s2 = pack2(s.x, s.y);
#pragma unroll
              for (int hf = 0; hf < 2; hf++) {
                float x0, x1;
                unpack2(mul2(pack2(__uint_as_float(sv[4 * i + 2 * hf]), __uint_as_float(sv[4 * i + 2 * hf + 1])), s2), x0, x1);
                sv[4 * i + 2 * hf] = __float_as_uint(x0);
                sv[4 * i + 2 * hf + 1] = __float_as_uint(x1);
              }
            }
          }
          const bool whole = from >= kTile;
          if (!whole) {
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
              const uint64_t see = bars->see[128 * b + row_in + 8 * hf];
              const int all = c.tree ? from : from + (int)see;   // keys below it are seen, and of the nodes some
              const uint64_t some = c.tree ? see : 0;
#pragma unroll
              for (int w = 0; w < 4; w++) {
                const int sh = all - 32 * w;   // bit i of `shown`: key 32 w + i
                uint32_t shown = sh >= 32 ? 0xffffffffu : sh >= 0 ? (uint32_t)(some << sh) | ((1u << sh) - 1u) : sh > -64 ? (uint32_t)(some >> -sh) : 0u;
                shown >>= 2 * (lane & 3);
#pragma unroll
                for (int i = 0; i < 8; i++)
                  if (!(shown >> (8 * (i >> 1) + (i & 1)) & 1u)) sv[16 * w + 4 * (i >> 1) + 2 * hf + (i & 1)] = 0xFF800000u;   // -inf
              }
            }
          }
          // row maxima of the raw scores: four chains of three-input maxima
          float mx[2];
#pragma unroll
          for (int hf = 0; hf < 2; hf++) {
            float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 16; i++) m4[i & 3] = max3(m4[i & 3], __uint_as_float(sv[4 * i + 2 * hf]), __uint_as_float(sv[4 * i + 2 * hf + 1]));
            mx[hf] = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * st.f[hf];
          }
          float alpha[2] = {shrink, shrink};
          bool rescale = kI8 && shrink != 1.f;
          if (__any_sync(0xffffffffu, mx[0] > st.m[0] + kRescaleThreshold || mx[1] > st.m[1] + kRescaleThreshold)) {
#pragma unroll
            for (int o = 1; o < 4; o <<= 1)
#pragma unroll
              for (int hf = 0; hf < 2; hf++) mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], o));
#pragma unroll
            for (int hf = 0; hf < 2; hf++)
              if (mx[hf] > st.m[hf] + kRescaleThreshold) {
                if (st.m[hf] != -INFINITY) {
                  const float a = ex2_approx(st.m[hf] - mx[hf]);
                  alpha[hf] *= a;
                  st.l[hf] *= a;
                  rescale = true;
                }
                st.m[hf] = mx[hf];
              }
          }
          uint64_t factor2[2], neg_m2[2], ps2[2];
#pragma unroll
          for (int hf = 0; hf < 2; hf++) {
            const float neg_m = (st.m[hf] == -INFINITY ? 0.f : -st.m[hf]) + (kI8 ? kPUp : 0.f);
            factor2[hf] = pack2(st.f[hf], st.f[hf]);
            neg_m2[hf] = pack2(neg_m, neg_m);
            ps2[hf] = pack2(0.f, 0.f);
          }
          uint32_t pw[32];
          exp_scores<kI8>(sv, factor2, neg_m2, pw, ps2);
          tmem_st_16x128b_x16(tmem_s, pw);
#pragma unroll
          for (int hf = 0; hf < 2; hf++) {
            float ps0, ps1;
            unpack2(ps2[hf], ps0, ps1);
            st.l[hf] += ps0 + ps1;
          }
          // O may be rescaled only behind the PV before this one on it.  With two blocks, or two halves, that is the one before QK(k) in the pipe, else
          // PV(k - 1), which QK(k) was ahead of: `pv` has then completed k - 1 or k phases, so its parity is no riddle.
          if (t > first && __any_sync(0xffffffffu, rescale)) {
            if (nb == 1 && !two) {
              wait_bar(&bars->pv, (step - 1) & 1, bars);
              tc_fence_after();
            }
#pragma unroll 1
            for (int col = 0; col < kD; col += 64) {
              uint32_t ov[32];
              tmem_ld_16x256b_x8(tmem_o + col, ov);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; i++) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha[(i >> 1) & 1]);
              tmem_st_16x256b_x8(tmem_o + col, ov);
            }
          }
          tmem_st_wait();
          tc_fence_before();
        }
        __syncwarp();
        const bool last = b + 1 == nb;
        if (lane == 0) {
          mbar_arrive(&bars->p_full[step & 1]);
          if (kI8 && last) mbar_arrive(&bars->info_empty[tile & 3]);
        }
        next_block();
        b = last ? 0 : b + 1;
        if (last) t += two ? 2 : 1;
      }
      k0 += tiles * nb;
      tt0 += tiles;
      // ---- results out: through the queries' place, which nothing reads any more, to whole lines ----
      wait_bar(&bars->fin, n & 1, bars);
      tc_fence_after();
      const bool ok = bars->abort_flag == 0;
      const uint64_t bad_nodes = kI8 ? bars->bad[n & 7].nodes : bars->bad_nodes;
      const bool bad_all = kI8 && bars->bad[n & 7].all, whole = p.tb == 0 && p.te == p.tiles;
      const int slot = 2 * (int)blockIdx.x + (p.us + p.tb == streams.u_begin ? 0 : 1);
#pragma unroll 1
      for (int b = 0; b < nb; b++, next_block()) {
        if (128 * b + 16 * row_warp >= rows) continue;
        float f[2], f2[2] = {0.f, 0.f};   // of this O, and (two) of the other half's
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
          float l = st.l[hf], m = st.m[hf], w = v_unit;
          l += __shfl_xor_sync(0xffffffffu, l, 1);
          l += __shfl_xor_sync(0xffffffffu, l, 2);
          if (two) {   // every row has been through one half or the other, or both
            const int x = row_in + 8 * hf;
            if ((lane & 3) == 0) {
              bars->halves[set][0][x] = m;
              bars->halves[set][1][x] = l;
              bars->halves[set][2][x] = v_unit;
            }
            asm volatile("bar.sync %0, 64;" ::"r"(1 + row_warp) : "memory");   // the two warps of these rows
            const float o_m = bars->halves[set ^ 1][0][x], o_l = bars->halves[set ^ 1][1][x];
            const float top = fmaxf(m, o_m), w0 = m == -INFINITY ? 0.f : ex2_approx(m - top), w1 = o_m == -INFINITY ? 0.f : ex2_approx(o_m - top);
            l = l * w0 + o_l * w1;
            w *= w0;
            f2[hf] = bars->halves[set ^ 1][2][x] * w1;
            m = top;
          }
          const int row = 128 * b + row_in + 8 * hf;
          const uint64_t see = bars->see[row];   // nobody's where the piece has none, and then no node of it is bad
          if (bad_all || (c.tree ? (see & bad_nodes) != 0 : bad_nodes != 0 && (int)see > (int)~(uint32_t)bad_nodes)) l = __uint_as_float(0x7FC00000u);
          const bool there = ok && row < rows && (!c.tree || token_of(c, sq.row0 + row) < sq.end - sq.len0);
          // no part of a sum that nobody has added to, of a row that is not there: zero whatever the accumulator holds
          const float inv = !whole ? 1.f : l == 0.f ? 0.f : __fdividef(1.f, l);
          f[hf] = !there || (st.m[hf] == -INFINITY && l == l) ? 0.f : w * inv;   // (the weights of a row that is not there may be NaN: its query is anything)
          f2[hf] = there ? f2[hf] * inv : 0.f;
          if (!whole && (lane & 3) == 0 && set == 0 && row < rows)
            *reinterpret_cast<float2*>(c.part_ml + ((size_t)slot * c.rows_rb + row) * 2) = there ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
        }
        uint8_t* place = smem + PL::kQ + b * kSlot + (r16 + 16 * set) * 128;   // 16 rows of 32 + 32 columns
#pragma unroll 1
        for (int col = two ? 64 * set : 0; col < (two ? 64 * set + 64 : kD); col += 64) {   // two: a half of the columns each
          uint32_t ov[32];
          tmem_ld_16x256b_x8(tmem + lane_addr + kTmemO + (two ? set : b) * 128 + col, ov);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; i++) ov[i] = f[(i >> 1) & 1] == 0.f ? 0u : __float_as_uint(__uint_as_float(ov[i]) * f[(i >> 1) & 1]);
          if (two) {
            uint32_t o2[32];
            tmem_ld_16x256b_x8(tmem + lane_addr + kTmemO + (set ^ 1) * 128 + col, o2);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; i++)
              if (f2[(i >> 1) & 1] != 0.f) ov[i] = __float_as_uint(fmaf(__uint_as_float(o2[i]), f2[(i >> 1) & 1], __uint_as_float(ov[i])));
          }
          __syncwarp();   // the columns before these have been read
#pragma unroll
          for (int i = 0; i < 16; i++) {   // columns 8 (i >> 1) + 2 (lane & 3) + {0, 1} of row (lane / 4) + 8 (i & 1)
            const int r = (lane >> 2) + 8 * (i & 1), chunk = 2 * ((i >> 1) & 3) + ((lane >> 1) & 1);
            *reinterpret_cast<float2*>(place + (i >> 3) * kHalf + r * 128 + ((chunk ^ (r & 7)) << 4) + (lane & 1) * 8) =
                make_float2(__uint_as_float(ov[2 * i]), __uint_as_float(ov[2 * i + 1]));
          }
          __syncwarp();
#pragma unroll 4
          for (int i = 0; i < 8; i++) {   // 16 lanes a row, four columns each
            const int r = 2 * i + (lane >> 4), row = 128 * b + 16 * row_warp + r, ch = lane & 15;
            if (row >= rows) continue;
            const float4 o = *reinterpret_cast<const float4*>(place + (ch >> 3) * kHalf + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
            const int s = token_of(c, sq.row0 + row);
            const size_t at = (whole ? (((size_t)sq.i * c.S + s) * c.H + (size_t)p.kvh * c.g + (sq.row0 + row - s * c.g)) * kD : ((size_t)slot * c.rows_rb + row) * kD) + col + 4 * ch;
            if (!whole) *reinterpret_cast<float4*>(c.part_o + at) = o;
            else if (c.out_bf16) *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(c.out) + at) = make_uint2(pack_bf16x2(o.x, o.y), pack_bf16x2(o.z, o.w));
            else *reinterpret_cast<float4*>(reinterpret_cast<float*>(c.out) + at) = o;
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (two) asm volatile("bar.sync %0, 64;" ::"r"(1 + row_warp) : "memory");   // before the next piece's queries come to the place of the other warp's results
    }
  } else if constexpr (kI8) {
    if (warp > kWarpScale) {
      regs_down<PL::kRegsOther, kI8>();   // nothing to do
    } else if (warp == kWarpScale) {
      // =============================== scales ===============================
      regs_down<PL::kRegsOther, kI8>();
      int tt = 0, n = 0;
      for (Piece p = first_piece(); streams.valid(p); p = streams.next(p), n++) {
        const TreeSeq sq = streams.seq(p.e);
        ValueUnit unit;
        uint64_t bad_nodes = 0;   // this lane's of the piece
        bool bad_all = false;
        for (int t = p.tb; t < p.te; t++, tt++) {
          const int at = tt & 3, r = 4 * lane;   // four rows a lane
          if (tt >= 4) wait_bar(&bars->info_empty[at], ((tt >> 2) - 1) & 1, bars);
          wait_bar(&bars->scale_full[at], (tt >> 2) & 1, bars);
          const float* scales = reinterpret_cast<const float*>(smem + PL::kScaleAt + at * 1024) + (r >> 6) * 128 + (r & 63);
          *reinterpret_cast<float4*>(&bars->k_scale[at][r]) = *reinterpret_cast<const float4*>(scales);
          const float4 v4 = *reinterpret_cast<const float4*>(scales + 64);
          float v[4] = {v4.x, v4.y, v4.z, v4.w};
          const int pos = t * kTile + r, there = sq.end - pos;
          float top = 0.f;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            if (i >= there) v[i] = 0.f;   // behind the drafted rows, where anything may lie
            if (!(v[i] == v[i])) {        // the row held an infinity or a NaN
              const int node = pos + i - sq.len0;
              if (node < 0) bad_all = true;
              else if (!c.tree) bad_nodes = max(bad_nodes, (uint64_t)~(uint32_t)node);   // the first one counts
              else if (node < kTreeNodes) bad_nodes |= 1ull << node;
              v[i] = 0.f;
            }
            top = fmaxf(top, v[i]);
          }
          if (__any_sync(0xffffffffu, top >= unit.limit)) unit.grow<8>(warp_max(top));   // values come below 2^15
          uint32_t s[4];
#pragma unroll
          for (int i = 0; i < 4; i++) s[i] = round_f16x2(v[i] * unit.down, v[i] * unit.down);
          *reinterpret_cast<uint4*>(&bars->v_scale[at][r]) = make_uint4(s[0], s[1], s[2], s[3]);
          if (lane == 0) bars->v_unit[at] = __uint_as_float((254u << 23) - __float_as_uint(unit.down));   // 1 / down, a power of two
          if (t + 1 == p.te) {
            const uint32_t lo = (uint32_t)bad_nodes, hi = (uint32_t)(bad_nodes >> 32);
            const uint32_t all_lo = c.tree ? __reduce_or_sync(0xffffffffu, lo) : __reduce_max_sync(0xffffffffu, lo), all_hi = __reduce_or_sync(0xffffffffu, hi);
            const bool any = __any_sync(0xffffffffu, bad_all);
            if (lane == 0) {
              bars->bad[n & 7].nodes = (uint64_t)all_hi << 32 | all_lo;
              bars->bad[n & 7].all = any;
            }
          }
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&bars->info[at]);
            mbar_arrive(&bars->scale_empty[at]);
          }
        }
      }
    } else {
      // =============================== converters ===============================
      // 16 threads a row, eight codes each: eight rows at a time, the same place of the swizzle in all of them, so that every address is a constant away.
      regs_down<PL::kRegsConv, kI8>();
      // K on two of the schedulers, V on the other two: warps of a scheduler in step share what it fetches of instructions.
      const bool of_v = (warp & 2) != 0;
      const int ct = 64 * ((warp >> 2) & 1) + (threadIdx.x & 63), hc = ct & 15, r0 = ct >> 4;
      const uint8_t* src0 = smem + PL::kRawAt + swz128(r0, hc >> 1) + (hc & 1) * 8;
      const uint32_t dst0 = swz128(r0, hc & 7);
      constexpr int kAtOnce = 4;
      int raw = 0, raw_phase = 0;   // the next slot of the ring of codes
      // A page of codes to dst; its slot is free again.
      auto convert = [&](uint8_t* dst, const uint32_t* v_scale, auto values) {
        constexpr int kFirst = decltype(values)::value ? PL::kRawK : 0, kNum = decltype(values)::value ? PL::kRawV : PL::kRawK;
        wait_bar(&bars->raw_full[kFirst + raw], raw_phase, bars);
        const uint8_t* src = src0 + (kFirst + raw) * kRawSlot;
#pragma unroll 1
        for (int i0 = 0; i0 < 8; i0 += kAtOnce, src += kAtOnce * 1024, dst += kAtOnce * 1024) {
          uint2 w[kAtOnce];
          uint32_t s[kAtOnce];
#pragma unroll
          for (int i = 0; i < kAtOnce; i++) {
            w[i] = *reinterpret_cast<const uint2*>(src + i * 1024);
            if constexpr (decltype(values)::value) s[i] = v_scale[8 * (i0 + i)];
          }
#pragma unroll
          for (int i = 0; i < kAtOnce; i++) {
            uint32_t x[4];
            int8x4_to_f16(w[i].x, x[0], x[1]);
            int8x4_to_f16(w[i].y, x[2], x[3]);
            if constexpr (decltype(values)::value) {
#pragma unroll
              for (int j = 0; j < 4; j++) {
                const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&x[j]), *reinterpret_cast<const __half2*>(&s[i]));
                x[j] = *reinterpret_cast<const uint32_t*>(&y);
              }
            }
            *reinterpret_cast<uint4*>(dst + i * 1024) = make_uint4(x[0], x[1], x[2], x[3]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->raw_empty[kFirst + raw]);
        if (++raw == kNum) {
          raw = 0;
          raw_phase ^= 1;
        }
      };
      int tt = 0, st = 0, phase = 1;   // tiles so far; the next slot of the ring of operands, whose first use waits for nothing
      for (Piece p = first_piece(); streams.valid(p); p = streams.next(p))
        for (int t = p.tb; t < p.te; t++, tt++) {
          if (!of_v) {
            wait_bar(&bars->empty[st], phase, bars);
            uint8_t* dst = smem + PL::kRing + st * kSlot + (hc >> 3) * kHalf + dst0;
#pragma unroll 1
            for (int k = 0; k < 2; k++) convert(dst + k * kRawSlot, nullptr, std::false_type{});
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->full[st]);
            if (++st == PL::kSlots) {
              st = 0;
              phase ^= 1;
            }
          } else {
            wait_bar(&bars->info[tt & 3], (tt >> 2) & 1, bars);
#pragma unroll 1
            for (int k = 0; k < 2; k++) {
              wait_bar(&bars->empty[PL::kSlots + st], phase, bars);
              convert(smem + PL::kRingV + st * kHalf + (hc >> 3) * (kHalf / 2) + dst0, &bars->v_scale[tt & 3][64 * k + r0], std::true_type{});
              fence_proxy_async();
              __syncwarp();
              if (lane == 0) mbar_arrive(&bars->full[PL::kSlots + st]);
              if (++st == PL::kSlotsV) {
                st = 0;
                phase ^= 1;
              }
            }
            if (lane == 0) mbar_arrive(&bars->info_empty[tt & 3]);
          }
        }
    }
  }
  if (c.out_bf16) fence_chained_writes();   // activations, which a later launch may read by TMA
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) {
    stamp_end(c.time);
    if (bars->abort_flag) set_status(c.status, RELUX_ERR_TIMEOUT);
  }
  if (warp == 0) tmem_dealloc<1>(tmem, kTmemCols);
}

// Joins the partials of the streams that more than one range has a part of: block x is the range behind a stream's first part, a warp every 8 gridDim.y-th
// row.  What a block costs is the search for its stream, so that it is given several rows a warp, and a row's parts are read at once, in one pass with a
// running maximum (a row a warp, and the maxima before the sums: 24 us for 148 ranges of 2 x 240 rows, 35 MB).
constexpr int kMergeRows = 4;   // of a warp
template <int N>
__global__ void __launch_bounds__(256, 4) merge_tree_kernel(const __grid_constant__ TreeParams<N> prm) {
  chain_release();
  chain_wait();   // every block: the launch behind this one takes it that the one before is complete
  const TreeCommon& c = prm.c;
  const Streams<N> streams(prm, blockIdx.x + 1);
  const int u = streams.u_begin, lane = threadIdx.x & 31;
  const Piece p = streams.at(u);
  const int w0 = blockIdx.x;
  if (p.tb <= 0 || p.tb >= p.tiles || prm.cuts[w0] > p.us) return;   // no stream goes on here, or its first part is further back
  int np = 2;
  while (w0 + np <= (int)gridDim.x && prm.cuts[w0 + np] < p.us + p.tiles) np++;
  const TreeSeq sq = streams.seq(p.e);
  const int rows = min(c.rows_rb, c.R - sq.row0), first = prm.cuts[w0] == p.us ? 0 : 1;
#pragma unroll 2
  for (int r = blockIdx.y * 8 + (threadIdx.x >> 5); r < rows; r += gridDim.y * 8) {
    float M = -INFINITY, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j0 = 0; j0 < np; j0 += 4) {
      float2 ml[4];
      float4 x[4];
#pragma unroll
      for (int q = 0; q < 4; q++) {
        ml[q] = make_float2(-INFINITY, 0.f);
        if (j0 + q < np) {
          const size_t at = (size_t)(2 * (w0 + j0 + q) + (j0 + q ? 0 : first)) * c.rows_rb + r;
          ml[q] = load_chained(reinterpret_cast<const float2*>(c.part_ml) + at);
          x[q] = load_chained(reinterpret_cast<const float4*>(c.part_o + at * kD) + lane);
        }
      }
      const float top = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), M);
      if (M != -INFINITY && top > M) {
        const float w = ex2_approx(M - top);
        L *= w;
        o.x *= w;
        o.y *= w;
        o.z *= w;
        o.w *= w;
      }
      M = top;
#pragma unroll
      for (int q = 0; q < 4; q++)
        // A part whose scores of this row are all NaN has a maximum of nothing and a sum of NaN: exp2(-inf - M) of that is NaN or nothing, and so is L then NaN.
        if (ml[q].x != -INFINITY || ml[q].y != ml[q].y) {
          const float w = ex2_approx(ml[q].x - M);
          L = fmaf(ml[q].y, w, L);
          o.x = fmaf(x[q].x, w, o.x);
          o.y = fmaf(x[q].y, w, o.y);
          o.z = fmaf(x[q].z, w, o.z);
          o.w = fmaf(x[q].w, w, o.w);
        }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int row = sq.row0 + r, s = token_of(c, row);
    const size_t at = (((size_t)sq.i * c.S + s) * c.H + (size_t)p.kvh * c.g + (row - s * c.g)) * kD + 4 * lane;
    if (c.out_bf16) *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(c.out) + at) = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
    else *reinterpret_cast<float4*>(reinterpret_cast<float*>(c.out) + at) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  }
  if (c.out_bf16) fence_chained_writes();
  __syncthreads();
  if (threadIdx.x == 0) stamp_end(c.time);   // of every block that joined rows: the attention's time ends with the last of them
}

template <bool kI8, int kNB, int N>
int32_t launch(Pool* p, const TreeParams<N>& prm, int workers, bool parts) {
  using PL = Plan<kI8, kNB>;
  const bool chained = p->tune.get(RELUX_TUNE_CHAINED_LAUNCHES) != 0;
  if (int32_t rc = allow_smem(p->dev, tree_sm100_kernel<kI8, kNB, N>, PL::kTotal)) return rc;
  RELUX_CUDA_TRY(launch_chained(chained, tree_sm100_kernel<kI8, kNB, N>, dim3(workers), dim3(PL::kThreads), (size_t)PL::kTotal, p->dev->stream, p->tmap_gqa, prm));
  count_launch(p->dev);
  if (parts) {
    RELUX_CUDA_TRY(launch_chained(chained, merge_tree_kernel<N>, dim3(workers - 1, (prm.c.rows_rb + 8 * kMergeRows - 1) / (8 * kMergeRows)), dim3(256), 0, p->dev->stream, prm));
    count_launch(p->dev);
  }
  return RELUX_OK;
}
// The ranges.  Equal ones cut nearly every stream where there are about as many streams as SMs: two parts an SM, each with its queries, its float32 sums out and
// in again, and a launch that joins them.  So where there are few streams a range (kPackStreams), whole ones are dealt out as well, in their order and none cut that
// is no longer than the longest range, and taken where that longest range is no more than what the parts would cost.  (Calls of 240 rows: 128 streams of 3000
// tokens 86 us with equal ranges, 74 with whole streams, on 8 bits 112 and 100; 144 of 1000 57 and 45; 296 of 2000 118 and 115; a prompt's 256 of 1564 to 2000
// 143 and 138.)
struct Ranges {
  int32_t cuts[kMaxWorkers + 1];
  int workers;
  bool parts;   // some stream is in several ranges
};
constexpr int kPackStreams = 3;             // of a range, at most

// Whole streams in their order, ranges of up to `most` units; false: that takes more than `workers`.
bool pack_streams(const TreeSeq* seqs, int n, int n_rb, int Hkv, int workers, int64_t most, int part, Ranges& out) {
  int w = 0;
  int64_t room = most, pos = 0;
  out.cuts[0] = 0;
  out.parts = false;
  for (int i = 0; i < n; i++)
    for (int h = 0; h < Hkv; h++)
      for (int e = i * n_rb; e < (i + 1) * n_rb; e++) {
        const int units = seqs[e + 1].unit0 - seqs[e].unit0, tiles = units - kFixUnits;
        for (int done = 0; done < tiles;) {
          const int rest = tiles - done, need = rest + kFixUnits + (done ? part : 0);
          if (need <= room) {
            room -= need;
            done = tiles;
          } else {
            const int64_t fit = room - kFixUnits - part;   // tiles of a part
            if (units > most && fit >= 4) {
              done += (int)std::min<int64_t>(fit, rest - 1);
              out.parts = true;
            } else if (room == most) {
              return false;
            }
            if (++w == workers) return false;
            out.cuts[w] = (int32_t)(pos + done);
            room = most;
          }
        }
        pos += units;
      }
  out.workers = w + 1;
  out.cuts[w + 1] = (int32_t)pos;
  return true;
}
Ranges make_ranges(const TreeSeq* seqs, int n, int n_rb, int Hkv, int units, int sm_count, int blocks) {
  const int part = blocks, join = blocks == 2 ? 5 : 2;   // tiles: what a part costs beyond a whole stream, and the join of all (parts of one block: half the bytes)
  Ranges r;
  r.workers = std::max(1, std::min({sm_count, kMaxWorkers, units / (kFixUnits + 1)}));
  for (int w = 0; w <= r.workers; w++) r.cuts[w] = w * (units / r.workers) + std::min(w, units % r.workers);
  r.parts = r.workers > 1;
  const int64_t streams = (int64_t)n * n_rb * Hkv;
  if (2 * streams >= r.workers && streams <= (int64_t)kPackStreams * r.workers) {
    const int64_t equal = (units + r.workers - 1) / r.workers, cost = equal + kFixUnits + 2 * part + join;
    Ranges best;
    int64_t lo = equal - 1, hi = cost + 1;   // lo: too few; hi: not looked at, or found
    while (hi - lo > 1) {
      const int64_t most = (lo + hi) / 2;
      Ranges some;
      if (pack_streams(seqs, n, n_rb, Hkv, r.workers, most, part, some)) {
        best = some;
        hi = most;
      } else {
        lo = most;
      }
    }
    if (hi + (hi <= cost && best.parts ? join : 0) <= cost) return best;
  }
  return r;
}

template <int N>
int32_t launch_n(Pool* p, const TreeCommon& c, const TreeSeq* seqs, const GqaTree* tree, const Ranges& ranges) {
  const int workers = ranges.workers;
  TreeParams<N> prm;
  prm.c = c;
  memcpy(prm.cuts, ranges.cuts, sizeof(int32_t) * ((size_t)workers + 1));
  if (!c.seqs) {
    memcpy(prm.seqs, seqs, sizeof(TreeSeq) * ((size_t)c.n_seqs * c.n_rb + 1));
    if (tree) memcpy(prm.parents, tree->parents, (size_t)kTreeNodes * (tree->one ? 1 : c.n_seqs));
  }
  if (p->int8) return c.rows_rb <= 128 ? launch<true, 1, N>(p, prm, workers, ranges.parts) : launch<true, 2, N>(p, prm, workers, ranges.parts);
  return c.rows_rb <= 128 ? launch<false, 1, N>(p, prm, workers, ranges.parts) : launch<false, 2, N>(p, prm, workers, ranges.parts);
}

}  // namespace

// q: device bf16 [n][S][H][128] token-major.  out: device, same shape, f32 or bf16.  All rows are in the cache.  tree: with `nodes`, host, those of
// every sequence, which lie behind its length; nullptr: the call's own mask (causal or none).
int32_t launch_gqa_tree_sm100(Pool* p, const SeqBatch& sb, const relux_attn_args& a, const void* d_q, void* d_out, bool out_bf16, const GqaTree* tree,
                              const int32_t* nodes) {
  const relux_pool_params& prm = p->prm;
  const int n = sb.n_seqs, Hkv = prm.gqa_num_kv_heads, g = a.num_heads / Hkv, S = a.q_tokens;
  const int64_t R = (int64_t)g * S;
  if (a.q_dtype != RELUX_DTYPE_BF16) { set_error("queries of this kernel are bf16"); return RELUX_ERR_UNSUPPORTED; }
  TreeCommon c{};
  c.n_rb = (int)((R + 255) / 256);
  c.rows_rb = (int)((R + c.n_rb - 1) / c.n_rb + 15) / 16 * 16;
  c.n_rb = (int)((R + c.rows_rb - 1) / c.rows_rb);
  const int64_t groups = (int64_t)n * c.n_rb;
  // R g: over_g g is less than 2^31 + g, so that a row times it stays below the next whole number while row g is below 2^31
  if (R >= ((int64_t)1 << 26) || R * g > ((int64_t)1 << 31) || groups >= ((int64_t)1 << 24)) { set_error("more query rows than one attention launch addresses"); return RELUX_ERR_UNSUPPORTED; }
  std::vector<TreeSeq> seqs;
  try {
    seqs.resize((size_t)groups + 1);
  } catch (const std::bad_alloc&) {
    set_error("out of host memory for %lld groups of query rows", (long long)groups);
    return RELUX_ERR_OUT_OF_MEMORY;
  }
  int64_t units64 = 0;
  for (int i = 0; i < n; i++) {
    const int s = sb.seq[i], len = p->h_len[(size_t)a.layer * prm.max_seqs + s], T = len + (tree ? nodes[i] : a.extra_tokens);
    for (int rb = 0; rb < c.n_rb; rb++) {
      const int row0 = rb * c.rows_rb, s0 = row0 / g, s1 = (int)(std::min<int64_t>(row0 + c.rows_rb, R) - 1) / g;   // first and last query token
      // causal: token s sees the first T - S + s + 1
      const int len0 = tree ? len : a.causal ? T - S + s0 + 1 : T, end = tree || !a.causal ? T : T - S + s1 + 1;
      seqs[(size_t)i * c.n_rb + rb] = TreeSeq{s, i, len0, end, row0, (int32_t)units64};
      units64 += std::max(1, (end + kTile - 1) / kTile) + kFixUnits;
      if (units64 * Hkv >= ((int64_t)1 << 31)) { set_error("more cached pages than one attention launch addresses"); return RELUX_ERR_UNSUPPORTED; }
    }
  }
  seqs[(size_t)groups] = TreeSeq{0, 0, 0, 0, 0, (int32_t)units64};
  const int units = (int)(units64 * Hkv);
  const Ranges ranges = make_ranges(seqs.data(), n, c.n_rb, Hkv, units, p->dev->sm_count, c.rows_rb <= 128 ? 1 : 2);
  const size_t part_rows = (size_t)2 * ranges.workers * c.rows_rb;
  int32_t rc = grow(p->dev, p->part_o, part_rows * (kD + 2) * sizeof(float));
  if (rc) return rc;
  if (groups > kInlineLarge) {
    if (stream_captured(p->dev)) {   // the list is this call's
      set_error("a call of %lld groups of query rows cannot be captured (%d can)", (long long)groups, kInlineLarge);
      return RELUX_ERR_UNSUPPORTED;
    }
    const size_t list = sizeof(TreeSeq) * seqs.size(), bytes = list + (tree ? (size_t)kTreeNodes * (tree->one ? 1 : n) : 0);
    if ((rc = grow(p->dev, p->seq_list, bytes))) return rc;
    // (pageable memory: the copies have read it when they return)
    RELUX_CUDA_TRY(cudaMemcpyAsync(p->seq_list.p, seqs.data(), list, cudaMemcpyHostToDevice, p->dev->stream));
    if (tree) RELUX_CUDA_TRY(cudaMemcpyAsync((char*)p->seq_list.p + list, tree->parents, bytes - list, cudaMemcpyHostToDevice, p->dev->stream));
    c.seqs = (const TreeSeq*)p->seq_list.p;
    c.parents = (const int8_t*)(c.seqs + seqs.size());
  }
  c.one_tree = tree && tree->one;
  c.tree = tree != nullptr;
  c.causal = a.causal;
  c.table = p->d_table;
  c.table_stride = prm.max_pages_per_seq;
  c.num_pages = prm.num_pages;
  c.n_seqs = n;
  c.Hkv = Hkv;
  c.H = a.num_heads;
  c.g = g;
  c.over_g = (uint32_t)((((uint64_t)1 << 31) + g - 1) / g);
  c.S = S;
  c.R = (int)R;
  const int64_t rows_per_block = (int64_t)prm.num_pages * Hkv * kPage;
  c.krow0 = (int32_t)((int64_t)a.layer * 2 * rows_per_block);
  c.vrow0 = (int32_t)((int64_t)a.layer * 2 * rows_per_block + rows_per_block);
  if (p->int8) {
    c.scales = p->scales_at(a.layer);
    c.codes = (const uint8_t*)p->storage;
  }
  c.scale_log2 = a.scale * 1.4426950408889634f;
  c.q = (const uint16_t*)d_q;
  c.out_bf16 = out_bf16;
  c.out = d_out;
  c.part_o = (float*)p->part_o.p;
  c.part_ml = c.part_o + part_rows * kD;
  c.status = p->d_status;
  c.time = time_stamp_next(p, p->attn_times);
  rc = groups <= kInlineSmall || c.seqs ? launch_n<kInlineSmall>(p, c, seqs.data(), tree, ranges) : launch_n<kInlineLarge>(p, c, seqs.data(), tree, ranges);
  if (rc) return rc;
  time_stamp_done(p->attn_times, c.time);
  return RELUX_OK;
}

}  // namespace relux
