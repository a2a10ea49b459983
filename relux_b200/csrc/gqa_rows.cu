// Rows of a grouped-query cache, bf16 or 8-bit, read back to dense device memory, and the commit of a drafted tree's accepted path.
//
// Both are byte movement.  Read back: n tokens are n * Hkv * 264 B of an 8-bit cache (512 of bf16) in and n * Hkv * 512 B of bf16 out; of a bf16 cache a block takes
// kRowsAhead tokens at a time, all their loads, then all their stores, as the append does.  Commit: a few rows of each sequence and layer, bound by the launch
// and by the latency of a length, a page id and a row, one after the other.
#include <algorithm>

#include "common.cuh"
#include "gqa_int8_parts.cuh"
#include "internal.h"
#include "softmax_parts.cuh"

namespace relux {

namespace {

constexpr int kRowsAhead = 4;
constexpr int kSeqsSmall = 32, kSeqsLarge = 256;   // sequences carried as kernel arguments; more go in several launches

struct RowSeq {
  int32_t seq, tok0, n, row0;   // pool sequence, first token, tokens, row of the result
};
struct ReadCommon {
  const void* k;          // layer `layer0`
  const void* v;
  size_t layer_bytes;     // between two layers
  const float* scales;    // 8-bit caches
  size_t layer_scales;
  const int32_t* table;
  int32_t table_stride, num_pages, page_tokens, Hkv, D;
  void* k_out;            // [layers][rows][Hkv][D]
  void* v_out;
  int64_t rows;           // of all sequences of the call
  int32_t* status;
  bool wide;              // k_out and v_out are multiples of 32
  int32_t parts;          // 8-bit caches: blocks that share a page's heads
};
template <int N>
struct ReadParams {
  ReadCommon c;
  RowSeq seqs[N];
};

// Eight bf16 values of a row, as they are or as float32.
template <bool kF32>
__device__ __forceinline__ void put8(void* to, size_t off, uint4 w) {
  if constexpr (kF32) {
    float4* f = reinterpret_cast<float4*>(reinterpret_cast<float*>(to) + off);
    f[0] = make_float4(bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y));
    f[1] = make_float4(bf16_lo(w.z), bf16_hi(w.z), bf16_lo(w.w), bf16_hi(w.w));
  } else {
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(to) + off) = w;
  }
}

// 32 bytes, in one store where the place is a multiple of 32.
__device__ __forceinline__ void store32(bool wide, void* to, const uint32_t (&w)[8]) {
  if (!wide) {
    reinterpret_cast<uint4*>(to)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(to)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    return;
  }
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(__cvta_generic_to_global(to)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
// 16 codes times their scale, to 16 values.  The product is rounded to float32, and that to bf16.
template <bool kF32>
__device__ __forceinline__ void put_codes(bool wide, void* to, size_t off, uint4 codes, float s) {
  const uint32_t c[4] = {codes.x, codes.y, codes.z, codes.w};
  const uint64_t s2 = pack2(s, s), zero2 = pack2(-8388736.f, -8388736.f);
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 8; i++) {   // a byte under 0x4B0000 is 2^23 + it, of which 2^23 + 128 is nothing
    const uint32_t lo = __byte_perm(c[i >> 1], 0x4B000000u, i & 1 ? 0x7442 : 0x7440), hi = __byte_perm(c[i >> 1], 0x4B000000u, i & 1 ? 0x7443 : 0x7441);
    float x0, x1;
    unpack2(mul2(add2(pack2(__uint_as_float(lo), __uint_as_float(hi)), zero2), s2), x0, x1);
    if constexpr (kF32) {
      w[2 * i] = __float_as_uint(x0);
      w[2 * i + 1] = __float_as_uint(x1);
    } else {
      w[i] = round_bf16x2(x0, x1);
    }
  }
  if constexpr (kF32) {
    float* f = reinterpret_cast<float*>(to) + off;
    store32(wide, f, reinterpret_cast<const uint32_t(&)[8]>(w[0]));
    store32(wide, f + 8, reinterpret_cast<const uint32_t(&)[8]>(w[8]));
  } else {
    store32(wide, reinterpret_cast<uint16_t*>(to) + off, reinterpret_cast<const uint32_t(&)[8]>(w[0]));
  }
}

// 8-bit cache: grid (sequences, pages of one times parts, layers), a warp a head's rows of a page, of K or of V: eight lanes a row, 16 codes each, kCodesAhead
// loads of four rows on their way.  kFew: fewer rows of any page than those, and the warp takes them one head behind another (64 x 5 tokens of 32 layers: 20 us
// one head at a time, 15 so; 8 x 2048 tokens 18 and 23).  (With a row's codes eight a lane, and blocks that looked up a page for every four tokens, 4 x 8192 tokens took 48 us.)
constexpr int kCodesAhead = 8, kCodesWarps = 4;
template <bool kF32, bool kFew, int N>
__global__ void __launch_bounds__(32 * kCodesWarps, 8) read_codes_kernel(const __grid_constant__ ReadParams<N> prm) {
  chain_release();
  chain_wait();
  const ReadCommon& c = prm.c;
  const RowSeq sq = prm.seqs[blockIdx.x];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane >> 3, d = (lane & 7) * 16;
  const int end = sq.tok0 + sq.n, first = (int)blockIdx.y / c.parts, part = (int)blockIdx.y - first * c.parts;
  for (int slot = sq.tok0 / kGqaPageTok + first; slot < (end + kGqaPageTok - 1) / kGqaPageTok && sq.n > 0; slot += gridDim.y / c.parts) {
    const int32_t pg = __ldg(c.table + (size_t)sq.seq * c.table_stride + slot);   // the page table is written by host calls that wait for their copy
    if (pg < 0 || pg >= c.num_pages) {
      set_status(c.status, RELUX_ERR_BAD_PAGE);
      continue;
    }
    const int base = slot * kGqaPageTok, lo = max(sq.tok0 - base, 0), hi = min(end - base, kGqaPageTok);
    const int64_t row0 = (int64_t)blockIdx.z * c.rows + sq.row0 + base - sq.tok0;
    // kCodesAhead groups of four rows at a time
    const int step = c.parts * kCodesWarps;
    auto load = [&](int u, int r, uint4& w, float& s) {   // K or V of a head, u, row r
      if (u >= 2 * c.Hkv || r >= hi) return;
      const int which = u >= c.Hkv;
      const size_t head = (size_t)pg * c.Hkv + (u - which * c.Hkv);
      const uint8_t* codes = (const uint8_t*)(which ? c.v : c.k) + (size_t)blockIdx.z * c.layer_bytes;
      w = load_chained(reinterpret_cast<const uint4*>(codes + (head * kGqaPageTok + r) * kGqaD + d));
      s = load_chained(c.scales + (size_t)blockIdx.z * c.layer_scales + (head * 2 + which) * kGqaPageTok + r);
    };
    auto put = [&](int u, int r, const uint4& w, float s) {
      if (u >= 2 * c.Hkv || r >= hi) return;
      const int which = u >= c.Hkv;
      put_codes<kF32>(c.wide, which ? c.v_out : c.k_out, (size_t)((row0 + r) * c.Hkv + (u - which * c.Hkv)) * kGqaD + d, w, s);
    };
    uint4 w[kCodesAhead];
    float s[kCodesAhead];
    int u = part * kCodesWarps + warp;
    if constexpr (kFew) {
      auto next = [&](int& u, int& r) {
        if ((r += 4) >= hi) {
          r = lo;
          u += step;
        }
      };
      for (int r = lo; u < 2 * c.Hkv;) {
        int u1 = u, r1 = r;
#pragma unroll
        for (int q = 0; q < kCodesAhead; q++, next(u1, r1)) load(u1, r1 + sub, w[q], s[q]);
#pragma unroll
        for (int q = 0; q < kCodesAhead; q++, next(u, r)) put(u, r + sub, w[q], s[q]);
      }
    } else {
      for (; u < 2 * c.Hkv; u += step)
        for (int r0 = lo + sub; r0 < hi; r0 += 4 * kCodesAhead) {
#pragma unroll
          for (int q = 0; q < kCodesAhead; q++) load(u, r0 + 4 * q, w[q], s[q]);
#pragma unroll
          for (int q = 0; q < kCodesAhead; q++) put(u, r0 + 4 * q, w[q], s[q]);
        }
    }
  }
  fence_chained_writes();
}

// bf16 cache: grid (sequences, slices of their tokens, layers).
template <bool kF32, int N>
__global__ void read_kv_kernel(const __grid_constant__ ReadParams<N> prm) {
  chain_release();
  chain_wait();
  const ReadCommon& c = prm.c;
  const RowSeq sq = prm.seqs[blockIdx.x];
  const int layer = blockIdx.z, per_head = c.D / 8, per_tok = c.Hkv * per_head;
  const int32_t* row = c.table + (size_t)sq.seq * c.table_stride;
  constexpr int kN = kRowsAhead;
  for (int r = blockIdx.y * kN; r < sq.n; r += gridDim.y * kN) {
    int32_t pg[kN], tok[kN];
#pragma unroll
    for (int q = 0; q < kN; q++) {
      const int pos = sq.tok0 + r + q, slot = pos / c.page_tokens;
      tok[q] = pos - slot * c.page_tokens;
      pg[q] = -1;
      if (r + q < sq.n) {
        pg[q] = __ldg(row + slot);   // the page table is written by host calls that wait for their copy
        if (pg[q] < 0 || pg[q] >= c.num_pages) {
          set_status(c.status, RELUX_ERR_BAD_PAGE);
          pg[q] = -1;
        }
      }
    }
    for (int u = threadIdx.x; u < 2 * per_tok; u += blockDim.x) {
      const int which = u >= per_tok, e = u - which * per_tok, h = e / per_head, d = (e - h * per_head) * 8;
      const uint16_t* base = (const uint16_t*)((const char*)(which ? c.v : c.k) + (size_t)layer * c.layer_bytes);
      uint4 x[kN];
#pragma unroll
      for (int q = 0; q < kN; q++)
        if (pg[q] >= 0) x[q] = load_chained(reinterpret_cast<const uint4*>(base + (((size_t)pg[q] * c.Hkv + h) * c.page_tokens + tok[q]) * c.D + d));
#pragma unroll
      for (int q = 0; q < kN; q++)
        if (pg[q] >= 0)
          put8<kF32>(which ? c.v_out : c.k_out, (((size_t)layer * c.rows + sq.row0 + r + q) * c.Hkv + h) * c.D + d, x[q]);
    }
  }
  fence_chained_writes();
}

template <bool kF32, int N>
int32_t launch_read_n(Pool* p, const ReadCommon& c, const RowSeq* seqs, int n, int layers) {
  ReadParams<N> prm;
  prm.c = c;
  memcpy(prm.seqs, seqs, sizeof(RowSeq) * n);
  int most = 1;
  for (int i = 0; i < n; i++) most = std::max(most, seqs[i].n);
  // bf16: about five blocks an SM in all.  8-bit: a page of tokens a block (rows that lie across two pages do not make two), or where those are few, several
  // blocks a page, up to a head a warp (8 x 2048 tokens, 256 pages: 27 us with one, 21 with four; 64 x 5 tokens of 32 layers: 18 with one, 22 with four)
  const int64_t pages = (most + kGqaPageTok - 1) / kGqaPageTok, blocks = pages * n * layers;
  prm.c.parts = (int)std::min<int64_t>((2 * c.Hkv + kCodesWarps - 1) / kCodesWarps, std::max<int64_t>(1, 12 * p->dev->sm_count / blocks));
  const int slices = p->int8 ? prm.c.parts * (int)std::max<int64_t>(1, std::min<int64_t>(pages, 65535 / prm.c.parts))
                             : std::min((most + kRowsAhead - 1) / kRowsAhead, std::max(1, 5 * p->dev->sm_count / (n * layers)));
  const int threads = p->int8 ? 32 * kCodesWarps : std::min(256, (2 * c.Hkv * (c.D / 8) + 31) / 32 * 32);
  RELUX_CUDA_TRY(launch_chained(p->tune.get(RELUX_TUNE_CHAINED_LAUNCHES) != 0, !p->int8 ? read_kv_kernel<kF32, N> : most < 4 * kCodesAhead ? read_codes_kernel<kF32, true, N> : read_codes_kernel<kF32, false, N>,
                                dim3(n, slices, layers), dim3(threads), 0, p->dev->stream, prm));
  count_launch(p->dev);
  return RELUX_OK;
}
template <bool kF32>
int32_t launch_read(Pool* p, const ReadCommon& c, const std::vector<RowSeq>& seqs, int layers) {
  for (size_t at = 0; at < seqs.size(); at += kSeqsLarge) {
    const int n = (int)std::min<size_t>(kSeqsLarge, seqs.size() - at);
    const int32_t rc = n <= kSeqsSmall ? launch_read_n<kF32, kSeqsSmall>(p, c, &seqs[at], n, layers) : launch_read_n<kF32, kSeqsLarge>(p, c, &seqs[at], n, layers);
    if (rc) return rc;
  }
  return RELUX_OK;
}

}  // namespace

// Tokens [tok0[i], tok0[i] + n[i]) of the batch's sequences, layers layer0 .. layer0 + layers - 1.
int32_t launch_read_kv(Pool* p, const SeqBatch& sb, int layer0, int layers, const int32_t* tok0, const int32_t* n, int dtype, void* k_out, void* v_out) {
  const relux_pool_params& prm = p->prm;
  std::vector<RowSeq> seqs(sb.n_seqs);
  int32_t row = 0;
  for (int i = 0; i < sb.n_seqs; i++) {
    seqs[i] = RowSeq{sb.seq[i], tok0 ? tok0[i] : 0, n[i], row};
    row += n[i];
  }
  ReadCommon c{};
  c.k = p->rows_at(layer0, 0);
  c.v = p->rows_at(layer0, 1);
  c.layer_bytes = p->layer_elems * p->elem_bytes();
  if (p->int8) {
    c.scales = p->scales_at(layer0);
    c.layer_scales = p->layer_scales();
  }
  c.table = p->d_table;
  c.table_stride = prm.max_pages_per_seq;
  c.num_pages = prm.num_pages;
  c.page_tokens = prm.page_tokens;
  c.Hkv = prm.gqa_num_kv_heads;
  c.D = prm.gqa_head_dim;
  c.k_out = k_out;
  c.v_out = v_out;
  c.wide = (((uintptr_t)k_out | (uintptr_t)v_out) & 31) == 0;
  c.rows = row;
  c.status = p->d_status;
  return dtype == RELUX_DTYPE_F32 ? launch_read<true>(p, c, seqs, layers) : launch_read<false>(p, c, seqs, layers);
}

int32_t do_read_kv(Pool* p, const relux_read_kv_args* a) {
  if (!a) { set_error("nil argument struct"); return RELUX_ERR_INVALID_ARG; }
  const relux_pool_params& prm = p->prm;
  if (prm.kind != RELUX_POOL_GQA) { set_error("relux_gqa_read_kv needs a GQA pool"); return RELUX_ERR_INVALID_ARG; }
  if (a->layer >= prm.num_layers) { set_error("layerIdx=%d out of range [0, %d)", a->layer, prm.num_layers); return RELUX_ERR_INVALID_ARG; }
  if (!a->n_tokens || !a->k || !a->v) { set_error("read_kv: nil n_tokens, k or v"); return RELUX_ERR_INVALID_ARG; }
  if (a->dtype != RELUX_DTYPE_F32 && a->dtype != RELUX_DTYPE_BF16) { set_error("read_kv: bad dtype"); return RELUX_ERR_INVALID_ARG; }
  for (int32_t r : a->reserved)
    if (r) { set_error("reserved fields must be zero"); return RELUX_ERR_INVALID_ARG; }
  int32_t rc;
  if ((rc = check_dev_align(a->k, "k")) || (rc = check_dev_align(a->v, "v"))) return rc;
  SeqBatch sb;
  if ((rc = stage_batch(p, a->n_seqs, a->seq_ids, a->n_tokens, 1, &sb, false))) return rc;
  int64_t total = 0;
  for (int i = 0; i < sb.n_seqs; i++) {
    const int64_t t0 = a->tok0 ? a->tok0[i] : 0, cap = (int64_t)p->seq_pages[sb.seq[i]] * prm.page_tokens;
    if (t0 < 0 || t0 + a->n_tokens[i] > cap) {
      set_error("read_kv: sequence %d rows [%lld,%lld) outside its capacity", sb.seq[i], (long long)t0, (long long)(t0 + a->n_tokens[i]));
      return RELUX_ERR_INVALID_ARG;
    }
    total += a->n_tokens[i];
  }
  if (total >= ((int64_t)1 << 31)) { set_error("read_kv: more rows than one call addresses"); return RELUX_ERR_UNSUPPORTED; }
  if (total == 0) return RELUX_OK;
  const int layer0 = a->layer < 0 ? 0 : a->layer, layers = a->layer < 0 ? prm.num_layers : 1;
  constexpr int kGridZ = 65535;
  const size_t row_bytes = (size_t)total * prm.gqa_num_kv_heads * prm.gqa_head_dim * (a->dtype == RELUX_DTYPE_F32 ? 4 : 2);
  for (int l = 0; l < layers; l += kGridZ) {
    rc = launch_read_kv(p, sb, layer0 + l, std::min(kGridZ, layers - l), a->tok0, a->n_tokens, a->dtype, (char*)a->k + l * row_bytes, (char*)a->v + l * row_bytes);
    if (rc) return rc;
  }
  return RELUX_OK;
}

// ---- commit of a tree's path -----------------------------------------------------------------------------------------------
namespace {

struct CommitSeq {
  int32_t seq, n;
  uint8_t path[kTreeNodes];
};
struct CommitCommon {
  char* k;                // layer 0 of the call
  char* v;
  size_t layer_bytes;
  float* scales;          // 8-bit caches
  size_t layer_scales;
  const int32_t* table;
  int32_t table_stride, num_pages, page_tokens, Hkv, row_bytes, max_seqs;
  int32_t* len;           // [layers][max_seqs]
  int32_t* status;
};
template <int N>
struct CommitParams {
  CommitCommon c;
  CommitSeq seqs[N];
};

// grid (sequences, layers): a block is all that writes a sequence's rows and length of a layer.
// Node path[k] >= k (the path is increasing), so a place k that is written was read by no later step of the path: a thread that takes the
// same columns of all rows may go through the path in order, kAtOnce rows at a time, all their loads before their stores.
template <int N>
__global__ void tree_commit_kernel(const __grid_constant__ CommitParams<N> prm) {
  chain_release();
  chain_wait();
  const CommitCommon& c = prm.c;
  const CommitSeq& sq = prm.seqs[blockIdx.x];
  __shared__ int64_t from[kTreeNodes], to[kTreeNodes];   // row 0 of kv head 0: page * Hkv * page_tokens + token; -1: not to be moved
  int32_t* len_at = c.len + (size_t)blockIdx.y * c.max_seqs + sq.seq;
  const int len = load_chained(len_at), n = sq.n;
  if (threadIdx.x < 2 * n) {
    const int k = threadIdx.x >> 1;
    const int pos = len + (threadIdx.x & 1 ? k : (int)sq.path[k]), slot = pos / c.page_tokens;
    int64_t at = -1;
    int32_t pg;
    if (slot >= c.table_stride) set_status(c.status, RELUX_ERR_OVERFLOW);
    else if (page_of(c.table, c.table_stride, sq.seq, slot, c.num_pages, c.status, &pg)) at = (int64_t)pg * c.Hkv * c.page_tokens + (pos - slot * c.page_tokens);
    (threadIdx.x & 1 ? to : from)[k] = at;
  }
  __syncthreads();
  constexpr int kAtOnce = 4;
  auto move = [&](auto* base, size_t step, int e0) {   // element e0 of every row of the path; `step` elements from row to row
    for (int k0 = 0; k0 < n; k0 += kAtOnce) {
      typename std::remove_reference<decltype(*base)>::type x[kAtOnce];
#pragma unroll
      for (int q = 0; q < kAtOnce; q++)
        if (k0 + q < n && from[k0 + q] >= 0) x[q] = load_chained(base + from[k0 + q] * step + e0);
#pragma unroll
      for (int q = 0; q < kAtOnce; q++)
        if (k0 + q < n && from[k0 + q] >= 0 && to[k0 + q] >= 0 && from[k0 + q] != to[k0 + q]) base[to[k0 + q] * step + e0] = x[q];
    }
  };
  const int per_row = c.row_bytes / 16, per_kind = c.Hkv * per_row;
  for (int u = threadIdx.x; u < 2 * per_kind; u += blockDim.x) {
    const int which = u >= per_kind, e = u - which * per_kind, h = e / per_row;
    uint4* base = reinterpret_cast<uint4*>((which ? c.v : c.k) + (size_t)blockIdx.y * c.layer_bytes);
    move(base, per_row, h * c.page_tokens * per_row + (e - h * per_row));
  }
  if (c.scales) {   // [page][kv head][K, V][token]: the same places with two rows of scales a kv head
    float* base = c.scales + (size_t)blockIdx.y * c.layer_scales;
    for (int u = threadIdx.x; u < 2 * c.Hkv; u += blockDim.x) {
      auto place = [&](int64_t at) { const int64_t pg = at / (c.Hkv * c.page_tokens); return pg * (2 * c.Hkv * c.page_tokens) + (at - pg * (c.Hkv * c.page_tokens)) + (int64_t)u * c.page_tokens; };
      for (int k = 0; k < n; k++)
        if (from[k] >= 0 && to[k] >= 0 && from[k] != to[k]) base[place(to[k])] = load_chained(base + place(from[k]));
    }
  }
  if (threadIdx.x == 0) *len_at = len + n;
  fence_chained_writes();
}

template <int N>
int32_t launch_commit(Pool* p, const CommitCommon& c, const CommitSeq* seqs, int n, int layers) {
  CommitParams<N> prm;
  prm.c = c;
  memcpy(prm.seqs, seqs, sizeof(CommitSeq) * n);
  const int units = 2 * c.Hkv * (c.row_bytes / 16), threads = std::max(2 * kTreeNodes, std::min(256, (units + 31) / 32 * 32));
  RELUX_CUDA_TRY(launch_chained(p->tune.get(RELUX_TUNE_CHAINED_LAUNCHES) != 0, tree_commit_kernel<N>, dim3(n, layers), dim3(threads), 0, p->dev->stream, prm));
  count_launch(p->dev);
  return RELUX_OK;
}

}  // namespace

int32_t do_tree_commit(Pool* p, const relux_tree_commit_args* a) {
  if (!a) { set_error("nil argument struct"); return RELUX_ERR_INVALID_ARG; }
  const relux_pool_params& prm = p->prm;
  if (prm.kind != RELUX_POOL_GQA) { set_error("relux_gqa_tree_commit needs a GQA pool"); return RELUX_ERR_INVALID_ARG; }
  if (a->layer >= prm.num_layers) { set_error("layerIdx=%d out of range [0, %d)", a->layer, prm.num_layers); return RELUX_ERR_INVALID_ARG; }
  if (!a->path || !a->path_len || a->path_stride <= 0) { set_error("tree_commit: nil path or path_len, or path_stride <= 0"); return RELUX_ERR_INVALID_ARG; }
  for (int32_t r : a->reserved)
    if (r) { set_error("reserved fields must be zero"); return RELUX_ERR_INVALID_ARG; }
  SeqBatch sb;
  int32_t rc = stage_batch(p, a->n_seqs, a->seq_ids, a->path_len, 1, &sb, false);
  if (rc) return rc;
  const int l0 = a->layer < 0 ? 0 : a->layer, l1 = a->layer < 0 ? prm.num_layers : a->layer + 1;
  std::vector<CommitSeq> seqs;
  seqs.reserve(sb.n_seqs);
  for (int i = 0; i < sb.n_seqs; i++) {
    const int n = sb.rows[i];
    if (n > a->path_stride || n > kTreeNodes) {
      set_error("tree_commit: path of %d nodes for sequence %d (path_stride=%d, at most %d)", n, sb.seq[i], a->path_stride, kTreeNodes);
      return RELUX_ERR_INVALID_ARG;
    }
    if (n == 0) continue;
    CommitSeq s{sb.seq[i], n, {}};
    const int32_t* path = a->path + (size_t)i * a->path_stride;
    for (int k = 0; k < n; k++) {
      if (path[k] < 0 || path[k] >= kTreeNodes || (k && path[k] <= path[k - 1])) {
        set_error("tree_commit: path[%d][%d]=%d: nodes are numbers of [0, %d), each larger than the one before it", i, k, path[k], kTreeNodes);
        return RELUX_ERR_INVALID_ARG;
      }
      s.path[k] = (uint8_t)path[k];
    }
    seqs.push_back(s);
  }
  for (int l = l0; l < l1; l++) {
    const int32_t* len = &p->h_len[(size_t)l * prm.max_seqs];
    for (const CommitSeq& s : seqs)
      if (len[s.seq] + s.path[s.n - 1] >= p->seq_pages[s.seq] * prm.page_tokens) {
        set_error("tree_commit: node %d lies past the capacity of sequence %d on layer %d", (int)s.path[s.n - 1], s.seq, l);
        return RELUX_ERR_OVERFLOW;
      }
  }
  CommitCommon c{};
  c.layer_bytes = p->layer_elems * p->elem_bytes();
  c.layer_scales = p->int8 ? p->layer_scales() : 0;
  c.table = p->d_table;
  c.table_stride = prm.max_pages_per_seq;
  c.num_pages = prm.num_pages;
  c.page_tokens = prm.page_tokens;
  c.Hkv = prm.gqa_num_kv_heads;
  c.row_bytes = (int)(prm.gqa_head_dim * p->elem_bytes());
  c.max_seqs = prm.max_seqs;
  c.status = p->d_status;
  constexpr int kGridY = 65535;
  for (int l = l0; l < l1; l += kGridY)
    for (size_t at = 0; at < seqs.size(); at += kSeqsLarge) {
      const int n = (int)std::min<size_t>(kSeqsLarge, seqs.size() - at), layers = std::min(kGridY, l1 - l);
      c.k = (char*)p->rows_at(l, 0);
      c.v = (char*)p->rows_at(l, 1);
      c.scales = p->int8 ? p->scales_at(l) : nullptr;
      c.len = p->d_len + (size_t)l * prm.max_seqs;
      rc = n <= kSeqsSmall ? launch_commit<kSeqsSmall>(p, c, &seqs[at], n, layers) : launch_commit<kSeqsLarge>(p, c, &seqs[at], n, layers);
      if (rc) return rc;
    }
  for (int l = l0; l < l1; l++) {
    int32_t* len = &p->h_len[(size_t)l * prm.max_seqs];
    for (const CommitSeq& s : seqs) {
      if (p->compat) note_set_len(p, l, s.seq, len[s.seq], len[s.seq] + s.n);
      len[s.seq] += s.n;
    }
  }
  return RELUX_OK;
}

}  // namespace relux
