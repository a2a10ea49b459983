// Rows of the 8-bit grouped-query cache, and per-warp attention over one 64-token page of them (gqa_stream_kernel.cuh,
// gqa_tree_sm100.cu, append.cu).
//
// A row of a kv head, 128 values x of K or of V, is 128 codes c (int8) and a float32 scale s:
//   a = max |x|,  s = a / 127,  c = x * (127 / a) to the nearest whole number, even where two are as near
// with every operation rounded to float32.  |c| <= 127: x * (127 / a) is at most 127 (1 + 2^-23).  A row with a < 1e-36, whose 127 / a might not be
// finite, is s = 0, c = 0.  A row that holds an infinity or a NaN is s = NaN, c = 0: a code is always a number, so a row that no query sees adds
// exactly nothing to a tensor-core product, whatever it held (0 * c, where bf16 rows have 0 * NaN).
// Whole numbers and not an 8-bit float: the same bytes, and a fourth of the error (half a step of 1 / 127 of the row's largest value against 2^-4 of each
// value); both are exact in binary16 and bfloat16.
//
// A page of a kv head is 64 rows of 128 bytes of K codes, the same of V, and 2 x 64 scales.  Both kinds of rows arrive by TMA with the 128-byte swizzle and
// are read 16 bytes a thread without bank conflicts, straight into the B fragments of mma.sync m16n8k16: what a fragment wants side by side are
// four consecutive K indices of one column, and the order of the indices is the reader's own as long as A has the same.
//   K: thread (n, c) = (lane / 4, lane % 4) takes bytes 32 c .. 32 c + 31 of token n of a block of eight; K slice ks is its word ks.
//   V: thread (n, c) takes bytes 16 n .. 16 n + 15 of tokens 2c, 2c + 1, 2c + 8, 2c + 9; output block j's column n is dim 16 n + j.
// A code is stored as c + 128: below the exponent of 1024 that is a binary16 number, and one subtraction (two instructions for two codes) makes it c, which
// binary16 holds exactly.  Queries are brought to binary16 with a power of two per row, which keeps 11 bits of a float32 query where bf16 keeps 8.  P carries
// s^v over a power of two that grows with the largest s^v seen so far (O is then rescaled as for a new maximum): 11 bits of it, 2^20 between the
// largest row and one that may lose bits.  (P s^v in bf16, whose range needs no unit, was off by 2.5e-3 of the result where this is 1.7e-3, the rounding of a
// bf16 output alone, and takes four instructions for two codes.)
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "gqa_parts.cuh"
#include "softmax_parts.cuh"

namespace relux {

constexpr int kInt8StageBytes = 2 * kGqaPageTok * kGqaD;                      // K codes, V codes
constexpr int kInt8ScaleBytes = 2 * kGqaPageTok * (int)sizeof(float);         // K scales, V scales
constexpr float kInt8Tiny = 1e-36f;
constexpr uint32_t kInt8Zeros = 0x80808080u;   // four codes of 0

// Untiled bulk copy global -> shared (multiples of 16 bytes), completion on an mbarrier of this CTA.
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem_dst)),
               "l"(__cvta_generic_to_global(src)), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// ---- a row's values, eight a lane ----
__device__ __forceinline__ void load8(float (&x)[8], const float* src) {
  const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void load8(float (&x)[8], const uint16_t* src) {
  const uint4 a = *reinterpret_cast<const uint4*>(src);
  x[0] = bf16_lo(a.x); x[1] = bf16_hi(a.x); x[2] = bf16_lo(a.y); x[3] = bf16_hi(a.y);
  x[4] = bf16_lo(a.z); x[5] = bf16_hi(a.z); x[6] = bf16_lo(a.w); x[7] = bf16_hi(a.w);
}
// Largest magnitude of a row, as bits (larger for an infinity or a NaN than for any number), by the 16 lanes that hold it; the warp is converged.
__device__ __forceinline__ float max_nan(float a, float b) {   // a NaN stays one
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ uint32_t row_top(const float (&x)[8]) {
  float m[4];
#pragma unroll
  for (int i = 0; i < 4; i++) m[i] = max_nan(fabsf(x[i]), fabsf(x[i + 4]));
  float top = max_nan(max_nan(m[0], m[1]), max_nan(m[2], m[3]));
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  return __float_as_uint(top);
}
struct Int8Row {
  uint2 codes;   // this lane's eight
  float scale;
};
// The warp is converged.  Of the two divisions a row needs, its even lanes do one and its odd lanes the other.
__device__ __forceinline__ Int8Row int8_quantise(const float (&x)[8], uint32_t top) {
  const bool odd = threadIdx.x & 1, some = top < 0x7F800000u && __uint_as_float(top) >= kInt8Tiny;
  const float a = some ? __uint_as_float(top) : 127.f;
  const float mine = __fdiv_rn(odd ? a : 127.f, odd ? 127.f : a), other = __shfl_xor_sync(0xffffffffu, mine, 1);
  const float inv = odd ? other : mine;
  Int8Row r;
  r.scale = some ? (odd ? mine : other) : top >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : 0.f;
  // 1.5 * 2^23 more is rounded to a whole number, as a conversion would (at a fourth of the rate), and has it in its low bits.  (One value at a time: a packed
  // product and a packed sum came out as one rounding, which takes 63.5 of half of the largest value to 63, not 64.)
  uint32_t c[8], w[2];
#pragma unroll
  for (int i = 0; i < 8; i++) c[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[i], inv), 12582912.f));
#pragma unroll
  for (int h = 0; h < 2; h++) w[h] = __byte_perm(__byte_perm(c[4 * h], c[4 * h + 1], 0x0040), __byte_perm(c[4 * h + 2], c[4 * h + 3], 0x0040), 0x5410) ^ kInt8Zeros;
  r.codes = some ? make_uint2(w[0], w[1]) : make_uint2(kInt8Zeros, kInt8Zeros);
  return r;
}
template <typename T>
__device__ __forceinline__ Int8Row int8_row(const T* src) {
  float x[8];
  load8(x, src);
  return int8_quantise(x, row_top(x));
}

// ---- codes -> matrix operands ----
// Two bytes under 0x64, binary16 1024 + (c + 128) -> c.
__device__ __forceinline__ uint32_t int8x2_to_f16(uint32_t t) {
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&t), __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&x);
}
// Four codes -> two pairs of binary16.
__device__ __forceinline__ void int8x4_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  lo = int8x2_to_f16(__byte_perm(w, 0x64646464u, 0x4140));
  hi = int8x2_to_f16(__byte_perm(w, 0x64646464u, 0x4342));
}
__device__ __forceinline__ uint32_t round_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The unit of the values' scales: those below `limit` come below 2^kUp times `down`.  For the largest scale of new rows that reaches the limit.
struct ValueUnit {
  float limit = 0.f, down = 1.f;
  template <int kUp>
  __device__ __forceinline__ void grow(float top) {
    const int e = max((int)(__float_as_uint(top) >> 23), kUp + 1);                // 2^(e - 127) <= top < 2^(e - 126)
    limit = __uint_as_float((uint32_t)min(e + 1, 254) << 23);
    down = __uint_as_float((uint32_t)(min(253 + kUp - e, 253)) << 23);            // 2^(kUp - 1 - (e - 127))
  }
};

// ---- queries ----
// The power of two that brings a row's largest value, of bits `top`, to [2^14, 2^15), and its inverse.  (Not rows of zeros or of subnormal numbers.)
__device__ __forceinline__ void query_factor(uint32_t top, float& up, float& down) {
  const int k = min(141 - (int)(top >> 23), 126);
  up = __uint_as_float((uint32_t)(127 + k) << 23);
  down = __uint_as_float((uint32_t)(127 - k) << 23);
}
// What a score is multiplied by: the softmax scale (times log2 e) over the row's power of two.  Not nothing, even of a row of zeros, whose power is the largest, under a
// scale below 2^-23: minus infinity, a hidden key's score, times nothing is NaN.
__device__ __forceinline__ float score_factor(float scale_log2, float down) { return fmaxf(scale_log2 * down, __uint_as_float(1u)); }
// Row of queries in shared memory: 128 binary16 values, the row's factor (what a score of theirs is multiplied by, softmax scale and log2 e included),
// and what the row sees of the new rows.  By 16 lanes of a converged warp, eight dims each.
__device__ __forceinline__ void int8_put_query(uint16_t* row, int ch, bool there, const void* q, size_t off, bool q_bf16, float scale_log2) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; i++) x[i] = 0.f;
  if (there) {
    if (q_bf16) load8(x, reinterpret_cast<const uint16_t*>(q) + off);
    else load8(x, reinterpret_cast<const float*>(q) + off);
  }
  float up, down;
  query_factor(row_top(x), up, down);
  if (!there) return;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const __half2 h = __floats2half2_rn(x[2 * i] * up, x[2 * i + 1] * up);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(row + ch) = make_uint4(w[0], w[1], w[2], w[3]);
  if (ch == 0) *reinterpret_cast<float*>(row + kGqaD) = score_factor(scale_log2, down);
}
// 16 such rows -> A fragments in the order of K's bytes, and the factors of this lane's two rows.
__device__ __forceinline__ void int8_load_q(uint32_t (&qa)[8][4], float (&q_scale)[2], const uint16_t* qs, int lane) {
#pragma unroll
  for (int hf = 0; hf < 2; hf++) {
    const uint16_t* row = qs + ((lane >> 2) + 8 * hf) * kGqaQStride;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint4 w = *reinterpret_cast<const uint4*>(row + 32 * (lane & 3) + 8 * i);
      qa[2 * i][hf] = w.x;
      qa[2 * i][2 + hf] = w.y;
      qa[2 * i + 1][hf] = w.z;
      qa[2 * i + 1][2 + hf] = w.w;
    }
    q_scale[hf] = *reinterpret_cast<const float*>(row + kGqaD);
  }
}

// D(16x8,f32) += A(16x16,f16,row) * B(16x8,f16,col)
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A maximum is followed only once it has grown by more than this (base 2): with random scores three visits of a page in five found a larger one, and
// moved 64 sums for it.
constexpr float kInt8Lazy = 8.f;
constexpr int kInt8Up = 7;   // P s^v is kept below 2^(kInt8Up + kInt8Lazy), the upper end of binary16

// Scores of a warp's 16 tokens of a page, but for the queries' factors.
__device__ __forceinline__ void int8_scores(float (&s)[2][4], const uint32_t (&qa)[8][4], const uint8_t* page, const float* scales, int tb, int lane) {
  const int n = lane >> 2, c = lane & 3;
  float odd[2][4];   // even and odd K slices: two chains of dependent MMAs a block
#pragma unroll
  for (int nt = 0; nt < 2; nt++) {
#pragma unroll
    for (int e = 0; e < 4; e++) s[nt][e] = odd[nt][e] = 0.f;
    const uint32_t row = tb + nt * 8 + n;
    const uint4 k0 = *reinterpret_cast<const uint4*>(page + swz128(row, 2 * c)), k1 = *reinterpret_cast<const uint4*>(page + swz128(row, 2 * c + 1));
    const uint32_t w[8] = {k0.x, k0.y, k0.z, k0.w, k1.x, k1.y, k1.z, k1.w};
#pragma unroll
    for (int ks = 0; ks < 8; ks++) {
      uint32_t b0, b1;
      int8x4_to_f16(w[ks], b0, b1);
      mma_f16_16816(ks & 1 ? odd[nt] : s[nt], qa[ks], b0, b1);
    }
    const float2 sk = *reinterpret_cast<const float2*>(scales + tb + nt * 8 + 2 * c);
#pragma unroll
    for (int e = 0; e < 4; e++) s[nt][e] = (s[nt][e] + odd[nt][e]) * (e & 1 ? sk.y : sk.x);
  }
}

// gqa_consume_page for a page of codes whose scores are in s.  next_scores(s) then computes those of the next page, beside this one's exponentials and values:
// with two such warps on a scheduler, one page's chain of latencies after another left it idle half of the time.
template <bool kTree, typename Next>
__device__ __forceinline__ void int8_consume_page(GqaState<1>& st, ValueUnit& unit, float (&s)[2][4], const float (&q_scale)[2], const uint8_t* page,
                                                  const float* scales, int tb, int tok0, int T, int S, int g, int causal, int lane, int row0,
                                                  const TreeRows& tree, Next next_scores) {
  const int n = lane >> 2, c = lane & 3;
  float sv[2][2];
#pragma unroll
  for (int nt = 0; nt < 2; nt++) {
    const float2 s2 = *reinterpret_cast<const float2*>(scales + kGqaPageTok + tb + nt * 8 + 2 * c);
    sv[nt][0] = s2.x;
    sv[nt][1] = s2.y;
  }
  // rows that nobody sees yet, or ever, have a part in the unit too if they are the sequence's; what lies behind T may hold anything
  const int there = T - tok0 - 2 * c;
  float top = fmaxf(fmaxf(there > 0 ? sv[0][0] : 0.f, there > 1 ? sv[0][1] : 0.f), fmaxf(there > 8 ? sv[1][0] : 0.f, there > 9 ? sv[1][1] : 0.f));   // NaN drop out
  uint32_t hidden = 0;   // bit 4 hf + 2 nt + e
  const bool need_mask = tok0 + 16 > (kTree ? tree.len0 : T - (causal ? S : 0));
  if (need_mask) {
#pragma unroll
    for (int hf = 0; hf < 2; hf++) {
      const int limit = causal ? (T - S + (row0 + hf * 8 + n) / g) : (T - 1);   // last visible token
#pragma unroll
      for (int nt = 0; nt < 2; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int tok = tok0 + nt * 8 + 2 * c + e;
          if (kTree ? tree.hides(hf, tok) : tok > limit || tok >= T) {
            hidden |= 1u << (4 * hf + 2 * nt + e);
            s[nt][hf * 2 + e] = -INFINITY;
          }
        }
    }
  }
  float mx[2];   // of this lane's tokens
  bool grow = false;
#pragma unroll
  for (int hf = 0; hf < 2; hf++) {
    mx[hf] = fmaxf(fmaxf(s[0][hf * 2], s[0][hf * 2 + 1]), fmaxf(s[1][hf * 2], s[1][hf * 2 + 1])) * q_scale[hf];
    grow |= mx[hf] > st.m[0][hf] + kInt8Lazy;
  }
  if (__any_sync(0xffffffffu, grow || top >= unit.limit)) {
    float shrink = 1.f;
    top = warp_max(top);
    if (top >= unit.limit) {
      const float before = unit.down;
      const bool first = unit.limit == 0.f;
      unit.grow<kInt8Up>(top);
      if (!first) shrink = unit.down / before;
    }
#pragma unroll
    for (int hf = 0; hf < 2; hf++) {
      mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 1));
      mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 2));
      const float m_new = fmaxf(st.m[0][hf], mx[hf]);
      float alpha = (m_new == -INFINITY) ? 0.f : gqa_ex2(st.m[0][hf] - m_new);
      st.m[0][hf] = m_new;
      st.l[0][hf] *= alpha;
      alpha *= shrink;
#pragma unroll
      for (int j = 0; j < 16; j++) {
        st.o[0][j][hf * 2] *= alpha;
        st.o[0][j][hf * 2 + 1] *= alpha;
      }
    }
  }
  float s_next[2][4];
  next_scores(s_next);
  // P times the values' scales over their unit, rounded to binary16: 2^-11 of each, or 2^-25 where the largest come to 2^7 and more
  uint32_t pa[4];
  float p[2][4];
#pragma unroll
  for (int hf = 0; hf < 2; hf++) {
    const float neg_m = (st.m[0][hf] == -INFINITY) ? 0.f : -st.m[0][hf];
    float ps = 0.f;
#pragma unroll
    for (int nt = 0; nt < 2; nt++) {
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const float x = gqa_ex2(fmaf(s[nt][hf * 2 + e], q_scale[hf], neg_m));
        ps += x;
        p[nt][hf * 2 + e] = x * (sv[nt][e] * unit.down);
      }
    }
    st.l[0][hf] += ps;
  }
  if (need_mask)   // the scale of a hidden row may be NaN
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (hidden >> i & 1u) p[i >> 1 & 1][(i >> 2) * 2 + (i & 1)] = 0.f;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    pa[i] = round_f16x2(p[i >> 1][(i & 1) * 2], p[i >> 1][(i & 1) * 2 + 1]);
#pragma unroll
    for (int nt = 0; nt < 2; nt++) s[nt][i] = s_next[nt][i];
  }
  const uint8_t* vt = page + kGqaPageTok * kGqaD;
  uint4 v[4];
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = *reinterpret_cast<const uint4*>(vt + swz128(tb + 2 * c + (i & 1) + (i >> 1) * 8, n));
#pragma unroll
  for (int w = 0; w < 4; w++) {
    uint32_t x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = w == 0 ? v[i].x : w == 1 ? v[i].y : w == 2 ? v[i].z : v[i].w;
    const uint32_t a01 = __byte_perm(x[0], x[1], 0x5140), a23 = __byte_perm(x[0], x[1], 0x7362);
    const uint32_t b01 = __byte_perm(x[2], x[3], 0x5140), b23 = __byte_perm(x[2], x[3], 0x7362);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t sel = j & 1 ? 0x4342 : 0x4140;
      mma_f16_16816(st.o[0][4 * w + j], pa, int8x2_to_f16(__byte_perm(j < 2 ? a01 : a23, 0x64646464u, sel)),
                    int8x2_to_f16(__byte_perm(j < 2 ? b01 : b23, 0x64646464u, sel)));
    }
  }
}

// gqa_store_state: output block j's column 2c + e is dim 16 (2c + e) + j.
__device__ __forceinline__ void int8_store_state(const GqaState<1>& st, const ValueUnit& unit, float* dst0, int rows, int lane, bool alive) {
  const float up = 1.f / unit.down;
#pragma unroll
  for (int hf = 0; hf < 2; hf++) {
    float l = st.l[0][hf];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    const int row = hf * 8 + (lane >> 2);
    if (row >= rows) continue;
    float* dst = dst0 + row * kGqaStateStride;
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
      for (int j = 0; j < 16; j += 4)
        *reinterpret_cast<float4*>(dst + 16 * (2 * (lane & 3) + e) + j) =
            make_float4(st.o[0][j][hf * 2 + e] * up, st.o[0][j + 1][hf * 2 + e] * up, st.o[0][j + 2][hf * 2 + e] * up, st.o[0][j + 3][hf * 2 + e] * up);
    if ((lane & 3) == 0) {
      dst[kGqaD] = alive ? st.m[0][hf] : -INFINITY;
      dst[kGqaD + 1] = alive ? l : 0.f;
    }
  }
}

}  // namespace relux
