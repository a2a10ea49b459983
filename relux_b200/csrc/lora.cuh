// What lora.cu asks of lora_gemm.cu.
#pragma once

#include "common.cuh"
#include "internal.h"

namespace relux {

constexpr int kNarrowRows = 16;     // calls of up to so many rows: one block of rows, float32 ones split by lora_gemm_kernel, adapters on the CUDA cores
constexpr int kNarrowSums = 512;    // rows x rank of them, of float32 ones half as many
constexpr int kOneT = 16;           // rows x rank of calls in one launch
constexpr int kMaxLoraTiles = 1024; // row tiles of a longer call

// Tiles of up to 128 neighbouring rows of one adapter.
struct LoraTiles {
  int32_t n;
  int32_t row[kMaxLoraTiles], slot[kMaxLoraTiles];
  int16_t rows[kMaxLoraTiles];
};

// f v as two bf16 halves, 16 bits of it.  Both have its sign, and not both are zero where it is not (down to 2^-133): the first is the largest of smaller magnitude, the second the rest.  So an infinity that
// they are multiplied with comes out as the formula has it (with the nearest value first the rest is zero or of the other sign, and the sum of both products NaN).  Of an infinity the
// first half is the largest number and the rest the infinity; a NaN's rest is NaN.  The rest is up to 2^-7 of the value, rounded by 2^-9 of itself.
__device__ __forceinline__ void split_halves(float4 v, float f, uint2& hi, uint2& lo) {
  auto times = [f](float x) { return __fadd_rn(__fmul_rn(x, f), 0.f); };   // never -0, of which there is no smaller magnitude
  auto first = [](float x) { return (max(__float_as_uint(x), 1u) - 1u) & 0xFFFF0000u; };
  v = make_float4(times(v.x), times(v.y), times(v.z), times(v.w));
  const uint32_t x = first(v.x), y = first(v.y), z = first(v.z), w = first(v.w);
  hi = make_uint2(__byte_perm(x, y, 0x7632), __byte_perm(z, w, 0x7632));
  lo = make_uint2(round_bf16x2(v.x - __uint_as_float(x), v.y - __uint_as_float(y)), round_bf16x2(v.z - __uint_as_float(z), v.w - __uint_as_float(w)));
}

// out = x W (+ out) + t B_s^T.  x: bf16 [M][K], the caller's or what the launch before this one has rounded; nullptr: up to kNarrowRows float32 rows of the
// caller's.  Without tiles or t: lora_gemm_kernel takes t itself.  Without tiles (up to kNarrowRows rows): row_slots
// [M], t [M][rank] without factors; with tiles: t as two bf16 halves [M][rank], factors included.
int32_t launch_lora_gemm(Pool* p, const relux_matmul_lora_args* a, const uint16_t* x, const int32_t* row_slots, const LoraTiles* tiles, const float* t,
                         const uint16_t* t_hi, const uint16_t* t_lo);

// t = f_s x A_s^T of the rows of `tiles` as two bf16 halves [M][rank].  x: bf16 rows [M][K]; nullptr: the caller's float32 ones, which are rounded to `rounded` as well.
int32_t launch_lora_rows(Pool* p, const relux_matmul_lora_args* a, const LoraTiles& tiles, const uint16_t* x, uint16_t* rounded, uint16_t* t_hi, uint16_t* t_lo);

}  // namespace relux
