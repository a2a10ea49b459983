// What lora.cu asks of lora_gemm.cu.
#pragma once

#include "common.cuh"
#include "internal.h"

namespace relux {

constexpr int kNarrowRows = 16;     // calls of up to so many rows: one block of rows, float32 ones split by lora_gemm_kernel, adapters on the CUDA cores
constexpr int kOneT = 16;           // rows x rank of calls in one launch
constexpr int kMaxLoraTiles = 1024; // row tiles of a longer call

// Tiles of up to 128 neighbouring rows of one adapter.
struct LoraTiles {
  int32_t n;
  int32_t row[kMaxLoraTiles], slot[kMaxLoraTiles];
  int16_t rows[kMaxLoraTiles];
};

// f v as two bf16 halves, 16 bits of it.
__device__ __forceinline__ void split_halves(float4 v, float f, uint2& hi, uint2& lo) {
  auto rest = [](float x, float h) { return fabsf(h) < __uint_as_float(0x7F800000u) ? x - h : 0.f; };   // an infinity has no second half
  v.x *= f; v.y *= f; v.z *= f; v.w *= f;
  hi = make_uint2(round_bf16x2(v.x, v.y), round_bf16x2(v.z, v.w));
  lo = make_uint2(round_bf16x2(rest(v.x, bf16_lo(hi.x)), rest(v.y, bf16_hi(hi.x))), round_bf16x2(rest(v.z, bf16_lo(hi.y)), rest(v.w, bf16_hi(hi.y))));
}

// out = x W (+ out) + t B_s^T.  x: bf16 [M][K], the caller's or what the launch before this one has rounded; nullptr: up to kNarrowRows float32 rows of the
// caller's.  Without tiles or t: lora_gemm_kernel takes t itself.  Without tiles (up to kNarrowRows rows): row_slots
// [M], t [M][rank] without factors; with tiles: t as two bf16 halves [M][rank], factors included.
int32_t launch_lora_gemm(Pool* p, const relux_matmul_lora_args* a, const uint16_t* x, const int16_t* row_slots, const LoraTiles* tiles, const float* t,
                         const uint16_t* t_hi, const uint16_t* t_lo);

// t = f_s x A_s^T of the rows of `tiles` as two bf16 halves [M][rank].  x: bf16 rows [M][K]; nullptr: the caller's float32 ones, which are rounded to `rounded` as well.
int32_t launch_lora_rows(Pool* p, const relux_matmul_lora_args* a, const LoraTiles& tiles, const uint16_t* x, uint16_t* rounded, uint16_t* t_hi, uint16_t* t_lo);

}  // namespace relux
