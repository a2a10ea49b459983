// What lora.cu asks of lora_gemm.cu.
#pragma once

#include "internal.h"

namespace relux {

constexpr int kNarrowRows = 16;     // calls of up to so many rows: one block of rows, rounded by lora_gemm_kernel, adapters on the CUDA cores
constexpr int kMaxLoraTiles = 1024; // row tiles of a longer call

// Tiles of up to 128 neighbouring rows of one adapter.
struct LoraTiles {
  int32_t n;
  int32_t row[kMaxLoraTiles], slot[kMaxLoraTiles];
  int16_t rows[kMaxLoraTiles];
};

// out = x W (+ out) + t B_s^T.  x: bf16 [M][K], the caller's or what the launch before this one has rounded; nullptr: up to kNarrowRows float32 rows of the
// caller's.  Without tiles (up to kNarrowRows rows): row_slots
// [M], t [M][rank] without factors; with tiles: t as two bf16 halves [M][rank], factors included.
int32_t launch_lora_gemm(Pool* p, const relux_matmul_lora_args* a, const uint16_t* x, const int16_t* row_slots, const LoraTiles* tiles, const float* t,
                         const uint16_t* t_hi, const uint16_t* t_lo);

}  // namespace relux
