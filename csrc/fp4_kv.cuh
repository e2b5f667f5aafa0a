// Shared by the 4-bit K / V cache's kernels: the page format and the attention arguments.
//
// Page of R rows of one sequence, for each K / V head a slab of R * d * 17 / 16 bytes:
//   K codes (R x d/2) | V codes (R x d/2) | K scales (R x d/32) | V scales (R x d/32)
// Byte j of a row's codes holds dim 2j (low four bits) and 2j + 1.  A code is E2M1 (sign, two
// exponent bits, one mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6); 32 dims share the scale
// 2^(byte - 127).  The scale's exponent is the smallest e with amax <= 6 * 2^e, at least -126;
// byte 255 marks a block that held a NaN or an infinity and reads as NaN.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace sv4 {

struct Fp4AttnArgs {
  const void* q;
  int64_t q_b, q_h, q_t;  // strides in elements
  const uint8_t* pages;
  int64_t page_stride, n_pages;
  const int* table;
  const int* lengths;
  const float* sink;
  void* out;  // (B, H, T, d) contiguous
  // what is cut between blocks: block i has two parts of `rows` rows, (2 i + which) * rows ..
  float* part_out;  // (blocks, 2, rows, d): mean of v under the part's own weights
  float2* part_ml;  // (blocks, 2, rows): maximum score (log2 units), sum of p
  int B, H, Hk, T, P, R, slab, window, blocks;
  float scale, softcap;
  int* err;
};

// How a kernel divides the work: a bound on its units, the blocks of its grid, the rows of a part.
struct Fp4AttnPlan {
  int64_t units;
  int blocks, rows;
};

// Few query rows per K / V head: head_dim d (32, 64, 128), q in fp16 or bf16.
Fp4AttnPlan fp4_attn_rows_plan(const Fp4AttnArgs& a, int d);
void fp4_attn_rows(const Fp4AttnArgs& a, int d, bool half, cudaStream_t stream);

// Many: head_dim 64 or 128.
Fp4AttnPlan fp4_attn_tile_plan(const Fp4AttnArgs& a);
void fp4_attn_tile(const Fp4AttnArgs& a, int d, bool half, cudaStream_t stream);

}  // namespace sv4
