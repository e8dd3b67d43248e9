// The products of a few rows (few_rows.cu), as the entry points of the grouped and the block-scaled products call them.
#pragma once
#include "moe_common.cuh"

namespace comfy_b200 {

constexpr int kFewRows = 16, kFewRowsBlock = 8;                      // rows that one pass over the weights serves
constexpr int kFewRowsQuantise = COMFY_MOE_FEW_ROWS_BLOCK;           // block-scaled, quantised on the way
constexpr int kFewQuantiseMaxK = COMFY_MOE_FEW_ROWS_BLOCK_MAX_K;     // what of them fits into shared memory

struct FewParams {
  const uint8_t* x;
  const uint8_t* w;
  uint8_t* out;
  const int32_t* offsets;
  const int32_t* counts;
  const float* ws;                             // block-scaled: scales of the weights,
  const float* xs;                             // and of the rows [blocks][ld_xs], if x holds quantised ones
  const void* bias;
  long long ld_x, ld_w, w_group, ld_out;       // bytes
  long long ws_group, ld_xs;
  int groups, rows, n, k, zero_unused;
};

int launch_few_rows(const FewParams& p, bool fp16, cudaStream_t stream);
int launch_few_rows_block(const FewParams& p, bool fp16, cudaStream_t stream);

}  // namespace comfy_b200
