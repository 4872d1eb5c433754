// Kernel parameters of the row operators (norm + rotation, the 4-bit append and read-back), shared by the kernels
// and the C-ABI layer.
#pragma once

#include "common.cuh"

namespace mlb {

struct RowArgs {
  const char *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;  // strides (tokens, heads) in elements
  char *q_out, *k_out;
  int64_t qo_st, qo_sh, ko_st, ko_sh;
  int64_t num_tokens;
  int h, hkv, rot;
  const int64_t* positions;
  const float* cos_sin;  // [num_positions][rot]: cos of rot / 2 angles, then sin
  int64_t num_positions;
  const char *q_weight, *k_weight;
  float eps;
  uint8_t *k_cache, *v_cache;
  const int64_t* slots;
  int64_t num_slots;
  int vec;  // every row start and stride is 16-byte aligned
  int32_t* err;
};

}  // namespace mlb
