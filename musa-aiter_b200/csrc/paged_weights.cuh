// What the kernels for few and for many rows of the attention weights share.
#pragma once

#include "paged_attn_tc.cuh"

namespace mak {

struct WeightParams {
  PagedParams a;
  const float* lse;     // [rows][heads], row stride lse_sr
  float* sums;          // [sequences or more][heads][max_tokens]
  const int32_t* rows;  // row of sums of each sequence, or null
  int64_t lse_sr, sum_sr, sum_sh, sum_rows;
  int32_t max_tokens, add;
  float scale;
};

// Row of sums of a sequence, -1: none.
__device__ __forceinline__ int64_t sum_row(const WeightParams& w, int s) {
  const int64_t r = w.rows != nullptr ? __ldg(w.rows + s) : s;
  return r >= 0 && r < w.sum_rows ? r : -1;
}

bool weights_tc_fits(const WeightParams& w);
// `work`: scratch of one number per sequence.
int launch_weights_tc(const WeightParams& w, int head_dim, bool bf16, const char* name, const CUtensorMap& k, int64_t* work, cudaStream_t st);

}  // namespace mak
