// The kernel for many rows of the attention over paged 16-bit caches, as its entry point calls it.
#pragma once

#include "paged_attn.cuh"

namespace mak {

constexpr int64_t kPagedCounterBytes = 4096;  // of a workspace, at its beginning

int64_t paged_tc_partial_bytes();
int64_t paged_tc_plan_bytes();
bool paged_tc_fits(const PagedParams& p);
int paged_tc_box(int bs);  // tokens of the boxes that it loads
int launch_paged_tc(const PagedParams& p, int head_dim, bool bf16, const char* name, const CUtensorMap& k, const CUtensorMap& v, void* plan,
                    cudaStream_t st);
// A plane [num_blocks][block_size][num_heads][head_dim] as boxes of `tokens` tokens of one head, 64 columns of them, lines of
// 128 bytes swizzled.  `none`: an address for a plane without blocks.  False where strides make no tensor map.
bool paged_map(CUtensorMap* map, const uint16_t* base, int64_t sb, int64_t st, int64_t sh, int64_t num_blocks, int nh, int hd, int bs, bool bf16,
               int tokens, const void* none);
// A tensor map over 16-bit elements; strides in bytes.
bool paged_encode(CUtensorMap* map, const void* base, int rank, const int64_t* dims, const int64_t* strides, const uint32_t* box, bool bf16);

// Of the entry points.
int check_paged_cache(const mak_paged_cache_desc& c, bool values, const char* name);
int check_paged_workspace(const void* workspace, int64_t bytes, const char* name);
PagedParams paged_params(const mak_paged_cache_desc& c);
struct PagedSpace {
  int32_t* counters;
  void* plan;
  int64_t plan_bytes;
  float* partial;
};
PagedSpace paged_space(void* workspace);

}  // namespace mak
