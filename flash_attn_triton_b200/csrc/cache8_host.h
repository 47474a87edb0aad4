// The 8-bit KV cache: what its launchers hand to one another.
#pragma once
#include <cuda_runtime.h>

#include "../../include/fa_b200.h"

namespace fa {

// Tokens to append; index 0 = keys, 1 = values.
struct Append8 {
  const void* x[2];
  int64_t x_stride[2][3];              // (sequence, token, head)
  void* cache[2];
  int64_t c_stride[2][3];              // (page, row, head)
  float* scale[2];
  int64_t s_stride[2][3];              // (page, block, head)
  int64_t tokens, longest_run;
  int heads, head_dim, dim_log2;
  int block, block_shift, page_size, page_shift, num_pages;   // shifts: -1 where no power of two
  const int64_t* slots;                // packed tokens
};
struct AppendGeom {
  int span;                            // tokens whose runs a CTA takes
  int per_y, warps_log2;
  unsigned grid_x, grid_y;
};

Append8 append_of(const fa_decode_args& call, const fa_cache8& cache);
// call: a cache call (null: packed tokens).  host, dev, check_here: value checks as in cache_append_kernel.
int append8_launch(const Append8& p, const fa_decode_args* call, int dtype, int code, int device, uint32_t* host, uint32_t* dev,
                   bool check_here, cudaStream_t st);

}  // namespace fa
