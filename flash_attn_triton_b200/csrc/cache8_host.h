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
  int per_y, warps_log2, held;
  unsigned grid_x, grid_y;
};

// A division by n that kernels make by a product.
struct Div32 {
  uint32_t m;
  int shift;
};
inline Div32 div_by(int n) {
  int l = 0;
  while ((1ll << l) < n) ++l;
  const int shift = 31 + l;
  return Div32{(uint32_t)(((1ull << shift) + (uint64_t)n - 1) / (uint64_t)n), shift};
}

// Decode: how a call is cut, and where its cache lies (strides in 16 bytes: an address is then two 32-bit products).
struct Geom8 {
  int ranges;      // CTAs per unit
  int rows;        // of the workspace: pieces
  int splits;      // 0: ranges sized on the device; else that many pieces of every sequence
  int resident;    // CTAs the GPU runs at a time
  int max_tiles;   // tiles of a full cache
  int row_groups;  // ceil(seqlen_q * group / rows of a unit)
  Div32 page, block;
  uint32_t k_page, k_row, v_page, v_row;
};

Append8 append_of(const fa_decode_args& call, const fa_cache8& cache);
// call: a cache call (null: packed tokens).  host, dev, check_here: value checks as in cache_append_kernel.
int append8_launch(const Append8& p, const fa_decode_args* call, int dtype, int code, int device, uint32_t* host, uint32_t* dev,
                   bool check_here, cudaStream_t st);

}  // namespace fa
