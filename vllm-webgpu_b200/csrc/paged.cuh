// paged.cuh -- the paged key-value cache as the kernels see it, and the checks that the
// entry points over it share.
#pragma once

#include "common.cuh"

namespace ggufmm {

int record_cuda_status(cudaError_t e);  // capi.cu
int check_device();                     // capi.cu

constexpr int64_t kI32Max = (int64_t(1) << 31) - 1;

inline bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
// A stride in 16-bit elements that keeps 16-byte alignment and that a tensor map can hold (< 2^40 bytes).
inline bool stride16_ok(int64_t s, int64_t least) { return s >= least && s % 8 == 0 && s < (int64_t(1) << 39); }

// Shape and alignment of a cache [num_pages, kv_heads, page_size, head_dim] of 16-bit
// values; strides in elements, the innermost one 1.
inline int check_cache(const void* k, const void* v, int64_t dtype, int64_t kv_heads, int64_t head_dim,
                       int64_t page_size, int64_t num_pages, const int64_t* ks, const int64_t* vs) {
  if (!k || !v) return GGUFMM_ERR_ARG;
  if (dtype != GGUFMM_F16 && dtype != GGUFMM_BF16) return GGUFMM_ERR_DTYPE;
  if (head_dim < 8 || head_dim > GGUFMM_MAX_HEAD_DIM || head_dim % 8 || kv_heads < 1 || kv_heads > 65535 ||
      page_size < 8 || page_size > 65536 || page_size % 8 || num_pages < 1 || num_pages > kI32Max)
    return GGUFMM_ERR_SHAPE;
  if (!aligned_to(k, 16) || !aligned_to(v, 16)) return GGUFMM_ERR_ALIGN;
  for (int i = 0; i < 3; ++i) {
    if (ks[i] < head_dim || vs[i] < head_dim) return GGUFMM_ERR_SHAPE;
    if (!stride16_ok(ks[i], head_dim) || !stride16_ok(vs[i], head_dim)) return GGUFMM_ERR_ALIGN;
  }
  return GGUFMM_OK;
}

}  // namespace ggufmm
