// attn.cu -- attention over a paged key-value cache: ggufmm_paged_attention (one new
// token per sequence) and ggufmm_paged_prompt_attention (ragged causal prompts).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max),  j in [lo, hi)
//
// The reference runs a score, a softmax and an output shader over one sequence
// (vllm_webgpu/models/llama.py:314-326; shaders/generic/{attn_score,softmax,attn_output}.wgsl).
#include <cmath>

#include "paged.cuh"

namespace ggufmm {

size_t paged_decode_workspace(int64_t head_dim);  // attn_decode.cu
cudaError_t launch_paged_decode(const ggufmm_attention_args& p, void* workspace, cudaStream_t st);

namespace {

struct AttnArgs {
  ggufmm_attention_args p;
};

template <int DT>
__device__ __forceinline__ float ld16(const void* b, int64_t i) {
  return DT == GGUFMM_F16 ? __half2float(static_cast<const __half*>(b)[i])
                          : __bfloat162float(static_cast<const __nv_bfloat16*>(b)[i]);
}

// One warp per (query, head): lane l holds values l, l + 32, ... of the head.
template <int DT>
__global__ void __launch_bounds__(128) attn_simple_kernel(const __grid_constant__ AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  const ggufmm_attention_args& p = a.p;
  const int lane = threadIdx.x & 31;
  const int64_t b = blockIdx.z;
  const int head = static_cast<int>(blockIdx.y);
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int d = static_cast<int>(p.head_dim);
  const int kvh = head / static_cast<int>(p.q_heads / p.kv_heads);
  int64_t row = b, n = 1;
  if (p.q_starts) {
    const int32_t* qs = static_cast<const int32_t*>(p.q_starts);
    row = qs[b] + i;
    n = qs[b + 1] - qs[b];
    if (row < 0 || row >= p.total_q) n = 0;
  }
  if (i >= n) return;
  int64_t len = static_cast<const int32_t*>(p.lens)[b];
  const int64_t room = p.table_width * p.page_size;
  if (len > room) {
    len = room;
    if (lane == 0) atomicOr(&g_device_error, kErrIndex);
  }
  const int64_t hi = len - n + i + 1;
  int64_t lo = p.window > 0 ? hi - p.window : 0;
  if (lo < 0) lo = 0;
  const int32_t* tab = static_cast<const int32_t*>(p.tables) + b * p.table_row;
  float q[8], o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = lane + 32 * e;
    q[e] = c < d ? ld16<DT>(p.q, row * p.q_row + head * p.q_head + c) * static_cast<float>(p.scale) : 0.f;
    o[e] = 0.f;
  }
  float mx = -INFINITY, sum = 0.f;
  for (int64_t j = lo; j < hi; ++j) {
    const int64_t page = tab[j / p.page_size];
    float k[8], v[8], s = 0.f;
    const bool there = page >= 0 && page < p.num_pages;
    if (!there && lane == 0) atomicOr(&g_device_error, kErrIndex);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = lane + 32 * e;
      const bool in = there && c < d;
      k[e] = in ? ld16<DT>(p.k, page * p.k_page + kvh * p.k_head + j % p.page_size * p.k_slot + c) : 0.f;
      v[e] = in ? ld16<DT>(p.v, page * p.v_page + kvh * p.v_head + j % p.page_size * p.v_slot + c) : 0.f;
      s = fmaf(q[e], k[e], s);
    }
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, w);
    const float m2 = fmaxf(mx, s);
    const float old = mx == -INFINITY ? 0.f : __expf(mx - m2), pj = m2 == -INFINITY ? 0.f : __expf(s - m2);
    sum = sum * old + pj;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = o[e] * old + pj * v[e];
    mx = m2;
  }
  const float inv = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = lane + 32 * e;
    if (c < d) store_y<DT>(p.out, row * p.o_row + head * p.o_head + c, o[e] * inv);
  }
}

int check_attention(const ggufmm_attention_args& p, bool prompt) {
  const int64_t ks[3] = {p.k_page, p.k_head, p.k_slot}, vs[3] = {p.v_page, p.v_head, p.v_slot};
  const int s = check_cache(p.k, p.v, p.dtype, p.kv_heads, p.head_dim, p.page_size, p.num_pages, ks, vs);
  if (s) return s;
  if (p.batch < 0 || p.batch > 65535 || p.total_q < 0 || p.total_q > kI32Max || p.q_heads < 1 || p.q_heads > 65535 ||
      p.q_heads % p.kv_heads || p.q_heads / p.kv_heads > GGUFMM_MAX_GROUP || p.table_width < 0 ||
      p.table_row < p.table_width || p.table_width * p.page_size > kI32Max / 2 || p.window < 0 || p.window > kI32Max)
    return GGUFMM_ERR_SHAPE;
  if (prompt ? (p.max_q < 0 || p.max_q > p.total_q) : p.total_q != p.batch) return GGUFMM_ERR_SHAPE;
  if (!std::isfinite(p.scale)) return GGUFMM_ERR_ARG;
  if (p.batch == 0 || p.total_q == 0) return GGUFMM_OK;
  if (!p.q || !p.out || !p.lens || (p.table_width && !p.tables) || (prompt && !p.q_starts)) return GGUFMM_ERR_ARG;
  if (p.q_row < p.head_dim || p.q_head < p.head_dim || p.o_row < p.head_dim || p.o_head < p.head_dim)
    return GGUFMM_ERR_SHAPE;
  if (!aligned_to(p.q, 16) || !aligned_to(p.out, 16) || !aligned_to(p.lens, 4) || !aligned_to(p.tables, 4) ||
      !aligned_to(p.q_starts, 4) || !stride16_ok(p.q_row, p.head_dim) || !stride16_ok(p.q_head, p.head_dim) ||
      !stride16_ok(p.o_row, p.head_dim) || !stride16_ok(p.o_head, p.head_dim))
    return GGUFMM_ERR_ALIGN;
  return GGUFMM_OK;
}

int launch_simple(const ggufmm_attention_args& p, int64_t max_q, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>((max_q + 3) / 4), static_cast<unsigned>(p.q_heads),
                  static_cast<unsigned>(p.batch));
  return record_cuda_status(p.dtype == GGUFMM_F16
                                ? pdl_launch(attn_simple_kernel<GGUFMM_F16>, grid, dim3(128), 0, st, AttnArgs{p})
                                : pdl_launch(attn_simple_kernel<GGUFMM_BF16>, grid, dim3(128), 0, st, AttnArgs{p}));
}

}  // namespace

cudaError_t attn_device_error(int* v, int clear, cudaStream_t st) { return tu_device_error(v, clear, st); }

}  // namespace ggufmm

using namespace ggufmm;

extern "C" size_t ggufmm_paged_attention_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                        int64_t head_dim) {
  if (batch < 1 || q_heads < 1 || kv_heads < 1 || head_dim < 8 || head_dim > GGUFMM_MAX_HEAD_DIM) return 0;
  return paged_decode_workspace(head_dim);
}

extern "C" int ggufmm_paged_attention(const ggufmm_attention_args* args, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  if (!args) return GGUFMM_ERR_ARG;
  ggufmm_attention_args p = *args;
  p.q_starts = nullptr;
  int s = check_attention(p, false);
  if (s || p.batch == 0) return s;
  if (!workspace || workspace_bytes < ggufmm_paged_attention_workspace_size(p.batch, p.q_heads, p.kv_heads, p.head_dim))
    return GGUFMM_ERR_WORKSPACE;
  if (!aligned_to(workspace, 256)) return GGUFMM_ERR_ALIGN;
  s = check_device();
  if (s) return s;
  return record_cuda_status(launch_paged_decode(p, workspace, static_cast<cudaStream_t>(stream)));
}

extern "C" int ggufmm_paged_prompt_attention(const ggufmm_attention_args* args, void* stream) {
  if (!args) return GGUFMM_ERR_ARG;
  const ggufmm_attention_args& p = *args;
  int s = check_attention(p, true);
  if (s || p.batch == 0 || p.total_q == 0 || p.max_q == 0) return s;
  s = check_device();
  if (s) return s;
  return launch_simple(p, p.max_q, static_cast<cudaStream_t>(stream));
}
