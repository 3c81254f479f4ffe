// attn.cu -- the entry points of attention over a paged key-value cache,
// ggufmm_paged_attention (one new token per sequence, attn_decode.cu) and
// ggufmm_paged_prompt_attention (ragged causal prompts, attn_prompt.cu), and their checks.
//
// The reference runs a score, a softmax and an output shader over one sequence
// (vllm_webgpu/models/llama.py:239-367; shaders/generic/{attn_score,softmax,attn_output}.wgsl).
#include <cmath>

#include "paged.cuh"

namespace ggufmm {

size_t paged_decode_workspace(int64_t group, int64_t head_dim);  // attn_decode.cu
cudaError_t launch_paged_decode(const ggufmm_attention_args& p, void* workspace, cudaStream_t st);
size_t paged_prompt_workspace(const ggufmm_attention_args& p, int sms);  // attn_prompt.cu
cudaError_t launch_paged_prompt(const ggufmm_attention_args& p, int sms, void* workspace, size_t workspace_bytes,
                                cudaStream_t st);
struct DevInfo {
  int sms = 0;
  int smem_optin = 0;
};
DevInfo device_info(int dev);  // capi.cu

namespace {

int check_attention(const ggufmm_attention_args& p, bool prompt) {
  const int64_t ks[3] = {p.k_page, p.k_head, p.k_slot}, vs[3] = {p.v_page, p.v_head, p.v_slot};
  const int s = check_cache(p.k, p.v, p.dtype, p.kv_heads, p.head_dim, p.page_size, p.num_pages, ks, vs);
  if (s) return s;
  if (p.batch < 0 || p.batch > 65535 || p.total_q < 0 || p.total_q > kI32Max || p.q_heads < 1 || p.q_heads > 65535 ||
      p.q_heads % p.kv_heads || p.q_heads / p.kv_heads > GGUFMM_MAX_GROUP || p.table_width < 0 ||
      p.table_width > kI32Max || p.table_row < p.table_width || p.table_width * p.page_size > kI32Max / 2 || p.window < 0 || p.window > kI32Max)
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

}  // namespace

}  // namespace ggufmm

using namespace ggufmm;

extern "C" size_t ggufmm_paged_attention_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                        int64_t head_dim) {
  if (batch < 1 || q_heads < 1 || kv_heads < 1 || head_dim < 8 || head_dim > GGUFMM_MAX_HEAD_DIM) return 0;
  if (q_heads % kv_heads) return 0;
  return paged_decode_workspace(q_heads / kv_heads, head_dim);
}

extern "C" int ggufmm_paged_attention(const ggufmm_attention_args* args, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  if (!args) return GGUFMM_ERR_ARG;
  ggufmm_attention_args p = *args;
  p.q_starts = nullptr;
  int s = check_attention(p, false);
  if (s || p.batch == 0) return s;
  // the kernel counts blocks of at least 64 tokens of every (sequence, kv head, 16 query heads)
  if (p.batch * p.kv_heads * ((p.q_heads / p.kv_heads + 15) / 16) > kI32Max / (p.table_width * p.page_size / 64 + 3))
    return GGUFMM_ERR_SHAPE;
  if (!workspace || workspace_bytes < ggufmm_paged_attention_workspace_size(p.batch, p.q_heads, p.kv_heads, p.head_dim))
    return GGUFMM_ERR_WORKSPACE;
  if (!aligned_to(workspace, 256)) return GGUFMM_ERR_ALIGN;
  s = check_device();
  if (s) return s;
  return record_cuda_status(launch_paged_decode(p, workspace, static_cast<cudaStream_t>(stream)));
}

extern "C" size_t ggufmm_paged_prompt_attention_workspace_size(const ggufmm_attention_args* args) {
  int dev = 0;
  if (!args || check_attention(*args, true) || args->batch == 0 || args->max_q == 0 || check_device() ||
      cudaGetDevice(&dev) != cudaSuccess || args->max_q > kI32Max / (args->batch * args->kv_heads))
    return 0;
  return paged_prompt_workspace(*args, device_info(dev).sms);
}

extern "C" int ggufmm_paged_prompt_attention(const ggufmm_attention_args* args, void* workspace, size_t workspace_bytes,
                                             void* stream) {
  if (!args) return GGUFMM_ERR_ARG;
  const ggufmm_attention_args& p = *args;
  int s = check_attention(p, true);
  if (s || p.batch == 0 || p.total_q == 0 || p.max_q == 0) return s;
  if (p.max_q > kI32Max / (p.batch * p.kv_heads)) return GGUFMM_ERR_SHAPE;  // tiles of the grid
  if (!aligned_to(workspace, 256)) return GGUFMM_ERR_ALIGN;
  s = check_device();
  if (s) return s;
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return record_cuda_status(e);
  return record_cuda_status(
      launch_paged_prompt(p, device_info(dev).sms, workspace, workspace_bytes, static_cast<cudaStream_t>(stream)));
}
