// rope.cu -- ggufmm_rope_append: rotary positions on q and k, and the append of k and v
// to a paged key-value cache, in one launch.
//
// A pair (a, b) of the first rot_dim values of a head turns by phi = position * f_i:
//   a' = factor * (a cos phi - b sin phi),  b' = factor * (a sin phi + b cos phi)
// with (a, b) = (i, i + rot_dim/2) or, interleaved, (2i, 2i + 1). The reference runs this
// as its rope shader on q and on k and its kv_cache_store shader on k and on v
// (vllm_webgpu/models/llama.py:286-312; shaders/generic/{rope,kv_cache_store}.wgsl).
//
// The frequencies come as turns per position in units of 2^-64 (a 64-bit integer), so the
// product with the position, reduced modulo one turn by the integer's own overflow, is
// exact for every position: an fp32 product of a position near 10^6 and a frequency
// would be off by hundredths of a radian.
#include "paged.cuh"

namespace ggufmm {

namespace {

struct RopeArgs {
  ggufmm_rope_args p;
};

__device__ __forceinline__ void turn(int64_t pos, int64_t step, float factor, float* c, float* s) {
  // signed 64-bit product = turns modulo 1 in [-1/2, 1/2) * 2^64; in half turns: * 2^-63
  const float t = static_cast<float>(static_cast<int64_t>(static_cast<uint64_t>(pos) * static_cast<uint64_t>(step))) *
                  1.0842021724855044e-19f;
  sincospif(t, s, c);
  *c *= factor;
  *s *= factor;
}

// One token per CTA, one value per thread and step.
__global__ void __launch_bounds__(256) rope_append_kernel(const __grid_constant__ RopeArgs a) {
  pdl_wait();
  pdl_trigger();
  const ggufmm_rope_args& p = a.p;
  const int64_t t = blockIdx.x;
  const int64_t pos = static_cast<const int64_t*>(p.positions)[t];
  const int d = static_cast<int>(p.head_dim), half = static_cast<int>(p.rot_dim) / 2;
  const int units = d - half;  // per head: pairs, then the values that pass
  const int hq = static_cast<int>(p.q_heads), hkv = p.k ? static_cast<int>(p.kv_heads) : 0;
  const int xt = static_cast<int>(p.x_dtype), ct = static_cast<int>(p.cache_dtype);
  int64_t slot = -1, base_k = 0, base_v = 0;
  if (hkv) {
    slot = static_cast<const int64_t*>(p.slots)[t];
    if (slot >= p.num_pages * p.page_size) {
      if (threadIdx.x == 0) atomicOr(&g_device_error, kErrIndex);
      slot = -1;
    }
    if (slot >= 0) {
      base_k = slot / p.page_size * p.kc_page + slot % p.page_size * p.kc_slot;
      base_v = slot / p.page_size * p.vc_page + slot % p.page_size * p.vc_slot;
    }
  }
  const int nq = hq * units, nk = slot >= 0 ? hkv * units : 0, nv = slot >= 0 ? hkv * d : 0;
  for (int i = threadIdx.x; i < nq + nk; i += 256) {
    const bool isq = i < nq;
    const int j = isq ? i : i - nq, h = j / units, u = j % units;
    const void* src = isq ? p.q : p.k;
    void* dst = isq ? p.q_out : p.k_cache;
    const int dt = isq ? static_cast<int>(p.q_out_dtype) : ct;
    const int64_t in = isq ? t * p.q_row + h * p.q_head : t * p.k_row + h * p.k_head;
    const int64_t out = isq ? t * p.qo_row + h * p.qo_head : base_k + h * p.kc_head;
    if (u < half) {
      const int e0 = p.interleaved ? 2 * u : u, e1 = p.interleaved ? 2 * u + 1 : u + half;
      float c, s;
      turn(pos, static_cast<const int64_t*>(p.steps)[u], static_cast<float>(p.factor), &c, &s);
      const float x0 = load_y_rt(src, xt, in + e0), x1 = load_y_rt(src, xt, in + e1);
      store_y_rt(dst, dt, out + e0, x0 * c - x1 * s);
      store_y_rt(dst, dt, out + e1, x0 * s + x1 * c);
    } else {
      store_y_rt(dst, dt, out + u + half, load_y_rt(src, xt, in + u + half));
    }
  }
  for (int i = threadIdx.x; i < nv; i += 256) {
    const int h = i / d, e = i % d;
    store_y_rt(p.v_cache, ct, base_v + h * p.vc_head + e, load_y_rt(p.v, xt, t * p.v_row + h * p.v_head + e));
  }
}

int elem(int64_t dtype) { return dtype == GGUFMM_F32 ? 4 : dtype == GGUFMM_F16 || dtype == GGUFMM_BF16 ? 2 : 0; }

}  // namespace

cudaError_t rope_device_error(int* v, int clear, cudaStream_t st) { return tu_device_error(v, clear, st); }

}  // namespace ggufmm

using namespace ggufmm;

extern "C" int ggufmm_rope_append(const ggufmm_rope_args* args, void* stream) {
  if (!args) return GGUFMM_ERR_ARG;
  const ggufmm_rope_args& p = *args;
  const int xe = elem(p.x_dtype), qe = elem(p.q_out_dtype);
  if (!xe || !qe) return GGUFMM_ERR_DTYPE;
  const int64_t d = p.head_dim;
  if (p.tokens < 0 || p.tokens > kI32Max || p.q_heads < 1 || p.q_heads > 65535 || d < 8 || d > GGUFMM_MAX_HEAD_DIM ||
      d % 8 || p.rot_dim < 0 || p.rot_dim > d || p.rot_dim % 2)
    return GGUFMM_ERR_SHAPE;
  if (p.q_row < 0 || p.q_head < 0 || p.qo_row < 0 || p.qo_head < 0) return GGUFMM_ERR_SHAPE;
  if (p.k) {
    const int64_t ks[3] = {p.kc_page, p.kc_head, p.kc_slot}, vs[3] = {p.vc_page, p.vc_head, p.vc_slot};
    const int s = check_cache(p.k_cache, p.v_cache, p.cache_dtype, p.kv_heads, d, p.page_size, p.num_pages, ks, vs);
    if (s) return s;
    if (p.k_row < 0 || p.k_head < 0 || p.v_row < 0 || p.v_head < 0) return GGUFMM_ERR_SHAPE;
  }
  if (p.tokens == 0) return GGUFMM_OK;
  if (!p.q || !p.q_out || !p.positions || (p.rot_dim && !p.steps) || (p.k && (!p.v || !p.slots))) return GGUFMM_ERR_ARG;
  if (!aligned_to(p.q, xe) || !aligned_to(p.q_out, qe) || !aligned_to(p.k, xe) || !aligned_to(p.v, xe) ||
      !aligned_to(p.positions, 8) || !aligned_to(p.slots, 8) || !aligned_to(p.steps, 8))
    return GGUFMM_ERR_ALIGN;
  const int s = check_device();
  if (s) return s;
  return record_cuda_status(pdl_launch(rope_append_kernel, dim3(static_cast<unsigned>(p.tokens)), dim3(256), 0,
                                       static_cast<cudaStream_t>(stream), RopeArgs{p}));
}
