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
#include <initializer_list>

#include "mma16.cuh"
#include "paged.cuh"

namespace ggufmm {

namespace {

struct RopeArgs {
  ggufmm_rope_args p;
  int per_cta;  // tokens of a CTA
};

__device__ __forceinline__ float2 turn(int64_t pos, int64_t step, float factor) {
  // signed 64-bit product = turns modulo 1 in [-1/2, 1/2) * 2^64; in half turns: * 2^-63
  const float t = static_cast<float>(static_cast<int64_t>(static_cast<uint64_t>(pos) * static_cast<uint64_t>(step))) *
                  1.0842021724855044e-19f;
  float c, s;
  sincospif(t, &s, &c);
  return make_float2(c * factor, s * factor);
}

// N consecutive values as they lie in memory (16-byte aligned where N * ES is).
template <int ES, int N>
struct Vals {
  uint32_t u[N * ES >= 4 ? N * ES / 4 : 1];
};

template <int ES, int N>
__device__ __forceinline__ void load_vals(Vals<ES, N>& d, const void* p, int64_t i) {
  const uint8_t* q = static_cast<const uint8_t*>(p) + i * ES;
  if constexpr (N == 1) {
    d.u[0] = ES == 4 ? *reinterpret_cast<const uint32_t*>(q) : *reinterpret_cast<const uint16_t*>(q);
  } else {
#pragma unroll
    for (int k = 0; k < N * ES / 16; ++k) reinterpret_cast<uint4*>(d.u)[k] = reinterpret_cast<const uint4*>(q)[k];
  }
}

template <int XT, int ES, int N>
__device__ __forceinline__ void to_float(const Vals<ES, N>& d, float* f) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const uint32_t u = XT == GGUFMM_F32 ? d.u[k] : N == 1 ? d.u[0] : (k & 1 ? d.u[k / 2] >> 16 : d.u[k / 2] & 0xFFFFu);
    if (XT == GGUFMM_F32) f[k] = __uint_as_float(u);
    else if (XT == GGUFMM_BF16) f[k] = __uint_as_float(u << 16);
    else f[k] = half_bits_to_float(u);
  }
}

template <int N>
__device__ __forceinline__ void store_vals(void* p, int dt, int64_t i, const float* f) {
  if constexpr (N == 1) {
    store_y_rt(p, dt, i, f[0]);
  } else if (dt == GGUFMM_F32) {
#pragma unroll
    for (int k = 0; k < N / 4; ++k)
      reinterpret_cast<float4*>(static_cast<float*>(p) + i)[k] = make_float4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
  } else {
#pragma unroll
    for (int k = 0; k < N / 8; ++k) {
      uint32_t u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float lo = f[8 * k + 2 * e], hi = f[8 * k + 2 * e + 1];
        u[e] = dt == GGUFMM_F16 ? pack16<GGUFMM_F16>(lo, hi) : pack16<GGUFMM_BF16>(lo, hi);
      }
      reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i)[k] = make_uint4(u[0], u[1], u[2], u[3]);
    }
  }
}

// A CTA takes per_cta tokens: it makes their sines and cosines once, in shared memory, for
// all heads, then runs over the units of q, k and v: N pairs (2 N values) that turn, or 2 N
// values that pass. N is 8, where whole 16-byte groups allow it, or 1.
template <int XT, int N>
__global__ void __launch_bounds__(256) rope_append_kernel(const __grid_constant__ RopeArgs a) {
  extern __shared__ float2 table[];  // [per_cta][half]
  constexpr int ES = XT == GGUFMM_F32 ? 4 : 2;
  pdl_wait();
  pdl_trigger();
  const ggufmm_rope_args& p = a.p;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.per_cta;
  const int nt = static_cast<int>(min(static_cast<int64_t>(a.per_cta), p.tokens - t0));
  const int d = static_cast<int>(p.head_dim), half = static_cast<int>(p.rot_dim) / 2;
  const int hq = static_cast<int>(p.q_heads), hkv = p.k ? static_cast<int>(p.kv_heads) : 0;
  const int ct = static_cast<int>(p.cache_dtype);
  const int64_t* positions = static_cast<const int64_t*>(p.positions) + t0;
  for (int i = threadIdx.x; i < nt * half; i += 256)
    table[i] = turn(positions[i / half], static_cast<const int64_t*>(p.steps)[i % half], static_cast<float>(p.factor));
  __syncthreads();
  // units of a head that turns: pairs first, then what passes; a head of v passes whole
  const int ut = half / N, uh = ut + (d - 2 * half) / (2 * N), uv = d / (2 * N);
  const int turning = (hq + hkv) * uh, per = turning + hkv * uv;
  for (int i = threadIdx.x; i < nt * per; i += 256) {
    const int t = i / per, j = i - t * per;
    const bool isv = j >= turning;
    int h = isv ? (j - turning) / uv : j / uh;
    const int u = isv ? (j - turning) - h * uv : j - h * uh;
    const bool isk = !isv && h >= hq;
    if (isk) h -= hq;
    const void* src;
    void* dst;
    int64_t in, out;
    int dt;
    if (!isk && !isv) {
      src = p.q;
      dst = p.q_out;
      dt = static_cast<int>(p.q_out_dtype);
      in = (t0 + t) * p.q_row + h * p.q_head;
      out = (t0 + t) * p.qo_row + h * p.qo_head;
    } else {
      const int64_t slot = static_cast<const int64_t*>(p.slots)[t0 + t];
      if (slot < 0) continue;
      const int64_t page = slot / p.page_size, off = slot - page * p.page_size;
      if (page >= p.num_pages) {
        atomicOr(&g_device_error, kErrIndex);
        continue;
      }
      dt = ct;
      src = isk ? p.k : p.v;
      dst = isk ? p.k_cache : p.v_cache;
      in = (t0 + t) * (isk ? p.k_row : p.v_row) + h * (isk ? p.k_head : p.v_head);
      out = isk ? page * p.kc_page + h * p.kc_head + off * p.kc_slot : page * p.vc_page + h * p.vc_head + off * p.vc_slot;
    }
    if (isv || u >= ut) {
      const int e = isv ? u * 2 * N : 2 * half + (u - ut) * 2 * N;
      Vals<ES, N> x, y;
      load_vals(x, src, in + e);
      load_vals(y, src, in + e + N);
      float f[2 * N];
      to_float<XT>(x, f);
      to_float<XT>(y, f + N);
      store_vals<N>(dst, dt, out + e, f);
      store_vals<N>(dst, dt, out + e + N, f + N);
      continue;
    }
    const float2* cs = table + t * half + u * N;
    const int e0 = p.interleaved ? u * 2 * N : u * N, e1 = p.interleaved ? e0 + N : e0 + half;
    Vals<ES, N> x, y;
    load_vals(x, src, in + e0);
    load_vals(y, src, in + e1);
    float f[2 * N], g[2 * N];
    to_float<XT>(x, f);
    to_float<XT>(y, f + N);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float2 w = cs[k];
      // both orders by selects: the arrays stay in registers
      const float v0 = p.interleaved ? f[2 * k] : f[k], v1 = p.interleaved ? f[2 * k + 1] : f[k + N];
      const float r0 = v0 * w.x - v1 * w.y, r1 = v0 * w.y + v1 * w.x;
      if (p.interleaved) {
        g[2 * k] = r0;
        g[2 * k + 1] = r1;
      } else {
        g[k] = r0;
        g[k + N] = r1;
      }
    }
    store_vals<N>(dst, dt, out + e0, g);
    store_vals<N>(dst, dt, out + e1, g + N);
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
  // whole 16-byte groups: units of 8 pairs
  auto whole = [](const void* ptr, int64_t e, std::initializer_list<int64_t> strides) {
    bool ok = aligned_to(ptr, 16);
    for (const int64_t v : strides) ok = ok && v * e % 16 == 0;
    return ok;
  };
  const bool vec = d % 16 == 0 && p.rot_dim % 16 == 0 && whole(p.q, xe, {p.q_row, p.q_head}) &&
                   whole(p.q_out, qe, {p.qo_row, p.qo_head}) &&
                   (!p.k || (whole(p.k, xe, {p.k_row, p.k_head}) && whole(p.v, xe, {p.v_row, p.v_head})));
  RopeArgs a{p, 1};
  if (p.tokens > 2048) a.per_cta = 4;
  const dim3 grid(static_cast<unsigned>((p.tokens + a.per_cta - 1) / a.per_cta));
  const size_t smem = static_cast<size_t>(a.per_cta) * (p.rot_dim / 2) * sizeof(float2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto* fn) { return record_cuda_status(pdl_launch(fn, grid, dim3(256), smem, st, a)); };
  if (p.x_dtype == GGUFMM_F32) return vec ? go(rope_append_kernel<GGUFMM_F32, 8>) : go(rope_append_kernel<GGUFMM_F32, 1>);
  if (p.x_dtype == GGUFMM_F16) return vec ? go(rope_append_kernel<GGUFMM_F16, 8>) : go(rope_append_kernel<GGUFMM_F16, 1>);
  return vec ? go(rope_append_kernel<GGUFMM_BF16, 8>) : go(rope_append_kernel<GGUFMM_BF16, 1>);
}
