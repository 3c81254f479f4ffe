// rope.cu -- ggufmm_rope_append: rotary positions on q and k, and the append of k and v
// to a paged key-value cache, in one launch.
//
// A pair (a, b) of the first rot_dim values of a head turns by phi = position * f_i:
//   a' = factor * (a cos phi - b sin phi),  b' = factor * (a sin phi + b cos phi)
// with (a, b) = (i, i + rot_dim/2) or, interleaved, (2i, 2i + 1). The reference runs this
// as its rope shader on q and on k and its kv_cache_store shader on k and on v
// (vllm_webgpu/models/llama.py:239-367; shaders/generic/{rope,kv_cache_store}.wgsl).
//
// The frequencies come as turns per position in units of 2^-64 (a 64-bit integer), so the
// product with the position, reduced modulo one turn by the integer's own overflow, is
// exact for every position: an fp32 product of a position near 10^6 and a frequency
// would be off by hundredths of a radian.
#include <algorithm>
#include <type_traits>

#include "mma16.cuh"
#include "paged.cuh"

namespace ggufmm {

namespace {

struct RopeArgs {
  ggufmm_rope_args p;
};

__device__ __forceinline__ float2 turn(int64_t pos, int64_t step, float factor) {
  // signed 64-bit product = turns modulo 1 in [-1/2, 1/2) * 2^64; in half turns: * 2^-63
  const float t = static_cast<float>(static_cast<int64_t>(static_cast<uint64_t>(pos) * static_cast<uint64_t>(step))) *
                  1.0842021724855044e-19f;
  float c, s;
  sincospif(t, &s, &c);
  return make_float2(c * factor, s * factor);
}

// N consecutive values as they lie in memory, aligned to 16 bytes or to all of them.
template <int ES, int N>
struct alignas(N * ES >= 16 ? 16 : N * ES >= 8 ? 8 : 4) Vals {
  uint32_t u[N * ES >= 4 ? N * ES / 4 : 1];
};

template <int ES, int N>
__device__ __forceinline__ void load_vals(Vals<ES, N>& d, const void* p, int64_t i) {
  const uint8_t* q = static_cast<const uint8_t*>(p) + i * ES;
  if constexpr (N == 1) {
    d.u[0] = ES == 4 ? *reinterpret_cast<const uint32_t*>(q) : *reinterpret_cast<const uint16_t*>(q);
  } else if constexpr (N * ES == 8) {
    *reinterpret_cast<uint2*>(d.u) = *reinterpret_cast<const uint2*>(q);
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
  } else if constexpr (N == 4) {
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) =
        dt == GGUFMM_F16 ? make_uint2(pack16<GGUFMM_F16>(f[0], f[1]), pack16<GGUFMM_F16>(f[2], f[3]))
                         : make_uint2(pack16<GGUFMM_BF16>(f[0], f[1]), pack16<GGUFMM_BF16>(f[2], f[3]));
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

// A CTA takes TB tokens: it makes their sines and cosines once, in shared memory, for all
// heads, then runs over the units of q, k and v: N pairs (2 N values) that turn, or 2 N values
// that pass. A thread has the same unit of all TB tokens, so that several loads are under way at
// a time and the unit's place is found once; the first ones go out before the sines are made. N is
// 8 or 4, where the widths and strides allow whole groups of 16 (8) bytes, or 1.
// HBM bound: 8192 tokens of 32 / 8 heads of 128 (201 MB) in 35 us, 5.7 TB/s, 89% of the measured
// copy rate, with two tokens and 128 threads a CTA; 256 threads 45 us (their waits coincide), four
// tokens 36 us, sines before loads 47 us. A few tokens take 3 us, a launch and two memory latencies.
// Rotary widths that are no multiple of 8 go value by value: 8192 tokens, heads of 80 with 20 turning
// (126 MB) 68 us, 1.9 TB/s; all 80 turning 28 us, 4.5 TB/s.
template <int XT, int N, int TB, int NT>
__global__ void __launch_bounds__(NT) rope_append_kernel(const __grid_constant__ RopeArgs a) {
  extern __shared__ float2 table[];  // [TB][half]
  __shared__ int64_t place[2][TB];   // where a token's k and v go, negative for nowhere
  constexpr int ES = XT == GGUFMM_F32 ? 4 : 2;
  pdl_wait();
  pdl_trigger();
  const ggufmm_rope_args& p = a.p;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * TB;
  const int nt = static_cast<int>(min(static_cast<int64_t>(TB), p.tokens - t0));
  const int d = static_cast<int>(p.head_dim), half = static_cast<int>(p.rot_dim) / 2;
  const int hq = static_cast<int>(p.q_heads), hkv = p.k ? static_cast<int>(p.kv_heads) : 0;
  // units of a head that turns: pairs first, then what passes; a head of v passes whole
  const int ut = half / N, uh = ut + (d - 2 * half) / (2 * N), uv = d / (2 * N);
  const int turning = (hq + hkv) * uh, per = turning + hkv * uv;
  for (int j0 = 0; j0 < per; j0 += NT) {
    const int j = min(j0 + static_cast<int>(threadIdx.x), per - 1);
    const int rows = j0 + static_cast<int>(threadIdx.x) < per ? nt : 0;  // 0: past the last unit
    const bool isv = j >= turning;
    int h = isv ? (j - turning) / uv : j / uh;
    const int u = isv ? (j - turning) - h * uv : j - h * uh;
    const bool isk = !isv && h >= hq, cached = isk || isv;
    if (isk) h -= hq;
    const bool turns = !isv && u < ut;
    // two groups of N values, each in a row with those of the lanes beside: the halves of what
    // turns (in either order of pairs), of what passes, of a head of v; N == 1 and interleaved: a pair
    const bool apart = !(N == 1 && turns && p.interleaved);
    const int first = isv || turns ? 0 : 2 * half, span = isv ? d / 2 : turns ? half : d / 2 - half;
    const int e0 = first + (apart ? (turns || isv ? u : u - ut) * N : 2 * u), e1 = apart ? e0 + span : e0 + 1;
    const void* src = isv ? p.v : isk ? p.k : p.q;
    const int64_t in_row = isv ? p.v_row : isk ? p.k_row : p.q_row;
    const int64_t in = t0 * in_row + h * (isv ? p.v_head : isk ? p.k_head : p.q_head);
    void* dst = isv ? p.v_cache : isk ? p.k_cache : p.q_out;
    const int dt = static_cast<int>(cached ? p.cache_dtype : p.q_out_dtype);
    const int64_t out_head = h * (isv ? p.vc_head : isk ? p.kc_head : p.qo_head);
    Vals<ES, N> x[TB], y[TB];
#pragma unroll
    for (int t = 0; t < TB; ++t)
      if (t < rows) {
        load_vals(x[t], src, in + t * in_row + e0);
        load_vals(y[t], src, in + t * in_row + e1);
      }
    if (j0 == 0) {  // while the first loads are under way
      const int64_t* positions = static_cast<const int64_t*>(p.positions) + t0;
      if (hkv && threadIdx.x < nt) {
        const int64_t slot = static_cast<const int64_t*>(p.slots)[t0 + threadIdx.x];
        const int64_t page = slot < 0 ? 0 : slot / p.page_size, off = slot - page * p.page_size;
        const bool in = slot >= 0 && page < p.num_pages;
        if (slot >= 0 && !in) atomicOr(&g_device_error, kErrIndex);
        place[0][threadIdx.x] = in ? page * p.kc_page + off * p.kc_slot : -1;
        place[1][threadIdx.x] = in ? page * p.vc_page + off * p.vc_slot : -1;
      }
      for (int i = threadIdx.x; i < nt * half; i += NT)
        table[i] = turn(positions[i / half], static_cast<const int64_t*>(p.steps)[i % half], static_cast<float>(p.factor));
      __syncthreads();
    }
#pragma unroll
    for (int t = 0; t < TB; ++t) {
      if (t >= rows) break;
      const int64_t at = cached ? place[isv][t] : (t0 + t) * p.qo_row;
      if (at < 0) continue;
      const int64_t out = at + out_head;
      float f[2 * N], g[2 * N];
      to_float<XT>(x[t], f);
      to_float<XT>(y[t], f + N);
      if (!turns) {
#pragma unroll
        for (int k = 0; k < 2 * N; ++k) g[k] = f[k];
      } else if (N > 1 && p.interleaved) {  // pairs inside each group
        const float2* cs = table + t * half + e0 / 2;
#pragma unroll
        for (int k = 0; k < 2 * N; k += 2) {
          const float2 w = cs[k < N ? k / 2 : half / 2 + (k - N) / 2];
          g[k] = f[k] * w.x - f[k + 1] * w.y;
          g[k + 1] = f[k] * w.y + f[k + 1] * w.x;
        }
      } else {
        const float2* cs = table + t * half + u * N;
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float2 w = cs[k];
          g[k] = f[k] * w.x - f[k + N] * w.y;
          g[k + N] = f[k] * w.y + f[k + N] * w.x;
        }
      }
      store_vals<N>(dst, dt, out + e0, g);
      store_vals<N>(dst, dt, out + e1, g + N);
    }
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
  // the widest groups of values that all widths, strides and addresses allow
  auto whole = [&](int n) {
    auto fits = [n](const void* ptr, int64_t e, int64_t row, int64_t head) {
      const int64_t bytes = std::min<int64_t>(n * e, 16);
      return reinterpret_cast<uintptr_t>(ptr) % bytes == 0 && row * e % bytes == 0 && head * e % bytes == 0;
    };
    return p.rot_dim % (2 * n) == 0 && d % (2 * n) == 0 && fits(p.q, xe, p.q_row, p.q_head) &&
           fits(p.q_out, qe, p.qo_row, p.qo_head) &&
           (!p.k || (fits(p.k, xe, p.k_row, p.k_head) && fits(p.v, xe, p.v_row, p.v_head)));
  };
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool many = p.tokens >= 592;  // two tokens a CTA leave several CTAs to every SM
  const int tb = many ? 2 : 1;
  const dim3 grid(static_cast<unsigned>((p.tokens + tb - 1) / tb));
  const size_t smem = static_cast<size_t>(tb) * (p.rot_dim / 2) * sizeof(float2);
  auto typed = [&](auto xt, auto n) {
    constexpr int XT = decltype(xt)::value, N = decltype(n)::value;
    return many ? pdl_launch(rope_append_kernel<XT, N, 2, 128>, grid, dim3(128), smem, st, RopeArgs{p})
                : pdl_launch(rope_append_kernel<XT, N, 1, 256>, grid, dim3(256), smem, st, RopeArgs{p});
  };
  auto sized = [&](auto n) {
    return record_cuda_status(p.x_dtype == GGUFMM_F32   ? typed(std::integral_constant<int, GGUFMM_F32>{}, n)
                              : p.x_dtype == GGUFMM_F16 ? typed(std::integral_constant<int, GGUFMM_F16>{}, n)
                                                        : typed(std::integral_constant<int, GGUFMM_BF16>{}, n));
  };
  if (whole(8)) return sized(std::integral_constant<int, 8>{});
  if (whole(4)) return sized(std::integral_constant<int, 4>{});
  return sized(std::integral_constant<int, 1>{});
}
