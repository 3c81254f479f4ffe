// norm.cu -- ggufmm_rms_norm: root-mean-square norm of each row, with the residual's
// addition in front of it.
//
//   s = x + r,  y = s * rsqrt(mean(s^2) + eps) * (w + c),  r' = s
//
// The reference runs its add shader and its rms_norm shader as two dispatches
// (vllm_webgpu/models/llama.py:239-367; shaders/generic/{add,rms_norm}.wgsl),
// with the stream rounded to f16 between them. Here the sum stays in 32 bits: it is
// rounded once into r' and, after the norm, once into y.
//
// HBM bound: a row is read once, held in registers over the sum of its squares, and written.
// 8192 rows of 4096, x in 32 bits, r, r' and y in bf16 (336 MB): 51.5 us, 6.5 TB/s, the measured
// copy rate. One row takes 2.2 us, a launch and two memory latencies. Rows of odd width start
// between 16-byte boundaries: without gaps they are read by the tensor's aligned groups (8192 rows
// of 4095: 59 us, 5.7 TB/s; 94 value by value, as rows with odd gaps still go).
#include "mma16.cuh"
#include "shifted.cuh"

namespace ggufmm {

int record_cuda_status(cudaError_t e);  // capi.cu
int check_device();                     // capi.cu

namespace {

struct NormArgs {
  const void* x;
  const void* r;
  void* ro;
  const void* w;
  void* y;
  int64_t ldx, ldr, ldro, ldy;
  int m, n;
  int xt, rt, wt, yt;
  float c, eps, inv_n;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// The sum over a CTA of up to 32 warps, the same bits in every thread.
__device__ __forceinline__ float cta_sum(float v, float* part) {
  v = warp_sum(v);
  const int nw = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return warp_sum(lane < nw ? part[lane] : 0.f);
}

// Eight values of one row: raw bytes first, so that all of a thread's loads are in flight
// before the first is converted.
template <int ES>
struct Raw8 {
  uint4 v[ES / 2];
};
template <>
struct Raw8<0> {};

template <int ES>
__device__ __forceinline__ void raw_load(Raw8<ES>& d, const void* p, int64_t i) {
  const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + i * ES);
#pragma unroll
  for (int k = 0; k < ES / 2; ++k) d.v[k] = q[k];
}

__device__ __forceinline__ void widen(uint32_t u, int t, float* f) {
  if (t == GGUFMM_BF16) {
    f[0] = __uint_as_float(u << 16);
    f[1] = __uint_as_float(u & 0xFFFF0000u);
  } else {
    const float2 h = __half22float2(*reinterpret_cast<__half2*>(&u));
    f[0] = h.x;
    f[1] = h.y;
  }
}

template <int ES>
__device__ __forceinline__ void raw_float(const Raw8<ES>& d, int t, float* f) {
  const uint32_t* u = reinterpret_cast<const uint32_t*>(d.v);
  if constexpr (ES == 4) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = __uint_as_float(u[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) widen(u[k], t, f + 2 * k);
  }
}

__device__ __forceinline__ void store8(void* p, int t, int64_t i, const float* f) {
  if (t == GGUFMM_F32) {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
    q[0] = make_float4(f[0], f[1], f[2], f[3]);
    q[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    uint4 v;
    v.x = t == GGUFMM_F16 ? pack16<GGUFMM_F16>(f[0], f[1]) : pack16<GGUFMM_BF16>(f[0], f[1]);
    v.y = t == GGUFMM_F16 ? pack16<GGUFMM_F16>(f[2], f[3]) : pack16<GGUFMM_BF16>(f[2], f[3]);
    v.z = t == GGUFMM_F16 ? pack16<GGUFMM_F16>(f[4], f[5]) : pack16<GGUFMM_BF16>(f[4], f[5]);
    v.w = t == GGUFMM_F16 ? pack16<GGUFMM_F16>(f[6], f[7]) : pack16<GGUFMM_BF16>(f[6], f[7]);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = v;
  }
}

// The same of the tensor's last group, which ends behind it.
template <int ES>
__device__ __forceinline__ void raw_load_last(Raw8<ES>& d, const void* p, int64_t row, int i, int n) {
  uint32_t* u = reinterpret_cast<uint32_t*>(d.v);
#pragma unroll
  for (int e = 0; e < 2 * ES; ++e) u[e] = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (i + e < 0 || i + e >= n) continue;
    if (ES == 4) u[e] = static_cast<const uint32_t*>(p)[row + i + e];
    else u[e / 2] |= static_cast<uint32_t>(static_cast<const uint16_t*>(p)[row + i + e]) << (e % 2 * 16);
  }
}

__device__ __forceinline__ void store8_edge(void* p, int t, int64_t row, int i, int n, const float* f) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (i + e >= 0 && i + e < n) store_y_rt(p, t, row + i + e, f[e]);
}

__device__ __forceinline__ void weights8(const void* p, int t, int i, float* w) {
  if (t == GGUFMM_F32) {
    Raw8<4> q;
    raw_load(q, p, i);
    raw_float(q, t, w);
  } else {
    Raw8<2> q;
    raw_load(q, p, i);
    raw_float(q, t, w);
  }
}

// A row is held in the registers of WARP ? one warp : one CTA, V groups of eight values a
// thread; XS, RS: bytes of a value of x and of r (0: none). Rows of whole 16-byte groups, or,
// SHIFT, rows of any width from 8 without a gap: the groups are then those of the whole tensor,
// each on 16 bytes; what a row's first and last hold of its neighbours is read and dropped. (A
// row's squares are then added in an order that depends on where it begins.)
template <int XS, int RS, int V, bool WARP, bool SHIFT>
__global__ void __launch_bounds__(WARP ? 256 : SHIFT ? 512 : 1024, SHIFT && V == 1 ? 3 : 1) rms_norm_vec_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float part[32];
  pdl_wait();
  pdl_trigger();
  const int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= a.m) return;  // whole warps
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, nt = WARP ? 32 : blockDim.x;
  const int shift = SHIFT ? static_cast<int>(row * a.n & 7) : 0;
  auto inside = [&](int i) { return !SHIFT || (i >= 0 && i + 8 <= a.n); };
  Raw8<XS> xr[V];
  Raw8<RS> rr[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int i = (tid + k * nt) * 8 - shift;
    if (i >= a.n) continue;
    if (!SHIFT || row + 1 < a.m || i + 8 <= a.n) {
      raw_load(xr[k], a.x, row * a.ldx + i);
      if constexpr (RS != 0) raw_load(rr[k], a.r, row * a.ldr + i);
    } else {
      raw_load_last(xr[k], a.x, row * a.ldx, i, a.n);
      if constexpr (RS != 0) raw_load_last(rr[k], a.r, row * a.ldr, i, a.n);
    }
  }
  float s[V][8], ss = 0.f;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int i = (tid + k * nt) * 8 - shift;
    if (i < a.n) {
      raw_float(xr[k], a.xt, s[k]);
      if constexpr (RS != 0) {
        float r[8];
        raw_float(rr[k], a.rt, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[k][e] += r[e];
        if (a.ro) {
          if (inside(i)) store8(a.ro, a.rt, row * a.ldro + i, s[k]);
          else store8_edge(a.ro, a.rt, row * a.ldro, i, a.n, s[k]);
        }
      }
      if (inside(i)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(s[k][e], s[k][e], ss);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e >= 0 && i + e < a.n) ss = fmaf(s[k][e], s[k][e], ss);
      }
    }
  }
  ss = WARP ? warp_sum(ss) : cta_sum(ss, part);
  const float inv = rsqrtf(fmaf(ss, a.inv_n, a.eps));
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int i = (tid + k * nt) * 8 - shift;
    if (i < a.n) {
      float w[8];
      if (a.w) {
        if (SHIFT)
          shifted8(i, shift, a.n, [&](int j, float* v) { weights8(a.w, a.wt, j, v); },
                   [&](int j) { return load_y_rt(a.w, a.wt, j); }, w);
        else
          weights8(a.w, a.wt, i, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = s[k][e] * inv * (w[e] + a.c);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = s[k][e] * inv;
      }
      if (inside(i)) store8(a.y, a.yt, row * a.ldy + i, w);
      else store8_edge(a.y, a.yt, row * a.ldy, i, a.n, w);
    }
  }
}

// Any width and alignment: one row per CTA, value by value, E of them held by a thread (raw
// first, as above). XS, RS: bytes of a value of x and of r (0: none).
template <int E, int XS, int RS>
__global__ void __launch_bounds__(512) rms_norm_any_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float part[32];
  pdl_wait();
  pdl_trigger();
  const int64_t row = blockIdx.x;
  auto raw = [](const void* p, int es, int64_t i) -> uint32_t {
    return es == 4 ? static_cast<const uint32_t*>(p)[i] : static_cast<const uint16_t*>(p)[i];
  };
  auto value = [](uint32_t u, int t) {
    return t == GGUFMM_F16 ? half_bits_to_float(u) : __uint_as_float(t == GGUFMM_BF16 ? u << 16 : u);
  };
  uint32_t x[E], r[E];
#pragma unroll
  for (int k = 0; k < E; ++k) {
    const int i = threadIdx.x + k * blockDim.x;
    x[k] = i < a.n ? raw(a.x, XS, row * a.ldx + i) : 0u;
    if (RS) r[k] = i < a.n ? raw(a.r, RS, row * a.ldr + i) : 0u;
  }
  float s[E], ss = 0.f;
#pragma unroll
  for (int k = 0; k < E; ++k) {
    s[k] = value(x[k], a.xt);
    if (RS) s[k] += value(r[k], a.rt);
    ss = fmaf(s[k], s[k], ss);
  }
  const float inv = rsqrtf(fmaf(cta_sum(ss, part), a.inv_n, a.eps));
#pragma unroll
  for (int k = 0; k < E; ++k) {
    const int i = threadIdx.x + k * blockDim.x;
    if (i >= a.n) break;
    if (RS && a.ro) store_y_rt(a.ro, a.rt, row * a.ldro + i, s[k]);
    float v = s[k] * inv;
    if (a.w) v *= load_y_rt(a.w, a.wt, i) + a.c;
    store_y_rt(a.y, a.yt, row * a.ldy + i, v);
  }
}

// Wider rows yet: read twice, each value again by the thread that read it first (so that y may
// be x and ro may be r).
__global__ void __launch_bounds__(1024) rms_norm_wide_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float part[32];
  pdl_wait();
  pdl_trigger();
  const int64_t row = blockIdx.x;
  auto sum_at = [&](int i) {
    float v = load_y_rt(a.x, a.xt, row * a.ldx + i);
    if (a.r) v += load_y_rt(a.r, a.rt, row * a.ldr + i);
    return v;
  };
  float ss = 0.f;
  for (int i = threadIdx.x; i < a.n; i += blockDim.x) {
    const float v = sum_at(i);
    ss = fmaf(v, v, ss);
  }
  const float inv = rsqrtf(fmaf(cta_sum(ss, part), a.inv_n, a.eps));
  for (int i = threadIdx.x; i < a.n; i += blockDim.x) {
    float v = sum_at(i);
    if (a.ro) store_y_rt(a.ro, a.rt, row * a.ldro + i, v);
    v *= inv;
    if (a.w) v *= load_y_rt(a.w, a.wt, i) + a.c;
    store_y_rt(a.y, a.yt, row * a.ldy + i, v);
  }
}

template <int XS, int RS>
cudaError_t launch_any(const NormArgs& a, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(a.m));
  auto block = [&](int e) { return dim3(static_cast<unsigned>((((a.n + e - 1) / e) + 31) / 32 * 32)); };
  if (a.n <= 4096) return pdl_launch(rms_norm_any_kernel<8, XS, RS>, grid, block(8), 0, st, a);
  if (a.n <= 8192) return pdl_launch(rms_norm_any_kernel<16, XS, RS>, grid, block(16), 0, st, a);
  return pdl_launch(rms_norm_wide_kernel, grid, dim3(1024), 0, st, a);
}

template <int XS, int RS>
cudaError_t launch_vec(const NormArgs& a, cudaStream_t st) {
  const int groups = a.n / 8;
  const dim3 rows8(static_cast<unsigned>((static_cast<int64_t>(a.m) + 7) / 8)), rows(static_cast<unsigned>(a.m));
  // a warp per row up to 1024 values, above it a CTA with two (up to 16384) or four groups
  if (groups <= 32) return pdl_launch(rms_norm_vec_kernel<XS, RS, 1, true, false>, rows8, dim3(256), 0, st, a);
  if (groups <= 64) return pdl_launch(rms_norm_vec_kernel<XS, RS, 2, true, false>, rows8, dim3(256), 0, st, a);
  if (groups <= 128) return pdl_launch(rms_norm_vec_kernel<XS, RS, 4, true, false>, rows8, dim3(256), 0, st, a);
  const int v = groups <= 2048 ? 2 : 4;
  const dim3 block(static_cast<unsigned>(((groups + v - 1) / v + 31) / 32 * 32));
  if (v == 2) return pdl_launch(rms_norm_vec_kernel<XS, RS, 2, false, false>, rows, block, 0, st, a);
  return pdl_launch(rms_norm_vec_kernel<XS, RS, 4, false, false>, rows, block, 0, st, a);
}

// One group a thread where that makes a CTA of up to 512: 38 registers, so that three of them hide
// each other's loads, sums and weights (8192 bf16 rows of 4095 without r 45 us; two groups 54).
template <int XS, int RS>
cudaError_t launch_shift(const NormArgs& a, cudaStream_t st) {
  const int groups = (a.n + 14) / 8;  // at the largest shift
  if (groups <= 128)
    return pdl_launch(rms_norm_vec_kernel<XS, RS, 4, true, true>, dim3(static_cast<unsigned>((static_cast<int64_t>(a.m) + 7) / 8)),
                      dim3(256), 0, st, a);
  const int v = groups <= 512 ? 1 : groups <= 1024 ? 2 : 4;
  const dim3 rows(static_cast<unsigned>(a.m)), block(static_cast<unsigned>(((groups + v - 1) / v + 31) / 32 * 32));
  if (v == 1) return pdl_launch(rms_norm_vec_kernel<XS, RS, 1, false, true>, rows, block, 0, st, a);
  if (v == 2) return pdl_launch(rms_norm_vec_kernel<XS, RS, 2, false, true>, rows, block, 0, st, a);
  return pdl_launch(rms_norm_vec_kernel<XS, RS, 4, false, true>, rows, block, 0, st, a);
}

cudaError_t launch_norm(const NormArgs& a, cudaStream_t st) {
  auto whole = [](const void* p, int dt, int64_t ld) {  // null, or 16-byte aligned in every row
    return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * (dt == GGUFMM_F32 ? 4 : 2) % 16 == 0);
  };
  if (a.n % 8 == 0 && a.n <= 32768 && whole(a.x, a.xt, a.ldx) && whole(a.r, a.rt, a.ldr) &&
      whole(a.ro, a.rt, a.ldro) && whole(a.w, a.wt, 0) && whole(a.y, a.yt, a.ldy)) {
    const bool x4 = a.xt == GGUFMM_F32;
    if (!a.r) return x4 ? launch_vec<4, 0>(a, st) : launch_vec<2, 0>(a, st);
    if (a.rt == GGUFMM_F32) return x4 ? launch_vec<4, 4>(a, st) : launch_vec<2, 4>(a, st);
    return x4 ? launch_vec<4, 2>(a, st) : launch_vec<2, 2>(a, st);
  }
  const bool x4 = a.xt == GGUFMM_F32;
  auto packed = [&](const void* p, int64_t ld) {  // null, or on 16 bytes and without a gap
    return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld == a.n);
  };
  if (a.n >= 8 && a.n <= 16368 && packed(a.x, a.ldx) && packed(a.r, a.ldr) && packed(a.ro, a.ldro) && packed(a.w, a.n) &&
      packed(a.y, a.ldy)) {
    if (!a.r) return x4 ? launch_shift<4, 0>(a, st) : launch_shift<2, 0>(a, st);
    if (a.rt == GGUFMM_F32) return x4 ? launch_shift<4, 4>(a, st) : launch_shift<2, 4>(a, st);
    return x4 ? launch_shift<4, 2>(a, st) : launch_shift<2, 2>(a, st);
  }
  if (!a.r) return x4 ? launch_any<4, 0>(a, st) : launch_any<2, 0>(a, st);
  if (a.rt == GGUFMM_F32) return x4 ? launch_any<4, 4>(a, st) : launch_any<2, 4>(a, st);
  return x4 ? launch_any<4, 2>(a, st) : launch_any<2, 2>(a, st);
}

int elem(int64_t dtype) { return dtype == GGUFMM_F32 ? 4 : dtype == GGUFMM_F16 || dtype == GGUFMM_BF16 ? 2 : 0; }
bool al(const void* p, int a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

}  // namespace

}  // namespace ggufmm

using namespace ggufmm;

extern "C" int ggufmm_rms_norm(const ggufmm_norm_args* args, void* stream) {
  if (!args) return GGUFMM_ERR_ARG;
  const ggufmm_norm_args& p = *args;
  const int xe = elem(p.x_dtype), ye = elem(p.y_dtype), we = p.w ? elem(p.w_dtype) : 1, re = p.resid ? elem(p.r_dtype) : 1;
  if (!xe || !ye || !we || !re) return GGUFMM_ERR_DTYPE;
  if (p.m < 0 || p.m > (int64_t(1) << 31) - 1 || p.n <= 0 || p.n > GGUFMM_NORM_MAX_N || p.ldx < p.n || p.ldy < p.n ||
      (p.resid && p.ldr < p.n) || (p.resid_out && p.ldro < p.n))
    return GGUFMM_ERR_SHAPE;
  if (p.resid_out && !p.resid) return GGUFMM_ERR_ARG;
  if (!(p.eps >= 0.)) return GGUFMM_ERR_ARG;
  if (p.m == 0) return GGUFMM_OK;
  if (!p.x || !p.y) return GGUFMM_ERR_ARG;
  if (!al(p.x, xe) || !al(p.y, ye) || !al(p.w, we) || !al(p.resid, re) || !al(p.resid_out, re)) return GGUFMM_ERR_ALIGN;
  const int s = check_device();
  if (s) return s;
  NormArgs a;
  a.x = p.x;
  a.r = p.resid;
  a.ro = p.resid_out;
  a.w = p.w;
  a.y = p.y;
  a.ldx = p.ldx;
  a.ldr = p.ldr;
  a.ldro = p.ldro;
  a.ldy = p.ldy;
  a.m = static_cast<int>(p.m);
  a.n = static_cast<int>(p.n);
  a.xt = static_cast<int>(p.x_dtype);
  a.rt = static_cast<int>(p.r_dtype);
  a.wt = static_cast<int>(p.w_dtype);
  a.yt = static_cast<int>(p.y_dtype);
  a.c = static_cast<float>(p.w_add);
  a.eps = static_cast<float>(p.eps);
  a.inv_n = 1.f / static_cast<float>(a.n);
  return record_cuda_status(launch_norm(a, static_cast<cudaStream_t>(stream)));
}
