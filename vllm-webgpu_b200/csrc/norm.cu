// norm.cu -- ggufmm_rms_norm: root-mean-square norm of each row, with the residual's
// addition in front of it.
//
//   s = x + r,  y = s * rsqrt(mean(s^2) + eps) * (w + c),  r' = s
//
// The reference runs its add shader and its rms_norm shader as two dispatches
// (vllm_webgpu/models/llama.py:262-270, :335-341; shaders/generic/{add,rms_norm}.wgsl),
// with the stream rounded to f16 between them. Here the sum stays in 32 bits: it is
// rounded once into r' and, after the norm, once into y.
#include "common.cuh"

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
  int n;
  int xt, rt, wt, yt;
  float c, eps;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// One row per CTA, two passes over it.
__global__ void __launch_bounds__(256) rms_norm_kernel(NormArgs a) {
  __shared__ float part[8];
  pdl_wait();
  pdl_trigger();
  const int64_t row = blockIdx.x;
  float ss = 0.f;
  for (int i = threadIdx.x; i < a.n; i += 256) {
    float s = load_y_rt(a.x, a.xt, row * a.ldx + i);
    if (a.r) s += load_y_rt(a.r, a.rt, row * a.ldr + i);
    ss = fmaf(s, s, ss);
  }
  ss = warp_sum(ss);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = ss;
  __syncthreads();
  float tot = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) tot += part[i];
  const float inv = rsqrtf(tot / static_cast<float>(a.n) + a.eps);
  // each element is read again and written by the thread that read it: y may be x and
  // ro may be r, element for element
  for (int i = threadIdx.x; i < a.n; i += 256) {
    float s = load_y_rt(a.x, a.xt, row * a.ldx + i);
    if (a.r) s += load_y_rt(a.r, a.rt, row * a.ldr + i);
    if (a.ro) store_y_rt(a.ro, a.rt, row * a.ldro + i, s);
    float v = s * inv;
    if (a.w) v *= load_y_rt(a.w, a.wt, i) + a.c;
    store_y_rt(a.y, a.yt, row * a.ldy + i, v);
  }
}

int elem(int dtype) { return dtype == GGUFMM_F32 ? 4 : dtype == GGUFMM_F16 || dtype == GGUFMM_BF16 ? 2 : 0; }
bool al(const void* p, int a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

}  // namespace

}  // namespace ggufmm

using namespace ggufmm;

extern "C" int ggufmm_rms_norm(const void* x, int x_dtype, int64_t m, int64_t n, int64_t ldx, const void* resid,
                               int r_dtype, int64_t ldr, void* resid_out, int64_t ldro, const void* w, int w_dtype,
                               float w_add, float eps, void* y, int y_dtype, int64_t ldy, void* stream) {
  const int xe = elem(x_dtype), ye = elem(y_dtype), we = w ? elem(w_dtype) : 1, re = resid ? elem(r_dtype) : 1;
  if (!xe || !ye || !we || !re) return GGUFMM_ERR_DTYPE;
  if (m < 0 || m > (int64_t(1) << 31) - 1 || n <= 0 || n > GGUFMM_NORM_MAX_N || ldx < n || ldy < n ||
      (resid && ldr < n) || (resid_out && ldro < n))
    return GGUFMM_ERR_SHAPE;
  if (resid_out && !resid) return GGUFMM_ERR_ARG;
  if (!(eps >= 0.f)) return GGUFMM_ERR_ARG;
  if (m == 0) return GGUFMM_OK;
  if (!x || !y) return GGUFMM_ERR_ARG;
  if (!al(x, xe) || !al(y, ye) || !al(w, we) || !al(resid, re) || !al(resid_out, re)) return GGUFMM_ERR_ALIGN;
  const int s = check_device();
  if (s) return s;
  const NormArgs a{x, resid, resid_out, w, y, ldx, ldr, ldro, ldy, static_cast<int>(n), x_dtype, r_dtype, w_dtype,
                   y_dtype, w_add, eps};
  return record_cuda_status(pdl_launch(rms_norm_kernel, dim3(static_cast<unsigned>(m)), dim3(256), 0,
                                       static_cast<cudaStream_t>(stream), a));
}
