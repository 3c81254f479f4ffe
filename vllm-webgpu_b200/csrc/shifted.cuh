// shifted.cuh -- eight consecutive values out of the two aligned groups of eight that hold
// them. Plain C++ too, so that its reads are checked without a GPU.
#pragma once

#ifdef __CUDACC__
#define GGUFMM_HD __host__ __device__ __forceinline__
#else
#define GGUFMM_HD inline
#endif

namespace ggufmm {

// The values of a vector of n from i = 8 g - shift on (0 <= shift < 8) into w. load8(j, v) reads
// v[0..7] from the aligned j, load1(j) one value, both of them inside the vector alone: i is that of
// a row's group, so for the last ones not only the second but also the first group may end behind
// n. What lies outside the vector is 0.
template <class Load8, class Load1>
GGUFMM_HD void shifted8(int i, int shift, int n, const Load8& load8, const Load1& load1, float* w) {
  float v[16], a[12], b[10];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int j = i + shift - 8 + 8 * h;
    if (j >= 0 && j + 8 <= n) {
      load8(j, v + 8 * h);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[8 * h + e] = j >= 0 && j + e < n ? load1(j + e) : 0.f;
    }
  }
#pragma unroll
  for (int e = 0; e < 12; ++e) a[e] = shift & 4 ? v[e] : v[e + 4];
#pragma unroll
  for (int e = 0; e < 10; ++e) b[e] = shift & 2 ? a[e] : a[e + 2];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = shift & 1 ? b[e + 1] : b[e + 2];
}

}  // namespace ggufmm
