// Internal interface of the 8-bit integer product.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "annc_b200.h"

namespace annc {
namespace gemm_i8 {

struct Params {
  const int8_t* a;  // [m, k], rows lda bytes apart
  const int8_t* b;  // [n, k], rows ldb bytes apart
  const float* scale_a;
  const float* scale_b;
  const float* bias;  // or null
  void* c;
  long long lda, ldb, ldc;
  int m, n, k;
  int c_dtype, act;
};

// How a product is run: on CUDA cores, by the split kernel (tokens per tile, CTAs per tile), or
// by the pair kernel.
enum RouteKind { ROUTE_SIMT = 0, ROUTE_SPLIT = 1, ROUTE_PAIR = 2 };
struct Route {
  RouteKind kind;
  int tokens, split;
};
Route route_of(const Params& p);
int run_tc(const Params& p, const Route& r, cudaStream_t s);

#ifdef __CUDACC__
// act(sum * scale_a * scale_b + bias).  The sum of products is exact (32-bit integers); it is rounded to fp32 once
// (sums above 2^24), and the two scalings, the addition and C's type round once each.
__device__ __forceinline__ float scaled(int sum, float scale_a, float scale_b, float bias) {
  return fmaf((float)sum * scale_a, scale_b, bias);
}
// Out of line: the loops that hardly ever take it stay small.  (The quotient within 2 ulp; correctly rounded it took a
// third of what 1999 x 1003 x 1001 takes.)
static __device__ __noinline__ float4 sigmoid4(float4 v) {
  return make_float4(__fdividef(1.0f, 1.0f + expf(-v.x)), __fdividef(1.0f, 1.0f + expf(-v.y)), __fdividef(1.0f, 1.0f + expf(-v.z)),
                     __fdividef(1.0f, 1.0f + expf(-v.w)));
}
template <int N>
__device__ __forceinline__ void activate(int act, float (&v)[N]) {
  static_assert(N % 4 == 0, "");
  if (act == ANNC_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = v[j] < 0.0f ? 0.0f : v[j];  // (a NaN stays one)
  } else if (act == ANNC_ACT_SIGMOID) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const float4 t = sigmoid4(make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]));
      v[j] = t.x; v[j + 1] = t.y; v[j + 2] = t.z; v[j + 3] = t.w;
    }
  }
}
template <typename T>
__device__ __forceinline__ T to_type(float v);
template <>
__device__ __forceinline__ float to_type<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 to_type<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half to_type<__half>(float v) { return __float2half_rn(v); }
#endif

}  // namespace gemm_i8
}  // namespace annc
