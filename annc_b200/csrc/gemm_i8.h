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
// Two values of one token, of two channels: the same roundings, two to an instruction.
__device__ __forceinline__ void scaled2(int sum0, int sum1, float scale_a, float2 scale_b, float2 bias, float* v0, float* v1) {
  asm("{\n\t.reg .b64 s, a, b, c;\n\t"
      "mov.b64 s, {%2, %3};\n\t"
      "mov.b64 a, {%4, %4};\n\t"
      "mov.b64 b, {%5, %6};\n\t"
      "mov.b64 c, {%7, %8};\n\t"
      "mul.rn.f32x2 s, s, a;\n\t"
      "fma.rn.f32x2 s, s, b, c;\n\t"
      "mov.b64 {%0, %1}, s;\n\t}"
      : "=f"(*v0), "=f"(*v1)
      : "f"((float)sum0), "f"((float)sum1), "f"(scale_a), "f"(scale_b.x), "f"(scale_b.y), "f"(bias.x), "f"(bias.y));
}
// 1 / (1 + 2^(-v log2 e)) by the special-function unit, both instructions within 2 ulp.  The product in the exponent
// rounds once, which moves the power by |v| 2^-24, as the rounding of v itself did; below -87.3, where the value is less than the
// smallest normal number, it is zero.  (With expf and a division 16384 x 1024 x 64 took 28 us, without activation 14.5.)
__device__ __forceinline__ float sigmoid(float v) {
  float e, y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.0f + e));
  return y;
}
template <int N>
__device__ __forceinline__ void activate(int act, float (&v)[N]) {
  if (act == ANNC_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(v[j]));  // (a NaN stays one)
  } else if (act == ANNC_ACT_SIGMOID) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = sigmoid(v[j]);
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
