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

// How a product is run: on CUDA cores, by the split kernel (tokens per tile, CTAs per tile), or by the pair kernel.
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
__device__ __forceinline__ float finish(const Params& p, int sum, float scale_a, float scale_b, float bias) {
  const float v = fmaf((float)sum * scale_a, scale_b, bias);
  if (p.act == ANNC_ACT_RELU) return v < 0.0f ? 0.0f : v;  // (a NaN stays one)
  if (p.act == ANNC_ACT_SIGMOID) return __fdiv_rn(1.0f, 1.0f + expf(-v));
  return v;
}
__device__ __forceinline__ void store_out(const Params& p, long long row, int col, float v) {
  const long long at = row * p.ldc + col;
  if (p.c_dtype == ANNC_F32) static_cast<float*>(p.c)[at] = v;
  else if (p.c_dtype == ANNC_BF16) static_cast<__nv_bfloat16*>(p.c)[at] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p.c)[at] = __float2half_rn(v);
}
#endif

}  // namespace gemm_i8
}  // namespace annc
