// Attention of a batch whose sequences share one long prefix of keys and values.
//
//   out[t, h, :] = sum_j p_j V_j,   p = softmax(scale * q[t, h, :] . K_j)
//
// over the keys j of the prefix, which every token sees, and those of the token's own sequence: token i of its
// sequence's n tokens sees all own keys but the last n - 1 - i.  A token without any key gets zeros.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <cstdint>

#include "common.h"
#include "prefix_attention.h"

namespace annc {
namespace attention {

namespace {

__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_float(float x, __nv_bfloat16* y) { *y = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_float(float x, __half* y) { *y = __float2half_rn(x); }

constexpr int kMaxDim = 256;

// One warp a token and head, lanes along the head's values, four keys at a time: takes every stride, head size, group and
// scale, for the calls that the tensor-core kernels do not (tc_supported).
template <typename T>
__global__ void __launch_bounds__(128) attention_rows_kernel(Params p) {
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const long long token = row / p.heads;
  const int h = (int)(row - token * p.heads), g = h / p.group;
  if (token >= p.tokens) return;
  long long first;
  int count;
  if (!own_keys(p, token, &first, &count)) return;
  constexpr int N = kMaxDim / 32, U = 4;
  // (the maximum starts at the lowest number, not at -inf: scores of -inf alone then have weights of 0, not of exp(-inf + inf))
  float q[N], acc[N] = {}, top = -3.402823466e38f, sum = 0.0f;
  const T* qp = static_cast<const T*>(p.q.data) + token * p.q.row + h * p.q.head;
#pragma unroll
  for (int i = 0; i < N; ++i) q[i] = lane + 32 * i < p.dim ? to_float(qp[lane + 32 * i]) : 0.0f;
  for (int part = 0; part < 2; ++part) {
    const Rows& k = part ? p.ko : p.kp;
    const Rows& v = part ? p.vo : p.vp;
    const long long from = part ? first : 0, to = part ? first + count : p.prefix;
    for (long long j = from; j < to; j += U) {
      float s[U], w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[u] = 0.0f;
        if (j + u >= to) continue;
        const T* kr = static_cast<const T*>(k.data) + (j + u) * k.row + g * k.head;
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (lane + 32 * i < p.dim) s[u] = fmaf(q[i], to_float(kr[lane + 32 * i]), s[u]);
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], d);
      float now = top;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[u] = j + u < to ? __fmul_rn(s[u], p.scale) : -INFINITY;
        now = fmaxf(now, s[u]);
      }
      const float keep = expf(top - now);
      top = now;
      sum *= keep;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        w[u] = j + u < to ? expf(__fsub_rn(s[u], now)) : 0.0f;
        sum += w[u];
      }
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] *= keep;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (j + u >= to) continue;
        const T* vr = static_cast<const T*>(v.data) + (j + u) * v.row + g * v.head;
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (lane + 32 * i < p.dim) acc[i] = fmaf(w[u], to_float(vr[lane + 32 * i]), acc[i]);
      }
    }
  }
  const bool none = p.prefix + count == 0;
  T* o = static_cast<T*>(p.out) + token * p.out_row + h * p.out_head;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (lane + 32 * i < p.dim) from_float(none ? 0.0f : acc[i] / sum, &o[lane + 32 * i]);
  if (p.lse && lane == 0) p.lse[token * p.heads + h] = none ? -INFINITY : top + logf(sum);
}

int run_rows(const Params& p, int dtype, cudaStream_t s) {
  const long long blocks = (p.tokens * p.heads + 3) / 4;
  ANNC_REQUIRE(blocks <= 0x7fffffffLL, ANNC_ERR_UNSUPPORTED, "prefix attention: too many tokens");
  if (dtype == ANNC_BF16) attention_rows_kernel<__nv_bfloat16><<<(unsigned)blocks, 128, 0, s>>>(p);
  else attention_rows_kernel<__half><<<(unsigned)blocks, 128, 0, s>>>(p);
  ANNC_CUDA(cudaGetLastError());
  return ANNC_OK;
}

int validate(const annc_prefix_attention_desc& d) {
  ANNC_REQUIRE(d.dtype == ANNC_BF16 || d.dtype == ANNC_F16, ANNC_ERR_INVALID_ARGUMENT, "prefix attention: operands are bf16 or f16");
  ANNC_REQUIRE(d.kv_heads >= 1 && d.heads >= d.kv_heads && d.heads % d.kv_heads == 0 && d.heads <= 65536,
               ANNC_ERR_INVALID_ARGUMENT, "prefix attention: heads have to be a multiple of kv_heads");
  ANNC_REQUIRE(d.head_dim >= 1 && d.head_dim <= kMaxDim, ANNC_ERR_INVALID_ARGUMENT, "prefix attention: head_dim is 1 to 256");
  ANNC_REQUIRE(d.tokens >= 0 && d.tokens < (1LL << 31) && d.prefix_len >= 0 && d.prefix_len < (1LL << 31) && d.own_rows >= 0 &&
                   d.sequences >= 0 && d.sequences < (1LL << 31), ANNC_ERR_INVALID_ARGUMENT, "prefix attention: bad extents");
  ANNC_REQUIRE(d.q_begin || d.sequences == d.tokens, ANNC_ERR_INVALID_ARGUMENT,
               "prefix attention: without q_begin every token is a sequence");
  ANNC_REQUIRE(std::isfinite(d.scale), ANNC_ERR_INVALID_ARGUMENT, "prefix attention: bad scale");
  if (d.tokens == 0) return ANNC_OK;
  const bool own = d.own_len != nullptr;
  ANNC_REQUIRE(d.q && d.out && (d.prefix_len == 0 || (d.k_prefix && d.v_prefix)), ANNC_ERR_INVALID_ARGUMENT,
               "prefix attention: null operand");
  ANNC_REQUIRE(!own || (d.own_begin && (d.own_rows == 0 || (d.k_own && d.v_own))), ANNC_ERR_INVALID_ARGUMENT,
               "prefix attention: own keys need k_own, v_own, own_begin and own_len");
  const uintptr_t all = reinterpret_cast<uintptr_t>(d.q) | reinterpret_cast<uintptr_t>(d.out) |
                        reinterpret_cast<uintptr_t>(d.k_prefix) | reinterpret_cast<uintptr_t>(d.v_prefix) |
                        reinterpret_cast<uintptr_t>(d.k_own) | reinterpret_cast<uintptr_t>(d.v_own);
  const uintptr_t words = reinterpret_cast<uintptr_t>(d.lse) | reinterpret_cast<uintptr_t>(d.own_len) |
                          reinterpret_cast<uintptr_t>(d.q_begin);
  ANNC_REQUIRE((all & 1) == 0 && (words & 3) == 0 && (reinterpret_cast<uintptr_t>(d.own_begin) & 7) == 0,
               ANNC_ERR_INVALID_ARGUMENT, "prefix attention: operand not aligned to its type");
  return ANNC_OK;
}

Params params_of(const annc_prefix_attention_desc& d) {
  Params p = {};
  p.q = Rows{d.q, d.q_row, d.q_head};
  p.kp = Rows{d.k_prefix, d.k_prefix_row, d.k_prefix_head};
  p.vp = Rows{d.v_prefix, d.v_prefix_row, d.v_prefix_head};
  p.ko = Rows{d.k_own, d.k_own_row, d.k_own_head};
  p.vo = Rows{d.v_own, d.v_own_row, d.v_own_head};
  p.out = d.out;
  p.out_row = d.out_row;
  p.out_head = d.out_head;
  p.lse = d.lse;
  p.own_begin = d.own_begin;
  p.own_len = d.own_len;
  p.q_begin = d.q_begin;
  p.tokens = d.tokens;
  p.sequences = d.sequences;
  p.prefix = d.prefix_len;
  p.own_rows = d.own_rows;
  p.heads = d.heads;
  p.kv_heads = d.kv_heads;
  p.group = d.heads / d.kv_heads;
  p.dim = d.head_dim;
  p.scale = d.scale;
  return p;
}

}  // namespace
}  // namespace attention
}  // namespace annc

using namespace annc;

extern "C" {

size_t annc_prefix_attention_workspace_bytes(int64_t tokens, int32_t heads, int32_t kv_heads, int32_t head_dim) {
  if (tokens < 1 || kv_heads < 1 || heads < kv_heads || heads % kv_heads || head_dim < 1) return 0;
  return attention::tc_workspace_bytes(tokens, heads, kv_heads, head_dim);
}

int annc_prefix_attention_dev(const annc_prefix_attention_desc* desc, void* stream) {
  ANNC_REQUIRE(desc, ANNC_ERR_INVALID_ARGUMENT, "prefix attention: null descriptor");
  ANNC_TRY(attention::validate(*desc));
  if (desc->tokens == 0) return ANNC_OK;
  const size_t need = annc_prefix_attention_workspace_bytes(desc->tokens, desc->heads, desc->kv_heads, desc->head_dim);
  ANNC_REQUIRE(need == 0 || (desc->workspace && (reinterpret_cast<uintptr_t>(desc->workspace) & 15) == 0 &&
                             desc->workspace_bytes >= need), ANNC_ERR_INVALID_ARGUMENT,
               "prefix attention: workspace missing, too small or not 16-byte aligned");
  const attention::Params p = attention::params_of(*desc);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return attention::tc_supported(p, desc->dtype) ? attention::run_tc(p, desc->dtype, desc->workspace, s)
                                                 : attention::run_rows(p, desc->dtype, s);
}

}  // extern "C"
