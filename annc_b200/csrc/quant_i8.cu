// 8-bit integer layers: quantisation per row, weights quantised per output channel, and the dispatcher of the
// product  C[m,n] = act(sum_k A[m,k] B[n,k] * scale_a[m] * scale_b[n] + bias[n]).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <cstring>

#include "common.h"
#include "gemm_i8.h"
#include "pdl.cuh"

namespace annc {
namespace gemm_i8 {

namespace {

// ---------------------------------------------------------------- quantisation
// A row's step is scale = max(max|x| / 127, 2^-126), nearest in fp32 (the lower end keeps it a normal number, so
// that nothing below divides by zero), and q the whole number nearest to x / scale, halves to even.  A row with an
// infinity or a NaN has the step NaN and q = 0: its products are NaN, as they would be in floating point.

// The nearest whole number exactly, also where the quotient of two fp32 numbers lies next to a half.  The guess comes
// from adding 1.5 * 2^23 (the sum's last place is one, its low byte the number) and may be one off there; the
// remainder x - q * scale has no more bits than fp32 holds (both are multiples of the smaller one's last place and the
// difference is little more than half a step), so that comparing it decides.
constexpr float kRound = 12582912.0f;
struct Guess {
  float sum, rem;
};
__device__ __forceinline__ Guess guess_of(float x, float scale, float inv) {
  Guess g;
  g.sum = __fmaf_rn(x, inv, kRound);
  g.rem = __fmaf_rn(kRound - g.sum, scale, x);
  return g;
}
// Below half a step either way the guess stands; beyond, or just half and odd, it is the neighbour.
__device__ __forceinline__ float settled(Guess g, float half) {
  const bool odd = __float_as_int(g.sum) & 1;
  if (fabsf(g.rem) > half || (fabsf(g.rem) == half && odd)) return g.sum + (g.rem > 0.0f ? 1.0f : -1.0f);
  return g.sum;
}
__device__ __forceinline__ int8_t quantize_one(float x, float scale, float inv) {
  return (int8_t)__float_as_int(settled(guess_of(x, scale, inv), 0.5f * scale));
}
// Largest |x| as the bits of a non-negative float, which order as the floats do, infinities and NaN on top.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
struct Step {
  float scale, inv;
  bool finite;
};
__device__ __forceinline__ Step step_of(uint32_t top) {
  Step s;
  s.finite = top < 0x7f800000u;
  s.scale = s.finite ? fmaxf(__fdiv_rn(__uint_as_float(top), 127.0f), 1.17549435e-38f) : __uint_as_float(0x7fc00000u);
  s.inv = __frcp_rn(s.scale);
  return s;
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

// The same over a piece of values: of two-byte types two at a time, as they lie.
template <typename T, int V>
__device__ __forceinline__ void top_of(const T (&v)[V], uint32_t& top) {
  if (sizeof(T) == 4 || V == 1) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      uint32_t w = 0;
      memcpy(&w, &v[e], sizeof(T));
      top = max(top, w & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fffu));
    }
  } else {
#pragma unroll
    for (int e = 0; e + 1 < V; e += 2) {
      uint32_t w;
      memcpy(&w, &v[e], 4);
      top = __vmaxu2(top, w & 0x7fff7fffu);
    }
  }
}
// ... to the bits of a float.
template <typename T>
__device__ __forceinline__ uint32_t top_bits(uint32_t top) {
  if (sizeof(T) == 4) return top;
  const uint16_t most = (uint16_t)max(top & 0xffffu, top >> 16);
  T v;
  memcpy(&v, &most, 2);
  return __float_as_uint(to_float(v));
}

template <int BYTES>
struct Words;
template <>
struct Words<16> { using type = uint4; };
template <>
struct Words<8> { using type = uint2; };
template <>
struct Words<4> { using type = uint32_t; };
struct QuantParams {
  const void* x;
  long long ld;
  int8_t* q;
  long long ldq;
  float* scale;
  long long rows;
  int cols;
  int unit;  // (QUADS) values of a load: 4, 2 or 1
};
// WIDE: rows of x are whole 16-byte pieces at 16-byte addresses.  QUADS: four values, loaded as x's addresses allow and
// stored as a word (rows of q at 4-byte addresses); the last piece of a row may have fewer.  SINGLES: one value at a time.
// us by quads / singles: 4730 x 2583 bf16 15.4 / 21.0, 1756 x 1121 f32 4.6 / 6.9, 15000 x 213 f16 7.3 / 6.6.
enum Pieces { WIDE, QUADS, SINGLES };

// TPR threads take a row; a thread keeps NV pieces of V values in registers between the maximum and the rounding, so
// that a row of up to TPR * NV * V values is read once; what is longer is read again, from L2.  Bound by memory once the
// rounding takes few enough instructions (8192 x 2048 bf16 31 us with rintf, a conversion and a branch for every value) and a
// thread has several pieces on their way (65536 x 256 bf16, a warp a row, one piece a lane, 27 us).
template <typename T, int TPR, Pieces KIND>
__global__ void __launch_bounds__(256) quantize_rows_kernel(QuantParams p) {
  constexpr int V = KIND == WIDE ? 16 / (int)sizeof(T) : KIND == QUADS ? 4 : 1;
  constexpr int NV = KIND == SINGLES ? 16 : 8;
  const int t = threadIdx.x % TPR, lane = threadIdx.x & 31;
  const long long at_row = (long long)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  pdl_trigger();
  pdl_wait();
  const bool there = at_row < p.rows;
  const long long row = there ? at_row : 0;
  const T* x = static_cast<const T*>(p.x) + row * p.ld;
  int8_t* q = p.q + row * p.ldq;
  const int pieces = there ? (p.cols + V - 1) / V : 0;

  alignas(16) T keep[NV][V];
  auto load = [&](int piece, T (&to)[V]) {
    if constexpr (KIND == WIDE) {
      *reinterpret_cast<uint4*>(to) = *(reinterpret_cast<const uint4*>(x) + piece);
    } else if constexpr (KIND == QUADS) {
      using Four = typename Words<4 * sizeof(T)>::type;
      using Two = typename Words<2 * sizeof(T)>::type;
      if (4 * piece + 4 > p.cols) {
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = 4 * piece + e < p.cols ? x[4 * piece + e] : T(0.0f);
      } else if (p.unit == 4) {
        *reinterpret_cast<Four*>(to) = *(reinterpret_cast<const Four*>(x) + piece);
      } else if (p.unit == 2) {
        reinterpret_cast<Two*>(to)[0] = reinterpret_cast<const Two*>(x)[2 * piece];
        reinterpret_cast<Two*>(to)[1] = reinterpret_cast<const Two*>(x)[2 * piece + 1];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = x[4 * piece + e];
      }
    } else {
      to[0] = x[piece];
    }
  };
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (t + i * TPR < pieces) load(t + i * TPR, keep[i]);
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (t + i * TPR < pieces) top_of(keep[i], top);
  for (int c = t + NV * TPR; c < pieces; c += TPR) {
    alignas(16) T v[V];
    load(c, v);
    top_of(v, top);
  }
  top = top_bits<T>(top);
#pragma unroll
  for (int d = 1; d < 32 && d < TPR; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (TPR > 32) {
    __shared__ uint32_t tops[8];
    const int warp = threadIdx.x >> 5;
    if (lane == 0) tops[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TPR / 32; ++w) top = max(top, tops[warp / (TPR / 32) * (TPR / 32) + w]);
  }
  const Step s = step_of(top);
  const float half = 0.5f * s.scale;
  if (t == 0 && there) p.scale[row] = s.scale;

  auto store = [&](int piece, const T (&v)[V]) {
    Guess g[V];
    float worst = 0.0f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      g[e] = guess_of(to_float(v[e]), s.scale, s.inv);
      worst = fmaxf(worst, fabsf(g[e].rem));
    }
    if (!(worst < half)) {  // hardly ever: a quotient next to a half, or a row that is not finite (half is NaN then)
#pragma unroll
      for (int e = 0; e < V; ++e) g[e].sum = s.finite ? settled(g[e], half) : 0.0f;
    }
    if (V == 1) {
      q[piece] = (int8_t)__float_as_int(g[0].sum);
    } else {
      uint32_t w[V < 4 ? 1 : V / 4];
#pragma unroll
      for (int j = 0; j < V / 4; ++j) {
        const uint32_t lo = __byte_perm(__float_as_uint(g[4 * j].sum), __float_as_uint(g[4 * j + 1].sum), 0x0040);
        const uint32_t hi = __byte_perm(__float_as_uint(g[4 * j + 2].sum), __float_as_uint(g[4 * j + 3].sum), 0x0040);
        w[j] = __byte_perm(lo, hi, 0x5410);
      }
      if (KIND == QUADS && 4 * piece + 4 > p.cols) {
        for (int e = 0; 4 * piece + e < p.cols; ++e) q[4 * piece + e] = (int8_t)(w[0] >> (8 * e));
      } else if (V == 8) *(reinterpret_cast<uint2*>(q) + piece) = make_uint2(w[0], w[V / 4 - 1]);
      else *(reinterpret_cast<uint32_t*>(q) + piece) = w[0];
    }
  };
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (t + i * TPR < pieces) store(t + i * TPR, keep[i]);
  for (int c = t + NV * TPR; c < pieces; c += TPR) {
    alignas(16) T v[V];
    load(c, v);
    store(c, v);
  }
}

// fp32 [K,N] -> int8 [N,K] with a step per column: a block takes 32 columns, reads them for their maxima and
// again (from L2) to round and turn them in shared memory.  A weight is converted once.
__global__ void __launch_bounds__(256)
i8_weight_kernel(const float* __restrict__ src, long long ldb, int8_t* __restrict__ dst, long long ldq,
                 float* __restrict__ scale, int K, int N) {
  __shared__ uint32_t tops[8][32];
  __shared__ int8_t tile[32][132];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int n0 = blockIdx.x * 32, n = n0 + tx;
  uint32_t top = 0;
  if (n < N)
    for (int k = ty; k < K; k += 8) top = max(top, abs_bits(src[(long long)k * ldb + n]));
  tops[ty][tx] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) top = max(top, tops[w][tx]);
  const Step s = step_of(top);
  if (ty == 0 && n < N) scale[n] = s.scale;
  for (int k0 = 0; k0 < K; k0 += 128) {
    for (int r = ty; r < 128; r += 8)
      tile[tx][r] = n < N && k0 + r < K && s.finite
                        ? quantize_one(src[(long long)(k0 + r) * ldb + n], s.scale, s.inv) : (int8_t)0;
    __syncthreads();
    for (int c = ty; c < 32; c += 8)
      if (n0 + c < N)
        for (int r = tx; r < 128; r += 32)
          if (k0 + r < K) dst[(long long)(n0 + c) * ldq + k0 + r] = tile[c][r];
    __syncthreads();
  }
}

// ---------------------------------------------------------------- CUDA-core product
// Takes every pitch and address: tiles of 64 x 64, k in steps of 64 bytes, four products a __dp4a; a thread holds
// 4 x 4 sums.  For operands whose rows are not at 16-byte addresses, which the tensor-core kernels do not take.
constexpr int ST = 64;

template <typename T>
__global__ void __launch_bounds__(256) gemm_i8_simt_kernel(Params p) {
  __shared__ __align__(16) int8_t sa[ST][ST + 4], sb[ST][ST + 4];  // rows of 17 words: no bank twice
  const int m0 = blockIdx.y * ST, n0 = blockIdx.x * ST;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < p.k; k0 += ST) {
    for (int e = threadIdx.x; e < ST * ST; e += 256) {
      const int r = e / ST, c = e % ST;
      const bool in = k0 + c < p.k;
      sa[r][c] = in && m0 + r < p.m ? p.a[(long long)(m0 + r) * p.lda + k0 + c] : (int8_t)0;
      sb[r][c] = in && n0 + r < p.n ? p.b[(long long)(n0 + r) * p.ldb + k0 + c] : (int8_t)0;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < ST; kk += 4) {
      int va[4], vb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        va[i] = *reinterpret_cast<const int*>(&sa[ty + 16 * i][kk]);
        vb[i] = *reinterpret_cast<const int*>(&sb[tx + 16 * i][kk]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(va[i], vb[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = m0 + ty + 16 * i;
    if (r >= p.m) continue;
    const float s = p.scale_a[r];
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = n0 + tx + 16 * j;
      v[j] = c < p.n ? scaled(acc[i][j], s, p.scale_b[c], p.bias ? p.bias[c] : 0.0f) : 0.0f;
    }
    activate(p.act, v);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n0 + tx + 16 * j < p.n) static_cast<T*>(p.c)[r * p.ldc + n0 + tx + 16 * j] = to_type<T>(v[j]);
  }
}

// A grid has at most 65535 tiles of rows: more than that, some 4 million rows, take several launches.  (Tiles along x alone, or along
// y and z, cost every product 5 to 10 %: 16384 x 1024 x 1001 620 us, with z 648, with x 655.)
template <typename T>
int run_simt_as(Params p, cudaStream_t s) {
  constexpr int most = 65535 * ST;
  for (int rows = p.m; rows > 0; rows -= p.m) {
    p.m = rows < most ? rows : most;
    gemm_i8_simt_kernel<T><<<dim3((unsigned)((p.n + ST - 1) / ST), (unsigned)((p.m + ST - 1) / ST)), 256, 0, s>>>(p);
    ANNC_CUDA(cudaGetLastError());
    if (p.a) p.a += p.m * p.lda;
    p.scale_a += p.m;
    p.c = static_cast<T*>(p.c) + p.m * p.ldc;
  }
  return ANNC_OK;
}
int run_simt(const Params& p, cudaStream_t s) {
  if (p.c_dtype == ANNC_F32) return run_simt_as<float>(p, s);
  if (p.c_dtype == ANNC_BF16) return run_simt_as<__nv_bfloat16>(p, s);
  return run_simt_as<__half>(p, s);
}

template <typename T>
int launch_quantize(QuantParams p, cudaStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  if (p.rows == 1) p.ld = p.ldq = 0;  // (where a next row would be does not matter)
  const bool wide = p.cols % V == 0 && p.ld % V == 0 && (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 && p.ldq % V == 0 &&
                    (reinterpret_cast<uintptr_t>(p.q) & (V - 1)) == 0;
  const bool quads = !wide && p.ldq % 4 == 0 && (reinterpret_cast<uintptr_t>(p.q) & 3) == 0;
  for (p.unit = 4; p.unit > 1 && (p.ld % p.unit || (reinterpret_cast<uintptr_t>(p.x) & (p.unit * sizeof(T) - 1))); p.unit /= 2) {
  }
  const int each = wide ? V : quads ? 4 : 1, pieces = (p.cols + each - 1) / each;
  // As few threads a row as hold it in registers (eight pieces each, 16 singles), but two blocks an SM if the rows give them.
  // 64 threads read up to half of a row again before 256 take it, which wait for one another: 8192 x 5120 bf16 33 / 43 us,
  // 16384 x 8192 80 / 95, 2000 x 6000 11.6 / 10.8.  (16 threads that do so: 8192 x 2048 14.8 us, 64 threads 12.0.)
  int tpr = 4;
  while (tpr < 256 && (pieces > (tpr == 64 || each == 1 ? 16 : 8) * tpr || p.rows * tpr < 2 * 148 * 256)) tpr *= 4;
  const long long blocks = (p.rows + 256 / tpr - 1) / (256 / tpr);
  ANNC_REQUIRE(blocks <= 0x7fffffffLL, ANNC_ERR_UNSUPPORTED, "quantize rows: too many rows");
  static void (*const kernels[3][4])(QuantParams) = {
      {quantize_rows_kernel<T, 4, WIDE>, quantize_rows_kernel<T, 16, WIDE>, quantize_rows_kernel<T, 64, WIDE>, quantize_rows_kernel<T, 256, WIDE>},
      {quantize_rows_kernel<T, 4, QUADS>, quantize_rows_kernel<T, 16, QUADS>, quantize_rows_kernel<T, 64, QUADS>, quantize_rows_kernel<T, 256, QUADS>},
      {quantize_rows_kernel<T, 4, SINGLES>, quantize_rows_kernel<T, 16, SINGLES>, quantize_rows_kernel<T, 64, SINGLES>, quantize_rows_kernel<T, 256, SINGLES>}};
  ANNC_CUDA(launch_pdl(kernels[wide ? WIDE : quads ? QUADS : SINGLES][tpr == 4 ? 0 : tpr == 16 ? 1 : tpr == 64 ? 2 : 3], dim3((unsigned)blocks), dim3(256), 0, s, p));
  return ANNC_OK;
}

int validate(const annc_gemm_i8_desc& d) {
  ANNC_REQUIRE(d.m >= 0 && d.n >= 0 && d.k >= 0 && d.m <= (1LL << 30) && d.n <= (1LL << 30), ANNC_ERR_INVALID_ARGUMENT,
               "gemm i8: bad extents");
  // 131071 * 128 * 128 is below 2^31: no sum of so many products leaves 32 bits
  ANNC_REQUIRE(d.k <= 131071, ANNC_ERR_UNSUPPORTED, "gemm i8: k above 131071 (the sums are kept in 32 bits)");
  ANNC_REQUIRE(d.lda >= d.k && d.ldb >= d.k && d.ldc >= d.n, ANNC_ERR_INVALID_ARGUMENT, "gemm i8: bad leading dimension");
  ANNC_REQUIRE(d.activation >= ANNC_ACT_NONE && d.activation <= ANNC_ACT_SIGMOID, ANNC_ERR_INVALID_ARGUMENT,
               "gemm i8: bad activation");
  ANNC_REQUIRE(d.c_dtype == ANNC_F32 || d.c_dtype == ANNC_BF16 || d.c_dtype == ANNC_F16, ANNC_ERR_INVALID_ARGUMENT,
               "gemm i8: C is f32, bf16 or f16");
  if (d.m == 0 || d.n == 0) return ANNC_OK;
  ANNC_REQUIRE((d.k == 0 || (d.a && d.b)) && d.c && d.scale_a && d.scale_b, ANNC_ERR_INVALID_ARGUMENT, "gemm i8: null operand");
  const uintptr_t es = d.c_dtype == ANNC_F32 ? 4 : 2;
  ANNC_REQUIRE(((reinterpret_cast<uintptr_t>(d.scale_a) | reinterpret_cast<uintptr_t>(d.scale_b) |
                 reinterpret_cast<uintptr_t>(d.bias)) & 3) == 0 && (reinterpret_cast<uintptr_t>(d.c) & (es - 1)) == 0,
               ANNC_ERR_INVALID_ARGUMENT, "gemm i8: operand not aligned to its type");
  return ANNC_OK;
}

Params params_of(const annc_gemm_i8_desc& d) {
  // the pitch of a single row does not matter: one that the tensor-core kernels take
  const long long whole = (d.k + 15) / 16 * 16;
  return Params{d.a, d.b, d.scale_a, d.scale_b, d.bias, d.c, d.m == 1 ? whole : d.lda, d.n == 1 ? whole : d.ldb, d.ldc, (int)d.m, (int)d.n, (int)d.k,
                d.c_dtype, d.activation};
}

}  // namespace
}  // namespace gemm_i8
}  // namespace annc

using namespace annc;

extern "C" {

int annc_gemm_i8_run(const annc_gemm_i8_desc* desc, void* stream) {
  ANNC_REQUIRE(desc, ANNC_ERR_INVALID_ARGUMENT, "gemm i8: null descriptor");
  ANNC_TRY(gemm_i8::validate(*desc));
  if (desc->m == 0 || desc->n == 0) return ANNC_OK;
  const gemm_i8::Params p = gemm_i8::params_of(*desc);
  const gemm_i8::Route r = gemm_i8::route_of(p);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return r.kind == gemm_i8::ROUTE_SIMT ? gemm_i8::run_simt(p, s) : gemm_i8::run_tc(p, r, s);
}

const char* annc_gemm_i8_kernel_name(const annc_gemm_i8_desc* desc) {
  if (!desc) return "";
  switch (gemm_i8::route_of(gemm_i8::params_of(*desc)).kind) {
    case gemm_i8::ROUTE_PAIR: return "tcgen05_pair_i8";
    case gemm_i8::ROUTE_SPLIT: return "tcgen05_i8";
    default: return "simt_i8";
  }
}

int annc_quantize_rows_dev(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t ld, int8_t* q,
                           int64_t ldq, float* scale, void* stream) {
  ANNC_REQUIRE(dtype == ANNC_F32 || dtype == ANNC_BF16 || dtype == ANNC_F16, ANNC_ERR_INVALID_ARGUMENT,
               "quantize rows: x is f32, bf16 or f16");
  ANNC_REQUIRE(rows >= 0 && cols >= 0 && cols < (1LL << 30) && ld >= cols && ldq >= cols, ANNC_ERR_INVALID_ARGUMENT,
               "quantize rows: bad extents");
  if (rows == 0) return ANNC_OK;
  ANNC_REQUIRE((cols == 0 || (x && q)) && scale, ANNC_ERR_INVALID_ARGUMENT, "quantize rows: null operand");
  const uintptr_t es = dtype == ANNC_F32 ? 4 : 2;
  ANNC_REQUIRE((reinterpret_cast<uintptr_t>(x) & (es - 1)) == 0 && (reinterpret_cast<uintptr_t>(scale) & 3) == 0,
               ANNC_ERR_INVALID_ARGUMENT, "quantize rows: operand not aligned to its type");
  const gemm_i8::QuantParams p{x, ld, q, ldq, scale, rows, (int)cols};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == ANNC_F32) return gemm_i8::launch_quantize<float>(p, s);
  if (dtype == ANNC_BF16) return gemm_i8::launch_quantize<__nv_bfloat16>(p, s);
  return gemm_i8::launch_quantize<__half>(p, s);
}

int annc_i8_weight_dev(const float* b_kn, int64_t ldb, int8_t* b_nk, int64_t ldq, float* scale, int64_t k, int64_t n,
                       void* stream) {
  ANNC_REQUIRE(b_kn && b_nk && scale && k >= 1 && n >= 1 && k < (1LL << 30) && n < (1LL << 30) && ldb >= n && ldq >= k,
               ANNC_ERR_INVALID_ARGUMENT, "i8 weight: bad arguments");
  ANNC_REQUIRE(((reinterpret_cast<uintptr_t>(b_kn) | reinterpret_cast<uintptr_t>(scale)) & 3) == 0, ANNC_ERR_INVALID_ARGUMENT,
               "i8 weight: operand not aligned to its type");
  gemm_i8::i8_weight_kernel<<<(unsigned)((n + 31) / 32), 256, 0, static_cast<cudaStream_t>(stream)>>>(b_kn, ldb, b_nk, ldq,
                                                                                                     scale, (int)k, (int)n);
  ANNC_CUDA(cudaGetLastError());
  return ANNC_OK;
}

}  // extern "C"
