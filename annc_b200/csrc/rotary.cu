// Rotary positions: pairs (a, b) of a head's first rot_dim values are turned by angle = position * freq[pair],
//   (a, b) -> size * (a cos - b sin, b cos + a sin),
// the rest of the head is passed through.  Pairs are (j, j + rot/2) in the half layout, (2j, 2j + 1) interleaved.
//
// Bound by memory: every value is read and written once.  A block takes a few tokens: it first works out their
// sines and cosines, once for all heads of queries and keys (in 64 bits up to the fraction of a turn, since
// position * freq of a far position has no bits left behind the point in 32; then in 32), and then moves the heads
// through in pieces of 16 bytes, two pieces a thread in flight.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <cstdint>

#include "common.h"
#include "pdl.cuh"

namespace annc {
namespace rotary {

namespace {

struct Heads {
  const void* in;
  void* out;
  long long in_token, in_head, out_token, out_head;  // in elements
};
struct Params {
  Heads x[2];
  const void* positions;
  const double* freq;
  float size;
  int heads0, heads;  // of the first tensor, of both
  int dim, rot, pos64, transposed, pass, pass_pieces;  // pass: values behind rot_dim that have to be copied
  int tokens_per_block;
  uint32_t units_magic, heads_magic;
  long long tokens;
};

constexpr int kMaxRot = 512;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_float(float x, float* y) { *y = x; }
__device__ __forceinline__ void from_float(float x, __nv_bfloat16* y) { *y = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_float(float x, __half* y) { *y = __float2half_rn(x); }

template <int BYTES>
struct Piece;
template <>
struct Piece<16> { using type = uint4; };
template <>
struct Piece<8> { using type = uint2; };
template <>
struct Piece<4> { using type = uint32_t; };
template <>
struct Piece<2> { using type = uint16_t; };

// i / d by one multiplication where i * d stays below 2^32 (magic = 2^32 / d rounded up), else (magic 0) by division.
__device__ __forceinline__ int quotient(int i, int d, uint32_t magic) { return magic ? (int)__umulhi((uint32_t)i, magic) : i / d; }

// V values make a piece.  A unit of work is the two pieces that hold V pairs (in the half layout pairs / 2 values apart,
// interleaved adjacent), behind rot_dim two pieces that are copied, or one.  (Interleaved units of one piece, with three divisions
// each, were bound by their instructions: 8191 tokens of 40 heads of 128 bf16 42 us.)
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(256) rotary_kernel(Params p) {
  using P = typename Piece<V * (int)sizeof(T)>::type;
  extern __shared__ float turns[];  // cosines [tokens][pairs], then sines
  constexpr int U = 2;  // units of a thread in flight
  const int pairs = p.rot >> 1;
  const long long t0 = (long long)blockIdx.x * p.tokens_per_block;
  const int nt = (int)min((long long)p.tokens_per_block, p.tokens - t0);
  float* const cosines = turns;
  float* const sines = turns + p.tokens_per_block * pairs;
  const int turned = pairs / V, units = turned + p.pass / (p.pass_pieces * V);
  const int total = nt * p.heads * units, other = HALF ? pairs : V;  // from a unit's one piece to its other
  P a[U], b[U];
  T* out[U];
  int pair[U];

  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + 256 * u;
      out[u] = nullptr;
      if (i >= total) continue;
      const int th = quotient(i, units, p.units_magic), unit = i - th * units;
      const int t = quotient(th, p.heads, p.heads_magic);
      int h = th - t * p.heads;
      const Heads& x = p.x[h >= p.heads0];
      if (h >= p.heads0) h -= p.heads0;
      const bool turn = unit < turned;
      const int first = !turn ? p.rot + (unit - turned) * p.pass_pieces * V : (HALF ? V : 2 * V) * unit;
      pair[u] = turn ? t * pairs + unit * V : -1;
      const T* in = static_cast<const T*>(x.in) + (t0 + t) * x.in_token + h * x.in_head + first;
      out[u] = static_cast<T*>(x.out) + (t0 + t) * x.out_token + h * x.out_head + first;
      a[u] = *reinterpret_cast<const P*>(in);
      if (turn || p.pass_pieces == 2) b[u] = *reinterpret_cast<const P*>(in + (turn ? other : V));
    }
  };
  pdl_trigger();
  pdl_wait();
  load(threadIdx.x);  // (on their way while the sines are worked out)

  for (int i = threadIdx.x; i < nt * pairs; i += 256) {
    const int t = i / pairs;
    const double at = p.pos64 ? (double)static_cast<const int64_t*>(p.positions)[t0 + t]
                              : (double)static_cast<const int32_t*>(p.positions)[t0 + t];
    double turn = at * p.freq[i - t * pairs] * 0.15915494309189533577;  // 1 / (2 pi)
    turn -= rint(turn);
    float s, c;
    sincospif((float)(2.0 * turn), &s, &c);
    cosines[i] = c * p.size;
    sines[i] = (p.transposed ? -s : s) * p.size;
  }
  __syncthreads();

  for (int i0 = threadIdx.x; i0 < total; i0 += 256 * U) {
    if (i0 != (int)threadIdx.x) load(i0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!out[u]) continue;
      if (pair[u] >= 0) {
        const float* c = cosines + pair[u];
        const float* s = sines + pair[u];
        T* va = reinterpret_cast<T*>(&a[u]);
        T* vb = reinterpret_cast<T*>(&b[u]);
        if (HALF || V == 1) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float x = to_float(va[e]), y = to_float(vb[e]);
            from_float(x * c[e] - y * s[e], &va[e]);
            from_float(y * c[e] + x * s[e], &vb[e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            T* const v = e < V / 2 ? va + 2 * e : vb + 2 * e - V;
            const float x = to_float(v[0]), y = to_float(v[V > 1 ? 1 : 0]);
            from_float(x * c[e] - y * s[e], &v[0]);
            from_float(y * c[e] + x * s[e], &v[V > 1 ? 1 : 0]);
          }
        }
        *reinterpret_cast<P*>(out[u] + other) = b[u];
      } else if (p.pass_pieces == 2) {
        *reinterpret_cast<P*>(out[u] + V) = b[u];
      }
      *reinterpret_cast<P*>(out[u]) = a[u];
    }
  }
}

// Largest piece that every address, stride and boundary inside a head allows, in values.
template <typename T>
int piece_values(const annc_rotary_desc& d, int pass) {
  for (int v : {16 / (int)sizeof(T), 8 / (int)sizeof(T)}) {
    bool ok = d.rot_dim / 2 % v == 0 && (pass == 0 || (pass % v == 0 && d.rot_dim % v == 0));
    for (const annc_rotary_heads& x : d.x) {
      if (x.heads == 0) continue;
      ok = ok && ((reinterpret_cast<uintptr_t>(x.in) | reinterpret_cast<uintptr_t>(x.out)) & (v * sizeof(T) - 1)) == 0 &&
           ((x.in_token | x.in_head | x.out_token | x.out_head) & (v - 1)) == 0;
    }
    if (ok) return v;
  }
  return 1;
}

template <typename T>
int launch(const annc_rotary_desc& d, cudaStream_t s) {
  Params p = {};
  bool in_place = true;
  int n = 0;
  for (const annc_rotary_heads& x : d.x) {
    if (x.heads == 0) continue;
    p.x[n++] = Heads{x.in, x.out, x.in_token, x.in_head, x.out_token, x.out_head};
    in_place = in_place && x.in == x.out && x.in_token == x.out_token && x.in_head == x.out_head;
    if (n == 1) p.heads0 = x.heads;
    p.heads += x.heads;
  }
  p.positions = d.positions;
  p.freq = d.freq;
  p.size = d.size;
  p.dim = d.head_dim;
  p.rot = d.rot_dim;
  p.pos64 = d.positions_dtype == ANNC_I64;
  p.transposed = d.transposed;
  p.pass = in_place ? 0 : d.head_dim - d.rot_dim;
  p.tokens = d.tokens;
  const int v = piece_values<T>(d, p.pass);
  p.pass_pieces = p.pass % (2 * v) == 0 ? 2 : 1;
  // Tokens of a block: about 2048 pieces of work, at most what 16 KB of sines hold, but first of all a grid that
  // fills the 148 SMs four times over.
  const long long per_token = (long long)p.heads * (d.head_dim / v);
  long long tb = 2048 / (per_token > 0 ? per_token : 1);
  if (tb > 2048 / (d.rot_dim / 2)) tb = 2048 / (d.rot_dim / 2);
  if (tb > d.tokens / 592) tb = d.tokens / 592;
  if (tb < 1) tb = 1;
  p.tokens_per_block = (int)tb;
  const long long units = d.rot_dim / 2 / v + p.pass / (p.pass_pieces * v), total = tb * p.heads * units;
  if (units > 1 && total * units < (1LL << 32)) p.units_magic = (uint32_t)(((1ULL << 32) + units - 1) / units);
  if (p.heads > 1 && total * p.heads < (1LL << 32)) p.heads_magic = (uint32_t)(((1ULL << 32) + p.heads - 1) / p.heads);
  const long long blocks = (d.tokens + tb - 1) / tb;
  ANNC_REQUIRE(blocks <= 0x7fffffffLL, ANNC_ERR_UNSUPPORTED, "rotary: too many tokens");
  const size_t smem = (size_t)tb * d.rot_dim * sizeof(float);
  const bool half = d.layout == ANNC_ROTARY_HALF;
  constexpr int V16 = 16 / (int)sizeof(T), V8 = 8 / (int)sizeof(T);
  void (*const kernel)(Params) = v == V16 ? (half ? rotary_kernel<T, V16, true> : rotary_kernel<T, V16, false>)
                               : v == V8  ? (half ? rotary_kernel<T, V8, true> : rotary_kernel<T, V8, false>)
                                          : (half ? rotary_kernel<T, 1, true> : rotary_kernel<T, 1, false>);
  ANNC_CUDA(launch_pdl(kernel, dim3((unsigned)blocks), dim3(256), smem, s, p));
  return ANNC_OK;
}

int validate(const annc_rotary_desc& d) {
  ANNC_REQUIRE(d.dtype == ANNC_F32 || d.dtype == ANNC_BF16 || d.dtype == ANNC_F16, ANNC_ERR_INVALID_ARGUMENT,
               "rotary: the heads are f32, bf16 or f16");
  ANNC_REQUIRE(d.layout == ANNC_ROTARY_HALF || d.layout == ANNC_ROTARY_INTERLEAVED, ANNC_ERR_INVALID_ARGUMENT,
               "rotary: bad layout");
  ANNC_REQUIRE(d.positions_dtype == ANNC_I32 || d.positions_dtype == ANNC_I64, ANNC_ERR_INVALID_ARGUMENT,
               "rotary: positions are i32 or i64");
  ANNC_REQUIRE(d.rot_dim >= 2 && d.rot_dim % 2 == 0 && d.rot_dim <= kMaxRot && d.head_dim >= d.rot_dim &&
                   d.head_dim <= (1 << 20), ANNC_ERR_INVALID_ARGUMENT,
               "rotary: rot_dim is even, from 2 to 512, and not above head_dim");
  ANNC_REQUIRE(d.tokens >= 0, ANNC_ERR_INVALID_ARGUMENT, "rotary: bad extents");
  const uintptr_t es = d.dtype == ANNC_F32 ? 4 : 2;
  long long heads = 0;
  for (const annc_rotary_heads& x : d.x) {
    ANNC_REQUIRE(x.heads >= 0 && x.heads <= 65536, ANNC_ERR_INVALID_ARGUMENT, "rotary: bad number of heads");
    heads += x.heads;
    if (x.heads == 0 || d.tokens == 0) continue;
    ANNC_REQUIRE(x.in && x.out, ANNC_ERR_INVALID_ARGUMENT, "rotary: null operand");
    ANNC_REQUIRE(((reinterpret_cast<uintptr_t>(x.in) | reinterpret_cast<uintptr_t>(x.out)) & (es - 1)) == 0,
                 ANNC_ERR_INVALID_ARGUMENT, "rotary: operand not aligned to its type");
  }
  if (d.tokens == 0 || heads == 0) return ANNC_OK;
  ANNC_REQUIRE(heads * d.head_dim <= (1LL << 26), ANNC_ERR_UNSUPPORTED, "rotary: more than 2^26 values a token");
  ANNC_REQUIRE(d.positions && d.freq && (reinterpret_cast<uintptr_t>(d.freq) & 7) == 0 &&
                   (reinterpret_cast<uintptr_t>(d.positions) & (d.positions_dtype == ANNC_I64 ? 7 : 3)) == 0,
               ANNC_ERR_INVALID_ARGUMENT, "rotary: positions or frequencies missing or not aligned to their type");
  return ANNC_OK;
}

}  // namespace
}  // namespace rotary
}  // namespace annc

using namespace annc;

extern "C" {

int annc_rotary_frequencies(int32_t rot_dim, double base, int32_t scaling, double factor, int64_t original_len,
                            double beta_fast, double beta_slow, double* freq, float* size) {
  ANNC_REQUIRE(rot_dim >= 2 && rot_dim % 2 == 0 && rot_dim <= rotary::kMaxRot, ANNC_ERR_INVALID_ARGUMENT,
               "rotary: rot_dim is even, from 2 to 512");
  ANNC_REQUIRE(freq && size, ANNC_ERR_INVALID_ARGUMENT, "rotary: null output");
  ANNC_REQUIRE(base > 1.0 && std::isfinite(base), ANNC_ERR_INVALID_ARGUMENT, "rotary: base has to be above 1");
  ANNC_REQUIRE(scaling >= ANNC_ROTARY_UNSCALED && scaling <= ANNC_ROTARY_YARN, ANNC_ERR_INVALID_ARGUMENT, "rotary: bad scaling");
  ANNC_REQUIRE(scaling == ANNC_ROTARY_UNSCALED || (factor >= 1.0 && std::isfinite(factor)), ANNC_ERR_INVALID_ARGUMENT,
               "rotary: factor has to be 1 or more");
  ANNC_REQUIRE(scaling != ANNC_ROTARY_YARN || (original_len >= 1 && beta_slow > 0.0 && beta_fast >= beta_slow && std::isfinite(beta_fast)),
               ANNC_ERR_INVALID_ARGUMENT, "rotary: yarn needs original_len >= 1 and beta_fast >= beta_slow > 0");
  const double pi = 3.14159265358979323846, d = rot_dim;
  *size = 1.0f;
  if (scaling == ANNC_ROTARY_NTK && rot_dim > 2) base *= std::pow(factor, d / (d - 2.0));
  double low = 0.0, high = 0.0;
  if (scaling == ANNC_ROTARY_YARN) {
    // the pair that turns `turns` times within original_len
    auto pair_of = [&](double turns) { return d * std::log((double)original_len / (turns * 2.0 * pi)) / (2.0 * std::log(base)); };
    low = std::fmax(std::floor(pair_of(beta_fast)), 0.0);
    high = std::fmin(std::ceil(pair_of(beta_slow)), d - 1.0);
    *size = (float)(0.1 * std::log(factor) + 1.0);
  }
  for (int j = 0; j < rot_dim / 2; ++j) {
    const double f = std::pow(base, -2.0 * j / d);
    if (scaling == ANNC_ROTARY_LINEAR) {
      freq[j] = f / factor;
    } else if (scaling == ANNC_ROTARY_YARN) {
      const double ramp = std::fmin(std::fmax((j - low) / std::fmax(high - low, 0.001), 0.0), 1.0);
      freq[j] = f / factor * ramp + f * (1.0 - ramp);
    } else {
      freq[j] = f;
    }
  }
  return ANNC_OK;
}

int annc_rotary_dev(const annc_rotary_desc* desc, void* stream) {
  ANNC_REQUIRE(desc, ANNC_ERR_INVALID_ARGUMENT, "rotary: null descriptor");
  ANNC_TRY(rotary::validate(*desc));
  if (desc->tokens == 0 || (desc->x[0].heads == 0 && desc->x[1].heads == 0)) return ANNC_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (desc->dtype == ANNC_F32) return rotary::launch<float>(*desc, s);
  if (desc->dtype == ANNC_BF16) return rotary::launch<__nv_bfloat16>(*desc, s);
  return rotary::launch<__half>(*desc, s);
}

}  // extern "C"
