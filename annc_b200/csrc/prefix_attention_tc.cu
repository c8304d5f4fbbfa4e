// Shared-prefix attention on the 5th-generation tensor cores: one kernel takes all rows against the prefix, a second
// one adds the keys of each sequence and joins the parts.
//
// Prefix kernel.  A CTA walks through its share of key tiles (plan_of in prefix_attention.h).  Per key tile of 128 keys and
// tile of 128 rows:  S = Q K^T (tcgen05, operands in shared memory, S in tensor memory), softmax numerators P in
// registers (a thread per row), P back to tensor memory as the operand of  O += P V  (V as it lies, N-major).  Heads of
// more than 64 values leave P no place but over S, so the next S waits for that product; with up to 64 values P has
// columns of its own and the next S is made while the exponentials are taken.
// Two such chains run side by side so that one's products cover the other's exponentials: with more than 128 rows
// in the item the two are its two row tiles, sharing the key tiles; else they take the key tiles in turn and are added
// at the end of the segment, the first one reading the other's O from tensor memory.  The running maximum of a row only
// moves when a score passes it by more than 2^8 in the exponential: until then O keeps its scale, the numerators grow to
// at most 256, and O is rescaled hardly ever.  (Of f16 they are raised by 2^7 on top, so that small ones keep their bits.)
// A tile with a row whose maximum is beyond 2^21, or -inf, goes a longer way: 2048 tokens of 16 heads
// (two key heads) of 64 over 1024 keys 25 us, 20 else.
//
// What bounds it: with 64 values the 16 exponentials a cycle of the SM (2048 of some 2560 cycles for two tiles of 128 x 128;
// a half, a third, a quarter or a sixth of them on the multiply-add units by a polynomial: 212, 187, 181 and 188 us where
// it is 184 without), with 128 values the way from P to the next S, which waits for two products (2048 cycles of
// products in some 3700).  Sixteen softmax warps, two for a row, had 96 registers each and were slower (210 us for 134), and so
// were half tiles of 64 keys with two places for S, which need no wait (161 us): half of a softmax step's time does not
// depend on the number of keys.
//
//   warps 0-3, 4-7   softmax of the two chains, rescaling of O, parts
//   warp 8           TMA: rows, then keys and values through a ring of tiles
//   warp 9           tensor memory, all products
//
// Join kernel.  Warps take (token, key head): its heads against the token's own keys with mma.sync straight from global
// memory (each lane reads 16-byte pieces; the order of the head's values in the products is permuted alike on both
// sides), and the parts of the prefix are added in registers.  Without own keys, items that one CTA has all of are
// written by the prefix kernel.
//
// Sums, maxima and O are held in fp32; the numerators are rounded to the operands' type for the second product, as the
// tensor cores want them, while their sum is of the unrounded ones: half a step a weight, which the row kernel, on fp32
// weights, does not have (error relative to 64 bits 2.3e-3 in bf16, 2.9e-4 in f16; with fp32 weights 1.7e-3 and 2.1e-4).
#include <cuda.h>

#include <cmath>
#include <cstdint>
#include <cstring>
#include <type_traits>

#include "common.h"
#include "pdl.cuh"
#include "prefix_attention.h"
#include "tc_host.h"
#include "tc_ptx.cuh"

namespace annc {
namespace gemm {
int* gemm_error_word();  // device address of the tensor-core kernels' error word (gemm_tc.cu)
}
namespace attention {

namespace {

using namespace annc::tc;

constexpr int kThreads = 384;  // eight softmax warps, loads, products, and two that complete the group of four
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kSlack = 8.0f * kLn2;  // what a score may pass the maximum by before that moves: a numerator of 2^8
constexpr float kFar = 2097152.0f;     // scores from here on are rounded before their maximum is subtracted (softmax_tile)
// Maxima start here, not at -inf: where every score is -inf the numerators are then 0, not exp(-inf + inf).
constexpr float kLowest = -3.402823466e38f;

// Numerators of f16 are raised by a power of two, so that its range goes to small ones: 2^8 of slack and 2^7 are half of
// 65504, and a numerator is off by at most 2^-25 of what it is then, 2^-32 of the row's largest.  (As they are, 2^17 weights of 2^-26
// beside one of 1 were lost.)  The join kernel, whose maxima move at once, has 2^15.
template <typename T>
__host__ __device__ constexpr int raise_of(int slack) { return std::is_same<T, __half>::value ? 15 - slack : 0; }

template <int DP>
struct Shape {
  static constexpr int kTile = kTileKeys * DP * 2;  // bytes of 128 rows: DP / 64 blocks of 128 bytes x 128
  static constexpr int kSlots = DP == 128 ? 5 : 9;
  // Tensor memory: S of the chains at columns 0 and 128, then O, then P if it has room of its own.
  static constexpr bool kOwnP = DP == 64;
  static constexpr uint32_t kO = 256, kP = kOwnP ? 384 : 0, kPStep = kOwnP ? 64 : 128;
  static constexpr int kExchange = 2 * kTile + kSlots * kTile;  // the second chain's [128] (maximum, sum)
  static constexpr int kBars = kExchange + kTileRows * 8;
  static constexpr size_t kSmem = 1024 + kBars + 320;
};

// The own keys that a token sees; row < 0: a token of no sequence.
struct Own {
  long long row;
  int count, reserved;
};

// Whether the join kernel takes the prefix too, and there is no prefix kernel: always up to 64 keys, further with few
// (token, key head).  us with / without the prefix kernel: 500 ragged sequences, 8 heads of 64, 64 keys 30 / 27, 100 30 /
// 32; 2048 tokens, 2 key heads of 128, 64 keys 35 / 32, 100 35 / 43; 64 tokens, 8 key heads, 128 keys 18 / 14, 200 16 / 18;
// one token, 8 heads, 256 keys 9.7 / 6.0, 400 10.2 / 8.0.
inline bool is_short(long long prefix, long long units) {
  return prefix <= 64 || (units <= 512 && prefix <= 128) || (units <= 64 && prefix <= 320);
}

struct PrefixParams {
  Plan plan;
  Params a;
  long long tokens;
  int kv_heads, group, prefix, dim;
  float scale, scale2;  // scale2: scale * log2(e)
  // [part][DP / 4][256] pieces of four values: a lane writes its row, so rows are adjacent (row by row the writes, 32
  // pieces at 512 bytes from one another, took 5 us a segment)
  float4* parts;
  float2* stats;  // [part][256]: maximum, sum
  Own* own;       // per token, or null
  // no own keys, every token a sequence: what a CTA has all of goes out at once
  int direct;
  void* out;
  long long out_row, out_head;
  float* lse;
  int* error_word;
};

// ---------------------------------------------------------------- PTX
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}
// Products and their commits are issued by a whole warp, of which one lane is elected in the instruction itself: its
// operands then stay in uniform registers.  (From a branch that one lane takes, every product cost some 140 cycles to
// issue, where 128 x 128 x 16 takes 64: 2048 tokens of 16 heads against 8192 keys 165 us.)
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_commit_elected(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// As mbar_wait, but the clock is only looked at now and then: most waits here are as short as reading it.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* error_word) {
  unsigned long long t0 = 0;
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 0) {
      if (*abort_flag) return false;
      const unsigned long long now = global_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > 1000000000ull) {
        *abort_flag = 1;
        atomicExch(error_word, 1);
        return false;
      }
    }
  }
}
__device__ __forceinline__ bool all_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* error_word) {
  return __all_sync(0xffffffffu, wait(bar, parity, abort_flag, error_word)) != 0;
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Registers of the calling group of four warps: a softmax thread holds the 128 scores of its row.  Launched with 168 each,
// and 2 x 128 x 208 + 128 x 88 is what 384 x 168 makes.
__device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 208;"); }
__device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 88;"); }
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  uint32_t w;
  memcpy(&w, &v, 4);
  return w;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  uint32_t w;
  memcpy(&w, &v, 4);
  return w;
}

// ---------------------------------------------------------------- prefix kernel

// What a CTA does of one item: key tiles first .. first + count - 1.
struct Segment {
  int item, head, tile;  // key head, pair of row tiles
  int first, count;
  int part;
  bool whole;  // all of the item
  bool dual;   // two row tiles; else the chains take the key tiles in turn
  __device__ __forceinline__ int steps(int chain) const { return dual ? count : (count - chain + 1) / 2; }
  __device__ __forceinline__ int key_tile(int chain, int step) const { return first + (dual ? step : 2 * step + chain); }
};
__device__ __forceinline__ Segment segment_at(const PrefixParams& p, int at, int begin, int end) {
  Segment s;
  s.item = at / p.plan.kv_tiles;
  s.first = at - s.item * p.plan.kv_tiles;
  s.count = min(p.plan.kv_tiles - s.first, end - at);
  s.head = s.item / p.plan.row_items;
  s.tile = s.item - s.head * p.plan.row_items;
  s.dual = p.tokens - (long long)s.tile * 2 * p.plan.tile_tokens > p.plan.tile_tokens;
  s.whole = s.count == p.plan.kv_tiles;
  s.part = s.whole ? 2 * kMaxCtas + s.item : 2 * (int)blockIdx.x + (at == begin ? 0 : 1);
  return s;
}

// A row's 128 scores of one key tile (in tensor memory, a lane each) -> numerators in the operands' type in their
// place; the row's maximum `top` (of scale * q . k) and sum follow, and O where the maximum moves.  `half_ready` is
// signalled when the first 64 keys' numerators are written.  TAIL: only the first `valid` keys are there.
template <bool TAIL>
__device__ __forceinline__ float max32(const uint32_t (&r)[32], int first, int valid, float top) {
  float m[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int j = 0; j < 32; j += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = TAIL && first + j + i >= valid ? -INFINITY : __uint_as_float(r[j + i]);
      const float y = TAIL && first + j + 4 + i >= valid ? -INFINITY : __uint_as_float(r[j + 4 + i]);
      m[i] = max3(m[i], x, y);
    }
  return max3(max3(m[0], m[1], m[2]), m[3], m[3]);
}
template <typename T, bool TAIL>
__device__ __forceinline__ void exp32(const uint32_t (&r)[32], int first, int valid, float2 by, float2 minus, float2 (&sum)[2],
                                      uint32_t (&w)[16]) {
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    const float2 x = fma2(make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), by, minus);
    float2 e = make_float2(exp2_approx(x.x), exp2_approx(x.y));
    if (TAIL) {
      if (first + j >= valid) e.x = 0.0f;
      if (first + j + 1 >= valid) e.y = 0.0f;
    }
    sum[j / 2 & 1] = add2(sum[j / 2 & 1], e);
    w[j / 2] = pack2<T>(e.x, e.y);
  }
}
template <typename T, int DP, bool TAIL>
__device__ __forceinline__ bool softmax_tile(uint32_t t_s, uint32_t t_p, uint32_t t_o, float scale, float scale2, bool mine, bool first, int valid,
                                             float& top, float& sum, uint32_t half_ready, uint32_t scores_read, uint32_t p_used, uint32_t p_phase,
                                             volatile int* abort_flag, int* error_word) {
  bool ok = true;
  uint32_t r0[32], r1[32], r2[32], r3[32];
  tmem_ld32(t_s, r0);
  tmem_ld32(t_s + 32, r1);
  tmem_ld_wait();
  tmem_ld32(t_s + 64, r2);
  tmem_ld32(t_s + 96, r3);
  const float m0 = max32<TAIL>(r0, 0, valid, -INFINITY), m1 = max32<TAIL>(r1, 32, valid, -INFINITY);
  tmem_ld_wait();
  const float m2 = max32<TAIL>(r2, 64, valid, -INFINITY), m3 = max32<TAIL>(r3, 96, valid, -INFINITY);
  // (A row of the tile that is not there holds what lay in shared memory: it must not send the warp the long ways below.
  // 2000 tokens of three heads to each of two key heads of 64 over 8192 keys: 60 us, 44 so.)
  const float most = mine ? max3(max3(m0, m1, m2), m3, m3) : 0.0f, now = most * scale;
  if (Shape<DP>::kOwnP) {
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(scores_read);
    ok = all_wait(p_used, p_phase, abort_flag, error_word);  // the product before this one: it reads P and adds to O
    tc_fence_after();
  }
  // The numerator is 2^(score * scale2 - top * log2 e) in one operation, whose product is not rounded while the maximum is:
  // nothing as long as that is small.  Far out it is a power of anything, and where no score is above -inf that of NaN.
  const bool moves = first || now - top > kSlack, far = fabsf(now) >= kFar;
  const float old_top = top;
  if (moves) top = fmaxf(now, kLowest);
  constexpr float kRaise = raise_of<T>(8);
  float minus = kRaise - top * kLog2e;
  if (__any_sync(0xffffffffu, far || (moves && !first))) {
    if (!first) {
      // (the products before this are complete)
      const float keep = moves ? exp2_approx((old_top - top) * kLog2e) : 1.0f;
      sum *= keep;
#pragma unroll 1
      for (int b = 0; b < DP / 16; ++b) {
        uint32_t o[16];
        tmem_ld16(t_o + 16 * b, o);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
        tmem_st16(t_o + 16 * b, o);
      }
    }
    if (__any_sync(0xffffffffu, far)) {
      // Scores are rounded, then the maximum is subtracted, so that equal ones stay equal, and what is left is put in
      // their place as if it had come out of the product.  (Finite products that the scale takes to -inf, with nothing
      // above them so far, become NaN.)
      const float base = top == kLowest && most != -INFINITY ? now : top, up = 1.0f / scale;
      minus = kRaise;
      auto settle = [&](uint32_t (&r)[32]) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          asm volatile("{\n\t.reg .f32 x;\n\tmov.b32 x, %0;\n\tmul.rn.f32 x, x, %1;\n\tsub.rn.f32 x, x, %2;\n\tmul.rn.f32 x, x, %3;\n\tmov.b32 %0, x;\n\t}"
                       : "+r"(r[j]) : "f"(scale), "f"(base), "f"(up));
      };
      settle(r0);
      settle(r1);
      settle(r2);
      settle(r3);
    }
  }
  float2 sums[2] = {make_float2(sum, 0.0f), make_float2(0.0f, 0.0f)};
  const float2 by = make_float2(scale2, scale2), minus2 = make_float2(minus, minus);
  uint32_t w[16];
  exp32<T, TAIL>(r0, 0, valid, by, minus2, sums, w);
  tmem_st16(t_p, w);
  exp32<T, TAIL>(r1, 32, valid, by, minus2, sums, w);
  tmem_st16(t_p + 16, w);
  exp32<T, TAIL>(r2, 64, valid, by, minus2, sums, w);
  tmem_st_wait();  // (of the first 64, long done by now)
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(half_ready);
  tmem_st16(t_p + 32, w);
  exp32<T, TAIL>(r3, 96, valid, by, minus2, sums, w);
  tmem_st16(t_p + 48, w);
  sums[0] = add2(sums[0], sums[1]);
  sum = sums[0].x + sums[0].y;
  tmem_st_wait();
  return ok;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
prefix_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
              const __grid_constant__ CUtensorMap tmap_v, PrefixParams p) {
  using S = Shape<DP>;
  constexpr int kBlock = kTileKeys * 128;  // bytes of a block of 64 values x 128 rows
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t q_smem = base, ring = base + 2 * S::kTile, bars = base + S::kBars;
  const uint32_t bar_full = bars, bar_empty = bars + 8 * S::kSlots;
  const uint32_t bar_q = bars + 16 * S::kSlots, bar_qfree = bar_q + 8;
  const uint32_t bar_s = bar_q + 16, bar_p = bar_q + 32, bar_o = bar_q + 48, bar_ofree = bar_q + 64, bar_h = bar_q + 80;  // per chain
  const uint32_t bar_x = bar_q + 96, bar_read = bar_q + 104, bar_pv = bar_q + 120, bar_out = bar_q + 136;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_raw + (bar_q + 144 - raw));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* issued = tmem_slot + 2;  // by the loader: tiles of keys and values, segments' rows

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // (known to be uniform)
  if (threadIdx.x == 0) {
    prefetch_tensormap(&tmap_q);
    prefetch_tensormap(&tmap_k);
    prefetch_tensormap(&tmap_v);
    for (int s = 0; s < S::kSlots; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    mbar_init(bar_q, 1);
    mbar_init(bar_qfree, 1);
    for (int c = 0; c < 2; ++c) {
      mbar_init(bar_s + 8 * c, 1);
      mbar_init(bar_h + 8 * c, 4);  // the first 64 numerators of every row, all of them
      mbar_init(bar_p + 8 * c, 4);
      mbar_init(bar_o + 8 * c, 1);
      mbar_init(bar_ofree + 8 * c, 4);
      mbar_init(bar_read + 8 * c, 4);  // (P apart) S is in registers
      mbar_init(bar_pv + 8 * c, 1);    // (P apart) P is used
    }
    mbar_init(bar_x, 4);
    mbar_init(bar_out, 1);
    *abort_flag = 0;
    issued[0] = issued[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  pdl_wait();
  const int total = p.plan.items * p.plan.kv_tiles;
  const int begin = (int)blockIdx.x * p.plan.per_cta, end = min(total, begin + p.plan.per_cta);
  const bool poisoned = *reinterpret_cast<volatile int*>(p.error_word) != 0;  // an earlier launch gave up
  bool ok = !poisoned;

  if (warp >= 8) {
  registers_down();
  if (warp == 8) {
    if (ok && lane == 0) {
      uint32_t n = 0, segments = 0, rows_issued = 0;
      const uint32_t q_bytes = (uint32_t)(p.plan.tile_tokens * p.group) * 128u * (DP / 64);
      auto load = [&](const CUtensorMap* map, int head, int tile) {
        const int s = n % S::kSlots;
        ok = wait(bar_empty + 8 * s, ((n / S::kSlots) & 1u) ^ 1u, abort_flag, p.error_word);
        if (!ok) return;
        mbar_expect_tx(bar_full + 8 * s, S::kTile);
#pragma unroll
        for (int b = 0; b < DP / 64; ++b)
          tma_load_3d(ring + s * S::kTile + b * kBlock, map, 64 * b, head, tile * kTileKeys, bar_full + 8 * s);
        ++n;
      };
      for (int at = begin; at < end && ok; ++segments) {
        const Segment g = segment_at(p, at, begin, end);
        at += g.count;
        ok = wait(bar_qfree, (segments & 1u) ^ 1u, abort_flag, p.error_word);
        if (!ok) break;
        ++rows_issued;
        mbar_expect_tx(bar_q, g.dual ? 2 * q_bytes : q_bytes);
        for (int c = 0; c < (g.dual ? 2 : 1); ++c)
#pragma unroll
          for (int b = 0; b < DP / 64; ++b)
            tma_load_4d(q_smem + c * S::kTile + b * kBlock, &tmap_q, 64 * b, 0, g.head, (2 * g.tile + c) * p.plan.tile_tokens, bar_q);
        for (int t = 0; t < g.count && ok; ++t) {
          load(&tmap_k, g.head, g.first + t);
          if (ok) load(&tmap_v, g.head, g.first + t);
        }
      }
      issued[0] = n;
      issued[1] = rows_issued;
    }
  } else if (warp == 9) {
    if (ok) {
      constexpr uint32_t fmt = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      constexpr uint32_t idesc_s = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(kTileKeys >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
      constexpr uint32_t idesc_o =
          (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | ((uint32_t)(DP >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
      // (an address further on is a descriptor further on: the address field counts 16 bytes and cannot overflow)
      const uint64_t q_desc = smem_desc(q_smem, 16, 1024, 2), k_desc = smem_desc(ring, 16, 1024, 2),
                     v_desc = smem_desc(ring, kBlock, 1024, 2);
      uint32_t n0 = 0, segments = 0;  // ring number of the segment's first key tile
      uint32_t steps_done[2] = {0, 0};
      for (int at = begin; at < end && ok; ++segments) {
        const Segment g = segment_at(p, at, begin, end);
        at += g.count;
        ok = all_wait(bar_q, segments & 1u, abort_flag, p.error_word);
        if (!ok) break;
        const int most = g.steps(0);
        for (int step = 0; step <= most && ok; ++step) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int steps = g.steps(c);
            const uint32_t t_s = tmem + 128 * c, t_o = tmem + S::kO + DP * c, t_p = tmem + S::kP + S::kPStep * c;
            auto scores = [&]() {  // S = Q K^T
              const uint32_t i = n0 + 2 * (uint32_t)(g.key_tile(c, step) - g.first), s = i % S::kSlots;
              ok = all_wait(bar_full + 8 * s, (i / S::kSlots) & 1u, abort_flag, p.error_word);
              if (ok && S::kOwnP) ok = all_wait(bar_read + 8 * c, ((steps_done[c] + step) & 1u) ^ 1u, abort_flag, p.error_word);
              if (!ok) return;
              tc_fence_after();
              const uint64_t k = k_desc + s * (S::kTile >> 4), q = q_desc + (g.dual ? c : 0) * (S::kTile >> 4);
#pragma unroll
              for (int kk = 0; kk < DP / 16; ++kk) {
                const uint32_t off = ((kk / 4) * kBlock + (kk % 4) * 32) >> 4;
                umma_f16_ss(t_s, q + off, k + off, idesc_s, kk > 0 ? 1u : 0u);
              }
              if (!g.dual || c == 1) umma_commit_elected(bar_empty + 8 * s);
              umma_commit_elected(bar_s + 8 * c);
            };
            if (S::kOwnP && step < steps) scores();
            if (!ok) break;
            if (step > 0 && step <= steps) {  // O += P V of the step before
              const uint32_t i = n0 + 2 * (uint32_t)(g.key_tile(c, step - 1) - g.first) + 1, s = i % S::kSlots;
              const uint32_t phase = (steps_done[c] + step - 1) & 1u;
              ok = all_wait(bar_full + 8 * s, (i / S::kSlots) & 1u, abort_flag, p.error_word);
              if (ok && step == 1) ok = all_wait(bar_ofree + 8 * c, (segments & 1u) ^ 1u, abort_flag, p.error_word);
              const uint64_t v = v_desc + s * (S::kTile >> 4);
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                if (ok) ok = all_wait((half ? bar_p : bar_h) + 8 * c, phase, abort_flag, p.error_word);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int kk = 4 * half; kk < 4 * half + 4; ++kk)
                  umma_f16_ts(t_o, t_p + 8 * kk, v + (kk * 2048 >> 4), idesc_o, step > 1 || kk > 0 ? 1u : 0u);
              }
              if (!ok) break;
              if (!g.dual || c == 1) umma_commit_elected(bar_empty + 8 * s);
              if (S::kOwnP) umma_commit_elected(bar_pv + 8 * c);
              if (step == steps) umma_commit_elected(bar_o + 8 * c);
            }
            if (!S::kOwnP && step < steps) scores();
            if (!ok) break;
          }
          if (step == most - 1 && ok) umma_commit_elected(bar_qfree);  // the segment's last use of its rows
        }
        steps_done[0] += g.steps(0);
        steps_done[1] += g.steps(1);
        n0 += 2 * g.count;
      }
    }
  } else if (p.own) {
    // the two warps that have nothing else to do look up, for the join, what every token sees of its sequence
    for (long long t = (long long)blockIdx.x * 64 + (threadIdx.x - 320); t < p.tokens; t += (long long)gridDim.x * 64) {
      Own own = {0, 0, 0};
      if (!own_keys(p.a, t, &own.row, &own.count)) own.row = -1;
      p.own[t] = own;
    }
  }
  } else {
  registers_up();
  if (ok) {
    const int c = warp >> 2, q = warp & 3;
    const int row = q * 32 + lane;  // of the tile
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    const uint32_t t_s = tmem + 128 * c + lanes, t_o = tmem + S::kO + DP * c + lanes, t_p = tmem + S::kP + S::kPStep * c + lanes;
    uint32_t parts = 0, done = 0, joins = 0;  // segments with key tiles, steps, segments joined: of this chain so far
    for (int at = begin; at < end && ok;) {
      const Segment g = segment_at(p, at, begin, end);
      at += g.count;
      const int steps = g.steps(c);
      // rows of the tile that there are
      const long long token0 = (long long)(2 * g.tile + (g.dual ? c : 0)) * p.plan.tile_tokens;
      const int rows = (int)min((long long)p.plan.tile_tokens, p.tokens - token0) * p.group;
      const bool any = q * 32 < rows;  // of this warp's
      float top = kLowest, sum = 0.0f;
      for (int step = 0; step < steps; ++step, ++done) {
        ok = all_wait(bar_s + 8 * c, done & 1u, abort_flag, p.error_word);
        if (!ok) break;
        if (any) {
          tc_fence_after();
          const int valid = p.prefix - g.key_tile(c, step) * kTileKeys;
          // (two copies of the code: selects for every value of every tile would be a third of its instructions)
          const uint32_t p_phase = (done & 1u) ^ 1u;
          if (valid >= kTileKeys)
            ok = softmax_tile<T, DP, false>(t_s, t_p, t_o, p.scale, p.scale2, row < rows, step == 0, valid, top, sum, bar_h + 8 * c, bar_read + 8 * c,
                                            bar_pv + 8 * c, p_phase, abort_flag, p.error_word);
          else
            ok = softmax_tile<T, DP, true>(t_s, t_p, t_o, p.scale, p.scale2, row < rows, step == 0, valid, top, sum, bar_h + 8 * c, bar_read + 8 * c,
                                           bar_pv + 8 * c, p_phase, abort_flag, p.error_word);
          if (!ok) break;
          tc_fence_before();
        } else {
          if (S::kOwnP) {  // (the waits are kept in step: a warp without rows must not run two phases ahead)
            if (lane == 0) mbar_arrive(bar_read + 8 * c);
            ok = all_wait(bar_pv + 8 * c, (done & 1u) ^ 1u, abort_flag, p.error_word);
            if (!ok) break;
          }
          if (lane == 0) mbar_arrive(bar_h + 8 * c);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p + 8 * c);
      }
      if (!ok) break;
      // O and sums of the segment: of two row tiles each chain its own, else both add up to one
      if (steps > 0) {
        ok = all_wait(bar_o + 8 * c, parts & 1u, abort_flag, p.error_word);
        if (!ok) break;
        ++parts;
      }
      constexpr float kLower = 1.0f / (1 << raise_of<T>(8));
      sum *= kLower;
      float weight = kLower, other = 0.0f;  // of this chain's O, of the other one's
      if (!g.dual && g.steps(1) > 0) {
        float2* const exchange = reinterpret_cast<float2*>(smem_raw + (base + S::kExchange - raw));
        if (c == 1) {
          exchange[row] = make_float2(top, sum);
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_x);
          continue;
        }
        ok = all_wait(bar_x, joins & 1u, abort_flag, p.error_word);
        if (!ok) break;
        ++joins;
        const float2 o = exchange[row];
        const float now = fmaxf(top, o.x);
        weight = exp2_approx((top - now) * kLog2e);
        other = exp2_approx((o.x - now) * kLog2e);
        sum = sum * weight + o.y * other;
        weight *= kLower;
        other *= kLower;
        top = now;
      } else if (!g.dual && c == 1) {
        continue;
      }
      if (any) {
        tc_fence_after();
        const bool mine = row < rows;
        const bool direct = p.direct && g.whole;
        const long long part_row = (long long)g.part * kPartRows + (g.dual ? c : 0) * kTileRows + row;
        const long long token = token0 + row / p.group;
        const int head = g.head * p.group + row % p.group;
        if (mine) {
          if (!direct) p.stats[part_row] = make_float2(top, sum);
          else if (p.lse) p.lse[token * p.kv_heads * p.group + head] = top + log2f(sum) * kLn2;
        }
        if (direct) {
          const float inv = 1.0f / sum;
          weight *= inv;
          other *= inv;
        }
        const uint32_t t_o1 = tmem + S::kO + DP + lanes;
        for (int b = 0; b < DP / 32; ++b) {
          uint32_t o[32];
          float v[32];
          tmem_ld32(t_o + 32 * b, o);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(o[j]) * weight;
          if (!g.dual && g.steps(1) > 0) {
            tmem_ld32(t_o1 + 32 * b, o);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = fmaf(__uint_as_float(o[j]), other, v[j]);
          }
          if (!mine) continue;
          if (!direct) {
            float4* out = p.parts + ((long long)g.part * (DP / 4) + 8 * b) * kPartRows + (g.dual ? c : 0) * kTileRows + row;
#pragma unroll
            for (int j = 0; j < 8; ++j) out[j * kPartRows] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          } else {
            T* out = static_cast<T*>(p.out) + token * p.out_row + head * p.out_head + 32 * b;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (32 * b + 8 * j < p.dim)
                *reinterpret_cast<uint4*>(out + 8 * j) = make_uint4(pack2<T>(v[8 * j], v[8 * j + 1]), pack2<T>(v[8 * j + 2], v[8 * j + 3]),
                                                                    pack2<T>(v[8 * j + 4], v[8 * j + 5]), pack2<T>(v[8 * j + 6], v[8 * j + 7]));
          }
        }
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) {  // the first chain has read both
        mbar_arrive(bar_ofree + 8 * c);
        if (!g.dual) mbar_arrive(bar_ofree + 8);
      }
    }
  }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {  // given up
    if (warp == 8 && lane == 0) {
      ring_settle(bar_full, S::kSlots, issued[0]);
      if (issued[1] > 0) mbar_settle(bar_q, (issued[1] - 1) & 1u);
    }
    if (warp == 9) {
      umma_commit_elected(bar_out);
      mbar_settle(bar_out, 0);
    }
    __syncwarp();
  }
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// ---------------------------------------------------------------- join kernel

template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The 8 x 8 matrix of 16-bit values that the warp holds (a row per four lanes), transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// own_keys with a whole warp: of the entries of q_begin 32 are looked at at once.
__device__ __forceinline__ bool own_keys_of_warp(const Params& p, int token, int lane, long long* first, int* count) {
  *first = 0;
  *count = 0;
  int seq = token, behind = 0;  // tokens of the sequence behind this one
  if (p.q_begin) {
    int lo = 0, hi = (int)p.sequences;  // q_begin[lo] <= token < q_begin[hi]
    if (hi == 0 || token < p.q_begin[0] || token >= p.q_begin[hi]) return false;
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) >> 5, at = lo + step * (lane + 1);
      const int below = __popc(__ballot_sync(0xffffffffu, at < hi && p.q_begin[at] <= token));
      lo += step * below;
      hi = min(hi, lo + step);
    }
    seq = lo;
    behind = p.q_begin[seq + 1] - 1 - token;
  }
  if (!p.own_len) return true;
  const long long begin = p.own_begin[seq], len = (long long)p.own_len[seq] - behind;
  if (len <= 0 || begin < 0 || begin >= p.own_rows) return true;
  *first = begin;
  *count = (int)min(len, p.own_rows - begin);
  return true;
}

__device__ __forceinline__ void prefetch_l1(const void* at) { asm volatile("prefetch.global.L1 [%0];" ::"l"(at)); }

struct JoinParams {
  Params a;
  Plan plan;
  int short_prefix;  // keys of a prefix that is taken here, like own keys; else 0
  int tokens;        // of a unit of work
  uint32_t kv_heads_magic, item_magic, per_cta_magic;  // for quotient()
  int per_token_magic;                                 // 64 / columns a token, rounded up: x / columns = x * it >> 6 for x < 8
  const float4* parts;
  const float2* stats;
  const Own* own;
};

// i / d by one multiplication where i * d stays below 2^32 (magic = 2^32 / d rounded up), else (magic 0) by division.
inline uint32_t magic_of(int d, long long most) { return d > 1 && most * d < (1LL << 32) ? (uint32_t)(((1ULL << 32) + d - 1) / d) : 0u; }
__device__ __forceinline__ int quotient(int i, int d, uint32_t magic) {
  return magic ? (int)__umulhi((uint32_t)i, magic) : d == 1 ? i : i / d;
}

// WPU warps work on the eight columns of a product: eight heads of a (token, key head) at a time, or with smaller groups
// the heads of p.tokens adjacent tokens.  S^T = K Q^T: keys are the 16 rows; a lane reads 16-byte pieces of two key
// rows, whose four words take the places of the k indices that the fragment layout gives the lane, in Q alike.
// O^T = V^T P^T: a lane reads values dn * DP/8 .. of four key rows (dn = lane / 4); rows dn and dn + 8 of product t are
// values dn * DP/8 + 2 t and + 2 t + 1, so that it ends with DP/8 adjacent values of columns 2 (lane % 4) and + 1, onto which
// the parts of the prefix are added in place.  Tokens take their own keys one after the other, and only their columns
// take what a product gives: what another token's values hold (infinities, NaN) reaches no other.
// SHORT: the whole prefix is taken here (in a kernel of its own: the registers that this takes cost the other one 3 to 10 us).
template <typename T, int DP, int WPU, bool SHORT>
__global__ void __launch_bounds__(WPU > 1 ? 32 * WPU : 128, WPU > 1 ? 1 : DP == 128 ? 4 : 5) join_kernel(JoinParams p) {
  constexpr int NT = DP / 8;  // values a lane holds of a column
  constexpr float kRaise = raise_of<T>(0);  // (of all sums: it drops out of the quotient)
  extern __shared__ float join_smem[];  // (WPU > 1) per warp: 8 columns of DP, 8 x (maximum, sum)
  constexpr int kWarp = 8 * DP + 16;
  pdl_trigger();
  pdl_wait();
  const Params& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wi = warp % WPU;
  const int quad = lane & 3, dn = lane >> 2;
  // (32-bit arithmetic by multiplication: with 64-bit divisions the indexes took most of the kernel's time, with 32-bit ones a tenth)
  const int unit = WPU > 1 ? (int)blockIdx.x : (int)blockIdx.x * 4 + warp;
  const int slice = quotient(unit, a.kv_heads, p.kv_heads_magic), h = unit - slice * a.kv_heads, token0 = slice * p.tokens;
  if (token0 >= (int)a.tokens) return;
  const int tokens = min(p.tokens, (int)a.tokens - token0);

  // Where the rows lie in the parts of the prefix (a unit's tokens are in one tile).
  int part0 = 0, parts = 0, row0 = 0, item = 0;
  if (p.plan.kv_tiles > 0) {
    const int tile = quotient(token0, 2 * p.plan.tile_tokens, p.item_magic), within = token0 - tile * 2 * p.plan.tile_tokens;
    const int second = within >= p.plan.tile_tokens;
    item = h * p.plan.row_items + tile;
    const int from = item * p.plan.kv_tiles;
    part0 = quotient(from, p.plan.per_cta, p.per_cta_magic);
    parts = quotient(from + p.plan.kv_tiles - 1, p.plan.per_cta, p.per_cta_magic) - part0 + 1;
    row0 = second * kTileRows + (within - second * p.plan.tile_tokens) * a.group;
  }
  const int per_token = p.tokens > 1 ? a.group : 8;  // columns
  int of[2];                                         // the token of this lane's columns
#pragma unroll
  for (int e = 0; e < 2; ++e) of[e] = (2 * quad + e) * p.per_token_magic >> 6;
  const int of_dn = dn * p.per_token_magic >> 6;

  long long own_first = -1;  // of token `lane`
  int own_count = 0;
  if (!SHORT && p.own && lane < tokens) {
    const int4 own = *reinterpret_cast<const int4*>(p.own + token0 + lane);
    own_first = (long long)own.y << 32 | (uint32_t)own.x;
    own_count = own.z;
  }
  for (int g0 = 0; g0 < a.group; g0 += 8) {
    const int columns = p.tokens > 1 ? tokens * a.group : min(8, a.group - g0);
    float o[2][NT];  // [column 2 quad + e][value dn * NT + i]
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
    int seen[2] = {-1, -1};  // own keys of the columns' tokens; -1: of no sequence
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int i = 0; i < NT; ++i) o[e][i] = 0.0f;

    uint4 q[DP / 32];  // of column dn
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) {
      q[b] = make_uint4(0, 0, 0, 0);
      if (dn < columns && 32 * b + 8 * quad < a.dim)
        q[b] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q.data) + (long long)(token0 + of_dn) * a.q.row +
                                               ((long long)h * a.group + g0 + dn - of_dn * per_token) * a.q.head + 32 * b + 8 * quad);
    }
    // The prefix's parts, each lane its own columns' values; a part's maximum and sum are read by eight lanes.  (First, so
    // that their way from memory is under the own keys'.)
    auto fold = [&](int e, float2 st, const float4 (&v)[NT / 4]) {
      const float now = fmaxf(top[e], st.x);
      const float keep = exp2_approx((top[e] - now) * kLog2e), weight = exp2_approx(fmaf(st.x - now, kLog2e, kRaise));
      top[e] = now;
      sum[e] = sum[e] * keep + st.y * weight;
#pragma unroll
      for (int x = 0; x < NT / 4; ++x) {
        o[e][4 * x] = o[e][4 * x] * keep + v[x].x * weight;
        o[e][4 * x + 1] = o[e][4 * x + 1] * keep + v[x].y * weight;
        o[e][4 * x + 2] = o[e][4 * x + 2] * keep + v[x].z * weight;
        o[e][4 * x + 3] = o[e][4 * x + 3] * keep + v[x].w * weight;
      }
    };
    const int row = row0 + g0 + 2 * quad;
    const auto stats_of = [&](int slot, int e) { return p.stats[(long long)slot * kPartRows + row + e]; };
    const auto value_of = [&](int slot, int e, int x) { return p.parts[((long long)slot * (DP / 4) + dn * (NT / 4) + x) * kPartRows + row + e]; };
    if constexpr (WPU == 1) {
      if (parts > 0) {  // (most often the only one: straight to its place, the loads wait for the first use)
        const int slot = p.plan.part_of(item, part0, parts);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (2 * quad + e >= columns) continue;
          const float2 st = stats_of(slot, e);
          constexpr float up = 1 << raise_of<T>(0);
          top[e] = st.x;
          sum[e] = st.y * up;
#pragma unroll
          for (int x = 0; x < NT / 4; ++x) {
            const float4 v = value_of(slot, e, x);
            o[e][4 * x] = v.x * up; o[e][4 * x + 1] = v.y * up; o[e][4 * x + 2] = v.z * up; o[e][4 * x + 3] = v.w * up;
          }
        }
      }
#pragma unroll 1
      for (int i = 1; i < parts; ++i) {
        const int slot = p.plan.part_of(item, part0 + i, parts);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (2 * quad + e >= columns) continue;
          const float2 st = stats_of(slot, e);
          float4 v[NT / 4];
#pragma unroll
          for (int x = 0; x < NT / 4; ++x) v[x] = value_of(slot, e, x);
          fold(e, st, v);
        }
      }
    } else {
      // Few units with many parts wait for memory: two parts' loads go out together (371 rows of 3 heads over 10450
      // keys: 32.4 us, one part at a time 34.2). With one warp to a unit there are other warps to run meanwhile, and
      // the second part's registers cost more than they bring (4096 rows of 16 heads over 2048 keys: 104 us, 94 so).
#pragma unroll 1
      for (int i = wi; i < parts; i += 2 * WPU) {
        float2 st[2][2];
        float4 v[2][2][NT / 4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int slot = p.plan.part_of(item, part0 + min(i + n * WPU, parts - 1), parts);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (2 * quad + e >= columns) continue;
            st[n][e] = stats_of(slot, e);
#pragma unroll
            for (int x = 0; x < NT / 4; ++x) v[n][e][x] = value_of(slot, e, x);
          }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          if (i + n * WPU >= parts) break;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (2 * quad + e < columns) fold(e, st[n][e], v[n][e]);
          }
        }
      }
    }
    if (dn > 0) sum[0] = sum[1] = 0.0f;  // (from here on a column's sum is spread over the eight lanes)

    for (int tt = SHORT ? -1 : 0; tt < tokens; ++tt) {  // -1: a short prefix, which all columns see
      const int token = token0 + tt;
      long long first = 0;
      int count = p.short_prefix;
      const bool own = !SHORT || tt >= 0;
      if (own) {
        if (!SHORT && p.own) {
          first = __shfl_sync(0xffffffffu, own_first, tt);
          count = __shfl_sync(0xffffffffu, own_count, tt);
          if (first < 0) continue;
          // the next token's first keys are on their way meanwhile
          const long long next = __shfl_sync(0xffffffffu, own_first, tt + 1);
          const int there = __shfl_sync(0xffffffffu, own_count, tt + 1);
          if (WPU == 1 && tt + 1 < tokens && (lane & 15) < there) {
            const Rows& rows = lane < 16 ? a.ko : a.vo;
            const T* at = static_cast<const T*>(rows.data) + (next + (lane & 15)) * rows.row + h * rows.head;
            prefetch_l1(at);
            if (DP == 128) prefetch_l1(at + 64);
          }
        } else if (!own_keys_of_warp(a, token, lane, &first, &count)) {
          continue;
        }
      }
      bool active[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        active[e] = (!own || of[e] == tt) && 2 * quad + e < columns;
        if (own && active[e]) seen[e] = count;
      }
      if (count <= 16 * wi) continue;
      const Rows& key_rows = own ? a.ko : a.kp;
      const Rows& value_rows = own ? a.vo : a.vp;
      const T* const keys = static_cast<const T*>(key_rows.data) + first * key_rows.row + h * key_rows.head;
      const T* const values = static_cast<const T*>(value_rows.data) + first * value_rows.row + h * value_rows.head;
      for (int k0 = 16 * wi; k0 < count; k0 += 16 * WPU) {
        uint4 k[2][DP / 32];  // keys dn, dn + 8
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int b = 0; b < DP / 32; ++b) {
            k[r][b] = make_uint4(0, 0, 0, 0);
            if (k0 + dn + 8 * r < count && 32 * b + 8 * quad < a.dim)
              k[r][b] = *reinterpret_cast<const uint4*>(keys + (k0 + dn + 8 * r) * key_rows.row + 32 * b + 8 * quad);
          }
        uint4 v[4][NT / 8];  // keys 2 quad, 2 quad + 1, + 8, + 9 (on their way during the softmax)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = k0 + 2 * quad + (i & 1) + 8 * (i >> 1);
#pragma unroll
          for (int x = 0; x < NT / 8; ++x) {
            v[i][x] = make_uint4(0, 0, 0, 0);
            if (key < count && dn * NT + 8 * x < a.dim)
              v[i][x] = *reinterpret_cast<const uint4*>(values + key * value_rows.row + dn * NT + 8 * x);
          }
        }
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // keys dn, dn, dn + 8, dn + 8; columns 2 quad, + 1
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) {
          const uint32_t a0[4] = {k[0][b].x, k[1][b].x, k[0][b].y, k[1][b].y}, a1[4] = {k[0][b].z, k[1][b].z, k[0][b].w, k[1][b].w};
          mma_16816<T>(s, a0, q[b].x, q[b].y);
          mma_16816<T>(s, a1, q[b].z, q[b].w);
        }
        float pr[4], keep[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const bool in0 = active[e] && k0 + dn < count, in1 = active[e] && k0 + dn + 8 < count;
          const float s0 = in0 ? __fmul_rn(s[e], a.scale) : -INFINITY, s1 = in1 ? __fmul_rn(s[2 + e], a.scale) : -INFINITY;
          float now = max3(fmaxf(top[e], kLowest), s0, s1);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, d));
          keep[e] = exp2_approx((top[e] - now) * kLog2e);
          pr[e] = in0 ? exp2_approx(fmaf(__fsub_rn(s0, now), kLog2e, kRaise)) : 0.0f;
          pr[2 + e] = in1 ? exp2_approx(fmaf(__fsub_rn(s1, now), kLog2e, kRaise)) : 0.0f;
          if (active[e]) {
            top[e] = now;
            sum[e] = sum[e] * keep[e] + pr[e] + pr[2 + e];
          }
        }
        const uint32_t p0 = transposed(pack2<T>(pr[0], pr[1])), p1 = transposed(pack2<T>(pr[2], pr[3]));
#pragma unroll
        for (int t = 0; t < NT / 2; ++t) {
          auto word = [&](int i) { return (t & 3) == 0 ? v[i][t / 4].x : (t & 3) == 1 ? v[i][t / 4].y : (t & 3) == 2 ? v[i][t / 4].z : v[i][t / 4].w; };
          const uint32_t av[4] = {__byte_perm(word(0), word(1), 0x5410), __byte_perm(word(0), word(1), 0x7632),
                                  __byte_perm(word(2), word(3), 0x5410), __byte_perm(word(2), word(3), 0x7632)};
          float d[4] = {o[0][2 * t] * keep[0], o[1][2 * t] * keep[1], o[0][2 * t + 1] * keep[0], o[1][2 * t + 1] * keep[1]};
          mma_16816<T>(d, av, p0, p1);
          if (active[0]) { o[0][2 * t] = d[0]; o[0][2 * t + 1] = d[2]; }
          if (active[1]) { o[1][2 * t] = d[1]; o[1][2 * t + 1] = d[3]; }
        }
      }
    }
    // (a column's sum is spread over the lanes of its keys; so far every one of them added to the same maximum)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], d);

    if (WPU > 1) {  // the warps' states, joined by the first one
      float* const mine = join_smem + warp * kWarp;
      if (wi > 0) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int i = 0; i < NT; i += 4)
            *reinterpret_cast<float4*>(mine + (2 * quad + e) * DP + dn * NT + i) = make_float4(o[e][i], o[e][i + 1], o[e][i + 2], o[e][i + 3]);
          if (dn == 0) {
            mine[8 * DP + 2 * (2 * quad + e)] = top[e];
            mine[8 * DP + 2 * (2 * quad + e) + 1] = sum[e];
          }
        }
      }
      __syncthreads();
      if (wi == 0) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float* const from = join_smem + warp * kWarp + (2 * quad + e) * DP + dn * NT;
          const float2* const stats = reinterpret_cast<const float2*>(join_smem + warp * kWarp + 8 * DP) + 2 * quad + e;
          float2 st[WPU];
          float now = fmaxf(top[e], kLowest);
#pragma unroll
          for (int w = 1; w < WPU; ++w) {
            st[w] = stats[w * (kWarp / 2)];
            now = fmaxf(now, st[w].x);
          }
          const float keep = exp2_approx((top[e] - now) * kLog2e);
          top[e] = now;
          sum[e] *= keep;
#pragma unroll
          for (int i = 0; i < NT; ++i) o[e][i] *= keep;
#pragma unroll
          for (int w = 1; w < WPU; ++w) {
            if (st[w].x == -INFINITY) continue;  // nothing was left for that warp
            const float weight = exp2_approx((st[w].x - now) * kLog2e);
            sum[e] += st[w].y * weight;
#pragma unroll
            for (int i = 0; i < NT; ++i) o[e][i] += from[w * kWarp + i] * weight;
          }
        }
      }
    }
    if (wi == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (seen[e] < 0) continue;
        const bool none = seen[e] == 0 && a.prefix == 0;  // no key at all (keys whose scores are all -inf give 0 / 0)
        const float inv = none ? 0.0f : 1.0f / sum[e];
        const long long token = token0 + of[e], head = (long long)h * a.group + g0 + 2 * quad + e - of[e] * per_token;
        T* const out = static_cast<T*>(a.out) + token * a.out_row + head * a.out_head + dn * NT;
#pragma unroll
        for (int x = 0; x < NT / 8; ++x)
          if (dn * NT + 8 * x < a.dim)
            *reinterpret_cast<uint4*>(out + 8 * x) =
                make_uint4(pack2<T>(o[e][8 * x] * inv, o[e][8 * x + 1] * inv), pack2<T>(o[e][8 * x + 2] * inv, o[e][8 * x + 3] * inv),
                           pack2<T>(o[e][8 * x + 4] * inv, o[e][8 * x + 5] * inv), pack2<T>(o[e][8 * x + 6] * inv, o[e][8 * x + 7] * inv));
        if (a.lse && dn == 0) a.lse[token * a.heads + head] = none ? -INFINITY : top[e] + (log2f(sum[e]) - kRaise) * kLn2;
      }
    }
    if (WPU > 1) __syncthreads();
  }
}

// ---------------------------------------------------------------- cut items without own keys

// Without own keys, and every token a sequence, only items that a share's end cuts are left to add up, at most one per
// CTA.  Block (b, y): rows 32 y .. of the item that the share of CTA b ends in.  Parts are read with rows across the lanes,
// as they lie, and turned in shared memory.
template <typename T, int DP>
__global__ void __launch_bounds__(256) cut_items_kernel(JoinParams p) {
  __shared__ float turned[32][DP + 1];
  pdl_trigger();
  pdl_wait();
  const Params& a = p.a;
  const int end = ((int)blockIdx.x + 1) * p.plan.per_cta;  // of the share
  const int item = end / p.plan.kv_tiles, from = item * p.plan.kv_tiles;
  if (item >= p.plan.items || end == from || (int)blockIdx.x != from / p.plan.per_cta) return;  // not cut here, or cut before already
  const int parts = (from + p.plan.kv_tiles - 1) / p.plan.per_cta - (int)blockIdx.x + 1;
  const int h = item / p.plan.row_items, tile = item - h * p.plan.row_items;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = 32 * (int)blockIdx.y + lane, second = row >= kTileRows;
  const int in_tile = row - second * kTileRows, tokens = p.plan.tile_tokens;
  const long long token0 = ((long long)2 * tile + second) * tokens;
  const bool there = in_tile < tokens * a.group && token0 + in_tile / a.group < a.tokens;
  float top = kLowest, sum = 0.0f;
  if (there) {
    for (int i = 0; i < parts; ++i) top = fmaxf(top, p.stats[(long long)p.plan.part_of(item, (int)blockIdx.x + i, parts) * kPartRows + row].x);
    // warp w: pieces w, w + 8, ..
    float4 acc[DP / 32];
#pragma unroll
    for (int x = 0; x < DP / 32; ++x) acc[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i = 0; i < parts; ++i) {
      const int slot = p.plan.part_of(item, (int)blockIdx.x + i, parts);
      const float2 st = p.stats[(long long)slot * kPartRows + row];
      const float weight = exp2_approx((st.x - top) * kLog2e);
      sum += st.y * weight;
#pragma unroll
      for (int x = 0; x < DP / 32; ++x) {
        const float4 v = p.parts[((long long)slot * (DP / 4) + warp + 8 * x) * kPartRows + row];
        acc[x].x += v.x * weight; acc[x].y += v.y * weight; acc[x].z += v.z * weight; acc[x].w += v.w * weight;
      }
    }
    const float inv = 1.0f / sum;
#pragma unroll
    for (int x = 0; x < DP / 32; ++x) {
      float* const to = &turned[lane][4 * (warp + 8 * x)];
      to[0] = acc[x].x * inv; to[1] = acc[x].y * inv; to[2] = acc[x].z * inv; to[3] = acc[x].w * inv;
    }
    if (warp == 0 && a.lse) a.lse[(token0 + in_tile / a.group) * a.heads + (long long)h * a.group + in_tile % a.group] = top + log2f(sum) * kLn2;
  }
  __syncthreads();
  constexpr int PER = DP / 8;  // lanes a row: eight values each
  for (int r = threadIdx.x / PER; r < 32; r += 256 / PER) {
    const int at = 32 * (int)blockIdx.y + r - second * kTileRows, d = threadIdx.x % PER * 8;
    const long long token = token0 + at / a.group;
    if (at >= tokens * a.group || token >= a.tokens || d >= a.dim) continue;
    const float* v = &turned[r][d];
    *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + token * a.out_row + ((long long)h * a.group + at % a.group) * a.out_head + d) =
        make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
  }
}

// ---------------------------------------------------------------- host

int heads_map(CUtensorMap* map, bool bf16, const void* ptr, int rank, const long long* dims, const long long* strides_elements,
              const int* box) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(ANNC_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  cuuint64_t d[4], st[3];
  cuuint32_t b[4], one[4] = {1, 1, 1, 1};
  for (int i = 0; i < rank; ++i) {
    d[i] = (cuuint64_t)dims[i];
    b[i] = (cuuint32_t)box[i];
    // (the stride of a dimension of one does not matter, but has to be a multiple of 16 bytes)
    if (i > 0) st[i - 1] = dims[i] == 1 ? 16 : (cuuint64_t)strides_elements[i - 1] * 2;
  }
  const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (cuuint32_t)rank,
                        const_cast<void*>(ptr), d, st, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(ANNC_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return ANNC_OK;
}

// 16-byte pieces of every row; TMA wants positive strides below 2^40 bytes.
bool rows_ok(const Rows& r, long long rows, long long heads, bool tma) {
  if (reinterpret_cast<uintptr_t>(r.data) & 15) return false;
  auto stride_ok = [&](long long s, long long n) {
    return n <= 1 || (s % 8 == 0 && (!tma || (s > 0 && s < (1LL << 39))));
  };
  return stride_ok(r.row, rows) && stride_ok(r.head, heads);
}

template <typename T, int DP>
int launch_prefix(const Params& a, const PrefixParams& p, cudaStream_t s) {
  void (*const kernel)(CUtensorMap, CUtensorMap, CUtensorMap, PrefixParams) = prefix_kernel<T, DP>;
  static bool attr_done[kMaxDevices] = {};
  const int dev = device_slot();
  if (!attr_done[dev]) {
    ANNC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<DP>::kSmem));
    attr_done[dev] = true;
  }
  const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  CUtensorMap tq, tk, tv;
  {
    const long long dims[4] = {a.dim, a.group, a.kv_heads, a.tokens}, strides[3] = {a.q.head, a.q.head * a.group, a.q.row};
    const int box[4] = {64, a.group, 1, p.plan.tile_tokens};
    ANNC_TRY(heads_map(&tq, bf16, a.q.data, 4, dims, strides, box));
  }
  for (int v = 0; v < 2; ++v) {
    const Rows& r = v ? a.vp : a.kp;
    const long long dims[3] = {a.dim, a.kv_heads, a.prefix}, strides[2] = {r.head, r.row};
    const int box[3] = {64, 1, kTileKeys};
    ANNC_TRY(heads_map(v ? &tv : &tk, bf16, r.data, 3, dims, strides, box));
  }
  ANNC_CUDA(launch_pdl(kernel, dim3((unsigned)p.plan.ctas), dim3(kThreads), Shape<DP>::kSmem, s, tq, tk, tv, p));
  return ANNC_OK;
}

template <typename T, int DP, int WPU>
int launch_join(JoinParams p, cudaStream_t s) {
  p.kv_heads_magic = magic_of(p.a.kv_heads, p.a.tokens * p.a.kv_heads);
  p.item_magic = magic_of(2 * p.plan.tile_tokens, p.a.tokens);
  p.per_cta_magic = magic_of(p.plan.per_cta, (long long)p.plan.items * p.plan.kv_tiles);
  const int per_token = p.tokens > 1 ? p.a.group : 8;
  p.per_token_magic = (64 + per_token - 1) / per_token;
  void (*const kernel)(JoinParams) = p.short_prefix ? join_kernel<T, DP, WPU, true> : join_kernel<T, DP, WPU, false>;
  const long long units = (p.a.tokens + p.tokens - 1) / p.tokens * p.a.kv_heads, blocks = WPU > 1 ? units : (units + 3) / 4;  // (tc_supported: they fit 30 bits)
  const size_t smem = WPU > 1 ? WPU * (8 * DP + 16) * sizeof(float) : 0;
  ANNC_CUDA(launch_pdl(kernel, dim3((unsigned)blocks), dim3(WPU > 1 ? 32 * WPU : 128), smem, s, p));
  return ANNC_OK;
}

template <typename T, int DP>
int run_as(const Params& a, void* workspace, cudaStream_t s) {
  PrefixParams p = {};
  const bool short_prefix = is_short(a.prefix, a.tokens * a.kv_heads);
  p.plan = plan_of(a.tokens, a.kv_heads, a.group, short_prefix ? 0 : a.prefix);
  p.tokens = a.tokens;
  p.kv_heads = a.kv_heads;
  p.group = a.group;
  p.prefix = (int)a.prefix;
  p.dim = a.dim;
  p.scale = a.scale;
  p.scale2 = a.scale * kLog2e;
  const size_t slots = 2 * kMaxCtas + (size_t)p.plan.items;
  p.a = a;
  p.parts = static_cast<float4*>(workspace);
  p.stats = reinterpret_cast<float2*>(p.parts + slots * kPartRows * (DP / 4));
  p.own = !short_prefix && (a.own_len || a.q_begin) ? reinterpret_cast<Own*>(p.stats + slots * kPartRows) : nullptr;
  p.error_word = gemm::gemm_error_word();
  if (!p.error_word) return fail(ANNC_ERR_CUDA, "the tensor-core error word is not addressable");
  p.direct = !a.own_len && !a.q_begin;
  p.out = a.out;
  p.out_row = a.out_row;
  p.out_head = a.out_head;
  p.lse = a.lse;
  if (!short_prefix) ANNC_TRY((launch_prefix<T, DP>(a, p, s)));
  JoinParams j = {};
  j.a = a;
  j.plan = p.plan;
  j.short_prefix = short_prefix ? (int)a.prefix : 0;
  j.tokens = 1;
  j.parts = p.parts;
  j.stats = p.stats;
  j.own = p.own;
  if (p.direct && !short_prefix) {
    if (p.plan.ctas > 1 && p.plan.per_cta % p.plan.kv_tiles != 0)
      ANNC_CUDA(launch_pdl(cut_items_kernel<T, DP>, dim3((unsigned)p.plan.ctas - 1, kPartRows / 32), dim3(256), 0, s, j));
    return ANNC_OK;
  }
  // A unit of work fills a warp.  Small groups: several tokens' heads, if that leaves eight warps for every SM.  Few units with
  // something to do for more than one warp (chunks of own keys, going by the size of their buffer, and parts): four
  // or eight warps for each.  The lengths themselves are on the device: a buffer of wide slots with few keys in each gets
  // more warps than they need (four keys a token, packed / in slots of 512: 500 tokens of two key heads over 40 keys 6.9 / 12.9 us, 100
  // tokens of eight over 300 17.0 / 22.5; with 64 tokens over 16 or 4096 keys the same).
  const long long units = a.tokens * a.kv_heads;
  const long long own = a.own_len && a.sequences > 0 ? a.own_rows / a.sequences : 0;
  const long long chunks = (own + j.short_prefix + 15) / 16 + (short_prefix ? 0 : p.plan.kv_tiles / p.plan.per_cta + 1);
  if (units <= 148 && chunks > 4) return launch_join<T, DP, 8>(j, s);
  if (units < 1184 && chunks > 4) return launch_join<T, DP, 4>(j, s);
  while (2 * j.tokens * a.group <= 8 && units / (2 * j.tokens) >= 148 * 8) j.tokens *= 2;
  return launch_join<T, DP, 1>(j, s);
}

}  // namespace

size_t tc_workspace_bytes(long long tokens, int heads, int kv_heads, int dim) {
  const int group = heads / kv_heads;
  if (group > kTileRows || dim > 128) return 0;
  const long long per_item = 2LL * (kTileRows / group);
  const unsigned long long slots = 2ULL * kMaxCtas + (unsigned long long)((tokens + per_item - 1) / per_item) * kv_heads;
  return (size_t)(slots * kPartRows * ((unsigned long long)part_width(dim) * 4 + 8) + (unsigned long long)tokens * sizeof(Own));
}

bool tc_supported(const Params& p, int) {
  if (p.dim % 8 || p.dim > 128 || p.group > kTileRows) return false;
  // the prefix kernel takes the maximum of the unscaled scores, multiplies by scale * log2 e, and far out by 1 / scale
  if (p.prefix > 0 && p.scale != 0.0f && !(p.scale >= 1e-30f && std::isfinite(p.scale * kLog2e))) return false;
  const Plan plan = plan_of(p.tokens, p.kv_heads, p.group, p.prefix);
  if ((long long)plan.row_items * p.kv_heads * (plan.kv_tiles > 0 ? plan.kv_tiles : 1) >= (1LL << 30) || p.tokens * p.kv_heads >= (1LL << 30)) return false;
  if (!rows_ok(p.q, p.tokens, p.heads, true) || p.q.head * p.group >= (1LL << 39)) return false;
  if (p.prefix > 0 && (!rows_ok(p.kp, p.prefix, p.kv_heads, true) || !rows_ok(p.vp, p.prefix, p.kv_heads, true))) return false;
  if (p.own_len && (!rows_ok(p.ko, p.own_rows, p.kv_heads, false) || !rows_ok(p.vo, p.own_rows, p.kv_heads, false))) return false;
  return (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 && (p.tokens == 1 || p.out_row % 8 == 0) && (p.heads == 1 || p.out_head % 8 == 0);
}

int run_tc(const Params& p, int dtype, void* workspace, cudaStream_t s) {
  if (dtype == ANNC_BF16)
    return p.dim <= 64 ? run_as<__nv_bfloat16, 64>(p, workspace, s) : run_as<__nv_bfloat16, 128>(p, workspace, s);
  return p.dim <= 64 ? run_as<__half, 64>(p, workspace, s) : run_as<__half, 128>(p, workspace, s);
}

}  // namespace attention
}  // namespace annc
