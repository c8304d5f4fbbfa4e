// 8-bit integer products on the 5th-generation tensor cores (tcgen05, kind::i8, 32-bit integer sums).
//
//   C[m,n] = act(sum_k A[m,k] B[n,k] * scale_a[m] * scale_b[n] + bias[n])
//
// Operands come by TMA in k-steps of 128 bytes (128-byte swizzle, out-of-range bytes read as zero).
//
//   split kernel  one CTA takes 128 channels x 16 to 256 tokens.  The channels (rows of B) lie on the 128 accumulator
//                 rows, so that a tile of few tokens wastes none, and since tensor memory is read with a lane per
//                 accumulator row, a warp's 32 values of one token are adjacent in C and are stored as they come.
//                 The CTAs of a cluster share a tile and split its k-steps, leave their integer sums in shared
//                 memory and add them over distributed shared memory (integers: any order gives the same).  For
//                 products whose tiles do not fill the chip, down to one token, where the weight's bytes are all
//                 there is to do.
//   pair kernel   persistent, a cluster of two CTAs takes 256 tokens x 256 channels (cta_group::2, each loads its own
//                 half of both operands), accumulators double-buffered in tensor memory, so that a tile is written
//                 under the next one's products.  Here tokens lie on the rows: a lane then holds adjacent channels, which
//                 leave through shared memory in whole lines by TMA.  (With a store of 32 channels per token and
//                 warp, as in the split kernel, the epilogue took 3.7 us a tile and bounded every product with k
//                 below 1024: 16384 x 8192 x 256 103 us.)
//
// Every wait is bounded; a role that gives up raises the error word that annc_gemm_check reads.
#include <cuda.h>

#include <cstdint>
#include <cstring>

#include "common.h"
#include "gemm_i8.h"
#include "pdl.cuh"
#include "tc_host.h"
#include "tc_ptx.cuh"

namespace annc {
namespace gemm {
int* gemm_error_word();  // device address of the tcgen05 GEMM error word (gemm_tc.cu)
}
namespace gemm_i8 {

namespace {

using namespace annc::tc;

constexpr int KB = 128;  // bytes (values) of k per stage

// Products and their commits are issued by a whole warp, of which one lane is elected in the instruction itself: its
// operands then stay in uniform registers.  (From a branch that one lane takes, a product costs some 140 cycles to issue.)
__device__ __forceinline__ void commit_elected(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
      : "memory");
}
__device__ __forceinline__ void commit_pair_elected(uint32_t bar) {
  const uint16_t mask = 3;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar),
      "h"(mask)
      : "memory");
}
__device__ __forceinline__ bool all_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* error_word) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, error_word)) != 0;
}
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_pair_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// 16 lanes x 32 columns; a thread gets, of each eight columns c = 8 g .., columns 2 (lane % 4) and the next of rows lane / 4
// (r[4 g], r[4 g + 1]) and lane / 4 + 8 (r[4 g + 2], r[4 g + 3]).
__device__ __forceinline__ void tmem_ld_16x256(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// D s32; A and B signed 8-bit, both K-major.
__host__ __device__ constexpr uint32_t i8_idesc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

template <int BYTES>
struct Vector4;  // four values of so many bytes
template <>
struct Vector4<4> { using type = uint4; };
template <>
struct Vector4<2> { using type = uint2; };

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const T v[2] = {to_type<T>(lo), to_type<T>(hi)};
  uint32_t w = 0;
  memcpy(&w, v, sizeof(v) < 4 ? sizeof(v) : 4);
  return w;
}

// N accumulator columns (tokens) of this lane's channel: finished, and stored N times one value of 32 adjacent
// channels per warp.  `out` is the place of the first token, `count` how many tokens there are.
template <typename T, int N>
__device__ __forceinline__ void finish_columns(const Params& p, const uint32_t (&r)[N], const float* scale_a, float scale_b,
                                               float bias, T* out, int count, bool in) {
  float v[N];
#pragma unroll
  for (int j = 0; j < N; j += 4) {
    const float4 sa = *reinterpret_cast<const float4*>(scale_a + j);
    v[j] = scaled((int)r[j], sa.x, scale_b, bias);
    v[j + 1] = scaled((int)r[j + 1], sa.y, scale_b, bias);
    v[j + 2] = scaled((int)r[j + 2], sa.z, scale_b, bias);
    v[j + 3] = scaled((int)r[j + 3], sa.w, scale_b, bias);
  }
  activate(p.act, v);
  if (!in) return;
  if (count >= N) {
#pragma unroll
    for (int j = 0; j < N; ++j) out[j * p.ldc] = to_type<T>(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < count) out[j * p.ldc] = to_type<T>(v[j]);
  }
}

// ---------------------------------------------------------------- split kernel

constexpr int kSplitThreads = 320;  // producer, MMA issuer, eight epilogue warps
constexpr int kChannels = 128;

// Rows of an operand's box: no more than there are.  (Rows that TMA has to fill with zeros cost far more than rows that it
// loads, 4730 x 24 x 2583 15.0 us with boxes of 128 rows, 6.6 so.  What lies in the stage behind the box gives sums of
// channels or tokens that are not there.)
__host__ __device__ __forceinline__ int box_rows(int rows, int tile) { return rows < tile ? rows : tile; }

template <int TN>
struct SplitShape {
  static constexpr int kStage = (kChannels + TN) * KB;
  static constexpr int kStages = TN <= 64 ? 8 : TN <= 128 ? 6 : 4;
  static constexpr int kCols = TN < 32 ? 32 : TN;
  // The sums of a tile lie where the stages were: kChannels * TN words fit there for every TN.
  static_assert(kStages * kStage >= kChannels * TN * 4, "");
  static constexpr int kScales = TN * 4;  // of the tile's tokens
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage + kScales + 256;
};

template <int TN, typename T>
__global__ void __launch_bounds__(kSplitThreads, 1)
gemm_i8_split_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_t, Params p, int split,
                     int* error_word) {
  using S = SplitShape<TN>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gen_base = smem_raw + (base - raw);
  float* const scales = reinterpret_cast<float*>(gen_base + S::kStages * S::kStage);
  constexpr int kBars = S::kStages * S::kStage + S::kScales;
  const uint32_t bars = base + kBars;
  const uint32_t bar_full = bars, bar_empty = bars + 8 * S::kStages, bar_done = bars + 16 * S::kStages, bar_out = bar_done + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gen_base + kBars + 16 * S::kStages + 16);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // (known to be uniform)
  const int channel_tiles = (p.n + kChannels - 1) / kChannels, tile = blockIdx.x / split;
  const int n0 = tile % channel_tiles * kChannels, m0 = tile / channel_tiles * TN;
  const int rank = split > 1 ? (int)cluster_ctarank() : 0;
  const int KT_all = (p.k + KB - 1) / KB;
  const int kt0 = (int)((long long)KT_all * rank / split), KT = (int)((long long)KT_all * (rank + 1) / split) - kt0;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&tmap_w);
    prefetch_tensormap(&tmap_t);
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    mbar_init(bar_done, 1);
    mbar_init(bar_out, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    // The weight's bytes are on their way to L2 while the kernel before this one (which quantises the tokens)
    // drains; L2 is where all its writes would be seen, so that nothing stale is read later.
    for (int kt = 0; kt < KT && kt < S::kStages; ++kt) tma_prefetch_2d(&tmap_w, (kt0 + kt) * KB, n0);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"((uint32_t)S::kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();
  pdl_wait();
  const bool poisoned = *reinterpret_cast<volatile int*>(error_word) != 0;  // an earlier launch gave up
  bool ok = !poisoned;
  uint32_t issued = 0;  // k-steps, by the producer

  if (ok && warp == 0) {
    if (lane == 0) {
      for (int kt = 0; kt < KT && ok; ++kt, ++issued) {
        const int s = kt % S::kStages;
        ok = mbar_wait(bar_empty + 8 * s, ((kt / S::kStages) & 1u) ^ 1u, abort_flag, error_word);
        if (!ok) break;
        const uint32_t sw = base + s * S::kStage;
        mbar_expect_tx(bar_full + 8 * s, (box_rows(p.n, kChannels) + box_rows(p.m, TN)) * KB);
        tma_load_2d(sw, &tmap_w, (kt0 + kt) * KB, n0, bar_full + 8 * s);
        tma_load_2d(sw + kChannels * KB, &tmap_t, (kt0 + kt) * KB, m0, bar_full + 8 * s);
      }
    }
  } else if (ok && warp == 1) {
    // (an address further on is a descriptor further on: the address field counts 16 bytes and cannot overflow)
    const uint64_t w_desc = smem_desc(base, 16, 1024, 2), t_desc = smem_desc(base + kChannels * KB, 16, 1024, 2);
    for (int kt = 0; kt < KT; ++kt) {
      const int s = kt % S::kStages;
      ok = all_wait(bar_full + 8 * s, (kt / S::kStages) & 1u, abort_flag, error_word);
      if (!ok) break;
      tc_fence_after();
      const uint32_t off = s * (S::kStage >> 4);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        umma_i8(tmem_base, w_desc + off + 2 * kk, t_desc + off + 2 * kk, i8_idesc(kChannels, TN), (kt | kk) != 0 ? 1u : 0u);
      commit_elected(bar_empty + 8 * s);
    }
    if (ok) commit_elected(bar_done);
  }

  __syncwarp();
  const int tokens = min(TN, p.m - m0);
  if (warp >= 2 && ok) {  // while the MMAs run
    for (int j = threadIdx.x - 64; j < TN; j += kSplitThreads - 64) scales[j] = j < tokens ? p.scale_a[m0 + j] : 0.0f;
  }
  // warp (q, half): channels 32 q .., every other piece of 16 tokens
  const int q = warp & 3, half = (warp - 2) >> 2;
  bool done = false;
  if (warp >= 2 && ok) {
    done = __all_sync(0xffffffffu, mbar_wait(bar_done, 0, abort_flag, error_word)) != 0;
    tc_fence_after();
  }
  const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16);
  T* const c = static_cast<T*>(p.c);
  if (split == 1) {
    if (warp >= 2) asm volatile("bar.sync 1, 256;" ::: "memory");  // the scales are there
    if (done) {
      const int n = n0 + q * 32 + lane;
      const bool in = n < p.n;
      const float sb = in ? p.scale_b[n] : 0.0f, bias = in && p.bias ? p.bias[n] : 0.0f;
#pragma unroll 1
      for (int c0 = 16 * half; c0 < tokens; c0 += 32) {
        uint32_t r[16];
        tmem_ld16(taddr + c0, r);
        tmem_ld_wait();
        finish_columns<T, 16>(p, r, scales + c0, sb, bias, c + (m0 + c0) * p.ldc + n, tokens - c0, in);
      }
    }
  } else {
    // Sums [token][channel] in shared memory, where the stages were: every MMA that read them is done.
    int* part = reinterpret_cast<int*>(gen_base);
    if (done) {
#pragma unroll 1
      for (int c0 = 16 * half; c0 < tokens; c0 += 32) {
        uint32_t r[16];
        tmem_ld16(taddr + c0, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c0 + j) * kChannels + q * 32 + lane] = (int)r[j];
      }
    }
    cluster_sync_all();
    if (ok) {
      // A piece of work is four adjacent channels of a token; the ranks take tokens in turn.
      constexpr int per_token = kChannels / 4;
      const int pieces = (tokens - rank + split - 1) / split * per_token;
      for (int i = threadIdx.x; i < pieces; i += kSplitThreads) {
        const int t = rank + i / per_token * split, n = n0 + i % per_token * 4;
        if (n >= p.n) continue;
        const uint32_t at = base + (uint32_t)(t * kChannels + i % per_token * 4) * 4u;
        int sum[8][4];
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r < split)
            asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(sum[r][0]), "=r"(sum[r][1]), "=r"(sum[r][2]), "=r"(sum[r][3])
                         : "r"(mapa_u32(at, (uint32_t)r)));
        const float sa = p.scale_a[m0 + t];
        const int more = min(4, p.n - n);
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
          for (int r = 1; r < 8; ++r)
            if (r < split) sum[0][e] += sum[r][e];
          v[e] = e < more ? scaled(sum[0][e], sa, p.scale_b[n + e], p.bias ? p.bias[n + e] : 0.0f) : 0.0f;
        }
        activate(p.act, v);
        T* const out = c + (m0 + t) * p.ldc + n;
        T o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = to_type<T>(v[e]);
        if (more == 4 && (reinterpret_cast<uintptr_t>(out) & (4 * sizeof(T) - 1)) == 0) {
          using V = typename Vector4<sizeof(T)>::type;
          V w;
          memcpy(&w, o, sizeof(w));
          *reinterpret_cast<V*>(out) = w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e < more) out[e] = o[e];
        }
      }
    }
    cluster_sync_all();  // a peer may still read this CTA's sums
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {  // given up
    if (warp == 0 && lane == 0) ring_settle(bar_full, S::kStages, issued);
    if (warp == 1) {
      commit_elected(bar_out);
      mbar_settle(bar_out, 0);
    }
    __syncwarp();
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)S::kCols) : "memory");
  }
}

// ---------------------------------------------------------------- pair kernel

constexpr int kPairStage = 32768;  // 128 tokens and 128 channels x 128 bytes per CTA
constexpr int kPairStages = 6;
constexpr int kPairThreads = 320;  // producer, MMA issuer, eight epilogue warps
constexpr int kPairTile = 256;     // tokens and channels
constexpr int kPairStaging = 8 * 4096;  // per epilogue warp 32 tokens x 128 bytes of C, swizzled
constexpr size_t kPairSmem = 1024 + (size_t)kPairStages * kPairStage + kPairStaging + 256;
constexpr int kBand = 8;

struct PairTiles {
  int channels, tokens;  // tiles along each
  int count;
};
// Bands of eight token tiles, inside a band the channel tile advances slowest: the tiles in flight share the
// panels of both operands through L2.
__device__ __forceinline__ void tile_coords(const PairTiles& t, int tile, int* token0, int* channel0) {
  const int band = tile / (kBand * t.channels), rem = tile - band * (kBand * t.channels);
  const int rows = min(kBand, t.tokens - band * kBand);
  const int c = rem / rows;
  *channel0 = c * kPairTile;
  *token0 = (band * kBand + rem - c * rows) * kPairTile;
}

// TMA_STORE: C goes out by TMA from the staging tiles (rows of whole 16-byte pieces at 16-byte addresses); else a
// warp writes its staging tile row by row, one or two values a lane.
template <typename T, bool TMA_STORE>
__global__ void __launch_bounds__(kPairThreads, 1)
gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                    const __grid_constant__ CUtensorMap tmap_c, Params p, PairTiles tiles, int* error_word) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gen_base = smem_raw + (base - raw);
  constexpr int kBars = kPairStages * kPairStage + kPairStaging;
  const uint32_t bars = base + kBars;
  const uint32_t bar_full = bars, bar_empty = bars + 8 * kPairStages;
  const uint32_t bar_tfull = bars + 16 * kPairStages, bar_tempty = bar_tfull + 16, bar_out = bar_tempty + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gen_base + kBars + 16 * kPairStages + 40);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // (known to be uniform)
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int KT = (p.k + KB - 1) / KB;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&tmap_a);
    prefetch_tensormap(&tmap_b);
    if (TMA_STORE) prefetch_tensormap(&tmap_c);
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);   // the leader's expect_tx arrival; bytes come from both CTAs
      mbar_init(bar_empty + 8 * s, 1);  // one commit
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(bar_tfull + 8 * a, 1);
      mbar_init(bar_tempty + 8 * a, 16);  // the epilogue warps of both CTAs
    }
    mbar_init(bar_out, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc_pair(smem_u32(tmem_slot), 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before anything signals across the pair
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();
  pdl_wait();
  const bool poisoned = *reinterpret_cast<volatile int*>(error_word) != 0;  // an earlier launch gave up

  uint32_t kit = 0;  // k-steps: issued by the producer, multiplied by the issuer of the products
  if (!poisoned) {
    if (warp == 0) {
      if (lane == 0) {
        bool ok = true;
        for (int tile = pair; tile < tiles.count && ok; tile += pairs) {
          int m0, n0;
          tile_coords(tiles, tile, &m0, &n0);
          m0 += (int)rank * (kPairTile / 2);
          n0 += (int)rank * (kPairTile / 2);
          for (int kt = 0; kt < KT; ++kt, ++kit) {
            const int s = kit % kPairStages;
            ok = mbar_wait(bar_empty + 8 * s, ((kit / kPairStages) & 1u) ^ 1u, abort_flag, error_word);
            if (!ok) break;
            const uint32_t sa = base + s * kPairStage;
            const uint32_t full_leader = mapa_u32(bar_full + 8 * s, 0);
            if (leader) mbar_expect_tx(bar_full + 8 * s, 2 * kPairStage);
            tma_load_2d_pair(sa, &tmap_a, kt * KB, m0, full_leader);
            tma_load_2d_pair(sa + kPairStage / 2, &tmap_b, kt * KB, n0, full_leader);
          }
        }
      }
    } else if (warp == 1) {
      if (leader) {
        const uint64_t a_desc = smem_desc(base, 16, 1024, 2), b_desc = smem_desc(base + kPairStage / 2, 16, 1024, 2);
        uint32_t count = 0;
        bool ok = true;
        for (int tile = pair; tile < tiles.count && ok; tile += pairs, ++count) {
          const uint32_t acc = count & 1u;
          ok = all_wait(bar_tempty + 8 * acc, ((count >> 1) & 1u) ^ 1u, abort_flag, error_word);
          if (!ok) break;
          tc_fence_after();
          const uint32_t tmem_d = tmem_base + acc * (uint32_t)kPairTile;
          for (int kt = 0; kt < KT; ++kt, ++kit) {
            const int s = kit % kPairStages;
            ok = all_wait(bar_full + 8 * s, (kit / kPairStages) & 1u, abort_flag, error_word);
            if (!ok) break;
            tc_fence_after();
            const uint32_t off = s * (kPairStage >> 4);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_pair_i8(tmem_d, a_desc + off + 2 * kk, b_desc + off + 2 * kk, i8_idesc(kPairTile, kPairTile), (kt | kk) != 0 ? 1u : 0u);
            commit_pair_elected(bar_empty + 8 * s);
          }
          if (ok) commit_pair_elected(bar_tfull + 8 * acc);
        }
      }
    } else {
      // warp (q, half): tokens 32 q .. of this CTA's 128, channels 128 half ..  A lane takes two of each eight channels for
      // four tokens, so that it needs 32 channels' scales and biases, not 128, and gets them by shuffles: with a token
      // a lane the two shuffles a value bounded the epilogue.
      constexpr int COLS = 128 / (int)sizeof(T);  // channels of a chunk: 128 bytes of C
      const int q = warp & 3, half = (warp - 2) >> 2, quad = lane & 3, row = lane >> 2;
      uint8_t* const stg = gen_base + kPairStages * kPairStage + (warp - 2) * 4096;
      // Of the warp's channels 8 G + 2 u + e this lane fetches u = quad, G = row and row + 8; tokens row + 8 h are its own.
      struct Scales {
        float sb[2][2], bias[2][2], sa[4];
      };
      auto fetch = [&](int tile) {
        Scales f;
        int m0, n0;
        tile_coords(tiles, tile, &m0, &n0);
        m0 += (int)rank * (kPairTile / 2) + q * 32;
        n0 += half * (kPairTile / 2);
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int n = n0 + 8 * (row + 8 * g) + 2 * quad + e;
            f.sb[g][e] = n < p.n ? p.scale_b[n] : 0.0f;
            f.bias[g][e] = n < p.n && p.bias ? p.bias[n] : 0.0f;
          }
#pragma unroll
        for (int h = 0; h < 4; ++h) f.sa[h] = m0 + row + 8 * h < p.m ? p.scale_a[m0 + row + 8 * h] : 0.0f;
        return f;
      };
      uint32_t count = 0;
      bool ok = true;
      Scales next = fetch(pair);  // (the grid has no more pairs than tiles)
      for (int tile = pair; tile < tiles.count && ok; tile += pairs, ++count) {
        int m0, n0;
        tile_coords(tiles, tile, &m0, &n0);
        m0 += (int)rank * (kPairTile / 2) + q * 32;
        n0 += half * (kPairTile / 2);
        const uint32_t acc = count & 1u;
        const Scales at = next;
        if (tile + pairs < tiles.count) next = fetch(tile + pairs);  // on their way under this tile
        ok = __all_sync(0xffffffffu, mbar_wait(bar_tfull + 8 * acc, (count >> 1) & 1u, abort_flag, error_word)) != 0;
        if (!ok) break;
        tc_fence_after();
        const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + acc * (uint32_t)kPairTile + half * (kPairTile / 2);
        uint32_t r[2][16];  // tokens 0 .. 15 and 16 .. 31 of the warp's
        if (m0 < p.m && n0 < p.n) {
          tmem_ld_16x256(taddr, r[0]);
          tmem_ld_16x256(taddr + (16u << 16), r[1]);
        }
#pragma unroll 1
        for (int c0 = 0; c0 < kPairTile / 2; c0 += COLS) {
          if (m0 >= p.m || n0 + c0 >= p.n) break;  // warp-uniform
          bool free_to_write = !TMA_STORE;
#pragma unroll
          for (int x = 0; x < COLS / 32; ++x) {
            const int first = c0 + 32 * x;
            float v[32];  // [channel group g][token h][e]
            tmem_ld_wait();
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              // group first / 8 + g: the same half of the warp's sixteen for all g
              const int from = ((first / 8 + g) & 7) * 4 + quad;
              float s2[2], b2[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                s2[e] = __shfl_sync(0xffffffffu, first < 64 ? at.sb[0][e] : at.sb[1][e], from);
                b2[e] = __shfl_sync(0xffffffffu, first < 64 ? at.bias[0][e] : at.bias[1][e], from);
              }
#pragma unroll
              for (int h = 0; h < 4; ++h)
                scaled2((int)r[h >> 1][4 * g + 2 * (h & 1)], (int)r[h >> 1][4 * g + 2 * (h & 1) + 1], at.sa[h], make_float2(s2[0], s2[1]),
                        make_float2(b2[0], b2[1]), &v[8 * g + 2 * h], &v[8 * g + 2 * h + 1]);
            }
            // (channels behind n are products of zeros with a scale of zero)
            if (first + 32 < kPairTile / 2) {
              tmem_ld_16x256(taddr + first + 32, r[0]);
              tmem_ld_16x256(taddr + (16u << 16) + first + 32, r[1]);
            }
            activate(p.act, v);
            if (!free_to_write) {
              if (lane == 0) bulk_wait_read<0>();  // the chunk before has left the staging tile
              __syncwarp();
              free_to_write = true;
            }
            if (sizeof(T) == 4) {
              // 8 bytes a lane; odd rows take group g ^ 2, so that the sixteen lanes of a store meet all banks
#pragma unroll
              for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                  const bool odd = row & 1;
                  const float lo = odd ? v[8 * (g ^ 2) + 2 * h] : v[8 * g + 2 * h], hi = odd ? v[8 * (g ^ 2) + 2 * h + 1] : v[8 * g + 2 * h + 1];
                  const int piece = 2 * (g ^ (odd ? 2 : 0)) + (quad >> 1);
                  *reinterpret_cast<float2*>(stg + (row + 8 * h) * 128 + ((piece ^ row) << 4) + (quad & 1) * 8) = make_float2(lo, hi);
                }
            } else {
#pragma unroll
              for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int h = 0; h < 4; ++h)
                  *reinterpret_cast<uint32_t*>(stg + (row + 8 * h) * 128 + (((4 * x + g) ^ row) << 4) + quad * 4) =
                      pack2<T>(v[8 * g + 2 * h], v[8 * g + 2 * h + 1]);
            }
          }
          if (TMA_STORE) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmap_c, n0 + c0, m0, smem_u32(stg));
              bulk_commit();
            }
          } else {
            __syncwarp();
            constexpr int PER = COLS / 32;  // values a lane
            const int n = n0 + c0 + lane * PER;
#pragma unroll 4
            for (int t = 0; t < 32; ++t) {
              if (m0 + t >= p.m) break;
              const T* from = reinterpret_cast<const T*>(stg + t * 128 + (((lane >> 2) ^ (t & 7)) << 4) + (lane & 3) * 4);
              T* const out = static_cast<T*>(p.c) + (m0 + t) * p.ldc + n;
#pragma unroll
              for (int e = 0; e < PER; ++e)
                if (n + e < p.n) out[e] = from[e];
            }
            __syncwarp();
          }
        }
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_u32(bar_tempty + 8 * acc, 0));
      }
      if (TMA_STORE && lane == 0) bulk_wait_all();  // the stores read this CTA's shared memory
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {  // given up
    if (warp == 0 && lane == 0) {
      // both CTAs' copies count on the leader's barriers; the other one cannot wait there and gives its own their time
      if (leader) ring_settle(bar_full, kPairStages, kit);
      else for (const unsigned long long t0 = global_ns(); global_ns() - t0 < 1000000ull;) {}
    }
    if (warp == 1 && leader) {
      commit_pair_elected(bar_out);
      mbar_settle(bar_out, 0);
    }
    __syncwarp();
  }
  cluster_sync_all();  // the peer may read this CTA's shared memory until its last MMA is done
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ---------------------------------------------------------------- host

int make_map(CUtensorMap* map, CUtensorMapDataType type, int bytes, const void* ptr, long long rows, long long cols, long long ld,
             int box_cols, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(ANNC_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * bytes};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, type, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(ANNC_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return ANNC_OK;
}
int operand_map(CUtensorMap* map, const int8_t* ptr, long long rows, long long k, long long ld, int box_rows) {
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, ptr, rows, k, ld, KB, box_rows);
}

template <int TN, typename T>
int launch_split(const Params& p, int split, int* error_word, cudaStream_t s) {
  void (*const kernel)(CUtensorMap, CUtensorMap, Params, int, int*) = gemm_i8_split_kernel<TN, T>;
  static bool attr_done[kMaxDevices] = {};
  const int dev = device_slot();
  if (!attr_done[dev]) {
    ANNC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)SplitShape<TN>::kSmem));
    attr_done[dev] = true;
  }
  CUtensorMap tw, tt;
  ANNC_TRY(operand_map(&tw, p.b, p.n, p.k, p.ldb, box_rows(p.n, kChannels)));
  ANNC_TRY(operand_map(&tt, p.a, p.m, p.k, p.lda, box_rows(p.m, TN)));
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cudaLaunchAttribute attr[2];
  attr[0] = pdl_attribute();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)split;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)split * (unsigned)((p.n + kChannels - 1) / kChannels) * (unsigned)((p.m + TN - 1) / TN), 1, 1);
  cfg.blockDim = dim3(kSplitThreads, 1, 1);
  cfg.dynamicSmemBytes = SplitShape<TN>::kSmem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  ANNC_CUDA(cudaLaunchKernelEx(&cfg, kernel, tw, tt, p, split, error_word));
  return ANNC_OK;
}

template <typename T, bool TMA_STORE>
int launch_pair_as(const Params& p, int* error_word, cudaStream_t s) {
  void (*const kernel)(CUtensorMap, CUtensorMap, CUtensorMap, Params, PairTiles, int*) = gemm_i8_pair_kernel<T, TMA_STORE>;
  static int max_pairs_dev[kMaxDevices] = {};
  int& max_pairs = max_pairs_dev[device_slot()];
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1] = pdl_attribute();
  cfg.gridDim = dim3(2, 1, 1);
  cfg.blockDim = dim3(kPairThreads, 1, 1);
  cfg.dynamicSmemBytes = kPairSmem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (max_pairs == 0) {
    ANNC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPairSmem));
    int n = 0;
    ANNC_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
    if (n < 1) return fail(ANNC_ERR_CUDA, "no CTA pair fits this device");
    max_pairs = n;
  }
  CUtensorMap ta, tb, tc;
  ANNC_TRY(operand_map(&ta, p.a, p.m, p.k, p.lda, kPairTile / 2));
  ANNC_TRY(operand_map(&tb, p.b, p.n, p.k, p.ldb, kPairTile / 2));
  if (TMA_STORE)
    ANNC_TRY(make_map(&tc, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, sizeof(T), p.c, p.m,
                      p.n, p.ldc, 128 / (int)sizeof(T), 32));
  else tc = ta;
  PairTiles t;
  t.channels = (p.n + kPairTile - 1) / kPairTile;
  t.tokens = (p.m + kPairTile - 1) / kPairTile;
  t.count = t.channels * t.tokens;
  cfg.gridDim.x = 2u * (unsigned)(t.count < max_pairs ? t.count : max_pairs);
  cfg.stream = s;
  cfg.numAttrs = 2;
  ANNC_CUDA(cudaLaunchKernelEx(&cfg, kernel, ta, tb, tc, p, t, error_word));
  return ANNC_OK;
}
// (a TMA store clips at the tensor's edge in pieces of 16 bytes)
bool pair_stores_by_tma(const Params& p) {
  const int size = p.c_dtype == ANNC_F32 ? 4 : 2, piece = 16 / size;
  return (reinterpret_cast<uintptr_t>(p.c) & 15) == 0 && p.ldc % piece == 0 && p.n % piece == 0 && p.ldc * (long long)size < (1LL << 40);
}
template <typename T>
int launch_pair(const Params& p, int* error_word, cudaStream_t s) {
  return pair_stores_by_tma(p) ? launch_pair_as<T, true>(p, error_word, s) : launch_pair_as<T, false>(p, error_word, s);
}

}  // namespace

// Which kernel and shape: the smallest of their times as these sums model them (us, bf16 output, figures fitted to
// 64 products from 1 x 512 x 256 to 16384 x 8192 x 256; 148 SMs).
//   split  2.4 for launch and prologue; per round of CTAs a k-step 0.165 + 0.00014 TN (latency: a CTA streams alone on
//          its SM; 0.286 for 256 tokens, 48 KB) and, unsplit, 0.0098 TN to write the tile; 2.6 for each further round (its
//          CTAs start, allocate tensor memory and fill their stages); split, once 0.6 + 0.022 TN for the sums of the
//          cluster
//   pair   2.9 for launch and prologue and the last tile's epilogue; a k-step 0.31, a tile at least what the epilogue under
//          it takes, 3.0, and 5.2 if C's rows do not allow TMA
// Measured, split kernel's best / pair: 1024 x 1024 x 1024 4.8 / 8.3, 512 x 4096 x 2048 7.2 / 10.8, 1024 x 4096 x 2048 10.2 /
// 11.5, 2048 x 1024 x 8192 16.1 / 24.3, 4096 x 1024 x 8192 24.8 / 25.1, 700 x 8192 x 4096 28.1 / 25.6, 2048 x 4096 x 2048
// 19.7 / 15.4, 16384 x 256 x 1024 7.8 / 8.3, 16384 x 512 x 1024 15.3 / 11.3, 16384 x 1024 x 64 21.7 / 15.3, 8192 x 4096 x 2048
// 74 / 46.
Route route_of(const Params& p) {
  Route best = {ROUTE_SIMT, 0, 0};
  // TMA wants rows on 16 bytes
  if (p.k < 1 || ((reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b)) & 15) || p.lda % 16 || p.ldb % 16) return best;
  const int kt = (p.k + KB - 1) / KB;
  const long long pair_tiles = ((p.m + 255LL) / 256) * ((p.n + 255LL) / 256);
  if (pair_tiles > (1LL << 30)) return best;
  const double main = 0.31 * kt;
  const long long pair_rounds = (pair_tiles + 73) / 74;
  const double epilogue = pair_stores_by_tma(p) ? 3.0 : 5.2;
  double us = 2.9 + epilogue + main + (double)(pair_rounds - 1) * (main > epilogue ? main : epilogue);
  best.kind = ROUTE_PAIR;
  for (int tn = 16; tn <= 256; tn *= 2) {
    const long long tiles = ((p.n + 127LL) / 128) * ((p.m + tn - 1LL) / tn);
    if (tiles > (1LL << 20)) continue;
    // (15 clusters of eight, 33 of four and 74 of two CTAs fit the chip at once)
    for (int split = 1; split <= 8 && split <= kt; split *= 2) {
      if (split > 1 && tiles > (split == 8 ? 15 : split == 4 ? 33 : 74)) break;
      const long long rounds = (tiles * split + 147) / 148;
      const double step = tn == 256 ? 0.286 : 0.165 + 0.00014 * tn;
      const double t = 2.4 + (double)rounds * ((kt + split - 1) / split * step + (split == 1 ? 0.0098 * tn : 0.0)) + 2.6 * (double)(rounds - 1) +
                       (split > 1 ? 0.6 + 0.022 * tn : 0.0);
      if (t < us) {
        us = t;
        best = {ROUTE_SPLIT, tn, split};
      }
    }
  }
  return best;
}

namespace {
template <typename T>
int run_as(const Params& p, const Route& r, cudaStream_t s) {
  int* word = gemm::gemm_error_word();
  if (!word) return fail(ANNC_ERR_CUDA, "gemm error word is not addressable");
  if (r.kind == ROUTE_PAIR) return launch_pair<T>(p, word, s);
  switch (r.tokens) {
    case 16: return launch_split<16, T>(p, r.split, word, s);
    case 32: return launch_split<32, T>(p, r.split, word, s);
    case 64: return launch_split<64, T>(p, r.split, word, s);
    case 128: return launch_split<128, T>(p, r.split, word, s);
    default: return launch_split<256, T>(p, r.split, word, s);
  }
}
}  // namespace

int run_tc(const Params& p, const Route& r, cudaStream_t s) {
  if (p.c_dtype == ANNC_F32) return run_as<float>(p, r, s);
  if (p.c_dtype == ANNC_BF16) return run_as<__nv_bfloat16>(p, r, s);
  return run_as<__half>(p, r, s);
}

}  // namespace gemm_i8
}  // namespace annc
