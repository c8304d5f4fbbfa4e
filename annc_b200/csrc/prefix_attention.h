// Internal interface of the shared-prefix attention.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "annc_b200.h"

namespace annc {
namespace attention {

struct Rows {  // [rows, heads, head_dim] with strides in elements
  const void* data;
  long long row, head;
};
struct Params {
  Rows q, kp, vp, ko, vo;
  void* out;
  long long out_row, out_head;
  float* lse;
  const int64_t* own_begin;
  const int32_t* own_len;
  const int32_t* q_begin;
  long long tokens, sequences, prefix, own_rows;
  int heads, kv_heads, group, dim;
  float scale;
};

// ---- The prefix on tensor cores, its parts and the own keys joined (prefix_attention_tc.cu)
//
// The rows (token, head of the group) of a key head form one matrix.  An item is up to 256 of its rows (two tiles of
// `tile_tokens` tokens) against the whole prefix, `kv_tiles` tiles of 128 keys.  All items' key tiles, one item after
// the other, are dealt to the CTAs in equal contiguous shares of `per_cta`; so an item is cut where a share ends, and what
// a CTA has of an item (a part) is left in the workspace as unnormalised sums with their maximum and weight.
constexpr int kTileRows = 128, kTileKeys = 128, kPartRows = 2 * kTileRows;
constexpr int kMaxCtas = 148;

struct Plan {
  int tile_tokens;  // tokens of a tile: as many whole groups of heads as fit 128 rows
  int row_items;    // items of a key head
  int items, kv_tiles;
  int per_cta, ctas;

  // Parts: CTA c leaves what it has of the item its share starts in at 2 c, of the one it ends in at 2 c + 1, and an item
  // that it has all of (`parts` is 1) behind all these, at the item's number.
#ifdef __CUDACC__
  __device__ __forceinline__ int part_of(int item, int cta, int parts) const {
    return parts == 1 ? 2 * kMaxCtas + item : 2 * cta + (cta * per_cta < item * kv_tiles ? 1 : 0);
  }
#endif
};

inline Plan plan_of(long long tokens, int kv_heads, int group, long long prefix) {
  Plan p;
  p.tile_tokens = kTileRows / group;
  p.row_items = (int)((tokens + 2LL * p.tile_tokens - 1) / (2LL * p.tile_tokens));
  p.items = p.row_items * kv_heads;
  p.kv_tiles = (int)((prefix + kTileKeys - 1) / kTileKeys);
  const long long total = (long long)p.items * p.kv_tiles;
  long long per = (total + kMaxCtas - 1) / kMaxCtas;
  if (per < 2 && p.kv_tiles > 1) per = 2;  // (two key tiles of a small item run side by side)
  if (per < 1) per = 1;
  p.per_cta = (int)per;
  p.ctas = (int)((total + per - 1) / per);
  return p;
}
inline int part_width(int dim) { return dim <= 64 ? 64 : 128; }

bool tc_supported(const Params& p, int dtype);
size_t tc_workspace_bytes(long long tokens, int heads, int kv_heads, int dim);
int run_tc(const Params& p, int dtype, void* workspace, cudaStream_t s);

#ifdef __CUDACC__
// The keys of a token's own sequence that it sees: rows first .. first + count - 1 of the own keys.  False for a
// token that belongs to no sequence.  Bounds are clamped, whatever the arrays hold: no row outside the buffer is read.
__device__ __forceinline__ bool own_keys(const Params& p, long long token, long long* first, int* count) {
  *first = 0;
  *count = 0;
  long long seq = token;
  long long behind = 0;  // tokens of the sequence behind this one
  if (p.q_begin) {
    if (p.sequences == 0 || token < p.q_begin[0] || token >= p.q_begin[p.sequences]) return false;
    long long lo = 0, hi = p.sequences;  // q_begin[lo] <= token < q_begin[hi]
    while (hi - lo > 1) {
      const long long mid = (lo + hi) >> 1;
      if (p.q_begin[mid] <= token) lo = mid;
      else hi = mid;
    }
    seq = lo;
    behind = (long long)p.q_begin[seq + 1] - 1 - token;
  }
  if (!p.own_len) return true;
  const long long begin = p.own_begin[seq], len = p.own_len[seq] - behind;
  if (len <= 0 || begin < 0 || begin >= p.own_rows) return true;
  *first = begin;
  *count = (int)min(len, p.own_rows - begin);
  return true;
}
#endif

}  // namespace attention
}  // namespace annc
