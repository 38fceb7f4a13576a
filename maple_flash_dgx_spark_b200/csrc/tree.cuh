// Attention over a KV cache for trees of drafted tokens: what the mma.sync and
// the tcgen05 kernels share (arguments, visibility, the split of a row's
// keys and the layout of the partial results).
//
// A sequence has s = seqlen[b] cached positions and N <= 64 drafted nodes
// whose K/V rows stand behind them, node j at slot s + j.  mask_i has bit j
// set where node i sees node j (its ancestors and itself); the node's position
// is p_i = s + popcount(mask_i) - 1.  Node i sees key t < s, and key s + j
// where bit j is set; with a window W > 0 only keys whose position is above
// p_i - W.  mask_i = 0 marks padding: its output is zero.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace mb {

// Two fp32 in one 64-bit register: a * b + c and a + b, each rounded once.
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void f2_get(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
constexpr int kTreeMaxNodes = 64;
constexpr int kTreeMaxSplits = 64;
constexpr int kTreeMaxGroup = 4096;  // query heads per KV head: (row of 64 nodes) x group stays below 2^32

struct TreeAttnParams {
  const void* q;              // [B, N, H, D], D contiguous
  const void* kc;             // [Bc, Hkv, T, D]
  const void* vc;
  const int64_t* seqlen;      // [B]
  const unsigned long long* mask;  // [B, N]
  const int32_t* row_map;     // [B] cache row, or null: b
  void* out;                  // [B, N, H, D] contiguous
  float* ws_acc;              // unnormalised partial sums of each row, split and dim
  float* ws_ml;               // maximum and sum of weights of each row and split
  int* err;
  int64_t q_sb, q_sn, q_sh, c_sb, c_sh;
  int B, N, H, Hkv, G, Bc, T, NS, window, join;
  float scale;
};

// The keys of a sequence of length s in cache row cb: [lo, hi) of slots, hi = s + (nodes in use); every
// node's visible keys are inside.  Empty (lo = hi) where the sequence has no
// node or its length or cache row is not in the cache.
struct TreeRange {
  int s, lo, hi, cb;
  bool bad;
};

__device__ __forceinline__ TreeRange tree_range(const TreeAttnParams& p, int64_t s, int cb, unsigned long long used) {
  TreeRange r;
  r.cb = cb;
  const int n = 64 - __clzll((long long)used);  // nodes up to the last one that is real or seen
  r.bad = s < 0 || s > p.T || cb < 0 || cb >= p.Bc || s + n > p.T;
  if (r.bad || n == 0) {
    r.bad = r.bad && n > 0;
    r.s = r.lo = r.hi = 0;
    return r;
  }
  r.s = (int)s;
  r.hi = r.s + n;
  r.lo = p.window > 0 ? max(0, r.s + 1 - p.window) : 0;  // depth 0 reaches back the furthest
  return r;
}

// Split sp of NS: tiles [t0, t1) of `tile` keys each, counted from lo.  The
// number of splits is fixed by the shapes, the split's length by the row's own
// length: a row's result depends on no other row.
__device__ __forceinline__ void tree_split(int lo, int hi, int tile, int ns, int sp, int& k0, int& k1) {
  const int tiles = (hi - lo + tile - 1) / tile;
  const int per = (tiles + ns - 1) / ns;
  k0 = min(hi, lo + sp * per * tile);
  k1 = min(hi, k0 + per * tile);
}

// How many splits hold keys.
__device__ __forceinline__ int tree_splits_used(int lo, int hi, int tile, int ns) {
  const int tiles = (hi - lo + tile - 1) / tile;
  if (tiles == 0) return 0;
  const int per = (tiles + ns - 1) / ns;
  return (tiles + per - 1) / per;
}

// tree_tc.cu: the tcgen05 kernel (bf16, heads of 64 or 128).
// pair: two row tiles per CTA; join: the splits are joined by their cluster, without partials in memory
int tree_tc_splits(int64_t ctas, int64_t max_len, bool pair, bool* join);
int tree_tc_groups(int64_t rows);
int64_t tree_tc_partial_rows(int64_t rows);  // rows that a split's partials take
cudaError_t tree_tc_launch(const TreeAttnParams& p, int D, cudaStream_t st);

}  // namespace mb
