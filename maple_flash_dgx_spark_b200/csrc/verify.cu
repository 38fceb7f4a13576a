// Verification of drafted tokens against the target's probabilities, from the
// caller's uniforms (speculative decoding).  No counterpart in the reference,
// which samples one token per step (kernels/sampler.py:24-206).
//
// At node n of a sequence's tree the target's distribution is the fused
// sampler's: the top_k largest logits (ties to the lowest id), weights
// e^((v - v_max) / T), normalised, kept while the sum before them is <= top_p,
// normalised again.  From node 0 the children of the current node are tried in
// index order: token x of child c is accepted where u_c q(x) < p(x), q being
// the draft's distribution at the current node (all on x without one);
// otherwise p <- norm(max(p - q, 0)), and q loses x unless the draft drew with
// replacement.  The walk goes on at the accepted child; where none is left the
// next token comes from p by the inverse of its distribution at u_0, ids in
// order of falling logits.  The emitted tokens follow the target's
// distribution exactly (for drafts drawn from q).
//
// Comparisons with a uniform decide which token comes out, so everything after
// the selection (at most 64 values per node) is held in 64 bits.
#include <cooperative_groups.h>
#include <utility>

#include "bulk.cuh"
#include "common.cuh"
#include "launch.cuh"

namespace mb {

namespace cg = cooperative_groups;

constexpr int kVerMaxK = 64;
constexpr int kVerMaxNodes = 64;
constexpr int kVerThreads = 256;
constexpr int kVerVecs = 8;      // 16-byte vectors per thread and tile
constexpr int kVerCap = 128;     // candidates that a tile may hand on

struct VerifyParams {
  const void* logits;     // [B, N, V], V contiguous
  const int64_t* tokens;  // [B, N]
  const int32_t* parents; // [B, N]
  const float* uniform;   // [B, N]
  const void* draft;      // [B, N, V] or null, V contiguous
  uint2* cand;            // [B * N, tiles, kVerCap] candidates: key, id
  int32_t* n_cand;        // [B * N, tiles]
  int32_t* path;          // [B, N]
  int32_t* n_path;        // [B]
  int64_t* out;           // [B, N]
  int* err;
  int64_t l_sb, l_sn, d_sb, d_sn;
  double inv_t, top_p;
  int B, N, V, K, tiles, replacement;
};

// Order-preserving word of a logit: larger logit, larger word; NaN as -inf,
// -0 as +0 (equal logits are ties).
__device__ __forceinline__ uint32_t logit_key(float v) {
  if (v != v) v = __int_as_float(0xff800000);
  const uint32_t u = __float_as_uint(v + 0.0f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}
// Inclusive prefixes of 64 values, value j in lane j % 32 of a[j / 32].
__device__ __forceinline__ void warp_prefix_d(const double (&a)[2], double (&c)[2], int lane) {
#pragma unroll
  for (int u = 0; u < 2; ++u) c[u] = a[u];
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const double o0 = __shfl_up_sync(0xffffffffu, c[0], m), o1 = __shfl_up_sync(0xffffffffu, c[1], m);
    if (lane >= m) {
      c[0] += o0;
      c[1] += o1;
    }
  }
  c[1] += __shfl_sync(0xffffffffu, c[0], 31);
}

// ------------------------------------------------------------- tile kernel --
// The logits are read once.  A CTA takes a tile of a row, eight 16-byte vectors
// per thread in flight together, and keeps each vector's maximum.  T, just
// below the K-th largest of the 256 threads' maxima, is at most the tile's
// K-th largest logit, and few logits reach it (about K of 16384: threads seldom
// hold two); the vectors that do are looked into again.  T is found bit
// by bit, one warp counting the maxima with votes, from the first bit in which
// they differ until close to K of them reach it: a T a little too low only lets
// a few more through.  Where more than kVerCap come through (ties, large logits
// side by side) the tile's K largest are selected exactly, ties to the lowest
// ids.  -inf and NaN are not handed on: they have no weight, and a row of
// nothing else is known by having no candidates.  Five CTAs per SM: their loads
// cover each other's search for T, and their tiles stay in L1 for the second
// look.  64 x 8 rows of 151936 bf16 at K = 50: 33 us, 4.7 TB/s, 25 without the
// second look; past L1 it took 37, with each thread looking at its own vectors
// instead of the CTA's put together 37 as well, from a ring of tiles in shared
// memory with two CTAs per SM 45.  16 x 24 rows at K = 20: 25 us.
// One word whose order is larger logit, then lower id.
__device__ __forceinline__ unsigned long long cand_word(const uint2& v) {
  return (unsigned long long)v.x << 32 | (0xffffffffu - v.y);
}
// Larger of two words of logits (two bf16, or one fp32), NaN giving way.
template <int XT>
__device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b) {
  if constexpr (XT == kBF16) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
    return r;
  } else {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
}
template <int XT>
__device__ __forceinline__ float word_max(uint32_t w) {
  if constexpr (XT == kBF16) return fmaxf(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __uint_as_float(w);
}

// Exactly the K largest logits above -inf of a tile (elements k0 .. of row x),
// all of them where there are fewer, in no order, into `list`; their number.
// The smallest one's word by halving, all above it, and its first ties in order
// of ids, the tile read again each time (it fits L1 as the CTAs lie).  For all
// threads of the CTA at once.
template <int XT>
__device__ __noinline__ int verify_tile_exact(const VerifyParams& p, const char* x, int k0, uint2* list, int* s_cnt,
                                              int* s_warp) {
  constexpr int EPC = XT == kBF16 ? 8 : 4, SH = XT == kBF16 ? 16 : 0, TILE = kVerThreads * kVerVecs * EPC;
  constexpr uint32_t kInf = 0x007fffffu >> SH;  // word of -inf
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto word = [&](int j) -> uint32_t {  // 0 outside of the row
    const int k = k0 + j;
    return k >= 0 && k < p.V ? logit_key(load_f<XT>(x, k)) >> SH : 0u;
  };
  int flip = 0;
  auto count = [&](uint32_t c) {  // words at or above c
    if (tid == 0) s_cnt[flip] = 0;
    __syncthreads();
    int cnt = 0;
#pragma unroll 8
    for (int j = tid; j < TILE; j += kVerThreads) cnt += word(j) >= c;
    cnt = __reduce_add_sync(0xffffffffu, cnt);
    if (lane == 0) atomicAdd(&s_cnt[flip], cnt);
    __syncthreads();
    cnt = s_cnt[flip];
    flip ^= 1;
    return cnt;
  };
  const int want = min(p.K, count(kInf + 1));
  if (want == 0) return 0;
  uint32_t kth = 0;
  for (int bit = 31 - SH; bit >= 0; --bit)
    if (count(kth | (1u << bit)) >= want) kth |= 1u << bit;
  __syncthreads();  // everyone has the last count
  if (tid == 0) s_cnt[0] = 0;
  __syncthreads();
  auto key_of = [](uint32_t w) {  // the whole word again
    return XT == kBF16 ? (w & 0x8000u ? w << 16 : w << 16 | 0xffffu) : w;
  };
  for (int j = tid; j < TILE; j += kVerThreads) {
    const uint32_t w = word(j);
    if (w > kth) list[atomicAdd(&s_cnt[0], 1)] = make_uint2(key_of(w), (uint32_t)(k0 + j));
  }
  __syncthreads();
  int base = s_cnt[0];  // fewer than `want`
  for (int j0 = 0; j0 < TILE && base < want; j0 += kVerThreads) {
    const unsigned vote = __ballot_sync(0xffffffffu, word(j0 + tid) == kth);
    if (lane == 0) s_warp[warp] = __popc(vote);
    __syncthreads();
    int at = base + __popc(vote & ((1u << lane) - 1u)), all = 0;
    for (int w = 0; w < kVerThreads / 32; ++w) {
      if (w < warp) at += s_warp[w];
      all += s_warp[w];
    }
    if (((vote >> lane) & 1u) && at < want) list[at] = make_uint2(key_of(kth), (uint32_t)(k0 + j0 + tid));
    base += all;
    __syncthreads();
  }
  return want;
}

// A word that at least K, and not many more, of 32 x PER words reach, for one
// warp: bit by bit from the first bit in which they differ, counting with votes.
template <int PER, typename At>
__device__ __forceinline__ uint32_t warp_threshold(At at, int K, int last_bit, int lane) {
  uint32_t key[PER], hi = 0, lo = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    key[i] = at(lane + 32 * i);
    hi = max(hi, key[i]);
    lo = min(lo, key[i]);
  }
  hi = __reduce_max_sync(0xffffffffu, hi);
  lo = __reduce_min_sync(0xffffffffu, lo);
  if (K == 1) return hi;
  const int top = 31 - __clz((int)(hi ^ lo));  // -1: they are all equal
  uint32_t t = top < 0 ? lo : lo & ~((2u << top) - 1u);
  int reach = 32 * PER;
  for (int bit = top; bit >= last_bit && reach > K + (K >> 3); --bit) {
    const uint32_t c = t | (1u << bit);
    int cnt = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) cnt += __popc(__ballot_sync(0xffffffffu, key[i] >= c));
    if (cnt >= K) {
      t = c;
      reach = cnt;
    }
  }
  return t;
}

// Vector v of a tile (its first element k of the row): the row's logits, -inf
// outside of it.
template <int XT>
__device__ __forceinline__ uint4 edge_vector(const char* x, int k, int V) {
  constexpr int EPC = XT == kBF16 ? 8 : 4;
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < EPC; ++e) {
    const bool in = k + e >= 0 && k + e < V;
    if constexpr (XT == kBF16) {
      const uint32_t h = in ? reinterpret_cast<const uint16_t*>(x)[k + e] : 0xff80u;
      w[e >> 1] |= h << (16 * (e & 1));
    } else {
      w[e] = in ? reinterpret_cast<const uint32_t*>(x)[k + e] : 0xff800000u;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int XT>
__global__ void __launch_bounds__(kVerThreads, 5) verify_tile_kernel(VerifyParams p) {
  constexpr int ES = XT == kBF16 ? 2 : 4, EPC = 16 / ES, SH = XT == kBF16 ? 16 : 0;  // SH: low key bits that say nothing
  constexpr int VECS = kVerVecs * kVerThreads, TILE = VECS * EPC;
  __shared__ float s_max[kVerThreads];
  __shared__ uint32_t s_t;
  __shared__ int s_n, s_vecs, s_cnt[2];
  __shared__ int s_warp[kVerThreads / 32];
  __shared__ uint16_t s_vec[VECS];
  __shared__ uint2 s_list[kVerCap];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int tile = blockIdx.x, n = blockIdx.y, b = blockIdx.z;
  pdl_wait();
  pdl_trigger();
  const int64_t row = (int64_t)b * p.N + n;
  const char* x = static_cast<const char*>(p.logits) + (b * p.l_sb + n * p.l_sn) * ES;
  const int off = (int)(reinterpret_cast<uintptr_t>(x) & 15) / ES;  // elements between a 16-byte boundary and the row
  const int k0 = tile * TILE - off;                                 // the tile's first element; < 2^30 + a tile
  const bool inner = k0 >= 0 && k0 + TILE <= p.V;
  if (p.parents[row] < -1) return;  // padding
  const char* src = x + ((int64_t)k0 + tid * EPC) * ES;
  uint4 r[kVerVecs];
  if (inner) {
#pragma unroll
    for (int i = 0; i < kVerVecs; ++i) r[i] = ld_u4(src + i * kVerThreads * 16);
  } else {
#pragma unroll
    for (int i = 0; i < kVerVecs; ++i) {
      const int k = k0 + (i * kVerThreads + tid) * EPC;
      r[i] = k >= 0 && k + EPC <= p.V ? ld_u4(src + i * kVerThreads * 16) : edge_vector<XT>(x, k, p.V);
    }
  }
  if (tid == 0) s_n = s_vecs = 0;
  float vm[kVerVecs], mx = __int_as_float(0xff800000);
#pragma unroll
  for (int i = 0; i < kVerVecs; ++i) {
    vm[i] = word_max<XT>(max_word<XT>(max_word<XT>(r[i].x, r[i].y), max_word<XT>(r[i].z, r[i].w)));
    mx = fmaxf(mx, vm[i]);
  }
  s_max[tid] = mx;
  __syncthreads();
  constexpr uint32_t kLowest = 0x00800000u;  // word of the lowest finite value
  if (warp == 0) {
    const uint32_t t = warp_threshold<kVerThreads / 32>([&](int j) { return logit_key(s_max[j]); }, p.K, SH, lane);
    if (lane == 0) s_t = max(t, kLowest);  // fewer than K finite maxima: all that is above -inf
  }
  __syncthreads();
  const float tf = key_logit(s_t);
  // the vectors that reach T, put together so that few warps look into them
  uint32_t in = 0;
#pragma unroll
  for (int i = 0; i < kVerVecs; ++i) in |= (vm[i] >= tf ? 1u : 0u) << i;
  if (in) {
    int at = atomicAdd(&s_vecs, __popc(in));
    for (; in; in &= in - 1) s_vec[at++] = (uint16_t)((__ffs((int)in) - 1) * kVerThreads + tid);
  }
  __syncthreads();
#pragma unroll 1
  for (int j = tid; j < s_vecs; j += kVerThreads) {
    const int k = k0 + s_vec[j] * EPC;
    const uint4 v = k >= 0 && k + EPC <= p.V ? ld_u4(x + (int64_t)k * ES) : edge_vector<XT>(x, k, p.V);
    const uint32_t q[4] = {v.x, v.y, v.z, v.w};
    auto value = [&](int e) {  // e a constant
      const uint32_t w = q[e * ES / 4];
      return __uint_as_float(XT == kBF16 ? (e & 1 ? w & 0xffff0000u : w << 16) : w);
    };
    uint32_t reach = 0;
#pragma unroll
    for (int e = 0; e < EPC; ++e) reach |= (value(e) >= tf && k + e >= 0 && k + e < p.V ? 1u : 0u) << e;
    int at = atomicAdd(&s_n, __popc(reach));
#pragma unroll
    for (int e = 0; e < EPC; ++e) {
      if ((reach >> e) & 1u) {
        if (at < kVerCap) s_list[at] = make_uint2(logit_key(value(e)), (uint32_t)(k + e));
        ++at;
      }
    }
  }
  __syncthreads();
  int found = s_n;
  if (found > kVerCap) {
    found = verify_tile_exact<XT>(p, x, k0, s_list, s_cnt, s_warp);
    __syncthreads();
  }
  const int64_t slot = row * p.tiles + tile;
  if (tid < found) p.cand[slot * kVerCap + tid] = s_list[tid];
  if (tid == 0) p.n_cand[slot] = found;
}

// ------------------------------------------------------------------- walk --
// One cluster of CTAs per sequence, four warps per node: the K largest of the
// node's candidates in order, their weights, and the draft's probabilities at
// them, into the shared memory of the cluster's first CTA, where one warp then
// walks with nothing left to fetch.  Bound by latency, so the work is spread: a
// thread per candidate of a tile (kVerCap = 128 of them), and per kept one that
// counts what stands before it.  64 x 8, 50 kept of 600 candidates: 13 us, of
// which the candidates take 3, their limit and order 3.5, weights and draft 1,
// the cluster 1 and the walk down eight nodes 3.5; with one warp per node 28.
constexpr int kVerBuf = 1024;                 // candidates of a node held at a time
constexpr int kVerRank = kVerCap;             // of which at most so many are put in order by counting
constexpr int kVerWalkThreads = 512;
constexpr int kVerGroups = kVerWalkThreads / kVerCap;  // nodes at a time in a CTA

struct VerGroup {
  unsigned long long buf[kVerBuf];
  unsigned long long lim[kVerCap / 32][2];
  int cnt[2][kVerCap / 32];
  int n;
};

__device__ __forceinline__ void group_sync(int group) {
  asm volatile("bar.sync %0, %1;\n" ::"r"(1 + group), "n"(kVerCap) : "memory");
}

// The K best of a row's candidates, in order, in g.buf[0 ..]; their number.
// first_counts: lane's count among the first 32 tiles, fetched ahead.
__device__ __forceinline__ int row_select(const VerifyParams& p, int64_t row, int first_counts, VerGroup& g, int group,
                                          int gt) {
  constexpr int WARPS = kVerCap / 32;
  const int lane = gt & 31, warp = gt >> 5;
  static_assert(kVerMaxK + kVerCap <= kVerBuf, "a tile fits behind what is carried");
  int have = 0, flip = 0;  // carried from the batches before
  for (int t0 = 0; t0 < p.tiles;) {
    // as many of the next 32 tiles as fit
    const int c = t0 == 0 ? first_counts : t0 + lane < p.tiles ? __ldcg(&p.n_cand[row * p.tiles + t0 + lane]) : 0;
    int pre = c;  // c and its prefixes: 0 and the total past the last tile
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, pre, m);
      if (lane >= m) pre += o;
    }
    const int nt = min(__popc(__ballot_sync(0xffffffffu, have + pre <= kVerBuf)), p.tiles - t0);
    const int total = have + __shfl_sync(0xffffffffu, pre, nt - 1);
    const uint2* src = p.cand + (row * p.tiles + t0) * kVerCap + gt;
#pragma unroll 1
    for (int t = 0; t < nt; t += 8) {
      uint2 v[8];
      int at[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int cnt = __shfl_sync(0xffffffffu, c, (t + i) & 31), end = __shfl_sync(0xffffffffu, pre, (t + i) & 31);
        at[i] = t + i < nt && gt < cnt ? have + end - cnt + gt : -1;
        if (at[i] >= 0) v[i] = __ldcg(src + (t + i) * kVerCap);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (at[i] >= 0) g.buf[at[i]] = cand_word(v[i]);
    }
    group_sync(group);
    const int want = min(p.K, total);
    int m = total;
    if (total > kVerRank) {
      // a word that between `want` and kVerRank of them reach, from the first bit in which they differ
      unsigned long long hi = 0, lo = ~0ull;
      for (int e = gt; e < total; e += kVerCap) {
        hi = max(hi, g.buf[e]);
        lo = min(lo, g.buf[e]);
      }
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) {
        hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      }
      if (lane == 0) {
        g.lim[warp][0] = hi;
        g.lim[warp][1] = lo;
      }
      if (gt == 0) g.n = 0;
      group_sync(group);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        hi = max(hi, g.lim[w][0]);
        lo = min(lo, g.lim[w][1]);
      }
      const int top = 63 - __clzll((long long)(hi ^ lo));  // the words are all different
      unsigned long long t = top == 63 ? 0ull : lo & ~((2ull << top) - 1ull);
#pragma unroll 1
      for (int bit = top; bit >= 0 && m > kVerRank; --bit) {
        const unsigned long long d = t | (1ull << bit);
        int cnt = 0;
#pragma unroll 4
        for (int e = gt; e < total; e += kVerCap) cnt += g.buf[e] >= d;
        cnt = __reduce_add_sync(0xffffffffu, cnt);
        if (lane == 0) g.cnt[flip][warp] = cnt;
        group_sync(group);
        cnt = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) cnt += g.cnt[flip][w];
        flip ^= 1;
        if (cnt >= want) {
          t = d;
          m = cnt;
        }
      }
      unsigned long long v[kVerBuf / kVerCap];
#pragma unroll
      for (int i = 0; i < kVerBuf / kVerCap; ++i) v[i] = gt + i * kVerCap < total ? g.buf[gt + i * kVerCap] : 0ull;
      group_sync(group);
#pragma unroll
      for (int i = 0; i < kVerBuf / kVerCap; ++i)
        if (gt + i * kVerCap < total && v[i] >= t) g.buf[atomicAdd(&g.n, 1)] = v[i];
      group_sync(group);
    }
    // in order: each counts what stands before it
    const unsigned long long v = gt < m ? g.buf[gt] : 0ull;
    int r = gt < m ? 0 : kVerMaxK;
    if (gt < m) {
#pragma unroll 8
      for (int j = 0; j < m; ++j) r += g.buf[j] > v;
    }
    group_sync(group);
    if (r < want) g.buf[r] = v;
    group_sync(group);
    have = want;
    t0 += nt;
  }
  return have;
}

template <int DT>
__global__ void __launch_bounds__(kVerWalkThreads) verify_walk_kernel(VerifyParams p) {
  extern __shared__ __align__(16) unsigned char dyn[];
  VerGroup* s_group = reinterpret_cast<VerGroup*>(dyn);                     // [kVerGroups]
  double* s_w = reinterpret_cast<double*>(s_group + kVerGroups);            // [N][64] weights, falling
  int* s_id = reinterpret_cast<int*>(s_w + p.N * kVerMaxK);                 // [N][64] their token ids
  float* s_q = reinterpret_cast<float*>(s_id + p.N * kVerMaxK);             // [N][64] the draft's probabilities of them
  float* s_raw = s_q + p.N * kVerMaxK;                                      // [N] that of the node's token at its parent
  const cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, group = tid / kVerCap, gt = tid % kVerCap;
  const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks(), b = (int)(blockIdx.x / ranks);
  auto here = cluster.barrier_arrive();  // every CTA has begun before one writes to another's shared memory
  pdl_wait();
  pdl_trigger();
  cluster.barrier_wait(std::move(here));
  const int64_t base = (int64_t)b * p.N;
  for (int n = rank * kVerGroups + group; n < p.N; n += ranks * kVerGroups) {
    const int parent = p.parents[base + n];
    const int64_t own = p.tokens[base + n];
    const int counts = lane < p.tiles ? __ldcg(&p.n_cand[(base + n) * p.tiles + lane]) : 0;
    if (parent < -1) continue;  // padding: never looked at
    VerGroup& g = s_group[group];
    const int have = row_select(p, base + n, counts, g, group, gt);
    if (gt < 32) {
      // `have` of K logits above -inf (none: the lowest ids share alike)
      constexpr int DS = DT == kBF16 ? 2 : 4;
      float q[2] = {0.0f, 0.0f}, raw = 0.0f;
      int id[2];
      unsigned long long word[2];
      if (p.draft != nullptr && parent >= 0 && parent < n && own >= 0 && own < p.V)
        raw = load_f<DT>(static_cast<const char*>(p.draft) + (b * p.d_sb + parent * p.d_sn) * DS, own);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int j = lane + 32 * u;
        word[u] = j < have ? g.buf[j] : 0ull;
        id[u] = j < have ? (int)(0xffffffffu - (uint32_t)word[u]) : have == 0 && j < p.K ? j : -1;
        if (p.draft != nullptr && id[u] >= 0)
          q[u] = load_f<DT>(static_cast<const char*>(p.draft) + (b * p.d_sb + n * p.d_sn) * DS, id[u]);
      }
      const float v0 = key_logit((uint32_t)(g.buf[0] >> 32));
      double w[2], c[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float v = key_logit((uint32_t)(word[u] >> 32));
        w[u] = id[u] < 0 ? 0.0 : have == 0 || v == v0 ? 1.0 : exp(((double)v - (double)v0) * p.inv_t);
      }
      // the nucleus: falling weights are kept while the sum before them is at most top_p of all
      warp_prefix_d(w, c, lane);
      const double most = p.top_p * __shfl_sync(0xffffffffu, c[1], 31);
      bool keep[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) keep[u] = c[u] - w[u] <= most;
      const unsigned long long kept = ((unsigned long long)__ballot_sync(0xffffffffu, keep[1]) << 32) |
                                      __ballot_sync(0xffffffffu, keep[0]);
      const int last = 63 - __clzll((long long)kept);  // the first one always is
      const double inv = 1.0 / __shfl_sync(0xffffffffu, last < 32 ? c[0] : c[1], last & 31);
      double* l_w = cluster.map_shared_rank(s_w, 0) + n * kVerMaxK;
      int* l_id = cluster.map_shared_rank(s_id, 0) + n * kVerMaxK;
      float* l_q = cluster.map_shared_rank(s_q, 0) + n * kVerMaxK;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        l_w[lane + 32 * u] = keep[u] ? w[u] * inv : 0.0;
        l_id[lane + 32 * u] = id[u];
        l_q[lane + 32 * u] = q[u];
      }
      if (lane == 0) cluster.map_shared_rank(s_raw, 0)[n] = raw;
    }
    group_sync(group);  // the buffer is free again
  }
  cluster.sync();
  if (rank != 0 || tid >= 32) return;
  int par[2];
  int64_t tok[2];
  float un[2], rw[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = lane + 32 * u;
    par[u] = i < p.N ? p.parents[base + i] : -2;
    tok[u] = i < p.N ? p.tokens[base + i] : -1;
    un[u] = i < p.N ? p.uniform[base + i] : 0.0f;
    rw[u] = i < p.N && p.draft != nullptr ? s_raw[i] : 0.0f;
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = lane + 32 * u;
    if (i < p.N) {
      p.path[base + i] = -1;
      p.out[base + i] = -1;
    }
  }
  const bool wrong = par[0] >= lane || par[1] >= lane + 32;
  if (wrong) atomicOr(p.err, kErrFlagBounds);
  __syncwarp();
  int kept = 0;
  if (__shfl_sync(0xffffffffu, par[0], 0) == -1) {  // below it padding, above it not before its node: padding too
    const float u0 = __shfl_sync(0xffffffffu, un[0], 0);
    int cur = 0, done = 0;  // children up to `done` have been tried
    double pr[2], q[2], left = 1.0;
    int id[2];
    auto enter = [&]() {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int j = cur * kVerMaxK + lane + 32 * u;
        pr[u] = s_w[j];
        id[u] = s_id[j];
        q[u] = (double)s_q[j];
      }
      left = 1.0;
      if (lane == 0) p.path[base + kept] = cur;
      ++kept;
    };
    enter();
    for (;;) {
      const unsigned long long kids =
          ((unsigned long long)__ballot_sync(0xffffffffu, par[1] == cur && lane + 32 > cur) << 32) |
          __ballot_sync(0xffffffffu, par[0] == cur && lane > cur);
      const unsigned long long todo = done >= 63 ? 0ull : kids & (~0ull << (done + 1));
      if (todo == 0) break;
      const int c = __ffsll((long long)todo) - 1;
      done = c;
      const int64_t x = __shfl_sync(0xffffffffu, c < 32 ? tok[0] : tok[1], c & 31);
      const double uc = (double)__shfl_sync(0xffffffffu, c < 32 ? un[0] : un[1], c & 31);
      const bool in = x >= 0 && x < p.V;
      if (!in && lane == 0) atomicOr(p.err, kErrFlagBounds);
      bool hit[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) hit[u] = in && id[u] == (int)x;
      const unsigned h0 = __ballot_sync(0xffffffffu, hit[0]), h1 = __ballot_sync(0xffffffffu, hit[1]);  // one at most
      const double px = (h0 | h1) ? __shfl_sync(0xffffffffu, h0 ? pr[0] : pr[1], __ffs((int)(h0 | h1)) - 1) : 0.0;
      double qx = 1.0, raw = 0.0;
      if (p.draft != nullptr) {
        // a token refused before is no longer there to draw
        const unsigned long long twin =
            (((unsigned long long)__ballot_sync(0xffffffffu, tok[1] == x) << 32) |
             __ballot_sync(0xffffffffu, tok[0] == x)) & kids & ((1ull << c) - 1ull);
        raw = (double)__shfl_sync(0xffffffffu, c < 32 ? rw[0] : rw[1], c & 31);
        if (!p.replacement && twin != 0) raw = 0.0;
        qx = fmin(raw / left, 1.0);
      }
      if (uc * qx < px) {
        if (lane == 0) p.out[base + kept - 1] = x;
        cur = c;
        enter();
        continue;
      }
      double r[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const double qn = p.draft != nullptr ? fmin(q[u] / left, 1.0) : (hit[u] ? 1.0 : 0.0);
        r[u] = fmax(pr[u] - qn, 0.0);
      }
      const double total = warp_sum_d(r[0] + r[1]);
      if (total > 0.0) {
        const double inv = 1.0 / total;
        pr[0] = r[0] * inv;
        pr[1] = r[1] * inv;
      }
      if (p.draft != nullptr && !p.replacement) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (hit[u]) q[u] = 0.0;
        left = fmax(left - raw, 1e-30);
      }
    }
    double c[2];
    warp_prefix_d(pr, c, lane);
    const double target = (double)u0 * __shfl_sync(0xffffffffu, c[1], 31);
    const unsigned long long below =
        ((unsigned long long)__ballot_sync(0xffffffffu, c[1] <= target) << 32) | __ballot_sync(0xffffffffu, c[0] <= target);
    const unsigned long long some =
        ((unsigned long long)__ballot_sync(0xffffffffu, pr[1] > 0.0) << 32) | __ballot_sync(0xffffffffu, pr[0] > 0.0);
    const int last = some ? 63 - __clzll((long long)some) : 0;
    const int pick = min(__popcll(below), last);
    const int nxt = __shfl_sync(0xffffffffu, pick < 32 ? id[0] : id[1], pick & 31);
    if (lane == 0) p.out[base + kept - 1] = nxt;
  }
  if (lane == 0) p.n_path[b] = kept;
}

// Tiles of a row of `vocab` logits, `per` of them in 16 bytes, wherever the row starts.
inline int64_t verify_tiles(int64_t vocab, int64_t per) {
  const int64_t tile = (int64_t)kVerThreads * kVerVecs * per;
  return (vocab + per - 1 + tile - 1) / tile;
}

}  // namespace mb

using namespace mb;

extern "C" int64_t maple_verify_tree_workspace_bytes(int64_t batch, int64_t nodes, int64_t vocab, int64_t top_k) {
  if (batch < 0 || nodes <= 0 || nodes > kVerMaxNodes || vocab <= 0 || vocab > (1LL << 30) || top_k <= 0) return -1;
  return batch * nodes * verify_tiles(vocab, 4) * (kVerCap * 8 + 4) + 16;  // fp32 rows have the more tiles
}

extern "C" int maple_verify_tree(const void* logits, int x_dtype, int64_t batch, int64_t nodes, int64_t vocab,
                                 int64_t l_sb, int64_t l_sn, const int64_t* tokens, const int32_t* parents,
                                 const float* uniform, const void* draft_probs, int d_dtype, int64_t d_sb,
                                 int64_t d_sn, float temperature, float top_p, int64_t top_k, int replacement,
                                 int32_t* path, int32_t* n_path, int64_t* out, void* workspace,
                                 int64_t workspace_bytes, int* err, void* stream) {
  if (batch < 0 || nodes <= 0 || nodes > kVerMaxNodes || vocab <= 0 || vocab > (1LL << 30) || batch > 65535)
    return kErrShape;
  if (batch == 0) return kOk;
  if (top_k <= 0 || top_k > kVerMaxK || !(temperature > 0.0f) || !(top_p > 0.0f)) return kErrShape;
  if ((x_dtype != kF32 && x_dtype != kBF16) || (draft_probs && d_dtype != kF32 && d_dtype != kBF16)) return kErrDtype;
  if (!logits || !tokens || !parents || !uniform || !path || !n_path || !out || !err) return kErrShape;
  if (!workspace || workspace_bytes < maple_verify_tree_workspace_bytes(batch, nodes, vocab, top_k)) return kErrWorkspace;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return kErrAlign;
  VerifyParams p{};
  p.logits = logits; p.tokens = tokens; p.parents = parents; p.uniform = uniform; p.draft = draft_probs;
  const int64_t rows = batch * nodes;
  p.tiles = (int)verify_tiles(vocab, x_dtype == kBF16 ? 8 : 4);
  p.cand = static_cast<uint2*>(workspace);
  p.n_cand = reinterpret_cast<int32_t*>(p.cand + rows * p.tiles * kVerCap);
  p.path = path; p.n_path = n_path; p.out = out; p.err = err;
  p.l_sb = l_sb; p.l_sn = l_sn; p.d_sb = d_sb; p.d_sn = d_sn;
  p.inv_t = 1.0 / (double)temperature; p.top_p = (double)top_p;
  p.B = (int)batch; p.N = (int)nodes; p.V = (int)vocab; p.K = (int)(top_k < vocab ? top_k : vocab);
  p.replacement = replacement != 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)p.tiles, (unsigned)nodes, (unsigned)batch);
  cudaError_t e = x_dtype == kBF16 ? launch_k(verify_tile_kernel<kBF16>, grid, dim3(kVerThreads), 0, st, p)
                                   : launch_k(verify_tile_kernel<kF32>, grid, dim3(kVerThreads), 0, st, p);
  if (e == cudaSuccess) {
    auto* walk = (draft_probs && d_dtype == kBF16) ? verify_walk_kernel<kBF16> : verify_walk_kernel<kF32>;
    const unsigned want = (unsigned)((nodes + kVerGroups - 1) / kVerGroups), ranks = want < 8 ? want : 8;  // portable
    const int smem = (int)(kVerGroups * sizeof(VerGroup)) + (int)nodes * kVerMaxK * 16 + kVerMaxNodes * 4;
    static std::atomic<uint64_t> done[2];
    const int most = (int)(kVerGroups * sizeof(VerGroup)) + kVerMaxNodes * (kVerMaxK * 16 + 4);
    e = smem_once(done[draft_probs && d_dtype == kBF16], walk, most);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)batch * ranks);
    cfg.blockDim = dim3(kVerWalkThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, walk, p);
  }
  return e == cudaSuccess ? kOk : kErrCuda;
}
