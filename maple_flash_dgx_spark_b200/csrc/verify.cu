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
#include "bulk.cuh"
#include "common.cuh"
#include "launch.cuh"

namespace mb {

constexpr int kVerMaxK = 64;
constexpr int kVerMaxNodes = 64;
constexpr int kVerThreads = 256;
constexpr int kVerVecs = 8;      // 16-byte vectors per thread and tile
constexpr int kVerCap = 128;     // candidates that a tile may hand on
constexpr int kVerBatch = 4096;  // candidates that a row's selection holds at a time

struct VerifyParams {
  const void* logits;     // [B, N, V], V contiguous
  const int64_t* tokens;  // [B, N]
  const int32_t* parents; // [B, N]
  const float* uniform;   // [B, N]
  const void* draft;      // [B, N, V] or null, V contiguous
  uint2* cand;            // [B * N, tiles, kVerCap] candidates: key, id
  int32_t* n_cand;        // [B * N, tiles]
  double* w;              // [B * N, 64] kept weights, falling
  int32_t* id;            // [B * N, 64] their token ids
  float* q;               // [B * N, 64] the draft's probabilities of them
  float* raw;             // [B * N] the draft's probability of the node's token at its parent
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
  for (int u = 0; u < 2; ++u) {
    c[u] = a[u];
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const double o = __shfl_up_sync(0xffffffffu, c[u], m);
      if (lane >= m) c[u] += o;
    }
  }
  c[1] += __shfl_sync(0xffffffffu, c[0], 31);
}

// A node's distribution from its `have` <= K largest logits above -inf, in order
// (none: all alike).
__device__ __forceinline__ void node_weights(const VerifyParams& p, const uint32_t* key, const int* ids, int have,
                                             int64_t row, int lane) {
  const float v0 = have > 0 ? key_logit(key[0]) : 0.0f;
  double w[2], c[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j = lane + 32 * u;
    w[u] = 0.0;
    if (j < have || (have == 0 && j < p.K)) {
      const float v = have > 0 ? key_logit(key[j]) : 0.0f;
      w[u] = v == v0 ? 1.0 : exp(((double)v - (double)v0) * p.inv_t);
    }
  }
  const double s = warp_sum_d(w[0] + w[1]);
#pragma unroll
  for (int u = 0; u < 2; ++u) w[u] /= s;
  warp_prefix_d(w, c, lane);
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (!(c[u] - w[u] <= p.top_p)) w[u] = 0.0;
  const double t = warp_sum_d(w[0] + w[1]);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j = lane + 32 * u;
    p.w[row * kVerMaxK + j] = w[u] / t;
    p.id[row * kVerMaxK + j] = j < have || (have == 0 && j < p.K) ? ids[j] : -1;
  }
}

// ------------------------------------------------------------- tile kernel --
// The logits are read once.  A CTA takes a tile of a row, eight 16-byte vectors
// per thread in flight together, and keeps each vector's maximum.  T, just
// below the K-th largest of the 256 threads' maxima, is at most the tile's
// K-th largest logit, and few logits reach it (about K of 16384: threads seldom
// hold two); the vectors that do are looked at again, one element per thread.
// T is found bit by bit, one warp counting the maxima with votes, from the
// first bit in which they differ until close to K of them reach it: a T a
// little too low only lets a few more through.  Where more than kVerCap come
// through (ties, large logits side by side) the tile's K largest are selected
// exactly, ties to the lowest ids.  -inf and NaN are not handed on: they have no weight, and a row
// of nothing else is known by having no candidates.
__device__ __forceinline__ uint4 ld_once_u4(const void* p) {  // written by the launch before: not the read-only path
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
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

template <int XT>
struct VerWord { using type = uint32_t; };
template <>
struct VerWord<kBF16> { using type = uint16_t; };

template <int XT>
__global__ void __launch_bounds__(kVerThreads, 5) verify_tile_kernel(VerifyParams p) {
  constexpr int ES = XT == kBF16 ? 2 : 4, EPC = 16 / ES, SH = XT == kBF16 ? 16 : 0;  // SH: low key bits that say nothing
  __shared__ float s_max[kVerThreads];
  __shared__ uint32_t s_t;
  __shared__ int s_n, s_vecs, s_cnt[2];
  __shared__ int s_warp[kVerThreads / 32];
  __shared__ uint4 s_tile[kVerThreads * kVerVecs];  // vectors of interest (their numbers), or the tile's words
  int* s_vec = reinterpret_cast<int*>(s_tile);
  __shared__ uint2 s_list[kVerCap];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int tile = blockIdx.x, n = blockIdx.y, b = blockIdx.z;
  const float ninf = __int_as_float(0xff800000);
  pdl_wait();
  pdl_trigger();
  const int64_t row = (int64_t)b * p.N + n;
  if (p.parents[row] < -1) return;  // padding
  const char* x = static_cast<const char*>(p.logits) + (b * p.l_sb + n * p.l_sn) * ES;
  const int off = (int)(reinterpret_cast<uintptr_t>(x) & 15) / ES;  // elements between a 16-byte boundary and the row
  const int k0 = tile * (kVerVecs * kVerThreads) * EPC - off;       // the tile's first element; < 2^30 + a tile
  uint4 r[kVerVecs];
#pragma unroll
  for (int i = 0; i < kVerVecs; ++i) {
    const int k = k0 + (i * kVerThreads + tid) * EPC;
    if (k >= 0 && k + EPC <= p.V) {
      r[i] = ld_once_u4(x + (int64_t)k * ES);
    } else {  // the row's ends, element by element; -inf outside
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < EPC; ++e) {
        const bool in = k + e >= 0 && k + e < p.V;
        if constexpr (XT == kBF16) {
          const uint32_t h = in ? reinterpret_cast<const uint16_t*>(x)[k + e] : 0xff80u;
          w[e >> 1] |= h << (16 * (e & 1));
        } else {
          w[e] = in ? reinterpret_cast<const uint32_t*>(x)[k + e] : 0xff800000u;
        }
      }
      r[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if (tid == 0) s_n = s_vecs = 0;
  float vm[kVerVecs], mx = ninf;
#pragma unroll
  for (int i = 0; i < kVerVecs; ++i) {
    const uint32_t w = max_word<XT>(max_word<XT>(r[i].x, r[i].y), max_word<XT>(r[i].z, r[i].w));
    vm[i] = word_max<XT>(w);
    mx = fmaxf(mx, vm[i]);
  }
  s_max[tid] = mx;
  __syncthreads();
  if (warp == 0) {
    uint32_t key[kVerThreads / 32], hi = 0, lo = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < kVerThreads / 32; ++i) {
      key[i] = logit_key(s_max[lane + 32 * i]);
      hi = max(hi, key[i]);
      lo = min(lo, key[i]);
    }
    hi = __reduce_max_sync(0xffffffffu, hi);
    lo = __reduce_min_sync(0xffffffffu, lo);
    const int top = 31 - __clz((int)(hi ^ lo));  // first bit in which they differ; -1: they are all equal
    uint32_t t = top < 0 ? lo : lo & ~((2u << top) - 1u);
    int reach = kVerThreads;
    for (int bit = top; bit >= SH && reach > p.K + (p.K >> 3); --bit) {
      const uint32_t c = t | (1u << bit);
      int cnt = 0;
#pragma unroll
      for (int i = 0; i < kVerThreads / 32; ++i) cnt += __popc(__ballot_sync(0xffffffffu, key[i] >= c));
      if (cnt >= p.K) {
        t = c;
        reach = cnt;
      }
    }
    if (lane == 0) s_t = t;
  }
  __syncthreads();
  // just above -inf where T is not above it (fewer than K finite maxima)
  const uint32_t t = max(s_t, 0x00800000u);
  const float tf = key_logit(t);
  if (mx >= tf) {
#pragma unroll
    for (int i = 0; i < kVerVecs; ++i)
      if (vm[i] >= tf) s_vec[atomicAdd(&s_vecs, 1)] = i * kVerThreads + tid;
  }
  __syncthreads();
  for (int j = tid; j < s_vecs * EPC; j += kVerThreads) {
    const int k = k0 + s_vec[j / EPC] * EPC + j % EPC;
    if (k < 0 || k >= p.V) continue;
    const float v = load_f<XT>(x, k);
    if (v >= tf) {
      const int at = atomicAdd(&s_n, 1);
      if (at < kVerCap) s_list[at] = make_uint2(logit_key(v), (uint32_t)k);
    }
  }
  __syncthreads();
  int found = s_n;
  if (found > kVerCap) {
    // exactly the K largest of the tile, from its words in shared memory: their
    // smallest by halving, all above it, and its first ties in order of ids
    using Word = typename VerWord<XT>::type;
    Word* words = reinterpret_cast<Word*>(s_tile);
    constexpr int TILE = kVerThreads * kVerVecs * EPC;
#pragma unroll 8
    for (int j = tid; j < TILE; j += kVerThreads) {
      const int k = k0 + j;
      const uint32_t key = k >= 0 && k < p.V ? logit_key(load_f<XT>(x, k)) : 0u;
      words[j] = (Word)(key >= t ? key >> SH : 0u);  // 0: not of interest
    }
    uint32_t kth = 0;
    int flip = 0;
#pragma unroll 1
    for (int bit = 31 - SH; bit >= 0; --bit) {
      const uint32_t c = kth | (1u << bit);
      if (tid == 0) s_cnt[flip] = 0;
      __syncthreads();
      int cnt = 0;
#pragma unroll 2
      for (int i = 0; i < kVerVecs; ++i) {
        const uint4 v = s_tile[i * kVerThreads + tid];
        const uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (XT == kBF16) cnt += ((q[e] & 0xffffu) >= c) + ((q[e] >> 16) >= c);
          else cnt += q[e] >= c;
        }
      }
      cnt = __reduce_add_sync(0xffffffffu, cnt);
      if (lane == 0) atomicAdd(&s_cnt[flip], cnt);
      __syncthreads();
      if (s_cnt[flip] >= p.K) kth = c;
      flip ^= 1;
    }
    if (tid == 0) s_n = 0;
    __syncthreads();
    auto key_of = [](uint32_t w) {  // the whole word again
      return XT == kBF16 ? (w & 0x8000u ? w << 16 : w << 16 | 0xffffu) : w;
    };
    for (int j = tid; j < TILE; j += kVerThreads)
      if (words[j] > kth) s_list[atomicAdd(&s_n, 1)] = make_uint2(key_of(words[j]), (uint32_t)(k0 + j));
    __syncthreads();
    int base = s_n;  // fewer than K
#pragma unroll 1
    for (int j0 = 0; j0 < TILE && base < p.K; j0 += kVerThreads) {
      const unsigned vote = __ballot_sync(0xffffffffu, words[j0 + tid] == kth);
      if (lane == 0) s_warp[warp] = __popc(vote);
      __syncthreads();
      int at = base + __popc(vote & ((1u << lane) - 1u)), all = 0;
      for (int w = 0; w < kVerThreads / 32; ++w) {
        if (w < warp) at += s_warp[w];
        all += s_warp[w];
      }
      if (((vote >> lane) & 1u) && at < p.K) s_list[at] = make_uint2(key_of(kth), (uint32_t)(k0 + j0 + tid));
      base += all;
      __syncthreads();
    }
    found = p.K;
  }
  const int64_t slot = row * p.tiles + tile;
  if (tid < found) p.cand[slot * kVerCap + tid] = s_list[tid];
  if (tid == 0) p.n_cand[slot] = found;
}

// -------------------------------------------------------------- row kernel --
// One CTA per node: the K largest of the tiles' candidates in order, their
// weights, and the draft's probabilities at them (so that the walk has nothing
// left to fetch token by token).  The K-th largest word is found bit by bit
// over the candidates in shared memory, what reaches it is put in order by
// counting what stands before each.
constexpr int kVerRank = 128;  // candidates that are put in order by counting

// One word whose order is larger logit, then lower id.
__device__ __forceinline__ unsigned long long cand_word(const uint2& v) {
  return (unsigned long long)v.x << 32 | (0xffffffffu - v.y);
}

template <int DT>
__global__ void __launch_bounds__(kVerThreads) verify_row_kernel(VerifyParams p) {
  __shared__ uint2 s_c[kVerBatch];
  __shared__ unsigned long long s_best[kVerRank];
  __shared__ uint2 s_sorted[kVerMaxK];
  __shared__ uint32_t s_key[kVerMaxK];
  __shared__ int s_id[kVerMaxK];
  __shared__ int s_red[2][kVerThreads / 32];
  __shared__ int s_off[33];
  __shared__ int s_m;
  constexpr int PER = (kVerBatch - kVerMaxK) / kVerCap;  // tiles per batch
  static_assert(PER <= 32, "a warp scans a batch's counts");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = blockIdx.x, b = blockIdx.y;
  pdl_wait();
  pdl_trigger();
  const int64_t row = (int64_t)b * p.N + n;
  const int parent = p.parents[row];
  if (parent < -1) return;
  int flip = 0;
  auto count = [&](auto pred, int m) {  // candidates of the batch for which pred holds
    int c = 0;
    for (int e = tid; e < m; e += kVerThreads) c += pred(s_c[e]);
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0) s_red[flip][warp] = c;
    __syncthreads();
    c = 0;
#pragma unroll
    for (int w = 0; w < kVerThreads / 32; ++w) c += s_red[flip][w];
    flip ^= 1;
    return c;
  };
  int have = 0;  // candidates carried from the batches before
  for (int t0 = 0; t0 < p.tiles; t0 += PER) {
    const int nt = min(PER, p.tiles - t0);
    if (warp == 0) {
      int c = lane < nt ? __ldcg(&p.n_cand[row * p.tiles + t0 + lane]) : 0, pre = c;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, pre, m);
        if (lane >= m) pre += o;
      }
      s_off[lane] = have + pre - c;
      if (lane == 31) s_off[32] = have + pre;
    }
    __syncthreads();
    for (int t = warp; t < nt; t += kVerThreads / 32) {
      const int at = s_off[t], c = s_off[t + 1] - at;
      for (int e = lane; e < c; e += 32) s_c[at + e] = __ldcg(&p.cand[(row * p.tiles + t0 + t) * kVerCap + e]);
    }
    if (tid < have) s_c[tid] = s_sorted[tid];
    __syncthreads();
    const int total = s_off[32], want = min(p.K, total);
    int m = total;
    if (total > kVerRank) {
      // cut down to between `want` and kVerRank: T from the first bit in which the words differ
      uint32_t hi = 0, lo = 0xffffffffu;
      for (int e = tid; e < total; e += kVerThreads) {
        hi = max(hi, s_c[e].x);
        lo = min(lo, s_c[e].x);
      }
      hi = __reduce_max_sync(0xffffffffu, hi);
      lo = __reduce_min_sync(0xffffffffu, lo);
      if (lane == 0) {
        s_red[0][warp] = (int)hi;
        s_red[1][warp] = (int)lo;
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kVerThreads / 32; ++w) {
        hi = max(hi, (uint32_t)s_red[0][w]);
        lo = min(lo, (uint32_t)s_red[1][w]);
      }
      __syncthreads();
      const int top = 31 - __clz((int)(hi ^ lo));
      uint32_t t = top < 0 ? lo : lo & ~((2u << top) - 1u);
      int k = total;
      for (int bit = top; bit >= 0 && k > kVerRank; --bit) {
        const uint32_t c = t | (1u << bit);
        const int kc = count([&](const uint2& v) { return v.x >= c; }, total);
        if (kc >= want) {
          t = c;
          k = kc;
        }
      }
      uint32_t last = 0xffffffffu;  // highest id taken among the words equal to t
      if (k > kVerRank) {
        const int ties = want - count([&](const uint2& v) { return v.x > t; }, total);
        last = 0;
        for (int bit = 30; bit >= 0; --bit) {  // ids are below 2^30; last + 1 such that `ties` are below it
          const uint32_t c = last | (1u << bit);
          if (count([&](const uint2& v) { return v.x == t && v.y < c; }, total) < ties) last = c;
        }
      }
      if (tid == 0) s_m = 0;
      __syncthreads();
      for (int e = tid; e < total; e += kVerThreads) {
        const uint2 v = s_c[e];
        if (v.x > t || (v.x == t && v.y <= last)) s_best[atomicAdd(&s_m, 1)] = cand_word(v);
      }
      __syncthreads();
      m = s_m;
    } else {
      if (tid < total) s_best[tid] = cand_word(s_c[tid]);
      __syncthreads();
    }
    if (tid < m) {
      const unsigned long long v = s_best[tid];
      int r = 0;
#pragma unroll 8
      for (int j = 0; j < m; ++j) r += s_best[j] > v;
      if (r < want) s_sorted[r] = make_uint2((uint32_t)(v >> 32), 0xffffffffu - (uint32_t)v);
    }
    __syncthreads();
    have = want;
  }
  if (tid < kVerMaxK) {
    const uint2 v = tid < have ? s_sorted[tid] : make_uint2(0u, 0u);
    s_key[tid] = v.x;
    s_id[tid] = have > 0 ? (int)v.y : tid;  // nothing above -inf: the lowest ids share alike
    if (p.draft != nullptr) {
      const bool used = tid < have || (have == 0 && tid < p.K);
      p.q[row * kVerMaxK + tid] =
          used ? load_f<DT>(static_cast<const char*>(p.draft) + (b * p.d_sb + n * p.d_sn) * (DT == kBF16 ? 2 : 4), s_id[tid])
               : 0.0f;
    }
  }
  if (tid == kVerMaxK && p.draft != nullptr) {
    const int64_t x = p.tokens[row];
    p.raw[row] = parent >= 0 && parent < n && x >= 0 && x < p.V
                     ? load_f<DT>(static_cast<const char*>(p.draft) +
                                  (b * p.d_sb + parent * p.d_sn) * (DT == kBF16 ? 2 : 4), x)
                     : 0.0f;
  }
  __syncthreads();
  if (warp == 0) node_weights(p, s_key, s_id, have, row, lane);
}

// ------------------------------------------------------------------- walk --
// One CTA per sequence: all of its nodes' distributions into shared memory at
// once, then one warp walks, nodes and candidates two per lane.
__global__ void __launch_bounds__(kVerThreads) verify_walk_kernel(VerifyParams p) {
  extern __shared__ __align__(16) unsigned char dyn[];
  double* s_w = reinterpret_cast<double*>(dyn);                 // [N][64]
  int* s_id = reinterpret_cast<int*>(s_w + p.N * kVerMaxK);     // [N][64]
  float* s_q = reinterpret_cast<float*>(s_id + p.N * kVerMaxK); // [N][64]
  const int tid = threadIdx.x, lane = tid & 31, b = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  const int64_t base = (int64_t)b * p.N;
  for (int e = tid; e < p.N * kVerMaxK; e += kVerThreads) {
    s_w[e] = __ldcg(p.w + base * kVerMaxK + e);  // a padding node's is never looked at
    s_id[e] = __ldcg(p.id + base * kVerMaxK + e);
    s_q[e] = p.draft != nullptr ? __ldcg(p.q + base * kVerMaxK + e) : 0.0f;
  }
  int par[2];
  int64_t tok[2];
  float un[2], rw[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = lane + 32 * u;
    par[u] = i < p.N ? p.parents[base + i] : -2;
    tok[u] = i < p.N ? p.tokens[base + i] : -1;
    un[u] = i < p.N ? p.uniform[base + i] : 0.0f;
    rw[u] = i < p.N && p.draft != nullptr ? __ldcg(p.raw + base + i) : 0.0f;
  }
  __syncthreads();
  if (tid >= 32) return;
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
  if (__shfl_sync(0xffffffffu, par[0], 0) >= -1) {
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
      const double px = warp_sum_d((hit[0] ? pr[0] : 0.0) + (hit[1] ? pr[1] : 0.0));
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
        pr[0] = r[0] / total;
        pr[1] = r[1] / total;
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
  const int64_t tiles = verify_tiles(vocab, 4);  // fp32 rows have the more tiles
  return batch * nodes * (tiles * (kVerCap * 8 + 4) + kVerMaxK * 16 + 8) + 64;
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
  p.w = static_cast<double*>(workspace);
  p.cand = reinterpret_cast<uint2*>(p.w + rows * kVerMaxK);
  p.id = reinterpret_cast<int32_t*>(p.cand + rows * p.tiles * kVerCap);
  p.q = reinterpret_cast<float*>(p.id + rows * kVerMaxK);
  p.raw = p.q + rows * kVerMaxK;
  p.n_cand = reinterpret_cast<int32_t*>(p.raw + rows);
  p.path = path; p.n_path = n_path; p.out = out; p.err = err;
  p.l_sb = l_sb; p.l_sn = l_sn; p.d_sb = d_sb; p.d_sn = d_sn;
  p.inv_t = 1.0 / (double)temperature; p.top_p = (double)top_p;
  p.B = (int)batch; p.N = (int)nodes; p.V = (int)vocab; p.K = (int)(top_k < vocab ? top_k : vocab);
  p.replacement = replacement != 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)p.tiles, (unsigned)nodes, (unsigned)batch), rgrid((unsigned)nodes, (unsigned)batch);
  cudaError_t e = x_dtype == kBF16 ? launch_k(verify_tile_kernel<kBF16>, grid, dim3(kVerThreads), 0, st, p)
                                   : launch_k(verify_tile_kernel<kF32>, grid, dim3(kVerThreads), 0, st, p);
  if (e == cudaSuccess)
    e = (draft_probs && d_dtype == kBF16) ? launch_k(verify_row_kernel<kBF16>, rgrid, dim3(kVerThreads), 0, st, p)
                                          : launch_k(verify_row_kernel<kF32>, rgrid, dim3(kVerThreads), 0, st, p);
  if (e == cudaSuccess) {
    const int smem = (int)nodes * kVerMaxK * 16;
    e = cudaFuncSetAttribute(verify_walk_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = launch_k(verify_walk_kernel, dim3((unsigned)batch), dim3(kVerThreads), smem, st, p);
  }
  return e == cudaSuccess ? kOk : kErrCuda;
}
