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
constexpr int kVerThreads = 512;

struct VerifyParams {
  const void* logits;     // [B, N, V], V contiguous
  const int64_t* tokens;  // [B, N]
  const int32_t* parents; // [B, N]
  const float* uniform;   // [B, N]
  const void* draft;      // [B, N, V] or null, V contiguous
  double* w;              // [B * N, 64] kept weights, falling
  int32_t* id;            // [B * N, 64] their token ids
  int32_t* path;          // [B, N]
  int32_t* n_path;        // [B]
  int64_t* out;           // [B, N]
  int* err;
  int64_t l_sb, l_sn, d_sb, d_sn;
  double inv_t, top_p;
  int B, N, V, K, replacement;
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

// A node's distribution from its K largest logits (sorted in v / id).
__device__ __forceinline__ void node_weights(const VerifyParams& p, const uint32_t* key, const int* ids, int64_t row,
                                             int lane) {
  const float v0 = key_logit(key[0]);
  double w[2], c[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j = lane + 32 * u;
    w[u] = 0.0;
    if (j < p.K) {
      const float v = key_logit(key[j]);
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
    p.id[row * kVerMaxK + j] = j < p.K ? ids[j] : -1;
  }
}

// One CTA per node: its K largest logits by radix selection.  Four passes of
// 8 bits over the row (from L2 after the first) find the K-th largest word;
// a last pass collects what is above it and the lowest ids of its ties.
template <int XT>
__global__ void __launch_bounds__(kVerThreads) verify_topk_kernel(VerifyParams p) {
  __shared__ unsigned hist[256];
  __shared__ unsigned s_prefix, s_need, s_count, s_ties;
  __shared__ uint32_t ck[kVerMaxK], sk[kVerMaxK];
  __shared__ int ci[kVerMaxK], si[kVerMaxK];
  __shared__ unsigned wcount[kVerThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = blockIdx.x, b = blockIdx.y;
  pdl_wait();
  pdl_trigger();
  const int64_t row = (int64_t)b * p.N + n;
  if (p.parents[row] < -1) return;  // padding
  const void* x = static_cast<const char*>(p.logits) + (b * p.l_sb + n * p.l_sn) * (XT == kBF16 ? 2 : 4);
  const unsigned K = p.K;
  if (tid == 0) { s_prefix = 0; s_need = K; s_count = 0; s_ties = 0; }
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    const uint32_t prefix = s_prefix;
    for (int k = tid; k < p.V; k += kVerThreads) {
      const uint32_t key = logit_key(load_f<XT>(x, k));
      if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      unsigned need = s_need;
      int d = 255;
      while (d > 0 && hist[d] < need) need -= hist[d--];
      s_need = need;
      s_prefix = (prefix << 8) | (unsigned)d;
    }
    __syncthreads();
  }
  const uint32_t kth = s_prefix;
  const unsigned above = K - s_need;  // words above the K-th; the rest are its first ties
  for (int k0 = 0; k0 < p.V; k0 += kVerThreads) {
    const int k = k0 + tid;
    const uint32_t key = k < p.V ? logit_key(load_f<XT>(x, k)) : 0u;
    if (k < p.V && key > kth) {
      const unsigned at = atomicAdd(&s_count, 1u);
      ck[at] = key;
      ci[at] = k;
    }
    const unsigned vote = __ballot_sync(0xffffffffu, k < p.V && key == kth);
    if (lane == 0) wcount[warp] = __popc(vote);
    __syncthreads();
    unsigned at = s_ties;
    for (int w = 0; w < warp; ++w) at += wcount[w];
    at += __popc(vote & ((1u << lane) - 1u));
    if (((vote >> lane) & 1u) && above + at < K) {
      ck[above + at] = key;
      ci[above + at] = k;
    }
    __syncthreads();
    if (tid == 0)
      for (int w = 0; w < kVerThreads / 32; ++w) s_ties += wcount[w];
  }
  __syncthreads();
  if (tid < (int)K) {  // in order: larger logit first, then the lower id
    int r = 0;
    for (int j = 0; j < (int)K; ++j) r += ck[j] > ck[tid] || (ck[j] == ck[tid] && ci[j] < ci[tid]);
    sk[r] = ck[tid];
    si[r] = ci[tid];
  }
  __syncthreads();
  if (warp == 0) node_weights(p, sk, si, row, lane);
}

// The walk: one warp per sequence, nodes and candidates two per lane.
template <int DT>
__global__ void __launch_bounds__(32) verify_walk_kernel(VerifyParams p) {
  const int lane = threadIdx.x, b = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  const int64_t base = (int64_t)b * p.N;
  int par[2];
  int64_t tok[2];
  float un[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = lane + 32 * u;
    par[u] = i < p.N ? p.parents[base + i] : -2;
    tok[u] = i < p.N ? p.tokens[base + i] : -1;
    un[u] = i < p.N ? p.uniform[base + i] : 0.0f;
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
        const int j = lane + 32 * u;
        pr[u] = __ldcg(p.w + (base + cur) * kVerMaxK + j);
        id[u] = __ldcg(p.id + (base + cur) * kVerMaxK + j);
        q[u] = 0.0;
        if (p.draft != nullptr && id[u] >= 0)
          q[u] = (double)load_f<DT>(static_cast<const char*>(p.draft) +
                                    (b * p.d_sb + cur * p.d_sn) * (DT == kBF16 ? 2 : 4), id[u]);
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
        if (in && (p.replacement || twin == 0))
          raw = (double)load_f<DT>(static_cast<const char*>(p.draft) +
                                   (b * p.d_sb + cur * p.d_sn) * (DT == kBF16 ? 2 : 4), x);
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

}  // namespace mb

using namespace mb;

extern "C" int64_t maple_verify_tree_workspace_bytes(int64_t batch, int64_t nodes, int64_t vocab, int64_t top_k) {
  if (batch < 0 || nodes <= 0 || nodes > kVerMaxNodes || vocab <= 0 || top_k <= 0) return -1;
  return batch * nodes * kVerMaxK * 12;
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
  p.w = static_cast<double*>(workspace);
  p.id = reinterpret_cast<int32_t*>(p.w + batch * nodes * kVerMaxK);
  p.path = path; p.n_path = n_path; p.out = out; p.err = err;
  p.l_sb = l_sb; p.l_sn = l_sn; p.d_sb = d_sb; p.d_sn = d_sn;
  p.inv_t = 1.0 / (double)temperature; p.top_p = (double)top_p;
  p.B = (int)batch; p.N = (int)nodes; p.V = (int)vocab; p.K = (int)(top_k < vocab ? top_k : vocab);
  p.replacement = replacement != 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)nodes, (unsigned)batch);
  cudaError_t e = x_dtype == kBF16 ? launch_k(verify_topk_kernel<kBF16>, grid, dim3(kVerThreads), 0, st, p)
                                   : launch_k(verify_topk_kernel<kF32>, grid, dim3(kVerThreads), 0, st, p);
  if (e == cudaSuccess)
    e = (draft_probs && d_dtype == kBF16) ? launch_k(verify_walk_kernel<kBF16>, dim3((unsigned)batch), dim3(32), 0, st, p)
                                          : launch_k(verify_walk_kernel<kF32>, dim3((unsigned)batch), dim3(32), 0, st, p);
  return e == cudaSuccess ? kOk : kErrCuda;
}
