// Trees of drafted tokens (speculative decoding): the ancestors' masks, the
// attention of every node over the cache and its branch, and the move of the
// accepted rows.  No counterpart in the reference, which decodes one token per
// step (generate.py:168-373).
#include <type_traits>

#include "bulk.cuh"
#include "launch.cuh"
#include "tree.cuh"

namespace mb {

// ------------------------------------------------------------------- plan --
// mask_i = 2^i | mask_parent(i) by pointer doubling: after round r a node's
// mask holds its ancestors within 2^r steps and `up` points 2^r steps up, so
// six rounds cover 64 nodes.  One warp per sequence, nodes `lane` and
// `lane + 32` in registers: no shared memory, no barrier; the 16 bytes per
// node make the launch itself the bound: 1.5 us for 1 x 8, 1.6 for 256 x 64.
__global__ void __launch_bounds__(128) tree_plan_kernel(const int32_t* parents, int64_t sb, int64_t sn, int B, int N,
                                                        unsigned long long* mask, int32_t* depth, int* err) {
  const int lane = threadIdx.x & 31, b = blockIdx.x * 4 + (threadIdx.x >> 5);
  pdl_wait();
  pdl_trigger();
  if (b >= B) return;
  unsigned long long m[2];
  int up[2];
  bool off[2], wrong = false;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = lane + 32 * u;
    const int par = i < N ? parents[(int64_t)b * sb + i * sn] : -2;
    wrong |= i < N && par >= i;
    off[u] = par < -1 || par >= i;
    up[u] = (off[u] || par < 0) ? i : par;
    m[u] = 1ull << i;
  }
#pragma unroll
  for (int r = 0; r < 6; ++r) {
    unsigned long long nm[2];
    int nu[2];
    bool no[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int a = up[u] & 31;
      const bool high = up[u] >= 32;
      const unsigned long long m0 = __shfl_sync(0xffffffffu, m[0], a), m1 = __shfl_sync(0xffffffffu, m[1], a);
      const int u0 = __shfl_sync(0xffffffffu, up[0], a), u1 = __shfl_sync(0xffffffffu, up[1], a);
      const int f0 = __shfl_sync(0xffffffffu, (int)off[0], a), f1 = __shfl_sync(0xffffffffu, (int)off[1], a);
      nm[u] = m[u] | (high ? m1 : m0);
      nu[u] = high ? u1 : u0;
      no[u] = off[u] || (high ? f1 : f0);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) { m[u] = nm[u]; up[u] = nu[u]; off[u] = no[u]; }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = lane + 32 * u;
    if (i >= N) continue;
    mask[(int64_t)b * N + i] = off[u] ? 0ull : m[u];
    depth[(int64_t)b * N + i] = off[u] ? 0 : __popcll(m[u]) - 1;
  }
  if (wrong) atomicOr(err, kErrFlagBounds);
}

// ----------------------------------------------------------------- narrow --
// Saturating, so that no number past int32 turns into a node or a cache row.
// A few hundred numbers: the launch is the bound.
__global__ void __launch_bounds__(256) narrow_kernel(const int64_t* x, int64_t n, int32_t* out) {
  pdl_wait();
  pdl_trigger();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t v = x[i];
    out[i] = v > INT32_MAX ? INT32_MAX : v < INT32_MIN ? INT32_MIN : (int32_t)v;
  }
}

// ------------------------------------- attention, fp32 and heads of 256 --
// One CTA per (split of the keys, KV head and tile of query rows, sequence).
// Row r of a KV head is node r / G, query head h G + r % G; a warp has 16 rows
// and a part of each tile's keys; the parts are joined in shared memory.
// Products on the tensor pipe as tf32 (mma.sync m16n8k8), each fp32 operand x
// split into hi (x in tf32) and lo = x - hi (exact, then rounded to tf32):
// lo hi + hi lo + hi hi leaves out 2^-23 of a product.  The pipe cuts its sums
// instead of rounding them, so an fp32 sum takes at most four steps on it
// before it is added to the rest with fp32's own rounding: 7e-7 of error at
// 4 x 1500, where straight sums had 2.6e-6 (and 8 % less time).  bf16 values are
// their own hi, which saves two of the three products for the scores and one for
// the output; their results' rounding to 2^-8 hides the cut sums, which stay
// straight.  Tiles of 32 keys stand in shared memory as fp32 in two stages
// (cp.async under the tile before); a pitch of D + 4 floats keeps ldmatrix (K, Q)
// and the V reads free of bank conflicts.  The weights stay in registers: key 2t
// of a block of eight takes the place of the product's index t and key 2t + 1
// that of t + 4, which is how the scores' accumulators lie, and V's rows are read
// in that order.
// Infinities do not survive the split (0 x inf), and a masked weight of 0 does
// not keep NaN out: K and V are cleared of both as they arrive.  A score with a
// cleared key is computed again from the cache (each such key by its threads);
// cleared values of V are added at the end for the rows that see them.
// 16 query heads of 256 on 4 KV heads, 8 nodes, 4 x 4096 bf16: 69 us, 980 GB/s
// of cache (115 with four warps that shared no keys); 32 heads of 128 on 8 with
// 64 nodes, 8 x 4000 fp32: 859 us, 39 TFLOP/s (1160).  Bound by the latency of
// its instructions: a scheduler issues in two cycles of five at 8 x 4000, eight
// instructions per product (splits, ldmatrix, V's 4-byte reads), and the
// registers hold no more than four warps on it.
constexpr int kMmaKeys = 32;
constexpr int kMmaWarps = 8, kMmaThreads = 32 * kMmaWarps;

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four 8 x 4 blocks of fp32, a lane's 32 bits as the tf32 fragments want them.
__device__ __forceinline__ void ldsm4(const float* p, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p)));
}
// hi is x rounded to tf32, or cut to it where x may be the largest fp32; lo is
// half a step up, as the pipe ignores the low 13 bits.
template <bool CUT>
__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t& hi, uint32_t& lo) {
  hi = (CUT ? x : x + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi)) + 0x1000u;
}
__device__ __forceinline__ bool odd_f32(uint32_t x) { return (x & 0x7f800000u) == 0x7f800000u; }  // NaN, infinity
__device__ __forceinline__ bool huge_f32(uint32_t x) { return (x & 0x7fffffffu) >= 0x7f7ff000u; }  // or rounds to it
// Without the two bits by which lo would round hi + lo up past fp32 (2^-22 of it).
__device__ __forceinline__ uint32_t cut_huge(uint32_t x) { return huge_f32(x) && !odd_f32(x) ? x & ~3u : x; }

// RW warps of 16 rows beside each other, KW = 8 / RW groups of them with 32 / KW
// keys of each tile, joined at the end.
template <int XT, int D, int RW>
__global__ void __launch_bounds__(kMmaThreads, D == 256 ? 1 : 2)
    tree_mma_kernel(TreeAttnParams p, int row_tiles) {
  constexpr int JG = 4;  // products of V side by side, for their latency
  constexpr int ROWS = 16 * RW, KW = kMmaWarps / RW, JW = 4 / KW;  // JW: blocks of eight keys per warp and tile
  constexpr int PITCH = D + 4, es = XT == kBF16 ? 2 : 4, EPC = 16 / es, CH = D / EPC;
  constexpr int STAGE = 2 * kMmaKeys * PITCH;             // floats: K, then V
  constexpr int PER = kMmaKeys * CH / kMmaThreads;                // 16-byte chunks of K (and of V) per thread
  extern __shared__ __align__(16) float sm[];
  float* sq = sm;                                         // [ROWS][PITCH]
  float* ring = sq + ROWS * PITCH;                    // [2][STAGE]
  __shared__ unsigned long long s_mask[kTreeMaxNodes];
  __shared__ unsigned s_used[2];
  __shared__ int s_dmax, s_fix;
  __shared__ unsigned s_odd[4];                           // keys that were cleared, four tiles in turn
  const int tid = threadIdx.x, lane = tid & 31, warp = (tid >> 5) % RW, kw = (tid >> 5) / RW;
  const int g = lane >> 2, t = lane & 3;
  const int sp = blockIdx.x, h = blockIdx.y / row_tiles, rt = blockIdx.y % row_tiles, b = blockIdx.z;
  const float ninf = __int_as_float(0xff800000);
  const float scale = p.scale * 1.44269504088896341f;  // scores in powers of 2
  pdl_wait();
  pdl_trigger();
  const int64_t len = p.seqlen[b];
  const int cb = p.row_map != nullptr ? p.row_map[b] : b;
  const int rows = p.N * p.G, r0 = rt * ROWS;
  const uint64_t per_g = (1ull << 32) / (unsigned)p.G + 1;  // row / G by a multiplication, exact while row x G < 2^32
  if (tid < 32) {
    const unsigned long long keep = p.N < 64 ? (1ull << p.N) - 1 : ~0ull;
    unsigned long long used = 0;
    int dm = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = lane + 32 * u;
      const unsigned long long m = i < p.N ? p.mask[(int64_t)b * p.N + i] & keep : 0ull;
      s_mask[i] = m;
      used |= m | (m ? 1ull << i : 0ull);
      dm = max(dm, __popcll(m) - 1);
    }
    const unsigned lo = __reduce_or_sync(0xffffffffu, (unsigned)used);
    const unsigned hi = __reduce_or_sync(0xffffffffu, (unsigned)(used >> 32));
    dm = __reduce_max_sync(0xffffffffu, dm);
    if (lane == 0) {
      s_used[0] = lo;
      s_used[1] = hi;
      s_dmax = dm;
      s_fix = 0;
      s_odd[0] = s_odd[1] = s_odd[2] = s_odd[3] = 0;
    }
  }
  __syncthreads();
  const TreeRange rg = tree_range(p, len, cb, ((unsigned long long)s_used[1] << 32) | s_used[0]);
  if (rg.bad && tid == 0) atomicOr(p.err, kErrFlagBounds);
  int k0, k1;
  tree_split(rg.lo, rg.hi, kMmaKeys, p.NS, sp, k0, k1);
  if (sp > 0 && k0 >= k1) return;  // nothing here; split 0 always answers
  const char* kb = static_cast<const char*>(p.kc) + (rg.cb * p.c_sb + h * p.c_sh) * es;
  const char* vb = static_cast<const char*>(p.vc) + (rg.cb * p.c_sb + h * p.c_sh) * es;

  // this thread's chunks of a tile (rows past the split's end as zeros)
  auto load = [&](int t0, int stage) {
    float* st = ring + stage * STAGE;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int c = tid + kMmaThreads * e, r = c / CH, cc = c % CH * EPC;
      const int64_t at = ((int64_t)(t0 + r) * D + cc) * es;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        float* dst = st + kv * kMmaKeys * PITCH + r * PITCH + cc;
        const char* src = (kv ? vb : kb) + at;
        if constexpr (XT == kF32) {
          if (t0 + r < k1) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(smem_u32(dst)), "l"(src) : "memory");
          else *reinterpret_cast<float4*>(dst) = make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
          float f[8];
          widen_u4<kBF16>(t0 + r < k1 ? ld_u4(src) : make_uint4(0u, 0u, 0u, 0u), f);
          *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
          *reinterpret_cast<float4*>(dst + 4) = make_float4(f[4], f[5], f[6], f[7]);
        }
      }
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
  // clears this thread's chunks of NaN and infinities
  auto clear = [&](int stage, int turn) {
    float* st = ring + stage * STAGE;
    uint32_t any = 0;
#pragma unroll
    for (int e = 0; e < 2 * PER; ++e) {
      const int c = tid + kMmaThreads * (e >> 1), r = c / CH, cc = c % CH * EPC;
#pragma unroll
      for (int u = 0; u < EPC; u += 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(st + (e & 1) * kMmaKeys * PITCH + r * PITCH + cc + u);
        any |= huge_f32(x.x) | huge_f32(x.y) | huge_f32(x.z) | huge_f32(x.w);
      }
    }
    if (!any) return;
#pragma unroll 1
    for (int e = 0; e < 2 * PER; ++e) {  // rare
      const int c = tid + kMmaThreads * (e >> 1), r = c / CH, cc = c % CH * EPC;
      for (int u = 0; u < EPC; ++u) {
        uint32_t* x = reinterpret_cast<uint32_t*>(st + (e & 1) * kMmaKeys * PITCH + r * PITCH + cc + u);
        if (!huge_f32(*x)) continue;
        if ((e & 1) && !odd_f32(*x)) {
          *x = cut_huge(*x);
          continue;
        }
        *x = 0u;
        if (e & 1) s_fix = 1;
        else atomicOr(&s_odd[turn & 3], 1u << r);
      }
    }
  };

  if (k0 < k1) load(k0, 0);
  // q rows, zero past the last one; a thread's loads in flight together
  constexpr int QN = ROWS * CH / kMmaThreads, QU = QN < 8 ? QN : 8;
#pragma unroll 1
  for (int e0 = 0; e0 < QN; e0 += QU) {
    uint4 v[QU];
#pragma unroll
    for (int e = 0; e < QU; ++e) {
      const int c = tid + kMmaThreads * (e0 + e), gr = r0 + c / CH;
      v[e] = make_uint4(0u, 0u, 0u, 0u);
      if (gr < rows) {
        const int i = (int)((uint64_t)(unsigned)gr * per_g >> 32), qg = gr - i * p.G;
        v[e] = ld_u4(static_cast<const char*>(p.q) +
                     (b * p.q_sb + i * p.q_sn + (int64_t)(h * p.G + qg) * p.q_sh + c % CH * EPC) * es);
      }
    }
#pragma unroll
    for (int e = 0; e < QU; ++e) {
      const int c = tid + kMmaThreads * (e0 + e);
      float f[EPC];
      widen_u4<XT>(v[e], f);
      if constexpr (XT == kF32) {
#pragma unroll
        for (int u = 0; u < EPC; ++u) f[u] = __uint_as_float(cut_huge(__float_as_uint(f[u])));
      }
#pragma unroll
      for (int u = 0; u < EPC; u += 4)
        *reinterpret_cast<float4*>(&sq[c / CH * PITCH + c % CH * EPC + u]) = make_float4(f[u], f[u + 1], f[u + 2], f[u + 3]);
    }
  }
  // rows g and g + 8 of the warp's 16
  unsigned long long mine[2];
  float m[2] = {ninf, ninf}, l[2] = {0.0f, 0.0f}, acc[D / 8][4];
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    const int r = r0 + warp * 16 + g + 8 * a;
    mine[a] = r < rows ? s_mask[(int)((uint64_t)(unsigned)r * per_g >> 32)] : 0ull;
  }
#pragma unroll
  for (int j = 0; j < D / 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
  auto sees = [&](int a, int key) {  // whether row a sees slot `key` of this split
    const int x = key - rg.s;        // its node, below 0: a cached position
    bool vis = key < k1 && mine[a] != 0 && (x < 0 || ((mine[a] >> (x & 63)) & 1));
    if (p.window > 0) {
      const int kpos = x < 0 ? key : x < kTreeMaxNodes ? rg.s + __popcll(s_mask[x]) - 1 : 0;
      vis = vis && kpos > rg.s + __popcll(mine[a]) - 1 - p.window;
    }
    return vis;
  };
  auto is_mixed = [&](int t0) {
    return t0 + kMmaKeys > min(rg.s, k1) || (p.window > 0 && t0 <= rg.s + s_dmax - p.window);
  };
  const bool idle = r0 + warp * 16 >= rows;  // a warp without rows only loads
  const float* a_at = sq + (warp * 16 + (lane & 7) + (lane >> 3 & 1) * 8) * PITCH + (lane >> 4) * 4;
  int stage = 0;
  for (int t0 = k0, turn = 0; t0 < k1; t0 += kMmaKeys, stage ^= 1, ++turn) {
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    clear(stage, turn);
    __syncthreads();  // the tile is there, and everyone is done with the one before
    if (tid == 0) s_odd[(turn + 2) & 3] = 0;  // read two tiles ago, written in two
    if (t0 + kMmaKeys < k1) load(t0 + kMmaKeys, stage ^ 1);
    const float* sk = ring + stage * STAGE;
    const float* sv = sk + kMmaKeys * PITCH;
    if (!idle) {
      // 16 rows x 8 JW keys: block j, keys 8 j + 2 t, + 1 of rows g (0, 1) and g + 8 (2, 3)
      float s[JW][4] = {};
      const float* b_at = JW == 1 ? sk + (8 * kw + (lane & 7)) * PITCH + (lane >> 3) * 4
                                  : sk + (8 * JW * kw + (lane & 7) + (lane >> 4) * 8) * PITCH + (lane >> 3 & 1) * 4;
#pragma unroll 2
      for (int k4 = 0; k4 < D / 8; k4 += 4) {
        float fresh[JW][4] = {};
        float(&part)[JW][4] = XT == kBF16 ? s : fresh;
        uint32_t y[4];
#pragma unroll
        for (int kk = k4; kk < k4 + 4; ++kk) {
          uint32_t a[4], ah[4], al[4], yh[JW][2], yl[JW][2];
          ldsm4(a_at + 8 * kk, a);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (XT == kBF16) ah[i] = a[i];
            else split_tf32<true>(a[i], ah[i], al[i]);
          }
          auto part_of = [&](int j, int i, uint32_t x) {
            if constexpr (XT == kBF16) yh[j][i] = x;
            else split_tf32<false>(x, yh[j][i], yl[j][i]);
          };
          if constexpr (JW == 1) {
            if (!(kk & 1)) ldsm4(b_at + 8 * kk, y);  // eight keys, two steps
            part_of(0, 0, y[2 * (kk & 1)]);
            part_of(0, 1, y[2 * (kk & 1) + 1]);
          } else {
#pragma unroll
            for (int j = 0; j < JW; j += 2) {
              ldsm4(b_at + 8 * j * PITCH + 8 * kk, y);
#pragma unroll
              for (int i = 0; i < 4; ++i) part_of(j + i / 2, i & 1, y[i]);
            }
          }
          if constexpr (XT != kBF16) {
#pragma unroll
            for (int j = 0; j < JW; ++j) mma_tf32(part[j], al, yh[j][0], yh[j][1]);
#pragma unroll
            for (int j = 0; j < JW; ++j) mma_tf32(part[j], ah, yl[j][0], yl[j][1]);
          }
#pragma unroll
          for (int j = 0; j < JW; ++j) mma_tf32(part[j], ah, yh[j][0], yh[j][1]);
        }
        if constexpr (XT != kBF16) {
#pragma unroll
          for (int j = 0; j < JW; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[j][c] += fresh[j][c];
        }
      }
      if (const unsigned odd = s_odd[turn & 3]; odd) {  // rare: keys with a NaN or an infinity, from the cache
#pragma unroll
        for (int j = 0; j < JW; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int key = 8 * (JW * kw + j) + 2 * t + (c & 1);
            if (!((odd >> key) & 1u)) continue;
            float x = 0.0f;
            const float* qr = sq + (warp * 16 + g + (c >> 1) * 8) * PITCH;
#pragma unroll 1
            for (int d = 0; d < D; ++d) x = fmaf(qr[d], load_f<XT>(kb, (int64_t)(t0 + key) * D + d), x);
            s[j][c] = x;
          }
      }
      const bool mixed = is_mixed(t0);
      float fix[2];
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        float mt = m[a];
#pragma unroll
        for (int j = 0; j < JW; ++j)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float& x = s[j][2 * a + c];
            x = mixed && !sees(a, t0 + 8 * (JW * kw + j) + 2 * t + c) ? ninf : x * scale;
            mt = fmaxf(mt, x);
          }
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
        const float base = mt == ninf ? 0.0f : mt;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < JW; ++j)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float& x = s[j][2 * a + c];
            x = x == ninf ? 0.0f : ex2(x - base);
            sum += x;
          }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        fix[a] = mt == m[a] ? 1.0f : ex2(m[a] - base);
        l[a] = fmaf(l[a], fix[a], sum);
        m[a] = mt;
      }
      if (__any_sync(0xffffffffu, fix[0] != 1.0f || fix[1] != 1.0f)) {
#pragma unroll
        for (int j = 0; j < D / 8; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[j][c] *= fix[c >> 1];
      }
      uint32_t ah[JW][4], al[JW][4];
#pragma unroll
      for (int kk = 0; kk < JW; ++kk) {
        const int order[4] = {0, 2, 1, 3};
#pragma unroll
        for (int i = 0; i < 4; ++i) split_tf32<false>(__float_as_uint(s[kk][order[i]]), ah[kk][i], al[kk][i]);
      }
      const float* v_at = sv + (8 * JW * kw + 2 * t) * PITCH + g;
#pragma unroll
      for (int j0 = 0; j0 < D / 8; j0 += JG) {
        float part[JG][4];
#pragma unroll
        for (int j = 0; j < JG; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) part[j][c] = XT == kBF16 ? acc[j0 + j][c] : 0.0f;
#pragma unroll
        for (int kk = 0; kk < JW; ++kk) {
          uint32_t yh[JG][2], yl[JG][2];
#pragma unroll
          for (int j = 0; j < JG; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t y = __float_as_uint(v_at[(8 * kk + u) * PITCH + 8 * (j0 + j)]);
              if constexpr (XT == kBF16) yh[j][u] = y;
              else split_tf32<true>(y, yh[j][u], yl[j][u]);
            }
#pragma unroll
          for (int j = 0; j < JG; ++j) mma_tf32(part[j], al[kk], yh[j][0], yh[j][1]);
          if constexpr (XT != kBF16) {
#pragma unroll
            for (int j = 0; j < JG; ++j) mma_tf32(part[j], ah[kk], yl[j][0], yl[j][1]);
          }
#pragma unroll
          for (int j = 0; j < JG; ++j) mma_tf32(part[j], ah[kk], yh[j][0], yh[j][1]);
        }
#pragma unroll
        for (int j = 0; j < JG; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[j0 + j][c] = XT == kBF16 ? part[j][c] : acc[j0 + j][c] + part[j][c];
      }
    }
  }
  __syncthreads();  // the tiles' place may be written again
  // the groups' parts of each row, in their order
  float* join = ring;  // [KW - 1][RW][D / 2 + 4][32]
  if (kw > 0 && !idle) {
    float* at = join + ((kw - 1) * RW + warp) * (D / 2 + 4) * 32 + lane;
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) at[(4 * j + c) * 32] = acc[j][c];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      at[(D / 2 + a) * 32] = m[a];
      at[(D / 2 + 2 + a) * 32] = l[a];
    }
  }
  __syncthreads();
  if (kw > 0 || idle) return;
#pragma unroll 1
  for (int k = 0; k < KW - 1; ++k) {
    const float* at = join + (k * RW + warp) * (D / 2 + 4) * 32 + lane;
    float w0[2], w1[2];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const float mo = at[(D / 2 + a) * 32], mt = fmaxf(m[a], mo), base = mt == ninf ? 0.0f : mt;
      w0[a] = ex2(m[a] - base);
      w1[a] = ex2(mo - base);
      l[a] = l[a] * w0[a] + at[(D / 2 + 2 + a) * 32] * w1[a];
      m[a] = mt;
    }
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[j][c] = acc[j][c] * w0[c >> 1] + at[(4 * j + c) * 32] * w1[c >> 1];
  }
  if (s_fix) {  // rare: what was cleared from V, to the rows that see it
    for (int key = k0; key < k1; ++key) {
      const bool v0 = sees(0, key), v1 = sees(1, key);
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float y = load_f<XT>(vb, (int64_t)key * D + 8 * j + 2 * t + c);
          if (odd_f32(__float_as_uint(y))) {
            if (v0) acc[j][c] += y;
            if (v1) acc[j][2 + c] += y;
          }
        }
    }
  }
  const bool alone = tree_splits_used(rg.lo, rg.hi, kMmaKeys, p.NS) <= 1;
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    const int r = r0 + warp * 16 + g + 8 * a;
    if (r >= rows) continue;
    const int i = (int)((uint64_t)(unsigned)r * per_g >> 32), qg = r - i * p.G;
    const int64_t o = (((int64_t)b * p.N + i) * p.H + h * p.G + qg) * D, R = ((int64_t)b * p.Hkv + h) * rows + r;
    if (mine[a] == 0) {  // padding, whatever it met in tiles that the others see whole
      m[a] = ninf;
      l[a] = 0.0f;
    }
    const bool none = m[a] == ninf && l[a] == 0.0f;  // sees nothing; NaN scores stay NaN
    const float inv = none ? 0.0f : 1.0f / l[a];
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      const float x0 = acc[j][2 * a], x1 = acc[j][2 * a + 1];
      const int d = 8 * j + 2 * t;
      if (!alone) {
        *reinterpret_cast<float2*>(p.ws_acc + (R * p.NS + sp) * D + d) = make_float2(x0, x1);
      } else {
        store_f<XT>(p.out, o + d, none ? 0.0f : x0 * inv);
        store_f<XT>(p.out, o + d + 1, none ? 0.0f : x1 * inv);
      }
    }
    if (!alone && t == 0) {
      p.ws_ml[(R * p.NS + sp) * 2] = m[a];
      p.ws_ml[(R * p.NS + sp) * 2 + 1] = l[a];
    }
  }
}

// Joins the splits of each row: M = max m_j, out = sum e^(m_j - M) acc_j / sum
// e^(m_j - M) l_j, in split order.  A warp per row, its lanes the dimensions;
// the partials were just written and come from L2.  7 us cold for 4 x 272 rows of
// 64 in 12 splits, bound by latency.
template <int XT, int D>
__global__ void __launch_bounds__(256) tree_merge_kernel(TreeAttnParams p, int tile) {
  constexpr int U = D / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = p.N * p.G, hr = blockIdx.x * 8 + warp, b = blockIdx.y;
  pdl_wait();
  pdl_trigger();
  const int64_t len = p.seqlen[b];
  const int cb = p.row_map != nullptr ? p.row_map[b] : b;
  const unsigned long long keep = p.N < 64 ? (1ull << p.N) - 1 : ~0ull;
  unsigned long long used = 0;
  for (int i = lane; i < p.N; i += 32) {
    const unsigned long long mi = p.mask[(int64_t)b * p.N + i] & keep;
    used |= mi | (mi ? 1ull << i : 0ull);
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) used |= __shfl_xor_sync(0xffffffffu, used, o);
  const TreeRange rg = tree_range(p, len, cb, used);
  const int ns = tree_splits_used(rg.lo, rg.hi, tile, p.NS);
  if (hr >= p.Hkv * rows || ns <= 1) return;  // one split wrote its output itself
  const int h = hr / rows, r = hr - h * rows;
  const int64_t R = (int64_t)b * p.Hkv * rows + hr;
  const float ninf = __int_as_float(0xff800000);
  const float* ml = p.ws_ml + R * p.NS * 2;
  const float* ac = p.ws_acc + R * p.NS * D;
  float mj[2], lj[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j = lane + 32 * u;
    mj[u] = j < ns ? __ldcg(ml + 2 * j) : ninf;
    lj[u] = j < ns ? __ldcg(ml + 2 * j + 1) : 0.0f;
  }
  const float M = warp_max(fmaxf(mj[0], mj[1]));
  const float base = M == ninf ? 0.0f : M;
  float wj[2] = {ex2(mj[0] - base), ex2(mj[1] - base)};
  float den = 0.0f, num[U];
#pragma unroll
  for (int u = 0; u < U; ++u) num[u] = 0.0f;
  constexpr int kB = 8;
  for (int j0 = 0; j0 < ns; j0 += kB) {
    float a[kB][U];
#pragma unroll
    for (int i = 0; i < kB; ++i)
      if (j0 + i < ns) {
#pragma unroll
        for (int u = 0; u < U; ++u) a[i][u] = __ldcg(ac + (int64_t)(j0 + i) * D + lane + 32 * u);
      }
#pragma unroll
    for (int i = 0; i < kB; ++i)
      if (j0 + i < ns) {
        const int j = j0 + i;
        const float w = __shfl_sync(0xffffffffu, j < 32 ? wj[0] : wj[1], j & 31);
        const float lw = __shfl_sync(0xffffffffu, j < 32 ? lj[0] : lj[1], j & 31);
        if (w == 0.0f && lw == 0.0f) continue;  // a split that this row sees nothing of
        den = fmaf(w, lw, den);
#pragma unroll
        for (int u = 0; u < U; ++u) num[u] = fmaf(w, a[i][u], num[u]);
      }
  }
  const int i = r / p.G, g = r - i * p.G;
  const int64_t o = (((int64_t)b * p.N + i) * p.H + h * p.G + g) * D;
#pragma unroll
  for (int u = 0; u < U; ++u) store_f<XT>(p.out, o + lane + 32 * u, den == 0.0f ? 0.0f : num[u] / den);
}

// ----------------------------------------------------------------- commit --
// cache[row, :, seqlen + d] <- cache[row, :, seqlen + path[d]] for d < n_path,
// every layer's K and V in one launch.  path rises (path[d] >= d), so one
// thread that walks d upwards with its own 16-byte column may move in place:
// what it overwrites at d it has read already.  Batches of eight loads keep the
// column's reads in flight.  Bound by latency at the sizes of a draft: 48 layers
// of 4 heads of 128, one sequence 2.3 us, 16 with up to 32 nodes 3.9 us for up
// to 10.4 MB (2.7 TB/s); a launch alone takes 1.5.
constexpr int kCommitLayers = 128;

struct CommitParams {
  void* ptr[2 * kCommitLayers];  // K and V of each layer
  const int64_t* seqlen;
  const int32_t* path;
  const int32_t* n_path;
  const int32_t* row_map;
  int32_t* kept;  // [B] rows kept of each sequence, or null
  int* err;
  int64_t sb, sh, sbh;  // cache strides in 16-byte units (batch, KV head); sbh: units per row
  int B, N, Hkv, Bc, T, nptr;
};

__global__ void __launch_bounds__(256) commit_kernel(const __grid_constant__ CommitParams p) {
  __shared__ int s_path[kTreeMaxNodes];
  __shared__ int s_bad;
  const int tid = threadIdx.x, b = blockIdx.y;
  pdl_wait();
  pdl_trigger();
  const int n = p.n_path[b];
  const int64_t s = p.seqlen[b];
  const int cb = p.row_map != nullptr ? p.row_map[b] : b;
  const bool tells = p.kept != nullptr && blockIdx.x == 0 && tid == 0;
  if (tid == 0) s_bad = 0;
  __syncthreads();
  if (n <= 0) {
    if (tells) p.kept[b] = 0;
    return;
  }
  const bool ok = n <= p.N && s >= 0 && s <= p.T && cb >= 0 && cb < p.Bc;
  if (ok && tid < n) {
    const int d = tid, x = p.path[(int64_t)b * p.N + d];
    const int before = d > 0 ? p.path[(int64_t)b * p.N + d - 1] : -1;
    if (x <= before || x >= p.N || s + x >= p.T) s_bad = 1;
    s_path[d] = x;
  }
  __syncthreads();
  const bool bad = !ok || s_bad;  // a path that does not rise or leaves the cache: nothing moves
  if (tells) p.kept[b] = bad ? 0 : n;
  if (bad) {
    if (tid == 0) atomicOr(p.err, kErrFlagBounds);
    return;
  }
  const int64_t cols = (int64_t)p.nptr * p.Hkv * p.sbh;
  for (int64_t c = (int64_t)blockIdx.x * 256 + tid; c < cols; c += (int64_t)gridDim.x * 256) {
    const int64_t lane = c % p.sbh, hl = c / p.sbh;
    uint4* base = static_cast<uint4*>(p.ptr[hl / p.Hkv]) + cb * p.sb + (hl % p.Hkv) * p.sh + s * p.sbh + lane;
    for (int d0 = 0; d0 < n; d0 += 8) {
      uint4 r[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (d0 + e < n && s_path[d0 + e] != d0 + e) r[e] = base[s_path[d0 + e] * p.sbh];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (d0 + e < n && s_path[d0 + e] != d0 + e) base[(d0 + e) * p.sbh] = r[e];
    }
  }
}

// How many splits a row's keys are cut into: as many as the resident CTAs
// (two or one per SM) take at once, no more than the join can hold.
inline int tree_mma_splits(int64_t ctas, int64_t max_len, int64_t head_dim) {
  const int64_t want = (head_dim == 256 ? 1 : 2) * 148 / ctas, most = (max_len + kMmaKeys - 1) / kMmaKeys;
  const int64_t ns = want < most ? want : most;
  return (int)(ns < 1 ? 1 : ns > kTreeMaxSplits ? kTreeMaxSplits : ns);
}
// Rows per CTA: 32 with four groups of warps on a tile's keys, or 64 with two.
// Four rows, 16 x 1500 fp32 with heads of 128: 72 us with 32, 105 with 64; more
// rows than 32 would read each key again: 512 rows, 8 x 4000, 1219 us and 975.
inline int tree_mma_rows(int64_t rows) { return rows <= 32 ? 32 : 64; }

inline bool tree_use_tc(int x_dtype, int64_t head_dim) {
  return x_dtype == kBF16 && (head_dim == 64 || head_dim == 128);
}

inline int tree_splits(int64_t batch, int64_t nodes, int64_t num_heads, int64_t num_kv_heads, int64_t max_len,
                       int x_dtype, int64_t head_dim, int64_t window, bool* join) {
  *join = false;
  if (window > 0 && window < max_len - nodes) max_len = window + nodes;  // no row's keys span more
  const int64_t rows = nodes * (num_heads / num_kv_heads);
  if (tree_use_tc(x_dtype, head_dim))
    return tree_tc_splits(batch * num_kv_heads * tree_tc_groups(rows), max_len, rows > tree_tc_partial_rows(1), join);
  const int64_t per = tree_mma_rows(rows), tiles = (rows + per - 1) / per;
  return tree_mma_splits(batch * num_kv_heads * tiles, max_len, head_dim);
}

// Rows of partials per split and KV head, and the bytes of all of them.
inline int64_t tree_partial_rows(int64_t rows, int x_dtype, int64_t head_dim) {
  return tree_use_tc(x_dtype, head_dim) ? tree_tc_partial_rows(rows) : rows;
}
inline int64_t tree_partial_bytes(int64_t batch, int64_t num_kv_heads, int64_t rows, int64_t ns, bool join,
                                  int64_t head_dim) {
  return ns <= 1 || join ? 0 : batch * num_kv_heads * rows * ns * (head_dim + 2) * 4;
}

}  // namespace mb

using namespace mb;

extern "C" int maple_narrow_int64(const int64_t* x, int64_t n, int32_t* out, void* stream) {
  if (n < 0) return kErrShape;
  if (n == 0) return kOk;
  if (!x || !out) return kErrShape;
  const int64_t blocks = (n + 255) / 256;
  const cudaError_t e = launch_k(narrow_kernel, dim3((unsigned)(blocks < 592 ? blocks : 592)), dim3(256), 0,
                                 static_cast<cudaStream_t>(stream), x, n, out);
  return e == cudaSuccess ? kOk : kErrCuda;
}

extern "C" int maple_tree_plan(const int32_t* parents, int64_t batch, int64_t nodes, int64_t p_sb, int64_t p_sn,
                               int64_t* mask, int32_t* depth, int* err, void* stream) {
  if (batch < 0 || nodes <= 0 || nodes > kTreeMaxNodes || batch > (1LL << 30)) return kErrShape;
  if (batch == 0) return kOk;
  if (!parents || !mask || !depth || !err) return kErrShape;
  const cudaError_t e = launch_k(tree_plan_kernel, dim3((unsigned)((batch + 3) / 4)), dim3(128), 0,
                                 static_cast<cudaStream_t>(stream), parents, p_sb, p_sn, (int)batch, (int)nodes,
                                 reinterpret_cast<unsigned long long*>(mask), depth, err);
  return e == cudaSuccess ? kOk : kErrCuda;
}

extern "C" int64_t maple_tree_gqa_workspace_bytes(int64_t batch, int64_t nodes, int64_t num_heads,
                                                  int64_t num_kv_heads, int64_t head_dim, int64_t max_len,
                                                  int64_t window, int x_dtype) {
  if (batch <= 0 || nodes <= 0 || nodes > kTreeMaxNodes || num_heads <= 0 || num_kv_heads <= 0 ||
      num_heads % num_kv_heads || num_heads / num_kv_heads > kTreeMaxGroup || head_dim <= 0 || max_len <= 0 || window < 0)
    return -1;
  bool join;
  const int64_t ns = tree_splits(batch, nodes, num_heads, num_kv_heads, max_len, x_dtype, head_dim, window, &join);
  const int64_t rows = tree_partial_rows(nodes * (num_heads / num_kv_heads), x_dtype, head_dim);
  return tree_partial_bytes(batch, num_kv_heads, rows, ns, join, head_dim);
}

extern "C" int maple_tree_gqa_attn(const void* q, int x_dtype, int64_t batch, int64_t nodes, int64_t num_heads,
                                   int64_t q_sb, int64_t q_sn, int64_t q_sh, const void* k_cache, const void* v_cache,
                                   int64_t cache_batch, int64_t num_kv_heads, int64_t cache_sb, int64_t cache_sh,
                                   int64_t max_len, int64_t head_dim, const int64_t* seqlen, const int64_t* tree_mask,
                                   const int32_t* row_map, float scale, int64_t window, void* out, void* workspace,
                                   int64_t workspace_bytes, int* err, void* stream) {
  if (batch < 0 || nodes <= 0 || nodes > kTreeMaxNodes || num_heads <= 0 || num_kv_heads <= 0 || max_len <= 0 ||
      cache_batch < 0 || window < 0 || !(scale * 2.0f - scale * 2.0f == 0.0f))  // also as powers of 2
    return kErrShape;
  if (batch == 0) return kOk;
  if (x_dtype != kF32 && x_dtype != kBF16) return kErrDtype;
  if (num_heads % num_kv_heads != 0 || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return kErrShape;
  if (num_heads / num_kv_heads > kTreeMaxGroup) return kErrShape;
  if (!q || !k_cache || !v_cache || !seqlen || !tree_mask || !out || !err || batch > 65535 || cache_batch < 1 ||
      num_heads > 65535 || max_len > (1LL << 30) || cache_batch > (1LL << 30))
    return kErrShape;
  const int es = x_dtype == kBF16 ? 2 : 4;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
        reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15) ||
      (((q_sb | q_sn | q_sh | cache_sb | cache_sh) * es) & 15))
    return kErrAlign;
  TreeAttnParams p{};
  p.q = q; p.kc = k_cache; p.vc = v_cache; p.seqlen = seqlen; p.row_map = row_map; p.out = out; p.err = err;
  p.mask = reinterpret_cast<const unsigned long long*>(tree_mask);
  p.q_sb = q_sb; p.q_sn = q_sn; p.q_sh = q_sh; p.c_sb = cache_sb; p.c_sh = cache_sh;
  p.B = (int)batch; p.N = (int)nodes; p.H = (int)num_heads; p.Hkv = (int)num_kv_heads;
  p.G = (int)(num_heads / num_kv_heads); p.Bc = (int)cache_batch; p.T = (int)max_len;
  p.window = (int)(window > max_len ? 0 : window);  // a window past the cache hides nothing
  p.scale = scale;
  const int64_t rows = (int64_t)p.N * p.G, per = tree_mma_rows(rows), tiles = (rows + per - 1) / per;
  if (num_kv_heads * tiles > 65535) return kErrShape;
  bool join;
  p.NS = tree_splits(batch, nodes, num_heads, num_kv_heads, max_len, x_dtype, head_dim, window, &join);
  p.join = join;
  const int64_t prows = tree_partial_rows(rows, x_dtype, head_dim);
  const int64_t need = tree_partial_bytes(batch, num_kv_heads, prows, p.NS, join, head_dim);
  if (need > 0 && (!workspace || workspace_bytes < need)) return kErrWorkspace;
  p.ws_acc = static_cast<float*>(workspace);
  p.ws_ml = p.ws_acc ? p.ws_acc + batch * num_kv_heads * prows * p.NS * head_dim : nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
#define MB_TREE_MMA(XT, DD, RW)                                                                             \
  do {                                                                                                      \
    const size_t smem = (size_t)(16 * RW + 4 * kMmaKeys) * (DD + 4) * 4;                                     \
    static std::atomic<uint64_t> done{0};                                                                   \
    e = smem_once(done, tree_mma_kernel<XT, DD, RW>, (int)smem);                                            \
    if (e == cudaSuccess)                                                                                   \
      e = launch_k(tree_mma_kernel<XT, DD, RW>,                                                             \
                   dim3((unsigned)p.NS, (unsigned)(num_kv_heads * tiles), (unsigned)batch), dim3(kMmaThreads), \
                   smem, st, p, (int)tiles);                                                                \
  } while (0)
#define MB_TREE(XT, DD)                                                                                              \
  do {                                                                                                               \
    if (per == 32) MB_TREE_MMA(XT, DD, 2); else MB_TREE_MMA(XT, DD, 4);                                              \
    if (e == cudaSuccess && p.NS > 1)                                                                                \
      e = launch_k(tree_merge_kernel<XT, DD>,                                                                        \
                   dim3((unsigned)((num_kv_heads * rows + 7) / 8), (unsigned)batch), dim3(256), 0, st, p, kMmaKeys); \
  } while (0)
  if (tree_use_tc(x_dtype, head_dim)) {
    if (batch * num_kv_heads * p.NS * tree_tc_groups(rows) > (1LL << 30)) return kErrShape;
    e = tree_tc_launch(p, (int)head_dim, st);
  } else if (x_dtype == kBF16) {
    MB_TREE(kBF16, 256);
  } else {
    if (head_dim == 64) MB_TREE(kF32, 64); else if (head_dim == 128) MB_TREE(kF32, 128); else MB_TREE(kF32, 256);
  }
#undef MB_TREE
#undef MB_TREE_MMA
  return e == cudaSuccess ? kOk : kErrCuda;
}

extern "C" int maple_commit_tree_kept(void* const* k_caches, void* const* v_caches, int64_t layers, int x_dtype,
                                      int64_t batch, int64_t nodes, int64_t cache_batch, int64_t num_kv_heads,
                                      int64_t cache_sb, int64_t cache_sh, int64_t max_len, int64_t head_dim,
                                      const int64_t* seqlen, const int32_t* path, const int32_t* n_path,
                                      const int32_t* row_map, int32_t* kept, int* err, void* stream) {
  if (layers < 0 || batch < 0 || nodes <= 0 || nodes > kTreeMaxNodes || num_kv_heads <= 0 || max_len <= 0 ||
      head_dim <= 0 || batch > 65535 || cache_batch < 0 || cache_batch > (1LL << 30) || max_len > (1LL << 30))
    return kErrShape;
  if (layers == 0 || batch == 0) return kOk;
  if (x_dtype != kF32 && x_dtype != kBF16) return kErrDtype;
  if (!k_caches || !v_caches || !seqlen || !path || !n_path || !err || cache_batch < 1) return kErrShape;
  if ((num_kv_heads > 1 && cache_sh == 0) || (cache_batch > 1 && cache_sb == 0)) return kErrShape;  // shared rows
  const int64_t epu = x_dtype == kBF16 ? 8 : 4;  // elements per 16 bytes
  if (head_dim % epu || cache_sb % epu || cache_sh % epu) return kErrAlign;
  for (int64_t i = 0; i < layers; ++i) {
    if (!k_caches[i] || !v_caches[i]) return kErrShape;
    if ((reinterpret_cast<uintptr_t>(k_caches[i]) | reinterpret_cast<uintptr_t>(v_caches[i])) & 15) return kErrAlign;
  }
  for (int64_t l0 = 0; l0 < layers; l0 += kCommitLayers) {
    const int64_t nl = layers - l0 < kCommitLayers ? layers - l0 : kCommitLayers;
    CommitParams p{};
    for (int64_t i = 0; i < nl; ++i) {
      p.ptr[2 * i] = k_caches[l0 + i];
      p.ptr[2 * i + 1] = v_caches[l0 + i];
    }
    p.seqlen = seqlen; p.path = path; p.n_path = n_path; p.row_map = row_map; p.err = err;
    p.kept = l0 == 0 ? kept : nullptr;  // the same for all layers
    p.sb = cache_sb / epu; p.sh = cache_sh / epu; p.sbh = head_dim / epu;
    p.B = (int)batch; p.N = (int)nodes; p.Hkv = (int)num_kv_heads; p.Bc = (int)cache_batch; p.T = (int)max_len;
    p.nptr = (int)(2 * nl);
    const int64_t cols = (int64_t)p.nptr * num_kv_heads * p.sbh, blocks = (cols + 255) / 256;
    const cudaError_t e = launch_k(commit_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024), (unsigned)batch),
                                   dim3(256), 0, static_cast<cudaStream_t>(stream), p);
    if (e != cudaSuccess) return kErrCuda;
  }
  return kOk;
}

extern "C" int maple_commit_tree(void* const* k_caches, void* const* v_caches, int64_t layers, int x_dtype,
                                 int64_t batch, int64_t nodes, int64_t cache_batch, int64_t num_kv_heads,
                                 int64_t cache_sb, int64_t cache_sh, int64_t max_len, int64_t head_dim,
                                 const int64_t* seqlen, const int32_t* path, const int32_t* n_path,
                                 const int32_t* row_map, int* err, void* stream) {
  return maple_commit_tree_kept(k_caches, v_caches, layers, x_dtype, batch, nodes, cache_batch, num_kv_heads, cache_sb,
                                cache_sh, max_len, head_dim, seqlen, path, n_path, row_map, nullptr, err, stream);
}
