// Attention over a KV cache for trees of drafted tokens on the 5th-generation
// tensor cores (bf16 caches, heads of 64 or 128).
//
// The rows of a KV head are (node, query head of the group) pairs, row r =
// node r / G, head r % G, in tiles of 128 = the MMA's M; a tile of 128 keys is
// its N.  Per key tile S = Q K^T (K-major operands from 128-byte-swizzled
// shared memory), softmax in registers, then O += P V with P as bf16 in tensor
// memory (over the scores it came from) and V read as stored, [keys][dims], an
// MN-major operand.  Each K/V row crosses HBM once per 256 rows.
//
// Roles (384 threads, one CTA per SM, persistent over work items): warp 9
// works the items out and streams K and V tiles by TMA into two rings; warp 8
// issues the MMAs; two warpgroups of four warps do the softmax, a thread per
// row.  Up to 128 rows (PAIR = false) both warpgroups share the row tile and
// take alternate key tiles, each with its own scores, output, maximum and sum,
// joined at the item's end; more rows (PAIR = true) give each its own row tile.
// Either way one's softmax runs under the other's MMAs.  A unit = one key tile
// of one warpgroup; the tensor pipe runs S(0) S(1) O(0) S(2) O(1) S(3) ..., so
// a unit's scores overwrite its predecessor's weights right behind the product
// that read them.  Because scores are committed behind that product, a
// warpgroup that sees them knows its output is at rest, and may rescale it;
// it does so only when a row's maximum has grown by more than 2^8.  The weights
// are relative to 2^8 times the maximum of the last time, so that they are at
// most 1, as are their products with V at most V: fp32 holds these for any V.
//
// An item is one split of one sequence's keys for one KV head and row tile (or
// pair).  With JOIN a CTA has one item, and the splits of a row tile form a
// cluster, which joins their parts through its shared memory.  A tile that some
// row sees only in part is masked in registers; its V tile is cleared of NaN and
// infinities in shared memory first (0 x NaN is NaN), and where a visible one was
// cleared the item's end adds it back to the rows that see it.
//
// Up to 128 rows HBM bounds it: 64 sequences x 8150 with eight nodes (32 heads
// on 4 of 128), 1.08 GB in 164 us = 6.57 TB/s, what a plain copy reaches; held
// for seconds the power limit makes it 181.  With more rows the chain of a unit
// does (scores, loads from tensor memory, exponentials, stores, product), of
// which two run in turn: 64 nodes x 65440, 68.7 GFLOP in 72 us = 950 TFLOP/s; at
// 1 x 32768 the exponential unit is busy 45 % of the time, the tensor pipe 44 %,
// the issue slots 32 %, so that no unit is full.  Exponentials by a polynomial on the FMA pipes gave 280 to 316 us for 273 (37 x 8192, 64 nodes),
// units of 64 keys with their scores a unit ahead 320.
//
// Waits are bounded: one that gives up sets the error word; every role then
// leaves, waits (bounded) for its copies and MMAs in flight, frees the tensor
// memory and returns.  Loads read this GPU's own memory, without multicast.
#include <cooperative_groups.h>

#include "bulk.cuh"
#include "launch.cuh"
#include "tcgen05.cuh"
#include "tmap.cuh"
#include "tree.cuh"

namespace mb {

namespace cg = cooperative_groups;

constexpr int kTtKeys = 128;   // keys per tile: MMA N of the scores, K of the output
constexpr int kTtRows = 128;   // rows per tile: MMA M
constexpr int kTtThreads = 384;
constexpr int kTtInfo = 2;     // items known ahead
constexpr int kTtCluster = 8;  // splits that a cluster joins (the portable size)
constexpr float kTtGrow = 8.0f;  // log2 growth of a row's maximum that rescales, and what weights leave for it

struct TtItem {
  int b, h, rt, sp;     // sequence, KV head, row tile (pair), split
  int s, k0, k1;        // cached positions, this split's keys
  int item, tiles, used, fix, dmax;  // key tiles; splits that hold keys; V was cleared; largest depth
  unsigned long long mask[kTreeMaxNodes];
};

template <int D, bool PAIR>
struct TtShape {
  static constexpr int kTile = kTtKeys * D * 2;              // one K, V or Q tile
  static constexpr int kQ = PAIR ? 2 : 1;
  static constexpr int NK = D == 128 ? 3 : 4;                // ring depths
  static constexpr int NV = D == 128 ? (PAIR ? 2 : 3) : 4;
  static constexpr int kTiles = (kQ + NK + NV) * kTile;
  static constexpr int kSmem = kTiles + kTtInfo * (int)sizeof(TtItem) + 288;
};

__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Not zero where either half is a NaN or an infinity (exponent bits all set).
__device__ __forceinline__ uint32_t odd_bf16x2(uint32_t w) { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A barrier among warps on an mbarrier (one arrival per warp), so that a warp
// that gave up cannot leave the others waiting for good.
__device__ __forceinline__ bool tt_sync(uint64_t* bar, int& count, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
  const bool ok = mbar_wait_bounded(bar, (unsigned)(count & 1));
  ++count;
  return __all_sync(0xffffffffu, ok);
}

// Whether some row of the item misses a key of the tile at t0: it reaches into
// the tree, past the split's end, or before a window.
__device__ __forceinline__ bool tt_mixed(const TtItem& it, int t0, int window) {
  return t0 + kTtKeys > min(it.s, it.k1) || (window > 0 && t0 <= it.s + it.dmax - window);
}

// This row's view of a tile as 128 bits: cached positions past the window's
// start, and its nodes' bits.
struct TtView {
  unsigned long long nodes;  // nodes seen, the window applied
  int first;                 // first cached position seen
  bool real;
};
// Columns 32 q .. 32 q + 31 of the tile at t0, one bit each.
__device__ __forceinline__ uint32_t tt_low(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }
__device__ __forceinline__ uint32_t tt_bits(const TtView& v, int s, int k1, int t0, int q) {
  const int t = t0 + 32 * q;
  const int sh = t - s;  // node of bit 0
  uint32_t nb = 0;
  if (sh >= 0 && sh < 64) nb = (uint32_t)(v.nodes >> sh);
  else if (sh < 0 && sh > -32) nb = (uint32_t)(v.nodes << -sh);
  const uint32_t cached = tt_low(s - t) & ~tt_low(v.first - t);
  return v.real ? (cached | nb) & tt_low(k1 - t) : 0u;  // past the split's end: the next split's
}

// A cluster's join, one split per CTA: M = max m_j, out = sum 2^(m_j - M) acc_j
// / sum 2^(m_j - M) l_j in split order.  The warps of the CTAs with keys each
// take 32 rows, whose weights they form once, and every so many blocks of four
// dims of them: loads from the other CTAs take some 0.5 us, so few may wait on
// one another.
template <int D, bool PAIR>
__device__ __forceinline__ void tt_join(const TreeAttnParams& p, const TtItem& it, float* part, float2* part_ml, int warp,
                                        int lane) {
  const cg::cluster_group cluster = cg::this_cluster();
  constexpr int R = PAIR ? 2 * kTtRows : kTtRows;
  const float ninf = __int_as_float(0xff800000);
  const int used = it.used, first = it.rt * R, rows = min(p.N * p.G - first, R);
  const int blocks = (rows + 31) / 32, at = it.sp * 8 + warp;  // at most 8 blocks for 16 warps or more
  const int row = at % blocks * 32 + lane, step = (used * 8 - at % blocks + blocks - 1) / blocks;
  if (row >= rows) return;
  float w[kTtCluster], M = ninf, den = 0.0f;
  {
    float2 y[kTtCluster];
#pragma unroll
    for (int j = 0; j < kTtCluster; ++j) {
      y[j] = j < used ? cluster.map_shared_rank(part_ml, j)[row] : make_float2(ninf, 0.0f);
      M = fmaxf(M, y[j].x);
    }
    const float base = M == ninf ? 0.0f : M;
#pragma unroll
    for (int j = 0; j < kTtCluster; ++j) {  // none for a split that this row sees nothing of; NaN scores stay NaN
      w[j] = y[j].x == ninf && y[j].y == 0.0f ? 0.0f : ex2(y[j].x - base);
      if (w[j] != 0.0f || y[j].y != 0.0f) den = fmaf(w[j], y[j].y, den);
    }
  }
  const float inv = den == 0.0f ? 0.0f : 1.0f / den;
  const int node = (first + row) / p.G, g = first + row - node * p.G;
  uint16_t* out = static_cast<uint16_t*>(p.out) + (((int64_t)it.b * p.N + node) * p.H + it.h * p.G + g) * D;
  const int src = row / kTtRows * D * kTtRows + row % kTtRows;
#pragma unroll 2
  for (int col = at / blocks * 4; col < D; col += step * 4) {
    float num[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < kTtCluster; ++j) {
      if (j < used) {
        const float* a = cluster.map_shared_rank(part, j) + src + col * kTtRows;
#pragma unroll
        for (int i = 0; i < 4; ++i) num[i] = fmaf(w[j], a[i * kTtRows], num[i]);
      }
    }
    *reinterpret_cast<uint2*>(out + col) = den == 0.0f ? make_uint2(0u, 0u) : make_uint2(bf16x2(num[0] * inv, num[1] * inv),
                                                                                         bf16x2(num[2] * inv, num[3] * inv));
  }
}

template <int D, bool PAIR, bool JOIN>
__global__ void __launch_bounds__(kTtThreads, 1)
    tree_tc_kernel(TreeAttnParams p, int row_groups, int items, const __grid_constant__ CUtensorMap tmk,
                   const __grid_constant__ CUtensorMap tmv) {
  using Sh = TtShape<D, PAIR>;
  constexpr int TILE = Sh::kTile, NK = Sh::NK, NV = Sh::NV, HALVES = D / 64, BOX = kTtKeys * 128;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* sq = smem;
  unsigned char* sk = sq + Sh::kQ * TILE;
  unsigned char* sv = sk + NK * TILE;
  TtItem* info = reinterpret_cast<TtItem*>(sv + NV * TILE);
  float2* s_ml = reinterpret_cast<float2*>(sq);  // [2][128] maximum and sum, once the queries are done with
  // JOIN: this split's part for the cluster, once the tiles are done with: [dim][128] per row tile, [row]
  float* s_part = reinterpret_cast<float*>(sk);
  float2* s_part_ml = s_ml + 2 * kTtRows;
  static_assert(Sh::kQ * kTtRows * D * 4 <= (NK + NV) * TILE && (2 + Sh::kQ) * kTtRows * 8 <= TILE, "parts in the tiles' place");
  uint64_t* bars = reinterpret_cast<uint64_t*>(info + kTtInfo);
  uint64_t *kfull = bars, *kempty = kfull + NK, *vfull = kempty + NK, *vempty = vfull + NV, *sfull = vempty + NV,
           *phalf = sfull + 2, *pready = phalf + 2, *ofull = pready + 2, *oempty = ofull + 2, *qfull = oempty + 1, *ifull = qfull + 1,
           *iempty = ifull + kTtInfo, *both = iempty + kTtInfo, *each = both + 1, *drain = each + 2;
  unsigned* s_tmem = reinterpret_cast<unsigned*>(drain + 1);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (warp == 8) tmem_alloc(s_tmem, 512);
  if (tid == 0) {
    for (int i = 0; i < NK; ++i) { mbar_init(&kfull[i], 1); mbar_init(&kempty[i], 1); }
    for (int i = 0; i < NV; ++i) { mbar_init(&vfull[i], 1); mbar_init(&vempty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&sfull[i], 1); mbar_init(&phalf[i], 4); mbar_init(&pready[i], 4); mbar_init(&ofull[i], 1); }
    mbar_init(oempty, 8);
    mbar_init(qfull, 8);
    for (int i = 0; i < kTtInfo; ++i) { mbar_init(&ifull[i], 1); mbar_init(&iempty[i], 9); }
    mbar_init(both, 8);
    for (int i = 0; i < 2; ++i) mbar_init(&each[i], 4);
    mbar_init(drain, 1);
    if (JOIN) info[0].tiles = -1;  // stays where this split has no keys
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = *s_tmem;
  pdl_wait();
  pdl_trigger();
  bool ok = (smem_u32(smem) & 1023u) == 0;  // the swizzled tiles need it; the launch gives it

  // 384 threads launch with 168 registers each (64512): 2 x 128 x 208 + 128 x 80 = 63488 of them
  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 80;\n");
  if (warp == 9) {
    // -------------------------------------------------- items, K and V tiles --
    const unsigned long long keep = p.N < 64 ? (1ull << p.N) - 1 : ~0ull;
    int n_items = 0, kt_all = 0;
    for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
      // a cluster's CTAs lie side by side: the splits of one row tile
      const int rt = JOIN ? item / p.NS % row_groups : item % row_groups;
      const int sp = JOIN ? item % p.NS : item / row_groups % p.NS, bh = item / row_groups / p.NS;
      const int h = bh % p.Hkv, b = bh / p.Hkv;
      const int64_t len = p.seqlen[b];
      const int cb = p.row_map != nullptr ? p.row_map[b] : b;
      unsigned long long m[2], used = 0;
      int dm = 0;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int i = lane + 32 * u;
        m[u] = i < p.N ? p.mask[(int64_t)b * p.N + i] & keep : 0ull;
        used |= m[u] | (m[u] ? 1ull << i : 0ull);
        dm = max(dm, __popcll(m[u]) - 1);
      }
      const unsigned ul = __reduce_or_sync(0xffffffffu, (unsigned)used);
      const unsigned uh = __reduce_or_sync(0xffffffffu, (unsigned)(used >> 32));
      dm = __reduce_max_sync(0xffffffffu, dm);
      const TreeRange rg = tree_range(p, len, cb, ((unsigned long long)uh << 32) | ul);
      if (rg.bad && lane == 0) atomicOr(p.err, kErrFlagBounds);
      const int mh = p.c_sh ? h : 0, mb = p.c_sb ? rg.cb : 0;  // a stride of 0 is a map of one
      int k0, k1;
      tree_split(rg.lo, rg.hi, kTtKeys, p.NS, sp, k0, k1);
      if (sp > 0 && k0 >= k1) continue;  // nothing here; split 0 always answers
      const int tiles = (k1 - k0 + kTtKeys - 1) / kTtKeys, slot = n_items % kTtInfo, use = n_items / kTtInfo;
      if (use > 0) ok = mbar_wait_bounded(&iempty[slot], (unsigned)((use - 1) & 1));
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      TtItem& it = info[slot];
      it.mask[lane] = m[0];
      it.mask[lane + 32] = m[1];
      if (lane == 0) {
        it.item = item; it.b = b; it.h = h; it.rt = rt; it.sp = sp;
        it.s = rg.s; it.k0 = k0; it.k1 = k1; it.tiles = tiles; it.fix = 0; it.dmax = dm;
        it.used = tree_splits_used(rg.lo, rg.hi, kTtKeys, p.NS);
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&ifull[slot]);
        // K runs ahead of V by one tile (two where the warpgroups take turns), as the MMAs use them
        constexpr int AHEAD = PAIR ? 1 : 2;
        for (int c = 0; c < tiles + AHEAD && ok; ++c) {
          if (c < tiles) {
            const int g = kt_all + c, st = g % NK;
            if (g >= NK) ok = mbar_wait_bounded(&kempty[st], (unsigned)((g / NK - 1) & 1));
            if (!ok) break;
            mbar_expect_tx(&kfull[st], (unsigned)TILE);
#pragma unroll
            for (int hf = 0; hf < HALVES; ++hf)
              tma_load_4d(sk + st * TILE + hf * BOX, &tmk, 64 * hf, k0 + c * kTtKeys, mh, mb, &kfull[st]);
          }
          if (c >= AHEAD) {
            const int g = kt_all + c - AHEAD, st = g % NV;
            if (g >= NV) ok = mbar_wait_bounded(&vempty[st], (unsigned)((g / NV - 1) & 1));
            if (!ok) break;
            mbar_expect_tx(&vfull[st], (unsigned)TILE);
#pragma unroll
            for (int hf = 0; hf < HALVES; ++hf)
              tma_load_4d(sv + st * TILE + hf * BOX, &tmv, 64 * hf, k0 + (c - AHEAD) * kTtKeys, mh, mb, &vfull[st]);
          }
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      kt_all += tiles;
      ++n_items;
    }
    if (ok) {  // the end
      const int slot = n_items % kTtInfo, use = n_items / kTtInfo;
      if (use > 0) ok = mbar_wait_bounded(&iempty[slot], (unsigned)((use - 1) & 1));
      if (ok && lane == 0) {
        info[slot].tiles = -1;
        mbar_arrive(&ifull[slot]);
      }
    }
    if (lane == 0) {
      if (!ok) atomicOr(p.err, kErrFlagTimeout);
      // copies in flight land before the CTA's memory is given up: no use for the ones that were consumed
      for (int i = 0; i < NK; ++i)
        if (kt_all > i) mbar_wait_bounded(&kfull[i], (unsigned)(((kt_all - 1 - i) / NK) & 1));
      for (int i = 0; i < NV; ++i)
        if (kt_all > i) mbar_wait_bounded(&vfull[i], (unsigned)(((kt_all - 1 - i) / NV) & 1));
    }
    __syncwarp();
  } else if (warp == 8) {
    // --------------------------------------------------------------- MMAs --
    // The whole warp walks the units and one elected lane issues: with values
    // that are the same in all lanes the descriptors stay in uniform registers
    // (built per lane, each MMA waited some 50 cycles for its operands' move).
    constexpr unsigned id_s = umma_idesc_bf16(kTtRows, kTtKeys, false), id_o = umma_idesc_bf16(kTtRows, D, true);
    const uint64_t dq = umma_desc_sw128(smem_u32(sq)), dk = umma_desc_sw128(smem_u32(sk)),
                   dv = umma_desc_sw128_mn(smem_u32(sv), BOX);
    int work = 0, ks = 0, kp = 0, vs = 0, vp = 0, pp[2] = {0, 0};  // ring stages and phases
    for (int n = 0; ok; ++n) {
      const int slot = n % kTtInfo;
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ifull[slot], (unsigned)((n / kTtInfo) & 1)));
      if (!ok) break;
      const int tiles = __shfl_sync(0xffffffffu, info[slot].tiles, 0);
      __syncwarp();
      if (elect_one()) mbar_arrive(&iempty[slot]);
      if (tiles < 0) break;
      if (tiles == 0) continue;
      const int units = PAIR ? 2 * tiles : tiles;
      auto scores = [&](int w) {
        if (!PAIR || w == 0) ok = __all_sync(0xffffffffu, mbar_wait_bounded(&kfull[ks], (unsigned)kp));
        if (!ok) return;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t a = dq + (unsigned)((PAIR ? w : 0) * (TILE >> 4)), k = dk + (unsigned)(ks * (TILE >> 4));
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const unsigned o = ((kk >> 2) * BOX + (kk & 3) * 32) >> 4;
            umma_bf16(tmem + w * kTtKeys, a + o, k + o, id_s, kk > 0);
          }
          umma_commit(&sfull[w]);
          if (!PAIR || w == 1) umma_commit(&kempty[ks]);
        }
        __syncwarp();
        if (!PAIR || w == 1) {
          if (++ks == NK) { ks = 0; kp ^= 1; }
        }
      };
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(qfull, (unsigned)(work & 1)));
      if (ok) scores(0);
      if (ok && units > 1) scores(1);
      // the item before has read its output
      if (ok && work > 0) ok = __all_sync(0xffffffffu, mbar_wait_bounded(oempty, (unsigned)((work - 1) & 1)));
      auto step = [&](int u, int w) {
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&phalf[w], (unsigned)pp[w]));
        if (ok && (!PAIR || w == 0)) ok = __all_sync(0xffffffffu, mbar_wait_bounded(&vfull[vs], (unsigned)vp));
        if (!ok) return;
        const uint64_t v = dv + (unsigned)(vs * (TILE >> 4));
        auto half = [&](int k0) {
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < kTtKeys / 32; ++k) {
              const int kk = k0 + k;
              umma_bf16_ta(tmem + 2 * kTtKeys + w * D, tmem + w * kTtKeys + 8 * kk, v + (unsigned)(128 * kk), id_o,
                           u >= 2 || kk > 0);
            }
          }
          __syncwarp();
        };
        half(0);
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&pready[w], (unsigned)pp[w]));
        pp[w] ^= 1;
        if (!ok) return;
        half(kTtKeys / 32);
        if ((!PAIR || w == 1) && elect_one()) umma_commit(&vempty[vs]);
        __syncwarp();
        if (!PAIR || w == 1) {
          if (++vs == NV) { vs = 0; vp ^= 1; }
        }
        if (u + 2 < units) scores(w);
      };
      for (int u = 0; u < units && ok; u += 2) {
        step(u, 0);
        if (ok && u + 1 < units) step(u + 1, 1);
      }
      if (ok && elect_one()) {
        umma_commit(&ofull[0]);
        umma_commit(&ofull[1]);
      }
      __syncwarp();
      ++work;
    }
    if (elect_one()) {
      if (!ok) atomicOr(p.err, kErrFlagTimeout);
      umma_commit(drain);  // nothing of the tensor pipe is left behind
      mbar_wait_bounded(drain, 0);
    }
    __syncwarp();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;\n");
    // ------------------------------------------------------------ softmax --
    const int w = warp >> 2, r = tid & 127;
    const unsigned lanes = (unsigned)(warp & 3) << 21;  // TMEM lane base of this warp, in bits 31:16
    const unsigned t_s = tmem + lanes + w * kTtKeys, t_o = tmem + lanes + 2 * kTtKeys;
    const float ninf = __int_as_float(0xff800000);
    // above 0, so that a masked score of -inf stays one under scale 0: by the least fp32, 2^-149, which makes
    // no more than 2^-21 of any score
    const float c = fmaxf(fabsf(p.scale) * 1.44269504088896341f, __int_as_float(1));
    const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u;  // the queries carry the scale's sign
    const int rows = p.N * p.G;
    // row / G by a multiplication: exact while row x G < 2^32
    const uint64_t per_g = (1ull << 32) / (unsigned)p.G + 1;
    auto tt_node = [&](int x) { return (int)((uint64_t)(unsigned)x * per_g >> 32); };
    int kbase = 0, work = 0, scount = 0, n_both = 0, n_each = 0;
    constexpr int CH = D / 8, QT = PAIR ? 128 : 256, QN = kTtRows * CH / QT;  // Q's 16-byte chunks per row, per thread
    int guess = (int)blockIdx.x;  // the next item, if it has keys
    for (int n = 0; ok; ++n) {
      // the guessed item's Q rows come near under the wait: they depend on its number alone
      if (guess < items) {
        const int bh = guess / row_groups / p.NS, rt = JOIN ? guess / p.NS % row_groups : guess % row_groups;
        constexpr int LINES = D / 64;  // 128 bytes each
        for (int x = PAIR ? r : tid; x < kTtRows * LINES; x += QT) {
          const int gr = (PAIR ? 2 * rt + w : rt) * kTtRows + x / LINES;
          if (gr < rows) {
            const int i = tt_node(gr), g = gr - i * p.G;
            asm volatile("prefetch.global.L1 [%0];\n" ::"l"(
                static_cast<const char*>(p.q) + (bh / p.Hkv * p.q_sb + i * p.q_sn +
                                                 (int64_t)(bh % p.Hkv * p.G + g) * p.q_sh + x % LINES * 64) * 2));
          }
        }
      }
      const int slot = n % kTtInfo;
      ok = mbar_wait_bounded(&ifull[slot], (unsigned)((n / kTtInfo) & 1));
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      TtItem& it = info[slot];
      const int tiles = it.tiles;
      if (tiles < 0) break;
      const int b = it.b, h = it.h, s = it.s, k0 = it.k0, k1 = it.k1;
      const int row = (PAIR ? 2 * it.rt + w : it.rt) * kTtRows + r;
      const int node = tt_node(row), head = h * p.G + row - node * p.G;
      TtView view{};
      const unsigned long long mine = row < rows ? it.mask[node] : 0ull;
      view.real = mine != 0;
      view.nodes = mine;
      if (p.window > 0) {
        const int first = s + __popcll(mine) - p.window;  // lowest position seen
        view.first = max(0, first);
        for (unsigned long long left = mine; left; left &= left - 1) {
          const int j = __ffsll((long long)left) - 1;
          if (s + __popcll(it.mask[j]) - 1 < first) view.nodes &= ~(1ull << j);
        }
      }
      const int64_t out = (((int64_t)b * p.N + node) * p.H + head) * D;
      float mc = ninf, l = 0.0f;  // what weights are relative to (a maximum times c, and kTtGrow), their sum
      int mine_units = 0;
      if (tiles > 0) {
        // Q, 128-byte swizzled: the warpgroup's own tile, or half of the shared one each
        guess = it.item + (int)gridDim.x;
        uint4 qv[QN];
#pragma unroll
        for (int e = 0; e < QN; ++e) {
          const int x = (PAIR ? r : tid) + e * QT, gr = (PAIR ? 2 * it.rt + w : it.rt) * kTtRows + x / CH;
          qv[e] = make_uint4(0u, 0u, 0u, 0u);
          if (gr < rows) {
            const int i = tt_node(gr), g = gr - i * p.G;
            qv[e] = ld_u4(static_cast<const char*>(p.q) +
                          (b * p.q_sb + i * p.q_sn + (int64_t)(h * p.G + g) * p.q_sh + x % CH * 8) * 2);
          }
        }
        unsigned char* tile = sq + (PAIR ? w : 0) * TILE;
#pragma unroll
        for (int e = 0; e < QN; ++e) {
          const int x = (PAIR ? r : tid) + e * QT, qr = x / CH, cc = x % CH;
          *reinterpret_cast<uint4*>(tile + (cc >> 3) * BOX + qr * 128 + (((cc & 7) ^ (qr & 7)) << 4)) =
              make_uint4(qv[e].x ^ flip, qv[e].y ^ flip, qv[e].z ^ flip, qv[e].w ^ flip);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(qfull);
        const bool idle = __all_sync(0xffffffffu, row >= rows);  // this warp has no row: it only keeps step
        for (int kt = PAIR ? 0 : w; kt < tiles && ok; kt += PAIR ? 1 : 2, ++mine_units) {
          ok = mbar_wait_bounded(&sfull[w], (unsigned)(scount & 1));
          ++scount;
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          tc_fence_after();
          const int t0 = k0 + kt * kTtKeys;
          const bool mixed = tt_mixed(it, t0, p.window);
          if (mixed) {
            // clear the V tile of NaN and infinities before its product
            const int g = kbase + kt, st = g % NV;
            ok = mbar_wait_bounded(&vfull[st], (unsigned)((g / NV) & 1));
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
              uint4* tile = reinterpret_cast<uint4*>(sv + st * TILE) + (PAIR ? tid : r);
              constexpr int STEP = PAIR ? 256 : 128, UNITS = TILE / 16 / STEP;
              uint32_t odd = 0;
#pragma unroll
              for (int x = 0; x < UNITS; ++x) {
                const uint4 v = tile[x * STEP];
                odd |= odd_bf16x2(v.x) | odd_bf16x2(v.y) | odd_bf16x2(v.z) | odd_bf16x2(v.w);
              }
              if (odd) {  // rare
#pragma unroll 1
                for (int x = 0; x < UNITS; ++x) {
                  uint4 v = tile[x * STEP];
                  if (!(odd_bf16x2(v.x) | odd_bf16x2(v.y) | odd_bf16x2(v.z) | odd_bf16x2(v.w))) continue;
                  uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    const uint32_t y = odd_bf16x2(e[i]);
                    e[i] &= ~((y >> 15 & 1u) * 0xffffu | (y >> 31) * 0xffff0000u);
                  }
                  tile[x * STEP] = make_uint4(e[0], e[1], e[2], e[3]);
                  if (t0 + ((PAIR ? tid : r) + x * STEP) % (BOX / 16) / 8 < k1) it.fix = 1;
                }
              }
              fence_proxy_async_smem();
            }
            const bool met = PAIR ? tt_sync(both, n_both, lane) : tt_sync(&each[w], n_each, lane);
            ok = ok && met;
            if (!ok) break;
          }
          if (!idle) {
            // a row's new maximum, and its output and sum brought to it where it has grown enough
            auto settle = [&](float top) {
              const float tc = top * c;
              const bool grow = tc > mc;
              if (!__any_sync(0xffffffffu, grow)) return;
              const float f = grow ? (mc == ninf ? 0.0f : ex2(mc - (tc + kTtGrow))) : 1.0f;
              if (grow) mc = tc + kTtGrow;
              l *= f;
              if (mine_units == 0) return;
#pragma unroll 1
              for (int q = 0; q < D / 32; ++q) {
                uint32_t o[32];
                tmem_ld32(t_o + w * D + 32 * q, o);
                tmem_wait32(o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                tmem_st32(t_o + w * D + 32 * q, o);
              }
            };
            uint32_t x[kTtKeys];
#pragma unroll
            for (int q = 0; q < 4; ++q) tmem_ld32(t_s + 32 * q, x + 32 * q);
            uint32_t bits[4];
            if (mixed) {
#pragma unroll
              for (int q = 0; q < 4; ++q) bits[q] = tt_bits(view, s, k1, t0, q);
            }
            float top[4] = {ninf, ninf, ninf, ninf};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              tmem_wait32(x + 32 * q);
              if (mixed) {
#pragma unroll
                for (int i = 0; i < 32; ++i) x[32 * q + i] = (bits[q] >> i) & 1u ? x[32 * q + i] : 0xff800000u;
              }
#pragma unroll
              for (int i = 0; i < 32; i += 2)
                top[(i >> 1) & 3] = max3(top[(i >> 1) & 3], __uint_as_float(x[32 * q + i]), __uint_as_float(x[32 * q + i + 1]));
            }
            settle(max3(fmaxf(top[0], top[1]), top[2], top[3]));
            const float sub = mc == ninf ? 0.0f : -mc;
            const uint64_t c2 = f2(c, c), sub2 = f2(sub, sub);
            uint64_t sum[2] = {0, 0};
            // the product starts on the first half of the weights while the second is formed
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
              for (int i = 64 * hf; i < 64 * hf + 64; i += 2) {
                const uint64_t y = f2_fma(f2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), c2, sub2);
                float a, e;
                f2_get(y, a, e);
                a = ex2(a);
                e = ex2(e);
                sum[(i >> 1) & 1] = f2_add(sum[(i >> 1) & 1], f2(a, e));
                x[i >> 1] = bf16x2(a, e);
              }
              tmem_st32(t_s + 32 * hf, x + 32 * hf);
              if (hf == 0) {
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&phalf[w]);
              }
            }
            float a, e;
            f2_get(f2_add(sum[0], sum[1]), a, e);
            l += a + e;
            tmem_wait_st();
          } else if (lane == 0) {
            mbar_arrive(&phalf[w]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&pready[w]);
        }
        if (!ok) break;
        // the end: the output of every unit is in
        ok = mbar_wait_bounded(&ofull[w], (unsigned)(work & 1));
        if (!PAIR) ok = mbar_wait_bounded(&ofull[w ^ 1], (unsigned)(work & 1)) && ok;
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc_fence_after();
      }
      float f0 = 1.0f, f1 = 0.0f;  // weights of this warpgroup's output and the other's
      int other_units = 0;
      if (!PAIR && tiles > 0) {
        s_ml[w * kTtRows + r] = make_float2(mc, l);
        ok = tt_sync(both, n_both, lane);
        if (!ok) break;
        const float2 o = s_ml[(w ^ 1) * kTtRows + r];
        other_units = w == 0 ? tiles / 2 : (tiles + 1) / 2;
        const float M = fmaxf(mc, o.x);
        f0 = mc == ninf ? 0.0f : ex2(mc - M);
        f1 = o.x == ninf ? 0.0f : ex2(o.x - M);
        // the same order in both warpgroups
        const float la = w == 0 ? f0 * l : f1 * o.y, lb = w == 0 ? f1 * o.y : f0 * l;
        l = la + lb;
        mc = M;
      }
      const bool zero = !(row < rows && mine != 0) || (mc == ninf && l == 0.0f);  // sees nothing; NaN scores stay NaN
      const float inv = zero ? 0.0f : 1.0f / l;
      // partials [item][dim][row of the tile]: a warp's 32 rows store side by side
      const int64_t part = (((int64_t)b * p.Hkv + h) * p.NS + it.sp) * ((rows + kTtRows - 1) / kTtRows) + row / kTtRows;
      constexpr int COLS = PAIR ? D : D / 2;  // sharing the rows, each warpgroup writes half of the dimensions
#pragma unroll 1
      for (int q = 0; q < COLS / 32; ++q) {
        const int col = (PAIR ? 0 : w * COLS) + 32 * q;
        uint32_t o[32];
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0.0f;
        if (mine_units > 0) {
          tmem_ld32(t_o + w * D + col, o);
          tmem_wait32(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = f0 * __uint_as_float(o[i]);
        }
        if (other_units > 0) {
          tmem_ld32(t_o + (w ^ 1) * D + col, o);
          tmem_wait32(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] += f1 * __uint_as_float(o[i]);
        }
        if (it.fix && row < rows) {
          // NaN and infinities that were cleared, to the rows that see them
          const uint16_t* vb = static_cast<const uint16_t*>(p.vc) +
                               (p.row_map != nullptr ? p.row_map[b] : b) * p.c_sb + h * p.c_sh + col;
#pragma unroll 1
          for (int t0 = k0; t0 < k1; t0 += kTtKeys) {
            if (!tt_mixed(it, t0, p.window)) continue;
#pragma unroll 1
            for (int x = 0; x < kTtKeys && t0 + x < k1; ++x) {
              if (!((tt_bits(view, s, k1, t0, x >> 5) >> (x & 31)) & 1u)) continue;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const uint16_t y = vb[(int64_t)(t0 + x) * D + i];
                if ((y & 0x7f80u) == 0x7f80u) v[i] += bf16_to_f32(y);
              }
            }
          }
        }
        if (row < rows) {
          if (it.used <= 1) {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + out + col);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t y[4];
#pragma unroll
              for (int j = 0; j < 4; ++j)
                y[j] = zero ? 0u : bf16x2(v[8 * i + 2 * j] * inv, v[8 * i + 2 * j + 1] * inv);
              dst[i] = make_uint4(y[0], y[1], y[2], y[3]);
            }
          } else {
            float* dst = JOIN ? s_part + ((PAIR ? w * D : 0) + col) * kTtRows + r : p.ws_acc + (part * D + col) * kTtRows + r;
#pragma unroll
            for (int i = 0; i < 32; ++i) dst[i * kTtRows] = zero ? 0.0f : v[i];
          }
        }
      }
      if (it.used > 1 && row < rows && (PAIR || w == 0)) {
        if (JOIN)
          s_part_ml[(PAIR ? w * kTtRows : 0) + r] = zero ? make_float2(ninf, 0.0f) : make_float2(mc, l);
        else
          reinterpret_cast<float2*>(p.ws_ml)[part * kTtRows + r] =
              zero ? make_float2(ninf, 0.0f) : make_float2(mc * 0.693147180559945309f, l);
      }
      tc_fence_before();
      __syncwarp();
      if (tiles > 0) {
        // both have read the exchange: the queries may be overwritten
        if (!PAIR) ok = tt_sync(both, n_both, lane);
        if (lane == 0) mbar_arrive(oempty);
        ++work;
        kbase += tiles;
      }
      if (lane == 0) mbar_arrive(&iempty[slot]);
    }
    if (!ok && lane == 0) atomicOr(p.err, kErrFlagTimeout);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) tmem_dealloc(tmem, 512);
  if constexpr (JOIN) {
    // every thread of the cluster comes here, whatever gave up before
    const cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const TtItem& it = info[0];
    if (warp < 8 && it.tiles > 0 && it.used > 1) tt_join<D, PAIR>(p, it, s_part, s_part_ml, warp, lane);
    cluster.sync();  // nobody leaves while its part is read
  }
}

// Joins the splits: M = max m_j, out = sum e^(m_j - M) acc_j / sum e^(m_j - M)
// l_j, in split order.  A CTA takes 32 rows (the lanes, as the partials lie) x
// 32 dims (four per warp); eight splits' loads are in flight at a time.  Bound
// by latency: 13 us for 18 splits of 4 x 512 rows with nothing in L2, where the
// partials are when they are read.
template <int D>
__global__ void __launch_bounds__(256) tree_tc_merge_kernel(TreeAttnParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = p.N * p.G, rtiles = (rows + kTtRows - 1) / kTtRows;
  const int h = blockIdx.y, b = blockIdx.z, rb = blockIdx.x / (D / 32), col = (blockIdx.x % (D / 32)) * 32 + warp * 4;
  const int row = rb * 32 + lane;
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
  const unsigned ul = __reduce_or_sync(0xffffffffu, (unsigned)used);
  const unsigned uh = __reduce_or_sync(0xffffffffu, (unsigned)(used >> 32));
  const TreeRange rg = tree_range(p, len, cb, ((unsigned long long)uh << 32) | ul);
  const int ns = tree_splits_used(rg.lo, rg.hi, kTtKeys, p.NS);
  if (row >= rows || ns <= 1) return;  // one split wrote its output itself
  const int64_t first = ((int64_t)b * p.Hkv + h) * p.NS * rtiles + row / kTtRows;  // this row's tile in split 0
  const float2* ml = reinterpret_cast<const float2*>(p.ws_ml) + first * kTtRows + row % kTtRows;
  const float* ac = p.ws_acc + (first * D + col) * kTtRows + row % kTtRows;
  const int64_t step_ml = (int64_t)rtiles * kTtRows, step_ac = (int64_t)rtiles * D * kTtRows;
  const float ninf = __int_as_float(0xff800000);
  constexpr int kB = 8;
  float M = ninf;
  for (int j0 = 0; j0 < ns; j0 += kB) {
    float m[kB];
#pragma unroll
    for (int i = 0; i < kB; ++i) m[i] = j0 + i < ns ? __ldcg(ml + (j0 + i) * step_ml).x : ninf;
#pragma unroll
    for (int i = 0; i < kB; ++i) M = fmaxf(M, m[i]);
  }
  const float base = M == ninf ? 0.0f : M;
  float den = 0.0f, num[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int j0 = 0; j0 < ns; j0 += kB) {
    float2 y[kB];
    float a[kB][4];
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      if (j0 + i < ns) {
        y[i] = __ldcg(ml + (j0 + i) * step_ml);
#pragma unroll
        for (int u = 0; u < 4; ++u) a[i][u] = __ldcg(ac + (j0 + i) * step_ac + u * kTtRows);
      }
    }
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      if (j0 + i < ns && !(y[i].x == ninf && y[i].y == 0.0f)) {  // not a split that this row sees nothing of
        const float w = mexp(y[i].x - base);
        den = fmaf(w, y[i].y, den);
#pragma unroll
        for (int u = 0; u < 4; ++u) num[u] = fmaf(w, a[i][u], num[u]);
      }
    }
  }
  const int node = row / p.G, g = row - node * p.G;
  const float inv = den == 0.0f ? 0.0f : 1.0f / den;
  uint2 out = make_uint2(0u, 0u);
  if (den != 0.0f) out = make_uint2(bf16x2(num[0] * inv, num[1] * inv), bf16x2(num[2] * inv, num[3] * inv));
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + (((int64_t)b * p.N + node) * p.H + h * p.G + g) * D + col) = out;
}

// Splits of a sequence's keys: the number with the least expected time.  A key
// tile takes 0.95 us while few SMs read (1.9 with two row tiles), 1.4 when all
// share the HBM; an item 4 us to start and end, a launch 3.  Up to 8 splits, as
// far as such clusters fit the GPU at once, are joined by their cluster in 2.3
// us (4.5 with two row tiles); otherwise a second launch takes 1.5 on the GPU and
// as much again on the host, 0.25 per split that it walks through and 0.02 per
// 128 rows of an item's partials.
// Measured (8 nodes, 8 heads per KV head), us, joined by a second launch:
//   splits            1     2     3     5     9    18    37
//   1 x 600        12.3  12.4  11.6  11.2
//   1 x 8192       67.5  40.3  30.4  22.9  18.8  16.7  19.7
//   4 x 4000       37.4  25.9  20.9  18.0  17.0  22.2  33.7
//   16 x 8192      70.0  55.0  71.3  73.1  67.9  89.8   135
//   37 x 4096      55.0  71.7  75.5  81.5   103   157   249
//   1 x 65440, 64 nodes  941   479   327   204   122  74.8  87.8
// and as the rule takes them: 1 x 600 in a cluster of 5 10.8, 4 x 1000 in 5 11.4
// (one split 15.2), 4 x 4000 in 6 16.5, 16 x 8192 in 2 51, 1 x 8192 in 8 17.9 (a
// launch and an allocation fewer on the host, 4 us), 37 x 4096 55 in one split,
// 1 x 65440 73 in 18; 22 x 3800 on 2 KV heads in 3 19.2, in 2 23.5.
int tree_tc_splits(int64_t ctas, int64_t max_len, bool pair, bool* join) {
  const int64_t tiles = (max_len + kTtKeys - 1) / kTtKeys;
  int64_t best = 1;
  double least = 1e30;
  *join = false;
  // clusters of 2 to 8 CTAs that fit a B200 at once (one that fits fewer takes a second turn)
  constexpr int kFit[kTtCluster + 1] = {0, 0, 74, 45, 33, 26, 22, 15, 15};
  for (int64_t ns = 1; ns <= kTreeMaxSplits && ns <= tiles; ++ns) {
    const int64_t items = ctas * ns, per = (tiles + ns - 1) / ns;
    auto wave = [&](int64_t n) {  // n items side by side
      const double alone = pair ? 1.9 : 0.95, shared = 1.4 / 148 * (double)n;
      return n == 0 ? 0.0 : (double)per * (alone > shared ? alone : shared) + 4.0;
    };
    double t = (double)(items / 148) * wave(148) + wave(items % 148) + 3.0;
    const bool cluster = ns > 1 && ns <= kTtCluster && ctas <= kFit[ns];
    if (cluster) t += pair ? 4.5 : 2.3;
    else if (ns > 1) t += 1.5 + 0.25 * (double)ns + (pair ? 0.04 : 0.02) * (double)items + 1.5;
    if (t < least) {
      least = t;
      best = ns;
      *join = cluster;
    }
  }
  return (int)best;
}

int tree_tc_groups(int64_t rows) { return rows <= kTtRows ? 1 : (int)((rows + 2 * kTtRows - 1) / (2 * kTtRows)); }

int64_t tree_tc_partial_rows(int64_t rows) { return (rows + kTtRows - 1) / kTtRows * kTtRows; }

template <int D, bool PAIR>
cudaError_t tree_tc_launch1(const TreeAttnParams& p, int groups, const CUtensorMap& tmk, const CUtensorMap& tmv,
                            cudaStream_t st) {
  constexpr int smem = TtShape<D, PAIR>::kSmem;
  static_assert(smem <= 232448, "shared memory of one SM");
  const int items = p.B * p.Hkv * p.NS * groups;
  if (p.join) {
    static std::atomic<uint64_t> done{0};
    cudaError_t e = smem_once(done, tree_tc_kernel<D, PAIR, true>, smem);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)items);
    cfg.blockDim = dim3(kTtThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.NS;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return e == cudaSuccess ? cudaLaunchKernelEx(&cfg, tree_tc_kernel<D, PAIR, true>, p, groups, items, tmk, tmv) : e;
  }
  static std::atomic<uint64_t> done{0};
  cudaError_t e = smem_once(done, tree_tc_kernel<D, PAIR, false>, smem);
  if (e == cudaSuccess)
    e = launch_k(tree_tc_kernel<D, PAIR, false>, dim3((unsigned)(items < 148 ? items : 148)), dim3(kTtThreads), smem, st, p,
                 groups, items, tmk, tmv);
  if (e == cudaSuccess && p.NS > 1)
    e = launch_k(tree_tc_merge_kernel<D>,
                 dim3((unsigned)((p.N * p.G + 31) / 32 * (D / 32)), (unsigned)p.Hkv, (unsigned)p.B), dim3(256), 0, st, p);
  return e;
}

cudaError_t tree_tc_launch(const TreeAttnParams& p, int D, cudaStream_t st) {
  // (dim, position, KV head, cache row); heads or rows that share one are a map of one
  CUtensorMap tmk, tmv;
  const int64_t heads = p.c_sh ? p.Hkv : 1, hs = p.c_sh ? p.c_sh : (int64_t)p.T * D;
  const int64_t caches = p.c_sb ? p.Bc : 1, bs = p.c_sb ? p.c_sb : hs * heads;
  if (!tmap_encode_bf16_4d(p.kc, D, p.T, heads, caches, D, hs, bs, 64, kTtKeys, &tmk) ||
      !tmap_encode_bf16_4d(p.vc, D, p.T, heads, caches, D, hs, bs, 64, kTtKeys, &tmv))
    return cudaErrorInvalidValue;
  const int rows = p.N * p.G, groups = tree_tc_groups(rows);
  const bool pair = rows > kTtRows;
  if (D == 64) return pair ? tree_tc_launch1<64, true>(p, groups, tmk, tmv, st) : tree_tc_launch1<64, false>(p, groups, tmk, tmv, st);
  return pair ? tree_tc_launch1<128, true>(p, groups, tmk, tmv, st) : tree_tc_launch1<128, false>(p, groups, tmk, tmv, st);
}

}  // namespace mb
