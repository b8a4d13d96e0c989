// Attention of a tree of drafted tokens over a key/value cache.
//
// The cache holds lens[b] rows of context and, behind them, one row for each of the N nodes of
// the drafted tree.  Node n's query sees the context, its ancestors and itself:
//     o[b, n, h] = sum_t softmax_t(scale q[b, n, h] . k[b, h / G, t]) v[b, h / G, t]
//     over t < lens[b] and t = lens[b] + j, j an ancestor of n or n itself.
// N = 1 is a decode step of a single token; parents absent: node n - 1 is node n's parent.
//
// One pass over the cached rows with a running maximum and sum.  The query rows that share a
// key/value head (nodes x the heads of its group) are packed into 128-row tiles, so a 128-key
// tile is read once for all of them: S = Q K^T and O += P V on the tensor cores (tcgen05, P from
// TMEM), one row a thread in between.  What bounds it is the cache's bytes while the packed rows
// are few, and the tensor cores from about two tiles (256 rows) on.
//
// Work is cut by keys, not by sequences: all (sequence, head, row group, key tile) quadruples
// form one line, of which every CTA takes an equal part, whatever the lengths are -- the host
// never needs them.  A part that covers a unit's key tiles only partly leaves its unnormalised
// output with its maximum and sum in a workspace, and a second, small kernel adds the parts of
// such a unit in order; results do not depend on timing.
//
// Quantised caches: four warps turn the e4m3 tiles into bf16 ones in shared memory, the
// row's power-of-two scale included (exactly, see kv_cache.cuh), since a product of a 16-bit
// and an 8-bit operand does not exist and q in 8 bits would lose half its significand.
//
// A row behind the context that no node uses may hold anything: its scores are masked, and its
// values are zeroed in shared memory before the product (0 * NaN is NaN).  A drafted row that is
// used but holds an infinity or a NaN is zeroed likewise and added afterwards, entry by entry,
// to the nodes that see it.
// The reference has no decode path; the attention is the math of train.py:2564-2567.
#include "kv_cache.cuh"

namespace tfb {

CUtensorMap make_tmap_nd(const void* ptr, CUtensorMapDataType type, int rank, const uint64_t* dims, const uint64_t* strides,
                         const uint32_t* box, CUtensorMapSwizzle swizzle);
int num_sms(int dev);

constexpr int kTreeNodes = 64;
constexpr uint32_t kTreePanel = 128u * 128u;   // bytes of one 64-column panel of 128 bf16 rows
constexpr int kSegRing = 8;                    // segments whose poison masks are kept

struct TreeArgs {
  __nv_bfloat16* o;          // [B, N, Hq, D]
  const int* lens;
  const int* parents;        // null: a chain
  int B, N, Hq, Hkv, G;
  int gb, nb;                // heads and nodes of a 128-row tile
  int gg, rt, rg;            // head groups, row tiles and row groups (of NT tiles) a key/value head
  float scale_log2;          // |scale| log2(e), never 0
  int neg;                   // scale < 0
  float* part;               // [2 * grid][NT * 128][D] unnormalised partial outputs
  float2* part_ml;           // [2 * grid][NT * 128] their maximum (log2 units) and sum
  int* err;
};

__device__ __forceinline__ int tree_len(const TreeArgs& a, const KvView& c, int b) { return max(0, min(a.lens[b], c.tmax)); }
// Key tiles of sequence b: its context and as many node rows as the cache has room for.
__device__ __forceinline__ int tree_tiles(const TreeArgs& a, const KvView& c, int b) {
  return (int)((min((long long)tree_len(a, c, b) + a.N, (long long)c.tmax) + 127) >> 7);
}

// The key tiles of a CTA, in order: [pos, end) of the line of all tiles.
struct TreeIter {
  long long pos, end, base;   // base: first tile of sequence b on the line
  int b, kt, units;           // kt: key tiles of sequence b; units: (head, row group) pairs
  int h, rgi, len, k, k0, k1; // present segment: head, row group, context length, key tile and its range
  int seg;                    // segments begun so far, less one

  // Present tile -> next one; false at the end.
  __device__ __forceinline__ bool next(const TreeArgs& a, const KvView& c) {
    if (seg >= 0 && k + 1 < k1) {
      ++k;
      return true;
    }
    if (pos >= end) return false;
    while (pos >= base + (long long)kt * units) {
      base += (long long)kt * units;
      kt = tree_tiles(a, c, ++b);
    }
    len = tree_len(a, c, b);
    const long long rel = pos - base;
    const int u = (int)(rel / kt);
    k0 = k = (int)(rel - (long long)u * kt);
    k1 = (int)min((long long)kt, k0 + (end - pos));
    h = u / a.rg;
    rgi = u - h * a.rg;
    pos += k1 - k0;
    ++seg;
    return true;
  }
  __device__ __forceinline__ bool first() const { return k == k0; }
  __device__ __forceinline__ bool last() const { return k + 1 == k1; }
};

// Start of CTA `cta` of `grid` on the line of tiles (warp-collective); total: the line's length.
__device__ __forceinline__ TreeIter tree_begin(const TreeArgs& a, const KvView& c, int cta, int grid, long long& total) {
  const int lane = threadIdx.x & 31;
  TreeIter it;
  it.units = a.Hkv * a.rg;
  long long sum = 0;
  for (int b = lane; b < a.B; b += 32) sum += tree_tiles(a, c, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  total = sum * it.units;
  grid = (int)min((long long)grid, total);   // CTAs that have work
  it.pos = cta < grid ? total * cta / grid : total;
  it.end = cta < grid ? total * (cta + 1) / grid : total;
  it.base = 0;
  it.b = 0;
  it.seg = -1;
  it.k = it.k0 = it.k1 = 0;
  // the sequence in which pos lies
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const long long mine = b0 + lane < a.B ? (long long)tree_tiles(a, c, b0 + lane) * it.units : 0;
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const unsigned in = __ballot_sync(0xffffffffu, it.pos < it.base + inc);
    const int at = in ? __ffs(in) - 1 : 31;
    const long long before = __shfl_sync(0xffffffffu, inc - mine, at);
    const long long all = __shfl_sync(0xffffffffu, inc, 31);
    if (in || b0 + 32 >= a.B) {
      it.b = min(b0 + at, a.B - 1);
      it.base += before;
      break;
    }
    it.base += all;
  }
  it.kt = tree_tiles(a, c, it.b);
  return it;
}

// Ancestors-or-self masks of nodes `lane` and `lane + 32` (warp-collective, by pointer
// doubling); 0 for an unused node: one whose line of parents meets an entry that is neither -1
// nor an earlier node, or whose own row the cache has no room for (`fit` rows fit).
__device__ __forceinline__ void tree_lines(const int* par, int N, int fit, unsigned long long& m0, unsigned long long& m1) {
  const int lane = threadIdx.x & 31;
  unsigned long long m[2];
  int j[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int n = lane + 32 * i;
    m[i] = 1ull << n;
    j[i] = -2;
    if (n < N && n < fit) {
      if (par == nullptr) {
        m[i] = n == 63 ? ~0ull : (2ull << n) - 1;
        j[i] = -1;
      } else {
        const int p = par[n];
        j[i] = p >= -1 && p < n ? p : -2;
      }
    }
  }
  while (__any_sync(0xffffffffu, j[0] >= 0 || j[1] >= 0)) {
    unsigned long long am[2];
    int aj[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int src = j[i] & 31;
      const unsigned long long x0 = __shfl_sync(0xffffffffu, m[0], src), x1 = __shfl_sync(0xffffffffu, m[1], src);
      const int y0 = __shfl_sync(0xffffffffu, j[0], src), y1 = __shfl_sync(0xffffffffu, j[1], src);
      am[i] = j[i] >= 32 ? x1 : x0;
      aj[i] = j[i] >= 32 ? y1 : y0;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (j[i] >= 0) {
        m[i] |= am[i];
        j[i] = aj[i];
      }
  }
  m0 = j[0] == -2 ? 0 : m[0];
  m1 = j[1] == -2 ? 0 : m[1];
}
__device__ __forceinline__ unsigned long long used_nodes(unsigned long long m0, unsigned long long m1) {
  return (unsigned long long)__ballot_sync(0xffffffffu, m0 != 0) | ((unsigned long long)__ballot_sync(0xffffffffu, m1 != 0) << 32);
}

// Visible columns s .. s + 31 (relative to the first node's row) as a bit mask.
__device__ __forceinline__ uint32_t tree_word(unsigned long long line, int s) {
  if (s >= kTreeNodes) return 0;
  if (s >= 0) return (uint32_t)(line >> s);
  return s > -32 ? (uint32_t)(line << -s) | ((1u << -s) - 1) : 0xffffffffu;
}

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}
__device__ __forceinline__ float tree_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint64_t tree_desc_k(uint32_t base, int kk) {   // K-major operand, 16 of D at step kk
  return umma_desc_sw128(base + (uint32_t)(kk >> 2) * kTreePanel + (uint32_t)(kk & 3) * 32u, 16, 1024);
}
__device__ __forceinline__ uint64_t tree_desc_mn(uint32_t base, int kk) {  // MN-major operand, 16 keys at step kk
  return umma_desc_sw128(base + (uint32_t)kk * 2048u, kTreePanel, 1024);
}

// 4 e4m3 codes -> 4 bf16 (two words), times m1 (and m2 unless it is 1).  The code's exponent and
// significand bits, moved to a bf16's place, are the value times 2^-120 (subnormals included),
// so a multiplication by 2^120 times the row's scale is all that is left; scales whose
// exponent does not fit that factor take a second one.
__device__ __forceinline__ uint2 codes4(uint32_t x, __nv_bfloat162 m1) {
  const uint32_t lo = __byte_perm(x, 0, 0x1404), hi = __byte_perm(x, 0, 0x3424);
  uint32_t a = (lo & 0x80008000u) | ((lo >> 4) & 0x07f007f0u);
  uint32_t b = (hi & 0x80008000u) | ((hi >> 4) & 0x07f007f0u);
  const __nv_bfloat162 u = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a), m1);
  const __nv_bfloat162 v = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&b), m1);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&u), *reinterpret_cast<const uint32_t*>(&v));
}
__device__ __forceinline__ __nv_bfloat162 bf16x2_bits(uint32_t h) {
  const uint32_t w = h | (h << 16);
  return *reinterpret_cast<const __nv_bfloat162*>(&w);
}

template <int D, bool QUANT, int NT>
struct TreeCfg {
  static constexpr uint32_t TILE = 128u * D * 2u;
  static constexpr uint32_t RAW = 128u * D;
  static constexpr int QS = 2 / NT;            // stages of NT query tiles
  static constexpr int NS = QUANT ? 3 : 5;     // bf16 key / value tiles
  static constexpr int RS = QUANT ? 4 : 0;     // e4m3 key / value tiles
  static constexpr int AUX = QUANT ? 4 : 1;    // warps that convert, or clear unused rows
  static constexpr int THREADS = 32 * (2 + 4 * NT + AUX);
  static constexpr size_t SMEM = 1024 + 2 * TILE + NS * TILE + RS * RAW + 40 * 8 + kSegRing * 8 + 16;
  static constexpr int LEAD = NT == 1 ? 2 : 1; // key tiles ahead of the first value tile
};
static_assert(TreeCfg<128, false, 1>::SMEM <= 232448 && TreeCfg<128, true, 1>::SMEM <= 232448, "shared memory");

// Roles: warp 0 loads (TMA), warp 1 issues the products, NT groups of four warps run the softmax
// of a row tile each, the rest converts quantised tiles or clears unused rows of value tiles.
// Key and value tiles share one ring in the order in which the products take them.
//   NT = 1: S is double-buffered in TMEM (S(g + 2) is issued behind P(g) V(g)), so the softmax
//           never waits for a product.  TMEM: S 2 x 128 | O 128.
//   NT = 2: one S a row tile; the tiles alternate.  TMEM: S 2 x 128 | O 2 x 128.
// P overwrites the first 64 columns of its S as packed bf16 pairs.
template <int D, bool QUANT, int NT>
__global__ void __launch_bounds__(TreeCfg<D, QUANT, NT>::THREADS, 1)
    tree_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                          const __grid_constant__ CUtensorMap tmV, const TreeArgs a, const KvView c) {
  using Cfg = TreeCfg<D, QUANT, NT>;
  constexpr uint32_t TILE = Cfg::TILE, RAW = Cfg::RAW;
  constexpr int NS = Cfg::NS, RS = Cfg::RS, QS = Cfg::QS, LEAD = Cfg::LEAD;
  constexpr int PANELS = D / 64;
  constexpr uint32_t IDESC_S = umma_idesc_bf16(128, 128, false, false);
  constexpr uint32_t IDESC_O = umma_idesc_bf16(128, D, false, true);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                          // [2] tiles: QS stages of NT
  uint8_t* sKV = sQ + 2 * TILE;                // [NS] tiles
  uint8_t* sRaw = sKV + NS * TILE;             // [RS] tiles
  uint64_t* bars = reinterpret_cast<uint64_t*>(sRaw + RS * RAW);
  uint64_t* q_full = bars;                     // [2]
  uint64_t* q_empty = bars + 2;                // [2]
  uint64_t* kv_full = bars + 4;                // [NS <= 5]
  uint64_t* kv_empty = bars + 9;               // [NS]
  uint64_t* v_ready = bars + 14;               // [NS] value tiles whose unused rows are cleared (not QUANT)
  uint64_t* raw_full = bars + 19;              // [RS <= 4]
  uint64_t* raw_empty = bars + 23;             // [RS]
  uint64_t* s_full = bars + 27;                // [2]
  uint64_t* p_full = bars + 29;                // [2]
  uint64_t* pv_done = bars + 31;               // [2]
  uint64_t* drain = bars + 33;
  // value tiles land on a barrier of their own (not QUANT): the warp that waits for them waits for
  // no key tile, and a wait by parity must see every phase of its barrier
  uint64_t* v_full = bars + 34;                // [NS]
  unsigned long long* s_poison = reinterpret_cast<unsigned long long*>(bars + 40);   // [kSegRing] drafted rows not finite
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_poison + kSegRing);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&pv_done[i], 1);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(&kv_full[i], QUANT ? 128 : 1);
      mbar_init(&kv_empty[i], 1);
      mbar_init(&v_ready[i], 32);
      mbar_init(&v_full[i], 1);
    }
    for (int i = 0; i < RS; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], 128);
    }
    mbar_init(drain, 1);
    for (int i = 0; i < kSegRing; ++i) s_poison[i] = 0;
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  long long total;
  TreeIter it = tree_begin(a, c, (int)blockIdx.x, (int)gridDim.x, total);
  const int tiles = (int)(it.end - it.pos);    // of this CTA
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch_dependents();
  const uint32_t tmem = *tmem_slot;
  constexpr uint32_t O_COL = 256;
  // position in the ring of the value tile of tile g
  auto v_item = [&](int g) { return NT == 1 ? min(2 * g + 2, 2 * tiles - 1) : 2 * g + 1; };

  if (warp == 0) {
    // ------------------------------------------------------------------ loads
    if (lane == 0 && tiles > 0) {
      bool ok = true;
      int item = 0, q_segs = 0;
      uint64_t* const empty = QUANT ? raw_empty : kv_empty;
      constexpr int R = QUANT ? RS : NS;
      uint32_t is_v = 0, phase[2] = {0, 0};     // per slot: what it holds, and the parities of its barriers
      auto full = [&](int slot, int v) { return QUANT ? &raw_full[slot] : v ? &v_full[slot] : &kv_full[slot]; };
      auto tile = [&](const TreeIter& t, int v) -> bool {
        const int slot = item % R;
        if (item >= R && !mbar_wait(&empty[slot], ((item / R) + 1) & 1, abort_flag, a.err, ERR_TIMEOUT_PRODUCER)) return false;
        uint64_t* bar = full(slot, v);
        const CUtensorMap* map = v ? &tmV : &tmK;
        mbar_arrive_expect_tx(bar, QUANT ? RAW : TILE);
        is_v = (is_v & ~(1u << slot)) | ((uint32_t)v << slot);
        phase[QUANT ? 0 : v] ^= 1u << slot;
        if constexpr (QUANT) {
          tma_load_4d(sRaw + slot * RAW, map, bar, 0, t.k * 128, t.h, t.b);
        } else {
#pragma unroll
          for (int p = 0; p < PANELS; ++p)
            tma_load_4d(sKV + slot * TILE + p * kTreePanel, map, bar, p * 64, t.k * 128, t.h, t.b);
        }
        ++item;
        return true;
      };
      auto queries = [&](const TreeIter& t) -> bool {
        const int st = t.seg % QS;
        if (t.seg >= QS && !mbar_wait(&q_empty[st], ((t.seg / QS) + 1) & 1, abort_flag, a.err, ERR_TIMEOUT_PRODUCER)) return false;
        mbar_arrive_expect_tx(&q_full[st], (uint32_t)(NT * PANELS * a.gb * a.nb) * 128u);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const int rt = t.rgi * NT + i;
          const int ng = rt / a.gg, hg = rt - ng * a.gg;
#pragma unroll
          for (int p = 0; p < PANELS; ++p)
            tma_load_5d(sQ + (st * NT + i) * TILE + p * kTreePanel, &tmQ, &q_full[st], p * 64, hg * a.gb, ng * a.nb, t.h, t.b);
        }
        q_segs = t.seg + 1;
        return true;
      };
      TreeIter ki = it, vi = it;
      auto key = [&]() -> bool {   // the next key tile, behind its queries; true also at the end
        if (!ki.next(a, c)) return true;
        if (ki.first() && !queries(ki)) return false;
        return tile(ki, 0);
      };
      for (int i = 0; i < LEAD && ok; ++i) ok = key();
      while (ok && vi.next(a, c)) ok = tile(vi, 1) && key();
      if (!ok) {   // let the copies in flight land before the CTA ends
        const unsigned long long t0 = globaltimer_ns();
        for (int i = max(0, item - R); i < item; ++i) {
          const int slot = i % R, v = (is_v >> slot) & 1;
          while (!mbar_try_wait(full(slot, v), ((phase[QUANT ? 0 : v] >> slot) & 1) ^ 1))
            if (globaltimer_ns() - t0 > 100000000ull) break;
        }
        for (int i = max(0, q_segs - QS); i < q_segs; ++i)
          while (!mbar_try_wait(&q_full[i % QS], (i / QS) & 1))
            if (globaltimer_ns() - t0 > 100000000ull) break;
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ products
    if (lane == 0 && tiles > 0) {
      bool ok = true;
      uint32_t vphase = 0, kphase = 0;          // per slot (not QUANT: keys and values land on separate barriers)
      TreeIter si[NT], pi[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) si[i] = pi[i] = it;
      int sg[NT] = {}, pg[NT] = {};
      auto k_item = [&](int g) { return NT == 1 ? (g < 2 ? g : 2 * g - 1) : 2 * g; };
      // S of the next tile of row tile t; true also at the end
      auto scores = [&](int t) -> bool {
        if (!si[t].next(a, c)) return true;
        const int g = sg[t]++, kit = k_item(g), st = si[t].seg % QS;
        if (si[t].first() && !mbar_wait(&q_full[st], (si[t].seg / QS) & 1, abort_flag, a.err, ERR_TIMEOUT_MMA)) return false;
        if (!mbar_wait(&kv_full[kit % NS], QUANT ? (kit / NS) & 1 : (kphase >> (kit % NS)) & 1, abort_flag, a.err, ERR_TIMEOUT_MMA))
          return false;
        tc_fence_after();
        const uint32_t q_addr = smem_u32(sQ + (st * NT + t) * TILE), k_addr = smem_u32(sKV + (kit % NS) * TILE);
        const int buf = NT == 1 ? g & 1 : t;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_bf16(tmem + buf * 128, tree_desc_k(q_addr, kk), tree_desc_k(k_addr, kk), IDESC_S, kk > 0 ? 1u : 0u);
        umma_commit(&s_full[buf]);
        if (t == NT - 1) {
          kphase ^= 1u << (kit % NS);
          umma_commit(&kv_empty[kit % NS]);
          if (si[t].last()) umma_commit(&q_empty[st]);
        }
        return true;
      };
      auto outputs = [&](int t) -> bool {
        pi[t].next(a, c);
        const int g = pg[t]++, vit = v_item(g), slot = vit % NS, buf = NT == 1 ? g & 1 : t;
        if (t == 0) {
          if constexpr (QUANT) {
            if (!mbar_wait(&kv_full[slot], (vit / NS) & 1, abort_flag, a.err, ERR_TIMEOUT_MMA)) return false;
          } else {
            if (!mbar_wait(&v_ready[slot], (vphase >> slot) & 1, abort_flag, a.err, ERR_TIMEOUT_MMA)) return false;
            vphase ^= 1u << slot;
          }
        }
        if (!mbar_wait(&p_full[buf], NT == 1 ? (g >> 1) & 1 : g & 1, abort_flag, a.err, ERR_TIMEOUT_MMA)) return false;
        tc_fence_after();
        const uint32_t v_addr = smem_u32(sKV + slot * TILE);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          umma_bf16_tmem_a(tmem + O_COL + t * 128, tmem + buf * 128 + kk * 8, tree_desc_mn(v_addr, kk), IDESC_O,
                           (!pi[t].first() || kk > 0) ? 1u : 0u);
        if (t == NT - 1) umma_commit(&kv_empty[slot]);
        umma_commit(&pv_done[buf]);
        return true;
      };
      for (int i = 0; i < LEAD && ok; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) ok = ok && scores(t);
      for (int g = 0; g < tiles && ok; ++g)
#pragma unroll
        for (int t = 0; t < NT; ++t) ok = ok && outputs(t) && scores(t);
      if (!ok) {
        *abort_flag = 1;
        umma_commit(drain);
        const unsigned long long t0 = globaltimer_ns();
        while (!mbar_try_wait(drain, 0))
          if (globaltimer_ns() - t0 > 100000000ull) break;
      }
    }
  } else if (warp < 2 + 4 * NT) {
    // ------------------------------------------------------------------ softmax of row tile t
    const int t = (warp - 2) >> 2, q4 = warp & 3, r = q4 * 32 + lane;
    const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
    const uint32_t tO = tmem + O_COL + t * 128 + lane_off;
    const float cl = a.scale_log2;
    const int rn = r / a.gb, rh = r - rn * a.gb;
    float m_run = -INFINITY, l = 0.f;
    unsigned long long line = 0;
    int n = 0, head = 0, g = 0;
    bool live = false, warp_live = false, ok = true;
    while (ok && it.next(a, c)) {
      if (it.first()) {
        const int rt = it.rgi * NT + t;
        const int ng = rt / a.gg, hg = rt - ng * a.gg;
        n = ng * a.nb + rn;
        head = hg * a.gb + rh;
        live = rn < a.nb && n < a.N && head < a.G && rt < a.rt;
        warp_live = __any_sync(0xffffffffu, live);
        unsigned long long m0, m1;
        tree_lines(a.parents ? a.parents + (long long)it.b * a.N : nullptr, a.N, c.tmax - it.len, m0, m1);
        const unsigned long long x0 = __shfl_sync(0xffffffffu, m0, n & 31), x1 = __shfl_sync(0xffffffffu, m1, n & 31);
        line = !live ? 0 : n >= 32 ? x1 : x0;
        m_run = -INFINITY;
        l = 0.f;
      }
      const int buf = NT == 1 ? g & 1 : t, sph = NT == 1 ? (g >> 1) & 1 : g & 1;
      const uint32_t tS = tmem + buf * 128 + lane_off;
      if (!mbar_wait_warp(&s_full[buf], sph, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) { ok = false; break; }
      // products into O up to tile g - 2 (NT = 1) or g - 1 were issued before S(g): these waits
      // only keep count of the barrier's phases
      if (NT == 1 ? g >= 2 : g >= 1) {
        if (!mbar_wait_warp(&pv_done[buf], sph ^ 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) { ok = false; break; }
      }
      tc_fence_after();
      if (warp_live) {
        const int off = it.k * 128 - it.len;          // of the tile's first key from the first node's row
        const bool masked = off + 128 > 0;
        float x[64];
        // half hf of the row of S: scaled by the sign, masked columns -inf
        auto half_row = [&](int hf) {
          uint32_t* xr = reinterpret_cast<uint32_t*>(x);
          __syncwarp();
          tmem_ld_32x32b_x32(tS + hf * 64, *reinterpret_cast<uint32_t(*)[32]>(xr));
          tmem_ld_32x32b_x32(tS + hf * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(xr + 32));
          tmem_ld_wait();
          if (a.neg) {
#pragma unroll
            for (int i = 0; i < 64; ++i) x[i] = -x[i];
          }
          if (masked) {
            const uint32_t w0 = tree_word(line, off + hf * 64), w1 = tree_word(line, off + hf * 64 + 32);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (!((w0 >> i) & 1u)) x[i] = -INFINITY;
              if (!((w1 >> i) & 1u)) x[32 + i] = -INFINITY;
            }
          }
        };
        auto half_max = [&](float mx) -> float {
          float m4[4] = {mx, x[0], x[1], x[2]};
#pragma unroll
          for (int i = 3; i < 63; i += 4)
#pragma unroll
            for (int k = 0; k < 4; ++k) m4[k] = fmaxf(m4[k], x[i + k]);
          return fmaxf(fmaxf(fmaxf(m4[0], x[63]), m4[1]), fmaxf(m4[2], m4[3]));
        };
        half_row(0);
        float mx = half_max(-INFINITY);
        half_row(1);
        mx = half_max(mx) * cl;
        // the exponents' reference moves only when the maximum grows by more than 8 (p stays below 2^8)
        float alpha = 1.f;
        const bool grow = live && mx > m_run + 8.f;
        if (grow) {
          alpha = tree_ex2(m_run - mx);
          m_run = mx;
        }
        const float mref = m_run == -INFINITY ? 0.f : m_run;   // nothing seen so far: every p is 2^-inf = 0
        const float2 c2 = make_float2(cl, cl), nm2 = make_float2(-mref, -mref);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t pk[2][32];
        auto half_exp = [&](uint32_t (&p)[32]) {
#pragma unroll
          for (int i = 0; i < 64; i += 2) {
            const float2 v = __ffma2_rn(make_float2(x[i], x[i + 1]), c2, nm2);
            const float2 e = make_float2(tree_ex2(v.x), tree_ex2(v.y));
            p[i >> 1] = pack_bf16x2(e.x, e.y);
            sum[(i >> 1) & 1] = __fadd2_rn(sum[(i >> 1) & 1], e);
          }
        };
        half_exp(pk[1]);
        half_row(0);
        half_exp(pk[0]);
        const float2 s2 = __fadd2_rn(sum[0], sum[1]);
        l = l * alpha + (s2.x + s2.y);
        if (!it.first() && __any_sync(0xffffffffu, grow)) {
          if (NT == 1 && !mbar_wait_warp(&pv_done[buf ^ 1], ((g - 1) >> 1) & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) { ok = false; break; }
          tc_fence_after();
#pragma unroll 1
          for (int cc = 0; cc < D / 32; ++cc) {
            uint32_t o[32];
            __syncwarp();
            tmem_ld_32x32b_x32(tO + cc * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st_32x32b_x32(tO + cc * 32, o);
          }
        }
        __syncwarp();
        tmem_st_32x32b_x32(tS, pk[0]);
        tmem_st_32x32b_x32(tS + 32, pk[1]);
        tmem_st_wait();
        tc_fence_before();
      }
      mbar_arrive(&p_full[buf]);
      if (it.last()) {
        if (!mbar_wait_warp(&pv_done[buf], sph, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) { ok = false; break; }
        tc_fence_after();
        if (warp_live) {
          const bool whole = it.k0 == 0 && it.k1 == it.kt;
          const long long slot = 2LL * blockIdx.x + (it.k0 == 0 ? 1 : 0);
          const float inv = line == 0 || l == 0.f ? 0.f : 1.f / l;
          unsigned long long bad = s_poison[it.seg & (kSegRing - 1)] & line;
          __nv_bfloat16* dst = a.o + (((long long)it.b * a.N + n) * a.Hq + it.h * a.G + head) * D;
          float* pd = a.part + ((slot * NT + t) * 128 + r) * D;
#pragma unroll 1
          for (int cc = 0; cc < D / 32; ++cc) {
            uint32_t o[32];
            __syncwarp();
            tmem_ld_32x32b_x32(tO + cc * 32, o);
            tmem_ld_wait();
            float f[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = line != 0 && l != 0.f ? __uint_as_float(o[i]) : 0.f;
            for (unsigned long long w = bad; w; w &= w - 1) {   // rows with an infinity or a NaN: those entries
              const int j = __ffsll((long long)w) - 1;
              if constexpr (QUANT) {
#pragma unroll
                for (int i = 0; i < 32; ++i) f[i] = __int_as_float(0x7fffffff);
              } else {
                const __nv_bfloat16* row = reinterpret_cast<const __nv_bfloat16*>(c.p[1] + it.b * c.b + it.h * c.h +
                                                                                  ((long long)it.len + j) * c.t) + cc * 32;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                  const float v = __bfloat162float(row[i]);
                  if (!(fabsf(v) < INFINITY)) f[i] += v;
                }
              }
            }
            if (live) {
              if (whole) {
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                  uint4 u;
                  u.x = pack_bf16x2(f[i] * inv, f[i + 1] * inv);
                  u.y = pack_bf16x2(f[i + 2] * inv, f[i + 3] * inv);
                  u.z = pack_bf16x2(f[i + 4] * inv, f[i + 5] * inv);
                  u.w = pack_bf16x2(f[i + 6] * inv, f[i + 7] * inv);
                  *reinterpret_cast<uint4*>(dst + cc * 32 + i) = u;
                }
              } else {
#pragma unroll
                for (int i = 0; i < 32; i += 4)
                  *reinterpret_cast<float4*>(pd + cc * 32 + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
              }
            }
          }
          if (live && !whole) a.part_ml[(slot * NT + t) * 128 + r] = line != 0 ? make_float2(m_run, l) : make_float2(-INFINITY, 0.f);
        }
        tc_fence_before();
      }
      ++g;
    }
  } else {
    // ------------------------------------------------------------------ e4m3 -> bf16, unused rows
    const int tid = (int)threadIdx.x - 32 * (2 + 4 * NT);
    unsigned long long used = 0;
    int used_seg = -1;
    auto enter = [&](const TreeIter& v) {       // a value tile's segment (warp-collective)
      if (v.seg == used_seg) return;
      used_seg = v.seg;
      unsigned long long m0, m1;
      tree_lines(a.parents ? a.parents + (long long)v.b * a.N : nullptr, a.N, c.tmax - v.len, m0, m1);
      used = used_nodes(m0, m1);
      if (tid == 0) s_poison[(v.seg + 3) & (kSegRing - 1)] = 0;   // last used five segments ago
    };
    if constexpr (!QUANT) {
      constexpr int CH = D / 8;                 // 16-byte chunks a row
      int g = 0;
      uint32_t vphase = 0;
      while (it.next(a, c)) {
        enter(it);
        const int slot = v_item(g++) % NS;
        if (!mbar_wait_warp(&v_full[slot], (vphase >> slot) & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) break;
        vphase ^= 1u << slot;
        const int off = it.k * 128 - it.len;
        if (off + 128 > 0) {
          uint8_t* tile = sKV + slot * TILE;
          unsigned long long bad = 0;
          for (int row = max(0, -off) + lane / CH; row < 128; row += 32 / CH) {
            const int j = row + off, ch = lane % CH;
            uint4* p = reinterpret_cast<uint4*>(tile + (ch >> 3) * kTreePanel + sw128_chunk_offset(row, ch & 7));
            if (j >= kTreeNodes || !((used >> j) & 1)) {
              *p = make_uint4(0, 0, 0, 0);
            } else {
              uint4 u = *p;
              uint32_t* w = reinterpret_cast<uint32_t*>(&u);
              bool hit = false;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if ((w[i] & 0x7f80u) == 0x7f80u) { w[i] &= 0xffff0000u; hit = true; }
                if ((w[i] & 0x7f800000u) == 0x7f800000u) { w[i] &= 0xffffu; hit = true; }
              }
              if (hit) {
                *p = u;
                bad |= 1ull << j;
              }
            }
          }
          uint32_t lo = __reduce_or_sync(0xffffffffu, (uint32_t)bad), hi = __reduce_or_sync(0xffffffffu, (uint32_t)(bad >> 32));
          if (lane == 0 && (lo | hi)) s_poison[it.seg & (kSegRing - 1)] |= ((unsigned long long)hi << 32) | lo;
          fence_proxy_async_smem();
        }
        mbar_arrive(&v_ready[slot]);
      }
    } else {
      // chunk q of a tile: 16 codes of row q / CH; a thread's rows are tid / CH + i * (128 / CH)
      constexpr int CH = D / 16, RPT = CH;      // chunks a row = rows a thread
      const int ch = tid % CH, row0 = tid / CH;
      constexpr int STEP = 128 / CH;
      TreeIter ki = it, vi = it;
      int item = 0;
      uint32_t sc[RPT];
      auto scales = [&](const TreeIter& x, int kv) {
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          const long long tt = (long long)x.k * 128 + row0 + i * STEP;
          sc[i] = tt < c.tmax ? c.s[kv][x.b * c.sb + x.h * c.sh + tt * c.st] : 127u;
        }
      };
      auto convert = [&](const TreeIter& x, int kv) -> bool {
        const int rslot = item % RS, slot = item % NS;
        if (!mbar_wait_warp(&raw_full[rslot], (item / RS) & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) return false;
        if (item >= NS && !mbar_wait_warp(&kv_empty[slot], ((item / NS) + 1) & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) return false;
        const uint8_t* src = sRaw + rslot * RAW;
        uint8_t* dst = sKV + slot * TILE + (ch >> 2) * kTreePanel;
        const int off = x.k * 128 - x.len;
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          const int row = row0 + i * STEP;
          const uint4 u = *reinterpret_cast<const uint4*>(src + row * D + ch * 16);
          uint32_t e = sc[i];
          bool clear = false;
          if (kv == 1 && row + off >= 0) {      // behind the context
            const int j = row + off;
            clear = j >= kTreeNodes || !((used >> j) & 1);
            if (!clear && e == (uint32_t)kScaleNan) {
              clear = true;
              if (ch == 0) atomicOr(&s_poison[x.seg & (kSegRing - 1)], 1ull << j);
            }
          }
          const __nv_bfloat162 m1 = bf16x2_bits(e == (uint32_t)kScaleNan ? 0x7fffu : min(e + 120u, 254u) << 7);
          const uint2 p0 = codes4(u.x, m1), p1 = codes4(u.y, m1), p2 = codes4(u.z, m1), p3 = codes4(u.w, m1);
          uint4 o0 = make_uint4(p0.x, p0.y, p1.x, p1.y), o1 = make_uint4(p2.x, p2.y, p3.x, p3.y);
          if (e > 134u && e != (uint32_t)kScaleNan) {   // scales above 2^7
            const __nv_bfloat162 m2 = bf16x2_bits((e - 7u) << 7);
            uint32_t* w0 = reinterpret_cast<uint32_t*>(&o0);
            uint32_t* w1 = reinterpret_cast<uint32_t*>(&o1);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const __nv_bfloat162 y0 = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&w0[k]), m2);
              const __nv_bfloat162 y1 = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&w1[k]), m2);
              w0[k] = *reinterpret_cast<const uint32_t*>(&y0);
              w1[k] = *reinterpret_cast<const uint32_t*>(&y1);
            }
          }
          if (clear) o0 = o1 = make_uint4(0, 0, 0, 0);
          const int c0 = 2 * (ch & 3);
          // the two panels' lanes store their chunks in opposite order: no bank is hit twice
          const bool swap = ch >= 4;
          *reinterpret_cast<uint4*>(dst + sw128_chunk_offset(row, swap ? c0 + 1 : c0)) = swap ? o1 : o0;
          *reinterpret_cast<uint4*>(dst + sw128_chunk_offset(row, swap ? c0 : c0 + 1)) = swap ? o0 : o1;
        }
        fence_proxy_async_smem();
        mbar_arrive(&kv_full[slot]);
        mbar_arrive(&raw_empty[rslot]);
        ++item;
        return true;
      };
      bool ok = true;
      auto key = [&]() -> bool {
        if (!ki.next(a, c)) return true;
        scales(ki, 0);
        return convert(ki, 0);
      };
      for (int i = 0; i < LEAD && ok; ++i) ok = key();
      while (ok && vi.next(a, c)) {
        enter(vi);
        scales(vi, 1);
        ok = convert(vi, 1) && key();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Adds the parts of the units that more than one CTA worked on: one warp a query row.
template <int D>
__global__ void __launch_bounds__(128) tree_combine_kernel(const TreeArgs a, const KvView c, int grid, int NT) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const bool on = w < (long long)a.B * a.N * a.Hq;
  long long c0 = 0, c1 = 0;
  int row = 0;
  if (on) {
    const int hq = (int)(w % a.Hq), n = (int)(w / a.Hq % a.N), b = (int)(w / a.Hq / a.N);
    const int h = hq / a.G, hd = hq - h * a.G, units = a.Hkv * a.rg;
    long long all = 0, before = 0;
    for (int i = lane; i < a.B; i += 32) {
      const long long k = tree_tiles(a, c, i);
      all += k;
      if (i < b) before += k;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      all += __shfl_xor_sync(0xffffffffu, all, o);
      before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    const int rt = (n / a.nb) * a.gg + hd / a.gb;
    row = (rt % NT) * 128 + (n % a.nb) * a.gb + hd % a.gb;
    const long long W = all * units, kt = tree_tiles(a, c, b);
    grid = (int)min((long long)grid, W);
    const long long p0 = before * units + (long long)(h * a.rg + rt / NT) * kt;
    c0 = ((p0 + 1) * grid - 1) / W;          // the CTA that owns a position of the line
    c1 = ((p0 + kt) * grid - 1) / W;
  }
  griddep_wait();                            // every thread: this grid ends after the one before it
  if (!on || c0 == c1) return;               // one CTA had the whole unit and wrote it
  // CTA c0 ends with this unit's first part (slot 1), the others begin with theirs (slot 0)
  float M = -INFINITY;
  for (long long i = c0; i <= c1; ++i) {
    const float2 ml = __ldcg(&a.part_ml[(2 * i + (i == c0 ? 1 : 0)) * NT * 128 + row]);
    if (ml.y != 0.f) M = fmaxf(M, ml.x);
  }
  float acc[E] = {}, L = 0.f;
  for (long long i = c0; i <= c1; ++i) {
    const long long at = (2 * i + (i == c0 ? 1 : 0)) * NT * 128 + row;
    const float2 ml = __ldcg(&a.part_ml[at]);
    if (ml.y == 0.f) continue;
    const float f = tree_ex2(ml.x - M);
    L += f * ml.y;
    const float* p = a.part + at * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += f * __ldcg(p + e);
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  __nv_bfloat16* dst = a.o + w * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack_bf16x2(acc[e] * inv, acc[e + 1] * inv);
}

template <int D, bool QUANT, int NT>
static void tree_launch(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const TreeArgs& a, const KvView& c,
                        int grid, cudaStream_t s) {
  using Cfg = TreeCfg<D, QUANT, NT>;
  static bool set[64] = {};                  // a function's attributes are kept by device
  int dev = 0;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev >= 64 || !set[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(tree_attention_kernel<D, QUANT, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg::SMEM));
    if (dev < 64) set[dev] = true;
  }
  tree_attention_kernel<D, QUANT, NT><<<grid, Cfg::THREADS, Cfg::SMEM, s>>>(tq, tk, tv, a, c);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)(((long long)a.B * a.N * a.Hq + 3) / 4), 1, 1);
  cfg.blockDim = dim3(128, 1, 1);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, tree_combine_kernel<D>, a, c, grid, NT));
}

at::Tensor tree_attention(at::Tensor q, at::Tensor kc, at::Tensor vc, at::Tensor lens,
                             c10::optional<at::Tensor> parents, double scale, c10::optional<at::Tensor> ks,
                             c10::optional<at::Tensor> vs, at::Tensor err) {
  bool quant;
  const KvView c = kv_view(kc, vc, ks, vs, quant);
  TORCH_CHECK(q.dim() == 4 && q.scalar_type() == at::kBFloat16 && q.device() == kc.device(),
              "q: bfloat16 [B, N, Hq, D] on the caches' device");
  const int64_t B = kc.size(0), H = kc.size(1), T = kc.size(2), D = kc.size(3), N = q.size(1), Hq = q.size(2);
  TORCH_CHECK(q.size(0) == B && q.size(3) == D, "q: the caches' B and D");
  TORCH_CHECK(N >= 1 && N <= kTreeNodes, "1 to 64 nodes");
  TORCH_CHECK(H >= 1 && Hq >= 1 && Hq % H == 0, "the query heads: a multiple of the caches' heads");
  TORCH_CHECK(q.stride(3) == 1 && (B <= 1 || q.stride(0) % 8 == 0) && (N == 1 || q.stride(1) % 8 == 0) &&
                  (Hq == 1 || q.stride(2) % 8 == 0) && (reinterpret_cast<uintptr_t>(q.data_ptr()) & 15) == 0,
              "q: unit inner stride and 16-byte aligned rows");
  TORCH_CHECK((B <= 1 || q.stride(0) > 0) && (N == 1 || q.stride(1) > 0) && (Hq == 1 || q.stride(2) > 0), "q: no broadcast dimension");
  TreeArgs a{};
  a.lens = kv_ints(lens, "lens", kc.device(), B);
  a.parents = parents.has_value() ? kv_ints(*parents, "parents", kc.device(), B, N) : nullptr;
  TORCH_CHECK(B * N * Hq < (1LL << 31), "too many query rows");
  const int G = (int)(Hq / H);
  a.B = (int)B; a.N = (int)N; a.Hq = (int)Hq; a.Hkv = (int)H; a.G = G;
  // rows of a tile: nb nodes of gb heads each
  a.gb = std::min(G, 128);
  a.nb = std::min((int)N, 128 / a.gb);
  a.gg = (G + a.gb - 1) / a.gb;
  a.rt = (((int)N + a.nb - 1) / a.nb) * a.gg;
  const int NT = a.rt > 1 ? 2 : 1;           // two row tiles share each key / value tile
  a.rg = (a.rt + NT - 1) / NT;
  a.scale_log2 = std::max((float)(std::abs(scale) * 1.4426950408889634), 1e-30f);   // -inf * 0 is NaN
  a.neg = scale < 0;
  c10::cuda::CUDAGuard guard(kc.device());
  auto o = at::empty({B, N, Hq, D}, q.options());
  if (o.numel() == 0) return o;
  a.o = reinterpret_cast<__nv_bfloat16*>(o.data_ptr());
  a.err = err.data_ptr<int>();
  const int64_t most = B * H * a.rg * ((T + 127) / 128);
  TORCH_CHECK(most < (1LL << 36), "too much work for one call");
  const int grid = (int)std::min<int64_t>(num_sms(kc.device().index()), most);
  auto part = at::empty({(int64_t)2 * grid * NT * 128 * (D + 2)}, q.options().dtype(at::kFloat));
  a.part = part.data_ptr<float>();
  a.part_ml = reinterpret_cast<float2*>(a.part + (int64_t)2 * grid * NT * 128 * D);

  const uint64_t u = 2;
  const uint64_t qd[5] = {(uint64_t)D, (uint64_t)G, (uint64_t)N, (uint64_t)H, (uint64_t)B};
  const uint64_t qs[4] = {q.stride(2) * u, q.stride(1) * u, (uint64_t)G * q.stride(2) * u, q.stride(0) * u};
  const uint32_t qb[5] = {64, (uint32_t)a.gb, (uint32_t)a.nb, 1, 1};
  const CUtensorMap tq = make_tmap_nd(q.data_ptr(), CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, qd, qs, qb, CU_TENSOR_MAP_SWIZZLE_128B);
  const uint64_t kd[4] = {(uint64_t)D, (uint64_t)T, (uint64_t)H, (uint64_t)B};
  const uint64_t kst[3] = {(uint64_t)c.t, (uint64_t)c.h, (uint64_t)c.b};
  const uint32_t kb[4] = {quant ? (uint32_t)D : 64u, 128, 1, 1};
  const auto type = quant ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const auto sw = quant ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B;
  const CUtensorMap tk = make_tmap_nd(c.p[0], type, 4, kd, kst, kb, sw), tv = make_tmap_nd(c.p[1], type, 4, kd, kst, kb, sw);
  auto s = at::cuda::getCurrentCUDAStream();
#define TFB_TREE(DD, QQ) (NT == 1 ? tree_launch<DD, QQ, 1>(tq, tk, tv, a, c, grid, s) : tree_launch<DD, QQ, 2>(tq, tk, tv, a, c, grid, s))
  if (D == 128) { if (quant) TFB_TREE(128, true); else TFB_TREE(128, false); }
  else { if (quant) TFB_TREE(64, true); else TFB_TREE(64, false); }
#undef TFB_TREE
  return o;
}

}  // namespace tfb
