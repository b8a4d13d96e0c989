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
// Quantised caches: eight warps turn the e4m3 tiles into bf16 ones in shared memory, the
// row's power-of-two scale included (exactly, see kv_cache.cuh), since a product of a 16-bit
// and an 8-bit operand does not exist and q in 8 bits would lose half its significand.  (f16 tiles
// brought to the largest scale of 32 rows convert in a fifth of the instructions, but a small row
// beside a large one that the query does not see then loses its bits.)
//
// Up to 16 query rows a key/value head (8 of bf16 heads of 128) take the kernel of tree_attention_few.cuh.
//
// Measured on a B200 (calls replayed from a graph; the floor is the bytes at 6.54 TB/s or the
// products at 1.68 PFLOP/s).  64-node trees, 32 / 8 heads, 16 sequences of 4096 .. 8191 bf16 rows: 136 us
// of 65 (160 in a long loop, where the power cap holds the SMs at 1.6 GHz).  By clock stamps a CTA takes
// 193 to 234 thousand cycles, 211 in the mean, at 1.80 GHz: 84 half tiles of 2130 cycles, 1350 of them
// exponentials, and segment starts and ends; the slowest ends at 129 us, then comes the second kernel.
// Parts left out in a copy: 132 us without exponentials, 134 with an eighth of the products, 105 with
// neither, so the two hide each other, and the rest is loads, reads of TMEM and hand-overs.
// 24-node trees, 32 / 8 heads, 8 sequences of 32768 .. 65535 e4m3 rows: 375 us of 125 (391 in a long
// loop).  318 without conversion, 386 without exponentials, 340 without either, 317 without either and an
// eighth of the products: of these only the conversion counts.  By stamps a group is busy for 2100 of a
// tile's 3790 cycles, and some 1200 lie between one tile's P and its first step of the next.
// Tiles of 64 keys with deeper rings were slower (145 and 705 us).
//
// A row behind the context that no node uses may hold anything: its scores are masked, and its
// values are zeroed in shared memory before the product (0 * NaN is NaN).  A drafted row that is
// used but holds an infinity or a NaN (in e4m3: a NaN code, or the scale NaN) is zeroed likewise and
// added afterwards, entry by entry, to the nodes that see it.
// The reference has no decode path; the attention is the math of train.py:2564-2567.
#include <climits>

#include "kv_cache.cuh"

namespace tfb {

CUtensorMap make_tmap_nd(const void* ptr, CUtensorMapDataType type, int rank, const uint64_t* dims, const uint64_t* strides,
                         const uint32_t* box, CUtensorMapSwizzle swizzle);
int num_sms(int dev);

constexpr int kTreeNodes = 64;
constexpr uint32_t kTreePanel = 128u * 128u;   // bytes of one 64-column panel of 128 bf16 rows
constexpr int kSegRing = 8;                    // segments whose poison masks are kept
constexpr int kLineRing = 4;                   // segments whose ancestor masks are kept
constexpr int kLenCache = 128;                 // context lengths kept in shared memory (of larger batches: none)

struct TreeArgs {
  __nv_bfloat16* o;          // [B, N, Hq, D]
  const int* lens;
  const int* parents;        // null: a chain
  int B, N, Hq, Hkv, G;
  int gb, nb;                // heads and nodes of a 128-row tile
  int gg, rt, rg;            // head groups, row tiles and row groups (of NT tiles) a key/value head
  float scale_log2;          // |scale| log2(e), never 0
  int neg;                   // scale < 0
  float4* part;              // [2 * grid][NT][D / 4][128 rows] unnormalised partial outputs
  float2* part_ml;           // [2 * grid][NT * 128] their maximum (log2 units) and sum: (-inf, 0) where no score
                             // is above -inf, (inf, 0) for an unused node
  float2* pair_ml;           // [grid][128] group 1's, for group 0 (NT = 1)
  int* err;
};

// Context lengths, from shared memory where the batch is small enough.
struct TreeLens {
  const int* lens;
  const int* cache;           // null: read lens
  int n, tmax;
  __device__ __forceinline__ int len(int b) const { return cache ? cache[b] : max(0, min(lens[b], tmax)); }
  // key tiles of sequence b: its context and as many node rows as the cache has room for
  __device__ __forceinline__ int tiles(int b) const { return (int)((min((long long)len(b) + n, (long long)tmax) + 127) >> 7); }
};

// The key tiles of a CTA, in order: [pos, end) of the line of all tiles.
struct TreeIter {
  int pos, end, base;         // base: first tile of sequence b on the line
  int b, kt, units;           // kt: key tiles of sequence b; units: (head, row group) pairs
  int h, rgi, len, k, k0, k1; // present segment: head, row group, context length, key tile and its range
  int seg;                    // segments begun so far, less one

  // Present tile -> next one; false at the end.
  __device__ __forceinline__ bool next(const TreeLens& lens, int rg) {
    if (seg >= 0 && k + 1 < k1) {
      ++k;
      return true;
    }
    if (pos >= end) return false;
    while (pos >= base + kt * units) {
      base += kt * units;
      kt = lens.tiles(++b);
    }
    len = lens.len(b);
    const unsigned rel = (unsigned)(pos - base);
    const int u = (int)(rel / (unsigned)kt);
    k0 = k = (int)rel - u * kt;
    k1 = min(kt, k0 + (end - pos));
    h = u / rg;
    rgi = u - h * rg;
    pos += k1 - k0;
    ++seg;
    return true;
  }
  __device__ __forceinline__ bool first() const { return k == k0; }
  __device__ __forceinline__ bool last() const { return k + 1 == k1; }
};

// Start of CTA `cta` of `grid` on the line of tiles (warp-collective).  total * grid < 2^32.
__device__ __forceinline__ TreeIter tree_begin(const TreeArgs& a, const TreeLens& lens, int cta, int grid) {
  const int lane = threadIdx.x & 31;
  TreeIter it;
  it.units = a.Hkv * a.rg;
  int sum = 0;
  for (int b = lane; b < a.B; b += 32) sum += lens.tiles(b);
  const int total = __reduce_add_sync(0xffffffffu, sum) * it.units;
  grid = min(grid, total);                   // CTAs that have work
  it.pos = cta < grid ? (int)((unsigned)total * (unsigned)cta / (unsigned)grid) : total;
  it.end = cta < grid ? (int)((unsigned)total * (unsigned)(cta + 1) / (unsigned)grid) : total;
  it.base = 0;
  it.b = 0;
  it.seg = -1;
  it.k = it.k0 = it.k1 = 0;
  // the sequence in which pos lies
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int mine = b0 + lane < a.B ? lens.tiles(b0 + lane) * it.units : 0;
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const unsigned in = __ballot_sync(0xffffffffu, it.pos < it.base + inc);
    const int at = in ? __ffs(in) - 1 : 31;
    const int before = __shfl_sync(0xffffffffu, inc - mine, at);
    const int all = __shfl_sync(0xffffffffu, inc, 31);
    if (in || b0 + 32 >= a.B) {
      it.b = min(b0 + at, a.B - 1);
      it.base += before;
      break;
    }
    it.base += all;
  }
  it.kt = lens.tiles(it.b);
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
// 2^v of a pair on the FMA pipe, for v <= 8 (0 below -126): v = n + f, n the nearest integer (it
// lands in the low bits of v + 1.5 * 2^23), 2^f on [-1/2, 1/2] by a polynomial of degree 4 fitted
// here for the least relative error (2.7e-6), n added to its exponent.  A quarter of the
// exponentials goes this way, since the two groups' 128 a row pair are all that the MUFU unit
// of a sub-core does in 1024 cycles (bf16 caches: 132 instead of 135 us without any exponentials at
// all, so little is left; beside the conversion of quantised tiles the extra instructions cost
// more than they save, 376 against 350 us).  NaN stays NaN.
__device__ __forceinline__ float2 tree_exp2_pair(float2 v) {
  const float2 c = make_float2(fmaxf(v.x, -126.f), fmaxf(v.y, -126.f));
  const float2 t = __fadd2_rn(c, make_float2(12582912.f, 12582912.f));
  const float2 n = __fadd2_rn(t, make_float2(-12582912.f, -12582912.f));
  const float2 f = __fadd2_rn(c, make_float2(-n.x, -n.y));
  float2 p = __ffma2_rn(make_float2(0.009570102207362652f, 0.009570102207362652f), f, make_float2(0.05591785907745361f, 0.05591785907745361f));
  p = __ffma2_rn(p, f, make_float2(0.240247443318367f, 0.240247443318367f));
  p = __ffma2_rn(p, f, make_float2(0.6931217908859253f, 0.6931217908859253f));
  p = __ffma2_rn(p, f, make_float2(0.9999992847442627f, 0.9999992847442627f));
  const float x = __int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23));
  const float y = __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23));
  return make_float2(v.x >= -126.f ? x : v.x == v.x ? 0.f : v.x, v.y >= -126.f ? y : v.y == v.y ? 0.f : v.y);
}

// Low word of an operand's descriptor (128-byte swizzle; the high word is the same for all), and
// what a step of 16 along the contraction adds to it: 32 bytes within a 64-column panel of a
// K-major operand, 16 rows of 128 bytes of an MN-major one.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t tree_desc_k(uint32_t addr) { return ((addr >> 4) & 0x3fffu) | (1u << 16); }
__device__ __forceinline__ uint32_t tree_desc_mn(uint32_t addr) { return ((addr >> 4) & 0x3fffu) | ((kTreePanel >> 4) << 16); }
__host__ __device__ constexpr uint32_t tree_step_k(int kk) { return (uint32_t)(kk >> 2) * (kTreePanel >> 4) + (uint32_t)(kk & 3) * 2u; }
__host__ __device__ constexpr uint32_t tree_step_mn(int kk) { return (uint32_t)kk * 128u; }
__device__ __forceinline__ void tree_mma(uint32_t d, uint32_t alo, uint32_t blo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d), "r"(alo), "r"(blo), "r"(idesc), "r"(accumulate),
      "r"(kDescHi));
}
__device__ __forceinline__ void tree_mma_p(uint32_t d, uint32_t a_tmem, uint32_t blo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d), "r"(a_tmem), "r"(blo), "r"(idesc), "r"(accumulate),
      "r"(kDescHi));
}

// Bit 7 of every byte: whether that e4m3 code is one of the two NaNs.
__device__ __forceinline__ uint32_t code4_nan(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// 4 e4m3 codes -> 4 bf16 (two words), times m1.  The code's exponent and
// significand bits, moved to a bf16's place, are the value times 2^-120 (subnormals included),
// so a multiplication by 2^120 times the row's scale is all that is left; scales whose
// exponent does not fit that factor take a second one.  la, ha: the moved bits, 0x07f0 of a NaN code,
// which the multiplication would make +-480 times the scale.
__device__ __forceinline__ uint2 codes4(uint32_t x, __nv_bfloat162 m1, uint32_t& la, uint32_t& ha) {
  const uint32_t lo = __byte_perm(x, 0, 0x1404), hi = __byte_perm(x, 0, 0x3424);
  la = (lo >> 4) & 0x07f007f0u;
  ha = (hi >> 4) & 0x07f007f0u;
  uint32_t a = (lo & 0x80008000u) | la;
  uint32_t b = (hi & 0x80008000u) | ha;
  const __nv_bfloat162 u = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a), m1);
  const __nv_bfloat162 v = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&b), m1);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&u), *reinterpret_cast<const uint32_t*>(&v));
}
__device__ __forceinline__ __nv_bfloat162 bf16x2_bits(uint32_t h) {
  const uint32_t w = h | (h << 16);
  return *reinterpret_cast<const __nv_bfloat162*>(&w);
}

__device__ __forceinline__ void tree_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// Adds what is not finite in the drafted value rows `bad` (nodes that the query sees) to 16
// columns from `col` on; those entries were zeroed for the product.
template <bool QUANT>
__device__ __noinline__ void tree_add_bad(float (&f)[16], unsigned long long bad, const KvView& c, int b, int h, int len, int col) {
  for (; bad; bad &= bad - 1) {
    const long long t = (long long)len + __ffsll((long long)bad) - 1;
    const uint8_t* base = c.p[1] + b * c.b + h * c.h + t * c.t;
    if (QUANT) {                             // NaN codes, or all of them where the row's scale is NaN
      const bool all = c.s[1][b * c.sb + h * c.sh + t * c.st] == kScaleNan;
      for (int k = 0; k < 16; ++k)
        if (all || (base[col + k] & 0x7f) == 0x7f) f[k] = __int_as_float(0x7fffffff);
    } else {
      const __nv_bfloat16* row = reinterpret_cast<const __nv_bfloat16*>(base) + col;
      for (int k = 0; k < 16; ++k) {
        const float v = __bfloat162float(row[k]);
        if (!(fabsf(v) < INFINITY)) f[k] += v;
      }
    }
  }
}

// Mends the bf16 forms of NaN codes, which codes4 turns into +-480 times the scale, in a converting lane's part
// (16 codes from `src` on of every RPI-th row) of a warp's 32 rows, cw * 32 .. of the tile at `dst`.  off: the
// tile's first row from the first node's.  A NaN where a row is seen by all; in drafted value rows 0 and a bit in
// `poison`, for the nodes that see them.  Rows whose factor (`mine`, a row a lane) is 0 are nobody's.
template <int D>
__device__ __noinline__ void tree_fix_nan(const uint8_t* src, uint8_t* dst, int cw, uint32_t mine, int off, unsigned long long* poison) {
  constexpr int CH = D / 16, RPI = 32 / CH;
  const int lane = threadIdx.x & 31, ch = lane % CH;
#pragma unroll 1
  for (int i = 0; i < CH; ++i) {
    const int r32 = i * RPI + lane / CH, at = off + cw * 32 + r32;
    const bool zeroed = __shfl_sync(0xffffffffu, mine, r32) == 0;
    bool hit = false;
#pragma unroll 1
    for (int q = 0; q < 16; ++q)
      if ((src[i * RPI * D + q] & 0x7f) == 0x7f && !zeroed) {
        hit = true;
        *reinterpret_cast<uint16_t*>(dst + sw128_chunk_offset(cw * 32 + r32, 2 * (ch & 3) + (q >> 3)) + (q & 7) * 2) = at >= 0 ? 0 : 0x7fff;
      }
    if (hit && at >= 0) atomicOr(poison, 1ull << at);
  }
}

template <int D, bool QUANT, int NT>
struct TreeCfg {
  static constexpr uint32_t TILE = 128u * D * 2u;
  static constexpr uint32_t RAW = 128u * D;
  static constexpr int NK = QUANT ? 2 : 3;                      // bf16 key tiles
  static constexpr int NV = QUANT ? 3 - NT : 4 - NT;            // bf16 value tiles
  static constexpr int NR = QUANT ? 2 : 0;                      // e4m3 tiles of either kind
  static constexpr int AUX = QUANT ? 8 : 1;                     // warps that convert, or clear unused rows
  static constexpr int THREADS = 32 * (3 + 8 + AUX);
  static constexpr int BARS = 48;
  static constexpr size_t SMEM = (NT + NK + NV) * TILE + 2 * NR * RAW + BARS * 8 + kSegRing * 8 + kLineRing * kTreeNodes * 8 + kLenCache * 4 + 16;
};
static_assert(TreeCfg<128, false, 1>::SMEM <= 232448 && TreeCfg<128, true, 1>::SMEM <= 232448 && TreeCfg<128, false, 2>::SMEM <= 232448 &&
              TreeCfg<128, true, 2>::SMEM <= 232448, "shared memory");

// Roles: warp 0 loads (TMA: one lane keys and queries, one lane values), warps 1 and 2 issue the
// products of a group each (one warp for both was busy with nothing else: 158 against 143 us), two
// groups of four warps run the softmax, the rest converts quantised tiles or clears unused rows of
// value tiles.  A group works
// through half tiles of 64 keys:
//   NT = 2: group t has row tile t and takes both halves of every key tile in turn;
//   NT = 1: both groups have the one row tile, group t half t of every key tile, each with a
//           maximum, sum and O of its own; at the end of a segment group 0 adds group 1's.
// A group's S is double-buffered in TMEM: S(i + 2) is issued behind P(i) V(i), so the softmax never
// waits for a product, and its 64 scores a row stay in registers from the maximum to the
// exponentials.  (With 128-key tiles and one S a group, each tile's chain S -> softmax -> P V ran
// serially, 4300 cycles for what the softmax needs 2300 of.)
// TMEM: group t's S at 128 t + 64 (i & 1), P over its first 32 columns; O at 256 + 128 t.
template <int D, bool QUANT, int NT>
__global__ void __launch_bounds__(TreeCfg<D, QUANT, NT>::THREADS, 1)
    tree_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                          const __grid_constant__ CUtensorMap tmV, const TreeArgs a, const __grid_constant__ KvView c) {
  using Cfg = TreeCfg<D, QUANT, NT>;
  constexpr uint32_t TILE = Cfg::TILE, RAW = Cfg::RAW;
  constexpr int NK = Cfg::NK, NV = Cfg::NV, NR = Cfg::NR;
  constexpr int PANELS = D / 64;
  constexpr int NH = NT;                       // half tiles of a key tile that a group takes
  constexpr uint32_t IDESC_S = umma_idesc_bf16(128, 64, false, false);
  constexpr uint32_t IDESC_O = umma_idesc_bf16(128, D, false, true);

  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {         // the swizzled tiles need it
    if (threadIdx.x == 0) atomicOr(a.err, ERR_BAD_ARG);
    return;
  }
  uint8_t* sQ = smem;                          // [NT] tiles
  uint8_t* sK = sQ + NT * TILE;                // [NK]
  uint8_t* sV = sK + NK * TILE;                // [NV]
  uint8_t* sRaw = sV + NV * TILE;              // [2][NR]: keys, values
  uint64_t* bars = reinterpret_cast<uint64_t*>(sRaw + 2 * NR * RAW);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* k_full = bars + 2;                 // [NK <= 3]
  uint64_t* k_empty = bars + 5;                // [NK]
  uint64_t* v_full = bars + 8;                 // [NV <= 3]
  uint64_t* v_empty = bars + 11;               // [NV]
  uint64_t* v_ready = bars + 14;               // [NV] value tiles whose unused rows are cleared (not QUANT)
  uint64_t* raw_full = bars + 17;              // [2][NR]
  uint64_t* raw_empty = bars + 21;             // [2][NR]
  uint64_t* s_full = bars + 25;                // [2 groups][2 buffers]
  uint64_t* p_full = bars + 29;                // [2][2]
  uint64_t* pv_done = bars + 33;               // [2][2]
  uint64_t* line_full = bars + 37;             // [kLineRing]
  uint64_t* ml_full = bars + 41;               // group 1's maximum and sum are written, its O is done (NT = 1)
  uint64_t* o_free = bars + 42;                // group 0 has read them (NT = 1)
  uint64_t* drain = bars + 43;                 // [2]
  unsigned long long* s_poison = reinterpret_cast<unsigned long long*>(bars + Cfg::BARS);   // [kSegRing] drafted rows not finite
  unsigned long long* s_line = s_poison + kSegRing;                                         // [kLineRing][kTreeNodes]
  int* s_len = reinterpret_cast<int*>(s_line + kLineRing * kTreeNodes);                     // [kLenCache]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_len + kLenCache);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 2);
    for (int i = 0; i < NK; ++i) {
      mbar_init(&k_full[i], QUANT ? 128 : 1);
      mbar_init(&k_empty[i], 2);
    }
    for (int i = 0; i < NV; ++i) {
      mbar_init(&v_full[i], QUANT ? 128 : 1);
      mbar_init(&v_empty[i], 2);
      mbar_init(&v_ready[i], 32);
    }
    for (int i = 0; i < 2 * NR; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], 128);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&pv_done[i], 1);
    }
    for (int i = 0; i < kLineRing; ++i) mbar_init(&line_full[i], 32);
    mbar_init(ml_full, 128);
    mbar_init(o_free, 128);
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
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
  const TreeLens lens{a.lens, a.B <= kLenCache ? s_len : nullptr, a.N, c.tmax};
  if (threadIdx.x >= 64)
    for (int i = (int)threadIdx.x - 64; i < a.B && i < kLenCache; i += (int)blockDim.x - 64) s_len[i] = max(0, min(a.lens[i], c.tmax));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch_dependents();
  TreeIter it = tree_begin(a, lens, (int)blockIdx.x, (int)gridDim.x);
  const int tiles = it.end - it.pos;           // of this CTA
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------------ loads: lane 0 keys and queries, lane 1 values
    if (lane < 2 && tiles > 0) {
      const int v = lane, R = QUANT ? NR : v ? NV : NK;
      const CUtensorMap* map = v ? &tmV : &tmK;
      uint64_t* const full = QUANT ? raw_full + v * NR : v ? v_full : k_full;
      uint64_t* const empty = QUANT ? raw_empty + v * NR : v ? v_empty : k_empty;
      uint8_t* const dst = QUANT ? sRaw + v * NR * RAW : v ? sV : sK;
      bool ok = true;
      int g = 0, segs = 0;                     // tiles begun, query tiles begun
      auto queries = [&](const TreeIter& t) -> bool {
        if (segs > 0 && !mbar_wait(q_empty, (segs + 1) & 1, abort_flag, a.err, ERR_TIMEOUT_PRODUCER)) return false;
        mbar_arrive_expect_tx(q_full, (uint32_t)(NT * PANELS * a.gb * a.nb) * 128u);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const int rt = t.rgi * NT + i;
          const int ng = rt / a.gg, hg = rt - ng * a.gg;
#pragma unroll
          for (int p = 0; p < PANELS; ++p)
            tma_load_5d(sQ + i * TILE + p * kTreePanel, &tmQ, q_full, p * 64, hg * a.gb, ng * a.nb, t.h, t.b);
        }
        ++segs;
        return true;
      };
      while (it.next(lens, a.rg)) {
        if (v == 0 && it.first() && !queries(it)) { ok = false; break; }
        const int slot = g % R;
        if (g >= R && !mbar_wait(&empty[slot], ((g / R) + 1) & 1, abort_flag, a.err, ERR_TIMEOUT_PRODUCER)) { ok = false; break; }
        mbar_arrive_expect_tx(&full[slot], QUANT ? RAW : TILE);
        if constexpr (QUANT) {
          tma_load_4d(dst + slot * RAW, map, &full[slot], 0, it.k * 128, it.h, it.b);
        } else {
#pragma unroll
          for (int p = 0; p < PANELS; ++p)
            tma_load_4d(dst + slot * TILE + p * kTreePanel, map, &full[slot], p * 64, it.k * 128, it.h, it.b);
        }
        ++g;
      }
      if (!ok) {   // let the copies in flight land before the CTA ends
        const unsigned long long t0 = globaltimer_ns();
        for (int i = max(0, g - R); i < g; ++i)
          while (!mbar_try_wait(&full[i % R], (i / R) & 1))
            if (globaltimer_ns() - t0 > 100000000ull) break;
        if (segs > 0)
          while (!mbar_try_wait(q_full, (segs - 1) & 1))
            if (globaltimer_ns() - t0 > 100000000ull) break;
      }
    }
  } else if (warp <= 2) {
    // ------------------------------------------------------------------ products of group t
    if (tiles > 0) {   // the whole warp keeps the schedule (in uniform registers), one lane issues
      const int t = warp - 1;
      bool ok = true, more = true;
      TreeIter si = it, pi = it;               // tiles of the scores and of the outputs
      int ks = NK - 1, vs = NV - 1;            // their places in the rings, and the phases of those
      uint32_t kph = 1, vph = 1;
      const uint32_t qd = tree_desc_k(smem_u32(sQ)) + (NT == 1 ? 0u : (uint32_t)t * (TILE >> 4));
      const uint32_t kd0 = tree_desc_k(smem_u32(sK)), vd0 = tree_desc_mn(smem_u32(sV));
      const uint32_t tS = tmem + t * 128, tO = tmem + 256 + t * 128;
      uint64_t* const in_v = QUANT ? v_full : v_ready;
      // the scores of the group's half tile i; true also at the end
      auto scores = [&](int i) -> bool {
        const int half = NT == 1 ? t : i & 1, buf = i & 1;
        if (NH == 1 || half == 0) {
          more = more && si.next(lens, a.rg);
          if (more) {
            if (++ks == NK) { ks = 0; kph ^= 1; }
            if (si.first() && !mbar_wait_warp(q_full, si.seg & 1, abort_flag, a.err, ERR_TIMEOUT_MMA)) return false;
            if (!mbar_wait_warp(&k_full[ks], kph, abort_flag, a.err, ERR_TIMEOUT_MMA)) return false;
            tc_fence_after();
          }
        }
        if (!more) return true;
        const uint32_t kd = kd0 + (uint32_t)ks * (TILE >> 4) + (uint32_t)half * (8192u >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            tree_mma(tS + buf * 64, qd + tree_step_k(kk), kd + tree_step_k(kk), IDESC_S, kk > 0 ? 1u : 0u);
          umma_commit(&s_full[t * 2 + buf]);
          if (NH == 1 || half == 1) {
            umma_commit(&k_empty[ks]);
            if (si.last()) umma_commit(q_empty);
          }
        }
        __syncwarp();
        return true;
      };
      auto outputs = [&](int i) -> bool {
        const int half = NT == 1 ? t : i & 1, buf = i & 1;
        if (NH == 1 || half == 0) {
          pi.next(lens, a.rg);
          if (++vs == NV) { vs = 0; vph ^= 1; }
          if (!mbar_wait_warp(&in_v[vs], vph, abort_flag, a.err, ERR_TIMEOUT_MMA)) return false;
        }
        if (!mbar_wait_warp(&p_full[t * 2 + buf], (i >> 1) & 1, abort_flag, a.err, ERR_TIMEOUT_MMA)) return false;
        tc_fence_after();
        const uint32_t vd = vd0 + (uint32_t)vs * (TILE >> 4) + (uint32_t)half * tree_step_mn(4);
        const uint32_t add = pi.first() && (NH == 1 || half == 0) ? 0u : 1u;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) tree_mma_p(tO, tS + buf * 64 + kk * 8, vd + tree_step_mn(kk), IDESC_O, kk > 0 ? 1u : add);
          if (NH == 1 || half == 1) umma_commit(&v_empty[vs]);
          umma_commit(&pv_done[t * 2 + buf]);
        }
        __syncwarp();
        return true;
      };
      ok = scores(0) && scores(1);
      for (int i = 0; i < tiles * NH && ok; ++i) ok = outputs(i) && scores(i + 2);
      if (!ok) {
        *abort_flag = 1;
        if (elect_one()) umma_commit(&drain[t]);
        __syncwarp();
        const unsigned long long t0 = globaltimer_ns();
        while (!mbar_try_wait(&drain[t], 0))
          if (globaltimer_ns() - t0 > 100000000ull) break;
      }
    }
  } else if (warp < 11) {
    // ------------------------------------------------------------------ softmax, group t
    const int t = (warp - 3) >> 2, q4 = warp & 3, r = q4 * 32 + lane;
    const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
    const uint32_t tO = tmem + 256 + t * 128 + lane_off;
    const float cl = a.scale_log2;
    const int rn = r / a.gb, rh = r - rn * a.gb;
    float m_run = -INFINITY, l = 0.f;
    unsigned long long line = 0;
    int n = 0, head = 0, i = 0;                // i: half tile of the group
    bool live = false, warp_live = false, ok = true;
    while (ok && it.next(lens, a.rg)) {
      if (it.first()) {
        const int rt = it.rgi * NT + (NT == 1 ? 0 : t);
        const int ng = rt / a.gg, hg = rt - ng * a.gg;
        n = ng * a.nb + rn;
        head = hg * a.gb + rh;
        live = rn < a.nb && n < a.N && head < a.G && rt < a.rt;
        warp_live = __any_sync(0xffffffffu, live);
        const int lr = it.seg & (kLineRing - 1);
        if (!mbar_wait_warp(&line_full[lr], (it.seg / kLineRing) & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) { ok = false; break; }
        line = live ? s_line[lr * kTreeNodes + n] : 0;
        m_run = -INFINITY;
        l = 0.f;
      }
#pragma unroll 1
      for (int hf = 0; hf < NH; ++hf, ++i) {
        const int half = NT == 1 ? t : hf, buf = i & 1, ph = (i >> 1) & 1;
        const uint32_t tS = tmem + t * 128 + buf * 64 + lane_off;
        // P(i - 2) V was issued before S(i): the second wait only keeps count of its barrier's phases
        ok = mbar_wait(&s_full[t * 2 + buf], ph, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE) &&
             (i < 2 || mbar_wait(&pv_done[t * 2 + buf], ph ^ 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE));
        ok = __all_sync(0xffffffffu, ok) != 0;
        if (!ok) break;
        tc_fence_after();
        if (warp_live) {
          const int off = it.k * 128 + half * 64 - it.len;   // of the first key from the first node's row
          float x[64];
          {
            uint32_t* xr = reinterpret_cast<uint32_t*>(x);
            __syncwarp();
            tmem_ld_32x32b_x32(tS, *reinterpret_cast<uint32_t(*)[32]>(xr));
            tmem_ld_32x32b_x32(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(xr + 32));
            tmem_ld_wait();
          }
          if (a.neg) {
#pragma unroll
            for (int k = 0; k < 64; ++k) x[k] = -x[k];
          }
          if (off + 64 > 0) {
            const uint32_t w0 = tree_word(line, off), w1 = tree_word(line, off + 32);
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              if (!((w0 >> k) & 1u)) x[k] = -INFINITY;
              if (!((w1 >> k) & 1u)) x[32 + k] = -INFINITY;
            }
          }
          float m4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
          for (int k = 4; k < 64; k += 8)
#pragma unroll
            for (int j = 0; j < 4; ++j) m4[j] = fmaxf(fmaxf(m4[j], x[k + j]), k + 4 < 64 ? x[k + 4 + j] : x[k + j]);
          const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * cl;
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
          uint32_t p[32];
#pragma unroll
          for (int k = 0; k < 64; k += 2) {
            const float2 v = __ffma2_rn(make_float2(x[k], x[k + 1]), c2, nm2);
            const float2 e = QUANT || k < 48 ? make_float2(tree_ex2(v.x), tree_ex2(v.y)) : tree_exp2_pair(v);
            p[k >> 1] = pack_bf16x2(e.x, e.y);   // P in 8 bits of significand for the product, its sum in 32 bits
            sum[(k >> 1) & 1] = __fadd2_rn(sum[(k >> 1) & 1], e);
          }
          __syncwarp();
          tmem_st_32x32b_x32(tS, p);
          const float2 s2 = __fadd2_rn(sum[0], sum[1]);
          l = l * alpha + (s2.x + s2.y);
          if (!(it.first() && hf == 0) && __any_sync(0xffffffffu, grow)) {
            if (!mbar_wait_warp(&pv_done[t * 2 + (buf ^ 1)], ((i - 1) >> 1) & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) { ok = false; break; }
            tc_fence_after();
#pragma unroll 1
            for (int cc = 0; cc < D / 32; ++cc) {
              uint32_t o[32];
              __syncwarp();
              tmem_ld_32x32b_x32(tO + cc * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
              tmem_st_32x32b_x32(tO + cc * 32, o);
            }
          }
          tmem_st_wait();
          tc_fence_before();
        }
        // group 1's O of the segment before is still to be read
        if (NT == 1 && t == 1 && it.first() && it.seg > 0 &&
            !mbar_wait_warp(o_free, (it.seg - 1) & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) { ok = false; break; }
        mbar_arrive(&p_full[t * 2 + buf]);
      }
      if (!ok || !it.last()) continue;
      // end of the segment: O is complete
      if (!mbar_wait_warp(&pv_done[t * 2 + ((i - 1) & 1)], ((i - 1) >> 1) & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) { ok = false; break; }
      tc_fence_after();
      float2* other = a.pair_ml + (long long)blockIdx.x * 128 + r;
      if (NT == 1 && t == 1) {
        *other = make_float2(m_run, l);
        tc_fence_before();
        mbar_arrive(ml_full);
        continue;
      }
      float f0 = 1.f, f1 = 0.f;
      if constexpr (NT == 1) {
        if (!mbar_wait_warp(ml_full, it.seg & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) { ok = false; break; }
        tc_fence_after();
        const volatile float2* ov = other;
        const float2 ml = make_float2(ov->x, ov->y);
        // the two halves at the larger of their references; one that saw nothing counts nothing
        const float mm = l == 0.f ? ml.x : ml.y == 0.f ? m_run : fmaxf(m_run, ml.x);
        f0 = l == 0.f ? 0.f : tree_ex2(m_run - mm);
        f1 = ml.y == 0.f ? 0.f : tree_ex2(ml.x - mm);
        l = (l == 0.f ? 0.f : l * f0) + (ml.y == 0.f ? 0.f : ml.y * f1);
        m_run = mm;
      }
      if (warp_live) {
        const bool whole = it.k0 == 0 && it.k1 == it.kt;
        const long long slot = 2LL * blockIdx.x + (it.k0 == 0 ? 1 : 0);
        const float inv = line != 0 ? 1.f / l : 0.f;   // l = 0: all scores are -inf, and 0 / 0 is NaN
        const unsigned long long bad = s_poison[it.seg & (kSegRing - 1)] & line;
        __nv_bfloat16* dst = a.o + (((long long)it.b * a.N + n) * a.Hq + it.h * a.G + head) * D;
        float4* pd = a.part + (slot * NT + (NT == 1 ? 0 : t)) * (D / 4) * 128 + r;
        // a short loop: this code runs once a segment, and fetching it costs more than running it
#pragma unroll 1
        for (int cc = 0; cc < D / 16; ++cc) {
          uint32_t o[16], o1[16];
          float f[16];
          __syncwarp();
          tree_ld16(tO + cc * 16, o);
          if constexpr (NT == 1) tree_ld16(tO + 128 + cc * 16, o1);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            f[k] = __uint_as_float(o[k]) * f0;       // the factors may be 0: a NaN stays
            if constexpr (NT == 1) f[k] += __uint_as_float(o1[k]) * f1;
            if (line == 0) f[k] = 0.f;
          }
          if (bad) tree_add_bad<QUANT>(f, bad, c, it.b, it.h, it.len, cc * 16);
          if (!live) continue;
          if (whole) {
            uint4* d4 = reinterpret_cast<uint4*>(dst + cc * 16);
#pragma unroll
            for (int k = 0; k < 2; ++k)
              d4[k] = make_uint4(pack_bf16x2(f[8 * k] * inv, f[8 * k + 1] * inv), pack_bf16x2(f[8 * k + 2] * inv, f[8 * k + 3] * inv),
                                 pack_bf16x2(f[8 * k + 4] * inv, f[8 * k + 5] * inv), pack_bf16x2(f[8 * k + 6] * inv, f[8 * k + 7] * inv));
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) pd[(cc * 4 + k) * 128] = make_float4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
          }
        }
        if (live && !whole) a.part_ml[(slot * NT + (NT == 1 ? 0 : t)) * 128 + r] = line != 0 ? make_float2(m_run, l) : make_float2(INFINITY, 0.f);
      }
      tc_fence_before();
      if (NT == 1) mbar_arrive(o_free);
    }
  } else {
    // ------------------------------------------------------------------ e4m3 -> bf16, unused rows
    const int tid = (int)threadIdx.x - 352;
    unsigned long long used = 0;
    // a value tile's segment (warp-collective): which drafted rows are used, and the lines for the softmax
    auto enter = [&](const TreeIter& v, bool publish) {
      unsigned long long m0, m1;
      tree_lines(a.parents ? a.parents + (long long)v.b * a.N : nullptr, a.N, c.tmax - v.len, m0, m1);
      used = used_nodes(m0, m1);
      if (publish) {
        const int lr = v.seg & (kLineRing - 1);
        s_line[lr * kTreeNodes + lane] = m0;
        s_line[lr * kTreeNodes + 32 + lane] = m1;
        if (lane == 0) s_poison[(v.seg + 3) & (kSegRing - 1)] = 0;   // last used five segments ago
        mbar_arrive(&line_full[lr]);
      }
    };
    if constexpr (!QUANT) {
      constexpr int CH = D / 8;                 // 16-byte chunks a row
      for (int g = 0; it.next(lens, a.rg); ++g) {
        if (it.first()) enter(it, true);
        const int slot = g % NV;
        if (!mbar_wait_warp(&v_full[slot], (g / NV) & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) break;
        const int off = it.k * 128 - it.len;
        if (off + 128 > 0) {
          uint8_t* tile = sV + slot * TILE;
          unsigned long long bad = 0;
          const int ch = lane % CH, r0 = max(0, -off);
          const int nodes = min(128, max(r0, a.N - off));      // rows from r0 to here are nodes', those behind nobody's
          auto at = [&](int row) { return reinterpret_cast<uint4*>(tile + (ch >> 3) * kTreePanel + sw128_chunk_offset(row, ch & 7)); };
#pragma unroll 8
          for (int row = nodes + lane / CH; row < 128; row += 32 / CH) *at(row) = make_uint4(0, 0, 0, 0);
#pragma unroll 4
          for (int row = r0 + lane / CH; row < nodes; row += 32 / CH) {
            const int j = row + off;
            uint4 u = *at(row);
            uint32_t* w = reinterpret_cast<uint32_t*>(&u);
            bool hit = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if ((w[i] & 0x7f80u) == 0x7f80u) { w[i] &= 0xffff0000u; hit = true; }
              if ((w[i] & 0x7f800000u) == 0x7f800000u) { w[i] &= 0xffffu; hit = true; }
            }
            if (!((used >> j) & 1)) u = make_uint4(0, 0, 0, 0);
            else if (hit) bad |= 1ull << j;
            if (hit || !((used >> j) & 1)) *at(row) = u;
          }
          const uint32_t lo = __reduce_or_sync(0xffffffffu, (uint32_t)bad), hi = __reduce_or_sync(0xffffffffu, (uint32_t)(bad >> 32));
          if (lane == 0 && (lo | hi)) s_poison[it.seg & (kSegRing - 1)] |= ((unsigned long long)hi << 32) | lo;
          fence_proxy_async_smem();
        }
        mbar_arrive(&v_ready[slot]);
      }
    } else {
      // four warps convert the keys, four the values, 32 neighbouring rows of a tile each: a lane
      // looks after one row's scale, fetched while the tile before is converted, and has 16 codes of
      // every RPI-th row.  The loop stays short on purpose: unrolled over all rows it ran out of the
      // instruction caches (3.3 of 11.7 warps stalled on that; 525 against 375 us).
      constexpr int CH = D / 16, RPI = 32 / CH;             // 16-code chunks a row, rows an iteration
      const int v = tid >> 7, cw = (tid >> 5) & 3, ch = lane % CH, own = cw * 32 + lane;
      const int R = v ? NV : NK;
      uint64_t* const out_full = v ? v_full : k_full;
      uint64_t* const out_empty = v ? v_empty : k_empty;
      const uint8_t* sb = v ? c.s[1] : c.s[0];
      uint32_t ahead = 127u;
      TreeIter nx = it;                         // one tile ahead of `it`
      auto scale = [&]() {
        const int row = nx.k * 128 + own;
        ahead = row < c.tmax ? sb[nx.b * c.sb + nx.h * c.sh + (long long)row * c.st] : 127u;
      };
      if (nx.next(lens, a.rg)) scale();
      int rslot = NR - 1, slot = R - 1;
      uint32_t rph = 1, ph = 0;
      for (int g = 0; it.next(lens, a.rg); ++g) {
        if (it.first() && v) enter(it, tid == 128 + lane);
        const int j = it.k * 128 - it.len + own;            // the lane's row from the first node's
        const uint32_t e = ahead;
        // the row's factor: 2^120 times its scale; scales above 2^7 take a second one
        uint32_t mine = e == (uint32_t)kScaleNan ? 0x7fffu : min(e + 120u, 254u) << 7;
        if (v && j >= 0) {                                  // behind the context: 0 for a row that nothing may see
          const bool seen = j < kTreeNodes && ((used >> j) & 1);
          if (seen && e == (uint32_t)kScaleNan) atomicOr(&s_poison[it.seg & (kSegRing - 1)], 1ull << j);
          if (!seen || e == (uint32_t)kScaleNan) mine = 0;
        }
        const uint32_t second = e > 134u && e != (uint32_t)kScaleNan ? (e - 7u) << 7 : 0x3f80u;
        if (nx.next(lens, a.rg)) scale();
        if (++rslot == NR) { rslot = 0; rph ^= 1; }
        if (++slot == R) { slot = 0; ph ^= 1; }
        if (!mbar_wait_warp(&raw_full[v * NR + rslot], rph, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) break;
        if (g >= R && !mbar_wait_warp(&out_empty[slot], ph, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) break;
        const uint8_t* src = sRaw + (v * NR + rslot) * RAW + (cw * 32 + lane / CH) * D + ch * 16;
        uint8_t* dst = (v ? sV : sK) + slot * TILE + (ch >> 2) * kTreePanel;
        // the two panels' lanes store their two chunks in opposite order: no bank is hit twice
        const bool swap = ch >= 4;
        const int c0 = 2 * (ch & 3) + (swap ? 1 : 0);
        const bool wide = __any_sync(0xffffffffu, second != 0x3f80u);
        // the largest codes: looking for NaNs costs 335 against 319 us (8 sequences of 32768 .. 65535 rows, 32 / 8
        // heads, 24 nodes; 341 with what mends them in line, 349 by a carry trick on the codes)
        uint32_t top = 0;
#pragma unroll 2
        for (int i = 0; i < CH; ++i) {
          const uint4 u = *reinterpret_cast<const uint4*>(src + i * RPI * D);
          const __nv_bfloat162 f = bf16x2_bits(__shfl_sync(0xffffffffu, mine, i * RPI + lane / CH));
          uint32_t m[8];
          const uint2 p0 = codes4(u.x, f, m[0], m[1]), p1 = codes4(u.y, f, m[2], m[3]), p2 = codes4(u.z, f, m[4], m[5]), p3 = codes4(u.w, f, m[6], m[7]);
          top = __vimax3_u16x2(__vimax3_u16x2(m[0], m[1], m[2]), __vimax3_u16x2(m[3], m[4], m[5]), __vimax3_u16x2(top, m[6], m[7]));
          const uint4 o0 = make_uint4(p0.x, p0.y, p1.x, p1.y), o1 = make_uint4(p2.x, p2.y, p3.x, p3.y);
          const int row = cw * 32 + i * RPI + lane / CH;
          *reinterpret_cast<uint4*>(dst + sw128_chunk_offset(row, c0)) = swap ? o1 : o0;
          *reinterpret_cast<uint4*>(dst + sw128_chunk_offset(row, c0 ^ 1)) = swap ? o0 : o1;
        }
        if (wide) {
#pragma unroll 1
          for (int i = 0; i < 2 * CH; ++i) {
            const __nv_bfloat162 f = bf16x2_bits(__shfl_sync(0xffffffffu, second, (i >> 1) * RPI + lane / CH));
            uint32_t* w = reinterpret_cast<uint32_t*>(dst + sw128_chunk_offset(cw * 32 + (i >> 1) * RPI + lane / CH, c0 ^ (i & 1)));
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[q]), f);
              w[q] = *reinterpret_cast<const uint32_t*>(&y);
            }
          }
        }
        if (__any_sync(0xffffffffu, max(top >> 16, top & 0xffffu) == 0x07f0u)) {
          tree_fix_nan<D>(src, dst, cw, mine, v != 0 ? it.k * 128 - it.len : INT_MIN, &s_poison[it.seg & (kSegRing - 1)]);
        }
        fence_proxy_async_smem();
        mbar_arrive(&out_full[slot]);
        mbar_arrive(&raw_empty[v * NR + rslot]);
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

}  // namespace tfb

#include "tree_attention_few.cuh"

namespace tfb {

// Adds the parts of the units that more than one CTA worked on.  A CTA has RP neighbouring rows
// of a row tile (RP: the rows of the tile, at most 32, rounded up to a power of two); the lanes of
// a warp are RP rows x 32 / RP parts, its warps share the D / 4 columns of four.  Parts are added
// lane by lane and then by a fixed tree over the lanes, so the order never changes.
template <int D>
__global__ void __launch_bounds__(128) tree_combine_kernel(const TreeArgs a, const KvView c, int grid, int NT, int RP, int blocks) {
  constexpr int Q = D / 16;                  // columns of four a warp
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blk = (int)(blockIdx.x % blocks);
  long long u = blockIdx.x / blocks;
  const int rt = (int)(u % a.rt);
  u /= a.rt;
  const int h = (int)(u % a.Hkv), b = (int)(u / a.Hkv), units = a.Hkv * a.rg;
  const TreeLens lens{a.lens, nullptr, a.N, c.tmax};
  int all = 0, before = 0;
  for (int i = lane; i < a.B; i += 32) {
    const int k = lens.tiles(i);
    all += k;
    if (i < b) before += k;
  }
  all = __reduce_add_sync(0xffffffffu, all);
  before = __reduce_add_sync(0xffffffffu, before);
  const unsigned W = (unsigned)(all * units), kt = (unsigned)lens.tiles(b), G = min((unsigned)grid, W);
  const unsigned p0 = (unsigned)(before * units) + (unsigned)(h * a.rg + rt / NT) * kt;
  const int c0 = (int)(((p0 + 1) * G - 1) / W), c1 = (int)(((p0 + kt) * G - 1) / W);   // CTAs that own the unit's ends
  griddep_wait();                            // every thread: this grid ends after the one before it
  if (c0 == c1) return;                      // one CTA had the whole unit and wrote it
  const int PS = 32 / RP, ps = lane / RP, r = blk * RP + lane % RP;
  const int ng = rt / a.gg, hg = rt - ng * a.gg, rn = r / a.gb, rh = r - rn * a.gb;
  const int n = ng * a.nb + rn, head = hg * a.gb + rh;
  const bool live = r < 128 && rn < a.nb && n < a.N && head < a.G;
  // CTA c0 ends with this unit's first part (slot 1), the others begin with theirs (slot 0)
  auto place = [&](int i) { return (2LL * i + (i == c0 ? 1 : 0)) * NT + rt % NT; };
  float M = -INFINITY;
  if (live)
    for (int i = c0 + ps; i <= c1; i += PS) {
      const float2 ml = __ldcg(&a.part_ml[place(i) * 128 + r]);
      M = fmaxf(M, ml.x);
    }
  for (int o = RP; o < 32; o *= 2) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  float4 acc[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) acc[q] = make_float4(0.f, 0.f, 0.f, 0.f);
  float L = 0.f;
  if (live) {
#pragma unroll 2
    for (int i = c0 + ps; i <= c1; i += PS) {
      const float2 ml = __ldcg(&a.part_ml[place(i) * 128 + r]);
      const float4* p = a.part + (place(i) * (D / 4) + warp * Q) * 128 + r;
      float4 v[Q];
#pragma unroll
      for (int q = 0; q < Q; ++q) v[q] = __ldcg(p + q * 128);
      const float f = ml.y == 0.f ? 0.f : tree_ex2(ml.x - M);   // 0: the row saw nothing there, or -inf only
      L += f * ml.y;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        acc[q].x += f * v[q].x; acc[q].y += f * v[q].y; acc[q].z += f * v[q].z; acc[q].w += f * v[q].w;
      }
    }
  }
  for (int o = RP; o < 32; o *= 2) {
    L += __shfl_xor_sync(0xffffffffu, L, o);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      acc[q].x += __shfl_xor_sync(0xffffffffu, acc[q].x, o);
      acc[q].y += __shfl_xor_sync(0xffffffffu, acc[q].y, o);
      acc[q].z += __shfl_xor_sync(0xffffffffu, acc[q].z, o);
      acc[q].w += __shfl_xor_sync(0xffffffffu, acc[q].w, o);
    }
  }
  if (!live || ps != 0) return;
  const bool used = !(L == 0.f && M == INFINITY);
  const float inv = used ? 1.f / L : 0.f;    // L = 0: all scores are -inf, and 0 / 0 is NaN
  if (!used) {
#pragma unroll
    for (int q = 0; q < Q; ++q) acc[q] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __nv_bfloat16* dst = a.o + (((long long)b * a.N + n) * a.Hq + h * a.G + head) * D + warp * Q * 4;
#pragma unroll
  for (int q = 0; q < Q; q += 2) {
    uint4 w;
    w.x = pack_bf16x2(acc[q].x * inv, acc[q].y * inv);
    w.y = pack_bf16x2(acc[q].z * inv, acc[q].w * inv);
    w.z = pack_bf16x2(acc[q + 1].x * inv, acc[q + 1].y * inv);
    w.w = pack_bf16x2(acc[q + 1].z * inv, acc[q + 1].w * inv);
    *reinterpret_cast<uint4*>(dst + 4 * q) = w;
  }
}

template <int D>
static void combine_launch(const TreeArgs& a, const KvView& c, int grid, int NT, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  const int rows = a.nb * a.gb;              // of a row tile
  int RP = 1;
  while (RP < 32 && RP < rows) RP *= 2;
  const int blocks = (rows + RP - 1) / RP;
  cfg.gridDim = dim3((unsigned)((long long)a.B * a.Hkv * a.rt * blocks), 1, 1);
  cfg.blockDim = dim3(128, 1, 1);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, tree_combine_kernel<D>, a, c, grid, NT, RP, blocks));
}

template <typename K>
static void tree_smem(K kernel, size_t bytes, bool (&set)[64]) {   // a function's attributes are kept by device
  int dev = 0;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev >= 64 || !set[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    if (dev < 64) set[dev] = true;
  }
}

template <int D, bool QUANT, int EH>
static void few_launch(const CUtensorMap& tk, const CUtensorMap& tv, const at::Tensor& q, const TreeArgs& a, const KvView& c, int grid,
                       cudaStream_t s) {
  using Cfg = FewCfg<D, QUANT, EH>;
  static bool set[64] = {};
  tree_smem(tree_few_kernel<D, QUANT, EH>, Cfg::SMEM, set);
  tree_few_kernel<D, QUANT, EH><<<grid, kFewThreads, Cfg::SMEM, s>>>(tk, tv, reinterpret_cast<const __nv_bfloat16*>(q.data_ptr()), q.stride(0),
                                                                     q.stride(1), q.stride(2), a, c);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  combine_launch<D>(a, c, grid, 1, s);
}

template <int D, bool QUANT, int NT>
static void tree_launch(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const TreeArgs& a, const KvView& c,
                        int grid, cudaStream_t s) {
  using Cfg = TreeCfg<D, QUANT, NT>;
  static bool set[64] = {};
  tree_smem(tree_attention_kernel<D, QUANT, NT>, Cfg::SMEM, set);
  tree_attention_kernel<D, QUANT, NT><<<grid, Cfg::THREADS, Cfg::SMEM, s>>>(tq, tk, tv, a, c);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  combine_launch<D>(a, c, grid, NT, s);
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
  // Few rows a key/value head: the register kernel, up to 16 rows of e4m3 caches or heads of 64, up to 8 of bf16
  // rows of 128, whose 16-row form keeps too much in registers.  Register kernel / tensor-core tiles, us, 16
  // sequences of 4095 .. 8190 rows, 8 heads; and 64 sequences of 100 .. 200 rows:
  //   bf16, 128: 8 rows 74 / 76, 38 / 42;  9 rows 83 / 79, 52 / 42;  16 rows 83 / 79, 52 / 44
  //   bf16, 64:  8 rows 53 / 63, 27 / 34;  9 rows 62 / 64, 35 / 35;  16 rows 63 / 64, 36 / 37
  //   e4m3, 128: 8 rows 70 / 107, 41 / 47;  9 rows 87 / 111, 54 / 50;  16 rows 88 / 112, 60 / 52
  //   e4m3, 64:  8 rows 58 / 96, 29 / 40;  9 rows 71 / 98, 39 / 41;  16 rows 72 / 99, 40 / 42
  // With 32 rows it spilled: 180 against 83.
  const int rows = (int)std::min<int64_t>(N * G, 1 << 20), EH = rows <= 8 ? 1 : rows <= 16 && (quant || D == 64) ? 2 : 0;
  // rows of a tile: nb nodes of gb heads each
  a.gb = std::min(G, 128);
  a.nb = std::min((int)N, 128 / a.gb);
  a.gg = (G + a.gb - 1) / a.gb;
  a.rt = (((int)N + a.nb - 1) / a.nb) * a.gg;
  const int NT = a.rt > 1 ? 2 : 1;           // two row tiles share each key / value tile (none with EH)
  a.rg = (a.rt + NT - 1) / NT;
  a.scale_log2 = std::max((float)(std::abs(scale) * 1.4426950408889634), 1e-30f);   // -inf * 0 is NaN
  a.neg = scale < 0;
  c10::cuda::CUDAGuard guard(kc.device());
  auto o = at::empty({B, N, Hq, D}, q.options());
  if (o.numel() == 0) return o;
  a.o = reinterpret_cast<__nv_bfloat16*>(o.data_ptr());
  a.err = err.data_ptr<int>();
  const int64_t most = B * H * a.rg * ((T + 127) / 128);
  const int grid = (int)std::min<int64_t>(num_sms(kc.device().index()), most);
  TORCH_CHECK(most * (grid + 1) < (1LL << 31), "too many key tiles for one call");   // the kernels count in 32 bits
  auto part = at::empty({(int64_t)2 * grid * NT * 128 * (D + 2) + (int64_t)grid * 256}, q.options().dtype(at::kFloat));
  a.part = reinterpret_cast<float4*>(part.data_ptr<float>());
  a.part_ml = reinterpret_cast<float2*>(part.data_ptr<float>() + (int64_t)2 * grid * NT * 128 * D);
  a.pair_ml = a.part_ml + (int64_t)2 * grid * NT * 128;

  const uint64_t kd[4] = {(uint64_t)D, (uint64_t)T, (uint64_t)H, (uint64_t)B};
  const uint64_t kst[3] = {(uint64_t)c.t, (uint64_t)c.h, (uint64_t)c.b};
  const uint32_t kb[4] = {quant ? (uint32_t)D : 64u, 128, 1, 1};
  const auto type = quant ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const auto sw = quant && !EH ? CU_TENSOR_MAP_SWIZZLE_NONE : quant && D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  const CUtensorMap tk = make_tmap_nd(c.p[0], type, 4, kd, kst, kb, sw), tv = make_tmap_nd(c.p[1], type, 4, kd, kst, kb, sw);
  auto s = at::cuda::getCurrentCUDAStream();
  if (EH) {
#define TFB_FEW(DD, QQ) \
  (EH == 1 ? few_launch<DD, QQ, 1>(tk, tv, q, a, c, grid, s) : few_launch<DD, QQ, 2>(tk, tv, q, a, c, grid, s))
    if (D == 128) { if (quant) TFB_FEW(128, true); else few_launch<128, false, 1>(tk, tv, q, a, c, grid, s); }
    else { if (quant) TFB_FEW(64, true); else TFB_FEW(64, false); }
#undef TFB_FEW
    return o;
  }
  const uint64_t u = 2;
  const uint64_t qd[5] = {(uint64_t)D, (uint64_t)G, (uint64_t)N, (uint64_t)H, (uint64_t)B};
  const uint64_t qs[4] = {q.stride(2) * u, q.stride(1) * u, (uint64_t)G * q.stride(2) * u, q.stride(0) * u};
  const uint32_t qb[5] = {64, (uint32_t)a.gb, (uint32_t)a.nb, 1, 1};
  const CUtensorMap tq = make_tmap_nd(q.data_ptr(), CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, qd, qs, qb, CU_TENSOR_MAP_SWIZZLE_128B);
#define TFB_TREE(DD, QQ) (NT == 1 ? tree_launch<DD, QQ, 1>(tq, tk, tv, a, c, grid, s) : tree_launch<DD, QQ, 2>(tq, tk, tv, a, c, grid, s))
  if (D == 128) { if (quant) TFB_TREE(128, true); else TFB_TREE(128, false); }
  else { if (quant) TFB_TREE(64, true); else TFB_TREE(64, false); }
#undef TFB_TREE
  return o;
}

}  // namespace tfb
