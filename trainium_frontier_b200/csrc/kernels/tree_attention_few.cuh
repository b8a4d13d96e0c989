// Tree attention of few query rows (at most 16 a key/value head): see tree_attention.cu, which
// includes this file.
//
// With so few rows the cache's bytes bound the time, and a 128-row tcgen05 tile leaves most of its
// lanes without work while every hand-over between its roles costs latency.  Here a key tile is
// cut over eight warps instead, 16 keys each, and a warp keeps everything of its keys in
// registers: scores, exponentials and products by 16 x 8 x 16 warp-level matrix instructions, with
// a maximum, a sum and an output of its own.  Nothing is handed over but the tiles themselves (TMA,
// a ring of key + value stages); the eight outputs are added once a segment.
//
// Quantised tiles are read as they are and become f16 fragments in registers, one conversion for
// two codes.  The rows' scales never touch the codes: a key's is a factor of its score, and a
// value's joins the exponent: w = 2^(score + log2 scale - m') against plain codes is p times the
// value, with a reference m' of its own, so that w fits f16 (11 bits of significand) whatever the
// scales are.  Weights below 2^-14 of the reference lose bits, and those below 2^-25 count nothing,
// also in columns where the rows of large weight hold zeros.  The sum of p = 2^(score - m) is kept
// apart in 32 bits.
//
// Measured on a B200 (calls replayed from a graph).  A decode step of 32 sequences x 10 heads over
// 288 .. 575 rows: bf16 30 us of 11, e4m3 32 of 5.5 (each CTA has two or three short segments, whose starts and
// ends cost more than the tiles, and the second kernel takes 7 us by itself).  16 sequences of 4095 .. 8190
// rows, 8 heads, 8 rows: bf16 74 us of 62, e4m3 70 of 31 (with two warps a sub-core the chain of
// instructions of a tile is the limit).  One sequence of 1023 e4m3 rows, 6 nodes x 10 heads of 64: 11 to 12 us, two
// dependent launches.  Two CTAs of 128 registers a SM spilled (101 us).
#pragma once

#include "warp_mma.cuh"

namespace tfb {

constexpr int kFewWarps = 8;
constexpr int kFewThreads = 32 * kFewWarps;

template <int D, bool QUANT, int EH>
struct FewCfg {
  static_assert(EH == 1 || EH == 2, "8 or 16 rows");
  static constexpr int MT = 1;                                     // 16-row tiles (two do not fit the registers)
  static constexpr uint32_t TILE = 128u * D * (QUANT ? 1u : 2u);   // a key or value tile
  static constexpr int NS = QUANT ? 6 : D == 128 ? 3 : 6;          // stages of one of each (at most a warp's worth)
  static constexpr int OUTF = 512;                                 // output values of a warp added at a time
  static constexpr uint32_t OUT = kFewWarps * (OUTF + 4 * 16) * 4; // rows padded
  static constexpr uint32_t QF = MT * (D / 16) * 512u;             // query fragments
  static constexpr size_t SMEM = 2 * NS * TILE + QF + OUT + kFewWarps * 16 * MT * 8 + 2 * NS * 8 + 16 + 16 * MT * 8 + kLenCache * 4 + 16;
};
static_assert(FewCfg<128, true, 2>::NS <= kFewWarps && FewCfg<64, true, 2>::NS <= kFewWarps, "a warp a stage");
static_assert(FewCfg<128, false, 1>::SMEM <= 232448 && FewCfg<128, true, 2>::SMEM <= 232448 && FewCfg<64, false, 2>::SMEM <= 232448,
              "shared memory");

template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16-byte chunk of a row of an e4m3 tile as TMA lays it out (128- or 64-byte swizzle).
template <int D>
__device__ __forceinline__ uint32_t code_chunk(int row, int chunk) {
  return D == 128 ? (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4)) : (uint32_t)(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
}
__device__ __forceinline__ bool bf16_bad(uint32_t h) { return (h & 0x7f80u) == 0x7f80u; }
// bits 15 and 31: whether the halves are infinite or NaN
__device__ __forceinline__ uint32_t bf16x2_bad(uint32_t w) { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }

// x plus four columns of an e4m3 value row, times its weight and scale.  Out of line since it is rare, and in
// line it cost the loop over the tiles registers (16 rows: 114 against 111 us).
template <int D>
__device__ __noinline__ float4 tree_add_row(float4 x, const __nv_bfloat16* q, const uint8_t* key, const uint8_t* value, float scale, float M,
                                          float vscale) {
  float y = 0.f;
  for (int d = 0; d < D; ++d) y += __bfloat162float(q[d]) * e4m3_float(key[d]);
  const float p = tree_ex2(y * scale - M) * vscale;
  x.x += p * e4m3_float(value[0]);
  x.y += p * e4m3_float(value[1]);
  x.z += p * e4m3_float(value[2]);
  x.w += p * e4m3_float(value[3]);
  return x;
}

// EH: halves of the 16-row tile that hold rows
template <int D, bool QUANT, int EH>
__global__ void __launch_bounds__(kFewThreads, 1)
    tree_few_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __nv_bfloat16* __restrict__ Q,
                    long long qb, long long qn, long long qh, const TreeArgs a, const __grid_constant__ KvView c) {
  using Cfg = FewCfg<D, QUANT, EH>;
  constexpr uint32_t TILE = Cfg::TILE;
  constexpr int NS = Cfg::NS, KS = D / 16, NTILE = D / 8, MT = Cfg::MT;
  constexpr int E = EH == 1 ? 1 : 2;           // halves of a tile that hold rows
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {         // the swizzled tiles need it
    if (threadIdx.x == 0) atomicOr(a.err, ERR_BAD_ARG);
    return;
  }
  uint8_t* sKV = smem;                         // [NS][key tile, value tile]
  uint4* sQ = reinterpret_cast<uint4*>(sKV + 2 * NS * TILE);                  // [MT][KS][32 lanes]
  float* sO = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(sQ) + Cfg::QF);   // [warps][rows][columns + 4]
  float2* sML = reinterpret_cast<float2*>(sO + Cfg::OUT / 4);                 // [warps][16 MT]
  uint64_t* full = reinterpret_cast<uint64_t*>(sML + kFewWarps * 16 * MT);
  uint64_t* empty = full + NS;
  unsigned long long* s_bad = reinterpret_cast<unsigned long long*>(empty + NS);
  unsigned long long* s_line = s_bad + 2;      // [16 MT]
  int* s_len = reinterpret_cast<int*>(s_line + 16 * MT);
  volatile int* abort_flag = s_len + kLenCache;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kFewWarps);
    }
    s_bad[0] = s_bad[1] = 0;
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  const TreeLens lens{a.lens, a.B <= kLenCache ? s_len : nullptr, a.N, c.tmax};
  for (int i = threadIdx.x; i < a.B && i < kLenCache; i += kFewThreads) s_len[i] = max(0, min(a.lens[i], c.tmax));
  __syncthreads();
  griddep_launch_dependents();
  TreeIter it = tree_begin(a, lens, (int)blockIdx.x, (int)gridDim.x);

  // One thread loads: the ring is filled, and a stage refilled once all warps have left it.  (A warp
  // for it alone would cost the others a quarter of their registers.)
  TreeIter ld = it;
  int loads = 0;
  bool load_ok = lane == 0;
  auto issue = [&](int s) {
    mbar_arrive_expect_tx(&full[s], 2 * TILE);
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      uint8_t* dst = sKV + (2 * s + v) * TILE;
      const CUtensorMap* map = v ? &tmV : &tmK;
      if constexpr (QUANT) {
        tma_load_4d(dst, map, &full[s], 0, ld.k * 128, ld.h, ld.b);
      } else {
#pragma unroll
        for (int p = 0; p < D / 64; ++p) tma_load_4d(dst + p * kTreePanel, map, &full[s], p * 64, ld.k * 128, ld.h, ld.b);
      }
    }
  };
  // the ring is filled by a warp a stage
#pragma unroll 1
  while (loads < NS && ld.next(lens, a.rg)) {
    if (loads == warp && lane == 0) issue(loads);
    ++loads;
  }
  auto load = [&]() {
    if (threadIdx.x != 0 || !load_ok || !ld.next(lens, a.rg)) return;
    const int s = loads % NS;
    load_ok = mbar_wait(&empty[s], ((loads / NS) + 1) & 1, abort_flag, a.err, ERR_TIMEOUT_PRODUCER);
    if (!load_ok) return;
    issue(s);
    ++loads;
  };
  __syncwarp();

  // ------------------------------------------------------------------ 16 keys of every tile a warp
  // A wait that runs out ends nothing here: the warps meet at barriers, so all of them go on to the
  // end with whatever the tiles hold, and the error word says so.
  const int gq = lane >> 2, j = lane & 3;      // row (of 8) and column pair of a fragment
  const int R = a.N * a.G;
  float o[MT][NTILE][4], m[MT][2], l[MT][2], cr[MT][2];
  float mw[MT][2];                             // reference of the weights (QUANT; else m)
  unsigned long long line[MT][2], used = 0;
  uint32_t ahead = 127u;                       // scale byte of the next tile: keys (lanes 0-15) and values of the warp's keys
  int g = 0, seg = 0;
  // row of fragment half e of row tile mt
  auto row_of = [&](int mt, int e) { return mt * 16 + e * 8 + gq; };
  int node[MT][2];                             // of the lane's rows, -1 where there is none
  long long qrow[MT][2];                       // their queries' places
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = row_of(mt, e), n = r / a.G;
      node[mt][e] = r < R ? n : -1;
      qrow[mt][e] = n * qn + (r - n * a.G) * qh;
    }
  // this lane's keys 2j, 2j + 1, 8 + 2j, 9 + 2j of the warp's 16
  auto key_of = [&](int i) { return warp * 16 + (i >> 1) * 8 + 2 * j + (i & 1); };
  const uint8_t* const sbase = QUANT ? (lane < 16 ? c.s[0] : c.s[1]) : nullptr;
  auto fetch_scales = [&](const TreeIter& t) {
    if constexpr (QUANT) {
      const int row = t.k * 128 + warp * 16 + (lane & 15);
      ahead = row < c.tmax ? sbase[t.b * c.sb + t.h * c.sh + (long long)row * c.st] : 127u;
    }
  };
  TreeIter nx = it;                            // one tile ahead
  if (nx.next(lens, a.rg)) fetch_scales(nx);
  while (it.next(lens, a.rg)) {
    if (it.first()) {
      // Drafted value rows (at most 16) that hold a NaN code (0 * NaN is NaN): they are left out of the
      // product like unused ones, and what the nodes that see them get of them is added at the segment's
      // end.  (Looked for in every tile, the branch alone cost 2 to 7 %: 118 against 109 us for 16 rows.)
      uint32_t drafted[2] = {0, 0};
      if constexpr (QUANT) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = warp + i * kFewWarps;
          if (lane < D / 4 && it.k1 * 128 > it.len && n < a.N && it.len + n < c.tmax)
            drafted[i] = reinterpret_cast<const uint32_t*>(c.p[1] + it.b * c.b + it.h * c.h + ((long long)it.len + n) * c.t)[lane];
        }
      }
      // queries as fragments, a step of 16 dimensions a warp at a time
      if constexpr (QUANT) {
        // f16, each row by a power of two that takes its largest value to 2^14 .. 2^15.  Entries below
        // 2^-31 of that value lose bits, those below 2^-40 are 0.
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const __nv_bfloat16* src = Q + it.b * qb + (long long)it.h * a.G * qh + qrow[mt][e];
            uint32_t mx = 0;
            uint2 mine = make_uint2(0, 0);
            if (node[mt][e] >= 0) {
#pragma unroll
              for (int s = 0; s < KS; ++s) {   // dimensions 2 KS j .. : what this lane's chunks of a key row hold
                const uint2 u = *reinterpret_cast<const uint2*>(src + (D / 4) * j + 4 * s);
                mx = __vmaxu2(mx, __vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu));
                if (s == warp % KS) mine = u;
              }
            }
            uint32_t top = max(mx & 0xffffu, mx >> 16);
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // exponent bytes of the maximum and of the factor: 2^111 at most, which takes bf16's least step,
            // 2^-133, to 2^-22 (exact in f16) and leaves its inverse a normal number
            const int ex = (int)(top >> 7), fe = min(268 - ex, 238);
            const float f = __uint_as_float((uint32_t)fe << 23);
            cr[mt][e] = a.scale_log2 * __uint_as_float((uint32_t)(254 - fe) << 23);
            if (a.neg) cr[mt][e] = -cr[mt][e];
            const uint32_t lo = pack_f16x2(__uint_as_float(mine.x << 16) * f, __uint_as_float(mine.x & 0xffff0000u) * f);
            const uint32_t hi = pack_f16x2(__uint_as_float(mine.y << 16) * f, __uint_as_float(mine.y & 0xffff0000u) * f);
            if (warp < KS) {
              uint32_t* d = reinterpret_cast<uint32_t*>(&sQ[(mt * KS + warp) * 32 + lane]);
              d[e] = lo;
              d[2 + e] = hi;
            }
          }
      } else {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t lo = 0, hi = 0;
            if (node[mt][e] >= 0 && warp < KS) {
              const __nv_bfloat16* src = Q + it.b * qb + (long long)it.h * a.G * qh + qrow[mt][e] + warp * 16 + 2 * j;
              lo = *reinterpret_cast<const uint32_t*>(src);
              hi = *reinterpret_cast<const uint32_t*>(src + 8);
            }
            if (warp < KS) {
              uint32_t* d = reinterpret_cast<uint32_t*>(&sQ[(mt * KS + warp) * 32 + lane]);
              d[e] = lo;
              d[2 + e] = hi;
            }
            cr[mt][e] = a.neg ? -a.scale_log2 : a.scale_log2;
          }
      }
      if constexpr (QUANT) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (__any_sync(0xffffffffu, code4_nan(drafted[i]) != 0) && lane == 0) atomicOr(&s_bad[seg & 1], 1ull << (warp + i * kFewWarps));
      }
      unsigned long long m0, m1;
      tree_lines(a.parents ? a.parents + (long long)it.b * a.N : nullptr, a.N, c.tmax - it.len, m0, m1);
      used = used_nodes(m0, m1);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = row_of(mt, e), n = max(node[mt][e], 0);
          const unsigned long long x0 = __shfl_sync(0xffffffffu, m0, n & 31), x1 = __shfl_sync(0xffffffffu, m1, n & 31);
          line[mt][e] = node[mt][e] < 0 ? 0 : n >= 32 ? x1 : x0;
          m[mt][e] = mw[mt][e] = -INFINITY;
          l[mt][e] = 0.f;
          if (warp == 0 && j == 0) s_line[r] = line[mt][e];
        }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < NTILE; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[mt][i][k] = 0.f;
      __syncthreads();
      if constexpr (QUANT) used &= ~s_bad[seg & 1];
    }
    // the lane's scale: a key's as it is, a value's as its log2 (decoded by its lane: once, not by every lane that needs it)
    const float factor = ahead == (uint32_t)kScaleNan ? __int_as_float(0x7fffffff)
                         : lane >= 16                 ? (float)((int)ahead - 127)
                                                      : __uint_as_float(ahead == 0 ? 1u << 22 : ahead << 23);
    if (nx.next(lens, a.rg)) fetch_scales(nx);
    const int slot = g % NS;
    mbar_wait(&full[slot], (g / NS) & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE);
    if (g > 0) load();                         // into the stage of the tile before
    ++g;
    __syncwarp();
    const uint8_t* sK = sKV + 2 * slot * TILE;
    const uint8_t* sV = sK + TILE;
    const int off = it.k * 128 + warp * 16 - it.len;      // of the warp's first key from the first node's row
    const bool masked = off + 16 > 0;

    // ---- scores
    float s[MT][2][4], s2[MT][2][4];                      // even and odd steps: two short chains instead of a long one
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[mt][t][k] = s2[mt][t][k] = 0.f;
    if constexpr (QUANT) {
      uint32_t u[2][KS];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int q = 0; q < KS / 4; ++q) {
          const uint4 x = *reinterpret_cast<const uint4*>(sK + code_chunk<D>(warp * 16 + 8 * t + gq, (KS / 4) * j + q));
          u[t][4 * q] = x.x; u[t][4 * q + 1] = x.y; u[t][4 * q + 2] = x.z; u[t][4 * q + 3] = x.w;
        }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const uint4 q = sQ[(mt * KS + ks) * 32 + lane];
          const uint32_t qa[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int t = 0; t < 2; ++t) mma16816<true>(ks & 1 ? s2[mt][t] : s[mt][t], qa, codes2(u[t][ks]), codes2(u[t][ks] >> 16));
        }
    } else {
      const int mi = lane >> 3, row = warp * 16 + (mi >> 1) * 8 + (lane & 7);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int ch = 2 * ks + (mi & 1);
        uint32_t kf[4];
        ldmatrix4<false>(smem_u32(sK) + (uint32_t)(ch >> 3) * kTreePanel + sw128_chunk_offset(row, ch & 7), kf);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const uint4 q = sQ[(mt * KS + ks) * 32 + lane];
          const uint32_t qa[4] = {q.x, q.y, q.z, q.w};
          mma16816<false>(ks & 1 ? s2[mt][0] : s[mt][0], qa, kf[0], kf[1]);
          mma16816<false>(ks & 1 ? s2[mt][1] : s[mt][1], qa, kf[2], kf[3]);
        }
      }
    }

    // ---- exponentials: element k of fragment t is (row half k >> 1, key 8 t + 2 j + (k & 1))
    float fk[4], ev[4];
    bool alive[4];                                        // the key's row holds something that counts
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = off + key_of(i) - warp * 16;
      alive[i] = !masked || at < 0 || (at < kTreeNodes && ((used >> at) & 1));
      if constexpr (QUANT) {
        fk[i] = __shfl_sync(0xffffffffu, factor, key_of(i) - warp * 16);
        ev[i] = __shfl_sync(0xffffffffu, factor, 16 + key_of(i) - warp * 16);
        alive[i] = alive[i] && ev[i] == ev[i];            // NaN: the weight is NaN for the queries that see the row
      }
    }
    uint32_t pa[MT][4];
    bool grow = false;
    float alpha[MT][2];
    auto quad_max = [](float x) {
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
      return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
    };
    // moves a reference to a maximum that is larger by more than 8; the factor for what stands at the old one
    auto refer = [](float mx, float& ref) -> float {
      const bool up = mx > ref + 8.f;
      const float al = up ? tree_ex2(ref - mx) : 1.f;
      ref = up ? mx : ref;
      return al;
    };
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int k = 0; k < 2 * E; ++k) {
          const int i = 2 * t + (k & 1), e = k >> 1;
          float x = (s[mt][t][k] + s2[mt][t][k]) * cr[mt][e];
          if constexpr (QUANT) x *= fk[i];
          if (masked) {
            const int at = off + 8 * t + 2 * j + (k & 1);
            if (at >= 0 && (at >= kTreeNodes || !((line[mt][e] >> at) & 1))) x = -INFINITY;
          }
          s[mt][t][k] = x;
        }
      if constexpr (E == 1) {
        alpha[mt][1] = 1.f;
        pa[mt][1] = pa[mt][3] = 0;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float x[4] = {s[mt][0][2 * e], s[mt][0][2 * e + 1], s[mt][1][2 * e], s[mt][1][2 * e + 1]};
        float y[4];
        float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), my = mx;
        if constexpr (QUANT) {
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = x[i] == -INFINITY ? -INFINITY : x[i] + ev[i];
          my = quad_max(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])));
        }
        mx = quad_max(mx);
        const float al = refer(mx, m[mt][e]);
        const float ref = m[mt][e] == -INFINITY ? 0.f : m[mt][e];
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = tree_ex2(x[i] - ref);
        l[mt][e] = l[mt][e] * al + ((p[0] + p[1]) + (p[2] + p[3]));
        if constexpr (QUANT) {
          float w[4];
          alpha[mt][e] = refer(my, mw[mt][e]);
          const float rw = mw[mt][e] == -INFINITY ? 0.f : mw[mt][e];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = tree_ex2(y[i] - rw);
          pa[mt][e] = pack_f16x2(w[0], w[1]);
          pa[mt][2 + e] = pack_f16x2(w[2], w[3]);
        } else {
          alpha[mt][e] = al;
          pa[mt][e] = pack_bf16x2(p[0], p[1]);              // 8 bits of significand for the product, the sum in 32 bits
          pa[mt][2 + e] = pack_bf16x2(p[2], p[3]);
        }
        grow |= alpha[mt][e] != 1.f;
      }
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < NTILE; ++i)
#pragma unroll
          for (int k = 0; k < 2 * E; ++k) o[mt][i][k] *= alpha[mt][k >> 1];
    }

    // ---- outputs
    if constexpr (QUANT) {
      // dimension (D / 8) n + i is column n of fragment i
      constexpr int W = D / 32;                           // words of a lane's piece of a row
      uint32_t v[4][W];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = key_of(i);
        if constexpr (D == 128) {
          const uint4 x = *reinterpret_cast<const uint4*>(sV + code_chunk<D>(row, gq));
          v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(sV + code_chunk<D>(row, gq >> 1) + (gq & 1) * 8);
          v[i][0] = x.x; v[i][1] = x.y;
        }
        if (!alive[i]) {
#pragma unroll
          for (int w = 0; w < W; ++w) v[i][w] = 0;
        }
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        uint32_t f[2][4];                                 // [keys 2j.., 8 + 2j..][dimension of the word]
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint32_t x = __byte_perm(v[2 * t][w], v[2 * t + 1][w], 0x5140), y = __byte_perm(v[2 * t][w], v[2 * t + 1][w], 0x7362);
          f[t][0] = codes2(x); f[t][1] = codes2(x >> 16); f[t][2] = codes2(y); f[t][3] = codes2(y >> 16);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) mma16816<true>(o[mt][4 * w + q], pa[mt], f[0][q], f[1][q]);
      }
    } else {
      const int mi = lane >> 3, row = warp * 16 + (mi & 1) * 8 + (lane & 7);
      uint32_t keep[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) keep[t] = (alive[2 * t] ? 0xffffu : 0u) | (alive[2 * t + 1] ? 0xffff0000u : 0u);
      uint32_t bad = 0;                                   // the lane's keys whose drafted row is not finite
      bool dirty = false;
      if (masked) {
        uint32_t any = 0;
#pragma unroll 2
        for (int i = 0; i < NTILE; i += 2) {
          const int ch = i + (mi >> 1);
          uint32_t vf[4];
          ldmatrix4<true>(smem_u32(sV) + (uint32_t)(ch >> 3) * kTreePanel + sw128_chunk_offset(row, ch & 7), vf);
#pragma unroll
          for (int q = 0; q < 4; ++q) any |= bf16x2_bad(vf[q] & keep[q & 1]);
        }
        dirty = __any_sync(0xffffffffu, any != 0);
      }
#pragma unroll
      for (int i = 0; i < NTILE; i += 2) {
        const int ch = i + (mi >> 1);
        uint32_t vf[4];
        ldmatrix4<true>(smem_u32(sV) + (uint32_t)(ch >> 3) * kTreePanel + sw128_chunk_offset(row, ch & 7), vf);
#pragma unroll
        for (int q = 0; q < 4; ++q) vf[q] &= keep[q & 1];
        if (dirty) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int t = q & 1;
            const int at = off + 8 * t + 2 * j;
            if (at >= 0 && bf16_bad(vf[q])) { vf[q] &= 0xffff0000u; bad |= 1u << (2 * t); }
            if (at + 1 >= 0 && bf16_bad(vf[q] >> 16)) { vf[q] &= 0xffffu; bad |= 2u << (2 * t); }
          }
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma16816<false>(o[mt][i], pa[mt], vf[0], vf[1]);
          mma16816<false>(o[mt][i + 1], pa[mt], vf[2], vf[3]);
        }
      }
      if (bad) {
        for (int i = 0; i < 4; ++i)
          if ((bad >> i) & 1) atomicOr(&s_bad[seg & 1], 1ull << (off + key_of(i) - warp * 16));
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[slot]);
    if (!it.last()) continue;

    // ---- end of the segment: the eight warps' outputs at their common reference, added
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float x = l[mt][e];
        x += __shfl_xor_sync(0xffffffffu, x, 1);
        x += __shfl_xor_sync(0xffffffffu, x, 2);
        if (j == 0) sML[warp * 16 * MT + row_of(mt, e)] = make_float2(m[mt][e], x);
      }
    __syncthreads();
    const bool whole = it.k0 == 0 && it.k1 == it.kt;
    const long long part = 2LL * blockIdx.x + (it.k0 == 0 ? 1 : 0);
    auto common = [&](int r) {
      float M = -INFINITY;
      for (int w = 0; w < kFewWarps; ++w) {
        const float2 ml = sML[w * 16 * MT + r];
        if (ml.y != 0.f) M = fmaxf(M, ml.x);
      }
      return M;
    };
    const int rp = EH > 1 ? 16 : R <= 4 ? 4 : 8;          // rows added at a time, and the columns that fit
    const int hc = min(Cfg::OUTF / rp, D);
#pragma unroll 1
    for (int mt = 0; mt < MT; ++mt) {
      float f[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int r = row_of(mt, e);
        float x = 0.f;
#pragma unroll
        for (int q = 0; q < MT; ++q)
          if (q == mt) x = QUANT ? mw[q][e] : m[q][e];
        f[e] = sML[warp * 16 * MT + r].y == 0.f ? 0.f : tree_ex2(x - common(r));
      }
#pragma unroll 1
      for (int h0 = 0; h0 < D; h0 += hc) {
        float* dst = sO + warp * rp * (hc + 4);
#pragma unroll
        for (int i = 0; i < NTILE; ++i)
#pragma unroll
          for (int k = 0; k < 2 * E; ++k) {
            const int d = (QUANT ? (D / 8) * (2 * j + (k & 1)) + i : 8 * i + 2 * j + (k & 1)) - h0;
            float x = 0.f;
#pragma unroll
            for (int q = 0; q < MT; ++q)
              if (q == mt) x = o[q][i][k];
            if (d >= 0 && d < hc && (k >> 1) * 8 + gq < rp) dst[((k >> 1) * 8 + gq) * (hc + 4) + d] = x * f[k >> 1];   // f may be 0: a NaN stays
          }
        __syncthreads();
        const int per = hc / 4, rr = threadIdx.x / per, r = mt * 16 + rr, c4 = threadIdx.x - rr * per;
        if (rr < rp && r < R) {
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kFewWarps; ++w) {
            const float4 y = *reinterpret_cast<const float4*>(sO + (w * rp + rr) * (hc + 4) + 4 * c4);
            x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
          }
          const float M = common(r);
          float L = 0.f;
          for (int w = 0; w < kFewWarps; ++w) {
            const float2 ml = sML[w * 16 * MT + r];
            if (ml.y != 0.f) L += ml.y * tree_ex2(ml.x - M);
          }
          const int n = r / a.G, hd = r - n * a.G;
          const unsigned long long ln = s_line[r];
          const int col = h0 + 4 * c4;
          unsigned long long bad = s_bad[seg & 1] & ln;
          for (; bad; bad &= bad - 1) {                    // drafted rows with an infinity or a NaN
            const long long t = (long long)it.len + __ffsll((long long)bad) - 1;
            const uint8_t* base = c.p[1] + it.b * c.b + it.h * c.h + t * c.t;
            if constexpr (QUANT) {                         // the whole row, with its weight once more
              if ((t >> 7) < it.k0 || (t >> 7) >= it.k1) continue;
              const long long si = it.b * c.sb + it.h * c.sh + t * c.st;
              x = tree_add_row<D>(x, Q + it.b * qb + ((long long)it.h * a.G + hd) * qh + n * qn, c.p[0] + (base - c.p[1]), base + col,
                              (a.neg ? -a.scale_log2 : a.scale_log2) * scale_float(c.s[0][si]), M, scale_float(c.s[1][si]));
              continue;
            }
            const __nv_bfloat16* row = reinterpret_cast<const __nv_bfloat16*>(base) + col;   // those entries
            float* xs = &x.x;
            for (int k = 0; k < 4; ++k) {
              const float y = __bfloat162float(row[k]);
              if (!(fabsf(y) < INFINITY)) xs[k] += y;
            }
          }
          if (whole) {
            const float inv = ln == 0 ? 0.f : 1.f / L;     // L = 0: all scores are -inf, and 0 / 0 is NaN
            if (ln == 0) x = make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<uint2*>(a.o + (((long long)it.b * a.N + n) * a.Hq + it.h * a.G + hd) * D + col) =
                make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
          } else {
            a.part[(part * (D / 4) + (col >> 2)) * 128 + r] = x;
            if (h0 == 0 && c4 == 0) a.part_ml[part * 128 + r] = ln == 0 ? make_float2(INFINITY, 0.f) : make_float2(M, L);
          }
        }
        __syncthreads();
      }
    }
    if (threadIdx.x == 0) s_bad[seg & 1] = 0;              // next used two segments on, with barriers between
    ++seg;
  }
  if (threadIdx.x == 0 && *abort_flag) {       // let the copies in flight land before the CTA ends
    const unsigned long long t0 = globaltimer_ns();
    for (int i = max(0, loads - NS); i < loads; ++i)
      while (!mbar_try_wait(&full[i % NS], (i / NS) & 1))
        if (globaltimer_ns() - t0 > 100000000ull) break;
  }
}

}  // namespace tfb
