// Attention of one new token of every sequence over a cache of pages.
//
//   o = sum_t softmax_t(scale q . k_t) v_t,   t < lens[b], row t being row t % page of page table[b, t / page].
//
// The cache's bytes bound the time: 2 D products a byte at most with 8 query heads a key/value head.  So
// nothing is staged: a warp takes 32 keys a step, reads their rows as 16-byte pieces straight into the
// registers of warp-level matrix instructions (16 keys or dimensions x 8 heads x 16), and the rows of its next
// step are on their way while it computes.  The order of the dimensions is free in q . k, and that of the
// output's rows in p v, so both operands' fragments are what a lane's own pieces hold:
//   scores   A = 16 keys x 16 dimensions: lane (r, j) has pieces j, j + 4, .. of keys r and r + 8;
//   output   A = 16 dimensions x 16 keys: lane (r, j) has piece r (and r + 8) of keys 2j, 2j + 1, 2j + 8, 2j + 9,
//            interleaved by byte permutations.  The weights, computed with the heads along the lanes,
//            are turned by the warp's 8 x 8 transposition.
// A piece of a sequence is a CTA of four warps, each with a maximum, a sum and an output of its own; a
// sequence is cut evenly into as many pieces as the batch needs to fill the GPU, whatever its length, and
// the pieces are joined in order by a second kernel that is launched under the first.
//
// Quantised rows: codes become f16 in registers.  A key's scale multiplies its score; a value's joins the
// exponent of its weight, 2^(score + log2 scale - m') with a maximum m' of its own, so that weights fit f16
// whatever the scales are.
#include <ATen/ops/empty.h>

#include "attention_tiles.cuh"
#include "warp_mma.cuh"

namespace tfb {

int num_sms(int dev);
int page_log(int64_t page);
const int* page_table(const at::Tensor& t, const at::Tensor& kp, int64_t B);

constexpr int kPaWarps = 4;
constexpr float kLowest = -3.4028234663852886e38f;

struct PaArgs {
  const __nv_bfloat16* q;
  long long qb, qh;              // in elements
  const int* table;
  long long tb;
  int width, pages, lg;
  const int* lens;
  int Hq, Hkv, G, rg;            // query heads a key/value head, groups of them
  int splits;
  float scale_log2;
  float* part;                   // [B, Hq, splits, D + 4]: output, then m, m', sum
  __nv_bfloat16* out;            // [B, Hq, D]
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// A 16-byte piece of a cached row; rows are read once.
__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) {
  uint4 u;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
  return u;
}
__device__ __forceinline__ uint2 ld_stream8(const uint8_t* p) {
  uint2 u;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(u.x), "=r"(u.y) : "l"(p));
  return u;
}

// KT: tiles of 16 keys a step of a warp; NT: groups of 8 query heads.
template <int D, bool QUANT, int KT, int NT>
__global__ void __launch_bounds__(32 * kPaWarps, NT == 1 && (QUANT || D == 64) ? 3 : 2)
    paged_attention_kernel(const PaArgs a, const __grid_constant__ KvView c) {
  constexpr int KEYS = 16 * KT;
  constexpr int KP = QUANT ? D / 64 : D / 32;      // pieces of a key row a lane
  constexpr int VP = QUANT ? 1 : D / 64;           // of a value row (e4m3 heads of 64: half a piece)
  constexpr int KS = D / 16, MT = D / 16;          // steps of 16 dimensions; tiles of them in the output
  constexpr int R = 8 * NT;                        // rows for query heads
  constexpr int TABLE = 32 / KT;                   // steps whose pages a warp holds, an entry a lane
  __shared__ float sO[kPaWarps][R][D + 4];
  __shared__ float sML[kPaWarps][R][3];
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, j = lane & 3;
  const int units = a.Hkv * a.rg;
  const int hr = (int)(blockIdx.x % units), split = (int)(blockIdx.x / units % a.splits);
  const int b = (int)(blockIdx.x / units / a.splits);
  const int h = hr / a.rg, g0 = (hr % a.rg) * R;   // key/value head, first query head of it
  const int rows = min(R, a.G - g0);
  const int len = (int)max(0LL, min((long long)a.lens[b], (long long)a.width << a.lg));
  const long long steps = ((long long)len + KEYS - 1) / KEYS;
  const int u0 = (int)(steps * split / a.splits), u1 = (int)(steps * (split + 1) / a.splits);
  const int* table = a.table + b * a.tb;

  // ------------------------------------------------------------------ queries: fragments of all dimensions
  uint32_t q[NT][2 * KS];
  float cr[NT][2];                                 // what a product is times, of heads 2j and 2j + 1
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = nt * 8 + gq;
    const __nv_bfloat16* src = a.q + b * a.qb + (long long)(h * a.G + g0 + r) * a.qh;
    if constexpr (!QUANT) {
#pragma unroll
      for (int p = 0; p < KP; ++p) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (r < rows) u = *reinterpret_cast<const uint4*>(src + 8 * (4 * p + j));
        q[nt][4 * p] = u.x; q[nt][4 * p + 1] = u.y; q[nt][4 * p + 2] = u.z; q[nt][4 * p + 3] = u.w;
      }
      cr[nt][0] = cr[nt][1] = a.scale_log2;
    } else {
      // f16: each head times a power of two that takes its largest value to 2^14 .. 2^15.  Entries below
      // 2^-31 of that value lose bits, those below 2^-40 are 0.
      uint32_t mx = 0;
#pragma unroll
      for (int p = 0; p < KP; ++p)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint4 u = make_uint4(0, 0, 0, 0);
          if (r < rows) u = *reinterpret_cast<const uint4*>(src + 16 * (4 * p + j) + 8 * i);
          mx = __vmaxu2(mx, absmax8(u));
          uint32_t* d = &q[nt][8 * p + 4 * i];
          d[0] = u.x; d[1] = u.y; d[2] = u.z; d[3] = u.w;
        }
      uint32_t top = max(mx & 0xffffu, mx >> 16);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // exponent bytes of the maximum and of the factor: 2^111 at most, whose inverse is a normal number
      const int ex = (int)(top >> 7), fe = min(268 - ex, 238);
      const float f = __uint_as_float((uint32_t)fe << 23);
      const float back = a.scale_log2 * __uint_as_float((uint32_t)(254 - fe) << 23);
#pragma unroll
      for (int i = 0; i < 2; ++i) cr[nt][i] = __shfl_sync(0xffffffffu, back, (2 * j + i) * 4);
#pragma unroll
      for (int i = 0; i < 2 * KS; ++i)
        q[nt][i] = pack_f16x2(__uint_as_float(q[nt][i] << 16) * f, __uint_as_float(q[nt][i] & 0xffff0000u) * f);
    }
  }

  // ------------------------------------------------------------------ loads of a step
  uint4 kr[KT][2][KP], vr[KT][4][VP];
  bool see[KT][2];                                 // keys gq and gq + 8 of a tile
  uint32_t sc = 0;                                 // scale bytes of key and value row `lane`
  int page[KT];                                    // of the step's tiles, -1: not there
  // the pages of the warp's next TABLE steps from step u on, one a lane
  auto fetch = [&](int u) {
    u += (lane / KT) * kPaWarps;
    const long long key = (long long)u * KEYS + 16 * (lane % KT);
    int pg = -1;
    if (u < u1 && key < len) pg = table[key >> a.lg];
    return pg >= 0 && pg < a.pages ? pg : -1;
  };
  auto load_k = [&](int u, int pages, int slot) {
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      page[t] = __shfl_sync(0xffffffffu, pages, slot * KT + t);
      const int key = u * KEYS + 16 * t + gq, in = key & ((1 << a.lg) - 1);
      const uint8_t* src = c.p[0] + page[t] * c.b + h * c.h + in * c.t + 16 * j;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        see[t][i] = page[t] >= 0 && key + 8 * i < len;
#pragma unroll
        for (int p = 0; p < KP; ++p) {
          kr[t][i][p] = make_uint4(0, 0, 0, 0);
          if (see[t][i]) kr[t][i][p] = ld_stream(src + 8 * i * c.t + 64 * p);
        }
      }
    }
    if constexpr (QUANT) {
      int pg = page[0];
#pragma unroll
      for (int t = 1; t < KT; ++t) pg = lane / 16 == t ? page[t] : pg;
      const int key = u * KEYS + lane;
      sc = 127u | (127u << 8);
      if (lane < KEYS && pg >= 0 && key < len) {
        const long long at = pg * c.sb + h * c.sh + (key & ((1 << a.lg) - 1)) * c.st;
        sc = c.s[0][at] | ((uint32_t)c.s[1][at] << 8);
      }
    }
  };
  auto load_v = [&](int u) {                       // rows that are not seen: zeros
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const int key = u * KEYS + 16 * t + 2 * j, in = key & ((1 << a.lg) - 1);
      const uint8_t* src = c.p[1] + page[t] * c.b + h * c.h + in * c.t + (QUANT && D == 64 ? 8 : 16) * gq;
#pragma unroll
      for (int i = 0; i < 4; ++i) {                // keys 2j, 2j + 1, 2j + 8, 2j + 9
        const int off = (i >> 1) * 8 + (i & 1);
#pragma unroll
        for (int p = 0; p < VP; ++p) {
          vr[t][i][p] = make_uint4(0, 0, 0, 0);
          if (page[t] >= 0 && key + off < len) {
            if constexpr (QUANT && D == 64) {
              const uint2 w = ld_stream8(src + off * c.t);
              vr[t][i][p].x = w.x; vr[t][i][p].y = w.y;
            } else {
              vr[t][i][p] = ld_stream(src + off * c.t + 128 * p);
            }
          }
        }
      }
    }
  };

  float o[NT][MT][4], m[NT][2], mw[NT][2], l[NT][2];   // mw: the weights' reference (QUANT; else m)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < MT; ++e) o[nt][e][0] = o[nt][e][1] = o[nt][e][2] = o[nt][e][3] = 0.f;
    m[nt][0] = m[nt][1] = mw[nt][0] = mw[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
  }

  // ------------------------------------------------------------------ the warp's steps
  int u = u0 + warp, slot = 0;
  int here = fetch(u), next = fetch(u + TABLE * kPaWarps);
  if (u < u1) {
    load_k(u, here, 0);
    load_v(u);
  }
#pragma unroll 1
  for (; u < u1; u += kPaWarps) {
    float x[KT][NT][4];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) x[t][nt][0] = x[t][nt][1] = x[t][nt][2] = x[t][nt][3] = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        uint32_t f[4];
        if constexpr (QUANT) {
          const uint4 r0 = kr[t][0][s >> 2], r1 = kr[t][1][s >> 2];
          const uint32_t w0 = (s & 3) == 0 ? r0.x : (s & 3) == 1 ? r0.y : (s & 3) == 2 ? r0.z : r0.w;
          const uint32_t w1 = (s & 3) == 0 ? r1.x : (s & 3) == 1 ? r1.y : (s & 3) == 2 ? r1.z : r1.w;
          f[0] = codes2(w0); f[1] = codes2(w1); f[2] = codes2(w0 >> 16); f[3] = codes2(w1 >> 16);
        } else {
          const uint4 r0 = kr[t][0][s >> 1], r1 = kr[t][1][s >> 1];
          f[0] = s & 1 ? r0.z : r0.x; f[1] = s & 1 ? r1.z : r1.x; f[2] = s & 1 ? r0.w : r0.y; f[3] = s & 1 ? r1.w : r1.y;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816<QUANT>(x[t][nt], f, q[nt][2 * s], q[nt][2 * s + 1]);
      }
    }
    float lv[KT][2];                               // log2 of the values' scales
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float ks = 1.f;
        lv[t][i] = 0.f;
        if constexpr (QUANT) {
          const uint32_t s2 = __shfl_sync(0xffffffffu, sc, 16 * t + 8 * i + gq);
          ks = scale_float((uint8_t)s2);
          lv[t][i] = (s2 >> 8) == kScaleNan ? __int_as_float(0x7fffffff) : (float)((int)(s2 >> 8) - 127);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float& y = x[t][nt][2 * i + k];
            y = see[t][i] ? y * cr[nt][k] * ks : -INFINITY;
          }
      }
    // maxima of the heads 2j, 2j + 1; a visible score of -inf counts as the lowest number
    bool grow = false;
    float nm[NT][2], nw[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float v = -INFINITY, w = -INFINITY;
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float y = x[t][nt][2 * i + k];
            v = fmaxf(v, see[t][i] ? fmaxf(y, kLowest) : -INFINITY);
            if constexpr (QUANT) w = fmaxf(w, see[t][i] ? fmaxf(y + lv[t][i], kLowest) : -INFINITY);
          }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
          if constexpr (QUANT) w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, d));
        }
        nm[nt][k] = fmaxf(m[nt][k], v);
        nw[nt][k] = QUANT ? fmaxf(mw[nt][k], w) : nm[nt][k];
        grow |= nm[nt][k] > m[nt][k] || (QUANT && nw[nt][k] > mw[nt][k]);
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float al = m[nt][k] == nm[nt][k] ? 1.f : ex2_approx(m[nt][k] - nm[nt][k]);
          const float aw = QUANT ? (mw[nt][k] == nw[nt][k] ? 1.f : ex2_approx(mw[nt][k] - nw[nt][k])) : al;
          l[nt][k] *= al;
#pragma unroll
          for (int e = 0; e < MT; ++e) {
            o[nt][e][k] *= aw;
            o[nt][e][2 + k] *= aw;
          }
          m[nt][k] = nm[nt][k];
          mw[nt][k] = nw[nt][k];
        }
    }
    uint32_t p[KT][NT][2];                         // weights: 16 keys x 8 heads a fragment
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float w[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float y = x[t][nt][2 * i + k];
            const float e = ex2_approx(y - (m[nt][k] == -INFINITY ? 0.f : m[nt][k]));
            l[nt][k] += e;
            w[k] = QUANT ? ex2_approx(y + lv[t][i] - (mw[nt][k] == -INFINITY ? 0.f : mw[nt][k])) : e;
          }
          p[t][nt][i] = transpose8x8(QUANT ? pack_f16x2(w[0], w[1]) : pack_bf16x2(w[0], w[1]));
        }
    // the next step's keys, before this one's values are used
    const int un = u + kPaWarps;
    if (un < u1) {
      if (++slot == TABLE) {
        slot = 0;
        here = next;
        next = fetch(un + TABLE * kPaWarps);
      }
      load_k(un, here, slot);
    }
#pragma unroll
    for (int t = 0; t < KT; ++t) {
#pragma unroll
      for (int e = 0; e < MT; ++e) {
        uint32_t f[4];
        if constexpr (QUANT) {
          // rows: code e of the lane's first 8 (4) codes, and of its last ones; two codes of two keys a word
          constexpr int HALF = D / 16;             // codes of a half
#pragma unroll
          for (int i = 0; i < 4; ++i) {            // f[0], f[1]: keys 2j, 2j + 1; f[2], f[3]: 2j + 8, 2j + 9
            const int code = e + (i & 1) * HALF, w = code >> 2;
            const uint4 ra = vr[t][i & 2][0], rb = vr[t][(i & 2) + 1][0];
            const uint32_t x0 = w == 0 ? ra.x : w == 1 ? ra.y : w == 2 ? ra.z : ra.w;
            const uint32_t x1 = w == 0 ? rb.x : w == 1 ? rb.y : w == 2 ? rb.z : rb.w;
            const uint32_t pair = __byte_perm(x0, x1, code & 2 ? 0x7362 : 0x5140);
            f[i] = codes2(code & 1 ? pair >> 16 : pair);
          }
        } else {
          // rows: entry e of the lane's first piece and of its second (heads of 64: e and e + 4 of its only one)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int entry = VP == 2 ? e : e + 4 * (i & 1), pc = VP == 2 ? (i & 1) : 0, w = entry >> 1;
            const uint4 ra = vr[t][i & 2][pc], rb = vr[t][(i & 2) + 1][pc];
            const uint32_t x0 = w == 0 ? ra.x : w == 1 ? ra.y : w == 2 ? ra.z : ra.w;
            const uint32_t x1 = w == 0 ? rb.x : w == 1 ? rb.y : w == 2 ? rb.z : rb.w;
            f[i] = __byte_perm(x0, x1, entry & 1 ? 0x7632 : 0x5410);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816<QUANT>(o[nt][e], f, p[t][nt][0], p[t][nt][1]);
      }
    }
    if (un < u1) load_v(un);
  }

  // ------------------------------------------------------------------ the four warps' outputs
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float s = l[nt][k];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      const int r = nt * 8 + 2 * j + k;
      if (gq == 0) {
        sML[warp][r][0] = m[nt][k];
        sML[warp][r][1] = QUANT ? mw[nt][k] : m[nt][k];
        sML[warp][r][2] = s;
      }
#pragma unroll
      for (int e = 0; e < MT; ++e) {
        // the dimensions of the tile's rows gq and gq + 8
        const int d0 = QUANT ? (D / 8) * gq + e : 8 * gq + e;
        const int d1 = QUANT ? d0 + D / 16 : VP == 2 ? d0 + 64 : d0 + 4;
        sO[warp][r][d0] = o[nt][e][k];
        sO[warp][r][d1] = o[nt][e][2 + k];
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * D; i += 32 * kPaWarps) {
    const int r = i / D, d = i % D;
    float M = -INFINITY, W = -INFINITY;
#pragma unroll
    for (int w = 0; w < kPaWarps; ++w) {
      M = fmaxf(M, sML[w][r][0]);
      W = fmaxf(W, sML[w][r][1]);
    }
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < kPaWarps; ++w) {
      const bool any = sML[w][r][0] != -INFINITY;
      L += any ? ex2_approx(sML[w][r][0] - M) * sML[w][r][2] : 0.f;
      O += any ? ex2_approx(sML[w][r][1] - W) * sO[w][r][d] : 0.f;
    }
    const long long at = (long long)b * a.Hq + h * a.G + g0 + r;
    if (a.splits == 1) {
      const float y = M == -INFINITY ? 0.f : O / L * (QUANT ? ex2_approx(W - M) : 1.f);
      a.out[at * D + d] = __float2bfloat16_rn(y);
    } else {
      float* dst = a.part + (at * a.splits + split) * (D + 4);
      dst[d] = O;
      if (d == 0) { dst[D] = M; dst[D + 1] = W; dst[D + 2] = L; }
    }
  }
}

// The pieces of a (sequence, head) joined in order, a dimension a thread.
template <int D, bool QUANT>
__global__ void __launch_bounds__(D) paged_join_kernel(const float* __restrict__ part, __nv_bfloat16* __restrict__ out, int splits) {
  griddep_wait();
  const float* src = part + (long long)blockIdx.x * splits * (D + 4);
  const int d = threadIdx.x;
  float M = -INFINITY, W = -INFINITY;
  for (int i = 0; i < splits; ++i) {
    M = fmaxf(M, src[i * (D + 4) + D]);
    W = fmaxf(W, src[i * (D + 4) + D + 1]);
  }
  float L = 0.f, O = 0.f;
  for (int i = 0; i < splits; ++i) {
    const float* s = src + i * (D + 4);
    if (s[D] == -INFINITY) continue;
    L += ex2_approx(s[D] - M) * s[D + 2];
    O += ex2_approx(s[D + 1] - W) * s[d];
  }
  const float y = M == -INFINITY ? 0.f : O / L * (QUANT ? ex2_approx(W - M) : 1.f);
  out[(long long)blockIdx.x * D + d] = __float2bfloat16_rn(y);
}

template <int D, bool QUANT>
static void pa_launch(PaArgs& a, const KvView& c, int64_t B, cudaStream_t s) {
  const unsigned grid = (unsigned)(B * a.splits * a.Hkv * a.rg);
  if (a.G <= 8) paged_attention_kernel<D, QUANT, 2, 1><<<grid, 32 * kPaWarps, 0, s>>>(a, c);
  else paged_attention_kernel<D, QUANT, 1, 2><<<grid, 32 * kPaWarps, 0, s>>>(a, c);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (a.splits == 1) return;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((unsigned)(B * a.Hq));
  cfg.blockDim = dim3(D);
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, paged_join_kernel<D, QUANT>, (const float*)a.part, a.out, a.splits));
}

at::Tensor paged_attention(at::Tensor q, at::Tensor kp, at::Tensor vp, at::Tensor table, at::Tensor lens, double scale,
                           c10::optional<at::Tensor> ks, c10::optional<at::Tensor> vs) {
  TORCH_CHECK(kp.is_cuda(), "pages: CUDA tensors");
  bool quant;
  const KvView c = kv_view(kp, vp, ks, vs, quant);
  PaArgs a{};
  a.lg = page_log(kp.size(2));
  const int64_t Hkv = kp.size(1), D = kp.size(3);
  TORCH_CHECK(q.dim() == 3 && q.scalar_type() == at::kBFloat16 && q.device() == kp.device() && q.size(2) == D,
              "q: bfloat16 [B, Hq, D] of the pages' D on their device");
  const int64_t B = q.size(0), Hq = q.size(1);
  TORCH_CHECK(Hq >= 1 && Hkv >= 1 && Hq % Hkv == 0, "the query heads: a multiple of the pages' heads");
  a.qb = q.stride(0); a.qh = q.stride(1);
  TORCH_CHECK(q.stride(2) == 1 && (B <= 1 || a.qb % 8 == 0) && (Hq == 1 || a.qh % 8 == 0) &&
                  (reinterpret_cast<uintptr_t>(q.data_ptr()) & 15) == 0, "q: unit inner stride and 16-byte aligned rows");
  TORCH_CHECK(std::isfinite(scale) && std::isfinite((float)(scale * 1.4426950408889634)), "scale: a finite number");
  a.lens = kv_ints(lens, "lens", kp.device(), B);
  a.table = page_table(table, kp, B);
  a.tb = table.stride(0);
  a.width = (int)table.size(1);
  a.pages = (int)kp.size(0);
  c10::cuda::CUDAGuard guard(kp.device());
  auto out = at::empty({B, Hq, D}, q.options());
  if (B == 0) return out;
  a.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.G = (int)(Hq / Hkv);
  a.rg = a.G <= 8 ? 1 : (a.G + 15) / 16;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  // pieces: as many as give every SM some eight CTAs, of 128 keys at the least
  const int64_t base = B * Hkv * a.rg, room = ((int64_t)a.width << a.lg) / 128;
  a.splits = (int)std::max<int64_t>(1, std::min<int64_t>({(8LL * num_sms(kp.get_device()) + base - 1) / base, room, 256}));
  TORCH_CHECK(base * a.splits < (1LL << 31), "too many sequences and heads");
  at::Tensor part;
  if (a.splits > 1) {
    part = at::empty({B * Hq * a.splits * (D + 4)}, q.options().dtype(at::kFloat));
    a.part = part.data_ptr<float>();
  }
  auto s = at::cuda::getCurrentCUDAStream();
  if (D == 128) { if (quant) pa_launch<128, true>(a, c, B, s); else pa_launch<128, false>(a, c, B, s); }
  else { if (quant) pa_launch<64, true>(a, c, B, s); else pa_launch<64, false>(a, c, B, s); }
  return out;
}

}  // namespace tfb
