// Attention of one new token of every sequence over a cache of pages.
//
//   o = sum_t softmax_t(scale q . k_t) v_t,   t < lens[b], row t being row t % page of page table[b, t / page].
//
// The cache's bytes bound the time: 2 D products a byte at most with 8 query heads a key/value head.  So
// nothing is staged: a warp takes 16 keys a step, reads their rows as 16-byte pieces straight into the
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
// Quantised rows: codes become f16 in registers.  A key's scale multiplies its score; a value's multiplies its
// weight, which is taken relative to a maximum m' of score + log2 scale, so that weights fit f16 whatever the
// scales are.
//
// Measured on a B200 (calls replayed from a graph; floors at 6.56 TB/s).  One sequence of 131071 bf16 rows, 32 / 8 heads:
// 84 us of 82.  64 sequences of 8192 .. 16384 e4m3 rows, 32 / 8 heads, pages of 16: 288 us of 248; 360
// instructions a step, half of the issue slots, 80 of them conversions and interleaving of codes.  A decode step of 32
// sequences of 288 .. 576 bf16 rows, 10 heads, pages of 16: 16 us of 11; every CTA has one short sequence, whose
// start (lengths, pages, first rows one after another) costs as much as its rows.  Rows loaded into registers instead of
// bulk copies into a ring: 350 (e4m3 batch) and 111 us (one sequence), since a wait for one load waits for the ones
// issued after it; copies by each lane for itself: 320 and 127.
#include <ATen/ops/empty.h>

#include <atomic>

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
  int* err;
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float min_nan(float a, float b) {   // min that keeps a NaN
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ uint4 ld_shared(uint32_t at) {
  uint4 u;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(at) : "memory");
  return u;
}
__device__ __forceinline__ uint2 ld_shared8(uint32_t at) {
  uint2 u;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(u.x), "=r"(u.y) : "r"(at) : "memory");
  return u;
}

template <int D, bool QUANT, int NT>
struct PaCfg {
  static constexpr int R = 8 * NT;                 // rows for query heads
  static constexpr int KP = QUANT ? D / 64 : D / 32;      // pieces of a key row a lane
  static constexpr int VP = QUANT ? 1 : D / 64;           // of a value row (e4m3 heads of 64: half a piece)
  static constexpr int VB = QUANT && D == 64 ? 8 : 16;    // bytes of one
  static constexpr int NS = QUANT || D == 64 ? 3 : 2;     // steps of a warp in flight and in use
  static constexpr uint32_t ROW = D * (QUANT ? 1u : 2u);
  static constexpr uint32_t STEP = 2 * 16 * ROW;          // 16 key rows, 16 value rows
  static constexpr uint32_t RING = kPaWarps * NS * STEP;
  static constexpr uint32_t OUT = kPaWarps * R * (D + 4) * 4u;
  static constexpr uint32_t REST = (RING > OUT ? RING : OUT);
  static constexpr uint32_t SMEM = REST + kPaWarps * R * 3 * 4u + kPaWarps * NS * 8u + 16;
};

template <int D, bool QUANT, int NT>
__global__ void __launch_bounds__(32 * kPaWarps, NT == 2 ? 2 : D == 64 || QUANT ? 4 : 3)
    paged_attention_kernel(const PaArgs a, const __grid_constant__ KvView c) {
  using Cfg = PaCfg<D, QUANT, NT>;
  constexpr int KP = Cfg::KP, VP = Cfg::VP, VB = Cfg::VB, R = Cfg::R, NS = Cfg::NS;
  constexpr int KS = D / 16, MT = D / 16;          // steps of 16 dimensions; tiles of them in the output
  extern __shared__ __align__(128) uint8_t smem[];
  float (*sO)[R][D + 4] = reinterpret_cast<float (*)[R][D + 4]>(smem);   // over the ring, once all is read
  float (*sML)[R][3] = reinterpret_cast<float (*)[R][3]>(smem + Cfg::REST);
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + Cfg::REST + kPaWarps * R * 3 * 4);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(bars + kPaWarps * NS);
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, j = lane & 3;
  const int units = a.Hkv * a.rg;
  const int hr = (int)(blockIdx.x % units), split = (int)(blockIdx.x / units % a.splits);
  const int b = (int)(blockIdx.x / units / a.splits);
  const int h = hr / a.rg, g0 = (hr % a.rg) * R;   // key/value head, first query head of it
  const int rows = min(R, a.G - g0);
  const int len = (int)max(0LL, min((long long)a.lens[b], (long long)a.width << a.lg));
  const long long steps = ((long long)len + 15) / 16;
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
  // A warp has a ring of its own, filled by bulk copies: one for a tile whose rows are one behind another, else one a
  // lane for a row.
  uint64_t* const full = bars + warp * NS;
  if (lane == 0) {
    for (int i = 0; i < NS; ++i) mbar_init(&full[i], 1);
    if (warp == 0) *abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  uint8_t* const ring = smem + warp * (NS * Cfg::STEP);
  constexpr uint32_t VAT = 16 * Cfg::ROW;          // values behind the keys
  const bool dense = c.t == Cfg::ROW;
  // lanes 0-15 copy key rows, the others value rows (dense: lanes 0 and 16 all of them)
  const uint8_t* const r0 = (lane < 16 ? c.p[0] : c.p[1]) + h * c.h + (lane & 15) * c.t;
  const uint8_t* const s0 = QUANT ? (lane < 16 ? c.s[0] : c.s[1]) + h * c.sh + (lane & 15) * c.st : nullptr;
  const int inside = (1 << a.lg) - 1;
  // the pages of the warp's next 32 steps from step u on, one a lane
  auto fetch = [&](int u) {
    u += lane * kPaWarps;
    int pg = -1;
    if (u < u1) pg = table[(u * 16) >> a.lg];
    return pg >= 0 && pg < a.pages ? pg : -1;
  };
  int ul = u0 + warp, slot = 0, stage = 0;         // next step to load, where its page and its rows are
  int here = fetch(ul), next = fetch(ul + 32 * kPaWarps);
  int pages[NS];                                   // of the steps in flight, oldest first (-1: not there)
  uint32_t scale = 127u;                           // scale byte of key row `lane` or of value row lane - 16, of the oldest
  // starts the loads of step ul, into the stage that all lanes have left; returns its page
  auto load = [&]() -> int {
    if (ul >= u1) return -1;
    const int page = __shfl_sync(0xffffffffu, here, slot);
    uint8_t* const to = ring + stage * Cfg::STEP + (lane < 16 ? 0 : VAT);
    const uint8_t* const src = r0 + page * c.b + (ul * 16 & inside) * c.t;
    if (page < 0) {
      if (lane == 0) mbar_arrive(&full[stage]);
    } else if (dense) {
      if (lane == 0) mbar_arrive_expect_tx(&full[stage], Cfg::STEP);
      __syncwarp();
      if ((lane & 15) == 0) bulk_load(to, src, VAT, &full[stage]);
    } else {
      if (lane == 0) mbar_arrive_expect_tx(&full[stage], Cfg::STEP);
      __syncwarp();
      bulk_load(to + (lane & 15) * Cfg::ROW, src, Cfg::ROW, &full[stage]);
    }
    if (++stage == NS) stage = 0;
    ul += kPaWarps;
    if (++slot == 32) {
      slot = 0;
      here = next;
      next = fetch(ul + 32 * kPaWarps);
    }
    return page;
  };
  // the scale byte of step u in page `page`
  auto load_scale = [&](int u, int page) -> uint32_t {
    const int key = u * 16, in = key & inside;
    if (!QUANT || page < 0 || key + (lane & 15) >= len) return 127u;
    return s0[page * c.sb + in * c.st];
  };

  // References of the weights: m of the sum's, mw of those that the values are multiplied by (QUANT; else m).  They move
  // when a score is above them by more than 8 (in log2), so weights are at most 2^8 and outputs rarely rescaled.
  float o[NT][MT][4];
  float2 m[NT], mw[NT], nref[NT], back[NT], l[NT];  // of heads 2j, 2j + 1; -m (0 for none), 2^(m - mw)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < MT; ++e) o[nt][e][0] = o[nt][e][1] = o[nt][e][2] = o[nt][e][3] = 0.f;
    m[nt] = mw[nt] = make_float2(-INFINITY, -INFINITY);
    nref[nt] = l[nt] = make_float2(0.f, 0.f);
    back[nt] = make_float2(1.f, 1.f);
  }

  // ------------------------------------------------------------------ the warp's steps
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) pages[i] = load();
  uint32_t at = smem_u32(ring), phase = 0;
  int cur = 0;
  scale = load_scale(u0 + warp, pages[0]);
#pragma unroll 1
  for (int u = u0 + warp; u < u1; u += kPaWarps) {
    if (!mbar_wait_warp(&full[cur], phase, abort_flag, a.err, ERR_TIMEOUT_PRODUCER)) {
      // give up, once what was started has come or had its time
      const unsigned long long t0 = globaltimer_ns();
      for (int v = u; v < ul; v += kPaWarps) {
        while (!mbar_try_wait(&full[cur], phase))
          if (globaltimer_ns() - t0 > 100000000ull) break;
        if (++cur == NS) { cur = 0; phase ^= 1; }
      }
      break;
    }
    uint4 kr[2][KP];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int p = 0; p < KP; ++p) kr[i][p] = ld_shared(at + (gq + 8 * i) * Cfg::ROW + 64 * p + 16 * j);
    const uint32_t sc = scale;
    const int left = pages[0] >= 0 ? len - u * 16 : 0;   // rows that are seen (16 or more: all)
    const bool seen[2] = {gq < left, gq + 8 < left};
    if (QUANT) scale = load_scale(u + kPaWarps, u + kPaWarps < u1 ? pages[1] : -1);
    // into the stage of the step before
    __syncwarp();
    pages[NS - 1] = load();
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) pages[i] = pages[i + 1];
    float x[NT][4], x1[NT][4];                     // of even and odd steps: two chains of products
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = x1[nt][0] = x1[nt][1] = x1[nt][2] = x1[nt][3] = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      uint32_t f[4];
      if constexpr (QUANT) {
        const uint4 r0 = kr[0][s >> 2], r1 = kr[1][s >> 2];
        const uint32_t w0 = (s & 3) == 0 ? r0.x : (s & 3) == 1 ? r0.y : (s & 3) == 2 ? r0.z : r0.w;
        const uint32_t w1 = (s & 3) == 0 ? r1.x : (s & 3) == 1 ? r1.y : (s & 3) == 2 ? r1.z : r1.w;
        f[0] = codes2(w0); f[1] = codes2(w1); f[2] = codes2_high(w0); f[3] = codes2_high(w1);
      } else {
        const uint4 r0 = kr[0][s >> 1], r1 = kr[1][s >> 1];
        f[0] = s & 1 ? r0.z : r0.x; f[1] = s & 1 ? r1.z : r1.x; f[2] = s & 1 ? r0.w : r0.y; f[3] = s & 1 ? r1.w : r1.y;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma16816<QUANT>(s & 1 ? x1[nt] : x[nt], f, q[nt][2 * s], q[nt][2 * s + 1]);
    }
    float ks[2] = {1.f, 1.f}, vs[2] = {1.f, 1.f}, lv[2] = {0.f, 0.f};   // scales of keys gq (0) and gq + 8, log2 of the values'
    if constexpr (QUANT) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ks[i] = scale_float((uint8_t)__shfl_sync(0xffffffffu, sc, 8 * i + gq));
        const uint32_t e = __shfl_sync(0xffffffffu, sc, 16 + 8 * i + gq);
        vs[i] = scale_float((uint8_t)e);
        lv[i] = __uint_as_float(0x4b000000u | e) - 8388735.f;   // 2^23 + e less 2^23 + 127 (a NaN's is not used)
      }
    }
    float2 y[NT][2];                               // scores, heads 2j and 2j + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 f = QUANT ? __fmul2_rn(make_float2(cr[nt][0], cr[nt][1]), make_float2(ks[i], ks[i])) : make_float2(cr[nt][0], cr[nt][1]);
        y[nt][i] = __fmul2_rn(__fadd2_rn(make_float2(x[nt][2 * i], x[nt][2 * i + 1]), make_float2(x1[nt][2 * i], x1[nt][2 * i + 1])), f);
        if (!seen[i]) y[nt][i] = make_float2(-INFINITY, -INFINITY);
      }
    // the lane's maxima; a visible score of -inf counts as the lowest number, so that something is seen
    const float low = seen[0] || seen[1] ? kLowest : -INFINITY;
    float2 v[NT], w[NT];
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      v[nt] = make_float2(max3f(y[nt][0].x, y[nt][1].x, low), max3f(y[nt][0].y, y[nt][1].y, low));
      grow |= v[nt].x > m[nt].x + 8.f || v[nt].y > m[nt].y + 8.f;
      if constexpr (QUANT) {
        const float2 w0 = __fadd2_rn(y[nt][0], make_float2(lv[0], lv[0])), w1 = __fadd2_rn(y[nt][1], make_float2(lv[1], lv[1]));
        w[nt] = make_float2(max3f(w0.x, w1.x, low), max3f(w0.y, w1.y, low));
        grow |= w[nt].x > mw[nt].x + 8.f || w[nt].y > mw[nt].y + 8.f;
      }
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if constexpr (!QUANT) w[nt] = v[nt];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          v[nt].x = fmaxf(v[nt].x, __shfl_xor_sync(0xffffffffu, v[nt].x, d));
          v[nt].y = fmaxf(v[nt].y, __shfl_xor_sync(0xffffffffu, v[nt].y, d));
          if constexpr (QUANT) {
            w[nt].x = fmaxf(w[nt].x, __shfl_xor_sync(0xffffffffu, w[nt].x, d));
            w[nt].y = fmaxf(w[nt].y, __shfl_xor_sync(0xffffffffu, w[nt].y, d));
          }
        }
        if constexpr (!QUANT) w[nt] = v[nt];
        auto step = [](float& ref, float to, float& factor) {   // ref moves up to `to`: what it scales, times factor
          factor = to > ref ? ex2_approx(ref - to) : 1.f;
          ref = fmaxf(ref, to);
        };
        float2 al, aw;
        step(m[nt].x, v[nt].x, al.x);
        step(m[nt].y, v[nt].y, al.y);
        if constexpr (QUANT) {
          step(mw[nt].x, w[nt].x, aw.x);
          step(mw[nt].y, w[nt].y, aw.y);
        } else {
          mw[nt] = m[nt];
          aw = al;
        }
        l[nt] = __fmul2_rn(l[nt], al);
#pragma unroll
        for (int e = 0; e < MT; ++e) {
          o[nt][e][0] *= aw.x; o[nt][e][1] *= aw.y;
          o[nt][e][2] *= aw.x; o[nt][e][3] *= aw.y;
        }
        nref[nt] = make_float2(m[nt].x == -INFINITY ? 0.f : -m[nt].x, m[nt].y == -INFINITY ? 0.f : -m[nt].y);
        if constexpr (QUANT)
          back[nt] = make_float2(m[nt].x == -INFINITY ? 1.f : ex2_approx(m[nt].x - mw[nt].x), m[nt].y == -INFINITY ? 1.f : ex2_approx(m[nt].y - mw[nt].y));
      }
    }
    uint32_t p[NT][2];                             // weights: 16 keys x 8 heads a fragment
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float2 e = __fadd2_rn(y[nt][i], nref[nt]);
        e = make_float2(ex2_approx(e.x), ex2_approx(e.y));
        l[nt] = __fadd2_rn(l[nt], e);
        if constexpr (QUANT) {
          // 2^(score - mw) times the value's scale.  The factor is 2^126 at most, so that 0 times it is 0 (a weight of 0 with a
          // factor beyond that counts less than 2^-100 of the others unless scales are that far apart); a NaN stays.
          const float2 f = __fmul2_rn(back[nt], make_float2(vs[i], vs[i]));
          e = __fmul2_rn(e, make_float2(min_nan(f.x, 0x1p126f), min_nan(f.y, 0x1p126f)));
        }
        p[nt][i] = transpose8x8(QUANT ? pack_f16x2(e.x, e.y) : pack_bf16x2(e.x, e.y));
      }
    uint4 vr[4][VP];                               // keys 2j, 2j + 1, 2j + 8, 2j + 9; rows that are not seen: zeros
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = 2 * j + (i >> 1) * 8 + (i & 1);
#pragma unroll
      for (int p = 0; p < VP; ++p) {
        const uint32_t from = at + VAT + key * Cfg::ROW + VB * gq + 128 * p;
        if constexpr (VB == 8) {
          const uint2 w2 = ld_shared8(from);
          vr[i][p] = make_uint4(w2.x, w2.y, 0, 0);
        } else {
          vr[i][p] = ld_shared(from);
        }
      }
    }
    if (left < 16) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (2 * j + (i >> 1) * 8 + (i & 1) >= left)
#pragma unroll
          for (int p = 0; p < VP; ++p) vr[i][p] = make_uint4(0, 0, 0, 0);
    }
    at += Cfg::STEP;
    if (++cur == NS) {
      cur = 0;
      at = smem_u32(ring);
      phase ^= 1;
    }
#pragma unroll
    for (int e = 0; e < MT; ++e) {
      uint32_t f[4];
      if constexpr (QUANT) {
        // rows: code e of the lane's first 8 (4) codes, and of its last ones; two codes of two keys a word
        constexpr int HALF = D / 16;               // codes of a half
#pragma unroll
        for (int i = 0; i < 4; ++i) {              // f[0], f[1]: keys 2j, 2j + 1; f[2], f[3]: 2j + 8, 2j + 9
          const int code = e + (i & 1) * HALF, wd = code >> 2;
          const uint4 ra = vr[i & 2][0], rb = vr[(i & 2) + 1][0];
          const uint32_t x0 = wd == 0 ? ra.x : wd == 1 ? ra.y : wd == 2 ? ra.z : ra.w;
          const uint32_t x1 = wd == 0 ? rb.x : wd == 1 ? rb.y : wd == 2 ? rb.z : rb.w;
          const uint32_t pair = __byte_perm(x0, x1, code & 2 ? 0x7362 : 0x5140);
          f[i] = code & 1 ? codes2_high(pair) : codes2(pair);
        }
      } else {
        // rows: entry e of the lane's first piece and of its second (heads of 64: e and e + 4 of its only one)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int entry = VP == 2 ? e : e + 4 * (i & 1), pc = VP == 2 ? (i & 1) : 0, wd = entry >> 1;
          const uint4 ra = vr[i & 2][pc], rb = vr[(i & 2) + 1][pc];
          const uint32_t x0 = wd == 0 ? ra.x : wd == 1 ? ra.y : wd == 2 ? ra.z : ra.w;
          const uint32_t x1 = wd == 0 ? rb.x : wd == 1 ? rb.y : wd == 2 ? rb.z : rb.w;
          f[i] = __byte_perm(x0, x1, entry & 1 ? 0x7632 : 0x5410);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma16816<QUANT>(o[nt][e], f, p[nt][0], p[nt][1]);
    }
  }

  __syncthreads();                                 // no warp is in its ring any more

  // ------------------------------------------------------------------ the four warps' outputs
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float s = k ? l[nt].y : l[nt].x;
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      const int r = nt * 8 + 2 * j + k;
      if (gq == 0) {
        sML[warp][r][0] = k ? m[nt].y : m[nt].x;
        sML[warp][r][1] = k ? mw[nt].y : mw[nt].x;
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
      if (d == 0) *reinterpret_cast<float4*>(dst + D) = make_float4(M, W, L, 0.f);
    }
  }
}

// The pieces of a (sequence, head) joined: eight warps take every eighth piece, in order, and their sums are added in order.
constexpr int kJoinWarps = 8;
template <int D, bool QUANT>
__global__ void __launch_bounds__(32 * kJoinWarps) paged_join_kernel(const float* __restrict__ part, __nv_bfloat16* __restrict__ out, int splits) {
  constexpr int E = D / 32;
  __shared__ float sO[kJoinWarps][D], sL[kJoinWarps];
  griddep_wait();
  const float* src = part + (long long)blockIdx.x * splits * (D + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float M = -INFINITY, W = -INFINITY;
  for (int i = lane; i < splits; i += 32) {
    M = fmaxf(M, src[(long long)i * (D + 4) + D]);
    W = fmaxf(W, src[(long long)i * (D + 4) + D + 1]);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
    W = fmaxf(W, __shfl_xor_sync(0xffffffffu, W, d));
  }
  float L = 0.f, O[E];
#pragma unroll
  for (int e = 0; e < E; ++e) O[e] = 0.f;
#pragma unroll 4
  for (int i = warp; i < splits; i += kJoinWarps) {
    const float* s = src + (long long)i * (D + 4);
    const float4 ml = *reinterpret_cast<const float4*>(s + D);
    float o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = s[e * 32 + lane];
    const bool any = ml.x != -INFINITY;            // a piece that saw nothing
    L += any ? ex2_approx(ml.x - M) * ml.z : 0.f;
    const float f = any ? ex2_approx(ml.y - W) : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) O[e] += any ? f * o[e] : 0.f;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) sO[warp][e * 32 + lane] = O[e];
  if (lane == 0) sL[warp] = L;
  __syncthreads();
  if (threadIdx.x >= D) return;
  L = 0.f;
  float y = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) {
    L += sL[w];
    y += sO[w][threadIdx.x];
  }
  y = M == -INFINITY ? 0.f : y / L * (QUANT ? ex2_approx(W - M) : 1.f);
  out[(long long)blockIdx.x * D + threadIdx.x] = __float2bfloat16_rn(y);
}

template <int D, bool QUANT, int NT>
static void pa_run(const PaArgs& a, const KvView& c, unsigned grid, cudaStream_t s, bool on) {
  if (!on) return;
  constexpr uint32_t smem = PaCfg<D, QUANT, NT>::SMEM;
  // said once a device: the call takes longer than the launch
  static std::atomic<uint64_t> done{0};
  int dev;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (!(done.load(std::memory_order_relaxed) & bit)) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(paged_attention_kernel<D, QUANT, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    done.fetch_or(bit, std::memory_order_relaxed);
  }
  paged_attention_kernel<D, QUANT, NT><<<grid, 32 * kPaWarps, smem, s>>>(a, c);
}

template <int D, bool QUANT>
static void pa_launch(PaArgs& a, const KvView& c, int64_t B, cudaStream_t s) {
  const unsigned grid = (unsigned)(B * a.splits * a.Hkv * a.rg);
  pa_run<D, QUANT, 1>(a, c, grid, s, a.G <= 8);
  pa_run<D, QUANT, 2>(a, c, grid, s, a.G > 8);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (a.splits == 1) return;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((unsigned)(B * a.Hq));
  cfg.blockDim = dim3(32 * kJoinWarps);
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, paged_join_kernel<D, QUANT>, (const float*)a.part, a.out, a.splits));
}

at::Tensor paged_attention(at::Tensor q, at::Tensor kp, at::Tensor vp, at::Tensor table, at::Tensor lens, double scale,
                           c10::optional<at::Tensor> ks, c10::optional<at::Tensor> vs, at::Tensor err) {
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
  a.err = err.data_ptr<int>();
  // Pieces.  One sequence: as many as fill the GPU once, since they are alike, of 128 rows at the least.  More
  // sequences, whose lengths the host does not know: six times as many as fit, so that long ones do not stand out, of
  // 512 rows at the least.
  const int64_t base = Hkv * a.rg, slots = (int64_t)num_sms(kp.get_device()) * (quant ? 3 : 2), rows = (int64_t)a.width << a.lg;
  const int64_t want = B == 1 ? std::min(slots / base, rows / 128) : std::min((6 * slots + B * base - 1) / (B * base), rows / 512);
  a.splits = (int)std::max<int64_t>(1, std::min<int64_t>(want, 256));
  TORCH_CHECK(B * base * a.splits < (1LL << 31), "too many sequences and heads");
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
