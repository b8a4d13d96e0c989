// Log probabilities of given tokens, entropies and the likeliest alternatives of rows of logits,
// and the gradient of the first two.
//
// With m the row's maximum, S = sum e^(z - m) and T = sum e^(z - m) (z - m):
//   log p_v = (z_v - m) - log S,   H = log S - T / S,
//   dz_v = g ([v = token] - p_v) - h p_v (log p_v + H)     (g, h: gradients of log p_token and H).
// All of it is held in 32 bits; m and log S are kept apart for the gradient, since their sum would
// round away what a small log p is made of.
//
// The bytes bound both directions, so a row is read once, as a stream: a warp has a share of it, 512 bytes a
// load, four loads ahead; a lane keeps a maximum and sums of its own, and its maxima over 16 blocks of the share.
// Alternatives are found afterwards: the k-th largest of the lanes' maxima is a bound that only few (block, lane) pairs
// reach (some 7 of 512 for five alternatives), and only their logits are read again, and taken in one by one,
// by (logit, lowest token first).  (Keeping the best so far while streaming took in 42 logits of a row of 8192 instead
// of 7: 134 us for 16384 rows.)  Nothing waits for another warp until the row's end.
// With many rows a warp has a whole one; with fewer a CTA's eight warps, or those of a cluster of up to 8
// CTAs, share it and are joined through (distributed) shared memory.
// Measured on a B200 (calls replayed from a graph).  16384 rows of 8192 fp32 logits with five alternatives: 107 us of 82 (HBM,
// 76 % of the copy rate; 3800 instructions a row).  4096 rows of 131072 bf16 logits: 234 us of 164 forward (the
// exponentials alone, 16 a cycle of an SM, take 120), gradient 358 of 327.  8 rows of 131072 fp32 logits with eight
// alternatives: 10.8 us; a chain of loads, sums, candidates and a cluster's joins.
// The reference has no counterpart; its losses are those of fused_ops.cu.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>

#include <tuple>
#include <vector>

#include "attention_tiles.cuh"

namespace tfb {

int num_sms(int dev);

constexpr int kLpWarps = 8;      // of a CTA
constexpr int kLpLoads = 4;      // of a lane a step
constexpr int kLpBlocks = 16;    // of a warp's share, for the alternatives
constexpr int kLpMaxTop = 32;
constexpr int kLpCand = 64;
typedef unsigned long long u64;

struct LpArgs {
  const void* z;
  long long ld;                  // elements between rows
  const void* tok;
  int tok64;
  int V, top;
  int W, C;                      // warps and CTAs a row (C > 1: W is all of a CTA's)
  long long N;
  float *lp, *ent, *stat;        // stat [N, 3]: m, log S, H
  int* top_tok;
  float* top_lp;
};

__device__ __forceinline__ long long lp_token(const void* t, int is64, long long row) {
  return is64 ? static_cast<const long long*>(t)[row] : static_cast<const int*>(t)[row];
}

// Order of the logits as unsigned numbers: -inf .. +inf, then NaN; -0 as +0.
__device__ __forceinline__ uint32_t lp_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lp_unkey(uint32_t k) {
  return __uint_as_float(k == 0xffffffffu ? 0x7fffffffu : (k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ u64 ld_dsmem_u64(uint32_t addr) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What logits of a share whose maximum is m are taken relative to: -inf (nothing in it counts) would give NaN
__device__ __forceinline__ float lp_ref(float m) { return m == -INFINITY ? 0.f : m; }

// Sums S and T against the maximum m as sums against M >= m.  An m of -inf comes with sums of 0 (or of NaN, which
// stay); e^-1e4 is 0, and 0 * inf never comes up.
__device__ __forceinline__ void lp_rebase(float m, float M, float& S, float& T) {
  const float d = m - M;
  const float e = m == -INFINITY ? 1.f : __expf(d);
  if (m != -INFINITY) T += fmaxf(d, -1e4f) * S;
  T *= e;
  S *= e;
}

// BF: bf16 logits, else fp32.  VEC: 16-byte loads (rows 16-byte aligned), else one element each.
template <bool BF, bool VEC>
struct LpStep {
  static constexpr int EPL = VEC ? (BF ? 8 : 4) : 1;           // elements of a load
  static constexpr int LOADS = VEC ? (BF ? kLpLoads / 2 : kLpLoads) : 4 * kLpLoads;   // 16 elements a lane
  static constexpr int EL = EPL * LOADS;                       // elements of a lane
  static constexpr int SIZE = 32 * EL;                         // of a step
  static constexpr int WORDS = VEC ? 4 * LOADS : LOADS;
  uint32_t r[WORDS];

  // a lane's i-th element's place in the row
  static __device__ __forceinline__ int place(int first, int i, int lane) { return first + (i / EPL * 32 + lane) * EPL + i % EPL; }
  // elements past the row's end are -inf
  __device__ __forceinline__ void load(const void* row, int first, int V) {
    const bool whole = first + SIZE <= V;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int e = place(first, j * EPL, threadIdx.x & 31);
      if constexpr (VEC) {
        uint4 u;
        if (whole || e + EPL <= V) {
          u = __ldg(reinterpret_cast<const uint4*>(static_cast<const char*>(row) + (long long)e * (BF ? 2 : 4)));
        } else {
          uint32_t w[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            if constexpr (BF) {
              const uint32_t lo = e + 2 * x < V ? static_cast<const uint16_t*>(row)[e + 2 * x] : 0xff80u;
              const uint32_t hi = e + 2 * x + 1 < V ? static_cast<const uint16_t*>(row)[e + 2 * x + 1] : 0xff80u;
              w[x] = lo | (hi << 16);
            } else {
              w[x] = e + x < V ? static_cast<const uint32_t*>(row)[e + x] : 0xff800000u;
            }
          }
          u = make_uint4(w[0], w[1], w[2], w[3]);
        }
        r[4 * j] = u.x; r[4 * j + 1] = u.y; r[4 * j + 2] = u.z; r[4 * j + 3] = u.w;
      } else {
        r[j] = 0xff800000u;
        if (e < V) r[j] = BF ? (uint32_t)static_cast<const uint16_t*>(row)[e] << 16 : static_cast<const uint32_t*>(row)[e];
      }
    }
  }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (BF && VEC) return __uint_as_float(i & 1 ? r[i >> 1] & 0xffff0000u : r[i >> 1] << 16);
    else return __uint_as_float(r[i]);
  }
};

// The best logits so far, lane i's the i-th: key 0 is none.
struct LpBest {
  uint32_t key = 0;
  int at = 0;
  // a logit better than one of the top ones (all lanes agree on it) takes its place
  __device__ __forceinline__ void insert(uint32_t k, int a) {
    const bool better = key > k || (key == k && at < a);
    const int place = __popc(__ballot_sync(0xffffffffu, better));
    const uint32_t pk = __shfl_up_sync(0xffffffffu, key, 1);
    const int pa = __shfl_up_sync(0xffffffffu, at, 1), lane = threadIdx.x & 31;
    if (lane > place) { key = pk; at = pa; }
    if (lane == place) { key = k; at = a; }
  }
};

// What a warp keeps for the alternatives of its share.
struct LpShare {
  float block[kLpBlocks * 32];             // the lanes' maxima over the blocks
  uint16_t pair[kLpBlocks * 32];           // (block, lane) pairs that reach the bound
  u64 cand[kLpCand];                       // logits that do
  u64 best[kLpMaxTop];
};

// The top best logits of a warp's share, steps c0 .. c1 - 1 in blocks of `per`, as lane i's i-th (0: none).  The
// top-th largest of the lanes' maxima (`mine`) is at most the top-th largest logit, so only (block, lane) pairs that
// reach it have some.  Their logits are read again, 32 at a time, and those that reach it are collected and ranked; more than
// kLpCand of them (equal logits) are taken in one by one instead.
template <bool BF, bool VEC>
__device__ __forceinline__ u64 best_of_share(const char* z, int V, int top, int c0, int c1, int per, float mine, LpShare& sh) {
  typedef LpStep<BF, VEC> Step;
  const int lane = threadIdx.x & 31;
  uint32_t k = lp_key(mine), least = 0;
  for (int i = 0; i < top; ++i) {
    least = __reduce_max_sync(0xffffffffu, k);
    if (lane == __ffs(__ballot_sync(0xffffffffu, k == least)) - 1) k = 0;
  }
  int pairs = 0;
  const int nb = (c1 - c0 + per - 1) / per;
  for (int b = 0; b < nb; ++b) {
    const bool hot = lp_key(sh.block[b * 32 + lane]) >= least;
    const unsigned in = __ballot_sync(0xffffffffu, hot);
    if (hot) sh.pair[pairs + __popc(in & ((1u << lane) - 1))] = (uint16_t)(b * 32 + lane);
    pairs += __popc(in);
  }
  sh.best[lane] = 0;
  __syncwarp();
  // the i-th logit of all pairs' logits, 0: there is none
  const int each = per * Step::EL, all = pairs * each;
  auto logit = [&](int i, int& e) -> uint32_t {
    if (i >= all) return 0u;
    const int p = sh.pair[i / each], x = i % each, c = c0 + (p >> 5) * per + x / Step::EL;
    e = Step::place(c * Step::SIZE, x % Step::EL, p & 31);
    if (c >= c1 || e >= V) return 0u;
    return lp_key(BF ? __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(z)[e] << 16) : reinterpret_cast<const float*>(z)[e]);
  };
  int n = 0;
  for (int i0 = 0; i0 < all && n <= kLpCand; i0 += 128) {
    uint32_t q[4];
    int e[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = logit(i0 + 32 * j + lane, e[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool ok = q[j] != 0 && q[j] >= least;
      const unsigned in = __ballot_sync(0xffffffffu, ok);
      const int at = n + __popc(in & ((1u << lane) - 1));
      if (ok && at < kLpCand) sh.cand[at] = ((u64)q[j] << 32) | (uint32_t)~e[j];
      n += __popc(in);
    }
  }
  __syncwarp();
  if (n <= kLpCand) {
    for (int i = lane; i < n; i += 32) {
      const u64 me = sh.cand[i];
      int place = 0;
      for (int j = 0; j < n; ++j) place += sh.cand[j] > me;
      if (place < top) sh.best[place] = me;
    }
    __syncwarp();
    return sh.best[lane];
  }
  LpBest best;
  int last = 0x7fffffff;                   // what a logit has to be better than: (least, last), there being `top` such
  for (int i0 = 0; i0 < all; i0 += 32) {
    int e = 0;
    const uint32_t q = logit(i0 + lane, e);
    unsigned in = __ballot_sync(0xffffffffu, q != 0 && (q > least || (q == least && e < last)));
    while (in) {
      const int l = __ffs(in) - 1;
      best.insert(__shfl_sync(0xffffffffu, q, l), __shfl_sync(0xffffffffu, e, l));
      const uint32_t full = __shfl_sync(0xffffffffu, best.key, top - 1);
      if (full) {
        least = full;
        last = __shfl_sync(0xffffffffu, best.at, top - 1);
      }
      in = (in & (in - 1)) & __ballot_sync(0xffffffffu, q > least || (q == least && e < last));
    }
  }
  return lane < top && best.key ? ((u64)best.key << 32) | (uint32_t)~best.at : 0;
}

template <bool BF, bool VEC>
__global__ void __launch_bounds__(32 * kLpWarps, 4) token_logprobs_kernel(const LpArgs a) {
  typedef LpStep<BF, VEC> Step;
  __shared__ LpShare sShare[kLpWarps];
  __shared__ float sStat[kLpWarps][3];
  __shared__ u64 sCand[kLpWarps * kLpMaxTop];
  __shared__ u64 sTop[kLpWarps * kLpMaxTop];   // of the rows (W > 1), best first (0: none)
  __shared__ float sRow[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = a.C > 1 ? (int)(blockIdx.x % a.C) : 0;
  const long long row = a.C > 1 ? blockIdx.x / a.C : (long long)blockIdx.x * (kLpWarps / a.W) + warp / a.W;
  const int part = a.C > 1 ? rank * kLpWarps + warp : warp % a.W;
  const char* z = static_cast<const char*>(a.z) + row * a.ld * (BF ? 2 : 4);
  const bool real = row < a.N;

  // ------------------------------------------------------------------ the warp's share
  float m = -INFINITY, S = 0.f, T = 0.f;
  float mine = -INFINITY, block = -INFINITY;   // maxima of the lane, NaN where there is one: of the share, of the block
  const long long steps = ((long long)a.V + Step::SIZE - 1) / Step::SIZE;
  const int parts = a.W * a.C;
  const int c0 = (int)(steps * part / parts), c1 = real ? (int)(steps * (part + 1) / parts) : 0;
  const int per = (c1 - c0 + kLpBlocks - 1) / kLpBlocks;
  int left = per;                          // steps until the block's end
  float* blocks = sShare[warp].block + lane;
  auto take = [&](const Step& x, int c) {
    float mx[4];                           // NaN where there is one
#pragma unroll
    for (int i = 0; i < 4; ++i) mx[i] = x.value(i);
#pragma unroll
    for (int i = 4; i < Step::EL; i += 8)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        mx[k] = i + 4 < Step::EL ? max3_nan(mx[k], x.value(i + k), x.value(i + 4 + k < Step::EL ? i + 4 + k : i + k)) : max_nan(mx[k], x.value(i + k));
    const float mc = max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3]));
    if (mc > m) {
      lp_rebase(m, mc, S, T);
      m = mc;
    }
    const float ref = -lp_ref(m);
    float2 s2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)}, t2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int i = 0; i < Step::EL; i += 2) {
      const float2 d = __fadd2_rn(make_float2(x.value(i), x.value(i + 1)), make_float2(ref, ref));
      const float2 l = __fmul2_rn(d, make_float2(kLog2e, kLog2e));
      const float2 e = make_float2(ex2_approx(l.x), ex2_approx(l.y));
      s2[i >> 1 & 1] = __fadd2_rn(s2[i >> 1 & 1], e);
      // e^-1e4 is 0: 0 * inf never comes up
      t2[i >> 1 & 1] = __ffma2_rn(e, make_float2(fmaxf(d.x, -1e4f), fmaxf(d.y, -1e4f)), t2[i >> 1 & 1]);
    }
    const float2 ss = __fadd2_rn(s2[0], s2[1]), tt = __fadd2_rn(t2[0], t2[1]);
    S += ss.x + ss.y;
    T += tt.x + tt.y;
    if (a.top) {
      block = max_nan(block, mc);
      if (--left == 0 || c + 1 == c1) {
        *blocks = block;
        blocks += 32;
        mine = max_nan(mine, block);
        block = -INFINITY;
        left = per;
      }
    }
  };
  Step x, y;                               // a step ahead
  if (c0 < c1) x.load(z, c0 * Step::SIZE, a.V);
#pragma unroll 1
  for (int c = c0; c < c1; c += 2) {
    if (c + 1 < c1) y.load(z, (c + 1) * Step::SIZE, a.V);
    take(x, c);
    if (c + 1 >= c1) break;
    if (c + 2 < c1) x.load(z, (c + 2) * Step::SIZE, a.V);
    take(y, c + 1);
  }
  u64 mykey = 0;                           // lane i's: the i-th best, 0: none
  if (a.top) {
    __syncwarp();
    mykey = best_of_share<BF, VEC>(z, a.V, a.top, c0, c1, max(per, 1), mine, sShare[warp]);
  }

  // ------------------------------------------------------------------ the row's
  float M = warp_max(m);
  lp_rebase(m, M, S, T);
  S = warp_sum(S);
  T = warp_sum(T);
  if (a.W > 1) {
    if (lane == 0) { sStat[warp][0] = M; sStat[warp][1] = S; sStat[warp][2] = T; }
    if (lane < a.top) sCand[warp * a.top + lane] = mykey;
    __syncthreads();
    // the row's first warp joins its W shares
    const int w0 = warp / a.W * a.W;
    for (int w = w0; w < w0 + a.W; ++w) M = fmaxf(M, sStat[w][0]);
    S = T = 0.f;
    for (int w = w0; w < w0 + a.W; ++w) {
      float sw = sStat[w][1], tw = sStat[w][2];
      lp_rebase(sStat[w][0], M, sw, tw);
      S += sw;
      T += tw;
    }
    if (a.top) {
      // a thread a share's alternative: its place is how many of the row's are better
      const int n = a.W * a.top, i = threadIdx.x - 32 * w0;
      const u64* all = sCand + w0 * a.top;
      const u64 me = i < n ? all[i] : 0;
      int place = 0;
      for (int k = 0; k < n; ++k) place += all[k] > me;
      u64* out = sTop + w0 * a.top;
      if (i < a.top) out[i] = 0;
      __syncthreads();
      if (me != 0 && place < a.top) out[place] = me;
      __syncthreads();
      mykey = lane < a.top ? out[lane] : 0;
    }
    if (warp != w0 && a.C == 1) return;
  }
  if (a.C > 1) {                           // W is 8: warp 0 has the CTA's
    if (threadIdx.x == 0) { sRow[0] = M; sRow[1] = S; sRow[2] = T; }   // its alternatives are in sTop
    cluster_sync();
    if (rank == 0 && warp == 0) {
      // lanes 0 .. C - 1 fetch the CTAs' sums, all lanes their alternatives
      float cm = -INFINITY, cs = 0.f, ct = 0.f;
      if (lane < a.C) {
        const uint32_t at = mapa_shared(smem_u32(sRow), lane);
        cm = ld_dsmem_f32(at); cs = ld_dsmem_f32(at + 4); ct = ld_dsmem_f32(at + 8);
      }
      M = warp_max(cm);
      lp_rebase(cm, M, cs, ct);
      S = warp_sum(cs);
      T = warp_sum(ct);
    }
    if (rank == 0 && a.top) {
      const int n = a.C * a.top, i = threadIdx.x;
      if (i < n) sCand[i] = ld_dsmem_u64(mapa_shared(smem_u32(sTop), i / a.top) + 8 * (i % a.top));
      __syncthreads();
      const u64 me = i < n ? sCand[i] : 0;
      int place = 0;
      for (int k = 0; k < n; ++k) place += sCand[k] > me;
      u64* out = sCand + kLpWarps * kLpMaxTop - kLpMaxTop;   // n <= 256 entries are in use while places are found
      __syncthreads();
      if (i < a.top) out[i] = 0;
      __syncthreads();
      if (me != 0 && place < a.top) out[place] = me;
      __syncthreads();
      mykey = lane < a.top ? out[lane] : 0;
    }
    cluster_sync();                        // shared memory lives until rank 0 has read it
    if (rank != 0 || warp != 0) return;
  }
  if (!real) return;
  const float logs = M == -INFINITY ? __int_as_float(0x7fffffff) : logf(S);   // nothing but -inf: NaN
  if (lane == 0) {
    const long long v = lp_token(a.tok, a.tok64, row);
    float lp = 0.f;
    if (v >= 0 && v < a.V)
      lp = (BF ? __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(z)[v] << 16) : reinterpret_cast<const float*>(z)[v]) - M - logs;
    const float H = logs - T / S;
    a.lp[row] = lp;
    a.ent[row] = H;
    if (a.stat) {
      a.stat[3 * row] = M;
      a.stat[3 * row + 1] = logs;
      a.stat[3 * row + 2] = H;
    }
  }
  if (lane < a.top) {
    a.top_tok[row * a.top + lane] = (int)~(uint32_t)mykey;
    a.top_lp[row * a.top + lane] = lp_unkey((uint32_t)(mykey >> 32)) - M - logs;
  }
}

struct LpGradArgs {
  const void* z;
  long long ld, ldo;
  void* dz;
  const void* tok;
  int tok64, V, chunks;
  const float *g, *h, *stat;     // g or h null: zero
};

// Elementwise: a CTA has 256 threads' loads of one row, four each, and their stores.
template <bool BF, bool VEC>
__global__ void __launch_bounds__(256) token_logprobs_grad_kernel(const LpGradArgs a) {
  constexpr int EPL = VEC ? (BF ? 8 : 4) : 1, U = 4;
  const long long row = blockIdx.x / a.chunks;
  const int i0 = (int)(blockIdx.x % a.chunks) * (U * 256) + threadIdx.x;
  const char* z = static_cast<const char*>(a.z) + row * a.ld * (BF ? 2 : 4);
  char* dz = static_cast<char*>(a.dz) + row * a.ldo * (BF ? 2 : 4);
  uint4 u[U];
#pragma unroll
  for (int j = 0; j < U; ++j) {
    const int e = (i0 + j * 256) * EPL;
    u[j] = make_uint4(0, 0, 0, 0);
    if constexpr (VEC) {
      if (e + EPL <= a.V) {
        u[j] = __ldg(reinterpret_cast<const uint4*>(z) + i0 + j * 256);
      } else if (e < a.V) {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < EPL; ++x)
          if (e + x < a.V) {
            if constexpr (BF) w[x >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(z)[e + x] << (16 * (x & 1));
            else w[x] = reinterpret_cast<const uint32_t*>(z)[e + x];
          }
        u[j] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else if (e < a.V) {
      u[j].x = BF ? (uint32_t)reinterpret_cast<const uint16_t*>(z)[e] << 16 : reinterpret_cast<const uint32_t*>(z)[e];
    }
  }
  const float m = a.stat[3 * row], logs = a.stat[3 * row + 1], H = a.stat[3 * row + 2];
  const long long tok = lp_token(a.tok, a.tok64, row);
  const float g = a.g && tok >= 0 && tok < a.V ? a.g[row] : 0.f, h = a.h ? a.h[row] : 0.f;
  auto grad = [&](float v, long long e) {
    const float l = v - m - logs, p = __expf(l);
    return (e == tok ? g : 0.f) - p * (g + h * (fmaxf(l, -1e4f) + H));   // e^-1e4 is 0
  };
#pragma unroll
  for (int j = 0; j < U; ++j) {
    const long long e = (long long)(i0 + j * 256) * EPL;
    if (e >= a.V) continue;
    if constexpr (VEC) {
      uint32_t w[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if constexpr (BF) w[x] = pack_bf16x2(grad(__uint_as_float(w[x] << 16), e + 2 * x), grad(__uint_as_float(w[x] & 0xffff0000u), e + 2 * x + 1));
        else w[x] = __float_as_uint(grad(__uint_as_float(w[x]), e + x));
      }
      if (e + EPL <= a.ldo) {    // the gradient's rows are padded to whole stores
        reinterpret_cast<uint4*>(dz)[i0 + j * 256] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else if constexpr (BF) {
      reinterpret_cast<__nv_bfloat16*>(dz)[e] = __float2bfloat16_rn(grad(__uint_as_float(u[j].x), e));
    } else {
      reinterpret_cast<float*>(dz)[e] = grad(__uint_as_float(u[j].x), e);
    }
  }
}

struct LpShape {
  at::Tensor z, tok;             // [N, V] and packed [N]
  bool bf, vec;
  int64_t N, V, ld;
};

static LpShape lp_check(const at::Tensor& logits, const at::Tensor& tokens, int64_t top) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() >= 1 && (logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16),
              "logits: float32 or bfloat16 [..., V]");
  LpShape s{};
  s.bf = logits.scalar_type() == at::kBFloat16;
  s.V = logits.size(-1);
  TORCH_CHECK(s.V >= 1 && s.V <= (1 << 30), "vocabulary of 1 .. 2^30 tokens");
  TORCH_CHECK(s.V == 1 || logits.stride(-1) == 1, "logits: unit inner stride");
  TORCH_CHECK((tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt) && tokens.device() == logits.device() &&
                  tokens.sizes() == logits.sizes().slice(0, logits.dim() - 1),
              "tokens: int64 or int32, one for each row of the logits, on their device");
  TORCH_CHECK(top >= 0 && top <= kLpMaxTop && top <= s.V, "top: 0 .. 32 alternatives, at most the vocabulary");
  s.N = tokens.numel();
  TORCH_CHECK(s.N <= (1 << 27), "at most 2^27 rows");
  s.z = logits.dim() == 2 ? logits : logits.reshape({s.N, s.V});
  s.tok = tokens.contiguous();
  s.ld = s.z.stride(0);
  s.vec = (reinterpret_cast<uintptr_t>(s.z.data_ptr()) & 15) == 0 && (s.N <= 1 || s.ld * s.z.element_size() % 16 == 0);
  return s;
}

// (log probabilities, entropies, alternatives and their log probabilities, what the gradient needs or nothing)
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, c10::optional<at::Tensor>> token_logprobs(at::Tensor logits, at::Tensor tokens,
                                                                                                     int64_t top, bool stats) {
  const LpShape s = lp_check(logits, tokens, top);
  const at::Tensor &z = s.z, &tok = s.tok;
  c10::cuda::CUDAGuard guard(z.device());
  const auto f32 = z.options().dtype(at::kFloat);
  auto lp = at::empty(tokens.sizes(), f32), ent = at::empty(tokens.sizes(), f32);
  std::vector<int64_t> wide(tokens.sizes().begin(), tokens.sizes().end());
  wide.push_back(top);
  auto top_lp = at::empty(wide, f32), top_tok = at::empty(wide, z.options().dtype(at::kInt));
  c10::optional<at::Tensor> stat;
  if (stats) stat = at::empty({s.N, 3}, f32);
  if (s.N == 0) return {lp, ent, top_tok, top_lp, stat};
  LpArgs a{};
  a.z = z.data_ptr(); a.ld = s.ld; a.tok = tok.data_ptr(); a.tok64 = tok.scalar_type() == at::kLong;
  a.V = (int)s.V; a.top = (int)top; a.N = s.N;
  // warps a row: one where the rows alone give every SM's 24 warps several rows each, else more while each has 16
  // steps of it, or, to have a warp for every scheduler four times over, two
  const int64_t step = 512, sms = num_sms(z.get_device());
  int W = 1, C = 1;
  while (W < kLpWarps && ((s.N * W < 192 * sms && 32 * W * step <= s.V) || (s.N * W < 16 * sms && 2 * W * step < s.V))) W *= 2;
  while (W == kLpWarps && C < 8 && s.N * W * C < 16 * sms && 2 * W * C * step < s.V) C *= 2;
  a.W = W; a.C = C;
  a.lp = lp.data_ptr<float>(); a.ent = ent.data_ptr<float>(); a.stat = stats ? stat->data_ptr<float>() : nullptr;
  a.top_tok = top_tok.data_ptr<int>(); a.top_lp = top_lp.data_ptr<float>();
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((unsigned)(C > 1 ? s.N * C : (s.N * W + kLpWarps - 1) / kLpWarps));
  cfg.blockDim = dim3(32 * kLpWarps);
  cfg.stream = at::cuda::getCurrentCUDAStream();
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 1 : 0;
  auto* kern = s.bf ? (s.vec ? token_logprobs_kernel<true, true> : token_logprobs_kernel<true, false>)
                    : (s.vec ? token_logprobs_kernel<false, true> : token_logprobs_kernel<false, false>);
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, a));
  return {lp, ent, top_tok, top_lp, stat};
}

// dz [..., V], a view of rows padded to 16 bytes.
at::Tensor token_logprobs_grad(at::Tensor logits, at::Tensor tokens, at::Tensor stat, c10::optional<at::Tensor> g, c10::optional<at::Tensor> h) {
  const LpShape s = lp_check(logits, tokens, 0);
  const at::Tensor &z = s.z, &tok = s.tok;
  TORCH_CHECK(stat.scalar_type() == at::kFloat && stat.device() == z.device() && stat.is_contiguous() && stat.numel() == 3 * s.N, "stat: float32 [N, 3]");
  for (const auto* t : {&g, &h})
    TORCH_CHECK(!t->has_value() || ((*t)->scalar_type() == at::kFloat && (*t)->device() == z.device() && (*t)->is_contiguous() &&
                                    (*t)->numel() == s.N), "gradients: contiguous float32, one for each row");
  c10::cuda::CUDAGuard guard(z.device());
  const int64_t pad = s.bf ? 8 : 4, ldo = (s.V + pad - 1) / pad * pad;
  std::vector<int64_t> wide(tokens.sizes().begin(), tokens.sizes().end());
  wide.push_back(ldo);
  auto dz = at::empty(wide, z.options());
  if (s.N == 0) return dz.narrow(-1, 0, s.V);
  LpGradArgs a{};
  a.z = z.data_ptr(); a.ld = s.ld; a.ldo = ldo; a.dz = dz.data_ptr(); a.tok = tok.data_ptr(); a.tok64 = tok.scalar_type() == at::kLong;
  a.V = (int)s.V;
  const int64_t per = 256 * 4 * (s.vec ? pad : 1);
  a.chunks = (int)((s.V + per - 1) / per);
  TORCH_CHECK(s.N * a.chunks < (1LL << 31), "too many logits");
  a.g = g.has_value() ? g->data_ptr<float>() : nullptr;
  a.h = h.has_value() ? h->data_ptr<float>() : nullptr;
  a.stat = stat.data_ptr<float>();
  auto* kern = s.bf ? (s.vec ? token_logprobs_grad_kernel<true, true> : token_logprobs_grad_kernel<true, false>)
                    : (s.vec ? token_logprobs_grad_kernel<false, true> : token_logprobs_grad_kernel<false, false>);
  kern<<<(unsigned)(s.N * a.chunks), 256, 0, at::cuda::getCurrentCUDAStream()>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return dz.narrow(-1, 0, s.V);
}

}  // namespace tfb
