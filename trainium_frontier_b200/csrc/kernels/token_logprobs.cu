// Log probabilities of given tokens, entropies and the likeliest alternatives of rows of logits,
// and the gradient of the first two.
//
// With m the row's maximum, S = sum e^(z - m) and T = sum e^(z - m) (z - m):
//   log p_v = (z_v - m) - log S,   H = log S - T / S,
//   dz_v = g ([v = token] - p_v) - h p_v (log p_v + H)     (g, h: gradients of log p_token and H).
// All of it is held in 32 bits; m and log S are kept apart for the gradient, since their sum would
// round away what a small log p is made of.
//
// The bytes bound both directions, so a row is read once: a thread keeps up to 128 bytes of it in
// registers, a CTA up to 64 KB, a cluster of up to 8 CTAs a longer row (or, with few rows, a shorter
// share of it each), and sums and alternatives of the CTAs are joined through distributed shared
// memory.  Only alternatives of rows beyond that are looked for in a second read.
//
// Alternatives: the k-th largest of 32 groups' maxima is at most the k-th largest logit, so the few
// logits that are not below it (6 on average for k = 5) are collected and ranked by (logit, lowest
// token first).  Where more than 1024 are collected (equal logits everywhere), k passes over the
// registers take the next one each.
// The reference has no counterpart; its losses are those of fused_ops.cu.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>

#include "sm100_common.cuh"

namespace tfb {

int num_sms(int dev);

constexpr int kLpRegs = 32;      // 32-bit words of a row a thread
constexpr int kLpMaxTop = 32;
constexpr int kLpCap = 1024;     // collected logits
typedef unsigned long long u64;

struct LpArgs {
  const void* z;
  long long ld;                  // elements between rows
  const void* tok;
  int tok64;
  int V, top;
  int items, per, nch;           // loads of a row, of a CTA, and rounds of them
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

// BF: bf16 logits, else fp32.  VEC: 16-byte loads (rows 16-byte aligned), else one element each.
template <bool BF, bool VEC>
struct LpRow {
  static constexpr int EPR = BF && VEC ? 2 : 1;                // elements of a word
  static constexpr int EPL = VEC ? (BF ? 8 : 4) : 1;           // of a load
  static constexpr int LOADS = VEC ? kLpRegs / 4 : kLpRegs;    // of a thread
  uint32_t r[kLpRegs];
  int i0, end, V;                // first load, end of the CTA's loads

  __device__ __forceinline__ void load(const void* row, int first) {
    i0 = first + threadIdx.x;
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int i = i0 + j * blockDim.x;
        uint4 u = make_uint4(0, 0, 0, 0);
        if (i < end) {
          const int e = i * EPL;
          if (e + EPL <= V) {
            u = __ldg(static_cast<const uint4*>(row) + i);
          } else {               // the row's last elements
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < EPL; ++x)
              if (e + x < V) {
                if constexpr (BF) w[x >> 1] |= (uint32_t)static_cast<const uint16_t*>(row)[e + x] << (16 * (x & 1));
                else w[x] = static_cast<const uint32_t*>(row)[e + x];
              }
            u = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        r[4 * j] = u.x; r[4 * j + 1] = u.y; r[4 * j + 2] = u.z; r[4 * j + 3] = u.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int i = i0 + j * blockDim.x;
        r[j] = 0;
        if (i < end) r[j] = BF ? (uint32_t)static_cast<const uint16_t*>(row)[i] << 16 : static_cast<const uint32_t*>(row)[i];
      }
    }
  }
  // f(element's index in the row, its value) of every element that is there
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int j = 0; j < kLpRegs; ++j) {
      const int i = i0 + (VEC ? j >> 2 : j) * blockDim.x;
      if (i >= end) continue;
#pragma unroll
      for (int h = 0; h < EPR; ++h) {
        const int e = VEC ? i * EPL + (j & 3) * EPR + h : i;
        if (VEC && e >= V) continue;
        f(e, __uint_as_float(EPR == 2 ? (h ? r[j] & 0xffff0000u : r[j] << 16) : r[j]));
      }
    }
  }
};

// Sums S and T against the maximum m as sums against M >= m.  An m of -inf comes with sums of 0 (or of NaN, which
// stay); e^-1e4 is 0, and 0 * inf never comes up.
__device__ __forceinline__ void lp_rebase(float m, float M, float& S, float& T) {
  const float d = m - M;
  const float e = m == -INFINITY ? 1.f : __expf(d);
  if (m != -INFINITY) T += fmaxf(d, -1e4f) * S;
  T *= e;
  S *= e;
}

template <bool BF, bool VEC>
__global__ void __launch_bounds__(512) token_logprobs_kernel(const LpArgs a, int C) {
  __shared__ float sM[16], sS[16], sT[16];
  __shared__ uint32_t sG[32];
  __shared__ u64 sTop[kLpMaxTop];          // the CTA's alternatives, best first (0: none)
  __shared__ float sStat[4];
  __shared__ u64 sCand[kLpCap];
  __shared__ int sCount;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const long long row = blockIdx.x / C;
  const int rank = (int)(blockIdx.x % C);
  const void* z = static_cast<const char*>(a.z) + row * a.ld * (BF ? 2 : 4);
  if (threadIdx.x == 0) sCount = 0;

  // ------------------------------------------------------------------ one read: maximum and sums
  LpRow<BF, VEC> x;
  x.V = a.V;
  const int first = rank * a.per;
  x.end = min(first + a.per, a.items);
  float m = -INFINITY, S = 0.f, T = 0.f;
  uint32_t key = 0;                        // the largest logit's, 0: none
  for (int c = 0; c < a.nch; ++c) {
    x.load(z, first + c * LpRow<BF, VEC>::LOADS * blockDim.x);
    float mc = m;
    bool some = false;
    x.each([&](int, float v) { mc = fmaxf(mc, v); some = true; });
    if (mc > m) {
      lp_rebase(m, mc, S, T);
      m = mc;
    }
    const float ref = lp_ref(m);
    float s4[4] = {0.f, 0.f, 0.f, 0.f}, t4[4] = {0.f, 0.f, 0.f, 0.f};
    int k = 0;
    bool nan = false;
    x.each([&](int, float v) {
      const float d = v - ref, e = __expf(d);
      s4[k & 3] += e;
      t4[k & 3] += e * fmaxf(d, -1e4f);    // e^-1e4 is 0: 0 * inf never comes up
      nan |= v != v;
      ++k;
    });
    S += (s4[0] + s4[1]) + (s4[2] + s4[3]);
    T += (t4[0] + t4[1]) + (t4[2] + t4[3]);
    if (some) key = nan ? 0xffffffffu : max(key, lp_key(m));
  }
  // the warp's, then the CTA's
  const float mw = warp_max(m);
  lp_rebase(m, mw, S, T);
  S = warp_sum(S);
  T = warp_sum(T);
  if (lane == 0) { sM[warp] = mw; sS[warp] = S; sT[warp] = T; }
  if (a.top) {
    uint32_t g = key;
    for (int o = (blockDim.x >> 5) >> 1; o > 0; o >>= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (threadIdx.x % (blockDim.x >> 5) == 0) sG[threadIdx.x / (blockDim.x >> 5)] = g;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float M = sM[0];
    for (int w = 1; w < warps; ++w) M = fmaxf(M, sM[w]);
    float s = 0.f, t = 0.f;
    for (int w = 0; w < warps; ++w) {
      float sw = sS[w], tw = sT[w];
      lp_rebase(sM[w], M, sw, tw);
      s += sw;
      t += tw;
    }
    sStat[0] = M; sStat[1] = s; sStat[2] = t;
  }

  // ------------------------------------------------------------------ the CTA's alternatives
  if (a.top) {
    uint32_t g = sG[lane], thr = 0;
    for (int i = 0; i < a.top; ++i) {      // the top-th largest of the groups' maxima
      thr = __reduce_max_sync(0xffffffffu, g);
      const unsigned who = __ballot_sync(0xffffffffu, g == thr);
      if (lane == __ffs(who) - 1) g = 0;
    }
    for (int c = 0; c < a.nch; ++c) {
      if (a.nch > 1) x.load(z, first + c * LpRow<BF, VEC>::LOADS * blockDim.x);
      if (key >= thr)
        x.each([&](int e, float v) {
          const uint32_t q = lp_key(v);
          if (q >= thr) {
            const int at = atomicAdd(&sCount, 1);
            if (at < kLpCap) sCand[at] = ((u64)q << 32) | (uint32_t)~e;
          }
        });
    }
    if (threadIdx.x < a.top) sTop[threadIdx.x] = 0;
    __syncthreads();
    const int n = sCount;
    if (n <= kLpCap) {
      for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const u64 me = sCand[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += sCand[j] > me;
        if (r < a.top) sTop[r] = me;
      }
    } else {
      u64 last = ~0ull;
      for (int i = 0; i < a.top; ++i) {
        u64 best = 0;
        for (int c = 0; c < a.nch; ++c) {
          if (a.nch > 1) x.load(z, first + c * LpRow<BF, VEC>::LOADS * blockDim.x);
          x.each([&](int e, float v) {
            const u64 q = ((u64)lp_key(v) << 32) | (uint32_t)~e;
            if (q < last && q > best) best = q;
          });
        }
        for (int o = 16; o > 0; o >>= 1) {
          const u64 other = __shfl_xor_sync(0xffffffffu, best, o);
          if (other > best) best = other;
        }
        __syncthreads();
        if (lane == 0) sCand[warp] = best;
        __syncthreads();
        for (int w = 0; w < warps; ++w) best = sCand[w] > best ? sCand[w] : best;
        if (threadIdx.x == 0) sTop[i] = best;
        last = best;
      }
    }
  }

  // ------------------------------------------------------------------ the row's
  if (C > 1) cluster_sync(); else __syncthreads();
  if (rank == 0) {
    float M = -INFINITY;
    float ms[8], ss[8], ts[8];
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < C) {
        const uint32_t at = C > 1 ? mapa_shared(smem_u32(sStat), c) : 0;
        ms[c] = C > 1 ? ld_dsmem_f32(at) : sStat[0];
        ss[c] = C > 1 ? ld_dsmem_f32(at + 4) : sStat[1];
        ts[c] = C > 1 ? ld_dsmem_f32(at + 8) : sStat[2];
        M = fmaxf(M, ms[c]);
      }
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < C) {
        lp_rebase(ms[c], M, ss[c], ts[c]);
        s += ss[c];
        t += ts[c];
      }
    const float logs = M == -INFINITY ? __int_as_float(0x7fffffff) : logf(s);   // nothing but -inf: NaN
    if (threadIdx.x == 0) {
      const long long v = lp_token(a.tok, a.tok64, row);
      float lp = 0.f;
      if (v >= 0 && v < a.V)
        lp = (BF ? __uint_as_float((uint32_t)static_cast<const uint16_t*>(z)[v] << 16) : static_cast<const float*>(z)[v]) - M - logs;
      const float H = logs - t / s;
      a.lp[row] = lp;
      a.ent[row] = H;
      if (a.stat) {
        a.stat[3 * row] = M;
        a.stat[3 * row + 1] = logs;
        a.stat[3 * row + 2] = H;
      }
    }
    if (a.top && C == 1) {
      if (threadIdx.x < a.top) {
        const u64 k = sTop[threadIdx.x];
        a.top_tok[row * a.top + threadIdx.x] = (int)~(uint32_t)k;
        a.top_lp[row * a.top + threadIdx.x] = lp_unkey((uint32_t)(k >> 32)) - M - logs;
      }
    } else if (a.top) {
      for (int i = threadIdx.x; i < C * a.top; i += blockDim.x)
        sCand[i] = ld_dsmem_u64(mapa_shared(smem_u32(sTop), i / a.top) + 8 * (i % a.top));
      __syncthreads();
      for (int i = threadIdx.x; i < C * a.top; i += blockDim.x) {
        const u64 k = sCand[i];
        int r = 0;
        for (int j = 0; j < C * a.top; ++j) r += sCand[j] > k;
        if (k != 0 && r < a.top) {
          a.top_tok[row * a.top + r] = (int)~(uint32_t)k;
          a.top_lp[row * a.top + r] = lp_unkey((uint32_t)(k >> 32)) - M - logs;
        }
      }
    }
  }
  if (C > 1) cluster_sync();               // shared memory lives until rank 0 has read it
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
  bool bf, vec;
  int64_t N, V, ld;
};

static LpShape lp_check(const at::Tensor& z, const at::Tensor& tok) {
  TORCH_CHECK(z.is_cuda() && z.dim() == 2 && (z.scalar_type() == at::kFloat || z.scalar_type() == at::kBFloat16),
              "logits: float32 or bfloat16 [..., V]");
  LpShape s{};
  s.bf = z.scalar_type() == at::kBFloat16;
  s.N = z.size(0); s.V = z.size(1);
  TORCH_CHECK(s.V >= 1 && s.V <= (1 << 30), "vocabulary of 1 .. 2^30 tokens");
  TORCH_CHECK(s.V == 1 || z.stride(1) == 1, "logits: unit inner stride");
  s.ld = z.stride(0);
  TORCH_CHECK(s.N <= (1 << 27), "at most 2^27 rows");
  TORCH_CHECK((tok.scalar_type() == at::kLong || tok.scalar_type() == at::kInt) && tok.device() == z.device() && tok.dim() == 1 &&
                  tok.size(0) == s.N && tok.is_contiguous(), "tokens: int64 or int32, one for each row of the logits, on their device");
  s.vec = (reinterpret_cast<uintptr_t>(z.data_ptr()) & 15) == 0 && (s.N == 1 || s.ld * z.element_size() % 16 == 0);
  return s;
}

std::vector<at::Tensor> token_logprobs(at::Tensor z, at::Tensor tok, int64_t top, bool stats) {
  const LpShape s = lp_check(z, tok);
  TORCH_CHECK(top >= 0 && top <= kLpMaxTop && top <= s.V, "top: 0 .. 32 alternatives, at most the vocabulary");
  c10::cuda::CUDAGuard guard(z.device());
  const auto f32 = z.options().dtype(at::kFloat);
  auto lp = at::empty({s.N}, f32), ent = at::empty({s.N}, f32), top_lp = at::empty({s.N, top}, f32);
  auto top_tok = at::empty({s.N, top}, z.options().dtype(at::kInt));
  auto stat = at::empty({stats ? s.N : 0, 3}, f32);
  if (s.N == 0) return {lp, ent, top_tok, top_lp, stat};
  const int epl = s.vec ? (s.bf ? 8 : 4) : 1, loads = s.vec ? kLpRegs / 4 : kLpRegs;
  LpArgs a{};
  a.z = z.data_ptr(); a.ld = s.ld; a.tok = tok.data_ptr(); a.tok64 = tok.scalar_type() == at::kLong;
  a.V = (int)s.V; a.top = (int)top;
  a.items = (int)((s.V + epl - 1) / epl);
  // threads: as few as hold the row, then more (down to one load each) while the rows alone do not fill
  // the GPU; CTAs of a cluster likewise
  const int64_t fill = (int64_t)num_sms(z.get_device()) * 1024;
  int T = 32, C = 1;
  while (T < 512 && ((int64_t)T * loads < a.items || (s.N * T < fill && T < a.items))) T *= 2;
  while (C < 8 && ((top > 0 && (int64_t)T * C * loads < a.items) || (s.N * T * C < fill && (int64_t)T * C < a.items))) C *= 2;
  a.per = (a.items + C - 1) / C;
  a.nch = (a.per + T * loads - 1) / (T * loads);
  a.lp = lp.data_ptr<float>(); a.ent = ent.data_ptr<float>(); a.stat = stats ? stat.data_ptr<float>() : nullptr;
  a.top_tok = top_tok.data_ptr<int>(); a.top_lp = top_lp.data_ptr<float>();
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((unsigned)(s.N * C));
  cfg.blockDim = dim3(T);
  cfg.stream = at::cuda::getCurrentCUDAStream();
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 1 : 0;
  auto* kern = s.bf ? (s.vec ? token_logprobs_kernel<true, true> : token_logprobs_kernel<true, false>)
                    : (s.vec ? token_logprobs_kernel<false, true> : token_logprobs_kernel<false, false>);
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, a, C));
  return {lp, ent, top_tok, top_lp, stat};
}

// dz [N, V], a view of rows padded to 16 bytes.
at::Tensor token_logprobs_grad(at::Tensor z, at::Tensor tok, at::Tensor stat, c10::optional<at::Tensor> g, c10::optional<at::Tensor> h) {
  const LpShape s = lp_check(z, tok);
  TORCH_CHECK(stat.scalar_type() == at::kFloat && stat.device() == z.device() && stat.is_contiguous() && stat.numel() == 3 * s.N, "stat: float32 [N, 3]");
  for (const auto* t : {&g, &h})
    TORCH_CHECK(!t->has_value() || ((*t)->scalar_type() == at::kFloat && (*t)->device() == z.device() && (*t)->is_contiguous() &&
                                    (*t)->numel() == s.N), "gradients: contiguous float32 [N]");
  c10::cuda::CUDAGuard guard(z.device());
  const int64_t pad = s.bf ? 8 : 4, ldo = (s.V + pad - 1) / pad * pad;
  auto dz = at::empty({s.N, ldo}, z.options());
  if (s.N == 0) return dz.narrow(1, 0, s.V);
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
  return dz.narrow(1, 0, s.V);
}

}  // namespace tfb
