// Drafted tokens verified against the target's probabilities (speculative sampling over a tree).
//
// Node 0 is the tree's root (a token that is already part of the text); node n > 0 is a drafted
// token, child of parents[n] < n.  Row n of p (q) holds the target's (the draft's) distribution
// of the token after node n, and the children of a node were drawn from its row of q, each by
// itself (q absent: a rule proposed them).  From the root on, the children of the last accepted
// node cur are tried in order with the remainder r (at first p[cur], Z = 1):
//     accept n      iff  u[n] q[cur][t] Z < r[t],  t = tokens[n]     (q absent: q[cur][t] = 1)
//     reject n:     r <- max(r - Z q[cur], 0),  Z <- sum r           (q absent: r[t] <- 0)
//                   (r / Z is the remainder's distribution; an empty one becomes p[cur], Z = 1)
// When no child is left, the next token is the least j with r[0] + .. + r[j] > u[0] sum r.
// The accepted tokens and that one are together distributed as if drawn from p one by one.
//
// Answers are whole numbers that a last bit can turn, so r, Z and every sum are in 64 bits
// (fp32 products are then exact, and a sum's order moves it by 1e-16 only).
//
// What a sequence has to read whole is one row of p, and of q after a rejection: the tests
// themselves read single entries, gathered for all nodes at once by one thread a node.  r is
// not stored: each pass recomputes it from p and q as max(p - S q, 0), S the sum of the Z's of the
// rejections so far, which is all of them in one step, since q and Z are not negative.  Its error is
// 2^-53 of p, the same as a single step's, but the steps one by one keep a remainder that has become
// small exact to 2^-53 of itself: below Z = 2^-20 they are taken one by one.  A
// cluster of CTAs shares a row, every warp a contiguous range of it, and all CTAs take the same
// decisions from the same sums, read from each other's shared memory.  The last pass leaves the
// warps' sums behind, so the draw re-reads only the range in which its token lies.
//
// Measured on a B200 (calls replayed from a graph).  8 chains of 6 nodes, vocabulary 8192: 7.5 us with q, 6.2
// without.  64 x 24 nodes, 131072: 39 us with q (47 with one subtraction a rejection and eight CTAs a row), where
// the last rows alone are 10 us at the memory's rate, and 50 without, of 5: every rejection is a pass over the
// row, though without q it changes one entry.  The bound is the slowest sequence's chain of passes, with q up to
// four there, each of which waits for the one before and takes 8 to 10 us.
// The reference has no decode path.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>

#include "sm100_common.cuh"

namespace tfb {

int num_sms(int dev);

constexpr int kVerThreads = 512;
constexpr int kVerWarps = kVerThreads / 32;
constexpr int kVerNodes = 64;
constexpr int kVerCluster = 8;   // CTAs of a cluster at most

struct VerArgs {
  const int* tokens;
  const int* parents;
  const float* p;
  const float* q;                // null: deterministic drafts
  const float* u;
  long long pb, pn, qb, qn;      // strides in elements
  int* path;
  int* count;
  int* out;
  int N, V, range;               // range: row entries a warp owns (a multiple of 128)
};

__device__ __forceinline__ double ld_dsmem_f64(uint32_t addr) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
  return v;
}

template <bool VEC>
__device__ __forceinline__ void load4(const float* row, int j, int end, float (&f)[4]) {
  if constexpr (VEC) {
    if (j + 4 <= end) {
      const float4 v = *reinterpret_cast<const float4*>(row + j);
      f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = j + i < end ? row[j + i] : 0.f;
}

// max(r, 0) without the 64-bit compare: the sign bit clears both words.
__device__ __forceinline__ double clear_negative(double r) {
  const int keep = ~(__double2hiint(r) >> 31);
  return __hiloint2double(__double2hiint(r) & keep, __double2loint(r) & keep);
}

// VEC: rows start on 16-byte boundaries.
template <bool VEC, bool HASQ>
__global__ void __launch_bounds__(kVerThreads, 2) verify_tree_kernel(const VerArgs a) {
  __shared__ int s_tok[kVerNodes], s_par[kVerNodes], s_path[kVerNodes];
  __shared__ float s_u[kVerNodes], s_p[kVerNodes], s_q[kVerNodes];
  __shared__ double s_z[kVerNodes];          // Z before each rejection at the current node
  __shared__ int s_rej[kVerNodes];           // the rejected tokens (q absent)
  __shared__ double s_sum[kVerWarps];        // the warps' sums of the last pass
  __shared__ double s_tot[2];                // this CTA's sum, two passes in turn
  __shared__ double s_scan[kVerWarps];
  __shared__ int s_pick, s_lastpos;

  const int C = (int)(gridDim.x / nclusters_x());
  const int rank = (int)cluster_ctarank();
  const int b = (int)(blockIdx.x / C);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int N = a.N, V = a.V;
  const float* P = a.p + b * a.pb;
  const float* Q = HASQ ? a.q + b * a.qb : nullptr;

  if (tid < N) {
    const int tok = a.tokens[(long long)b * N + tid], par = a.parents[(long long)b * N + tid];
    const bool real = tid > 0 && tok >= 0 && tok < V && par >= 0 && par < tid;   // else no node's child
    s_tok[tid] = tok;
    s_par[tid] = real ? par : -1;
    s_u[tid] = a.u[(long long)b * N + tid];
    s_p[tid] = real ? P[par * a.pn + tok] : 0.f;
    s_q[tid] = real && HASQ ? Q[par * a.qn + tok] : 1.f;
  }
  __syncthreads();

  int cur = 0, cnt = 1, rej = 0, turn = 0;
  double Z = 1.0, S = 0.0, share = 0.0;      // S: sum of Z over the rejections; share: lane i has CTA i's part of the last pass's total
  bool deep = false;                         // Z is small: rejections one by one (q given)
  bool summed = false;                       // s_sum and share belong to the present r
  const long long w0 = (long long)(rank * kVerWarps + warp) * a.range;   // this warp's range
  const int lo = (int)min((long long)V, w0), hi = (int)min((long long)V, w0 + a.range);

  // r at M neighbouring entries from j on, after the rejections so far; f: p there, g: q there
  auto rest = [&](auto& r, const auto& f, const auto& g, int j, int M) {
#pragma unroll
    for (int i = 0; i < M; ++i) r[i] = (double)f[i];
    if constexpr (HASQ) {
      if (deep) {
#pragma unroll 1
        for (int k = 0; k < rej; ++k) {
          const double z = s_z[k];
#pragma unroll
          for (int i = 0; i < M; ++i) r[i] = clear_negative(__dsub_rn(r[i], __dmul_rn(z, (double)g[i])));
        }
      } else if (rej > 0) {
#pragma unroll
        for (int i = 0; i < M; ++i) r[i] = clear_negative(__fma_rn(-S, (double)g[i], r[i]));
      }
    } else {
#pragma unroll 1
      for (int k = 0; k < rej; ++k) {
        const int t = s_rej[k] - j;
#pragma unroll
        for (int i = 0; i < M; ++i)
          if (t == i) r[i] = 0.0;
      }
    }
  };
  // the sum of r, and with it s_sum and share
  auto pass = [&]() -> double {
    const float* pr = P + cur * a.pn;
    const float* qr = HASQ ? Q + cur * a.qn : nullptr;
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    if (HASQ && deep) {                      // in a loop of its own: 38 against 42 us
#pragma unroll 1
      for (int j = lo + lane; j < hi; j += 32) {
        const float f[1] = {pr[j]}, g[1] = {qr[j]};
        double r[1];
        rest(r, f, g, j, 1);
        acc[0] += r[0];
      }
    } else {
      for (int j = lo + lane * 4; j < hi; j += 512) {
        float f[4][4], g[4][4] = {};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          load4<VEC>(pr, j + 128 * k, hi, f[k]);
          if constexpr (HASQ) {
            if (rej > 0) load4<VEC>(qr, j + 128 * k, hi, g[k]);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          double r[4];
          if constexpr (HASQ) {
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = clear_negative(__fma_rn(-S, (double)g[k][i], (double)f[k][i]));   // S = 0: r = p
          } else {
            rest(r, f[k], g[k], j + 128 * k, 4);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i] += r[i];
        }
      }
    }
    double s = (acc[0] + acc[1]) + (acc[2] + acc[3]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    __syncthreads();                         // s_sum of the pass before is no longer read
    if (lane == 0) s_sum[warp] = s;
    __syncthreads();
    double t = lane < kVerWarps ? s_sum[lane] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    share = lane == 0 ? t : 0.0;
    if (C > 1) {
      if (tid == 0) s_tot[turn] = t;
      cluster_sync();
      share = lane < C ? ld_dsmem_f64(mapa_shared(smem_u32(&s_tot[turn]), (uint32_t)lane)) : 0.0;
      t = share;
#pragma unroll
      for (int o = kVerCluster / 2; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
      t = __shfl_sync(0xffffffffu, t, 0);
      turn ^= 1;
    }
    summed = true;
    return t;
  };

  if (tid == 0) s_path[0] = 0;
  for (int n = 1; n < N; ++n) {
    if (s_par[n] != cur) continue;
    const float f[1] = {s_p[n]}, g[1] = {s_q[n]};
    double r[1];
    rest(r, f, g, s_tok[n], 1);
    if (__dmul_rn(__dmul_rn((double)s_u[n], (double)g[0]), Z) < r[0]) {
      __syncthreads();                       // s_path, and s_z / s_rej of the node left behind
      cur = n;
      if (tid == 0) s_path[cnt] = n;
      ++cnt;
      rej = 0;
      Z = 1.0;
      S = 0.0;
      deep = false;
      summed = false;
    } else {
      __syncthreads();
      if (tid == 0) {
        s_z[rej] = Z;
        s_rej[rej] = s_tok[n];
      }
      ++rej;
      S += Z;
      __syncthreads();
      Z = pass();
      if (HASQ && !deep && Z < 0x1p-20) {
        deep = true;
        if (rej > 1) Z = pass();             // the first rejection is one step in any case
      }
      if (!(Z > 0.0)) {                      // nothing is left (p = q up to rounding): p itself
        rej = 0;
        Z = 1.0;
        S = 0.0;
        deep = false;
        summed = false;
      }
    }
  }
  if (!summed) Z = pass();

  // the draw: the CTA and the warp's range in which the running sum passes the target, then the
  // entry.  By rounding none may pass it: then the last one that holds anything.
  const double target = __dmul_rn((double)s_u[0], Z);
  double before = 0.0;
  int at = 0;
  auto find = [&](int n, auto part) {
    double run = before;
    bool found = false;
    at = 0;
    for (int i = 0; i < n; ++i) {
      const double s = part(i);
      if (s > 0.0 && !found) {
        at = i;
        before = run;
        found = run + s > target;
      }
      run += s;
    }
  };
  find(C, [&](int i) { return __shfl_sync(0xffffffffu, share, i); });
  if (rank == at) {
    find(kVerWarps, [&](int i) { return s_sum[i]; });
    const long long first = (long long)(rank * kVerWarps + at) * a.range;
    const int r0 = (int)min((long long)V, first), r1 = (int)min((long long)V, first + a.range);
    const float* pr = P + cur * a.pn;
    const float* qr = HASQ ? Q + cur * a.qn : nullptr;
    if (tid == 0) { s_pick = V; s_lastpos = -1; }
    __syncthreads();
    for (int j0 = r0; j0 < r1; j0 += kVerThreads * 4) {
      const int j = j0 + tid * 4;
      float f[4], g[4] = {0.f, 0.f, 0.f, 0.f};
      load4<VEC>(pr, j, r1, f);
      if constexpr (HASQ) {
        if (rej > 0) load4<VEC>(qr, j, r1, g);
      }
      double r[4];
      rest(r, f, g, j, 4);
      int lastj = -1;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r[i] > 0.0 && j + i < r1) lastj = j + i;
      const double own = (r[0] + r[1]) + (r[2] + r[3]);
      double inc = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (lane == 31) s_scan[warp] = inc;
      if (lastj >= 0) atomicMax(&s_lastpos, lastj);
      __syncthreads();
      double base = before, all = before;
      for (int w = 0; w < kVerWarps; ++w) {
        if (w < warp) base += s_scan[w];
        all += s_scan[w];
      }
      double c = base + (inc - own);
      int pick = V;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c += r[i];
        if (pick == V && r[i] > 0.0 && c > target) pick = j + i;
      }
      if (pick < V) atomicMin(&s_pick, pick);
      before = all;
      __syncthreads();
      if (s_pick < V) break;
    }
    const int tok = s_pick < V ? s_pick : s_lastpos >= 0 ? s_lastpos : V - 1;
    if (tid < N) {
      const long long o = (long long)b * N + tid;
      a.path[o] = tid < cnt ? s_path[tid] : -1;
      a.out[o] = tid + 1 < cnt ? s_tok[s_path[tid + 1]] : tid + 1 == cnt ? tok : -1;
      if (tid == 0) a.count[b] = cnt;
    }
  }
  if (C > 1) cluster_sync();                 // no CTA leaves while another may read its sums
}

std::vector<at::Tensor> verify_tree(at::Tensor tokens, at::Tensor parents, at::Tensor p, c10::optional<at::Tensor> q,
                                       at::Tensor u) {
  TORCH_CHECK(p.is_cuda() && p.dim() == 3 && p.scalar_type() == at::kFloat, "p: float32 [B, N, V]");
  const int64_t B = p.size(0), N = p.size(1), V = p.size(2);
  TORCH_CHECK(N >= 1 && N <= kVerNodes, "1 to 64 nodes");
  TORCH_CHECK(V >= 1 && V <= (1 << 30), "vocabulary of 1 .. 2^30 tokens");
  auto ints = [&](const at::Tensor& t, const char* name) {
    TORCH_CHECK(t.scalar_type() == at::kInt && t.device() == p.device() && t.dim() == 2 && t.size(0) == B && t.size(1) == N &&
                    t.is_contiguous(), name, ": contiguous int32 [B, N] on p's device");
    return t.data_ptr<int>();
  };
  VerArgs a{};
  a.tokens = ints(tokens, "tokens");
  a.parents = ints(parents, "parents");
  TORCH_CHECK(u.scalar_type() == at::kFloat && u.device() == p.device() && u.dim() == 2 && u.size(0) == B && u.size(1) == N &&
                  u.is_contiguous(), "u: contiguous float32 [B, N] on p's device");
  auto rows = [&](const at::Tensor& t, const char* name, long long& sb, long long& sn) {
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.device() == p.device() && t.sizes() == p.sizes() && (t.size(2) == 1 || t.stride(2) == 1),
                name, ": float32 [B, N, V] with unit inner stride on p's device");
    sb = t.stride(0); sn = t.stride(1);
    return (B <= 1 || sb % 4 == 0) && (N <= 1 || sn % 4 == 0) && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
  };
  bool vec = rows(p, "p", a.pb, a.pn);
  if (q.has_value()) vec = rows(*q, "q", a.qb, a.qn) && vec;
  a.p = p.data_ptr<float>();
  a.q = q.has_value() ? q->data_ptr<float>() : nullptr;
  a.u = u.data_ptr<float>();
  c10::cuda::CUDAGuard guard(p.device());
  auto opt = p.options().dtype(at::kInt);
  auto path = at::empty({B, N}, opt), count = at::empty({B}, opt), out = at::empty({B, N}, opt);
  if (B == 0) return {path, count, out};
  a.path = path.data_ptr<int>(); a.count = count.data_ptr<int>(); a.out = out.data_ptr<int>();
  a.N = (int)N; a.V = (int)V;
  TORCH_CHECK(B <= (1LL << 31) / kVerCluster - 1, "too many sequences");
  // CTAs of a cluster: at most one for each 16384 entries, since exchanging sums costs every pass about 1 us.
  // Two CTAs fit on a SM; more than that wait their turn, which pays only while a CTA's range is long: turns
  // at most as many as times 16384 entries a CTA.  Trees with q, us with 1 / 2 / 4 / 8 CTAs (the rule's choice):
  //   131072 entries, 24 nodes: 8 sequences 56 / 35 / 25 / 19 (8), 32: 65 / 41 / 28 / 26 (8), 64: 72 / 46 / 37 / 41 (4),
  //                             128: 88 / 64 / 58 / 76 (4), 256: 115 / 94 / 99 / 141 (2)
  //   32768, 24:                32: 24 / 21 / 18 / 22 (2), 128: 30 / 29 / 37 / 64 (2), 512: 58 / 74 / 111 / 222 (1)
  //   8192, 6:                  8: 11 / 14 / 15 / 15 (1), 64: 12 / 17 / 21 / 29 (1), 512: 24 / 44 / 81 / 162 (1)
  const int64_t slots = 2 * num_sms(p.device().index());
  int C = 1;
  while (C < kVerCluster && (int64_t)C * 16384 < V && B * (2 * C) * (2 * C) * 16384 <= slots * V) C *= 2;
  a.range = (int)(((V + C * kVerWarps - 1) / (C * kVerWarps) + 127) / 128 * 128);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(B * C), 1, 1);
  cfg.blockDim = dim3(kVerThreads, 1, 1);
  cfg.stream = at::cuda::getCurrentCUDAStream();
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (vec) {
    if (a.q) C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, verify_tree_kernel<true, true>, a));
    else C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, verify_tree_kernel<true, false>, a));
  } else {
    if (a.q) C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, verify_tree_kernel<false, true>, a));
    else C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, verify_tree_kernel<false, false>, a));
  }
  return {path, count, out};
}

}  // namespace tfb
