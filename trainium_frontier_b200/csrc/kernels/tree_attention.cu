// Attention of a tree of drafted tokens over a key/value cache.
//
// The cache holds lens[b] rows of context and, behind them, one row for each of the N nodes of
// the drafted tree.  Node n's query sees the context, its ancestors and itself:
//     o[b, n, h] = sum_t softmax_t(scale q[b, n, h] . k[b, h / G, t]) v[b, h / G, t]
//     over t < lens[b] and t = lens[b] + j, j an ancestor of n or n itself.
// N = 1 is a decode step of a single token; parents absent: node n - 1 is node n's parent.
// The reference has no decode path; the attention is the math of train.py:2564-2567.
#include <cuda_fp8.h>

#include "kv_cache.cuh"

namespace tfb {

constexpr int kTreeNodes = 64;

struct TreeArgs {
  const __nv_bfloat16* q;
  long long qb, qn, qh;      // strides in elements
  __nv_bfloat16* o;          // [B, N, Hq, D]
  const int* lens;
  const int* parents;        // null: a chain
  int B, N, Hq, Hkv, G;
  float scale_log2;
};

// Ancestors of node n and n itself as a bit mask; 0 for an unused node: one whose line of
// parents meets an entry that is not -1 or an earlier node, or whose own row is not in the cache.
__device__ __forceinline__ unsigned long long tree_line(const int* par, int n, int fit) {
  if (n >= fit) return 0;
  if (par == nullptr) return n == 63 ? ~0ull : (2ull << n) - 1;
  unsigned long long m = 0;
  int i = n;
  while (true) {
    m |= 1ull << i;
    const int p = par[i];
    if (p == -1) return m;
    if (p < 0 || p >= i) return 0;
    i = p;
  }
}

template <int D, bool QUANT>
__global__ void __launch_bounds__(128) tree_attention_simple_kernel(const TreeArgs a, const KvView c) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (w >= (long long)a.B * a.N * a.Hq) return;
  const int hq = (int)(w % a.Hq), n = (int)(w / a.Hq % a.N), b = (int)(w / a.Hq / a.N), h = hq / a.G;
  const int len = max(0, min(a.lens[b], c.tmax));
  const int fit = min(a.N, c.tmax - len);
  const unsigned long long line = tree_line(a.parents ? a.parents + (long long)b * a.N : nullptr, n, fit);
  float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    q[i] = __bfloat162float(a.q[b * a.qb + n * a.qn + hq * a.qh + lane * E + i]) * a.scale_log2;
    o[i] = 0.f;
  }
  const int end = line ? len + n + 1 : 0;
  for (int t = 0; t < end; ++t) {
    if (t >= len && !((line >> (t - len)) & 1)) continue;
    float kv[2][E];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint8_t* row = c.p[s] + b * c.b + h * c.h + (long long)t * c.t;
      float sc = 1.f;
      if constexpr (QUANT) {
        const int e = c.s[s][b * c.sb + h * c.sh + (long long)t * c.st];
        sc = e == kScaleNan ? __int_as_float(0x7fffffff) : e == 0 ? 0x1p-127f : __uint_as_float((uint32_t)e << 23);
      }
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if constexpr (QUANT) {
          const __half_raw hr = __nv_cvt_fp8_to_halfraw(row[lane * E + i], __NV_E4M3);
          kv[s][i] = __half2float(__half(hr)) * sc;
        } else {
          kv[s][i] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[lane * E + i]);
        }
      }
    }
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) x += q[i] * kv[0][i];
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
    const float mn = fmaxf(m, x);
    const float f = mn == -INFINITY ? 1.f : exp2f(m - mn), p = exp2f(x - mn);
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = o[i] * f + p * kv[1][i];
    m = mn;
  }
  __nv_bfloat16* dst = a.o + w * D + lane * E;
#pragma unroll
  for (int i = 0; i < E; ++i) dst[i] = __float2bfloat16_rn(line ? o[i] / l : 0.f);
}

at::Tensor tree_attention(at::Tensor q, at::Tensor kc, at::Tensor vc, at::Tensor lens,
                             c10::optional<at::Tensor> parents, double scale, c10::optional<at::Tensor> ks,
                             c10::optional<at::Tensor> vs, at::Tensor err) {
  bool quant;
  const KvView c = kv_view(kc, vc, ks, vs, quant);
  TORCH_CHECK(q.dim() == 4 && q.scalar_type() == at::kBFloat16 && q.device() == kc.device(),
              "q: bfloat16 [B, N, Hq, D] on the caches' device");
  const int64_t B = kc.size(0), H = kc.size(1), D = kc.size(3), N = q.size(1), Hq = q.size(2);
  TORCH_CHECK(q.size(0) == B && q.size(3) == D, "q: the caches' B and D");
  TORCH_CHECK(N >= 1 && N <= kTreeNodes, "1 to 64 nodes");
  TORCH_CHECK(H >= 1 && Hq >= 1 && Hq % H == 0, "the query heads: a multiple of the caches' heads");
  TORCH_CHECK(q.stride(3) == 1 && (B == 1 || q.stride(0) % 8 == 0) && (N == 1 || q.stride(1) % 8 == 0) &&
                  (Hq == 1 || q.stride(2) % 8 == 0) && (reinterpret_cast<uintptr_t>(q.data_ptr()) & 15) == 0,
              "q: unit inner stride and 16-byte aligned rows");
  TreeArgs a{};
  a.lens = kv_ints(lens, "lens", kc.device(), B);
  a.parents = parents.has_value() ? kv_ints(*parents, "parents", kc.device(), B, N) : nullptr;
  a.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  a.qb = q.stride(0); a.qn = q.stride(1); a.qh = q.stride(2);
  a.B = (int)B; a.N = (int)N; a.Hq = (int)Hq; a.Hkv = (int)H; a.G = (int)(Hq / H);
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  c10::cuda::CUDAGuard guard(kc.device());
  auto o = at::empty({B, N, Hq, D}, q.options());
  if (o.numel() == 0) return o;
  a.o = reinterpret_cast<__nv_bfloat16*>(o.data_ptr());
  auto s = at::cuda::getCurrentCUDAStream();
  const int64_t blocks = (B * N * Hq + 3) / 4;
  TORCH_CHECK(blocks < (1LL << 31), "too many rows");
#define TFB_TREE(DD, QQ) tree_attention_simple_kernel<DD, QQ><<<(unsigned)blocks, 128, 0, s>>>(a, c)
  if (D == 128) { if (quant) TFB_TREE(128, true); else TFB_TREE(128, false); }
  else { if (quant) TFB_TREE(64, true); else TFB_TREE(64, false); }
#undef TFB_TREE
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return o;
}

}  // namespace tfb
