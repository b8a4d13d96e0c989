// Rows of new keys and values into a cache of pages: row r of sequence s, the n-th of its new rows,
// becomes row (pos[s] + n) % page of page table[s, (pos[s] + n) / page].  The format of quantised rows is
// that of kv_cache.cuh.
//
// Bytes bound the time, so the kernel is that of kv_cache_write: 16 (8) lanes of one 16-byte load a row of 128
// (64), a block on one head's neighbouring rows, which are one contiguous piece of each head-major page.
// A warp finds its first row's sequence with 32 probes a step and its further rows' by walking on.
//
// Measured on a B200 (calls replayed from a graph): 16 prompts of 2048 .. 4096 rows of 8 heads of 128, bf16, pages of 16: 71 us
// of 61 (87 % of the copy rate), e4m3 102 us of 46 (not looked into yet); one row for 32 sequences of 10 heads, e4m3: 2.9 us (a launch and three dependent loads).
#include "kv_cache.cuh"
#include "packed.cuh"

namespace tfb {

constexpr int kPagedThreads = 256;

struct PagedRows {               // rows [M, H, D]
  const uint8_t* p[2];
  long long n[2], h[2];          // strides in bytes
};

template <int D, bool QUANT, int U>
__global__ void __launch_bounds__(kPagedThreads) paged_cache_write_kernel(const PagedRows src, const KvView c, const int* __restrict__ table,
                                                                          long long tb, int width, const int* __restrict__ pos,
                                                                          const Pieces pc, int pages, int lg, int H) {
  constexpr int L = D / 8;       // lanes a row
  const int kv = blockIdx.y, h = blockIdx.x % H;
  const int l = threadIdx.x % L, rows = blockDim.x / L;
  const int n0 = ((int)(blockIdx.x / H) * rows + threadIdx.x / L) * U;
  int s;
  if (pc.cu) {                   // warp-collective: the sequence of the warp's first row
    const int first = ((int)(blockIdx.x / H) * rows + (int)(threadIdx.x & ~31u) / L) * U;
    s = last_piece(pc.S + 2, first, [&](int k) { return (long long)pc.begin(k); });
  } else {
    s = n0 + 1;                  // one row a sequence
  }
  uint4 u[U];
  long long dst[U], sdst[U];
  bool on[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int n = n0 + i;
    on[i] = n < pc.M;
    u[i] = make_uint4(0, 0, 0, 0);
    dst[i] = sdst[i] = 0;
    if (!on[i]) continue;
    int at = 0;
    if (pc.cu) {
      while (s <= pc.S && n >= pc.end(s)) ++s;
      on[i] = pc.real(s) && n >= pc.begin(s);
      if (!on[i]) continue;
      at = n - pc.begin(s);
    } else {
      s = n + 1;
    }
    const long long t = (long long)pos[s - 1] + at, w = t >> lg;
    const int page = t >= 0 && w < width ? table[(s - 1) * tb + w] : -1;
    on[i] = page >= 0 && page < pages;
    if (!on[i]) continue;
    const long long in = t & ((1 << lg) - 1);
    dst[i] = page * c.b + h * c.h + in * c.t;
    if constexpr (QUANT) sdst[i] = page * c.sb + h * c.sh + in * c.st;
    u[i] = *reinterpret_cast<const uint4*>(pick(src.p, kv) + n * pick(src.n, kv) + h * pick(src.h, kv) + 16 * l);
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if constexpr (!QUANT) {
      if (on[i]) reinterpret_cast<uint4*>(pick(c.p, kv) + dst[i])[l] = u[i];
    } else {
      uint32_t m = absmax8(u[i]);
      m = max(m & 0xffffu, m >> 16);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      const int e = scale_byte(m);
      if (on[i]) {
        uint2 codes = make_uint2(0, 0);        // a row with an inf or NaN: its scale says so
        if (e != kScaleNan) codes = quant8(u[i], __uint_as_float((uint32_t)(254 - e) << 23));
        if (e == kScaleMax) codes = make_uint2(hold_top(codes.x), hold_top(codes.y));
        reinterpret_cast<uint2*>(pick(c.p, kv) + dst[i])[l] = codes;
        if (l == 0) pick(c.s, kv)[sdst[i]] = (uint8_t)e;
      }
    }
  }
}

// Rows of a page (a power of two from 16 on) as their logarithm.
int page_log(int64_t page) {
  int lg = 0;
  while ((1LL << lg) < page) ++lg;
  TORCH_CHECK(page >= 16 && page <= 65536 && (1LL << lg) == page, "pages: a power of two from 16 to 65536 rows");
  return lg;
}

// The table [B, W] of page numbers: rows of unit inner stride on the pages' device.
const int* page_table(const at::Tensor& t, const at::Tensor& kp, int64_t B) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.device() == kp.device() && t.dim() == 2 && t.size(0) == B && (t.size(1) <= 1 || t.stride(1) == 1),
              "page_table: int32 [B, W] with unit inner stride on the pages' device");
  TORCH_CHECK(t.size(1) * kp.size(2) <= (1 << 30), "page_table: at most 2^30 rows a sequence");
  return t.data_ptr<int>();
}

void paged_cache_write(at::Tensor k, at::Tensor v, at::Tensor kp, at::Tensor vp, at::Tensor table, at::Tensor pos,
                       c10::optional<at::Tensor> cu, c10::optional<at::Tensor> ks, c10::optional<at::Tensor> vs) {
  TORCH_CHECK(kp.is_cuda(), "pages: CUDA tensors");
  bool quant;
  const KvView c = kv_view(kp, vp, ks, vs, quant);
  kv_check_scales_written(ks);
  const int lg = page_log(kp.size(2));
  const int64_t H = kp.size(1), D = kp.size(3), B = pos.dim() == 1 ? pos.size(0) : -1;
  const int* pp = kv_ints(pos, "pos", kp.device(), B);
  const int* tp = page_table(table, kp, B);
  TORCH_CHECK(k.dim() == 3, "k and v: bfloat16 [M, H, D]");
  const int64_t M = k.size(0);
  PagedRows r{};
  const at::Tensor* t[2] = {&k, &v};
  for (int i = 0; i < 2; ++i) {
    TORCH_CHECK(t[i]->scalar_type() == at::kBFloat16 && t[i]->device() == kp.device() && t[i]->dim() == 3 && t[i]->size(0) == M &&
                    t[i]->size(1) == H && t[i]->size(2) == D, "k and v: bfloat16 [M, H, D] of the pages' H, D on their device");
    r.p[i] = static_cast<const uint8_t*>(t[i]->data_ptr());
    r.n[i] = t[i]->stride(0) * 2; r.h[i] = t[i]->stride(1) * 2;
    TORCH_CHECK(t[i]->stride(2) == 1 && (M <= 1 || r.n[i] % 16 == 0) && (H == 1 || r.h[i] % 16 == 0) &&
                    (reinterpret_cast<uintptr_t>(r.p[i]) & 15) == 0, "k and v: unit inner stride and 16-byte aligned rows");
  }
  Pieces pc{};
  TORCH_CHECK(M <= (1 << 30) && B < (1 << 30), "at most 2^30 rows and sequences");
  pc.S = (int)B; pc.M = (int)M;
  if (cu.has_value()) pc.cu = kv_ints(*cu, "cu_seqlens", kp.device(), B + 1);
  else TORCH_CHECK(M == B, "without cu_seqlens: one row for each sequence");
  if (M == 0 || B == 0 || H == 0 || kp.size(0) == 0) return;
  c10::cuda::CUDAGuard guard(kp.device());
  auto s = at::cuda::getCurrentCUDAStream();
  const int64_t L = D / 8, most = kPagedThreads / L;
  const int U = M >= 4 * most ? 4 : 1;
  const int threads = (int)((std::min(most, M) * L + 31) / 32 * 32);
  const int64_t per = threads / L * U, gx = (M + per - 1) / per * H;
  TORCH_CHECK(gx < (1LL << 31), "too many rows");
  const dim3 grid((unsigned)gx, 2);
  const int W = (int)table.size(1), P = (int)kp.size(0);
  const long long tb = table.stride(0);
#define TFB_PAGED_WRITE(DD, QQ) \
  (U == 1 ? paged_cache_write_kernel<DD, QQ, 1><<<grid, threads, 0, s>>>(r, c, tp, tb, W, pp, pc, P, lg, (int)H) \
          : paged_cache_write_kernel<DD, QQ, 4><<<grid, threads, 0, s>>>(r, c, tp, tb, W, pp, pc, P, lg, (int)H))
  if (D == 128) { if (quant) TFB_PAGED_WRITE(128, true); else TFB_PAGED_WRITE(128, false); }
  else { if (quant) TFB_PAGED_WRITE(64, true); else TFB_PAGED_WRITE(64, false); }
#undef TFB_PAGED_WRITE
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace tfb
