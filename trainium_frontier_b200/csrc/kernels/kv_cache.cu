// Rows of a key/value cache: written (as they are or quantised), read back, and moved up when
// part of a drafted tree is accepted.  The format is described in kv_cache.cuh.
//
// All three move bytes and do nothing else that counts, so the floor is the bytes over the
// memory rate.  A row of D = 128 (64) bf16 is 8 (4) lanes of two 16-byte loads each: the row's
// largest magnitude is then three (two) shuffles away, and each lane's 16 codes leave as one
// 16-byte store.
// The reference has no decode path; these serve the cache of inference/generate.py.
#include <cuda_fp8.h>

#include "kv_cache.cuh"

namespace tfb {

constexpr int kKvThreads = 256;

struct KvRows {                  // rows [B, N, H, D] outside the cache
  const uint8_t* p[2];
  long long b[2], n[2], h[2];    // strides in bytes
};

// Exponent byte of the least power-of-two scale (2^-117 at the least) under which a row whose
// largest magnitude has the bf16 bits `amax` fits +-448 = 1.75 * 2^8; 255 if it is not finite.
__device__ __forceinline__ int scale_byte(uint32_t amax) {
  const int ex = (int)(amax >> 7);
  if (ex == 255) return kScaleNan;
  const int e = ex - 8 + ((amax & 127u) > 96u ? 1 : 0);
  return e < kScaleMin ? kScaleMin : e;
}

// 8 bf16 (one 16-byte load) times `inv` as 8 e4m3 codes, rounded to nearest even.
__device__ __forceinline__ uint2 quant8(const uint4& u, float inv) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = make_float2(__uint_as_float(w[i] << 16) * inv, __uint_as_float(w[i] & 0xffff0000u) * inv);
    c[i] = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}

__device__ __forceinline__ uint32_t absmax8(const uint4& u) {
  const uint32_t m = 0x7fff7fffu;
  return __vmaxu2(__vmaxu2(u.x & m, u.y & m), __vmaxu2(u.z & m, u.w & m));
}

// cache[b, :, pos[b] + n] = rows[b, n] for n < count[b]; rows outside the cache are left out.
template <int D, bool QUANT>
__global__ void __launch_bounds__(kKvThreads) kv_cache_write_kernel(const KvRows src, const KvView c, const int* __restrict__ pos,
                                                                    const int* __restrict__ count, int N, int H) {
  constexpr int L = D / 16;   // lanes a row
  const int b = blockIdx.y, kv = blockIdx.z;
  const long long r = (long long)blockIdx.x * (kKvThreads / L) + threadIdx.x / L;
  const int l = threadIdx.x % L;
  const int n = (int)(r / H), h = (int)(r % H);
  const long long t = (long long)pos[b] + n;
  const int live = count ? min(count[b], N) : N;
  const bool on = n < live && t >= 0 && t < c.tmax;
  uint4 u0 = make_uint4(0, 0, 0, 0), u1 = u0;
  if (on) {
    const uint4* p = reinterpret_cast<const uint4*>(src.p[kv] + b * src.b[kv] + n * src.n[kv] + h * src.h[kv]) + 2 * l;
    u0 = p[0];
    u1 = p[1];
  }
  uint8_t* dst = c.p[kv] + b * c.b + h * c.h + t * c.t;
  if constexpr (!QUANT) {
    if (on) {
      reinterpret_cast<uint4*>(dst)[2 * l] = u0;
      reinterpret_cast<uint4*>(dst)[2 * l + 1] = u1;
    }
  } else {
    uint32_t m = __vmaxu2(absmax8(u0), absmax8(u1));
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    const int e = scale_byte(max(m & 0xffffu, m >> 16));
    if (on) {
      uint4 codes = make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);  // a row with an inf or NaN: NaN codes too
      if (e != kScaleNan) {
        const float inv = __uint_as_float((uint32_t)(254 - e) << 23);   // 2^-(e - 127)
        const uint2 a = quant8(u0, inv), d = quant8(u1, inv);
        codes = make_uint4(a.x, a.y, d.x, d.y);
      }
      reinterpret_cast<uint4*>(dst)[l] = codes;
      if (l == 0) c.s[kv][b * c.sb + h * c.sh + t * c.st] = (uint8_t)e;
    }
  }
}

// out[b, t, h] = the cached row as bf16 for t < min(lens[b], T_max), zeros for the other t < T.
template <int D, bool QUANT>
__global__ void __launch_bounds__(kKvThreads) kv_cache_read_kernel(const KvView c, const int* __restrict__ lens, uint8_t* __restrict__ k,
                                                                   uint8_t* __restrict__ v, int T, int H) {
  constexpr int L = D / 16;
  const int b = blockIdx.y, kv = blockIdx.z;
  const long long r = (long long)blockIdx.x * (kKvThreads / L) + threadIdx.x / L;
  const int l = threadIdx.x % L;
  const int t = (int)(r / H), h = (int)(r % H);
  if (t >= T) return;
  uint4 o0 = make_uint4(0, 0, 0, 0), o1 = o0;
  if (t < lens[b] && t < c.tmax) {
    const uint4* p = reinterpret_cast<const uint4*>(c.p[kv] + b * c.b + h * c.h + (long long)t * c.t);
    if constexpr (!QUANT) {
      o0 = p[2 * l];
      o1 = p[2 * l + 1];
    } else {
      const uint4 u = p[l];
      const int e = c.s[kv][b * c.sb + h * c.sh + t * c.st];
      const float sc = e == kScaleNan ? __int_as_float(0x7fffffff) : e == 0 ? 0x1p-127f : __uint_as_float((uint32_t)e << 23);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
      uint32_t o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
        const float2 f = __half22float2(__half2(hr));
        o[i] = pack_bf16x2(f.x * sc, f.y * sc);
      }
      o0 = make_uint4(o[0], o[1], o[2], o[3]);
      o1 = make_uint4(o[4], o[5], o[6], o[7]);
    }
  }
  uint4* dst = reinterpret_cast<uint4*>((kv ? v : k) + (((long long)b * T + t) * H + h) * (D * 2)) + 2 * l;
  dst[0] = o0;
  dst[1] = o1;
}

// cache[b, h, lens[b] + i] = cache[b, h, lens[b] + path[b, i]], i < count[b], path ascending with
// path[i] >= i.  A source is then never below its own target and never a target of an earlier
// move, so moves in order of i are right in place; loading a batch of rows before storing any
// of it keeps that order (every row of a batch is loaded before the batch stores).  One lane
// owns 16 bytes of a row for all moves.
template <int ROW>   // bytes of a row
__global__ void __launch_bounds__(kKvThreads) kv_cache_commit_kernel(const KvView c, const int* __restrict__ lens, const int* __restrict__ path,
                                                                     const int* __restrict__ count, int B, int N, int H) {
  constexpr int L = ROW / 16, U = 8;
  const long long g = (long long)blockIdx.x * (kKvThreads / L) + threadIdx.x / L;
  if (g >= 2LL * B * H) return;
  const int l = threadIdx.x % L;
  const int kv = (int)(g & 1), b = (int)((g >> 1) / H), h = (int)((g >> 1) % H);
  const long long t0 = lens[b];
  const int m = min(count[b], N);
  const int* pp = path + (long long)b * N;
  uint8_t* base = c.p[kv] + b * c.b + h * c.h + 16 * l;
  uint8_t* sbase = c.s[kv] ? c.s[kv] + b * c.sb + h * c.sh : nullptr;
  if (t0 < 0) return;
  for (int i0 = 0; i0 < m; i0 += U) {
    uint4 u[U];
    uint8_t s[U];
    bool on[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = i0 + j;
      const int src = i < m ? pp[i] : -1;
      on[j] = src > i && src < N && t0 + src < c.tmax;
      if (on[j]) {
        u[j] = *reinterpret_cast<const uint4*>(base + (t0 + src) * c.t);
        if (sbase && l == 0) s[j] = sbase[(t0 + src) * c.st];
      }
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (on[j]) {
        *reinterpret_cast<uint4*>(base + (t0 + i0 + j) * c.t) = u[j];
        if (sbase && l == 0) sbase[(t0 + i0 + j) * c.st] = s[j];
      }
    }
  }
}

static KvRows kv_rows(const at::Tensor& k, const at::Tensor& v, const at::Tensor& kc) {
  KvRows r{};
  const at::Tensor* t[2] = {&k, &v};
  for (int i = 0; i < 2; ++i) {
    TORCH_CHECK(t[i]->scalar_type() == at::kBFloat16 && t[i]->device() == kc.device() && t[i]->dim() == 4 &&
                    t[i]->size(0) == kc.size(0) && t[i]->size(1) == k.size(1) && t[i]->size(2) == kc.size(1) &&
                    t[i]->size(3) == kc.size(3), "k and v: bfloat16 [B, N, H, D] of the caches' B, H, D on their device");
    r.p[i] = static_cast<const uint8_t*>(t[i]->data_ptr());
    r.b[i] = t[i]->stride(0) * 2; r.n[i] = t[i]->stride(1) * 2; r.h[i] = t[i]->stride(2) * 2;
    TORCH_CHECK(t[i]->stride(3) == 1 && (t[i]->size(0) == 1 || r.b[i] % 16 == 0) && (t[i]->size(1) == 1 || r.n[i] % 16 == 0) &&
                    (t[i]->size(2) == 1 || r.h[i] % 16 == 0) && (reinterpret_cast<uintptr_t>(r.p[i]) & 15) == 0,
                "k and v: unit inner stride and 16-byte aligned rows");
  }
  return r;
}

static void check_batch(int64_t B) { TORCH_CHECK(B <= 65535, "at most 65535 sequences"); }

void kv_cache_write(at::Tensor k, at::Tensor v, at::Tensor kc, at::Tensor vc, at::Tensor pos,
                    c10::optional<at::Tensor> count, c10::optional<at::Tensor> ks, c10::optional<at::Tensor> vs) {
  bool quant;
  const KvView c = kv_view(kc, vc, ks, vs, quant);
  TORCH_CHECK(k.dim() == 4, "k and v: bfloat16 [B, N, H, D]");
  const KvRows r = kv_rows(k, v, kc);
  const int64_t B = kc.size(0), N = k.size(1), H = kc.size(1), D = kc.size(3);
  const int* pp = kv_ints(pos, "pos", kc.device(), B);
  const int* cp = count.has_value() ? kv_ints(*count, "count", kc.device(), B) : nullptr;
  check_batch(B);
  TORCH_CHECK(N <= (1 << 30), "at most 2^30 rows");
  if (B == 0 || N == 0 || H == 0) return;
  c10::cuda::CUDAGuard guard(kc.device());
  auto s = at::cuda::getCurrentCUDAStream();
  const int64_t per = kKvThreads / (D / 16), gx = (N * H + per - 1) / per;
  TORCH_CHECK(gx < (1LL << 31), "too many rows");
  const dim3 grid((unsigned)gx, (unsigned)B, 2);
#define TFB_KV_WRITE(DD, QQ) kv_cache_write_kernel<DD, QQ><<<grid, kKvThreads, 0, s>>>(r, c, pp, cp, (int)N, (int)H)
  if (D == 128) { if (quant) TFB_KV_WRITE(128, true); else TFB_KV_WRITE(128, false); }
  else { if (quant) TFB_KV_WRITE(64, true); else TFB_KV_WRITE(64, false); }
#undef TFB_KV_WRITE
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

std::vector<at::Tensor> kv_cache_read(at::Tensor kc, at::Tensor vc, at::Tensor lens, int64_t T,
                                         c10::optional<at::Tensor> ks, c10::optional<at::Tensor> vs) {
  bool quant;
  const KvView c = kv_view(kc, vc, ks, vs, quant);
  const int64_t B = kc.size(0), H = kc.size(1), D = kc.size(3);
  TORCH_CHECK(T >= 0 && T <= kc.size(2), "T: 0 .. the cache's rows");
  const int* lp = kv_ints(lens, "lens", kc.device(), B);
  check_batch(B);
  c10::cuda::CUDAGuard guard(kc.device());
  auto opt = kc.options().dtype(at::kBFloat16);
  auto k = at::empty({B, T, H, D}, opt), v = at::empty({B, T, H, D}, opt);
  if (k.numel() == 0) return {k, v};
  auto s = at::cuda::getCurrentCUDAStream();
  const int64_t per = kKvThreads / (D / 16), gx = (T * H + per - 1) / per;
  TORCH_CHECK(gx < (1LL << 31), "too many rows");
  const dim3 grid((unsigned)gx, (unsigned)B, 2);
  auto* kp = static_cast<uint8_t*>(k.data_ptr());
  auto* vp = static_cast<uint8_t*>(v.data_ptr());
#define TFB_KV_READ(DD, QQ) kv_cache_read_kernel<DD, QQ><<<grid, kKvThreads, 0, s>>>(c, lp, kp, vp, (int)T, (int)H)
  if (D == 128) { if (quant) TFB_KV_READ(128, true); else TFB_KV_READ(128, false); }
  else { if (quant) TFB_KV_READ(64, true); else TFB_KV_READ(64, false); }
#undef TFB_KV_READ
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {k, v};
}

void kv_cache_commit(at::Tensor kc, at::Tensor vc, at::Tensor lens, at::Tensor path, at::Tensor count,
                     c10::optional<at::Tensor> ks, c10::optional<at::Tensor> vs) {
  bool quant;
  const KvView c = kv_view(kc, vc, ks, vs, quant);
  const int64_t B = kc.size(0), H = kc.size(1), D = kc.size(3);
  TORCH_CHECK(path.dim() == 2, "path: int32 [B, N]");
  const int64_t N = path.size(1);
  const int* lp = kv_ints(lens, "lens", kc.device(), B);
  const int* pp = kv_ints(path, "path", kc.device(), B, N);
  const int* cp = kv_ints(count, "count", kc.device(), B);
  check_batch(B);
  if (B == 0 || H == 0 || N == 0) return;
  c10::cuda::CUDAGuard guard(kc.device());
  auto s = at::cuda::getCurrentCUDAStream();
  const int64_t row = D * (quant ? 1 : 2), per = kKvThreads / (row / 16), gx = (2 * B * H + per - 1) / per;
  TORCH_CHECK(gx < (1LL << 31), "too many rows");
#define TFB_KV_COMMIT(RR) kv_cache_commit_kernel<RR><<<(unsigned)gx, kKvThreads, 0, s>>>(c, lp, pp, cp, (int)B, (int)N, (int)H)
  if (row == 256) TFB_KV_COMMIT(256);
  else if (row == 128) TFB_KV_COMMIT(128);
  else TFB_KV_COMMIT(64);
#undef TFB_KV_COMMIT
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace tfb
