// Rows of a key/value cache: written (as they are or quantised), read back, and moved up when
// part of a drafted tree is accepted.  The format is described in kv_cache.cuh.
//
// All three move bytes and do nothing else that counts, so the floor is the bytes over the
// memory rate.  A row of D = 128 (64) bf16 is 16 (8) lanes of one 16-byte load each, whole lines
// a warp: the row's largest magnitude is then four (three) shuffles away, and a lane's 8 codes
// leave as one 8-byte store.  A block has one head's neighbouring rows, so that it writes (or
// reads) one contiguous piece of a head-major cache and of its scales.
//
// Measured on a B200 (calls replayed from a graph; floors at 6.54 TB/s): one row for 32 sequences of 10 heads
// 2.1 us, e4m3 or bf16; 16 x 4096 rows of 8 heads e4m3 71 us of 62, bf16 83 of 82; read of 8 x 16384 rows e4m3
// 119 us of 118, bf16 150 of 154; commit of 256 trees of 64 nodes, 8 heads, bf16 22.5 us of 10, e4m3 13.7 of 5
// (4096 blocks of a unit each, some five waves of them, and in every one the loads wait for each other: length,
// count, path, row).
// The reference has no decode path; these serve the cache of inference/generate.py.
#include <cuda_fp8.h>

#include "kv_cache.cuh"

namespace tfb {

constexpr int kKvThreads = 256;

struct KvRows {                  // rows [B, N, H, D] outside the cache
  const uint8_t* p[2];
  long long b[2], n[2], h[2];    // strides in bytes
};

// Keys' or values' entry of a parameter array.  Indexed, the array is copied to local memory by every
// thread: 109 instead of 70 us for 16 x 4096 written rows of 8 heads, 159 instead of 119 for 8 x 16384 read.
template <typename T>
__device__ __forceinline__ T pick(const T (&a)[2], int kv) { return kv ? a[1] : a[0]; }

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

// Codes under the largest scale: 256 (0x78), which stands for 2^128, becomes 240.  No other code is above 240 there.
__device__ __forceinline__ uint32_t hold_top(uint32_t c) { return c - ((((c & 0x7f7f7f7fu) + 0x08080808u) & 0x80808080u) >> 7); }

__device__ __forceinline__ uint32_t absmax8(const uint4& u) {
  const uint32_t m = 0x7fff7fffu;
  return __vmaxu2(__vmaxu2(u.x & m, u.y & m), __vmaxu2(u.z & m, u.w & m));
}

// cache[b, h, pos[b] + n] = rows[b, n, h] for n < count[b]; rows outside the cache are left out.
// A block has one (sequence, head, keys or values) and blockDim / L * U neighbouring rows, a
// thread U of them in a row.  With U = 4 the four rows' maxima are found together: two 16-bit
// maxima a word, and the two words of a thread are halved between its lanes in the first step
// (5 shuffles instead of 16: 109 instead of 114 us for 16 x 4096
// rows of 8 heads, when the parameters still were copied to local memory).
template <int D, bool QUANT, int U>
__global__ void __launch_bounds__(kKvThreads) kv_cache_write_kernel(const KvRows src, const KvView c, const int* __restrict__ pos,
                                                                    const int* __restrict__ count, int N, int H) {
  static_assert(U == 1 || U == 4, "rows a thread");
  constexpr int L = D / 8;   // lanes a row
  const int b = blockIdx.y, kv = blockIdx.z, h = blockIdx.x % H;
  const int l = threadIdx.x % L, rows = blockDim.x / L;
  const int n0 = ((int)(blockIdx.x / H) * rows + threadIdx.x / L) * U;
  const int live = count ? min(count[b], N) : N;
  const long long t0 = pos[b];
  const uint8_t* sp = pick(src.p, kv) + b * pick(src.b, kv) + h * pick(src.h, kv) + n0 * pick(src.n, kv) + 16 * l;
  uint8_t* dp = pick(c.p, kv) + b * c.b + h * c.h + (t0 + n0) * c.t;
  uint4 u[U];
  bool on[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    on[i] = n0 + i < live && t0 + n0 + i >= 0 && t0 + n0 + i < c.tmax;
    u[i] = make_uint4(0, 0, 0, 0);
    if (on[i]) u[i] = *reinterpret_cast<const uint4*>(sp + i * pick(src.n, kv));
  }
  if constexpr (!QUANT) {
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (on[i]) reinterpret_cast<uint4*>(dp + i * c.t)[l] = u[i];
  } else {
    uint32_t top[U];                           // the rows' largest magnitudes, as bf16 bits
    uint32_t m[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      m[i] = absmax8(u[i]);
      m[i] = max(m[i] & 0xffffu, m[i] >> 16);
    }
    if constexpr (U == 4) {
      const uint32_t w0 = m[0] | (m[1] << 16), w1 = m[2] | (m[3] << 16);
      const bool up = (l & (L / 2)) != 0;      // the upper lanes go on with rows 2 and 3
      uint32_t w = __vmaxu2(up ? w1 : w0, __shfl_xor_sync(0xffffffffu, up ? w0 : w1, L / 2));
#pragma unroll
      for (int o = L / 4; o > 0; o >>= 1) w = __vmaxu2(w, __shfl_xor_sync(0xffffffffu, w, o));
      const uint32_t x = __shfl_xor_sync(0xffffffffu, w, L / 2);
      const uint32_t a = up ? x : w, d = up ? w : x;
      top[0] = a & 0xffffu; top[1] = a >> 16; top[2] = d & 0xffffu; top[3] = d >> 16;
    } else {
      uint32_t w = m[0];
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) w = max(w, __shfl_xor_sync(0xffffffffu, w, o));
      top[0] = w;
    }
    uint32_t byte = 0;
    bool byte_on = false;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int e = scale_byte(top[i]);
      if (on[i]) {
        uint2 codes = make_uint2(0, 0);        // a row with an inf or NaN: its scale says so
        if (e != kScaleNan) codes = quant8(u[i], __uint_as_float((uint32_t)(254 - e) << 23));   // times 2^-(e - 127)
        if (e == kScaleMax) codes = make_uint2(hold_top(codes.x), hold_top(codes.y));
        reinterpret_cast<uint2*>(dp + i * c.t)[l] = codes;
      }
      if (l == i) {                            // lane i stores row i's scale
        byte = (uint32_t)e;
        byte_on = on[i];
      }
    }
    if (byte_on) pick(c.s, kv)[b * c.sb + h * c.sh + (t0 + n0 + l) * c.st] = (uint8_t)byte;
  }
}

// out[b, t, h] = the cached row as bf16 for t < min(lens[b], T_max), zeros for the other t < T.
// Blocks as above.
template <int D, bool QUANT, int U>
__global__ void __launch_bounds__(kKvThreads) kv_cache_read_kernel(const KvView c, const int* __restrict__ lens, uint8_t* __restrict__ k,
                                                                   uint8_t* __restrict__ v, int T, int H) {
  constexpr int L = D / 8;
  const int b = blockIdx.y, kv = blockIdx.z, h = blockIdx.x % H;
  const int l = threadIdx.x % L, rows = blockDim.x / L;
  const int t0 = (int)(blockIdx.x / H) * rows * U + threadIdx.x / L;
  const int live = min(min(lens[b], c.tmax), T);
  uint4 o[U];
  uint2 u[U];
  int e[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int t = t0 + i * rows;
    o[i] = make_uint4(0, 0, 0, 0);
    u[i] = make_uint2(0, 0);
    e[i] = 127;
    if (t < live) {
      const uint8_t* p = pick(c.p, kv) + b * c.b + h * c.h + (long long)t * c.t;
      if constexpr (QUANT) {
        u[i] = reinterpret_cast<const uint2*>(p)[l];
        e[i] = pick(c.s, kv)[b * c.sb + h * c.sh + t * c.st];
      } else {
        o[i] = reinterpret_cast<const uint4*>(p)[l];
      }
    }
  }
  uint8_t* out = (kv ? v : k) + ((long long)b * T * H + h) * (D * 2);
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int t = t0 + i * rows;
    if constexpr (QUANT) {
      const float sc = e[i] == kScaleNan ? __int_as_float(0x7fffffff) : e[i] == 0 ? 0x1p-127f : __uint_as_float((uint32_t)e[i] << 23);
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((j < 2 ? u[i].x : u[i].y) >> (16 * (j & 1))), __NV_E4M3);
        const float2 f = __half22float2(__half2(hr));
        w[j] = pack_bf16x2(f.x * sc, f.y * sc);
      }
      o[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (t < T) reinterpret_cast<uint4*>(out + (long long)t * H * (D * 2))[l] = o[i];
  }
}

// cache[b, h, lens[b] + i] = cache[b, h, lens[b] + path[b, i]], i < count[b], path ascending with
// path[i] >= i.  A source is then never below its own target and never a target of an earlier
// move, so moves in order of i are right in place -- and so are batches of moves of which all
// rows are loaded before any is stored.  A block of 256 threads has units of at most 64 rows, a unit
// being one (sequence, head, keys or values): `rows` rows of L lanes at a time, U times, held in
// registers between the two barriers.
template <int ROW>   // bytes of a row
__global__ void __launch_bounds__(kKvThreads, 6) kv_cache_commit_kernel(const KvView c, const int* __restrict__ lens, const int* __restrict__ path,
                                                                        const int* __restrict__ count, int B, int N, int H, int rows) {
  constexpr int L = ROW / 16, U = ROW / 64;   // 64 rows a batch: U * 256 / L
  const int threads = rows * L;
  const int slot = threadIdx.x / threads, id = threadIdx.x - slot * threads;
  const int units = kKvThreads / threads;
  const long long unit = (long long)blockIdx.x * units + slot;
  const bool real = slot < units && unit < 2LL * B * H;
  const int kv = (int)(unit & 1), b = real ? (int)((unit >> 1) / H) : 0, h = (int)((unit >> 1) % H);
  const long long t0 = lens[b];
  const int m = real && t0 >= 0 ? min(count[b], N) : 0;
  const int* pp = path + (long long)b * N;
  const int l = id % L, i1 = id / L;
  uint8_t* base = pick(c.p, kv) + b * c.b + h * c.h + t0 * c.t + 16 * l;
  uint8_t* sbase = pick(c.s, kv) && l == 0 ? pick(c.s, kv) + b * c.sb + h * c.sh + t0 * c.st : nullptr;
  const int room = (int)min((long long)N, c.tmax - t0);   // rows behind the context
  for (int i0 = i1; i0 - i1 < N; i0 += U * rows) {
    uint4 u[U];
    uint8_t s[U];
    int src[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = i0 + j * rows;
      src[j] = i < m ? pp[i] : -1;
      if (src[j] <= i || src[j] >= room) src[j] = -1;
    }
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (src[j] >= 0) {
        u[j] = *reinterpret_cast<const uint4*>(base + src[j] * c.t);
        if (sbase) s[j] = sbase[src[j] * c.st];
      }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (src[j] >= 0) {
        const int i = i0 + j * rows;
        *reinterpret_cast<uint4*>(base + i * c.t) = u[j];
        if (sbase) sbase[i * c.st] = s[j];
      }
    if (N > U * rows) __syncthreads();
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

// Blocks of the row kernels: up to 256 threads of D / 8 lanes a row, four rows a thread where
// there are enough rows to fill the GPU with fewer threads.
static dim3 kv_grid(int64_t N, int64_t H, int64_t B, int64_t D, int& threads, int& U) {
  const int64_t L = D / 8, most = kKvThreads / L;
  U = N >= 4 * most ? 4 : 1;
  const int64_t rows = std::min(most, N);
  threads = (int)((rows * L + 31) / 32 * 32);
  const int64_t per = threads / L * U, gx = (N + per - 1) / per * H;
  TORCH_CHECK(gx < (1LL << 31), "too many rows");
  return dim3((unsigned)gx, (unsigned)B, 2);
}

static void check_batch(int64_t B) { TORCH_CHECK(B <= 65535, "at most 65535 sequences"); }

void kv_cache_write(at::Tensor k, at::Tensor v, at::Tensor kc, at::Tensor vc, at::Tensor pos,
                    c10::optional<at::Tensor> count, c10::optional<at::Tensor> ks, c10::optional<at::Tensor> vs) {
  bool quant;
  const KvView c = kv_view(kc, vc, ks, vs, quant);
  kv_check_scales_written(ks);
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
  int threads, U;
  const dim3 grid = kv_grid(N, H, B, D, threads, U);
#define TFB_KV_WRITE(DD, QQ) \
  (U == 1 ? kv_cache_write_kernel<DD, QQ, 1><<<grid, threads, 0, s>>>(r, c, pp, cp, (int)N, (int)H) \
          : kv_cache_write_kernel<DD, QQ, 4><<<grid, threads, 0, s>>>(r, c, pp, cp, (int)N, (int)H))
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
  int threads, U;
  const dim3 grid = kv_grid(T, H, B, D, threads, U);
  auto* kp = static_cast<uint8_t*>(k.data_ptr());
  auto* vp = static_cast<uint8_t*>(v.data_ptr());
#define TFB_KV_READ(DD, QQ) \
  (U == 1 ? kv_cache_read_kernel<DD, QQ, 1><<<grid, threads, 0, s>>>(c, lp, kp, vp, (int)T, (int)H) \
          : kv_cache_read_kernel<DD, QQ, 4><<<grid, threads, 0, s>>>(c, lp, kp, vp, (int)T, (int)H))
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
  kv_check_scales_written(ks);
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
  const int64_t row = D * (quant ? 1 : 2);
  const int rows = (int)std::min<int64_t>(N, kKvThreads / (row / 16));
  const int64_t units = kKvThreads / (rows * (row / 16)), gx = (2 * B * H + units - 1) / units;
  TORCH_CHECK(gx < (1LL << 31), "too many rows");
#define TFB_KV_COMMIT(RR) kv_cache_commit_kernel<RR><<<(unsigned)gx, kKvThreads, 0, s>>>(c, lp, pp, cp, (int)B, (int)N, (int)H, rows)
  if (row == 256) TFB_KV_COMMIT(256);
  else if (row == 128) TFB_KV_COMMIT(128);
  else TFB_KV_COMMIT(64);
#undef TFB_KV_COMMIT
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace tfb
