// A key/value cache as the serving kernels address it: [B, H, T, D] by strides (so head-major
// and token-major storage alike), bf16 rows or quantised rows.
//
// Quantised rows: e4m3 codes and one e8m0 scale byte a row (value = code * 2^(byte - 127),
// 255 = NaN).  The scale is a power of two, so quantising is one exact multiplication and one
// rounding, and every cached value is exactly a bf16 number: reading back never rounds.  (Under the
// largest scale that a bf16 row can need, 2^120, code 256 would stand for 2^128: such a value is held
// as 240 instead.  Under larger ones, which only a caller's own cache can hold, values past bf16's
// range may become infinite.)  An
// fp32 scale would use the top of the e4m3 range up to one binade better, which changes no
// significand bit of a value above the subnormals, and costs four bytes a row instead of one.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>

#include "sm100_common.cuh"

namespace tfb {

constexpr int kScaleMin = 10;    // exponent byte of the least scale, 2^-117: every e4m3 normal times it is a bf16 normal
constexpr int kScaleMax = 247;   // of the largest one that is written, 2^120
constexpr int kScaleNan = 255;

struct KvView {
  uint8_t* p[2];            // key / value rows
  uint8_t* s[2];            // scale bytes (quantised caches), else null
  long long b, h, t;        // strides in bytes
  long long sb, sh, st;     // strides of the scale bytes
  int tmax;
};

// Checks a pair of caches (and their scales) and returns the view; `quant`: whether they are e4m3.
inline KvView kv_view(const at::Tensor& kc, const at::Tensor& vc, const c10::optional<at::Tensor>& ks,
                      const c10::optional<at::Tensor>& vs, bool& quant) {
  TORCH_CHECK(kc.dim() == 4 && kc.sizes() == vc.sizes() && kc.strides() == vc.strides(),
              "k_cache and v_cache: [B, H, T, D] of the same sizes and strides");
  TORCH_CHECK(kc.scalar_type() == vc.scalar_type() && kc.device() == vc.device(), "k_cache and v_cache: one type and device");
  quant = kc.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(quant || kc.scalar_type() == at::kBFloat16, "caches: bfloat16 or float8_e4m3fn");
  const int64_t D = kc.size(3);
  TORCH_CHECK(D == 64 || D == 128, "head_dim 64 or 128");
  TORCH_CHECK(kc.size(2) >= 1 && kc.size(2) <= (1 << 30), "cache rows 1 .. 2^30");
  const int64_t es = quant ? 1 : 2;
  KvView v{};
  v.b = kc.stride(0) * es; v.h = kc.stride(1) * es; v.t = kc.stride(2) * es;
  v.tmax = (int)kc.size(2);
  // a dimension of one entry is never stepped over: give it a stride that every path accepts
  if (kc.size(0) == 1) v.b = D * es;
  if (kc.size(1) == 1) v.h = D * es;
  if (kc.size(2) == 1) v.t = D * es;
  v.p[0] = static_cast<uint8_t*>(kc.data_ptr());
  v.p[1] = static_cast<uint8_t*>(vc.data_ptr());
  TORCH_CHECK(kc.stride(3) == 1 && v.b > 0 && v.h > 0 && v.t > 0 && v.b % 16 == 0 && v.h % 16 == 0 && v.t % 16 == 0 &&
                  ((reinterpret_cast<uintptr_t>(v.p[0]) | reinterpret_cast<uintptr_t>(v.p[1])) & 15) == 0,
              "caches: unit inner stride, 16-byte aligned rows, no broadcast dimension");
  TORCH_CHECK(quant == ks.has_value() && quant == vs.has_value(),
              "k_scale and v_scale: given with float8_e4m3fn caches, and only with them");
  if (quant) {
    TORCH_CHECK(ks->scalar_type() == at::kFloat8_e8m0fnu && vs->scalar_type() == at::kFloat8_e8m0fnu &&
                    ks->device() == kc.device() && vs->device() == kc.device(),
                "scales: float8_e8m0fnu on the caches' device");
    TORCH_CHECK(ks->dim() == 3 && ks->sizes() == kc.sizes().slice(0, 3) && vs->sizes() == ks->sizes() &&
                    vs->strides() == ks->strides(), "scales: [B, H, T] of the same strides");
    v.s[0] = static_cast<uint8_t*>(ks->data_ptr());
    v.s[1] = static_cast<uint8_t*>(vs->data_ptr());
    v.sb = ks->stride(0); v.sh = ks->stride(1); v.st = ks->stride(2);
  }
  return v;
}

// Whether every row has a scale byte of its own, as storing one needs.
inline void kv_check_scales_written(const c10::optional<at::Tensor>& ks) {
  if (!ks.has_value()) return;
  for (int i = 0; i < 3; ++i)
    TORCH_CHECK(ks->size(i) <= 1 || ks->stride(i) > 0, "scales that are written: no broadcast dimension");
}

// An int32 tensor [B] (or [B, N]) on the caches' device, packed.
inline const int* kv_ints(const at::Tensor& t, const char* name, c10::Device dev, int64_t B, int64_t N = -1) {
  const bool fits = N < 0 ? t.dim() == 1 && t.size(0) == B : t.dim() == 2 && t.size(0) == B && t.size(1) == N;
  TORCH_CHECK(t.scalar_type() == at::kInt && t.device() == dev && fits && t.is_contiguous(), name, ": contiguous int32 of ",
              N < 0 ? "[B]" : "[B, N]", " entries on the caches' device");
  return t.data_ptr<int>();
}

}  // namespace tfb
