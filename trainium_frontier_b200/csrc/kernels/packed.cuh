// Sequences that lie behind one another in one buffer of M rows, as the packed kernels find them:
// cu [S + 1] ascending, sequence s being rows cu[s] .. cu[s + 1] - 1.  Whatever cu holds, no row
// outside 0 .. M - 1 is reached.
#pragma once

#include "sm100_common.cuh"

namespace tfb {

// Rows in front of the first sequence and behind the last one are taken as two more "sequences",
// 0 and S + 1, so that pieces 0 .. S + 1 cover all rows.
struct Pieces {
  const int* cu;
  int S, M;
  __device__ __forceinline__ int begin(int k) const { return k == 0 ? 0 : max(0, min(cu[k - 1], M)); }
  __device__ __forceinline__ int end(int k) const { return k == S + 1 ? M : max(begin(k), min(cu[k], M)); }
  __device__ __forceinline__ bool real(int k) const { return k >= 1 && k <= S; }
};

// Units of U rows, cut from every piece's start on, are numbered so that the number of a piece's first
// one, begin / U + k, needs no sum over the pieces before it; some numbers stay unused.
__host__ __device__ __forceinline__ long long piece_slots(long long M, long long S, int U) { return M / U + S + 2; }

// The last piece k with key(k) <= x, key ascending and key(0) <= x (warp-collective: 32 probes a step).
template <typename F>
__device__ __forceinline__ int last_piece(int n, long long x, F key) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int step = (hi - lo + 32) / 32;
    const int k = lo + lane * step;
    const unsigned hit = __ballot_sync(0xffffffffu, k <= hi && (lane == 0 || key(k) <= x));
    lo += (31 - __clz(hit)) * step;
    hi = min(hi, lo + step - 1);
  }
  return lo;
}

struct PieceUnit {
  int piece, begin, len, unit;   // unit < 0: the slot is unused
};
// What slot `slot` of the units of U rows is (warp-collective).
template <int U>
__device__ __forceinline__ PieceUnit piece_unit(const Pieces& p, int slot) {
  // as last_piece; the last step's probes hold the piece's begin and the next one's, which is its end
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = p.S + 1, begin = -1, end = -1;
  while (lo < hi) {
    const int step = (hi - lo + 32) / 32, i = lo + lane * step;
    const int at = i <= hi ? p.begin(i) : 0;
    const unsigned hit = __ballot_sync(0xffffffffu, i <= hi && (lane == 0 || (long long)at / U + i <= slot));
    const int top = 31 - __clz(hit);
    begin = __shfl_sync(0xffffffffu, at, top);
    end = __shfl_sync(0xffffffffu, at, (top + 1) & 31);
    if (step > 1 || top == 31 || lo + top + 1 > hi) end = -1;   // not probed
    lo += top * step;
    hi = min(hi, lo + step - 1);
  }
  const int k = lo;
  PieceUnit u;
  u.piece = k;
  u.begin = begin;
  if (end < 0) end = p.end(k);
  u.len = max(end, begin) - begin;
  u.unit = slot - (u.begin / U + k);
  if (u.unit < 0 || (long long)u.unit * U >= u.len) u.unit = -1;
  return u;
}

}  // namespace tfb
