// Causal attention of sequences that lie behind one another in one buffer, with shared key/value
// heads, forward and backward, on the 5th-generation tensor cores.
//
//   o_i = sum_{j <= i} p_ij v_j,   p_ij = exp(scale q_i . k_j - lse_i),   i, j rows of one sequence;
//   D_i = dO_i . o_i,  ds_ij = p_ij (dO_i . v_j - D_i),   (o_i to 16 bits of significand: the forward keeps what the
//                                                         rounding to bf16 took off; see below)
//   dQ_i = scale sum_j ds_ij k_j,  dK_j = scale sum_i ds_ij q_i,  dV_j = sum_i p_ij dO_i.
//
// q [M, Hq, D], k and v [M, Hkv, D] are read where they lie (TMA tiles of 128 rows from any row on); a
// tile that reaches past its sequence holds rows of the next one.  Those keys lie behind every
// query of the sequence, so the causal mask hides them, and what they hold never enters a product: score
// and weight are chosen, not multiplied by 0, and rows of an operand that the tensor core would multiply by
// a weight of 0 are cleared in shared memory first.  In the forward's diagonal tiles the infinities and NaN of a
// sequence's own values are taken out too, by the producer warp when it has nothing left to load, and the
// queries that see them get them back at the end: 0.49 ms instead of 0.24 for a sequence of 16384 whose values are all NaN (2 / 1
// heads).  (Computing such rows again one by one, over all of their keys, would take some 0.1 s by count of operations.)
//
// Which rows a CTA has follows from cu_seqlens alone (packed.cuh): no plan, no launch before the kernel, nothing
// kept between calls, and rows outside all sequences get zeros.
//
// Forward: two 128-row tiles a CTA, which share every K / V tile and alternate on the tensor core: while one
// tile's softmax runs, the other's products do.  The tiles are two query heads of one key/value head
// where there are an even number of them (both see the same keys: no tile waits for the other's end, and
// short sequences fill both), else neighbouring rows of one head.
//   warp 0      TMA: Q tiles, then K_0, V_0, K_1, .. through a ring; looks over the last V
//   warp 1      MMA: per step P0 V, S0(next), P1 V, S1(next); P from TMEM, over its own scores
//   warps 2-9   softmax of tile 0 / 1, a row a thread
// The running maximum moves only when it grows by more than 8 (in log2), so outputs are rarely rescaled.
//
// Backward: two kernels and no sum through memory.  One has 128 queries and goes over the keys (dQ, three
// products a tile); one has 128 keys of a key/value head and goes over all queries of its query heads (dK and
// dV, four).  Scores are formed twice, seven products instead of the five of a single pass, but that
// pass would add every dQ tile into 32-bit memory (an accumulator written, added to, read and rounded, in an
// order that changes from run to run).  Here each gradient is a sum in TMEM, in order, and rounded once.
// A sequence's first token sees itself alone: its weight is 1 and its ds 0 whatever the score is, but a weight formed again from a
// rounded lse is off by some 2^-24 of it, and ds with it.  So that ds is chosen to be 0, as masked ones are (what is no number
// stays).  Where all sequences are one token, dQ and dK are zeros, not rounding errors.
// D of the rounded output would be the largest error of short sequences' gradients: 3.4e-3 of their size.  So a forward that
// a backward follows writes the rest of the output too, 2 bytes an entry (2 to 4 % of the forward's
// time): 2.6e-3.  A sequence's first 128 rows, whose weights are all in one tile, take D from those in 32 bits:
// 2.4e-3, of which 1.7e-3 is the rounding of the result.
//
// Measured on a B200, head_dim 128 (counters: profiles/packed_attention.md).  Forward: 16 sequences of 4096 .. 8191 rows, 32 / 8
// heads, 5.2 ms = 0.98 PFLOP/s, power capped (floor 3.1 at the burst rate of a library product, 3.7 at the sustained one);
// a step of two 128 x 128 tiles takes 3700 cycles of which the tensor core's products are 2048: a tile's
// softmax (2150) and its own two products follow one another, and only the other tile's lie under them.  192 documents of
// 340 rows on average, 10 heads: 0.35 ms with what a backward needs (0.34 without), starts and ends of 4200 CTAs.
// Backward: 4 sequences of 4096 .. 8192, 32 / 8 heads, 4.4 ms (dQ 1.9, dK and dV 2.6) = 0.74 PFLOP/s of the formula's five
// products, 1.04 of the seven; the documents 0.95 ms.  With one key/value head dK and dV have few CTAs: one sequence of 4096 rows, 8 / 1
// heads, 0.54 ms where the products would take 0.05 spread evenly.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/ops/clone.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>

#include <atomic>
#include <tuple>
#include <vector>

#include "attention_tiles.cuh"
#include "packed.cuh"

namespace tfb {

CUtensorMap make_tmap_bf16(const void* ptr, uint64_t inner, uint64_t outer, uint64_t row_stride_elems,
                           uint32_t box_inner, uint32_t box_outer, uint64_t batch, uint64_t batch_stride_elems);

constexpr float kPkLowest = -3.4028234663852886e38f;

struct PkArgs {
  Pieces pc;
  int Hq, Hkv, G;
  int by_heads;                  // the forward's two tiles are two heads (else neighbouring rows)
  float scale, scale_log2;
  const __nv_bfloat16 *q, *k, *v, *o, *dout;           // rows and heads, strides in elements
  long long qr, qh, kr, kh, vr, vh, gr, gh;
  __nv_bfloat16 *out, *low, *dq, *dk, *dv;             // [M, H, D]; low: what out's rounding took off, for the gradients
  float *lse, *dvec;             // [Hq, M]
  int* err;
};

// Operand descriptors of a tile, whose address is `d`'s first field (in 16 bytes), at k-step kk: as desc_kmajor and
// desc_mnmajor, but a base that is computed once and constants.  (Computed anew for each product, the
// descriptors took the issuing thread 97 cycles a product; the product takes 64.)
__device__ __forceinline__ uint64_t kmajor_base(const void* tile) { return umma_desc_sw128(smem_u32(tile), 16, 1024); }
__device__ __forceinline__ uint64_t mnmajor_base(const void* tile) { return umma_desc_sw128(smem_u32(tile), kPanel, 1024); }
__device__ __forceinline__ uint64_t kmajor_at(uint64_t d, int kk) { return d + (((uint32_t)(kk >> 2) * kPanel + (uint32_t)(kk & 3) * 32u) >> 4); }
__device__ __forceinline__ uint64_t mnmajor_at(uint64_t d, int kk) { return d + ((uint32_t)kk * 2048u >> 4); }

// D += A B over a tile, A and B by descriptors: 16 dimensions a step
template <int STEPS>
__device__ __forceinline__ void mma_kk(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
#pragma unroll
  for (int kk = 0; kk < STEPS; ++kk) umma_bf16(d, kmajor_at(a, kk), kmajor_at(b, kk), idesc, kk > 0 ? 1u : 0u);
}
// D (+)= A B, A the weights of 128 columns in TMEM, packed: 16 of them a step, those of every 32 columns GAP behind the
// ones before
template <int GAP>
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
#pragma unroll
  for (int kk = 0; kk < 8; ++kk)
    umma_bf16_tmem_a(d, a + (kk >> 1) * GAP + (kk & 1) * 8, mnmajor_at(b, kk), idesc, kk > 0 ? 1u : add ? 1u : 0u);
}

// Of 8 bf16: which are infinities or NaN (all bits of their halves, else none).
__device__ __forceinline__ uint4 not_finite8(const uint4& u) {
  auto of = [](uint32_t w) { return __vcmpeq2(w & 0x7f807f80u, 0x7f807f80u); };
  return make_uint4(of(u.x), of(u.y), of(u.z), of(u.w));
}
// Row `row` of a tile of D columns (swizzled panels of 64): whether it holds an infinity or a NaN.
template <int D>
__device__ __forceinline__ bool tile_row_bad(const uint8_t* tile, int row) {
  uint32_t bad = 0;
#pragma unroll
  for (int c = 0; c < D / 8; ++c) {
    const uint4 u = *reinterpret_cast<const uint4*>(tile + (c >> 3) * kPanel + sw128_chunk_offset(row, c & 7));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w;
      bad |= ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
    }
  }
  return bad != 0;
}
// Zeros in their places.  (In line: as a function of its own the forward of 16 x 8191 rows took 4 % longer, for want of registers.)
template <int D>
__device__ __forceinline__ void tile_row_mend(uint8_t* tile, int row) {
#pragma unroll 1
  for (int c = 0; c < D / 8; ++c) {
    uint4* at = reinterpret_cast<uint4*>(tile + (c >> 3) * kPanel + sw128_chunk_offset(row, c & 7));
    const uint4 u = *at, m = not_finite8(u);
    *at = make_uint4(u.x & ~m.x, u.y & ~m.y, u.z & ~m.z, u.w & ~m.w);
  }
}
template <int D>
__device__ __forceinline__ void tile_row_clear(uint8_t* tile, int row) {
#pragma unroll
  for (int c = 0; c < D / 8; ++c)
    *reinterpret_cast<uint4*>(tile + (c >> 3) * kPanel + sw128_chunk_offset(row, c & 7)) = make_uint4(0, 0, 0, 0);
}

// One arrival for a warp, once all its lanes have come here: an mbarrier takes the arrivals of 32 lanes one after
// another (dQ of 4 x 8192 rows took 2.3 instead of 1.8 ms with 512 of them a barrier).
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// Zeros into rows [row0, row0 + n) x heads of out [M, H, D] (rows outside all sequences).
template <int D>
__device__ __forceinline__ void clear_rows(__nv_bfloat16* out, int H, int h0, int heads, long long row0, int n) {
  for (int i = threadIdx.x; i < n * heads * (D / 8); i += blockDim.x) {
    const int c = i % (D / 8), h = i / (D / 8) % heads, r = i / (D / 8) / heads;
    reinterpret_cast<uint4*>(out + ((row0 + r) * H + h0 + h) * D)[c] = make_uint4(0, 0, 0, 0);
  }
}

// A warp's 32 rows of 16-byte CHUNKS, from TMEM columns at `from` on, each row times its lane's `by`, rounded and stored
// through `stage`, PASS chunks of all rows at a time, so that a store covers whole pieces of rows (shared memory of the
// warp's own, 16-byte aligned, 512 x PASS bytes, and as many again with `low`).  dst: the first row's, `stride` elements between
// rows; low (or null): what the rounding took off them, rounded, likewise; n: rows that are there.
// (Rows stored by their own lanes took 4500 of a one-tile CTA's 15000 cycles.)
template <int CHUNKS, int PASS>
__device__ __forceinline__ void store_rows(uint32_t from, float by, uint8_t* stage, __nv_bfloat16* dst, __nv_bfloat16* low, long long stride, int n) {
  static_assert(CHUNKS % PASS == 0 && PASS % 2 == 0, "chunks");
  const int lane = threadIdx.x & 31;
  auto place = [](int row, int c) { return row * (16 * PASS) + ((c ^ (row & (PASS - 1) & 7)) << 4); };
#pragma unroll
  for (int c0 = 0; c0 < CHUNKS; c0 += PASS) {
#pragma unroll
    for (int c = 0; c < PASS; c += 2) {
      uint32_t o[16];
      __syncwarp();
      tmem_ld_32x32b_x16(from + (c0 + c) * 8, o);
      tmem_ld_wait();
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t w[4], v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = __uint_as_float(o[8 * k + 2 * i]) * by, y = __uint_as_float(o[8 * k + 2 * i + 1]) * by;
          w[i] = pack_bf16x2(x, y);
          v[i] = pack_bf16x2(x - __uint_as_float(w[i] << 16), y - __uint_as_float(w[i] & 0xffff0000u));
        }
        *reinterpret_cast<uint4*>(stage + place(lane, c + k)) = make_uint4(w[0], w[1], w[2], w[3]);
        if (low) *reinterpret_cast<uint4*>(stage + 512 * PASS + place(lane, c + k)) = make_uint4(v[0], v[1], v[2], v[3]);
      }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < PASS; ++i) {
      const int row = (i * 32 + lane) / PASS, c = (i * 32 + lane) % PASS;
      if (row < n) {
        reinterpret_cast<uint4*>(dst + row * stride)[c0 + c] = *reinterpret_cast<const uint4*>(stage + place(row, c));
        if (low) reinterpret_cast<uint4*>(low + row * stride)[c0 + c] = *reinterpret_cast<const uint4*>(stage + 512 * PASS + place(row, c));
      }
    }
    __syncwarp();
  }
}

// Infinities and NaN of values were taken out of the tile of V before its product; a query row (a lane each, whose output of D
// columns is at `out` in TMEM) gets those of the rows that it sees, j <= seen of the tile.  `rows`: a bit for each of them;
// v: the tile's first row.  All of them NaN: 128 rows of loads that the warp shares.
template <int D>
__device__ __noinline__ void add_not_finite(uint32_t out, const uint32_t* rows, const __nv_bfloat16* v, long long vr, int seen) {
  if (!(rows[0] | rows[1] | rows[2] | rows[3])) return;
#pragma unroll 1
  for (int d0 = 0; d0 < D; d0 += 32) {
    uint32_t o[32];
    __syncwarp();
    tmem_ld_32x32b_x32(out + d0, o);
    tmem_ld_wait();
#pragma unroll 1
    for (int w = 0; w < 4; ++w) {
#pragma unroll 1
      for (uint32_t left = rows[w]; left; left &= left - 1) {
        const int j = w * 32 + __ffs(left) - 1;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint4 u = *reinterpret_cast<const uint4*>(v + j * vr + d0 + 8 * c), m = not_finite8(u);
          const uint32_t x[4] = {u.x & m.x, u.y & m.y, u.z & m.z, u.w & m.w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (j <= seen) {
              o[8 * c + 2 * i] = __float_as_uint(__uint_as_float(o[8 * c + 2 * i]) + __uint_as_float(x[i] << 16));
              o[8 * c + 2 * i + 1] = __float_as_uint(__uint_as_float(o[8 * c + 2 * i + 1]) + __uint_as_float(x[i] & 0xffff0000u));
            }
        }
      }
    }
    __syncwarp();
    tmem_st_32x32b_x32(out + d0, o);
    tmem_st_wait();
  }
}

// The same for tile t of a CTA of the forward, `out` being the warp's lanes of it.  All is found again from the unit, so that the
// loop over the keys keeps no registers for it.
template <int D, int TILES>
__device__ __noinline__ void give_back(uint32_t out, const uint32_t* bad, int t, const PieceUnit& un, int by_heads, int Hq, int G,
                                       const __nv_bfloat16* v, long long vr, long long vh) {
  const bool pair = TILES == 2 && by_heads;
  const int nh = pair ? Hq / 2 : Hq, hk = (int)(blockIdx.x % nh) * (pair ? 2 : 1) / G;
  const int r = (threadIdx.x >> 5 & 3) * 32 + (threadIdx.x & 31), r0 = un.unit * (TILES == 1 || pair ? 128 : 256);
  const __nv_bfloat16* first = v + (long long)(un.begin + r0) * vr + hk * vh;
  if (pair || t == 0) {
    add_not_finite<D>(out, bad + 4 * t, first, vr, r);
  } else {                               // of neighbouring tiles the second sees all rows of the first one's last V
    add_not_finite<D>(out, bad, first, vr, 127);
    add_not_finite<D>(out, bad + 4, first + 128 * vr, vr, r);
  }
}

template <int D, int TILES>
struct PkFwd {
  static constexpr uint32_t TILE = 128u * D * 2u;
  static constexpr int NS = TILES == 1 ? (D == 128 ? 2 : 4) : D == 128 ? 5 : 8;   // K / V ring
  static constexpr size_t SMEM = 1024 + (TILES + NS) * TILE + 32 * 8 + 64;
  static constexpr int THREADS = 64 + 128 * TILES;
  static constexpr uint32_t COLUMNS = 256 * TILES;     // of TMEM: S and O of each tile
};
static_assert(2 * PkFwd<128, 1>::SMEM <= 227 * 1024 && PkFwd<128, 2>::SMEM <= 227 * 1024, "shared memory");
// The producer looks over the last V of each tile when all loads are issued, so none of them may wait for a product with it:
// the last load waits for the slot NS items before, and behind tile 0's last V come at most two items.
static_assert(PkFwd<128, 1>::NS >= 2 && PkFwd<64, 1>::NS >= 2 && PkFwd<128, 2>::NS >= 4 && PkFwd<64, 2>::NS >= 4, "K / V ring");

template <int D, int TILES>
__global__ void __launch_bounds__(64 + 128 * TILES, 3 - TILES)
    packed_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const PkArgs a) {
  using Cfg = PkFwd<D, TILES>;
  constexpr uint32_t TILE = Cfg::TILE;
  constexpr int NS = Cfg::NS, PANELS = D / 64;
  constexpr uint32_t IDESC_S = umma_idesc_bf16(128, 128, false, false);
  constexpr uint32_t IDESC_O = umma_idesc_bf16(128, D, false, true);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                 // [TILES]
  uint8_t* sKV = sQ + TILES * TILE;       // [NS] slots
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + NS * TILE);
  uint64_t* bar_q = bars + 0;
  uint64_t* kv_full = bars + 1;          // [NS]
  uint64_t* kv_empty = bars + 1 + NS;    // [NS]
  uint64_t* s_full = bars + 1 + 2 * NS;  // [2]
  uint64_t* p_full = s_full + 2;         // [2]
  uint64_t* o_done = p_full + 2;         // [2]
  uint64_t* looked = o_done + 2;         // [2] the tile's last V holds finite numbers alone, bad_rows says whether it did before
  uint64_t* drain = looked + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  PieceUnit* s_unit = reinterpret_cast<PieceUnit*>(tmem_slot + 4);
  uint32_t* bad_rows = tmem_slot + 8;    // [2][4] the rows of the tiles' last V that held an infinity or a NaN, a bit each
  volatile uint32_t* any_bad = tmem_slot + 2;          // whether one of them did

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nh = TILES == 2 && a.by_heads ? a.Hq / 2 : a.Hq;
  const int hx = (int)(blockIdx.x % nh);
  const int slot_id = (int)(gridDim.x / nh - 1 - blockIdx.x / nh);   // a sequence's last rows have the most keys: first
  if (warp == 0) {
    const PieceUnit u = TILES == 1 || a.by_heads ? piece_unit<128>(a.pc, slot_id) : piece_unit<256>(a.pc, slot_id);
    if (lane == 0) *s_unit = u;
  } else if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::COLUMNS);
    tmem_relinquish();
  } else if (threadIdx.x == 64) {
    mbar_init(bar_q, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_done[t], 1);
      mbar_init(&looked[t], 1);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    *any_bad = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = TILES == 2 ? 0 : *tmem_slot;   // all 512 columns start at 0
  if (TILES == 2 && threadIdx.x == 0 && *tmem_slot != tmem) atomicOr(a.err, ERR_BAD_ARG);
  constexpr uint32_t OAT = 128 * TILES;                // outputs behind the scores
  const PieceUnit un = *s_unit;
  const bool pair = TILES == 2 && a.by_heads;
  const int U = TILES == 1 || pair ? 128 : 256;
  const bool live = un.unit >= 0 && a.pc.real(un.piece);
  // tile t: its head, first row in the sequence, and number of K / V tiles (0: there is none)
  const int h0 = pair ? 2 * hx : hx, h1 = pair ? h0 + 1 : hx;
  const int r0 = un.unit * U, r1 = pair ? r0 : r0 + 128;
  const int n0 = live ? r0 / 128 + 1 : 0, n1 = TILES == 2 && live && r1 < un.len ? r1 / 128 + 1 : 0;
  const int nk = max(n0, n1);
  const int hk = h0 / a.G;

  if (!live) {
    if (un.unit >= 0) clear_rows<D>(a.out, a.Hq, h0, pair ? 2 : 1, un.begin + r0, min(U, un.len - r0));
  } else if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    bool ok = true;
    if (lane == 0) {
      uint32_t out_valid = 0, out_parity = 0;
      mbar_arrive_expect_tx(bar_q, (n1 ? 2 : 1) * TILE);
#pragma unroll
      for (int p = 0; p < PANELS; ++p) {
        tma_load_3d(sQ + p * kPanel, &tmQ, bar_q, p * 64, un.begin + r0, h0);
        if (n1) tma_load_3d(sQ + TILE + p * kPanel, &tmQ, bar_q, p * 64, un.begin + r1, h1);
      }
      const int items = 2 * nk;
      for (int i = 0; i < items && ok; ++i) {
        const int slot = i % NS;
        if (i >= NS && !mbar_wait(&kv_empty[slot], ((i / NS) + 1) & 1, abort_flag, a.err, ERR_TIMEOUT_PRODUCER)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&kv_full[slot], TILE);
        out_valid |= 1u << slot;
        out_parity = (out_parity & ~(1u << slot)) | ((uint32_t)((i / NS) & 1) << slot);
        const int krow = un.begin + (i >> 1) * 128;
        const CUtensorMap* map = (i & 1) ? &tmV : &tmK;
#pragma unroll
        for (int p = 0; p < PANELS; ++p) tma_load_3d(sKV + slot * TILE + p * kPanel, map, &kv_full[slot], p * 64, krow, hk);
      }
      if (!ok) {
        for (int s = 0; s < NS; ++s) {
          if (!((out_valid >> s) & 1u)) continue;
          const unsigned long long t0 = globaltimer_ns();
          while (!mbar_try_wait(&kv_full[s], (out_parity >> s) & 1u))
            if (globaltimer_ns() - t0 > 100000000ull) break;
        }
        const unsigned long long t0 = globaltimer_ns();
        while (!mbar_try_wait(bar_q, 0))
          if (globaltimer_ns() - t0 > 100000000ull) break;
      }
    }
    // The last V of a tile has rows that some of its queries do not see, but the tensor core multiplies by their weights of 0: no
    // infinity or NaN may be among them.  They are looked over and taken out under the tile's softmax; who sees them gets them back
    // at the end.
    ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    for (int t = 0; t < TILES && ok; ++t) {
      const int j = (t == 0 ? n0 : n1) - 1, i = 2 * j + 1;
      if (j < 0) break;
      if (pair && t == 1) {              // the same V
        __syncwarp();
        if (lane < 4) bad_rows[4 + lane] = bad_rows[lane];
        warp_arrive(&looked[1]);
        break;
      }
      ok = mbar_wait_warp(&kv_full[i % NS], (i / NS) & 1, abort_flag, a.err, ERR_TIMEOUT_PRODUCER);
      if (!ok) break;
      uint8_t* tile = sKV + (i % NS) * TILE;
      bool any = false;
#pragma unroll 1
      for (int w = 0; w < 4; ++w) {
        const int r = w * 32 + lane;
        const bool bad = j * 128 + r < un.len && tile_row_bad<D>(tile, r);
        if (bad) tile_row_mend<D>(tile, r);
        any |= bad;
        const uint32_t rows = __ballot_sync(0xffffffffu, bad);
        if (lane == 0) {
          bad_rows[4 * t + w] = rows;
          if (rows) *any_bad = 1;
        }
      }
      if (any) fence_proxy_async_smem();
      warp_arrive(&looked[t]);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    // The warp runs as one, so that operands stay in uniform registers; one lane issues.
    bool ok = mbar_wait_warp(bar_q, 0, abort_flag, a.err, ERR_TIMEOUT_MMA);
    const bool leader = elect_one();
    const uint64_t qd[2] = {kmajor_base(sQ), kmajor_base(sQ + TILE)};
    const uint64_t kd = kmajor_base(sKV), vd = mnmajor_base(sKV);
    constexpr uint64_t STEP = TILE >> 4;
    // slots and parities of the K / V tiles: S takes K_j, the products after it V_j
    int ks = 0, vs = 1;
    uint32_t kp = 0, vp = 0;
    auto issue_s = [&](int t) {
      tc_fence_after();
      if (leader) {
        mma_kk<D / 16>(tmem + t * 128, qd[t], kd + ks * STEP, IDESC_S);
        umma_commit(&s_full[t]);
      }
      __syncwarp();
    };
    auto issue_pv = [&](int t, int j) -> bool {
      if (j == (t == 0 ? n0 : n1) - 1 && !mbar_wait_warp(&looked[t], 0, abort_flag, a.err, ERR_TIMEOUT_MMA)) return false;
      if (!mbar_wait_warp(&p_full[t], j & 1, abort_flag, a.err, ERR_TIMEOUT_MMA)) return false;
      tc_fence_after();
      if (leader) mma_tmem<16>(tmem + OAT + t * 128, tmem + t * 128, vd + vs * STEP, IDESC_O, j > 0);
      __syncwarp();
      return true;
    };
    auto commit = [&](uint64_t* bar) {
      if (leader) umma_commit(bar);
      __syncwarp();
    };
    if (ok) ok = mbar_wait_warp(&kv_full[0], 0, abort_flag, a.err, ERR_TIMEOUT_MMA);
    if (ok) {
      issue_s(0);
      if (n1) issue_s(1);
      commit(&kv_empty[0]);              // K_0 read by both tiles
    }
    for (int j = 0; j < nk && ok; ++j) {
      // one thread's tcgen05 MMAs run in issue order: S_t(j + 1) may overwrite P_t(j)
      const bool more = j + 1 < nk;
      if (more) {
        ks += 2;
        if (ks >= NS) { ks -= NS; kp ^= 1; }
      }
      if (!mbar_wait_warp(&kv_full[vs], vp, abort_flag, a.err, ERR_TIMEOUT_MMA)) { ok = false; break; }
      if (j < n0) {
        if (!issue_pv(0, j)) { ok = false; break; }
        if (j + 1 < n0) {
          if (!mbar_wait_warp(&kv_full[ks], kp, abort_flag, a.err, ERR_TIMEOUT_MMA)) { ok = false; break; }
          issue_s(0);
        } else {
          commit(&o_done[0]);
        }
      }
      if (j < n1) {
        if (!issue_pv(1, j)) { ok = false; break; }
        if (j + 1 < n1) {
          if (!mbar_wait_warp(&kv_full[ks], kp, abort_flag, a.err, ERR_TIMEOUT_MMA)) { ok = false; break; }
          issue_s(1);
        } else {
          commit(&o_done[1]);
        }
      }
      if (more) commit(&kv_empty[ks]);   // K_{j+1} read by both tiles
      commit(&kv_empty[vs]);             // V_j done
      vs += 2;
      if (vs >= NS) { vs -= NS; vp ^= 1; }
    }
    if (!ok) {
      *abort_flag = 1;
      commit(drain);
      const unsigned long long t0 = globaltimer_ns();
      while (!mbar_try_wait(drain, 0))
        if (globaltimer_ns() - t0 > 100000000ull) break;
    }
  } else {
    // ------------------------------------------------------------------ softmax (tile t)
    const int t = (warp - 2) >> 2;
    const int q4 = warp & 3;
    const int r = q4 * 32 + lane;
    const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
    const uint32_t tS = tmem + t * 128, tO = tmem + OAT + t * 128;
    const int n_t = t == 0 ? n0 : n1;
    const int row = (t == 0 ? r0 : r1) + r, head = t == 0 ? h0 : h1;   // row of the sequence
    const float c = a.scale_log2;
    float m_run = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n_t; ++j) {
      if (!mbar_wait_warp(&s_full[t], j & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) { ok = false; break; }
      tc_fence_after();
      float x[128];
      {
        uint32_t* xr = reinterpret_cast<uint32_t*>(x);
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          __syncwarp();
          tmem_ld_32x32b_x32(tS + lane_off + cc * 32, *reinterpret_cast<uint32_t(*)[32]>(xr + 32 * cc));
        }
        tmem_ld_wait();
      }
      const bool diag = j == n_t - 1;
      if (diag) {  // keys after this query row are masked, those past the sequence among them
#pragma unroll
        for (int cc = 0; cc < 4; ++cc)
          if (cc >= q4)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (cc * 32 + i > r) x[cc * 32 + i] = -INFINITY;
        // rows of V past the sequence (another's) are cleared
        if (j * 128 + r >= un.len) {
          mbar_wait(&kv_full[(2 * j + 1) % NS], ((2 * j + 1) / NS) & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE);
          tile_row_clear<D>(sKV + ((2 * j + 1) % NS) * TILE, r);
          fence_proxy_async_smem();
        }
        __syncwarp();
      }
      // four independent max chains, two new elements per three-input max
      float mx4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
      for (int i = 4; i < 128; i += 8)
#pragma unroll
        for (int k = 0; k < 4; ++k) mx4[k] = max3_nan(mx4[k], x[i + k], x[i + 4 + k]);
      // visible scores of -inf count as the lowest number, so that their weights are 0
      float mxs = max_nan(max_nan(max_nan(mx4[0], mx4[1]), max_nan(mx4[2], mx4[3])) * c, kPkLowest);
      if (mxs == INFINITY) mxs = NAN;            // inf - inf
      float alpha = 1.f;
      const bool grow = !(mxs <= m_run + 8.f);   // true for a NaN, which then stays
      if (grow) {
        alpha = ex2_approx(m_run - mxs);
        m_run = mxs;
      }
      // p = 2^(x c - m): packed pairs
      const float2 c2 = make_float2(c, c), nm2 = make_float2(-m_run, -m_run);
      float2 sm4[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      uint32_t pk[64];  // the row of P as packed bf16 pairs
#pragma unroll
      for (int i = 0; i < 128; i += 2) {
        const float2 v = __ffma2_rn(make_float2(x[i], x[i + 1]), c2, nm2);
        // a quarter on the FMA pipe, which the MUFU unit's 16 a cycle of an SM leave idle (5.6 ms without, for 16 x 8191 rows).  A
        // NaN is lost there, but then the row's maximum is NaN and with it all of its other weights.
        float2 p2;
        if (i >= 96) p2 = exp2_poly2(v);
        else p2 = make_float2(ex2_approx(v.x), ex2_approx(v.y));
        pk[i >> 1] = pack_bf16x2(p2.x, p2.y);
        sm4[(i >> 1) & 3] = __fadd2_rn(sm4[(i >> 1) & 3], p2);
      }
      const float2 s01 = __fadd2_rn(__fadd2_rn(sm4[0], sm4[1]), __fadd2_rn(sm4[2], sm4[3]));
      l = l * alpha + (s01.x + s01.y);
      // O_t is stable: the commit that signalled S_t(j) covered P_t(j-1) V_{j-1}
      if (j >= 1 && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
        for (int cc = 0; cc < D / 32; ++cc) {
          uint32_t o[32];
          __syncwarp();
          tmem_ld_32x32b_x32(tO + lane_off + cc * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st_32x32b_x32(tO + lane_off + cc * 32, o);
        }
      }
      // P_t(j) over the first 64 columns of S_t(j) (already in registers)
      __syncwarp();
      tmem_st_32x32b_x32(tS + lane_off, *reinterpret_cast<const uint32_t(*)[32]>(pk));
      tmem_st_32x32b_x32(tS + lane_off + 32, *reinterpret_cast<const uint32_t(*)[32]>(pk + 32));
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&p_full[t]);
    }
    if (n_t > 0 && ok && mbar_wait_warp(&o_done[t], 0, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE) &&
        mbar_wait_warp(&looked[t], 0, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) {
      tc_fence_after();
      const bool mine = row < un.len;
      const int first = row - lane;      // the warp's first row; Q's tile is free: all products of it are done
      // no weight at all (every visible score is -inf): NaN, an infinity of v's among them
      const float inv_l = l == 0.f ? NAN : 1.f / l, lse2 = m_run + log2f(l);
      if (*any_bad) give_back<D, TILES>(tO + lane_off, bad_rows, t, *s_unit, a.by_heads, a.Hq, a.G, a.v, a.vr, a.vh);
      __nv_bfloat16* dst = a.out + ((long long)(un.begin + first) * a.Hq + head) * D;
      store_rows<D / 8, D / 16>(tO + lane_off, inv_l, sQ + t * TILE + q4 * (32 * D * 2), dst, a.low ? a.low + (dst - a.out) : nullptr,
                                (long long)a.Hq * D, un.len - first);
      if (mine && a.lse) a.lse[(long long)head * a.pc.M + un.begin + row] = lse2 * kLn2;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::COLUMNS);
  }
}

// ================================================================================ backward: dQ
// One CTA per 128 queries of a head, over the keys.  TMEM: S | dP | dQ | two dS (bf16).
//   warp 0      TMA: Q and dO, then K_0, V_0, K_1, .. through a ring each
//   warp 1      MMA: S(next) = Q K^T, dP(next) = dO V^T
//   warp 18     MMA: dQ += dS K with dS from TMEM (by itself, so that it waits for nothing but dS)
//   warps 2-17  p = 2^(S c - lse), dS = p (dP - D): four warps a lane quarter, 32 columns each
// S and dP are given back as soon as they are in registers, so the next ones are formed meanwhile.
template <int D>
struct PkDq {
  static constexpr uint32_t TILE = 128u * D * 2u;
  static constexpr int NK = D == 128 ? 3 : 5, NV = D == 128 ? 2 : 4, NS = NK + NV;   // rings of K (held until dQ has read it) and V
  static constexpr size_t SMEM = 1024 + (2 + NS) * TILE + 512 + 32 * 8 + 64;
};

template <int D>
__global__ void __launch_bounds__(608, 1)
    packed_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmG, const PkArgs a) {
  constexpr uint32_t TILE = PkDq<D>::TILE;
  constexpr int NK = PkDq<D>::NK, NS = PkDq<D>::NS, PANELS = D / 64;
  constexpr uint32_t IDESC_S = umma_idesc_bf16(128, 128, false, false);
  constexpr uint32_t IDESC_Q = umma_idesc_bf16(128, D, false, true);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sG = sQ + TILE;
  uint8_t* sKV = sG + TILE;
  float* sD = reinterpret_cast<float*>(sKV + NS * TILE);   // [128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sD + 128);
  uint64_t* bar_q = bars + 0;
  uint64_t* kv_full = bars + 1;          // [NK + NV]
  uint64_t* kv_empty = bars + 1 + NS;    // [NK + NV]
  uint64_t* s_full = bars + 1 + 2 * NS;
  uint64_t* s_free = s_full + 1;
  uint64_t* dp_full = s_full + 2;
  uint64_t* dp_free = s_full + 3;
  uint64_t* ds_full = s_full + 4;      // [2]: the compute warps may be a tile ahead of dQ
  uint64_t* ds_free = s_full + 6;      // [2]
  uint64_t* done = s_full + 8;
  uint64_t* drain = s_full + 9;        // [2]
  uint64_t* part_full = s_full + 11;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(part_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  PieceUnit* s_unit = reinterpret_cast<PieceUnit*>(tmem_slot + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = (int)(blockIdx.x % a.Hq), hk = h / a.G;
  if (warp == 0) {
    const PieceUnit u = piece_unit<128>(a.pc, (int)(gridDim.x / a.Hq - 1 - blockIdx.x / a.Hq));
    if (lane == 0) *s_unit = u;
  } else if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  } else if (threadIdx.x == 64) {
    mbar_init(bar_q, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_free, 16);
    mbar_init(dp_full, 1);
    mbar_init(dp_free, 16);
    mbar_init(&ds_full[0], 16);
    mbar_init(&ds_full[1], 16);
    mbar_init(&ds_free[0], 1);
    mbar_init(&ds_free[1], 1);
    mbar_init(done, 1);
    mbar_init(part_full, 16);
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmG);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;           // all 512 columns are this CTA's: they start at 0
  if (threadIdx.x == 0 && *tmem_slot != tmem) atomicOr(a.err, ERR_BAD_ARG);
  const uint32_t tS = tmem, tP = tmem + 128, tQ = tmem + 256, tD = tmem + 384;
  const PieceUnit un = *s_unit;
  const int row0 = un.unit * 128, n = un.unit + 1;

  if (un.unit < 0 || !a.pc.real(un.piece)) {
    if (un.unit >= 0) clear_rows<D>(a.dq, a.Hq, h, 1, un.begin + row0, min(128, un.len - row0));
  } else if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      uint32_t out_valid = 0, out_parity = 0;
      mbar_arrive_expect_tx(bar_q, 2 * TILE);
#pragma unroll
      for (int p = 0; p < PANELS; ++p) {
        tma_load_3d(sQ + p * kPanel, &tmQ, bar_q, p * 64, un.begin + row0, h);
        tma_load_3d(sG + p * kPanel, &tmG, bar_q, p * 64, un.begin + row0, h);
      }
      int slot[2] = {0, NK};             // K's and V's next
      uint32_t lap[2] = {0, 0};          // times round
      for (int i = 0; i < 2 * n && ok; ++i) {
        const int w = i & 1, sl = w ? slot[1] : slot[0];
        const uint32_t r = w ? lap[1] : lap[0];
        if (r > 0 && !mbar_wait(&kv_empty[sl], (r - 1) & 1, abort_flag, a.err, ERR_TIMEOUT_PRODUCER)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&kv_full[sl], TILE);
        out_valid |= 1u << sl;
        out_parity = (out_parity & ~(1u << sl)) | ((r & 1) << sl);
        const CUtensorMap* map = w ? &tmV : &tmK;
#pragma unroll
        for (int p = 0; p < PANELS; ++p)
          tma_load_3d(sKV + sl * TILE + p * kPanel, map, &kv_full[sl], p * 64, un.begin + (i >> 1) * 128, hk);
        if (w) { if (++slot[1] == NS) { slot[1] = NK; ++lap[1]; } }
        else if (++slot[0] == NK) { slot[0] = 0; ++lap[0]; }
      }
      if (!ok) {
        for (int s = 0; s < NS; ++s) {
          if (!((out_valid >> s) & 1u)) continue;
          const unsigned long long t0 = globaltimer_ns();
          while (!mbar_try_wait(&kv_full[s], (out_parity >> s) & 1u))
            if (globaltimer_ns() - t0 > 100000000ull) break;
        }
        const unsigned long long t0 = globaltimer_ns();
        while (!mbar_try_wait(bar_q, 0))
          if (globaltimer_ns() - t0 > 100000000ull) break;
      }
    }
  } else if (warp == 1) {
    bool ok = mbar_wait_warp(bar_q, 0, abort_flag, a.err, ERR_TIMEOUT_MMA);
    const bool leader = elect_one();
    const uint64_t qd = kmajor_base(sQ), gd = kmajor_base(sG), kd = kmajor_base(sKV);
    constexpr uint64_t STEP = TILE >> 4;
    int ks = 0, vs = NK;                 // slots of the next K and V
    uint32_t kp = 0, vp = 0;
    auto commit = [&](uint64_t* bar) {
      if (leader) umma_commit(bar);
      __syncwarp();
    };
    // S(j) = Q K_j^T, dP(j) = dO V_j^T, once the compute warps have the tiles before in registers
    auto issue_s = [&](int j) -> bool {
      if (!mbar_wait_warp(&kv_full[ks], kp, abort_flag, a.err, ERR_TIMEOUT_MMA)) return false;
      if (j >= 1 && !mbar_wait_warp(s_free, (j - 1) & 1, abort_flag, a.err, ERR_TIMEOUT_MMA)) return false;
      tc_fence_after();
      if (leader) {
        mma_kk<D / 16>(tS, qd, kd + ks * STEP, IDESC_S);
        umma_commit(s_full);
      }
      __syncwarp();
      if (++ks == NK) { ks = 0; kp ^= 1; }
      return true;
    };
    auto issue_dp = [&](int j) -> bool {
      if (!mbar_wait_warp(&kv_full[vs], vp, abort_flag, a.err, ERR_TIMEOUT_MMA)) return false;
      if (j >= 1 && !mbar_wait_warp(dp_free, (j - 1) & 1, abort_flag, a.err, ERR_TIMEOUT_MMA)) return false;
      tc_fence_after();
      if (leader) {
        mma_kk<D / 16>(tP, gd, kd + vs * STEP, IDESC_S);
        umma_commit(dp_full);
        umma_commit(&kv_empty[vs]);
      }
      __syncwarp();
      if (++vs == NS) { vs = NK; vp ^= 1; }
      return true;
    };
    for (int j = 0; j < n && ok; ++j) ok = issue_s(j) && issue_dp(j);
    if (!ok) {
      *abort_flag = 1;
      commit(&drain[0]);
      const unsigned long long t0 = globaltimer_ns();
      while (!mbar_try_wait(&drain[0], 0))
        if (globaltimer_ns() - t0 > 100000000ull) break;
    }
  } else if (warp == 18) {
    const bool leader = elect_one();
    const uint64_t kn = mnmajor_base(sKV);
    constexpr uint64_t STEP = TILE >> 4;
    int kq = 0;                          // slot of K_j
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      if (!mbar_wait_warp(&ds_full[j & 1], (j >> 1) & 1, abort_flag, a.err, ERR_TIMEOUT_MMA)) { ok = false; break; }
      tc_fence_after();
      if (leader) {
        mma_tmem<16>(tQ, tD + (j & 1) * 64, kn + kq * STEP, IDESC_Q, j > 0);
        umma_commit(&kv_empty[kq]);
        umma_commit(&ds_free[j & 1]);
        if (j == n - 1) umma_commit(done);
      }
      __syncwarp();
      if (++kq == NK) kq = 0;
    }
    if (!ok) {
      *abort_flag = 1;
      if (leader) umma_commit(&drain[1]);
      __syncwarp();
      const unsigned long long t0 = globaltimer_ns();
      while (!mbar_try_wait(&drain[1], 0))
        if (globaltimer_ns() - t0 > 100000000ull) break;
    }
  } else {
    const int q4 = warp & 3, quarter = (warp - 2) >> 2, cb = quarter * 32;
    const int r = q4 * 32 + lane, row = row0 + r;
    const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
    const bool mine = row < un.len;
    const bool first = row == 0 && quarter == 0;         // holds the ds that is 0 by definition
    const long long at = (long long)h * a.pc.M + un.begin + row;
    // D_i = dO_i . o_i, kept for the other kernel: eight rows a warp, 16-byte loads of whole rows.  (A row a thread took 9000
    // cycles, longer than three tiles of keys.)  A sequence's first 128 rows take it from their one tile of weights, below.
    if (n > 1) {
      constexpr int L = D / 8;           // lanes a row
      const int w8 = (warp - 2) * 8;
      uint4 x[8 * L / 32], y[8 * L / 32], z[8 * L / 32];
#pragma unroll
      for (int i = 0; i < 8 * L / 32; ++i) {
        const int rr = row0 + w8 + i * (32 / L) + lane / L;
        x[i] = y[i] = z[i] = make_uint4(0, 0, 0, 0);
        if (rr < un.len) {
          x[i] = reinterpret_cast<const uint4*>(a.dout + (long long)(un.begin + rr) * a.gr + h * a.gh)[lane % L];
          const long long at = ((long long)(un.begin + rr) * a.Hq + h) * D;
          y[i] = reinterpret_cast<const uint4*>(a.o + at)[lane % L];
          z[i] = reinterpret_cast<const uint4*>(a.low + at)[lane % L];
        }
      }
#pragma unroll
      for (int i = 0; i < 8 * L / 32; ++i) {
        const uint32_t xw[4] = {x[i].x, x[i].y, x[i].z, x[i].w}, yw[4] = {y[i].x, y[i].y, y[i].z, y[i].w}, zw[4] = {z[i].x, z[i].y, z[i].z, z[i].w};
        float d = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          d += __uint_as_float(xw[w] << 16) * (__uint_as_float(yw[w] << 16) + __uint_as_float(zw[w] << 16));
          d += __uint_as_float(xw[w] & 0xffff0000u) * (__uint_as_float(yw[w] & 0xffff0000u) + __uint_as_float(zw[w] & 0xffff0000u));
        }
#pragma unroll
        for (int k = L / 2; k > 0; k >>= 1) d += __shfl_xor_sync(0xffffffffu, d, k);
        if (lane % L == 0) sD[w8 + i * (32 / L) + lane / L] = d;
      }
      named_bar_sync(1, 512);            // no wait comes before it: all 512 threads arrive
    }
    const float nlse = mine ? -a.lse[at] * kLog2e : -INFINITY;
    const float2 c2 = make_float2(a.scale_log2, a.scale_log2), nl2 = make_float2(nlse, nlse);
    bool ok = true;
    float dsum = 0.f;
    if (n > 1) {
      dsum = sD[r];
    } else {
      // D_i = sum of p dP over the row, of 32-bit weights: those that o was summed with are rounded, which is as much as
      // the rounding of ds where a row has few keys (gradients of sequences of 20 rows off by 2.4e-3 instead of 2.6e-3 of their
      // size).  dO's tile is free: its product is done.  (Within the loop below long sequences' dQ took 6 % longer.)
      float* part = reinterpret_cast<float*>(sG);        // [4][128]
      ok = mbar_wait_warp(s_full, 0, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE) && mbar_wait_warp(dp_full, 0, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE);
      if (ok) {
        tc_fence_after();
#pragma unroll 1
        for (int c = cb; c < cb + 32; c += 16) {
          uint32_t x[16], y[16];
          __syncwarp();
          tmem_ld_32x32b_x16(tS + lane_off + c, x);
          tmem_ld_32x32b_x16(tP + lane_off + c, y);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float w = ex2_approx(fmaf(__uint_as_float(x[e]), a.scale_log2, nlse));
            if (c + e <= r) dsum = fmaf(w, __uint_as_float(y[e]), dsum);
          }
        }
        part[quarter * 128 + r] = dsum;
        warp_arrive(part_full);
        ok = mbar_wait_warp(part_full, 0, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE);
        dsum = (part[r] + part[128 + r]) + (part[256 + r] + part[384 + r]);
      }
    }
    if (mine && quarter == 0) a.dvec[at] = dsum;
    const float2 nd2 = make_float2(-dsum, -dsum);
    for (int j = 0; j < n && ok; ++j) {
      const bool diag = j == n - 1;
      if (!mbar_wait_warp(s_full, j & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) { ok = false; break; }
      tc_fence_after();
      float p[32];
      __syncwarp();
      tmem_ld_32x32b_x32(tS + lane_off + cb, *reinterpret_cast<uint32_t(*)[32]>(p));
      tmem_ld_wait();
      tc_fence_before();
      warp_arrive(s_free);
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const float2 v = __ffma2_rn(make_float2(p[e], p[e + 1]), c2, nl2);
        p[e] = ex2_approx(v.x);
        p[e + 1] = ex2_approx(v.y);
      }
      if (diag) {
        // rows of K past the sequence, which weights of 0 would meet
        if (quarter == 0 && j * 128 + r >= un.len) {
          mbar_wait(&kv_full[j % NK], (j / NK) & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE);
          tile_row_clear<D>(sKV + (j % NK) * TILE, r);
          fence_proxy_async_smem();
        }
        __syncwarp();
      }
      if (!mbar_wait_warp(dp_full, j & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) { ok = false; break; }
      tc_fence_after();
      uint32_t dp[32], pk[16];
      __syncwarp();
      tmem_ld_32x32b_x32(tP + lane_off + cb, dp);
      tmem_ld_wait();
      tc_fence_before();
      warp_arrive(dp_free);
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        float2 y = __fmul2_rn(make_float2(p[e], p[e + 1]), __fadd2_rn(make_float2(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1])), nd2));
        if (diag) {
          if (cb + e > r) y.x = 0.f;
          if (cb + e + 1 > r) y.y = 0.f;
          if (e == 0 && first) y.x *= 0.f;
        }
        pk[e >> 1] = pack_bf16x2(y.x, y.y);
      }
      if (j >= 2 && !mbar_wait_warp(&ds_free[j & 1], ((j - 2) >> 1) & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) { ok = false; break; }
      __syncwarp();
      tmem_st_32x32b_x16(tD + (j & 1) * 64 + lane_off + quarter * 16, pk);
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&ds_full[j & 1]);
    }
    if (ok && mbar_wait_warp(done, 0, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) {
      tc_fence_after();
      // Q's tile is free: all products of it are done
      __nv_bfloat16* dst = a.dq + ((long long)(un.begin + row0 + q4 * 32) * a.Hq + h) * D + quarter * (D / 4);
      store_rows<D / 32, D / 32>(tQ + lane_off + quarter * (D / 4), a.scale, sQ + (warp - 2) * (32 * (D / 4) * 2), dst, nullptr, (long long)a.Hq * D, un.len - row0 - q4 * 32);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ================================================================================ backward: dK, dV
// One CTA per 128 keys of a key/value head, over the queries from there on of all its query heads, in the
// transposed frame (a key a TMEM lane).  TMEM: S^T | dP^T | dV | dK; P^T and dS^T lie over the scores they came
// from, each warp's over columns that it alone has read (four warps a lane quarter, 32 columns each).  MMA order dV(i), S(i+1), dK(i), dP(i+1): while the
// compute warps turn dP into dS the tensor core runs dV and the next S, and while they take the next exponentials dK
// and the next dP.
template <int D>
struct PkDkv {
  static constexpr uint32_t TILE = 128u * D * 2u;
  static constexpr size_t SMEM = 1024 + 6 * TILE + 4 * 512 + 32 * 8 + 64;
};

template <int D>
__global__ void __launch_bounds__(576, 1)
    packed_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmG, const PkArgs a) {
  constexpr uint32_t TILE = PkDkv<D>::TILE;
  constexpr int PANELS = D / 64;
  constexpr uint32_t IDESC_S = umma_idesc_bf16(128, 128, false, false);
  constexpr uint32_t IDESC_KV = umma_idesc_bf16(128, D, false, true);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;
  uint8_t* sV = sK + TILE;
  uint8_t* sQ = sV + TILE;             // [2]
  uint8_t* sG = sQ + 2 * TILE;         // [2]
  float* sL = reinterpret_cast<float*>(sG + 2 * TILE);   // [2][128] -lse in log2
  float* sD = sL + 256;                                  // [2][128] -D
  uint64_t* bars = reinterpret_cast<uint64_t*>(sD + 256);
  uint64_t* bar_kv = bars + 0;
  uint64_t* q_full = bars + 1;         // [2]
  uint64_t* q_empty = bars + 3;        // [2]
  uint64_t* g_full = bars + 5;         // [2]
  uint64_t* g_empty = bars + 7;        // [2]
  uint64_t* l_full = bars + 9;         // [2]
  uint64_t* s_full = bars + 11;
  uint64_t* p_full = bars + 12;
  uint64_t* dp_full = bars + 13;
  uint64_t* ds_full = bars + 14;
  uint64_t* done = bars + 15;
  uint64_t* drain = bars + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 17);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  PieceUnit* s_unit = reinterpret_cast<PieceUnit*>(tmem_slot + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = (int)(blockIdx.x % a.Hkv);
  if (warp == 0) {
    const PieceUnit u = piece_unit<128>(a.pc, (int)(blockIdx.x / a.Hkv));   // a sequence's first keys have the most queries
    if (lane == 0) *s_unit = u;
  } else if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  } else if (threadIdx.x == 64) {
    mbar_init(bar_kv, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&g_full[i], 1);
      mbar_init(&g_empty[i], 1);
      mbar_init(&l_full[i], 8);
    }
    mbar_init(s_full, 1);
    mbar_init(p_full, 16);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, 16);
    mbar_init(done, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmG);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;           // all 512 columns are this CTA's: they start at 0
  if (threadIdx.x == 0 && *tmem_slot != tmem) atomicOr(a.err, ERR_BAD_ARG);
  const uint32_t tS = tmem, tP = tmem + 128, tDV = tmem + 256, tDK = tmem + 384;
  const PieceUnit un = *s_unit;
  const int kt = un.unit, row0 = kt * 128;
  const int tiles = (un.len + 127) / 128, nq = tiles - kt, n = nq * a.G;   // steps: query tiles kt .. of every query head

  if (un.unit < 0 || !a.pc.real(un.piece)) {
    if (un.unit >= 0) {
      clear_rows<D>(a.dk, a.Hkv, hk, 1, un.begin + row0, min(128, un.len - row0));
      clear_rows<D>(a.dv, a.Hkv, hk, 1, un.begin + row0, min(128, un.len - row0));
    }
  } else if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      uint32_t valid = 0, parity = 0;    // bits 0, 1: Q; 2, 3: dO
      mbar_arrive_expect_tx(bar_kv, 2 * TILE);
#pragma unroll
      for (int p = 0; p < PANELS; ++p) {
        tma_load_3d(sK + p * kPanel, &tmK, bar_kv, p * 64, un.begin + row0, hk);
        tma_load_3d(sV + p * kPanel, &tmV, bar_kv, p * 64, un.begin + row0, hk);
      }
      int qi = kt, h = hk * a.G;
      for (int it = 0; it < n && ok; ++it) {
        const int b = it & 1;
#pragma unroll
        for (int w = 0; w < 2 && ok; ++w) {
          if (it >= 2 && !mbar_wait(w ? &g_empty[b] : &q_empty[b], ((it - 2) >> 1) & 1, abort_flag, a.err, ERR_TIMEOUT_PRODUCER)) {
            ok = false;
            break;
          }
          uint64_t* bar = w ? &g_full[b] : &q_full[b];
          mbar_arrive_expect_tx(bar, TILE);
          valid |= 1u << (2 * w + b);
          parity = (parity & ~(1u << (2 * w + b))) | ((uint32_t)((it >> 1) & 1) << (2 * w + b));
#pragma unroll
          for (int p = 0; p < PANELS; ++p)
            tma_load_3d((w ? sG : sQ) + b * TILE + p * kPanel, w ? &tmG : &tmQ, bar, p * 64, un.begin + qi * 128, h);
        }
        if (++qi == tiles) { qi = kt; ++h; }
      }
      if (!ok) {
        *abort_flag = 1;
        const unsigned long long t0 = globaltimer_ns();
        for (int s = 0; s < 4; ++s) {
          if (!((valid >> s) & 1u)) continue;
          while (!mbar_try_wait(s < 2 ? &q_full[s] : &g_full[s - 2], (parity >> s) & 1u))
            if (globaltimer_ns() - t0 > 200000000ull) break;
        }
        while (!mbar_try_wait(bar_kv, 0))
          if (globaltimer_ns() - t0 > 300000000ull) break;
      }
    }
  } else if (warp == 1) {
    bool ok = mbar_wait_warp(bar_kv, 0, abort_flag, a.err, ERR_TIMEOUT_MMA);
    const bool leader = elect_one();
    const uint64_t kd = kmajor_base(sK), vd = kmajor_base(sV), qk = kmajor_base(sQ), gk = kmajor_base(sG), qm = mnmajor_base(sQ), gm = mnmajor_base(sG);
    constexpr uint64_t STEP = TILE >> 4;
    auto commit = [&](uint64_t* bar) {
      if (leader) umma_commit(bar);
      __syncwarp();
    };
    auto issue_s = [&](int it) -> bool {   // S^T = K Q^T
      const int b = it & 1;
      if (!mbar_wait_warp(&q_full[b], (it >> 1) & 1, abort_flag, a.err, ERR_TIMEOUT_MMA)) return false;
      tc_fence_after();
      if (leader) {
        mma_kk<D / 16>(tS, kd, qk + b * STEP, IDESC_S);
        umma_commit(s_full);
      }
      __syncwarp();
      return true;
    };
    auto issue_dp = [&](int it) -> bool {  // dP^T = V dO^T
      const int b = it & 1;
      if (!mbar_wait_warp(&g_full[b], (it >> 1) & 1, abort_flag, a.err, ERR_TIMEOUT_MMA)) return false;
      tc_fence_after();
      if (leader) {
        mma_kk<D / 16>(tP, vd, gk + b * STEP, IDESC_S);
        umma_commit(dp_full);
      }
      __syncwarp();
      return true;
    };
    if (ok) ok = issue_s(0) && issue_dp(0);
    for (int it = 0; it < n && ok; ++it) {
      const int b = it & 1;
      if (!mbar_wait_warp(p_full, it & 1, abort_flag, a.err, ERR_TIMEOUT_MMA)) { ok = false; break; }
      tc_fence_after();
      if (leader) {
        // dV += P^T dO: the weights of 32 queries in the first 16 of their scores' columns
        mma_tmem<32>(tDV, tS, gm + b * STEP, IDESC_KV, it > 0);
        umma_commit(&g_empty[b]);
      }
      __syncwarp();
      if (it + 1 < n && !issue_s(it + 1)) { ok = false; break; }
      if (!mbar_wait_warp(ds_full, it & 1, abort_flag, a.err, ERR_TIMEOUT_MMA)) { ok = false; break; }
      tc_fence_after();
      if (leader) {
        mma_tmem<32>(tDK, tP, qm + b * STEP, IDESC_KV, it > 0);   // dK += dS^T Q
        umma_commit(&q_empty[b]);
      }
      __syncwarp();
      if (it + 1 < n && !issue_dp(it + 1)) { ok = false; break; }
    }
    if (ok) {
      commit(done);
    } else {
      *abort_flag = 1;
      commit(drain);
      const unsigned long long t0 = globaltimer_ns();
      while (!mbar_try_wait(drain, 0))
        if (globaltimer_ns() - t0 > 100000000ull) break;
    }
  } else {
    const int q4 = warp & 3, quarter = (warp - 2) >> 2, cb = quarter * 32;
    const int r = q4 * 32 + lane;
    const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
    const float2 c2 = make_float2(a.scale_log2, a.scale_log2);
    const bool first = row0 + r == 0 && quarter == 0;    // holds the ds that is 0 by definition, in the diagonal tiles
    const bool reads = quarter < 2;      // the first 256 threads: a query's lse (quarter 0) or D
    const float* stats = quarter == 0 ? a.lse : a.dvec;
    int qi = kt, h = hk * a.G;
    // a step ahead and as it is (what is computed from it waits for it); a query past the sequence weighs nothing
    auto stat = [&](int i, int hh) -> float {
      const int qrow = i * 128 + r;
      return reads && qrow < un.len ? stats[(long long)hh * a.pc.M + un.begin + qrow] : quarter == 0 ? INFINITY : 0.f;
    };
    const float turn = quarter == 0 ? -kLog2e : -1.f;
    float next = stat(qi, h);
    bool ok = true;
    for (int it = 0; it < n; ++it) {
      const int b = it & 1;
      float *nl = sL + b * 128, *nd = sD + b * 128;
      if (reads) {
        (quarter == 0 ? nl : nd)[r] = next * turn;
        warp_arrive(&l_full[b]);
      }
      const bool diag = qi == kt;
      const int lim = un.len - qi * 128;     // queries of this tile
      if (++qi == tiles) { qi = kt; ++h; }
      if (it + 1 < n) next = stat(qi, h);
      if (!mbar_wait_warp(s_full, it & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) { ok = false; break; }
      tc_fence_after();
      const bool part = diag || lim < 128;   // some of its weights are chosen to be 0
      if (lim < 128) {
        // rows of dO and Q past the sequence, which weights of 0 would meet
        if (reads && r >= lim) {
          mbar_wait(quarter == 0 ? &g_full[b] : &q_full[b], (it >> 1) & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE);
          tile_row_clear<D>((quarter == 0 ? sG : sQ) + b * TILE, r);
          fence_proxy_async_smem();
        }
        __syncwarp();
      }
      float p[32];      // this thread's 32 columns of the P^T row
      uint32_t pk[16];  // packed bf16 pairs of it, then of dS^T
      __syncwarp();
      tmem_ld_32x32b_x32(tS + lane_off + cb, *reinterpret_cast<uint32_t(*)[32]>(p));
      if (!mbar_wait_warp(&l_full[b], (it >> 1) & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) { ok = false; break; }
      tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        const int cc = cb + e;
        const float4 n4 = *reinterpret_cast<const float4*>(nl + cc);
        const float2 v0 = __ffma2_rn(make_float2(p[e], p[e + 1]), c2, make_float2(n4.x, n4.y));
        const float2 v1 = __ffma2_rn(make_float2(p[e + 2], p[e + 3]), c2, make_float2(n4.z, n4.w));
        float2 p0 = make_float2(ex2_approx(v0.x), ex2_approx(v0.y)), p1 = make_float2(ex2_approx(v1.x), ex2_approx(v1.y));
        if (part) {
          const int lo = diag ? r : 0;       // queries lo .. lim - 1 see this key
          if (cc < lo || cc >= lim) p0.x = 0.f;
          if (cc + 1 < lo || cc + 1 >= lim) p0.y = 0.f;
          if (cc + 2 < lo || cc + 2 >= lim) p1.x = 0.f;
          if (cc + 3 < lo || cc + 3 >= lim) p1.y = 0.f;
        }
        p[e] = p0.x; p[e + 1] = p0.y; p[e + 2] = p1.x; p[e + 3] = p1.y;
        pk[e >> 1] = pack_bf16x2(p0.x, p0.y);
        pk[(e >> 1) + 1] = pack_bf16x2(p1.x, p1.y);
      }
      __syncwarp();
      tmem_st_32x32b_x16(tS + lane_off + cb, pk);
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(p_full);
      if (!mbar_wait_warp(dp_full, it & 1, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) { ok = false; break; }
      tc_fence_after();
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2) {       // (all 32 at once: registers ran out)
        uint32_t dp[16];
        __syncwarp();
        tmem_ld_32x32b_x16(tP + lane_off + cb + h2 * 16, dp);
        tmem_ld_wait();
#pragma unroll
        for (int e0 = 0; e0 < 16; e0 += 4) {
          const int e = h2 * 16 + e0, cc = cb + e;
          const float4 d4 = *reinterpret_cast<const float4*>(nd + cc);
          float2 da = __fmul2_rn(make_float2(p[e], p[e + 1]), __fadd2_rn(make_float2(__uint_as_float(dp[e0]), __uint_as_float(dp[e0 + 1])), make_float2(d4.x, d4.y)));
          float2 db = __fmul2_rn(make_float2(p[e + 2], p[e + 3]), __fadd2_rn(make_float2(__uint_as_float(dp[e0 + 2]), __uint_as_float(dp[e0 + 3])), make_float2(d4.z, d4.w)));
          if (part) {
            const int lo = diag ? r : 0;
            if (cc < lo || cc >= lim) da.x = 0.f;
            if (cc + 1 < lo || cc + 1 >= lim) da.y = 0.f;
            if (cc + 2 < lo || cc + 2 >= lim) db.x = 0.f;
            if (cc + 3 < lo || cc + 3 >= lim) db.y = 0.f;
            if (e == 0 && first && diag) da.x *= 0.f;
          }
          pk[e >> 1] = pack_bf16x2(da.x, da.y);
          pk[(e >> 1) + 1] = pack_bf16x2(db.x, db.y);
        }
      }
      __syncwarp();
      tmem_st_32x32b_x16(tP + lane_off + cb, pk);
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(ds_full);
    }
    if (ok && mbar_wait_warp(done, 0, abort_flag, a.err, ERR_TIMEOUT_EPILOGUE)) {
      tc_fence_after();
      // K's and V's tiles are free: all products of them are done
      const int first = row0 + q4 * 32, n_rows = un.len - first;
      const long long at = ((long long)(un.begin + first) * a.Hkv + hk) * D + quarter * (D / 4), stride = (long long)a.Hkv * D;
      const uint32_t stage = (warp - 2) * (32 * (D / 4) * 2);
      store_rows<D / 32, D / 32>(tDV + lane_off + quarter * (D / 4), 1.f, sV + stage, a.dv + at, nullptr, stride, n_rows);
      store_rows<D / 32, D / 32>(tDK + lane_off + quarter * (D / 4), a.scale, sK + stage, a.dk + at, nullptr, stride, n_rows);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------------------ host
// A kernel's shared memory, said once a device: the call takes longer than the launch.
template <auto KERN>
static void pk_smem(size_t bytes, int dev) {
  static std::atomic<uint64_t> done{0};
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return;
  C10_CUDA_CHECK(cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  done.fetch_or(bit, std::memory_order_relaxed);
}

template <auto KERN>
struct PkKern {
  static constexpr auto value = KERN;
};

struct PkView {
  at::Tensor t;                  // a copy where the rows cannot be read in place
  const __nv_bfloat16* p;
  long long r, h;
  CUtensorMap map;
};

static PkView pk_view(const at::Tensor& given, const char* name, const at::Tensor& q, int64_t H) {
  TORCH_CHECK(given.is_cuda() && given.device() == q.device() && given.scalar_type() == at::kBFloat16 && given.dim() == 3 &&
                  given.size(0) == q.size(0) && given.size(1) == H && given.size(2) == q.size(2),
              name, ": bfloat16 [M, H, D] of q's M and D on its device");
  const int64_t M = given.size(0), D = given.size(2);
  PkView v{};
  auto take = [&](const at::Tensor& t) {
    v.t = t;
    v.p = reinterpret_cast<const __nv_bfloat16*>(t.data_ptr());
    v.h = H > 1 ? t.stride(1) : D;
    v.r = M > 1 ? t.stride(0) : H * D;
    return t.stride(2) == 1 && v.r > 0 && v.h > 0 && v.r % 8 == 0 && v.h % 8 == 0 && (reinterpret_cast<uintptr_t>(v.p) & 15) == 0;
  };
  if (!take(given)) take(given.clone(at::MemoryFormat::Contiguous));   // broadcast, misaligned or strided inside
  if (M > 0) v.map = make_tmap_bf16(v.p, D, M, v.r, 64, 128, H, v.h);
  return v;
}

struct PkCall {
  PkArgs a;
  PkView q, k, v;
  int64_t M, D;
};

static PkCall pk_check(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& cu, double scale, const at::Tensor& err) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && q.scalar_type() == at::kBFloat16, "q: bfloat16 [M, Hq, D]");
  TORCH_CHECK(k.dim() == 3 && v.dim() == 3, "k and v: bfloat16 [M, Hkv, D]");
  PkCall c{};
  const int64_t Hq = q.size(1), Hkv = k.size(1);
  c.M = q.size(0); c.D = q.size(2);
  TORCH_CHECK(c.D == 64 || c.D == 128, "head_dim 64 or 128");
  TORCH_CHECK(Hq >= 1 && Hkv >= 1 && Hq % Hkv == 0, "the query heads: a multiple of the key/value heads");
  TORCH_CHECK(c.M <= (1 << 30), "at most 2^30 rows");
  TORCH_CHECK(cu.scalar_type() == at::kInt && cu.device() == q.device() && cu.dim() == 1 && cu.size(0) >= 1 && cu.size(0) <= (1 << 30) && cu.is_contiguous(),
              "cu_seqlens: contiguous int32 [S + 1] on q's device");
  const float scale_log2 = (float)(scale * 1.4426950408889634);
  TORCH_CHECK(scale > 0 && scale_log2 > 0 && std::isfinite(scale_log2), "scale: a number within float32's range");
  c.q = pk_view(q, "q", q, Hq);
  c.k = pk_view(k, "k", q, Hkv);
  c.v = pk_view(v, "v", q, Hkv);
  PkArgs& a = c.a;
  a.pc.cu = cu.data_ptr<int>(); a.pc.S = (int)cu.size(0) - 1; a.pc.M = (int)c.M;
  a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.G = (int)(Hq / Hkv);
  a.scale = (float)scale; a.scale_log2 = scale_log2;
  a.q = c.q.p; a.qr = c.q.r; a.qh = c.q.h;
  a.k = c.k.p; a.kr = c.k.r; a.kh = c.k.h;
  a.v = c.v.p; a.vr = c.v.r; a.vh = c.v.h;
  a.err = err.data_ptr<int>();
  return c;
}

static unsigned pk_grid(long long slots, long long heads) {
  TORCH_CHECK(slots * heads < (1LL << 31), "too many rows and heads");
  return (unsigned)(slots * heads);
}

// (out [M, Hq, D]; for a backward also lse [Hq, M] and the rest of the output [M, Hq, D])
std::tuple<at::Tensor, c10::optional<at::Tensor>, c10::optional<at::Tensor>> packed_attention_fwd(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor cu, double scale, bool want_lse,
                                             at::Tensor err) {
  TORCH_CHECK(q.is_cuda(), "q: a CUDA tensor");
  c10::cuda::CUDAGuard guard(q.device());
  PkCall c = pk_check(q, k, v, cu, scale, err);
  PkArgs& a = c.a;
  auto out = at::empty({c.M, a.Hq, c.D}, q.options());
  c10::optional<at::Tensor> lse, low;
  if (want_lse) {
    lse = at::empty({a.Hq, c.M}, q.options().dtype(at::kFloat));
    low = at::empty({c.M, a.Hq, c.D}, q.options());
  }
  if (c.M == 0) return {out, lse, low};
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.lse = want_lse ? lse->data_ptr<float>() : nullptr;
  a.low = want_lse ? reinterpret_cast<__nv_bfloat16*>(low->data_ptr()) : nullptr;
  a.by_heads = a.G % 2 == 0;
  auto s = at::cuda::getCurrentCUDAStream();
  auto launch = [&](auto cfg, auto kern, int64_t slots, int64_t heads) {
    typedef decltype(cfg) Cfg;
    constexpr auto KERN = decltype(kern)::value;
    pk_smem<KERN>(Cfg::SMEM, q.get_device());
    KERN<<<pk_grid(slots, heads), Cfg::THREADS, Cfg::SMEM, s>>>(c.q.map, c.k.map, c.v.map, a);
  };
  // One tile a CTA, two CTAs an SM, where a tile has few keys and no second head shares them: one's start and end lie under the
  // other's products (10 heads, 65536 rows: 236 instead of 256 us for sequences of 512, 379 instead of 588 for 64; from 1024 on
  // two tiles that share their keys are as fast or faster).  The lengths are in device memory, so the mean over all entries of
  // cu_seqlens has to do: where most of them are empty, long sequences get the one-tile form too, at 10971 instead of 9648 us for one of
  // 65535 rows, 1524 instead of 1392 for eight of 8192 (10 heads).
  const bool one = !a.by_heads && c.M < 1024 * (int64_t)a.pc.S;
  if (one) {
    const int64_t slots = piece_slots(c.M, a.pc.S, 128);
    if (c.D == 128) launch(PkFwd<128, 1>{}, PkKern<packed_fwd_kernel<128, 1>>{}, slots, a.Hq);
    else launch(PkFwd<64, 1>{}, PkKern<packed_fwd_kernel<64, 1>>{}, slots, a.Hq);
  } else {
    const int64_t slots = piece_slots(c.M, a.pc.S, a.by_heads ? 128 : 256), heads = a.by_heads ? a.Hq / 2 : a.Hq;
    if (c.D == 128) launch(PkFwd<128, 2>{}, PkKern<packed_fwd_kernel<128, 2>>{}, slots, heads);
    else launch(PkFwd<64, 2>{}, PkKern<packed_fwd_kernel<64, 2>>{}, slots, heads);
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {out, lse, low};
}

// {dq, dk, dv}, packed [M, H, D]; out and lse are the forward's.
std::vector<at::Tensor> packed_attention_bwd(at::Tensor dout, at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor out, at::Tensor low,
                                             at::Tensor lse, at::Tensor cu, double scale, at::Tensor err) {
  TORCH_CHECK(q.is_cuda(), "q: a CUDA tensor");
  c10::cuda::CUDAGuard guard(q.device());
  PkCall c = pk_check(q, k, v, cu, scale, err);
  PkArgs& a = c.a;
  const PkView g = pk_view(dout, "the output's gradient", q, a.Hq);
  for (const auto* t : {&out, &low})
    TORCH_CHECK(t->device() == q.device() && t->scalar_type() == at::kBFloat16 && t->sizes() == q.sizes() && t->is_contiguous(),
                "out and its rest: the forward's");
  TORCH_CHECK(lse.device() == q.device() && lse.scalar_type() == at::kFloat && lse.numel() == a.Hq * c.M && lse.is_contiguous(), "lse: the forward's");
  auto dq = at::empty({c.M, a.Hq, c.D}, q.options()), dk = at::empty({c.M, a.Hkv, c.D}, q.options()), dv = at::empty({c.M, a.Hkv, c.D}, q.options());
  if (c.M == 0) return {dq, dk, dv};
  auto dvec = at::empty({a.Hq, c.M}, lse.options());
  a.o = reinterpret_cast<const __nv_bfloat16*>(out.data_ptr());
  a.low = reinterpret_cast<__nv_bfloat16*>(low.data_ptr());
  a.dout = g.p; a.gr = g.r; a.gh = g.h;
  a.dq = reinterpret_cast<__nv_bfloat16*>(dq.data_ptr());
  a.dk = reinterpret_cast<__nv_bfloat16*>(dk.data_ptr());
  a.dv = reinterpret_cast<__nv_bfloat16*>(dv.data_ptr());
  a.lse = lse.data_ptr<float>(); a.dvec = dvec.data_ptr<float>();
  const long long slots = piece_slots(c.M, a.pc.S, 128);
  const unsigned gq = pk_grid(slots, a.Hq), gk = pk_grid(slots, a.Hkv);
  auto s = at::cuda::getCurrentCUDAStream();
  if (c.D == 128) {
    pk_smem<packed_dq_kernel<128>>(PkDq<128>::SMEM, q.get_device());
    pk_smem<packed_dkv_kernel<128>>(PkDkv<128>::SMEM, q.get_device());
    packed_dq_kernel<128><<<gq, 608, PkDq<128>::SMEM, s>>>(c.q.map, c.k.map, c.v.map, g.map, a);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    packed_dkv_kernel<128><<<gk, 576, PkDkv<128>::SMEM, s>>>(c.q.map, c.k.map, c.v.map, g.map, a);
  } else {
    pk_smem<packed_dq_kernel<64>>(PkDq<64>::SMEM, q.get_device());
    pk_smem<packed_dkv_kernel<64>>(PkDkv<64>::SMEM, q.get_device());
    packed_dq_kernel<64><<<gq, 608, PkDq<64>::SMEM, s>>>(c.q.map, c.k.map, c.v.map, g.map, a);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    packed_dkv_kernel<64><<<gk, 576, PkDkv<64>::SMEM, s>>>(c.q.map, c.k.map, c.v.map, g.map, a);
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {dq, dk, dv};
}

}  // namespace tfb
