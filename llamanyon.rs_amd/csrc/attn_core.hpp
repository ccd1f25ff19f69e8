// attn_core.hpp -- causal attention of a batch's new tokens over the paged cache
// (swamp_attn_paged): o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q.k_j).
//
// Mathematics.  One pass over the keys with the softmax's running maximum m and
// sum l: a tile's scores s, m' = max(m, c max s) with c = scale log2 e, p =
// 2^(c s - m'), l and o scaled by 2^(m - m') where m grows by more than kSlack
// (p then reaches 2^kSlack at most; sums and the last division do not care).
// For fp16 weights m lies below the maximum, and follows the tiles down as well
// (Rows::kFall).
//
// Tiles.  The rows of one cache head -- new tokens times the query heads that
// share it -- are cut into blocks of 128, and a block takes its keys in tiles.
// Scores are taken as S^T = K Q^T with 32 x 32 x 16 matrix instructions: a lane
// then holds 16 of 32 keys of ONE row (lane % 32), so that maximum and sum stay
// within the lane but for one exchange with lane ^ 32, and P^T is already the B
// operand of O^T = V^T P^T (keys are summed in the order that S^T left them in,
// V is read in the same order by the transposing LDS read).  Neither P nor the
// statistics pass through LDS.
//
// Feeding.  Keys and values reach LDS by direct-to-LDS DMA, 16 bytes a lane in
// groups of 16 keys.  A row of dim elements lies at a stride of S 16-byte
// chunks: dims of 64, 128 and 256 XOR the chunk with the row (K: all rows of a
// fragment read in different banks; V: the four rows of a transposing read),
// other dims take an odd stride of chunks instead.
//
// Bounds and measures.  Decoding is HBM's: all keys once, 5.2 to 5.5 TB/s of the
// 6.0 that a long read reaches (one token over 131072 keys 98 us).  Prompts are
// the matrix pipe's and its power's: 4096 tokens of 64 heads of 128 dims take 274
// us, 1000 TFLOP/s, where a bf16 product of the library reaches 1130 to 1230; of
// 296 us on a slower card the exponentials cost 19, the DMAs 33, and what is left
// without them, products, maximum and conversion, runs at 1175 TFLOP/s.  Two waves a
// SIMD (201 registers) fill each other's gaps; blocks of 256 rows in workgroups of
// eight waves halve the DMAs and lost more to their common barrier (64 dims: 93 ->
// 107 us).
//
// Rows outside a block's keys are loaded from its nearest key: their weights
// are 0 and what they hold is finite wherever the keys are.  A weight of 0 times
// an infinity or NaN that only OTHER rows see would still spoil a row.  So a
// result that is not finite is computed once more with such values taken out of
// the tiles and added, row by row, to the rows that see them.
#pragma once
#include "attn_plan.hpp"
#include "paging.hpp"
#include "swamp_common.hpp"

#include <type_traits>

namespace swamp_attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896341f;

struct Work {
  swamp::PagedCache cache;
  swamp::SeqBatch b;
  const uint16_t *q;
  int64_t q_stride;
  void *out;
  int64_t out_stride;
  uint32_t out_type;
  int n_heads, group, window;
  float scale;
  int blocks;      // blocks of the grid (per head and split)
  int one_block;   // no sequence has more than one
  int few;         // no sequence has more than kFew rows
  int splits;      // pieces of a sequence's keys
  int chunk;       // keys of a piece (a multiple of kTile); the last takes the rest
  float *part;     // [split][row][dim]: sums of a piece, splits > 1
  f32x2 *stat;     // [split][row]: (m, l); l = -1: the row sees no key at all
};

}  // namespace swamp_attn

namespace {

using namespace swamp_attn;

// ---- LDS and DMA ----------------------------------------------------------
// LDS is addressed by byte offset.  Not templates: the host pass rejects the
// address-space cast inside a template instantiation.
__device__ __forceinline__ uint32_t lds_base(uint8_t *smem) {
  return uint32_t(uintptr_t((__attribute__((address_space(3))) uint8_t *)smem));
}
// at + off, off a constant: the sum stays in the instruction's offset.
#define SWAMP_LDS(T, at, off)                                          \
  ((__attribute__((address_space(3))) T *)((__attribute__((            \
       address_space(3))) uint8_t *)(uintptr_t)(at) + (off)))
__device__ __forceinline__ s16x8 lds16(uint32_t at, uint32_t off = 0) {
  return *SWAMP_LDS(s16x8, at, off);
}
__device__ __forceinline__ void lds16_put(uint32_t at, s16x8 v) {
  *(__attribute__((address_space(3))) s16x8 *)(uintptr_t)at = v;
}
__device__ __forceinline__ f32x4 ldsf4(uint32_t at) {
  return *(__attribute__((address_space(3))) f32x4 *)(uintptr_t)at;
}
__device__ __forceinline__ void ldsf4_put(uint32_t at, f32x4 v) {
  *(__attribute__((address_space(3))) f32x4 *)(uintptr_t)at = v;
}
__device__ __forceinline__ float ldsf(uint32_t at) {
  return *(__attribute__((address_space(3))) float *)(uintptr_t)at;
}
__device__ __forceinline__ void ldsf_put(uint32_t at, float v) {
  *(__attribute__((address_space(3))) float *)(uintptr_t)at = v;
}
// Four rows' elements of one column: lane i of 16 names 8 bytes of row i / 4 and
// gets column i of the 4 x 16 block.
__device__ __forceinline__ s16x4 lds_tr(uint32_t at, uint32_t off) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(SWAMP_LDS(s16x4, at, off));
}

__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ float uni(float x) {
  return __uint_as_float(uint32_t(uni(int(__float_as_uint(x)))));
}
__device__ __forceinline__ const void *uni(const void *p) {
  const uint64_t x = uint64_t(uintptr_t(p));
  const uint32_t lo = uint32_t(uni(int(uint32_t(x)))), hi = uint32_t(uni(int(x >> 32)));
  return reinterpret_cast<const void *>(uintptr_t(uint64_t(hi) << 32 | lo));
}

// DMA, 16 bytes a lane into LDS (lane L writes at + 16 L).  Written as assembly
// because the compiler waits for every DMA in flight before it lets a transposing
// read pass.  They have no output register, every read of what they bring stands
// behind a wait of wait_dma or wait_all, and m0 has no other user in these kernels.
//
// N of them, from base + off[j] to at + 1024 j.  The instruction's offset counts
// for both addresses, so that one m0 serves four; off[j] holds dma_lift(j) to
// make up for it.
constexpr uint32_t dma_lift(int j) { return 1024u * (3 - j % 4); }
template <int N>
__device__ __forceinline__ void dma_uniform(const uint8_t *base, const uint32_t *off, uint32_t at) {
#ifdef __HIP_DEVICE_COMPILE__
  const void *from = uni(base - dma_lift(0));
#pragma unroll
  for (int j = 0; j < N; j += 4) {
    const uint32_t to = uint32_t(uni(int(at + 1024 * j)));
    if (N - j >= 4)
      asm volatile(
          "s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %5\n\t"
          "global_load_lds_dwordx4 %2, %5 offset:1024\n\t"
          "global_load_lds_dwordx4 %3, %5 offset:2048\n\t"
          "global_load_lds_dwordx4 %4, %5 offset:3072"
          :
          : "s"(to), "v"(off[j]), "v"(off[j + 1]), "v"(off[j + 2]), "v"(off[j + 3]), "s"(from));
    else if (N - j == 3)
      asm volatile(
          "s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %4\n\t"
          "global_load_lds_dwordx4 %2, %4 offset:1024\n\t"
          "global_load_lds_dwordx4 %3, %4 offset:2048"
          :
          : "s"(to), "v"(off[j]), "v"(off[j + 1]), "v"(off[j + 2]), "s"(from));
    else
      asm volatile(
          "s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\t"
          "global_load_lds_dwordx4 %2, %3 offset:1024"
          :
          : "s"(to), "v"(off[j]), "v"(off[j + 1]), "s"(from));
  }
  static_assert(N % 4 != 1, "no form of one");
#endif
}
// One, with every lane's own address.
__device__ __forceinline__ void dma_lane(const void *p, uint32_t at) {
#ifdef __HIP_DEVICE_COMPILE__
  at = uint32_t(uni(int(at)));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(at), "v"(p));
#endif
}
// At most N DMAs (and loads) of this wave in flight; its LDS reads are done.
template <int N>
__device__ __forceinline__ void wait_dma() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
// The same for all waves of the workgroup, and nothing in flight.
__device__ __forceinline__ void wait_all() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
__device__ __forceinline__ void lds_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// x, which the compiler no longer knows: what rare paths compute from it is not
// computed ahead of the loop and kept in registers meanwhile.
template <typename T>
__device__ __forceinline__ T fresh(T x) {
#ifdef __HIP_DEVICE_COMPILE__
  asm volatile("" : "+v"(x));
#endif
  return x;
}

// Whether x holds anywhere in the workgroup; 4 bytes a wave of LDS at `at`.
__device__ __forceinline__ bool anywhere(bool x, uint32_t at) {
  const uint32_t mine = __any(x) ? 1u : 0u;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) ldsf_put(at + (threadIdx.x >> 6) * 4, __uint_as_float(mine));
  __syncthreads();
  uint32_t all = 0;
#pragma unroll
  for (int i = 0; i < kWaves; i++) all |= __float_as_uint(ldsf(at + 4 * i));
  return uni(int(all)) != 0;
}

// ---- element types --------------------------------------------------------
template <typename CT>
struct Op;
template <>
struct Op<_Float16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  static constexpr uint16_t kExp = 0x7C00;
  static constexpr float kMax = 65504.f;
  static constexpr int kParts = 2;  // 11 bits each: 22
  static constexpr bool kNarrow = true;  // a weight's range, see Rows::kFall
  static __device__ __forceinline__ f32x16 mma(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a),
                                                  __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};
template <>
struct Op<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  static constexpr uint16_t kExp = 0x7F80;
  static constexpr float kMax = 3.38953139e38f;
  static constexpr int kParts = 3;  // 8 bits each: 24
  static constexpr bool kNarrow = false;
  static __device__ __forceinline__ f32x16 mma(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a),
                                                   __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};

// ---- how the keys lie -----------------------------------------------------
// D: the head's dims, or (not exact) the most of them.
template <int D, bool kExact>
struct Geo {
  static constexpr bool kPow2 = kExact && (D & (D - 1)) == 0;
  static constexpr int KS = (D + 15) / 16;  // score steps of 16 dims
  static constexpr int DB = (D + 31) / 32;  // output blocks of 32 dims
  static constexpr int kStride = kPow2 ? D / 8 : kExact ? (D / 8) | 1 : D / 8 - 1;
  static constexpr int NI = (kStride + 3) / 4;      // DMAs of a group of 16 keys (1 KB each)
  static constexpr uint32_t kGroup = NI * 1024;     // bytes of a group
  static constexpr uint32_t kBuf = 8 * kGroup;      // K and V of a tile
  static constexpr uint32_t kSmem = 2 * kBuf;       // and the next tile's
  static constexpr uint32_t kExtra = 4 * 32 * 2 * 4;  // statistics of the waves
  int nch, stride;  // 16-byte chunks of a row, and from row to row
  __device__ __forceinline__ Geo(int dim) {
    nch = kExact ? D / 8 : dim / 8;
    stride = kExact ? kStride : (nch | 1);
  }
  __device__ __forceinline__ bool within(int d) const { return kPow2 || d < 8 * nch; }
  static __device__ __forceinline__ int k_chunk(int r, int c) {
    return !kPow2 ? c : D == 64 ? c ^ ((r >> 1) & 7) : c ^ (r & 15);
  }
  static __device__ __forceinline__ int v_chunk(int r, int c) {
    return !kPow2 ? c : D == 64 ? c ^ (((r >> 1) & 1) << 2) : c ^ ((r & 3) << 2);
  }
};

// The keys lo .. hi - 1 of one sequence and cache head, on their way into LDS.
// kWhole: a group of 16 keys lies within a page, pages and the way from page to
// page are below 4 GB; a group's address is then the scalar unit's.  Else every
// lane has its own, and reads page 0 in place of one that is none (q's first row
// where the cache has no pages).  kOne: this wave brings keys only or values only,
// whose pointer and offsets are k and koff then.
template <int D, bool kExact, bool kWhole, bool kOne>
struct Feed {
  typedef Geo<D, kExact> G;
  const uint8_t *k, *v;     // slot 0 of page 0 of this head
  const int32_t *table;
  int64_t page_bytes, slot_bytes, cols;
  int n_pages, shift, lo, hi;
  bool near;                // page_bytes and a group's way in a page fit 32 bits
  int bad;                  // this lane met a position without a page
  uint32_t rows;            // row of the group (0..15) of DMA j at bits 4 j
  uint32_t koff[G::NI], voff[G::NI];

  // Where a group of 16 keys lies: page ids (kWhole: one, the scalar unit's, and,
  // once it is there, the group's offset; else a lane's own for each DMA).
  struct Place {
    int32_t id[kWhole ? 1 : G::NI];
    int64_t at;
    int p0;
  };

  __device__ __forceinline__ void init(const Work &w, const G &g, int s, int head, int lane,
                                       bool values = false) {
    k = reinterpret_cast<const uint8_t *>(w.cache.k + int64_t(head) * w.cache.head_stride);
    v = reinterpret_cast<const uint8_t *>(w.cache.v + int64_t(head) * w.cache.head_stride);
    if (kOne && values) k = v;
    table = w.b.pages + int64_t(s) * w.b.pages_stride;
    page_bytes = w.cache.page_stride * 2;
    slot_bytes = w.cache.slot_stride * 2;
    cols = w.b.pages_stride;
    n_pages = w.cache.n_pages;
    if (!kWhole && n_pages == 0) {
      k = v = reinterpret_cast<const uint8_t *>(w.q);
      page_bytes = slot_bytes = 0;
    }
    shift = w.cache.page_shift;
    near = (page_bytes >> 32) == 0 && slot_bytes < (1 << 26);
    const int in_page = min((1 << shift) - 1, 15);
    bad = 0;
    rows = 0;
#pragma unroll
    for (int j = 0; j < G::NI; j++) {
      const int i = 64 * j + lane, r = min(i / g.stride, 15), c = min(i - r * g.stride, g.nch - 1);
      // a row's way within its group's part of a page, where it fits
      const uint32_t row = kWhole ? uint32_t(r) * uint32_t(slot_bytes) + dma_lift(j)
                           : near ? uint32_t(r & in_page) * uint32_t(slot_bytes)
                                  : 0;
      rows |= uint32_t(r) << (4 * j);
      koff[j] = row + 16 * (kOne && values ? G::v_chunk(r, c) : G::k_chunk(r, c));
      voff[j] = row + 16 * G::v_chunk(r, c);
    }
  }
  __device__ __forceinline__ int row_of(int j) const { return int((rows >> (4 * j)) & 15); }
  // All 16 keys from p0 on are among lo .. hi - 1.
  __device__ __forceinline__ bool inside(int p0) const { return p0 >= lo && p0 + 15 < hi; }
  __device__ __forceinline__ int within(int p) const { return min(max(p, lo), hi - 1); }
  // Entry `col` of the page table, by the scalar unit; -1 past its end.
  __device__ __forceinline__ int entry(int64_t col) const {
    return col < cols ? *(const __attribute__((address_space(4))) int32_t *)(uintptr_t)(
                            table + uni(int(col)))
                      : -1;
  }
  // Page ids of the group at p0 (a multiple of 16), on their way.  kNow: they are
  // needed before other loads of this wave have come in, whose wait they would
  // share as vector loads; the scalar unit then brings them page by page.
  template <bool kNow>
  __device__ __forceinline__ Place find(int p0) const {
    Place g;
    g.p0 = p0;
    if constexpr (kWhole) {
      g.id[0] = entry(swamp::page_col(within(p0), shift));
    } else if constexpr (kNow) {
      const int first = within(p0) >> shift, last = within(p0 + 15) >> shift;
#pragma unroll
      for (int j = 0; j < G::NI; j++) g.id[j] = -1;
      for (int c = first; c <= last; c++) {
        const int id = entry(c);
#pragma unroll
        for (int j = 0; j < G::NI; j++)
          if (within(p0 + row_of(j)) >> shift == c) g.id[j] = id;
      }
    } else if (inside(p0) && swamp::page_col_ok(p0, swamp::page_col(p0 + 15, shift), cols)) {
      const int32_t *from = table + swamp::page_col(p0, shift);
#pragma unroll
      for (int j = 0; j < G::NI; j++) g.id[j] = from[uint32_t(row_of(j)) >> shift];
    } else {
      const uint32_t rows = fresh(this->rows);
#pragma unroll
      for (int j = 0; j < G::NI; j++) {
        const int p = within(p0 + int((rows >> (4 * j)) & 15));
        const int64_t col = swamp::page_col(p, shift);
        g.id[j] = swamp::page_col_ok(p, col, cols) ? table[col] : -1;
      }
    }
    return g;
  }
  // The ids are there.
  __device__ __forceinline__ void arrive(Place &g) {
    if constexpr (kWhole) {
      const uint32_t slot = uint32_t(within(g.p0)) & ((1u << shift) - 16);
      g.at = int64_t(uint64_t(uint32_t(g.id[0])) * uint32_t(page_bytes) +
                     uint64_t(slot) * uint32_t(slot_bytes));
      bad |= swamp::page_ok(g.id[0], n_pages) ? 0 : 1;
    } else {
#pragma unroll
      for (int j = 0; j < G::NI; j++) {
        const bool ok = swamp::page_ok(g.id[j], n_pages);
        bad |= ok ? 0 : 1;
        if (!ok) g.id[j] = 0;
      }
    }
  }
  // DMAs of the group's keys (kK) or values to LDS; kWhole: none without a page
  // (the result is NaN then).
  template <bool kK>
  __device__ __forceinline__ void issue(const Place &g, uint32_t to) {
    const uint8_t *base = kK || kOne ? k : v;
    const uint32_t *off = kK || kOne ? koff : voff;
    if constexpr (kWhole) {
      if (!swamp::page_ok(g.id[0], n_pages)) return;
      if (inside(g.p0)) {
        dma_uniform<G::NI>(base + g.at, off, to);
        return;
      }
      const uint32_t rows = fresh(this->rows);
      const int first = within(g.p0) & ~15;
      uint32_t moved[G::NI];
#pragma unroll
      for (int j = 0; j < G::NI; j++) {
        const int r = (rows >> (4 * j)) & 15;
        moved[j] = off[j] + uint32_t(within(g.p0 + r) - first - r) * uint32_t(slot_bytes);
      }
      dma_uniform<G::NI>(base + g.at, moved, to);
    } else {
      const int in_page = (1 << shift) - 1;
      if (near && inside(g.p0)) {
        const uint8_t *first = base + (g.p0 & in_page) * slot_bytes;
#pragma unroll
        for (int j = 0; j < G::NI; j++)
          dma_lane(first + uint64_t(uint32_t(g.id[j])) * uint32_t(page_bytes) + off[j],
                   to + 1024 * j);
        return;
      }
      const uint32_t rows = fresh(this->rows);
#pragma unroll
      for (int j = 0; j < G::NI; j++) {
        const int r = (rows >> (4 * j)) & 15, slot = within(g.p0 + r) & in_page;
        dma_lane(base + g.id[j] * page_bytes + (slot - (near ? r & in_page & 15 : 0)) * slot_bytes +
                     off[j],
                 to + 1024 * j);
      }
    }
  }
};

// ---- one wave's 32 rows ---------------------------------------------------
template <typename CT, int D, bool kExact, int NP>
struct Rows {
  typedef Geo<D, kExact> G;
  typedef Op<CT> O;
  // Weights are 2^(c s - m).  A tile that moves m puts it kLift below its largest
  // score, and its largest may pass that by kSlack.
  //
  // fp16 has no step below 2^-24, so that a weight loses bits below 2^-14, or with
  // two parts, whose second begins 11 bits down, below 2^-3.  Weights are lifted to
  // the top of its range, 2^15; and where a tile's largest would be lifted by less
  // than kLift - kFall, m falls to it, or the many small weights of a row whose first
  // key takes nearly all would lose them (one 16 nats above 3000 others, of a value
  // of 0: the result off by 6% without either, at 18 all of it gone).  What a weight
  // loses is then 2^-25 against its own tile's largest, 2^(kLift - kFall) at least:
  // 2^-24 of it, with two parts 2^-31.  l and o grow where m falls: it falls no
  // further than takes l to 2^kTop, and o, 2^16 times that at most, stays within fp32.
  // Scores have their own rounding, 2^-24 of them: m keeps clear of the range's end
  // by that much (scores of 2^24 and more; from 2^25 on the range is too short to
  // hold it and weights lose bits again).
  static constexpr bool kNarrow = O::kNarrow;
  static constexpr float kLift = !kNarrow ? 0.f : NP > 1 ? 14.f : 7.f;
  static constexpr float kSlack = kNarrow && NP > 1 ? 0.f : 8.f;
  static constexpr float kFall = 8.f, kTop = 80.f;

  s16x8 q[G::KS];
  f32x16 o[G::DB];
  float m, l, c;
  int lo, hi;  // keys that this lane's row sees
  uint32_t k_at, v_at;  // LDS offsets of this lane's part of a fragment

  __device__ __forceinline__ void addresses(const G &g, int lane) {
    const int r = lane & 15, half = lane >> 5;
    k_at = ((lane >> 4) & 1) * G::kGroup + 16 * (r * g.stride + G::k_chunk(r, half));
    const int vr = 4 * half + ((lane & 15) >> 2);  // and vr + 8, with the same swizzle
    v_at = 16 * (vr * g.stride + G::v_chunk(vr, ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1))) +
           (lane & 1) * 8;
  }
  // Step ks of the scores, block db of the values.  The swizzles leave their
  // bits to an exclusive or (buffers begin at multiples of 1 KB).
  static __device__ __forceinline__ s16x8 k_frag(uint32_t at, int ks, int kb) {
    return G::kPow2 ? lds16(at ^ (32 * ks), kb * 2 * G::kGroup)
                    : lds16(at, 32 * ks + kb * 2 * G::kGroup);
  }
  static __device__ __forceinline__ s16x8 v_frag(const G &g, uint32_t at, int db, int kg) {
    const uint32_t x = G::kPow2 ? at ^ (64 * db) : at;
    const uint32_t off = kg * G::kGroup + (G::kPow2 ? 0 : 64 * db);
    const s16x4 a = lds_tr(x, off);
    const s16x4 b = kExact ? lds_tr(x, off + 128 * G::kStride) : lds_tr(x + 128 * g.stride, off);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }

  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int db = 0; db < G::DB; db++)
#pragma unroll
      for (int i = 0; i < 16; i++) o[db][i] = 0.f;
  }

  // q's row as B operand; a negative scale goes into its signs.
  __device__ __forceinline__ void load_q(const G &g, const uint16_t *row, float scale, int lane) {
    c = fmaxf(fabsf(scale) * kLog2e, 1e-37f);  // 0 would make NaN of a hidden key's -inf
    // (the scalar unit's where vector registers are few; prompts of 64 dims lose by it,
    // 85 us and 88)
    if constexpr (D >= 128) c = uni(c);
    const short sign = scale < 0.f ? short(0x8000) : short(0);
#pragma unroll
    for (int ks = 0; ks < G::KS; ks++) {
      const int ch = 2 * ks + (lane >> 5);
      s16x8 x = {0, 0, 0, 0, 0, 0, 0, 0};
      if (ch < g.nch) {
        x = *reinterpret_cast<const s16x8 *>(row + 8 * ch);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] ^= sign;
      }
      q[ks] = x;
    }
#ifdef __HIP_DEVICE_COMPILE__
    // (above 128 dims in accumulator registers, where products read it as well: with
    // the sums they are more than half of those)
    if constexpr (D > 128) {
#pragma unroll
      for (int ks = 0; ks < G::KS; ks++) asm volatile("" : "+a"(q[ks]));
    }
#endif
  }

  // Scores of KB x 32 keys in LDS at k.
  template <int KB>
  __device__ __forceinline__ void scores(const G &g, uint32_t k, f32x16 *s, int lane) const {
#pragma unroll
    for (int kb = 0; kb < KB; kb++)
#pragma unroll
      for (int i = 0; i < 16; i++) s[kb][i] = 0.f;
    const uint32_t at = k + k_at;
#pragma unroll
    for (int ks = 0; ks < G::KS; ks++) {
#pragma unroll
      for (int kb = 0; kb < KB; kb++) {
        s16x8 a = k_frag(at, ks, kb);
        // past the row's chunks lies the next row, which may hold NaN
        if (!kExact && 2 * ks + (lane >> 5) >= g.nch) a = s16x8{0, 0, 0, 0, 0, 0, 0, 0};
        s[kb] = O::mma(a, q[ks], s[kb]);
      }
    }
    // fragments are read kAhead products before their own
    constexpr int kAhead = 4;
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);  // LDS reads
#pragma unroll
    for (int i = 0; i < KB * G::KS - kAhead; i++) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix product
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
  }

  // Keys from position p on that this row does not see: score -infinity.
  template <int KB>
  __device__ __forceinline__ void hide(f32x16 *s, int p, int lane) const {
    const uint32_t first = uint32_t(p + 4 * (fresh(lane) >> 5) - lo), n = uint32_t(max(hi - lo, 0));
#pragma unroll
    for (int kb = 0; kb < KB; kb++)
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (first + uint32_t(32 * kb + 8 * (i >> 2) + (i & 3)) >= n) s[kb][i] = -INFINITY;
  }
  // c times the row's largest score, from the two halves' largest.
  __device__ __forceinline__ float join_halves(float top) const {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top),
                                                       false, false);
    return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1])) * c;
  }
  // Some row's m has to follow a tile with the largest scores top.
  __device__ __forceinline__ bool falls(float top) const {
    return kNarrow && top < m + (kLift - kFall);
  }
  __device__ __forceinline__ bool moves(float top) const {
    const float most = m + (kLift + kSlack);
    return __any(top > (kNarrow ? __builtin_fmaf(fabsf(m), -0x1p-22f, most) : most) || falls(top));
  }
  // Where it goes.
  __device__ __forceinline__ float follow(float top) const {
    if (!kNarrow) return fmaxf(m, top);
    const float at = top == -INFINITY ? top : __builtin_fmaf(fabsf(top), 0x1p-23f, top - kLift);
    const float room = kTop - float(__builtin_amdgcn_frexp_expf(sum()));
    return fmaxf(at, falls(top) ? m - fmaxf(room, 0.f) : m);
  }
  // m follows; l and o with it.
  __device__ __forceinline__ void move(float top) {
    if (moves(top)) {
      const float to = follow(top), base = to == -INFINITY ? 0.f : to;
      const float keep = __builtin_amdgcn_exp2f(m - base);
      m = to;
      l *= keep;
#pragma unroll
      for (int db = 0; db < G::DB; db++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[db][i] *= keep;
    }
  }
  template <int KB>
  __device__ __forceinline__ float largest(const f32x16 *s) const {
    float top = s[0][0];
#pragma unroll
    for (int e = 1; e < 16 * KB; e++) top = fmaxf(top, s[e >> 4][e & 15]);
    return join_halves(top);
  }
  __device__ __forceinline__ float base_of() const { return m == -INFINITY ? 0.f : m; }

  // Weights 2 j and 2 j + 1 of the group kg, in three stages, so that none waits for
  // the one before it where steps take them in turn: x = c s - base, ...
  __device__ __forceinline__ void weigh_in(const f32x16 *s, int kg, int j, float base,
                                           float *x) const {
#pragma unroll
    for (int i = 0; i < 2; i++)
      x[i] = fresh(__builtin_fmaf(s[kg >> 1][8 * (kg & 1) + 2 * j + i], c, -base));
  }
  // ... 2^x, ...
  static __device__ __forceinline__ void weigh_up(float *x) {
#pragma unroll
    for (int i = 0; i < 2; i++) x[i] = fresh(__builtin_amdgcn_exp2f(x[i]));
  }
  // ... and its parts in the group's operands p: the nearest of the cache's type and,
  // where the output is fp32, what is left of the weight, again and again.  (fresh:
  // not moved to where they are used, past the products that hide this.)
  __device__ __forceinline__ void weigh_out(const float *x, int j, u32x4 *p) {
    typedef typename O::v2 v2;
    f32x2 r = {x[0], x[1]};
    l += r[0];
    l += r[1];
#pragma unroll
    for (int n = 0; n < NP; n++) {
      const v2 h = __builtin_convertvector(r, v2);
      p[n][j] = __builtin_bit_cast(uint32_t, h);
      if (n + 1 < NP) r -= f32x2{float(h[0]), float(h[1])};
    }
#pragma unroll
    for (int n = 0; n < NP; n++) p[n][j] = fresh(p[n][j]);
    l = fresh(l);
  }
  // Groups from kg0 on, their pairs of weights counted through: what step f of kSteps
  // does for kPairs of them (steps up to kSteps + 1 finish the last).
  template <int kPairs, int kSteps>
  __device__ __forceinline__ void weigh_step(const f32x16 *s, int kg0, int f, float base,
                                             float (*x)[2], u32x4 (*p)[NP]) {
    auto first = [](int g) { return g < 0 ? 0 : g > kSteps ? kPairs : kPairs * g / kSteps; };
#pragma unroll
    for (int q = first(f - 2); q < first(f - 1); q++) weigh_out(x[q], q & 3, p[kg0 + (q >> 2)]);
#pragma unroll
    for (int q = first(f - 1); q < first(f); q++) weigh_up(x[q]);
#pragma unroll
    for (int q = first(f); q < first(f + 1); q++) weigh_in(s, kg0 + (q >> 2), q & 3, base, x[q]);
  }
  // A tile of 32 keys after its scores and move(): weights, and o = o + V^T P^T
  // over the values in LDS at v.  A step is one block of dims of one group of 16
  // keys: its product, the read of the values four steps on, and a share of the
  // next group's weights, which the matrix pipe's time hides.
  __device__ __forceinline__ void rest(const G &g, uint32_t v, const f32x16 *s) {
    constexpr int kSteps = 2 * G::DB, kRing = 4, kIn = G::DB > 2 ? G::DB - 2 : 1;
    const float base = base_of();
    const uint32_t at = v + v_at;
    s16x8 ring[kRing];
    u32x4 p[2][NP];
#pragma unroll
    for (int f = 0; f < kRing; f++)
      if (f < kSteps) ring[f] = v_frag(g, at, f % G::DB, f / G::DB);
    float x[4][2], y[4][2];
#pragma unroll
    for (int f = 0; f < 3; f++) weigh_step<4, 1>(s, 0, f, base, x, p);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int f = 0; f < kSteps; f++) {
      const int kg = f / G::DB;
#pragma unroll
      for (int n = 0; n < NP; n++)
        o[f % G::DB] = O::mma(ring[f % kRing], __builtin_bit_cast(s16x8, p[kg][n]), o[f % G::DB]);
      if (f + kRing < kSteps)
        ring[f % kRing] = v_frag(g, at, (f + kRing) % G::DB, (f + kRing) / G::DB);
      if (kg == 0) weigh_step<4, kIn>(s, 1, f, base, y, p);
      if (f + 1 == G::DB) {
#pragma unroll
        for (int h = G::DB; h < kIn + 2; h++) weigh_step<4, kIn>(s, 1, h, base, y, p);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // ---- scores a tile ahead of the sums (attn_many_kernel) ----
  // p holds a tile's weights; those of its last group are made with the next
  // tile's scores (KB 2: from the half of s that the first products leave alone).

  // Scores of the tile whose keys are in LDS at k; kPending: and the last group
  // of the tile before.
  template <int KB, bool kPending>
  __device__ __forceinline__ void scores_ahead(const G &g, uint32_t k, f32x16 *s, u32x4 (&p)[2 * KB][NP],
                                               float base, int lane) {
    constexpr int kSteps = KB * G::KS, kRing = 4;
    const uint32_t at = k + k_at;
    s16x8 ring[kRing];
    f32x16 other = {};
    float w[4][2];
#pragma unroll
    for (int f = 0; f < kRing; f++) ring[f] = k_frag(at, f % G::KS, f / G::KS);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int f = 0; f < kSteps; f++) {
      const int kb = f / G::KS, ks = f % G::KS;
      s16x8 a = ring[f % kRing];
      if (!kExact && 2 * ks + (lane >> 5) >= g.nch) a = s16x8{0, 0, 0, 0, 0, 0, 0, 0};
      // (KB 1: one wave a SIMD, so that a chain of products each on the last's
      // result would leave the pipe idle: two chains)
      if (KB == 1 && ks % 2 == 1) other = O::mma(a, q[ks], ks == 1 ? f32x16{} : other);
      else s[kb] = O::mma(a, q[ks], ks == 0 ? f32x16{} : s[kb]);
      if (f + kRing < kSteps)
        ring[f % kRing] = k_frag(at, (f + kRing) % G::KS, (f + kRing) / G::KS);
      // (weigh_in reads s[1], whose own products begin at step KS)
      if (KB == 2 && kPending && f < G::KS + 2) weigh_step<4, G::KS>(s, 3, f, base, w, p);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (KB == 1) {
#pragma unroll
      for (int i = 0; i < 16; i++) s[0][i] += other[i];
    }
  }
  // The maximum over the scores s, then the weights of all groups but a pending
  // one; kSums: while o = o + V^T P^T runs with the weights in p, which the new
  // ones replace group by group.
  template <int KB, bool kSums>
  __device__ __forceinline__ void weigh_ahead(const G &g, uint32_t v, const f32x16 *s,
                                              u32x4 (&p)[2 * KB][NP], float &base) {
    constexpr int kSteps = 2 * KB * G::DB, kRing = 4;
    const uint32_t at = v + v_at;
    s16x8 ring[kRing];
    if (kSums) {
#pragma unroll
      for (int f = 0; f < kRing; f++)
        if (f < kSteps) ring[f] = v_frag(g, at, f % G::DB, f / G::DB);
    }
    // of all groups but the last, each behind the sums that its old weights are for
    constexpr int kPairs = KB == 2 ? 12 : 4;
    float top = s[0][0], keep = 1.f, w[kPairs][2];
    bool moved = false;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int f = 0; f < kSteps; f++) {
      const int kg = f / G::DB, db = f % G::DB;
      if (kSums) {
#pragma unroll
        for (int n = 0; n < NP; n++)
          o[db] = O::mma(ring[f % kRing], __builtin_bit_cast(s16x8, p[kg][n]), o[db]);
        if (f + kRing < kSteps)
          ring[f % kRing] = v_frag(g, at, (f + kRing) % G::DB, (f + kRing) / G::DB);
      }
      if (kg == 0) {
#pragma unroll
        for (int e = 16 * KB * db / G::DB; e < 16 * KB * (db + 1) / G::DB; e++)
          top = fmaxf(top, s[e >> 4][e & 15]);
        if (db + 1 == G::DB) {
          top = join_halves(top);
          moved = moves(top);
          const float to = moved ? follow(top) : m;
          base = to == -INFINITY ? 0.f : to;
          keep = __builtin_amdgcn_exp2f(m - base);
          m = to;
          l *= keep;
        }
      } else {
        weigh_step<kPairs, kSteps - G::DB>(s, 0, f - G::DB, base, w, p);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int f = kSteps - G::DB; f < kSteps - G::DB + 2; f++)
      weigh_step<kPairs, kSteps - G::DB>(s, 0, f, base, w, p);
    if (KB == 1) {
#pragma unroll
      for (int f = 0; f < 3; f++) weigh_step<4, 1>(s, 1, f, base, w, p);
    }
    if (kSums && moved) {
#pragma unroll
      for (int db = 0; db < G::DB; db++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[db][i] *= keep;
    }
    if (kSums) stay();
  }
  // Sums of heads above 128 dims keep to the accumulator registers: with the rest
  // they would not fit, and the compiler moves all of them forth and back.
  __device__ __forceinline__ void stay() {
#ifdef __HIP_DEVICE_COMPILE__
    if constexpr (D > 128) {
#pragma unroll
      for (int db = 0; db < G::DB; db++) asm volatile("" : "+a"(o[db]));
    }
#endif
  }
  // The last tile's sums.
  template <int KB>
  __device__ __forceinline__ void sums(const G &g, uint32_t v, const f32x16 *s,
                                       u32x4 (&p)[2 * KB][NP], float base) {
    const uint32_t at = v + v_at;
    float w[4][2];
    if (KB == 2) {
#pragma unroll
      for (int f = 0; f < 3; f++) weigh_step<4, 1>(s, 3, f, base, w, p);
    }
#pragma unroll
    for (int f = 0; f < 2 * KB * G::DB; f++) {
      const int kg = f / G::DB, db = f % G::DB;
      const s16x8 vf = v_frag(g, at, db, kg);
#pragma unroll
      for (int n = 0; n < NP; n++)
        o[db] = O::mma(vf, __builtin_bit_cast(s16x8, p[kg][n]), o[db]);
    }
  }

  // Bit 15 of every 16-bit half whose exponent is all ones.
  static __device__ __forceinline__ uint32_t odd_halves(uint32_t x) {
    constexpr uint32_t e = uint32_t(O::kExp) * 0x10001u, one = e & ~(e << 1);
    return ((x & e) + one) & 0x80008000u;
  }
  // The values that are not finite among the 16 keys of the group in LDS at v:
  // whether there are any (uniform).
  __device__ __forceinline__ bool odd_values(const G &g, uint32_t v, int lane) const {
    uint32_t odd = 0;
    lane = fresh(lane);
    for (int i = lane; i < 16 * g.stride; i += 64) {
      if (!G::kPow2 && i % g.stride >= g.nch) continue;
      const u32x4 x = __builtin_bit_cast(u32x4, lds16(v + 16 * i));
#pragma unroll
      for (int j = 0; j < 4; j++) odd |= odd_halves(x[j]);
    }
    return __any(odd != 0);
  }
  // Adds them to the rows that see them (y less its nearest finite value: 0 for
  // all others); p: position of the group's first key.
  __device__ __forceinline__ void add_odd_values(const G &g, uint32_t v, int p, int lane) {
    lane = fresh(lane);
    for (int r = 0; r < 16; r++) {
      if (p + r < lo || p + r >= hi) continue;
#pragma unroll
      for (int db = 0; db < G::DB; db++) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int d = 32 * db + 8 * i + 4 * (lane >> 5);
          if (!g.within(d)) continue;
          const uint32_t at = v + 16 * (r * g.stride + G::v_chunk(r, d >> 3)) + 2 * (d & 7);
          const s16x4 x = *(__attribute__((address_space(3))) s16x4 *)(uintptr_t)at;
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const short e = x[j];  // (a bit cast of x[j] itself takes element 0)
            const float y = float(__builtin_bit_cast(CT, e));
            o[db][4 * i + j] += y - __builtin_amdgcn_fmed3f(y, -O::kMax, O::kMax);
          }
        }
      }
    }
  }
  // ... and puts 0 in their place.
  __device__ __forceinline__ void clear_odd_values(const G &g, uint32_t v, int lane) const {
    lane = fresh(lane);
    for (int i = lane; i < 16 * g.stride; i += 64) {
      u32x4 x = __builtin_bit_cast(u32x4, lds16(v + 16 * i));
#pragma unroll
      for (int j = 0; j < 4; j++) x[j] &= ~((odd_halves(x[j]) >> 15) * 0xFFFFu);
      lds16_put(v + 16 * i, __builtin_bit_cast(s16x8, x));
    }
  }

  // An infinity or NaN among the sums of a row (dims below dim).
  __device__ __forceinline__ bool not_finite(const G &g, int lane) const {
    float z = 0.f;
#pragma unroll
    for (int db = 0; db < G::DB; db++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int d = 32 * db + 8 * (i >> 2) + 4 * (lane >> 5);
        if (g.within(d)) z = __builtin_fmaf(o[db][i], 0.f, z);
      }
    return z != 0.f;
  }
  // l of both halves.
  __device__ __forceinline__ float sum() const {
    const auto both =
        __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    return __uint_as_float(both[0]) + __uint_as_float(both[1]);
  }
};

__device__ __forceinline__ void put4(const Work &w, int64_t row, int head, int dim, int d, f32x4 x) {
  const int64_t at = row * w.out_stride + int64_t(head) * dim + d;
  if (w.out_type == SWAMP_F32) {
    *reinterpret_cast<f32x4 *>(static_cast<float *>(w.out) + at) = x;
  } else if (w.out_type == SWAMP_F16) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<h4 *>(static_cast<_Float16 *>(w.out) + at) = __builtin_convertvector(x, h4);
  } else {
    typedef __bf16 b4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<b4 *>(static_cast<__bf16 *>(w.out) + at) = __builtin_convertvector(x, b4);
  }
}

// Sequence and block of the unit `at`: sequences 64 at a time, a lane each.
__device__ __forceinline__ bool find_block(const Work &w, int at, int &s, int &blk, int lane) {
  if (w.one_block) {
    s = at;
    blk = 0;
    return s < w.b.n_seq;
  }
  for (int s0 = 0; s0 < w.b.n_seq; s0 += 64) {
    int n = 0;
    if (s0 + lane < w.b.n_seq) {
      const swamp::Seq q = swamp::seq_of(w.b.first[s0 + lane], w.b.first[s0 + lane + 1], 0, w.b.n_tok);
      n = int((int64_t(q.n) * w.group + kRows - 1) / kRows);
    }
    int upto = n;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int x = __shfl_up(upto, off, 64);
      if (lane >= off) upto += x;
    }
    const uint64_t past = __ballot(upto > at);
    if (past) {
      const int who = __builtin_ctzll(past);
      s = s0 + who;
      blk = at - (__shfl(upto, who, 64) - __shfl(n, who, 64));
      return true;
    }
    at -= __shfl(upto, 63, 64);
  }
  return false;
}

// ---- a workgroup's share ---------------------------------------------------
// Rows r0 .. r0 + rows - 1 of a sequence and cache head (row r: new token r /
// group, head r % group), and a piece of the keys that they see.
struct Piece {
  swamp::Seq sq;
  int64_t r0;
  int rows;
  int before;       // position of the first new token
  int begin, end;   // keys of the piece
  int tile0, stop;  // where its tiles begin; no tile begins at or past stop
  bool over;        // the rows see positions that the page table cannot hold

  __device__ __forceinline__ int64_t token(int64_t r, int group) const { return sq.t0 + r / group; }
  __device__ __forceinline__ swamp::Span seen(int64_t r, const Work &w) const {
    return swamp::seen_by(before + int(r / w.group), w.window);
  }
};

// False: no rows, or no keys in this piece (its statistics are written here).
__device__ __forceinline__ bool find_piece(const Work &w, int s, int64_t r0, int max_rows,
                                           int split, int head, Piece &p) {
  p.sq = swamp::seq_of(w.b.first[s], w.b.first[s + 1], w.b.len[s], w.b.n_tok);
  const int64_t n_rows = int64_t(p.sq.n) * w.group;
  p.r0 = r0;
  if (r0 >= n_rows) return false;
  p.rows = int(min(n_rows - r0, int64_t(max_rows)));
  p.before = p.sq.len - p.sq.n;
  const swamp::Span ka = p.seen(r0, w), kz = p.seen(r0 + p.rows - 1, w);
  const int64_t room = swamp::walked(w.b.pages_stride, w.cache.page_shift);
  const int last = int(min(int64_t(kz.hi), room));
  const int64_t from = (ka.lo & ~(kTile - 1)) + int64_t(split) * w.chunk;
  p.over = kz.hi > room;
  p.begin = int(min(max(int64_t(ka.lo), from), int64_t(last)));
  p.end = split == w.splits - 1 ? last : int(min(from + w.chunk, int64_t(last)));
  p.tile0 = p.begin & ~(kTile - 1);
  p.stop = p.end > p.begin ? p.end : p.tile0;
  if (w.splits > 1 && p.stop == p.tile0 && !p.over) {
    for (int i = int(threadIdx.x); i < p.rows; i += kThreads) {
      const int64_t r = r0 + i, t = p.token(r, w.group);
      const swamp::Span seen = p.seen(r, w);
      w.stat[(int64_t(split) * w.b.n_tok + t) * w.n_heads + head * w.group + int(r % w.group)] =
          f32x2{-INFINITY, seen.hi > seen.lo ? 0.f : -1.f};
    }
    return false;
  }
  return true;
}

// Blocks of up to kFew rows: the four waves share the rows, and each takes its
// own 32-key tiles through its own quarter of LDS (K: 2 groups, V: 2 groups).
// No barrier: a wave waits for its own DMAs only; K of the next tile is on its
// way from the end of the scores, V from the end of the sums.
// A wave has a tile of K and one of V on their way, 8 KB each of 128 dims, a CU's four
// waves up to 64 KB: one token over 131072 keys, one workgroup a CU, 98 us; 64 ragged
// sequences of up to 8192 in 2048 workgroups 225 us.
template <typename CT, int D, bool kExact, bool kWhole, int NP>
__global__ void __launch_bounds__(kThreads, D <= 128 ? 2 : 1) attn_few_kernel(Work w) {
  typedef Geo<D, kExact> G;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int tid = int(threadIdx.x), lane = tid & 63, wave = uni(tid >> 6);
  const uint32_t lds = lds_base(smem), extra = lds + G::kSmem;
  const G g(w.cache.dim);
  const int dim = kExact ? D : w.cache.dim;
  const int head = int(blockIdx.x) % w.cache.n_kv, unit = int(blockIdx.x) / w.cache.n_kv;
  const int split = unit % w.splits, s = unit / w.splits;
  Piece pc;
  if (!find_piece(w, s, 0, kFew, split, head, pc)) return;

  const int64_t rr = min(lane & 31, pc.rows - 1);
  const int hq = head * w.group + int(rr % w.group);
  const int64_t t = pc.token(rr, w.group);
  Rows<CT, D, kExact, NP> a;
  a.addresses(g, lane);
  a.load_q(g, w.q + t * w.q_stride + int64_t(hq) * dim, w.scale, lane);
  const swamp::Span mine = pc.seen(rr, w);
  a.lo = max(mine.lo, pc.begin);
  a.hi = min(mine.hi, pc.end);
  const int all_lo = max(pc.seen(pc.rows - 1, w).lo, pc.begin);
  const int all_hi = min(pc.seen(0, w).hi, pc.end);
  typedef Feed<D, kExact, kWhole, false> F;
  F f;
  f.init(w, g, s, head, lane);
  f.bad = pc.over;
  f.lo = pc.begin;
  f.hi = pc.end;

  const uint32_t at_k = lds + wave * (G::kSmem / kWaves), at_v = at_k + 2 * G::kGroup;
  bool bad = false;
  for (int safe = 0; safe < 2; safe++) {
    a.clear();
    // (fresh, or the first tile's addresses are kept for the second pass)
    int p = uni(fresh(pc.tile0 + 32 * wave));
    typename F::Place at[2];
    if (p < pc.stop) {
#pragma unroll
      for (int i = 0; i < 2; i++) at[i] = f.template find<true>(p + 16 * i);
#pragma unroll
      for (int i = 0; i < 2; i++) {
        f.arrive(at[i]);
        f.template issue<true>(at[i], at_k + i * G::kGroup);
      }
#pragma unroll
      for (int i = 0; i < 2; i++) f.template issue<false>(at[i], at_v + i * G::kGroup);
    }
    while (p < pc.stop) {
      const int next = p + 32 * kWaves;
      const bool more = next < pc.stop;
      if (more) {
#pragma unroll
        for (int i = 0; i < 2; i++) at[i] = f.template find<true>(next + 16 * i);
      }
      f32x16 sc[1];
      wait_dma<2 * G::NI>();
      a.template scores<1>(g, at_k, sc, lane);
      lds_done();
      if (more) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
          f.arrive(at[i]);
          f.template issue<true>(at[i], at_k + i * G::kGroup);
        }
      }
      if (p < all_lo || p + 32 > all_hi) a.template hide<1>(sc, p, lane);
      a.move(a.template largest<1>(sc));
      if (more) wait_dma<2 * G::NI>();
      else wait_dma<0>();
      if (safe) {
        for (int i = 0; i < 2; i++)
          if (a.odd_values(g, at_v + i * G::kGroup, lane)) {
            a.add_odd_values(g, at_v + i * G::kGroup, p + 16 * i, lane);
            lds_done();
            a.clear_odd_values(g, at_v + i * G::kGroup, lane);
            lds_done();
          }
      }
      a.rest(g, at_v, sc);
      lds_done();
      if (more) {
#pragma unroll
        for (int i = 0; i < 2; i++) f.template issue<false>(at[i], at_v + i * G::kGroup);
      }
      p = next;
    }
    bad = __any(f.bad);
    if (bad || !__any(a.not_finite(g, lane))) break;
  }

  // the waves' sums meet in LDS, rows of dim floats (16-byte chunks swizzled by
  // the row where there are enough of them)
  const float l = bad ? __builtin_nanf("") : a.sum();
  const uint32_t flip = dim % 32 == 0 ? 7 : 0;
  const uint32_t mine_at = lds + wave * (G::kSmem / kWaves);
  const int r = lane & 31;
  if (lane < 32) {
    ldsf_put(extra + 8 * (32 * wave + r), a.m);
    ldsf_put(extra + 8 * (32 * wave + r) + 4, l);
  }
  if (r < pc.rows) {
#pragma unroll
    for (int db = 0; db < G::DB; db++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int d = 32 * db + 8 * i + 4 * (lane >> 5);
        if (d < dim)
          ldsf4_put(mine_at + 4 * r * dim + 16 * ((d >> 2) ^ (r & flip)),
                    f32x4{a.o[db][4 * i], a.o[db][4 * i + 1], a.o[db][4 * i + 2],
                          a.o[db][4 * i + 3]});
      }
  }
  if (bad && w.b.bad && lane == 0) *w.b.bad = 1;
  __syncthreads();
  const int per = dim >> 2;
  for (int i = tid; i < pc.rows * per; i += kThreads) {
    const int row = i / per, d = 4 * (i - row * per);
    float mw[kWaves], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int x = 0; x < kWaves; x++) {
      mw[x] = ldsf(extra + 8 * (32 * x + row));
      top = fmaxf(top, mw[x]);
    }
    const float base = top == -INFINITY ? 0.f : top;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < kWaves; x++) {
      const float k = __builtin_amdgcn_exp2f(mw[x] - base);
      sum += k * ldsf(extra + 8 * (32 * x + row) + 4);
      if (mw[x] != -INFINITY)
        acc += k * ldsf4(lds + x * (G::kSmem / kWaves) + 4 * row * dim +
                         16 * ((d >> 2) ^ (row & flip)));
    }
    const int64_t to = pc.token(row, w.group);
    const int h = head * w.group + row % w.group;
    const swamp::Span seen = pc.seen(row, w);
    const bool sees = seen.hi > seen.lo;
    if (w.splits == 1) {
      put4(w, to, h, dim, d, sees ? acc * (1.f / sum) : f32x4{0.f, 0.f, 0.f, 0.f});
    } else {
      const int64_t pr = (int64_t(split) * w.b.n_tok + to) * w.n_heads + h;
      *reinterpret_cast<f32x4 *>(w.part + pr * dim + d) = acc;
      if (d == 0) w.stat[pr] = f32x2{top, sees ? sum : -1.f};
    }
  }
}

// Blocks of up to kRows rows, 32 a wave.  A tile of 32 KB keys is shared, each wave
// brings in a part of it.  Scores run a tile ahead of the sums: while tile i is
// summed and tile i + 1 scored, K of i + 2 and V of i + 1 are on their way, and
// one barrier a tile orders all of it.  K and V have two buffers each.
template <typename CT, int D, bool kExact, bool kWhole, int NP>
__global__ void __launch_bounds__(kThreads, D <= 128 ? 2 : 1) attn_many_kernel(Work w) {
  typedef Geo<D, kExact> G;
  // heads of 256 dims: the sums alone are 128 registers
  constexpr int KB = D <= 128 ? 2 : 1, kKeys = 32 * KB;
  constexpr uint32_t kPart = 2 * KB * G::kGroup;  // K or V of a tile
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int tid = int(threadIdx.x), lane = tid & 63, wave = uni(tid >> 6);
  const uint32_t lds = lds_base(smem), extra = lds + G::kSmem;
  const G g(w.cache.dim);
  const int dim = kExact ? D : w.cache.dim;
  // heads first: eight heads' workgroups keep to one XCD each, whose L2 then
  // holds one head's keys; late blocks, which see the most keys, go first
  const int head = int(blockIdx.x) % w.cache.n_kv, unit = int(blockIdx.x) / w.cache.n_kv;
  const int split = unit % w.splits;
  int s, blk;
  if (!find_block(w, w.blocks - 1 - unit / w.splits, s, blk, lane)) return;
  s = uni(s);
  blk = uni(blk);
  Piece pc;
  if (!find_piece(w, s, int64_t(blk) * kRows, kRows, split, head, pc)) return;

  // this lane's row
  const bool store = 32 * wave + (lane & 31) < pc.rows;
  const int64_t rr = pc.r0 + min(32 * wave + (lane & 31), pc.rows - 1);
  const int hq = head * w.group + int(rr % w.group);
  const int t = int(pc.token(rr, w.group));
  Rows<CT, D, kExact, NP> a;
  a.addresses(g, lane);
  a.load_q(g, w.q + t * w.q_stride + int64_t(hq) * dim, w.scale, lane);
  const swamp::Span mine = pc.seen(rr, w);
  a.lo = max(mine.lo, pc.begin);
  a.hi = min(mine.hi, pc.end);
  // keys that any row of the wave sees, and that all do
  const swamp::Span wa = pc.seen(pc.r0 + min(32 * wave, pc.rows - 1), w);
  const swamp::Span wz = pc.seen(pc.r0 + min(32 * wave + 31, pc.rows - 1), w);
  const int any_lo = max(wa.lo, pc.begin), any_hi = min(wz.hi, pc.end);
  const int all_lo = max(wz.lo, pc.begin), all_hi = min(wa.hi, pc.end);
  typedef Feed<D, kExact, kWhole, KB == 1> F;
  F f;
  f.init(w, g, s, head, lane, wave >= 2);
  f.bad = pc.over;
  f.lo = pc.begin;
  f.hi = pc.end;
  int tile0 = pc.tile0;
  const int n_tiles = (pc.stop - pc.tile0 + kKeys - 1) / kKeys;

  // K and V of tile i.  Tiles of 64 keys: each wave a group of either; of 32: two
  // waves K, two waves V.
  const int part = 16 * (KB == 2 ? wave : wave & 1);
  // Places of the tiles whose K and V are next.  Tiles of 32: a wave brings one of
  // the two and knows `ahead` only, `lead` tiles from the turn's.
  typename F::Place ahead, behind;
  const int lead = KB == 2 || wave < 2 ? 2 : 1;
  const uint32_t part_at = lds + (part >> 4) * G::kGroup;
  auto bring_k = [&](int i) {
    if (KB == 2 || wave < 2) f.template issue<true>(ahead, part_at + (i & 1) * kPart);
  };
  auto bring_v = [&](int i) {
    if (KB == 2) f.template issue<false>(behind, part_at + (2 + (i & 1)) * kPart);
    else if (wave >= 2) f.template issue<false>(ahead, part_at + (2 + (i & 1)) * kPart);
  };
  auto find = [&](int i) { return f.template find<false>(tile0 + i * kKeys + part); };
  auto k_of = [&](int i) { return lds + (i & 1) * kPart; };
  auto v_of = [&](int i) { return lds + (2 + (i & 1)) * kPart; };
  // tiles with keys that rows of this wave see, and of which they see every key
  const int first = any_hi > any_lo ? (any_lo - pc.tile0) / kKeys : n_tiles;
  const int last = any_hi > any_lo ? (any_hi - pc.tile0 + kKeys - 1) / kKeys : n_tiles;
  auto plain = [&](int i) {
    const int p = tile0 + i * kKeys;
    return p >= all_lo && p + kKeys <= all_hi;
  };
  auto run = [&](auto safe) {
    // (nor are the first tile's addresses, or q, kept for the second pass where
    // registers are few)
    if constexpr (decltype(safe)::value && D > 128) {
      tile0 = uni(fresh(tile0));
      a.load_q(g, w.q + fresh(t * w.q_stride + int64_t(hq) * dim), w.scale, lane);
    }
    // (A wave on its way through products goes before one that prepares a tile: 4096
    // tokens over themselves 274 -> 272 us, 512 over 16384 keys 146 -> 141.)
    // Turn i = -1 .. n_tiles - 1: K of tile i + 1 and V of tile i are there, and
    // nobody reads what K of i + 2 and V of i + 1 go over.  ahead = the place of
    // tile i + lead, behind = of i + 1.
    auto turn = [&](int i) {
      wait_all();
      if (i + lead < n_tiles) f.arrive(ahead);
      const typename F::Place then = find(min(i + lead + 1, n_tiles));
      if (i + 2 < n_tiles) bring_k(i + 2);
      if (i + 1 < n_tiles) bring_v(i + 1);
      if (KB == 2) behind = ahead;
      ahead = then;
      if constexpr (decltype(safe)::value) {
        if (i < 0) return;
        const uint32_t v = v_of(i), mine_v = v + (part >> 4) * G::kGroup;
        if (anywhere(a.odd_values(g, mine_v, lane), extra)) {
          for (int j = 0; j < 2 * KB; j++)
            a.add_odd_values(g, v + j * G::kGroup, tile0 + i * kKeys + 16 * j, lane);
          __syncthreads();
          a.clear_odd_values(g, mine_v, lane);
          __syncthreads();
        }
      }
    };
    a.clear();
    if (n_tiles == 0) return;
    ahead = find(0);
    if (lead == 2) {
      f.arrive(ahead);
      bring_k(0);
      if (KB == 2) behind = ahead;
      ahead = find(1);
    }
    int i = -1;
    for (; i + 1 < first; i++) turn(i);
    if (first < last) {
      f32x16 sc[KB];
      u32x4 wt[2 * KB][NP];
      float base = 0.f;
      turn(i);
      a.template scores_ahead<KB, false>(g, k_of(i + 1), sc, wt, base, lane);
      if (!plain(i + 1)) a.template hide<KB>(sc, tile0 + (i + 1) * kKeys, lane);
      a.template weigh_ahead<KB, false>(g, 0, sc, wt, base);
      for (i++; i + 1 < last; i++) {
        turn(i);
        __builtin_amdgcn_s_setprio(1);
        a.template scores_ahead<KB, true>(g, k_of(i + 1), sc, wt, base, lane);
        if (!plain(i + 1)) a.template hide<KB>(sc, tile0 + (i + 1) * kKeys, lane);
        a.template weigh_ahead<KB, true>(g, v_of(i), sc, wt, base);
        __builtin_amdgcn_s_setprio(0);
      }
      turn(i);
      a.template sums<KB>(g, v_of(i), sc, wt, base);
      i++;
    }
    for (; i < n_tiles; i++) turn(i);
  };
  run(std::false_type{});
  const bool bad = anywhere(f.bad, extra);
  if (!bad && anywhere(store && a.not_finite(g, lane), extra)) run(std::true_type{});
  const float l = bad ? __builtin_nanf("") : a.sum();
  if (bad && w.b.bad && tid == 0) *w.b.bad = 1;
  if (!store) return;
  const bool sees = mine.hi > mine.lo;
  const int64_t pr = (int64_t(split) * w.b.n_tok + t) * w.n_heads + hq;
  const float inv = 1.f / l;
  if (w.splits > 1 && lane < 32) w.stat[pr] = f32x2{a.m, sees ? l : -1.f};
#pragma unroll
  for (int db = 0; db < G::DB; db++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int d = 32 * db + 8 * i + 4 * (lane >> 5);
      if (!g.within(d)) continue;
      const f32x4 x = {a.o[db][4 * i], a.o[db][4 * i + 1], a.o[db][4 * i + 2], a.o[db][4 * i + 3]};
      if (w.splits == 1) put4(w, t, hq, dim, d, sees ? x * inv : f32x4{0.f, 0.f, 0.f, 0.f});
      else *reinterpret_cast<f32x4 *>(w.part + pr * dim + d) = x;
    }
}

template <typename CT, int D, bool kExact, bool kWhole, int NP>
void launch_kind(const Work &w, hipStream_t s) {
  typedef Geo<D, kExact> G;
  const dim3 grid(unsigned(w.blocks) * unsigned(w.splits) * unsigned(w.cache.n_kv));  // (kMaxGroups)
  const uint32_t smem = G::kSmem + G::kExtra;
  if (w.few) attn_few_kernel<CT, D, kExact, kWhole, NP><<<grid, kThreads, smem, s>>>(w);
  else attn_many_kernel<CT, D, kExact, kWhole, NP><<<grid, kThreads, smem, s>>>(w);
}

template <typename CT, int D, bool kExact>
int launch(const Work &w, int parts, hipStream_t s) {
  // (heads of other sizes take every lane's own pages: the general form)
  const bool whole = kExact && w.cache.page_shift >= 4 &&
                     w.cache.page_stride < (int64_t(1) << 31) &&
                     (w.cache.slot_stride << w.cache.page_shift) < (int64_t(1) << 30);
  auto go = [&](auto np) {
    if (whole) launch_kind<CT, D, kExact, kExact, decltype(np)::value>(w, s);
    else launch_kind<CT, D, kExact, false, decltype(np)::value>(w, s);
  };
  if (parts == 1) go(std::integral_constant<int, 1>{});
  else if (parts == 2) go(std::integral_constant<int, 2>{});
  else go(std::integral_constant<int, Op<CT>::kParts>{});
  return hipGetLastError() == hipSuccess ? SWAMP_OK : SWAMP_ELAUNCH;
}

template <typename CT>
int launch_dim(const Work &w, int parts, hipStream_t s) {
  switch (w.cache.dim) {
    case 64: return launch<CT, 64, true>(w, parts, s);
    case 80: return launch<CT, 80, true>(w, parts, s);
    case 96: return launch<CT, 96, true>(w, parts, s);
    case 128: return launch<CT, 128, true>(w, parts, s);
    case 256: return launch<CT, 256, true>(w, parts, s);
  }
  return w.cache.dim < 128 ? launch<CT, 128, false>(w, parts, s)
                           : launch<CT, 256, false>(w, parts, s);
}

}  // namespace
