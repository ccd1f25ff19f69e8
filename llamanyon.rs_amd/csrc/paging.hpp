// paging.hpp -- where the tokens of a batch lie: which sequence and position a
// row has, which keys it sees, and the page of a position.  Plain index
// arithmetic, the same source on the device and (without HIP) on the host, so
// that its bounds can be checked without a GPU.
//
// Every index that comes from device memory is checked here before it is used:
// row ranges against n_tok, page-table columns against the table's width and
// page ids against the cache's pages.
#pragma once

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#endif
#include <stddef.h>
#include <stdint.h>

#include "swamp_qmm.h"

#ifdef __HIPCC__
#define SWAMP_HD __host__ __device__ __forceinline__
#else
#define SWAMP_HD inline
#endif

namespace swamp {

// swamp_kv_pages and swamp_seq_batch as the kernels take them: strides filled
// in, the page size as a shift.
struct PagedCache {
  uint16_t *k, *v;
  int64_t page_stride, head_stride, slot_stride;
  int n_pages, page_shift, n_kv, dim;
};
struct SeqBatch {
  const int32_t *first, *len, *pages;
  int64_t pages_stride;
  int32_t *bad;
  int n_seq, n_tok;
};

// swamp_page_pool, swamp_page_tables and swamp_page_moves, checked.
constexpr int kMaxPageSeqs = 2048;
struct PagePool {
  int n_pages, shift;
  int32_t *refs;
  uint32_t *used;
};
struct PageTables {
  int n_seq;
  int32_t *len, *pages;
  int64_t stride;
  int32_t *bad;
};
struct PageMoves {
  int cap;
  int32_t *src, *dst, *count;
};

// One swamp_beam_select call, checked.
struct BeamCall {
  int n_seq, n_beam, vocab, n_out, eos;
  uint32_t type;
  const void *logits;
  int64_t stride;
  const float *score;
  const int32_t *done;
  int32_t *parent, *token;
  float *out_score;
  int32_t *out_done;
};

// One swamp_gemm_rows_i8 call, checked.
struct GemmI8Call {
  const int8_t *x, *w;
  const float *x_scale, *w_scale;
  void *y;
  uint32_t y_type;
  int64_t x_stride, w_stride, y_stride;
  int m, n, k, accumulate;
};

// One swamp_attn_paged call, checked.
struct AttnCall {
  PagedCache cache;
  SeqBatch batch;
  uint32_t dtype, out_type;
  int max_new, max_len, n_heads, window;
  float scale;
  const void *q;
  void *out;
  int64_t q_stride, out_stride;
};

// A sequence's new tokens as rows t0 .. t0 + n - 1 of the batch, and its
// tokens in the cache; ranges that leave the batch or run backwards are cut.
struct Seq {
  int t0, n;
  int len;
};
SWAMP_HD Seq seq_of(int32_t first, int32_t next, int32_t len, int n_tok) {
  Seq s;
  s.t0 = first < 0 ? 0 : first > n_tok ? n_tok : first;
  const int t1 = next > n_tok ? n_tok : next;
  s.n = t1 > s.t0 ? t1 - s.t0 : 0;
  s.len = len < 0 ? 0 : len;
  return s;
}

// Keys lo .. hi - 1 that the row at position pos sees (window 0: all).  pos < 0:
// none.  pos < len <= 2^31 - 1 for every row of a sequence.
struct Span {
  int lo, hi;
};
SWAMP_HD Span seen_by(int pos, int window) {
  Span k;
  k.hi = pos < 0 ? 0 : pos + 1;
  k.lo = window > 0 && k.hi > window ? k.hi - window : 0;
  return k;
}

// The page-table column of position pos, which is a column of the table only
// if page_col_ok says so.
SWAMP_HD int64_t page_col(int pos, int shift) { return int64_t(pos >> shift); }
SWAMP_HD bool page_col_ok(int pos, int64_t col, int64_t pages_stride) {
  return pos >= 0 && col < pages_stride;
}
// Table entries that a sequence of len tokens holds.
SWAMP_HD int64_t held_cols(int len, int shift, int64_t stride) {
  const int64_t n = len <= 0 ? 0 : (int64_t(len) + (int64_t(1) << shift) - 1) >> shift;
  return n < stride ? n : stride;
}
// Element offset of slot 0, dim 0 of `head` at position pos on page id.
SWAMP_HD bool page_ok(int32_t id, int n_pages) { return uint32_t(id) < uint32_t(n_pages); }
SWAMP_HD int64_t slot_offset(int32_t id, int pos, int head, int shift, int64_t page_stride,
                             int64_t head_stride, int64_t slot_stride) {
  return int64_t(id) * page_stride + int64_t(head) * head_stride +
         int64_t(pos & ((1 << shift) - 1)) * slot_stride;
}

}  // namespace swamp
