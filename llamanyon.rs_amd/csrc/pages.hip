// pages.hip -- who holds the pages of a paged cache, and copies of pages: forking
// (swamp_pages_fork), growing (swamp_pages_extend), cutting (swamp_pages_trim),
// compacting (swamp_pages_compact) and swamp_kv_copy.
//
// A page's count is the number of page tables that name it, so a call's results are
// sums and lowest places, which no order of atomics changes.
#include "swamp_common.hpp"
#include "wave.hpp"

#include <algorithm>
#include <mutex>

namespace {

using swamp::held_cols;
using swamp::page_ok;
using swamp::PageMoves;
using swamp::PagePool;
using swamp::PageTables;

constexpr int kSeqs = swamp::kMaxPageSeqs;
constexpr int kTile = 16;     // table columns that a workgroup turns at a time

// ---- fork -----------------------------------------------------------------
// T'[s] = T[parent s], in place: a workgroup takes 16 columns of all rows into LDS.
// A page gains (children of its row) - 1 per row that names it.  Rows that share
// pages lie together and name them in the same column: a thread runs down a column
// and adds a run of equal pages' gains at once, and where a prompt's beams only
// change places the sum is 0 and nothing is written.
//
// A chain of two loads, LDS and stores: 64 sequences of 31 pages 6.3 us, 64 of up to 2048
// 7.1, and 1.6 and 2.2 for the second launch.
//
// kOne: the one workgroup of a small call also does what else comes in a launch of its
// own, when every count is final: which pages are in use, and the lengths (4 sequences of 7
// pages 4.0 us).
template <bool kOne>
__global__ void __launch_bounds__(256) fork_kernel(PagePool pool, PageTables t,
                                                   const int32_t *__restrict__ d_parent) {
  extern __shared__ int smem[];
  const int n = t.n_seq, tid = int(threadIdx.x), c = tid % kTile;
  int *tile = smem, *gain = tile + n * kTile, *lens = gain + n, *parent = lens + n;
  __shared__ int most;
  // the first tile's entries, on their way while lengths and parents come in
  constexpr int kAhead = 8;
  int ahead[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; j++) {
    const int s = j * (256 / kTile) + tid / kTile;
    ahead[j] = s < n ? t.len[s] : 0;
  }
#pragma unroll
  for (int j = 0; j < kAhead; j++) {
    const int s = j * (256 / kTile) + tid / kTile;
    const int64_t col = int64_t(blockIdx.x) * kTile + c;
    ahead[j] = col < held_cols(ahead[j], pool.shift, t.stride) ? t.pages[s * t.stride + col] : -1;
  }
  if (tid == 0) most = 0;
  for (int s = tid; s < n; s += 256) gain[s] = -1;
  __syncthreads();
  int top = 0;
  for (int s = tid; s < n; s += 256) {
    const int p = d_parent[s];
    parent[s] = uint32_t(p) < uint32_t(n) ? p : -1;
    lens[s] = t.len[s];
    top = max(top, int(held_cols(lens[s], pool.shift, t.stride)));
    if (uint32_t(p) < uint32_t(n)) atomicAdd(&gain[p], 1);
  }
  if (top > 0) atomicMax(&most, top);
  __syncthreads();
  const int rows = (n + 15) / 16, r0 = min(tid / kTile * rows, n), r1 = min(r0 + rows, n);
  const int64_t mine = int64_t(blockIdx.x) * kTile;
  for (int64_t c0 = mine; c0 < most; c0 += int64_t(gridDim.x) * kTile) {
    auto held = [&](int s) { return c0 + c < held_cols(lens[s], pool.shift, t.stride); };
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      const int s = j * (256 / kTile) + tid / kTile;
      if (s < n)
        tile[s * kTile + c] = c0 == mine ? ahead[j] : held(s) ? t.pages[s * t.stride + c0 + c] : -1;
    }
    for (int s = kAhead * (256 / kTile) + tid / kTile; s < n; s += 256 / kTile)
      tile[s * kTile + c] = held(s) ? t.pages[s * t.stride + c0 + c] : -1;
    __syncthreads();
    int id = -1, sum = 0;
    for (int s = r0; s < r1; s++) {
      const int e = tile[s * kTile + c];
      if (e != id) {
        if (sum != 0 && page_ok(id, pool.n_pages)) atomicAdd(&pool.refs[id], sum);
        id = e;
        sum = 0;
      }
      sum += gain[s];
    }
    if (sum != 0 && page_ok(id, pool.n_pages)) atomicAdd(&pool.refs[id], sum);
    for (int s = tid / kTile; s < n; s += 256 / kTile) {
      const int p = parent[s];
      if (p != s && p >= 0 && held(p)) t.pages[s * t.stride + c0 + c] = tile[p * kTile + c];
    }
    __syncthreads();
  }
  if constexpr (kOne) {
    __threadfence();
    __syncthreads();
    for (int s = tid; s < n; s += 256) t.len[s] = parent[s] < 0 ? 0 : lens[parent[s]];
    for (int64_t first = 0; first < pool.n_pages; first += 256) {
      const int64_t p = first + tid;
      // (counts as the adds left them, not as a cache may hold them)
      const bool held = p < pool.n_pages && __hip_atomic_load(&pool.refs[p], __ATOMIC_RELAXED,
                                                              __HIP_MEMORY_SCOPE_AGENT) > 0;
      const uint64_t used = __ballot(held);
      if (tid % 32 == 0 && p < pool.n_pages)
        pool.used[p / 32] = uint32_t(tid % 64 ? used >> 32 : used);
    }
  }
}

// Every table and count is final: which pages are in use, and the lengths.
__global__ void __launch_bounds__(256) fork_finish_kernel(PagePool pool, PageTables t,
                                                          const int32_t *__restrict__ d_parent) {
  const int64_t id = int64_t(blockIdx.x) * 256 + threadIdx.x;
  const uint64_t used = __ballot(id < pool.n_pages && pool.refs[id] > 0);
  if (threadIdx.x % 32 == 0 && id < pool.n_pages)
    pool.used[id / 32] = uint32_t(threadIdx.x % 64 ? used >> 32 : used);
  if (blockIdx.x != 0) return;
  __shared__ int lens[kSeqs];
  for (int s = int(threadIdx.x); s < t.n_seq; s += 256) lens[s] = t.len[s];
  __syncthreads();
  for (int s = int(threadIdx.x); s < t.n_seq; s += 256) {
    const int p = d_parent[s];
    t.len[s] = uint32_t(p) < uint32_t(t.n_seq) ? lens[p] : 0;
  }
}

// ---- one workgroup's sums -------------------------------------------------
// The sum of x over the threads before this one, and over all; `part` holds a value
// for each wave and is free again on return.
template <int kBlock>
__device__ __forceinline__ int64_t scan(int64_t x, int64_t *part, int64_t &total) {
  const int lane = int(threadIdx.x) & 63, wave = int(threadIdx.x) >> 6;
  const int64_t incl = swamp::sum_to_here(x);
  if (lane == 63) part[wave] = incl;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kBlock / 64; w++) {
    const int64_t p = part[w];
    if (w < wave) before += p;
    total += p;
  }
  __syncthreads();
  return before + incl - x;
}

// Word w of the pages in use; pages past the last count as used where `fill`.
__device__ __forceinline__ uint32_t used_word(const PagePool &pool, int64_t w, bool fill) {
  const int64_t first = 32 * w;
  if (first >= pool.n_pages) return fill ? ~0u : 0u;
  const int64_t n = pool.n_pages - first;
  const uint32_t there = n >= 32 ? ~0u : (1u << n) - 1, x = pool.used[w];
  return fill ? x | ~there : x & there;
}

constexpr int kWords = 2;  // of a thread in a round, at most

// ---- extend ---------------------------------------------------------------
// One workgroup: what every sequence needs (two a thread), where its pages begin in
// the row of all pages handed out, then one pass over the free pages in rising
// order: a thread a page, which finds the page's word and its owner by bisection.  Of the h
// sequences that would write one shared page in turn, the j-th finds refs - j tables naming
// it.  A chain of loads and sums: 64 sequences of 31 pages take 6.8 us.
template <int kBlock>
__global__ void __launch_bounds__(kBlock) extend_kernel(PagePool pool, PageTables t,
                                                        const int32_t *__restrict__ d_new,
                                                        PageMoves moves, int per) {
  constexpr int kMost = 2 * kBlock;  // sequences
  __shared__ __attribute__((aligned(16))) int tail[kMost];  // the shared page it would write, or -1
  __shared__ int copy[kMost];     // its place in the list, or -1
  __shared__ int first[kMost];    // its first new column
  __shared__ int64_t off[kMost];
  __shared__ uint32_t word[kWords * kBlock];  // free pages of a round's words
  __shared__ int word_at[kWords * kBlock];    // and how many lie before each
  __shared__ int64_t part[kBlock / 64];
  __shared__ int listed;
  const int n = t.n_seq, tid = int(threadIdx.x);
  const int mask = (1 << pool.shift) - 1;
  const int64_t words = (int64_t(pool.n_pages) + 31) / 32;
  uint32_t free[kWords];  // of the first round, on their way
#pragma unroll
  for (int i = 0; i < kWords; i++) free[i] = i < per ? ~used_word(pool, tid * per + i, true) : 0u;
  bool bad = false;
  int refs[2], grown[2], fresh[2];
  if (tid == 0) listed = 0;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int s = 2 * tid + i;
    tail[s] = -1;
    refs[i] = grown[i] = fresh[i] = 0;
    if (s >= n) continue;
    const int len = max(t.len[s], 0);
    const int want = d_new ? max(d_new[s], 0) : 1, more = min(want, INT32_MAX - len);
    const int64_t last = len >> pool.shift;
    const int64_t c0 = (int64_t(len) + mask) >> pool.shift;
    const int64_t c1 = (int64_t(len) + more + mask) >> pool.shift;
    grown[i] = len + more;
    first[s] = int(min(c0, t.stride));
    fresh[i] = int(min(c1, t.stride) - min(c0, t.stride));
    bad |= more > 0 && c1 > t.stride;
    bad |= want > more;
    if (more > 0 && (len & mask) != 0 && last < t.stride) {
      const int id = t.pages[s * t.stride + last];
      if (page_ok(id, pool.n_pages)) {
        refs[i] = pool.refs[id];
        if (refs[i] > 1) tail[s] = id;
      } else {
        bad = true;
      }
    }
  }
  __syncthreads();
  const int mine[2] = {tail[2 * tid], tail[2 * tid + 1]};
  int before[2] = {0, 0}, copies[2];
  if (mine[0] >= 0 || mine[1] >= 0)
#pragma unroll 4
    for (int o = 0; o < 2 * tid; o += 2) {
      const int a = tail[o], b = tail[o + 1];
      before[0] += (a == mine[0] ? 1 : 0) + (b == mine[0] ? 1 : 0);
      before[1] += (a == mine[1] ? 1 : 0) + (b == mine[1] ? 1 : 0);
    }
  before[1] += mine[0] == mine[1] ? 1 : 0;
#pragma unroll
  for (int i = 0; i < 2; i++) copies[i] = mine[i] >= 0 && before[i] < refs[i] - 1 ? 1 : 0;
  // pages in the low 48 bits (2048 times less than 2^31 at most), copies above
  constexpr int kCopy = 48;
  int64_t total;
  int64_t at = scan<kBlock>(int64_t(copies[0]) + fresh[0] + copies[1] + fresh[1] +
                                (int64_t(copies[0] + copies[1]) << kCopy),
                            part, total);
  const int place = int(at >> kCopy);
  at &= (int64_t(1) << kCopy) - 1;
  total &= (int64_t(1) << kCopy) - 1;
  off[2 * tid] = at;
  off[2 * tid + 1] = at + copies[0] + fresh[0];
  copy[2 * tid] = copies[0] ? place : -1;
  copy[2 * tid + 1] = copies[1] ? place + copies[0] : -1;
#pragma unroll
  for (int i = 0; i < 2; i++)
    if (copies[i]) atomicSub(&pool.refs[mine[i]], 1);
  __syncthreads();

  int64_t base = 0;  // free pages before this round's
  for (int64_t w0 = 0; base < total && w0 < words; w0 += kBlock * per) {
    if (w0 > 0)
#pragma unroll
      for (int i = 0; i < kWords; i++)
        free[i] = i < per ? ~used_word(pool, w0 + tid * per + i, true) : 0u;
    int count = 0;
#pragma unroll
    for (int i = 0; i < kWords; i++) count += __builtin_popcount(free[i]);
    int64_t found;
    const int64_t rank = base + scan<kBlock>(count, part, found);
    int64_t before = rank;
#pragma unroll
    for (int i = 0; i < kWords; i++) {
      if (i >= per) continue;
      word[tid * per + i] = free[i];
      word_at[tid * per + i] = int(before - base);
      const int have = __builtin_popcount(free[i]);
      if (before < total && have > 0) {
        // the lowest of the word's free pages are taken, all of them but in the last word
        uint32_t left = 0;
        if (before + have > total) {
          left = free[i];
          for (int64_t r = before; r < total; r++) left &= left - 1;
        }
        const int64_t w = w0 + tid * per + i;
        pool.used[w] = used_word(pool, w, false) | (free[i] & ~left);
      }
      before += have;
    }
    __syncthreads();
    // a thread a page
    for (int64_t r = base + tid; r < min(base + found, total); r += kBlock) {
      int at = 0, end = kBlock * per;  // word_at[at] <= r - base < word_at[end]
      while (end - at > 1) {
        const int mid = (at + end) / 2;
        if (word_at[mid] <= int(r - base)) at = mid;
        else end = mid;
      }
      uint32_t left = word[at];
      int bit = 0, nth = int(r - base) - word_at[at];  // the nth bit that is set
#pragma unroll
      for (int half = 16; half >= 1; half /= 2) {
        const int low = __builtin_popcount(left & ((1u << half) - 1));
        if (nth >= low) {
          nth -= low;
          left >>= half;
          bit += half;
        }
      }
      const int id = int(32 * (w0 + at)) + bit;
      int lo = 0, hi = n;  // off[lo] <= r < off[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (off[mid] <= r) lo = mid;
        else hi = mid;
      }
      const int which = int(r - off[lo]);
      int32_t *row = t.pages + lo * t.stride;
      const int c = copy[lo];
      if (c >= 0 && which == 0) {
        row[first[lo] - 1] = id;
        moves.src[c] = tail[lo];
        moves.dst[c] = id;
        atomicAdd(&listed, 1);
      } else {
        row[first[lo] + which - (c >= 0 ? 1 : 0)] = id;
      }
      pool.refs[id] = 1;
    }
    __syncthreads();
    base += found;
  }
  // what no page was left for
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int s = 2 * tid + i;
    if (s >= n) continue;
    const int64_t all = copies[i] + fresh[i], got = min(max(base - off[s], int64_t(0)), all);
    bad |= got < all;
    for (int64_t k = got; k < all; k++)
      t.pages[s * t.stride + first[s] + k - copies[i]] = -1;
    t.len[s] = grown[i];
  }
  if (bad && t.bad) *t.bad = 1;
  __syncthreads();
  if (tid == 0) *moves.count = listed;
}

// ---- trim -----------------------------------------------------------------
// A workgroup a sequence, a thread a page: the last table that names a page frees it.
// Latency: 128 sequences of up to 47 pages 4.8 us.
__global__ void __launch_bounds__(256) trim_kernel(PagePool pool, PageTables t,
                                                   const int32_t *__restrict__ d_keep) {
  const int s = int(blockIdx.x);
  const int len = max(t.len[s], 0), keep = min(len, d_keep ? max(d_keep[s], 0) : 0);
  const int64_t c1 = held_cols(len, pool.shift, t.stride);
  for (int64_t c = held_cols(keep, pool.shift, t.stride) + threadIdx.x; c < c1; c += 256) {
    const int id = t.pages[s * t.stride + c];
    if (page_ok(id, pool.n_pages) && atomicSub(&pool.refs[id], 1) == 1)
      atomicAnd(&pool.used[id / 32], ~(1u << (id % 32)));
  }
  __syncthreads();
  if (threadIdx.x == 0) t.len[s] = keep;
}

// ---- compact --------------------------------------------------------------
// One workgroup: the words of a round, with the holes below U and the pages at U and
// above that lie before each, go to LDS; then a thread a page, whose rank is its place.
// 4790 pages 4.8 us, the time of its sums' steps.
constexpr int kListBlock = 1024, kListWords = 2;
__global__ void __launch_bounds__(kListBlock) compact_list_kernel(PagePool pool, PageMoves moves) {
  constexpr int kRound = kListBlock * kListWords;
  __shared__ int64_t part[kListBlock / 64];
  __shared__ uint32_t word[kRound], hole_at[kRound], up_at[kRound];
  const int tid = int(threadIdx.x);
  const int64_t words = (int64_t(pool.n_pages) + 31) / 32;
  int64_t n_used = 0, sum;
  for (int64_t w = tid; w < words; w += kListBlock)
    n_used += __builtin_popcount(used_word(pool, w, false));
  scan<kListBlock>(n_used, part, sum);
  n_used = sum;
  int64_t holes = 0, high = 0;  // before this round's words
  for (int64_t w0 = 0; w0 < words; w0 += kRound) {
    uint32_t x[kListWords], low[kListWords];
    int64_t mine = 0;  // holes, and 2^32 times the pages above
#pragma unroll
    for (int i = 0; i < kListWords; i++) {
      const int64_t w = w0 + tid * kListWords + i, below = n_used - 32 * w;
      low[i] = below >= 32 ? ~0u : below <= 0 ? 0u : (1u << below) - 1;
      x[i] = used_word(pool, w, false);
      mine += __builtin_popcount(~x[i] & low[i]) + (int64_t(__builtin_popcount(x[i] & ~low[i])) << 32);
    }
    const int64_t before = scan<kListBlock>(mine, part, sum);
    uint32_t h = uint32_t(holes + (before & 0xFFFFFFFF)), u = uint32_t(high + (before >> 32));
#pragma unroll
    for (int i = 0; i < kListWords; i++) {
      word[tid * kListWords + i] = x[i];
      hole_at[tid * kListWords + i] = h;
      up_at[tid * kListWords + i] = u;
      h += uint32_t(__builtin_popcount(~x[i] & low[i]));
      u += uint32_t(__builtin_popcount(x[i] & ~low[i]));
    }
    __syncthreads();
    const int64_t last = min(int64_t(pool.n_pages), 32 * (w0 + kRound));
    for (int64_t id = 32 * w0 + tid; id < last; id += kListBlock) {
      const int at = int(id / 32 - w0);
      const uint32_t bit = 1u << (id % 32), under = bit - 1, w = word[at];
      const int64_t below = n_used - id / 32 * 32;
      const uint32_t lower = below >= 32 ? ~0u : below <= 0 ? 0u : (1u << below) - 1;
      if (id < n_used && !(w & bit)) {
        const uint32_t r = hole_at[at] + uint32_t(__builtin_popcount(~w & lower & under));
        if (r < uint32_t(moves.cap)) moves.dst[r] = int(id);
      } else if (id >= n_used && (w & bit)) {
        const uint32_t r = up_at[at] + uint32_t(__builtin_popcount(w & ~lower & under));
        if (r < uint32_t(moves.cap)) moves.src[r] = int(id);
      }
    }
    __syncthreads();
    holes += sum & 0xFFFFFFFF;
    high += sum >> 32;
  }
  if (tid == 0) *moves.count = int(min(high, int64_t(moves.cap)));
}

// Counts of the pages that move (the last layer of workgroups), and the rows' entries
// (a workgroup a row and layer): where the list, which rises, holds an entry as a source it
// becomes the place it moves to, found by bisection.  Lists of up to 2048 lie in LDS whole;
// of longer ones every step-th source does.  Latency: 128 sequences of up to 47 pages 8.1 us.
constexpr int kProbes = 2048;
__global__ void __launch_bounds__(256) compact_move_kernel(PagePool pool, PageTables t,
                                                           PageMoves moves) {
  __shared__ int probe[kProbes], place[kProbes];
  const int s = int(blockIdx.x), tid = int(threadIdx.x);
  // (loads are on their way before the list's length is known; what lies behind it is not
  // used)
  if (blockIdx.y == gridDim.y - 1) {  // counts
    int64_t i = int64_t(s) * 256 + tid;
    int a = i < moves.cap ? moves.src[i] : -1, b = i < moves.cap ? moves.dst[i] : -1;
    int refs = page_ok(a, pool.n_pages) ? pool.refs[a] : 0;
    for (const int n = *moves.count; i < n;) {
      pool.refs[b] = refs;
      pool.refs[a] = 0;
      atomicAnd(&pool.used[a / 32], ~(1u << (a % 32)));
      atomicOr(&pool.used[b / 32], 1u << (b % 32));
      i += int64_t(gridDim.x) * 256;
      if (i >= n) break;
      a = moves.src[i];
      b = moves.dst[i];
      refs = pool.refs[a];
    }
    return;
  }
  int src[kProbes / 256], dst[kProbes / 256], id = -1;
#pragma unroll
  for (int j = 0; j < kProbes / 256; j++) {
    const int i = 256 * j + tid;
    src[j] = i < moves.cap ? moves.src[i] : 0;
    dst[j] = i < moves.cap ? moves.dst[i] : 0;
  }
  const int64_t first = int64_t(blockIdx.y) * 256 + tid;
  const int64_t cols = s < t.n_seq ? held_cols(t.len[s], pool.shift, t.stride) : 0;
  if (first < cols) id = t.pages[s * t.stride + first];
  const int n = *moves.count;
  if (n == 0) return;
  const int step = (n + kProbes - 1) / kProbes, probes = (n + step - 1) / step;
  if (int64_t(blockIdx.y) * 256 >= cols) return;
  if (step == 1) {
#pragma unroll
    for (int j = 0; j < kProbes / 256; j++) {
      probe[256 * j + tid] = src[j];
      place[256 * j + tid] = dst[j];
    }
  } else {
    for (int i = tid; i < probes; i += 256) probe[i] = moves.src[int64_t(i) * step];
  }
  __syncthreads();
  for (int64_t c = first; c < cols; c += int64_t(gridDim.y - 1) * 256) {
    if (c != first) id = t.pages[s * t.stride + c];
    if (id < probe[0]) continue;
    int lo = 0, hi = probes;  // probe[lo] <= id < probe[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (probe[mid] <= id) lo = mid;
      else hi = mid;
    }
    if (step == 1) {
      if (probe[lo] == id) t.pages[s * t.stride + c] = place[lo];
      continue;
    }
    int64_t a = int64_t(lo) * step, b = min(a + step, int64_t(n));
    while (b - a > 1) {
      const int64_t mid = (a + b) / 2;
      if (moves.src[mid] <= id) a = mid;
      else b = mid;
    }
    if (moves.src[a] == id) t.pages[s * t.stride + c] = moves.dst[a];
  }
}

// ---- copy -----------------------------------------------------------------
// HBM's: a page is read and written once, 4 KB a wave at a time.  The list's length
// is on the device, so a fixed grid runs over (pair, segment of a page).  307 MB of pages
// of 32 KB, keys and values of two layers, read and written in 54 us: 5.6 TB/s.
constexpr int kCaches = 64;  // of a launch
typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));

struct CopyWork {
  uint16_t *base[2 * kCaches];  // keys and values of each cache
  PageMoves moves;
  int64_t page_stride, head_stride, slot_stride;  // elements
  int n_pages, shift, row_chunks, chunks, segs;   // 16-byte chunks of a row and of a page
  int flat;                                       // a page's rows lie without gaps
};

__global__ void __launch_bounds__(256) copy_kernel(CopyWork w) {
  const int lane = int(threadIdx.x) & 63, wave = int(threadIdx.x) >> 6;
  uint16_t *base = w.base[blockIdx.y];
  const int n = min(*w.moves.count, w.moves.cap);
  const int64_t items = int64_t(n) * w.segs;
  for (int64_t item = int64_t(blockIdx.x) * 4 + wave; item < items; item += int64_t(gridDim.x) * 4) {
    const int pair = int(item / w.segs), seg = int(item - int64_t(pair) * w.segs);
    const int a = w.moves.src[pair], b = w.moves.dst[pair];
    if (!page_ok(a, w.n_pages) || !page_ok(b, w.n_pages)) continue;
    const uint16_t *src = base + a * w.page_stride;
    uint16_t *dst = base + b * w.page_stride;
    int64_t at[4];
    u32x4v v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int c = seg * 256 + 64 * i + lane;
      at[i] = int64_t(c) * 8;
      if (!w.flat) {
        const int row = c / w.row_chunks;
        at[i] = (row >> w.shift) * w.head_stride + (row & ((1 << w.shift) - 1)) * w.slot_stride +
                (c - row * w.row_chunks) * 8;
      }
      if (c < w.chunks) v[i] = *reinterpret_cast<const u32x4v *>(src + at[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (seg * 256 + 64 * i + lane < w.chunks) *reinterpret_cast<u32x4v *>(dst + at[i]) = v[i];
  }
}

// Forks of many sequences ask for more than 64 KB of dynamic LDS, which a kernel has to be
// allowed: once a device, the most that any call takes, so that no call lowers the limit
// between another thread's setting and its launch.
size_t fork_lds(int n_seq) { return size_t(n_seq) * (kTile + 3) * 4; }
bool fork_limit_set() {
  constexpr int kDevices = 64;  // (as many as the library initialises)
  static std::once_flag once[kDevices];
  static hipError_t err[kDevices];
  const int dev = swamp::device_info().device;
  if (dev < 0 || dev >= kDevices) return false;
  std::call_once(once[dev], [dev] {
    err[dev] = hipFuncSetAttribute(reinterpret_cast<const void *>(&fork_kernel<false>),
                                   hipFuncAttributeMaxDynamicSharedMemorySize, int(fork_lds(kSeqs)));
  });
  return err[dev] == hipSuccess;
}

int launched() { return hipGetLastError() == hipSuccess ? SWAMP_OK : SWAMP_ELAUNCH; }

}  // namespace

int swamp_launch_pages_fork(const PagePool &pool, const PageTables &t, const int32_t *d_parent,
                            hipStream_t s) {
  const size_t lds = fork_lds(t.n_seq);
  const int64_t tiles = std::max<int64_t>(1, (t.stride + kTile - 1) / kTile);
  // Two launches take 5.5 to 8 us (64 sequences 8).  One takes 3.4, 0.6 a thousand pages and,
  // a tile, 0.5 and 0.04 a sequence: 4 sequences of 30 pages among 512 take 4.8 us in one and
  // 6.4 in two, 64 of 30 among 2048 10.2 and 8.4, 4 of 8 among 8192 9.3 and 6.0.
  if (pool.n_pages / 1024 + tiles * (16 + t.n_seq) / 32 <= 4 && t.n_seq <= 256) {
    fork_kernel<true><<<1, 256, lds, s>>>(pool, t, d_parent);
    return launched();
  }
  if (lds > 64 * 1024 && !fork_limit_set()) return SWAMP_ELAUNCH;
  fork_kernel<false><<<unsigned(std::min<int64_t>(tiles, 1024)), 256, lds, s>>>(pool, t, d_parent);
  const unsigned blocks = unsigned(std::max<int64_t>(1, (int64_t(pool.n_pages) + 255) / 256));
  fork_finish_kernel<<<blocks, 256, 0, s>>>(pool, t, d_parent);
  return launched();
}

int swamp_launch_pages_extend(const PagePool &pool, const PageTables &t, const int32_t *d_new,
                              const PageMoves &moves, hipStream_t s) {
  // (a small workgroup waits less at its barriers)
  const int64_t words = (int64_t(pool.n_pages) + 31) / 32;
  auto per = [&](int block) { return int(std::max<int64_t>(1, std::min<int64_t>(kWords, (words + block - 1) / block))); };
  if (t.n_seq <= 512 && words <= 256 * kWords)
    extend_kernel<256><<<1, 256, 0, s>>>(pool, t, d_new, moves, per(256));
  else
    extend_kernel<1024><<<1, 1024, 0, s>>>(pool, t, d_new, moves, per(1024));
  return launched();
}

int swamp_launch_pages_trim(const PagePool &pool, const PageTables &t, const int32_t *d_keep,
                            hipStream_t s) {
  trim_kernel<<<unsigned(t.n_seq), 256, 0, s>>>(pool, t, d_keep);
  return launched();
}

int swamp_launch_pages_compact(const PagePool &pool, const PageTables &t, const PageMoves &moves,
                               hipStream_t s) {
  compact_list_kernel<<<1, kListBlock, 0, s>>>(pool, moves);
  const dim3 grid(unsigned(std::max(t.n_seq, 64)),
                  unsigned(1 + std::max<int64_t>(1, std::min<int64_t>(t.stride / 256, 16))));
  compact_move_kernel<<<grid, 256, 0, s>>>(pool, t, moves);
  return launched();
}

int swamp_launch_kv_copy(const swamp::PagedCache &c, const swamp_kv_pages *caches, int n_caches,
                         const PageMoves &moves, hipStream_t s) {
  CopyWork w;
  w.moves = moves;
  w.page_stride = c.page_stride;
  w.head_stride = c.head_stride;
  w.slot_stride = c.slot_stride;
  w.n_pages = c.n_pages;
  w.shift = c.page_shift;
  w.row_chunks = c.dim / 8;
  w.chunks = (c.n_kv << c.page_shift) * w.row_chunks;
  w.segs = (w.chunks + 255) / 256;
  const int64_t slots = int64_t(1) << c.page_shift;
  w.flat = (c.slot_stride == c.dim && (c.n_kv == 1 || c.head_stride == slots * c.dim)) ||
           ((c.n_kv == 1 || c.head_stride == c.dim) &&
            (slots == 1 || c.slot_stride == int64_t(c.n_kv) * c.dim));
  for (int i0 = 0; i0 < n_caches; i0 += kCaches) {
    const int n = std::min(n_caches - i0, kCaches);
    for (int i = 0; i < n; i++) {
      w.base[2 * i] = static_cast<uint16_t *>(caches[i0 + i].d_k);
      w.base[2 * i + 1] = static_cast<uint16_t *>(caches[i0 + i].d_v);
    }
    // (waves for every segment of the list's most, 16 workgroups a CU in all)
    const int64_t most = (int64_t(moves.cap) * w.segs + 3) / 4;
    const int64_t room = std::max(1, 16 * swamp::device_info().num_cus / (2 * n));
    const dim3 grid(unsigned(std::max<int64_t>(1, std::min(most, room))), unsigned(2 * n));
    copy_kernel<<<grid, 256, 0, s>>>(w);
  }
  return launched();
}
