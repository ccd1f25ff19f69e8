// beam.hip -- swamp_beam_select: the best continuations of every sequence over its
// beams and the vocabulary.  total(b, v) = score_b + x_bv - log sum_u exp x_bu, taken as
// score_b + ((x_bv - m_b) - log sum_u exp(x_bu - m_b)), m_b the row's largest logit.
//
// Two launches.  The first cuts every row of logits into chunks of 4096, one a
// workgroup, held in registers: the chunk's maximum m, its sum of exp(x - m), and its
// n_out largest logits in falling order.  The second, a workgroup a sequence, joins the
// sums and ranks the lists' tokens by their totals.
//
// Sums and totals are 64-bit: beams whose scores agree to 32 bits keep their order.  Equal
// totals go by beam, then the larger logit, then the lower token.  The exponential is
// 2^n 2^f, n = rint(x log2 e), 2^f a polynomial of degree 9 through the Chebyshev nodes of
// |f| <= 1/2 (off by 2e-14 of it): 16 operations of 64 bits an element, which the vector
// units issue at the rate of 32-bit ones.
//
// Largest tokens without a sort: a wave's lanes each have a largest value.  Where a quarter
// of n_out of every wave's reach a bound (found bit by bit with ballots), or n_out of one
// wave's do, so do n_out values of the chunk.  What reaches it, little more than n_out
// tokens, is collected in LDS and ranked by counting.  Where too many do (equal logits) the
// exact bound is found bit by bit over the whole chunk.  The lists of a sequence are cut
// alike: n_out / r lists whose r-th token reaches a bound have n_out tokens that do.
//
// Measured, the two kernels: 4 beams of 128256 f32 logits, 8 best, 5.6 + 6.3 us; 16 x 4 of
// them 13.4 + 6.5 (2.4 TB/s in the first); 4 x 32 of 32000 bf16, 64 best, 13.9 + 14.5; 50 x 5
// of 50257 f16, nearly all masked, 14.0 + 7.0.  The first is bound by the ballots of its
// bounds and the 64-bit polynomial (vector units busy half of the time), the second by its
// chain of steps in one workgroup (sums 2 us, bound 2, collection 1, ranks 1).
#include "swamp_common.hpp"
#include "wave.hpp"

#include <type_traits>

namespace {

using swamp::BeamCall;

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kEach = 16;                  // logits of a thread
constexpr int kChunk = kThreads * kEach;   // of a workgroup
constexpr int kList = 1024;                // tokens that it ranks
constexpr int kJoin = 2048;                // tokens that a sequence's workgroup ranks
constexpr int kBeams = 64;
constexpr int kJoinThreads = 512, kJoinWaves = kJoinThreads / 64;

struct Entry {
  float x;
  int32_t token;  // -1: none
};
struct Part {  // of a chunk
  double sum;
  float top, pad;
};

struct Work {
  BeamCall c;
  int chunks;    // of a row
  int pad;       // places of a list: n_out, a multiple of 4
  Entry *list;   // [row][chunk][pad]
  Part *part;    // [row][chunk]
};

// Floats in the order of their keys (-0 below 0: 0 is added where that counts).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}
constexpr uint32_t kNone = 0x007FFFFFu;  // key of -infinity

// x, which the compiler no longer knows: what a rare path computes from it is not kept in
// registers meanwhile.
template <typename T>
__device__ __forceinline__ T fresh(T x) {
#ifdef __HIP_DEVICE_COMPILE__
  asm volatile("" : "+v"(x));
#endif
  return x;
}

// 2^t for t of any size; NaN passes, and t far below 0 gives 0.
__device__ __forceinline__ double exp2_64(double t) {
  const double n = __builtin_rint(t), f = t - n;
  constexpr double c[10] = {1.000000000000013545e+00, 6.931471805599446201e-01,
                            2.402265069563986055e-01, 5.550410866470367743e-02,
                            9.618129194074795732e-03, 1.333355819593412062e-03,
                            1.540343361871355534e-04, 1.525267453819431725e-05,
                            1.325968083523608916e-06, 1.020575712504153700e-07};
  double p = c[9];
#pragma unroll
  for (int i = 8; i >= 0; i--) p = __builtin_fma(p, f, c[i]);
  return __builtin_amdgcn_ldexp(p, int(n));
}
constexpr double kLog2e64 = 1.4426950408889634074;
constexpr float kLowest = -3.402823466e38f;

// ---- a chunk --------------------------------------------------------------
template <typename XT>
struct __attribute__((packed, aligned(sizeof(XT)))) Vec {
  XT v[16 / sizeof(XT)];
};

// The chunk's elements: load j of a thread holds kPer neighbours; of a row's last chunk,
// which is short, every thread has one of each 256, so that all waves have their share.
template <typename XT>
struct Chunk {
  static constexpr int kPer = 16 / int(sizeof(XT)), kLoads = kEach / kPer;
  static __device__ __forceinline__ int at(int e, bool whole, int tid = int(threadIdx.x)) {
    return whole ? (e / kPer) * kThreads * kPer + tid * kPer + e % kPer : e * kThreads + tid;
  }
  static __device__ __forceinline__ void load(const XT *row, int n, bool whole, float *x) {
    if (whole) {
#pragma unroll
      for (int j = 0; j < kLoads; j++) {
        const Vec<XT> v = *reinterpret_cast<const Vec<XT> *>(row + at(j * kPer, true));
#pragma unroll
        for (int i = 0; i < kPer; i++) x[j * kPer + i] = float(v.v[i]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < kEach; e++) x[e] = at(e, false) < n ? float(row[at(e, false)]) : -INFINITY;
    }
  }
};

// Keys that at least k, and at least `few` (k over the waves), of the wave's 64 N reach:
// the largest such but for their low bits.
template <int N, int kLow>
__device__ __forceinline__ void reached_by(const uint32_t *keys, int k, int few, uint32_t &all,
                                           uint32_t &share) {
  all = share = 0;
#pragma unroll
  for (int bit = 31; bit >= kLow; bit--) {
    const uint32_t up = all | 1u << bit, up1 = share | 1u << bit;
    int n = 0, n1 = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
      n += __builtin_popcountll(__ballot(keys[i] >= up));
      n1 += __builtin_popcountll(__ballot(keys[i] >= up1));
    }
    if (n >= k) all = up;
    if (n1 >= few) share = up1;
  }
}
// What k of the workgroup's reach: the best of what k of a wave's do, or what every
// wave's share does.
template <int W>
__device__ __forceinline__ uint32_t joint_bound(const uint32_t *all, const uint32_t *share) {
  uint32_t a = all[0], q = share[0];
#pragma unroll
  for (int i = 1; i < W; i++) {
    a = max(a, all[i]);
    q = min(q, share[i]);
  }
  return max(a, q);
}

template <typename XT>
__global__ void __launch_bounds__(kThreads, 8) chunk_kernel(Work w) {
  typedef Chunk<XT> C;
  __shared__ uint64_t list[kList];  // key, then place from the end
  __shared__ int16_t kept[kList];
  __shared__ float tops[kWaves];
  __shared__ double sums[kWaves];
  __shared__ uint32_t bounds[kWaves], shares[kWaves];
  __shared__ int listed, left, counts[kWaves];
  const int row = int(blockIdx.x / uint32_t(w.chunks)), chunk = int(blockIdx.x % uint32_t(w.chunks));
  if (w.c.done && w.c.done[row]) return;
  const int tid = int(threadIdx.x), wave = tid >> 6, k = w.c.n_out;
  const int first = chunk * kChunk, n = min(w.c.vocab - first, kChunk);
  const bool whole = n == kChunk;
  float x[kEach];
  C::load(static_cast<const XT *>(w.c.logits) + row * w.c.stride + first, n, whole, x);
  if (tid == 0) listed = left = 0;
  float mine = -INFINITY;  // (and for NaN)
#pragma unroll
  for (int e = 0; e < kEach; e++) mine = fmaxf(mine, x[e]);
  float top = swamp::group_max(mine, 64);
  // n_out of one wave's lanes reach the one bound, a quarter of them of every wave's the other
  uint32_t bound, share;
  const uint32_t key = key_of(mine);
  reached_by<1, 15>(&key, k, (k + kWaves - 1) / kWaves, bound, share);
  if ((tid & 63) == 0) {
    tops[wave] = top;
    bounds[wave] = bound;
    shares[wave] = share;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; i++) top = fmaxf(top, tops[i]);
  const float least = value_of(max(joint_bound<kWaves>(bounds, shares), kNone + 1));
  if (__any(mine >= least)) {
#pragma unroll
    for (int e = 0; e < kEach; e++)
      if (x[e] >= least) {
        const int i = atomicAdd(&listed, 1);
        if (i < kList)
          list[i] = uint64_t(key_of(x[e] + 0.f)) << 32 | uint32_t(~C::at(e, whole, fresh(tid)));
      }
  }
  // (a chunk of nothing but -infinity: 0; an infinity: NaN, of inf - inf)
  const double base = top == -INFINITY ? 0.0 : double(top);
  double sum = 0.0;
  float low = x[0];
#pragma unroll
  for (int e = 1; e < kEach; e++) low = fminf(low, x[e]);
  if (__any(low == -INFINITY)) {  // masked tokens: no work where all of the wave's are
#pragma unroll
    for (int e = 0; e < kEach; e++)
      if (__any(x[e] != -INFINITY)) {
        __builtin_amdgcn_sched_barrier(0);
        // (0 itself: beside a top of the lowest value any finite stand-in would count)
        const double term = exp2_64((double(x[e]) - base) * kLog2e64);
        sum += x[e] == -INFINITY ? 0.0 : term;
      }
  } else {
#pragma unroll
    for (int e = 0; e < kEach; e++) {
      if (e % 4 == 0) __builtin_amdgcn_sched_barrier(0);
      sum += exp2_64((double(x[e]) - base) * kLog2e64);
    }
  }
  sum = swamp::group_sum(sum, 64);
  if ((tid & 63) == 0) sums[wave] = sum;
  __syncthreads();
  int c = listed;
  if (c > kList) {
    // the k-th largest (key, place) exactly: k or fewer reach it
    uint64_t t = 0;
    for (int bit = 43; bit >= 0; bit--) {  // 32 bits of key, 12 of place
      const uint64_t up = t | uint64_t(1) << bit;
      int reach = 0;
#pragma unroll
      for (int e = 0; e < kEach; e++) {
        const uint32_t key = key_of(fmaxf(fresh(x[e]), -INFINITY) + 0.f);
        const uint64_t place = uint64_t(key) << 12 | uint32_t(kChunk - 1 - C::at(e, whole, fresh(tid)));
        reach += __builtin_popcountll(__ballot(key > kNone && place >= up));
      }
      __syncthreads();
      if ((tid & 63) == 0) counts[wave] = reach;
      __syncthreads();
      reach = 0;
#pragma unroll
      for (int i = 0; i < kWaves; i++) reach += counts[i];
      if (reach >= k) t = up;
    }
    if (tid == 0) listed = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; e++) {
      const uint32_t key = key_of(fmaxf(fresh(x[e]), -INFINITY) + 0.f);
      const uint64_t place = uint64_t(key) << 12 | uint32_t(kChunk - 1 - C::at(e, whole, fresh(tid)));
      if (key > kNone && place >= t)
        list[atomicAdd(&listed, 1)] = uint64_t(key) << 32 | uint32_t(~C::at(e, whole, fresh(tid)));
    }
    __syncthreads();
    c = listed;
  }
  const int64_t at = int64_t(row) * w.chunks + chunk;
  Entry *out = w.list + at * w.pad;
  auto rank_all = [&](int n, auto at) {
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t me = list[at(i)];
      int rank = 0;
#pragma unroll 8
      for (int o = 0; o < n; o++) rank += list[at(o)] > me ? 1 : 0;
      if (rank < k) out[rank] = Entry{value_of(uint32_t(me >> 32)), first + int(~uint32_t(me))};
    }
  };
  if (c <= 256) {
    rank_all(c, [](int i) { return i; });
  } else {
    // a bound again, of all that is listed.  Up to 256 every thread ranks at most one: 4 x 32
    // beams of 32000 bf16 logits, 64 best, take 29 us in both kernels, 33 if the bound is
    // renewed from 97 on, and 4 of 128256, 8 best, 13 and, if it always is, 16.
    constexpr int kEachLane = kList / kThreads;
    uint32_t some[kEachLane], all, part;
#pragma unroll
    for (int i = 0; i < kEachLane; i++) {
      const int from = (64 * i + (tid & 63)) * kWaves + wave;
      some[i] = from < c ? uint32_t(list[from] >> 32) : 0;
    }
    reached_by<kEachLane, 8>(some, k, (k + kWaves - 1) / kWaves, all, part);
    if ((tid & 63) == 0) {
      bounds[wave] = all;
      shares[wave] = part;
    }
    __syncthreads();
    const uint32_t enough = joint_bound<kWaves>(bounds, shares);
    for (int i = tid; i < c; i += kThreads)
      if (uint32_t(list[i] >> 32) >= enough) kept[atomicAdd(&left, 1)] = int16_t(i);
    __syncthreads();
    rank_all(left, [&](int i) { return int(kept[i]); });
  }
  for (int i = min(c, k) + tid; i < w.pad; i += kThreads) out[i] = Entry{0.f, -1};
  if (tid == 0) {
    sum = sums[0];
#pragma unroll
    for (int i = 1; i < kWaves; i++) sum += sums[i];
    w.part[at] = Part{sum, top, 0.f};
  }
}

// ---- a sequence -----------------------------------------------------------
// The order of continuations: the larger total, then the lower place: the beam, above the
// logit's key turned round, above the token.  Totals of one beam fall with its logits or stay
// equal (a logit of 1e18 leaves no other two apart in 64 bits), so the chunks' lists, cut by
// logits, are in this order too, and the best n are the head of the best n + 1.
struct Best {
  double total;
  uint64_t place;
};
constexpr int kTokenBits = 20, kBeamShift = 52;  // vocabularies of up to 2^20
constexpr uint64_t kNobody = ~uint64_t(0);  // place of no continuation
__device__ __forceinline__ uint64_t place_of(int beam, float x, int token) {
  return uint64_t(beam) << kBeamShift | uint64_t(~key_of(x)) << kTokenBits | uint32_t(token);
}
__device__ __forceinline__ int beam_at(uint64_t place) { return int(place >> kBeamShift); }
__device__ __forceinline__ int token_at(uint64_t place) {
  return int(uint32_t(place) & ((1u << kTokenBits) - 1));
}
__device__ __forceinline__ bool before(const Best &a, const Best &b) {
  return a.place != kNobody &&
         (b.place == kNobody || a.total > b.total || (a.total == b.total && a.place < b.place));
}

// A total as a whole number of the same order, for comparisons without branches.
struct Ranked {
  uint64_t key, place;
};
__device__ __forceinline__ Ranked ranked(const Best &b) {
  const uint64_t u = __builtin_bit_cast(uint64_t, b.total + 0.0);
  return Ranked{u >> 63 ? ~u : u | uint64_t(1) << 63, b.place};
}
__device__ __forceinline__ double total_of(uint64_t key) {
  return __builtin_bit_cast(double, key >> 63 ? key & ~(uint64_t(1) << 63) : ~key);
}

// The largest logit and the log of the sum of exp(x - top) stay apart: in one number a top
// of 1e15, or one of the type's lowest value (a row whose mask leaves nothing), takes log_sum
// with it even in 64 bits.
struct Row {  // of a beam
  double score, top, log_sum;
  int state;  // 0: it has no continuation, 1: tokens, 2: it has ended
};

// x at place p of list l, of beam b.
__device__ __forceinline__ Best best_of(const Work &w, const Row &r, int b, int l, int p, Entry x) {
  Best e{0.0, kNobody};
  if (r.state == 1) {
    if (x.token >= 0)
      e = Best{r.score + ((double(x.x) - r.top) - r.log_sum), place_of(b, x.x, x.token)};
  } else if (r.state == 2 && p == 0 && l == b * w.chunks) {
    e = Best{r.score, place_of(b, 0.f, w.c.eos)};
  }
  return e;
}
__device__ __forceinline__ const Entry *list_of(const Work &w, int seq, int l) {
  return w.list + (int64_t(seq) * w.c.n_beam * w.chunks + l) * w.pad;
}
__device__ __forceinline__ uint32_t bound_key(const Best &e) {
  return e.place == kNobody ? 0u : key_of(float(e.total) + 0.f);
}
__device__ __forceinline__ Best wave_best(Best best) {
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) {
    const Best o{__shfl_xor(best.total, d, 64),
                 uint64_t(__shfl_xor(static_cast<unsigned long long>(best.place), d, 64))};
    if (before(o, best)) best = o;
  }
  return best;
}

__global__ void __launch_bounds__(kJoinThreads) join_kernel(Work w) {
  __shared__ Row rows[kBeams];
  __shared__ __attribute__((aligned(16))) Ranked list[kJoin];
  __shared__ uint32_t keys[kJoin];
  __shared__ int16_t kept[kJoin];
  __shared__ Best picked[kBeams];
  __shared__ Best waves[kJoinWaves];
  __shared__ uint32_t bounds[kJoinWaves], shares[kJoinWaves];
  __shared__ int listed, left;
  const int seq = int(blockIdx.x), tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6;
  const int nb = w.c.n_beam, k = w.c.n_out, lists = nb * w.chunks;
  if (tid == 0) listed = left = 0;
  // (on their way while the sums are joined) the first, 4th, 16th, 64th of a list
  constexpr int kProbes = 4;
  Entry probe[kProbes];
  // `full` waves have 64 lists or more and take them in turn, so that none has but one
  // beam's; another wave may have a few
  const int full = min(max(lists / 64, 1), kJoinWaves);
  const int mine = wave < full ? lane * full + wave : tid;
  const Entry *mine_at = list_of(w, seq, min(mine, lists - 1));
#pragma unroll
  for (int i = 0; i < kProbes; i++) probe[i] = mine_at[min((1 << 2 * i) - 1, k - 1)];
  // `team` lanes take a beam's chunks
  int team = 1;
  while (team < w.chunks && team < 64) team *= 2;
  const int at = lane & (team - 1);
  for (int b = tid / team; b < (nb + kJoinThreads / team - 1) / (kJoinThreads / team) * (kJoinThreads / team);
       b += kJoinThreads / team) {
    const int64_t row = int64_t(seq) * nb + min(b, nb - 1);
    const Part *part = w.part + row * w.chunks;
    const bool ended = w.c.done && w.c.done[row];
    const double score = double(w.c.score[row]);
    Part own = part[min(at, w.chunks - 1)];
    if (ended || at >= w.chunks) own = Part{0.0, -INFINITY, 0.f};
    float top = own.top;
    if (!ended)
      for (int i = at + 64; i < w.chunks; i += 64) top = fmaxf(top, part[i].top);
    top = swamp::group_max(top, team);
    const double base = top == -INFINITY ? 0.0 : double(top);
    // (a chunk of nothing but -infinity has the sum 0; NaN passes)
    auto term = [&](const Part &p) {
      const float a = p.top == -INFINITY ? kLowest : p.top;
      return p.sum * exp2_64((double(a) - base) * kLog2e64);
    };
    double sum = term(own);
    if (!ended)
      for (int i = at + 64; i < w.chunks; i += 64) sum += term(part[i]);
    sum = swamp::group_sum(sum, team);
    // (finite only where the row's top is: a row of -infinity has the sum 0, and one that holds
    // NaN or infinity a NaN)
    const double log_sum = ended ? 0.0 : log(sum);
    if (at == 0 && b < nb) {
      const bool fine = score - score == 0.0 && log_sum - log_sum == 0.0;  // both finite
      rows[b] = Row{score, double(top), log_sum, !fine ? 0 : ended ? 2 : 1};
    }
  }
  __syncthreads();
  // a bound that n_out totals reach: of the lists' r-th tokens, for several r
  uint32_t bound = 0, share = 0;
#pragma unroll
  for (int i = 0; i < kProbes; i++) {
    const int r = 1 << 2 * i;
    if (r > k) break;
    uint32_t key = 0;
    if (mine < lists) {
      const int b = mine / w.chunks;
      key = bound_key(best_of(w, rows[b], b, mine, r - 1, probe[i]));
    }
    for (int l = mine + kJoinThreads; l < lists; l += kJoinThreads) {
      const int b = l / w.chunks;
      key = max(key, bound_key(best_of(w, rows[b], b, l, r - 1, list_of(w, seq, l)[r - 1])));
    }
    uint32_t all, quarter;
    const int need = (k + r - 1) / r;
    reached_by<1, 14>(&key, need, (need + full - 1) / full, all, quarter);
    bound = max(bound, all);
    share = max(share, quarter);
  }
  if (wave >= full) share = ~0u;
  if (lane == 0) {
    bounds[wave] = bound;
    shares[wave] = share;
  }
  __syncthreads();
  uint32_t least = max(joint_bound<kJoinWaves>(bounds, shares), 1u);
  // Four places of a list at a time, `team` threads a list where there are few; a list
  // falls, and is left at the first place below the bound.
  team = 1;
  while (team * lists * 2 <= kJoinThreads && team * 4 < k) team *= 2;
  for (int l = tid / team; l < lists; l += kJoinThreads / team) {
    const int b = l / w.chunks;
    const Entry *from = list_of(w, seq, l);
    for (int p = tid % team * 4; p < k; p += 4 * team) {
      Entry x[4];
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = from[p + i];
      bool below = false;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const Best e = best_of(w, rows[b], b, l, p + i, x[i]);
        below = bound_key(e) < least;
        if (below) continue;
        const int to = atomicAdd(&listed, 1);
        if (to < kJoin) {
          list[to] = ranked(e);
          keys[to] = bound_key(e);
        }
      }
      if (below) break;
    }
  }
  __syncthreads();
  const int c = listed;
  if (c <= kJoin) {
    auto rank_all = [&](int n, auto at) {
      for (int i = tid; i < n; i += kJoinThreads) {
        const Ranked me = list[at(i)];
        int rank = 0;
#pragma unroll 8
        for (int o = 0; o < n; o++) {
          const Ranked x = list[at(o)];
          rank += int(x.key > me.key) | (int(x.key == me.key) & int(x.place < me.place));
        }
        if (rank < k) picked[rank] = Best{total_of(me.key), me.place};
      }
    };
    if (c <= 256) {
      rank_all(c, [](int i) { return i; });
    } else {
      // a bound again, of all that is listed: 3 x 28 beams of 99882 bf16 logits, 56 best, take
      // 33.5 us in both kernels without it and 36 with it from 97 on; 7 x 63 beams of 20764,
      // 64 best, 41 with it and 42 without.
      constexpr int kEachLane = kJoin / kJoinThreads;
      uint32_t some[kEachLane], all, part;
#pragma unroll
      for (int i = 0; i < kEachLane; i++) {
        const int at = (64 * i + lane) * kJoinWaves + wave;
        some[i] = at < c ? keys[at] : 0;
      }
      reached_by<kEachLane, 8>(some, k, (k + kJoinWaves - 1) / kJoinWaves, all, part);
      if (lane == 0) {
        bounds[wave] = all;
        shares[wave] = part;
      }
      __syncthreads();
      least = joint_bound<kJoinWaves>(bounds, shares);
      for (int i = tid; i < c; i += kJoinThreads)
        if (keys[i] >= least) kept[atomicAdd(&left, 1)] = int16_t(i);
      __syncthreads();
      rank_all(left, [&](int i) { return int(kept[i]); });
    }
    for (int i = c + tid; i < k; i += kJoinThreads) picked[i] = Best{0.0, kNobody};
  } else {
    // One after the other: the first of the lists' heads, whose list goes on.  A thread
    // keeps the first of its lists' heads; next[l] lies in the ranked list's place.
    uint8_t *next = reinterpret_cast<uint8_t *>(list);
    for (int l = tid; l < lists; l += kJoinThreads) next[l] = 0;
    int from = 0;
    auto first = [&]() {
      Best best{0.0, kNobody};
      for (int l = tid; l < lists; l += kJoinThreads) {
        const int b = l / w.chunks, p = next[l];
        const Best e = p < k ? best_of(w, rows[b], b, l, p, list_of(w, seq, l)[p]) : Best{0.0, kNobody};
        if (before(e, best)) best = e, from = l;
      }
      return best;
    };
    Best head = first();
    for (int r = 0; r < k; r++) {
      const Best top = wave_best(head);
      __syncthreads();
      if (lane == 0) waves[wave] = top;
      __syncthreads();
      Best best = waves[0];
#pragma unroll
      for (int i = 1; i < kJoinWaves; i++)
        if (before(waves[i], best)) best = waves[i];
      if (tid == 0) picked[r] = best;
      if (best.place != kNobody && head.place == best.place) {
        next[from]++;
        head = first();
      }
    }
  }
  __syncthreads();
  if (tid < k) {
    const Best e = picked[tid];
    const bool none = e.place == kNobody;
    const int b = none ? 0 : beam_at(e.place), token = token_at(e.place);
    const int64_t to = int64_t(seq) * k + tid;
    w.c.parent[to] = none ? -1 : seq * nb + b;
    w.c.token[to] = none ? -1 : token;
    w.c.out_score[to] = none ? -INFINITY : float(e.total);
    if (w.c.out_done)
      w.c.out_done[to] = !none && (rows[b].state == 2 || token == w.c.eos) ? 1 : 0;
  }
}

int64_t chunks_of(const BeamCall &c) { return (c.vocab + kChunk - 1) / kChunk; }
int pad_of(const BeamCall &c) { return (c.n_out + 3) / 4 * 4; }

}  // namespace

size_t swamp_beam_scratch_bytes(const BeamCall &c) {
  const size_t parts = size_t(c.n_seq) * size_t(c.n_beam) * size_t(chunks_of(c));
  return swamp::scratch_round(parts * size_t(pad_of(c)) * sizeof(Entry)) +
         swamp::scratch_round(parts * sizeof(Part));
}

int swamp_launch_beam_select(const BeamCall &c, swamp::Scratch &sc, hipStream_t s) {
  Work w;
  w.c = c;
  w.chunks = int(chunks_of(c));
  w.pad = pad_of(c);
  const int64_t parts = int64_t(c.n_seq) * c.n_beam * w.chunks;  // below 2^31
  w.list = static_cast<Entry *>(sc.get(size_t(parts) * size_t(w.pad) * sizeof(Entry)));
  w.part = static_cast<Part *>(sc.get(size_t(parts) * sizeof(Part)));
  if (!w.list || !w.part) return SWAMP_EWORKSPACE;
  if (c.type == SWAMP_F32) chunk_kernel<float><<<unsigned(parts), kThreads, 0, s>>>(w);
  else if (c.type == SWAMP_F16) chunk_kernel<_Float16><<<unsigned(parts), kThreads, 0, s>>>(w);
  else chunk_kernel<__bf16><<<unsigned(parts), kThreads, 0, s>>>(w);
  join_kernel<<<unsigned(c.n_seq), kJoinThreads, 0, s>>>(w);
  return hipGetLastError() == hipSuccess ? SWAMP_OK : SWAMP_ELAUNCH;
}
