// beam.hip -- swamp_beam_select: the best continuations of every sequence over its
// beams and the vocabulary.  total(b, v) = score_b + x_bv - log sum_u exp x_bu.
//
// Two launches.  The first cuts every row of logits into chunks of 4096, one a
// workgroup, held in registers: the chunk's maximum m, its sum of exp(x - m), and its
// n_out largest logits in falling order.  The second, a workgroup a sequence, joins the
// sums and ranks the lists' tokens by their totals.
//
// Sums and totals are 64-bit: beams whose scores agree to 32 bits keep their order, and
// equal ones the order of their tokens.  The exponential is 2^n 2^f, n = rint(x log2 e),
// 2^f by its Taylor polynomial of degree 11 (|f| <= 1/2: off by 6e-15 of it): 18
// operations of 64 bits an element, which the vector units issue at the rate of 32-bit
// ones.
//
// Largest tokens without a sort: a wave's lanes each have a largest value, and the
// n_out-th largest of those 64, found bit by bit with ballots, has n_out values at or
// above it in the chunk.  What reaches the largest of the four waves' bounds, a few
// times n_out tokens, is collected in LDS and ranked by counting.  Where too many do
// (equal logits) the exact bound is found bit by bit over the whole chunk.
#include "swamp_common.hpp"

#include <type_traits>

namespace {

using swamp::BeamCall;

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kEach = 16;                  // logits of a thread
constexpr int kChunk = kThreads * kEach;   // of a workgroup
constexpr int kList = 1024;                // tokens that it ranks
constexpr int kJoin = 2048;                // tokens that a sequence's workgroup ranks
constexpr int kBeams = 64;

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
  Entry *list;   // [row][chunk][n_out]
  Part *part;    // [row][chunk]
};

// Floats in the order of their keys (NaN: as -infinity, it takes its row with it).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}
constexpr uint32_t kNone = 0x007FFFFFu;  // key of -infinity

__device__ __forceinline__ double exp64(double x) {
  x = x < -750.0 ? -750.0 : x;  // (0 from there on; NaN passes)
  const double t = x * 1.4426950408889634074, n = __builtin_rint(t), f = t - n;
  constexpr double c[12] = {1.0,
                            6.931471805599453094e-1,
                            2.402265069591007123e-1,
                            5.550410866482157995e-2,
                            9.618129107628477232e-3,
                            1.333355814642844342e-3,
                            1.540353039338160996e-4,
                            1.525273380405984028e-5,
                            1.321548679014430948e-6,
                            1.017808600923969973e-7,
                            7.054911620801123329e-9,
                            4.445538271870811498e-10};
  double p = c[11];
#pragma unroll
  for (int i = 10; i >= 0; i--) p = __builtin_fma(p, f, c[i]);
  return __builtin_amdgcn_ldexp(p, int(n));
}

// ---- a chunk --------------------------------------------------------------
template <typename XT>
struct __attribute__((packed, aligned(sizeof(XT)))) Vec {
  XT v[16 / sizeof(XT)];
};

// The chunk's elements: load j of a thread holds kPer neighbours.
template <typename XT>
struct Chunk {
  static constexpr int kPer = 16 / int(sizeof(XT)), kLoads = kEach / kPer;
  static __device__ __forceinline__ int at(int e) {
    return (e / kPer) * kThreads * kPer + int(threadIdx.x) * kPer + e % kPer;
  }
  static __device__ __forceinline__ void load(const XT *row, int n, float *x) {
#pragma unroll
    for (int j = 0; j < kLoads; j++) {
      const int first = at(j * kPer);
      if (first + kPer <= n) {
        const Vec<XT> v = *reinterpret_cast<const Vec<XT> *>(row + first);
#pragma unroll
        for (int i = 0; i < kPer; i++) x[j * kPer + i] = float(v.v[i]) + 0.f;  // -0 counts as 0
      } else {
#pragma unroll
        for (int i = 0; i < kPer; i++)
          x[j * kPer + i] = first + i < n ? float(row[first + i]) + 0.f : -INFINITY;
      }
    }
  }
};

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) x = fmaxf(x, __shfl_xor(x, d, 64));
  return x;
}
__device__ __forceinline__ double wave_sum64(double x) {
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) x += __shfl_xor(x, d, 64);
  return x;
}
// A key that at least k of the wave's 64 reach, the largest such but for its low bits.
__device__ __forceinline__ uint32_t reached_by(uint32_t key, int k) {
  uint32_t t = 0;
#pragma unroll
  for (int bit = 31; bit >= 10; bit--) {
    const uint32_t up = t | 1u << bit;
    if (__builtin_popcountll(__ballot(key >= up)) >= k) t = up;
  }
  return t;
}

template <typename XT>
__global__ void __launch_bounds__(kThreads) chunk_kernel(Work w) {
  typedef Chunk<XT> C;
  __shared__ uint64_t list[kList];
  __shared__ float tops[kWaves];
  __shared__ double sums[kWaves];
  __shared__ uint32_t bounds[kWaves];
  __shared__ int listed, counts[kWaves];
  const int row = int(blockIdx.x / uint32_t(w.chunks)), chunk = int(blockIdx.x % uint32_t(w.chunks));
  if (w.c.done && w.c.done[row]) return;
  const int tid = int(threadIdx.x), wave = tid >> 6, k = w.c.n_out;
  const int first = chunk * kChunk, n = min(w.c.vocab - first, kChunk);
  float x[kEach];
  C::load(static_cast<const XT *>(w.c.logits) + row * w.c.stride + first, n, x);
  if (tid == 0) listed = 0;
  float top = x[0];
#pragma unroll
  for (int e = 1; e < kEach; e++) top = fmaxf(top, x[e]);
  const float mine = fmaxf(top, -INFINITY);
  top = wave_max(mine);
  if ((tid & 63) == 0) tops[wave] = top;
  const uint32_t bound = reached_by(key_of(mine), k);
  if ((tid & 63) == 0) bounds[wave] = bound;
  __syncthreads();
  uint32_t least = kNone + 1;
#pragma unroll
  for (int i = 0; i < kWaves; i++) {
    top = fmaxf(top, tops[i]);
    least = max(least, bounds[i]);
  }
  // (the sum's exponentials come between the barriers of the list's)
#pragma unroll
  for (int e = 0; e < kEach; e++) {
    const uint32_t key = key_of(fmaxf(x[e], -INFINITY));
    if (__ballot(key >= least) == 0) continue;
    if (key >= least) {
      const int i = atomicAdd(&listed, 1);
      if (i < kList) list[i] = uint64_t(key) << 32 | uint32_t(~C::at(e));
    }
  }
  const double base = top == -INFINITY ? 0.0 : double(top);
  double sum = 0.0;
#pragma unroll
  for (int e = 0; e < kEach; e++) sum += exp64(double(x[e]) - base);
  sum = wave_sum64(sum);
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
        const uint32_t key = key_of(fmaxf(x[e], -INFINITY));
        const uint64_t place = uint64_t(key) << 12 | uint32_t(kChunk - 1 - C::at(e));
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
      const uint32_t key = key_of(fmaxf(x[e], -INFINITY));
      const uint64_t place = uint64_t(key) << 12 | uint32_t(kChunk - 1 - C::at(e));
      if (key > kNone && place >= t)
        list[atomicAdd(&listed, 1)] = uint64_t(key) << 32 | uint32_t(~C::at(e));
    }
    __syncthreads();
    c = listed;
  }
  const int64_t at = int64_t(row) * w.chunks + chunk;
  Entry *out = w.list + at * k;
  for (int i = tid; i < c; i += kThreads) {
    const uint64_t me = list[i];
    int rank = 0;
    for (int o = 0; o < c; o++) rank += list[o] > me ? 1 : 0;
    if (rank < k) out[rank] = Entry{value_of(uint32_t(me >> 32)), first + int(~uint32_t(me))};
  }
  for (int i = c + tid; i < k; i += kThreads) out[i] = Entry{0.f, -1};
  if (tid == 0) {
    sum = sums[0];
#pragma unroll
    for (int i = 1; i < kWaves; i++) sum += sums[i];
    w.part[at] = Part{sum, top, 0.f};
  }
}

// ---- a sequence -----------------------------------------------------------
struct Best {
  double total;
  int flat;  // beam * vocab + token; -1: none
};
__device__ __forceinline__ bool before(const Best &a, const Best &b) {
  return a.flat >= 0 && (b.flat < 0 || a.total > b.total || (a.total == b.total && a.flat < b.flat));
}

struct Row {  // of a beam
  double score, lse;
  int state;  // 0: it has no continuation, 1: tokens, 2: it has ended
};

// Place p of list l of sequence `seq`.
__device__ __forceinline__ Best entry_of(const Work &w, const Row *rows, int seq, int l, int p) {
  const int b = l / w.chunks;
  const Row &r = rows[b];
  Best e{0.0, -1};
  if (r.state == 1) {
    const Entry x = w.list[(int64_t(seq) * w.c.n_beam * w.chunks + l) * w.c.n_out + p];
    if (x.token >= 0) e = Best{r.score + (double(x.x) - r.lse), b * w.c.vocab + x.token};
  } else if (r.state == 2 && p == 0 && l == b * w.chunks) {
    e = Best{r.score, b * w.c.vocab + w.c.eos};
  }
  return e;
}
__device__ __forceinline__ uint32_t bound_key(const Best &e) {
  return e.flat < 0 ? 0u : key_of(float(e.total) + 0.f);
}

__global__ void __launch_bounds__(kThreads) join_kernel(Work w) {
  __shared__ Row rows[kBeams];
  __shared__ Best list[kJoin];
  __shared__ Best picked[kBeams];
  __shared__ Best waves[kWaves];
  __shared__ uint32_t bounds[kWaves];
  __shared__ int listed;
  const int seq = int(blockIdx.x), tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6;
  const int nb = w.c.n_beam, k = w.c.n_out, lists = nb * w.chunks;
  if (tid == 0) listed = 0;
  for (int b = wave; b < nb; b += kWaves) {
    const int64_t row = int64_t(seq) * nb + b;
    const bool ended = w.c.done && w.c.done[row];
    float top = -INFINITY;
    double sum = 0.0;
    if (!ended) {
      for (int i = lane; i < w.chunks; i += 64) top = fmaxf(top, w.part[row * w.chunks + i].top);
      top = wave_max(top);
      const double base = top == -INFINITY ? 0.0 : double(top);
      for (int i = lane; i < w.chunks; i += 64) {
        const Part p = w.part[row * w.chunks + i];
        // (a chunk of nothing but -infinity has the sum 0; NaN and infinity pass)
        sum += p.sum * exp64(double(p.top) - base);
      }
      sum = wave_sum64(sum);
    }
    if (lane == 0) {
      Row r;
      r.score = double(w.c.score[row]);
      r.lse = ended ? 0.0 : double(top) + log(sum);
      const bool fine = r.score - r.score == 0.0 && r.lse - r.lse == 0.0;  // both finite
      r.state = !fine ? 0 : ended ? 2 : 1;
      rows[b] = r;
    }
  }
  __syncthreads();
  // a bound that n_out totals reach, from the lists' heads
  uint32_t head = 0;
  for (int l = tid; l < lists; l += kThreads) head = max(head, bound_key(entry_of(w, rows, seq, l, 0)));
  const uint32_t bound = reached_by(head, k);
  if (lane == 0) bounds[wave] = bound;
  __syncthreads();
  uint32_t least = 1;
#pragma unroll
  for (int i = 0; i < kWaves; i++) least = max(least, bounds[i]);
  for (int i = tid; i < lists * k; i += kThreads) {
    const Best e = entry_of(w, rows, seq, i / k, i % k);
    if (bound_key(e) >= least) {
      const int at = atomicAdd(&listed, 1);
      if (at < kJoin) list[at] = e;
    }
  }
  __syncthreads();
  const int c = listed;
  if (c <= kJoin) {
    for (int i = tid; i < c; i += kThreads) {
      const Best me = list[i];
      int rank = 0;
      for (int o = 0; o < c; o++) rank += before(list[o], me) ? 1 : 0;
      if (rank < k) picked[rank] = me;
    }
    for (int i = c + tid; i < k; i += kThreads) picked[i] = Best{0.0, -1};
  } else {
    // one after the other: of the tokens behind the last one that was taken the first
    Best last{INFINITY, -1};
    for (int r = 0; r < k; r++) {
      Best best{0.0, -1};
      for (int i = tid; i < lists * k; i += kThreads) {
        const Best e = entry_of(w, rows, seq, i / k, i % k);
        if ((r == 0 || before(last, e)) && before(e, best)) best = e;
      }
#pragma unroll
      for (int d = 32; d >= 1; d /= 2) {
        const Best o{__shfl_xor(best.total, d, 64), __shfl_xor(best.flat, d, 64)};
        if (before(o, best)) best = o;
      }
      __syncthreads();
      if (lane == 0) waves[wave] = best;
      __syncthreads();
      best = waves[0];
#pragma unroll
      for (int i = 1; i < kWaves; i++)
        if (before(waves[i], best)) best = waves[i];
      if (tid == 0) picked[r] = best;
      last = best;
      if (best.flat < 0) {
        for (int i = r + tid; i < k; i += kThreads) picked[i] = Best{0.0, -1};
        break;
      }
    }
  }
  __syncthreads();
  if (tid < k) {
    const Best e = picked[tid];
    const bool none = e.flat < 0;
    const int b = none ? 0 : e.flat / w.c.vocab, token = e.flat - b * w.c.vocab;
    const int64_t at = int64_t(seq) * k + tid;
    w.c.parent[at] = none ? -1 : seq * nb + b;
    w.c.token[at] = none ? -1 : token;
    w.c.out_score[at] = none ? -INFINITY : float(e.total);
    if (w.c.out_done)
      w.c.out_done[at] = !none && (rows[b].state == 2 || token == w.c.eos) ? 1 : 0;
  }
}

int64_t chunks_of(const BeamCall &c) { return (c.vocab + kChunk - 1) / kChunk; }

}  // namespace

size_t swamp_beam_scratch_bytes(const BeamCall &c) {
  const size_t parts = size_t(c.n_seq) * size_t(c.n_beam) * size_t(chunks_of(c));
  return swamp::scratch_round(parts * size_t(c.n_out) * sizeof(Entry)) +
         swamp::scratch_round(parts * sizeof(Part));
}

int swamp_launch_beam_select(const BeamCall &c, swamp::Scratch &sc, hipStream_t s) {
  Work w;
  w.c = c;
  w.chunks = int(chunks_of(c));
  const int64_t parts = int64_t(c.n_seq) * c.n_beam * w.chunks;  // below 2^31
  w.list = static_cast<Entry *>(sc.get(size_t(parts) * size_t(c.n_out) * sizeof(Entry)));
  w.part = static_cast<Part *>(sc.get(size_t(parts) * sizeof(Part)));
  if (!w.list || !w.part) return SWAMP_EWORKSPACE;
  if (c.type == SWAMP_F32) chunk_kernel<float><<<unsigned(parts), kThreads, 0, s>>>(w);
  else if (c.type == SWAMP_F16) chunk_kernel<_Float16><<<unsigned(parts), kThreads, 0, s>>>(w);
  else chunk_kernel<__bf16><<<unsigned(parts), kThreads, 0, s>>>(w);
  join_kernel<<<unsigned(c.n_seq), kThreads, 0, s>>>(w);
  return hipGetLastError() == hipSuccess ? SWAMP_OK : SWAMP_ELAUNCH;
}
