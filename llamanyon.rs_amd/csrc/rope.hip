// rope.hip -- rotary positions (swamp_rope) and the paged cache's append
// (swamp_kv_append): replaces the engine's rotation of q and k
// (swamp-engine/src/ops.rs:20-54) and the copy of k and v into its cache
// (cache.rs) for all new tokens of a batch.
//
// Mathematics: pair (a, b) of pair index i at position p becomes
//   (a c - b s, a s + b c),  c = m cos(p f_i),  s = m sin(p f_i).
// The angle is taken in 64 bits (p f_i has up to 20 integer bits at far
// positions, which fp32 would lose from the fraction), reduced to a quarter
// turn there and handed to fp32 Taylor sums: |x| <= pi/4, next term below
// 2e-9 (sine) and 2e-10 (cosine).  Everything else is fp32, rounded once to
// the output's type.
//
// Bound by HBM for prompts, by the launch for single tokens.  A workgroup takes
// one token and 256 / (units a head) heads at a time; a thread owns the same
// unit of every head it takes, so that its angles serve kHeads heads, whose
// loads are issued before the angles are computed.  A unit is V pairs (V = 4:
// 16 bytes of fp32, 8 of 16 bits a load), or 2 V passing dims.
//
// Measured: 4096 tokens of 32 heads of 128 dims in bf16 14.5 us, 5086 tokens of 48
// heads from fp32 into a bf16 cache 39.5 us, 4.6 TB/s both (a device copy: 4.9);
// one token 7.6 us, the call itself.
#include "paging.hpp"
#include "swamp_common.hpp"

#include <type_traits>

namespace {

constexpr int kThreads = 256;
constexpr int kHeads = 2;  // heads a thread takes

template <typename T>
struct Vec4 {
  typedef T type __attribute__((ext_vector_type(4)));
};

template <int V, typename T>
__device__ __forceinline__ void load(const T *p, float *r) {
  if constexpr (V == 4) {
    const auto v = *reinterpret_cast<const typename Vec4<T>::type *>(p);
#pragma unroll
    for (int j = 0; j < 4; j++) r[j] = float(v[j]);
  } else {
    r[0] = float(p[0]);
  }
}
template <int V, typename T>
__device__ __forceinline__ void store(T *p, const float *r) {
  if constexpr (V == 4) {
    typename Vec4<T>::type v;
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = T(r[j]);
    *reinterpret_cast<typename Vec4<T>::type *>(p) = v;
  } else {
    p[0] = T(r[0]);
  }
}

// cos and sin of p f radians, times m.
__device__ __forceinline__ void turn(double p, double f, float m, float &c, float &s) {
  constexpr double kQuarters = 0.63661977236758134308;  // 2 / pi
  double t = p * f * kQuarters;                         // quarter turns
  t -= 4.0 * __builtin_rint(0.25 * t);                  // -2 .. 2
  const double q = __builtin_rint(t);
  const float x = float(t - q) * 1.57079632679489662f;
  const float z = x * x;
  float sn = 2.7557319e-6f;  // 1 / 9!
  sn = __builtin_fmaf(sn, z, -1.9841270e-4f);
  sn = __builtin_fmaf(sn, z, 8.3333333e-3f);
  sn = __builtin_fmaf(sn, z, -1.6666667e-1f);
  sn = __builtin_fmaf(sn * z, x, x);
  float cs = -2.7557319e-7f;  // -1 / 10!
  cs = __builtin_fmaf(cs, z, 2.4801587e-5f);
  cs = __builtin_fmaf(cs, z, -1.3888889e-3f);
  cs = __builtin_fmaf(cs, z, 4.1666667e-2f);
  cs = __builtin_fmaf(cs, z, -0.5f);
  cs = __builtin_fmaf(cs, z, 1.0f);
  const int k = int(q) & 3;
  const float a = (k & 1) ? sn : cs, b = (k & 1) ? cs : sn;
  c = m * ((k == 1 || k == 2) ? -a : a);
  s = m * ((k & 2) ? -b : b);
}

// The pairs of a head, cut into units of V pairs (V divides n_rot / 2, or n_rot
// is 0) and 2 V passing dims.
struct Pairs {
  const double *freqs;
  float m;
  int rot;    // dims that turn
  int units;  // units of a head
  uint32_t active;  // threads of a workgroup with a unit: whole heads
};

// Values of unit u of one head: lo and hi are the pairs' first and second
// elements as they lie in memory (pairs layout: the unit's first and last V).
template <int V, bool kHalves>
__device__ __forceinline__ int place(const Pairs &g, int u, int &gap) {
  const int turning = g.rot / (2 * V);
  if (u >= turning) {
    gap = V;
    return g.rot + (u - turning) * 2 * V;
  }
  gap = kHalves ? g.rot / 2 : V;
  return kHalves ? u * V : u * 2 * V;
}

template <int V, bool kHalves>
__device__ __forceinline__ void rotate(float *lo, float *hi, const float *c, const float *s) {
  if constexpr (kHalves) {
#pragma unroll
    for (int j = 0; j < V; j++) {
      const float a = lo[j], b = hi[j];
      lo[j] = a * c[j] - b * s[j];
      hi[j] = a * s[j] + b * c[j];
    }
  } else {
    float v[2 * V];
#pragma unroll
    for (int j = 0; j < V; j++) v[j] = lo[j], v[V + j] = hi[j];
#pragma unroll
    for (int j = 0; j < V; j++) {
      const float a = v[2 * j], b = v[2 * j + 1];
      v[2 * j] = a * c[j] - b * s[j];
      v[2 * j + 1] = a * s[j] + b * c[j];
    }
#pragma unroll
    for (int j = 0; j < V; j++) lo[j] = v[j], hi[j] = v[V + j];
  }
}

template <int V>
__device__ __forceinline__ void angles(const Pairs &g, int u, double pos, float *c, float *s) {
#pragma unroll
  for (int j = 0; j < V; j++) c[j] = 1.0f, s[j] = 0.0f;
  if (u < g.rot / (2 * V)) {
#pragma unroll
    for (int j = 0; j < V; j++) turn(pos, g.freqs[u * V + j], g.m, c[j], s[j]);
  }
}

template <typename XT, typename OT, int V, bool kHalves>
__global__ void __launch_bounds__(kThreads)
    rope_kernel(Pairs g, const int32_t *__restrict__ d_pos, const XT *x, int64_t x_stride, OT *out,
                int64_t out_stride, int n_heads, int dim) {
  // x and out may be the same rows: a thread reads its elements before it
  // writes them, and nobody else touches them
  if (threadIdx.x >= g.active) return;
  const int u = int(threadIdx.x) % g.units, per = int(g.active) / g.units;
  const int h0 = int(blockIdx.y) * per * kHeads + int(threadIdx.x) / g.units;
  int gap;
  const int e = place<V, kHalves>(g, u, gap);
  const XT *xr = x + int64_t(blockIdx.x) * x_stride;
  OT *orow = out + int64_t(blockIdx.x) * out_stride;
  float lo[kHeads][V], hi[kHeads][V];
#pragma unroll
  for (int k = 0; k < kHeads; k++) {
    const int h = h0 + k * per;
    if (h < n_heads) {
      load<V>(xr + h * dim + e, lo[k]);
      load<V>(xr + h * dim + e + gap, hi[k]);
    }
  }
  float c[V], s[V];
  angles<V>(g, u, double(d_pos[blockIdx.x]), c, s);
  const bool turns = u < g.rot / (2 * V);
#pragma unroll
  for (int k = 0; k < kHeads; k++) {
    const int h = h0 + k * per;
    if (h >= n_heads) continue;
    if (turns) rotate<V, kHalves>(lo[k], hi[k], c, s);
    store<V>(orow + h * dim + e, lo[k]);
    store<V>(orow + h * dim + e + gap, hi[k]);
  }
}

// The sequence of row t: every wave counts the sequences that end at or before
// it, 64 at a time (loads that do not wait for one another).
__device__ __forceinline__ int seq_of_row(const swamp::SeqBatch &b, int t) {
  int n = 0;
  for (int s0 = 0; s0 < b.n_seq; s0 += 64) {
    const int s = s0 + int(threadIdx.x & 63);
    const bool past = s < b.n_seq && b.first[s + 1] <= t;
    n += __builtin_popcountll(__ballot(past));
  }
  return n;
}

// Heads 0 .. n_heads - 1 of a token are q (to q_out), then n_kv of k and n_kv of
// v (to the cache).
template <typename XT, typename CT, int V, bool kHalves>
__global__ void __launch_bounds__(kThreads)
    append_kernel(swamp::PagedCache cache, swamp::SeqBatch b, Pairs g, const XT *__restrict__ q,
                  const XT *__restrict__ k, const XT *__restrict__ v, int64_t q_stride,
                  int64_t k_stride, int64_t v_stride, CT *__restrict__ q_out, int64_t q_out_stride,
                  int n_heads) {
  const int t = int(blockIdx.x);
  const int u = int(threadIdx.x) % g.units, per = int(g.active) / g.units;
  const int h0 = int(blockIdx.y) * per * kHeads + int(threadIdx.x) / g.units;
  const bool idle = threadIdx.x >= g.active;
  const int total = n_heads + 2 * cache.n_kv;
  int gap;
  const int e = place<V, kHalves>(g, u, gap);
  float lo[kHeads][V], hi[kHeads][V];
#pragma unroll
  for (int j = 0; j < kHeads; j++) {
    const int h = h0 + j * per;
    if (idle || h >= total) continue;
    const int kh = h - n_heads, vh = kh - cache.n_kv;
    const XT *src = kh < 0   ? q + t * q_stride + h * cache.dim
                    : vh < 0 ? k + t * k_stride + kh * cache.dim
                             : v + t * v_stride + vh * cache.dim;
    load<V>(src + e, lo[j]);
    load<V>(src + e + gap, hi[j]);
  }
  const int sq = seq_of_row(b, t);
  if (sq >= b.n_seq || t < b.first[sq]) return;  // padding
  // first[sq + 1] > t >= 0, so the difference fits
  const int pos = int(max(int64_t(b.len[sq]) - (int64_t(b.first[sq + 1]) - t), int64_t(-1)));
  const int64_t col = swamp::page_col(pos, cache.page_shift);
  int32_t id = -1;
  if (swamp::page_col_ok(pos, col, b.pages_stride)) id = b.pages[sq * b.pages_stride + col];
  const bool cached = swamp::page_ok(id, cache.n_pages);
  if (!cached && b.bad && threadIdx.x == 0) *b.bad = 1;
  if (idle) return;
  float c[V], s[V];
  angles<V>(g, u, double(pos), c, s);
  const bool turns = u < g.rot / (2 * V);
#pragma unroll
  for (int j = 0; j < kHeads; j++) {
    const int h = h0 + j * per;
    if (h >= total) continue;
    const int kh = h - n_heads, vh = kh - cache.n_kv;
    if (turns && vh < 0) rotate<V, kHalves>(lo[j], hi[j], c, s);
    CT *dst;
    if (kh < 0) {
      dst = q_out + t * q_out_stride + h * cache.dim;
    } else {
      if (!cached) continue;
      dst = reinterpret_cast<CT *>(vh < 0 ? cache.k : cache.v) +
            swamp::slot_offset(id, pos, vh < 0 ? kh : vh, cache.page_shift, cache.page_stride,
                               cache.head_stride, cache.slot_stride);
    }
    store<V>(dst + e, lo[j]);
    store<V>(dst + e + gap, hi[j]);
  }
}

int launched() { return hipGetLastError() == hipSuccess ? SWAMP_OK : SWAMP_ELAUNCH; }

// V = 4 needs whole units (n_rot and dim multiples of 8) and rows that 4
// elements of either type load aligned.
bool wide(const void *p, uint32_t type, int64_t stride) {
  return reinterpret_cast<uintptr_t>(p) % (type == SWAMP_F32 ? 16 : 8) == 0 && stride % 4 == 0;
}

Pairs pairs_of(const swamp_rope_spec *r, int dim, int v) {
  Pairs g;
  g.freqs = r ? r->d_freqs : nullptr;
  g.m = r ? r->mscale : 1.0f;
  g.rot = r ? r->n_rot : 0;
  g.units = dim / (2 * v);
  g.active = uint32_t(kThreads / g.units * g.units);
  return g;
}

dim3 grid_of(const Pairs &g, int n_tok, int heads) {
  const int per = int(g.active) / g.units * kHeads;
  return dim3(unsigned(n_tok), unsigned((heads + per - 1) / per));
}

// f with the element type of a dtype code that api.hip has checked.
template <typename F>
void with_type(uint32_t t, F f) {
  if (t == SWAMP_F32) f(float{});
  else if (t == SWAMP_F16) f(_Float16{});
  else f(__bf16{});
}
// f with V and the layout as constants.
template <typename F>
void with_form(bool v4, bool halves, F f) {
  typedef std::integral_constant<int, 4> four;
  typedef std::integral_constant<int, 1> one;
  if (v4 && halves) f(four{}, std::true_type{});
  else if (v4) f(four{}, std::false_type{});
  else if (halves) f(one{}, std::true_type{});
  else f(one{}, std::false_type{});
}

}  // namespace

int swamp_launch_rope(const swamp_rope_spec *r, const int32_t *d_pos, const void *d_x,
                      uint32_t x_type, int64_t x_stride, void *d_out, uint32_t out_type,
                      int64_t out_stride, int n_tok, int n_heads, int head_dim, hipStream_t s) {
  const bool v4 = head_dim % 8 == 0 && r->n_rot % 8 == 0 && wide(d_x, x_type, x_stride) &&
                  wide(d_out, out_type, out_stride);
  const Pairs g = pairs_of(r, head_dim, v4 ? 4 : 1);
  const dim3 grid = grid_of(g, n_tok, n_heads);
  with_type(x_type, [&](auto xt) {
    with_type(out_type, [&](auto ot) {
      with_form(v4, r->layout == SWAMP_ROPE_HALVES, [&](auto v, auto halves) {
        rope_kernel<decltype(xt), decltype(ot), decltype(v)::value, decltype(halves)::value>
            <<<grid, kThreads, 0, s>>>(g, d_pos, static_cast<const decltype(xt) *>(d_x), x_stride,
                                       static_cast<decltype(ot) *>(d_out), out_stride, n_heads,
                                       head_dim);
      });
    });
  });
  return launched();
}

int swamp_launch_kv_append(const swamp::PagedCache &cache, const swamp::SeqBatch &b, uint32_t dtype,
                           const swamp_rope_spec *r, const void *d_q, const void *d_k,
                           const void *d_v, uint32_t x_type, int64_t q_stride, int64_t k_stride,
                           int64_t v_stride, void *d_q_out, int64_t q_out_stride, int n_heads,
                           hipStream_t s) {
  const bool v4 = (!r || r->n_rot % 8 == 0) && wide(d_k, x_type, k_stride) &&
                  wide(d_v, x_type, v_stride) &&
                  (n_heads == 0 ||
                   (wide(d_q, x_type, q_stride) && wide(d_q_out, dtype, q_out_stride)));
  const Pairs g = pairs_of(r, cache.dim, v4 ? 4 : 1);
  const dim3 grid = grid_of(g, b.n_tok, n_heads + 2 * cache.n_kv);
  auto go = [&](auto ct) {
    with_type(x_type, [&](auto xt) {
      with_form(v4, r && r->layout == SWAMP_ROPE_HALVES, [&](auto v, auto halves) {
        typedef decltype(xt) X;
        typedef decltype(ct) C;
        append_kernel<X, C, decltype(v)::value, decltype(halves)::value>
            <<<grid, kThreads, 0, s>>>(cache, b, g, static_cast<const X *>(d_q),
                                       static_cast<const X *>(d_k), static_cast<const X *>(d_v),
                                       q_stride, k_stride, v_stride, static_cast<C *>(d_q_out),
                                       q_out_stride, n_heads);
      });
    });
  };
  if (dtype == SWAMP_F16) go(_Float16{});
  else go(__bf16{});
  return launched();
}
