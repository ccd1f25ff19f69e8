// rows_i8.hip -- 8-bit codes with one scale a row (swamp_quantize_rows) and their
// products (swamp_gemm_rows_i8): y[i][r] = sx_i sw_r sum_k x[i][k] w[r][k].
//
// The scales stand outside the sum, so the sum is the matrix cores' own int32 (exact:
// 131071 terms of at most 2^14 stay below 2^31) and one product an output is left for
// the vector unit, where scales a block of 32 cost a conversion and an FMA for every 32
// terms (gemm_i8.hip).
//
// Tiles.  Eight waves a workgroup (64 x 128: four), WM x WN V_MFMA_I32_32X32X32_I8 blocks
// each: two waves a SIMD fill each other's waits at the barriers and in the epilogue (four
// waves of twice the blocks: 640 x 14336 x 4096 68 us, 58 so; 3000 x 5000 x 5000 107, 95).  A
// K step is 64 codes: a stage holds the tile's rows of x, then of w, 64 bytes each, 16-byte
// chunks XOR-swizzled by (row / 4) % 4, so that 16 consecutive lanes of a fragment read
// meet no bank twice.  Stages are filled by direct-to-LDS DMA, two steps at a time, four to
// twelve steps ahead; one barrier a step, between its halves, whose counted wait leaves
// the DMAs of the steps behind the next one in flight.
//
// The last step of a sum is taken apart from the loop: its codes of x behind column K
// are cleared, so that what lies in w there (a row's padding) counts for nothing.
//
// Measured: 4096 rows of x by 28672 x 4096 in tiles of 256 x 256 430 to 475 us (2.0 to 2.2
// POP/s, bf16 out), bound by the matrix pipes, busy 65% of the time at the clock that the
// card holds, and by each tile's start and end (about 12 of its 66 us); 64 rows by the same
// weights in tiles of 64 x 128 26.7 us, 4.7 TB/s, bound by HBM.
#include "rows_plan.hpp"
#include "swamp_common.hpp"
#include "swamp_items.hpp"
#include "wave.hpp"

#include <algorithm>
#include <mutex>
#include <type_traits>

namespace {

using swamp::GemmI8Call;
using swamp_rows::Plan;

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));

// ---- quantizer ------------------------------------------------------------
// A workgroup a row.  HBM's: a row is read once where it fits its threads' registers (8 to
// 64 elements each), else the second look is the cache's.
//
// A code is rint(x / s), the quotient rounded to fp32.  x times 1 / s lies within 127.1 2^-23
// of x / s, and that within 127 2^-24 of the rounded quotient, 2.3e-5 in all: where it is
// further than 2^-15 from half way between two codes it names the code, and only elsewhere
// (1024 elements of a wave meet one in 6 of 100) is there a division.  From HBM, into codes
// that go there: 4096 x 4096 bf16 15.9 us (3.2 TB/s; 19.0 with a division for each), f32 17.0
// (4.9 TB/s; 19.4), 4096 x 14336 bf16 41.0 (4.3 TB/s; 50.2).

// The largest |x| of a workgroup's elements, as bits: infinity and NaN come last.
__device__ __forceinline__ uint32_t raise(uint32_t top, float x) {
  return max(top, __float_as_uint(x) & 0x7FFFFFFFu);
}
__device__ __forceinline__ uint32_t workgroup_max(uint32_t top) {
  __shared__ uint32_t tops[16];
  top = swamp::group_max(top, 64);
  const int waves = int(blockDim.x) >> 6;
  if (waves == 1) return top;
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  top = tops[0];
  for (int i = 1; i < waves; i++) top = max(top, tops[i]);
  return top;
}
// The row's scale, written; 0 or less: its codes are 0.
__device__ __forceinline__ float scale_of(uint32_t top, float *to) {
  const bool fine = top < 0x7F800000u;
  float s = __uint_as_float(top) / 127.f;
  if (s < 1.17549435e-38f) s = 0.f;
  if (threadIdx.x == 0) *to = fine ? s : __builtin_nanf("");
  return fine ? s : -1.f;
}
// The codes of N elements of a row whose scale is s, 1 / s = r.
template <int N, typename XT>
__device__ __forceinline__ void codes_of(const XT *x, float s, float r, int8_t *c) {
  if (!(s > 0.f)) {
#pragma unroll
    for (int k = 0; k < N; k++) c[k] = 0;
    return;
  }
  float far = 0.f;
#pragma unroll
  for (int k = 0; k < N; k++) {
    const float t = float(x[k]) * r, whole = __builtin_rintf(t);
    far = fmaxf(far, fabsf(t - whole));
    c[k] = int8_t(int(whole));
  }
  if (far > 0.5f - 0x1p-15f) {
#pragma unroll
    for (int k = 0; k < N; k++) c[k] = int8_t(int(__builtin_rintf(float(x[k]) / s)));
  }
}

// N elements of any place that their type allows.
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Vec {
  T v[N];
};
// Those at place `at` of a row of n; zeros behind it.
template <typename XT, int V>
__device__ __forceinline__ Vec<XT, V> take(const XT *row, int at, int n) {
  if (at <= n - V) return *reinterpret_cast<const Vec<XT, V> *>(row + at);
  Vec<XT, V> x;
#pragma unroll
  for (int k = 0; k < V; k++) x.v[k] = k < n - at ? row[at + k] : XT(0);
  return x;
}
template <typename XT, int V>
__device__ __forceinline__ void give(int8_t *out, int at, int n, const Vec<XT, V> &x, float s,
                                     float r) {
  Vec<int8_t, V> c;
  codes_of<V>(x.v, s, r, c.v);
  if (at <= n - V) {
    *reinterpret_cast<Vec<int8_t, V> *>(out + at) = c;
  } else {
#pragma unroll
    for (int k = 0; k < V; k++)
      if (k < n - at) out[at + k] = c.v[k];
  }
}

// Rows of any length.
template <typename XT>
__global__ void __launch_bounds__(1024) quantize_any_kernel(const XT *__restrict__ x,
                                                            int64_t x_stride,
                                                            int8_t *__restrict__ q,
                                                            int64_t q_stride,
                                                            float *__restrict__ scale, int n) {
  constexpr int V = 16 / int(sizeof(XT));
  const XT *row = x + int64_t(blockIdx.x) * x_stride;
  int8_t *out = q + int64_t(blockIdx.x) * q_stride;
  uint32_t top = 0;
#pragma unroll 4
  for (int64_t at = int(threadIdx.x) * V; at < n; at += 1024 * V) {
    const Vec<XT, V> v = take<XT, V>(row, int(at), n);
#pragma unroll
    for (int k = 0; k < V; k++) top = raise(top, float(v.v[k]));
  }
  const float s = scale_of(workgroup_max(top), scale + blockIdx.x), r = 1.f / s;
  for (int64_t at = int(threadIdx.x) * V; at < n; at += 1024 * V)
    give<XT, V>(out, int(at), n, take<XT, V>(row, int(at), n), s, r);
}

// Rows of up to kEach times the threads, 16 bytes a load.
template <typename XT, int kEach>
__global__ void __launch_bounds__(1024) quantize_kernel(const XT *__restrict__ x, int64_t x_stride,
                                                        int8_t *__restrict__ q, int64_t q_stride,
                                                        float *__restrict__ scale, int n) {
  constexpr int V = 16 / int(sizeof(XT)), kLoads = kEach / V;
  const XT *row = x + int64_t(blockIdx.x) * x_stride;
  int8_t *out = q + int64_t(blockIdx.x) * q_stride;
  auto place = [](int j) { return (j * int(blockDim.x) + int(threadIdx.x)) * V; };
  Vec<XT, V> v[kLoads];
#pragma unroll
  for (int j = 0; j < kLoads; j++) v[j] = take<XT, V>(row, place(j), n);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < kLoads; j++)
#pragma unroll
    for (int k = 0; k < V; k++) top = raise(top, float(v[j].v[k]));
  const float s = scale_of(workgroup_max(top), scale + blockIdx.x), r = 1.f / s;
#pragma unroll
  for (int j = 0; j < kLoads; j++) give<XT, V>(out, place(j), n, v[j], s, r);
}

// ---- products -------------------------------------------------------------
template <int WM, int WN, int NWM, int NWN>
struct Shape {
  static constexpr int NW = NWM * NWN, kThreads = 64 * NW;
  static constexpr int TM = 32 * WM * NWM, TN = 32 * WN * NWN;  // tile: rows of x, of w
  static constexpr int kStage = (TM + TN) * 64;
  // Pairs of steps on their way, as many as LDS holds with one step more, 6 at most.
  static constexpr int kPairs = std::min(6, (160 * 1024 / kStage - 1) / 2);
  static constexpr int kStages = 2 * kPairs + 1;
  static constexpr int kSmem = kStages * kStage;
  static constexpr int kDma = (TM + TN) / (16 * NW);  // 1 KB DMAs of a wave and step
  static constexpr int kDma0 = (kDma + 1) / 2;        // of them in a step's first half
  static_assert(TM % (16 * NW) == 0 && TN % (16 * NW) == 0, "a DMA fills 16 rows of one operand");
  static_assert(kPairs >= 2 && kSmem <= 160 * 1024, "LDS");
  static_assert(2 * kPairs * kDma <= 63, "the memory counter");
};

// One 16-byte-per-lane DMA into LDS (lane L writes lds + 16 L).  Not a template: the
// host pass rejects the LDS address-space cast inside a template instantiation.
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint8_t *lds, uint32_t voff,
                                      uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)lds, 16,
                                           voff, soff, 0, 0);
}

struct Work {
  GemmI8Call c;
  int tiles_m, tiles_n;
  int group;                 // tiles of x that share a run of tiles of w
  int pieces, steps;         // pieces of the sum, 64-code steps of a piece
  int32_t *part;             // [piece][m][n], pieces > 1
};

// sum times both scales into y, added to what is there or not.
template <typename Y>
__device__ __forceinline__ void put(Y *y, int sum, float sx, double sw, int add) {
  float v = float(double(sx) * sw * double(sum));
#ifdef __HIP_DEVICE_COMPILE__
  asm volatile("" : "+v"(v));  // (or the compiler rounds to 16 bits from 64 at once)
#endif
  *y = Y(add ? float(*y) + v : v);
}
__device__ __forceinline__ void put_at(const GemmI8Call &c, int m, int n, int sum) {
  const int64_t at = int64_t(m) * c.y_stride + n;
  const float sx = c.x_scale[m];
  const double sw = double(c.w_scale[n]);
  if (c.y_type == SWAMP_F32) put(static_cast<float *>(c.y) + at, sum, sx, sw, c.accumulate);
  else if (c.y_type == SWAMP_F16) put(static_cast<_Float16 *>(c.y) + at, sum, sx, sw, c.accumulate);
  else put(static_cast<__bf16 *>(c.y) + at, sum, sx, sw, c.accumulate);
}

// Between LDS that a wave's lanes write and its other lanes read: LDS keeps a wave's order by
// itself, and this makes the compiler keep it.  No instruction of its own.
__device__ __forceinline__ void lanes_meet() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// 32 rows of kCols sums, in LDS, to rows m0 on and columns n0 on of y, whose ends may lie
// among them.
template <int kCols, int kPitch, typename Y>
__device__ __forceinline__ void store_strip(const GemmI8Call &c, const int32_t *strip,
                                            const float *scales, int m0, int n0, int lane) {
  constexpr int V = 16 / int(sizeof(Y)), kLanes = kCols / V, kRows = 64 / kLanes;
  const int col = lane % kLanes * V, n = n0 + col;
  if (n >= c.n) return;
  float sw[V];
#pragma unroll
  for (int v = 0; v < V; v++) sw[v] = c.w_scale[min(n + v, c.n - 1)];
  for (int row = lane / kLanes; row < 32 && m0 + row < c.m; row += kRows) {
    const float sx = scales[row];
    Y *y = static_cast<Y *>(c.y) + int64_t(m0 + row) * c.y_stride + n;
    const int32_t *sum = strip + row * kPitch + col;
#pragma unroll
    for (int v = 0; v < V; v++)
      if (n + v < c.n) put(y + v, sum[v], sx, double(sw[v]), c.accumulate);
  }
}

template <typename Y, int WM, int WN, int NWM, int NWN>
__global__ void __launch_bounds__(64 * NWM * NWN, 1) gemm_kernel(Work wk) {
  using S = Shape<WM, WN, NWM, NWN>;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const GemmI8Call &c = wk.c;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // Hardware ids i, i + 8, ... run on XCD i % 8: each takes a contiguous run of the
  // tiles in grouped order, so that its CUs share few rows of either side in its L2.
  const int units = int(gridDim.x), b = int(blockIdx.x);
  const int q = units / 8, rem = units % 8, xcd = b % 8;
  const int u = xcd * q + min(xcd, rem) + b / 8;
  const int t = u / wk.pieces, piece = u % wk.pieces;
  const int grp = t / (wk.group * wk.tiles_n), g0 = grp * wk.group;
  const int gs = min(wk.tiles_m - g0, wk.group), r = t - grp * wk.group * wk.tiles_n;
  const int m0 = (g0 + r % gs) * S::TM, n0 = r / gs * S::TN;
  const int K = c.k, KT = (K + 63) / 64;
  const int kt0 = piece * wk.steps, kt1 = min(KT, kt0 + wk.steps);
  // Where every row of w is one workgroup's, each begins its whole pairs of steps at
  // another place: side by side they would read the same columns of rows a power of two
  // apart, which are a few memory channels'.
  const int turn = wk.tiles_m == 1 && (kt1 - kt0) % 2 == 0 && K % 64 == 0
                       ? 2 * (5 * (t + piece) % ((kt1 - kt0) / 2)) : 0;

  const uint32_t xp = uint32_t(c.x_stride), wp = uint32_t(c.w_stride), k16 = uint32_t(K + 15) & ~15u;
  const uint32_t xm = uint32_t(min(S::TM, c.m - m0) - 1), wn_ = uint32_t(min(S::TN, c.n - n0) - 1);
  const uint32_t x_bytes = xm * xp + k16, w_bytes = wn_ * wp + k16;
  // DMA i of wave w fills stage rows R = 16 (NW i + w) .. R + 15: lane L writes row
  // R + L / 4, physical chunk L % 4, which holds logical chunk (L % 4) ^ (L / 16 % 4).
  const uint32_t lrow4 = uint32_t(lane >> 2), chunk = uint32_t((lane & 3) ^ ((lane >> 4) & 3)) << 4;
  const uint32_t xv = lrow4 * xp + chunk, wv = lrow4 * wp + chunk;

  // DMAs [i0, i1) of the steps kt and kt + 1: 64 bytes of a row and the 64 behind them
  // directly after one another, so that the first level cache gets the line once.
  auto dma_pair = [&](int kt, int stage, auto i0c, auto i1c) {
    constexpr int i0 = decltype(i0c)::value, i1 = decltype(i1c)::value;
    uint8_t *st = smem + S::kStage * stage;
    uint8_t *st1 = smem + S::kStage * (stage + 1 == S::kStages ? 0 : stage + 1);
    const int at = kt + turn < kt1 ? kt + turn : kt + turn - (kt1 - kt0);
    // (past the end: nothing is fetched, and the count of DMAs stays)
    const __amdgpu_buffer_rsrc_t xr =
        swamp::make_rsrc(c.x + m0 * c.x_stride, kt < kt1 ? x_bytes : 0u);
    const __amdgpu_buffer_rsrc_t wr =
        swamp::make_rsrc(c.w + n0 * c.w_stride, kt < kt1 ? w_bytes : 0u);
#pragma unroll
    for (int i = i0; i < i1; i++) {
      const int R = 16 * (S::NW * i + wave);
      if (16 * S::NW * i < S::TM) {
        dma16(xr, st + R * 64, xv, uint32_t(R) * xp + uint32_t(at) * 64u);
        dma16(xr, st1 + R * 64, xv, uint32_t(R) * xp + uint32_t(at) * 64u + 64u);
      } else {
        dma16(wr, st + R * 64, wv, uint32_t(R - S::TM) * wp + uint32_t(at) * 64u);
        dma16(wr, st1 + R * 64, wv, uint32_t(R - S::TM) * wp + uint32_t(at) * 64u + 64u);
      }
    }
  };
  using I0 = std::integral_constant<int, 0>;
  using IH = std::integral_constant<int, S::kDma0>;
  using IE = std::integral_constant<int, S::kDma>;

  // Fragment of half s (codes 32 s .. 32 s + 31 of the step): lane l reads row l % 32 of
  // its 32-row block, logical chunk 2 s + l / 32.
  const int wm = wave % NWM, wn = wave / NWM;
  const uint32_t lrow = uint32_t(lane & 31) * 64;
  const uint32_t sw = uint32_t((lane >> 2) & 3);
  const uint32_t loff0 = lrow + (((uint32_t(lane >> 5)) ^ sw) << 4);
  const uint32_t loff1 = lrow + (((2u + uint32_t(lane >> 5)) ^ sw) << 4);
  const uint32_t a_off = uint32_t(wm * WM * 32) * 64, b_off = uint32_t(S::TM + wn * WN * 32) * 64;

  auto read_frags = [&](const uint8_t *st, uint32_t loff, i32x4 (&fa)[WM], i32x4 (&fb)[WN]) {
#pragma unroll
    for (int i = 0; i < WM; i++)
      fa[i] = *reinterpret_cast<const i32x4 *>(st + a_off + 2048 * i + loff);
#pragma unroll
    for (int j = 0; j < WN; j++)
      fb[j] = *reinterpret_cast<const i32x4 *>(st + b_off + 2048 * j + loff);
  };

  i32x16 acc[WM][WN];
#pragma unroll
  for (int i = 0; i < WM; i++)
#pragma unroll
    for (int j = 0; j < WN; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[i][j][e] = 0;

  auto mfmas = [&](const i32x4 (&fa)[WM], const i32x4 (&fb)[WN]) {
#pragma unroll
    for (int i = 0; i < WM; i++)
#pragma unroll
      for (int j = 0; j < WN; j++)
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[i], fb[j], acc[i][j], 0, 0, 0);
  };

  // Steps go in pairs, 0 and 1, 2 and 3, ...: an odd step s issues the DMA of the pair
  // behind the last one on its way, into the stages of steps s - 2 and s - 1, which every
  // wave finished reading before the barrier of step s - 1.
  constexpr int NS = S::kStages, kPairs = S::kPairs;
#pragma unroll
  for (int p = 0; p < kPairs; p++) {
    dma_pair(kt0 + 2 * p, 2 * p, I0{}, IE{});
    __builtin_amdgcn_sched_barrier(0);
  }
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((kPairs - 1) * 2 * S::kDma) : "memory");

  i32x4 fa0[WM], fb0[WN], fa1[WM], fb1[WN];
  read_frags(smem, loff0, fa0, fb0);

  // A half's instruction order: its products, one fragment read after each of the first
  // WM + WN, its DMAs spread over the rest.
  auto order = [&](auto ndc) {
    constexpr int n_dma = decltype(ndc)::value, R = std::max(1, WM * WN - (WM + WN));
#pragma unroll
    for (int m = 0; m < WM * WN; m++) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // 1 MFMA
      if (m < WM + WN) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // 1 DS read
      } else {
        const int k = m - (WM + WN), nd = (k + 1) * n_dma / R - k * n_dma / R;
#pragma unroll
        for (int d = 0; d < nd; d++) __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);  // DMA
      }
    }
  };
  using N0 = std::integral_constant<int, 0>;
  using D0 = std::integral_constant<int, 2 * S::kDma0>;
  using D1 = std::integral_constant<int, 2 * (S::kDma - S::kDma0)>;

  int cur = 0;
  auto step = [&](int kt, auto odd_c) {
    constexpr bool odd = decltype(odd_c)::value;
    const int nxt = cur + 1 == NS ? 0 : cur + 1;
    const int fill = cur >= 2 ? cur - 2 : cur - 2 + NS, ktf = kt + 2 * kPairs - 1;
    read_frags(smem + S::kStage * cur, loff1, fa1, fb1);
    mfmas(fa0, fb0);
    if constexpr (odd) {
      dma_pair(ktf, fill, I0{}, IH{});
      order(D0{});
    } else {
      order(N0{});
    }
    __builtin_amdgcn_sched_barrier(0);
    // Step kt + 1 is there for every wave, and this one read.  (An even step's next came
    // with it; else all but the pairs behind the next and what this step has issued.)
    if constexpr (odd)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((kPairs - 2) * 2 * S::kDma +
                                                                       2 * S::kDma0)
                   : "memory");
    else
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    read_frags(smem + S::kStage * nxt, loff0, fa0, fb0);
    mfmas(fa1, fb1);
    if constexpr (odd) {
      dma_pair(ktf, fill, IH{}, IE{});
      order(D1{});
    } else {
      order(N0{});
    }
    __builtin_amdgcn_sched_barrier(0);
    cur = nxt;
  };
  int kt = kt0;
  for (; kt + 1 < kt1 - 1; kt += 2) {
    step(kt, std::false_type{});
    step(kt + 1, std::true_type{});
  }
  if (kt < kt1 - 1) step(kt, std::false_type{});
  // The last step, without what lies behind column K.
  read_frags(smem + S::kStage * cur, loff1, fa1, fb1);
  auto cut = [&](i32x4 (&f)[WM], int half) {
    const int left = K - (kt1 - 1) * 64 - 32 * half - 16 * (lane >> 5);  // codes of this lane's 16
    uint32_t keep[4];
#pragma unroll
    for (int d = 0; d < 4; d++) {
      const int k = left - 4 * d;
      keep[d] = k >= 4 ? ~0u : k <= 0 ? 0u : (1u << (8 * k)) - 1;
    }
#pragma unroll
    for (int i = 0; i < WM; i++)
#pragma unroll
      for (int d = 0; d < 4; d++) f[i][d] &= int32_t(keep[d]);
  };
  cut(fa0, 0);
  mfmas(fa0, fb0);
  cut(fa1, 1);
  mfmas(fa1, fb1);
  // A block's result: lane holds column (row of w) lane % 32, rows (of x) 8 (e / 4) +
  // 4 (lane / 32) + e % 4.
  const int fr = lane & 31, fc = lane >> 5;
  const int mw = m0 + wm * WM * 32 + 4 * fc, nw = n0 + wn * WN * 32 + fr;
  if (wk.pieces > 1) {
    int32_t *part = wk.part + int64_t(piece) * c.m * c.n;
#pragma unroll
    for (int i = 0; i < WM; i++)
#pragma unroll
      for (int j = 0; j < WN; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const int m = mw + 32 * i + 8 * (e >> 2) + (e & 3), n = nw + 32 * j;
          if (m < c.m && n < c.n) part[int64_t(m) * c.n + n] = acc[i][j][e];
        }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no DMA outlives the workgroup
    return;
  }
  // To y through LDS, 32 rows of a wave at a time, so that a store is 16 bytes a lane and
  // whole runs of a row (from the blocks' own layout, one element a lane, a tile of 256 x
  // 256 took 33 us).  Every wave is done with the stages.
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  float *scales = reinterpret_cast<float *>(smem);
  for (int i = tid; i < S::TM; i += S::kThreads) scales[i] = c.x_scale[min(m0 + i, c.m - 1)];
  __syncthreads();
  // (rows 4 apart are written together: 128 bytes apart in the banks)
  constexpr int kCols = 32 * WN, kPitch = kCols + 8;
  static_assert(S::TM * 4 + S::NW * 32 * kPitch * 4 <= S::kSmem, "strips");
  int32_t *strip = reinterpret_cast<int32_t *>(smem + S::TM * 4) + wave * 32 * kPitch;
  auto fill = [&](auto ic) {
    constexpr int i = decltype(ic)::value;
#pragma unroll
    for (int j = 0; j < WN; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) {
        int32_t x = acc[i][j][e];
#ifdef __HIP_DEVICE_COMPILE__
        asm volatile("" : "+v"(x));  // (one by one: as pairs they moved whole blocks to memory)
#endif
        strip[(8 * (e >> 2) + 4 * fc + (e & 3)) * kPitch + 32 * j + fr] = x;
      }
  };
  const int mr = wm * WM * 32, nr = n0 + wn * kCols;  // the wave's first row in the tile, column
  // Ragged tiles, and all tiles of a call that adds to y, element by element: 4096 x 28672 x
  // 4096 bf16 420 us, added 650; 4096 x 4096 x 14336 190 and 230.
  if (m0 + S::TM > c.m || n0 + S::TN > c.n || c.accumulate) {
    auto part = [&](auto ic) {
      constexpr int i = decltype(ic)::value;
      if constexpr (i < WM) {
        lanes_meet();
        fill(ic);
        lanes_meet();
        store_strip<kCols, kPitch, Y>(c, strip, scales + mr + 32 * i, m0 + mr + 32 * i, nr, lane);
      }
    };
    part(std::integral_constant<int, 0>{});
    part(std::integral_constant<int, 1>{});
    part(std::integral_constant<int, 2>{});
    part(std::integral_constant<int, 3>{});
    return;
  }
  // A whole tile: a strip's reads, the next one's writes (LDS keeps their order), and then
  // the first's arithmetic.
  constexpr int V = 16 / int(sizeof(Y)), kLanes = kCols / V, kRows = 64 / kLanes, T = 32 / kRows;
  const int col = lane % kLanes * V, row0 = lane / kLanes;
  double sw_n[V];
#pragma unroll
  for (int v = 0; v < V; v++) sw_n[v] = double(c.w_scale[nr + col + v]);
  Y *y = static_cast<Y *>(c.y) + int64_t(m0 + mr + row0) * c.y_stride + nr + col;
  fill(std::integral_constant<int, 0>{});
  lanes_meet();
  auto whole = [&](auto ic) {
    constexpr int i = decltype(ic)::value;
    if constexpr (i < WM) {
      i32x4 sum[T][V / 4];
      float sx[T];
#pragma unroll
      for (int t = 0; t < T; t++) {
#pragma unroll
        for (int v = 0; v < V / 4; v++)
          sum[t][v] = *reinterpret_cast<const i32x4 *>(strip + (t * kRows + row0) * kPitch + col + 4 * v);
        sx[t] = scales[mr + 32 * i + t * kRows + row0];
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (i + 1 < WM) {
        lanes_meet();
        fill(std::integral_constant<int, i + 1>{});
        lanes_meet();
      }
#pragma unroll
      for (int t = 0; t < T; t++) {
        Vec<Y, V> o;
#pragma unroll
        for (int v = 0; v < V; v++) put(&o.v[v], sum[t][v / 4][v % 4], sx[t], sw_n[v], 0);
        *reinterpret_cast<Vec<Y, V> *>(y) = o;
        y += kRows * c.y_stride;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  whole(std::integral_constant<int, 0>{});
  whole(std::integral_constant<int, 1>{});
  whole(std::integral_constant<int, 2>{});
  whole(std::integral_constant<int, 3>{});
}

// ---- few rows of x --------------------------------------------------------
// The weights' stream bounds it, so they go from memory to registers: a lane holds 16
// codes of one row of w (R tiles of 16 rows), V_MFMA_I32_16X16X64_I8 multiplies 16 rows
// by T times 16 of x.  A workgroup's waves take a share of the columns each, so that a
// short matrix has all its bytes in flight at once, and their sums meet in LDS.  What of
// x lies behind column K is cleared, rows behind the last are the descriptor's zeros.
// One row of 6144 x 4096: 7.6 us, 4.5 of them its bytes at 5.6 TB/s; 32 rows 10.4 (4.6); 64 rows
// of 4096 x 4096 11.9 (3.2): there every workgroup's own reading of x, 16 codes a lane and product.
//
// Waves and steps in flight are what the registers hold: 16 of 128 each, or 8 of 256.
template <int R, int T>
struct Few {
  static constexpr int kWaves = R * T >= 8 ? 8 : 16;
  static constexpr int U = R * T <= 2 || (R == 4 && T == 2) ? 4 : 2;  // and as many to come
};
template <int R, int T>
__global__ void __launch_bounds__((64 * Few<R, T>::kWaves)) few_kernel(GemmI8Call c) {
  constexpr int U = Few<R, T>::U;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  int32_t *parts = reinterpret_cast<int32_t *>(smem);
  const int lane = int(threadIdx.x) & 63, r = lane & 15, h = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int waves = int(blockDim.x) >> 6, KT = (c.k + 63) / 64, n0 = int(blockIdx.x) * 16 * R;
  const int share = (KT + waves - 1) / waves, s0 = min(wave * share, KT), s1 = min(s0 + share, KT);
  const uint32_t xp = uint32_t(c.x_stride), wp = uint32_t(c.w_stride);
  const uint32_t k16 = uint32_t(c.k + 15) & ~15u;
  const __amdgpu_buffer_rsrc_t xr = swamp::make_rsrc(c.x, uint32_t(c.m - 1) * xp + k16);
  const __amdgpu_buffer_rsrc_t wr = swamp::make_rsrc(
      c.w + n0 * c.w_stride, uint32_t(min(16 * R, c.n - n0) - 1) * wp + k16);
  uint32_t xv[T], wv[R];
#pragma unroll
  for (int j = 0; j < T; j++) xv[j] = uint32_t(16 * j + r) * xp + 16u * uint32_t(h);
#pragma unroll
  for (int i = 0; i < R; i++) wv[i] = uint32_t(16 * i + r) * wp + 16u * uint32_t(h);
  i32x4 acc[R][T];
#pragma unroll
  for (int i = 0; i < R; i++)
#pragma unroll
    for (int j = 0; j < T; j++) acc[i][j] = i32x4{0, 0, 0, 0};
  struct Stage {
    i32x4 w[U][R], x[U][T];
  };
  auto load = [&](Stage &st, int s) {
    if (s >= s1) return;
    // (a row's steps one after another: two are a cache line)
    auto from = [&](const __amdgpu_buffer_rsrc_t &rsrc, uint32_t at, int u) {
      return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                           rsrc, at, uint32_t(min(s + u, s1 - 1)) * 64u, 0));
    };
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
      for (int u = 0; u < U; u++) st.w[u][i] = from(wr, wv[i], u);
#pragma unroll
    for (int j = 0; j < T; j++)
#pragma unroll
      for (int u = 0; u < U; u++) st.x[u][j] = from(xr, xv[j], u);
  };
  auto multiply = [&](Stage &st, int s) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (s + u >= s1) break;
      const int left = c.k - (s + u) * 64 - 16 * h;  // columns of this lane's 16
      if ((s + u + 1) * 64 > c.k) {
#pragma unroll
        for (int d = 0; d < 4; d++) {
          const int n = left - 4 * d;
          const int32_t keep = n >= 4 ? ~0 : n <= 0 ? 0 : int32_t((1u << (8 * n)) - 1);
#pragma unroll
          for (int j = 0; j < T; j++) st.x[u][j][d] &= keep;
        }
      }
#pragma unroll
      for (int i = 0; i < R; i++)
#pragma unroll
        for (int j = 0; j < T; j++)
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(st.x[u][j], st.w[u][i], acc[i][j], 0, 0,
                                                            0);
    }
  };
  if (s0 < s1) {
    Stage a, b;
    load(a, s0);
    for (int s = s0; s < s1; s += 2 * U) {
      load(b, s + U);
      multiply(a, s);
      load(a, s + 2 * U);
      multiply(b, s + U);
    }
  }
  // lane: column (row of w) r, rows (of x) 4 h .. 4 h + 3
#pragma unroll
  for (int i = 0; i < R; i++)
#pragma unroll
    for (int j = 0; j < T; j++)
#pragma unroll
      for (int e = 0; e < 4; e++)
        parts[((wave * R + i) * T + j) * 256 + (4 * h + e) * 16 + r] = acc[i][j][e];
  __syncthreads();
  for (int o = int(threadIdx.x); o < R * T * 256; o += int(blockDim.x)) {
    int sum = 0;
    for (int w = 0; w < waves; w++) sum += parts[w * R * T * 256 + o];
    const int i = o / (T * 256), j = o / 256 % T;
    const int m = 16 * j + o % 256 / 16, n = n0 + 16 * i + o % 16;
    if (m < c.m && n < c.n) put_at(c, m, n, sum);
  }
}

// The pieces' sums (whole numbers: in any order the same) to y.
__global__ void __launch_bounds__(256) join_kernel(Work wk) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x, mn = int64_t(wk.c.m) * wk.c.n;
  if (i >= mn) return;
  int sum = 0;
  for (int p = 0; p < wk.pieces; p++) sum += wk.part[p * mn + i];
  const int m = int(i / wk.c.n);
  put_at(wk.c, m, int(i - int64_t(m) * wk.c.n), sum);
}

// A sum of nothing.
__global__ void __launch_bounds__(256) nothing_kernel(GemmI8Call c) {
  const int64_t mn = int64_t(c.m) * c.n;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < mn; i += int64_t(gridDim.x) * 256) {
    const int m = int(i / c.n);
    put_at(c, m, int(i - int64_t(m) * c.n), 0);
  }
}

template <int R, int T>
int launch_few(const GemmI8Call &c, hipStream_t s) {
  // (as many waves as take the same whole turns)
  using F = Few<R, T>;
  const int steps = (c.k + 63) / 64, each = (steps + F::U * F::kWaves - 1) / (F::U * F::kWaves) * F::U;
  const int waves = (steps + each - 1) / each;
  few_kernel<R, T><<<unsigned((c.n + 16 * R - 1) / (16 * R)), 64 * waves, R * T * 1024 * waves, s>>>(c);
  return hipGetLastError() == hipSuccess ? SWAMP_OK : SWAMP_ELAUNCH;
}

template <typename Y, int WM, int WN, int NWM, int NWN>
int launch_typed(const Work &wk, hipStream_t s) {
  using S = Shape<WM, WN, NWM, NWN>;
  static std::once_flag once;
  static hipError_t err = hipSuccess;
  std::call_once(once, [] {
    err = hipFuncSetAttribute(reinterpret_cast<const void *>(&gemm_kernel<Y, WM, WN, NWM, NWN>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  });
  if (err != hipSuccess) return SWAMP_ELAUNCH;
  const unsigned units = unsigned(wk.tiles_m) * unsigned(wk.tiles_n) * unsigned(wk.pieces);
  gemm_kernel<Y, WM, WN, NWM, NWN><<<units, S::kThreads, S::kSmem, s>>>(wk);
  return hipGetLastError() == hipSuccess ? SWAMP_OK : SWAMP_ELAUNCH;
}
template <int WM, int WN, int NWM, int NWN>
int launch(const Work &wk, hipStream_t s) {
  if (wk.c.y_type == SWAMP_F32) return launch_typed<float, WM, WN, NWM, NWN>(wk, s);
  if (wk.c.y_type == SWAMP_F16) return launch_typed<_Float16, WM, WN, NWM, NWN>(wk, s);
  return launch_typed<__bf16, WM, WN, NWM, NWN>(wk, s);
}

}  // namespace

int swamp_launch_quantize_rows(const void *d_x, uint32_t x_type, int64_t x_stride, int8_t *d_q,
                               int64_t q_stride, float *d_scale, int n_rows, int n_cols,
                               hipStream_t s) {
  // (a launch holds less than 2^32 threads)
  constexpr int kRows = 1 << 21;
  auto go = [&](auto t) {
    typedef decltype(t) X;
    for (int64_t r0 = 0; r0 < n_rows; r0 += kRows) {
      const X *x = static_cast<const X *>(d_x) + r0 * x_stride;
      int8_t *q = d_q + r0 * q_stride;
      float *scale = d_scale + r0;
      const unsigned n = unsigned(std::min<int64_t>(n_rows - r0, kRows));
      auto rows = [&](auto each_c) {
        constexpr int each = decltype(each_c)::value;
        const int threads = std::max(1, (n_cols + 64 * each - 1) / (64 * each)) * 64;
        quantize_kernel<X, each><<<n, threads, 0, s>>>(x, x_stride, q, q_stride, scale, n_cols);
      };
      // (rows in few waves wait less for each other; from HBM: 4096 x 14336 bf16 41 us with 32
      // elements a thread and 45 with 16, 4096 x 4096 18.6 and 15.3, 16384 x 512 9.1 with 8 and
      // 10.8 with 16, 512 x 40000 f32 24 with 64 and 32 in two looks)
      if (n_cols <= 512) rows(std::integral_constant<int, 8>{});
      else if (n_cols <= 1024 * 8) rows(std::integral_constant<int, 16>{});
      else if (n_cols <= 1024 * 32) rows(std::integral_constant<int, 32>{});
      else if (n_cols <= 1024 * 64) rows(std::integral_constant<int, 64>{});
      else quantize_any_kernel<X><<<n, 1024, 0, s>>>(x, x_stride, q, q_stride, scale, n_cols);
    }
  };
  if (x_type == SWAMP_F32) go(float{});
  else if (x_type == SWAMP_F16) go(_Float16{});
  else go(__bf16{});
  return hipGetLastError() == hipSuccess ? SWAMP_OK : SWAMP_ELAUNCH;
}

size_t swamp_gemm_rows_i8_scratch_bytes(int m, int n_rows, int n_cols) {
  if (n_cols == 0) return 0;
  const Plan p = swamp_rows::plan_of(m, n_rows, n_cols, swamp::device_info().num_cus);
  return p.pieces > 1 ? swamp::scratch_round(size_t(p.pieces) * size_t(m) * size_t(n_rows) * 4) : 0;
}

int swamp_launch_gemm_rows_i8(const GemmI8Call &c, swamp::Scratch &sc, hipStream_t s) {
  const int64_t blocks = (int64_t(c.m) * c.n + 255) / 256;
  if (c.k == 0) {
    nothing_kernel<<<unsigned(std::min<int64_t>(blocks, 1 << 16)), 256, 0, s>>>(c);
    return hipGetLastError() == hipSuccess ? SWAMP_OK : SWAMP_ELAUNCH;
  }
  const Plan p = swamp_rows::plan_of(c.m, c.n, c.k, swamp::device_info().num_cus);
  if (p.shape < 0) {
    auto few = [&](auto r) {
      constexpr int R = decltype(r)::value;
      if (c.m <= 16) return launch_few<R, 1>(c, s);
      if (c.m <= 32) return launch_few<R, 2>(c, s);
      if constexpr (R <= 2) return launch_few<R, 4>(c, s);
      return int(SWAMP_EINVAL);  // (no plan)
    };
    return p.tiles_n == 1   ? few(std::integral_constant<int, 1>{})
           : p.tiles_n == 2 ? few(std::integral_constant<int, 2>{})
                            : few(std::integral_constant<int, 4>{});
  }
  Work wk{c, p.tiles_m, p.tiles_n, 8, p.pieces, p.steps, nullptr};
  if (p.pieces > 1) {
    wk.part = static_cast<int32_t *>(sc.get(size_t(p.pieces) * size_t(c.m) * size_t(c.n) * 4));
    if (!wk.part) {
      wk.pieces = 1;
      wk.steps = (c.k + 63) / 64;
    }
  }
  const int rc = p.shape == 0   ? launch<1, 2, 2, 2>(wk, s)
                 : p.shape == 1 ? launch<2, 1, 2, 4>(wk, s)
                 : p.shape == 2 ? launch<2, 2, 4, 2>(wk, s)
                 : p.shape == 3 ? launch<2, 2, 2, 4>(wk, s)
                                : launch<4, 2, 2, 4>(wk, s);
  if (rc != SWAMP_OK || wk.pieces == 1) return rc;
  join_kernel<<<unsigned(blocks), 256, 0, s>>>(wk);
  return hipGetLastError() == hipSuccess ? SWAMP_OK : SWAMP_ELAUNCH;
}
