// rows_i8.hip -- 8-bit codes with one scale a row (swamp_quantize_rows) and their
// products (swamp_gemm_rows_i8): y[i][r] = sx_i sw_r sum_k x[i][k] w[r][k].
//
// The scales stand outside the sum, so the sum is the matrix cores' own int32 (exact:
// 131071 terms of at most 2^14 stay below 2^31) and one product an output is left for
// the vector unit, where scales a block of 32 cost a conversion and an FMA for every 32
// terms (gemm_i8.hip).
//
// Tiles.  Four waves a workgroup, WM x WN V_MFMA_I32_32X32X32_I8 blocks each.  A K step
// is 64 codes: a stage holds the tile's rows of x, then of w, 64 bytes each, 16-byte
// chunks XOR-swizzled by (row / 4) % 4, so that 16 consecutive lanes of a fragment read
// meet no bank twice.  Five stages, filled by direct-to-LDS DMA three steps ahead; one
// barrier a step, between its halves, whose counted wait leaves the last step and a half
// of DMAs in flight.
//
// The last step of a sum is taken apart from the loop: its codes of x behind column K
// are cleared, so that what lies in w there (a row's padding) counts for nothing.
#include "swamp_common.hpp"
#include "swamp_items.hpp"

#include <algorithm>
#include <mutex>
#include <type_traits>

namespace {

using swamp::GemmI8Call;

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));

// ---- quantizer ------------------------------------------------------------
// A workgroup a row.  HBM's: a row is read once (the second look is the cache's).
template <typename XT>
__global__ void __launch_bounds__(256) quantize_kernel(const XT *__restrict__ x, int64_t x_stride,
                                                       int8_t *__restrict__ q, int64_t q_stride,
                                                       float *__restrict__ scale, int n) {
  __shared__ float tops[4];
  const XT *row = x + int64_t(blockIdx.x) * x_stride;
  int8_t *out = q + int64_t(blockIdx.x) * q_stride;
  const int tid = int(threadIdx.x);
  float top = 0.f;
  for (int k = tid; k < n; k += 256) {
    const float a = fabsf(float(row[k]));
    top = !(a <= 3.402823466e38f) ? INFINITY : fmaxf(top, a);  // NaN counts as infinity
  }
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) top = fmaxf(top, __shfl_xor(top, d, 64));
  if ((tid & 63) == 0) tops[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const bool fine = top < INFINITY;
  float s = top / 127.f;
  if (s < 1.17549435e-38f) s = 0.f;
  if (tid == 0) scale[blockIdx.x] = fine ? s : __builtin_nanf("");
  for (int k = tid; k < n; k += 256)
    out[k] = fine && s > 0.f ? int8_t(__builtin_rintf(float(row[k]) / s)) : int8_t(0);
}

// ---- products -------------------------------------------------------------
template <int WM, int WN, int NWM, int NWN>
struct Shape {
  static constexpr int NW = NWM * NWN, kThreads = 64 * NW;
  static constexpr int TM = 32 * WM * NWM, TN = 32 * WN * NWN;  // tile: rows of x, of w
  static constexpr int kStage = (TM + TN) * 64;
  static constexpr int kStages = 5;
  static constexpr int kSmem = kStages * kStage;
  static constexpr int kDma = (TM + TN) / (16 * NW);  // 1 KB DMAs of a wave and step
  static constexpr int kDma0 = (kDma + 1) / 2;        // of them in a step's first half
  static_assert(TM % (16 * NW) == 0 && TN % (16 * NW) == 0, "a DMA fills 16 rows of one operand");
  static_assert(kSmem <= 160 * 1024, "LDS");
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
template <bool kAdd, typename Y>
__device__ __forceinline__ void put(Y *y, int sum, float sx, double sw) {
  float v = float(double(sx) * sw * double(sum));
#ifdef __HIP_DEVICE_COMPILE__
  asm volatile("" : "+v"(v));  // (or the compiler rounds to 16 bits from 64 at once)
#endif
  *y = Y(kAdd ? float(*y) + v : v);
}
// f with y's element type and whether to add.
template <typename F>
__device__ __forceinline__ void with_output(const GemmI8Call &c, F f) {
  if (c.y_type == SWAMP_F32) {
    if (c.accumulate) f(float{}, std::true_type{});
    else f(float{}, std::false_type{});
  } else if (c.y_type == SWAMP_F16) {
    if (c.accumulate) f(_Float16{}, std::true_type{});
    else f(_Float16{}, std::false_type{});
  } else {
    if (c.accumulate) f(__bf16{}, std::true_type{});
    else f(__bf16{}, std::false_type{});
  }
}
__device__ __forceinline__ void put_at(const GemmI8Call &c, int64_t i, int sum) {
  const int m = int(i / c.n), n = int(i - int64_t(m) * c.n);
  with_output(c, [&](auto yt, auto add) {
    put<decltype(add)::value>(static_cast<decltype(yt) *>(c.y) + int64_t(m) * c.y_stride + n, sum,
                              c.x_scale[m], double(c.w_scale[n]));
  });
}

template <int WM, int WN, int NWM, int NWN>
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

  const uint32_t xp = uint32_t(c.x_stride), wp = uint32_t(c.w_stride), k16 = uint32_t(K + 15) & ~15u;
  const uint32_t xm = uint32_t(min(S::TM, c.m - m0) - 1), wn_ = uint32_t(min(S::TN, c.n - n0) - 1);
  const __amdgpu_buffer_rsrc_t xr = swamp::make_rsrc(c.x + m0 * c.x_stride, xm * xp + k16);
  const __amdgpu_buffer_rsrc_t wr = swamp::make_rsrc(c.w + n0 * c.w_stride, wn_ * wp + k16);
  // DMA i of wave w fills stage rows R = 16 (NW i + w) .. R + 15: lane L writes row
  // R + L / 4, physical chunk L % 4, which holds logical chunk (L % 4) ^ (L / 16 % 4).
  const uint32_t lrow4 = uint32_t(lane >> 2), chunk = uint32_t((lane & 3) ^ ((lane >> 4) & 3)) << 4;
  const uint32_t xv = lrow4 * xp + chunk, wv = lrow4 * wp + chunk;

  auto dma_part = [&](uint8_t *st, int kt, auto i0c, auto i1c) {
    constexpr int i0 = decltype(i0c)::value, i1 = decltype(i1c)::value;
#pragma unroll
    for (int i = i0; i < i1; i++) {
      const int R = 16 * (S::NW * i + wave);
      if (16 * S::NW * i < S::TM)
        dma16(xr, st + R * 64, xv, uint32_t(R) * xp + uint32_t(kt) * 64u);
      else
        dma16(wr, st + R * 64, wv, uint32_t(R - S::TM) * wp + uint32_t(kt) * 64u);
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

  constexpr int NS = S::kStages;
  // Step kt issues the DMA of step kt + 3, half in each half, into the stage of step
  // kt - 2, which every wave finished reading before the previous barrier.  Past the
  // end: the last step again.
#pragma unroll
  for (int p = 0; p < 3; p++) {
    dma_part(smem + S::kStage * p, min(kt0 + p, kt1 - 1), I0{}, IE{});
    __builtin_amdgcn_sched_barrier(0);
  }
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * S::kDma) : "memory");

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
  using D0 = std::integral_constant<int, S::kDma0>;
  using D1 = std::integral_constant<int, S::kDma - S::kDma0>;

  int cur = 0;
  for (int kt = kt0; kt < kt1 - 1; kt++) {
    const int nxt = cur + 1 == NS ? 0 : cur + 1;
    const int fill = cur + 3 < NS ? cur + 3 : cur + 3 - NS;
    const int ktf = min(kt + 3, kt1 - 1);
    read_frags(smem + S::kStage * cur, loff1, fa1, fb1);
    mfmas(fa0, fb0);
    dma_part(smem + S::kStage * fill, ktf, I0{}, IH{});
    order(D0{});
    __builtin_amdgcn_sched_barrier(0);
    // step kt + 1 is there for every wave: only step kt + 2's DMA and the first half of
    // step kt + 3's stay in flight
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(S::kDma + S::kDma0) : "memory");
    read_frags(smem + S::kStage * nxt, loff0, fa0, fb0);
    mfmas(fa1, fb1);
    dma_part(smem + S::kStage * fill, ktf, IH{}, IE{});
    order(D1{});
    __builtin_amdgcn_sched_barrier(0);
    cur = nxt;
  }
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
  // The scales of the tile's rows, in the stages' place once every wave is done with them.
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  float *scales = reinterpret_cast<float *>(smem);
  for (int i = tid; i < S::TM; i += S::kThreads) scales[i] = c.x_scale[min(m0 + i, c.m - 1)];
  __syncthreads();
  auto store = [&](auto yt, auto acc_c) {
    typedef decltype(yt) Y;
    constexpr bool kAdd = decltype(acc_c)::value;
#pragma unroll
    for (int j = 0; j < WN; j++) {
      const int n = nw + 32 * j;
      const double sw_n = double(c.w_scale[min(n, c.n - 1)]);
#pragma unroll
      for (int i = 0; i < WM; i++) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const int row = wm * WM * 32 + 4 * fc + 32 * i + 8 * (e >> 2) + (e & 3), m = m0 + row;
          if (m < c.m && n < c.n) put<kAdd>(static_cast<Y *>(c.y) + int64_t(m) * c.y_stride + n,
                                            acc[i][j][e], scales[row], sw_n);
        }
      }
    }
  };
  with_output(c, store);
}

// The pieces' sums (whole numbers: in any order the same) to y.
__global__ void __launch_bounds__(256) join_kernel(Work wk) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x, mn = int64_t(wk.c.m) * wk.c.n;
  if (i >= mn) return;
  int sum = 0;
  for (int p = 0; p < wk.pieces; p++) sum += wk.part[p * mn + i];
  put_at(wk.c, i, sum);
}

// A sum of nothing.
__global__ void __launch_bounds__(256) nothing_kernel(GemmI8Call c) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i < int64_t(c.m) * c.n) put_at(c, i, 0);
}

struct Plan {
  int shape;  // 0: 64 x 256, 1: 128 x 128, 2: 256 x 256
  int tiles_m, tiles_n, pieces, steps;
};

Plan plan_of(int m, int n, int k) {
  const int cus = swamp::device_info().num_cus, KT = (k + 63) / 64;
  Plan p;
  auto tiles = [&](int tm, int tn) {
    p.tiles_m = (m + tm - 1) / tm;
    p.tiles_n = (n + tn - 1) / tn;
    return int64_t(p.tiles_m) * p.tiles_n;
  };
  p.shape = 2;
  if (m <= 64) p.shape = 0;
  else if (2 * tiles(256, 256) <= cus) p.shape = 1;
  const int64_t t = p.shape == 0 ? tiles(64, 256) : p.shape == 1 ? tiles(128, 128) : tiles(256, 256);
  p.pieces = int(std::max<int64_t>(1, std::min<int64_t>({cus / t, 8, KT / 8})));
  p.steps = (KT + p.pieces - 1) / p.pieces;
  p.pieces = (KT + p.steps - 1) / p.steps;
  return p;
}

template <int WM, int WN, int NWM, int NWN>
int launch(const Work &wk, hipStream_t s) {
  using S = Shape<WM, WN, NWM, NWN>;
  static std::once_flag once;
  static hipError_t err = hipSuccess;
  std::call_once(once, [] {
    err = hipFuncSetAttribute(reinterpret_cast<const void *>(&gemm_kernel<WM, WN, NWM, NWN>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  });
  if (err != hipSuccess) return SWAMP_ELAUNCH;
  const unsigned units = unsigned(wk.tiles_m) * unsigned(wk.tiles_n) * unsigned(wk.pieces);
  gemm_kernel<WM, WN, NWM, NWN><<<units, S::kThreads, S::kSmem, s>>>(wk);
  return hipGetLastError() == hipSuccess ? SWAMP_OK : SWAMP_ELAUNCH;
}

}  // namespace

int swamp_launch_quantize_rows(const void *d_x, uint32_t x_type, int64_t x_stride, int8_t *d_q,
                               int64_t q_stride, float *d_scale, int n_rows, int n_cols,
                               hipStream_t s) {
  auto go = [&](auto t) {
    typedef decltype(t) X;
    quantize_kernel<X><<<unsigned(n_rows), 256, 0, s>>>(static_cast<const X *>(d_x), x_stride, d_q,
                                                        q_stride, d_scale, n_cols);
  };
  if (x_type == SWAMP_F32) go(float{});
  else if (x_type == SWAMP_F16) go(_Float16{});
  else go(__bf16{});
  return hipGetLastError() == hipSuccess ? SWAMP_OK : SWAMP_ELAUNCH;
}

size_t swamp_gemm_rows_i8_scratch_bytes(int m, int n_rows, int n_cols) {
  if (n_cols == 0) return 0;
  const Plan p = plan_of(m, n_rows, n_cols);
  return p.pieces > 1 ? size_t(p.pieces) * size_t(m) * size_t(n_rows) * 4 : 0;
}

int swamp_launch_gemm_rows_i8(const GemmI8Call &c, swamp::Scratch &sc, hipStream_t s) {
  const int64_t blocks = (int64_t(c.m) * c.n + 255) / 256;
  if (c.k == 0) {
    nothing_kernel<<<unsigned(blocks), 256, 0, s>>>(c);
    return hipGetLastError() == hipSuccess ? SWAMP_OK : SWAMP_ELAUNCH;
  }
  Plan p = plan_of(c.m, c.n, c.k);
  Work wk{c, p.tiles_m, p.tiles_n, 8, p.pieces, p.steps, nullptr};
  if (p.pieces > 1) {
    wk.part = static_cast<int32_t *>(sc.get(size_t(p.pieces) * size_t(c.m) * size_t(c.n) * 4));
    if (!wk.part) {
      wk.pieces = 1;
      wk.steps = (c.k + 63) / 64;
    }
  }
  const int rc = p.shape == 0   ? launch<2, 2, 1, 4>(wk, s)
                 : p.shape == 1 ? launch<2, 2, 2, 2>(wk, s)
                                : launch<4, 4, 2, 2>(wk, s);
  if (rc != SWAMP_OK || wk.pieces == 1) return rc;
  join_kernel<<<unsigned(blocks), 256, 0, s>>>(wk);
  return hipGetLastError() == hipSuccess ? SWAMP_OK : SWAMP_ELAUNCH;
}
