// attn.hip -- swamp_attn_paged: how a call's keys are split over workgroups, and
// the join of the pieces.  The attention itself is in attn_core.hpp, built per
// cache type in attn_f16.hip and attn_bf16.hip.
#include "attn_core.hpp"

#include <algorithm>

int swamp_attn_f16(const swamp_attn::Work &w, bool precise, hipStream_t s);
int swamp_attn_bf16(const swamp_attn::Work &w, bool precise, hipStream_t s);

namespace {

constexpr int kJoinWide = 4;  // pieces up to which a thread joins them all

// out = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i over a row's pieces, in a
// fixed order.

// A thread takes four dims of a row and all pieces.
__global__ void __launch_bounds__(kThreads) join_kernel(Work w) {
  const int per = w.cache.dim >> 2;
  const int64_t n = int64_t(w.b.n_tok) * w.n_heads;  // rows of a piece
  const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t row = i / per;
  const int d = int(i - row * per) * 4;
  const int64_t t = row / w.n_heads;
  if (row >= n || t < w.b.first[0] || t >= w.b.first[w.b.n_seq]) return;  // padding
  float top = -INFINITY;
#pragma unroll 8
  for (int x = 0; x < w.splits; x++) top = fmaxf(top, w.stat[x * n + row][0]);
  const float base = top == -INFINITY ? 0.f : top;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
  bool sees = true;
#pragma unroll 4
  for (int x = 0; x < w.splits; x++) {
    const f32x2 st = w.stat[x * n + row];
    const float k = __builtin_amdgcn_exp2f(st[0] - base);
    sees = sees && st[1] != -1.f;
    sum += k * st[1];
    if (st[0] != -INFINITY)
      acc += k * *reinterpret_cast<const f32x4 *>(w.part + (x * n + row) * w.cache.dim + d);
  }
  put4(w, t, int(row - t * w.n_heads), w.cache.dim, d,
       sees ? acc * (1.f / sum) : f32x4{0.f, 0.f, 0.f, 0.f});
}

// A workgroup takes a row: `per` threads (dim / 4 rounded up to a power of two)
// for the dims, 256 / per shares of the pieces.  For few rows in many pieces,
// whose loads would otherwise wait for one another.
__global__ void __launch_bounds__(kThreads) join_wide_kernel(Work w, int per) {
  __shared__ f32x4 accs[kThreads];
  __shared__ float sums[kThreads], tops[kWaves];
  __shared__ int blind;
  const int64_t n = int64_t(w.b.n_tok) * w.n_heads, row = blockIdx.x, t = row / w.n_heads;
  if (t < w.b.first[0] || t >= w.b.first[w.b.n_seq]) return;  // padding
  const int tid = int(threadIdx.x), share = tid / per, shares = kThreads / per;
  const int d = 4 * (tid - share * per);
  float top = -INFINITY;
  for (int x = tid; x < w.splits; x += kThreads) top = fmaxf(top, w.stat[x * n + row][0]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  if ((tid & 63) == 0) tops[tid >> 6] = top;
  if (tid == 0) blind = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; i++) top = fmaxf(top, tops[i]);
  const float base = top == -INFINITY ? 0.f : top;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
#pragma unroll 4
  for (int x = share; x < w.splits; x += shares) {
    const f32x2 st = w.stat[x * n + row];
    const float k = __builtin_amdgcn_exp2f(st[0] - base);
    if (st[1] == -1.f) blind = 1;
    sum += k * st[1];
    if (st[0] != -INFINITY && d < w.cache.dim)
      acc += k * *reinterpret_cast<const f32x4 *>(w.part + (x * n + row) * w.cache.dim + d);
  }
  accs[tid] = acc;
  sums[tid] = sum;
  __syncthreads();
  if (share != 0 || d >= w.cache.dim) return;
  for (int i = 1; i < shares; i++) {
    acc += accs[i * per + tid];
    sum += sums[i * per + tid];
  }
  put4(w, t, int(row - t * w.n_heads), w.cache.dim, d,
       blind ? f32x4{0.f, 0.f, 0.f, 0.f} : acc * (1.f / sum));
}

struct Plan {
  int blocks, one_block, few, splits, chunk;
};

// blocks: at most this many, of all sequences, whatever the rows' distribution.
Plan plan_of(const swamp::AttnCall &c) {
  const int group = c.n_heads / c.cache.n_kv;
  const int64_t rows = int64_t(c.batch.n_tok) * group;
  const int64_t most = (int64_t(c.max_new) * group + kRows - 1) / kRows;  // of a sequence
  Plan p;
  p.one_block = most <= 1;
  p.blocks = int(p.one_block ? c.batch.n_seq
                             : std::min((rows + int64_t(kRows - 1) * c.batch.n_seq) / kRows,
                                        most * c.batch.n_seq));
  p.few = int64_t(c.max_new) * group <= kFew;
  const int slots = swamp::device_info().num_cus * (c.cache.dim <= 128 ? 2 : 1);
  const int64_t base = int64_t(p.blocks) * c.cache.n_kv;
  const int64_t keys =
      c.window ? std::min<int64_t>(c.max_len, int64_t(c.window) + c.max_new) : c.max_len;
  const int64_t least = p.few ? 2 * kTile : 4 * kTile;
  int64_t want = std::max<int64_t>(1, (p.few ? 2 : 1) * slots / std::max<int64_t>(base, 1));
  want = std::max<int64_t>(1, std::min<int64_t>(want, keys / least));
  p.chunk = int((((keys + want - 1) / want + 2 * kTile - 1) / (2 * kTile)) * 2 * kTile);
  p.chunk = std::max(p.chunk, 2 * kTile);
  p.splits = int(std::max<int64_t>(1, (keys + p.chunk - 1) / p.chunk));
  return p;
}

size_t part_bytes(const swamp::AttnCall &c, int splits) {
  return size_t(splits) * c.batch.n_tok * c.n_heads * c.cache.dim * 4;
}
size_t stat_bytes(const swamp::AttnCall &c, int splits) {
  return size_t(splits) * c.batch.n_tok * c.n_heads * 8;
}

}  // namespace

size_t swamp_attn_scratch_bytes(const swamp::AttnCall &c) {
  const Plan p = plan_of(c);
  if (p.splits <= 1) return 0;
  return swamp::scratch_round(part_bytes(c, p.splits)) +
         swamp::scratch_round(stat_bytes(c, p.splits));
}

int swamp_launch_attn_paged(const swamp::AttnCall &c, swamp::Scratch &sc, hipStream_t s) {
  const Plan p = plan_of(c);
  Work w;
  w.cache = c.cache;
  w.b = c.batch;
  w.q = static_cast<const uint16_t *>(c.q);
  w.q_stride = c.q_stride;
  w.out = c.out;
  w.out_stride = c.out_stride;
  w.out_type = c.out_type;
  w.n_heads = c.n_heads;
  w.group = c.n_heads / c.cache.n_kv;
  w.window = c.window;
  w.scale = c.scale;
  w.blocks = p.blocks;
  w.one_block = p.one_block;
  w.few = p.few;
  w.splits = p.splits;
  w.chunk = p.chunk;
  w.part = nullptr;
  w.stat = nullptr;
  if (p.splits > 1) {
    w.part = static_cast<float *>(sc.get(part_bytes(c, p.splits)));
    w.stat = static_cast<f32x2 *>(sc.get(stat_bytes(c, p.splits)));
    if (!w.part || !w.stat) w.splits = 1;
  }
  const bool precise = c.out_type == SWAMP_F32;
  const int rc = c.dtype == SWAMP_F16 ? swamp_attn_f16(w, precise, s) : swamp_attn_bf16(w, precise, s);
  if (rc != SWAMP_OK || w.splits == 1) return rc;
  const int64_t rows = int64_t(c.batch.n_tok) * c.n_heads;
  if (w.splits > kJoinWide) {
    int per = 2;
    while (4 * per < c.cache.dim) per *= 2;
    join_wide_kernel<<<dim3(unsigned(rows)), kThreads, 0, s>>>(w, per);
  } else {
    const int64_t n = rows * (c.cache.dim / 4);
    join_kernel<<<dim3(unsigned((n + kThreads - 1) / kThreads)), kThreads, 0, s>>>(w);
  }
  return hipGetLastError() == hipSuccess ? SWAMP_OK : SWAMP_ELAUNCH;
}
