// attn.hip -- swamp_attn_paged: how a call's keys are split over workgroups, and
// the join of the pieces.  The attention itself is in attn_core.hpp, built per
// cache type in attn_f16.hip and attn_bf16.hip.
#include "attn_core.hpp"

#include <algorithm>
#include <cmath>

int swamp_attn_f16(const swamp_attn::Work &w, bool precise, hipStream_t s);
int swamp_attn_bf16(const swamp_attn::Work &w, bool precise, hipStream_t s);

namespace {

// out = sum_x 2^(m_x - m) o_x / sum_x 2^(m_x - m) l_x over the pieces x of a row, in
// a fixed order.  `per` threads (dim / 4 rounded up to a power of two) times
// `shares` take a row: four dims and one run of the pieces each, kBatch pieces'
// loads at a time, and the runs meet in LDS.
//
// A kernel of its own.  Joined by the last workgroup of each row instead (a
// counter, and sums that bypass the L2 of an XCD, which others do not see), 64
// sequences of up to 8192 tokens in 4 pieces took 279 us against 231, one of
// 131072 in 32 pieces 117 against 100, and 700 tokens 12 as now.
template <int kBatch>
__global__ void __launch_bounds__(kThreads) join_kernel(Work w, int per, int shares) {
  __shared__ f32x4 accs[kThreads];
  __shared__ f32x2 stats[kThreads];
  const int tid = int(threadIdx.x), team = per * shares;
  const int64_t n = int64_t(w.b.n_tok) * w.n_heads;
  const int64_t row = int64_t(blockIdx.x) * (kThreads / team) + tid / team, t = row / w.n_heads;
  const int share = tid % team / per, d = 4 * (tid % per), dim = w.cache.dim;
  // (rows of no sequence are not touched)
  const bool mine = row < n && d < dim && t >= w.b.first[0] && t < w.b.first[w.b.n_seq];
  const int run = (w.splits + shares - 1) / shares;
  const int x1 = min((share + 1) * run, w.splits);
  float m = -INFINITY, l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  bool sees = true;
  for (int x0 = share * run; mine && x0 < x1; x0 += kBatch) {
    f32x2 st[kBatch];
    f32x4 o[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; i++) {
      const int64_t at = min(x0 + i, x1 - 1) * n + row;
      st[i] = w.stat[at];
      o[i] = *reinterpret_cast<const f32x4 *>(w.part + at * dim + d);
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < kBatch; i++) top = fmaxf(top, st[i][0]);
    const float base = top == -INFINITY ? 0.f : top, keep = __builtin_amdgcn_exp2f(m - base);
    m = top;
    acc *= keep;
    l *= keep;
#pragma unroll
    for (int i = 0; i < kBatch; i++) {
      if (x0 + i >= x1) break;
      const float k = __builtin_amdgcn_exp2f(st[i][0] - base);
      sees = sees && st[i][1] != -1.f;
      l += k * st[i][1];
      if (st[i][0] != -INFINITY) acc += k * o[i];  // (else nothing was written)
    }
  }
  if (shares > 1) {
    accs[tid] = acc;
    stats[tid] = f32x2{m, l};
    __syncthreads();
    if (share == 0) {
      float top = m;
      for (int i = 1; i < shares; i++) top = fmaxf(top, stats[tid + i * per][0]);
      const float base = top == -INFINITY ? 0.f : top, keep = __builtin_amdgcn_exp2f(m - base);
      acc *= keep;
      l *= keep;
      for (int i = 1; i < shares; i++) {
        const f32x2 st = stats[tid + i * per];
        const float k = __builtin_amdgcn_exp2f(st[0] - base);
        l += k * st[1];
        if (st[0] != -INFINITY) acc += k * accs[tid + i * per];
      }
    }
  }
  if (mine && share == 0)
    put4(w, t, int(row - t * w.n_heads), dim, d,
         sees ? acc * (1.f / l) : f32x4{0.f, 0.f, 0.f, 0.f});
}

struct Plan {
  int blocks, one_block, few, splits, chunk;
};

// Pieces of the keys that make attn_many_kernel shortest, by a model of its time
// on this card, us: a tile takes 0.55 + 0.007 dim where a CU has one workgroup
// and 0.6 more for each further one (heads of 128: 1.45 and 2.06 us measured), a
// workgroup's start and end three tiles, and a join 4 us and its sums' way
// through memory.  A last round that is not full costs its share, as most rows
// see less than the longest sequence, and a little more: without it 45
// workgroups of 256 dims go in 6 pieces instead of 5, 38.8 us and 30.8.  Down
// to one tile a piece pays (7 workgroups, 256 dims, 554 keys: pieces of four
// tiles 34.8 us, of one 23.7).
int many_splits(int64_t base, int64_t rows, int64_t keys, int dim, int cus) {
  const int most = dim <= 64 ? 3 : dim <= 128 ? 2 : 1;  // workgroups of a CU
  const double tiles = double(keys) / kTile;
  double best = 0;
  int want = 1;
  for (int n = 1; n <= 16 && n <= std::max<int64_t>(1, keys / kTile); n++) {
    const int64_t load = std::min<int64_t>(most, (base * n + cus - 1) / cus);
    const double rounds = std::max(1.0, double(base) * n / (double(cus) * most));
    double t = (0.95 * rounds + 0.05 * std::ceil(rounds)) * (tiles / n + 3) * (0.55 + 0.007 * dim + 0.6 * double(load - 1));
    if (n > 1) t += 4 + n * double(rows) * dim * 8 / 6e6;
    if (n == 1 || t < best) best = t, want = n;
  }
  return want;
}

// blocks: at most this many, of all sequences, whatever the rows' distribution.
Plan plan_of(const swamp::AttnCall &c) {
  const int group = c.n_heads / c.cache.n_kv, cus = swamp::device_info().num_cus;
  const int64_t rows = int64_t(c.batch.n_tok) * group;  // of a cache head
  const int64_t most = (int64_t(c.max_new) * group + kRows - 1) / kRows;  // blocks of a sequence
  Plan p;
  p.few = int64_t(c.max_new) * group <= kFew;
  p.one_block = most <= 1;
  p.blocks = int(p.one_block ? c.batch.n_seq
                             : std::min((rows + int64_t(kRows - 1) * c.batch.n_seq) / kRows,
                                        most * c.batch.n_seq));
  const int64_t base = std::max<int64_t>(1, int64_t(p.blocks) * c.cache.n_kv);
  const int64_t seen = int64_t(c.window) + (p.few ? c.max_new : kRows / group) + kTile;
  const int64_t keys = c.window ? std::min<int64_t>(c.max_len, seen) : c.max_len;
  int64_t want;
  if (p.few) {
    // one workgroup a CU, of short heads two while a piece keeps two steps (64
    // workgroups of 128 dims over 4001 keys: 256 in all 22.4 us, 512 25.2, 64 60;
    // 22 of 64 dims over up to 22634 keys: 528 in all 27.5, 242 41.5; 2 over 20345:
    // 160 in all 13.3, 318 14.8)
    want = cus / base;
    if (c.cache.dim <= 64) want = std::max(want, std::min(2 * cus / base, keys / (64 * kWaves)));
    // sequences of unequal length in a piece or two each: pieces of 2048 keys even
    // them out (256 workgroups over up to 6000 keys 39.9 us, whole 47.0; 115 over
    // up to 14540: 68.5, in two 78.9); where there are more pieces these are too
    // many (70 of 256 dims over up to 13260 keys: 124 us, in three 109)
    if (want < 3) want = std::max(want, keys / 2048);
    // none below the time of the join (8 workgroups, 128 dims, 512 keys: whole 9.6
    // us, in pieces 11.1; 1024 keys: 14.2 and 10.8; 64 dims, 1024 keys: 10.6 and 11)
    if (keys * c.cache.dim <= 65536) want = 1;
  } else {
    want = many_splits(base, rows * c.cache.n_kv, keys, c.cache.dim, cus);
  }
  // a piece is whole tiles; of a few rows one for each wave at least
  const int step = p.few ? 32 * kWaves : kTile;
  want = std::max<int64_t>(1, want);
  p.chunk = int(((keys + want - 1) / want + step - 1) / step * step);
  p.chunk = std::max(p.chunk, step);
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
  int per = 2, shares = 1;
  while (4 * per < c.cache.dim) per *= 2;
  while (shares * 2 * per <= kThreads && shares * 8 < w.splits) shares *= 2;
  const int64_t rows = int64_t(c.batch.n_tok) * c.n_heads, each = kThreads / (per * shares);
  const dim3 grid(unsigned((rows + each - 1) / each));
  if (w.splits <= 4) join_kernel<4><<<grid, kThreads, 0, s>>>(w, per, shares);
  else join_kernel<8><<<grid, kThreads, 0, s>>>(w, per, shares);
  return hipGetLastError() == hipSuccess ? SWAMP_OK : SWAMP_ELAUNCH;
}
