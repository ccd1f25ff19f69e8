// attn.hip -- swamp_attn_paged: its launches, and the join of a cache's pieces (their
// number: attn_plan.hpp).  The attention itself is in attn_core.hpp, built per cache
// type in attn_f16.hip and attn_bf16.hip.
#include "attn_core.hpp"

int swamp_attn_f16(const swamp_attn::Work &w, int parts, hipStream_t s);
int swamp_attn_bf16(const swamp_attn::Work &w, int parts, hipStream_t s);

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
      st[i] = w.stat[min(x0 + i, x1 - 1) * n + row];
    }
    // (a piece without keys of the row wrote no sums, and where max_len is far above
    // the lengths most are such)
#pragma unroll
    for (int i = 0; i < kBatch; i++) {
      o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (st[i][0] != -INFINITY)
        o[i] = *reinterpret_cast<const f32x4 *>(
            w.part + (min(x0 + i, x1 - 1) * n + row) * dim + d);
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
      acc += k * o[i];
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

}  // namespace

size_t swamp_attn_scratch_bytes(const swamp::AttnCall &c) {
  const swamp::AttnPlan p = swamp::plan_attn(c, swamp::device_info().num_cus);
  if (p.splits <= 1) return 0;
  return swamp::scratch_round(swamp::attn_part_bytes(c, p.splits)) +
         swamp::scratch_round(swamp::attn_stat_bytes(c, p.splits));
}

int swamp_launch_attn_paged(const swamp::AttnCall &c, swamp::Scratch &sc, hipStream_t s) {
  const swamp::AttnPlan p = swamp::plan_attn(c, swamp::device_info().num_cus);
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
    w.part = static_cast<float *>(sc.get(swamp::attn_part_bytes(c, p.splits)));
    w.stat = static_cast<f32x2 *>(sc.get(swamp::attn_stat_bytes(c, p.splits)));
    if (!w.part || !w.stat) w.splits = 1;
  }
  // Weights in as many parts of the cache's type as the output has bits for: 11 a part
  // in fp16, 8 in bf16.  With 16-bit output of the cache's own type, or less, one
  // rounding of theirs is as large as the output's.  (A further product for one of the
  // sums costs blocks of many rows about a third each: 4096 tokens of 32 heads of 128
  // dims, fp16 160 us and 218, bf16 151, 199 and 241; few rows 1 to 2% in full batches
  // and up to 15% in short calls, 16 drafts of 4 tokens over 2000 keys of 80 dims 17.9
  // us and 20.2.)
  const bool half_of_bf16 = c.dtype == SWAMP_BF16 && c.out_type == SWAMP_F16;
  const int parts = c.out_type == SWAMP_F32 ? 3 : half_of_bf16 ? 2 : 1;
  const int rc = c.dtype == SWAMP_F16 ? swamp_attn_f16(w, parts, s) : swamp_attn_bf16(w, parts, s);
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
