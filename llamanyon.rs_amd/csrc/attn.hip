// attn.hip -- causal attention of a batch's new tokens over the paged cache
// (swamp_attn_paged): o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q.k_j).
//
// One wave takes one row and one query head and walks the keys that the row
// sees, in order: four dims a lane, the score summed across the wave, the
// softmax's running maximum m and sum l beside the running output, which is
// scaled by exp(m_old - m_new) where m grows (one pass over K and V).
#include "paging.hpp"
#include "swamp_common.hpp"

namespace {

constexpr float kLog2e = 1.44269504088896341f;

template <typename CT, typename OT>
__global__ void __launch_bounds__(256)
    attn_rows_kernel(swamp::PagedCache cache, swamp::SeqBatch b, const CT *__restrict__ q,
                     int64_t q_stride, int n_heads, float scale, int window, OT *__restrict__ out,
                     int64_t out_stride) {
  const int lane = int(threadIdx.x & 63);
  const int s = int(blockIdx.y);
  const int64_t unit = int64_t(blockIdx.x) * 4 + int(threadIdx.x >> 6);
  const int row = int(unit / n_heads), head = int(unit % n_heads);
  const swamp::Seq sq = swamp::seq_of(b.first[s], b.first[s + 1], b.len[s], b.n_tok);
  if (row >= sq.n) return;
  const int64_t t = sq.t0 + row;
  const int pos = sq.len - sq.n + row;
  const swamp::Span keys = swamp::seen_by(pos, window);
  const int d0 = 4 * lane, kv_head = head / (n_heads / cache.n_kv);
  float qv[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 4; j++)
    qv[j] = d0 < cache.dim ? float(q[t * q_stride + head * cache.dim + d0 + j]) : 0.f;
  float m = -INFINITY, l = 0.f;
  bool bad = false;
  for (int p = keys.lo; p < keys.hi; p++) {
    const int64_t col = swamp::page_col(p, cache.page_shift);
    int32_t id = -1;
    if (swamp::page_col_ok(p, col, b.pages_stride)) id = b.pages[s * b.pages_stride + col];
    if (!swamp::page_ok(id, cache.n_pages)) {
      bad = true;
      break;
    }
    const int64_t at = swamp::slot_offset(id, p, kv_head, cache.page_shift, cache.page_stride,
                                          cache.head_stride, cache.slot_stride);
    float dot = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    if (d0 < cache.dim) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        dot += qv[j] * float(reinterpret_cast<const CT *>(cache.k)[at + d0 + j]);
        v[j] = float(reinterpret_cast<const CT *>(cache.v)[at + d0 + j]);
      }
    }
    const float x = swamp::wave_sum(dot) * scale * kLog2e;
    const float grown = fmaxf(m, x), base = grown == -INFINITY ? 0.f : grown;
    const float keep = __builtin_amdgcn_exp2f(m - base), w = __builtin_amdgcn_exp2f(x - base);
    m = grown;
    l = l * keep + w;
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = o[j] * keep + w * v[j];
  }
  if (bad && b.bad && lane == 0) *b.bad = 1;
  if (d0 < cache.dim) {
#pragma unroll
    for (int j = 0; j < 4; j++)
      out[t * out_stride + head * cache.dim + d0 + j] =
          OT(bad ? __builtin_nanf("") : keys.hi > keys.lo ? o[j] / l : 0.f);
  }
}

}  // namespace

size_t swamp_attn_scratch_bytes(const swamp::AttnCall &) { return 0; }

int swamp_launch_attn_paged(const swamp::AttnCall &c, swamp::Scratch &, hipStream_t s) {
  const dim3 grid(unsigned((int64_t(c.max_new) * c.n_heads + 3) / 4), unsigned(c.batch.n_seq));
  auto go = [&](auto ct, auto ot) {
    typedef decltype(ct) C;
    typedef decltype(ot) O;
    attn_rows_kernel<C, O><<<grid, 256, 0, s>>>(c.cache, c.batch, static_cast<const C *>(c.q),
                                                c.q_stride, c.n_heads, c.scale, c.window,
                                                static_cast<O *>(c.out), c.out_stride);
  };
  auto with_out = [&](auto ct) {
    if (c.out_type == SWAMP_F32) go(ct, float{});
    else if (c.out_type == SWAMP_F16) go(ct, _Float16{});
    else go(ct, __bf16{});
  };
  if (c.dtype == SWAMP_F16) with_out(_Float16{});
  else with_out(__bf16{});
  return hipGetLastError() == hipSuccess ? SWAMP_OK : SWAMP_ELAUNCH;
}
