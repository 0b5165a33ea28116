// Extend attention: causal attention of several new tokens per request over the paged cache, driven by the tables of
// ft_extend_plan.cu (items, segments, tokens; their layouts stand there).
//
//   o[t] = sum_j p_j v_j / sum_j p_j,   p_j = exp(cap(scale q[t] . k_j) - m),   j in sight of t
//
// This file: the tables' readers, one query row by one warp in scalar fp32 arithmetic (the generic kernel is made of it; the
// tensor-core kernel falls back to it for single rows), and the merge of an item's partial rows.
#pragma once

#include "ft_common.cuh"

namespace ft {

constexpr int EXT_ITEM_INTS = 24, EXT_SEG_INTS = 8;

struct ExtendParams {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  float* o_lse;
  const int32_t* kv_entries;
  const int32_t* items;
  const int32_t* segs;
  const int32_t* tokens;
  const int32_t* sm_offs;
  const int32_t* sm_tasks;
  const int32_t* merged;      // {row of q, first entry of its list, entries, 0}
  const int32_t* merge_rows;
  float* mid_o;
  float* mid_lse;
  int64_t q_s0, q_s1, k_s0, k_s1, v_s0, v_s1, o_s0, o_s1;
  int64_t kv_rows, q_rows, kv_entries_len;
  int32_t num_items, num_merged, partial_rows;
  int32_t heads, kv_heads, group, head_dim, window, tile;
  float sm_scale;
  float logit_cap;  // <= 0: none
};

// One stream of an item: its query tokens, its K/V tiles and where its rows go.
struct ExtendStream {
  int tok0, ntok, lo, hi, part, q_tile, first;  // first: the stream's first token within the block
};

__device__ __forceinline__ ExtendStream extend_stream(const int32_t* item, int w) {
  const int4 a = __ldg(reinterpret_cast<const int4*>(item + 8 + 8 * w));
  const int4 b = __ldg(reinterpret_cast<const int4*>(item + 12 + 8 * w));
  return {a.x, a.y, a.z, a.w, b.x, b.y, b.z};
}

struct ExtendSegment {
  int64_t kv_off;
  int len, pos0, tok_lo, tok_hi, voff;
};

__device__ __forceinline__ ExtendSegment extend_segment(const int32_t* segs, int s) {
  const int4 a = __ldg(reinterpret_cast<const int4*>(segs + (int64_t)EXT_SEG_INTS * s));
  const int4 b = __ldg(reinterpret_cast<const int4*>(segs + (int64_t)EXT_SEG_INTS * s + 4));
  return {(int64_t)(((uint64_t)(uint32_t)a.y << 32) | (uint32_t)a.x), a.z, a.w, b.x, b.y, b.z};
}

// The virtual positions [lo, hi) of segment g that the query at position `pos`, token `tok` of its block, sees.
__device__ __forceinline__ void extend_in_sight(const ExtendSegment& g, int tok, int pos, int window, int& lo, int& hi) {
  const bool mine = tok >= g.tok_lo && tok < g.tok_hi;
  hi = mine ? g.voff + min(g.len, pos + 1 - g.pos0) : g.voff;
  lo = g.voff + (window > 0 ? max(pos - window + 1 - g.pos0, 0) : 0);
}

// Where a stream's row goes: a row of o, or a partial row.
template <typename T>
__device__ __forceinline__ void extend_store(const ExtendParams& p, int part, int tok, int q_row, int head, int d, float x) {
  if (part >= 0)
    p.mid_o[((int64_t)(part + tok) * p.heads + head) * p.head_dim + d] = x;
  else
    reinterpret_cast<T*>(p.o)[(int64_t)q_row * p.o_s0 + (int64_t)head * p.o_s1 + d] = from_float<T>(x);
}
__device__ __forceinline__ void extend_store_lse(const ExtendParams& p, int part, int tok, int q_row, int head, float lse) {
  if (part >= 0)
    p.mid_lse[(int64_t)(part + tok) * p.heads + head] = lse;
  else if (p.o_lse != nullptr)
    p.o_lse[(int64_t)q_row * p.heads + head] = lse;
}

// Query row (token `tok` of the stream, query head `head`) over the stream's K/V tiles lo, lo + step, ..., by one warp: lanes
// span the head dimension, four tokens in flight, online softmax with warp-shuffle sums.
template <typename T>
__device__ __noinline__ void extend_row(const ExtendParams& p, const int32_t* item, const ExtendStream st, const int tok, const int head) {
  constexpr int MAXJ = 8, TB = 4;  // 8 x 32 lanes = head_dim up to 256
  const int lane = threadIdx.x & 31, D = p.head_dim, kvh = head / p.group;
  const int seg0 = item[0], nseg = item[1], step = item[4];
  const int q_row = p.tokens[2 * (st.tok0 + tok)], pos = p.tokens[2 * (st.tok0 + tok) + 1];
  if (q_row < 0 || q_row >= p.q_rows) {
    if (lane == 0) flag_error(FT_DEV_BAD_Q_INDEX);
    return;
  }
  const T* __restrict__ qp = reinterpret_cast<const T*>(p.q) + (int64_t)q_row * p.q_s0 + (int64_t)head * p.q_s1;
  const T* __restrict__ kbase = reinterpret_cast<const T*>(p.k) + (int64_t)kvh * p.k_s1;
  const T* __restrict__ vbase = reinterpret_cast<const T*>(p.v) + (int64_t)kvh * p.v_s1;
  float qreg[MAXJ], acc[MAXJ];
#pragma unroll
  for (int j = 0; j < MAXJ; ++j) {
    const int d = lane + 32 * j;
    qreg[j] = d < D ? to_float<T>(qp[d]) : 0.f;
    acc[j] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int sg = seg0; sg < seg0 + nseg; ++sg) {
    const ExtendSegment g = extend_segment(p.segs, sg);
    int lo, hi;
    extend_in_sight(g, st.first + tok, pos, p.window, lo, hi);
    lo = max(lo, st.lo * p.tile);
    hi = min(hi, st.hi * p.tile);
    const int32_t* __restrict__ ids = p.kv_entries + g.kv_off - g.voff;
    int t0 = lo;
    while (t0 < hi) {
      const int tile = t0 / p.tile;
      if (step == 2 && ((tile - st.lo) & 1) != 0) {  // a tile of the other stream
        t0 = (tile + 1) * p.tile;
        continue;
      }
      const int end = min(hi, (tile + 1) * p.tile), n = min(TB, end - t0);
      int64_t row[TB];
      float s[TB];
      bool bad = false;
#pragma unroll
      for (int u = 0; u < TB; ++u) {
        row[u] = -1;
        if (u < n) {
          const int64_t id = ids[t0 + u];
          if (id >= 0 && id < p.kv_rows) row[u] = id;
          else bad = true;
        }
      }
      if (bad && lane == 0) flag_error(FT_DEV_BAD_KV_INDEX);
#pragma unroll
      for (int u = 0; u < TB; ++u) {
        float part = 0.f;
        if (row[u] >= 0) {
          const T* __restrict__ kp = kbase + row[u] * p.k_s0;
#pragma unroll
          for (int j = 0; j < MAXJ; ++j) {
            const int d = lane + 32 * j;
            if (d < D) part = fmaf(qreg[j], to_float<T>(kp[d]), part);
          }
        }
        s[u] = part;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
        for (int u = 0; u < TB; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], o);
      }
      float m_new = m;
#pragma unroll
      for (int u = 0; u < TB; ++u) {
        s[u] *= p.sm_scale;
        if (p.logit_cap > 0.f) s[u] = p.logit_cap * tanhf(s[u] / p.logit_cap);
        if (row[u] < 0) s[u] = -INFINITY;
        m_new = fmaxf(m_new, s[u]);
      }
      t0 += n;
      if (m_new == -INFINITY) {  // nothing in sight yet, unless a score is NaN
        bool nan = false;
#pragma unroll
        for (int u = 0; u < TB; ++u) nan |= s[u] != s[u];
        if (!nan) continue;
      }
      const float corr = m == m_new ? 1.f : expf(m - m_new);
      l *= corr;
#pragma unroll
      for (int j = 0; j < MAXJ; ++j) acc[j] *= corr;
#pragma unroll
      for (int u = 0; u < TB; ++u) {
        if (row[u] < 0) continue;
        const float pr = expf(s[u] - m_new);
        l += pr;
        // the tensor-core kernels round the probabilities to the storage type; here nothing asks for it
        const T* __restrict__ vp = vbase + row[u] * p.v_s0;
#pragma unroll
        for (int j = 0; j < MAXJ; ++j) {
          const int d = lane + 32 * j;
          if (d < D) acc[j] = fmaf(pr, to_float<T>(vp[d]), acc[j]);
        }
      }
      m = m_new;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int j = 0; j < MAXJ; ++j) {
    const int d = lane + 32 * j;
    if (d < D) extend_store<T>(p, st.part, tok, q_row, head, d, acc[j] * inv);
  }
  if (lane == 0) extend_store_lse(p, st.part, tok, q_row, head, l == 0.f ? -INFINITY : logf(l) + m);
}

// Any type and head size: a CTA per (item, KV head), a warp per query row in turn.
template <typename T>
__global__ void __launch_bounds__(128) extend_generic_kernel(const ExtendParams p) {
  const int item_id = (int)(blockIdx.x / (unsigned)p.kv_heads), kvh = (int)(blockIdx.x - (unsigned)item_id * p.kv_heads);
  const int32_t* item = p.items + (int64_t)EXT_ITEM_INTS * item_id;
  for (int w = 0; w < 2; ++w) {
    const ExtendStream st = extend_stream(item, w);
    for (int r = threadIdx.x >> 5; r < st.ntok * p.group; r += blockDim.x >> 5)
      extend_row<T>(p, item, st, r / p.group, kvh * p.group + r % p.group);
  }
}

// Merge of partial rows: a warp per (merged token, query head), lanes over the head dimension.  Rows of LSE -inf (nothing in
// sight) do not count.  Two passes over the LSEs, which the first brings into L1, then the rows, four in flight.
template <typename T>
__global__ void __launch_bounds__(128) extend_merge_kernel(const ExtendParams p) {
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (w >= (int64_t)p.num_merged * p.heads) return;
  const int lane = threadIdx.x & 31, D = p.head_dim;
  const int mt = (int)(w / p.heads), head = (int)(w - (int64_t)mt * p.heads);
  const int4 rec = __ldg(reinterpret_cast<const int4*>(p.merged) + mt);
  if (rec.x < 0 || rec.x >= p.q_rows) {
    if (lane == 0) flag_error(FT_DEV_BAD_Q_INDEX);
    return;
  }
  wait_for_prior_grid();
  const int32_t* __restrict__ list = p.merge_rows + rec.y;
  const int n = rec.z;
  float mx = -INFINITY;
  bool nan = false;
  for (int i = lane; i < n; i += 32) {
    const float x = p.mid_lse[(int64_t)list[i] * p.heads + head];
    mx = fmaxf(mx, x);
    nan |= x != x;
  }
  mx = warp_max(mx);
  if (__any_sync(0xffffffffu, nan)) mx = __int_as_float(0x7fc00000);
  constexpr int MAXJ = 8;
  float acc[MAXJ];
#pragma unroll
  for (int j = 0; j < MAXJ; ++j) acc[j] = 0.f;
  float sum = 0.f;
  for (int i0 = 0; i0 < n; i0 += 4) {
    float wt[4], x[4][MAXJ];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool ok = i0 + u < n;
      const int64_t row = ((int64_t)(ok ? list[i0 + u] : list[0]) * p.heads + head);
      const float lse = p.mid_lse[row];
      wt[u] = !ok || lse == -INFINITY ? 0.f : expf(lse - mx);
#pragma unroll
      for (int j = 0; j < MAXJ; ++j) {
        const int d = lane + 32 * j;
        x[u][j] = d < D && wt[u] != 0.f ? p.mid_o[row * D + d] : 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      sum += wt[u];
#pragma unroll
      for (int j = 0; j < MAXJ; ++j) acc[j] = fmaf(wt[u], x[u][j], acc[j]);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int j = 0; j < MAXJ; ++j) {
    const int d = lane + 32 * j;
    if (d < D) extend_store<T>(p, -1, 0, rec.x, head, d, acc[j] * inv);
  }
  if (lane == 0) extend_store_lse(p, -1, 0, rec.x, head, sum == 0.f ? -INFINITY : logf(sum) + mx);
}

}  // namespace ft
