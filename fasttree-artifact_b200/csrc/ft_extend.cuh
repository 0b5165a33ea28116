// Extend attention: causal attention of several new tokens per request over the paged cache, driven by the tables of
// ft_extend_plan.cu (items, tiles, tokens; their layouts stand there).
//
//   o[t] = sum_j p_j v_j / sum_j p_j,   p_j = exp(cap(scale q[t] . k_j) - m),   j in sight of t
//
// This file: the tables' readers, one query row by one warp in scalar fp32 arithmetic (the generic kernel is made of it; the
// tensor-core kernel falls back to it for single rows), and the merge of an item's partial rows.
#pragma once

#include "ft_common.cuh"

namespace ft {

constexpr int EXT_ITEM_INTS = 32;

struct ExtendParams {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  float* o_lse;
  const int32_t* kv_entries;
  const int32_t* items;
  const int32_t* tokens;
  const int32_t* tiles;
  const int32_t* extra;
  const int32_t* sms;
  const int32_t* sm_tasks;
  const int32_t* merged;      // {row of q, first entry of its list, entries, 0}
  const int32_t* merge_rows;
  float* mid_o;
  float* mid_lse;
  int64_t q_s0, q_s1, k_s0, k_s1, v_s0, v_s1, o_s0, o_s1;
  int64_t kv_rows, q_rows, kv_entries_len;
  int32_t num_items, num_merged, partial_rows;
  int32_t heads, kv_heads, group, head_dim, tile;
  float sm_scale;
  float logit_cap;  // <= 0: none
};

// One stream of an item: its query tokens, its K/V tiles and where its rows go; first, block_tile: the stream's first token and its
// query tile within the block.
struct ExtendStream {
  int tok0, ntok, lo, hi, part, q_tile, first, block_tile;
};

__device__ __forceinline__ ExtendStream extend_stream(const int32_t* item, int w) {
  const int4 a = __ldg(reinterpret_cast<const int4*>(item + 8 + 8 * w));
  const int4 b = __ldg(reinterpret_cast<const int4*>(item + 12 + 8 * w));
  return {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}

// Where the rows of token `tok` of a stream go: to o (-1), to a partial row, or nowhere (-2: the token sees nothing there).
__device__ __forceinline__ int extend_part(const ExtendParams& p, const ExtendStream& st, int tok) {
  return st.part < 0 ? -1 : __ldg(p.extra + st.part + tok);
}

template <typename T>
__device__ __forceinline__ void extend_store(const ExtendParams& p, int part, int q_row, int head, int d, float x) {
  if (part >= 0)
    p.mid_o[((int64_t)part * p.heads + head) * p.head_dim + d] = x;
  else
    reinterpret_cast<T*>(p.o)[(int64_t)q_row * p.o_s0 + (int64_t)head * p.o_s1 + d] = from_float<T>(x);
}
__device__ __forceinline__ void extend_store_lse(const ExtendParams& p, int part, int q_row, int head, float lse) {
  if (part >= 0)
    p.mid_lse[(int64_t)part * p.heads + head] = lse;
  else if (p.o_lse != nullptr)
    p.o_lse[(int64_t)q_row * p.heads + head] = lse;
}

// entry of kv_entries of token i of the tile with record `rec` (its first four ints)
__device__ __forceinline__ int64_t extend_entry(const ExtendParams& p, const int4 rec, int i) {
  if (rec.w < 0) return (int64_t)(((uint64_t)(uint32_t)rec.y << 32) | (uint32_t)rec.x) + i;
  const int2 e = __ldg(reinterpret_cast<const int2*>(p.extra + rec.w) + i);
  return (int64_t)(((uint64_t)(uint32_t)e.y << 32) | (uint32_t)e.x);
}

// Query row (token `tok` of the stream, query head `head`) over the stream's K/V tiles lo, lo + step, ..., by one warp: lanes
// span the head dimension, four tokens in flight, online softmax with warp-shuffle sums.  steps: a counter in shared memory that
// goes up with every tile, for those who wait for this warp (0: none does).
template <typename T>
__device__ __noinline__ void extend_row(const ExtendParams& p, const int32_t* item, const ExtendStream st, const int tok, const int head,
                                        const uint32_t steps = 0) {
  constexpr int MAXJ = 8, TB = 4;  // 8 x 32 lanes = head_dim up to 256
  const int lane = threadIdx.x & 31, D = p.head_dim, kvh = head / p.group;
  const int step = item[2], tile0 = item[5], words = p.tile / 32;
  const int q_row = p.tokens[2 * (st.tok0 + tok)];
  if (q_row < 0 || q_row >= p.q_rows) {
    if (lane == 0) flag_error(FT_DEV_BAD_Q_INDEX);
    return;
  }
  const int part = extend_part(p, st, tok);
  if (part == -2) return;
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
  for (int t = st.lo; t < st.hi; t += step) {
    const int32_t* tile = p.tiles + 8 * ((int64_t)tile0 + t);
    const int4 rec = __ldg(reinterpret_cast<const int4*>(tile));
    const int bits_at = __ldg(tile + 4 + st.block_tile);
    if (steps != 0 && lane == 0) asm volatile("red.shared.add.u32 [%0], 1;\n" ::"r"(steps) : "memory");
    for (int k = 0; k < words; ++k) {
      uint32_t todo = bits_at < 0 ? 0xffffffffu : (uint32_t)__ldg(p.extra + bits_at + (st.first + tok) * words + k);
      while (todo != 0) {
        int64_t row[TB];
        float s[TB];
        bool bad = false;
#pragma unroll
        for (int u = 0; u < TB; ++u) {
          row[u] = -1;
          if (todo != 0) {
            const int64_t id = p.kv_entries[extend_entry(p, rec, 32 * k + __ffs(todo) - 1)];
            todo &= todo - 1;
            if (id >= 0 && id < p.kv_rows) row[u] = id;
            else bad = true;
          }
        }
        if (bad && lane == 0) flag_error(FT_DEV_BAD_KV_INDEX);
#pragma unroll
        for (int u = 0; u < TB; ++u) {
          float dot = 0.f;
          if (row[u] >= 0) {
            const T* __restrict__ kp = kbase + row[u] * p.k_s0;
#pragma unroll
            for (int j = 0; j < MAXJ; ++j) {
              const int d = lane + 32 * j;
              if (d < D) dot = fmaf(qreg[j], to_float<T>(kp[d]), dot);
            }
          }
          s[u] = dot;
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
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int j = 0; j < MAXJ; ++j) {
    const int d = lane + 32 * j;
    if (d < D) extend_store<T>(p, part, q_row, head, d, acc[j] * inv);
  }
  if (lane == 0) extend_store_lse(p, part, q_row, head, l == 0.f ? -INFINITY : logf(l) + m);
}

// How many row ids outside the pool a stream shows to a token: each lane for its own, by a whole warp.  steps as above.
__device__ __noinline__ int extend_bad_in_sight(const ExtendParams& p, const int32_t* item, const ExtendStream st, const int tok, const uint32_t steps) {
  const int lane = threadIdx.x & 31, step = item[2], tile0 = item[5], words = p.tile / 32;
  int n = 0;
  for (int t = st.lo; t < st.hi; t += step) {
    const int32_t* tile = p.tiles + 8 * ((int64_t)tile0 + t);
    const int4 rec = __ldg(reinterpret_cast<const int4*>(tile));
    const int bits_at = __ldg(tile + 4 + st.block_tile);
    if (lane == 0) asm volatile("red.shared.add.u32 [%0], 1;\n" ::"r"(steps) : "memory");
#pragma unroll 4
    for (int k = 0; k < words; ++k) {
      const int i = 32 * k + lane, id = i < rec.z ? __ldg(p.kv_entries + extend_entry(p, rec, i)) : 0;
      const uint32_t out = __ballot_sync(0xffffffffu, i < rec.z && (id < 0 || id >= p.kv_rows));
      if (out != 0) n += __popc(out & (bits_at < 0 ? 0xffffffffu : (uint32_t)__ldg(p.extra + bits_at + (st.first + tok) * words + k)));
    }
  }
  return n;
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

// Merge of partial rows: WARPS warps per (merged token, query head) share its list of rows, VEC floats of a row per lane, so that
// LANES lanes span a row and 32 / LANES rows go by at a time.  A row's LSE and the row itself are read together; a running
// maximum scales what a warp has, and the warps' results are merged through shared memory.  Rows of LSE -inf (nothing in sight)
// do not count.  Bound by the chain of round trips to L2: one warp where the lists are short, four where they are long (per
// call with one / four: one token on 30 000, 36 rows for each of 32 heads, 48 / 44 us; 443 tokens of two rows 188 / 202).
template <typename T, int D, int WARPS>
__global__ void __launch_bounds__(128) extend_merge_kernel(const ExtendParams p) {
  constexpr int VEC = D >= 128 ? 4 : D / 32 > 0 ? D / 32 : 1;  // floats per lane and piece
  constexpr int PIECES = D > 128 ? D / 128 : 1;
  constexpr int LANES = D >= 32 ? 32 : D, ROWS = 32 / LANES;   // lanes over a row, rows at a time
  constexpr int RB = D > 128 ? 2 : 4;                          // batches of rows in flight
  constexpr int GROUPS = 4 / WARPS;                            // (token, head) pairs per CTA
  __shared__ float sh_acc[WARPS > 1 ? WARPS * D : 1], sh_m[WARPS], sh_l[WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % WARPS;
  const int64_t pair = (int64_t)blockIdx.x * GROUPS + warp / WARPS;
  if (pair >= (int64_t)p.num_merged * p.heads) return;
  const int mt = (int)(pair / p.heads), head = (int)(pair - (int64_t)mt * p.heads);
  const int4 rec = __ldg(reinterpret_cast<const int4*>(p.merged) + mt);
  const int32_t* __restrict__ list = p.merge_rows + rec.y;
  const int n = rec.z, rsub = lane / LANES, at = (lane % LANES) * VEC;
  float m = -INFINITY, l = 0.f, acc[PIECES][VEC];
#pragma unroll
  for (int c = 0; c < PIECES; ++c)
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[c][e] = 0.f;
  constexpr int STRIDE = WARPS * ROWS;
  int ids[RB];
#pragma unroll
  for (int u = 0; u < RB; ++u) {
    const int i = sub * ROWS + rsub + u * STRIDE;
    ids[u] = i < n ? __ldg(list + i) : -1;
  }
  wait_for_prior_grid();
  for (int i0 = sub * ROWS + rsub; i0 - rsub < n; i0 += RB * STRIDE) {
    float lse[RB], x[RB][PIECES][VEC];
#pragma unroll
    for (int u = 0; u < RB; ++u) {
      const int64_t row = (int64_t)(ids[u] < 0 ? 0 : ids[u]) * p.heads + head;
      lse[u] = ids[u] < 0 ? -INFINITY : __ldcg(p.mid_lse + row);
#pragma unroll
      for (int c = 0; c < PIECES; ++c) {
        const float* src = p.mid_o + row * D + c * 128 + at;
        if constexpr (VEC == 4) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(src));
          x[u][c][0] = v.x, x[u][c][1] = v.y, x[u][c][2] = v.z, x[u][c][3] = v.w;
        } else if constexpr (VEC == 2) {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(src));
          x[u][c][0] = v.x, x[u][c][1] = v.y;
        } else {
          x[u][c][0] = __ldcg(src);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < RB; ++u) {  // the next rows' numbers travel meanwhile
      const int i = i0 + (RB + u) * STRIDE;
      ids[u] = i < n ? __ldg(list + i) : -1;
    }
    float mx = m;
#pragma unroll
    for (int u = 0; u < RB; ++u) mx = fmaxf(mx, lse[u]);
    const float corr = m == mx ? 1.f : expf(m - mx);
    m = mx;
    l *= corr;
#pragma unroll
    for (int c = 0; c < PIECES; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[c][e] *= corr;
#pragma unroll
    for (int u = 0; u < RB; ++u) {
      const float wt = lse[u] == -INFINITY ? 0.f : expf(lse[u] - mx);
      if (wt == 0.f) continue;  // (a row without weight may hold anything)
      l += wt;
#pragma unroll
      for (int c = 0; c < PIECES; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[c][e] = fmaf(wt, x[u][c][e], acc[c][e]);
    }
  }
  // a warp's row groups (head_dim 16), then its neighbours
  if constexpr (ROWS > 1) {
#pragma unroll
    for (int o = LANES; o < 32; o <<= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o), a2 = __shfl_xor_sync(0xffffffffu, acc[0][0], o);
      const float mx = fmaxf(m, m2), f1 = m == -INFINITY ? 0.f : expf(m - mx), f2 = m2 == -INFINITY ? 0.f : expf(m2 - mx);
      acc[0][0] = (f1 == 0.f ? 0.f : f1 * acc[0][0]) + (f2 == 0.f ? 0.f : f2 * a2);
      l = f1 * l + f2 * l2;
      m = mx;
    }
  }
  if constexpr (WARPS > 1) {
#pragma unroll
    for (int c = 0; c < PIECES; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (rsub == 0) sh_acc[sub * D + c * 128 + at + e] = acc[c][e];
    if (lane == 0) {
      sh_m[sub] = m;
      sh_l[sub] = l;
    }
    __syncthreads();
    if (sub != 0) return;
    float mx = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) {
      mx = fmaxf(mx, sh_m[k]);
      nan |= sh_l[k] != sh_l[k];
    }
    l = nan ? __int_as_float(0x7fc00000) : 0.f;
#pragma unroll
    for (int c = 0; c < PIECES; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[c][e] = 0.f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) {
      const float f = sh_m[k] == -INFINITY ? 0.f : expf(sh_m[k] - mx);
      if (f == 0.f) continue;
      l += f * sh_l[k];
#pragma unroll
      for (int c = 0; c < PIECES; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[c][e] = fmaf(f, sh_acc[k * D + c * 128 + at + e], acc[c][e]);
    }
    m = mx;
  }
  if (rec.x < 0 || rec.x >= p.q_rows) {
    if (lane == 0) flag_error(FT_DEV_BAD_Q_INDEX);
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (rsub == 0) {
#pragma unroll
    for (int c = 0; c < PIECES; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) extend_store<T>(p, -1, rec.x, head, c * 128 + at + e, acc[c][e] * inv);
  }
  if (lane == 0) extend_store_lse(p, -1, rec.x, head, l == 0.f ? -INFINITY : logf(l) + m);
}

}  // namespace ft
