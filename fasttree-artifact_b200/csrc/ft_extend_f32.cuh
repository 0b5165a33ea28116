// Extend attention for fp32 storage: exact fp32 arithmetic on the CUDA cores (no tensor core takes fp32 operands unrounded).
//
// 256 threads as 16 x 16 (ty, tx) over a query tile of R = 16 RPT rows and K/V tiles of 64 tokens:
//   S: a thread has RPT rows x 4 tokens (tx, tx + 16, ...), from float4 reads along head_dim: 4 (RPT + 4) floats read for
//      16 RPT products;
//   softmax: a row's 16 threads are half a warp, its maximum and sum stay in their registers;
//   P through shared memory; O: the same RPT rows x D / 16 columns per thread, kept in registers.
// Q, K, V and P tiles are swizzled by 16-byte chunks, so that neither product's reads meet in a bank.  V of a tile is loaded
// beside its scores, K of the next beside the product with V; the row ids one tile ahead.  Two CTAs per SM up to head_dim 128.
// Bound by shared-memory reads and FMAs in about equal parts: 512 tokens on 2048, 8/2 heads of 128, 180 us = 27 TFLOP/s (the
// CUDA cores' nominal rate is 72), heads of 256 the same; steps of few tokens by the chain of reads at the start.  64 rows where
// the step has them, 16 (a quarter of the work per tile, four times the tiles) where requests have few: the plan tries both.
// With 16 rows a score is summed in blocks of 32 products, which makes its error two to three times smaller (single tokens, heads of
// 256, scores capped at 50: outputs off by 9.1e-7, in blocks 3.3e-7) and takes no more time; with 64 rows the registers that it needs
// cost 7 %, and the error of one chain is that of a matrix product.
#pragma once

#include "ft_extend.cuh"
#include "ft_stage1_mma.cuh"

namespace ft {

template <int D_, int RPT_>
struct ExtF32Cfg {
  static constexpr int D = D_, RPT = RPT_, R = 16 * RPT, TILE = 64, THREADS = 256;
  static constexpr int CH = D / 4;  // 16-byte chunks of a row
  static constexpr int K_OFF = R * D * 4, V_OFF = K_OFF + TILE * D * 4, P_OFF = V_OFF + TILE * D * 4, IDS_OFF = P_OFF + R * TILE * 4,
                       SMEM_BYTES = IDS_OFF + 2 * TILE * 4;
  static constexpr int CTAS = SMEM_BYTES <= 115712 ? 2 : 1;
  static_assert(SMEM_BYTES <= 232448, "one CTA must fit in one SM's shared memory");
};

// byte position of 16-byte chunk c of row r in a tile of CH chunks a row
template <int CH>
__device__ __forceinline__ uint32_t ext_chunk(int r, int c) {
  constexpr int PER = CH >= 8 ? 1 : 8 / CH, MASK = CH >= 8 ? 7 : CH - 1;  // rows per 128 bytes
  return (uint32_t)(r * CH + (c ^ ((r / PER) & MASK))) * 16u;
}

template <int D, int RPT>
__global__ void __launch_bounds__(256, ExtF32Cfg<D, RPT>::CTAS) extend_f32_kernel(const ExtendParams p) {
  using C = ExtF32Cfg<D, RPT>;
  constexpr int CH = C::CH, TILE = C::TILE;
  constexpr int CPT = D >= 64 ? D / 64 : 1;  // float4 columns of O per thread (head_dim 16, 32: the first D / 4 threads of a row)
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sm = smem_u32(smem);
  int* ids = reinterpret_cast<int*>(smem + C::IDS_OFF);
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  allow_dependent_launch();
  wait_for_prior_grid();
  const int4 share = __ldg(reinterpret_cast<const int4*>(p.sms) + 4 * blockIdx.x);
  const float* qb = reinterpret_cast<const float*>(p.q);
  auto at4 = [&](uint32_t off) { return *reinterpret_cast<const float4*>(smem + off); };
  for (int n = share.x; n < share.y; ++n) {
    const int task = n == share.x ? share.z : __ldg(p.sm_tasks + n), kvh = task % p.kv_heads;
    const int32_t* item = p.items + (int64_t)EXT_ITEM_INTS * (task / p.kv_heads);
    const int tile0 = __ldg(item + 5);
    const ExtendStream st = extend_stream(item, 0);
    const int rows = st.ntok * p.group;
    const float* kb = reinterpret_cast<const float*>(p.k) + (int64_t)kvh * p.k_s1;
    const float* vb = reinterpret_cast<const float*>(p.v) + (int64_t)kvh * p.v_s1;
    auto fetch_id = [&](int t) {  // threads below TILE: the row id of a token of tile t; -1: none, -2: out of range
      int id = -1;
      if (t < st.hi) {
        const int4 rec = __ldg(reinterpret_cast<const int4*>(p.tiles) + 2 * ((int64_t)tile0 + t));
        if (tid < rec.z) {
          id = __ldg(p.kv_entries + extend_entry(p, rec, tid));
          if (id < 0 || id >= p.kv_rows) {
            flag_error(FT_DEV_BAD_KV_INDEX);
            id = -2;
          }
        }
      }
      return id;
    };
    auto load_rows = [&](int off, const float* base, int64_t stride, const int* of) {  // a K or V tile; rows without a token become zeros
      for (int i = tid; i < TILE * CH; i += 256) {
        const int r = i / CH, c = i % CH, id = of[r];
        cp_async16_zfill(sm + off + ext_chunk<CH>(r, c), base + (int64_t)(id < 0 ? 0 : id) * stride + c * 4, id >= 0);
      }
      cp_async_commit();
    };
    for (int row0 = 0; row0 < rows; row0 += C::R) {
      __syncthreads();  // the rows before are done with shared memory
      if (tid < TILE) ids[(st.lo & 1) * TILE + tid] = fetch_id(st.lo);
      for (int i = tid; i < C::R * CH; i += 256) {
        const int r = row0 + i / CH, c = i % CH;
        int q_row = -1;
        if (r < rows) q_row = __ldg(p.tokens + 2 * (st.tok0 + r / p.group));
        const bool ok = q_row >= 0 && q_row < p.q_rows;
        cp_async16_zfill(sm + ext_chunk<CH>(i / CH, c), qb + (int64_t)(ok ? q_row : 0) * p.q_s0 + (int64_t)(kvh * p.group + r % p.group) * p.q_s1 + c * 4, ok);
      }
      __syncthreads();
      load_rows(C::K_OFF, kb, p.k_s0, ids + (st.lo & 1) * TILE);
      float m[RPT], l[RPT], o[RPT][CPT][4];
      bool hidden[RPT];
      const int32_t* bits[RPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const int r = row0 + ty * RPT + i;
        m[i] = -INFINITY;
        l[i] = 0.f;
        hidden[i] = false;
        bits[i] = p.extra + (st.first + (r < rows ? r / p.group : 0)) * (TILE / 32);
#pragma unroll
        for (int c = 0; c < CPT; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][c][e] = 0.f;
      }
      for (int t = st.lo; t < st.hi; ++t) {
        cp_async_wait<0>();
        __syncthreads();  // K is there; V's and P's readers are done
        load_rows(C::V_OFF, vb, p.v_s0, ids + (t & 1) * TILE);
        const int next_id = tid < TILE ? fetch_id(t + 1) : -1;
        const int mask = __ldg(p.tiles + 8 * ((int64_t)tile0 + t) + 4 + st.block_tile);
        float s[RPT][4];
#pragma unroll
        for (int i = 0; i < RPT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
        auto products = [&](int c, float (&to)[RPT][4]) {
          float4 q[RPT], k[4];
#pragma unroll
          for (int i = 0; i < RPT; ++i) q[i] = at4(ext_chunk<CH>(ty * RPT + i, c));
#pragma unroll
          for (int j = 0; j < 4; ++j) k[j] = at4(C::K_OFF + ext_chunk<CH>(tx + 16 * j, c));
#pragma unroll
          for (int i = 0; i < RPT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              to[i][j] = fmaf(q[i].w, k[j].w, fmaf(q[i].z, k[j].z, fmaf(q[i].y, k[j].y, fmaf(q[i].x, k[j].x, to[i][j]))));
        };
        if constexpr (RPT == 1 && CH > 8) {
#pragma unroll 1
          for (int c0 = 0; c0 < CH; c0 += 8) {
            float part[RPT][4] = {};
#pragma unroll 4
            for (int c = c0; c < c0 + 8; ++c) products(c, part);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[0][j] += part[0][j];
          }
        } else {
#pragma unroll 4
          for (int c = 0; c < CH; ++c) products(c, s);
        }
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          float mx = -INFINITY;
          uint32_t in[2] = {0xffffffffu, 0xffffffffu};
          if (mask >= 0) {
            in[0] = extend_bits(bits[i] + mask);
            in[1] = extend_bits(bits[i] + mask + 1);
            hidden[i] |= (in[0] & in[1]) != 0xffffffffu;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[i][j] *= p.sm_scale;
            if (p.logit_cap > 0.f) s[i][j] = p.logit_cap * tanhf(s[i][j] / p.logit_cap);
            const bool seen = ((in[j >> 1] >> ((tx + 16 * j) & 31)) & 1u) != 0 && ids[(t & 1) * TILE + tx + 16 * j] >= 0;
            if (!seen) s[i][j] = -INFINITY;
            mx = fmaxf(mx, s[i][j]);
          }
#pragma unroll
          for (int d = 8; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const float m_new = fmaxf(m[i], mx);
          const float corr = m[i] == m_new ? 1.f : expf(m[i] - m_new);
          m[i] = m_new;
          const float base = m_new == -INFINITY ? 0.f : m_new;
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[i][j] = expf(s[i][j] - base);
            sum += s[i][j];
            *reinterpret_cast<float*>(smem + C::P_OFF + ext_chunk<16>(ty * RPT + i, (tx >> 2) + 4 * j) + (tx & 3) * 4) = s[i][j];
          }
#pragma unroll
          for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
          l[i] = l[i] * corr + sum;
#pragma unroll
          for (int c = 0; c < CPT; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][c][e] *= corr;
        }
        if (tid < TILE) ids[((t + 1) & 1) * TILE + tid] = next_id;
        cp_async_wait<0>();
        __syncthreads();  // V and P are there; K's readers are done
        if (t + 1 < st.hi) load_rows(C::K_OFF, kb, p.k_s0, ids + ((t + 1) & 1) * TILE);
        if (D >= 64 || tx < CH) {
#pragma unroll 2
          for (int k4 = 0; k4 < TILE / 4; ++k4) {
            float4 pr[RPT];
#pragma unroll
            for (int i = 0; i < RPT; ++i) pr[i] = at4(C::P_OFF + ext_chunk<16>(ty * RPT + i, k4));
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
              for (int c = 0; c < CPT; ++c) {
                const float4 v = at4(C::V_OFF + ext_chunk<CH>(4 * k4 + u, tx + 16 * c));
#pragma unroll
                for (int i = 0; i < RPT; ++i) {
                  const float w = u == 0 ? pr[i].x : u == 1 ? pr[i].y : u == 2 ? pr[i].z : pr[i].w;
                  o[i][c][0] = fmaf(w, v.x, o[i][c][0]);
                  o[i][c][1] = fmaf(w, v.y, o[i][c][1]);
                  o[i][c][2] = fmaf(w, v.z, o[i][c][2]);
                  o[i][c][3] = fmaf(w, v.w, o[i][c][3]);
                }
              }
          }
        }
      }
      cp_async_wait<0>();
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const int r = row0 + ty * RPT + i, tok = r < rows ? r / p.group : 0, head = kvh * p.group + r % p.group;
        const int q_row = __ldg(p.tokens + 2 * (st.tok0 + tok)), part = r < rows ? extend_part(p, st, tok) : -2;
        const bool store = part != -2 && q_row >= 0 && q_row < p.q_rows;
        if (part != -2 && !store) flag_error(FT_DEV_BAD_Q_INDEX);
        const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
        float zero = 0.f;  // 0 x every element: 0, or NaN
        if (D >= 64 || tx < CH) {
          float* dst = part >= 0 ? p.mid_o + ((int64_t)part * p.heads + head) * D
                                 : reinterpret_cast<float*>(p.o) + (int64_t)(store ? q_row : 0) * p.o_s0 + (int64_t)head * p.o_s1;
#pragma unroll
          for (int c = 0; c < CPT; ++c) {
            const float4 x = make_float4(o[i][c][0] * inv, o[i][c][1] * inv, o[i][c][2] * inv, o[i][c][3] * inv);
            zero += 0.f * x.x + 0.f * x.y + 0.f * x.z + 0.f * x.w;
            if (store) *reinterpret_cast<float4*>(dst + (tx + 16 * c) * 4) = x;
          }
        }
        if (store && tx == 0) extend_store_lse(p, part, q_row, head, l[i] == 0.f ? -INFINITY : logf(l[i]) + m[i]);
        // rows of V that this row does not see were multiplied by 0: if one of them was not finite, the row again, alone
        const uint32_t spoiled = __ballot_sync(0xffffffffu, store && hidden[i] && !(zero == 0.f));
#pragma unroll
        for (int half = 0; half < 2; ++half)
          if ((spoiled >> (16 * half) & 0xffffu) != 0) {
            const int rr = row0 + ((tid >> 5) * 2 + half) * RPT + i;
            __syncwarp();
            extend_row<float>(p, item, st, rr / p.group, kvh * p.group + rr % p.group);
          }
      }
    }
  }
}

}  // namespace ft
