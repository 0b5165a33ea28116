// A step's new tokens enter the paged cache: queries and keys are turned by their positions, keys and values go to the
// tokens' pool rows.
//
//   pair i of a head, (x1, x2) = elements (i, i + rot / 2), or (2 i, 2 i + 1) in the interleaved form:
//     (x1, x2)  ->  (x1 c - x2 s,  x2 c + x1 s),   c, s = table[pos][i], table[pos][rot / 2 + i]
//   with pos the token's position along the axis whose section i falls into; elements from rot on stay as they are.
//
// The table (fp32, [positions, rot]: cosines, then sines) is the caller's, so far positions are as exact as it is.  The
// turn is done in fp32 and rounded once.  Bound by memory: every element is read once and written once.
//
// One CTA per token.  The unit of work is two 16-byte vectors of one head - the two halves of VEC pairs, or 2 VEC
// adjacent elements - and a thread keeps its place in the head over the heads it takes, so its cosines and sines are
// read once per token and stay in registers.  A thread issues the loads of two heads before the first store.
#pragma once

#include "ft_common.cuh"

namespace ft {

struct AppendParams {
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  void* k_buffer;
  void* v_buffer;
  const void* slots;
  const void* positions;
  const float* cos_sin;
  int64_t q_s0, q_s1, k_s0, k_s1, v_s0, v_s1, qo_s0, qo_s1, kb_s0, kb_s1, vb_s0, vb_s1;
  int64_t kv_rows, positions_s0, cos_sin_rows, cos_sin_s0;
  int32_t tokens, q_heads, kv_heads, head_dim, rot;
  int32_t section_end[4];  // pair i belongs to the first axis whose end is above i
  int32_t axes;
  int32_t slots_64, positions_64, interleaved;
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) AppendVec {
  T x[VEC];
};

__device__ __forceinline__ int64_t append_index(const void* p, int64_t i, int is_64) {
  return is_64 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
}

template <typename T, int VEC>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  using Vec = AppendVec<T, VEC>;
  const int64_t t = blockIdx.x;
  const int units = p.head_dim / (2 * VEC);        // per head
  const int per_pass = (int)blockDim.x / units;    // heads at a time
  const int u = (int)threadIdx.x % units, h0 = (int)threadIdx.x / units;
  if (h0 >= per_pass) return;
  const int q_heads = p.q != nullptr ? p.q_heads : 0, heads = q_heads + 2 * p.kv_heads;

  // this unit's two vectors, and its pairs' cosines and sines
  const int half = p.rot / 2;
  const bool turned = p.interleaved ? 2 * VEC * u < p.rot : VEC * u < half;
  int at0, at1;
  if (turned && !p.interleaved) {
    at0 = VEC * u;
    at1 = half + VEC * u;
  } else {
    // adjacent: the interleaved form's pairs, or elements behind the turned ones (half / VEC units are the turned ones')
    at0 = p.interleaved ? 2 * VEC * u : p.rot + 2 * VEC * (u - half / VEC);
    at1 = at0 + VEC;
  }
  const int64_t slot = append_index(p.slots, t, p.slots_64);
  const bool keep = slot >= 0 && slot < p.kv_rows;
  if (!keep && slot != -1 && threadIdx.x == 0) flag_error(FT_DEV_BAD_KV_INDEX);
  bool bad = false;
  for (int axis = 0; axis < p.axes; ++axis) {
    const int64_t pos = append_index(p.positions, (int64_t)axis * p.positions_s0 + t, p.positions_64);
    bad |= pos < 0 || pos >= p.cos_sin_rows;
  }
  if (bad) {  // a position outside the table: nothing of the token is written
    if (threadIdx.x == 0) flag_error(FT_DEV_BAD_POSITION);
    return;
  }
  float c[VEC], s[VEC];
  if (turned) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int pair = VEC * u + i;  // in both forms
      int axis = 0;
      while (axis + 1 < p.axes && pair >= p.section_end[axis]) ++axis;
      const float* row = p.cos_sin + append_index(p.positions, (int64_t)axis * p.positions_s0 + t, p.positions_64) * p.cos_sin_s0;
      c[i] = row[pair];
      s[i] = row[half + pair];
    }
  }
  constexpr int HEADS = 2;  // in flight per thread
  for (int h = h0; h < heads; h += HEADS * per_pass) {
    Vec a[HEADS], b[HEADS];
#pragma unroll
    for (int n = 0; n < HEADS; ++n) {
      const int hh = h + n * per_pass;
      if (hh >= heads) break;
      const T* src = hh < q_heads              ? reinterpret_cast<const T*>(p.q) + t * p.q_s0 + (int64_t)hh * p.q_s1
                     : hh < q_heads + p.kv_heads ? reinterpret_cast<const T*>(p.k) + t * p.k_s0 + (int64_t)(hh - q_heads) * p.k_s1
                                               : reinterpret_cast<const T*>(p.v) + t * p.v_s0 + (int64_t)(hh - q_heads - p.kv_heads) * p.v_s1;
      // (values are not turned; which two vectors of the head a unit takes does not matter for them)
      a[n] = *reinterpret_cast<const Vec*>(src + at0);
      b[n] = *reinterpret_cast<const Vec*>(src + at1);
    }
#pragma unroll
    for (int n = 0; n < HEADS; ++n) {
      const int hh = h + n * per_pass;
      if (hh >= heads) break;
      const bool is_q = hh < q_heads, is_k = !is_q && hh < q_heads + p.kv_heads;
      if (turned && (is_q || is_k)) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          T* x1;
          T* x2;
          if (p.interleaved) {
            const int e = 2 * i;
            x1 = e < VEC ? &a[n].x[e % VEC] : &b[n].x[e % VEC];
            x2 = e + 1 < VEC ? &a[n].x[(e + 1) % VEC] : &b[n].x[(e + 1) % VEC];
          } else {
            x1 = &a[n].x[i];
            x2 = &b[n].x[i];
          }
          const float y1 = to_float<T>(*x1), y2 = to_float<T>(*x2);
          *x1 = from_float<T>(y1 * c[i] - y2 * s[i]);
          *x2 = from_float<T>(y2 * c[i] + y1 * s[i]);
        }
      }
      if (!is_q && !keep) continue;  // a padding token, or a slot outside the pool
      T* dst = is_q   ? reinterpret_cast<T*>(p.q_out) + t * p.qo_s0 + (int64_t)hh * p.qo_s1
               : is_k ? reinterpret_cast<T*>(p.k_buffer) + slot * p.kb_s0 + (int64_t)(hh - q_heads) * p.kb_s1
                      : reinterpret_cast<T*>(p.v_buffer) + slot * p.vb_s0 + (int64_t)(hh - q_heads - p.kv_heads) * p.vb_s1;
      *reinterpret_cast<Vec*>(dst + at0) = a[n];
      *reinterpret_cast<Vec*>(dst + at1) = b[n];
    }
  }
}

}  // namespace ft
