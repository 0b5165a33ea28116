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
// One CTA per token.  The unit of work is two 16-byte vectors of one head - the two halves of VEC pairs, or 2 VEC adjacent
// elements - and a thread keeps its place in the head over the heads it takes.  The token's cosines and sines come through
// shared memory, once for all heads; they are two loads deep (position, table row), so the first heads' elements are sent for
// before them.  128 threads of 64 registers, three heads in flight each: 8192 tokens at 32/8 heads of 128, bf16 (206 MB) 45 us =
// 4.6 TB/s, what a plain copy of as many bytes takes on the same GPU (43 us); 256 threads with two heads in flight 57 us, 384
// threads with one 65 us; one decode step's 64 tokens 8 us, a launch.
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
  int32_t slots_64, positions_64;
};

// VEC elements as 32-bit words (as an array of 16-bit elements they take a register each), or one element
template <typename T, int VEC>
struct alignas(16) AppendVec {
  uint32_t w[4];
};
template <typename T>
struct AppendVec<T, 1> {
  T w[1];
};

template <typename T>
__device__ __forceinline__ float2 append_unpack(uint32_t w);
template <>
__device__ __forceinline__ float2 append_unpack<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 append_unpack<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t append_pack(float a, float b);
template <>
__device__ __forceinline__ uint32_t append_pack<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t append_pack<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The turn of a unit's VEC pairs: those of a with those of b, or (PAIRS) the adjacent elements of a, then of b.
template <typename T, int VEC, bool PAIRS>
__device__ __forceinline__ void append_turn(AppendVec<T, VEC>& a, AppendVec<T, VEC>& b, const float (&c)[VEC], const float (&s)[VEC]) {
  if constexpr (VEC == 1) {
    const float x = to_float<T>(a.w[0]), y = to_float<T>(b.w[0]);
    a.w[0] = from_float<T>(x * c[0] - y * s[0]);
    b.w[0] = from_float<T>(y * c[0] + x * s[0]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t& p = PAIRS ? (i < 2 ? a.w[2 * i & 3] : b.w[2 * i & 3]) : a.w[i];
      uint32_t& q = PAIRS ? (i < 2 ? a.w[(2 * i + 1) & 3] : b.w[(2 * i + 1) & 3]) : b.w[i];
      const float x = __uint_as_float(p), y = __uint_as_float(q);
      p = __float_as_uint(x * c[i] - y * s[i]);
      q = __float_as_uint(y * c[i] + x * s[i]);
    }
  } else if constexpr (PAIRS) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t& w = i < 4 ? a.w[i & 3] : b.w[i & 3];
      const float2 x = append_unpack<T>(w);
      w = append_pack<T>(x.x * c[i] - x.y * s[i], x.y * c[i] + x.x * s[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = append_unpack<T>(a.w[i]), y = append_unpack<T>(b.w[i]);
      a.w[i] = append_pack<T>(x.x * c[2 * i] - y.x * s[2 * i], x.y * c[2 * i + 1] - y.y * s[2 * i + 1]);
      b.w[i] = append_pack<T>(y.x * c[2 * i] + x.x * s[2 * i], y.y * c[2 * i + 1] + x.y * s[2 * i + 1]);
    }
  }
}

__device__ __forceinline__ int64_t append_index(const void* p, int64_t i, int is_64) {
  return is_64 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
}

// PAIRS: adjacent elements are turned together (the interleaved form)
template <typename T, int VEC, bool PAIRS>
__global__ void __launch_bounds__(128, 8) append_kernel(const AppendParams p) {
  using Vec = AppendVec<T, VEC>;
  const int64_t t = blockIdx.x;
  const int units = p.head_dim / (2 * VEC);        // per head
  const int per_pass = (int)blockDim.x / units;    // heads at a time
  const int u = (int)threadIdx.x % units, h0 = (int)threadIdx.x / units;
  const bool works = h0 < per_pass;  // (a thread beyond the last whole head helps with the table)
  const int q_heads = p.q != nullptr ? p.q_heads : 0, heads = q_heads + 2 * p.kv_heads;

  // this unit's two vectors, and its pairs' cosines and sines
  const int half = p.rot / 2;
  const bool turned = PAIRS ? 2 * VEC * u < p.rot : VEC * u < half;
  int at0, at1;
  if (turned && !PAIRS) {
    at0 = VEC * u;
    at1 = half + VEC * u;
  } else {
    // adjacent: the interleaved form's pairs, or elements behind the turned ones (half / VEC units are the turned ones')
    at0 = PAIRS ? 2 * VEC * u : p.rot + 2 * VEC * (u - half / VEC);
    at1 = at0 + VEC;
  }
  constexpr int HEADS = 3;  // in flight per thread
  Vec a[HEADS], b[HEADS];
  auto fetch = [&](int h) {
#pragma unroll
    for (int n = 0; n < HEADS; ++n) {
      const int hh = h + n * per_pass;
      if (hh >= heads || !works) break;
      const T* src = hh < q_heads              ? reinterpret_cast<const T*>(p.q) + t * p.q_s0 + (int64_t)hh * p.q_s1
                     : hh < q_heads + p.kv_heads ? reinterpret_cast<const T*>(p.k) + t * p.k_s0 + (int64_t)(hh - q_heads) * p.k_s1
                                               : reinterpret_cast<const T*>(p.v) + t * p.v_s0 + (int64_t)(hh - q_heads - p.kv_heads) * p.v_s1;
      // (values are not turned; which two vectors of the head a unit takes does not matter for them)
      a[n] = *reinterpret_cast<const Vec*>(src + at0);
      b[n] = *reinterpret_cast<const Vec*>(src + at1);
    }
  };
  fetch(h0);
  const int64_t slot = append_index(p.slots, t, p.slots_64);
  const bool keep = slot >= 0 && slot < p.kv_rows;
  if (!keep && slot != -1 && threadIdx.x == 0) flag_error(FT_DEV_BAD_KV_INDEX);
  __shared__ __align__(16) float sh_cos[128], sh_sin[128];
  float c[VEC], s[VEC];
  if (p.axes > 0) {
    bool bad = false;
    for (int pair = threadIdx.x; pair < half; pair += blockDim.x) {
      int axis = 0;
      while (axis + 1 < p.axes && pair >= p.section_end[axis]) ++axis;
      const int64_t pos = append_index(p.positions, (int64_t)axis * p.positions_s0 + t, p.positions_64);
      if (pos >= 0 && pos < p.cos_sin_rows) {
        const float* row = p.cos_sin + pos * p.cos_sin_s0;
        sh_cos[pair] = row[pair];
        sh_sin[pair] = row[half + pair];
      } else {
        bad = true;
      }
    }
    if (__syncthreads_or(bad)) {  // a position outside the table: nothing of the token is written
      if (threadIdx.x == 0) flag_error(FT_DEV_BAD_POSITION);
      return;
    }
    if (turned) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {  // (pairs VEC u + i in both forms)
        c[i] = sh_cos[VEC * u + i];
        s[i] = sh_sin[VEC * u + i];
      }
    }
  }
  if (!works) return;
  for (int h = h0; h < heads; h += HEADS * per_pass) {
    if (h != h0) fetch(h);
#pragma unroll
    for (int n = 0; n < HEADS; ++n) {
      const int hh = h + n * per_pass;
      if (hh >= heads) break;
      const bool is_q = hh < q_heads, is_k = !is_q && hh < q_heads + p.kv_heads;
      if (turned && (is_q || is_k)) append_turn<T, VEC, PAIRS>(a[n], b[n], c, s);
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
