// Beam search: the best continuations of a request's beams, and the table rows that follow them.
//
//   score(b, x) = scores[b] + logits[b][x] - log sum_y exp(logits[b][y])
//
// Within a beam the order of scores is that of the logits, so a beam's share of the results is among its `best` largest
// logits.  beam_scan_kernel reads every logit once: a CTA goes through a slice of a row and leaves its sum of exponentials and its
// `best` largest logits; beam_merge_kernel puts a request's slices together.  Scores are made and compared in 64 bits, because those of
// different beams may lie close: what decides is the logits' own value.
#pragma once

#include <type_traits>

#include "ft_async.cuh"
#include "ft_draft.cuh"

namespace ft {

constexpr int BEAM_THREADS = 256, BEAM_WARPS = BEAM_THREADS / 32;
constexpr int BEAM_KEYS = 1024;  // candidates that a CTA lists; beyond that, which takes many equal logits, it picks one at a time

struct BeamParams {
  const void* logits;
  const float* scores;
  float* out_scores;
  void* out_beams;
  void* out_tokens;
  unsigned long long* keys;  // [rows][slices][best] {ordered logit, ~token}, 0: none
  float2* sums;              // [rows][slices] {c, sum of 2^(logit log2(e) - c)}
  int64_t logits_s0, logits_s1, scores_s0, scores_s1, out_scores_s0, out_beams_s0, out_tokens_s0;
  int32_t batch, beams, vocab, best, slices, slice_len, beams_64, tokens_64;  // slice_len: a multiple of 16 bytes
};

// A lower bound of the n-th largest of a block's values that n of them reach, from each thread's largest: the least of the
// largest of `groups` groups of threads, groups >= n a power of two up to BEAM_THREADS.  `largest`: of all.  A whole block; between
// calls with the same shared memory there has to be a barrier.
__device__ __forceinline__ float group_bound(float mine, int groups, float (&low)[BEAM_WARPS], float (&high)[BEAM_WARPS], float& largest) {
  const int lanes = BEAM_THREADS / groups;  // of a group, if that is less than a warp
  float top = mine, bound = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float other = __shfl_xor_sync(0xffffffffu, bound, o);
    bound = o < lanes ? fmaxf(bound, other) : fminf(bound, other);
  }
  if ((threadIdx.x & 31) == 0) {
    low[threadIdx.x >> 5] = bound;
    high[threadIdx.x >> 5] = top;
  }
  __syncthreads();
  bound = low[0], largest = high[0];
#pragma unroll
  for (int w = 1; w < BEAM_WARPS; ++w) {
    bound = fminf(bound, low[w]);
    largest = fmaxf(largest, high[w]);
  }
  return bound;
}

__device__ __forceinline__ unsigned long long warp_max_key(unsigned long long k) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
  return k;
}

// log2(e) as the kernels multiply by it: what a sum's offset is divided by to give a logarithm, in 64 bits.
constexpr float BEAM_LOG2E = 1.4426950408889634f;

// The best of a list of n keys into out[0 .. best), 0 where the list ends: ranked by counting, or one at a time, whichever
// takes fewer instructions.  A whole block, behind a barrier.
__device__ __forceinline__ void best_of_list(const unsigned long long* keys, int n, unsigned long long* __restrict__ out, int best,
                                             unsigned long long (&from_warp)[BEAM_WARPS]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (n <= 128 + 16 * best) {
    for (int i = threadIdx.x; i < n; i += BEAM_THREADS) {
      const unsigned long long key = keys[i];
      int rank = 0;
#pragma unroll 4
      for (int k = 0; k < n; ++k) rank += keys[k] > key;
      if (rank < best) out[rank] = key;
    }
    for (int i = n + (int)threadIdx.x; i < best; i += BEAM_THREADS) out[i] = 0;
    return;
  }
  unsigned long long last = ~0ull;
  for (int r = 0; r < best; ++r) {
    unsigned long long key = 0;
    for (int i = threadIdx.x; i < n; i += BEAM_THREADS)
      if (keys[i] < last) key = max(key, keys[i]);
    key = warp_max_key(key);
    if (lane == 0) from_warp[warp] = key;
    __syncthreads();
    last = warp_max_key(from_warp[lane & (BEAM_WARPS - 1)]);
    if (threadIdx.x == 0) out[r] = last;
    __syncthreads();
  }
}

// Shared memory of beam_scan_kernel: stages of a chunk each, as its bytes stand in memory from the 16-byte border below on.
template <int NV>
struct BeamScan {
  static constexpr int STAGES = 3, CHUNK_BYTES = BEAM_THREADS * NV * 16, STAGE_BYTES = CHUNK_BYTES + 32, SMEM_BYTES = STAGES * STAGE_BYTES;
  static constexpr int WAIT_LIMIT = 1 << 16;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// One slice of one row, in chunks of NV x 16 bytes a thread that come by bulk copies, three chunks ahead.
//
// VEC: rows start on 16 bytes, and a thread reads 16 bytes at a time; else it reads words of 4 (a rule of the call, not of the row, so
// that equal rows have equal sums).  Copies are of whole 16-byte pieces inside the row; what stands at its ends is filled in.
//
// The sum: each thread has its own running maximum and adds 2^(x log2(e) - c), c = maximum x log2(e).
// The `best` largest: in the first chunk each group of threads (a warp for up to 8 results) has a largest logit, and the least of them
// bounds the `best`-th from below; what reaches it, 22 of 8192 logits on average for 8 groups, is listed, and what of the other chunks
// does.  Where equal logits overflow the list, the best of the list and the chunk are picked one at a time.
template <typename T, int NV, bool VEC>
__global__ void __launch_bounds__(BEAM_THREADS, 3) beam_scan_kernel(const BeamParams p, const int groups) {
  using C = BeamScan<NV>;
  constexpr int S = (int)sizeof(T), N = 16 / S, CHUNK = BEAM_THREADS * NV * N;
  constexpr uint32_t NONE = S == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;  // -inf
  extern __shared__ __align__(128) uint8_t stages[];
  __shared__ unsigned long long keys[BEAM_KEYS];
  __shared__ float low[BEAM_WARPS], high[BEAM_WARPS];
  __shared__ float2 sums[BEAM_WARPS];
  __shared__ unsigned long long from_warp[BEAM_WARPS], picked[FT_MAX_BEAMS];
  __shared__ __align__(8) unsigned long long barrier[C::STAGES];
  __shared__ int more[3];  // listed by a chunk, by turns: the next chunk's is cleared before a chunk's last barrier
  allow_dependent_launch();
  wait_for_prior_grid();
  const int row = (int)(blockIdx.x / (unsigned)p.slices), slice = (int)(blockIdx.x - (unsigned)row * p.slices);
  const int req = row / p.beams, beam = row - req * p.beams, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned long long* __restrict__ out = p.keys + (int64_t)blockIdx.x * p.best;
  const int begin = slice * p.slice_len, end = min(p.vocab, begin + p.slice_len);
  const float score = __ldg(p.scores + req * p.scores_s0 + beam * p.scores_s1);
  if (!(fabsf(score) < INFINITY) || begin >= end) {  // nothing comes from this beam
    for (int i = tid; i < p.best; i += BEAM_THREADS) out[i] = 0;
    if (tid == 0) p.sums[blockIdx.x] = make_float2(-INFINITY, 0.f);
    return;
  }
  const T* __restrict__ base = static_cast<const T*>(p.logits) + req * p.logits_s0 + beam * p.logits_s1;
  const uintptr_t row_at = reinterpret_cast<uintptr_t>(base), row_end = row_at + (int64_t)p.vocab * S;
  const uint32_t bars = (uint32_t)__cvta_generic_to_shared(barrier), ring = (uint32_t)__cvta_generic_to_shared(stages);
  // a chunk's bytes: from `at` (its stage begins at the 16-byte border below), of which [from, to) are copied
  struct Span {
    uintptr_t at, from, to;
  };
  auto span_of = [&](int first) {
    const uintptr_t a = row_at + (int64_t)first * S, b = row_at + (int64_t)min(end, first + CHUNK) * S;
    Span s = {a, a & ~(uintptr_t)15, (b + 15) & ~(uintptr_t)15};
    if (s.from < row_at) s.from += 16;
    if (s.to > row_end) s.to -= 16;
    if (s.to < s.from) s.to = s.from;
    return s;
  };
  auto issue = [&](int chunk) {
    const int first = begin + chunk * CHUNK;
    if (first >= end) return;
    const Span s = span_of(first);
    const uint32_t bytes = (uint32_t)(s.to - s.from), bar = bars + 8 * (chunk % C::STAGES);
    mbar_arrive_expect_tx(bar, bytes);
    if (bytes > 0)
      bulk_load(ring + (chunk % C::STAGES) * C::STAGE_BYTES + (uint32_t)(s.from - (s.at & ~(uintptr_t)15)), reinterpret_cast<const void*>(s.from), bytes, bar);
  };
  if (tid == 0) {
    for (int i = 0; i < C::STAGES; ++i) mbar_init(bars + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    proxy_fence();
    for (int i = 0; i < C::STAGES; ++i) issue(i);
  }
  if (tid < 3) more[tid] = 0;
  __syncthreads();
  float top = -INFINITY, off = 0.f, sum = 0.f, least = -3.4028234e38f;
  int listed = 0, turn = 0, chunk = 0;
  uint32_t phase = 0;
  bool late = false;
#pragma unroll 1
  for (int first = begin; first < end; first += CHUNK, ++chunk) {
    const int stage = chunk % C::STAGES;
    const int len = min(end - first, CHUNK);
    const Span s = span_of(first);
    uint8_t* const bytes = stages + stage * C::STAGE_BYTES;
    const uint32_t shift = (uint32_t)(s.at & 15);
    late |= !mbar_wait_warp(bars + 8 * stage, phase, C::WAIT_LIMIT);
    if (stage == C::STAGES - 1) phase ^= 1u;
    const uintptr_t stop = s.at + (int64_t)len * S, whole = (stop + 15) & ~(uintptr_t)15;
    if (s.from > s.at || s.to < whole) {  // the row's ends, and -inf up to the next 16 bytes
      if (tid < 2 * N) {
        const uintptr_t at = tid < N ? s.at + tid * S : s.to + (tid - N) * S;
        if (tid < N ? at < s.from && at < stop : at < whole && at >= s.at && at >= s.from)
          *reinterpret_cast<T*>(bytes + (at - (s.at & ~(uintptr_t)15))) = at < stop ? *reinterpret_cast<const T*>(at) : from_float<T>(-INFINITY);
      }
      proxy_fence();
      __syncthreads();
    }
    // word w of piece j; number of its first element in the chunk
    auto number = [&](int j, int e) {
      if constexpr (VEC) return (j * BEAM_THREADS + tid) * N + e;
      if constexpr (S == 4) return (4 * j + e) * BEAM_THREADS + tid;
      return 2 * ((4 * j + (e >> 1)) * BEAM_THREADS + tid) + (e & 1);
    };
    uint4 x[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if constexpr (VEC) {
        x[j] = number(j, 0) < len ? *reinterpret_cast<const uint4*>(bytes + number(j, 0) * S) : make_uint4(NONE, NONE, NONE, NONE);
      } else {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = number(j, e * (4 / S));
          const uint8_t* const from = bytes + shift + i * S;
          if constexpr (S == 4) {
            w[e] = i < len ? *reinterpret_cast<const uint32_t*>(from) : NONE;
          } else {
            const uint32_t a = i < len ? *reinterpret_cast<const uint16_t*>(from) : NONE & 0xffffu;
            w[e] = a | (i + 1 < len ? (uint32_t)*reinterpret_cast<const uint16_t*>(from + 2) << 16 : NONE & 0xffff0000u);
          }
        }
        x[j] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    float piece[NV], mine = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      piece[j] = vec_max<T>(x[j]);
      mine = fmaxf(mine, piece[j]);
    }
    if (mine > top) {  // (with +inf, c is it too and the sum NaN, as with NaN)
      const float c = mine * BEAM_LOG2E;
      sum = top == -INFINITY ? sum : sum * fast_exp2(off - c);
      top = mine;
      off = c;
    }
    float2 sum2[2] = {make_float2(sum, 0.f), make_float2(0.f, 0.f)};
    const float2 scale2 = make_float2(BEAM_LOG2E, BEAM_LOG2E), off2 = make_float2(-off, -off);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
      for (int e = 0; e < N / 2; ++e) {
        float2 y;
        if constexpr (S == 4)
          y = make_float2(__uint_as_float(w[2 * e]), __uint_as_float(w[2 * e + 1]));
        else
          y = unpack2<T>(w[e]);
        y = __ffma2_rn(y, scale2, off2);
        sum2[e & 1] = __fadd2_rn(sum2[e & 1], make_float2(fast_exp2(y.x), fast_exp2(y.y)));
      }
    }
    sum = (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
    if (first == begin) {
      float all;
      least = fmaxf(least, group_bound(mine, groups, low, high, all));
    }
    // what reaches the bound (the pieces are unpacked anew: kept since the sum they would take 100 registers)
    if (__any_sync(0xffffffffu, mine >= least)) {
      uint32_t hits = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!__any_sync(0xffffffffu, piece[j] >= least)) continue;
        asm volatile("" : "+r"(x[j].x), "+r"(x[j].y), "+r"(x[j].z), "+r"(x[j].w));
#pragma unroll
        for (int e = 0; e < N; ++e) hits |= vec_at<T>(x[j], e) >= least ? 1u << (j * N + e) : 0u;
      }
      if (hits != 0) {
        int to = listed + atomicAdd(&more[turn], __popc(hits));
        for (; hits != 0; hits &= hits - 1, ++to) {
          const int bit = __ffs(hits) - 1, i = number(bit / N, bit % N);
          const float y = to_float<T>(*reinterpret_cast<const T*>(bytes + shift + i * S));
          if (to < BEAM_KEYS) keys[to] = ((unsigned long long)ordered(y) << 32) | (0xffffffffu - (uint32_t)(first + i));
        }
      }
    }
    const int next = turn == 2 ? 0 : turn + 1;
    if (tid == 0) more[next] = 0;
    __syncthreads();
    const int now = listed + more[turn];
    turn = next;
    if (tid == 0) issue(chunk + C::STAGES);
    if (now <= BEAM_KEYS) {
      listed = now;
      continue;
    }
    unsigned long long last = ~0ull;
#pragma unroll 1
    for (int r = 0; r < p.best; ++r) {
      unsigned long long key = 0;
      for (int i = tid; i < listed; i += BEAM_THREADS)
        if (keys[i] < last) key = max(key, keys[i]);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        asm volatile("" : "+r"(x[j].x), "+r"(x[j].y), "+r"(x[j].z), "+r"(x[j].w));
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float y = vec_at<T>(x[j], e);
          const unsigned long long k = ((unsigned long long)ordered(y) << 32) | (0xffffffffu - (uint32_t)(first + number(j, e)));
          if (y >= least && k < last) key = max(key, k);
        }
      }
      key = warp_max_key(key);
      if (lane == 0) from_warp[warp] = key;
      __syncthreads();
      last = warp_max_key(from_warp[lane & (BEAM_WARPS - 1)]);
      if (tid == 0) picked[r] = last;
      __syncthreads();
    }
    for (int i = tid; i < p.best; i += BEAM_THREADS) keys[i] = picked[i];
    listed = p.best;
    least = from_ordered((uint32_t)(last >> 32));  // (more than `best` were there, so none is missing)
    __syncthreads();
  }
  // the threads' sums, over the largest offset
  if (top == -INFINITY) off = -INFINITY;
  const float warp_off = warp_max(off), from = warp_off == -INFINITY ? 0.f : warp_off;
  const float total = warp_sum(sum == 0.f ? 0.f : sum * fast_exp2(off - from));
  if (lane == 0) sums[warp] = make_float2(warp_off, total);
  best_of_list(keys, listed, out, p.best, from_warp);
  if (__syncthreads_or(late)) {  // a copy that did not come: its bytes may not land in another CTA's memory
    if (tid == 0) flag_error(FT_DEV_WAIT_TIMEOUT);
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  }
  if (warp == 0) {
    const float2 x = lane < BEAM_WARPS ? sums[lane] : make_float2(-INFINITY, 0.f);
    const float most = warp_max(x.x), from_all = most == -INFINITY ? 0.f : most;
    const float all = warp_sum(x.y == 0.f ? 0.f : x.y * fast_exp2(x.x - from_all));
    if (lane == 0) p.sums[blockIdx.x] = make_float2(most, all);
  }
}

// A candidate of the merge: its score, and in their order its beam, logit and token.
struct BeamCandidate {
  double score;
  unsigned long long key;
  int beam;
};
__device__ __forceinline__ bool before(const BeamCandidate& a, const BeamCandidate& b) {
  return a.score != b.score ? a.score > b.score : a.beam != b.beam ? a.beam < b.beam : a.key > b.key;
}

// A CTA per request: each beam's sum from its slices (64 bits), each listed logit's score, and a threshold between the best
// and the rest, found by halving, that leaves few to be ranked.  REGS scores a thread stay in registers, in fp32 rounded down, which
// keeps their order; more are made anew each time.
template <int REGS>
__global__ void __launch_bounds__(BEAM_THREADS) beam_merge_kernel(const BeamParams p) {
  __shared__ double shift[FT_MAX_BEAMS];  // a beam's score less its logarithm; NaN: nothing comes from it
  __shared__ BeamCandidate list[BEAM_KEYS];
  __shared__ float high[BEAM_WARPS];
  __shared__ int counts[3][BEAM_WARPS], place[BEAM_KEYS];
  __shared__ BeamCandidate from_warp[BEAM_WARPS];
  __shared__ int listed;
  const int req = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) listed = 0;
  allow_dependent_launch();
  wait_for_prior_grid();
  const float2* __restrict__ sums = p.sums + (int64_t)req * p.beams * p.slices;
  const int per_beam = p.slices * p.best, total = p.beams * per_beam;
  const unsigned long long* __restrict__ keys = p.keys + (int64_t)req * total;
  unsigned long long mine[REGS];
#pragma unroll
  for (int k = 0; k < REGS; ++k) mine[k] = tid + k * BEAM_THREADS < total ? __ldcg(keys + tid + k * BEAM_THREADS) : 0;
  for (int b = warp; b < p.beams; b += BEAM_WARPS) {
    const float score = p.scores[req * p.scores_s0 + b * p.scores_s1];
    float top = -INFINITY;
    for (int s = lane; s < p.slices; s += 32) top = fmaxf(top, __ldcg(&sums[b * p.slices + s]).x);
    top = warp_max(top);
    double sum = 0;
    for (int s = lane; s < p.slices; s += 32) {
      const float2 x = __ldcg(&sums[b * p.slices + s]);
      if (x.y != 0.f) sum += (double)x.y * exp2((double)x.x - (double)top);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      // (the terms' exponents were taken x BEAM_LOG2E, which is not log2(e): by it the offset is a logit again, and what is left of
      // the difference, 1.3e-8 of the distance from the largest logit to the mean, is below fp32's half step)
      const double lse = (double)top / (double)BEAM_LOG2E + log(sum);
      shift[b] = fabsf(score) < INFINITY && fabs(lse) < (double)INFINITY ? (double)score - lse : (double)NAN;
    }
  }
  __syncthreads();
  // candidate i with this key; false: there is none
  auto candidate = [&](int i, unsigned long long key, BeamCandidate& c) {
    c.key = key;
    c.beam = i / per_beam;
    c.score = (double)from_ordered((uint32_t)(key >> 32)) + shift[c.beam];
    return key != 0 && c.score == c.score;
  };
  BeamCandidate c;
  float score[REGS], top = -INFINITY;
#pragma unroll
  for (int k = 0; k < REGS; ++k) {
    const int i = tid + k * BEAM_THREADS;
    score[k] = i < total && candidate(i, mine[k], c) ? __double2float_rd(c.score) : -INFINITY;
    top = fmaxf(top, score[k]);
  }
  auto beyond = [&](auto fn) {  // those that no register holds
    for (int i = tid + REGS * BEAM_THREADS; i < total; i += BEAM_THREADS)
      if (candidate(i, __ldcg(keys + i), c)) fn(__double2float_rd(c.score));
  };
  beyond([&](float x) { top = fmaxf(top, x); });
  top = warp_max(top);
  if (lane == 0) high[warp] = top;
  __syncthreads();
  top = high[0];
#pragma unroll
  for (int w = 1; w < BEAM_WARPS; ++w) top = fmaxf(top, high[w]);
  int turn = 0;
  auto reach = [&](float least) {  // how many do
    int n = 0;
#pragma unroll
    for (int k = 0; k < REGS; ++k) n += score[k] >= least;
    beyond([&](float x) { n += x >= least; });
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) counts[turn][warp] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < BEAM_WARPS; ++w) n += counts[turn][w];
    turn = turn == 2 ? 0 : turn + 1;
    return n;
  };
  // the threshold: steps that double away from the best until enough reach it, then halves between the last two
  const int enough = 2 * p.best + 32;
  float least = -3.4028234e38f;
  int n = 0;
  if (top > -INFINITY) {
    float above = top, step = 1.f;
    for (; step < 1e6f; step *= 4.f) {
      n = reach(top - step);
      if (n >= p.best) {
        least = top - step;
        break;
      }
      above = top - step;
    }
    if (step < 1e6f)
      for (int i = 0; i < 24 && n > enough; ++i) {
        const float middle = 0.5f * (above + least);
        const int m = reach(middle);
        if (m >= p.best) {
          least = middle;
          n = m;
        } else {
          above = middle;
        }
      }
  }
  auto put = [&](int i, unsigned long long key) {
    if (candidate(i, key, c) && __double2float_rd(c.score) >= least) {
      const int to = atomicAdd(&listed, 1);
      if (to < BEAM_KEYS) list[to] = c;
    }
  };
#pragma unroll
  for (int k = 0; k < REGS; ++k)
    if (score[k] >= least) put(tid + k * BEAM_THREADS, mine[k]);
  for (int i = tid + REGS * BEAM_THREADS; i < total; i += BEAM_THREADS) put(i, __ldcg(keys + i));
  for (int i = tid; i < BEAM_KEYS; i += BEAM_THREADS) place[i] = 0;
  __syncthreads();
  auto store = [&](int at, float score, int64_t beam, int64_t token) {
    p.out_scores[req * p.out_scores_s0 + at] = score;
    if (p.beams_64)
      static_cast<long long*>(p.out_beams)[req * p.out_beams_s0 + at] = beam;
    else
      static_cast<int*>(p.out_beams)[req * p.out_beams_s0 + at] = (int)beam;
    if (p.tokens_64)
      static_cast<long long*>(p.out_tokens)[req * p.out_tokens_s0 + at] = token;
    else
      static_cast<int*>(p.out_tokens)[req * p.out_tokens_s0 + at] = (int)token;
  };
  auto store_candidate = [&](int at, const BeamCandidate& x) { store(at, (float)x.score, x.beam, 0xffffffffu - (uint32_t)x.key); };
  n = listed;
  if (n <= BEAM_KEYS) {
    // ranked by counting; where they are few, several threads share one's count
    int parts = 1;
    while (parts < 8 && n * parts * 2 <= BEAM_THREADS) parts *= 2;
    for (int i = tid / parts; i < n; i += BEAM_THREADS / parts) {
      c = list[i];
      int rank = 0;
      for (int k = tid & (parts - 1); k < n; k += parts) rank += before(list[k], c);
      if (rank != 0) atomicAdd(&place[i], rank);
    }
    __syncthreads();
    for (int i = tid; i < n; i += BEAM_THREADS)
      if (place[i] < p.best) store_candidate(place[i], list[i]);
    for (int i = n + tid; i < p.best; i += BEAM_THREADS) store(i, -INFINITY, -1, -1);
    return;
  }
  // equal scores without end: one at a time, the best of what comes behind the last one
  BeamCandidate last = {(double)INFINITY, 0, -1};
  for (int r = 0; r < p.best; ++r) {
    BeamCandidate most = {-(double)INFINITY, 0, 0x7fffffff};
    for (int i = tid; i < total; i += BEAM_THREADS)
      if (candidate(i, __ldcg(keys + i), c) && before(last, c) && before(c, most)) most = c;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      BeamCandidate other;
      other.score = __shfl_xor_sync(0xffffffffu, most.score, o);
      other.key = __shfl_xor_sync(0xffffffffu, most.key, o);
      other.beam = __shfl_xor_sync(0xffffffffu, most.beam, o);
      if (before(other, most)) most = other;
    }
    if (lane == 0) from_warp[warp] = most;
    __syncthreads();
    last = from_warp[0];
#pragma unroll
    for (int w = 1; w < BEAM_WARPS; ++w)
      if (before(from_warp[w], last)) last = from_warp[w];
    if (tid == 0) store_candidate(r, last);
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ reordering

constexpr int REORDER_WORDS = 16;  // 4-byte words a thread moves

struct ReorderParams {
  uint32_t* table;  // in words of 4 bytes, as the widths and the stride
  const void* rows;
  const void* beams;
  const void* out_rows;
  const void* starts;
  const void* ends;
  int64_t table_rows, width, table_s0, rows_s0, beams_s0, out_rows_s0;
  int32_t from, to, words, rows_64, beams_64, out_rows_64, starts_64, ends_64;  // words: of an element
  int32_t shift;  // a CTA has 2^shift columns, in words
};

// A CTA has some columns of all of a request's rows: it reads every word that it moves before it writes any, so that rows may
// change places.
__global__ void __launch_bounds__(BEAM_THREADS) beam_reorder_kernel(const ReorderParams p) {
  __shared__ int64_t source[FT_MAX_BEAMS], target[FT_MAX_BEAMS];
  wait_for_prior_grid();
  const int req = blockIdx.y;
  const int64_t whole = p.width / p.words;
  int64_t lo = p.starts != nullptr ? load_index(p.starts, p.starts_64, req) : 0, hi = p.ends != nullptr ? load_index(p.ends, p.ends_64, req) : whole;
  bool bad = lo < 0 || lo > whole || hi < 0 || hi > whole;
  lo = (lo < 0 ? 0 : lo > whole ? whole : lo) * p.words;
  hi = (hi < 0 ? 0 : hi > whole ? whole : hi) * p.words;
  const int64_t first = lo + ((int64_t)blockIdx.x << p.shift);
  if (first >= hi && blockIdx.x > 0) return;
  if ((int)threadIdx.x < p.to) {
    int64_t s = -1, t = -1;
    const int64_t beam = load_index(p.beams, p.beams_64, req * p.beams_s0 + threadIdx.x);
    if (beam != -1) {
      t = load_index(p.out_rows, p.out_rows_64, req * p.out_rows_s0 + threadIdx.x);
      s = beam >= 0 && beam < p.from ? load_index(p.rows, p.rows_64, req * p.rows_s0 + beam) : -1;
      if (s < 0 || s >= p.table_rows || t < 0 || t >= p.table_rows) {
        bad = true;
        t = -1;
      }
    }
    source[threadIdx.x] = s == t ? -1 : s;
    target[threadIdx.x] = s == t ? -1 : t;
  }
  if (bad) flag_error(FT_DEV_BAD_ROW_INDEX);
  __syncthreads();
  const int columns = first >= hi ? 0 : (int)(hi - first < (1 << p.shift) ? hi - first : 1 << p.shift);
  uint32_t x[REORDER_WORDS];
#pragma unroll
  for (int j = 0; j < REORDER_WORDS; ++j) {
    const int i = j * BEAM_THREADS + (int)threadIdx.x, r = i >> p.shift, c = i & ((1 << p.shift) - 1);
    if (r < p.to && c < columns && target[r] >= 0) x[j] = p.table[source[r] * p.table_s0 + first + c];
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < REORDER_WORDS; ++j) {
    const int i = j * BEAM_THREADS + (int)threadIdx.x, r = i >> p.shift, c = i & ((1 << p.shift) - 1);
    if (r < p.to && c < columns && target[r] >= 0) p.table[target[r] * p.table_s0 + first + c] = x[j];
  }
}

}  // namespace ft
