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

// One slice of one row, in chunks of NV 16-byte pieces a thread, or as many elements one at a time where rows do not start on 16
// bytes (a rule of the call, not of the row, so that equal rows have equal sums).
//
// The sum: each thread has its own running maximum and adds 2^(x log2(e) - c), c = maximum x log2(e).
// The `best` largest: in the first chunk each group of threads (a warp for up to 8 results) has a largest logit, and the least of them
// bounds the `best`-th from below; what reaches it, 22 of 8192 logits on average for 8 groups, is listed, and what of the other chunks
// does.  Where equal logits overflow the list, the best of the list and the chunk are picked one at a time.
template <typename T, int NV, bool VEC>
__global__ void __launch_bounds__(BEAM_THREADS, 4) beam_scan_kernel(const BeamParams p, const int groups) {
  constexpr int N = Vec<T>::N, CHUNK = BEAM_THREADS * NV * N;
  __shared__ unsigned long long keys[BEAM_KEYS];
  __shared__ float low[BEAM_WARPS], high[BEAM_WARPS];
  __shared__ float2 sums[BEAM_WARPS];
  __shared__ unsigned long long from_warp[BEAM_WARPS], picked[FT_MAX_BEAMS];
  __shared__ int more[3];  // listed by a chunk, by turns: the next chunk's is cleared before a chunk's last barrier
  allow_dependent_launch();
  wait_for_prior_grid();
  const int row = (int)(blockIdx.x / (unsigned)p.slices), slice = (int)(blockIdx.x - (unsigned)row * p.slices);
  const int req = row / p.beams, beam = row - req * p.beams, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned long long* __restrict__ out = p.keys + (int64_t)blockIdx.x * p.best;
  const float score = __ldg(p.scores + req * p.scores_s0 + beam * p.scores_s1);
  if (!(fabsf(score) < INFINITY)) {  // nothing comes from this beam
    for (int i = threadIdx.x; i < p.best; i += BEAM_THREADS) out[i] = 0;
    if (threadIdx.x == 0) p.sums[blockIdx.x] = make_float2(-INFINITY, 0.f);
    return;
  }
  if (threadIdx.x < 3) more[threadIdx.x] = 0;
  const T* __restrict__ base = static_cast<const T*>(p.logits) + req * p.logits_s0 + beam * p.logits_s1;
  const int begin = slice * p.slice_len, end = min(p.vocab, begin + p.slice_len);
  float top = -INFINITY, off = 0.f, sum = 0.f, least = -3.4028234e38f;
  int listed = 0, turn = 0;
#pragma unroll 1
  for (int first = begin; first < end; first += CHUNK) {
    // element e of piece j of a thread is number first + (j * BEAM_THREADS + thread) * N + e, either way
    uint4 x[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = first + (j * BEAM_THREADS + (int)threadIdx.x) * N;
      if (VEC && at + N <= end) {
        x[j] = load_stream(base + at);
      } else {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (sizeof(T) == 4) {
            w[e] = at + e < end ? __float_as_uint(to_float<T>(base[at + e])) : 0xff800000u;
          } else {
            const uint16_t* raw = reinterpret_cast<const uint16_t*>(base);
            const uint32_t none = std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;  // -inf
            const uint32_t a = at + 2 * e < end ? raw[at + 2 * e] : none, b = at + 2 * e + 1 < end ? raw[at + 2 * e + 1] : none;
            w[e] = a | b << 16;
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
        if constexpr (sizeof(T) == 4)
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
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!__any_sync(0xffffffffu, piece[j] >= least)) continue;
        asm volatile("" : "+r"(x[j].x), "+r"(x[j].y), "+r"(x[j].z), "+r"(x[j].w));
        const int at = first + (j * BEAM_THREADS + (int)threadIdx.x) * N;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float y = vec_at<T>(x[j], e);
          if (y >= least) {
            const int to = listed + atomicAdd(&more[turn], 1);
            if (to < BEAM_KEYS) keys[to] = ((unsigned long long)ordered(y) << 32) | (0xffffffffu - (uint32_t)(at + e));
          }
        }
      }
    }
    const int next = turn == 2 ? 0 : turn + 1;
    if (threadIdx.x == 0) more[next] = 0;
    __syncthreads();
    const int now = listed + more[turn];
    turn = next;
    if (now <= BEAM_KEYS) {
      listed = now;
      continue;
    }
    unsigned long long last = ~0ull;
#pragma unroll 1
    for (int r = 0; r < p.best; ++r) {
      unsigned long long key = 0;
      for (int i = threadIdx.x; i < listed; i += BEAM_THREADS)
        if (keys[i] < last) key = max(key, keys[i]);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        asm volatile("" : "+r"(x[j].x), "+r"(x[j].y), "+r"(x[j].z), "+r"(x[j].w));
        const int at = first + (j * BEAM_THREADS + (int)threadIdx.x) * N;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float y = vec_at<T>(x[j], e);
          const unsigned long long k = ((unsigned long long)ordered(y) << 32) | (0xffffffffu - (uint32_t)(at + e));
          if (y >= least && k < last) key = max(key, k);
        }
      }
      key = warp_max_key(key);
      if (lane == 0) from_warp[warp] = key;
      __syncthreads();
      last = warp_max_key(from_warp[lane & (BEAM_WARPS - 1)]);
      if (threadIdx.x == 0) picked[r] = last;
      __syncthreads();
    }
    for (int i = threadIdx.x; i < p.best; i += BEAM_THREADS) keys[i] = picked[i];
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
  __syncthreads();
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

// A CTA per request: each beam's sum from its slices (64 bits), each listed logit's score, and as in the slices a bound that keeps most
// of them out of the ranking.
__global__ void __launch_bounds__(BEAM_THREADS) beam_merge_kernel(const BeamParams p, const int groups) {
  __shared__ double shift[FT_MAX_BEAMS];  // a beam's score less its logarithm; NaN: nothing comes from it
  __shared__ BeamCandidate list[BEAM_KEYS];
  __shared__ float low[BEAM_WARPS], high[BEAM_WARPS];
  __shared__ BeamCandidate from_warp[BEAM_WARPS];
  __shared__ int listed;
  const int req = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) listed = 0;
  allow_dependent_launch();
  wait_for_prior_grid();
  const float2* __restrict__ sums = p.sums + (int64_t)req * p.beams * p.slices;
  for (int b = warp; b < p.beams; b += BEAM_WARPS) {
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
    const float score = p.scores[req * p.scores_s0 + b * p.scores_s1];
    if (lane == 0) {
      // (the terms' exponents were taken x BEAM_LOG2E, which is not log2(e): by it the offset is a logit again, and what is left of
      // the difference, 1.3e-8 of the distance from the largest logit to the mean, is below fp32's half step)
      const double lse = (double)top / (double)BEAM_LOG2E + log(sum);
      shift[b] = fabsf(score) < INFINITY && fabs(lse) < (double)INFINITY ? (double)score - lse : (double)NAN;
    }
  }
  __syncthreads();
  const int lists = p.beams * p.slices, total = lists * p.best;
  const unsigned long long* __restrict__ keys = p.keys + (int64_t)req * total;
  // candidate i, the lists' first ones first (so that every group of threads has some of the best); false: there is none
  auto candidate = [&](int i, BeamCandidate& c) {
    const int rank = i / lists, list = i - rank * lists;
    c.key = __ldcg(keys + list * p.best + rank);
    c.beam = list / p.slices;
    c.score = (double)from_ordered((uint32_t)(c.key >> 32)) + shift[c.beam];
    return c.key != 0 && c.score == c.score;
  };
  BeamCandidate c;
  // (the bound in fp32, rounded towards -inf, so that it stays one)
  float mine = -INFINITY, top;
  for (int i = threadIdx.x; i < total; i += BEAM_THREADS)
    if (candidate(i, c)) mine = fmaxf(mine, __double2float_rd(c.score));
  const float bound = group_bound(mine, groups, low, high, top);
  for (int i = threadIdx.x; i < total; i += BEAM_THREADS)
    if (candidate(i, c) && c.score >= (double)bound) {
      const int to = atomicAdd(&listed, 1);
      if (to < BEAM_KEYS) list[to] = c;
    }
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
  const int n = listed;
  if (n <= BEAM_KEYS) {
    for (int i = threadIdx.x; i < n; i += BEAM_THREADS) {
      c = list[i];
      int rank = 0;
      for (int k = 0; k < n; ++k) rank += before(list[k], c);
      if (rank < p.best) store_candidate(rank, c);
    }
    for (int i = n + (int)threadIdx.x; i < p.best; i += BEAM_THREADS) store(i, -INFINITY, -1, -1);
    return;
  }
  // one at a time: the best of what comes behind the last one
  BeamCandidate last = {(double)INFINITY, 0, -1};
  for (int r = 0; r < p.best; ++r) {
    BeamCandidate most = {-(double)INFINITY, 0, 0x7fffffff};
    for (int i = threadIdx.x; i < total; i += BEAM_THREADS)
      if (candidate(i, c) && before(last, c) && before(c, most)) most = c;
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
    if (threadIdx.x == 0) store_candidate(r, last);
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
  int32_t columns;  // of a CTA, in words
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
  const int64_t first = lo + (int64_t)blockIdx.x * p.columns;
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
  const int columns = first >= hi ? 0 : (int)(hi - first < p.columns ? hi - first : p.columns);
  uint32_t x[REORDER_WORDS];
#pragma unroll
  for (int j = 0; j < REORDER_WORDS; ++j) {
    const int i = j * BEAM_THREADS + (int)threadIdx.x, r = i / p.columns, c = i - r * p.columns;
    if (r < p.to && c < columns && target[r] >= 0) x[j] = p.table[source[r] * p.table_s0 + first + c];
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < REORDER_WORDS; ++j) {
    const int i = j * BEAM_THREADS + (int)threadIdx.x, r = i / p.columns, c = i - r * p.columns;
    if (r < p.to && c < columns && target[r] >= 0) p.table[target[r] * p.table_s0 + first + c] = x[j];
  }
}

}  // namespace ft
