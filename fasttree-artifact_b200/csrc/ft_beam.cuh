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

constexpr int BEAM_CTAS = 4;  // of the scan on an SM
constexpr int BEAM_THREADS = 256, BEAM_WARPS = BEAM_THREADS / 32;
// Logits that a slice lists, and pieces with one that it sets aside until it lists them; where more reach its bound, it goes over the
// slice again with the list cut on the way.
constexpr int BEAM_LIST = 512, BEAM_ASIDE = 256;
constexpr int BEAM_KEYS = 1024;  // candidates that the merge lists; beyond that, which takes many equal scores, it picks one at a time

struct BeamParams {
  const void* logits;
  const float* scores;
  float* out_scores;
  void* out_beams;
  void* out_tokens;
  unsigned long long* keys;  // [rows][slices][best] {ordered logit, ~token}, 0: none
  float2* sums;              // [rows][slices] {top, sum of e^(logit - top)}, as the scan's threads add it
  int64_t logits_s0, logits_s1, scores_s0, scores_s1, out_scores_s0, out_beams_s0, out_tokens_s0;
  int32_t batch, beams, vocab, best, beams_64, tokens_64;
  int32_t slices, chunks, per_cta;  // most slices of a row, its chunks, chunks of a CTA
  int32_t pitch;                    // places for a row's chunks: as many as it has, or what its own CTAs have together
};

// The scan's BEAM_THREADS threads that read logits; one more warp sends for them.
__device__ __forceinline__ void beam_sync() { asm volatile("bar.sync 1, %0;\n" ::"n"(BEAM_THREADS) : "memory"); }

// A warp's values sorted, the largest in lane 0.
__device__ __forceinline__ float warp_sorted(float x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, x, o);
      // falling within blocks of `size` where the lane's bit of it is clear, rising where it is set
      x = ((lane & size) == 0) == ((lane & o) == 0) ? fmaxf(x, other) : fminf(x, other);
    }
  return x;
}

// A lower bound of the n-th largest of those threads' logits, which n of them reach, from each thread's largest; `holders`: the
// threads, from the first, that hold any.  Up to 16: the n-th of the largest of 32 groups of eight threads.  More: each full warp's
// r-th, r of them in every warp being enough, and the least of those.  -inf: none.  Between calls with the same shared
// memory there has to be a barrier.
__device__ __forceinline__ float logit_bound(float mine, int n, int holders, float (&low)[32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (n <= 16) {
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) mine = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, o));
    if ((lane & 7) == 0) low[threadIdx.x >> 3] = mine;
    beam_sync();
    return __shfl_sync(0xffffffffu, warp_sorted(low[lane]), n - 1);
  }
  const int full = min(holders >> 5, BEAM_WARPS), r = full > 0 ? (n + full - 1) / full : 33;
  mine = __shfl_sync(0xffffffffu, warp_sorted(mine), min(r, 32) - 1);
  if (lane == 0) low[warp] = r > 32 ? -INFINITY : warp < full ? mine : INFINITY;
  beam_sync();
  float bound = low[0];
#pragma unroll
  for (int w = 1; w < BEAM_WARPS; ++w) bound = fminf(bound, low[w]);
  return bound;
}

// A sum of exponentials around the logit `top` adds 2^(a x - a top): a is log2(e), by one fma with the product a top rounded
// before.  Beyond 2^30 a is 1: that rounding is then more than 2^6 and at last beyond fp32, while x - top is exact, and any logit but top
// itself is 64 or more away, so that its term is 0 in either form.
constexpr float BEAM_LOG2E = 1.4426950408889634f, BEAM_FAR = 1073741824.f;
__device__ __forceinline__ bool beam_near(float top) { return fabsf(top) < BEAM_FAR; }
__device__ __forceinline__ float beam_offset(float top) { return beam_near(top) ? __fmul_rn(top, BEAM_LOG2E) : top; }
// What a sum around `from` is multiplied by to be one around `to`, which is no less; -inf: an empty sum's.
__device__ __forceinline__ float beam_rescale(float from, float to) {
  if (beam_near(from) && beam_near(to)) return fast_exp2(__fsub_rn(__fmul_rn(from, BEAM_LOG2E), __fmul_rn(to, BEAM_LOG2E)));
  return from == to ? 1.f : 0.f;
}
__device__ __forceinline__ double beam_rescale64(float from, float to) {
  if (beam_near(from) && beam_near(to)) return exp2((double)beam_offset(from) - (double)beam_offset(to));
  return from == to ? 1.0 : 0.0;
}

// The best of a list of n keys into out[0 .. best), 0 where the list ends: ranked by counting, or one at a time, whichever
// takes fewer instructions.  By all threads of the scan, behind a barrier.
__device__ __forceinline__ void best_of_list(const unsigned long long* keys, int n, unsigned long long* out, int best,
                                             unsigned long long (&from_warp)[BEAM_WARPS]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (n <= 128 + 16 * best) {
    for (int i = threadIdx.x; i < n; i += BEAM_THREADS) {
      const unsigned long long key = keys[i];
      int rank = 0;
#pragma unroll 8
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
    key = warp_largest(key);
    if (lane == 0) from_warp[warp] = key;
    beam_sync();
    last = warp_largest(from_warp[lane & (BEAM_WARPS - 1)]);
    if (threadIdx.x == 0) out[r] = last;
    beam_sync();
  }
}

// Shared memory of beam_scan_kernel: stages of a chunk each, as its bytes stand in memory from the 16-byte border below on.
template <int NV>
struct BeamScan {
  static constexpr int STAGES = 2, CHUNK_BYTES = BEAM_THREADS * NV * 16, STAGE_BYTES = CHUNK_BYTES + 32, SMEM_BYTES = STAGES * STAGE_BYTES;
  static constexpr int WAIT_LIMIT = 1 << 16;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// Chunks of NV x 16 bytes a thread, that one warp sends for, two ahead of the eight that read them.  A row has p.chunks chunks in
// p.pitch places, and a CTA takes p.per_cta of the places as they follow one another.  What it has of a row is a slice: slice
// number s of a row is that of the s-th CTA that has some of it.  A slice costs about as much as seven chunks beside its own, so
// rows are cut into slices of CTAs of their own (whole rows if they are many) where that leaves few CTAs idle.
//
// VEC: rows start on 16 bytes, and a thread reads 16 bytes at a time; else it reads words of 4 (a rule of the call, not of the row, so
// that equal rows cut alike have equal sums).  Copies are of whole 16-byte pieces inside the row; what stands at its ends is filled in.
//
// The sum: each thread adds its terms around its largest logit (beam_offset), which may lag by 8 (then by 2^11.5 a term).
// The `best` largest: the largest of groups of threads in a slice's first chunk bound the `best`-th from below.  Up to 16 results: the
// `best`-th of 32 of them, which little more than `best` logits reach; else something looser (logit_bound), and what reaches it is
// listed, the list is cut to the best and the last one is the new bound.  It is cut (again) when four times as many chunks have passed
// (twice for more than 32 results), so that about three times `best` logits reach the bound in between, when the warps do not wait for
// each other.  A thread whose piece reaches the bound notes the piece, and the logits that do are found by all threads together:
// done on the spot it takes the whole warp for one thread's.
//
// What bounds it (64 x 4 beams of 131072 bf16 logits, 67 MB, 24 us = 2.8 TB/s): in cycles, a slice of ten chunks takes 30 000 - 1100 a chunk
// for the sum, of which the exponential unit is busy 512, and it serves four CTAs; 4000 until its first chunk is there, all CTAs asking
// at once; 2400 with the first bound, 2500 a cut, 2000 the end.  Without bounds and lists (dealt evenly, then 27 us in all) 22 us, without
// the exponentials too 19.
template <typename T, int NV, bool VEC>
__global__ void __launch_bounds__(BEAM_THREADS + 32, BEAM_CTAS) beam_scan_kernel(const BeamParams p) {
  using C = BeamScan<NV>;
  constexpr int S = (int)sizeof(T), N = 16 / S, CHUNK = BEAM_THREADS * NV * N, PAIR = NV > 1 ? 2 : 1;
  constexpr int PIECES = BEAM_THREADS * NV / PAIR, E = PAIR * N;  // pieces (of one or two vectors) of a chunk, their elements
  constexpr uint32_t NONE = S == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;  // -inf
  constexpr float LEAST = -3.4028234e38f, LAG = 8.f;
  extern __shared__ __align__(128) uint8_t stages[];
  __shared__ unsigned long long keys[BEAM_LIST];
  __shared__ float low[32];
  __shared__ float2 sums[BEAM_WARPS];
  __shared__ unsigned long long from_warp[BEAM_WARPS], picked[FT_MAX_BEAMS];
  __shared__ __align__(8) unsigned long long barrier[2 * C::STAGES];  // full, empty
  __shared__ __align__(16) uint4 aside[BEAM_ASIDE][PAIR];
  __shared__ uint32_t aside_at[BEAM_ASIDE];              // chunk of the row x PIECES + piece
  __shared__ uint16_t pieces[BEAM_THREADS * NV / PAIR];  // of the first chunk
  __shared__ int listed, noted, more[3];
  __shared__ volatile int dead;  // a wait has run out
  allow_dependent_launch();
  wait_for_prior_grid();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t all_places = (int64_t)p.batch * p.beams * p.pitch, place0 = (int64_t)blockIdx.x * p.per_cta;
  int todo = (int)(all_places - place0 < p.per_cta ? all_places - place0 : p.per_cta);
  const uint32_t full0 = (uint32_t)__cvta_generic_to_shared(barrier), empty0 = full0 + 8 * C::STAGES;
  struct Row {
    uintptr_t at;
    bool live;  // else nothing comes from this beam
  };
  auto row_of = [&](int row) {
    const int req = row / p.beams, beam = row - req * p.beams;
    const float score = __ldg(p.scores + req * p.scores_s0 + beam * p.scores_s1);
    return Row{reinterpret_cast<uintptr_t>(static_cast<const T*>(p.logits) + req * p.logits_s0 + beam * p.logits_s1), fabsf(score) < INFINITY};
  };
  int row = (int)(place0 / p.pitch), k = (int)(place0 - (int64_t)row * p.pitch), stage = 0;
  if (p.pitch > p.chunks) todo = min(todo, p.chunks - k);  // (a row's CTAs are its own: the last one's last places are empty)
  uint32_t phase = 0;
  Row here = {0, false};
  bool fresh = true;  // a slice begins
  auto await = [&](uint32_t bar, uint32_t parity) {
    if (dead == 0 && !mbar_wait_warp(bar, parity, C::WAIT_LIMIT)) dead = 1;
  };
  auto advance = [&]() {
    if (++stage == C::STAGES) {
      stage = 0;
      phase ^= 1u;
    }
    if (++k == p.chunks) {
      k = 0;
      ++row;
    }
  };
  if (tid == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(full0 + 8 * i, 1);
      mbar_init(empty0 + 8 * i, BEAM_WARPS);
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    proxy_fence();
    listed = noted = 0;
    dead = 0;
  }
  if (tid < 3) more[tid] = 0;
  __syncthreads();
  if (warp == BEAM_WARPS) {
    // ---- a chunk's bytes: from `at`, whose stage begins at the 16-byte border below; [from, to) are copied, the rest, at the row's ends,
    // is filled in, with -inf up to the next border
    // (a row's score is asked for a row ahead; the first row is copied without asking)
    const int rows = p.batch * p.beams;
    Row ahead = row_of(row);
    ahead.live = true;
    for (int n = 0; n < todo; ++n) {
      if (n == 0 || k == 0) {
        here = ahead;
        if (row + 1 < rows) ahead = row_of(row + 1);
      }
      const uint32_t full = full0 + 8 * stage;
      await(empty0 + 8 * stage, phase ^ 1u);
      uint32_t bytes = 0, to_stage = 0;
      uintptr_t from = 0;
      if (here.live) {
        const int first = k * CHUNK;
        const uintptr_t at = here.at + (int64_t)first * S, stop = here.at + (int64_t)min(p.vocab, first + CHUNK) * S;
        const uintptr_t border = at & ~(uintptr_t)15, whole = (stop + 15) & ~(uintptr_t)15;
        uintptr_t to = whole;
        from = border < here.at ? border + 16 : border;
        if (to > here.at + (int64_t)p.vocab * S) to -= 16;
        if (to < from) to = from;
        bytes = (uint32_t)(to - from);
        uint8_t* const mine = stages + stage * C::STAGE_BYTES;
        to_stage = (uint32_t)__cvta_generic_to_shared(mine + (from - border));
        if (lane < 2 * N) {
          const uintptr_t x = lane < N ? at + lane * S : to + (lane - N) * S;
          if (lane < N ? x < from && x < stop : x < whole && x >= at && x >= from)
            *reinterpret_cast<T*>(mine + (x - border)) = x < stop ? *reinterpret_cast<const T*>(x) : from_float<T>(-INFINITY);
        }
        proxy_fence();
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive_expect_tx(full, bytes);
        if (bytes > 0) bulk_load(to_stage, reinterpret_cast<const void*>(from), bytes, full);
      }
      __syncwarp();
      advance();
    }
  } else {
    // number in the chunk of element e of thread t's vector j
    auto number_of = [&](int t, int j, int e) {
      if constexpr (VEC) return (j * BEAM_THREADS + t) * N + e;
      if constexpr (S == 4) return (4 * j + e) * BEAM_THREADS + t;
      return 2 * ((4 * j + (e >> 1)) * BEAM_THREADS + t) + (e & 1);
    };
    auto number = [&](int j, int e) { return number_of(tid, j, e); };
    auto list = [&](float y, int at) {
      const int to = atomicAdd(&listed, 1);
      if (to < BEAM_LIST) keys[to] = ((unsigned long long)ordered(y) << 32) | (0xffffffffu - (uint32_t)at);
    };
    float top = -INFINITY, least = LEAST;
    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    int from_k = 0;     // the slice's first chunk
    const bool few = p.best <= 16;
    bool lost = false;  // more reached the bound than there was room for
#pragma unroll 1
    for (int n = 0; n < todo; ++n) {
      if (fresh) {
        here = row_of(row);
        from_k = k;
      }
      const int first = k * CHUNK, len = p.vocab - first;
      const uint32_t shift = VEC ? 0u : (uint32_t)(here.at & 15);
      const uint8_t* const bytes = stages + stage * C::STAGE_BYTES + shift;
      auto load = [&](auto full, int j) {
        constexpr bool FULL = decltype(full)::value;
        if constexpr (VEC) {
          return FULL || number(j, 0) < len ? *reinterpret_cast<const uint4*>(bytes + number(j, 0) * S) : make_uint4(NONE, NONE, NONE, NONE);
        } else {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = number(j, e * (4 / S));
            if constexpr (S == 4) {
              w[e] = FULL || i < len ? *reinterpret_cast<const uint32_t*>(bytes + i * S) : NONE;
            } else if (FULL && (shift & 2) == 0) {
              w[e] = *reinterpret_cast<const uint32_t*>(bytes + i * S);
            } else {
              const uint32_t a = FULL || i < len ? *reinterpret_cast<const uint16_t*>(bytes + i * S) : NONE & 0xffffu;
              w[e] = a | (FULL || i + 1 < len ? (uint32_t)*reinterpret_cast<const uint16_t*>(bytes + i * S + 2) << 16 : NONE & 0xffff0000u);
            }
          }
          return make_uint4(w[0], w[1], w[2], w[3]);
        }
      };
      auto pass = [&](auto full) {
        if (fresh) {
          float mine = -INFINITY;
#pragma unroll
          for (int j = 0; j < NV; ++j) mine = fmaxf(mine, vec_max<T>(load(full, j)));
          least = fmaxf(LEAST, logit_bound(mine, p.best, len >= CHUNK ? BEAM_THREADS : VEC ? (len + N - 1) / N : S == 4 ? len : (len + 1) / 2, low));
          top = mine;
        }
        float2 off2, mul2;
        auto around_top = [&]() {
          const float off = top == -INFINITY ? 0.f : beam_offset(top), mul = top == -INFINITY || beam_near(top) ? BEAM_LOG2E : 1.f;
          off2 = make_float2(-off, -off);
          mul2 = make_float2(mul, mul);
        };
        around_top();
        float gate = top == -INFINITY ? LEAST : fminf(least, top + LAG);  // below it a piece needs nothing but its sum
#pragma unroll
        for (int j = 0; j < NV; j += PAIR) {
          uint4 x[PAIR];
          float most = -INFINITY;
#pragma unroll
          for (int u = 0; u < PAIR; ++u) x[u] = load(full, j + u);
          if constexpr (PAIR == 2 && S == 2)
            most = vec_max<T>(make_uint4(max2(x[0].x, x[1].x, T()), max2(x[0].y, x[1].y, T()), max2(x[0].z, x[1].z, T()), max2(x[0].w, x[1].w, T())));
          else
#pragma unroll
            for (int u = 0; u < PAIR; ++u) most = fmaxf(most, vec_max<T>(x[u]));
          if (most >= gate) {
            if (most > top + LAG || top == -INFINITY) {  // (around +inf the sum is NaN, as with NaN)
              const float f = beam_rescale(top, most);
#pragma unroll
              for (int i = 0; i < 2; ++i) sum[i] = __fmul2_rn(sum[i], make_float2(f, f));
              top = most;
              around_top();
              gate = fminf(least, top + LAG);
            }
            if (most >= least) {
              const int to = atomicAdd(&noted, 1), piece = (j / PAIR) * BEAM_THREADS + tid;
              if (fresh && !few) {
                pieces[to] = (uint16_t)piece;
              } else if (to < BEAM_ASIDE) {
#pragma unroll
                for (int u = 0; u < PAIR; ++u) aside[to][u] = x[u];
                aside_at[to] = (uint32_t)k * PIECES + piece;
              }
            }
          }
#pragma unroll
          for (int u = 0; u < PAIR; ++u) {
            const uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
              float2 y;
              if constexpr (S == 4)
                y = make_float2(__uint_as_float(w[2 * e]), __uint_as_float(w[2 * e + 1]));
              else
                y = unpack2<T>(w[e]);
              y = __ffma2_rn(y, mul2, off2);
              sum[e & 1] = __fadd2_rn(sum[e & 1], make_float2(fast_exp2(y.x), fast_exp2(y.y)));
            }
          }
        }
      };
      await(full0 + 8 * stage, phase);
      if (here.live) {
        if (len >= CHUNK)
          pass(std::true_type{});
        else
          pass(std::false_type{});
      }
      __syncwarp();
      if (!(fresh && !few) && lane == 0) mbar_arrive(empty0 + 8 * stage);
      const bool ends = k == p.chunks - 1 || n == todo - 1;
      const int passed = k - from_k + 1;
      int count = 0;
      if (((passed & (passed - 1)) == 0 && (p.best > 32 || (passed & 0x2aaaaaaa) == 0) && !(few && passed == 1)) || ends) {
        // the logits of the noted pieces, of many results' first chunk in its stage
        beam_sync();
        const int n_pieces = noted;
        if (fresh && !few) {
          for (int i0 = tid; i0 < n_pieces * E; i0 += BEAM_THREADS) {
            const int piece = pieces[i0 / E], e = i0 % E, i = number_of(piece % BEAM_THREADS, piece / BEAM_THREADS * PAIR + e / N, e % N);
            const float y = i < len ? to_float<T>(*reinterpret_cast<const T*>(bytes + i * S)) : -INFINITY;
            if (y >= least) list(y, first + i);
          }
        } else {
          for (int i0 = tid; i0 < min(n_pieces, BEAM_ASIDE) * E; i0 += BEAM_THREADS) {
            const int q = i0 / E, e = i0 % E, piece = (int)(aside_at[q] % PIECES);
            const float y = to_float<T>(reinterpret_cast<const T*>(aside[q])[e]);
            if (y >= least)
              list(y, (int)(aside_at[q] / PIECES) * CHUNK + number_of(piece % BEAM_THREADS, piece / BEAM_THREADS * PAIR + e / N, e % N));
          }
          lost |= n_pieces > BEAM_ASIDE;
        }
        beam_sync();
        if (fresh && !few && lane == 0) mbar_arrive(empty0 + 8 * stage);
        count = listed;
        lost |= count > BEAM_LIST;
        if (!ends) {
          const bool cut = !lost && count > p.best;
          if (cut) {
            best_of_list(keys, count, picked, p.best, from_warp);
            beam_sync();
            if (tid < p.best) keys[tid] = picked[tid];
            least = from_ordered((uint32_t)(picked[p.best - 1] >> 32));
          } else if (lost) {
            least = INFINITY;  // the list is made anew in any case
            beam_sync();
          }
          if (tid == 0) {
            noted = 0;
            listed = cut ? p.best : count;
          }
          beam_sync();
        }
      }
      fresh = ends;
      if (ends) {
        // ---- the slice's list, and the threads' sums around the largest of their logits
        const int64_t slice = (int64_t)blockIdx.x - (int64_t)row * p.pitch / p.per_cta, at = (int64_t)row * p.slices + slice;
        const float mine = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        const float warp_top = warp_max(top), total = warp_sum(mine * beam_rescale(top, warp_top));
        if (lane == 0) sums[warp] = make_float2(warp_top, total);
        if (lost) {
          // more than there was room for (the largest logits late in the slice, or many equal ones): all of the slice's logits twice
          // again, for a bound by the threads' largest of all and for the list, which is cut when it may overflow
          constexpr int AT_ONCE = 8;
          const T* const logits = reinterpret_cast<const T*>(here.at);
          const int stop = min(p.vocab, first + CHUNK);
          float largest = -INFINITY;
          for (int i0 = from_k * CHUNK; i0 < stop; i0 += AT_ONCE * BEAM_THREADS) {
            float y[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) y[u] = i0 + u * BEAM_THREADS + tid < stop ? to_float<T>(logits[i0 + u * BEAM_THREADS + tid]) : -INFINITY;
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) largest = fmaxf(largest, y[u]);
          }
          const float low_bound = logit_bound(largest, p.best, min(stop - from_k * CHUNK, BEAM_THREADS), low);
          unsigned long long bound = (unsigned long long)ordered(fmaxf(low_bound, LEAST)) << 32;  // (below every key of that value)
          int turn = 0;
          count = 0;
          auto cut_list = [&](int most) {
            if (count <= most) return;
            best_of_list(keys, count, picked, p.best, from_warp);
            beam_sync();
            if (tid < p.best) keys[tid] = picked[tid];
            bound = picked[p.best - 1];
            count = p.best;
            beam_sync();
          };
          for (int i0 = from_k * CHUNK; i0 < stop; i0 += AT_ONCE * BEAM_THREADS) {
            unsigned long long key[AT_ONCE];
            int mine = 0;
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
              const int i = i0 + u * BEAM_THREADS + tid;
              const float y = i < stop ? to_float<T>(logits[i]) : -INFINITY;
              key[u] = y > -INFINITY ? ((unsigned long long)ordered(y) << 32) | (0xffffffffu - (uint32_t)i) : 0ull;
              mine += key[u] > bound;
            }
            // all of them if they are few, else one of each thread at a time
            const int next = turn == 2 ? 0 : turn + 1;
            if (mine > 0) atomicAdd(&more[turn], mine);
            if (tid == 0) {
              more[next] = 0;
              listed = count;
            }
            beam_sync();
            const bool fits = count + more[turn] <= BEAM_LIST;
            turn = next;
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
              if (key[u] > bound) keys[atomicAdd(&listed, 1)] = key[u];
              if (!fits) {
                beam_sync();
                count = listed;
                beam_sync();
                cut_list(BEAM_LIST - BEAM_THREADS);
                if (tid == 0) listed = count;
                beam_sync();
              }
            }
            beam_sync();
            count = listed;
            beam_sync();
            cut_list(BEAM_LIST - BEAM_THREADS);
          }
          beam_sync();
          if (tid < 3) more[tid] = 0;
        }
        best_of_list(keys, count, p.keys + at * p.best, p.best, from_warp);
        beam_sync();
        if (tid == 0) listed = noted = 0;
        if (warp == 0) {
          const float2 x = lane < BEAM_WARPS ? sums[lane] : make_float2(-INFINITY, 0.f);
          const float most = warp_max(x.x), all = warp_sum(x.y * beam_rescale(x.x, most));
          if (lane == 0) p.sums[at] = make_float2(most, all);
        }
        if (k == p.chunks - 1)  // the row's other places stay empty
          for (int s = (int)slice + 1; s < p.slices; ++s) {
            if (tid < p.best) p.keys[(at + s - slice) * p.best + tid] = 0;
            if (tid == 0) p.sums[at + s - slice] = make_float2(-INFINITY, 0.f);
          }
        beam_sync();
        lost = false;
        top = -INFINITY, least = LEAST;
        sum[0] = sum[1] = make_float2(0.f, 0.f);
      }
      advance();
    }
  }
  __syncthreads();
  if (dead != 0) {  // a copy that did not come: its bytes may not land in another CTA's memory
    if (tid == 0) flag_error(FT_DEV_WAIT_TIMEOUT);
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  }
}

// A candidate of the merge: its score as a whole number in the same order, and in their order its beam, logit and token.
struct BeamCandidate {
  unsigned long long score, key;
  int beam;
};
__device__ __forceinline__ bool before(const BeamCandidate& a, const BeamCandidate& b) {
  return a.score != b.score ? a.score > b.score : a.beam != b.beam ? a.beam < b.beam : a.key > b.key;
}
__device__ __forceinline__ unsigned long long ordered64(double x) {
  const long long b = __double_as_longlong(x + 0.0);
  return b < 0 ? ~(unsigned long long)b : (unsigned long long)b | (1ull << 63);
}
__device__ __forceinline__ double from_ordered64(unsigned long long k) { return __longlong_as_double((long long)((k >> 63) != 0 ? k & ~(1ull << 63) : ~k)); }

// A CTA per request: each beam's sum from its slices (64 bits) and its listed logits' scores, by a warp; then a threshold between
// the best and the rest, found by halving, that leaves few to be ranked.  It goes by the scores in fp32 rounded down, which keep their order.
// Bound by its chain of steps.
__global__ void __launch_bounds__(BEAM_THREADS) beam_merge_kernel(const BeamParams p) {
  extern __shared__ float scores[];       // of all listed logits, -inf where there is none
  // of a beam the logit that its sum is around, and its score less the sum's logarithm (not one number: the logit may dwarf the
  // others); NaN: nothing comes from it
  __shared__ double around[FT_MAX_BEAMS], shift[FT_MAX_BEAMS];
  __shared__ unsigned long long list_score[BEAM_KEYS], list_key[BEAM_KEYS];
  __shared__ uint8_t list_beam[BEAM_KEYS];
  __shared__ float high[BEAM_WARPS];
  __shared__ int counts[3][BEAM_WARPS];
  __shared__ BeamCandidate from_warp[BEAM_WARPS];
  __shared__ int listed;
  const int req = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) listed = 0;
  allow_dependent_launch();
  wait_for_prior_grid();
  const float2* __restrict__ sums = p.sums + (int64_t)req * p.beams * p.slices;
  const int per_beam = p.slices * p.best, total = p.beams * per_beam;
  const unsigned long long* __restrict__ keys = p.keys + (int64_t)req * total;
  constexpr float LEAST = -3.4028234e38f;
  auto score_of = [&](unsigned long long key, int beam) { return ((double)from_ordered((uint32_t)(key >> 32)) - around[beam]) + shift[beam]; };
  auto put_score = [&](int i, unsigned long long key) {
    const double x = score_of(key, i / per_beam);
    // (one that is lower than all of fp32 is a candidate still)
    return scores[i] = key != 0 && x == x ? fmaxf(__double2float_rd(x), LEAST) : -INFINITY;
  };
  const unsigned long long early = tid < total ? __ldcg(keys + tid) : 0;  // asked for before it is needed
  // 2^wide lanes to a beam, at least its slices if they are no more than 32
  int wide = 2;
  while (wide < 5 && (1 << wide) < p.slices) ++wide;
  const int lanes = 1 << wide;
  for (int b0 = warp << (5 - wide); b0 < p.beams; b0 += BEAM_WARPS << (5 - wide)) {
    const int b = b0 + (lane >> wide);
    const bool there = b < p.beams;
    const float score = there ? p.scores[req * p.scores_s0 + b * p.scores_s1] : -INFINITY;
    float2 x = make_float2(-INFINITY, 0.f);  // of the lane's slices
    double sum = 0;
    for (int s = lane & (lanes - 1); there && s < p.slices; s += lanes) {
      const float2 y = __ldcg(&sums[b * p.slices + s]);
      if (s < lanes) {
        x = y;
        sum = (double)x.y;
      } else {
        const float most = fmaxf(x.x, y.x);
        sum = sum * beam_rescale64(x.x, most) + (double)y.y * beam_rescale64(y.x, most);
        x.x = most;
      }
    }
    float most = x.x;
    for (int o = 1; o < lanes; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    sum *= beam_rescale64(x.x, most);
    for (int o = 1; o < lanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    // (the terms' exponents were taken x BEAM_LOG2E, which is not log2(e): by it the offset is a logit again, and what is left of the
    // difference, 1.3e-8 of the distance from the largest logit to the mean, is below fp32's half step)
    const double logit = beam_near(most) ? (double)beam_offset(most) * (1.0 / (double)BEAM_LOG2E) : (double)most, lse = log(sum);
    if (there && (lane & (lanes - 1)) == 0) {
      around[b] = logit;
      shift[b] = fabsf(score) < INFINITY && fabs(logit + lse) < (double)INFINITY ? (double)score - lse : (double)NAN;
    }
  }
  __syncthreads();
  float top = -INFINITY;
#pragma unroll 1
  for (int i = tid; i < total; i += BEAM_THREADS) top = fmaxf(top, put_score(i, i == tid ? early : __ldcg(keys + i)));
  top = warp_max(top);
  if (lane == 0) high[warp] = top;
  __syncthreads();
  top = high[0];
#pragma unroll
  for (int w = 1; w < BEAM_WARPS; ++w) top = fmaxf(top, high[w]);
  // candidate i, which has a score
  auto candidate = [&](int i) {
    BeamCandidate c;
    c.key = __ldcg(keys + i);
    c.beam = i / per_beam;
    c.score = ordered64(score_of(c.key, c.beam));
    return c;
  };
  int turn = 0;
  auto reach = [&](float least) {  // how many do
    int n = 0;
#pragma unroll 2
    for (int i = tid; i < total; i += BEAM_THREADS) n += scores[i] >= least;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) counts[turn][warp] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < BEAM_WARPS; ++w) n += counts[turn][w];
    turn = turn == 2 ? 0 : turn + 1;
    return n;
  };
  // the threshold: steps that grow away from the best until enough reach it, then halves between the last two
  const int enough = 2 * p.best + 32;
  float least = LEAST;
  int n = total;
  if (top > -INFINITY && total > enough) {
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
        const float middle = 0.5f * above + 0.5f * least;  // (their sum may be beyond fp32)
        const int m = reach(middle);
        if (m >= p.best) {
          least = middle;
          n = m;
        } else {
          above = middle;
        }
      }
  }
  for (int i = tid; i < total; i += BEAM_THREADS)
    if (scores[i] >= least) {
      const int to = atomicAdd(&listed, 1);
      if (to < BEAM_KEYS) {
        const BeamCandidate c = candidate(i);
        list_score[to] = c.score;
        list_key[to] = c.key;
        list_beam[to] = (uint8_t)c.beam;
      }
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
  auto store_candidate = [&](int at, const BeamCandidate& x) { store(at, (float)from_ordered64(x.score), x.beam, 0xffffffffu - (uint32_t)x.key); };
  auto listed_candidate = [&](int i) { return BeamCandidate{list_score[i], list_key[i], list_beam[i]}; };
  n = listed;
  if (n <= BEAM_KEYS) {
    // ranked by counting, four threads to a candidate; the order among equal scores is asked for where there are any
    for (int i0 = 0; i0 < n; i0 += BEAM_THREADS / 4) {
      const int i = i0 + (tid >> 2);
      const unsigned long long score = i < n ? list_score[i] : 0;
      int rank = 0, equal = 0;
#pragma unroll 4
      for (int k = tid & 3; k < n; k += 4) {
        const unsigned long long other = list_score[k];
        rank += other > score;
        equal += other == score;
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        rank += __shfl_xor_sync(0xffffffffu, rank, o);
        equal += __shfl_xor_sync(0xffffffffu, equal, o);
      }
      if (i < n && (tid & 3) == 0) {
        const BeamCandidate c = listed_candidate(i);
        if (equal > 1)
          for (int k = 0; k < n; ++k)
            if (list_score[k] == score) rank += before(listed_candidate(k), c);
        if (rank < p.best) store_candidate(rank, c);
      }
    }
    for (int i = n + tid; i < p.best; i += BEAM_THREADS) store(i, -INFINITY, -1, -1);
    return;
  }
  // equal scores without end: one at a time, the best of what comes behind the last one
  BeamCandidate last = {~0ull, 0, -1};
  for (int r = 0; r < p.best; ++r) {
    BeamCandidate most = {0, 0, 0x7fffffff};
    for (int i = tid; i < total; i += BEAM_THREADS)
      if (scores[i] > -INFINITY) {
        const BeamCandidate c = candidate(i);
        if (before(last, c) && before(c, most)) most = c;
      }
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

// (not by ld.global.nc: the selection's merge may write them while this kernel, launched early, waits for it)
__device__ __forceinline__ int64_t load_number(const void* p, int is_64, int64_t i) {
  long long x;
  int y;
  if (is_64) {
    asm volatile("ld.global.b64 %0, [%1];\n" : "=l"(x) : "l"(static_cast<const long long*>(p) + i));
    return x;
  }
  asm volatile("ld.global.b32 %0, [%1];\n" : "=r"(y) : "l"(static_cast<const int*>(p) + i));
  return y;
}

// A CTA has some columns of all of a request's rows: it reads every word that it moves before it writes any, so that rows may
// change places.
__global__ void __launch_bounds__(BEAM_THREADS) beam_reorder_kernel(const ReorderParams p) {
  __shared__ int64_t source[FT_MAX_BEAMS], target[FT_MAX_BEAMS];
  wait_for_prior_grid();
  const int req = blockIdx.y;
  const int64_t whole = p.width / p.words;
  // (what does not depend on one another is asked for at once: the call's length is this chain, the rows' numbers, the rows)
  int64_t beam = -1, t = -1;
  if ((int)threadIdx.x < p.to) {
    beam = load_number(p.beams, p.beams_64, req * p.beams_s0 + threadIdx.x);
    t = load_number(p.out_rows, p.out_rows_64, req * p.out_rows_s0 + threadIdx.x);
  }
  int64_t lo = p.starts != nullptr ? load_number(p.starts, p.starts_64, req) : 0, hi = p.ends != nullptr ? load_number(p.ends, p.ends_64, req) : whole;
  bool bad = lo < 0 || lo > whole || hi < 0 || hi > whole;
  lo = (lo < 0 ? 0 : lo > whole ? whole : lo) * p.words;
  hi = (hi < 0 ? 0 : hi > whole ? whole : hi) * p.words;
  const int64_t first = lo + ((int64_t)blockIdx.x << p.shift);
  if (first >= hi && blockIdx.x > 0) return;
  if ((int)threadIdx.x < p.to) {
    int64_t s = -1;
    if (beam != -1) {
      s = beam >= 0 && beam < p.from ? load_number(p.rows, p.rows_64, req * p.rows_s0 + beam) : -1;
      if (s < 0 || s >= p.table_rows || t < 0 || t >= p.table_rows) {
        bad = true;
        s = t = -1;
      }
    }
    source[threadIdx.x] = s;
    target[threadIdx.x] = beam == -1 || s == t ? -1 : t;
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
