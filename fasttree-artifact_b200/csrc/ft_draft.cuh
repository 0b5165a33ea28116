// Drafted tokens: their trees into a plan's masks, and which of them the model agrees with.
//
// Kernels here and in ft_beam.cuh that write row tables let no later launch start early.  That of a tree does: no kernel reads what it
// writes before its own wait.
//
// A request's drafted tokens are numbered so that a parent comes before its children.  The attention itself is ft_extend's: its
// kernels read what a row sees from bits of the plan, and ft_draft_tree sets the few words of them that trees decide.
#pragma once

#include "ft_common.cuh"
#include "ft_draft_span.cuh"

namespace ft {

struct DraftParams {
  const int32_t* drafts;  // the plan's requests (ft_extend_plan.cu)
  const DraftSpan* spans;
  int32_t* extra;
  const void* parents;
  void* positions;
  int32_t parents_64, positions_64, window, words;  // words: of a token's bits in a tile
};

struct Draft {
  int row, n, cached, id, span0, spans;
  int64_t entries;
};

__device__ __forceinline__ Draft load_draft(const int32_t* drafts, int i) {
  const int4 a = __ldg(reinterpret_cast<const int4*>(drafts) + 2 * i), b = __ldg(reinterpret_cast<const int4*>(drafts) + 2 * i + 1);
  return {a.x, a.y, a.z, b.y, b.z, b.w, (int64_t)(((uint64_t)(uint32_t)b.x << 32) | (uint32_t)a.w)};
}

__device__ __forceinline__ int64_t load_index(const void* p, int is_64, int64_t i) {
  return is_64 ? __ldg(static_cast<const long long*>(p) + i) : (int64_t)__ldg(static_cast<const int*>(p) + i);
}

// (by plain loads: slots may be written by the same kernel)
__device__ __forceinline__ int64_t load_slot(const void* p, int is_64, int64_t i) {
  return is_64 ? static_cast<const volatile long long*>(p)[i] : (int64_t)static_cast<const volatile int*>(p)[i];
}

constexpr int DRAFT_THREADS = 128;

// A request's tree in shared memory.
struct Tree {
  int16_t parent[FT_MAX_DRAFT];                      // -1: a root, -2: padding, else an earlier token
  int16_t jump[2][FT_MAX_DRAFT], depth[2][FT_MAX_DRAFT];  // by turns, see load_tree
};

// Reads the tree; a parent that is none, and what hangs on padding, makes a token padding.  Depths by doubling: jump is a token's
// 2^n-th ancestor, or what its climb ends on (below 0), depth the steps to it, so ten rounds do for the longest chain.  Returns
// the depths.  A whole block; ends with a barrier.  (Loops are not unrolled: the kernel is as long as its way from memory.)
__device__ __forceinline__ const int16_t* load_tree(const void* parents, int is_64, const Draft& d, Tree& t) {
  bool bad = false;
#pragma unroll 1
  for (int i = threadIdx.x; i < d.n; i += DRAFT_THREADS) {
    const int64_t p = load_index(parents, is_64, (int64_t)d.row + i);
    const bool ok = p >= -2 && p < i;
    bad |= !ok;
    t.parent[i] = t.jump[0][i] = (int16_t)(ok ? (int)p : -2);
    t.depth[0][i] = ok && p >= 0;
  }
  __syncthreads();
  int now = 0;
  bool more;
#pragma unroll 1
  do {
    more = false;
#pragma unroll 1
    for (int i = threadIdx.x; i < d.n; i += DRAFT_THREADS) {
      int to = t.jump[now][i], steps = t.depth[now][i];
      if (to >= 0) {
        steps += t.depth[now][to];
        to = t.jump[now][to];
        more |= to >= 0;
      }
      t.jump[now ^ 1][i] = (int16_t)to;
      t.depth[now ^ 1][i] = (int16_t)steps;
    }
    now ^= 1;
  } while (__syncthreads_or(more));
#pragma unroll 1
  for (int i = threadIdx.x; i < d.n; i += DRAFT_THREADS)
    if (t.jump[now][i] == -2 && t.depth[now][i] > 0) {  // it hangs on padding
      bad = true;
      t.parent[i] = -2;
      t.depth[now][i] = 0;
    }
  if (bad) flag_error(FT_DEV_BAD_PARENT);
  __syncthreads();
  return t.depth[now];
}

// A CTA per request (several, with the spans shared out, where drafts are long): positions of its tokens, and the words that its tree
// decides.  Bound by a chain of three reads (request, parents and spans, words), the rounds of the depths and a span's climb: 3.1 to
// 5.6 us for drafts of 5 to 64 tokens.  Two stretches of a tile may share a word, in different bits: clearing and setting are atomic, and
// their order does not matter.
__global__ void __launch_bounds__(DRAFT_THREADS) draft_tree_kernel(const DraftParams p) {
  __shared__ Tree tree;
  allow_dependent_launch();
  const Draft d = load_draft(p.drafts, blockIdx.x);
  if (d.n == 0) return;
  const int warp = (threadIdx.x >> 5) + blockIdx.y * (DRAFT_THREADS / 32), warps = gridDim.y * (DRAFT_THREADS / 32);
  int4 a = make_int4(0, 0, 0, 0), b = a;  // the warp's next span
  auto fetch = [&](int s) {
    const int4* raw = reinterpret_cast<const int4*>(p.spans + d.span0 + s);
    a = __ldg(raw);
    b = __ldg(raw + 1);
  };
  if (warp < d.spans) fetch(warp);
  const int16_t* const depth = load_tree(p.parents, p.parents_64, d, tree);
  if (p.positions != nullptr && blockIdx.y == 0)
    for (int i = threadIdx.x; i < d.n; i += DRAFT_THREADS) {
      const int64_t at = (int64_t)d.row + i;
      if (p.positions_64)
        static_cast<long long*>(p.positions)[at] = d.cached + depth[i];
      else
        static_cast<int*>(p.positions)[at] = d.cached + depth[i];
    }
  for (int s = warp; s < d.spans; s += warps) {
    const DraftSpan span = {a.x, a.y, a.z, a.w, b.x, b.y, 0, 0};
    for (int k = threadIdx.x & 31; k < span.tokens; k += 32)
      draft_span_words(span, k, p.window, tree.parent, depth, [&](int word, uint32_t mask, uint32_t bits) {
        int32_t* at = p.extra + span.bits + k * p.words + word;
        if (mask == 0xffffffffu) {
          *at = (int32_t)bits;
        } else {
          atomicAnd(at, (int32_t)(~mask | bits));
          atomicOr(at, (int32_t)bits);
        }
      });
    if (s + warps < d.spans) fetch(s + warps);
  }
}

// ------------------------------------------------------------------------------------------------ acceptance

struct AcceptParams {
  const int32_t* drafts;
  const void* logits;
  const void* targets;
  const void* tokens;
  const void* parents;
  int32_t* accepted;
  int32_t* counts;
  void* next_tokens;
  const void* slots;
  int32_t* kv_entries;
  int64_t logits_s0, accepted_s0, kv_entries_len;
  int32_t vocab, width, targets_64, tokens_64, parents_64, next_64, slots_64;
};

// Whole numbers in the order of floats; -0 and 0 are one, NaN stands below all.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0u : (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t k) { return __uint_as_float((k & 0x80000000u) != 0 ? k & 0x7fffffffu : ~k); }

// 16 bytes of a row as floats
template <typename T>
struct Vec {
  static constexpr int N = 16 / (int)sizeof(T);
};
__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 x;
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "l"(p));
  return x;
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// the larger of each half; a number and NaN: the number
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b, __half) {
  const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b, __nv_bfloat16) {
  const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
// largest of a vector's elements
template <typename T>
__device__ __forceinline__ float vec_max(const uint4& v) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  } else {
    const float2 m = unpack2<T>(max2(max2(v.x, v.y, T()), max2(v.z, v.w, T()), T()));
    return fmaxf(m.x, m.y);
  }
}
template <typename T>
__device__ __forceinline__ float vec_at(const uint4& v, int e) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(w[e]);
  } else {
    const float2 x = unpack2<T>(w[e >> 1]);
    return (e & 1) != 0 ? x.y : x.x;
  }
}

// The largest of a warp's keys, by its halves.
__device__ __forceinline__ unsigned long long warp_largest(unsigned long long key) {
  const uint32_t high = __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32));
  return ((unsigned long long)high << 32) | __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32) == high ? (uint32_t)key : 0u);
}

constexpr int ACCEPT_THREADS = 512;

// Largest logit of one rank's share of a row, as {ordered value, ~index}: a thread's candidates come in rising order, so a larger one
// only replaces the first of equals.  Vectors from the row's first 16-byte border on; what stands before it and behind the last
// vector goes to the first and the last rank.
template <typename T>
__device__ __forceinline__ unsigned long long row_argmax(const T* __restrict__ row, int vocab, int rank, int ranks) {
  constexpr int N = Vec<T>::N, U = 4;
  const int head = min(vocab, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T)), nv = (vocab - head) / N, tail = head + nv * N;
  const int lo = (int)((int64_t)nv * rank / ranks), hi = (int)((int64_t)nv * (rank + 1) / ranks), tid = threadIdx.x;
  float best = -INFINITY;
  uint32_t at = 0xffffffffu;
  if (rank == 0 && tid < head) {
    const float x = to_float<T>(row[tid]);
    if (x > best) best = x, at = (uint32_t)tid;
  }
  uint4 held = make_uint4(0, 0, 0, 0);  // the first vector with the largest so far; which element it is is asked once
  int held_at = -1;
  for (int v0 = lo + tid; v0 < hi; v0 += U * ACCEPT_THREADS) {
    uint4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = load_stream(row + head + (int64_t)min(v0 + u * ACCEPT_THREADS, hi - 1) * N);
#pragma unroll
    for (int u = 0; u < U; ++u) {  // (the last vector once more changes nothing)
      const float m = vec_max<T>(x[u]);
      const bool more = m > best;
      best = more ? m : best;
      held_at = more ? v0 + u * ACCEPT_THREADS : held_at;
      held.x = more ? x[u].x : held.x, held.y = more ? x[u].y : held.y, held.z = more ? x[u].z : held.z, held.w = more ? x[u].w : held.w;
    }
  }
  if (held_at >= 0) {
    int first = 0;
#pragma unroll
    for (int e = N - 1; e >= 0; --e) first = vec_at<T>(held, e) == best ? e : first;
    at = (uint32_t)(head + min(held_at, hi - 1) * N + first);
  }
  if (rank == ranks - 1 && tail + tid < vocab) {
    const float x = to_float<T>(row[tail + tid]);
    if (x > best) best = x, at = (uint32_t)(tail + tid);
  }
  // (nothing above -inf: the row's first element will do)
  return at == 0xffffffffu ? 0xffffffffull - (rank == 0 ? 0u : 1u) : ((unsigned long long)ordered(best) << 32) | (0xffffffffu - at);
}

__device__ __forceinline__ void cluster_arrive_wait() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

// A cluster of CTAs per request walks down its tree: the row of the token it stands at is split among them, each gives its largest
// logit to all (through the cluster's shared memory, in two sets by turns: a CTA that is ahead writes the next step's), and all
// go on to the same child.  So only the rows along the path are read: one to a handful of, say, 32.  Each step costs a row's
// way from memory and the exchange.
template <typename T>
__global__ void __launch_bounds__(ACCEPT_THREADS, 2) draft_accept_kernel(const AcceptParams p) {
  __shared__ int16_t parent[FT_MAX_DRAFT];
  __shared__ int32_t token[FT_MAX_DRAFT];
  __shared__ int16_t path[FT_MAX_DRAFT];
  __shared__ unsigned long long from_cta[2][8], from_warp[ACCEPT_THREADS / 32];
  __shared__ int child_at[3];  // by turns: a step's, the next one's, which is cleared before the step's barrier, and the one before's
  uint32_t rank, ranks;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const Draft d = load_draft(p.drafts, blockIdx.x / ranks);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // (a token that hangs on padding, or has no valid parent, is not reached)
  for (int i = threadIdx.x; i < d.n; i += ACCEPT_THREADS) {
    const int64_t t = load_index(p.tokens, p.tokens_64, (int64_t)d.row + i), up = load_index(p.parents, p.parents_64, (int64_t)d.row + i);
    token[i] = t >= 0 && t <= 0x7fffffff ? (int)t : -1;
    parent[i] = (int16_t)(up >= -1 && up < i ? (int)up : -2);
  }
  if (threadIdx.x < 3) child_at[threadIdx.x] = FT_MAX_DRAFT;
  __syncthreads();
  if (ranks > 1) cluster_arrive_wait();  // all of them run before any writes to another
  int count = 0;
  int64_t next = -1;
  if (d.n > 0 && parent[0] == -1) {
    for (int cur = 0; cur < FT_MAX_DRAFT;) {
      if (threadIdx.x == 0) path[count] = (int16_t)cur;
      ++count;
      if (p.targets != nullptr) {
        next = load_index(p.targets, p.targets_64, (int64_t)d.row + cur);
      } else {
        unsigned long long key = row_argmax(static_cast<const T*>(p.logits) + ((int64_t)d.row + cur) * p.logits_s0, p.vocab, (int)rank, (int)ranks);
        key = warp_largest(key);
        if (lane == 0) from_warp[warp] = key;
        __syncthreads();
        const int set = count & 1;
        key = warp_largest(from_warp[lane & (ACCEPT_THREADS / 32 - 1)]);
        if (ranks > 1) {
          if (threadIdx.x < ranks) {
            uint32_t there;
            const uint32_t here = (uint32_t)__cvta_generic_to_shared(&from_cta[set][rank]);
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(there) : "r"(here), "r"(threadIdx.x));
            asm volatile("st.shared::cluster.u64 [%0], %1;\n" ::"r"(there), "l"(key) : "memory");
          }
          cluster_arrive_wait();
          key = 0;
          for (uint32_t r = 0; r < ranks; ++r) key = max(key, from_cta[set][r]);
        }
        next = (int64_t)(0xffffffffu - (uint32_t)key);
      }
      // the first child that holds it (-1 stands for a token that is none, which no target is)
      const int turn = count % 3;
      int found = FT_MAX_DRAFT;
      for (int i = cur + 1 + (int)threadIdx.x; i < d.n; i += ACCEPT_THREADS)
        if (parent[i] == cur && next >= 0 && (int64_t)token[i] == next) found = min(found, i);
      found = __reduce_min_sync(0xffffffffu, found);
      if (lane == 0 && found < FT_MAX_DRAFT) atomicMin(&child_at[turn], found);
      if (threadIdx.x == 0) child_at[(count + 1) % 3] = FT_MAX_DRAFT;
      __syncthreads();
      cur = child_at[turn];
    }
  }
  if (rank != 0) return;
  __syncthreads();
  const int64_t out = d.id;
  if (threadIdx.x == 0) {
    p.counts[out] = count;
    if (p.next_64)
      static_cast<long long*>(p.next_tokens)[out] = next;
    else
      static_cast<int*>(p.next_tokens)[out] = next == (int64_t)(int)next ? (int)next : -1;
  }
  for (int i = threadIdx.x; i < p.width; i += ACCEPT_THREADS) p.accepted[out * p.accepted_s0 + i] = i < count ? path[i] : -1;
  if (p.slots == nullptr) return;
  // the path's rows first, then the others', each in order: the path rises.  All are read before any is written: they may stand at
  // these entries.
  bool bad = false;
  for (int i = threadIdx.x; i < d.n; i += ACCEPT_THREADS) {
    const int64_t slot = load_slot(p.slots, p.slots_64, (int64_t)d.row + i);
    const bool ok = slot == (int64_t)(int32_t)slot;
    bad |= !ok;
    token[i] = ok ? (int32_t)slot : -1;
  }
  if (bad) flag_error(FT_DEV_BAD_KV_INDEX);
  __syncthreads();
  for (int i = threadIdx.x; i < d.n; i += ACCEPT_THREADS) {
    int before = 0;
    while (before < count && path[before] < i) ++before;
    const int to = before < count && path[before] == i ? before : count + i - before;
    const int64_t entry = d.entries + d.cached + to;
    if (entry < p.kv_entries_len) p.kv_entries[entry] = token[i];
  }
}

}  // namespace ft
