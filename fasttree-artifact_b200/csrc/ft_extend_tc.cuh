// Extend attention on the 5th-generation tensor cores: a CTA per SM walks its share of the plan's (item, KV head) tasks.
//
//   S_w[128 x TILE] = Q_w[128 x D] . K_tile^T      tcgen05.mma, A and B K-major
//   O_w[128 x D]   += P_w[128 x TILE] . V_tile     tcgen05.mma, A = P in tensor memory, B MN-major
//
// At head_dim 64 and 128 two streams w = 0, 1 run through the K/V tiles: two query tiles (128 packed rows of tokens x GQA
// group each) that share every K/V tile in shared memory, or one query tile whose even and odd K/V tiles are streams of
// their own, so that either way one stream's softmax runs beside the other's products.  At head_dim 256, where O alone is
// half of tensor memory, there is one stream, and the scores of a tile are computed beside the softmax of the one before.
//
// Roles (warps): one softmax warpgroup per stream (thread = query row = TMEM lane), then one warp each for the MMA issue,
// K loads, V loads, and the tiles' row ids and Q loads.  All of them walk the same task list on their own; mbarriers (full / empty per buffer) are
// the only hand-offs, and the counters behind their phases run on from task to task, so the next task's Q and K are loaded
// and its first scores computed while the last rows of the task before are normalised and stored.  Every wait is bounded
// and unwinds the CTA through a state word.
//
// A K/V tile whose rows are consecutive in the pool is one TMA box per 64 columns; any other is gathered four rows at a
// time through the TMA unit, its last rows with 16-byte copies.  Rows of V behind the last token are zeroed up to the next
// 16, where the product ends; rows of K are not: their scores are masked.  Row ids outside the pool become zeros; the K loader notes
// the task, and what such keys of score 0 have put into a row's sum is taken out of it at the task's end (a check of every tile instead
// costs all calls 1 to 8 %).
//
// Softmax: a thread reads its row of S, masks what the row does not see (bits from the plan; a tile that all of the query tile's
// rows see whole has none), keeps a running maximum that may lag by 2^8 before O is rescaled in
// tensor memory, and writes P in the storage type; the row's sum is of the unrounded probabilities in fp32.  P takes the
// place of S, except at head_dim 64, where the products have different shapes and their order is not the order of issue:
// there P has columns of its own, and a stream's next scores are computed as soon as the ones before are in registers (2048 on
// 2048 tokens, 32/4 heads of 64: 101 -> 94 us).  At head_dim 128 a stream's scores are ready only when its earlier products are
// done (tcgen05.commit covers every MMA issued before it), so nothing is waited for before O is rescaled; at 64 and 256 there is
// a barrier for that.
//
// What bounds it: at head_dim 128 the chain scores -> softmax -> product of a stream, which the other stream hides but for a
// third (the tensor pipe is busy 55 % of an SM's active cycles in 2048 on 2048 tokens), and power: 4096 tokens behind 12288
// cached ones, 64/8 heads, bf16, 1710 us = 1125 TFLOP/s run on end, 0.81 of what a large library product settles at; 1486 us =
// 1295 in short runs; 2048 on 2048, 32/4 heads 109 us = 950.  At 64 the exponentials, 16 a clock and SM, at 63 % of the active
// cycles: 94 us = 548 TFLOP/s for the same (the two softmax warps of a scheduler taking turns at them: 111 for 94).  At 256 the products,
// whose 64-column shapes read shared memory more often than they multiply: 254 us = 811 TFLOP/s.  Few tokens: the K/V rows' way from
// memory, 4.0 to 4.6 TB/s where each request has a cache of its own, and below about 30 us the chain of dependent reads at the
// start (schedule, tile record, row ids, first tile) and the merge's launch.  Scattered pools: the TMA unit's row gathers, about
// 27 ns for four rows of 128 bytes and SM (sixteen prompts 332 us, with consecutive rows 297); 16-byte copies beside or instead
// of them were slower in every mixture (half of the rows 375).
//
// Rows of V that a query does not see are multiplied by P = 0, and 0 x Inf is NaN: a row that is not shown everything and did
// not come out finite is computed again from its own tokens (extend_row).
#pragma once

#include "ft_extend.cuh"
#include "ft_stage1_tc.cuh"

namespace ft {

struct alignas(64) ExtendTcParams {
  CUtensorMap k_map;       // [rows, kv heads, head_dim], box 64 x 1 x TILE
  CUtensorMap v_map;
  CUtensorMap k_rows_map;  // [rows, all heads' elements], box 64 x 1, for gathers
  CUtensorMap v_rows_map;
  CUtensorMap q_map;       // [q rows, heads, head_dim], box 64 x G x 1 (at most 8 heads where G is a multiple of 8)
  CUtensorMap q_map_tile;  // box 64 x G x 128 / G
  ExtendParams p;
  int has_tma, has_gather4, q_box_heads;
};

template <int D_>
struct ExtCfg {
  static constexpr int D = D_;
  static constexpr int NW = D <= 128 ? 2 : 1;       // streams
  static constexpr int TILE = D <= 128 ? 128 : 64;  // tokens of a K/V tile
  static constexpr int NB = D / 64;                 // 64-element column blocks of an operand row
  static constexpr int THREADS = 128 * NW + 128;
  static constexpr int Q_BYTES = NB * 16384;        // one query tile
  static constexpr int KV_BLOCK = TILE * 128;       // one column block of a K/V tile
  static constexpr int KV_BYTES = NB * KV_BLOCK;
  static constexpr int NSK = D == 64 ? 5 : D == 128 ? 2 : 3, NSV = D == 64 ? 5 : D == 128 ? 3 : 2;
  static constexpr int Q_OFF = 0, K_OFF = NW * Q_BYTES, V_OFF = K_OFF + NSK * KV_BYTES;
  static constexpr int NSI = 4;                           // tiles whose row ids are known or under way
  static constexpr int IDS_OFF = V_OFF + NSV * KV_BYTES;  // NSI x {TILE row ids}, then NSI x {tokens, KV head, task, 0}
  static constexpr int META_OFF = IDS_OFF + NSI * TILE * 4;
  static constexpr int BAD_OFF = META_OFF + NSI * 16;     // first and last task with a row id outside the pool
  static constexpr int BAR_OFF = BAD_OFF + 8;
  static constexpr int K_FULL = 0, K_EMPTY = K_FULL + NSK, V_FULL = K_EMPTY + NSK, V_EMPTY = V_FULL + NSV, S_FULL = V_EMPTY + NSV,
                       P_HALF = S_FULL + 2, P_FULL = P_HALF + 2, O_FULL = P_FULL + 2, PV_DONE = O_FULL + 2, S_READ = PV_DONE + 2, Q_FULL = S_READ + 2, Q_EMPTY = Q_FULL + 1,
                       IDS_FULL = Q_EMPTY + 1, IDS_EMPTY = IDS_FULL + NSI, NBARS = IDS_EMPTY + NSI;
  static constexpr int STATE_OFF = BAR_OFF + NBARS * 8, TMEM_SLOT_OFF = STATE_OFF + 4, SMEM_BYTES = TMEM_SLOT_OFF + 4;
  // tensor memory columns.  Two streams: S_w, then O_w, then (head_dim 64) P_w.  One: two S buffers, O.
  static constexpr int S_COL = 0, O_COL = 256, P_COL = D == 64 ? 384 : S_COL;
  static constexpr int S_STEP = NW == 2 ? 128 : 64, P_STEP = D == 64 ? 64 : S_STEP;
  static constexpr bool EARLY = D == 64;            // scores of a stream's next tile as soon as those before are read: P is elsewhere
  static constexpr int PV_N = D == 128 ? 128 : 64;  // columns of O per product
  static constexpr int CPR = D / 8;                 // 16-byte chunks of a row
  static constexpr int REGS_SOFTMAX = 224, REGS_OTHER = 56, REGS_LAUNCH = 168;
  static_assert(SMEM_BYTES <= 232448, "one CTA must fit in one SM's shared memory");
  static_assert(NW != 2 || (2 * REGS_SOFTMAX + REGS_OTHER) * 128 <= REGS_LAUNCH * THREADS, "register trade must balance");
};

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// One lane of the (whole) warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(one));
  return one != 0;
}

__device__ __forceinline__ int lds_int(uint32_t addr) {
  int x;
  asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(x) : "r"(addr) : "memory");
  return x;
}

__device__ __forceinline__ int2 lds_int2(uint32_t addr) {
  int2 x;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];\n" : "=r"(x.x), "=r"(x.y) : "r"(addr) : "memory");
  return x;
}

// Operand descriptors as two words: the low one holds the address and the leading offset, the high one the stride of 8 rows (1024
// bytes), the version and the 128-byte swizzle, which are the same for every operand here.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo_bytes) { return ((addr >> 4) & 0x3fffu) | ((lbo_bytes >> 4) << 16); }
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);

__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(acc), "r"(DESC_HI)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(acc), "r"(DESC_HI)
      : "memory");
}

// A CTA's state word: negative once a role has given up, else the count of its steps: K/V tiles whose row ids were sent for, and tiles
// of rows that are computed again one by one.
__device__ __forceinline__ int ext_state(uint32_t state) {
  int x;
  asm volatile("ld.volatile.shared.b32 %0, [%1];\n" : "=r"(x) : "r"(state) : "memory");
  return x;
}
__device__ __forceinline__ bool ext_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return __all_sync(0xffffffffu, ok != 0);
}

// Probes of mbarrier.try_wait before a wait gives up, about 4 us each where nothing comes: 0.26 s.
constexpr int EXT_WAIT_LIMIT = 1 << 16;

// Bounded wait of a whole warp for the phase of `bar` with the given parity, with one answer for its lanes: false after `limit` probes
// without a step of the CTA, or once another role has given up.  A stream may have nothing to do for many long tasks, and others wait
// for rows computed again, so the time alone does not tell a long wait from one that nothing will end.
// The form counts: the first probe stands apart because most waits end with it, and the warp's vote keeps its lanes together (2048 on
// 2048 tokens at head_dim 256: 255 us; a loop that each lane left by itself, with a look at the state in every sixteenth probe, 283).
__device__ __forceinline__ bool ext_wait(uint32_t bar, uint32_t parity, uint32_t state, int limit = EXT_WAIT_LIMIT) {
  if (ext_try(bar, parity)) return true;
  int seen = 0, left = limit;
#pragma unroll 1
  while (true) {
    if (ext_try(bar, parity)) return true;
    const int now = ext_state(state);
    left = __any_sync(0xffffffffu, now != seen) ? limit : left - 1;
    seen = now;
    if (__any_sync(0xffffffffu, now < 0) || left <= 0) return false;
  }
}

// Capped scores: tanh(x), x = S scale / cap, which the softmax multiplies by cap log2(e).
//
// Up to |x| = 1 by tanh(x) = x (1 + x^2 r(x^2)), r of six coefficients fitted with the Remez exchange for the smallest relative
// error: 6e-8, about fp32's half step, so a cap far above the scores changes nothing near 0.  The coefficients are those of x and
// stay normal numbers whatever scale and cap are: with the powers of scale / cap multiplied into them, which saves one
// multiplication in nine, the thirteenth is 0 from about scale / cap = 8e-4 on (sm_scale 1/128, cap 30: scores off by 0.3).
// Two tanh or one exponential more per score on the special-function unit, which the softmax already keeps busy, cost more than
// nine packed FMAs for two scores.
// Larger |x|: tanh(x) = 1 - 2 / (1 + e^(2 x)), one reciprocal for two scores, for every 32 columns in which the warp has such a score.
// Which of the two a score takes goes by that score alone, so what stands in a tile beside the scores in sight (rows of K that
// nobody wrote among them) is never seen in a result.
// 2048 on 2048 tokens, 32/4 heads of 128: not capped 109 us; capped 169, where most columns have a score beyond the cap 272.
struct Capped {
  static constexpr float LOG2E = 1.4426950408889634f, MOST = 1.f;
  float k, c2;
  // (limits that keep k and c2 finite; a cap of 1e36 hides nothing from fp32 that 1e38 would show)
  __device__ __forceinline__ Capped(float scale, float cap) {
    cap = fminf(cap, 1e36f);
    k = fminf(scale / cap, 1e36f);
    c2 = cap * LOG2E;
  }
  __device__ __forceinline__ static float2 fit(float2 x, float2 u) {
    constexpr float q[6] = {-0.33332987f, 0.13326409f, -0.053498708f, 0.02035976f, -0.0062593398f, 0.0010582648f};
    float2 y = make_float2(q[5], q[5]);
#pragma unroll
    for (int j = 4; j >= 0; --j) y = __ffma2_rn(y, u, make_float2(q[j], q[j]));
    return __fmul2_rn(__ffma2_rn(y, u, make_float2(1.f, 1.f)), x);
  }
  // tanh(k s) in place, right up to MOST; the largest x^2 of every 32 scores
  template <int N>
  __device__ __forceinline__ void apply(float (&s)[N], float (&most)[N / 32]) const {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 x = __fmul2_rn(make_float2(s[2 * i], s[2 * i + 1]), make_float2(k, k)), u = __fmul2_rn(x, x);
      if (i % 16 == 0)
        most[i / 16] = fmaxf(u.x, u.y);
      else
        asm("max.f32 %0, %0, %1, %2;" : "+f"(most[i / 16]) : "f"(u.x), "f"(u.y));
      const float2 y = fit(x, u);
      s[2 * i] = y.x;
      s[2 * i + 1] = y.y;
    }
  }
  // what apply() left of the scores z beyond MOST
  __device__ __forceinline__ void large(float* s, const float (&z)[32]) const {
    const float2 one = make_float2(1.f, 1.f);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      // (2^60 and above is as good as infinite: 1 + 2^60 squared still is a number; a NaN becomes one here, and keeps to itself)
      const float2 x = __fmul2_rn(make_float2(z[2 * i], z[2 * i + 1]), make_float2(k, k));
      float2 y = __fmul2_rn(x, make_float2(2.f * LOG2E, 2.f * LOG2E));
      y = __fadd2_rn(make_float2(fast_exp2(fminf(y.x, 60.f)), fast_exp2(fminf(y.y, 60.f))), one);
      float r;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y.x * y.y));
      y = __ffma2_rn(__fmul2_rn(make_float2(r, r), make_float2(y.y, y.x)), make_float2(-2.f, -2.f), one);
      s[2 * i] = fabsf(x.x) > MOST ? y.x : s[2 * i];
      s[2 * i + 1] = fabsf(x.y) > MOST ? y.y : s[2 * i + 1];
    }
  }
};

template <typename T, int D, bool CAP>
__global__ void __launch_bounds__(ExtCfg<D>::THREADS, 1) extend_tc_kernel(const __grid_constant__ ExtendTcParams tp) {
  using C = ExtCfg<D>;
  constexpr int TILE = C::TILE, NB = C::NB, NW = C::NW;
  extern __shared__ __align__(1024) uint8_t smem[];
  const ExtendParams& p = tp.p;
  const uint32_t sm = smem_u32(smem), bars = sm + C::BAR_OFF;
  const uint32_t state = sm + C::STATE_OFF;
  auto set_state = [&](int x) { asm volatile("st.volatile.shared.b32 [%0], %1;\n" ::"r"(state), "r"(x) : "memory"); };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + C::TMEM_SLOT_OFF);
  auto bar = [&](int i) { return bars + 8u * i; };
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  allow_dependent_launch();
  wait_for_prior_grid();
  const int4* my_share = reinterpret_cast<const int4*>(p.sms) + 4 * blockIdx.x;
  const int4 share = __ldg(my_share);
  const int task_lo = share.x, task_hi = share.y;
  if (task_lo >= task_hi) return;
  if ((sm & 1023u) != 0u) {  // the swizzled operand layout needs a 1024-byte aligned window
    if (tid == 0) flag_error(FT_DEV_WAIT_TIMEOUT);
    return;
  }
  if (tid == C::THREADS - 32) {  // the first copies would otherwise pay for fetching their descriptors
    const CUtensorMap* maps[] = {&tp.k_map, &tp.v_map, &tp.q_map, &tp.q_map_tile, &tp.k_rows_map, &tp.v_rows_map};
#pragma unroll
    for (int i = 0; i < 6; ++i) asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(maps[i])) : "memory");
  }
  if (tid == 0) {
    for (int b = 0; b < C::NSK; ++b) {
      mbar_init(bar(C::K_FULL + b), 32);
      mbar_init(bar(C::K_EMPTY + b), 1);
    }
    for (int b = 0; b < C::NSV; ++b) {
      mbar_init(bar(C::V_FULL + b), 32);
      mbar_init(bar(C::V_EMPTY + b), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar(C::S_FULL + b), 1);
      mbar_init(bar(C::P_HALF + b), 128);
      mbar_init(bar(C::P_FULL + b), 128);
      mbar_init(bar(C::O_FULL + b), 1);
      mbar_init(bar(C::PV_DONE + b), 1);
      mbar_init(bar(C::S_READ + b), 128);
    }
    mbar_init(bar(C::Q_FULL), 1);
    mbar_init(bar(C::Q_EMPTY), 1);
    for (int b = 0; b < C::NSI; ++b) {
      mbar_init(bar(C::IDS_FULL + b), 33);  // the copies of 32 lanes, and what lane 0 writes beside them
      mbar_init(bar(C::IDS_EMPTY + b), 2);  // both loaders
    }
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};\n" ::"r"(sm + C::BAD_OFF), "r"(0x7fffffff), "r"(-1) : "memory");
    set_state(0);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(sm + C::TMEM_SLOT_OFF), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  // the end of the set-up, which every role passes once, before it waits for or touches anything that was set up
  auto set_up = [&]() {
    tc_fence_before();
    asm volatile("bar.sync 0;\n" ::: "memory");
    tc_fence_after();
    return *tmem_slot;
  };
  const int G = p.group;
  bool dead = false;
  auto give_up = [&]() {
    set_state(INT_MIN);
    flag_error(FT_DEV_WAIT_TIMEOUT);
    dead = true;
  };
  auto item_of = [&](int n, int& kvh) {
    const int task = n == task_lo ? share.z : __ldg(p.sm_tasks + n);
    kvh = task % p.kv_heads;
    return p.items + (int64_t)EXT_ITEM_INTS * (task / p.kv_heads);
  };

  if (warp < 4 * NW) {
    const uint32_t tmem = set_up();
    // ====================================================================== softmax, one query row per thread
    if constexpr (NW == 2) reg_grow<C::REGS_SOFTMAX>();
    const int w = warp >> 2, row = tid & 127;
    const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t o_col = t_lane + C::O_COL + w * D;
    const float scale = p.sm_scale == 0.f ? 1.17549435e-38f : fabsf(p.sm_scale);
    constexpr float LOG2E = 1.4426950408889634f;
    const Capped capped = CAP ? Capped(scale, p.logit_cap) : Capped(0.f, 1.f);
    // scores in powers of two: scale2 x S, or x what Capped makes of S
    const float scale2 = CAP ? capped.c2 : scale * LOG2E;
    int tiles_done = 0, items_done = 0;
    for (int n = task_lo; n < task_hi && !dead; ++n) {
      int lo, hi, step, rows;    // of the stream: K/V tiles lo, lo + step, ... below hi, rows of the query tile
      const int32_t* mask_of;    // per K/V tile, every eighth int: where its bits are, or -1
      const int32_t* bits = nullptr;  // of this row's token
      {
        int kvh;
        const int32_t* item = item_of(n, kvh);
        const ExtendStream st = extend_stream(item, w);
        lo = st.lo;
        hi = st.hi;
        rows = st.ntok * G;
        step = __ldg(item + 2);
        mask_of = p.tiles + 8 * (int64_t)__ldg(item + 5) + 4 + st.block_tile;
        bits = p.extra + (st.first + (row < rows ? row / G : 0)) * (TILE / 32);
      }
      if (rows == 0) continue;
      const bool warp_live = (row & ~31) < rows;
      float m_used = -INFINITY, l_run = 0.f;
      bool hidden = false;  // this row was shown less than all of its tiles
      uint32_t see[TILE / 32];
      bool any = true;
      auto tile = [&](auto masked, const int t) {
        constexpr bool MASKED = decltype(masked)::value;
        const int buf = NW == 2 ? w : tiles_done & 1;
        const uint32_t phase = NW == 2 ? (uint32_t)tiles_done & 1u : (uint32_t)(tiles_done >> 1) & 1u;
        ++tiles_done;
        const uint32_t s_col = t_lane + C::S_COL + buf * C::S_STEP, p_col = t_lane + C::P_COL + buf * C::P_STEP;
        // (one answer for the warp: it goes on, or gives up, as a whole)
        if (!ext_wait(bar(C::S_FULL + buf), phase, state)) {
          give_up();
          return;
        }
        tc_fence_after();
        // P's columns, and O if it is rescaled: the product with V of the stream's tile before has to be done with them
        auto wait_pv = [&]() {
          const int before = tiles_done - 2, b = NW == 2 ? w : before & 1;
          const uint32_t ph = NW == 2 ? (uint32_t)before & 1u : (uint32_t)(before >> 1) & 1u;
          if (before >= 0 && !ext_wait(bar(C::PV_DONE + b), ph, state)) give_up();
          tc_fence_after();
        };
        if (MASKED && !__any_sync(0xffffffffu, any)) {  // nothing in sight of the warp's rows
          if constexpr (C::EARLY) {
            mbar_arrive(bar(C::S_READ + buf));
            wait_pv();
          }
          if (warp_live) {
            float zero[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) zero[c] = 0.f;
#pragma unroll
            for (int c = 0; c < TILE / 64; ++c) tmem_st32(p_col + 32 * c, zero);
            tmem_wait_st();
          }
          tc_fence_before();
          mbar_arrive(bar(C::P_HALF + buf));
          mbar_arrive(bar(C::P_FULL + buf));
          return;
        }
        float s[TILE];
#pragma unroll
        for (int c = 0; c < TILE / 32; ++c) tmem_ld32_nowait(s_col + 32 * c, *reinterpret_cast<float(*)[32]>(&s[32 * c]));
        tmem_wait_ld();
        if constexpr (CAP) {
          float most[TILE / 32];
          capped.apply(s, most);
          auto beyond = [&](float x) { return __any_sync(0xffffffffu, row < rows && x > Capped::MOST * Capped::MOST); };
          if (beyond(TILE == 128 ? fmaxf(fmaxf(most[0], most[1]), fmaxf(most[TILE / 32 - 2], most[TILE / 32 - 1])) : fmaxf(most[0], most[1]))) {
#pragma unroll
            for (int c = 0; c < TILE / 32; ++c)
              if (beyond(most[c])) {
                float z[32];
                tmem_ld32(s_col + 32 * c, z);
                capped.large(s + 32 * c, z);
              }
          }
        }
        if constexpr (C::EARLY) {
          tc_fence_before();
          mbar_arrive(bar(C::S_READ + buf));
        }
        if constexpr (MASKED) {
#pragma unroll
          for (int k = 0; k < TILE / 32; ++k)
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if ((see[k] & (1u << c)) == 0) s[32 * k + c] = -INFINITY;
        }
        float mx4[4] = {fmaxf(s[0], s[1]), fmaxf(s[2], s[3]), fmaxf(s[4], s[5]), fmaxf(s[6], s[7])};
#pragma unroll
        for (int c = 8; c < TILE; c += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k) asm("max.f32 %0, %0, %1, %2;" : "+f"(mx4[k]) : "f"(s[c + 2 * k]), "f"(s[c + 2 * k + 1]));
        float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        mx *= scale2;
        float corr = 1.f;
        bool grow = false;
        if (mx > m_used + 8.f || m_used == -INFINITY) {  // the offset may lag the true maximum by up to 2^8
          if (mx > -INFINITY) {
            grow = m_used > -INFINITY;
            corr = fast_exp2(m_used - mx);  // 0 at the row's first tokens
            m_used = mx;
          }
        }
        l_run *= corr;
        const float neg_off = m_used == -INFINITY ? 0.f : -m_used;
        const float2 sc2 = make_float2(scale2, scale2), no2 = make_float2(neg_off, neg_off);
        float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        // P, in halves: the first is handed over while the second is made
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t wds[TILE / 4];
#pragma unroll
          for (int i = 0; i < TILE / 4; ++i) {
            float2 x = make_float2(s[h * (TILE / 2) + 2 * i], s[h * (TILE / 2) + 2 * i + 1]);
            x = __ffma2_rn(x, sc2, no2);
            x.x = fast_exp2(x.x);
            x.y = fast_exp2(x.y);
            sum2[i & 1] = __fadd2_rn(sum2[i & 1], x);
            wds[i] = pack2<T>(x.x, x.y);
          }
          if (C::EARLY && h == 0) wait_pv();
          if constexpr (TILE == 128)
            tmem_st32(p_col + 32 * h, *reinterpret_cast<float(*)[32]>(&wds[0]));
          else
            tmem_st16(p_col + 16 * h, *reinterpret_cast<uint32_t(*)[16]>(&wds[0]));
          if (h == 0 && t > lo && __any_sync(0xffffffffu, grow)) {
            if constexpr (NW == 1) wait_pv();
#pragma unroll
            for (int cb = 0; cb < D / 32; ++cb) {
              float o[32];
              tmem_ld32(o_col + cb * 32, o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] *= corr;
              tmem_st32(o_col + cb * 32, o);
            }
          }
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(bar((h == 1 ? C::P_FULL : C::P_HALF) + buf));
        }
        l_run += (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
      };
      // Two loops, so that the one over tiles that every row sees whole has no masks in it: with one loop the scores do not all fit
      // the registers (4096 tokens behind 12288, 64/8 heads: 1910 us, with two 1620).  Where the next tile's bits are is read a
      // tile ahead.
      auto mask_at = [&](int t) { return t < hi ? __ldg(mask_of + 8 * t) : -1; };
      int mask = mask_at(lo);
      for (int t = lo; t < hi && !dead;) {
        while (mask < 0 && t < hi && !dead) {
          mask = mask_at(t + step);
          tile(std::false_type{}, t);
          t += step;
        }
        if (t >= hi || dead) break;
        uint32_t some = 0, every = 0xffffffffu;
#pragma unroll
        for (int k = 0; k < TILE / 32; ++k) {
          see[k] = row < rows ? (uint32_t)__ldg(bits + mask + k) : 0u;
          some |= see[k];
          every &= see[k];
        }
        any = some != 0;
        hidden |= every != 0xffffffffu;
        mask = mask_at(t + step);
        tile(std::true_type{}, t);
        t += step;
      }
      if (dead) break;
      // ---- the row's result: normalised, to o or to its partial row
      if (!ext_wait(bar(C::O_FULL + w), (uint32_t)items_done & 1u, state)) {
        give_up();
        break;
      }
      ++items_done;
      tc_fence_after();
      if (!warp_live) continue;
      int kvh;
      const int32_t* item = item_of(n, kvh);
      const ExtendStream st = extend_stream(item, w);
      const bool live = row < rows;
      const int tok = live ? row / G : 0, head = kvh * G + (live ? row - tok * G : 0);
      const int2 tk = __ldg(reinterpret_cast<const int2*>(p.tokens) + st.tok0 + tok);
      const int part = live ? extend_part(p, st, tok) : -2;
      const bool store = part != -2 && tk.x >= 0 && tk.x < p.q_rows;
      if (part != -2 && !store) flag_error(FT_DEV_BAD_Q_INDEX);
      // Row ids outside the pool were zeros: keys of score 0 and no value, which nothing but the row's sum has met.  What they put
      // there is taken out, if the offset is a real key's (then P has its full precision) and enough of the sum is left.
      // (The K loader notes the task before it hands the tile over; the tasks between the first and the last are looked at too.)
      bool again = false;
      const int2 bad = lds_int2(sm + C::BAD_OFF);
      if (n >= bad.x && n <= bad.y) {
        const int in_sight = extend_bad_in_sight(p, item, st, tok, state);
        if (in_sight > 0) {
          const float rest = l_run - (float)in_sight * fast_exp2(-m_used);
          again = !(m_used > 0.f && rest >= 0.015625f * l_run);
          l_run = rest;
        }
      }
      const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
      float2 finite = make_float2(0.f, 0.f);  // 0 x every element: 0, or NaN
      uint8_t* dst = nullptr;
      if (store)
        dst = part >= 0 ? reinterpret_cast<uint8_t*>(p.mid_o + ((int64_t)part * p.heads + head) * D)
                           : reinterpret_cast<uint8_t*>(reinterpret_cast<T*>(p.o) + (int64_t)tk.x * p.o_s0 + (int64_t)head * p.o_s1);
      auto load_32 = [&](int cb, float (&o)[32]) {
        tmem_ld32(o_col + cb * 32, o);
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const float2 x = __fmul2_rn(make_float2(o[2 * c], o[2 * c + 1]), make_float2(inv, inv));
          finite = __ffma2_rn(x, make_float2(0.f, 0.f), finite);
          o[2 * c] = x.x;
          o[2 * c + 1] = x.y;
        }
      };
#pragma unroll
      for (int cb = 0; cb < D / 32; ++cb) {
        float o[32];
        load_32(cb, o);
        if (dst != nullptr) {
          if (st.part >= 0) {
#pragma unroll
            for (int c = 0; c < 8; ++c)
              reinterpret_cast<float4*>(dst + cb * 128)[c] = make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
          } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
              reinterpret_cast<uint4*>(dst + cb * 64)[c] = make_uint4(pack2<T>(o[8 * c], o[8 * c + 1]), pack2<T>(o[8 * c + 2], o[8 * c + 3]),
                                                                     pack2<T>(o[8 * c + 4], o[8 * c + 5]), pack2<T>(o[8 * c + 6], o[8 * c + 7]));
          }
        }
      }
      if (store)
        extend_store_lse(p, part, tk.x, head, l_run == 0.f ? -INFINITY : (m_used + log2f(l_run)) * 0.6931471805599453f);
      const bool spoiled = store && (again || (hidden && !(finite.x + finite.y == 0.f)));
      for (uint32_t todo = __ballot_sync(0xffffffffu, spoiled); todo != 0; todo &= todo - 1) {
        const int r = (row & ~31) + __ffs(todo) - 1;
        __syncwarp();
        extend_row<T>(p, item, st, r / G, kvh * G + r % G, state);
      }
    }
  } else {
    if constexpr (NW == 2) reg_shrink<C::REGS_OTHER>();
    const int role = warp - 4 * NW;
    if (role == 0) {
      const uint32_t tmem = set_up();
      // ==================================================================== MMA issue
      // The whole warp walks the loop, on values that are the same in every lane (broadcast where they come from memory), so that
      // the operands of an MMA stand in uniform registers; one lane issues.  With a loop for one lane alone, every MMA waits
      // for its operands' way into uniform registers: 120 cycles an MMA that takes 64 (4096 tokens behind 12288, 64/8 heads:
      // 1980 -> 1590 us).
      const uint32_t idesc_s = tc_idesc<T>(128, TILE, false, p.sm_scale < 0.f), idesc_o = tc_idesc<T>(128, C::PV_N, true);
      const uint32_t bars_u = __shfl_sync(0xffffffffu, bars, 0), sm_u = __shfl_sync(0xffffffffu, sm, 0), tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
      const bool issuer = elect_one();
      auto ubar = [&](int i) { return bars_u + 8u * (uint32_t)i; };
      auto wait = [&](uint32_t b, uint32_t phase) {
        if (!ext_wait(b, phase, state)) give_up();
      };
      // (Loops are kept short on purpose: the roles run at the same time from one instruction cache.)
      int k_stage = 0, v_stage = 0;
      uint32_t k_phase = 0, v_phase = 0, q_phase = 0, p_phases = 0;  // p_phases: a bit per P buffer
      int s_count = 0;        // score tiles issued (one stream)
      uint32_t s_phases = 0;  // a bit per stream
      const int tasks_u = __shfl_sync(0xffffffffu, task_hi - task_lo, 0);
      for (int n = 0; n < tasks_u && !dead; ++n) {
        int t0, t1, step, len, lo0, hi0, lo1 = 0, hi1 = 0, tile1 = 0;
        {
          int kvh;
          const int32_t* item = item_of(task_lo + n, kvh);
          t0 = __shfl_sync(0xffffffffu, __ldg(item), 0);
          t1 = __shfl_sync(0xffffffffu, __ldg(item + 1), 0);
          step = __shfl_sync(0xffffffffu, __ldg(item + 2), 0);
          len = __shfl_sync(0xffffffffu, __ldg(item + 4), 0);
          const ExtendStream a = extend_stream(item, 0);
          lo0 = __shfl_sync(0xffffffffu, a.lo, 0);
          hi0 = __shfl_sync(0xffffffffu, a.hi, 0);
          if constexpr (NW == 2) {
            const ExtendStream b = extend_stream(item, 1);
            lo1 = __shfl_sync(0xffffffffu, b.lo, 0);
            hi1 = __shfl_sync(0xffffffffu, b.hi, 0);
            tile1 = __shfl_sync(0xffffffffu, b.q_tile, 0);
          }
        }
        wait(ubar(C::Q_FULL), q_phase);
        q_phase ^= 1u;
        if (dead) break;
        bool k_here = false, v_here = false;
        auto wait_k = [&]() {
          if (!k_here) wait(ubar(C::K_FULL + k_stage), k_phase);
          k_here = true;
        };
        auto wait_v = [&]() {
          if (!v_here) wait(ubar(C::V_FULL + v_stage), v_phase);
          v_here = true;
        };
        auto issue_qk = [&](int buf, int tile) {
          wait_k();
          if (dead) return;
          proxy_fence();
          tc_fence_after();
          uint32_t a = desc_lo(sm_u + C::Q_OFF + tile * C::Q_BYTES, 16), b = desc_lo(sm_u + C::K_OFF + k_stage * C::KV_BYTES, 16);
          const uint32_t d = tmem_u + C::S_COL + buf * C::S_STEP;
          if (issuer) {
#pragma unroll
            for (int blk = 0; blk < NB; ++blk) {  // k-steps of 16 along head_dim: +32 B inside a block, +1 block after 4
#pragma unroll
              for (int ks = 0; ks < 4; ++ks) mma_ss(d, a + ks * 2, b + ks * 2, idesc_s, (uint32_t)(blk | ks));
              a += 16384 >> 4;
              b += C::KV_BLOCK >> 4;
            }
            tc_commit(ubar(C::S_FULL + buf));
          }
          __syncwarp();
        };
        auto issue_pv = [&](int w, int buf, int t, bool first, bool last) {
          const uint32_t a = tmem_u + C::P_COL + buf * C::P_STEP, b = desc_lo(sm_u + C::V_OFF + v_stage * C::KV_BYTES, C::KV_BLOCK);
          const uint32_t d = tmem_u + C::O_COL + w * D;
          const int ksteps = min(TILE, len - t * TILE + 15) >> 4;  // the rows of V behind the next 16 are not defined
          constexpr int HALF = TILE / 32;                          // k-steps of 16 tokens in half a tile
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            wait(ubar((half == 0 ? C::P_HALF : C::P_FULL) + buf), (p_phases >> buf) & 1u);
            if (half == 0 && !dead) wait_v();
            if (dead) return;
            proxy_fence();
            tc_fence_after();
            if (issuer) {
#pragma unroll
              for (int h = 0; h < D / C::PV_N; ++h) {
                const uint32_t ah = a + half * (HALF * 8), bh = b + h * (C::KV_BLOCK >> 4) + half * (HALF * 128);
                if (ksteps >= (half + 1) * HALF) {
#pragma unroll
                  for (int ks = 0; ks < HALF; ++ks)
                    mma_ts(d + h * C::PV_N, ah + ks * 8, bh + ks * 128, idesc_o, !first || half + ks > 0 ? 1u : 0u);
                } else {
#pragma unroll 1
                  for (int ks = 0; ks < ksteps - half * HALF; ++ks)
                    mma_ts(d + h * C::PV_N, ah + ks * 8, bh + ks * 128, idesc_o, !first || half + ks > 0 ? 1u : 0u);
                }
              }
              if (half == 1) {
                if (NW == 1 || C::EARLY) tc_commit(ubar(C::PV_DONE + buf));
                if (last) tc_commit(ubar(C::O_FULL + w));
              }
            }
            __syncwarp();
          }
          p_phases ^= 1u << buf;
        };
        auto release_k = [&]() {
          wait_k();
          if (dead) return;
          if (issuer) tc_commit(ubar(C::K_EMPTY + k_stage));
          if (++k_stage == C::NSK) {
            k_stage = 0;
            k_phase ^= 1u;
          }
          k_here = false;
        };
        auto release_v = [&]() {
          wait_v();
          if (dead) return;
          if (issuer) tc_commit(ubar(C::V_EMPTY + v_stage));
          if (++v_stage == C::NSV) {
            v_stage = 0;
            v_phase ^= 1u;
          }
          v_here = false;
        };
        if constexpr (C::EARLY) {
          // iteration t: the scores of tile t for both streams, then the products with V of tile t - step
#pragma unroll 1
          for (int t = t0; t < t1 + step && !dead; ++t) {
            const int before = t - step;
#pragma unroll 1
            for (int w = 0; w < 2 && !dead; ++w) {
              const int lo = w == 0 ? lo0 : lo1, hi = w == 0 ? hi0 : hi1;
              if (t < lo || t >= hi || (step == 2 && ((t - lo) & 1) != 0)) continue;
              wait(ubar(C::S_READ + w), ((s_phases >> w) & 1u) ^ 1u);
              s_phases ^= 1u << w;
              if (!dead) issue_qk(w, w == 0 ? 0 : tile1);
            }
            if (t < t1 && !dead) release_k();
            if (t == t1 - 1 && !dead && issuer) tc_commit(ubar(C::Q_EMPTY));
#pragma unroll 1
            for (int w = 0; w < 2 && !dead; ++w) {
              const int lo = w == 0 ? lo0 : lo1, hi = w == 0 ? hi0 : hi1;
              if (before < lo || before >= hi || (step == 2 && ((before - lo) & 1) != 0)) continue;
              issue_pv(w, w, before, before == lo, before + step >= hi);
            }
            if (before >= t0 && before < t1 && !dead) release_v();
          }
        } else if constexpr (NW == 2) {
          // iteration t: the products with V of tile t - step, then the scores of tile t, stream by stream
#pragma unroll 1
          for (int t = t0; t < t1 + step && !dead; ++t) {
            const int before = t - step;
#pragma unroll 1
            for (int w = 0; w < 2 && !dead; ++w) {
              const int lo = w == 0 ? lo0 : lo1, hi = w == 0 ? hi0 : hi1;
              if (step == 2 && ((t - lo) & 1) != 0) continue;  // (t and t - step are the same stream's)
              if (before >= lo && before < hi) issue_pv(w, w, before, before == lo, before + step >= hi);
              if (!dead && t >= lo && t < hi) issue_qk(w, w == 0 ? 0 : tile1);
            }
            if (dead) break;
            if (t < t1) release_k();
            if (t == t1 - 1 && !dead && issuer) tc_commit(ubar(C::Q_EMPTY));
            if (before >= t0 && before < t1 && !dead) release_v();
          }
        } else {
          // (buffers by the tile's number over all tasks: its parity is s_count's)
#pragma unroll 1
          for (int t = t0; t <= t1 && !dead; ++t) {
            if (t < t1) {
              issue_qk(s_count++ & 1, 0);
              if (!dead) release_k();
              if (t == t1 - 1 && !dead && issuer) tc_commit(ubar(C::Q_EMPTY));
            }
            if (t > t0 && !dead) {
              issue_pv(0, (s_count - (t < t1 ? 2 : 1)) & 1, t - 1, t - 1 == lo0, t == t1);
              if (!dead) release_v();
            }
          }
        }
      }
      __syncwarp();
    } else if (role <= 2) {
      // ==================================================================== K loads (role 1), V loads (role 2)
      const bool is_k = role == 1;
      const CUtensorMap* map = is_k ? &tp.k_map : &tp.v_map;
      const CUtensorMap* rows_map = is_k ? &tp.k_rows_map : &tp.v_rows_map;
      const int64_t s0 = is_k ? p.k_s0 : p.v_s0, s1 = is_k ? p.k_s1 : p.v_s1;
      const T* base0 = reinterpret_cast<const T*>(is_k ? p.k : p.v);
      const uint32_t full0 = bar(is_k ? C::K_FULL : C::V_FULL), empty0 = bar(is_k ? C::K_EMPTY : C::V_EMPTY);
      const uint32_t ring = sm + (is_k ? C::K_OFF : C::V_OFF);
      const int stages = is_k ? C::NSK : C::NSV;
      const uint32_t row_lim = (uint32_t)(p.kv_rows < 0x7fffffffLL ? p.kv_rows : 0x7fffffffLL);
      int stage = 0, slot = 0;
      uint32_t phase = 1, ids_phase = 0;
      set_up();
      while (true) {
        if (!ext_wait(bar(C::IDS_FULL + slot), ids_phase, state)) {
          give_up();
          break;
        }
        const uint32_t ids = sm + C::IDS_OFF + slot * (TILE * 4);
        int id[TILE / 32];
        const int2 meta = lds_int2(sm + C::META_OFF + slot * 16);
        const int valid = meta.x, kvh = meta.y;
        if (valid == 0) break;  // the end
        const int first = __shfl_sync(0xffffffffu, lds_int(ids), 0);
        bool dense = true, in_pool = true;
#pragma unroll
        for (int h = 0; h < TILE / 32; ++h) {
          id[h] = lds_int(ids + (lane + 32 * h) * 4);
          dense &= id[h] == first + lane + 32 * h;
          in_pool &= lane + 32 * h >= valid || (uint32_t)id[h] < row_lim;
        }
        in_pool = __all_sync(0xffffffffu, in_pool);
        dense = tp.has_tma && valid == TILE && in_pool && __all_sync(0xffffffffu, dense);
        if (!ext_wait(empty0 + 8u * stage, phase, state)) {
          give_up();
          break;
        }
        const uint32_t buf = ring + stage * C::KV_BYTES, full = full0 + 8u * stage;
        if (dense) {
          if (lane == 0) {
            mbar_arrive_expect_tx(full, C::KV_BYTES);
#pragma unroll
            for (int h = 0; h < NB; ++h) tma_load_3d(buf + h * C::KV_BLOCK, map, 64 * h, kvh, first, full);
          } else {
            mbar_arrive(full);
          }
        } else {
          int done = 0;
          if (tp.has_gather4 && in_pool) {
            done = valid & ~3;
            if (lane == 0 && done > 0) mbar_expect_tx(full, (uint32_t)done * (2u * D));
            __syncwarp();
#pragma unroll 1
            for (int i = lane; i < done / 4 * NB; i += 32) {
              const int blk = i % NB, r = i / NB * 4;
              int r0, r1, r2, r3;
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(ids + r * 4));
              tma_gather4(buf + blk * C::KV_BLOCK + r * 128, rows_map, kvh * (int)s1 + 64 * blk, r0, r1, r2, r3, full);
            }
          }
          // what is left, 16 bytes at a time; of V zeros up to the next 16 rows
          const T* base = base0 + (int64_t)kvh * s1;
          const int end = is_k ? valid : (valid + 15) & ~15, c16 = lane % C::CPR;
#pragma unroll 1
          for (int r = done + lane / C::CPR; r < end; r += 32 / C::CPR) {
            const int row_id = lds_int(ids + r * 4);
            const bool ok = r < valid && (uint32_t)row_id < row_lim;
            cp_async16_zfill(buf + (uint32_t)((c16 >> 3) * C::KV_BLOCK) + tc_swz(r, c16 & 7, 0), base + (int64_t)(ok ? row_id : 0) * s0 + c16 * 8, ok);
          }
          if (!in_pool && lane == 0) {
            if (is_k) {
              const int task = lds_int(sm + C::META_OFF + slot * 16 + 8), before = lds_int(sm + C::BAD_OFF);
              asm volatile("st.shared.v2.b32 [%0], {%1, %2};\n" ::"r"(sm + C::BAD_OFF), "r"(min(task, before)), "r"(task) : "memory");
              __threadfence_block();
            }
            flag_error(FT_DEV_BAD_KV_INDEX);
          }
          mbar_arrive_on_cp_async(full);
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(bar(C::IDS_EMPTY + slot));
        if (++slot == C::NSI) {
          slot = 0;
          ids_phase ^= 1u;
        }
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      cp_async_wait<0>();
    } else {
      // ==================================================================== row ids of the K/V tiles, Q loads
      // The ids of a tile go to a slot of a ring that both loaders read, NSI tiles ahead of them: a plain load that is sent off
      // beside a hundred kilobytes of tile copies comes back after them.  A task's first tiles come before its Q, for which
      // this warp may have to wait until the task before is through with its own.
      int slot = 0, items = 0;
      uint32_t ids_phase = 1;
      auto put_ids = [&](const int4 rec, int kvh, int task) {  // rec.z 0: the end
        if (!ext_wait(bar(C::IDS_EMPTY + slot), ids_phase, state)) {
          give_up();
          return;
        }
        const uint32_t ids = sm + C::IDS_OFF + slot * (TILE * 4);
#pragma unroll
        for (int h = 0; h < TILE / 32; ++h)
          if (lane + 32 * h < rec.z) cp_async4(ids + (lane + 32 * h) * 4, p.kv_entries + extend_entry(p, rec, lane + 32 * h));
        if (lane == 0) {
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %3};\n" ::"r"(sm + C::META_OFF + slot * 16), "r"(rec.z), "r"(kvh), "r"(task) : "memory");
          mbar_arrive(bar(C::IDS_FULL + slot));
          asm volatile("red.shared.add.u32 [%0], 1;\n" ::"r"(state) : "memory");
        }
        mbar_arrive_on_cp_async(bar(C::IDS_FULL + slot));
        if (++slot == C::NSI) {
          slot = 0;
          ids_phase ^= 1u;
        }
      };
      set_up();
      for (int n = task_lo; n < task_hi && !dead; ++n, ++items) {
        int kvh, t0, t1, tile0;
        int4 rec;
        const int32_t* item = item_of(n, kvh);
        if (n == task_lo) {
          const int4 head = __ldg(my_share + 1);
          t0 = head.x;
          t1 = head.y;
          tile0 = head.z;
          rec = __ldg(my_share + 2);
        } else {
          t0 = __ldg(item);
          t1 = __ldg(item + 1);
          tile0 = __ldg(item + 5);
          rec = __ldg(reinterpret_cast<const int4*>(item + 24));
        }
        int t = t0;
        auto put_until = [&](int end) {
#pragma unroll 1
          for (; t < end && !dead; ++t) {
            const int4 next = t + 1 < t1 ? __ldg(reinterpret_cast<const int4*>(p.tiles) + 2 * ((int64_t)tile0 + t + 1)) : rec;
            put_ids(rec, kvh, n);
            rec = next;
          }
        };
        put_until(min(t1, t0 + 2));
        if (dead) break;
        const int q_tiles = __ldg(item + 3);
        if (!ext_wait(bar(C::Q_EMPTY), ((uint32_t)items & 1u) ^ 1u, state)) {
          give_up();
          break;
        }
        // bytes first: a whole tile if its tokens' rows are consecutive, else a box per token
        uint32_t bytes = 0, in_order = 0;
#pragma unroll 1
        for (int w = 0; w < q_tiles; ++w) {
          const ExtendStream st = extend_stream(item, w);
          const int first = __ldg(p.tokens + 2 * st.tok0);
          bool mine = true;
          int rows = 0;
          for (int i = lane; i < st.ntok; i += 32) {
            const int r = __ldg(p.tokens + 2 * (st.tok0 + i));
            mine &= r == first + i && r >= 0 && r < p.q_rows;
            rows += r >= 0 && r < p.q_rows;
          }
          const bool whole = __all_sync(0xffffffffu, mine);
          rows = __reduce_add_sync(0xffffffffu, rows);
          in_order |= whole ? 1u << w : 0u;
          bytes += whole ? (uint32_t)(128 / G * G) * (2u * D) : (uint32_t)rows * G * (2u * D);
        }
        if (lane == 0) mbar_arrive_expect_tx(bar(C::Q_FULL), bytes);
        __syncwarp();
#pragma unroll 1
        for (int w = 0; w < q_tiles; ++w) {
          const ExtendStream st = extend_stream(item, w);
          const uint32_t dst = sm + C::Q_OFF + w * C::Q_BYTES;
          if ((in_order >> w & 1u) != 0) {
            if (lane < NB) tma_load_3d(dst + lane * 16384, &tp.q_map_tile, 64 * lane, kvh * G, __ldg(p.tokens + 2 * st.tok0), bar(C::Q_FULL));
          } else {
#pragma unroll 1
            for (int i = lane; i < st.ntok; i += 32) {
              const int r = __ldg(p.tokens + 2 * (st.tok0 + i));
              if (r < 0 || r >= p.q_rows) continue;
#pragma unroll 1
              for (int sub = 0; sub < G; sub += tp.q_box_heads)
#pragma unroll
                for (int h = 0; h < NB; ++h)
                  tma_load_3d(dst + (uint32_t)(i * G + sub) * 128 + h * 16384, &tp.q_map, 64 * h, kvh * G + sub, r, bar(C::Q_FULL));
            }
          }
        }
        put_until(t1);
      }
      if (!dead) put_ids(make_int4(0, 0, 0, -1), 0, 0);
      cp_async_wait<0>();
    }
  }

  // ---- release tensor memory
  tc_fence_before();
  __syncthreads();
  if (ext_state(state) < 0)  // copies that nobody waits for any more land before the CTA ends
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(*tmem_slot), "r"(512) : "memory");
  }
}

}  // namespace ft
