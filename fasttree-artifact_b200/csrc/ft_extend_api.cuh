// C entry points of ft_append and ft_extend (part of ft_api.cu: they use its error text, launch counter and descriptor cache).
#pragma once

#include "ft_append.cuh"
#include "ft_extend.cuh"
#include "ft_extend_f32.cuh"
#include "ft_extend_tc.cuh"

namespace {

bool known_head_dim(int d) { return d == 16 || d == 32 || d == 64 || d == 128 || d == 256; }

int check_heads(int dtype, int hq, int hkv, int d) {
  if (dtype != FT_F16 && dtype != FT_BF16 && dtype != FT_F32)
    return fail(FT_ERR_INVALID_ARGUMENT, "dtype %d is not one of FT_F16/FT_BF16/FT_F32", dtype);
  if (hq <= 0 || hkv <= 0) return fail(FT_ERR_INVALID_ARGUMENT, "head counts must be positive (hq %d, hkv %d)", hq, hkv);
  if (!known_head_dim(d)) return fail(FT_ERR_UNSUPPORTED, "head_dim %d is not one of 16, 32, 64, 128, 256", d);
  return FT_OK;
}

// Can a tensor's rows be read and written as vectors of `elems` elements of `size` bytes?
bool vector_rows(const void* p, int64_t s0, int64_t s1, int elems, int size) {
  return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(elems * size - 1)) == 0 && s0 % elems == 0 && s1 % elems == 0;
}

// A [rows, heads, head_dim] tensor's place in memory, strides in bytes; an axis of one entry has stride 0.
struct Place {
  int64_t at, n[2], s[2], inner;
  Place(const void* p, int64_t rows, int heads, int d, int64_t s0, int64_t s1, int size)
      : at((int64_t) reinterpret_cast<uintptr_t>(p)), n{rows, heads}, s{rows > 1 ? s0 * size : 0, heads > 1 ? s1 * size : 0}, inner((int64_t)d * size) {}
  bool operator==(const Place& b) const {
    return at == b.at && n[0] == b.n[0] && n[1] == b.n[1] && s[0] == b.s[0] && s[1] == b.s[1] && inner == b.inner;
  }
  int64_t edge(bool high) const {  // lowest address, or one past the highest
    int64_t x = at + (high ? inner : 0);
    for (int i = 0; i < 2; ++i) {
      const int64_t far = (n[i] - 1) * s[i];
      if ((far > 0) == high) x += far;
    }
    return x;
  }
  // bytes from the tensor's start that it touches in each period, or -1: its strides are not of that period
  int64_t in_period(int64_t period) const {
    int64_t x = inner;
    for (int i = 0; i < 2; ++i) {
      if (s[i] < 0) return -1;
      if (s[i] % period != 0) x += (n[i] - 1) * s[i];
    }
    return x <= period ? x : -1;
  }
};

// May two tensors share a byte?  No, if their address ranges are apart, or if they touch different bytes of a period that both are
// laid out in (columns of one buffer, heads in turn).  Layouts that this does not tell apart count as overlapping.
bool may_overlap(const Place& a, const Place& b) {
  if (a.n[0] <= 0 || a.n[1] <= 0 || b.n[0] <= 0 || b.n[1] <= 0) return false;
  if (a.edge(true) <= b.edge(false) || b.edge(true) <= a.edge(false)) return false;
  const int64_t periods[] = {a.s[0], a.s[1], b.s[0], b.s[1]};
  for (const int64_t p : periods) {
    if (p <= 0) continue;
    const int64_t ea = a.in_period(p), eb = b.in_period(p), r = ((b.at - a.at) % p + p) % p;
    if (ea >= 0 && eb >= 0 && r >= ea && r + eb <= p) return false;
  }
  return true;
}

template <typename T, int VEC, bool PAIRS>
int launch_append(const ft::AppendParams& p, cudaStream_t st) {
  const int units = p.head_dim / (2 * VEC), heads = (p.q != nullptr ? p.q_heads : 0) + 2 * p.kv_heads;
  // a thread per unit, in whole warps, at most 128 (which hold every unit of a head: units is at most 128)
  int threads = (units * heads + 31) / 32 * 32;
  threads = threads > 128 ? 128 : threads;
  ft::append_kernel<T, VEC, PAIRS><<<(unsigned)p.tokens, (unsigned)threads, 0, st>>>(p);
  FT_CUDA_OK(cudaGetLastError());
  count_launch();
  return FT_OK;
}

template <typename T>
int launch_append_for(const ft::AppendParams& p, bool pairs, cudaStream_t st) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const int size = (int)sizeof(T), half = p.rot / 2;
  bool vec = p.head_dim % (2 * VEC) == 0 && half % VEC == 0 && (p.head_dim - p.rot) % (2 * VEC) == 0 &&
             vector_rows(p.k, p.k_s0, p.k_s1, VEC, size) && vector_rows(p.v, p.v_s0, p.v_s1, VEC, size) &&
             vector_rows(p.k_buffer, p.kb_s0, p.kb_s1, VEC, size) && vector_rows(p.v_buffer, p.vb_s0, p.vb_s1, VEC, size);
  if (p.q != nullptr) vec = vec && vector_rows(p.q, p.q_s0, p.q_s1, VEC, size) && vector_rows(p.q_out, p.qo_s0, p.qo_s1, VEC, size);
  if (pairs) return vec ? launch_append<T, VEC, true>(p, st) : launch_append<T, 1, true>(p, st);
  return vec ? launch_append<T, VEC, false>(p, st) : launch_append<T, 1, false>(p, st);
}

// Can the tensor-core kernel take these arguments?  A reason, or NULL.
const char* extend_tc_obstacle(const ft_extend_args* a) {
  if (a->dtype == FT_F32) return "fp32 inputs";
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) return "head_dim not 64, 128 or 256";
  if (a->plan.rows_per_tile != 128) return "more than 128 query heads per KV head";
  // (a stride along one head is never used)
  const int64_t q1 = a->num_qo_heads > 1 ? a->q_stride1 : 0, o1 = a->num_qo_heads > 1 ? a->o_stride1 : 0;
  const int64_t k1 = a->num_kv_heads > 1 ? a->k_stride1 : 0, v1 = a->num_kv_heads > 1 ? a->v_stride1 : 0;
  if (!vector_rows(a->q, a->q_stride0, q1, 8, 2) || !vector_rows(a->k_buffer, a->k_stride0, k1, 8, 2) ||
      !vector_rows(a->v_buffer, a->v_stride0, v1, 8, 2) || !vector_rows(a->o, a->o_stride0, o1, 8, 2))
    return "q, k_buffer, v_buffer and o need 16-byte aligned rows";
  return nullptr;
}

// The descriptors of a call.  They are made anew for each: a step's queries are new tensors every time.  false: the queries'
// layout has none, and the scalar kernel takes the call.
template <int D>
bool extend_maps(ft::ExtendTcParams& tp, const ft_extend_args* a) {
  const int G = a->num_qo_heads / a->num_kv_heads, tile = ft::ExtCfg<D>::TILE, dt = a->dtype;
  const int64_t q1 = a->num_qo_heads > 1 ? a->q_stride1 : D, k1 = a->num_kv_heads > 1 ? a->k_stride1 : D, v1 = a->num_kv_heads > 1 ? a->v_stride1 : D;
  tp.q_box_heads = G % 8 == 0 ? 8 : G;
  if (!encode_map(&tp.q_map, a->q, dt, D, a->q_rows, a->num_qo_heads, a->q_stride0, q1, tp.q_box_heads, 1) ||
      !encode_map(&tp.q_map_tile, a->q, dt, D, a->q_rows, a->num_qo_heads, a->q_stride0, q1, G, 128 / G))
    return false;
  tp.has_tma = encode_map(&tp.k_map, a->k_buffer, dt, D, a->kv_rows, a->num_kv_heads, a->k_stride0, k1, 1, tile) &&
               encode_map(&tp.v_map, a->v_buffer, dt, D, a->kv_rows, a->num_kv_heads, a->v_stride0, v1, 1, tile);
  tp.has_gather4 = encode_map(&tp.k_rows_map, a->k_buffer, dt, D, a->kv_rows, a->num_kv_heads, a->k_stride0, k1, 0, 1) &&
                   encode_map(&tp.v_rows_map, a->v_buffer, dt, D, a->kv_rows, a->num_kv_heads, a->v_stride0, v1, 0, 1);
  return true;
}

template <typename T, int D, bool CAP>
int launch_extend_tc(const ft::ExtendTcParams& tp, int ctas, cudaStream_t st) {
  using C = ft::ExtCfg<D>;
  auto kernel = ft::extend_tc_kernel<T, D, CAP>;
  static OncePerDevice once;
  FT_CUDA_OK(raise_smem_limit(once, kernel, C::SMEM_BYTES));
  if (C::NW == 2) {  // the warpgroups trade the registers that the block is launched with: it has to have them
    static const int regs = [&] {
      cudaFuncAttributes at;
      return cudaFuncGetAttributes(&at, kernel) == cudaSuccess ? at.numRegs : 0;
    }();
    if (regs != C::REGS_LAUNCH) return fail(FT_ERR_UNSUPPORTED, "the kernel was built with %d registers a thread, not %d", regs, C::REGS_LAUNCH);
  }
  FT_CUDA_OK(launch_early(kernel, (unsigned)ctas, C::THREADS, C::SMEM_BYTES, st, tp));
  count_launch();
  return FT_OK;
}

// 1: launched (or named), 0: this call's layout has no descriptors, < 0: an error
template <typename T, int D>
int try_extend_tc(const ft::ExtendParams& p, const ft_extend_args* a, cudaStream_t st) {
  ft::ExtendTcParams tp;
  memset(&tp, 0, sizeof(tp));
  tp.p = p;
  if (!extend_maps<D>(tp, a)) return 0;
  if (dry_run("extend_tc_kernel")) return 1;
  const int rc = p.logit_cap > 0.f ? launch_extend_tc<T, D, true>(tp, a->plan.num_sms, st) : launch_extend_tc<T, D, false>(tp, a->plan.num_sms, st);
  return rc == FT_OK ? 1 : rc;
}

// fp32 rows that the tiled kernel can copy 16 bytes at a time
bool extend_f32_ok(const ft_extend_args* a) {
  return (a->plan.rows_per_tile == 64 || a->plan.rows_per_tile == 16) && vector_rows(a->q, a->q_stride0, a->num_qo_heads > 1 ? a->q_stride1 : 0, 4, 4) &&
         vector_rows(a->o, a->o_stride0, a->num_qo_heads > 1 ? a->o_stride1 : 0, 4, 4) &&
         vector_rows(a->k_buffer, a->k_stride0, a->num_kv_heads > 1 ? a->k_stride1 : 0, 4, 4) &&
         vector_rows(a->v_buffer, a->v_stride0, a->num_kv_heads > 1 ? a->v_stride1 : 0, 4, 4);
}

template <int D, int RPT>
int launch_extend_f32_as(const ft::ExtendParams& p, int ctas, cudaStream_t st) {
  auto kernel = ft::extend_f32_kernel<D, RPT>;
  static OncePerDevice once;
  FT_CUDA_OK(raise_smem_limit(once, kernel, ft::ExtF32Cfg<D, RPT>::SMEM_BYTES));
  FT_CUDA_OK(launch_early(kernel, (unsigned)ctas, 256, ft::ExtF32Cfg<D, RPT>::SMEM_BYTES, st, p));
  count_launch();
  return FT_OK;
}

template <int D>
int launch_extend_f32(const ft::ExtendParams& p, const ft_extend_args* a, cudaStream_t st) {
  return a->plan.rows_per_tile == 64 ? launch_extend_f32_as<D, 4>(p, a->plan.num_sms, st) : launch_extend_f32_as<D, 1>(p, a->plan.num_sms, st);
}

// scheduled early: it reads the plan's lists, which the launch before it reads too, before it waits for that launch
template <typename T, int D>
int launch_extend_merge(const ft::ExtendParams& p, cudaStream_t st) {
  const int64_t pairs = (int64_t)p.num_merged * p.heads;
  const bool split = p.partial_rows > 8LL * p.num_merged;  // more than eight rows a token
  if (split)
    FT_CUDA_OK(launch_early(ft::extend_merge_kernel<T, D, 4>, (unsigned)pairs, 128, 0, st, p));
  else
    FT_CUDA_OK(launch_early(ft::extend_merge_kernel<T, D, 1>, (unsigned)((pairs + 3) / 4), 128, 0, st, p));
  count_launch();
  return FT_OK;
}

template <typename T>
int launch_extend(const ft::ExtendParams& p, const ft_extend_args* a, bool tensor, cudaStream_t st) {
  int done = 0;
  if constexpr (sizeof(T) == 2) {
    if (tensor) done = p.head_dim == 64 ? try_extend_tc<T, 64>(p, a, st) : p.head_dim == 128 ? try_extend_tc<T, 128>(p, a, st) : try_extend_tc<T, 256>(p, a, st);
    if (done < 0) return done;
    if (tensor && done == 0 && a->path == FT_EXTEND_TCGEN05) return fail(FT_ERR_UNSUPPORTED, "tcgen05 path: no TMA descriptor for the layout of q");
  }
  if constexpr (sizeof(T) == 4) {
    if (a->path == FT_EXTEND_AUTO && extend_f32_ok(a)) {
      done = 1;
      if (!dry_run("extend_f32_kernel")) {
        const int rc = p.head_dim == 16   ? launch_extend_f32<16>(p, a, st)
                       : p.head_dim == 32 ? launch_extend_f32<32>(p, a, st)
                       : p.head_dim == 64 ? launch_extend_f32<64>(p, a, st)
                       : p.head_dim == 128 ? launch_extend_f32<128>(p, a, st)
                                           : launch_extend_f32<256>(p, a, st);
        if (rc != FT_OK) return rc;
      }
    }
  }
  if (done == 0 && !dry_run("extend_generic_kernel")) {
    ft::extend_generic_kernel<T><<<(unsigned)(p.num_items * p.kv_heads), 128, 0, st>>>(p);
    FT_CUDA_OK(cudaGetLastError());
    count_launch();
  }
  if (p.num_merged > 0 && !dry_run("extend_merge_kernel")) {
    switch (p.head_dim) {
      case 16: return launch_extend_merge<T, 16>(p, st);
      case 32: return launch_extend_merge<T, 32>(p, st);
      case 64: return launch_extend_merge<T, 64>(p, st);
      case 128: return launch_extend_merge<T, 128>(p, st);
      default: return launch_extend_merge<T, 256>(p, st);
    }
  }
  return FT_OK;
}

// Two warps.  The first waits as the roles of extend_tc_kernel do: (1) for a barrier that nothing arrives at; (2) for the same where
// another role has given up, with probes for seconds; (3) for a completed barrier, with no probe to spare; (4) for a barrier that
// the second warp arrives at long after `limit` probes, counting steps until then; (5) for its next phase, which nothing completes, after the last
// step.  No copy, MMA or tensor memory is involved.
__global__ void extend_wait_selftest_kernel(int limit, int* result) {
  __shared__ __align__(8) unsigned long long barrier_word[3];
  __shared__ int state_word;
  const uint32_t never = ft::smem_u32(barrier_word), done = never + 8, late = never + 16, state = ft::smem_u32(&state_word);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 3; ++i) ft::mbar_init(never + 8 * i, 1);
    state_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    ft::mbar_arrive(done);
  }
  __syncthreads();
  bool plain = false, gone = false, there = true, patient = true, last = false;
  if (warp == 0) plain = ft::ext_wait(never, 0, state, limit);
  __syncthreads();
  if (threadIdx.x == 0) state_word = INT_MIN;
  __syncthreads();
  if (warp == 0) gone = ft::ext_wait(never, 0, state, 1 << 20);
  __syncthreads();
  if (threadIdx.x == 0) state_word = 0;
  __syncthreads();
  if (warp == 0) there = ft::ext_wait(done, 0, state, 0);
  __syncthreads();
  if (warp == 0) {
    patient = ft::ext_wait(late, 0, state, limit);
  } else {
    for (int i = 0; i < 32; ++i) {  // (8 `limit` probes, of the time that the first warp's take, and more)
      for (int n = 0; n < (limit + 7) / 8; ++n)
        if (ft::ext_wait(never, 0, state, 1)) break;
      if (lane == 0) asm volatile("red.shared.add.u32 [%0], 1;\n" ::"r"(state) : "memory");
      __syncwarp();
    }
    if (lane == 0) ft::mbar_arrive(late);
  }
  __syncthreads();
  if (warp == 0) last = ft::ext_wait(late, 1, state, limit);
  if (threadIdx.x == 0) {
    ft::flag_error(FT_DEV_WAIT_TIMEOUT);
    result[0] = (plain ? 1 : 0) + (gone ? 2 : 0) + (there ? 0 : 4) + (patient ? 0 : 8) + (last ? 16 : 0);
    result[1] = ft::EXT_WAIT_LIMIT;
  }
}

}  // namespace

extern "C" {

int ft_selftest_extend_wait(int limit, int* result_host, void* stream) {
  if (result_host == nullptr) return fail(FT_ERR_INVALID_ARGUMENT, "result_host is NULL");
  if (limit < 64 || limit > (1 << 16)) return fail(FT_ERR_INVALID_ARGUMENT, "limit must be in [64, 2^16] probes");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int* dev = nullptr;
  FT_CUDA_OK(cudaMalloc(&dev, 2 * sizeof(int)));
  extend_wait_selftest_kernel<<<1, 64, 0, st>>>(limit, dev);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = cudaMemcpyAsync(result_host, dev, 2 * sizeof(int), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  cudaFree(dev);
  if (e != cudaSuccess) return fail(FT_ERR_CUDA, "extend wait self-test failed: %s", cudaGetErrorString(e));
  count_launch();
  return FT_OK;
}

int ft_append_args_size(void) { return static_cast<int>(sizeof(ft_append_args)); }
int ft_extend_args_size(void) { return static_cast<int>(sizeof(ft_extend_args)); }

int ft_append(const ft_append_args* a) {
  if (a == nullptr) return fail(FT_ERR_INVALID_ARGUMENT, "args is NULL");
  const int rc = check_heads(a->dtype, a->q != nullptr ? a->num_qo_heads : 1, a->num_kv_heads, a->head_dim);
  if (rc != FT_OK) return rc;
  if (a->tokens < 0) return fail(FT_ERR_INVALID_ARGUMENT, "tokens is negative");
  if (a->rot_dim < 0 || a->rot_dim > a->head_dim || a->rot_dim % 2 != 0)
    return fail(FT_ERR_INVALID_ARGUMENT, "rot_dim %d is not an even number up to head_dim %d", a->rot_dim, a->head_dim);
  ft::AppendParams p;
  memset(&p, 0, sizeof(p));
  if (a->rot_dim > 0) {
    if (a->num_axes < 1 || a->num_axes > 4) return fail(FT_ERR_INVALID_ARGUMENT, "num_axes %d is not 1 to 4", a->num_axes);
    int64_t end = 0;
    for (int i = 0; i < a->num_axes; ++i) {
      if (a->sections[i] < 0) return fail(FT_ERR_INVALID_ARGUMENT, "sections[%d] is negative", i);
      end += a->sections[i];
      p.section_end[i] = (int32_t)(end < 0x7fffffff ? end : 0x7fffffff);
    }
    if (end != a->rot_dim / 2)
      return fail(FT_ERR_INVALID_ARGUMENT, "the sections hold %lld pairs, rot_dim %d has %d", (long long)end, a->rot_dim, a->rot_dim / 2);
    if (a->cos_sin_stride0 < 0) return fail(FT_ERR_INVALID_ARGUMENT, "cos_sin_stride0 is negative");
  }
  if (a->tokens == 0) return FT_OK;
  if (a->k == nullptr || a->v == nullptr || a->k_buffer == nullptr || a->v_buffer == nullptr || a->slots == nullptr)
    return fail(FT_ERR_INVALID_ARGUMENT, "k / v / k_buffer / v_buffer / slots is NULL");
  if ((a->q == nullptr) != (a->q_out == nullptr)) return fail(FT_ERR_INVALID_ARGUMENT, "one of q and q_out is NULL");
  if (a->kv_rows <= 0) return fail(FT_ERR_INVALID_ARGUMENT, "kv_rows must be positive");
  if (a->rot_dim > 0 && (a->positions == nullptr || a->cos_sin == nullptr || a->cos_sin_rows <= 0))
    return fail(FT_ERR_INVALID_ARGUMENT, "a rotation needs positions and a table of cosines and sines");
  const int size = a->dtype == FT_F32 ? 4 : 2;
  if (a->q != nullptr) {
    const Place out(a->q_out, a->tokens, a->num_qo_heads, a->head_dim, a->q_out_stride0, a->q_out_stride1, size),
        q(a->q, a->tokens, a->num_qo_heads, a->head_dim, a->q_stride0, a->q_stride1, size);
    const struct {
      const char* name;
      Place place;
    } others[] = {{"k", Place(a->k, a->tokens, a->num_kv_heads, a->head_dim, a->k_stride0, a->k_stride1, size)},
                  {"v", Place(a->v, a->tokens, a->num_kv_heads, a->head_dim, a->v_stride0, a->v_stride1, size)},
                  {"k_buffer", Place(a->k_buffer, a->kv_rows, a->num_kv_heads, a->head_dim, a->k_buffer_stride0, a->k_buffer_stride1, size)},
                  {"v_buffer", Place(a->v_buffer, a->kv_rows, a->num_kv_heads, a->head_dim, a->v_buffer_stride0, a->v_buffer_stride1, size)}};
    if (!(out == q) && may_overlap(out, q)) return fail(FT_ERR_INVALID_ARGUMENT, "q_out overlaps q and is not q");
    for (const auto& other : others)
      if (may_overlap(out, other.place)) return fail(FT_ERR_INVALID_ARGUMENT, "q_out overlaps %s", other.name);
  }
  p.q = a->q, p.k = a->k, p.v = a->v, p.q_out = a->q_out, p.k_buffer = a->k_buffer, p.v_buffer = a->v_buffer;
  p.slots = a->slots, p.positions = a->positions, p.cos_sin = a->cos_sin;
  p.q_s0 = a->q_stride0, p.q_s1 = a->q_stride1, p.k_s0 = a->k_stride0, p.k_s1 = a->k_stride1;
  p.v_s0 = a->v_stride0, p.v_s1 = a->v_stride1, p.qo_s0 = a->q_out_stride0, p.qo_s1 = a->q_out_stride1;
  p.kb_s0 = a->k_buffer_stride0, p.kb_s1 = a->k_buffer_stride1, p.vb_s0 = a->v_buffer_stride0, p.vb_s1 = a->v_buffer_stride1;
  p.kv_rows = a->kv_rows, p.positions_s0 = a->positions_stride0, p.cos_sin_rows = a->cos_sin_rows, p.cos_sin_s0 = a->cos_sin_stride0;
  p.tokens = a->tokens, p.q_heads = a->num_qo_heads, p.kv_heads = a->num_kv_heads, p.head_dim = a->head_dim, p.rot = a->rot_dim;
  p.axes = a->rot_dim > 0 ? a->num_axes : 0;
  p.slots_64 = a->slots_64, p.positions_64 = a->positions_64;
  cudaStream_t st = static_cast<cudaStream_t>(a->stream);
  if (a->dtype == FT_F16) return launch_append_for<__half>(p, a->interleaved != 0, st);
  if (a->dtype == FT_BF16) return launch_append_for<__nv_bfloat16>(p, a->interleaved != 0, st);
  return launch_append_for<float>(p, a->interleaved != 0, st);
}

int ft_extend(const ft_extend_args* a) {
  if (a == nullptr) return fail(FT_ERR_INVALID_ARGUMENT, "args is NULL");
  const int rc = check_heads(a->dtype, a->num_qo_heads, a->num_kv_heads, a->head_dim);
  if (rc != FT_OK) return rc;
  const ft_extend_plan_info& pl = a->plan;
  if (pl.num_qo_heads != a->num_qo_heads || pl.num_kv_heads != a->num_kv_heads || pl.head_dim != a->head_dim ||
      pl.elem_bytes != (a->dtype == FT_F32 ? 4 : 2))
    return fail(FT_ERR_INVALID_ARGUMENT, "the plan was made for %d/%d heads of %d, %d bytes an element", pl.num_qo_heads, pl.num_kv_heads,
                pl.head_dim, pl.elem_bytes);
  if (a->path != FT_EXTEND_AUTO && a->path != FT_EXTEND_GENERIC && a->path != FT_EXTEND_TCGEN05)
    return fail(FT_ERR_INVALID_ARGUMENT, "unknown path %d", a->path);
  if (pl.num_items < 0 || pl.num_tokens < 0 || pl.num_merged < 0 || pl.partial_rows < 0)
    return fail(FT_ERR_INVALID_ARGUMENT, "the plan's counts are negative");
  if (pl.num_items == 0) return FT_OK;  // no query
  const struct {
    int64_t off, ints;
  } parts[] = {{pl.items_off, (int64_t)pl.num_items * ft::EXT_ITEM_INTS}, {pl.tokens_off, 2LL * pl.num_tokens}, {pl.tiles_off, 8LL * pl.num_tiles},
               {pl.extra_off, 0}, {pl.sms_off, 16LL * pl.num_sms}, {pl.sm_tasks_off, (int64_t)pl.num_items * pl.num_kv_heads},
               {pl.merge_off, 4LL * pl.num_merged}, {pl.merge_rows_off, 0}};
  for (const auto& part : parts)
    if (part.off < 0 || part.off % 4 != 0 || part.ints < 0 || part.off + part.ints > pl.table_ints)
      return fail(FT_ERR_INVALID_ARGUMENT, "the plan's parts do not lie in its table");
  // the sizes that the kernels are compiled for, as ft_extend_plan_build chooses them
  const int group = a->num_qo_heads / a->num_kv_heads;
  const bool tensor_form = pl.elem_bytes == 2 && a->head_dim >= 64 && group <= 128;
  if (a->num_qo_heads % a->num_kv_heads != 0 || pl.num_sms <= 0 || pl.tile_tokens != (tensor_form && a->head_dim <= 128 ? 128 : 64) ||
      !(pl.rows_per_tile == (tensor_form ? 128 : 64) || (!tensor_form && pl.rows_per_tile == 16)))
    return fail(FT_ERR_INVALID_ARGUMENT, "the plan's sizes are not a plan's");
  if (a->q == nullptr || a->k_buffer == nullptr || a->v_buffer == nullptr || a->o == nullptr || a->kv_entries == nullptr || a->plan_table == nullptr)
    return fail(FT_ERR_INVALID_ARGUMENT, "q / k_buffer / v_buffer / o / kv_entries / plan_table is NULL");
  if (!aligned16(a->plan_table)) return fail(FT_ERR_UNSUPPORTED, "plan_table must be 16-byte aligned");
  if (a->kv_rows <= 0) return fail(FT_ERR_INVALID_ARGUMENT, "kv_rows must be positive");
  if (pl.kv_entries_len > a->kv_entries_len)
    return fail(FT_ERR_INVALID_ARGUMENT, "the plan names %lld entries of kv_entries, which has %lld", (long long)pl.kv_entries_len,
                (long long)a->kv_entries_len);
  if (pl.q_rows > a->q_rows)
    return fail(FT_ERR_INVALID_ARGUMENT, "the plan names %lld rows of q, which has %lld", (long long)pl.q_rows, (long long)a->q_rows);
  if (pl.partial_rows > 0 && (a->mid_o == nullptr || a->mid_lse == nullptr || !aligned16(a->mid_o)))
    return fail(FT_ERR_INVALID_ARGUMENT, "the plan has partial rows: mid_o (16-byte aligned) and mid_lse are needed");
  if ((int64_t)pl.num_items * a->num_kv_heads > 0x7fffffffLL || (int64_t)pl.num_merged * a->num_qo_heads > 0x7fffffffLL)
    return fail(FT_ERR_TOO_LARGE, "more tasks than one launch takes");
  // (rows of q are read after rows of o are written)
  const int size = pl.elem_bytes;
  const Place out(a->o, pl.q_rows, a->num_qo_heads, a->head_dim, a->o_stride0, a->o_stride1, size);
  if (may_overlap(out, Place(a->q, pl.q_rows, a->num_qo_heads, a->head_dim, a->q_stride0, a->q_stride1, size)))
    return fail(FT_ERR_INVALID_ARGUMENT, "o overlaps q");
  if (may_overlap(out, Place(a->k_buffer, a->kv_rows, a->num_kv_heads, a->head_dim, a->k_stride0, a->k_stride1, size)) ||
      may_overlap(out, Place(a->v_buffer, a->kv_rows, a->num_kv_heads, a->head_dim, a->v_stride0, a->v_stride1, size)))
    return fail(FT_ERR_INVALID_ARGUMENT, "o overlaps the pool");
  const char* obstacle = extend_tc_obstacle(a);
  if (a->path == FT_EXTEND_TCGEN05 && obstacle != nullptr) return fail(FT_ERR_UNSUPPORTED, "tcgen05 path: %s", obstacle);
  const bool tensor = a->path != FT_EXTEND_GENERIC && obstacle == nullptr;

  ft::ExtendParams p;
  memset(&p, 0, sizeof(p));
  p.q = a->q, p.k = a->k_buffer, p.v = a->v_buffer, p.o = a->o, p.o_lse = a->o_lse, p.kv_entries = a->kv_entries;
  p.items = a->plan_table + pl.items_off, p.tokens = a->plan_table + pl.tokens_off;
  p.tiles = a->plan_table + pl.tiles_off, p.extra = a->plan_table + pl.extra_off, p.sms = a->plan_table + pl.sms_off, p.sm_tasks = a->plan_table + pl.sm_tasks_off;
  p.merged = a->plan_table + pl.merge_off, p.merge_rows = a->plan_table + pl.merge_rows_off;
  p.mid_o = a->mid_o, p.mid_lse = a->mid_lse;
  p.q_s0 = a->q_stride0, p.q_s1 = a->q_stride1, p.k_s0 = a->k_stride0, p.k_s1 = a->num_kv_heads > 1 ? a->k_stride1 : 0;
  p.v_s0 = a->v_stride0, p.v_s1 = a->num_kv_heads > 1 ? a->v_stride1 : 0, p.o_s0 = a->o_stride0, p.o_s1 = a->o_stride1;
  p.kv_rows = a->kv_rows, p.q_rows = a->q_rows, p.kv_entries_len = a->kv_entries_len;
  p.num_items = pl.num_items, p.num_merged = pl.num_merged, p.partial_rows = pl.partial_rows;
  p.heads = a->num_qo_heads, p.kv_heads = a->num_kv_heads, p.group = a->num_qo_heads / a->num_kv_heads, p.head_dim = a->head_dim;
  p.tile = pl.tile_tokens;
  p.sm_scale = a->sm_scale, p.logit_cap = a->logit_cap > 0.f && a->logit_cap < INFINITY ? a->logit_cap : 0.f;  // (an infinite cap is none)
  cudaStream_t st = static_cast<cudaStream_t>(a->stream);
  if (a->dtype == FT_F16) return launch_extend<__half>(p, a, tensor, st);
  if (a->dtype == FT_BF16) return launch_extend<__nv_bfloat16>(p, a, tensor, st);
  return launch_extend<float>(p, a, false, st);
}

const char* ft_extend_path_name(const ft_extend_args* args) {
  g_kernel_names[0] = '\0';
  g_dry_run = true;
  const int rc = ft_extend(args);
  g_dry_run = false;
  if (rc != FT_OK) return nullptr;
  return g_kernel_names;
}

}  // extern "C"
