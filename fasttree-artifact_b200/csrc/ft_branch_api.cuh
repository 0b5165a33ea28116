// C entry points for branching continuations: ft_draft_tree, ft_draft_accept, ft_beam_select, ft_beam_reorder (part of ft_api.cu, as
// ft_extend_api.cuh).
#pragma once

#include "ft_beam.cuh"
#include "ft_draft.cuh"

namespace {

// A draft plan's parts lie in its table, and its requests' rows within `rows`.
int check_draft_plan(const ft_extend_plan_info& pl, const int32_t* table, int64_t rows) {
  if (pl.draft != 1) return fail(FT_ERR_INVALID_ARGUMENT, "the plan was not made for drafted tokens");
  if (pl.num_drafts < 0 || pl.num_spans < 0 || pl.longest_draft < 0 || pl.longest_draft > FT_MAX_DRAFT || pl.num_tokens < 0)
    return fail(FT_ERR_INVALID_ARGUMENT, "the plan's counts are not a plan's");
  if (pl.drafts_off < 0 || pl.drafts_off % 4 != 0 || pl.drafts_off + 8LL * pl.num_drafts > pl.table_ints || pl.spans_off < 0 || pl.spans_off % 4 != 0 ||
      pl.spans_off + 8LL * pl.num_spans > pl.table_ints || pl.extra_off < 0 || pl.extra_off % 4 != 0 || pl.extra_off > pl.table_ints)
    return fail(FT_ERR_INVALID_ARGUMENT, "the plan's parts do not lie in its table");
  if (pl.tile_tokens != 64 && pl.tile_tokens != 128) return fail(FT_ERR_INVALID_ARGUMENT, "the plan's sizes are not a plan's");
  if (pl.num_tokens == 0) return FT_OK;
  if (table == nullptr) return fail(FT_ERR_INVALID_ARGUMENT, "plan_table is NULL");
  if (!aligned16(table)) return fail(FT_ERR_UNSUPPORTED, "plan_table must be 16-byte aligned");
  if (pl.q_rows > rows) return fail(FT_ERR_INVALID_ARGUMENT, "the plan names %lld tokens, the call has %lld", (long long)pl.q_rows, (long long)rows);
  return FT_OK;
}

// A row of `n` elements, or `rows` of them, as a place in memory.
Place rows_at(const void* p, int64_t rows, int64_t n, int64_t s0, int size) { return Place(p, n > 0 ? rows : 0, 1, (int)n, s0, 0, size); }
Place row_at(const void* p, int64_t n, int size) { return rows_at(p, p != nullptr ? n : 0, 1, 1, size); }
int index_size(int is_64) { return is_64 ? 8 : 4; }

int current_sms() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess ? sm_count(dev) : 148;
}

template <typename T>
int launch_accept(const ft::AcceptParams& p, int requests, int64_t row_bytes, cudaStream_t st) {
  // CTAs per request: as many as the SMs hold two of, so that all are there at once, as long as each has 16 KB of a row to read (with
  // 1, 2, 4, 8: 64 requests, 131072 bf16 logits, 1 to 6 rows a path 45, 35, 29, 41 us; 33 requests, 100003 fp32, 1 to 5 rows 53, 38, 29, 24)
  int ranks = 1;
  const int room = 2 * current_sms();
  while (p.targets == nullptr && ranks < 8 && (int64_t)requests * ranks * 2 <= room && row_bytes / (2 * ranks) >= 16384) ranks *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(requests * ranks));
  cfg.blockDim = dim3(ft::ACCEPT_THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  FT_CUDA_OK(cudaLaunchKernelEx(&cfg, ft::draft_accept_kernel<T>, p));
  count_launch();
  return FT_OK;
}

struct BeamShape {
  int pieces, slices, chunks, per_cta, pitch;
  int64_t ctas, keys, bytes;  // of the workspace: keys, then sums
};

int dtype_size(int dtype) { return dtype == FT_F32 ? 4 : 2; }

int check_beam_select(const ft_beam_select_args* a) {
  if (a == nullptr) return fail(FT_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->dtype != FT_F16 && a->dtype != FT_BF16 && a->dtype != FT_F32)
    return fail(FT_ERR_INVALID_ARGUMENT, "dtype %d is not one of FT_F16/FT_BF16/FT_F32", a->dtype);
  if (a->batch < 0 || a->beams <= 0 || a->beams > FT_MAX_BEAMS || a->best <= 0 || a->best > FT_MAX_BEAMS)
    return fail(FT_ERR_INVALID_ARGUMENT, "beams %d and best %d must be 1 to %d", a->beams, a->best, FT_MAX_BEAMS);
  if (a->vocab <= 0 || a->vocab > FT_MAX_VOCAB) return fail(FT_ERR_INVALID_ARGUMENT, "vocab must be 1 to 2^30");
  return FT_OK;
}

// Shared memory for the listed logits of a request, 4 bytes each: 64 results of 592 slices (rows with CTAs of their own, all CTAs at once)
// take 148 KB of it.
constexpr int BEAM_MERGE_SMEM = 176 << 10;

// Chunks of a call and how many a CTA takes, all CTAs at once.  Chunks of 16 KB, smaller ones where the call would leave SMs without any or
// rows are shorter.  In chunks, a slice costs seven beside its own: dealt evenly, a CTA has the ends of two rows or more; with CTAs
// of their own, or whole rows to a CTA, rows have no more slices than they need (64 x 4 rows of 16 chunks, two CTAs to a row: 29 us,
// seven chunks to a CTA 31).  Few long rows dealt evenly can have more slices than the merge holds (1 x 59 rows: 708): they get CTAs of their own
// too.  (148 SMs whatever the device: the workspace's size goes by this.)
BeamShape beam_shape(const ft_beam_select_args* a) {
  BeamShape s;
  const int n = 16 / dtype_size(a->dtype);
  const int64_t rows = std::max<int64_t>(1, (int64_t)a->batch * a->beams), ctas = ft::BEAM_CTAS * 148;
  int64_t chunk = 0;
  for (s.pieces = 4;; s.pieces /= 2) {
    chunk = (int64_t)ft::BEAM_THREADS * n * s.pieces;
    s.chunks = (int)((a->vocab + chunk - 1) / chunk);
    if (s.pieces == 1 || (rows * s.chunks >= 2 * 148 && chunk <= a->vocab)) break;
  }
  const int64_t even = (rows * s.chunks + ctas - 1) / ctas;
  s.per_cta = (int)even;
  s.pitch = s.chunks;
  auto dealt_slices = [&]() {
    return s.chunks % s.per_cta == 0 ? s.chunks / s.per_cta : s.per_cta % s.chunks == 0 ? 1 : std::min((s.chunks - 1) / s.per_cta + 2, s.chunks);
  };
  if (rows <= ctas) {
    const int64_t own = (s.chunks + ctas / rows - 1) / (ctas / rows);  // chunks of a CTA, with ctas / rows of them to a row
    if (own <= even + 7 || 4LL * a->beams * dealt_slices() * a->best > BEAM_MERGE_SMEM) {
      s.per_cta = (int)own;
      s.pitch = (int)((s.chunks + own - 1) / own * own);
    }
  } else {
    const int64_t each = (rows + ctas - 1) / ctas;  // rows of a CTA; dealt evenly it has one more slice
    if (each * s.chunks <= even + 7) s.per_cta = (int)(each * s.chunks);
  }
  s.ctas = (rows * s.pitch + s.per_cta - 1) / s.per_cta;
  s.slices = s.pitch > s.chunks ? s.pitch / s.per_cta : dealt_slices();
  s.keys = rows * s.slices * a->best;
  s.bytes = s.keys * 8 + rows * s.slices * 8;
  return s;
}

int pow2_at_least(int n, int low) {
  while (low < n) low *= 2;
  return low;
}

template <typename T, int NV, bool VEC>
int launch_scan_as(const ft::BeamParams& p, const BeamShape& s, cudaStream_t st) {
  auto kernel = ft::beam_scan_kernel<T, NV, VEC>;
  static OncePerDevice once;
  FT_CUDA_OK(raise_smem_limit(once, kernel, ft::BeamScan<NV>::SMEM_BYTES));
  kernel<<<(unsigned)s.ctas, ft::BEAM_THREADS + 32, ft::BeamScan<NV>::SMEM_BYTES, st>>>(p);
  FT_CUDA_OK(cudaGetLastError());
  count_launch();
  return FT_OK;
}

template <typename T>
int launch_beam_select(const ft::BeamParams& p, const BeamShape& s, bool vec, cudaStream_t st) {
  const int rc = s.pieces == 1   ? (vec ? launch_scan_as<T, 1, true>(p, s, st) : launch_scan_as<T, 1, false>(p, s, st))
                 : s.pieces == 2 ? (vec ? launch_scan_as<T, 2, true>(p, s, st) : launch_scan_as<T, 2, false>(p, s, st))
                                 : (vec ? launch_scan_as<T, 4, true>(p, s, st) : launch_scan_as<T, 4, false>(p, s, st));
  if (rc != FT_OK) return rc;
  const int64_t smem = 4LL * p.beams * p.slices * p.best;
  static OncePerDevice once;
  FT_CUDA_OK(raise_smem_limit(once, ft::beam_merge_kernel, BEAM_MERGE_SMEM));
  FT_CUDA_OK(launch_early(ft::beam_merge_kernel, dim3((unsigned)p.batch), ft::BEAM_THREADS, (size_t)smem, st, p));
  count_launch();
  return FT_OK;
}

}  // namespace

extern "C" {

int ft_draft_tree_args_size(void) { return static_cast<int>(sizeof(ft_draft_tree_args)); }
int ft_draft_accept_args_size(void) { return static_cast<int>(sizeof(ft_draft_accept_args)); }
int ft_beam_select_args_size(void) { return static_cast<int>(sizeof(ft_beam_select_args)); }
int ft_beam_reorder_args_size(void) { return static_cast<int>(sizeof(ft_beam_reorder_args)); }

int ft_draft_tree(const ft_draft_tree_args* a) {
  if (a == nullptr) return fail(FT_ERR_INVALID_ARGUMENT, "args is NULL");
  const int rc = check_draft_plan(a->plan, a->plan_table, a->rows);
  if (rc != FT_OK) return rc;
  if (a->plan.num_tokens == 0) return FT_OK;
  if (a->parents == nullptr) return fail(FT_ERR_INVALID_ARGUMENT, "parents is NULL");
  if (may_overlap(row_at(a->positions, a->plan.q_rows, index_size(a->positions_64)), row_at(a->parents, a->plan.q_rows, index_size(a->parents_64))))
    return fail(FT_ERR_INVALID_ARGUMENT, "positions overlaps parents");
  ft::DraftParams p;
  memset(&p, 0, sizeof(p));
  p.drafts = a->plan_table + a->plan.drafts_off;
  p.spans = reinterpret_cast<const DraftSpan*>(a->plan_table + a->plan.spans_off);
  p.extra = a->plan_table + a->plan.extra_off;
  p.parents = a->parents, p.positions = a->positions;
  p.parents_64 = a->parents_64, p.positions_64 = a->positions_64;
  p.window = a->plan.window, p.words = a->plan.tile_tokens / 32;
  // (a token of a long chain climbs through all of its spans: a CTA for every 128 tokens of the longest draft)
  const dim3 grid((unsigned)a->plan.num_drafts, (unsigned)((a->plan.longest_draft + 127) / 128));
  ft::draft_tree_kernel<<<grid, ft::DRAFT_THREADS, 0, static_cast<cudaStream_t>(a->stream)>>>(p);
  FT_CUDA_OK(cudaGetLastError());
  count_launch();
  return FT_OK;
}

int ft_draft_accept(const ft_draft_accept_args* a) {
  if (a == nullptr) return fail(FT_ERR_INVALID_ARGUMENT, "args is NULL");
  const int rc = check_draft_plan(a->plan, a->plan_table, a->rows);
  if (rc != FT_OK) return rc;
  const ft_extend_plan_info& pl = a->plan;
  if ((a->logits == nullptr) == (a->targets == nullptr) && pl.num_tokens > 0)
    return fail(FT_ERR_INVALID_ARGUMENT, "one of logits and targets must be given");
  if (a->dtype != FT_F16 && a->dtype != FT_BF16 && a->dtype != FT_F32)
    return fail(FT_ERR_INVALID_ARGUMENT, "dtype %d is not one of FT_F16/FT_BF16/FT_F32", a->dtype);
  if (a->logits != nullptr && (a->vocab <= 0 || a->vocab > FT_MAX_VOCAB)) return fail(FT_ERR_INVALID_ARGUMENT, "vocab must be 1 to 2^30");
  if (a->num_requests < pl.num_drafts) return fail(FT_ERR_INVALID_ARGUMENT, "the plan has %d requests, the results %d", pl.num_drafts, a->num_requests);
  if (a->accepted_width < pl.longest_draft)
    return fail(FT_ERR_INVALID_ARGUMENT, "accepted has %d entries a request, the longest draft %d tokens", a->accepted_width, pl.longest_draft);
  if (pl.num_drafts == 0) return FT_OK;
  if (a->plan_table == nullptr || !aligned16(a->plan_table)) return fail(FT_ERR_INVALID_ARGUMENT, "plan_table is NULL or not 16-byte aligned");
  if (a->accepted == nullptr || a->counts == nullptr || a->next_tokens == nullptr ||
      (pl.num_tokens > 0 && (a->tokens == nullptr || a->parents == nullptr)))
    return fail(FT_ERR_INVALID_ARGUMENT, "tokens / parents / accepted / counts / next_tokens is NULL");
  if ((a->slots == nullptr) != (a->kv_entries == nullptr) && pl.num_tokens > 0)
    return fail(FT_ERR_INVALID_ARGUMENT, "slots and kv_entries go together");
  if (a->slots != nullptr && pl.kv_entries_len > a->kv_entries_len)
    return fail(FT_ERR_INVALID_ARGUMENT, "the plan names %lld entries of kv_entries, which has %lld", (long long)pl.kv_entries_len,
                (long long)a->kv_entries_len);
  // a request's tokens are read while another's results are written
  const Place results[] = {rows_at(a->accepted, a->num_requests, a->accepted_width, a->accepted_stride0, 4), row_at(a->counts, a->num_requests, 4),
                           row_at(a->next_tokens, a->num_requests, index_size(a->next_64)), row_at(a->slots != nullptr ? a->kv_entries : nullptr, a->kv_entries_len, 4)};
  const char* const result_names[] = {"accepted", "counts", "next_tokens", "kv_entries"};
  const Place inputs[] = {row_at(a->tokens, pl.q_rows, index_size(a->tokens_64)), row_at(a->parents, pl.q_rows, index_size(a->parents_64)),
                          row_at(a->targets, pl.q_rows, index_size(a->targets_64)),
                          rows_at(a->logits, a->logits != nullptr ? pl.q_rows : 0, a->vocab, a->logits_stride0, dtype_size(a->dtype)),
                          row_at(a->slots, pl.q_rows, index_size(a->slots_64))};
  const char* const input_names[] = {"tokens", "parents", "targets", "logits", "slots"};
  for (int r = 0; r < 4; ++r) {
    for (int i = 0; i < 5; ++i) {
      if (r == 3 && i == 4 && pl.num_drafts == 1) continue;  // one request's rows may stand at their entries: they are read first
      if (may_overlap(results[r], inputs[i])) return fail(FT_ERR_INVALID_ARGUMENT, "%s overlaps %s", result_names[r], input_names[i]);
    }
    for (int i = 0; i < r; ++i)
      if (may_overlap(results[r], results[i])) return fail(FT_ERR_INVALID_ARGUMENT, "%s overlaps %s", result_names[r], result_names[i]);
  }
  ft::AcceptParams p;
  memset(&p, 0, sizeof(p));
  p.drafts = a->plan_table + pl.drafts_off;
  p.logits = a->logits, p.targets = a->targets, p.tokens = a->tokens, p.parents = a->parents;
  p.accepted = a->accepted, p.counts = a->counts, p.next_tokens = a->next_tokens;
  p.slots = a->kv_entries != nullptr ? a->slots : nullptr, p.kv_entries = a->kv_entries;
  p.logits_s0 = a->logits_stride0, p.accepted_s0 = a->accepted_stride0, p.kv_entries_len = a->kv_entries_len;
  p.vocab = a->vocab, p.width = a->accepted_width;
  p.targets_64 = a->targets_64, p.tokens_64 = a->tokens_64, p.parents_64 = a->parents_64, p.next_64 = a->next_64, p.slots_64 = a->slots_64;
  const int64_t row_bytes = (int64_t)a->vocab * dtype_size(a->dtype);
  cudaStream_t st = static_cast<cudaStream_t>(a->stream);
  if (a->dtype == FT_F16) return launch_accept<__half>(p, pl.num_drafts, row_bytes, st);
  if (a->dtype == FT_BF16) return launch_accept<__nv_bfloat16>(p, pl.num_drafts, row_bytes, st);
  return launch_accept<float>(p, pl.num_drafts, row_bytes, st);
}

int64_t ft_beam_select_workspace(const ft_beam_select_args* a) {
  const int rc = check_beam_select(a);
  return rc != FT_OK ? rc : beam_shape(a).bytes;
}

int ft_beam_select(const ft_beam_select_args* a) {
  const int rc = check_beam_select(a);
  if (rc != FT_OK) return rc;
  if (a->batch == 0) return FT_OK;
  if (a->logits == nullptr || a->scores == nullptr || a->out_scores == nullptr || a->out_beams == nullptr || a->out_tokens == nullptr)
    return fail(FT_ERR_INVALID_ARGUMENT, "logits / scores / out_scores / out_beams / out_tokens is NULL");
  if (a->workspace == nullptr || !aligned16(a->workspace)) return fail(FT_ERR_INVALID_ARGUMENT, "workspace is NULL or not 16-byte aligned");
  // scores may be the results' rows, or the start of each: a request's are read before its results are written
  const Place scores(a->scores, a->batch, a->beams, 1, a->scores_stride0, a->scores_stride1, 4);
  const Place results[] = {rows_at(a->out_scores, a->batch, a->best, a->out_scores_stride0, 4),
                           rows_at(a->out_beams, a->batch, a->best, a->out_beams_stride0, index_size(a->beams_64)),
                           rows_at(a->out_tokens, a->batch, a->best, a->out_tokens_stride0, index_size(a->tokens_64))};
  const bool in_place = static_cast<const void*>(a->scores) == a->out_scores && (a->batch == 1 || a->scores_stride0 == a->out_scores_stride0) &&
                        (a->beams == 1 || a->scores_stride1 == 1) && (a->batch == 1 || a->beams <= a->scores_stride0);
  const Place logits[] = {Place(a->logits, a->batch, a->beams, a->vocab, a->logits_stride0, a->logits_stride1, dtype_size(a->dtype))};
  for (int r = 0; r < 3; ++r) {
    if (may_overlap(results[r], logits[0])) return fail(FT_ERR_INVALID_ARGUMENT, "a result overlaps logits");
    if (!(r == 0 && in_place) && may_overlap(results[r], scores)) return fail(FT_ERR_INVALID_ARGUMENT, "a result overlaps scores, whose rows are not its own");
    for (int i = 0; i < r; ++i)
      if (may_overlap(results[r], results[i])) return fail(FT_ERR_INVALID_ARGUMENT, "two results overlap");
  }
  const BeamShape s = beam_shape(a);
  if ((int64_t)a->batch * a->beams > 0x7fffffffLL / 64 || s.ctas > 0x7fffffffLL || (int64_t)a->beams * s.slices * a->best > 0x7fffffffLL / 2)
    return fail(FT_ERR_TOO_LARGE, "more slices of logits than one launch takes");
  ft::BeamParams p;
  memset(&p, 0, sizeof(p));
  p.logits = a->logits, p.scores = a->scores, p.out_scores = a->out_scores, p.out_beams = a->out_beams, p.out_tokens = a->out_tokens;
  p.keys = static_cast<unsigned long long*>(a->workspace);
  p.sums = reinterpret_cast<float2*>(p.keys + s.keys);
  p.logits_s0 = a->logits_stride0, p.logits_s1 = a->logits_stride1, p.scores_s0 = a->scores_stride0, p.scores_s1 = a->scores_stride1;
  p.out_scores_s0 = a->out_scores_stride0, p.out_beams_s0 = a->out_beams_stride0, p.out_tokens_s0 = a->out_tokens_stride0;
  p.batch = a->batch, p.beams = a->beams, p.vocab = a->vocab, p.best = a->best, p.slices = s.slices, p.chunks = s.chunks, p.per_cta = s.per_cta, p.pitch = s.pitch;
  p.beams_64 = a->beams_64, p.tokens_64 = a->tokens_64;
  const int n = 16 / dtype_size(a->dtype);
  const bool vec = aligned16(a->logits) && (a->batch == 1 || a->logits_stride0 % n == 0) && (a->beams == 1 || a->logits_stride1 % n == 0);
  cudaStream_t st = static_cast<cudaStream_t>(a->stream);
  if (a->dtype == FT_F16) return launch_beam_select<__half>(p, s, vec, st);
  if (a->dtype == FT_BF16) return launch_beam_select<__nv_bfloat16>(p, s, vec, st);
  return launch_beam_select<float>(p, s, vec, st);
}

int ft_beam_reorder(const ft_beam_reorder_args* a) {
  if (a == nullptr) return fail(FT_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->elem_bytes != 4 && a->elem_bytes != 8) return fail(FT_ERR_INVALID_ARGUMENT, "elements of %d bytes, not 4 or 8", a->elem_bytes);
  if (a->batch < 0 || a->from <= 0 || a->from > FT_MAX_BEAMS || a->to <= 0 || a->to > FT_MAX_BEAMS)
    return fail(FT_ERR_INVALID_ARGUMENT, "rows of %d and %d beams a request must be 1 to %d", a->from, a->to, FT_MAX_BEAMS);
  if (a->table_rows < 0 || a->width < 0) return fail(FT_ERR_INVALID_ARGUMENT, "the table's sizes are negative");
  if (a->batch == 0 || a->table_rows == 0 || a->width == 0) return FT_OK;
  if (a->table == nullptr || a->rows == nullptr || a->beams == nullptr || a->out_rows == nullptr)
    return fail(FT_ERR_INVALID_ARGUMENT, "table / rows / beams / out_rows is NULL");
  if (a->batch > 65535) return fail(FT_ERR_TOO_LARGE, "more than 65535 requests");
  if (a->width > 0x7fffffffLL / 8) return fail(FT_ERR_TOO_LARGE, "the table's rows are too long for one launch");
  const Place table = rows_at(a->table, a->table_rows, a->width, a->table_stride0, a->elem_bytes);
  const Place numbers[] = {rows_at(a->rows, a->batch, a->from, a->rows_stride0, index_size(a->rows_64)),
                           rows_at(a->beams, a->batch, a->to, a->beams_stride0, index_size(a->beams_64)),
                           rows_at(a->out_rows, a->batch, a->to, a->out_rows_stride0, index_size(a->out_rows_64)),
                           row_at(a->starts, a->batch, index_size(a->starts_64)), row_at(a->ends, a->batch, index_size(a->ends_64))};
  for (const Place& n : numbers)
    if (may_overlap(table, n)) return fail(FT_ERR_INVALID_ARGUMENT, "the table overlaps the rows' or beams' numbers");
  ft::ReorderParams p;
  memset(&p, 0, sizeof(p));
  p.words = a->elem_bytes / 4;
  p.table = static_cast<uint32_t*>(a->table);
  p.rows = a->rows, p.beams = a->beams, p.out_rows = a->out_rows, p.starts = a->starts, p.ends = a->ends;
  p.table_rows = a->table_rows, p.width = a->width * p.words, p.table_s0 = a->table_stride0 * p.words;
  p.rows_s0 = a->rows_stride0, p.beams_s0 = a->beams_stride0, p.out_rows_s0 = a->out_rows_stride0;
  p.from = a->from, p.to = a->to;
  p.rows_64 = a->rows_64, p.beams_64 = a->beams_64, p.out_rows_64 = a->out_rows_64, p.starts_64 = a->starts_64, p.ends_64 = a->ends_64;
  for (p.shift = 12; pow2_at_least(a->to, 1) << p.shift > ft::REORDER_WORDS * ft::BEAM_THREADS;) --p.shift;
  const int64_t chunks = (p.width + (1 << p.shift) - 1) >> p.shift;
  FT_CUDA_OK(launch_early(ft::beam_reorder_kernel, dim3((unsigned)chunks, (unsigned)a->batch), ft::BEAM_THREADS, 0, static_cast<cudaStream_t>(a->stream), p));
  count_launch();
  return FT_OK;
}

}  // extern "C"
