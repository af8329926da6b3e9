// pf_paged.cpp — entry points of the paged-cache operators: argument checks, and
// the launches (pf_paged.hip, pf_attend_*.hip, pf_shared_*.hip).
#include <algorithm>
#include <cmath>

#include "pf_paged_args.h"

struct pf_attend_workspace {
  int device = 0;
  uint64_t data = 0;
  uint64_t bytes = 0;
};

namespace pf {

namespace {

int move_rows(bool write, const pf_kv_pages* pages, const pf_kv_rows* k, const pf_kv_rows* v,
              uint64_t slots, uint64_t n, pf_stream stream) {
  Ranges ranges;
  PagedView pv;
  if (int rc = view_pages(pages, ranges, &pv)) return rc;
  if (!k || !v) return invalid("null rows");
  if (k->type != v->type) return invalid("K and V rows differ in type");
  if (is_row_type(pv.type) && is_row_type(k->type) && pv.type != k->type)
    return invalid("16-bit pages hold the rows' own type");
  if (n == 0) return PF_OK;
  if (!write && k->data == v->data) return invalid("K and V rows overlap");
  if (n >= kMaxTokens) return invalid("too many rows");
  RowsView kv, vv;
  bool aligned = true;
  if (int rc = view_rows(*k, "K rows", n, pv.heads, pv.dim, !write, ranges, &kv, &aligned))
    return rc;
  if (int rc = view_rows(*v, "V rows", n, pv.heads, pv.dim, !write, ranges, &vv, &aligned))
    return rc;
  if (int rc = add_array("slots", slots, n * 8, 8, ranges)) return rc;
  if (int rc = ranges.check()) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  OnDevice on;
  if (int rc = on.enter(s, ranges)) return rc;
  const int64_t* at = reinterpret_cast<const int64_t*>(slots);
  const uint32_t rows = static_cast<uint32_t>(n);
  PF_HIP(write ? launch_kv_write(pv, kv, vv, k->type, at, rows, aligned, s)
               : launch_kv_read(pv, kv, vv, k->type, at, rows, aligned, s));
  return PF_OK;
}

// `shared`: the groups of sequences that share their first tokens, or null.
int attend(const pf_kv_pages* pages, const pf_attend_args* a, const pf_shared_args* shared,
           pf_attend_workspace* ws, pf_stream stream) {
  Ranges ranges;
  AttendParams p{};
  if (int rc = view_pages(pages, ranges, &p.pages)) return rc;
  const PagedView& pv = p.pages;
  if (!a) return invalid("null arguments");
  if (!is_row_type(a->q.type) || a->q.type != a->out.type)
    return invalid("q and out are of one type, bf16 or fp16");
  if (is_row_type(pv.type) && pv.type != a->q.type)
    return invalid("16-bit pages hold the rows' own type");
  if (a->num_q_heads == 0 || a->num_q_heads % pv.heads)
    return invalid(strf("%u query heads are no multiple of %u KV heads", a->num_q_heads, pv.heads));
  if (a->window && !a->causal) return invalid("a window needs causal attention");
  p.scale_log2 = static_cast<float>(std::fabs(a->scale) * 1.4426950408889634);
  if (!std::isfinite(p.scale_log2)) return invalid("the scale is not finite");
  if (a->num_seqs == 0 || a->num_rows == 0) return PF_OK;
  if (a->table_width == 0) return invalid("the block table has no entries");
  if (static_cast<uint64_t>(a->table_width) * pv.block_size > kMaxTokens - kAttendSlack)
    return invalid("the block table spans more than 2^31 - 65536 tokens");
  if (a->table_stride < a->table_width && a->num_seqs > 1)
    return invalid("rows of the block table overlap");
  if (a->num_seqs >= (1u << 24) || a->num_rows >= kMaxTokens / a->num_q_heads)
    return invalid("too many rows");
  bool aligned = true;
  if (int rc = view_rows(a->q, "q", a->num_rows, a->num_q_heads, pv.dim, false, ranges, &p.q,
                         &aligned))
    return rc;
  if (int rc = view_rows(a->out, "out", a->num_rows, a->num_q_heads, pv.dim, true, ranges, &p.out,
                         &aligned))
    return rc;
  uint64_t entries = 0;
  if (__builtin_mul_overflow(static_cast<uint64_t>(a->num_seqs) - 1, a->table_stride, &entries) ||
      entries > (1ull << 40))
    return invalid("the block table's strides overflow");
  entries += a->table_width;
  if (int rc = add_array("block table", a->block_table, entries * 4, 4, ranges)) return rc;
  if (int rc = add_array("seq_lens", a->seq_lens, a->num_seqs * 4ull, 4, ranges)) return rc;
  if (int rc = add_array("query_starts", a->query_starts, (a->num_seqs + 1ull) * 4, 4, ranges))
    return rc;
  if (a->lse)
    if (int rc = add_array("lse", a->lse, a->num_rows * a->num_q_heads * 4, 4, ranges)) return rc;
  const uint32_t groups = shared ? shared->num_groups : 0;
  if (groups) {
    if (groups >= (1u << 24)) return invalid("too many groups");
    if (int rc = add_array("group_starts", shared->group_starts, (groups + 1ull) * 4, 4, ranges))
      return rc;
    if (int rc = add_array("shared_lens", shared->shared_lens, groups * 4ull, 4, ranges)) return rc;
    p.group_starts = reinterpret_cast<const int32_t*>(shared->group_starts);
    p.shared_lens = reinterpret_cast<const int32_t*>(shared->shared_lens);
    p.num_groups = groups;
  }
  if (int rc = ranges.check()) return rc;
  p.block_table = reinterpret_cast<const int32_t*>(a->block_table);
  p.table_stride = a->table_stride;
  p.seq_lens = reinterpret_cast<const int32_t*>(a->seq_lens);
  p.query_starts = reinterpret_cast<const int32_t*>(a->query_starts);
  p.lse = reinterpret_cast<float*>(a->lse);
  p.num_rows = static_cast<uint32_t>(a->num_rows);
  p.q_heads = a->num_q_heads;
  p.group = a->num_q_heads / pv.heads;
  p.num_seqs = a->num_seqs;
  p.table_width = a->table_width;
  // A window as long as the table hides nothing.
  const uint32_t room = a->table_width * pv.block_size;  // checked above
  p.window = a->window >= room ? 0 : a->window;
  p.causal = a->causal != 0;
  // The kernels hide a score by -infinity, which a scale of 0 would turn into NaN; this
  // one leaves every weight at 1 as 0 does.
  if (p.scale_log2 < 1e-37f) p.scale_log2 = 1e-37f;
  p.q_sign = a->scale < 0 ? 0x80008000u : 0;
  p.aligned = aligned;
  while (p.unit_shift < 4 && !(pv.block_size >> p.unit_shift & 1u)) ++p.unit_shift;
  const uint64_t work = ws ? ws->data : 0, bytes = ws ? ws->bytes : 0;
  // More rows than the sequences can have are not all theirs.
  const uint64_t most_new = a->max_query_len ? a->max_query_len : a->num_rows;
  const uint64_t rows = a->num_rows <= a->num_seqs * most_new ? a->num_rows : 0;
  const bool joined = groups && plan_shared(&p, a->max_query_len, shared->max_shared_len,
                                            shared->max_own_len, work, bytes, rows);
  uint64_t grid = 0;
  if (joined) {
    grid = std::max(shared_grid(p), shared_join_grid(p));
  } else {
    uint64_t longest = a->max_seq_len;
    if (shared && shared->max_shared_len && shared->max_own_len) {
      const uint64_t both = static_cast<uint64_t>(shared->max_shared_len) + shared->max_own_len;
      longest = longest ? std::min(longest, both) : both;
    }
    plan_attend(&p, a->max_query_len, longest, work, bytes);
    const uint64_t left = p.many_units - p.many_whole;
    grid = std::max({static_cast<uint64_t>(p.num_seqs) * p.few_splits,
                     p.many_whole + left * p.many_splits,
                     left * (p.many_rows / 32) * (padded_dim(pv.dim) / 32)}) *
           pv.heads;
  }
  if (grid > 0x7fffffffull) return invalid("too many rows");
  hipStream_t s = static_cast<hipStream_t>(stream);
  OnDevice on;
  if (int rc = on.enter(s, ranges)) return rc;
  int dev = 0;
  PF_HIP(hipGetDevice(&dev));
  if (ws && ws->device != dev)
    return invalid(strf("the workspace is on device %d, the stream on device %d", ws->device, dev));
  if (joined)
    PF_HIP(a->q.type == PF_KV_BF16 ? launch_shared_bf16(p, s) : launch_shared_fp16(p, s));
  else
    PF_HIP(a->q.type == PF_KV_BF16 ? launch_attend_bf16(p, s) : launch_attend_fp16(p, s));
  return PF_OK;
}

}  // namespace

}  // namespace pf

extern "C" {

int pf_kv_segment_bytes(uint32_t block_size, uint32_t num_heads, uint32_t head_dim, uint32_t type,
                        uint64_t* out) {
  return pf::guarded([&] {
    if (!out) return pf::invalid("null output");
    return pf::segment_bytes(block_size, num_heads, head_dim, type, out);
  });
}

int pf_kv_write(const pf_kv_pages* pages, const pf_kv_rows* k, const pf_kv_rows* v, uint64_t slots,
                uint64_t num_rows, pf_stream stream) {
  return pf::guarded([&] { return pf::move_rows(true, pages, k, v, slots, num_rows, stream); });
}

int pf_kv_read(const pf_kv_pages* pages, const pf_kv_rows* k, const pf_kv_rows* v, uint64_t slots,
               uint64_t num_rows, pf_stream stream) {
  return pf::guarded([&] { return pf::move_rows(false, pages, k, v, slots, num_rows, stream); });
}

int pf_attend_workspace_create(int device, uint64_t bytes, pf_attend_workspace** out) {
  return pf::guarded([&]() -> int {
    if (!out) return pf::invalid("null output");
    *out = nullptr;
    if (bytes == 0) return pf::fail(PF_ERR_ZERO_SIZE, "the workspace has no bytes");
    int prev = 0;
    const bool had = hipGetDevice(&prev) == hipSuccess;
    const int rc = pf_init(device);
    void* p = nullptr;
    hipError_t e = rc == PF_OK ? hipMalloc(&p, bytes) : hipSuccess;
    if (p) {  // its counts start at 0
      e = hipMemset(p, 0, pf::workspace_counts(bytes) * pf::kCountStride * 4);
      if (e == hipSuccess) e = hipDeviceSynchronize();
    }
    if (e != hipSuccess && p) (void)hipFree(p);
    if (had && prev != device) (void)hipSetDevice(prev);
    if (rc != PF_OK) return rc;
    if (e != hipSuccess) return pf::hip_fail(e, "pf_attend_workspace_create");
    *out = new pf_attend_workspace{device, reinterpret_cast<uint64_t>(p), bytes};
    return PF_OK;
  });
}

int pf_attend_workspace_destroy(pf_attend_workspace* workspace) {
  return pf::guarded([&]() -> int {
    if (!workspace) return PF_OK;
    (void)hipFree(reinterpret_cast<void*>(workspace->data));
    delete workspace;
    return PF_OK;
  });
}

int pf_kv_attend(const pf_kv_pages* pages, const pf_attend_args* args,
                 pf_attend_workspace* workspace, pf_stream stream) {
  return pf::guarded([&] { return pf::attend(pages, args, nullptr, workspace, stream); });
}

int pf_kv_attend_shared(const pf_kv_pages* pages, const pf_attend_args* args,
                        const pf_shared_args* shared, pf_attend_workspace* workspace,
                        pf_stream stream) {
  return pf::guarded([&]() -> int {
    if (!shared) return pf::invalid("null groups");
    return pf::attend(pages, args, shared, workspace, stream);
  });
}

}  // extern "C"
