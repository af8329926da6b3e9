// pf_paged.cpp — entry points of the paged-cache operators: argument checks, and
// the launches (pf_paged.hip, pf_attend_*.hip).
#include <algorithm>
#include <cmath>

#include "pf_common.h"
#include "pf_paged.h"

struct pf_attend_workspace {
  int device = 0;
  uint64_t data = 0;
  uint64_t bytes = 0;
};

namespace pf {

namespace {

constexpr uint64_t kMaxTokens = 1ull << 31;  // of a sequence, and rows of a call

bool is_row_type(uint32_t t) { return t == PF_KV_BF16 || t == PF_KV_FP16; }
bool is_code_type(uint32_t t) { return t == PF_KV_E4M3 || t == PF_KV_INT8; }

int invalid(const std::string& msg) { return fail(PF_ERR_INVALID_ARGUMENT, msg); }

int segment_bytes(uint32_t block_size, uint32_t heads, uint32_t dim, uint32_t type,
                  uint64_t* out) {
  if (!is_row_type(type) && !is_code_type(type))
    return invalid(strf("unknown KV type %u", type));
  if (block_size == 0 || heads == 0) return invalid("pages need block_size and num_heads > 0");
  if (dim == 0 || dim % 16 != 0 || dim > PF_KV_MAX_HEAD_DIM)
    return invalid(strf("head_dim %u is not a multiple of 16 up to %u", dim,
                        (unsigned)PF_KV_MAX_HEAD_DIM));
  const uint64_t tokens = static_cast<uint64_t>(block_size) * heads;
  if (tokens > (1ull << 22))
    return invalid(strf("block_size %u x num_heads %u is too large", block_size, heads));
  const uint64_t n = tokens * (is_code_type(type) ? dim + 4 : dim * 2);
  *out = (n + 15) / 16 * 16;
  return PF_OK;
}

// The ranges that a call's kernels touch: each inside one device or pinned
// allocation, checked after everything else that the arguments say, and on the stream's
// device (a kernel that reads another device's memory faults).
class Ranges {
 public:
  void add(const char* what, uint64_t addr, uint64_t bytes) { list_[n_++] = {what, addr, bytes, -1}; }
  int check() {
    RangeCache cache;
    for (int i = 0; i < n_; ++i) {
      if (!cache.check(list_[i].addr, list_[i].bytes))
        return invalid(strf("%s: range [0x%llx, +%llu) is not inside one device or pinned "
                            "allocation",
                            list_[i].what, (unsigned long long)list_[i].addr,
                            (unsigned long long)list_[i].bytes));
      list_[i].device = cache.device();
    }
    return PF_OK;
  }
  int check_device(int device) const {
    for (int i = 0; i < n_; ++i) {
      int at = list_[i].device;
      if (at < 0) {  // pinned, which every device reads, or another process's
        hipPointerAttribute_t attr;
        const hipError_t e =
            hipPointerGetAttributes(&attr, reinterpret_cast<void*>(list_[i].addr));
        if (e != hipSuccess) (void)hipGetLastError();  // clear the probe's error
        if (e != hipSuccess || attr.type != hipMemoryTypeDevice) continue;
        at = attr.device;
      }
      if (at != device)
        return invalid(
            strf("%s: on device %d, the stream on device %d", list_[i].what, at, device));
    }
    return PF_OK;
  }

 private:
  struct {
    const char* what;
    uint64_t addr, bytes;
    int device;
  } list_[8];
  int n_ = 0;
};

// Checks the pages and describes them for the kernels.
int view_pages(const pf_kv_pages* p, Ranges& ranges, PagedView* out) {
  if (!p) return invalid("null pages");
  uint64_t need = 0;
  if (int rc = segment_bytes(p->block_size, p->num_heads, p->head_dim, p->type, &need)) return rc;
  if (p->order != PF_KV_TOKEN_MAJOR && p->order != PF_KV_HEAD_MAJOR)
    return invalid(strf("unknown order %u of the pages", p->order));
  const pf_kv_layout& l = p->layout;
  if (l.num_blocks == 0 || l.num_blocks >= kMaxTokens)
    return invalid("pages need between 1 and 2^31 - 1 blocks");
  if (l.segments != 1 && l.segments != 2)
    return invalid(strf("pages need one or two segments, got %llu",
                        (unsigned long long)l.segments));
  const uint64_t segment = l.segments == 2 ? l.bytes_per_block : l.bytes_per_block / 2;
  const uint64_t v_offset = l.segments == 2 ? l.kv_stride_bytes : segment;
  if (segment < need)
    return invalid(strf("a segment of %llu bytes cannot hold K or V of a block (%llu bytes)",
                        (unsigned long long)segment, (unsigned long long)need));
  if (l.data_ptr % 16 || segment % 16 || v_offset % 16 ||
      (l.segments == 1 && l.bytes_per_block % 32))
    return invalid("pages are not 16-byte aligned");
  uint64_t end = 0, span = 0;
  if (__builtin_mul_overflow(l.num_blocks, l.bytes_per_block, &span) ||
      __builtin_add_overflow(span, l.segments == 2 ? v_offset : 0, &end) || end > l.size_bytes)
    return invalid("the pages exceed the registered memory");
  if (l.segments == 2 && v_offset < span) return invalid("K and V segments of the pages overlap");
  ranges.add("pages", l.data_ptr, end);
  const uint32_t value = is_code_type(p->type) ? 1 : 2;
  const bool token_major = p->order == PF_KV_TOKEN_MAJOR;
  out->k = l.data_ptr;
  out->v = l.data_ptr + v_offset;
  out->block_bytes = l.bytes_per_block;
  out->num_blocks = static_cast<uint32_t>(l.num_blocks);
  out->block_size = p->block_size;
  out->heads = p->num_heads;
  out->dim = p->head_dim;
  out->token_bytes = (token_major ? p->num_heads : 1) * p->head_dim * value;
  out->head_bytes = (token_major ? 1 : p->block_size) * p->head_dim * value;
  out->scale_offset = p->block_size * p->num_heads * p->head_dim * value;
  out->type = p->type;
  set_division(p->block_size, &out->div_mul, &out->div_shift);
  return PF_OK;
}

// Checks rows of `n` tokens and `heads` heads; *aligned is cleared where they
// cannot move by 16 bytes.
int view_rows(const pf_kv_rows& r, const char* what, uint64_t n, uint32_t heads, uint32_t dim,
              bool written, Ranges& ranges, RowsView* out, bool* aligned) {
  if (!is_row_type(r.type)) return invalid(strf("%s: rows are bf16 or fp16", what));
  if (r.data % 2) return invalid(strf("%s: unaligned address", what));
  uint64_t a = 0, b = 0, last = 0, bytes = 0;
  if (__builtin_mul_overflow(n - 1, r.token_stride, &a) ||
      __builtin_mul_overflow(static_cast<uint64_t>(heads) - 1, r.head_stride, &b) ||
      __builtin_add_overflow(a, b, &last) || __builtin_add_overflow(last, dim, &last) ||
      __builtin_mul_overflow(last, uint64_t{2}, &bytes))
    return invalid(strf("%s: strides overflow", what));
  if (written) {
    // Dimensions of one index have no stride.
    const bool by_token = n > 1, by_head = heads > 1;
    const uint64_t t = r.token_stride, h = r.head_stride;
    const bool apart =
        (!by_token && !by_head) || (!by_head && t >= dim) || (!by_token && h >= dim) ||
        (by_token && by_head && ((h >= dim && t >= b + dim) || (t >= dim && h >= a + dim)));
    if (!apart) return invalid(strf("%s: rows overlap", what));
  }
  ranges.add(what, r.data, bytes);
  if (r.data % 16 || (n > 1 && r.token_stride % 8) || (heads > 1 && r.head_stride % 8))
    *aligned = false;
  *out = {r.data, r.token_stride, r.head_stride};
  return PF_OK;
}

int add_array(const char* what, uint64_t addr, uint64_t bytes, uint64_t align, Ranges& ranges) {
  if (addr % align) return invalid(strf("%s: unaligned address", what));
  ranges.add(what, addr, bytes);
  return PF_OK;
}

// Makes the stream's device current while a call launches (the null stream's is the
// current one).  Every range must be there.
class OnDevice {
 public:
  int enter(hipStream_t stream, const Ranges& ranges) {
    int dev = 0;
    PF_HIP(hipGetDevice(&prev_));
    if (stream)
      PF_HIP(hipStreamGetDevice(stream, &dev));
    else
      dev = prev_;
    if (int rc = ranges.check_device(dev)) return rc;
    if (dev != prev_) {
      PF_HIP(hipSetDevice(dev));
      moved_ = true;
    }
    (void)hipGetLastError();
    return PF_OK;
  }
  ~OnDevice() {
    if (moved_) (void)hipSetDevice(prev_);
  }

 private:
  int prev_ = 0;
  bool moved_ = false;
};

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

int attend(const pf_kv_pages* pages, const pf_attend_args* a, pf_attend_workspace* ws,
           pf_stream stream) {
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
  plan_attend(&p, a->max_query_len, a->max_seq_len, ws ? ws->data : 0, ws ? ws->bytes : 0);
  const uint64_t left = p.many_units - p.many_whole;
  const uint64_t grid = std::max({static_cast<uint64_t>(p.num_seqs) * p.few_splits,
                                  p.many_whole + left * p.many_splits,
                                  left * (p.many_rows / 32) * (padded_dim(pv.dim) / 32)}) *
                        pv.heads;
  if (grid > 0x7fffffffull) return invalid("too many rows");
  hipStream_t s = static_cast<hipStream_t>(stream);
  OnDevice on;
  if (int rc = on.enter(s, ranges)) return rc;
  int dev = 0;
  PF_HIP(hipGetDevice(&dev));
  if (ws && ws->device != dev)
    return invalid(strf("the workspace is on device %d, the stream on device %d", ws->device, dev));
  PF_HIP(a->q.type == PF_KV_BF16 ? launch_attend_bf16(p, s) : launch_attend_fp16(p, s));
  return PF_OK;
}

// No exception leaves an entry point (an error text may fail to allocate).
template <class F>
int guarded(F&& f) {
  try {
    return f();
  } catch (...) {
    return PF_ERR_STORAGE;
  }
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
  return pf::guarded([&] { return pf::attend(pages, args, workspace, stream); });
}

}  // extern "C"
