// pf_paged_args.h — the checks of arguments that the paged-cache operators' entry points
// share (pf_paged.cpp, pf_rotary.cpp, pf_pages.cpp).
#pragma once

#include "pf_common.h"
#include "pf_paged.h"

namespace pf {

constexpr uint64_t kMaxTokens = 1ull << 31;  // of a sequence, and rows of a call

inline bool is_row_type(uint32_t t) { return t == PF_KV_BF16 || t == PF_KV_FP16; }
inline bool is_code_type(uint32_t t) { return t == PF_KV_E4M3 || t == PF_KV_INT8; }

inline int invalid(const std::string& msg) { return fail(PF_ERR_INVALID_ARGUMENT, msg); }

inline int segment_bytes(uint32_t block_size, uint32_t heads, uint32_t dim, uint32_t type,
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
  static constexpr int kMost = 16;  // of any call
  struct {
    const char* what;
    uint64_t addr, bytes;
    int device;
  } list_[kMost];
  int n_ = 0;
};

// Checks the pages and describes them for the kernels.
inline int view_pages(const pf_kv_pages* p, Ranges& ranges, PagedView* out) {
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
inline int view_rows(const pf_kv_rows& r, const char* what, uint64_t n, uint32_t heads,
                     uint32_t dim, bool written, Ranges& ranges, RowsView* out, bool* aligned) {
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

inline int add_array(const char* what, uint64_t addr, uint64_t bytes, uint64_t align,
                     Ranges& ranges) {
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

// No exception leaves an entry point (an error text may fail to allocate).
template <class F>
int guarded(F&& f) {
  try {
    return f();
  } catch (...) {
    return PF_ERR_STORAGE;
  }
}

}  // namespace pf
