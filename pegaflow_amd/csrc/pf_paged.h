// pf_paged.h — the paged-cache operators' arguments, shared by their entry
// points (pf_paged.cpp) and kernels (pf_paged.hip, pf_attend.hip).
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstdint>

#include "../../include/pegaflow_hip.h"

namespace pf {

// A layer's pages as the kernels see them.  Token t of a block lies at
// block * block_bytes + t * token_bytes + head * head_bytes of its segment, and
// for 8-bit kinds its scale at scale_offset + (head * block_size + t) * 4.
struct PagedView {
  uint64_t k, v;         // first block's K and V segment
  uint64_t block_bytes;  // from one block to the next
  uint32_t num_blocks, block_size, heads, dim;
  uint32_t token_bytes, head_bytes, scale_offset;
  uint32_t type;     // PF_KV_*
  uint32_t div_mul;  // token / block_size, see page_of
  uint32_t div_shift;
};

// Multiplier and shift with which x * mul >> (31 + shift) == x / d for every x <
// 2^31: mul = ceil(2^(31 + shift) / d) with shift = ceil(log2 d) exceeds
// 2^(31 + shift) / d by less than 1 <= 2^shift / d, so x times the excess stays
// under 2^(31 + shift) / d, too little to reach the next quotient.
inline void set_division(uint32_t d, uint32_t* mul, uint32_t* shift) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  *mul = static_cast<uint32_t>(((1ull << (31 + s)) + d - 1) / d);
  *shift = s;
}

struct RowsView {
  uint64_t data;
  uint64_t token_stride, head_stride;  // elements
};

struct AttendParams {
  PagedView pages;
  RowsView q, out;
  const int32_t* block_table;
  uint64_t table_stride;
  const int32_t* seq_lens;
  const int32_t* query_starts;
  float* lse;  // [num_rows, q_heads], may be null
  uint32_t num_rows, q_heads, group, num_seqs, table_width;
  uint32_t window;  // 0: none
  uint32_t causal;
  float scale_log2;  // score scale times log2(e)
};

hipError_t launch_kv_write(const PagedView& pages, const RowsView& k, const RowsView& v,
                           uint32_t row_type, const int64_t* slots, uint32_t n, bool aligned,
                           hipStream_t stream);
hipError_t launch_kv_read(const PagedView& pages, const RowsView& k, const RowsView& v,
                          uint32_t row_type, const int64_t* slots, uint32_t n, bool aligned,
                          hipStream_t stream);
hipError_t launch_attend(const AttendParams& p, uint32_t row_type, hipStream_t stream);

}  // namespace pf
