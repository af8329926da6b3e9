// pf_paged.h — the paged-cache operators' arguments, shared by their entry
// points (pf_paged.cpp) and kernels (pf_paged.hip, pf_attend_*.hip).
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
  float scale_log2;   // |score scale| times log2(e), above 0
  uint32_t q_sign;    // flips the sign of two 16-bit values where the scale is negative
  uint32_t aligned;   // q and out move by 16 bytes
  uint32_t unit_shift;  // 2^unit_shift aligned tokens, at most 16, share a block
  // The launch (plan_attend): sequences of up to few_rows rows of a KV head go to the
  // kernel for few, in few_splits shares of few_piece tokens (0: none do) of at most
  // few_rows_most rows, the others in many_units tiles of many_rows rows, of which those
  // from many_whole on go in many_splits shares of many_piece tokens.
  uint32_t few_rows, few_splits, few_piece, few_rows_most;
  uint32_t many_units, many_rows, many_whole, many_splits, many_piece;
  float *few_o, *few_ml, *many_o, *many_ml;  // shares, in the workspace
  uint32_t* few_count;  // finished shares of each sequence and head, 0 between calls
};

constexpr uint32_t kFewRows = 16;        // of attend_few_kernel's tile
constexpr uint32_t kManyRows = 128;      // of attend_many_kernel's, or where rows are many
constexpr uint32_t kWideRows = 256;      // and heads have up to kWideMaxDim values
constexpr uint32_t kWideMaxDim = 128;
constexpr uint32_t kFewMaxSplits = 192;
// A count of finished shares has a 128-byte line of its own: adds to one line run one
// after another.  The first kCounts of them (or a sixteenth of a small workspace) are at
// the workspace's start.
constexpr uint32_t kCountStride = 32;
constexpr uint64_t kCounts = 8192;
inline uint64_t workspace_counts(uint64_t bytes) {
  const uint64_t n = bytes / 16 / (kCountStride * 4);
  return n < kCounts ? n : kCounts;
}
constexpr uint32_t kAttendSlack = 1u << 16;  // tokens that a kernel's counting may run past the end

// Head sizes that the kernels are built for.
inline uint32_t padded_dim(uint32_t dim) {
  return dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128 : dim <= 192 ? 192 : 256;
}

// Tokens of a share of attend_few_kernel: `units` sequences and heads, the longest of
// `longest` tokens.  (Measured with 128 values a head, 4 rows, in us.)
//
// The chip holds 512 of its workgroups at once, and a launch of a few more than that
// takes twice as long: 384 units of 1,000 tokens whole 45.0, in two shares 55.2; 512 of
// 2,000 whole 97.3, in two 108.3; 128 of 4,000 in 2, 4 and 8 shares 55.4, 56.5 and 59.8.
// Many launches' worth of shares, though, even out lengths that the host does not
// know: 512 of up to 16,000 tokens, on average half, in shares of 1,024 tokens 226, of
// 8,192 277.  Where units are few, a share of s tokens takes about 7.5 ns a token and
// the join 200 to 280 ns a share, so shares of sqrt(37 * longest) are best: one sequence
// of 10,000 tokens and 8 heads in shares of 256, 512, 1,024 and 2,048 takes 20.5, 16.1,
// 18.7 and 27.1; of 30,000 (8-bit) 36.7, 26.0, 20.9 and 24.1; of 3,000 12.0, 14.2, 18.1
// and 22.4.
inline uint64_t few_piece(uint64_t units, uint64_t longest) {
  constexpr uint64_t kSlots = 512, kEven = 1024;
  if (units * longest >= 4 * kSlots * kEven) return kEven;
  const uint64_t most = units < kSlots ? kSlots / units : 1;
  const uint64_t whole = (longest + most - 1) / most;
  uint64_t piece = 128;
  while (piece * piece < 37 * longest) piece += 128;
  return piece > whole ? piece : whole;
}

// Whether attend_many_kernel's tiles are of kWideRows rows: half the loads and writes to
// LDS for a product, but one workgroup a compute unit, so that lengths even out less.
// (Measured with 8 heads of 128 and a group of 4, in us, wide and not.)
//
// A sequence alone, from 512 rows and 4,096 tokens on: 8,192 new tokens 532 and 578, 130
// behind 4,000 34.0 and 34.6; 2,000 new ones 66 and 62, 300 22 and 19.  Several, where the
// chip is filled twice or more: 9 of up to 701 behind 4,100 (int8) 297 and 312, 16 of 480
// behind 4,000 245 and 268, 8 of 960 (e4m3) 342 and 335; below that 8 of 240 behind 10,000
// 324 and 288.
inline bool wide_tiles(uint64_t seqs, uint64_t rows, uint64_t heads, uint64_t dim,
                       uint64_t longest) {
  constexpr uint64_t kLong = 4096, kUnits = 512;
  if (dim > kWideMaxDim || longest < kLong) return false;
  return seqs == 1 ? rows >= 2 * kWideRows
                   : rows >= kWideRows * seqs && rows / kWideRows * heads >= kUnits;
}

// Shapes the launch of a batch whose longest query has `most_new` rows and longest
// sequence `longest` tokens, joining in `bytes` of workspace at `ws`.  `longest` may be wrong:
// every row is attended whatever it says.  `most_new` may be loose but not too small: rows
// that a sequence has beyond it may stay as they were.
inline void plan_attend(AttendParams* p, uint64_t most_new, uint64_t longest, uint64_t ws,
                        uint64_t bytes) {
  constexpr uint64_t kCus = 256;
  const uint64_t heads = p->pages.heads, group = p->group, dim = padded_dim(p->pages.dim);
  const uint64_t room = static_cast<uint64_t>(p->table_width) * p->pages.block_size;
  if (longest == 0 || longest > room) longest = room;
  if (most_new == 0 || most_new > p->num_rows) most_new = p->num_rows;
  if (p->window && p->window + most_new < longest) longest = p->window + most_new;
  auto ceil_div = [](uint64_t a, uint64_t b) { return (a + b - 1) / b; };
  const bool all_few = most_new * group <= kFewRows;
  const bool any_few = all_few || (p->num_seqs > 1 && group <= kFewRows);
  p->few_rows = any_few && !all_few ? kFewRows : 0;
  p->few_splits = p->few_piece = 0;
  p->many_units = p->many_whole = p->many_splits = p->many_piece = 0;
  const uint64_t counts = workspace_counts(bytes);
  uint64_t at = ws + counts * kCountStride * 4;
  const uint64_t end = ws + bytes;
  p->few_count = reinterpret_cast<uint32_t*>(ws);
  if (any_few) {
    const uint64_t units = p->num_seqs * heads;
    p->few_rows_most = static_cast<uint32_t>(all_few ? most_new * group : kFewRows);
    const uint64_t slot = p->few_rows_most * (dim * 4 + 8);
    uint64_t piece = few_piece(units, longest);
    uint64_t splits = ceil_div(longest, piece);
    if (splits > kFewMaxSplits) splits = kFewMaxSplits;
    if (units > counts) splits = 1;
    if (splits * units * slot > end - at) splits = (end - at) / (units * slot);
    if (splits < 2) splits = 1;
    piece = ceil_div(ceil_div(longest, splits), 128) * 128;
    p->few_splits = static_cast<uint32_t>(splits);
    p->few_piece = static_cast<uint32_t>(piece);
    if (splits > 1) {
      const uint64_t n = units * splits * p->few_rows_most;
      p->few_o = reinterpret_cast<float*>(at);
      p->few_ml = reinterpret_cast<float*>(at + n * dim * 4);
      at += n * (dim * 4 + 8);
    }
  }
  if (!all_few) {
    const uint64_t rows = p->num_rows * group;
    const uint64_t seqs = p->num_seqs < p->num_rows ? p->num_seqs : p->num_rows;
    const uint64_t many = wide_tiles(seqs, rows, heads, dim, longest) ? kWideRows : kManyRows;
    const uint64_t tiles = seqs > 1 ? rows / many + seqs : ceil_div(rows, many);
    // The tiles that fill the chip, once or more, are passed over whole; those left over
    // are split among the workgroups that it holds at once, where they are long enough for
    // their join: the last tiles are those of the first rows, which attend little more than
    // what is cached.  2,100 rows of 32 heads behind 30,000 tokens took 1,156 us, whole
    // 1,627 (2,048 rows: 1,095); behind 4,000 216 and 251, 1,500 122 and 122, 1,000 106 and
    // 100; seven times 300 (8-bit) behind 10,000 435 and 595, 1,900 115 and 140; 2,500
    // behind 1,900 176 and 169.
    constexpr uint64_t kSplitCached = 1536;
    const uint64_t slots = kCus * (dim <= 128 && many == kManyRows ? 2 : 1);
    uint64_t whole = tiles * heads / slots * slots / heads;
    if (whole && longest < most_new + kSplitCached) whole = tiles;
    const uint64_t units = (tiles - whole) * heads;
    const uint64_t slot = many * (dim * 4 + 16);
    const uint64_t want = units && units < slots ? slots / units : 1;
    uint64_t piece = ceil_div(ceil_div(longest, want), 64) * 64;
    if (piece < 256) piece = 256;
    uint64_t splits = ceil_div(longest, piece);
    if (splits * units * slot > end - at) {
      splits = (end - at) / (units * slot);
      if (splits < 2) splits = 1;
      piece = ceil_div(ceil_div(longest, splits), 64) * 64;
    }
    if (splits == 1) whole = tiles;
    p->many_rows = static_cast<uint32_t>(many);
    p->many_whole = static_cast<uint32_t>(whole);
    p->many_units = static_cast<uint32_t>(tiles);
    p->many_splits = static_cast<uint32_t>(splits);
    p->many_piece = static_cast<uint32_t>(piece);
    if (splits > 1) {
      const uint64_t n = units * splits * many;
      p->many_o = reinterpret_cast<float*>(at);
      p->many_ml = reinterpret_cast<float*>(at + n * dim * 4);
    }
  }
}

hipError_t launch_kv_write(const PagedView& pages, const RowsView& k, const RowsView& v,
                           uint32_t row_type, const int64_t* slots, uint32_t n, bool aligned,
                           hipStream_t stream);
hipError_t launch_kv_read(const PagedView& pages, const RowsView& k, const RowsView& v,
                          uint32_t row_type, const int64_t* slots, uint32_t n, bool aligned,
                          hipStream_t stream);
hipError_t launch_attend_bf16(const AttendParams& p, hipStream_t stream);
hipError_t launch_attend_fp16(const AttendParams& p, hipStream_t stream);

}  // namespace pf
