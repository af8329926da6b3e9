// pf_pages.h — blocks and tokens that move within a cache, in all its layers at once: the
// arguments that their entry points (pf_pages.cpp) hand to their kernels (pf_pages.hip).
#pragma once

#include "pf_paged.h"

namespace pf {

// First block's K and V segment of a layer.
struct LayerView {
  uint64_t k, v;
};

struct ForkParams {
  const LayerView* layers;
  PagedView pages;  // of every layer, k and v aside
  uint32_t num_layers;
  uint32_t segment_chunks;  // 16-byte chunks of a block's K (or V)
  uint32_t parts;           // workgroups of one of them
  // A copy: child i's block, from blocks[i] to new_blocks[i].
  const int32_t* blocks;
  // A fork: the parents' table and lengths, and each child's parent.
  const int32_t* table;
  const int32_t* seq_lens;
  const int32_t* parents;
  int32_t* out_table;
  uint64_t table_stride, out_stride;
  uint32_t width, num_seqs;
  const int32_t* new_blocks;
  uint32_t num_children;
};

struct CompactParams {
  const LayerView* layers;
  PagedView pages;
  uint32_t num_layers;
  const int32_t* table;
  const int32_t* out_table;
  uint64_t table_stride, out_stride;
  uint32_t width, num_seqs;
  const int32_t* kept;         // [total]
  const int32_t* kept_starts;  // [num_seqs + 1]
  const int32_t* first;        // [num_seqs], or null: 0
  int32_t* out_lens;           // [num_seqs], or null
  uint32_t total;
  // The launch (plan_compact): a token's 16-byte columns go in `strips` workgroups of
  // 2^cols_shift, its scales in `scale_strips`; a sequence's tokens in `turns` workgroups
  // that take chunks in turn (1 in place, where a chunk is read before it is overwritten by
  // the next).
  uint32_t cols_shift, strips, scale_strips, turns;
  bool few;  // at most kCompactFew tokens of a sequence are said to move
};

constexpr uint32_t kPagesThreads = 256;
constexpr uint32_t kForkChunks = 4;     // of a thread
constexpr uint32_t kCompactTokens = 8;  // of a thread
constexpr uint32_t kMinShift = 3, kMaxShift = 7;

inline uint32_t compact_columns(const PagedView& p) {
  return p.heads * p.dim * (p.type == PF_KV_BF16 || p.type == PF_KV_FP16 ? 2 : 1) / 16;
}
// Tokens of a workgroup's chunk.
inline uint32_t compact_chunk(uint32_t cols_shift) {
  return (kPagesThreads >> cols_shift) * kCompactTokens;
}
inline uint64_t compact_grid(const CompactParams& p) {
  return static_cast<uint64_t>(p.num_seqs) * p.num_layers * 2 * (p.strips + p.scale_strips) *
         p.turns;
}

// Tokens up to which a sequence's moves are few: one chunk, whose launch is all latency.
constexpr uint64_t kCompactFew = 16;

// Columns of a strip: a power of two from kMinShift on.  A token-major row of 8 heads of 128 is 128
// of them, 2 KB that lie together, and moves best whole: 2,500 of 5,000 tokens in 32 layers (bf16)
// in strips of 16, 32, 64 and 128 columns 139, 135, 131 and 129 us, 4 of each of 32 sequences 27,
// 15.5, 9.7 and 8.4.  In place, though, a strip's tokens move one chunk after another, and strips
// are all there is to fill the chip: 2,400 of 4,800 tokens of one sequence (the same layers) 131,
// 134, 202 and 380 us, of four 529, 507, 511 and 508 (their bytes 123 and 491).  To other blocks the
// chunks go to so many workgroups that 8,192 are at work: 2,048 did in 131.
inline void plan_compact(CompactParams* p, uint64_t most, bool in_place) {
  const uint32_t columns = compact_columns(p->pages);
  const bool codes = p->pages.type == PF_KV_E4M3 || p->pages.type == PF_KV_INT8;
  if (most == 0 || most > p->total) most = p->total;
  p->turns = 1;
  auto cut = [&](uint32_t shift) {
    const uint32_t cols = 1u << shift;
    p->cols_shift = shift;
    p->strips = (columns + cols - 1) / cols;
    p->scale_strips = codes ? (p->pages.heads + cols - 1) / cols : 0;
  };
  uint32_t whole = kMinShift;
  while (whole < kMaxShift && (1u << whole) < columns) ++whole;
  cut(whole);
  p->few = most <= kCompactFew;
  if (p->few) return;
  if (in_place) {
    if (whole > 5) cut(5);
    if (whole > 4 && compact_grid(*p) < 1024) cut(4);
    return;
  }
  const uint64_t chunks = (most + compact_chunk(p->cols_shift) - 1) / compact_chunk(p->cols_shift);
  while (p->turns * 2 <= chunks && compact_grid(*p) < 8192) p->turns *= 2;
}

hipError_t launch_fork(const ForkParams& p, hipStream_t stream);
hipError_t launch_compact(const CompactParams& p, hipStream_t stream);

}  // namespace pf
