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
};

constexpr uint32_t kPagesThreads = 256;
constexpr uint32_t kForkChunks = 4;     // of a thread
constexpr uint32_t kCompactTokens = 8;  // of a thread

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

inline void plan_compact(CompactParams* p, uint64_t most, bool in_place) {
  const uint32_t columns = compact_columns(p->pages);
  const bool codes = p->pages.type == PF_KV_E4M3 || p->pages.type == PF_KV_INT8;
  if (most == 0 || most > p->total) most = p->total;
  p->cols_shift = most <= 16 ? 7 : 4;
  const uint32_t cols = 1u << p->cols_shift;
  p->strips = (columns + cols - 1) / cols;
  p->scale_strips = codes ? (p->pages.heads + cols - 1) / cols : 0;
  p->turns = 1;
  if (in_place) return;
  const uint64_t chunks = (most + compact_chunk(p->cols_shift) - 1) / compact_chunk(p->cols_shift);
  while (p->turns * 2 <= chunks && compact_grid(*p) < 2048) p->turns *= 2;
}

hipError_t launch_fork(const ForkParams& p, hipStream_t stream);
hipError_t launch_compact(const CompactParams& p, hipStream_t stream);

}  // namespace pf
