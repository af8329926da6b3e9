// pf_pages.hip — blocks copied for forked sequences, and kept tokens moved together, in all
// layers of a cache by one launch.
//
// Bound by HBM (bytes are read once and written once, as they are) or, for a few blocks, by
// the launch and the chain of loads that leads to a block's place: parent, length, table
// entry.
#include <hip/hip_runtime.h>

#include "pf_paged_device.h"
#include "pf_pages.h"

namespace pf {

namespace {

constexpr uint32_t kThreads = kPagesThreads;
typedef __attribute__((address_space(1))) int32_t g_i32;

// Workgroups of a child, its K and V of each layer in `parts`; then one for each child's row
// of the table.
//
// 64 children in 32 layers (e4m3, 121 MB) take 18.5 to 20 us, 6 TB/s (part of it stays in the
// caches between calls), 4 in 12 layers 3.8.
template <bool FORK>
__global__ void __launch_bounds__(kThreads) fork_kernel(ForkParams p) {
  const uint32_t tid = threadIdx.x;
  const uint32_t copies = p.num_layers * 2 * p.parts;
  const bool row = FORK && blockIdx.x >= p.num_children * copies;
  const uint32_t child = row ? blockIdx.x - p.num_children * copies : blockIdx.x / copies;
  const int32_t to = p.new_blocks[child];
  int32_t from = -1;
  if constexpr (FORK) {
    const int32_t parent = p.parents[child];
    if (parent < 0 || parent >= static_cast<int32_t>(p.num_seqs)) return;
    const int32_t* entries = p.table + parent * p.table_stride;
    const uint32_t len = static_cast<uint32_t>(max(p.seq_lens[parent], 0));
    const uint32_t page = page_of(p.pages, len);
    const bool fresh = to >= 0 && to < static_cast<int32_t>(p.pages.num_blocks);
    if (row) {
      int32_t* out = p.out_table + child * p.out_stride;
      for (uint32_t i = tid; i < p.width; i += kThreads)
        out[i] = fresh && i == page ? to : entries[i];
      return;
    }
    if (!fresh || page >= p.width || len == page * p.pages.block_size) return;
    from = entries[page];
  } else {
    from = p.blocks[child];
  }
  if (static_cast<uint32_t>(from) >= p.pages.num_blocks ||
      static_cast<uint32_t>(to) >= p.pages.num_blocks || from == to)
    return;
  const uint32_t rest = blockIdx.x % copies, part = rest % p.parts, layer = rest / p.parts / 2;
  const uint64_t base = rest / p.parts % 2 ? p.layers[layer].v : p.layers[layer].k;
  const uint64_t src = base + static_cast<uint32_t>(from) * p.pages.block_bytes;
  const uint64_t dst = base + static_cast<uint32_t>(to) * p.pages.block_bytes;
  u32x4 x[kForkChunks];
  const uint32_t first = part * (kThreads * kForkChunks) + tid;
#pragma unroll
  for (uint32_t i = 0; i < kForkChunks; ++i) {
    const uint32_t c = first + i * kThreads;
    if (c < p.segment_chunks) x[i] = *reinterpret_cast<const g_u32x4*>(src + c * 16ull);
  }
#pragma unroll
  for (uint32_t i = 0; i < kForkChunks; ++i) {
    const uint32_t c = first + i * kThreads;
    if (c < p.segment_chunks) *reinterpret_cast<g_u32x4*>(dst + c * 16ull) = x[i];
  }
}

// A workgroup moves one strip of columns of one sequence's kept tokens, in chunks of
// kCompactTokens tokens a thread.  In place a chunk is in registers before any of it is
// written, and the next one's tokens lie behind all that this one writes: kept positions
// ascend, and none moves up.
//
// 2,500 of 5,000 tokens in 32 layers (bf16, 655 MB) take 129 us, 5.1 TB/s, what a large copy
// reaches; 4 of each of 32 sequences (21 MB) 7.7, of which the memory works 4.  Where much moves
// (STREAM) neither its bytes nor their copies are kept in the caches: 137 us otherwise.
template <uint32_t SHIFT, bool STREAM>
__global__ void __launch_bounds__(kThreads) compact_kernel(CompactParams p) {
  constexpr uint32_t kCols = 1u << SHIFT, kRows = kThreads / kCols;
  constexpr uint32_t kChunk = kRows * kCompactTokens;
  // Where the chunk's tokens lie and go, as a block's place and a position in it; a token
  // that does not move goes nowhere.  Three in turn: the next chunk's are found while a wave
  // may still write the one before this.
  __shared__ uint64_t from_at[3][kChunk], to_at[3][kChunk];
  __shared__ uint32_t from_off[3][kChunk], to_off[3][kChunk];
  constexpr uint64_t kNowhere = ~0ull;
  const PagedView& pg = p.pages;
  const uint32_t tid = threadIdx.x, strips = p.strips + p.scale_strips;
  uint32_t rest = blockIdx.x;
  const uint32_t turn = rest % p.turns;
  rest /= p.turns;
  const uint32_t strip = rest % strips;
  rest /= strips;
  const bool value = rest % 2;
  rest /= 2;
  const uint32_t layer = rest % p.num_layers, seq = rest / p.num_layers;
  const int32_t total = static_cast<int32_t>(p.total);
  const int32_t begin = min(max(p.kept_starts[seq], 0), total);
  const int32_t end = min(max(p.kept_starts[seq + 1], begin), total);
  const int32_t first = p.first ? max(p.first[seq], 0) : 0;
  if (p.out_lens && tid == 0 && turn == 0 && strip == 0 && !value && layer == 0)
    p.out_lens[seq] = first + (end - begin);
  const uint64_t base = value ? p.layers[layer].v : p.layers[layer].k;
  const int32_t* table = p.table + seq * p.table_stride;
  const int32_t* out_table = p.out_table + seq * p.out_stride;
  const uint32_t room = p.width * pg.block_size;

  // This thread's column: 16 bytes of a head's row, or a head's scale.
  const bool scales = strip >= p.strips;
  const uint32_t col = (scales ? strip - p.strips : strip) * kCols + tid % kCols;
  const uint32_t row_bytes = pg.dim * (pg.type == PF_KV_BF16 || pg.type == PF_KV_FP16 ? 2 : 1);
  uint64_t col_at;
  uint32_t by_token;
  bool mine;
  if (scales) {
    mine = col < pg.heads;
    col_at = base + pg.scale_offset + static_cast<uint64_t>(col) * pg.block_size * 4;
    by_token = 4;
  } else {
    const uint32_t head = col * 16 / row_bytes;
    mine = head < pg.heads;
    col_at = base + static_cast<uint64_t>(head) * pg.head_bytes + (col * 16 - head * row_bytes);
    by_token = pg.token_bytes;
  }

  const int32_t step = static_cast<int32_t>(kChunk * p.turns);
  static_assert(kChunk <= kThreads, "a thread for each token of a chunk");
  auto find = [&](int32_t j0, uint32_t buffer) {
    if (tid >= kChunk) return;
    const int32_t j = j0 + static_cast<int32_t>(tid);
    uint64_t at = kNowhere, to = kNowhere;
    uint32_t at_off = 0, new_off = 0;
    if (j < end) {
      const uint32_t old = static_cast<uint32_t>(p.kept[j]);
      const uint32_t now = static_cast<uint32_t>(first) + static_cast<uint32_t>(j - begin);
      if (old < room && now < room) {
        const uint32_t page = page_of(pg, old), new_page = page_of(pg, now);
        at_off = old - page * pg.block_size;
        new_off = now - new_page * pg.block_size;
        const uint32_t block = static_cast<uint32_t>(table[page]);
        const uint32_t new_block = static_cast<uint32_t>(out_table[new_page]);
        if (block < pg.num_blocks && new_block < pg.num_blocks &&
            (block != new_block || at_off != new_off)) {
          at = block * pg.block_bytes;
          to = new_block * pg.block_bytes;
        }
      }
    }
    from_at[buffer][tid] = at;
    to_at[buffer][tid] = to;
    from_off[buffer][tid] = at_off;
    to_off[buffer][tid] = new_off;
  };
  int32_t j0 = begin + static_cast<int32_t>(kChunk * turn);
  if (j0 >= end) return;
  find(j0, 0);
  __syncthreads();
  uint32_t buffer = 0;
  for (; j0 < end; j0 += step) {
    const uint32_t next = buffer == 2 ? 0 : buffer + 1;
    u32x4 x[kCompactTokens];
#pragma unroll
    for (uint32_t i = 0; i < kCompactTokens; ++i) {
      const uint32_t t = i * kRows + tid / kCols;
      x[i] = u32x4{0, 0, 0, 0};
      if (mine && from_at[buffer][t] != kNowhere) {
        const uint64_t at =
            col_at + from_at[buffer][t] + static_cast<uint64_t>(from_off[buffer][t]) * by_token;
        if (scales)
          x[i][0] = *reinterpret_cast<const g_u32*>(at);
        else
          x[i] = STREAM ? __builtin_nontemporal_load(reinterpret_cast<const g_u32x4*>(at))
                        : *reinterpret_cast<const g_u32x4*>(at);
      }
    }
    if (j0 + step < end) find(j0 + step, next);
    // Every thread's loads have returned before any thread writes.
#pragma unroll
    for (uint32_t i = 0; i < kCompactTokens; ++i) asm volatile("" : "+v"(x[i]));
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kCompactTokens; ++i) {
      const uint32_t t = i * kRows + tid / kCols;
      if (mine && to_at[buffer][t] != kNowhere) {
        const uint64_t at =
            col_at + to_at[buffer][t] + static_cast<uint64_t>(to_off[buffer][t]) * by_token;
        if (scales)
          *reinterpret_cast<g_u32*>(at) = x[i][0];
        else if constexpr (STREAM)
          __builtin_nontemporal_store(x[i], reinterpret_cast<g_u32x4*>(at));
        else
          *reinterpret_cast<g_u32x4*>(at) = x[i];
      }
    }
    buffer = next;
  }
}

}  // namespace

hipError_t launch_fork(const ForkParams& p, hipStream_t stream) {
  const uint32_t copies = p.num_children * p.num_layers * 2 * p.parts;
  if (p.blocks)
    hipLaunchKernelGGL(fork_kernel<false>, dim3(copies), dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL(fork_kernel<true>, dim3(copies + p.num_children), dim3(kThreads), 0, stream,
                       p);
  return hipGetLastError();
}

hipError_t launch_compact(const CompactParams& p, hipStream_t stream) {
  static_assert(kMinShift == 3 && kMaxShift == 7, "a kernel for each strip");
  using Kernel = void (*)(CompactParams);
  static constexpr Kernel kKernels[2][5] = {
      {compact_kernel<3, true>, compact_kernel<4, true>, compact_kernel<5, true>,
       compact_kernel<6, true>, compact_kernel<7, true>},
      {compact_kernel<3, false>, compact_kernel<4, false>, compact_kernel<5, false>,
       compact_kernel<6, false>, compact_kernel<7, false>}};
  const Kernel f = kKernels[p.few][p.cols_shift - kMinShift];
  hipLaunchKernelGGL(f, dim3(static_cast<uint32_t>(compact_grid(p))), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace pf
