// pf_paged.h — the paged-cache operators' arguments, shared by their entry
// points (pf_paged.cpp) and kernels (pf_paged.hip, pf_attend_*.hip).
#pragma once

#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cmath>
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
  // Groups of sequences that share their first tokens (attend_shared_kernel; num_groups 0:
  // none do).  Group g has the sequences group_starts[g] to group_starts[g + 1].
  const int32_t* group_starts;
  const int32_t* shared_lens;
  uint32_t num_groups;
  // The launch (plan_shared): the groups' rows go in prefix_units tiles of kManyRows over the
  // shared tokens, in prefix_splits shares of prefix_piece tokens, each sequence's in own_tiles
  // tiles of kFewRows over its own, in own_splits shares of own_piece, by own_waves waves each.
  // Every row and query head then has prefix_splits + own_splits places for shares.
  uint32_t prefix_units, prefix_splits, prefix_piece, own_tiles, own_splits, own_piece, own_waves;
  float *share_o, *share_ml;  // in the workspace
  uint32_t* share_info;       // [num_rows], how many shares a row's heads have
};

constexpr uint32_t kFewRows = 16;        // of attend_few_kernel's tile
constexpr uint32_t kManyRows = 128;      // of attend_many_kernel's, or where rows are many
constexpr uint32_t kWideRows = 256;      // and heads have up to kWideMaxDim values
constexpr uint32_t kWideMaxDim = 128;
constexpr uint32_t kFewMaxSplits = 192;
constexpr uint32_t kFewWaves = 4;        // of a workgroup
constexpr uint32_t kCus = 256;
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
constexpr uint64_t kFewSlots = 512;
inline uint64_t few_piece(uint64_t units, uint64_t longest, uint64_t slots = kFewSlots) {
  constexpr uint64_t kEven = 1024;
  if (units * longest >= 4 * kFewSlots * kEven) return kEven;
  const uint64_t most = units < slots ? slots / units : 1;
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

// Rows of a sequence and KV head up to which shared tokens are passed over once for a group: a
// sequence with more fills tiles of its own, and reads them seldom enough.
constexpr uint32_t kSharedRows = 64;
constexpr uint32_t kSharedMaxSplits = 32;  // of the prefix, and of own tokens

// Bytes of shares, written once and read once, of the shared tokens and the own ones.
inline double share_bytes(const AttendParams& p) {
  return 4.0 * static_cast<double>(p.num_rows) * p.q_heads * (padded_dim(p.pages.dim) * 4 + 8);
}

// Bytes of K and V that sharing has to save before it is worth a second launch and the shares,
// where plan_attend has attend_few_kernel for all.  Sequences and heads that fill the chip read at
// its rate; fewer are split there too.  (In us, as attend_few_kernel's and shared, 8 heads of 128,
// bf16, if nothing else is said: 64 sequences of 4 rows that save 96 MB 16.0 and 18.7, 200 MB 23.4
// and 19.9; of 16 rows 128 MB 19.1 and 23.1, 200 MB 24.2 and 23.2; 192 of 16 rows of 96 values (int8)
// 128 MB 32.0 and 35.5, 200 MB 41.4 and 34.2; 16 of 4 rows 32 MB 14.8 and 16.3, 64 MB 17.6 and 16.5;
// of 16 rows 16 MB 16.2 and 17.7, 64 MB 20.6 and 18.1; 4 of 16 rows 8 MB 14.2 and 15.4, 32 MB 17.8
// and 16.9; 64 of 15 rows of one head of 192 16 MB 19.4 and 20.9, 64 MB 38.8 and 24.0.)
constexpr double kSharedSaves = 96 << 20;
inline double shared_saves(const AttendParams& p, uint64_t rows) {
  if (static_cast<uint64_t>(p.num_seqs) * p.pages.heads > 256)
    return kSharedSaves + 2 * share_bytes(p);
  return rows > kFewRows / 2 ? kSharedSaves / 3 : kSharedSaves / 2;
}

// For sequences of more rows than kFewRows the times of both ways, in us, are estimated and
// compared: neither way gains by a simple count of bytes, for attend reads a sequence's own tokens
// once, in a tile of kManyRows that its rows fill in part, and sharing reads them once for every
// kFewRows rows.  `most` rows of a sequence and KV head, `mean` on average, stand behind `shared`
// tokens and up to `own` of their own.  (14,675 random batches of 2 to 320 sequences, 1 to 12 heads
// of 64 to 256, 17 to 64 rows, timed both ways: by the better way each they take 888 ms, by this rule
// 902, by attend 1,542, all shared 937; the rule leaves 851 more than 6% slower than the better way and
// 25 more than 50%.  Of 5,865 others, from which no constant was taken, 367 and 16.)

// attend: the tiles' start, which looks for their sequences; their steps of 64 tokens; of few tiles,
// in shares of 4 steps or more, the join; and a launch for sequences of up to kFewRows rows, of
// which there are as many as if rows were spread evenly up to `most`.
inline double attend_us(const AttendParams& p, double most, double mean, double shared, double own,
                        bool codes) {
  const double heads = p.pages.heads, seqs = p.num_seqs, dim = padded_dim(p.pages.dim) / 128.0;
  const double slots = dim <= 1 ? 2 * kCus : kCus;
  const double few = std::min(1.0, 2 * (most - mean) / most * (kFewRows / most));
  const double steps = (shared + own) / 64;
  const double full = seqs * (1 + mean / kManyRows) * heads / slots;  // the chip, so many times
  const double shares = std::min(std::max(std::floor(1 / full), 1.0), std::max(steps / 4, 1.0));
  const double chain = full < 1 ? steps / shares
                                : std::max(steps, seqs * heads * (1 - few) * steps / slots);
  const double join = shares > 1 ? 4 + 9.4 * dim * shares * seqs * heads / slots : 0;
  return 6.4 + std::max(full, 1.0) * (2.9 + 5.4 * seqs / 64) +
         (codes ? 1.95 : 1.75) * (dim + 0.5) / 1.5 * chain + join +
         few * (20 + 2.7 * dim * seqs * heads * steps / 1024);
}

// Sharing, as plan_shared has shaped it: a tile's chain of steps over shared tokens and a wave's over
// own ones, what all tiles of either kind take of the chip, and the shares' bytes.
inline double shared_us(const AttendParams& p, double groups, double most, double mean,
                        double shared, double own, bool codes) {
  const double heads = p.pages.heads, seqs = p.num_seqs, dim = padded_dim(p.pages.dim) / 128.0;
  // A sequence's last tile may be part-filled.
  const double tiles = mean > 0.95 * most ? p.own_tiles
                                          : std::min(mean / kFewRows + 0.4, 1.0 * p.own_tiles);
  const double chain = 1.1 * std::min(shared, 1.0 * p.prefix_piece) / 64 +
                       0.27 * std::min(own, 1.0 * p.own_piece) / 32 / p.own_waves;
  const double prefix = (seqs * mean / kManyRows + 0.5 * groups) * heads * shared / 64;
  const double owns = seqs * heads * tiles * own;
  return 12.4 + dim * (chain + 1.2 * prefix / (2 * kCus) + (codes ? 2.9e-5 : 4.4e-5) * owns) +
         2.3e-6 * seqs * mean * heads * (512 * dim + 8);
}

// Workgroups that pass over shared tokens, of the 512 that the chip holds.  Each step of one,
// 64 tokens of 128 rows, takes some 1.4 us (heads of 128), a launch of them 9 more, and own tokens
// are read at 4.5 TB/s, on average half of the longest: the fewest that are done with the own ones
// leave the fewest shares to write and join, more leave too little room beside them.  (64, 128,
// 256 and 384 of them, in us, 64 bf16 sequences: behind 8,000 shared tokens and up to 500 of
// their own 58, 40, 34 and 42, with up to 2,000 84, 87, 92 and 99; behind 32,000 and up to 2,000
// 203, 131, 109 and 128; 16 behind 8,000 and up to 2,000 35, 35, 36 and 36.)  Of long prefixes two
// to a compute unit hide each other's loads: 64 sequences behind 32,000 with 256 72, 384 69; 256
// 210 and 195; but 64 behind 12,000 39 and 43.  Where there are several groups, shorter ones
// among them leave workgroups out: 64 sequences in four groups behind up to 4,000, with 256, 384
// and 512, 32, 29 and 32, up to 32,000 138, 108 and 110; 256 in four behind up to 12,000 153,
// 110 and 98.  Heads of more than 128 values leave room for one workgroup a compute unit, and own
// tokens wait where shared ones take them all: heads of 192 with 192 and with 256 or 384, 24
// sequences of 12 rows (e4m3) behind 4,000 and up to 20 of their own 34 and 40, 24 of 4 (bf16) behind
// 16,000 and up to 300 52 and 59, 120 of 12 behind 16,000 and up to 20 (4 heads) 114 and 126; but 64
// of 12 behind 16,000 and up to 300 165 and 156.
inline uint64_t prefix_workgroups(uint64_t steps, uint64_t groups, uint64_t dim, double own_bytes) {
  const double step = 1.4 * static_cast<double>(dim) / 128;
  const double own = 8 + own_bytes / 2 / 4.5e6;
  uint64_t n = 64;
  while (n < 256 && 9 + static_cast<double>(steps) / static_cast<double>(n) * step > own) n *= 2;
  if (n == 256 && groups == 1 && dim > 128) return 192;
  if (n == 256 && steps >= 24 * 256) return groups > 1 ? 512 : 384;
  return n == 256 && groups > 1 && steps >= 8 * 256 ? 384 : n;
}

// Shapes the launch of a batch whose groups share up to `most_shared` tokens, whose sequences
// have up to `most_own` more and `most_new` rows, joining in `bytes` of workspace at `ws`.  Like
// plan_attend's, lengths may be wrong and rows too few; a shared length counts for what the block
// table holds, whatever it says, or, from PF_SHARED_LEN_ANYWAY on, for as much as sharing takes.
// `rows`: of all sequences together, 0 if that is not known (num_rows may have others behind them).
// False where the batch is better off, or has to be, attended by plan_attend's kernels.
inline bool plan_shared(AttendParams* p, uint64_t most_new, uint64_t most_shared,
                        uint64_t most_own, uint64_t ws, uint64_t bytes, uint64_t rows = 0) {
  const uint64_t heads = p->pages.heads, group = p->group, dim = padded_dim(p->pages.dim);
  const uint64_t room = static_cast<uint64_t>(p->table_width) * p->pages.block_size;
  if (most_shared == 0) most_shared = room;
  if (most_new == 0 || most_new > p->num_rows) most_new = p->num_rows;
  auto ceil_div = [](uint64_t a, uint64_t b) { return (a + b - 1) / b; };
  if (p->num_groups == 0 || p->num_seqs < 2 || p->window || most_new * group > kSharedRows)
    return false;
  const bool codes = p->pages.type == PF_KV_E4M3 || p->pages.type == PF_KV_INT8;
  const double token = 2.0 * static_cast<double>(heads * p->pages.dim) * (codes ? 1 : 2);
  const uint64_t groups = p->num_groups < p->num_seqs ? p->num_groups : p->num_seqs;
  const bool anyway = most_shared >= PF_SHARED_LEN_ANYWAY;
  if (most_shared > room) most_shared = room;
  if (most_own == 0 || most_own > room) most_own = room;
  const double saved =
      static_cast<double>(p->num_seqs - groups) * static_cast<double>(most_shared) * token;
  const double own = static_cast<double>(p->num_seqs * most_own) * token;
  const bool few = most_new * group <= kFewRows;
  if (!anyway && few && saved < shared_saves(*p, most_new * group)) return false;
  // Each group's last tile may be part-filled.
  const uint64_t tiles = (p->num_rows * group + groups * (kManyRows - 1)) / kManyRows;
  const uint64_t prefix = prefix_workgroups(tiles * heads * ceil_div(most_shared, 64), groups, dim,
                                            own);
  uint64_t splits = prefix / (tiles * heads);
  if (splits < 1) splits = 1;
  if (splits > kSharedMaxSplits) splits = kSharedMaxSplits;
  uint64_t piece = ceil_div(ceil_div(most_shared, splits), 64) * 64;
  if (piece < 256) piece = 256;
  splits = ceil_div(most_shared, piece);
  const uint64_t own_tiles = ceil_div(most_new * group, kFewRows);
  const uint64_t units = p->num_seqs * own_tiles * heads;
  const uint64_t slots = kFewSlots - (prefix < 256 ? prefix : 256);
  uint64_t own_piece = few_piece(units, most_own, slots);
  uint64_t own_splits = ceil_div(most_own, own_piece);
  if (own_splits > kSharedMaxSplits) own_splits = kSharedMaxSplits;
  const uint64_t share = p->num_rows * p->q_heads * (dim * 4 + 8);
  const uint64_t counts = workspace_counts(bytes) * kCountStride * 4;
  const uint64_t info = ceil_div(p->num_rows * 4, 16) * 16;
  if (bytes < counts + info) return false;
  const uint64_t most = (bytes - counts - info) / share;
  if (most < 2) return false;
  if (own_splits > most / 2) own_splits = most / 2;
  if (splits > most - own_splits) splits = most - own_splits;
  piece = ceil_div(ceil_div(most_shared, splits), 64) * 64;
  own_piece = ceil_div(ceil_div(most_own, own_splits), 128) * 128;
  // The own tokens' workgroups start together, or nearly so (ragged lengths make room), beside
  // those of the shared ones, where fewer waves for each allow it: 64 sequences behind 8,000 and
  // up to 500 of their own 34 us with 2 waves and 39 with 4, and with up to 2,000 (64 workgroups
  // before them) 93 and 84; 128 behind 8,000 and up to 500 59 with one, 61 with 2, 66 with 4.
  uint32_t waves = kFewWaves;
  while (waves > 1 && units * own_splits * waves / kFewWaves + prefix > kFewSlots * 5 / 4) waves /= 2;
  // The kernel counts units in 32 bits, of sequences without rows as well, and both kinds make one
  // grid.
  constexpr uint64_t kMostUnits = 0x3fffffff;
  if (units * own_splits > kMostUnits || tiles * splits * heads > kMostUnits) return false;
  p->prefix_units = static_cast<uint32_t>(tiles);
  p->prefix_splits = static_cast<uint32_t>(splits);
  p->prefix_piece = static_cast<uint32_t>(piece);
  p->own_tiles = static_cast<uint32_t>(own_tiles);
  p->own_splits = static_cast<uint32_t>(own_splits);
  p->own_piece = static_cast<uint32_t>(own_piece);
  p->own_waves = waves;
  if (!anyway && !few) {
    const double most = static_cast<double>(most_new * group);
    const double mean = rows ? std::min(static_cast<double>(rows * group) / p->num_seqs, most) : most / 2;
    const double s = static_cast<double>(most_shared), o = static_cast<double>(most_own);
    if (shared_us(*p, static_cast<double>(groups), most, mean, s, o, codes) >
        1.05 * attend_us(*p, most, mean, s, o, codes))
      return false;
  }
  const uint64_t values = (splits + own_splits) * p->num_rows * p->q_heads;
  p->share_info = reinterpret_cast<uint32_t*>(ws + counts);
  p->share_o = reinterpret_cast<float*>(ws + counts + info);
  p->share_ml = reinterpret_cast<float*>(ws + counts + info + values * dim * 4);
  return true;
}
inline uint64_t shared_grid(const AttendParams& p) {
  const uint64_t own =
      static_cast<uint64_t>(p.num_seqs) * p.own_tiles * p.own_splits * p.pages.heads;
  const uint64_t per = kFewWaves / p.own_waves;
  return static_cast<uint64_t>(p.prefix_units) * p.prefix_splits * p.pages.heads +
         (own + per - 1) / per;
}
// Heads of a workgroup of attend_shared_join_kernel, one a wave.
constexpr uint32_t kJoinHeads = 4;
inline uint64_t shared_join_grid(const AttendParams& p) {
  return static_cast<uint64_t>(p.num_rows) * ((p.q_heads + kJoinHeads - 1) / kJoinHeads);
}

hipError_t launch_kv_write(const PagedView& pages, const RowsView& k, const RowsView& v,
                           uint32_t row_type, const int64_t* slots, uint32_t n, bool aligned,
                           hipStream_t stream);
hipError_t launch_kv_read(const PagedView& pages, const RowsView& k, const RowsView& v,
                          uint32_t row_type, const int64_t* slots, uint32_t n, bool aligned,
                          hipStream_t stream);
hipError_t launch_attend_bf16(const AttendParams& p, hipStream_t stream);
hipError_t launch_attend_fp16(const AttendParams& p, hipStream_t stream);
hipError_t launch_shared_bf16(const AttendParams& p, hipStream_t stream);
hipError_t launch_shared_fp16(const AttendParams& p, hipStream_t stream);

}  // namespace pf
