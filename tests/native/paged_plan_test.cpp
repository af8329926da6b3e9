// paged_plan_test.cpp — how a batch's attention is launched (plan_attend, pf_paged.h), on
// the host (no GPU), built by tests/test_paged_plan.py:
//   * every row of every batch that fits the bounds has a tile, whatever the hints say;
//   * shares fit the workspace and do not overlap, and their counts are there;
//   * tiles are split where the chip is not full, or the last round of it is not.
// Exit status 0 and "ok" on success; the first failed checks are printed.
#include <algorithm>
#include <cstdio>
#include <random>

#include "pf_paged.h"

using namespace pf;

namespace {

int failures = 0;
std::mt19937_64 rng(1);

uint64_t pick(uint64_t lo, uint64_t hi) { return lo + rng() % (hi - lo + 1); }
uint64_t spread(uint64_t hi) { return pick(1, 1ull << pick(0, 63 - __builtin_clzll(hi))); }

#define EXPECT(cond)                                                                       \
  if (!(cond) && ++failures <= 20)                                                         \
  std::printf("FAILED line %d: %s (%u sequences, %lu rows, %u heads of %u, group %u)\n",   \
              __LINE__, #cond, p.num_seqs, static_cast<unsigned long>(p.num_rows),         \
              p.pages.heads, p.pages.dim, p.group)

AttendParams batch(uint32_t seqs, uint32_t rows, uint32_t heads, uint32_t dim, uint32_t group,
                   uint32_t longest) {
  AttendParams p{};
  p.num_seqs = seqs;
  p.num_rows = rows;
  p.pages.heads = heads;
  p.pages.dim = dim;
  p.pages.block_size = 16;
  p.group = group;
  p.causal = 1;
  p.table_width = (longest + 15) / 16;
  return p;
}

void any_batch() {
  const uint32_t dims[] = {16, 64, 80, 128, 192, 256};
  const uint32_t seqs = spread(512);
  AttendParams p = batch(seqs, spread(16384), spread(64), dims[pick(0, 5)], pick(1, 20),
                         spread(65536));
  if (pick(0, 3) == 0) p.window = spread(4096);
  const uint64_t bytes = pick(0, 4) ? spread(1ull << 28) + 4096 : 0, ws = 1ull << 40;
  const uint64_t most = pick(0, 2) ? spread(p.num_rows) : 0;
  plan_attend(&p, most, pick(0, 2) ? spread(65536) : 0, bytes ? ws : 0, bytes);
  const uint64_t dim = padded_dim(p.pages.dim), bound = most ? std::min<uint64_t>(most, p.num_rows)
                                                             : p.num_rows;
  // A batch within the bounds: at most `bound` rows a sequence, num_rows in all.
  uint64_t left = p.num_rows, tiles = 0, few = 0;
  for (uint32_t i = 0; i < seqs && left; ++i) {
    const uint64_t n = std::min(left, i % 2 ? bound : pick(1, bound));
    left -= n;
    if (n * p.group > p.few_rows && p.many_units)
      tiles += (n * p.group + p.many_rows - 1) / p.many_rows;
    else if (n * p.group <= kFewRows)
      ++few;
    else
      EXPECT(!"a sequence has a kernel");
  }
  EXPECT(tiles <= p.many_units);
  EXPECT(few == 0 || p.few_splits);
  uint64_t at = ws + workspace_counts(bytes) * kCountStride * 4;
  if (p.few_splits > 1) {
    const uint64_t shares = static_cast<uint64_t>(seqs) * p.pages.heads * p.few_splits;
    EXPECT(p.few_splits <= kFewMaxSplits);
    EXPECT(static_cast<uint64_t>(seqs) * p.pages.heads <= workspace_counts(bytes));
    EXPECT(reinterpret_cast<uint64_t>(p.few_o) == at);
    EXPECT(reinterpret_cast<uint64_t>(p.few_ml) == at + shares * p.few_rows_most * dim * 4);
    at += shares * p.few_rows_most * (dim * 4 + 8);
    EXPECT(at <= ws + bytes);
  }
  EXPECT(p.many_whole <= p.many_units);
  if (p.many_whole < p.many_units) {
    EXPECT(p.many_splits > 1);
    const uint64_t shares = static_cast<uint64_t>(p.many_units - p.many_whole) * p.pages.heads *
                            p.many_splits;
    EXPECT(reinterpret_cast<uint64_t>(p.many_o) == at && at % 16 == 0);
    EXPECT(reinterpret_cast<uint64_t>(p.many_ml) == at + shares * p.many_rows * dim * 4);
    // A wave's 64 lanes each hold a maximum and a sum: two lanes a row.
    EXPECT(at + shares * p.many_rows * (dim * 4 + 16) <= ws + bytes);
    EXPECT(p.many_piece % 64 == 0 && p.many_piece >= 64);
  }
  if (!bytes) EXPECT(p.few_splits <= 1 && p.many_whole == p.many_units);
}

void rules() {
  const uint64_t ws = 1ull << 40, bytes = 64ull << 20;
  AttendParams p = batch(1, 500, 8, 128, 4, 10500);  // 64 workgroups: four shares each
  plan_attend(&p, 500, 10500, ws, bytes);
  EXPECT(p.many_rows == 256 && p.many_units == 8 && p.many_whole == 0 && p.many_splits == 4);
  p = batch(1, 2048, 8, 128, 4, 32048);  // 256: whole
  plan_attend(&p, 2048, 32048, ws, bytes);
  EXPECT(p.many_units == 32 && p.many_whole == 32);
  p = batch(1, 2100, 8, 128, 4, 32100);  // 8 more: split among as many
  plan_attend(&p, 2100, 32100, ws, bytes);
  EXPECT(p.many_units == 33 && p.many_whole == 32 && p.many_splits == 32);
  p = batch(1, 2100, 8, 128, 4, 3100);  // shorter: narrow tiles, not worth a join
  plan_attend(&p, 2100, 3100, ws, bytes);
  EXPECT(p.many_rows == 128 && p.many_units == 66 && p.many_whole == 66);
  p = batch(1, 2100, 8, 128, 4, 32100);  // no workspace
  plan_attend(&p, 2100, 32100, 0, 0);
  EXPECT(p.many_whole == 33);
  p = batch(1, 1100, 8, 256, 4, 9100);  // one workgroup a compute unit
  plan_attend(&p, 1100, 9100, ws, bytes);
  EXPECT(p.many_rows == 128 && p.many_units == 35 && p.many_whole == 32 && p.many_splits > 1);
  EXPECT(wide_tiles(16, 16384, 8, 128, 4500) && !wide_tiles(16, 16383, 8, 128, 4500));
  EXPECT(!wide_tiles(65, 16384, 64, 128, 4500) && wide_tiles(64, 16384, 64, 128, 4500));
  EXPECT(few_piece(8, 10001) < 1024 && few_piece(384, 1000) == 1000);
}

}  // namespace

int main() {
  rules();
  for (int i = 0; i < 200000; ++i) any_batch();
  if (failures) return 1;
  std::puts("ok");
  return 0;
}
