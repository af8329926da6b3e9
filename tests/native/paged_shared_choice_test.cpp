// paged_shared_choice_test.cpp — which way a batch of shared tokens runs whose sequences have 17 to
// 64 rows of a KV head (plan_shared, pf_paged.h), against both ways' measured times.  On the host
// (no GPU), built by tests/test_shared_choice.py.
// Exit status 0 and "ok" on success; each wrong choice is printed.
#include <cstdio>

#include "pf_paged.h"

using namespace pf;

namespace {

struct Measured {
  uint32_t seqs, groups, heads, group, dim, type, most_new, rows, shared, own;
  double us_shared, us_attend;
};

// The first 20 of either kind, by a factor of 1.6 or more, of 4,000 random batches that no constant
// of the rule was taken from; six in ten with as many new tokens for each sequence.
const Measured kBatches[] = {
    {25, 1, 12, 5, 64, PF_KV_INT8, 9, 225, 80, 104, 24.2, 14.7},
    {3, 1, 12, 5, 128, PF_KV_FP16, 7, 21, 16, 11047, 61.5, 33.4},
    {228, 228, 8, 7, 64, PF_KV_E4M3, 7, 1596, 112, 3524, 700.3, 410.4},
    {29, 5, 12, 5, 128, PF_KV_E4M3, 9, 261, 64, 54, 29.1, 16.5},
    {96, 96, 8, 7, 128, PF_KV_BF16, 7, 672, 336, 64, 76.5, 44.5},
    {55, 1, 4, 4, 256, PF_KV_INT8, 9, 495, 16, 1039, 107.0, 63.1},
    {116, 116, 8, 4, 128, PF_KV_INT8, 8, 928, 64, 921, 112.8, 69.6},
    {24, 2, 12, 7, 128, PF_KV_FP16, 8, 192, 240, 7959, 664.3, 270.5},
    {19, 19, 8, 3, 96, PF_KV_FP16, 10, 190, 6480, 5919, 263.1, 159.6},
    {29, 29, 2, 5, 96, PF_KV_INT8, 8, 232, 7632, 8587, 179.6, 98.3},
    {55, 5, 1, 7, 128, PF_KV_BF16, 7, 385, 5920, 5966, 155.1, 84.0},
    {34, 3, 8, 8, 128, PF_KV_INT8, 7, 238, 16, 25, 27.0, 15.3},
    {3, 1, 8, 4, 128, PF_KV_BF16, 14, 42, 224, 7218, 47.3, 27.4},
    {67, 67, 12, 8, 128, PF_KV_E4M3, 7, 469, 272, 185, 86.5, 50.6},
    {57, 1, 4, 8, 192, PF_KV_BF16, 8, 456, 16, 26, 40.5, 23.4},
    {52, 5, 8, 8, 256, PF_KV_BF16, 7, 364, 48, 1131, 253.7, 103.2},
    {61, 61, 8, 7, 128, PF_KV_INT8, 3, 183, 48, 462, 56.3, 32.9},
    {77, 5, 4, 5, 128, PF_KV_BF16, 10, 770, 32, 4901, 307.9, 184.0},
    {45, 11, 12, 4, 128, PF_KV_FP16, 16, 720, 80, 518, 95.5, 34.5},
    {182, 182, 2, 4, 128, PF_KV_BF16, 12, 2184, 432, 754, 104.8, 65.3},
    {3, 1, 1, 3, 128, PF_KV_INT8, 8, 12, 688, 4159, 17.0, 31.2},
    {5, 1, 1, 2, 64, PF_KV_FP16, 10, 33, 2000, 330, 14.0, 25.5},
    {23, 5, 8, 5, 96, PF_KV_E4M3, 8, 115, 8016, 25, 52.3, 149.9},
    {173, 1, 2, 5, 192, PF_KV_INT8, 9, 872, 11776, 27, 243.5, 642.0},
    {35, 1, 1, 5, 128, PF_KV_BF16, 6, 136, 48, 3771, 24.8, 45.0},
    {99, 24, 1, 7, 64, PF_KV_E4M3, 8, 792, 11264, 20, 59.7, 115.1},
    {311, 1, 1, 7, 256, PF_KV_INT8, 3, 644, 2880, 613, 88.6, 341.6},
    {3, 1, 2, 8, 128, PF_KV_E4M3, 4, 7, 3264, 1416, 18.0, 35.8},
    {123, 2, 4, 3, 128, PF_KV_BF16, 10, 690, 3568, 101, 47.4, 149.1},
    {11, 3, 8, 8, 128, PF_KV_INT8, 5, 32, 96, 11363, 78.3, 136.8},
    {85, 5, 8, 4, 128, PF_KV_E4M3, 14, 638, 4640, 28, 95.6, 166.3},
    {148, 5, 8, 7, 192, PF_KV_E4M3, 6, 473, 112, 23, 73.8, 135.8},
    {68, 1, 2, 8, 64, PF_KV_INT8, 8, 544, 6128, 121, 54.4, 104.2},
    {14, 3, 4, 3, 64, PF_KV_INT8, 9, 83, 12560, 666, 27.6, 69.5},
    {5, 2, 2, 4, 128, PF_KV_BF16, 5, 18, 160, 250, 15.0, 29.2},
    {129, 1, 8, 3, 64, PF_KV_BF16, 6, 445, 16, 36, 24.6, 39.8},
    {4, 1, 4, 8, 64, PF_KV_BF16, 4, 10, 160, 4692, 14.2, 27.1},
    {5, 1, 2, 2, 128, PF_KV_E4M3, 10, 38, 3248, 75, 17.8, 36.4},
    {31, 1, 8, 8, 256, PF_KV_BF16, 4, 75, 368, 2759, 130.7, 219.9},
    {202, 1, 4, 4, 64, PF_KV_INT8, 6, 1212, 2496, 116, 74.7, 144.4},
};

int failures = 0;

bool shares(const Measured& b) {
  AttendParams p{};
  p.num_seqs = b.seqs;
  p.num_groups = b.groups;
  p.num_rows = b.rows;
  p.pages.heads = b.heads;
  p.pages.dim = b.dim;
  p.pages.type = b.type;
  p.pages.block_size = 16;
  p.group = b.group;
  p.q_heads = b.heads * b.group;
  p.causal = 1;
  p.table_width = (b.shared + b.own + 15) / 16;
  return plan_shared(&p, b.most_new, b.shared, b.own, 1ull << 40, 64ull << 20, b.rows);
}

}  // namespace

int main() {
  for (const Measured& b : kBatches)
    if (shares(b) != (b.us_shared < b.us_attend) && ++failures)
      std::printf("FAILED: %u sequences in %u groups, %u heads of %u, up to %u rows behind %u and %u "
                  "tokens: shared %.1f us, attend %.1f\n",
                  b.seqs, b.groups, b.heads, b.dim, b.most_new * b.group, b.shared, b.own, b.us_shared,
                  b.us_attend);
  // 80 sequences of 48 rows each: 213.6 us shared, 107.3 by attend, on either side of any length.
  int changes = 0;
  Measured b{80, 1, 8, 4, 128, PF_KV_BF16, 12, 960, 250, 16, 0, 0};
  bool before = shares(b);
  for (; b.own < 30000; ++b.own) {
    const bool now = shares(b);
    changes += now != before;
    before = now;
  }
  if (changes > 1 && ++failures) std::printf("FAILED: the choice changes %d times with the length\n", changes);
  if (failures) return 1;
  std::puts("ok");
  return 0;
}
