// pf_rotary.h — rotary positions: the arguments that their entry points (pf_rotary.cpp)
// hand to their kernels (pf_rotary.hip).
#pragma once

#include "pf_paged.h"

namespace pf {

constexpr uint32_t kMaxPairs = PF_KV_MAX_HEAD_DIM / 2;

struct RotaryParams {
  PagedView pages;  // where the turned K and V go; of a call without them only `dim` is set
  RowsView q, q_out, k, v;
  const int64_t* positions;
  const int64_t* slots;
  const uint64_t* turns;  // each pair's turns a position, times 2^64
  float factor;           // of turned values
  uint32_t rotary;        // values of a head that are turned
  uint32_t layout;        // PF_ROTARY_*
  uint32_t n, q_heads, kv_heads;
  // The launch (plan_rotary): a workgroup takes part_heads heads of some tokens, of q in
  // the first q_parts workgroups of these tokens, then kv_parts of K and as many of V.
  uint32_t part_heads, q_parts, kv_parts;
  bool aligned;  // all rows move by 16 bytes
};

constexpr uint32_t kRotaryThreads = 256;
// Lanes of a row, 16 values each.
inline uint32_t rotary_lanes(uint32_t dim) { return dim <= 64 ? 4 : dim <= 128 ? 8 : 16; }
inline uint64_t rotary_units(const RotaryParams& p) {
  return (static_cast<uint64_t>(p.n) * rotary_lanes(p.pages.dim) + kRotaryThreads - 1) /
         kRotaryThreads;
}
inline uint64_t rotary_grid(const RotaryParams& p) {
  return rotary_units(p) * (p.q_parts + 2 * p.kv_parts);
}

// Heads of a workgroup.  Its lanes keep the sines and cosines of their pairs, some 240
// operations, for all of them: 2,000 tokens (32 heads of 128 on 8, e4m3) take 10.9 us with 2,
// 9.9 with 4 and 12.2 with 8.  Where keys need no coding 10,000 take 48.9 with 2, 50.9 with 4
// and 52.2 with 8.  Halves of a number of turned values that is no multiple of 16 have twice the
// sines and cosines: 13,900 tokens (12 heads of 128, fp16, 82 values) 76 with 2, 66 with 4 and 67
// with 12.  Few tokens fill the chip only with few heads each: 5 take 3.0 us with one
// head and 5.9 with 8, 500 4.7 from 256 workgroups on and 5.0 from 512.
inline void plan_rotary(RotaryParams* p) {
  const uint64_t units = rotary_units(*p);
  const bool codes = p->pages.type == PF_KV_E4M3 || p->pages.type == PF_KV_INT8;
  uint32_t heads = codes || (p->rotary % 16 && p->layout == PF_ROTARY_HALF) ? 4 : 2;
  auto parts = [&](uint32_t h) { return (h + heads - 1) / heads; };
  while (heads > 1 && units * (parts(p->q_heads) + 2 * parts(p->kv_heads)) < 256) heads /= 2;
  p->part_heads = heads;
  p->q_parts = parts(p->q_heads);
  p->kv_parts = parts(p->kv_heads);
}

hipError_t launch_rotary_bf16(const RotaryParams& p, hipStream_t stream);
hipError_t launch_rotary_fp16(const RotaryParams& p, hipStream_t stream);

}  // namespace pf
