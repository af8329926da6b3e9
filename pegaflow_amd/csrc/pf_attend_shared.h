// pf_attend_shared.h — attention of a batch whose sequences share their first tokens, included
// once for each row type (pf_shared_bf16.hip, pf_shared_fp16.hip).
//
// A softmax over a sequence's tokens is one over its parts, joined: with a part's maximum m_s,
// sum l_s and outputs o_s (not divided),
//   m = max m_s,  o = sum o_s exp(m_s - m) / sum l_s exp(m_s - m).
// Shared tokens are attended by the rows of all sequences of a group at once, as one matrix
// of rows in attend_many's tiles: their K and V are read once a tile instead of once a
// sequence, and meet the matrix cores with tiles that are full.  The tokens that a sequence
// has to itself are attended by its few rows, in attend_few's tiles.  Both kinds of tiles are
// workgroups of one launch, so that the first's products run beside the second's reads; all leave
// their shares in fp32, which a second launch joins.
//
// 64 sequences behind 10,000 shared tokens and up to 500 of their own (bf16, 32 heads of 128 on 8)
// take 38 to 42 us, 31.7 to 36.6 of them the tiles and 6.8 the join; attend, which reads the shared
// tokens 64 times, 224 to 231.  The bytes alone would take 21 and the products 9: a tile's start is a
// chain of loads (groups, lengths, table, K: some 7 us of a cold launch), its steps have one wave
// a vector unit where own tokens take the other, 1.4 us each, of which half are products and
// softmax and a third the wait for K and V, and 17 MB of shares are written and read.  256
// sequences behind 30,000 take 182 to 199 (attend 3,690 to 3,720), 690 TFLOP/s; there tiles of 256
// rows were no faster.  64 behind 16,000 and up to 2,000 (e4m3) take 66 to 71 (attend 242 to 249).
//
// The weights of shared tokens are rounded once to the rows' type, as attend rounds those of more
// than 16 rows: outputs are off by 0.0022 to 0.0023 relative (bf16; fp16 0.00025 to 0.00029) where
// the rounding of the output alone takes 0.0017 (0.00021).  The rest of each weight, multiplied as
// well, brought them to that, but the three batches above took 45, 242 and 74 us instead of 38, 183
// and 69 (29 drafts behind 4,100, int8, 47 instead of 39), and was left out: who needs it calls
// attend.
#pragma once

#include "pf_attend_kernels.h"

namespace pf {
namespace {

// Workgroup `index` of the tiles of shared tokens.
template <class Row, uint32_t TYPE, uint32_t DP>
__device__ __forceinline__ void attend_shared_tokens(const AttendParams& a, ManyLds<DP>& lds,
                                                     uint32_t index) {
  constexpr uint32_t ROWS = kManyRows;
  constexpr bool SHARED = true;
#include "pf_attend_many.inc"
}

// Workgroup `index` of the tiles of sequences' own tokens.
template <class Row, uint32_t TYPE, uint32_t DP>
__device__ __forceinline__ void attend_own_tokens(const AttendParams& a, FewLds<DP>& mem,
                                                  uint32_t index) {
  constexpr bool SHARED = true;
#include "pf_attend_few.inc"
}

template <class Row, uint32_t TYPE, uint32_t DP>
__global__ void __launch_bounds__(kFewThreads, DP <= 128 ? 2 : 1)
attend_shared_kernel(AttendParams a) {
  static_assert(kFewThreads == 2 * kManyRows, "one workgroup's threads for both");
  __shared__ union {
    ManyLds<DP> many;
    FewLds<DP> few;
  } lds;
  // Tiles of shared tokens take the longest: first.
  const uint32_t prefix = a.prefix_units * a.prefix_splits * a.pages.heads;
  if (blockIdx.x < prefix)
    attend_shared_tokens<Row, TYPE, DP>(a, lds.many, blockIdx.x);
  else
    attend_own_tokens<Row, TYPE, DP>(a, lds.few, blockIdx.x - prefix);
}

// Joins the shares of a row: a wave to a query head, 4 values a lane, shares in turn where a
// head's values take part of a wave only.  Everything that a wave reads is asked for at once, also
// the places of shares that turn out to be none: one wait instead of three.
template <class Row, uint32_t DP>
__global__ void __launch_bounds__(kJoinHeads * 64) attend_shared_join_kernel(AttendParams a) {
  constexpr uint32_t kLanes = DP / 4, kTurns = 64 / kLanes, kFlight = 8;
  static_assert(2 * kSharedMaxSplits <= 64, "a lane for each share");
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t per_row = (a.q_heads + kJoinHeads - 1) / kJoinHeads;
  const uint32_t row = blockIdx.x / per_row;
  const uint32_t q_head = __builtin_amdgcn_readfirstlane(blockIdx.x % per_row * kJoinHeads +
                                                         (threadIdx.x >> 6));
  if (q_head >= a.q_heads) return;
  const uint32_t turn = lane / kLanes, d = lane % kLanes * 4;
  const uint32_t places = a.prefix_splits + a.own_splits;
  f32x2 ml{kNegInf, 0.0f};
  if (lane < places) ml = reinterpret_cast<const f32x2*>(a.share_ml)[share_at(a, lane, row, q_head)];
  auto part = [&](uint32_t i) {
    f32x4 x{0, 0, 0, 0};
    if (turn < kTurns && i < places)
      x = *reinterpret_cast<const f32x4*>(a.share_o + share_at(a, i, row, q_head) * DP + d);
    return x;
  };
  f32x4 x[kFlight];
#pragma unroll
  for (uint32_t j = 0; j < kFlight; ++j) x[j] = part(j * kTurns + turn);
  const uint32_t info = a.share_info[row];
  const int32_t first = row_start(a, 0), last = row_start(a, a.num_seqs);
  // A row of no sequence, or beyond the rows that one was said to have, stays as it was.
  if (static_cast<int32_t>(row) < first || static_cast<int32_t>(row) >= last || info == 0) return;
  // Shares 0 to prefix - 1 and prefix_splits to `end` - 1 are there.
  const uint32_t prefix = info & 0xffu, end = a.prefix_splits + (info >> 8);
  if (lane >= end || (lane >= prefix && lane < a.prefix_splits)) ml = f32x2{kNegInf, 0.0f};
  float m = ml[0];
#pragma unroll
  for (int step = 1; step < 64; step *= 2) m = fmaxf(m, __shfl_xor(m, step));
  // A share without a maximum attended nothing, or only what is no number.
  const float factor =
      ml[0] == kNegInf ? (ml[1] == 0.0f ? 0.0f : 1.0f) : share_factor(ml[0] - m);
  float l = ml[1] * factor;
#pragma unroll
  for (int step = 1; step < 64; step *= 2) l += __shfl_xor(l, step);
  f32x4 o{0, 0, 0, 0};
  auto add = [&](uint32_t i0, const f32x4 (&y)[kFlight]) {
#pragma unroll
    for (uint32_t j = 0; j < kFlight; ++j) {
      const uint32_t i = i0 + j * kTurns + turn;
      const float f = __shfl(factor, static_cast<int>(i & 63u));
      const bool there = i < prefix || (i >= a.prefix_splits && i < end);
#pragma unroll
      for (int v = 0; v < 4; ++v) o[v] += there ? y[j][v] * f : 0.0f;
    }
  };
  add(0, x);
  for (uint32_t i0 = kTurns * kFlight; i0 < places; i0 += kTurns * kFlight) {
#pragma unroll
    for (uint32_t j = 0; j < kFlight; ++j) x[j] = part(i0 + j * kTurns + turn);
    add(i0, x);
  }
  if constexpr (kTurns > 1) {
    f32x4 sum = o;
#pragma unroll
    for (uint32_t t = 1; t < kTurns; ++t)
#pragma unroll
      for (int v = 0; v < 4; ++v)
        sum[v] += __shfl(o[v], static_cast<int>((lane + t * kLanes) & 63u));
    o = sum;
  }
  if (turn) return;
  const float inv = l == 0 ? 0.0f : 1.0f / l;
  store_out4<Row>(a.out.data + (row * a.out.token_stride + q_head * a.out.head_stride) * 2, d, a,
                  f32x4{o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv});
  if (a.lse && d == 0)
    a.lse[static_cast<uint64_t>(row) * a.q_heads + q_head] = log_sum_exp<Row>(a, m, l);
}

template <class Row, uint32_t TYPE, uint32_t DP>
hipError_t launch_shared_kernels(const AttendParams& p, hipStream_t stream) {
  hipLaunchKernelGGL((attend_shared_kernel<Row, TYPE, DP>),
                     dim3(static_cast<uint32_t>(shared_grid(p))), dim3(kFewThreads), 0, stream, p);
  hipLaunchKernelGGL((attend_shared_join_kernel<Row, DP>),
                     dim3(static_cast<uint32_t>(shared_join_grid(p))), dim3(kJoinHeads * 64), 0,
                     stream, p);
  return hipGetLastError();
}

template <class Row, uint32_t TYPE>
hipError_t launch_shared_dim(const AttendParams& p, hipStream_t stream) {
  switch (padded_dim(p.pages.dim)) {
    case 64: return launch_shared_kernels<Row, TYPE, 64>(p, stream);
    case 96: return launch_shared_kernels<Row, TYPE, 96>(p, stream);
    case 128: return launch_shared_kernels<Row, TYPE, 128>(p, stream);
    case 192: return launch_shared_kernels<Row, TYPE, 192>(p, stream);
    default: return launch_shared_kernels<Row, TYPE, 256>(p, stream);
  }
}

template <class Row>
hipError_t launch_shared_type(const AttendParams& p, hipStream_t stream) {
  if (p.pages.type == PF_KV_E4M3) return launch_shared_dim<Row, PF_KV_E4M3>(p, stream);
  if (p.pages.type == PF_KV_INT8) return launch_shared_dim<Row, PF_KV_INT8>(p, stream);
  return launch_shared_dim<Row, Row::kType>(p, stream);
}

}  // namespace
}  // namespace pf
