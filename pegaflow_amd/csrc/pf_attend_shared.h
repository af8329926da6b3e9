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
#pragma once

#include "pf_attend_kernels.h"

namespace pf {
namespace {

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
    attend_many<Row, TYPE, DP, kManyRows, true>(a, lds.many, blockIdx.x);
  else
    attend_few<Row, TYPE, DP, true>(a, lds.few, blockIdx.x - prefix);
}

// Joins the shares of a row: a wave to a query head, 4 values a lane, shares in turn where a
// head's values take part of a wave only.
template <class Row, uint32_t DP>
__global__ void __launch_bounds__(kJoinHeads * 64) attend_shared_join_kernel(AttendParams a) {
  constexpr uint32_t kLanes = DP / 4, kTurns = 64 / kLanes;
  static_assert(2 * kSharedMaxSplits <= 64, "a lane for each share");
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t per_row = (a.q_heads + kJoinHeads - 1) / kJoinHeads;
  const uint32_t row = blockIdx.x / per_row;
  const uint32_t q_head = __builtin_amdgcn_readfirstlane(blockIdx.x % per_row * kJoinHeads +
                                                         (threadIdx.x >> 6));
  if (q_head >= a.q_heads) return;
  // The row's sequence.
  uint32_t seq = a.num_seqs;
  for (uint32_t b0 = 0; b0 < a.num_seqs; b0 += 64) {
    const uint32_t b = b0 + lane;
    const uint64_t in = __ballot(b < a.num_seqs && a.query_starts[b] <= static_cast<int32_t>(row) &&
                                 static_cast<int32_t>(row) < a.query_starts[b + 1]);
    if (in) {
      seq = b0 + __builtin_ctzll(in);
      break;
    }
  }
  if (seq == a.num_seqs) return;  // of none: stays as it was
  const Seq sq = seq_of(a, seq);
  const uint32_t head = q_head / a.group;
  const uint32_t in_seq = (row - static_cast<uint32_t>(sq.first)) * a.group + q_head - head * a.group;
  const uint32_t tile = in_seq / kFewRows;
  if (tile >= a.own_tiles) return;  // more rows than the batch was said to have
  const int32_t shared = shared_of(a, static_cast<int32_t>(seq));
  int32_t begin = 0, end = shared;
  const uint32_t prefix =
      shared ? split_range(begin, end, 0, a.prefix_splits, a.prefix_piece) : 0;
  // Of its tile, as attend_few counts them.
  const uint32_t rows = static_cast<uint32_t>(sq.rows) * a.group;
  const uint32_t last = min((tile + 1) * kFewRows, rows) - 1;
  begin = shared;
  end = row_end(a, sq.len, sq.len - sq.rows + static_cast<int32_t>(last / a.group));
  const uint32_t used = prefix + split_range(begin, end, 0, a.own_splits, a.own_piece);
  auto share = [&](uint32_t i) {
    return share_at(a, i < prefix ? i : a.prefix_splits + i - prefix, row, q_head);
  };
  f32x2 ml{kNegInf, 0.0f};
  if (lane < used) ml = reinterpret_cast<const f32x2*>(a.share_ml)[share(lane)];
  float m = ml[0];
#pragma unroll
  for (int step = 1; step < 64; step *= 2) m = fmaxf(m, __shfl_xor(m, step));
  // A share without a maximum attended nothing, or only what is no number.
  const float factor =
      ml[0] == kNegInf ? (ml[1] == 0.0f ? 0.0f : 1.0f) : share_factor(ml[0] - m);
  float l = ml[1] * factor;
#pragma unroll
  for (int step = 1; step < 64; step *= 2) l += __shfl_xor(l, step);
  const uint32_t turn = lane / kLanes, d = lane % kLanes * 4;
  f32x4 o{0, 0, 0, 0};
  constexpr uint32_t kFlight = 4;  // loads under way together
  for (uint32_t i0 = 0; i0 < used; i0 += kTurns * kFlight) {
    f32x4 x[kFlight];
    float f[kFlight];
#pragma unroll
    for (uint32_t j = 0; j < kFlight; ++j) {
      const uint32_t i = i0 + j * kTurns + turn;
      x[j] = f32x4{0, 0, 0, 0};
      f[j] = __shfl(factor, static_cast<int>(i & 63u));
      if (turn < kTurns && i < used)
        x[j] = *reinterpret_cast<const f32x4*>(a.share_o + share(i) * DP + d);
    }
#pragma unroll
    for (uint32_t j = 0; j < kFlight; ++j) {
      const bool mine = turn < kTurns && i0 + j * kTurns + turn < used;
#pragma unroll
      for (int v = 0; v < 4; ++v) o[v] += mine ? x[j][v] * f[j] : 0.0f;
    }
  }
  if constexpr (kTurns > 1) {
    f32x4 sum = o;
#pragma unroll
    for (uint32_t t = 1; t < kTurns; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        sum[j] += __shfl(o[j], static_cast<int>((lane + t * kLanes) & 63u));
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
