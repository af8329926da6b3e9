// pf_paged.hip — writing rows of K and V into a layer's pages and reading them
// back, at 16 bits or as 8-bit codes with one scale for each token and head.
//
// Row x (one token, one head, `dim` values) is held as codes c and scale s:
//   s = max|x| * (1 / L) (L = 448 for e4m3, 127 for int8),  c = round(x / s),
// 1 / L, the product and the quotient each rounded to 32 bits, to nearest, ties to even:
// s is off by an ulp at most, and costs one multiplication.  A row of zeros has
// s = 0 and codes 0.  A row with an infinity or NaN has s = NaN and codes 0, so it
// reads back as NaN throughout.  |x| / s exceeds L at most by the roundings of 1 / L, s
// and the quotient: by a factor under 1 + 2^-8 even where s is subnormal (the
// smallest max|x| is 2^-133, which leaves s 7 bits), and both conversions round
// such a quotient back to L, so nothing is clamped.
//
// Bound by HBM: a row is read once and written once.  A row belongs to a group of
// lanes, 8 values each; a workgroup covers as many consecutive tokens as it has
// groups, and kHeads heads, so the scales of one head's tokens, which are
// neighbours in the block, leave one XCD's L2 together.
//
// 10,000 tokens of 8 heads of 128 (62 MB) are written as int8 in 13.0 us and read from
// e4m3 in 10.7, 4.8 and 5.8 TB/s (part of it stays in the caches between calls; a large
// copy moves 5.2).  16 values a lane, 8 heads a workgroup and non-temporal accesses were
// no faster.
#include <hip/hip_runtime.h>

#include "pf_paged_device.h"

namespace pf {

namespace {

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kThreads = 256;
constexpr uint32_t kHeads = 2;  // heads of a workgroup: independent loads in flight

// The 8 values of this lane as codes of scale s (s > 0).
template <class Row, uint32_t TYPE>
__device__ __forceinline__ u32x2 encode_row8(u32x4 x, float s) {
  float q[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    q[2 * i] = Row::to_float(x[i] & 0xffffu);
    q[2 * i + 1] = Row::to_float(x[i] >> 16);
  }
  return encode<TYPE>(q, s);
}

// Workgroup b: tokens (b / (2 * head_groups)) * groups + group, K or V, kHeads heads.
template <class Row, uint32_t TYPE, uint32_t LANES, bool ALIGNED>
__global__ void __launch_bounds__(kThreads)
kv_write_kernel(PagedView p, RowsView k, RowsView v, const int64_t* __restrict__ slots, uint32_t n,
                uint32_t head_groups) {
  const uint32_t lane = threadIdx.x % LANES;
  const uint32_t unit = blockIdx.x / (2 * head_groups), part = blockIdx.x % (2 * head_groups);
  const uint32_t row = unit * (kThreads / LANES) + threadIdx.x / LANES;
  const uint32_t h0 = (part >> 1) * kHeads;
  if (row >= n) return;
  const int64_t slot = slots[row];
  if (slot < 0 || slot >= static_cast<int64_t>(static_cast<uint64_t>(p.num_blocks) * p.block_size))
    return;
  const uint64_t block = static_cast<uint64_t>(slot) / p.block_size;
  const uint32_t token = static_cast<uint32_t>(static_cast<uint64_t>(slot) - block * p.block_size);
  const RowsView& rows = part & 1 ? v : k;
  const uint64_t segment = (part & 1 ? p.v : p.k) + block * p.block_bytes;
  const uint32_t d = lane * 8;
  const bool mine = d < p.dim;
  u32x4 x[kHeads];
#pragma unroll
  for (uint32_t i = 0; i < kHeads; ++i) {
    x[i] = u32x4{0, 0, 0, 0};
    if (mine && h0 + i < p.heads)
      x[i] = load_row8<ALIGNED>(rows.data +
                                (row * rows.token_stride + (h0 + i) * rows.head_stride + d) * 2);
  }
#pragma unroll
  for (uint32_t i = 0; i < kHeads; ++i) {
    const uint32_t h = h0 + i;
    if (h >= p.heads) break;
    const uint64_t at = segment + static_cast<uint64_t>(token) * p.token_bytes +
                        static_cast<uint64_t>(h) * p.head_bytes;
    if constexpr (TYPE == PF_KV_BF16 || TYPE == PF_KV_FP16) {
      if (mine) *reinterpret_cast<g_u32x4*>(at + d * 2) = x[i];
    } else {
      // The largest magnitude, as bits: they order as the values do, with
      // infinity and NaN on top.
      u16x2 pair{0, 0};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t word = x[i][w] & 0x7fff7fffu;
        pair = __builtin_elementwise_max(pair, __builtin_bit_cast(u16x2, word));
      }
      const uint32_t m = group_max<LANES>(umax(pair[0], pair[1]));
      float s = Row::to_float(m) * kInverseLargest<TYPE>;
      u32x2 c{0, 0};
      if (m >= Row::kInf)
        s = __builtin_nanf("");
      else if (m)
        c = encode_row8<Row, TYPE>(x[i], s);
      if (mine) *reinterpret_cast<g_u32x2*>(at + d) = c;
      if (lane == 0)
        *reinterpret_cast<g_f32*>(segment + p.scale_offset + (h * p.block_size + token) * 4ull) = s;
    }
  }
}

template <class Row, uint32_t TYPE, uint32_t LANES, bool ALIGNED>
__global__ void __launch_bounds__(kThreads)
kv_read_kernel(PagedView p, RowsView k, RowsView v, const int64_t* __restrict__ slots, uint32_t n,
               uint32_t head_groups) {
  const uint32_t lane = threadIdx.x % LANES;
  const uint32_t unit = blockIdx.x / (2 * head_groups), part = blockIdx.x % (2 * head_groups);
  const uint32_t row = unit * (kThreads / LANES) + threadIdx.x / LANES;
  const uint32_t h0 = (part >> 1) * kHeads;
  const uint32_t d = lane * 8;
  if (row >= n || d >= p.dim) return;
  const int64_t slot = slots[row];
  if (slot < 0 || slot >= static_cast<int64_t>(static_cast<uint64_t>(p.num_blocks) * p.block_size))
    return;
  const uint64_t block = static_cast<uint64_t>(slot) / p.block_size;
  const uint32_t token = static_cast<uint32_t>(static_cast<uint64_t>(slot) - block * p.block_size);
  const RowsView& rows = part & 1 ? v : k;
  const uint64_t segment = (part & 1 ? p.v : p.k) + block * p.block_bytes;
  u32x4 x[kHeads];
  float s[kHeads];
#pragma unroll
  for (uint32_t i = 0; i < kHeads; ++i) {
    const uint32_t h = h0 + i;
    if (h >= p.heads) break;
    const uint64_t at = segment + static_cast<uint64_t>(token) * p.token_bytes +
                        static_cast<uint64_t>(h) * p.head_bytes;
    if constexpr (TYPE == PF_KV_BF16 || TYPE == PF_KV_FP16) {
      x[i] = *reinterpret_cast<const g_u32x4*>(at + d * 2);
    } else {
      const u32x2 c = *reinterpret_cast<const g_u32x2*>(at + d);
      x[i] = u32x4{c[0], c[1], 0, 0};
      s[i] = *reinterpret_cast<const g_f32*>(segment + p.scale_offset +
                                             (h * p.block_size + token) * 4ull);
    }
  }
#pragma unroll
  for (uint32_t i = 0; i < kHeads; ++i) {
    const uint32_t h = h0 + i;
    if (h >= p.heads) break;
    u32x4 y = x[i];
    if constexpr (!(TYPE == PF_KV_BF16 || TYPE == PF_KV_FP16)) {
      float f[8];
      codes_to_float<TYPE>(x[i][0], f);
      codes_to_float<TYPE>(x[i][1], f + 4);
#pragma unroll
      for (int w = 0; w < 4; ++w)
        y[w] = Row::from_float(f[2 * w] * s[i]) | Row::from_float(f[2 * w + 1] * s[i]) << 16;
    }
    store_row8<ALIGNED>(rows.data + (row * rows.token_stride + h * rows.head_stride + d) * 2, y);
  }
}

using RowsKernel = void (*)(PagedView, RowsView, RowsView, const int64_t*, uint32_t, uint32_t);

template <bool WRITE, class Row, uint32_t TYPE, uint32_t LANES, bool ALIGNED>
constexpr RowsKernel kernel() {
  if constexpr (WRITE)
    return kv_write_kernel<Row, TYPE, LANES, ALIGNED>;
  else
    return kv_read_kernel<Row, TYPE, LANES, ALIGNED>;
}

template <bool WRITE, class Row, uint32_t TYPE>
RowsKernel pick(uint32_t lanes, bool aligned) {
  switch (lanes) {
    case 8:
      return aligned ? kernel<WRITE, Row, TYPE, 8, true>() : kernel<WRITE, Row, TYPE, 8, false>();
    case 16:
      return aligned ? kernel<WRITE, Row, TYPE, 16, true>() : kernel<WRITE, Row, TYPE, 16, false>();
    default:
      return aligned ? kernel<WRITE, Row, TYPE, 32, true>() : kernel<WRITE, Row, TYPE, 32, false>();
  }
}

template <bool WRITE, class Row>
RowsKernel pick(uint32_t type, uint32_t lanes, bool aligned) {
  if (type == PF_KV_E4M3) return pick<WRITE, Row, PF_KV_E4M3>(lanes, aligned);
  if (type == PF_KV_INT8) return pick<WRITE, Row, PF_KV_INT8>(lanes, aligned);
  return pick<WRITE, Row, Row::kType>(lanes, aligned);
}

template <bool WRITE>
hipError_t launch_rows(const PagedView& pages, const RowsView& k, const RowsView& v,
                       uint32_t row_type, const int64_t* slots, uint32_t n, bool aligned,
                       hipStream_t stream) {
  if (n == 0) return hipSuccess;
  const uint32_t lanes = pages.dim <= 64 ? 8 : pages.dim <= 128 ? 16 : 32;
  const RowsKernel f = row_type == PF_KV_BF16 ? pick<WRITE, BF16>(pages.type, lanes, aligned)
                                              : pick<WRITE, FP16>(pages.type, lanes, aligned);
  const uint32_t head_groups = (pages.heads + kHeads - 1) / kHeads;
  const uint32_t per = kThreads / lanes;
  const uint64_t grid = static_cast<uint64_t>((n + per - 1) / per) * 2 * head_groups;
  if (grid > 0x7fffffffull) return hipErrorInvalidValue;
  hipLaunchKernelGGL(f, dim3(static_cast<uint32_t>(grid)), dim3(kThreads), 0, stream, pages, k, v,
                     slots, n, head_groups);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_write(const PagedView& pages, const RowsView& k, const RowsView& v,
                           uint32_t row_type, const int64_t* slots, uint32_t n, bool aligned,
                           hipStream_t stream) {
  return launch_rows<true>(pages, k, v, row_type, slots, n, aligned, stream);
}

hipError_t launch_kv_read(const PagedView& pages, const RowsView& k, const RowsView& v,
                          uint32_t row_type, const int64_t* slots, uint32_t n, bool aligned,
                          hipStream_t stream) {
  return launch_rows<false>(pages, k, v, row_type, slots, n, aligned, stream);
}

}  // namespace pf
