// pf_attend.hip — attention of new tokens over a paged cache.
//
// Row r (one new token at position p of a sequence of L tokens, one query head)
// attends the tokens t with t < L, t <= p (causal) and t > p - window:
//   z_t = scale * q . k_t,  m = max z,  w_t = exp(z_t - m),
//   o = sum w_t v_t / sum w_t,  lse = m + log(sum w_t);
// a row that attends none has o = 0 and lse = -inf.  8-bit pages hold codes and a
// scale for each token, which multiplies z_t and w_t instead of the codes.
#include <hip/hip_runtime.h>

#include "pf_paged_device.h"

namespace pf {

namespace {

constexpr float kLn2 = 0.6931471805599453f;

// 8 values of a token at `at` as floats (codes for 8-bit pages).
template <class Row, uint32_t TYPE>
__device__ __forceinline__ void load8(uint64_t at, float* out) {
  if constexpr (TYPE == PF_KV_E4M3 || TYPE == PF_KV_INT8) {
    const u32x2 c = *reinterpret_cast<const g_u32x2*>(at);
    codes_to_float<TYPE>(c[0], out);
    codes_to_float<TYPE>(c[1], out + 4);
  } else {
    const u32x4 x = *reinterpret_cast<const g_u32x4*>(at);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      out[2 * w] = Row::to_float(x[w] & 0xffffu);
      out[2 * w + 1] = Row::to_float(x[w] >> 16);
    }
  }
}

// One wave a row: 64 tokens at a time, a token a lane for the scores, 4 values of
// the output a lane.
template <class Row, uint32_t TYPE>
__global__ void __launch_bounds__(64) attend_kernel(AttendParams a) {
  constexpr bool kCodes = TYPE == PF_KV_E4M3 || TYPE == PF_KV_INT8;
  const PagedView& pg = a.pages;
  const uint32_t lane = threadIdx.x, row = blockIdx.x, qh = blockIdx.y, h = qh / a.group;
  const int32_t total = static_cast<int32_t>(a.num_rows);
  uint32_t seq = a.num_seqs;
  int32_t first = 0, last = 0;
  for (uint32_t b = 0; b < a.num_seqs; ++b) {
    first = min(max(a.query_starts[b], 0), total);
    last = min(max(a.query_starts[b + 1], 0), total);
    if (static_cast<int32_t>(row) >= first && static_cast<int32_t>(row) < last) {
      seq = b;
      break;
    }
  }
  if (seq == a.num_seqs) return;
  const int32_t room = static_cast<int32_t>(a.table_width * pg.block_size);
  const int32_t len = min(max(a.seq_lens[seq], 0), room);
  const int32_t pos = len - (last - first) + (static_cast<int32_t>(row) - first);
  int32_t end = a.causal ? min(len, pos + 1) : len;
  const int32_t window = static_cast<int32_t>(a.window);
  int32_t begin = window && pos >= window ? pos - window + 1 : 0;
  __shared__ float q[256];
  const uint64_t q_at = a.q.data + (row * a.q.token_stride + qh * a.q.head_stride) * 2;
  for (uint32_t d = lane; d < 256; d += 64)
    q[d] = d < pg.dim ? Row::to_float(reinterpret_cast<const g_u16*>(q_at)[d]) : 0.0f;
  __syncthreads();
  float m = -__builtin_inff(), l = 0, o[4] = {0, 0, 0, 0};
  const int32_t* table = a.block_table + seq * a.table_stride;
  for (int32_t t0 = begin; t0 < end; t0 += 64) {
    const int32_t t = t0 + static_cast<int32_t>(lane);
    float z = -__builtin_inff(), vs = 1.0f;
    uint64_t at = 0;
    bool in = false;
    if (t < end) {
      const uint32_t slot = page_of(pg, t), off = t - slot * pg.block_size;
      const int32_t block = table[slot];
      if (block >= 0 && block < static_cast<int32_t>(pg.num_blocks)) {
        in = true;
        const uint64_t base = static_cast<uint64_t>(block) * pg.block_bytes;
        at = base + static_cast<uint64_t>(off) * pg.token_bytes +
             static_cast<uint64_t>(h) * pg.head_bytes;
        float sum = 0;
        for (uint32_t d = 0; d < pg.dim; d += 8) {
          float k[8];
          load8<Row, TYPE>(pg.k + at + d * (kCodes ? 1 : 2), k);
#pragma unroll
          for (int i = 0; i < 8; ++i) sum += q[d + i] * k[i];
        }
        if constexpr (kCodes) {
          const uint64_t s = base + pg.scale_offset + (h * pg.block_size + off) * 4ull;
          sum *= *reinterpret_cast<const g_f32*>(pg.k + s);
          vs = *reinterpret_cast<const g_f32*>(pg.v + s);
        }
        z = sum * a.scale_log2;
      }
    }
    float top = z;
    for (int s = 32; s > 0; s /= 2) top = fmaxf(top, __shfl_xor(top, s));
    const float m_new = fmaxf(m, top), m_use = m_new == -__builtin_inff() ? 0.0f : m_new;
    const float w = in ? exp2f(z - m_use) : 0.0f;
    const float keep = exp2f(m - m_use);
    float sum = w;
    for (int s = 32; s > 0; s /= 2) sum += __shfl_xor(sum, s);
    l = l * keep + sum;
    m = m_new;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] *= keep;
    const int32_t count = min(64, end - t0);
    for (int32_t j = 0; j < count; ++j) {
      if (!__shfl(static_cast<int>(in), j)) continue;
      const float wv = __shfl(w * vs, j);
      const uint64_t v_at = pg.v + __shfl(at, j);
      if (lane * 4 < pg.dim) {
        float v[8];
        load8<Row, TYPE>(v_at + (lane & ~1u) * 4 * (kCodes ? 1 : 2), v);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += wv * (lane & 1 ? v[4 + i] : v[i]);
      }
    }
  }
  const uint64_t out = a.out.data + (row * a.out.token_stride + qh * a.out.head_stride) * 2;
  if (lane * 4 < pg.dim)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<g_u16*>(out)[lane * 4 + i] = Row::from_float(l == 0 ? 0.0f : o[i] / l);
  if (a.lse && lane == 0)
    a.lse[static_cast<uint64_t>(row) * a.q_heads + qh] =
        l == 0 ? -__builtin_inff() : (m + log2f(l)) * kLn2;
}

template <class Row>
hipError_t launch(const AttendParams& p, hipStream_t stream) {
  const dim3 grid(p.num_rows, p.q_heads);
  if (p.pages.type == PF_KV_E4M3)
    hipLaunchKernelGGL((attend_kernel<Row, PF_KV_E4M3>), grid, dim3(64), 0, stream, p);
  else if (p.pages.type == PF_KV_INT8)
    hipLaunchKernelGGL((attend_kernel<Row, PF_KV_INT8>), grid, dim3(64), 0, stream, p);
  else
    hipLaunchKernelGGL((attend_kernel<Row, Row::kType>), grid, dim3(64), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_attend(const AttendParams& p, uint32_t row_type, hipStream_t stream) {
  if (p.num_rows == 0) return hipSuccess;
  return row_type == PF_KV_BF16 ? launch<BF16>(p, stream) : launch<FP16>(p, stream);
}

}  // namespace pf
