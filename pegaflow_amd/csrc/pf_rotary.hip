// pf_rotary.hip — queries and keys turned to their positions, keys and values written
// into a layer's pages in the same pass.
//
// Pair i of a head, (a, b), of the token at position p becomes
//   (c (a cos t - b sin t), c (b cos t + a sin t)),  t = 2 pi p f_i,
// f_i turns a position.  The fraction of p f_i is all that matters, and in fixed point it
// comes by itself: f_i is held as a 64-bit fraction, the product with p is taken modulo
// 2^64, and no position, however far, loses a bit of its angle (p = 2^31 leaves 2^-33
// turns).  The nearest quarter turn is taken off, and sine and cosine of the rest, at most
// pi / 4, are their Taylor sums up to x^9 and x^10: what follows is less than 2^-29, and their fp32
// operations are off by less than 2^-23 in all (2^-23.4 and 2^-23.2 over all 2^30 arguments).  Values
// stay in fp32 from the rows to their one rounding, to the rows' type or to a code.
//
// Bound by HBM: rows are read once and written once, no table of angles is read.  A lane
// takes 8 pairs of a row, its two runs of 8 neighbours, so that a pair never crosses
// lanes (and rows may be turned in place), and keeps their sines and cosines for all heads
// of its workgroup.
//
// 10,000 tokens (32 heads of 128 on 8, bf16, 246 MB) take 48.9 us, 5.0 TB/s where a large copy
// moves 5.1; 64 tokens of a decode step 3.4, 500 4.7, of which the memory works 2.4.  With the
// loads of 4 heads under way, or of 8, 2,000 tokens take 10.2 and 10.9 us, with those of 2 9.8.
#include <hip/hip_runtime.h>

#include "pf_paged_device.h"
#include "pf_rotary.h"

namespace pf {

namespace {

constexpr uint32_t kThreads = kRotaryThreads;
typedef uint16_t __attribute__((may_alias)) any_u16;
constexpr uint32_t kFlight = 2;  // heads whose loads are under way together

// How rows are cut: kWide, kNarrow: whole runs of 8 pairs, loaded by 16 bytes or value by
// value; kPart: neighbours as pairs, of which the last run has some, by 16 bytes; kAnyWide, kAny:
// any even number of turned values, by 16 bytes or value by value, each with a look at its partner
// in shared memory.  (13,900 tokens of 12 heads of 128, fp16, 82 values turned, take 57.8 us by
// kPart and 66.4, in halves, by kAnyWide, 112 where values and partners were loaded one by one; 96
// values 53 by kWide, where tests for a run's pairs, as kPart has them, cost 10,000 tokens 5 of 48.)
enum Path { kWide, kNarrow, kPart, kAnyWide, kAny };

// Cosine and sine of t / 2^64 turns.
__device__ __forceinline__ void turn(uint64_t t, float* c, float* s) {
  const uint32_t u = static_cast<uint32_t>((t + 0x80000000ull) >> 32);
  const uint32_t quarter = (u + 0x20000000u) >> 30;
  const float x = static_cast<float>(static_cast<int32_t>(u - (quarter << 30))) *
                  1.46291807926715968e-9f;  // 2 pi / 2^32
  const float z = x * x;
  float p = __builtin_fmaf(z, 1.0f / 362880, -1.0f / 5040);
  p = __builtin_fmaf(z, p, 1.0f / 120);
  p = __builtin_fmaf(z, p, -1.0f / 6);
  const float sine = __builtin_fmaf(x * z, p, x);
  p = __builtin_fmaf(z, -1.0f / 3628800, 1.0f / 40320);
  p = __builtin_fmaf(z, p, -1.0f / 720);
  p = __builtin_fmaf(z, p, 1.0f / 24);
  p = __builtin_fmaf(z, p, -0.5f);
  const float cosine = __builtin_fmaf(z, p, 1.0f);
  const float cc = quarter & 1 ? sine : cosine, ss = quarter & 1 ? cosine : sine;
  *c = (quarter + 1) & 2 ? -cc : cc;
  *s = quarter & 2 ? -ss : ss;
}

__device__ __forceinline__ void rotate(float& a, float& b, float c, float s) {
  const float x = a, y = b;
  a = __builtin_fmaf(x, c, -(y * s));
  b = __builtin_fmaf(y, c, x * s);
}

template <class Row>
__device__ __forceinline__ void unpack8(u32x4 x, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = Row::to_float(x[i] & 0xffffu);
    f[2 * i + 1] = Row::to_float(x[i] >> 16);
  }
}
template <class Row>
__device__ __forceinline__ u32x4 pack8(const float* f) {
  u32x4 x;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = Row::from_float(f[2 * i]) | Row::from_float(f[2 * i + 1]) << 16;
  return x;
}

// Workgroup b: tokens (b / parts) * groups + group, part b % parts (RotaryParams).
template <class Row, uint32_t TYPE, uint32_t LANES, Path PATH>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryParams p) {
  constexpr bool kAligned = PATH != kNarrow && PATH != kAny;
  constexpr bool kPartners = PATH == kAnyWide || PATH == kAny;
  constexpr uint32_t kAngles = kPartners ? 16 : 8;
  // Rows as they were, for a look at partners: 16 bytes between rows put those of 4 lanes that
  // ask together in other banks.
  constexpr uint32_t kRowWords = LANES * 8 + 4, kRows = 64 / LANES;
  __shared__ uint32_t seen[kPartners ? kThreads / 64 : 1][kPartners ? kFlight : 1]
                          [kPartners ? kRows * kRowWords : 1] __attribute__((aligned(16)));
  const uint32_t lane = threadIdx.x % LANES, parts = p.q_parts + 2 * p.kv_parts;
  const uint32_t unit = blockIdx.x / parts;
  uint32_t part = blockIdx.x % parts;
  const uint32_t row = unit * (kThreads / LANES) + threadIdx.x / LANES;
  if (row >= p.n) return;
  const uint32_t dim = p.pages.dim, r = p.rotary;
  const bool to_pages = part >= p.q_parts;
  bool value = false;  // V, which is not turned
  RowsView rows = p.q;
  uint32_t heads = p.q_heads;
  if (to_pages) {
    part -= p.q_parts;
    value = part >= p.kv_parts;
    if (value) part -= p.kv_parts;
    rows = value ? p.v : p.k;
    heads = p.kv_heads;
  }
  uint64_t segment = 0;  // the block's
  uint32_t token = 0;
  if (to_pages) {
    const int64_t slot = p.slots[row];
    if (slot < 0 ||
        slot >= static_cast<int64_t>(static_cast<uint64_t>(p.pages.num_blocks) * p.pages.block_size))
      return;
    const uint64_t block = static_cast<uint64_t>(slot) / p.pages.block_size;
    token = static_cast<uint32_t>(static_cast<uint64_t>(slot) - block * p.pages.block_size);
    segment = (value ? p.pages.v : p.pages.k) + block * p.pages.block_bytes;
  }
  // This lane's values: d0 to d0 + 7 and d1 to d1 + 7.
  const bool mine = lane * 16 < dim;
  constexpr bool kRuns = PATH == kWide || PATH == kNarrow;
  const bool turned = !value && (kRuns ? lane * 16 + 15 : lane * 16) < r;
  const bool half = PATH != kPart && p.layout == PF_ROTARY_HALF;
  // Of this lane's 8 pairs, those that are turned.
  const uint32_t pairs = PATH != kPart ? 8 : turned ? min((r - lane * 16) / 2, 8u) : 0;
  uint32_t d0 = lane * 16, d1 = d0 + 8;
  if (!kPartners && turned && half) {
    d0 = lane * 8;
    d1 = r / 2 + d0;
  }
  // Value d's pair in a row of any number of turned values, and its partner.
  auto pair_of = [&](uint32_t d) { return half ? (d < r / 2 ? d : d - r / 2) : d / 2; };
  auto partner_of = [&](uint32_t d) { return half ? (d < r / 2 ? d + r / 2 : d - r / 2) : d ^ 1u; };
  float c[kAngles], s[kAngles];
#pragma unroll
  for (uint32_t i = 0; i < kAngles; ++i) {
    c[i] = 1.0f;
    s[i] = 0.0f;
  }
  if (turned) {
    const uint64_t position = static_cast<uint64_t>(p.positions[row]);
    if constexpr (kPartners) {
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i)
        if (d0 + i < r) turn(position * p.turns[pair_of(d0 + i)], &c[i], &s[i]);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i)
        if (i < pairs) turn(position * p.turns[lane * 8 + i], &c[i], &s[i]);
    }
#pragma unroll
    for (uint32_t i = 0; i < kAngles; ++i) {
      if (kPartners && d0 + i >= r) continue;
      c[i] *= p.factor;
      s[i] *= p.factor;
    }
  }
  const uint32_t first = part * p.part_heads, last = min(first + p.part_heads, heads);
  const uint64_t from = rows.data + row * rows.token_stride * 2;
  for (uint32_t h0 = first; h0 < last; h0 += kFlight) {
    u32x4 x[kFlight][2], other[kFlight][2];
#pragma unroll
    for (uint32_t j = 0; j < kFlight; ++j) {
      x[j][0] = x[j][1] = other[j][0] = other[j][1] = u32x4{0, 0, 0, 0};
      const uint64_t at = from + (h0 + j) * rows.head_stride * 2;
      if (mine && h0 + j < last) {
        x[j][0] = load_row8<kAligned>(at + d0 * 2);
        x[j][1] = load_row8<kAligned>(at + d1 * 2);
      }
    }
    if constexpr (kPartners) {
      // A row's lanes are of one wave, whose accesses to shared memory are in order.
#pragma unroll
      for (uint32_t j = 0; j < kFlight; ++j) {
        uint32_t* mem = seen[threadIdx.x / 64][j] + threadIdx.x % 64 / LANES * kRowWords;
        *reinterpret_cast<u32x4*>(mem + lane * 8) = x[j][0];
        *reinterpret_cast<u32x4*>(mem + lane * 8 + 4) = x[j][1];
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (turned) {
#pragma unroll
        for (uint32_t j = 0; j < kFlight; ++j) {
          const any_u16* values = reinterpret_cast<const any_u16*>(
              seen[threadIdx.x / 64][j] + threadIdx.x % 64 / LANES * kRowWords);
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i)
            if (d0 + i < r)
              other[j][i / 8][i / 2 % 4] |= static_cast<uint32_t>(values[partner_of(d0 + i)])
                                            << (i % 2 * 16);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    // Rows that are turned in place are read before they are written.
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (uint32_t j = 0; j < kFlight; ++j) {
      const uint32_t h = h0 + j;
      if (h >= last) break;
      float f[2][8];
      unpack8<Row>(x[j][0], f[0]);
      unpack8<Row>(x[j][1], f[1]);
      if (turned) {
        if constexpr (kPartners) {
          float g[2][8];
          unpack8<Row>(other[j][0], g[0]);
          unpack8<Row>(other[j][1], g[1]);
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i) {
            const uint32_t d = d0 + i;
            if (d >= r) continue;
            const bool second = half ? d >= r / 2 : d & 1u;
            float &x = f[i / 8][i % 8], y = g[i / 8][i % 8] * s[i];
            x = __builtin_fmaf(x, c[i], second ? y : -y);
          }
        } else if (half) {
#pragma unroll
          for (int i = 0; i < 8; ++i) rotate(f[0][i], f[1][i], c[i], s[i]);
        } else {
#pragma unroll
          for (uint32_t i = 0; i < 8; ++i)
            if (i < pairs) rotate(f[i / 4][2 * i % 8], f[i / 4][2 * i % 8 + 1], c[i], s[i]);
        }
      }
      // Values that are not turned go as they are, bit by bit.
      auto words = [&](const float* y, u32x4 was, uint32_t d) {
        if (!turned) return was;
        u32x4 is = pack8<Row>(y);
        if (!kRuns)
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) is[i] = d + 2 * i < r ? is[i] : was[i];
        return is;
      };
      if (!to_pages) {
        const uint64_t to = p.q_out.data + (row * p.q_out.token_stride + h * p.q_out.head_stride) * 2;
        if (mine) {
          store_row8<kAligned>(to + d0 * 2, words(f[0], x[j][0], d0));
          store_row8<kAligned>(to + d1 * 2, words(f[1], x[j][1], d1));
        }
        continue;
      }
      const uint64_t at = segment + static_cast<uint64_t>(token) * p.pages.token_bytes +
                          static_cast<uint64_t>(h) * p.pages.head_bytes;
      if constexpr (TYPE == PF_KV_BF16 || TYPE == PF_KV_FP16) {
        if (mine) {
          store_row8<true>(at + d0 * 2, words(f[0], x[j][0], d0));
          store_row8<true>(at + d1 * 2, words(f[1], x[j][1], d1));
        }
      } else {
        // The largest magnitude, as bits: they order as the values do, with infinity and
        // NaN on top.
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          m = umax(m, __builtin_bit_cast(uint32_t, f[i / 8][i % 8]) & 0x7fffffffu);
        m = group_max<LANES>(m);
        float scale = __builtin_bit_cast(float, m) * kInverseLargest<TYPE>;
        u32x2 c0{0, 0}, c1{0, 0};
        if (m >= 0x7f800000u) {
          scale = __builtin_nanf("");
        } else if (scale > 0.0f) {
          c0 = encode<TYPE>(f[0], scale);
          c1 = encode<TYPE>(f[1], scale);
        }
        if (mine) {
          *reinterpret_cast<g_u32x2*>(at + d0) = c0;
          *reinterpret_cast<g_u32x2*>(at + d1) = c1;
        }
        if (lane == 0)
          *reinterpret_cast<g_f32*>(segment + p.pages.scale_offset +
                                    (h * p.pages.block_size + token) * 4ull) = scale;
      }
    }
  }
}

using RotaryKernel = void (*)(RotaryParams);

template <class Row, uint32_t TYPE, uint32_t LANES>
RotaryKernel pick_path(const RotaryParams& p) {
  if (p.rotary % 16)
    return p.aligned && p.layout == PF_ROTARY_INTERLEAVED ? rotary_kernel<Row, TYPE, LANES, kPart>
           : p.aligned                                    ? rotary_kernel<Row, TYPE, LANES, kAnyWide>
                                                          : rotary_kernel<Row, TYPE, LANES, kAny>;
  return p.aligned ? rotary_kernel<Row, TYPE, LANES, kWide> : rotary_kernel<Row, TYPE, LANES, kNarrow>;
}

template <class Row, uint32_t TYPE>
RotaryKernel pick_lanes(const RotaryParams& p, uint32_t lanes) {
  switch (lanes) {
    case 4: return pick_path<Row, TYPE, 4>(p);
    case 8: return pick_path<Row, TYPE, 8>(p);
    default: return pick_path<Row, TYPE, 16>(p);
  }
}

template <class Row>
hipError_t launch_rotary(const RotaryParams& p, hipStream_t stream) {
  const uint32_t lanes = rotary_lanes(p.pages.dim);
  const RotaryKernel f = p.pages.type == PF_KV_E4M3   ? pick_lanes<Row, PF_KV_E4M3>(p, lanes)
                         : p.pages.type == PF_KV_INT8 ? pick_lanes<Row, PF_KV_INT8>(p, lanes)
                                                      : pick_lanes<Row, Row::kType>(p, lanes);
  hipLaunchKernelGGL(f, dim3(static_cast<uint32_t>(rotary_grid(p))), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rotary_bf16(const RotaryParams& p, hipStream_t stream) {
  return launch_rotary<BF16>(p, stream);
}

hipError_t launch_rotary_fp16(const RotaryParams& p, hipStream_t stream) {
  return launch_rotary<FP16>(p, stream);
}

}  // namespace pf
