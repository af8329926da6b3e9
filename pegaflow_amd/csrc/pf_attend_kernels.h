// pf_attend_kernels.h — attention of new tokens over a paged cache: the kernels,
// included once for each row type (pf_attend_bf16.hip, pf_attend_fp16.hip).
//
// Row r (one new token at position p of a sequence of L tokens, one query head)
// attends the tokens t with t < L, t <= p (causal) and t > p - window:
//   z_t = scale * q . k_t,  m = max z,  w_t = exp(z_t - m),
//   o = sum w_t v_t / sum w_t,  lse = m + log(sum w_t);
// a row that attends none has o = 0 and lse = -inf.  8-bit pages hold codes and a
// scale for each token, which multiplies z_t and w_t instead of the codes: the codes
// are exact in 16 bits.
//
// The rows of a sequence and KV head, its new tokens times the `group` query heads
// that share the head, are one matrix of rows, cut into tiles; a tile passes once over
// the tokens it attends with a running maximum and sum.  Both products are taken
// transposed, S^T = K Q^T and O^T = V^T W^T, so that a lane of the matrix core's result
// holds one row's scores: its maximum and sum need one exchange between two (or four)
// lanes, and the weights are already where the second product reads them.  That product
// reads V^T from LDS with the transposing 16-bit loads.
//
// Weights are rounded to the rows' 16 bits for the product with V: the matrix core takes
// no more, and the rounding, at most half a step of each weight (of fp16 weights 2^-37 of the
// largest at least), is of the size of the output's own.  (Of few rows the rest of each weight
// is multiplied as well.)  Scores, maxima, sums and outputs stay in fp32 until the end.
#pragma once

#include <hip/hip_runtime.h>

#include <utility>

#include "pf_paged_device.h"

namespace pf {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 l_s16x4;

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_inff();

template <class T>
struct Mat;
template <>
struct Mat<BF16> {
  static __device__ __forceinline__ f32x16 mul32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mul16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(x), static_cast<__bf16>(y)});
  }
  static __device__ __forceinline__ f32x2 unpack(uint32_t w) {
    return f32x2{__builtin_bit_cast(float, w << 16), __builtin_bit_cast(float, w & 0xffff0000u)};
  }
};
template <>
struct Mat<FP16> {
  static __device__ __forceinline__ f32x16 mul32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mul16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t,
                              f16x2{static_cast<_Float16>(x), static_cast<_Float16>(y)});
  }
  static __device__ __forceinline__ f32x2 unpack(uint32_t w) {
    const f16x2 h = __builtin_bit_cast(f16x2, w);
    return f32x2{static_cast<float>(h[0]), static_cast<float>(h[1])};
  }
};

constexpr bool is_codes(uint32_t type) { return type == PF_KV_E4M3 || type == PF_KV_INT8; }

// The four codes of a word as 16-bit values of M (exact: 4 and 8 significant bits).
template <class M, uint32_t TYPE>
__device__ __forceinline__ u32x2 codes_to_16(uint32_t word) {
  if constexpr (TYPE == PF_KV_E4M3) {
    if constexpr (M::kType == PF_KV_BF16)
      return u32x2{
          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, 1.0f, false)),
          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, 1.0f, true))};
    else
      return u32x2{
          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.0f, false)),
          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.0f, true))};
  } else if constexpr (M::kType == PF_KV_BF16) {
    // The high halves of the floats hold all of them.
    uint32_t f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f[i] = __builtin_bit_cast(uint32_t,
                                static_cast<float>(static_cast<int8_t>(word >> (8 * i))));
    return u32x2{__builtin_amdgcn_perm(f[1], f[0], 0x07060302u),
                 __builtin_amdgcn_perm(f[3], f[2], 0x07060302u)};
  } else {
    // 0x6400 | u is 1024 + u in fp16; u = code + 128.
    const uint32_t u = word ^ 0x80808080u;
    const f16x2 bias{static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    const uint32_t lo = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
    const uint32_t hi = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, lo) - bias),
                 __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, hi) - bias)};
  }
}

// x of lanes l and l ^ 32, in both lanes and the same order.
__device__ __forceinline__ f32x2 both_halves(float x) {
  const uint32_t y = __builtin_bit_cast(uint32_t, x);
  const u32x2 r = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  const uint32_t r0 = r[0], r1 = r[1];  // a bit_cast of a vector's element takes its first
  return f32x2{__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1)};
}
__device__ __forceinline__ float max32(float x) {
  const f32x2 b = both_halves(x);
  return fmaxf(b[0], b[1]);
}
__device__ __forceinline__ float sum32(float x) {
  const f32x2 b = both_halves(x);
  return b[0] + b[1];
}

// 8 values of a query row (zeros past its end), negated where the scale is negative.
__device__ __forceinline__ u32x4 load_q8(uint64_t row, uint32_t d, const AttendParams& a,
                                         bool valid) {
  u32x4 v{0, 0, 0, 0};
  if (valid && d < a.pages.dim) {
    if (a.aligned) {
      v = *reinterpret_cast<const g_u32x4*>(row + d * 2);
    } else {
      const g_u16* p = reinterpret_cast<const g_u16*>(row + d * 2);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = p[2 * i] | static_cast<uint32_t>(p[2 * i + 1]) << 16;
    }
  }
  return v ^ a.q_sign;
}

// 4 values of an output row.
template <class Row>
__device__ __forceinline__ void store_out4(uint64_t row, uint32_t d, const AttendParams& a,
                                           f32x4 o) {
  if (d >= a.pages.dim) return;
  const u32x2 v{Mat<Row>::pack(o[0], o[1]), Mat<Row>::pack(o[2], o[3])};
  if (a.aligned) {
    *reinterpret_cast<g_u32x2*>(row + d * 2) = v;
  } else {
    g_u16* p = reinterpret_cast<g_u16*>(row + d * 2);
    p[0] = static_cast<uint16_t>(v[0]);
    p[1] = static_cast<uint16_t>(v[0] >> 16);
    p[2] = static_cast<uint16_t>(v[1]);
    p[3] = static_cast<uint16_t>(v[1] >> 16);
  }
}

// Lane N of this lane's 16, an operand of the instruction that uses it.
template <int N>
__device__ __forceinline__ float of16(float x) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x150 + N, 0xf, 0xf, true));
}
// x[i] *= lane FIRST + i of these 16's y.
template <int FIRST, int... I>
__device__ __forceinline__ void scale_by(float* x, float y, std::integer_sequence<int, I...>) {
  ((x[I] *= of16<FIRST + I>(y)), ...);
}

// The maximum that a row's weights are taken against follows its largest score only where that
// has grown by more than 2^lag: until then weights up to that serve as well, and sums and
// outputs need no rescaling.  But the largest weight is 1, which 16 bits hold, only where it
// has followed: 2,000 new bf16 tokens are off by 0.0021 against 64 bits with a lag of 2^3 as of
// 2^8, but where scores are six times as large by 0.0017 and 0.0019.  Prompts of 8,192 tokens
// take 547 and 545 us, and 554 with a lag of 2^1.  Rescaling heads of 256 takes more: 2,000
// behind 2,000 170 and 163, so that bf16 heads of more than 128 keep 2^8 (fp16 ones, whose
// weights need the room, 173 and 163).
template <class Row, uint32_t DP>
constexpr float lag() {
  return Row::kType == PF_KV_FP16 || DP <= 128 ? 3.0f : 8.0f;
}

// fp16 weights over 16-bit pages are held as 2^12 times what they are, l and the outputs with
// them: fp16's smallest step is 2^-24, and a weight off by half of it is then off by 2^-37 of
// its row's largest, so that many small ones keep their sum.  (Held as they are, all under
// 2^-25 were lost, of 30,000 tokens that far under one the whole output.)  With its lag
// none is over 2^15.
constexpr float kFp16Room = 12.0f, kFp16Down = 0x1p-12f;

// A row's maximum m is held in base 2, as its weights exp2(score - m) are taken.  Under a lift
// of its own it is the whole part only: the lift then adds to it exactly, and the weight meets a
// scale before it is rounded anyway.  Elsewhere the largest weight is 1 (or the lift), which 16
// bits hold: with the whole part there as well 2,000 new bf16 tokens were off by 0.0023.

// The log-sum-exp of a row of maximum m and sum l.
template <class Row>
__device__ __forceinline__ float log_sum_exp(const AttendParams& a, float m, float l) {
  if (l == 0) return kNegInf;
  if (Row::kType == PF_KV_FP16 && !is_codes(a.pages.type)) l *= kFp16Down;
  return m * kLn2 + logf(l);
}

// fp16 weights over codes.  A weight meets a code as w s, s the scale of V's token, and s
// may be anything that 32 bits hold, so all weights of a row, its sum l and its outputs
// carry a power of two, 2^lift, until the end: with the largest scale that the row has
// attended s 2^lift is at most 2^12, and w, at most 2^3, makes 2^15 of it.  A product is then a
// normal number down to 2^-25 of the largest scale, and off by 2^-36 of that below.  (bf16
// weights need none of it, but are off by up to 2^-8 where the outputs hold 2^-11.)  A lift
// stops at 2^28: products with scales under 2^-16 are then off by up to 2^-53, of which fp16
// outputs show nothing, and exponents, which it is part of, stay under 32 and are off by 2^-20
// at most, of which a log-sum-exp would show more.
constexpr float kLiftStart = 28.0f, kLiftNone = -100.0f;
// Lowers `lift` (kLiftStart before the first token; kLiftNone for no row) to suit scales
// up to `big` (or 2^66, so that the factor is a normal number: values as large as that
// are infinite in fp16), and returns the factor that the row's sums take.  Other rows of
// the wave have lifts of their own: `limit` is the largest scale that suits them all.
__device__ __forceinline__ float lower_lift(float big, float* lift, float* limit) {
  const float room =
      kFp16Room - static_cast<float>(__builtin_amdgcn_frexp_expf(fminf(big, 0x1p66f)));
  const float old = *lift;
  if (big > 0.0f) *lift = fminf(old, room);
  float most = *lift;
#pragma unroll
  for (int step = 1; step < 64; step *= 2) most = fmaxf(most, __shfl_xor(most, step));
  *limit = __builtin_amdgcn_exp2f(kFp16Room - most);
  return __builtin_amdgcn_exp2f(*lift - old);
}

// V in a tile that some row attends only in part, or that has tokens without a block: a
// weight of 0 must not meet an infinity or NaN, so those values are taken as zero, and the
// tile's caller returns for them at the end (add_odd).  Returns whether there were any among
// these 16 bytes.
template <class Row, uint32_t TYPE>
__device__ __forceinline__ bool clear_odd(u32x4& v) {
  if constexpr (TYPE == PF_KV_INT8) return false;
  u32x4 odd;  // all ones in the values to clear
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (TYPE == PF_KV_E4M3) {  // NaN: 0x7f and a sign
      const uint32_t top = ((v[w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
      odd[w] = (top >> 7) * 0xffu;
    } else {
      const int32_t lo = static_cast<int32_t>(Row::kInf - 1 - (v[w] & 0x7fffu)) >> 31;
      const int32_t hi = static_cast<int32_t>(Row::kInf - 1 - ((v[w] >> 16) & 0x7fffu)) >> 31;
      odd[w] = (static_cast<uint32_t>(lo) & 0xffffu) | (static_cast<uint32_t>(hi) << 16);
    }
    v[w] &= ~odd[w];
  }
  return (odd[0] | odd[1] | odd[2] | odd[3]) != 0;
}

// Adds the infinities and NaN among values d to d + 3 of V of the token at `at` (their
// weights are positive, and infinite either way) to 4 outputs.
template <class Row, uint32_t TYPE>
__device__ __forceinline__ void add_odd(uint64_t at, uint32_t d, uint32_t dim, float* o) {
  if (d + 4 > dim) return;
  float v[4];
  if constexpr (is_codes(TYPE)) {
    codes_to_float<TYPE>(*reinterpret_cast<const g_u32*>(at + d), v);
  } else {
    const u32x2 x = *reinterpret_cast<const g_u32x2*>(at + d * 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = Row::to_float((x[i / 2] >> (16 * (i & 1))) & 0xffffu);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)  // v - v is 0 or NaN
    o[i] += v[i] - v[i] == 0.0f ? 0.0f : v[i];
}

// An output that is NaN while its row's sum is a number met an infinity in V: times a weight
// that 16 bits hold as 0, times the two halves of a weight, of different signs or one of them
// 0, or with one of the other sign.  Only the values themselves tell which: the output is set to
// kLost, those values are added (odd_tokens, add_odd), and where none was it is NaN again.
constexpr float kLost = 3.402823466e38f;
template <int N, uint32_t COUNT, class V>
__device__ __forceinline__ bool any_nan(const V (&o)[COUNT]) {
  // Their sum, by 4 chains: also where two infinities meet, which costs a look in vain.
  float sum[4] = {o[0][0], o[0][1], o[0][2], o[0][3]};
#pragma unroll
  for (uint32_t i = 4; i < COUNT * N; ++i) sum[i % 4] += o[i / N][i % N];
  return __builtin_isunordered(sum[0] + sum[1], sum[2] + sum[3]);
}
template <int N, class V>
__device__ __forceinline__ void lose_nan(V& o) {
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = o[i] != o[i] ? kLost : o[i];
}
template <int N, class V>
__device__ __forceinline__ void restore_nan(V& o) {
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = o[i] == kLost ? __builtin_nanf("") : o[i];
}

// exp2(x), x <= 0, as the factor of a share in a join: never 0, which an infinity would not
// survive (and too small to show in a number).
__device__ __forceinline__ float share_factor(float x) {
  return fmaxf(__builtin_amdgcn_exp2f(x), 0x1p-126f);
}

// A sequence of the batch: its first row, its rows, its tokens.  Starts and lengths
// come from device memory and are bounded here.
struct Seq {
  int32_t first, rows, len;
};
__device__ __forceinline__ Seq seq_of(const AttendParams& a, uint32_t b) {
  const int32_t total = static_cast<int32_t>(a.num_rows);
  const int32_t first = min(max(a.query_starts[b], 0), total);
  const int32_t last = min(max(a.query_starts[b + 1], 0), total);
  const int32_t room = static_cast<int32_t>(a.table_width * a.pages.block_size);
  return {first, max(last - first, 0), min(max(a.seq_lens[b], 0), room)};
}

// The lowest n bits (none for n < 0, all for n > 63).
__device__ __forceinline__ uint64_t bits_below(int32_t n) {
  return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1;
}

// Tokens that the row at position `pos` attends: [begin, end).
__device__ __forceinline__ int32_t row_end(const AttendParams& a, int32_t len, int32_t pos) {
  return a.causal ? max(min(len, pos + 1), 0) : len;
}
__device__ __forceinline__ int32_t row_begin(const AttendParams& a, int32_t pos) {
  const int32_t w = static_cast<int32_t>(a.window);
  return w && pos >= w ? pos - w + 1 : 0;
}

// The share [begin, end) of a tile's tokens that split `split` of `splits` passes over,
// in pieces of `piece` tokens; the last split takes what is left.  Returns the number
// of splits that have a share (at least 1); begin and end mean nothing for the others.
__device__ __forceinline__ uint32_t split_range(int32_t& begin, int32_t& end, uint32_t split,
                                                uint32_t splits, uint32_t piece) {
  const uint32_t n = static_cast<uint32_t>(max(end - begin, 0));
  const uint32_t used = min(max((n + piece - 1) / piece, 1u), splits);
  if (split < used) {
    begin += static_cast<int32_t>(split * piece);
    if (split + 1 < used) end = begin + static_cast<int32_t>(piece);
  }
  return used;
}

// Byte offset of token t's values in K's (or V's) pages, and of its scale; false where
// its block does not exist.
__device__ __forceinline__ bool token_at(const PagedView& p, int32_t block, uint32_t t,
                                         uint32_t page, uint32_t h, uint64_t* at,
                                         uint64_t* scale_at) {
  const uint32_t off = t - page * p.block_size;
  const uint64_t base = static_cast<uint64_t>(static_cast<uint32_t>(block)) * p.block_bytes;
  *at = base + off * p.token_bytes + h * p.head_bytes;
  *scale_at = base + p.scale_offset + (h * p.block_size + off) * 4u;
  return static_cast<uint32_t>(block) < p.num_blocks;
}

// The tokens t0 to t0 + 63 under `end` that have a block and hold V that is not finite, as
// bits: each lane looks at one.
template <class Row, uint32_t TYPE>
__device__ __forceinline__ uint64_t odd_tokens(const PagedView& p, const int32_t* table,
                                               uint32_t head, int32_t t0, int32_t end) {
  const int32_t tok = t0 + static_cast<int32_t>(threadIdx.x & 63u);
  bool odd = false;
  if (tok < end) {
    uint64_t at, scale_at;
    const uint32_t page = page_of(p, tok);
    if (token_at(p, table[page], tok, page, head, &at, &scale_at))
      for (uint32_t d = 0; d < p.dim * (is_codes(TYPE) ? 1 : 2); d += 16) {
        u32x4 v = *reinterpret_cast<const g_u32x4*>(p.v + at + d);
        odd |= clear_odd<Row, TYPE>(v);
      }
  }
  return __ballot(odd);
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup of 4 waves takes 128 rows, or of 8 waves 256, 32 a wave, and 64
// tokens at a time.  K and V of those tokens go through registers into LDS, converted to
// 16 bits, under the previous tile's products; each wave then multiplies its rows with
// them.
//
// Bound by the matrix cores and, close behind, by the softmax on the vector units: 64
// tokens x 32 rows take a wave 32 products of 32 cycles at head size 128, and 2,048
// weights 32 times (multiply-add, exponential, maximum, sum, rounding).  Two waves share
// each vector unit, of two workgroups or one, so that one's products run under the
// other's softmax.  Under such load the clock falls from 2.4 to 1.7-1.9 GHz.
//
// 8,192 new tokens (bf16, 32 heads of 128 on 8) take 532 us, 1,030 TFLOP/s where a large
// product of matrices reaches 1,240; 578 in tiles of 128 rows, which load and store K and
// V twice as often (without that work 484).  2,048 behind 30,000: 963.
// ---------------------------------------------------------------------------
constexpr uint32_t kTileTokens = 64;
constexpr uint32_t kRing = 256;

// Bytes from one token to the next in LDS.  K: 16-byte reads of 16 neighbouring tokens
// fall into different banks.  V: a transposing read takes 64 bytes of each of 4 tokens.
constexpr uint32_t k_pitch(uint32_t dp) { return 2 * dp + 16; }
constexpr uint32_t v_pitch(uint32_t dp) {
  uint32_t p = 2 * dp;
  while (p % 256 != 64 && p % 256 != 192) p += 16;
  return p;
}

template <uint32_t DP>
struct ManyLds {
  // Two tiles in turn where two workgroups still fit the compute unit's 160 KB.
  static constexpr uint32_t kBuffers = DP <= 128 ? 2 : 1;
  struct K {
    __attribute__((aligned(16))) uint8_t data[kTileTokens * k_pitch(DP)];
    __attribute__((aligned(16))) float k_scale[kTileTokens], v_scale[kTileTokens];
  } k[kBuffers];
  struct V {
    __attribute__((aligned(16))) uint8_t data[kTileTokens * v_pitch(DP)];
  } v[kBuffers];
  // Where units of tokens lie in K's (or V's) pages, and their scales, for the tiles to
  // come: a ring of two halves, each filled as the other is used up.  A unit is the tokens
  // that surely share a block (AttendParams::unit_shift); one without a block has a place
  // that may be read, and is not there.
  uint64_t at[kRing], scale_at[kRing];
  uint8_t there[kRing];
  uint32_t odd;  // some tile attended in part holds V that is not finite
};

// The rows tile `index` of the batch, of the sequences with more than `least` rows: its
// sequence and tile in it, false if there is none.  Workgroups start in the order of their
// index, so tiles that attend much come first: up to 64 sequences go by their length, and
// a sequence's tiles from the last.  (Nine sequences of up to 700 new and 4,100 cached
// tokens 305 us, in the order of the batch 347.)
__device__ __forceinline__ bool find_tile(const AttendParams& a, uint32_t index, uint32_t tile_rows,
                                          uint32_t least, uint32_t* seq, uint32_t* tile) {
  const uint32_t lane = threadIdx.x & 63u;
  for (uint32_t b0 = 0; b0 < a.num_seqs; b0 += 64) {
    uint32_t tiles = 0;
    int32_t len = -1;
    if (b0 + lane < a.num_seqs) {
      const Seq s = seq_of(a, b0 + lane);
      const uint32_t rows = static_cast<uint32_t>(s.rows) * a.group;
      if (rows > least) tiles = (rows + tile_rows - 1) / tile_rows;
      len = s.len;
    }
    // Tiles before this lane's sequence, of the 64 at hand.
    uint32_t before = 0;
    const uint32_t count = min(a.num_seqs - b0, 64u);
    for (uint32_t j = 0; j < count; ++j) {
      const int32_t other = __builtin_amdgcn_readlane(len, j);
      const uint32_t n = __builtin_amdgcn_readlane(tiles, j);
      if (other > len || (other == len && j < lane)) before += n;
    }
    const uint64_t here = __ballot(index >= before && index < before + tiles);
    if (here) {
      const int at = __builtin_ctzll(here);
      *seq = b0 + at;
      *tile = __builtin_amdgcn_readlane(before + tiles, at) - 1 - index;
      return true;
    }
#pragma unroll
    for (int step = 1; step < 64; step *= 2) tiles += __shfl_xor(static_cast<int>(tiles), step);
    index -= tiles;
  }
  return false;
}

// A tile of rows: its sequence, the tokens it passes over and this lane's row.
struct ManyTile {
  Seq s;
  uint32_t seq, head, rows, row;  // rows of the sequence and head, and this lane's
  int32_t begin, end;             // tokens of the tile
  int32_t pos0;                   // position of the sequence's first new token
  bool valid;
};
template <uint32_t ROWS>
__device__ __forceinline__ bool many_tile(const AttendParams& a, uint32_t unit, uint32_t head,
                                          uint32_t wave, ManyTile* t) {
  uint32_t tile = 0;
  if (!find_tile(a, unit, ROWS, a.few_rows, &t->seq, &tile)) return false;
  t->seq = __builtin_amdgcn_readfirstlane(t->seq);
  tile = __builtin_amdgcn_readfirstlane(tile);
  t->s = seq_of(a, t->seq);
  t->head = head;
  t->rows = static_cast<uint32_t>(t->s.rows) * a.group;
  const uint32_t row0 = tile * ROWS, last = min(row0 + ROWS, t->rows) - 1;
  t->pos0 = t->s.len - t->s.rows;
  t->begin = row_begin(a, t->pos0 + static_cast<int32_t>(row0 / a.group)) &
             ~static_cast<int32_t>(kTileTokens - 1);
  t->end = row_end(a, t->s.len, t->pos0 + static_cast<int32_t>(last / a.group));
  t->row = row0 + wave * 32 + (threadIdx.x & 31);
  t->valid = t->row < t->rows;
  return true;
}

__device__ __forceinline__ uint64_t row_address(const AttendParams& a, const RowsView& v,
                                                const ManyTile& t) {
  const uint32_t token = t.row / a.group, g = t.row - token * a.group;
  return v.data + ((t.s.first + static_cast<uint64_t>(token)) * v.token_stride +
                   static_cast<uint64_t>(t.head * a.group + g) * v.head_stride) *
                      2;
}

// The log-sum-exp of this lane's row, where asked for.
template <class Row>
__device__ __forceinline__ void many_lse(const AttendParams& a, const ManyTile& t, float m,
                                         float l) {
  if (!a.lse || !t.valid || (threadIdx.x & 32)) return;
  const uint32_t token = t.row / a.group, g = t.row - token * a.group;
  a.lse[(t.s.first + static_cast<uint64_t>(token)) * a.q_heads + t.head * a.group + g] =
      log_sum_exp<Row>(a, m, l);
}

// Outputs of this lane's row, o / l, and its log-sum-exp.
template <class Row, uint32_t DP>
__device__ __forceinline__ void many_store(const AttendParams& a, const ManyTile& t,
                                           const f32x16* o, float m, float l) {
  if (!t.valid) return;
  const uint32_t half = (threadIdx.x >> 5) & 1;
  const float inv = l == 0 ? 0.0f : 1.0f / l;
  const uint64_t row = row_address(a, a.out, t);
#pragma unroll
  for (uint32_t dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      store_out4<Row>(row, dt * 32 + 8 * i + 4 * half, a,
                      f32x4{o[dt][4 * i] * inv, o[dt][4 * i + 1] * inv, o[dt][4 * i + 2] * inv,
                            o[dt][4 * i + 3] * inv});
  many_lse<Row>(a, t, m, l);
}

template <class Row, uint32_t TYPE, uint32_t DP, uint32_t ROWS>
__global__ void __launch_bounds__(2 * ROWS, DP <= 128 ? 2 : 1)
attend_many_kernel(AttendParams a) {
  constexpr uint32_t kThreads = 2 * ROWS, kWaves = ROWS / 32;
  constexpr bool kCodes = is_codes(TYPE);
  constexpr bool kLift = kCodes && Row::kType == PF_KV_FP16;
  constexpr bool kFixed = !kCodes && Row::kType == PF_KV_FP16;
  constexpr uint32_t kPer = kCodes ? 16 : 8;  // values of a 16-byte load
  // Lanes of a token: a power of two, so that a wave's load stays within 16 tokens.
  constexpr uint32_t kCols = (DP <= 64 ? 64 : DP <= 128 ? 128 : 256) / kPer;
  // Tokens of one load of the workgroup, whose threads may be more than a tile needs: then
  // its halves load and store the same.
  constexpr uint32_t kLoadTokens = kThreads / kCols < kTileTokens ? kThreads / kCols : kTileTokens;
  constexpr uint32_t kLoads = kTileTokens / kLoadTokens;
  constexpr uint32_t kKP = k_pitch(DP), kVP = v_pitch(DP);
  constexpr int32_t kStep = kTileTokens;
  using Lds = ManyLds<DP>;
  __shared__ Lds lds;
  const PagedView& pg = a.pages;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, half = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // Heads of one tile are neighbours: with 8 of them each has an XCD's L2 for its pages.
  const uint32_t head = blockIdx.x % pg.heads;
  const uint32_t rest = blockIdx.x / pg.heads;
  uint32_t unit = rest, split = 0, splits = 1;
  if (rest >= a.many_whole) {
    splits = a.many_splits;
    split = (rest - a.many_whole) % splits;
    unit = a.many_whole + (rest - a.many_whole) / splits;
  }
  ManyTile t;
  if (!many_tile<ROWS>(a, unit, head, wave, &t)) return;
  int32_t begin = t.begin, end = t.end;
  const uint32_t used = split_range(begin, end, split, splits, a.many_piece);
  if (split >= used) return;
  begin = __builtin_amdgcn_readfirstlane(begin);
  end = __builtin_amdgcn_readfirstlane(end);
  const int32_t* table = a.block_table + t.seq * a.table_stride;

  // Tokens that every row of the workgroup attends, and this wave's and row's.
  const uint32_t wave0 = __builtin_amdgcn_readfirstlane(t.row), group = a.group;
  const uint32_t tile0 = wave0 - wave * 32, tile_last = min(tile0 + ROWS, t.rows) - 1;
  const int32_t all_begin = row_begin(a, t.pos0 + static_cast<int32_t>(tile_last / group));
  const int32_t all_end = row_end(a, t.s.len, t.pos0 + static_cast<int32_t>(tile0 / group));
  const int32_t pos = t.pos0 + static_cast<int32_t>(t.row / group);
  const int32_t my_begin = row_begin(a, pos);
  const int32_t my_end = t.valid ? row_end(a, t.s.len, pos) : 0;
  const bool wave_rows = wave0 < t.rows;

  u32x4 q[DP / 16];
  const uint64_t q_row = row_address(a, a.q, t);
#pragma unroll
  for (uint32_t kk = 0; kk < DP / 16; ++kk) q[kk] = load_q8(q_row, kk * 16 + half * 8, a, t.valid);

  f32x16 o[DP / 32];
#pragma unroll
  for (uint32_t dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.0f;
  float m = kNegInf, l = 0.0f;
  float lift = t.valid ? kLiftStart : kLiftNone, lift_limit = 0.0f;  // kLift

  // This thread's part of a tile: 16 bytes of tokens my_tok + kLoadTokens * i, values
  // my_d and on, and of 8-bit pages the scales of token 16 * wave + lane (lanes 0 to 15 of
  // the first 4 waves).
  const uint32_t my_tok = tid / kCols % kTileTokens, my_d = (tid % kCols) * kPer;
  const bool my_col = my_d < pg.dim;
  const uint32_t shift = a.unit_shift, in_unit = (1u << shift) - 1, tile_units = kTileTokens >> shift;
  // A load's tokens repeat their place in their unit after at most two loads.
  constexpr uint32_t kOffsets = kLoadTokens < 16 ? 2 : 1;
  uint32_t lane_at[kOffsets];
#pragma unroll
  for (uint32_t i = 0; i < kOffsets; ++i)
    lane_at[i] = ((my_tok + i * kLoadTokens) & in_unit) * pg.token_bytes +
                 (my_col ? my_d : 0) * (kCodes ? 1 : 2);
  const uint32_t lane_scale = (lane & in_unit & 15u) * 4u;
  u32x4 kr[kLoads], vr[kLoads];
  float k_sr = 0.0f, v_sr = 0.0f;
  // The half of the ring that starts with tile n.
  auto fill_ring = [&](uint32_t n) {
    if (tid >= kRing / 2) return;
    const uint32_t unit = n * tile_units + tid;
    const int32_t tok = begin + static_cast<int32_t>(unit << shift);
    const uint32_t page = page_of(pg, min(tok, end - 1));
    const int32_t block = tok < end ? table[page] : -1;
    uint64_t at, scale_at;
    const bool in = token_at(pg, block, tok, page, head, &at, &scale_at);
    lds.at[unit % kRing] = in ? at : 0;
    if constexpr (kCodes) lds.scale_at[unit % kRing] = in ? scale_at : pg.scale_offset;
    lds.there[unit % kRing] = in;
  };
  auto unit_of = [&](uint32_t n, uint32_t tok) {
    return (n * tile_units & (kRing - 1)) + (tok >> shift);
  };
  auto load_k = [&](uint32_t n) {
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i)
      kr[i] = *reinterpret_cast<const g_u32x4*>(
          pg.k + lds.at[unit_of(n, my_tok + i * kLoadTokens)] + lane_at[i % kOffsets]);
    if constexpr (kCodes)
      if (lane < 16 && wave < 4) {
        const uint64_t at = lds.scale_at[unit_of(n, wave * 16 + lane)] + lane_scale;
        k_sr = *reinterpret_cast<const g_f32*>(pg.k + at);
        v_sr = *reinterpret_cast<const g_f32*>(pg.v + at);
      }
  };
  auto load_v = [&](uint32_t n) {
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i)
      vr[i] = *reinterpret_cast<const g_u32x4*>(
          pg.v + lds.at[unit_of(n, my_tok + i * kLoadTokens)] + lane_at[i % kOffsets]);
  };
  auto tokens_there = [&](uint32_t n) { return __ballot(lds.there[unit_of(n, lane)] != 0); };
  // K into LDS.
  auto store_k = [&](uint32_t n) {
    typename Lds::K& tile = lds.k[n % Lds::kBuffers];
    if (my_col)
#pragma unroll
      for (uint32_t i = 0; i < kLoads; ++i) {
        u32x4* to = reinterpret_cast<u32x4*>(tile.data + (my_tok + i * kLoadTokens) * kKP + my_d * 2);
        if constexpr (kCodes) {
          const u32x2 x0 = codes_to_16<Row, TYPE>(kr[i][0]), x1 = codes_to_16<Row, TYPE>(kr[i][1]);
          const u32x2 x2 = codes_to_16<Row, TYPE>(kr[i][2]), x3 = codes_to_16<Row, TYPE>(kr[i][3]);
          to[0] = u32x4{x0[0], x0[1], x1[0], x1[1]};
          to[1] = u32x4{x2[0], x2[1], x3[0], x3[1]};
        } else {
          to[0] = kr[i];
        }
      }
    if constexpr (kCodes)
      if (lane < 16 && wave < 4) {
        tile.k_scale[wave * 16 + lane] = k_sr;
        tile.v_scale[wave * 16 + lane] = v_sr;
      }
  };
  // V of tile n into LDS; `masked`: some row does not attend every token; bit j of
  // `there`: token j has a block.
  auto store_v = [&](uint32_t n, bool masked, uint64_t there) {
    typename Lds::V& tile = lds.v[n % Lds::kBuffers];
    if (masked) {
      bool odd = false;
#pragma unroll
      for (uint32_t i = 0; i < kLoads; ++i) {
        const uint32_t tok = my_tok + i * kLoadTokens;
        if (!(there >> tok & 1u) || begin + static_cast<int32_t>(n * kTileTokens + tok) >= end)
          vr[i] = u32x4{0, 0, 0, 0};
        odd |= clear_odd<Row, TYPE>(vr[i]);
      }
      if (odd && my_col) lds.odd = 1;
    }
    if (my_col)
#pragma unroll
      for (uint32_t i = 0; i < kLoads; ++i) {
        u32x4* to = reinterpret_cast<u32x4*>(tile.data + (my_tok + i * kLoadTokens) * kVP + my_d * 2);
        if constexpr (kCodes) {
          const u32x2 x0 = codes_to_16<Row, TYPE>(vr[i][0]), x1 = codes_to_16<Row, TYPE>(vr[i][1]);
          const u32x2 x2 = codes_to_16<Row, TYPE>(vr[i][2]), x3 = codes_to_16<Row, TYPE>(vr[i][3]);
          to[0] = u32x4{x0[0], x0[1], x1[0], x1[1]};
          to[1] = u32x4{x2[0], x2[1], x3[0], x3[1]};
        } else {
          to[0] = vr[i];
        }
      }
  };
  // S^T of tile n: this lane's row, tokens 32 tt + 8 (i / 4) + 4 half + i % 4.  The reads
  // of one group of products are under way during the group before.
  f32x16 s[2];
  constexpr uint32_t kGroup = 2;  // steps of 16 values: 4 products
  u32x4 kf[2][kGroup][2];
  auto read_k = [&](uint32_t n, uint32_t g, u32x4 (&f)[kGroup][2]) {
    const uint8_t* at = lds.k[n % Lds::kBuffers].data + (lane & 31u) * kKP + half * 16;
#pragma unroll
    for (uint32_t j = 0; j < kGroup; ++j)
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
        f[j][tt] = *reinterpret_cast<const u32x4*>(at + tt * 32 * kKP + (g * kGroup + j) * 32);
  };
  // Scales of the tile: lane i of 16 holds that of this half's token i, and 32 tt on.
  float ks[2], vs[2];
  const uint32_t my_scale = 8 * ((lane & 15u) / 4) + 4 * half + (lane & 3u);
  auto scores = [&](uint32_t n) {
    if constexpr (kCodes)
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        ks[tt] = lds.k[n % Lds::kBuffers].k_scale[32 * tt + my_scale];
        vs[tt] = lds.k[n % Lds::kBuffers].v_scale[32 * tt + my_scale];
      }
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[tt][i] = 0.0f;
#pragma unroll
    for (uint32_t g = 0; g < DP / 16 / kGroup; ++g) {
      if (g + 1 < DP / 16 / kGroup) read_k(n, g + 1, kf[(g + 1) & 1]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (uint32_t j = 0; j < kGroup; ++j)
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
          s[tt] = Mat<Row>::mul32(kf[g & 1][j][tt], q[g * kGroup + j], s[tt]);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (kCodes) {
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = s[tt][i];
        scale_by<0>(x, ks[tt], std::make_integer_sequence<int, 16>());
#pragma unroll
        for (int i = 0; i < 16; ++i) s[tt][i] = x[i];
      }
    }
  };
  // V^T of 16 tokens of tile n, from 16 u on.  They are taken in the order in which a
  // lane holds their weights: 4 half + (0..3), then 8 + 4 half + (0..3).
  const uint32_t quad = lane & 15u;
  const uint32_t v_lane = (half * 4 + quad / 4) * kVP + ((lane >> 4) & 1u) * 32 + (quad & 3u) * 8;
  u32x4 vf[2][DP / 32];
  auto read_v = [&](uint32_t n, int u, u32x4 (&f)[DP / 32]) {
#pragma unroll
    for (uint32_t dt = 0; dt < DP / 32; ++dt) {
      const uint8_t* from = lds.v[n % Lds::kBuffers].data + v_lane + u * 16 * kVP + dt * 64;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((l_s16x4*)(from));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((l_s16x4*)(from + 8 * kVP));
      const u32x2 x = __builtin_bit_cast(u32x2, lo), y = __builtin_bit_cast(u32x2, hi);
      f[dt] = u32x4{x[0], x[1], y[0], y[1]};
    }
  };
  // O^T += V^T W^T.
  auto add_v = [&](const u32x4 (&f)[DP / 32], u32x4 w) {
#pragma unroll
    for (uint32_t dt = 0; dt < DP / 32; ++dt) o[dt] = Mat<Row>::mul32(f[dt], w, o[dt]);
  };
  // Tile n's scores and softmax.  Its product with V follows in the next step, under that
  // tile's softmax: p are the weights of tile n - 1 at first, of tile n at the end.
  u32x4 p[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) p[u] = u32x4{0, 0, 0, 0};
  auto step = [&](int32_t t0, uint32_t n, bool masked, uint64_t hole) {
    __builtin_amdgcn_s_setprio(1);  // ahead of the other workgroup's softmax
    scores(n);
    read_v(n + 1, 0, vf[0]);  // the buffer of tile n - 1
    if (masked) {
      // Bit j of `seen`: this half's token j, of 64, is attended; its scores are tokens
      // 32 tt + 8 (i / 4) + i % 4.
      const int32_t lo = my_begin - t0 - static_cast<int32_t>(4 * half);
      const int32_t hi = my_end - t0 - static_cast<int32_t>(4 * half);
      const uint64_t seen = bits_below(hi) & ~bits_below(lo) & ~(hole >> (4 * half));
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const int32_t word = static_cast<int32_t>(seen >> (32 * tt));
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int b = 8 * (i / 4) + i % 4;
          const uint32_t keep = static_cast<uint32_t>(word << (31 - b) >> 31);
          const float x = s[tt][i];
          s[tt][i] = __builtin_bit_cast(
              float, (__builtin_bit_cast(uint32_t, x) & keep) | (0xff800000u & ~keep));
        }
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[tt][i]);
    top = max32(top);
    top *= a.scale_log2;
    bool grown = __any(top - m > lag<Row, DP>());
    float keep = 1.0f;
    if (grown) {
      const float m_new = fmaxf(m, kLift ? floorf(top) : top);
      keep = m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
    }
    float base = m == kNegInf ? 0.0f : -m;
    if constexpr (kLift) {
      if (__any(fmaxf(vs[0], vs[1]) > lift_limit)) {  // some row may not have room for it
        const float* scale = lds.k[n % Lds::kBuffers].v_scale + 4 * half;
        float big = 0.0f;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            big = fmaxf(big, s[tt][i] == kNegInf ? 0.0f : scale[32 * tt + 8 * (i / 4) + i % 4]);
        keep *= lower_lift(max32(big), &lift, &lift_limit);
        grown = true;
      }
      base += lift;
    }
    if constexpr (kFixed) base += kFp16Room;
    float sum = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (u < 3) read_v(n + 1, u + 1, vf[(u + 1) & 1]);
      __builtin_amdgcn_sched_barrier(0);
      add_v(vf[u & 1], p[u]);
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float z = s[u / 2][8 * (u & 1) + i];
        x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(z, a.scale_log2, base));
        sum += x[i];
      }
      if constexpr (kCodes) {
        if (u & 1)
          scale_by<8>(x, vs[u / 2], std::make_integer_sequence<int, 8>());
        else
          scale_by<0>(x, vs[u / 2], std::make_integer_sequence<int, 8>());
        if (masked) {  // a hidden token's scale may be anything
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (s[u / 2][8 * (u & 1) + i] == kNegInf) x[i] = 0.0f;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) p[u][j] = Mat<Row>::pack(x[2 * j], x[2 * j + 1]);
      asm volatile("" : "+v"(p[u]), "+v"(sum));  // here, beside the products
#pragma unroll
      for (uint32_t i = 0; i < DP / 32; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);    // a product
        __builtin_amdgcn_sched_group_barrier(0x402, 8, 0);  // vector and exponentials
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    l = l * keep + sum;
    if (grown) {  // the outputs up to tile n - 1
#pragma unroll
      for (uint32_t dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] *= keep;
    }
  };

  if (tid == 0) lds.odd = 0;
  // Values past the head's size, and V before the first tile, which meets weights of 0.
#pragma unroll
  for (uint32_t i = 0; i < kLoads; ++i)
#pragma unroll
    for (uint32_t j = 0; j < kPer / 8; ++j) {
      const uint32_t tok = my_tok + i * kLoadTokens;
      if (my_d >= DP) continue;
#pragma unroll
      for (uint32_t b = 0; b < Lds::kBuffers; ++b) {
        if (!my_col)
          reinterpret_cast<u32x4*>(lds.k[b].data + tok * kKP + my_d * 2)[j] = u32x4{0, 0, 0, 0};
        reinterpret_cast<u32x4*>(lds.v[b].data + tok * kVP + my_d * 2)[j] = u32x4{0, 0, 0, 0};
      }
    }
  if (begin < end) {
    fill_ring(0);
    __syncthreads();
    load_k(0);
    uint64_t there = tokens_there(0), v_there = ~0ull;
    bool v_masked = false;
    uint32_t n = 0;
    for (int32_t t0 = begin; t0 < end; t0 += kStep, ++n) {
      const bool masked = t0 < all_begin || t0 + kStep > all_end || ~there;
      if (Lds::kBuffers == 1) __syncthreads();  // the tiles before have been read
      store_k(n);
      if (n) store_v(n - 1, v_masked, v_there);
      if ((n + 1) * tile_units % (kRing / 2) == 0) fill_ring(n + 1);
      __syncthreads();
      read_k(n, 0, kf[0]);
      v_masked = masked;
      v_there = there;
      there = tokens_there(n + 1);
      load_v(n);
      load_k(n + 1);
      if (wave_rows) step(t0, n, masked, ~v_there);
    }
    if (Lds::kBuffers == 1) __syncthreads();
    store_v(n - 1, v_masked, v_there);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      read_v(n - 1, u, vf[u & 1]);
      add_v(vf[u & 1], p[u]);
    }
  }

  if constexpr (kLift) {
    const float down = __builtin_amdgcn_exp2f(-lift);
    l *= down;
#pragma unroll
    for (uint32_t dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[dt][i] *= down;
  }
  __syncthreads();
  bool odd = TYPE != PF_KV_INT8 && lds.odd;
  if constexpr (!kCodes) odd |= __any(t.valid & (l == l) & any_nan<16>(o));
  // Those of every tile: where none was cleared the products have them already, and once
  // more changes nothing.
  if (__builtin_expect(odd, 0)) {
#pragma unroll
    for (uint32_t dt = 0; dt < DP / 32; ++dt) lose_nan<16>(o[dt]);
    for (int32_t t0 = begin; t0 < end; t0 += kStep) {
      const uint64_t tokens = odd_tokens<Row, TYPE>(pg, table, head, t0, end);
      for (uint64_t left = tokens; left; left &= left - 1) {
        const int32_t tok = t0 + __builtin_ctzll(left);
        if (tok < my_begin || tok >= my_end) continue;
        uint64_t at, scale_at;
        const uint32_t page = page_of(pg, tok);
        token_at(pg, table[page], tok, page, head, &at, &scale_at);
#pragma unroll
        for (uint32_t dt = 0; dt < DP / 32; ++dt)
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) {
            float x[4] = {o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2], o[dt][4 * i + 3]};
            add_odd<Row, TYPE>(pg.v + at, dt * 32 + 8 * i + 4 * half, pg.dim, x);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[dt][4 * i + j] = x[j];
          }
      }
      if (!tokens) continue;
      bool settled = true;  // NaN throughout, which nothing changes
#pragma unroll
      for (uint32_t dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i)
          settled &= o[dt][i] != o[dt][i] || dt * 32 + 8 * (i / 4) + 4 * half >= pg.dim;
      if (!__any(t.valid && !settled)) break;
    }
#pragma unroll
    for (uint32_t dt = 0; dt < DP / 32; ++dt) restore_nan<16>(o[dt]);
  }

  l = sum32(l);
  if (used == 1) {
    many_store<Row, DP>(a, t, o, m, l);
    return;
  }
  // This split's share for attend_many_join_kernel: 16 bytes a lane at a time.
  if (!wave_rows) return;
  const uint64_t slot = (rest - a.many_whole) * static_cast<uint64_t>(pg.heads) + head;
  f32x4* part = reinterpret_cast<f32x4*>(a.many_o) + (slot * kWaves + wave) * (DP / 8) * 64 + lane;
#pragma unroll
  for (uint32_t dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      part[(dt * 4 + i) * 64] = f32x4{o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2],
                                      o[dt][4 * i + 3]};
  reinterpret_cast<f32x2*>(a.many_ml)[(slot * kWaves + wave) * 64 + lane] = f32x2{m, l};
}

// Joins the shares of split tiles.  A wave takes 32 rows and 32 values of each, in the
// lanes that held them.  Of more than kJoinFew shares (TURNS) the 4 waves of a workgroup
// take turns and join in LDS: 20 rows of 32 heads behind 2,000 tokens, in 8 shares, 17.8
// us and otherwise 22.2; behind 10,000, in 40, 27.3 (48.7 where a wave joined the rows'
// whole outputs).  Of few shares each wave takes other values, in a quarter of the
// workgroups: 500 rows behind 10,000, in 4 shares, 9.1 us of this kernel and otherwise 10.7.
constexpr uint32_t kJoinThreads = 256;
constexpr uint32_t kJoinFew = 4;
// Workgroups of 32 rows.
constexpr uint32_t join_parts(uint32_t dp, bool turns) {
  return turns ? dp / 32 : (dp / 32 + 3) / 4;
}
template <class Row, uint32_t DP, uint32_t ROWS, bool TURNS>
__global__ void __launch_bounds__(kJoinThreads) attend_many_join_kernel(AttendParams a) {
  constexpr uint32_t kWaves = ROWS / 32, kJoinWaves = kJoinThreads / 64;
  __shared__ f32x4 join_o[kJoinWaves][4][64];
  __shared__ f32x2 join_ml[kJoinWaves][64];
  const PagedView& pg = a.pages;
  const uint32_t lane = threadIdx.x & 63u, mine = threadIdx.x >> 6, half = lane >> 5;
  constexpr uint32_t kParts = join_parts(DP, TURNS), kStep = TURNS ? kJoinWaves : 1;
  const uint32_t dt = TURNS ? blockIdx.x % kParts : blockIdx.x % kParts * kJoinWaves + mine;
  const uint32_t wave = blockIdx.x / kParts % kWaves, rest = blockIdx.x / kParts / kWaves;
  const uint32_t head = rest % pg.heads, left = rest / pg.heads;
  ManyTile t;
  if (!many_tile<ROWS>(a, a.many_whole + left, head, wave, &t)) return;
  if (__builtin_amdgcn_readfirstlane(t.row) >= t.rows) return;
  int32_t begin = t.begin, end = t.end;
  const uint32_t used = split_range(begin, end, 0, a.many_splits, a.many_piece);
  if (used == 1) return;
  auto slot = [&](uint32_t split) {
    return ((static_cast<uint64_t>(left) * a.many_splits + split) * pg.heads + head) * kWaves + wave;
  };
  const f32x2* ml = reinterpret_cast<const f32x2*>(a.many_ml) + lane;
  const f32x4* part = reinterpret_cast<const f32x4*>(a.many_o) + dt * 4 * 64 + lane;
  if (!TURNS && dt >= DP / 32) return;
  const uint32_t first = TURNS ? mine : 0;
  float m = kNegInf, l = 0.0f;
#pragma unroll 4
  for (uint32_t s = first; s < used; s += kStep) m = fmaxf(m, ml[slot(s) * 64][0]);
  // A share without a maximum attended nothing, or only what is no number (l is NaN).
  auto factor = [&](f32x2 x, float top) {
    return x[0] == kNegInf ? (x[1] == 0.0f ? 0.0f : 1.0f)
                           : share_factor(x[0] - top);
  };
  f32x4 o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = f32x4{0, 0, 0, 0};
#pragma unroll 4
  for (uint32_t s = first; s < used; s += kStep) {
    const f32x2 x = ml[slot(s) * 64];
    const float keep = factor(x, m);
    l += x[1] * keep;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 y = part[slot(s) * (DP / 8) * 64 + i * 64];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] += y[j] * keep;
    }
  }
  auto store = [&](uint32_t i, f32x4 x, float sum) {
    const float inv = sum == 0 ? 0.0f : 1.0f / sum;
    store_out4<Row>(row_address(a, a.out, t), dt * 32 + 8 * i + 4 * half, a,
                    f32x4{x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv});
  };
  if constexpr (!TURNS) {
    if (!t.valid) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) store(i, o[i], l);
    if (dt == 0) many_lse<Row>(a, t, m, l);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) join_o[mine][i][lane] = o[i];
  join_ml[mine][lane] = f32x2{m, l};
  __syncthreads();
  float top = kNegInf, sum = 0.0f;
#pragma unroll
  for (uint32_t w = 0; w < kJoinWaves; ++w) top = fmaxf(top, join_ml[w][lane][0]);
  f32x4 x{0, 0, 0, 0};
#pragma unroll
  for (uint32_t w = 0; w < kJoinWaves; ++w) {
    const f32x2 y = join_ml[w][lane];
    const float keep = factor(y, top);
    sum += y[1] * keep;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] += join_o[w][mine][lane][j] * keep;
  }
  if (!t.valid) return;
  store(mine, x, sum);
  if (dt == 0 && mine == 0) many_lse<Row>(a, t, top, sum);
}

// ---------------------------------------------------------------------------
// Few rows: single tokens and short drafts, up to 16 rows of a KV head.  Bound by
// reading the pages.  Each wave of a workgroup passes over tokens of its own, 32 at a
// time, with no barrier: K goes from memory straight into the operand's registers
// (lane: token lane % 16, 8 or 16 values), V through the wave's own part of LDS.  The
// next 32 tokens are on their way meanwhile.  At the end the 4 waves join in LDS, and
// the shares of a split sequence in the workgroup that finishes last.
//
// 64 sequences of up to 16,000 e4m3 tokens (8 heads of 128, 1.03 GB) take 227 us, 4.5
// TB/s where a large copy moves 5.2.  32 sequences behind 1,000 fp16 tokens (12 heads of
// 64, 57 MB) take 16, of which the memory works some 10 and the rest is the start, the
// first loads and the end; one behind 10,000 (8 heads of 128, 41 MB) 16, 12.8 of them the
// pass and 3.2 the join (4.5 where a share's values were not asked for before its factor
// was known).  Eight waves a workgroup, or tokens under way two tiles ahead (16.1 ->
// 17.5), gained nothing.
// ---------------------------------------------------------------------------
constexpr uint32_t kFewWaves = 4, kFewThreads = kFewWaves * 64;
constexpr uint32_t kFewTokens = 32;
constexpr uint32_t few_v_pitch(uint32_t dp) { return 2 * dp + 32; }

// Values d to d + 3 of an output row, o / l, and with the first the log-sum-exp.
template <class Row>
__device__ __forceinline__ void few_store(const AttendParams& a, const Seq& sq, uint32_t head,
                                          uint32_t row, uint32_t d, f32x4 o, float m, float l) {
  const float inv = l == 0 ? 0.0f : 1.0f / l;
  const uint32_t token = row / a.group, g = row - token * a.group;
  const uint64_t at = sq.first + static_cast<uint64_t>(token), qh = head * a.group + g;
  store_out4<Row>(a.out.data + (at * a.out.token_stride + qh * a.out.head_stride) * 2, d, a,
                  f32x4{o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv});
  if (a.lse && d == 0) a.lse[at * a.q_heads + qh] = log_sum_exp<Row>(a, m, l);
}

template <class Row, uint32_t TYPE, uint32_t DP>
__global__ void __launch_bounds__(kFewThreads, DP <= 128 ? 2 : 1)
attend_few_kernel(AttendParams a) {
  constexpr bool kCodes = is_codes(TYPE);
  constexpr bool kLift = kCodes && Row::kType == PF_KV_FP16;
  constexpr bool kFixed = !kCodes && Row::kType == PF_KV_FP16;
  constexpr uint32_t kPer = kCodes ? 16 : 8;
  constexpr uint32_t kKLoads = DP / (4 * kPer) + (DP % (4 * kPer) ? 1 : 0);  // of 16 tokens
  constexpr uint32_t kCols = DP / kPer;
  constexpr uint32_t kVLoads = (kFewTokens * kCols + 63) / 64;
  constexpr uint32_t kVP = few_v_pitch(DP);
  constexpr uint32_t kSteps = kKLoads * (kCodes ? 2 : 1);  // products of 32 values
  struct WaveLds {
    __attribute__((aligned(16))) uint8_t v[kFewTokens * kVP];
    // Of 32 tokens to load next: where they lie; of the tile at hand: its scales.
    uint64_t at[kFewTokens];
    __attribute__((aligned(16))) float k_scale[kFewTokens], v_scale[kFewTokens];
  };
  __shared__ WaveLds lds[kFewWaves];
  __shared__ float join_m[kFewWaves][16], join_l[kFewWaves][16];
  __shared__ bool finished;
  const PagedView& pg = a.pages;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, col = lane & 15u, quarter = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t head = blockIdx.x % pg.heads;
  const uint32_t rest = blockIdx.x / pg.heads;
  const uint32_t split = rest % a.few_splits, seq = rest / a.few_splits;
  const int32_t* table = a.block_table + seq * a.table_stride;
  // Without a window a share starts at a token known from here on: a launch that is all
  // latency asks for its first block beside the sequence's length (a token behind 10,000
  // gains 0.8 us; where shares wait for their turn it costs 2%).
  const bool ask_early = !a.window && gridDim.x <= 512;
  int32_t early_block = -1;
  if (ask_early)
    early_block = table[page_of(pg, min(split * a.few_piece + wave * kFewTokens + (lane & 31u),
                                        a.table_width * pg.block_size - 1))];
  const Seq sq = seq_of(a, seq);
  uint32_t rows = static_cast<uint32_t>(sq.rows) * a.group;
  if (rows > kFewRows) {
    if (a.many_units) return;  // attend_many_kernel's
    rows = kFewRows;
  }
  if (rows > a.few_rows_most) rows = a.few_rows_most;  // more than the batch was said to have
  if (rows == 0) return;
  const int32_t pos0 = sq.len - sq.rows;
  uint8_t* v_lds = lds[wave].v;

  const uint32_t row = col, last = rows - 1;
  const bool valid = row < rows;
  const int32_t pos = pos0 + static_cast<int32_t>(row / a.group);
  const int32_t my_begin = row_begin(a, pos);
  const int32_t my_end = valid ? row_end(a, sq.len, pos) : 0;
  int32_t begin = row_begin(a, pos0) &
                  ~static_cast<int32_t>(kFewTokens - 1);
  int32_t end = row_end(a, sq.len, pos0 + static_cast<int32_t>(last / a.group));
  const int32_t all_begin = row_begin(a, pos0 + static_cast<int32_t>(last / a.group));
  const int32_t all_end = row_end(a, sq.len, pos0);
  const uint32_t used = split_range(begin, end, split, a.few_splits, a.few_piece);
  if (split >= used) return;
  const uint32_t token = row / a.group, g = row - token * a.group;
  const uint64_t q_row = a.q.data + ((sq.first + static_cast<uint64_t>(token)) * a.q.token_stride +
                                     static_cast<uint64_t>(head * a.group + g) * a.q.head_stride) *
                                        2;
  u32x4 q[kSteps];
#pragma unroll
  for (uint32_t i = 0; i < kSteps; ++i)
    q[i] = load_q8(q_row,
                   kCodes ? (i / 2) * 64 + quarter * 16 + (i & 1) * 8 : i * 32 + quarter * 8, a,
                   valid);
  f32x4 o[DP / 16];
#pragma unroll
  for (uint32_t dt = 0; dt < DP / 16; ++dt) o[dt] = f32x4{0, 0, 0, 0};
  float m = kNegInf, l = 0.0f;
  bool odd = false;  // some tile attended in part holds V that is not finite
  float lift = valid ? kLiftStart : kLiftNone, lift_limit = 0.0f;  // kLift

  u32x4 kr[2][kKLoads], vr[kVLoads];
  // Token t0 + lane of a tile, lanes 0 to 31: its block (of the tile to load next), its
  // place and, once the tile is on its way, its scales.  A token past the end or
  // without a block reads some other place: it is masked and its V zeroed.
  int32_t block = -1;
  float k_scale = 0.0f, v_scale = 0.0f;
  uint32_t there = 0;  // bit j: token j of the tile has a block
  auto load_block = [&](int32_t t0) {
    const int32_t tok = t0 + static_cast<int32_t>(lane & 31u);
    block = tok < end ? table[page_of(pg, tok)] : -1;
  };
  // d of this lane's part of K and V (some other value where there is none).
  uint32_t k_at[kKLoads], v_at[kVLoads];
#pragma unroll
  for (uint32_t i = 0; i < kKLoads; ++i) {
    const uint32_t d = (i * 4 + quarter) * kPer;
    k_at[i] = (d < pg.dim ? d : 0) * (kCodes ? 1 : 2);
  }
#pragma unroll
  for (uint32_t i = 0; i < kVLoads; ++i) {
    const uint32_t d = (lane + i * 64) % kCols * kPer;
    v_at[i] = (d < pg.dim ? d : 0) * (kCodes ? 1 : 2);
  }
  auto load = [&](int32_t t0) {
    const int32_t tok = t0 + static_cast<int32_t>(lane & 31u);
    uint64_t place, scale_place;
    const bool in =
        token_at(pg, block, tok, page_of(pg, tok), head, &place, &scale_place);
    there = static_cast<uint32_t>(__ballot(in));
    if (lane < 32) {
      lds[wave].at[lane] = in ? place : 0;
      if constexpr (kCodes) {
        if (!in) scale_place = pg.scale_offset;
        k_scale = *reinterpret_cast<const g_f32*>(pg.k + scale_place);
        v_scale = *reinterpret_cast<const g_f32*>(pg.v + scale_place);
      }
    }
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const uint64_t at = pg.k + lds[wave].at[tt * 16 + col];
#pragma unroll
      for (uint32_t i = 0; i < kKLoads; ++i)
        kr[tt][i] = *reinterpret_cast<const g_u32x4*>(at + k_at[i]);
    }
#pragma unroll
    for (uint32_t i = 0; i < kVLoads; ++i)
      vr[i] = *reinterpret_cast<const g_u32x4*>(
          pg.v + lds[wave].at[(lane + i * 64) / kCols] + v_at[i]);
  };

  constexpr int32_t kStep = kFewTokens * kFewWaves;
  auto tile = [&](int32_t t0) {
    const bool partial = t0 < all_begin || t0 + static_cast<int32_t>(kFewTokens) > all_end;
    const bool masked = partial || there != 0xffffffffu;
    // V into LDS.
    if (masked) {
#pragma unroll
      for (uint32_t i = 0; i < kVLoads; ++i) {
        const uint32_t j = (lane + i * 64) / kCols;
        if (!(there >> j & 1u)) vr[i] = u32x4{0, 0, 0, 0};
        odd |= clear_odd<Row, TYPE>(vr[i]);
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < kVLoads; ++i) {
      const uint32_t c = lane + i * 64, j = c / kCols, cc = c % kCols;
      u32x4 v0 = vr[i], v1{0, 0, 0, 0};
      if constexpr (kCodes) {
        const u32x2 b0 = codes_to_16<Row, TYPE>(vr[i][0]), b1 = codes_to_16<Row, TYPE>(vr[i][1]);
        const u32x2 b2 = codes_to_16<Row, TYPE>(vr[i][2]), b3 = codes_to_16<Row, TYPE>(vr[i][3]);
        v0 = u32x4{b0[0], b0[1], b1[0], b1[1]};
        v1 = u32x4{b2[0], b2[1], b3[0], b3[1]};
      }
      u32x4* vd = reinterpret_cast<u32x4*>(v_lds + j * kVP + cc * (kCodes ? 32 : 16));
      vd[0] = v0;
      if constexpr (kCodes) vd[1] = v1;
    }
    if constexpr (kCodes) {
      if (lane < 32) {
        lds[wave].k_scale[lane] = k_scale;
        lds[wave].v_scale[lane] = v_scale;
      }
    }
    if (pg.dim != DP) {  // values past the head's size
#pragma unroll
      for (uint32_t i = 0; i < kKLoads; ++i)
        if ((i * 4 + quarter) * kPer >= pg.dim) kr[0][i] = kr[1][i] = u32x4{0, 0, 0, 0};
    }
    // S^T: this lane's row `col`, tokens 16 tt + 4 quarter + i.
    f32x4 s[2];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      s[tt] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (uint32_t i = 0; i < kKLoads; ++i) {
        if constexpr (kCodes) {
          const u32x2 a0 = codes_to_16<Row, TYPE>(kr[tt][i][0]);
          const u32x2 a1 = codes_to_16<Row, TYPE>(kr[tt][i][1]);
          const u32x2 a2 = codes_to_16<Row, TYPE>(kr[tt][i][2]);
          const u32x2 a3 = codes_to_16<Row, TYPE>(kr[tt][i][3]);
          s[tt] = Mat<Row>::mul16(u32x4{a0[0], a0[1], a1[0], a1[1]}, q[2 * i], s[tt]);
          s[tt] = Mat<Row>::mul16(u32x4{a2[0], a2[1], a3[0], a3[1]}, q[2 * i + 1], s[tt]);
        } else {
          s[tt] = Mat<Row>::mul16(kr[tt][i], q[i], s[tt]);
        }
      }
    }
    float wv[2][4];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      f32x4 x{1, 1, 1, 1}, y{1, 1, 1, 1};
      if constexpr (kCodes) {
        x = *reinterpret_cast<const f32x4*>(lds[wave].k_scale + tt * 16 + quarter * 4);
        y = *reinterpret_cast<const f32x4*>(lds[wave].v_scale + tt * 16 + quarter * 4);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (kCodes) s[tt][i] *= x[i];
        wv[tt][i] = y[i];
      }
    }
    const uint32_t seen_blocks = there;
    const bool lower = kLift && __any(v_scale > lift_limit);
    if (t0 + kStep < end) {
      load(t0 + kStep);
      load_block(t0 + 2 * kStep);
    }
    if (masked) {
      // Bit 16 tt + i: this lane's token 16 tt + 4 quarter + i is attended.
      const int32_t at = t0 + static_cast<int32_t>(quarter) * 4;
      const uint32_t seen =
          static_cast<uint32_t>(bits_below(my_end - at) & ~bits_below(my_begin - at)) &
          (seen_blocks >> (quarter * 4));
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t keep =
              static_cast<uint32_t>(static_cast<int32_t>(seen << (31 - tt * 16 - i)) >> 31);
          const float x = s[tt][i], y = wv[tt][i];
          s[tt][i] = __builtin_bit_cast(
              float, (__builtin_bit_cast(uint32_t, x) & keep) | (0xff800000u & ~keep));
          wv[tt][i] = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, y) & keep);
        }
    }
    float top = kNegInf;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, s[tt][i]);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = max32(top);
    top *= a.scale_log2;
    if (__any(top - m > lag<Row, DP>())) {
      const float m_new = fmaxf(m, kLift ? floorf(top) : top);
      const float keep = m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= keep;
#pragma unroll
      for (uint32_t dt = 0; dt < DP / 16; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[dt][i] *= keep;
    }
    float base = m == kNegInf ? 0.0f : -m;
    if constexpr (kLift) {
      if (lower) {  // a scale that some row may not have room for; hidden ones are 0 here
        float big = 0.0f;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) big = fmaxf(big, wv[tt][i]);
        big = fmaxf(big, __shfl_xor(big, 16));
        const float keep = lower_lift(max32(big), &lift, &lift_limit);
        l *= keep;
#pragma unroll
        for (uint32_t dt = 0; dt < DP / 16; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[dt][i] *= keep;
      }
      base += lift;
    }
    if constexpr (kFixed) base += kFp16Room;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[tt][i], a.scale_log2, base));
        l += w;
        wv[tt][i] *= w;
      }
    // Each weight as two numbers of 16 bits, the second what the first's rounding left: the
    // matrix cores have time here, and outputs are off by little more than their own
    // rounding (twice that with the first alone, of a few tokens).  The product costs 2% at
    // 32 sequences behind 1,000 tokens, and nothing measurable elsewhere.
    u32x4 w, rest;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = wv[i / 2][2 * (i & 1)], y = wv[i / 2][2 * (i & 1) + 1];
      const uint32_t word = Mat<Row>::pack(x, y);
      const f32x2 held = Mat<Row>::unpack(word);
      w[i] = word;
      float rest_x = x - held[0], rest_y = y - held[1];
      if constexpr (kCodes) {  // an infinite scale leaves no number
        rest_x = rest_x == rest_x ? rest_x : 0.0f;
        rest_y = rest_y == rest_y ? rest_y : 0.0f;
      }
      rest[i] = Mat<Row>::pack(rest_x, rest_y);
    }
    // Every lane of the wave has stored its part of V before any reads another's.
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const uint8_t* v_from = v_lds + (quarter * 4 + col / 4) * kVP + (col & 3u) * 8;
#pragma unroll
    for (uint32_t dt = 0; dt < DP / 16; ++dt) {
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((l_s16x4*)(v_from + dt * 32));
      const s16x4 hi =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((l_s16x4*)(v_from + 16 * kVP + dt * 32));
      const u32x2 x = __builtin_bit_cast(u32x2, lo), y = __builtin_bit_cast(u32x2, hi);
      o[dt] = Mat<Row>::mul16(u32x4{x[0], x[1], y[0], y[1]}, w, o[dt]);
      o[dt] = Mat<Row>::mul16(u32x4{x[0], x[1], y[0], y[1]}, rest, o[dt]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  int32_t t0 = begin + static_cast<int32_t>(wave * kFewTokens);
  if (t0 < end) {
    if (ask_early)
      block = t0 + static_cast<int32_t>(lane & 31u) < end ? early_block : -1;
    else
      load_block(t0);
    load(t0);
    load_block(t0 + kStep);
  }
  for (; t0 < end; t0 += kStep) tile(t0);
  if constexpr (kLift) {
    const float down = __builtin_amdgcn_exp2f(-lift);
    l *= down;
#pragma unroll
    for (uint32_t dt = 0; dt < DP / 16; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[dt][i] *= down;
  }
  // Those of all of this wave's tiles, as in attend_many_kernel.
  if constexpr (!kCodes) odd |= valid & (l == l) & any_nan<4>(o);
  if (TYPE != PF_KV_INT8 && __builtin_expect(__any(odd), 0)) {
#pragma unroll
    for (uint32_t dt = 0; dt < DP / 16; ++dt) lose_nan<4>(o[dt]);
    for (int32_t t1 = begin + static_cast<int32_t>(wave * kFewTokens); t1 < end; t1 += kStep) {
      const uint64_t tokens = odd_tokens<Row, TYPE>(
          pg, table, head, t1, min(end, t1 + static_cast<int32_t>(kFewTokens)));
      for (uint64_t left = tokens; left; left &= left - 1) {
        const int32_t tok = t1 + __builtin_ctzll(left);
        if (tok < my_begin || tok >= my_end) continue;
        uint64_t at, scale_at;
        const uint32_t page = page_of(pg, tok);
        token_at(pg, table[page], tok, page, head, &at, &scale_at);
#pragma unroll
        for (uint32_t dt = 0; dt < DP / 16; ++dt) {
          float x[4] = {o[dt][0], o[dt][1], o[dt][2], o[dt][3]};
          add_odd<Row, TYPE>(pg.v + at, dt * 16 + quarter * 4, pg.dim, x);
          o[dt] = f32x4{x[0], x[1], x[2], x[3]};
        }
      }
      if (!tokens) continue;
      bool settled = true;
#pragma unroll
      for (uint32_t dt = 0; dt < DP / 16; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          settled &= o[dt][i] != o[dt][i] || dt * 16 + quarter * 4 >= pg.dim;
      if (!__any(valid && !settled)) break;
    }
#pragma unroll
    for (uint32_t dt = 0; dt < DP / 16; ++dt) restore_nan<4>(o[dt]);
  }

  // Join the waves: each puts its outputs, 16 rows x DP in fp32, into its own part of
  // LDS (which V no longer needs), and the threads share the sums.
  l += __shfl_xor(l, 16);
  l = sum32(l);
  float* mine = reinterpret_cast<float*>(lds[wave].v);
  static_assert(sizeof(WaveLds) >= 16 * DP * sizeof(float), "a wave's outputs fit its LDS");
#pragma unroll
  for (uint32_t dt = 0; dt < DP / 16; ++dt)
    *reinterpret_cast<f32x4*>(mine + col * DP + dt * 16 + quarter * 4) = o[dt];
  if (quarter == 0) {
    join_m[wave][col] = m;
    join_l[wave][col] = l;
  }
  __syncthreads();
  const uint64_t slot = (static_cast<uint64_t>(seq) * a.few_splits + split) * pg.heads + head;
  const __amdgpu_buffer_rsrc_t share = __builtin_amdgcn_make_buffer_rsrc(
      a.few_o + (used > 1 ? slot * a.few_rows_most * DP : 0), 0,
      static_cast<int>(a.few_rows_most * DP * 4), 0x00027000);
  for (uint32_t i = tid; i < 16 * DP / 4; i += kFewThreads) {
    const uint32_t r = i / (DP / 4), d = i % (DP / 4) * 4;
    if (r >= rows) continue;
    float top = kNegInf;
#pragma unroll
    for (uint32_t w = 0; w < kFewWaves; ++w) top = fmaxf(top, join_m[w][r]);
    float sum = 0.0f;
    f32x4 x{0, 0, 0, 0};
#pragma unroll
    for (uint32_t w = 0; w < kFewWaves; ++w) {
      const float mw = join_m[w][r], lw = join_l[w][r];
      const float keep = mw == kNegInf ? (lw == 0.0f ? 0.0f : 1.0f)
                                       : share_factor(mw - top);
      sum += lw * keep;
      const f32x4 y =
          *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds[w].v) + r * DP + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] += y[j] * keep;
    }
    if (used > 1) {
      // Written through the XCD's L2 (the sc1 policy of agent-scope stores, which the
      // language offers for at most 8 bytes at a time).
      constexpr int kSc1 = 16;
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), share,
                                             static_cast<int>((r * DP + d) * 4), 0, kSc1);
      if (d == 0)
        __hip_atomic_store(reinterpret_cast<uint64_t*>(a.few_ml) + slot * a.few_rows_most + r,
                           __builtin_bit_cast(uint64_t, f32x2{top, sum}), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
    } else {
      few_store<Row>(a, sq, head, r, d, x, top, sum);
    }
  }
  if (used == 1) return;
  // The split that finishes last joins them all, in order.  Shares go through the XCD's
  // L2 to where every XCD sees them; a workgroup counts itself once its stores have been
  // acknowledged, and the last one puts the count back to 0 for the next call.
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  uint32_t* count = a.few_count + (static_cast<uint64_t>(seq) * pg.heads + head) * kCountStride;
  if (tid == 0) {
    const uint32_t before =
        __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (before + 1 == used)
      __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    finished = before + 1 == used;
  }
  __syncthreads();
  if (!finished) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  const uint64_t slot0 = static_cast<uint64_t>(seq) * a.few_splits * pg.heads + head;
  const f32x2* ml = reinterpret_cast<const f32x2*>(a.few_ml);
  // 4 values an item; where there are fewer items than threads, groups of threads share
  // the splits out and add up in LDS.
  const uint32_t items = rows * (DP / 4);
  uint32_t groups = 1;
  while (groups * 2 * items <= kFewThreads) groups *= 2;
  const uint32_t group = tid / items;
  const uint64_t stride = static_cast<uint64_t>(pg.heads) * a.few_rows_most * DP;
  const uint32_t first = groups > 1 ? group : 0;
  auto part = [&](uint32_t i, uint32_t s) {
    return *reinterpret_cast<const f32x4*>(a.few_o + (slot0 * a.few_rows_most + i / (DP / 4)) * DP +
                                           i % (DP / 4) * 4 + s * stride);
  };
  // The first shares' values are under way while their factors are computed.
  constexpr uint32_t kAhead = 8;
  const uint32_t item = groups > 1 ? tid - group * items : tid;
  f32x4 ahead[kAhead];
#pragma unroll
  for (uint32_t j = 0; j < kAhead; ++j)
    if (group < groups && item < items && first + j * groups < used)
      ahead[j] = part(item, first + j * groups);
  // Each share's factor exp(m - largest m), of every row, and the rows' sums.
  static_assert(sizeof(lds) >= kFewMaxSplits * 64 + kFewThreads * 16, "factors and sums fit");
  float* factor = reinterpret_cast<float*>(lds);  // [used][16]
  for (uint32_t r = wave; r < rows; r += kFewWaves) {
    constexpr uint32_t kEach = kFewMaxSplits / 64;
    f32x2 y[kEach];
    float largest = kNegInf;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
      const uint32_t s = lane + j * 64;
      y[j] = f32x2{kNegInf, 0.0f};
      if (s < used) y[j] = ml[(slot0 + s * pg.heads) * a.few_rows_most + r];
    }
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) largest = fmaxf(largest, y[j][0]);
    // Lanes from `used` on hold nothing.
    for (uint32_t step = 1; step < 64 && step < used; step *= 2)
      largest = fmaxf(largest, __shfl_xor(largest, step));
    float sum = 0.0f;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
      // A share without a maximum attended nothing, or only what is no number.
      const float f = y[j][0] == kNegInf
                          ? (y[j][1] == 0.0f ? 0.0f : 1.0f)
                          : share_factor(y[j][0] - largest);
      if (lane + j * 64 < used) factor[(lane + j * 64) * 16 + r] = f;
      sum += y[j][1] * f;
    }
    for (uint32_t step = 1; step < 64 && step < used; step *= 2) sum += __shfl_xor(sum, step);
    if (lane == 0) {
      join_m[0][r] = largest;
      join_l[0][r] = sum;
    }
  }
  __syncthreads();
  f32x4* sums = reinterpret_cast<f32x4*>(factor + used * 16);
  for (uint32_t i0 = 0; i0 < items; i0 += kFewThreads) {
    const uint32_t i = groups > 1 ? tid - group * items : i0 + tid;
    const uint32_t r = i / (DP / 4), d = i % (DP / 4) * 4;
    const bool mine = groups > 1 ? group < groups : i < items;
    f32x4 x{0, 0, 0, 0};
    if (mine) {
      auto add = [&](uint32_t s, f32x4 y) {
        const float f = factor[s * 16 + r];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] += y[j] * f;
      };
      uint32_t s = first;
      if (i0 == 0)
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j, s += groups)
          if (s < used) add(s, ahead[j]);
#pragma unroll 8
      for (; s < used; s += groups) add(s, part(i, s));
    }
    if (groups > 1) {
      if (mine) sums[tid] = x;
      __syncthreads();
      if (group == 0)
        for (uint32_t g = 1; g < groups; ++g) {
          const f32x4 y = sums[g * items + i];
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] += y[j];
        }
    }
    if (mine && group * (groups > 1) == 0)
      few_store<Row>(a, sq, head, r, d, x, join_m[0][r], join_l[0][r]);
  }
}

template <class Row, uint32_t TYPE, uint32_t DP, uint32_t ROWS>
void launch_many(const AttendParams& p, hipStream_t stream) {
  const uint32_t left = p.many_units - p.many_whole;
  hipLaunchKernelGGL((attend_many_kernel<Row, TYPE, DP, ROWS>),
                     dim3((p.many_whole + left * p.many_splits) * p.pages.heads), dim3(2 * ROWS), 0,
                     stream, p);
  if (!left) return;
  const bool turns = p.many_splits > kJoinFew;
  const dim3 grid(left * p.pages.heads * (ROWS / 32) * join_parts(DP, turns)), block(kJoinThreads);
  if (turns)
    hipLaunchKernelGGL((attend_many_join_kernel<Row, DP, ROWS, true>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((attend_many_join_kernel<Row, DP, ROWS, false>), grid, block, 0, stream, p);
}

template <class Row, uint32_t TYPE, uint32_t DP>
hipError_t launch_kernels(const AttendParams& p, hipStream_t stream) {
  if (p.few_splits) {
    const uint32_t units = p.num_seqs * p.pages.heads;
    hipLaunchKernelGGL((attend_few_kernel<Row, TYPE, DP>), dim3(units * p.few_splits),
                       dim3(kFewThreads), 0, stream, p);
  }
  if (p.many_units) {
    if constexpr (DP <= kWideMaxDim) {
      if (p.many_rows == kWideRows)
        launch_many<Row, TYPE, DP, kWideRows>(p, stream);
      else
        launch_many<Row, TYPE, DP, kManyRows>(p, stream);
    } else {
      launch_many<Row, TYPE, DP, kManyRows>(p, stream);
    }
  }
  return hipGetLastError();
}

template <class Row, uint32_t TYPE>
hipError_t launch_dim(const AttendParams& p, hipStream_t stream) {
  switch (padded_dim(p.pages.dim)) {
    case 64: return launch_kernels<Row, TYPE, 64>(p, stream);
    case 96: return launch_kernels<Row, TYPE, 96>(p, stream);
    case 128: return launch_kernels<Row, TYPE, 128>(p, stream);
    case 192: return launch_kernels<Row, TYPE, 192>(p, stream);
    default: return launch_kernels<Row, TYPE, 256>(p, stream);
  }
}

template <class Row>
hipError_t launch_type(const AttendParams& p, hipStream_t stream) {
  if (p.pages.type == PF_KV_E4M3) return launch_dim<Row, PF_KV_E4M3>(p, stream);
  if (p.pages.type == PF_KV_INT8) return launch_dim<Row, PF_KV_INT8>(p, stream);
  return launch_dim<Row, Row::kType>(p, stream);
}

}  // namespace
}  // namespace pf
