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

// The smallest x of a wave, in a scalar: within 16 lanes by cross-lane operands, which cost no trip
// through LDS.
__device__ __forceinline__ int32_t wave_min(int32_t x) {
  constexpr int kSwap1 = 0xb1, kSwap2 = 0x4e, kMirror8 = 0x141, kMirror16 = 0x140;
  x = min(x, __builtin_amdgcn_mov_dpp(x, kSwap1, 0xf, 0xf, true));
  x = min(x, __builtin_amdgcn_mov_dpp(x, kSwap2, 0xf, 0xf, true));
  x = min(x, __builtin_amdgcn_mov_dpp(x, kMirror8, 0xf, 0xf, true));
  x = min(x, __builtin_amdgcn_mov_dpp(x, kMirror16, 0xf, 0xf, true));
  const int32_t a = __builtin_amdgcn_readlane(x, 0), b = __builtin_amdgcn_readlane(x, 16);
  const int32_t c = __builtin_amdgcn_readlane(x, 32), d = __builtin_amdgcn_readlane(x, 48);
  return min(min(a, b), min(c, d));
}

// Groups of sequences that share their first tokens.  Starts are bounded as in seq_of.
__device__ __forceinline__ int32_t group_start(const AttendParams& a, uint32_t g) {
  return min(max(a.group_starts[g], 0), static_cast<int32_t>(a.num_seqs));
}
__device__ __forceinline__ int32_t row_start(const AttendParams& a, uint32_t b) {
  return min(max(a.query_starts[b], 0), static_cast<int32_t>(a.num_rows));
}
// Tokens that all rows of a sequence attend, if it shares them: none of its new ones.
__device__ __forceinline__ int32_t cached_of(const AttendParams& a, const Seq& s) {
  return max(a.causal ? s.len - s.rows : s.len, 0);
}
// How many tokens sequence `seq` shares: its group's, of those that it has cached.  The whole
// wave calls.
__device__ __forceinline__ int32_t shared_of(const AttendParams& a, int32_t seq, const Seq& s) {
  const uint32_t lane = threadIdx.x & 63u;
  for (uint32_t g0 = 0; g0 < a.num_groups; g0 += 64) {
    const uint32_t g = g0 + lane;
    int32_t shared = 0;
    bool mine = false;
    if (g < a.num_groups) {
      shared = a.shared_lens[g];
      mine = group_start(a, g) <= seq && seq < group_start(a, g + 1);
    }
    const uint64_t in = __ballot(mine);
    if (in) {
      shared = __builtin_amdgcn_readlane(shared, __builtin_ctzll(in));
      return min(max(shared, 0), cached_of(a, s));
    }
  }
  return 0;
}

// Tile `index` of the rows of group `g`: those of its sequences one after another.  A row
// attends as many of the shared tokens, `my_end`, as its sequence has cached, all rows at least
// `all_end`; the tile passes over those that any sequence has, in that one's blocks.
template <uint32_t ROWS>
__device__ __forceinline__ bool group_tile(const AttendParams& a, uint32_t g, uint32_t index,
                                           uint32_t wave, ManyTile* t, int32_t* all_end,
                                           int32_t* my_end) {
  const uint32_t lane = threadIdx.x & 63u;
  const int32_t first = group_start(a, g), last = max(group_start(a, g + 1), first);
  const int32_t first_row = row_start(a, first);
  const int32_t room = static_cast<int32_t>(a.table_width * a.pages.block_size);
  int32_t shared = min(max(a.shared_lens[g], 0), room);
  t->rows = static_cast<uint32_t>(max(row_start(a, last) - first_row, 0)) * a.group;
  t->s = {first_row, 0, 0};
  t->row = index * ROWS + wave * 32 + (lane & 31u);
  t->valid = t->row < t->rows;
  constexpr int32_t kNone = 0x7fffffff;
  constexpr uint32_t kChunks = 4;  // of 64 sequences, whose loads are under way together
  int32_t least = kNone, most = -1;
  for (int32_t b0 = first; b0 < last; b0 += 64 * kChunks) {
    int32_t cached[kChunks];
#pragma unroll
    for (uint32_t c = 0; c < kChunks; ++c) {
      const int32_t b = b0 + static_cast<int32_t>(c * 64 + lane);
      cached[c] = -1;
      if (b < last) {
        const Seq s = seq_of(a, b);
        if (s.rows) cached[c] = cached_of(a, s);
      }
    }
#pragma unroll
    for (uint32_t c = 0; c < kChunks; ++c) {
      least = min(least, wave_min(cached[c] < 0 ? kNone : cached[c]));
      const int32_t hi = -wave_min(-cached[c]);
      if (hi > most) {
        most = hi;
        t->seq = b0 + c * 64 + __builtin_ctzll(__ballot(cached[c] == hi));
      }
    }
  }
  shared = min(shared, most);
  if (shared <= 0) return false;
  int32_t mine = shared;
  if (least < shared) {  // some sequence has cached less: each row's own
    const int32_t token = first_row + static_cast<int32_t>(t->row / a.group);
    for (int32_t b0 = first; b0 < last; b0 += 64) {
      const int32_t b = b0 + static_cast<int32_t>(lane);
      int32_t start = kNone, end = 0, cached = 0;
      if (b < last) {
        const Seq s = seq_of(a, b);
        start = s.first;
        end = s.first + s.rows;
        cached = cached_of(a, s);
      }
      // The last sequence that starts at this lane's token or before: starts ascend.
      int at = 0;
#pragma unroll
      for (int step = 32; step; step /= 2) {
        const int32_t then = __shfl(start, at + step);
        at += then <= token ? step : 0;
      }
      // All lanes read before any decides: a lane reads nothing of one that does not take part.
      const int32_t from = __shfl(start, at), to = __shfl(end, at), has = __shfl(cached, at);
      mine = from <= token && token < to ? min(has, shared) : mine;
    }
  }
  t->begin = 0;
  t->end = shared;
  *all_end = min(shared, least);
  *my_end = t->valid ? mine : 0;
  return true;
}

// Tile `index` of all groups' rows, false if there is none or its group shares nothing.
template <uint32_t ROWS>
__device__ __forceinline__ bool shared_tile(const AttendParams& a, uint32_t index, uint32_t head,
                                            uint32_t wave, ManyTile* t, int32_t* all_end,
                                            int32_t* my_end) {
  const uint32_t lane = threadIdx.x & 63u;
  t->head = head;
  t->pos0 = 0;
  for (uint32_t g0 = 0; g0 < a.num_groups; g0 += 64) {
    uint32_t tiles = 0;
    const uint32_t count = min(a.num_groups - g0, 64u);
    if (lane < count) {
      const int32_t first = group_start(a, g0 + lane);
      const int32_t last = max(group_start(a, g0 + lane + 1), first);
      const uint32_t rows = static_cast<uint32_t>(max(row_start(a, last) - row_start(a, first), 0));
      tiles = (rows * a.group + ROWS - 1) / ROWS;
    }
    for (uint32_t j = 0; j < count; ++j) {
      const uint32_t n = __builtin_amdgcn_readlane(tiles, j);
      if (index < n) return group_tile<ROWS>(a, g0 + j, index, wave, t, all_end, my_end);
      index -= n;
    }
  }
  return false;
}

// A share of one row and query head, as an index to their outputs, and maxima and sums.
__device__ __forceinline__ uint64_t share_at(const AttendParams& a, uint32_t share, uint32_t row,
                                             uint32_t q_head) {
  return (static_cast<uint64_t>(share) * a.num_rows + row) * a.q_heads + q_head;
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
  __shared__ ManyLds<DP> lds;
  constexpr bool SHARED = false;
  const uint32_t index = blockIdx.x;
#include "pf_attend_many.inc"
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
constexpr uint32_t kFewThreads = kFewWaves * 64;
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

template <uint32_t DP>
struct FewLds {
  struct Wave {
    __attribute__((aligned(16))) uint8_t v[kFewTokens * few_v_pitch(DP)];
    // Of 32 tokens to load next: where they lie; of the tile at hand: its scales.
    uint64_t at[kFewTokens];
    __attribute__((aligned(16))) float k_scale[kFewTokens], v_scale[kFewTokens];
  } wave[kFewWaves];
  float join_m[kFewWaves][16], join_l[kFewWaves][16];
  bool finished;
};

template <class Row, uint32_t TYPE, uint32_t DP>
__global__ void __launch_bounds__(kFewThreads, DP <= 128 ? 2 : 1)
attend_few_kernel(AttendParams a) {
  __shared__ FewLds<DP> mem;
  constexpr bool SHARED = false;
  const uint32_t index = blockIdx.x;
#include "pf_attend_few.inc"
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
