// pf_rotary.cpp — entry points of rotary positions: the table of frequencies, argument
// checks, and the launch (pf_rotary.hip).
#include <cmath>

#include "pf_paged_args.h"
#include "pf_rotary.h"

struct pf_rotary {
  int device = 0;
  uint64_t turns = 0;  // device memory, [pairs]
  uint32_t pairs = 0, layout = 0;
  float factor = 1;
};

namespace pf {

namespace {

// f radians a position as turns times 2^64, of which only the fraction of a turn counts.
// Rounded from a long double's 64 bits: frequencies of up to a turn are off by 2^-64 turns.
uint64_t turns_of(double f) {
  const long double t = static_cast<long double>(f) / 6.283185307179586476925286766559005768L;
  const long double part = (t - std::floor(t)) * 0x1p64L;
  return part >= 0x1p64L ? 0 : static_cast<uint64_t>(part);
}

int check_rows_type(const pf_rotary* rotary, uint32_t dim) {
  if (!rotary) return invalid("null rotary positions");
  if (dim == 0 || dim % 16 != 0 || dim > PF_KV_MAX_HEAD_DIM)
    return invalid(strf("head_dim %u is not a multiple of 16 up to %u", dim,
                        (unsigned)PF_KV_MAX_HEAD_DIM));
  if (2 * rotary->pairs > dim)
    return invalid(strf("%u turned values of heads of %u", 2 * rotary->pairs, dim));
  return PF_OK;
}

int launch(RotaryParams& p, const pf_rotary* rotary, uint32_t type, uint64_t positions,
           uint64_t slots, uint64_t n, Ranges& ranges, pf_stream stream) {
  if (int rc = add_array("positions", positions, n * 8, 8, ranges)) return rc;
  if (p.kv_heads)
    if (int rc = add_array("slots", slots, n * 8, 8, ranges)) return rc;
  if (int rc = ranges.check()) return rc;
  p.positions = reinterpret_cast<const int64_t*>(positions);
  p.slots = reinterpret_cast<const int64_t*>(slots);
  p.turns = reinterpret_cast<const uint64_t*>(rotary->turns);
  p.factor = rotary->factor;
  p.rotary = 2 * rotary->pairs;
  p.layout = rotary->layout;
  p.n = static_cast<uint32_t>(n);
  plan_rotary(&p);
  if (rotary_grid(p) > 0x7fffffffull) return invalid("too many rows");
  hipStream_t s = static_cast<hipStream_t>(stream);
  OnDevice on;
  if (int rc = on.enter(s, ranges)) return rc;
  int dev = 0;
  PF_HIP(hipGetDevice(&dev));
  if (rotary->device != dev)
    return invalid(
        strf("the rotary positions are on device %d, the stream on device %d", rotary->device, dev));
  PF_HIP(type == PF_KV_BF16 ? launch_rotary_bf16(p, s) : launch_rotary_fp16(p, s));
  return PF_OK;
}

// Rows that are turned from `x` to `out`.
int view_turned(const pf_kv_rows* x, const pf_kv_rows* out, uint64_t n, uint32_t heads,
                uint32_t dim, Ranges& ranges, RotaryParams* p) {
  if (!is_row_type(x->type) || x->type != out->type)
    return invalid("turned rows are of one type, bf16 or fp16");
  if (int rc = view_rows(*x, "q", n, heads, dim, false, ranges, &p->q, &p->aligned)) return rc;
  return view_rows(*out, "q_out", n, heads, dim, true, ranges, &p->q_out, &p->aligned);
}

int rotate(const pf_rotary* rotary, const pf_kv_rows* x, const pf_kv_rows* out, uint64_t positions,
           uint64_t n, uint32_t heads, uint32_t dim, pf_stream stream) {
  if (int rc = check_rows_type(rotary, dim)) return rc;
  if (!x || !out) return invalid("null rows");
  if (n == 0 || heads == 0) return PF_OK;
  if (n >= kMaxTokens || heads >= kMaxTokens / n) return invalid("too many rows");
  Ranges ranges;
  RotaryParams p{};
  p.aligned = true;
  p.pages.dim = dim;
  p.pages.type = x->type;
  p.q_heads = heads;
  if (int rc = view_turned(x, out, n, heads, dim, ranges, &p)) return rc;
  return launch(p, rotary, x->type, positions, 0, n, ranges, stream);
}

int write_rotated(const pf_kv_pages* pages, const pf_rotary* rotary, const pf_kv_rows* q,
                  const pf_kv_rows* q_out, uint32_t q_heads, const pf_kv_rows* k,
                  const pf_kv_rows* v, uint64_t positions, uint64_t slots, uint64_t n,
                  pf_stream stream) {
  Ranges ranges;
  RotaryParams p{};
  p.aligned = true;
  if (int rc = view_pages(pages, ranges, &p.pages)) return rc;
  if (int rc = check_rows_type(rotary, p.pages.dim)) return rc;
  if (!k || !v || (q_heads && (!q || !q_out))) return invalid("null rows");
  if (k->type != v->type) return invalid("K and V rows differ in type");
  if (is_row_type(p.pages.type) && is_row_type(k->type) && p.pages.type != k->type)
    return invalid("16-bit pages hold the rows' own type");
  if (q_heads && q->type != k->type) return invalid("q, K and V rows are of one type");
  if (n == 0) return PF_OK;
  if (n >= kMaxTokens || q_heads >= kMaxTokens / n) return invalid("too many rows");
  p.q_heads = q_heads;
  p.kv_heads = p.pages.heads;
  if (q_heads)
    if (int rc = view_turned(q, q_out, n, q_heads, p.pages.dim, ranges, &p)) return rc;
  if (int rc = view_rows(*k, "K rows", n, p.kv_heads, p.pages.dim, false, ranges, &p.k, &p.aligned))
    return rc;
  if (int rc = view_rows(*v, "V rows", n, p.kv_heads, p.pages.dim, false, ranges, &p.v, &p.aligned))
    return rc;
  return launch(p, rotary, k->type, positions, slots, n, ranges, stream);
}

}  // namespace

}  // namespace pf

extern "C" {

int pf_rotary_create(int device, const double* frequencies, uint32_t num_pairs, uint32_t layout,
                     float factor, pf_rotary** out) {
  return pf::guarded([&]() -> int {
    if (!out) return pf::invalid("null output");
    *out = nullptr;
    if (!frequencies) return pf::invalid("null frequencies");
    if (num_pairs == 0 || num_pairs > pf::kMaxPairs)
      return pf::invalid(pf::strf("%u pairs of a head (1 to %u)", num_pairs, pf::kMaxPairs));
    if (layout != PF_ROTARY_HALF && layout != PF_ROTARY_INTERLEAVED)
      return pf::invalid(pf::strf("unknown layout %u of the pairs", layout));
    if (!std::isfinite(factor)) return pf::invalid("the factor is not finite");
    uint64_t turns[pf::kMaxPairs];
    for (uint32_t i = 0; i < num_pairs; ++i) {
      if (!std::isfinite(frequencies[i])) return pf::invalid("a frequency is not finite");
      turns[i] = pf::turns_of(frequencies[i]);
    }
    int prev = 0;
    const bool had = hipGetDevice(&prev) == hipSuccess;
    const int rc = pf_init(device);
    void* p = nullptr;
    hipError_t e = rc == PF_OK ? hipMalloc(&p, sizeof(turns)) : hipSuccess;
    if (p) e = hipMemcpy(p, turns, num_pairs * 8, hipMemcpyHostToDevice);
    if (e != hipSuccess && p) (void)hipFree(p);
    if (had && prev != device) (void)hipSetDevice(prev);
    if (rc != PF_OK) return rc;
    if (e != hipSuccess) return pf::hip_fail(e, "pf_rotary_create");
    *out = new pf_rotary{device, reinterpret_cast<uint64_t>(p), num_pairs, layout, factor};
    return PF_OK;
  });
}

int pf_rotary_destroy(pf_rotary* rotary) {
  return pf::guarded([&]() -> int {
    if (!rotary) return PF_OK;
    (void)hipFree(reinterpret_cast<void*>(rotary->turns));
    delete rotary;
    return PF_OK;
  });
}

int pf_rotary_rotate(const pf_rotary* rotary, const pf_kv_rows* x, const pf_kv_rows* out,
                     uint64_t positions, uint64_t num_rows, uint32_t num_heads, uint32_t head_dim,
                     pf_stream stream) {
  return pf::guarded(
      [&] { return pf::rotate(rotary, x, out, positions, num_rows, num_heads, head_dim, stream); });
}

int pf_kv_write_rotated(const pf_kv_pages* pages, const pf_rotary* rotary, const pf_kv_rows* q,
                        const pf_kv_rows* q_out, uint32_t num_q_heads, const pf_kv_rows* k,
                        const pf_kv_rows* v, uint64_t positions, uint64_t slots, uint64_t num_rows,
                        pf_stream stream) {
  return pf::guarded([&] {
    return pf::write_rotated(pages, rotary, q, q_out, num_q_heads, k, v, positions, slots, num_rows,
                             stream);
  });
}

}  // extern "C"
