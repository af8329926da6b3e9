// paged_overlap_test.cpp — memory that a call on all layers of a cache may not be given twice, on
// the host (no GPU): this program's own versions of the HIP calls that say where memory and
// streams are, allocate, and launch kernels, come before the runtime's.  Built by
// tests/test_paged_overlaps.py against the library.
// Exit status 0 and "ok" on success; each failed check is printed.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <vector>

#include "pegaflow_hip.h"

namespace {

// One allocation on device 0.
constexpr uint64_t kBase = 1ull << 40, kSize = 1ull << 30;
int launches = 0, failures = 0;

#define EXPECT(cond) \
  if (!(cond) && ++failures <= 20) std::printf("FAILED line %d: %s (%s)\n", __LINE__, #cond, pf_last_error())

}  // namespace

extern "C" {
hipError_t hipGetDevice(int* device) {
  *device = 0;
  return hipSuccess;
}
hipError_t hipGetDeviceCount(int* n) {
  *n = 1;
  return hipSuccess;
}
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipDeviceGetAttribute(int* value, hipDeviceAttribute_t, int) {
  *value = 100000;
  return hipSuccess;
}
hipError_t hipGetSymbolAddress(void** p, const void*) {
  static char memory[1 << 20];
  *p = memory;
  return hipSuccess;
}
hipError_t hipMalloc(void** p, size_t n) {
  *p = std::malloc(n);
  return hipSuccess;
}
hipError_t hipFree(void* p) {
  std::free(p);
  return hipSuccess;
}
hipError_t hipMemcpy(void* dst, const void* src, size_t n, hipMemcpyKind) {
  std::memcpy(dst, src, n);
  return hipSuccess;
}
hipError_t hipMemset(void* p, int v, size_t n) {
  std::memset(p, v, n);
  return hipSuccess;
}
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipStreamGetDevice(hipStream_t, hipDevice_t* device) {
  *device = 0;
  return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipPointerGetAttributes(hipPointerAttribute_t* attr, const void* p) {
  if (reinterpret_cast<uint64_t>(p) / kBase != 1) return hipErrorInvalidValue;
  std::memset(attr, 0, sizeof(*attr));
  attr->type = hipMemoryTypeDevice;
  return hipSuccess;
}
hipError_t hipMemGetAddressRange(hipDeviceptr_t* base, size_t* size, hipDeviceptr_t) {
  *base = reinterpret_cast<hipDeviceptr_t>(kBase);
  *size = kSize;
  return hipSuccess;
}
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3*, dim3*, size_t*, hipStream_t*) { return hipSuccess; }
hipError_t hipLaunchKernel(const void*, dim3, dim3, void**, size_t, hipStream_t) {
  ++launches;
  return hipSuccess;
}
}  // extern "C"

namespace {

std::mt19937_64 rng(1);
uint64_t pick(uint64_t lo, uint64_t hi) { return lo + rng() % (hi - lo + 1); }

// Pages of one token, one head and 16 values of a 16-bit type: segments of 32 bytes.
pf_kv_pages pages(uint64_t at, uint64_t blocks, uint64_t step, uint64_t v_offset) {
  pf_kv_pages p{};
  p.block_size = 1;
  p.num_heads = 1;
  p.head_dim = 16;
  p.type = PF_KV_BF16;
  p.layout.data_ptr = kBase + at;
  p.layout.num_blocks = blocks;
  p.layout.bytes_per_block = step;
  p.layout.segments = v_offset ? 2 : 1;
  p.layout.kv_stride_bytes = v_offset;
  p.layout.size_bytes = blocks * step + v_offset;
  return p;
}

// Layers anywhere in a few hundred bytes: refused where a byte of a block is in two segments, and
// only there.
void layers() {
  int apart = 0, met = 0;
  for (int i = 0; i < 100000; ++i) {
    const uint64_t blocks = pick(1, 5), step = 32 * pick(2, 8);
    const uint64_t v_offset = pick(0, 2) ? blocks * step + 16 * pick(0, 4) : 0;
    const uint64_t segment = v_offset ? step : step / 2, n = pick(1, 4);
    std::vector<pf_kv_pages> list;
    std::vector<int> owners(1 << 14, 0);
    bool meet = false;
    for (uint64_t layer = 0; layer < n; ++layer) {
      const uint64_t at = 16 * pick(0, pick(0, 3) ? 16 : 300);
      list.push_back(pages(at, blocks, step, v_offset));
      for (uint64_t kv = 0; kv < 2; ++kv)
        for (uint64_t b = 0; b < blocks; ++b)
          for (uint64_t x = 0; x < 32; ++x)
            meet |= owners[at + kv * (v_offset ? v_offset : segment) + b * step + x]++ > 0;
    }
    pf_kv_layers* l = nullptr;
    const int rc = pf_kv_layers_create(0, list.data(), static_cast<uint32_t>(n), &l);
    EXPECT(rc == (meet ? PF_ERR_INVALID_ARGUMENT : PF_OK));
    EXPECT(!meet || std::strstr(pf_last_error(), "same memory"));
    EXPECT((l != nullptr) == (rc == PF_OK));
    pf_kv_layers_destroy(l);
    ++(meet ? met : apart);
  }
  EXPECT(apart > 10000 && met > 10000);
  // As caches lay them out: each by itself, and a block's Ks, then its Vs, of all layers.
  for (const bool mixed : {false, true}) {
    std::vector<pf_kv_pages> list;
    for (uint64_t i = 0; i < 64; ++i)
      list.push_back(mixed ? pages(i * 32, 1000, 64 * 64, 0) : pages(i * 64000, 1000, 32, 32000));
    pf_kv_layers* l = nullptr;
    EXPECT(pf_kv_layers_create(0, list.data(), 64, &l) == PF_OK);
    pf_kv_layers_destroy(l);
    list[7].layout.data_ptr -= 16;
    EXPECT(pf_kv_layers_create(0, list.data(), 64, &l) == PF_ERR_INVALID_ARGUMENT);
  }
}

// Lengths that are written may be none of the entries that are read.
void lengths() {
  const pf_kv_pages one = pages(1 << 20, 10, 64, 0);
  pf_kv_layers* l = nullptr;
  EXPECT(pf_kv_layers_create(0, &one, 1, &l) == PF_OK);
  const uint32_t seqs = 5, width = 4, kept = 9;
  const uint64_t out = kBase + 4096, far = kBase + 65536;
  pf_compact_args args{};
  args.block_table = args.out_table = far;
  args.table_stride = args.out_stride = args.table_width = width;
  args.num_seqs = seqs;
  args.num_kept = kept;
  args.out_lens = out;
  const struct {
    uint64_t pf_compact_args::*at;
    int entries;
  } arrays[] = {{&pf_compact_args::first, seqs},
                {&pf_compact_args::kept_starts, seqs + 1},
                {&pf_compact_args::kept, kept}};
  for (const auto& array : arrays)
    for (int shift = -12; shift <= 12; ++shift) {
      pf_compact_args a = args;
      a.kept = far + 4096;
      a.kept_starts = far + 8192;
      a.first = far + 12288;
      a.*array.at = out + 4 * shift;
      const bool meet = shift < static_cast<int>(seqs) && shift + array.entries > 0;
      launches = 0;
      EXPECT(pf_kv_compact(l, &a, nullptr) == (meet ? PF_ERR_INVALID_ARGUMENT : PF_OK));
      EXPECT(launches == (meet ? 0 : 1) && (!meet || std::strstr(pf_last_error(), "out_lens")));
    }
  pf_compact_args a = args;  // without firsts, and without kept tokens
  a.kept_starts = far + 8192;
  a.num_kept = 0;
  a.kept = out;
  EXPECT(pf_kv_compact(l, &a, nullptr) == PF_OK);
  pf_kv_layers_destroy(l);
}

}  // namespace

int main() {
  layers();
  lengths();
  if (failures) return 1;
  std::puts("ok");
  return 0;
}
