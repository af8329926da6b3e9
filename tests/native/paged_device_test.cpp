// paged_device_test.cpp — the paged-cache operators refuse arrays on another device than
// the stream's, on the host (no GPU): this program's own versions of the HIP calls that say
// where memory and streams are, and that launch kernels, come before the runtime's.  Built
// by tests/test_paged_devices.py against the library.
// Exit status 0 and "ok" on success; each failed check is printed.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstring>

#include "pegaflow_hip.h"

namespace {

// Allocation i of kSize bytes lies at kBase * (i + 1), on device where[i].
constexpr uint64_t kBase = 1ull << 40, kSize = 1ull << 30;
enum Array { kPages, kK, kV, kSlots, kQ, kOut, kTable, kLens, kStarts, kLse, kArrays };
const char* const kNames[kArrays] = {"pages", "K rows", "V rows",   "slots",        "q",
                                     "out",   "block table", "seq_lens", "query_starts", "lse"};
int where[kArrays];
int current = 0, launches = 0, launch_device = -1, failures = 0;

uint64_t at(int array) { return kBase * (array + 1) + 4096; }

#define EXPECT(cond) \
  if (!(cond) && ++failures) std::printf("FAILED line %d: %s (%s)\n", __LINE__, #cond, pf_last_error())

}  // namespace

extern "C" {
hipError_t hipGetDevice(int* device) {
  *device = current;
  return hipSuccess;
}
hipError_t hipSetDevice(int device) {
  current = device;
  return hipSuccess;
}
hipError_t hipStreamGetDevice(hipStream_t stream, hipDevice_t* device) {  // stream d + 1 is device d's
  *device = static_cast<int>(reinterpret_cast<uintptr_t>(stream)) - 1;
  return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipPointerGetAttributes(hipPointerAttribute_t* attr, const void* p) {
  const uint64_t i = reinterpret_cast<uint64_t>(p) / kBase;
  if (i == 0 || i > kArrays) return hipErrorInvalidValue;
  std::memset(attr, 0, sizeof(*attr));
  attr->type = hipMemoryTypeDevice;
  attr->device = where[i - 1];
  return hipSuccess;
}
hipError_t hipMemGetAddressRange(hipDeviceptr_t* base, size_t* size, hipDeviceptr_t p) {
  *base = reinterpret_cast<hipDeviceptr_t>(reinterpret_cast<uint64_t>(p) / kBase * kBase);
  *size = kSize;
  return hipSuccess;
}
// What a launch's syntax becomes before and in the kernel's host function.
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3*, dim3*, size_t*, hipStream_t*) { return hipSuccess; }
hipError_t hipLaunchKernel(const void*, dim3, dim3, void**, size_t, hipStream_t) {
  ++launches;
  launch_device = current;
  return hipSuccess;
}
}  // extern "C"

namespace {

pf_kv_rows rows(int array, uint32_t heads) {
  return {at(array), heads * 64, 64, PF_KV_BF16, 0};
}

int call(int op, pf_stream stream) {
  pf_kv_pages p{};
  p.block_size = 16;
  p.num_heads = 2;
  p.head_dim = 64;
  p.type = PF_KV_BF16;
  p.layout.data_ptr = at(kPages);
  p.layout.num_blocks = 10;
  p.layout.bytes_per_block = 4096;
  p.layout.kv_stride_bytes = 40960;
  p.layout.size_bytes = 81920;
  p.layout.segments = 2;
  const pf_kv_rows k = rows(kK, 2), v = rows(kV, 2);
  if (op == 0) return pf_kv_write(&p, &k, &v, at(kSlots), 5, stream);
  if (op == 1) return pf_kv_read(&p, &k, &v, at(kSlots), 5, stream);
  pf_attend_args a{};
  a.q = rows(kQ, 4);
  a.out = rows(kOut, 4);
  a.num_rows = 5;
  a.block_table = at(kTable);
  a.table_stride = a.table_width = 4;
  a.seq_lens = at(kLens);
  a.query_starts = at(kStarts);
  a.lse = at(kLse);
  a.num_q_heads = 4;
  a.num_seqs = 2;
  a.causal = 1;
  a.scale = 0.125f;
  return pf_kv_attend(&p, &a, nullptr, stream);
}

bool takes(int op, int array) {
  return array == kPages || (op < 2 ? array <= kSlots : array >= kQ);
}

}  // namespace

int main() {
  for (int op = 0; op < 3; ++op)
    for (int device = 0; device < 3; ++device)
      for (int null = 0; null < 2; ++null) {
        // Everything on one device: on a stream of it, or on its null stream.
        const pf_stream stream = null ? nullptr : reinterpret_cast<pf_stream>(device + 1ull);
        for (int i = 0; i < kArrays; ++i) where[i] = device;
        current = null ? device : 1;
        const int before = current;
        launches = 0;
        EXPECT(call(op, stream) == PF_OK);
        EXPECT(launches > 0 && launch_device == device && current == before);
        // Each array in turn on another.
        for (int i = 0; i < kArrays; ++i) {
          where[i] = (device + 1) % 3;
          launches = 0;
          if (takes(op, i)) {
            EXPECT(call(op, stream) == PF_ERR_INVALID_ARGUMENT);
            EXPECT(launches == 0 && current == before);
            EXPECT(std::strstr(pf_last_error(), kNames[i]) &&
                   std::strstr(pf_last_error(), "the stream on device"));
          } else {
            EXPECT(call(op, stream) == PF_OK && launches > 0);
          }
          where[i] = device;
        }
      }
  if (failures) return 1;
  std::puts("ok");
  return 0;
}
