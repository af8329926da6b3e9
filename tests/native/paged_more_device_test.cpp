// paged_more_device_test.cpp — the operators on rotary positions, all layers of a cache and
// shared tokens refuse arrays on another device than the stream's, and arguments that make no
// sense, on the host (no GPU): this program's own versions of the HIP calls that say where memory
// and streams are, allocate, and launch kernels, come before the runtime's.  Built by
// tests/test_paged_devices_more.py against the library.
// Exit status 0 and "ok" on success; each failed check is printed.
#include <hip/hip_runtime_api.h>

#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <vector>

#include "pegaflow_hip.h"

namespace {

// Allocation i of kSize bytes lies at kBase * (i + 1), on device where[i].
constexpr uint64_t kBase = 1ull << 40, kSize = 1ull << 30;
enum Array {
  kPages, kK, kV, kSlots, kQ, kOut, kTable, kLens, kStarts, kLse, kPositions, kGroups, kShared,
  kParents, kNew, kOutTable, kKept, kFirst, kOutLens, kArrays
};
const char* const kNames[kArrays] = {
    "pages", "K rows", "V rows", "slots", "q", "q_out", "block table", "seq_lens", "query_starts",
    "lse", "positions", "group_starts", "shared_lens", "parents", "new_blocks", "out_table", "kept",
    "first", "out_lens"};
int where[kArrays];
int current = 0, launches = 0, launch_device = -1, failures = 0, held = 0;

uint64_t at(int array) { return kBase * (array + 1) + 4096; }

#define EXPECT(cond) \
  if (!(cond) && ++failures) std::printf("FAILED line %d: %s (%s)\n", __LINE__, #cond, pf_last_error())

}  // namespace

extern "C" {
hipError_t hipGetDevice(int* device) {
  *device = current;
  return hipSuccess;
}
hipError_t hipGetDeviceCount(int* n) {
  *n = 3;
  return hipSuccess;
}
hipError_t hipSetDevice(int device) {
  current = device;
  return hipSuccess;
}
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
  ++held;
  *p = std::malloc(n);
  return hipSuccess;
}
hipError_t hipFree(void* p) {
  --held;
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

pf_kv_pages pages() {
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
  return p;
}

pf_fork_args forks() {
  return {at(kTable), 4, at(kLens), at(kParents), at(kNew), at(kOutTable), 4, 2, 4, 3, 0};
}

pf_compact_args moves() {
  return {at(kTable), 4, at(kOutTable), 4, at(kKept), 9, at(kStarts), at(kFirst), at(kOutLens),
          2, 4, 0, 0};
}

pf_attend_args batch() {
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
  a.num_seqs = 3;
  a.causal = 1;
  a.scale = 0.125f;
  a.max_query_len = 2;
  return a;
}

// The handles of a device, and one call of each operator with them.
struct Handles {
  pf_rotary* rotary = nullptr;
  pf_kv_layers* layers = nullptr;
  pf_attend_workspace* workspace = nullptr;
};

Handles handles(int device) {
  Handles h;
  const double f[32] = {1.0, 0.5};
  pf_kv_pages p[2] = {pages(), pages()};
  p[1].layout.data_ptr += 1 << 20;
  EXPECT(pf_rotary_create(device, f, 32, PF_ROTARY_HALF, 1.0f, &h.rotary) == PF_OK);
  EXPECT(pf_kv_layers_create(device, p, 2, &h.layers) == PF_OK);
  EXPECT(pf_attend_workspace_create(device, 1 << 20, &h.workspace) == PF_OK);
  return h;
}

int call(int op, const Handles& h, pf_stream stream) {
  const pf_kv_pages p = pages();
  const pf_kv_rows q = rows(kQ, 4), out = rows(kOut, 4), k = rows(kK, 2), v = rows(kV, 2);
  switch (op) {
    case 0: return pf_rotary_rotate(h.rotary, &q, &out, at(kPositions), 5, 4, 64, stream);
    case 1:
      return pf_kv_write_rotated(&p, h.rotary, &q, &out, 4, &k, &v, at(kPositions), at(kSlots), 5,
                                 stream);
    case 2: return pf_kv_copy_blocks(h.layers, at(kParents), at(kNew), 3, stream);
    case 3: {
      const pf_fork_args a = forks();
      return pf_kv_fork(h.layers, &a, stream);
    }
    case 4: {
      const pf_compact_args a = moves();
      return pf_kv_compact(h.layers, &a, stream);
    }
    default: {
      const pf_attend_args a = batch();
      // As many shared tokens as make it worth while, or none.
      const pf_shared_args s{at(kGroups), at(kShared), 1, op == 5 ? ~0u : 1u, 8, 0};
      return pf_kv_attend_shared(&p, &a, &s, h.workspace, stream);
    }
  }
}

std::vector<int> takes(int op) {
  switch (op) {
    case 0: return {kQ, kOut, kPositions};
    case 1: return {kPages, kK, kV, kSlots, kQ, kOut, kPositions};
    case 2: return {kParents, kNew};
    case 3: return {kTable, kLens, kParents, kNew, kOutTable};
    case 4: return {kTable, kOutTable, kKept, kStarts, kFirst, kOutLens};
    default: return {kPages, kQ, kOut, kTable, kLens, kStarts, kLse, kGroups, kShared};
  }
}

void devices() {
  for (int op = 0; op < 7; ++op)
    for (int device = 0; device < 3; ++device) {
      for (int i = 0; i < kArrays; ++i) where[i] = device;
      const Handles mine = handles(device);
      for (int i = 0; i < kArrays; ++i) where[i] = (device + 1) % 3;
      const Handles other = handles((device + 1) % 3);
      for (int i = 0; i < kArrays; ++i) where[i] = device;
      for (int null = 0; null < 2; ++null) {
        // Everything on one device: on a stream of it, or on its null stream.
        const pf_stream stream = null ? nullptr : reinterpret_cast<pf_stream>(device + 1ull);
        current = null ? device : 1;
        const int before = current;
        launches = 0;
        EXPECT(call(op, mine, stream) == PF_OK);
        EXPECT(launches == (op == 5 ? 2 : launches) && launches > 0 && launch_device == device);
        EXPECT(current == before);
        // The handles of another device, and each array in turn on it.
        launches = 0;
        EXPECT(call(op, other, stream) == PF_ERR_INVALID_ARGUMENT);
        EXPECT(launches == 0 && current == before && std::strstr(pf_last_error(), "the stream on device"));
        for (int i : takes(op)) {
          where[i] = (device + 1) % 3;
          EXPECT(call(op, mine, stream) == PF_ERR_INVALID_ARGUMENT);
          EXPECT(launches == 0 && current == before);
          const char* name = op >= 5 && i == kOut ? "out" : op == 2 && i == kParents ? "from_blocks"
                             : op == 2 && i == kNew ? "to_blocks"
                             : op == 4 && i == kStarts ? "kept_starts" : kNames[i];
          EXPECT(std::strstr(pf_last_error(), name) &&
                 std::strstr(pf_last_error(), "the stream on device"));
          where[i] = device;
        }
      }
      for (const Handles& h : {mine, other}) {
        EXPECT(pf_rotary_destroy(h.rotary) == PF_OK);
        EXPECT(pf_kv_layers_destroy(h.layers) == PF_OK);
        EXPECT(pf_attend_workspace_destroy(h.workspace) == PF_OK);
      }
    }
  EXPECT(pf_rotary_destroy(nullptr) == PF_OK && pf_kv_layers_destroy(nullptr) == PF_OK);
}

void refused(int line, const char* text, const std::function<int()>& f) {
  launches = 0;
  if (f() == PF_ERR_INVALID_ARGUMENT && launches == 0 && std::strstr(pf_last_error(), text)) return;
  ++failures;
  std::printf("FAILED line %d: not refused for \"%s\" (%s)\n", line, text, pf_last_error());
}
#define REFUSED(text, ...) refused(__LINE__, text, [&]() -> int { __VA_ARGS__; })

void arguments() {
  for (int i = 0; i < kArrays; ++i) where[i] = 0;
  current = 0;
  const int before = held;
  double f[200] = {1.0};
  pf_rotary* r = nullptr;
  REFUSED("pairs", return pf_rotary_create(0, f, 0, PF_ROTARY_HALF, 1, &r));
  REFUSED("pairs", return pf_rotary_create(0, f, 129, PF_ROTARY_HALF, 1, &r));
  REFUSED("layout", return pf_rotary_create(0, f, 4, 3, 1, &r));
  REFUSED("factor", return pf_rotary_create(0, f, 4, PF_ROTARY_HALF, INFINITY, &r));
  REFUSED("null freq", return pf_rotary_create(0, nullptr, 4, PF_ROTARY_HALF, 1, &r));
  REFUSED("null output", return pf_rotary_create(0, f, 4, PF_ROTARY_HALF, 1, nullptr));
  f[2] = NAN;
  REFUSED("not finite", return pf_rotary_create(0, f, 4, PF_ROTARY_HALF, 1, &r));
  EXPECT(!r && held == before);
  f[2] = 0;
  pf_kv_layers* l = nullptr;
  pf_kv_pages p[2] = {pages(), pages()};
  REFUSED("no layers", return pf_kv_layers_create(0, p, 0, &l));
  REFUSED("no layers", return pf_kv_layers_create(0, nullptr, 2, &l));
  REFUSED("same memory", return pf_kv_layers_create(0, p, 2, &l));
  p[1].layout.data_ptr += 40960;  // its K the other's V
  REFUSED("same memory", return pf_kv_layers_create(0, p, 2, &l));
  p[1].block_size = 8;
  REFUSED("another shape", return pf_kv_layers_create(0, p, 2, &l));
  p[1] = pages();
  p[1].layout.size_bytes -= 1;
  REFUSED("exceed", return pf_kv_layers_create(0, p, 2, &l));
  p[1] = pages();
  where[kPages] = 1;
  REFUSED("on device", return pf_kv_layers_create(0, p, 2, &l));
  where[kPages] = 0;
  EXPECT(!l && held == before);

  const Handles h = handles(0);
  const pf_kv_rows q = rows(kQ, 4), k = rows(kK, 2);
  REFUSED("head_dim", return pf_rotary_rotate(h.rotary, &q, &q, at(kPositions), 5, 4, 40, nullptr));
  REFUSED("turned values", return pf_rotary_rotate(h.rotary, &q, &q, at(kPositions), 5, 4, 48, nullptr));
  REFUSED("null rows", return pf_rotary_rotate(h.rotary, &q, nullptr, at(kPositions), 5, 4, 64, nullptr));
  REFUSED("too many", return pf_rotary_rotate(h.rotary, &q, &q, at(kPositions), 1ull << 31, 1, 64, nullptr));
  REFUSED("positions", return pf_rotary_rotate(h.rotary, &q, &q, at(kPositions) + 4, 5, 4, 64, nullptr));
  REFUSED("not inside", return pf_rotary_rotate(h.rotary, &q, &q, at(kPositions) + kSize - 4104, 5, 4, 64, nullptr));
  EXPECT(pf_rotary_rotate(h.rotary, &q, &q, 0, 0, 4, 64, nullptr) == PF_OK);
  const pf_kv_pages page = pages();
  REFUSED("null rows", return pf_kv_write_rotated(&page, h.rotary, nullptr, nullptr, 4, &k, &k,
                                                  at(kPositions), at(kSlots), 5, nullptr));
  EXPECT(pf_kv_write_rotated(&page, h.rotary, nullptr, nullptr, 0, &k, &k, at(kPositions),
                             at(kSlots), 5, nullptr) == PF_OK);

  REFUSED("null layers", return pf_kv_copy_blocks(nullptr, at(kParents), at(kNew), 3, nullptr));
  REFUSED("too many", return pf_kv_copy_blocks(h.layers, at(kParents), at(kNew), 1ull << 31, nullptr));
  EXPECT(pf_kv_copy_blocks(h.layers, 0, 0, 0, nullptr) == PF_OK);
  pf_fork_args a = forks();
  a.out_stride = 3;
  REFUSED("overlap", return pf_kv_fork(h.layers, &a, nullptr));
  a = forks();
  a.out_table = a.block_table;
  REFUSED("itself", return pf_kv_fork(h.layers, &a, nullptr));
  a = forks();
  a.table_width = 0;
  REFUSED("no entries", return pf_kv_fork(h.layers, &a, nullptr));
  a = forks();
  a.num_seqs = 0;
  REFUSED("without sequences", return pf_kv_fork(h.layers, &a, nullptr));
  a.num_children = 0;
  EXPECT(pf_kv_fork(h.layers, &a, nullptr) == PF_OK);
  pf_compact_args m = moves();
  m.out_lens = m.first;
  REFUSED("out_lens", return pf_kv_compact(h.layers, &m, nullptr));
  m = moves();
  m.out_table = m.block_table;
  m.out_stride = 5;
  REFUSED("two strides", return pf_kv_compact(h.layers, &m, nullptr));
  m = moves();
  m.table_width = 1u << 28;
  m.table_stride = m.out_stride = 1u << 28;
  REFUSED("2^31", return pf_kv_compact(h.layers, &m, nullptr));
  m = moves();
  m.num_kept = 1ull << 30;
  REFUSED("too many", return pf_kv_compact(h.layers, &m, nullptr));
  m = moves();
  m.num_kept = 0;
  m.kept = 0;
  EXPECT(pf_kv_compact(h.layers, &m, nullptr) == PF_OK);
  m.num_seqs = 0;
  EXPECT(pf_kv_compact(h.layers, &m, nullptr) == PF_OK);

  const pf_attend_args b = batch();
  REFUSED("null groups", return pf_kv_attend_shared(&page, &b, nullptr, h.workspace, nullptr));
  pf_shared_args s{at(kGroups), at(kShared), 1u << 24, 0, 0, 0};
  REFUSED("groups", return pf_kv_attend_shared(&page, &b, &s, h.workspace, nullptr));
  s.num_groups = 1;
  s.group_starts += 2;
  REFUSED("group_starts", return pf_kv_attend_shared(&page, &b, &s, h.workspace, nullptr));
  s = {0, 0, 0, 0, 0, 0};
  EXPECT(pf_kv_attend_shared(&page, &b, &s, nullptr, nullptr) == PF_OK);
  pf_rotary_destroy(h.rotary);
  pf_kv_layers_destroy(h.layers);
  pf_attend_workspace_destroy(h.workspace);
  EXPECT(held == before);
}

}  // namespace

int main() {
  devices();
  arguments();
  if (failures) return 1;
  std::puts("ok");
  return 0;
}
