// pf_pages.cpp — entry points of the operators on all layers of a cache: the layers' handle,
// argument checks, and the launches (pf_pages.hip).
#include <algorithm>
#include <vector>

#include "pf_paged_args.h"
#include "pf_pages.h"

struct pf_kv_layers {
  int device = 0;
  uint64_t views = 0;  // device memory, LayerView of each
  uint32_t count = 0;
  pf::PagedView pages{};
};

namespace pf {

namespace {

bool same_shape(const PagedView& a, const PagedView& b) {
  return a.block_bytes == b.block_bytes && a.num_blocks == b.num_blocks &&
         a.block_size == b.block_size && a.heads == b.heads && a.dim == b.dim &&
         a.token_bytes == b.token_bytes && a.head_bytes == b.head_bytes && a.type == b.type;
}

// Whether `count` segments of `bytes`, each `step` behind the one before it, have bytes in common
// with as many that start `apart` behind them.
bool segments_meet(uint64_t apart, uint64_t step, uint64_t count, uint64_t bytes) {
  const uint64_t whole = apart / step, rest = apart % step;
  return (whole < count && rest < bytes) || (whole + 1 < count && step - rest < bytes);
}

int create_layers(int device, const pf_kv_pages* pages, uint32_t n, pf_kv_layers** out) {
  if (!out) return invalid("null output");
  *out = nullptr;
  if (!pages || n == 0) return invalid("no layers");
  if (n > (1u << 16)) return invalid("too many layers");
  std::vector<LayerView> views(n);
  PagedView shape{};
  for (uint32_t i = 0; i < n; ++i) {
    Ranges ranges;
    PagedView v;
    if (int rc = view_pages(pages + i, ranges, &v)) return rc;
    if (i && !same_shape(shape, v)) return invalid(strf("layer %u has pages of another shape", i));
    if (i == 0) shape = v;
    if (int rc = ranges.check()) return rc;
    if (int rc = ranges.check_device(device)) return rc;
    views[i] = {v.k, v.v};
  }
  // Twice the same memory would be moved twice, by workgroups that do not wait for each other.
  // Layers may lie between each other's blocks.
  std::vector<uint64_t> starts;
  for (const LayerView& v : views) {
    starts.push_back(v.k);
    starts.push_back(v.v);
  }
  std::sort(starts.begin(), starts.end());
  uint64_t bytes = 0;
  if (int rc = segment_bytes(shape.block_size, shape.heads, shape.dim, shape.type, &bytes)) return rc;
  const uint64_t span = (shape.num_blocks - 1ull) * shape.block_bytes + bytes;
  for (size_t i = 0; i < starts.size(); ++i)
    for (size_t j = i + 1; j < starts.size() && starts[j] - starts[i] < span; ++j)
      if (segments_meet(starts[j] - starts[i], shape.block_bytes, shape.num_blocks, bytes))
        return invalid("two layers have some of the same memory");
  int prev = 0;
  const bool had = hipGetDevice(&prev) == hipSuccess;
  const int rc = pf_init(device);
  const uint64_t table = n * sizeof(LayerView);
  void* p = nullptr;
  hipError_t e = rc == PF_OK ? hipMalloc(&p, table) : hipSuccess;
  if (p) e = hipMemcpy(p, views.data(), table, hipMemcpyHostToDevice);
  if (e != hipSuccess && p) (void)hipFree(p);
  if (had && prev != device) (void)hipSetDevice(prev);
  if (rc != PF_OK) return rc;
  if (e != hipSuccess) return hip_fail(e, "pf_kv_layers_create");
  *out = new pf_kv_layers{device, reinterpret_cast<uint64_t>(p), n, shape};
  return PF_OK;
}

// Makes the stream's device current where the layers and the call's arrays lie on it.
int enter(OnDevice& on, const pf_kv_layers* layers, hipStream_t stream, Ranges& ranges) {
  if (int rc = ranges.check()) return rc;
  if (int rc = on.enter(stream, ranges)) return rc;
  int dev = 0;
  PF_HIP(hipGetDevice(&dev));
  if (layers->device != dev)
    return invalid(strf("the layers are on device %d, the stream on device %d", layers->device, dev));
  return PF_OK;
}

int add_table(const char* what, uint64_t addr, uint64_t rows, uint64_t width, uint64_t stride,
              Ranges& ranges) {
  if (stride < width && rows > 1) return invalid(strf("%s: rows overlap", what));
  uint64_t entries = 0;
  if (__builtin_mul_overflow(rows - 1, stride, &entries) || entries > (1ull << 40))
    return invalid(strf("%s: strides overflow", what));
  return add_array(what, addr, (entries + width) * 4, 4, ranges);
}

int launch_copies(const pf_kv_layers* layers, ForkParams& p, Ranges& ranges, pf_stream stream) {
  p.layers = reinterpret_cast<const LayerView*>(layers->views);
  p.pages = layers->pages;
  p.num_layers = layers->count;
  uint64_t bytes = 0;
  if (int rc = segment_bytes(p.pages.block_size, p.pages.heads, p.pages.dim, p.pages.type, &bytes))
    return rc;
  p.segment_chunks = static_cast<uint32_t>(bytes / 16);
  p.parts = (p.segment_chunks + kPagesThreads * kForkChunks - 1) / (kPagesThreads * kForkChunks);
  const uint64_t each = static_cast<uint64_t>(p.num_layers) * 2 * p.parts + 1;
  if (p.num_children > 0x7fffffffull / each) return invalid("too many blocks to copy");
  hipStream_t s = static_cast<hipStream_t>(stream);
  OnDevice on;
  if (int rc = enter(on, layers, s, ranges)) return rc;
  PF_HIP(launch_fork(p, s));
  return PF_OK;
}

int copy_blocks(const pf_kv_layers* layers, uint64_t from, uint64_t to, uint64_t n,
                pf_stream stream) {
  if (!layers) return invalid("null layers");
  if (n == 0) return PF_OK;
  if (n >= kMaxTokens) return invalid("too many blocks to copy");
  Ranges ranges;
  if (int rc = add_array("from_blocks", from, n * 4, 4, ranges)) return rc;
  if (int rc = add_array("to_blocks", to, n * 4, 4, ranges)) return rc;
  ForkParams p{};
  p.blocks = reinterpret_cast<const int32_t*>(from);
  p.new_blocks = reinterpret_cast<const int32_t*>(to);
  p.num_children = static_cast<uint32_t>(n);
  return launch_copies(layers, p, ranges, stream);
}

int fork(const pf_kv_layers* layers, const pf_fork_args* a, pf_stream stream) {
  if (!layers) return invalid("null layers");
  if (!a) return invalid("null arguments");
  if (a->num_children == 0) return PF_OK;
  if (a->num_seqs == 0) return invalid("children without sequences to fork");
  if (a->table_width == 0) return invalid("the block table has no entries");
  if (a->num_seqs >= (1u << 24) || a->num_children >= (1u << 24))
    return invalid("too many sequences");
  Ranges ranges;
  if (int rc = add_table("block table", a->block_table, a->num_seqs, a->table_width,
                         a->table_stride, ranges))
    return rc;
  if (int rc = add_table("out_table", a->out_table, a->num_children, a->table_width,
                         a->out_stride, ranges))
    return rc;
  if (a->block_table == a->out_table) return invalid("out_table is the block table itself");
  if (int rc = add_array("seq_lens", a->seq_lens, a->num_seqs * 4ull, 4, ranges)) return rc;
  if (int rc = add_array("parents", a->parents, a->num_children * 4ull, 4, ranges)) return rc;
  if (int rc = add_array("new_blocks", a->new_blocks, a->num_children * 4ull, 4, ranges)) return rc;
  ForkParams p{};
  p.table = reinterpret_cast<const int32_t*>(a->block_table);
  p.table_stride = a->table_stride;
  p.seq_lens = reinterpret_cast<const int32_t*>(a->seq_lens);
  p.parents = reinterpret_cast<const int32_t*>(a->parents);
  p.new_blocks = reinterpret_cast<const int32_t*>(a->new_blocks);
  p.out_table = reinterpret_cast<int32_t*>(a->out_table);
  p.out_stride = a->out_stride;
  p.width = a->table_width;
  p.num_seqs = a->num_seqs;
  p.num_children = a->num_children;
  return launch_copies(layers, p, ranges, stream);
}

int compact(const pf_kv_layers* layers, const pf_compact_args* a, pf_stream stream) {
  if (!layers) return invalid("null layers");
  if (!a) return invalid("null arguments");
  if (a->num_seqs == 0) return PF_OK;
  if (a->table_width == 0) return invalid("the block table has no entries");
  if (static_cast<uint64_t>(a->table_width) * layers->pages.block_size >= kMaxTokens)
    return invalid("the block table spans 2^31 tokens or more");
  // A chunk's end stays within 31 bits.
  if (a->num_seqs >= (1u << 24) || a->num_kept >= kMaxTokens / 2) return invalid("too many tokens");
  // A sequence's length is written by one workgroup while others still read the arrays.
  auto written = [&](uint64_t at, uint64_t entries) {
    return a->out_lens && at && at < a->out_lens + a->num_seqs * 4ull &&
           a->out_lens < at + entries * 4;
  };
  if (written(a->first, a->num_seqs) || written(a->kept_starts, a->num_seqs + 1ull) ||
      written(a->kept, a->num_kept))
    return invalid("out_lens is, in part, one of the arrays that are read");
  Ranges ranges;
  if (int rc = add_table("block table", a->block_table, a->num_seqs, a->table_width,
                         a->table_stride, ranges))
    return rc;
  if (int rc = add_table("out_table", a->out_table, a->num_seqs, a->table_width, a->out_stride,
                         ranges))
    return rc;
  const bool in_place = a->block_table == a->out_table;
  if (in_place && a->table_stride != a->out_stride && a->num_seqs > 1)
    return invalid("the block table has two strides");
  // Without a kept token there is only the length to write, and nothing is read of `kept`.
  if (a->num_kept)
    if (int rc = add_array("kept", a->kept, a->num_kept * 4, 4, ranges)) return rc;
  if (int rc = add_array("kept_starts", a->kept_starts, (a->num_seqs + 1ull) * 4, 4, ranges))
    return rc;
  if (a->first)
    if (int rc = add_array("first", a->first, a->num_seqs * 4ull, 4, ranges)) return rc;
  if (a->out_lens)
    if (int rc = add_array("out_lens", a->out_lens, a->num_seqs * 4ull, 4, ranges)) return rc;
  CompactParams p{};
  p.layers = reinterpret_cast<const LayerView*>(layers->views);
  p.pages = layers->pages;
  p.num_layers = layers->count;
  p.table = reinterpret_cast<const int32_t*>(a->block_table);
  p.out_table = reinterpret_cast<const int32_t*>(a->out_table);
  p.table_stride = a->table_stride;
  p.out_stride = a->out_stride;
  p.width = a->table_width;
  p.num_seqs = a->num_seqs;
  p.kept = reinterpret_cast<const int32_t*>(a->kept);
  p.kept_starts = reinterpret_cast<const int32_t*>(a->kept_starts);
  p.first = reinterpret_cast<const int32_t*>(a->first);
  p.out_lens = reinterpret_cast<int32_t*>(a->out_lens);
  p.total = static_cast<uint32_t>(a->num_kept);
  plan_compact(&p, a->max_kept, in_place);
  if (compact_grid(p) > 0x7fffffffull) return invalid("too many sequences and layers");
  hipStream_t s = static_cast<hipStream_t>(stream);
  OnDevice on;
  if (int rc = enter(on, layers, s, ranges)) return rc;
  PF_HIP(launch_compact(p, s));
  return PF_OK;
}

}  // namespace

}  // namespace pf

extern "C" {

int pf_kv_layers_create(int device, const pf_kv_pages* layers, uint32_t num_layers,
                        pf_kv_layers** out) {
  return pf::guarded([&] { return pf::create_layers(device, layers, num_layers, out); });
}

int pf_kv_layers_destroy(pf_kv_layers* layers) {
  return pf::guarded([&]() -> int {
    if (!layers) return PF_OK;
    (void)hipFree(reinterpret_cast<void*>(layers->views));
    delete layers;
    return PF_OK;
  });
}

int pf_kv_copy_blocks(const pf_kv_layers* layers, uint64_t from_blocks, uint64_t to_blocks,
                      uint64_t num_blocks, pf_stream stream) {
  return pf::guarded(
      [&] { return pf::copy_blocks(layers, from_blocks, to_blocks, num_blocks, stream); });
}

int pf_kv_fork(const pf_kv_layers* layers, const pf_fork_args* args, pf_stream stream) {
  return pf::guarded([&] { return pf::fork(layers, args, stream); });
}

int pf_kv_compact(const pf_kv_layers* layers, const pf_compact_args* args, pf_stream stream) {
  return pf::guarded([&] { return pf::compact(layers, args, stream); });
}

}  // extern "C"
