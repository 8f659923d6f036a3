// Copies inside the cache: the first rows of pages to other pages, or whole state slots to other slots, in every layer of several
// tensors at once.  A forked request takes its parent's last, partly filled page and its recurrent states this way, and compaction
// moves whole pages.
//
// A tensor is [entries][blocks][parts][rows][row bytes]: a slab of the cache has a part per KV head and a row per token, a state
// tensor one part of one row.  pairs holds (from, to, rows) or (from, to) per copy: tensor[e][to][h][0 : rows] =
// tensor[e][from][h][0 : rows] for every entry e and part h.  A pair that names a block outside the tensor is left out.
//
// What bounds it: memory, each byte read and written once, and for a few pages the launch.  So one launch takes up to kCopyTensors
// tensors, a thread's loads are all under way before the first store, and a block has 32 KB to move (whole pages of 16 tokens, 8
// heads of 128 in bfloat16), which fills the GPU from about 300 such pages on.  Measured: 1,500 pages in four layers, 786 MB read and written,
// 119 us (6.6 TB/s, what a plain copy reaches); partly filled pages of 63 forks in twelve layers, 25 MB, 8.5 us; seven slots of six
// layers' matrix states, 51 MB, 12.8 us; four pages of a small model 8.5 us, a launch on cold caches.
#include "common.cuh"

namespace ftk {

constexpr int kCopyTensors = 16, kCopyThreads = 256, kCopyLoads = 8;

struct CopyTensor {
  unsigned char* base;
  long long entry_vecs, block_vecs;  // in words of the launch's size
  int n_blocks, rows, first_entry;   // first_entry: entries of the tensors before this one
  unsigned int parts, row_vecs;
};
struct CopyArgs {
  CopyTensor t[kCopyTensors];
  int n_tensors, pair_ints, splits;
  const int32_t* pairs;
};

template <typename V>
__global__ void __launch_bounds__(kCopyThreads) copy_blocks_kernel(const __grid_constant__ CopyArgs a) {
  pdl_wait();
  pdl_trigger();
  int at = 0;
#pragma unroll
  for (int i = 1; i < kCopyTensors; ++i)
    if (i < a.n_tensors && (int)blockIdx.y >= a.t[i].first_entry) at = i;
  const CopyTensor& t = a.t[at];
  const int pair = blockIdx.x / a.splits, split = blockIdx.x - pair * a.splits;
  const int32_t* w = a.pairs + (size_t)pair * a.pair_ints;
  const int from = w[0], to = w[1], rows = a.pair_ints == 3 ? min(w[2], t.rows) : t.rows;
  if (from < 0 || to < 0 || from >= t.n_blocks || to >= t.n_blocks || from == to || rows <= 0) return;
  V* entry = reinterpret_cast<V*>(t.base) + (blockIdx.y - t.first_entry) * t.entry_vecs;
  const V* src = entry + from * t.block_vecs;
  V* dst = entry + to * t.block_vecs;
  // a part's copied rows lie together; all of its rows are the whole block
  const unsigned int run = (unsigned int)rows * t.row_vecs, part = (unsigned int)t.rows * t.row_vecs, total = run * t.parts;
  const unsigned int chunk = kCopyThreads * kCopyLoads;
  for (unsigned int i0 = split * chunk; i0 < total; i0 += (unsigned int)a.splits * chunk) {
    V v[kCopyLoads];
    unsigned int o[kCopyLoads];
#pragma unroll
    for (int u = 0; u < kCopyLoads; ++u) {
      const unsigned int i = i0 + u * kCopyThreads + threadIdx.x;
      o[u] = run == part ? i : i / run * part + i % run;
      if (i < total) v[u] = src[o[u]];
    }
#pragma unroll
    for (int u = 0; u < kCopyLoads; ++u)
      if (i0 + u * kCopyThreads + threadIdx.x < total) dst[o[u]] = v[u];
  }
}

}  // namespace ftk

using namespace ftk;

extern "C" int ftk_copy_blocks(const FtkCopyTensor* tensors, int n_tensors, const int32_t* pairs, int pair_ints, int n_pairs, void* stream) {
  FTK_REQUIRE(n_tensors >= 0 && n_pairs >= 0 && (pair_ints == 2 || pair_ints == 3), "copy_blocks: bad counts");
  if (n_tensors == 0 || n_pairs == 0) return 0;
  FTK_REQUIRE(tensors && pairs, "copy_blocks: null pointer");
  for (int i = 0; i < n_tensors; ++i) {
    const FtkCopyTensor& t = tensors[i];
    FTK_REQUIRE(t.base && t.entries >= 1 && t.blocks >= 1 && t.parts >= 1 && t.rows >= 1 && t.row_bytes >= 1, "copy_blocks: tensor %d is empty", i);
    FTK_REQUIRE((long long)t.parts * t.rows <= 0x7fffffffLL / t.row_bytes, "copy_blocks: a block of tensor %d has 2^31 bytes or more", i);
  }
  for (int first = 0; first < n_tensors;) {
    CopyArgs a = {};
    int entries = 0, n = 0;
    unsigned long long align = 16;
    long long most = 0;  // bytes of the largest block
    for (; first + n < n_tensors && n < kCopyTensors; ++n) {
      const FtkCopyTensor& t = tensors[first + n];
      FTK_REQUIRE(t.entries <= 65535, "copy_blocks: %d entries of tensor %d", t.entries, first + n);
      if (entries + t.entries > 65535) break;
      align |= (unsigned long long)(uintptr_t)t.base | (unsigned long long)t.row_bytes;
      entries += t.entries;
      const long long block = (long long)t.parts * t.rows * t.row_bytes;
      if (block > most) most = block;
    }
    const int size = (int)(align & (~align + 1));  // the largest power of two, 16 at most, that divides every address and row
    entries = 0;
    for (int i = 0; i < n; ++i) {
      const FtkCopyTensor& t = tensors[first + i];
      CopyTensor& c = a.t[i];
      c.base = static_cast<unsigned char*>(t.base);
      c.row_vecs = (unsigned int)(t.row_bytes / size);
      c.parts = (unsigned int)t.parts;
      c.rows = t.rows;
      c.n_blocks = t.blocks;
      c.block_vecs = (long long)t.parts * t.rows * c.row_vecs;
      c.entry_vecs = c.block_vecs * t.blocks;
      c.first_entry = entries;
      entries += t.entries;
    }
    a.n_tensors = n;
    a.pairs = pairs;
    a.pair_ints = pair_ints;
    const long long chunk = (long long)kCopyThreads * kCopyLoads * size;
    const long long splits = (most + chunk - 1) / chunk;
    a.splits = (int)(splits < 1024 ? splits : 1024);
    FTK_REQUIRE((long long)n_pairs * a.splits <= 0x7fffffffLL, "copy_blocks: %d pairs are too many for one launch", n_pairs);
    const dim3 grid(n_pairs * a.splits, entries);
    note_variant(pair_ints == 3 ? "copy: rows of pages" : "copy: state slots");
    auto kern = size == 16 ? copy_blocks_kernel<uint4> : size == 8 ? copy_blocks_kernel<uint2> : size == 4 ? copy_blocks_kernel<unsigned int>
                : size == 2 ? copy_blocks_kernel<unsigned short> : copy_blocks_kernel<unsigned char>;
    FTK_LAUNCH(kern, grid, kCopyThreads, 0, (cudaStream_t)stream, a);
    FTK_LAUNCH_CHECK("copy_blocks");
    first += n;
  }
  return 0;
}
