// What stands around a drafted tree's attention: who sees whom (forge_tree_mask), the accepted branch's keys and values
// closing up in the cache (forge_kv_compact), copies of whole pages (forge_copy_pages).
#include <limits.h>

#include <algorithm>
#include <functional>
#include <vector>

#include "common.h"
#include "forge_internal.h"

namespace forge {

// ---------------------------------------------------------------- who sees whom
// vis(t) = {t} and vis(parent of t). Doubling: after k rounds a node has its 2^k nearest ancestors, itself among them, and
// knows the one after those, whose set it takes next; a chain of 1,024 takes ten rounds, a usual tree three. One block a
// row. Bound by its start and the rounds, a barrier and a row of LDS each: 1.9 us for a row of 12 nodes, 5.2 for 64 rows of 256.
template <int W> __global__ __launch_bounds__(1024) void tree_mask_kernel(const int32_t* parents, int64_t spb,
                                                                        const int32_t* new_lens, int T, uint64_t* mask,
                                                                        int32_t* depth) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int words = (T + 63) / 64;
  uint64_t* vis = reinterpret_cast<uint64_t*>(smem);   // [T][words]
  int* up = reinterpret_cast<int*>(vis + T * words);   // [T]
  const int b = blockIdx.x, t = threadIdx.x;
  int n = new_lens ? new_lens[b] : T;
  n = n < 0 ? 0 : n < T ? n : T;
  uint64_t own[W];
  int next = -1;
#pragma unroll
  for (int w = 0; w < W; ++w) own[w] = t < n && t / 64 == w ? 1ull << (t & 63) : 0;
  if (t < n) {
    const int a = parents[b * spb + t];
    next = a >= 0 && a < t ? a : -1;
  }
  __shared__ int more[2];   // whether a node of this round, or the next, has an ancestor left to take
  if (t == 0) more[0] = 0;
  __syncthreads();
  for (int round = 0; round <= 10; ++round) {
    if (t < T) {
#pragma unroll
      for (int w = 0; w < W; ++w)
        if (w < words) vis[t * words + w] = own[w];
      up[t] = next;
    }
    if (t == 0) more[(round + 1) & 1] = 0;
    if (next >= 0) more[round & 1] = 1;
    __syncthreads();
    if (!more[round & 1]) break;   // (in round ten at the latest: the ancestor that is next is 2^round nodes up)
    if (next >= 0) {
#pragma unroll
      for (int w = 0; w < W; ++w)
        if (w < words) own[w] |= vis[next * words + w];
      next = up[next];
    }
    __syncthreads();
  }
  if (t >= T) return;
  int d = -1;
  const int64_t at = (int64_t)b * T + t;
#pragma unroll
  for (int w = 0; w < W; ++w)
    if (w < words) {
      mask[at * words + w] = own[w];
      d += __popcll(own[w]);
    }
  depth[at] = d < 0 ? 0 : d;
}

// ---------------------------------------------------------------- moves within the cache
constexpr int kMoveLayers = 64;   // layers of one launch (their pointers are kernel arguments)
struct MoveParams {
  const void* kv[2 * kMoveLayers];  // K and V of each layer
  int64_t skp, skh, sks;            // bytes between pages (contiguous: batch rows), heads, positions
  int K, chunks;                    // KV heads; 16-byte chunks of a position
  int npages, page_shift, page_mask;
  // compaction
  const int32_t* table;
  int64_t spt;
  int limit;
  const int32_t* row_pos;
  const int64_t* pos_dev;
  int64_t pos0;
  const int32_t* path;
  int64_t s_path;
  const int32_t* counts;
  int T;
  // copies
  const int32_t* src;
  const int32_t* dst;
  int n, page;
};

// The accepted branch closes up: slot base + i takes what slot base + path[i] holds, for i below the row's count. Entries
// with path[i] < i or beyond the cache move nothing; all others lie at or behind their place, so that in rising order,
// eight at a time, each is read before anything is written to it. A thread owns one 16-byte chunk of one head of one
// layer's K or V, for the whole path. Latency, position, entry, pages, chunk: 3.4 us for one row of 28 layers, 8.3 for 64
// rows' 19 MB over pages (12.4 with all sixteen pages of a batch looked up at once, 10.7 by scalar loads: most entries of
// a path are not there).
__global__ __launch_bounds__(256) void kv_compact_kernel(MoveParams p) {
  const int b = blockIdx.z, unit = blockIdx.x * 256 + threadIdx.x;
  const int head = unit / p.chunks, chunk = unit - head * p.chunks;
  if (head >= p.K) return;
  char* kv = static_cast<char*>(const_cast<void*>(p.kv[blockIdx.y])) + head * p.skh + chunk * 16;
  int64_t base = row_base(p.row_pos, p.pos_dev, p.pos0, b);
  if (base < 0 || base > p.limit) return;
  int n = p.counts[b];
  n = n < p.T ? n : p.T;
  const auto slot = [&](int64_t key) -> char* {
    int64_t page = b;
    if (p.table) {
      page = p.table[b * p.spt + (key >> p.page_shift)];
      if (page < 0 || page >= p.npages) return nullptr;
    }
    return kv + page * p.skp + (key & p.page_mask) * p.sks;
  };
  for (int i0 = 0; i0 < n; i0 += 8) {
    uint4 x[8];
    char* to[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      to[j] = nullptr;
      const int i = i0 + j;
      if (i >= n) continue;
      const int of = p.path[b * p.s_path + i];
      if (of <= i || base + of >= p.limit) continue;
      const char* from = slot(base + of);
      if (!from) continue;
      to[j] = slot(base + i);
      x[j] = load16(from);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (to[j]) store16(to[j], x[j]);
  }
}

// Page dst[i] takes what page src[i] holds. A block takes 256 chunks x 4 of one page of one layer's K or V. As fast as a
// copy: 64 pages of 128 KB in 28 layers 178 us, 5.3 TB/s (a 1 GiB copy 5.15).
constexpr int kCopyPer = 4;
__global__ __launch_bounds__(256) void copy_pages_kernel(MoveParams p) {
  const int i = blockIdx.y;
  const int from = p.src[i], to = p.dst[i];
  if (from < 0 || from >= p.npages || to < 0 || to >= p.npages || from == to) return;
  char* kv = static_cast<char*>(const_cast<void*>(p.kv[blockIdx.z]));
  const int all = p.K * p.page * p.chunks;
  uint4 x[kCopyPer];
  int64_t at[kCopyPer];
#pragma unroll
  for (int j = 0; j < kCopyPer; ++j) {
    const int c = (blockIdx.x * kCopyPer + j) * 256 + threadIdx.x;
    at[j] = -1;
    if (c >= all) continue;
    const int row = c / p.chunks, head = row / p.page;
    at[j] = head * p.skh + (row - head * p.page) * p.sks + (c - row * p.chunks) * 16;
    x[j] = load16(kv + from * p.skp + at[j]);
  }
#pragma unroll
  for (int j = 0; j < kCopyPer; ++j)
    if (at[j] >= 0) store16(kv + to * p.skp + at[j], x[j]);
}

// What both moves check, and the layers' strides in bytes.
static const char* move_setup(MoveParams& p, int esize, int layers, const void* const* k, const void* const* v, int K, int D,
                              int64_t skp, int64_t skh, int64_t sks) {
  if (esize != 2 && esize != 4) return "elements have 2 or 4 bytes";
  if (layers < 0 || K <= 0 || D <= 0) return "bad sizes";
  if (D * esize % 16) return "a head's channels must be a multiple of 16 bytes";
  if ((int64_t)K * (D * esize / 16) > INT_MAX / 256) return "too many heads";
  if (layers > 0 && (!k || !v)) return "null layer pointers";
  for (const int64_t s : {skp, skh, sks})
    if (s < 0 || s * esize % 16) return "strides must be multiples of 16 bytes";
  for (int l = 0; l < layers; ++l)
    if (!k[l] || !v[l] || (uintptr_t)k[l] % 16 || (uintptr_t)v[l] % 16) return "the caches must be 16-byte aligned";
  p.skp = skp * esize; p.skh = skh * esize; p.sks = sks * esize;
  p.K = K; p.chunks = D * esize / 16;
  return nullptr;
}
// A cache named twice would be moved by two blocks at once, one of which may read what the other has moved already.
static bool named_twice(int layers, const void* const* k, const void* const* v) {
  const std::less<const void*> before;
  const auto rises = [&](const void* const* x) {
    for (int l = 1; l < layers; ++l)
      if (!before(x[l - 1], x[l])) return false;
    return true;
  };
  if (rises(k) && rises(v)) {   // (as allocated one after the other: no memory of its own needed)
    for (int i = 0, j = 0; i < layers && j < layers;) {
      if (k[i] == v[j]) return true;
      if (before(k[i], v[j])) ++i;
      else ++j;
    }
    return false;
  }
  std::vector<const void*> all(k, k + layers);
  all.insert(all.end(), v, v + layers);
  std::sort(all.begin(), all.end(), before);
  return std::adjacent_find(all.begin(), all.end()) != all.end();
}
static int take_layers(MoveParams& p, int l0, int layers, const void* const* k, const void* const* v) {
  const int n = layers - l0 < kMoveLayers ? layers - l0 : kMoveLayers;
  for (int l = 0; l < n; ++l) {
    p.kv[2 * l] = k[l0 + l];
    p.kv[2 * l + 1] = v[l0 + l];
  }
  return n;
}

}  // namespace forge

using namespace forge;

extern "C" int forge_tree_mask(int B, int T, const int32_t* parents, int64_t s_parents_b, const int32_t* new_lens, int64_t* mask,
                               int32_t* depth, void* stream) {
  clear_error();
  if (B < 0 || T < 0) return set_error("bad sizes");
  if (T > FORGE_TREE_MAX_TOKENS) return set_error("a tree has at most 1024 tokens");
  if (B == 0 || T == 0) return 0;
  if (!parents || !mask || !depth || s_parents_b < 0) return set_error("null tensor pointer");
  const int words = (T + 63) / 64;
  const size_t lds = (size_t)T * (words * 8 + 4);
  const dim3 threads((unsigned)words * 64);
  const hipStream_t s = (hipStream_t)stream;
  uint64_t* m = reinterpret_cast<uint64_t*>(mask);
  if (words == 1) hipLaunchKernelGGL(tree_mask_kernel<1>, dim3(B), threads, lds, s, parents, s_parents_b, new_lens, T, m, depth);
  else if (words <= 4) hipLaunchKernelGGL(tree_mask_kernel<4>, dim3(B), threads, lds, s, parents, s_parents_b, new_lens, T, m, depth);
  else {
    if (lds > 64 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void*>(&tree_mask_kernel<16>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
      return set_error("cannot reserve the LDS the kernel needs");
    hipLaunchKernelGGL(tree_mask_kernel<16>, dim3(B), threads, lds, s, parents, s_parents_b, new_lens, T, m, depth);
  }
  return check_launch();
}

extern "C" int forge_kv_compact(int esize, int layers, int B, int K, int D, const void* const* k, const void* const* v,
                                int64_t skp, int64_t skh, int64_t sks, int n_pages, int64_t page_size,
                                const int32_t* page_table, int64_t s_table, int max_pages, const int32_t* row_pos,
                                const int64_t* pos_dev, int64_t pos0, const int32_t* path, int64_t s_path, int T,
                                const int32_t* counts, void* stream) {
  clear_error();
  MoveParams p{};
  if (const char* why = move_setup(p, esize, layers, k, v, K, D, skp, skh, sks)) return set_error(why);
  if (B < 0 || B > 65535 || T < 0) return set_error("bad sizes (at most 65,535 rows)");
  if (page_size <= 0) return set_error("the cache's length must be positive");
  if (page_table && (page_size < 16 || (page_size & (page_size - 1)) || page_size > INT_MAX))
    return set_error("the page size must be a power of two of at least 16");
  if (page_table && (n_pages <= 0 || max_pages <= 0 || s_table < 0)) return set_error("bad page table sizes");
  if (page_table && !row_pos) return set_error("a paged cache needs row positions");
  if (layers == 0 || B == 0 || T == 0) return 0;
  if (!path || !counts || s_path < 0) return set_error("null path or counts");
  const int64_t limit = page_table ? max_pages * page_size : page_size;
  if (limit > INT_MAX) return set_error("rows are limited to 2^31 - 1 keys");
  try {
    if (named_twice(layers, k, v)) return set_error("a cache is named twice: its keys would move twice");
  } catch (...) {
    return set_error("no memory");
  }
  p.limit = (int)limit;
  p.table = page_table; p.spt = s_table; p.npages = n_pages;
  p.page_shift = page_table ? __builtin_ctz((unsigned)page_size) : 31;
  p.page_mask = page_table ? (int)page_size - 1 : 0x7fffffff;
  p.row_pos = row_pos; p.pos_dev = pos_dev; p.pos0 = pos0;
  p.path = path; p.s_path = s_path; p.counts = counts; p.T = T;
  for (int l0 = 0; l0 < layers; l0 += kMoveLayers) {
    const int n = take_layers(p, l0, layers, k, v);
    hipLaunchKernelGGL(kv_compact_kernel, dim3((K * p.chunks + 255) / 256, 2 * n, B), dim3(256), 0, (hipStream_t)stream, p);
    if (const int st = check_launch()) return st;
  }
  return 0;
}

extern "C" int forge_copy_pages(int esize, int layers, int K, int D, const void* const* k, const void* const* v, int64_t skp,
                                int64_t skh, int64_t sks, int n_pages, int page_size, int n, const int32_t* src,
                                const int32_t* dst, void* stream) {
  clear_error();
  MoveParams p{};
  if (const char* why = move_setup(p, esize, layers, k, v, K, D, skp, skh, sks)) return set_error(why);
  if (page_size < 16 || (page_size & (page_size - 1))) return set_error("the page size must be a power of two of at least 16");
  if (n_pages <= 0 || n < 0) return set_error("bad sizes");
  if (layers == 0 || n == 0) return 0;
  if (!src || !dst) return set_error("null page numbers");
  if ((int64_t)K * page_size * p.chunks > INT_MAX / 2) return set_error("pages are too large");
  p.npages = n_pages; p.page = page_size;
  const int all = K * page_size * p.chunks, blocks = (all + 256 * kCopyPer - 1) / (256 * kCopyPer);
  for (int i0 = 0; i0 < n; i0 += 65535) {
    p.src = src + i0; p.dst = dst + i0;
    const int m = n - i0 < 65535 ? n - i0 : 65535;
    for (int l0 = 0; l0 < layers; l0 += kMoveLayers) {
      const int c = take_layers(p, l0, layers, k, v);
      hipLaunchKernelGGL(copy_pages_kernel, dim3(blocks, m, 2 * c), dim3(256), 0, (hipStream_t)stream, p);
      if (const int st = check_launch()) return st;
    }
  }
  return 0;
}
