// What the parts of the paged / windowed attention share: its parameters, a block's keys, the merge.
#pragma once

#include "common.h"
#include "forge_internal.h"

namespace forge {

// Table entries are read with scalar loads (the address is the same for the whole wave).
__device__ __forceinline__ int scalar_load(const int32_t* p) {
  return *(const __attribute__((address_space(4))) int32_t*)p;
}

struct PagedParams {
  const void* q;
  int64_t sqb, sqh, sqt;
  const float* qw;
  float eps;
  int flags;
  const float* cos;
  const float* sin;
  int64_t csb, cst;
  const void* k;
  const void* v;
  int64_t skp, skh, sks;  // elements between pages (contiguous: batch rows), heads, positions
  const int32_t* table;   // [B][max_pages] page ids, or null: contiguous, batch row b is page b
  int64_t spt;
  int npages;
  int page_shift, page_mask;  // contiguous: 31 and 0x7fffffff
  const int32_t* row_pos;
  const int64_t* pos_dev;
  int64_t pos0;
  const int32_t* new_lens;  // or null: T each
  int B, T, H, K, G;
  int rows;   // G * T
  int limit;  // keys at or past it do not exist
  int window, sinks;
  float scale_log2;
  void* out;
  int64_t sob, sot, soh;
  // Key split: a row block's tiles go to ceil(tiles / part_tiles) blocks (at most nparts) in equal shares, each
  // writing an fp32 partial that the combine kernel merges in part order. nparts 1: no split.
  int nparts, part_tiles;
  float2* ws_ml;  // [B][K][rows][nparts]
  float* ws_o;    // ... [D]

  // The page that holds position `key` (below limit, so the table has an entry for it) of batch row b; -1
  // where the table names none of the pool.
  __device__ __forceinline__ int page_of(int b, int key) const {
    if (!table) return b;
    const int id = scalar_load(table + b * spt + (key >> page_shift));
    return (unsigned)id < (unsigned)npages ? id : -1;
  }
};

// The split kernel's largest row block and its keys per wave tile, by element size and head dim: what the
// registers hold (fewer keys in flight with more rows or wider ones).
constexpr int step_rows_most(int esize, int D) {
  return esize == 4 ? (D <= 64 ? 64 : D == 128 ? 32 : 16) : D <= 128 ? 64 : D == 256 ? 32 : 16;
}
constexpr int step_keys(int esize, int D, int rows) { return esize * D * (rows / 16) >= 1024 ? 16 : 32; }
// Its blocks per CU (registers, and 160 KB of LDS).
constexpr int step_blocks_per_cu(int esize, int D, int rows) {
  const int bytes = esize * D * (rows == 64 ? 2 : 1);
  return bytes <= 128 && rows == 16 ? 4 : bytes <= 256 ? 2 : 1;
}

// How the host cuts a call: rows per block, keys per tile, parts.
struct PagedPlan {
  bool chunk;  // paged_chunk.hip's kernel (rows 128), or paged.hip's
  int rows, keys;
  int nparts, part_tiles;
};

// Batch row b: the position of its first new token, and its real query rows (new_lens * G). A position
// outside the cache leaves nothing visible, and tokens past `limit` are not real.
__device__ __forceinline__ void row_extent(const PagedParams& p, int b, int& base, int& rows) {
  int64_t at = p.row_pos ? (int64_t)p.row_pos[b] : p.pos_dev ? *p.pos_dev : p.pos0;
  if (at < 0 || at > p.limit) at = p.limit;
  base = (int)at;
  int nl = p.new_lens ? p.new_lens[b] : p.T;
  nl = nl < 0 ? 0 : nl < p.T ? nl : p.T;
  if (nl > p.limit - base) nl = p.limit - base;
  rows = nl * p.G;
}

// The keys of query rows row0 .. row0 + nrows - 1 of a batch row, as tiles of KT keys: the tiles that hold
// first tokens (from key 0 on), then those from the first query's window to the last query.
struct RowSpan {
  int base;         // position of the row's first new token
  int rows;         // query rows of the batch row that are real
  int first, last;  // positions of the block's first and last real query
  int sink_tiles, main_tile, tiles;
  __device__ __forceinline__ int tile_key(int i, int KT) const {
    return (i < sink_tiles ? i : main_tile + i - sink_tiles) * KT;
  }
};

__device__ __forceinline__ RowSpan make_span(const PagedParams& p, int base, int rows, int row0, int nrows, int KT) {
  RowSpan w;
  w.base = base;
  w.rows = rows;
  w.sink_tiles = w.main_tile = w.tiles = 0;
  w.first = w.last = 0;
  if (row0 >= rows) return w;
  const int row1 = (row0 + nrows < rows ? row0 + nrows : rows) - 1;
  w.first = base + row0 / p.G;
  w.last = base + row1 / p.G;
  const int lo = p.window > 0 && w.first >= p.window ? w.first - p.window + 1 : 0;
  w.main_tile = lo / KT;
  const int se = p.sinks < lo ? p.sinks : lo;
  const int st = (se + KT - 1) / KT;
  w.sink_tiles = st < w.main_tile ? st : w.main_tile;
  w.tiles = w.sink_tiles + w.last / KT - w.main_tile + 1;
  return w;
}

// The same for batch row b of a block (uniform: scalar registers).
__device__ __forceinline__ RowSpan row_span(const PagedParams& p, int b, int row0, int nrows, int KT) {
  int base, rows;
  row_extent(p, b, base, rows);
  return make_span(p, __builtin_amdgcn_readfirstlane(base), __builtin_amdgcn_readfirstlane(rows), row0, nrows, KT);
}

// Part `part` of a row block's tiles; how many parts it has (0 or 1: no partials).
__device__ __forceinline__ int take_tiles(const PagedParams& p, const RowSpan& w, int part, int& begin, int& end) {
  const int parts = p.nparts < 2 ? 1 : (w.tiles + p.part_tiles - 1) / p.part_tiles;
  begin = (int)((int64_t)part * w.tiles / (parts > 1 ? parts : 1));
  end = (int)((int64_t)(part + 1) * w.tiles / (parts > 1 ? parts : 1));
  return parts;
}

// blockIdx.x -> (part, row block, batch row, KV head). Late row blocks first (a causal chunk's have the
// most keys). The (batch row, KV head, part) triples follow each other, so where they are a multiple of 8
// in number all blocks that read the same keys run on one XCD and meet in its L2.
__device__ __forceinline__ void block_unit(const PagedParams& p, int nrb, int& part, int& rblk, int& b, int& kvh) {
  const int pairs = p.B * p.K;
  const int x = blockIdx.x;
  rblk = nrb - 1 - x / (pairs * p.nparts);
  const int y = x % (pairs * p.nparts);
  const int pair = y % pairs;
  part = y / pairs;
  b = pair / p.K;
  kvh = pair % p.K;
}

// Four output channels of query row `flat` of (b, kvh).
template <typename T>
__device__ __forceinline__ void store_row(const PagedParams& p, int b, int kvh, int flat, int ch, float4 a, float f) {
  T* dst = static_cast<T*>(p.out) + b * p.sob + (int64_t)(flat / p.G) * p.sot + (kvh * p.G + flat % p.G) * p.soh + ch;
  T v[4] = {from_f32<T>(a.x * f), from_f32<T>(a.y * f), from_f32<T>(a.z * f), from_f32<T>(a.w * f)};
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(dst) = *reinterpret_cast<float4*>(v);
  else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(v);
}

// Merges the parts of the rows whose tiles were split: D / 4 lanes per row, four channels each, the
// parts in order.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_combine_kernel(PagedParams p, int block_rows, int KT) {
  constexpr int LPR = D / 4;
  const int pair = (int)blockIdx.x % (p.B * p.K);
  const int flat = (int)blockIdx.x / (p.B * p.K) * (256 / LPR) + threadIdx.x / LPR;
  const int x = 4 * (threadIdx.x % LPR);
  const int kvh = pair % p.K, b = pair / p.K;
  int base, rows;
  row_extent(p, b, base, rows);
  if (flat >= rows) return;
  const RowSpan w = make_span(p, base, rows, flat / block_rows * block_rows, block_rows, KT);
  const int parts = (w.tiles + p.part_tiles - 1) / p.part_tiles;
  if (parts < 2) return;  // written by its block
  const int64_t slot = (((int64_t)b * p.K + kvh) * p.rows + flat) * p.nparts;
  float M = kNegInf;
  for (int i = 0; i < parts; ++i) M = fmaxf(M, p.ws_ml[slot + i].x);
  float L = 0.0f;
  float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i = 0; i < parts; ++i) {
    const float2 e = p.ws_ml[slot + i];
    const float4 o = *reinterpret_cast<const float4*>(p.ws_o + (slot + i) * D + x);
    const float a = rescale(e.x, M);
    L += a * e.y;
    O.x += a * o.x;
    O.y += a * o.y;
    O.z += a * o.z;
    O.w += a * o.w;
  }
  store_row<T>(p, b, kvh, flat, x, O, L > 0.0f ? 1.0f / L : 0.0f);
}

template <typename T, int D>
static int launch_paged_combine(const PagedParams& p, int block_rows, int KT, hipStream_t s) {
  constexpr int RPB = 256 / (D / 4);
  const int64_t blocks = (int64_t)((p.rows + RPB - 1) / RPB) * p.K * p.B;
  if (blocks > 0x7fffffff) return set_error("forge_attn_paged: grid too large");
  hipLaunchKernelGGL((paged_combine_kernel<T, D>), dim3((unsigned)blocks), dim3(256), 0, s, p, block_rows, KT);
  return check_launch();
}

template <typename T> int launch_paged(const PagedParams& p, const PagedPlan& plan, int D, hipStream_t s);
template <typename T> int launch_paged_chunk(const PagedParams& p, int D, hipStream_t s);

}  // namespace forge
