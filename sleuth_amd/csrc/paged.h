// What the parts of the paged / windowed attention share: its parameters, a block's keys, the merge.
#pragma once

#include <atomic>

#include "common.h"
#include "forge_internal.h"

namespace forge {

// Table entries are read with scalar loads (the address is the same for the whole wave).
__device__ __forceinline__ int scalar_load(const int32_t* p) {
  return *(const __attribute__((address_space(4))) int32_t*)p;
}

// A block's share of a planned call: part `part` of `parts` of row block `pair` (b * row blocks + row block).
struct PagedItem {
  int pair, part, parts, slot;
};

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
  unsigned g_inv;  // ceil(2^32 / G): the token of a query row is one high product (rows * G < 2^32)
  int rows;        // G * T
  int limit;  // keys at or past it do not exist
  int window, sinks;
  float scale_log2;
  void* out;
  int64_t sob, sot, soh;
  // Key split: a row block's tiles go to ceil(tiles / part_tiles) blocks (at most nparts) in equal shares, each
  // writing an fp32 partial that the combine kernel merges in part order. nparts 1: no split.
  int nparts, part_tiles;
  // Fixed cut: key tile a (of the whole cache) is wave a % 4's of part a / 4 % nparts, so that what a wave adds up
  // for a query hangs on the query's own position alone, not on the other queries of its block.
  bool fixed;
  // Planned calls (the chunk kernel, rows of different lengths): block x takes item items[x / K] of KV head
  // x % K; the pairs say where the merge finds a row block's partials. Null: the static split above.
  const PagedItem* items;
  const int4* pairs;  // [B][row blocks]: (its first slot, parts, the batch row's real query rows)
  int slots;          // blocks that the device holds at a time
  float2* ws_ml;      // [slot][block's rows]
  float* ws_o;        // ... [D]
  // Arrival counters [row block of a (batch row, KV head)], all zero between calls: the last part of a row block
  // merges it. Null: the combine kernel does, launched behind.
  unsigned* counters;

  // Token of query row r (r / G).
  __device__ __forceinline__ int token(int r) const { return G == 1 ? r : (int)__umulhi((unsigned)r, g_inv); }

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
constexpr int step_rows_most(int esize, int D) { return esize * D <= 512 ? 32 : 16; }
constexpr int step_keys(int esize, int D, int rows) { return esize * D * (rows / 16) >= 1024 ? 16 : 32; }
// Its blocks per CU (registers, and 160 KB of LDS).
constexpr int step_blocks_per_cu(int esize, int D, int rows) {
  return esize * D <= 128 && rows == 16 ? 4 : esize * D <= 256 ? 2 : 1;
}

// The chunk kernel's: its launch bounds hold the compiler to the registers, its LDS is asserted. (Three at 128 bytes a
// key: a 512-token chunk at 15,360, 12 q / 4 KV heads of 64, 53 -> 45 us.)
constexpr int chunk_blocks_per_cu(int esize, int D) { return esize * D >= 1024 ? 1 : esize * D <= 128 ? 3 : 2; }

// How the host cuts a call: rows per block, keys per tile, parts.
struct PagedPlan {
  bool chunk;    // paged_chunk.hip's kernel (rows 128), or paged.hip's
  bool fixed;    // (paged.hip's) parts and waves by the tile's number in the cache
  bool planned;  // the parts are planned on the device
  int rows, keys;
  int nparts, part_tiles;
  int slots;   // blocks that the device holds at a time
  int nitems;  // planned: room for this many
};
constexpr int kPlanPairs = 4096;  // row blocks (of all batch rows) that a plan can hold

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
  int lo, se;       // what the block's queries see: keys below se (first tokens) and those from lo to last
  int sink_tiles, main_tile, tiles;
  __device__ __forceinline__ int tile_key(int i, int KT) const {
    return (i < sink_tiles ? i : main_tile + i - sink_tiles) * KT;
  }
  // A tile's ends may hold keys that no query of the block sees: past the last one, between the first tokens and the
  // window. Their weights are 0, but 0 * NaN of such a value would be NaN, so rows of keys that are seen are read in
  // their place (and a page behind the window costs no traffic). Of R keys from `group` on (a multiple of R) in the
  // tile that starts at key0: where the R keys to read start, and the key to read for `key` among those.
  template <int R> __device__ __forceinline__ int group_from(int group, int key0) const {
    if (group > last) return last & ~(R - 1);
    if (group >= se && group + R <= lo) return (key0 < se ? se - 1 : lo) & ~(R - 1);
    return group;
  }
  __device__ __forceinline__ int row_key(int from, int key) const {
    key = key < last ? key : last;
    return key >= se && key < lo ? (from < se ? se - 1 : lo) : key;
  }
};

__device__ __forceinline__ RowSpan make_span(const PagedParams& p, int base, int rows, int row0, int nrows, int KT) {
  RowSpan w;
  w.base = base;
  w.rows = rows;
  w.sink_tiles = w.main_tile = w.tiles = 0;
  w.first = w.last = w.lo = w.se = 0;
  if (row0 >= rows) return w;
  const int row1 = (row0 + nrows < rows ? row0 + nrows : rows) - 1;
  w.first = base + p.token(row0);
  w.last = base + p.token(row1);
  w.lo = p.window > 0 && w.first >= p.window ? w.first - p.window + 1 : 0;
  w.main_tile = w.lo / KT;
  w.se = p.sinks < w.lo ? p.sinks : w.lo;
  const int st = (w.se + KT - 1) / KT;
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

// What a block does: part `part` of `parts` (0 or 1: the whole) of row block rblk of (b, kvh); its tiles, and the
// slot that its partial goes to.
struct BlockWork {
  int b, kvh, rblk, part, parts, begin, end, slot;
  RowSpan span;
  bool none;  // nothing to do
};

// The parts of a row block's tiles, where the device does not plan them.
__device__ __forceinline__ int row_parts(const PagedParams& p, int tiles) {
  if (p.nparts < 2 || tiles == 0) return 1;
  return p.fixed ? p.nparts : (tiles + p.part_tiles - 1) / p.part_tiles;
}

// Grid: x (batch row, KV head), y part, z row block, late ones first (a causal chunk's have the most keys). Blocks
// start in that order, x first, so where (batch row, KV head) pairs times parts are a multiple of 8 all blocks that
// read the same keys run on one XCD and meet in its L2.
template <int BM, int KT> __device__ __forceinline__ BlockWork block_work(const PagedParams& p) {
  BlockWork w;
  const int nrb = (p.rows + BM - 1) / BM;
  w.none = true;
  if (p.items) {
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    const int x = blockIdx.x;
    w.kvh = x % p.K;
    const i32x4 it = *(const __attribute__((address_space(4))) i32x4*)(p.items + x / p.K);
    w.part = it[1];
    w.parts = it[2];
    w.slot = it[3] * p.K + w.kvh;
    w.b = it[0] / nrb;
    w.rblk = it[0] % nrb;
    if (w.parts < 0) return w;  // behind the last item
    w.span = row_span(p, w.b, w.rblk * BM, BM, KT);
  } else {
    const int pair = blockIdx.x;
    w.part = blockIdx.y;
    w.rblk = nrb - 1 - (int)blockIdx.z;
    w.b = pair / p.K;
    w.kvh = pair - w.b * p.K;
    w.span = row_span(p, w.b, w.rblk * BM, BM, KT);
    w.parts = row_parts(p, w.span.tiles);
    w.slot = (pair * nrb + w.rblk) * p.nparts + w.part;
    if (w.part > 0 && w.part >= w.parts) return w;
  }
  w.none = false;
  w.begin = 0;
  w.end = w.span.tiles;
  if (w.parts > 1) {  // equal shares: the first `more` parts take one tile more
    const int per = w.span.tiles / w.parts, more = w.span.tiles - per * w.parts;
    w.begin = w.part * per + (w.part < more ? w.part : more);
    w.end = w.begin + per + (w.part < more);
  }
  return w;
}

// The low n bits (none for n <= 0, all for n >= 32), and a score where its bit is set, else -inf.
__device__ __forceinline__ unsigned low_bits(int n) {
  return (unsigned)((1ull << (n < 0 ? 0 : n < 32 ? n : 32)) - 1);
}
__device__ __forceinline__ float masked(float s, unsigned see, int bit) {
  const int keep = (int)__builtin_amdgcn_sbfe((int)see, bit, 1);
  return __int_as_float((__float_as_int(s) & keep) | (__float_as_int(kNegInf) & ~keep));
}

// Four output channels of query row `flat` of (b, kvh).
template <typename T>
__device__ __forceinline__ void store_row(const PagedParams& p, int b, int kvh, int flat, int ch, float4 a, float f) {
  const int t = p.token(flat);
  T* dst = static_cast<T*>(p.out) + b * p.sob + (int64_t)t * p.sot + (kvh * p.G + flat - t * p.G) * p.soh + ch;
  T v[4] = {from_f32<T>(a.x * f), from_f32<T>(a.y * f), from_f32<T>(a.z * f), from_f32<T>(a.w * f)};
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(dst) = *reinterpret_cast<float4*>(v);
  else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(v);
}

// Memory that blocks on other XCDs, with L2 caches of their own, write or read in the same launch: agent-scope
// accesses go past those caches.
__device__ __forceinline__ float2 load_shared(const float2* p) {
  const uint64_t u = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((unsigned)u), __uint_as_float((unsigned)(u >> 32)));
}
__device__ __forceinline__ void store_shared(float2* p, float x, float y) {
  const uint64_t u = __float_as_uint(x) | (uint64_t)__float_as_uint(y) << 32;
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Merges a row's parts, in part order, over four channels: (m, l) at ml[i * step], outputs at o[i * step * D].
// Returns the sum of the weights. SHARED: written in this launch.
template <int D, int U, bool SHARED>
__device__ __forceinline__ float merge_parts(const float2* ml, const float* po, int parts, int64_t step, float4& O) {
  // U parts' loads go out together; the running maximum as in the kernels
  float M = kNegInf, L = 0.0f;
  O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i0 = 0; i0 < parts; i0 += U) {
    float2 e[U];
    float4 o[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = (i0 + u < parts ? i0 + u : parts - 1) * step;
      if constexpr (SHARED) {
        e[u] = load_shared(ml + at);
        const float2 x = load_shared(reinterpret_cast<const float2*>(po + at * D));
        const float2 y = load_shared(reinterpret_cast<const float2*>(po + at * D) + 1);
        o[u] = make_float4(x.x, x.y, y.x, y.y);
      } else {
        e[u] = ml[at];
        o[u] = *reinterpret_cast<const float4*>(po + at * D);
      }
    }
    float top = M;
#pragma unroll
    for (int u = 0; u < U; ++u) top = fmaxf(top, e[u].x);
    const float keep = rescale(M, top);
    L *= keep;
    O.x *= keep;
    O.y *= keep;
    O.z *= keep;
    O.w *= keep;
    M = top;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float a = i0 + u < parts ? rescale(e[u].x, M) : 0.0f;
      L += a * e[u].y;
      O.x += a * o[u].x;
      O.y += a * o[u].y;
      O.z += a * o[u].z;
      O.w += a * o[u].w;
    }
  }
  return L;
}

// Rows of a merging block: 256 threads of D / 4 lanes a row, within one row block.
constexpr int combine_rows(int D, int BM) { return 1024 / D < BM ? 1024 / D : BM; }

// Merges the parts of the rows whose tiles were split: D / 4 lanes per row, four channels each, the
// parts in order, eight at a time; four in planned calls, whose many rows of few parts want the registers for more
// waves.
template <typename T, int D, int BM, int KT, bool PLANNED>
__global__ __launch_bounds__(256) void paged_combine_kernel(PagedParams p) {
  constexpr int LPR = D / 4, RPB = combine_rows(D, BM);
  const int nrb = (p.rows + BM - 1) / BM;
  const int b = (int)blockIdx.x / p.K, kvh = (int)blockIdx.x - b * p.K;
  const int sub = blockIdx.y, rblk = blockIdx.z, pair = b * nrb + rblk;
  const int in = sub * RPB + threadIdx.x / LPR, flat = rblk * BM + in;
  const int x = 4 * (threadIdx.x % LPR);
  int rows, parts, stride;
  int64_t slot;
  if constexpr (PLANNED) {
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    const i32x4 e = *(const __attribute__((address_space(4))) i32x4*)(p.pairs + pair);
    slot = (int64_t)e[0] * p.K + kvh;
    parts = e[1];
    rows = e[2];
    stride = p.K;
  } else {
    const RowSpan w = row_span(p, b, rblk * BM, BM, KT);
    rows = w.rows;
    parts = row_parts(p, w.tiles);
    slot = ((int64_t)(b * p.K + kvh) * nrb + rblk) * p.nparts;
    stride = 1;
  }
  if (parts < 2 || flat >= rows) return;  // written by its block
  float4 O;
  const float2* ml = p.ws_ml + slot * BM + in;
  const float* po = p.ws_o + (slot * BM + in) * D + x;
  const float L = merge_parts<D, PLANNED ? 4 : 8, false>(ml, po, parts, (int64_t)stride * BM, O);
  store_row<T>(p, b, kvh, flat, x, O, L > 0.0f ? 1.0f / L : 0.0f);
}

template <typename T, int D, int BM, int KT, bool PLANNED = false> static int launch_paged_combine(const PagedParams& p, hipStream_t s) {
  constexpr int RPB = combine_rows(D, BM);
  const int64_t nrb = (p.rows + BM - 1) / BM;
  const int subs = p.rows < BM ? (p.rows + RPB - 1) / RPB : BM / RPB;  // (blocks of a row block)
  if (nrb > 65535) return set_error("forge_attn_paged: too many query rows");
  hipLaunchKernelGGL((paged_combine_kernel<T, D, BM, KT, PLANNED>), dim3((unsigned)(p.B * p.K), subs, (unsigned)nrb), dim3(RPB * (D / 4)),
                     0, s, p);
  return check_launch();
}

// Lets a kernel have `bytes` of LDS on the current device; `done` remembers on which devices (a bit each) it has them.
inline int reserve_lds(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
  if (bytes <= 64 * 1024) return 0;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return set_error("forge_attn_paged: no current device");
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return 0;
  if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
    return set_error("forge_attn_paged: cannot reserve the LDS the kernel needs");
  done.fetch_or(bit, std::memory_order_relaxed);
  return 0;
}

template <typename T> int launch_paged(const PagedParams& p, const PagedPlan& plan, int D, hipStream_t s);
template <typename T> int launch_paged_chunk(const PagedParams& p, const PagedPlan& plan, int D, hipStream_t s);

}  // namespace forge
