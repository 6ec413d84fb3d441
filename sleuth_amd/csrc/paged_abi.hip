// Entry points of the paged cache and of attention with sinks (kernels: paged.hip): argument checks, the
// cut of a call into blocks, the launch.
#include <limits.h>
#include <math.h>

#include "paged.h"

namespace forge {

extern template int launch_paged<bf16>(const PagedParams&, const PagedPlan&, int, hipStream_t);
extern template int launch_paged<f16>(const PagedParams&, const PagedPlan&, int, hipStream_t);
extern template int launch_paged_chunk<bf16>(const PagedParams&, const PagedPlan&, int, hipStream_t);
extern template int launch_paged_chunk<f16>(const PagedParams&, const PagedPlan&, int, hipStream_t);
extern template int launch_paged_chunk<float>(const PagedParams&, const PagedPlan&, int, hipStream_t);
extern template int launch_paged<float>(const PagedParams&, const PagedPlan&, int, hipStream_t);

static bool paged_dim_ok(int dtype, int D) {
  return D == 32 || D == 64 || D == 128 || D == 256 || (D == 512 && dtype != FORGE_F32);
}

// Rows per block, keys per tile and the key split of a call whose rows hold at most max_kv keys.
// ragged: the rows may have different lengths (row_pos).
static PagedPlan paged_plan(int dtype, int B, int T, int H, int K, int D, int64_t max_kv, int window, int sinks,
                            bool ragged, bool split) {
  PagedPlan plan{};
  const int es = dtype == FORGE_F32 ? 4 : 2, G = H / K, cus = device_cus();
  const int64_t rows = (int64_t)G * T;
  // tiles that a block can have: its queries' window and the first tokens (whose ends may lie inside tiles), or
  // the whole row; and the call's blocks
  const auto tiles_of = [&] {
    const int64_t tokens = rows < plan.rows ? T : (plan.rows - 1) / G + 2;
    const int64_t all = (max_kv + plan.keys - 1) / plan.keys;
    if (window <= 0) return all;
    const int64_t seen = (window + tokens + plan.keys - 3) / plan.keys + 1 + (sinks + plan.keys - 1) / plan.keys;
    return seen < all ? seen : all;
  };
  const auto units_of = [&] { return (int64_t)B * K * ((rows + plan.rows - 1) / plan.rows); };
  plan.rows = 16;
  plan.keys = step_keys(es, D, 16);
  const int64_t work = units_of() * tiles_of(), round = (int64_t)cus * step_blocks_per_cu(es, D, 16);
  // More than 32 rows go to the chunk kernel, whose waves share each key tile; up to 32 the split kernel's waves keep
  // more bytes in flight. us, split / chunk: 34 rows (8 batch rows of 2,000 keys, 8 KV heads, head dim 128) 27.8 / 23.9,
  // 40 rows (32 of 8,000) 239 / 194, 32 rows 183 / 196; head dim 256, one KV head, 16 batch rows of 8,000: 40 rows
  // 50.6 / 45.4, 32 rows (64 batch rows) 99.6 / 118. Head dim 512, where the split kernel has room for 16 rows, from 17
  // on: 32 rows (8 batch rows of 4,000) 30.1 / 26.9, 8,192 (1 of 4,600) 404 / 113. In fp32, where a tile's products take
  // 3.4 us a wave, from 65 rows and head dim 64 on: 80 rows (8 of 2,000) 111 / 85, 40 rows 64.7 / 79; 600 new tokens 143 /
  // 127, 700 at head dim 256 116 / 92; head dim 32 (2 rows of 333) 15.5 / 23.8.
  // A call whose 16-row blocks have few tiles is a matter of latency, and goes to them whatever its rows: up to six
  // tiles for each block that the device holds. us, split / chunk: 256 new tokens at head dim 256 12.1 / 16.7 (4 tiles
  // each), 12 behind 8,000 22.2 / 24.6 (5.9), 60 behind 300 at head dim 512 21.2 / 26.7 (5.6); four rows of 48 behind 500
  // at head dim 256 23.9 / 17.4 (6.8), 100 fp32 tokens behind 500 26.0 / 21.3 (7.7).
  // Head dim 32 in 16 bits, four split blocks a CU, from 60 tiles each on: 6 rows of 3,898 tokens, window 897, 62.5 /
  // 44.3, 500 tokens behind 8,000 24.2 / 20.1; four prompts of 700 (30 tiles) 8.7 / 13.5.
  const bool rows_enough = rows > (es == 4 ? 64 : D == 512 ? 16 : 32);
  if (rows_enough && (D >= 64 ? work > 6 * round : es == 2 && work > 60 * round)) {
    plan.chunk = true;
    plan.rows = 128;
    plan.keys = es * D >= 512 ? 32 : 64;
  } else if (rows > 16 && work > 16 * round && step_rows_most(es, D) >= 32) {
    // 32 rows a block read the keys half as often, 16 rows make twice the blocks: up to 16 tiles for each that the device
    // holds. us, 16 / 32 rows: 32 query rows over 1,500 keys at head dim 256 14.1 / 17.6, over 8,000 (15.6 tiles each)
    // 24.7 / 27.0; 16 batch rows of 1,024-key windows at head dim 128 (17 tiles) 27.1 / 21.2, 32 of 8,000 341 / 182;
    // 333 tokens at head dim 32 in fp32 12.6 / 13.1, 2,000 in bf16 37.9 / 29.2 (64 rows a block 31.8).
    plan.rows = 32;
    plan.keys = step_keys(es, D, 32);
  }
  plan.nparts = 1;
  if (!split) return plan;
  const int64_t tiles = tiles_of(), units = units_of();
  plan.slots = cus * (plan.chunk ? chunk_blocks_per_cu(es, D) : step_blocks_per_cu(es, D, plan.rows));
  const int64_t slots = plan.slots;
  const int64_t blocks = units / K;
  // (the plan adds up tiles in 32 bits)
  if (plan.chunk && ragged && B > 1 && K <= 64 && units < 2 * slots && blocks <= kPlanPairs && units * tiles > 16 * slots &&
      blocks * tiles <= INT_MAX / 4) {
    plan.planned = true;
    plan.nitems = (int)(plan.slots / K + blocks);
    return plan;
  }
  // Parts that are on the device together: one more would wait for a whole part of the others (us, with parts rounded
  // up / down: 1,548 tokens, window 882, 32 q / 8 KV heads 52.0 / 32.2; 56 at head dim 512 28.3 / 14.3).
  const int64_t fit = slots / units < 1 ? 1 : slots / units;
  int64_t per = (tiles + fit - 1) / fit;
  if (plan.chunk) {
    // n tiles in p parts take n / p of a tile's time, then the merge: p of its steps one after the other, the partials
    // of all units, and a launch; in 16 bits about p (4 + units) / 64 + 3 tiles' time, an eighth of the long ones' in
    // fp32. us, eight tiles at least / so: 100 new tokens behind 2,000 at head dim 128 18.6 / 15.1, 234 behind 319 at 256
    // 22.7 / 20.1, 788 with a window of 256 24.3 / 22.6; at 7 rows of 432 (window 256) two parts 31.5, one 17.2.
    const int64_t tile = es == 4 ? 512 : 64;
    int64_t p = (int64_t)sqrt((double)(tile * tiles) / (double)(4 + units));
    p = p < 1 ? 1 : p < fit ? p : fit;
    const int64_t n = (tiles + p - 1) / p;
    per = n * tile + p * (4 + units) + 192 < tiles * tile ? n : tiles;
  } else {
    // two tiles at least for each wave, one of the long ones from 512 bytes a key on (us, two / one: 32 rows of 1,500 keys
    // at head dim 256 15.7 / 14.1, 2 rows of 800 at head dim 512 19.2 / 16.3, but one of 8,000 at 128 14.2 / 15.8).
    // Rows of different lengths end at different times, so long ones are cut though the blocks fill the device already, as
    // long as those are fewer than eight for each that it holds: us, cut / whole, a step of 128 rows of up to 32,767 keys (8 KV
    // heads, head dim 128, 2 blocks for each) 1,274 / 1,460, of 512 of up to 16,000 (8) 2,652 / 2,681, of 1,024 of up to 8,000
    // (16) 2,718 / 2,674; fp32 prompts of 4,096 at head dim 32 behind 15,000 (8) 2,848 / 2,456 and four of them behind 28,000
    // (32) 21,947 / 18,660, whose partials were 1.1 GB.
    const int64_t least = es * D >= 512 ? 4 : 8, most = (step_blocks_per_cu(es, D, plan.rows) > 1 ? 2048 : 4096) / plan.keys;
    if (per > most && units < 8 * slots) per = most;
    if (per < least) per = least;
  }
  int64_t parts = (tiles + per - 1) / per;
  if (parts > 65535) parts = 65535;  // (the grid's)
  if (parts > 1) {
    plan.nparts = (int)parts;
    plan.part_tiles = (int)((tiles + parts - 1) / parts);
  }
  return plan;
}

// A step whose sums must not hang on how many tokens it has, or on the bound of its keys: everything as for one token
// of rows that hold all that the cache can (max_len) or the window lets them see. Where a call's query rows are more
// than a block's, 32 rows a block read the keys half as often, if their tiles are the same. What it costs (us, free /
// fixed cut, window 1,024): a token of 16 rows, 8 KV heads of 128, 17.2 / 18.1, of one row 9.0 / 9.0; 5 tokens of 8 rows there
// 13.1 / 13.6; 4 of 8 rows, one KV head of 256 with 8 query heads, 12.2 / 13.9. Verify steps of many rows, which the chunk
// kernel would take, pay most: 5 tokens of 32 rows, 28 q / 4 KV heads of 128, 24.3 / 33.3; 8 of 16 rows, 16 q / 1 KV head of
// 512, 36 / 124.
static PagedPlan fixed_plan(int dtype, int B, int T, int H, int K, int D, int64_t max_len, int window, int sinks, bool split) {
  PagedPlan plan{};
  const int es = dtype == FORGE_F32 ? 4 : 2, G = H / K;
  plan.fixed = true;
  plan.keys = step_keys(es, D, 16);
  plan.rows = G * T > 16 && step_rows_most(es, D) >= 32 && step_keys(es, D, 32) == plan.keys ? 32 : 16;
  plan.nparts = 1;
  if (!split) return plan;
  const int64_t all = (max_len + plan.keys - 1) / plan.keys;
  const int64_t seen = ((int64_t)window + FORGE_FIXED_CUT_MAX_T + plan.keys - 3) / plan.keys + 1 +
                       ((int64_t)sinks + plan.keys - 1) / plan.keys;
  const int64_t tiles = seen < all ? seen : all, units = (int64_t)B * K * ((G + 15) / 16);
  const int64_t slots = (int64_t)device_cus() * step_blocks_per_cu(es, D, 16);
  // Two tiles at most for each wave, one of the long ones, where the device has room for that many blocks.
  const int64_t least = es * D >= 512 ? 4 : 8, most = (tiles + least - 1) / least;
  int64_t parts = slots / units;
  if (parts > most) parts = most;
  plan.nparts = (int)(parts < 1 ? 1 : parts > 4096 ? 4096 : parts);
  return plan;
}

// The workspace: the counters, [items | row blocks' parts] of a planned call, then (m, l) and the output of every
// slot's rows.
struct PagedWs {
  size_t items, pairs, ml, o, bytes;
};
static PagedWs paged_ws(const PagedPlan& plan, int B, int T, int H, int K, int D) {
  PagedWs w{};
  if (plan.nparts < 2 && !plan.planned) return w;
  const auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  const size_t blocks = (size_t)B * (((size_t)(H / K) * T + plan.rows - 1) / plan.rows);
  const size_t rows = (plan.planned ? (size_t)plan.nitems : blocks * plan.nparts) * K * plan.rows;
  w.items = FORGE_PAGED_COUNTER_BYTES;
  w.pairs = w.items + (plan.planned ? up(plan.nitems * sizeof(PagedItem)) : 0);
  w.ml = w.pairs + (plan.planned ? up(blocks * sizeof(int4)) : 0);
  w.o = w.ml + up(rows * sizeof(float2));
  w.bytes = w.o + rows * D * sizeof(float);
  return w;
}

static bool unaligned(const void* p) { return (uintptr_t)p % 16 != 0; }

// Checks what both entry points share, cuts the call and launches it.
static int paged_run(int dtype, int D, PagedParams p, int64_t max_kv, float scale, void* workspace,
                     size_t workspace_bytes, int ws_flags, hipStream_t s) {
  if (dtype != FORGE_F32 && dtype != FORGE_BF16 && dtype != FORGE_F16) return set_error("unknown dtype code");
  if (p.B < 0 || p.T < 0 || p.H <= 0 || p.K <= 0 || p.H % p.K) return set_error("bad sizes (H must be a multiple of K)");
  if (!paged_dim_ok(dtype, D)) return set_error("head dim must be 32, 64, 128, 256 (or 512 in bf16/fp16)");
  if (!p.q || !p.k || !p.v || !p.out) return set_error("null tensor pointer");
  if (p.window < 0 || p.sinks < 0 || p.window > INT_MAX / 2 || p.sinks > INT_MAX / 2)
    return set_error("window and sinks must not be negative");
  if (p.sinks > 0 && p.window == 0) return set_error("sinks need a window (without one every key is visible)");
  if (!scale_ok(scale)) return set_error("scale must be positive and finite");
  const int64_t es = dtype == FORGE_F32 ? 4 : 2, e16 = 16 / es;
  for (const int64_t st : {p.sqb, p.sqh, p.sqt, p.skp, p.skh, p.sks, p.sob, p.soh, p.sot})
    if (st < 0 || st % e16) return set_error("strides must be multiples of 16 bytes");
  if ((p.B > 1 && p.sob == 0) || (p.T > 1 && p.sot == 0) || (p.H > 1 && p.soh == 0)) return set_error("out's rows overlap");
  if (unaligned(p.q) || unaligned(p.k) || unaligned(p.v) || unaligned(p.out))
    return set_error("q, k, v and out must be 16-byte aligned");
  if (p.sks < D || p.sks > INT_MAX / 16 / 64) return set_error("cache positions must be head dim to 2^21 elements apart");
  if ((p.flags & FORGE_NORM_QK) && p.qw && unaligned(p.qw)) return set_error("the norm gain must be 16-byte aligned");
  if ((p.flags & FORGE_ROPE) && (!p.cos || !p.sin)) return set_error("FORGE_ROPE needs cos and sin");
  p.G = p.H / p.K;
  if ((int64_t)p.G * p.G * p.T > INT_MAX || (int64_t)p.B * p.K > INT_MAX) return set_error("too many query rows");
  p.g_inv = (unsigned)(((1ull << 32) + p.G - 1) / p.G);
  p.rows = p.G * p.T;
  p.scale_log2 = scale * kLog2e;
  const bool split = workspace != nullptr;
  const PagedPlan plan = p.fixed ? fixed_plan(dtype, p.B, p.T, p.H, p.K, D, max_kv, p.window, p.sinks, split)
                                 : paged_plan(dtype, p.B, p.T, p.H, p.K, D, max_kv, p.window, p.sinks, p.row_pos != nullptr, split);
  p.nparts = plan.nparts;
  p.part_tiles = plan.part_tiles;
  p.slots = plan.slots;
  const PagedWs ws = paged_ws(plan, p.B, p.T, p.H, p.K, D);
  if (ws.bytes) {
    if (workspace_bytes < ws.bytes) return set_error("workspace too small");
    if ((uintptr_t)workspace % 256) return set_error("the workspace must be 256-byte aligned");
    char* at = static_cast<char*>(workspace);
    if (plan.planned) {
      p.items = reinterpret_cast<PagedItem*>(at + ws.items);
      p.pairs = reinterpret_cast<int4*>(at + ws.pairs);
    }
    p.ws_ml = reinterpret_cast<float2*>(at + ws.ml);
    p.ws_o = reinterpret_cast<float*>(at + ws.o);
    // The last part merges where that is little for one block; else the combine kernel spreads it over many. us, last
    // part / combine: 4 rows of 1,000 keys (6 KB) 7.3 / 9.4, 16 rows of 1,024-key windows (4 KB) 18.1 / 19.2; one row
    // of 8,000 keys (32 KB) 15.2 / 13.7, one KV head of 256 with 32 query rows (288 KB) 29.4 / 17.7.
    const int64_t units = (int64_t)p.B * p.K * ((p.rows + plan.rows - 1) / plan.rows);
    const int64_t bytes = (int64_t)(p.rows < plan.rows ? p.rows : plan.rows) * D * 4 * plan.nparts;
    if ((ws_flags & FORGE_WS_ZEROED) && !plan.chunk && units <= FORGE_PAGED_COUNTER_BYTES / 4 && bytes <= 16 * 1024)
      p.counters = reinterpret_cast<unsigned*>(at);
  }
  switch (dtype) {
    case FORGE_F32: return plan.chunk ? launch_paged_chunk<float>(p, plan, D, s) : launch_paged<float>(p, plan, D, s);
    case FORGE_BF16: return plan.chunk ? launch_paged_chunk<bf16>(p, plan, D, s) : launch_paged<bf16>(p, plan, D, s);
    default: return plan.chunk ? launch_paged_chunk<f16>(p, plan, D, s) : launch_paged<f16>(p, plan, D, s);
  }
}

}  // namespace forge

using namespace forge;

extern "C" size_t forge_attn_paged_workspace_bytes(int dtype, int B, int T, int H, int K, int D, int64_t max_kv_len,
                                                   int window, int sinks) {
  if (B <= 0 || T <= 0 || H <= 0 || K <= 0 || H % K || !paged_dim_ok(dtype, D) || max_kv_len <= 0 || window < 0 ||
      sinks < 0 || max_kv_len > INT_MAX)
    return 0;
  const auto bytes = [&](bool ragged, bool* planned) {
    const PagedPlan plan = paged_plan(dtype, B, T, H, K, D, max_kv_len, window, sinks, ragged, true);
    *planned = plan.planned;
    return paged_ws(plan, B, T, H, K, D).bytes;
  };
  bool planned;
  const size_t a = bytes(true, &planned);
  if (!planned) return a;
  const size_t b = bytes(false, &planned);  // (without row positions nothing is planned: what either needs)
  return a > b ? a : b;
}

extern "C" int forge_attn_paged(int dtype, int B, int T, int H, int K, int D, const void* q, int64_t sqb, int64_t sqh,
                                int64_t sqt, const float* q_weight, float eps, int flags, const float* cos,
                                const float* sin, int64_t s_cos_b, int64_t s_cos_t, const void* k_pages,
                                const void* v_pages, int64_t skp, int64_t skh, int64_t sks, int n_pages, int page_size,
                                const int32_t* page_table, int64_t s_table, int max_pages, const int32_t* row_pos,
                                const int32_t* new_lens, int64_t max_kv_len, int window, int sinks, float scale,
                                void* out, int64_t sob, int64_t sot, int64_t soh, void* workspace,
                                size_t workspace_bytes, int ws_flags, void* stream) {
  clear_error();
  if (page_size < 16 || (page_size & (page_size - 1))) return set_error("the page size must be a power of two of at least 16");
  if (n_pages <= 0 || max_pages <= 0 || s_table < 0) return set_error("bad page table sizes");
  if (flags & FORGE_FIXED_CUT) return set_error("FORGE_FIXED_CUT is for forge_attn_sinks");
  if (max_kv_len <= 0) return set_error("max_kv_len must be positive");
  if (B == 0 || T == 0) return 0;  // (torch's empty tensors have no address)
  if (!page_table || !row_pos) return set_error("null page table or row positions");
  int64_t limit = (int64_t)max_pages * page_size;
  if (max_kv_len < limit) limit = max_kv_len;
  if (limit > INT_MAX - 65536) return set_error("rows are limited to 2^31 - 65536 keys");
  if (max_kv_len > INT_MAX) max_kv_len = limit;
  PagedParams p{};
  p.q = q; p.sqb = sqb; p.sqh = sqh; p.sqt = sqt;
  p.qw = q_weight; p.eps = eps; p.flags = flags;
  p.cos = cos; p.sin = sin; p.csb = s_cos_b; p.cst = s_cos_t;
  p.k = k_pages; p.v = v_pages; p.skp = skp; p.skh = skh; p.sks = sks;
  p.table = page_table; p.spt = s_table; p.npages = n_pages;
  p.page_shift = __builtin_ctz((unsigned)page_size); p.page_mask = page_size - 1;
  p.row_pos = row_pos; p.new_lens = new_lens;
  p.B = B; p.T = T; p.H = H; p.K = K; p.limit = (int)limit; p.window = window; p.sinks = sinks;
  p.out = out; p.sob = sob; p.sot = sot; p.soh = soh;
  return paged_run(dtype, D, p, max_kv_len, scale, workspace, workspace_bytes, ws_flags, (hipStream_t)stream);
}

extern "C" size_t forge_attn_sinks_workspace_bytes(int dtype, int B, int T, int H, int K, int D, int64_t max_kv_len,
                                                   int window, int sinks) {
  return forge_attn_paged_workspace_bytes(dtype, B, T, H, K, D, max_kv_len, window, sinks);
}

extern "C" size_t forge_attn_sinks_fixed_workspace_bytes(int dtype, int B, int T, int H, int K, int D, int64_t max_len,
                                                         int window, int sinks) {
  if (B <= 0 || T <= 0 || T > FORGE_FIXED_CUT_MAX_T || H <= 0 || K <= 0 || H % K || !paged_dim_ok(dtype, D) || max_len <= 0 ||
      window <= 0 || sinks < 0)
    return 0;
  return paged_ws(fixed_plan(dtype, B, T, H, K, D, max_len, window, sinks, true), B, T, H, K, D).bytes;
}

extern "C" int forge_attn_sinks(int dtype, int B, int T, int H, int K, int D, const void* q, int64_t sqb, int64_t sqh,
                                int64_t sqt, const float* q_weight, float eps, int flags, const float* cos,
                                const float* sin, int64_t s_cos_b, int64_t s_cos_t, const void* k_cache,
                                const void* v_cache, int64_t skb, int64_t skh, int64_t sks, int64_t max_len,
                                const int32_t* row_pos, const int64_t* pos_dev, int64_t pos0, int64_t max_kv_len,
                                int window, int sinks, float scale, void* out, int64_t sob, int64_t sot, int64_t soh,
                                void* workspace, size_t workspace_bytes, int ws_flags, void* stream) {
  clear_error();
  if (window <= 0) return set_error("forge_attn_sinks needs a window");
  if (max_kv_len <= 0 || max_len <= 0) return set_error("max_kv_len and max_len must be positive");
  const int64_t limit = max_kv_len < max_len ? max_kv_len : max_len;
  if (limit > INT_MAX - 65536) return set_error("rows are limited to 2^31 - 65536 keys");
  if (B == 0 || T == 0) return 0;
  if (!row_pos && !pos_dev && (pos0 < 0 || T < 0 || pos0 > limit - T))
    return set_error("pos + T exceeds max_kv_len or the cache length");
  const bool fixed = flags & FORGE_FIXED_CUT;
  if (fixed && T > FORGE_FIXED_CUT_MAX_T) return set_error("FORGE_FIXED_CUT is for steps of at most 16 tokens");
  PagedParams p{};
  p.fixed = fixed;
  p.q = q; p.sqb = sqb; p.sqh = sqh; p.sqt = sqt;
  p.qw = q_weight; p.eps = eps; p.flags = flags;
  p.cos = cos; p.sin = sin; p.csb = s_cos_b; p.cst = s_cos_t;
  p.k = k_cache; p.v = v_cache; p.skp = skb; p.skh = skh; p.sks = sks;
  p.page_shift = 31; p.page_mask = 0x7fffffff; p.npages = B;
  p.row_pos = row_pos; p.pos_dev = pos_dev; p.pos0 = pos0;
  p.B = B; p.T = T; p.H = H; p.K = K; p.limit = (int)limit; p.window = window; p.sinks = sinks;
  p.out = out; p.sob = sob; p.sot = sot; p.soh = soh;
  return paged_run(dtype, D, p, fixed ? max_len : max_kv_len, scale, workspace, workspace_bytes, ws_flags, (hipStream_t)stream);
}
