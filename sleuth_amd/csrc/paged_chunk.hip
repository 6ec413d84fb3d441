// Chunks of many query rows over a paged cache, or over a contiguous one with a window and first tokens:
// bf16/fp16, head dims 32 to 512, on v_mfma_f32_32x32x16, and fp32, head dims 64 to 256, on v_mfma_f32_32x32x2
// (the split kernel of paged.hip serves the rest).
//
// A block of 4 waves (8 at head dim 512) owns 128 query rows of one (batch row, KV head) -- row r is token r / G, head r % G of the
// group, so the heads of a group share each key tile they read -- and streams that row's visible key tiles through
// two LDS stages, as the causal prefill kernel does: direct loads into LDS in swizzled chunk order, S^T = K . Q^T
// with Q^T in registers, one lane per query row (two lanes share a row's keys), P^T fed to O^T = V^T . P^T straight
// from the score registers. Bound by the matrix units and the softmax's VALU work, which take turns on a SIMD: 512 tokens
// behind 15,360 at head dim 128 80 us (817 TFLOP/s, 0.59 of a large library product; 0.48 of the cycles MFMA, 0.41 VALU),
// two prompts of 8,192 506 us at head dim 256 (1,086 TFLOP/s), 562 at 128, 317 at 64.
// See prefill.hip for the operand layouts; what differs here:
//   * A wave loads RW (BN / 4, or / 8) consecutive key rows of a tile, which never straddle pages (pages are multiples of 16
//     positions), so a tile costs each wave one table entry: a scalar load, issued one tile ahead.
//   * A page id outside the pool leaves zeros in LDS and a flag for the stage; its keys are masked.
//   * With a window, the tiles that hold first tokens come before those of the window.
#include <limits.h>

#include "paged.h"
#include "prefill_tile.h"

namespace forge {

// Block shape: 128 query rows, BN keys per tile, two LDS stages of a K and a V tile. At head dim 512 a wave's
// registers hold the queries and the output of 256 channels, so two waves share 32 rows: each sums the scores of its
// half of the channels, the two exchange those sums, and each takes the products with its half of V. (One wave with all
// 512 would need 384 registers for them: the compiler spills the queries.) 16 heads, one KV head: 4,096 tokens behind
// 4,096 959 us, 860 TFLOP/s; 512 behind 4,096 113 us, 404 on the split kernel.
constexpr int chunk_halves(int D) { return D > 256 ? 2 : 1; }
template <typename T, int D> struct ChunkTile {
  static constexpr int HALVES = chunk_halves(D);
  static constexpr int WAVES = 4 * HALVES, STAGES = 2, BM = 128;
  static constexpr int THREADS = WAVES * 64;
  static constexpr int ROWB = D * (int)sizeof(T);        // bytes per key row
  static constexpr int NCH = ROWB / 16;                  // 16-byte chunks of it
  static constexpr int BN = ROWB >= 512 ? 32 : 64;
  static constexpr int TILEB = BN * ROWB;
  static constexpr int LOADS = TILEB / (WAVES * 1024);   // 16-byte loads per lane per tile
  static constexpr int LDS_BYTES = STAGES * 2 * TILEB + (HALVES == 2 ? WAVES * 4096 : 64);  // and sums, or flags
  static constexpr int QS = D / HALVES * (int)sizeof(T) / 32;  // 16-byte pieces of a lane's share of a query row
  static constexpr int BLOCKS = chunk_blocks_per_cu(sizeof(T), D);
  static_assert(BLOCKS * LDS_BYTES <= 160 * 1024, "LDS");
};
// Chunk swizzles by key row: as prefill_tile.h's in 16 bits; in fp32 a V read is 32 channels of two rows 4 apart.
template <typename T, int D> __device__ __forceinline__ int chunk_swz_k(int row) {
  constexpr int NCH = ChunkTile<T, D>::NCH, RP = NCH >= 16 ? 1 : 16 / NCH;  // key rows per 256-byte bank line
  return (row / RP) & ((NCH >= 16 ? 16 : NCH) - 1);
}
template <typename T, int D> __device__ __forceinline__ int chunk_swz_v(int row) {
  if constexpr (sizeof(T) == 2) return D == 32 ? 0 : swz_v<D>(row);
  else return ((row >> 2) & 1) << 3;
}

// Query row (b, h, t) as MFMA B operands, RMSNorm and RoPE in fp32 with one rounding: lane half hi holds the
// 16-byte pieces 2s + hi (in 16 bits the k-slots of one product, in fp32 of four). Of two waves that share the
// row, wave `half` takes half of each half of the channels, so that RoPE's pairs stay together.
template <typename T, int D>
__device__ __forceinline__ void chunk_load_q(const PagedParams& p, int b, int h, int t, int hi, int half,
                                             uint4 (&q)[ChunkTile<T, D>::QS]) {
  constexpr int S = ChunkTile<T, D>::QS, E = 16 / sizeof(T), HALVES = ChunkTile<T, D>::HALVES;
  const T* src = static_cast<const T*>(p.q) + b * p.sqb + h * p.sqh + t * p.sqt;
  const auto channel = [&](int s, int of) {  // first channel of piece s of wave `of`
    return HALVES == 1 ? (2 * s + hi) * E : (2 * (s % (S / 2)) + hi) * E + s / (S / 2) * (D / 2) + of * (D / 4);
  };
#pragma unroll
  for (int s = 0; s < S; ++s) q[s] = load16(src + channel(s, half));
  const bool norm = p.flags & FORGE_NORM_QK, rope = p.flags & FORGE_ROPE;
  if (!norm && !rope) return;
  float f[S][E];
#pragma unroll
  for (int s = 0; s < S; ++s) unpack16<T>(q[s], f[s]);
  if (norm) {
    float ss = 0.0f;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int e = 0; e < E; ++e) ss += f[s][e] * f[s][e];
    if constexpr (HALVES == 2) {  // (the other wave's channels)
#pragma unroll
      for (int s = 0; s < S; ++s) {
        float o[E];
        unpack16<T>(load16(src + channel(s, half ^ 1)), o);
#pragma unroll
        for (int e = 0; e < E; ++e) ss += o[e] * o[e];
      }
    }
    ss += __shfl_xor(ss, 32, kWave);
    const float rs = rsqrtf(ss / (float)D + p.eps);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float w[E];
      if (p.qw) {
#pragma unroll
        for (int e = 0; e < E; e += 4)
          *reinterpret_cast<float4*>(w + e) = *reinterpret_cast<const float4*>(p.qw + channel(s, half) + e);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) f[s][e] = p.qw ? f[s][e] * rs * w[e] : f[s][e] * rs;
    }
  }
  if (rope) {
    const float* cr = p.cos + b * p.csb + t * p.cst;
    const float* sr = p.sin + b * p.csb + t * p.cst;
#pragma unroll
    for (int s = 0; s < S / 2; ++s)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = channel(s, half) + e;
        const float a = f[s][e], z = f[s + S / 2][e];
        f[s][e] = a * cr[c] - z * sr[c];
        f[s + S / 2][e] = z * cr[c + D / 2] + a * sr[c + D / 2];
      }
  }
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if constexpr (sizeof(T) < 4) {
#pragma unroll
      for (int e = 0; e < E; ++e) f[s][e] = fp32_result(f[s][e]);
    }
    q[s] = pack16<T>(f[s]);
  }
}

// One step of S^T: 16 bytes of K against 16 bytes of Q^T.
template <typename T> __device__ __forceinline__ floatx16 chunk_score(uint4 a, uint4 b, floatx16 c) {
  if constexpr (sizeof(T) == 2) {
    using V8 = typename Mfma<T>::vec;
    return Mfma<T>::run(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c);
  } else {
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
  }
}

// sum + a[0] + a[1] in fp32.
template <typename T, typename V> __device__ __forceinline__ float pair_sum(V a, float sum) {
  if constexpr (__is_same(T, bf16)) return __builtin_amdgcn_fdot2_f32_bf16(a, V{(__bf16)1.0f, (__bf16)1.0f}, sum, false);
  else return __builtin_amdgcn_fdot2(a, V{(_Float16)1.0f, (_Float16)1.0f}, sum, false);
}

template <typename T, int D, bool TREE>
__global__ __launch_bounds__(256 * chunk_halves(D))
__attribute__((amdgpu_waves_per_eu(ChunkTile<T, D>::BLOCKS * chunk_halves(D))))
void paged_chunk_kernel(PagedParams p) {
  using TL = ChunkTile<T, D>;
  constexpr int BN = TL::BN, BM = TL::BM;
  constexpr int HALVES = TL::HALVES;
  constexpr int KB = BN / 32, KSTEPS = TL::QS, DB = D / HALVES / 32;
  constexpr int RW = BN / TL::WAVES;      // key rows of a tile that a wave loads
  constexpr int RL = kWave / TL::NCH;     // of which one load instruction covers RL
  static_assert(TL::STAGES == 2 && RW == RL * TL::LOADS && RW <= 16, "a wave's rows lie in one page");

  extern __shared__ __attribute__((aligned(1024))) char smem[];  // [stage][K|V][TILEB], then the flags [stage][wave]
  int* flags = reinterpret_cast<int*>(smem + TL::STAGES * 2 * TL::TILEB);
  float4* sums = reinterpret_cast<float4*>(smem + TL::STAGES * 2 * TL::TILEB);  // (two halves) [wave][4][lane]

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int n = lane & 31, hi = lane >> 5;
  const int half = HALVES == 2 ? wave >> 2 : 0;

  const BlockWork work = block_work<BM, BN, TREE>(p);
  if (work.none) return;
  const RowSpan w = work.span;
  const int b = work.b, kvh = work.kvh, rblk = work.rblk, part = work.part, begin = work.begin, end = work.end;
  const bool whole = work.parts < 2;

  // rows without a real token come out as zeros
  if (part == 0 && w.rows < rblk * BM + BM) {
    const int r0 = w.rows > rblk * BM ? w.rows : rblk * BM;
    const int r1 = rblk * BM + BM < p.rows ? rblk * BM + BM : p.rows;
    for (int x = threadIdx.x; x < (r1 - r0) * (D / 4); x += TL::THREADS)
      store_row<T>(p, b, kvh, r0 + x / (D / 4), 4 * (x % (D / 4)), make_float4(0.0f, 0.0f, 0.0f, 0.0f), 0.0f);
  }
  if (w.tiles == 0) return;

  // ---- key tiles: load i of this wave fills LDS slots (wave * LOADS + i) * 64 + lane, key rows RL * i + lane / NCH
  // of the wave's RW, in swizzled chunk order (kept offsets; in 16 bits at head dim 256, where registers are short,
  // one xor each from shared ones)
  constexpr bool KEEP = !(sizeof(T) == 2 && D >= 256);
  constexpr int ES = sizeof(T);
  const int64_t pageb = p.skp * ES;
  const int rowb = (int)p.sks * ES;
  const char* kgb = static_cast<const char*>(p.k) + kvh * p.skh * ES;
  const char* vgb = static_cast<const char*>(p.v) + kvh * p.skh * ES;
  const int ld_row = lane / TL::NCH, pch = lane % TL::NCH;
  const int wr0 = wave * RW;
  const int ld_k = (pch ^ chunk_swz_k<T, D>(ld_row)) << 4, ld_v = (pch ^ chunk_swz_v<T, D>(ld_row)) << 4;
  int kept_k[KEEP ? TL::LOADS : 1], kept_v[KEEP ? TL::LOADS : 1];
  if constexpr (KEEP) {
#pragma unroll
    for (int i = 0; i < TL::LOADS; ++i) {
      const int in = RL * i + ld_row;
      kept_k[i] = in * rowb + ((pch ^ chunk_swz_k<T, D>(wr0 + in)) << 4);
      kept_v[i] = in * rowb + ((pch ^ chunk_swz_v<T, D>(wr0 + in)) << 4);
    }
  }
  // Whose rows of a stage are zeros: each wave's flag, or, where a tile has only two groups of 16 rows (the least
  // that a page holds) and the sums take the LDS, bits that every wave looks up itself.
  int flagged[2] = {0, 0};   // what this wave's flag of each stage holds, or the stage's bits
  if (HALVES == 1 && lane < 2) flags[4 * lane + wave] = 0;
  int part_key = 0;     // first row of the wave's part of the tile that `page` belongs to, or of what stands for it
  unsigned groups = 0;  // (two halves) bit j: group j of the tile that `page` belongs to has no page
  auto page_at = [&](int i) {
    const int key0 = w.tile_key(i, BN), left = w.last - key0;
    part_key = w.group_from<RW>(key0 + wr0, key0);
    if constexpr (HALVES == 1) return p.page_of(b, part_key);
    const int p0 = p.page_of(b, key0), p1 = p.page_of(b, key0 + (left >= 16 ? 16 : 0));
    groups = (unsigned)(p0 < 0) | (unsigned)(p1 < 0) << 1;
    return part_key - key0 < 16 ? p0 : p1;
  };
  auto issue = [&](int stage, int page) {
    const unsigned kdst = lds_offset(smem + (2 * stage) * TL::TILEB + wave * TL::LOADS * 1024);
    const unsigned vdst = kdst + TL::TILEB;
    const int miss = page < 0;
    if constexpr (HALVES == 2) {
      if (stage == 0) flagged[0] = (int)groups;
      else flagged[1] = (int)groups;
    } else if (miss != flagged[stage]) {
      if (lane == 0) flags[4 * stage + wave] = miss;
      flagged[stage] = miss;
    }
    if (miss) {
      char* kd = smem + (2 * stage) * TL::TILEB + wave * TL::LOADS * 1024 + lane * 16;
#pragma unroll
      for (int x = 0; x < TL::LOADS; ++x) {
        *reinterpret_cast<uint4*>(kd + x * 1024) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(kd + TL::TILEB + x * 1024) = make_uint4(0, 0, 0, 0);
      }
      return;
    }
    const int key = part_key;
    const int64_t at = page * pageb + (int64_t)(key & p.page_mask) * rowb;
    const bool edge = w.last - key < RW - 1 || (key < w.lo && key + RW > w.se);  // it holds keys that no query sees
    const char* ks = kgb + at;
    const char* vs = vgb + at;
    int lk = ld_k, lv = ld_v;
    if constexpr (!KEEP) asm volatile("" : "+v"(lk), "+v"(lv));  // (not kept over the loop)
    if (TREE && KEEP && !edge && p.rows <= BM) {
      // A tree of one row block has its keys to itself, unless rows share pages (forks of a prompt), which is not seen here. us,
      // kept in the caches / not, 64 tokens, 16 q / 8 KV heads of 128: 32 rows of 2,000 to 16,383 keys of their own 269 / 256, of
      // a contiguous cache 283 / 270, 8 rows of up to 2,000 28.8 / 29.8; 32 rows that share 16,000 keys 283 / 296, by fours
      // 321 / 329, 4 rows 52.1 / 54.5; 64 channels and fp32 within 1 % of each other either way.
#pragma unroll
      for (int x = 0; x < (KEEP ? TL::LOADS : 0); ++x) {
        lds_dma16_once(ks, (unsigned)kept_k[x], kdst + x * 1024);
        lds_dma16_once(vs, (unsigned)kept_v[x], vdst + x * 1024);
      }
    } else if (!edge) {
#pragma unroll
      for (int x = 0; x < TL::LOADS; ++x) {
        if constexpr (KEEP) {
          lds_dma16(ks, (unsigned)kept_k[x], kdst + x * 1024);
          lds_dma16(vs, (unsigned)kept_v[x], vdst + x * 1024);
        } else {
          const int r0 = wr0 + RL * x;
          const unsigned lo = (unsigned)(ld_row * rowb);
          lds_dma16(ks + RL * x * rowb, lo + (lk ^ (chunk_swz_k<T, D>(r0) << 4)), kdst + x * 1024);
          lds_dma16(vs + RL * x * rowb, lo + (lv ^ (chunk_swz_v<T, D>(r0) << 4)), vdst + x * 1024);
        }
      }
    } else {
#pragma unroll
      for (int x = 0; x < TL::LOADS; ++x) {
        const int in = RL * x + ld_row, row = w.row_key(key, key + in) - key;
        lds_dma16(ks, (unsigned)(row * rowb + ((pch ^ chunk_swz_k<T, D>(wr0 + in)) << 4)), kdst + x * 1024);
        lds_dma16(vs, (unsigned)(row * rowb + ((pch ^ chunk_swz_v<T, D>(wr0 + in)) << 4)), vdst + x * 1024);
      }
    }
  };
  int page = page_at(begin);
  issue(0, page);
  page = page_at(begin + 1 < end ? begin + 1 : begin);

  // ---- this lane's query row; the wave's span of positions
  const int w_row = rblk * BM + (wave & 3) * 32;
  const bool wave_any = w_row < w.rows;
  const int flat = w_row + n;
  const bool valid = flat < w.rows;
  const int t = p.token(valid ? flat : w.rows - 1), h = kvh * p.G + (valid ? flat : w.rows - 1) - t * p.G;
  const int ntok = TREE ? w.last - w.base + 1 : 0;   // the tree's real tokens
  const int qpos = TREE ? tree_position(p, b, w.base, ntok, t) : w.base + t;
  TreeRow qtree{};
  if constexpr (TREE) qtree = tree_row(p, b, t);
  // positions between which the wave's queries lie; keys up to wq_all that all of them see
  const int wq_lo = TREE ? w.base : w.base + p.token(w_row), wq_all = TREE ? w.first : wq_lo;
  const int wq_hi = TREE ? w.last : w.base + p.token(w_row + 31 < w.rows ? w_row + 31 : w.rows - 1);
  uint4 qreg[KSTEPS];
  chunk_load_q<T, D>(p, b, h, t, hi, half, qreg);

  // LDS read offsets of a lane within a stage's K and V tiles: in 16 bits prefill.hip's; in fp32 a V operand is channel
  // 32d + n of key 8i + 4hi + j, whose swizzle is the lane's own bit hi
  const unsigned k_rd = n * TL::ROWB + ((hi ^ chunk_swz_k<T, D>(n)) << 4);
  unsigned v_rd;
  if constexpr (ES == 2) {
    const int g = lane >> 4, kq = (lane >> 2) & 3, qq = lane & 3;
    const int v_row = 4 * (g >> 1) + kq;
    v_rd = v_row * TL::ROWB + (((2 * (g & 1) + (qq >> 1)) ^ chunk_swz_v<T, D>(v_row)) << 4) + 8 * (qq & 1);
  } else {
    v_rd = 4 * hi * TL::ROWB + (((n >> 2) ^ chunk_swz_v<T, D>(4 * hi)) << 4) + 4 * (n & 3);
  }
  const unsigned lds0 = lds_offset(smem);

  floatx16 oacc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int x = 0; x < 16; ++x) oacc[d][x] = 0.0f;
  float m_run = kNegInf, l_run = 0.0f;
  const float c = p.scale_log2;

  int odd = 0;   // (trees) values were taken out of the wave's rows of a tile
  const auto whole_tile = [&](int key0) {
    return key0 + BN - 1 <= w.first && (p.window <= 0 || w.last - key0 < p.window || key0 + BN <= p.sinks);
  };
  for (int it = begin; it < end; ++it) {
    const int stage = (it - begin) & 1;
    wait_vm<0>();
    if constexpr (TREE) {   // (paged.h; each wave looks at the rows that it loaded, before the others read them)
      if (!whole_tile(w.tile_key(it, BN))) {
        char* mine = smem + (2 * stage + 1) * TL::TILEB + wave * TL::LOADS * 1024 + lane * 16;
        OddValues<T> values;
#pragma unroll
        for (int x = 0; x < TL::LOADS; ++x) {
          const uint4 v = load16(mine + x * 1024);
          values.add(v.x), values.add(v.y), values.add(v.z), values.add(v.w);
        }
        if (__any(values.bad())) {
          odd = 1;
#pragma unroll 1
          for (int x = 0; x < 4 * TL::LOADS; ++x) {
            unsigned* at = reinterpret_cast<unsigned*>(mine + (x >> 2) * 1024) + (x & 3);
            *at = finite_dword<T>(*at);
          }
        }
      }
    }
    __syncthreads();  // tile `it` is in LDS for every wave; the other stage is free
    if (it + 1 < end) {
      issue(stage ^ 1, page);
      page = page_at(it + 2 < end ? it + 2 : it + 1);
    }
    const int key0 = w.tile_key(it, BN);
    const bool needed = wave_any && key0 <= wq_hi &&
                        (p.window <= 0 || key0 + BN - 1 > wq_lo - p.window || key0 < p.sinks);
    if (HALVES == 1 && !needed) continue;
    unsigned bad = 0;
    if constexpr (HALVES == 2) bad = (unsigned)(stage ? flagged[1] : flagged[0]);
    else if (p.table) bad = (unsigned)__ballot(flags[4 * stage + (lane & 3)] != 0) & 15u;
    const bool full = bad == 0 && key0 + BN - 1 <= wq_all &&
                      (p.window <= 0 || wq_hi - key0 < p.window || key0 + BN <= p.sinks);

    const unsigned kl = lds0 + (2 * stage) * TL::TILEB + k_rd + 256 * half;
    const unsigned vl = lds0 + (2 * stage + 1) * TL::TILEB + v_rd + 512 * half;

    // S^T = K . Q^T, K operands read two steps ahead (pinned: left alone each step waits for its reads)
    floatx16 sacc[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int x = 0; x < 16; ++x) sacc[kb][x] = 0.0f;
    if (HALVES == 1 || needed) {
      auto kread = [&](int kb, int st) {
        typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
        return __builtin_bit_cast(uint4, *(__attribute__((address_space(3))) const u32x4*)((kl ^ (32 * (st & 7))) +
                                                                                           256 * HALVES * (st >> 3) + kb * 32 * TL::ROWB));
      };
      uint4 a0[KB], a1[KB], a2[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) a0[kb] = kread(kb, 0);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) a1[kb] = kread(kb, 1);
      __builtin_amdgcn_sched_group_barrier(0x100, 2 * KB, 0);
#pragma unroll
      for (int st = 0; st < KSTEPS; ++st) {
        if (st + 2 < KSTEPS) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) a2[kb] = kread(kb, st + 2);
          __builtin_amdgcn_sched_group_barrier(0x100, KB, 0);
        }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) sacc[kb] = chunk_score<T>(a0[kb], qreg[st], sacc[kb]);
        __builtin_amdgcn_sched_group_barrier(0x008, KB * (ES == 4 ? 4 : 1), 0);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          a0[kb] = a1[kb];
          a1[kb] = a2[kb];
        }
      }
    }
    if constexpr (HALVES == 2) {
      // the sums of the other half of the channels (every wave meets here, whatever it needs)
      float4* mine = sums + wave * 256 + lane;
      if (needed) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mine[64 * i] = make_float4(sacc[0][4 * i], sacc[0][4 * i + 1], sacc[0][4 * i + 2], sacc[0][4 * i + 3]);
      }
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // (LDS only: the next tile's loads go on)
      if (!needed) continue;
      const float4* other = sums + (wave ^ 4) * 256 + lane;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 z = other[64 * i];
        sacc[0][4 * i] += z.x;
        sacc[0][4 * i + 1] += z.y;
        sacc[0][4 * i + 2] += z.z;
        sacc[0][4 * i + 3] += z.w;
      }
    }

    // Element (kb, x) of this lane is key key0 + 4hi + 32kb + ce, ce = 8(x/4) + x%4. What its query sees of the 32 from
    // there on is a mask of bits: the run from the window's first key to the query, and the first tokens (up to the
    // query). An element then takes two instructions, where compares took three and a branch each when written with
    // && and || (two prompts of 4,093 tokens, window 1,024, head dim 64: 55 us with the branches, 46 with compares, 45).
    if (!full) {
      const int base = key0 + 4 * hi;
      const int top = (qpos < w.last ? qpos : w.last) - base + 1;   // past the last visible key
      const int lo = (p.window > 0 ? qpos - p.window + 1 : 0) - base;
      const int first = p.sinks - base < top ? p.sinks - base : top;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        unsigned see = (low_bits(top - 32 * kb) & ~low_bits(lo - 32 * kb)) | low_bits(first - 32 * kb);
        if constexpr (TREE) see = tree_sees(p, b, w.base, ntok, qtree, qpos, base + 32 * kb);
        if (bad) {
#pragma unroll
          for (int x = 0; x < 16; x += 4)
            if (bad >> ((32 * kb + 2 * x) / (HALVES == 2 ? 16 : RW)) & 1) see &= ~(0xffu << (2 * x));
        }
#pragma unroll
        for (int x = 0; x < 16; ++x) sacc[kb][x] = masked(sacc[kb][x], see, 8 * (x >> 2) + (x & 3));
      }
    }

    // online softmax in base 2, the scale in the exponent's fma; the maximum moves when a score passes it by 2^8. In 16
    // bits the sum takes the rounded weights, two to an instruction, as the products do (prompts of 8,192 tokens at head
    // dim 256: 549 -> 506 us; a ragged batch of chunks 227 -> 222; at head dim 64 the same)
    float mx[2] = {sacc[0][0], sacc[0][2]};
#pragma unroll
    for (int x = 0; x < 16 * KB; ++x) mx[x >> 1 & 1] = fmaxf(mx[x >> 1 & 1], sacc[x >> 4][x & 15]);
    const float mxc = max_xor32(fmaxf(mx[0], mx[1])) * c;
    if (mxc > m_run + kLazyLog2) {
      const float alpha = m_run == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m_run - mxc);
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int x = 0; x < 16; ++x) oacc[d][x] *= alpha;
      m_run = mxc;
    }
    const float neg_m = m_run == kNegInf ? 0.0f : -m_run;
    float rs[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const float pv = __builtin_amdgcn_exp2f(fmaf(sacc[kb][x], c, neg_m));
        sacc[kb][x] = pv;
        if constexpr (ES == 4) rs[x & 3] += pv;
      }
    if constexpr (ES == 4) l_run += (rs[0] + rs[1]) + (rs[2] + rs[3]);

    // O^T += V^T . P^T. In 16 bits the weights are rounded to the type once, as the prefill kernels' are: as two numbers
    // of it, like the split kernel's, they would cost a second product, and products are half of this kernel's time. us,
    // once / as two, and the outputs' 2-norm error against 64 bits: 512 tokens behind 15,360 80 / 109, 0.0023 / 0.0017 (the
    // last is the output's own rounding); a ragged batch of chunks 225 / 293; fp16 prompts of 4,093 43 / 59, 0.00026 /
    // 0.00021; 8,192 tokens with a window of 2,048 144 / 201, 0.0022 / 0.0017.
    if constexpr (ES == 4) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const unsigned row = (32 * kb + 8 * (x >> 2) + (x & 3)) * TL::ROWB;
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            const float a = *(__attribute__((address_space(3))) const float*)((vl ^ (128 * (d & 1))) + 256 * (d >> 1) + row);
            oacc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, sacc[kb][x], oacc[d], 0, 0, 0);
          }
        }
    } else {
      using V8 = typename Mfma<T>::vec;
#pragma unroll
      for (int hf = 0; hf < BN / 16; ++hf) {
        const int kb = hf >> 1, half = hf & 1;
        V8 pb;
#pragma unroll
        for (int e = 0; e < 8; ++e) pb[e] = from_f32<T>(sacc[kb][8 * half + e]);
        rs[0] = pair_sum<T>(__builtin_shufflevector(pb, pb, 0, 1), rs[0]);
        rs[1] = pair_sum<T>(__builtin_shufflevector(pb, pb, 2, 3), rs[1]);
        rs[2] = pair_sum<T>(__builtin_shufflevector(pb, pb, 4, 5), rs[2]);
        rs[3] = pair_sum<T>(__builtin_shufflevector(pb, pb, 6, 7), rs[3]);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const unsigned va = (vl ^ (64 * (d & 3))) + 256 * (d >> 2) + 16 * hf * TL::ROWB;
          const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)va);
          const i16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) i16x4*)(va + 8 * TL::ROWB));
          typedef short i16x8 __attribute__((ext_vector_type(8)));
          const i16x8 av = __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
          oacc[d] = Mfma<T>::run(__builtin_bit_cast(V8, av), pb, oacc[d]);
        }
      }
      l_run += (rs[0] + rs[1]) + (rs[2] + rs[3]);
    }
  }

  l_run += __shfl_xor(l_run, 32, kWave);
  if constexpr (TREE) {   // whether any wave took values out (the tiles' LDS is free)
    int* all = reinterpret_cast<int*>(smem);
    __syncthreads();
    if (lane == 0) all[wave] = odd;
    __syncthreads();
    odd = 0;
#pragma unroll
    for (int y = 0; y < TL::WAVES; ++y) odd |= all[y];
  }
  if (!valid) return;
  if constexpr (TREE) {
#pragma unroll 1
    for (int y = begin; odd && y < end; ++y) {   // those, for the rows that see them
      const int key0 = w.tile_key(y, BN);
      if (whole_tile(key0)) continue;
#pragma unroll 1
      for (int key = key0; key < key0 + BN && key <= w.last; ++key) {
        const int page = p.page_of(b, key);
        if (page < 0 || !(tree_sees(p, b, w.base, ntok, qtree, qpos, key) & 1)) continue;
        const T* src = reinterpret_cast<const T*>(vgb + page * pageb + (int64_t)(key & p.page_mask) * rowb);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const T v = src[half * (D / 2) + d * 32 + 8 * (x >> 2) + 4 * hi + (x & 3)];
            if (not_finite(v)) oacc[d][x] += to_f32<T>(v);
          }
      }
    }
  }
  if (!whole) {
    const int64_t slot = (int64_t)work.slot * BM + (wave & 3) * 32 + n;
    float* po = p.ws_o + slot * D + half * (D / 2) + 4 * hi;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<float4*>(po + d * 32 + 8 * i) =
            make_float4(oacc[d][4 * i], oacc[d][4 * i + 1], oacc[d][4 * i + 2], oacc[d][4 * i + 3]);
    if (hi == 0 && half == 0) p.ws_ml[slot] = make_float2(m_run, l_run);
    return;
  }
  const float inv = l_run > 0.0f ? 1.0f / l_run : 0.0f;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      store_row<T>(p, b, kvh, flat, half * (D / 2) + d * 32 + 8 * i + 4 * hi,
                   make_float4(oacc[d][4 * i], oacc[d][4 * i + 1], oacc[d][4 * i + 2], oacc[d][4 * i + 3]), inv);
}

// Plans a call whose rows have different lengths, which only the device knows: one block, a thread per row
// block. Each row block's tiles are cut into equal parts of at most `per` tiles, the smallest `per` of 16 tried
// (wave w tries one, over the row blocks in turn) with which all parts are resident at once; the parts go out
// longest first (64 classes of length), so that a CU that got a long one gets a short one beside it.
constexpr int kPlanThreads = 1024;
template <int BM, int KT, bool TREE> __global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PagedParams p, PagedItem* items,
                                                                                        int4* pairs, int nitems) {
  __shared__ int tiles[kPlanPairs];
  __shared__ int wave_of[16], wave_tot[16], cls[64], pick;
  const int nrb = (p.rows + BM - 1) / BM, n = p.B * nrb;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  if (threadIdx.x < 64) cls[threadIdx.x] = 0;
  int sum = 0;
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    int base, rows;
    row_extent(p, i / nrb, base, rows);
    tiles[i] = make_span<TREE>(p, base, rows, i % nrb * BM, BM, KT).tiles;
    sum += tiles[i];
  }
  for (int d = 1; d < kWave; d <<= 1) sum += __shfl_xor(sum, d, kWave);
  if (lane == 0) wave_tot[wave] = sum;
  __syncthreads();
  int total = 0;
  for (int w = 0; w < 16; ++w) total += wave_tot[w];
  // equal shares of all slots, and up to 2.5 times that; fewer than 8 tiles a part cost more than they even out
  const int room = p.slots / p.K;
  const int least = max(8, (total + room - 1) / room);
  auto per_of = [&](int w) { return w == 15 ? 1 << 30 : least + (int)((int64_t)least * w / 10); };
  int per;
  if constexpr (!TREE) {
    const int tried = per_of(wave);
    int parts = 0;
    for (int i = lane; i < n; i += kWave) parts += (tiles[i] + tried - 1) / tried;
    for (int d = 1; d < kWave; d <<= 1) parts += __shfl_xor(parts, d, kWave);
    if (lane == 0) wave_of[wave] = parts;
    __syncthreads();
    if (threadIdx.x == 0) {
      int w = 0;
      while (w < 15 && wave_of[w] > room) ++w;
      pick = w;
    }
    __syncthreads();
    per = per_of(pick);
  } else {
    // Few rows of different lengths leave much of one round empty (32 of up to 16,383 keys: 62 parts, the longest 93 tiles
    // where 69 would be an equal share), and two rounds of half as long parts less: for each the least of 32 steps of 5 %
    // that fits, and the one whose longest parts take less time, with what a part costs by itself, three tiles' time
    // (there 238 us in one round, 216 in two, 232 in three).
    const int half = max(8, (total + 2 * room - 1) / (2 * room));
    __shared__ int best[2];
    if (threadIdx.x < 2) best[threadIdx.x] = 1 << 30;
    __syncthreads();
    const int from = wave < 8 ? least : half, fits = (wave < 8 ? 1 : 2) * room;   // (a wave tries four)
    int tried[4], parts[4] = {0, 0, 0, 0};
#pragma unroll
    for (int x = 0; x < 4; ++x) tried[x] = from + (int)((int64_t)from * (4 * (wave & 7) + x) / 20);
    for (int i = lane; i < n; i += kWave)
#pragma unroll
      for (int x = 0; x < 4; ++x) parts[x] += (tiles[i] + tried[x] - 1) / tried[x];
    for (int d = 1; d < kWave; d <<= 1)
#pragma unroll
      for (int x = 0; x < 4; ++x) parts[x] += __shfl_xor(parts[x], d, kWave);
    if (lane == 0)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (parts[x] <= fits) atomicMin(&best[wave >> 3], tried[x]);
    __syncthreads();
    per = best[1] < 1 << 30 && 2 * (int64_t)best[1] + 6 < best[0] + 3 ? best[1] : best[0];
  }
  // lengths relative to the longest part: class 0 is the longest; a row block without a real query is one part
  // of no tiles, which writes its zeros
  auto parts_of = [&](int i) { return tiles[i] > 0 ? (tiles[i] + per - 1) / per : 1; };
  auto class_of = [&](int i, int parts) {
    const int len = tiles[i] / parts;
    const int scale = per < (1 << 30) ? per : p.limit / KT + 1;
    return 63 - (int)min((int64_t)63, (int64_t)len * 64 / (scale + 1));
  };
  int mine = 0;
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int parts = parts_of(i);
    mine += parts;
    atomicAdd(&cls[class_of(i, parts)], parts);
  }
  // slots: row blocks in the order of the threads that hold them
  int before = mine;
  for (int d = 1; d < kWave; d <<= 1) {
    const int y = __shfl_up(before, d, kWave);
    if (lane >= d) before += y;
  }
  if (lane == kWave - 1) wave_tot[wave] = before;
  before -= mine;
  __syncthreads();
  for (int w = 0; w < wave; ++w) before += wave_tot[w];
  if (threadIdx.x == 0) {
    int at = 0;
    for (int c = 0; c < 64; ++c) {
      const int k = cls[c];
      cls[c] = at;
      at += k;
    }
    pick = at;  // all parts
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int parts = parts_of(i);
    int base, rows;
    row_extent(p, i / nrb, base, rows);
    pairs[i] = make_int4(before, parts, rows, 0);
    const int at = atomicAdd(&cls[class_of(i, parts)], parts);
    for (int j = 0; j < parts; ++j) items[at + j] = PagedItem{i, j, parts, before + j};
    before += parts;
  }
  for (int i = pick + threadIdx.x; i < nitems; i += kPlanThreads) items[i] = PagedItem{0, 0, -1, 0};
}

template <typename T, int D, bool TREE> static int launch_chunk_d(PagedParams p, const PagedPlan& plan, hipStream_t s) {
  using TL = ChunkTile<T, D>;
  static std::atomic<uint64_t> done{0};
  if (const int st = reserve_lds(reinterpret_cast<const void*>(&paged_chunk_kernel<T, D, TREE>), TL::LDS_BYTES, done)) return st;
  const int nrb = (p.rows + TL::BM - 1) / TL::BM;
  if (nrb > 65535) return set_error("forge_attn_paged: too many query rows");
  dim3 grid((unsigned)(p.B * p.K), p.nparts, nrb);
  if (plan.planned) {
    grid = dim3((unsigned)(plan.nitems * p.K));
    hipLaunchKernelGGL((paged_plan_kernel<TL::BM, TL::BN, TREE>), dim3(1), dim3(kPlanThreads), 0, s, p,
                       const_cast<PagedItem*>(p.items), const_cast<int4*>(p.pairs), plan.nitems);
    const int st = check_launch();
    if (st) return st;
  }
  hipLaunchKernelGGL((paged_chunk_kernel<T, D, TREE>), grid, dim3(TL::THREADS), TL::LDS_BYTES, s, p);
  const int st = check_launch();
  if (st) return st;
  if (plan.planned) return launch_paged_combine<T, D, TL::BM, TL::BN, true, TREE>(p, s);
  return p.nparts > 1 ? launch_paged_combine<T, D, TL::BM, TL::BN, false, TREE>(p, s) : 0;
}

template <typename T, bool TREE> int launch_paged_chunk(const PagedParams& p, const PagedPlan& plan, int D, hipStream_t s) {
  switch (D) {
    case 32:
      if constexpr (sizeof(T) == 2) return launch_chunk_d<T, 32, TREE>(p, plan, s);
      break;
    case 64: return launch_chunk_d<T, 64, TREE>(p, plan, s);
    case 128: return launch_chunk_d<T, 128, TREE>(p, plan, s);
    case 256: return launch_chunk_d<T, 256, TREE>(p, plan, s);
    case 512:
      if constexpr (sizeof(T) == 2) return launch_chunk_d<T, 512, TREE>(p, plan, s);
  }
  return set_error("forge_attn_paged: unsupported head dim");
}
#if FORGE_PAGED_PART == 1
template int launch_paged_chunk<bf16, false>(const PagedParams&, const PagedPlan&, int, hipStream_t);
#elif FORGE_PAGED_PART == 2
template int launch_paged_chunk<f16, false>(const PagedParams&, const PagedPlan&, int, hipStream_t);
#elif FORGE_PAGED_PART == 3
template int launch_paged_chunk<float, false>(const PagedParams&, const PagedPlan&, int, hipStream_t);
#elif FORGE_PAGED_PART == 4
template int launch_paged_chunk<bf16, true>(const PagedParams&, const PagedPlan&, int, hipStream_t);
#elif FORGE_PAGED_PART == 5
template int launch_paged_chunk<f16, true>(const PagedParams&, const PagedPlan&, int, hipStream_t);
#elif FORGE_PAGED_PART == 6
template int launch_paged_chunk<float, true>(const PagedParams&, const PagedPlan&, int, hipStream_t);
#endif

}  // namespace forge
