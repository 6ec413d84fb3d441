// Attention of new tokens over a paged cache, and over a contiguous one with a sliding window whose
// first tokens stay visible (forge_attn_paged, forge_attn_sinks).
//
// Row b's new token t sits at position p = base_b + t and sees key s iff
//   s <= p  and  (no window, or s > p - window, or s < sinks),
// so a row's visible keys are one run, or two with a window: the first `sinks` keys and the window.
// out = sum_s w_s v_s / sum_s w_s,  w_s = exp(scale q.k_s - m), m the running maximum: one pass over
// the keys, statistics and sums in fp32. A contiguous cache is a paged one with one page per batch row.
//
// The G * T query rows (token, head of the group) of one KV head share its keys: row r is token r / G,
// head r % G of the group. Both kernels below take blocks of such rows, so a key row loaded once serves
// every head of the group, and a step of few tokens still fills matrix-core tiles.
#include <limits.h>

#include "paged.h"

namespace forge {

// ---------------------------------------------------------------- matrix-core steps
// 16x16 tiles. Lane (n, g) = (lane % 16, lane / 16) gives row n of A and column n of B, k-slots of
// group g, and receives column n, rows 4g .. 4g+3 of C. Scores are computed transposed
// (S^T = K . Q^T: A = 16 keys, B = 16 query rows), so a lane owns ONE query row and four keys of each
// key block: the row maximum takes two exchanges (lanes 16 and 32 away), the row sum none until the
// end, and the weights are already where the second product O^T = V^T . P^T wants its B operand.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Mma;
template <> struct Mma<bf16> {
  static __device__ __forceinline__ f32x4 k32(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 k16(i16x4 a, i16x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
  }
};
template <> struct Mma<f16> {
  static __device__ __forceinline__ f32x4 k32(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 k16(i16x4 a, i16x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
  }
};
template <> struct Mma<float> {
  // 16 bytes are four channels: four products of one channel per group
  static __device__ __forceinline__ f32x4 k32(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
    return c;
  }
};

// max / sum over lanes l, l ^ 16, l ^ 32, l ^ 48 (the four groups of one query row). Swapping x with
// itself returns both halves of each pair, so both lanes combine the same two values.
template <bool MAX> __device__ __forceinline__ float over_groups(float x) {
  unsigned u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const unsigned a0 = a[0], a1 = a[1];
  x = MAX ? fmaxf(__uint_as_float(a0), __uint_as_float(a1)) : __uint_as_float(a0) + __uint_as_float(a1);
  u = __float_as_uint(x);
  const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const unsigned b0 = b[0], b1 = b[1];
  return MAX ? fmaxf(__uint_as_float(b0), __uint_as_float(b1)) : __uint_as_float(b0) + __uint_as_float(b1);
}

// ---------------------------------------------------------------- split kernel
// A block of four waves takes ROWS = 16 RB query rows of one (batch row, KV head) and a part of their
// key tiles. Each wave streams tiles of its own (tile i goes to wave i % 4) through registers into LDS
// that only it uses, so no wave waits for another until the end: the tile in registers is the prefetch
// of the next one. The waves' (m, l, O) meet in LDS once, at the end.
//
// Bound by the keys' bytes where there are many, 710 us (6.5 TB/s) for one token of 64 rows of 1,024 to 32,767 keys, 8 KV
// heads of 128 in bf16, as fast as a streaming read; by latency where there are few, 7 us for one row of 212 keys:
// position, page, keys, a tile or two a wave and the merge follow one another. 16 rows a block leave the matrix units
// half empty at a step, but nothing waits for them; a second register tile in flight per wave gained nothing.
template <typename T, int D, int RB> struct StepTile {
  static_assert(16 * RB <= step_rows_most(sizeof(T), D), "registers");
  static constexpr int ROWB = D * (int)sizeof(T);        // bytes of a key row
  static constexpr int NCH = ROWB / 16;                  // 16-byte chunks of it
  static constexpr int KT = step_keys(sizeof(T), D, 16 * RB);  // keys per wave tile
  static constexpr int KB = KT / 16;                     // 16-key blocks
  static constexpr int RPI = 64 / NCH;                   // key rows per wave load instruction
  static constexpr int NL = KT / RPI;                    // load instructions per K (or V) tile
  static constexpr int TILEB = KT * ROWB;
  static constexpr int RP = ROWB >= 256 ? 1 : 256 / ROWB;  // key rows per 256-byte bank line
};

// Chunk swizzles by key row. K operands: 16 rows of one chunk at a time, so the chunk index turns with
// the row. V operands: in 16 bits 16 rows of two neighbouring chunks (32 bytes), in fp32 four rows 4
// apart of four chunks (64 bytes).
template <typename T, int D> __device__ __forceinline__ int step_swz_k(int row) {
  using TL = StepTile<T, D, 1>;
  return (row / TL::RP) & ((TL::NCH < 16 ? TL::NCH : 16) - 1);
}
template <typename T, int D> __device__ __forceinline__ int step_swz_v(int row) {
  using TL = StepTile<T, D, 1>;
  if constexpr (sizeof(T) == 4) return ((row >> 2) << 2) & ((TL::NCH < 16 ? TL::NCH : 16) - 1);
  else return ((row / TL::RP) << 1) & ((TL::NCH < 16 ? TL::NCH : 16) - 1);
}

// Query row `row` (a row that exists) as B operands: chunk 4s + g in q[s], with RMSNorm and RoPE in
// fp32 and one rounding.
template <typename T, int D>
__device__ __forceinline__ void step_load_q(const PagedParams& p, int b, int kvh, int row, int g,
                                            u32x4 (&q)[StepTile<T, D, 1>::NCH / 4]) {
  constexpr int NCH = StepTile<T, D, 1>::NCH, S = NCH / 4, E = 16 / sizeof(T);
  const int t = p.token(row), h = kvh * p.G + row - t * p.G;
  const T* src = static_cast<const T*>(p.q) + b * p.sqb + h * p.sqh + t * p.sqt;
#pragma unroll
  for (int s = 0; s < S; ++s) q[s] = *reinterpret_cast<const u32x4*>(src + (4 * s + g) * E);
  const bool norm = p.flags & FORGE_NORM_QK, rope = p.flags & FORGE_ROPE;
  if (!norm && !rope) return;
  float f[S][E];
#pragma unroll
  for (int s = 0; s < S; ++s) unpack16<T>(__builtin_bit_cast(uint4, q[s]), f[s]);
  if (norm) {
    float ss = 0.0f;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int e = 0; e < E; ++e) ss += f[s][e] * f[s][e];
    const float rs = rsqrtf(over_groups<false>(ss) / (float)D + p.eps);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float w[E];
      if (p.qw) {
#pragma unroll
        for (int e = 0; e < E; e += 4) *reinterpret_cast<float4*>(w + e) = *reinterpret_cast<const float4*>(p.qw + (4 * s + g) * E + e);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) f[s][e] = p.qw ? f[s][e] * rs * w[e] : f[s][e] * rs;
    }
  }
  if (rope) {
    const float* cr = p.cos + b * p.csb + t * p.cst;
    const float* sr = p.sin + b * p.csb + t * p.cst;
    if constexpr (S >= 2) {  // the pair (c, c + D/2) is in one lane
#pragma unroll
      for (int s = 0; s < S / 2; ++s)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int c = (4 * s + g) * E + e;
          const float a = f[s][e], z = f[s + S / 2][e];
          f[s][e] = a * cr[c] - z * sr[c];
          f[s + S / 2][e] = z * cr[c + D / 2] + a * sr[c + D / 2];
        }
    } else {  // 16 bits, head dim 32: the partner channel is two groups away
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = g * E + e;
        const float o = __shfl_xor(f[0][e], 32, kWave);
        f[0][e] = f[0][e] * cr[c] + (g < 2 ? -o : o) * sr[c];
      }
    }
  }
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if constexpr (sizeof(T) < 4) {
#pragma unroll
      for (int e = 0; e < E; ++e) f[s][e] = fp32_result(f[s][e]);
    }
    q[s] = __builtin_bit_cast(u32x4, pack16<T>(f[s]));
  }
}

template <typename T, int D, int RB> struct StepLds {
  using TL = StepTile<T, D, RB>;
  static constexpr int ROWS = 16 * RB;
  static constexpr int OUT = ROWS * D * 4;                                // a wave's output in fp32
  static constexpr int WAVE = 2 * TL::TILEB > OUT ? 2 * TL::TILEB : OUT;  // a wave's K and V tile, later its output
  // The query operands are read from LDS in each tile where the output and the tile in flight take the
  // registers: a reload of a spilled one would wait for the tile loads it queues behind.
  static constexpr bool Q_LDS = TL::ROWB * RB >= 1024;
  static constexpr int ML = 5 * ROWS * 8;                                 // (m, l) of every wave's rows, and of all
  static constexpr int Q_OFF = 4 * WAVE + ML;
  static constexpr int BYTES = Q_OFF + (Q_LDS ? ROWS * TL::ROWB : 0);
  static constexpr int BLOCKS = step_blocks_per_cu(sizeof(T), D, ROWS);
  static_assert(BLOCKS * BYTES <= 160 * 1024, "LDS");
};

// How a call's keys are cut and seen: freely, at places fixed in the cache, or freely by the rows of a tree.
enum StepMode { kFree, kFixed, kTree };

template <typename T, int D, int RB, StepMode MODE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(StepLds<T, D, RB>::BLOCKS >= 2 ? 2 : 1)))
void paged_step_kernel(PagedParams p) {
  using TL = StepTile<T, D, RB>;
  using LD = StepLds<T, D, RB>;
  constexpr int KT = TL::KT, KB = TL::KB, NL = TL::NL, S = TL::NCH / 4, DB = D / 16, ROWS = LD::ROWS;
  constexpr int GROUPS = KT / 16;
  constexpr bool FIXED = MODE == kFixed, TREE = MODE == kTree;

  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int n = lane & 15, g = lane >> 4;

  const BlockWork work = block_work<ROWS, KT, TREE>(p);
  if (work.none) return;
  const RowSpan w = work.span;
  const int b = work.b, kvh = work.kvh, rblk = work.rblk;
  const bool whole = work.parts < 2;

  // ---- key tiles of this wave: begin + wave, + 4, ...; with a fixed cut those whose number in the cache is the wave's
  // own below 4 nparts, modulo 4 nparts: tiles of the first tokens, then, `hop` behind the first one of the window, those
  const int own = 4 * work.part + wave, step = FIXED ? 4 * p.nparts : 4;
  const int sink_end = FIXED ? w.sink_tiles : 0;
  int hop = FIXED ? (own - w.main_tile) % step : 0;
  hop += hop < 0 ? step : 0;
  const auto next = [&](int i) { return FIXED && i < sink_end && i + step >= sink_end ? sink_end + hop : i + step; };
  u32x4 kr[NL], vr[NL];
  const int lrow = lane / TL::NCH, lch = lane % TL::NCH;
  const char* kb0 = static_cast<const char*>(p.k) + kvh * p.skh * (int64_t)sizeof(T);
  const char* vb0 = static_cast<const char*>(p.v) + kvh * p.skh * (int64_t)sizeof(T);
  const int64_t pageb = p.skp * (int64_t)sizeof(T);
  const int rowb = (int)(p.sks * (int64_t)sizeof(T));
  unsigned bad = 0;  // bit i: 16-key group i of the tile in kr/vr lies in no page of the pool
  auto load = [&](int i) {
    const int key0 = w.tile_key(i, KT);
    const bool edge = w.last - key0 < KT - 1 || key0 < w.lo;  // rows of it stand for keys that no query sees
    unsigned miss = 0;
    int from[GROUPS];
    int64_t base[GROUPS];
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) {
      from[j] = edge ? w.group_from<16>(key0 + 16 * j, key0) : key0 + 16 * j;
      const int page = p.page_of(b, from[j]);
      if (page < 0) miss |= 1u << j;
      base[j] = page * pageb + (int64_t)(from[j] & p.page_mask) * rowb;
    }
    if (miss == 0) {
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const int in = j * TL::RPI / 16;   // the load's group
        int row = j * TL::RPI % 16 + lrow;
        if (edge) row = w.row_key(from[in], from[in] + row) - from[in];
        const unsigned off = (unsigned)(row * rowb + lch * 16);
        kr[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kb0 + base[in] + off));
        vr[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(vb0 + base[in] + off));
      }
    } else {
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const int in = j * TL::RPI / 16;
        const int row = w.row_key(from[in], from[in] + j * TL::RPI % 16 + lrow) - from[in];
        const unsigned off = (unsigned)(row * rowb + lch * 16);
        kr[j] = u32x4{0, 0, 0, 0};
        vr[j] = u32x4{0, 0, 0, 0};
        if (!(miss >> in & 1)) {
          kr[j] = *reinterpret_cast<const u32x4*>(kb0 + base[in] + off);
          vr[j] = *reinterpret_cast<const u32x4*>(vb0 + base[in] + off);
        }
      }
    }
    bad = miss;
  };
  int i = !FIXED ? work.begin + wave : own < sink_end ? own : sink_end + hop;
  const int end = FIXED ? w.tiles : work.end;
  if (i < end) load(i);

  // ---- query rows, as B operands; rows behind the row's last one stand for that one (never written)
  u32x4 q[LD::Q_LDS ? 1 : RB][S];
  int qpos[RB];
  TreeRow qtree[TREE ? RB : 1];
  const int ntok = TREE ? w.last - w.base + 1 : 0;   // the tree's real tokens
  char* ql = smem + LD::Q_OFF;  // [ROWS][chunks turned with the row]
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int row = rblk * ROWS + 16 * r + n;
    const int at = row < w.rows ? row : w.rows - 1;
    qpos[r] = w.base + p.token(at);
    if constexpr (TREE) {
      qtree[r] = tree_row(p, b, w.rows > 0 ? p.token(at) : 0);
      qpos[r] = w.rows > 0 ? tree_position(p, b, w.base, ntok, p.token(at)) : w.base;
    }
    if constexpr (LD::Q_LDS) {
      if (r % 4 == wave && w.rows > 0) {
        step_load_q<T, D>(p, b, kvh, at, g, q[0]);
#pragma unroll
        for (int st = 0; st < S; ++st)
          *reinterpret_cast<u32x4*>(ql + (16 * r + n) * TL::ROWB + (((4 * st + g) ^ n) << 4)) = q[0][st];
      }
    } else if (w.rows > 0) {
      step_load_q<T, D>(p, b, kvh, at, g, q[r]);
    }
  }
  if constexpr (LD::Q_LDS) __syncthreads();

  f32x4 o[RB][DB];
  float m[RB], l[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    m[r] = kNegInf;
    l[r] = 0.0f;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[r][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const float c = p.scale_log2;
  char* kt = smem + wave * LD::WAVE;
  char* vt = kt + TL::TILEB;

  int odd_from = -1, odd_to = -2;   // (trees) the wave's tiles among which are those with values taken out
  for (; i < end; i = next(i)) {
    const int key0 = w.tile_key(i, KT);
    // whether every row of the block sees the tile whole
    const bool whole_tile = key0 + KT - 1 <= w.first && (p.window <= 0 || key0 > w.last - p.window || key0 + KT <= p.sinks);
    if constexpr (TREE) {
      if (!whole_tile) {   // (paged.h)
        OddValues<T> odd;
#pragma unroll
        for (int j = 0; j < NL; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) odd.add(vr[j][e]);
        if (__any(odd.bad())) {
          odd_from = odd_from < 0 ? i : odd_from;
          odd_to = i;
#pragma unroll
          for (int j = 0; j < NL; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) vr[j][e] = finite_dword<T>(vr[j][e]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NL; ++j) {
      const int row = j * TL::RPI + lrow;
      *reinterpret_cast<u32x4*>(kt + row * TL::ROWB + ((lch ^ step_swz_k<T, D>(row)) << 4)) = kr[j];
      *reinterpret_cast<u32x4*>(vt + row * TL::ROWB + ((lch ^ step_swz_v<T, D>(row)) << 4)) = vr[j];
    }
    const unsigned miss = bad;
    if (next(i) < end) load(next(i));
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // (this wave's tile: LDS keeps a wave's order)
    __builtin_amdgcn_wave_barrier();

    f32x4 s[RB][KB];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) s[r][kb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int st = 0; st < S; ++st)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int row = 16 * kb + n;
        const u32x4 a = *reinterpret_cast<const u32x4*>(kt + row * TL::ROWB + (((4 * st + g) ^ step_swz_k<T, D>(row)) << 4));
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          u32x4 x;
          if constexpr (LD::Q_LDS) x = *reinterpret_cast<const u32x4*>(ql + (16 * r + n) * TL::ROWB + (((4 * st + g) ^ n) << 4));
          else x = q[r][st];
          s[r][kb] = Mma<T>::k32(a, x, s[r][kb]);
        }
      }

    // a tile that every row sees whole, in pages that are there, needs no mask
    if (miss || !whole_tile) {
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        // bits of the keys from key0 + 4g on: the window up to the query, and the first tokens up to it
        const int base = key0 + 4 * g;
        const int top = (qpos[r] < w.last ? qpos[r] : w.last) - base + 1;
        const int lo = (p.window > 0 ? qpos[r] - p.window + 1 : 0) - base;
        const int first = p.sinks - base < top ? p.sinks - base : top;
        unsigned see = (low_bits(top) & ~low_bits(lo)) | low_bits(first);
        if constexpr (TREE) see = tree_sees(p, b, w.base, ntok, qtree[r], qpos[r], base);
        if (miss & 1) see &= ~0xffffu;
        if (miss & 2) see &= 0xffffu;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[r][kb][j] = masked(s[r][kb][j], see, 16 * kb + j);
      }
    }

    // online softmax in base 2, the scale folded into the exponent; the reference maximum moves only
    // when a score passes it by 2^8 (weights stay <= 2^8, safe in 16 bits), so rescaling is rare
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      float mx = s[r][0][0];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, s[r][kb][j]);
      mx = over_groups<true>(mx) * c;
      if (mx > m[r] + 8.0f) {
        const float a = m[r] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m[r] - mx);
        l[r] *= a;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[r][d] *= a;
        m[r] = mx;
      }
      const float neg = m[r] == kNegInf ? 0.0f : -m[r];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float w8 = __builtin_amdgcn_exp2f(fmaf(s[r][kb][j], c, neg));
          s[r][kb][j] = w8;
          l[r] += w8;
        }
    }

    // O^T += V^T . P^T; the k-slots of a lane are the keys whose weights it holds
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = 16 * kb + 4 * g + j;
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            const int ch = 4 * d + (n >> 2);
            const float a = *reinterpret_cast<const float*>(vt + row * TL::ROWB + ((ch ^ step_swz_v<T, D>(row)) << 4) + 4 * (n & 3));
#pragma unroll
            for (int r = 0; r < RB; ++r)
              o[r][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, s[r][kb][j], o[r][d], 0, 0, 0);
          }
        }
    } else {
      // transposing LDS reads: in each 16-lane group lane 4k + i/4 addresses 4 channels of key k and
      // lane i receives channel i of the four keys
      // A weight goes to the product as two numbers of the type, its rounding and what that left out: rounded once, a
      // row whose softmax rests on few keys had up to 1.5 times the error of fp32 weights, and the second product takes
      // 1 % (one step of 64 ragged rows 711 -> 712 us, a verify step 29.0 -> 29.4, head dim 512 56.8 -> 58.2).
      i16x4 w4[RB][KB], w4b[RB][KB];
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          T x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = from_f32<T>(s[r][kb][j]);
          w4[r][kb] = *reinterpret_cast<const i16x4*>(x);
          T y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = from_f32<T>(s[r][kb][j] - (float)x[j]);
          w4b[r][kb] = *reinterpret_cast<const i16x4*>(y);
        }
      const int vrow = 4 * g + (n >> 2);
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        i16x4 a4[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const int row = 16 * kb + vrow, ch = 2 * d + ((n & 3) >> 1);
          const unsigned at = lds_offset(vt) + row * TL::ROWB + ((ch ^ step_swz_v<T, D>(row)) << 4) + 8 * (n & 1);
          a4[kb] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)at);
        }
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          if constexpr (KB == 2) {
            const i16x8 a = __builtin_shufflevector(a4[0], a4[1], 0, 1, 2, 3, 4, 5, 6, 7);
            const i16x8 x = __builtin_shufflevector(w4[r][0], w4[r][1], 0, 1, 2, 3, 4, 5, 6, 7);
            o[r][d] = Mma<T>::k32(__builtin_bit_cast(u32x4, a), __builtin_bit_cast(u32x4, x), o[r][d]);
            const i16x8 z = __builtin_shufflevector(w4b[r][0], w4b[r][1], 0, 1, 2, 3, 4, 5, 6, 7);
            o[r][d] = Mma<T>::k32(__builtin_bit_cast(u32x4, a), __builtin_bit_cast(u32x4, z), o[r][d]);
          } else {
            o[r][d] = Mma<T>::k16(a4[0], w4[r][0], o[r][d]);
            o[r][d] = Mma<T>::k16(a4[0], w4b[r][0], o[r][d]);
          }
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  if constexpr (TREE) {
#pragma unroll 1
    for (int y = odd_from; y >= 0 && y <= odd_to; y += 4) {   // the values that were taken out, for the rows that see them
      const int key0 = w.tile_key(y, KT);
#pragma unroll 1
      for (int key = key0; key < key0 + KT && key <= w.last; ++key) {
        const int page = p.page_of(b, key);
        if (page < 0) continue;
        const char* src = vb0 + page * pageb + (int64_t)(key & p.page_mask) * rowb;
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          if (!(tree_sees(p, b, w.base, ntok, qtree[r], qpos[r], key) & 1)) continue;
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const T v = reinterpret_cast<const T*>(src)[16 * d + 4 * g + j];
              if (not_finite(v)) o[r][d][j] += to_f32<T>(v);
            }
        }
      }
    }
  }

  // ---- the four waves' rows meet: each scales its own to the common maximum and puts it into its LDS
  // region (16-byte pieces turned with the row), then all threads add the four
  float2* ml = reinterpret_cast<float2*>(smem + 4 * LD::WAVE);  // [wave][ROWS]
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    l[r] = over_groups<false>(l[r]);
    if (g == 0) ml[wave * ROWS + 16 * r + n] = make_float2(m[r], l[r]);
  }
  __syncthreads();
  constexpr int Q4 = D / 4;  // float4 pieces of a row
  const int row0 = rblk * ROWS;
  const int here = w.rows - row0 < ROWS ? w.rows - row0 : ROWS;   // real rows of the block, and those that exist
  const int exist = p.rows - row0 < ROWS ? p.rows - row0 : ROWS;
  float4* mine = reinterpret_cast<float4*>(smem + wave * LD::WAVE);
  float2* all = ml + 4 * ROWS;  // [ROWS] of the four together
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int row = 16 * r + n;
    float2 e[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) e[y] = ml[y * ROWS + row];
    const float M = fmaxf(fmaxf(e[0].x, e[1].x), fmaxf(e[2].x, e[3].x));
    const float a = rescale(m[r], M);
    if (row < here) {
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const int piece = (4 * d + g) ^ (n & (Q4 < 16 ? Q4 - 1 : 15));
        mine[row * Q4 + piece] = make_float4(o[r][d][0] * a, o[r][d][1] * a, o[r][d][2] * a, o[r][d][3] * a);
      }
    }
    if (wave == 0 && g == 0) {
      float L = 0.0f;
#pragma unroll
      for (int y = 0; y < 4; ++y) L += rescale(e[y].x, M) * e[y].y;
      all[row] = make_float2(M, L);
    }
  }
  __syncthreads();
  constexpr int PIECES = ROWS * Q4, PER = PIECES < 256 ? 1 : PIECES / 256;   // of a thread
  constexpr int BATCH = PER < 4 ? PER : 4;                                   // whose reads go out together
#pragma unroll
  for (int x0 = 0; x0 < PER; x0 += BATCH) {
    if (x0 * 256 / Q4 >= exist) break;
    float4 f[BATCH][4];
    float2 e[BATCH];
#pragma unroll
    for (int x = 0; x < BATCH; ++x) {
      const int at = ((x0 + x) * 256 + (int)threadIdx.x) % PIECES, row = at / Q4, c4 = at % Q4;
#pragma unroll
      for (int y = 0; y < 4; ++y)
        f[x][y] = reinterpret_cast<const float4*>(smem + y * LD::WAVE)[row * Q4 + (c4 ^ (row & (Q4 < 16 ? Q4 - 1 : 15)))];
      e[x] = all[row];
    }
#pragma unroll
    for (int x = 0; x < BATCH; ++x) {
      const int at = (x0 + x) * 256 + (int)threadIdx.x, row = at / Q4, c4 = at % Q4;
      if (row >= exist) continue;
      const float4 acc = make_float4((f[x][0].x + f[x][1].x) + (f[x][2].x + f[x][3].x), (f[x][0].y + f[x][1].y) + (f[x][2].y + f[x][3].y),
                                     (f[x][0].z + f[x][1].z) + (f[x][2].z + f[x][3].z), (f[x][0].w + f[x][1].w) + (f[x][2].w + f[x][3].w));
      if (row >= here) {
        store_row<T>(p, b, kvh, row0 + row, 4 * c4, make_float4(0.0f, 0.0f, 0.0f, 0.0f), 0.0f);
      } else if (whole) {
        store_row<T>(p, b, kvh, row0 + row, 4 * c4, acc, e[x].y > 0.0f ? 1.0f / e[x].y : 0.0f);
      } else {
        const int64_t slot = (int64_t)work.slot * ROWS + row;
        float* po = p.ws_o + slot * D + 4 * c4;
        if (p.counters) {
          store_shared(reinterpret_cast<float2*>(po), acc.x, acc.y);
          store_shared(reinterpret_cast<float2*>(po) + 1, acc.z, acc.w);
          if (c4 == 0) store_shared(p.ws_ml + slot, e[x].x, e[x].y);
        } else {
          *reinterpret_cast<float4*>(po) = acc;
          if (c4 == 0) p.ws_ml[slot] = e[x];
        }
      }
    }
  }
  if (whole || !p.counters) return;

  // ---- the part that arrives last merges the row block (the others' partials are where agent-scope accesses find
  // them once their stores are acknowledged; the counter wraps to zero for the next call)
  __shared__ int last;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const int unit = work.slot / p.nparts;
    last = atomicInc(p.counters + unit, (unsigned)work.parts - 1) == (unsigned)work.parts - 1;
  }
  __syncthreads();
  if (!last) return;
  const int64_t slot0 = (int64_t)(work.slot - work.part) * ROWS;
  for (int x = threadIdx.x; x < here * Q4; x += 256) {
    const int row = x / Q4, ch = 4 * (x % Q4);
    float4 O;
    const float L = merge_parts<D, 8, true>(p.ws_ml + slot0 + row, p.ws_o + (slot0 + row) * D + ch, work.parts, ROWS, O);
    store_row<T>(p, b, kvh, row0 + row, ch, O, L > 0.0f ? 1.0f / L : 0.0f);
  }
}

template <typename T, int D, int RB, StepMode MODE> static int launch_step_rb(PagedParams p, hipStream_t s) {
  using LD = StepLds<T, D, RB>;
  static std::atomic<uint64_t> done{0};
  if (const int st = reserve_lds(reinterpret_cast<const void*>(&paged_step_kernel<T, D, RB, MODE>), LD::BYTES, done)) return st;
  const int nrb = (p.rows + LD::ROWS - 1) / LD::ROWS;
  if (nrb > 65535) return set_error("forge_attn_paged: too many query rows");
  hipLaunchKernelGGL((paged_step_kernel<T, D, RB, MODE>), dim3((unsigned)(p.B * p.K), p.nparts, nrb), dim3(256), LD::BYTES, s, p);
  int st = check_launch();
  if (st == 0 && p.nparts > 1 && !p.counters) st = launch_paged_combine<T, D, LD::ROWS, StepTile<T, D, RB>::KT, false, MODE == kTree>(p, s);
  return st;
}

template <typename T, int D, int RB, bool TREE> static int launch_step_rows(const PagedParams& p, hipStream_t s) {
  if constexpr (TREE) return launch_step_rb<T, D, RB, kTree>(p, s);
  else return p.fixed ? launch_step_rb<T, D, RB, kFixed>(p, s) : launch_step_rb<T, D, RB, kFree>(p, s);
}

template <typename T, int D, bool TREE> static int launch_step(const PagedParams& p, const PagedPlan& plan, hipStream_t s) {
  if constexpr (step_rows_most(sizeof(T), D) >= 32) {
    if (plan.rows == 32) return launch_step_rows<T, D, 2, TREE>(p, s);
  }
  if (plan.rows == 16) return launch_step_rows<T, D, 1, TREE>(p, s);
  return set_error("forge_attn_paged: no kernel of this row block");
}

template <typename T, bool TREE> int launch_paged(const PagedParams& p, const PagedPlan& plan, int D, hipStream_t s) {
  switch (D) {
    case 32: return launch_step<T, 32, TREE>(p, plan, s);
    case 64: return launch_step<T, 64, TREE>(p, plan, s);
    case 128: return launch_step<T, 128, TREE>(p, plan, s);
    case 256: return launch_step<T, 256, TREE>(p, plan, s);
    case 512:
      if constexpr (sizeof(T) == 2) return launch_step<T, 512, TREE>(p, plan, s);
    default: return set_error("forge_attn_paged: unsupported head dim");
  }
}

// (one type a translation unit, trees apart: they build side by side)
#if FORGE_PAGED_PART == 1
template int launch_paged<bf16, false>(const PagedParams&, const PagedPlan&, int, hipStream_t);
#elif FORGE_PAGED_PART == 2
template int launch_paged<f16, false>(const PagedParams&, const PagedPlan&, int, hipStream_t);
#elif FORGE_PAGED_PART == 3
template int launch_paged<float, false>(const PagedParams&, const PagedPlan&, int, hipStream_t);
#elif FORGE_PAGED_PART == 4
template int launch_paged<bf16, true>(const PagedParams&, const PagedPlan&, int, hipStream_t);
#elif FORGE_PAGED_PART == 5
template int launch_paged<f16, true>(const PagedParams&, const PagedPlan&, int, hipStream_t);
#elif FORGE_PAGED_PART == 6
template int launch_paged<float, true>(const PagedParams&, const PagedPlan&, int, hipStream_t);
#endif

}  // namespace forge
