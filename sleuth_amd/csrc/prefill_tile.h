// The 32x32 matrix-core tiles of the prefill kernels (prefill.hip) and of the paged chunk kernel
// (paged_chunk.hip): MFMA steps, block shape per head dim, LDS swizzles, the wait for loads into LDS.
#pragma once

#include "common.h"

namespace forge {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

template <typename T> struct Mfma;
template <> struct Mfma<bf16> {
  typedef bf16x8 vec;
  static __device__ __forceinline__ floatx16 run(vec a, vec b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mfma<f16> {
  typedef f16x8 vec;
  static __device__ __forceinline__ floatx16 run(vec a, vec b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

constexpr float kLazyLog2 = 8.0f;

// Block shape per head dim: WAVES waves of 32 queries each, STAGES LDS stages of one K
// and one V tile of BN keys (loads run STAGES - 1 tiles ahead of the compute).
template <int D> struct Tile {
  static constexpr int WAVES = 4;
  static constexpr int STAGES = 2;
  static constexpr int BM = 32 * WAVES;                // queries per block
  static constexpr int BN = D >= 256 ? 32 : 64;        // keys per tile
  static constexpr int NCH = D / 8;                    // 16-byte chunks per key row
  static constexpr int ROWB = 2 * D;                   // bytes per key row
  static constexpr int TILEB = BN * ROWB;              // bytes of one K (or V) tile
  static constexpr int LOADS = TILEB / (WAVES * 1024);   // 16-byte loads per lane per tile
  static constexpr int LDS_BYTES = STAGES * 2 * TILEB;
  static_assert(LOADS * WAVES * 1024 == TILEB, "tile must split into whole wave loads");
};

// XOR swizzles of the 16-byte chunk index by key row (see the reads below).
template <int D> __device__ __forceinline__ int swz_k(int row) {
  return row & ((D / 8 >= 16 ? 16 : D / 8) - 1);
}
template <int D> __device__ __forceinline__ int swz_v(int row) {
  return D / 8 >= 16 ? (row & 3) << 2 : ((row >> 1) & 1) << 2;
}

// Wait until at most N vector-memory loads of this wave are outstanding (loads retire in
// issue order, so everything issued before the last N has landed).
template <int N> __device__ __forceinline__ void wait_vm() {
  static_assert(N == 0 || N == 2 || N == 4 || N == 8, "add the count");
  if constexpr (N == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  else if constexpr (N == 2) asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
  else if constexpr (N == 4) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
}

}  // namespace forge
