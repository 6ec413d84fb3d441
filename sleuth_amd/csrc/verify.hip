// Verification of drafted tokens against the target's logits (forge_verify_drafts).
//
// Node 0 of a row is its last token that stands; node t hangs on an earlier one, parents[t], and was drafted as what
// follows it. With e = exp((l - max l) / temperature) over a node's logits l, Z = sum e, and q what the drafter gave each
// token there, the walk starts at node 0 and asks its children in order. Child j is accepted iff
//   u q(x) W_j < r_j(x),   r_j(v) = max(e(v) - a_j q(v), 0),  W_j = sum_v r_j(v),  a_0 = 0,  a_{j+1} = a_j + W_j:
// repeated rejection takes q, scaled to what was left, out of what was left, and since q >= 0 all the steps so far fold
// into one difference. Without the drafter's probabilities a rejected child takes its own token out (q is one there). An
// accepted child is where the walk goes on; where all are rejected (or there are none) the next token is the first v
// with r(0) + .. + r(v) > u W. Temperature 0: a child is accepted iff its token is the argmax, which is the next token.
//
// The answers are whole numbers, so sums and weights are held in 64 bits: in 32, one draw in thirty of a vocabulary of
// 131,072 would come out one token off.
//
// Every node's logits are read once, whichever the walk needs, by one launch over chunks of all nodes (each chunk's
// maximum and sum); a block per row then walks, and draws within the one chunk that its number falls into. Waiting for the
// walk to know which nodes it needs would read less and take a launch a level. What a rejected child's probabilities leave
// has to be summed over a whole row of the vocabulary: a launch more, whose blocks end at once for the rows that need
// none, and whose last one draws. Greedy calls of few chunks walk in the scan's own launch.
//
// us a call (and each launch): one greedy chain of 5 over 32,768 tokens 7.9; 32 sampled chains of 6 over 131,072 in bf16 with
// the drafter's probabilities 44 (scan 22: VALU, 0.86 of the SIMDs' cycles; walk 11 and rest 15: latency, a chain of loads and
// cross-lane sums); 8 trees of up to 40 over 100,003 in fp32 30 (scan 19: 3.5 TB/s, VALU 0.67; walk 12).
#include <limits.h>

#include "common.h"
#include "forge_internal.h"

namespace forge {

constexpr int kVerifyChunk = 4096;  // elements of a row that a block takes
constexpr int kScanThreads = 256, kWalkThreads = 512;
constexpr int kVerifyNodes = FORGE_TREE_MAX_TOKENS;
static_assert(2 * kWalkThreads >= kVerifyNodes, "a thread of the walk takes two nodes");

struct VerifyParams {
  const void* logits;
  int64_t slb, slt;
  const int64_t* tokens;
  int64_t stb;
  const int32_t* parents;  // null: a chain
  int64_t spb;
  const float* uniform;
  int64_t sub;
  const float* temps;  // [B], or null: `temperature`
  double temperature;
  const void* probs;  // null: none
  int64_t sqb, sqt;
  const int32_t* new_lens;
  int B, T, V, C;  // C: chunks of a row
  int64_t* out;    // [B][T]
  int32_t* path;
  int32_t* count;
  // workspace: each chunk's sum, maximum and its first place; a row's state between launches; the sums of what is left
  struct Part* parts;  // [B][T][C]
  unsigned* counters;  // [B], zero between calls: the block that scans a row's last chunk walks. Null: a launch of its own does
  double scale_hi, scale_lo;  // of `temperature`
  struct State* state;  // [B]
  double* rest;         // [B][C]

  __device__ __forceinline__ int nodes(int b) const {
    const int n = new_lens ? new_lens[b] : T;
    return n < 0 ? 0 : n < T ? n : T;
  }
  __device__ __forceinline__ double heat(int b) const {
    return !temps ? temperature : temps[b] > 1e30f ? 1e30 : (double)temps[b];
  }
};

struct Part {
  double z;
  float m;
  int i;
};

// Where a row's walk ended, if its next token is drawn from what the drafter's probabilities left.
struct State {
  double taken;  // a
  float most;    // max l
  int node, at;  // where; which of the row's outputs the token is
  int left;      // 0: drawn already
  unsigned done;  // blocks that have summed their chunk
};

// log2(e) / temperature in two parts.
struct Scale {
  double hi, lo;
};
__host__ __device__ inline Scale scale_of(double temperature) {
  constexpr double l_hi = 0x1.71547652b82fep+0, l_lo = 0x1.777d0ffda0d24p-56;
  Scale s;
  s.hi = l_hi / temperature;
  s.lo = (fma(-s.hi, temperature, l_hi) + l_lo) / temperature;
  return s;
}
__device__ __forceinline__ Scale row_scale(const VerifyParams& p, int b) {
  if (!p.temps) return Scale{p.scale_hi, p.scale_lo};
  const double heat = p.heat(b);
  return scale_of(heat > 0.0 ? heat : 1.0);
}

// 2^f = 1 + f P(f), |f| <= 1/2: P interpolates (2^f - 1) / f at ten Chebyshev points (off by 6e-16 at most).
__device__ __forceinline__ double exp2_part(double f) {
  double p = 0x1.e5e83cccccccdp-28;
  p = fma(p, f, 0x1.b657203333333p-24);
  p = fma(p, f, 0x1.62bfe55000000p-20);
  p = fma(p, f, 0x1.ffcb767660000p-17);
  p = fma(p, f, 0x1.4309130322a00p-13);
  p = fma(p, f, 0x1.5d87fe909032ap-10);
  p = fma(p, f, 0x1.3b2ab6fba39c7p-7);
  p = fma(p, f, 0x1.c6b08d7044115p-5);
  p = fma(p, f, 0x1.ebfbdff82c590p-3);
  p = fma(p, f, 0x1.62e42fefa39f7p-1);
  return fma(p, f, 1.0);
}
// exp((x - m) / temperature) to about 1e-15, exactly 1 at x = m, 0 for -inf and for a NaN (which no maximum takes): 2^t with t = k + f, k from the low bits of
// t + 1.5 2^52.
__device__ __forceinline__ double weight(float x, float m, Scale c) {
  const double d = x == m ? 0.0 : (double)x - (double)m;   // (infinite logits share the mass)
  const double t = d * c.hi, lo = fma(d, c.lo, fma(d, c.hi, -t));
  const double big = t + 0x1.8p52, f = (t - (big - 0x1.8p52)) + lo;
  return t > -1100.0 ? ldexp(exp2_part(f), __double2loint(big)) : 0.0;   // (NaN: 0)
}

// 64-bit numbers across lanes without a way through LDS (the walk is one chain of such steps).
template <int CTRL, int ROWS = 0xF> __device__ __forceinline__ double dpp64(double x) {   // 0 where a lane has no partner
  return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(x), CTRL, ROWS, 0xF, true),
                          __builtin_amdgcn_update_dpp(0, __double2loint(x), CTRL, ROWS, 0xF, true));
}
// Sum over aligned groups of 16 or 64 lanes: every lane receives it.
template <int W> __device__ __forceinline__ double lanes_sum(double x) {
  x += dpp64<kDppQuadXor1>(x);
  x += dpp64<kDppQuadXor2>(x);
  x += dpp64<kDppRowHalfMirror>(x);
  x += dpp64<kDppRowMirror>(x);
  if constexpr (W == 64) {
    const auto halves = [](double y, auto swap) {   // both halves of each pair, added in one order
      const auto lo = swap((unsigned)__double2loint(y)), hi = swap((unsigned)__double2hiint(y));
      const unsigned l0 = lo[0], l1 = lo[1], h0 = hi[0], h1 = hi[1];
      return __hiloint2double((int)h0, (int)l0) + __hiloint2double((int)h1, (int)l1);
    };
    x = halves(x, [](unsigned u) { return __builtin_amdgcn_permlane16_swap(u, u, false, false); });
    x = halves(x, [](unsigned u) { return __builtin_amdgcn_permlane32_swap(u, u, false, false); });
  }
  return x;
}
// Sum of the lanes up to one's own.
__device__ __forceinline__ double lanes_upto(double x) {
  x += dpp64<0x111>(x);         // row_shr 1, 2, 4, 8: within rows of 16
  x += dpp64<0x112>(x);
  x += dpp64<0x114>(x);
  x += dpp64<0x118>(x);
  x += dpp64<0x142, 0xA>(x);    // a row's last lane to the next row
  x += dpp64<0x143, 0xC>(x);    // lane 31 to the upper half
  return x;
}

// Sum over the block, in one fixed order; every thread receives it. `lds`: one double a wave.
template <int THREADS> __device__ __forceinline__ double block_sum(double x, double* lds) {
  x = lanes_sum<64>(x);
  __syncthreads();   // (the last call's readers)
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = x;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) s += lds[w];
  return s;
}

// Numbers of blocks on several XCDs, whose caches are their own, are written past those, counted, and read by the block that
// counts last.
__device__ __forceinline__ void store_agent(double* p, double x) {
  __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double load_agent(const double* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_part(Part* p, Part x) {
  store_agent(&p->z, x.z);
  store_agent(reinterpret_cast<double*>(&p->m), __hiloint2double(x.i, __float_as_int(x.m)));
}
template <bool FUSED> __device__ __forceinline__ Part load_part(const Part* p) {   // (of another launch: as any memory)
  if constexpr (!FUSED) return *p;
  const double z = load_agent(&p->z), mi = load_agent(reinterpret_cast<const double*>(&p->m));
  return Part{z, __int_as_float(__double2loint(mi)), __double2hiint(mi)};
}

// A row of logits, whose 16-byte pieces start `shift` elements before it; chunk c is elements c * 4096 - shift on.
template <typename T> struct Row {
  static constexpr int E = 16 / sizeof(T);
  const T* at;
  int V, shift;
  __device__ __forceinline__ Row(const T* p, int V) : at(p), V(V), shift((int)((uintptr_t)p % 16 / sizeof(T))) {}
  // the E elements from i on (a piece's first), -inf where there are none
  __device__ __forceinline__ void piece(int i, float (&x)[E]) const {
    if (i >= 0 && i + E <= V) {
      unpack16<T>(load16(at + i), x);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = i + e >= 0 && i + e < V ? to_f32<T>(at[i + e]) : kNegInf;
    }
  }
  __device__ __forceinline__ float one(int i) const { return to_f32<T>(at[i]); }
};
template <typename T> __device__ __forceinline__ Row<T> logits_row(const VerifyParams& p, int b, int t) {
  return Row<T>(static_cast<const T*>(p.logits) + b * p.slb + t * p.slt, p.V);
}

// Chunk c of node t of row b: its maximum, the first element that holds it, the sum of its weights against it.
//
// The draw takes a chunk's elements apart with weights of 1e-15, so what a sum here may be off by moves a few chunks' ends
// and a threshold, not every element's: 1e-10 of itself turns one answer in 10^8. So the scan has its own form of a weight,
// with the temperature's scale in one part and a polynomial through seven points (1.2e-10), the exponent added as a whole
// number, and nothing below 2^-1000: 19 instructions a logit, which are what it waits for (a bf16 logit comes from memory
// in half that time). The argmax is looked for where it decides, at temperature 0.
template <typename T, bool GREEDY> __device__ __forceinline__ Part scan_chunk(const VerifyParams& p, int b, int t, int c) {
  constexpr int E = Row<T>::E, U = kVerifyChunk / kScanThreads / E, WAVES = kScanThreads / kWave;
  const Row<T> row = logits_row<T>(p, b, t);
  const int first = c * kVerifyChunk - row.shift;
  float x[U][E];
#pragma unroll
  for (int u = 0; u < U; ++u) row.piece(first + (u * kScanThreads + (int)threadIdx.x) * E, x[u]);
  float m = kNegInf;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) m = fmaxf(m, x[u][e]);
  __shared__ float wm[WAVES];
  __shared__ int wi[WAVES];
  __shared__ double wz[WAVES];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  m = group_max<64>(m);
  if (lane == 0) wm[wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) m = fmaxf(m, wm[w]);
  double z = 0.0;
  int i = 0;
  if (GREEDY || !(p.heat(b) > 0.0)) {
    i = p.V;
#pragma unroll
    for (int u = U - 1; u >= 0; --u)
#pragma unroll
      for (int e = E - 1; e >= 0; --e)
        if (x[u][e] == m) i = first + (u * kScanThreads + (int)threadIdx.x) * E + e;
    for (int d = 32; d; d >>= 1) i = min(i, __shfl_xor(i, d, kWave));
  } else if (m > kNegInf) {
    const Scale s = row_scale(p, b);
    if (m == -kNegInf) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) z += x[u][e] == m ? 1.0 : 0.0;
    } else {
      const double md = m, least = -1000.0 / s.hi;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const double d = fmax((double)x[u][e] - md, least), big = fma(d, s.hi, 0x1.8p52);
          const double f = fma(d, s.hi, -(big - 0x1.8p52));
          double q = 0x1.00a581599a492p-16;
          q = fma(q, f, 0x1.443fffc90e1b7p-13);
          q = fma(q, f, 0x1.5d879ead062cep-10);
          q = fma(q, f, 0x1.3b2a1b7152be9p-7);
          q = fma(q, f, 0x1.c6b08d883dca7p-5);
          q = fma(q, f, 0x1.ebfbe045f4d3cp-3);
          q = fma(q, f, 0x1.62e42fefa39efp-1);
          q = fma(q, f, 1.0);
          z += __hiloint2double(__double2hiint(q) + (int)((unsigned)__double2loint(big) << 20), __double2loint(q));
        }
    }
    for (int d = 32; d; d >>= 1) z += __shfl_xor(z, d, kWave);
  }
  if (lane == 0) wi[wave] = i, wz[wave] = z;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) i = w == 0 ? wi[0] : min(i, wi[w]), z = w == 0 ? wz[0] : z + wz[w];
  return Part{z, m, i};
}

// The chunk that `target` falls into by the sums mass(0), mass(1), ..: the first c with mass(0) + .. + mass(c) > target, and
// what it has to pass there; where rounding leaves none, the last one that has any. All threads receive both.
struct Found {
  int c;
  double target;
};
template <typename F> __device__ __forceinline__ Found find_chunk(int C, double target, F mass) {
  __shared__ Found found;
  if (threadIdx.x < kWave) {
    const int lane = threadIdx.x;
    double before = 0.0;
    Found f{-1, 0.0};
    int last = 0;
    for (int c0 = 0; c0 < C && f.c < 0; c0 += kWave) {
      const double own = c0 + lane < C ? mass(c0 + lane) : 0.0;
      const double upto = lanes_upto(own);
      const uint64_t over = __ballot(before + upto > target && own > 0.0), some = __ballot(own > 0.0);
      if (some) last = c0 + 63 - __builtin_clzll(some);
      if (over) {
        const int l = __builtin_ctzll(over);
        f.c = c0 + l;
        f.target = target - before - (l ? __shfl(upto, l - 1, kWave) : 0.0);
      }
      before += __shfl(upto, kWave - 1, kWave);
    }
    if (f.c < 0) f = Found{last, 1.7e308};
    if (lane == 0) found = f;
  }
  __syncthreads();
  return found;
}

// The first element of a chunk at which the running sum of what the threads hold (PER elements each, r) passes the target,
// or the last that has any.
template <int THREADS, int PER = kVerifyChunk / THREADS>
__device__ __forceinline__ int find_element(int first, double target, const double (&r)[PER]) {
  __shared__ double sums[THREADS / kWave];
  __shared__ int hit, most;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int i0 = first + (int)threadIdx.x * PER;
  if (threadIdx.x == 0) hit = INT_MAX, most = -1;
  double own = 0.0;
#pragma unroll
  for (int e = 0; e < PER; ++e) own += r[e];
  const double upto = lanes_upto(own);
  if (lane == kWave - 1) sums[wave] = upto;
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) sum += w < wave ? sums[w] : 0.0;
  sum += upto - own;
  int at = INT_MAX, last = -1;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    sum += r[e];
    if (r[e] > 0.0) {
      last = i0 + e;
      if (sum > target) at = min(at, i0 + e);
    }
  }
  if (at < INT_MAX) atomicMin(&hit, at);
  if (last >= 0) atomicMax(&most, last);
  __syncthreads();
  return hit < INT_MAX ? hit : most < 0 ? 0 : most;
}

// The first element that holds the row's maximum (where rejections left nothing: once in a blue moon).
template <int THREADS, typename T> __device__ __forceinline__ int argmax_of(Row<T> row, float top) {
  __shared__ int first;
  if (threadIdx.x == 0) first = INT_MAX;
  __syncthreads();
  int i = threadIdx.x;
  while (i < row.V && row.one(i) != top) i += THREADS;
  if (i < row.V) atomicMin(&first, i);
  __syncthreads();
  return first < INT_MAX ? first : 0;
}

// max(e - a q, 0) over a row whose next token is drawn from there.
template <typename T, typename Q> struct Rest {
  Row<T> row;
  const Q* q;
  double taken;
  float most;
  Scale s;
  __device__ __forceinline__ Rest(const VerifyParams& p, int b, int node, double taken, float most, Scale s)
      : row(logits_row<T>(p, b, node)), q(static_cast<const Q*>(p.probs) + b * p.sqb + node * p.sqt), taken(taken), most(most),
        s(s) {}
  __device__ __forceinline__ double of(float x, double q) const { return fmax(weight(x, most, s) - taken * q, 0.0); }
  __device__ __forceinline__ double one(int v) const { return of(row.one(v), (double)to_f32<Q>(q[v])); }
  // the 8 N elements from i0 on, a piece's first; 0 where there are none
  template <int N> __device__ __forceinline__ void eights(int i0, double (&r)[8 * N]) const {
    constexpr int E = Row<T>::E, F = 16 / (int)sizeof(Q);
    float x[8 * N], y[8 * N];
#pragma unroll
    for (int u = 0; u < 8 * N / E; ++u) row.piece(i0 + u * E, reinterpret_cast<float(&)[E]>(x[u * E]));
    if (i0 >= 0 && i0 + 8 * N <= row.V && (uintptr_t)(q + i0) % 16 == 0) {
#pragma unroll
      for (int u = 0; u < 8 * N / F; ++u) unpack16<Q>(load16(q + i0 + u * F), y + u * F);
    } else {
#pragma unroll
      for (int e = 0; e < 8 * N; ++e) y[e] = i0 + e >= 0 && i0 + e < row.V ? to_f32<Q>(q[i0 + e]) : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 8 * N; ++e) r[e] = of(x[e], (double)y[e]);
  }
};

// The walk's shared memory: a few numbers a node, a sum a chunk, and all chunks' numbers where they are few.
struct WalkLds {
  static constexpr int KEPT = 1024;   // chunks of all nodes
  double *zs, *es, *masses, *sums;   // (es, par and tok are read four nodes at a time)
  Part* parts;
  float *most, *us, *qs;
  int *args, *tok, *par, *child, *sib;
  bool* yes;
  __host__ __device__ static bool keeps(int T, int C) { return T <= 512 && T * C <= KEPT; }   // (all of it below 64 KB)
  __host__ __device__ static size_t bytes(int T, int C) {
    const size_t nodes = (T + 3) / 4 * 4;
    return 8 * (2 * nodes + C + C % 2 + 16) + (keeps(T, C) ? sizeof(Part) * T * C : 0) + 33 * nodes;
  }
  __device__ __forceinline__ WalkLds(char* at, int T, int C) {
    const auto take = [&](auto*& p, size_t n) {
      p = reinterpret_cast<decltype(p + 0)>(at);
      at += n * sizeof(*p);
    };
    const int nodes = (T + 3) / 4 * 4;
    take(parts, keeps(T, C) ? T * C : 0);
    take(zs, nodes);
    take(es, nodes);
    take(masses, C + C % 2);
    take(sums, 16);
    take(most, nodes);
    take(us, nodes);
    take(qs, nodes);
    take(args, nodes);
    take(tok, nodes);
    take(par, nodes);
    take(child, nodes);
    take(sib, nodes);
    take(yes, nodes);
  }
};

// A row's walk, by one block: from the chunks' numbers to its new tokens. Latency: what is read hangs on what was read
// before, the tokens, their logits, the chunks' numbers, the one chunk that the draw falls into. FUSED: behind the scan, in its
// launch, greedily.
template <typename T, typename Q, int THREADS, bool FUSED> __device__ __forceinline__ void walk_row(const VerifyParams& p, int b, char* smem) {
  constexpr int PER = kVerifyChunk / THREADS, WAVES = THREADS / kWave;
  const WalkLds l(smem, p.T, p.C);
  const int n = p.nodes(b), tid = threadIdx.x, lane = tid % kWave;
  int64_t* out = p.out + (int64_t)b * p.T;
  int32_t* path = p.path + (int64_t)b * p.T;
  const bool warm = !FUSED && p.heat(b) > 0.0;
  const Scale s = FUSED ? Scale{} : row_scale(p, b);
  const Q* probs = FUSED ? nullptr : static_cast<const Q*>(p.probs);

  // Each drafted token, its parent, and the logit and probability it is judged by; the first chunks' numbers are on their
  // way meanwhile.
  constexpr int MINE = 2;   // (nodes a thread: the launch sees to it)
  struct Drafted {
    int64_t token;
    int up;
    float u;
  };
  const auto drafted = [&](int t) {
    return Drafted{p.tokens[b * p.stb + t], t == 0 ? -1 : p.parents ? p.parents[b * p.spb + t] : t - 1,
                   warm ? p.uniform[b * p.sub + t] : 0.0f};
  };
  const auto judged = [&](int t, Drafted d, float& x, float& q) {
    const bool real = d.token >= 0 && d.token < p.V && d.up >= 0 && d.up < t;   // (others are passed over)
    l.tok[t] = real ? (int)d.token : -1;
    l.par[t] = real ? d.up : -1;
    l.us[t] = d.u;
    l.child[t] = p.T;
    x = real && warm ? logits_row<T>(p, b, d.up).one((int)d.token) : kNegInf;
    q = real && warm && probs ? to_f32<Q>(probs[b * p.sqb + d.up * p.sqt + d.token]) : 0.0f;
  };
  float logit[MINE], prob[MINE];
  Drafted d[MINE];
#pragma unroll
  for (int y = 0; y < MINE; ++y)
    if (tid + y * THREADS < n) d[y] = drafted(tid + y * THREADS);
  const bool keep = WalkLds::keeps(p.T, p.C);
  const Part* parts = p.parts + (int64_t)b * p.T * p.C;
  const int wide = n <= THREADS / kWave ? 64 : 16, mine = tid & (wide - 1);   // lanes a node: a wave where those are enough
  const auto two = [&](int t, int c0, Part (&x)[2]) {
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int c = c0 + y * wide + mine;
      x[y] = t < n && c < p.C ? load_part<FUSED>(parts + t * p.C + c) : Part{0.0, kNegInf, p.V};
    }
  };
  Part early[2];
  two(tid / wide, 0, early);
#pragma unroll
  for (int y = 0; y < MINE; ++y)
    if (tid + y * THREADS < n) judged(tid + y * THREADS, d[y], logit[y], prob[y]);
  for (int t = tid; t < p.T; t += THREADS) {
    out[t] = -1;
    path[t] = t == 0 && n > 0 ? 0 : -1;
  }
  if (probs && tid == 0) {
    p.state[b].left = 0;
    p.state[b].done = 0;
  }
  if (n == 0) {
    if (tid == 0) p.count[b] = 0;
    return;
  }

  // each node's maximum, argmax and sum
  for (int t = tid / wide; t < n; t += THREADS / wide) {
    float m = kNegInf;
    int i = p.V;
    double z = 0.0;
    for (int c0 = 0; c0 < p.C; c0 += 2 * wide) {
      Part x[2] = {early[0], early[1]};
      if (t >= THREADS / wide || c0 > 0) two(t, c0, x);
      if (keep) {
#pragma unroll
        for (int y = 0; y < 2; ++y)
          if (c0 + y * wide + mine < p.C) l.parts[t * p.C + c0 + y * wide + mine] = x[y];
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) {   // (the running sum against the running maximum)
        if (x[y].m > m) {
          z = warm ? x[y].z + (m > kNegInf ? z * weight(m, x[y].m, s) : 0.0) : 0.0;
          m = x[y].m;
          i = x[y].i;
        } else if (x[y].m == m) {
          z += x[y].z;
          i = min(i, x[y].i);
        } else if (warm && x[y].m > kNegInf) {
          z += x[y].z * weight(x[y].m, m, s);
        }
      }
    }
    float top = group_max<16>(m);
    if (wide == 64) top = fmaxf(top, __shfl_xor(top, 16, kWave)), top = fmaxf(top, __shfl_xor(top, 32, kWave));
    if (m < top) i = p.V;
    if (warm) z = m > kNegInf ? z * weight(m, top, s) : 0.0;
    z = wide == 64 ? lanes_sum<64>(z) : lanes_sum<16>(z);
    if (!warm)
      for (int d = wide / 2; d; d >>= 1) i = min(i, __shfl_xor(i, d, kWave));
    if (mine == 0) l.most[t] = top, l.args[t] = top > kNegInf ? i : 0, l.zs[t] = z;   // (nothing: the first)
  }
  __syncthreads();
  const auto weigh = [&](int t, float x, float q) {
    const int up = l.par[t];
    double e = warm && up >= 0 && l.most[up] > kNegInf ? weight(x, l.most[up], s) : 0.0;
    l.qs[t] = q;
    if (warm && !probs && up >= 0) {   // a token that an earlier sibling has is out already
      const int mine = l.tok[t];
      bool twice = false;
#pragma unroll 2
      for (int j = (up + 1) & ~3; j < t; j += 4) {
        const int4 a = *reinterpret_cast<const int4*>(l.par + j), k = *reinterpret_cast<const int4*>(l.tok + j);
        twice |= a.x == up && k.x == mine;
        twice |= a.y == up && k.y == mine && j + 1 < t;
        twice |= a.z == up && k.z == mine && j + 2 < t;
        twice |= a.w == up && k.w == mine && j + 3 < t;
      }
      if (twice) e = 0.0;
    }
    l.es[t] = e;
  };
#pragma unroll
  for (int y = 0; y < MINE; ++y)
    if (tid + y * THREADS < n) weigh(tid + y * THREADS, logit[y], prob[y]);
  __syncthreads();

  // Who would be accepted if the walk came to its parent. With the drafter's probabilities that is known for first
  // children only: child[] are a node's first children, sib[] their next siblings. Else child[] are the accepted ones.
  for (int t = tid; t < n; t += THREADS) {
    const int up = l.par[t];
    if (up < 0) continue;
    if (!warm) {
      if (l.tok[t] == l.args[up]) atomicMin(&l.child[up], t);
    } else if (probs) {
      l.yes[t] = l.us[t] * (double)l.qs[t] * l.zs[up] < l.es[t];
      atomicMin(&l.child[up], t);
      int next = p.T;
#pragma unroll 2
      for (int j = (n - 1) & ~3; j + 3 > t; j -= 4) {
        const int4 a = *reinterpret_cast<const int4*>(l.par + j);
        next = a.w == up && j + 3 < n ? j + 3 : next;
        next = a.z == up && j + 2 < n && j + 2 > t ? j + 2 : next;
        next = a.y == up && j + 1 < n && j + 1 > t ? j + 1 : next;
        next = a.x == up && j > t ? j : next;
      }
      l.sib[t] = next;
    } else {
      double left = l.zs[up];
#pragma unroll 2
      for (int j = (up + 1) & ~3; j < t; j += 4) {
        const int4 a = *reinterpret_cast<const int4*>(l.par + j);
        const double2 e0 = *reinterpret_cast<const double2*>(l.es + j), e1 = *reinterpret_cast<const double2*>(l.es + j + 2);
        left -= a.x == up ? e0.x : 0.0;
        left -= a.y == up && j + 1 < t ? e0.y : 0.0;
        left -= a.z == up && j + 2 < t ? e1.x : 0.0;
        left -= a.w == up && j + 3 < t ? e1.y : 0.0;
      }
      if (l.us[t] * fmax(left, 0.0) < l.es[t]) atomicMin(&l.child[up], t);
    }
  }
  __syncthreads();

  // the walk: every thread takes it
  int at = 0, count = 1;
  double taken = 0.0;
  while (true) {
    int t = l.child[at];
    if (t >= p.T) break;
    if (warm && probs && !l.yes[t]) {
      // (a sibling more is a row of the vocabulary more, by this one block: 52 us at 131,072 tokens in bf16)
      taken = l.zs[at];
      for (t = l.sib[t]; t < p.T; t = l.sib[t]) {
        const Rest<T, Q> rest(p, b, at, taken, l.most[at], s);
        double w = 0.0;
#pragma unroll 2
        for (int i = tid * 8 - rest.row.shift; i < p.V; i += THREADS * 8) {
          double x[8];
          rest.template eights<1>(i, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) w += x[e];
        }
        w = block_sum<THREADS>(w, l.sums);
        const double q = l.qs[t];
        if (l.us[t] * q * w < l.es[t] - taken * q) break;
        taken += w;
      }
      if (t >= p.T) break;
      taken = 0.0;
    }
    if (tid == 0) {
      out[count - 1] = l.tok[t];
      path[count] = t;
    }
    at = t;
    ++count;
  }

  int token = warm ? 0 : l.args[at];
  if (warm && l.most[at] > kNegInf && taken > 0.0) {   // what the drafter's probabilities left is drawn from below
    if (tid == 0) p.state[b] = State{taken, l.most[at], at, count - 1, 1, 0};
    token = -1;
  } else if (warm && l.most[at] > kNegInf) {
    const Row<T> row = logits_row<T>(p, b, at);
    const float top = l.most[at];
    double* masses = l.masses;
    int* gone = l.child;     // the rejected children's tokens and weights, and chunks that are summed again
    double* weights = l.zs;
    int* again = l.sib;
    __shared__ int nagain;
    int ngone = 0;
    __syncthreads();
    if (tid == 0) nagain = 0;
    for (int c = tid; c < p.C; c += THREADS) {
      const Part x = keep ? l.parts[at * p.C + c] : parts[at * p.C + c];
      masses[c] = x.m > kNegInf ? x.z * weight(x.m, top, s) : 0.0;
    }
    __syncthreads();
    if (!probs) {
      // (in the nodes' order, in which their weights are added up: every wave counts them, and keeps its own nodes')
      for (int j0 = at + 1; j0 < n; j0 += kWave) {
        const int j = j0 + lane;
        const bool mine = j < n && l.par[j] == at && l.es[j] > 0.0;
        const uint64_t all = __ballot(mine);
        if (mine && (j0 - at - 1) / kWave % WAVES == tid / kWave) {
          const int g = ngone + __popcll(all & ((1ull << lane) - 1));
          gone[g] = l.tok[j];
          weights[g] = l.es[j];
        }
        ngone += __popcll(all);
      }
      __syncthreads();
      // a chunk that loses all but a thousandth of its sum is summed again: the difference could leave what is not there
      for (int g = tid; g < ngone; g += THREADS) {
        const int c = (gone[g] + row.shift) / kVerifyChunk;
        double out_of = 0.0;
        bool first = true;
#pragma unroll 4
        for (int h = 0; h < ngone; ++h) {
          const bool here = (gone[h] + row.shift) / kVerifyChunk == c;
          first &= !here || h >= g;
          out_of += here ? weights[h] : 0.0;
        }
        if (!first) continue;
        const double left = masses[c] - out_of;
        if (left < masses[c] * 0x1p-10) again[atomicAdd(&nagain, 1)] = c;
        else masses[c] = left;
      }
    }
    __syncthreads();
    const auto piece = [&](int c, double (&r)[PER]) {   // the thread's weights of chunk c, without rejected tokens
      constexpr int E = Row<T>::E;
      const int i0 = c * kVerifyChunk - row.shift + tid * PER;
      float x[PER];
#pragma unroll
      for (int u = 0; u < PER / E; ++u) row.piece(i0 + u * E, reinterpret_cast<float(&)[E]>(x[u * E]));
      unsigned cut = 0;
#pragma unroll 4
      for (int g = 0; g < ngone; ++g) {
        const int d = gone[g] - i0;
        cut |= (unsigned)d < PER ? 1u << (d & 31) : 0u;
      }
#pragma unroll
      for (int e = 0; e < PER; ++e) r[e] = cut >> e & 1 ? 0.0 : weight(x[e], top, s);
    };
    double x[PER];
    for (int g = 0; g < nagain; ++g) {
      piece(again[g], x);
      double w = 0.0;
#pragma unroll
      for (int e = 0; e < PER; ++e) w += x[e];
      w = block_sum<THREADS>(w, l.sums);
      if (tid == 0) masses[again[g]] = w;
    }
    if (nagain) __syncthreads();
    double total = 0.0;   // (each wave for itself)
    for (int c = lane; c < p.C; c += kWave) total += masses[c];
    total = lanes_sum<64>(total);
    if (total > 0.0) {
      const Found f = find_chunk(p.C, l.us[0] * total, [&](int c) { return masses[c]; });
      piece(f.c, x);
      token = find_element<THREADS>(f.c * kVerifyChunk - row.shift, f.target, x);
    } else {
      token = argmax_of<THREADS>(row, top);
    }
  }
  if (tid == 0) {
    if (token >= 0) out[count - 1] = token;
    p.count[b] = count;
  }
}

// The scan, a block a chunk. FUSED (greedy calls of few chunks): the block that ends a row's scan walks it too.
template <typename T, bool FUSED>
__global__ __launch_bounds__(kScanThreads) void verify_scan_kernel(VerifyParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int c = blockIdx.x, t = blockIdx.y, b = blockIdx.z, n = p.nodes(b);
  if (t < n) {
    const Part x = scan_chunk<T, FUSED>(p, b, t, c);
    Part* to = p.parts + ((int64_t)b * p.T + t) * p.C + c;
    if constexpr (!FUSED) {
      if (threadIdx.x == 0) *to = x;
      return;
    } else {
      __shared__ bool last;
      if (threadIdx.x == 0) {
        store_part(to, x);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const unsigned all = (unsigned)(n * p.C);   // (the counter wraps to zero for the next call)
        last = atomicInc(p.counters + b, all - 1) == all - 1;
      }
      __syncthreads();
      if (!last) return;
    }
  } else if (!FUSED || n > 0 || t > 0 || c > 0) {
    return;
  }
  if constexpr (FUSED) walk_row<T, float, kScanThreads, true>(p, b, smem);
}
template <typename T, typename Q> __global__ __launch_bounds__(kWalkThreads) void verify_walk_kernel(VerifyParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  walk_row<T, Q, kWalkThreads, false>(p, blockIdx.x, smem);
}

// What the drafter's probabilities left of a row, chunk by chunk; a row's last block draws from it.
template <typename T, typename Q> __global__ __launch_bounds__(kWalkThreads) void verify_rest_kernel(VerifyParams p) {
  constexpr int PER = kVerifyChunk / kWalkThreads;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  double* all = reinterpret_cast<double*>(smem);   // [C]
  __shared__ double lds[kWalkThreads / kWave];
  __shared__ bool last;
  const int c = blockIdx.x, b = blockIdx.y;
  const State st = p.state[b];
  if (!st.left) return;
  const Rest<T, Q> rest(p, b, st.node, st.taken, st.most, row_scale(p, b));
  double* sums = p.rest + (int64_t)b * p.C;
  double x[PER], w = 0.0;
  rest.template eights<PER / 8>(c * kVerifyChunk - rest.row.shift + (int)threadIdx.x * PER, x);
#pragma unroll
  for (int e = 0; e < PER; ++e) w += x[e];
  w = block_sum<kWalkThreads>(w, lds);
  if (threadIdx.x == 0) {
    store_agent(sums + c, w);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    last = atomicAdd(&p.state[b].done, 1u) == (unsigned)p.C - 1;
  }
  __syncthreads();
  if (!last) return;
  const float u = p.uniform[b * p.sub];
  for (int i = threadIdx.x; i < p.C; i += kWalkThreads) all[i] = load_agent(sums + i);
  __syncthreads();
  double total = 0.0;   // (each wave for itself)
  for (int i = threadIdx.x % kWave; i < p.C; i += kWave) total += all[i];
  total = lanes_sum<64>(total);
  int token;
  if (total > 0.0) {
    const Found f = find_chunk(p.C, u * total, [&](int i) { return all[i]; });
    const int first = f.c * kVerifyChunk - rest.row.shift;
    rest.template eights<PER / 8>(first + (int)threadIdx.x * PER, x);
    token = find_element<kWalkThreads>(first, f.target, x);
  } else {
    token = argmax_of<kWalkThreads>(rest.row, st.most);
  }
  if (threadIdx.x == 0) p.out[(int64_t)b * p.T + st.at] = token;
}

struct VerifyWs {
  size_t parts, state, rest, bytes;
};
static int verify_chunks(int V) { return (V + 7 + kVerifyChunk - 1) / kVerifyChunk; }   // (a row may start inside a piece)
static VerifyWs verify_ws(int B, int T, int V, bool probs) {
  const auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  const size_t C = verify_chunks(V);
  VerifyWs w{};
  w.parts = FORGE_PAGED_COUNTER_BYTES;
  w.state = w.parts + up((size_t)B * T * C * sizeof(Part));
  w.rest = w.state + (probs ? up((size_t)B * sizeof(State)) : 0);
  w.bytes = w.rest + (probs ? up((size_t)B * C * sizeof(double)) : 0);
  return w;
}

template <typename T, typename Q> static int launch_verify(const VerifyParams& p, hipStream_t s) {
  const size_t lds = WalkLds::bytes(p.T, p.C);
  const dim3 scan(p.C, p.T, p.B);
  if (p.counters) {
    hipLaunchKernelGGL((verify_scan_kernel<T, true>), scan, dim3(kScanThreads), lds, s, p);
  } else {
    hipLaunchKernelGGL((verify_scan_kernel<T, false>), scan, dim3(kScanThreads), 0, s, p);
    if (const int st = check_launch()) return st;
    hipLaunchKernelGGL((verify_walk_kernel<T, Q>), dim3(p.B), dim3(kWalkThreads), lds, s, p);
  }
  if (const int st = check_launch(); st || !p.probs) return st;
  hipLaunchKernelGGL((verify_rest_kernel<T, Q>), dim3(p.C, p.B), dim3(kWalkThreads), p.C * sizeof(double), s, p);
  return check_launch();
}

}  // namespace forge

using namespace forge;

static bool verify_sizes_ok(int B, int T, int V) {
  // (the grid's limits; the chunks' sums of a node fit the walk's shared memory)
  return B > 0 && B <= 65535 && T > 0 && T <= FORGE_TREE_MAX_TOKENS && V > 0 && verify_chunks(V) <= kVerifyNodes;
}

extern "C" size_t forge_verify_drafts_workspace_bytes(int B, int T, int V, int draft_probs) {
  return verify_sizes_ok(B, T, V) ? verify_ws(B, T, V, draft_probs != 0).bytes : 0;
}

extern "C" int forge_verify_drafts(int dtype, int B, int T, int V, const void* logits, int64_t s_logits_b,
                                   int64_t s_logits_t, const int64_t* tokens, int64_t s_tokens_b, const int32_t* parents,
                                   int64_t s_parents_b, const float* uniform, int64_t s_uniform_b, const float* temperatures,
                                   double temperature, int probs_dtype, const void* draft_probs, int64_t s_probs_b,
                                   int64_t s_probs_t, const int32_t* new_lens, int64_t* out, int32_t* path, int32_t* count,
                                   void* workspace, size_t workspace_bytes, int ws_flags, void* stream) {
  clear_error();
  if (dtype != FORGE_F32 && dtype != FORGE_BF16 && dtype != FORGE_F16) return set_error("unknown dtype code");
  if (B < 0 || T <= 0 || V <= 0) return set_error("bad sizes");
  if (B == 0) return 0;
  if (!verify_sizes_ok(B, T, V))
    return set_error("at most 65,535 rows of 1,024 nodes over 2^22 - 8 tokens");
  if (!logits || !tokens || !out || !path || !count) return set_error("null tensor pointer");
  if (!temperatures && !(temperature >= 0.0 && temperature <= 1e30)) return set_error("the temperature must be 0 or positive and finite");
  const bool warm = temperatures || temperature > 0.0;
  if (warm && !uniform) return set_error("temperatures need random numbers");
  if (!temperatures && temperature > 0.0 && temperature < 1e-30) return set_error("a positive temperature must be at least 1e-30");
  if (draft_probs && probs_dtype != FORGE_F32 && probs_dtype != dtype) return set_error("draft probabilities are fp32 or of the logits' type");
  for (const int64_t st : {s_logits_b, s_logits_t, s_tokens_b, s_parents_b, s_uniform_b, s_probs_b, s_probs_t})
    if (st < 0) return set_error("strides must not be negative");
  if (!warm) draft_probs = nullptr;   // (greedy: they decide nothing)
  const VerifyWs ws = verify_ws(B, T, V, draft_probs != nullptr);
  if (!workspace || workspace_bytes < ws.bytes) return set_error("workspace too small");
  if ((uintptr_t)workspace % 256) return set_error("the workspace must be 256-byte aligned");
  char* at = static_cast<char*>(workspace);
  VerifyParams p{};
  p.logits = logits; p.slb = s_logits_b; p.slt = s_logits_t;
  p.tokens = tokens; p.stb = s_tokens_b; p.parents = parents; p.spb = s_parents_b;
  p.uniform = uniform; p.sub = s_uniform_b; p.temps = temperatures; p.temperature = temperature;
  p.probs = draft_probs; p.sqb = s_probs_b; p.sqt = s_probs_t;
  if (!temperatures) {
    const Scale scale = scale_of(temperature > 0.0 ? temperature : 1.0);
    p.scale_hi = scale.hi; p.scale_lo = scale.lo;
  }
  p.new_lens = new_lens;
  p.B = B; p.T = T; p.V = V; p.C = verify_chunks(V);
  p.out = out; p.path = path; p.count = count;
  p.parts = reinterpret_cast<Part*>(at + ws.parts);
  // One launch saves an eager caller the time of making the second, 3 us; its walk waits for a counter and has half the
  // threads. us, two launches / one, 6 nodes over 32,768 tokens, greedy, recorded: 54 chunks 7.0 / 5.8, 108 7.2 / 6.3, 216 7.3 /
  // 7.7, 432 7.6 / 10.0, 1,296 8.4 / 17.4 (eager, 45 chunks 11.5 / 8.1). Sampled calls gain nothing (54 chunks 12.6 / 13.4, 216
  // 12.8 / 15.0; with probabilities, 198 16.5 / 18.7): without their walk the kernel has 38 registers in place of 181.
  if ((ws_flags & FORGE_WS_ZEROED) && !warm && T <= 2 * kScanThreads && (int64_t)p.C * T * B <= device_cus() / 2)
    p.counters = reinterpret_cast<unsigned*>(at);
  p.state = reinterpret_cast<State*>(at + ws.state);
  p.rest = reinterpret_cast<double*>(at + ws.rest);
  const hipStream_t s = (hipStream_t)stream;
  const bool wide = !draft_probs || probs_dtype == FORGE_F32;
  switch (dtype) {
    case FORGE_F32: return launch_verify<float, float>(p, s);
    case FORGE_BF16: return wide ? launch_verify<bf16, float>(p, s) : launch_verify<bf16, bf16>(p, s);
    default: return wide ? launch_verify<f16, float>(p, s) : launch_verify<f16, f16>(p, s);
  }
}
