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
// maximum and sum); a block per row then walks, and draws within the one chunk that its number falls into. What a
// rejected child's probabilities leave has to be summed over a whole row of the vocabulary: a launch more, whose blocks
// end at once for the rows that need none, and whose last one draws.
#include <limits.h>

#include "common.h"
#include "forge_internal.h"

namespace forge {

constexpr int kVerifyChunk = 4096;  // elements of a row that a block takes
constexpr int kScanThreads = 256, kWalkThreads = 512;

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
  // workspace: each chunk's maximum, its first place, its sum; a row's state between launches; the sums of what is left
  double* part_z;  // [B][T][C]
  float* part_m;
  int32_t* part_i;
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
// exp((x - m) / temperature) to about 1e-15, exactly 1 at x = m, 0 for -inf: 2^t with t = k + f, k from the low bits of
// t + 1.5 2^52.
__device__ __forceinline__ double weight(float x, float m, Scale c) {
  if (m == -kNegInf) return x == m ? 1.0 : 0.0;   // infinite logits share the mass
  const double d = (double)x - (double)m;
  const double t = d * c.hi, lo = fma(d, c.lo, fma(d, c.hi, -t));
  const double big = t + 0x1.8p52, f = (t - (big - 0x1.8p52)) + lo;
  return t > -1100.0 ? ldexp(exp2_part(f), __double2loint(big)) : 0.0;   // (NaN: 0)
}

// Sum over the block, in one fixed order; every thread receives it. `lds`: one double a wave.
template <int THREADS> __device__ __forceinline__ double block_sum(double x, double* lds) {
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d, kWave);
  __syncthreads();   // (the last call's readers)
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = x;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) s += lds[w];
  return s;
}

// A row of logits, whose 16-byte pieces start `shift` elements before it; chunk c is elements c * 4096 - shift on.
template <typename T> struct Row {
  static constexpr int E = 16 / sizeof(T);
  const T* at;
  int V, shift;
  __device__ __forceinline__ Row(const T* p, int V) : at(p), V(V), shift((int)((uintptr_t)p % 16 / sizeof(T))) {}
  // the E elements from i on (a piece's first), -inf where there are none; a NaN counts as -inf
  __device__ __forceinline__ void piece(int i, float (&x)[E]) const {
    if (i >= 0 && i + E <= V) {
      unpack16<T>(load16(at + i), x);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = i + e >= 0 && i + e < V ? to_f32<T>(at[i + e]) : kNegInf;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = fmaxf(x[e], kNegInf);   // (of a NaN and a number the number)
  }
  __device__ __forceinline__ float one(int i) const {
    const float x = to_f32<T>(at[i]);
    return x == x ? x : kNegInf;
  }
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
template <typename T> __global__ __launch_bounds__(kScanThreads) void verify_scan_kernel(VerifyParams p) {
  const int c = blockIdx.x, t = blockIdx.y, b = blockIdx.z;
  if (t >= p.nodes(b)) return;
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
  const double heat = p.heat(b);
  double z = 0.0;
  int i = 0;
  if (!(heat > 0.0)) {
    i = p.V;
#pragma unroll
    for (int u = U - 1; u >= 0; --u)
#pragma unroll
      for (int e = E - 1; e >= 0; --e)
        if (x[u][e] == m) i = first + (u * kScanThreads + (int)threadIdx.x) * E + e;
    if (i < 0) i = 0;   // (-inf before the row's first element)
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
  if (threadIdx.x == 0) {
    const int64_t at = ((int64_t)b * p.T + t) * p.C + c;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) i = min(i, wi[w]), z += wz[w];
    p.part_m[at] = m;
    p.part_i[at] = i;
    p.part_z[at] = z;
  }
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
      double upto = own;
      for (int d = 1; d < kWave; d <<= 1) {
        const double y = __shfl_up(upto, d, kWave);
        if (lane >= d) upto += y;
      }
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
  double upto = own;
  for (int d = 1; d < kWave; d <<= 1) {
    const double y = __shfl_up(upto, d, kWave);
    if (lane >= d) upto += y;
  }
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
template <typename T> __device__ __forceinline__ int argmax_of(Row<T> row, float top) {
  __shared__ int first;
  if (threadIdx.x == 0) first = INT_MAX;
  __syncthreads();
  int i = threadIdx.x;
  while (i < row.V && row.one(i) != top) i += kWalkThreads;
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
  // the 8 elements from i0 on, a piece's first; 0 where there are none
  __device__ __forceinline__ void eight(int i0, double (&r)[8]) const {
    constexpr int E = Row<T>::E;
    float x[8], y[8];
#pragma unroll
    for (int u = 0; u < 8 / E; ++u) row.piece(i0 + u * E, reinterpret_cast<float(&)[E]>(x[u * E]));
    if (i0 >= 0 && i0 + 8 <= row.V && (uintptr_t)(q + i0) % 16 == 0) {
#pragma unroll
      for (int u = 0; u < 8 * (int)sizeof(Q) / 16; ++u) unpack16<Q>(load16(q + i0 + u * (16 / (int)sizeof(Q))), y + u * (16 / (int)sizeof(Q)));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = i0 + e >= 0 && i0 + e < row.V ? to_f32<Q>(q[i0 + e]) : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = of(x[e], (double)y[e]);
  }
};

constexpr int kVerifyNodes = FORGE_TREE_MAX_TOKENS;
static_assert(kVerifyChunk / kWalkThreads == 8, "a thread of the walk's draw holds eight elements");

// One block per row: from the chunks' numbers to its new tokens. Latency: the nodes' numbers, their tokens' logits and the one
// chunk that the draw falls into are read one after the other.
template <typename T, typename Q> __global__ __launch_bounds__(kWalkThreads) void verify_walk_kernel(VerifyParams p) {
  __shared__ float most[kVerifyNodes], us[kVerifyNodes];
  __shared__ double zs[kVerifyNodes], es[kVerifyNodes];
  __shared__ int args[kVerifyNodes], tok[kVerifyNodes], par[kVerifyNodes], child[kVerifyNodes], sib[kVerifyNodes];
  __shared__ bool yes[kVerifyNodes];
  __shared__ double lds[kWalkThreads / kWave];
  const int b = blockIdx.x, n = p.nodes(b), tid = threadIdx.x;
  int64_t* out = p.out + (int64_t)b * p.T;
  int32_t* path = p.path + (int64_t)b * p.T;
  const double heat = p.heat(b);
  const bool warm = heat > 0.0;
  const Scale s = row_scale(p, b);
  const Q* probs = static_cast<const Q*>(p.probs);
  const auto q_of = [&](int node, int v) { return (double)to_f32<Q>(probs[b * p.sqb + node * p.sqt + v]); };

  // each drafted token, its parent and the logit it is judged by (the loads go out before the chunks' numbers are met)
  constexpr int MINE = kVerifyNodes / kWalkThreads;
  float logit[MINE];
#pragma unroll
  for (int y = 0; y < MINE; ++y) {
    const int t = tid + y * kWalkThreads;
    logit[y] = kNegInf;
    if (t < p.T) {
      out[t] = -1;
      path[t] = t == 0 && n > 0 ? 0 : -1;
    }
    if (t >= n) continue;
    const int64_t x = p.tokens[b * p.stb + t];
    const int up = t == 0 ? -1 : p.parents ? p.parents[b * p.spb + t] : t - 1;
    const bool real = x >= 0 && x < p.V && up >= 0 && up < t;   // (others are passed over)
    tok[t] = real ? (int)x : -1;
    par[t] = real ? up : -1;
    us[t] = warm ? p.uniform[b * p.sub + t] : 0.0f;
    child[t] = p.T;
    if (real && warm) logit[y] = logits_row<T>(p, b, up).one((int)x);
  }
  if (probs && tid == 0) {
    p.state[b].left = 0;
    p.state[b].done = 0;
  }
  if (n == 0) {
    if (tid == 0) p.count[b] = 0;
    return;
  }

  // each node's maximum, argmax and sum: 16 lanes a node
  for (int t = tid / 16; t < n; t += kWalkThreads / 16) {
    const int64_t at = ((int64_t)b * p.T + t) * p.C;
    const int l = tid % 16;
    float m = kNegInf;
    int i = p.V;
    double z = 0.0;
    for (int c = l; c < p.C; c += 16) {   // (the running sum against the running maximum)
      const float mc = p.part_m[at + c];
      const int ic = p.part_i[at + c];
      const double zc = p.part_z[at + c];
      if (mc > m) {
        z = warm ? zc + (m > kNegInf ? z * weight(m, mc, s) : 0.0) : 0.0;
        m = mc;
        i = ic;
      } else if (mc == m) {   // (in rising order: the first stays)
        z += zc;
        i = min(i, ic);
      } else if (warm && mc > kNegInf) {
        z += zc * weight(mc, m, s);
      }
    }
    const float top = group_max<16>(m);
    if (m < top) i = p.V;
    if (warm) z = m > kNegInf ? z * weight(m, top, s) : 0.0;
    for (int d = 8; d; d >>= 1) {
      i = min(i, __shfl_xor(i, d, kWave));
      z += __shfl_xor(z, d, kWave);
    }
    if (l == 0) most[t] = top, args[t] = i, zs[t] = z;
  }
  __syncthreads();
#pragma unroll
  for (int y = 0; y < MINE; ++y) {
    const int t = tid + y * kWalkThreads;
    if (t >= n) continue;
    const int up = par[t];
    es[t] = warm && up >= 0 && most[up] > kNegInf ? weight(logit[y], most[up], s) : 0.0;
    if (!warm || probs || up < 0) continue;
    bool twice = false;   // an earlier sibling has the token
#pragma unroll 4
    for (int j = up + 1; j < t; ++j) twice |= par[j] == up && tok[j] == tok[t];
    yes[t] = !twice;
  }
  __syncthreads();

  // Who would be accepted if the walk came to its parent. With the drafter's probabilities that is known for first
  // children only: child[] are a node's first children, sib[] their next siblings. Else child[] are the accepted ones.
  for (int t = tid; t < n; t += kWalkThreads) {
    const int up = par[t];
    if (up < 0) continue;
    if (!warm) {
      if (tok[t] == args[up]) atomicMin(&child[up], t);
    } else if (probs) {
      yes[t] = us[t] * q_of(up, tok[t]) * zs[up] < es[t];
      atomicMin(&child[up], t);
      int next = p.T;
#pragma unroll 4
      for (int j = n - 1; j > t; --j) next = par[j] == up ? j : next;
      sib[t] = next;
    } else if (yes[t]) {
      double left = zs[up];
#pragma unroll 4
      for (int j = up + 1; j < t; ++j) left -= par[j] == up && yes[j] ? es[j] : 0.0;
      if (us[t] * fmax(left, 0.0) < es[t]) atomicMin(&child[up], t);
    }
  }
  __syncthreads();

  // the walk: every thread takes it
  int at = 0, count = 1;
  double taken = 0.0;
  while (true) {
    int t = child[at];
    if (t >= p.T) break;
    if (warm && probs && !yes[t]) {
      taken = zs[at];
      for (t = sib[t]; t < p.T; t = sib[t]) {
        const Rest<T, Q> rest(p, b, at, taken, most[at], s);
        double w = 0.0;
#pragma unroll 2
        for (int i = tid * 8 - rest.row.shift; i < p.V; i += kWalkThreads * 8) {
          double x[8];
          rest.eight(i, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) w += x[e];
        }
        w = block_sum<kWalkThreads>(w, lds);
        const double q = q_of(at, tok[t]);
        if (us[t] * q * w < es[t] - taken * q) break;
        taken += w;
      }
      if (t >= p.T) break;
      taken = 0.0;
    }
    if (tid == 0) {
      out[count - 1] = tok[t];
      path[count] = t;
    }
    at = t;
    ++count;
  }

  int token = warm ? 0 : args[at];
  if (warm && most[at] > kNegInf && taken > 0.0) {   // what the drafter's probabilities left is drawn from below
    if (tid == 0) p.state[b] = State{taken, most[at], at, count - 1, 1, 0};
    token = -1;
  } else if (warm && most[at] > kNegInf) {
    const Row<T> row = logits_row<T>(p, b, at);
    const int64_t base = ((int64_t)b * p.T + at) * p.C;
    const float top = most[at];
    double* masses = zs;   // (the nodes' are done with: [chunk])
    double* whole = es;    // a chunk's, before tokens were taken out
    int* gone = child;     // the rejected children's tokens, and the chunks they are in
    int* again = sib;
    __shared__ int ngone, nagain;
    __syncthreads();
    if (tid == 0) ngone = nagain = 0;
    for (int c = tid; c < p.C; c += kWalkThreads) {
      const float mc = p.part_m[base + c];
      masses[c] = mc > kNegInf ? p.part_z[base + c] * weight(mc, top, s) : 0.0;
    }
    __syncthreads();
    if (!probs) {
      for (int j = at + 1 + tid; j < n; j += kWalkThreads)
        if (par[j] == at && yes[j]) gone[atomicAdd(&ngone, 1)] = tok[j];
      __syncthreads();
      // a chunk that loses all but a thousandth of its sum is summed again: the difference could leave what is not there
      for (int g = tid; g < ngone; g += kWalkThreads) {
        const int c = (gone[g] + row.shift) / kVerifyChunk;
        double out_of = 0.0;
        bool first = true;
        for (int h = 0; h < ngone; ++h) {
          if ((gone[h] + row.shift) / kVerifyChunk != c) continue;
          first &= h >= g;
          out_of += weight(row.one(gone[h]), top, s);
        }
        if (!first) continue;
        const double left = masses[c] - out_of;
        if (left < masses[c] * 0x1p-10) again[atomicAdd(&nagain, 1)] = c;
        else masses[c] = left;
      }
    }
    __syncthreads();
    const auto eight = [&](int i0, double (&r)[8]) {   // the weights of the 8 elements from i0 on, without rejected ones
      constexpr int E = Row<T>::E;
      float x[8];
#pragma unroll
      for (int u = 0; u < 8 / E; ++u) row.piece(i0 + u * E, reinterpret_cast<float(&)[E]>(x[u * E]));
      unsigned cut = 0;
      for (int g = 0; g < ngone; ++g)
        if ((unsigned)(gone[g] - i0) < 8) cut |= 1u << (gone[g] - i0);
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = cut >> e & 1 ? 0.0 : weight(x[e], top, s);
    };
    double x[8];
    for (int g = 0; g < nagain; ++g) {
      const int c = again[g];
      eight(c * kVerifyChunk - row.shift + tid * 8, x);
      double w = 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) w += x[e];
      w = block_sum<kWalkThreads>(w, lds);
      if (tid == 0) masses[c] = w;
    }
    __syncthreads();
    double total = 0.0;
    for (int c = tid; c < p.C; c += kWalkThreads) total += masses[c];
    total = block_sum<kWalkThreads>(total, lds);
    if (total > 0.0) {
      const Found f = find_chunk(p.C, us[0] * total, [&](int c) { return masses[c]; });
      const int first = f.c * kVerifyChunk - row.shift;
      eight(first + tid * 8, x);
      token = find_element<kWalkThreads>(first, f.target, x);
    } else {
      token = argmax_of(row, top);
    }
  }
  if (tid == 0) {
    if (token >= 0) out[count - 1] = token;
    p.count[b] = count;
  }
}

// Sums over blocks on several XCDs, whose caches are their own: written past them, counted, and read by the block that
// counts last.
__device__ __forceinline__ void store_agent(double* p, double x) {
  __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double load_agent(const double* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// What the drafter's probabilities left of a row, chunk by chunk; a row's last block draws from it.
template <typename T, typename Q> __global__ __launch_bounds__(kWalkThreads) void verify_rest_kernel(VerifyParams p) {
  __shared__ double lds[kWalkThreads / kWave];
  __shared__ bool last;
  const int c = blockIdx.x, b = blockIdx.y;
  const State st = p.state[b];
  if (!st.left) return;
  const Rest<T, Q> rest(p, b, st.node, st.taken, st.most, row_scale(p, b));
  double* sums = p.rest + (int64_t)b * p.C;
  double x[8], w = 0.0;
  rest.eight(c * kVerifyChunk - rest.row.shift + (int)threadIdx.x * 8, x);
#pragma unroll
  for (int e = 0; e < 8; ++e) w += x[e];
  w = block_sum<kWalkThreads>(w, lds);
  if (threadIdx.x == 0) {
    store_agent(sums + c, w);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    last = atomicAdd(&p.state[b].done, 1u) == (unsigned)p.C - 1;
  }
  __syncthreads();
  if (!last) return;
  double total = 0.0;
  for (int i = threadIdx.x; i < p.C; i += kWalkThreads) total += load_agent(sums + i);
  total = block_sum<kWalkThreads>(total, lds);
  int token;
  if (total > 0.0) {
    const Found f = find_chunk(p.C, (double)p.uniform[b * p.sub] * total, [&](int i) { return load_agent(sums + i); });
    const int first = f.c * kVerifyChunk - rest.row.shift;
    rest.eight(first + (int)threadIdx.x * 8, x);
    token = find_element<kWalkThreads>(first, f.target, x);
  } else {
    token = argmax_of(rest.row, st.most);
  }
  if (threadIdx.x == 0) p.out[(int64_t)b * p.T + st.at] = token;
}

struct VerifyWs {
  size_t z, m, i, state, rest, bytes;
};
static int verify_chunks(int V) { return (V + 7 + kVerifyChunk - 1) / kVerifyChunk; }   // (a row may start inside a piece)
static VerifyWs verify_ws(int B, int T, int V, bool probs) {
  const auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  const size_t n = (size_t)B * T * verify_chunks(V);
  VerifyWs w{};
  w.m = up(n * sizeof(double));
  w.i = w.m + up(n * sizeof(float));
  w.state = w.i + up(n * sizeof(int32_t));
  w.rest = w.state + (probs ? up((size_t)B * sizeof(State)) : 0);
  w.bytes = w.rest + (probs ? up((size_t)B * verify_chunks(V) * sizeof(double)) : 0);
  return w;
}

template <typename T, typename Q> static int launch_verify(const VerifyParams& p, hipStream_t s) {
  hipLaunchKernelGGL((verify_scan_kernel<T>), dim3(p.C, p.T, p.B), dim3(kScanThreads), 0, s, p);
  int st = check_launch();
  if (st) return st;
  hipLaunchKernelGGL((verify_walk_kernel<T, Q>), dim3(p.B), dim3(kWalkThreads), 0, s, p);
  st = check_launch();
  if (st || !p.probs) return st;
  hipLaunchKernelGGL((verify_rest_kernel<T, Q>), dim3(p.C, p.B), dim3(kWalkThreads), 0, s, p);
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
                                   void* workspace, size_t workspace_bytes, void* stream) {
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
  p.part_z = reinterpret_cast<double*>(at);
  p.part_m = reinterpret_cast<float*>(at + ws.m);
  p.part_i = reinterpret_cast<int32_t*>(at + ws.i);
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
