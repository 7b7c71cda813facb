// Token routing from router scores, with what training needs of it and its gradient:
//
//   l[t,e]    = s[t,e]                             rule 0 (pure_torch_mlx/model.py:75-77)
//             = cap * tanh(s[t,e] / cap) / temp    rule 1 (sft_cot_bundle/scripts/model.py:318-329)
//   p[t,:]    = softmax(l[t,:]) over all experts,  lse[t] = log sum_e exp(l[t,e])
//   idx[t,:]  = the k largest scores, equal scores lowest expert first (tanh is increasing: the order of l is the order of s)
//   gates     = softmax over the k winners (rule 0),  p_j / (sum of the k winners' p + 1e-6) (rule 1)
//   counts[e] = number of slots that chose e,  f_e = counts[e] / (n k),  P_e = (1/n) sum_t p[t,e]
//   balance   = E * sum_e f_e P_e,   z = (1/n) sum_t lse[t]^2,   n = number of tokens that count
//
// A score of -inf switches an expert off for that token: it is never chosen and has no probability, under either rule.  Slots
// left over are empty (idx -1, gate 0).  A token that is masked, or that has no expert left, is all empty slots and counts
// nowhere; whatever its scores hold (NaN included) has no influence.  NaN in a token that counts sorts first, as in torch.topk,
// and makes its gates and the losses NaN.
//
// All arithmetic is fp32 whatever the scores' type; the logits of rule 1 are not rounded to the scores' type (the layer's own
// bf16 kernels do round them, as the reference's inference does; there the saturated ones tie).
//
// Gradient (f_e is a count and has none), with A_e = dB * E * f_e / n, and for the gates G = sum_j gate_j dgate_j:
//   dl[t,e] = p[t,e] * (A_e - sum_e' p A + (2/n) dz * lse - [rule 1] G * (1 - sum_j gate_j))
//             + [e chosen in slot j] gate_j * (dgate_j - G)
//   ds = dl (rule 0),  dl * sech^2(s / cap) / temp (rule 1)
#include "common.cuh"
#include "kernels.h"
#include "pair.cuh"
#include "ptx.cuh"

#include <cmath>

namespace tmoe {
namespace {

constexpr int kRouteThreads = 256;                       // backward
constexpr int kRouteWarps = kRouteThreads / 32;
// Forward: 512 where a lane holds 8 columns, so that fewer blocks leave partial rows; 256 where it holds more
constexpr int forward_threads(int NC) { return NC == 1 ? 512 : 256; }
constexpr int kRouteMaxExperts = 1024;

struct RouteArgs {
  const void *scores;
  const uint8_t *mask;       // [tokens] or nullptr
  int64_t tokens, stride;    // stride: elements between score rows
  int E, k, rule;
  float inv_cap, scale;      // logit = scale * tanh(score * inv_cap)
  int32_t *idx;              // [tokens, k]
  float *gates;              // [tokens, k]
  int32_t *counts;           // [E]
  float *losses;             // balance, z, n
  float *stats;              // [tokens, 2]: largest logit and sum of exp(logit - largest) of a token, or nullptr
  float *part_p;             // [blocks, E]
  int32_t *part_c;           // [blocks, E]
  float *part_zn;            // [blocks, 2]
  // backward
  const float *d_gates, *d_balance, *d_z;
  void *d_scores;            // [tokens, E]
};

// Selection keys: unsigned order = higher score first, equal scores lower column first.  Adding zero beforehand makes -0 equal to +0 and
// every NaN the positive one, which sorts above +inf.  -inf is the lowest key that a score can have and marks an expert that is off.
template <typename TS> struct Key;
template <> struct Key<bf16> {
  using type = uint32_t;   // order-preserving bits of the score << 16 | 0xffff - column
  // the keys of 8 scores, two to a word; low[i] = 0xffff - column of score i
  __device__ static __forceinline__ void make(const uint4 &v, const uint32_t (&low)[8], uint32_t (&key)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 c = __hadd2(*reinterpret_cast<const __nv_bfloat162 *>(&w[i]), __nv_bfloat162{__ushort_as_bfloat16(0), __ushort_as_bfloat16(0)});
      const uint32_t u = *reinterpret_cast<const uint32_t *>(&c);
      uint32_t neg;                                            // 0xffff in the halves whose sign is set
      asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(neg) : "r"(u));
      const uint32_t o = u ^ (neg | 0x80008000u);
      asm("mad.lo.u32 %0, %1, 65536, %2;" : "=r"(key[2 * i]) : "r"(o), "r"(low[2 * i]));
      key[2 * i + 1] = (o & 0xffff0000u) | low[2 * i + 1];
    }
  }
  __device__ static __forceinline__ bool empty(uint32_t key) { return (key >> 16) <= 0x7fu; }
  __device__ static __forceinline__ int col(uint32_t key) { return (int)(0xffffu - (key & 0xffffu)); }
  __device__ static __forceinline__ float value(uint32_t key) {
    const uint32_t u = key >> 16;
    return __uint_as_float(((u & 0x8000u) ? (u & 0x7fffu) : (~u & 0xffffu)) << 16);
  }
};
template <> struct Key<float> {
  using type = unsigned long long;   // order-preserving bits << 32 | 0xffffffff - column
  __device__ static __forceinline__ unsigned long long one(float v, int col) {
    const uint32_t b = __float_as_uint(__fadd_rn(v, 0.f));
    const uint32_t u = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return ((unsigned long long)u << 32) | (0xffffffffu - (uint32_t)col);
  }
  __device__ static __forceinline__ bool empty(unsigned long long key) { return (uint32_t)(key >> 32) <= 0x007fffffu; }
  __device__ static __forceinline__ int col(unsigned long long key) { return (int)(0xffffffffu - (uint32_t)key); }
  __device__ static __forceinline__ float value(unsigned long long key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
  }
};

// 4 keys of bf16 scores or 2 of fp32 ones behind a list keep its rows 16-byte aligned
template <typename TS> struct Lists { static constexpr int kPad = sizeof(TS) == 2 ? 4 : 2; };

// Slots that one lane of a token's G lanes keeps: slot j lives in lane j % G.  k is at most 16 and at most E <= 8 * G here.
template <int G> struct Slots { static constexpr int N = G <= 2 ? 8 : G == 4 ? 4 : G == 8 ? 2 : 1; };

// Reductions over the G lanes that share a token (all 32 lanes of the warp call them).
template <int G> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int G> __device__ __forceinline__ uint32_t group_max(uint32_t v) {
  if (G == 32) return __reduce_max_sync(0xffffffffu, v);
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int G> __device__ __forceinline__ unsigned long long group_max(unsigned long long v) {
  if (G == 32) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
    return ((unsigned long long)hi << 32) | lo;
  }
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    const unsigned long long w = __shfl_xor_sync(0xffffffffu, v, o);
    v = v > w ? v : w;
  }
  return v;
}

// The 8 scores of one lane in columns e0 .. e0 + 7, as pairs.  What is not there (column, token, masked token) reads as -inf.
template <typename TS, bool WIDE> struct Chunk;
template <bool WIDE> struct Chunk<bf16, WIDE> {
  uint4 v;
  __device__ __forceinline__ void load(const bf16 *row, int e0, int E, bool want) {
    v = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
    if (WIDE) {
      if (want && e0 < E) v = __ldg(reinterpret_cast<const uint4 *>(row + e0));   // E % 8 == 0
    } else if (want) {
      uint32_t h[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) h[q] = e0 + q < E ? (uint32_t)__bfloat16_as_ushort(row[e0 + q]) : 0xff80u;
      v = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
  }
  __device__ __forceinline__ void keys(int, const uint32_t (&low)[8], uint32_t (&key)[8]) const { Key<bf16>::make(v, low, key); }
  __device__ __forceinline__ f2 get(int j) const {
    const uint32_t w = j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w;
    return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
};
template <bool WIDE> struct Chunk<float, WIDE> {
  float v[8];
  __device__ __forceinline__ void load(const float *row, int e0, int E, bool want) {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = -INFINITY;
    if (WIDE) {
      if (want && e0 < E) {
        const float4 a = __ldg(reinterpret_cast<const float4 *>(row + e0)), b = __ldg(reinterpret_cast<const float4 *>(row + e0) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
      }
    } else if (want) {
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (e0 + q < E) v[q] = row[e0 + q];
    }
  }
  __device__ __forceinline__ void keys(int e0, const uint32_t (&)[8], unsigned long long (&key)[8]) const {
#pragma unroll
    for (int q = 0; q < 8; ++q) key[q] = Key<float>::one(v[q], e0 + q);
  }
  __device__ __forceinline__ f2 get(int j) const { return pair(v[2 * j], v[2 * j + 1]); }
};

// Capped, tempered logits l = scale * tanh(score * inv_cap) of N2 pairs and, for GRAD, their derivatives.  tanh up to 1 in magnitude is the Pade
// approximant x (945 + 105 x^2 + x^4) / (945 + 420 x^2 + 15 x^4) that Lambert's continued fraction gives (6e-8 off at 1, less below) with
// derivative 1 - t^2.  Beyond that, where 1 - t^2 cancels, both come from e = exp(-2|x|), and a score of -inf, which the cap would make a number
// again, is put back to -inf (the score itself is asked: a finite one over a small cap may overflow, and stays on).  That second part is
// skipped unless a lane of the warp may need it, told by the sum of its x^2 (paired FMAs; compares would go to the pipe that the selection
// fills): scores seldom reach the cap.  NaN stays NaN.
template <int N2, bool GRAD, typename SCORE>
__device__ __forceinline__ void cap_logits(const RouteArgs &a, const SCORE &score, f2 (&l)[N2], f2 (&d)[GRAD ? N2 : 1]) {
  f2 all = both(0.f);
#pragma unroll
  for (int j = 0; j < N2; ++j) {
    float da, db;
    const f2 x = mul2(score(j), both(a.inv_cap)), q = mul2(x, x);
    all = add2(all, q);
    split(fma2(q, fma2(q, both(15.f), both(420.f)), both(945.f)), da, db);
    const f2 t = mul2(mul2(x, fma2(q, add2(q, both(105.f)), both(945.f))), pair(fast_rcp(da), fast_rcp(db)));
    l[j] = mul2(t, both(a.scale));
    if (GRAD) d[j] = mul2(fma2(mul2(t, both(-1.f)), t, both(1.f)), both(a.scale * a.inv_cap));
  }
  if (!__any_sync(0xffffffffu, !(sum2(all) <= 1.f))) return;
#pragma unroll
  for (int j = 0; j < N2; ++j) {
    float s[2], lj[2], dj[2] = {0.f, 0.f};
    split(score(j), s[0], s[1]);
    split(l[j], lj[0], lj[1]);
    if (GRAD) split(d[j], dj[0], dj[1]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float v = s[h] * a.inv_cap, e = fast_exp2(fabsf(v) * (-2.f * kLog2e)), i = fast_rcp(1.f + e);
      if (fabsf(v) > 1.f) {
        lj[h] = s[h] == -INFINITY ? -INFINITY : copysignf(fmaf(-2.f * e, i, 1.f), v) * a.scale;
        dj[h] = 4.f * e * i * i * (a.scale * a.inv_cap);
      }
    }
    l[j] = pair(lj[0], lj[1]);
    if (GRAD) d[j] = pair(dj[0], dj[1]);
  }
}

__device__ __forceinline__ float fast_log2(float x) { float r; asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
constexpr float kLn2 = 0.6931471805599453f;

template <typename K> __device__ __forceinline__ void sort_two(K &a, K &b) {   // larger first
  const K hi = a > b ? a : b, lo = a > b ? b : a;
  a = hi; b = lo;
}
// The DEPTH largest of 8 keys, sorted, in the first places: all 8 by Batcher's network of 19 exchanges, or the first two by a
// tournament of pairs.
template <int DEPTH, typename K> __device__ __forceinline__ void sort_keys(K (&k)[8]) {
  sort_two(k[0], k[1]); sort_two(k[2], k[3]); sort_two(k[4], k[5]); sort_two(k[6], k[7]);
  if (DEPTH == 2) {
#pragma unroll
    for (int w = 2; w < 8; w *= 2) {
#pragma unroll
      for (int i = 0; i < 8; i += 2 * w) {
        const K lo = k[i] > k[i + w] ? k[i + w] : k[i], second = k[i + 1] > k[i + w + 1] ? k[i + 1] : k[i + w + 1];
        k[i] = k[i] > k[i + w] ? k[i] : k[i + w];
        k[i + 1] = lo > second ? lo : second;
      }
    }
    return;
  }
  sort_two(k[0], k[2]); sort_two(k[1], k[3]); sort_two(k[4], k[6]); sort_two(k[5], k[7]);
  sort_two(k[1], k[2]); sort_two(k[5], k[6]);
  sort_two(k[0], k[4]); sort_two(k[1], k[5]); sort_two(k[2], k[6]); sort_two(k[3], k[7]);
  sort_two(k[2], k[4]); sort_two(k[3], k[5]);
  sort_two(k[1], k[2]); sort_two(k[3], k[4]); sort_two(k[5], k[6]);
}

// The losses from the whole batch's sums; `dot` = sum_e counts_e * sum_t p[t, e]
__device__ __forceinline__ void write_losses(const RouteArgs &a, float dot, float z, float n) {
  const float inv = n > 0.f ? 1.f / n : 0.f;
  a.losses[0] = (float)a.E * (dot * inv) * (inv / (float)a.k);
  a.losses[1] = z * inv;
  a.losses[2] = n;
}

// G lanes per token, 8 columns of NC chunks each; a warp walks over tokens with all its groups, and every lane owns the same columns in all
// of them, so P is a sum in its registers; the choices are counted in shared memory (integers: the order of the atomics does not matter).
// A lane sorts its keys once and leaves them in shared memory, so that a round of the selection is one maximum over the lanes' heads and one
// load by the winner (shifting the list in registers instead kept the integer pipe busy for two thirds of the kernel).
// Blocks write one row of partial sums each; a block that is alone finishes the losses itself.  Bound by instruction issue (78 % of the
// slots): 131072 tokens x 256 bf16 scores, k = 8, rule 1 take 460 instructions a token, 67 us (and 9 us of losses), where reading the
// scores alone is 10 us; 32768 x 64, k = 2 take 11 us in all.
template <typename TS, int G, int NC, int DEPTH, bool WIDE>
__global__ void __launch_bounds__(forward_threads(NC)) route_kernel(const __grid_constant__ RouteArgs a) {
  using K = Key<TS>;
  constexpr int THREADS = forward_threads(NC), WARPS = THREADS / 32;
  constexpr int N = NC * 8, SL = Slots<G>::N, PER = 32 / G;   // columns and slots per lane, tokens per warp
  extern __shared__ __align__(16) float sm[];                 // the lanes' lists; after the walk [warps][G * N] sums
  __shared__ int hist[G * N];
  // a lane's NC lists of DEPTH keys, each with a 0 behind it (an exhausted list; equal to no chosen key but an exhausted row's), 16-byte rows
  constexpr int kPad = Lists<TS>::kPad;
  typename K::type *list = reinterpret_cast<typename K::type *>(sm) + (size_t)threadIdx.x * NC * (DEPTH + kPad);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gl = lane % G, grp = lane / G;
  ptx::griddep_launch_dependents();
  for (int i = threadIdx.x; i < G * N; i += THREADS) hist[i] = 0;
  __syncthreads();
  ptx::griddep_wait();   // the scores may come from the kernel before this one
  f2 acc[N / 2];
#pragma unroll
  for (int x = 0; x < N / 2; ++x) acc[x] = both(0.f);
  float zsum = 0.f, nsum = 0.f;
  uint32_t low[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    list[c * (DEPTH + kPad) + DEPTH] = 0;
#pragma unroll
    for (int q = 0; q < 8; ++q) low[c][q] = 0xffffu - (uint32_t)((c * G + gl) * 8 + q);
  }
  const int64_t step = (int64_t)gridDim.x * WARPS * PER;
  int64_t t = ((int64_t)blockIdx.x * WARPS + warp) * PER + grp;
  Chunk<TS, WIDE> next[NC];                                   // one token ahead
  auto fetch = [&](int64_t at) {
    const bool want = at < a.tokens && (!a.mask || a.mask[at]);
#pragma unroll
    for (int c = 0; c < NC; ++c) next[c].load((const TS *)a.scores + at * a.stride, (c * G + gl) * 8, a.E, want);
  };
  fetch(t);
  for (; t - grp < a.tokens; t += step) {
    const bool here = t < a.tokens;
    Chunk<TS, WIDE> s[NC];
    typename K::type head[NC], mine[SL], first = 0;
    const typename K::type *at[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) s[c] = next[c];
    fetch(t + step);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      typename K::type key[8];
      s[c].keys((c * G + gl) * 8, low[c], key);
      sort_keys<DEPTH>(key);
      typename K::type *to = list + c * (DEPTH + kPad);
#pragma unroll
      for (int q = 0; q < DEPTH; ++q) to[q] = key[q];
      head[c] = key[0];
      at[c] = to;
    }
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      mine[i] = 0;
      const int last = min(G, a.k - i * G);
#pragma unroll 4
      for (int jj = 0; jj < last; ++jj) {
        typename K::type m = head[0];
#pragma unroll
        for (int c = 1; c < NC; ++c) m = head[c] > m ? head[c] : m;
        m = group_max<G>(m);
        if (i == 0 && jj == 0) first = m;
        if (gl == jj) mine[i] = m;
#pragma unroll
        for (int c = 0; c < NC; ++c)
          if (head[c] == m) head[c] = *++at[c];
      }
    }
    const bool live = !K::empty(first);
    // logits of the chosen, then of all; the largest is the first chosen one's
    const auto pick = [&](int i) {
      return pair(K::value(mine[2 * i]), 2 * i + 1 < SL ? K::value(mine[2 * i + 1 < SL ? 2 * i + 1 : 0]) : 0.f);
    };
    const auto score = [&](int x) { return s[x / 4].get(x % 4); };
    f2 lm[(SL + 1) / 2], none[1];
    if (a.rule == 1) {
      cap_logits<(SL + 1) / 2, false>(a, pick, lm, none);
    } else {
#pragma unroll
      for (int i = 0; i < (SL + 1) / 2; ++i) lm[i] = pick(i);
    }
    float la, lb;
    split(lm[0], la, lb);
    const float lead = __shfl_sync(0xffffffffu, la, lane - gl);
    const float top = live ? lead : 0.f;
    f2 ex[N / 2], sum = both(0.f);
    if (a.rule == 1) {
      cap_logits<N / 2, false>(a, score, ex, none);
    } else {
#pragma unroll
      for (int x = 0; x < N / 2; ++x) ex[x] = score(x);
    }
#pragma unroll
    for (int x = 0; x < N / 2; ++x) {
      // (the difference first: exact for what matters, whatever the scores' size)
      split(mul2(add2(ex[x], both(-top)), both(kLog2e)), la, lb);
      ex[x] = pair(fast_exp2(la), fast_exp2(lb));
      sum = add2(sum, ex[x]);
    }
    const float den = group_sum<G>(sum2(sum));
    const float inv = live ? fast_rcp(den) : 0.f;
    if (live) {
#pragma unroll
      for (int x = 0; x < N / 2; ++x) acc[x] = fma2(ex[x], both(inv), acc[x]);
      if (gl == 0) {
        const float lse = fmaf(fast_log2(den), kLn2, top);
        zsum = fmaf(lse, lse, zsum);
        nsum += 1.f;
        if (a.stats) reinterpret_cast<float2 *>(a.stats)[t] = make_float2(top, den);
      }
    }
    float g[SL], total = 0.f;
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      split(lm[i / 2], la, lb);
      g[i] = K::empty(mine[i]) ? 0.f : fast_exp2(((i & 1 ? lb : la) - top) * kLog2e) * (a.rule == 1 ? inv : 1.f);
      total += g[i];
    }
    total = group_sum<G>(total);
    const float over = live ? fast_rcp(a.rule == 1 ? total + 1e-6f : total) : 0.f;
    if (here) {
#pragma unroll
      for (int i = 0; i < SL; ++i) {
        const int j = i * G + gl;
        if (j < a.k) {
          const bool full = !K::empty(mine[i]);
          const int col = K::col(mine[i]);
          a.idx[t * a.k + j] = full ? col : -1;
          a.gates[t * a.k + j] = g[i] * over;
          if (full) atomicAdd(&hist[col], 1);
        }
      }
    }
  }
  __syncthreads();   // the lists' memory is reused
  // the block's sums: groups of a warp by shuffles, then the warps in order
#pragma unroll
  for (int x = 0; x < N; ++x) {
    float lo, hi;
    split(acc[x / 2], lo, hi);
    float v = (x & 1) ? hi : lo;
#pragma unroll
    for (int o = G; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (grp == 0) sm[warp * (G * N) + ((x / 8) * G + gl) * 8 + x % 8] = v;
  }
  __shared__ float szn[WARPS][3];
  zsum = warp_sum(zsum); nsum = warp_sum(nsum);
  if (lane == 0) { szn[warp][0] = zsum; szn[warp][1] = nsum; }
  __syncthreads();
  const bool alone = gridDim.x == 1;
  float dot = 0.f;
  for (int e = threadIdx.x; e < a.E; e += THREADS) {
    float p = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) p += sm[w * (G * N) + e];
    if (alone) {
      a.counts[e] = hist[e];
      dot = fmaf((float)hist[e], p, dot);
    } else {
      a.part_p[(int64_t)blockIdx.x * a.E + e] = p;
      a.part_c[(int64_t)blockIdx.x * a.E + e] = hist[e];
    }
  }
  if (alone) {
    dot = warp_sum(dot);
    if (lane == 0) szn[warp][2] = dot;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    float z = 0.f, n = 0.f, d = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) { z += szn[w][0]; n += szn[w][1]; d += alone ? szn[w][2] : 0.f; }
    if (alone) {
      write_losses(a, d, z, n);
    } else {
      a.part_zn[blockIdx.x * 2] = z;
      a.part_zn[blockIdx.x * 2 + 1] = n;
    }
  }
}

// Sums the blocks' rows in a fixed order: counts, and the two losses.  One cluster of 8 blocks (one block alone took 45 us at 296 rows);
// each takes an eighth of the columns, `width` threads side by side on them and the others on other rows, and block 0 puts the eight
// parts of the balance loss together.
constexpr int kLossBlocks = 8, kLossThreads = 1024;
__global__ void __launch_bounds__(kLossThreads) route_losses_kernel(const __grid_constant__ RouteArgs a, int blocks, int width) {
  __shared__ float sp[kLossThreads];
  __shared__ int sc[kLossThreads];
  __shared__ float parts[kLossBlocks];
  __shared__ float red[kLossThreads / 32][3];
  ptx::griddep_wait();
  ptx::cluster_arrive();   // block 0 runs before anything is stored to its shared memory
  ptx::cluster_wait();
  const int rank = blockIdx.x, per = (a.E + kLossBlocks - 1) / kLossBlocks, e0 = rank * per;
  const int slices = kLossThreads / width, col = threadIdx.x % width, slice = threadIdx.x / width;
  float dot = 0.f;
  for (int c0 = 0; c0 < per; c0 += width) {
    const int e = e0 + c0 + col;
    const bool in = c0 + col < per && e < a.E && slice < slices;
    float p = 0.f;
    int c = 0;
    if (in) {
#pragma unroll 8
      for (int b = slice; b < blocks; b += slices) {
        p += a.part_p[(int64_t)b * a.E + e];
        c += a.part_c[(int64_t)b * a.E + e];
      }
    }
    sp[threadIdx.x] = p; sc[threadIdx.x] = c;
    __syncthreads();
    for (int n = slices / 2; n > 0; n >>= 1) {   // slices is a power of two
      if (slice < n) {
        sp[threadIdx.x] += sp[threadIdx.x + n * width];
        sc[threadIdx.x] += sc[threadIdx.x + n * width];
      }
      __syncthreads();
    }
    if (in && slice == 0) {
      a.counts[e] = sc[threadIdx.x];
      dot = fmaf((float)sc[threadIdx.x], sp[threadIdx.x], dot);
    }
    __syncthreads();
  }
  float z = 0.f, n = 0.f;
  if (rank == 0) {
    for (int b = threadIdx.x; b < blocks; b += kLossThreads) { z += a.part_zn[2 * b]; n += a.part_zn[2 * b + 1]; }
    z = warp_sum(z);
    n = warp_sum(n);
  }
  dot = warp_sum(dot);
  if ((threadIdx.x & 31) == 0) { red[threadIdx.x >> 5][0] = dot; red[threadIdx.x >> 5][1] = z; red[threadIdx.x >> 5][2] = n; }
  __syncthreads();
  if (threadIdx.x == 0) {
    dot = 0.f;
    for (int w = 0; w < kLossThreads / 32; ++w) dot += red[w][0];
    ptx::st_cluster_u32(ptx::mapa_u32(ptx::smem_u32(&parts[rank]), 0), __float_as_uint(dot));
  }
  __syncthreads();
  ptx::cluster_arrive();
  ptx::cluster_wait();
  if (rank == 0 && threadIdx.x == 0) {
    dot = z = n = 0.f;
    for (int r = 0; r < kLossBlocks; ++r) dot += parts[r];
    for (int w = 0; w < kLossThreads / 32; ++w) { z += red[w][1]; n += red[w][2]; }
    write_losses(a, dot, z, n);
  }
}

// p comes from the kept largest logit and sum, so a token needs one pass over its row.  The gates' parts of the gradient go through a row of shared memory
// per token: the lanes that hold slots put them at their columns, and every lane picks up its own eight.  131072 x 256 bf16, rule 1: 62 us for
// 147 MB, 327 instructions a token in about 65 % of the issue slots.
template <typename TS, int G, int NC, bool WIDE>
__global__ void __launch_bounds__(kRouteThreads, NC == 1 && G >= 16 ? 3 : 1) route_backward_kernel(const __grid_constant__ RouteArgs a) {
  constexpr int N = NC * 8, SL = Slots<G>::N, PER = 32 / G;
  extern __shared__ __align__(16) float sm[];   // [warps][PER][G * N]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gl = lane % G, grp = lane / G;
  float *row = sm + (warp * PER + grp) * (G * N);
  ptx::griddep_launch_dependents();
  for (int i = gl; i < G * N; i += G) row[i] = 0.f;
  __syncwarp();
  ptx::griddep_wait();
  const float n = a.losses[2], inv_n = n > 0.f ? 1.f / n : 0.f;
  const float z2 = a.d_z ? *a.d_z * 2.f * inv_n : 0.f;
  const float bal = a.d_balance ? *a.d_balance * ((float)a.E * inv_n) * (inv_n / (float)a.k) : 0.f;
  f2 A[N / 2];
#pragma unroll
  for (int x = 0; x < N / 2; ++x) {
    const int col = ((x / 4) * G + gl) * 8 + x % 4 * 2;
    A[x] = pair(col < a.E ? bal * (float)a.counts[col] : 0.f, col + 1 < a.E ? bal * (float)a.counts[col + 1] : 0.f);
  }
  const int64_t step = (int64_t)gridDim.x * kRouteWarps * PER;
  int64_t t = ((int64_t)blockIdx.x * kRouteWarps + warp) * PER + grp;
  struct Token {
    Chunk<TS, WIDE> s[NC];
    float2 stat;
    int col[SL];              // slots: lane j % G holds slot j
    float g[SL], dg[SL];
    bool live;                // a token that counts has a chosen expert in slot 0
  };
  auto fetch = [&](Token &n, int64_t at) {
    const bool want = at < a.tokens && (!a.mask || a.mask[at]);
#pragma unroll
    for (int c = 0; c < NC; ++c) n.s[c].load((const TS *)a.scores + at * a.stride, (c * G + gl) * 8, a.E, want);
    n.live = false;
    n.stat = make_float2(0.f, 1.f);
    if (want) {
      n.live = a.idx[at * a.k] >= 0;
      n.stat = reinterpret_cast<const float2 *>(a.stats)[at];   // (not used unless live)
    }
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const int j = i * G + gl;
      n.col[i] = -1; n.g[i] = n.dg[i] = 0.f;
      if (a.d_gates && want && j < a.k) {
        n.col[i] = a.idx[at * a.k + j];
        n.g[i] = a.gates[at * a.k + j];
        n.dg[i] = a.d_gates[at * a.k + j];
      }
    }
  };
  Token next;
  fetch(next, t);
  for (; t - grp < a.tokens; t += step) {
    const bool here = t < a.tokens;
    Token now = next;
    fetch(next, t + step);                       // one token ahead
    const float top = now.live ? now.stat.x : 0.f, den = now.live ? now.stat.y : 1.f;
    const float lse = now.live ? fmaf(fast_log2(den), kLn2, top) : 0.f, inv = fast_rcp(den);
    float inner = 0.f, total = 0.f;
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const bool full = now.live && (unsigned)now.col[i] < (unsigned)a.E;   // (an empty slot's gradient may be anything)
      now.col[i] = full ? now.col[i] : -1;
      now.g[i] = full ? now.g[i] : 0.f;
      now.dg[i] = full ? now.dg[i] : 0.f;
      inner = fmaf(now.g[i], now.dg[i], inner);
      total += now.g[i];
    }
    const auto score = [&](int x) { return now.s[x / 4].get(x % 4); };
    f2 p[N / 2], th[N / 2], dot2 = both(0.f);
    if (a.rule == 1) {
      cap_logits<N / 2, true>(a, score, p, th);
    } else {
#pragma unroll
      for (int x = 0; x < N / 2; ++x) { p[x] = score(x); th[x] = both(1.f); }
    }
#pragma unroll
    for (int x = 0; x < N / 2; ++x) {
      float la, lb;
      split(mul2(add2(p[x], both(-top)), both(kLog2e)), la, lb);
      p[x] = mul2(pair(fast_exp2(la), fast_exp2(lb)), both(inv));
      dot2 = fma2(p[x], A[x], dot2);
    }
    float base = z2 * lse - group_sum<G>(sum2(dot2));
    if (a.d_gates) {
      inner = group_sum<G>(inner);
      if (a.rule == 1) base -= inner * (1.f - group_sum<G>(total));
#pragma unroll
      for (int i = 0; i < SL; ++i)
        if (now.col[i] >= 0) row[now.col[i]] = now.g[i] * (now.dg[i] - inner);
      __syncwarp();
    }
    TS *dst = (TS *)a.d_scores + t * a.E;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int e0 = (c * G + gl) * 8;
      float4 r0 = make_float4(0.f, 0.f, 0.f, 0.f), r1 = r0;
      if (a.d_gates) { r0 = *reinterpret_cast<const float4 *>(row + e0); r1 = *reinterpret_cast<const float4 *>(row + e0 + 4); }
      const f2 chosen[4] = {pair(r0.x, r0.y), pair(r0.z, r0.w), pair(r1.x, r1.y), pair(r1.z, r1.w)};
      float f[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int x = c * 4 + j;
        split(mul2(fma2(p[x], add2(A[x], both(base)), chosen[j]), th[x]), f[2 * j], f[2 * j + 1]);
      }
      if (!now.live) {      // (whatever the upstream gradients hold)
#pragma unroll
        for (int q = 0; q < 8; ++q) f[q] = 0.f;
      }
      if (here) {
        if (WIDE) {
          if (e0 < a.E) {
            if (sizeof(TS) == 2) {
              *reinterpret_cast<uint4 *>(dst + e0) =
                  make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
            } else {
              reinterpret_cast<float4 *>(dst + e0)[0] = make_float4(f[0], f[1], f[2], f[3]);
              reinterpret_cast<float4 *>(dst + e0)[1] = make_float4(f[4], f[5], f[6], f[7]);
            }
          }
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (e0 + q < a.E) dst[e0 + q] = from_f32<TS>(f[q]);
        }
      }
    }
    if (a.d_gates) {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < SL; ++i)
        if (now.col[i] >= 0) row[now.col[i]] = 0.f;
      __syncwarp();
    }
  }
}

int lanes_per_token(int E) {
  int g = 1;
  while (g < 32 && g * 8 < E) g <<= 1;
  return g;
}
int route_blocks(int64_t tokens, int E, int sms) {
  const int64_t per = forward_threads((E + 255) / 256) / 32 * (32 / lanes_per_token(E));
  const int64_t want = (tokens + per - 1) / per, cap = (int64_t)sms * 2;
  return (int)(want < cap ? want : cap);
}

int check_route(const tmoe_route_t *p) {
  if (!p) return TMOE_ERR_NULL;
  if (p->dtype != TMOE_F32 && p->dtype != TMOE_BF16) return TMOE_ERR_DTYPE;
  if (p->tokens < 0 || p->tokens > ((int64_t)1 << 30) || p->n_experts <= 0 || p->top_k <= 0 || p->top_k > p->n_experts ||
      p->top_k > TMOE_MAX_TOPK || p->scores_stride < 0)
    return TMOE_ERR_SHAPE;
  if (p->n_experts > kRouteMaxExperts) return TMOE_ERR_UNSUPPORTED;
  if (p->router_mode != TMOE_ROUTER_TOPK_SOFTMAX && p->router_mode != TMOE_ROUTER_CAPPED_SOFTMAX) return TMOE_ERR_UNSUPPORTED;
  if (p->router_mode == TMOE_ROUTER_CAPPED_SOFTMAX) {
    const float cap = p->router_cap, temperature = p->router_temperature;
    if (!(cap > 0.f) || !(temperature > 0.f) || std::isinf(cap) || std::isinf(temperature)) return TMOE_ERR_SHAPE;
    // what the kernels multiply by; an infinite one would make NaN of a score of 0, a subnormal one has lost its digits
    if (!std::isnormal(1.f / cap) || !std::isnormal(cap / temperature) || !std::isnormal(1.f / temperature)) return TMOE_ERR_SHAPE;
  }
  if (p->tokens == 0) return TMOE_OK;
  if (!p->scores) return TMOE_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(p->scores) & (p->dtype == TMOE_F32 ? 3 : 1)) return TMOE_ERR_ALIGN;
  return TMOE_OK;
}

RouteArgs route_args(const tmoe_route_t &p) {
  RouteArgs a{};
  a.scores = p.scores; a.mask = p.token_mask; a.tokens = p.tokens; a.stride = p.scores_stride;
  a.E = p.n_experts; a.k = p.top_k; a.rule = p.router_mode;
  a.scale = a.inv_cap = 1.f;
  if (a.rule == 1) { a.inv_cap = 1.f / p.router_cap; a.scale = p.router_cap / p.router_temperature; }
  return a;
}

bool route_wide(const tmoe_route_t &p, const void *d_scores) {
  const int size = p.dtype == TMOE_F32 ? 4 : 2;
  return p.n_experts % 8 == 0 && (p.scores_stride * size) % 16 == 0 && !(reinterpret_cast<uintptr_t>(p.scores) & 15) &&
         !(reinterpret_cast<uintptr_t>(d_scores) & 15);
}

// The kernel for E experts: G lanes x NC pieces of 8 columns cover them
#define TMOE_ROUTE_G(CALL, TS, W)                              \
  (a.E <= 8     ? CALL(TS, 1, 1, W)                            \
   : a.E <= 16  ? CALL(TS, 2, 1, W)                            \
   : a.E <= 32  ? CALL(TS, 4, 1, W)                            \
   : a.E <= 64  ? CALL(TS, 8, 1, W)                            \
   : a.E <= 128 ? CALL(TS, 16, 1, W)                           \
   : a.E <= 256 ? CALL(TS, 32, 1, W)                           \
   : a.E <= 512 ? CALL(TS, 32, 2, W)                           \
                : CALL(TS, 32, 4, W))

template <typename TS, int G, int NC, int DEPTH, bool WIDE>
int launch_route_as(const RouteArgs &a, int blocks, cudaStream_t st) {
  constexpr int threads = forward_threads(NC);
  constexpr int lists = threads * NC * (DEPTH + Lists<TS>::kPad) * (int)sizeof(typename Key<TS>::type), sums = threads / 32 * G * NC * 8 * 4;
  constexpr int smem = lists > sums ? lists : sums;
  if (smem > 40 * 1024) {   // (with the static part above what needs no declaration)
    static std::atomic<uint64_t> opted{0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return TMOE_ERR_CUDA;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(opted.load(std::memory_order_relaxed) & bit)) {
      cudaFuncSetAttribute(route_kernel<TS, G, NC, DEPTH, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      opted.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  count_launch();
  return cuda_ok(launch_pdl(route_kernel<TS, G, NC, DEPTH, WIDE>, dim3((unsigned)blocks), dim3(threads), smem, st, a));
}
template <typename TS>
int launch_route(const RouteArgs &a, bool wide, int blocks, cudaStream_t st) {
#define TMOE_RT(TS_, G, NC, W) (a.k <= 2 ? launch_route_as<TS_, G, NC, 2, W>(a, blocks, st) : launch_route_as<TS_, G, NC, 8, W>(a, blocks, st))
  return wide ? TMOE_ROUTE_G(TMOE_RT, TS, true) : TMOE_ROUTE_G(TMOE_RT, TS, false);
#undef TMOE_RT
}
template <typename TS>
int launch_route_backward(const RouteArgs &a, bool wide, int blocks, cudaStream_t st) {
#define TMOE_RTB(TS_, G, NC, W) \
  cuda_ok(launch_pdl(route_backward_kernel<TS_, G, NC, W>, dim3((unsigned)blocks), dim3(kRouteThreads), kRouteWarps * 32 * NC * 8 * 4, st, a))
  count_launch();
  return wide ? TMOE_ROUTE_G(TMOE_RTB, TS, true) : TMOE_ROUTE_G(TMOE_RTB, TS, false);
#undef TMOE_RTB
}

// partial rows of the blocks; a block that is alone keeps none
int64_t route_ws(int blocks, int E) {
  return blocks == 1 ? 0 : align_up((int64_t)blocks * E * 4, 256) * 2 + align_up((int64_t)blocks * 8, 256);
}

}  // namespace
}  // namespace tmoe

using namespace tmoe;

extern "C" {

int64_t tmoe_route_workspace_bytes(const tmoe_route_t *p) {
  int rc = check_route(p);
  if (rc) return rc;
  // sized for up to 160 SMs, whatever device the sizing query runs on
  return route_ws(p->tokens ? route_blocks(p->tokens, p->n_experts, 160) : 1, p->n_experts);
}

int tmoe_route_tokens(const tmoe_route_t *p, int32_t *idx, float *gates, int32_t *counts, float *losses, float *stats, void *workspace,
                      int64_t workspace_bytes, void *stream) {
  int rc = check_route(p);
  if (rc) return rc;
  if (!counts || !losses) return TMOE_ERR_NULL;
  cudaStream_t st = (cudaStream_t)stream;
  if (p->tokens == 0) {
    rc = cuda_ok(cudaMemsetAsync(counts, 0, (size_t)p->n_experts * 4, st));
    return rc ? rc : cuda_ok(cudaMemsetAsync(losses, 0, 12, st));
  }
  if (!idx || !gates) return TMOE_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(idx) | reinterpret_cast<uintptr_t>(gates) | reinterpret_cast<uintptr_t>(counts) |
       reinterpret_cast<uintptr_t>(losses)) & 3)
    return TMOE_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(stats) & 7) return TMOE_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return TMOE_ERR_ALIGN;
  const int sms = current_device_sms();
  if (sms <= 0) return TMOE_ERR_CUDA;
  const int blocks = route_blocks(p->tokens, p->n_experts, sms < 160 ? sms : 160);
  const int64_t need = route_ws(blocks, p->n_experts);
  if (need && !workspace) return TMOE_ERR_NULL;
  if (workspace_bytes < need) return TMOE_ERR_WORKSPACE;
  RouteArgs a = route_args(*p);
  a.idx = idx; a.gates = gates; a.counts = counts; a.losses = losses; a.stats = stats;
  char *ws = reinterpret_cast<char *>(workspace);
  const int64_t one = align_up((int64_t)blocks * a.E * 4, 256);
  a.part_p = reinterpret_cast<float *>(ws);
  a.part_c = reinterpret_cast<int32_t *>(ws + one);
  a.part_zn = reinterpret_cast<float *>(ws + 2 * one);
  const bool wide = route_wide(*p, nullptr);
  rc = p->dtype == TMOE_F32 ? launch_route<float>(a, wide, blocks, st) : launch_route<bf16>(a, wide, blocks, st);
  if (rc || blocks == 1) return rc;
  const int per = (a.E + kLossBlocks - 1) / kLossBlocks;
  int width = 1;
  while (width < per && width < 64) width *= 2;
  rc = cuda_ok(launch_pdl_cluster(route_losses_kernel, dim3(kLossBlocks), dim3(kLossThreads), 0, st, kLossBlocks, a, blocks, width));
  count_launch();
  return rc;
}

int tmoe_route_tokens_backward(const tmoe_route_t *p, const int32_t *idx, const float *gates, const int32_t *counts,
                               const float *losses, const float *stats, const float *d_gates, const float *d_balance,
                               const float *d_z, void *d_scores, void *stream) {
  int rc = check_route(p);
  if (rc) return rc;
  if (p->tokens == 0) return TMOE_OK;
  if (!idx || !gates || !counts || !losses || !stats || !d_scores) return TMOE_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(idx) | reinterpret_cast<uintptr_t>(gates) | reinterpret_cast<uintptr_t>(counts) |
       reinterpret_cast<uintptr_t>(losses) | reinterpret_cast<uintptr_t>(d_gates) | reinterpret_cast<uintptr_t>(d_balance) |
       reinterpret_cast<uintptr_t>(d_z)) & 3)
    return TMOE_ERR_ALIGN;
  if ((reinterpret_cast<uintptr_t>(d_scores) & (p->dtype == TMOE_F32 ? 3 : 1)) || (reinterpret_cast<uintptr_t>(stats) & 7)) return TMOE_ERR_ALIGN;
  const int sms = current_device_sms();
  if (sms <= 0) return TMOE_ERR_CUDA;
  RouteArgs a = route_args(*p);
  a.idx = const_cast<int32_t *>(idx); a.gates = const_cast<float *>(gates); a.counts = const_cast<int32_t *>(counts);
  a.losses = const_cast<float *>(losses);
  a.stats = const_cast<float *>(stats);
  a.d_gates = d_gates; a.d_balance = d_balance; a.d_z = d_z; a.d_scores = d_scores;
  const bool wide = route_wide(*p, d_scores);
  const int64_t per = kRouteWarps * (32 / lanes_per_token(a.E)), want = (a.tokens + per - 1) / per;
  const int blocks = (int)(want < (int64_t)sms * 3 ? want : (int64_t)sms * 3);
  cudaStream_t st = (cudaStream_t)stream;
  return p->dtype == TMOE_F32 ? launch_route_backward<float>(a, wide, blocks, st) : launch_route_backward<bf16>(a, wide, blocks, st);
}

}  // extern "C"
