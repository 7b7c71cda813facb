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
#include "ptx.cuh"

#include <cmath>

namespace tmoe {
namespace {

constexpr int kRouteThreads = 256;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kRouteMaxExperts = 1024;

struct RouteArgs {
  const void *scores;
  const uint8_t *mask;       // [tokens] or nullptr
  int64_t tokens, stride;    // stride: elements between score rows
  int E, k, rule;
  float cap, inv_cap, inv_temp;
  int32_t *idx;              // [tokens, k]
  float *gates;              // [tokens, k]
  int32_t *counts;           // [E]
  float *losses;             // balance, z, n
  float *part_p;             // [blocks, E]
  int32_t *part_c;           // [blocks, E]
  float *part_zn;            // [blocks, 2]
  // backward
  const float *d_gates, *d_balance, *d_z;
  void *d_scores;            // [tokens, E]
};

// Selection keys: unsigned order = higher score first, equal scores lower column first; 0 = switched off.
template <typename TS> struct Key;
template <> struct Key<bf16> {
  using type = uint32_t;
  __device__ static __forceinline__ uint32_t make(float v, int col) {
    uint32_t b = __float_as_uint(v) >> 16;
    if ((b & 0x7fffu) > 0x7f80u) b = 0x7fffu;            // NaN above everything
    if (b == 0xff80u) return 0u;                         // -inf
    if (b == 0x8000u) b = 0u;                            // -0 equals +0
    const uint32_t u = (b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u);
    return (u << 16) | (0xffffu - (uint32_t)col);
  }
  __device__ static __forceinline__ int col(uint32_t key) { return (int)(0xffffu - (key & 0xffffu)); }
  __device__ static __forceinline__ float value(uint32_t key) {
    const uint32_t u = key >> 16;
    return __uint_as_float(((u & 0x8000u) ? (u & 0x7fffu) : (~u & 0xffffu)) << 16);
  }
};
template <> struct Key<float> {
  using type = unsigned long long;
  __device__ static __forceinline__ unsigned long long make(float v, int col) {
    uint32_t b = __float_as_uint(v);
    if ((b & 0x7fffffffu) > 0x7f800000u) b = 0x7fffffffu;
    if (b == 0xff800000u) return 0ull;
    if (b == 0x80000000u) b = 0u;
    const uint32_t u = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return ((unsigned long long)u << 32) | (0xffffffffu - (uint32_t)col);
  }
  __device__ static __forceinline__ int col(unsigned long long key) { return (int)(0xffffffffu - (uint32_t)key); }
  __device__ static __forceinline__ float value(unsigned long long key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
  }
};

// Slots that one lane of a token's G lanes keeps: slot j lives in lane j % G.  k is at most 16 and at most E <= 8 * G here.
template <int G> struct Slots { static constexpr int N = G <= 2 ? 8 : G == 4 ? 4 : G == 8 ? 2 : 1; };

// Reductions over the G lanes that share a token (all 32 lanes of the warp call them).
template <int G> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int G> __device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
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

// The 8 * NC scores of one lane: columns (c * G + gl) * 8 + q.  Columns beyond E read as -inf.
template <typename TS, int G, int NC, bool WIDE>
__device__ __forceinline__ void load_scores(const TS *row, int gl, int E, bool want, float (&s)[NC * 8]) {
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int e0 = (c * G + gl) * 8;
    if (WIDE) {
      if (want && e0 < E) {   // E % 8 == 0
        if (sizeof(TS) == 2) {
          const uint4 v = __ldg(reinterpret_cast<const uint4 *>(row + e0));
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int q = 0; q < 8; ++q) s[c * 8 + q] = __uint_as_float((q & 1) ? (w[q >> 1] & 0xffff0000u) : (w[q >> 1] << 16));
        } else {
          const float4 a = __ldg(reinterpret_cast<const float4 *>(row + e0)), b = __ldg(reinterpret_cast<const float4 *>(row + e0) + 1);
          const float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
          for (int q = 0; q < 8; ++q) s[c * 8 + q] = f[q];
        }
      } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) s[c * 8 + q] = -INFINITY;
      }
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) s[c * 8 + q] = (want && e0 + q < E) ? to_f32(row[e0 + q]) : -INFINITY;
    }
  }
}

__device__ __forceinline__ float logit_of(const RouteArgs &a, float s) {
  return a.rule == 1 ? a.cap * tanhf(s * a.inv_cap) * a.inv_temp : s;
}

// G lanes per token, a warp walks over tokens with all its groups; every lane owns the same columns in all of them, so P and the
// counts are sums in its registers.  Blocks write one row of partial sums each.
template <typename TS, int G, int NC, bool WIDE>
__global__ void __launch_bounds__(kRouteThreads) route_kernel(const __grid_constant__ RouteArgs a) {
  using K = Key<TS>;
  constexpr int N = NC * 8, SL = Slots<G>::N;          // columns and slots per lane
  extern __shared__ float sm[];                        // [warps][G * N]: P, then the counts
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gl = lane % G, grp = lane / G;
  constexpr int PER = 32 / G;
  float acc[N];
  int cnt[N];
#pragma unroll
  for (int x = 0; x < N; ++x) { acc[x] = 0.f; cnt[x] = 0; }
  float zsum = 0.f, nsum = 0.f;
  for (int64_t t0 = ((int64_t)blockIdx.x * kRouteWarps + warp) * PER; t0 < a.tokens; t0 += (int64_t)gridDim.x * kRouteWarps * PER) {
    const int64_t t = t0 + grp;
    const bool here = t < a.tokens;
    const bool want = here && (!a.mask || a.mask[t]);
    float s[N];
    load_scores<TS, G, NC, WIDE>((const TS *)a.scores + t * a.stride, gl, a.E, want, s);
    typename K::type key[N];
#pragma unroll
    for (int x = 0; x < N; ++x) key[x] = K::make(s[x], ((x / 8) * G + gl) * 8 + x % 8);
    typename K::type mine[SL];
    float top = 0.f;
    bool live = false;
#pragma unroll
    for (int i = 0; i < SL; ++i) mine[i] = 0;
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const int last = min(G, a.k - i * G);
#pragma unroll 1
      for (int jj = 0; jj < last; ++jj) {
        typename K::type m = key[0];
#pragma unroll
        for (int x = 1; x < N; ++x) m = key[x] > m ? key[x] : m;
        m = group_max<G>(m);
        if (i == 0 && jj == 0) { live = m != 0; top = live ? logit_of(a, K::value(m)) : 0.f; }
        if (gl == jj) mine[i] = m;
#pragma unroll
        for (int x = 0; x < N; ++x) key[x] = key[x] == m ? 0 : key[x];
      }
    }
    float den = 0.f;
#pragma unroll
    for (int x = 0; x < N; ++x) {
      const bool on = s[x] != -INFINITY;
      cnt[x] += (on && key[x] == 0) ? 1 : 0;
      s[x] = on ? expf(logit_of(a, s[x]) - top) : 0.f;
      den += s[x];
    }
    den = group_sum<G>(den);
    const float inv = live ? 1.f / den : 0.f;
    if (live) {
#pragma unroll
      for (int x = 0; x < N; ++x) acc[x] = fmaf(s[x], inv, acc[x]);
      if (gl == 0) {
        const float lse = top + logf(den);
        zsum = fmaf(lse, lse, zsum);
        nsum += 1.f;
      }
    }
    float g[SL], sum = 0.f;
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      g[i] = mine[i] != 0 ? expf(logit_of(a, K::value(mine[i])) - top) : 0.f;
      if (a.rule == 1) g[i] *= inv;
      sum += g[i];
    }
    sum = group_sum<G>(sum);
    if (a.rule == 1) sum += 1e-6f;
    if (here) {
#pragma unroll
      for (int i = 0; i < SL; ++i) {
        const int j = i * G + gl;
        if (j < a.k) {
          a.idx[t * a.k + j] = mine[i] != 0 ? K::col(mine[i]) : -1;
          a.gates[t * a.k + j] = mine[i] != 0 ? g[i] / sum : 0.f;
        }
      }
    }
  }
  // the block's sums: groups of a warp by shuffles, then the warps in order
#pragma unroll
  for (int x = 0; x < N; ++x) {
#pragma unroll
    for (int o = G; o < 32; o <<= 1) {
      acc[x] += __shfl_xor_sync(0xffffffffu, acc[x], o);
      cnt[x] += __shfl_xor_sync(0xffffffffu, cnt[x], o);
    }
    if (grp == 0) sm[warp * (G * N) + ((x / 8) * G + gl) * 8 + x % 8] = acc[x];
  }
  __shared__ float szn[kRouteWarps][2];
  zsum = warp_sum(zsum); nsum = warp_sum(nsum);
  if (lane == 0) { szn[warp][0] = zsum; szn[warp][1] = nsum; }
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += kRouteThreads) {
    float p = 0.f;
#pragma unroll
    for (int w = 0; w < kRouteWarps; ++w) p += sm[w * (G * N) + e];
    a.part_p[(int64_t)blockIdx.x * a.E + e] = p;
  }
  __syncthreads();
  int *si = reinterpret_cast<int *>(sm);
  if (grp == 0) {
#pragma unroll
    for (int x = 0; x < N; ++x) si[warp * (G * N) + ((x / 8) * G + gl) * 8 + x % 8] = cnt[x];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += kRouteThreads) {
    int c = 0;
#pragma unroll
    for (int w = 0; w < kRouteWarps; ++w) c += si[w * (G * N) + e];
    a.part_c[(int64_t)blockIdx.x * a.E + e] = c;
  }
  if (threadIdx.x < 2) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kRouteWarps; ++w) v += szn[w][threadIdx.x];
    a.part_zn[blockIdx.x * 2 + threadIdx.x] = v;
  }
}

// Sums the blocks' rows in order: counts, and the two losses.  One block.
__global__ void __launch_bounds__(1024) route_losses_kernel(const __grid_constant__ RouteArgs a, int blocks) {
  __shared__ float red[32];
  float dot = 0.f;
  for (int e = threadIdx.x; e < a.E; e += 1024) {
    float p = 0.f; int c = 0;
    for (int b = 0; b < blocks; ++b) { p += a.part_p[(int64_t)b * a.E + e]; c += a.part_c[(int64_t)b * a.E + e]; }
    a.counts[e] = c;
    dot = fmaf((float)c, p, dot);
  }
  dot = warp_sum(dot);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = dot;
  __syncthreads();
  if (threadIdx.x == 0) {
    float z = 0.f, n = 0.f;
    for (int b = 0; b < blocks; ++b) { z += a.part_zn[2 * b]; n += a.part_zn[2 * b + 1]; }
    dot = 0.f;
    for (int w = 0; w < 32; ++w) dot += red[w];
    const float inv = n > 0.f ? 1.f / n : 0.f;
    a.losses[0] = (float)a.E * (dot * inv) * (inv / (float)a.k);
    a.losses[1] = z * inv;
    a.losses[2] = n;
  }
}

template <typename TS, int G, int NC, bool WIDE>
__global__ void __launch_bounds__(kRouteThreads) route_backward_kernel(const __grid_constant__ RouteArgs a) {
  constexpr int N = NC * 8, SL = Slots<G>::N, PER = 32 / G;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gl = lane % G, grp = lane / G;
  const float n = a.losses[2], inv_n = n > 0.f ? 1.f / n : 0.f;
  const float z2 = a.d_z ? *a.d_z * 2.f * inv_n : 0.f;
  const float bal = a.d_balance ? *a.d_balance * ((float)a.E * inv_n) * (inv_n / (float)a.k) : 0.f;
  float A[N];
#pragma unroll
  for (int x = 0; x < N; ++x) {
    const int col = ((x / 8) * G + gl) * 8 + x % 8;
    A[x] = col < a.E ? bal * (float)a.counts[col] : 0.f;
  }
  for (int64_t t0 = ((int64_t)blockIdx.x * kRouteWarps + warp) * PER; t0 < a.tokens; t0 += (int64_t)gridDim.x * kRouteWarps * PER) {
    const int64_t t = t0 + grp;
    const bool here = t < a.tokens;
    const bool want = here && (!a.mask || a.mask[t]);
    float s[N], th[N];
    load_scores<TS, G, NC, WIDE>((const TS *)a.scores + t * a.stride, gl, a.E, want, s);
    float top = -INFINITY;
    bool any = false;
#pragma unroll
    for (int x = 0; x < N; ++x) {
      const bool on = s[x] != -INFINITY;
      any |= on;
      if (a.rule == 1) {
        // sech^2 from exp(-2|s/cap|): no cancellation where the cap saturates
        const float e = expf(-2.f * fabsf(s[x] * a.inv_cap)), d = 1.f / (1.f + e);
        th[x] = on ? 4.f * e * d * d * a.inv_temp : 0.f;
        s[x] = on ? logit_of(a, s[x]) : -INFINITY;
      } else {
        th[x] = on ? 1.f : 0.f;
      }
      top = fmaxf(top, s[x]);
    }
    top = group_max<G>(top);
    const bool live = (__ballot_sync(0xffffffffu, any) >> (grp * G) & (G == 32 ? 0xffffffffu : ((1u << G) - 1u))) != 0u;
    float den = 0.f, dot = 0.f;
#pragma unroll
    for (int x = 0; x < N; ++x) {
      s[x] = s[x] != -INFINITY ? expf(s[x] - top) : 0.f;
      den += s[x];
    }
    den = group_sum<G>(den);
    const float inv = live ? 1.f / den : 0.f;
    const float lse = live ? top + logf(den) : 0.f;
#pragma unroll
    for (int x = 0; x < N; ++x) {
      s[x] *= inv;
      dot = fmaf(s[x], A[x], dot);
    }
    dot = group_sum<G>(dot);
    // the gates' part: lane j % G holds slot j
    int col[SL];
    float val[SL], inner = 0.f, total = 0.f;
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const int j = i * G + gl;
      col[i] = -1; val[i] = 0.f;
      if (a.d_gates && want && j < a.k) {
        col[i] = a.idx[t * a.k + j];
        if (col[i] >= 0) {
          const float g = a.gates[t * a.k + j], dg = a.d_gates[t * a.k + j];
          inner = fmaf(g, dg, inner);
          total += g;
          val[i] = g;
        }
      }
    }
    inner = group_sum<G>(inner);
    total = group_sum<G>(total);
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const int j = i * G + gl;
      if (col[i] >= 0) val[i] *= a.d_gates[t * a.k + j] - inner;
    }
    const float base = z2 * lse - dot - (a.rule == 1 ? inner * (1.f - total) : 0.f);
#pragma unroll
    for (int x = 0; x < N; ++x) s[x] *= A[x] + base;
    if (a.d_gates) {
#pragma unroll
      for (int i = 0; i < SL; ++i) {
        const int last = min(G, a.k - i * G);
#pragma unroll 1
        for (int jj = 0; jj < last; ++jj) {
          const int cj = __shfl_sync(0xffffffffu, col[i], grp * G + jj);
          const float vj = __shfl_sync(0xffffffffu, val[i], grp * G + jj);
#pragma unroll
          for (int x = 0; x < N; ++x) s[x] += cj == ((x / 8) * G + gl) * 8 + x % 8 ? vj : 0.f;
        }
      }
    }
#pragma unroll
    for (int x = 0; x < N; ++x) s[x] = th[x] != 0.f ? s[x] * th[x] : 0.f;
    if (here) {
      TS *dst = (TS *)a.d_scores + t * a.E;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int e0 = (c * G + gl) * 8;
        if (WIDE) {
          if (e0 < a.E) {
            if (sizeof(TS) == 2) {
              *reinterpret_cast<uint4 *>(dst + e0) = make_uint4(pack_bf16x2(s[c * 8], s[c * 8 + 1]), pack_bf16x2(s[c * 8 + 2], s[c * 8 + 3]),
                                                                pack_bf16x2(s[c * 8 + 4], s[c * 8 + 5]), pack_bf16x2(s[c * 8 + 6], s[c * 8 + 7]));
            } else {
              reinterpret_cast<float4 *>(dst + e0)[0] = make_float4(s[c * 8], s[c * 8 + 1], s[c * 8 + 2], s[c * 8 + 3]);
              reinterpret_cast<float4 *>(dst + e0)[1] = make_float4(s[c * 8 + 4], s[c * 8 + 5], s[c * 8 + 6], s[c * 8 + 7]);
            }
          }
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (e0 + q < a.E) dst[e0 + q] = from_f32<TS>(s[c * 8 + q]);
        }
      }
    }
  }
}

int lanes_per_token(int E) {
  int g = 1;
  while (g < 32 && g * 8 < E) g <<= 1;
  return g;
}
int route_blocks(int64_t tokens, int E, int sms) {
  const int64_t per = kRouteWarps * (32 / lanes_per_token(E));
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
  if (p->router_mode == TMOE_ROUTER_CAPPED_SOFTMAX &&
      (!(p->router_cap > 0.f) || !(p->router_temperature > 0.f) || std::isinf(p->router_cap) || std::isinf(p->router_temperature)))
    return TMOE_ERR_SHAPE;
  if (p->tokens == 0) return TMOE_OK;
  if (!p->scores) return TMOE_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(p->scores) & (p->dtype == TMOE_F32 ? 3 : 1)) return TMOE_ERR_ALIGN;
  return TMOE_OK;
}

RouteArgs route_args(const tmoe_route_t &p) {
  RouteArgs a{};
  a.scores = p.scores; a.mask = p.token_mask; a.tokens = p.tokens; a.stride = p.scores_stride;
  a.E = p.n_experts; a.k = p.top_k; a.rule = p.router_mode;
  a.cap = a.inv_cap = a.inv_temp = 1.f;
  if (a.rule == 1) { a.cap = p.router_cap; a.inv_cap = 1.f / p.router_cap; a.inv_temp = 1.f / p.router_temperature; }
  return a;
}

bool route_wide(const tmoe_route_t &p, const void *d_scores) {
  const int size = p.dtype == TMOE_F32 ? 4 : 2;
  return p.n_experts % 8 == 0 && (p.scores_stride * size) % 16 == 0 && !(reinterpret_cast<uintptr_t>(p.scores) & 15) &&
         !(reinterpret_cast<uintptr_t>(d_scores) & 15);
}

// The kernel for E experts: G lanes x NC pieces of 8 columns cover them
#define TMOE_ROUTE_G(CALL, TS, W)                \
  do {                                           \
    if (a.E <= 8) CALL(TS, 1, 1, W);             \
    else if (a.E <= 16) CALL(TS, 2, 1, W);       \
    else if (a.E <= 32) CALL(TS, 4, 1, W);       \
    else if (a.E <= 64) CALL(TS, 8, 1, W);       \
    else if (a.E <= 128) CALL(TS, 16, 1, W);     \
    else if (a.E <= 256) CALL(TS, 32, 1, W);     \
    else if (a.E <= 512) CALL(TS, 32, 2, W);     \
    else CALL(TS, 32, 4, W);                     \
  } while (0)

template <typename TS>
void launch_route(const RouteArgs &a, bool wide, int blocks, cudaStream_t st) {
#define TMOE_RT(TS_, G, NC, W) route_kernel<TS_, G, NC, W><<<blocks, kRouteThreads, kRouteWarps * G * NC * 8 * 4, st>>>(a)
  if (wide) TMOE_ROUTE_G(TMOE_RT, TS, true);
  else TMOE_ROUTE_G(TMOE_RT, TS, false);
#undef TMOE_RT
}
template <typename TS>
void launch_route_backward(const RouteArgs &a, bool wide, int blocks, cudaStream_t st) {
#define TMOE_RTB(TS_, G, NC, W) route_backward_kernel<TS_, G, NC, W><<<blocks, kRouteThreads, 0, st>>>(a)
  if (wide) TMOE_ROUTE_G(TMOE_RTB, TS, true);
  else TMOE_ROUTE_G(TMOE_RTB, TS, false);
#undef TMOE_RTB
}

int64_t route_ws(int blocks, int E) { return align_up((int64_t)blocks * E * 4, 256) * 2 + align_up((int64_t)blocks * 8, 256); }

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

int tmoe_route_tokens(const tmoe_route_t *p, int32_t *idx, float *gates, int32_t *counts, float *losses, void *workspace,
                      int64_t workspace_bytes, void *stream) {
  int rc = check_route(p);
  if (rc) return rc;
  if (!counts || !losses) return TMOE_ERR_NULL;
  cudaStream_t st = (cudaStream_t)stream;
  if (p->tokens == 0) {
    rc = cuda_ok(cudaMemsetAsync(counts, 0, (size_t)p->n_experts * 4, st));
    return rc ? rc : cuda_ok(cudaMemsetAsync(losses, 0, 12, st));
  }
  if (!idx || !gates || !workspace) return TMOE_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(idx) | reinterpret_cast<uintptr_t>(gates) | reinterpret_cast<uintptr_t>(counts) |
       reinterpret_cast<uintptr_t>(losses)) & 3)
    return TMOE_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return TMOE_ERR_ALIGN;
  const int sms = current_device_sms();
  if (sms <= 0) return TMOE_ERR_CUDA;
  const int blocks = route_blocks(p->tokens, p->n_experts, sms < 160 ? sms : 160);
  if (workspace_bytes < route_ws(blocks, p->n_experts)) return TMOE_ERR_WORKSPACE;
  RouteArgs a = route_args(*p);
  a.idx = idx; a.gates = gates; a.counts = counts; a.losses = losses;
  char *ws = reinterpret_cast<char *>(workspace);
  const int64_t one = align_up((int64_t)blocks * a.E * 4, 256);
  a.part_p = reinterpret_cast<float *>(ws);
  a.part_c = reinterpret_cast<int32_t *>(ws + one);
  a.part_zn = reinterpret_cast<float *>(ws + 2 * one);
  const bool wide = route_wide(*p, nullptr);
  if (p->dtype == TMOE_F32) launch_route<float>(a, wide, blocks, st);
  else launch_route<bf16>(a, wide, blocks, st);
  count_launch();
  if ((rc = launch_status())) return rc;
  route_losses_kernel<<<1, 1024, 0, st>>>(a, blocks);
  count_launch();
  return launch_status();
}

int tmoe_route_tokens_backward(const tmoe_route_t *p, const int32_t *idx, const float *gates, const int32_t *counts,
                               const float *losses, const float *d_gates, const float *d_balance, const float *d_z, void *d_scores,
                               void *stream) {
  int rc = check_route(p);
  if (rc) return rc;
  if (p->tokens == 0) return TMOE_OK;
  if (!idx || !gates || !counts || !losses || !d_scores) return TMOE_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(idx) | reinterpret_cast<uintptr_t>(gates) | reinterpret_cast<uintptr_t>(counts) |
       reinterpret_cast<uintptr_t>(losses) | reinterpret_cast<uintptr_t>(d_gates) | reinterpret_cast<uintptr_t>(d_balance) |
       reinterpret_cast<uintptr_t>(d_z)) & 3)
    return TMOE_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(d_scores) & (p->dtype == TMOE_F32 ? 3 : 1)) return TMOE_ERR_ALIGN;
  const int sms = current_device_sms();
  if (sms <= 0) return TMOE_ERR_CUDA;
  RouteArgs a = route_args(*p);
  a.idx = const_cast<int32_t *>(idx); a.gates = const_cast<float *>(gates); a.counts = const_cast<int32_t *>(counts);
  a.losses = const_cast<float *>(losses);
  a.d_gates = d_gates; a.d_balance = d_balance; a.d_z = d_z; a.d_scores = d_scores;
  const bool wide = route_wide(*p, d_scores);
  const int64_t per = kRouteWarps * (32 / lanes_per_token(a.E)), want = (a.tokens + per - 1) / per;
  const int blocks = (int)(want < (int64_t)sms * 8 ? want : (int64_t)sms * 8);
  cudaStream_t st = (cudaStream_t)stream;
  if (p->dtype == TMOE_F32) launch_route_backward<float>(a, wide, blocks, st);
  else launch_route_backward<bf16>(a, wide, blocks, st);
  count_launch();
  return launch_status();
}

}  // extern "C"
