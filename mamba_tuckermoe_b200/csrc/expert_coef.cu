// Coefficient vectors of the core mixing from given routing, with their gradients:
//
//   c[t, a]      = sum_j gates[t, j] * U_expert[idx[t, j], a]          (the gather of pure_torch_mlx/model.py:93)
//   d_gates[t,j] = sum_a U_expert[idx[t, j], a] * d_c[t, a]
//   d_U[e, a]    = sum over the slots (t, j) with idx[t, j] = e of gates[t, j] * d_c[t, a]
//
// A slot whose index lies outside 0 .. E-1 is empty: it adds nothing and its d_gates is 0.
//
// d_U is a scatter of T * k rows onto E; float atomics would add them in another order on every run.  Here each group of lanes keeps a
// table [E, columns] of its own in shared memory and adds its tokens' slots to it in order; a block adds its groups' tables in order
// and writes one partial table, coef_reduce_kernel adds the blocks' tables in order.
#include "column_sum.cuh"
#include "common.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace tmoe {
namespace {

constexpr int kCoefMaxExperts = 8192;    // a table of 4 columns: 128 KB
constexpr int kCoefSmem = 192 * 1024;    // shared memory for the tables of one block
constexpr int kDuThreads = 640;          // 20 warps of up to 96 registers
constexpr int kDuClear = 512;            // threads that clear and fold the tables at least
constexpr int kAhead = 4;                // rounds of slots whose operands are in flight

struct CoefArgs {
  const int32_t *idx;     // [T, k]
  const float *gates;     // [T, k]
  const void *u;          // [E, r1]
  int64_t T;
  int E, k, r1;
  float *c;               // [T, r1]
  const float *d_c;       // [T, r1]
  float *d_gates;         // [T, k]
  float *partial;         // [blocks, E, r1]
};

// C consecutive values of a U_expert row or an fp32 row (C = 4: one 8- or 16-byte load)
template <int C> __device__ __forceinline__ void load_cols(const float *p, float (&f)[C]) {
  if constexpr (C == 4) {
    const float4 v = __ldg(reinterpret_cast<const float4 *>(p));
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  } else {
    f[0] = __ldg(p);
  }
}
template <int C> __device__ __forceinline__ void load_cols(const bf16 *p, float (&f)[C]) {
  if constexpr (C == 4) {
    const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
    f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
    f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
  } else {
    f[0] = to_f32(*p);
  }
}
// up to 4 slots of a token (KV = 4: one 16-byte load each)
template <int KV> struct SlotPack {
  int e[KV];
  float g[KV];
  __device__ __forceinline__ void load(const CoefArgs &a, int64_t at) {
    if constexpr (KV == 4) {
      const int4 i = __ldg(reinterpret_cast<const int4 *>(a.idx + at));
      const float4 f = __ldg(reinterpret_cast<const float4 *>(a.gates + at));
      e[0] = i.x; e[1] = i.y; e[2] = i.z; e[3] = i.w;
      g[0] = f.x; g[1] = f.y; g[2] = f.z; g[3] = f.w;
    } else if constexpr (KV == 2) {
      const int2 i = __ldg(reinterpret_cast<const int2 *>(a.idx + at));
      const float2 f = __ldg(reinterpret_cast<const float2 *>(a.gates + at));
      e[0] = i.x; e[1] = i.y; g[0] = f.x; g[1] = f.y;
    } else {
      e[0] = __ldg(a.idx + at); g[0] = __ldg(a.gates + at);
    }
  }
};

// One thread makes C neighbouring coefficients of a token; the U_expert table comes from L1.  131072 x 8, r1 = 8: 4.6 us = 2.7 TB/s.
template <typename TU, int C, int KV>
__global__ void __launch_bounds__(256) coef_kernel(const __grid_constant__ CoefArgs a) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();   // the routing may come from the kernel before this one
  const int per = a.r1 / C;
  const int64_t n = a.T * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / per;
    const int col = (int)(i - t * per) * C;
    float s[C];
#pragma unroll
    for (int q = 0; q < C; ++q) s[q] = 0.f;
    for (int j = 0; j < a.k; j += KV) {
      SlotPack<KV> p;
      p.load(a, t * a.k + j);
#pragma unroll
      for (int v = 0; v < KV; ++v) {
        if ((unsigned)p.e[v] < (unsigned)a.E) {
          float u[C];
          load_cols<C>((const TU *)a.u + (int64_t)p.e[v] * a.r1 + col, u);
#pragma unroll
          for (int q = 0; q < C; ++q) s[q] = fmaf(p.g[v], u[q], s[q]);
        }
      }
    }
    if constexpr (C == 4) *reinterpret_cast<float4 *>(a.c + t * a.r1 + col) = make_float4(s[0], s[1], s[2], s[3]);
    else a.c[t * a.r1 + col] = s[0];
  }
}

// One thread makes KV neighbouring slots of a token.
template <typename TU, int C, int KV>
__global__ void __launch_bounds__(256) coef_d_gates_kernel(const __grid_constant__ CoefArgs a) {
  // in this order: once the next kernel may start, what was before this one is complete (coef_d_u_kernel counts on it)
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int per = a.k / KV;
  const int64_t n = a.T * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / per, at = i * KV;
    SlotPack<KV> p;
    p.load(a, at);
    float s[KV];
#pragma unroll
    for (int v = 0; v < KV; ++v) {
      s[v] = 0.f;
      if ((unsigned)p.e[v] >= (unsigned)a.E) p.e[v] = -1;
    }
    for (int q = 0; q < a.r1; q += C) {
      float d[C];
      load_cols<C>(a.d_c + t * a.r1 + q, d);
#pragma unroll
      for (int v = 0; v < KV; ++v) {
        if (p.e[v] >= 0) {
          float u[C];
          load_cols<C>((const TU *)a.u + (int64_t)p.e[v] * a.r1 + q, u);
#pragma unroll
          for (int x = 0; x < C; ++x) s[v] = fmaf(u[x], d[x], s[v]);
        }
      }
    }
    if constexpr (KV == 4) *reinterpret_cast<float4 *>(a.d_gates + at) = make_float4(s[0], s[1], s[2], s[3]);
    else if constexpr (KV == 2) *reinterpret_cast<float2 *>(a.d_gates + at) = make_float2(s[0], s[1]);
    else a.d_gates[at] = s[0];
  }
}

// A group of S * L lanes (a power of two up to 32) takes S slots of a token at once, 4 columns a lane, with a private table.  The experts of
// a token usually differ, so the S slots touch different rows of it; where an expert is given twice the lanes take turns.  The operands of
// kAhead rounds are in flight while the ones before are added.  blockIdx.y picks the columns; threads beyond the last group only
// clear and fold tables.  Bound by the rounds' read-modify-write on few warps (the tables fill shared memory): 131072 tokens x 8 slots, 256
// experts, r1 = 8 take 17 us, with the lane layout as arguments of the kernel they took 25; 32768 x 2, 64 experts, r1 = 4 take 6 us.
template <int L, int S>
__global__ void __launch_bounds__(kDuThreads) coef_d_u_kernel(const __grid_constant__ CoefArgs a, int groups, int wide) {
  constexpr int lanes = S * L;
  extern __shared__ __align__(16) float4 tab[];   // [groups][E * L]
  const int grp = threadIdx.x / lanes, in = threadIdx.x - grp * lanes, lane = threadIdx.x & 31;
  const int s = in / L, col = in - s * L, c = (blockIdx.y * L + col) * 4, width = a.E * L;
  ptx::griddep_launch_dependents();
  for (int i = threadIdx.x; i < groups * width; i += blockDim.x) tab[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  // the lanes of this group that hold the same columns of the slots before this one
  const int lane0 = (lane & ~(lanes - 1)) + col;
  uint32_t before = 0;
#pragma unroll
  for (int q = 0; q < S; ++q) before |= q < s ? 1u << (lane0 + q * L) : 0u;
  const int64_t lo = a.T * blockIdx.x / gridDim.x, hi = a.T * (blockIdx.x + 1) / gridDim.x;
  // every lane of the block walks the same number of rounds: the turns need whole warps (rounds beyond the last are empty)
  const int rounds = (int)((hi - lo + groups - 1) / groups) * ((a.k + S - 1) / S);
  int left = grp < groups && c < a.r1 ? (int)((hi - lo - grp + groups - 1) / groups) : 0;   // tokens of this group
  int base = 0;                                             // slots of the current token that are done
  const int64_t t0 = lo + (grp < groups ? grp : 0);
  const int32_t *idx = a.idx + t0 * a.k + s;
  const float *gates = a.gates + t0 * a.k + s, *d_c = a.d_c + t0 * a.r1 + c;
  const int64_t k_step = (int64_t)groups * a.k, d_step = (int64_t)groups * a.r1;
  int e_next[kAhead], e[kAhead];
  float g_next[kAhead], g[kAhead];
  float4 d_next[kAhead], d[kAhead];
  auto fetch = [&]() {
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      e_next[q] = -1;
      g_next[q] = 0.f;
      d_next[q] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (left > 0 && base + s < a.k) {
        e_next[q] = __ldg(idx + base);
        g_next[q] = __ldg(gates + base);
        if (wide) {
          d_next[q] = __ldg(reinterpret_cast<const float4 *>(d_c));
        } else {
          d_next[q].x = __ldg(d_c);
          if (c + 1 < a.r1) d_next[q].y = __ldg(d_c + 1);
          if (c + 2 < a.r1) d_next[q].z = __ldg(d_c + 2);
          if (c + 3 < a.r1) d_next[q].w = __ldg(d_c + 3);
        }
      }
      base += S;
      if (base >= a.k) { base = 0; --left; idx += k_step; gates += k_step; d_c += d_step; }
    }
  };
  fetch();
  __syncthreads();
  float4 *mine = tab + (grp < groups ? grp * width + col : 0);
  auto add = [&](int row, float w, const float4 &x) {
    float4 v = mine[row * L];
    v.x = fmaf(w, x.x, v.x); v.y = fmaf(w, x.y, v.y); v.z = fmaf(w, x.z, v.z); v.w = fmaf(w, x.w, v.w);
    mine[row * L] = v;
  };
  const bool idle = (int)(threadIdx.x & ~31u) >= groups * lanes;   // a warp without a group only clears and folds
  for (int r = idle ? rounds : 0; r < rounds; r += kAhead) {
#pragma unroll
    for (int q = 0; q < kAhead; ++q) { e[q] = e_next[q]; g[q] = g_next[q]; d[q] = d_next[q]; }
    if (r + kAhead < rounds) fetch();
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const bool have = (unsigned)e[q] < (unsigned)a.E;
      bool twice = false;
#pragma unroll
      for (int o = 1; o <= S / 2; ++o) {   // of every two slots one sees the other; by every lane, whatever it has found
        const int other = __shfl_sync(0xffffffffu, e[q], lane0 + (s + o) % S * L);
        twice |= other == e[q];
      }
      if (!__any_sync(0xffffffffu, have && twice)) {
        if (have) add(e[q], g[q], d[q]);
      } else {
        const int turn = __popc(__match_any_sync(0xffffffffu, have ? e[q] : -1 - lane) & before);
        for (int w = 0; w < S; ++w) {
          if (have && turn == w) add(e[q], g[q], d[q]);
          __syncwarp();
        }
      }
      __syncwarp();   // the group's other lanes may hold this row next
    }
  }
  __syncthreads();
  // the kernel before this one in the stream (d_gates, whose output nothing here reads) may still run until here
  ptx::griddep_wait();
  for (int i = threadIdx.x; i < width; i += blockDim.x) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int q = 0; q < groups; ++q) {
      const float4 w = tab[q * width + i];
      v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
    }
    const int x = i / L, q = (blockIdx.y * L + i - x * L) * 4;
    float *to = a.partial + ((int64_t)blockIdx.x * a.E + x) * a.r1 + q;
    if (a.r1 % 4 == 0) {
      if (q < a.r1) *reinterpret_cast<float4 *>(to) = v;
    } else {
      const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int y = 0; y < 4; ++y)
        if (q + y < a.r1) to[y] = f[y];
    }
  }
}

template <typename TU>
__global__ void __launch_bounds__(kColumnSumThreads) coef_reduce_kernel(const float *__restrict__ partial, int blocks, int n, TU *__restrict__ d_u) {
  __shared__ float part[32][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31);
  ptx::griddep_wait();
  const float t = column_sum(partial, blocks, n, col, part);
  if (threadIdx.x < 32 && col < n) d_u[col] = from_f32<TU>(t);
}

int check_coef(const tmoe_expert_coef_t *p) {
  if (!p) return TMOE_ERR_NULL;
  if (p->dtype != TMOE_F32 && p->dtype != TMOE_BF16) return TMOE_ERR_DTYPE;
  if (p->tokens < 0 || p->tokens > ((int64_t)1 << 30) || p->n_experts <= 0 || p->top_k <= 0 || p->top_k > TMOE_MAX_TOPK || p->r1 <= 0 ||
      p->r1 > TMOE_MAX_R1)
    return TMOE_ERR_SHAPE;
  if (p->n_experts > kCoefMaxExperts) return TMOE_ERR_UNSUPPORTED;
  if (p->tokens == 0) return TMOE_OK;
  if (!p->idx || !p->gates || !p->U_expert) return TMOE_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(p->idx) | reinterpret_cast<uintptr_t>(p->gates)) & 3) return TMOE_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(p->U_expert) & (p->dtype == TMOE_F32 ? 3 : 1)) return TMOE_ERR_ALIGN;
  return TMOE_OK;
}

CoefArgs coef_args(const tmoe_expert_coef_t &p) {
  CoefArgs a{};
  a.idx = p.idx; a.gates = p.gates; a.u = p.U_expert; a.T = p.tokens; a.E = p.n_experts; a.k = p.top_k; a.r1 = p.r1;
  return a;
}

// Lanes over the columns of a block (4 columns each), slots taken at once, groups with a table each, blocks over the tokens.  Tables of at
// most 32 KB leave room for several groups; a group wants some rounds of work for the table it clears and folds.
struct DuShape { int L, S, parts, groups, blocks; };
DuShape du_shape(int64_t T, int E, int k, int r1, int sms) {
  DuShape s;
  s.L = 1;
  while (s.L < 16 && s.L * 4 < r1 && (int64_t)E * s.L * 2 * 16 <= 32 * 1024) s.L *= 2;
  s.parts = (r1 + s.L * 4 - 1) / (s.L * 4);
  s.S = 1;
  while (s.S < k && s.S * 2 * s.L <= 32) s.S *= 2;
  const int most = (int)(kCoefSmem / ((int64_t)E * s.L * 16)), lanes = s.S * s.L, per_token = (k + s.S - 1) / s.S;
  const int64_t cap = (sms + s.parts - 1) / s.parts, want = (T + 31) / 32;
  s.blocks = (int)(want < cap ? want : cap);
  const int64_t each = (T + s.blocks - 1) / s.blocks, tokens = per_token < 8 ? 8 / per_token : 1;
  s.groups = (int)((each + tokens - 1) / tokens < most ? (each + tokens - 1) / tokens : most);
  if (s.groups > kDuThreads / lanes) s.groups = kDuThreads / lanes;
  return s;
}

template <int L, int S>
int launch_d_u_as(const CoefArgs &a, const DuShape &s, bool overlap, cudaStream_t st) {
  static std::atomic<uint64_t> opted{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return TMOE_ERR_CUDA;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(opted.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(coef_d_u_kernel<L, S>, cudaFuncAttributeMaxDynamicSharedMemorySize, kCoefSmem) != cudaSuccess) return TMOE_ERR_CUDA;
    opted.fetch_or(bit, std::memory_order_relaxed);
  }
  const int need = (s.groups * S * L + 31) / 32 * 32, threads = need > kDuClear ? need : kDuClear, wide = a.r1 % 4 == 0 && !(reinterpret_cast<uintptr_t>(a.d_c) & 15);
  const size_t smem = (size_t)s.groups * a.E * L * 16;
  const dim3 grid((unsigned)s.blocks, (unsigned)s.parts), block((unsigned)threads);
  count_launch();
  // after d_gates of the same call it may begin while that runs: both only read what was there before
  if (overlap) return cuda_ok(launch_pdl(coef_d_u_kernel<L, S>, grid, block, smem, st, a, s.groups, wide));
  coef_d_u_kernel<L, S><<<grid, block, smem, st>>>(a, s.groups, wide);
  return launch_status();
}
template <int L>
int launch_d_u(const CoefArgs &a, const DuShape &s, bool overlap, cudaStream_t st) {
  switch (s.S) {   // S * L is at most 32
    case 1: return launch_d_u_as<L, 1>(a, s, overlap, st);
    case 2: return launch_d_u_as<L, 2>(a, s, overlap, st);
    case 4: if constexpr (L <= 8) return launch_d_u_as<L, 4>(a, s, overlap, st); break;
    case 8: if constexpr (L <= 4) return launch_d_u_as<L, 8>(a, s, overlap, st); break;
    case 16: if constexpr (L <= 2) return launch_d_u_as<L, 16>(a, s, overlap, st); break;
  }
  return TMOE_ERR_UNSUPPORTED;
}

// wide: rows of U_expert, c and d_c are whole 4-column pieces
bool cols_by_4(const CoefArgs &a, int size, const void *rows) {
  return a.r1 % 4 == 0 && !(reinterpret_cast<uintptr_t>(a.u) & (4 * size - 1)) && !(reinterpret_cast<uintptr_t>(rows) & 15);
}
// slots per 16- or 8-byte load of idx, gates and (backward) d_gates
int slots_wide(const CoefArgs &a) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(a.idx) | reinterpret_cast<uintptr_t>(a.gates) | reinterpret_cast<uintptr_t>(a.d_gates);
  return a.k % 4 == 0 && !(all & 15) ? 4 : a.k % 2 == 0 && !(all & 7) ? 2 : 1;
}
int spread(int64_t threads, int sms) {
  const int64_t want = (threads + 255) / 256, cap = (int64_t)sms * 16;
  return (int)(want < cap ? want : cap);
}
template <typename TU, int C>
int launch_coef(const CoefArgs &a, int sms, cudaStream_t st) {
  const int blocks = spread(a.T * (a.r1 / C), sms), kv = slots_wide(a);
  const dim3 grid((unsigned)blocks), block(256);
  count_launch();
  return cuda_ok(kv == 4   ? launch_pdl(coef_kernel<TU, C, 4>, grid, block, 0, st, a)
                 : kv == 2 ? launch_pdl(coef_kernel<TU, C, 2>, grid, block, 0, st, a)
                           : launch_pdl(coef_kernel<TU, C, 1>, grid, block, 0, st, a));
}
template <typename TU, int C>
int launch_d_gates(const CoefArgs &a, int sms, cudaStream_t st) {
  const int kv = slots_wide(a), blocks = spread(a.T * (a.k / kv), sms);
  const dim3 grid((unsigned)blocks), block(256);
  count_launch();
  return cuda_ok(kv == 4   ? launch_pdl(coef_d_gates_kernel<TU, C, 4>, grid, block, 0, st, a)
                 : kv == 2 ? launch_pdl(coef_d_gates_kernel<TU, C, 2>, grid, block, 0, st, a)
                           : launch_pdl(coef_d_gates_kernel<TU, C, 1>, grid, block, 0, st, a));
}

}  // namespace
}  // namespace tmoe

using namespace tmoe;

extern "C" {

int tmoe_expert_coef(const tmoe_expert_coef_t *p, float *c, void *stream) {
  int rc = check_coef(p);
  if (rc) return rc;
  if (p->tokens == 0) return TMOE_OK;
  if (!c) return TMOE_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(c) & 3) return TMOE_ERR_ALIGN;
  const int sms = current_device_sms();
  if (sms <= 0) return TMOE_ERR_CUDA;
  CoefArgs a = coef_args(*p);
  a.c = c;
  const bool four = cols_by_4(a, p->dtype == TMOE_F32 ? 4 : 2, c);
  cudaStream_t st = (cudaStream_t)stream;
  if (p->dtype == TMOE_F32) return four ? launch_coef<float, 4>(a, sms, st) : launch_coef<float, 1>(a, sms, st);
  return four ? launch_coef<bf16, 4>(a, sms, st) : launch_coef<bf16, 1>(a, sms, st);
}

int64_t tmoe_expert_coef_workspace_bytes(const tmoe_expert_coef_t *p) {
  int rc = check_coef(p);
  if (rc) return rc;
  // sized for up to 160 SMs, whatever device the sizing query runs on
  return p->tokens ? (int64_t)du_shape(p->tokens, p->n_experts, p->top_k, p->r1, 160).blocks * p->n_experts * p->r1 * 4 : 0;
}

int tmoe_expert_coef_backward(const tmoe_expert_coef_t *p, const float *d_c, float *d_gates, void *d_U_expert, void *workspace,
                              int64_t workspace_bytes, void *stream) {
  int rc = check_coef(p);
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const int size = p->dtype == TMOE_F32 ? 4 : 2;
  if (!d_gates && !d_U_expert) return TMOE_ERR_NULL;
  if (p->tokens == 0)
    return d_U_expert ? cuda_ok(cudaMemsetAsync(d_U_expert, 0, (size_t)p->n_experts * p->r1 * size, st)) : (int)TMOE_OK;
  if (!d_c) return TMOE_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(d_c) | reinterpret_cast<uintptr_t>(d_gates)) & 3) return TMOE_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(d_U_expert) & (size - 1)) return TMOE_ERR_ALIGN;
  const int sms = current_device_sms();
  if (sms <= 0) return TMOE_ERR_CUDA;
  CoefArgs a = coef_args(*p);
  a.d_c = d_c; a.d_gates = d_gates;
  if (d_gates) {
    const bool four = cols_by_4(a, size, d_c);
    if (p->dtype == TMOE_F32) rc = four ? launch_d_gates<float, 4>(a, sms, st) : launch_d_gates<float, 1>(a, sms, st);
    else rc = four ? launch_d_gates<bf16, 4>(a, sms, st) : launch_d_gates<bf16, 1>(a, sms, st);
    if (rc) return rc;
  }
  if (d_U_expert) {
    const DuShape s = du_shape(a.T, a.E, a.k, a.r1, sms < 160 ? sms : 160);
    const int n = a.E * a.r1;
    if (!workspace) return TMOE_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return TMOE_ERR_ALIGN;
    if (workspace_bytes < (int64_t)s.blocks * n * 4) return TMOE_ERR_WORKSPACE;
    a.partial = reinterpret_cast<float *>(workspace);
    switch (s.L) {
      case 1: rc = launch_d_u<1>(a, s, d_gates != nullptr, st); break;
      case 2: rc = launch_d_u<2>(a, s, d_gates != nullptr, st); break;
      case 4: rc = launch_d_u<4>(a, s, d_gates != nullptr, st); break;
      case 8: rc = launch_d_u<8>(a, s, d_gates != nullptr, st); break;
      default: rc = launch_d_u<16>(a, s, d_gates != nullptr, st); break;
    }
    if (rc) return rc;
    const dim3 grid((unsigned)((n + 31) / 32)), block(kColumnSumThreads);
    rc = p->dtype == TMOE_F32 ? cuda_ok(launch_pdl(coef_reduce_kernel<float>, grid, block, 0, st, a.partial, s.blocks, n, (float *)d_U_expert))
                              : cuda_ok(launch_pdl(coef_reduce_kernel<bf16>, grid, block, 0, st, a.partial, s.blocks, n, (bf16 *)d_U_expert));
    count_launch();
  }
  return rc;
}

}  // extern "C"
