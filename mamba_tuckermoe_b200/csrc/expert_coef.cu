// Coefficient vectors of the core mixing from given routing, with their gradients:
//
//   c[t, a]      = sum_j gates[t, j] * U_expert[idx[t, j], a]          (the gather of pure_torch_mlx/model.py:93)
//   d_gates[t,j] = sum_a U_expert[idx[t, j], a] * d_c[t, a]
//   d_U[e, a]    = sum over the slots (t, j) with idx[t, j] = e of gates[t, j] * d_c[t, a]
//
// A slot whose index lies outside 0 .. E-1 is empty: it adds nothing and its d_gates is 0.
//
// d_U is a scatter of T * k rows onto E; float atomics would add them in another order on every run.  Here each group of lanes
// keeps a table [E, columns] of its own in shared memory and adds its slots to it in order; a block adds its groups' tables in
// order and writes one partial table, coef_reduce_kernel adds the blocks' tables in order.
#include "common.cuh"
#include "kernels.h"

namespace tmoe {
namespace {

constexpr int kCoefMaxExperts = 16384;
constexpr int kCoefSmem = 160 * 1024;    // shared memory for the tables of one block

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

template <typename TU>
__global__ void __launch_bounds__(256) coef_kernel(const __grid_constant__ CoefArgs a) {
  const int64_t n = a.T * a.r1;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / a.r1;
    const int col = (int)(i - t * a.r1);
    float s = 0.f;
    for (int j = 0; j < a.k; ++j) {
      const int e = a.idx[t * a.k + j];
      if ((unsigned)e < (unsigned)a.E) s = fmaf(a.gates[t * a.k + j], to_f32(((const TU *)a.u)[(int64_t)e * a.r1 + col]), s);
    }
    a.c[i] = s;
  }
}

template <typename TU>
__global__ void __launch_bounds__(256) coef_d_gates_kernel(const __grid_constant__ CoefArgs a) {
  const int64_t n = a.T * a.k;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int e = a.idx[i];
    float s = 0.f;
    if ((unsigned)e < (unsigned)a.E) {
      const float *d = a.d_c + (i / a.k) * a.r1;
      const TU *u = (const TU *)a.u + (int64_t)e * a.r1;
      for (int q = 0; q < a.r1; ++q) s = fmaf(to_f32(u[q]), d[q], s);
    }
    a.d_gates[i] = s;
  }
}

// blockDim = groups * cols; blockIdx.y picks the columns.
__global__ void __launch_bounds__(1024) coef_d_u_kernel(const __grid_constant__ CoefArgs a, int cols) {
  extern __shared__ float tab[];   // [groups][E * cols]
  const int groups = blockDim.x / cols, grp = threadIdx.x / cols, col = threadIdx.x - grp * cols;
  const int c0 = blockIdx.y * cols, width = a.E * cols;
  for (int i = threadIdx.x; i < groups * width; i += blockDim.x) tab[i] = 0.f;
  __syncthreads();
  if (c0 + col < a.r1) {
    float *mine = tab + grp * width + col;
    const int64_t lo = a.T * blockIdx.x / gridDim.x, hi = a.T * (blockIdx.x + 1) / gridDim.x;
    for (int64_t t = lo + grp; t < hi; t += groups) {
      const float d = a.d_c[t * a.r1 + c0 + col];
      for (int j = 0; j < a.k; ++j) {
        const int e = a.idx[t * a.k + j];
        if ((unsigned)e < (unsigned)a.E) mine[e * cols] = fmaf(a.gates[t * a.k + j], d, mine[e * cols]);
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < width; i += blockDim.x) {
    float s = 0.f;
    for (int g = 0; g < groups; ++g) s += tab[g * width + i];
    const int e = i / cols, q = i - e * cols;
    if (c0 + q < a.r1) a.partial[((int64_t)blockIdx.x * a.E + e) * a.r1 + c0 + q] = s;
  }
}

template <typename TU>
__global__ void __launch_bounds__(256) coef_reduce_kernel(const float *__restrict__ partial, int blocks, int n, TU *__restrict__ d_u) {
  __shared__ float part[8][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  float s = 0.f;
  if (col < n)
    for (int b = row; b < blocks; b += 8) s += partial[(int64_t)b * n + col];
  part[row][lane] = s;
  __syncthreads();
  if (row == 0 && col < n) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += part[i][lane];
    d_u[col] = from_f32<TU>(t);
  }
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

// Columns of one block and its lane groups: as many private tables as fit
struct DuShape { int cols, groups, parts; };
DuShape du_shape(int E, int r1) {
  DuShape s;
  s.cols = 1;
  while (s.cols < 32 && s.cols < r1 && (int64_t)E * s.cols * 2 * 4 <= 32 * 1024) s.cols *= 2;
  s.parts = (r1 + s.cols - 1) / s.cols;
  s.groups = (int)(kCoefSmem / ((int64_t)E * s.cols * 4));
  if (s.groups > 512 / s.cols) s.groups = 512 / s.cols;
  return s;
}
int du_blocks(int64_t T, int E, int r1, int sms) {
  const DuShape s = du_shape(E, r1);
  const int64_t want = (T + s.groups * 4 - 1) / (s.groups * 4), cap = (sms + s.parts - 1) / s.parts;
  return (int)(want < cap ? want : cap);
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
  const int64_t want = (a.T * a.r1 + 255) / 256, cap = (int64_t)sms * 16;
  const int blocks = (int)(want < cap ? want : cap);
  if (p->dtype == TMOE_F32) coef_kernel<float><<<blocks, 256, 0, (cudaStream_t)stream>>>(a);
  else coef_kernel<bf16><<<blocks, 256, 0, (cudaStream_t)stream>>>(a);
  count_launch();
  return launch_status();
}

int64_t tmoe_expert_coef_workspace_bytes(const tmoe_expert_coef_t *p) {
  int rc = check_coef(p);
  if (rc) return rc;
  // sized for up to 160 SMs, whatever device the sizing query runs on
  return p->tokens ? (int64_t)du_blocks(p->tokens, p->n_experts, p->r1, 160) * p->n_experts * p->r1 * 4 : 0;
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
    const int64_t want = (a.T * a.k + 255) / 256, cap = (int64_t)sms * 16;
    const int blocks = (int)(want < cap ? want : cap);
    if (p->dtype == TMOE_F32) coef_d_gates_kernel<float><<<blocks, 256, 0, st>>>(a);
    else coef_d_gates_kernel<bf16><<<blocks, 256, 0, st>>>(a);
    count_launch();
    if ((rc = launch_status())) return rc;
  }
  if (d_U_expert) {
    const DuShape s = du_shape(a.E, a.r1);
    const int blocks = du_blocks(a.T, a.E, a.r1, sms < 160 ? sms : 160), n = a.E * a.r1;
    if (!workspace) return TMOE_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return TMOE_ERR_ALIGN;
    if (workspace_bytes < (int64_t)blocks * n * 4) return TMOE_ERR_WORKSPACE;
    a.partial = reinterpret_cast<float *>(workspace);
    const int smem = s.groups * a.E * s.cols * 4;
    if (cudaFuncSetAttribute(coef_d_u_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kCoefSmem) != cudaSuccess) return TMOE_ERR_CUDA;
    coef_d_u_kernel<<<dim3(blocks, s.parts), s.groups * s.cols, smem, st>>>(a, s.cols);
    count_launch();
    if ((rc = launch_status())) return rc;
    if (p->dtype == TMOE_F32) coef_reduce_kernel<float><<<(n + 31) / 32, 256, 0, st>>>(a.partial, blocks, n, (float *)d_U_expert);
    else coef_reduce_kernel<bf16><<<(n + 31) / 32, 256, 0, st>>>(a.partial, blocks, n, (bf16 *)d_U_expert);
    count_launch();
    rc = launch_status();
  }
  return rc;
}

}  // extern "C"
