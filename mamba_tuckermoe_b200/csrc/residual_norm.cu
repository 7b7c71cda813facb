// The tail of a block as one pass over its rows, with its gradients:
//
//   a      = y * rstd(y) * post_w        (norm after the block; a = y without it)
//   v      = silu(gate) * a              (v = a without a gate)
//   out    = residual + layer_scale * v  (either may be absent)
//   normed = out * rstd(out) * next_w    (norm in front of the next block),      rstd(x) = 1 / sqrt(mean(x^2) + eps)
//
// The order is the one of the layer's own epilogue (pure_torch_mlx/model.py:25-27, 258-260, 340-341): layer output, silu gate,
// layer scale and residual, then the next block's pre-norm.
//
// Everything between the loads and the stores is fp32; `normed` is made from the unrounded sum, so `out` and `normed` are each
// rounded once, to their storage types.
//
// Gradients, with x = out * rstd1, h = y * rstd0, s = silu(gate) and the upstream gradients dO (of out) and dN (of normed):
//   u  = next_w * dN,   dR = dO + rstd1 * (u - x * mean(u * x))                  d_residual = dR
//   dv = layer_scale * dR,   da = dv * s                                         d_gate = dv * a * silu'(gate)
//   dy = rstd0 * (post_w * da - h * mean(post_w * da * h))
//   d_layer_scale = sum_t dR * v,   d_post_w = sum_t da * h,   d_next_w = sum_t dN * x
// The two row means need one team reduction, not two: with b = dO + rstd1 * u and q = post_w * layer_scale * s * h,
//   mean(post_w * da * h) = (sum q*b - rstd1 * mean(u*x) * sum q*x) / d.
// `out` is recomputed in fp32 from y, gate and residual (the same bytes as reading it back, and no rounding in between); only
// the two rstd of a row are kept from the forward pass.
#include "common.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace tmoe {
namespace {

constexpr int kMaxWidth = 8192;      // widest row: 512 threads x 16 elements
constexpr int kNormThreads = 512;    // upper bound of the block size
constexpr int kNormWarps = kNormThreads / 32;

// VEC consecutive elements of a row as they lie in memory (VEC = 8: 16-byte loads; VEC = 1: any width, stride and base).
template <typename T, int VEC> struct Piece;
template <> struct Piece<bf16, 8> {
  uint4 r;
  __device__ __forceinline__ void load(const bf16 *p) { r = *reinterpret_cast<const uint4 *>(p); }
  __device__ __forceinline__ void zero() { r = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ float get(int q) const {
    const uint32_t w = (q >> 1) == 0 ? r.x : (q >> 1) == 1 ? r.y : (q >> 1) == 2 ? r.z : r.w;
    return __uint_as_float((q & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  __device__ static __forceinline__ void store(bf16 *p, const float (&f)[8]) {
    *reinterpret_cast<uint4 *>(p) =
        make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
};
template <> struct Piece<float, 8> {
  float4 a, b;
  __device__ __forceinline__ void load(const float *p) {
    a = reinterpret_cast<const float4 *>(p)[0];
    b = reinterpret_cast<const float4 *>(p)[1];
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ float get(int q) const {
    const float4 v = q < 4 ? a : b;
    return (q & 3) == 0 ? v.x : (q & 3) == 1 ? v.y : (q & 3) == 2 ? v.z : v.w;
  }
  __device__ static __forceinline__ void store(float *p, const float (&f)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
};
template <typename T> struct Piece<T, 1> {
  T r;
  __device__ __forceinline__ void load(const T *p) { r = *p; }
  __device__ __forceinline__ void zero() { r = from_f32<T>(0.f); }
  __device__ __forceinline__ float get(int) const { return to_f32(r); }
  __device__ static __forceinline__ void store(T *p, const float (&f)[1]) { *p = from_f32<T>(f[0]); }
};

struct NormArgs {
  const void *y, *res, *ls, *gate, *w0, *w1;  // inputs; nullptr = the term is absent
  int64_t ys, rs, gs;                          // row strides in elements
  int64_t rows;
  int d, tw;                                   // row width; warps per row ("team")
  float eps0, eps1;
  void *out, *normed;                          // forward outputs [rows, d]; either may be nullptr
  float *rstd;                                 // [2, rows]: 1/rms of y and of out; nullptr = not kept
  // backward
  const void *d_out, *d_normed;
  int64_t dos, dns;
  void *d_y, *d_res, *d_gate;                  // [rows, d]; nullptr = not wanted
  float *partial;                              // [blocks, n_sums, d] column sums; nullptr = no parameter gradient wanted
  int sum_ls, sum_w0, sum_w1;                  // slot of each parameter gradient in `partial`, or -1
  int n_sums;
};

// Sum over the `tw` warps of a team, in warp order; `slot` alternates between calls, so one barrier per call is enough.
template <int N>
__device__ __forceinline__ void team_sum(float (&v)[N], int tw, int team, float (*red)[kNormWarps][N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if (tw == 1) return;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) (*red)[warp][i] = v[i];
  }
  ptx::named_bar_sync(1 + team, tw * 32);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.f;
  for (int w = 0; w < tw; ++w) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += (*red)[team * tw + w][i];
  }
}

__device__ __forceinline__ float sigmoid(float g) { return 1.f / (1.f + expf(-g)); }

template <typename TY, typename TR, int VEC, int NV>
__global__ void __launch_bounds__(kNormThreads) residual_norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[2][kNormWarps][1];
  const int tpr = a.tw * 32, team = threadIdx.x / tpr, lt = threadIdx.x - team * tpr;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / tpr) + team;
  if (row >= a.rows) return;   // whole teams leave
  const TY *y = (const TY *)a.y + row * a.ys;
  const TY *gate = a.gate ? (const TY *)a.gate + row * a.gs : nullptr;
  const TR *res = a.res ? (const TR *)a.res + row * a.rs : nullptr;
  Piece<TY, VEC> py[NV], pg[NV];
  Piece<TR, VEC> pr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * tpr + lt) * VEC;
    py[i].zero(); pg[i].zero(); pr[i].zero();
    if (e < a.d) {
      py[i].load(y + e);
      if (gate) pg[i].load(gate + e);
      if (res) pr[i].load(res + e);
    }
  }
  float rho0 = 1.f;
  if (a.w0) {
    float ss[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int q = 0; q < VEC; ++q) ss[0] = fmaf(py[i].get(q), py[i].get(q), ss[0]);
    }
    team_sum<1>(ss, a.tw, team, &red[0]);
    rho0 = 1.f / sqrtf(ss[0] / (float)a.d + a.eps0);
    if (a.rstd && lt == 0) a.rstd[row] = rho0;
  }
  float v[NV][VEC];
  float ss[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * tpr + lt) * VEC;
    Piece<TY, VEC> w, l;
    w.zero(); l.zero();
    if (e < a.d) {
      if (a.w0) w.load((const TY *)a.w0 + e);
      if (a.ls) l.load((const TY *)a.ls + e);
    }
#pragma unroll
    for (int q = 0; q < VEC; ++q) {
      float t = py[i].get(q);
      if (a.w0) t = t * rho0 * w.get(q);
      if (gate) { const float g = pg[i].get(q); t *= g * sigmoid(g); }
      if (a.ls) t *= l.get(q);
      t += pr[i].get(q);
      v[i][q] = t;
      ss[0] = fmaf(t, t, ss[0]);
    }
    if (a.out && e < a.d) Piece<TR, VEC>::store((TR *)a.out + row * a.d + e, v[i]);
  }
  if (!a.normed) return;
  team_sum<1>(ss, a.tw, team, &red[1]);
  const float rho1 = 1.f / sqrtf(ss[0] / (float)a.d + a.eps1);
  if (a.rstd && lt == 0) a.rstd[a.rows + row] = rho1;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * tpr + lt) * VEC;
    if (e < a.d) {
      Piece<TY, VEC> w;
      w.load((const TY *)a.w1 + e);
#pragma unroll
      for (int q = 0; q < VEC; ++q) v[i][q] = v[i][q] * rho1 * w.get(q);
      Piece<TY, VEC>::store((TY *)a.normed + row * a.d + e, v[i]);
    }
  }
}

// A team walks over rows blockIdx * teams + team, + gridDim * teams, ...; every thread owns the same columns in all of them, so
// the parameter gradients are sums in its registers.  At the end a block adds its teams in order and writes one row of partial
// sums; norm_params_kernel adds the blocks in order.  The result depends on the sizes and the grid only.
template <typename TY, typename TR, int VEC, int NV>
__global__ void __launch_bounds__(kNormThreads) residual_norm_backward_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[2][kNormWarps][3];
  extern __shared__ float fold[];   // [d] when a block has several teams
  const int tpr = a.tw * 32, team = threadIdx.x / tpr, lt = threadIdx.x - team * tpr, teams = blockDim.x / tpr;
  float acc_ls[NV][VEC], acc_w0[NV][VEC], acc_w1[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int q = 0; q < VEC; ++q) acc_ls[i][q] = acc_w0[i][q] = acc_w1[i][q] = 0.f;
  }
  const float inv_d = 1.f / (float)a.d;
  int slot = 0;
  for (int64_t row = (int64_t)blockIdx.x * teams + team; row < a.rows; row += (int64_t)gridDim.x * teams) {
    const TY *y = (const TY *)a.y + row * a.ys;
    const TY *gate = a.gate ? (const TY *)a.gate + row * a.gs : nullptr;
    const TR *res = a.res ? (const TR *)a.res + row * a.rs : nullptr;
    const TR *d_out = a.d_out ? (const TR *)a.d_out + row * a.dos : nullptr;
    const TY *d_n = a.d_normed ? (const TY *)a.d_normed + row * a.dns : nullptr;
    Piece<TY, VEC> py[NV], pg[NV], pn[NV];
    Piece<TR, VEC> pr[NV], po[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * tpr + lt) * VEC;
      py[i].zero(); pg[i].zero(); pr[i].zero(); po[i].zero(); pn[i].zero();
      if (e < a.d) {
        py[i].load(y + e);
        if (gate) pg[i].load(gate + e);
        if (res) pr[i].load(res + e);
        if (d_out) po[i].load(d_out + e);
        if (d_n) pn[i].load(d_n + e);
      }
    }
    const float rho0 = a.w0 ? a.rstd[row] : 1.f;
    const float rho1 = d_n ? a.rstd[a.rows + row] : 0.f;   // without dN nothing flows through the next norm
    float s3[3] = {0.f, 0.f, 0.f};                          // sum u*x, sum q*b, sum q*x
    if (d_n || a.w0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = (i * tpr + lt) * VEC;
        Piece<TY, VEC> w0, l, w1;
        w0.zero(); l.zero(); w1.zero();
        if (e < a.d) {
          if (a.w0) w0.load((const TY *)a.w0 + e);
          if (a.ls) l.load((const TY *)a.ls + e);
          if (d_n) w1.load((const TY *)a.w1 + e);
        }
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
          const float h = py[i].get(q) * rho0;
          float c = a.ls ? l.get(q) : 1.f;                  // d out / d a
          if (gate) { const float g = pg[i].get(q); c *= g * sigmoid(g); }
          const float w = a.w0 ? w0.get(q) : 1.f;
          const float x = fmaf(c * w, h, pr[i].get(q)) * rho1;
          const float u = w1.get(q) * pn[i].get(q);
          const float b = fmaf(rho1, u, po[i].get(q)), qq = c * w * h;
          s3[0] = fmaf(u, x, s3[0]);
          s3[1] = fmaf(qq, b, s3[1]);
          s3[2] = fmaf(qq, x, s3[2]);
        }
      }
      team_sum<3>(s3, a.tw, team, &red[slot]);
      slot ^= 1;
    }
    const float m1 = s3[0] * inv_d;
    const float m0 = (s3[1] - rho1 * m1 * s3[2]) * inv_d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * tpr + lt) * VEC;
      if (e < a.d) {
        Piece<TY, VEC> w0, l, w1;
        w0.zero(); l.zero(); w1.zero();
        if (a.w0) w0.load((const TY *)a.w0 + e);
        if (a.ls) l.load((const TY *)a.ls + e);
        if (d_n) w1.load((const TY *)a.w1 + e);
        float f_y[VEC], f_r[VEC], f_g[VEC];
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
          const float h = py[i].get(q) * rho0, w = a.w0 ? w0.get(q) : 1.f, ls = a.ls ? l.get(q) : 1.f;
          const float g = pg[i].get(q), sg = gate ? sigmoid(g) : 0.f, s = gate ? g * sg : 1.f;
          const float aa = h * w, v = aa * s;
          const float x = fmaf(ls, v, pr[i].get(q)) * rho1;
          const float dn = pn[i].get(q), u = w1.get(q) * dn;
          const float dr = po[i].get(q) + rho1 * (u - x * m1);
          const float dv = ls * dr, da = dv * s;
          f_r[q] = dr;
          f_g[q] = dv * aa * (sg * (1.f + g * (1.f - sg)));
          f_y[q] = a.w0 ? rho0 * (w * da - h * m0) : da;
          acc_ls[i][q] = fmaf(dr, v, acc_ls[i][q]);
          acc_w0[i][q] = fmaf(da, h, acc_w0[i][q]);
          acc_w1[i][q] = fmaf(dn, x, acc_w1[i][q]);
        }
        if (a.d_y) Piece<TY, VEC>::store((TY *)a.d_y + row * a.d + e, f_y);
        if (a.d_res) Piece<TR, VEC>::store((TR *)a.d_res + row * a.d + e, f_r);
        if (a.d_gate) Piece<TY, VEC>::store((TY *)a.d_gate + row * a.d + e, f_g);
      }
    }
  }
  if (!a.partial) return;
  float *dst = a.partial + (int64_t)blockIdx.x * a.n_sums * a.d;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const int at = k == 0 ? a.sum_ls : k == 1 ? a.sum_w0 : a.sum_w1;
    if (at < 0) continue;
    for (int m = 0; m < teams; ++m) {            // teams add themselves to the block's row one after the other
      if (teams > 1) __syncthreads();
      if (m == team) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int e = (i * tpr + lt) * VEC;
          if (e < a.d) {
#pragma unroll
            for (int q = 0; q < VEC; ++q) {
              float t = k == 0 ? acc_ls[i][q] : k == 1 ? acc_w0[i][q] : acc_w1[i][q];
              if (m > 0) t += fold[e + q];
              if (m == teams - 1) dst[(int64_t)at * a.d + e + q] = t;
              else fold[e + q] = t;
            }
          }
        }
      }
    }
  }
}

// Sum of the blocks' partial rows, one column per thread column of a 32 x 8 block: each of the 8 rows of threads adds every
// eighth block's value, then the eight are added in order.
template <typename TY>
__global__ void __launch_bounds__(256) norm_params_kernel(const float *__restrict__ partial, int blocks, int n_sums, int d,
                                                          TY *d_ls, TY *d_w0, TY *d_w1, int s_ls, int s_w0, int s_w1) {
  __shared__ float part[8][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x & 31, part_i = threadIdx.x >> 5;
  const int n = n_sums * d;
  float s = 0.f;
  if (col < n)
    for (int b = part_i; b < blocks; b += 8) s += partial[(int64_t)b * n + col];
  part[part_i][lane] = s;
  __syncthreads();
  if (part_i == 0 && col < n) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += part[i][lane];
    const int which = col / d, e = col - which * d;
    TY *dst = which == s_ls ? d_ls : which == s_w0 ? d_w0 : d_w1;
    dst[e] = from_f32<TY>(t);
  }
}

struct NormShape { int tw, nv, teams; };

// Warps per row and 8-element pieces per thread.  Up to 1024 columns one warp owns a row (no barriers); wider rows are shared by
// just enough warps for two pieces per thread.
NormShape norm_shape(int d, int max_nv1) {
  NormShape s;
  const int pieces = (d + 7) / 8;
  if (pieces <= 32 * max_nv1) {
    s.tw = 1;
    s.nv = (pieces + 31) / 32;
    if (s.nv == 3) s.nv = 4;
  } else {
    s.nv = pieces <= 256 ? 1 : 2;
    s.tw = (pieces + 32 * s.nv - 1) / (32 * s.nv);
  }
  s.teams = s.tw >= 8 ? 1 : 8 / s.tw;
  return s;
}

bool bad_align(const void *p, int size) { return p && (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(size - 1)); }
bool wide_ok(const void *p, int64_t stride, int size) {
  return !p || (!(reinterpret_cast<uintptr_t>(p) & 15) && (stride * size) % 16 == 0);
}

int check_norm(const tmoe_residual_norm_t *p) {
  if (!p) return TMOE_ERR_NULL;
  if (p->dtype != TMOE_F32 && p->dtype != TMOE_BF16) return TMOE_ERR_DTYPE;
  if (p->residual_dtype != p->dtype && p->residual_dtype != TMOE_F32) return TMOE_ERR_DTYPE;
  if (p->rows < 0 || p->rows > ((int64_t)1 << 30) || p->d <= 0) return TMOE_ERR_SHAPE;
  if (p->d > kMaxWidth) return TMOE_ERR_UNSUPPORTED;
  if (p->y_stride < 0 || p->residual_stride < 0 || p->gate_stride < 0) return TMOE_ERR_SHAPE;
  if (!p->residual && p->residual_dtype != p->dtype) return TMOE_ERR_DTYPE;   // out has y's type then
  if (p->rows == 0) return TMOE_OK;
  if (!p->y) return TMOE_ERR_NULL;
  const int sy = p->dtype == TMOE_F32 ? 4 : 2, sr = p->residual_dtype == TMOE_F32 ? 4 : 2;
  if (bad_align(p->y, sy) || bad_align(p->gate, sy) || bad_align(p->layer_scale, sy) || bad_align(p->post_w, sy) ||
      bad_align(p->next_w, sy) || bad_align(p->residual, sr))
    return TMOE_ERR_ALIGN;
  return TMOE_OK;
}

NormArgs norm_args(const tmoe_residual_norm_t &p) {
  NormArgs a{};
  a.y = p.y; a.res = p.residual; a.ls = p.layer_scale; a.gate = p.gate; a.w0 = p.post_w; a.w1 = p.next_w;
  a.ys = p.y_stride; a.rs = p.residual_stride; a.gs = p.gate_stride;
  a.rows = p.rows; a.d = p.d; a.eps0 = p.post_eps; a.eps1 = p.next_eps;
  a.sum_ls = a.sum_w0 = a.sum_w1 = -1;
  return a;
}

// 16-byte pieces when every row of every tensor starts on a 16-byte boundary and the width is a multiple of 8
bool norm_wide(const tmoe_residual_norm_t &p) {
  const int sy = p.dtype == TMOE_F32 ? 4 : 2, sr = p.residual_dtype == TMOE_F32 ? 4 : 2;
  return p.d % 8 == 0 && wide_ok(p.y, p.y_stride, sy) && wide_ok(p.gate, p.gate_stride, sy) &&
         wide_ok(p.residual, p.residual_stride, sr) && wide_ok(p.layer_scale, 0, sy) && wide_ok(p.post_w, 0, sy) &&
         wide_ok(p.next_w, 0, sy);
}

template <typename TY, typename TR>
void launch_forward(const NormArgs &a0, bool wide, cudaStream_t st) {
  NormArgs a = a0;
  const NormShape s = norm_shape(a.d, 4);
  a.tw = s.tw;
  const dim3 grid((unsigned)((a.rows + s.teams - 1) / s.teams)), block(s.teams * s.tw * 32);
#define TMOE_RN(V, N) residual_norm_kernel<TY, TR, V, N><<<grid, block, 0, st>>>(a)
  if (wide) { if (s.nv == 1) TMOE_RN(8, 1); else if (s.nv == 2) TMOE_RN(8, 2); else TMOE_RN(8, 4); }
  else { if (s.nv == 1) TMOE_RN(1, 8); else if (s.nv == 2) TMOE_RN(1, 16); else TMOE_RN(1, 32); }
#undef TMOE_RN
}

NormShape backward_shape(int d) { return norm_shape(d, 1); }
int backward_blocks(int64_t rows, int d, int sms) {
  const NormShape s = backward_shape(d);
  const int64_t want = (rows + s.teams - 1) / s.teams, cap = (int64_t)sms * (s.tw * s.teams > 8 ? 1 : 2);
  return (int)(want < cap ? want : cap);
}

template <typename TY, typename TR>
void launch_backward(const NormArgs &a0, bool wide, int blocks, cudaStream_t st) {
  NormArgs a = a0;
  const NormShape s = backward_shape(a.d);
  a.tw = s.tw;
  const dim3 grid((unsigned)blocks), block(s.teams * s.tw * 32);
  const size_t smem = s.teams > 1 ? (size_t)a.d * 4 : 0;
#define TMOE_RNB(V, N) residual_norm_backward_kernel<TY, TR, V, N><<<grid, block, smem, st>>>(a)
  if (wide) { if (s.nv == 1) TMOE_RNB(8, 1); else TMOE_RNB(8, 2); }
  else { if (s.nv == 1) TMOE_RNB(1, 8); else TMOE_RNB(1, 16); }
#undef TMOE_RNB
}

}  // namespace
}  // namespace tmoe

using namespace tmoe;

extern "C" {

int tmoe_residual_norm(const tmoe_residual_norm_t *p, void *out, void *normed, float *rstd, void *stream) {
  int rc = check_norm(p);
  if (rc) return rc;
  if (p->rows == 0) return TMOE_OK;
  if ((normed != nullptr) != (p->next_w != nullptr)) return TMOE_ERR_NULL;
  if (!out && !normed) return TMOE_ERR_NULL;
  const int sy = p->dtype == TMOE_F32 ? 4 : 2, sr = p->residual_dtype == TMOE_F32 ? 4 : 2;
  if (bad_align(out, sr) || bad_align(normed, sy) || bad_align(rstd, 4)) return TMOE_ERR_ALIGN;
  NormArgs a = norm_args(*p);
  a.out = out; a.normed = normed; a.rstd = rstd;
  const bool wide = norm_wide(*p) && wide_ok(out, p->d, sr) && wide_ok(normed, p->d, sy);
  cudaStream_t st = (cudaStream_t)stream;
  if (p->dtype == TMOE_F32) launch_forward<float, float>(a, wide, st);
  else if (p->residual_dtype == TMOE_F32) launch_forward<bf16, float>(a, wide, st);
  else launch_forward<bf16, bf16>(a, wide, st);
  count_launch();
  return launch_status();
}

int64_t tmoe_residual_norm_workspace_bytes(const tmoe_residual_norm_t *p) {
  int rc = check_norm(p);
  if (rc) return rc;
  // sized for up to 160 SMs, whatever device the sizing query runs on
  return p->rows == 0 ? 0 : (int64_t)backward_blocks(p->rows, p->d, 160) * 3 * p->d * 4;
}

int tmoe_residual_norm_backward(const tmoe_residual_norm_t *p, const float *rstd, const void *d_out, int64_t d_out_stride,
                                const void *d_normed, int64_t d_normed_stride, void *d_y, void *d_residual, void *d_gate,
                                void *d_layer_scale, void *d_post_w, void *d_next_w, void *workspace, int64_t workspace_bytes,
                                void *stream) {
  int rc = check_norm(p);
  if (rc) return rc;
  const int sy = p->dtype == TMOE_F32 ? 4 : 2, sr = p->residual_dtype == TMOE_F32 ? 4 : 2;
  cudaStream_t st = (cudaStream_t)stream;
  // a gradient of something that is not there
  if ((d_residual && !p->residual) || (d_gate && !p->gate) || (d_layer_scale && !p->layer_scale) || (d_post_w && !p->post_w) ||
      (d_next_w && !p->next_w) || (d_normed && !p->next_w))
    return TMOE_ERR_NULL;
  const bool params = d_layer_scale || d_post_w || d_next_w;
  if (p->rows == 0) {   // sums over no rows
    void *g[3] = {d_layer_scale, d_post_w, d_next_w};
    for (void *q : g)
      if (q && cudaMemsetAsync(q, 0, (size_t)p->d * sy, st) != cudaSuccess) return TMOE_ERR_CUDA;
    return TMOE_OK;
  }
  if (!d_out && !d_normed) return TMOE_ERR_NULL;
  if ((p->post_w || d_normed) && !rstd) return TMOE_ERR_NULL;
  if (d_out_stride < 0 || d_normed_stride < 0) return TMOE_ERR_SHAPE;
  if (bad_align(d_out, sr) || bad_align(d_normed, sy) || bad_align(d_y, sy) || bad_align(d_residual, sr) || bad_align(d_gate, sy) ||
      bad_align(d_layer_scale, sy) || bad_align(d_post_w, sy) || bad_align(d_next_w, sy) || bad_align(rstd, 4) ||
      bad_align(workspace, 16))
    return TMOE_ERR_ALIGN;
  NormArgs a = norm_args(*p);
  a.rstd = const_cast<float *>(rstd);
  a.d_out = d_out; a.dos = d_out_stride; a.d_normed = d_normed; a.dns = d_normed_stride;
  a.d_y = d_y; a.d_res = d_residual; a.d_gate = d_gate;
  if (d_layer_scale) a.sum_ls = a.n_sums++;
  if (d_post_w) a.sum_w0 = a.n_sums++;
  if (d_next_w) a.sum_w1 = a.n_sums++;
  const int sms = current_device_sms();
  if (sms <= 0) return TMOE_ERR_CUDA;
  const int blocks = backward_blocks(p->rows, p->d, sms < 160 ? sms : 160);
  if (params) {
    if (!workspace) return TMOE_ERR_NULL;
    if (workspace_bytes < (int64_t)blocks * a.n_sums * p->d * 4) return TMOE_ERR_WORKSPACE;
    a.partial = reinterpret_cast<float *>(workspace);
  }
  const bool wide = norm_wide(*p) && wide_ok(d_out, d_out_stride, sr) && wide_ok(d_normed, d_normed_stride, sy) &&
                    wide_ok(d_y, p->d, sy) && wide_ok(d_residual, p->d, sr) && wide_ok(d_gate, p->d, sy);
  if (p->dtype == TMOE_F32) launch_backward<float, float>(a, wide, blocks, st);
  else if (p->residual_dtype == TMOE_F32) launch_backward<bf16, float>(a, wide, blocks, st);
  else launch_backward<bf16, bf16>(a, wide, blocks, st);
  count_launch();
  if ((rc = launch_status())) return rc;
  if (params) {
    const dim3 grid((unsigned)((a.n_sums * p->d + 31) / 32));
    if (p->dtype == TMOE_F32)
      norm_params_kernel<float><<<grid, 256, 0, st>>>(a.partial, blocks, a.n_sums, p->d, (float *)d_layer_scale, (float *)d_post_w,
                                                      (float *)d_next_w, a.sum_ls, a.sum_w0, a.sum_w1);
    else
      norm_params_kernel<bf16><<<grid, 256, 0, st>>>(a.partial, blocks, a.n_sums, p->d, (bf16 *)d_layer_scale, (bf16 *)d_post_w,
                                                     (bf16 *)d_next_w, a.sum_ls, a.sum_w0, a.sum_w1);
    count_launch();
    rc = launch_status();
  }
  return rc;
}

}  // extern "C"
