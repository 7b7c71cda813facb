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
// The sums of d_layer_scale and d_post_w differ by a column factor only: with S = sum_t dR * s * h they are post_w * S and
// layer_scale * S.
// `out` is recomputed in fp32 from y, gate and residual (the same bytes as reading it back, and no rounding in between); only
// the two rstd of a row are kept from the forward pass.
#include "column_sum.cuh"
#include "common.cuh"
#include "kernels.h"
#include "pair.cuh"
#include "ptx.cuh"

namespace tmoe {
namespace {

constexpr int kMaxWidth = 8192;      // widest row: 512 threads x 16 elements
// Warps that an SM is meant to hold, by the registers a thread needs.  Forward 32 (64 registers) in blocks of 8 or of one row each;
// backward one block of 20 (96 registers), or 16 (128) in fp32; 16 where a thread has 16 elements, 18 (96 registers) in the fp32 forward without
// a gate, so that two blocks of 9 fit (4608 columns: 51 us against 75).
constexpr int resident_warps(int nv, bool back, bool f32, bool gate) {
  return nv == 2 ? (f32 && !back && !gate ? 18 : 16) : back ? (f32 ? 16 : 20) : 32;
}
// Warps of the largest block
constexpr int block_warps(int nv, bool back, bool f32) { return back ? resident_warps(nv, back, f32, true) : 16; }
constexpr int kMaxTeams = 10;           // teams of several warps in a block (a named barrier each)
constexpr int kRingBytes = 208 * 1024;

// sigmoid to a few ulp (the gate is one factor of a sum that is rounded to the storage type).  exp(-g) beyond the range is 0 or infinite,
// and its reciprocal 1 or 0.
__device__ __forceinline__ f2 sigmoid2(f2 g) {
  float a, b;
  split(mul2(g, both(-kLog2e)), a, b);
  split(add2(pair(fast_exp2(a), fast_exp2(b)), both(1.f)), a, b);
  return pair(fast_rcp(a), fast_rcp(b));
}

__device__ __forceinline__ void cp_async16(void *smem, const void *gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ptx::smem_u32(smem)), "l"(gmem) : "memory");
}
// through L1: for two copies that share a 32-byte sector, so that it crosses from L2 once
__device__ __forceinline__ void cp_async16_l1(void *smem, const void *gmem) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(ptx::smem_u32(smem)), "l"(gmem) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// VEC consecutive elements of a row as they lie in memory (VEC = 8: 16-byte loads; VEC = 1: any width, stride and base).
// kPlanes 16-byte parts, part p of a thread at slot[p * pitch] of a shared-memory ring.
template <typename T, int VEC> struct Piece;
template <> struct Piece<bf16, 8> {
  static constexpr int kPlanes = 1;
  uint4 r;
  __device__ static __forceinline__ void copy(uint4 *slot, int, const bf16 *p) { cp_async16(slot, p); }
  __device__ __forceinline__ void fetch(const uint4 *slot, int) { r = *slot; }
  __device__ __forceinline__ void load(const bf16 *p) { r = *reinterpret_cast<const uint4 *>(p); }
  __device__ __forceinline__ void zero() { r = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void one() { r = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u); }
  __device__ __forceinline__ f2 get2(int j) const {   // elements 2j, 2j + 1
    const uint32_t w = j == 0 ? r.x : j == 1 ? r.y : j == 2 ? r.z : r.w;
    return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  __device__ static __forceinline__ uint32_t pack(f2 v) { float a, b; split(v, a, b); return pack_bf16x2(a, b); }
  __device__ static __forceinline__ void store(bf16 *p, const f2 *f) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack(f[0]), pack(f[1]), pack(f[2]), pack(f[3]));
  }
};
template <> struct Piece<float, 8> {
  static constexpr int kPlanes = 2;
  float4 a, b;
  __device__ static __forceinline__ void copy(uint4 *slot, int pitch, const float *p) { cp_async16_l1(slot, p); cp_async16_l1(slot + pitch, p + 4); }
  __device__ __forceinline__ void fetch(const uint4 *slot, int pitch) {
    a = *reinterpret_cast<const float4 *>(slot);
    b = *reinterpret_cast<const float4 *>(slot + pitch);
  }
  __device__ __forceinline__ void load(const float *p) {
    a = reinterpret_cast<const float4 *>(p)[0];
    b = reinterpret_cast<const float4 *>(p)[1];
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void one() { a = b = make_float4(1.f, 1.f, 1.f, 1.f); }
  __device__ __forceinline__ f2 get2(int j) const {
    const float4 v = j < 2 ? a : b;
    return (j & 1) ? pair(v.z, v.w) : pair(v.x, v.y);
  }
  __device__ static __forceinline__ void store(float *p, const f2 *f) {
    asm volatile("st.global.v4.b64 [%0], {%1, %2, %3, %4};" ::"l"(p), "l"(f[0]), "l"(f[1]), "l"(f[2]), "l"(f[3]) : "memory");
  }
};
template <typename T> struct Piece<T, 1> {
  static constexpr int kPlanes = 0;
  T r;
  __device__ static __forceinline__ void copy(uint4 *, int, const T *) {}
  __device__ __forceinline__ void fetch(const uint4 *, int) {}
  __device__ __forceinline__ void load(const T *p) { r = *p; }
  __device__ __forceinline__ void zero() { r = from_f32<T>(0.f); }
  __device__ __forceinline__ void one() { r = from_f32<T>(1.f); }
  __device__ __forceinline__ float get() const { return to_f32(r); }
};

// Pairs over a thread's NV * VEC elements: neighbours in a piece, or two pieces where a piece is one element.
template <typename T, int NV> __device__ __forceinline__ f2 pair_of(const Piece<T, 8> (&p)[NV], int j) { return p[j / 4].get2(j % 4); }
template <typename T, int NV> __device__ __forceinline__ f2 pair_of(const Piece<T, 1> (&p)[NV], int j) { return pair(p[2 * j].get(), p[2 * j + 1].get()); }
// Stores a thread's pairs to columns (i * tpr + lt) * VEC ... of one row of width d.
template <typename T, int VEC, int NV>
__device__ __forceinline__ void store_row(T *row, int tpr, int lt, int d, const f2 (&f)[NV * VEC / 2]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * tpr + lt) * VEC;
    if (e < d) {
      if constexpr (VEC == 8) {
        Piece<T, 8>::store(row + e, f + i * 4);
      } else {
        float a, b;
        split(f[i / 2], a, b);
        row[e] = from_f32<T>((i & 1) ? b : a);
      }
    }
  }
}

struct NormArgs {
  const void *y, *res, *ls, *gate, *w0, *w1;  // inputs; nullptr = the term is absent
  int64_t ys, rs, gs;                          // row strides in elements
  int64_t rows;
  int d, tw;                                   // row width; warps per row ("team")
  int step;                                    // rows between two rows of one team: blocks * teams of a block
  int64_t y_step, r_step, g_step, do_step, dn_step, o_step;   // step times the row strides, and times d
  float eps0, eps1;
  void *out, *normed;                          // forward outputs [rows, d]; either may be nullptr
  float *rstd;                                 // [2, rows]: 1/rms of y and of out; nullptr = not kept
  // backward
  const void *d_out, *d_normed;
  int64_t dos, dns;
  void *d_y, *d_res, *d_gate;                  // [rows, d]; nullptr = not wanted
  float *partial;                              // [blocks, n_sums, d] column sums; nullptr = no parameter gradient wanted
  int sum_a, sum_x;                            // slot in `partial` of sum_t dR * s * h and of sum_t dN * x, or -1
  int n_sums;
};

// Sums over the `tw` warps of a team, in a fixed order.  A team has 20 places of shared memory for each sum, zero beyond its own warps
// (TeamRed::init), which every thread reads back with wide loads; `slot` alternates between calls, so one barrier per call is enough.
template <int N> struct TeamRed {
  float at[2][kMaxTeams][N][20];   // [slot][team][sum][warp]
  __device__ __forceinline__ void init() {
    for (int i = threadIdx.x; i < 2 * kMaxTeams * N * 20; i += blockDim.x) (&at[0][0][0][0])[i] = 0.f;
    __syncthreads();
  }
};
__device__ __forceinline__ float sum_places(const float (&v)[20], int tw) {
  const ulonglong2 *p = reinterpret_cast<const ulonglong2 *>(v);
  f2 s = add2(p[0].x, p[0].y);
  if (tw > 4) {
    s = add2(s, add2(p[1].x, p[1].y));
    if (tw > 8) {
      s = add2(s, add2(add2(p[2].x, p[2].y), add2(p[3].x, p[3].y)));
      if (tw > 16) s = add2(s, add2(p[4].x, p[4].y));
    }
  }
  return sum2(s);
}
__device__ __forceinline__ float team_sum(float v, int tw, int team, int slot, TeamRed<1> &red) {
  v = warp_sum(v);
  if (tw == 1) return v;
  if ((threadIdx.x & 31) == 0) red.at[slot][team][0][(threadIdx.x >> 5) - team * tw] = v;
  ptx::named_bar_sync(1 + team, tw * 32);
  return sum_places(red.at[slot][team][0], tw);
}

// The same for three sums at once.  The first two steps of the butterfly halve the number of values a lane carries, so three sums
// take 6 shuffles instead of 15.
__device__ __forceinline__ float3 team_sum3(float a, float b, float c, int tw, int team, int slot, TeamRed<3> &red) {
  const int lane = threadIdx.x & 31;
  const bool hi = lane & 16, up = lane & 8;
  float p = (hi ? c : a) + __shfl_xor_sync(0xffffffffu, hi ? a : c, 16);
  float q = (hi ? 0.f : b) + __shfl_xor_sync(0xffffffffu, hi ? b : 0.f, 16);
  p = (up ? q : p) + __shfl_xor_sync(0xffffffffu, up ? p : q, 8);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) p += __shfl_xor_sync(0xffffffffu, p, o);
  // lanes 0.. hold a, 8.. b, 16.. c
  if (tw == 1)
    return make_float3(__shfl_sync(0xffffffffu, p, 0), __shfl_sync(0xffffffffu, p, 8), __shfl_sync(0xffffffffu, p, 16));
  if ((lane & 7) == 0 && lane < 24) red.at[slot][team][lane >> 3][(threadIdx.x >> 5) - team * tw] = p;
  ptx::named_bar_sync(1 + team, tw * 32);
  return make_float3(sum_places(red.at[slot][team][0], tw), sum_places(red.at[slot][team][1], tw), sum_places(red.at[slot][team][2], tw));
}

extern __shared__ uint4 norm_ring[];

// One row's inputs as they lie in memory, and the walk of a team over its rows.  Where the ring has stages, a row's pieces are copied to
// shared memory some rows ahead; a thread copies and reads its own pieces only, so the ring needs no barrier, just the thread's own
// wait for its copies.  What is never copied (an absent operand, a column beyond the row) is zero in the ring from the start, so reading
// needs no conditions.
template <typename TY, typename TR, int VEC, int NV, bool GATE, bool BACK> struct RowIn {
  using PY = Piece<TY, VEC>;
  using PR = Piece<TR, VEC>;
  static constexpr int kPlanes = NV * ((1 + (GATE ? 1 : 0) + (BACK ? 1 : 0)) * PY::kPlanes + (BACK ? 2 : 1) * PR::kPlanes);
  // as many rows ahead as fit for the warps that an SM is meant to run; below 2 stages rows are loaded when their turn comes
  // (backward, the parameters' columns of a thread lie behind the ring, in fp32).  The fp32 forward loads without a ring: its 32-byte pieces
  // keep as much in flight from registers (18.9 M elements with a gate, 2304 columns: 60.5 us against 70.9 with a ring, 768: 59.3 / 70.8, 8192:
  // 70.1 / 83.1, without a gate 1520: 49.4 / 58.1; only the gated blocks of 9 to 15 warps lose, 4608: 84.2 / 79.5); bf16 needs it (37.7 M elements of
  // 2304 columns: 49.4 us against 73.8 without).
  static constexpr int kParamPlanes = BACK && VEC == 8 ? 4 * NV : 0;
  static constexpr int kFit = kPlanes ? (kRingBytes / (resident_warps(NV, BACK, sizeof(TY) == 4, GATE) * 512) - kParamPlanes) / kPlanes : 0;
  static constexpr int kStages = sizeof(TY) == 4 && !BACK ? 1 : kFit >= 3 ? 3 : kFit == 2 ? 2 : 1;
  static constexpr bool kRing = kStages > 1;
  PY y[NV], g[GATE ? NV : 1], dn[BACK ? NV : 1];
  PR r[NV], dout[BACK ? NV : 1];
};

template <typename TY, typename TR, int VEC, int NV, bool GATE, bool BACK> struct RowWalk {
  using In = RowIn<TY, TR, VEC, NV, GATE, BACK>;
  using PY = Piece<TY, VEC>;
  using PR = Piece<TR, VEC>;
  // this thread's first piece in the row that is copied (or, without a ring, loaded) next
  const TY *y, *g, *dn;
  const TR *r, *o;
  int ahead;           // that row (rows + 3 * step < 2^31)
  uint4 *slot;
  int stage;

  __device__ __forceinline__ RowWalk(const NormArgs &a, int row, int lt) : ahead(row), slot(norm_ring + threadIdx.x), stage(0) {
    y = (const TY *)a.y + (int64_t)row * a.ys + lt * VEC;
    g = (const TY *)a.gate + (int64_t)row * a.gs + lt * VEC;
    dn = (const TY *)a.d_normed + (int64_t)row * a.dns + lt * VEC;
    r = (const TR *)a.res + (int64_t)row * a.rs + lt * VEC;
    o = (const TR *)a.d_out + (int64_t)row * a.dos + lt * VEC;
    if (In::kRing) {
#pragma unroll
      for (int i = 0; i < In::kStages * In::kPlanes; ++i) slot[i * blockDim.x] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int s = 0; s < In::kStages - 1; ++s) copy(a, lt, at(s));
    }
  }
  __device__ __forceinline__ uint4 *at(int s) const { return slot + s * In::kPlanes * blockDim.x; }
  __device__ __forceinline__ uint4 *behind() const { return at(In::kStages); }
  __device__ __forceinline__ void advance(const NormArgs &a) {
    ahead += a.step;
    y += a.y_step;
    r += a.r_step;
    if (GATE) g += a.g_step;
    if (BACK) { dn += a.dn_step; o += a.do_step; }
  }
  __device__ __forceinline__ void copy(const NormArgs &a, int lt, uint4 *to) {
    if (ahead < (int)a.rows) {
      const int pitch = blockDim.x, tpr = a.tw * 32;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = i * tpr * VEC;
        if (lt * VEC + e < a.d) {
          PY::copy(to, pitch, y + e);
          if (GATE) PY::copy(to + PY::kPlanes * pitch, pitch, g + e);
          if (a.res) PR::copy(to + kR * pitch, pitch, r + e);
          if (BACK && a.d_normed) PY::copy(to + kN * pitch, pitch, dn + e);
          if (BACK && a.d_out) PR::copy(to + kO * pitch, pitch, o + e);
        }
        to += In::kPlanes / NV * pitch;
      }
    }
    advance(a);
    cp_async_commit();
  }
  // planes of one piece: y, gate, residual, d_normed, d_out
  static constexpr int kR = (GATE ? 2 : 1) * PY::kPlanes, kN = kR + PR::kPlanes, kO = kN + PY::kPlanes;
  __device__ __forceinline__ void fetch(const uint4 *from, In &in) const {
    const int pitch = blockDim.x;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      in.y[i].fetch(from, pitch);
      if (GATE) in.g[i].fetch(from + PY::kPlanes * pitch, pitch);
      in.r[i].fetch(from + kR * pitch, pitch);
      if (BACK) { in.dn[i].fetch(from + kN * pitch, pitch); in.dout[i].fetch(from + kO * pitch, pitch); }
      from += In::kPlanes / NV * pitch;
    }
  }
  __device__ __forceinline__ void take(const NormArgs &a, int lt, In &in) {
    if (In::kRing) {
      copy(a, lt, at(stage == 0 ? In::kStages - 1 : stage - 1));
      cp_async_wait<In::kStages - 1>();
      fetch(at(stage), in);
      stage = stage + 1 == In::kStages ? 0 : stage + 1;
    } else {
      const int tpr = a.tw * 32;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = i * tpr * VEC;
        in.y[i].zero(); in.r[i].zero();
        if (GATE) in.g[i].zero();
        if (BACK) { in.dn[i].zero(); in.dout[i].zero(); }
        if (lt * VEC + e < a.d) {
          in.y[i].load(y + e);
          if (a.res) in.r[i].load(r + e);
          if (GATE) in.g[i].load(g + e);
          if (BACK) {
            if (a.d_out) in.dout[i].load(o + e);
            if (a.d_normed) in.dn[i].load(dn + e);
          }
        }
      }
      advance(a);
    }
  }
  // the row taken last, once more
  __device__ __forceinline__ void again(In &in) const { fetch(at(stage == 0 ? In::kStages - 1 : stage - 1), in); }
};

// The parameter vectors' columns of one thread (1 where a factor is absent): c = post_w * layer_scale, w1 = next_w.
template <typename TY, int VEC, int NV> struct Params {
  static constexpr int N2 = NV * VEC / 2;
  f2 c[N2], w1[N2];
  __device__ __forceinline__ void load(const NormArgs &a, int lt) {
    Piece<TY, VEC> p0[NV], pl[NV], p1[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * a.tw * 32 + lt) * VEC;
      p0[i].zero(); pl[i].zero(); p1[i].zero();
      if (e < a.d) {
        if (a.w0) p0[i].load((const TY *)a.w0 + e); else p0[i].one();
        if (a.ls) pl[i].load((const TY *)a.ls + e); else pl[i].one();
        if (a.w1) p1[i].load((const TY *)a.w1 + e);
      }
    }
#pragma unroll
    for (int j = 0; j < N2; ++j) { c[j] = mul2(pair_of(p0, j), pair_of(pl, j)); w1[j] = pair_of(p1, j); }
  }
  // 16-byte parts: c first, then w1
  __device__ __forceinline__ void keep(uint4 *slot) const {
#pragma unroll
    for (int j = 0; j < N2; j += 2) {
      *reinterpret_cast<ulonglong2 *>(slot + j / 2 * blockDim.x) = make_ulonglong2(c[j], c[j + 1]);
      *reinterpret_cast<ulonglong2 *>(slot + (N2 / 2 + j / 2) * blockDim.x) = make_ulonglong2(w1[j], w1[j + 1]);
    }
  }
  __device__ __forceinline__ void fetch(const uint4 *slot) {
#pragma unroll
    for (int j = 0; j < N2; j += 2) {
      const ulonglong2 p = *reinterpret_cast<const ulonglong2 *>(slot + j / 2 * blockDim.x);
      const ulonglong2 q = *reinterpret_cast<const ulonglong2 *>(slot + (N2 / 2 + j / 2) * blockDim.x);
      c[j] = p.x; c[j + 1] = p.y; w1[j] = q.x; w1[j + 1] = q.y;
    }
  }
};

// A team walks over rows blockIdx * teams + team, + gridDim * teams, ...  Bound by memory: 32768 x 768 bf16 with every operand in 43 us
// = 5.8 TB/s of 252 MB, 16384 x 2304 without a gate in 50 us = 6.1 TB/s.
template <typename TY, typename TR, int VEC, int NV, bool GATE>
__global__ void __launch_bounds__(VEC == 8 && NV == 2 && sizeof(TY) == 4 && !GATE ? 576 : 512, VEC == 8 && NV == 1 ? 2 : 1) residual_norm_kernel(const __grid_constant__ NormArgs a) {
  using In = RowIn<TY, TR, VEC, NV, GATE, false>;
  __shared__ __align__(16) TeamRed<1> red;
  ptx::griddep_launch_dependents();
  red.init();
  ptx::griddep_wait();   // the operands may come from the kernel before this one
  const int tpr = a.tw * 32, team = threadIdx.x / tpr, lt = threadIdx.x - team * tpr;
  int row = blockIdx.x * (blockDim.x / tpr) + team;
  int64_t off = (int64_t)row * a.d;     // of the row in the outputs
  const float inv_d = 1.f / (float)a.d;
  RowWalk<TY, TR, VEC, NV, GATE, false> walk(a, row, lt);
  Params<TY, VEC, NV> w;
  w.load(a, lt);
  int slot = 0;
  for (; row < (int)a.rows; row += a.step, off += a.o_step) {
    In in;
    walk.take(a, lt, in);
    constexpr int N2 = NV * VEC / 2;
    float rho0 = 1.f;
    if (a.w0) {
      f2 ss = both(0.f);
#pragma unroll
      for (int j = 0; j < N2; ++j) ss = fma2(pair_of(in.y, j), pair_of(in.y, j), ss);
      rho0 = rsqrtf(fmaf(team_sum(sum2(ss), a.tw, team, slot, red), inv_d, a.eps0));
      slot ^= 1;
      if (a.rstd && lt == 0) a.rstd[row] = rho0;
    }
    f2 v[N2], ss = both(0.f);
#pragma unroll
    for (int j = 0; j < N2; ++j) {
      f2 t = mul2(mul2(pair_of(in.y, j), both(rho0)), w.c[j]);
      if (GATE) { const f2 g = pair_of(in.g, j); t = mul2(t, mul2(g, sigmoid2(g))); }
      v[j] = add2(t, pair_of(in.r, j));
      ss = fma2(v[j], v[j], ss);
    }
    if (a.out) store_row<TR, VEC, NV>((TR *)a.out + off, tpr, lt, a.d, v);
    if (!a.normed) continue;
    const float rho1 = rsqrtf(fmaf(team_sum(sum2(ss), a.tw, team, slot, red), inv_d, a.eps1));
    slot ^= 1;
    if (a.rstd && lt == 0) a.rstd[a.rows + row] = rho1;
#pragma unroll
    for (int j = 0; j < N2; ++j) v[j] = mul2(v[j], mul2(both(rho1), w.w1[j]));
    store_row<TY, VEC, NV>((TY *)a.normed + off, tpr, lt, a.d, v);
  }
}

// Without a norm nothing ties a row's elements together: threads walk over the 8-element pieces of all rows, `per_row` to a row, a grid of
// pieces ahead (row_step rows and col_step pieces, so that no division is needed), two of them in flight.  The arithmetic is the row
// kernel's.  For whole pieces only: 8398 x 1520 fp32 + residual in 23.9 us = 6.4 TB/s (the row walk: 30.5), 32768 x 768 bf16 with a gate
// 31.8 us (34.3); element by element it is slower than the row walk (20000 x 1001 bf16: 60.7 against 42.7 us), which those widths keep.
constexpr int kMapThreads = 256, kMapAhead = 2;
template <typename TY, typename TR, bool GATE>
__global__ void __launch_bounds__(kMapThreads) residual_map_kernel(const __grid_constant__ NormArgs a, int per_row, int row_step, int col_step) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const uint32_t first = blockIdx.x * kMapThreads + threadIdx.x;
  int row = (int)(first / (uint32_t)per_row), col = (int)(first - (uint32_t)row * per_row);
  while (row < (int)a.rows) {   // (rows + kMapAhead * (row_step + 1) < 2^31)
    Piece<TY, 8> y[kMapAhead], g[kMapAhead], s[kMapAhead];
    Piece<TR, 8> r[kMapAhead];
    int at_row[kMapAhead], at[kMapAhead];
#pragma unroll
    for (int b = 0; b < kMapAhead; ++b) {
      at_row[b] = row; at[b] = col * 8;
      if (row < (int)a.rows) {
        y[b].load((const TY *)a.y + row * a.ys + at[b]);
        if (GATE) g[b].load((const TY *)a.gate + row * a.gs + at[b]);
        if (a.res) r[b].load((const TR *)a.res + row * a.rs + at[b]); else r[b].zero();
        if (a.ls) s[b].load((const TY *)a.ls + at[b]); else s[b].one();
      }
      row += row_step;
      col += col_step;
      if (col >= per_row) { col -= per_row; ++row; }
    }
#pragma unroll
    for (int b = 0; b < kMapAhead; ++b) {
      if (at_row[b] < (int)a.rows) {
        f2 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f2 t = mul2(y[b].get2(j), s[b].get2(j));
          if (GATE) { const f2 q = g[b].get2(j); t = mul2(t, mul2(q, sigmoid2(q))); }
          v[j] = add2(t, r[b].get2(j));
        }
        Piece<TR, 8>::store((TR *)a.out + (int64_t)at_row[b] * a.d + at[b], v);
      }
    }
  }
}

// The same walk; every thread owns the same columns in all rows, so the parameter gradients are sums in its registers:
// d_next_w = sum dN * x, and d_layer_scale and d_post_w are post_w and layer_scale times the same sum dR * s * h.  At the end a block
// adds its teams in order and writes one row of partial sums; norm_params_kernel adds the blocks in order.  The result depends on the
// sizes and the grid only.  16384 x 2304 bf16 with every operand but the gate: 453 MB in 85 us = 5.35 TB/s, the instruction slots 56 % busy;
// what is missing to the forward's rate is the chain of a row (wait, sum, barrier, second pass) that 15 warps an SM do not cover.
template <typename TY, typename TR, int VEC, int NV, bool GATE>
__global__ void __launch_bounds__(32 * block_warps(VEC == 8 ? NV : NV / 8, true, sizeof(TY) == 4)) residual_norm_backward_kernel(const __grid_constant__ NormArgs a) {
  using In = RowIn<TY, TR, VEC, NV, GATE, true>;
  __shared__ __align__(16) TeamRed<3> red;
  ptx::griddep_launch_dependents();
  red.init();
  ptx::griddep_wait();
  const int tpr = a.tw * 32, team = threadIdx.x / tpr, lt = threadIdx.x - team * tpr, teams = blockDim.x / tpr;
  int row = blockIdx.x * teams + team;
  int64_t off = (int64_t)row * a.d;     // of the row in the outputs
  const float inv_d = 1.f / (float)a.d;
  RowWalk<TY, TR, VEC, NV, GATE, true> walk(a, row, lt);
  // Registers are what decides how many rows an SM works on.  With a ring a thread reads its pieces of the row and of the parameters
  // from shared memory in both passes over the row, so that only x, b and the sums stay in registers across the reduction.
  Params<TY, VEC, NV> w;
  w.load(a, lt);
  if (In::kRing) w.keep(walk.behind());
  constexpr int N2 = NV * VEC / 2;
  f2 acc_a[N2], acc_x[N2];
#pragma unroll
  for (int j = 0; j < N2; ++j) acc_a[j] = acc_x[j] = both(0.f);
  int slot = 0;
  // without dN nothing flows through the next norm; one row's rstd are loaded a row ahead
  const float *rstd0 = a.rstd + row, *rstd1 = rstd0 + a.rows;
  float next0 = a.w0 && row < (int)a.rows ? *rstd0 : 1.f, next1 = a.d_normed && row < (int)a.rows ? *rstd1 : 0.f;
  for (; row < (int)a.rows; row += a.step, off += a.o_step) {
    const float rho0 = next0, rho1 = next1;
    rstd0 += a.step;
    rstd1 += a.step;
    if (row + a.step < (int)a.rows) {
      if (a.w0) next0 = *rstd0;
      if (a.d_normed) next1 = *rstd1;
    }
    In in;
    walk.take(a, lt, in);
    if (In::kRing) w.fetch(walk.behind());
    f2 x[N2], b[N2], s1 = both(0.f), s2 = s1, s3 = s1;   // sum u*x, sum q*b, sum q*x
    const f2 r0 = both(rho0), r1 = both(rho1);
#pragma unroll
    for (int j = 0; j < N2; ++j) {
      f2 t = mul2(mul2(pair_of(in.y, j), r0), w.c[j]);
      if (GATE) { const f2 g = pair_of(in.g, j); t = mul2(t, mul2(g, sigmoid2(g))); }
      x[j] = mul2(add2(pair_of(in.r, j), t), r1);
      const f2 u = mul2(w.w1[j], pair_of(in.dn, j));
      b[j] = fma2(r1, u, pair_of(in.dout, j));
      s1 = fma2(u, x[j], s1);
      s2 = fma2(t, b[j], s2);
      s3 = fma2(t, x[j], s3);
    }
    float k1 = 0.f, k0 = 0.f;
    if (a.w0 || a.d_normed) {
      const float3 r = team_sum3(sum2(s1), sum2(s2), sum2(s3), a.tw, team, slot, red);
      slot ^= 1;
      k1 = rho1 * r.x * inv_d;
      k0 = a.w0 ? rho0 * inv_d * (r.y - k1 * r.z) : 0.f;
    }
    if (In::kRing) {
      walk.again(in);
      w.fetch(walk.behind());
    }
    const f2 n1 = both(-k1), n0 = both(-k0);
#pragma unroll
    for (int j = 0; j < N2; ++j) {
      b[j] = fma2(n1, x[j], b[j]);                                     // dR
      acc_x[j] = fma2(pair_of(in.dn, j), x[j], acc_x[j]);
    }
    if (a.d_res) store_row<TR, VEC, NV>((TR *)a.d_res + off, tpr, lt, a.d, b);
    if (GATE) {
      f2 f[N2];
#pragma unroll
      for (int j = 0; j < N2; ++j) {
        const f2 g = pair_of(in.g, j), sg = sigmoid2(g), s = mul2(g, sg);
        const f2 ch = mul2(mul2(pair_of(in.y, j), r0), w.c[j]);
        // silu'(g) = sg + silu(g) * (1 - sg)
        f[j] = mul2(mul2(b[j], ch), fma2(s, fma2(sg, both(-1.f), both(1.f)), sg));
        b[j] = mul2(b[j], s);                                          // dR * s
      }
      if (a.d_gate) store_row<TY, VEC, NV>((TY *)a.d_gate + off, tpr, lt, a.d, f);
    }
#pragma unroll
    for (int j = 0; j < N2; ++j) {
      const f2 h = mul2(pair_of(in.y, j), r0);
      acc_a[j] = fma2(b[j], h, acc_a[j]);
      b[j] = fma2(mul2(b[j], r0), w.c[j], mul2(n0, h));
    }
    if (a.d_y) store_row<TY, VEC, NV>((TY *)a.d_y + off, tpr, lt, a.d, b);
  }
  if (!a.partial) return;
  // [d] floats where the ring was, when a block has several teams: all of its copies have landed and been read by then
  cp_async_wait<0>();
  float *fold = reinterpret_cast<float *>(norm_ring);
  float *dst = a.partial + (int64_t)blockIdx.x * a.n_sums * a.d;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int at = k == 0 ? a.sum_a : a.sum_x;
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
              const int n = i * VEC + q;
              float lo, hi;
              split(k == 0 ? acc_a[n / 2] : acc_x[n / 2], lo, hi);
              float t = (n & 1) ? hi : lo;
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

// Adds the blocks' partial rows and turns the sums into the parameter gradients.
template <typename TY>
__global__ void __launch_bounds__(kColumnSumThreads) norm_params_kernel(const __grid_constant__ NormArgs a, int blocks, TY *d_ls, TY *d_w0, TY *d_w1) {
  __shared__ float part[32][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), n = a.n_sums * a.d;
  ptx::griddep_wait();
  const float t = column_sum(a.partial, blocks, n, col, part);
  if (threadIdx.x < 32 && col < n) {
    const int which = col / a.d, e = col - which * a.d;
    if (which == a.sum_x) {
      d_w1[e] = from_f32<TY>(t);
    } else {
      if (d_ls) d_ls[e] = from_f32<TY>(a.w0 ? t * to_f32(((const TY *)a.w0)[e]) : t);
      if (d_w0) d_w0[e] = from_f32<TY>(a.ls ? t * to_f32(((const TY *)a.ls)[e]) : t);
    }
  }
}

struct NormShape { int tw, nv, teams, blocks; };

// Warps per row, 8-element pieces per thread, rows worked on at once by a block, blocks.
//
// Two pieces a thread halve what a row costs besides its elements (reduction, barrier, addresses); one piece leaves room for more
// threads and, on few rows, is quicker through its chain.  Measured over 37.7 M elements with all operands but the gate, one / two:
// forward d = 384: 52.9 / 55.4 us, 768: 64.0 / 50.8, 2304: 54.4 / 49.6, 4096: 53.9 / 49.5; backward d = 768: 85.3 / 88.4, 1536:
// 93.8 / 82.1, 2304: 107.8 / 87.9, 4096: 112.2 / 88.1.  Backward with a gate, or in fp32, two pieces' ring does not fit (or their registers
// spill): 310 us against 78 us at 768 with a gate.  Few rows are spread over the SMs before a block takes several.
NormShape norm_shape(const tmoe_residual_norm_t &p, bool back, int sms) {
  NormShape s;
  const bool f32 = p.dtype == TMOE_F32;
  const int64_t rows = p.rows;
  const int pieces = (p.d + 7) / 8;
  const bool two = back ? pieces > 128 && !f32 && p.residual_dtype == TMOE_BF16 && !p.gate : pieces > 64;
  s.nv = pieces > 32 * block_warps(1, back, f32) || (two && rows > sms) ? 2 : 1;
  s.tw = (pieces + 32 * s.nv - 1) / (32 * s.nv);
  const int resident = resident_warps(s.nv, back, f32, p.gate != nullptr), full = back ? resident : 8;
  s.teams = s.tw >= full ? 1 : full / s.tw;
  if (s.tw > 1 && s.teams > kMaxTeams) s.teams = kMaxTeams;
  const int64_t each = (rows + sms - 1) / sms;
  if (each < s.teams) s.teams = each < 1 ? 1 : (int)each;
  const int per_sm = back || s.tw * s.teams > resident ? 1 : resident / (s.tw * s.teams);
  const int64_t want = (rows + s.teams - 1) / s.teams, cap = (int64_t)sms * per_sm;
  s.blocks = (int)(want < cap ? want : cap);
  return s;
}

// Blocks of the backward walk at most: one on each SM (sized for up to 160, whatever device a sizing query runs on)
int64_t max_partials(int64_t rows) { return rows < 160 ? rows : 160; }

bool bad_align(const void *p, int size) { return p && (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(size - 1)); }
// rows of 8-element pieces that each start on a multiple of their size (16 bytes in bf16, 32 in fp32)
bool wide_ok(const void *p, int64_t stride, int size) { return !p || (!(reinterpret_cast<uintptr_t>(p) & (8 * size - 1)) && stride % 8 == 0); }

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
  a.sum_a = a.sum_x = -1;
  return a;
}

// 8-element pieces when every row of every tensor starts on a piece's boundary and the width is a multiple of 8
bool norm_wide(const tmoe_residual_norm_t &p) {
  const int sy = p.dtype == TMOE_F32 ? 4 : 2, sr = p.residual_dtype == TMOE_F32 ? 4 : 2;
  return p.d % 8 == 0 && wide_ok(p.y, p.y_stride, sy) && wide_ok(p.gate, p.gate_stride, sy) &&
         wide_ok(p.residual, p.residual_stride, sr) && wide_ok(p.layer_scale, 0, sy) && wide_ok(p.post_w, 0, sy) &&
         wide_ok(p.next_w, 0, sy);
}

// Launch with the ring's shared memory; its size (and that the SM should be split for it: without that fewer blocks are resident
// than the grid counts on) is declared once per kernel and device
template <typename In, typename Kernel>
int launch_walk(Kernel kernel, const NormArgs &a, const NormShape &s, bool fold, cudaStream_t st) {
  static std::atomic<uint64_t> opted{0};
  const int threads = s.teams * s.tw * 32;
  size_t smem = In::kRing ? (size_t)(In::kStages * In::kPlanes + In::kParamPlanes) * threads * 16 : 0;
  if (fold && s.teams > 1 && smem < (size_t)a.d * 4) smem = (size_t)a.d * 4;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return TMOE_ERR_CUDA;
  const uint64_t bit = 1ull << (dev & 63);
  if (In::kRing && !(opted.load(std::memory_order_relaxed) & bit)) {
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes);
    cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    opted.fetch_or(bit, std::memory_order_relaxed);
  }
  NormArgs b = a;
  b.step = s.blocks * s.teams;
  b.y_step = b.step * a.ys; b.r_step = b.step * a.rs; b.g_step = b.step * a.gs; b.do_step = b.step * a.dos; b.dn_step = b.step * a.dns;
  b.o_step = (int64_t)b.step * a.d;
  count_launch();
  return cuda_ok(launch_pdl(kernel, dim3((unsigned)s.blocks), dim3((unsigned)threads), smem, st, b));
}

template <typename TY, typename TR, bool GATE>
int launch_forward(const NormArgs &a, const NormShape &s, bool wide, cudaStream_t st) {
#define TMOE_RN(V, N) launch_walk<RowIn<TY, TR, V, N, GATE, false>>(residual_norm_kernel<TY, TR, V, N, GATE>, a, s, false, st)
  if (wide) return s.nv == 1 ? TMOE_RN(8, 1) : TMOE_RN(8, 2);
  return s.nv == 1 ? TMOE_RN(1, 8) : TMOE_RN(1, 16);
#undef TMOE_RN
}

template <typename TY, typename TR, bool GATE>
int launch_map(const NormArgs &a, int sms, cudaStream_t st) {
  const int per_row = a.d / 8;
  const int64_t want = (a.rows * per_row + kMapThreads - 1) / kMapThreads, cap = (int64_t)sms * 8;
  const int blocks = (int)(want < cap ? want : cap), step = blocks * kMapThreads;
  count_launch();
  return cuda_ok(launch_pdl(residual_map_kernel<TY, TR, GATE>, dim3((unsigned)blocks), dim3(kMapThreads), 0, st, a, per_row, step / per_row, step % per_row));
}

template <typename TY, typename TR, bool GATE>
int launch_backward(const NormArgs &a, const NormShape &s, bool wide, cudaStream_t st) {
#define TMOE_RNB(V, N) launch_walk<RowIn<TY, TR, V, N, GATE, true>>(residual_norm_backward_kernel<TY, TR, V, N, GATE>, a, s, true, st)
  if (wide) return s.nv == 1 ? TMOE_RNB(8, 1) : TMOE_RNB(8, 2);
  return s.nv == 1 ? TMOE_RNB(1, 8) : TMOE_RNB(1, 16);
#undef TMOE_RNB
}

// CALL<y type, residual type, gate>(...) for the call's types
#define TMOE_NORM_TYPES(CALL, p, ...)                                                                                              \
  ((p)->dtype == TMOE_F32 ? ((p)->gate ? CALL<float, float, true>(__VA_ARGS__) : CALL<float, float, false>(__VA_ARGS__))           \
   : (p)->residual_dtype == TMOE_F32 ? ((p)->gate ? CALL<bf16, float, true>(__VA_ARGS__) : CALL<bf16, float, false>(__VA_ARGS__))  \
                                     : ((p)->gate ? CALL<bf16, bf16, true>(__VA_ARGS__) : CALL<bf16, bf16, false>(__VA_ARGS__)))

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
  const int sms = current_device_sms();
  if (sms <= 0) return TMOE_ERR_CUDA;
  if (wide && !p->post_w && !p->next_w) return TMOE_NORM_TYPES(launch_map, p, a, sms, st);
  const NormShape s = norm_shape(*p, false, sms);
  a.tw = s.tw;
  return TMOE_NORM_TYPES(launch_forward, p, a, s, wide, st);
}

int64_t tmoe_residual_norm_workspace_bytes(const tmoe_residual_norm_t *p) {
  int rc = check_norm(p);
  if (rc) return rc;
  return p->rows == 0 ? 0 : max_partials(p->rows) * 2 * p->d * 4;
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
  if (d_layer_scale || d_post_w) a.sum_a = a.n_sums++;
  if (d_next_w) a.sum_x = a.n_sums++;
  const int sms = current_device_sms();
  if (sms <= 0) return TMOE_ERR_CUDA;
  const NormShape s = norm_shape(*p, true, sms < 160 ? sms : 160);
  if (params) {
    if (!workspace) return TMOE_ERR_NULL;
    if (workspace_bytes < max_partials(p->rows) * a.n_sums * p->d * 4) return TMOE_ERR_WORKSPACE;
    a.partial = reinterpret_cast<float *>(workspace);
  }
  const bool wide = norm_wide(*p) && wide_ok(d_out, d_out_stride, sr) && wide_ok(d_normed, d_normed_stride, sy) &&
                    wide_ok(d_y, p->d, sy) && wide_ok(d_residual, p->d, sr) && wide_ok(d_gate, p->d, sy);
  a.tw = s.tw;
  if ((rc = TMOE_NORM_TYPES(launch_backward, p, a, s, wide, st))) return rc;
  if (params) {
    const dim3 grid((unsigned)((a.n_sums * p->d + 31) / 32)), block(kColumnSumThreads);
    if (p->dtype == TMOE_F32)
      rc = cuda_ok(launch_pdl(norm_params_kernel<float>, grid, block, 0, st, a, s.blocks, (float *)d_layer_scale, (float *)d_post_w, (float *)d_next_w));
    else
      rc = cuda_ok(launch_pdl(norm_params_kernel<bf16>, grid, block, 0, st, a, s.blocks, (bf16 *)d_layer_scale, (bf16 *)d_post_w, (bf16 *)d_next_w));
    count_launch();
  }
  return rc;
}

}  // extern "C"
