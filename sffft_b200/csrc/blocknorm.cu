// The joint between two blocks of a network, on rows of C channels:
//
//   a = y * rstd_g(y) * post_weight      norm of the block's output, over each of `groups` equal runs of channels
//   h = x + scale * act(gate) * a        gate, residual scale and residual stream
//   n = h * rstd(h) * weight             norm before the next block
//
// with rstd(z) = (mean z^2 + eps)^-1/2; each norm, the gate and x may be absent.  One pass: x, y and gate are read
// once, h and n written once, a row's values stay in fp32 registers between the two norms.
//
// Backward, with u = y rstd_g(y), z = h rstd(h), f = act(gate) and the two norms' rstd kept from the forward pass:
//   t  = dn * weight          dx    = dh + rstd(h) (t - z mean(t z))                 dweight      = sum_rows dn z
//   da = scale f dx           dgate = scale dx a act'(gate)                          dpost_weight = sum_rows da u
//   s  = da * post_weight     dy    = rstd_g(y) (s - u mean_g(s u))
// h is computed again from x, y and gate, which are read anyway (it would cost as much to read, and in bf16 the kept h is
// rounded).  The sums over rows are taken in a fixed order: each block of a fixed grid adds its rows in registers (or,
// channels first, in shared memory), a second launch adds the blocks.
//
// Two layouts: rows of contiguous channels, and the convolution's [B][C][L], where a row is a column of stride L.
#include <cuda_bf16.h>
#include <stdint.h>

#include <climits>
#include <cmath>

#include "../../include/sffft.h"
#include "launch.h"

int sffft_note_cuda_error(cudaError_t e);

namespace sffft {
namespace {

constexpr int kMaxChannels = 8192;   // what a block's registers hold in the backward pass

enum { GATE_NONE = 0, GATE_FULL = 1, GATE_CHANNEL = 2 };

struct NormParams {
  const void *x, *y, *gate, *pw, *w;
  void *h, *n;
  float *r1, *r2;             // rstd of the groups of y [rows][groups] and of h [rows] (written forward, read backward)
  const void *dh, *dn;
  void *dx, *dy, *dgate;
  float* part;                // [blocks][3][C]: sums of dweight, dpost_weight, dgate of a channel gate
  long long rows, xs, ys, gs; // rows layout: row strides
  int C, groups, gc, inner;   // gc channels in a group; inner: L of [B][C][L]
  int gate_kind, act, w_bf16;
  unsigned gmul;              // 2^31 / gc, rounded up: group_of
  int blocks;                 // backward: blocks of the grid
  int sums_shared;            // channels first, backward: sums over rows in shared memory
  float scale, eps;
};

__device__ __forceinline__ float ldf(const float* p) { return *p; }
__device__ __forceinline__ float ldf(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// VEC consecutive values; VEC > 1 in 16-byte (fp32 x 4, bf16 x 8) or 8-byte (bf16 x 4) pieces.
template <int VEC>
__device__ __forceinline__ void ldv(const float* p, float (&v)[VEC]) {
  if constexpr (VEC == 1) v[0] = *p;
  else
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 a = *(const float4*)(p + i);
      v[i] = a.x, v[i + 1] = a.y, v[i + 2] = a.z, v[i + 3] = a.w;
    }
}
__device__ __forceinline__ void unpack(uint32_t u, float& a, float& b) {
  a = __uint_as_float(u << 16);
  b = __uint_as_float(u & 0xffff0000u);
}
__device__ __forceinline__ uint32_t pack(float a, float b) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
  return *(const uint32_t*)&t;
}
template <int VEC>
__device__ __forceinline__ void ldv(const __nv_bfloat16* p, float (&v)[VEC]) {
  if constexpr (VEC == 1) v[0] = __bfloat162float(*p);
  else if constexpr (VEC == 4) {
    const uint2 a = *(const uint2*)p;
    unpack(a.x, v[0], v[1]);
    unpack(a.y, v[2], v[3]);
  } else {
    const uint4 a = *(const uint4*)p;
    unpack(a.x, v[0], v[1]);
    unpack(a.y, v[2], v[3]);
    unpack(a.z, v[4], v[5]);
    unpack(a.w, v[6], v[7]);
  }
}
template <int VEC>
__device__ __forceinline__ void stv(float* p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) *p = v[0];
  else
#pragma unroll
    for (int i = 0; i < VEC; i += 4) *(float4*)(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}
template <int VEC>
__device__ __forceinline__ void stv(__nv_bfloat16* p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) *p = __float2bfloat16_rn(v[0]);
  else if constexpr (VEC == 4) *(uint2*)p = make_uint2(pack(v[0], v[1]), pack(v[2], v[3]));
  else *(uint4*)p = make_uint4(pack(v[0], v[1]), pack(v[2], v[3]), pack(v[4], v[5]), pack(v[6], v[7]));
}
template <int VEC>
__device__ __forceinline__ void ldw(const void* w, int bf16, int c, float (&v)[VEC]) {
  if (bf16) ldv<VEC>((const __nv_bfloat16*)w + c, v);
  else ldv<VEC>((const float*)w + c, v);
}

// The approximate division is off by at most 2 units in the last place; the exact one, with the exact exp, was a third of the
// instructions of a kernel that their issue held back, 65 -> 55 us for 32768 rows of 768.  A gate in fp32 has the
// exact exp (2 units).  A gate in bf16 has the approximate one, whose error grows with |x| to 32 units at 87, 2^-18: the
// gate, rounded to 2^-8 of itself, moves the result by |x| times that (61 us for the same rows; 65 with the exact one).
template <class T>
__device__ __forceinline__ float sigmoidf(float x) {
  if constexpr (sizeof(T) == 4) return __fdividef(1.f, 1.f + expf(-x));
  else return __fdividef(1.f, 1.f + __expf(-x));
}

// act(gate) of a thread's values, gate of type T, and its derivative (one branch for all of them)
template <class T, int VEC>
__device__ __forceinline__ void act_fwd(int act, const float (&g)[VEC], float (&f)[VEC]) {
  if (act == SFFFT_ACT_NONE) {
#pragma unroll
    for (int e = 0; e < VEC; e++) f[e] = g[e];
  } else if (act == SFFFT_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < VEC; e++) f[e] = g[e] * sigmoidf<T>(g[e]);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; e++) f[e] = sigmoidf<T>(g[e]);
  }
}
template <class T, int VEC>
__device__ __forceinline__ void act_both(int act, const float (&g)[VEC], float (&f)[VEC], float (&df)[VEC]) {
  if (act == SFFFT_ACT_NONE) {
#pragma unroll
    for (int e = 0; e < VEC; e++) f[e] = g[e], df[e] = 1.f;
  } else if (act == SFFFT_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < VEC; e++) {
      const float s = sigmoidf<T>(g[e]);
      f[e] = g[e] * s;
      df[e] = fmaf(f[e], 1.f - s, s);
    }
  } else {
#pragma unroll
    for (int e = 0; e < VEC; e++) {
      f[e] = sigmoidf<T>(g[e]);
      df[e] = fmaf(-f[e], f[e], f[e]);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Rows of contiguous channels.  A row's threads (a warp, or a block) hold VEC x NV channels each.  Bound by memory; what
// costs is latency: a row is a chain of loads, sums over its threads and stores.  So all of a row's loads are issued before
// the first use (they are kept as they come, RawV), backward also the next row's before this one's arithmetic, and the sums
// that backward needs are taken together: with s = scale f post_weight,
//   m = sum t z,  A_g = sum_g s u (dh + rstd t),  B_g = sum_g s u z   give   sum_g s u dx = A_g - rstd m / C * B_g.
// Measured: 32768 rows of 768 in bf16 with an fp32 residual stream, 12 groups: 56 us forward (6.3 TB/s); 14329 rows of 1024 in
// bf16: 25 us forward (4.7 TB/s), 66 backward (2.7 TB/s), which is bound by the issue of its instructions (61 % of the slots
// at the 512 threads an SM that 128 registers each allow).
// ---------------------------------------------------------------------------------------------------------------
template <class T, int VEC>
struct RawV {
  static constexpr int bytes = VEC * (int)sizeof(T);
  uint32_t w[(bytes + 3) / 4];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (bytes >= 16) {
#pragma unroll
      for (int i = 0; i < bytes / 16; i++) {
        const uint4 a = ((const uint4*)p)[i];
        w[4 * i] = a.x, w[4 * i + 1] = a.y, w[4 * i + 2] = a.z, w[4 * i + 3] = a.w;
      }
    } else if constexpr (bytes == 8) {
      const uint2 a = *(const uint2*)p;
      w[0] = a.x, w[1] = a.y;
    } else if constexpr (bytes == 4) {
      w[0] = *(const uint32_t*)p;
    } else {
      w[0] = (uint32_t) * (const uint16_t*)p << 16;
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (uint32_t& x : w) x = 0;
  }
  __device__ __forceinline__ void get(float (&v)[VEC]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < VEC; i++) v[i] = __uint_as_float(w[i]);
    } else if constexpr (VEC == 1) {
      v[0] = __uint_as_float(w[0]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; i += 2) unpack(w[i / 2], v[i], v[i + 1]);
    }
  }
};

// N sums over the threads of a row: a warp, or (BLOCK) the nw warps of the block, through red[2][N][32], whose halves take
// turns (`turn`), so that one barrier does.
template <bool BLOCK, int N>
__device__ __forceinline__ void row_sums(float (&s)[N], float* red, int nw, int& turn) {
#pragma unroll
  for (int k = 0; k < N; k++)
#pragma unroll
    for (int o = 16; o; o >>= 1) s[k] += __shfl_xor_sync(~0u, s[k], o);
  if constexpr (BLOCK) {
    float* r = red + turn * N * 32;
    turn ^= 1;
    const int lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
      for (int k = 0; k < N; k++) r[k * 32 + (threadIdx.x >> 5)] = s[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; k++) {
      s[k] = lane < nw ? r[k * 32 + lane] : 0.f;
#pragma unroll
      for (int o = 16; o; o >>= 1) s[k] += __shfl_xor_sync(~0u, s[k], o);
    }
  }
}

template <bool BLOCK>
__device__ __forceinline__ void row_sync() {
  if constexpr (BLOCK) __syncthreads();
  else __syncwarp();
}

// Sums over several groups of channels: v[j] is the sum over the thread's j-th vector, replaced by its group's sum.  Where
// a group is a power of two of at most 32 vectors its vectors lie in neighbouring lanes (a row's threads start at a
// multiple of 32); otherwise the vectors' sums go through shared memory, one warp adding up a group.
template <bool BLOCK, int NV>
__device__ __forceinline__ void group_sums(float (&v)[NV], int nvec, int per, int groups, float* vec, int t, int tpr) {
  if (per <= 32 && (per & (per - 1)) == 0) {
#pragma unroll
    for (int j = 0; j < NV; j++)
      for (int o = per >> 1; o; o >>= 1) v[j] += __shfl_xor_sync(~0u, v[j], o);
    return;
  }
  float* grp = vec + nvec;
  row_sync<BLOCK>();
#pragma unroll
  for (int j = 0; j < NV; j++)
    if (j * tpr + t < nvec) vec[j * tpr + t] = v[j];
  row_sync<BLOCK>();
  for (int g = t >> 5; g < groups; g += tpr >> 5) {
    float s = 0.f;
    for (int e = t & 31; e < per; e += 32) s += vec[g * per + e];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if ((t & 31) == 0) grp[g] = s;
  }
  row_sync<BLOCK>();
#pragma unroll
  for (int j = 0; j < NV; j++) v[j] = j * tpr + t < nvec ? grp[(j * tpr + t) / per] : 0.f;
}

// Shared memory of a row: vector sums and group sums (only where group_sums needs them).  All of it is dynamic, row_sums' too:
// a launch's limit counts both kinds.
__host__ __device__ inline int rows_smem_floats(int nvec, int groups) { return groups > 1 ? nvec + groups : 0; }
constexpr int kRedForward = 2 * 32, kRedBackward = 2 * 3 * 32;   // floats of row_sums, where a row is a block's

constexpr int kRowsPerBlock = 4;   // where a row is a warp's

template <class TX, class TY, int VEC, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 1024 : 32 * kRowsPerBlock) norm_rows_kernel(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(16) float red[];
  const int tpr = BLOCK ? blockDim.x : 32, t = BLOCK ? threadIdx.x : threadIdx.x & 31, nvec = p.C / VEC;
  const int sub = BLOCK ? 0 : threadIdx.x >> 5, nw = tpr >> 5, per = p.gc / VEC;
  float* vec = red + (BLOCK ? kRedForward : 0) + sub * rows_smem_floats(nvec, p.groups);
  const long long r = BLOCK ? (long long)blockIdx.x : blockIdx.x * (long long)kRowsPerBlock + sub;
  if (r >= p.rows) return;   // whole warps
  int turn = 0;
  RawV<TY, VEC> ry[NV], rg[NV];
  RawV<TX, VEC> rx[NV];
#pragma unroll
  for (int j = 0; j < NV; j++) {
    const int i = j * tpr + t;
    ry[j].zero(), rg[j].zero(), rx[j].zero();
    if (i < nvec) {
      if (p.y) ry[j].load((const TY*)p.y + r * p.ys + i * VEC);
      if (p.x) rx[j].load((const TX*)p.x + r * p.xs + i * VEC);
      if (p.gate_kind) rg[j].load((const TY*)p.gate + r * p.gs + i * VEC);
    }
  }
  float v[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; j++) ry[j].get(v[j]);
  if (p.pw) {
    float s[NV], all[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NV; j++) {
      s[j] = 0.f;
#pragma unroll
      for (int e = 0; e < VEC; e++) s[j] = fmaf(v[j][e], v[j][e], s[j]);
      all[0] += s[j];
    }
    if (p.groups == 1) {
      row_sums<BLOCK, 1>(all, red, nw, turn);
#pragma unroll
      for (int j = 0; j < NV; j++) s[j] = all[0];
    } else {
      group_sums<BLOCK, NV>(s, nvec, per, p.groups, vec, t, tpr);
    }
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const int i = j * tpr + t;
      if (i >= nvec) continue;
      const float rs = rsqrtf(s[j] / (float)p.gc + p.eps);
      if (p.r1) {
        if (p.groups == 1) {
          if (i == 0) p.r1[r] = rs;
        } else if (i % per == 0) {
          p.r1[r * p.groups + i / per] = rs;
        }
      }
      float w[VEC];
      ldw<VEC>(p.pw, p.w_bf16, i * VEC, w);
#pragma unroll
      for (int e = 0; e < VEC; e++) v[j][e] *= rs * w[e];
    }
  }
  float ss[1] = {0.f};
#pragma unroll
  for (int j = 0; j < NV; j++) {
    const int i = j * tpr + t;
    if (i >= nvec) continue;
    float a[VEC];
    rx[j].get(a);
    if (p.y) {
      if (p.gate_kind) {
        float g[VEC], f[VEC];
        rg[j].get(g);
        act_fwd<TY, VEC>(p.act, g, f);
#pragma unroll
        for (int e = 0; e < VEC; e++) v[j][e] *= f[e];
      }
#pragma unroll
      for (int e = 0; e < VEC; e++) v[j][e] = fmaf(p.scale, v[j][e], a[e]);
      stv<VEC>((TX*)p.h + r * p.C + i * VEC, v[j]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; e++) v[j][e] = a[e];
    }
#pragma unroll
    for (int e = 0; e < VEC; e++) ss[0] = fmaf(v[j][e], v[j][e], ss[0]);
  }
  if (!p.w) return;
  row_sums<BLOCK, 1>(ss, red, nw, turn);
  const float rs = rsqrtf(ss[0] / (float)p.C + p.eps);
  if (p.r2 && t == 0) p.r2[r] = rs;
#pragma unroll
  for (int j = 0; j < NV; j++) {
    const int i = j * tpr + t;
    if (i >= nvec) continue;
    float w[VEC];
    ldw<VEC>(p.w, p.w_bf16, i * VEC, w);
#pragma unroll
    for (int e = 0; e < VEC; e++) v[j][e] *= rs * w[e];
    stv<VEC>((TY*)p.n + r * p.C + i * VEC, v[j]);
  }
}

template <class TX, class TY, int VEC, int NV>
struct RawRow {
  RawV<TY, VEC> y[NV], g[NV], dn[NV];
  RawV<TX, VEC> x[NV], dh[NV];
  float r1[NV], r2;
  __device__ __forceinline__ void load(const NormParams& p, long long r, int t, int tpr, int nvec, const int (&grp)[NV]) {
    r2 = p.w ? p.r2[r] : 0.f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const int i = j * tpr + t;
      y[j].zero(), g[j].zero(), dn[j].zero(), x[j].zero(), dh[j].zero();
      r1[j] = 1.f;
      if (i >= nvec) continue;
      if (p.y) y[j].load((const TY*)p.y + r * p.ys + i * VEC);
      if (p.gate_kind == GATE_FULL) g[j].load((const TY*)p.gate + r * p.gs + i * VEC);
      if (p.dh) dh[j].load((const TX*)p.dh + r * p.C + i * VEC);
      if (p.w) {
        if (p.x) x[j].load((const TX*)p.x + r * p.xs + i * VEC);
        dn[j].load((const TY*)p.dn + r * p.C + i * VEC);
      }
      if (p.pw) r1[j] = p.r1[r * p.groups + grp[j]];
    }
  }
};

// Threads of a row in the backward pass: 512 at most, which leaves each 128 registers.
template <class TX, class TY, int VEC, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 512 : 32 * kRowsPerBlock) norm_rows_bwd_kernel(const __grid_constant__ NormParams p) {
  constexpr bool AHEAD = NV == 1;   // registers for the next row
  extern __shared__ __align__(16) float red[];
  const int tpr = BLOCK ? blockDim.x : 32, t = BLOCK ? threadIdx.x : threadIdx.x & 31, nvec = p.C / VEC;
  const int sub = BLOCK ? 0 : threadIdx.x >> 5, nw = tpr >> 5, per = p.gc / VEC;
  float* vec = red + (BLOCK ? kRedBackward : 0) + sub * rows_smem_floats(nvec, p.groups);
  int turn = 0, grp[NV];
  float sw[NV][VEC], sp[NV][VEC], sg[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; j++) {
    grp[j] = p.groups > 1 ? min((j * tpr + t) / per, p.groups - 1) : 0;
#pragma unroll
    for (int e = 0; e < VEC; e++) sw[j][e] = sp[j][e] = sg[j][e] = 0.f;
  }
  const long long step = BLOCK ? (long long)p.blocks : (long long)p.blocks * kRowsPerBlock;
  long long r = BLOCK ? (long long)blockIdx.x : blockIdx.x * (long long)kRowsPerBlock + sub;
  RawRow<TX, TY, VEC, NV> now, next;
  if (r < p.rows) now.load(p, r, t, tpr, nvec, grp);
  const float inv_c = 1.f / (float)p.C, inv_g = 1.f / (float)p.gc;

  for (; r < p.rows; r += step) {
    if (AHEAD && r + step < p.rows) next.load(p, r + step, t, tpr, nvec, grp);
    float u[NV][VEC], z[NV][VEC], d[NV][VEC], s[NV][VEC];   // d: dh + rstd t, then dx;  s: scale f post_weight
    float A[NV], B[NV], sum[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const int i = j * tpr + t;
      float x[VEC], tn[VEC], w[VEC], pw[VEC], g[VEC];
      now.y[j].get(u[j]);
      now.x[j].get(x);
      now.dn[j].get(tn);
      now.dh[j].get(d[j]);
      now.g[j].get(g);
#pragma unroll
      for (int e = 0; e < VEC; e++) w[e] = 0.f, pw[e] = 1.f;
      if (i < nvec) {
        if (p.w) ldw<VEC>(p.w, p.w_bf16, i * VEC, w);
        if (p.pw) ldw<VEC>(p.pw, p.w_bf16, i * VEC, pw);
        if (p.gate_kind == GATE_CHANNEL) ldv<VEC>((const TY*)p.gate + i * VEC, g);
      }
      A[j] = B[j] = 0.f;
      float f[VEC];
#pragma unroll
      for (int e = 0; e < VEC; e++) f[e] = 1.f;
      if (p.gate_kind) act_fwd<TY, VEC>(p.act, g, f);
      if (!p.pw) {   // without y u is zero
#pragma unroll
        for (int e = 0; e < VEC; e++) s[j][e] = p.scale * f[e];
      } else {
#pragma unroll
        for (int e = 0; e < VEC; e++) s[j][e] = p.scale * f[e] * pw[e];
      }
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        u[j][e] *= now.r1[j];
        z[j][e] = fmaf(s[j][e], u[j][e], x[e]) * now.r2;
        sw[j][e] = fmaf(tn[e], z[j][e], sw[j][e]);
        const float tt = tn[e] * w[e], su = s[j][e] * u[j][e];
        d[j][e] = fmaf(now.r2, tt, d[j][e]);
        sum[0] = fmaf(tt, z[j][e], sum[0]);
        A[j] = fmaf(su, d[j][e], A[j]);
        B[j] = fmaf(su, z[j][e], B[j]);
      }
    }
    if (p.pw && p.groups == 1) {
#pragma unroll
      for (int j = 0; j < NV; j++) sum[1] += A[j], sum[2] += B[j];
      row_sums<BLOCK, 3>(sum, red, nw, turn);
#pragma unroll
      for (int j = 0; j < NV; j++) A[j] = sum[1], B[j] = sum[2];
    } else {
      if (p.w) {
        float one[1] = {sum[0]};
        row_sums<BLOCK, 1>(one, red, nw, turn);
        sum[0] = one[0];
      }
      if (p.pw) {
        group_sums<BLOCK, NV>(A, nvec, per, p.groups, vec, t, tpr);
        group_sums<BLOCK, NV>(B, nvec, per, p.groups, vec, t, tpr);
      }
    }
    const float m = sum[0] * now.r2 * inv_c;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const int i = j * tpr + t;
      if (i >= nvec) continue;
#pragma unroll
      for (int e = 0; e < VEC; e++) d[j][e] = fmaf(-m, z[j][e], d[j][e]);
      if (p.dx) stv<VEC>((TX*)p.dx + r * p.C + i * VEC, d[j]);
      if (!p.y) continue;
      float pw[VEC];
#pragma unroll
      for (int e = 0; e < VEC; e++) pw[e] = 1.f;
      if (p.pw) ldw<VEC>(p.pw, p.w_bf16, i * VEC, pw);
      if (p.gate_kind) {
        float g[VEC], f[VEC], df[VEC];
        if (p.gate_kind == GATE_FULL) now.g[j].get(g);
        else ldv<VEC>((const TY*)p.gate + i * VEC, g);
        act_both<TY, VEC>(p.act, g, f, df);
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          const float du = p.scale * d[j][e] * u[j][e];
          sp[j][e] = fmaf(f[e], du, sp[j][e]);
          g[e] = du * pw[e] * df[e];
        }
        if (p.gate_kind == GATE_FULL) {
          stv<VEC>((TY*)p.dgate + r * p.C + i * VEC, g);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; e++) sg[j][e] += g[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < VEC; e++) sp[j][e] = fmaf(p.scale * d[j][e], u[j][e], sp[j][e]);
      }
      const float mu = p.pw ? fmaf(-m, B[j], A[j]) * inv_g : 0.f;
#pragma unroll
      for (int e = 0; e < VEC; e++) d[j][e] = now.r1[j] * fmaf(-mu, u[j][e], s[j][e] * d[j][e]);
      stv<VEC>((TY*)p.dy + r * p.C + i * VEC, d[j]);
    }
    if (AHEAD) now = next;
    else if (r + step < p.rows) now.load(p, r + step, t, tpr, nvec, grp);
  }
  // this block's sums over its rows, its warps' one after the other
  float* out = p.part + (long long)blockIdx.x * 3 * p.C;
  for (int q = 0; q < (BLOCK ? 1 : kRowsPerBlock); q++) {
    if (q == sub) {
#pragma unroll
      for (int j = 0; j < NV; j++) {
        const int i = j * tpr + t;
        if (i >= nvec) continue;
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          const int c = i * VEC + e;
          if (p.w) out[c] = (q ? out[c] : 0.f) + sw[j][e];
          if (p.pw) out[p.C + c] = (q ? out[p.C + c] : 0.f) + sp[j][e];
          if (p.gate_kind == GATE_CHANNEL) out[2 * p.C + c] = (q ? out[2 * p.C + c] : 0.f) + sg[j][e];
        }
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Channels first: [B][C][L].  A block takes kPos positions of one row of the batch, all channels: a warp's lanes lie
// across the positions, VEC each, and down 32 VEC / kPos channels, so that it reads whole 128-byte (bf16: 64-byte) pieces.
//
// Sums over a group's channels: each thread adds its own channels, lanes of a position are added by shuffles, warps
// through shared memory.  With many groups (kManyGroups) each is left to one warp instead.
//
// Forward, y's tile is kept in shared memory in fp32 (then h's in its place) as long as it fits, so that y, x and gate are
// read once.  Backward would have to keep five tiles; instead all three sums that a position needs are taken in one
// reading,
//   m = mean(t z),  A_g = sum_g s u (dh + rstd t),  B_g = sum_g s u z   (s = scale f post_weight):  sum_g s u dx = A - m B
// and the second reading, which writes the results, finds the tile in L2: two blocks on each SM keep 296 tiles at work,
// 145 MB for 768 channels in fp32 and 73 in bf16, of 126 (two blocks: 76 us for [8][768][1024] in fp32; one: 85).
//
// What bounds both is the latency of a thread's loads: 1024 threads on an SM with 64 registers (forward: 40 to 64, and 98 KB
// of tile for 768 channels) hold no more of them in flight.  Measured, of the bytes that must move: [8][768][1024] fp32, one
// group: 33 us forward (3.8 TB/s), 76 backward (2.6); [8][768][4096] bf16, 12 groups: 87 and 211 us (2.9, 1.9 TB/s).
// Forward's loads are taken two (fp32) or four channels at a time, which was 125 -> 87 us of the latter; backward has no
// registers for a second channel (212 -> 259 us where it was made to) but where threads hold single values.  They do where L
// is no multiple of 4, and their instructions then bound both: [3][768][2187] fp32: 32 and 101 us (3.1, 1.6 TB/s);
// [8][768][4095] bf16, 12 groups: 151 and 536 (1.7, 0.75 TB/s; 691 one channel at a time).
// ---------------------------------------------------------------------------------------------------------------
constexpr int kPos = 32, kFirstThreads = 512, kFirstWarps = kFirstThreads / 32, kManyGroups = 8;

template <int VEC>
struct FirstShape {
  static constexpr int TX = kPos / VEC, TR = 32 / TX, TY = kFirstWarps * TR;   // lanes across, channels in a warp, in the block
};

// c / gc: c gmul / 2^31 is above it by less than c / 2^31, which is less than 1 / gc (both are at most kMaxChannels).
__device__ __forceinline__ int group_of(const NormParams& p, int c) { return (int)__umulhi(2u * (unsigned)c, p.gmul); }

// Channels c, c + step, .. below `end`, the loads of U of them before the first one's use: results that are stored in between
// may be anyone's memory to the compiler, which therefore does not move a load ahead of them itself.
template <int U, class R, class L, class F>
__device__ __forceinline__ void channels(int c, int end, int step, L load, F use) {
  for (; c + (U - 1) * step < end; c += U * step) {
    R r[U];
#pragma unroll
    for (int i = 0; i < U; i++) load(c + i * step, r[i]);
#pragma unroll
    for (int i = 0; i < U; i++) use(c + i * step, r[i]);
  }
  if constexpr (U > 1)
    for (; c < end; c += step) {
      R r;
      load(c, r);
      use(c, r);
    }
}

// Sums of N quantities over each group: `add(c, r, s)` adds channel c's, loaded by load(c, r), to the thread's s[N][VEC].
// out[k]: [groups][kPos].  part: [min(groups, kManyGroups - 1)][kFirstWarps][kPos] floats for each quantity.  Ends with the
// block in step.
template <int VEC, int N, int U, class R, class L, class F>
__device__ __forceinline__ void first_sums(int groups, int gc, float* part, float* const (&out)[N], bool in, L load, F add) {
  using SH = FirstShape<VEC>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tx = lane % SH::TX, tr = lane / SH::TX;
  const bool many = groups >= kManyGroups;
  const int first = many ? tr : warp * SH::TR + tr, step = many ? SH::TR : SH::TY;
  for (int g = many ? warp : 0; g < groups; g += many ? kFirstWarps : 1) {
    float s[N][VEC] = {};
    if (in) channels<U, R>(g * gc + first, (g + 1) * gc, step, load, [&](int c, const R& r) { add(c, r, s); });
#pragma unroll
    for (int k = 0; k < N; k++) {
#pragma unroll
      for (int e = 0; e < VEC; e++)
#pragma unroll
        for (int o = SH::TX; o < 32; o <<= 1) s[k][e] += __shfl_xor_sync(~0u, s[k][e], o);
      if (tr == 0) {
        float* to = many ? out[k] + g * kPos : part + ((k * groups + g) * kFirstWarps + warp) * kPos;
#pragma unroll
        for (int e = 0; e < VEC; e++) to[tx * VEC + e] = s[k][e];
      }
    }
  }
  __syncthreads();
  if (many) return;
  for (int i = threadIdx.x; i < N * groups * kPos; i += kFirstThreads) {
    const int k = i / (groups * kPos), gp = i % (groups * kPos);
    const float* from = part + ((k * groups + gp / kPos) * kFirstWarps) * kPos + gp % kPos;
    float z = 0.f;
#pragma unroll
    for (int w = 0; w < kFirstWarps; w++) z += from[w * kPos];
    out[k][gp] = z;
  }
  __syncthreads();
}

__host__ __device__ inline int first_part_floats(int groups, int n) {
  return groups >= kManyGroups ? kFirstWarps * kPos : n * groups * kFirstWarps * kPos;
}

// Tiles of a row of the batch (inner + kPos - 1 may pass 31 bits).
__host__ __device__ inline int first_tiles(int inner) { return inner / kPos + (inner % kPos != 0); }

struct FirstTile {
  long long base;   // element (channel 0, first position of the thread)
  long long row;    // row index of that position
  bool in;          // inside L (VEC 4: L is a multiple of 4)
};

template <int VEC>
__device__ __forceinline__ FirstTile first_tile(const NormParams& p, long long tile) {
  const int per = first_tiles(p.inner);
  const long long b = tile / per, l = tile % per * kPos + (threadIdx.x % FirstShape<VEC>::TX) * VEC;
  return {b * p.C * p.inner + l, b * p.inner + l, l < p.inner};
}

template <class TX, class TY, int VEC, bool KEEP>
__global__ void __launch_bounds__(kFirstThreads) norm_first_kernel(const __grid_constant__ NormParams p) {
  using SH = FirstShape<VEC>;
  extern __shared__ __align__(16) float dyn[];
  float* r1 = dyn;                                     // [groups][kPos]
  float* r2 = r1 + p.groups * kPos;                    // [kPos]
  float* part = r2 + kPos;
  float* tile = part + first_part_floats(p.groups, 1); // KEEP: [C][kPos]
  const int tx = threadIdx.x % SH::TX, ty = threadIdx.x / SH::TX;
  const FirstTile ft = first_tile<VEC>(p, blockIdx.x);
  const TY *y = (const TY*)p.y + ft.base, *gate = (const TY*)p.gate;
  const TX* x = (const TX*)p.x + ft.base;
  const long long L = p.inner;
  // Channels ahead, two against four (us): with fp32 alone [8][768][1024] 41, 45, [8][768][4096] 121, 135, [8][256][8192] 88,
  // 141, but [4][1024][2048] 53, 49 and [2][2048][2048] 72, 66; in bf16 [8][768][4096] 108, 105, [8][256][8192] 76, 74,
  // [2][2048][4096] 82, 74.
  constexpr int kAhead = VEC == 1 || sizeof(TX) + sizeof(TY) <= 6 ? 4 : 2;
  if (p.pw) {
    float* const out[1] = {r1};
    if constexpr (KEEP) {   // y's tile first, many loads at a time: the sums over groups would wait for each
      if (ft.in)
#pragma unroll 8
        for (int c = ty; c < p.C; c += SH::TY) {
          float v[VEC];
          ldv<VEC>(y + c * L, v);
          stv<VEC>(tile + c * kPos + tx * VEC, v);
        }
      __syncthreads();
    }
    first_sums<VEC, 1, 4, RawV<TY, VEC>>(
        p.groups, p.gc, part, out, ft.in,
        [&](int c, RawV<TY, VEC>& r) {
          if constexpr (!KEEP) r.load(y + c * L);
        },
        [&](int c, const RawV<TY, VEC>& r, float (&s)[1][VEC]) {
          float v[VEC];
          if constexpr (KEEP) ldv<VEC>(tile + c * kPos + tx * VEC, v);
          else r.get(v);
#pragma unroll
          for (int e = 0; e < VEC; e++) s[0][e] = fmaf(v[e], v[e], s[0][e]);
        });
    for (int i = threadIdx.x; i < p.groups * kPos; i += kFirstThreads) r1[i] = rsqrtf(r1[i] / (float)p.gc + p.eps);
    __syncthreads();
    if (p.r1 && ft.in)
      for (int g = ty; g < p.groups; g += SH::TY)
#pragma unroll
        for (int e = 0; e < VEC; e++) p.r1[(ft.row + e) * p.groups + g] = r1[g * kPos + tx * VEC + e];
  }
  struct Raw {
    RawV<TY, VEC> y, g;
    RawV<TX, VEC> x;
    float pw, gc;
  };
  auto load = [&](int c, Raw& r) {
    r.y.zero(), r.g.zero(), r.x.zero();
    float t[1] = {1.f};
    if (p.y && !(KEEP && p.pw)) r.y.load(y + c * L);
    if (p.gate_kind == GATE_FULL) r.g.load(gate + ft.base + c * L);
    if (p.x) r.x.load(x + c * L);
    if (p.pw) ldw<1>(p.pw, p.w_bf16, c, t);
    r.pw = t[0];
    r.gc = p.gate_kind == GATE_CHANNEL ? ldf(gate + c) : 0.f;
  };
  auto value = [&](int c, const Raw& r, float (&h)[VEC]) {
    float xv[VEC];
    r.x.get(xv);
    r.y.get(h);
    if (p.y) {
      if (KEEP && p.pw) ldv<VEC>(tile + c * kPos + tx * VEC, h);
      if (p.pw) {
        const float* rs = r1 + group_of(p, c) * kPos + tx * VEC;
#pragma unroll
        for (int e = 0; e < VEC; e++) h[e] *= rs[e] * r.pw;
      }
      if (p.gate_kind) {
        float gv[VEC], f[VEC];
        if (p.gate_kind == GATE_FULL) r.g.get(gv);
        else
#pragma unroll
          for (int e = 0; e < VEC; e++) gv[e] = r.gc;
        act_fwd<TY, VEC>(p.act, gv, f);
#pragma unroll
        for (int e = 0; e < VEC; e++) h[e] *= f[e];
      }
    }
#pragma unroll
    for (int e = 0; e < VEC; e++) h[e] = p.x ? fmaf(p.scale, h[e], xv[e]) : p.scale * h[e];
  };
  if (!p.w) {
    if (ft.in)
      channels<kAhead, Raw>(ty, p.C, SH::TY, load, [&](int c, const Raw& r) {
        float h[VEC];
        value(c, r, h);
        stv<VEC>((TX*)p.h + ft.base + c * L, h);
      });
    return;
  }
  float* const out[1] = {r2};
  first_sums<VEC, 1, kAhead, Raw>(1, p.C, part, out, ft.in, load, [&](int c, const Raw& r, float (&s)[1][VEC]) {
    float h[VEC];
    value(c, r, h);
    if (p.h) stv<VEC>((TX*)p.h + ft.base + c * L, h);
    if (KEEP) stv<VEC>(tile + c * kPos + tx * VEC, h);
#pragma unroll
    for (int e = 0; e < VEC; e++) s[0][e] = fmaf(h[e], h[e], s[0][e]);
  });
  if (!ft.in) return;
  float rs[VEC];
#pragma unroll
  for (int e = 0; e < VEC; e++) {
    rs[e] = rsqrtf(r2[tx * VEC + e] / (float)p.C + p.eps);
    if (p.r2 && ty == 0) p.r2[ft.row + e] = rs[e];
  }
  struct Last {
    Raw r;
    float w;
  };
  channels<kAhead, Last>(
      ty, p.C, SH::TY,
      [&](int c, Last& l) {
        if constexpr (!KEEP) load(c, l.r);
        float w[1];
        ldw<1>(p.w, p.w_bf16, c, w);
        l.w = w[0];
      },
      [&](int c, const Last& l) {
        float h[VEC];
        if constexpr (KEEP) ldv<VEC>(tile + c * kPos + tx * VEC, h);
        else value(c, l.r, h);
#pragma unroll
        for (int e = 0; e < VEC; e++) h[e] *= rs[e] * l.w;
        stv<VEC>((TY*)p.n + ft.base + c * L, h);
      });
}

template <class TX, class TY, int VEC>
__global__ void __launch_bounds__(kFirstThreads, 2) norm_first_bwd_kernel(const __grid_constant__ NormParams p) {
  using SH = FirstShape<VEC>;
  extern __shared__ __align__(16) float dyn[];
  constexpr int kAhead = VEC == 1 ? 2 : 1;   // what 64 registers hold
  float* sA = dyn;                           // [groups][kPos]
  float* sB = sA + p.groups * kPos;
  float* sM = sB + p.groups * kPos;          // [groups][kPos], then [kPos]
  float* sQ = sM + p.groups * kPos;          // [groups][kPos]: rstd of y's groups
  float* part = sQ + p.groups * kPos;
  const int tx = threadIdx.x % SH::TX, ty = threadIdx.x / SH::TX;
  // this block's sums; a channel always belongs to one ty
  float* out = p.part + (long long)blockIdx.x * 3 * p.C;
  float* acc = p.sums_shared ? part + first_part_floats(p.groups, 3) : out;
  const long long L = p.inner;
  const int per = first_tiles(p.inner);
  const long long tiles = (p.rows / p.inner) * per;
  const TY* gate = (const TY*)p.gate;
  bool first = true;
  for (long long tile = blockIdx.x; tile < tiles; tile += p.blocks, first = false) {
    const FirstTile ft = first_tile<VEC>(p, tile);
    if (p.pw) {
      const long long row0 = tile / per * p.inner + tile % per * kPos;
      const int there = min(kPos, p.inner - (int)(tile % per) * kPos) * p.groups;
      for (int i = threadIdx.x; i < kPos * p.groups; i += kFirstThreads)
        sQ[i % p.groups * kPos + i / p.groups] = i < there ? p.r1[row0 * p.groups + i] : 0.f;
      __syncthreads();
    }
    float r2[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) r2[e] = p.w && ft.in ? p.r2[ft.row + e] : 0.f;
    struct Raw {
      RawV<TY, VEC> y, g, dn;
      RawV<TX, VEC> x, dh;
      float pw, w, gc;
    };
    auto load = [&](int c, Raw& r) {
      const long long at = ft.base + c * L;
      r.y.zero(), r.g.zero(), r.dn.zero(), r.x.zero(), r.dh.zero();
      float t[1] = {1.f}, w[1] = {0.f};
      if (p.y) r.y.load((const TY*)p.y + at);
      if (p.gate_kind == GATE_FULL) r.g.load(gate + at);
      if (p.dh) r.dh.load((const TX*)p.dh + at);
      if (p.w) {
        if (p.x) r.x.load((const TX*)p.x + at);
        r.dn.load((const TY*)p.dn + at);
        ldw<1>(p.w, p.w_bf16, c, w);
      }
      if (p.pw) ldw<1>(p.pw, p.w_bf16, c, t);
      r.pw = t[0];
      r.w = w[0];
      r.gc = p.gate_kind == GATE_CHANNEL ? ldf(gate + c) : 0.f;
    };
    struct Values {
      float u[VEC], f[VEC], df[VEC], z[VEC], d[VEC], tn[VEC];   // d: dh + rstd t
    };
    auto values = [&](const float* q, const Raw& r, Values& v, bool with_df) {   // q: rstd of y's group
      float xv[VEC];
      r.y.get(v.u);
      r.dh.get(v.d);
      r.dn.get(v.tn);
      r.x.get(xv);
#pragma unroll
      for (int e = 0; e < VEC; e++) v.f[e] = 1.f, v.df[e] = 0.f;
      if (p.pw)
#pragma unroll
        for (int e = 0; e < VEC; e++) v.u[e] *= q[e];
      if (p.gate_kind) {
        float gv[VEC];
        if (p.gate_kind == GATE_FULL) r.g.get(gv);
        else
#pragma unroll
          for (int e = 0; e < VEC; e++) gv[e] = r.gc;
        if (with_df) act_both<TY, VEC>(p.act, gv, v.f, v.df);
        else act_fwd<TY, VEC>(p.act, gv, v.f);
      }
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        v.z[e] = (p.y ? fmaf(p.scale * v.f[e], v.u[e] * r.pw, xv[e]) : xv[e]) * r2[e];
        v.d[e] = fmaf(r2[e], v.tn[e] * r.w, v.d[e]);
      }
    };
    if (p.w || p.pw) {
      float* const sums[3] = {sA, sB, sM};
      first_sums<VEC, 3, kAhead, Raw>(p.groups, p.gc, part, sums, ft.in, load, [&](int c, const Raw& r, float (&s)[3][VEC]) {
        Values v;
        values(sQ + group_of(p, c) * kPos + tx * VEC, r, v, false);
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          const float su = p.scale * v.f[e] * r.pw * v.u[e];
          s[0][e] = fmaf(su, v.d[e], s[0][e]);
          s[1][e] = fmaf(su, v.z[e], s[1][e]);
          s[2][e] = fmaf(v.tn[e] * r.w, v.z[e], s[2][e]);
        }
      });
      if (p.groups > 1) {
        float m = 0.f;
        if (threadIdx.x < kPos)
          for (int g = 0; g < p.groups; g++) m += sM[g * kPos + threadIdx.x];
        __syncthreads();
        if (threadIdx.x < kPos) sM[threadIdx.x] = m;
        __syncthreads();
      }
    }
    float m2[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) m2[e] = p.w ? sM[tx * VEC + e] * r2[e] / (float)p.C : 0.f;
    const float inv_g = 1.f / (float)p.gc;
    // Positions beyond L take part with zeros: the TX lanes of a channel are neighbours and add up.
    channels<kAhead, Raw>(
        ty, p.C, SH::TY,
        [&](int c, Raw& r) {
          if (ft.in) load(c, r);
        },
        [&](int c, const Raw& r) {
          float sw = 0.f, sp = 0.f, sg = 0.f;
          if (ft.in) {
            const int g = group_of(p, c) * kPos + tx * VEC;
            Values v;
            values(sQ + g, r, v, true);
            float dg[VEC];
#pragma unroll
            for (int e = 0; e < VEC; e++) {
              sw = fmaf(v.tn[e], v.z[e], sw);
              v.d[e] = fmaf(-m2[e], v.z[e], v.d[e]);
            }
            if (p.dx) stv<VEC>((TX*)p.dx + ft.base + c * L, v.d);
            if (p.y) {
#pragma unroll
              for (int e = 0; e < VEC; e++) {
                dg[e] = p.scale * v.d[e] * v.u[e] * r.pw * v.df[e];
                sg += dg[e];
                const float da = p.scale * v.f[e] * v.d[e];
                sp = fmaf(da, v.u[e], sp);
                v.d[e] = p.pw ? sQ[g + e] * fmaf(-fmaf(-m2[e], sB[g + e], sA[g + e]) * inv_g, v.u[e], da * r.pw) : da;
              }
              if (p.gate_kind == GATE_FULL) stv<VEC>((TY*)p.dgate + ft.base + c * L, dg);
              stv<VEC>((TY*)p.dy + ft.base + c * L, v.d);
            }
          }
          // lanes of a warp whose channel is beyond C have left together
          const unsigned mask = SH::TX == 32 ? ~0u : ((1u << SH::TX) - 1) << ((threadIdx.x & 31) / SH::TX * SH::TX);
#pragma unroll
          for (int o = SH::TX / 2; o; o >>= 1) {
            sw += __shfl_xor_sync(mask, sw, o);
            sp += __shfl_xor_sync(mask, sp, o);
            sg += __shfl_xor_sync(mask, sg, o);
          }
          if (tx == 0) {
            if (p.w) acc[c] = (first ? 0.f : acc[c]) + sw;
            if (p.pw) acc[p.C + c] = (first ? 0.f : acc[p.C + c]) + sp;
            if (p.gate_kind == GATE_CHANNEL) acc[2 * p.C + c] = (first ? 0.f : acc[2 * p.C + c]) + sg;
          }
        });
    __syncthreads();
  }
  if (p.sums_shared)
    for (int i = threadIdx.x; i < 3 * p.C; i += kFirstThreads) {
      const int k = i / p.C;
      if (k == 0 ? p.w != nullptr : k == 1 ? p.pw != nullptr : p.gate_kind == GATE_CHANNEL) out[i] = acc[i];
    }
}

// Sums the blocks' parts: a block takes 32 channels, 32 threads down the parts, added in a fixed order.
struct PartParams {
  const float* part;
  void* out[3];       // dweight, dpost_weight, dgate (null: not wanted)
  int C, blocks, w_bf16, g_bf16;
};

__global__ void __launch_bounds__(1024) norm_part_kernel(const __grid_constant__ PartParams p) {
  __shared__ float sm[32][33];
  const int tx = threadIdx.x % 32, ty = threadIdx.x / 32, c = blockIdx.x * 32 + tx, k = blockIdx.y;
  if (!p.out[k]) return;
  float s = 0.f;
  if (c < p.C)
#pragma unroll 8
    for (int b = ty; b < p.blocks; b += 32) s += p.part[((long long)b * 3 + k) * p.C + c];
  sm[ty][tx] = s;
  __syncthreads();
  s = sm[tx][ty];   // a warp adds up one channel
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  const int mine = blockIdx.x * 32 + ty;
  if (tx == 0 && mine < p.C) {
    if (k == 2 ? p.g_bf16 : p.w_bf16) ((__nv_bfloat16*)p.out[k])[mine] = __float2bfloat16_rn(s);
    else ((float*)p.out[k])[mine] = s;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------------------------------------------
template <class TX, class TY, int VEC, int NV, bool BLOCK>
cudaError_t rows_fwd(const NormParams& p, cudaStream_t st) {
  const int nvec = p.C / VEC, tpr = BLOCK ? ((nvec + NV - 1) / NV + 31) / 32 * 32 : 32, rpb = BLOCK ? 1 : kRowsPerBlock;
  return launch(norm_rows_kernel<TX, TY, VEC, NV, BLOCK>, dim3((unsigned)((p.rows + rpb - 1) / rpb)), tpr * rpb,
                4 * ((BLOCK ? kRedForward : 0) + rpb * rows_smem_floats(nvec, p.groups)), st, p);
}
template <class TX, class TY, int VEC, int NV, bool BLOCK>
cudaError_t rows_bwd(const NormParams& p, cudaStream_t st) {
  const int nvec = p.C / VEC, tpr = BLOCK ? ((nvec + NV - 1) / NV + 31) / 32 * 32 : 32, rpb = BLOCK ? 1 : kRowsPerBlock;
  return launch(norm_rows_bwd_kernel<TX, TY, VEC, NV, BLOCK>, dim3((unsigned)p.blocks), tpr * rpb,
                4 * ((BLOCK ? kRedBackward : 0) + rpb * rows_smem_floats(nvec, p.groups)), st, p);
}

// Vectors of a thread: one, as long as a block's threads do.
template <class TX, class TY, int VEC>
cudaError_t rows_v(const NormParams& p, bool bwd, cudaStream_t st) {
  constexpr int kVecs = kMaxChannels / VEC;   // the most of a row
  const int nvec = p.C / VEC;
  if (bwd) {
    if (nvec <= 32) return rows_bwd<TX, TY, VEC, 1, false>(p, st);
    if (nvec <= 512) return rows_bwd<TX, TY, VEC, 1, true>(p, st);
    if (nvec <= 1024) return rows_bwd<TX, TY, VEC, 2, true>(p, st);
    if constexpr (kVecs > 1024) {
      if (nvec <= 2048) return rows_bwd<TX, TY, VEC, 4, true>(p, st);
      if constexpr (kVecs > 2048) return rows_bwd<TX, TY, VEC, 16, true>(p, st);
    }
    return cudaErrorInvalidValue;
  }
  if (nvec <= 32) return rows_fwd<TX, TY, VEC, 1, false>(p, st);
  if (nvec <= 1024) return rows_fwd<TX, TY, VEC, 1, true>(p, st);
  if constexpr (kVecs > 1024) {
    if (nvec <= 2048) return rows_fwd<TX, TY, VEC, 2, true>(p, st);
    if constexpr (kVecs > 2048) return rows_fwd<TX, TY, VEC, 8, true>(p, st);
  }
  return cudaErrorInvalidValue;
}

template <class TX, class TY, int VEC>
cudaError_t first_v(const NormParams& p, bool bwd, cudaStream_t st) {
  const long long tiles = (p.rows / p.inner) * first_tiles(p.inner);
  if (bwd) {
    const int smem = 4 * (4 * p.groups * kPos + first_part_floats(p.groups, 3)), with = smem + 4 * 3 * p.C;
    NormParams q = p;
    q.sums_shared = with <= kMaxShared / 2;   // two blocks on an SM
    return launch(norm_first_bwd_kernel<TX, TY, VEC>, dim3((unsigned)p.blocks), kFirstThreads, q.sums_shared ? with : smem, st, q);
  }
  const int smem = 4 * ((p.groups + 1) * kPos + first_part_floats(p.groups, 1)), kept = smem + 4 * p.C * kPos;
  if (kept <= kMaxShared)
    return launch(norm_first_kernel<TX, TY, VEC, true>, dim3((unsigned)tiles), kFirstThreads, kept, st, p);
  return launch(norm_first_kernel<TX, TY, VEC, false>, dim3((unsigned)tiles), kFirstThreads, smem, st, p);
}

bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

template <class TX, class TY>
cudaError_t norm_t(const NormParams& p, bool bwd, cudaStream_t st) {
  if (p.inner) {
    const bool v4 = p.inner % 4 == 0 && aligned(p.x, 4 * sizeof(TX)) && aligned(p.h, 4 * sizeof(TX)) &&
                    aligned(p.dh, 4 * sizeof(TX)) && aligned(p.dx, 4 * sizeof(TX)) && aligned(p.y, 4 * sizeof(TY)) &&
                    aligned(p.n, 4 * sizeof(TY)) && aligned(p.dn, 4 * sizeof(TY)) && aligned(p.dy, 4 * sizeof(TY)) &&
                    (p.gate_kind != GATE_FULL || (aligned(p.gate, 4 * sizeof(TY)) && aligned(p.dgate, 4 * sizeof(TY))));
    return v4 ? first_v<TX, TY, 4>(p, bwd, st) : first_v<TX, TY, 1>(p, bwd, st);
  }
  constexpr int V = 16 / sizeof(TY);
  const bool vec = p.C % V == 0 && p.gc % V == 0 && p.xs % V == 0 && p.ys % V == 0 && p.gs % V == 0 && aligned(p.x, 16) &&
                   aligned(p.y, 16) && aligned(p.gate, 16) && aligned(p.h, 16) && aligned(p.n, 16) && aligned(p.dh, 16) &&
                   aligned(p.dn, 16) && aligned(p.dx, 16) && aligned(p.dy, 16) &&
                   (p.gate_kind != GATE_FULL || aligned(p.dgate, 16)) && aligned(p.pw, 16) && aligned(p.w, 16);
  return vec ? rows_v<TX, TY, V>(p, bwd, st) : rows_v<TX, TY, 1>(p, bwd, st);
}

cudaError_t norm_any(const NormParams& p, int res_io, int io, bool bwd, cudaStream_t st) {
  if (res_io == SFFFT_IO_FP32 && io == SFFFT_IO_FP32) return norm_t<float, float>(p, bwd, st);
  if (res_io == SFFFT_IO_FP32) return norm_t<float, __nv_bfloat16>(p, bwd, st);
  return norm_t<__nv_bfloat16, __nv_bfloat16>(p, bwd, st);
}

size_t io_size(int io) { return io == SFFFT_IO_BF16 ? 2 : 4; }

int check(const sffft_block_norm_t* d, const void* x, const void* y, const void* gate, const void* pw, const void* w) {
  auto io_ok = [](int v) { return v == SFFFT_IO_FP32 || v == SFFFT_IO_BF16; };
  if (!d || d->rows < 0 || d->channels < 1 || d->inner < 0 || d->groups < 1 || d->channels % d->groups != 0 ||
      !io_ok(d->io) || !io_ok(d->res_io) || !io_ok(d->weight_io) || d->gate < 0 || d->gate > 2 || d->act < 0 || d->act > 2 ||
      !std::isfinite(d->scale) || !(d->eps >= 0.f) || !std::isfinite(d->eps) || d->device < 0)
    return SFFFT_ERR_INVALID_ARGUMENT;
  if (d->inner && d->rows % d->inner != 0) return SFFFT_ERR_INVALID_ARGUMENT;
  if (!y && (!x || gate || pw || d->gate)) return SFFFT_ERR_INVALID_ARGUMENT;   // nothing to norm, or a gate of nothing
  if (!y && !w) return SFFFT_ERR_INVALID_ARGUMENT;                              // nothing to do
  if ((d->gate != 0) != (gate != nullptr)) return SFFFT_ERR_INVALID_ARGUMENT;
  if (d->res_io == SFFFT_IO_BF16 && d->io == SFFFT_IO_FP32) return SFFFT_ERR_UNSUPPORTED;
  if (!x && d->res_io != d->io) return SFFFT_ERR_UNSUPPORTED;
  if (d->channels > kMaxChannels || d->rows > INT_MAX) return SFFFT_ERR_UNSUPPORTED;
  if (d->inner && pw && d->groups > 256) return SFFFT_ERR_UNSUPPORTED;
  if (!on_elements(io_size(d->io), {y, gate}) || !on_elements(io_size(d->res_io), {x}) || !on_elements(io_size(d->weight_io), {pw, w}))
    return SFFFT_ERR_INVALID_ARGUMENT;
  return SFFFT_OK;
}

int backward_blocks(const sffft_block_norm_t* d, int sms) {
  const long long units = d->inner ? (d->rows / d->inner) * first_tiles(d->inner) : d->rows;
  // rows: as many blocks of a row's threads as an SM's registers hold at 128 each; channels first: two
  const int threads = (d->channels / (d->io == SFFFT_IO_BF16 ? 8 : 4) + 31) / 32 * 32;
  const int per_sm = d->inner ? 2 : threads > 256 ? 1 : threads <= 32 ? 4 : 512 / threads;
  const long long most = (long long)per_sm * sms;
  return (int)(units < most ? units : most);
}

int facts(int device, int* sms) {
  int major = 0, minor = 0;
  cudaError_t ce = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device);
  if (ce == cudaSuccess) ce = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
  if (ce == cudaSuccess) ce = cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, device);
  if (ce != cudaSuccess) return sffft_note_cuda_error(ce);
  return major == 10 && minor == 0 ? SFFFT_OK : SFFFT_ERR_DEVICE;
}

NormParams params(const sffft_block_norm_t* d, const void* x, const void* y, const void* gate, const void* pw, const void* w) {
  NormParams p = {};
  p.x = x; p.y = y; p.gate = gate; p.pw = pw; p.w = w;
  p.rows = d->rows; p.xs = d->x_stride; p.ys = d->y_stride; p.gs = d->gate_stride;
  if (d->gate != GATE_FULL) p.gs = 0;
  if (!x) p.xs = 0;
  if (!y) p.ys = 0;
  p.C = d->channels; p.groups = pw ? d->groups : 1; p.gc = p.C / p.groups; p.inner = d->inner;
  p.gmul = ((1u << 31) + p.gc - 1) / p.gc;
  p.gate_kind = d->gate; p.act = d->act; p.w_bf16 = d->weight_io == SFFFT_IO_BF16;
  p.scale = d->scale; p.eps = d->eps;
  return p;
}

}  // namespace
}  // namespace sffft

using namespace sffft;

extern "C" {

int sffft_block_norm(const sffft_block_norm_t* d, const void* x, const void* y, const void* gate, const void* post_weight,
                     const void* weight, void* h, void* n, float* rstd_post, float* rstd, void* stream) {
  int rc = check(d, x, y, gate, post_weight, weight);
  if (rc) return rc;
  if ((y && !h) || (weight && !n)) return SFFFT_ERR_INVALID_ARGUMENT;
  if (!on_elements(io_size(d->res_io), {h}) || !on_elements(io_size(d->io), {n}) || !on_elements(4, {rstd_post, rstd}))
    return SFFFT_ERR_INVALID_ARGUMENT;
  if (d->rows == 0) return SFFFT_OK;
  int sms;
  if ((rc = facts(d->device, &sms))) return rc;
  NormParams p = params(d, x, y, gate, post_weight, weight);
  p.h = y ? h : nullptr;
  p.n = n;
  p.r1 = rstd_post;
  p.r2 = rstd;
  DeviceScope scope(d->device);
  if (scope.err != cudaSuccess) return sffft_note_cuda_error(scope.err);
  const cudaError_t ce = norm_any(p, d->res_io, d->io, false, (cudaStream_t)stream);
  return ce == cudaSuccess ? SFFFT_OK : sffft_note_cuda_error(ce);
}

int sffft_block_norm_workspace_bytes(const sffft_block_norm_t* d, size_t* bytes) {
  if (!d || !bytes || d->rows < 0 || d->channels < 1 || d->inner < 0 || d->device < 0) return SFFFT_ERR_INVALID_ARGUMENT;
  if (d->channels > kMaxChannels || d->rows > INT_MAX) return SFFFT_ERR_UNSUPPORTED;
  int sms;
  const int rc = facts(d->device, &sms);
  if (rc) return rc;
  *bytes = (size_t)backward_blocks(d, sms) * 3 * d->channels * sizeof(float);
  return SFFFT_OK;
}

int sffft_block_norm_backward(const sffft_block_norm_t* d, const void* x, const void* y, const void* gate,
                              const void* post_weight, const void* weight, const float* rstd_post, const float* rstd,
                              const void* dh, const void* dn, void* dx, void* dy, void* dgate, void* dpost_weight,
                              void* dweight, void* work, size_t work_bytes, void* stream) {
  int rc = check(d, x, y, gate, post_weight, weight);
  if (rc) return rc;
  if ((x && !dx) || (y && !dy) || (gate && !dgate) || (post_weight && (!dpost_weight || !rstd_post)) ||
      (weight && (!dweight || !rstd || !dn)) || (!weight && !dh))
    return SFFFT_ERR_INVALID_ARGUMENT;
  if (((uintptr_t)work & 255) != 0) return SFFFT_ERR_INVALID_ARGUMENT;
  if (!on_elements(io_size(d->res_io), {dh, dx}) || !on_elements(io_size(d->io), {dn, dy, dgate}) ||
      !on_elements(io_size(d->weight_io), {dpost_weight, dweight}) || !on_elements(4, {rstd_post, rstd}))
    return SFFFT_ERR_INVALID_ARGUMENT;
  int sms;
  if ((rc = facts(d->device, &sms))) return rc;
  NormParams p = params(d, x, y, gate, post_weight, weight);
  p.r1 = const_cast<float*>(rstd_post);
  p.r2 = const_cast<float*>(rstd);
  p.dh = dh; p.dn = weight ? dn : nullptr; p.dx = x ? dx : nullptr; p.dy = dy; p.dgate = dgate;
  p.blocks = backward_blocks(d, sms);
  p.part = (float*)work;
  const size_t need = (size_t)p.blocks * 3 * d->channels * sizeof(float);
  if (need && (!work || work_bytes < need)) return SFFFT_ERR_WORKSPACE;
  DeviceScope scope(d->device);
  if (scope.err != cudaSuccess) return sffft_note_cuda_error(scope.err);
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t ce = cudaSuccess;
  if (p.blocks) ce = norm_any(p, d->res_io, d->io, true, st);
  const bool cg = d->gate == GATE_CHANNEL;
  if (ce == cudaSuccess && (weight || post_weight || cg)) {   // with no rows the sums are zero
    PartParams q = {p.part, {weight ? dweight : nullptr, post_weight ? dpost_weight : nullptr, cg ? dgate : nullptr},
                    d->channels, p.blocks, p.w_bf16, d->io == SFFFT_IO_BF16};
    ce = launch(norm_part_kernel, dim3((unsigned)((d->channels + 31) / 32), 3), 1024, 0, st, q);
  }
  return ce == cudaSuccess ? SFFFT_OK : sffft_note_cuda_error(ce);
}

}  // extern "C"
