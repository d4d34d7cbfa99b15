// Linear attention with a decay for each head, fp32 arithmetic on CUDA cores.
//
// A block takes one head of one row, up to 64 columns of v and one segment of positions, C at a time.  With P the
// C x C products q_i . k_j times lambda^(i-j) for j <= i, and S the state before the chunk (D x 64, in shared memory):
//   y_i = scale * (sum_j P_ij v_j + lambda^(i+1) q_i^T S),   S <- lambda^C S + sum_j lambda^(C-1-j) k_j v_j^T
// so that a token costs 2 C (D + 64) + 4 * 64 D flop instead of L (D + 64).
//
// Few heads and a long row leave most SMs idle, so the positions are then cut into G segments: a first launch leaves
// the state that each segment builds from zero, a second sums them up in segment order, and a block of the main launch
// starts from the sum before it.  The price is a second reading of k and v.
//
// Time reversal (the gradients of k and v) is a matter of addressing: processing position p reads token n-1-p.
//
// Bound by the issue of its instructions: 2 x 12 heads x 2047 x 64 in fp32 take 106 us in three launches, of which the
// multiply-adds alone would be 25 and the bytes 8; each FMA comes with half a shared-memory load and the chunk's set-up, and
// the issue slots are 56 to 61 % busy at 16 warps an SM (what its registers and shared memory hold).  Chunks of 64 positions
// up to head size 128, 32 above: what shared memory holds beside the state.
#include <cuda_bf16.h>

#include "launch.h"
#include "linattn.h"

namespace sffft {
namespace {

constexpr int kCols = 64;   // columns of v in a block
constexpr int kThreads = 256;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f(float& d, float x) { d = x; }
__device__ __forceinline__ void from_f(__nv_bfloat16& d, float x) { d = __float2bfloat16_rn(x); }

// N consecutive floats of shared memory, 16 (N = 2: 8) byte aligned
template <int N>
__device__ __forceinline__ void lds(const float* p, float (&v)[N]) {
  if constexpr (N == 4) {
    const float4 a = *(const float4*)p;
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  } else {
    const float2 a = *(const float2*)p;
    v[0] = a.x, v[1] = a.y;
  }
}

template <int DM, int C>
struct GeneralSmem {
  static constexpr int PT = C + 4;   // pitch of the [d][token] images: a multiple of 4, and 4-way conflicts at worst
  static constexpr int bytes = 4 * (2 * DM * PT + C * kCols + C * PT + DM * kCols + C + 4);
};

template <class T, int DM, int C, bool LOCAL>
__global__ void __launch_bounds__(kThreads, DM == 64 ? 2 : 1) la_general_kernel(const __grid_constant__ LaParams prm) {
  constexpr int PT = GeneralSmem<DM, C>::PT, TI = C / 16;
  extern __shared__ __align__(16) float sm[];
  float* Qt = sm;                  // [DM][PT]
  float* Kt = Qt + DM * PT;        // [DM][PT]
  float* V = Kt + DM * PT;         // [C][kCols]
  float* Pt = V + C * kCols;       // [C][PT], transposed: Pt[j][i]
  float* S = Pt + C * PT;          // [DM][kCols]
  float* pw = S + DM * kCols;      // lambda^0 .. lambda^C
  const LaTask& tk = prm.task[blockIdx.z];
  const int D = tk.D, Dv = tk.Dv, c0 = blockIdx.y * kCols;
  if (c0 >= Dv) return;
  const int g = blockIdx.x % prm.G, bh = blockIdx.x / prm.G, b = bh / prm.H, h = bh % prm.H;
  if (LOCAL && g == prm.G - 1) return;   // nothing follows the last segment
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  int n = prm.L;
  if (prm.len) n = min(max(prm.len[b], 0), prm.L);
  const int ps = min(g * prm.seg, n), pe = min((g + 1) * prm.seg, n);
  const LaDecay dec(prm.ld[h]);
  for (int i = tid; i <= C; i += kThreads) pw[i] = dec.pow(i);
  const float whole_lo = dec.pow_rest(C, dec.pow(C));

  const T* q = (const T*)tk.q + b * tk.qs[0] + (h / tk.qdiv) * tk.qs[1];
  const T* k = (const T*)tk.k + b * tk.ks[0] + (h / tk.kdiv) * tk.ks[1];
  const T* v = (const T*)tk.v + b * tk.vs[0] + (h / tk.vdiv) * tk.vs[1];
  const long long ybase = b * tk.ys[0] + h * tk.ys[1];

  // state before the segment: the start state, or what the earlier segments leave
  const float* in = LOCAL || g == 0 ? nullptr : tk.loc + ((long long)bh * prm.G + g - 1) * D * Dv;
  for (int e = tid; e < DM * kCols; e += kThreads) {
    const int d = e / kCols, c = c0 + e % kCols;
    float s = 0.f;
    if (!LOCAL && d < D && c < Dv) {
      if (in) s = in[(long long)d * Dv + c];
      else if (tk.s0) s = tk.s0[b * tk.s0s[0] + h * tk.s0s[1] + d * tk.s0s[2] + c * tk.s0s[3]] * tk.s0_mul;
    }
    S[e] = s;
  }
  __syncthreads();

  // The next chunk's q, k and v are on their way (in registers) while a chunk is worked on: read element by element, as any
  // stride and size allow, each would otherwise cost the memory's latency.
  constexpr int NQ = DM * C / kThreads, NV = C * kCols / kThreads;
  float rq[LOCAL ? 1 : NQ], rk[NQ], rv[NV];
  auto fetch = [&](int p0) {
    const int m = min(C, pe - p0);
#pragma unroll
    for (int x = 0; x < NQ; x++) {
      const int e = x * kThreads + tid, d = e % DM, i = e / DM;
      const bool there = i < m && d < D;
      const long long t = tk.rev ? n - 1 - (p0 + i) : p0 + i;
      if (!LOCAL) rq[x] = there ? to_f(q[t * tk.qs[2] + d]) : 0.f;
      rk[x] = there ? to_f(k[t * tk.ks[2] + d]) : 0.f;
    }
#pragma unroll
    for (int x = 0; x < NV; x++) {
      const int e = x * kThreads + tid, i = e / kCols, c = c0 + e % kCols;
      const long long t = tk.rev ? n - 1 - (p0 + i) : p0 + i;
      rv[x] = i < m && c < Dv ? to_f(v[t * tk.vs[2] + c]) : 0.f;
    }
  };
  if (ps < pe) fetch(ps);
  for (int p0 = ps; p0 < pe; p0 += C) {
    const int m = min(C, pe - p0);
    const int off = (tk.off && p0 == 0) ? 1 : 0;
#pragma unroll
    for (int x = 0; x < NQ; x++) {
      const int e = x * kThreads + tid, d = e % DM, i = e / DM;
      if (!LOCAL) Qt[d * PT + i] = rq[x];
      Kt[d * PT + i] = LOCAL ? rk[x] * pw[max(m - 1 - i, 0)] : rk[x];
    }
#pragma unroll
    for (int x = 0; x < NV; x++) V[x * kThreads + tid] = rv[x];
    __syncthreads();
    if (p0 + C < pe) fetch(p0 + C);
    if (!LOCAL) {
      {
        float acc[TI][TI] = {};
#pragma unroll 4
        for (int d = 0; d < D; d++) {
          float a[TI], c[TI];
          lds<TI>(Qt + d * PT + ty * TI, a);
          lds<TI>(Kt + d * PT + tx * TI, c);
#pragma unroll
          for (int x = 0; x < TI; x++)
#pragma unroll
            for (int y = 0; y < TI; y++) acc[x][y] = fmaf(a[x], c[y], acc[x][y]);
        }
#pragma unroll
        for (int y = 0; y < TI; y++)
#pragma unroll
          for (int x = 0; x < TI; x++) {
            const int i = ty * TI + x, j = tx * TI + y;
            Pt[j * PT + i] = i >= j ? acc[x][y] * pw[max(i - j, 0)] : 0.f;
          }
      }
      __syncthreads();
      float o[TI][4] = {}, r[TI][4] = {};
#pragma unroll 4
      for (int j = 0; j < m; j++) {
        float a[TI], c[4];
        lds<TI>(Pt + j * PT + ty * TI, a);
        lds<4>(V + j * kCols + tx * 4, c);
#pragma unroll
        for (int x = 0; x < TI; x++)
#pragma unroll
          for (int y = 0; y < 4; y++) o[x][y] = fmaf(a[x], c[y], o[x][y]);
      }
#pragma unroll 4
      for (int d = 0; d < D; d++) {
        float a[TI], c[4];
        lds<TI>(Qt + d * PT + ty * TI, a);
        lds<4>(S + d * kCols + tx * 4, c);
#pragma unroll
        for (int x = 0; x < TI; x++)
#pragma unroll
          for (int y = 0; y < 4; y++) r[x][y] = fmaf(a[x], c[y], r[x][y]);
      }
#pragma unroll
      for (int x = 0; x < TI; x++) {
        const int i = ty * TI + x;
        if (i >= m) continue;
        const long long t = tk.rev ? n - 1 - (p0 + i) : p0 + i;
        const float w = pw[i + 1 - off];
#pragma unroll
        for (int y = 0; y < 4; y++) {
          const int c = c0 + tx * 4 + y;
          if (c >= Dv) continue;
          const float z = tk.scale * fmaf(w, r[x][y], o[x][y]);
          const long long at = ybase + t * tk.ys[2] + c;
          if (tk.y_f32) ((float*)tk.y)[at] = z;
          else from_f(((T*)tk.y)[at], z);
        }
      }
      __syncthreads();
      for (int e = tid; e < DM * C; e += kThreads) Kt[(e % DM) * PT + e / DM] *= pw[max(m - 1 - e / DM, 0)];
      __syncthreads();
    }
    // lambda^C as a sum of two floats: its rounding would come back with every chunk
    const float ws = pw[m - off], ws_lo = m - off == C ? whole_lo : 0.f;
    for (int d0 = ty * 4; d0 < D; d0 += 64) {
      float acc[4][4];
#pragma unroll
      for (int x = 0; x < 4; x++)
#pragma unroll
        for (int y = 0; y < 4; y++) acc[x][y] = 0.f;
      for (int j = 0; j < m; j += 4) {   // behind the last position there are zeros
        float a[4][4], c[4][4];   // [d][j], [j][column]
#pragma unroll
        for (int x = 0; x < 4; x++) lds<4>(Kt + (d0 + x) * PT + j, a[x]), lds<4>(V + (j + x) * kCols + tx * 4, c[x]);
#pragma unroll
        for (int z = 0; z < 4; z++)
#pragma unroll
          for (int x = 0; x < 4; x++)
#pragma unroll
            for (int y = 0; y < 4; y++) acc[x][y] = fmaf(a[x][z], c[z][y], acc[x][y]);
      }
#pragma unroll
      for (int x = 0; x < 4; x++)
#pragma unroll
        for (int y = 0; y < 4; y++) {
          float& s = S[(d0 + x) * kCols + tx * 4 + y];
          s = fmaf(ws, s, fmaf(ws_lo, s, acc[x][y]));
        }
    }
    __syncthreads();
  }

  if (LOCAL) {
    float* out = tk.loc + ((long long)bh * prm.G + g) * D * Dv;
    for (int e = tid; e < DM * kCols; e += kThreads) {
      const int d = e / kCols, c = c0 + e % kCols;
      if (d < D && c < Dv) out[(long long)d * Dv + c] = S[e];
    }
    return;
  }
  if (tk.s1 && g == prm.G - 1) {
    const float w = tk.s1_mul * (tk.s1_decay && n > 0 ? pw[1] : 1.f);
    for (int e = tid; e < DM * kCols; e += kThreads) {
      const int d = e / kCols, c = c0 + e % kCols;
      if (d < D && c < Dv) tk.s1[b * tk.s1s[0] + h * tk.s1s[1] + d * tk.s1s[2] + c * tk.s1s[3]] = w * S[e];
    }
  }
  // positions behind the row's last token
  const int z0 = max(g * prm.seg, n), z1 = min((g + 1) * prm.seg, prm.L);
  for (long long e = tid; e < (long long)(z1 - z0) * kCols; e += kThreads) {
    const long long t = z0 + e / kCols;
    const int c = c0 + (int)(e % kCols);
    if (c >= Dv) continue;
    const long long at = ybase + t * tk.ys[2] + c;
    if (tk.y_f32) ((float*)tk.y)[at] = 0.f;
    else from_f(((T*)tk.y)[at], 0.f);
  }
}

// What the segments up to each one leave, the start state's part included, from what each leaves alone; in place.  A
// thread takes one element of a state.
__global__ void __launch_bounds__(256) la_general_prefix_kernel(const __grid_constant__ LaParams prm) {
  const LaTask& tk = prm.task[blockIdx.z];
  const int size = tk.D * tk.Dv, e = blockIdx.y * 256 + threadIdx.x;
  const int bh = blockIdx.x, b = bh / prm.H, h = bh % prm.H;
  if (e >= size) return;
  int n = prm.L;
  if (prm.len) n = min(max(prm.len[b], 0), prm.L);
  const LaDecay dec(prm.ld[h]);
  float s = 0.f;
  if (tk.s0) s = tk.s0[b * tk.s0s[0] + h * tk.s0s[1] + (e / tk.Dv) * tk.s0s[2] + (e % tk.Dv) * tk.s0s[3]] * tk.s0_mul;
  float* loc = tk.loc + (long long)bh * prm.G * size + e;
  for (int g0 = 0; g0 < prm.G - 1; g0 += 8) {
    float x[8];   // the loads do not wait for the sums
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (g0 + i < prm.G - 1) x[i] = loc[(long long)(g0 + i) * size];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int g = g0 + i;
      if (g >= prm.G - 1) break;
      const int a = min(g * prm.seg, n), m = min((g + 1) * prm.seg, n) - a;
      if (m > 0) s = fmaf(dec.pow(m - (tk.off && a == 0)), s, x[i]);
      loc[(long long)g * size] = s;
    }
  }
}

template <class T, int DM, int C>
cudaError_t launch_t(const LaParams& prm, int dv_max, cudaStream_t st) {
  const dim3 grid((unsigned)(prm.B * prm.H * prm.G), (unsigned)((dv_max + kCols - 1) / kCols), (unsigned)prm.ntask);
  constexpr int bytes = GeneralSmem<DM, C>::bytes;
  if (prm.G > 1) {
    cudaError_t ce = launch(la_general_kernel<T, DM, C, true>, grid, kThreads, bytes, st, prm);
    if (ce != cudaSuccess) return ce;
    int size = 0;
    for (int i = 0; i < prm.ntask; i++) size = max(size, prm.task[i].D * prm.task[i].Dv);
    ce = launch(la_general_prefix_kernel, dim3((unsigned)(prm.B * prm.H), (unsigned)((size + 255) / 256), (unsigned)prm.ntask), 256, 0, st, prm);
    if (ce != cudaSuccess) return ce;
  }
  return launch(la_general_kernel<T, DM, C, false>, grid, kThreads, bytes, st, prm);
}

template <class T>
cudaError_t launch_d(const LaParams& prm, cudaStream_t st) {
  int d = 0, dv = 0;
  for (int i = 0; i < prm.ntask; i++) d = max(d, prm.task[i].D), dv = max(dv, prm.task[i].Dv);
  if (d <= 64) return launch_t<T, 64, 64>(prm, dv, st);
  if (d <= 128) return launch_t<T, 128, 64>(prm, dv, st);
  return launch_t<T, 256, 32>(prm, dv, st);
}

}  // namespace

cudaError_t launch_la_general(const LaParams& prm, bool bf16, cudaStream_t st) {
  return bf16 ? launch_d<__nv_bfloat16>(prm, st) : launch_d<float>(prm, st);
}

}  // namespace sffft
