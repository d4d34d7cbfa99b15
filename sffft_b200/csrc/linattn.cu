// Linear attention with a decay for each head: C ABI, planning, the single-token kernel and the sum over the heads
// that share a key and value head.
#include <cuda_bf16.h>

#include <algorithm>
#include <climits>
#include <type_traits>
#include <cmath>

#include "../../include/sffft.h"
#include "launch.h"
#include "linattn.h"

int sffft_note_cuda_error(cudaError_t e);

namespace sffft {
namespace {

__device__ __forceinline__ float ldf(const float* p) { return *p; }
__device__ __forceinline__ float ldf(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void stf(float* p, float x) { *p = x; }
__device__ __forceinline__ void stf(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// ---------------------------------------------------------------------------------------------------------------
// Single tokens: S <- lambda S + k v^T, y = scale q^T S.
//
// Bound by the state, D Dv fp32 values read and written once for each head and row.  A block takes 32 columns of one
// state (128-byte rows): 8 threads across with 4 columns each, 16 rows at a time, so that a single row of 12 heads
// still spreads over 24 blocks at Dv = 64; each thread issues kStepAhead loads before it uses the first.
// Measured: 200 rows of 8 heads of 128 x 128: 43 us with the launch for 210 MB (4.9 TB/s); 512 rows of 12: 130 us for 805 MB
// (6.2 TB/s); one row of 12 heads of 64 x 64 is a launch.
// ---------------------------------------------------------------------------------------------------------------
struct LaStepParams {
  const void *q, *k, *v;
  void* y;
  float* state;
  const int* slots;
  const float* ld;
  long long qs[2], ks[2], vs[2], ys[2], ss;   // row, head; state: slot
  int B, H, kv_div, D, Dv, pool;
  float scale;
};

constexpr int kStepThreads = 128, kStepCols = 32, kStepAhead = 8;

template <class T, int VEC>
__global__ void __launch_bounds__(kStepThreads) la_step_kernel(const __grid_constant__ LaStepParams prm) {
  constexpr int TX = kStepCols / VEC, TY = kStepThreads / TX;
  __shared__ float part[TY][kStepCols];
  const int bh = blockIdx.x, b = bh / prm.H, h = bh % prm.H;
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  const int c = blockIdx.y * kStepCols + tx * VEC;
  const bool in = c < prm.Dv;   // VEC 4: Dv is a multiple of 4
  const int slot = prm.slots ? prm.slots[b] : b;
  const bool ok = slot >= 0 && slot < prm.pool;
  const T* q = (const T*)prm.q + b * prm.qs[0] + h * prm.qs[1];
  const T* k = (const T*)prm.k + b * prm.ks[0] + (h / prm.kv_div) * prm.ks[1];
  const T* v = (const T*)prm.v + b * prm.vs[0] + (h / prm.kv_div) * prm.vs[1];
  float* S = prm.state + (ok ? slot : 0) * prm.ss + (long long)h * prm.D * prm.Dv + c;
  float st[kStepAhead][VEC];
  auto load = [&](int d0) {
#pragma unroll
    for (int a = 0; a < kStepAhead; a++) {
      const int d = d0 + a * TY;
      if (d >= prm.D) continue;
      if constexpr (VEC == 4) {
        const float4 x = __ldcs((const float4*)(S + (long long)d * prm.Dv));
        st[a][0] = x.x, st[a][1] = x.y, st[a][2] = x.z, st[a][3] = x.w;
      } else {
        st[a][0] = __ldcs(S + (long long)d * prm.Dv);
      }
    }
  };
  // The first rows of the state are on their way while the slots are looked through.
  const bool there = ok && in;
  if (there) load(ty);
  const float lam = LaDecay(prm.ld[h]).pow(1);
  float vv[VEC], acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; e++) vv[e] = in ? ldf(v + c + e) : 0.f, acc[e] = 0.f;
  // Rows that name a slot again after an earlier row of the call leave it alone: the first one alone updates it.
  int again = 0;
  if (prm.slots)
    for (int r = threadIdx.x; r < b; r += kStepThreads) again |= prm.slots[r] == slot;
  if (!__syncthreads_or(again) && there) {
    for (int d0 = ty; d0 < prm.D; d0 += TY * kStepAhead) {
      if (d0 > ty) load(d0);
#pragma unroll
      for (int a = 0; a < kStepAhead; a++) {
        const int d = d0 + a * TY;
        if (d >= prm.D) continue;
        const float kd = ldf(k + d), qd = ldf(q + d);
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          st[a][e] = fmaf(lam, st[a][e], kd * vv[e]);
          acc[e] = fmaf(qd, st[a][e], acc[e]);
        }
        if constexpr (VEC == 4) __stcs((float4*)(S + (long long)d * prm.Dv), make_float4(st[a][0], st[a][1], st[a][2], st[a][3]));
        else __stcs(S + (long long)d * prm.Dv, st[a][0]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; e++) part[ty][tx * VEC + e] = acc[e];
  __syncthreads();
  const int col = threadIdx.x, cc = blockIdx.y * kStepCols + col;
  if (col < kStepCols && cc < prm.Dv) {
    float z = 0.f;
#pragma unroll
    for (int r = 0; r < TY; r++) z += part[r][col];
    stf((T*)prm.y + b * prm.ys[0] + h * prm.ys[1] + cc, prm.scale * z);
  }
}

// Sum over the query heads that share a key and value head, in head order: out[b][g][t] = sum_r w[b][g R + r][t].  Bound by
// memory: a thread takes VEC values of a position; blockIdx.y is the row and head, so that no index needs a division but
// that by the D / VEC pieces of a position.
struct LaReduceParams {
  const float* w;   // [B][G R][L][D]
  void* out;
  long long os[3];
  int B, G, R, L, D;
};

template <class T, int VEC>
__global__ void __launch_bounds__(256) la_reduce_kernel(const __grid_constant__ LaReduceParams p) {
  const long long plane = (long long)p.L * p.D;
  const unsigned pieces = p.D / VEC;
  // pieces of a row and head: within 32 bits where they are 8 values (2^32 of them for two heads alone would be 256 GB)
  typedef typename std::conditional<VEC == 8, unsigned, unsigned long long>::type Index;
  const Index total = (Index)p.L * pieces;
  for (int bg = blockIdx.y; bg < p.B * p.G; bg += gridDim.y) {
    const float* w = p.w + (long long)bg * p.R * plane;
    T* out = (T*)p.out + (bg / p.G) * p.os[0] + (bg % p.G) * p.os[1];
    for (Index e = blockIdx.x * 256u + threadIdx.x; e < total; e += gridDim.x * 256u) {
      const unsigned t = (unsigned)(e / pieces), d = (unsigned)(e - (Index)t * pieces) * VEC;
      float s[VEC] = {};
      for (int r = 0; r < p.R; r++) {
        const float* x = w + r * plane + (long long)e * VEC;
        if constexpr (VEC == 8) {
          const float4 a = *(const float4*)x, c = *(const float4*)(x + 4);
          s[0] += a.x, s[1] += a.y, s[2] += a.z, s[3] += a.w, s[4] += c.x, s[5] += c.y, s[6] += c.z, s[7] += c.w;
        } else {
          s[0] += *x;
        }
      }
      T* to = out + (long long)t * p.os[2] + d;
#pragma unroll
      for (int i = 0; i < VEC; i++) stf(to + i, s[i]);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Planning
// ---------------------------------------------------------------------------------------------------------------
constexpr int kMaxSegments = 32;

// sffft_debug_linear_attention's, for the calls of its thread
thread_local unsigned long long t_wait_ns = kLaWaitNs;
thread_local int t_withhold = LA_WITHHOLD_NONE;

struct DeviceFacts {
  int sms = 0, ok = 0;
};

cudaError_t device_facts(int device, DeviceFacts* f) {
  int major = 0, minor = 0;
  cudaError_t ce = cudaDeviceGetAttribute(&f->sms, cudaDevAttrMultiProcessorCount, device);
  if (ce == cudaSuccess) ce = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
  if (ce == cudaSuccess) ce = cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, device);
  f->ok = major == 10 && minor == 0;
  return ce;
}

// How many segments the rows are cut into.  Few heads leave SMs idle, which segments fill; they cost a second reading of k and
// v and two more launches, so rows of many heads stay whole.  The choice is the least of, in us,
//   whole:       start + waves * chunks * one           cut: cut + waves * (start_cut + chunks of a segment * both)
// where `both` takes the segment's own state, too, and a wave is what the SMs hold at once.  The constants fit 572
// measured times (head sizes 64, 128 and 256, forward and backward, 3 to 400 heads of 4 to 128 chunks, 1 to 32 segments): the choice is
// within 12 % of the best of them, 0.7 % on average.  E.g. 96 heads x 4096 x 128 in bf16: whole 168 us, two segments 224, twelve 306;
// 16 heads: whole 161, six segments 65.
struct ChunkTimes {
  double one, both, start, start_cut, cut;
  bool pairs;   // two blocks on an SM, which together take 1.72 times as long as one
};

struct LaunchPlan {
  long long blocks;   // in a segment
  ChunkTimes t;
};

double waves(long long blocks, bool pairs, int sms) {
  if (!pairs) return (double)((blocks + sms - 1) / sms);
  const long long full = blocks / (2 * sms), rest = blocks % (2 * sms);
  return (double)full * 1.72 + (rest == 0 ? 0.0 : rest <= sms ? 1.0 : 1.72);
}

void plan_segments(const LaunchPlan* l, int n, long long chunks, int sms, int* G, long long* per) {
  double best = 0;
  *G = 1, *per = chunks;
  for (int g = 1; g <= kMaxSegments && g <= chunks; g++) {
    const long long m = (chunks + g - 1) / g;
    if ((chunks + m - 1) / m != g) continue;   // as many chunks a segment as with fewer of them
    double cost = 0;
    for (int i = 0; i < n; i++) {
      const ChunkTimes& t = l[i].t;
      const double w = waves(l[i].blocks * g, t.pairs, sms);
      cost += g == 1 ? t.start + w * (double)m * t.one : t.cut + w * (t.start_cut + (double)m * t.both);
    }
    if (g == 1 || cost < best) best = cost, *G = g, *per = m;
  }
}

void plan_general(int B, int H, int L, int D, int Dv, int ntask, int sms, int* G, int* seg) {
  const int chunk = la_general_chunk(D);
  const LaunchPlan l = {(long long)B * H * ((Dv + 63) / 64) * ntask, D <= 64    ? ChunkTimes{12.6, 16, 11, 4, 18, true}
                                                                     : D <= 128 ? ChunkTimes{19.8, 26, 12, 8, 20, false}
                                                                                : ChunkTimes{23.3, 35, 16, 8, 30, false}};
  long long per;
  plan_segments(&l, 1, ((long long)L + chunk - 1) / chunk, sms, G, &per);
  *seg = (int)(per < 1 ? chunk : per * chunk);
}

// One launch for each tile shape.  `out`: the state is an output, whose third part of X waits for the product of the others
// at head sizes above 64; with segments that is the last one's lot alone.
void plan_tc(int B, int H, int L, int D, int Dv, bool backward, int sms, int* G, int* seg) {
  auto launch = [&](int d, int dv, int tasks, bool out) {
    const bool wide = la_tc_tile(d, dv) == 128;
    return LaunchPlan{(long long)B * H * tasks * la_tc_slices(d, dv),
                      d <= 64 ? ChunkTimes{2.1, 3.5, 11, 10, 16, false}
                      : wide  ? (out ? ChunkTimes{4.6, 6.4, 14, 17, 20, false} : ChunkTimes{3.4, 5.4, 11, 16, 16, false})
                              : (out ? ChunkTimes{3.6, 5.4, 13, 14, 16, false} : ChunkTimes{2.9, 4.6, 11, 14, 16, false})};
  };
  LaunchPlan l[2];
  int n = 1;
  if (!backward) l[0] = launch(D, Dv, 1, true);
  else if ((D > 64) == (Dv > 64)) l[0] = launch(D > Dv ? D : Dv, D > Dv ? D : Dv, 3, false);   // of one shape
  else l[0] = launch(Dv, D, 2, false), l[1] = launch(D, Dv, 1, false), n = 2;
  long long per;
  plan_segments(l, n, ((long long)L + kLaTcChunk - 1) / kLaTcChunk, sms, G, &per);
  *seg = (int)(per < 1 ? kLaTcChunk : per * kLaTcChunk);
}

size_t io_size(int io) { return io == SFFFT_IO_BF16 ? 2 : 4; }

struct Sizes {
  size_t loc[kLaMaxTasks], grad_k, grad_v, total;
};

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

bool bad_shape(const sffft_linear_attention_t* p) {
  return !p || p->B < 0 || p->H < 1 || p->Hkv < 1 || p->H % p->Hkv != 0 || p->L < 0 || p->D < 1 || p->Dv < 1 ||
         (p->io != SFFFT_IO_FP32 && p->io != SFFFT_IO_BF16) || p->device < 0 || !std::isfinite(p->scale) || p->scale == 0.f;
}

int too_large(const sffft_linear_attention_t* p) {
  if (p->D > 256 || p->Dv > 4096) return 1;
  return (long long)p->B * p->H * kMaxSegments > INT_MAX || p->L > (1 << 30);
}

Sizes sizes(const sffft_linear_attention_t* p, int backward, int G) {
  Sizes s = {};
  const size_t bh = (size_t)p->B * p->H, st = bh * (size_t)p->D * p->Dv * 4;
  for (int i = 0; i < (backward ? 3 : 1); i++) {
    s.loc[i] = G > 1 ? up256(st * G) : 0;
    s.total += s.loc[i];
  }
  if (backward && p->Hkv < p->H) {
    s.grad_k = up256(bh * p->L * (size_t)p->D * 4);
    s.grad_v = up256(bh * p->L * (size_t)p->Dv * 4);
    s.total += s.grad_k + s.grad_v;
  }
  return s;
}

void plan(const sffft_linear_attention_t* p, int backward, bool tc, int sms, int* G, int* seg) {
  const int D = backward ? (p->D > p->Dv ? p->D : p->Dv) : p->D, Dv = backward ? D : p->Dv;
  if (tc) plan_tc(p->B, p->H, p->L, p->D, p->Dv, backward != 0, sms, G, seg);
  else plan_general(p->B, p->H, p->L, D, Dv, backward ? 3 : 1, sms, G, seg);
}

// Chooses the kernel and the segments, hands out the workspace, and launches.
int run(const sffft_linear_attention_t* p, int backward, LaParams* prm, const DeviceFacts& f, char* work, size_t work_bytes,
        cudaStream_t st) {
  const bool bf = p->io == SFFFT_IO_BF16, tc = bf && la_tc_takes(*prm);
  prm->wait_ns = t_wait_ns;
  prm->withhold = t_withhold;
  plan(p, backward, tc, f.sms, &prm->G, &prm->seg);
  if (tc) {
    long long slices = 0;
    for (int i = 0; i < prm->ntask; i++) slices += la_tc_slices(prm->task[i].D, prm->task[i].Dv);
    if ((long long)p->B * p->H * prm->G * slices * prm->ntask > INT_MAX) return SFFFT_ERR_UNSUPPORTED;   // CTAs of a launch
  }
  const Sizes sz = sizes(p, backward, prm->G);
  const size_t need = sz.total - sz.grad_k - sz.grad_v;
  if (need && (!work || work_bytes < need)) return SFFFT_ERR_WORKSPACE;
  for (int i = 0; i < prm->ntask; i++) {
    prm->task[i].loc = (float*)work;
    work += sz.loc[i];
  }
  cudaError_t ce = tc ? la_tc_word(p->device, &prm->status) : cudaSuccess;
  if (ce == cudaSuccess) ce = tc ? launch_la_tc(*prm, st) : launch_la_general(*prm, bf, st);
  return ce == cudaSuccess ? SFFFT_OK : sffft_note_cuda_error(ce);
}

template <class T>
void copy3(long long (&d)[3], const T* s) {
  for (int i = 0; i < 3; i++) d[i] = s[i];
}

// Element strides of a contiguous state [B][H][D][Dv], or of its transposed use.
void state_strides(long long (&s)[4], const sffft_linear_attention_t* p, bool transposed) {
  const long long n = (long long)p->D * p->Dv;
  s[0] = p->H * n;
  s[1] = n;
  s[2] = transposed ? 1 : p->Dv;
  s[3] = transposed ? p->Dv : 1;
}

int common_checks(const sffft_linear_attention_t* p, const void* log_decay) {
  if (bad_shape(p) || !log_decay) return SFFFT_ERR_INVALID_ARGUMENT;
  if (too_large(p)) return SFFFT_ERR_UNSUPPORTED;
  return SFFFT_OK;
}

int start(const sffft_linear_attention_t* p, DeviceFacts* f) {
  const cudaError_t ce = device_facts(p->device, f);
  if (ce != cudaSuccess) return sffft_note_cuda_error(ce);
  return f->ok ? SFFFT_OK : SFFFT_ERR_DEVICE;
}

template <class T>
cudaError_t reduce_t(const LaReduceParams& r, int sms, cudaStream_t st) {
  if (r.B == 0 || r.L == 0) return cudaSuccess;
  const bool vec = r.D % 8 == 0;
  const long long per = ((long long)r.L * (vec ? r.D / 8 : r.D) + 255) / 256;
  const long long heads = (long long)r.B * r.G, most = std::max(1ll, 16ll * sms / heads);
  const dim3 grid((unsigned)std::min(per, most), (unsigned)std::min(heads, 65535ll));
  return vec ? launch(la_reduce_kernel<T, 8>, grid, 256, 0, st, r) : launch(la_reduce_kernel<T, 1>, grid, 256, 0, st, r);
}

}  // namespace
}  // namespace sffft

using namespace sffft;

extern "C" {

int sffft_linear_attention_workspace_bytes(const sffft_linear_attention_t* p, int backward, size_t* bytes) {
  if (bad_shape(p) || !bytes) return SFFFT_ERR_INVALID_ARGUMENT;
  if (too_large(p)) return SFFFT_ERR_UNSUPPORTED;
  *bytes = 0;
  if (p->B == 0) return SFFFT_OK;
  DeviceFacts f;
  const int rc = start(p, &f);
  if (rc) return rc;
  for (int tc = 0; tc < 2; tc++) {   // which kernel runs also depends on the tensors' addresses and strides
    int G, seg;
    plan(p, backward, tc != 0, f.sms, &G, &seg);
    const size_t n = sizes(p, backward, G).total;
    if (n > *bytes) *bytes = n;
  }
  return SFFFT_OK;
}

int sffft_linear_attention(const sffft_linear_attention_t* p, const void* q, const void* k, const void* v,
                           const float* log_decay, const int* lengths, const float* initial_state, void* y,
                           float* final_state, void* work, size_t work_bytes, void* stream) {
  int rc = common_checks(p, log_decay);
  if (rc) return rc;
  if (p->B == 0) return SFFFT_OK;
  if (p->L > 0 && (!q || !k || !v || !y)) return SFFFT_ERR_INVALID_ARGUMENT;
  if (((uintptr_t)work & 255) != 0) return SFFFT_ERR_INVALID_ARGUMENT;
  if (!on_elements(io_size(p->io), {q, k, v, y}) || !on_elements(4, {log_decay, lengths, initial_state, final_state}))
    return SFFFT_ERR_INVALID_ARGUMENT;
  if (initial_state && initial_state == final_state) return SFFFT_ERR_INVALID_ARGUMENT;   // segments start from it all along
  if ((rc = la_tc_reported(p->device))) return rc;
  DeviceFacts f;
  if ((rc = start(p, &f))) return rc;
  LaParams prm = {};
  prm.ld = log_decay; prm.len = lengths;
  prm.ntask = 1; prm.B = p->B; prm.H = p->H; prm.L = p->L; prm.sms = f.sms;
  LaTask& t = prm.task[0];
  t.q = q; t.k = k; t.v = v; t.y = y;
  copy3(t.qs, p->q_stride); copy3(t.ks, p->k_stride); copy3(t.vs, p->v_stride); copy3(t.ys, p->y_stride);
  t.qdiv = 1; t.kdiv = t.vdiv = p->H / p->Hkv;
  t.s0 = initial_state; t.s0_mul = 1.f; state_strides(t.s0s, p, false);
  t.s1 = final_state; t.s1_mul = 1.f; state_strides(t.s1s, p, false);
  t.D = p->D; t.Dv = p->Dv; t.scale = p->scale;
  DeviceScope scope(p->device);
  if (scope.err != cudaSuccess) return sffft_note_cuda_error(scope.err);
  return run(p, 0, &prm, f, (char*)work, work_bytes, (cudaStream_t)stream);
}

int sffft_linear_attention_backward(const sffft_linear_attention_t* p, const sffft_linear_attention_grads_t* g,
                                    const void* q, const void* k, const void* v, const float* log_decay,
                                    const int* lengths, const float* initial_state, const void* dy,
                                    const float* dfinal_state, void* dq, void* dk, void* dv, float* dinitial_state,
                                    void* work, size_t work_bytes, void* stream) {
  int rc = common_checks(p, log_decay);
  if (rc) return rc;
  if (!g || !std::isfinite(1.f / p->scale)) return SFFFT_ERR_INVALID_ARGUMENT;
  if (p->Dv > 256) return SFFFT_ERR_UNSUPPORTED;   // v takes the place of q in two of the three passes
  if (p->B == 0) return SFFFT_OK;
  if (p->L > 0 && (!q || !k || !v || !dy || !dq || !dk || !dv)) return SFFFT_ERR_INVALID_ARGUMENT;
  if (((uintptr_t)work & 255) != 0) return SFFFT_ERR_INVALID_ARGUMENT;
  if (!on_elements(io_size(p->io), {q, k, v, dy, dq, dk, dv}) ||
      !on_elements(4, {log_decay, lengths, initial_state, dfinal_state, dinitial_state}))
    return SFFFT_ERR_INVALID_ARGUMENT;
  if (dinitial_state && dinitial_state == dfinal_state) return SFFFT_ERR_INVALID_ARGUMENT;   // as forward
  if ((rc = la_tc_reported(p->device))) return rc;
  DeviceFacts f;
  if ((rc = start(p, &f))) return rc;
  LaParams prm = {};
  prm.ld = log_decay; prm.len = lengths;
  prm.ntask = 3; prm.B = p->B; prm.H = p->H; prm.L = p->L; prm.sms = f.sms;
  for (int i = 0; i < 3; i++) {
    prm.task[i].scale = p->scale;
    prm.task[i].s0_mul = prm.task[i].s1_mul = 1.f;
  }
  const int share = p->H / p->Hkv;
  // the workspace begins with the query heads' gradients, whose size does not depend on the kernel
  const Sizes whole = sizes(p, 1, 1);
  if (whole.total && (!work || work_bytes < whole.total)) return SFFFT_ERR_WORKSPACE;
  float *wk = (float*)work, *wv = (float*)((char*)work + whole.grad_k);
  LaTask& a = prm.task[0];   // dq
  a.q = dy; a.k = v; a.v = k; a.y = dq;
  copy3(a.qs, g->dy_stride); copy3(a.ks, p->v_stride); copy3(a.vs, p->k_stride); copy3(a.ys, g->dq_stride);
  a.qdiv = 1; a.kdiv = a.vdiv = share;
  a.s0 = initial_state; state_strides(a.s0s, p, true);
  a.D = p->Dv; a.Dv = p->D;
  LaTask& c = prm.task[1];   // dk
  c.q = v; c.k = dy; c.v = q;
  copy3(c.qs, p->v_stride); copy3(c.ks, g->dy_stride); copy3(c.vs, p->q_stride);
  c.qdiv = share; c.kdiv = c.vdiv = 1;
  c.s0 = dfinal_state; c.s0_mul = 1.f / p->scale; state_strides(c.s0s, p, true);
  c.D = p->Dv; c.Dv = p->D; c.rev = c.off = 1;
  LaTask& e = prm.task[2];   // dv and the start state's gradient
  e.q = k; e.k = q; e.v = dy;
  copy3(e.qs, p->k_stride); copy3(e.ks, p->q_stride); copy3(e.vs, g->dy_stride);
  e.qdiv = share; e.kdiv = e.vdiv = 1;
  e.s0 = dfinal_state; e.s0_mul = 1.f / p->scale; state_strides(e.s0s, p, false);
  e.s1 = dinitial_state; e.s1_mul = p->scale; e.s1_decay = 1; state_strides(e.s1s, p, false);
  e.D = p->D; e.Dv = p->Dv; e.rev = e.off = 1;
  if (share > 1) {   // a gradient for each query head in fp32, then their sum
    const long long hk[3] = {(long long)p->H * p->L * p->D, (long long)p->L * p->D, p->D};
    const long long hv[3] = {(long long)p->H * p->L * p->Dv, (long long)p->L * p->Dv, p->Dv};
    c.y = wk; c.y_f32 = 1; copy3(c.ys, hk);
    e.y = wv; e.y_f32 = 1; copy3(e.ys, hv);
  } else {
    c.y = dk; copy3(c.ys, g->dk_stride);
    e.y = dv; copy3(e.ys, g->dv_stride);
  }
  DeviceScope scope(p->device);
  if (scope.err != cudaSuccess) return sffft_note_cuda_error(scope.err);
  const bool bf = p->io == SFFFT_IO_BF16;
  const cudaStream_t st = (cudaStream_t)stream;
  if ((rc = run(p, 1, &prm, f, (char*)work + whole.total, work_bytes - whole.total, st))) return rc;
  cudaError_t ce = cudaSuccess;
  if (share > 1) {
    LaReduceParams r = {wk, dk, {}, p->B, p->Hkv, share, p->L, p->D};
    copy3(r.os, g->dk_stride);
    ce = bf ? reduce_t<__nv_bfloat16>(r, f.sms, st) : reduce_t<float>(r, f.sms, st);
    if (ce == cudaSuccess) {
      r.w = wv; r.out = dv; r.D = p->Dv;
      copy3(r.os, g->dv_stride);
      ce = bf ? reduce_t<__nv_bfloat16>(r, f.sms, st) : reduce_t<float>(r, f.sms, st);
    }
  }
  return ce == cudaSuccess ? SFFFT_OK : sffft_note_cuda_error(ce);
}

int sffft_linear_attention_check(int device) {
  if (device < 0) return SFFFT_ERR_INVALID_ARGUMENT;
  DeviceScope scope(device);
  if (scope.err != cudaSuccess) return sffft_note_cuda_error(scope.err);
  int status = 0;
  const cudaError_t ce = la_tc_status(device, &status);
  return ce == cudaSuccess ? status : sffft_note_cuda_error(ce);
}

int sffft_debug_linear_attention(int limit_us, int withhold) {
  if (limit_us < 0 || limit_us > 1000000 || withhold < LA_WITHHOLD_NONE || withhold > LA_WITHHOLD_OOUT || (withhold && !limit_us))
    return SFFFT_ERR_INVALID_ARGUMENT;
  t_wait_ns = limit_us ? 1000ull * (unsigned long long)limit_us : kLaWaitNs;
  t_withhold = withhold;
  return SFFFT_OK;
}

int sffft_linear_attention_step(const sffft_linear_attention_step_t* p, const void* q, const void* k, const void* v,
                                const float* log_decay, float* state, const int* slots, void* y, void* stream) {
  if (!p || p->B < 0 || p->H < 1 || p->Hkv < 1 || p->H % p->Hkv != 0 || p->D < 1 || p->Dv < 1 || p->pool < 0 ||
      (p->io != SFFFT_IO_FP32 && p->io != SFFFT_IO_BF16) || p->device < 0 || !std::isfinite(p->scale))
    return SFFFT_ERR_INVALID_ARGUMENT;
  if (!slots && p->pool < p->B) return SFFFT_ERR_INVALID_ARGUMENT;
  if (p->pool > 1 && p->state_stride < (long long)p->H * p->D * p->Dv) return SFFFT_ERR_INVALID_ARGUMENT;   // slots that overlap
  if ((long long)p->B * p->H > INT_MAX || (long long)p->D * p->Dv > INT_MAX || p->Dv > 32 * 65535) return SFFFT_ERR_UNSUPPORTED;
  if (p->B == 0) return SFFFT_OK;
  if (!q || !k || !v || !log_decay || (!state && p->pool > 0) || !y) return SFFFT_ERR_INVALID_ARGUMENT;
  if (!on_elements(io_size(p->io), {q, k, v, y}) || !on_elements(4, {log_decay, state, slots})) return SFFFT_ERR_INVALID_ARGUMENT;
  if (const int rc = la_tc_reported(p->device)) return rc;   // the states may come from the call that reported it
  DeviceFacts f;
  const cudaError_t fe = device_facts(p->device, &f);
  if (fe != cudaSuccess) return sffft_note_cuda_error(fe);
  if (!f.ok) return SFFFT_ERR_DEVICE;
  LaStepParams s = {q, k, v, y, state, slots, log_decay, {}, {}, {}, {}, p->state_stride,
                    p->B, p->H, p->H / p->Hkv, p->D, p->Dv, p->pool, p->scale};
  for (int i = 0; i < 2; i++) {
    s.qs[i] = p->q_stride[i]; s.ks[i] = p->k_stride[i]; s.vs[i] = p->v_stride[i]; s.ys[i] = p->y_stride[i];
  }
  DeviceScope scope(p->device);
  if (scope.err != cudaSuccess) return sffft_note_cuda_error(scope.err);
  const dim3 grid((unsigned)(p->B * p->H), (unsigned)((p->Dv + kStepCols - 1) / kStepCols));
  const bool vec = p->Dv % 4 == 0 && p->state_stride % 4 == 0 && ((uintptr_t)state & 15) == 0;
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t ce;
  if (p->io == SFFFT_IO_BF16)
    ce = vec ? launch(la_step_kernel<__nv_bfloat16, 4>, grid, kStepThreads, 0, st, s)
             : launch(la_step_kernel<__nv_bfloat16, 1>, grid, kStepThreads, 0, st, s);
  else
    ce = vec ? launch(la_step_kernel<float, 4>, grid, kStepThreads, 0, st, s)
             : launch(la_step_kernel<float, 1>, grid, kStepThreads, 0, st, s);
  return ce == cudaSuccess ? SFFFT_OK : sffft_note_cuda_error(ce);
}

}  // extern "C"
