// Linear attention with a decay for each head: the problem as its kernels see it.
//
//   S_n = lambda S_{n-1} + k_n v_n^T,   y_n = scale * q_n^T S_n          (S_0 given or zero)
//
// The backward pass is the same recurrence on other operands, so one description ("task") serves all of it:
//   dq_n = scale * dy_n^T (S_n)^T          forward in time,  (q, k, v) <- (dy, v, k), start S_0^T
//   dk_n = scale * v_n^T R_n^T             backward in time, (q, k, v) <- (v, dy, q), start dS_L^T / scale
//   dv_n = scale * k_n^T R_n               backward in time, (q, k, v) <- (k, q, dy), start dS_L / scale
// with R_n = lambda R_{n+1} + q_n dy_n^T, R_{L+1} = dS_L / (scale * lambda), and dS_0 = scale * lambda * R_1.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace sffft {

struct LaTask {
  const void *q, *k, *v;
  void* y;
  long long qs[3], ks[3], vs[3], ys[3];   // element strides: row, head, position; a head's values are contiguous
  int qdiv, kdiv, vdiv;                   // head h reads head h / div of the tensor
  const float* s0;                        // start state (may be null), element (b, h, d, e) at s0s
  long long s0s[4];
  float s0_mul;
  float* s1;                              // end state (may be null)
  long long s1s[4];
  float s1_mul;
  int s1_decay;                           // the end state takes one more factor lambda (where there is a token)
  float* loc;                             // G > 1: state that each segment alone leaves, [B*H][G][D Dv] in a kernel's own order
  int D, Dv;
  int rev;                                // tokens are taken from the last one to the first
  int off;                                // the first token takes the start state as it is, without a factor lambda
  int y_f32;                              // y is fp32 whatever the type of q, k, v
  float scale;
};

constexpr int kLaMaxTasks = 3;

struct LaParams {
  LaTask task[kLaMaxTasks];
  const float* ld;   // natural logarithm of lambda, [H]
  const int* len;    // tokens of each row (null: L)
  int ntask, B, H, L;
  int G, seg;        // segments that the positions are cut into, and positions in each
  int sms;
  unsigned long long wait_ns;   // tensor cores: the limit of a wait
  int* status;                  // and where one that runs out is reported
  int withhold;                 // test hook of sffft_debug_linear_attention: an arrival that one thread leaves out
};

// X of a segment's last chunk; the scaling of O; O's staging.
enum { LA_WITHHOLD_NONE = 0, LA_WITHHOLD_X = 1, LA_WITHHOLD_OS = 2, LA_WITHHOLD_OOUT = 3 };
constexpr unsigned long long kLaWaitNs = 2000000000ull;

// lambda^n from log2(lambda) held as the sum hi + lo of two floats: hi * n is split exactly, so that the error is
// that of one exp2f, not of |hi * n| roundings.
struct LaDecay {
  float hi, lo;
  __device__ __forceinline__ explicit LaDecay(float ld) {
    const double l2 = (double)ld * 1.4426950408889634074;
    hi = (float)l2;
    lo = isinf(hi) ? 0.f : (float)(l2 - (double)hi);
  }
  __device__ __forceinline__ float pow(int n) const {
    if (n <= 0) return 1.f;
    const float x = (float)n, p = hi * x;
    if (p < -160.f) return 0.f;   // below the smallest float (also lambda = 0, where p is -inf)
    const float e = fmaf(hi, x, -p) + lo * x;
    return exp2f(p) * fmaf(e, 0.69314718f, 1.f);
  }
  // what the float `r` = pow(n) leaves of lambda^n
  __device__ __forceinline__ float pow_rest(int n, float r) const {
    if (n <= 0 || r == 0.f) return 0.f;
    return (float)(exp2(((double)hi + (double)lo) * n) - (double)r);
  }
};

// fp32 on CUDA cores: any type, strides and head sizes up to 256 (G > 1: three launches, else one).
cudaError_t launch_la_general(const LaParams& prm, bool bf16, cudaStream_t st);
// positions in a chunk of the general kernel for head sizes up to dmax
inline int la_general_chunk(int dmax) { return dmax > 128 ? 32 : 64; }

// bf16 on the tensor cores: D up to 128, D and Dv multiples of 8, 16-byte aligned rows (la_tc_takes), any length.
bool la_tc_takes(const LaParams& prm);
cudaError_t launch_la_tc(const LaParams& prm, cudaStream_t st);
// The status word of a device (where kernels write it), what has been reported there so far, and, having waited for the current
// device, the same with the word cleared.
constexpr int kLaMaxDevices = 64;
cudaError_t la_tc_word(int device, int** word);
int la_tc_reported(int device);
cudaError_t la_tc_status(int device, int* status);
constexpr int kLaTcChunk = 128;
int la_tc_tile(int D, int Dv);     // columns of v in a CTA
int la_tc_slices(int D, int Dv);   // CTAs over the columns of v

}  // namespace sffft
