/* sffft — B200 (sm_100a) fused causal long convolution, C ABI.
 *
 *   y[b,h,n] = sum_{m<=n} u[b,h,m] * k[h,n-m],   0 <= n < L
 *
 * Drop-in for the operator surface of sfFFT (github.com/solidsf-inc/sfFFT, src/sffft.cu and
 * src/selection.h).  All device buffers are caller-owned; calls are asynchronous on the given CUDA
 * stream (cudaStream_t passed as void*, NULL = default stream); every call returns an int status
 * (SFFFT_OK = 0) and never exits the process.  Plans are immutable after creation and may be shared
 * by host threads.  There is no CPU fallback: without a B200-class device, plan creation fails.
 *
 * Layouts (identical to the reference):
 *   u, y : [B][H][L] contiguous, fp32 or bf16 (plan io), 16-byte aligned
 *   k    : [H][L] contiguous real filter, fp32 or bf16 (k_dtype)
 *   Kf   : [H][N] complex fp32 (float pairs), N = 2L, unnormalised DFT of the zero-padded filter in the
 *          plan's digit order: position p = k0*R1*R2 + k1*R2 + k2 holds frequency k0 + R0*k1 + R0*R1*k2
 *          (the layout permuteK writes, src/sffft.cu:283-288)
 */
#ifndef SFFFT_H_
#define SFFFT_H_

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SFFFT_OK 0
#define SFFFT_ERR_INVALID_ARGUMENT 1
#define SFFFT_ERR_UNSUPPORTED 2
#define SFFFT_ERR_CUDA 3
#define SFFFT_ERR_DEVICE 4
#define SFFFT_ERR_TIMEOUT 5
#define SFFFT_ERR_NO_MATCH 6
#define SFFFT_ERR_ALLOC 7
#define SFFFT_ERR_SCRATCH_LIMIT 8 /* problem too large for sffft_conv_noalloc's fixed scratch */
#define SFFFT_ERR_WORKSPACE 9     /* the call needs a larger workspace (composite plans, linear attention, norms' backward) */

#define SFFFT_IO_FP32 0
#define SFFFT_IO_BF16 1
#define SFFFT_ACC_FP32 0
#define SFFFT_ACC_FP16 1
#define SFFFT_KERNEL_LEGACY 0 /* DFT matrices computed inside every CTA (reference --kernel legacy) */
#define SFFFT_KERNEL_CACHED 1 /* DFT matrices copied from a precomputed table (reference --kernel cached) */

typedef struct sffft_plan* sffft_plan_t;

typedef struct {
  int L, N, stages, R0, R1, R2;
  int pairs_per_cta;   /* G: pairs of batch elements (same channel) per CTA */
  int warps, threads, smem_bytes, tmem_cols, occupancy;
  int io, acc, kernel_mode, device;
  int blocks;          /* 1, or the block count of a composite plan (L = blocks * block length) */
  char config[96];     /* catalog name, e.g. "64x32/w4", or "2x[32x32x32/w8]" for a composite plan */
} sffft_plan_info_t;

/* Creates a plan for length L (power of two).  config: catalog name ("64x32/w4") for L = 128..16384, or
 * NULL / "" for the built-in B200 default for L.  Replaces the compile-time choice of fftconv<Plan<R0,R1,R2>,
 * W,TIO,TAcc,CACHED> plus its cudaFuncSetAttribute / occupancy setup (src/sffft.cu:243-245, 385-388).
 * Composite plans (no reference counterpart; the reference stops at L = 8192 and lists multi-pass plans
 * as missing, README.md:175): config "<P>x[<catalog name>]" runs L = P * Lb (P = 2..16) as a partitioned
 * convolution on the catalog plan of length Lb (a forward transform per input block, then per output block
 * the sum of block spectra times filter-segment spectra and one inverse transform; block plans: the default
 * plan of each length up to 16384, and 16x16/w4), and the default for L = 32768 .. 262144 is
 * "<L/16384>x[<default for 16384>]".  For a composite plan Kf holds the P filter-segment spectra
 * [P][H][2 Lb] (the same H * 2L complex values), filter layouts other than causal are unsupported, and the
 * convolution needs a caller-owned workspace (sffft_conv_workspace_bytes): passed to sffft_conv_ws, or
 * attached to the plan for sffft_conv with sffft_plan_set_workspace. */
int sffft_plan_create(sffft_plan_t* plan, int L, int io, int acc, const char* config, int kernel_mode, int device);
int sffft_plan_destroy(sffft_plan_t plan);
int sffft_plan_info(sffft_plan_t plan, sffft_plan_info_t* info);

/* Filter spectrum in the plan's digit order, once per channel (untimed prep).  k_dtype: SFFFT_IO_FP32 or
 * SFFFT_IO_BF16.  Replaces host zero-padding + cufftExecC2C + permuteK (src/sffft.cu:342-344, 365,
 * 283-288, 384). */
int sffft_filter_spectrum(sffft_plan_t plan, const void* k, int k_dtype, int H, void* Kf, void* stream);

/* Filter layouts: which convolution sffft_conv computes, for n in [0, L), with the spectrum of k. */
#define SFFFT_FILTER_CAUSAL 0    /* k [H][L]:    y[n] = sum_{m<=n} u[m] k[n-m]           (the reference's) */
#define SFFFT_FILTER_TWO_SIDED 1 /* k [H][2L-1]: y[n] = sum_{m<L} u[m] k[L-1+n-m]        (non-causal) */
#define SFFFT_FILTER_CIRCULAR 2  /* k [H][L]:    y[n] = sum_{m<L} u[m] k[(n-m) mod L]    (period L) */

/* sffft_filter_spectrum for a filter in the given layout (SFFFT_FILTER_*); the fused convolution is the
 * same kernel for all three.  The reference exposes only the causal form; non-causal and circular
 * convolution are listed as not yet exposed (README.md:174). */
int sffft_filter_spectrum_ex(sffft_plan_t plan, const void* k, int k_dtype, int layout, int H, void* Kf,
                             void* stream);

/* Standalone real FFTs of length N = 2L (the plan's N) over B rows, on the same digit decomposition as
 * the filter-spectrum prep (fp32 CUDA cores, exact twiddles); no reference counterpart (README.md:174
 * lists standalone forward and inverse FFTs as not yet exposed).
 *   sffft_rfft:  x [B][N] real (x_dtype SFFFT_IO_FP32 or SFFFT_IO_BF16) -> X [B][N/2+1] complex fp32,
 *                X[f] = sum_n x[n] exp(-2 pi i f n / N)              (numpy.fft.rfft)
 *   sffft_irfft: X [B][N/2+1] complex fp32 -> x [B][N] fp32,
 *                x[n] = (1/N) sum_f Xfull[f] exp(+2 pi i f n / N)    (numpy.fft.irfft; the imaginary
 *                parts of X[0] and X[N/2] are ignored)
 * work: caller-owned device buffer of sffft_fft_workspace_bytes(plan, B) bytes, 8-byte aligned. */
int sffft_fft_workspace_bytes(sffft_plan_t plan, int B, size_t* bytes);
int sffft_rfft(sffft_plan_t plan, const void* x, int x_dtype, int B, void* X, void* work, void* stream);
int sffft_irfft(sffft_plan_t plan, const void* X, int B, float* x, void* work, void* stream);

/* The fused convolution: one kernel launch per call (four for a composite plan, which needs a workspace: see
 * sffft_conv_ws).  Replaces the launch fftconv<P,W,TIO,TAcc,CACHED><<<B*H, 32*W, smem>>>(u, Kf, tw, dft, y, B, H)
 * (src/sffft.cu:243-280, 389-390); the unused twiddle table and the DFT table are owned by the plan.  The kernel
 * is a programmatic dependent of the stream's previous kernel: its prologue may overlap that kernel's end, and it
 * reads u and Kf only after that kernel has completed. */
int sffft_conv(sffft_plan_t plan, const void* u, const void* Kf, void* y, int B, int H, void* stream);

/* Workspace of a composite plan's convolution of a B x H batch, in bytes: the forward spectra of every
 * input block (ceil(B/2) * H * L * 16 bytes) and the row energies; 0 for single-pass plans. */
int sffft_conv_workspace_bytes(sffft_plan_t plan, int B, int H, size_t* bytes);
/* sffft_conv with a caller-owned device workspace (256-byte aligned, at least sffft_conv_workspace_bytes;
 * NULL for single-pass plans).  A composite call is four launches in stream order (row energies, forward
 * transforms, spectrum sums, inverse transforms); the workspace must not be shared by calls that can overlap.
 * Returns SFFFT_ERR_WORKSPACE when a composite plan gets no workspace or too small a one. */
int sffft_conv_ws(sffft_plan_t plan, const void* u, const void* Kf, void* y, int B, int H, void* work,
                  size_t work_bytes, void* stream);
/* Attaches a caller-owned workspace (256-byte aligned; NULL detaches) that sffft_conv uses for composite
 * plans, which otherwise return SFFFT_ERR_WORKSPACE.  The plan does not free it. */
int sffft_plan_set_workspace(sffft_plan_t plan, void* work, size_t bytes);

/* Waits for the plan's device and returns (and clears) the device-side status word: SFFFT_OK, or
 * SFFFT_ERR_TIMEOUT when a kernel barrier wait gave up.  No reference counterpart (the reference has no
 * device-side error reporting; its CUDA errors surface through cudaGetLastError, src/sffft.cu:324). */
int sffft_plan_check(sffft_plan_t plan);

/* Plan catalog (the candidates of the reference's RUN rows, src/sffft.cu:506-513, plus L = 16384). */
int sffft_catalog_count(void);
int sffft_catalog_entry(int index, int* L, char* name, int name_cap);
int sffft_default_config(int L, char* name, int name_cap);

/* Empirical selector with the semantics of select_candidate / relative_l2 (src/selection.h:13-29):
 * returns the index of the fastest candidate with finite ms > 0 and finite 0 <= rel_err <= max_error
 * whose io matches (or io == "any"); ties go to the lower error; -1 when nothing qualifies or the budget
 * or io is invalid. */
typedef struct {
  const char* method;
  const char* io;
  const char* config;
  double ms, rel_err;
} sffft_candidate_t;
int sffft_select_candidate(const sffft_candidate_t* candidates, int count, double max_error, const char* io);
double sffft_relative_l2(double squared_error, double squared_reference);

/* Channel sharding across devices: shard g of G owns channels [h0, h1) (contiguous, sizes differ by at
 * most one).  No reference counterpart (the reference is single-GPU, src/sffft.cu:490). */
int sffft_shard_range(int H, int shards, int shard, int* h0, int* h1);

const char* sffft_status_string(int status);
int sffft_last_cuda_error(void);

/* cuFFT baseline pipeline on the same device (src/sffft.cu:289-305, 365-371): spectrum from the
 * fp32 filter k_dev [H][L]; run(full=1) = pad -> R2C -> multiply -> C2R -> slice, run(full=0) = core
 * only (reuses the padded input of the previous full run). */
typedef struct sffft_baseline* sffft_baseline_t;
int sffft_baseline_create(sffft_baseline_t* bl, int L, int B, int H, const float* k_dev, int device);
int sffft_baseline_run(sffft_baseline_t bl, const float* u, float* y, int full, void* stream);
int sffft_baseline_destroy(sffft_baseline_t bl);

/* Debug: one tcgen05.mma through the fused kernel's layout writers and descriptors (no reference
 * counterpart).  a_kind: 0 = MN-major 128-B swizzle, 32/64/128 = K-major row pitch; A: 128x16 halves,
 * B: n x 16 halves (B[n][k]), D: 128 x n raw TMEM words. */
int sffft_debug_umma_probe(int a_kind, int a_slice, int b_pitch, int b_slice, int n, int acc16,
                           const unsigned short* A, const unsigned short* B, unsigned int* D);

/* Allocation-free convolution, for callers that cannot allocate device memory while they run (an
 * inference-engine plugin whose execute step must not allocate, a process whose device memory is all
 * reserved by another allocator).  No counterpart in the reference.  The caller passes u [B][H][L], the
 * real filter k [H][L] (k_dtype fp32 or bf16) and y; the filter spectrum and a status word live in a fixed
 * array inside the library (16 MiB of spectrum, i.e. H * 2L * 8 bytes <= 16 MiB, plus 256 bytes), which
 * every GPU that loads the library holds until the process exits.  Larger problems return
 * SFFFT_ERR_SCRATCH_LIMIT without launching anything.  Uses the built-in plan for L with DFT matrices built
 * in-kernel; results equal sffft_filter_spectrum + sffft_conv on a "legacy" plan.  The first call on a
 * device sets up that device (looks up the array's device address, sets kernel attributes); make it
 * before any stream capture.  All calls on a device share the array, so calls whose work overlaps on the
 * GPU race.  sync != 0 waits for the stream and returns the kernel's device-side status; with sync == 0 the
 * call returns once the work is queued and a device-side error of that call (a barrier timeout) is not
 * reported, since the next call on the device clears the status word before it launches. */
int sffft_conv_noalloc(int L, int io, int acc, const void* u, const void* k, int k_dtype, void* y, int B, int H,
                       void* stream, int sync);

/* Host-buffer pipeline (no reference counterpart: the reference keeps u and y on the device and times the
 * kernel alone).  sffft_pipe_create sizes device staging for a B x H batch cut into about `chunks` chunks
 * (0 = 4) of whole batch-row pairs (contiguous, one copy each way), or of pairs and channel ranges when B/2
 * is smaller than `chunks`, and creates one stream per stage (upload, convolution, download) with three
 * staging slots; sffft_conv_host then computes y_host = causal_conv(u_host, k) for host buffers u_host,
 * y_host [B][H][L] (the plan's I/O type; pinned for overlap) and the device spectrum Kf [H][N]: chunk i goes
 * through slot i % 3, so uploads, kernels and downloads of different chunks overlap.  Ordered after earlier work on `stream`; later work on
 * `stream` waits for it.  Calls on one pipe must not overlap. */
typedef struct sffft_pipe* sffft_pipe_t;
int sffft_pipe_create(sffft_pipe_t* pipe, sffft_plan_t plan, int B, int H, int chunks);
int sffft_conv_host(sffft_pipe_t pipe, const void* u_host, const void* Kf, void* y_host, void* stream);
int sffft_pipe_destroy(sffft_pipe_t pipe);

/* Channel-sharded convolution over several devices.  No reference counterpart: the reference runs on device 0
 * only (src/sffft.cu:490).  Shard g of G owns channels [h0, h1) = sffft_shard_range(H, G, g) and runs on the
 * device of plans[g] (plans share L and the I/O type; one device may hold several shards).
 *   sffft_conv_multi: device-resident shards, asynchronous: u[g], y[g] are [B][h1 - h0][L] and Kf[g] is
 *     [h1 - h0][N] on plans[g]'s device; one sffft_conv per shard on streams[g] (NULL: default streams).
 *   sffft_multi_pipe_create / sffft_conv_host_multi: one [B][H][L] batch in host memory (pinned for overlap);
 *     every device uploads its channel slice, convolves it with its spectrum rows Kf[g] ([h1 - h0][N] on that
 *     device) and downloads its slice of y_host, all devices concurrently, each through a host pipe of its own
 *     (as sffft_pipe_create with `chunks`) driven by a host thread of its own (started by
 *     sffft_multi_pipe_create, joined by sffft_multi_pipe_destroy); the call returns when every device has
 *     finished, with the first error or device-side status (SFFFT_ERR_TIMEOUT) of any shard.  Composite plans
 *     in sffft_conv_multi use the workspace attached to each plan (sffft_plan_set_workspace); the pipes
 *     allocate their own. */
int sffft_conv_multi(const sffft_plan_t* plans, int G, const void* const* u, const void* const* Kf, void* const* y,
                     int B, int H, void* const* streams);
typedef struct sffft_multi* sffft_multi_t;
int sffft_multi_pipe_create(sffft_multi_t* multi, const sffft_plan_t* plans, int G, int B, int H, int chunks);
int sffft_conv_host_multi(sffft_multi_t multi, const void* u_host, const void* const* Kf, void* y_host);
int sffft_multi_pipe_destroy(sffft_multi_t multi);

/* ---------------------------------------------------------------------------------------------------------------
 * Linear attention with a decay for each head (no reference counterpart): the causal mixer whose filter depends on
 * the data.  For a head with decay lambda = exp(log_decay), lambda in [0, 1], and state S [D][Dv] in fp32,
 *
 *   S_n = lambda S_{n-1} + k_n v_n^T,     y_n = scale * S_n^T q_n,        n = 1 .. length
 *
 * i.e. y_n = scale * (sum_{m<=n} lambda^(n-m) (q_n . k_m) v_m + lambda^n S_0^T q_n): with D = Dv = 1 and q = k = 1 it
 * is sffft_conv with the filter lambda^n.
 *
 *   q, y [B][H][L][D or Dv], k [B][Hkv][L][D], v [B][Hkv][L][Dv]   of type io; a position's D (Dv) values are
 *        contiguous, the other axes have the element strides {row, head, position} of the descriptor, so that
 *        [B][L][H][D] buffers and parts of a fused projection work as they are.  Query head h uses key and value head
 *        h / (H / Hkv).
 *   log_decay [H] fp32, <= 0 (-inf: no memory); a constant of the model, not trained.
 *   lengths [B] int32 on the device, or NULL: tokens of each row (clamped to 0 .. L).  What q, k and v hold behind a
 *        row's last token is not used, not even where it is NaN; y there is set to zero.
 *   initial_state, final_state [B][H][D][Dv] fp32 contiguous; NULL: zero, not wanted.
 *
 * D up to 256 and Dv up to 4096 (backward: 256), any L; other sizes return SFFFT_ERR_UNSUPPORTED.  A value of q, k or v
 * that is not finite may reach all outputs of its row and head.  Outputs must not overlap inputs (final_state ==
 * initial_state is refused).  `work`: caller-owned
 * device memory of sffft_linear_attention_workspace_bytes (256-byte aligned), not shared by calls that can overlap.
 * Calls run on `device` in stream order and can be captured in graphs; the caller's current device is left as it was.
 * Results do not depend on scheduling: no atomics.
 *
 * Accuracy.  Outputs are rounded once to their type, and states are sums in fp32, whichever kernel runs (on the tensor cores
 * of terms held to 2^-24, or to 2^-16 where final_state is NULL and only y uses them).  bf16 with D up to 128, D and Dv
 * multiples of 8 and rows on 16 bytes (strides multiples of 8) runs on the tensor cores, where one factor of each of y's
 * products (the weighted q . k, and the state) is rounded to bf16 first: y, dq, dk and dv are off by up to 2^-8 of their
 * terms' magnitudes beside their own rounding (relative L2 2.35e-3, the rounding alone 1.66e-3).  Other sizes, addresses
 * and strides, and fp32, run on the CUDA cores in fp32 throughout; the same bf16 values in a view that lies between have
 * the smaller error.  To have it everywhere, pass fp32 tensors. */
typedef struct {
  int B, H, Hkv, L, D, Dv;
  int io;                 /* SFFFT_IO_* of q, k, v, y and their gradients */
  int device;
  float scale;            /* finite, not 0 (backward: 1 / scale finite) */
  long long q_stride[3], k_stride[3], v_stride[3], y_stride[3];
} sffft_linear_attention_t;
int sffft_linear_attention_workspace_bytes(const sffft_linear_attention_t* p, int backward, size_t* bytes);
int sffft_linear_attention(const sffft_linear_attention_t* p, const void* q, const void* k, const void* v,
                           const float* log_decay, const int* lengths, const float* initial_state, void* y,
                           float* final_state, void* work, size_t work_bytes, void* stream);

/* Gradients of q, k, v and the initial state from those of y and of the final state (dfinal_state NULL: zero;
 * dinitial_state NULL: not wanted).  dk and dv of a shared head are summed over its query heads in fp32.  Gradients
 * behind a row's last token are zero.  y_stride of the descriptor is not used. */
typedef struct {
  long long dy_stride[3], dq_stride[3], dk_stride[3], dv_stride[3];
} sffft_linear_attention_grads_t;
int sffft_linear_attention_backward(const sffft_linear_attention_t* p, const sffft_linear_attention_grads_t* g,
                                    const void* q, const void* k, const void* v, const float* log_decay,
                                    const int* lengths, const float* initial_state, const void* dy,
                                    const float* dfinal_state, void* dq, void* dk, void* dv, float* dinitial_state,
                                    void* work, size_t work_bytes, void* stream);

/* Waits for the device and returns (and clears) what its linear attention kernels reported: SFFFT_OK, or
 * SFFFT_ERR_TIMEOUT when a barrier wait of one gave up, and its outputs are not valid.  Until then every later call on the
 * device (the single-token one too, whose states may come from there) returns the same status and does nothing,
 * without waiting: as soon as the kernel that reported it has ended. */
int sffft_linear_attention_check(int device);

/* One token for each of B rows: S <- lambda S + k v^T in place, y = scale * S^T q.  The states lie in a pool of slots
 * of [H][D][Dv] fp32, state_stride elements apart (at least H D Dv where there is more than one); row b uses slot
 * slots[b] (int32, device), or slot b where slots is NULL.  A row whose slot is not in [0, pool) is padding: it gets y = 0
 * and no state changes.  The same holds for a row that names a slot which an earlier row of the call names.  Strides are
 * {row, head}. */
typedef struct {
  int B, H, Hkv, D, Dv, pool;
  int io, device;
  float scale;
  long long q_stride[2], k_stride[2], v_stride[2], y_stride[2], state_stride;
} sffft_linear_attention_step_t;
int sffft_linear_attention_step(const sffft_linear_attention_step_t* p, const void* q, const void* k, const void* v,
                                const float* log_decay, float* state, const int* slots, void* y, void* stream);

/* ---------------------------------------------------------------------------------------------------------------
 * The joint between two blocks (no reference counterpart): the norm behind a block, its gate and residual scale, the
 * residual stream, and the norm before the next block, in one pass.  On each row of `channels` values
 *
 *   a = y * rstd_g(y) * post_weight     (a = y where post_weight is NULL, whatever groups; rstd over each of `groups` runs of channels)
 *   h = x + scale * act(gate) * a       (without x where it is NULL; without the gate where gate is NULL)
 *   n = h * rstd(h) * weight            (not computed where weight is NULL)
 *
 * with rstd(z) = (mean(z^2) + eps)^(-1/2).  y NULL: h = x (not written), n alone.
 *
 *   inner = 0: x, y and gate are rows of contiguous channels, x_stride (..) elements apart; h and n are contiguous
 *   inner > 0: all tensors are [rows / inner][channels][inner] contiguous, the layout of sffft_conv's u and y
 *   gate: SFFFT_GATE_NONE, _FULL (shaped like y) or _CHANNEL ([channels])
 *   y, gate and n are of type io, x and h of type res_io (io, or fp32 beside bf16), the weights [channels] of weight_io
 *   rstd_post [rows][groups] and rstd [rows] fp32: written for the backward pass, NULL: not wanted
 *
 * All arithmetic is in fp32; an act of a gate in bf16 is off by up to 2^-18 of its value, of one in fp32 by 2^-20.
 * Up to 8192 channels (and 256 groups with inner > 0).  h may be x's and n y's own buffer where the strides agree and inner = 0. */
#define SFFFT_GATE_NONE 0
#define SFFFT_GATE_FULL 1
#define SFFFT_GATE_CHANNEL 2
#define SFFFT_ACT_NONE 0
#define SFFFT_ACT_SILU 1
#define SFFFT_ACT_SIGMOID 2
typedef struct {
  long long rows;
  int channels, inner, groups;
  int io, res_io, weight_io;
  int gate, act;
  float scale, eps;
  int device;
  long long x_stride, y_stride, gate_stride;
} sffft_block_norm_t;
int sffft_block_norm(const sffft_block_norm_t* p, const void* x, const void* y, const void* gate, const void* post_weight,
                     const void* weight, void* h, void* n, float* rstd_post, float* rstd, void* stream);
/* Gradients from dh (NULL: zero) and dn, which are laid out like h and n, and the forward pass's rstd_post and rstd.
 * dx, dy and a full dgate are contiguous in the same layout; dpost_weight, dweight and a channel's dgate are summed
 * over the rows in fp32 and a fixed order.  work: sffft_block_norm_workspace_bytes, 256-byte aligned. */
int sffft_block_norm_workspace_bytes(const sffft_block_norm_t* p, size_t* bytes);
int sffft_block_norm_backward(const sffft_block_norm_t* p, const void* x, const void* y, const void* gate,
                              const void* post_weight, const void* weight, const float* rstd_post, const float* rstd,
                              const void* dh, const void* dn, void* dx, void* dy, void* dgate, void* dpost_weight,
                              void* dweight, void* work, size_t work_bytes, void* stream);

/* Debug: a kernel waits on a barrier that nothing arrives at, using the same bounded wait as the fused
 * kernel; returns SFFFT_ERR_TIMEOUT after about limit_us microseconds (1..1e6) with the context intact.
 * No reference counterpart (the reference has no device-side timeouts). */
int sffft_debug_wait_timeout(int limit_us);

/* Debug: sffft_conv with every barrier wait of the fused kernel limited to limit_us microseconds (1..1e6) and
 * one arrival withheld (the first warp of the team that converts the first group skips its arrival on the
 * "operand ready" barrier), so the stage-0 MMAs are never issued and the bounded waits run out: the kernel's
 * roles see the abort flag, wait for their MMAs in flight, free TMEM and return; sffft_plan_check then reports
 * SFFFT_ERR_TIMEOUT and the context stays usable.  Exercises the fused kernel's failure path without a fault.
 * No reference counterpart (the reference fails fast on host errors only, src/sffft.cu:22-23). */
int sffft_debug_conv_timeout(sffft_plan_t plan, const void* u, const void* Kf, void* y, int B, int H, int limit_us,
                             void* stream);

/* Debug: from here on, linear attention on the tensor cores that this host thread launches limits each barrier wait to
 * limit_us microseconds (1..1e6; 0: the default, 2 s), and with `withhold` one thread leaves out an arrival: 1: that the last
 * chunk's keys are ready for the state's product, 2: that the outputs are scaled, 3: that they are staged.  The
 * waits that need it run out, every role sees the flag, lets its copies and products in flight end, frees TMEM and
 * returns; sffft_linear_attention_check then reports SFFFT_ERR_TIMEOUT and the context stays usable.  (0, 0) puts the
 * defaults back. */
int sffft_debug_linear_attention(int limit_us, int withhold);

#ifdef __cplusplus
}
#endif
#endif /* SFFFT_H_ */
