// Linear attention with a decay for each head on the tensor cores (bf16 operands, fp32 accumulators in TMEM).
//
// A CTA takes one head of one row and a segment of its positions, 128 at a time (the MMA's M).  With S the state before the
// chunk, P = (Q K^T) * lambda^(i-j) for j <= i, m tokens in the chunk:
//   O = lambda^(i+1) (Q S) + P V              S <- lambda^m S + X^T V,    X_j = lambda^(m-1-j) k_j
// Four products a chunk; each of 128 x 128 x 128 takes 512 cycles of an SM, while the chunk's 128 KB of q, k, v and y
// (head size 128) take about 5700 cycles of its share of the memory's bandwidth: the kernel is bound by memory as long as
// what lies between the products is overlapped with the loads.  So the work is split over warps:
//   4 warps     P: TMEM -> scale, mask, round -> TMEM;  O: lambda^(i+1) scale between the two products;  output
//   4 per 64 columns of v   X: shared memory -> TMEM, transposed;  S in fp32 registers -> bf16 in shared memory
//   1 thread    TMA loads, two stages of (Q, K, V), and the store of O, which is staged where V was
//   1 thread    tcgen05.mma
//
// Rounding.  y takes P and S rounded to bf16, one rounding beside its own, as any tensor-core product must.  The state is an
// fp32 result that lives for the whole row, so X is held as a sum of bf16 values: two (2^-17) where only y uses the state,
// three (2^-25) where it is an output; and S is added up in registers, not in the accumulator, whose additions truncate.
// With a head size of 64 the first two parts fill the 128 lanes together (lanes 0-63 and 64-127), and so does S, whose two
// halves the product with Q adds up.
//
// Time reversal (gradients of k and v): chunks from the last to the first, P and X mirrored.
//
// Every wait is bounded: after kWaitLimit ns the waiting role raises the CTA's flag, all roles leave, and the device's
// status word says so.
#include <cuda.h>
#include <cuda_bf16.h>

#include "../../include/sffft.h"
#include "launch.h"
#include "linattn.h"
#include "plan.h"
#include "tc.cuh"

namespace sffft {

static __device__ int g_la_status;

namespace {

constexpr int kTok = 128;   // positions in a chunk
constexpr uint64_t kWaitLimit = 2000000000ull;
constexpr uint32_t kBlk = kTok * 128;   // bytes of a 64-column tile of 128 positions: 128-byte rows, 128-byte swizzle

struct __align__(64) LaTcParams {
  CUtensorMap map[kLaMaxTasks][4];   // q, k, v, y
  LaParams p;
  int blocks;   // chunks in a segment
};

template <int DQ, int DV>
struct Shape {
  static constexpr int NB = DV / 64;                    // state warpgroups
  static constexpr int threads = 128 + 128 * NB + 64;
  static constexpr bool alias = DQ == 64 && DV == 64;   // two CTAs on an SM: 256 columns each, O lies in S's upper half
  static constexpr uint32_t q_bytes = DQ / 64 * kBlk, v_bytes = DV / 64 * kBlk, stage = 2 * q_bytes + v_bytes;
  static constexpr uint32_t off_s = 2 * stage, off_tab = off_s + NB * kBlk, off_bar = off_tab + 544;
  static constexpr uint32_t smem = off_bar + 16 * 8 + 16;
  static constexpr uint32_t cols = alias ? 256 : 512;
  // TMEM columns: products Q K^T (P over their first half), O, increment of S, X
  static constexpr uint32_t c_p = 0, c_o = alias ? 64 : 128, c_kv = alias ? 128 : 128 + DV, c_x = c_kv + DV;
  static constexpr uint32_t x_cols = DQ == 64 ? 64 : 128;
  static_assert(c_x + x_cols <= cols, "TMEM");
};

enum { B_FULL0, B_FULL1, B_S, B_P, B_O1, B_OS, B_O, B_OOUT, B_OFREE, B_X, B_KV, B_X2, B_KV2, B_ST, B_FIN, B_COUNT };

__host__ __device__ constexpr uint32_t idesc_bf16(int N, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t t, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(t));
}
__device__ __forceinline__ void tmem_st32(uint32_t t, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(t),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t t, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(t),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* m, int x, int t, int h, int b, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
                   dst),
               "l"(m), "r"(x), "r"(t), "r"(h), "r"(b), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* m, uint32_t src, int x, int t, int h, int b) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(m), "r"(x), "r"(t),
               "r"(h), "r"(b), "r"(src)
               : "memory");
}

__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ float lds32(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// {lo, hi} halves of a word
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float lo_f(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float hi_f(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// among the 128 threads of a state warpgroup
__device__ __forceinline__ void wg_sync(int wg) {
  if (wg == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
  else asm volatile("bar.sync 2, 128;" ::: "memory");
}

struct Waiter {
  uint64_t* bars;
  volatile int* stop;
  // false: the CTA gives up
  __device__ __forceinline__ bool operator()(int b, uint32_t parity) const {
    if (mbar_try_wait(bars + b, parity)) return true;
    return slow(b, parity);
  }
  __device__ __noinline__ bool slow(int b, uint32_t parity) const {
    const uint64_t t0 = global_ns();
    while (!mbar_try_wait(bars + b, parity)) {
      if (*stop) return false;
      if (global_ns() - t0 > kWaitLimit) {
        *stop = 1;
        atomicExch(&g_la_status, SFFFT_ERR_TIMEOUT);
        return false;
      }
    }
    return true;
  }
};

// The same for a warp whose lanes go on together (tcgen05.ld and st are collective).
struct WarpWaiter {
  Waiter w;
  __device__ __forceinline__ bool operator()(int b, uint32_t parity) const { return __all_sync(~0u, w(b, parity)); }
};

// Tokens of a row of n, in processing order, before chunk `c` of nblk.
__device__ __forceinline__ int tokens_before(int c, int n, int nblk, bool rev) {
  if (c >= nblk) return n;
  return rev ? (c == 0 ? 0 : n - (nblk - c) * kTok) : c * kTok;
}

template <int DQ, int DV, bool LOCAL>
__global__ void __launch_bounds__(Shape<DQ, DV>::threads, Shape<DQ, DV>::alias ? 2 : 1)
    la_tc_kernel(const __grid_constant__ LaTcParams prm) {
  using SH = Shape<DQ, DV>;
  constexpr int NB = SH::NB;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t sm = smem_u32(smem);
  float* tab = (float*)(smem + SH::off_tab);   // lambda^0 .. lambda^128
  uint64_t* bars = (uint64_t*)(smem + SH::off_bar);
  volatile int* stop = (volatile int*)(smem + SH::off_bar + 16 * 8);
  uint32_t* slot = (uint32_t*)(smem + SH::off_bar + 16 * 8 + 4);

  const LaParams& lp = prm.p;
  const int ti = blockIdx.x % lp.ntask, u = blockIdx.x / lp.ntask;
  const LaTask& tk = lp.task[ti];
  const int g = u % lp.G, bh = u / lp.G, b = bh / lp.H, h = bh % lp.H;
  if (LOCAL && g == lp.G - 1) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int n = lp.L;
  if (lp.len) n = min(max(lp.len[b], 0), lp.L);
  const bool rev = tk.rev;
  const int nblk = (n + kTok - 1) / kTok;
  const int c0 = min(g * prm.blocks, nblk), c1 = min(c0 + prm.blocks, nblk), nc = c1 - c0;
  const int before = tokens_before(c0, n, nblk, rev);
  const LaDecay dec(lp.ld[h]);
  const bool three = tk.s1 != nullptr;   // the state is an output: three parts of X
  // the first chunk meets no state
  const bool fresh = !LOCAL && before == 0 && !tk.s0;

  if (threadIdx.x == 0) {
    const int count[B_COUNT] = {1, 1, 1, 128, 1, 128, 1, 128, 128, 128 * NB, 1, 128 * NB, 1, 128 * NB, 1};
    for (int i = 0; i < B_COUNT; i++) mbar_init(bars + i, (uint32_t)count[i]);
    *stop = (sm & 1023u) != 0;   // swizzled tiles need the alignment that the launch gives
    if (*stop) atomicExch(&g_la_status, SFFFT_ERR_DEVICE);
    fence_mbar_init();
  }
  for (int i = threadIdx.x; i <= kTok; i += blockDim.x) tab[i] = dec.pow(i);
  if (warp == SH::threads / 32 - 1) {
    tmem_alloc(slot, SH::cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = *slot;
  const Waiter wait{bars, stop};
  const WarpWaiter wwait{wait};
  const uint32_t tabs = sm + SH::off_tab;

  auto tokens = [&](int c) {   // of chunk c0 + c
    const int blk = rev ? nblk - 1 - (c0 + c) : c0 + c;
    return min(kTok, n - blk * kTok);
  };

  if (*stop) {
    // nothing has been started
  } else if (warp == SH::threads / 32 - 2) {
    // ---- loads, stores ----
    if (lane == 0) {
      const CUtensorMap* m = prm.map[ti];
      const int hq = h / tk.qdiv, hk = h / tk.kdiv, hv = h / tk.vdiv;
      auto load = [&](int c) {
        const uint32_t st = sm + (uint32_t)(c & 1) * SH::stage;
        uint64_t* bar = bars + B_FULL0 + (c & 1);
        const int t = (rev ? nblk - 1 - (c0 + c) : c0 + c) * kTok;
        mbar_expect(bar, (LOCAL ? SH::q_bytes : 2 * SH::q_bytes) + SH::v_bytes);
        for (int i = 0; i < DQ / 64; i++) tma_load(st + SH::q_bytes + i * kBlk, m + 1, i * 64, t, hk, b, bar);
        if (!LOCAL)
          for (int i = 0; i < DQ / 64; i++) tma_load(st + i * kBlk, m + 0, i * 64, t, hq, b, bar);
        for (int i = 0; i < NB; i++) tma_load(st + 2 * SH::q_bytes + i * kBlk, m + 2, i * 64, t, hv, b, bar);
      };
      int issued = 0;
      for (; issued < min(nc, 2); issued++) load(issued);
      for (int c = 0; c < nc; c++) {
        if (!wait(LOCAL ? B_ST : B_OOUT, c & 1)) break;
        if (!LOCAL && !tk.y_f32) {
          const uint32_t st = sm + (uint32_t)(c & 1) * SH::stage + 2 * SH::q_bytes;
          const int t = (rev ? nblk - 1 - (c0 + c) : c0 + c) * kTok;
          for (int i = 0; i < NB; i++) tma_store(m + 3, st + i * kBlk, i * 64, t, h, b);
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          if (c + 2 < nc || c + 1 == nc) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        }
        if (c + 2 < nc) load(issued++);
      }
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
      if (*stop)   // copies in flight end before the block does
        for (int c = max(0, issued - 2); c < issued; c++) mbar_wait_bounded(bars + B_FULL0 + (c & 1), (c >> 1) & 1, kWaitLimit);
    }
  } else if (warp == SH::threads / 32 - 1) {
    // ---- products ----
    if (lane == 0) {
      constexpr uint32_t id_s = idesc_bf16(128, false), id_v = idesc_bf16(DV, true);
      for (int c = 0; c < nc; c++) {
        const uint32_t ph = c & 1, st = sm + (uint32_t)(c & 1) * SH::stage;
        if (!wait(B_FULL0 + (c & 1), (c >> 1) & 1)) break;
        const uint64_t qd = make_sdesc(st, 16, 1024, LT_SW128), kd = make_sdesc(st + SH::q_bytes, 16, 1024, LT_SW128);
        const uint64_t vd = make_sdesc(st + 2 * SH::q_bytes, kBlk, 1024, LT_SW128);
        const uint64_t sd = make_sdesc(sm + SH::off_s, kBlk, 1024, LT_SW128);
        auto at = [](uint64_t d, uint32_t bytes) { return d + (uint64_t)(bytes >> 4); };
        auto kstep = [](int k) { return (uint32_t)(k >> 2) * kBlk + (uint32_t)(k & 3) * 32; };   // K-major: 16 values on
        if (!LOCAL) {
          if (SH::alias && c > 0 && !wait(B_OFREE, ph ^ 1)) break;
          tc_fence_after();
          for (int k = 0; k < DQ / 16; k++) mma_f16_ss(tm + SH::c_p, at(qd, kstep(k)), at(kd, kstep(k)), id_s, k > 0);
          mma_commit(bars + B_S);
        }
        if (!wait(B_X, ph)) break;
        tc_fence_after();
        for (int part = 0; part < DQ / 64; part++)
          for (int k = 0; k < 8; k++)
            mma_ts(tm + SH::c_kv, tm + SH::c_x + part * 64 + k * 8, at(vd, k * 2048), id_v, (part | k) > 0);
        mma_commit(bars + B_KV);
        if (!LOCAL) {
          if (!wait(B_ST, ph)) break;
          if (!SH::alias && c > 0 && !wait(B_OFREE, ph ^ 1)) break;
          if (SH::alias && !wait(B_P, ph)) break;
          tc_fence_after();
          if (!(fresh && c == 0))
            for (int k = 0; k < 8; k++)
              mma_f16_ss(tm + SH::c_o, at(qd, kstep(DQ == 64 ? k & 3 : k)), at(sd, k * 2048), id_v, k > 0);
          mma_commit(bars + B_O1);
        }
        if (three) {
          if (!wait(B_X2, ph)) break;
          tc_fence_after();
          for (int k = 0; k < 8; k++) mma_ts(tm + SH::c_kv, tm + SH::c_x + k * 8, at(vd, k * 2048), id_v, 1);
          mma_commit(bars + B_KV2);
        }
        if (!LOCAL) {
          if (!SH::alias && !wait(B_P, ph)) break;
          if (!wait(B_OS, ph)) break;
          tc_fence_after();
          for (int k = 0; k < 8; k++)
            mma_ts(tm + SH::c_o, tm + SH::c_p + k * 8, at(vd, k * 2048), id_v, k > 0 || !(fresh && c == 0));
          mma_commit(bars + B_O);
        }
      }
      if (*stop) {   // products in flight end before TMEM is given back
        mma_commit(bars + B_FIN);
        mbar_wait_bounded(bars + B_FIN, 0, kWaitLimit);
      }
    }
  } else if (warp < 4) {
    // ---- P and O ----
    if (!LOCAL) {
      const int i = threadIdx.x;   // position in the chunk
      const uint32_t tl = tm + ((uint32_t)(warp * 32) << 16);
      for (int c = 0; c < nc; c++) {
        const uint32_t ph = c & 1;
        const int m = tokens(c), blk = rev ? nblk - 1 - (c0 + c) : c0 + c;
        const int off = tk.off && before == 0 && c == 0;
        if (!wwait(B_S, ph)) break;
        tc_fence_after();
#pragma unroll 1
        for (int jb = 0; jb < 4; jb++) {
          uint32_t r[32], o[16];
          const bool some = rev ? jb >= warp : jb <= warp;
          if (some) {
            tmem_ld32(tl + SH::c_p + jb * 32, r);
            // lambda^|i-j|: within the diagonal block the other side is masked, and its table index held in range
            const int d0 = rev ? jb * 32 - i : i - jb * 32;   // |i - j| = d0 -+ jj
            tmem_wait_ld();
            if (rev) {
#pragma unroll
              for (int jj = 0; jj < 32; jj++) {
                const int d = d0 + jj;
                const float w = lds32(tabs + 4u * (uint32_t)max(d, 0));
                const float x = __uint_as_float(r[jj]) * w;
                r[jj] = __float_as_uint(d >= 0 && jb * 32 + jj < m ? x : 0.f);
              }
            } else {
#pragma unroll
              for (int jj = 0; jj < 32; jj++) {
                const int d = d0 - jj;
                const float w = lds32(tabs + 4u * (uint32_t)max(d, 0));
                const float x = __uint_as_float(r[jj]) * w;
                r[jj] = __float_as_uint(d >= 0 && i < m ? x : 0.f);
              }
            }
#pragma unroll
            for (int e = 0; e < 16; e++) o[e] = pack_bf16(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]));
          } else {
#pragma unroll
            for (int e = 0; e < 16; e++) o[e] = 0;
          }
          tmem_st16(tl + SH::c_p + jb * 16, o);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bars + B_P);
        // lambda^(i+1) Q S (in reverse lambda^(m-i)); rows behind the last token hold whatever q holds: zero
        if (!wwait(B_O1, ph)) break;
        tc_fence_after();
        if (!(fresh && c == 0)) {
          const float w = i < m ? tab[(rev ? m - i : i + 1) - off] : 0.f;
#pragma unroll 1
          for (int q = 0; q < DV / 32; q++) {
            uint32_t r[32];
            tmem_ld32(tl + SH::c_o + q * 32, r);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; e++) r[e] = __float_as_uint(i < m ? __uint_as_float(r[e]) * w : 0.f);
            tmem_st32(tl + SH::c_o + q * 32, r);
          }
          tmem_wait_st();
        }
        tc_fence_before();
        mbar_arrive(bars + B_OS);
        if (!wwait(B_O, ph)) break;
        tc_fence_after();
        const uint32_t out = sm + (uint32_t)(c & 1) * SH::stage + 2 * SH::q_bytes + (uint32_t)i * 128;
#pragma unroll 1
        for (int q = 0; q < DV / 32; q++) {
          uint32_t r[32];
          tmem_ld32(tl + SH::c_o + q * 32, r);
          tmem_wait_ld();
          if (!tk.y_f32) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
              uint32_t w[4];
#pragma unroll
              for (int x = 0; x < 4; x++)
                w[x] = pack_bf16(tk.scale * __uint_as_float(r[8 * e + 2 * x]), tk.scale * __uint_as_float(r[8 * e + 2 * x + 1]));
              const uint32_t chunk = (uint32_t)((q & 1) * 4 + e);
              sts128(out + (uint32_t)(q >> 1) * kBlk + ((chunk ^ (uint32_t)(i & 7)) << 4), w[0], w[1], w[2], w[3]);
            }
          } else if (blk * kTok + i < lp.L) {
            float* y = (float*)tk.y + b * tk.ys[0] + h * tk.ys[1] + (long long)(blk * kTok + i) * tk.ys[2] + q * 32;
#pragma unroll
            for (int e = 0; e < 32; e += 4)   // Dv is a multiple of 8
              if (q * 32 + e < tk.Dv)
                *(float4*)(y + e) = make_float4(tk.scale * __uint_as_float(r[e]), tk.scale * __uint_as_float(r[e + 1]),
                                                tk.scale * __uint_as_float(r[e + 2]), tk.scale * __uint_as_float(r[e + 3]));
          }
        }
        fence_async_smem();
        tc_fence_before();
        mbar_arrive(bars + B_OFREE);
        mbar_arrive(bars + B_OOUT);
      }
      // chunks of the segment behind the row's last token
      const int z0 = max(g * prm.blocks, nblk) * kTok, z1 = min((long long)(g + 1) * prm.blocks * kTok, (long long)lp.L);
      const int pieces = tk.Dv / 8;
      for (long long e = i; e < (long long)(z1 - z0) * pieces; e += 128) {
        const long long at = b * tk.ys[0] + h * tk.ys[1] + (z0 + e / pieces) * tk.ys[2] + (e % pieces) * 8;
        if (tk.y_f32) {
          *(float4*)((float*)tk.y + at) = make_float4(0.f, 0.f, 0.f, 0.f);
          *(float4*)((float*)tk.y + at + 4) = make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
          *(uint4*)((__nv_bfloat16*)tk.y + at) = make_uint4(0, 0, 0, 0);
        }
      }
    }
  } else {
    // ---- X and S ----
    const int wg = (warp - 4) >> 2, t = threadIdx.x & 127;
    const uint32_t tl = tm + ((uint32_t)((warp & 3) * 32) << 16);
    const int d = DQ == 64 ? t & 63 : t;        // the thread's row of the state
    const bool main_part = DQ == 128 || t < 64; // lanes 64-127 hold the second part where the head size is 64
    float s[64];
#pragma unroll
    for (int e = 0; e < 64; e++) s[e] = 0.f;
    if (!LOCAL && main_part && d < tk.D) {
      const float* loc = tk.loc + ((long long)bh * lp.G * tk.D + d) * tk.Dv + wg * 64;
      const long long step = (long long)tk.D * tk.Dv;
      for (int gg = 0; gg < g; gg++) {
        const int a = tokens_before(min(gg * prm.blocks, nblk), n, nblk, rev);
        const int z = tokens_before(min((gg + 1) * prm.blocks, nblk), n, nblk, rev);
        if (z == a) break;
        const float w = dec.pow(z - a);
#pragma unroll
        for (int e = 0; e < 64; e++)
          if (wg * 64 + e < tk.Dv) s[e] = fmaf(w, s[e], loc[gg * step + e]);
      }
      if (tk.s0) {
        const float w = dec.pow(before - (tk.off && before > 0));
        const float* s0 = tk.s0 + b * tk.s0s[0] + h * tk.s0s[1] + d * tk.s0s[2] + (long long)(wg * 64) * tk.s0s[3];
#pragma unroll
        for (int e = 0; e < 64; e++)
          if (wg * 64 + e < tk.Dv) s[e] = fmaf(w, s0[e * tk.s0s[3]] * tk.s0_mul, s[e]);
      }
    }
    const uint32_t srow = sm + SH::off_s + (uint32_t)wg * kBlk + (uint32_t)t * 128;
    auto publish = [&]() {   // S in bf16 for the next chunk's product
#pragma unroll
      for (int e = 0; e < 8; e++)
        sts128(srow + (((uint32_t)e ^ (uint32_t)(t & 7)) << 4), pack_bf16(s[8 * e], s[8 * e + 1]), pack_bf16(s[8 * e + 2], s[8 * e + 3]),
               pack_bf16(s[8 * e + 4], s[8 * e + 5]), pack_bf16(s[8 * e + 6], s[8 * e + 7]));
      fence_async_smem();
    };
    if (!LOCAL) {
      publish();
      mbar_arrive(bars + B_ST);
    }
    // lambda^128 as a sum of two floats: its rounding would come back with every chunk
    const float whole = dec.pow(kTok), whole_lo = dec.pow_rest(kTok, whole);
    constexpr int TPW = kTok / NB;   // positions whose X this warpgroup makes
    const uint32_t kcol = (uint32_t)(d >> 6) * kBlk + (uint32_t)(d & 7) * 2;
    const uint32_t cd = (uint32_t)(d & 63) >> 3;
    for (int c = 0; c < nc; c++) {
      const uint32_t ph = c & 1, st = sm + (uint32_t)(c & 1) * SH::stage;
      const int m = tokens(c);
      const int off = tk.off && before == 0 && c == 0;
      if (!wwait(B_FULL0 + (c & 1), (c >> 1) & 1)) break;
      if (m < kTok && n < lp.L) {   // v behind the last token may hold anything, and 0 * NaN is NaN
        const uint32_t v = st + 2 * SH::q_bytes + (uint32_t)wg * kBlk;
        for (int e = t; e < (kTok - m) * 8; e += 128) sts128(v + (uint32_t)m * 128 + (uint32_t)e * 16, 0, 0, 0, 0);
        fence_async_smem();
      }
      // the first two parts of X, or the third
      auto make_x = [&](bool third) {
        const uint32_t kb = st + SH::q_bytes + kcol;
#pragma unroll 1
        for (int j0 = wg * TPW; j0 < (wg + 1) * TPW; j0 += 32) {
          uint32_t a[16], z[16];
#pragma unroll
          for (int e = 0; e < 16; e++) {
            float x[2];
#pragma unroll
            for (int q = 0; q < 2; q++) {
              const int jj = 2 * e + q, j = j0 + jj;
              const uint32_t raw = lds16(kb + (uint32_t)j0 * 128 + (uint32_t)jj * 128 + ((cd ^ (uint32_t)(jj & 7)) << 4));
              const float w = lds32(tabs + 4u * (uint32_t)(rev ? j : max(m - 1 - j, 0)));
              const float y = __uint_as_float(raw << 16) * w;
              x[q] = j < m ? y : 0.f;
            }
            const uint32_t p1 = pack_bf16(x[0], x[1]);
            const float r0 = x[0] - lo_f(p1), r1 = x[1] - hi_f(p1);
            const uint32_t p2 = pack_bf16(r0, r1);
            if (third) {
              a[e] = main_part ? pack_bf16(r0 - lo_f(p2), r1 - hi_f(p2)) : 0u;
            } else if (DQ == 64) {
              a[e] = t < 64 ? p1 : p2;
            } else {
              a[e] = p1;
              z[e] = p2;
            }
          }
          tmem_st16(tl + SH::c_x + j0 / 2, a);
          if (DQ == 128 && !third) tmem_st16(tl + SH::c_x + 64 + j0 / 2, z);
        }
        tmem_wait_st();
        tc_fence_before();
      };
      make_x(false);
      mbar_arrive(bars + B_X);
      if (!wwait(B_KV, ph)) break;
      if (three) {
        tc_fence_after();
        make_x(true);
        mbar_arrive(bars + B_X2);
        if (!wwait(B_KV2, ph)) break;
      }
      if (!LOCAL && !wwait(B_O1, ph)) break;   // the product with the old S has been taken
      tc_fence_after();
      float w = whole, w_lo = whole_lo;
      if (m - off < kTok) w = tab[m - off], w_lo = 0.f;
#pragma unroll
      for (int q = 0; q < 4; q++) {
        uint32_t r[16];
        tmem_ld16(tl + SH::c_kv + wg * 64 + q * 16, r);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; e++) {
          float& x = s[q * 16 + e];
          x = fmaf(w, x, fmaf(w_lo, x, __uint_as_float(r[e])));
        }
      }
      tc_fence_before();
      if (!LOCAL) publish();
      mbar_arrive(bars + B_ST);
    }
    // the state that the segment leaves (after a wait that gave up: whatever it is, but every thread comes by)
    if (LOCAL || (tk.s1 && g == lp.G - 1)) {
      if constexpr (DQ == 64) {   // add the two parts; S's shared memory is free: nothing reads it any more
        wg_sync(wg);
        float* x = (float*)(smem + SH::off_s + wg * kBlk);
        if (t >= 64) {
#pragma unroll
          for (int e = 0; e < 64; e++) x[e * 64 + d] = s[e];
        }
        wg_sync(wg);
        if (t < 64) {
#pragma unroll
          for (int e = 0; e < 64; e++) s[e] += x[e * 64 + d];
        }
      }
      if (main_part && d < tk.D) {
        if (LOCAL) {
          float* out = tk.loc + (((long long)bh * lp.G + g) * tk.D + d) * tk.Dv + wg * 64;
#pragma unroll
          for (int e = 0; e < 64; e++)
            if (wg * 64 + e < tk.Dv) out[e] = s[e];
        } else {
          const float w = tk.s1_mul * (tk.s1_decay && n > 0 ? tab[1] : 1.f);
          float* out = tk.s1 + b * tk.s1s[0] + h * tk.s1s[1] + d * tk.s1s[2] + (long long)(wg * 64) * tk.s1s[3];
#pragma unroll
          for (int e = 0; e < 64; e++)
            if (wg * 64 + e < tk.Dv) out[e * tk.s1s[3]] = w * s[e];
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == SH::threads / 32 - 1) tmem_dealloc(tm, SH::cols);
}

// ---------------------------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (EncodeFn)p;
  }();
  return fn;
}

// What a tensor map of [B][H][L][D] bf16 needs: 16-byte aligned rows, and strides of their own.
bool mappable(const void* p, const long long (&s)[3], int B, int H, int L, int D) {
  if (((uintptr_t)p & 15) != 0 || D % 8 != 0 || D > 128) return false;
  const int n[3] = {B, H, L};
  for (int i = 0; i < 3; i++)
    if (n[i] > 1 && (s[i] <= 0 || s[i] % 8 != 0 || s[i] >= (1ll << 38))) return false;
  return true;
}

bool make_map(CUtensorMap* m, const void* p, const long long (&s)[3], int B, int H, int L, int D) {
  const cuuint64_t dim[4] = {(cuuint64_t)D, (cuuint64_t)L, (cuuint64_t)H, (cuuint64_t)B};
  auto bytes = [](int n, long long st) { return (cuuint64_t)(n > 1 ? st * 2 : 256); };   // an axis of one has no stride
  const cuuint64_t str[3] = {bytes(L, s[2]), bytes(H, s[1]), bytes(B, s[0])};
  const cuuint32_t box[4] = {64, kTok, 1, 1}, one[4] = {1, 1, 1, 1};
  return encode_fn()(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(p), dim, str, box, one,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DQ, int DV>
cudaError_t launch_shape(const LaTcParams& prm, cudaStream_t st) {
  using SH = Shape<DQ, DV>;
  const dim3 grid((unsigned)(prm.p.B * prm.p.H * prm.p.G * prm.p.ntask));
  if (prm.p.G > 1) {
    const cudaError_t ce = launch(la_tc_kernel<DQ, DV, true>, grid, SH::threads, (int)SH::smem, st, prm);
    if (ce != cudaSuccess) return ce;
  }
  return launch(la_tc_kernel<DQ, DV, false>, grid, SH::threads, (int)SH::smem, st, prm);
}

}  // namespace

bool la_tc_takes(const LaParams& p) {
  if (p.L < 1 || !encode_fn()) return false;
  for (int i = 0; i < p.ntask; i++) {
    const LaTask& t = p.task[i];
    if (!mappable(t.q, t.qs, p.B, p.H / t.qdiv, p.L, t.D) || !mappable(t.k, t.ks, p.B, p.H / t.kdiv, p.L, t.D) ||
        !mappable(t.v, t.vs, p.B, p.H / t.vdiv, p.L, t.Dv) || t.Dv % 8 != 0)
      return false;
    if (!mappable(t.y, t.ys, p.B, p.H, p.L, t.Dv)) return false;
  }
  return true;
}

cudaError_t launch_la_tc(const LaParams& p, cudaStream_t st) {
  // tasks of one tile shape go into one launch
  bool done[kLaMaxTasks] = {};
  for (int i = 0; i < p.ntask; i++) {
    if (done[i]) continue;
    LaTcParams prm = {};
    prm.p = p;
    prm.p.ntask = 0;
    prm.blocks = p.seg / kTok;
    const bool q2 = p.task[i].D > 64, v2 = p.task[i].Dv > 64;
    for (int j = i; j < p.ntask; j++) {
      const LaTask& t = p.task[j];
      if (done[j] || (t.D > 64) != q2 || (t.Dv > 64) != v2) continue;
      done[j] = true;
      const int k = prm.p.ntask++;
      prm.p.task[k] = t;
      if (!make_map(&prm.map[k][0], t.q, t.qs, p.B, p.H / t.qdiv, p.L, t.D) ||
          !make_map(&prm.map[k][1], t.k, t.ks, p.B, p.H / t.kdiv, p.L, t.D) ||
          !make_map(&prm.map[k][2], t.v, t.vs, p.B, p.H / t.vdiv, p.L, t.Dv) ||
          (!t.y_f32 && !make_map(&prm.map[k][3], t.y, t.ys, p.B, p.H, p.L, t.Dv)))
        return cudaErrorInvalidValue;
    }
    const cudaError_t ce = q2 ? (v2 ? launch_shape<128, 128>(prm, st) : launch_shape<128, 64>(prm, st))
                              : (v2 ? launch_shape<64, 128>(prm, st) : launch_shape<64, 64>(prm, st));
    if (ce != cudaSuccess) return ce;
  }
  return cudaSuccess;
}

cudaError_t la_tc_status(int* status) {
  void* p = nullptr;
  cudaError_t ce = cudaGetSymbolAddress(&p, g_la_status);
  const int zero = 0;
  if (ce == cudaSuccess) ce = cudaDeviceSynchronize();
  if (ce == cudaSuccess) ce = cudaMemcpy(status, p, sizeof(int), cudaMemcpyDeviceToHost);
  if (ce == cudaSuccess && *status) ce = cudaMemcpy(p, &zero, sizeof(int), cudaMemcpyHostToDevice);
  return ce;
}

}  // namespace sffft
