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
  static constexpr int NB = DV / 64, NW = DV / 32;      // 64-column tiles of v; state warpgroups, 32 columns each
  static constexpr int threads = 128 + 128 * NW + 64;
  static constexpr bool alias = DQ == 64 && DV == 64;   // two CTAs on an SM: 256 columns each, O lies in S's upper half
  static constexpr bool out_q = DQ >= DV;               // O is staged where Q was, else where V was
  static constexpr uint32_t q_bytes = DQ / 64 * kBlk, v_bytes = NB * kBlk, stage = 2 * q_bytes + v_bytes;
  static constexpr uint32_t off_s = 2 * stage, off_tab = off_s + NB * kBlk, off_bar = off_tab + 4 * 160;
  static constexpr uint32_t smem = off_bar + 17 * 8 + 8;
  static constexpr uint32_t cols = alias ? 256 : 512;
  // TMEM columns: products Q K^T (P over their first half), O, increment of S, X
  static constexpr uint32_t c_p = 0, c_o = alias ? 64 : 128, c_kv = alias ? 128 : 128 + DV, c_x = c_kv + DV;
  static constexpr uint32_t x_cols = DQ == 64 ? 64 : 128;
  static_assert(c_x + x_cols <= cols, "TMEM");
};

// Barriers; each completes once a chunk (the first two pairs once for every other chunk).
enum {
  B_KV0, B_KV1, B_Q0, B_Q1,   // K and V, Q loaded
  B_S, B_P,                   // products ready; P ready
  B_O1, B_OS, B_O,            // Q S taken; scaled; O complete
  B_OOUT, B_OFREE,            // O staged; O's TMEM read
  B_X, B_INC, B_X2, B_INC2,   // X ready, its product taken; third part ready, its product taken
  B_ST,                       // S published (once more before the first chunk)
  B_FIN, B_COUNT
};
static_assert(B_COUNT <= 17, "barriers");

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

// Four 8 x 8 tiles of 16-bit values, transposed: lane l gives the address of row l % 8 of tile l / 8, and gets of each tile
// rows 2 (l % 4) and 2 (l % 4) + 1 of column l / 4, in one word.
__device__ __forceinline__ void ldsm_t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
// 16 lanes x 16 columns: word 2 i + k of lane l goes to TMEM lane 8 k + l / 4, column 4 i + l % 4.
__device__ __forceinline__ void tmem_st_16x128b_x4(uint32_t t, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(t), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
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
  switch (wg) {
    case 0: asm volatile("bar.sync 1, 128;" ::: "memory"); break;
    case 1: asm volatile("bar.sync 2, 128;" ::: "memory"); break;
    case 2: asm volatile("bar.sync 3, 128;" ::: "memory"); break;
    default: asm volatile("bar.sync 4, 128;" ::: "memory");
  }
}

// two floats in one instruction
struct F2 {
  float a, b;
};
__device__ __forceinline__ F2 mul2(F2 x, F2 y) {
  F2 r;
  asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmul.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "=f"(r.a), "=f"(r.b)
      : "f"(x.a), "f"(x.b), "f"(y.a), "f"(y.b));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 x, F2 y, F2 c) {
  F2 r;
  asm("{\n\t.reg .b64 p, q, m;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmov.b64 m, {%6, %7};\n\t"
      "fma.rn.f32x2 p, p, q, m;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "=f"(r.a), "=f"(r.b)
      : "f"(x.a), "f"(x.b), "f"(y.a), "f"(y.b), "f"(c.a), "f"(c.b));
  return r;
}
__device__ __forceinline__ F2 sub2(F2 x, F2 y) {   // x + (-y)
  F2 r;
  asm("{\n\t.reg .b64 p, q, m;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmov.b64 m, 0xbf800000bf800000;\n\t"
      "fma.rn.f32x2 p, q, m, p;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "=f"(r.a), "=f"(r.b)
      : "f"(x.a), "f"(x.b), "f"(y.a), "f"(y.b));
  return r;
}
// cut off behind bf16's eighth bit; the same packed
__device__ __forceinline__ F2 cut2(F2 x) {
  return {__uint_as_float(__float_as_uint(x.a) & 0xffff0000u), __uint_as_float(__float_as_uint(x.b) & 0xffff0000u)};
}
__device__ __forceinline__ uint32_t upper2(F2 x) { return __byte_perm(__float_as_uint(x.a), __float_as_uint(x.b), 0x7632); }

// Waits asleep for up to about a millisecond.
__device__ __forceinline__ bool try_wait_for(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P1;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 P1, [%1], %2, %3;\n\t"
      "selp.b32 %0, 1, 0, P1;\n\t}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
      : "memory");
  return ok != 0;
}

struct Waiter {
  uint64_t* bars;
  volatile int* stop;
  // false: the CTA gives up
  __device__ __forceinline__ bool operator()(int b, uint32_t parity) const {
    if (try_wait_for(bars + b, parity)) return true;
    return slow(b, parity);
  }
  __device__ __noinline__ bool slow(int b, uint32_t parity) const {
    const uint64_t t0 = global_ns();
    while (!try_wait_for(bars + b, parity)) {
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
  constexpr int NB = SH::NB, NW = SH::NW;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t sm = smem_u32(smem);
  // Powers of lambda in the order in which they are wanted, so that a loop over positions has fixed offsets.  Forward:
  // lambda^127 .. lambda^0 and 32 zeros; in reverse: 32 zeros, lambda^0 .. lambda^127.  The zeros are the masked side of a
  // diagonal block.
  float* tab = (float*)(smem + SH::off_tab);
  uint64_t* bars = (uint64_t*)(smem + SH::off_bar);
  volatile int* stop = (volatile int*)(smem + SH::off_bar + 17 * 8);
  uint32_t* slot = (uint32_t*)(smem + SH::off_bar + 17 * 8 + 4);

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
    for (int i = 0; i < B_COUNT; i++) {
      const bool a = i == B_P || i == B_OS || i == B_OOUT || i == B_OFREE, x = i == B_X || i == B_X2 || i == B_ST;
      mbar_init(bars + i, a ? 128u : x ? 128u * NW : 1u);
    }
    *stop = (sm & 1023u) != 0;   // swizzled tiles need the alignment that the launch gives
    if (*stop) atomicExch(&g_la_status, SFFFT_ERR_DEVICE);
    fence_mbar_init();
  }
  for (int i = threadIdx.x; i < 160; i += blockDim.x) {
    const int e = rev ? i - 32 : 127 - i;
    tab[i] = e >= 0 ? dec.pow(e) : 0.f;
  }
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
  auto power = [&](int e) { return tab[rev ? 32 + e : 127 - e]; };   // 0 <= e < 128

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
      auto load_kv = [&](int c) {
        const uint32_t st = sm + (uint32_t)(c & 1) * SH::stage;
        uint64_t* bar = bars + B_KV0 + (c & 1);
        const int t = (rev ? nblk - 1 - (c0 + c) : c0 + c) * kTok;
        mbar_expect(bar, SH::q_bytes + SH::v_bytes);
        for (int i = 0; i < DQ / 64; i++) tma_load(st + SH::q_bytes + i * kBlk, m + 1, i * 64, t, hk, b, bar);
        for (int i = 0; i < NB; i++) tma_load(st + 2 * SH::q_bytes + i * kBlk, m + 2, i * 64, t, hv, b, bar);
      };
      auto load_q = [&](int c) {
        const uint32_t st = sm + (uint32_t)(c & 1) * SH::stage;
        uint64_t* bar = bars + B_Q0 + (c & 1);
        const int t = (rev ? nblk - 1 - (c0 + c) : c0 + c) * kTok;
        mbar_expect(bar, SH::q_bytes);
        for (int i = 0; i < DQ / 64; i++) tma_load(st + i * kBlk, m + 0, i * 64, t, hq, b, bar);
      };
      int kv = 0, qs = 0;   // loads issued
      for (; kv < min(nc, 2); kv++) load_kv(kv);
      if (!LOCAL)
        for (; qs < min(nc, 2); qs++) load_q(qs);
      // a parity names the phase that follows a completed one: the first publication goes by before the loop
      const bool go = LOCAL || nc == 0 || wait(B_ST, 0);
      for (int c = 0; go && c < nc; c++) {
        // K and V have been read: by X and its products, and by P V
        if (!wait(B_ST, (LOCAL ? c : c + 1) & 1) || (!LOCAL && !wait(B_O, c & 1))) break;
        if ((LOCAL || SH::out_q) && c + 2 < nc) load_kv(kv++);
        if (LOCAL) continue;
        if (!wait(B_OOUT, c & 1)) break;
        if (!tk.y_f32) {
          const uint32_t st = sm + (uint32_t)(c & 1) * SH::stage + (SH::out_q ? 0 : 2 * SH::q_bytes);
          const int t = (rev ? nblk - 1 - (c0 + c) : c0 + c) * kTok;
          for (int i = 0; i < NB; i++) tma_store(m + 3, st + i * kBlk, i * 64, t, h, b);
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          if (c + 2 < nc) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        }
        if (c + 2 < nc) {
          if (!SH::out_q) load_kv(kv++);
          load_q(qs++);
        }
      }
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
      if (*stop) {   // copies in flight end before the block does
        for (int c = max(0, kv - 2); c < kv; c++) mbar_wait_bounded(bars + B_KV0 + (c & 1), (c >> 1) & 1, kWaitLimit);
        for (int c = max(0, qs - 2); c < qs; c++) mbar_wait_bounded(bars + B_Q0 + (c & 1), (c >> 1) & 1, kWaitLimit);
      }
    }
  } else if (warp == SH::threads / 32 - 1) {
    // ---- products ----
    if (lane == 0) {
      constexpr uint32_t id_s = idesc_bf16(128, false), id_v = idesc_bf16(DV, true);
      auto at = [](uint64_t d, uint32_t bytes) { return d + (uint64_t)(bytes >> 4); };
      auto kstep = [](int k) { return (uint32_t)(k >> 2) * kBlk + (uint32_t)(k & 3) * 32; };   // K-major: 16 values on
      const uint64_t sd = make_sdesc(sm + SH::off_s, kBlk, 1024, LT_SW128);
      bool ok = true;
      for (int c = 0; ok && c < nc; c++) {
        const uint32_t ph = c & 1, st = sm + (uint32_t)(c & 1) * SH::stage;
        if (!wait(B_KV0 + (c & 1), (c >> 1) & 1)) break;
        const uint64_t qd = make_sdesc(st, 16, 1024, LT_SW128), kd = make_sdesc(st + SH::q_bytes, 16, 1024, LT_SW128);
        const uint64_t vd = make_sdesc(st + 2 * SH::q_bytes, kBlk, 1024, LT_SW128);
        if (!LOCAL) {
          if (!wait(B_Q0 + (c & 1), (c >> 1) & 1)) break;
          if (SH::alias && c > 0 && !wait(B_OFREE, ph ^ 1)) break;
          tc_fence_after();
          for (int k = 0; k < DQ / 16; k++) mma_f16_ss(tm + SH::c_p, at(qd, kstep(k)), at(kd, kstep(k)), id_s, k > 0);
          mma_commit(bars + B_S);
        }
        // the chunk's other products in the order in which their operands become ready
        bool inc = false, inc2 = !three, qs = LOCAL, pv = LOCAL;
        const bool dirty = tokens(c) < kTok && n < lp.L;   // v is cleaned before X arrives
        uint64_t t0 = 0;
        uint32_t idle = 0;
        while (!(inc && inc2 && qs && pv)) {
          if (!qs && mbar_test_wait(bars + B_ST, ph) &&
              (SH::alias ? mbar_test_wait(bars + B_P, ph) : c == 0 || mbar_test_wait(bars + B_OFREE, ph ^ 1))) {
            tc_fence_after();
            if (!(fresh && c == 0))
              for (int k = 0; k < 8; k++)
                mma_f16_ss(tm + SH::c_o, at(qd, kstep(DQ == 64 ? k & 3 : k)), at(sd, k * 2048), id_v, k > 0);
            mma_commit(bars + B_O1);
            qs = true;
          } else if (qs && !pv && (inc || !dirty) && mbar_test_wait(bars + B_OS, ph) && mbar_test_wait(bars + B_P, ph)) {
            tc_fence_after();
            for (int k = 0; k < 8; k++)
              mma_ts(tm + SH::c_o, tm + SH::c_p + k * 8, at(vd, k * 2048), id_v, k > 0 || !(fresh && c == 0));
            mma_commit(bars + B_O);
            pv = true;
          } else if (!inc && mbar_test_wait(bars + B_X, ph)) {
            tc_fence_after();
            for (int part = 0; part < DQ / 64; part++)
              for (int k = 0; k < 8; k++)
                mma_ts(tm + SH::c_kv, tm + SH::c_x + part * 64 + k * 8, at(vd, k * 2048), id_v, (part | k) > 0);
            mma_commit(bars + B_INC);
            inc = true;
          } else if (inc && !inc2 && mbar_test_wait(bars + B_X2, ph)) {
            tc_fence_after();
            for (int k = 0; k < 8; k++) mma_ts(tm + SH::c_kv, tm + SH::c_x + k * 8, at(vd, k * 2048), id_v, 1);
            mma_commit(bars + B_INC2);
            inc2 = true;
          } else {
            if ((++idle & 63) == 0) {
              const uint64_t now = global_ns();
              if (!t0) t0 = now;
              if (now - t0 > kWaitLimit) {
                *stop = 1;
                atomicExch(&g_la_status, SFFFT_ERR_TIMEOUT);
              }
              if (*stop) {
                ok = false;
                break;
              }
            }
            __nanosleep(20);
          }
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
      const float whole = dec.pow(kTok);
      for (int c = 0; c < nc; c++) {
        const uint32_t ph = c & 1;
        const int m = tokens(c), blk = rev ? nblk - 1 - (c0 + c) : c0 + c;
        const int off = tk.off && before == 0 && c == 0;
        if (!wwait(B_S, ph)) break;
        tc_fence_after();
#pragma unroll 1
        for (int jb = 0; jb < 4; jb++) {
          uint32_t r[32], o[16];
          if (rev ? jb < warp : jb > warp) {   // a block on the masked side of the diagonal
#pragma unroll
            for (int e = 0; e < 16; e++) o[e] = 0;
          } else {
            tmem_ld32(tl + SH::c_p + jb * 32, r);
            const float* w = tab + (rev ? 32 + jb * 32 - i : 127 - i + jb * 32);
            tmem_wait_ld();
            if (m < kTok) {   // products with what k holds behind the last token may not be finite
#pragma unroll
              for (int e = 0; e < 32; e++)
                if (jb * 32 + e >= m) r[e] = 0;
            }
#pragma unroll
            for (int e = 0; e < 16; e++)
              o[e] = pack_bf16(__uint_as_float(r[2 * e]) * w[2 * e], __uint_as_float(r[2 * e + 1]) * w[2 * e + 1]);
          }
          tmem_st16(tl + SH::c_p + jb * 16, o);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bars + B_P);
        // lambda^(i+1) Q S, in reverse lambda^(m-i)
        if (!wwait(B_O1, ph)) break;
        tc_fence_after();
        if (!(fresh && c == 0)) {
          const int e = (rev ? m - i : i + 1) - off;
          const float w = e < 0 ? 0.f : e < kTok ? power(e) : whole;
#pragma unroll 1
          for (int q = 0; q < DV / 32; q++) {
            uint32_t r[32];
            tmem_ld32(tl + SH::c_o + q * 32, r);
            tmem_wait_ld();
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              const F2 z = mul2({__uint_as_float(r[x]), __uint_as_float(r[x + 1])}, {w, w});
              r[x] = __float_as_uint(z.a), r[x + 1] = __float_as_uint(z.b);
            }
            tmem_st32(tl + SH::c_o + q * 32, r);
          }
          tmem_wait_st();
        }
        tc_fence_before();
        mbar_arrive(bars + B_OS);
        if (!wwait(B_O, ph)) break;
        tc_fence_after();
        if (!SH::out_q && !wwait(three ? B_INC2 : B_INC, ph)) break;   // V's last reader
        const uint32_t out = sm + (uint32_t)(c & 1) * SH::stage + (SH::out_q ? 0 : 2 * SH::q_bytes) + (uint32_t)i * 128;
#pragma unroll 1
        for (int q = 0; q < DV / 32; q++) {
          uint32_t r[32];
          tmem_ld32(tl + SH::c_o + q * 32, r);
          tmem_wait_ld();
          // rows behind the last token: whatever q holds has come through
          if (m < kTok && i >= m) {
#pragma unroll
            for (int e = 0; e < 32; e++) r[e] = 0;
          }
          if (!tk.y_f32) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
              uint32_t w[4];
#pragma unroll
              for (int x = 0; x < 4; x++) {
                const F2 z = mul2({__uint_as_float(r[8 * e + 2 * x]), __uint_as_float(r[8 * e + 2 * x + 1])}, {tk.scale, tk.scale});
                w[x] = pack_bf16(z.a, z.b);
              }
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
    float s[32];                                // columns 32 wg ..
    const int col = wg * 32;
#pragma unroll
    for (int e = 0; e < 32; e++) s[e] = 0.f;
    if (!LOCAL && main_part && d < tk.D) {
      const float* loc = tk.loc + ((long long)bh * lp.G * tk.D + d) * tk.Dv + col;
      const long long step = (long long)tk.D * tk.Dv;
      for (int gg = 0; gg < g; gg++) {
        const int a = tokens_before(min(gg * prm.blocks, nblk), n, nblk, rev);
        const int z = tokens_before(min((gg + 1) * prm.blocks, nblk), n, nblk, rev);
        if (z == a) break;
        const float w = dec.pow(z - a);
#pragma unroll
        for (int e = 0; e < 32; e += 4)   // Dv is a multiple of 8
          if (col + e < tk.Dv) {
            const float4 x = *(const float4*)(loc + gg * step + e);
            s[e] = fmaf(w, s[e], x.x), s[e + 1] = fmaf(w, s[e + 1], x.y);
            s[e + 2] = fmaf(w, s[e + 2], x.z), s[e + 3] = fmaf(w, s[e + 3], x.w);
          }
      }
      if (tk.s0) {
        const float w = dec.pow(before - (tk.off && before > 0));
        const float* s0 = tk.s0 + b * tk.s0s[0] + h * tk.s0s[1] + d * tk.s0s[2] + (long long)col * tk.s0s[3];
#pragma unroll
        for (int e = 0; e < 32; e++)
          if (col + e < tk.Dv) s[e] = fmaf(w, s0[e * tk.s0s[3]] * tk.s0_mul, s[e]);
      }
    }
    const uint32_t srow = sm + SH::off_s + (uint32_t)(wg >> 1) * kBlk + (uint32_t)t * 128;
    auto publish = [&]() {   // S in bf16 for the next chunk's product
#pragma unroll
      for (int e = 0; e < 4; e++)
        sts128(srow + (((uint32_t)(4 * (wg & 1) + e) ^ (uint32_t)(t & 7)) << 4), pack_bf16(s[8 * e], s[8 * e + 1]),
               pack_bf16(s[8 * e + 2], s[8 * e + 3]), pack_bf16(s[8 * e + 4], s[8 * e + 5]), pack_bf16(s[8 * e + 6], s[8 * e + 7]));
      fence_async_smem();
    };
    // Zeroes v behind the last token of the chunk, where it may hold anything, and 0 * NaN is NaN.  Products with v wait
    // for X in such a chunk.
    auto clean_v = [&](int c) {
      const int m = tokens(c);
      if (m == kTok || n == lp.L) return;
      const uint32_t v = sm + (uint32_t)(c & 1) * SH::stage + 2 * SH::q_bytes + (uint32_t)(wg >> 1) * kBlk;
      for (int e = t; e < (kTok - m) * 4; e += 128)
        sts128(v + (uint32_t)(m + (e >> 2)) * 128 + (uint32_t)(4 * (wg & 1) + (e & 3)) * 16, 0, 0, 0, 0);
      fence_async_smem();
    };
    if (!LOCAL) {
      publish();
      mbar_arrive(bars + B_ST);
    }
    // lambda^128 as a sum of two floats: its rounding would come back with every chunk
    const float whole = dec.pow(kTok), whole_lo = dec.pow_rest(kTok, whole);
    constexpr int TPW = kTok / NW;   // positions whose X this warpgroup makes
    // Address of the lane's row of the K tiles of the warp's first 16 rows d and first 16 positions: tiles (d, position) are
    // (0-7, 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15); 16 rows d on is two 16-byte pieces on, under the swizzle.
    const int dw = DQ == 64 ? (warp & 1) * 32 : (warp & 3) * 32;
    const uint32_t kaddr = SH::q_bytes + (uint32_t)(dw >> 6) * kBlk + (uint32_t)(((lane >> 4) & 1) * 8 + (lane & 7)) * 128 +
                           ((((uint32_t)(dw & 63) >> 3) + ((uint32_t)(lane >> 3) & 1)) ^ (uint32_t)(lane & 7)) * 16;
    for (int c = 0; c < nc; c++) {
      const uint32_t ph = c & 1, st = sm + (uint32_t)(c & 1) * SH::stage;
      const int m = tokens(c);
      const int off = tk.off && before == 0 && c == 0;
      if (!wwait(B_KV0 + (c & 1), (c >> 1) & 1)) break;
      clean_v(c);
      // The first two parts of X, or the third.  Lanes of X are rows d of the state, its columns pairs of positions: K's
      // tiles come transposed from shared memory in the very arrangement that the 16 x 128b store takes.
      auto make_x = [&](bool third) {
#pragma unroll 1
        for (int j0 = wg * TPW; j0 < (wg + 1) * TPW; j0 += 32) {
          if (DQ == 64 && third && (j0 < kTok / 2) != (t < 64)) {   // each half of the lanes takes half the positions
            const uint32_t none[8] = {};
            tmem_st_16x128b_x4(tl + SH::c_x + j0 / 2, none);
            tmem_st_16x128b_x4(tl + (16u << 16) + SH::c_x + j0 / 2, none);
            continue;
          }
          float w[8];   // of positions j0 + 8 i + 2 (lane % 4) + {0, 1}
          const int wi = (rev ? 32 : kTok - m) + j0 + 2 * (lane & 3);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float* at = tab + min(wi + 8 * i, 158);   // behind the last token: the zeros
            w[2 * i] = at[0], w[2 * i + 1] = at[1];
          }
#pragma unroll 1
          for (int half = 0; half < 2; half++) {   // 16 rows each
            uint32_t r[8], z[8];
            const uint32_t addr = (kaddr + st + (uint32_t)j0 * 128) ^ (uint32_t)(32 * half);
            ldsm_t(addr, *(uint32_t(*)[4]) & r[0]);
            ldsm_t(addr + 16 * 128, *(uint32_t(*)[4]) & r[4]);
            if (m < kTok) {   // behind the last token k may hold anything
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const int j = j0 + 8 * i + 2 * (lane & 3);
                const uint32_t mask = (j < m ? 0xffffu : 0u) | (j + 1 < m ? 0xffff0000u : 0u);
                r[2 * i] &= mask;
                r[2 * i + 1] &= mask;
              }
            }
            const uint32_t to = tl + ((uint32_t)(16 * half) << 16) + SH::c_x + j0 / 2;
            // each part but the last is cut off, so that what is left is exact
            if (DQ == 64 && !third && t < 64) {
#pragma unroll
              for (int i = 0; i < 8; i++) r[i] = upper2(mul2({lo_f(r[i]), hi_f(r[i])}, {w[i & ~1], w[i | 1]}));
            } else if (!third) {
#pragma unroll
              for (int i = 0; i < 8; i++) {
                F2 x = mul2({lo_f(r[i]), hi_f(r[i])}, {w[i & ~1], w[i | 1]});
                if (DQ == 128) z[i] = upper2(x);
                x = sub2(x, cut2(x));
                r[i] = pack_bf16(x.a, x.b);
              }
              if (DQ == 128) tmem_st_16x128b_x4(to, z);
            } else {
#pragma unroll
              for (int i = 0; i < 8; i++) {
                F2 x = mul2({lo_f(r[i]), hi_f(r[i])}, {w[i & ~1], w[i | 1]});
                x = sub2(x, cut2(x));
                x = sub2(x, cut2(x));
                r[i] = pack_bf16(x.a, x.b);
              }
            }
            tmem_st_16x128b_x4(DQ == 128 && !third ? to + 64 : to, r);
          }
        }
        tmem_wait_st();
        tc_fence_before();
      };
      make_x(false);
      mbar_arrive(bars + B_X);
      if (!wwait(B_INC, ph)) break;
      tc_fence_after();
      if (three) {
        make_x(true);
        mbar_arrive(bars + B_X2);
        if (!wwait(B_INC2, ph)) break;
      }
      if (!LOCAL && !wwait(B_O1, ph)) break;   // the product with the old S has been taken
      tc_fence_after();
      float w = whole, w_lo = whole_lo;
      if (m - off < kTok) w = power(m - off), w_lo = 0.f;
#pragma unroll
      for (int q = 0; q < 2; q++) {
        uint32_t r[16];
        tmem_ld16(tl + SH::c_kv + col + q * 16, r);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          float &x = s[q * 16 + e], &y = s[q * 16 + e + 1];
          const F2 z = fma2({w, w}, {x, y}, fma2({w_lo, w_lo}, {x, y}, {__uint_as_float(r[e]), __uint_as_float(r[e + 1])}));
          x = z.a, y = z.b;
        }
      }
      tc_fence_before();
      if (!LOCAL && c + 1 < nc) publish();
      mbar_arrive(bars + B_ST);
    }
    // the state that the segment leaves (after a wait that gave up: whatever it is, but every thread comes by)
    if (LOCAL || (tk.s1 && g == lp.G - 1)) {
      if constexpr (DQ == 64) {   // add the two parts; S's shared memory is free: nothing reads it any more
        // every warpgroup is behind its last use of the tile
        asm volatile("bar.sync 5, %0;" ::"n"(128 * SH::NW) : "memory");
        float* x = (float*)(smem + SH::off_s + wg * (kBlk / 2));
        if (t >= 64) {
#pragma unroll
          for (int e = 0; e < 32; e++) x[e * 64 + d] = s[e];
        }
        wg_sync(wg);
        if (t < 64) {
#pragma unroll
          for (int e = 0; e < 32; e++) s[e] += x[e * 64 + d];
        }
      }
      if (main_part && d < tk.D) {
        if (LOCAL) {
          float* out = tk.loc + (((long long)bh * lp.G + g) * tk.D + d) * tk.Dv + col;
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            if (col + e < tk.Dv) *(float4*)(out + e) = make_float4(s[e], s[e + 1], s[e + 2], s[e + 3]);
        } else {
          const float w = tk.s1_mul * (tk.s1_decay && n > 0 ? power(1) : 1.f);
          float* out = tk.s1 + b * tk.s1s[0] + h * tk.s1s[1] + d * tk.s1s[2] + (long long)col * tk.s1s[3];
#pragma unroll
          for (int e = 0; e < 32; e++)
            if (col + e < tk.Dv) out[e * tk.s1s[3]] = w * s[e];
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
