// Linear attention with a decay for each head on the tensor cores (bf16 operands, fp32 accumulators in TMEM).
//
// A CTA takes one head of one row, up to 64 or 128 columns of v and a segment of the positions, 128 at a time (the MMA's M).
// With S the state before the chunk, P = (Q K^T) * lambda^(i-j) for j <= i, m tokens in the chunk:
//   O = lambda^(i+1) (Q S) + P V              S <- lambda^m S + X^T V,    X_j = lambda^(m-1-j) k_j
// Four products a chunk.  A chunk's q, k, v and y take about 5700 cycles of an SM's share of the memory's bandwidth at head
// size 128 (128 KB) and 2850 at 64; the products take 2050 to 2560 and 1020 to 1280.  So the kernel is bound by memory as
// far as what lies between the products keeps up, and that is spread over warps:
//   A warpgroups     P: TMEM -> scale, mask, round -> TMEM;  O: lambda^(i+1) between the two products;  output.  One, or
//                    two that take turns at head size 64, where a chunk has half the time
//   state warpgroups, one for each 32 columns of v    X: shared memory -> TMEM, transposed;  S: fp32 registers, and in bf16
//                    in shared memory for the next chunk's product
//   1 thread         TMA loads, 2 to 6 stages, and the store of O, which is staged where Q was
//   1 warp           tcgen05.mma, each product as soon as its operands are there
//
// Rounding.  y takes P and S rounded to bf16, one rounding beside its own, as any tensor-core product must.  The state is an
// fp32 result that lives for the whole row, so X is held as a sum of bf16 values: two (2^-16) where only y uses the state,
// three (2^-24) where it is an output; and S is added up in registers, not in the accumulator, whose additions truncate.
//
// Head size 64 would leave half of the 128 lanes of X^T V idle.  So lanes 0-63 take the chunk's first 64 positions and lanes
// 64-127 the others, against both halves of V side by side (N = 128): of the four 64 x 64 results the two mixed ones are
// not looked at, and S is the sum of two halves that Q S adds up, each with its own copy of Q.
//
// Time reversal (gradients of k and v): chunks from the last to the first, P and X mirrored.
//
// A segment's own contribution to the state (LOCAL) needs X^T V alone.
//
// Measured (bytes: q, k, v and y once).  8 x 12 heads x 4096 x 64: 74 us, 2.7 TB/s on 96 of 148
// SMs, 3800 cycles a chunk: bound by the chain from one chunk's state to the next's, X (1100), its product (1170), taking it
// over (470) and the wake-up between them (490), with the issuing warp's own 500 a step.  2 x 8 heads x 16384 x 128 in
// segments: 110 us in three launches, 2.4 TB/s (3.7 with the second reading of k and v), 5800 cycles a chunk.  The tensor
// pipe is busy for 31 to 35 %.  Tried and slower: four state warpgroups at head size 64 (85 us), the third part of X kept in
// registers at 128 (spills, 167 -> 194 us), the next launch's prologue overlapped with the last one's end (no gain).
//
// Every wait on an mbarrier is bounded: after LaParams::wait_ns the waiting role raises the CTA's flag, all roles leave, and
// the device's status word says so, which lies in host memory so that a later call can look at it without waiting.  The
// named barriers (bar.sync) stand where every thread of theirs comes by, given up or not: behind the state warpgroups' loop.
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "../../include/sffft.h"
#include "launch.h"
#include "linattn.h"
#include "plan.h"
#include "tc.cuh"

namespace sffft {

namespace {

constexpr int kTok = 128;   // positions in a chunk
constexpr uint64_t kCopyLimit = 2000000000ull;   // of what is in flight when a CTA gives up
constexpr uint32_t kBlk = kTok * 128;   // bytes of a 64-column tile of 128 positions: 128-byte rows, 128-byte swizzle

struct __align__(64) LaTcParams {
  CUtensorMap map[kLaMaxTasks][4];   // q, k, v, y
  LaParams p;
  int blocks;   // chunks in a segment
  int slices;   // CTAs over the columns of v
  int by_length;   // CTAs take the rows from the longest to the shortest
};

// The row that the CTAs numbered b take.  Where they come to between one and two for each SM, a long row that starts last
// leaves the other SMs idle behind it.  Own order against longest first, rows of random lengths, and two long ones among rows
// of a quarter (us):
//   8 rows x 12 heads x 1999 x 64 x 128, 192 CTAs     71, 70     68, 53
//   16 x 16 x 2000 x 64, 256                          84, 74     74, 58
//   30 x 8 x 4000 x 64, 240                          141, 131   123, 91
//   24 x 12 x 1024 x 128 x 64, 288                    78, 68     66, 64
//   10 x 15 x 3000 x 128, 150                        187, 176   205, 164
//   16 x 32 x 2000 x 64, 512                         137, 141   119, 105
// and no shape of up to two CTAs an SM was slower.  Beyond, either order may win.  Called by whole warps, each for itself: a
// lane ranks one row, ties by number.
constexpr int kMaxSorted = 32;
__device__ __forceinline__ int row_of(const LaTcParams& prm, int b) {
  if (!prm.by_length) return b;
  const int i = threadIdx.x & 31, mine = i < prm.p.B ? min(max(prm.p.len[i], 0), prm.p.L) : -1;
  int rank = 0;
#pragma unroll
  for (int j = 0; j < kMaxSorted; j++) {
    const int other = __shfl_sync(~0u, mine, j);
    rank += other > mine || (other == mine && j < i);
  }
  return __ffs(__ballot_sync(~0u, rank == b)) - 1;   // ranks are a permutation of the lanes, the rows' first
}

template <int DQ, int DV, bool LOCAL>
struct Shape {
  static constexpr bool split = DQ == 64;               // positions over the halves of the lanes
  static_assert(!split || DV == 64, "head size 64 takes 64 columns of v");
  static constexpr int NB = DV / 64, NW = DV / 32;      // 64-column tiles of v; state warpgroups, 32 columns each
  static constexpr int NA = LOCAL ? 0 : split ? 2 : 1;
  static constexpr int NS = LOCAL ? (split ? 6 : 3) : split ? 4 : 2;   // stages: what shared memory holds
  static constexpr int threads = 128 * NA + 128 * NW + 64;
  static constexpr uint32_t q_bytes = DQ / 64 * kBlk, v_bytes = NB * kBlk;
  static constexpr uint32_t off_k = LOCAL ? 0 : q_bytes, off_v = off_k + q_bytes, stage = off_v + v_bytes;
  static constexpr uint32_t off_s = NS * stage, off_tab = off_s + NB * kBlk, off_bar = off_tab + 4 * 160;
  static constexpr uint32_t smem = off_bar + 42 * 8 + 16;
  static_assert(smem <= 227 * 1024 && smem > 114 * 1024, "one CTA on an SM: each takes all of TMEM");
  // TMEM columns.  Products Q K^T (P over their first half) and O of A warpgroup a; the increment of S; X.
  __host__ __device__ static constexpr uint32_t c_p(int a) { return (uint32_t)a * 128; }
  __host__ __device__ static constexpr uint32_t c_o(int a) { return split ? (uint32_t)a * 128 + 64 : 128; }
  static constexpr uint32_t inc_cols = split ? 128 : DV;
  __host__ __device__ static constexpr uint32_t c_inc(int c) { return LOCAL ? (uint32_t)(c & 1) * 128 : 256; }   // LOCAL: two, in turn
  static constexpr uint32_t c_x = LOCAL ? 256 : 256 + inc_cols;
  static constexpr bool whole_x = split || LOCAL;       // all parts of X at once; else the third after the others
  static constexpr uint32_t part_cols = split ? 32 : 64;
  static_assert(c_x + part_cols * (whole_x ? 3 : 2) <= 512, "TMEM");
};

// Barriers.  A wait names a phase by its parity alone, so whoever waits must not fall two phases behind: that holds where the
// next phase needs something that the waiting role does after it has seen this one.  The thread that loads is ahead of
// nothing, so what it waits for has a barrier for each stage, whose next phase needs that thread's own next load.
// Those of the stages complete once for each NS chunks, those of an A warpgroup once for each NA, the others once a chunk.
// tests/test_mixer_protocol.py restates the roles and checks these rules, and that accesses to TMEM and to the tiles are
// ordered, for every shape: who changes a role changes it there too.
enum {
  B_KV = 0, B_Q = 6,          // K and V, Q loaded [stage]
  B_REL = 10,                 // K and V read by the state warpgroups and X^T V [stage]
  B_PV = 14,                  // V read by P V; LOCAL: by X^T V [stage]
  B_OOUT = 20,                // O staged [stage]
  B_S = 24, B_P = 26,         // products ready; P ready [A]
  B_O1 = 28, B_OS = 30,       // Q S taken; scaled [A]
  B_O = 32, B_OFREE = 34,     // O complete; its TMEM read [A]
  B_X = 36, B_INC,            // X ready (split: of even chunks), its product taken
  B_X2, B_INC2,               // third part ready (split: X of odd chunks), its product taken
  B_ST,                       // S taken over and published; once more before the first chunk (not LOCAL)
  B_FIN, B_COUNT
};
static_assert(B_COUNT <= 42, "barriers");

__host__ __device__ constexpr uint32_t idesc_bf16(int N, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// One lane of a warp whose control flow is uniform.  Behind this instruction the compiler keeps a product's descriptors in
// uniform registers; on a branch `lane == 0` (or with the products predicated) it moves them there anew for each product:
// 8 products of 128 x 64 x 16 are issued in 252 cycles here, in 600 (714) there, and execute in about 260.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
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
__device__ __forceinline__ float4 lds_f4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
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
  volatile int* stop;   // the limit of a wait lies two words behind
  volatile int* status;
  // false: the CTA gives up
  __device__ __forceinline__ bool operator()(int b, uint32_t parity) const {
    if (try_wait_for(bars + b, parity)) return true;
    return slow(b, parity);
  }
  __device__ __noinline__ bool slow(int b, uint32_t parity) const {
    const uint64_t t0 = global_ns();
    while (!try_wait_for(bars + b, parity)) {
      if (*stop) return false;
      if (global_ns() - t0 > *(volatile uint64_t*)(stop + 2)) {
        *stop = 1;
        *status = SFFFT_ERR_TIMEOUT;
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
__global__ void __launch_bounds__(Shape<DQ, DV, LOCAL>::threads, 1) la_tc_kernel(const __grid_constant__ LaTcParams prm) {
  using SH = Shape<DQ, DV, LOCAL>;
  constexpr int NB = SH::NB, NW = SH::NW, NA = SH::NA, NS = SH::NS;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t sm = smem_u32(smem);
  // Powers of lambda in the order in which they are wanted, so that a loop over positions has fixed offsets.  Forward:
  // lambda^127 .. lambda^0 and 32 zeros; in reverse: 32 zeros, lambda^0 .. lambda^127.  The zeros are the masked side of a
  // diagonal block.
  float* tab = (float*)(smem + SH::off_tab);
  uint64_t* bars = (uint64_t*)(smem + SH::off_bar);
  volatile int* stop = (volatile int*)(smem + SH::off_bar + 42 * 8);
  uint32_t* slot = (uint32_t*)(smem + SH::off_bar + 42 * 8 + 4);

  const LaParams& lp = prm.p;
  uint32_t u = blockIdx.x;
  const int vi = u % prm.slices;   // the CTA's columns of v
  u /= prm.slices;
  const int ti = u % lp.ntask;
  u /= lp.ntask;
  const LaTask& tk = lp.task[ti];
  const int cb = vi * DV;
  const int g = u % lp.G, h = u / lp.G % lp.H, b = row_of(prm, u / lp.G / lp.H), bh = b * lp.H + h;
  if (cb >= tk.Dv || (LOCAL && g == lp.G - 1)) return;   // nothing follows the last segment
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int n = lp.L;
  if (lp.len) n = min(max(lp.len[b], 0), lp.L);
  const bool rev = tk.rev;
  const int nblk = (n + kTok - 1) / kTok;
  const int c0 = min(g * prm.blocks, nblk), c1 = min(c0 + prm.blocks, nblk), nc = c1 - c0;
  const int before = tokens_before(c0, n, nblk, rev);
  const LaDecay dec(lp.ld[h]);
  const bool three = tk.s1 != nullptr && (LOCAL || g == lp.G - 1);   // the state, or what it is made of, is an output
  const bool fresh = !LOCAL && before == 0 && !tk.s0;                // the first chunk meets no state

  if (threadIdx.x == 0) {
    for (int i = 0; i < B_COUNT; i++) {
      const bool a = (i >= B_OOUT && i < B_S) || (i >= B_P && i < B_O1) || (i >= B_OS && i < B_O) || (i >= B_OFREE && i < B_X);
      const bool x = (i >= B_REL && i < B_PV) || i == B_X || i == B_X2 || i == B_ST;
      mbar_init(bars + i, a ? 128u : x ? 128u * NW : 1u);
    }
    *stop = 0;
    *(volatile uint64_t*)(stop + 2) = lp.wait_ns;
    fence_mbar_init();
  }
  for (int i = threadIdx.x; i < 160; i += blockDim.x) {
    const int e = rev ? i - 32 : 127 - i;
    tab[i] = e >= 0 ? dec.pow(e) : 0.f;
  }
  if (warp == SH::threads / 32 - 1) {
    tmem_alloc(slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // The CTA holds all 512 columns, which begin at address 0: a constant, so that the products' operands need no registers.
  constexpr uint32_t tm = 0;
  // Swizzled tiles need the alignment that the launch gives.  Not by `stop`, which an early role may raise before a late one
  // has looked: all threads have to decide alike.
  const bool dead = *slot != tm || (sm & 1023u) != 0;
  if (dead && threadIdx.x == 0) *(volatile int*)lp.status = SFFFT_ERR_DEVICE;
  const Waiter wait{bars, stop, lp.status};
  const WarpWaiter wwait{wait};
  auto power = [&](int e) { return tab[rev ? 32 + e : 127 - e]; };   // 0 <= e < 128

  auto block = [&](int c) { return rev ? nblk - 1 - (c0 + c) : c0 + c; };
  auto tokens = [&](int c) { return min(kTok, n - block(c) * kTok); };
  auto stage_at = [&](int c) { return sm + (uint32_t)(c % NS) * SH::stage; };
  auto sph = [](int c) { return (uint32_t)(c / NS) & 1; };         // phase of a stage's barrier
  auto aph = [](int c) { return (uint32_t)(c / (NA ? NA : 1)) & 1; };   // of an A warpgroup's
  auto grp = [](int c) { return NA ? c % NA : 0; };
  // Split: two parts of X leave room for the next chunk's, which is then made before this one's product is taken; so X has a
  // barrier for every other chunk.
  const bool two_x = SH::split && !LOCAL && !three;
  auto x_bar = [](int c) { return SH::split && !LOCAL && (c & 1) ? (int)B_X2 : (int)B_X; };
  auto x_ph = [](int c) { return (uint32_t)(SH::split && !LOCAL ? c >> 1 : c) & 1; };
  auto x_col = [&](int c) { return SH::c_x + (two_x ? (uint32_t)(c & 1) * 64 : 0u); };

  if (dead) {
    // nothing has been started
  } else if (warp == SH::threads / 32 - 2) {
    // ---- loads, stores ----
    if (lane == 0) {
      const CUtensorMap* mp = prm.map[ti];
      const int hq = h / tk.qdiv, hk = h / tk.kdiv, hv = h / tk.vdiv;
      int kv = 0, qs = 0;   // loads issued
      auto load_kv = [&]() {
        const int c = kv++;
        uint64_t* bar = bars + B_KV + c % NS;
        mbar_expect(bar, (SH::split && !LOCAL ? 2 : 1) * SH::q_bytes + SH::v_bytes);   // split: with Q
        for (int i = 0; i < DQ / 64; i++) tma_load(stage_at(c) + SH::off_k + i * kBlk, mp + 1, i * 64, block(c) * kTok, hk, b, bar);
        for (int i = 0; i < NB; i++) tma_load(stage_at(c) + SH::off_v + i * kBlk, mp + 2, cb + i * 64, block(c) * kTok, hv, b, bar);
      };
      auto load_q = [&]() {
        const int c = qs++;
        uint64_t* bar = bars + (SH::split ? B_KV : B_Q) + c % NS;
        if (!SH::split) mbar_expect(bar, SH::q_bytes);
        for (int i = 0; i < DQ / 64; i++) tma_load(stage_at(c) + i * kBlk, mp + 0, i * 64, block(c) * kTok, hq, b, bar);
      };
      while (kv < min(nc, NS)) {
        load_kv();
        if (!LOCAL) load_q();
      }
      for (int c = 0; c < nc; c++) {
        const int r = c % NS;
        if (LOCAL) {
          if (!wait(B_PV + r, sph(c))) break;
          if (kv < nc) load_kv();
          continue;
        }
        if (!SH::split) {   // with two stages K and V are wanted back before O is staged
          if (!wait(B_REL + r, sph(c)) || !wait(B_PV + r, sph(c))) break;
          if (kv < nc) load_kv();
        }
        if (!wait(B_OOUT + r, sph(c))) break;
        if (!tk.y_f32) {
          for (int i = 0; i < NB; i++) tma_store(mp + 3, stage_at(c) + i * kBlk, cb + i * 64, block(c) * kTok, h, b);
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        if (qs < nc) {
          if (SH::split && !wait(B_REL + r, sph(c))) break;   // and P V: O is out
          asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          if (SH::split) load_kv();
          load_q();
        }
      }
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
      if (*stop) {   // copies in flight end before the block does
        for (int c = max(0, kv - NS); c < kv; c++) mbar_wait_bounded(bars + B_KV + c % NS, sph(c), kCopyLimit);
        for (int c = max(0, qs - NS); !SH::split && c < qs; c++) mbar_wait_bounded(bars + B_Q + c % NS, sph(c), kCopyLimit);
      }
    }
  } else if (warp == SH::threads / 32 - 1) {
    // ---- products ----
    constexpr uint32_t id_s = idesc_bf16(128, false), id_v = idesc_bf16(DV, true), id_inc = idesc_bf16(SH::inc_cols, true);
    // a descriptor moved on by `bytes`: its address field is in the low word and never carries
    auto at = [](uint64_t d, uint32_t bytes) { return (d & 0xffffffff00000000ull) | (uint32_t)((uint32_t)d + (bytes >> 4)); };
    auto kstep = [](int k) { return (uint32_t)(k >> 2) * kBlk + (uint32_t)(k & 3) * 32; };   // K-major: 16 values on
    const bool later = three && !SH::whole_x;
    auto any = [](bool x) { return __any_sync(~0u, x) != 0; };   // a condition that the compiler too sees to be uniform
    // Each waits for its operands and issues its product; false: the CTA gives up.  A wait costs a hundred cycles, so what an
    // earlier one implies is not asked again.
    auto q_k = [&](int c) {
      if (!wwait(B_KV + c % NS, sph(c)) || (!SH::split && !wwait(B_Q + c % NS, sph(c)))) return false;
      // P of an earlier chunk lies where the product goes, and products with different accumulators are not kept in order.
      if (SH::split ? c >= NA && !wwait(B_OFREE + grp(c), aph(c - NA)) : c > 0 && !wwait(B_O, (c - 1) & 1)) return false;
      const uint64_t qd = make_sdesc(stage_at(c), 16, 1024, LT_SW128), kd = make_sdesc(stage_at(c) + SH::off_k, 16, 1024, LT_SW128);
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < DQ / 16; k++) mma_f16_ss(tm + SH::c_p(grp(c)), at(qd, kstep(k)), at(kd, kstep(k)), id_s, k > 0);
        mma_commit(bars + B_S + grp(c));
      }
      __syncwarp();
      return true;
    };
    auto q_s = [&](int c) {   // after x_v, which has seen S
      if (SH::split ? !wwait(B_P + grp(c), aph(c)) : c > 0 && !wwait(B_OFREE, (c - 1) & 1)) return false;
      const uint64_t qd = make_sdesc(stage_at(c), 16, 1024, LT_SW128), sd = make_sdesc(sm + SH::off_s, kBlk, 1024, LT_SW128);
      tc_fence_after();
      const bool state = any(!fresh || c > 0);
      if (elect_one()) {
        if (state)
#pragma unroll
          for (int k = 0; k < 8; k++)
            mma_f16_ss(tm + SH::c_o(grp(c)), at(qd, kstep(SH::split ? k & 3 : k)), at(sd, k * 2048), id_v, k > 0);
        mma_commit(bars + B_O1 + grp(c));
      }
      __syncwarp();
      return true;
    };
    auto p_v = [&](int c) {
      if (!wwait(B_OS + grp(c), aph(c))) return false;   // and P, from the same threads before
      const uint64_t vd = make_sdesc(stage_at(c) + SH::off_v, kBlk, 1024, LT_SW128);
      tc_fence_after();
      const bool state = any(!fresh || c > 0);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 8; k++)
          mma_ts(tm + SH::c_o(grp(c)), tm + SH::c_p(grp(c)) + k * 8, at(vd, k * 2048), id_v, k > 0 || state);
        mma_commit(bars + B_O + grp(c));
        if (!SH::split) mma_commit(bars + B_PV + c % NS);
      }
      __syncwarp();
      return true;
    };
    // X^T V: parts first .. last - 1 of X.  Split: 64 positions against both halves of V, 64 rows of 128 bytes apart.
    auto increment = [&](int c, uint32_t x_at, int first, int last, bool keep) {
      const uint64_t vd = make_sdesc(stage_at(c) + SH::off_v, SH::split ? kBlk / 2 : kBlk, 1024, LT_SW128);
#pragma unroll
      for (int part = first; part < last; part++)
#pragma unroll
        for (int k = 0; k < (SH::split ? 4 : 8); k++)
          mma_ts(tm + SH::c_inc(c), tm + x_at + part * SH::part_cols + k * 8, at(vd, k * 2048), id_inc, keep || part > first || k > 0);
    };
    auto x_v = [&](int c) {
      // The increment's columns have been taken over: from the last chunk, once its state is published; LOCAL, from the last
      // but one, before X of this one came.
      if ((LOCAL && !wwait(B_KV + c % NS, sph(c))) || !wwait(x_bar(c), x_ph(c)) || (!LOCAL && !wwait(B_ST, c & 1))) return false;
      const bool all = any(SH::whole_x && three), odd = any(x_col(c) != SH::c_x);
      tc_fence_after();
      if (elect_one()) {
        if (all) increment(c, SH::c_x, 0, 3, false);
        else if (odd) increment(c, SH::c_x + 64, 0, 2, false);
        else increment(c, SH::c_x, 0, 2, false);
        mma_commit(bars + B_INC);
        if (LOCAL) mma_commit(bars + B_PV + c % NS);
      }
      __syncwarp();
      return true;
    };
    auto x_v_third = [&](int c) {
      if (!wwait(B_X2, c & 1)) return false;
      tc_fence_after();
      if (elect_one()) {
        increment(c, SH::c_x, 0, 1, true);
        mma_commit(bars + B_INC2);
      }
      __syncwarp();
      return true;
    };
    // The order in which operands become ready (asking for whichever is took 10 questions a product, 500 cycles and more).
    // The state's product goes first: the chain from one to the next (X, and taking the state over) is the longest.
    if constexpr (LOCAL) {
      for (int c = 0; any(c < nc); c++)
        if (!x_v(c)) break;
    } else if constexpr (SH::split) {
      if (any(nc > 0) && q_k(0))
        for (int c = 0; any(c < nc); c++)
          if (!x_v(c) || !q_s(c) || (any(c + 1 < nc) && !q_k(c + 1)) || !p_v(c)) break;
    } else {
      for (int c = 0; any(c < nc); c++)
        if (!q_k(c) || !x_v(c) || !q_s(c) || !p_v(c) || (any(later) && !x_v_third(c))) break;
    }
    if (any(*stop != 0)) {   // products in flight end before TMEM is given back; the election needs the whole warp
      if (elect_one()) {
        mma_commit(bars + B_FIN);
        mbar_wait_bounded(bars + B_FIN, 0, kCopyLimit);
      }
      __syncwarp();
    }
  } else if (warp < 4 * NA) {
    // ---- P and O ----
    if constexpr (!LOCAL) {
      const int i = threadIdx.x & 127, a = warp >> 2, quad = warp & 3;   // position in the chunk
      const uint32_t tl = tm + ((uint32_t)(quad * 32) << 16), tp = tl + SH::c_p(a), to = tl + SH::c_o(a);
      const float whole = dec.pow(kTok);
      for (int c = a; c < nc; c += NA) {
        const uint32_t ph = aph(c);
        const int m = tokens(c), blk = block(c);
        const int off = tk.off && before == 0 && c == 0;
        if (!wwait(B_S + a, ph)) break;
        tc_fence_after();
#pragma unroll 1
        for (int jb = 0; jb < 4; jb++) {
          uint32_t r[32], o[16];
          if (rev ? jb < quad : jb > quad) {   // a block on the masked side of the diagonal
#pragma unroll
            for (int e = 0; e < 16; e++) o[e] = 0;
          } else {
            tmem_ld32(tp + jb * 32, r);
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
          tmem_st16(tp + jb * 16, o);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bars + B_P + a);
        // lambda^(i+1) Q S, in reverse lambda^(m-i)
        if (!wwait(B_O1 + a, ph)) break;
        tc_fence_after();
        if (!(fresh && c == 0)) {
          const int e = (rev ? m - i : i + 1) - off;
          const float w = e < 0 ? 0.f : e < kTok ? power(e) : whole;
#pragma unroll 1
          for (int q = 0; q < DV / 32; q++) {
            uint32_t r[32];
            tmem_ld32(to + q * 32, r);
            tmem_wait_ld();
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              const F2 z = mul2({__uint_as_float(r[x]), __uint_as_float(r[x + 1])}, {w, w});
              r[x] = __float_as_uint(z.a), r[x + 1] = __float_as_uint(z.b);
            }
            tmem_st32(to + q * 32, r);
          }
          tmem_wait_st();
        }
        tc_fence_before();
        if (!(lp.withhold == LA_WITHHOLD_OS && i == 0)) mbar_arrive(bars + B_OS + a);
        if (!wwait(B_O + a, ph)) break;
        tc_fence_after();
        // staged where Q was, whose products are complete: bf16 in the swizzled rows that the TMA store takes, or fp32, 64
        // (split: 32) columns at a time, from where the warp writes its 32 rows as whole ones (a lane's own row would be
        // pieces of 16 bytes in 32 rows at once).  A warp's rows are its own business: a barrier among the warps would not
        // be bounded, and one of them may have given up.
        const uint32_t out = stage_at(c) + (uint32_t)i * 128;
#pragma unroll 1
        for (int q = 0; q < DV / 32; q++) {
          uint32_t r[32];
          tmem_ld32(to + q * 32, r);
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
          } else {
            // 128-byte rows of 32 columns; Q's tile holds one such block, or two
            const uint32_t blk_at = stage_at(c) + (SH::q_bytes > kBlk ? (uint32_t)(q & 1) * kBlk : 0u);
#pragma unroll
            for (int e = 0; e < 8; e++)
              sts128(blk_at + (uint32_t)i * 128 + (((uint32_t)e ^ (uint32_t)(i & 7)) << 4), __float_as_uint(tk.scale * __uint_as_float(r[4 * e])),
                     __float_as_uint(tk.scale * __uint_as_float(r[4 * e + 1])), __float_as_uint(tk.scale * __uint_as_float(r[4 * e + 2])),
                     __float_as_uint(tk.scale * __uint_as_float(r[4 * e + 3])));
            __syncwarp();
            float* y = (float*)tk.y + b * tk.ys[0] + h * tk.ys[1] + (long long)(blk * kTok) * tk.ys[2] + cb + q * 32;
#pragma unroll 4
            for (int x = 0; x < 8; x++) {   // 4 rows of 8 pieces at a time; Dv is a multiple of 8
              const int row = quad * 32 + x * 4 + (lane >> 3), e = lane & 7;
              if (blk * kTok + row < lp.L && cb + q * 32 + e * 4 < tk.Dv)
                *(float4*)(y + (long long)row * tk.ys[2] + e * 4) = lds_f4(blk_at + (uint32_t)row * 128 + ((uint32_t)(e ^ (row & 7)) << 4));
            }
            if (SH::q_bytes == kBlk || (q & 1)) __syncwarp();
          }
        }
        fence_async_smem();
        tc_fence_before();
        mbar_arrive(bars + B_OFREE + a);
        if (!(lp.withhold == LA_WITHHOLD_OOUT && i == 0)) mbar_arrive(bars + B_OOUT + c % NS);
      }
      // chunks of the segment behind the row's last token
      const int z0 = max(g * prm.blocks, nblk) * kTok, z1 = min((long long)(g + 1) * prm.blocks * kTok, (long long)lp.L);
      const int pieces = min(tk.Dv - cb, DV) / 8;
      for (long long e = threadIdx.x; e < (long long)(z1 - z0) * pieces; e += 128 * NA) {
        const long long at = b * tk.ys[0] + h * tk.ys[1] + (z0 + e / pieces) * tk.ys[2] + cb + (e % pieces) * 8;
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
    const int wg = (warp >> 2) - NA, t = threadIdx.x & 127, quad = warp & 3;
    const uint32_t tl = tm + ((uint32_t)(quad * 32) << 16);
    const int d = SH::split ? t & 63 : t;         // the thread's row of the state
    const bool main_part = !SH::split || t < 64;  // split: lanes 64-127 hold the second halves' sum
    float s[32];                                  // columns 32 wg ..
    const int col = cb + wg * 32;
#pragma unroll
    for (int e = 0; e < 32; e++) s[e] = 0.f;
    const long long mine = (long long)col * tk.D + d;   // of the segments' states, which are kept transposed: lanes are rows
    if (!LOCAL && main_part && d < tk.D) {
      if (g > 0) {   // what the earlier segments leave, s0 included
        const float* in = tk.loc + ((long long)bh * lp.G + g - 1) * tk.D * tk.Dv + mine;
#pragma unroll
        for (int e = 0; e < 32; e++)
          if (col + e < tk.Dv) s[e] = in[(long long)e * tk.D];
      } else if (tk.s0) {
        const float* s0 = tk.s0 + b * tk.s0s[0] + h * tk.s0s[1] + d * tk.s0s[2] + (long long)col * tk.s0s[3];
        if (tk.s0s[3] == 1 && ((uintptr_t)s0 & 15) == 0) {   // a lane's values lie together
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            if (col + e < tk.Dv) {
              const float4 x = *(const float4*)(s0 + e);
              s[e] = x.x * tk.s0_mul, s[e + 1] = x.y * tk.s0_mul, s[e + 2] = x.z * tk.s0_mul, s[e + 3] = x.w * tk.s0_mul;
            }
        } else {
#pragma unroll
          for (int e = 0; e < 32; e++)
            if (col + e < tk.Dv) s[e] = s0[e * tk.s0s[3]] * tk.s0_mul;
        }
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
    if (!LOCAL) {
      publish();
      mbar_arrive(bars + B_ST);
    }
    // lambda^128 as a sum of two floats: its rounding would come back with every chunk
    const float whole = dec.pow(kTok), whole_lo = dec.pow_rest(kTok, whole);
    // Address of the lane's row of the K tiles of the warp's first 16 rows d and first 16 positions: tiles (d, position) are
    // (0-7, 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15); 16 rows d on is two 16-byte pieces on, under the swizzle.
    const int dw = SH::split ? (quad & 1) * 32 : quad * 32;
    const uint32_t kaddr = SH::off_k + (uint32_t)(dw >> 6) * kBlk + (uint32_t)(((lane >> 4) & 1) * 8 + (lane & 7)) * 128 +
                           ((((uint32_t)(dw & 63) >> 3) + ((uint32_t)(lane >> 3) & 1)) ^ (uint32_t)(lane & 7)) * 16;
    // Positions whose X the warp makes, and the column of X that the first of them has.
    constexpr int kMine = SH::split ? 64 / NW : kTok / NW;
    const int first = SH::split ? (quad >> 1) * 64 + wg * kMine : wg * kMine;
    const uint32_t xcol = (uint32_t)(wg * kMine) / 2;
    static_assert(kMine % 32 == 0, "32 positions at a time");

    // Parts of X of chunk c: the first two (and the third, whole_x), or the third alone.  Lanes of X are rows d of the state,
    // its columns pairs of positions: K's tiles come transposed from shared memory in the very arrangement that the 16 x 128b
    // store takes.  Each part but the last is cut off, not rounded, so that what is left is exact.
    auto make_x = [&](int c, int m, bool third) {
      const uint32_t st = stage_at(c);
#pragma unroll 1
      for (int jj = 0; jj < kMine; jj += 32) {
        const int j0 = first + jj;
        float w[8];   // of positions j0 + 8 i + 2 (lane % 4) + {0, 1}
        const int wi = (rev ? 32 : kTok - m) + j0 + 2 * (lane & 3);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float* at = tab + min(wi + 8 * i, 158);   // behind the last token: the zeros
          w[2 * i] = at[0], w[2 * i + 1] = at[1];
        }
#pragma unroll 1
        for (int half = 0; half < 2; half++) {   // 16 rows each
          uint32_t r[8], y[8], z[8];
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
          const uint32_t to = tl + ((uint32_t)(16 * half) << 16) + x_col(c) + xcol + jj / 2;
          if (SH::whole_x && three) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
              F2 x = mul2({lo_f(r[i]), hi_f(r[i])}, {w[i & ~1], w[i | 1]});
              r[i] = upper2(x);
              x = sub2(x, cut2(x));
              y[i] = upper2(x);
              x = sub2(x, cut2(x));
              z[i] = pack_bf16(x.a, x.b);
            }
            tmem_st_16x128b_x4(to, r);
            tmem_st_16x128b_x4(to + SH::part_cols, y);
            tmem_st_16x128b_x4(to + 2 * SH::part_cols, z);
          } else if (!third) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
              F2 x = mul2({lo_f(r[i]), hi_f(r[i])}, {w[i & ~1], w[i | 1]});
              r[i] = upper2(x);
              x = sub2(x, cut2(x));
              y[i] = three ? upper2(x) : pack_bf16(x.a, x.b);   // cut off where a third follows
            }
            tmem_st_16x128b_x4(to, r);
            tmem_st_16x128b_x4(to + SH::part_cols, y);
          } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
              F2 x = mul2({lo_f(r[i]), hi_f(r[i])}, {w[i & ~1], w[i | 1]});
              x = sub2(x, cut2(x));
              x = sub2(x, cut2(x));
              r[i] = pack_bf16(x.a, x.b);
            }
            tmem_st_16x128b_x4(to, r);
          }
        }
      }
      tmem_wait_st();
      tc_fence_before();
    };
    // S <- lambda^m S + X^T V of chunk c, whose product is complete
    auto take = [&](int c) {
      const int m = tokens(c), off = tk.off && before == 0 && c == 0;
      float w = whole, w_lo = whole_lo;
      if (m - off < kTok) w = power(m - off), w_lo = 0.f;
      const uint32_t from = tl + SH::c_inc(c) + (SH::split ? (uint32_t)(quad >> 1) * 64 : 0) + wg * 32;
      uint32_t r[32];
      tmem_ld32(from, r);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const F2 z = fma2({w, w}, {s[e], s[e + 1]}, fma2({w_lo, w_lo}, {s[e], s[e + 1]}, {__uint_as_float(r[e]), __uint_as_float(r[e + 1])}));
        s[e] = z.a, s[e + 1] = z.b;
      }
      tc_fence_before();
    };
    // X of chunk c, once its tiles are there
    auto give_x = [&](int c) {
      const int m = tokens(c);
      if (!wwait(B_KV + c % NS, sph(c))) return false;
      if (m < kTok && n < lp.L) {   // v behind the last token may hold anything, and 0 * NaN is NaN
        const uint32_t v = stage_at(c) + SH::off_v + (uint32_t)(wg >> 1) * kBlk;
        for (int e = t; e < (kTok - m) * 4; e += 128)
          sts128(v + (uint32_t)(m + (e >> 2)) * 128 + (uint32_t)(4 * (wg & 1) + (e & 3)) * 16, 0, 0, 0, 0);
        fence_async_smem();
      }
      make_x(c, m, false);
      if (!(lp.withhold == LA_WITHHOLD_X && c == nc - 1 && wg == 0 && t == 0)) mbar_arrive(bars + x_bar(c));
      return true;
    };
    // X of the next chunk goes before this one's state: it needs only the columns that this one's product has read, or, with
    // columns of its own (two_x), the last one's.
    if (nc > 0 && give_x(0))
      for (int c = 0; c < nc; c++) {
        if (two_x && c + 1 < nc && !give_x(c + 1)) break;
        if (!wwait(B_INC, c & 1)) break;
        tc_fence_after();
        if (three && !SH::whole_x) {
          make_x(c, tokens(c), true);
          mbar_arrive(bars + B_X2);
          if (!wwait(B_INC2, c & 1)) break;
          tc_fence_after();
        }
        if (!two_x && c + 1 < nc && !give_x(c + 1)) break;
        if (!LOCAL && !wwait(B_O1 + grp(c), aph(c))) break;   // the product with the old S has been taken
        take(c);
        if (LOCAL) continue;
        if (c + 1 < nc) publish();
        mbar_arrive(bars + B_ST);
        mbar_arrive(bars + B_REL + c % NS);
      }
    // the state that the segment leaves (after a wait that gave up: whatever it is, but every thread comes by)
    if (LOCAL || (tk.s1 && g == lp.G - 1)) {
      if constexpr (SH::split) {   // add the two halves, in S's shared memory, once all warpgroups are through with it
        asm volatile("bar.sync 5, %0;" ::"n"(128 * NW) : "memory");
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
          float* out = tk.loc + ((long long)bh * lp.G + g) * tk.D * tk.Dv + mine;
#pragma unroll
          for (int e = 0; e < 32; e++)
            if (col + e < tk.Dv) out[(long long)e * tk.D] = s[e];
        } else {
          const float w = tk.s1_mul * (tk.s1_decay && n > 0 ? power(1) : 1.f);
          float* out = tk.s1 + b * tk.s1s[0] + h * tk.s1s[1] + d * tk.s1s[2] + (long long)col * tk.s1s[3];
          if (tk.s1s[3] == 1 && ((uintptr_t)out & 15) == 0) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              if (col + e < tk.Dv) *(float4*)(out + e) = make_float4(w * s[e], w * s[e + 1], w * s[e + 2], w * s[e + 3]);
          } else {
#pragma unroll
            for (int e = 0; e < 32; e++)
              if (col + e < tk.Dv) out[e * tk.s1s[3]] = w * s[e];
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == SH::threads / 32 - 1) tmem_dealloc(*slot, 512);
}

// What the segments up to each one leave, from what each leaves alone, in place; the last one's is not needed.  A thread
// takes one element of a state; the loads of all segments are independent of the sums.
__global__ void __launch_bounds__(256) la_prefix_kernel(const __grid_constant__ LaTcParams prm) {
  const LaParams& lp = prm.p;
  const LaTask& tk = lp.task[blockIdx.z];
  const int size = tk.D * tk.Dv, e = blockIdx.y * 256 + threadIdx.x;   // [Dv][D]
  const int bh = blockIdx.x, b = bh / lp.H, h = bh % lp.H;
  if (e >= size) return;
  int n = lp.L;
  if (lp.len) n = min(max(lp.len[b], 0), lp.L);
  const int nblk = (n + kTok - 1) / kTok;
  const LaDecay dec(lp.ld[h]);
  float s = 0.f;
  if (tk.s0) s = tk.s0[b * tk.s0s[0] + h * tk.s0s[1] + (e % tk.D) * tk.s0s[2] + (e / tk.D) * tk.s0s[3]] * tk.s0_mul;
  float* loc = tk.loc + (long long)bh * lp.G * size + e;
  for (int g0 = 0; g0 < lp.G - 1; g0 += 8) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (g0 + i < lp.G - 1) x[i] = loc[(long long)(g0 + i) * size];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int g = g0 + i;
      if (g >= lp.G - 1) break;
      const int a = tokens_before(min(g * prm.blocks, nblk), n, nblk, tk.rev);
      const int m = tokens_before(min((g + 1) * prm.blocks, nblk), n, nblk, tk.rev) - a;
      if (m > 0) s = fmaf(dec.pow(m - (tk.off && a == 0)), s, x[i]);
      loc[(long long)g * size] = s;
    }
  }
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
  if (((uintptr_t)p & 15) != 0 || D % 8 != 0) return false;
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
cudaError_t launch_shape(LaTcParams& prm, cudaStream_t st) {
  const dim3 grid((unsigned)(prm.p.B * prm.p.H * prm.p.G * prm.p.ntask * prm.slices));
  prm.by_length = prm.p.len && prm.p.B <= kMaxSorted && prm.p.G == 1 && grid.x > (unsigned)prm.p.sms &&
                  grid.x <= 2u * (unsigned)prm.p.sms;
  if (prm.p.G > 1) {
    using SH = Shape<DQ, DV, true>;
    cudaError_t ce = launch(la_tc_kernel<DQ, DV, true>, grid, SH::threads, (int)SH::smem, st, prm);
    if (ce != cudaSuccess) return ce;
    int size = 0;
    for (int i = 0; i < prm.p.ntask; i++) size = std::max(size, prm.p.task[i].D * prm.p.task[i].Dv);
    ce = launch(la_prefix_kernel, dim3((unsigned)(prm.p.B * prm.p.H), (unsigned)((size + 255) / 256), (unsigned)prm.p.ntask), 256, 0, st, prm);
    if (ce != cudaSuccess) return ce;
  }
  using SH = Shape<DQ, DV, false>;
  return launch(la_tc_kernel<DQ, DV, false>, grid, SH::threads, (int)SH::smem, st, prm);
}

}  // namespace

bool la_tc_takes(const LaParams& p) {
  if (p.L < 1 || !encode_fn()) return false;
  for (int i = 0; i < p.ntask; i++) {
    const LaTask& t = p.task[i];
    if (t.D > 128 || !mappable(t.q, t.qs, p.B, p.H / t.qdiv, p.L, t.D) || !mappable(t.k, t.ks, p.B, p.H / t.kdiv, p.L, t.D) ||
        !mappable(t.v, t.vs, p.B, p.H / t.vdiv, p.L, t.Dv) || !mappable(t.y, t.ys, p.B, p.H, p.L, t.Dv))
      return false;
  }
  return true;
}

int la_tc_tile(int D, int Dv) { return D > 64 && Dv > 64 ? 128 : 64; }

int la_tc_slices(int D, int Dv) { return (Dv + la_tc_tile(D, Dv) - 1) / la_tc_tile(D, Dv); }

cudaError_t launch_la_tc(const LaParams& p, cudaStream_t st) {
  // tasks of one tile shape go into one launch
  bool done[kLaMaxTasks] = {};
  for (int i = 0; i < p.ntask; i++) {
    if (done[i]) continue;
    LaTcParams prm = {};
    prm.p = p;
    prm.p.ntask = 0;
    prm.blocks = p.seg / kTok;
    prm.slices = 1;
    const bool q2 = p.task[i].D > 64;
    const int dv = la_tc_tile(p.task[i].D, p.task[i].Dv);
    for (int j = i; j < p.ntask; j++) {
      const LaTask& t = p.task[j];
      if (done[j] || (t.D > 64) != q2 || la_tc_tile(t.D, t.Dv) != dv) continue;
      done[j] = true;
      const int k = prm.p.ntask++;
      prm.p.task[k] = t;
      const int sl = la_tc_slices(t.D, t.Dv);
      if (sl > prm.slices) prm.slices = sl;
      if (!make_map(&prm.map[k][0], t.q, t.qs, p.B, p.H / t.qdiv, p.L, t.D) ||
          !make_map(&prm.map[k][1], t.k, t.ks, p.B, p.H / t.kdiv, p.L, t.D) ||
          !make_map(&prm.map[k][2], t.v, t.vs, p.B, p.H / t.vdiv, p.L, t.Dv) ||
          (!t.y_f32 && !make_map(&prm.map[k][3], t.y, t.ys, p.B, p.H, p.L, t.Dv)))
        return cudaErrorInvalidValue;
    }
    const cudaError_t ce = !q2 ? launch_shape<64, 64>(prm, st) : dv == 128 ? launch_shape<128, 128>(prm, st)
                                                                           : launch_shape<128, 64>(prm, st);
    if (ce != cudaSuccess) return ce;
  }
  return cudaSuccess;
}

// Status words of the devices, in page-locked host memory that every device can write.
namespace {
std::atomic<int*> g_words{nullptr}, g_device_word[kLaMaxDevices];   // and their addresses on the devices
}

cudaError_t la_tc_word(int device, int** word) {
  static std::mutex mutex;
  if (device < 0 || device >= kLaMaxDevices) return cudaErrorInvalidDevice;
  if ((*word = g_device_word[device].load(std::memory_order_acquire))) return cudaSuccess;
  int* p = g_words.load(std::memory_order_acquire);
  if (!p) {
    std::lock_guard<std::mutex> lock(mutex);
    p = g_words.load(std::memory_order_relaxed);
    if (!p) {
      // The first call may be one that a graph captures, where allocations are refused unless the thread says otherwise.
      cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
      cudaError_t ce = cudaThreadExchangeStreamCaptureMode(&mode);
      if (ce != cudaSuccess) return ce;
      void* m = nullptr;
      ce = cudaHostAlloc(&m, kLaMaxDevices * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
      cudaThreadExchangeStreamCaptureMode(&mode);
      if (ce != cudaSuccess) return ce;
      p = (int*)m;
      std::fill(p, p + kLaMaxDevices, 0);
      g_words.store(p, std::memory_order_release);
    }
  }
  void* on_device = nullptr;
  const cudaError_t ce = cudaHostGetDevicePointer(&on_device, p + device, 0);
  if (ce == cudaSuccess) g_device_word[device].store(*word = (int*)on_device, std::memory_order_release);
  return ce;
}

int la_tc_reported(int device) {
  const int* p = g_words.load(std::memory_order_acquire);
  return p && device >= 0 && device < kLaMaxDevices ? *(const volatile int*)(p + device) : SFFFT_OK;
}

cudaError_t la_tc_status(int device, int* status) {
  const cudaError_t ce = cudaDeviceSynchronize();
  *status = ce == cudaSuccess ? la_tc_reported(device) : SFFFT_OK;
  if (*status) ((volatile int*)g_words.load())[device] = 0;
  return ce;
}

}  // namespace sffft
