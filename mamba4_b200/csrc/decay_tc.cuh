// Decay attention on the fifth-generation tensor cores: bfloat16 operands.
//
// One CTA walks the chunks of one (pass, batch row, head, segment of the time
// axis); see decay.cu for the recurrence. Everything with a head dim in its
// rows is computed transposed, so that 128-wide head dims fill the 128 lanes
// of tensor memory with chunks of 64 tokens:
//   P   [t, s]    = Q K^T                          (64 x 64)
//   O1^T[dv, t]   = V^T P'^T,  P' = masked, decayed P in two bfloat16 terms
//   O2^T[dv, t]   = S^T Q^T,   S^T [dv, dk] the state before, in two terms
//   dS^T[dv, dk]  = (w V)^T K, the weighted values in three terms
// (an fp32 factor times a bfloat16 value has 32 significant bits: three terms
// keep 24 of them, the float32 that a state is held in; two, which keep 16, let
// contributions that cancel leave little behind, and cost 2.4 % less in a
// training step. The scores and a state that is read keep 16: they end in a
// bfloat16 result at once, to which they add 2^-16 of the sum of absolute values
// at most. In a training step, 64 x 128, 0.25 % of the results are not the
// rounded exact ones, 0.02 % with float32 products, and the error against 64 bits
// is the same.) The running state stays in registers in float32: S' = e^{g L} S +
// dS, so chunks join with one rounding each. (The weights go on the narrower of V
// and K.)
//
// Warps: XW for scores and weights, 4 for outputs, SW for the state, one each
// for loads, products and stores. They meet on mbarriers only; every wait
// is bounded. Tiles are [64 tokens][64 columns] panels with the 128-byte
// swizzle; a chunk's output is gathered in its own, then idle, input tiles.
//
// What bounds it: the chunk-to-chunk hand-overs. A chunk's state is needed by
// the next one's outputs, and its weighted terms by its state, so that the
// groups work on neighbouring chunks in turn. Measured (B200; 148 CTAs, dims
// key x value, us a chunk of 64 tokens and CTA, of the SM's share of bandwidth):
//   64 x 64 (two CTAs an SM)  2.45   4.0 TB/s        128 x 64   1.68   4.3 TB/s
//   64 x 128                  1.52   4.8 TB/s        128 x 128  2.40   4.0 TB/s
// against 6.6 TB/s of a copy, and about 7 us to start a CTA (tables, tensor
// memory, first loads). At 64 x 128 the tensor pipe is busy 24 (forward) to 32 %
// of the time (backward) and 41 % of the issue slots are taken; with the barriers
// alone a chunk takes 0.72 us, with a quarter of its products, or without loads,
// stores or weights, 1.41, so no one part bounds it. Whole sequences of few heads
// are cut into segments, which read the keys and values twice.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "tc05.cuh"

namespace m4 {
namespace decay {

constexpr int PANEL = 64 * 128;  // bytes of a [64][64] bfloat16 panel

struct alignas(64) TcProblem {
  CUtensorMap maps[4];
  CUtensorMap out_maps[3];  // of each pass's output (bfloat16 outputs)
  Problem pr;
  int map_of[3][3];         // tensor map of each pass's a, b, c
  int segments, segment_tokens;
  float* seg_state;     // [passes][B][H][segments][da][dc]: states at segment starts (phase 1: at their ends)
  size_t seg_pass;      // floats per pass in seg_state
};

template <int DA, int DC, bool READ>
struct Geo {
  static constexpr int NA = DA / 64, NC = DC / 64;
  static constexpr bool SMALL = DA + DC == 128;           // two CTAs an SM
  // State in tensor memory as the A operand (128 rows of dv), or in shared
  // memory (64 rows; its two terms then stand in one operand of 128 rows, 16
  // and 16 alternating, so that a lane quarter gets both parts of its rows).
  static constexpr bool S_TMEM = DC == 128;
  // The two terms of the scores side by side in one product of N = 128, summed
  // when the outputs are read, where tensor memory has room.
  static constexpr bool P_WIDE = DC == 64 && !SMALL;
  static constexpr int NQ = READ ? NA : 0;                // panels of the a operand
  static constexpr int STAGE = (NQ + NA + NC) * PANEL;
  // As many chunks ahead as shared memory holds: a load under full HBM traffic
  // takes about 3000 cycles, a chunk 2000 to 4500.
  static constexpr int STAGES = SMALL ? 2 : (!READ || DA < DC ? 4 : 3);
  static constexpr int WB = READ || SMALL ? 1 : 2;        // buffers of weighted terms and of what they add
  static constexpr int XW = SMALL ? 4 : 8;                // warps for scores and weights
  static constexpr int SW = SMALL ? 4 : 8;                // state warps
  // Three warps work in the last group. 768 threads of 80 registers; the groups
  // then share them out as they need: 2 x 64 + 104 + 2 x 104 + 40 = 6 x 80.
  static constexpr bool SHARE_REGS = !SMALL;
  static constexpr int THREADS = 32 * (XW + 4 + SW + (SHARE_REGS ? 4 : 3));
  static constexpr bool W_ON_K = NA < NC;                 // which operand of the state's product is weighted
  static constexpr int NW = W_ON_K ? NA : NC;             // its panels
  static constexpr int S_ROWS = 128 * 128;                // bytes of a panel of S^T (shared memory, both terms)
  static constexpr int W_TERM = NW * PANEL;
  static constexpr int OFF_P = STAGES * STAGE;            // two panels
  static constexpr int OFF_W = OFF_P + (READ ? 2 * PANEL : 0);
  static constexpr int OFF_S = OFF_W + WB * 3 * W_TERM;
  static constexpr int BYTES = OFF_S + (S_TMEM || !READ ? 0 : NA * S_ROWS);
  static constexpr int SMEM = BYTES + 1024;
  // Tensor-memory columns. With two sets of output accumulators a chunk's
  // scores lie where its output's own part goes once they are read.
  static constexpr int OB = SMALL ? 1 : 2;
  static constexpr int O1 = P_WIDE ? 128 : 64, OSET = O1 + 64;
  static constexpr int COL_O = !READ || OB == 2 ? 0 : 64;
  static constexpr int COL_S = READ ? COL_O + OSET * OB : 0, COL_A = COL_S + DA * WB;
  static constexpr int USED = COL_A + (READ && S_TMEM ? DA : 0);
  static constexpr int COLS = USED <= 256 ? 256 : 512;
  static_assert(USED <= COLS && BYTES + 1024 + 2048 <= 227 * 1024, "tensor and shared memory");
  static constexpr int SC = DA / (SW / 4);                // state columns of a state warp
};

constexpr int MAX_STAGES = 4;
// No barrier completes a phase before its waiters have seen the one before:
// each is signalled for chunk n + 1 only after something its waiter does after
// its wait for chunk n. (full, staged, empty: n + STAGES, one barrier a stage;
// with two output accumulators o_full and o_free: n + 2, one barrier each.)
struct Bars {
  uint64_t full[MAX_STAGES], staged[MAX_STAGES], empty[MAX_STAGES];
  uint64_t w_ready[2], ds_full[2], ds_free[2], p_full, p_ready, s_ready, q_done, o_full[2], o_free[2], clean;
};

__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::su32(bar)) : "memory");
}
// One arrival for a warp's work (32 arrivals at one address are done one after another).
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) bar_arrive(bar);
}
__device__ __forceinline__ void tma_load_4d(void* dst, const void* map, int c0, int c1, int c2, int c3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(tc::su32(dst)), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(tc::su32(bar)) : "memory");
}
__device__ __forceinline__ void tma_store_4d(const void* map, const void* src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(map),
               "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(tc::su32(src)) : "memory");
}
// Named barrier of the 128 output threads.
__device__ __forceinline__ void output_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
template <bool ON, int N, bool MORE>
__device__ __forceinline__ void registers() {
  if constexpr (ON) {
    if constexpr (MORE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
  }
}
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is != 0;
}
// Wait until the barrier's phase `parity` has completed. A wait that gives up
// sets `gone`, which ends every later wait of the CTA at once. (In assembly: a
// wait is a few instructions in a kernel whose roles share the instruction
// cache; the compiler's version of this loop was 2 KB long.)
__device__ __forceinline__ void bar_wait(uint64_t* bar, uint32_t parity, const int* gone) {
  asm volatile(
      "{\n\t"
      ".reg .pred done, end;\n\t"
      ".reg .u32 polls, dead, far;\n\t"
      "mov.u32 polls, 0;\n"
      "POLL_%=:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 done, [%0], %1;\n\t"
      "@done bra DONE_%=;\n\t"
      "ld.volatile.shared.u32 dead, [%2];\n\t"
      "add.u32 polls, polls, 1;\n\t"
      "shr.u32 far, polls, 21;\n\t"
      "or.b32 dead, dead, far;\n\t"
      "setp.eq.u32 end, dead, 0;\n\t"
      "@end bra POLL_%=;\n\t"
      "st.volatile.shared.u32 [%2], 1;\n"
      "DONE_%=:\n\t"
      "}" ::"r"(tc::su32(bar)), "r"(parity), "r"(tc::su32(gone)) : "memory");
}

// 16 rows x 32 columns of an accumulator: v[4 k + 2 hh + j] is row
// lane / 4 + 8 hh, column 8 k + 2 (lane % 4) + j.
__device__ __forceinline__ void tm_load(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void stm4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d) : "memory");
}
__device__ __forceinline__ void stm4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b),
               "r"(c), "r"(d) : "memory");
}
// The thread's row (tensor-memory lane), 16 columns.
__device__ __forceinline__ void tm_load_row(uint32_t taddr, float (&v)[16]) { tc::ld16(taddr, v); }
__device__ __forceinline__ void tm_store_row(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void tm_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// bfloat16 pair (x0 in the low half) and what it leaves of x0, x1.
__device__ __forceinline__ uint32_t last_pair(float x0, float x1) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x0, x1);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t take_pair(float& x0, float& x1) {
  const uint32_t u = last_pair(x0, x1);
  x0 -= __uint_as_float(u << 16);
  x1 -= __uint_as_float(u & 0xffff0000u);
  return u;
}

// Operand descriptors: panels read along their contiguous axis (K-major) or
// across it (MN-major: 64-wide blocks of M or N a panel apart). A step of 16
// values of k advances the address by 32 (2048) bytes. `at`: shared-memory
// address / 16. One thread issues every product, in order: the fewer
// instructions between two of them, the fuller the tensor pipe, so everything
// but `at` is a constant.
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);  // 8-row groups 1024 bytes apart, 128-byte swizzle
__device__ __forceinline__ uint64_t desc(uint32_t at, bool mn, int ks) {
  const uint32_t lo = at + (((mn ? PANEL >> 4 : 1u) << 16) + ks * (mn ? 128u : 2u));
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(DESC_HI));
  return d;
}
// d (+)= A B over 64 values of k.
template <int M, int N, bool A_MN, bool B_MN>
__device__ __forceinline__ void product(uint32_t d, uint32_t a, uint32_t b, bool accumulate) {
  constexpr uint32_t id = tc::idesc_bf16(M, N, A_MN, B_MN);
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
    const uint32_t acc = accumulate || ks > 0;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(desc(a, A_MN, ks)), "l"(desc(b, B_MN, ks)), "r"(id), "r"(acc) : "memory");
  }
}
// The same with A (M = 128) in tensor memory: two values of k a column.
template <int N, bool B_MN>
__device__ __forceinline__ void product_ta(uint32_t d, uint32_t a, uint32_t b, bool accumulate) {
  constexpr uint32_t id = tc::idesc_bf16(128, N, 0, B_MN);
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
    const uint32_t acc = accumulate || ks > 0;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a + 8 * ks), "l"(desc(b, B_MN, ks)), "r"(id), "r"(acc) : "memory");
  }
}

// NaN if `m` or one of the values is.
__device__ __forceinline__ float any_nan(float m, const float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 16; i += 2) asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(v[i]), "f"(v[i + 1]));
  return m;
}
// The outputs of a segment anew, by the recurrence. A masked score is 0, and 0
// times a value that is not finite is NaN: where the walk meets a NaN in a
// chunk's own part of its outputs, it may come from a token that the output does
// not depend on. N threads from FIRST_WARP on, each a column and ROWS rows of the
// state. Slow, for what is rare: 1.1 (64 x 64) to 1.8 us (128 x 128) a token (8
// heads x 32 rows x 1024 tokens, 64 x 128: 63 us, with one NaN 1.5 ms).
template <int DA, int DC, int FIRST_WARP, int N>
__device__ __noinline__ void by_token(const TcProblem& tp, int pass) {
  constexpr int GROUPS = N / DC, ROWS = ((DA + GROUPS - 1) / GROUPS + 3) & ~3;
  extern __shared__ float4 spare[];
  const Problem& pr = tp.pr;
  const Pass& ps = pr.pass[pass];
  const int b = int(blockIdx.x) / tp.segments, h = blockIdx.y, seg = int(blockIdx.x) % tp.segments;
  const int base = seg * tp.segment_tokens, u = int(threadIdx.x) - 32 * FIRST_WARP;
  int end = min(base + tp.segment_tokens, pr.T);
  if (pr.lengths) end = min(end, pr.lengths[b]);
  const int c = u % DC, r0 = u / DC * ROWS, da = ps.da, dc = ps.dc;
  // Shared: the state, a thread's rows by four; two each of a token's a and b and of the parts of its outputs.
  float4* state = spare + u;
  float* ab = reinterpret_cast<float*>(spare + ROWS / 4 * N);
  float* part = ab + 4 * GROUPS * ROWS;
  auto sync = [] { asm volatile("bar.sync 2, %0;" ::"n"(N) : "memory"); };
  const size_t bh = size_t(b) * pr.H + h;
  const float* init = ps.init ? ps.init + bh * da * dc : nullptr;
  int ir = ps.init_r, ic = ps.init_c;
  if (tp.segments > 1) init = tp.seg_state + pass * tp.seg_pass + (bh * tp.segments + seg) * da * dc, ir = dc, ic = 1;
  auto at_start = [&](int r) { return init && c < dc && r < da ? init[r * ir + c * ic] : 0.f; };
  for (int i = 0; i < ROWS; i += 4) {
    const int r = r0 + i;
    state[i / 4 * N] = make_float4(at_start(r), at_start(r + 1), at_start(r + 2), at_start(r + 3));
  }
  const bf16* a = operand_at<bf16>(ps.a, b, h);
  const bf16* k = operand_at<bf16>(ps.b, b, h);
  const bf16* v = operand_at<bf16>(ps.c, b, h);
  // (a reverse walk decays the state after it is read)
  const float gamma = expf(pr.log_decay[h]), before = ps.reverse ? 1.f : gamma, after = ps.reverse ? gamma : 1.f;
  float na = 0.f, nb = 0.f, nv = 0.f;  // the next token's
  auto token = [&](int n) { return int64_t(ps.reverse ? base + end - 1 - n : n); };
  auto fetch = [&](int n) {
    if (n >= end) return;
    const int64_t t = token(n);
    if (u < da) na = to_f<bf16>(a[t * ps.a.st + u]), nb = to_f<bf16>(k[t * ps.b.st + u]);
    if (c < dc) nv = ps.write_scale * to_f<bf16>(v[t * ps.c.st + c]);
  };
  fetch(base);
  for (int n = base; n <= end; ++n) {
    float* now = ab + 2 * GROUPS * ROWS * (n & 1);
    if (u < GROUPS * ROWS) now[u] = na, now[GROUPS * ROWS + u] = nb;
    const float w = nv;
    fetch(n + 1);
    sync();
    if (n > base && u < dc) {
      float o = 0.f;
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) o += part[((n - 1) & 1) * N + i * DC + u];
      const int64_t at = ((int64_t(b) * pr.T + token(n - 1)) * pr.H + h) * dc + u;
      if (ps.out_f32) static_cast<float*>(ps.out)[at] = ps.read_scale * o;
      else static_cast<bf16*>(ps.out)[at] = from_f<bf16>(ps.read_scale * o);
    }
    float o = 0.f;
#pragma unroll 2
    for (int i = 0; i < ROWS; i += 4) {
      const float4 x = ld4(now + r0 + i), y = ld4(now + GROUPS * ROWS + r0 + i);
      float4 z = state[i / 4 * N];
      z.x = fmaf(y.x, w, before * z.x), z.y = fmaf(y.y, w, before * z.y);
      z.z = fmaf(y.z, w, before * z.z), z.w = fmaf(y.w, w, before * z.w);
      o = fmaf(x.x, z.x, fmaf(x.y, z.y, fmaf(x.z, z.z, fmaf(x.w, z.w, o))));
      state[i / 4 * N] = make_float4(after * z.x, after * z.y, after * z.z, after * z.w);
    }
    part[(n & 1) * N + u] = o;
  }
}

// The walk. READ = false: only the state (a segment's own contribution).
template <int DA, int DC, bool READ>
__device__ __forceinline__ void walk(const TcProblem& tp, int pass) {
  using G = Geo<DA, DC, READ>;
  constexpr int NA = G::NA, NC = G::NC, SW = G::SW, NW = G::NW, XW = G::XW, STAGES = G::STAGES, WB = G::WB;
  extern __shared__ unsigned char raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ Bars bars;
  __shared__ uint32_t tmem_at;
  __shared__ int dead, again;
  __shared__ float pw[C + 4];                      // e^{g i}
  __shared__ float inner[2 * C];                   // e^{g gap} in_scale at gap + 63, 0 for gap < 0
  __shared__ __align__(8) float reads[2][C];       // factor of the state's read per token: a full chunk, the short one
  const Problem& pr = tp.pr;
  const Pass& ps = pr.pass[pass];
  const int b = int(blockIdx.x) / tp.segments, h = blockIdx.y, seg = int(blockIdx.x) % tp.segments;
  const int t = threadIdx.x, lane = t & 31, warp = __shfl_sync(0xffffffffu, t >> 5, 0);
  const bool rev = ps.reverse;
  int len = pr.T;
  if (pr.lengths) len = max(0, min(pr.T, pr.lengths[b]));
  const int base = seg * tp.segment_tokens, bound = min(base + tp.segment_tokens, pr.T);
  const int end = max(base, min(len, bound));
  const int chunks = (end - base + C - 1) / C;
  const int last_tokens = end - base - (chunks - 1) * C;
  const int short_chunk = last_tokens < C ? (rev ? 0 : chunks - 1) : -1;
  auto chunk_start = [&](int n) { return base + (rev ? chunks - 1 - n : n) * C; };
  auto chunk_tokens = [&](int n) { return n == short_chunk ? last_tokens : C; };
  // The chunk that holds the sequence's end before T: its tiles carry places that are not the sequence's.
  const int dirty = end == len && len < pr.T ? short_chunk : -1;

  // Chunk n's tiles into its stage (one thread).
  auto load_chunk = [&](int n) {
    const int ma = tp.map_of[pass][0], mb = tp.map_of[pass][1], mc = tp.map_of[pass][2];
    const int ha = h / ps.a.group, hb = h / ps.b.group, hc = h / ps.c.group;
    uint64_t* bar = &bars.full[n % STAGES];
    tc::mbar_expect_tx(bar, G::STAGE);
    unsigned char* st = sm + (n % STAGES) * G::STAGE;
    const int t0 = chunk_start(n);
#pragma unroll
    for (int p = 0; p < NA; ++p) tma_load_4d(st + (G::NQ + p) * PANEL, &tp.maps[mb], 64 * p, hb, t0, b, bar);
#pragma unroll
    for (int p = 0; p < NC; ++p) tma_load_4d(st + (G::NQ + NA + p) * PANEL, &tp.maps[mc], 64 * p, hc, t0, b, bar);
    if (READ)
#pragma unroll
      for (int p = 0; p < NA; ++p) tma_load_4d(st + p * PANEL, &tp.maps[ma], 64 * p, ha, t0, b, bar);
  };
  if (warp == XW + 4 + SW && lane == 0) {
    dead = again = 0;
    for (int i = 0; i < STAGES; ++i) {
      tc::mbar_init(&bars.full[i], 1);
      tc::mbar_init(&bars.empty[i], 1);
      tc::mbar_init(&bars.staged[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&bars.w_ready[i], XW);
      tc::mbar_init(&bars.ds_full[i], 1);
      tc::mbar_init(&bars.ds_free[i], SW);
      tc::mbar_init(&bars.o_full[i], 1);
      tc::mbar_init(&bars.o_free[i], 4);
    }
    tc::mbar_init(&bars.p_full, 1);
    tc::mbar_init(&bars.p_ready, XW);
    tc::mbar_init(&bars.s_ready, SW);
    tc::mbar_init(&bars.q_done, 1);
    tc::mbar_init(&bars.clean, XW);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tc::fence_proxy_async();
    // The first loads are on their way while the tables are made.
#pragma unroll 1
    for (int n = 0; n < min(chunks, STAGES); ++n) load_chunk(n);
  }
  const float g = pr.log_decay[h];
  for (int i = t; i <= C; i += G::THREADS) pw[i] = i ? expf(g * float(i)) : 1.f;
  for (int i = t; i < 2 * C; i += G::THREADS) {
    const int gap = i - (C - 1);
    inner[i] = gap < 0 ? 0.f : gap ? ps.in_scale * expf(g * float(gap)) : ps.in_scale;
    const int tokens = i < C ? C : last_tokens, e = rev ? max(tokens - 1 - (i & (C - 1)), 0) : (i & (C - 1)) + 1;
    reads[i / C][i & (C - 1)] = e ? ps.read_scale * expf(g * float(e)) : ps.read_scale;
  }
  if (warp == 0) {
    tc::tmem_alloc(&tmem_at, G::COLS);
    tc::tmem_relinquish();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tm = tmem_at;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    bar_wait(bar, parity & 1, &dead);
  };
  auto stage = [&](int n) { return (n % STAGES) * G::STAGE; };
  // Lane's part in stmatrix: row lane % 8 of matrix lane / 8 = hh + 2 (odd k).
  const int mrow = lane & 7, mh = (lane >> 3) & 1, mk = lane >> 4;
  const int gr = lane >> 2, c2 = 2 * (lane & 3);

  if (warp < XW) {
    // ---- weights of chunk n + 1, scores of chunk n --------------------------------------
    registers<G::SHARE_REGS, 64, false>();
    const uint32_t P = tc::su32(sm + G::OFF_P);
    auto weights = [&](int n) {
      const int L = chunk_tokens(n);
      wait(&bars.full[n % STAGES], n / STAGES);
      unsigned char* st = sm + stage(n);
      if (n == dirty) {  // places past the sequence: zero, whatever is there
        constexpr int VECS = G::STAGE / 16;
        for (int u = t; u < VECS; u += 32 * XW)
          if (((u >> 3) & 63) >= L) reinterpret_cast<uint4*>(st)[u] = make_uint4(0, 0, 0, 0);
        tc::fence_proxy_async();
        warp_arrive(&bars.clean, lane);
      }
      const unsigned char* X = st + (G::W_ON_K ? G::NQ : G::NQ + NA) * PANEL;
      if (n >= WB) wait(&bars.ds_full[n % WB], n / WB - 1);  // the products that read W are done
      unsigned char* W = sm + G::OFF_W + (n % WB) * 3 * G::W_TERM;
#pragma unroll 2
      for (int u = t; u < NW * PANEL / 16; u += 32 * XW) {  // 16-byte pieces of panel rows, in memory order
        const int tok = (u >> 3) & 63;
        const uint4 x = *reinterpret_cast<const uint4*>(X + 16 * u);
        const float f = ps.write_scale * pw[rev ? tok + 1 : max(L - 1 - tok, 0)];
        uint32_t in[4] = {x.x, x.y, x.z, x.w}, w1[4], w2[4], w3[4];
        if (n == dirty && tok >= L) in[0] = in[1] = in[2] = in[3] = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float x0 = f * __uint_as_float(in[k] << 16), x1 = f * __uint_as_float(in[k] & 0xffff0000u);
          w1[k] = take_pair(x0, x1);
          w2[k] = take_pair(x0, x1);
          w3[k] = last_pair(x0, x1);
        }
        *reinterpret_cast<uint4*>(W + 16 * u) = make_uint4(w1[0], w1[1], w1[2], w1[3]);
        *reinterpret_cast<uint4*>(W + G::W_TERM + 16 * u) = make_uint4(w2[0], w2[1], w2[2], w2[3]);
        *reinterpret_cast<uint4*>(W + 2 * G::W_TERM + 16 * u) = make_uint4(w3[0], w3[1], w3[2], w3[3]);
      }
      tc::fence_proxy_async();
      warp_arrive(&bars.w_ready[n % WB], lane);
    };
    // (one place for the weights' code: chunk n's scores, then chunk n + 1's weights)
#pragma unroll 1
    for (int n = -1; n < chunks; ++n) {
      if (READ && n >= 0) {
        wait(&bars.p_full, n);
        tc::fence_after();
        const int q = warp & 3;
        // Column c of row r: factor inner[63 + (r - c)], or (c - r) in a reverse walk.
        const int step = rev ? 1 : -1, first = C - 1 + (rev ? c2 - 16 * q - gr : 16 * q + gr - c2);
#pragma unroll 1
        for (int c0 = XW == 8 ? 32 * (warp >> 2) : 0; c0 < C; c0 += XW == 8 ? C : 32) {  // 32 columns at a time
          float v[16];
          tm_load(tm + (G::OB == 2 ? G::OSET * (n & 1) : 0) + c0 + (uint32_t(32 * q) << 16), v);
          tc::wait_ld();
          uint32_t hi[8], lo[8];
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              const float* f = inner + first + step * (c0 + 8 * k - 8 * hh);
              float x0 = v[4 * k + 2 * hh] * f[0], x1 = v[4 * k + 2 * hh + 1] * f[step];
              hi[2 * k + hh] = take_pair(x0, x1);
              lo[2 * k + hh] = last_pair(x0, x1);
            }
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            const uint32_t at = P + tc::sw(16 * q + 8 * mh + mrow, c0 + 8 * (k + mk));
            stm4(at, hi[2 * k], hi[2 * k + 1], hi[2 * k + 2], hi[2 * k + 3]);
            stm4(at + PANEL, lo[2 * k], lo[2 * k + 1], lo[2 * k + 2], lo[2 * k + 3]);
          }
        }
        tc::fence_before();
        tc::fence_proxy_async();
        warp_arrive(&bars.p_ready, lane);
      }
      if (n + 1 < chunks) weights(n + 1);
    }
  } else if (warp < XW + 4) {
    // ---- outputs: O = O1 + e^{g ..} O2 ----------------------------------------------------
    registers<G::SHARE_REGS, 104, true>();
    if constexpr (READ) {
      const int q = warp & 3, u0 = t - 32 * XW;
      const int64_t row = int64_t(pr.H) * ps.dc;
      const int64_t out0 = int64_t(b) * pr.T * row + int64_t(h) * ps.dc;
      float nan = 0.f;
      for (int n = 0; n < chunks; ++n) {
        const int t0 = chunk_start(n), L = chunk_tokens(n);
        unsigned char* st = sm + stage(n);
        const float* factor = reads[n == short_chunk];
        const uint32_t acc = tm + G::COL_O + G::OSET * (n % G::OB) + (uint32_t(32 * q) << 16);
        wait(&bars.o_full[n % G::OB], n / G::OB);
        tc::fence_after();
        // 16 head-dim rows x 32 tokens at a time.
#pragma unroll 1
        for (int part = 0; part < 2 * NC; ++part) {
          const int c0 = 32 * (part & 1), hb = part >> 1;
          float o1[16], o2[16];
          tm_load(acc + c0 + (uint32_t(16 * hb) << 16), o1);
          tm_load(acc + G::O1 + c0 + (uint32_t(16 * hb) << 16), o2);
          float e1[16], e2[16];
          if (!G::S_TMEM) tm_load(acc + G::O1 + c0 + (16u << 16), e2);
          if (G::P_WIDE) tm_load(acc + 64 + c0, e1);
          tc::wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (!G::S_TMEM) o2[i] += e2[i];
            if (G::P_WIDE) o1[i] += e1[i];
          }
          if (part == 2 * NC - 1) {
            tc::fence_before();
            warp_arrive(&bars.o_free[n % G::OB], lane);
          }
          nan = any_nan(nan, o1);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = *reinterpret_cast<const float2*>(factor + c0 + 8 * k + c2);
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              o1[4 * k + 2 * hh] = fmaf(f.x, o2[4 * k + 2 * hh], o1[4 * k + 2 * hh]);
              o1[4 * k + 2 * hh + 1] = fmaf(f.y, o2[4 * k + 2 * hh + 1], o1[4 * k + 2 * hh + 1]);
            }
          }
          const int r0 = NC == 2 ? 32 * q + 16 * hb : 16 * q;  // first head-dim row
          if (n == dirty)  // zeros past the sequence, whatever the state holds
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (c0 + 8 * (i >> 2) + c2 + (i & 1) >= L) o1[i] = 0.f;
          if (ps.out_f32) {
            float* tile = reinterpret_cast<float*>(st) + (c0 + c2) * DC + r0 + gr;
#pragma unroll
            for (int i = 0; i < 16; ++i) tile[(8 * (i >> 2) + (i & 1)) * DC + 8 * ((i >> 1) & 1)] = o1[i];
          } else {
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
              const int d = r0 + 8 * mh;
              const uint32_t at = tc::su32(st) + (d >> 6) * PANEL + tc::sw(c0 + 8 * (k + mk) + mrow, d & 63);
              stm4_trans(at, last_pair(o1[4 * k], o1[4 * k + 1]), last_pair(o1[4 * k + 2], o1[4 * k + 3]),
                         last_pair(o1[4 * k + 4], o1[4 * k + 5]), last_pair(o1[4 * k + 6], o1[4 * k + 7]));
            }
          }
        }
        if (ps.out_f32) {  // (a part of a shared head's gradient)
          output_sync();
          float* out = static_cast<float*>(ps.out) + out0 + int64_t(t0) * row;
          const int rows = n == dirty ? min(C, pr.T - t0) : L;
#pragma unroll 1
          for (int u = u0; u < C * DC / 4; u += 128) {
            const int tok = u / (DC / 4), d = 4 * (u % (DC / 4));
            if (tok < rows && d < ps.dc) st4(out + tok * row + d, reinterpret_cast<const float4*>(st)[u]);
          }
        }
        tc::fence_proxy_async();
        warp_arrive(&bars.staged[n % STAGES], lane);
      }
      if (nan != nan) again = 1;
    }
  } else if (warp < XW + 4 + SW) {
    // ---- the state ----------------------------------------------------------------------
    registers<G::SHARE_REGS, 104, true>();
    const int w = warp - XW - 4, q = w & 3, c0 = (w >> 2) * G::SC;
    const size_t bh = (size_t(b) * pr.H + h);
    float* seg_at = tp.seg_state ? tp.seg_state + pass * tp.seg_pass + (bh * tp.segments + seg) * ps.da * ps.dc : nullptr;
    const float* init = nullptr;
    int ir = ps.dc, ic = 1;
    if (READ) {
      init = tp.segments > 1 ? seg_at : ps.init;
      if (tp.segments == 1 && init) init += bh * ps.da * ps.dc, ir = ps.init_r, ic = ps.init_c;
    }
    float* fin = READ ? (tp.segments == 1 ? ps.fin : nullptr) : seg_at;
    if (READ && fin) fin += bh * ps.da * ps.dc;
    if (READ) after_previous();  // (the segments' states; all else was there before the kernels that make them)
    if constexpr (G::S_TMEM) {
      // Row dv of S^T in one thread, SC of its columns.
      const int dv = 32 * q + lane;
      const uint32_t ln = uint32_t(32 * q) << 16;
      float s[G::SC];
#pragma unroll
      for (int i = 0; i < G::SC; ++i) s[i] = 0.f;
      if (init && dv < ps.dc) {
        const float* at = init + c0 * ir + dv * ic;
#pragma unroll
        for (int i = 0; i < G::SC; ++i, at += ir)
          if (c0 + (i & ~7) < ps.da) s[i] = *at;  // (dims are multiples of 8)
      }
      for (int n = 0; n < chunks; ++n) {
        if constexpr (READ) {
          if (n) wait(&bars.q_done, n - 1);  // the products that read the terms are done
          tc::fence_after();
#pragma unroll
          for (int i = 0; i < G::SC; i += 16) {
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int m = 0; m < 8; ++m) {
              float x0 = s[i + 2 * m], x1 = s[i + 2 * m + 1];
              hi[m] = take_pair(x0, x1);
              lo[m] = last_pair(x0, x1);
            }
            tm_store_row(tm + G::COL_A + (c0 + i) / 2 + ln, hi);
            tm_store_row(tm + G::COL_A + DA / 2 + (c0 + i) / 2 + ln, lo);
          }
          tm_wait_store();
          tc::fence_before();
          warp_arrive(&bars.s_ready, lane);
        }
        const float f = pw[chunk_tokens(n)];
        wait(&bars.ds_full[n % WB], n / WB);
        tc::fence_after();
#pragma unroll
        for (int i = 0; i < G::SC; i += 16) {
          float v[16];
          tm_load_row(tm + G::COL_S + DA * (n % WB) + c0 + i + ln, v);
          tc::wait_ld();
          if (i + 16 >= G::SC) {
            tc::fence_before();
            warp_arrive(&bars.ds_free[n % WB], lane);
          }
#pragma unroll
          for (int k = 0; k < 16; ++k) s[i + k] = fmaf(f, s[i + k], v[k]);
        }
      }
      if (fin && dv < ps.dc) {
        float* at = fin + c0 * ps.dc + dv;
#pragma unroll
        for (int i = 0; i < G::SC; ++i, at += ps.dc)
          if (c0 + (i & ~7) < ps.da) *at = s[i];
      }
    } else {
      // 16 rows x SC columns a warp: s[4 k + 2 hh + j] is row 16 q + gr + 8 hh, column c0 + 8 k + c2 + j.
      constexpr int NG = G::SC / 8;
      const uint32_t S = tc::su32(sm + G::OFF_S);
      float s[4 * NG];
#pragma unroll
      for (int i = 0; i < 4 * NG; ++i) {
        const int dv = 16 * q + gr + 8 * ((i >> 1) & 1), d = c0 + 8 * (i >> 2) + c2 + (i & 1);
        s[i] = init && dv < ps.dc && d < ps.da ? init[d * ir + dv * ic] : 0.f;
      }
      for (int n = 0; n < chunks; ++n) {
        if constexpr (READ) {
          if (n) wait(&bars.q_done, n - 1);  // the products that read the terms are done
#pragma unroll
          for (int k = 0; k < NG; k += 2) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              float x0 = s[4 * k + 2 * m], x1 = s[4 * k + 2 * m + 1];
              hi[m] = take_pair(x0, x1);
              lo[m] = last_pair(x0, x1);
            }
            const int d = c0 + 8 * (k + mk);
            const uint32_t at = S + (d >> 6) * G::S_ROWS + tc::sw(32 * q + 8 * mh + mrow, d & 63);
            stm4(at, hi[0], hi[1], hi[2], hi[3]);
            stm4(at + 16 * 128, lo[0], lo[1], lo[2], lo[3]);  // 16 rows on: the same swizzle
          }
          tc::fence_proxy_async();
          warp_arrive(&bars.s_ready, lane);
        }
        const float f = pw[chunk_tokens(n)];
        wait(&bars.ds_full[n % WB], n / WB);
        tc::fence_after();
        float v[NG / 4][16];
#pragma unroll
        for (int k = 0; k < NG; k += 4) tm_load(tm + G::COL_S + DA * (n % WB) + c0 + 8 * k + (uint32_t(32 * q) << 16), v[k / 4]);
        tc::wait_ld();
        tc::fence_before();
        warp_arrive(&bars.ds_free[n % WB], lane);
#pragma unroll
        for (int i = 0; i < 4 * NG; ++i) s[i] = fmaf(f, s[i], v[i >> 4][i & 15]);
      }
      if (fin)
#pragma unroll
        for (int i = 0; i < 4 * NG; ++i) {
          const int dv = 16 * q + gr + 8 * ((i >> 1) & 1), d = c0 + 8 * (i >> 2) + c2 + (i & 1);
          if (dv < ps.dc && d < ps.da) fin[d * ps.dc + dv] = s[i];
        }
    }
  } else {
   registers<G::SHARE_REGS, 40, false>();
   if (warp == XW + 4 + SW) {
    // ---- TMA ----------------------------------------------------------------------------
    if (lane == 0) {
      int n = min(chunks, STAGES);
      for (; n < chunks; ++n) {
        wait(&bars.empty[n % STAGES], n / STAGES - 1);
        if (*static_cast<volatile int*>(&dead)) break;
        load_chunk(n);
      }
      // Before the CTA ends: no copy in flight, and every stage's last use done (its barrier arrived).
      for (int m = max(0, n - STAGES); m < n; ++m) {
        tc::mbar_wait(&bars.full[m % STAGES], (m / STAGES) & 1, 1 << 16);
        wait(&bars.empty[m % STAGES], m / STAGES);
      }
    }
   } else if (warp == XW + 4 + SW + 2) {
    // ---- output tiles to memory (places past T or the head dim are clipped) -----------------
    if (READ && lane == 0) {
      for (int n = 0; n < chunks; ++n) {
        wait(&bars.staged[n % STAGES], n / STAGES);
        if (!ps.out_f32) {
          const int t0 = chunk_start(n);
#pragma unroll
          for (int p = 0; p < NC; ++p) tma_store_4d(&tp.out_maps[pass], sm + stage(n) + p * PANEL, 64 * p, h, t0, b);
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        }
        bar_arrive(&bars.empty[n % STAGES]);
      }
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
   } else if (warp == XW + 4 + SW + 1) {
    // ---- products -------------------------------------------------------------------------
    if (elect_one()) {
      // Shared-memory places in units of 16 bytes.
      constexpr uint32_t PN = PANEL >> 4;
      const uint32_t s0 = tc::su32(sm) >> 4, P = s0 + (G::OFF_P >> 4), W = s0 + (G::OFF_W >> 4), S = s0 + (G::OFF_S >> 4);
#pragma unroll 1
      for (int n = 0; n < chunks; ++n) {
        const uint32_t Q = s0 + (stage(n) >> 4), K = Q + G::NQ * PN, V = K + NA * PN;
        const uint32_t acc = tm + G::COL_O + G::OSET * (n % G::OB);
        wait(&bars.full[n % STAGES], n / STAGES);
        if (n == dirty) wait(&bars.clean, 0);
        if constexpr (READ) {
          if (G::OB == 2 && n >= 2) wait(&bars.o_free[n & 1], n / 2 - 1);
          tc::fence_after();
#pragma unroll
          for (int p = 0; p < NA; ++p)
            product<64, 64, false, false>(G::OB == 2 ? acc : tm, Q + p * PN, K + p * PN, p > 0);
          tc::commit(&bars.p_full);
        }
        wait(&bars.w_ready[n % WB], n / WB);
        if (n >= WB) wait(&bars.ds_free[n % WB], n / WB - 1);
        tc::fence_after();
        auto add = [&](int term) {
          const uint32_t w = W + ((n % WB) * 3 + term) * (G::W_TERM >> 4);
          product<DC, DA, true, true>(tm + G::COL_S + DA * (n % WB), G::W_ON_K ? V : w, G::W_ON_K ? w : K, term > 0);
        };
        add(0);
        add(1);
        add(2);
        tc::commit(&bars.ds_full[n % WB]);
        if constexpr (READ) {
          wait(&bars.s_ready, n);
          if (G::OB == 1 && n) wait(&bars.o_free[0], n - 1);
          tc::fence_after();
          if constexpr (G::S_TMEM) {
#pragma unroll
            for (int i = 0; i < 2 * NA; ++i)  // terms, panels
              product_ta<64, false>(acc + G::O1, tm + G::COL_A + (i / NA) * (DA / 2) + 32 * (i % NA), Q + (i % NA) * PN,
                                    i > 0);
          } else {
#pragma unroll
            for (int p = 0; p < NA; ++p)
              product<128, 64, false, false>(acc + G::O1, S + p * (G::S_ROWS >> 4), Q + p * PN, p > 0);
          }
          tc::commit(&bars.q_done);
          wait(&bars.p_ready, n);
          tc::fence_after();
          if constexpr (G::P_WIDE) {
            product<DC, 128, true, false>(acc, V, P, false);
          } else {
#pragma unroll
            for (int term = 0; term < 2; ++term) product<DC, 64, true, false>(acc, V, P + term * PN, term > 0);
          }
          tc::commit(&bars.o_full[n % G::OB]);
        } else {
          tc::commit(&bars.empty[n % STAGES]);
        }
      }
    }
   }
  }
  // Rows of this segment past its chunks: zero, a warp a row. (Those past the
  // sequence within its last chunk are in that chunk's tile.)
  if (READ && len < bound) {
    const int64_t row = int64_t(pr.H) * ps.dc, out0 = int64_t(b) * pr.T * row + int64_t(h) * ps.dc;
    const int size = ps.out_f32 ? 4 : 2, pieces = ps.dc * size / 16;  // (dims are multiples of 8)
    for (int r = base + chunks * C + warp; r < bound; r += G::THREADS / 32)
      for (int i = lane; i < pieces; i += 32)
        reinterpret_cast<uint4*>(static_cast<char*>(ps.out) + (out0 + r * row) * size)[i] = make_uint4(0, 0, 0, 0);
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 0) tc::tmem_dealloc(tm, G::COLS);
  if (t == 0 && dead) tc::flag_timeout();
  // (the warps with the most registers)
  if (READ && again && !dead && warp >= XW && warp < XW + 4 + SW)
    by_token<DA, DC, XW, 32 * (4 + SW)>(tp, pass);
}

template <int DA, int DC, bool READ>
__global__ void __launch_bounds__(Geo<DA, DC, READ>::THREADS, Geo<DA, DC, READ>::SMALL ? 2 : 1)
    walk_tc(const __grid_constant__ TcProblem tp) {
  walk<DA, DC, READ>(tp, int(blockIdx.z));
}
// Passes of both mixed shapes in one launch (a backward pass with unequal
// dims): no wave of idle SMs between them.
template <bool READ>
__global__ void __launch_bounds__(Geo<64, 128, READ>::THREADS, 1)
    walk_mixed(const __grid_constant__ TcProblem tp) {
  static_assert(int(Geo<64, 128, READ>::THREADS) == int(Geo<128, 64, READ>::THREADS), "one block size");
  const int pass = int(blockIdx.z);
  if (tp.pr.pass[pass].da > 64) walk<128, 64, READ>(tp, pass);
  else walk<64, 128, READ>(tp, pass);
}

// Segment ends (walked from zero) -> the states at segment starts, and the
// state after the whole walk.
__global__ void __launch_bounds__(256) join_segments(const __grid_constant__ TcProblem tp) {
  const Problem& pr = tp.pr;
  const Pass& ps = pr.pass[blockIdx.z];
  const int n = ps.da * ps.dc, i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  after_previous();
  const size_t bh = blockIdx.y;
  const int b = int(bh) / pr.H, h = int(bh) % pr.H;
  int len = pr.T;
  if (pr.lengths) len = max(0, min(pr.T, pr.lengths[b]));
  const float g = pr.log_decay[h];
  const int r = i / ps.dc, c = i - r * ps.dc;
  float s = ps.init ? ps.init[bh * n + r * ps.init_r + c * ps.init_c] : 0.f;
  float* seg = tp.seg_state + blockIdx.z * tp.seg_pass + bh * tp.segments * n + i;
  for (int k0 = 0; k0 < tp.segments; k0 += 8) {
    float local[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int k = k0 + u, at = ps.reverse ? tp.segments - 1 - k : k;
      local[u] = k < tp.segments ? seg[size_t(at) * n] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int k = k0 + u, at = ps.reverse ? tp.segments - 1 - k : k;
      if (k >= tp.segments) break;
      const int base = at * tp.segment_tokens;
      const int tokens = max(0, min(len, base + tp.segment_tokens) - base);
      seg[size_t(at) * n] = s;
      s = fmaf(tokens ? expf(g * float(tokens)) : 1.f, s, local[u]);
    }
  }
  if (ps.fin) ps.fin[bh * n + i] = s;
}

}  // namespace decay
}  // namespace m4
