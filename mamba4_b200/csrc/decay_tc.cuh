// Decay attention on the fifth-generation tensor cores: bfloat16 operands.
//
// One CTA walks the chunks of one (pass, batch row, head, segment of the time
// axis); see decay.cu for the recurrence. Everything with a head dim in its
// rows is computed transposed, so that 128-wide head dims fill the 128 lanes
// of tensor memory with chunks of 64 tokens:
//   P   [t, s]    = Q K^T                          (64 x 64)
//   O1^T[dv, t]   = V^T P'^T,  P' = masked, decayed P in two bfloat16 terms
//   O2^T[dv, t]   = S^T Q^T,   S^T [dv, dk] the state before, in two terms
//   dS^T[dv, dk]  = (w V)^T K, w V the weighted values in three terms
// (an fp32 factor times a bfloat16 value has 32 significant bits; two terms
// keep 16 of them, which leaves a bfloat16 output with its own rounding only,
// three keep 24, the state's float32). The running state stays in registers
// in float32: S' = e^{g L} S + dS, so chunks join with one rounding each.
//
// Warps: 4 score/output warps, SW state warps, 4 value warps, one for TMA,
// one that issues the products. They meet on mbarriers only; every wait is
// bounded. Tiles are [64 tokens][64 columns] panels with the 128-byte swizzle.
//
// Bound by HBM when heads and rows fill the GPU: a chunk moves 4 x 8 KB per 64
// columns, the products take about half that time on the tensor pipe.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "tc05.cuh"

namespace m4 {
namespace decay {

constexpr int PANEL = 64 * 128;  // bytes of a [64][64] bfloat16 panel
constexpr int STAGES = 2;

struct alignas(64) TcProblem {
  CUtensorMap maps[4];
  Problem pr;
  int map_of[3][3];     // tensor map of each pass's a, b, c
  int segments, segment_tokens;
  float* seg_state;     // [passes][B][H][segments][da][dc]: states at segment starts (phase 1: at their ends)
  size_t seg_pass;      // floats per pass in seg_state
};

template <int DA, int DC>
struct Geo {
  static constexpr int NA = DA / 64, NC = DC / 64;
  static constexpr int STAGE = (2 * NA + NC) * PANEL;
  static constexpr int SW = DA * DC >= 8192 ? 8 : 4;      // state warps
  static constexpr int THREADS = 32 * (4 + SW + 4 + 2);
  static constexpr int S_TERM = DC * DA * 2;              // one bfloat16 term of S^T
  static constexpr int W_TERM = NC * PANEL;
  static constexpr int OFF_P = STAGES * STAGE;            // two panels; the output tile afterwards
  static constexpr int P_BYTES = 2 * PANEL;
  static constexpr int OFF_W = OFF_P + P_BYTES;
  static constexpr int OFF_S = OFF_W + 3 * W_TERM;
  static constexpr int BYTES = OFF_S + 2 * S_TERM;
  static constexpr int SMEM = BYTES + 1024;
  // Tensor-memory columns.
  static constexpr int COL_P = 0, COL_O1 = 64, COL_O2 = 128, COL_S = 192;
  static constexpr int COLS = COL_S + DA <= 256 ? 256 : 512;
  // State registers: per warp HB blocks of 16 rows x SC columns.
  static constexpr int HB = DC / 64, SC = DA / (SW / 4);
};

struct Bars {
  uint64_t full[STAGES], empty[STAGES];
  uint64_t p_full, p_ready, w_ready, s_full, s_ready, o_full, o_free, clean;
};

__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::su32(bar)) : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const void* map, int c0, int c1, int c2, int c3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(tc::su32(dst)), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(tc::su32(bar)) : "memory");
}
// Named barrier of the 128 score/output threads.
__device__ __forceinline__ void group_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

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
// bfloat16 pair (x0 in the low half) and what it leaves of x0, x1.
__device__ __forceinline__ uint32_t take_pair(float& x0, float& x1) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x0, x1);
  const uint32_t u = *reinterpret_cast<const uint32_t*>(&h);
  x0 -= __uint_as_float(u << 16);
  x1 -= __uint_as_float(u & 0xffff0000u);
  return u;
}
__device__ __forceinline__ uint32_t last_pair(float x0, float x1) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x0, x1);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// d (+)= A B over 64 values of k, four products of 16; operands are panels
// read along their contiguous axis (K-major) or across it (MN-major; 64-wide
// blocks of M or N one panel apart).
template <int M, int N, bool A_MN, bool B_MN>
__device__ __forceinline__ void product(uint32_t d, const unsigned char* a, const unsigned char* b, bool accumulate) {
  constexpr uint32_t id = tc::idesc_bf16(M, N, A_MN, B_MN);
#pragma unroll 1
  for (int ks = 0; ks < 4; ++ks)
    tc::mma_bf16(d, A_MN ? tc::sdesc_sw128(a + 2048 * ks, PANEL, 1024) : tc::sdesc_sw128(a + 32 * ks, 16, 1024),
                 B_MN ? tc::sdesc_sw128(b + 2048 * ks, PANEL, 1024) : tc::sdesc_sw128(b + 32 * ks, 16, 1024), id,
                 accumulate || ks > 0);
}

// The walk. READ = false: only the state (a segment's own contribution).
template <int DA, int DC, bool READ>
__global__ void __launch_bounds__(Geo<DA, DC>::THREADS, DA + DC == 128 ? 2 : 1)
    walk_tc(const __grid_constant__ TcProblem tp, int first_pass) {
  using G = Geo<DA, DC>;
  constexpr int NA = G::NA, NC = G::NC, SW = G::SW;
  extern __shared__ unsigned char raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ Bars bars;
  __shared__ uint32_t tmem_at;
  __shared__ int dead;
  __shared__ float pw[C + 4];            // e^{g i}
  __shared__ float inner[2 * C];         // e^{g gap} in_scale at gap + 63, 0 for gap < 0
  const Problem& pr = tp.pr;
  const int pass = first_pass + int(blockIdx.z);
  const Pass& ps = pr.pass[pass];
  const int b = int(blockIdx.x) / tp.segments, h = blockIdx.y, seg = int(blockIdx.x) % tp.segments;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const bool rev = ps.reverse;
  int len = pr.T;
  if (pr.lengths) len = max(0, min(pr.T, pr.lengths[b]));
  const int base = seg * tp.segment_tokens, bound = min(base + tp.segment_tokens, pr.T);
  const int end = max(base, min(len, bound));
  const int chunks = (end - base + C - 1) / C;
  const int last_tokens = end - base - (chunks - 1) * C;
  auto chunk_start = [&](int n) { return base + (rev ? chunks - 1 - n : n) * C; };
  auto chunk_tokens = [&](int n) { return (rev ? n == 0 : n == chunks - 1) ? last_tokens : C; };
  // The chunk that holds the sequence's end before T: its tiles carry places that are not the sequence's.
  const int dirty = end == len && len < pr.T && last_tokens < C && chunks > 0 ? (rev ? 0 : chunks - 1) : -1;

  const float g = pr.log_decay[h];
  for (int i = t; i <= C; i += G::THREADS) pw[i] = i ? expf(g * float(i)) : 1.f;
  for (int i = t; i < 2 * C; i += G::THREADS) {
    const int gap = i - (C - 1);
    inner[i] = gap < 0 ? 0.f : gap ? ps.in_scale * expf(g * float(gap)) : ps.in_scale;
  }
  if (t == 0) {
    dead = 0;
    for (int i = 0; i < STAGES; ++i) tc::mbar_init(&bars.full[i], 1), tc::mbar_init(&bars.empty[i], 1);
    tc::mbar_init(&bars.p_full, 1);
    tc::mbar_init(&bars.p_ready, 128);
    tc::mbar_init(&bars.w_ready, 128);
    tc::mbar_init(&bars.s_full, 1);
    tc::mbar_init(&bars.s_ready, 32 * SW);
    tc::mbar_init(&bars.o_full, 1);
    tc::mbar_init(&bars.o_free, 128);
    tc::mbar_init(&bars.clean, 128);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tc::fence_proxy_async();
  }
  if (warp == 0) {
    tc::tmem_alloc(&tmem_at, G::COLS);
    tc::tmem_relinquish();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tm = tmem_at;
  volatile int* gone = &dead;
  // Bounded wait; after one has given up, none waits any more.
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (*gone) return;
    if (!tc::mbar_wait(bar, parity & 1, tc::WAIT_LIMIT)) {
      *gone = 1;
      tc::flag_timeout();
    }
  };
  auto stage = [&](int n) { return sm + (n % STAGES) * G::STAGE; };

  if (warp < 4) {
    // ---- scores and outputs -------------------------------------------------------------
    if constexpr (READ) {
      const int q = warp, gr = lane >> 2, c2 = 2 * (lane & 3);
      unsigned char* P = sm + G::OFF_P;
      // stmatrix rows of this lane: matrix lane / 8 = hh + 2 (k odd), row lane % 8.
      const int mrow = lane & 7, mh = (lane >> 3) & 1, mk = lane >> 4;
      const int64_t row = int64_t(pr.H) * ps.dc;
      const int64_t out0 = int64_t(b) * pr.T * row + int64_t(h) * ps.dc;
      for (int n = 0; n < chunks; ++n) {
        const int t0 = chunk_start(n), L = chunk_tokens(n);
        wait(&bars.p_full, n);
        tc::fence_after();
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float v[16];
          tm_load(tm + G::COL_P + 32 * half + (uint32_t(32 * q) << 16), v);
          tc::wait_ld();
          uint32_t hi[8], lo[8];
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              const int r = 16 * q + gr + 8 * hh, c = 32 * half + 8 * k + c2;
              const int gap = rev ? c - r : r - c, step = rev ? 1 : -1;
              float x0 = v[4 * k + 2 * hh] * inner[gap + C - 1];
              float x1 = v[4 * k + 2 * hh + 1] * inner[gap + step + C - 1];
              hi[2 * k + hh] = take_pair(x0, x1);
              lo[2 * k + hh] = last_pair(x0, x1);
            }
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            const uint32_t at = tc::sw(16 * q + 8 * mh + mrow, 32 * half + 8 * (k + mk));
            stm4(tc::su32(P) + at, hi[2 * k], hi[2 * k + 1], hi[2 * k + 2], hi[2 * k + 3]);
            stm4(tc::su32(P) + PANEL + at, lo[2 * k], lo[2 * k + 1], lo[2 * k + 2], lo[2 * k + 3]);
          }
        }
        tc::fence_before();
        tc::fence_proxy_async();
        bar_arrive(&bars.p_ready);
        wait(&bars.o_full, n);
        tc::fence_after();
        // O = O1 + e^{g ..} O2, 16 head-dim rows x 32 tokens at a time.
#pragma unroll
        for (int hb = 0; hb < G::HB; ++hb) {
          const int r0 = G::HB == 2 ? 32 * q + 16 * hb : 16 * q;  // first row; its tensor-memory lane:
          const uint32_t ln = uint32_t(32 * q + 16 * hb) << 16;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float o1[16], o2[16];
            tm_load(tm + G::COL_O1 + 32 * half + ln, o1);
            tm_load(tm + G::COL_O2 + 32 * half + ln, o2);
            tc::wait_ld();
            if (hb == G::HB - 1 && half == 1) {
              tc::fence_before();
              bar_arrive(&bars.o_free);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const int tok = 32 * half + 8 * k + c2 + j;
                const float f = ps.read_scale * pw[rev ? max(L - 1 - tok, 0) : tok + 1];
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) o1[4 * k + 2 * hh + j] += f * o2[4 * k + 2 * hh + j];
              }
            if (ps.out_f32) {
              float* out = static_cast<float*>(ps.out);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int tok = 32 * half + 8 * (i >> 2) + c2 + (i & 1), d = r0 + gr + 8 * ((i >> 1) & 1);
                if (tok < L && d < ps.dc) out[out0 + (t0 + tok) * row + d] = o1[i];
              }
            } else {
#pragma unroll
              for (int k = 0; k < 4; k += 2) {
                const int d = r0 + 8 * mh;
                const uint32_t at = tc::su32(P) + (d >> 6) * PANEL + tc::sw(32 * half + 8 * (k + mk) + mrow, d & 63);
                stm4_trans(at, last_pair(o1[4 * k], o1[4 * k + 1]), last_pair(o1[4 * k + 2], o1[4 * k + 3]),
                           last_pair(o1[4 * k + 4], o1[4 * k + 5]), last_pair(o1[4 * k + 6], o1[4 * k + 7]));
              }
            }
          }
        }
        if (!ps.out_f32) {
          group_sync();
          bf16* out = static_cast<bf16*>(ps.out) + out0 + int64_t(t0) * row;
#pragma unroll
          for (int i = 0; i < 4 * NC; ++i) {
            const int u = i * 128 + t, tok = u / (8 * NC), d = 8 * (u % (8 * NC));
            const uint4 x = *reinterpret_cast<const uint4*>(P + (d >> 6) * PANEL + tc::sw(tok, d & 63));
            if (tok < L && d < ps.dc) *reinterpret_cast<uint4*>(out + tok * row + d) = x;
          }
          group_sync();
        }
      }
    }
  } else if (warp < 4 + SW) {
    // ---- the state ----------------------------------------------------------------------
    const int w = warp - 4, q = w & 3, c0 = (w >> 2) * G::SC, gr = lane >> 2, c2 = 2 * (lane & 3);
    constexpr int HB = G::HB, NG = G::SC / 8;  // blocks of 16 rows, groups of 8 columns
    const int mrow = lane & 7, mh = (lane >> 3) & 1, mk = lane >> 4;
    float s[HB][4 * NG];  // [..][4 k + 2 hh + j]: S^T row r0 + gr + 8 hh, column c0 + 8 k + c2 + j
    const size_t bh = (size_t(b) * pr.H + h);
    float* seg_at = tp.seg_state ? tp.seg_state + pass * tp.seg_pass + (bh * tp.segments + seg) * ps.da * ps.dc : nullptr;
    const float* init = nullptr;
    int ir = ps.dc, ic = 1;
    if (READ) {
      init = tp.segments > 1 ? seg_at : ps.init;
      if (tp.segments == 1 && init) init += bh * ps.da * ps.dc, ir = ps.init_r, ic = ps.init_c;
    }
    auto row0 = [&](int hb) { return HB == 2 ? 32 * q + 16 * hb : 16 * q; };
#pragma unroll
    for (int hb = 0; hb < HB; ++hb)
#pragma unroll
      for (int i = 0; i < 4 * NG; ++i) {
        const int dv = row0(hb) + gr + 8 * ((i >> 1) & 1), d = c0 + 8 * (i >> 2) + c2 + (i & 1);
        s[hb][i] = init && dv < ps.dc && d < ps.da ? init[d * ir + dv * ic] : 0.f;
      }
    unsigned char* S = sm + G::OFF_S;
    for (int n = 0; n < chunks; ++n) {
      if constexpr (READ) {
#pragma unroll
        for (int hb = 0; hb < HB; ++hb)
#pragma unroll
          for (int k = 0; k < NG; k += 2) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              float x0 = s[hb][4 * k + 2 * m], x1 = s[hb][4 * k + 2 * m + 1];
              hi[m] = take_pair(x0, x1);
              lo[m] = last_pair(x0, x1);
            }
            const int d = c0 + 8 * (k + mk);
            const uint32_t at =
                tc::su32(S) + (d >> 6) * (DC * 128) + tc::sw(row0(hb) + 8 * mh + mrow, d & 63);
            stm4(at, hi[0], hi[1], hi[2], hi[3]);
            stm4(at + G::S_TERM, lo[0], lo[1], lo[2], lo[3]);
          }
        tc::fence_proxy_async();
      }
      tc::fence_before();
      bar_arrive(&bars.s_ready);
      const float f = pw[chunk_tokens(n)];
      wait(&bars.s_full, n);
      tc::fence_after();
#pragma unroll
      for (int hb = 0; hb < HB; ++hb)
#pragma unroll
        for (int k = 0; k < NG; k += 4) {
          float v[16];
          tm_load(tm + G::COL_S + c0 + 8 * k + (uint32_t(32 * q + 16 * hb) << 16), v);
          tc::wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) s[hb][4 * k + i] = fmaf(f, s[hb][4 * k + i], v[i]);
        }
    }
    float* fin = READ ? (tp.segments == 1 ? ps.fin : nullptr) : seg_at;
    if (READ && fin) fin += bh * ps.da * ps.dc;
    if (fin) {
#pragma unroll
      for (int hb = 0; hb < HB; ++hb)
#pragma unroll
        for (int i = 0; i < 4 * NG; ++i) {
          const int dv = row0(hb) + gr + 8 * ((i >> 1) & 1), d = c0 + 8 * (i >> 2) + c2 + (i & 1);
          if (dv < ps.dc && d < ps.da) fin[d * ps.dc + dv] = s[hb][i];
        }
    }
  } else if (warp < 8 + SW) {
    // ---- weighted values ----------------------------------------------------------------
    const int u0 = t - 32 * (4 + SW);
    unsigned char* W = sm + G::OFF_W;
    for (int n = 0; n < chunks; ++n) {
      const int L = chunk_tokens(n);
      wait(&bars.full[n % STAGES], n / STAGES);
      unsigned char* st = stage(n);
      if (n == dirty) {  // places past the sequence: zero, whatever is there
        constexpr int VECS = (2 * NA + NC) * PANEL / 16;
        for (int u = u0; u < VECS; u += 128) {
          const int tok = (u * 16 / 128) & 63;
          if (tok >= L) reinterpret_cast<uint4*>(st)[u] = make_uint4(0, 0, 0, 0);
        }
        tc::fence_proxy_async();
        bar_arrive(&bars.clean);
        // (the values read below are this thread's own or valid ones: tok >= L is skipped)
      }
      if (n) wait(&bars.s_full, n - 1);  // the products that read W are done
      const unsigned char* V = st + 2 * NA * PANEL;
#pragma unroll
      for (int i = 0; i < 4 * NC; ++i) {
        const int u = i * 128 + u0, tok = (u >> 3) & 63;  // 16-byte piece of a panel row, in memory order
        uint4 x = *reinterpret_cast<const uint4*>(V + 16 * u);
        const float f = ps.write_scale * pw[rev ? tok + 1 : max(L - 1 - tok, 0)];
        uint32_t in[4] = {x.x, x.y, x.z, x.w}, w1[4], w2[4], w3[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float x0 = f * __uint_as_float(in[k] << 16), x1 = f * __uint_as_float(in[k] & 0xffff0000u);
          if (n == dirty && tok >= L) x0 = x1 = 0.f;
          w1[k] = take_pair(x0, x1);
          w2[k] = take_pair(x0, x1);
          w3[k] = last_pair(x0, x1);
        }
        *reinterpret_cast<uint4*>(W + 16 * u) = make_uint4(w1[0], w1[1], w1[2], w1[3]);
        *reinterpret_cast<uint4*>(W + G::W_TERM + 16 * u) = make_uint4(w2[0], w2[1], w2[2], w2[3]);
        *reinterpret_cast<uint4*>(W + 2 * G::W_TERM + 16 * u) = make_uint4(w3[0], w3[1], w3[2], w3[3]);
      }
      tc::fence_proxy_async();
      bar_arrive(&bars.w_ready);
    }
  } else if (warp == 8 + SW) {
    // ---- TMA ----------------------------------------------------------------------------
    if (lane == 0) {
      const int ma = tp.map_of[pass][0], mb = tp.map_of[pass][1], mc = tp.map_of[pass][2];
      const int ha = h / ps.a.group, hb = h / ps.b.group, hc = h / ps.c.group;
      for (int n = 0; n < chunks; ++n) {
        uint64_t* bar = &bars.full[n % STAGES];
        if (n >= STAGES) wait(&bars.empty[n % STAGES], n / STAGES - 1);
        tc::mbar_expect_tx(bar, (READ ? 2 * NA + NC : NA + NC) * PANEL);
        unsigned char* st = stage(n);
        const int t0 = chunk_start(n);
#pragma unroll
        for (int p = 0; p < NA; ++p) tma_load_4d(st + (NA + p) * PANEL, &tp.maps[mb], 64 * p, hb, t0, b, bar);
#pragma unroll
        for (int p = 0; p < NC; ++p) tma_load_4d(st + (2 * NA + p) * PANEL, &tp.maps[mc], 64 * p, hc, t0, b, bar);
        if (READ)
#pragma unroll
          for (int p = 0; p < NA; ++p) tma_load_4d(st + p * PANEL, &tp.maps[ma], 64 * p, ha, t0, b, bar);
      }
      // Every stage's last use has completed (and its barrier arrived) before the CTA ends.
      for (int n = max(0, chunks - STAGES); n < chunks; ++n) wait(&bars.empty[n % STAGES], n / STAGES);
    }
  } else if (lane == 0) {
    // ---- products -----------------------------------------------------------------------
    for (int n = 0; n < chunks; ++n) {
      const unsigned char* Q = stage(n);
      const unsigned char *K = Q + NA * PANEL, *V = K + NA * PANEL;
      const unsigned char *P = sm + G::OFF_P, *W = sm + G::OFF_W, *S = sm + G::OFF_S;
      wait(&bars.full[n % STAGES], n / STAGES);
      if (n == dirty) wait(&bars.clean, 0);
      tc::fence_after();
      if constexpr (READ) {
#pragma unroll
        for (int p = 0; p < NA; ++p)
          product<64, 64, false, false>(tm + G::COL_P, Q + p * PANEL, K + p * PANEL, p > 0);
        tc::commit(&bars.p_full);
      }
      wait(&bars.s_ready, n);
      if constexpr (READ) {
        if (n) wait(&bars.o_free, n - 1);
        tc::fence_after();
#pragma unroll
        for (int term = 0; term < 2; ++term)
#pragma unroll
          for (int p = 0; p < NA; ++p)
            product<DC, 64, false, false>(tm + G::COL_O2, S + term * G::S_TERM + p * (DC * 128), Q + p * PANEL,
                                          term + p > 0);
      }
      wait(&bars.w_ready, n);
      tc::fence_after();
#pragma unroll
      for (int term = 0; term < 3; ++term)
        product<DC, DA, true, true>(tm + G::COL_S, W + term * G::W_TERM, K, term > 0);
      tc::commit(&bars.s_full);
      if constexpr (READ) {
        wait(&bars.p_ready, n);
        tc::fence_after();
#pragma unroll
        for (int term = 0; term < 2; ++term)
          product<DC, 64, true, false>(tm + G::COL_O1, V, P + term * PANEL, term > 0);
        tc::commit(&bars.o_full);
      }
      tc::commit(&bars.empty[n % STAGES]);
    }
  }
  // Rows of this segment past the sequence's end.
  if (READ && len < bound) {
    const int z0 = max(len, base);
    const int64_t row = int64_t(pr.H) * ps.dc, out0 = int64_t(b) * pr.T * row + int64_t(h) * ps.dc;
    for (int64_t i = t; i < int64_t(bound - z0) * ps.dc; i += G::THREADS) {
      const int64_t at = out0 + (z0 + i / ps.dc) * row + i % ps.dc;
      if (ps.out_f32) static_cast<float*>(ps.out)[at] = 0.f;
      else static_cast<bf16*>(ps.out)[at] = __float2bfloat16_rn(0.f);
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 0) tc::tmem_dealloc(tm, G::COLS);
}

// Segment ends (walked from zero) -> the states at segment starts, and the
// state after the whole walk.
__global__ void __launch_bounds__(256) join_segments(const __grid_constant__ TcProblem tp) {
  const Problem& pr = tp.pr;
  const Pass& ps = pr.pass[blockIdx.z];
  const int n = ps.da * ps.dc, i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const size_t bh = blockIdx.y;
  const int b = int(bh) / pr.H, h = int(bh) % pr.H;
  int len = pr.T;
  if (pr.lengths) len = max(0, min(pr.T, pr.lengths[b]));
  const float g = pr.log_decay[h];
  const int r = i / ps.dc, c = i - r * ps.dc;
  float s = ps.init ? ps.init[bh * n + r * ps.init_r + c * ps.init_c] : 0.f;
  float* seg = tp.seg_state + blockIdx.z * tp.seg_pass + bh * tp.segments * n + i;
#pragma unroll 4
  for (int k = 0; k < tp.segments; ++k) {
    const int at = ps.reverse ? tp.segments - 1 - k : k;
    const int base = at * tp.segment_tokens;
    const int tokens = max(0, min(len, base + tp.segment_tokens) - base);
    const float local = seg[size_t(at) * n];
    seg[size_t(at) * n] = s;
    s = fmaf(tokens ? expf(g * float(tokens)) : 1.f, s, local);
  }
  if (ps.fin) ps.fin[bh * n + i] = s;
}

}  // namespace decay
}  // namespace m4
