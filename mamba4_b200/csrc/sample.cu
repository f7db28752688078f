// Token sampling with temperature, top-k, top-p and min-p from given uniform
// numbers (sm_100a).
//
// Per row: z_i = (max x - x_i) / T >= 0 (float32), e_i = exp(-z_i) and the mass
// m_i = trunc(2^35 e_i), a 64-bit integer: sums of masses are exact, so every
// order of summation (threads, blocks, atomics) gives the same token. Tokens
// are ranked by (z, index). A token is kept when its rank is below top_k, the
// mass ranked before it is below ceil(top_p * mass of the top_k), and
// e_i >= min_p; the first-ranked token always is. All three keep a prefix of
// the ranking, so the kept set is {(z, index) <= (tau, tau_index)}, found
// without sorting the row:
//   - a small top_k: the k-th largest of 256 maxima of groups of logits is a
//     bound that at least k logits reach; the few whose z is at most the bound's
//     go to a list, and one block ranks it and finishes; a top_k in the hundreds:
//     the same with a bound from the histogram below and binary digits in place
//     of the ranking;
//   - else an approximate histogram of z (all of the head, a quarter of the
//     tail) says about where the boundary lies; one exact pass sums the mass
//     below that place and lists the tokens around it, among which the boundary
//     is found exactly. If it is not there, the pass is made again around where
//     its exact sum puts the boundary, and after three such passes exact
//     histograms of the whole row narrow it down.
// The token is the first in vocabulary order whose running kept mass exceeds
// floor(u * kept mass). Tokens with z >= 24.5 have no mass and are never drawn.
//
// One thread-block cluster per row, from 16 blocks (a single row: bound by the
// latency of the cluster's barriers) to one (a large batch: bound by the
// arithmetic on each logit, an exponential and its integer). A row is read from
// HBM once; later passes find it in L1 or L2. Measured (B200), us: one row of
// 50304 float32 logits: greedy 5, top_k 50 and top_p 0.95 12, top_p 0.9 21,
// none 8; 64 rows: 9, 18, 35, 16; 512 rows of 131072 bfloat16 logits (134 MB, 20
// at the copy bandwidth): 67, 87, 297, 136, at 63 % of the issue slots.
// Without the list for a small top_k the second would be 21, 35 and 182; with
// top_k 1000, 19, 29 and 160, without its list 21, 37 and 284.
#include <cooperative_groups.h>

#include "common.cuh"

namespace m4 {
namespace sample {

namespace cg = cooperative_groups;
using bf16 = __nv_bfloat16;
using u32 = uint32_t;
using u64 = unsigned long long;

constexpr int NT = 512, NW = NT / 32;
constexpr int MAX_CTAS = 16;
constexpr int NB = 1024;             // histogram bins (2 a thread)
constexpr int GROUPS = 256;          // maxima of groups of logits, over the cluster
constexpr int SMALL_K = 128;         // top_k up to which the group maxima bound the list well
constexpr int LONG_K = 2048;         // top_k up to which the whole choice is made in a list
constexpr int RANKED = 1024;         // tokens ranked against each other
constexpr int LIST = 4096;           // tokens around the boundary
constexpr float Z_END = 24.5f;       // 2^35 e^-24.5 < 1
constexpr u32 Z_KEY = 0x41c40000u;   // its bits
constexpr int Z_BINS = 784;          // bins of z of width 1/32 below Z_END
constexpr float MASS_UNITS = 8192.f; // of the estimate, a token

// Estimated tokens listed on either side of the boundary: about three standard
// deviations of the estimate, of the number k of tokens before it (a quarter of
// them sampled: sqrt(3 k)) or of the mass. The list costs by its length, a miss
// one more pass: 512 rows of 131072 at top_p 0.9 took 290 us with 800 tokens,
// 306 with 1400, 500 with 500; 64 rows of 50304 33.8 us with 500, 38.9 with
// 1400, 41.3 with 150.
M4_DEV u32 slack_of(bool by_mass, int top_k, int vocab) {
  const float most = 2.2f * sqrtf(float(vocab)) + 20.f;
  return u32(by_mass ? most : fminf(most, 100.f + 5.2f * sqrtf(float(top_k))));
}

struct Settings {
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
};

// Mass of a token in two parts, m = hi 2^18 + lo: hi <= 2^17 and lo < 2^18, so
// 32-bit sums hold thousands of tokens. (Truncation by adding 2^23 towards
// zero: e 2^17 has 24 significant bits, its remainder is exact.)
M4_DEV void mass_parts(float e, u32& hi, u32& lo) {
  const float s = e * 131072.f, t = __fadd_rz(s, 8388608.f);
  hi = __float_as_uint(t) - 0x4b000000u;
  lo = __float_as_uint(__fmaf_rz(s - (t - 8388608.f), 262144.f, 8388608.f)) - 0x4b000000u;
}
M4_DEV u64 join(u32 hi, u32 lo) { return (u64(hi) << 18) + lo; }
M4_DEV u64 mass_of(float z) {
  u32 hi, lo;
  mass_parts(expf(-z), hi, lo);
  return join(hi, lo);
}
M4_DEV u64 warp_inclusive(u64 v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 n = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += n;
  }
  return v;
}
// Warp sum of parts (thread sums of at most 512 tokens).
M4_DEV u64 warp_total(u32 hi, u32 lo) {
  return join(__reduce_add_sync(0xffffffffu, hi), 0) + __reduce_add_sync(0xffffffffu, lo);
}

// What a CTA shows to its cluster.
struct Shared {
  u32 count[NB], hi[NB], lo[NB];  // this CTA's histogram: tokens, mass
  u32 all_count[NB];              // the cluster's
  u64 all_mass[NB];
  u64 list[LIST];                 // rank 0: key << 32 | index
  float group_max[GROUPS];
  u64 slot_a[MAX_CTAS], slot_b[MAX_CTAS], slot_d[MAX_CTAS], slot_e[2];  // one value of every CTA
  u64 warp_a[NW], warp_b[NW];
  u32 warp_n[NW];
  int n_list;
  u32 bin, bin_count, before_count;
  u64 before_mass;
  u32 tau_key;
  int tau_index;
  u32 lo_bin, hi_bin, centre;
  float lo_sum;
};

template <typename T>
struct Row {
  static constexpr int VEC = 16 / int(sizeof(T));
  Shared& s;
  u64* chunk;             // kept mass of each warp's step, in vocabulary order (+ 1)
  cg::cluster_group cl;
  const int rank, ctas, t, lane, warp;
  const T* src;           // the row
  int first, last;        // this CTA's slice
  bool vec;
  float top, inv;
  bool odd;               // an infinite largest logit or 1 / T: products may not be numbers
  // Members: (key, index) <= (tau_key, tau_index); at first, the tokens with mass.
  u32 tau_key;
  int tau_index = -1;
  bool summed = false;    // `chunk` holds the kept mass

  M4_DEV Row(Shared& s_, u64* c)
      : s(s_), chunk(c), cl(cg::this_cluster()), rank(int(cl.block_rank())), ctas(int(cl.num_blocks())),
        t(int(threadIdx.x)), lane(t & 31), warp(t >> 5), tau_key(Z_KEY) {}

  M4_DEV int steps() const { return (last - first + NT * VEC - 1) / (NT * VEC); }
  // f(values, index of the first, step), one vector of logits at a time, the
  // next two on their way; a NaN, and a place past the slice, is passed on as
  // -inf. All threads make equally many steps.
  template <class F>
  M4_DEV void each(F f) const {
    const int n = steps();
    uint4 next = fetch(0), after = fetch(1);
#pragma unroll 1
    for (int q = 0; q < n; ++q) {
      const uint4 now = next;
      next = after;
      if (q + 2 < n) after = fetch(q + 2);
      float x[VEC];
      unpack(now, x);
      f(x, first + (q * NT + t) * VEC, q);
    }
  }
  M4_DEV uint4 fetch(int q) const {
    const int i0 = first + (q * NT + t) * VEC;
    if (vec && i0 + VEC <= last) return *reinterpret_cast<const uint4*>(src + i0);
    alignas(16) T v[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = i0 + i < last ? src[i0 + i] : from_f<T>(-INFINITY);
    return *reinterpret_cast<const uint4*>(v);
  }
  static M4_DEV void unpack(uint4 raw, float (&x)[VEC]) {
    const u32 w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (VEC == 8) {
        const __nv_bfloat162 low = __float2bfloat162_rn(-INFINITY);
        const __nv_bfloat162 h = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), low);
        const u32 u = *reinterpret_cast<const u32*>(&h);
        x[2 * i] = __uint_as_float(u << 16);
        x[2 * i + 1] = __uint_as_float(u & 0xffff0000u);
      } else {
        x[i] = fmaxf(__uint_as_float(w[i]), -INFINITY);
      }
    }
  }
  // 0 for the largest logit, inf (no member) for -inf.
  M4_DEV float z_of(float x) const {
    const float z = (top - x) * inv;
    return odd ? (x == top ? 0.f : x > -INFINITY && z == z ? z : INFINITY) : z;
  }
  // A logit below which no z is at most z_of(bound). Different logits may have
  // one z, which ranks them by index, so what a bound selects is decided by z;
  // this spares most logits the product. z = fl(fl(top - x) inv) is within
  // 2^-23 of (top - x) inv, or 2^-149 where that underflows (inv within a factor
  // of two of 1 / temperature), so z <= z_of(bound) needs top - x <= (top -
  // bound)(1 + 2^-20) + 2^-147 temperature.
  M4_DEV float lowest(float bound, float temperature) const {
    if (odd) return -INFINITY;
    return __fsub_rd(top, __fadd_ru(__fmul_ru(top - bound, 1.f + 0x1p-20f), __fmul_ru(temperature, 0x1p-147f)));
  }
  M4_DEV bool member(u32 key, int index) const { return key < tau_key || (key == tau_key && index <= tau_index); }

  M4_DEV void clear_bins() {
    for (int b = t; b < NB; b += NT) s.count[b] = s.hi[b] = s.lo[b] = 0;
    __syncthreads();
  }
  // (a bin may hold a whole row: its sum has 54 bits, the low word's carries go to the high one)
  M4_DEV void add_mass(int b, u64 m) {
    const u32 low = u32(m);
    const u32 high = u32(m >> 32) + (low && atomicAdd(&s.lo[b], low) > ~low);
    if (high) atomicAdd(&s.hi[b], high);
  }
  M4_DEV u64 mass_in(const Shared& o, int b) const { return (u64(o.hi[b]) << 32) + o.lo[b]; }
  M4_DEV void add_to_bin(int b, float z) {
    atomicAdd(&s.count[b], 1u);
    add_mass(b, mass_of(z));
  }
  // Bins of the whole cluster: CTA r sums its share and hands it to everyone.
  M4_DEV void reduce_bins() {
    cl.sync();
    const int share = NB / ctas;
    for (int i = t; i < share; i += NT) {
      const int b = rank * share + i;
      u32 c = 0;
      u64 m = 0;
      for (int r = 0; r < ctas; ++r) {
        const Shared& o = *cl.map_shared_rank(&s, r);
        c += o.count[b];
        m += mass_in(o, b);
      }
      for (int r = 0; r < ctas; ++r) {
        Shared& o = *cl.map_shared_rank(&s, r);
        o.all_count[b] = c;
        o.all_mass[b] = m;
      }
    }
    cl.sync();
  }
  // This CTA's bins alone.
  M4_DEV void own_bins() {
    __syncthreads();
    for (int b = t; b < NB; b += NT) s.all_count[b] = s.count[b], s.all_mass[b] = mass_in(s, b);
    __syncthreads();
  }
  // The bin in which the running count (or mass), from what precedes, reaches `need`.
  M4_DEV void locate(bool by_mass, u64 need, u32& before_count, u64& before_mass, u32& bin, u32& bin_count) {
    const u32 c0 = s.all_count[2 * t], c1 = s.all_count[2 * t + 1];
    const u64 m0 = s.all_mass[2 * t], m1 = s.all_mass[2 * t + 1];
    u32 ci = c0 + c1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u32 n = __shfl_up_sync(0xffffffffu, ci, o);
      if (lane >= o) ci += n;
    }
    const u64 mi = warp_inclusive(m0 + m1, lane);
    if (lane == 31) s.warp_n[warp] = ci, s.warp_a[warp] = mi;
    __syncthreads();
    u32 c = before_count + ci - c0 - c1;
    u64 m = before_mass + mi - m0 - m1;
    for (int w = 0; w < warp; ++w) c += s.warp_n[w], m += s.warp_a[w];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const u32 bc = i ? c1 : c0;
      const u64 bm = i ? m1 : m0;
      if (by_mass ? m < need && need <= m + bm : c < need && need <= u64(c) + bc)
        s.bin = 2 * t + i, s.bin_count = bc, s.before_count = c, s.before_mass = m;
      c += bc;
      m += bm;
    }
    __syncthreads();
    bin = s.bin, bin_count = s.bin_count, before_count = s.before_count, before_mass = s.before_mass;
    __syncthreads();
  }

  // The boundary: the member at which the running count (mass) reaches `need`,
  // known to have a key in [lo, hi) with (before_count, before_mass) below lo.
  // Bins of the key's bits, then of the index, until one token is left. WHOLE:
  // over the row, by the cluster; else over this CTA's list.
  template <bool WHOLE>
  M4_DEV void narrow(bool by_mass, u64 need, u32 lo, u32 hi, u32 before_count, u64 before_mass, int n_list,
                     int vocab) {
    bool on_index = false;
    u32 key = 0;
    // (31 bits of a key and 18 of an index, 10 a pass: at most 4 + 2; the count ends the loop whatever the sums are)
#pragma unroll 1
    for (int pass = 0; pass < 6; ++pass) {
      const int shift = max(0, 22 - __clz(hi - lo - 1));  // at most NB bins (hi - lo = 1: one)
      const int sh = hi - lo == 1 ? 0 : shift;
      clear_bins();
      auto take = [&](u32 k, int index, float z) {
        const u32 d = on_index ? u32(index) : k;
        if (d >= lo && d < hi && (!on_index || k == key)) add_to_bin(int((d - lo) >> sh), z);
      };
      if (WHOLE) {
        each([&](const float(&x)[VEC], int i0, int) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float z = z_of(x[i]);
            if (member(__float_as_uint(z), i0 + i)) take(__float_as_uint(z), i0 + i, z);
          }
        });
        reduce_bins();
      } else {
        for (int i = t; i < n_list; i += NT) {
          const u64 c = s.list[i];
          take(u32(c >> 32), int(u32(c)), __uint_as_float(u32(c >> 32)));
        }
        own_bins();
      }
      u32 bin, n;
      locate(by_mass, need, before_count, before_mass, bin, n);
      lo += bin << sh;
      hi = min(hi, lo + (1u << sh));
      if (n == 1) {  // the one token left says where it is
        auto found = [&](u32 k, int index) {
          const u32 d = on_index ? u32(index) : k;
          if (d >= lo && d < hi && (!on_index || k == key)) s.tau_key = k, s.tau_index = index;
        };
        if (WHOLE) {
          if (t == 0) s.tau_index = -1;
          __syncthreads();
          each([&](const float(&x)[VEC], int i0, int) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const u32 k = __float_as_uint(z_of(x[i]));
              if (member(k, i0 + i)) found(k, i0 + i);
            }
          });
          __syncthreads();
          if (s.tau_index >= 0 && t < ctas) {
            Shared& o = *cl.map_shared_rank(&s, t);
            o.slot_e[0] = s.tau_key, o.slot_e[1] = u64(s.tau_index);
          }
          cl.sync();
          tau_key = u32(s.slot_e[0]), tau_index = int(s.slot_e[1]);
        } else {
          for (int i = t; i < n_list; i += NT) found(u32(s.list[i] >> 32), int(u32(s.list[i])));
          __syncthreads();
          tau_key = s.tau_key, tau_index = s.tau_index;
          __syncthreads();
        }
        return;
      }
      if (hi - lo == 1) {
        if (on_index) break;
        on_index = true;
        key = lo;
        lo = 0;
        hi = u32(vocab);
      }
    }
    tau_key = key;
    tau_index = int(lo);
  }

  // Every CTA's two sums, over the cluster.
  M4_DEV void cluster_sums(u64& a, u64& b) {
    if (lane == 0) s.warp_a[warp] = a, s.warp_b[warp] = b;
    __syncthreads();
    if (t < ctas) {
      u64 x = 0, y = 0;
      for (int k = 0; k < NW; ++k) x += s.warp_a[k], y += s.warp_b[k];
      Shared& o = *cl.map_shared_rank(&s, t);
      o.slot_a[rank] = x, o.slot_b[rank] = y;
    }
    cl.sync();
    a = b = 0;
    for (int k = 0; k < ctas; ++k) a += s.slot_a[k], b += s.slot_b[k];
  }

  // About how the members' mass (by_mass; every logit from x_head on counts:
  // few hold much of it) or number lies over the bins of z.
  M4_DEV void estimate(bool by_mass, float x_head) {
    // One sum per bin: the mass, or the count; each about gives the other. Masses
    // are integers, whose shared-memory atomics are single instructions, in units
    // of e^(-b / 32) / MASS_UNITS for bin b: at most MASS_UNITS a token, and a block's
    // 2^18 tokens, of which a sampled one counts four beside its head, stay below 2^32.
    for (int b = t; b < NB; b += NT) s.count[b] = 0;
    __syncthreads();
    each([&](const float(&x)[VEC], int i0, int q) {
      u32 head = 0;
      if (by_mass) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) head |= u32(x[i] >= x_head) << i;
      }
      auto add = [&](float v, int i, u32 times) {
        const float z = z_of(v);
        if (member(__float_as_uint(z), i0 + i)) {
          const float b = truncf(z * 32.f);
          atomicAdd(&s.count[int(b)], by_mass ? times * __float2uint_rn(__expf(fmaf(b, 1.f / 32.f, -z)) * MASS_UNITS) : times);
        }
      };
      // (a quarter of the tail)
#pragma unroll
      for (int i = 1; i < VEC; i += 4)
        if (!(head >> i & 1)) add(x[i], i, 4);
      while (head) {
        const int i = __ffs(head) - 1;
        head &= head - 1;
        float v = x[0];
#pragma unroll
        for (int j = 1; j < VEC; ++j) v = i == j ? x[j] : v;
        add(v, i, 1);
      }
    });
    cl.sync();
    const int part = NB / ctas;
    for (int i = t; i < part; i += NT) {
      const int b = rank * part + i;
      float m = 0.f;
      for (int r = 0; r < ctas; ++r) m += float(cl.map_shared_rank(&s, r)->count[b]);
      if (by_mass) m *= __expf(float(b) * (-1.f / 32.f)) / MASS_UNITS;
      for (int r = 0; r < ctas; ++r) reinterpret_cast<float*>(cl.map_shared_rank(&s, r)->all_count)[b] = m;
    }
    cl.sync();
  }

  // Bins [s.lo_bin, s.hi_bin) with about 2 `slack` tokens around where the running
  // estimate reaches: `share` of all of it; `goal`; or (again) `goal` more than at
  // s.lo_bin, where an exact sum is known.
  M4_DEV void place(bool by_mass, float share, float goal, bool again, u32 slack) {
    const float* all_sum = reinterpret_cast<const float*>(s.all_count);
    if (again) goal += s.lo_sum;
    __syncthreads();
    const float v0 = all_sum[2 * t], v1 = all_sum[2 * t + 1];
    const float scale = by_mass ? __expf(float(2 * t + 1) / 32.f) : 1.f;  // (a mass of e^-z: so many tokens)
    const u32 c0 = u32(v0 * scale), c1 = u32(v1 * scale);
    u32 ci = c0 + c1;
    float mi = v0 + v1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u32 n = __shfl_up_sync(0xffffffffu, ci, o);
      const float f = __shfl_up_sync(0xffffffffu, mi, o);
      if (lane >= o) ci += n, mi += f;
    }
    if (lane == 31) s.warp_n[warp] = ci, s.warp_a[warp] = __float_as_uint(mi);
    if (t == 0) s.centre = 0xffffffffu, s.lo_bin = Z_BINS - 1, s.hi_bin = 0;
    __syncthreads();
    u32 c = ci - c0 - c1, all_c = 0;
    float m = mi - v0 - v1, all = 0.f;
    for (int w = 0; w < NW; ++w) {
      const float f = __uint_as_float(u32(s.warp_a[w]));
      if (w < warp) c += s.warp_n[w], m += f;
      all_c += s.warp_n[w], all += f;
    }
    if (share > 0.f) goal = share * all;
    if (m < goal && goal <= m + v0 + v1) atomicMin(&s.centre, c + (c0 + c1) / 2);
    __syncthreads();
    const u32 centre = s.centre != 0xffffffffu ? s.centre : goal > 0.f ? all_c : 0;  // (before or past all of it)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const u32 b = 2 * t + i, upto = c + (i ? c0 + c1 : c0), from = i ? c + c0 : c;
      if (b < Z_BINS && int(upto) > int(centre) - int(slack)) atomicMin(&s.lo_bin, b);
      if (b < Z_BINS && from < centre + slack) atomicMax(&s.hi_bin, b + 1);
    }
    __syncthreads();
    if (int(s.lo_bin) >> 1 == t) s.lo_sum = m + (s.lo_bin & 1 ? v0 : 0.f);
    __syncthreads();
  }

  M4_DEV u64 block_total(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) s.warp_b[warp] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < NW; ++w) v += s.warp_b[w];
    return v;
  }

  // Moves the boundary to where the running count of the ranking reaches
  // top_k, or (MASS) its running mass top_p of the members' mass.
  template <bool MASS>
  M4_DEV void cut(int top_k, float top_p, float min_p, int vocab, float x_head) {
    estimate(MASS, x_head);
    const u32 slack = slack_of(MASS, top_k, vocab);
    place(MASS, MASS ? top_p : 0.f, float(top_k), false, slack);
    Shared& o = *cl.map_shared_rank(&s, 0);
    u64 need, under;
    int n;
#pragma unroll 1
    for (int attempt = 0;; ++attempt) {
      const u32 lo = __float_as_uint(float(s.lo_bin) / 32.f), hi = __float_as_uint(float(s.hi_bin) / 32.f);
      if (rank == 0 && t == 0) s.n_list = 0;
      cl.sync();
      u32 ah = 0, al = 0, bh = 0, bl = 0, live = 0, below = 0;
      u64 kept = 0;  // this warp's, below lo
      // (without an earlier bound masses past Z_END are 0 anyway; without min_p the kept mass below lo is all of it)
      const bool bounded = tau_key != Z_KEY, filter = min_p > 0.f;
      each([&](const float(&x)[VEC], int i0, int q) {
        u32 kh = 0, kl = 0;  // kept for sure: below lo
        u32 near = 0;        // in [lo, hi)
  #pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float z = z_of(x[i]);
          const u32 key = __float_as_uint(z);
          bool in = true;
          if (!MASS || bounded) in = member(key, i0 + i);
          const bool under = key < lo;
          if (MASS) {
            const float e = expf(-z);
            u32 h, l;
            mass_parts(e, h, l);
            if (bounded && !in) h = l = 0;
            ah += h, al += l;
            if (under) {
              if (filter) {
                bh += h, bl += l;
                if (!(e >= min_p)) h = l = 0;
              }
              kh += h, kl += l;
            }
          } else {
            live += in;
            below += in && under;
          }
          near |= u32(in && key - lo < hi - lo) << i;
        }
        if (near) {
          int at = atomicAdd(&o.n_list, __popc(near));
  #pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (near >> i & 1) {
              if (at < LIST) o.list[at] = (u64(__float_as_uint(z_of(x[i]))) << 32) | u32(i0 + i);
              ++at;
            }
        }
        if (MASS) {
          const u64 sum = warp_total(kh, kl);
          kept += sum;
          if (lane == 0) chunk[q * NW + warp] = sum;
        }
      });
      need = u64(top_k);
      u64 a = MASS ? warp_total(ah, al) : __reduce_add_sync(0xffffffffu, live);
      under = MASS ? (filter ? warp_total(bh, bl) : kept) : __reduce_add_sync(0xffffffffu, below);
      cluster_sums(a, under);
      n = o.n_list;
      if (MASS) {
        need = u64(ceil(double(top_p) * double(a)));
        if (need == 0) need = 1;
      } else if (a < need) {  // every token with mass is among the first top_k
        cl.sync();
        return;
      }
      // The list decides, if it reaches the boundary.
      if (rank == 0) {
        bool reached = under < need && n <= LIST;
        if (reached) {
          u64 inside = 0;
          for (int i = t; i < n; i += NT) inside += MASS ? mass_of(__uint_as_float(u32(s.list[i] >> 32))) : 1;
          reached = need <= under + block_total(inside);
        }
        if (reached) narrow<false>(MASS, need, lo, hi, u32(under), under, n, vocab);
        if (t < ctas) {
          Shared& to = *cl.map_shared_rank(&s, t);
          to.slot_e[0] = tau_key | u64(reached) << 32, to.slot_e[1] = u64(tau_index);
        }
      }
      cl.sync();
      if (s.slot_e[0] >> 32 || attempt == 2) break;
      // Once more, from the exact sum at lo.
      const double off = (double(need) - double(under)) * (MASS ? 0x1p-35 : 1.0);
      place(MASS, 0.f, float(off), true, n > LIST ? slack / 4 : slack);
    }
    if (s.slot_e[0] >> 32) {
      tau_key = u32(s.slot_e[0]), tau_index = int(s.slot_e[1]);
      if (MASS) {  // the list's kept tokens of this CTA join its sums
        for (int i = t; i < n; i += NT) {
          const u64 c = o.list[i];
          const u32 key = u32(c >> 32);
          const int index = int(u32(c));
          const float e = expf(-__uint_as_float(key));
          if (index >= first && index < last && member(key, index) && e >= min_p) {
            u32 h, l;
            mass_parts(e, h, l);
            atomicAdd(&chunk[(index - first) / (32 * VEC)], join(h, l));
          }
        }
        summed = true;
      }
    } else {
      cl.sync();  // (rank 0's count has been read)
      Row<T> whole = *this;  // (the boundary so far stays the members' bound while it narrows)
      whole.template narrow<true>(MASS, need, 0, Z_KEY, 0, 0, 0, vocab);
      tau_key = whole.tau_key, tau_index = whole.tau_index;
    }
  }

  // Rank 0 alone: the list holds every token up to some z, the first top_k
  // among them (more than finish_list ranks).
  M4_DEV void finish_long_list(int n, int top_k, float top_p, float min_p, float u, int vocab, int64_t* token,
                               float* log_prob) {
    if (n > top_k) narrow<false>(false, u64(top_k), 0, Z_KEY, 0, 0, n, vocab);
    auto mass = [&](u64 c, bool likely) {
      const float e = expf(-__uint_as_float(u32(c >> 32)));
      u32 h = 0, l = 0;
      if (member(u32(c >> 32), int(u32(c))) && (!likely || e >= min_p)) mass_parts(e, h, l);
      return join(h, l);
    };
    u64 sum = 0;
    if (top_p < 1.f) {
      for (int i = t; i < n; i += NT) sum += mass(s.list[i], false);
      const u64 need = u64(ceil(double(top_p) * double(block_total(sum))));
      narrow<false>(true, need > 0 ? need : 1, 0, Z_KEY, 0, 0, n, vocab);
    }
    sum = 0;
    for (int i = t; i < n; i += NT) sum += mass(s.list[i], true);
    const u64 kept = block_total(sum);
    const double d = double(u) * double(kept);
    u64 target = d > 0 ? u64(fmin(d, 1e18)) : 0;
    target = target < kept ? target : kept - 1;
    // By index: the bin, then the place, at which the running kept mass exceeds the target.
    u32 lo = 0, hi = u32(vocab), before_count = 0, bin, in_bin;
    u64 before_mass = 0;
    for (int pass = 0; pass < 3 && hi - lo > 1; ++pass) {  // (18 bits, 10 a pass)
      const int sh = max(0, 22 - __clz(hi - lo - 1));
      clear_bins();
      for (int i = t; i < n; i += NT) {
        const u64 c = s.list[i], m = mass(c, true);
        const u32 index = u32(c);
        if (m && index >= lo && index < hi) add_mass(int((index - lo) >> sh), m);
      }
      own_bins();
      locate(true, target + 1, before_count, before_mass, bin, in_bin);
      lo += bin << sh;
      hi = min(hi, lo + (1u << sh));
    }
    for (int i = t; i < n; i += NT)
      if (u32(s.list[i]) == lo) {
        *token = int64_t(lo);
        *log_prob = -__uint_as_float(u32(s.list[i] >> 32)) - logf(float(double(kept) * 0x1p-35));
      }
  }

  // Rank 0 alone: the list holds every token up to some z, the first top_k among them.
  M4_DEV void finish_list(int n, int top_k, float top_p, float min_p, float u, int64_t* token, float* log_prob) {
    u64* ranked = s.all_mass;  // [RANKED]
    for (int i = t; i < n; i += NT) {
      const u64 me = s.list[i];
      int r = 0;
      for (int j = 0; j < n; ++j) r += s.list[j] < me;
      ranked[r] = me;
    }
    __syncthreads();
    if (warp) return;  // one warp: at most SMALL_K tokens are left
    n = min(n, top_k);
    constexpr int PER = SMALL_K / 32;
    u64 key[PER], m[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = lane * PER + i;
      key[i] = at < n ? ranked[at] : 0;
      m[i] = at < n ? mass_of(__uint_as_float(u32(key[i] >> 32))) : 0;
      sum += m[i];
    }
    const u64 incl = warp_inclusive(sum, lane);
    u64 run = incl - sum;
    const u64 all = __shfl_sync(0xffffffffu, incl, 31);
    u64 need = all;
    if (top_p < 1.f) need = max(1ull, u64(ceil(double(top_p) * double(all))));
    u64 kept = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool keep = run < need && expf(-__uint_as_float(u32(key[i] >> 32))) >= min_p;
      run += m[i];
      if (!keep) m[i] = 0;
      kept += m[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) kept += __shfl_xor_sync(0xffffffffu, kept, o);
    const double d = double(u) * double(kept);
    u64 target = d > 0 ? u64(fmin(d, 1e18)) : 0;
    target = target < kept ? target : kept - 1;
    // Kept mass with a lower index than each token's.
    u64 below[PER] = {};
    for (int src_lane = 0; src_lane < 32; ++src_lane)
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const u64 om = __shfl_sync(0xffffffffu, m[j], src_lane);
        const u32 oi = __shfl_sync(0xffffffffu, u32(key[j]), src_lane);
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (oi < u32(key[i])) below[i] += om;
      }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (m[i] && below[i] <= target && target < below[i] + m[i]) {
        *token = int64_t(u32(key[i]));
        *log_prob = -__uint_as_float(u32(key[i] >> 32)) - logf(float(double(kept) * 0x1p-35));
      }
  }
};

template <typename T>
__global__ void __launch_bounds__(NT, 2) sample_kernel(int vocab, int64_t ld, int slice, bool vec,
                                                    const T* __restrict__ logits,
                                                    const float* __restrict__ uniform, Settings set,
                                                    int64_t* __restrict__ tokens, float* __restrict__ log_prob) {
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& s = *reinterpret_cast<Shared*>(raw);
  Row<T> row(s, reinterpret_cast<u64*>(raw + sizeof(Shared)));
  constexpr int VEC = Row<T>::VEC;
  const int t = row.t, lane = row.lane, warp = row.warp, rank = row.rank, ctas = row.ctas;
  const int r = blockIdx.x / ctas;
  row.first = min(rank * slice, vocab);
  row.last = min(row.first + slice, vocab);
  row.src = logits + int64_t(r) * ld;
  row.vec = vec;
  row.cl.barrier_arrive();  // every CTA of the cluster has started before its shared memory is written
  // Maxima of groups of 2 ctas neighbouring threads: 256 over the cluster.
  float best = -INFINITY;
  row.each([&](const float(&x)[VEC], int, int) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) best = fmaxf(best, x[i]);
  });
  for (int o = 1; o < 2 * ctas && o < 32; o <<= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
  const int width = min(32, 2 * ctas), per = NT / width;
  row.cl.barrier_wait();
  if ((t & (width - 1)) == 0)
    for (int k = 0; k < ctas; ++k) row.cl.map_shared_rank(&s, k)->group_max[rank * per + t / width] = best;
  row.cl.sync();
  static_assert(GROUPS == NT / 2 && MAX_CTAS <= 16, "per x ctas groups, for every size of a cluster");
  float top = t < GROUPS ? s.group_max[t] : -INFINITY;
  {
    float low = t < GROUPS ? top : INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    }
    if (lane == 0) s.warp_a[warp] = __float_as_uint(top), s.warp_b[warp] = __float_as_uint(low);
    __syncthreads();
    for (int w = 0; w < NW; ++w) {
      top = fmaxf(top, __uint_as_float(u32(s.warp_a[w])));
      low = fminf(low, __uint_as_float(u32(s.warp_b[w])));
    }
    best = low;  // the least of the group maxima
  }
  __syncthreads();

  const float temperature = set.temperature ? set.temperature[r] : set.temperature_all;
  const float top_p = set.top_p ? set.top_p[r] : set.top_p_all;
  const float min_p = set.min_p ? set.min_p[r] : set.min_p_all;
  int top_k = set.top_k ? set.top_k[r] : set.top_k_all;
  // Settings that leave the first-ranked token alone (a NaN does).
  if (!(temperature > 0.f) || !(top_p > 0.f) || !(min_p <= 1.f)) top_k = 1;
  if (top_k <= 0 || top_k > vocab) top_k = vocab;
  if (top == -INFINITY) {  // the mask leaves nothing
    if (rank == 0 && t == 0) tokens[r] = -1, log_prob[r] = -INFINITY;
    return;
  }
  const bool hot = temperature > 0.f;
  row.top = top;
  row.inv = 1.f / temperature;
  row.odd = !(top < INFINITY) || !(row.inv < INFINITY) || row.inv == 0.f;
  if (top_k == 1) {  // the lowest index of z = 0 (without a temperature: of the largest logit)
    const float least = hot ? row.lowest(top, temperature) : top;
    int idx = 0x7fffffff;
    row.each([&](const float(&x)[VEC], int i0, int) {
#pragma unroll
      for (int i = VEC - 1; i >= 0; --i)
        if (x[i] >= least && (x[i] == top || (hot && row.z_of(x[i]) == 0.f)) && i0 + i < idx) idx = i0 + i;
    });
    idx = __reduce_min_sync(0xffffffffu, idx);
    if (lane == 0) s.warp_n[warp] = u32(idx);
    __syncthreads();
    if (t == 0) {
      for (int w = 0; w < NW; ++w) idx = min(idx, int(s.warp_n[w]));
      row.cl.map_shared_rank(&s, 0)->slot_a[rank] = u64(idx);
    }
    row.cl.sync();
    if (rank == 0 && t == 0) {
      for (int k = 0; k < ctas; ++k) idx = min(idx, int(s.slot_a[k]));
      tokens[r] = idx;
      log_prob[r] = 0.f;
    }
    return;
  }
  if (top_k <= SMALL_K) {
    // The k-th largest group maximum: at least top_k logits reach it.
    if (t < GROUPS) {
      const float me = s.group_max[t];
      int above = 0;
      for (int j = 0; j < GROUPS; ++j) {
        const float x = s.group_max[j];
        above += x > me || (x == me && j < t);
      }
      if (above == top_k - 1) s.centre = __float_as_uint(me);
    }
    if (rank == 0 && t == 0) s.n_list = 0;
    row.cl.sync();
    const float bound = __uint_as_float(s.centre), z_bound = row.z_of(bound), least = row.lowest(bound, temperature);
    Shared& o = *row.cl.map_shared_rank(&s, 0);
    row.each([&](const float(&x)[VEC], int i0, int) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (x[i] >= least) {
          const float z = row.z_of(x[i]);
          if (z <= z_bound && z < Z_END) {
            const int at = atomicAdd(&o.n_list, 1);
            if (at < RANKED) o.list[at] = (u64(__float_as_uint(z)) << 32) | u32(i0 + i);
          }
        }
    });
    row.cl.sync();
    const int n = o.n_list;
    row.cl.sync();  // (rank 0's memory is not read below, and may be reused)
    if (n <= RANKED) {
      if (rank == 0) row.finish_list(n, top_k, top_p, min_p, uniform[r], tokens + r, log_prob + r);
      return;
    }
  }
  const float x_head = best;  // the least group maximum: reached by about 1400 logits
  if (top_k <= LONG_K) {
    // About top_k tokens and the slack, again from a bound on z.
    row.estimate(false, x_head);
    row.place(false, 0.f, float(top_k), false, slack_of(false, top_k, vocab));
    const u32 hi = __float_as_uint(float(s.hi_bin) / 32.f);
    if (rank == 0 && t == 0) s.n_list = 0;
    row.cl.sync();
    Shared& o = *row.cl.map_shared_rank(&s, 0);
    row.each([&](const float(&x)[VEC], int i0, int) {
      u32 near = 0;
#pragma unroll
      for (int i = 0; i < VEC; ++i) near |= u32(__float_as_uint(row.z_of(x[i])) < hi) << i;
      if (near) {
        int at = atomicAdd(&o.n_list, __popc(near));
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (near >> i & 1) {
            if (at < LIST) o.list[at] = (u64(__float_as_uint(row.z_of(x[i]))) << 32) | u32(i0 + i);
            ++at;
          }
      }
    });
    row.cl.sync();
    const int n = o.n_list;
    row.cl.sync();
    // (every token with mass, or at least top_k)
    if (n <= LIST && (n >= top_k || s.hi_bin == Z_BINS)) {
      if (rank == 0)
        row.finish_long_list(n, top_k, top_p, min_p, uniform[r], vocab, tokens + r, log_prob + r);
      return;
    }
  }
  if (top_k < vocab) row.template cut<false>(top_k, 1.f, min_p, vocab, x_head);
  if (top_p < 1.f) row.template cut<true>(0, top_p, min_p, vocab, x_head);
  // Mass of the kept tokens in vocabulary order, per warp and step.
  auto kept_parts = [&](float x, int index, u32& h, u32& l, float& z) {
    h = l = 0;
    z = row.z_of(x);
    const float e = expf(-z);
    if (row.member(__float_as_uint(z), index) && e >= min_p) mass_parts(e, h, l);
  };
  if (!row.summed)
    row.each([&](const float(&x)[VEC], int i0, int q) {
      u32 hi = 0, lo = 0;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        u32 h, l;
        float z;
        kept_parts(x[i], i0 + i, h, l, z);
        hi += h;
        lo += l;
      }
      const u64 sum = warp_total(hi, lo);
      if (lane == 0) row.chunk[q * NW + warp] = sum;
    });
  __syncthreads();
  // Running sums over the steps of this CTA.
  const int n_chunks = row.steps() * NW;
  u64 mine = 0;
  const int per_thread = (n_chunks + NT - 1) / NT;
  for (int i = 0; i < per_thread; ++i) {
    const int at = t * per_thread + i;
    if (at < n_chunks) mine += row.chunk[at];
  }
  const u64 incl = warp_inclusive(mine, lane);
  if (lane == 31) s.warp_a[warp] = incl;
  __syncthreads();
  u64 run = incl - mine, cta = 0;
  for (int w = 0; w < NW; ++w) {
    if (w < warp) run += s.warp_a[w];
    cta += s.warp_a[w];
  }
  if (t < ctas) row.cl.map_shared_rank(&s, t)->slot_d[rank] = cta;
  row.cl.sync();
  u64 total = 0, before = 0;
  for (int k = 0; k < ctas; ++k) {
    if (k < rank) before += s.slot_d[k];
    total += s.slot_d[k];
  }
  const double d = double(uniform[r]) * double(total);
  u64 target = d > 0 ? u64(fmin(d, 1e18)) : 0;
  target = target < total ? target : total - 1;
  if (target < before || target >= before + cta) return;  // another CTA's token
  target -= before;
  for (int i = 0; i < per_thread; ++i) {
    const int at = t * per_thread + i;
    if (at >= n_chunks) break;
    const u64 m = row.chunk[at];
    if (run <= target && target < run + m) s.bin = u32(at), s.before_mass = run;
    run += m;
  }
  __syncthreads();
  if (warp == 0) {  // the step's 32 vectors
    const int i0 = row.first + (int(s.bin) * 32 + lane) * VEC;
    u64 m[VEC], sum = 0;
    float z[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float x = i0 + i < row.last ? fmaxf(to_f<T>(row.src[i0 + i]), -INFINITY) : -INFINITY;
      u32 h, l;
      kept_parts(x, i0 + i, h, l, z[i]);
      m[i] = join(h, l);
      sum += m[i];
    }
    u64 at = s.before_mass + warp_inclusive(sum, lane) - sum;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if (at <= target && target < at + m[i]) {
        tokens[r] = i0 + i;
        log_prob[r] = -z[i] - logf(float(double(total) * 0x1p-35));
      }
      at += m[i];
    }
  }
}

constexpr int MAX_VOCAB = 262144;

template <auto K>
bool allow_clusters_of_16() {
  static std::atomic<bool> done[64];
  int device;
  if (cudaGetDevice(&device) != cudaSuccess) return false;
  if (device < 64 && done[device]) return true;
  if (cudaFuncSetAttribute(K, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return false;
  if (device < 64) done[device] = true;  // (set twice by two threads it is the same)
  return true;
}

template <typename T>
int launch(int rows, int vocab, int64_t ld, const void* logits, const float* uniform, const Settings& set,
           int64_t* tokens, float* log_prob, cudaStream_t st) {
  // As many CTAs a row as the GPU has room for (two of 512 threads an SM), each
  // with at least a vector a thread. Twice as many: 64 rows of 50304 at top_p 0.9
  // 55 us for 35, 256 rows 92 for 74; four times: 512 rows of 131072 300 for 295.
  int ctas = 1;
  while (ctas < MAX_CTAS && int64_t(rows) * ctas * 2 <= 296 && ctas * NT * 4 < vocab) ctas *= 2;
  const int slice = ((vocab + ctas - 1) / ctas + 7) & ~7;
  const bool vec = (ld * sizeof(T)) % 16 == 0 && aligned16(logits);
  const int per_step = NT * Row<T>::VEC;
  const size_t smem = sizeof(Shared) + size_t((slice + per_step - 1) / per_step) * NW * 8;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(rows) * ctas);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (!allow_shared<sample_kernel<T>>(smem) ||
      (ctas > 8 && !allow_clusters_of_16<sample_kernel<T>>()))
    return M4_ERR_LAUNCH;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<T>, vocab, ld, slice, vec,
                                           static_cast<const T*>(logits), uniform, set, tokens, log_prob);
  return e == cudaSuccess ? launch_status() : M4_ERR_LAUNCH;
}

}  // namespace sample
}  // namespace m4

extern "C" int m4_sample(int rows, int vocab, int64_t ld, const void* logits, int bf16_logits, const float* uniform,
                         const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                         float temperature_all, int top_k_all, float top_p_all, float min_p_all, int64_t* tokens,
                         float* log_prob, void* stream) {
  using namespace m4::sample;
  if (rows <= 0 || vocab <= 0 || ld < vocab) return M4_ERR_DIMS;
  if (vocab > MAX_VOCAB || rows > 0x7fffffff / MAX_CTAS) return M4_ERR_UNSUPPORTED;
  if (!logits || !uniform || !tokens || !log_prob) return M4_ERR_NULL;
  const Settings set{temperature, top_k, top_p, min_p, temperature_all, top_p_all, min_p_all, top_k_all};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return bf16_logits ? launch<bf16>(rows, vocab, ld, logits, uniform, set, tokens, log_prob, st)
                     : launch<float>(rows, vocab, ld, logits, uniform, set, tokens, log_prob, st);
}
