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
// without sorting: a histogram of z in 1024 bins of width 1/32 locates the
// bin of the boundary, sub-histograms of the float's bits narrow a crowded bin
// down, and the few tokens left are ranked against each other. The token is
// the first in vocabulary order whose running kept mass exceeds
// floor(u * kept mass).
//
// One thread-block cluster per row: the row is read once, stays in registers
// (up to 32 values a thread), and partial results cross in distributed shared
// memory. A large batch is bound by the arithmetic on each logit (an
// exponential and its integer), a single row by the latency of the cluster's
// barriers.
#include <cooperative_groups.h>

#include "common.cuh"

namespace m4 {
namespace sample {

namespace cg = cooperative_groups;
using bf16 = __nv_bfloat16;
using u32 = uint32_t;
using u64 = unsigned long long;

constexpr int NT = 512, NW = NT / 32;
constexpr int NB = 1024;        // histogram bins
constexpr int MAX_CTAS = 16;
constexpr int CAP = 1024;       // tokens ranked against each other
constexpr u32 ABSENT = 0xffffffffu;  // key of a place past the row's end (above every z, inf included)
constexpr u32 KEY_END = 0x7f800001u; // one above the key of z = inf

struct Settings {
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
};

// Mass of a token in two parts, m = hi 2^18 + lo: hi <= 2^17 and lo < 2^18, so
// 32-bit sums hold the 16384 tokens of a CTA. (e 2^17 has 24 significant bits:
// its remainder below the integer part is exact.)
M4_DEV void mass_parts(float e, u32& hi, u32& lo) {
  const float s = e * 131072.f;
  hi = __float2uint_rz(s);
  lo = __float2uint_rz((s - __uint2float_rz(hi)) * 262144.f);
}
M4_DEV u64 mass_of(float e) {
  u32 hi, lo;
  mass_parts(e, hi, lo);
  return (u64(hi) << 18) + lo;
}
M4_DEV u64 warp_inclusive_u64(u64 v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 n = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += n;
  }
  return v;
}
// Warp sum of values below 2^36 each (thread sums of at most 8 masses or counts: parts below 2^21).
M4_DEV u64 warp_sum_parts(u32 hi, u32 lo) {
  return (u64(__reduce_add_sync(0xffffffffu, hi)) << 18) + __reduce_add_sync(0xffffffffu, lo);
}

// What one CTA shows to its cluster.
struct Shared {
  u32 count[NB], hi[NB], lo[NB];  // this CTA's histogram
  u32 total_count[NB];            // the cluster's
  u64 total_mass[NB];
  u64 cand[CAP];                  // rank 0: key << 32 | index
  u64 warp_mass[8 * NW + 1];      // running sums per (round, warp)
  u64 cta_mass[MAX_CTAS];
  float cta_max[MAX_CTAS];
  int cta_first[MAX_CTAS];
  u64 scan_mass[NW];
  u32 scan_count[NW];
  float scan_f[NW];
  int scan_i[NW];
  int n_cand;
  // Located bin and what precedes it.
  u32 bin, bin_count, before_count;
  u64 before_mass;
  // Boundary, and the mass of the tokens up to it.
  u32 tau_key;
  int tau_index;
  u64 mass_upto;
};

// A row's slice in one CTA: E values a thread, in ROUNDS vectors of VEC.
template <typename T, int E>
struct Row {
  static constexpr int VEC = 16 / int(sizeof(T));
  static constexpr int ROUNDS = E / VEC;
  static_assert(ROUNDS * VEC == E && ROUNDS <= 8, "slices are whole vectors");

  float z[E];  // its bits are the ranking key; ABSENT past the end
  Shared& s;
  cg::cluster_group cl;
  const int rank, ctas, t, lane, warp;
  int base;
  u32 tau_key = KEY_END;  // members are the tokens with (key, index) <= (tau_key, tau_index)
  int tau_index = 0;

  M4_DEV explicit Row(Shared& s_)
      : s(s_), cl(cg::this_cluster()), rank(int(cl.block_rank())), ctas(int(cl.num_blocks())), t(int(threadIdx.x)),
        lane(t & 31), warp(t >> 5) {}

  M4_DEV int index(int j) const { return base + (j / VEC) * NT * VEC + t * VEC + j % VEC; }
  M4_DEV u32 key(int j) const { return __float_as_uint(z[j]); }
  M4_DEV bool member(int j) const {
    const u32 k = key(j);
    return k < tau_key || (k == tau_key && index(j) <= tau_index);
  }

  // Cluster histogram of the members with lo <= key < hi: bins of z of width
  // 1/32 when shift < 0, of the key's distance from lo otherwise.
  M4_DEV void histogram(u32 lo, u32 hi, int shift) {
    for (int b = t; b < NB; b += NT) s.count[b] = s.hi[b] = s.lo[b] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const u32 k = key(j);
      if (k < lo || k >= hi || !member(j)) continue;
      const int b = shift < 0 ? int(fminf(z[j] * 32.f, float(NB - 1))) : int((k - lo) >> shift);
      atomicAdd(&s.count[b], 1u);
      u32 mh, ml;
      mass_parts(expf(-z[j]), mh, ml);
      if (mh | ml) {
        atomicAdd(&s.hi[b], mh);
        atomicAdd(&s.lo[b], ml);
      }
    }
    cl.sync();
    // CTA r sums its share of the bins over the cluster and hands them to everyone.
    const int share = NB / ctas;
    for (int i = t; i < share; i += NT) {
      const int b = rank * share + i;
      u32 c = 0;
      u64 m = 0;
      for (int r = 0; r < ctas; ++r) {
        const Shared& o = *cl.map_shared_rank(&s, r);
        c += o.count[b];
        m += (u64(o.hi[b]) << 18) + o.lo[b];
      }
      for (int r = 0; r < ctas; ++r) {
        Shared& o = *cl.map_shared_rank(&s, r);
        o.total_count[b] = c;
        o.total_mass[b] = m;
      }
    }
    cl.sync();
  }

  // The bin in which the running count (or mass) from (before_count, before_mass)
  // reaches `need` (>= 1), and what precedes it; the last bin if none does.
  M4_DEV void locate(bool by_mass, u64 need, u32& before_count, u64& before_mass, u32& bin, u32& bin_count) {
    constexpr int PER = NB / NT;
    u32 c = 0;
    u64 m = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      c += s.total_count[t * PER + i];
      m += s.total_mass[t * PER + i];
    }
    u32 ci = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u32 n = __shfl_up_sync(0xffffffffu, ci, o);
      if (lane >= o) ci += n;
    }
    u64 mi = warp_inclusive_u64(m, lane);
    if (lane == 31) s.scan_count[warp] = ci, s.scan_mass[warp] = mi;
    __syncthreads();
    u32 c0 = before_count + ci - c;
    u64 m0 = before_mass + mi - m;
    for (int w = 0; w < warp; ++w) c0 += s.scan_count[w], m0 += s.scan_mass[w];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int b = t * PER + i;
      const u32 bc = s.total_count[b];
      const u64 bm = s.total_mass[b];
      const bool reaches = by_mass ? m0 < need && need <= m0 + bm : u64(c0) < need && need <= u64(c0) + bc;
      if (reaches || (b == NB - 1 && (by_mass ? m0 + bm < need : u64(c0) + bc < need)))
        s.bin = b, s.bin_count = bc, s.before_count = c0, s.before_mass = m0;
      c0 += bc;
      m0 += bm;
    }
    __syncthreads();
    bin = s.bin, bin_count = s.bin_count, before_count = s.before_count, before_mass = s.before_mass;
    __syncthreads();
  }

  // Running sums of the per-round warp sums in warp_mass (exclusive; the total
  // last), and every CTA's total in cta_mass. warp_mass is filled by the caller.
  M4_DEV void scan_cta() {
    __syncthreads();
    if (warp == 0) {
      constexpr int N = ROUNDS * NW, PER = (N + 31) / 32;
      u64 v[PER], sum = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        v[i] = lane * PER + i < N ? s.warp_mass[lane * PER + i] : 0;
        sum += v[i];
      }
      const u64 incl = warp_inclusive_u64(sum, lane);
      u64 run = incl - sum;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (lane * PER + i < N) s.warp_mass[lane * PER + i] = run;
        run += v[i];
      }
      const u64 total = __shfl_sync(0xffffffffu, incl, 31);
      if (lane == 0) s.warp_mass[N] = total;
      if (lane < ctas) cl.map_shared_rank(&s, lane)->cta_mass[rank] = total;
    }
    cl.sync();
  }

  // The token of this CTA at which the running weight (weight(j) as two parts)
  // first exceeds `target`, given the CTA's running sums; called by every thread
  // of the CTA that owns the target, true in the one thread that found it.
  template <class F>
  M4_DEV bool find(u64 target, F weight, int& found_index, float& found_z) const {
    bool hit = false;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const u64 first = s.warp_mass[r * NW + warp], next = s.warp_mass[r * NW + warp + 1];
      if (target < first || target >= next) continue;  // one (round, warp) only
      u64 mine = 0;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        u32 hi, lo;
        weight(r * VEC + i, hi, lo);
        mine += (u64(hi) << 18) + lo;
      }
      const u64 incl = warp_inclusive_u64(mine, lane);
      u64 run = first + incl - mine;
      if (run <= target && target < run + mine) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          u32 hi, lo;
          weight(r * VEC + i, hi, lo);
          const u64 w = (u64(hi) << 18) + lo;
          if (!hit && target < run + w) hit = true, found_index = index(r * VEC + i), found_z = z[r * VEC + i];
          run += w;
        }
      }
    }
    return hit;
  }

  template <class F>
  M4_DEV void warp_sums(F weight) {
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      u32 hi = 0, lo = 0;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        u32 h, l;
        weight(r * VEC + i, h, l);
        hi += h;
        lo += l;
      }
      const u64 sum = warp_sum_parts(hi, lo);
      if (lane == 0) s.warp_mass[r * NW + warp] = sum;
    }
  }

  // Moves the boundary to the member at which the running count (by_mass:
  // mass) of the ranking reaches `need`. Returns the members' mass up to it.
  // `fresh`: total_count / total_mass hold the histogram of all bins of z.
  M4_DEV u64 cut(bool by_mass, u64 need, bool& fresh) {
    u32 lo = 0, hi = KEY_END, before_count = 0, bin, n;
    u64 before_mass = 0;
    int shift = -1;
    while (true) {
      if (shift >= 0 || !fresh) histogram(lo, hi, shift);
      fresh = shift < 0;
      locate(by_mass, need, before_count, before_mass, bin, n);
      if (shift < 0) {
        lo = __float_as_uint(float(bin) * (1.f / 32));
        if (bin + 1 < NB) hi = __float_as_uint(float(bin + 1) * (1.f / 32));
      } else {
        lo += bin << shift;
        hi = min(hi, lo + (1u << shift));
      }
      if (n <= CAP || hi - lo == 1) break;
      shift = max(0, 22 - __clz(hi - lo - 1));  // at most NB bins
    }
    if (n <= CAP) {
      // Rank 0 ranks the few tokens left against each other.
      Shared& o = *cl.map_shared_rank(&s, 0);
      if (rank == 0 && t == 0) s.n_cand = 0;
      cl.sync();
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (key(j) >= lo && key(j) < hi && member(j)) {
          const int at = atomicAdd(&o.n_cand, 1);
          if (at < CAP) o.cand[at] = (u64(key(j)) << 32) | u32(index(j));
        }
      cl.sync();
      if (rank == 0) {
        const int have = min(s.n_cand, CAP);
        for (int i = t; i < have; i += NT) {
          const u64 me = s.cand[i];
          u32 below = before_count;
          u64 mass = before_mass;
          for (int k = 0; k < have; ++k) {
            const u64 other = s.cand[k];
            if (other < me) {
              ++below;
              if (by_mass) mass += mass_of(expf(-__uint_as_float(u32(other >> 32))));
            }
          }
          const u64 m = mass_of(expf(-__uint_as_float(u32(me >> 32))));
          const bool last = by_mass ? mass < need && need <= mass + m : u64(below) + 1 == need;
          if (last) {
            if (!by_mass)
              for (int k = 0; k < have; ++k)
                if (s.cand[k] < me) mass += mass_of(expf(-__uint_as_float(u32(s.cand[k] >> 32))));
            for (int r = 0; r < ctas; ++r) {
              Shared& to = *cl.map_shared_rank(&s, r);
              to.tau_key = u32(me >> 32);
              to.tau_index = int(u32(me));
              to.mass_upto = mass + m;
            }
          }
        }
      }
      cl.sync();
    } else {
      // Many tokens with one z: the boundary is the r-th of them by index.
      const u64 m = mass_of(expf(-__uint_as_float(lo)));
      const u64 r = by_mass ? (need - before_mass + m - 1) / m : need - before_count;
      auto weight = [&](int j, u32& h, u32& l) { h = 0, l = key(j) == lo && member(j); };
      warp_sums(weight);
      scan_cta();
      u64 before = 0;
      for (int k = 0; k < rank; ++k) before += s.cta_mass[k];
      int idx;
      float zf;
      if (r - 1 >= before && r - 1 < before + s.cta_mass[rank] && find(r - 1 - before, weight, idx, zf))
        for (int k = 0; k < ctas; ++k) {
          Shared& to = *cl.map_shared_rank(&s, k);
          to.tau_key = lo;
          to.tau_index = idx;
          to.mass_upto = before_mass + r * m;
        }
      cl.sync();
    }
    tau_key = s.tau_key;
    tau_index = s.tau_index;
    return s.mass_upto;
  }
};

template <typename T, int E>
__global__ void __launch_bounds__(NT) sample_kernel(int vocab, int64_t ld, int slice, bool vec,
                                                    const T* __restrict__ logits,
                                                    const float* __restrict__ uniform, Settings set,
                                                    int64_t* __restrict__ tokens, float* __restrict__ log_prob) {
  __shared__ Shared s;
  Row<T, E> row(s);
  constexpr int VEC = Row<T, E>::VEC;
  const int t = row.t, lane = row.lane, warp = row.warp, rank = row.rank, ctas = row.ctas;
  const int r = blockIdx.x / ctas;
  const int first = min(rank * slice, vocab), last = min(first + slice, vocab);
  row.base = first;
  row.cl.barrier_arrive();  // every CTA of the cluster has started before its shared memory is written
  const T* src = logits + int64_t(r) * ld;
  float (&z)[E] = row.z;
  // The slice (16 bytes a load when rows allow it), and its largest logit.
  float top = -INFINITY;
#pragma unroll
  for (int q = 0; q < Row<T, E>::ROUNDS; ++q) {
    const int i0 = row.index(q * VEC);
    if (vec && i0 + VEC <= last) {
      alignas(16) T v[VEC];
      *reinterpret_cast<uint4*>(v) = __ldcs(reinterpret_cast<const uint4*>(src + i0));
#pragma unroll
      for (int i = 0; i < VEC; ++i) z[q * VEC + i] = to_f<T>(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) z[q * VEC + i] = i0 + i < last ? to_f<T>(src[i0 + i]) : -INFINITY;
    }
  }
#pragma unroll
  for (int j = 0; j < E; ++j) top = fmaxf(top, z[j]);  // a NaN is passed over
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s.scan_f[warp] = top;
  __syncthreads();
  row.cl.barrier_wait();
  if (t < ctas) {
    float m = s.scan_f[0];
    for (int w = 1; w < NW; ++w) m = fmaxf(m, s.scan_f[w]);
    row.cl.map_shared_rank(&s, t)->cta_max[rank] = m;
  }
  row.cl.sync();
  top = s.cta_max[0];
  for (int k = 1; k < ctas; ++k) top = fmaxf(top, s.cta_max[k]);

  const float temperature = set.temperature ? set.temperature[r] : set.temperature_all;
  const float top_p = set.top_p ? set.top_p[r] : set.top_p_all;
  const float min_p = set.min_p ? set.min_p[r] : set.min_p_all;
  int top_k = set.top_k ? set.top_k[r] : set.top_k_all;
  const bool greedy = !(temperature > 0.f);
  // Settings that leave the first-ranked token alone (a NaN does).
  if (!(top_p > 0.f) || !(min_p <= 1.f)) top_k = 1;
  if (top == -INFINITY) {  // the mask leaves nothing
    if (rank == 0 && t == 0) tokens[r] = -1, log_prob[r] = -INFINITY;
    row.cl.sync();
    return;
  }
  if (greedy || top_k == 1) {  // the lowest index of the largest logit
    int best = 0x7fffffff;
#pragma unroll
    for (int j = E - 1; j >= 0; --j)
      if (z[j] == top && row.index(j) < last) best = row.index(j);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = min(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) s.scan_i[warp] = best;
    __syncthreads();
    if (t == 0) {
      for (int w = 1; w < NW; ++w) best = min(best, s.scan_i[w]);
      row.cl.map_shared_rank(&s, 0)->cta_first[rank] = best;
    }
    row.cl.sync();
    if (rank == 0 && t == 0) {
      for (int k = 0; k < ctas; ++k) best = min(best, s.cta_first[k]);
      tokens[r] = best;
      log_prob[r] = 0.f;
    }
    return;
  }
  const float inv = 1.f / temperature;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    const float x = z[j];
    // Equal to the maximum: 0 (also where inf - inf is not a number). -inf, NaN: never drawn.
    float d = x == top ? 0.f : x > -INFINITY ? (top - x) * inv : INFINITY;
    z[j] = row.index(j) < last ? d : __uint_as_float(ABSENT);
  }
  bool fresh = false;
  if (top_k > 0 && top_k < vocab) row.cut(false, u64(top_k), fresh);
  if (top_p < 1.f) {
    u64 all;
    if (top_k > 0 && top_k < vocab) {
      all = s.mass_upto;
    } else {
      row.histogram(0, KEY_END, -1);
      fresh = true;
      all = 0;
      u64 m = 0;
      for (int b = t; b < NB; b += NT) m += s.total_mass[b];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
      if (lane == 0) s.scan_mass[warp] = m;
      __syncthreads();
      for (int w = 0; w < NW; ++w) all += s.scan_mass[w];
      __syncthreads();
    }
    const u64 need = u64(ceil(double(top_p) * double(all)));
    // A histogram of every token serves as one of the members: what the count
    // cut off lies past the boundary of the mass.
    row.cut(true, need > 0 ? need : 1, fresh);
  }
  // Mass of the kept tokens in vocabulary order.
  auto weight = [&](int j, u32& hi, u32& lo) {
    const float e = expf(-z[j]);
    hi = lo = 0;
    if (row.key(j) != ABSENT && row.member(j) && e >= min_p) mass_parts(e, hi, lo);
  };
  row.warp_sums(weight);
  row.scan_cta();
  u64 total = 0, before = 0;
  for (int k = 0; k < ctas; ++k) {
    if (k < rank) before += s.cta_mass[k];
    total += s.cta_mass[k];
  }
  const double u = double(uniform[r]) * double(total);
  u64 target = u > 0 ? u64(fmin(u, 1e18)) : 0;
  target = target < total ? target : total - 1;
  int idx;
  float zf;
  if (target >= before && target < before + s.cta_mass[rank] && row.find(target - before, weight, idx, zf)) {
    tokens[r] = idx;
    log_prob[r] = -zf - logf(float(double(total) * 0x1p-35));
  }
}

// Largest vocabulary: 16 CTAs of 32 values a thread.
constexpr int MAX_VOCAB = MAX_CTAS * NT * 32;

template <typename T, int E>
int launch(int rows, int vocab, int64_t ld, int ctas, const void* logits, const float* uniform, const Settings& set,
           int64_t* tokens, float* log_prob, cudaStream_t st) {
  const int slice = ((vocab + ctas - 1) / ctas + 7) & ~7;
  const bool vec = (ld * sizeof(T)) % 16 == 0 && aligned16(logits);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(rows) * ctas);
  cfg.blockDim = dim3(NT);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (ctas > 8 && cudaFuncSetAttribute(sample_kernel<T, E>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) !=
                      cudaSuccess)
    return M4_ERR_LAUNCH;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<T, E>, vocab, ld, slice, vec,
                                           static_cast<const T*>(logits), uniform, set, tokens, log_prob);
  return e == cudaSuccess ? launch_status() : M4_ERR_LAUNCH;
}

template <typename T>
int dispatch(int rows, int vocab, int64_t ld, const void* logits, const float* uniform, const Settings& set,
             int64_t* tokens, float* log_prob, cudaStream_t st) {
  int ctas = 1;
  while (ctas < 8 && ctas * NT * 16 < vocab) ctas *= 2;
  if (ctas * NT * 16 >= vocab)
    return launch<T, 16>(rows, vocab, ld, ctas, logits, uniform, set, tokens, log_prob, st);
  if (ctas * NT * 32 < vocab) ctas = 16;
  return launch<T, 32>(rows, vocab, ld, ctas, logits, uniform, set, tokens, log_prob, st);
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
  return bf16_logits ? dispatch<bf16>(rows, vocab, ld, logits, uniform, set, tokens, log_prob, st)
                     : dispatch<float>(rows, vocab, ld, logits, uniform, set, tokens, log_prob, st);
}
