// Decay attention (linear attention with a decay for each head), sm_100a.
//
//   S_t = e^g S_(t-1) + k_t v_t^T  [dk, dv],    o_t = scale q_t S_t
//
// over chunks of C = 64 tokens: with i, j counted inside a chunk of L tokens
// and S the state before it,
//   o_i = scale (sum_{j <= i} e^{g (i - j)} (q_i . k_j) v_j + e^{g (i + 1)} q_i S)
//   S'  = e^{g L} S + sum_j e^{g (L - 1 - j)} k_j v_j^T.
// The gradients are the same walk with its roles exchanged (D = dL/dS from the
// later tokens; a reverse walk counts from the sequence's end):
//   dq = walk(q = do, k = v, v = k),  dk = reverse(q = v, k = do, v = q),
//   dv = reverse(q = k, k = q, v = do), whose last state is dL/dS_initial.
// So one kernel, given operands, strides, direction and where the scale goes,
// is the forward pass and each part of the backward pass.
#include "common.cuh"

namespace m4 {
namespace decay {

using bf16 = __nv_bfloat16;
constexpr int C = 64;          // tokens per chunk
constexpr int MAX_DIM = 128;   // largest key or value dim

// An operand [B, T, heads, dim] (dim contiguous; strides in elements).
struct Operand {
  const void* p;
  int64_t sb, st, sh;
  int group;  // query heads per head of this operand
};

// One walk: a, b [.., da] in the places of q and k, c [.., dc] in that of v.
struct Pass {
  Operand a, b, c;
  int da, dc;
  void* out;            // [B, T, H, dc] dense
  int out_f32;
  const float* init;    // state [da, dc] before the walk, element (r, c) at r init_r + c init_c; NULL: zero
  float* fin;           // state after it, [da, dc] row-major; NULL: not wanted
  int init_r, init_c;
  int reverse;
  float in_scale;       // on a chunk's own products
  float read_scale;     // on reads of the carried state
  float write_scale;    // on what a chunk adds to the state
};
struct Problem {
  int B, T, H;
  const float* log_decay;
  const int* lengths;   // [B] or NULL
  Pass pass[3];
};

template <typename T>
M4_DEV const T* operand_at(const Operand& o, int b, int h) {
  return static_cast<const T*>(o.p) + b * o.sb + (h / o.group) * o.sh;
}

// e^{g i}, i = 0 .. 64 (g = -inf: 1, 0, 0, ...).
M4_DEV void decay_table(float* pw, float g) {
  for (int i = threadIdx.x; i <= C; i += blockDim.x) pw[i] = i ? expf(g * float(i)) : 1.f;
}

// ---------------------------------------------------------------------------
// The walk on the CUDA cores, fp32 throughout: float32 operands. 256 threads,
// tiles in shared memory, 4 x 4 scores and 4 x J outputs and state entries a
// thread. A CTA takes 16 J columns of the c operand and of the state (they do
// not interact): few heads and rows are spread over the GPU with J = 1 at the
// price of computing the scores once per CTA. Bound by shared-memory reads.
// ---------------------------------------------------------------------------
constexpr int ST = 256;

struct SimpleLayout {
  int da, q, k, v, s, p, pw, floats;
};
__host__ __device__ inline SimpleLayout simple_layout(int da, int width) {
  SimpleLayout l;
  l.da = (da + 15) & ~15;  // zero beyond the dim
  l.q = 0;
  l.k = l.q + C * (l.da + 4);
  l.v = l.k + C * (l.da + 4);
  l.s = l.v + C * (width + 4);
  l.p = l.s + l.da * (width + 4);
  l.pw = l.p + C * (C + 4);
  l.floats = l.pw + C + 4;
  return l;
}

M4_DEV void load_tile(float* dst, int width, const float* src, int64_t st, int dim, int valid) {
  if (dim % 4 == 0 && st % 4 == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
    const int w4 = width / 4;
    for (int i = threadIdx.x; i < C * w4; i += ST) {
      const int r = i / w4, c = 4 * (i - r * w4);
      cp16(dst + r * (width + 4) + c, r < valid && c < dim ? src + r * st + c : src, r < valid && c < dim);
    }
    return;
  }
  for (int i = threadIdx.x; i < C * width; i += ST) {
    const int r = i / width, c = i - r * width;
    cp4(dst + r * (width + 4) + c, r < valid && c < dim ? src + r * st + c : src, r < valid && c < dim);
  }
}
template <int J>
M4_DEV void load_cols(const float* p, float (&v)[J]) {
  if constexpr (J == 4) {
    const float4 x = ld4(p);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
  } else if constexpr (J == 2) {
    const float2 x = *reinterpret_cast<const float2*>(p);
    v[0] = x.x, v[1] = x.y;
  } else {
    v[0] = *p;
  }
}

// Output (r, c) of a chunk of L tokens from its tiles, without the places that the order masks.
__device__ __noinline__ float own_sum(const float* sm, const SimpleLayout& l, int r, int c, int wc, int L, bool rev,
                                      float read_scale) {
  const float* q = sm + l.q + r * (l.da + 4);
  float sum = 0.f;
  for (int d = 0; d < l.da; ++d) sum += q[d] * sm[l.s + d * wc + c];
  sum *= read_scale * sm[l.pw + (rev ? max(L - 1 - r, 0) : r + 1)];
  for (int j = rev ? r : 0; rev ? j < L : j <= r; ++j) sum += sm[l.p + r * (C + 4) + j] * sm[l.v + j * wc + c];
  return sum;
}

template <int J>
__global__ void __launch_bounds__(ST) walk_simple(const __grid_constant__ Problem pr) {
  constexpr int WIDTH = 16 * J, WC = WIDTH + 4, WP = C + 4;
  extern __shared__ float4 smem4[];
  float* sm = reinterpret_cast<float*>(smem4);
  const Pass& ps = pr.pass[blockIdx.z];
  const int h = blockIdx.x % pr.H, col0 = blockIdx.x / pr.H * WIDTH, b = blockIdx.y;
  if (col0 >= ps.dc) return;
  const int t = threadIdx.x, tx = t & 15, ty = t >> 4, dc = min(WIDTH, ps.dc - col0);
  const SimpleLayout l = simple_layout(ps.da, WIDTH);
  const int wa = l.da + 4;
  float *Q = sm + l.q, *K = sm + l.k, *V = sm + l.v, *S = sm + l.s, *P = sm + l.p, *pw = sm + l.pw;
  decay_table(pw, pr.log_decay[h]);
  int len = pr.T;
  if (pr.lengths) len = max(0, min(pr.T, pr.lengths[b]));
  const size_t state = (size_t(b) * pr.H + h) * ps.da * ps.dc;
  for (int i = t; i < l.da * WIDTH; i += ST) {
    const int r = i / WIDTH, c = i - r * WIDTH;
    S[r * WC + c] = ps.init && r < ps.da && c < dc ? ps.init[state + r * ps.init_r + (col0 + c) * ps.init_c] : 0.f;
  }
  const float* qa = operand_at<float>(ps.a, b, h);
  const float* kb = operand_at<float>(ps.b, b, h);
  const float* vc = operand_at<float>(ps.c, b, h) + col0;
  const int64_t row = int64_t(pr.H) * ps.dc;
  float* out = static_cast<float*>(ps.out) + int64_t(b) * pr.T * row + int64_t(h) * ps.dc + col0;
  const int chunks = (len + C - 1) / C;
  const bool rev = ps.reverse;
  const int c0 = J * tx;
  for (int n = 0; n < chunks; ++n) {
    const int t0 = (rev ? chunks - 1 - n : n) * C, L = min(C, len - t0);
    __syncthreads();
    load_tile(Q, l.da, qa + t0 * ps.a.st, ps.a.st, ps.da, L);
    load_tile(K, l.da, kb + t0 * ps.b.st, ps.b.st, ps.da, L);
    load_tile(V, WIDTH, vc + t0 * ps.c.st, ps.c.st, dc, L);
    cp_wait();
    __syncthreads();
    // Scores: rows 4 ty .., columns tx + 16 j; a block of 16 columns that the order masks is skipped.
    const int first = rev ? (4 * ty) / 16 : 0, past = rev ? 4 : (4 * ty + 3) / 16 + 1;
    {
      float acc[4][4] = {};
      for (int d = 0; d < l.da; d += 4) {
        float4 q[4], k[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          q[i] = ld4(Q + (4 * ty + i) * wa + d);
          if (i >= first && i < past) k[i] = ld4(K + (tx + 16 * i) * wa + d);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j >= first && j < past)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[i][j] += q[i].x * k[j].x + q[i].y * k[j].y + q[i].z * k[j].z + q[i].w * k[j].w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 4 * ty + i, c = tx + 16 * j, gap = rev ? c - r : r - c;
          P[r * WP + c] = gap >= 0 ? acc[i][j] * (ps.in_scale * pw[gap]) : 0.f;
        }
    }
    __syncthreads();
    {  // outputs
      float acc[4][J] = {};
      for (int d = 0; d < l.da; d += 4) {
        float4 q[4];
        float s[4][J];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = ld4(Q + (4 * ty + i) * wa + d), load_cols<J>(S + (d + i) * WC + c0, s[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < J; ++j)
            acc[i][j] += q[i].x * s[0][j] + q[i].y * s[1][j] + q[i].z * s[2][j] + q[i].w * s[3][j];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * ty + i, e = rev ? L - 1 - r : r + 1;
        const float f = ps.read_scale * pw[max(e, 0)];
#pragma unroll
        for (int j = 0; j < J; ++j) acc[i][j] *= f;
      }
      for (int j0 = 16 * first; j0 < 16 * past; j0 += 4) {
        float4 p[4];
        float v[4][J];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = ld4(P + (4 * ty + i) * WP + j0), load_cols<J>(V + (j0 + i) * WC + c0, v[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < J; ++j)
            acc[i][j] += p[i].x * v[0][j] + p[i].y * v[1][j] + p[i].z * v[2][j] + p[i].w * v[3][j];
      }
      // A masked place's zero times a value that is not finite is NaN: the sums anew, over each row's own places
      // (32 rows x 1024 tokens x 8 heads, 64 x 128: 645 us, 2.5 ms where every value is NaN).
      bool nan = false;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < J; ++j) nan |= acc[i][j] != acc[i][j];
      if (nan)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < J; ++j) acc[i][j] = own_sum(sm, l, 4 * ty + i, c0 + j, WC, L, rev, ps.read_scale);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (4 * ty + i < L && c0 + j < dc) out[(t0 + 4 * ty + i) * row + c0 + j] = acc[i][j];
    }
    __syncthreads();
    // The weights go on the values once, then the state: rows 4 ty + r0 .., columns c0 ...
    for (int i = t; i < C * WIDTH; i += ST) {
      const int r = i / WIDTH;
      V[r * WC + i - r * WIDTH] *= ps.write_scale * pw[rev ? r + 1 : max(L - 1 - r, 0)];
    }
    __syncthreads();
    const float f = pw[L];
    for (int r0 = 4 * ty; r0 < l.da; r0 += 64) {
      float acc[4][J] = {};
#pragma unroll 4
      for (int j = 0; j < L; ++j) {
        const float4 k = ld4(K + j * wa + r0);
        float v[J];
        load_cols<J>(V + j * WC + c0, v);
#pragma unroll
        for (int c = 0; c < J; ++c) acc[0][c] += k.x * v[c], acc[1][c] += k.y * v[c], acc[2][c] += k.z * v[c], acc[3][c] += k.w * v[c];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < J; ++c) {
          float* s = S + (r0 + i) * WC + c0 + c;
          *s = f * *s + acc[i][c];
        }
    }
  }
  __syncthreads();
  if (ps.fin)
    for (int i = t; i < ps.da * WIDTH; i += ST) {
      const int r = i / WIDTH, c = i - r * WIDTH;
      if (c < dc) ps.fin[state + size_t(r) * ps.dc + col0 + c] = S[r * WC + c];
    }
  // Rows past the sequence's end.
  for (int64_t r = len + ty; r < pr.T; r += 16)
    for (int c = tx; c < dc; c += 16) out[r * row + c] = 0.f;
}

// Sum of the query heads' parts of a shared head: part [B, T, H, D] -> out [B, T, H / group, D].
template <typename T>
__global__ void __launch_bounds__(256) group_sum(int64_t n, int group, int dim, const float* __restrict__ part,
                                                 T* __restrict__ out) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t head = i / dim;
  const float* p = part + head * group * dim + i % dim;
  float s = 0.f;
  for (int g = 0; g < group; ++g) s += p[int64_t(g) * dim];
  out[i] = from_f<T>(s);
}

// ---------------------------------------------------------------------------
// One token: S' = e^g S + k v^T, o = scale q S'. Bound by HBM (the state is
// read and written once). A CTA per (b, h); `lanes` neighbouring threads hold
// a state row as float4, so a warp's accesses are whole lines; a thread has 8
// of them on their way. 64 sequences of 16 heads, 128 x 128 states (135 MB):
// 25.5 us, 5.3 TB/s (a copy: 6.6); one sequence 3.3 us, latency.
// ---------------------------------------------------------------------------
constexpr int DT = 256;

template <typename T>
__global__ void __launch_bounds__(DT) step_kernel(int H, int group, int dk, int dv, int lanes, bool vec, float scale,
                                                  const float* state, const T* __restrict__ q,
                                                  const T* __restrict__ k, const T* __restrict__ v,
                                                  const float* __restrict__ log_decay, T* __restrict__ out,
                                                  float* state_out) {
  __shared__ float ks[MAX_DIM], qs[MAX_DIM];
  __shared__ float sums[DT * 4];
  const int bh = blockIdx.x, b = bh / H, h = bh - b * H, t = threadIdx.x;
  const int kvh = b * (H / group) + h / group;
  for (int i = t; i < dk; i += DT) ks[i] = to_f<T>(k[size_t(kvh) * dk + i]), qs[i] = to_f<T>(q[size_t(bh) * dk + i]);
  const float gamma = expf(log_decay[h]);
  const int c = 4 * (t & (lanes - 1)), r0 = t / lanes, rows = DT / lanes;
  float vv[4], acc[4] = {};
#pragma unroll
  for (int j = 0; j < 4; ++j) vv[j] = c + j < dv ? to_f<T>(v[size_t(kvh) * dv + c + j]) : 0.f;
  __syncthreads();
  const float* src = state + size_t(bh) * dk * dv + c;
  float* dst = state_out + size_t(bh) * dk * dv + c;
  if (vec) {
    if (c < dv)
      for (int r = r0; r < dk; r += 8 * rows) {
        float4 s[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (r + u * rows < dk) s[u] = ld4(src + size_t(r + u * rows) * dv);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int i = r + u * rows;
          if (i >= dk) break;
          const float kk = ks[i], qq = qs[i];
          s[u].x = gamma * s[u].x + kk * vv[0];
          s[u].y = gamma * s[u].y + kk * vv[1];
          s[u].z = gamma * s[u].z + kk * vv[2];
          s[u].w = gamma * s[u].w + kk * vv[3];
          st4(dst + size_t(i) * dv, s[u]);
          acc[0] += qq * s[u].x, acc[1] += qq * s[u].y, acc[2] += qq * s[u].z, acc[3] += qq * s[u].w;
        }
      }
  } else {
    for (int r = r0; r < dk; r += rows)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < dv) {
          const float s = gamma * src[size_t(r) * dv + j] + ks[r] * vv[j];
          dst[size_t(r) * dv + j] = s;
          acc[j] += qs[r] * s;
        }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) sums[r0 * 4 * lanes + c + j] = acc[j];
  __syncthreads();
  if (t < dv) {
    float s = 0.f;
    for (int r = 0; r < rows; ++r) s += sums[r * 4 * lanes + t];
    out[size_t(bh) * dv + t] = from_f<T>(scale * s);
  }
}

}  // namespace decay
}  // namespace m4

#include "decay_tc.cuh"

namespace m4 {
namespace decay {

inline int check(const M4DecayDims* d) {
  if (!d) return M4_ERR_NULL;
  if (d->batch <= 0 || d->time <= 0 || d->heads <= 0 || d->kv_heads <= 0 || d->key_dim <= 0 || d->value_dim <= 0 ||
      d->heads % d->kv_heads)
    return M4_ERR_DIMS;
  if (d->key_dim > MAX_DIM || d->value_dim > MAX_DIM || d->batch > 65535 || d->heads > 65535)
    return M4_ERR_UNSUPPORTED;
  if (d->bf16 && (d->key_dim % 8 || d->value_dim % 8)) return M4_ERR_UNSUPPORTED;
  return M4_OK;
}

template <int J>
int launch_simple(const Problem& pr, int passes, cudaStream_t st) {
  int floats = 0, tiles = 0;
  for (int i = 0; i < passes; ++i) {
    const int n = simple_layout(pr.pass[i].da, 16 * J).floats, m = (pr.pass[i].dc + 16 * J - 1) / (16 * J);
    floats = n > floats ? n : floats;
    tiles = m > tiles ? m : tiles;
  }
  if (!allow_shared<walk_simple<J>>(floats * 4)) return M4_ERR_LAUNCH;
  walk_simple<J><<<dim3(pr.H * tiles, pr.B, passes), ST, floats * 4, st>>>(pr);
  return launch_status();
}
// Columns per CTA: 16, 32 or 64, whichever gives the SM with the most CTAs the
// least to do. A CTA alone takes 1 : 1.07 : 1.29 of the time (64 x 128, T 512:
// 82, 88, 107 us), each further one on its SM about 0.7 of that. Measured with
// 16, 32 and 64 columns, us: 12 walks of 64 x 128: 82, 88, 107; 48: 182, 124,
// 108; 160: 497, 332, 268; 48 walks of 40 x 72: 91, 78, 94; 64: 157, 104, 94;
// 80: 158, 105, 137; 320: 516, 383, 365.
inline int run_simple(const Problem& pr, int passes, cudaStream_t st) {
  const float alone[3] = {1.f, 1.07f, 1.29f};
  int best = 0;
  float least = INFINITY;
  for (int i = 0; i < 3; ++i) {
    int64_t ctas = 0;
    for (int p = 0; p < passes; ++p) ctas += int64_t(pr.H) * pr.B * ((pr.pass[p].dc + (16 << i) - 1) / (16 << i));
    const float cost = alone[i] * (1.f + 0.7f * float((ctas + 147) / 148 - 1));
    if (cost < least) best = i, least = cost;
  }
  return best == 0 ? launch_simple<1>(pr, passes, st)
                   : best == 1 ? launch_simple<2>(pr, passes, st) : launch_simple<4>(pr, passes, st);
}

// Segments of the time axis (bfloat16): one where the heads and rows fill the
// GPU; else as many as fill it, of at least MIN_SEGMENT chunks, if there are
// MIN_COUNT of them. Each segment's own contribution to the state is walked
// first (keys and values are read twice, two launches more): 8 chunks of 30
// heads ran 23 us whole and 30 us in two segments, 13 chunks 34 us whole and
// 33 us in three, 512 chunks of 8 heads about 1200 us whole and 114 us in 18.
constexpr int MIN_SEGMENT = 4, MIN_COUNT = 4;
struct Segments {
  int count, tokens;
  size_t floats;  // per pass
};
inline Segments segments_of(const M4DecayDims* d, int passes) {
  const int64_t walks = int64_t(d->batch) * d->heads * passes;
  const int chunks = (d->time + C - 1) / C;
  const int slots = d->key_dim <= 64 && d->value_dim <= 64 ? 296 : 148;
  int count = 1;
  if (d->bf16) {
    count = int(slots / walks);
    if (count > chunks / MIN_SEGMENT) count = chunks / MIN_SEGMENT;
    if (count < MIN_COUNT) count = 1;
  }
  const int per = (chunks + count - 1) / count;
  count = (chunks + per - 1) / per;
  return Segments{count, per * C, size_t(d->batch) * d->heads * count * d->key_dim * d->value_dim};
}

// Tensor map of an operand [B][T][heads][dim] (bfloat16): boxes of 64 columns
// x 1 head x 64 tokens x 1 row, 128-byte swizzle; places outside read as 0.
inline int encode(CUtensorMap* map, const Operand& o, int B, int T, int heads, int dim) {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    PFN_cuTensorMapEncodeTiled_v12000 f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", reinterpret_cast<void**>(&f), cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return f;
  }();
  // (a driver call wants the device's context current in this host thread: a
  // framework's backward thread may not have made a runtime call yet)
  int device;
  if (!fn || cudaGetDevice(&device) != cudaSuccess || cudaSetDevice(device) != cudaSuccess) return M4_ERR_LAUNCH;
  const cuuint64_t size[4] = {cuuint64_t(dim), cuuint64_t(heads), cuuint64_t(T), cuuint64_t(B)};
  const int64_t st[3] = {o.sh, o.st, o.sb};
  cuuint64_t stride[3];
  for (int i = 0; i < 3; ++i) {
    stride[i] = size[i + 1] > 1 ? cuuint64_t(st[i]) * 2 : 16;  // (an axis of one place has no stride)
    if (size[i + 1] > 1 && st[i] <= 0) return M4_ERR_UNSUPPORTED;
    if (stride[i] % 16) return M4_ERR_ALIGN;
  }
  if (!aligned16(o.p)) return M4_ERR_ALIGN;
  const cuuint32_t box[4] = {64, 1, 64, 1}, elem[4] = {1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(o.p), size, stride, box, elem,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? M4_OK
             : M4_ERR_UNSUPPORTED;
}

template <auto K, int THREADS, int SMEM, bool SHARED_REGS>
int launch_walk(const TcProblem& tp, int passes, bool after, cudaStream_t st) {
  if (!allow_shared<K>(SMEM)) return M4_ERR_LAUNCH;
  if (SHARED_REGS) {
    // The groups' shares add up to 80 registers a thread: with fewer at launch they would wait for ever.
    static const int registers = [] {
      cudaFuncAttributes a;
      return cudaFuncGetAttributes(&a, K) == cudaSuccess ? a.numRegs : 0;
    }();
    if (registers < 80) return M4_ERR_LAUNCH;
  }
  const dim3 grid(unsigned(tp.pr.B) * tp.segments, tp.pr.H, passes);
  if (after) return launch_after(K, grid, THREADS, SMEM, st, tp);
  K<<<grid, THREADS, SMEM, st>>>(tp);
  return launch_status();
}
template <bool READ, int DA, int DC>
int launch_one(const TcProblem& tp, int passes, bool after, cudaStream_t st) {
  using G = Geo<DA, DC, READ>;
  return launch_walk<walk_tc<DA, DC, READ>, G::THREADS, G::SMEM, G::SHARE_REGS>(tp, passes, after, st);
}
template <bool READ>
int launch_any(const TcProblem& tp, int passes, bool after, cudaStream_t st) {
  const bool wa = tp.pr.pass[0].da > 64, wc = tp.pr.pass[0].dc > 64;
  if (passes > 1 && wa != wc) {
    using G = Geo<64, 128, READ>;
    using H = Geo<128, 64, READ>;
    return launch_walk<walk_mixed<READ>, G::THREADS, (G::SMEM > H::SMEM ? G::SMEM : H::SMEM), true>(tp, passes, after, st);
  }
  return wa ? (wc ? launch_one<READ, 128, 128>(tp, passes, after, st) : launch_one<READ, 128, 64>(tp, passes, after, st))
            : (wc ? launch_one<READ, 64, 128>(tp, passes, after, st) : launch_one<READ, 64, 64>(tp, passes, after, st));
}

// One pass (forward) or the three of the backward, whose dims are the forward's in either order.
inline int run_tc(TcProblem& tp, int passes, cudaStream_t st) {
  for (int i = 0; i < passes; ++i) {
    const Pass& p = tp.pr.pass[i];
    const int64_t row = int64_t(tp.pr.H) * p.dc;
    const Operand out{p.out, row * tp.pr.T, row, p.dc, 1};
    if (!p.out_f32)
      if (const int e = encode(&tp.out_maps[i], out, tp.pr.B, tp.pr.T, tp.pr.H, p.dc)) return e;
  }
  if (tp.segments > 1) {  // (the launches overlap: a long prompt among others 117 us, 120 one after another)
    if (const int e = launch_any<false>(tp, passes, false, st)) return e;
    const Pass& p = tp.pr.pass[0];
    if (const int e = launch_after(join_segments, dim3((p.da * p.dc + 255) / 256, tp.pr.B * tp.pr.H, passes), 256, 0,
                                   st, tp))
      return e;
  }
  return launch_any<true>(tp, passes, tp.segments > 1, st);
}

inline Problem problem_of(const M4DecayDims* d, const float* log_decay, const int* lengths) {
  Problem pr = {};
  pr.B = d->batch;
  pr.T = d->time;
  pr.H = d->heads;
  pr.log_decay = log_decay;
  pr.lengths = lengths;
  return pr;
}
inline Operand operand(const void* p, const int64_t* strides, int group) {
  return Operand{p, strides[0], strides[1], strides[2], group};
}

}  // namespace decay
}  // namespace m4

extern "C" size_t m4_decay_fwd_workspace_bytes(const M4DecayDims* d) {
  using namespace m4::decay;
  if (check(d) != M4_OK) return 0;
  const Segments s = segments_of(d, 1);
  return 256 + (s.count > 1 ? m4::align256(s.floats * 4) : 0);
}

extern "C" int m4_decay_fwd(const M4DecayDims* d, const void* q, const void* k, const void* v, const float* log_decay,
                            const int* lengths, const float* initial, void* output, float* final_state,
                            void* workspace, size_t workspace_bytes, void* stream) {
  using namespace m4::decay;
  if (const int e = check(d)) return e;
  if (!q || !k || !v || !log_decay || !output || !final_state || !workspace) return M4_ERR_NULL;
  if (workspace_bytes < m4_decay_fwd_workspace_bytes(d)) return M4_ERR_WORKSPACE;
  const int group = d->heads / d->kv_heads;
  Problem pr = problem_of(d, log_decay, lengths);
  pr.pass[0] = Pass{operand(q, d->q_strides, 1), operand(k, d->k_strides, group), operand(v, d->v_strides, group),
                    d->key_dim, d->value_dim, output, 0, initial, final_state, d->value_dim, 1, 0,
                    d->scale, d->scale, 1.f};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!d->bf16) return run_simple(pr, 1, st);
  if (!m4::all_aligned16(output, workspace)) return M4_ERR_ALIGN;
  const Segments sg = segments_of(d, 1);
  TcProblem tp = {};
  tp.pr = pr;
  const Pass& p = pr.pass[0];
  if (const int e = encode(&tp.maps[0], p.a, pr.B, pr.T, d->heads, d->key_dim)) return e;
  if (const int e = encode(&tp.maps[1], p.b, pr.B, pr.T, d->kv_heads, d->key_dim)) return e;
  if (const int e = encode(&tp.maps[2], p.c, pr.B, pr.T, d->kv_heads, d->value_dim)) return e;
  for (int i = 0; i < 3; ++i) tp.map_of[0][i] = i;
  tp.segments = sg.count;
  tp.segment_tokens = sg.tokens;
  tp.seg_state = reinterpret_cast<float*>(static_cast<char*>(workspace) + 256);
  tp.seg_pass = sg.floats;
  return run_tc(tp, 1, st);
}

extern "C" size_t m4_decay_bwd_workspace_bytes(const M4DecayDims* d) {
  using namespace m4::decay;
  if (check(d) != M4_OK) return 0;
  const Segments s = segments_of(d, 2);
  size_t n = 256 + (s.count > 1 ? 3 * m4::align256(s.floats * 4) : 0);
  if (d->heads != d->kv_heads)
    n += m4::align256(size_t(d->batch) * d->time * d->heads * d->key_dim * 4) +
         m4::align256(size_t(d->batch) * d->time * d->heads * d->value_dim * 4);
  return n;
}

extern "C" int m4_decay_bwd(const M4DecayDims* d, const void* q, const void* k, const void* v, const float* log_decay,
                            const int* lengths, const float* initial, const void* d_output, const float* d_final,
                            void* dq, void* dk, void* dv, float* d_initial, void* workspace, size_t workspace_bytes,
                            void* stream) {
  using namespace m4::decay;
  if (const int e = check(d)) return e;
  if (!q || !k || !v || !log_decay || !d_output || !dq || !dk || !dv || !workspace) return M4_ERR_NULL;
  if (workspace_bytes < m4_decay_bwd_workspace_bytes(d)) return M4_ERR_WORKSPACE;
  const int group = d->heads / d->kv_heads, n = d->key_dim, p = d->value_dim;
  const size_t tokens = size_t(d->batch) * d->time;
  const Segments sg = segments_of(d, 2);
  float* seg_state = reinterpret_cast<float*>(static_cast<char*>(workspace) + 256);
  float* dk_part = seg_state + (sg.count > 1 ? 3 * m4::align256(sg.floats * 4) / 4 : 0);
  float* dv_part = dk_part + m4::align256(tokens * d->heads * n * 4) / 4;
  const Operand Q = operand(q, d->q_strides, 1), K = operand(k, d->k_strides, group),
                V = operand(v, d->v_strides, group);
  const Operand G{d_output, int64_t(d->time) * d->heads * p, int64_t(d->heads) * p, p, 1};
  Problem pr = problem_of(d, log_decay, lengths);
  const float s = d->scale;
  const bool shared = group > 1;
  pr.pass[0] = Pass{G, V, K, p, n, dq, 0, initial, nullptr, 1, p, 0, s, s, 1.f};
  pr.pass[1] = Pass{V, G, Q, p, n, shared ? dk_part : dk, shared, d_final, nullptr, 1, p, 1, s, 1.f, s};
  pr.pass[2] = Pass{K, Q, G, n, p, shared ? dv_part : dv, shared, d_final, d_initial, p, 1, 1, s, 1.f, s};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!d->bf16) {
    if (const int e = run_simple(pr, 3, st)) return e;
  } else {
    if (!m4::all_aligned16(dq, dk, dv, workspace)) return M4_ERR_ALIGN;
    TcProblem tp = {};
    tp.pr = pr;
    if (const int e = encode(&tp.maps[0], Q, pr.B, pr.T, d->heads, n)) return e;
    if (const int e = encode(&tp.maps[1], K, pr.B, pr.T, d->kv_heads, n)) return e;
    if (const int e = encode(&tp.maps[2], V, pr.B, pr.T, d->kv_heads, p)) return e;
    if (const int e = encode(&tp.maps[3], G, pr.B, pr.T, d->heads, p)) return e;
    const int of[3][3] = {{3, 2, 1}, {2, 3, 0}, {1, 0, 3}};
    for (int i = 0; i < 9; ++i) tp.map_of[i / 3][i % 3] = of[i / 3][i % 3];
    tp.segments = sg.count;
    tp.segment_tokens = sg.tokens;
    tp.seg_state = seg_state;
    tp.seg_pass = m4::align256(sg.floats * 4) / 4;
    if (const int e = run_tc(tp, 3, st)) return e;
  }
  if (shared) {
    const int64_t nk = int64_t(tokens) * d->kv_heads * n, nv = int64_t(tokens) * d->kv_heads * p;
    if (d->bf16) {
      group_sum<bf16><<<unsigned((nk + 255) / 256), 256, 0, st>>>(nk, group, n, dk_part, static_cast<bf16*>(dk));
      group_sum<bf16><<<unsigned((nv + 255) / 256), 256, 0, st>>>(nv, group, p, dv_part, static_cast<bf16*>(dv));
    } else {
      group_sum<float><<<unsigned((nk + 255) / 256), 256, 0, st>>>(nk, group, n, dk_part, static_cast<float*>(dk));
      group_sum<float><<<unsigned((nv + 255) / 256), 256, 0, st>>>(nv, group, p, dv_part, static_cast<float*>(dv));
    }
  }
  return m4::launch_status();
}

int m4::decay_timeout() { return m4::tc::take_timeout(); }

extern "C" int m4_decay_step(const M4DecayDims* d, const float* state, const void* q, const void* k, const void* v,
                             const float* log_decay, void* output, float* state_out, void* stream) {
  using namespace m4::decay;
  if (!d) return M4_ERR_NULL;
  M4DecayDims one = *d;
  one.time = 1;
  one.bf16 = 0;  // (any dims)
  one.batch = one.batch > 0 ? 1 : one.batch;  // (batch has no grid limit here)
  if (const int e = check(&one)) return e;
  if (int64_t(d->batch) * d->heads > 0x7fffffff) return M4_ERR_UNSUPPORTED;
  if (!state || !q || !k || !v || !log_decay || !output || !state_out) return M4_ERR_NULL;
  int lanes = 1;
  while (4 * lanes < d->value_dim) lanes *= 2;
  const bool vec = d->value_dim % 4 == 0 && m4::all_aligned16(state, state_out);
  const int group = d->heads / d->kv_heads;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned grid = unsigned(d->batch) * d->heads;
  if (d->bf16)
    step_kernel<bf16><<<grid, DT, 0, st>>>(d->heads, group, d->key_dim, d->value_dim, lanes, vec, d->scale, state,
                                           static_cast<const bf16*>(q), static_cast<const bf16*>(k),
                                           static_cast<const bf16*>(v), log_decay, static_cast<bf16*>(output),
                                           state_out);
  else
    step_kernel<float><<<grid, DT, 0, st>>>(d->heads, group, d->key_dim, d->value_dim, lanes, vec, d->scale, state,
                                            static_cast<const float*>(q), static_cast<const float*>(k),
                                            static_cast<const float*>(v), log_decay, static_cast<float*>(output),
                                            state_out);
  return m4::launch_status();
}
