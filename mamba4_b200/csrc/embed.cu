// Embedding lookup with scaling, and its gradient by sorted tokens (sm_100a).
//
//   out[i] = round(scale W[tok_i])            (zero for ids outside [0, V))
//   dW[v]  = scale sum_{i : tok_i = v} g_i    (fp32)
//
// Both are bound by HBM: the lookup reads the N rows it needs and writes N
// rows, the gradient reads N rows and writes all V. The gradient needs the
// positions of every id, in order. No full sort: ids are put in ranges of
// R = 2^s ids and
//   1. tile_kernel   sorts each tile of 1024 tokens by range (stable), and
//                    writes how many of the tile's tokens precede each range;
//   2. sort_kernel   one CTA per range: its tokens from all tiles (their place
//                    in the whole order is the sum of the preceding counts)
//                    and a stable counting sort by id;
//   3. sum_kernel    a block per ROWS gradient rows: a warp writes the zeros or
//                    adds the row where at most SHORT tokens ask for the id,
//                    the block's warps share a row of at most LONG. Ids with
//                    more come in pieces of LONG positions, which the first
//                    blocks take; the piece that finishes last adds the partial
//                    sums in the order of the pieces.
// Every sum has a fixed order, so results repeat bit for bit: up to SHORT places
// in ascending order; above, ascending runs of them, whose sums are joined in
// order.
//
// The choices below, as lookup and gradient in us at (32768 tokens x 512, 65536
// x 768): as they are 57, 105; QT 128: 62, 115, 512: 65, 107; SHORT 1: 63, 121,
// 16: 61, 106; LONG 32: 58, 110; ROWS 64: 59, 106; PIECE_BLOCKS 148: 57, 106,
// 592: 59, 108.
//
// Measured (B200; each alone, cold L2): 65536 tokens of a 50304 x 768 table,
// bfloat16 gradients to a float32 table (405 MB with the lookup of 15750 different
// rows, 62 us at the copy bandwidth): lookup 28 us, tiles 10, sort 21, sums 53;
// together, warm, 105 us. 32768 tokens x 512: 57 us against 29. What is left above
// the bandwidth is the sort, 31 us of dependent steps (counts, scan, places; it
// moves 1 MB), and the latency of rows with few tokens. Float32 gradients: 166 us
// against 92, and 76 against 39. Width 1024: 140 us against 82 (bfloat16).
#include "common.cuh"

namespace m4 {
namespace embed {

using bf16 = __nv_bfloat16;

constexpr int TILE = 1024;       // tokens per tile (one thread each)
constexpr int MAX_RANGES = 1024;
constexpr int MAX_R = 2048;      // ids per range
constexpr int RT = 256;          // threads of sum_kernel
constexpr int RW = RT / 32;
constexpr int QT = 256;          // threads of sort_kernel: a range has tens of tokens as a rule
constexpr int QW = QT / 32;
constexpr int LONG = 64;         // positions per piece
constexpr int SHORT = 4;         // positions that one warp adds
constexpr int CACHED = 4096;     // tokens of a range held in shared memory
constexpr int ROWS = 32;         // gradient rows per block of sum_kernel
constexpr int HELD = 1024;       // their positions held in shared memory
constexpr int PIECE_BLOCKS = 296; // blocks of sum_kernel that take the pieces

// Eight consecutive elements as float.
template <typename T> struct Vec8;
template <> struct Vec8<float> {
  static M4_DEV void load(const float* p, float (&v)[8]) {
    const float4 a = ld4(p), b = ld4(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  static M4_DEV void store(float* p, const float (&v)[8]) {
    st4(p, make_float4(v[0], v[1], v[2], v[3]));
    st4(p + 4, make_float4(v[4], v[5], v[6], v[7]));
  }
};
template <> struct Vec8<bf16> {
  static M4_DEV void load(const bf16* p, float (&v)[8]) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static M4_DEV void store(bf16* p, const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// Eight floats as one 32-byte store (`wide`: the address is a multiple of 32):
// two 16-byte stores leave each 32-byte sector half written at a time (lookup and
// gradient of 32768 x 512: 57 us, with them 60; 65536 x 768: 105, 108).
M4_DEV void store_wide(float* p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]),
               "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
M4_DEV void store_wide(bf16* p, const float (&v)[8]) { Vec8<bf16>::store(p, v); }

// Columns c .. c + 7 of a row (those below dim; `vec`: 16-byte access allowed).
template <typename T>
M4_DEV void load8(const T* row, int c, int dim, bool vec, float (&v)[8]) {
  if (vec) return Vec8<T>::load(row + c, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = c + i < dim ? to_f<T>(row[c + i]) : 0.f;
}
template <typename T>
M4_DEV void store8(T* row, int c, int dim, bool vec, const float (&v)[8]) {
  if (vec) return Vec8<T>::store(row + c, v);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c + i < dim) row[c + i] = from_f<T>(v[i]);
}

// `lanes` (a power of two) neighbouring threads per row, 8 columns each per
// step. 64 rows: 2.3 us, the latency of an id's load, its row's and the store.
template <typename W, typename O>
__global__ void __launch_bounds__(256) lookup_kernel(int64_t rows, int vocab, int dim, int lanes, bool vec,
                                                     const int64_t* __restrict__ tokens,
                                                     const W* __restrict__ weight, float scale,
                                                     O* __restrict__ out) {
  const int64_t i = (int64_t(blockIdx.x) * 256 + threadIdx.x) / lanes;
  if (i >= rows) return;
  const int64_t tok = tokens[i];
  const bool inside = tok >= 0 && tok < vocab;
  const W* src = weight + (inside ? tok : 0) * int64_t(dim);
  O* dst = out + i * int64_t(dim);
#pragma unroll 2
  for (int c = 8 * (threadIdx.x & (lanes - 1)); c < dim; c += 8 * lanes) {
    float v[8] = {};
    if (inside) load8(src, c, dim, vec, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = inside ? v[j] * scale : 0.f;
    store8(dst, c, dim, vec, v);
  }
}

// Workspace of the gradient.
struct Work {
  uint16_t* offs;    // [ranges + 1][tiles]: tokens of the tile in ranges below
  uint32_t* local;   // [tiles * TILE]: (id in range << 10) | place in tile, by range
  int32_t* perm;     // [rows]: positions sorted by id
  uint64_t* list;    // [rows]: ids and positions in token order, for ranges that exceed shared memory
  int* items;        // [max_items][4]: id, first, count, head item of the id
  float* part;       // [max_items][part_width] partial sums
  int* arrived;      // [max_items] pieces done (at the id's head item)
  int* start;        // [ranges << shift, + 1]: first place of each id in perm
  int* n_items;
};

struct Plan {
  int64_t rows;
  int vocab, dim, shift, ranges, tiles;
  int64_t max_items;
  size_t offs_at, local_at, perm_at, list_at, items_at, part_at, arrived_at, start_at, bytes;
};

// Columns of a partial sum (whole vectors).
__host__ __device__ inline size_t part_width(int dim) { return size_t(dim + 7) & ~size_t(7); }

// Range size: the smallest power of two that gives at most MAX_RANGES ranges
// (at least 16 ids). Many small ranges keep every SM busy to the end.
inline bool plan_for(int64_t rows, int vocab, int dim, Plan* p) {
  if (rows <= 0 || rows > (int64_t(1) << 28) || vocab <= 0 || dim <= 0) return false;
  p->rows = rows;
  p->vocab = vocab;
  p->dim = dim;
  p->shift = 4;
  while (((int64_t(vocab) + (1 << p->shift) - 1) >> p->shift) > MAX_RANGES) ++p->shift;
  if ((1 << p->shift) > MAX_R) return false;
  p->ranges = (vocab + (1 << p->shift) - 1) >> p->shift;
  p->tiles = int((rows + TILE - 1) / TILE);
  // A long id has more than LONG tokens and ceil(tokens / LONG) pieces: at most 2 rows / LONG.
  p->max_items = 2 * rows / LONG + 1;
  size_t at = 0;
  auto take = [&](size_t n) { const size_t o = at; at += align256(n); return o; };
  take(sizeof(int));
  p->offs_at = take(size_t(p->ranges + 1) * p->tiles * 2);
  p->local_at = take(size_t(p->tiles) * TILE * 4);
  p->perm_at = take(size_t(rows) * 4);
  p->list_at = take(size_t(rows) * 8);
  p->items_at = take(size_t(p->max_items) * 16);
  p->part_at = take(size_t(p->max_items) * part_width(dim) * 4);
  p->arrived_at = take(size_t(p->max_items) * 4);
  p->start_at = take((size_t(p->ranges) << p->shift) * 4 + 4);
  p->bytes = at;
  return true;
}

inline Work work_of(const Plan& p, void* w) {
  char* b = static_cast<char*>(w);
  return Work{reinterpret_cast<uint16_t*>(b + p.offs_at), reinterpret_cast<uint32_t*>(b + p.local_at),
              reinterpret_cast<int32_t*>(b + p.perm_at),  reinterpret_cast<uint64_t*>(b + p.list_at),
              reinterpret_cast<int*>(b + p.items_at),
              reinterpret_cast<float*>(b + p.part_at),    reinterpret_cast<int*>(b + p.arrived_at),
              reinterpret_cast<int*>(b + p.start_at),     reinterpret_cast<int*>(b)};
}

// Exclusive scan of one value per thread over a block of NW warps; `total` for everyone.
template <int NW>
M4_DEV int block_exclusive(int v, int* scratch, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += n;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = s;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const int n = scratch[w];
    before += w < warp ? n : 0;
    all += n;
  }
  total = all;
  return before + s - v;
}

// Stable sort of a tile by range: place = tokens of lower ranges + of the same
// range in lower warps + in lower lanes (a match within the warp), so no
// atomics. Shared: counts [32 warps][ranges] (16 bits). Bound by its barriers
// and shared-memory passes (10 us for 64 tiles, one a block).
__global__ void __launch_bounds__(TILE) tile_kernel(int64_t rows, int vocab, int shift, int ranges, int tiles,
                                                    const int64_t* __restrict__ tokens, Work w) {
  extern __shared__ uint16_t cnt[];
  __shared__ int scratch[32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, tile = blockIdx.x;
  if (tile == 0 && t == 0) *w.n_items = 0;
  const int64_t i = int64_t(tile) * TILE + t;
  const int64_t tok = i < rows ? tokens[i] : -1;
  const bool inside = tok >= 0 && tok < vocab;
  const int range = inside ? int(tok) >> shift : ranges;
  for (int j = t; j < 16 * ranges; j += TILE) reinterpret_cast<uint32_t*>(cnt)[j] = 0;
  __syncthreads();
  const unsigned same = __match_any_sync(0xffffffffu, range);
  const int rank = __popc(same & ((1u << lane) - 1));
  if (inside && rank == 0) cnt[warp * ranges + range] = uint16_t(__popc(same));
  __syncthreads();
  // Thread r: tokens of range r in the warps before each warp, then the ranges before r.
  int mine = 0;
  if (t < ranges) {
#pragma unroll 8
    for (int k = 0; k < 32; ++k) {
      const int n = cnt[k * ranges + t];
      cnt[k * ranges + t] = uint16_t(mine);
      mine += n;
    }
  }
  int total;
  const int base = block_exclusive<32>(mine, scratch, total);
  __syncthreads();
  if (t < ranges) {
    w.offs[size_t(t) * tiles + tile] = uint16_t(base);
#pragma unroll 8
    for (int k = 0; k < 32; ++k) cnt[k * ranges + t] = uint16_t(cnt[k * ranges + t] + base);
  }
  if (t == 0) w.offs[size_t(ranges) * tiles + tile] = uint16_t(total);
  __syncthreads();
  if (inside)
    w.local[size_t(tile) * TILE + cnt[warp * ranges + range] + rank] =
        (uint32_t(int(tok) & ((1 << shift) - 1)) << 10) | uint32_t(t);
}

// One CTA per range. Shared: the range's list in token order (while it fits; a
// range with more than CACHED tokens uses the workspace) and per-warp id
// counts [QW][R]. Bound by the latency of its dependent steps.
__global__ void __launch_bounds__(QT) sort_kernel(int vocab, int shift, int tiles, Work w) {
  extern __shared__ uint64_t list_cache[];  // [CACHED]: id in range << 32 | position
  __shared__ int scratch[QW];
  const int R = 1 << shift, range = blockIdx.x, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  int* cnt = reinterpret_cast<int*>(list_cache + CACHED);  // [QW][R]
  const uint16_t* lo = w.offs + size_t(range) * tiles;
  const uint16_t* hi = lo + tiles;
  // The range's place in the whole order, and its number of tokens.
  int below = 0, mine = 0;
  for (int k = t; k < tiles; k += QT) {
    below += lo[k];
    mine += hi[k] - lo[k];
  }
  int base, m;
  block_exclusive<QW>(below, scratch, base);
  block_exclusive<QW>(mine, scratch, m);
  for (int j = t; j < QW * R; j += QT) cnt[j] = 0;
  const bool fits = m <= CACHED;
  uint64_t* list = fits ? list_cache : w.list + base;
  int32_t* perm = w.perm + base;
  // The list in token order: QT tiles at a time, a warp copies a tile's tokens.
  __shared__ int tile_at[QT], tile_lo[QT], tile_n[QT];
  for (int k0 = 0, at = 0; k0 < tiles; k0 += QT) {
    const int k = k0 + t, first = k < tiles ? lo[k] : 0, n = k < tiles ? hi[k] - first : 0;
    int total;
    const int before = block_exclusive<QW>(n, scratch, total);
    tile_at[t] = at + before;
    tile_lo[t] = first;
    tile_n[t] = n;
    at += total;
    __syncthreads();
    const int here = min(QT, tiles - k0);
    for (int j = warp; j < here; j += QW)
      for (int e = lane; e < tile_n[j]; e += 32) {
        const uint32_t x = w.local[size_t(k0 + j) * TILE + tile_lo[j] + e];
        list[tile_at[j] + e] = (uint64_t(x >> 10) << 32) | uint32_t((k0 + j) * TILE + int(x & 1023u));
      }
    __syncthreads();
  }
  // Stable counting sort by id: each warp counts and then places one span of the list.
  const int span = ((m + QW - 1) / QW + 31) & ~31;
  const int s0 = min(warp * span, m), s1 = min(s0 + span, m);
  int* my = cnt + warp * R;
  for (int e0 = s0; e0 < s1; e0 += 128) {
    int id[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int e = e0 + 32 * u + lane;
      id[u] = e < s1 ? int(list[e] >> 32) : R;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const unsigned same = __match_any_sync(0xffffffffu, id[u]);
      if (id[u] < R && (same & ((1u << lane) - 1)) == 0) my[id[u]] += __popc(same);
      __syncwarp();
    }
  }
  __syncthreads();
  int carry = 0;
  for (int j0 = 0; j0 < R; j0 += QT) {
    const int j = j0 + t;
    int n = 0;
    if (j < R)
#pragma unroll
      for (int k = 0; k < QW; ++k) {
        const int c = cnt[k * R + j];
        cnt[k * R + j] = n;
        n += c;
      }
    int total;
    const int before = carry + block_exclusive<QW>(n, scratch, total);
    if (j < R) {
      w.start[(range << shift) + j] = base + before;
#pragma unroll
      for (int k = 0; k < QW; ++k) cnt[k * R + j] += before;
      const int id = (range << shift) + j;
      if (n > LONG && id < vocab) {
        // Pieces for sum_kernel (their order in the list does not matter: sums are joined per id).
        const int pieces = (n + LONG - 1) / LONG;
        const int head = atomicAdd(w.n_items, pieces);
        w.arrived[head] = 0;
        for (int q = 0; q < pieces; ++q)
          reinterpret_cast<int4*>(w.items)[head + q] =
              make_int4(id, base + before + q * LONG, min(LONG, n - q * LONG) | (pieces << 7), head);
      }
    }
    carry += total;
  }
  if (t == 0 && range == int(gridDim.x) - 1) w.start[(range + 1) << shift] = base + m;
  __syncthreads();
  for (int e0 = s0; e0 < s1; e0 += 128) {
    uint64_t x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int e = e0 + 32 * u + lane;
      x[u] = e < s1 ? list[e] : uint64_t(R) << 32;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int id = int(x[u] >> 32);
      const unsigned same = __match_any_sync(0xffffffffu, id);
      const int rank = __popc(same & ((1u << lane) - 1));
      const int to = id < R ? my[id] + rank : 0;
      __syncwarp();
      if (id < R) {
        perm[to] = int32_t(uint32_t(x[u]));
        if (rank == 0) my[id] += __popc(same);
      }
      __syncwarp();
    }
  }
}

// Eight elements as they lie in memory, on their way.
template <typename T> struct Raw8;
template <> struct Raw8<bf16> {
  uint4 a;
  M4_DEV void load(const bf16* p) { a = *reinterpret_cast<const uint4*>(p); }
  M4_DEV void add(float (&acc)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc[2 * i] += __uint_as_float(w[i] << 16);
      acc[2 * i + 1] += __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <> struct Raw8<float> {
  float4 a, b;
  M4_DEV void load(const float* p) { a = ld4(p), b = ld4(p + 4); }
  M4_DEV void add(float (&acc)[8]) const {
    acc[0] += a.x, acc[1] += a.y, acc[2] += a.z, acc[3] += a.w;
    acc[4] += b.x, acc[5] += b.y, acc[6] += b.z, acc[7] += b.w;
  }
};

// Adds columns c + 256 u .. c + 256 u + 7 (u < U) of the rows at pos[0 .. n), in ascending order.
template <typename G, int U>
M4_DEV void sum_rows(const G* __restrict__ g, const int32_t* pos, int n, int c, int dim, bool vec,
                     float (&acc)[U][8]) {
  constexpr int J = U == 1 ? 4 : 2;  // rows on their way
  if (vec) {
    for (int j = 0; j < n; j += J) {
      Raw8<G> v[J][U];
#pragma unroll
      for (int r = 0; r < J; ++r)
        if (j + r < n) {
          const G* row = g + int64_t(pos[j + r]) * dim + c;
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (c + 256 * u < dim) v[r][u].load(row + 256 * u);
        }
#pragma unroll
      for (int r = 0; r < J; ++r)
        if (j + r < n)
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (c + 256 * u < dim) v[r][u].add(acc[u]);
    }
  } else {
    for (int j = 0; j < n; ++j)
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c + 256 * u < dim) {
          float v[8];
          load8(g + int64_t(pos[j]) * dim, c + 256 * u, dim, false, v);
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[u][i] += v[i];
        }
  }
}

// Blocks below `piece_blocks`: pieces of ids with more than LONG tokens (the
// warps take LONG / RW positions each; joined in order). The others: ROWS
// gradient rows; first those of more than SHORT tokens, an eighth of a row's
// tokens a warp, joined in order; then one row, 256 U columns at a time, a warp.
// Bound by HBM and latency: 255 MB in 53 us (65536 x 768, cold L2), 39 at the
// copy bandwidth. In copies of the kernel zero rows alone took 21 us, rows of at
// most 4 tokens 34, all rows without the pieces 48 to 60 where one warp added
// up to 32. Four blocks an SM, three where a thread holds 24 columns and 64
// registers would spill (bfloat16 gradients: 57, 105 us; three: 60, 105). With
// float32 gradients 24 columns and two rows on their way spill at 80 registers
// too, and above width 768 the last sweep over the columns leaves lanes idle.
template <typename G, typename W, int U>
__global__ void __launch_bounds__(RT, U == 3 ? 3 : 4) sum_kernel(int vocab, int dim, bool vec, bool wide, float scale,
                                                                 int piece_blocks, const G* __restrict__ grad, Work w,
                                                                 W* __restrict__ d_weight) {
  __shared__ __align__(16) float sums[RW][256 * U];
  __shared__ int start[ROWS + 1], mids[ROWS], n_mid, last;
  __shared__ int32_t held[HELD];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  // Joins the warps' sums in order: sum u of thread t is column c0 + 256 u + t.
  auto join = [&](const float(&acc)[U][8], float(&s)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) Vec8<float>::store(&sums[warp][256 * u + 8 * lane], acc[u]);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[u] = 0.f;
#pragma unroll
      for (int k = 0; k < RW; ++k) s[u] += sums[k][256 * u + t];
    }
    __syncthreads();
  };
  if (int(blockIdx.x) >= piece_blocks) {
    const int row0 = (int(blockIdx.x) - piece_blocks) * ROWS, rows = min(ROWS, vocab - row0);
    if (t <= rows) start[t] = w.start[row0 + t];
    if (t == 0) n_mid = 0;
    __syncthreads();
    const int base = start[0], all = start[rows] - base;
    for (int i = t; i < min(all, HELD); i += RT) held[i] = w.perm[base + i];
    if (t < rows) {
      const int n = start[t + 1] - start[t];
      if (n > SHORT && n <= LONG) mids[atomicAdd(&n_mid, 1)] = t;
    }
    __syncthreads();
    auto positions = [&](int first, int n) {
      return first + n <= HELD ? static_cast<const int32_t*>(held + first) : w.perm + base + first;
    };
    for (int i = 0; i < n_mid; ++i) {  // rows that all warps share
      const int j = mids[i], first = start[j] - base, n = start[j + 1] - base - first;
      const int32_t* pos = positions(first, n);
      const int per = (n + RW - 1) / RW, p0 = min(warp * per, n), p1 = min(p0 + per, n);
      for (int c0 = 0; c0 < dim; c0 += 256 * U) {
        float acc[U][8] = {}, s[U];
        sum_rows<G, U>(grad, pos + p0, p1 - p0, c0 + 8 * lane, dim, vec, acc);
        join(acc, s);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (c0 + 256 * u + t < dim) d_weight[int64_t(row0 + j) * dim + c0 + 256 * u + t] = from_f<W>(s[u] * scale);
      }
    }
    for (int j = warp; j < rows; j += RW) {
      const int first = start[j] - base, n = start[j + 1] - base - first;
      if (n > SHORT) continue;
      const int32_t* pos = positions(first, n);
      W* out = d_weight + int64_t(row0 + j) * dim;
      for (int c = 8 * lane; c < dim; c += 256 * U) {
        float acc[U][8] = {};
        sum_rows<G, U>(grad, pos, n, c, dim, vec, acc);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (c + 256 * u < dim) {
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[u][i] *= scale;
            if (wide) store_wide(out + c + 256 * u, acc[u]);
            else store8(out, c + 256 * u, dim, vec, acc[u]);
          }
      }
    }
    return;
  }
  const int n_items = *w.n_items;
  const size_t width = part_width(dim);
  for (int it = blockIdx.x; it < n_items; it += piece_blocks) {
    const int4 item = reinterpret_cast<const int4*>(w.items)[it];
    const int n = item.z & 127, pieces = item.z >> 7;
    constexpr int PER = LONG / RW;
    const int p0 = min(warp * PER, n), p1 = min(p0 + PER, n);
    for (int c0 = 0; c0 < dim; c0 += 256 * U) {
      float acc[U][8] = {}, s[U];
      sum_rows<G, U>(grad, w.perm + item.y + p0, p1 - p0, c0 + 8 * lane, dim, vec, acc);
      join(acc, s);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + 256 * u + t < width) w.part[size_t(it) * width + c0 + 256 * u + t] = s[u];
    }
    __threadfence();
    __syncthreads();
    if (t == 0) last = atomicAdd(w.arrived + item.w, 1) == pieces - 1;
    __syncthreads();
    if (last) {  // the id's pieces in order, an eighth of them a warp
      __threadfence();
      const int per = (pieces + RW - 1) / RW, q0 = min(warp * per, pieces), q1 = min(q0 + per, pieces);
      for (int c0 = 0; c0 < dim; c0 += 256 * U) {
        float acc[U][8] = {}, s[U];
        const float* from = w.part + size_t(item.w) * width + c0 + 8 * lane;
#pragma unroll 2
        for (int q = q0; q < q1; ++q)
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (c0 + 256 * u + 8 * lane < width) {
              const float4 a = __ldcg(reinterpret_cast<const float4*>(from + q * width + 256 * u));
              const float4 b = __ldcg(reinterpret_cast<const float4*>(from + q * width + 256 * u + 4));
              acc[u][0] += a.x, acc[u][1] += a.y, acc[u][2] += a.z, acc[u][3] += a.w;
              acc[u][4] += b.x, acc[u][5] += b.y, acc[u][6] += b.z, acc[u][7] += b.w;
            }
        join(acc, s);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (c0 + 256 * u + t < dim)
            d_weight[int64_t(item.x) * dim + c0 + 256 * u + t] = from_f<W>(s[u] * scale);
      }
    }
    __syncthreads();
  }
}

template <typename W, typename O>
int lookup(int64_t rows, int vocab, int dim, const int64_t* tokens, const void* weight, float scale, void* out,
           cudaStream_t st) {
  const bool vec = dim % 8 == 0 && all_aligned16(weight, out);
  int lanes = 1;
  while (lanes < 32 && 8 * lanes < dim) lanes *= 2;
  const int64_t blocks = (rows * lanes + 255) / 256;
  if (blocks > 0x7fffffff) return M4_ERR_UNSUPPORTED;
  lookup_kernel<W, O><<<unsigned(blocks), 256, 0, st>>>(rows, vocab, dim, lanes, vec, tokens,
                                                        static_cast<const W*>(weight), scale, static_cast<O*>(out));
  return launch_status();
}

template <typename G, typename W>
int gradient(const Plan& p, const int64_t* tokens, const void* grad, float scale, void* d_weight, void* workspace,
             cudaStream_t st) {
  const Work w = work_of(p, workspace);
  const bool vec = p.dim % 8 == 0 && all_aligned16(grad, d_weight);
  const bool wide = vec && (reinterpret_cast<uintptr_t>(d_weight) & 31u) == 0;
  const int R = 1 << p.shift;
  const int tile_smem = 32 * ((p.ranges + 1) & ~1) * 2;
  const int sort_smem = CACHED * 8 + QW * R * 4;
  if (!allow_shared<tile_kernel>(tile_smem) || !allow_shared<sort_kernel>(sort_smem)) return M4_ERR_LAUNCH;
  tile_kernel<<<p.tiles, TILE, tile_smem, st>>>(p.rows, p.vocab, p.shift, p.ranges, p.tiles, tokens, w);
  sort_kernel<<<p.ranges, QT, sort_smem, st>>>(p.vocab, p.shift, p.tiles, w);
  const int pieces = p.rows <= LONG ? 0 : int(p.max_items < PIECE_BLOCKS ? p.max_items : PIECE_BLOCKS);
  const unsigned blocks = unsigned(pieces + (p.vocab + ROWS - 1) / ROWS);
  const G* g = static_cast<const G*>(grad);
  W* d = static_cast<W*>(d_weight);
  if (p.dim <= 256) sum_kernel<G, W, 1><<<blocks, RT, 0, st>>>(p.vocab, p.dim, vec, wide, scale, pieces, g, w, d);
  else if (p.dim <= 512) sum_kernel<G, W, 2><<<blocks, RT, 0, st>>>(p.vocab, p.dim, vec, wide, scale, pieces, g, w, d);
  else sum_kernel<G, W, 3><<<blocks, RT, 0, st>>>(p.vocab, p.dim, vec, wide, scale, pieces, g, w, d);
  return launch_status();
}

}  // namespace embed
}  // namespace m4

extern "C" size_t m4_embedding_workspace_bytes(int64_t rows, int vocab, int dim) {
  m4::embed::Plan p;
  return m4::embed::plan_for(rows, vocab, dim, &p) ? p.bytes : 0;
}

extern "C" int m4_embedding_fwd(int64_t rows, int vocab, int dim, const int64_t* tokens, const void* weight,
                                int weight_bf16, float scale, void* out, int out_bf16, void* stream) {
  using namespace m4::embed;
  if (rows <= 0 || vocab <= 0 || dim <= 0) return M4_ERR_DIMS;
  if (!tokens || !weight || !out) return M4_ERR_NULL;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (weight_bf16)
    return out_bf16 ? lookup<bf16, bf16>(rows, vocab, dim, tokens, weight, scale, out, st)
                    : lookup<bf16, float>(rows, vocab, dim, tokens, weight, scale, out, st);
  return out_bf16 ? lookup<float, bf16>(rows, vocab, dim, tokens, weight, scale, out, st)
                  : lookup<float, float>(rows, vocab, dim, tokens, weight, scale, out, st);
}

extern "C" int m4_embedding_bwd(int64_t rows, int vocab, int dim, const int64_t* tokens, const void* grad,
                                int grad_bf16, float scale, void* d_weight, int weight_bf16, void* workspace,
                                size_t workspace_bytes, void* stream) {
  using namespace m4::embed;
  if (rows <= 0 || vocab <= 0 || dim <= 0) return M4_ERR_DIMS;
  Plan p;
  if (!plan_for(rows, vocab, dim, &p)) return M4_ERR_UNSUPPORTED;
  if (!tokens || !grad || !d_weight || !workspace) return M4_ERR_NULL;
  if (!m4::aligned16(workspace)) return M4_ERR_ALIGN;
  if (workspace_bytes < p.bytes) return M4_ERR_WORKSPACE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (grad_bf16)
    return weight_bf16 ? gradient<bf16, bf16>(p, tokens, grad, scale, d_weight, workspace, st)
                       : gradient<bf16, float>(p, tokens, grad, scale, d_weight, workspace, st);
  return weight_bf16 ? gradient<float, bf16>(p, tokens, grad, scale, d_weight, workspace, st)
                     : gradient<float, float>(p, tokens, grad, scale, d_weight, workspace, st);
}
