// Attention for trees of drafted tokens over a paged cache.  Row cu[s] + i is token i of sequence s; it sees the C = start[s] cached positions,
// its ancestors in the tree and itself, each within the window of its own position C + depth(i).
//
// Work.  The query rows of a sequence that read the same key/value head g are its tokens times the query heads of the group: row r of them is
// token r / qpk, head g qpk + r % qpk.  An item is (sequence, kv head, tile of rows), a unit one tile of keys of an item.  The units of all items,
// in order, are dealt out to the blocks in equal runs, so that sequences of any lengths load all SMs alike; a block that has a part of an item leaves
// (max, sum, unnormalised output) of its keys in the workspace, and combine_kernel adds the parts up in order.  Where the parts lie follows from the
// lengths alone: no counters, and the same sums on every run.
//
//   tree_prep_kernel      depths; rotates and appends the new keys and values; zeroes the output's padding columns
//   tree_plain_kernel     any type, any widths up to 256: fp32 products on the CUDA cores
//   combine_kernel        sums the parts of the items that several blocks shared
// Scores, softmax and sums are fp32.
#include "chunk.cuh"

namespace pt {
namespace ta {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int MAX_SEQ = 1024, MAX_NODES = 256, WORDS = MAX_NODES / 32;

__device__ __forceinline__ float val(float x) { return x; }
__device__ __forceinline__ float val(__half x) { return __half2float(x); }
__device__ __forceinline__ float val(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T rounded(float x);
template <> __device__ __forceinline__ float rounded<float>(float x) { return x; }
template <> __device__ __forceinline__ __half rounded<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

struct Params {
  int n_seq, n_head, n_kv, qpk, dim, vdim, page, max_pages, max_len, window, most;
  int q_ld, kv_ld, out_ld, out_cols, rope_half;
  int rows_tile, keys_tile, blocks;        // of an item, of a unit, of the attention kernel
  float scale, softcap;
  const void *q, *k, *v;
  void *pool, *out;
  const float2 *rope;
  const int *page_table, *cu, *start, *slot, *parent;
  int *error_flag;
  float *part_o;      // [2 blocks][vdim / 4][rows_tile][4]
  float2 *part_ml;    // [2 blocks][rows_tile]
};

// ------------------------------------------------------------------------------------------ the work and its parts
struct Seq {
  int row0, n, start;      // n = 0: nothing is done for it
};
__device__ __forceinline__ Seq sequence(const Params &p, int s) {
  Seq x{p.cu[s], 0, p.start[s]};
  const int n = p.cu[s + 1] - x.row0;
  if (n > 0 && n <= p.most && x.start >= 0 && x.start <= p.max_len - n) x.n = n;
  return x;
}
struct Span {
  int first, tiles, row_tiles;      // key tiles of an item, items per kv head
};
__device__ __forceinline__ Span span(const Params &p, const Seq &x) {
  const int lo = p.window ? max(0, x.start - p.window + 1) / p.keys_tile : 0;
  return Span{lo, (x.start + x.n + p.keys_tile - 1) / p.keys_tile - lo, (x.n * p.qpk + p.rows_tile - 1) / p.rows_tile};
}
// Units in front of every sequence (units[n_seq]: all), by the whole block.
__device__ __forceinline__ void count_units(const Params &p, int *units) {
  __shared__ int warp_sum[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
  int base = 0;
  for (int s0 = 0; s0 < p.n_seq; s0 += blockDim.x) {
    const int s = s0 + tid;
    int v = 0;
    if (s < p.n_seq) {
      const Seq x = sequence(p, s);
      if (x.n) {
        const Span y = span(p, x);
        v = p.n_kv * y.row_tiles * y.tiles;
      }
    }
    int t = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += u;
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = t;
    __syncthreads();
    int before = base;
    for (int i = 0; i < nw; ++i) {
      if (i < warp) before += warp_sum[i];
      base += warp_sum[i];
    }
    if (s < p.n_seq) units[s] = before + t - v;
  }
  if (tid == 0) units[p.n_seq] = base;
  __syncthreads();
}
// The sequence of a unit: the last one that begins at or before it and has units.
__device__ __forceinline__ int seq_of(const int *units, int n_seq, int u) {
  int lo = 0, hi = n_seq - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (units[mid] <= u) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
struct Share {
  int all, quota;
};
__device__ __forceinline__ Share share(const Params &p, const int *units) {
  const int all = units[p.n_seq];
  return Share{all, (all + p.blocks - 1) / p.blocks};
}
// A part of an item: key tiles t0 .. t0 + nt - 1 of row tile rt of kv head g of sequence s.
struct Piece {
  int s, g, rt, t0, nt;
  Seq x;
  bool whole;            // the item's only part
  int slot;              // else: where it goes.  A block has at most two such parts: one of an item that began before its run, one that goes on behind it
};
__device__ __forceinline__ Piece piece_at(const Params &p, const int *units, const Share &sh, int block, int u) {
  Piece k;
  k.s = seq_of(units, p.n_seq, u);
  k.x = sequence(p, k.s);
  const Span y = span(p, k.x);
  const int item = (u - units[k.s]) / y.tiles, first = units[k.s] + item * y.tiles;
  k.g = item / y.row_tiles;
  k.rt = item - k.g * y.row_tiles;
  const int end = min(min(first + y.tiles, (block + 1) * sh.quota), sh.all);
  k.t0 = y.first + u - first;
  k.nt = end - u;
  k.whole = k.nt == y.tiles;
  k.slot = 2 * block + (u == first ? 1 : 0);
  return k;
}

// ------------------------------------------------------------------------------------------ trees
// A token's parent, -1 for one that follows the cached positions (and for a parent that is none: *bad).
__device__ __forceinline__ int parent_of(const Params &p, const Seq &x, int i, bool *bad = nullptr) {
  if (!p.parent) return i - 1;
  const int u = p.parent[x.row0 + i];
  if (u >= -1 && u < i) return u;
  if (bad) *bad = true;
  return -1;
}
struct Tree {
  int parent[MAX_NODES];
  int depth[MAX_NODES];
  uint32_t seen[MAX_NODES][WORDS];   // the tokens that a token sees
};
// By `threads` threads, between two barriers of theirs (`sync`).  MASKS: also what every token sees.
template <bool MASKS, typename Sync> __device__ __forceinline__ void build_tree(const Params &p, const Seq &x, Tree &t, int tid, int threads, Sync sync, bool *bad = nullptr) {
  for (int i = tid; i < x.n; i += threads) t.parent[i] = parent_of(p, x, i, bad);
  sync();
  for (int i = tid; i < x.n; i += threads) {
    uint32_t w[WORDS] = {};
    int d = 0;
    if (!p.parent) {
      d = i;
      if (MASKS) {
        const int lo = p.window ? max(0, i - p.window + 1) : 0;
#pragma unroll
        for (int k = 0; k < WORDS; ++k) {
          const int a = max(lo - 32 * k, 0), b = min(i - 32 * k, 31);      // bits a .. b
          if (a <= b) w[k] = (0xffffffffu >> (31 - (b - a))) << a;
        }
      }
    } else {
      for (int u = i; u >= 0; u = t.parent[u], ++d)
        if (MASKS && (p.window == 0 || d < p.window)) {
#pragma unroll
          for (int k = 0; k < WORDS; ++k)
            if (u >> 5 == k) w[k] |= 1u << (u & 31);
        }
      --d;
    }
    t.depth[i] = d;
    if (MASKS) {
#pragma unroll
      for (int k = 0; k < WORDS; ++k) t.seen[i][k] = w[k];
    }
  }
  sync();
}
// Whether token i sees position j (below C + n).
__device__ __forceinline__ bool sees(const Params &p, const Seq &x, const Tree &t, int i, int j) {
  const int d = j - x.start;
  if (d >= 0) return t.seen[i][d >> 5] >> (d & 31) & 1;
  return p.window == 0 || x.start + t.depth[i] - j < p.window;
}

template <typename T> __device__ __forceinline__ T *k_page(const Params &p, int phys, int g) {
  return reinterpret_cast<T *>(p.pool) + (size_t)phys * p.n_kv * p.page * (p.dim + p.vdim) + (size_t)g * p.page * p.dim;
}
template <typename T> __device__ __forceinline__ T *v_page(const Params &p, int phys, int g) {
  return reinterpret_cast<T *>(p.pool) + (size_t)phys * p.n_kv * p.page * (p.dim + p.vdim) + (size_t)p.n_kv * p.page * p.dim + (size_t)g * p.page * p.vdim;
}
// Element c of a head's row, rotated by the angles of `pos`.
template <typename T> __device__ __forceinline__ float turned(const Params &p, const T *row, int c, int pos) {
  const int h = p.rope_half;
  if (c >= 2 * h) return val(row[c]);
  const float2 a = p.rope[(size_t)pos * h + (c < h ? c : c - h)];
  return c < h ? val(row[c]) * a.x - val(row[c + h]) * a.y : val(row[c]) * a.x + val(row[c - h]) * a.y;
}

constexpr int PREP_THREADS = 256;
// Block: a sequence's tokens (x strided), one at a time.
template <typename T> __global__ void __launch_bounds__(PREP_THREADS) tree_prep_kernel(const Params p) {
  early_start();
  __shared__ Tree tree;
  __shared__ bool bad;
  const int s = blockIdx.y, tid = threadIdx.x;
  const Seq x = sequence(p, s);
  const int n = p.cu[s + 1] - x.row0;
  if (n <= 0) return;
  if (!x.n) {
    if (tid == 0 && blockIdx.x == 0 && p.error_flag) atomicExch(p.error_flag, n > p.most ? 14 : 12);
    return;
  }
  if (tid == 0) bad = false;
  __syncthreads();
  build_tree<false>(p, x, tree, tid, PREP_THREADS, [] { __syncthreads(); }, &bad);
  if (bad && tid == 0 && blockIdx.x == 0 && p.error_flag) atomicExch(p.error_flag, 14);
  const int *table = p.page_table + (size_t)p.slot[s] * p.max_pages;
  for (int i = blockIdx.x; i < x.n; i += gridDim.x) {
    const int at = x.start + i, pos = x.start + tree.depth[i], phys = table[at / p.page], place = at % p.page;
    const T *k = reinterpret_cast<const T *>(p.k) + (size_t)(x.row0 + i) * p.kv_ld, *v = reinterpret_cast<const T *>(p.v) + (size_t)(x.row0 + i) * p.kv_ld;
    for (int e = tid; e < p.n_kv * p.dim; e += PREP_THREADS) {
      const int g = e / p.dim, c = e - g * p.dim;
      k_page<T>(p, phys, g)[(size_t)place * p.dim + c] = rounded<T>(turned<T>(p, k + g * p.dim, c, pos));
    }
    for (int e = tid; e < p.n_kv * p.vdim; e += PREP_THREADS) {
      const int g = e / p.vdim, c = e - g * p.vdim;
      v_page<T>(p, phys, g)[(size_t)place * p.vdim + c] = v[e];
    }
    for (int c = p.n_head * p.vdim + tid; c < p.out_cols; c += PREP_THREADS) reinterpret_cast<T *>(p.out)[(size_t)(x.row0 + i) * p.out_ld + c] = rounded<T>(0.f);
  }
}

// Scores in the units of exp2 from raw products.
__device__ __forceinline__ float score2(const Params &p, float s) {
  s *= p.scale;
  return (p.softcap > 0.f ? p.softcap * tanhf(s / p.softcap) : s) * kLog2e;
}

// ------------------------------------------------------------------------------------------ any sizes
// Rows and keys of a tile in shared memory as fp32; thread (ty, tx) has rows 2 ty, 2 ty + 1 and keys tx, tx + 8, .. of the scores, and columns 4 tx + 32 j of
// the output.  What bounds it: fp32 multiply-adds, six shared loads of 16 bytes for 32 of them.
constexpr int PLAIN_THREADS = 128, PROWS = 32, PKEYS = 32;
static size_t plain_smem(int dim, int vdim) { return (size_t)(PROWS + PKEYS) * (dim + 8) * 4 + (size_t)PKEYS * (vdim + 36) * 4 + (size_t)PROWS * (PKEYS + 4) * 4 + PROWS * 8; }
template <typename T, int VJ> __global__ void __launch_bounds__(PLAIN_THREADS) tree_plain_kernel(const Params p) {
  early_start();
  extern __shared__ __align__(16) float sm[];
  __shared__ int units[MAX_SEQ + 1];
  __shared__ Tree tree;
  const int d4 = (p.dim + 3) / 4 * 4, v32 = VJ * 32, kld = d4 + 4, vld = v32 + 4, pld = PKEYS + 4;
  float *Q = sm, *K = Q + PROWS * kld, *V = K + PKEYS * kld, *P = V + PKEYS * vld, *corr = P + PROWS * pld, *sum = corr + PROWS;
  const int tid = threadIdx.x, tx = tid & 7, ty = tid >> 3;
  count_units(p, units);
  const Share sh = share(p, units);
  const int end = min((int)(blockIdx.x + 1) * sh.quota, sh.all);
  int had = -1;
  for (int u = blockIdx.x * sh.quota; u < end;) {
    const Piece k = piece_at(p, units, sh, blockIdx.x, u);
    u += k.nt;
    const Seq x = k.x;
    const int rows = min(PROWS, x.n * p.qpk - k.rt * PROWS), r0 = k.rt * PROWS;
    __syncthreads();
    if (k.s != had) build_tree<true>(p, x, tree, tid, PLAIN_THREADS, [] { __syncthreads(); });
    had = k.s;
    for (int e = tid; e < PROWS * d4; e += PLAIN_THREADS) {
      const int r = e / d4, c = e - r * d4;
      float y = 0.f;
      if (r < rows && c < p.dim) {
        const int i = (r0 + r) / p.qpk, h = k.g * p.qpk + (r0 + r) % p.qpk;
        y = turned<T>(p, reinterpret_cast<const T *>(p.q) + (size_t)(x.row0 + i) * p.q_ld + (size_t)h * p.dim, c, x.start + tree.depth[i]);
      }
      Q[r * kld + c] = y;
    }
    float o[2][VJ][4];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int j = 0; j < VJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[a][j][e] = 0.f;
    float m = -INFINITY, l = 0.f;        // of row tid / 4, the same in its four threads
    const int *table = p.page_table + (size_t)p.slot[k.s] * p.max_pages;
    for (int t = k.t0; t < k.t0 + k.nt; ++t) {
      const int j0 = t * PKEYS, keys = min(PKEYS, x.start + x.n - j0);
      __syncthreads();
      for (int e = tid; e < PKEYS * d4; e += PLAIN_THREADS) {
        const int r = e / d4, c = e - r * d4, j = j0 + r;
        K[r * kld + c] = r < keys && c < p.dim ? val(k_page<T>(p, table[j / p.page], k.g)[(size_t)(j % p.page) * p.dim + c]) : 0.f;
      }
      for (int e = tid; e < PKEYS * v32; e += PLAIN_THREADS) {
        const int r = e / v32, c = e - r * v32, j = j0 + r;
        V[r * vld + c] = r < keys && c < p.vdim ? val(v_page<T>(p, table[j / p.page], k.g)[(size_t)(j % p.page) * p.vdim + c]) : 0.f;
      }
      __syncthreads();
      float sc[2][4] = {};
      for (int c = 0; c < d4; c += 4) {
        float4 a[2], b[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) a[i] = *reinterpret_cast<const float4 *>(Q + (2 * ty + i) * kld + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = *reinterpret_cast<const float4 *>(K + (tx + 8 * i) * kld + c);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[i][j] = fmaf(a[i].w, b[j].w, fmaf(a[i].z, b[j].z, fmaf(a[i].y, b[j].y, fmaf(a[i].x, b[j].x, sc[i][j]))));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 2 * ty + i, key = tx + 8 * j;
          P[r * pld + key] = r < rows && key < keys && sees(p, x, tree, (r0 + r) / p.qpk, j0 + key) ? score2(p, sc[i][j]) : -INFINITY;
        }
      __syncthreads();
      {
        float *row = P + (tid >> 2) * pld + (tid & 3) * 8, top = m, add = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, row[j]);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float base = top == -INFINITY ? 0.f : top, f = exp2f(m - base);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float w = exp2f(row[j] - base);
          row[j] = w;
          add += w;
        }
        add += __shfl_xor_sync(0xffffffffu, add, 1);
        add += __shfl_xor_sync(0xffffffffu, add, 2);
        l = l * f + add;
        m = top;
        if ((tid & 3) == 0) corr[tid >> 2] = f;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float f = corr[2 * ty + i];
#pragma unroll
        for (int j = 0; j < VJ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][j][e] *= f;
      }
      // (a value that a row does not see may be infinite or NaN: it is left out, not multiplied by zero)
      const bool all_seen = j0 + keys <= x.start && (p.window == 0 || x.start + x.n - 1 - j0 < p.window);
      for (int key = 0; key < keys; ++key) {
        const float w0 = P[2 * ty * pld + key], w1 = P[(2 * ty + 1) * pld + key];
        if (!all_seen) {
#pragma unroll
          for (int j = 0; j < VJ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y = V[key * vld + 4 * tx + 32 * j + e];
              if (w0 != 0.f) o[0][j][e] = fmaf(w0, y, o[0][j][e]);
              if (w1 != 0.f) o[1][j][e] = fmaf(w1, y, o[1][j][e]);
            }
          continue;
        }
#pragma unroll
        for (int j = 0; j < VJ; ++j) {
          const float4 y = *reinterpret_cast<const float4 *>(V + key * vld + 4 * tx + 32 * j);
          o[0][j][0] = fmaf(w0, y.x, o[0][j][0]); o[0][j][1] = fmaf(w0, y.y, o[0][j][1]); o[0][j][2] = fmaf(w0, y.z, o[0][j][2]); o[0][j][3] = fmaf(w0, y.w, o[0][j][3]);
          o[1][j][0] = fmaf(w1, y.x, o[1][j][0]); o[1][j][1] = fmaf(w1, y.y, o[1][j][1]); o[1][j][2] = fmaf(w1, y.z, o[1][j][2]); o[1][j][3] = fmaf(w1, y.w, o[1][j][3]);
        }
      }
    }
    if ((tid & 3) == 0) {
      sum[tid >> 2] = l;
      if (!k.whole) p.part_ml[(size_t)k.slot * PROWS + (tid >> 2)] = make_float2(m, l);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 2 * ty + i, tok = (r0 + r) / p.qpk, h = k.g * p.qpk + (r0 + r) % p.qpk;
      if (r >= rows) continue;
      const float inv = 1.0f / sum[r];
      T *out = reinterpret_cast<T *>(p.out) + (size_t)(x.row0 + tok) * p.out_ld + (size_t)h * p.vdim;
#pragma unroll
      for (int j = 0; j < VJ; ++j) {
        const int c = 4 * tx + 32 * j;
        if (c >= p.vdim) continue;
        if (k.whole) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e < p.vdim) out[c + e] = rounded<T>(o[i][j][e] * inv);
        } else {
          *reinterpret_cast<float4 *>(p.part_o + (((size_t)k.slot * ((p.vdim + 3) / 4) + c / 4) * PROWS + r) * 4) = make_float4(o[i][j][0], o[i][j][1], o[i][j][2], o[i][j][3]);
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------ parts of an item
// Block (x: an item, by the most that a sequence can have; y: sequence): adds up the parts in the order of the keys.
constexpr int COMBINE_THREADS = 256;
template <typename T> __global__ void __launch_bounds__(COMBINE_THREADS) combine_kernel(const Params p) {
  early_start();
  __shared__ int units[MAX_SEQ + 1];
  const int s = blockIdx.y, tid = threadIdx.x;
  const Seq x = sequence(p, s);
  if (!x.n) return;
  const Span y = span(p, x);
  const int most_tiles = (p.most * p.qpk + p.rows_tile - 1) / p.rows_tile, g = blockIdx.x / most_tiles, rt = blockIdx.x - g * most_tiles;
  if (rt >= y.row_tiles) return;
  count_units(p, units);
  const Share sh = share(p, units);
  const int first = units[s] + (g * y.row_tiles + rt) * y.tiles, b0 = first / sh.quota, b1 = (first + y.tiles - 1) / sh.quota;
  if (b0 == b1) return;
  const int r0 = rt * p.rows_tile, rows = min(p.rows_tile, x.n * p.qpk - r0), v4 = (p.vdim + 3) / 4;
  for (int e = tid; e < rows * v4; e += COMBINE_THREADS) {
    const int r = e / v4, c = e - r * v4;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int b = b0; b <= b1; ++b) {
      const size_t slot = 2 * b + (b == b0 ? 1 : 0);
      const float2 ml = p.part_ml[slot * p.rows_tile + r];
      const float4 w = *reinterpret_cast<const float4 *>(p.part_o + ((slot * v4 + c) * p.rows_tile + r) * 4);
      const float top = fmaxf(m, ml.x);
      if (top == -INFINITY) continue;
      const float a = exp2f(m - top), f = exp2f(ml.x - top);
      o.x = o.x * a + w.x * f; o.y = o.y * a + w.y * f; o.z = o.z * a + w.z * f; o.w = o.w * a + w.w * f;
      l = l * a + ml.y * f;
      m = top;
    }
    const float inv = 1.0f / l;
    const int tok = (r0 + r) / p.qpk, h = g * p.qpk + (r0 + r) % p.qpk;
    T *out = reinterpret_cast<T *>(p.out) + (size_t)(x.row0 + tok) * p.out_ld + (size_t)h * p.vdim + 4 * c;
    const float z[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * c + i < p.vdim) out[i] = rounded<T>(z[i]);
  }
}

static int max_blocks() { return sm_count() * 4; }

template <typename T, int VJ> static int launch_plain(Params &p, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  const size_t smem = plain_smem(p.dim, VJ * 32);
  if (smem > 32 * 1024) PT_CUDA(allow_smem(tree_plain_kernel<T, VJ>, (int)plain_smem(256, VJ * 32), done));
  p.rows_tile = PROWS; p.keys_tile = PKEYS;
  p.blocks = sm_count() * 2;
  PT_CUDA(launch_early(tree_plain_kernel<T, VJ>, Grid(p.blocks), PLAIN_THREADS, smem, st, p));
  PT_LAUNCH_CHECK("pt_tree_attn");
  return PT_OK;
}
template <typename T> static int run(Params &p, cudaStream_t st) {
  PT_CUDA(launch_early(tree_prep_kernel<T>, Grid(dim3(std::min(p.most, 64), p.n_seq)), PREP_THREADS, 0, st, p));
  PT_LAUNCH_CHECK("pt_tree_attn");
  const int rc = p.vdim <= 64 ? launch_plain<T, 2>(p, st) : p.vdim <= 128 ? launch_plain<T, 4>(p, st) : launch_plain<T, 8>(p, st);
  if (rc) return rc;
  const int tiles = ceil_div(p.most * p.qpk, p.rows_tile);
  PT_CUDA(launch_early(combine_kernel<T>, Grid(dim3(p.n_kv * tiles, p.n_seq)), COMBINE_THREADS, 0, st, p));
  PT_LAUNCH_CHECK("pt_tree_attn");
  return PT_OK;
}

}  // namespace ta
}  // namespace pt

using namespace pt;

// (n_seq, max_tokens_per_seq and the heads do not matter to the present kernels: every block has two parts of one tile of rows.)
extern "C" size_t pt_tree_attn_workspace_bytes(int n_seq, int max_tokens_per_seq, int n_head, int n_kv, int vdim) {
  (void)n_seq; (void)max_tokens_per_seq; (void)n_head; (void)n_kv;
  return (size_t)2 * ta::max_blocks() * ta::PROWS * (sizeof(float2) + (size_t)(vdim + 3) / 4 * 16);
}

extern "C" int pt_tree_attn(const pt_tree_attn_args *a, void *stream) {
  PT_REQUIRE(a, "pt_tree_attn: null args");
  const pt_batch_view &b = a->batch;
  PT_REQUIRE(b.n_seq > 0 && b.n_seq <= ta::MAX_SEQ && b.n_tok > 0 && b.cu && b.start && b.slot, "pt_tree_attn: bad batch (%d sequences of at most %d, %d tokens)", b.n_seq, ta::MAX_SEQ,
             b.n_tok);
  PT_REQUIRE(a->n_head > 0 && a->n_kv > 0 && a->n_head % a->n_kv == 0, "pt_tree_attn: n_head=%d must be a positive multiple of n_kv=%d", a->n_head, a->n_kv);
  PT_REQUIRE(a->dim > 0 && a->dim <= 256 && a->vdim > 0 && a->vdim <= 256 && a->page_size > 0 && a->max_pages > 0, "pt_tree_attn: bad shape dim=%d vdim=%d (at most 256) page_size=%d max_pages=%d",
             a->dim, a->vdim, a->page_size, a->max_pages);
  PT_REQUIRE(a->dtype == PT_DT_F16 || a->dtype == PT_DT_F32 || a->dtype == PT_DT_BF16, "pt_tree_attn: type %d (fp16, fp32 or bf16)", a->dtype);
  PT_REQUIRE(a->q && a->k && a->v && a->pool && a->page_table && a->out, "pt_tree_attn: null pointer argument");
  PT_REQUIRE(a->q_ld >= a->n_head * a->dim && a->out_ld >= a->n_head * a->vdim && a->kv_ld >= a->n_kv * std::max(a->dim, a->vdim),
             "pt_tree_attn: row strides q %d, kv %d, out %d too small", a->q_ld, a->kv_ld, a->out_ld);
  PT_REQUIRE(a->window >= 0 && a->softcap >= 0.f, "pt_tree_attn: window=%d softcap=%f", a->window, a->softcap);
  PT_REQUIRE(a->rope_dims >= 0 && a->rope_dims % 2 == 0 && a->rope_dims <= a->dim && (!a->rope_dims || a->rope), "pt_tree_attn: %d rotated dimensions of %d", a->rope_dims, a->dim);
  const long long positions = (long long)a->page_size * a->max_pages;
  PT_REQUIRE(positions < (1ll << 31) && a->max_len <= positions, "pt_tree_attn: max_len=%d exceeds the %lld positions of the page table", a->max_len, positions);
  ta::Params p{};
  p.n_seq = b.n_seq; p.n_head = a->n_head; p.n_kv = a->n_kv; p.qpk = a->n_head / a->n_kv; p.dim = a->dim; p.vdim = a->vdim;
  p.page = a->page_size; p.max_pages = a->max_pages; p.max_len = a->max_len > 0 ? a->max_len : (int)positions; p.window = a->window;
  p.most = a->max_tokens_per_seq > 0 ? a->max_tokens_per_seq : b.n_tok;
  PT_REQUIRE(p.most <= ta::MAX_NODES, "pt_tree_attn: %d tokens of one sequence (at most %d)", p.most, ta::MAX_NODES);
  // (a unit is 32 positions of a row tile: their number is an int)
  PT_REQUIRE((double)b.n_seq * a->n_kv * (p.most * p.qpk / 32 + 1) * (p.max_len / 32 + 2) < 2e9, "pt_tree_attn: %d sequences of up to %d positions and %d heads are too much for one call", b.n_seq,
             p.max_len, a->n_head);
  p.q_ld = a->q_ld; p.kv_ld = a->kv_ld; p.out_ld = a->out_ld; p.rope_half = a->rope_dims / 2;
  p.out_cols = a->out_cols > 0 ? a->out_cols : a->out_ld;
  PT_REQUIRE(p.out_cols >= a->n_head * a->vdim && p.out_cols <= a->out_ld, "pt_tree_attn: out_cols=%d", a->out_cols);
  p.scale = a->scale; p.softcap = a->softcap; p.q = a->q; p.k = a->k; p.v = a->v; p.pool = a->pool; p.out = a->out; p.rope = (const float2 *)a->rope;
  p.page_table = a->page_table; p.cu = b.cu; p.start = b.start; p.slot = b.slot; p.parent = a->parent; p.error_flag = a->error_flag;
  const size_t need = pt_tree_attn_workspace_bytes(b.n_seq, p.most, a->n_head, a->n_kv, a->vdim);
  PT_REQUIRE(a->workspace && a->workspace_bytes >= need && aligned_to(a->workspace, 16), "pt_tree_attn: %zu workspace bytes on a 16-byte boundary needed, got %zu", need, a->workspace_bytes);
  p.part_o = (float *)a->workspace;
  p.part_ml = (float2 *)(p.part_o + (size_t)2 * ta::max_blocks() * ta::PROWS * ((a->vdim + 3) / 4 * 4));
  cudaStream_t st = as_stream(stream);
  if (a->dtype == PT_DT_F32) return ta::run<float>(p, st);
  return a->dtype == PT_DT_F16 ? ta::run<__half>(p, st) : ta::run<__nv_bfloat16>(p, st);
}
