// Attention for trees of drafted tokens over a paged cache.  Row cu[s] + i is token i of sequence s; it sees the C = start[s] cached positions,
// its ancestors in the tree and itself, each within the window of its own position C + depth(i).
//
// Work.  The query rows of a sequence that read the same key/value head g are its tokens times the query heads of the group: row r of them is
// token r / qpk, head g qpk + r % qpk.  An item is (sequence, kv head, tile of rows); its units are its key tiles, behind `extra` units that stand for what an item costs
// beside them.  The units of all items, in order, are dealt out to the blocks in equal runs, so that sequences of any lengths load all SMs alike; a block
// that has a part of an item leaves (max, sum, unnormalised output) of its keys in the workspace, and combine_kernel adds the parts up in order.  Where
// the parts lie follows from the lengths alone: no counters, and the same sums on every run.
//
//   tree_prep_kernel      rotates and appends the new keys and values, writes down what every token sees and who does what, and lays out the queries for the
//                         tensor cores
//   tree_plain_kernel     any type, any widths up to 256: fp32 products on the CUDA cores
//   tree_tensor_kernel    fp16 and bf16, widths up to 128 in steps of 8: both products on tcgen05
//   combine_kernel        sums the parts of the items that several blocks shared
// Scores, softmax and sums are fp32.  All three in a captured graph: 5 tokens behind 700 positions (32 heads over 8 of 128) 18 us, 16 sequences of 16 tokens behind up to
// 4000 68 us, 63 tokens behind 60000 187 us.
#include <cuda.h>

#include <type_traits>

#include "chunk.cuh"
#include "mbarrier.cuh"
#include "tmem.cuh"

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
  int n_seq, n_tok, n_head, n_kv, qpk, dim, vdim, page, max_pages, max_len, window, most;
  int q_ld, kv_ld, out_ld, out_cols, rope_half;
  int rows_tile, keys_tile, extra, blocks; // of an item, of a unit (powers of two); units of an item beside its key tiles; blocks of the attention kernel
  int rows_shift, keys_shift, part_ld;      // part_ld: rows of a part in the workspace
  float scale, softcap;
  const void *q, *k, *v;
  void *pool, *out;
  const float2 *rope;
  const int *page_table, *cu, *start, *slot, *parent;
  int *error_flag;
  int box;            // cache rows of a TMA box: the largest power of two up to 128 that divides a page; 0: no boxes
  bool out16;         // the output can be written in units of 16 bytes
  // workspace
  int *plan;          // units of a block, of all blocks; from PLAN_HEAD on a Start of every block
  int *units;         // [n_seq + 1] units in front of a sequence
  int *depth;         // [n_seq][most]
  uint32_t *seen;     // [n_seq][most][WORDS]: the tokens that a token sees
  uint4 *queries;     // tensor cores: of sequence s and kv head g from unit (s most n_head + g rows) 2 dim / 8 on: [part][dim / 8][rows], rows = n qpk;
                      // plain: [n_seq][most][n_head][dim up to a multiple of 4] as fp32
  float *part_o;      // [2 blocks][vdim / 4][part_ld][4]
  float2 *part_ml;    // [2 blocks][part_ld]
};

// ------------------------------------------------------------------------------------------ the work and its parts
struct Seq {
  int row0, n, start;      // n = 0: nothing is done for it
};
__device__ __forceinline__ Seq sequence(const Params &p, int s) {
  Seq x{p.cu[s], 0, p.start[s]};
  const int n = p.cu[s + 1] - x.row0;
  if (n > 0 && n <= p.most && x.row0 >= 0 && x.row0 <= p.n_tok - n && x.start >= 0 && x.start <= p.max_len - n) x.n = n;
  return x;
}
struct Span {
  int first, tiles, row_tiles;      // key tiles of an item, items per kv head
};
__device__ __forceinline__ Span span(const Params &p, const Seq &x) {
  const int lo = p.window ? max(0, x.start - p.window + 1) >> p.keys_shift : 0;
  return Span{lo, ((x.start + x.n + p.keys_tile - 1) >> p.keys_shift) - lo, (x.n * p.qpk + p.rows_tile - 1) >> p.rows_shift};
}
// What a block has to know of the sequence of its first unit, in one place: two loads instead of a chain of five.
struct __align__(16) Start {
  int s, units, next, slot;      // next: the next sequence's first unit
  Seq x;
  int unused;
};
constexpr int PLAN_HEAD = 4;
// Who does what, by one block of tree_prep_kernel.  Sequences that nothing is done for set the flag.
constexpr int PREP_THREADS = 256;
__device__ __noinline__ void write_plan(const Params &p) {
  __shared__ int units[MAX_SEQ + 1], warp_sum[PREP_THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int base = 0;
  for (int s0 = 0; s0 < p.n_seq; s0 += PREP_THREADS) {
    const int s = s0 + tid;
    int v = 0;
    if (s < p.n_seq) {
      const Seq x = sequence(p, s);
      if (x.n) {
        const Span y = span(p, x);
        v = p.n_kv * y.row_tiles * (y.tiles + p.extra);
      } else if (p.error_flag) {
        const int n = p.cu[s + 1] - x.row0;
        if (n > 0) atomicExch(p.error_flag, n > p.most || x.row0 < 0 || x.row0 > p.n_tok - n ? 14 : 12);
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
    for (int i = 0; i < PREP_THREADS / 32; ++i) {
      if (i < warp) before += warp_sum[i];
      base += warp_sum[i];
    }
    if (s < p.n_seq) p.units[s] = units[s] = before + t - v;
  }
  if (tid == 0) p.units[p.n_seq] = units[p.n_seq] = base;
  __syncthreads();
  const int quota = (base + p.blocks - 1) / p.blocks;
  if (tid == 0) {
    p.plan[0] = quota;
    p.plan[1] = base;
  }
  for (int b = tid; b < p.blocks; b += PREP_THREADS) {
    // the last sequence that begins at or before the block's first unit
    const int u = b * quota;
    int lo = 0, hi = p.n_seq - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (units[mid] <= u) lo = mid;
      else hi = mid - 1;
    }
    *reinterpret_cast<Start *>(p.plan + PLAN_HEAD + b * (sizeof(Start) / 4)) = Start{lo, units[lo], units[lo + 1], p.slot[lo], sequence(p, lo), 0};
  }
}
// A part of an item: key tiles t0 .. t0 + nt - 1 of row tile rt of kv head g of sequence s.
struct Piece {
  int s, g, rt, t0, nt;    // nt = 0: there is no more
  Seq x;
  int table;               // the sequence's row of the page table
  bool whole, first;       // the item's only part, its first
  int slot;                // else: where it goes.  A block has at most two such parts: one of an item that began before its run, one that goes on behind it
};
struct Cursor {
  int u, end;              // next unit of the block, behind its last one
  Start at;                // the sequence of unit u, or one in front of it
  __device__ __forceinline__ Cursor(const Params &p) {
    const int2 all = *reinterpret_cast<const int2 *>(p.plan);
    const int4 *from = reinterpret_cast<const int4 *>(p.plan + PLAN_HEAD) + 2 * blockIdx.x, a = from[0], b = from[1];
    at = Start{a.x, a.y, a.z, a.w, Seq{b.x, b.y, b.z}, 0};
    u = blockIdx.x * all.x;
    end = min(u + all.x, all.y);
  }
};
__device__ __noinline__ Piece next_piece(const Params &p, Cursor &c) {
  Piece k;
  k.nt = 0;
  while (c.u < c.end) {
    if (c.u >= c.at.next) {
      do c.at.units = c.at.next, c.at.next = p.units[++c.at.s + 1]; while (c.u >= c.at.next);
      c.at.x = sequence(p, c.at.s);
      c.at.slot = p.slot[c.at.s];
    }
    const int units = c.at.units;
    k.s = c.at.s;
    k.x = c.at.x;
    k.table = c.at.slot;
    const Span y = span(p, k.x);
    const int item = (c.u - units) / (y.tiles + p.extra), first = units + item * (y.tiles + p.extra), stop = min(first + y.tiles + p.extra, c.end);
    const int t0 = max(c.u - first - p.extra, 0), t1 = stop - first - p.extra;
    c.u = stop;
    if (t1 <= t0) continue;
    k.g = item / y.row_tiles;
    k.rt = item - k.g * y.row_tiles;
    k.t0 = y.first + t0;
    k.nt = t1 - t0;
    k.first = t0 == 0;
    k.whole = k.first && t1 == y.tiles;
    k.slot = 2 * blockIdx.x + (k.first ? 1 : 0);
    break;
  }
  return k;
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

// Half: pairs of 16-bit values and fp32
// Weights are 2^kBias times as large as their row's largest allows, which may be 2^kRaise above: in fp16 a part of 2^-14 or less has fewer bits (2^-25 is gone), and 2^16 is
// infinite.  So the largest lies between 2^13.9 and 2^15.9, and weights down to 2^-28 of it keep eleven bits or more, as where they are rounded once; from 2^-23 of it on, in two
// parts, the 15 that bf16 keeps.  (Between 2^7 and 2^15 a flat tail 19 below a high score was off by 2.5 roundings; but the output is rescaled more often: 60000 positions
// 186 -> 198 us, 16 sequences 68 -> 71.5.)
template <typename T> struct Half2;
template <> struct Half2<__half> {
  static constexpr float kBias = 13.9f, kRaise = 2.f;
  static __device__ __forceinline__ uint32_t pack(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
  static __device__ __forceinline__ float2 wide(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }
  // a and b in two parts
  static __device__ __forceinline__ void split(float a, float b, uint32_t &hi, uint32_t &lo) {
    hi = pack(a, b);
    const float2 back = wide(hi);
    lo = pack(a - back.x, b - back.y);
  }
  static constexpr uint32_t kExponent = 0x7c00u;
};
template <> struct Half2<__nv_bfloat16> {
  static constexpr float kBias = 0.f, kRaise = 8.f;
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf2(a, b); }
  static __device__ __forceinline__ float2 wide(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
  // (By cutting off bits, which costs no conversion: the upper half of a float is a bf16.  What is lost is below 2^-15 of the value.)
  static __device__ __forceinline__ void split(float a, float b, uint32_t &hi, uint32_t &lo) {
    const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
    hi = __byte_perm(x, y, 0x7632);
    lo = __byte_perm(__float_as_uint(a - __uint_as_float(x & 0xffff0000u)), __float_as_uint(b - __uint_as_float(y & 0xffff0000u)), 0x7632);
  }
  static constexpr uint32_t kExponent = 0x7f80u;
};
// Of a pair: whether a value is infinite or NaN, and the pair with zeros for those.
template <typename T> __device__ __forceinline__ bool bad(uint32_t v) {
  constexpr uint32_t e = Half2<T>::kExponent;
  return (v & e) == e || (v & e << 16) == e << 16;
}
template <typename T> __device__ __forceinline__ uint32_t finite(uint32_t v) {
  constexpr uint32_t e = Half2<T>::kExponent;
  return ((v & e) == e ? 0u : v & 0xffffu) | ((v & e << 16) == e << 16 ? 0u : v & 0xffff0000u);
}
// Eight neighbouring dimensions d .. d + 7 of a head's row, rotated by the angles of `pos`; `own`: their values.
template <typename T> __device__ __forceinline__ void turn8(const Params &p, const T *src, int d, int pos, const uint4 &own, float2 (&y)[4]) {
  const int h = p.rope_half;
  if (h % 8 == 0) {
    const bool second = d >= h;
    const uint4 other = *reinterpret_cast<const uint4 *>(src + (second ? d - h : d + h));
    const uint32_t o[4] = {own.x, own.y, own.z, own.w}, z[4] = {other.x, other.y, other.z, other.w};
    const float4 *cs = reinterpret_cast<const float4 *>(p.rope + (size_t)pos * h + (second ? d - h : d));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 m = Half2<T>::wide(o[i]), t = Half2<T>::wide(z[i]);
      const float4 an = __ldg(cs + i);
      y[i] = second ? make_float2(m.x * an.x + t.x * an.y, m.y * an.z + t.y * an.w) : make_float2(m.x * an.x - t.x * an.y, m.y * an.z - t.y * an.w);
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
      const float2 v = make_float2(turned<T>(p, src, d + 2 * i, pos), turned<T>(p, src, d + 2 * i + 1, pos));
      if (i == 0) y[0] = v; else if (i == 1) y[1] = v; else if (i == 2) y[2] = v; else y[3] = v;
    }
  }
}

// Block: token x of sequence y; one more block writes the plan.  EIGHTS: rows in units of 16 bytes.
template <typename T, bool EIGHTS> __global__ void __launch_bounds__(PREP_THREADS) tree_prep_kernel(const __grid_constant__ Params p) {
  early_start();
  const int s = blockIdx.y, i = blockIdx.x, tid = threadIdx.x;
  if (s == p.n_seq) {
    if (i == 0) write_plan(p);
    return;
  }
  __shared__ int parent[MAX_NODES];
  __shared__ uint32_t seen[WORDS];
  __shared__ int depth;
  const Seq x = sequence(p, s);
  if (i >= x.n) return;
  const int at = x.start + i, phys = p.page_table[(size_t)p.slot[s] * p.max_pages + at / p.page], place = at % p.page;
  if (p.parent) {
    for (int j = tid; j <= i; j += PREP_THREADS) parent[j] = p.parent[x.row0 + j];
    if (tid < WORDS) seen[tid] = 0;
    __syncthreads();
    if (tid == 0) {
      // (a parent that is none: the token follows the cached positions)
      int d = 0;
      for (int u = i; u >= 0; ++d) {
        if (p.window == 0 || d < p.window) seen[u >> 5] |= 1u << (u & 31);
        const int up = parent[u];
        if (u == i && (up < -1 || up >= i) && p.error_flag) atomicExch(p.error_flag, 14);
        u = up < u ? max(up, -1) : -1;
      }
      depth = d - 1;
    }
    __syncthreads();
  } else {
    if (tid < WORDS) {
      const int a = max((p.window ? max(0, i - p.window + 1) : 0) - 32 * tid, 0), b = min(i - 32 * tid, 31);      // bits a .. b
      seen[tid] = a <= b ? (0xffffffffu >> (31 - (b - a))) << a : 0u;
    }
    if (tid == 0) depth = i;
    __syncthreads();
  }
  const int pos = x.start + depth;
  if (tid < WORDS) p.seen[((size_t)s * p.most + i) * WORDS + tid] = seen[tid];
  if (tid == WORDS) p.depth[(size_t)s * p.most + i] = depth;
  const T *k = reinterpret_cast<const T *>(p.k) + (size_t)(x.row0 + i) * p.kv_ld, *v = reinterpret_cast<const T *>(p.v) + (size_t)(x.row0 + i) * p.kv_ld;
  if constexpr (EIGHTS) {
    const int nk = p.n_kv * (p.dim / 8), all = nk + p.n_kv * (p.vdim / 8);
    for (int e = tid; e < all; e += PREP_THREADS) {
      if (e < nk) {
        const int per = p.dim / 8, g = e / per, c = (e - g * per) * 8;
        uint4 w = *reinterpret_cast<const uint4 *>(k + g * p.dim + c);
        if (c < 2 * p.rope_half) {
          float2 y[4];
          turn8<T>(p, k + g * p.dim, c, pos, w, y);
          w = make_uint4(Half2<T>::pack(y[0].x, y[0].y), Half2<T>::pack(y[1].x, y[1].y), Half2<T>::pack(y[2].x, y[2].y), Half2<T>::pack(y[3].x, y[3].y));
        }
        *reinterpret_cast<uint4 *>(k_page<T>(p, phys, g) + (size_t)place * p.dim + c) = w;
      } else {
        const int per = p.vdim / 8, g = (e - nk) / per, c = (e - nk - g * per) * 8;
        *reinterpret_cast<uint4 *>(v_page<T>(p, phys, g) + (size_t)place * p.vdim + c) = *reinterpret_cast<const uint4 *>(v + g * p.vdim + c);
      }
    }
    // queries, rotated (in two parts), and negated where the scale is negative; a row's units lie as far apart as there are rows, so that the threads that have a
    // row each read them side by side
    const T *q = reinterpret_cast<const T *>(p.q) + (size_t)(x.row0 + i) * p.q_ld;
    const int per = p.dim / 8, rows = x.n * p.qpk;
    const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
    for (int e = tid; e < p.n_head * per; e += PREP_THREADS) {
      const int head = e / per, c = e - head * per, g = head / p.qpk, r = i * p.qpk + head - g * p.qpk;
      const T *src = q + (size_t)head * p.dim;
      uint4 w = *reinterpret_cast<const uint4 *>(src + c * 8), lo = make_uint4(0u, 0u, 0u, 0u);
      if (c * 8 < 2 * p.rope_half) {
        float2 y[4];
        uint32_t a[4], b[4];
        turn8<T>(p, src, c * 8, pos, w, y);
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          a[z] = Half2<T>::pack(y[z].x, y[z].y);
          const float2 back = Half2<T>::wide(a[z]);
          b[z] = Half2<T>::pack(y[z].x - back.x, y[z].y - back.y) ^ flip;
        }
        w = make_uint4(a[0], a[1], a[2], a[3]);
        lo = make_uint4(b[0], b[1], b[2], b[3]);
      }
      w.x ^= flip; w.y ^= flip; w.z ^= flip; w.w ^= flip;
      uint4 *to = p.queries + ((size_t)s * p.most * p.n_head + (size_t)g * rows) * 2 * per + r;
      to[(size_t)c * rows] = w;
      if (p.rope_half) to[(size_t)(per + c) * rows] = lo;
    }
  } else {
    for (int e = tid; e < p.n_kv * p.dim; e += PREP_THREADS) {
      const int g = e / p.dim, c = e - g * p.dim;
      k_page<T>(p, phys, g)[(size_t)place * p.dim + c] = rounded<T>(turned<T>(p, k + g * p.dim, c, pos));
    }
    for (int e = tid; e < p.n_kv * p.vdim; e += PREP_THREADS) {
      const int g = e / p.vdim, c = e - g * p.vdim;
      v_page<T>(p, phys, g)[(size_t)place * p.vdim + c] = v[e];
    }
    const T *q = reinterpret_cast<const T *>(p.q) + (size_t)(x.row0 + i) * p.q_ld;
    const int d4 = (p.dim + 3) / 4 * 4;
    float *to = reinterpret_cast<float *>(p.queries) + ((size_t)s * p.most + i) * p.n_head * d4;
    for (int e = tid; e < p.n_head * d4; e += PREP_THREADS) {
      const int head = e / d4, c = e - head * d4;
      to[e] = c < p.dim ? turned<T>(p, q + (size_t)head * p.dim, c, pos) : 0.f;
    }
  }
  for (int c = p.n_head * p.vdim + tid; c < p.out_cols; c += PREP_THREADS) reinterpret_cast<T *>(p.out)[(size_t)(x.row0 + i) * p.out_ld + c] = rounded<T>(0.f);
}

// Which of the keys base .. base + 31 token i sees.
__device__ __forceinline__ uint32_t seen_word(const Params &p, const Seq &x, const uint32_t *seen, int depth, int base) {
  const int ctx = min(max(x.start - base, 0), 32), low = p.window ? min(max(x.start + depth - p.window + 1 - base, 0), 32) : 0;
  uint32_t v = ctx == 32 ? 0xffffffffu : (1u << ctx) - 1u;
  v = low == 32 ? 0u : v & ~((1u << low) - 1u);
  const int d = base - x.start;      // drafted token of the first key
  if (d >= 0) {
    const int k = d >> 5;
    if (k < WORDS) v |= __funnelshift_r(seen[k], k + 1 < WORDS ? seen[k + 1] : 0u, d & 31);
  } else if (d > -32) {
    v |= seen[0] << -d;
  }
  return v;
}

// tanh without a branch: below 0.55 its Taylor series (the coefficients are 2^2n (2^2n - 1) B_2n / (2n)!; what is left out is below 2^-24 of it), else
// 1 - 2 / (e^2x + 1).
__device__ __forceinline__ float tanh_of(float x) {
  const float y = x * x;
  float t = -929569.f / 638512875.f;
  t = fmaf(t, y, 21844.f / 6081075.f);
  t = fmaf(t, y, -1382.f / 155925.f);
  t = fmaf(t, y, 62.f / 2835.f);
  t = fmaf(t, y, -17.f / 315.f);
  t = fmaf(t, y, 2.f / 15.f);
  t = fmaf(t, y, -1.f / 3.f);
  return fabsf(x) < 0.55f ? fmaf(x * y, t, x) : 1.0f - __fdividef(2.0f, exp2f(2.0f * kLog2e * x) + 1.0f);
}

// ------------------------------------------------------------------------------------------ any sizes
// Rows and keys of a tile in shared memory as fp32; thread (ty, tx) has rows 2 ty, 2 ty + 1 and keys tx, tx + 8, .. of the scores, and columns 4 tx + 32 j of
// the output.  The next keys come in behind the scores, the next values behind the output, four threads a row; fp32 rows of whole 16 bytes by asynchronous copies.
// What bounds it: fp32 multiply-adds, six shared loads of 16 bytes for 32 of them; where blocks have two tiles or so, the latency of one warp a scheduler (11 tokens of
// three sequences behind a window of 512, 16 heads over 4 of 80: 35 us; 73 when rows came in one element after the other).
constexpr int PLAIN_THREADS = 128, PROWS = 32, PKEYS = 32, PLAIN_BLOCKS = 2;      // blocks: of an SM
static size_t plain_smem(int dim, int vdim) { return (size_t)(PROWS + PKEYS) * (dim + 8) * 4 + (size_t)PKEYS * (vdim + 36) * 4 + (size_t)PROWS * (PKEYS + 4) * 4 + PROWS * 8; }
// 16 bytes, zeros where bytes is 0.
__device__ __forceinline__ void cp_async(uint32_t dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// This thread's part of a row of `have` elements (zeros, where it is not `there`) to `to`, up to a multiple of four.
template <typename T> __device__ __noinline__ void row_in(float *to, const T *from, bool there, int have, bool async) {
  const int part = threadIdx.x & 3;
  if (std::is_same<T, float>::value && async) {
    for (int c = 4 * part; c < have; c += 16) cp_async(tc::sa(to + c), from + (there ? c : 0), there ? 16 : 0);
    return;
  }
#pragma unroll 4
  for (int c = part; c < (have + 3) / 4 * 4; c += 4) to[c] = there && c < have ? val(from[c]) : 0.f;
}
template <typename T, int VJ> __global__ void __launch_bounds__(PLAIN_THREADS) tree_plain_kernel(const __grid_constant__ Params p) {
  early_start();
  extern __shared__ __align__(16) float sm[];
  const int d4 = (p.dim + 3) / 4 * 4, v32 = VJ * 32, kld = d4 + 4, vld = v32 + 4, pld = PKEYS + 4;
  float *Q = sm, *K = Q + PROWS * kld, *V = K + PKEYS * kld, *P = V + PKEYS * vld, *corr = P + PROWS * pld, *sum = corr + PROWS;
  const int tid = threadIdx.x, tx = tid & 7, ty = tid >> 3, mine = tid >> 2;      // mine: the row that the thread brings in and whose softmax it shares
  const bool async = p.dim % 4 == 0 && p.vdim % 4 == 0 && (reinterpret_cast<uintptr_t>(p.pool) & 15) == 0;
  const float inv_cap = p.softcap > 0.f ? 1.0f / p.softcap : 0.f;
  Cursor cursor(p);
  for (Piece k = next_piece(p, cursor); k.nt; k = next_piece(p, cursor)) {
    const Seq x = k.x;
    const int rows = min(PROWS, x.n * p.qpk - k.rt * PROWS), r0 = k.rt * PROWS, last = x.start + x.n, lowest = p.window ? max(0, x.start - p.window + 1) : 0;
    const int *table = p.page_table + (size_t)k.table * p.max_pages;
    // the thread's row of a tile: its page (-1: it is not the sequence's, or nobody sees it), looked up a tile ahead, and its place in the page
    auto page_of = [&](int t, int &in) {
      const int j = t * PKEYS + mine, page = j / p.page;
      in = j - page * p.page;
      return t < k.t0 + k.nt && j >= lowest && j < last ? table[page] : -1;
    };
    int in, in_next, phys = page_of(k.t0, in), phys_next = page_of(k.t0 + 1, in_next);
    auto keys_in = [&](int phys, int in) { row_in<T>(K + mine * kld, k_page<T>(p, max(phys, 0), k.g) + (size_t)in * p.dim, phys >= 0, p.dim, async); };
    auto values_in = [&](int phys, int in) { row_in<T>(V + mine * vld, v_page<T>(p, max(phys, 0), k.g) + (size_t)in * p.vdim, phys >= 0, p.vdim, async); };
    const int row = min(r0 + mine, x.n * p.qpk - 1), tok = row / p.qpk;      // (rows behind the last: anything)
    __syncthreads();
    row_in<float>(Q + mine * kld, reinterpret_cast<const float *>(p.queries) + (((size_t)k.s * p.most + tok) * p.n_head + k.g * p.qpk + row - tok * p.qpk) * d4, true, d4, true);
    keys_in(phys, in);
    asm volatile("cp.async.commit_group;" ::: "memory");
    values_in(phys, in);
    asm volatile("cp.async.commit_group;" ::: "memory");
    const int depth = p.depth[(size_t)k.s * p.most + tok];
    const uint32_t *seen = p.seen + ((size_t)k.s * p.most + tok) * WORDS;
    float o[2][VJ][4];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int j = 0; j < VJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[a][j][e] = 0.f;
    float m = -INFINITY, l = 0.f;        // of row tid / 4, the same in its four threads
    for (int t = k.t0; t < k.t0 + k.nt; ++t) {
      const int j0 = t * PKEYS;
      const bool all_seen = j0 + PKEYS <= x.start && (p.window == 0 || last - 1 - j0 < p.window);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncthreads();
      const uint32_t see = all_seen ? 0xffffffffu : seen_word(p, x, seen, depth, j0) >> (tid & 3) * 8;      // of the eight keys whose weights the thread works out
      float sc[2][4] = {};
#pragma unroll 2
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
        for (int j = 0; j < 4; ++j) P[(2 * ty + i) * pld + tx + 8 * j] = sc[i][j] * p.scale;
      __syncthreads();
      in = in_next;
      phys = phys_next;
      phys_next = page_of(t + 2, in_next);
      if (t + 1 < k.t0 + k.nt) keys_in(phys, in);
      asm volatile("cp.async.commit_group;" ::: "memory");
      {
        float4 *row = reinterpret_cast<float4 *>(P + mine * pld + (tid & 3) * 8);
        const float4 y = row[0], z = row[1];
        float w[8] = {y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w}, top = m, add = 0.f;
        if (p.softcap > 0.f) {
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = p.softcap * tanh_of(w[i] * inv_cap);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] = see >> i & 1 ? w[i] * kLog2e : -INFINITY;
          top = fmaxf(top, w[i]);
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float base = top == -INFINITY ? 0.f : top, f = exp2f(m - base);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] = exp2f(w[i] - base);
          add += w[i];
        }
        row[0] = make_float4(w[0], w[1], w[2], w[3]);
        row[1] = make_float4(w[4], w[5], w[6], w[7]);
        add += __shfl_xor_sync(0xffffffffu, add, 1);
        add += __shfl_xor_sync(0xffffffffu, add, 2);
        l = l * f + add;
        m = top;
        if ((tid & 3) == 0) corr[mine] = f;
      }
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float f = corr[2 * ty + i];
#pragma unroll
        for (int j = 0; j < VJ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][j][e] *= f;
      }
#pragma unroll 2
      for (int key = 0; key < PKEYS; ++key) {
        const float a = P[2 * ty * pld + key], b = P[(2 * ty + 1) * pld + key];
        // (a value that a row does not see may be infinite or NaN: it is left out, not multiplied by zero)
        const bool first = all_seen || a != 0.f, second = all_seen || b != 0.f;
#pragma unroll
        for (int j = 0; j < VJ; ++j) {
          const float4 y = *reinterpret_cast<const float4 *>(V + key * vld + 4 * tx + 32 * j);
          if (first) {
            o[0][j][0] = fmaf(a, y.x, o[0][j][0]); o[0][j][1] = fmaf(a, y.y, o[0][j][1]); o[0][j][2] = fmaf(a, y.z, o[0][j][2]); o[0][j][3] = fmaf(a, y.w, o[0][j][3]);
          }
          if (second) {
            o[1][j][0] = fmaf(b, y.x, o[1][j][0]); o[1][j][1] = fmaf(b, y.y, o[1][j][1]); o[1][j][2] = fmaf(b, y.z, o[1][j][2]); o[1][j][3] = fmaf(b, y.w, o[1][j][3]);
          }
        }
      }
      __syncthreads();
      if (t + 1 < k.t0 + k.nt) values_in(phys, in);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    if ((tid & 3) == 0) {
      sum[tid >> 2] = l;
      if (!k.whole && mine < rows) p.part_ml[(size_t)k.slot * p.part_ld + mine] = make_float2(m, l);
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
          *reinterpret_cast<float4 *>(p.part_o + (((size_t)k.slot * ((p.vdim + 3) / 4) + c / 4) * p.part_ld + r) * 4) = make_float4(o[i][j][0], o[i][j][1], o[i][j][2], o[i][j][3]);
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------ tensor cores
// One block per SM, 128 query rows against tiles of 128 keys.  Queries stay in tensor memory: shared memory is the ring of keys and values, whose depth decides how
// fast they come (32 KB of queries in two parts took two of its six slots: 234 us behind 60000 positions, 222 without).  S = Q K^T goes to tensor memory
// (lane = row), two softmax threads per row, one for each half of the keys, turn it into weights in place, and O += P V takes those from there and V, keys
// outermost as the cache has it, from shared memory.  A row's weights would lose 8 or 11 bits' worth when rounded once; as two parts (hi + lo) they keep 15 or
// more, for a second product with V; rotated queries come in two parts likewise.  Scores have two buffers, so that the products of one tile run beside the
// exponentials of the other.
//   warps 0-3, 4-7   softmax of the first and the second 64 keys; query rows in, results out
//   warps 8, 9       keys and values into a ring of tiles in the swizzled layout, by TMA: a box per page and 64 columns; pages of sizes that no box fits by
//                    asynchronous copies of 16 bytes.  Values that some rows do not see are gone over before they are used: zeros where the sequence has none.
//   warp 10          issues the products; owns the tensor memory: 2 x 128 columns of scores, 128 of output, 2 x 64 of queries.  (All 512 are asked for: they
//                    begin at 0.)
// (Twelve warps: an SM quarter's registers are shared by three.)
// A tile is 64 KB of keys and values for 1536 or, with rotation, 2048 cycles of products (128-wide heads), and 2600 cycles at this SM's share of memory.  Measured
// are 3700 behind 60000 positions: one warp asks for boxes (700 for a tile of keys or values), one issues products, and each tile's softmax, products and copies
// hand it on to one another.  Behind some hundred positions a block has one or two tiles, and what bounds it is the way from the plan to the first weights.
// The running maximum is only raised, and the output rescaled, when a score exceeds it by 2^kRaise: weights stay below 2^8 (2^15.9 in fp16, where they are kept 2^13.9 times
// as large, so that small ones keep their bits).
constexpr int SOFT_WARPS = 8, COPY_WARPS = 2, MMA_WARP = SOFT_WARPS + COPY_WARPS, TENSOR_THREADS = 384, TROWS = 128, TKEYS = 128, MAX_SLOTS = 10;
constexpr int RING_BYTES = 192 * 1024, O_COL = 256, Q_COL = 384, Q_LOW = 64;      // columns of output and queries, from there of the queries' second part

struct TcShared {
  // landed: by slot, like full.  A slot is sent for again when its products are done, which wait for both copying warps: so both have seen its phase before the next
  // can begin.  (One barrier for all slots had no such bound: the first warp could go on by two phases while the second was still at a tile.)
  uint64_t full[MAX_SLOTS], empty[MAX_SLOTS], landed[MAX_SLOTS], s_full[2], p_full[2], o_done[2], q_full, drained;
  uint32_t tmem;               // where the tensor memory begins (at 0: all of it is ours)
  volatile int abort;
  float top[2][2][TROWS], sum[2][2][TROWS];      // of a half of the keys: by tile, by piece (a warp may be one ahead of its partner)
  // Whether a piece has values that are not finite and that not every row sees: they are zeroed in shared memory (0 * inf would reach rows that do not see them),
  // and infinite_values gives them back to the rows that do.
  int any_bad[8];
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint64_t both(float x) {
  uint64_t y;
  asm("mov.b64 %0, {%1, %1};" : "=l"(y) : "f"(x));
  return y;
}
// Values with the keys outermost: 64 columns (128 bytes) of a key are a swizzled row, eight keys 1024 bytes, 64 columns more a block of 128 rows.
__device__ __forceinline__ uint64_t value_desc(uint32_t addr) { return (tc::smem_desc_sw128(addr) & ~((uint64_t)0x3fff << 16)) | (uint64_t)(TKEYS * 128 >> 4) << 16; }
__device__ __forceinline__ uint32_t product_desc(bool bf16, int n, bool b_by_rows) {
  return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (b_by_rows ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(TROWS >> 4) << 24;
}
// Byte of 16-byte unit c of row r of a tile of rows of 128 swizzled bytes (blocks of 128 rows).
__device__ __forceinline__ uint32_t swizzled(int r, int c) { return (uint32_t)((c >> 3) * (128 * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }
// A box of a tensor map into shared memory; its bytes arrive on `bar`.
__device__ __forceinline__ void box_load(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint64_t &bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map), "r"(tc::sa(&bar)), "r"(x), "r"(y), "r"(z)
               : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&v)[16]) {      // (to be waited for)
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
                 "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(taddr)
               : "memory");
}
// (The registers pass through, so that nothing reads them before.)
__device__ __forceinline__ void tmem_landed(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]),
                 "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
               : "memory");
}

struct Waits {          // a role's bounded waits: the whole warp goes the same way
  TcShared &sm;
  int *error_flag;
  __device__ __forceinline__ bool operator()(uint64_t &bar, uint32_t parity) const {
    const uint32_t b = tc::sa(&bar);
    bool ok = false;
    for (int i = 0; i < 64 && !ok; ++i) ok = mbar_test(b, parity);      // (a warp that lets itself be suspended wakes late)
    ok = __all_sync(0xffffffffu, ok || mbar_wait(b, parity, &sm.abort));
    if (!ok) {
      if (!sm.abort && error_flag) atomicCAS(error_flag, 0, 11);
      sm.abort = 1;
    }
    return ok;
  }
  __device__ __forceinline__ void arrive(uint64_t &bar) const {      // one arrival of the warp
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(tc::sa(&bar));
  }
};

// Columns c0 .. c0 + 63 of a row's output, as it was stored: those with an infinite or NaN value that the row sees become the sum of these.  (What the products made of them is
// none: a weight comes in two parts, of which the second may be 0 or negative, and where not all rows see a value it was 0.)  all: look at every key of the piece, else only at
// those that not every row sees, which are the first MAX_NODES from the lowest that any row sees, where there is a window, and the drafted ones.  Four keys are asked for at
// once: others wait meanwhile, with a limit.  (Behind the stores and not in them: there it cost 0.4 us of 16, and 1.4 of 17.4 with a cap.)
template <typename T> __device__ __noinline__ void infinite_values(const Params &p, const Piece &k, int row, const uint32_t *seen, int depth, int c0, bool all) {
  const int start = k.x.start, low = p.window ? start + depth - p.window + 1 : 0, first = max(max(k.t0 * TKEYS, low), 0), last = min((k.t0 + k.nt) * TKEYS, start + k.x.n);
  const int skip = all ? last : p.window ? max(first, max(start - p.window + 1, 0) + MAX_NODES) : first;      // from here to `start` all rows see all
  const int *table = p.page_table + (size_t)k.table * p.max_pages;
  const int at = k.rt * TROWS + row, node = at / p.qpk, head = k.g * p.qpk + at - node * p.qpk;
  for (int c = c0; c < min(p.vdim, c0 + 64); c += 8) {
    float sum[8] = {};
    for (int j0 = first; j0 < last; j0 += 4) {
      if (j0 >= skip && j0 < start) j0 = start;
      uint4 w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = j0 + u, d = j - start, page = j / p.page;
        w[u] = make_uint4(0u, 0u, 0u, 0u);
        if (j < last && (d < 0 || (seen[d >> 5] >> (d & 31) & 1)))
          w[u] = *reinterpret_cast<const uint4 *>(v_page<T>(p, table[page], k.g) + (size_t)(j - page * p.page) * p.vdim + c);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t y[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!bad<T>(y[i])) continue;
          const float2 z = Half2<T>::wide(y[i]);
          if (!isfinite(z.x)) sum[2 * i] += z.x;
          if (!isfinite(z.y)) sum[2 * i + 1] += z.y;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (sum[i] == 0.f) continue;
      if (k.whole) reinterpret_cast<T *>(p.out)[(size_t)(k.x.row0 + node) * p.out_ld + (size_t)head * p.vdim + c + i] = rounded<T>(sum[i]);
      else p.part_o[(((size_t)k.slot * (p.vdim / 4) + (c + i) / 4) * p.part_ld + row) * 4 + (i & 3)] = sum[i];
    }
  }
}

// A piece's tile that some rows see in part: keys from `start` on are drafted, those in front of start + n - window are not seen by all.
__device__ __forceinline__ bool partial(const Params &p, const Seq &x, int j0) { return j0 + TKEYS > x.start || (p.window && x.start + x.n - 1 - j0 >= p.window); }
// CAP: scores go through cap tanh(score / cap).  As cap (1 - 2 / (e^2x + 1)) alone that is off by cap 2^-21, whatever the score: up to LOW_CAP less than what the weights lose
// as two parts and the output by its rounding.  Larger caps, which scores hardly reach, take tanh_of, which is right to 2^-20 of the score and costs twice the time
// (16 sequences: 68 us without a cap, 86 with a low one, 161; behind 60000 positions 187, 237, 508).
enum Cap { NO_CAP, LOW, ANY };
constexpr float LOW_CAP = 256.f;
template <typename T, Cap CAP> __global__ void __launch_bounds__(TENSOR_THREADS, 1) tree_tensor_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap keys, const __grid_constant__ CUtensorMap values) {
  early_start();
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) unsigned char raw[];
  unsigned char *base = raw + ((1024 - (tc::sa(raw) & 1023)) & 1023);
  const int kblocks = (p.dim + 63) / 64, vblocks = (p.vdim + 63) / 64, slot_bytes = max(kblocks, vblocks) * TKEYS * 128;
  const bool split_q = p.rope_half > 0;                     // query rows in two parts
  const int slots = min(MAX_SLOTS, RING_BYTES / slot_bytes);
  unsigned char *ring = base;
  TcShared &sm = *reinterpret_cast<TcShared *>(base + RING_BYTES);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  if (tid == 0) {
    for (int i = 0; i < slots; ++i) {
      mbar_init(tc::sa(&sm.full[i]), COPY_WARPS * 32);
      mbar_init(tc::sa(&sm.empty[i]), 1);
      mbar_init(tc::sa(&sm.landed[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(tc::sa(&sm.s_full[i]), 1);
      mbar_init(tc::sa(&sm.p_full[i]), SOFT_WARPS);
      mbar_init(tc::sa(&sm.o_done[i]), 1);
    }
    mbar_init(tc::sa(&sm.q_full), SOFT_WARPS);
    mbar_init(tc::sa(&sm.drained), 1);
    sm.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid < 8) sm.any_bad[tid] = 0;
  if (warp == MMA_WARP) tc::tmem_alloc(tc::sa(&sm.tmem), 512);
  tc::fence_before();
  Cursor cursor(p);
  __syncthreads();
  tc::fence_after();
  const Waits wait{sm, p.error_flag};

  if (warp >= SOFT_WARPS && warp < MMA_WARP) {
    // ---- keys and values
    const int w = warp - SOFT_WARPS;
    const int box = p.box, boxes = box ? TKEYS / box : 0;   // rows of a box, and how many make a tile
    const bool one = tc::elect_one();
    int slot = 0, phase = 1, e = 0, pieces = 0;             // where the next tile goes; tiles asked for
    uint32_t fixed = 0;                                     // by slot: the phase of `landed` that the next tile of values to be gone over has there
    bool ok = true, flying = false;                         // flying: a tile that was given up has not landed
    for (Piece k = next_piece(p, cursor); k.nt && ok; k = next_piece(p, cursor), ++pieces) {
      const Seq x = k.x;
      const int *table = p.page_table + (size_t)k.table * p.max_pages;
      const int lowest = p.window ? max(0, x.start - p.window + 1) : 0, last = x.start + x.n;
      auto page_of = [&](int j) { return j >= lowest && j < last ? table[j / p.page] : 0; };      // (what is not the sequence's: any page)
      // Page and row in it of a tile's boxes, one per lane, looked up a tile ahead (here and not where they are used: a division takes as long as a box)
      auto box_at = [&](int t) {
        const int j = t * TKEYS + lane * box, page = box ? j / p.page : 0;      // (a box lies in one page)
        return make_int2(w == 0 && lane < boxes && j + box > lowest && j < last ? table[page] : 0, k.g * p.page + j - page * p.page);
      };
      int2 ahead = box_at(k.t0);
      for (int t = 0; t < k.nt && ok; ++t) {
        const int j0 = (k.t0 + t) * TKEYS;
        const int2 here = ahead;
        ahead = box_at(k.t0 + t + 1);
        const bool part = partial(p, x, j0);
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv, ++e, phase ^= ++slot == slots, slot = slot == slots ? 0 : slot) {
          if (e >= slots && !wait(sm.empty[slot], phase)) { ok = false; break; }
          const uint32_t to = tc::sa(ring + slot * slot_bytes);
          const int dims = kv ? p.vdim : p.dim, blocks = kv ? vblocks : kblocks, have = dims / 8, pad = (dims + 15) / 16 * 2;
          const bool look = kv && part;                     // what is seen in part
          if (box) {
            uint64_t &bar = look ? sm.landed[slot] : sm.full[slot];
            if (w == 0) {
              if (tc::elect_one()) mbar_expect_tx(tc::sa(&bar), blocks * TKEYS * 128);
              __syncwarp();
#pragma unroll 1
              for (int i = 0; i < boxes; ++i) {
                const int page = __shfl_sync(0xffffffffu, here.x, i), y = __shfl_sync(0xffffffffu, here.y, i);
                if (tc::elect_one()) {                      // (said here, so that the compiler knows that one lane goes in: the instruction wants its operands the same in all)
                  box_load(to + i * box * 128, kv ? &values : &keys, 0, y, page, bar);
                  if (blocks > 1) box_load(to + TKEYS * 128 + i * box * 128, kv ? &values : &keys, 64, y, page, bar);
                }
                __syncwarp();
              }
            }
            if (!look) {
              if (w || !one) mbar_arrive(tc::sa(&bar));
              continue;
            }
            if (!wait(sm.landed[slot], fixed >> slot & 1)) { ok = false; flying = true; break; }
            fixed ^= 1u << slot;
          } else {
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              const int r0 = w * 64 + h * 32, j = j0 + r0 + lane;
              const bool in = j >= lowest && j < last;
              const T *src = (kv ? v_page<T>(p, page_of(j), k.g) : k_page<T>(p, page_of(j), k.g)) + (size_t)(in ? j % p.page : 0) * dims;
              const int cols = blocks * 8, c = lane % cols;
              for (int q0 = 0; q0 < 32; q0 += 32 / cols) {
                const int r = q0 + lane / cols;
                const unsigned long long from = __shfl_sync(0xffffffffu, (unsigned long long)src, r);
                const bool there = __shfl_sync(0xffffffffu, in ? 1 : 0, r) && c < have;
                if (c < pad) cp_async(to + swizzled(r0 + r, c), reinterpret_cast<const T *>(from) + (there ? c * 8 : 0), there ? 16 : 0);
              }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
          }
          if (look) {
            // rows that the sequence has not: zeros; rows that not all see: made finite, and said
            const int cols = blocks * 8, c = lane % cols, r1 = w * 64 + 64;
            int r = w * 64 + lane / cols;
            if (!p.window) r += max(0, (x.start - j0 - r) / (32 / cols)) * (32 / cols);      // (those in front all see)
#pragma unroll 2
            for (; r < r1; r += 32 / cols) {
              const int key = j0 + r, d = key - x.start, b = key - lowest;
              if (c >= have || (d < 0 && b >= MAX_NODES)) continue;
              uint4 *at = reinterpret_cast<uint4 *>(ring + slot * slot_bytes + swizzled(r, c));
              const bool in = key >= lowest && key < last;
              if (in) {
                const uint4 v = *at;
                if ((!bad<T>(v.x) && !bad<T>(v.y) && !bad<T>(v.z) && !bad<T>(v.w)) || (d < 0 && !p.window)) continue;
                sm.any_bad[pieces & 7] = 1;
                *at = make_uint4(finite<T>(v.x), finite<T>(v.y), finite<T>(v.z), finite<T>(v.w));
              } else {
                *at = make_uint4(0u, 0u, 0u, 0u);
              }
            }
          }
          tc::fence_operands();
          mbar_arrive(tc::sa(&sm.full[slot]));
        }
      }
    }
    // nothing is in flight when the block ends, after a failure either
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (w == 0 && box) {
      mbar_wait_ring(tc::sa(&sm.full[0]), e, slots);
      if (flying) mbar_wait_all(tc::sa(&sm.landed[slot]), fixed >> slot & 1);
    }
  } else if (warp == MMA_WARP) {
    // ---- products.  (What they take is the same in all lanes, and the compiler knows it: counters that go up by known steps, in loops whose bounds come
    // out of a reduction.  After a wait that ran out they go on: nobody reads what they give.)
    const int ksteps = (p.dim + 15) / 16, vcols = (p.vdim + 15) / 16 * 16;
    const uint32_t kdesc = product_desc(BF16, TKEYS, false), vdesc = product_desc(BF16, vcols, true);
    const uint64_t r0 = tc::smem_desc_sw128(tc::sa(ring)), rv0 = value_desc(tc::sa(ring));
    struct Place { int slot, phase; } at_k{0, 0}, at_v{1, 0};      // of the next tiles of keys and of values
    auto on = [&](Place &x) {
      x.slot += 2;
      if (x.slot >= slots) { x.slot -= slots; x.phase ^= 1; }
    };
    int pieces = 0, done = 0;                               // tiles done
    auto scores = [&](int b) {
      wait(sm.full[at_k.slot], at_k.phase);
      tc::fence_after();
      if (tc::elect_one()) {
        const uint64_t kt = r0 + (uint64_t)(uint32_t)(at_k.slot * (slot_bytes / 16));
        for (int part = 0; part < (split_q ? 2 : 1); ++part) {
          const uint32_t qt = Q_COL + part * Q_LOW;
          if (ksteps == 8) {
#pragma unroll
            for (int s = 0; s < 8; ++s) tc::umma_ta(b * 128, qt + s * 8, kt + (s >> 2) * (128 * 128 / 16) + (s & 3) * 2, kdesc, part > 0 || s > 0);
          } else {
            for (int s = 0; s < ksteps; ++s) tc::umma_ta(b * 128, qt + s * 8, kt + (s >> 2) * (128 * 128 / 16) + (s & 3) * 2, kdesc, part > 0 || s > 0);
          }
        }
        tc::umma_commit(tc::sa(&sm.empty[at_k.slot]));
        tc::umma_commit(tc::sa(&sm.s_full[b]));
      }
      __syncwarp();
      on(at_k);
    };
    // (Tiles come as K V K V ..; the scores of the next tile but one are asked for behind this one's output.)
    int used0 = 0, used1 = 0;                               // of either buffer
    for (;; ++pieces) {
      const int nt = __reduce_max_sync(0xffffffffu, next_piece(p, cursor).nt);
      if (!nt) break;
      wait(sm.q_full, pieces & 1);
      tc::fence_after();
      scores(0);
      if (nt > 1) scores(1);
      for (int t = 0; t < nt; ++t, ++done) {
        const int b = t & 1;
        wait(sm.full[at_v.slot], at_v.phase);
        wait(sm.p_full[b], (b ? used1++ : used0++) & 1);
        tc::fence_after();
        if (tc::elect_one()) {
          const uint64_t vt = rv0 + (uint64_t)(uint32_t)(at_v.slot * (slot_bytes / 16));
#pragma unroll
          for (int s = 0; s < 16; ++s)                      // (hi and lo of 16 keys: 8 columns each)
            tc::umma_ta(O_COL, b * 128 + (s >> 1) * 16 + (s & 1) * 8, vt + (s >> 1) * (2048 / 16), vdesc, t > 0 || s > 0);
          tc::umma_commit(tc::sa(&sm.empty[at_v.slot]));
          tc::umma_commit(tc::sa(&sm.o_done[done & 1]));
        }
        __syncwarp();
        on(at_v);
        if (t + 2 < nt) scores(b);
      }
    }
    // nothing may be on its way to tensor or shared memory when the block ends
    if (tc::elect_one()) {
      tc::umma_commit(tc::sa(&sm.drained));
      mbar_wait_all(tc::sa(&sm.drained), 0);
    }
    __syncwarp();
  } else if (warp < SOFT_WARPS) {
    // ---- softmax
    const int half = warp >> 2, q = warp & 3, row = q * 32 + lane;
    const uint32_t lanes = (uint32_t)(q * 32) << 16, S = lanes + half * 64, O = lanes + O_COL;
    int pieces = 0, n_s[2] = {0, 0}, n_o = 0;
    const float a1 = fmaxf(fabsf(p.scale), 1e-30f) * kLog2e, a2 = CAP == LOW ? 2.0f * a1 / p.softcap : CAP ? fmaxf(fabsf(p.scale), 1e-30f) / p.softcap : 0.f, b2 = p.softcap * kLog2e;
    // (a scale of zero: so small that all scores are equal, but -inf, which marks what is not seen, times it is -inf)
    auto score = [&](float s) { return CAP == LOW ? b2 * (1.0f - __fdividef(2.0f, ex2(a2 * s) + 1.0f)) : __fmul_rn(b2, tanh_of(a2 * s)); };      // of a cap; grows with s
    const float unit = CAP ? 1.f : a1;                      // of what the maximum is kept in: capped scores in powers of 2, or scores as the products gave them
    auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(SOFT_WARPS * 32) : "memory"); };
    auto meet_partner = [&] { asm volatile("bar.sync %0, 64;" ::"r"(2 + q) : "memory"); };       // the warp with the same rows
    // The output of the block's tile i.  (By turns on two barriers: of either the phase before is done when the scores of tile i are, and the phase behind
    // needs weights that come later.)
    auto output_of = [&](int i) { wait(sm.o_done[i & 1], (i >> 1) & 1); };
    // (After a wait that ran out all go on without waiting: everybody comes to every meeting, and what is computed does not matter.)
    // Query rows of a piece to tensor memory, 64 dimensions a thread (rows that there are none of hold anything: they stay by themselves).
    auto stage = [&](const Piece &k) {
      const int all = k.x.n * p.qpk, r0 = k.rt * TROWS, per = p.dim / 8;
      if (q * 32 < all - r0 && half * 64 < p.dim) {
        const uint4 *from = p.queries + ((size_t)k.s * p.most * p.n_head + (size_t)k.g * all) * 2 * per + min(r0 + row, all - 1);
        for (int part = 0; part < (split_q ? 2 : 1); ++part) {
          uint32_t v[32];
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const int d = half * 8 + c;
            const uint4 w = d < per ? __ldcg(from + (size_t)(part * per + d) * all) : make_uint4(0u, 0u, 0u, 0u);
            v[4 * c] = w.x; v[4 * c + 1] = w.y; v[4 * c + 2] = w.z; v[4 * c + 3] = w.w;
          }
          tc::tmem_st32(lanes + Q_COL + part * Q_LOW + half * 32, v);
        }
        tc::tmem_wait_st();
        tc::fence_before();
      }
      wait.arrive(sm.q_full);
    };
    Piece k = next_piece(p, cursor);
    if (k.nt) stage(k);
    for (; k.nt; ++pieces) {
      const Seq x = k.x;
      const int r0 = k.rt * TROWS, rows = min(TROWS, x.n * p.qpk - r0);
      const bool live = q * 32 < rows;                      // (uniform over the warp)
      const int at = min(r0 + row, x.n * p.qpk - 1), node = at / p.qpk, head = k.g * p.qpk + at - node * p.qpk, depth = p.parent ? p.depth[(size_t)k.s * p.most + node] : node;
      const uint32_t *seen = p.seen + ((size_t)k.s * p.most + node) * WORDS;
      float m = -INFINITY, l = 0.f;                         // m: the maximum that the exponents are relative to; l: of this half
      // Scores of a tile's half to weights.  (In loops of 32 keys: a block that has a tile or two fetches this code once, and waits for it.  Measured with 64 keys
      // in line and the mask in a copy of it, 5 tokens behind 700: a third of all waiting was for instructions.)
      auto weigh = [&](int t) {
        const uint32_t at = S + (t & 1) * 128;
        const int j0 = (k.t0 + t) * TKEYS;
        if (partial(p, x, j0)) {
#pragma unroll 1
          for (int c = 0; c < 64; c += 16) {
            uint32_t v[16];
            tc::tmem_ld16(at + c, v);
            const uint32_t see = seen_word(p, x, seen, depth, j0 + half * 64 + c);
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (!(see >> i & 1)) v[i] = 0xff800000u;       // -inf
            tmem_store16(at + c, v);
          }
          tc::tmem_wait_st();
        }
        uint32_t a[16], b[16];
        tmem_load(at, a);
        float tops[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
        for (int c = 0; c < 64; c += 32) {
          tmem_landed(a);
          tmem_load(at + c + 16, b);
#pragma unroll
          for (int i = 0; i < 16; ++i) tops[i & 1] = fmaxf(tops[i & 1], __uint_as_float(a[i]));
          tmem_landed(b);
          tmem_load(at + (c + 32 & 63), a);                  // (the last: the first again)
#pragma unroll
          for (int i = 0; i < 16; ++i) tops[i & 1] = fmaxf(tops[i & 1], __uint_as_float(b[i]));
        }
        float top = fmaxf(tops[0], tops[1]);
        sm.top[t & 1][half][row] = top;
        meet_partner();
        top = fmaxf(top, sm.top[t & 1][1 - half][row]);
        if (CAP && top != -INFINITY) top = score(top);
        // (keys that went before lie far below, or none was seen: the sums so far are scaled to the new maximum)
        const bool raise = row < rows && (top - m) * unit > Half2<T>::kRaise;
        if (__any_sync(0xffffffffu, raise) && t > 0) {
          const float f = raise ? ex2((m - top) * unit) : 1.f;        // (m = -inf: 0, of sums that are 0)
          l *= f;
          output_of(n_o - 1);
          tc::fence_after();
          tmem_landed(a);
#pragma unroll 1
          for (int c = half * 64; c < min(p.vdim, half * 64 + 64); c += 16) {
            tc::tmem_ld16(O + c, b);
#pragma unroll
            for (int i = 0; i < 16; ++i) b[i] = __float_as_uint(__uint_as_float(b[i]) * f);
            tmem_store16(O + c, b);
          }
        }
        if (raise) m = top;
        const float base = m == -INFINITY ? 0.f : m, ref = base - Half2<T>::kBias;
        // Exponents of two weights.  The maximum is taken off first and as it is: of large scores a product in full lies far beside a rounded one, and floats next to it are further
        // apart than weights may be.
        const uint64_t less = both(-base), times = both(a1), plus = both(Half2<T>::kBias);
        auto exponents = [&](float &y, float &z) {
          if (CAP) {                                         // (-inf stays what is not seen)
            if (y != -INFINITY) y = CAP == LOW ? score(y) - ref : (score(y) - base) + Half2<T>::kBias;
            if (z != -INFINITY) z = CAP == LOW ? score(z) - ref : (score(z) - base) + Half2<T>::kBias;
          } else {
            asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%0, %1};\n\tadd.rn.f32x2 t, t, %2;\n\tfma.rn.f32x2 t, t, %3, %4;\n\tmov.b64 {%0, %1}, t;\n\t}" : "+f"(y), "+f"(z) : "l"(less), "l"(times), "l"(plus));
          }
        };
        float add[4] = {0.f, 0.f, 0.f, 0.f};
        // 16 keys: eight columns of their weights' first parts, eight of the second
        auto sixteen = [&](const uint32_t (&v)[16], uint32_t to) {
          uint32_t o[16];
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            float y = __uint_as_float(v[i]), z = __uint_as_float(v[i + 1]);
            exponents(y, z);
            y = ex2(y);
            z = ex2(z);
            add[i & 2] += y;
            add[(i & 2) + 1] += z;
            Half2<T>::split(y, z, o[i / 2], o[8 + i / 2]);
          }
          tmem_store16(to, o);
        };
#pragma unroll 1
        for (int c = 0; c < 64; c += 32) {
          tmem_landed(a);
          tmem_load(at + c + 16, b);
          sixteen(a, at + c);
          tmem_landed(b);
          if (c == 0) tmem_load(at + 32, a);
          sixteen(b, at + c + 16);
        }
        l += (add[0] + add[1]) + (add[2] + add[3]);
      };
      for (int t = 0; t < k.nt; ++t, ++n_o) {               // (n_o: tiles whose output was asked for before this one)
        wait(sm.s_full[t & 1], n_s[t & 1]++ & 1);
        tc::fence_after();
        if (live) {
          weigh(t);
          tc::tmem_wait_st();
          tc::fence_before();
        }
        wait.arrive(sm.p_full[t & 1]);
      }
      // ---- the next piece's queries (all scores of this one are there: nobody reads its queries any more), then this one out; either half of the threads takes
      // half of the columns
      const Piece next = next_piece(p, cursor);
      if (next.nt) stage(next);
      sm.sum[pieces & 1][half][row] = l;
      meet();
      if (tid == 0) sm.any_bad[(pieces + 7) & 7] = 0;       // (of the piece before: everybody is past it)
      output_of(n_o - 1);
      tc::fence_after();
      if (live) {
        const float sum = sm.sum[pieces & 1][0][row] + sm.sum[pieces & 1][1][row];
        const bool store = row < rows;
        float odd = 0.f;                                    // NaN, if something came out infinite or NaN
        const float inv = k.whole ? 1.0f / sum : 1.0f;
        T *out = reinterpret_cast<T *>(p.out) + (size_t)(x.row0 + node) * p.out_ld + (size_t)head * p.vdim;
        if (!k.whole && half == 0 && store) p.part_ml[(size_t)k.slot * p.part_ld + row] = make_float2(m * unit - Half2<T>::kBias, sum);
#pragma unroll 1
        for (int c = half * 64; c < min(p.vdim, half * 64 + 64); c += 16) {
          uint32_t v[16];
          __syncwarp();
          tc::tmem_ld16(O + c, v);
          if (!store) continue;
#pragma unroll
          for (int z = 0; z < 16; z += 8) {
            if (c + z >= p.vdim) break;
#pragma unroll
            for (int b = 0; b < 8; ++b) odd = fmaf(__uint_as_float(v[z + b]), 0.f, odd);
            if (k.whole) {
              uint32_t y[4];
#pragma unroll
              for (int b = 0; b < 4; ++b) y[b] = Half2<T>::pack(__uint_as_float(v[z + 2 * b]) * inv, __uint_as_float(v[z + 2 * b + 1]) * inv);
              if (p.out16) {
                *reinterpret_cast<uint4 *>(out + c + z) = make_uint4(y[0], y[1], y[2], y[3]);
              } else {
                const T *e = reinterpret_cast<const T *>(y);
#pragma unroll
                for (int b = 0; b < 8; ++b) out[c + z + b] = e[b];
              }
            } else {
              uint4 *to = reinterpret_cast<uint4 *>(p.part_o + (((size_t)k.slot * (p.vdim / 4) + (c + z) / 4) * p.part_ld + row) * 4);
              to[0] = make_uint4(v[z], v[z + 1], v[z + 2], v[z + 3]);
              to[p.part_ld] = make_uint4(v[z + 4], v[z + 5], v[z + 6], v[z + 7]);
            }
          }
        }
        // (where the sum of the weights is NaN all is; what came out finite holds no infinite value of a tile that all rows see)
        if (store && (sm.any_bad[pieces & 7] || isnan(odd)) && !isnan(sum)) infinite_values<T>(p, k, row, seen, depth, half * 64, isnan(odd));
        __syncwarp();
        tc::fence_before();
      }
      k = next;
    }
  }
  __syncthreads();
  if (warp == MMA_WARP) {
    tc::fence_after();
    tc::tmem_dealloc(sm.tmem, 512);
  }
}
constexpr size_t tensor_smem() { return 1024 + RING_BYTES + sizeof(TcShared); }
static_assert(tensor_smem() + tc::TMEM_SHARED + 2 * tc::BLOCK_SHARED > tc::SM_SHARED, "the next kernel starts before a block has its columns: none that allocates some may fit beside it");

// ------------------------------------------------------------------------------------------ parts of an item
// Block (x: eight rows of an item, by the most that a sequence can have; y: sequence): adds up the parts in the order of the keys, in one pass with a running
// maximum and sum.  What bounds it is the latency of its loads: six parts are asked for at once (two passes of four loads took 18.2 us for 5 tokens behind 700
// and 29.3 for two kv heads of 8 sequences, this 17.3 and 27.0).
constexpr int COMBINE_THREADS = 256, COMBINE_ROWS = 8, AHEAD = 6;
template <typename T> __global__ void __launch_bounds__(COMBINE_THREADS) combine_kernel(const __grid_constant__ Params p) {
  early_start();
  const int s = blockIdx.y, tid = threadIdx.x, quota = p.plan[0], units = p.units[s];
  const Seq x = sequence(p, s);
  if (!x.n) return;
  const Span y = span(p, x);
  const int eights = (p.most * p.qpk + COMBINE_ROWS - 1) / COMBINE_ROWS, g = blockIdx.x / eights, r0 = (blockIdx.x - g * eights) * COMBINE_ROWS;   // (first row, of all of the kv head's)
  const int rows = min(COMBINE_ROWS, x.n * p.qpk - r0), rt = r0 >> p.rows_shift;
  if (rows <= 0) return;
  const int first = units + (g * y.row_tiles + rt) * (y.tiles + p.extra) + p.extra, b0 = first / quota, b1 = (first + y.tiles - 1) / quota;
  if (b0 == b1) return;
  const int v4 = (p.vdim + 3) / 4;
  const int mine = tid % COMBINE_ROWS, r = (r0 & (p.rows_tile - 1)) + mine;      // eight rows of a column lie side by side: 128 bytes
  if (mine >= rows) return;
  for (int c = tid / COMBINE_ROWS; c < v4; c += COMBINE_THREADS / COMBINE_ROWS) {
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int b = b0; b <= b1; b += AHEAD) {
      float2 ml[AHEAD];
      float4 w[AHEAD];
      float top = m;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const size_t slot = 2 * min(b + i, b1) + (b + i == b0 ? 1 : 0);
        ml[i] = p.part_ml[slot * p.part_ld + r];
        w[i] = *reinterpret_cast<const float4 *>(p.part_o + ((slot * v4 + c) * p.part_ld + r) * 4);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) top = fmaxf(top, ml[i].x);
      const float ref = top == -INFINITY ? 0.f : top, old = exp2f(m - ref);
      o.x *= old; o.y *= old; o.z *= old; o.w *= old;
      l *= old;
      m = top;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (b + i > b1) break;
        const float f = exp2f(ml[i].x - ref);
        o.x = fmaf(w[i].x, f, o.x); o.y = fmaf(w[i].y, f, o.y); o.z = fmaf(w[i].z, f, o.z); o.w = fmaf(w[i].w, f, o.w);
        l = fmaf(ml[i].y, f, l);
      }
    }
    const float inv = 1.0f / l;
    const int row = r0 + mine, tok = row / p.qpk, h = g * p.qpk + row % p.qpk;
    T *out = reinterpret_cast<T *>(p.out) + (size_t)(x.row0 + tok) * p.out_ld + (size_t)h * p.vdim + 4 * c;
    const float z[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * c + i < p.vdim) out[i] = rounded<T>(z[i]);
  }
}

static size_t plan_ints() { return PLAN_HEAD + (size_t)sm_count() * PLAIN_BLOCKS * (sizeof(Start) / 4); }
// Rows of the parts: two tiles of every block of either kernel.
static size_t part_rows() { return (size_t)2 * sm_count() * std::max(TROWS + 8, PLAIN_BLOCKS * (PROWS + 8)); }

template <typename T, int VJ> static int launch_plain(Params &p, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  const size_t smem = plain_smem(p.dim, VJ * 32);
  if (smem > 32 * 1024) PT_CUDA(allow_smem(tree_plain_kernel<T, VJ>, (int)plain_smem(256, VJ * 32), done));
  PT_CUDA(launch_early(tree_plain_kernel<T, VJ>, Grid(p.blocks), PLAIN_THREADS, smem, st, p));
  PT_LAUNCH_CHECK("pt_tree_attn");
  return PT_OK;
}
using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// The rows of all pages' keys or values: [pages][n_kv page][width], boxes of 64 columns of `box` rows of one page.  (How many pages there are is the
// caller's to know: none that the table does not name is read.)
static bool page_map(CUtensorMap *map, CUtensorMapDataType dt, const void *base, int width, const Params &p) {
  static EncodeTiled fn = [] {
    void *ptr = nullptr;
    cudaDriverEntryPointQueryResult res;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &res) == cudaSuccess && res == cudaDriverEntryPointSuccess ? (EncodeTiled)ptr : nullptr;
  }();
  const cuuint64_t dims[3] = {(cuuint64_t)width, (cuuint64_t)p.n_kv * p.page, 1u << 30}, strides[2] = {(cuuint64_t)width * 2, (cuuint64_t)p.n_kv * p.page * (p.dim + p.vdim) * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)p.box, 1}, steps[3] = {1, 1, 1};
  return fn && fn(map, dt, 3, const_cast<void *>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, Cap CAP> static int launch_tensor(Params &p, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  PT_CUDA(allow_smem(tree_tensor_kernel<T, CAP>, (int)tensor_smem(), done));
  CUtensorMap keys{}, values{};
  p.box = 1;
  while (p.box < TKEYS && p.page % (2 * p.box) == 0) p.box *= 2;
  const CUtensorMapDataType dt = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if (p.box < 8 || !page_map(&keys, dt, p.pool, p.dim, p) || !page_map(&values, dt, (T *)p.pool + (size_t)p.n_kv * p.page * p.dim, p.vdim, p)) p.box = 0;      // (a swizzled box has rows in eights)
  PT_CUDA(launch_early(tree_tensor_kernel<T, CAP>, Grid(p.blocks), TENSOR_THREADS, tensor_smem(), st, p, keys, values));
  PT_LAUNCH_CHECK("pt_tree_attn");
  return PT_OK;
}
template <typename T> static int run(Params &p, bool tensor, cudaStream_t st) {
  int rc;
  const Grid prep(dim3(p.most, p.n_seq + 1));
  if constexpr (std::is_same<T, float>::value) tensor = false;
  // (an odd number of eights: rows of the same column of parts lie apart by no power of two)
  p.part_ld = (std::min(tensor ? TROWS : PROWS, p.most * p.qpk) + 7) / 8 * 8 | 8;
  if (tensor) {
    // (A piece beside its tiles costs about as much as two of them: queries in, the last weights and products, the output.  19 calls of all sizes, on average: 23.2 us; with
    // one, three or four 23.4.)
    p.rows_tile = TROWS; p.keys_tile = TKEYS; p.rows_shift = p.keys_shift = 7; p.extra = 2; p.blocks = sm_count();
    if constexpr (!std::is_same<T, float>::value) PT_CUDA(launch_early(tree_prep_kernel<T, true>, prep, PREP_THREADS, 0, st, p));
  } else {
    p.rows_tile = PROWS; p.keys_tile = PKEYS; p.rows_shift = p.keys_shift = 5; p.extra = 0; p.blocks = sm_count() * PLAIN_BLOCKS;
    PT_CUDA(launch_early(tree_prep_kernel<T, false>, prep, PREP_THREADS, 0, st, p));
  }
  PT_LAUNCH_CHECK("pt_tree_attn");
  if constexpr (!std::is_same<T, float>::value) {
    if (tensor) rc = p.softcap == 0.f ? launch_tensor<T, NO_CAP>(p, st) : p.softcap <= LOW_CAP ? launch_tensor<T, LOW>(p, st) : launch_tensor<T, ANY>(p, st);
  }
  if (!tensor) rc = p.vdim <= 64 ? launch_plain<T, 2>(p, st) : p.vdim <= 128 ? launch_plain<T, 4>(p, st) : launch_plain<T, 8>(p, st);
  if (rc) return rc;
  PT_CUDA(launch_early(combine_kernel<T>, Grid(dim3(p.n_kv * ceil_div(p.most * p.qpk, COMBINE_ROWS), p.n_seq)), COMBINE_THREADS, 0, st, p));
  PT_LAUNCH_CHECK("pt_tree_attn");
  return PT_OK;
}

}  // namespace ta
}  // namespace pt

using namespace pt;

// Workspace: the plan, units, depths and masks of all tokens; the queries as the attention kernel takes them (fp32, or of widths up to 128 two
// parts of 16 bits); the parts.
static size_t queries_offset(int n_seq, int most) { return ((ta::plan_ints() + n_seq + 1 + (size_t)n_seq * most * (1 + ta::WORDS)) * 4 + 255) / 256 * 256; }
static size_t part_offset(int n_seq, int most, int n_head) { return queries_offset(n_seq, most) + (size_t)n_seq * most * n_head * 256 * 4; }
extern "C" size_t pt_tree_attn_workspace_bytes(int n_seq, int max_tokens_per_seq, int n_head, int n_kv, int vdim) {
  (void)n_kv;
  return part_offset(n_seq, max_tokens_per_seq, n_head) + ta::part_rows() * (sizeof(float2) + (size_t)(vdim + 3) / 4 * 16);
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
  PT_REQUIRE(a->window >= 0 && (a->softcap == 0.f || (a->softcap >= 1e-20f && a->softcap <= 1e20f)), "pt_tree_attn: window=%d softcap=%g (0, or 1e-20 .. 1e20)", a->window, a->softcap);
  PT_REQUIRE(a->rope_dims >= 0 && a->rope_dims % 2 == 0 && a->rope_dims <= a->dim && (!a->rope_dims || a->rope), "pt_tree_attn: %d rotated dimensions of %d", a->rope_dims, a->dim);
  const long long positions = (long long)a->page_size * a->max_pages;
  PT_REQUIRE(positions < (1ll << 31) - 1024 && a->max_len <= positions, "pt_tree_attn: max_len=%d exceeds the %lld positions of the page table, or those are 2^31 or nearly", a->max_len,
             positions);
  ta::Params p{};
  p.n_seq = b.n_seq; p.n_tok = b.n_tok; p.n_head = a->n_head; p.n_kv = a->n_kv; p.qpk = a->n_head / a->n_kv; p.dim = a->dim; p.vdim = a->vdim;
  p.page = a->page_size; p.max_pages = a->max_pages; p.max_len = a->max_len > 0 ? a->max_len : (int)positions; p.window = a->window;
  p.most = a->max_tokens_per_seq > 0 ? a->max_tokens_per_seq : b.n_tok;
  PT_REQUIRE(p.most <= ta::MAX_NODES, "pt_tree_attn: %d tokens of one sequence (at most %d)", p.most, ta::MAX_NODES);
  // (a unit is 32 positions of a row tile: their number is an int)
  PT_REQUIRE((double)b.n_seq * a->n_kv * (p.most * p.qpk / 32 + 1) * (p.max_len / 32 + 4) < 2e9, "pt_tree_attn: %d sequences of up to %d positions and %d heads are too much for one call", b.n_seq,
             p.max_len, a->n_head);
  p.q_ld = a->q_ld; p.kv_ld = a->kv_ld; p.out_ld = a->out_ld; p.rope_half = a->rope_dims / 2;
  p.out_cols = a->out_cols > 0 ? a->out_cols : a->out_ld;
  PT_REQUIRE(p.out_cols >= a->n_head * a->vdim && p.out_cols <= a->out_ld, "pt_tree_attn: out_cols=%d", a->out_cols);
  p.scale = a->scale; p.softcap = a->softcap; p.q = a->q; p.k = a->k; p.v = a->v; p.pool = a->pool; p.out = a->out; p.rope = (const float2 *)a->rope;
  p.page_table = a->page_table; p.cu = b.cu; p.start = b.start; p.slot = b.slot; p.parent = a->parent; p.error_flag = a->error_flag;
  const size_t need = pt_tree_attn_workspace_bytes(b.n_seq, p.most, a->n_head, a->n_kv, a->vdim);
  PT_REQUIRE(a->workspace && a->workspace_bytes >= need && aligned_to(a->workspace, 16), "pt_tree_attn: %zu workspace bytes on a 16-byte boundary needed, got %zu", need, a->workspace_bytes);
  p.plan = (int *)a->workspace;
  p.units = p.plan + ta::plan_ints();
  p.depth = p.units + b.n_seq + 1;
  p.seen = (uint32_t *)(p.depth + (size_t)b.n_seq * p.most);
  p.queries = (uint4 *)((char *)a->workspace + queries_offset(b.n_seq, p.most));
  p.part_o = (float *)((char *)a->workspace + part_offset(b.n_seq, p.most, a->n_head));
  p.part_ml = (float2 *)(p.part_o + ta::part_rows() * ((a->vdim + 3) / 4 * 4));
  cudaStream_t st = as_stream(stream);
  p.out16 = a->out_ld % 8 == 0 && aligned_to(a->out, 16);
  const bool tensor = !a->plain && a->dtype != PT_DT_F32 && a->dim <= 128 && a->vdim <= 128 && a->dim % 8 == 0 && a->vdim % 8 == 0 && a->q_ld % 8 == 0 && a->kv_ld % 8 == 0 && aligned_to(a->q, 16) && aligned_to(a->k, 16) && aligned_to(a->v, 16) &&
                      aligned_to(a->pool, 16) && (p.rope_half % 8 || aligned_to(a->rope, 16));
  if (a->dtype == PT_DT_F32) return ta::run<float>(p, false, st);
  return a->dtype == PT_DT_F16 ? ta::run<__half>(p, tensor, st) : ta::run<__nv_bfloat16>(p, tensor, st);
}
