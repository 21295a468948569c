// Paged caches of eight bits: keys and values as bytes (int8 or E4M3), with a scale for every position and head.
//   pool[page] = K [n_kv][page_size][dim] and then V [n_kv][page_size][vdim], a byte each; scales[page] = fp32 [2][n_kv][page_size], K's and then V's.
// A row x of one position and head is kept as  byte_i = round(x_i (top / m)),  scale = m / top,  m = max_i |x_i|  (top: 127 or 448).  m is at least 2^-64, so that
// top / m is finite; a row that has a NaN, an infinity or a magnitude above 2^64 gets the scale NaN and bytes of 0, and reads back as NaN.
#include <type_traits>

#include "rotate.cuh"

namespace pt {
namespace kv8 {

constexpr int THREADS = 256;
constexpr float SMALL = 0x1p-64f, LARGE = 0x1p64f;

// Division by what a launch has but once: n / d = (n + high word of n mul) >> shift for 0 <= n < 2^31, mul = ceil(2^32 (2^shift - d) / d), 2^shift the power of two at or above d.
struct Divide {
  uint32_t d, mul, shift;
  __host__ static Divide by(uint32_t d) {
    Divide r{d, 0, 0};
    while ((1ull << r.shift) < d) ++r.shift;
    r.mul = (uint32_t)((((1ull << r.shift) - d) << 32) / d + 1);
    return r;
  }
  __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift); }
};

struct Cache {
  unsigned char *pool;
  float *scales;
  const int *page_table;
  int n_kv, dim, vdim, page, max_pages, max_len;
  size_t page_bytes;
};
struct Batch {
  int n_seq, n_tok;
  const int *cu, *start, *slot, *tok_seq;
};

template <bool E4M3> __device__ __forceinline__ float top_byte() { return E4M3 ? 448.f : 127.f; }
template <bool E4M3> __device__ __forceinline__ float from_byte(unsigned char b) {
  if constexpr (E4M3) {
    __nv_fp8_e4m3 x;
    x.__x = b;
    return float(x);
  }
  return (float)(signed char)b;
}
template <bool E4M3> __device__ __forceinline__ uint32_t to_byte(float x) {
  if constexpr (E4M3) return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
  return (uint32_t)max(-127, min(127, __float2int_rn(x))) & 0xFFu;
}
// The largest magnitude of three values; NaN if one of them is.
__device__ __forceinline__ float larger(float a, float b, float c) {
  float m;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
// Four values as a word.
template <bool E4M3> __device__ __forceinline__ uint32_t to_word(float a, float b, float c, float d) {
  if constexpr (E4M3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3), hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
  }
  // (|x| is at most 127 (1 + 2^-23): behind 1.5 2^23 the nearest whole number, ties to even, is in the lowest byte)
  const uint32_t w = __float_as_uint(__fadd_rn(a, 12582912.f)), x = __float_as_uint(__fadd_rn(b, 12582912.f)), y = __float_as_uint(__fadd_rn(c, 12582912.f)), z = __float_as_uint(__fadd_rn(d, 12582912.f));
  return __byte_perm(__byte_perm(w, x, 0x0040), __byte_perm(y, z, 0x0040), 0x5410);
}

// Whether a sequence's new positions can be there, and the page and place of one.
__device__ __forceinline__ bool in_table(const Cache &c, int start, int count) { return start >= 0 && count <= c.max_len - start; }

// ------------------------------------------------------------------------------------------ rotation
struct Rotary {
  int rows, heads, dim, rot, x_ld, out_ld, positions;
  const int *position;
  const float2 *rope;
  int *error_flag;
  Divide by_heads;
};
// LANES lanes (16 elements each) for a head of a row; a thread has one.  Bound by memory: rows in and out once.  So nothing waits for the position before the row has been asked for, and no lane
// loops (4000 rows of 34 heads of 128, half of each turned: 13.3 us, 5.3 TB/s; a block a row, whose lanes went
// through its heads in turn with the angles in registers, 16.1).
template <typename T, int LANES, bool WHOLE, bool INVERSE, bool NEIGHBOURS>
__global__ void __launch_bounds__(THREADS, 4) rotary_kernel(const T *x, T *out, const Rotary p) {
  early_start();
  const int item = blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES, t = threadIdx.x % LANES, row = p.by_heads(item), h = item - row * p.heads;
  if (row >= p.rows || 16 * t >= p.dim) return;
  const T *from = x + (size_t)row * p.x_ld + (size_t)h * p.dim;
  T *to = out + (size_t)row * p.out_ld + (size_t)h * p.dim;
  const Runs runs = runs_of(t, p.dim, p.rot, NEIGHBOURS);
  Raw<T> raw;
  if constexpr (WHOLE) raw = load_raw(from, runs);
  const int pos = p.position[row];
  if (pos < 0 || pos >= p.positions) {
    if (h == 0 && t == 0 && p.error_flag) atomicExch(p.error_flag, 12);
    return;
  }
  const float2 *angles = p.rope + (size_t)pos * (p.rot / 2);
  const float sign = INVERSE ? -1.f : 1.f;
  if constexpr (WHOLE) {
    Item v = item_of<T>(raw);
    turn_item(v, load_angles(angles, runs, NEIGHBOURS), runs, NEIGHBOURS, sign);
    store_run(to + runs.lo, v.lo);
    store_run(to + runs.hi, v.hi);
  } else {
    Item v = load_pairs(from, t, p.dim, p.rot, NEIGHBOURS);
    turn_pairs(v, angles, t, p.rot, sign);
    store_pairs(to, v, t, p.dim, p.rot, NEIGHBOURS);
  }
}

// ------------------------------------------------------------------------------------------ appending
struct Append {
  Batch b;
  Cache c;
  int heads, rot, ld, q_out_ld;
  const float2 *rope;
  int *error_flag;
  Divide by_page, by_q, by_kv;      // a page's positions; a token's query heads and its kv heads in groups of ROWS
  int q_blocks, kv_blocks;          // blocks of query heads, of keys (and as many of values)
};
enum Kind { QUERY, KEY, VALUE };
// LANES lanes have the same sixteenth elements of ROWS neighbouring heads of a token: of queries, which are rotated, of keys, rotated and kept as bytes, or of values, kept as bytes.
template <typename T, int LANES, int ROWS, bool WHOLE, bool NEIGHBOURS, bool E4M3, Kind KIND>
__device__ __forceinline__ void append_rows(const T *src, T *q_out, const Append &p, int block) {
  const int heads = KIND == QUERY ? p.heads : p.c.n_kv, dim = KIND == VALUE ? p.c.vdim : p.c.dim, rot = KIND == VALUE ? 0 : p.rot;
  const Divide &by = KIND == QUERY ? p.by_q : p.by_kv;
  const int item = block * (THREADS / LANES) + threadIdx.x / LANES, t = threadIdx.x % LANES, tok = by(item), h0 = (item - tok * (int)by.d) * ROWS;
  const bool there = tok < p.b.n_tok, mine = there && 16 * t < dim;
  const Runs runs = runs_of(t, dim, rot, NEIGHBOURS);
  const T *from = src + (size_t)tok * p.ld + h0 * dim;
  const int used = p.b.cu[p.b.n_seq], seq = there ? p.b.tok_seq[tok] : 0;
  Raw<T> raw[ROWS];
  if constexpr (WHOLE) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
      if (mine && h0 + i < heads) raw[i] = load_raw(from + i * dim, runs);
  }
  int pos = -1, page = -1;
  if (there && tok < used) {
    const int first = p.b.cu[seq], start = p.b.start[seq];
    if (in_table(p.c, start, p.b.cu[seq + 1] - first)) {
      pos = start + tok - first;
      page = p.c.page_table[(size_t)p.b.slot[seq] * p.c.max_pages + p.by_page(pos)];
    }
    if (page < 0 && h0 == 0 && t == 0 && p.error_flag) atomicExch(p.error_flag, 12);
  }
  const bool fits = mine && page >= 0;
  const float2 *row = p.rope + (size_t)max(pos, 0) * (rot / 2);
  Angles angles{};
  if (WHOLE && KIND != VALUE && fits) angles = load_angles(row, runs, NEIGHBOURS);
  const int place = pos - p.by_page(max(pos, 0)) * p.c.page;
  unsigned char *to = p.c.pool + (size_t)max(page, 0) * p.c.page_bytes + (KIND == VALUE ? (size_t)p.c.n_kv * p.c.page * p.c.dim : 0) + ((size_t)h0 * p.c.page + place) * dim;
  float *scale = p.c.scales + ((size_t)max(page, 0) * 2 + (KIND == VALUE)) * p.c.n_kv * p.c.page + h0 * p.c.page + place;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {      // (whole warps stay together: the lanes of a row exchange their maxima)
    const bool in = fits && h0 + i < heads;
    Item x{};
    if (in) {
      if constexpr (WHOLE) {
        x = item_of<T>(raw[i]);
        if (KIND != VALUE) turn_item(x, angles, runs, NEIGHBOURS, 1.f);
      } else {
        x = load_pairs(from + i * dim, t, dim, rot, NEIGHBOURS);
        if (KIND != VALUE) turn_pairs(x, row, t, rot, 1.f);
      }
    }
    if constexpr (KIND == QUERY) {
      T *out = q_out + (size_t)tok * p.q_out_ld + (h0 + i) * dim;
      if (!in) continue;
      if constexpr (WHOLE) {
        store_run(out + runs.lo, x.lo);
        store_run(out + runs.hi, x.hi);
      } else {
        store_pairs(out, x, t, dim, rot, NEIGHBOURS);
      }
    } else {
      float m = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = larger(m, x.lo[j], x.hi[j]);
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) m = larger(m, __shfl_xor_sync(0xffffffffu, m, o), 0.f);
      if (!in) continue;
      const bool fine = m <= LARGE;
      const float most = fmaxf(m, SMALL), times = __fdiv_rn(top_byte<E4M3>(), most);
      if (t == 0) scale[i * p.c.page] = fine ? __fdiv_rn(most, top_byte<E4M3>()) : __uint_as_float(0x7fffffffu);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x.lo[j] = __fmul_rn(x.lo[j], times);
        x.hi[j] = __fmul_rn(x.hi[j], times);
      }
      if (!fine) x = Item{};
      unsigned char *bytes = to + (size_t)i * p.c.page * dim;
      if constexpr (WHOLE) {
        *reinterpret_cast<uint2 *>(bytes + runs.lo) = make_uint2(to_word<E4M3>(x.lo[0], x.lo[1], x.lo[2], x.lo[3]), to_word<E4M3>(x.lo[4], x.lo[5], x.lo[6], x.lo[7]));
        *reinterpret_cast<uint2 *>(bytes + runs.hi) = make_uint2(to_word<E4M3>(x.hi[0], x.hi[1], x.hi[2], x.hi[3]), to_word<E4M3>(x.hi[4], x.hi[5], x.hi[6], x.hi[7]));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int2 e = pair_at(8 * t + j, rot, NEIGHBOURS);
          if (e.x < dim) bytes[e.x] = (unsigned char)to_byte<E4M3>(x.lo[j]);
          if (e.y < dim) bytes[e.y] = (unsigned char)to_byte<E4M3>(x.hi[j]);
        }
      }
    }
  }
}
// Bound by memory, and before that by the way to a token's place (sequence, position, page, angles), which is gone once for all of a lane's rows, after they have been asked for.  11,000 tokens
// of 32 + 8 + 8 heads of 128, 250 MB: 46.0 us, 5.4 TB/s; a row a lane 69.7, two rows of any kind 59.0 (selects and addresses of three kinds).  Where there is less than a wave of rows one is
// faster: a token 2.4 us.
template <typename T, int LANES, int ROWS, bool WHOLE, bool NEIGHBOURS, bool E4M3>
__global__ void __launch_bounds__(THREADS, 4) append_kernel(const T *q, const T *k, const T *v, T *q_out, const Append p) {
  early_start();
  const int block = blockIdx.x;
  if (block < p.kv_blocks) append_rows<T, LANES, ROWS, WHOLE, NEIGHBOURS, E4M3, KEY>(k, nullptr, p, block);
  else if (block < 2 * p.kv_blocks) append_rows<T, LANES, ROWS, WHOLE, NEIGHBOURS, E4M3, VALUE>(v, nullptr, p, block - p.kv_blocks);
  else append_rows<T, LANES, ROWS, WHOLE, NEIGHBOURS, E4M3, QUERY>(q, q_out, p, block - 2 * p.kv_blocks);
}

// ------------------------------------------------------------------------------------------ pages in a wider type
struct Unpack {
  Batch b;
  Cache c;
  const int *into_table;
  int into_page, into_max_pages, into_max_len, rows_each, heads_each;
  int *error_flag;
  Divide by_page, by_into_page;
};
template <bool E4M3> __device__ __forceinline__ void from_word(uint32_t w, float scale, float *v) {
  if constexpr (E4M3) {
    const float2 a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3))), b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3)));
    v[0] = a.x * scale; v[1] = a.y * scale; v[2] = b.x * scale; v[3] = b.y * scale;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)(signed char)(w >> (8 * j)) * scale;
  }
}
// Block: rows_each positions of a sequence, keys or values of heads_each heads.  Bound by memory: a thread finds its places once and asks for four heads' bytes together, and a warp's stores are whole
// sectors.  4 sequences of up to 16500 positions, 8 heads of 128, E4M3 to fp16, 299 MB: 49.7 us, 6.0 TB/s (a block a head, which found its places again, 63.4; stores of half sectors 60.4).
template <typename T, bool WHOLE, bool E4M3> __global__ void __launch_bounds__(THREADS) unpack_kernel(T *into, const Unpack p) {
  early_start();
  const int parts = gridDim.z / 2;
  const bool is_v = blockIdx.z >= parts;
  const int seq = blockIdx.y, G = p.c.n_kv, h0 = (blockIdx.z - (is_v ? parts : 0)) * p.heads_each, h1 = min(G, h0 + p.heads_each), first = blockIdx.x * p.rows_each;
  const int start = p.b.start[seq], count = p.b.cu[seq + 1] - p.b.cu[seq], slot = p.b.slot[seq];
  if (!in_table(p.c, start, count) || count > p.into_max_len - start) {
    if (blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0 && p.error_flag) atomicExch(p.error_flag, 12);
    return;
  }
  const int rows = min(p.rows_each, start + count - first), dim = is_v ? p.c.vdim : p.c.dim;
  if (rows <= 0) return;
  const int *table = p.c.page_table + (size_t)slot * p.c.max_pages, *into_table = p.into_table + (size_t)slot * p.into_max_pages;
  const size_t into_page_elements = (size_t)G * p.into_page * (p.c.dim + p.c.vdim);
  constexpr int UNIT = WHOLE ? 16 / (int)sizeof(T) : 1, TOGETHER = 4;      // (16 bytes of the wider type: the warps' stores are whole)
  using Bytes = std::conditional_t<UNIT == 4, uint32_t, uint2>;
  const int units = dim / UNIT;
  for (int i = threadIdx.x; i < rows * units; i += THREADS) {
    const int r = i / units, u = i - r * units, pos = first + r, pg = p.by_page(pos), to_pg = p.by_into_page(pos);
    const int page = table[pg], to_page = into_table[to_pg];
    if (page < 0 || to_page < 0) {
      if (p.error_flag) atomicExch(p.error_flag, 12);
      continue;
    }
    const int place = pos - pg * p.c.page;
    const float *scale = p.c.scales + ((size_t)page * 2 * G + (is_v ? G : 0)) * p.c.page + place;
    const unsigned char *from = p.c.pool + (size_t)page * p.c.page_bytes + (is_v ? (size_t)G * p.c.page * p.c.dim : 0) + (size_t)place * dim + (size_t)u * UNIT;
    T *to = into + (size_t)to_page * into_page_elements + (is_v ? (size_t)G * p.into_page * p.c.dim : 0) + (size_t)(pos - to_pg * p.into_page) * dim + (size_t)u * UNIT;
    if constexpr (WHOLE) {
      for (int h = h0; h < h1; h += TOGETHER) {
        Bytes w[TOGETHER];
        float s[TOGETHER];
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k)
          if (h + k < h1) {
            w[k] = *reinterpret_cast<const Bytes *>(from + (size_t)(h + k) * p.c.page * dim);
            s[k] = scale[(size_t)(h + k) * p.c.page];
          }
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k)
          if (h + k < h1) {
            T *at = to + (size_t)(h + k) * p.into_page * dim;
            if constexpr (UNIT == 4) {
              float v[4];
              from_word<E4M3>(w[k], s[k], v);
              *reinterpret_cast<float4 *>(at) = make_float4(v[0], v[1], v[2], v[3]);
            } else {
              float v[8];
              from_word<E4M3>(w[k].x, s[k], v); from_word<E4M3>(w[k].y, s[k], v + 4);
              store_run(at, v);
            }
          }
      }
    } else {
      for (int h = h0; h < h1; ++h) to[(size_t)h * p.into_page * dim] = from_f<T>(from_byte<E4M3>(from[(size_t)h * p.c.page * dim]) * scale[(size_t)h * p.c.page]);
    }
  }
}

// ------------------------------------------------------------------------------------------ attention
struct Attn {
  Batch b;
  Cache c;
  int heads, window, q_ld, out_ld;
  float scale, softcap;
  int *error_flag;
};
}  // namespace kv8
}  // namespace pt
#include "kv8_attn.cuh"
namespace pt {
namespace kv8 {
// Any sizes (and 54 times the time of the tensor cores' on 48 sequences of up to 8000 positions): a block per token and head, whose warps take every fourth key each with a running maximum and sum, lanes across the dimensions.
constexpr int PLAIN_WARPS = 4, MOST_DIM = 256;
template <typename T, bool E4M3> __global__ void __launch_bounds__(PLAIN_WARPS * 32) attn_plain_kernel(const T *q, T *out, const Attn p) {
  early_start();
  __shared__ float top[PLAIN_WARPS], total[PLAIN_WARPS], sums[PLAIN_WARPS][MOST_DIM];
  const int tok = blockIdx.x, head = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = p.c.n_kv, g = head / (p.heads / G);
  if (tok >= p.b.cu[p.b.n_seq]) return;
  const int seq = p.b.tok_seq[tok], first = p.b.cu[seq], start = p.b.start[seq];
  if (!in_table(p.c, start, p.b.cu[seq + 1] - first)) {
    if (threadIdx.x == 0 && p.error_flag) atomicExch(p.error_flag, 12);
    return;
  }
  const int pos = start + tok - first, from = p.window > 0 ? max(0, pos - p.window + 1) : 0;
  const int *table = p.c.page_table + (size_t)p.b.slot[seq] * p.c.max_pages;
  constexpr int PER = MOST_DIM / 32;
  float x[PER], o[PER], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int d = lane + 32 * i;
    x[i] = d < p.c.dim ? to_f(q[(size_t)tok * p.q_ld + (size_t)head * p.c.dim + d]) : 0.f;
    o[i] = 0.f;
  }
  for (int j = from + warp; j <= pos; j += PLAIN_WARPS) {
    int page = table[j / p.c.page];
    if (page < 0) {
      if (lane == 0 && p.error_flag) atomicExch(p.error_flag, 12);
      page = 0;
    }
    const size_t row = (size_t)g * p.c.page + j % p.c.page, at = (size_t)page * 2 * G * p.c.page + row;
    const unsigned char *k = p.c.pool + (size_t)page * p.c.page_bytes + row * p.c.dim, *v = p.c.pool + (size_t)page * p.c.page_bytes + (size_t)G * p.c.page * p.c.dim + row * p.c.vdim;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 32 * i < p.c.dim) s = fmaf(x[i], from_byte<E4M3>(k[lane + 32 * i]), s);
    s = warp_sum(s) * (p.c.scales[at] * p.scale);
    if (p.softcap > 0.f) s = p.softcap * tanhf(s / p.softcap);
    const float t = fmaxf(m, s), was = m == t ? 1.f : expf(m - t), w = expf(s - (t == -INFINITY ? 0.f : t)), wv = w * p.c.scales[at + (size_t)G * p.c.page];
    m = t;
    l = l * was + w;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 32 * i < p.c.vdim) o[i] = o[i] * was + wv * from_byte<E4M3>(v[lane + 32 * i]);
  }
  if (lane == 0) { top[warp] = m; total[warp] = l; }
#pragma unroll
  for (int i = 0; i < PER; ++i) sums[warp][lane + 32 * i] = o[i];
  __syncthreads();
  float most = top[0], whole = 0.f, share[PLAIN_WARPS];
#pragma unroll
  for (int w = 1; w < PLAIN_WARPS; ++w) most = fmaxf(most, top[w]);
#pragma unroll
  for (int w = 0; w < PLAIN_WARPS; ++w) {
    share[w] = total[w] == 0.f ? 0.f : expf(top[w] - most);
    whole += total[w] * share[w];
  }
  for (int d = threadIdx.x; d < p.c.vdim; d += PLAIN_WARPS * 32) {
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < PLAIN_WARPS; ++w) y += total[w] == 0.f ? 0.f : sums[w][d] * share[w];
    out[(size_t)tok * p.out_ld + (size_t)head * p.c.vdim + d] = from_f<T>(y / whole);
  }
}

static int check_cache(const pt_kv8_cache &c, const char *who) {
  PT_REQUIRE(c.pool && c.scales && c.page_table, "%s: null pool, scales or page table", who);
  PT_REQUIRE(c.fmt == PT_KV8_INT8 || c.fmt == PT_KV8_E4M3, "%s: cache format %d (int8 or E4M3)", who, c.fmt);
  PT_REQUIRE(c.n_kv > 0 && c.dim > 0 && c.dim <= MOST_DIM && c.vdim > 0 && c.vdim <= MOST_DIM, "%s: n_kv=%d, heads of %d and %d (1 .. %d)", who, c.n_kv, c.dim, c.vdim, MOST_DIM);
  PT_REQUIRE(c.page_size > 0 && c.max_pages > 0 && (long long)c.page_size * c.max_pages < (1ll << 31) && c.max_len >= 0 && c.max_len <= (long long)c.page_size * c.max_pages,
             "%s: %d pages of %d positions, max_len=%d", who, c.max_pages, c.page_size, c.max_len);
  PT_REQUIRE((long long)c.n_kv * c.page_size * (c.dim + c.vdim) < (1ll << 31), "%s: a page of 2 GB or more", who);
  PT_REQUIRE(((uintptr_t)c.scales & 3) == 0, "%s: scales on a multiple of 4 bytes", who);
  return PT_OK;
}
static int check_batch(const pt_batch_view &b, const char *who) {
  PT_REQUIRE(b.n_seq > 0 && b.n_tok >= 0 && b.cu && b.start && b.slot && (b.tok_seq || b.n_tok == 0), "%s: bad batch (%d sequences, %d tokens)", who, b.n_seq, b.n_tok);
  return PT_OK;
}
static int check_rope(const float *rope, int rope_dims, int dim, const char *who) {
  PT_REQUIRE(rope_dims >= 0 && rope_dims % 2 == 0 && rope_dims <= dim, "%s: %d rotated dimensions of %d (an even number)", who, rope_dims, dim);
  PT_REQUIRE(rope_dims == 0 || (rope && aligned_to(rope, 8)), "%s: %d rotated dimensions want a table (on a multiple of 8 bytes)", who, rope_dims);
  return PT_OK;
}
// Whether rows of `width` that are read and rows of `to_width` that are written while others are still read have no element in common.
static bool apart(const void *x, long long ld, long long width, const void *to, long long to_ld, long long to_width, long long rows, int es) {
  const char *a = (const char *)x, *b = (const char *)to;
  if (rows <= 0 || a + ((rows - 1) * ld + width) * es <= b || b + ((rows - 1) * to_ld + to_width) * es <= a) return true;
  if (ld != to_ld || (b - a) % es != 0) return false;
  const long long d = (((b - a) / es) % ld + ld) % ld;      // columns of the same wider rows
  return d >= width && d + to_width <= ld;
}
static Cache cache_of(const pt_kv8_cache &c) {
  return {(unsigned char *)c.pool, c.scales, c.page_table, c.n_kv, c.dim, c.vdim, c.page_size, c.max_pages, c.max_len ? c.max_len : c.page_size * c.max_pages,
          (size_t)c.n_kv * c.page_size * (c.dim + c.vdim)};
}
static Batch batch_of(const pt_batch_view &b) { return {b.n_seq, b.n_tok, b.cu, b.start, b.slot, b.tok_seq}; }
static int elem_bytes(int dtype) { return dtype == PT_DT_F32 ? 4 : 2; }
static int lanes_of(int dim) { return dim <= 64 ? 4 : dim <= 128 ? 8 : 16; }

template <typename T, int LANES, bool WHOLE> static cudaError_t launch_rotary(const pt_rotary_args &a, const Rotary &p, dim3 grid, cudaStream_t st) {
  const T *x = (const T *)a.x;
  T *out = (T *)a.out;
  const auto kernel = a.inverse ? (a.interleaved ? rotary_kernel<T, LANES, WHOLE, true, true> : rotary_kernel<T, LANES, WHOLE, true, false>)
                                : (a.interleaved ? rotary_kernel<T, LANES, WHOLE, false, true> : rotary_kernel<T, LANES, WHOLE, false, false>);
  return launch_early(kernel, Grid(grid), THREADS, 0, st, x, out, p);
}
template <typename T> static cudaError_t launch_rotary(const pt_rotary_args &a, const Rotary &p, bool whole, cudaStream_t st) {
  const int lanes = lanes_of(a.dim);
  const dim3 grid(ceil_div(a.rows * a.heads, THREADS / lanes));
  if (lanes == 4) return whole ? launch_rotary<T, 4, true>(a, p, grid, st) : launch_rotary<T, 4, false>(a, p, grid, st);
  if (lanes == 8) return whole ? launch_rotary<T, 8, true>(a, p, grid, st) : launch_rotary<T, 8, false>(a, p, grid, st);
  return whole ? launch_rotary<T, 16, true>(a, p, grid, st) : launch_rotary<T, 16, false>(a, p, grid, st);
}

template <typename T, int LANES, int ROWS, bool WHOLE> static cudaError_t launch_append(const pt_kv8_append_args &a, Append p, cudaStream_t st) {
  p.by_q = Divide::by(std::max(1, ceil_div(p.heads, ROWS)));
  p.by_kv = Divide::by(ceil_div(p.c.n_kv, ROWS));
  p.q_blocks = p.heads ? ceil_div(a.batch.n_tok * (int)p.by_q.d, THREADS / LANES) : 0;
  p.kv_blocks = ceil_div(a.batch.n_tok * (int)p.by_kv.d, THREADS / LANES);
  const bool e4m3 = a.cache.fmt == PT_KV8_E4M3;
  const auto kernel = e4m3 ? (a.interleaved ? append_kernel<T, LANES, ROWS, WHOLE, true, true> : append_kernel<T, LANES, ROWS, WHOLE, false, true>)
                           : (a.interleaved ? append_kernel<T, LANES, ROWS, WHOLE, true, false> : append_kernel<T, LANES, ROWS, WHOLE, false, false>);
  return launch_early(kernel, Grid(p.q_blocks + 2 * p.kv_blocks), THREADS, 0, st, (const T *)a.q, (const T *)a.k, (const T *)a.v, (T *)a.q_out, p);
}
template <typename T, int LANES> static cudaError_t launch_append(const pt_kv8_append_args &a, const Append &p, bool whole, cudaStream_t st) {
  constexpr int MANY = 2;      // rows of a lane, where there are more than a wave of rows one by one (four: fewer warps, 61.6 us where two took 59.0)
  const bool many = (long long)a.batch.n_tok * (p.heads + 2 * p.c.n_kv) * LANES > 1024ll * sm_count();
  if (!whole) return launch_append<T, LANES, 1, false>(a, p, st);
  return many ? launch_append<T, LANES, MANY, true>(a, p, st) : launch_append<T, LANES, 1, true>(a, p, st);
}
template <typename T> static cudaError_t launch_append(const pt_kv8_append_args &a, const Append &p, bool whole, cudaStream_t st) {
  const int lanes = lanes_of(std::max(a.cache.dim, a.cache.vdim));
  return lanes == 4 ? launch_append<T, 4>(a, p, whole, st) : lanes == 8 ? launch_append<T, 8>(a, p, whole, st) : launch_append<T, 16>(a, p, whole, st);
}

template <typename T> static cudaError_t launch_unpack(const pt_kv8_unpack_args &a, Unpack p, bool whole, cudaStream_t st) {
  // Heads of a block: all, unless the longest histories that there may be would not fill the GPU then.
  p.rows_each = std::max(1, THREADS / std::max(1, std::min(p.c.dim, p.c.vdim) / (whole ? 16 / (int)sizeof(T) : 1)));      // (a thread has one place)
  const int chunks = ceil_div(std::min(p.c.max_len, p.into_max_len), p.rows_each);
  p.heads_each = p.c.n_kv;
  while (p.heads_each > 1 && (long long)chunks * a.batch.n_seq * 2 * ceil_div(p.c.n_kv, p.heads_each) < 8ll * sm_count()) p.heads_each = (p.heads_each + 1) / 2;
  const dim3 grid(chunks, a.batch.n_seq, 2 * ceil_div(p.c.n_kv, p.heads_each));
  const bool e4m3 = a.cache.fmt == PT_KV8_E4M3;
  const auto kernel = whole ? (e4m3 ? unpack_kernel<T, true, true> : unpack_kernel<T, true, false>) : (e4m3 ? unpack_kernel<T, false, true> : unpack_kernel<T, false, false>);
  return launch_early(kernel, Grid(grid), THREADS, 0, st, (T *)a.into, p);
}

template <typename T> static cudaError_t launch_plain(const pt_kv8_attn_args &a, const Attn &p, cudaStream_t st) {
  const auto kernel = a.cache.fmt == PT_KV8_E4M3 ? attn_plain_kernel<T, true> : attn_plain_kernel<T, false>;
  return launch_early(kernel, Grid(dim3(a.batch.n_tok, a.n_head)), PLAIN_WARPS * 32, 0, st, (const T *)a.q, (T *)a.out, p);
}
// A workspace: counters, then (by the width of the heads) pieces of every block.
static size_t workspace_bytes(int width) {
  const size_t pieces = width > 128 ? (Shape<256>::WARPS + 2) * Shape<256>::PIECE : width > 64 ? (Shape<128>::WARPS + 2) * Shape<128>::PIECE : (Shape<64>::WARPS + 2) * Shape<64>::PIECE;
  return sizeof(int) * COUNTERS + sizeof(float) * sm_count() * pieces;
}
template <int SIZE, bool FULL> static cudaError_t launch_attn(const pt_kv8_attn_args &a, const Attn &p, const Split &sp, cudaStream_t st) {
  const bool e4m3 = a.cache.fmt == PT_KV8_E4M3, wide = a.dtype != PT_DT_BF16;      // (weights in two fp16 parts: one would double the error of an fp16 output)
  const auto kernel = e4m3 ? (wide ? attn_kernel<SIZE, FULL, true, 2> : attn_kernel<SIZE, FULL, true, 1>) : (wide ? attn_kernel<SIZE, FULL, false, 2> : attn_kernel<SIZE, FULL, false, 1>);
  static std::atomic<uint64_t> allowed[4];
  constexpr int WARPS = Shape<SIZE>::WARPS, FIXED = WARPS * Shape<SIZE>::RING;
  const cudaError_t e = allow_smem(kernel, FIXED + (3 * MAX_TOKENS + 1) * (int)sizeof(int), allowed[2 * e4m3 + wide]);
  if (e != cudaSuccess) return e;
  return launch_early(kernel, Grid(sp.grid), WARPS * 32, FIXED + (3 * sp.tokens + 1) * sizeof(int), st, p, sp);
}
template <int SIZE> static cudaError_t launch_attn(const pt_kv8_attn_args &a, const Attn &p, Split sp, cudaStream_t st) {
  sp.parts = sp.heads + (size_t)sp.grid * Shape<SIZE>::WARPS * Shape<SIZE>::PIECE;
  return p.c.dim == SIZE && p.c.vdim == SIZE ? launch_attn<SIZE, true>(a, p, sp, st) : launch_attn<SIZE, false>(a, p, sp, st);
}

}  // namespace kv8
}  // namespace pt

using namespace pt;

extern "C" int pt_rotary(const pt_rotary_args *a, void *stream) {
  PT_REQUIRE(a, "pt_rotary: null args");
  PT_REQUIRE(a->dtype == PT_DT_F16 || a->dtype == PT_DT_BF16 || a->dtype == PT_DT_F32, "pt_rotary: type %d", a->dtype);
  PT_REQUIRE(a->rows >= 0 && a->heads > 0 && a->heads <= 65535 && a->dim > 0 && a->dim <= kv8::MOST_DIM, "pt_rotary: %d rows of %d heads of %d (heads of 1 .. %d)", a->rows, a->heads, a->dim,
             kv8::MOST_DIM);
  if (a->rows == 0) return PT_OK;
  PT_REQUIRE(a->x && a->out && a->position, "pt_rotary: null pointer argument");
  PT_REQUIRE(a->x_ld >= (long long)a->heads * a->dim && a->out_ld >= (long long)a->heads * a->dim, "pt_rotary: rows of %d and %d elements, %d heads of %d", a->x_ld, a->out_ld, a->heads, a->dim);
  const int es = kv8::elem_bytes(a->dtype);
  const long long width = (long long)a->heads * a->dim;
  PT_REQUIRE((a->x == a->out && a->x_ld == a->out_ld) || kv8::apart(a->x, a->x_ld, width, a->out, a->out_ld, width, a->rows, es), "pt_rotary: out is x itself (with its stride, %d, not %d) or apart from it",
             a->x_ld, a->out_ld);
  PT_REQUIRE(a->positions > 0 && a->rope_dims > 0, "pt_rotary: %d rotated dimensions, a table of %d positions", a->rope_dims, a->positions);
  if (int rc = kv8::check_rope(a->rope, a->rope_dims, a->dim, "pt_rotary")) return rc;
  PT_REQUIRE((long long)a->rows * a->heads < (1ll << 30), "pt_rotary: %d rows of %d heads", a->rows, a->heads);
  const bool whole = a->dim % 16 == 0 && a->rope_dims % 16 == 0 && aligned_to(a->rope, 16) && aligned_to(a->x, 16) && aligned_to(a->out, 16) && (long long)a->x_ld * es % 16 == 0 && (long long)a->out_ld * es % 16 == 0;
  const kv8::Rotary p{a->rows, a->heads, a->dim, a->rope_dims, a->x_ld, a->out_ld, a->positions, a->position, (const float2 *)a->rope, a->error_flag, kv8::Divide::by(a->heads)};
  const cudaStream_t st = as_stream(stream);
  PT_CUDA(a->dtype == PT_DT_F32   ? kv8::launch_rotary<float>(*a, p, whole, st)
          : a->dtype == PT_DT_F16 ? kv8::launch_rotary<__half>(*a, p, whole, st)
                                  : kv8::launch_rotary<__nv_bfloat16>(*a, p, whole, st));
  PT_LAUNCH_CHECK("pt_rotary");
  return PT_OK;
}

extern "C" int pt_kv8_append(const pt_kv8_append_args *a, void *stream) {
  PT_REQUIRE(a, "pt_kv8_append: null args");
  PT_REQUIRE(a->dtype == PT_DT_F16 || a->dtype == PT_DT_BF16 || a->dtype == PT_DT_F32, "pt_kv8_append: type %d", a->dtype);
  if (int rc = kv8::check_batch(a->batch, "pt_kv8_append")) return rc;
  if (int rc = kv8::check_cache(a->cache, "pt_kv8_append")) return rc;
  if (a->batch.n_tok == 0) return PT_OK;       // (tensors without elements have no address)
  PT_REQUIRE(a->k && a->v && a->ld > 0, "pt_kv8_append: null pointer argument, or rows of %d elements", a->ld);
  PT_REQUIRE(!a->q_out || (a->q && a->n_head > 0 && a->q_out_ld >= (long long)a->n_head * a->cache.dim), "pt_kv8_append: q_out wants q and rows of %d heads of %d, got %d elements", a->n_head,
             a->cache.dim, a->q_out_ld);
  const int es = kv8::elem_bytes(a->dtype);
  if (a->q_out) {
    const long long n = a->batch.n_tok, width = (long long)a->n_head * a->cache.dim, kv = a->cache.n_kv;
    PT_REQUIRE(((a->q == a->q_out && a->ld == a->q_out_ld) || kv8::apart(a->q, a->ld, width, a->q_out, a->q_out_ld, width, n, es)) &&
                   kv8::apart(a->k, a->ld, kv * a->cache.dim, a->q_out, a->q_out_ld, width, n, es) && kv8::apart(a->v, a->ld, kv * a->cache.vdim, a->q_out, a->q_out_ld, width, n, es),
               "pt_kv8_append: q_out is q itself (with its stride, %d, not %d) or apart from the rows", a->ld, a->q_out_ld);
  }
  if (int rc = kv8::check_rope(a->rope, a->rope_dims, a->cache.dim, "pt_kv8_append")) return rc;
  PT_REQUIRE((long long)a->batch.n_tok * ((a->q_out ? a->n_head : 0) + 2ll * a->cache.n_kv) < (1ll << 30), "pt_kv8_append: %d tokens of %d and %d heads", a->batch.n_tok, a->n_head,
             a->cache.n_kv);
  const kv8::Append p{kv8::batch_of(a->batch), kv8::cache_of(a->cache), a->q_out ? a->n_head : 0, a->rope_dims, a->ld, a->q_out_ld, (const float2 *)a->rope, a->error_flag,
                      kv8::Divide::by(a->cache.page_size), {}, {}, 0, 0};
  const bool whole = a->cache.dim % 16 == 0 && a->cache.vdim % 16 == 0 && a->rope_dims % 16 == 0 && aligned_to(a->rope, 16) && aligned_to(a->cache.pool, 16) && aligned_to(a->k, 16) && aligned_to(a->v, 16) &&
                     (long long)a->ld * es % 16 == 0 && (!a->q_out || (aligned_to(a->q, 16) && aligned_to(a->q_out, 16) && (long long)a->q_out_ld * es % 16 == 0));
  const cudaStream_t st = as_stream(stream);
  PT_CUDA(a->dtype == PT_DT_F32   ? kv8::launch_append<float>(*a, p, whole, st)
          : a->dtype == PT_DT_F16 ? kv8::launch_append<__half>(*a, p, whole, st)
                                  : kv8::launch_append<__nv_bfloat16>(*a, p, whole, st));
  PT_LAUNCH_CHECK("pt_kv8_append");
  return PT_OK;
}

extern "C" int pt_kv8_unpack(const pt_kv8_unpack_args *a, void *stream) {
  PT_REQUIRE(a, "pt_kv8_unpack: null args");
  PT_REQUIRE(a->dtype == PT_DT_F16 || a->dtype == PT_DT_BF16 || a->dtype == PT_DT_F32, "pt_kv8_unpack: type %d", a->dtype);
  if (int rc = kv8::check_batch(a->batch, "pt_kv8_unpack")) return rc;
  if (int rc = kv8::check_cache(a->cache, "pt_kv8_unpack")) return rc;
  PT_REQUIRE(a->into && a->into_table && a->into_page_size > 0 && a->into_max_pages > 0 && (long long)a->into_page_size * a->into_max_pages < (1ll << 31),
             "pt_kv8_unpack: null pointer argument, or %d pages of %d positions", a->into_max_pages, a->into_page_size);
  PT_REQUIRE(a->into_max_len >= 0 && a->into_max_len <= (long long)a->into_page_size * a->into_max_pages, "pt_kv8_unpack: %d pages of %d positions, max_len=%d", a->into_max_pages,
             a->into_page_size, a->into_max_len);
  PT_REQUIRE(a->batch.n_seq <= 65535 && a->cache.n_kv <= 32767, "pt_kv8_unpack: %d sequences (65535 at most), %d heads (32767)", a->batch.n_seq, a->cache.n_kv);
  const kv8::Unpack p{kv8::batch_of(a->batch), kv8::cache_of(a->cache), a->into_table, a->into_page_size, a->into_max_pages,
                      a->into_max_len ? a->into_max_len : a->into_page_size * a->into_max_pages, 1, 1, a->error_flag, kv8::Divide::by(a->cache.page_size), kv8::Divide::by(a->into_page_size)};
  const bool whole = a->cache.dim % 16 == 0 && a->cache.vdim % 16 == 0 && aligned_to(a->cache.pool, 16) && aligned_to(a->into, 16);
  const cudaStream_t st = as_stream(stream);
  PT_CUDA(a->dtype == PT_DT_F32   ? kv8::launch_unpack<float>(*a, p, whole, st)
          : a->dtype == PT_DT_F16 ? kv8::launch_unpack<__half>(*a, p, whole, st)
                                  : kv8::launch_unpack<__nv_bfloat16>(*a, p, whole, st));
  PT_LAUNCH_CHECK("pt_kv8_unpack");
  return PT_OK;
}

extern "C" size_t pt_kv8_attn_workspace_bytes(int n_tok, int n_head, int n_kv, int width) { return n_tok < 1 || n_kv < 1 || n_head < n_kv ? 0 : kv8::workspace_bytes(width); }

extern "C" int pt_kv8_attn(const pt_kv8_attn_args *a, void *stream) {
  PT_REQUIRE(a, "pt_kv8_attn: null args");
  PT_REQUIRE(a->dtype == PT_DT_F16 || a->dtype == PT_DT_BF16 || a->dtype == PT_DT_F32, "pt_kv8_attn: type %d", a->dtype);
  if (int rc = kv8::check_batch(a->batch, "pt_kv8_attn")) return rc;
  if (int rc = kv8::check_cache(a->cache, "pt_kv8_attn")) return rc;
  if (a->batch.n_tok == 0) return PT_OK;
  PT_REQUIRE(a->q && a->out, "pt_kv8_attn: null pointer argument");
  PT_REQUIRE(a->n_head > 0 && a->n_head <= 65535 && a->n_head % a->cache.n_kv == 0, "pt_kv8_attn: %d heads over %d", a->n_head, a->cache.n_kv);
  PT_REQUIRE(a->q_ld >= (long long)a->n_head * a->cache.dim && a->out_ld >= (long long)a->n_head * a->cache.vdim, "pt_kv8_attn: rows of %d and %d elements, %d heads of %d and %d", a->q_ld,
             a->out_ld, a->n_head, a->cache.dim, a->cache.vdim);
  const int es = kv8::elem_bytes(a->dtype);
  PT_REQUIRE((a->q == a->out && a->q_ld == a->out_ld && a->cache.dim == a->cache.vdim) || kv8::apart(a->q, a->q_ld, (long long)a->n_head * a->cache.dim, a->out, a->out_ld, (long long)a->n_head * a->cache.vdim,
                                                                                                      a->batch.n_tok, es),
             "pt_kv8_attn: out is q itself (with its stride and width) or apart from it");
  PT_REQUIRE(a->window >= 0, "pt_kv8_attn: window=%d", a->window);
  PT_REQUIRE(a->softcap == 0.f || (a->softcap >= 1e-20f && a->softcap <= 1e20f), "pt_kv8_attn: softcap=%g (0, or 1e-20 .. 1e20)", (double)a->softcap);
  PT_REQUIRE(a->scale - a->scale == 0.f, "pt_kv8_attn: scale=%g", (double)a->scale);
  const kv8::Attn p{kv8::batch_of(a->batch), kv8::cache_of(a->cache), a->n_head, a->window, a->q_ld, a->out_ld, a->scale, a->softcap, a->error_flag};
  const cudaStream_t st = as_stream(stream);
  const int width = std::max(a->cache.dim, a->cache.vdim);
  // (16 bytes of a row a lane, 16 positions of a page a group)
  if (a->plain || a->cache.dim % 16 || a->cache.vdim % 16 || a->cache.page_size % 16 || !aligned_to(a->cache.pool, 16)) {
    PT_CUDA(a->dtype == PT_DT_F32   ? kv8::launch_plain<float>(*a, p, st)
            : a->dtype == PT_DT_F16 ? kv8::launch_plain<__half>(*a, p, st)
                                    : kv8::launch_plain<__nv_bfloat16>(*a, p, st));
    PT_LAUNCH_CHECK("pt_kv8_attn");
    return PT_OK;
  }
  const size_t need = pt_kv8_attn_workspace_bytes(a->batch.n_tok, a->n_head, a->cache.n_kv, width);
  PT_REQUIRE(a->workspace && aligned_to(a->workspace, 16) && a->workspace_bytes >= need, "pt_kv8_attn: %zu workspace bytes (on a multiple of 16) are wanted, got %zu", need,
             a->workspace ? a->workspace_bytes : 0);
  kv8::Split sp{};
  sp.chunks = ceil_div(a->n_head / a->cache.n_kv, kv8::HEADS);
  sp.dtype = a->dtype;
  sp.q_whole = aligned_to(a->q, 16) && (long long)a->q_ld * es % 16 == 0;
  sp.out_whole = aligned_to(a->out, 16) && (long long)a->out_ld * es % 16 == 0;
  sp.counters = (int *)a->workspace;
  sp.heads = (float *)(sp.counters + kv8::COUNTERS);
  sp.q = a->q;
  sp.out = a->out;
  sp.grid = sm_count();
  sp.segs = a->cache.n_kv * sp.chunks;
  sp.by_segs = kv8::Divide::by(sp.segs);
  sp.by_chunks = kv8::Divide::by(sp.chunks);
  sp.by_page = kv8::Divide::by(p.c.page);
  sp.by_grid = kv8::Divide::by(sp.grid);
  // Tokens of a launch: what its blocks plan in shared memory, a counter for every segment, and tiles that an int counts.
  const long long segs = (long long)a->cache.n_kv * sp.chunks, tiles = segs * (ceil_div(p.c.max_len, 16) + 1);
  PT_REQUIRE(tiles < 1ll << 30, "pt_kv8_attn: %lld heads of a history of %d positions", segs, p.c.max_len);
  const int most = (int)std::min<long long>({kv8::MAX_TOKENS, kv8::COUNTERS / segs, (1ll << 30) / tiles});
  for (; sp.tok0 < a->batch.n_tok; sp.tok0 += most) {
    sp.tokens = std::min(a->batch.n_tok - sp.tok0, most);
    PT_CUDA(width > 128 ? kv8::launch_attn<256>(*a, p, sp, st) : width > 64 ? kv8::launch_attn<128>(*a, p, sp, st) : kv8::launch_attn<64>(*a, p, sp, st));
    PT_LAUNCH_CHECK("pt_kv8_attn");
  }
  return PT_OK;
}
