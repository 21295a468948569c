// Filling and emptying caches of eight bits (kv8.cuh): rotation of rows, appending, pages back in a wider type.
#include "kv8.cuh"

namespace pt {
namespace kv8 {

constexpr int THREADS = 256;
constexpr float SMALL = 0x1p-64f, LARGE = 0x1p64f;

template <bool E4M3> __device__ __forceinline__ float top_byte() { return E4M3 ? 448.f : 127.f; }
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
// through its heads in turn with the angles in registers, 16.1).  Rotated parts, heads or addresses that are no multiples of 16 go element by element: 4000 rows of 34 heads of 80, 20 of each turned, 55 us
// (neighbours 62) for 6.7 of bytes.
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
// faster: a token 2.4 us.  Element by element (as in the rotation; heads of 80, 20 of each turned) 204 us for 23 of bytes; heads of 80 that turn whole 40.
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
// Blocks are launched for what the tables can hold: 8 sequences of 700 positions 6.2 us, in tables of 131072 136.
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
