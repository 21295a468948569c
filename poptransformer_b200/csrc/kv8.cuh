// Paged caches of eight bits: keys and values as bytes (int8 or E4M3), with a scale for every position and head.
//   pool[page] = K [n_kv][page_size][dim] and then V [n_kv][page_size][vdim], a byte each; scales[page] = fp32 [2][n_kv][page_size], K's and then V's.
// A row x of one position and head is kept as  byte_i = round(x_i (top / m)),  scale = m / top,  m = max_i |x_i|  (top: 127 or 448).  m is at least 2^-64, so that
// top / m is finite; a row that has a NaN, an infinity or a magnitude above 2^64 gets the scale NaN and bytes of 0, and reads back as NaN.
#pragma once
#include <type_traits>

#include "rotate.cuh"

namespace pt {
namespace kv8 {

constexpr int MOST_DIM = 256;

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

template <bool E4M3> __device__ __forceinline__ float from_byte(unsigned char b) {
  if constexpr (E4M3) {
    __nv_fp8_e4m3 x;
    x.__x = b;
    return float(x);
  }
  return (float)(signed char)b;
}
// Whether a sequence's new positions can be there.
__device__ __forceinline__ bool in_table(const Cache &c, int start, int count) { return start >= 0 && count <= c.max_len - start; }

inline int check_cache(const pt_kv8_cache &c, const char *who) {
  PT_REQUIRE(c.pool && c.scales && c.page_table, "%s: null pool, scales or page table", who);
  PT_REQUIRE(c.fmt == PT_KV8_INT8 || c.fmt == PT_KV8_E4M3, "%s: cache format %d (int8 or E4M3)", who, c.fmt);
  PT_REQUIRE(c.n_kv > 0 && c.dim > 0 && c.dim <= MOST_DIM && c.vdim > 0 && c.vdim <= MOST_DIM, "%s: n_kv=%d, heads of %d and %d (1 .. %d)", who, c.n_kv, c.dim, c.vdim, MOST_DIM);
  PT_REQUIRE(c.page_size > 0 && c.max_pages > 0 && (long long)c.page_size * c.max_pages < (1ll << 31) && c.max_len >= 0 && c.max_len <= (long long)c.page_size * c.max_pages,
             "%s: %d pages of %d positions, max_len=%d", who, c.max_pages, c.page_size, c.max_len);
  PT_REQUIRE((long long)c.n_kv * c.page_size * (c.dim + c.vdim) < (1ll << 31), "%s: a page of 2 GB or more", who);
  PT_REQUIRE(((uintptr_t)c.scales & 3) == 0, "%s: scales on a multiple of 4 bytes", who);
  return PT_OK;
}
inline int check_batch(const pt_batch_view &b, const char *who) {
  PT_REQUIRE(b.n_seq > 0 && b.n_tok >= 0 && b.cu && b.start && b.slot && (b.tok_seq || b.n_tok == 0), "%s: bad batch (%d sequences, %d tokens)", who, b.n_seq, b.n_tok);
  return PT_OK;
}
inline int check_rope(const float *rope, int rope_dims, int dim, const char *who) {
  PT_REQUIRE(rope_dims >= 0 && rope_dims % 2 == 0 && rope_dims <= dim, "%s: %d rotated dimensions of %d (an even number)", who, rope_dims, dim);
  PT_REQUIRE(rope_dims == 0 || (rope && aligned_to(rope, 8)), "%s: %d rotated dimensions want a table (on a multiple of 8 bytes)", who, rope_dims);
  return PT_OK;
}
// Whether rows of `width` that are read and rows of `to_width` that are written while others are still read have no element in common.
inline bool apart(const void *x, long long ld, long long width, const void *to, long long to_ld, long long to_width, long long rows, int es) {
  const char *a = (const char *)x, *b = (const char *)to;
  if (rows <= 0 || a + ((rows - 1) * ld + width) * es <= b || b + ((rows - 1) * to_ld + to_width) * es <= a) return true;
  if (ld != to_ld || (b - a) % es != 0) return false;
  const long long d = (((b - a) / es) % ld + ld) % ld;      // columns of the same wider rows
  return d >= width && d + to_width <= ld;
}
inline Cache cache_of(const pt_kv8_cache &c) {
  return {(unsigned char *)c.pool, c.scales, c.page_table, c.n_kv, c.dim, c.vdim, c.page_size, c.max_pages, c.max_len ? c.max_len : c.page_size * c.max_pages,
          (size_t)c.n_kv * c.page_size * (c.dim + c.vdim)};
}
inline Batch batch_of(const pt_batch_view &b) { return {b.n_seq, b.n_tok, b.cu, b.start, b.slot, b.tok_seq}; }
inline int elem_bytes(int dtype) { return dtype == PT_DT_F32 ? 4 : 2; }

}  // namespace kv8
}  // namespace pt
