// Rotation of rows by their positions, a lane at a time: what the rotation and appending kernels share.
//
// A lane has eight pairs of a row: pairs 8 t .. 8 t + 7 of item t.  Pair p < rot / 2 is elements (p, p + rot / 2), or (2 p, 2 p + 1) where neighbours
// turn together; behind the rotated part it is (2 p, 2 p + 1).  So a lane holds both elements of each of its pairs (a row can be rotated where it lies), and
// sixteen elements that are one run of 16 or two runs of 8.
#pragma once
#include "elem.cuh"

namespace pt {

__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

struct Pairs { float a[8], b[8]; };
// What a lane reads of a row, as it lies there (two runs of eight): asked for before it is known how far the row turns.
template <typename T> struct Runs { uint4 v[sizeof(T) / 2 * 2]; };

// Eight values that lie together, from or to a multiple of 16 bytes.
__device__ __forceinline__ void load_run(const float *p, float (&v)[8]) {
  const float4 x = reinterpret_cast<const float4 *>(p)[0], y = reinterpret_cast<const float4 *>(p)[1];
  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
}
template <typename T> __device__ __forceinline__ void load_run(const T *p, float (&v)[8]) {
  const uint4 r = *reinterpret_cast<const uint4 *>(p);
  T h[8];
  *reinterpret_cast<uint4 *>(h) = r;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = to_f(h[j]);
}
__device__ __forceinline__ void store_run(float *p, const float (&v)[8]) {
  reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
template <typename T> __device__ __forceinline__ void store_run(T *p, const float (&v)[8]) {
  __align__(16) T h[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) h[j] = from_f<T>(v[j]);
  *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(h);
}

// Elements of pair p of a row.
__device__ __forceinline__ int2 pair_at(int p, int rot, bool neighbours) { return p < rot / 2 && !neighbours ? make_int2(p, p + rot / 2) : make_int2(2 * p, 2 * p + 1); }

// Of rows that lie on multiples of 16 bytes, with dim and rot multiples of 16: every item is two whole runs, rot / 2 apart or one behind the other.
template <typename T> __device__ __forceinline__ Runs<T> load_runs(const T *x, int t, int rot, bool neighbours) {
  constexpr int N = sizeof(T) / 2;
  const bool apart = !neighbours && 16 * t < rot;
  const uint4 *lo = reinterpret_cast<const uint4 *>(x + (apart ? 8 * t : 16 * t)), *hi = reinterpret_cast<const uint4 *>(x + (apart ? 8 * t + rot / 2 : 16 * t + 8));
  Runs<T> r;
#pragma unroll
  for (int i = 0; i < N; ++i) { r.v[i] = lo[i]; r.v[N + i] = hi[i]; }
  return r;
}
template <typename T> __device__ __forceinline__ Pairs pairs_of(const Runs<T> &r, int t, int rot, bool neighbours) {
  const bool apart = !neighbours && 16 * t < rot;
  T e[16];
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) reinterpret_cast<uint4 *>(e)[i] = r.v[i];
  Pairs v;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v.a[j] = to_f(apart ? e[j] : e[2 * j]);
    v.b[j] = to_f(apart ? e[8 + j] : e[2 * j + 1]);
  }
  return v;
}
// Of any rows.
template <typename T> __device__ __forceinline__ Pairs load_pairs(const T *x, int t, int dim, int rot, bool neighbours) {
  Pairs v;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int2 e = pair_at(8 * t + j, rot, neighbours);
    v.a[j] = e.x < dim ? to_f(x[e.x]) : 0.f;
    v.b[j] = e.y < dim ? to_f(x[e.y]) : 0.f;
  }
  return v;
}
// WHOLE: as load_runs wants them.
template <bool WHOLE, typename T> __device__ __forceinline__ void store_pairs(T *x, const Pairs &v, int t, int dim, int rot, bool neighbours) {
  if constexpr (WHOLE) {
    const bool apart = !neighbours && 16 * t < rot;
    float lo[8], hi[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lo[j] = apart ? v.a[j] : j & 1 ? v.b[j >> 1] : v.a[j >> 1];
      hi[j] = apart ? v.b[j] : j & 1 ? v.b[4 + (j >> 1)] : v.a[4 + (j >> 1)];
    }
    store_run(x + (apart ? 8 * t : 16 * t), lo);
    store_run(x + (apart ? 8 * t + rot / 2 : 16 * t + 8), hi);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int2 e = pair_at(8 * t + j, rot, neighbours);
      if (e.x < dim) x[e.x] = from_f<T>(v.a[j]);
      if (e.y < dim) x[e.y] = from_f<T>(v.b[j]);
    }
  }
}

// (cos, sin) of an item's pairs; (1, 0) behind the rotated part.  WHOLE: a row of the table lies on a multiple of 16 bytes, and an item is rotated as a whole or not at all.
struct Turn { float c[8], s[8]; };
template <bool WHOLE> __device__ __forceinline__ Turn load_turn(const float2 *row, int t, int rot, bool inverse) {
  Turn r;
  if constexpr (WHOLE) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 cs = 16 * t < rot ? __ldg(reinterpret_cast<const float4 *>(row + 8 * t) + j) : make_float4(1.f, 0.f, 1.f, 0.f);
      r.c[2 * j] = cs.x; r.c[2 * j + 1] = cs.z;
      r.s[2 * j] = inverse ? -cs.y : cs.y; r.s[2 * j + 1] = inverse ? -cs.w : cs.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 cs = 8 * t + j < rot / 2 ? __ldg(row + 8 * t + j) : make_float2(1.f, 0.f);
      r.c[j] = cs.x;
      r.s[j] = inverse ? -cs.y : cs.y;
    }
  }
  return r;
}
// Three roundings, as written: what is cached does not depend on which products a compiler joins.
__device__ __forceinline__ void turn_pairs(Pairs &v, const Turn &r, int t, int rot) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (8 * t + j >= rot / 2) continue;
    const float x = v.a[j], y = v.b[j];
    v.a[j] = __fsub_rn(__fmul_rn(x, r.c[j]), __fmul_rn(y, r.s[j]));
    v.b[j] = __fadd_rn(__fmul_rn(y, r.c[j]), __fmul_rn(x, r.s[j]));
  }
}

}  // namespace pt
