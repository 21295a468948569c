// Rotation of rows by their positions, a lane at a time: what the rotation, appending and rounding kernels share.
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

// WHOLE: rows lie on multiples of 16 bytes, dim is a multiple of 16, and so is rot: every item is two whole runs.  apart: the runs are rot / 2 apart.
template <bool WHOLE, typename T> __device__ __forceinline__ Pairs load_pairs(const T *x, int t, int dim, int rot, bool neighbours) {
  Pairs v;
  if constexpr (WHOLE) {
    const bool apart = !neighbours && 16 * t < rot;
    float lo[8], hi[8];
    load_run(x + (apart ? 8 * t : 16 * t), lo);
    load_run(x + (apart ? 8 * t + rot / 2 : 16 * t + 8), hi);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v.a[j] = apart ? lo[j] : j < 4 ? lo[2 * (j & 3)] : hi[2 * (j & 3)];
      v.b[j] = apart ? hi[j] : j < 4 ? lo[2 * (j & 3) + 1] : hi[2 * (j & 3) + 1];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int2 e = pair_at(8 * t + j, rot, neighbours);
      v.a[j] = e.x < dim ? to_f(x[e.x]) : 0.f;
      v.b[j] = e.y < dim ? to_f(x[e.y]) : 0.f;
    }
  }
  return v;
}
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

// (cos, sin) of an item's pairs; (1, 0) behind the rotated part.
struct Turn { float c[8], s[8]; };
__device__ __forceinline__ Turn load_turn(const float2 *row, int t, int rot, bool inverse) {
  Turn r;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float2 cs = 8 * t + j < rot / 2 ? __ldg(row + 8 * t + j) : make_float2(1.f, 0.f);
    r.c[j] = cs.x;
    r.s[j] = inverse ? -cs.y : cs.y;
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
