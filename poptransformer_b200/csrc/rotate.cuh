// Rotation of rows by their positions, a lane at a time: what the rotation and appending kernels share.
//
// Pair p < rot / 2 of a row is elements (p, p + rot / 2), or (2 p, 2 p + 1) where neighbours turn together.  A lane has sixteen elements, both of every pair that it has any of, so
// that a row can be rotated where it lies.
#pragma once
#include "elem.cuh"

namespace pt {

__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// Eight values that lie together, to a multiple of 16 bytes.
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

// Three roundings, as written: what is cached does not depend on which products a compiler joins.
__device__ __forceinline__ void turn(float &x, float &y, float c, float s) {
  const float a = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
  y = __fadd_rn(__fmul_rn(y, c), __fmul_rn(x, s));
  x = a;
}

// ---- rows on multiples of 16 bytes, dim and rot multiples of 16: lane t has two runs of eight, and neighbouring lanes neighbouring runs
struct Item { float lo[8], hi[8]; };
struct Runs { int lo, hi; bool turns_lo, turns_hi; };
__device__ __forceinline__ Runs runs_of(int t, int dim, int rot, bool neighbours) {
  if (neighbours) return {8 * t, 8 * t + dim / 2, 8 * t < rot, 8 * t + dim / 2 < rot};
  if (16 * t < rot) return {8 * t, 8 * t + rot / 2, true, true};
  return {rot / 2 + 8 * t, rot / 2 + 8 * t + (dim - rot) / 2, false, false};      // (behind the rotated part, from element rot on)
}
// As they lie there: asked for before it is known how far the row turns.
template <typename T> struct Raw { uint4 v[sizeof(T)]; };
template <typename T> __device__ __forceinline__ Raw<T> load_raw(const T *x, const Runs &r) {
  constexpr int N = sizeof(T) / 2;
  Raw<T> w;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    w.v[i] = reinterpret_cast<const uint4 *>(x + r.lo)[i];
    w.v[N + i] = reinterpret_cast<const uint4 *>(x + r.hi)[i];
  }
  return w;
}
template <typename T> __device__ __forceinline__ Item item_of(const Raw<T> &w) {
  T e[16];
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) reinterpret_cast<uint4 *>(e)[i] = w.v[i];
  Item v;
#pragma unroll
  for (int j = 0; j < 8; ++j) { v.lo[j] = to_f(e[j]); v.hi[j] = to_f(e[8 + j]); }
  return v;
}
// (cos, sin) of a lane's pairs; row: those of the position, on a multiple of 16 bytes.
struct Angles { float4 v[4]; };
__device__ __forceinline__ Angles load_angles(const float2 *row, const Runs &r, bool neighbours) {
  const float4 *cs = reinterpret_cast<const float4 *>(row);
  Angles a{};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (neighbours ? (j < 2 ? r.turns_lo : r.turns_hi) : r.turns_lo) a.v[j] = __ldg(cs + (neighbours ? (j < 2 ? r.lo / 4 + j : r.hi / 4 + j - 2) : r.lo / 2 + j));
  }
  return a;
}
__device__ __forceinline__ void turn_item(Item &v, const Angles &a, const Runs &r, bool neighbours, float sign) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float4 cs = make_float4(a.v[j].x, sign * a.v[j].y, a.v[j].z, sign * a.v[j].w);
    if (neighbours) {
      float(&run)[8] = j < 2 ? v.lo : v.hi;
      if (j < 2 ? r.turns_lo : r.turns_hi) {
        turn(run[4 * (j & 1)], run[4 * (j & 1) + 1], cs.x, cs.y);
        turn(run[4 * (j & 1) + 2], run[4 * (j & 1) + 3], cs.z, cs.w);
      }
    } else if (r.turns_lo) {
      turn(v.lo[2 * j], v.hi[2 * j], cs.x, cs.y);
      turn(v.lo[2 * j + 1], v.hi[2 * j + 1], cs.z, cs.w);
    }
  }
}

// ---- any rows: lane t has pairs 8 t .. 8 t + 7, those behind the rotated part being (2 p, 2 p + 1)
__device__ __forceinline__ int2 pair_at(int p, int rot, bool neighbours) { return p < rot / 2 && !neighbours ? make_int2(p, p + rot / 2) : make_int2(2 * p, 2 * p + 1); }
template <typename T> __device__ __forceinline__ Item load_pairs(const T *x, int t, int dim, int rot, bool neighbours) {
  Item v;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int2 e = pair_at(8 * t + j, rot, neighbours);
    v.lo[j] = e.x < dim ? to_f(x[e.x]) : 0.f;
    v.hi[j] = e.y < dim ? to_f(x[e.y]) : 0.f;
  }
  return v;
}
template <typename T> __device__ __forceinline__ void store_pairs(T *x, const Item &v, int t, int dim, int rot, bool neighbours) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int2 e = pair_at(8 * t + j, rot, neighbours);
    if (e.x < dim) x[e.x] = from_f<T>(v.lo[j]);
    if (e.y < dim) x[e.y] = from_f<T>(v.hi[j]);
  }
}
__device__ __forceinline__ void turn_pairs(Item &v, const float2 *row, int t, int rot, float sign) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (8 * t + j < rot / 2) {
      const float2 cs = __ldg(row + 8 * t + j);
      turn(v.lo[j], v.hi[j], cs.x, sign * cs.y);
    }
}

}  // namespace pt
