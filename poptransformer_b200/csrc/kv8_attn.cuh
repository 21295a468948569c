// Attention of new tokens over a cache of eight bits, on tensor cores (included by kv8.cu).
//
// A segment is one token, one kv head and up to eight of its query heads; its keys are tiles of KT positions.  All tiles of a launch lie in one row, segment
// after segment; every block takes an equal run of them, and every warp an equal run of its block's, so that unequal histories cost nobody a wait and warps meet
// once, at their end.  A segment that lies in one warp's run leaves from there; the pieces of others are added up by the block that has all of them, or by the last of the blocks that
// have some to come (in the order of the pieces, so that the sum does not depend on who was last).
//   scores [16 keys x 8 heads] = K . q^T,   out^T [16 dims x 8 heads] += V^T . W^T      (mma m16n8k16, fp16 operands, fp32 sums)
// A lane copies to shared memory (cp.async) exactly what it reads back, so the ring of a warp needs no barrier and no swizzle: 16 bytes of two key rows (row of the fragment), 16
// bytes of four value rows (its keys).  Which dimension of the head is which k of an instruction does not matter as long as K and q agree: a lane's k are the dimensions of
// its bytes.  Bytes become fp16 exactly: int8 b as (1024 + 128 + b) - 1152, E4M3 by its bits (times 2^-8, which the scales take back).
//
// Numbers.  q comes in fp16 times a power of two that brings its row's largest element to [1, 2): what is lost lies below 2^-25 of that; queries of 32 bits have a second fp16 part.
// With x = score log2(e), v_j = bytes times vs_j, and e_j about log2 vs_j, a segment keeps R = max (x_j + e_j), l = sum 2^(x_j - R + 14) in 32 bits, and sums
// w_j (bytes of v_j) with w_j = 2^(x_j - R + 14) vs_j, below 2^15: rounded to fp16 once (2^-11; two parts for rows of 32 bits), whole down to 2^-29 of the largest and then off by
// 2^-40 of it, however far the scales of the values lie apart.
#pragma once
#include <type_traits>

#include "tile_math.cuh"

namespace pt {
namespace kv8 {

constexpr int HEADS = 8, MAX_TOKENS = 1024;
constexpr int COUNTERS = 1 << 16;      // of a workspace, always in front: whichever calls share one, nothing else is written there

// SIZE: the widest head, 64, 128 or 256.
template <int SIZE> struct Shape {
  static constexpr int WARPS = SIZE == 256 ? 8 : 12;    // one block to an SM: 168 registers a thread (254), 16.5 KB of shared memory a warp
  static constexpr int KT = SIZE == 256 ? 16 : 32, GROUPS = KT / 16, STAGES = SIZE == 64 ? 4 : 2;   // 8 KB of a warp's ring are on their way while 8 KB are in use
  static constexpr int NK = SIZE / 64;                  // 16-byte runs of a key row per lane
  static constexpr int VB = SIZE == 64 ? 8 : 16, NV = SIZE == 256 ? 2 : 1;   // bytes of a run of a value row, runs per lane
  static constexpr int MT = SIZE / 16;                  // tiles of 16 output dimensions
  static constexpr int K_BYTES = GROUPS * 2 * NK * 512, V_BYTES = GROUPS * 4 * NV * VB * 32, STAGE = K_BYTES + V_BYTES + GROUPS * 128, RING = STAGES * STAGE;
  static constexpr int PIECE = MT * 4 * 32 + 2 * HEADS; // floats of a piece of a segment: a warp's sums, maxima and totals
  static_assert(PIECE * 4 <= RING, "a warp's last piece takes the place of its keys and values");
};

struct Plan {     // of a launch, in the shared memory of every block
  int *cum, *pos, *slot;      // [tokens + 1] tiles before, [tokens] position (of the token), [tokens]
};
struct Split {
  int tok0, tokens, chunks;   // the launch's tokens; parts of a kv head's query heads
  int grid, dtype, q_whole, out_whole;
  int *counters;              // [COUNTERS], zero between launches; [token][segment]
  float *heads;               // [grid][WARPS][PIECE]: the pieces that warps begin with and do not end with
  float *parts;               // [grid][2][PIECE]: what blocks have of segments that are not theirs alone, in front and at their end
  const void *q;
  void *out;
};

// Asynchronous copies of B bytes; zeros where !in (the source is then not read).
template <int B> __device__ __forceinline__ void copy_whole(uint32_t dst, const void *src) {
  if constexpr (B == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(B) : "memory");
}
template <int B> __device__ __forceinline__ void copy_async(uint32_t dst, const void *src, bool in) {
  if constexpr (B == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(B), "r"(in ? B : 0) : "memory");
}
template <int N> __device__ __forceinline__ void copies_left() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// Bytes 0 and 2, and 1 and 3, of a word as fp16 pairs.
template <bool E4M3> __device__ __forceinline__ void widen(uint32_t w, uint32_t &even, uint32_t &odd) {
  if constexpr (E4M3) {
    const uint32_t w8 = w << 8;
    odd = ((w >> 1) & 0x3f803f80u) | (w & 0x80008000u);
    even = ((w8 >> 1) & 0x3f803f80u) | (w8 & 0x80008000u);
  } else {
    const __half2 off = __float2half2_rn(1152.f);
    uint32_t e = (w & 0x00ff00ffu) ^ 0x64806480u, o = ((w >> 8) & 0x00ff00ffu) ^ 0x64806480u;
    const __half2 he = __hsub2(*reinterpret_cast<__half2 *>(&e), off), ho = __hsub2(*reinterpret_cast<__half2 *>(&o), off);
    even = *reinterpret_cast<const uint32_t *>(&he);
    odd = *reinterpret_cast<const uint32_t *>(&ho);
  }
}
template <bool E4M3> __device__ __forceinline__ float byte_unit() { return E4M3 ? 256.f : 1.f; }

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turn8x8(uint32_t v) {
  uint32_t t;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(v));
  return t;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void load16(const void *q, size_t at, int dtype, bool whole, int n, float (&v)[16]) {
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] = 0.f;
  if (n <= 0) return;
  auto run = [&](auto *p) {
    if (whole) {
      float lo[8], hi[8];
      load_run(p + at, lo);
      load_run(p + at + 8, hi);
#pragma unroll
      for (int j = 0; j < 8; ++j) { v[j] = lo[j]; v[8 + j] = hi[j]; }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = to_f(p[at + j]);
    }
  };
  if (dtype == PT_DT_F32) run((const float *)q);
  else if (dtype == PT_DT_F16) run((const __half *)q);
  else run((const __nv_bfloat16 *)q);
}
template <int N> __device__ __forceinline__ void store_n(void *out, size_t at, int dtype, bool whole, const float (&v)[N]) {     // 8 or 16 of them
  auto run = [&](auto *p) {
    if (whole) {
#pragma unroll
      for (int i = 0; i < N / 8; ++i) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = v[8 * i + j];
        store_run(p + at + 8 * i, x);
      }
    } else {
      using T = std::remove_pointer_t<decltype(p)>;
#pragma unroll
      for (int j = 0; j < N; ++j) p[at + j] = from_f<T>(v[j]);
    }
  };
  if (dtype == PT_DT_F32) run((float *)out);
  else if (dtype == PT_DT_F16) run((__half *)out);
  else run((__nv_bfloat16 *)out);
}

__device__ __forceinline__ void store_one(void *out, size_t at, int dtype, float v) {
  if (dtype == PT_DT_F32) ((float *)out)[at] = v;
  else if (dtype == PT_DT_F16) ((__half *)out)[at] = from_f<__half>(v);
  else ((__nv_bfloat16 *)out)[at] = from_f<__nv_bfloat16>(v);
}

// Where a run of tiles has come to: token, segment of it, tile of that.
struct Walk {
  int tok, seg, tile, tiles;
};
__device__ __forceinline__ void settle(Walk &w, const Plan &pl, int segs, int tokens) {
  while (w.tok < tokens && w.tile >= w.tiles) {
    w.tile -= w.tiles;
    if (++w.seg == segs) {
      w.seg = 0;
      do ++w.tok;
      while (w.tok < tokens && pl.cum[w.tok + 1] == pl.cum[w.tok]);
      w.tiles = w.tok < tokens ? pl.cum[w.tok + 1] - pl.cum[w.tok] : 0;
    }
  }
}
__device__ __forceinline__ Walk walk_to(int at, const Plan &pl, int segs, int tokens) {
  Walk w;
  const int x = at / segs;
  int lo = 0, hi = tokens - 1;       // the last token whose tiles begin at or before x: it has some
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (pl.cum[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  w.tok = lo;
  w.tiles = pl.cum[lo + 1] - pl.cum[lo];
  const int rest = at - pl.cum[lo] * segs;
  w.seg = rest / w.tiles;
  w.tile = rest - w.seg * w.tiles;
  return w;
}

// Pieces of one segment added up, unit j (four floats of every lane) of each: the sum, and l and R of heads 2 tg and 2 tg + 1.
struct Joined { float4 o; float L[2], R[2]; };
// OTHERS: other blocks have written them; else they may lie in shared memory.
template <int SIZE, bool OTHERS, typename At> __device__ __forceinline__ Joined add_pieces(int from, int to, int j, int lane, const At &at) {
  constexpr int SUMS = Shape<SIZE>::PIECE - 2 * HEADS;
  auto load = [](const float *p, int i) { return OTHERS ? __ldcg(reinterpret_cast<const float4 *>(p) + i) : reinterpret_cast<const float4 *>(p)[i]; };
  Joined r;
  r.o = make_float4(0.f, 0.f, 0.f, 0.f);
  r.R[0] = r.R[1] = -INFINITY;
  r.L[0] = r.L[1] = 0.f;
#pragma unroll 4
  for (int i = from; i < to; ++i) {
    const float *p = at(i);
    if (!p) continue;
    const float4 ml = load(p + SUMS, lane & 3);
    r.R[0] = fmaxf(r.R[0], ml.x);
    r.R[1] = fmaxf(r.R[1], ml.z);
  }
#pragma unroll 4
  for (int i = from; i < to; ++i) {
    const float *p = at(i);
    if (!p) continue;
    const float4 ml = load(p + SUMS, lane & 3), o = load(p, j * 32 + lane);
    const float f0 = ml.x == r.R[0] ? 1.f : exp2_fast(ml.x - r.R[0]), f1 = ml.z == r.R[1] ? 1.f : exp2_fast(ml.z - r.R[1]);
    r.L[0] += ml.y * f0;
    r.L[1] += ml.w * f1;
    r.o.x += o.x * f0; r.o.y += o.y * f1; r.o.z += o.z * f0; r.o.w += o.w * f1;
  }
  return r;
}

// FULL: keys and values are as wide as SIZE.
template <int SIZE, bool FULL, bool E4M3, int PARTS>
__global__ void __launch_bounds__(Shape<SIZE>::WARPS * 32, 1) attn_kernel(const Attn p, const Split sp) {
  early_start();
  using S = Shape<SIZE>;
  constexpr int NW = S::WARPS, KT = S::KT, GROUPS = S::GROUPS, STAGES = S::STAGES, NK = S::NK, NV = S::NV, VB = S::VB, MT = S::MT;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int scan[NW], piece[2 * NW], last;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), g = lane >> 2, tg = lane & 3;
  const int dim = FULL ? SIZE : p.c.dim, vdim = FULL ? SIZE : p.c.vdim;
  const int G = p.c.n_kv, qpk = p.heads / G, segs = G * sp.chunks, tokens = sp.tokens;
  Plan pl;
  pl.cum = reinterpret_cast<int *>(smem + NW * S::RING);
  pl.pos = pl.cum + tokens + 1;
  pl.slot = pl.pos + tokens;

  // ---- how many tiles every token has, and the sums in front of it
  const int used = p.b.cu[p.b.n_seq];
  int before = 0;
  for (int t0 = 0; t0 < tokens; t0 += NW * 32) {
    const int t = t0 + tid, tok = sp.tok0 + t;
    int n = 0;
    if (t < tokens) {
      int pos = -1, slot = 0;
      if (tok < used) {
        const int seq = p.b.tok_seq[tok], first = p.b.cu[seq], start = p.b.start[seq];
        slot = p.b.slot[seq];
        if (in_table(p.c, start, p.b.cu[seq + 1] - first)) {
          pos = start + tok - first;
          n = pos / KT - (p.window > 0 ? max(0, pos - p.window + 1) : 0) / KT + 1;
        } else if (blockIdx.x == 0 && p.error_flag) {
          atomicExch(p.error_flag, 12);
        }
      }
      pl.pos[t] = pos;
      pl.slot[t] = slot;
    }
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) scan[warp] = sum;
    __syncthreads();
    int base = before;
    for (int w = 0; w < NW; ++w) {
      if (w < warp) base += scan[w];
      before += scan[w];
    }
    if (t < tokens) pl.cum[t + 1] = base + sum;
    __syncthreads();
  }
  if (tid == 0) pl.cum[0] = 0;
  if (tid < 2 * NW) piece[tid] = -1;
  __syncthreads();
  const int all = before * segs, per = max(NW, (all + sp.grid - 1) / sp.grid), block0 = blockIdx.x * per, block_n = min(per, all - block0);
  if (block_n <= 0) return;

  // ---- this warp's run
  const int run0 = block0 + block_n * warp / NW, count = block0 + block_n * (warp + 1) / NW - run0;
  unsigned char *ring = smem + warp * S::RING;
  if (count > 0) {
    Walk w = walk_to(run0, pl, segs, tokens), ahead = w;
    const uint32_t ring_s = smem_addr(ring) + lane * 16;
    // copies: a tile a call, STAGES - 1 ahead of what is used.  A lane knows the page and the row in it of one of the next 32 groups of 16 positions.
    int ahead_at = 0, stage_in = 0, listed = 0, list_end = 0, page_l = 0, row_l = 0, kvh_in = 0;
    auto fetch = [&]() {
      if (ahead_at < count) {
        if (ahead_at >= list_end) {      // (a segment's first tile, or the list has been used up)
          const int pos = pl.pos[ahead.tok], first = (p.window > 0 ? max(0, pos - p.window + 1) : 0) / KT;
          const int at = (first + ahead.tile) * KT + lane * 16, pg = at <= pos ? at / p.c.page : 0;
          row_l = at <= pos ? at - pg * p.c.page : -1;      // (-1: behind the last position)
          page_l = at <= pos ? p.c.page_table[(size_t)pl.slot[ahead.tok] * p.c.max_pages + pg] : 0;
          if (page_l < 0) {
            if (p.error_flag) atomicExch(p.error_flag, 12);
            page_l = 0;
          }
          listed = ahead_at;
          list_end = ahead_at + min(32 / GROUPS, ahead.tiles - ahead.tile);
          kvh_in = ahead.seg / sp.chunks;
        }
        const uint32_t st = ring_s + stage_in * S::STAGE;
#pragma unroll
        for (int u = 0; u < GROUPS; ++u) {
          const int page = __shfl_sync(0xffffffffu, page_l, (ahead_at - listed) * GROUPS + u), row = __shfl_sync(0xffffffffu, row_l, (ahead_at - listed) * GROUPS + u);
          const unsigned char *base = p.c.pool + (size_t)page * p.c.page_bytes;
          const unsigned char *k = base + (kvh_in * p.c.page + row + g) * dim + 16 * tg;
          const unsigned char *v = base + (G * p.c.page) * dim + (kvh_in * p.c.page + row + 2 * tg) * vdim + VB * g;
          const float *sc = p.c.scales + (size_t)page * (2 * G * p.c.page) + ((lane >> 4) * G + kvh_in) * p.c.page + row + (lane & 15);
          const uint32_t st_v = st + S::K_BYTES + u * (4 * NV * VB * 32) - (VB == 8 ? lane * 8 : 0), st_s = st + S::K_BYTES + S::V_BYTES + u * 128 - lane * 12;
          if (FULL && row >= 0) {
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int i = 0; i < NK; ++i) copy_whole<16>(st + ((u * 2 + r) * NK + i) * 512, k + 8 * r * SIZE + 64 * i);
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int i = 0; i < NV; ++i) copy_whole<VB>(st_v + (r * NV + i) * (VB * 32), v + ((r & 1) + 8 * (r >> 1)) * SIZE + 128 * i);
            copy_whole<4>(st_s, sc);
          } else {
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int i = 0; i < NK; ++i) {
                const bool here = row >= 0 && 16 * tg + 64 * i < dim;
                copy_async<16>(st + ((u * 2 + r) * NK + i) * 512, here ? k + 8 * r * dim + 64 * i : base, here);
              }
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int i = 0; i < NV; ++i) {
                const bool here = row >= 0 && VB * g + 128 * i < vdim;
                copy_async<VB>(st_v + (r * NV + i) * (VB * 32), here ? v + ((r & 1) + 8 * (r >> 1)) * vdim + 128 * i : base, here);
              }
            copy_async<4>(st_s, row >= 0 ? sc : p.c.scales, row >= 0);
          }
        }
        ++ahead_at;
        ++ahead.tile;
        settle(ahead, pl, segs, tokens);
        if (++stage_in == STAGES) stage_in = 0;
      }
      copies_end();       // (the groups are counted)
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) fetch();

    int done = 0, stage = 0;
    while (done < count) {      // segment after segment
      const int here = min(count - done, w.tiles - w.tile), tok = w.tok;      // tiles of this segment that are the warp's
      const int kvh = w.seg / sp.chunks, chunk = w.seg - kvh * sp.chunks, head0 = kvh * qpk + chunk * HEADS, heads = min(HEADS, qpk - chunk * HEADS);
      const int pos = pl.pos[tok], begin = p.window > 0 ? max(0, pos - p.window + 1) : 0;
      float O[MT][4], R[2] = {-INFINITY, -INFINITY}, L[2] = {0.f, 0.f};
#pragma unroll
      for (int j = 0; j < MT; ++j) O[j][0] = O[j][1] = O[j][2] = O[j][3] = 0.f;
      // q as B operand: lane (g, tg) holds head g's dimensions 64 i + 16 tg + 4 c + {0, 2} and {1, 3} of k step 4 i + c
      uint32_t qf[PARTS][NK * 4][2];
      float by[2];          // factors of the scores of heads 2 tg and 2 tg + 1
      {
        float x[NK][16], most = 0.f;
        const size_t at = (size_t)(sp.tok0 + tok) * p.q_ld + (size_t)(head0 + g) * dim + 16 * tg;
#pragma unroll
        for (int i = 0; i < NK; ++i) load16(sp.q, at + 64 * i, sp.dtype, sp.q_whole, g < heads ? dim - 64 * i - 16 * tg : 0, x[i]);
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) most = fmaxf(most, fabsf(x[i][j]));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // the power of two at or below the largest element (1 for a row of zeros or infinities; within 2^-120 .. 2^120, so that its reciprocal is a number)
        const uint32_t e = __float_as_uint(most) >> 23, f = most == 0.f || e == 255 ? 127u : min(max(e, 7u), 247u);
        const float turn = __uint_as_float((254u - f) << 23), unit = __uint_as_float(f << 23);
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int o = 0; o < 2; ++o) {
              const float a = x[i][4 * c + o] * turn, b = x[i][4 * c + o + 2] * turn;
              qf[0][4 * i + c][o] = pack2(a, b);
              if constexpr (PARTS == 2) {
                const float2 h = unpack2(qf[0][4 * i + c][o]);
                qf[PARTS - 1][4 * i + c][o] = pack2(a - h.x, b - h.y);
              }
            }
#pragma unroll
        for (int h = 0; h < 2; ++h) by[h] = __shfl_sync(0xffffffffu, unit, 8 * tg + 4 * h) * (p.scale * byte_unit<E4M3>());     // (lanes 8 tg and 8 tg + 4 have their rows)
      }
      const float log2e = 1.4426950408889634f;
      if (!(p.softcap > 0.f)) { by[0] *= log2e; by[1] *= log2e; }
      int key0 = (begin / KT + w.tile) * KT;
      for (int t = 0; t < here; ++t, key0 += KT) {
        fetch();
        copies_left<STAGES - 1>();
        __syncwarp();
        const unsigned char *st = ring + stage * S::STAGE;
        const float *sc = reinterpret_cast<const float *>(st + S::K_BYTES + S::V_BYTES);
        float x[GROUPS][4];
#pragma unroll
        for (int u = 0; u < GROUPS; ++u) {
          float c[2][4] = {};
#pragma unroll
          for (int i = 0; i < NK; ++i) {
            const uint4 a = *reinterpret_cast<const uint4 *>(st + ((u * 2 + 0) * NK + i) * 512 + lane * 16), b = *reinterpret_cast<const uint4 *>(st + ((u * 2 + 1) * NK + i) * 512 + lane * 16);
            const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t a0, a1, a2, a3;
              widen<E4M3>(wa[k], a0, a2);
              widen<E4M3>(wb[k], a1, a3);
#pragma unroll
              for (int q = 0; q < PARTS; ++q) mma(c[k & 1], a0, a1, a2, a3, qf[q][4 * i + k][0], qf[q][4 * i + k][1]);
            }
          }
          const float ks[2] = {sc[u * 32 + g], sc[u * 32 + 8 + g]};
#pragma unroll
          for (int e = 0; e < 4; ++e) x[u][e] = (c[0][e] + c[1][e]) * (ks[e >> 1] * by[e & 1]);
        }
        if (p.softcap > 0.f) {
#pragma unroll
          for (int u = 0; u < GROUPS; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[u][e] = p.softcap * tanhf(x[u][e] / p.softcap) * log2e;
        }
        // about log2 of the value scales: exponent and mantissa as one number (at most 0.09 below; no less than -80: appended scales are above that)
        float vs[GROUPS][2], ev[GROUPS][2];
#pragma unroll
        for (int u = 0; u < GROUPS; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            vs[u][r] = sc[u * 32 + 16 + 8 * r + g];
            ev[u][r] = fmaxf(fmaf((float)__float_as_int(vs[u][r]), 1.f / (1 << 23), -127.f), -80.f);
          }
        if (key0 < begin || key0 + KT > pos + 1) {
#pragma unroll
          for (int u = 0; u < GROUPS; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int key = key0 + 16 * u + 8 * r + g;
              if (key < begin || key > pos) {
                x[u][2 * r] = x[u][2 * r + 1] = -INFINITY;
                vs[u][r] = 0.f;
                ev[u][r] = 0.f;
              }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float m = R[h];
#pragma unroll
          for (int u = 0; u < GROUPS; ++u) m = fmaxf(m, fmaxf(x[u][h] + ev[u][0], x[u][2 + h] + ev[u][1]));
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
          if (__any_sync(0xffffffffu, R[h] != m)) {
            const float was = R[h] == m ? 1.f : exp2_fast(R[h] - m);
            R[h] = m;
            L[h] *= was;
#pragma unroll
            for (int j = 0; j < MT; ++j) { O[j][h] *= was; O[j][2 + h] *= was; }
          }
          const float ref = (m == -INFINITY ? 0.f : m) - 14.f;
#pragma unroll
          for (int u = 0; u < GROUPS; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float e = exp2_fast(x[u][2 * r + h] - ref);
              L[h] += e;
              x[u][2 * r + h] = e * vs[u][r];
            }
        }
#pragma unroll
        for (int u = 0; u < GROUPS; ++u) {
          uint32_t wf[PARTS][2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t hi = pack2(x[u][2 * r], x[u][2 * r + 1]);
            wf[0][r] = turn8x8(hi);
            if constexpr (PARTS == 2) {
              const float2 f = unpack2(hi);
              wf[PARTS - 1][r] = turn8x8(pack2(x[u][2 * r] - f.x, x[u][2 * r + 1] - f.y));
            }
          }
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            uint32_t v[4][VB / 4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const unsigned char *at = st + S::K_BYTES + ((u * 4 + r) * NV + i) * (VB * 32) + lane * VB;
              if constexpr (VB == 16) {
                const uint4 y = *reinterpret_cast<const uint4 *>(at);
                v[r][0] = y.x; v[r][1] = y.y; v[r][VB / 4 - 2] = y.z; v[r][VB / 4 - 1] = y.w;
              } else {
                const uint2 y = *reinterpret_cast<const uint2 *>(at);
                v[r][0] = y.x; v[r][1] = y.y;
              }
            }
#pragma unroll
            for (int k = 0; k < VB / 4; ++k)
#pragma unroll
              for (int half = 0; half < 2; ++half) {     // dimensions 4 k + 2 half and the next, of keys (0, 1) and (2, 3)
                uint32_t a0, a1, a2, a3;
                widen<E4M3>(__byte_perm(v[0][k], v[1][k], half ? 0x7632 : 0x5410), a0, a1);
                widen<E4M3>(__byte_perm(v[2][k], v[3][k], half ? 0x7632 : 0x5410), a2, a3);
#pragma unroll
                for (int q = 0; q < PARTS; ++q) mma(O[i * 8 + 2 * k + half], a0, a1, a2, a3, wf[q][0], wf[q][1]);
              }
          }
        }
        __syncwarp();      // the scales have been read by all lanes
        if (++stage == STAGES) stage = 0;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) L[h] += __shfl_xor_sync(0xffffffffu, L[h], o);

      done += here;
      if (here == w.tiles) {          // a whole segment leaves
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (2 * tg + h >= heads) continue;
          const float f = byte_unit<E4M3>() / L[h];
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            if (VB * g + 128 * i >= vdim) continue;
            float y[VB];
#pragma unroll
            for (int j = 0; j < VB / 2; ++j) {
              y[2 * j] = O[i * 8 + j][h] * f;
              y[2 * j + 1] = O[i * 8 + j][2 + h] * f;
            }
            store_n<VB>(sp.out, (size_t)(sp.tok0 + tok) * p.out_ld + (size_t)(head0 + 2 * tg + h) * vdim + VB * g + 128 * i, sp.dtype, sp.out_whole, y);
          }
        }
      } else {                        // a piece stays: the last one in shared memory, where no tile is needed any more
        const bool end = done == count;
        float *to = end ? reinterpret_cast<float *>(ring) : sp.heads + ((size_t)blockIdx.x * NW + warp) * S::PIECE;
        if (end) {
          copies_left<0>();
          __syncwarp();
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) reinterpret_cast<float4 *>(to)[j * 32 + lane] = make_float4(O[j][0], O[j][1], O[j][2], O[j][3]);
        if (g == 0) reinterpret_cast<float4 *>(to + MT * 128)[tg] = make_float4(R[0], L[0], R[1], L[1]);
        if (lane == 0) piece[2 * warp + end] = tok * segs + w.seg;
      }
      w.tile += here;
      settle(w, pl, segs, tokens);
    }
    copies_left<0>();
  }
  __syncthreads();

  // ---- pieces of a segment come together
  auto leave = [&](const Joined &r, int id, int j) {
    const int tok = id / segs, seg = id - tok * segs, kvh = seg / sp.chunks, chunk = seg - kvh * sp.chunks, heads = min(HEADS, qpk - chunk * HEADS);
    const int d = VB * g + 128 * (j / 8) + 2 * (j % 8);
    const float o[2][2] = {{r.o.x, r.o.z}, {r.o.y, r.o.w}};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (2 * tg + h >= heads || d >= vdim) continue;
      const float f = byte_unit<E4M3>() / r.L[h];
      const size_t at = (size_t)(sp.tok0 + tok) * p.out_ld + (size_t)(kvh * qpk + chunk * HEADS + 2 * tg + h) * vdim + d;
#pragma unroll
      for (int e = 0; e < 2; ++e) store_one(sp.out, at + e, sp.dtype, o[h][e] * f);
    }
  };
  for (int i0 = 0; i0 < 2 * NW;) {
    const int id = piece[i0];
    int i1 = i0 + 1;
    if (id >= 0) {
      while (i1 < 2 * NW && (piece[i1] == id || piece[i1] < 0)) ++i1;
      auto mine = [&](int i) -> const float * {
        return piece[i] < 0 ? nullptr : i & 1 ? reinterpret_cast<const float *>(smem + (i >> 1) * S::RING) : sp.heads + ((size_t)blockIdx.x * NW + (i >> 1)) * S::PIECE;
      };
      const int tok = id / segs, tiles = pl.cum[tok + 1] - pl.cum[tok], tile0 = pl.cum[tok] * segs + (id - tok * segs) * tiles, b0 = tile0 / per, b1 = (tile0 + tiles - 1) / per;
      float *part = sp.parts + ((size_t)blockIdx.x * 2 + (tile0 > block0)) * S::PIECE;
      for (int j = warp; j < MT; j += NW) {
        const Joined r = add_pieces<SIZE, false>(i0, i1, j, lane, mine);
        if (b0 == b1) {
          leave(r, id, j);
        } else {
          __stcg(reinterpret_cast<float4 *>(part) + j * 32 + lane, r.o);
          if (j == 0 && g == 0) __stcg(reinterpret_cast<float4 *>(part + MT * 128) + tg, make_float4(r.R[0], r.L[0], r.R[1], r.L[1]));
        }
      }
      if (b0 != b1) {
        __threadfence();
        __syncthreads();
        if (tid == 0) {
          last = atomicAdd(sp.counters + id, 1) == b1 - b0;
          if (last) sp.counters[id] = 0;
          __threadfence();
        }
        __syncthreads();
        if (last) {
          auto theirs = [&](int b) -> const float * { return sp.parts + ((size_t)b * 2 + (tile0 > b * per)) * S::PIECE; };
          for (int j = warp; j < MT; j += NW) leave(add_pieces<SIZE, true>(b0, b1 + 1, j, lane, theirs), id, j);
        }
        __syncthreads();
      }
    }
    i0 = i1;
  }
}

}  // namespace kv8
}  // namespace pt
