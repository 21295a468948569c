// Attention of new tokens over a cache of eight bits, on tensor cores (included by kv8.cu).
//
// A segment is one token, one kv head and up to eight of its query heads; its keys are tiles of KT positions.  All tiles of a launch lie in one row, segment
// after segment, and every block takes an equal run of them, so that unequal histories cost nobody a wait; the warps of a block take every NW-th tile of its run.
//   scores [16 keys x 8 heads] = K . q^T,   out^T [16 dims x 8 heads] += V^T . W^T      (mma m16n8k16, fp16 operands, fp32 sums)
// A lane copies to shared memory (cp.async) exactly what it reads back, so the ring of a warp needs no barrier and no swizzle: 16 bytes of two key rows (row of the fragment), 16
// bytes of four value rows (its keys).  Which dimension of the head is which k of an instruction does not matter as long as K and q agree: a lane's k are the dimensions of
// its bytes.  Bytes become fp16 exactly: int8 b as (1024 + 128 + b) - 1152, E4M3 by its bits (times 2^-8, which the scales take back).
//
// Numbers.  q comes in fp16 times a power of two that brings its row's largest element to [1, 2): what is lost lies below 2^-25 of that; queries of 32 bits have a second fp16 part.
// With x = score log2(e), v_j = bytes times vs_j, and e_j the exponent of vs_j, a segment keeps R = max (x_j + e_j), l = sum 2^(x_j - R + 14) in 32 bits, and sums
// w_j (bytes of v_j) with w_j = 2^(x_j - R + 14) vs_j, at most 2^15: rounded to fp16 once (2^-11; two parts for rows of 32 bits), whole down to 2^-29 of the largest and then off by
// 2^-40 of it, however far the scales of the values lie apart.
#pragma once
#include <type_traits>

#include "tile_math.cuh"

namespace pt {
namespace kv8 {

constexpr int NW = 4, HEADS = 8, MAX_TOKENS = 1024;
constexpr int COUNTERS = 1 << 16;      // of a workspace, always in front: whichever calls share one, nothing else is written there

// SIZE: the widest head, 64, 128 or 256.
template <int SIZE> struct Shape {
  static constexpr int KT = SIZE == 256 ? 16 : 32, GROUPS = KT / 16, STAGES = SIZE == 64 ? 4 : 2;   // 8 KB of a warp's ring are on their way while 8 KB are in use
  static constexpr int NK = SIZE / 64;                  // 16-byte runs of a key row per lane
  static constexpr int VB = SIZE == 64 ? 8 : 16, NV = SIZE == 256 ? 2 : 1;   // bytes of a run of a value row, runs per lane
  static constexpr int MT = SIZE / 16;                  // tiles of 16 output dimensions
  static constexpr int K_BYTES = GROUPS * 2 * NK * 512, V_BYTES = GROUPS * 4 * NV * VB * 32, STAGE = K_BYTES + V_BYTES + GROUPS * 128;
  static constexpr int JOIN = MT * 4 * 32 * 4;          // a warp's sums
  static constexpr int PART = JOIN / 4 + 2 * HEADS;     // ... with maxima and totals, in floats
};
constexpr int BLOCKS_PER_SM = 3;

struct Plan {     // of a launch, in the shared memory of every block
  int *cum, *pos, *slot;      // [tokens + 1] tiles before, [tokens] position (of the token), [tokens]
};
struct Split {
  int tok0, tokens, chunks;   // the launch's tokens; parts of a kv head's query heads
  int grid, dtype, q_whole, out_whole;
  int *counters;              // [COUNTERS], zero between launches; [token][segment]
  float *parts;               // [grid][2][PART]
  const void *q;
  void *out;
};

__device__ __forceinline__ void copy_async(uint32_t dst, const void *src, int bytes, bool in) {
  if (bytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
  else if (bytes == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(in ? 8 : 0) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
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

template <int SIZE, bool E4M3, int PARTS>
__global__ void __launch_bounds__(NW * 32, SIZE == 256 ? 2 : BLOCKS_PER_SM) attn_kernel(const Attn p, const Split sp) {
  early_start();
  using S = Shape<SIZE>;
  constexpr int KT = S::KT, GROUPS = S::GROUPS, STAGES = S::STAGES, NK = S::NK, NV = S::NV, VB = S::VB, MT = S::MT;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float join_ml[2 * HEADS];
  __shared__ int scan[NW];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tg = lane & 3;
  const int G = p.c.n_kv, qpk = p.heads / G, segs = G * sp.chunks, tokens = sp.tokens;
  float *join = reinterpret_cast<float *>(smem + NW * STAGES * S::STAGE);
  Plan pl;
  pl.cum = reinterpret_cast<int *>(smem + NW * STAGES * S::STAGE + S::JOIN);
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
  __syncthreads();
  const long long all = (long long)before * segs, per = max((long long)NW, (all + sp.grid - 1) / sp.grid), run0 = blockIdx.x * per, run1 = min(all, run0 + per);
  if (run0 >= run1) return;

  // ---- the segment that the run begins in, and where this warp begins
  Walk from;
  {
    const int x = (int)(run0 / segs);
    int lo = 0, hi = tokens - 1;       // the last token whose tiles begin at or before x, and which has some
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (pl.cum[mid] <= x) lo = mid;
      else hi = mid - 1;
    }
    from.tok = lo;
    from.tiles = pl.cum[lo + 1] - pl.cum[lo];
    const long long rest = run0 - (long long)pl.cum[lo] * segs;
    from.seg = (int)(rest / from.tiles);
    from.tile = (int)(rest - (long long)from.seg * from.tiles);
  }
  const int count = (int)(run1 - run0);
  unsigned char *ring = smem + warp * STAGES * S::STAGE;
  const uint32_t ring_s = smem_addr(ring);

  // ---- copies: a tile a call, STAGES - 1 ahead of what is used
  Walk ahead = from;
  ahead.tile += warp;
  settle(ahead, pl, segs, tokens);
  int ahead_at = warp, stage_in = 0, listed_tok = -1, listed_seg = -1, listed_tile = 0, page_l = 0, row_l = 0;
  auto fetch = [&]() {
    if (ahead_at < count) {
      const int pos = pl.pos[ahead.tok], first = (p.window > 0 ? max(0, pos - p.window + 1) : 0) / KT;
      // (pages of the next tiles of this warp in this segment, one group of 16 positions a lane)
      if (ahead.tok != listed_tok || ahead.seg != listed_seg || ahead.tile - listed_tile >= 32 / GROUPS * NW) {
        listed_tok = ahead.tok; listed_seg = ahead.seg; listed_tile = ahead.tile;
        const int at = (first + ahead.tile + lane / GROUPS * NW) * KT + lane % GROUPS * 16;
        const int pg = at <= pos ? at / p.c.page : 0;
        page_l = at <= pos ? p.c.page_table[(size_t)pl.slot[ahead.tok] * p.c.max_pages + pg] : 0;
        row_l = at - pg * p.c.page;
        if (page_l < 0) {
          if (p.error_flag) atomicExch(p.error_flag, 12);
          page_l = 0;
        }
      }
      const int kvh = ahead.seg / sp.chunks, in_list = (ahead.tile - listed_tile) / NW * GROUPS;
      const uint32_t st = ring_s + stage_in * S::STAGE;
#pragma unroll
      for (int u = 0; u < GROUPS; ++u) {
        const int page = __shfl_sync(0xffffffffu, page_l, in_list + u), row = __shfl_sync(0xffffffffu, row_l, in_list + u);
        const bool in = (first + ahead.tile) * KT + 16 * u <= pos;
        const unsigned char *base = p.c.pool + (size_t)page * p.c.page_bytes;
        const unsigned char *k = base + ((size_t)kvh * p.c.page + (in ? row : 0) + g) * p.c.dim + 16 * tg;
        const unsigned char *v = base + (size_t)G * p.c.page * p.c.dim + ((size_t)kvh * p.c.page + (in ? row : 0) + 2 * tg) * p.c.vdim + VB * g;
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int i = 0; i < NK; ++i) {
            const bool here = in && 16 * tg + 64 * i < p.c.dim;
            copy_async(st + ((u * 2 + r) * NK + i) * 512 + lane * 16, here ? k + (size_t)(8 * r) * p.c.dim + 64 * i : base, 16, here);
          }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const bool here = in && VB * g + 128 * i < p.c.vdim;
            copy_async(st + S::K_BYTES + ((u * 4 + r) * NV + i) * (VB * 32) + lane * VB, here ? v + (size_t)((r & 1) + 8 * (r >> 1)) * p.c.vdim + 128 * i : base, VB, here);
          }
        copy_async(st + S::K_BYTES + S::V_BYTES + u * 128 + lane * 4,
                   p.c.scales + (((size_t)page * 2 + (lane >> 4)) * G + kvh) * p.c.page + (in ? row : 0) + (lane & 15), 4, in);
      }
      ahead_at += NW;
      ahead.tile += NW;
      settle(ahead, pl, segs, tokens);
      if (++stage_in == STAGES) stage_in = 0;
    }
    copies_end();       // (the groups are counted)
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) fetch();

  // ---- segment after segment
  Walk w = from;
  int done = 0, mine = warp, stage = 0;       // tiles of the run that lie behind; this warp's next
  while (done < count) {
    const int here = min(count - done, w.tiles - w.tile), tok = w.tok;      // tiles of this segment that are the block's
    const int kvh = w.seg / sp.chunks, chunk = w.seg - kvh * sp.chunks, head0 = kvh * qpk + chunk * HEADS, heads = min(HEADS, qpk - chunk * HEADS);
    const int pos = pl.pos[tok], begin = p.window > 0 ? max(0, pos - p.window + 1) : 0, first = begin / KT;
    float O[MT][4], R[2] = {-INFINITY, -INFINITY}, L[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < MT; ++j) O[j][0] = O[j][1] = O[j][2] = O[j][3] = 0.f;
    if (mine < done + here) {
      // q as B operand: lane (g, tg) holds head g's dimensions 64 i + 16 tg + 4 c + {0, 2} and {1, 3} of k step 4 i + c
      uint32_t qf[PARTS][NK * 4][2];
      float unit;
      {
        float x[NK][16], most = 0.f;
        const size_t at = (size_t)(sp.tok0 + tok) * p.q_ld + (size_t)(head0 + g) * p.c.dim + 16 * tg;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          load16(sp.q, at + 64 * i, sp.dtype, sp.q_whole, g < heads ? p.c.dim - 64 * i - 16 * tg : 0, x[i]);
#pragma unroll
          for (int j = 0; j < 16; ++j) most = fmaxf(most, fabsf(x[i][j]));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // the power of two at or below the largest element (1 for a row of zeros or infinities; 2^-120 at least, so that its reciprocal is a number)
        const uint32_t e = __float_as_uint(most) >> 23;
        const uint32_t f = e == 0 ? (most == 0.f ? 127u : 7u) : e == 255 ? 127u : min(max(e, 7u), 247u);
        const float by = __uint_as_float((254u - f) << 23);
        unit = __uint_as_float(f << 23);
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int o = 0; o < 2; ++o) {
              const float a = x[i][4 * c + o] * by, b = x[i][4 * c + o + 2] * by;
              qf[0][4 * i + c][o] = pack2(a, b);
              if constexpr (PARTS == 2) {
                const float2 h = unpack2(qf[0][4 * i + c][o]);
                qf[PARTS - 1][4 * i + c][o] = pack2(a - h.x, b - h.y);
              }
            }
      }
      // factors of the scores of heads 2 tg and 2 tg + 1, whose q rows lanes 8 tg and 8 tg + 4 have
      float by[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) by[h] = __shfl_sync(0xffffffffu, unit, 8 * tg + 4 * h) * (p.scale * byte_unit<E4M3>());
      const float log2e = 1.4426950408889634f;
      for (; mine < done + here; mine += NW) {
        fetch();
        copies_left<STAGES - 1>();
        __syncwarp();
        const unsigned char *st = ring + stage * S::STAGE;
        const float *sc = reinterpret_cast<const float *>(st + S::K_BYTES + S::V_BYTES);
        const int key0 = (first + w.tile + mine - done) * KT;
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
            for (int e = 0; e < 4; ++e) x[u][e] = p.softcap * tanhf(x[u][e] / p.softcap);
        }
        const bool border = key0 < begin || key0 + KT > pos + 1;
        float vs[GROUPS][2], ev[GROUPS][2];
#pragma unroll
        for (int u = 0; u < GROUPS; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            vs[u][r] = sc[u * 32 + 16 + 8 * r + g];
            ev[u][r] = (float)(min(max((int)(__float_as_uint(vs[u][r]) >> 23 & 255u), 47), 191) - 127);      // (2^-80 .. 2^64: appended scales are within)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              x[u][2 * r + h] *= log2e;
              if (border) {
                const int key = key0 + 16 * u + 8 * r + g;
                if (key < begin || key > pos) x[u][2 * r + h] = -INFINITY;
              }
            }
            if (border && (key0 + 16 * u + 8 * r + g < begin || key0 + 16 * u + 8 * r + g > pos)) vs[u][r] = 0.f;
          }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float m = R[h];
#pragma unroll
          for (int u = 0; u < GROUPS; ++u) m = fmaxf(m, fmaxf(x[u][h] + ev[u][0], x[u][2 + h] + ev[u][1]));
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
          const float was = R[h] == m ? 1.f : exp2_fast(R[h] - m);
          R[h] = m;
          if (__any_sync(0xffffffffu, was != 1.f)) {
            L[h] *= was;
#pragma unroll
            for (int j = 0; j < MT; ++j) { O[j][h] *= was; O[j][2 + h] *= was; }
          }
          const float ref = (m == -INFINITY ? 0.f : m) - 14.f;
#pragma unroll
          for (int u = 0; u < GROUPS; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float t = exp2_fast(x[u][2 * r + h] - ref);
              L[h] += t;
              x[u][2 * r + h] = t * vs[u][r];
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
    }

    // ---- the warps' sums come together in warp 0, one after the other
    for (int j0 = 0; j0 < min(here, NW); ++j0) {
      const int who = (int)((done + j0) % NW);       // (the warps that have tiles of it)
      if (who == 0) continue;
      __syncthreads();
      if (warp == who) {
#pragma unroll
        for (int j = 0; j < MT; ++j) reinterpret_cast<float4 *>(join)[j * 32 + lane] = make_float4(O[j][0], O[j][1], O[j][2], O[j][3]);
        if (g == 0) {
          join_ml[4 * tg] = R[0]; join_ml[4 * tg + 1] = L[0];
          join_ml[4 * tg + 2] = R[1]; join_ml[4 * tg + 3] = L[1];
        }
      }
      __syncthreads();
      if (warp == 0) {
        float mine_by[2], its_by[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float r = join_ml[4 * tg + 2 * h], l = join_ml[4 * tg + 2 * h + 1], m = fmaxf(R[h], r);
          mine_by[h] = R[h] == m ? 1.f : exp2_fast(R[h] - m);
          its_by[h] = r == m ? 1.f : exp2_fast(r - m);
          R[h] = m;
          L[h] = L[h] * mine_by[h] + l * its_by[h];
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const float4 o = reinterpret_cast<const float4 *>(join)[j * 32 + lane];
          O[j][0] = O[j][0] * mine_by[0] + o.x * its_by[0]; O[j][1] = O[j][1] * mine_by[1] + o.y * its_by[1];
          O[j][2] = O[j][2] * mine_by[0] + o.z * its_by[0]; O[j][3] = O[j][3] * mine_by[1] + o.w * its_by[1];
        }
      }
    }

    // ---- a whole segment leaves; of a part the last block to come finds the others'
    const long long seg_tile0 = run0 + done - w.tile, seg_tile1 = seg_tile0 + w.tiles;
    const int b0 = (int)(seg_tile0 / per), b1 = (int)((seg_tile1 - 1) / per);
    bool write = warp == 0;
    if (b1 > b0) {
      constexpr int PART = S::PART;
      const int id = tok * segs + w.seg;
      if (warp == 0) {
        float *to = sp.parts + ((size_t)blockIdx.x * 2 + (seg_tile0 > run0 ? 1 : 0)) * PART;
#pragma unroll
        for (int j = 0; j < MT; ++j) __stcg(reinterpret_cast<float4 *>(to) + j * 32 + lane, make_float4(O[j][0], O[j][1], O[j][2], O[j][3]));
        if (g == 0) __stcg(reinterpret_cast<float4 *>(to + S::JOIN / 4) + tg, make_float4(R[0], L[0], R[1], L[1]));
        __threadfence();
        __syncwarp();
        int last = lane == 0 ? atomicAdd(sp.counters + id, 1) == b1 - b0 : 0;
        write = __shfl_sync(0xffffffffu, last, 0);
      }
      if (write) {
        __threadfence();
        if (lane == 0) sp.counters[id] = 0;
        auto part_of = [&](int b) { return sp.parts + ((size_t)b * 2 + (seg_tile0 > b * per ? 1 : 0)) * PART; };
        R[0] = R[1] = -INFINITY;
        L[0] = L[1] = 0.f;
#pragma unroll
        for (int j = 0; j < MT; ++j) O[j][0] = O[j][1] = O[j][2] = O[j][3] = 0.f;
        for (int b = b0; b <= b1; ++b) {
          const float4 ml = __ldcg(reinterpret_cast<const float4 *>(part_of(b) + S::JOIN / 4) + tg);
          R[0] = fmaxf(R[0], ml.x);
          R[1] = fmaxf(R[1], ml.z);
        }
        for (int b = b0; b <= b1; ++b) {
          const float *from_part = part_of(b);
          const float4 ml = __ldcg(reinterpret_cast<const float4 *>(from_part + S::JOIN / 4) + tg);
          const float f0 = ml.x == R[0] ? 1.f : exp2_fast(ml.x - R[0]), f1 = ml.z == R[1] ? 1.f : exp2_fast(ml.z - R[1]);
          L[0] += ml.y * f0;
          L[1] += ml.w * f1;
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            const float4 o = __ldcg(reinterpret_cast<const float4 *>(from_part) + j * 32 + lane);
            O[j][0] += o.x * f0; O[j][1] += o.y * f1; O[j][2] += o.z * f0; O[j][3] += o.w * f1;
          }
        }
      }
    }
    if (write) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (2 * tg + h >= heads) continue;
        const float by = byte_unit<E4M3>() / L[h];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          constexpr int N = VB;            // dimensions VB g + 128 i .. of this lane
          if (VB * g + 128 * i >= p.c.vdim) continue;
          float y[N];
#pragma unroll
          for (int j = 0; j < N / 2; ++j) {
            y[2 * j] = O[i * 8 + j][h] * by;
            y[2 * j + 1] = O[i * 8 + j][2 + h] * by;
          }
          store_n<N>(sp.out, (size_t)(sp.tok0 + tok) * p.out_ld + (size_t)(head0 + 2 * tg + h) * p.c.vdim + VB * g + 128 * i, sp.dtype, sp.out_whole, y);
        }
      }
    }
    done += here;
    w.tile += here;
    settle(w, pl, segs, tokens);
  }
  copies_left<0>();
}

}  // namespace kv8
}  // namespace pt
