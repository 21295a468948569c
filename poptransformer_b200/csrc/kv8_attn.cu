// Attention of new tokens over a cache of eight bits (kv8.cuh), on tensor cores.
//
// A segment is one token, one kv head and up to eight of its query heads; its keys are tiles of KT positions.  All tiles of a launch lie in one row, segment
// after segment; every block takes an equal run of them, and every warp an equal run of its block's, so that unequal histories cost nobody a wait and warps meet
// once, at their end.  A segment that lies in one warp's run leaves from there; the pieces of others are added up by the block that has all of them, or by the last of the blocks that
// have some to come (in the order of the pieces, so that the sum does not depend on who was last).
//   scores [16 keys x 8 heads] = K . q^T,   out^T [16 dims x 8 heads] += V^T . W^T      (mma m16n8k16, fp16 operands, fp32 sums)
// Rows come to a warp's ring by asynchronous copies of 512 bytes that lie together (16 a lane; copies in the order of the fragments, four or eight rows each, reached 4.8 TB/s alone,
// these 6.5), and are read as fragments: a lane has 16 bytes of two key rows (row of the fragment), 16
// bytes of four value rows (its keys).  Which dimension of the head is which k of an instruction does not matter as long as K and q agree: a lane's k are the dimensions of
// its bytes.  Keys of int8 are multiplied as they are, with q in three parts of 8 bits (m16n8k32, whole numbers); all other bytes become fp16, exactly: E4M3 by conversion, int8 b as
// (1024 + 128 + b) - 1152.
// Bound by memory: 48 sequences of up to 8000 positions, 32 query over 8 kv heads of 128, 519 MB, 96 us, 5.4 TB/s (105 in a long run of such calls, when the power limit
// takes the clock from 1965 MHz to about 1700); 7 TB/s from a block's first tile to its last, 820 instructions a tile of 32 positions, which is half of the issue slots.  Two sequences of 100,000, E4M3: 79 us.
// One of 700: 10.2 us, latency.
//
// Numbers.  int8: q to 2^-22 of its row's largest element.  E4M3: q in fp16 times a power of two that brings its row's largest element to [1, 2), and for rows that are not bf16 a second part of
// what is left: what is lost lies below 2^-25 of the largest.
// With x = score log2(e), v_j = bytes times vs_j, and e_j about log2 vs_j, a segment keeps R = max (x_j + e_j), l = sum 2^(x_j - R + 14) in 32 bits, and sums
// w_j (bytes of v_j) with w_j = 2^(x_j - R + 14) vs_j, below 2^15, in two fp16 parts: 2^-21 of a weight, whole down to 2^-29 of the largest and then off by
// 2^-40 of it, however far the scales of the values lie apart.  (One part, 2^-11, for rows of bf16 moved outputs to the neighbouring number, 0.0011 of
// their size altogether where two parts are 0.0001 from the plain form.  It took 98 us for the 48 sequences, 100 in a long run, where it needs less power; two parts 96 and 105.  Long sequences: 78.2, 78.6.)
#include "kv8.cuh"
#include "tile_math.cuh"

namespace pt {
namespace kv8 {

struct Attn {
  Batch b;
  Cache c;
  int heads, window, q_ld, out_ld;
  float scale, softcap;
  int *error_flag;
};

constexpr int HEADS = 8, MAX_TOKENS = 1024;
constexpr int SHORT = 3;      // tiles of a warp up to which a segment stays in one block (32 query over 8 kv heads of 128, one token: 700 positions 10.2 us so, 13.0 dealt out; 1300 13.7 either way; both limits were measured at this width alone)
constexpr int ALIGNED = 6;    // ... and up to which a block has whole segments (64 sequences of 300 positions 21.0 us dealt out evenly, so 19.2; of 2000 48.5 and 46.3; from 9 on the blocks' loads differ too much)
constexpr int COUNTERS = 1 << 16;      // of a workspace, always in front: whichever calls share one, nothing else is written there

// SIZE: the widest head, 64, 128 or 256.
template <int SIZE> struct Shape {
  static constexpr int WARPS = SIZE == 256 ? 8 : 12;    // one block to an SM: 168 registers a thread (254), 16.5 KB of shared memory a warp
  static constexpr int KT = SIZE == 256 ? 16 : 32, GROUPS = KT / 16, STAGES = SIZE == 64 ? 4 : 2;   // 8 KB of a warp's ring are on their way while 8 KB are in use
  static constexpr int NK = SIZE / 64;                  // 16-byte runs of a key row per lane
  static constexpr int VB = SIZE == 64 ? 8 : 16, NV = SIZE == 256 ? 2 : 1;   // bytes of a run of a value row, runs per lane
  static constexpr int MT = SIZE / 16;                  // tiles of 16 output dimensions
  static constexpr int COPIES = SIZE / 32;              // of 512 bytes, 16 a lane, for 16 rows
  static constexpr int ROWS = KT * SIZE, STAGE = 2 * ROWS + GROUPS * 128, RING = STAGES * STAGE;      // keys, values, scales
  static constexpr int PIECE = MT * 4 * 32 + 2 * HEADS; // floats of a piece of a segment: a warp's sums, maxima and totals
  static_assert(PIECE * 4 <= RING, "a warp's last piece takes the place of its keys and values");
};

struct Plan {     // of a launch, in the shared memory of every block
  int *cum, *pos, *slot;      // [tokens + 1] tiles before, [tokens] position (of the token), [tokens]
};
struct Split {
  int tok0, tokens, chunks;   // the launch's tokens; parts of a kv head's query heads
  int segs, grid, dtype, q_whole, out_whole;
  Divide by_segs, by_chunks, by_page, by_grid;
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

// Bytes of two words as fp16 pairs: (byte 2 half of x, of y) and (byte 2 half + 1 of x, of y).
template <bool E4M3> __device__ __forceinline__ void widen(uint32_t x, uint32_t y, int half, uint32_t &first, uint32_t &second) {
  if constexpr (E4M3) {
    const uint32_t w = __byte_perm(x, y, half ? 0x7362 : 0x5140);
    asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h;}" : "=r"(first), "=r"(second) : "r"(w));
  } else {
    const uint32_t w = __byte_perm(x, y, half ? 0x7632 : 0x5410);
    const __half2 off = __float2half2_rn(1152.f);
    uint32_t a = (w & 0x00ff00ffu) ^ 0x64806480u, b = ((w >> 8) & 0x00ff00ffu) ^ 0x64806480u;     // 1024 + 128 + byte
    const __half2 ha = __hsub2(*reinterpret_cast<__half2 *>(&a), off), hb = __hsub2(*reinterpret_cast<__half2 *>(&b), off);
    first = *reinterpret_cast<const uint32_t *>(&ha);
    second = *reinterpret_cast<const uint32_t *>(&hb);
  }
}
// The first product of a sum.
__device__ __forceinline__ void mma_s8_first(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ void mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
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

// Sixteen elements of a query, as they lie there (`whole`: on a multiple of 16 bytes) or, of any other rows, as fp32; asked for before the tiles, used behind them.
__device__ __forceinline__ void load16(const void *q, size_t at, int dtype, bool whole, int n, uint32_t (&v)[16]) {
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] = 0;
  if (n <= 0) return;
  if (whole) {
    const uint4 *p = reinterpret_cast<const uint4 *>((const char *)q + at * (dtype == PT_DT_F32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < 2 || dtype == PT_DT_F32) {
        const uint4 w = p[i];
        v[4 * i] = w.x; v[4 * i + 1] = w.y; v[4 * i + 2] = w.z; v[4 * i + 3] = w.w;
      }
  } else {
#pragma unroll 1
    for (int j = 0; j < 16; ++j) {
      const uint32_t x = __float_as_uint(dtype == PT_DT_F32 ? ((const float *)q)[at + j] : dtype == PT_DT_F16 ? __half2float(((const __half *)q)[at + j]) : __bfloat162float(((const __nv_bfloat16 *)q)[at + j]));
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] = k == j ? x : v[k];
    }
  }
}
__device__ __forceinline__ void floats16(uint32_t (&v)[16], int dtype, bool whole) {
  if (!whole || dtype == PT_DT_F32) return;
#pragma unroll
  for (int j = 7; j >= 0; --j) {
    const uint32_t w = v[j];
    if (dtype == PT_DT_F16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
      v[2 * j] = __float_as_uint(f.x); v[2 * j + 1] = __float_as_uint(f.y);
    } else {
      v[2 * j] = w << 16; v[2 * j + 1] = w & 0xffff0000u;
    }
  }
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

// Two neighbouring dimensions of up to two heads, the sums o over l.
static __device__ __noinline__ void store_sums(void *out, size_t at, int vdim, int dtype, int heads, float4 o, float l0, float l1) {
  const float y[4] = {__fdividef(o.x, l0), __fdividef(o.z, l0), __fdividef(o.y, l1), __fdividef(o.w, l1)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i / 2 >= heads) return;
    const size_t to = at + (i & 1) + (i / 2) * vdim;
    if (dtype == PT_DT_F32) ((float *)out)[to] = y[i];
    else if (dtype == PT_DT_F16) ((__half *)out)[to] = from_f<__half>(y[i]);
    else ((__nv_bfloat16 *)out)[to] = from_f<__nv_bfloat16>(y[i]);
  }
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
__device__ __forceinline__ Walk walk_to(int at, const Plan &pl, int segs, const Divide &by_segs, int tokens) {
  Walk w;
  const int x = by_segs(at);
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

// FULL: keys and values are as wide as SIZE.  QUERY_PARTS: fp16 parts of queries over E4M3 keys: 1 for rows of bf16, which have eight bits, 2 for others.
template <int SIZE, bool FULL, bool E4M3, int QUERY_PARTS>
__global__ void __launch_bounds__(Shape<SIZE>::WARPS * 32, 1) attn_kernel(const Attn p, const Split sp) {
  early_start();
  using S = Shape<SIZE>;
  constexpr int QPARTS = E4M3 ? QUERY_PARTS : 3, QREGS = E4M3 ? 2 : 1, NW = S::WARPS, KT = S::KT, GROUPS = S::GROUPS, STAGES = S::STAGES, NK = S::NK, NV = S::NV, VB = S::VB, MT = S::MT;
  extern __shared__ __align__(128) unsigned char smem[];
  // The pieces of segments that warps begin and end with: which segments, and (R, l) of every head.
  __shared__ int scan[NW], widest[NW], front[NW], rear[NW], first_block[2], parts[2];
  __shared__ float2 ml[2 * NW][HEADS];      // rears, fronts
  __shared__ __align__(16) float2 share[2 * NW][HEADS];      // factors that bring the pieces of a segment to one R, and l times those
  __shared__ float top[2 * NW][HEADS];      // that R
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), g = lane >> 2, tg = lane & 3;
  const int dim = FULL ? SIZE : p.c.dim, vdim = FULL ? SIZE : p.c.vdim;
  const int G = p.c.n_kv, qpk = p.heads / G, segs = sp.segs, tokens = sp.tokens;
  Plan pl;
  pl.cum = reinterpret_cast<int *>(smem + NW * S::RING);
  pl.pos = pl.cum + tokens + 1;
  pl.slot = pl.pos + tokens;

  // ---- how many tiles every token has, and the sums in front of it
  const int used = p.b.cu[p.b.n_seq];
  int before = 0, most = 0;
  const bool few = tokens <= 32;      // (every warp counts them by itself)
  for (int t0 = 0; t0 < tokens; t0 += few ? 32 : NW * 32) {
    const int t = few ? lane : t0 + tid, tok = sp.tok0 + t;
    int n = 0;
    if (t < tokens) {
      int pos = -1, slot = 0;
      // (of a batch of one token a sequence these are asked for together; a row that no sequence has may name any)
      const int guess = min(tok, p.b.n_seq - 1), seq = p.b.tok_seq[tok];
      int first = p.b.cu[guess], end = p.b.cu[guess + 1], start = p.b.start[guess];
      slot = p.b.slot[guess];
      if (tok < used) {
        if (seq != guess) {
          first = p.b.cu[seq];
          end = p.b.cu[seq + 1];
          start = p.b.start[seq];
          slot = p.b.slot[seq];
        }
        if (in_table(p.c, start, end - first)) {
          pos = start + tok - first;
          n = pos / KT - (p.window > 0 ? max(0, pos - p.window + 1) : 0) / KT + 1;
        } else if (blockIdx.x == 0 && (!few || warp == 0) && p.error_flag) {
          atomicExch(p.error_flag, 12);
        }
      }
      if (!few || warp == 0) {
        pl.pos[t] = pos;
        pl.slot[t] = slot;
      }
    }
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const int w_most = (int)__reduce_max_sync(0xffffffffu, (unsigned)n);
    if (few) {
      before = __shfl_sync(0xffffffffu, sum, 31);
      most = w_most;
      if (warp == 0 && t < tokens) pl.cum[t + 1] = sum;
      break;
    }
    if (lane == 31) scan[warp] = sum;
    if (lane == 0) widest[warp] = w_most;
    __syncthreads();
    int base = before;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w < warp) base += scan[w];
      before += scan[w];
      most = max(most, widest[w]);
    }
    if (t < tokens) pl.cum[t + 1] = base + sum;
    __syncthreads();
  }
  if (tid == 0) pl.cum[0] = 0;
  if (tid < NW) front[tid] = rear[tid] = -1;
  __syncthreads();
  const int all = before * segs, per = max(NW, sp.by_grid(all + sp.grid - 1));
  int block0 = blockIdx.x * per, block_n = min(per, all - block0);
  Walk w;
  // (Few short segments: a block each, so that blocks need not wait for one another's sums.)
  const bool one_each = tokens * segs <= sp.grid && most <= SHORT * NW;
  if (one_each) {
    w.tok = sp.by_segs(blockIdx.x);
    w.seg = blockIdx.x - w.tok * segs;
    w.tiles = block_n = w.tok < tokens ? pl.cum[w.tok + 1] - pl.cum[w.tok] : 0;
    if (block_n) block0 = pl.cum[w.tok] * segs + w.seg * block_n;
  }
  // (Many short ones: whole segments to a block, those that begin in its run, for the same reason; not where most blocks would have none.)
  if (!one_each && most <= ALIGNED * NW && most <= 2 * per) {
    const int at = block0 + (lane & 1) * per;
    int begin = min(at, all);
    if (at < all) {
      const Walk x = walk_to(at, pl, segs, sp.by_segs, tokens);
      if (x.tile) begin = at + x.tiles - x.tile;
    }
    block0 = __shfl_sync(0xffffffffu, begin, 0);
    block_n = __shfl_sync(0xffffffffu, begin, 1) - block0;
  }
  if (block_n <= 0) return;

  // ---- this warp's run
  const int each = block_n / NW, more = block_n - each * NW, run0 = block0 + each * warp + min(warp, more), count = each + (warp < more);      // (warps without tiles are the last)
  unsigned char *ring = smem + warp * S::RING;
  if (count > 0) {
    if (one_each) w.tile = run0 - block0;
    else w = walk_to(run0, pl, segs, sp.by_segs, tokens);
    Walk ahead = w;
    // Rows of SIZE bytes; the 16-byte runs of a row are exchanged so that the lanes that read together hit different banks: run c of key row r lies at c ^ 4 (r & 1), of value row
    // r at c ^ (r & 6) (rows of 64 bytes: keys as they are, values at c ^ (r / 2 & 3)).  A copy's 32 lanes have neighbouring runs of ROW_LANES each: 512 bytes that lie together.
    constexpr int ROW_LANES = SIZE / 16;
    const int row_in = lane / ROW_LANES, run_in = lane % ROW_LANES;
    const uint32_t ring_s = smem_addr(ring), k_in = row_in * SIZE + ((run_in ^ (SIZE == 64 ? 0 : (row_in & 1) << 2)) << 4),
                   v_in = row_in * SIZE + ((run_in ^ (SIZE == 64 ? row_in >> 1 & 3 : row_in & 6)) << 4);
    const int k_at0 = g * SIZE + ((tg ^ (SIZE == 64 ? 0 : (g & 1) << 2)) << 4);
    const int v_at0 = 2 * tg * SIZE + (SIZE == 64 ? (((g >> 1) ^ tg) << 4) + (g & 1) * 8 : (g ^ 2 * tg) << 4);
    // copies: a tile a call, STAGES of them before the first is used and then one behind each.  A lane knows the page and the row in it of one of the next 32 groups of 16 positions.
    int ahead_at = 0, stage_in = 0, listed = 0, list_end = 0, page_l = 0, row_l = 0, k_l = 0, v_l = 0, s_l = 0;
    uint32_t whole_l = 0;        // groups that are there as a whole
    auto list = [&]() {
      const int pos = pl.pos[ahead.tok], first = (p.window > 0 ? max(0, pos - p.window + 1) : 0) / KT;
      const int at = (first + ahead.tile) * KT + lane * 16, pg = at <= pos ? sp.by_page(at) : 0;
      row_l = at <= pos ? at - pg * p.c.page : -1;      // (-1: behind the last position)
      page_l = at <= pos ? p.c.page_table[(size_t)pl.slot[ahead.tok] * p.c.max_pages + pg] : 0;
      listed = ahead_at;       // (nothing waits for the page yet: the queries are asked for behind it)
      list_end = ahead_at + min(32 / GROUPS, ahead.tiles - ahead.tile);
      const int kvh = sp.by_chunks(ahead.seg);       // this lane's first bytes and scale of a page, but for the row
      k_l = (kvh * p.c.page + row_in) * dim + 16 * run_in;
      v_l = G * p.c.page * dim + (kvh * p.c.page + row_in) * vdim + 16 * run_in;
      s_l = ((lane >> 4) * G + kvh) * p.c.page + (lane & 15);
    };
    list();
    auto fetch = [&]() {
      if (ahead_at < count) {
        if (ahead_at >= list_end) list();      // (a segment's first tile, or the list has been used up)
        const int at = (ahead_at - listed) * GROUPS;
        if (at == 0) whole_l = __ballot_sync(0xffffffffu, FULL && row_l >= 0 && page_l >= 0);
        const bool whole = (whole_l >> at & ((1 << GROUPS) - 1)) == (1 << GROUPS) - 1;
        const uint32_t st = ring_s + stage_in * S::STAGE;
        auto v_to = [&](uint32_t st_v, int j) { return (SIZE == 128 ? st_v ^ (j & 1) << 6 : SIZE == 256 ? st_v ^ (2 * j & 6) << 4 : st_v) + j * 512; };
        if (whole) {
#pragma unroll
          for (int u = 0; u < GROUPS; ++u) {
            const int page = __shfl_sync(0xffffffffu, page_l, at + u), row = __shfl_sync(0xffffffffu, row_l, at + u);
            const unsigned char *base = p.c.pool + (size_t)(uint32_t)page * p.c.page_bytes, *k = base + (k_l + row * SIZE), *v = base + (v_l + row * SIZE);
            const uint32_t st_k = st + u * (16 * SIZE) + k_in, st_v = st + S::ROWS + u * (16 * SIZE) + v_in;
#pragma unroll
            for (int j = 0; j < S::COPIES; ++j) copy_whole<16>(st_k + j * 512, k + j * 512);
#pragma unroll
            for (int j = 0; j < S::COPIES; ++j) copy_whole<16>(v_to(st_v, j), v + j * 512);
            copy_whole<4>(st + 2 * S::ROWS + u * 128 + lane * 4, p.c.scales + (size_t)(uint32_t)page * (2 * G * p.c.page) + (s_l + row));
          }
        } else {
#pragma unroll 1
          for (int u = 0; u < GROUPS; ++u) {
            int page = __shfl_sync(0xffffffffu, page_l, at + u);
            const int row = __shfl_sync(0xffffffffu, row_l, at + u);
            if (page < 0) {        // (one whose positions lie in front of the window may be gone: a tile has others of its own, and masks these)
              const int pos = pl.pos[ahead.tok], begin = p.window > 0 ? max(0, pos - p.window + 1) : 0, at0 = (begin / KT + ahead.tile) * KT + 16 * u;
              if (at0 + 15 >= begin && p.error_flag) atomicExch(p.error_flag, 12);
              page = 0;
            }
            const unsigned char *base = p.c.pool + (size_t)page * p.c.page_bytes, *k = base + (k_l + row * dim), *v = base + (v_l + row * vdim);
            const uint32_t st_k = st + u * (16 * SIZE) + k_in, st_v = st + S::ROWS + u * (16 * SIZE) + v_in;
            const bool k_here = row >= 0 && 16 * run_in < dim, v_here = row >= 0 && 16 * run_in < vdim;
            constexpr int AT_ONCE = 512 / SIZE;      // rows of a copy
#pragma unroll
            for (int j = 0; j < S::COPIES; ++j) copy_async<16>(st_k + j * 512, k_here ? k + j * AT_ONCE * dim : base, k_here);
#pragma unroll
            for (int j = 0; j < S::COPIES; ++j) copy_async<16>(v_to(st_v, j), v_here ? v + j * AT_ONCE * vdim : base, v_here);
            copy_async<4>(st + 2 * S::ROWS + u * 128 + lane * 4, row >= 0 ? p.c.scales + (size_t)page * (2 * G * p.c.page) + (s_l + row) : p.c.scales, row >= 0);
          }
        }
        ++ahead_at;
        ++ahead.tile;
        settle(ahead, pl, segs, tokens);
        if (++stage_in == STAGES) stage_in = 0;
      }
      copies_end();       // (the groups are counted)
    };

    int done = 0, stage = 0;
    while (done < count) {      // segment after segment
      const int here = min(count - done, w.tiles - w.tile), tok = w.tok;      // tiles of this segment that are the warp's
      const int kvh = sp.by_chunks(w.seg), chunk = w.seg - kvh * sp.chunks, head0 = kvh * qpk + chunk * HEADS, heads = min(HEADS, qpk - chunk * HEADS);
      const int pos = pl.pos[tok], begin = p.window > 0 ? max(0, pos - p.window + 1) : 0;
      float O[MT][4], R[2] = {-INFINITY, -INFINITY}, L[2] = {0.f, 0.f};
#pragma unroll
      for (int j = 0; j < MT; ++j) O[j][0] = O[j][1] = O[j][2] = O[j][3] = 0.f;
      // q as B operand: lane (g, tg) holds head g's dimensions 64 i + 16 tg + .. of the byte runs that it reads of the keys.  int8: three parts of 8 bits of (127 2^14 / the row's largest) q;
      // E4M3: fp16, after a power of two, in QPARTS parts.
      uint32_t qf[QPARTS][NK * 4][QREGS];
      float by[2];          // factors of the scores of heads 2 tg and 2 tg + 1
      {
        uint32_t x[NK][16], most = 0;           // (in the order of bits: NaN above infinity)
        const size_t at = (size_t)(sp.tok0 + tok) * p.q_ld + (size_t)(head0 + g) * dim + 16 * tg;
#pragma unroll
        for (int i = 0; i < NK; ++i) load16(sp.q, at + 64 * i, sp.dtype, sp.q_whole, g < heads ? dim - 64 * i - 16 * tg : 0, x[i]);
        if (done == 0) {        // (the first segment's queries are asked for before all tiles: they would come behind them)
#pragma unroll 1
          for (int s = 0; s < STAGES; ++s) fetch();
        }
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          floats16(x[i], sp.dtype, sp.q_whole);
#pragma unroll
          for (int j = 0; j < 16; ++j) most = max(most, x[i][j] & 0x7fffffffu);
        }
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        float unit;
        if constexpr (E4M3) {
          // the power of two at or below the largest element (1 for a row of zeros, infinities or NaN; within 2^-120 .. 2^120, so that its reciprocal is a number)
          const uint32_t e = most >> 23, f = most == 0 || e == 255 ? 127u : min(max(e, 7u), 247u);
          const float turn = __uint_as_float((254u - f) << 23);
          unit = __uint_as_float(f << 23);
#pragma unroll
          for (int i = 0; i < NK; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int o = 0; o < 2; ++o) {
                const float a = __uint_as_float(x[i][4 * c + 2 * o]) * turn, b = __uint_as_float(x[i][4 * c + 2 * o + 1]) * turn;
                qf[0][4 * i + c][o % QREGS] = pack2(a, b);
                if constexpr (QPARTS == 2) {
                  const float2 h = unpack2(qf[0][4 * i + c][o % QREGS]);
                  qf[QPARTS - 1][4 * i + c][o % QREGS] = pack2(a - h.x, b - h.y);
                }
              }
        } else {
          // v = round((127 2^14 / top) x) as digits 2^14 hi + 2^7 mid + lo, mid and lo in -64 .. 63: those of v + 64 + 64 2^7, less 64.  (1.5 2^23 is added in fp32: the sum's lowest bits are v.)
          const float top = fmaxf(__uint_as_float(most), 0x1p-100f), turn = 127.f * 16384.f / top;
          unit = __uint_as_float(most) == 0.f ? 0.f : most >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : top / (127.f * 16384.f);
#pragma unroll
          for (int i = 0; i < NK; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t v[4], part[3];
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = __float_as_uint(fmaf(__uint_as_float(x[i][4 * c + e]), turn, 12582912.f)) + (64u + (64u << 7) - 0x4B400000u);
#pragma unroll
              for (int q = 0; q < 3; ++q) {       // bits 0 .. 6, 7 .. 13 and 14 .. 21 as byte 0, 1 and 2
                const uint32_t sel = q == 0 ? 0x0040u : q == 1 ? 0x0051u : 0x0062u, sh = q;
                part[q] = __byte_perm(__byte_perm(v[0] << sh, v[1] << sh, sel), __byte_perm(v[2] << sh, v[3] << sh, sel), 0x5410);
              }
              qf[0][4 * i + c][0] = part[2];
#pragma unroll
              for (int q = 1; q < QPARTS; ++q) qf[q][4 * i + c][0] = (((part[2 - q] & 0x7f7f7f7fu) | 0x80808080u) - 0x40404040u) ^ 0x80808080u;
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) by[h] = __shfl_sync(0xffffffffu, unit, 8 * tg + 4 * h) * p.scale;     // (lanes 8 tg and 8 tg + 4 have their rows)
      }
      const float log2e = 1.4426950408889634f;
      if (!(p.softcap > 0.f)) { by[0] *= log2e; by[1] *= log2e; }
      int key0 = (begin / KT + w.tile) * KT;
      for (int t = 0; t < here; ++t, key0 += KT) {
        copies_left<STAGES - 1>();
        __syncwarp();
        const unsigned char *st = ring + stage * S::STAGE;
        const float *sc = reinterpret_cast<const float *>(st + 2 * S::ROWS);
        float x[GROUPS][4];
#pragma unroll
        for (int u = 0; u < GROUPS; ++u) {
          float c[2][4];
          int n[3][4];
#pragma unroll
          for (int i = 0; i < NK; ++i) {
            const unsigned char *at = st + u * (16 * SIZE) + (k_at0 ^ (i & 1) << 6) + (i >> 1) * 128;
            const uint4 a = *reinterpret_cast<const uint4 *>(at), b = *reinterpret_cast<const uint4 *>(at + 8 * SIZE);
            const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w};
            if constexpr (E4M3) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint32_t a0, a1, a2, a3;
                asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h;}" : "=r"(a0), "=r"(a2) : "r"(wa[k]));
                asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h;}" : "=r"(a1), "=r"(a3) : "r"(wb[k]));
#pragma unroll
                for (int q = 0; q < QPARTS; ++q) {
                  if (i == 0 && k < 2 && q == 0) mma_first(c[k & 1], a0, a1, a2, a3, qf[q][4 * i + k][0], qf[q][4 * i + k][QREGS - 1]);
                  else mma16816(c[k & 1], a0, a1, a2, a3, qf[q][4 * i + k][0], qf[q][4 * i + k][QREGS - 1]);
                }
              }
            } else {
#pragma unroll
              for (int k = 0; k < 4; k += 2)
#pragma unroll
                for (int q = 0; q < QPARTS; ++q) {
                  if (i == 0 && k == 0) mma_s8_first(n[q % 3], wa[k], wb[k], wa[k + 1], wb[k + 1], qf[q][4 * i + k][0], qf[q][4 * i + k + 1][0]);
                  else mma_s8(n[q % 3], wa[k], wb[k], wa[k + 1], wb[k + 1], qf[q][4 * i + k][0], qf[q][4 * i + k + 1][0]);
                }
            }
          }
          const float ks[2] = {sc[u * 32 + g], sc[u * 32 + 8 + g]};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float s = E4M3 ? c[0][e] + c[1][e] : fmaf((float)n[0][e], 16384.f, fmaf((float)n[1][e], 128.f, (float)n[2][e]));
            x[u][e] = s * (ks[e >> 1] * by[e & 1]);
          }
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
        const bool border = key0 < begin || key0 + KT > pos + 1;
        if (border) {
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
          uint32_t wf[2][2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t hi = pack2(x[u][2 * r], x[u][2 * r + 1]);
            wf[0][r] = turn8x8(hi);
            const float2 f = unpack2(hi);
            wf[1][r] = turn8x8(pack2(x[u][2 * r] - f.x, x[u][2 * r + 1] - f.y));
          }
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            uint32_t v[4][VB / 4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const unsigned char *at = st + S::ROWS + (u * 16 + (r & 1) + 8 * (r >> 1)) * SIZE + v_at0 + i * 128;
              if constexpr (VB == 16) {
                const uint4 y = *reinterpret_cast<const uint4 *>(at);
                v[r][0] = y.x; v[r][1] = y.y; v[r][VB / 4 - 2] = y.z; v[r][VB / 4 - 1] = y.w;
              } else {
                const uint2 y = *reinterpret_cast<const uint2 *>(at);
                v[r][0] = y.x; v[r][1] = y.y;
              }
              const int key = key0 + 16 * u + 2 * tg + (r & 1) + 8 * (r >> 1);
              if (E4M3 && border && (key < begin || key > pos)) {      // (whatever lies there may be NaN)
#pragma unroll
                for (int k = 0; k < VB / 4; ++k) v[r][k] = 0;
              }
            }
#pragma unroll
            for (int k = 0; k < VB / 4; ++k)
#pragma unroll
              for (int half = 0; half < 2; ++half) {     // dimensions 4 k + 2 half and the next, of keys (0, 1) and (2, 3)
                uint32_t a0, a1, a2, a3;
                widen<E4M3>(v[0][k], v[1][k], half, a0, a1);
                widen<E4M3>(v[2][k], v[3][k], half, a2, a3);
#pragma unroll
                for (int q = 0; q < 2; ++q) mma16816(O[i * 8 + 2 * k + half], a0, a1, a2, a3, wf[q][0], wf[q][1]);
              }
          }
        }
        __syncwarp();      // the scales have been read by all lanes
        if (++stage == STAGES) stage = 0;
        fetch();           // (to the stage that was used)
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
          const float f = 1.f / L[h];
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
        if (g == 0) {
          ml[end ? warp : NW + warp][2 * tg] = make_float2(R[0], L[0]);
          ml[end ? warp : NW + warp][2 * tg + 1] = make_float2(R[1], L[1]);
        }
        if (lane == 0) (end ? rear : front)[warp] = tok * segs + w.seg;
      }
      w.tile += here;
      settle(w, pl, segs, tokens);
    }
    copies_left<0>();
  }
  __syncthreads();

  // ---- pieces of a segment come together: the rears of some warps and the front of the next.  (Whoever has the block's last tile, the others wait for this: few instructions one after
  // the other.)  First their shares, a warp per head and a lane per piece ...
  static_assert(2 * NW <= 32 && NW >= HEADS, "a lane per piece, a warp per head");
  if (warp < HEADS) {
    const int id = lane < NW ? rear[lane] : lane < 2 * NW ? front[lane - NW] : -1;
    const float2 x = ml[min(lane, 2 * NW - 1)][warp];
    const int key = __float_as_int(x.x), most_key = __reduce_max_sync(__match_any_sync(0xffffffffu, id), key ^ (key >> 31 & 0x7fffffff));      // (floats in the order of whole numbers)
    const float r = __int_as_float(most_key ^ (most_key >> 31 & 0x7fffffff)), f = x.x == r ? 1.f : exp2_fast(x.x - r);
    if (lane < 2 * NW) {
      share[lane][warp] = make_float2(f, x.y * f);
      top[lane][warp] = r;
    }
  }
  __syncthreads();
  // ... then the sums, a unit of four floats a lane at a time, dealt out to the warps.  What is not the block's alone goes where the others find it.
  auto leave = [&](const float4 &o, float l0, float l1, int id, int j) {
    const int tok = sp.by_segs(id), seg = id - tok * segs, kvh = sp.by_chunks(seg), chunk = seg - kvh * sp.chunks, heads = min(HEADS, qpk - chunk * HEADS);
    const int d = VB * g + 128 * (j / 8) + 2 * (j % 8);
    const size_t at = (size_t)(sp.tok0 + tok) * p.out_ld + (size_t)(kvh * qpk + chunk * HEADS + 2 * tg) * vdim + d;
    if (d < vdim) store_sums(sp.out, at, vdim, sp.dtype, heads - 2 * tg, o, l0, l1);
  };
  const int rear_l = lane < NW ? rear[lane] : -1, front_l = lane < NW ? front[lane] : -1;
  int unit = 0, open0 = -1, open1 = -1;       // the segments that begin before the block's run, and that end behind it
  for (int w0 = -1; w0 < NW;) {               // (-1: what began before the block and ends in its first warp; every other front belongs to the rears before it)
    const int id = __shfl_sync(0xffffffffu, w0 < 0 ? front_l : rear_l, max(w0, 0));
    const uint32_t rears = __ballot_sync(0xffffffffu, rear_l == id), fronts = __ballot_sync(0xffffffffu, front_l == id);      // (rears of one segment are neighbours)
    if (id < 0) { ++w0; continue; }
    const int tok = sp.by_segs(id), tiles = pl.cum[tok + 1] - pl.cum[tok], tile0 = pl.cum[tok] * segs + (id - tok * segs) * tiles;
    const bool alone = tile0 >= block0 && tile0 + tiles <= block0 + block_n;
    const int side = tile0 >= block0;
    if (!alone) (side ? open1 : open0) = id;
    float *part = sp.parts + ((size_t)blockIdx.x * 2 + side) * S::PIECE;
    const int fw = __ffs(fronts) - 1, r0 = rears ? __ffs(rears) - 1 : 0, r1 = 32 - __clz(rears);
#pragma unroll 1
    for (int j = 0; j < MT; ++j, ++unit) {
      if (unit % NW != warp) continue;
      float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
      float l0 = 0.f, l1 = 0.f;
      if (fw >= 0) {
        const float4 o = __ldcg(reinterpret_cast<const float4 *>(sp.heads + ((size_t)blockIdx.x * NW + fw) * S::PIECE) + j * 32 + lane), f = *reinterpret_cast<const float4 *>(&share[NW + fw][2 * tg]);
        r = make_float4(o.x * f.x, o.y * f.z, o.z * f.x, o.w * f.z);
        l0 = f.y; l1 = f.w;
      }
#pragma unroll 2
      for (int k = r0; k < r1; ++k) {
        const float4 o = reinterpret_cast<const float4 *>(smem + k * S::RING)[j * 32 + lane], f = *reinterpret_cast<const float4 *>(&share[k][2 * tg]);
        r.x += o.x * f.x; r.y += o.y * f.z; r.z += o.z * f.x; r.w += o.w * f.z;
        l0 += f.y; l1 += f.w;
      }
      if (alone) {
        leave(r, l0, l1, id, j);
      } else {
        __stcg(reinterpret_cast<float4 *>(part) + j * 32 + lane, r);
        if (j == 0 && g == 0) {
          const int any = rears ? __ffs(rears) - 1 : NW + fw;
          __stcg(reinterpret_cast<float4 *>(part + MT * 128) + tg, make_float4(top[any][2 * tg], l0, top[any][2 * tg + 1], l1));
        }
      }
    }
    w0 = w0 < 0 ? 0 : 32 - __clz(rears);
  }
  if (open0 < 0 && open1 < 0) return;
  // ---- ... and the last block of a segment to come adds them up, in their order
  __threadfence();
  __syncthreads();
  if (tid < 2) {
    const int id = tid ? open1 : open0;
    parts[tid] = 0;
    if (id >= 0) {
      const int tok = sp.by_segs(id), tiles = pl.cum[tok + 1] - pl.cum[tok], tile0 = pl.cum[tok] * segs + (id - tok * segs) * tiles, b0 = tile0 / per, n = (tile0 + tiles - 1) / per - b0 + 1;
      if (atomicAdd(sp.counters + id, 1) == n - 1) {
        sp.counters[id] = 0;
        first_block[tid] = b0;
        parts[tid] = n;
      }
    }
    __threadfence();
  }
  __syncthreads();
  // (Of both segments at once.  Shares first, a warp per head and a lane per part.)
  if (!parts[0] && !parts[1]) return;
  auto part_of = [&](int side, int i) { return sp.parts + ((size_t)(first_block[side] + i) * 2 + (i == 0)) * S::PIECE; };     // (a segment begins in its first block)
  float2 *shares = reinterpret_cast<float2 *>(smem);      // [side][grid][head]: the pieces in shared memory have been used
  if (warp < HEADS) {
#pragma unroll 1
    for (int side = 0; side < 2; ++side) {
      const int n = parts[side];
      float m = -INFINITY;
#pragma unroll 1
      for (int i = lane; i < n; i += 32) m = fmaxf(m, __ldcg(reinterpret_cast<const float2 *>(part_of(side, i) + MT * 128) + warp).x);
      m = warp_max(m);
#pragma unroll 1
      for (int i = lane; i < n; i += 32) {
        const float2 x = __ldcg(reinterpret_cast<const float2 *>(part_of(side, i) + MT * 128) + warp);
        const float f = x.x == m ? 1.f : exp2_fast(x.x - m);
        shares[(side * sp.grid + i) * HEADS + warp] = make_float2(f, x.y * f);
      }
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int n = warp; n < 2 * MT; n += NW) {
    const int side = n >= MT, j = n - side * MT;
    if (!parts[side]) continue;
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
    float l0 = 0.f, l1 = 0.f;
#pragma unroll 4
    for (int i = 0; i < parts[side]; ++i) {
      const float4 o = __ldcg(reinterpret_cast<const float4 *>(part_of(side, i)) + j * 32 + lane), f = *reinterpret_cast<const float4 *>(&shares[(side * sp.grid + i) * HEADS + 2 * tg]);
      r.x += o.x * f.x; r.y += o.y * f.z; r.z += o.z * f.x; r.w += o.w * f.z;
      l0 += f.y; l1 += f.w;
    }
    leave(r, l0, l1, side ? open1 : open0, j);
  }
}

// Any sizes (and 54 times the time of the tensor cores' on 48 sequences of up to 8000 positions): a block per token and head, whose warps take every fourth key each with a running maximum and sum, lanes across the dimensions.
constexpr int PLAIN_WARPS = 4;
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
  const int which = a.cache.fmt != PT_KV8_E4M3 ? 0 : a.dtype == PT_DT_BF16 ? 1 : 2;
  const auto kernel = which == 0 ? attn_kernel<SIZE, FULL, false, 1> : which == 1 ? attn_kernel<SIZE, FULL, true, 1> : attn_kernel<SIZE, FULL, true, 2>;
  static std::atomic<uint64_t> allowed[3];
  constexpr int WARPS = Shape<SIZE>::WARPS, FIXED = WARPS * Shape<SIZE>::RING;
  const cudaError_t e = allow_smem(kernel, FIXED + (3 * MAX_TOKENS + 1) * (int)sizeof(int), allowed[which]);
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
