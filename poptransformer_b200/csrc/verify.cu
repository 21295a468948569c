// Verification of drafted tokens (speculative sampling): which of a tree's tokens the target accepts, and the token behind them.
//
// p = softmax(logits / T) of the row that is reached.  Its children are looked at in order.  When they are independent draws from a draft
// distribution q, child j with token x stands if u q(x) Z_j < r_j(x), with r_0 = p, Z_j = sum r_j and r_{j+1} = max(r_j - Z_j q, 0): the part of
// p that q has not covered.  Since max(max(p - a q, 0) - b q, 0) = max(p - (a + b) q, 0), r_j = max(p - S_j q, 0) with S_j = Z_0 + .. + Z_{j-1}: one
// number tells a row's whole past.  Without q the tokens that were refused leave p.  The last token is the first whose running sum of r exceeds
// u Z.  That the tokens follow the target's distribution whatever the draft is the point of these rules, and it holds as far as sums and
// residuals are exact: p - q cancels, and a step of the running sum can be 1e-6 of Z while a vocabulary of fp32 roundings drifts by 1e-7.
// They are kept in 64 bits, of weights that are right to 2^-42.
//
// A cluster of blocks has one sequence and walks down its path: it reads only the rows that the path reaches, each once.  Every block has a slice of the
// vocabulary, every warp a part of the slice in order, whose weights stay in shared memory in 64 bits.  A part's weights are 2^(z - K), z = logit log2(e) / T and K
// the whole number above the part's largest z: parts are brought together by adding to exponents, which costs and loses nothing.  With the sums of the parts
// known the drawing is a search: block, warp, then 32 tokens at a time.  Where every row has one child (a chain) the rows' sums come first, all of them
// without a meeting in between, and the tests of all children at once; the walk then begins at the last row that stands (32 chains of 6 over 50257 tokens:
// 70 us walked from the root).  What bounds it is the way down: per row the time of a load, of the 64-bit
// arithmetic in line (a dependent multiply-add takes several times as long as a 32-bit one) and of a meeting of the cluster; in large batches the instructions (64 a token, 15
// of them in 64 bits: those 32 chains take 43 us, of which memory needs 6).  One greedy chain of 5 over 32000 tokens takes 9.9 us, 16 trees of 32 over 65024 29.5.
#include <type_traits>

#include "elem.cuh"
#include "mbarrier.cuh"

namespace pt {
namespace vf {

// Warps of the rows, and one more that looks up the children meanwhile.
constexpr int WARPS = 16, ROW_THREADS = WARPS * 32, THREADS = ROW_THREADS + 32, MAX_BLOCKS = 16, MAX_ROWS = 512, CHAIN = 16;      // CHAIN: rows of a chain that are summed first, at most
constexpr int WEIGHT_BYTES = 192 * 1024;

struct Params {
  int n_seq, n_tok, vocab, logits_ld, draft_ld, max_path;
  int blocks, slice, part;      // of a cluster; tokens of a block and of a warp (multiples of 4)
  bool kept;                    // the weights of a slice fit in shared memory
  const int *cu, *token, *parent;
  const void *logits;
  const float *draft, *temperature, *uniform, *uniform_next;
  int *path, *count, *out_token;
  float *logprob;
};

__device__ __forceinline__ float value(float x) { return x; }
__device__ __forceinline__ float value(__half x) { return __half2float(x); }
__device__ __forceinline__ float value(__nv_bfloat16 x) { return __bfloat162float(x); }
// A logit; NaN is no token's.
template <typename T> __device__ __forceinline__ float logit(const T *row, int i) {
  const float x = value(row[i]);
  return x == x ? x : -INFINITY;
}

struct Part {         // of a row: the largest logit, its lowest place, K, and the sum of the weights relative to it
  double sum, k;
  float top;
  int at;
};
struct Shared {
  Part warp[2][WARPS], pair[MAX_BLOCKS / 2];      // warp: by turns, read by the whole cluster; pair: of two blocks
  double block[MAX_BLOCKS];            // the blocks' sums, relative to K of their pair
  Part row[CHAIN][WARPS], row_block[CHAIN], row_all[CHAIN];      // of a chain: the warps', the block's (read by the whole cluster), the rows'
  double part[WARPS], rest[2];         // sums of what is left, of the warps and (by turns) of the block
  struct Kids {                        // the children of a row, as block 0 found them
    int n, row[MAX_ROWS], token[MAX_ROWS];
    float u[MAX_ROWS], logit[MAX_ROWS], q[MAX_ROWS];
  } kids[2];                           // by turns: the others read block 0's while it goes on
  int drawn;
};

// ln(2)^n / n!
__constant__ double kSeries[11] = {1.0, 0.6931471805599453, 0.24022650695910072, 0.05550410866482158, 0.009618129107628477, 0.0013333558146428443, 0.0001540353039338161, 1.5252733804059841e-05, 1.321548679014431e-06, 1.01780860092397e-07, 7.054911620801123e-09};
// A finite float as a double, by its bits: conversions are a quarter as fast as additions.  (0 and what is smaller than 2^-126 becomes something below 2^-126.)
__device__ __forceinline__ double widened(float x) {
  const int b = __float_as_int(x);
  return __hiloint2double((b >> 3 & (int)0x8fffffff) + 0x38000000, b << 29);
}
// 2^(c x - K) for c x <= K: n = the whole number next to c x - K, r = c x - K - n without a rounding but its own, 2^r by its series up to r^10 (|r| <= 1/2: the
// next term is below 2^-42).  0 for x <= least, where c x - K is -1000 or less, which -inf is.  (least is rounded down: floats above it are those above (K - 1000) / c,
// however near that lies to the largest logit.  Fifteen 64-bit operations, of which an SM does 64 a cycle, and no
// table: look-ups at random places of shared memory, or by shuffles, cost more than the terms that they save.)
struct Scale {
  double c, shift;      // 1.5 2^52 - K: the last bit is 1
  float least;
  __device__ __forceinline__ Scale(double c, double k) : c(c), shift(6755399441055744.0 - k) { least = __double2float_rd((k - 1000.0) / c); }
  __device__ __forceinline__ double operator()(float x) const {
    const double v = widened(x), t = fma(v, c, shift), r = fma(v, c, shift - t);
    double e = fma(r, kSeries[10], kSeries[9]);
#pragma unroll
    for (int n = 8; n >= 0; --n) e = fma(r, e, kSeries[n]);
    const int hi = __double2hiint(e) + (__double2loint(t) << 20);
    return __hiloint2double(x > least ? hi : 0, __double2loint(e));      // (what is left without its upper half is below 2^-1000)
  }
};
// 2^d x, d a whole number <= 0, where that is at least 2^-1000 or so.
__device__ __forceinline__ double scaled(double x, double d) { return d > -1000.0 ? x * __hiloint2double((1023 + (int)d) << 20, 0) : 0.0; }
// Weight of a logit: 2^(c x - K), K of the row's largest.  Where that is infinite, or so large (a temperature next to 0) that no other logit's weight would differ from 0,
// the logits that are equal to it share the weight.
struct Weigh {
  double c;
  static __device__ __forceinline__ bool alone(double k) { return fabs(k) > 0x1p40; }
  __device__ __forceinline__ double operator()(float x, double k, float top) const { return alone(k) ? (x == top ? 1.0 : 0.0) : x > -INFINITY ? Scale(c, k)(x) : 0.0; }
  __device__ __forceinline__ double k(float top) const { return top == INFINITY ? 1e300 : top == -INFINITY ? -1e300 : ceil(widened(top) * c); }
  // log of the weight
  __device__ __forceinline__ double log(float x, double k) const { return alone(k) ? 0.0 : fma(widened(x), c, -k) * 0.6931471805599453; }
};
__device__ __forceinline__ double warp_add(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// The largest of a warp's values and the lowest place that has it (the same in all lanes).
__device__ __forceinline__ void warp_top(float &x, int &at) {
  x += 0.f;                                           // (-0 is 0)
  const int b = __float_as_int(x), key = b ^ (b >> 31 & 0x7fffffff), top = __reduce_max_sync(0xffffffffu, key);      // (ordered like the floats; -0 below 0)
  at = __reduce_min_sync(0xffffffffu, key == top ? at : 0x7fffffff);
  x = __int_as_float(top ^ (top >> 31 & 0x7fffffff));
}
// An address of this block's shared memory, in block `rank` of the cluster.
template <typename V> __device__ __forceinline__ const V *in_block(const V *p, int rank) {
  uint64_t a;
  asm volatile("mapa.u64 %0, %1, %2;" : "=l"(a) : "l"((uint64_t)p), "r"(rank));
  return reinterpret_cast<const V *>(a);
}

// Four values from an address on a boundary of four, or -inf if not `there`: loads without a branch, so that several are under way.
__device__ __forceinline__ void load4(const float *p, bool there, float (&v)[4]) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\tmov.f32 %0, 0fff800000;\n\tmov.f32 %1, 0fff800000;\n\tmov.f32 %2, 0fff800000;\n\tmov.f32 %3, 0fff800000;\n\t"
               "@q ld.global.nc.v4.f32 {%0, %1, %2, %3}, [%4];\n\t}"
               : "=&f"(v[0]), "=&f"(v[1]), "=&f"(v[2]), "=&f"(v[3])
               : "l"(p), "r"((int)there));
}
template <typename T> __device__ __forceinline__ void load4(const T *p, bool there, float (&v)[4]) {
  constexpr uint32_t least = std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  uint2 r;
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %3, 0;\n\tmov.b32 %0, %4;\n\tmov.b32 %1, %4;\n\t@q ld.global.nc.v2.b32 {%0, %1}, [%2];\n\t}"
               : "=&r"(r.x), "=&r"(r.y)
               : "l"(p), "r"((int)there), "n"(least));
  const T *h = reinterpret_cast<const T *>(&r);
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = value(h[k]);
}

// What a warp does with its part lo .. hi - 1 of a row (from lo on in fours that lie on their boundaries in memory; places below 0 do not exist): the largest logit,
// weights and their sum.  KEEP: the logits are kept in `logits` meanwhile (room for the part), and with `weights` the weights behind it.  PLACE: the largest one's place.
template <typename T, bool KEEP, bool PLACE> __device__ __forceinline__ Part sum_part(const T *row, int lo, int hi, int vocab, const Weigh &weigh, float *logits, double *weights) {
  const int lane = threadIdx.x & 31;
  float top = -INFINITY;
  int at = 0x7fffffff;
  constexpr int AHEAD = 4;
  // (Fours are inside a part or outside, but for those at the ends of the row.)
  const bool ends = lo < 0 || hi == vocab;
  const int whole = hi == vocab ? lo + (hi - lo) / 4 * 4 : hi;
  for (int i0 = lo; i0 < hi; i0 += AHEAD * 128) {
    float v[AHEAD][4];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int i = i0 + u * 128 + lane * 4;
      load4(row + i, i < whole && i >= 0, v[u]);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int i = i0 + u * 128 + lane * 4;
      if (i0 + u * 128 >= hi) break;                  // (uniform)
      if (ends && (i < 0 || i >= whole)) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (i + k >= 0 && i + k < hi) v[u][k] = value(row[i + k]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[u][k] = fmaxf(v[u][k], -INFINITY);          // (NaN)
        if (PLACE) {
          if (v[u][k] > top) { top = v[u][k]; at = i + k; }
        } else {
          top = fmaxf(top, v[u][k]);
        }
      }
      if (KEEP && i < hi) *reinterpret_cast<float4 *>(logits + i - lo) = make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
    }
  }
  warp_top(top, at);
  const double k = weigh.k(top);
  const Scale scale(weigh.c, k);
  if (KEEP) __syncwarp();
  auto at_place = [&](int i) { return KEEP ? logits[i - lo] : i >= 0 ? logit(row, i) : -INFINITY; };
  double sum = 0.0;
  if (!Weigh::alone(k)) {
    // (a token a lane: few lanes idle at the end of a part)
    int i = lo + lane;
    for (; i + 96 < hi; i += 128) {
      double w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) w[u] = scale(at_place(i + 32 * u));
      if (KEEP && weights) {
#pragma unroll
        for (int u = 0; u < 4; ++u) weights[i + 32 * u - lo] = w[u];
      }
      sum += (w[0] + w[1]) + (w[2] + w[3]);
    }
    for (; i < hi; i += 32) {
      const double w = scale(at_place(i));
      if (KEEP && weights) weights[i - lo] = w;
      sum += w;
    }
  } else {
    for (int i = lo + lane; i < hi; i += 32) {
      const double w = top > -INFINITY && at_place(i) == top ? 1.0 : 0.0;
      if (KEEP && weights) weights[i - lo] = w;
      sum += w;
    }
  }
  return Part{warp_add(sum), k, top, at};
}

template <typename T> __global__ void __launch_bounds__(THREADS, 2) verify_kernel(const Params p) {
  early_start();
  extern __shared__ __align__(16) double kept[];      // [WARPS part] weights, then as many logits
  __shared__ Shared sm;
  const int s = blockIdx.x, rank = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r0 = p.cu[s], all = p.cu[s + 1] - r0, n = r0 >= 0 && r0 + all <= p.n_tok ? min(all, MAX_ROWS) : 0;
  int *path = p.path + (size_t)s * p.max_path, *said = p.out_token + (size_t)s * p.max_path;
  float *lp = p.logprob ? p.logprob + (size_t)s * p.max_path : nullptr;
  const double t = p.temperature ? (double)p.temperature[s] : 0.0, log2e = 1.4426950408889634;
  const Weigh weigh{t > 0.0 ? log2e / t : log2e};
  const bool greedy = !(t > 0.0);
  double *mine = kept + warp * p.part;
  float *logits = reinterpret_cast<float *>(kept + WARPS * p.part) + warp * p.part;
  auto part_of = [&](const T *row, int lo, int hi, bool keep, double *weights) {
    if (greedy) return keep ? sum_part<T, true, true>(row, lo, hi, p.vocab, weigh, logits, weights) : sum_part<T, false, true>(row, lo, hi, p.vocab, weigh, logits, weights);
    return keep ? sum_part<T, true, false>(row, lo, hi, p.vocab, weigh, logits, weights) : sum_part<T, false, false>(row, lo, hi, p.vocab, weigh, logits, weights);
  };
  auto row_of = [&](int r) { return reinterpret_cast<const T *>(p.logits) + (size_t)(r0 + r) * p.logits_ld; };
  // This warp's tokens of a row.  (Counted from the boundary of four in memory in front of it; the row's address is one of T.)
  auto slice_of = [&](const T *row) { return rank * p.slice - (int)((uintptr_t)row / sizeof(T) & 3); };
  auto end_of = [&](int slice, int lo, int part) { return max(lo, min(min(lo + part, slice + p.slice), p.vocab)); };
  int done = 0, turn = 0, at = n > 0 ? 0 : -1;
  const int chain = p.parent || n < 3 ? 0 : min(min(n, CHAIN), p.max_path);
  if (chain > 2) {
    // ---- a chain: the sums of its rows, each cut into as many parts as there are warps, or, where those would be small, into fewer: all rows at once then
    const int cuts = p.part >= 256 ? WARPS : max(1, WARPS / chain), piece = cuts == WARPS ? p.part : (p.slice / 4 + cuts - 1) / cuts * 4;
    float x_top = -INFINITY, x_u = 0.f, x_q = 1.f;    // lane j of the last warp: row j's child
    int x = -1;
    if (warp < WARPS)
      for (int i = warp; i < chain * cuts; i += WARPS) {
        const int r = i / cuts, c = i - r * cuts;
        const T *row = row_of(r);
        const int slice = slice_of(row), lo = slice + c * piece;
        const Part part = part_of(row, lo, end_of(slice, lo, piece), p.kept && cuts == WARPS, nullptr);
        if (lane == 0) sm.row[r][c] = part;
      }
    else if (lane < chain - 1) {
      x = p.token[r0 + lane + 1];
      if (x < 0 || x >= p.vocab) x = -1;
      if (x >= 0) x_top = logit(row_of(lane), x);
      if (!greedy) {
        x_u = p.uniform[r0 + lane + 1];
        if (p.draft && x >= 0) x_q = p.draft[(size_t)(r0 + lane) * p.draft_ld + x];
      }
    }
    __syncthreads();
    auto join = [&](Part v) {                         // of the warp's lanes
      float top = v.top;
      int best = v.at;
      warp_top(top, best);
      const double k = weigh.k(top);
      return Part{warp_add(scaled(v.sum, v.k - k)), k, top, best};
    };
    const Part none{0.0, -1e300, -INFINITY, 0x7fffffff};
    if (warp < chain) {
      const Part v = join(lane < cuts ? sm.row[warp][lane] : none);
      if (lane == 0) sm.row_block[warp] = v;
    }
    stay_for_cluster();
    if (warp < chain) {
      const Part v = join(lane < p.blocks ? *in_block(&sm.row_block[warp], lane) : none);
      if (lane == 0) sm.row_all[warp] = v;
    }
    __syncthreads();
    // every child against its own row, by block 0; the first one that falls ends the chain
    if (rank == 0 && warp == WARPS) {
      bool ok = false;
      double log_p = 0.0;
      if (x >= 0) {
        const Part v = sm.row_all[lane];
        const double px = v.top > -INFINITY ? weigh(x_top, v.k, v.top) / v.sum : 0.0;
        ok = greedy ? v.top > -INFINITY && x == v.at : (double)x_u * (double)x_q < px;
        log_p = weigh.log(x_top, v.k) - log(v.sum);
      }
      const int stand = __ffs(~__ballot_sync(0xffffffffu, ok)) - 1;
      if (lane < stand) {
        path[lane] = lane;
        said[lane] = x;
        if (lp) lp[lane] = (float)log_p;
      }
      // the largest logit's token follows; one that is drawn needs its row's weights
      const bool over = greedy && (stand < chain - 1 || chain == min(n, p.max_path));
      if (over && lane == 0) {
        const Part v = sm.row_all[stand];
        const bool any = v.top > -INFINITY;
        path[stand] = stand;
        said[stand] = any ? v.at : -1;
        if (lp) lp[stand] = any ? (float)(weigh.log(v.top, v.k) - log(v.sum)) : 0.f;
      }
      if (lane == 0) sm.drawn = over ? -stand - 1 : stand;
    }
    stay_for_cluster();
    const int stand = *in_block(&sm.drawn, 0);
    at = stand < 0 ? -1 : stand;
    done = stand < 0 ? -stand : stand;
    // (nobody writes sm.drawn before the cluster has met again)
  }
  while (at >= 0) {
    const T *row = row_of(at);
    const float *q = greedy || !p.draft ? nullptr : p.draft + (size_t)(r0 + at) * p.draft_ld;
    const int slice = slice_of(row), lo = slice + warp * p.part, hi = warp < WARPS ? end_of(slice, lo, p.part) : lo;
    Shared::Kids &kid = sm.kids[done & 1];
    double my_k = 0.0;
    if (warp < WARPS) {
      // ---- the row
      const Part part = part_of(row, lo, hi, p.kept, mine);
      my_k = part.k;
      if (lane == 0) sm.warp[done & 1][warp] = part;
    } else {
      // ---- children; the first one's row is likely the next
      int k = 0, first = -1;
      if (done + 1 < p.max_path)
        for (int c0 = at + 1; c0 < n; c0 += 32) {
          const int c = c0 + lane;
          const bool is = c < n && (p.parent ? p.parent[r0 + c] : c - 1) == at;
          const unsigned who = __ballot_sync(0xffffffffu, is);
          if (first < 0 && who) {
            first = c0 + __ffs(who) - 1;
            const char *ahead = reinterpret_cast<const char *>(reinterpret_cast<const T *>(p.logits) + (size_t)(r0 + first) * p.logits_ld);
            const size_t a = (size_t)rank * p.slice * sizeof(T), b = (size_t)min((rank + 1) * p.slice, p.vocab) * sizeof(T);      // (three places more or less do not matter)
            for (size_t x = a + lane * 128; x < b; x += 32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(ahead + x));
          }
          if (rank == 0 && is) {
            const int i = k + __popc(who & ((1u << lane) - 1u)), x = p.token[r0 + c];
            const bool in = x >= 0 && x < p.vocab;
            kid.row[i] = c;
            kid.token[i] = in ? x : -1;
            kid.logit[i] = in ? logit(row, x) : -INFINITY;
            if (!greedy) {
              kid.u[i] = p.uniform[r0 + c];
              if (q) kid.q[i] = in ? q[x] : 0.f;
            }
          }
          k += __popc(who);
        }
      if (lane == 0 && rank == 0) kid.n = k;
    }
    stay_for_cluster();
    // ---- the parts of the whole row, two blocks a warp; the children that block 0 found
    if (warp < MAX_BLOCKS / 2) {
      const int b = tid / WARPS;
      Part x{0.0, -1e300, -INFINITY, 0x7fffffff};
      if (b < p.blocks) x = *in_block(&sm.warp[done & 1][tid % WARPS], b);
      float top = x.top;
      int best = x.at;
      warp_top(top, best);
      const double k = weigh.k(top);
      double sum = scaled(x.sum, x.k - k);
#pragma unroll
      for (int o = WARPS / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (tid % WARPS == 0) sm.block[b] = sum;
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      if (lane == 0) sm.pair[warp] = Part{sum, k, top, best};
    } else if (warp == WARPS && rank != 0) {
      const Shared::Kids *head = in_block(&kid, 0);
      const int kids = head->n;
      for (int i = lane; i < kids; i += 32) {
        kid.row[i] = head->row[i]; kid.token[i] = head->token[i]; kid.logit[i] = head->logit[i];
        if (!greedy) kid.u[i] = head->u[i];
        if (q) kid.q[i] = head->q[i];
      }
      if (lane == 0) kid.n = kids;
    }
    __syncthreads();
    // ---- every warp for itself, from the same numbers: the row's largest and sum, and which child stands
    Part whole_row = lane < MAX_BLOCKS / 2 ? sm.pair[lane] : Part{0.0, -1e300, -INFINITY, 0x7fffffff};
    float top = whole_row.top;
    int best = whole_row.at;
    warp_top(top, best);
    const double K = weigh.k(top);
    double total = scaled(whole_row.sum, whole_row.k - K);
#pragma unroll
    for (int o = MAX_BLOCKS / 4; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    total = __shfl_sync(0xffffffffu, total, 0);
    const bool any = top > -INFINITY;
    const double over = 1.0 / total;
    const int kids = any ? kid.n : 0;
    double S = 0.0, Z = 1.0;      // with q: r = max(p - S q, 0); without: Z is what the refused tokens left of p
    int stands = -1, tried = 0;
    auto kid_p = [&](int k) { return kid.token[k] >= 0 ? weigh(kid.logit[k], K, top) * over : 0.0; };
    if (!q)
      for (int k0 = 0; k0 < kids && stands < 0; k0 += 32) {
        const int mine_x = k0 + lane < kids ? kid.token[k0 + lane] : -1;
        double px = 0.0, u = 0.0;
        if (greedy) {
          const unsigned is = __ballot_sync(0xffffffffu, mine_x == best);
          if (is) stands = tried = k0 + __ffs(is) - 1;
          continue;
        }
        if (mine_x >= 0) {
          px = kid_p(k0 + lane);
          u = (double)kid.u[k0 + lane];
        }
        for (int i = 0; i < min(k0 + lane, kids) && k0 + lane < kids; ++i)
          if (kid.token[i] == mine_x) px = 0.0;       // (a token that was refused has no weight left)
        for (int i = 0; i < min(32, kids - k0); ++i) {
          const double pi = __shfl_sync(0xffffffffu, px, i);
          if (__shfl_sync(0xffffffffu, u, i) * Z < pi) { stands = tried = k0 + i; break; }
          Z = fmax(Z - pi, 0.0);      // (below 0 by a rounding, a random number of 1 or more would accept what has no weight)
        }
      }
    if (!q && stands < 0) tried = kids;
    // a token's weight (of this warp's part), and what the refused children left of it
    auto raw = [&](int i) { return p.kept ? scaled(mine[i - lo], my_k - K) : weigh(logit(row, i), K, top); };
    auto of_cluster = [&](double z) {                 // Z = sum over the cluster of what the warps have
      z = warp_add(z);
      turn ^= 1;
      if (lane == 0 && warp < WARPS) sm.part[warp] = z;
      __syncthreads();
      if (warp == 0) {
        const double v = warp_add(lane < WARPS ? sm.part[lane] : 0.0);
        if (lane == 0) sm.rest[turn] = v;
      }
      stay_for_cluster();
      Z = warp_add(lane < p.blocks ? *in_block(&sm.rest[turn], lane) : 0.0);
    };
    bool passed = false;                              // sm.part and sm.rest hold the sums of what is left
    if (q)
      while (tried < kids) {                          // (uniform over the cluster: all go by the same numbers)
        if (kid.token[tried] >= 0 && (double)kid.u[tried] * (double)kid.q[tried] * Z < fmax(kid_p(tried) - S * (double)kid.q[tried], 0.0)) {
          stands = tried;
          break;
        }
        ++tried;
        S += Z;
        double z = 0.0;
#pragma unroll 4
        for (int i = max(lo, 0) + lane; i < hi; i += 32) z += fmax(raw(i) * over - S * (double)q[i], 0.0);
        of_cluster(z);
        passed = true;
      }
    const int next = stands < 0 ? -1 : kid.row[stands];
    int token = next >= 0 ? kid.token[stands] : any && greedy ? best : -1;
    bool writes = rank == 0;                          // the block that knows the token
    if (next < 0 && any && !greedy) {
      // ---- drawing.  `everything`: nothing is left, p itself
      bool everything = passed && !(Z > 0.0);
      auto rest = [&](int i) {
        if (everything) return raw(i);
        if (q) return passed ? fmax(raw(i) * over - S * (double)q[i], 0.0) : raw(i);
        for (int k = 0; k < tried; ++k)
          if (kid.token[k] == i) return 0.0;
        return raw(i);
      };
      if (!q && tried) {
        // (parts without a refused token keep their sums)
        bool has = false;
        for (int k = 0; k < tried; ++k) has |= kid.token[k] >= lo && kid.token[k] < hi;
        double z = 0.0;
        if (has)
          for (int i = max(lo, 0) + lane; i < hi; i += 32) z += rest(i);
        else if (warp < WARPS && lane == 0) z = scaled(sm.warp[done & 1][warp].sum, my_k - K);
        of_cluster(z);
        passed = true;
        everything = !(Z > 0.0);
      }
      const bool left = passed && !everything;        // the sums are those of the last pass, else the row's
      if (!left) Z = total;
      auto block_sum = [&](int b) { return left ? *in_block(&sm.rest[turn], b) : scaled(sm.block[b], sm.pair[b / 2].k - K); };
      auto part_sum = [&](int w) { return left ? sm.part[w] : scaled(sm.warp[done & 1][w].sum, sm.warp[done & 1][w].k - K); };
      const float u = p.uniform_next[s];
      const double want = (u < 1.f ? (double)u : 1.0 - 0x1p-24) * Z;
      // the block, the warp, the token whose running sum exceeds it (where rounding leaves none: the last one with weight)
      auto find = [&](int count, double from, auto sum_of, double &before) {
        const double v = lane < count ? sum_of(lane) : 0.0;
        double upto = v;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += y;
        }
        const unsigned some = __ballot_sync(0xffffffffu, v > 0.0), over_it = __ballot_sync(0xffffffffu, v > 0.0 && from + upto > want);
        const int pick = max(over_it ? __ffs(over_it) - 1 : 31 - __clz(some), 0);      // (one in any case: some block has to write)
        before = from + __shfl_sync(0xffffffffu, upto - v, pick);
        return pick;
      };
      double before, c;
      writes = find(p.blocks, 0.0, block_sum, before) == rank;
      if (writes) {
        const int chosen = find(WARPS, before, part_sum, c);
        if (warp == chosen) {
          int last = -1;
          bool found = false;
          for (int i0 = lo; i0 < hi && !found; i0 += 32) {
            const int i = i0 + lane;
            const double v = i >= 0 && i < hi ? rest(i) : 0.0;
            double upto = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const double y = __shfl_up_sync(0xffffffffu, upto, o);
              if (lane >= o) upto += y;
            }
            const unsigned some = __ballot_sync(0xffffffffu, v > 0.0), over_it = __ballot_sync(0xffffffffu, v > 0.0 && c + upto > want);
            if (some) last = i0 + (over_it ? __ffs(over_it) - 1 : 31 - __clz(some));
            c += __shfl_sync(0xffffffffu, upto, 31);
            found = over_it != 0;
          }
          if (lane == 0) sm.drawn = last;
        }
        __syncthreads();
        token = sm.drawn;
      }
    }
    if (writes && warp == WARPS && lane == 0) {       // (the others are at the next row)
      path[done] = at;
      said[done] = token;
      if (lp) {
        const float x = token >= 0 ? logit(row, token) : 0.f;
        lp[done] = token >= 0 ? (float)(weigh.log(x, K) - log(total)) : 0.f;
      }
    }
    ++done;
    at = next;
  }
  if (rank == 0) {
    for (int i = done + tid; i < p.max_path; i += THREADS) {
      path[i] = said[i] = -1;
      if (lp) lp[i] = 0.f;
    }
    if (tid == 0) p.count[s] = done;
  }
  stay_for_cluster();                                 // nobody reads this block's shared memory any more
}

template <typename T> static int launch(const Params &p, size_t smem, cudaStream_t st) {
  static std::atomic<uint64_t> wide{0}, large{0};
  PT_CUDA(allow_wide_clusters(verify_kernel<T>, wide));
  PT_CUDA(allow_smem(verify_kernel<T>, WEIGHT_BYTES, large));
  PT_CUDA(launch_early(verify_kernel<T>, Grid(dim3(p.n_seq, p.blocks), p.blocks), THREADS, p.kept ? smem : 0, st, p));
  PT_LAUNCH_CHECK("pt_verify_drafts");
  return PT_OK;
}

}  // namespace vf
}  // namespace pt

using namespace pt;

extern "C" int pt_verify_drafts(const pt_verify_args *a, void *stream) {
  PT_REQUIRE(a, "pt_verify_drafts: null args");
  PT_REQUIRE(a->n_seq > 0 && a->n_tok >= 0 && a->vocab > 0 && a->max_path > 0, "pt_verify_drafts: n_seq=%d n_tok=%d vocab=%d max_path=%d", a->n_seq, a->n_tok, a->vocab, a->max_path);
  PT_REQUIRE(a->cu && a->logits && a->token && a->path && a->count && a->out_token, "pt_verify_drafts: null pointer argument");
  PT_REQUIRE(a->dtype == PT_DT_F16 || a->dtype == PT_DT_F32 || a->dtype == PT_DT_BF16, "pt_verify_drafts: type %d (fp16, fp32 or bf16)", a->dtype);
  PT_REQUIRE(a->logits_ld >= a->vocab && (!a->draft || a->draft_ld >= a->vocab), "pt_verify_drafts: row strides %d, %d of %d tokens", a->logits_ld, a->draft_ld, a->vocab);
  PT_REQUIRE(!a->temperature || (a->uniform && a->uniform_next), "pt_verify_drafts: sampling needs uniform and uniform_next");
  vf::Params p{};
  p.n_seq = a->n_seq; p.n_tok = a->n_tok; p.vocab = a->vocab; p.logits_ld = a->logits_ld; p.draft_ld = a->draft_ld; p.max_path = a->max_path;
  p.cu = a->cu; p.token = a->token; p.parent = a->parent; p.logits = a->logits; p.draft = a->draft; p.temperature = a->temperature;
  p.uniform = a->uniform; p.uniform_next = a->uniform_next; p.path = a->path; p.count = a->count; p.out_token = a->out_token; p.logprob = a->logprob;
  // Blocks of a cluster: as many as keep the GPU's SMs busy with two each, of 1024 tokens or more; more where the weights of a slice would not fit.
  int blocks = 1;
  while (blocks < vf::MAX_BLOCKS && (long long)a->n_seq * blocks <= sm_count() && (long long)a->vocab > 1024ll * blocks) blocks *= 2;
  auto slice = [&](int b) { return ceil_div(a->vocab + 3, b * 4) * 4; };
  while (blocks < vf::MAX_BLOCKS && (size_t)slice(blocks) * 12 > vf::WEIGHT_BYTES) blocks *= 2;
  p.blocks = blocks;
  p.slice = slice(blocks);
  p.part = ceil_div(p.slice, vf::WARPS * 4) * 4;
  const size_t smem = (size_t)vf::WARPS * p.part * 12;
  p.kept = smem <= vf::WEIGHT_BYTES;
  return a->dtype == PT_DT_F32 ? vf::launch<float>(p, smem, as_stream(stream)) : a->dtype == PT_DT_F16 ? vf::launch<__half>(p, smem, as_stream(stream))
                                                                                : vf::launch<__nv_bfloat16>(p, smem, as_stream(stream));
}
