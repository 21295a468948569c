// Verification of drafted tokens (speculative sampling): which of a tree's tokens the target accepts, and the token behind them.
//
// p = softmax(logits / T) of the row that is reached.  Its children are looked at in order.  When they are independent draws from a draft
// distribution q, child j with token x stands if u q(x) Z_j < r_j(x), with r_0 = p, Z_j = sum r_j and r_{j+1} = max(r_j - Z_j q, 0): the part of
// p that q has not covered.  Since max(max(p - a q, 0) - b q, 0) = max(p - (a + b) q, 0), r_j = max(p - S_j q, 0) with S_j = Z_0 + .. + Z_{j-1}: one
// number tells a row's whole past.  Without q the tokens that were refused leave p.  The last token is the first whose running sum of r exceeds
// u Z.  That the tokens follow the target's distribution whatever the draft is the point of these rules, and it holds as far as sums and
// residuals are exact: p - q cancels, and a step of the running sum can be 1e-6 of Z while a vocabulary of fp32 roundings drifts by 1e-7.
// They are kept in 64 bits.
//
// A cluster of blocks has one sequence and walks down its path: it reads only the rows that the path reaches, each once.  Every block has a slice of the
// vocabulary, every warp a part of the slice in order, whose weights exp((x - top of the part) / T) stay in shared memory in 64 bits.  With the sums of
// the parts known the drawing is a search: block, warp, then 128 tokens at a time.  What bounds it is the way down: per row the time of a load, two
// reductions and a meeting of the cluster; in large batches memory.  (64-bit multiply-adds are half as many a cycle as 32-bit ones; a weight takes a dozen.)
#include "elem.cuh"
#include "mbarrier.cuh"

namespace pt {
namespace vf {

// Warps of the rows, and one more that looks up the children meanwhile.
constexpr int WARPS = 16, ROW_THREADS = WARPS * 32, THREADS = ROW_THREADS + 32, MAX_BLOCKS = 16, MAX_ROWS = 512, STEP = 128;
constexpr int WEIGHT_BYTES = 192 * 1024;

struct Params {
  int n_seq, n_tok, vocab, logits_ld, draft_ld, max_path;
  int blocks, slice, part;      // of a cluster; tokens of a block and of a warp (multiples of 128)
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

struct Top {          // of a part of a row: the largest logit, its lowest place, the sum of the weights relative to it
  float x;
  int at;
  double sum;
};
struct Shared {
  double table[64];                    // 2^(j / 64)
  Top warp[WARPS], block[2];           // block: by turns, read by the whole cluster
  double part[WARPS], rest[2];         // sums of what is left, of the warps and (by turns) of the block
  double scale[WARPS];                 // of the warps' weights to the row's
  struct Kids {                        // the children of a row, as block 0 found them
    int n, row[MAX_ROWS], token[MAX_ROWS];
    float u[MAX_ROWS], logit[MAX_ROWS], q[MAX_ROWS];
  } kids[2];                           // by turns: the others read block 0's while it goes on
  // what the first warp made of it
  int next, tried, best, drawn;
  float top;
  double total, S, Z;
};

// exp(y) for y <= 0, after Tang (Table-driven implementation of the exponential function in IEEE floating-point arithmetic, 1989): y = (64 m + j) ln 2 / 64 + r,
// exp(y) = 2^m 2^(j / 64) exp(r), |r| <= ln 2 / 128, exp(r) by its series up to r^5 (the next term is below 2^-54).
__device__ __forceinline__ double exp_neg(double y, const double *table) {
  if (!(y > -700.0)) return 0.0;
  const double shift = 6755399441055744.0, t = fma(y, 92.33248261689366, shift), n = t - shift;      // 1.5 2^52; 64 / ln 2
  const int k = __double2loint(t);
  double r = fma(n, -0x1.62e42fef00000p-7, y);      // ln 2 / 64 in two parts, the first of 33 bits
  r = fma(n, -0x1.473de6af278edp-40, r);
  double e = fma(r, 1.0 / 120.0, 1.0 / 24.0);
  e = fma(r, e, 1.0 / 6.0);
  e = fma(r, e, 0.5);
  e = fma(r, e, 1.0);
  e = fma(r, e, 1.0);
  e *= table[k & 63];
  return __hiloint2double(__double2hiint(e) + ((k >> 6) << 20), __double2loint(e));
}
// Weight of logit x relative to `top`; equal infinities share the weight.
__device__ __forceinline__ double weight(float x, float top, double inv_t, const double *table) {
  return x == top ? 1.0 : exp_neg(((double)x - (double)top) * inv_t, table);
}
__device__ __forceinline__ double warp_add(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ void larger(float &x, int &at, float ox, int oat) {
  if (ox > x || (ox == x && oat < at)) { x = ox; at = oat; }
}
// An address of this block's shared memory, in block `rank` of the cluster.
template <typename V> __device__ __forceinline__ const V *in_block(const V *p, int rank) {
  uint64_t a;
  asm volatile("mapa.u64 %0, %1, %2;" : "=l"(a) : "l"((uint64_t)p), "r"(rank));
  return reinterpret_cast<const V *>(a);
}

// Four logits from place i on, -inf from `end` on.
template <typename T> __device__ __forceinline__ void four(const T *row, int i, int end, bool aligned, float (&v)[4]) {
  if (aligned && i + 4 <= end) {
    if constexpr (sizeof(T) == 4) {
      const float4 r = __ldg(reinterpret_cast<const float4 *>(row + i));
      v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
    } else {
      const uint2 r = __ldg(reinterpret_cast<const uint2 *>(row + i));
      const T *h = reinterpret_cast<const T *>(&r);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = value(h[k]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = i + k < end ? value(row[i + k]) : -INFINITY;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (!(v[k] == v[k])) v[k] = -INFINITY;
}

template <typename T> __global__ void __launch_bounds__(THREADS) verify_kernel(const Params p) {
  early_start();
  extern __shared__ __align__(16) double kept[];      // [slice] weights (first: logits)
  __shared__ Shared sm;
  const int s = blockIdx.x, rank = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r0 = p.cu[s], all = p.cu[s + 1] - r0, n = r0 >= 0 && r0 + all <= p.n_tok ? min(all, MAX_ROWS) : 0;
  int *path = p.path + (size_t)s * p.max_path, *said = p.out_token + (size_t)s * p.max_path;
  float *lp = p.logprob ? p.logprob + (size_t)s * p.max_path : nullptr;
  if (tid < 64) sm.table[tid] = exp2((double)tid / 64.0);
  const double t = p.temperature ? (double)p.temperature[s] : 0.0, inv_t = t > 0.0 ? 1.0 / t : 1.0;
  const bool greedy = !(t > 0.0), aligned = p.logits_ld % 4 == 0 && (uintptr_t)p.logits % (4 * sizeof(T)) == 0;
  const int lo = rank * p.slice + warp * p.part, hi = warp < WARPS ? min(min(lo + p.part, (rank + 1) * p.slice), p.vocab) : lo;      // this warp's tokens
  double *mine = kept + warp * p.part;
  __syncthreads();
  int done = 0, turn = 0;
  for (int at = n > 0 ? 0 : -1; at >= 0;) {
    const T *row = reinterpret_cast<const T *>(p.logits) + (size_t)(r0 + at) * p.logits_ld;
    const float *q = greedy || !p.draft ? nullptr : p.draft + (size_t)(r0 + at) * p.draft_ld;
    Shared::Kids &kid = sm.kids[done & 1];
    float my_top = -INFINITY;
    if (warp < WARPS) {
      // ---- the row: largest logit of the part, then weights relative to it and their sum
      int my_at = p.vocab;
#pragma unroll 4
      for (int i = lo + lane * 4; i < hi; i += STEP) {
        float v[4];
        four(row, i, hi, aligned, v);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (v[k] > my_top) { my_top = v[k]; my_at = i + k; }
          if (p.kept && i + k < hi) mine[i + k - lo] = v[k];
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) larger(my_top, my_at, __shfl_xor_sync(0xffffffffu, my_top, o), __shfl_xor_sync(0xffffffffu, my_at, o));
      double sum = 0.0;
      if (my_top > -INFINITY)
        for (int i = lo + lane * 4; i < hi; i += STEP) {
          float v[4];
          if (!p.kept) four(row, i, hi, aligned, v);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (i + k < hi) {
              const double w = weight(p.kept ? (float)mine[i + k - lo] : v[k], my_top, inv_t, sm.table);
              if (p.kept) mine[i + k - lo] = w;
              sum += w;
            }
        }
      sum = warp_add(sum);
      if (lane == 0) sm.warp[warp] = Top{my_top, my_at, sum};
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
            const size_t a = (size_t)rank * p.slice * sizeof(T), b = (size_t)min((rank + 1) * p.slice, p.vocab) * sizeof(T);
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
    __syncthreads();
    // ---- the block's largest and sum, then the cluster's (every block for itself, from the same numbers)
    turn ^= 1;
    if (warp == 0) {
      Top x = lane < WARPS ? sm.warp[lane] : Top{-INFINITY, p.vocab, 0.0};
      float top = x.x;
      int best = x.at;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) larger(top, best, __shfl_xor_sync(0xffffffffu, top, o), __shfl_xor_sync(0xffffffffu, best, o));
      const double sum = warp_add(lane < WARPS && x.x > -INFINITY ? x.sum * weight(x.x, top, inv_t, sm.table) : 0.0);
      if (lane == 0) sm.block[turn] = Top{top, best, sum};
    }
    stay_for_cluster();
    if (warp == 0) {
      Top x = lane < p.blocks ? *in_block(&sm.block[turn], lane) : Top{-INFINITY, p.vocab, 0.0};
      float top = x.x;
      int best = x.at;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) larger(top, best, __shfl_xor_sync(0xffffffffu, top, o), __shfl_xor_sync(0xffffffffu, best, o));
      top = __shfl_sync(0xffffffffu, top, 0);
      best = __shfl_sync(0xffffffffu, best, 0);
      const double total = warp_add(lane < p.blocks && x.x > -INFINITY ? x.sum * weight(x.x, top, inv_t, sm.table) : 0.0);
      if (lane < WARPS) sm.scale[lane] = sm.warp[lane].x > -INFINITY ? weight(sm.warp[lane].x, top, inv_t, sm.table) / total : 0.0;      // weights to probabilities
      const Shared::Kids *head = in_block(&kid, 0);
      const int kids = top > -INFINITY ? head->n : 0;
      if (rank != 0)
        for (int i = lane; i < kids; i += 32) {
          kid.row[i] = head->row[i]; kid.token[i] = head->token[i]; kid.logit[i] = head->logit[i];
          if (!greedy) kid.u[i] = head->u[i];
          if (q) kid.q[i] = head->q[i];
        }
      __syncwarp();
      if (lane == 0) {
        sm.top = top; sm.total = total; sm.best = best; sm.S = 0.0; sm.Z = 1.0; sm.drawn = -1;
        int next = -1, tried = 0;
        for (; tried < kids; ++tried) {
          const int x = kid.token[tried];
          if (greedy) {
            if (x == best) { next = tried; break; }
            continue;
          }
          const double px = x >= 0 ? weight(kid.logit[tried], top, inv_t, sm.table) / total : 0.0;
          if (q) {
            if (x >= 0 && (double)kid.u[tried] * (double)kid.q[tried] < px) next = tried;
            break;                                    // (behind a refusal comes a pass over the row)
          }
          bool before = x < 0;
          for (int i = 0; i < tried && !before; ++i) before = kid.token[i] == x;
          if (before) continue;
          if ((double)kid.u[tried] * sm.Z < px) { next = tried; break; }
          sm.Z -= px;
        }
        sm.next = next;
        sm.tried = tried;
        if (rank != 0) kid.n = kids;
      }
    }
    __syncthreads();
    const float top = sm.top;
    const bool any = top > -INFINITY;
    const int kids = any ? kid.n : 0;
    // ---- with draft probabilities: what a refused child leaves, until one is accepted
    bool passed = false;                              // sm.part and sm.rest hold the sums of what is left
    double S = 0.0;
    auto of_cluster = [&] {                           // sum over the blocks of the sums in sm.part, by the whole block
      __syncthreads();
      turn ^= 1;
      if (warp == 0) {
        const double v = warp_add(lane < WARPS ? sm.part[lane] : 0.0);
        if (lane == 0) sm.rest[turn] = v;
      }
      stay_for_cluster();
      if (warp == 0) {
        const double z = warp_add(lane < p.blocks ? *in_block(&sm.rest[turn], lane) : 0.0);
        if (lane == 0) sm.Z = z;
      }
      __syncthreads();
    };
    auto prob = [&](int i) { return p.kept ? mine[i - lo] * sm.scale[warp] : weight(logit(row, i), top, inv_t, sm.table) / sm.total; };
    if (q && any && kids)
      while (sm.next < 0 && sm.tried < kids) {        // (uniform over the cluster)
        S += sm.Z;
        double z = 0.0;
        if (warp < WARPS)
#pragma unroll 4
          for (int i = lo + lane; i < hi; i += 32) z += fmax(prob(i) - S * (double)q[i], 0.0);
        z = warp_add(z);
        if (warp < WARPS && lane == 0) sm.part[warp] = z;
        of_cluster();
        passed = true;
        if (tid == 0) {
          const int k = ++sm.tried;
          if (k < kids) {
            const int x = kid.token[k];
            const double px = x >= 0 ? weight(kid.logit[k], top, inv_t, sm.table) / sm.total : 0.0;
            if (x >= 0 && (double)kid.u[k] * (double)kid.q[k] * sm.Z < fmax(px - S * (double)kid.q[k], 0.0)) sm.next = k;
          }
        }
        __syncthreads();
      }
    const int next = sm.next < 0 ? -1 : kid.row[sm.next], tried = min(sm.tried, kids);
    int token = next >= 0 ? kid.token[sm.next] : any && greedy ? sm.best : -1;
    bool writes = rank == 0;                          // the block that knows the token
    if (next < 0 && any && !greedy) {
      // ---- drawing.  `whole`: nothing is left, p itself
      bool whole = passed && !(sm.Z > 0.0);
      auto gone = [&](int i) {
        for (int k = 0; k < tried; ++k)
          if (kid.token[k] == i) return true;
        return false;
      };
      auto rest = [&](int i) { return q && passed && !whole ? fmax(prob(i) - S * (double)q[i], 0.0) : !q && !whole && tried && gone(i) ? 0.0 : prob(i); };
      for (int round = 0; round < 2; ++round) {
        if (!(passed && !whole)) {
          double z = 0.0;
          if (warp < WARPS) {
            if (q || whole || !tried) z = lane == 0 ? sm.warp[warp].sum * sm.scale[warp] : 0.0;
            else
              for (int i = lo + lane; i < hi; i += 32) z += rest(i);
          }
          z = warp_add(z);
          __syncthreads();
          if (warp < WARPS && lane == 0) sm.part[warp] = z;
          of_cluster();
        }
        if (sm.Z > 0.0 || whole) break;               // (uniform over the cluster)
        whole = true;
        passed = false;
      }
      const float u = p.uniform_next[s];
      const double want = (u < 1.f ? (double)u : 1.0 - 0x1p-24) * sm.Z;
      // the block, the warp, the token whose running sum exceeds it (where rounding leaves none: the last one with weight)
      double before = 0.0, own_before = 0.0;
      int owner = 0;
      bool found = false;
      for (int b = 0; b < p.blocks && !found; ++b) {
        const double v = *in_block(&sm.rest[turn], b);
        if (v > 0.0) {
          owner = b;
          own_before = before;
          found = before + v > want;
        }
        before += v;
      }
      writes = owner == rank;
      if (writes && warp < WARPS) {
        double c = own_before, my_before = 0.0;
        int chosen = -1;
        found = false;
        for (int w = 0; w < WARPS && !found; ++w) {
          const double v = sm.part[w];
          if (v > 0.0) {
            chosen = w;
            my_before = c;
            found = c + v > want;
          }
          c += v;
        }
        if (warp == chosen) {
          c = my_before;
          int last = -1;
          found = false;
          for (int i0 = lo; i0 < hi && !found; i0 += STEP) {
            double v[4], sum = 0.0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int i = i0 + lane * 4 + k;
              v[k] = i < hi ? rest(i) : 0.0;
              sum += v[k];
            }
            double upto = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const double y = __shfl_up_sync(0xffffffffu, upto, o);
              if (lane >= o) upto += y;
            }
            const unsigned over = __ballot_sync(0xffffffffu, sum > 0.0 && c + upto > want), some = __ballot_sync(0xffffffffu, sum > 0.0);
            const int pick = over ? __ffs(over) - 1 : some ? 31 - __clz(some) : -1;
            int mine_at = -1;
            if (lane == pick) {
              double y = c + (upto - sum);
              for (int k = 0; k < 4; ++k)
                if (v[k] > 0.0) {
                  mine_at = i0 + lane * 4 + k;
                  y += v[k];
                  if (over && y > want) break;
                }
            }
            if (pick >= 0) last = __shfl_sync(0xffffffffu, mine_at, pick);
            c += __shfl_sync(0xffffffffu, upto, 31);
            found = over != 0;
          }
          if (lane == 0) sm.drawn = last;
        }
      }
      __syncthreads();
      token = sm.drawn;
    }
    if (writes && tid == 0) {
      path[done] = at;
      said[done] = token;
      if (lp) {
        const float x = token >= 0 ? logit(row, token) : 0.f;
        lp[done] = token >= 0 ? (float)((x == top ? 0.0 : ((double)x - (double)top) * inv_t) - log(sm.total)) : 0.f;
      }
    }
    ++done;
    at = next;
    __syncthreads();                                  // (the next row writes over what was read)
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
  while (blocks < vf::MAX_BLOCKS && ((long long)a->n_seq * blocks < 2 * sm_count() && (long long)a->vocab > 1024ll * blocks)) blocks *= 2;
  auto slice = [&](int b) { return ceil_div(ceil_div(a->vocab, b), vf::STEP) * vf::STEP; };
  while (blocks < vf::MAX_BLOCKS && (size_t)slice(blocks) * sizeof(double) > vf::WEIGHT_BYTES) blocks *= 2;
  p.blocks = blocks;
  p.slice = slice(blocks);
  p.part = ceil_div(ceil_div(p.slice, vf::WARPS), vf::STEP) * vf::STEP;
  const size_t smem = (size_t)vf::WARPS * p.part * sizeof(double);
  p.kept = smem <= vf::WEIGHT_BYTES;
  return a->dtype == PT_DT_F32 ? vf::launch<float>(p, smem, as_stream(stream)) : a->dtype == PT_DT_F16 ? vf::launch<__half>(p, smem, as_stream(stream))
                                                                                : vf::launch<__nv_bfloat16>(p, smem, as_stream(stream));
}
