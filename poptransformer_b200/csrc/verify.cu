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
// Block: one sequence; it reads only the rows that its path reaches.
#include "elem.cuh"

namespace pt {
namespace vf {

constexpr int THREADS = 512, WARPS = THREADS / 32;

struct Params {
  int n_seq, n_tok, vocab, logits_ld, draft_ld, max_path;
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
// exp((x - top) / T); equal infinities share the weight.
__device__ __forceinline__ double weight(float x, float top, double inv_t) { return x == top ? 1.0 : exp(((double)x - (double)top) * inv_t); }

struct Shared {
  double sum[WARPS];
  float top[WARPS];
  int at[WARPS];
};
__device__ __forceinline__ double block_add(double v, Shared &sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm.sum[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
  for (int i = 0; i < WARPS; ++i) t += sm.sum[i];
  return t;
}
// The largest logit and its lowest place.
template <typename T> __device__ __forceinline__ void row_top(const T *row, int vocab, Shared &sm, float &top, int &at) {
  float m = -INFINITY;
  int k = vocab;
  for (int i = threadIdx.x; i < vocab; i += THREADS) {
    const float x = logit(row, i);
    if (x > m) { m = x; k = i; }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o);
    const int ok = __shfl_xor_sync(0xffffffffu, k, o);
    if (om > m || (om == m && ok < k)) { m = om; k = ok; }
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) { sm.top[threadIdx.x >> 5] = m; sm.at[threadIdx.x >> 5] = k; }
  __syncthreads();
  top = sm.top[0]; at = sm.at[0];
  for (int i = 1; i < WARPS; ++i)
    if (sm.top[i] > top || (sm.top[i] == top && sm.at[i] < at)) { top = sm.top[i]; at = sm.at[i]; }
}

template <typename T> __global__ void __launch_bounds__(THREADS) verify_kernel(const Params p) {
  early_start();
  __shared__ Shared sm;
  __shared__ int drawn, behind;
  const int s = blockIdx.x, tid = threadIdx.x, r0 = p.cu[s], n = p.cu[s + 1] - r0;
  int *path = p.path + (size_t)s * p.max_path, *said = p.out_token + (size_t)s * p.max_path;
  float *lp = p.logprob ? p.logprob + (size_t)s * p.max_path : nullptr;
  int done = 0;
  if (n > 0 && r0 >= 0 && r0 + n <= p.n_tok) {
    const double t = p.temperature ? (double)p.temperature[s] : 0.0, inv_t = t > 0.0 ? 1.0 / t : 1.0;
    const bool greedy = !(t > 0.0);
    int at = 0;
    while (at >= 0) {
      const T *row = reinterpret_cast<const T *>(p.logits) + (size_t)(r0 + at) * p.logits_ld;
      const float *q = greedy || !p.draft ? nullptr : p.draft + (size_t)(r0 + at) * p.draft_ld;
      float top;
      int best;
      row_top(row, p.vocab, sm, top, best);
      const bool any = top > -INFINITY;
      double total = 0.0;
      if (any)
        for (int i = tid; i < p.vocab; i += THREADS) total += weight(logit(row, i), top, inv_t);
      total = block_add(total, sm);
      auto prob = [&](int x) { return weight(logit(row, x), top, inv_t) / total; };
      auto log_p = [&](int x) {
        const float l = logit(row, x);
        return (float)((l == top ? 0.0 : ((double)l - (double)top) * inv_t) - log(total));
      };
      // children, in order
      double S = 0.0, Z = 1.0;      // with q: r = max(p - S q, 0); without: Z is what the refused tokens left of p
      int next = -1, tried = 0;     // tried: children refused
      auto child = [&](int c) { return (p.parent ? p.parent[r0 + c] : c - 1) == at; };
      auto refused = [&](int x) {   // without q: whether x was the token of a refused child
        for (int c = at + 1, k = 0; k < tried && c < n; ++c)
          if (child(c)) {
            if (p.token[r0 + c] == x) return true;
            ++k;
          }
        return false;
      };
      if (any && done + 1 < p.max_path)
        for (int c = at + 1; c < n && next < 0; ++c) {
          if (!child(c)) continue;
          const int x = p.token[r0 + c];
          bool ok = false;
          if (x >= 0 && x < p.vocab) {
            if (greedy) ok = x == best;
            else if (q) ok = (double)p.uniform[r0 + c] * (double)q[x] * Z < fmax(prob(x) - S * (double)q[x], 0.0);
            else ok = !refused(x) && (double)p.uniform[r0 + c] * Z < prob(x);
          }
          if (ok) {
            next = c;
            break;
          }
          if (q) {
            S += Z;
            double z = 0.0;
            for (int i = tid; i < p.vocab; i += THREADS) z += fmax(weight(logit(row, i), top, inv_t) / total - S * (double)q[i], 0.0);
            Z = block_add(z, sm);
          } else if (!greedy && x >= 0 && x < p.vocab && !refused(x)) {
            Z -= prob(x);
          }
          ++tried;
        }
      int token = best, level = done;
      if (next >= 0) token = p.token[r0 + next];
      else if (!any) token = -1;
      else if (!greedy) {
        // r, in a contiguous share per thread; the running sum over the threads finds the one that holds the token
        bool whole = q ? !(Z > 0.0) : false;      // nothing is left: p itself
        const int share = (p.vocab + THREADS - 1) / THREADS, lo = min(tid * share, p.vocab), hi = min(lo + share, p.vocab);
        auto rest = [&](int i) {
          const double w = weight(logit(row, i), top, inv_t) / total;
          if (whole) return w;
          if (q) return fmax(w - S * (double)q[i], 0.0);
          return tried > 0 && refused(i) ? 0.0 : w;
        };
        double mine = 0.0, all = 0.0;
        for (int round = 0; round < 2; ++round) {
          mine = 0.0;
          for (int i = lo; i < hi; ++i) mine += rest(i);
          all = block_add(mine, sm);
          if (all > 0.0 || whole) break;          // (uniform: every thread has the same sum)
          whole = true;
        }
        double upto = mine;                       // inclusive running sum over the threads
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, upto, o);
          if ((tid & 31) >= o) upto += v;
        }
        __syncthreads();
        if ((tid & 31) == 31) sm.sum[tid >> 5] = upto;
        if (tid == 0) { drawn = p.vocab; behind = -1; }
        __syncthreads();
        for (int i = 0; i < (tid >> 5); ++i) upto += sm.sum[i];
        const double want = (double)p.uniform_next[s] * all, before = upto - mine;
        // the first value whose running sum exceeds `want`; where rounding leaves none, the last that has weight
        if (mine > 0.0) {
          double c = before;
          int last = -1;
          bool found = false;
          for (int i = lo; i < hi && !found; ++i) {
            const double w = rest(i);
            if (w > 0.0) {
              last = i;
              c += w;
              found = c > want;
            }
          }
          if (found) atomicMin(&drawn, last);
          else atomicMax(&behind, last);
        }
        __syncthreads();
        token = drawn < p.vocab ? drawn : behind;
      }
      if (tid == 0) {
        path[level] = at;
        said[level] = token;
        if (lp) lp[level] = token >= 0 ? log_p(token) : 0.f;
      }
      ++done;
      at = next;
    }
  }
  for (int i = done + tid; i < p.max_path; i += THREADS) {
    path[i] = said[i] = -1;
    if (lp) lp[i] = 0.f;
  }
  if (tid == 0) p.count[s] = done;
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
  const vf::Params p{a->n_seq, a->n_tok, a->vocab, a->logits_ld, a->draft_ld, a->max_path, a->cu, a->token, a->parent, a->logits, a->draft, a->temperature, a->uniform,
                     a->uniform_next, a->path, a->count, a->out_token, a->logprob};
  const auto kernel = a->dtype == PT_DT_F32 ? vf::verify_kernel<float> : a->dtype == PT_DT_F16 ? vf::verify_kernel<__half> : vf::verify_kernel<__nv_bfloat16>;
  PT_CUDA(launch_early(kernel, Grid(a->n_seq), vf::THREADS, 0, as_stream(stream), p));
  PT_LAUNCH_CHECK("pt_verify_drafts");
  return PT_OK;
}
