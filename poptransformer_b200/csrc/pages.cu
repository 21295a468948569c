// Pages and rows of paged caches: copying pages when sequences fork or a pool is compacted, and moving the rows of accepted tokens together.
// The caches of a model's layers share one page numbering, so that one launch serves all of them: the grid's second dimension is the layer.
// Both are copies: what bounds them is memory (each byte read and written once: 450 pages of 28 layers, 1.65 GB, in 285 us, 5.8 TB/s; 16 pages of 32 layers in
// 47 us), or the launch where little moves (rows of 24 sequences in 32 layers: 7.1 us).
#include "elem.cuh"

namespace pt {
namespace pg {

constexpr int MAX_POOLS = 64, THREADS = 256, MAX_PATH = 512;      // (a path: as long as verification makes them)

struct Pools {
  char *pool[MAX_POOLS];
  int n_kv[MAX_POOLS], k_row[MAX_POOLS], v_row[MAX_POOLS];   // bytes of a position's key and value of one head
};

__device__ __forceinline__ size_t page_bytes(const Pools &c, int l, int page) { return (size_t)c.n_kv[l] * page * (c.k_row[l] + c.v_row[l]); }

// V: the unit that all pages are whole multiples of.
template <typename V> __global__ void __launch_bounds__(THREADS) copy_pages_kernel(const Pools c, int page, int n_pages, const int *src, const int *dst, int n, int *error_flag) {
  early_start();
  constexpr int UNROLL = 4, CHUNK = THREADS * UNROLL;
  const int l = blockIdx.y;
  const size_t bytes = page_bytes(c, l, page), units = bytes / sizeof(V);
  const long long chunks = (long long)((units + CHUNK - 1) / CHUNK), all = chunks * n;
  for (long long w = blockIdx.x; w < all; w += gridDim.x) {
    const int i = (int)(w / chunks);
    const size_t at = (size_t)(w - i * chunks) * CHUNK + threadIdx.x;
    const int a = src[i], b = dst[i];
    if (a < 0 || b < 0 || a == b) continue;
    if (a >= n_pages || b >= n_pages) {
      if (threadIdx.x == 0 && error_flag) atomicExch(error_flag, 12);
      continue;
    }
    const V *from = reinterpret_cast<const V *>(c.pool[l] + (size_t)a * bytes);
    V *to = reinterpret_cast<V *>(c.pool[l] + (size_t)b * bytes), v[UNROLL];
#pragma unroll
    for (int j = 0; j < UNROLL; ++j)
      if (at + j * THREADS < units) v[j] = from[at + j * THREADS];
#pragma unroll
    for (int j = 0; j < UNROLL; ++j)
      if (at + j * THREADS < units) to[at + j * THREADS] = v[j];
  }
}

struct Rows {
  int page, max_pages, path_ld;
  const int *page_table, *cu, *start, *slot, *path, *count;
  int *error_flag;
};
// Block: one sequence, one layer.  A thread moves a unit of every row of the path, in order: a path increases, so that row i is read as a
// source, if it is one, before it is written, and the rows behind it are read later but lie behind all that was written.
template <typename V> __global__ void __launch_bounds__(THREADS) move_rows_kernel(const Pools c, const Rows p) {
  early_start();
  __shared__ int2 from[MAX_PATH], to[MAX_PATH];     // page and place in it
  __shared__ int bad;
  const int s = blockIdx.x, l = blockIdx.y, tid = threadIdx.x;
  const int len = p.cu[s + 1] - p.cu[s], start = p.start[s], n = p.count[s];
  if (n <= 0) return;
  if (tid == 0) bad = n > p.path_ld || n > MAX_PATH || n > len ? 14 : start < 0 || start > p.page * p.max_pages - len ? 12 : 0;
  __syncthreads();
  if (!bad) {
    const int *table = p.page_table + (size_t)p.slot[s] * p.max_pages, *path = p.path + (size_t)s * p.path_ld;
    for (int i = tid; i < n; i += THREADS) {
      const int r = path[i];
      if (r < 0 || r >= len || (i > 0 && path[i - 1] >= r)) {
        bad = 14;
        continue;
      }
      from[i] = make_int2(table[(start + r) / p.page], (start + r) % p.page);
      to[i] = make_int2(table[(start + i) / p.page], (start + i) % p.page);
      if (from[i].x < 0 || to[i].x < 0) bad = 12;
    }
  }
  __syncthreads();
  if (bad) {
    if (tid == 0 && p.error_flag) atomicExch(p.error_flag, bad);
    return;
  }
  const int kv = c.n_kv[l], ku = c.k_row[l] / (int)sizeof(V), vu = c.v_row[l] / (int)sizeof(V);
  const size_t bytes = page_bytes(c, l, p.page);
  for (int u = tid; u < kv * (ku + vu); u += THREADS) {
    const bool is_v = u >= kv * ku;
    const int w = is_v ? u - kv * ku : u, per = is_v ? vu : ku, g = w / per, col = w - g * per;
    const size_t base = (is_v ? (size_t)kv * p.page * ku : 0) + (size_t)g * p.page * per + col;   // in units
    auto at = [&](int2 x) { return reinterpret_cast<V *>(c.pool[l] + (size_t)x.x * bytes) + base + (size_t)x.y * per; };
    constexpr int AHEAD = 8;
    for (int i0 = 0; i0 < n; i0 += AHEAD) {
      V v[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (i0 + j < n) v[j] = *at(from[i0 + j]);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (i0 + j < n) *at(to[i0 + j]) = v[j];
    }
  }
}

static int fill(Pools &c, const pt_kv_pool *in, int n, int page, int &unit, const char *who) {
  for (int i = 0; i < n; ++i) {
    const pt_kv_pool &x = in[i];
    PT_REQUIRE(x.pool && x.n_kv > 0 && x.dim > 0 && x.vdim >= 0 && (x.elem_bytes == 1 || x.elem_bytes == 2 || x.elem_bytes == 4), "%s: pool %d: n_kv=%d dim=%d vdim=%d elem_bytes=%d",
               who, i, x.n_kv, x.dim, x.vdim, x.elem_bytes);
    PT_REQUIRE((long long)(x.dim + (long long)x.vdim) * x.elem_bytes * x.n_kv * page < (1ll << 31), "%s: pool %d: a page of 2 GB or more", who, i);
    c.pool[i] = (char *)x.pool;
    c.n_kv[i] = x.n_kv; c.k_row[i] = x.dim * x.elem_bytes; c.v_row[i] = x.vdim * x.elem_bytes;
    while ((uintptr_t)x.pool % unit || c.k_row[i] % unit || c.v_row[i] % unit) unit /= 2;
  }
  return PT_OK;
}

}  // namespace pg
}  // namespace pt

using namespace pt;

extern "C" int pt_kv_copy_pages(const pt_kv_pool *pools, int n_pools, int page_size, int n_pages, const int32_t *src, const int32_t *dst, int n, int32_t *error_flag, void *stream) {
  PT_REQUIRE(pools && n_pools > 0 && page_size > 0 && n_pages > 0 && n >= 0, "pt_kv_copy_pages: n_pools=%d page_size=%d n_pages=%d n=%d", n_pools, page_size, n_pages, n);
  PT_REQUIRE(n == 0 || (src && dst), "pt_kv_copy_pages: null pointer argument");
  for (int i0 = 0; i0 < n_pools; i0 += pg::MAX_POOLS) {
    const int k = std::min(n_pools - i0, pg::MAX_POOLS);
    pg::Pools c{};
    int unit = 16;
    if (int rc = pg::fill(c, pools + i0, k, page_size, unit, "pt_kv_copy_pages")) return rc;
    if (n == 0) continue;
    const auto kernel = unit == 16 ? pg::copy_pages_kernel<uint4> : unit == 8 ? pg::copy_pages_kernel<uint2> : unit == 4 ? pg::copy_pages_kernel<uint32_t>
                        : unit == 2 ? pg::copy_pages_kernel<uint16_t> : pg::copy_pages_kernel<uint8_t>;
    const int blocks = std::max(1, ceil_div(sm_count() * 8, k));
    PT_CUDA(launch_early(kernel, Grid(dim3(blocks, k)), pg::THREADS, 0, as_stream(stream), c, page_size, n_pages, src, dst, n, error_flag));
    PT_LAUNCH_CHECK("pt_kv_copy_pages");
  }
  return PT_OK;
}

extern "C" int pt_kv_move_rows(const pt_kv_pool *pools, int n_pools, int page_size, int max_pages, const int32_t *page_table, const pt_batch_view *b, const int32_t *path,
                               int path_ld, const int32_t *count, int32_t *error_flag, void *stream) {
  PT_REQUIRE(pools && n_pools > 0 && page_size > 0 && max_pages > 0 && page_table, "pt_kv_move_rows: n_pools=%d page_size=%d max_pages=%d", n_pools, page_size, max_pages);
  PT_REQUIRE((long long)page_size * max_pages < (1ll << 31), "pt_kv_move_rows: %d pages of %d positions", max_pages, page_size);
  PT_REQUIRE(b && b->n_seq > 0 && b->cu && b->start && b->slot && path && count && path_ld > 0, "pt_kv_move_rows: bad batch (%d sequences) or path (%d entries a row)", b ? b->n_seq : 0,
             path_ld);
  for (int i0 = 0; i0 < n_pools; i0 += pg::MAX_POOLS) {
    const int k = std::min(n_pools - i0, pg::MAX_POOLS);
    pg::Pools c{};
    int unit = 16;
    if (int rc = pg::fill(c, pools + i0, k, page_size, unit, "pt_kv_move_rows")) return rc;
    const auto kernel = unit == 16 ? pg::move_rows_kernel<uint4> : unit == 8 ? pg::move_rows_kernel<uint2> : unit == 4 ? pg::move_rows_kernel<uint32_t>
                        : unit == 2 ? pg::move_rows_kernel<uint16_t> : pg::move_rows_kernel<uint8_t>;
    const pg::Rows r{page_size, max_pages, path_ld, page_table, b->cu, b->start, b->slot, path, count, error_flag};
    PT_CUDA(launch_early(kernel, Grid(dim3(b->n_seq, k)), pg::THREADS, 0, as_stream(stream), c, r));
    PT_LAUNCH_CHECK("pt_kv_move_rows");
  }
  return PT_OK;
}
