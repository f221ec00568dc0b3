// Pages of a key-value cache: fork (share, copy, free, reorder), compact, extend
// and the write of new tokens' keys and values.
//
// State: a page table (rows x width page numbers), the rows' lengths, and a
// reference count per page.  A page is free when its count is 0; the lowest free
// page is taken first, so every result is a function of the inputs alone (no
// free list, no order of arrival).  The bookkeeping of one call is one launch of
// one thread-block cluster (its phases follow one another through cluster
// barriers, a microsecond each, where separate launches or a grid barrier cost
// more); the page contents then move in a second launch over the whole GPU.
//
// Nothing here computes: the bound is the bytes moved (the rows copied, once in
// and once out) plus the two launches.  Measured through the public calls: a fork of 4 beams
// over 96 pages 8.3 us (6.2 on the GPU), which is latency alone; of 16 groups of 8 beams with
// 142 MB moved 32 us (4.4 TB/s; 10 of them bookkeeping); a compaction of 1.2 GB moved (both
// ways) 210 to 214 us (5.8 TB/s); 16 ragged chunks of up to 512 tokens taken and written
// 15 us, most of them two launches' latency.
#include "qs_common.cuh"
#include "qs_launch.h"

namespace qs {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;

// Raised by the kernels, read and cleared by qs_device_status.
__device__ int g_cache_error;

__device__ __forceinline__ void flag_error(int bit) { atomicOr(&g_cache_error, bit); }

__global__ void clear_error_kernel(int bit) { atomicAnd(&g_cache_error, ~bit); }

__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return static_cast<int>(r);
}
__device__ __forceinline__ int cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return static_cast<int>(r);
}
// Barrier of every thread of the cluster; global writes before it are seen after it
// (within one CTA without the fence, which waits for them to reach L2).
__device__ __forceinline__ void cluster_barrier() {
  if (cluster_size() == 1) {
    __syncthreads();
    return;
  }
  __threadfence();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Exclusive prefix of v over the block's threads; *total gets the sum.
__device__ __forceinline__ int block_prefix(int v, int *total, int *tmp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) tmp[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = lane < kWarps ? tmp[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += y;
    }
    if (lane < kWarps) tmp[lane] = w;
  }
  __syncthreads();
  const int before = (warp ? tmp[warp - 1] : 0) + x - v;
  *total = tmp[kWarps - 1];
  __syncthreads();
  return before;
}

// Workspace of a bookkeeping launch (int32 words).
struct Work {
  int *head;    // [64]: 0 = entries of list, 1 = moves of a compaction, 8.. = one count per CTA
  int *a, *b;   // [pages] each
  int *map;     // [pages]
  int4 *list;   // copies: source page, destination page, tokens
};

Work split_work(void *ws, int64_t rows, int64_t pages) {
  Work w;
  w.head = static_cast<int *>(ws);
  w.list = reinterpret_cast<int4 *>(w.head + 64);
  w.a = w.head + 64 + 4 * (rows + pages);
  w.b = w.a + pages;
  w.map = w.b + pages;
  return w;
}

// This CTA's pages [lo, hi): equal shares in page order.
__device__ __forceinline__ void share_of(int pages, int *lo, int *hi) {
  const int each = (pages + cluster_size() - 1) / cluster_size();
  *lo = min(pages, each * cluster_rank());
  *hi = min(pages, *lo + each);
}

// Sum of the counts of the CTAs before this one (and of all), after every CTA wrote head[8 + rank].
__device__ __forceinline__ int counts_before(const int *head, int *total) {
  int before = 0, all = 0;
  for (int r = 0; r < cluster_size(); ++r) {
    const int c = __ldcg(head + 8 + r);
    if (r < cluster_rank()) before += c;
    all += c;
  }
  *total = all;
  return before;
}

// Numbers this CTA's share of the pages with pred true, in page order, from the
// cluster-wide prefix: emit(page, rank, pred, their number in all) for every page.  All
// threads call it; a first pass counts and a cluster barrier exchanges the counts (one
// CTA needs neither, unless emit asks for the number: kNeedAll), the second pass numbers.
template <bool kNeedAll, class Pred, class Emit>
__device__ __forceinline__ int number_pages(int pages, int *head, int *tmp, Pred pred, Emit emit) {
  int lo, hi;
  share_of(pages, &lo, &hi);
  int all = 0, base = 0;
  if (cluster_size() > 1 || kNeedAll) {
    int mine = 0;
#pragma unroll 4
    for (int p = lo + threadIdx.x; p < hi; p += kThreads) mine += pred(p) ? 1 : 0;
    block_prefix(mine, &all, tmp);
    if (cluster_size() > 1) {
      if (threadIdx.x == 0) head[8 + cluster_rank()] = all;
      cluster_barrier();
      base = counts_before(head, &all);
    }
  }
  for (int p0 = lo; p0 < hi; p0 += kThreads) {
    const int p = p0 + threadIdx.x;
    const bool is = p < hi && pred(p);
    int n;
    const int r = base + block_prefix(is ? 1 : 0, &n, tmp);
    if (p < hi) emit(p, r, is, all);
    base += n;
  }
  return cluster_size() > 1 || kNeedAll ? all : base;
}

struct Tables {
  int rows, width, pages, page_shift;
  const int *table, *lengths, *refcount;
  int *table_out, *lengths_out, *refcount_out;
};

__device__ __forceinline__ int pages_of(int64_t n, int shift, int width) {
  return static_cast<int>(min(static_cast<int64_t>(width), (n + (1 << shift) - 1) >> shift));
}

// ---- fork ------------------------------------------------------------------------
// Row i becomes a copy of row parent[i] of the input tables (-1: empty).  Whole
// pages are shared; a part-filled last page stays with the first child, and the
// other children get a page of their own, whose filled tokens the second launch
// copies.  Counts change by references after minus references before, so counts
// that the caller holds besides the table's stay.  NEAR (one CTA, counts that fit its
// shared memory): the counts are changed and searched there, which saves two trips to L2.
template <bool NEAR>
__global__ void __launch_bounds__(kThreads, 1) fork_kernel(Tables t, const int *parents, Work w) {
  extern __shared__ int sm[];
  __shared__ int tmp[32];
  int *first = sm, *kids = sm + t.rows, *rank = sm + 2 * t.rows, *par = sm + 3 * t.rows, *len = sm + 4 * t.rows;
  int *fresh = NEAR ? sm + 5 * t.rows : w.a, *count = NEAR ? sm + 6 * t.rows : t.refcount_out;
  pdl_wait();
  pdl_launch_dependents();
  const int nthreads = kThreads * cluster_size(), tid = cluster_rank() * kThreads + threadIdx.x;
  const int fill_mask = (1 << t.page_shift) - 1;
  int lo, hi;
  share_of(t.pages, &lo, &hi);
  for (int i = threadIdx.x; i < t.rows; i += kThreads) {
    const int p = parents[i];
    first[i] = t.rows;
    kids[i] = 0;
    len[i] = max(0, t.lengths[i]);
    par[i] = p >= 0 && p < t.rows ? p : -1;
    if (par[i] < 0 && p != -1 && cluster_rank() == 0) flag_error(kCacheErrParent);
  }
#pragma unroll 4
  for (int p = lo + threadIdx.x; p < hi; p += kThreads) count[p] = t.refcount[p];
  __syncthreads();
  for (int i = threadIdx.x; i < t.rows; i += kThreads)
    if (par[i] >= 0) {
      atomicAdd(&kids[par[i]], 1);
      atomicMin(&first[par[i]], i);
    }
  __syncthreads();
  // rows that need a page of their own, numbered in row order
  int want = 0;
  for (int i0 = 0; i0 < t.rows; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    bool dup = false;
    if (i < t.rows && par[i] >= 0 && first[par[i]] != i) {
      const int n = len[par[i]], c = n >> t.page_shift;
      if ((n & fill_mask) != 0 && c < t.width) {
        const int page = t.table[static_cast<int64_t>(par[i]) * t.width + c];
        dup = page >= 0 && page < t.pages;  // an absent page is absent in every child
      }
    }
    int n;
    const int r = want + block_prefix(dup ? 1 : 0, &n, tmp);
    if (i < t.rows) rank[i] = dup ? r : -1;
    want += n;
  }
  cluster_barrier();
  // entry by entry: the references of the old row that go or come, and the new row
  const int64_t entries = static_cast<int64_t>(t.rows) * t.width;
#pragma unroll 4
  for (int64_t e = tid; e < entries; e += nthreads) {
    const int i = static_cast<int>(static_cast<uint32_t>(e) / static_cast<uint32_t>(t.width));
    const int c = static_cast<int>(e - static_cast<int64_t>(i) * t.width);
    const int p = par[i];
    const int old_used = pages_of(len[i], t.page_shift, t.width), whole = min(old_used, len[i] >> t.page_shift);
    const int n = p < 0 ? 0 : len[p], used = pages_of(n, t.page_shift, t.width);
    const int d = c < whole ? kids[i] - 1 : (kids[i] ? 0 : -1);
    const int was = c < old_used && d != 0 ? t.table[e] : -1;
    const int is = c < used ? t.table[static_cast<int64_t>(p) * t.width + c] : -1;
    if (was >= 0 && was < t.pages) atomicAdd(count + was, d);
    if (rank[i] >= 0 && c == used - 1) w.list[rank[i]].x = is;  // a copying row's last entry follows below
    else t.table_out[e] = is;
    if (c == 0) t.lengths_out[i] = n;
  }
  if (t.width == 0)
    for (int i = tid; i < t.rows; i += nthreads) t.lengths_out[i] = par[i] < 0 ? 0 : len[par[i]];
  cluster_barrier();
  auto count_of = [&](int p) { return NEAR ? count[p] : __ldcg(count + p); };
  if (want == 0) {  // the same in every CTA
    if (NEAR)
      for (int p = tid; p < t.pages; p += nthreads) t.refcount_out[p] = count[p];
    if (tid == 0) w.head[0] = 0;
    return;
  }
  const int free_pages = number_pages<false>(
      t.pages, w.head, tmp, [&](int p) { return count_of(p) == 0; },
      [&](int p, int r, bool is, int) {
        const bool take = is && r < want;
        if (take) fresh[r] = p;
        if (NEAR) t.refcount_out[p] = take ? 1 : count[p];
      });
  cluster_barrier();
  for (int i = tid; i < t.rows; i += nthreads) {
    const int r = rank[i];
    if (r < 0) continue;
    const int n = len[par[i]], page = r < free_pages ? (NEAR ? fresh[r] : __ldcg(fresh + r)) : -1;
    t.table_out[static_cast<int64_t>(i) * t.width + (n >> t.page_shift)] = page;
    if (page < 0) flag_error(kCacheErrPages);
    else if (!NEAR) t.refcount_out[page] = 1;
    w.list[r].y = page;
    w.list[r].z = n & fill_mask;
  }
  if (tid == 0) w.head[0] = want;
}

// ---- compact ---------------------------------------------------------------------
// With U pages in use, the used pages from U on move to the holes below U, both in
// ascending order; tables and counts follow.
__global__ void __launch_bounds__(kThreads, 1) compact_kernel(Tables t, int *used_out, Work w) {
  __shared__ int tmp[32];
  pdl_wait();
  pdl_launch_dependents();
  const int nthreads = kThreads * cluster_size(), tid = cluster_rank() * kThreads + threadIdx.x;
  if (tid == 0) w.head[1] = 0;
  // rank = used pages before p.  A hole p < U is number p - rank among the holes; a
  // used page p >= U goes by its rank, and those ranks end at U - 1.
  const int used = number_pages<true>(
      t.pages, w.head, tmp, [&](int p) { return t.refcount[p] > 0; },
      [&](int p, int r, bool is, int all) {
        t.refcount_out[p] = t.refcount[p];
        w.map[p] = p;
        if (is && p >= all) w.a[r] = p;
        if (!is && p < all) w.b[p - r] = p;
        if (p == all) w.head[1] = all - r;  // holes below U
      });
  cluster_barrier();
  const int moves = __ldcg(w.head + 1);
  for (int m = tid; m < moves; m += nthreads) {
    const int src = __ldcg(w.a + used - moves + m), dst = __ldcg(w.b + m);
    w.map[src] = dst;
    t.refcount_out[dst] = t.refcount[src];
    t.refcount_out[src] = 0;
    w.list[m] = make_int4(src, dst, 1 << t.page_shift, 0);
  }
  if (tid == 0) {
    w.head[0] = moves;
    used_out[0] = used;
  }
  cluster_barrier();
  const int64_t entries = static_cast<int64_t>(t.rows) * t.width;
#pragma unroll 4
  for (int64_t e = tid; e < entries; e += nthreads) {
    const int i = static_cast<int>(static_cast<uint32_t>(e) / static_cast<uint32_t>(t.width));
    const int c = static_cast<int>(e - static_cast<int64_t>(i) * t.width);
    const int p = t.table[e];
    const bool held = c < pages_of(max(0, t.lengths[i]), t.page_shift, t.width) && p >= 0 && p < t.pages;
    t.table_out[e] = held ? __ldcg(w.map + p) : -1;
  }
}

// ---- extend ----------------------------------------------------------------------
// Row i grows by add[i] tokens; its new pages are the lowest free ones, numbered in
// row and then column order.  NEAR: as for fork.
template <bool NEAR>
__global__ void __launch_bounds__(kThreads, 1) extend_kernel(Tables t, const int *add, Work w) {
  extern __shared__ int sm[];
  __shared__ int tmp[32];
  int *start = sm, *had_s = sm + t.rows, *len_s = sm + 2 * t.rows;
  int *fresh = NEAR ? sm + 3 * t.rows : w.a, *count = NEAR ? fresh + t.pages : w.b;
  pdl_wait();
  pdl_launch_dependents();
  const int nthreads = kThreads * cluster_size(), tid = cluster_rank() * kThreads + threadIdx.x;
  if (NEAR) {
#pragma unroll 4
    for (int p = threadIdx.x; p < t.pages; p += kThreads) count[p] = t.refcount[p];
  }
  int want = 0;
  for (int i0 = 0; i0 < t.rows; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    int need = 0;
    if (i < t.rows) {
      const int n = max(0, t.lengths[i]), a = add[i];
      const int64_t m = static_cast<int64_t>(n) + max(0, a);
      const int had = pages_of(n, t.page_shift, t.width);
      need = pages_of(m, t.page_shift, t.width) - had;
      had_s[i] = had;
      len_s[i] = static_cast<int>(min(m, static_cast<int64_t>(0x7fffffff)));
      if (cluster_rank() == 0) {
        if (a < 0) flag_error(kCacheErrParent);
        if (m > (static_cast<int64_t>(t.width) << t.page_shift)) flag_error(kCacheErrPages);
      }
    }
    int n;
    const int before = want + block_prefix(need, &n, tmp);
    if (i < t.rows) start[i] = before;
    want += n;
  }
  const int free_pages = number_pages<false>(  // NEAR: a thread's own entries of count
      t.pages, w.head, tmp, [&](int p) { return (NEAR ? count[p] : t.refcount[p]) == 0; },
      [&](int p, int r, bool is, int) {
        const bool take = is && r < want;
        const int had = NEAR ? count[p] : t.refcount[p];
        if (take) fresh[r] = p;
        count[p] = take ? 1 : had;
      });
  if (tid == 0 && want > free_pages) flag_error(kCacheErrPages);
  cluster_barrier();
  // the outputs may be the inputs: every input value was read before the last barrier,
  // except the table entries that stay where they are
  for (int p = tid; p < t.pages; p += nthreads) t.refcount_out[p] = NEAR ? count[p] : __ldcg(count + p);
  const int64_t entries = static_cast<int64_t>(t.rows) * t.width;
#pragma unroll 4
  for (int64_t e = tid; e < entries; e += nthreads) {
    const int i = static_cast<int>(static_cast<uint32_t>(e) / static_cast<uint32_t>(t.width));
    const int c = static_cast<int>(e - static_cast<int64_t>(i) * t.width);
    const int had = had_s[i], has = pages_of(len_s[i], t.page_shift, t.width), r = start[i] + c - had;
    int p = -1;
    if (c < had) p = t.table[e];
    else if (c < has && r < free_pages) p = NEAR ? fresh[r] : __ldcg(fresh + r);
    t.table_out[e] = p;
  }
  for (int i = tid; i < t.rows; i += nthreads) t.lengths_out[i] = len_s[i];
}

// ---- moving page contents ------------------------------------------------------------
struct Pool {
  char *k, *v;
  int layers, pages, heads, chunks;  // chunks: 16-byte pieces of one token's row of one head
  int64_t ks[4], vs[4];              // strides in bytes: layer, page, head, token
};

Pool make_pool(const qs_kv_pool &p) {
  Pool q;
  q.k = static_cast<char *>(p.k);
  q.v = static_cast<char *>(p.v);
  q.layers = static_cast<int>(p.layers);
  q.pages = static_cast<int>(p.pages);
  q.heads = static_cast<int>(p.heads);
  q.chunks = static_cast<int>(p.dim / 8);
  for (int i = 0; i < 4; ++i) q.ks[i] = p.k_stride[i] * 2, q.vs[i] = p.v_stride[i] * 2;
  return q;
}

// A warp takes 4 KB (256 pieces of 16 bytes) of one (copy, layer, K or V, head) at a time:
// `tokens` rows of `chunks` pieces.  The list is kept in shared memory, so that the parts
// that lie beyond a part-filled page's tokens cost next to nothing.
constexpr int kCopyUnroll = 8;
constexpr int kCopyList = 1024;
__global__ void __launch_bounds__(256) copy_pages_kernel(Pool p, int page, const int *head, const int4 *list) {
  __shared__ int4 near[kCopyList];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, count = head[0];
  for (int i = threadIdx.x; i < min(count, kCopyList); i += blockDim.x) near[i] = list[i];
  __syncthreads();
  const uint32_t parts = (page * p.chunks + 32 * kCopyUnroll - 1) / (32 * kCopyUnroll);
  const uint32_t each = static_cast<uint32_t>(p.layers) * 2 * p.heads * parts;  // warps' shares per copy
  const int64_t units = static_cast<int64_t>(count) * each;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); u < units; u += step) {
    const int at = static_cast<int>(u / each);
    uint32_t r = static_cast<uint32_t>(u - static_cast<int64_t>(at) * each);
    const int4 e = at < kCopyList ? near[at] : list[at];
    const uint32_t part = r % parts;
    const int n = e.z * p.chunks, i0 = static_cast<int>(part) * 32 * kCopyUnroll + lane;
    if (i0 - lane >= n || e.x < 0 || e.x >= p.pages || e.y < 0 || e.y >= p.pages) continue;
    r /= parts;
    const uint32_t h = r % p.heads;
    r /= p.heads;
    const bool is_v = r & 1;
    const int64_t *st = is_v ? p.vs : p.ks;
    char *base = (is_v ? p.v : p.k) + (r >> 1) * st[0] + h * st[2];
    const char *src = base + e.x * st[1];
    char *dst = base + e.y * st[1];
    const int token = static_cast<int>(st[3]);
    uint4 x[kCopyUnroll];
    int off[kCopyUnroll];
#pragma unroll
    for (int j = 0; j < kCopyUnroll; ++j) {
      const int i = i0 + 32 * j;
      if (i < n) {
        const int row = i / p.chunks;
        off[j] = row * token + (i - row * p.chunks) * 16;
        x[j] = *reinterpret_cast<const uint4 *>(src + off[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < kCopyUnroll; ++j)
      if (i0 + 32 * j < n) *reinterpret_cast<uint4 *>(dst + off[j]) = x[j];
  }
}

// ---- writing new tokens ------------------------------------------------------------
struct WriteArgs {
  Pool p;
  int rows, width, page_shift, tokens;
  const int *table, *lengths, *cu;  // cu null: token t is the newest of row t
  const char *k, *v;
  int64_t k_token, k_head, v_token, v_head;  // bytes
};

// A warp per token: its place is its row's length before the call plus its number
// among the row's new tokens.  Tokens without a page, or of no row, are left out.
__global__ void __launch_bounds__(256) write_kernel(WriteArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int tok = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (tok >= a.tokens) return;
  int row = tok, back = 1;  // back: tokens from this one to the row's end
  if (a.cu) {
    // the first row whose end is past tok, 32 probes at a time
    int lo = 0, n = a.rows;
    while (n > 0) {
      const int step = (n + 31) >> 5, at = lo + lane * step + step - 1;
      const int c = __popc(__ballot_sync(0xffffffffu, at < lo + n && a.cu[at + 1] <= tok));
      const int end = lo + n;
      lo += c * step;
      n = min(step - 1, end - lo);
    }
    row = min(lo, a.rows);
    if (row < a.rows) {
      if (tok < a.cu[row]) return;  // before the first row's
      back = a.cu[row + 1] - tok;
    }
  }
  if (row >= a.rows) return;
  const int pos = a.lengths[row] - back;
  if (pos < 0 || (pos >> a.page_shift) >= a.width) return;
  const int page = a.table[static_cast<int64_t>(row) * a.width + (pos >> a.page_shift)];
  if (page < 0 || page >= a.p.pages) return;
  const int slot = pos & ((1 << a.page_shift) - 1);
  const int n = a.p.heads * a.p.chunks;
  for (int i = lane; i < n; i += 32) {
    const int h = i / a.p.chunks, c = i % a.p.chunks;
    const uint4 x = *reinterpret_cast<const uint4 *>(a.k + tok * a.k_token + h * a.k_head + c * 16);
    const uint4 y = *reinterpret_cast<const uint4 *>(a.v + tok * a.v_token + h * a.v_head + c * 16);
    *reinterpret_cast<uint4 *>(a.p.k + page * a.p.ks[1] + h * a.p.ks[2] + slot * a.p.ks[3] + c * 16) = x;
    *reinterpret_cast<uint4 *>(a.p.v + page * a.p.vs[1] + h * a.p.vs[2] + slot * a.p.vs[3] + c * 16) = y;
  }
}

constexpr int kNearBytes = 160 * 1024;

// One CTA while a scan of the counts and the tables is short; a cluster of eight
// shares longer ones.
int cluster_for(int64_t rows, int64_t width, int64_t pages) { return rows * width + pages <= 32768 ? 1 : 8; }

// The most shared memory that a kernel may ask for, whatever this call needs: a limit that
// followed the calls could be lowered by another thread between its setting and the launch.
template <bool NEAR>
constexpr int kForkMost = NEAR ? kNearBytes : kCacheMaxRows * 20;
template <bool NEAR>
constexpr int kExtendMost = NEAR ? kNearBytes : kCacheMaxRows * 12;

template <typename... KArgs, typename... Args>
int launch_kernel(const char *what, void (*kern)(KArgs...), int ctas, size_t smem, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  if (ctas == 1) return launch_pdl(what, kern, dim3(1), dim3(kThreads), smem, s, args...);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
  if (e != cudaSuccess) return fail(QS_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
  return QS_OK;
}

template <auto kern, int most, typename... Args>
int launch_cluster(const char *what, int ctas, size_t smem, cudaStream_t s, Args... args) {
  static std::atomic<uint64_t> allowed{0};
  const int st = most > 48 * 1024 ? allow_smem(what, kern, most, allowed) : QS_OK;
  return st ? st : launch_kernel(what, kern, ctas, smem, s, args...);
}

int log2_of(int64_t v) {
  int s = 0;
  while ((int64_t(1) << s) < v) ++s;
  return s;
}

int launch_copy(const qs_kv_pool &pool, const Work &w, cudaStream_t s) {
  return launch_pdl("copy_pages", copy_pages_kernel, dim3(device_sms() * 8), dim3(256), 0, s, make_pool(pool),
                    static_cast<int>(pool.page), static_cast<const int *>(w.head), static_cast<const int4 *>(w.list));
}

}  // namespace

int64_t cache_workspace_bytes(int64_t rows, int64_t pages) { return (64 + 4 * (rows + pages) + 3 * pages) * 4; }

int device_sms() {
  static int cached[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && cached[dev]) return cached[dev];
  int n = 148;
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  if (dev >= 0 && dev < 64) cached[dev] = n;
  return n;
}

int take_cache_error(int *bit, cudaStream_t s) {
  int bits = 0;
  QS_CUDA_TRY(cudaMemcpyFromSymbolAsync(&bits, g_cache_error, sizeof(int), 0, cudaMemcpyDeviceToHost, s));
  QS_CUDA_TRY(cudaStreamSynchronize(s));
  *bit = bits & kCacheErrPages ? kCacheErrPages : bits;
  if (*bit) {  // that one alone: what another stream raises meanwhile stays
    clear_error_kernel<<<1, 1, 0, s>>>(*bit);
    QS_CUDA_TRY(cudaGetLastError());
    QS_CUDA_TRY(cudaStreamSynchronize(s));
  }
  return QS_OK;
}

int launch_cache_fork(const qs_kv_pool &pool, int rows, int width, const int *table, const int *lengths,
                      const int *refcount, const int *parents, int *table_out, int *lengths_out, int *refcount_out,
                      void *ws, cudaStream_t s) {
  const Tables t{rows, width, static_cast<int>(pool.pages), log2_of(pool.page), table, lengths, refcount,
                 table_out, lengths_out, refcount_out};
  const Work w = split_work(ws, rows, pool.pages);
  const int ctas = cluster_for(rows, width, pool.pages);
  const size_t near = static_cast<size_t>(rows) * 24 + pool.pages * 4;
  const int st = ctas == 1 && near <= kNearBytes
                     ? launch_cluster<fork_kernel<true>, kForkMost<true>>("cache fork", ctas, near, s, t, parents, w)
                     : launch_cluster<fork_kernel<false>, kForkMost<false>>("cache fork", ctas, static_cast<size_t>(rows) * 20, s,
                                                                            t, parents, w);
  return st ? st : launch_copy(pool, w, s);
}

int launch_cache_compact(const qs_kv_pool &pool, int rows, int width, const int *table, const int *lengths,
                         const int *refcount, int *table_out, int *refcount_out, int *used_out, void *ws,
                         cudaStream_t s) {
  const Tables t{rows, width, static_cast<int>(pool.pages), log2_of(pool.page), table, lengths, refcount,
                 table_out, nullptr, refcount_out};
  const Work w = split_work(ws, rows, pool.pages);
  const int st = launch_cluster<compact_kernel, 0>("cache compact", cluster_for(rows, width, pool.pages), 0, s, t, used_out, w);
  return st ? st : launch_copy(pool, w, s);
}

int launch_cache_extend(int64_t page, int64_t pages, int rows, int width, const int *table, const int *lengths,
                        const int *refcount, const int *add, int *table_out, int *lengths_out, int *refcount_out,
                        void *ws, cudaStream_t s) {
  const Tables t{rows, width, static_cast<int>(pages), log2_of(page), table, lengths, refcount,
                 table_out, lengths_out, refcount_out};
  const Work w = split_work(ws, rows, pages);
  const int ctas = cluster_for(rows, width, pages);
  const size_t near = static_cast<size_t>(rows) * 12 + pages * 8;
  if (ctas == 1 && near <= kNearBytes)
    return launch_cluster<extend_kernel<true>, kExtendMost<true>>("cache extend", ctas, near, s, t, add, w);
  return launch_cluster<extend_kernel<false>, kExtendMost<false>>("cache extend", ctas, static_cast<size_t>(rows) * 12, s, t,
                                                                  add, w);
}

int launch_cache_write(const qs_kv_pool &pool, int rows, int width, const int *table, const int *lengths,
                       const int *cu, const void *k, int64_t k_token, int64_t k_head, const void *v, int64_t v_token,
                       int64_t v_head, int64_t tokens, cudaStream_t s) {
  const WriteArgs a{make_pool(pool), rows, width, log2_of(pool.page), static_cast<int>(tokens), table, lengths, cu,
                    static_cast<const char *>(k), static_cast<const char *>(v), k_token * 2, k_head * 2,
                    v_token * 2, v_head * 2};
  return launch_pdl("cache write", write_kernel, dim3(static_cast<unsigned>(ceil_div(tokens, 8))), dim3(256), 0, s, a);
}

}  // namespace qs
