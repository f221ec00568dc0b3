// Attention of one new token per row over the paged cache.
//
// The query heads that share a key head form the 16 rows of mma.sync m16n8k16 (more
// than 16 take further blocks of 16), so each key and value is read once for all of
// them.  A warp works alone: it streams groups of 16 keys (one page each) through its
// own cp.async ring, keeps the running maximum, sum and output of a softmax in
// registers, and meets the other warps of its CTA only when a segment ends.
//
// Rows differ in length, so the work is cut by keys, not by rows: the groups of all
// (row, key head) segments form one line that is dealt out in equal ranges, whatever the
// lengths, a few ranges for each place a CTA can run (SMs reach memory at different rates:
// with one range for each, the slowest made the others idle for a fifth of the time).  A
// segment that several ranges share leaves partial results (maximum, sum, output in
// float32), which attn_join_kernel puts together in order.  Where no row can see more than
// kWholeGroups groups (short tables, short windows), a CTA takes a segment whole and
// there is nothing to join; where segments are few, the CTAs of a cluster share it and join
// over each other's shared memory.
//
// Bound: the keys and values seen, once, at HBM rate.  Measured: 64 rows of 100 to 16000
// tokens, 64 query heads over 8 of 128, bfloat16: 318 to 330 us for 2.0 GB (6.1 to 6.3 TB/s);
// 48 rows under a window of 1000, 28 heads over 4 of 64: 13.7 us (46 MB, 3.4 TB/s: 192
// segments of unequal length, and a step's latency); one row of 203 tokens 5.4 us, latency
// alone; one row of 1500, 8 key heads, 6.9.
#include <cmath>
#include <type_traits>

#include "qs_attn.cuh"

namespace qs {
namespace {

constexpr int kRangesPerCta = 4;  // 64 rows of up to 16000 tokens: 337, 327, 321, 319, 322 us with 1, 2, 3, 4, 6
constexpr int kStages = 3;
constexpr int kKeys = 16;         // keys of a group
constexpr float kBias = 12.f;     // no weight is above 2^12
constexpr int kRows = 16;         // query heads of a block
constexpr int kCtasPerSm = 2;     // of four warps
constexpr int kDealWarps = 4;     // warps of a CTA that is dealt ranges
constexpr int kRanges = 148 * kCtasPerSm * kRangesPerCta;
constexpr int kMinRange = 16;     // groups of a range at least: 4 per warp, or the joins cost more than the split saves
constexpr int kLongRange = 128;   // the start of a shorter range is not paid for by the evener shares
constexpr int kWholeGroups = 80;  // for each CTA of a segment; one of four warps takes 20 steps for them

// The groups of 16 keys that a row's newest token sees: the first `sink` groups, then
// those from `from` on.
struct Seen {
  int n, lo, sink_keys;  // keys in places >= lo or < sink_keys are seen
  int sink, from, count;
};

__device__ __forceinline__ Seen seen_of(int length, const AttnArgs &a) {
  Seen s;
  const int64_t cap = static_cast<int64_t>(a.width) << a.page_shift;
  s.n = static_cast<int>(min(cap, static_cast<int64_t>(max(0, length))));
  s.lo = a.window > 0 && length > a.window ? static_cast<int>(length - a.window) : 0;
  s.lo = min(s.lo, s.n);
  s.sink_keys = static_cast<int>(min(static_cast<int64_t>(s.lo), a.sinks));
  s.sink = (s.sink_keys + kKeys - 1) / kKeys;
  s.from = max(s.lo / kKeys, s.sink);
  s.count = s.sink + max(0, (s.n + kKeys - 1) / kKeys - s.from);
  return s;
}

// How the line of groups is dealt (the same in every CTA and in the join).
struct Deal {
  int64_t total;  // padded groups of all segments
  int range;      // groups per range
  int pad;        // segments take multiples of this many groups
};

__device__ __forceinline__ int padded(int count, int pad) { return (count + pad - 1) / pad * pad; }

struct Ws {
  int64_t *start;  // [rows + 1]: padded groups of one head before the row
  int *deal;       // range, pad
  float *ml;       // [slot][16][2]
  float *o;        // [slot][16][DP]
};

template <typename T, int DP, int W>
struct Smem {
  T kv[W][kStages][2][kKeys * DP];
  float ml[W][kRows][2];
  float joined[kRows][2];  // of this CTA's warps
  int64_t sums[W * 32 + 1][2];
  int lengths[W * 32];  // of the first rows
};

// The CTAs of a cluster (where a segment is shared by several).
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
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float2 peer_pair(const float *mine, int rank) {  // the same place in another CTA's memory
  uint32_t at;
  float2 x;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(at) : "memory");
  return x;
}

// One warp's softmax state over 16 query rows (R8: only the first 8 are real).
template <typename T, int DP, bool R8>
struct Warp {
  uint32_t q[DP / 16][4];
  float o[DP / 8][4];
  float m[2], l[2];

  __device__ __forceinline__ void load_q(const AttnArgs &a, int64_t row, int head0, int heads, int lane) {
    const int g = lane >> 2, t = lane & 3;
    const T *base = static_cast<const T *>(a.q) + row * a.q_token;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = g + (i & 1) * 8, d = k * 16 + (i >> 1) * 8 + 2 * t;
        q[k][i] = r < heads && d < a.dim
                      ? *reinterpret_cast<const uint32_t *>(base + (head0 + r) * a.q_head + d) : 0u;
      }
  }
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int j = 0; j < DP / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  }
  // 16 keys at kv (keys, then values, swizzled rows); bit i of `mask`: key i is seen.
  __device__ __forceinline__ void step(uint32_t ks, uint32_t vs, uint32_t mask, float scale2, int lane) {
    float s[2][4] = {};
    const int r8 = lane & 7, hi = (lane >> 3) & 1, top = lane >> 4;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      uint32_t b[4];
      ldmatrix_x4(b, ks + swizzled<DP>(r8 + 8 * top, 2 * k + hi));
      mma16816<T>(s[0], q[k], b[0], b[1]);
      mma16816<T>(s[1], q[k], b[2], b[3]);
    }
    const int t = lane & 3;
    float top_s[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < (R8 ? 2 : 4); ++i) {
        s[j][i] *= scale2;
        if (mask != 0xffffu && !((mask >> (8 * j + 2 * t + (i & 1))) & 1)) s[j][i] = -INFINITY;
        top_s[i >> 1] = fmaxf(top_s[i >> 1], s[j][i]);
      }
    bool grew = false;
    float mn[2], alpha[2];
#pragma unroll
    for (int h = 0; h < (R8 ? 1 : 2); ++h) {
      top_s[h] = fmaxf(top_s[h], __shfl_xor_sync(0xffffffffu, top_s[h], 1));
      top_s[h] = fmaxf(top_s[h], __shfl_xor_sync(0xffffffffu, top_s[h], 2));
      mn[h] = fmaxf(m[h], top_s[h]);
      grew |= mn[h] > m[h];
      alpha[h] = mn[h] == -INFINITY ? 1.f : ex2(m[h] - mn[h]);
      m[h] = mn[h];
    }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int h = 0; h < (R8 ? 1 : 2); ++h) {
        l[h] *= alpha[h];
#pragma unroll
        for (int j = 0; j < DP / 8; ++j) o[j][2 * h] *= alpha[h], o[j][2 * h + 1] *= alpha[h];
      }
    }
    // The weights enter the second product as the sum of two 16-bit values (what the
    // first leaves of 24 bits, the second takes), so they lose nothing that the output's
    // rounding would show; the extra products are hidden behind the loads.  They are
    // 2^kBias times what the softmax has, which keeps small ones in float16's range.
    uint32_t ph[4] = {}, pl[4] = {};
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int h = 0; h < (R8 ? 1 : 2); ++h) {
        const float base = m[h] == -INFINITY ? 0.f : m[h] - kBias;
        const float x = ex2(s[j][2 * h] - base), y = ex2(s[j][2 * h + 1] - base);
        l[h] += x + y;
        const float2 back = split16<T>(x, y, ph[2 * j + h]);
        float2 unused;
        unused = split16<T>(x - back.x, y - back.y, pl[2 * j + h]);
        (void)unused;
      }
#pragma unroll
    for (int j = 0; j < DP / 16; ++j) {
      uint32_t b[4];
      ldmatrix_x4_trans(b, vs + swizzled<DP>(r8 + 8 * hi, 2 * j + top));
      mma16816<T>(o[2 * j], ph, b[0], b[1]);
      mma16816<T>(o[2 * j + 1], ph, b[2], b[3]);
      mma16816<T>(o[2 * j], pl, b[0], b[1]);
      mma16816<T>(o[2 * j + 1], pl, b[2], b[3]);
    }
  }
};

template <typename T, int DP, bool R8, int W, bool WHOLE>
__global__ void __launch_bounds__(W * 32, W == 4 || DP == 64 ? 2 : 1)
attn_decode_kernel(AttnArgs a, Ws ws, int blocks, int share) {
  extern __shared__ __align__(128) uint8_t dsm[];
  using S = Smem<T, DP, W>;
  S &sm = *reinterpret_cast<S *>(dsm);
  constexpr int kThreads = W * 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_launch_dependents();

  const T *kbase = static_cast<const T *>(a.k), *vbase = static_cast<const T *>(a.v);
  const float scale2 = a.scale * kLog2e;
  constexpr int CPR = DP / 8;            // 16-byte pieces of a key
  constexpr int RPI = 32 / CPR;          // keys per warp-wide copy
  const int piece = lane % CPR, sub = lane / CPR;
  const uint32_t ring = smem_u32(&sm.kv[warp][0][0][0]);

  // Groups [u0, u1) of one segment; `slot`: where a partial result goes.
  auto segment = [&](int row, int head, const Seen &seen, int u0, int u1, int64_t slot) {
    const int kvh = head / blocks, h0 = kvh * share + (head % blocks) * kRows;
    const int hn = min(kRows, share - (head % blocks) * kRows);
    const int *table = a.table + static_cast<int64_t>(row) * a.width;
    Warp<T, DP, R8> w;
    w.load_q(a, row, h0, hn, lane);

    const int mine = u1 - u0 - warp > 0 ? (u1 - u0 - warp + W - 1) / W : 0;
    auto group_of = [&](int it) {
      const int u = u0 + warp + it * W;
      return u < seen.sink ? u : seen.from + (u - seen.sink);
    };
    // lane i: the page of this warp's group 32 * block + i, for the groups being loaded and
    // for those being computed, which trail them
    int page_ids = -1, masks_page = -1;
    auto mask_of = [&](int g, int page) {  // bits of the group's keys that are seen
      if (page < 0 || page >= a.pages) return 0u;
      const int k0 = g * kKeys;
      if (k0 >= seen.lo && k0 + kKeys <= seen.n) return 0xffffu;  // most groups
      const uint32_t below = seen.n - k0 >= kKeys ? 0xffffu : (1u << (seen.n - k0)) - 1u;
      const int lo_k = seen.lo - k0, sink_k = seen.sink_keys - k0;
      const uint32_t recent = lo_k <= 0 ? 0xffffu : lo_k >= kKeys ? 0u : 0xffffu & ~((1u << lo_k) - 1u);
      const uint32_t sinks = sink_k <= 0 ? 0u : sink_k >= kKeys ? 0xffffu : (1u << sink_k) - 1u;
      return below & (recent | sinks);
    };
    // this lane's piece of a group's first key, and the step to its next one
    const bool real = piece * 8 < a.dim;
    const T *kp0 = kbase + kvh * a.ks[1] + sub * a.ks[2] + (real ? piece * 8 : 0);
    const T *vp0 = vbase + kvh * a.vs[1] + sub * a.vs[2] + (real ? piece * 8 : 0);
    const int64_t kstep = RPI * a.ks[2], vstep = RPI * a.vs[2];
    const int page_mask = (1 << a.page_shift) - 1;
    auto issue = [&](int it) {
      if (it < mine) {
        if ((it & 31) == 0) {
          page_ids = -1;
          if (it + lane < mine) page_ids = table[(group_of(it + lane) * kKeys) >> a.page_shift];
        }
        const int page = __shfl_sync(0xffffffffu, page_ids, it & 31);
        const int g = group_of(it);
        const uint32_t mask = mask_of(g, page);
        const int64_t pg = mask ? page : 0;
        const int slot_in_page = (g * kKeys) & page_mask;
        const T *kp = kp0 + pg * a.ks[0] + slot_in_page * a.ks[2];
        const T *vp = vp0 + pg * a.vs[0] + slot_in_page * a.vs[2];
        const uint32_t st = ring + (it % kStages) * (2 * kKeys * DP * 2);
        // a key that is not seen is not read: its place is zero, so nothing it holds can enter
#pragma unroll
        for (int i = 0; i < kKeys / RPI; ++i) {
          const int key = sub + i * RPI;
          const bool in = real && (mask == 0xffffu || ((mask >> key) & 1));
          const uint32_t dst = st + swizzled<DP>(key, piece);
          cp_async16(dst, kp + i * kstep, in);
          cp_async16(dst + kKeys * DP * 2, vp + i * vstep, in);
        }
      }
      cp_async_commit();
    };

    w.reset();
#pragma unroll
    for (int it = 0; it < kStages - 1; ++it) issue(it);
    masks_page = page_ids;
    for (int it = 0; it < mine; ++it) {
      if (it > 0 && (it & 31) == 0) masks_page = it + lane < mine ? table[(group_of(it + lane) * kKeys) >> a.page_shift] : -1;
      issue(it + kStages - 1);
      cp_async_wait<kStages - 1>();
      __syncwarp();
      const uint32_t st = ring + (it % kStages) * (2 * kKeys * DP * 2);
      const uint32_t mask = mask_of(group_of(it), __shfl_sync(0xffffffffu, masks_page, it & 31));
      w.step(st, st + kKeys * DP * 2, mask, scale2, lane);
      __syncwarp();
    }
    cp_async_wait<0>();

    // the CTA's warps meet: outputs through shared memory (their own rings)
    float *mine_o = reinterpret_cast<float *>(&sm.kv[warp][0][0][0]);
    const int g = lane >> 2, t = lane & 3;
    __syncwarp();
#pragma unroll
    for (int h = 0; h < (R8 ? 1 : 2); ++h) {
      float l = w.l[h];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (t == 0) sm.ml[warp][g + 8 * h][0] = w.m[h], sm.ml[warp][g + 8 * h][1] = l;
#pragma unroll
      for (int j = 0; j < DP / 8; ++j)
        *reinterpret_cast<float2 *>(mine_o + (g + 8 * h) * DP + 8 * j + 2 * t) =
            make_float2(w.o[j][2 * h], w.o[j][2 * h + 1]);
    }
    __syncthreads();
    const bool whole = u0 == 0 && u1 == seen.count;
    auto finish = [&](int r, int c2, float m, float l, float2 o) {
      const int64_t out = static_cast<int64_t>(row) * a.q_heads + h0 + r;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      uint32_t packed;
      split16<T>(o.x * inv, o.y * inv, packed);
      if (c2 < a.dim) *reinterpret_cast<uint32_t *>(static_cast<T *>(a.out) + out * a.dim + c2) = packed;
      if (c2 == 0 && a.lse) a.lse[out] = l == 0.f ? -INFINITY : (m - kBias + log2f(l)) * kLn2;
    };
    const int ctas = WHOLE ? cluster_size() : 1;
    float *first = reinterpret_cast<float *>(&sm.kv[0][0][0][0]);
    for (int i = tid; i < hn * (DP / 2); i += kThreads) {
      const int r = i / (DP / 2), c2 = i % (DP / 2) * 2;
      float m = -INFINITY, l = 0.f;
      float2 o = make_float2(0.f, 0.f);
#pragma unroll
      for (int v = 0; v < W; ++v) m = fmaxf(m, sm.ml[v][r][0]);
#pragma unroll
      for (int v = 0; v < W; ++v) {
        const float f = weight(sm.ml[v][r][0], m);
        const float2 x = *reinterpret_cast<const float2 *>(reinterpret_cast<const float *>(&sm.kv[v][0][0][0]) + r * DP + c2);
        l += f * sm.ml[v][r][1];
        o.x += f * x.x;
        o.y += f * x.y;
      }
      if (WHOLE && ctas > 1) {  // over what this thread alone has read
        *reinterpret_cast<float2 *>(first + r * DP + c2) = o;
        if (c2 == 0) sm.joined[r][0] = m, sm.joined[r][1] = l;
      } else if (WHOLE || whole) {
        finish(r, c2, m, l, o);
      } else {
        *reinterpret_cast<float2 *>(ws.o + (slot * kRows + r) * DP + c2) = o;
        if (c2 == 0) ws.ml[(slot * kRows + r) * 2] = m, ws.ml[(slot * kRows + r) * 2 + 1] = l;
      }
    }
    if (WHOLE && ctas > 1) {  // each CTA takes its part of the outputs, over all CTAs' sums
      cluster_barrier();
      for (int i = cluster_rank() * kThreads + tid; i < hn * (DP / 2); i += ctas * kThreads) {
        const int r = i / (DP / 2), c2 = i % (DP / 2) * 2;
        float m = -INFINITY, l = 0.f;
        float2 o = make_float2(0.f, 0.f);
        for (int v = 0; v < ctas; ++v) m = fmaxf(m, peer_pair(sm.joined[r], v).x);
        for (int v = 0; v < ctas; ++v) {
          const float2 ml = peer_pair(sm.joined[r], v), x = peer_pair(first + r * DP + c2, v);
          const float f = weight(ml.x, m);
          l += f * ml.y;
          o.x += f * x.x;
          o.y += f * x.y;
        }
        finish(r, c2, m, l, o);
      }
      cluster_barrier();  // no CTA leaves while another reads from it
      return;
    }
    __syncthreads();
  };

  const int heads = a.kv_heads * blocks;  // segments per row
  if (WHOLE) {
    const int ctas = cluster_size(), at = blockIdx.x / ctas, row = at / heads, rank = cluster_rank();
    const Seen seen = seen_of(a.lengths[row], a);
    segment(row, at % heads, seen, seen.count * rank / ctas, seen.count * (rank + 1) / ctas, 0);
    return;
  }

  // ---- the line of groups: counts per thread's rows, then their prefix
  const int per = (a.rows + kThreads - 1) / kThreads;
  const int first_row = min(a.rows, tid * per), last_row = min(a.rows, first_row + per);
  {
    int64_t c = 0, p = 0;
    for (int r = first_row; r < last_row; ++r) {
      const int length = a.lengths[r], n = seen_of(length, a).count;
      if (r == tid) sm.lengths[tid] = length;  // a row per thread: they are all here
      c += n;
      p += padded(n, kMinRange);
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, c, d), y = __shfl_up_sync(0xffffffffu, p, d);
      if (lane >= d) c += x, p += y;
    }
    sm.sums[tid + 1][0] = c;
    sm.sums[tid + 1][1] = p;
    if (tid == 0) sm.sums[0][0] = sm.sums[0][1] = 0;
    __syncthreads();
    int64_t before_c = 0, before_p = 0;
    for (int v = 0; v < warp; ++v) before_c += sm.sums[v * 32 + 32][0], before_p += sm.sums[v * 32 + 32][1];
    __syncthreads();
    sm.sums[tid + 1][0] = c + before_c;
    sm.sums[tid + 1][1] = p + before_p;
    __syncthreads();
  }
  // Enough groups for every CTA: one unpadded line in equal ranges.  Else short ranges
  // that begin with their segments, so that most segments need no join.
  Deal d;
  const int64_t groups = sm.sums[kThreads][0] * heads;
  const bool dense = groups >= static_cast<int64_t>(148 * kCtasPerSm) * kMinRange;
  const int col = dense ? 0 : 1;
  d.pad = dense ? 1 : kMinRange;
  d.total = sm.sums[kThreads][col] * heads;
  const int64_t one_each = (d.total + 148 * kCtasPerSm - 1) / (148 * kCtasPerSm);
  d.range = dense ? static_cast<int>(max(min(one_each, static_cast<int64_t>(kLongRange)), (d.total + kRanges - 1) / kRanges))
                  : kMinRange;
  if (blockIdx.x == 0) {  // for the join
    int64_t at = sm.sums[tid][col];
    for (int r = first_row; r < last_row; ++r) {
      ws.start[r] = at;
      at += padded(seen_of(a.lengths[r], a).count, d.pad);
    }
    if (tid == 0) {
      ws.start[a.rows] = sm.sums[kThreads][col];
      ws.deal[0] = d.range;
      ws.deal[1] = d.pad;
    }
  }

  const int64_t ranges = (d.total + d.range - 1) / d.range;
  for (int64_t range = blockIdx.x; range < ranges; range += gridDim.x) {
    const int64_t r0 = range * d.range, r1 = min(d.total, r0 + d.range);
    // the row that holds group r0: the thread's block of rows by its prefix, then row by row
    int lo = 0, hi = kThreads;
    while (lo + 1 < hi) {
      const int mid = (lo + hi) >> 1;
      if (sm.sums[mid][col] * heads <= r0) lo = mid;
      else hi = mid;
    }
    int row = lo * per;
    int64_t at = sm.sums[lo][col] * heads;  // the row's first group
    int64_t pos = r0;
    while (pos < r1 && row < a.rows) {
      const Seen seen = seen_of(per == 1 ? sm.lengths[row] : a.lengths[row], a);
      const int c = padded(seen.count, d.pad);
      if (at + static_cast<int64_t>(c) * heads <= pos) {
        at += static_cast<int64_t>(c) * heads;
        ++row;
        continue;
      }
      const int head = static_cast<int>((pos - at) / c);
      const int64_t seg = at + static_cast<int64_t>(head) * c;  // the segment's first group
      const int u0 = static_cast<int>(pos - seg);
      const int u1 = static_cast<int>(min(static_cast<int64_t>(seen.count), r1 - seg));
      pos = min(r1, seg + c);
      if (u0 < u1) segment(row, head, seen, u0, u1, dense ? 2 * range + (seg > r0 ? 1 : 0) : range);
    }
  }
}

// Joins the partial results of one segment's ranges, in their order; segments that no range
// covers (rows that see nothing) get zeros.  A warp for each query row, or, where the rows
// are few and their parts may be many, four (WPR) that take every fourth part each.
template <typename T, int DP, int WPR>
__global__ void __launch_bounds__(128) attn_join_kernel(AttnArgs a, Ws ws, int blocks, int share) {
  constexpr int PER = DP / 32, U = 4, ROWS = 4 / WPR;  // outputs per lane, parts at a time, rows of a CTA
  __shared__ float sums[WPR > 1 ? 4 : 1][DP + 1];
  pdl_wait();
  pdl_launch_dependents();
  const int heads = a.kv_heads * blocks, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int segment = blockIdx.x / (kRows / ROWS), r = blockIdx.x % (kRows / ROWS) * ROWS + warp / WPR;
  const int row = segment / heads, head = segment % heads;
  const int kvh = head / blocks, h0 = kvh * share + (head % blocks) * kRows;
  const int range = ws.deal[0], pad = ws.deal[1];
  const int64_t start = ws.start[row];
  const int count = seen_of(a.lengths[row], a).count;
  if (r >= min(kRows, share - (head % blocks) * kRows)) return;  // with several warps a row, the whole CTA
  const int64_t seg = start * heads + static_cast<int64_t>(head) * padded(count, pad);
  const int64_t f = seg / range, e = count ? (seg + count - 1) / range : f;
  if (count && f == e) return;  // one range had it whole
  const int parts = count ? static_cast<int>(e - f) + 1 : 0;
  auto slot_of = [&](int i) { return pad == 1 ? 2 * (f + i) + (i == 0 && seg > f * range ? 1 : 0) : f + i; };
  float m = -INFINITY;
  for (int i = lane; i < parts; i += 32) m = fmaxf(m, ws.ml[(slot_of(i) * kRows + r) * 2]);
#pragma unroll
  for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  float l = 0.f, o[PER] = {};
  for (int i0 = warp % WPR; i0 < parts; i0 += U * WPR) {
    float2 ml[U];
    float x[U][PER];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * WPR;
      if (i < parts) {
        const int64_t at = slot_of(i) * kRows + r;
        ml[u] = *reinterpret_cast<const float2 *>(ws.ml + at * 2);
#pragma unroll
        for (int c = 0; c < PER; ++c) x[u][c] = ws.o[at * DP + lane * PER + c];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u * WPR >= parts) break;
      const float p = weight(ml[u].x, m);
      l += p * ml[u].y;
#pragma unroll
      for (int c = 0; c < PER; ++c) o[c] += p * x[u][c];
    }
  }
  if (WPR > 1) {
#pragma unroll
    for (int c = 0; c < PER; ++c) sums[warp][lane * PER + c] = o[c];
    if (lane == 0) sums[warp][DP] = l;
    __syncthreads();
    if (warp) return;
#pragma unroll
    for (int v = 1; v < 4; ++v) {
      l += sums[v][DP];
#pragma unroll
      for (int c = 0; c < PER; ++c) o[c] += sums[v][lane * PER + c];
    }
  }
  const int64_t out = static_cast<int64_t>(row) * a.q_heads + h0 + r;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int c = 0; c < PER; c += 2) {
    uint32_t packed;
    split16<T>(o[c] * inv, o[c + 1] * inv, packed);
    if (lane * PER + c < a.dim)
      *reinterpret_cast<uint32_t *>(static_cast<T *>(a.out) + out * a.dim + lane * PER + c) = packed;
  }
  if (lane == 0 && a.lse) a.lse[out] = l == 0.f ? -INFINITY : (m - kBias + log2f(l)) * kLn2;
}

struct Shape {
  int64_t heads, slots;
  int dp;
};

Shape shape_of(int64_t rows, int64_t q_heads, int64_t kv_heads, int64_t dim) {
  Shape s;
  s.heads = kv_heads * ceil_div(q_heads / kv_heads, kRows);
  // equal ranges leave up to two partial results each; short ranges one, and there are
  // no more of them than the CTAs plus one for each segment's last
  const int64_t some = 148 * kCtasPerSm + rows * s.heads;
  s.slots = 2 * kRanges > some ? 2 * kRanges : some;
  s.dp = dim <= 64 ? 64 : 128;
  return s;
}

// Groups that a row can see at most, by its line and the window.
int64_t most_groups(int64_t page, int64_t width, int64_t window, int64_t sinks) {
  int64_t keys = width * page;
  if (window > 0 && window < keys && sinks < keys && window + sinks < keys)
    keys = window + sinks + 2 * kKeys;  // both ends inside a group
  return ceil_div(keys, kKeys);
}

// CTAs (of four warps) that share a segment as a cluster: where segments are few, as many as
// the SMs hold, each with two groups a warp or more.  Eight heads of 128 under a window of
// 1000: one row 11.5 us with one CTA of eight warps, 7.4 with clusters of 4, 6.0 of 8; 8 rows
// 12.7, 10.0, 15.1; 16 rows 15.2 and 21 (each CTA alone again).  30 keys: 3.6, 5.0, 5.1.
int ctas_of(int64_t segments, int64_t most) {
  if (segments * 8 <= 148 * kCtasPerSm && most >= 64) return 8;
  if (segments * 4 <= 148 * kCtasPerSm && most >= 32) return 4;
  return 1;
}

// Whether each segment is taken whole (see kWholeGroups).  More CTAs take longer ones: 1500
// keys of one row 9.9 us dealt and 6.9 whole, 3800 10.4 both; 8 rows of up to 2000 18.9 and 14.4.
bool taken_whole(int64_t segments, int64_t most) {
  const int ctas = ctas_of(segments, most);
  return most <= kWholeGroups * (ctas == 8 ? 3 : ctas == 4 ? 2 : 1);
}

template <typename... KArgs>
int launch_clusters(void (*kern)(KArgs...), int64_t clusters, int ctas, int threads, int smem, cudaStream_t s,
                    KArgs... args) {
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * ctas));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  return e == cudaSuccess ? QS_OK : fail(QS_ERR_CUDA, "attention (decode): %s", cudaGetErrorString(e));
}

template <typename T, int DP, bool R8, int W, bool WHOLE>
int run(const AttnArgs &a, const Ws &ws, int blocks, int share, int64_t grid, cudaStream_t s, int ctas = 1) {
  auto kern = attn_decode_kernel<T, DP, R8, W, WHOLE>;
  constexpr int smem = static_cast<int>(sizeof(Smem<T, DP, W>));
  static std::atomic<uint64_t> allowed{0};
  const int st = allow_smem("attention (decode)", kern, smem, allowed);
  if (st) return st;
  if (ctas > 1) return launch_clusters(kern, grid, ctas, W * 32, smem, s, a, ws, blocks, share);
  return launch_pdl("attention (decode)", kern, dim3(static_cast<unsigned>(grid)), dim3(W * 32), smem, s, a, ws, blocks,
                    share);
}

template <typename T, int DP, bool R8>
int run_shape(const AttnArgs &a, const Ws &ws, int blocks, int share, cudaStream_t s) {
  const int64_t segments = static_cast<int64_t>(a.rows) * a.kv_heads * blocks, most = most_groups(int64_t(1) << a.page_shift, a.width, a.window, a.sinks);
  if (taken_whole(segments, most)) {
    const int ctas = ctas_of(segments, most);
    if (ctas > 1) return run<T, DP, R8, 4, true>(a, ws, blocks, share, segments, s, ctas);
    // eight warps where all segments run at once anyway
    if (segments <= 148 * (DP == 64 ? 2 : 1)) return run<T, DP, R8, 8, true>(a, ws, blocks, share, segments, s);
    return run<T, DP, R8, 4, true>(a, ws, blocks, share, segments, s);
  }
  const int64_t fewest = ceil_div(most, kMinRange) * segments;  // ranges there can be
  const int st = run<T, DP, R8, kDealWarps, false>(a, ws, blocks, share, fewest < kRanges ? fewest : kRanges, s);
  if (st) return st;
  if (segments <= 148)
    return launch_pdl("attention (join)", attn_join_kernel<T, DP, 4>, dim3(static_cast<unsigned>(segments * kRows)),
                      dim3(128), 0, s, a, ws, blocks, share);
  return launch_pdl("attention (join)", attn_join_kernel<T, DP, 1>, dim3(static_cast<unsigned>(segments * (kRows / 4))),
                    dim3(128), 0, s, a, ws, blocks, share);
}

template <typename T>
int run_type(const AttnArgs &a, const Ws &ws, int blocks, int share, cudaStream_t s) {
  if (a.dim <= 64)
    return share <= 8 ? run_shape<T, 64, true>(a, ws, blocks, share, s) : run_shape<T, 64, false>(a, ws, blocks, share, s);
  return share <= 8 ? run_shape<T, 128, true>(a, ws, blocks, share, s) : run_shape<T, 128, false>(a, ws, blocks, share, s);
}

}  // namespace

int64_t attn_decode_workspace_bytes(int64_t rows, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t page,
                                    int64_t width, int64_t window, int64_t sinks) {
  const Shape s = shape_of(rows, q_heads, kv_heads, dim);
  const int64_t most = most_groups(page, width, window, sinks);
  if (taken_whole(rows * s.heads, most)) return 0;
  return round_up((rows + 1) * 8 + 8, 256) + s.slots * kRows * (s.dp + 2) * 4;
}

int launch_attn_decode(const AttnArgs &a, cudaStream_t s) {
  const int share = a.q_heads / a.kv_heads, blocks = static_cast<int>(ceil_div(share, kRows));
  const Shape sh = shape_of(a.rows, a.q_heads, a.kv_heads, a.dim);
  Ws ws;
  ws.start = static_cast<int64_t *>(a.ws);
  ws.deal = reinterpret_cast<int *>(ws.start + a.rows + 1);
  ws.ml = reinterpret_cast<float *>(static_cast<char *>(a.ws) + round_up((a.rows + 1) * int64_t(8) + 8, 256));
  ws.o = ws.ml + sh.slots * kRows * 2;
  return a.dtype == QS_F16 ? run_type<__half>(a, ws, blocks, share, s)
                           : run_type<__nv_bfloat16>(a, ws, blocks, share, s);
}

}  // namespace qs
