// Beam search's selection: the best n of beams x vocabulary continuations by
//   score[b] + (x - m) - log(sum exp(x - m)),   m = max x.
//
// One pass over the logits.  A beam's scores fall with its logits, so its n best
// continuations are its n largest logits, and the log-sum, which is not known until
// the row ends, is not needed to find them.  beam_scan: each CTA takes a chunk of
// one row; its threads keep a running maximum and sum of exponentials, and their
// largest logit.  The n-th largest of those thread maxima is a bound that at least
// n logits of the chunk reach and few others do, so only the few threads whose
// maximum reaches it look at their logits again.  beam_merge: one CTA per search
// joins the chunks' lists into the beams', and the beams' into the result; a candidate's
// place is the number of those ahead of it, so nothing is sorted and nothing depends on
// the order of arrival.
//
// Bound: the logits' bytes, once.
#include <cmath>

#include "qs_common.cuh"
#include "qs_launch.h"
#include "qs_pair.cuh"

namespace qs {
namespace {

constexpr int kT = 512;        // threads of the merge
constexpr int kS = 128;        // threads of the scan
constexpr int kStep = 4;       // 16-byte pieces that a scanning thread takes at a time
constexpr int kRing = 2;       // steps of its ring in shared memory
constexpr int kCap = 1024;     // candidates of a chunk kept in shared memory
constexpr int kItems = 512;    // pieces that are looked at again
constexpr int kMinChunk = 2048;
constexpr int kScanCtas = 8;   // scanning CTAs per SM
constexpr int kLists = 4096;   // candidates merged at a time
constexpr float kLog2e = 1.4426950408889634f;

template <typename T> struct Vec;  // a 16-byte piece of a row
template <> struct Vec<float> {
  static constexpr int n = 4;
  __device__ static void unpack(const uint4 &w, float (&v)[4]) {
    v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
  }
  template <int U>
  __device__ static float top(const uint4 (&w)[U]) {  // NaN only where all are
    float t = __uint_as_float(w[0].x);
#pragma unroll
    for (int u = 0; u < U; ++u)
      t = fmaxf(t, fmaxf(fmaxf(__uint_as_float(w[u].x), __uint_as_float(w[u].y)),
                         fmaxf(__uint_as_float(w[u].z), __uint_as_float(w[u].w))));
    return t;
  }
  __device__ static uint4 none() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }  // -inf
  __device__ static float one(const float *p) { return *p; }
};
template <> struct Vec<__half> {
  static constexpr int n = 8;
  __device__ static __half2 pair(uint32_t x) { return *reinterpret_cast<const __half2 *>(&x); }
  __device__ static void unpack(const uint4 &w, float (&v)[8]) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(pair(a[i]));
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
  template <int U>
  __device__ static float top(const uint4 (&w)[U]) {
    auto t = pair(w[0].x);
#pragma unroll
    for (int u = 0; u < U; ++u)
      t = __hmax2(t, __hmax2(__hmax2(pair(w[u].x), pair(w[u].y)), __hmax2(pair(w[u].z), pair(w[u].w))));
    const float2 f = __half22float2(t);
    return fmaxf(f.x, f.y);
  }
  __device__ static uint4 none() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
  __device__ static float one(const __half *p) { return __half2float(*p); }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int n = 8;
  __device__ static __nv_bfloat162 pair(uint32_t x) { return *reinterpret_cast<const __nv_bfloat162 *>(&x); }
  __device__ static void unpack(const uint4 &w, float (&v)[8]) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(a[i] << 16);
      v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
    }
  }
  template <int U>
  __device__ static float top(const uint4 (&w)[U]) {
    auto t = pair(w[0].x);
#pragma unroll
    for (int u = 0; u < U; ++u)
      t = __hmax2(t, __hmax2(__hmax2(pair(w[u].x), pair(w[u].y)), __hmax2(pair(w[u].z), pair(w[u].w))));
    const float2 f = __bfloat1622float2(t);
    return fmaxf(f.x, f.y);
  }
  __device__ static uint4 none() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
  __device__ static float one(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
};

// Unsigned keys in the order of the values; -0 counts as 0, nothing as 0 (below -inf).
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void copy16(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

struct ScanArgs {
  const void *logits;
  int64_t batch_stride, beam_stride;
  int beams, vocab, n, chunks, chunk;  // chunk: 16-byte pieces per CTA
  float2 *stats;                       // [row][chunk]: reference b, sum of 2^(x c - b), c = log2(e) in float32
  uint2 *cand;                         // [row][chunk][n]: key, token
};

// Pieces of a row: piece j holds elements [j * n - skew, ...), so that whole pieces
// are aligned; the first and last may be partial and are read element by element.
template <typename T>
struct Row {
  static constexpr int NV = Vec<T>::n;
  const T *p;
  int vocab, skew;
  __device__ Row(const T *base, int v) : p(base), vocab(v) {
    skew = static_cast<int>((reinterpret_cast<uintptr_t>(base) & 15) / sizeof(T));
  }
  __device__ int first(int j) const { return j * NV - skew; }
  __device__ bool whole(int j) const { return first(j) >= 0 && first(j) + NV <= vocab; }
  __device__ uint4 raw(int j) const { return __ldg(reinterpret_cast<const uint4 *>(p + first(j))); }
  __device__ bool in(int e) const { return e >= 0 && e < vocab; }
  // NaN becomes -inf, places outside the row too
  __device__ void values(int j, float (&v)[NV]) const {
    if (whole(j)) {
      Vec<T>::unpack(raw(j), v);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = in(first(j) + i) ? Vec<T>::one(p + first(j) + i) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = fmaxf(v[i], -INFINITY);
  }
};

// A thread's sum of 2^(x c - b).  The reference b is a float32 near the maximum times c
// and is itself exact: x c - b is rounded once, so no term is off by more than its own
// distance to b, and it may lag behind the maximum by kLag, which float32 sums hold.
constexpr float kLag = 8.f;
struct Sum {
  float ref = -INFINITY, b = -INFINITY, l = 0.f;  // b = ref * c

  __device__ __forceinline__ void renew(float top) {
    const float nb = top * kLog2e;
    l *= b == nb ? 1.f : ex2(b - nb);
    ref = top;
    b = nb;
  }
  // Whatever the values: +inf counts alone, -inf nothing.
  template <int NV>
  __device__ __noinline__ void add_any(const float (&v)[NV]) {
    float top = v[0];
#pragma unroll
    for (int i = 1; i < NV; ++i) top = fmaxf(top, v[i]);
    if (top == INFINITY) {
      if (ref != INFINITY) l = 0.f, ref = b = INFINITY;
#pragma unroll
      for (int i = 0; i < NV; ++i) l += v[i] == INFINITY ? 1.f : 0.f;
    } else if (ref != INFINITY) {
      if (top > ref) renew(top);
      if (ref != -INFINITY)
#pragma unroll
        for (int i = 0; i < NV; ++i) l += ex2(fmaf(v[i], kLog2e, -b));
    }
  }
  // Pieces of ordinary numbers with maximum `top`; false (and nothing added) where there
  // are others.  Per number: half a multiply-add and half an addition (two at a time)
  // and the exponential.
  template <typename T, int U>
  __device__ __forceinline__ bool add(const uint4 (&w)[U], float top) {
    if (!(top <= ref + kLag)) {
      if (!(fabsf(top) < INFINITY)) return false;
      renew(top);
    }
    const uint64_t c2 = pack2(kLog2e, kLog2e), b2 = pack2(-b, -b);
    uint64_t s2 = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[Vec<T>::n];
      Vec<T>::unpack(w[u], v);
#pragma unroll
      for (int i = 0; i < Vec<T>::n; i += 2) {
        const float2 e = unpack2(fma2(pack2(v[i], v[i + 1]), c2, b2));
        s2 = add2(s2, pack2(ex2(e.x), ex2(e.y)));
      }
    }
    const float2 s = unpack2(s2);
    if (!(s.x + s.y < INFINITY)) return false;  // NaN or infinities among them
    l += s.x + s.y;
    return true;
  }
};

// Joins (b2, l2) into (b, l).
__device__ __forceinline__ void join(float &b, float &l, float b2, float l2) {
  const float m = fmaxf(b, b2);
  l = l * (b == m ? 1.f : ex2(b - m)) + l2 * (b2 == m ? 1.f : ex2(b2 - m));
  b = m;
}

__device__ __forceinline__ bool before(uint32_t k1, int t1, uint32_t k2, int t2) {
  return k1 > k2 || (k1 == k2 && t1 < t2);
}

template <typename T>
__global__ void __launch_bounds__(kS, kScanCtas) beam_scan_kernel(ScanArgs a) {
  constexpr int NV = Vec<T>::n, U = kStep, W = kS / 32;
  // the ring of the first phase, then the candidates of the second
  __shared__ union {
    uint4 ring[kRing][U][kS];
    struct {
      uint2 cand[kCap];
      int items[kItems];
    } found;
  } sm;
  uint2 *cand = sm.found.cand;
  int *items = sm.found.items;
  __shared__ uint32_t tops[kS];
  __shared__ float2 part[W];
  __shared__ uint2 best[W];
  __shared__ uint32_t bound_s;
  __shared__ int count, item_count;
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Row<T> x(static_cast<const T *>(a.logits) + (row / a.beams) * a.batch_stride + (row % a.beams) * a.beam_stride,
                 a.vocab);
  const int pieces = (a.vocab + x.skew + NV - 1) / NV;
  const int lo = min(pieces, chunk * a.chunk), hi = min(pieces, lo + a.chunk);
  if (tid == 0) count = item_count = 0;
  Sum sum;
  // the thread's largest logit, the first piece of the step that holds it, and the largest
  // of its other steps
  float top = -INFINITY, next = -INFINITY;
  int top_at = -1;
  auto seen = [&](float t, int at) {
    next = fmaxf(next, fminf(top, t));
    if (t > top) top = t, top_at = at;
  };
  auto careful = [&](int j) {
    float v[NV];
    x.values(j, v);
    sum.add_any(v);
  };
  // whole pieces are [w0, w1); the row's first and last may be partial
  const int w0 = lo + (lo < hi && !x.whole(lo) ? 1 : 0), w1 = max(w0, hi - (lo < hi && !x.whole(hi - 1) ? 1 : 0));
  // Thread tid has the pieces lo + tid + i kS, here and below.  They come through a ring
  // of its own (asynchronous copies, no barrier), a step ahead of the arithmetic.
  const int j0 = lo + tid < w0 ? lo + tid + kS : lo + tid;
  const int steps = j0 < w1 ? (w1 - j0 + U * kS - 1) / (U * kS) : 0;
  auto fetch = [&](int i) {
    if (i < steps) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = j0 + (i * U + u) * kS;
        if (at < w1) copy16(&sm.ring[i % kRing][u][tid], x.p + x.first(at));
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kRing - 1; ++i) fetch(i);
  for (int i = 0; i < steps; ++i) {
    fetch(i + kRing - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
    const int at = j0 + i * U * kS;
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = sm.ring[i % kRing][u][tid];
    if (at + (U - 1) * kS >= w1) {
#pragma unroll
      for (int u = 1; u < U; ++u)
        if (at + u * kS >= w1) w[u] = Vec<T>::none();
    }
    const float t = fmaxf(Vec<T>::top(w), -INFINITY);
    seen(t, at);
    if (!sum.template add<T>(w, t))
      for (int u = 0; u < U && at + u * kS < w1; ++u) careful(at + u * kS);
  }
  // the partial ones belong to the threads whose turn they would be
  auto partial = [&](int at) {
    if ((at - lo) % kS != tid) return;
    float v[NV];
    x.values(at, v);
    float t = v[0];
#pragma unroll
    for (int i = 1; i < NV; ++i) t = fmaxf(t, v[i]);
    seen(t, at);
    sum.add_any(v);
  };
  if (w0 > lo) partial(lo);
  if (w1 < hi && hi - 1 >= w0) partial(hi - 1);

  const bool any = lo + tid < hi;
  const uint32_t key = any ? key_of(top) : 0u;
  tops[tid] = key;
#pragma unroll
  for (int d = 16; d; d >>= 1)
    join(sum.b, sum.l, __shfl_xor_sync(0xffffffffu, sum.b, d), __shfl_xor_sync(0xffffffffu, sum.l, d));
  if (lane == 0) part[warp] = make_float2(sum.b, sum.l);
  __syncthreads();
  if (warp == 0) {
    // a bound that at least n thread maxima, and so n logits, reach: the upper half of the
    // n-th largest key, bit by bit, by one warp (every thread counting the maxima ahead of
    // its own took 3 us more at 1024 CTAs: the others' instructions wait)
    uint32_t k[W];
#pragma unroll
    for (int i = 0; i < W; ++i) k[i] = tops[i * 32 + lane] >> 16;
    uint32_t bound = 0;
#pragma unroll 1
    for (int bit = 15; bit >= 0; --bit) {
      const uint32_t t = bound | (1u << bit);
      int c = 0;
#pragma unroll
      for (int i = 0; i < W; ++i) c += k[i] >= t ? 1 : 0;
      if (__reduce_add_sync(0xffffffffu, c) >= a.n) bound = t;
    }
    if (lane == 0) bound_s = bound << 16;
  } else if (tid == 32) {
    float b = part[0].x, l = part[0].y;
    for (int w = 1; w < W; ++w) join(b, l, part[w].x, part[w].y);
    a.stats[static_cast<int64_t>(row) * a.chunks + chunk] = make_float2(b, l);
  }
  __syncthreads();
  const uint32_t bound = bound_s;
  const float least = bound <= key_of(-INFINITY) ? -INFINITY : value_of(bound);  // the bound as a value
  auto look = [&](int at) {  // a piece's logits that reach the bound
    float v[NV];
    x.values(at, v);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (v[i] >= least && x.in(x.first(at) + i)) {
        const int c = atomicAdd(&count, 1);
        if (c < kCap) cand[c] = make_uint2(key_of(v[i]), x.first(at) + i);
      }
    }
  };
  // the threads that reach it: usually only the step with the thread's largest logit, else
  // all its pieces, go to a list that all threads then share
  for (uint32_t who = __ballot_sync(0xffffffffu, any && key >= bound); who; who &= who - 1) {
    const int src = __ffs(who) - 1;
    const bool one = __shfl_sync(0xffffffffu, next < least && top_at >= 0, src);
    const int first = lo + (tid - lane) + src, step = __shfl_sync(0xffffffffu, top_at, src);
    const int start = one ? step : first, stop = one ? min(hi, step + U * kS) : hi;
    const int need = (stop - start + kS - 1) / kS;
    int at = 0;
    if (lane == 0) at = atomicAdd(&item_count, need);
    at = __shfl_sync(0xffffffffu, at, 0);
    for (int i = lane; i < need; i += 32) {
      if (at + i < kItems) items[at + i] = start + i * kS;
      else look(start + i * kS);
    }
  }
  __syncthreads();
  for (int i = tid; i < min(item_count, kItems); i += kS)
    if (items[i] >= 0) look(items[i]);
  __syncthreads();
  uint2 *out = a.cand + (static_cast<int64_t>(row) * a.chunks + chunk) * a.n;
  const int have = count;
  if (have <= kCap) {
    for (int i = tid; i < have; i += kS) {
      const uint2 c = cand[i];
      int r = 0;
      for (int k = 0; k < have && r < a.n; ++k) r += before(cand[k].x, cand[k].y, c.x, c.y) ? 1 : 0;
      if (r < a.n) out[r] = c;
    }
    for (int i = have + tid; i < a.n; i += kS) out[i] = make_uint2(0u, 0u);  // a chunk of fewer than n logits
  } else {
    // More equal or huge logits than fit (a vocabulary masked to one value, say):
    // n rounds, each the best one after the last pick.
    uint2 last = make_uint2(0xffffffffu, 0u);
    for (int r = 0; r < a.n; ++r) {
      uint2 b = make_uint2(0u, 0x7fffffffu);
      for (int at = lo + tid; at < hi; at += kS) {
        float v[NV];
        x.values(at, v);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int e = x.first(at) + i;
          const uint32_t k = key_of(v[i]);
          if (x.in(e) && before(last.x, last.y, k, e) && before(k, e, b.x, b.y)) b = make_uint2(k, e);
        }
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) {
        const uint32_t k = __shfl_xor_sync(0xffffffffu, b.x, d);
        const int e = __shfl_xor_sync(0xffffffffu, b.y, d);
        if (before(k, e, b.x, b.y)) b = make_uint2(k, e);
      }
      if (lane == 0) best[warp] = b;
      __syncthreads();
      for (int w = 0; w < kS / 32; ++w)
        if (before(best[w].x, best[w].y, b.x, b.y)) b = best[w];
      if (tid == 0) out[r] = b;
      last = b;
      __syncthreads();
    }
  }
}

struct MergeArgs {
  int beams, n, chunks, pad;
  const float2 *stats;
  const uint2 *cand;
  const float *scores;
  const uint8_t *finished;
  float *scores_out;
  int *parents_out, *tokens_out;
};

// Entries of a list of n falling keys that come before key k: those >= k where the
// list goes first among equals (x >= k is x > k - 1: no key of an entry is 0), those > k
// where it goes later.  Short lists are counted through (their loads do not wait for one
// another), longer ones halved.
__device__ __forceinline__ int entries_before(const uint32_t *list, int stride, int n, uint32_t k, bool first) {
  const uint32_t above = first ? k - 1u : k;
  int lo = 0;
  if (n <= 16) {
#pragma unroll 4
    for (int i = 0; i < n; ++i) lo += list[i * stride] > above ? 1 : 0;
    return lo;
  }
  int hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (list[mid * stride] > above) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

__host__ __device__ constexpr int round4(int v) { return (v + 3) / 4 * 4; }

// A beam as the merge needs it.
struct Beam {
  double log_sum;  // log of the row's sum of e^(x - b / c) (see ScanArgs::stats)
  float b;
  float score;     // so far
  int ended;
};

__device__ __forceinline__ void copy8(void *dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__global__ void __launch_bounds__(kT) beam_merge_kernel(MergeArgs a) {
  extern __shared__ uint32_t sm[];
  uint2 *in = reinterpret_cast<uint2 *>(sm);                // chunks' lists of some beams
  uint16_t *left = reinterpret_cast<uint16_t *>(sm + 2 * kLists);  // entries of each beam that matter
  uint32_t *key = sm + 2 * kLists + kLists / 2;             // [beams][n]: score keys, falling
  int *tok = reinterpret_cast<int *>(key + a.beams * a.n);  // [beams][n]
  int *place = tok + a.beams * a.n;                         // [beams][n]: places in the joint list
  Beam *beams = reinterpret_cast<Beam *>(key + round4(3 * a.beams * a.n));
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
  const int per = a.chunks * a.n, group = min(a.beams, kLists / per);  // beams at a time
  const uint2 *lists = a.cand + static_cast<int64_t>(b) * a.beams * per;
  for (int i = tid; i < group * per; i += kT) copy8(&in[i], &lists[i]);
  for (int k = tid >> 5; k < a.beams; k += kT / 32) {
    const int64_t row = static_cast<int64_t>(b) * a.beams + k;
    const float score = a.scores[row];
    const int ended = a.finished ? a.finished[row] : 0;
    float sb = -INFINITY, sl = 0.f;
    for (int c = lane; c < a.chunks; c += 32) {
      const float2 s = a.stats[row * a.chunks + c];
      join(sb, sl, s.x, s.y);
    }
    for (int d = 1; d < a.chunks && d < 32; d <<= 1)
      join(sb, sl, __shfl_xor_sync(0xffffffffu, sb, d), __shfl_xor_sync(0xffffffffu, sl, d));
    if (lane == 0) beams[k] = Beam{log(static_cast<double>(sl)), sb, score, ended};
  }
  for (int k0 = 0; k0 < a.beams; k0 += group) {
    const int kn = min(group, a.beams - k0);
    if (k0)
      for (int i = tid; i < kn * per; i += kT) copy8(&in[i], &lists[static_cast<int64_t>(k0) * per + i]);
    copies_done();
    __syncthreads();
    // a warp for each beam: the upper half of its n-th largest key, bit by bit; the entries
    // that reach it; their places by counting those ahead
    for (int k = tid >> 5; k < kn; k += kT / 32) {
      const uint2 *mine = in + k * per;
      uint16_t *some = left + k * per;
      uint32_t bound = 0;
#pragma unroll 1
      for (int bit = 15; bit >= 0 && per > 48; --bit) {  // fewer are counted through as they are
        const uint32_t t = bound | (1u << bit);
        int c = 0;
#pragma unroll 4
        for (int i = lane; i < per; i += 32) c += (mine[i].x >> 16) >= t ? 1 : 0;
        if (__reduce_add_sync(0xffffffffu, c) >= a.n) bound = t;
      }
      bound <<= 16;
      int count = 0;
      for (int i0 = 0; i0 < per; i0 += 32) {
        const int i = i0 + lane;
        const uint32_t key_i = i < per ? mine[i].x : 0u;
        const uint32_t who = __ballot_sync(0xffffffffu, key_i != 0u && key_i >= bound);
        if ((who >> lane) & 1) some[count + __popc(who & ((1u << lane) - 1u))] = static_cast<uint16_t>(i);
        count += __popc(who);
      }
      __syncwarp();
      for (int s = lane; s < count; s += 32) {
        const uint2 x = mine[some[s]];
        int r = 0;
        for (int o = 0; o < count && r < a.n; ++o) {
          const uint2 y = mine[some[o]];
          r += before(y.x, static_cast<int>(y.y), x.x, static_cast<int>(x.y)) ? 1 : 0;
        }
        if (r >= a.n) continue;
        key[(k0 + k) * a.n + r] = x.x;
        tok[(k0 + k) * a.n + r] = static_cast<int>(x.y);
      }
    }
    __syncthreads();
  }
  // logits to scores: s + ((x - top) - log(sum of e^(x - top))), the last log from the
  // stored sum in 64 bits (once per beam and thread), rounded once
  for (int k = tid >> 5; k < a.beams; k += kT / 32) {
    const Beam x = beams[k];
    const float top = value_of(key[k * a.n]);
    const double shift = top == INFINITY ? 0.0 : static_cast<double>(x.b) - static_cast<double>(top) * kLog2e;
    const float log_sum = static_cast<float>(shift * 0.6931471805599453 + x.log_sum);
    __syncwarp();
    for (int j = lane; j < a.n; j += 32) {
      const float v = value_of(key[k * a.n + j]);
      float s = x.score;
      if (x.ended) {
        if (j > 0) s = -INFINITY;
        tok[k * a.n + j] = a.pad;
      } else {
        s += top == -INFINITY ? -INFINITY : (v == top ? 0.f : v - top) - log_sum;
      }
      key[k * a.n + j] = key_of(fmaxf(s, -INFINITY));
      place[k * a.n + j] = j;
    }
  }
  __syncthreads();
  // places in the joint list: a thread per candidate and other beam
  const int total = a.beams * a.n;
  for (int i = tid; i < total * a.beams; i += kT) {
    const int c = i / a.beams, o = i - c * a.beams, beam = c / a.n;
    if (o == beam) continue;
    const int r = entries_before(key + o * a.n, 1, a.n, key[c], o < beam);
    if (r) atomicAdd(&place[c], r);
  }
  __syncthreads();
  for (int i = tid; i < total; i += kT) {
    const int beam = i / a.n, r = place[i];
    if (r >= a.n) continue;
    const int64_t at = static_cast<int64_t>(b) * a.n + r;
    a.scores_out[at] = value_of(key[i]);
    a.parents_out[at] = beam;
    a.tokens_out[at] = tok[i];
  }
}

// Chunks of a row: as many CTAs as the GPU holds at once (kScanCtas per SM),
// none below kMinChunk logits, where a CTA's fixed cost outweighs its loads.
int chunks_of(int64_t rows, int64_t vocab, int64_t n) {
  int64_t c = (148 * kScanCtas) / (rows > 0 ? rows : 1);
  if (c > vocab / kMinChunk) c = vocab / kMinChunk;
  if (c > kLists / n) c = kLists / n;
  return static_cast<int>(c < 1 ? 1 : c);
}

template <typename T>
int run_scan(ScanArgs a, int64_t rows, cudaStream_t s) {
  const int pieces = static_cast<int>(ceil_div(a.vocab, Vec<T>::n)) + 1;  // a skewed row has one more
  a.chunk = static_cast<int>(ceil_div(pieces, a.chunks));
  return launch_pdl("beam scan", beam_scan_kernel<T>, dim3(a.chunks, static_cast<unsigned>(rows)), dim3(kS), 0, s, a);
}

}  // namespace

int64_t beam_workspace_bytes(int64_t batch, int64_t beams, int64_t vocab, int64_t n) {
  const int64_t rows = batch * beams, c = chunks_of(rows, vocab, n);
  return round_up(rows * c * 8, 256) + rows * c * n * 8;
}

int launch_beam_select(const void *logits, int dtype, int64_t batch_stride, int64_t beam_stride, int64_t batch,
                       int64_t beams, int64_t vocab, const float *scores, const uint8_t *finished, int n, int pad,
                       float *scores_out, int *parents_out, int *tokens_out, void *ws, cudaStream_t s) {
  const int64_t rows = batch * beams;
  const int chunks = chunks_of(rows, vocab, n);
  float2 *stats = static_cast<float2 *>(ws);
  uint2 *cand = reinterpret_cast<uint2 *>(static_cast<char *>(ws) + round_up(rows * chunks * 8, 256));
  const ScanArgs a{logits, batch_stride, beam_stride, static_cast<int>(beams), static_cast<int>(vocab), n, chunks, 0,
                   stats, cand};
  const int st = dtype == QS_F32 ? run_scan<float>(a, rows, s)
                 : dtype == QS_F16 ? run_scan<__half>(a, rows, s) : run_scan<__nv_bfloat16>(a, rows, s);
  if (st) return st;
  const MergeArgs m{static_cast<int>(beams), n, chunks, pad, stats, cand, scores, finished, scores_out, parents_out,
                    tokens_out};
  const size_t smem = static_cast<size_t>(kLists) * 10 + round4(static_cast<int>(3 * beams * n)) * 4 + beams * sizeof(Beam);
  static const cudaError_t attr = cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                       kLists * 10 + kBeamMaxBeams * kBeamMaxN * 12 + kBeamMaxBeams * (int)sizeof(Beam));
  if (attr != cudaSuccess) return fail(QS_ERR_CUDA, "beam merge: %s", cudaGetErrorString(attr));
  return launch_pdl("beam merge", beam_merge_kernel, dim3(static_cast<unsigned>(batch)), dim3(kT), smem, s, m);
}

}  // namespace qs
