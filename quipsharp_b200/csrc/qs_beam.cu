// Beam search's selection: the best n of beams x vocabulary continuations by
//   score[b] + (x - m) - log(sum exp(x - m)),   m = max x.
//
// One pass over the logits.  A beam's scores fall with its logits, so its n best
// continuations are its n largest logits, and the log-sum, which is not known until
// the row ends, is not needed to find them.  beam_scan: each CTA takes a chunk of
// one row; its threads keep a running maximum and sum of exponentials, and their
// largest logit.  A bound on the n-th largest of those thread maxima is one that at least
// n logits of the chunk reach and few others do, so only the few threads whose
// maximum reaches it look at their logits again.  beam_merge: one CTA per search
// joins the chunks' lists into the beams', and the beams' into the result; a candidate's
// place is the number of those ahead of it, so nothing is sorted and nothing depends on
// the order of arrival.
//
// Bound: the logits' bytes, once, for many rows; dependent steps for few.  Measured: 32
// searches of 8 beams over 128000 bfloat16 logits, n = 16: 28 us (2.3 TB/s; 8 of them after
// the stream's end); 4 beams over 32000 float32 logits, n = 4: 8.5 us (7.9 on the GPU).
#include <algorithm>
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
constexpr int kQuick = 16;     // n up to which the scan's bound comes from 32 maxima
constexpr int kMinChunk = 2048;
constexpr int kScanCtas = 8;   // scanning CTAs per SM
constexpr int kLists = 4096;   // candidates merged at a time
constexpr int kDirect = 32;    // candidates of a beam that are counted through as they are
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
  float2 *stats;                       // [row][chunk]: a logit r near the largest, sum of e^(x - r)
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

// A thread's sum.  Beside an ordinary reference (the largest logit, or kLag below it, which
// float32 sums hold) it is of 2^(x c - b) with c = log2(e) and b = ref c, both in float32:
// x c - b is rounded once, so no term is off by more than its own distance to b.  What b was
// rounded by grows with it, though, and past some 2^31 would take 2^(x c - b) out of float32's
// range (a vocabulary masked with the type's lowest number, in float32 or bfloat16), so beside
// a larger reference the sum is of 2^((x - ref) c).
constexpr float kLag = 8.f;
constexpr float kOrdinary = 0x1p20f;  // b is off by 2^-4 at most
struct Sum {
  float ref = -INFINITY, b = -INFINITY, l = 0.f;  // b = ref * c
  float limit = -INFINITY;                        // ordinary numbers up to here need no other reference

  __device__ __forceinline__ bool ordinary() const { return fabsf(ref) < kOrdinary; }
  __device__ __forceinline__ void renew(float top) {  // both references ordinary, or the old one -inf
    const float nb = top * kLog2e;
    l *= b == nb ? 1.f : ex2(b - nb);
    ref = top;
    b = nb;
    limit = ref + kLag;
  }
  // What b was rounded by: the sum is of e^(x - ref) times 2^this.
  __device__ __forceinline__ float off() const { return ordinary() ? fmaf(ref, kLog2e, -b) : 0.f; }
  __device__ __forceinline__ float natural() const { return l * ex2(-off()); }
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
      float s = natural();
      if (top > ref) s *= ex2((ref - top) * kLog2e), ref = top, b = top * kLog2e;
      if (ref != -INFINITY)
#pragma unroll
        for (int i = 0; i < NV; ++i) s += ex2((v[i] - ref) * kLog2e);
      l = s * ex2(off());
    }
    limit = ordinary() ? ref + kLag : -INFINITY;
  }
  // Pieces of ordinary numbers with maximum `top`; false (and nothing added) where there
  // are others, or were until now.  Per number: half a multiply-add and half an addition (two at a time)
  // and the exponential.
  template <typename T, int U>
  __device__ __forceinline__ bool add(const uint4 (&w)[U], float top) {
    if (!(top <= limit)) {
      if (!(fabsf(top) < kOrdinary) || !(ordinary() || ref == -INFINITY)) return false;
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

// Joins a sum l2 of e^(x - r2) into l, of e^(x - r).
__device__ __forceinline__ void join(float &r, float &l, float r2, float l2) {
  const float m = fmaxf(r, r2);
  l = l * (r == m ? 1.f : ex2((r - m) * kLog2e)) + l2 * (r2 == m ? 1.f : ex2((r2 - m) * kLog2e));
  r = m;
}

__device__ __forceinline__ bool before(uint32_t k1, int t1, uint32_t k2, int t2) {
  return k1 > k2 || (k1 == k2 && t1 < t2);
}

// How many of a list's entries come before x; at least n where they are no fewer (the list
// is then left early, eight entries at a time, so that their loads do not wait).
__device__ __forceinline__ int place_of(const uint2 *list, int count, uint2 x, int n) {
  int r = 0, k = 0;
  for (; k + 8 <= count && r < n; k += 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint2 y = list[k + i];
      r += before(y.x, static_cast<int>(y.y), x.x, static_cast<int>(x.y)) ? 1 : 0;
    }
  }
  for (; k < count && r < n; ++k)
    r += before(list[k].x, static_cast<int>(list[k].y), x.x, static_cast<int>(x.y)) ? 1 : 0;
  return r;
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
  float r = sum.ref, l = sum.natural();
#pragma unroll
  for (int d = 16; d; d >>= 1) join(r, l, __shfl_xor_sync(0xffffffffu, r, d), __shfl_xor_sync(0xffffffffu, l, d));
  if (lane == 0) part[warp] = make_float2(r, l);
  __syncthreads();
  if (warp == 0) {
    // A bound that at least n thread maxima, and so n logits, reach, by one warp (every
    // thread counting the maxima ahead of its own took 3 us more at 1024 CTAs: the others'
    // instructions wait).  For small n the n-th largest of 32 maxima of four threads each:
    // about n + n^2 / 64 threads reach it, and it takes 200 cycles for the 2000 of the other.
    // That one is the upper half of the n-th largest key, bit by bit.
    uint32_t k[W], bound = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) k[i] = tops[i * 32 + lane];
    if (a.n <= kQuick) {
      uint32_t top4 = k[0];
#pragma unroll
      for (int i = 1; i < W; ++i) top4 = max(top4, k[i]);
      int r = 0;
#pragma unroll
      for (int o = 0; o < 32; ++o) {
        const uint32_t y = __shfl_sync(0xffffffffu, top4, o);
        r += y > top4 || (y == top4 && o < lane) ? 1 : 0;
      }
      bound = __shfl_sync(0xffffffffu, top4, __ffs(__ballot_sync(0xffffffffu, r == a.n - 1)) - 1);
    } else {
#pragma unroll 1
      for (int bit = 31; bit >= 16; --bit) {
        const uint32_t t = bound | (1u << bit);
        int c = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) c += k[i] >= t ? 1 : 0;
        if (__reduce_add_sync(0xffffffffu, c) >= a.n) bound = t;
      }
    }
    if (lane == 0) bound_s = bound;
  } else if (tid == 32) {
    r = part[0].x, l = part[0].y;
    for (int w = 1; w < W; ++w) join(r, l, part[w].x, part[w].y);
    a.stats[static_cast<int64_t>(row) * a.chunks + chunk] = make_float2(r, l);
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
  if (any && key >= bound) {
    const bool one = next < least && top_at >= 0;
    const int start = one ? top_at : lo + tid, stop = one ? min(hi, top_at + U * kS) : hi;
    const int need = (stop - start + kS - 1) / kS, at = atomicAdd(&item_count, need);
    for (int i = 0; i < need; ++i) {
      if (at + i < kItems) items[at + i] = start + i * kS;
      else look(start + i * kS);
    }
  }
  __syncthreads();
  for (int i = tid; i < min(item_count, kItems); i += kS)
    look(items[i]);
  __syncthreads();
  uint2 *out = a.cand + (static_cast<int64_t>(row) * a.chunks + chunk) * a.n;
  const int have = count;
  if (have <= kCap) {
    for (int i = tid; i < have; i += kS) {
      const uint2 c = cand[i];
      const int r = place_of(cand, have, c, a.n);
      if (r < a.n) out[r] = c;
    }
    for (int i = have + tid; i < a.n; i += kS) out[i] = make_uint2(0u, 0u);  // a chunk of fewer than n logits
  } else {
    // More equal or huge logits than fit (a vocabulary masked to one value, say):
    // n rounds, each the best one after the last pick (32 x 8 x 128000 bfloat16 logits of
    // which all but 1000 are masked, n = 16: 680 us, for 28).
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
  int group, room;  // beams at a time; their entries, to a multiple of 4
  const float2 *stats;
  const uint2 *cand;
  const float *scores;
  const uint8_t *finished;
  float *scores_out;
  int *parents_out, *tokens_out;
};

__host__ __device__ constexpr int round4(int v) { return (v + 3) / 4 * 4; }

// A beam as the merge needs it.
struct Beam {
  double log_sum;  // log of the row's sum of e^(x - r) (see ScanArgs::stats)
  float r;
  float score;     // so far
  int ended;
};

__device__ __forceinline__ void copy8(void *dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__global__ void __launch_bounds__(kT) beam_merge_kernel(MergeArgs a) {
  extern __shared__ __align__(16) uint32_t sm[];
  uint2 *in = reinterpret_cast<uint2 *>(sm);                // chunks' lists of some beams
  uint2 *left = in + a.room;                                // entries of each beam that matter
  const int total = a.beams * a.n, total4 = round4(total);
  uint32_t *key = sm + (a.chunks * a.n <= kDirect ? 2 : 4) * a.room;  // [beams][n]: score keys; zeros to a multiple of 4
  int *tok = reinterpret_cast<int *>(key + total4);         // [beams][n]
  Beam *beams = reinterpret_cast<Beam *>(tok + total4);
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = a.chunks * a.n, group = a.group;
  const uint2 *lists = a.cand + static_cast<int64_t>(b) * a.beams * per;
  for (int i = total + tid; i < total4; i += kT) key[i] = 0u;
  // The beams' sums: by the warps that have no list while the others are at theirs, where
  // there are such, else afterwards.
  auto sums = [&] {
    for (int k = warp ^ (kT / 64); k < a.beams; k += kT / 32) {
      const int64_t row = static_cast<int64_t>(b) * a.beams + k;
      const float score = a.scores[row];
      const int ended = a.finished ? a.finished[row] : 0;
      float sr = -INFINITY, sl = 0.f;
      for (int c = lane; c < a.chunks; c += 32) {
        const float2 s = a.stats[row * a.chunks + c];
        join(sr, sl, s.x, s.y);
      }
      for (int d = 1; d < a.chunks && d < 32; d <<= 1)
        join(sr, sl, __shfl_xor_sync(0xffffffffu, sr, d), __shfl_xor_sync(0xffffffffu, sl, d));
      if (lane == 0) beams[k] = Beam{log(static_cast<double>(sl)), sr, score, ended};
    }
  };
  const bool apart = a.beams <= kT / 64 && group == a.beams;
  const int listing = apart ? kT / 2 : kT;
  auto listed = [&] { asm volatile("bar.sync 1, %0;" ::"r"(listing) : "memory"); };
  if (apart && warp >= kT / 64) sums();
  for (int k0 = 0; k0 < a.beams && tid < listing; k0 += group) {
    const int kn = min(group, a.beams - k0);
    for (int i = tid; i < kn * per; i += listing) copy8(&in[i], &lists[static_cast<int64_t>(k0) * per + i]);
    copies_done();
    listed();
    // A warp for each beam.  Its n best are no lower than a bound that n entries reach: the
    // n-th largest of the chunks' first ones where there are n chunks, else of their first m,
    // of which there are n and a half of n or more.  Each chunk's list falls, so a lane walks
    // it down to the bound; places come from counting those ahead.
    for (int k = warp; k < kn; k += listing / 32) {
      const uint2 *mine = in + k * per;
      uint2 *some = left + k * per;
      int count = per;
      if (per <= kDirect) {
        some = in + k * per;
      } else {
        uint32_t bound = 0;  // the same key may be there more than once
        if (a.chunks >= a.n) {
          for (int c = lane; c < a.chunks; c += 32) {
            const uint32_t x = mine[c * a.n].x;
            int r = 0;
#pragma unroll 8
            for (int d = 0; d < a.chunks; ++d) {
              const uint32_t y = mine[d * a.n].x;
              r += y > x || (y == x && d < c) ? 1 : 0;
            }
            if (r == a.n - 1) bound = x;
          }
        } else {
          const int m = min(a.n, (a.n + a.n / 2 + a.chunks - 1) / a.chunks);
          for (int i = lane; i < a.chunks * m; i += 32) {
            const uint32_t x = mine[i / m * a.n + i % m].x;
            int r = 0;
            for (int c = 0, d = 0; c < a.chunks; ++c)
#pragma unroll 2
              for (int j = 0; j < m; ++j, ++d) {
                const uint32_t y = mine[c * a.n + j].x;
                r += y > x || (y == x && d < i) ? 1 : 0;
              }
            if (r == a.n - 1) bound = x;
          }
        }
        bound = __reduce_max_sync(0xffffffffu, bound);
        bound = max(bound, 1u);  // 0 is no entry
        count = 0;
        for (int c0 = 0; c0 < a.chunks; c0 += 32) {
          const uint2 *list = mine + (c0 + lane) * a.n;
          int have = 0;
          if (c0 + lane < a.chunks)
            while (have < a.n && list[have].x >= bound) ++have;
          int before_me = have;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, before_me, d);
            if (lane >= d) before_me += y;
          }
          for (int i = 0; i < have; ++i) some[count + before_me - have + i] = list[i];
          count += __shfl_sync(0xffffffffu, before_me, 31);
        }
        __syncwarp();
      }
      for (int i = lane; i < count; i += 32) {
        const uint2 x = some[i];
        if (x.x == 0u) continue;
        const int r = place_of(some, count, x, a.n);
        if (r >= a.n) continue;
        key[(k0 + k) * a.n + r] = x.x;
        tok[(k0 + k) * a.n + r] = static_cast<int>(x.y);
      }
    }
    listed();
  }
  if (!apart) sums();
  __syncthreads();
  // logits to scores: s + ((x - top) - log(sum of e^(x - top))), the last log from the
  // stored sum in 64 bits (once per beam and thread), rounded once
  for (int k = tid >> 5; k < a.beams; k += kT / 32) {
    const Beam x = beams[k];
    const float top = value_of(key[k * a.n]);
    const double shift = x.r == top ? 0.0 : static_cast<double>(x.r) - static_cast<double>(top);
    const float log_sum = static_cast<float>(shift + x.log_sum);
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
    }
  }
  __syncthreads();
  // Places in the joint list: a candidate's is the number of those ahead, by score, then in
  // the order they stand (the beam, then its list).  A few neighbouring threads share one.
  int share = 1;
  while (share < 16 && share * 2 * total <= kT) share *= 2;
  const int part = tid & (share - 1);
  for (int c0 = 0; c0 < total; c0 += kT / share) {
    const int c = c0 + tid / share;
    const uint32_t x = c < total ? key[c] : 0xffffffffu;
    int r = 0;
#pragma unroll 4
    for (int d = part * 4; d < total4; d += share * 4) {
      const uint4 y = *reinterpret_cast<const uint4 *>(key + d);
      r += (y.x > x || (y.x == x && d < c) ? 1 : 0) + (y.y > x || (y.y == x && d + 1 < c) ? 1 : 0) +
           (y.z > x || (y.z == x && d + 2 < c) ? 1 : 0) + (y.w > x || (y.w == x && d + 3 < c) ? 1 : 0);
    }
    for (int d = 1; d < share; d <<= 1) r += __shfl_xor_sync(0xffffffffu, r, d);
    if (part == 0 && c < total && r < a.n) {
      const int64_t at = static_cast<int64_t>(b) * a.n + r;
      a.scores_out[at] = value_of(x);
      a.parents_out[at] = c / a.n;
      a.tokens_out[at] = tok[c];
    }
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
  int st = dtype == QS_F32 ? run_scan<float>(a, rows, s)
                 : dtype == QS_F16 ? run_scan<__half>(a, rows, s) : run_scan<__nv_bfloat16>(a, rows, s);
  if (st) return st;
  const int per = chunks * n, group = static_cast<int>(std::min<int64_t>(beams, kLists / per)), room = round4(group * per);
  const MergeArgs m{static_cast<int>(beams), n, chunks, pad, group, room, stats, cand, scores, finished, scores_out, parents_out,
                    tokens_out};
  // as much as this call needs: SMs that have to change their split of memory wait for the
  // kernel before (3 us)
  const size_t smem = static_cast<size_t>(room) * (per <= kDirect ? 8 : 16) + round4(static_cast<int>(beams * n)) * 8 + beams * sizeof(Beam);
  static std::atomic<uint64_t> allowed{0};
  st = allow_smem("beam merge", beam_merge_kernel,
                  kLists * 16 + kBeamMaxBeams * kBeamMaxN * 8 + kBeamMaxBeams * (int)sizeof(Beam), allowed);
  if (st) return st;
  return launch_pdl("beam merge", beam_merge_kernel, dim3(static_cast<unsigned>(batch)), dim3(kT), smem, s, m);
}

}  // namespace qs
