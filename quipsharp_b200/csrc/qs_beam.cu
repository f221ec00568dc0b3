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
// joins the chunks' sorted lists into the beams', and the beams' into the result;
// a candidate's place in the merged list is the sum of its places in each list
// (binary searches), so nothing is sorted and nothing depends on arrival order.
//
// Bound: the logits' bytes, once.
#include <cmath>

#include "qs_common.cuh"
#include "qs_launch.h"

namespace qs {
namespace {

constexpr int kT = 256;        // threads of both kernels
constexpr int kCap = 1024;     // candidates of a chunk kept in shared memory
constexpr int kMinChunk = 2048;
constexpr int kLists = 4096;   // candidates merged at a time
constexpr float kLog2e = 1.4426950408889634f;

template <typename T> struct Vec;  // a 16-byte piece of a row
template <> struct Vec<float> {
  static constexpr int n = 4;
  __device__ static void unpack(const uint4 &w, float (&v)[4]) {
    v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
  }
  __device__ static float one(const float *p) { return *p; }
};
template <> struct Vec<__half> {
  static constexpr int n = 8;
  __device__ static void unpack(const uint4 &w, float (&v)[8]) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&a[i]));
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
  __device__ static float one(const __half *p) { return __half2float(*p); }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int n = 8;
  __device__ static void unpack(const uint4 &w, float (&v)[8]) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(a[i] << 16);
      v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
    }
  }
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

struct ScanArgs {
  const void *logits;
  int64_t batch_stride, beam_stride;
  int beams, vocab, n, chunks, chunk;  // chunk: 16-byte pieces per CTA
  float2 *stats;                       // [row][chunk]: maximum, sum of exp(x - maximum)
  uint2 *cand;                         // [row][chunk][n]: key, token
};

// Pieces of a row: piece j holds elements [j * n - skew, ...), so that whole pieces
// are aligned; the first and last may be partial and are read element by element.
template <typename T>
struct Row {
  const T *p;
  int vocab, skew;
  __device__ Row(const T *base, int v) : p(base), vocab(v) {
    skew = static_cast<int>((reinterpret_cast<uintptr_t>(base) & 15) / sizeof(T));
  }
  __device__ int first(int j) const { return j * Vec<T>::n - skew; }
  // NaN becomes -inf; places outside the row become -inf and `in` false there
  __device__ void load(int j, float (&v)[Vec<T>::n]) const {
    const int e = first(j);
    if (e >= 0 && e + Vec<T>::n <= vocab) {
      Vec<T>::unpack(*reinterpret_cast<const uint4 *>(p + e), v);
    } else {
#pragma unroll
      for (int i = 0; i < Vec<T>::n; ++i) v[i] = in(e + i) ? Vec<T>::one(p + e + i) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < Vec<T>::n; ++i) v[i] = fmaxf(v[i], -INFINITY);
  }
  __device__ bool in(int e) const { return e >= 0 && e < vocab; }
};

// Adds a piece to a running maximum m and sum l of exp(x - m).
template <int NV>
__device__ __forceinline__ void accumulate(const float (&v)[NV], float &m, float &l) {
  float top = v[0];
#pragma unroll
  for (int i = 1; i < NV; ++i) top = fmaxf(top, v[i]);
  const float mn = fmaxf(m, top);
  if (mn == INFINITY) {  // only the +inf logits count
    float c = m == INFINITY ? l : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) c += v[i] == INFINITY ? 1.f : 0.f;
    l = c;
  } else if (mn != -INFINITY) {
    // subtract, then scale: the difference is (nearly) exact, where mn * log2(e) rounded
    // once would shift every term of the sum by |mn| 2^-24
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) s += ex2((v[i] - mn) * kLog2e);
    l = fmaf(l, ex2((m - mn) * kLog2e), s);
  }
  m = mn;
}

// Joins (m2, l2) into (m, l).
__device__ __forceinline__ void join(float &m, float &l, float m2, float l2) {
  const float mn = fmaxf(m, m2);
  const float a = m == mn ? 1.f : expf(m - mn), b = m2 == mn ? 1.f : expf(m2 - mn);
  l = l * a + l2 * b;
  m = mn;
}

__device__ __forceinline__ bool before(uint32_t k1, int t1, uint32_t k2, int t2) {
  return k1 > k2 || (k1 == k2 && t1 < t2);
}

template <typename T>
__global__ void __launch_bounds__(kT) beam_scan_kernel(ScanArgs a) {
  constexpr int NV = Vec<T>::n, U = 4;
  __shared__ uint32_t tops[kT];
  __shared__ uint2 cand[kCap];
  __shared__ float2 part[kT / 32];
  __shared__ uint2 best[kT / 32];
  __shared__ uint32_t bound_s;
  __shared__ int count;
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Row<T> x(static_cast<const T *>(a.logits) + (row / a.beams) * a.batch_stride + (row % a.beams) * a.beam_stride,
                 a.vocab);
  const int pieces = (a.vocab + x.skew + NV - 1) / NV;
  const int lo = min(pieces, chunk * a.chunk), hi = min(pieces, lo + a.chunk);
  if (tid == 0) count = 0, bound_s = 0;
  float m = -INFINITY, l = 0.f;
  bool any = false;
  for (int j0 = lo + tid; j0 < hi; j0 += kT * U) {
    float v[U][NV];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j0 + u * kT < hi) x.load(j0 + u * kT, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j0 + u * kT < hi) accumulate(v[u], m, l);
    any = true;
  }
  const uint32_t top = any ? key_of(m) : 0u;
  tops[tid] = top;
#pragma unroll
  for (int d = 16; d; d >>= 1)
    join(m, l, __shfl_xor_sync(0xffffffffu, m, d), __shfl_xor_sync(0xffffffffu, l, d));
  if (lane == 0) part[warp] = make_float2(m, l);
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kT / 32; ++w) join(m, l, part[w].x, part[w].y);
    a.stats[static_cast<int64_t>(row) * a.chunks + chunk] = make_float2(m, l);
  }
  // the n-th largest thread maximum (ties: the lower thread first)
  int ahead = 0;
  for (int t = 0; t < kT; ++t) ahead += before(tops[t], t, top, tid) ? 1 : 0;
  if (ahead == a.n - 1) bound_s = top;
  __syncthreads();
  const uint32_t bound = bound_s;
  if (any && top >= bound) {
    for (int j = lo + tid; j < hi; j += kT) {
      float v[NV];
      x.load(j, v);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = x.first(j) + i;
        const uint32_t k = key_of(v[i]);
        if (x.in(e) && k >= bound) {
          const int at = atomicAdd(&count, 1);
          if (at < kCap) cand[at] = make_uint2(k, e);
        }
      }
    }
  }
  __syncthreads();
  uint2 *out = a.cand + (static_cast<int64_t>(row) * a.chunks + chunk) * a.n;
  const int have = count;
  if (have <= kCap) {
    for (int i = tid; i < have; i += kT) {
      const uint2 c = cand[i];
      int r = 0;
      for (int k = 0; k < have && r < a.n; ++k) r += before(cand[k].x, cand[k].y, c.x, c.y) ? 1 : 0;
      if (r < a.n) out[r] = c;
    }
    for (int i = have + tid; i < a.n; i += kT) out[i] = make_uint2(0u, 0u);  // a chunk of fewer than n logits
  } else {
    // More equal or huge logits than fit (a vocabulary masked to one value, say):
    // n rounds, each the best one after the last pick.
    uint2 last = make_uint2(0xffffffffu, 0u);
    for (int r = 0; r < a.n; ++r) {
      uint2 b = make_uint2(0u, 0x7fffffffu);
      for (int j = lo + tid; j < hi; j += kT) {
        float v[NV];
        x.load(j, v);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int e = x.first(j) + i;
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
      for (int w = 0; w < kT / 32; ++w)
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
// list goes first among equals, those > k where it goes later.
__device__ __forceinline__ int entries_before(const uint32_t *list, int stride, int n, uint32_t k, bool first) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    const uint32_t x = list[mid * stride];
    if (first ? x >= k : x > k) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kT) beam_merge_kernel(MergeArgs a) {
  extern __shared__ uint32_t sm[];
  uint2 *in = reinterpret_cast<uint2 *>(sm);                        // chunks' lists of some beams
  uint32_t *key = sm + 2 * kLists;                                  // [beams][n]: score keys, falling
  int *tok = reinterpret_cast<int *>(key + a.beams * a.n);          // [beams][n]
  float2 *st = reinterpret_cast<float2 *>(tok + a.beams * a.n);
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.x, tid = threadIdx.x;
  const int per = a.chunks * a.n, group = min(a.beams, kLists / per);  // beams at a time
  for (int k = tid; k < a.beams; k += kT) {
    const float2 *s = a.stats + (static_cast<int64_t>(b) * a.beams + k) * a.chunks;
    float m = -INFINITY, l = 0.f;
    for (int c = 0; c < a.chunks; ++c) join(m, l, s[c].x, s[c].y);
    st[k] = make_float2(m, logf(l));
  }
  for (int k0 = 0; k0 < a.beams; k0 += group) {
    const int kn = min(group, a.beams - k0);
    __syncthreads();
    const uint2 *src = a.cand + (static_cast<int64_t>(b) * a.beams + k0) * per;
    for (int i = tid; i < kn * per; i += kT) in[i] = src[i];
    __syncthreads();
    for (int i = tid; i < kn * per; i += kT) {
      const int k = i / per, c = (i % per) / a.n, j = i % a.n;
      const uint2 x = in[i];
      int r = j;
      for (int o = 0; o < a.chunks && r < a.n; ++o)
        if (o != c) r += entries_before(&in[k * per + o * a.n].x, 2, a.n, x.x, o < c);
      if (x.x == 0u || r >= a.n) continue;
      const int beam = k0 + k;
      const float s0 = a.scores[static_cast<int64_t>(b) * a.beams + beam];
      float s = s0;
      int token = static_cast<int>(x.y);
      if (a.finished && a.finished[static_cast<int64_t>(b) * a.beams + beam]) {
        if (r > 0) s = -INFINITY;
        token = a.pad;
      } else {
        const float v = value_of(x.x), m = st[beam].x;
        s += m == -INFINITY ? -INFINITY : (v == m ? 0.f : v - m) - st[beam].y;
      }
      key[beam * a.n + r] = key_of(fmaxf(s, -INFINITY));
      tok[beam * a.n + r] = token;
    }
  }
  __syncthreads();
  for (int i = tid; i < a.beams * a.n; i += kT) {
    const int beam = i / a.n, j = i % a.n;
    const uint32_t k = key[i];
    int r = j;
    for (int o = 0; o < a.beams && r < a.n; ++o)
      if (o != beam) r += entries_before(key + o * a.n, 1, a.n, k, o < beam);
    if (r >= a.n) continue;
    const int64_t at = static_cast<int64_t>(b) * a.n + r;
    a.scores_out[at] = value_of(k);
    a.parents_out[at] = beam;
    a.tokens_out[at] = tok[i];
  }
}

// Chunks of a row: enough CTAs to fill the GPU once (eight of 256 threads per SM),
// none below kMinChunk logits, where a CTA's fixed cost outweighs its loads.
int chunks_of(int64_t rows, int64_t vocab, int64_t n) {
  int64_t c = (148 * 8) / (rows > 0 ? rows : 1);
  if (c > vocab / kMinChunk) c = vocab / kMinChunk;
  if (c > kLists / n) c = kLists / n;
  return static_cast<int>(c < 1 ? 1 : c);
}

template <typename T>
int run_scan(ScanArgs a, int64_t rows, cudaStream_t s) {
  const int pieces = static_cast<int>(ceil_div(a.vocab, Vec<T>::n)) + 1;  // a skewed row has one more
  a.chunk = static_cast<int>(ceil_div(pieces, a.chunks));
  return launch_pdl("beam scan", beam_scan_kernel<T>, dim3(a.chunks, static_cast<unsigned>(rows)), dim3(kT), 0, s, a);
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
  const size_t smem = static_cast<size_t>(kLists) * 8 + static_cast<size_t>(beams) * n * 8 + beams * 8;
  static const cudaError_t attr = cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                       kLists * 8 + kBeamMaxBeams * kBeamMaxN * 8 + kBeamMaxBeams * 8);
  if (attr != cudaSuccess) return fail(QS_ERR_CUDA, "beam merge: %s", cudaGetErrorString(attr));
  return launch_pdl("beam merge", beam_merge_kernel, dim3(static_cast<unsigned>(batch)), dim3(kT), smem, s, m);
}

}  // namespace qs
