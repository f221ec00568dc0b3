// Causal attention of many new tokens per row over the paged cache, with a sliding
// window and first tokens that stay visible.
//
// A CTA takes NQ tiles of 128 query rows of one key head: the tokens of a tile times
// the query heads that share the key head (token-major), so a key tile read once
// serves the whole group, and a tile spans few tokens, which keeps what a window or
// the diagonal cuts off small.  Keys come in tiles of 128 as whole-page boxes through
// TMA.  Per key tile and query tile: S = Q K^T on the tensor core into TMEM; one
// thread per query row takes its row of S into registers, keeps the running maximum
// and sum of the softmax, and writes the weights back over S as 16-bit values; O +=
// P V on the tensor core with P read from TMEM.  With two query tiles the tensor core
// works on one while the other's softmax runs.
//
// The weights are 2^(s - reference), the reference kBias below a maximum of the scores so
// far.  Most tiles keep it: whether it still will do shows in the weights' sum, and only
// then is a maximum taken and O rescaled.  Float16 weights have to stay below 65504, and
// the bias keeps those down to 2^-20 of the largest in float16's normal range (a first
// token that takes nearly all the weight and has next to no value is common).
//
// One CTA per SM stays and takes one group of tiles after another: the grid has a block
// for each, and a running CTA cancels the next one that has not started and does its work
// (so the longest are begun first and none waits for a fixed share).  The loads of a
// group begin while the one before is still being summed.
//
// Where the tiles are fewer than the SMs (few tokens over many keys), each is split along
// the keys: a block takes a share of its key tiles and leaves its sum, maximum and output
// in float32, and window_join_kernel puts the shares together.
//
// Bound: the exponentials.  A key tile of one query tile takes 128 x 128 of them, 1024
// cycles of an SM's sixteen a cycle, next to 1024 of the two products (dim 128) and the
// rest of the softmax's issue.  Measured: a prompt of 8192 tokens, 64 query heads over 8
// of 128, bfloat16: 940 to 967 us (1.14 to 1.17 PFLOP/s, by the clocks that the power limit
// leaves); four chunks of 300 to 2000 tokens under a window of 1024: 88 us (0.67 PFLOP/s of
// visible pairs; ten tiles a job, four of them with masks); up to 9 tokens of 3 rows: 10.4 us,
// latency alone.  (Passes through the public call; the figures of variants below are of the
// GPU alone, from a graph, where the chunks take 6 us less.)
//
// A tile of which 64 keys hold all that its tokens see (a window's edge, the diagonal, first
// tokens that stay) is computed for those 64 alone.  The loading warp, which has the time,
// works out what each query tile sees of a key tile and leaves it as a word for the others;
// the product instructions are the same for both kinds, with other addresses (a branch
// around two bodies of them, or one that leaves out tiles that nothing sees, cost the
// issuing warp more than the smaller tiles save: chunks 89 us).
//
// Warps: 0 loads, 1 issues the products, 2 and 3 sum rows again where an unseen value spoilt
// them (see amend_row), then four per query tile for the softmax, to which the first four
// leave most of the registers.
#include <cuda.h>

#include <cmath>

#include "qs_attn.cuh"
#include "qs_sm100.cuh"

namespace qs {
namespace {

constexpr int kTile = 128;            // query rows of a tile, keys of a tile
constexpr float kBias = 6.f;
// Of 64 weights with the reference kept.  None of them may overflow float16; a first tile
// with few keys seen leaves a low reference, from which this has room for 2^3 with scores
// of ordinary spread (bias 8: 2^1, and chunks under a window took 93 us for 84).
// Bfloat16 weights hold more, but their products with large values go into float32 sums: with
// 2^30 those stay finite up to values of 1e26 and a thousand such tiles.
template <typename T>
constexpr float kMaxSum = std::is_same<T, __half>::value ? 60000.f : 0x1p30f;
constexpr int kHalf = kTile * 128;    // bytes of 128 rows of 64 values
constexpr uint64_t kDrainNs = kDefaultWaitNs;

template <int DP, int NQ>
struct Cfg {
  static constexpr int halves = DP / 64;
  static constexpr int tile_bytes = halves * kHalf;
  static constexpr int out_bytes = NQ * 4 * 32 * 128;  // 32 rows of 64 outputs per softmax warp
  static constexpr int room = (224 * 1024 - NQ * tile_bytes - out_bytes) / tile_bytes;
  static constexpr int stages = room > 8 ? 8 : room;
  static constexpr int threads = 128 + NQ * 128;
  static constexpr int tmem_cols = NQ * (kTile + DP) <= 256 ? 256 : 512;
  static constexpr int bars = 3 * stages + 5 * NQ + 10;
  static constexpr int smem = (NQ + stages) * tile_bytes + out_bytes + bars * 8 + 16 + 1024;
};

struct WindowArgs {
  AttnArgs a;
  int share, tokens_per_tile, granule;  // granule: keys of a load box
  int splits;                           // shares of a tile's keys
  float *part_o;                        // [split][token, head][DP] where splits > 1
  float2 *part_ml;                      // [split][token, head]: reference (log2), sum
  uint64_t wait_ns;
  int *error;
};

// 32 lanes x 32 columns of 32 bits.
__device__ __forceinline__ void tmem_ld_32(uint32_t addr, uint32_t *v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32(uint32_t addr, const uint32_t *v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
      "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
      "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 64 scores of a row (float32 in raw) to weights 2^(s scale2 + shift), as 16-bit values in
// raw's first half; returns their sum before that rounding.  The rounding is what the tensor
// core takes beside 16-bit values, and about as large as the output's own: the prompt's error
// against 64 bits is 2.0e-3 with it and 1.6e-3 without, drafted float16 tokens' 2.8e-4 and
// 2.1e-4.  A second product with what it leaves, as in the decode kernel, would add half to
// the tensor core's time, which is as long as the exponentials' now.  The special-function unit
// takes 8 cycles for a warp's exponential and bounds it: 533 cycles a warp with two warps
// on a scheduler.  A quarter of them as polynomials on the multiply-add pipe (26 cycles a
// pair against 16) took as long.
template <typename T>
__device__ __forceinline__ float weights(uint32_t *raw, float scale2, float shift) {
  const uint64_t scale_2 = pack2(scale2, scale2), shift_2 = pack2(shift, shift);
  uint64_t sums[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const uint64_t e2 = fma2(pack2(__uint_as_float(raw[2 * j]), __uint_as_float(raw[2 * j + 1])), scale_2, shift_2);
    float2 e = unpack2(e2);
    e.x = ex2(e.x);
    e.y = ex2(e.y);
    sums[j & 1] = add2(sums[j & 1], pack2(e.x, e.y));
    split16<T>(e.x, e.y, raw[j]);
  }
  const float2 sum = unpack2(add2(sums[0], sums[1]));
  return sum.x + sum.y;
}

// The largest of three; NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The largest of 64 scores; NaN if one is.
__device__ __forceinline__ float top_of(const uint32_t *raw) {
  const float *s = reinterpret_cast<const float *>(raw);
  float tops[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
  for (int c = 4; c < 64; c += 8)
#pragma unroll
    for (int x = 0; x < 4; ++x) tops[x] = max3(tops[x], s[c + x], c + 4 + x < 64 ? s[c + 4 + x] : s[c + x]);
  return max3(max3(tops[0], tops[1], tops[2]), tops[3], tops[3]);
}

// D[tmem] (+)= A[tmem] * B[smem], issued by one thread.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void *map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void *map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
          "r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}

// Descriptor of a tile whose rows are the product's K dimension (the values: 128 keys x
// 64 dimensions of 128 bytes, swizzled): blocks of 64 dimensions kHalf apart, groups of
// 8 keys 1024 bytes apart.
__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(kHalf >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

template <typename T>
constexpr uint32_t idesc_of(int n, bool b_mn_major) {
  const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return sm100::idesc_f16_f32(kTile, n) | (f << 7) | (f << 10) | ((b_mn_major ? 1u : 0u) << 16);
}

template <typename T>
__device__ __forceinline__ float2 floats_of(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
  else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w));
}

// The lowest n bits (none for n <= 0, all for n >= 32).
__device__ __forceinline__ uint32_t ones_below(int n) {
  return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u;
}

// The tiles of one block of the grid.
struct Job {
  int row;          // -1: none
  int head;         // key head
  int q0, q1;       // the row's tokens in q; without a row, those of all rows
  int t0;           // first token (in q; without a row, counted over the tokens of no row)
  int pos0;         // its place in the row
  int keys;         // keys that any of the tokens sees end before this
  int sink_tiles;   // key tiles from 0
  int from;         // first key after them
  int first, tiles; // this share's first tile, its tiles (0: tokens to clear, -1: no more jobs)
  int split;        // which share
};

// Registers per thread: 168 at launch (65536 / 384, in eights); the sum over the
// warpgroups stays 3 x 168.
template <int N>
__device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

// True in one thread of a warp that is here as a whole.  The compiler knows that it is
// one: what the product instructions take from uniform registers stays there, where a
// test of the lane number has every operand moved there first (chunks under a window took
// 122 us that way, 98 this way).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// Takes over the next block of the grid that has not started: the answer goes to `answer`
// (16 bytes) and completes on the barrier.
__device__ __forceinline__ void ask_next_block(uint32_t answer, uint32_t bar) {
  sm100::mbar_arrive_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer),
               "r"(bar)
               : "memory");
}
// The block taken over, or false where none was left.
__device__ __forceinline__ bool next_block(uint32_t answer, int &x, int &y, int &z) {
  uint32_t taken, bx, by, bz;
  asm volatile(
      "{\n\t.reg .b128 a;\n\t.reg .pred p;\n\tld.shared.b128 a, [%4];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
      "mov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, %2, %3, _}, a;\n\t}"
      : "=r"(taken), "=r"(bx), "=r"(by), "=r"(bz)
      : "r"(answer)
      : "memory");
  sm100::fence_proxy_async_smem();  // read before the next answer is written
  x = static_cast<int>(bx);
  y = static_cast<int>(by);
  z = static_cast<int>(bz);
  return taken != 0;
}

// Block (x, y, z) of the grid as a job (a whole warp): the rows' tiles in row order, a row's
// last tile (the most keys) first; y the key head, z the share of the keys.
__device__ __forceinline__ Job job_of(const WindowArgs &w, int x, int y, int z, int per, int lane) {
  const AttnArgs &a = w.a;
  const int total_tokens = static_cast<int>(a.tokens);
  Job j;
  j.row = -1;
  j.head = y;
  j.split = z;
  j.first = 0;
  j.q0 = j.q1 = j.t0 = 0;
  int end = 0, want = x, length = 0;
  for (int r0 = 0; r0 < a.rows && j.row < 0; r0 += 32) {
    const int r = r0 + lane;
    int q0 = 0, q1 = 0, n = 0, len = 0;
    if (r < a.rows) {
      len = a.lengths[r];
      q0 = clampi(a.cu[r], 0, total_tokens);
      q1 = clampi(a.cu[r + 1], q0, total_tokens);
      n = (q1 - q0 + per - 1) / per;
    }
    int sum = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += v;
    }
    const uint32_t who = __ballot_sync(0xffffffffu, want >= sum - n && want < sum);
    end = max(end, __reduce_max_sync(0xffffffffu, q1));
    if (who) {
      const int src = __ffs(who) - 1;
      j.row = r0 + src;
      j.q0 = __shfl_sync(0xffffffffu, q0, src);
      j.q1 = __shfl_sync(0xffffffffu, q1, src);
      length = max(0, __shfl_sync(0xffffffffu, len, src));
      const int local = __shfl_sync(0xffffffffu, want - (sum - n), src), all = __shfl_sync(0xffffffffu, n, src);
      j.t0 = j.q0 + (all - 1 - local) * per;
    } else {
      want -= __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  if (j.row >= 0) {
    const int cap = static_cast<int>(min(static_cast<int64_t>(a.width) << a.page_shift, static_cast<int64_t>(0x7ffffff0)));
    const int back = length - (j.q1 - j.q0);
    j.pos0 = back + (j.t0 - j.q0);
    const int last = back + min(j.q1, j.t0 + per) - 1 - j.q0;
    j.keys = clampi(last + 1, 0, min(length, cap));
    const int lo = a.window > 0 && j.pos0 + 1 > a.window ? static_cast<int>(j.pos0 + 1 - a.window) : 0;
    const int sinks = static_cast<int>(min(static_cast<int64_t>(min(lo, j.keys)), a.sinks));
    j.sink_tiles = (sinks + kTile - 1) / kTile;
    j.from = max(lo / w.granule * w.granule, j.sink_tiles * kTile);
    const int all = j.sink_tiles + max(0, (j.keys - j.from + kTile - 1) / kTile);
    j.first = static_cast<int>(static_cast<int64_t>(all) * z / w.splits);
    j.tiles = static_cast<int>(static_cast<int64_t>(all) * (z + 1) / w.splits) - j.first;
  } else {  // a block beyond the tiles clears its share of the tokens that belong to no row:
            // with ceil(tokens / per) blocks and one for each row with tokens there are enough
    j.q0 = a.rows > 0 ? clampi(a.cu[0], 0, total_tokens) : 0;
    j.q1 = end;
    j.t0 = want * per;
    j.tiles = 0;
  }
  return j;
}

// What a query tile's tokens see of a key tile, as the loading warp tells it to the others:
// where 64 keys from a multiple of 32 on hold all that any of them sees (a window's or the
// diagonal's edge, first tokens that stay), the products and the softmax take only those.
constexpr uint32_t kPlain = 1, kNarrow = 2;  // every token sees every key; 64 keys are enough
constexpr int kFrom = 2;                     // two bits: where those begin, in 32s
constexpr int kGaps = 8;                     // eight bits: 16s of keys whose page is missing
__device__ __forceinline__ int narrow_from(uint32_t s) { return static_cast<int>((s >> kFrom) & 3) * 32; }

__device__ __forceinline__ uint32_t span_of(const WindowArgs &w, const Job &j, int t, int k0, uint32_t gaps) {
  const int ahead = t * w.tokens_per_tile, tokens = min(j.q1 - j.t0 - ahead, w.tokens_per_tile);
  const int first = j.pos0 + ahead;
  const int64_t window = w.a.window > 0 ? w.a.window : int64_t(1) << 40, sinks = w.a.sinks;
  int lo = first + 1 > window ? static_cast<int>(first + 1 - window) - k0 : 0;
  int hi = min(min(first + tokens, j.keys) - k0, kTile);
  const bool plain = k0 + kTile <= min(first + 1, j.keys) && gaps == 0 &&
                     (k0 + kTile <= sinks || k0 > first + w.tokens_per_tile - 1 - window);
  if (plain) return kPlain;
  if (lo > 0 && sinks > k0) {
    if (lo >= hi) hi = static_cast<int>(min(static_cast<int64_t>(hi), sinks - k0));
    lo = 0;
  }
  lo = clampi(lo, 0, kTile - 64) / 32;
  return gaps << kGaps | (tokens <= 0 || hi <= lo * 32 + 64 ? kNarrow | lo << kFrom : 0u);
}

// Key `key` (from 0) of the job's key tile i, in tile order.
__device__ __forceinline__ int first_key(const Job &j, int i) {
  i += j.first;
  return i < j.sink_tiles ? i * kTile : j.from + (i - j.sink_tiles) * kTile;
}

// A value that a row does not see has weight 0 in its sum, and 0 x inf is NaN.  So a row
// (r of query tile t) whose sum is not finite is looked at by a whole warp, a few dimensions to
// a lane: where a key of its tiles that it does not see has an infinite or NaN value, and its
// own key has none that would explain the output, that dimension is summed again, key by key.
// By a warp that has nothing else to do: in the softmax warps' epilogue the same code took
// registers from their loop (a prompt of 8192 tokens 968 -> 1022 us).
template <typename T, int DP>
struct Amend {
  static constexpr int PER = DP / 32;  // dimensions of a lane
  const WindowArgs &w;
  const int lane;
  int token = -1;       // the last one looked at,
  uint32_t unseen = 0;  // and this lane's dimensions with such values among the keys that it does not see

  __device__ Amend(const WindowArgs &w_, int lane_) : w(w_), lane(lane_) {}

  static __device__ __forceinline__ uint32_t strange_of(const T *v) {  // a bit for each dimension
    uint32_t bits = 0;
#pragma unroll
    for (int c = 0; c < PER; c += 2) {
      constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
      const uint32_t x = *reinterpret_cast<const uint32_t *>(v + c);
      bits |= ((x & e) == e ? 1u : 0u) << c | ((x >> 16 & e) == e ? 2u : 0u) << c;
    }
    return bits;
  }

  __device__ __forceinline__ void row(const Job &j, int t, int r) {
    const AttnArgs &a = w.a;
    const int ahead = t * w.tokens_per_tile + r / w.share, pos = j.pos0 + ahead;
    const int last = min(pos, j.keys - 1), page_mask = (1 << a.page_shift) - 1;
    const int low = a.window > 0 && pos >= a.window ? static_cast<int>(pos - a.window) : -1;
    const int head = j.head * w.share + r % w.share;
    const bool mine = lane * PER < a.dim;  // this lane has dimensions
    const int64_t at = static_cast<int64_t>(j.t0 + ahead) * a.q_heads + head;
    const int *table = a.table + static_cast<int64_t>(j.row) * a.width;
    auto seen = [&](int key) { return key <= last && (key > low || key < a.sinks); };
    auto page_of = [&](int key) {  // -1 where there is none
      if (key < 0 || key >= j.keys) return -1;
      const int p = table[key >> a.page_shift];
      return p >= 0 && p < a.pages ? p : -1;
    };
    auto place = [&](const void *pool, const int64_t (&st)[3], int page, int key) {
      return static_cast<const T *>(pool) + page * st[0] + j.head * st[1] + (key & page_mask) * st[2];
    };
    float *part = w.splits > 1 ? w.part_o + (j.split * a.tokens * a.q_heads + at) * DP + lane * PER : nullptr;
    T *out = static_cast<T *>(a.out) + at * a.dim + lane * PER;
    uint32_t bad = 0;  // dimensions whose sum is not finite
    if (mine) {
      if (w.splits > 1)
#pragma unroll
        for (int c = 0; c < PER; ++c) bad |= (fabsf(part[c]) < INFINITY ? 0u : 1u) << c;
      else
        bad = strange_of(out);
    }
    // a model gone NaN: the token's own value says it all
    const int own = seen(last) ? page_of(last) : -1;
    if (mine && own >= 0) bad &= ~strange_of(place(a.v, a.vs, own, last) + lane * PER);
    if (!__any_sync(0xffffffffu, bad)) return;
    if (token != ahead) {  // the heads of a token see the same keys
      token = ahead;
      unseen = 0;
      for (int i = 0; i < j.tiles; ++i) {
        const int k0 = first_key(j, i);
        if (k0 + kTile - 1 <= last && (k0 > low || k0 + kTile <= a.sinks)) continue;  // all seen
        for (int key = k0; key < k0 + kTile; key += 16) {  // of one page
          const int page = page_of(key);
          if (page < 0) continue;
          const T *v = place(a.v, a.vs, page, key) + lane * PER;
#pragma unroll
          for (int x = 0; x < 16; ++x)
            if (mine && key + x < j.keys && !seen(key + x)) unseen |= strange_of(v + x * a.vs[2]);
        }
      }
    }
    bad &= unseen;
    if (!__any_sync(0xffffffffu, bad)) return;

    const uint4 *q = reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + static_cast<int64_t>(j.t0 + ahead) * a.q_token +
                                                     head * a.q_head);
    const int pieces = a.dim / 8;
    const float scale2 = a.scale * kLog2e;
    float m = -INFINITY, l = 0.f, o[PER] = {};
    for (int i = 0; i < j.tiles; ++i) {
      const int k0 = first_key(j, i);
#pragma unroll 1
      for (int k32 = k0; k32 < k0 + kTile; k32 += 32) {
        const int key = k32 + lane, page = seen(key) ? page_of(key) : -1;
        const uint32_t some = __ballot_sync(0xffffffffu, page >= 0);
        if (!some) continue;
        float s = -INFINITY;
        if (page >= 0) {
          const uint4 *k = reinterpret_cast<const uint4 *>(place(a.k, a.ks, page, key));
          float dot = 0.f;
#pragma unroll 4
          for (int c = 0; c < pieces; ++c) {
            const uint4 x = q[c], y = k[c];
            auto add = [&](uint32_t u, uint32_t v) {
              const float2 f = floats_of<T>(u), g = floats_of<T>(v);
              dot = fmaf(f.x, g.x, fmaf(f.y, g.y, dot));
            };
            add(x.x, y.x), add(x.y, y.y), add(x.z, y.z), add(x.w, y.w);
          }
          s = dot * scale2;
        }
        float top = s;
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        if (top > m) {
          const float f = ex2(m - top);
          l *= f;
#pragma unroll
          for (int c = 0; c < PER; ++c) o[c] *= f;
          m = top;
        }
        const float p = s == -INFINITY ? 0.f : ex2(s - m);
        l += p;
#pragma unroll 8
        for (int x = 0; x < 32; ++x) {
          const float px = __shfl_sync(0xffffffffu, p, x);
          const int page_x = __shfl_sync(0xffffffffu, page, x);
          if (page_x < 0 || !mine) continue;
          const T *v = place(a.v, a.vs, page_x, k32 + x) + lane * PER;
#pragma unroll
          for (int c = 0; c < PER; c += 2) {
            const float2 f = floats_of<T>(*reinterpret_cast<const uint32_t *>(v + c));
            o[c] = fmaf(px, f.x, o[c]);
            o[c + 1] = fmaf(px, f.y, o[c + 1]);
          }
        }
      }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    // beside the reference that the other dimensions have, or over the sum
    const float f = l == 0.f ? 0.f : w.splits > 1 ? ex2(m - w.part_ml[j.split * a.tokens * a.q_heads + at].x) : 1.f / l;
#pragma unroll
    for (int c = 0; c < PER; ++c)
      if (bad >> c & 1) {
        if (w.splits > 1) part[c] = o[c] * f;
        else store1(out + c, o[c] * f);
      }
  }
};

template <typename T, int DP, int NQ>
__global__ void __launch_bounds__(Cfg<DP, NQ>::threads, 1)
attn_window_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap, const WindowArgs w) {
  using C = Cfg<DP, NQ>;
  constexpr int S = C::stages;
  extern __shared__ uint8_t dsm[];
  __shared__ Job jobs[2];  // the current one and the next
  constexpr int kSpans = 16;
  static_assert(kSpans >= S / 2 + 3, "loads run ahead by half the ring");
  __shared__ uint32_t spans[kSpans][NQ];  // of the last key tiles
  __shared__ __align__(16) uint8_t answer_s[16];
  __shared__ uint32_t bads[2][NQ * 4];  // a job's rows whose sums are not finite, by softmax warp
  __shared__ uint32_t amended;          // rows summed again so far
  const AttnArgs &a = w.a;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  uint8_t *base = dsm + ((1024u - (smem_u32(dsm) & 1023u)) & 1023u);
  const uint32_t q_sm = smem_u32(base), ring = q_sm + NQ * C::tile_bytes;
  const uint32_t out_sm = ring + S * C::tile_bytes, bar0 = out_sm + C::out_bytes;
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (S + s); };
  auto landed = [&](int s) { return bar0 + 8u * (2 * S + s); };  // loads of a tile that is then cleared in part
  auto s_full = [&](int t) { return bar0 + 8u * (3 * S + t); };
  auto p_full = [&](int t) { return bar0 + 8u * (3 * S + NQ + t); };
  auto o_full = [&](int t) { return bar0 + 8u * (3 * S + 2 * NQ + t); };
  auto p_half = [&](int t) { return bar0 + 8u * (3 * S + 3 * NQ + t); };    // the first 64 keys' weights are stored
  auto half_done = [&](int t) { return bar0 + 8u * (3 * S + 4 * NQ + t); };  // and in O
  auto job_full = [&](int s) { return bar0 + 8u * (3 * S + 5 * NQ + s); };
  auto job_empty = [&](int s) { return bar0 + 8u * (3 * S + 5 * NQ + 2 + s); };
  const uint32_t q_full = bar0 + 8u * (3 * S + 5 * NQ + 4), q_empty = q_full + 8, asked = q_full + 16, drain = q_full + 24;
  auto summed = [&](int s) { return q_full + 32 + 8u * s; };  // a job's outputs are stored
  uint32_t *holder = reinterpret_cast<uint32_t *>(base + (NQ + S) * C::tile_bytes + C::out_bytes + C::bars * 8);

  if (tid == 0) {
    amended = 0;
    for (int s = 0; s < S; ++s) {
      sm100::mbar_init(full(s), 1);
      sm100::mbar_init(empty(s), 1);
      sm100::mbar_init(landed(s), 1);
    }
    for (int t = 0; t < NQ; ++t) {
      sm100::mbar_init(s_full(t), 1);
      sm100::mbar_init(p_full(t), 4);
      sm100::mbar_init(p_half(t), 4);
      sm100::mbar_init(half_done(t), 1);
      sm100::mbar_init(o_full(t), 1);
    }
    for (int s = 0; s < 2; ++s) {
      sm100::mbar_init(job_full(s), 1);
      sm100::mbar_init(job_empty(s), 3 + NQ * 128);
      sm100::mbar_init(summed(s), NQ * 4);
    }
    sm100::mbar_init(q_full, 1);
    sm100::mbar_init(q_empty, 1);
    sm100::mbar_init(asked, 1);
    sm100::mbar_init(drain, 1);
    sm100::fence_barrier_init();
    sm100::prefetch_tmap(&qmap);
    sm100::prefetch_tmap(&kmap);
    sm100::prefetch_tmap(&vmap);
  }
  if (warp == 1) sm100::tmem_alloc(smem_u32(holder), C::tmem_cols);
  pdl_wait();
  pdl_launch_dependents();
  sm100::tc_fence_before_sync();
  __syncthreads();
  sm100::tc_fence_after_sync();
  const uint32_t tmem = *holder;
  const int per = NQ * w.tokens_per_tile;
  auto key_of_tile = [&](const Job &j, int i) { return first_key(j, i); };
  // A wait between jobs, which rows being summed again may hold up: its limit starts anew with
  // each of them.
  auto wait_job = [&](uint32_t bar, uint32_t parity) {
    for (uint32_t before = 0;;) {
      if (sm100::mbar_wait_warp(bar, parity, w.wait_ns)) return true;
      const uint32_t now = __shfl_sync(0xffffffffu, *const_cast<volatile uint32_t *>(&amended), 0);
      if (now == before) return false;
      before = now;
    }
  };

  if (warp < 4) {
    if (NQ == 2) registers_down<72>();
    if (warp == 0) {
      // ---- jobs, and loads: Q, then K and V tiles through one ring.  Lane b takes box b.
      const int boxes = kTile / w.granule, mask = (1 << a.page_shift) - 1;
      const uint32_t answer = smem_u32(answer_s);
      int issued = 0, tiles = 0, q_loads = 0, asks = 0, answers = 0;
      uint32_t landed_phase = 0;
      bool ok = true;
      int bx = blockIdx.x, by = blockIdx.y, bz = blockIdx.z;
      for (int num = 0; ok; ++num) {
        const int slot = num & 1;
        const Job j = job_of(w, bx, by, bz, per, lane);
        if (num >= 2) ok = wait_job(job_empty(slot), ((num >> 1) - 1) & 1);
        if (!ok) break;
        if (lane == 0) {
          jobs[slot] = j;
          sm100::mbar_arrive(job_full(slot));
        }
        __syncwarp();
        // The next block is asked for with the last tile's loads: early enough for its own
        // loads to follow, and no earlier, or this CTA keeps it from one that is idle.
        auto ask = [&] {
          if (lane == 0) ask_next_block(answer, asked);
          ++asks;
          __syncwarp();
        };
        const int n = j.tiles;
        if (n > 0) {
          if (q_loads > 0) ok = sm100::mbar_wait_warp(q_empty, (q_loads - 1) & 1, w.wait_ns);
          if (!ok) break;
          if (lane == 0) {
            sm100::mbar_arrive_expect_tx(q_full, NQ * C::halves * 128 * w.share * w.tokens_per_tile);
            for (int t = 0; t < NQ; ++t)
              for (int h = 0; h < C::halves; ++h)
                tma_load_3d(q_sm + t * C::tile_bytes + h * kHalf, &qmap, h * 64, j.head * w.share,
                            j.t0 + t * w.tokens_per_tile, q_full);
          }
          ++q_loads;
        }
        const int *table = a.table + static_cast<int64_t>(max(j.row, 0)) * a.width;
        auto page_at = [&](int i) {  // lane b: the page of box b of tile i, -1 where there is none
          const int k = key_of_tile(j, i) + lane * w.granule;
          if (i >= n || lane >= boxes || k >= j.keys) return -1;
          const int p = table[k >> a.page_shift];
          return p >= 0 && p < a.pages ? p : -1;
        };
        int next_page = page_at(0);
        if (n == 0) ask();
        for (int i = 0; i < n && ok; ++i) {
          if (i + 1 == n) ask();
          const int page = next_page;
          next_page = page_at(i + 1);
          const int k0 = key_of_tile(j, i), k = k0 + lane * w.granule;
          const uint32_t have = __ballot_sync(0xffffffffu, page >= 0);
          const int bytes = __popc(have) * w.granule * 128 * C::halves;
          uint32_t gaps = __ballot_sync(0xffffffffu, page < 0 && lane < boxes && k < j.keys);  // boxes, then 16s
          gaps = __ballot_sync(0xffffffffu, lane < kTile / 16 && (gaps >> (lane * 16 / w.granule)) & 1u);
          if (lane < NQ)  // before the tile's loads: what reads it comes after them
            *const_cast<volatile uint32_t *>(&spans[tiles % kSpans][lane]) = span_of(w, j, lane, k0, gaps);
          ++tiles;
          __syncwarp();
          // values of absent pages and past the last key must be zero: their weights are,
          // but zero times what stale memory may hold need not be
          const bool partial = __popc(have) != boxes || k0 + kTile > j.keys;
#pragma unroll
          for (int kv = 0; kv < 2 && ok; ++kv) {
            const int s = issued % S, use = issued / S;
            if (use > 0) ok = sm100::mbar_wait_warp(empty(s), (use - 1) & 1, w.wait_ns);
            if (!ok) break;
            const bool clear = kv == 1 && partial;
            const uint32_t bar = clear ? landed(s) : full(s), dst = ring + s * C::tile_bytes;
            if (lane == 0) sm100::mbar_arrive_expect_tx(bar, bytes);
            __syncwarp();
            if (page >= 0)
              for (int h = 0; h < C::halves; ++h)
                tma_load_4d(dst + h * kHalf + lane * w.granule * 128, kv ? &vmap : &kmap, h * 64, k & mask, j.head, page,
                            bar);
            ++issued;
            if (clear) {
              ok = sm100::mbar_wait_warp(bar, (landed_phase >> s) & 1, w.wait_ns);
              // given up, but the copies must not outlive the CTA
              if (!ok && !sm100::mbar_wait_warp(bar, (landed_phase >> s) & 1, kDrainNs)) *w.error = 1;
              landed_phase ^= 1u << s;
              for (int r = lane; r < kTile; r += 32) {
                const int p = __shfl_sync(0xffffffffu, page, r / w.granule);
                if (p < 0 || k0 + r >= j.keys)
                  for (int h = 0; h < C::halves; ++h)
                    for (int c = 0; c < 8; ++c)
                      asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(dst + h * kHalf + r * 128 + c * 16),
                                   "r"(0)
                                   : "memory");
              }
              sm100::fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) sm100::mbar_arrive(full(s));
            }
          }
        }
        if (!ok) break;
        ok = sm100::mbar_wait_warp(asked, num & 1, w.wait_ns);
        if (ok) ++answers;
        if (!ok || !next_block(answer, bx, by, bz)) {
          // no block is left: the job after this one says so
          const int last = (num + 1) & 1;
          if (ok && num >= 1) ok = wait_job(job_empty(last), (((num + 1) >> 1) - 1) & 1);
          if (ok && lane == 0) {
            jobs[last].tiles = -1;
            sm100::mbar_arrive(job_full(last));
          }
          break;
        }
      }
      if (!ok) *w.error = 1;
      // wind down: every load and answer must have landed before the CTA exits
      if (lane == 0) {
        if (asks > answers && !sm100::mbar_wait_bounded(asked, answers & 1, kDrainNs)) *w.error = 1;
        if (q_loads && !sm100::mbar_wait_bounded(q_full, (q_loads - 1) & 1, kDrainNs)) *w.error = 1;
        for (int x = issued > S ? issued - S : 0; x < issued; ++x)
          if (!sm100::mbar_wait_bounded(full(x % S), (x / S) & 1, kDrainNs)) *w.error = 1;
      }
    } else if (warp == 1) {
      // ---- products: the warp waits, one thread issues
      constexpr uint32_t id_s = idesc_of<T>(kTile, false), id_n = idesc_of<T>(kTile / 2, false), id_o = idesc_of<T>(DP, true);
      auto stage_of = [&](int x) { return ring + (x % S) * C::tile_bytes; };
      auto wait_tile = [&](int x) { return sm100::mbar_wait_warp(full(x % S), (x / S) & 1, w.wait_ns); };
      auto span_at = [&](int t, int i) {  // of key tile i, counted through the jobs
        const uint32_t span = *const_cast<volatile uint32_t *>(&spans[i % kSpans][t]);
        return __reduce_or_sync(0xffffffffu, span);  // a uniform register: see elect_one
      };
      auto scores = [&](int t, int x, int i) {  // S of query tile t over the keys of tile i, in ring place x
        const uint32_t span = span_at(t, i);
        const uint64_t qd = sm100::sw128_kmajor_desc(q_sm + t * C::tile_bytes), kd = sm100::sw128_kmajor_desc(stage_of(x));
        const bool narrow = span & kNarrow;
        const uint32_t id = narrow ? id_n : id_s, from = narrow ? narrow_from(span) : 0;
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < DP / 16; ++k) {
            const uint32_t off = ((k / 4) * kHalf + (k % 4) * 32) >> 4;
            sm100::umma_f16(tmem + t * kTile + from, qd + off, kd + (from * 128 >> 4) + off, id, k != 0);
          }
          sm100::umma_commit(s_full(t));
        }
        __syncwarp();
      };
      auto commit = [&](uint32_t bar) {
        if (elect_one()) sm100::umma_commit(bar);
        __syncwarp();
      };
      bool ok = true;
      int q_loads = 0, place = 0, step = 0;  // place: of the job's first tile in the ring; step: key tiles so far
      for (int num = 0; ok; ++num) {
        const int slot = num & 1;
        ok = wait_job(job_full(slot), (num >> 1) & 1);
        if (!ok) break;
        const int n = __shfl_sync(0xffffffffu, jobs[slot].tiles, 0);
        if (n < 0) break;
        if (lane == 0) sm100::mbar_arrive(job_empty(slot));
        __syncwarp();
        if (n == 0) continue;
        ok = sm100::mbar_wait_warp(q_full, q_loads & 1, w.wait_ns) && wait_tile(place);
        ++q_loads;
        if (!ok) break;
        sm100::tc_fence_after_sync();
        for (int t = 0; t < NQ; ++t) scores(t, place, step);
        commit(empty(place % S));
        if (n == 1) commit(q_empty);
        for (int i = 0; i < n && ok; ++i) {
          const int k_next = place + 2 * i + 2, v = place + 2 * i + 1;
          ok = wait_tile(v);
          for (int t = 0; t < NQ && ok; ++t) {
            const uint64_t vb = sw128_mnmajor_desc(stage_of(v));
            const uint32_t od = tmem + NQ * kTile + t * DP, pa = tmem + t * kTile;
            const uint32_t span = span_at(t, step + i);
            const bool narrow = span & kNarrow;
            const uint32_t from = narrow ? narrow_from(span) / 16 : 0;
            ok = sm100::mbar_wait_warp(p_half(t), (step + i) & 1, w.wait_ns);
            if (!ok) break;
            sm100::tc_fence_after_sync();
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < kTile / 32; ++k)
                umma_ts(od, pa + (from + k) * 8, vb + (from + k) * (16 * 128 >> 4), id_o, k != 0 || i != 0);
              sm100::umma_commit(half_done(t));
            }
            __syncwarp();
            ok = sm100::mbar_wait_warp(p_full(t), (step + i) & 1, w.wait_ns);
            if (!ok) break;
            sm100::tc_fence_after_sync();
            if (elect_one()) {
              if (!narrow) {
#pragma unroll
                for (int k = kTile / 32; k < kTile / 16; ++k) umma_ts(od, pa + k * 8, vb + k * (16 * 128 >> 4), id_o, 1);
              }
              if (i + 1 == n) sm100::umma_commit(o_full(t));
            }
            __syncwarp();
            if (i + 1 < n) {
              if (t == 0) ok = wait_tile(k_next);
              if (!ok) break;
              sm100::tc_fence_after_sync();
              scores(t, k_next, step + i + 1);
            }
          }
          if (!ok) break;
          commit(empty(v % S));
          if (i + 1 < n) commit(empty(k_next % S));
          if (i + 2 == n) commit(q_empty);  // the last scores are under way
        }
        place += 2 * n;
        step += n;
      }
      if (!ok) *w.error = 1;
      commit(drain);
      if (!sm100::mbar_wait_warp(drain, 0, kDrainNs)) *w.error = 1;
    } else {
      // ---- rows to be summed again, every second softmax warp's each
      Amend<T, DP> amend(w, lane);
      bool ok = true;
      uint32_t summed_phase = 0;
      for (int num = 0; ok; ++num) {
        const int slot = num & 1;
        ok = wait_job(job_full(slot), (num >> 1) & 1);
        if (!ok) break;
        const int n = __shfl_sync(0xffffffffu, jobs[slot].tiles, 0);
        if (n < 0) break;
        if (n > 0) {
          ok = sm100::mbar_wait_warp(summed(slot), (summed_phase >> slot) & 1, w.wait_ns);
          summed_phase ^= 1u << slot;
          if (!ok) break;
          for (int from = warp - 2; from < NQ * 4; from += 2) {
            uint32_t bad = *const_cast<volatile uint32_t *>(&bads[slot][from]);
            for (; bad; bad &= bad - 1) {
              amend.row(jobs[slot], from >> 2, (from & 3) * 32 + __ffs(bad) - 1);
              if (lane == 0) atomicAdd(&amended, 1u);
            }
          }
          amend.token = -1;
        }
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(job_empty(slot));
      }
      if (!ok) *w.error = 1;
    }
  } else {
    if (NQ == 2) registers_up<216>();
    // ---- softmax: one thread per query row
    const int t = (warp - 4) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_at = tmem + lanes + t * kTile, o_at = tmem + lanes + NQ * kTile + t * DP;
    const int tok = r / w.share;
    const int64_t win = a.window > 0 ? a.window : (int64_t(1) << 40);
    const int sinks = static_cast<int>(min(a.sinks, static_cast<int64_t>(0x7fffffff)));
    const float scale2 = a.scale * kLog2e;
    bool ok = true;
    int step = 0, outs = 0;
    for (int num = 0; ok; ++num) {
      const int slot = num & 1;
      ok = wait_job(job_full(slot), (num >> 1) & 1);
      if (!ok) break;
      const Job j = jobs[slot];
      const int n = j.tiles;
      if (n < 0) break;
      if (n == 0) {
        const int begin = jobs[slot].q0, held = jobs[slot].row >= 0 ? 0 : j.q1 - begin;  // tokens of the rows
        const int end = jobs[slot].row >= 0 ? j.q1 : static_cast<int>(a.tokens) - held;
        const int count = max(0, min(end - j.t0, per)) * w.share;
        for (int i = tid - 128; i < count * a.dim; i += NQ * 128) {
          int token = j.t0 + i / a.dim / w.share;
          if (token >= begin) token += held;
          const int64_t at = static_cast<int64_t>(token) * a.q_heads + j.head * w.share + i / a.dim % w.share;
          if (w.splits > 1) {  // an empty share
            if (i % a.dim == 0) w.part_ml[j.split * a.tokens * a.q_heads + at] = make_float2(-INFINITY, 0.f);
            continue;
          }
          store1(static_cast<T *>(a.out) + at * a.dim + i % a.dim, 0.f);
          if (i % a.dim == 0 && a.lse) a.lse[at] = -INFINITY;
        }
        sm100::mbar_arrive(job_empty(slot));
        continue;
      }
      const int token = j.t0 + t * w.tokens_per_tile + tok;
      const bool real = tok < w.tokens_per_tile && token < j.q1;
      const int pos = j.pos0 + t * w.tokens_per_tile + tok;
      // keys seen: k <= pos, where the row's line has so many, and k > pos - window or k < sinks
      const int last = min(pos, j.keys - 1);
      const int low = static_cast<int>(max(static_cast<int64_t>(-1), pos - win));  // keys above it are recent
      float m = -INFINITY, l = 0.f;  // m in the units of S
      for (int i = 0; i < n; ++i) {
        ok = sm100::mbar_wait_warp(s_full(t), (step + i) & 1, w.wait_ns);
        if (!ok) break;
        sm100::tc_fence_after_sync();
        uint32_t raw[kTile];
        auto load = [&] {
#pragma unroll
          for (int c = 0; c < kTile; c += 32) tmem_ld_32(s_at + c, raw + c);
          sm100::tmem_ld_wait();
        };
        auto tell = [&](uint32_t bar) {  // that weights are stored
          tmem_st_wait();
          sm100::tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) sm100::mbar_arrive(bar);
        };
        auto store = [&](int half) {  // the weights of 64 keys, over the first quarters of S
          tmem_st_32(s_at + 32 * half, raw + 64 * half);
          tell(half ? p_full(t) : p_half(t));
        };
        auto rescale = [&](float mn) {  // to a new reference
          const float f = m == mn ? 1.f : ex2((m - mn) * scale2);
#pragma unroll
          for (int c = 0; c < DP; c += 32) {
            uint32_t o[32];
            tmem_ld_32(o_at + c, o);
            sm100::tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
            tmem_st_32(o_at + c, o);
          }
          l *= f;
          m = mn;
        };
        const uint32_t span = *const_cast<volatile uint32_t *>(&spans[(step + i) % kSpans][t]);
        load();  // what no token sees of it holds anything, and is not looked at
        const int k0 = key_of_tile(j, i);
        const bool plain = span & kPlain, narrow = span & kNarrow;
        if (plain && i > 0) {
          // Most tiles: no mask, and the reference of the tiles before will do, which shows
          // afterwards.  No weight is above the sum's bound, which float16 holds.  The
          // product with the first 64 keys' values starts before the others' weights are
          // made.
          const float shift = kBias - m * scale2;
          const float sum = weights<T>(raw, scale2, shift);
          if (!__any_sync(0xffffffffu, real && !(sum <= kMaxSum<T> && m > -INFINITY))) {
            store(0);
            l += sum;
            float sum2 = weights<T>(raw + 64, scale2, shift);
            if (__any_sync(0xffffffffu, real && !(sum2 <= kMaxSum<T>))) {
              // a new reference in the middle: O takes it once the first half is in
              ok = sm100::mbar_wait_warp(half_done(t), (step + i) & 1, w.wait_ns);
              if (!ok) break;
              sm100::tc_fence_after_sync();
              tmem_ld_32(s_at + 64, raw + 64);
              tmem_ld_32(s_at + 96, raw + 96);
              sm100::tmem_ld_wait();
              const float top = top_of(raw + 64);
              rescale(top <= m ? m : top);
              sum2 = weights<T>(raw + 64, scale2, kBias - m * scale2);
            }
            l += sum2;
            store(1);
            continue;
          }
          load();  // S is still in its place
        }
        float *s = reinterpret_cast<float *>(raw);
        // of 32 keys from b on, what the row does not see becomes -inf: as bits, the places up
        // to hi that are above lo or below sk
        auto mask = [&](float *s, int b) {
          const int hi = last - k0, lo = low - k0, sk = sinks - k0;
          uint32_t see = ones_below(hi + 1 - b) & (~ones_below(lo + 1 - b) | ones_below(sk - b));
          const uint32_t gone = span >> (kGaps + b / 16);
          see &= ~((gone & 1u ? 0xffffu : 0u) | (gone & 2u ? 0xffff0000u : 0u));
#pragma unroll
          for (int c = 0; c < 32; ++c) s[c] = (see >> c) & 1 ? s[c] : -INFINITY;
        };
        const int from = narrow ? narrow_from(span) : 0;
        if (narrow) {
          tmem_ld_32(s_at + from, raw);
          tmem_ld_32(s_at + from + 32, raw + 32);
          sm100::tmem_ld_wait();
        }
        if (!plain) {
          mask(s, from);
          mask(s + 32, from + 32);
        }
        float top = top_of(raw);
        if (!narrow) {
          if (!plain) {
            mask(s + 64, 64);
            mask(s + 96, 96);
          }
          top = max3(top, top_of(raw + 64), top);
        }
        const bool renew = m == -INFINITY ? top != -INFINITY : !((top - m) * scale2 <= 7.f);  // NaN stays; 2^(7 + kBias) fits float16
        if (i == 0) m = top;
        else if (__any_sync(0xffffffffu, renew)) rescale(renew ? top : m);
        const float shift = m == -INFINITY ? 0.f : kBias - m * scale2;
        l += weights<T>(raw, scale2, shift);
        tmem_st_32(s_at + from / 2, raw);
        tell(p_half(t));
        if (!narrow) {
          l += weights<T>(raw + 64, scale2, shift);
          tmem_st_32(s_at + 32, raw + 64);
        }
        tell(p_full(t));
      }
      if (!ok) break;
      step += n;
      ok = sm100::mbar_wait_warp(o_full(t), outs & 1, w.wait_ns);
      ++outs;
      if (!ok) break;
      sm100::mbar_arrive(job_empty(slot));
      sm100::tc_fence_after_sync();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int64_t at = static_cast<int64_t>(token) * a.q_heads + j.head * w.share + r % w.share;
      // 32 words of each row at a time through shared memory, so that a warp stores whole
      // lines: four rows of 128 bytes where its threads' own rows would be 32 lines for 16
      // bytes each
      const uint32_t stage = out_sm + (warp - 4) * 4096, mine = stage + lane * 128;
      const uint32_t reals = __ballot_sync(0xffffffffu, real);
      const int64_t from = real ? at : 0;
      auto send = [&](const uint32_t *words, char *rows, int64_t row_bytes, int bytes) {
#pragma unroll
        for (int x = 0; x < 8; ++x)
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(mine + ((x ^ (lane & 7)) << 4)), "r"(words[4 * x]),
                       "r"(words[4 * x + 1]), "r"(words[4 * x + 2]), "r"(words[4 * x + 3])
                       : "memory");
        __syncwarp();
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int row = 4 * x + (lane >> 3), piece = lane & 7;
          const int64_t to = __shfl_sync(0xffffffffu, from, row);
          uint4 v;
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                       : "r"(stage + row * 128 + ((piece ^ (row & 7)) << 4))
                       : "memory");
          if (((reals >> row) & 1) && piece * 16 < bytes) *reinterpret_cast<uint4 *>(rows + to * row_bytes + piece * 16) = v;
        }
        __syncwarp();
      };
      // whether the sums are finite: 0 times them is then 0 (see Amend)
      uint64_t test[4] = {};
      auto look = [&](const uint32_t *o) {
#pragma unroll
        for (int x = 0; x < 32; x += 2)
          test[x / 2 % 4] = fma2(pack2(__uint_as_float(o[x]), __uint_as_float(o[x + 1])), 0, test[x / 2 % 4]);
      };
      uint32_t bad = 0;
      auto report = [&] {
        if (lane == 0) {
          *const_cast<volatile uint32_t *>(&bads[slot][warp - 4]) = bad;
          sm100::mbar_arrive(summed(slot));
        }
      };
      auto tested = [&] {  // the usual answer goes out while the outputs are being stored
        const float2 z = unpack2(add2(add2(test[0], test[1]), add2(test[2], test[3])));
        bad = __ballot_sync(0xffffffffu, real && l < INFINITY && !(z.x + z.y == 0.f));
        if (bad == 0) report();
      };
      auto stored = [&] {
        __syncwarp();
        if (bad) report();
      };
      if (w.splits > 1) {
        const int64_t base = j.split * a.tokens * a.q_heads;
#pragma unroll
        for (int c = 0; c < DP; c += 32) {
          uint32_t o[32];
          tmem_ld_32(o_at + c, o);
          sm100::tmem_ld_wait();
          look(o);
          if (c + 32 == DP) tested();
          send(o, reinterpret_cast<char *>(w.part_o + base * DP + c), DP * 4, 128);
        }
        if (real) w.part_ml[base + at] = make_float2(m == -INFINITY ? -INFINITY : m * scale2 - kBias, l);
        sm100::tc_fence_before_sync();
        stored();
        continue;
      }
#pragma unroll
      for (int c = 0; c < DP; c += 64) {
        uint32_t o[64];
        tmem_ld_32(o_at + c, o);
        tmem_ld_32(o_at + c + 32, o + 32);
        sm100::tmem_ld_wait();
        look(o);
        look(o + 32);
        if (c + 64 == DP) tested();
#pragma unroll
        for (int x = 0; x < 32; ++x)
          split16<T>(__uint_as_float(o[2 * x]) * inv, __uint_as_float(o[2 * x + 1]) * inv, o[x]);
        send(o, reinterpret_cast<char *>(static_cast<T *>(a.out) + c), a.dim * 2, (a.dim - c) * 2);
      }
      sm100::tc_fence_before_sync();  // O is read: the next job's first weights release it
      if (real && a.lse) a.lse[at] = l == 0.f ? -INFINITY : (m == -INFINITY ? 0.f : (m * scale2 - kBias) * kLn2) + logf(l);
      stored();
    }
    if (!ok) *w.error = 1;
  }
  sm100::tc_fence_before_sync();
  __syncthreads();
  sm100::tc_fence_after_sync();
  if (warp == 1) sm100::tmem_dealloc(tmem, C::tmem_cols);
}

// Joins a row's shares, a warp for each token and query head.
template <typename T, int DP>
__global__ void __launch_bounds__(256) window_join_kernel(WindowArgs w) {
  constexpr int PER = DP / 32, U = 4;  // outputs per lane, shares at a time
  pdl_wait();
  pdl_launch_dependents();
  const AttnArgs &a = w.a;
  const int lane = threadIdx.x & 31;
  const int64_t rows = a.tokens * a.q_heads, at = blockIdx.x * int64_t(8) + (threadIdx.x >> 5);
  if (at >= rows) return;
  float m = -INFINITY;
  for (int i = lane; i < w.splits; i += 32) m = fmaxf(m, w.part_ml[i * rows + at].x);
#pragma unroll
  for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  float l = 0.f, o[PER] = {};
  for (int i0 = 0; i0 < w.splits; i0 += U) {
    float2 ml[U];
    float x[U][PER];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u >= w.splits) break;
      ml[u] = w.part_ml[(i0 + u) * rows + at];
#pragma unroll
      for (int c = 0; c < PER; ++c) x[u][c] = w.part_o[((i0 + u) * rows + at) * DP + lane * PER + c];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u >= w.splits) break;
      if (ml[u].y == 0.f) continue;  // an empty share has no output
      const float p = weight(ml[u].x, m);
      l += p * ml[u].y;
#pragma unroll
      for (int c = 0; c < PER; ++c) o[c] += p * x[u][c];
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int c = 0; c < PER; c += 2) {
    uint32_t packed;
    split16<T>(o[c] * inv, o[c + 1] * inv, packed);
    if (lane * PER + c < a.dim) *reinterpret_cast<uint32_t *>(static_cast<T *>(a.out) + at * a.dim + lane * PER + c) = packed;
  }
  if (lane == 0 && a.lse) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// Query tiles of a block: one where the rows' tokens fill no more than one on average (a
// second would mostly be empty: 16 rows of 8 tokens over 16000 keys), else two.
int query_tiles(int64_t tokens, int64_t rows, int64_t share) { return tokens <= rows * (kTile / share) ? 1 : 2; }

// Shares of a tile's keys: as many as there are SMs for, of at least two key tiles each.
int splits_for(int64_t tokens, int64_t rows, int64_t q_heads, int64_t kv_heads, int64_t page, int64_t width,
               int64_t window, int64_t sinks) {
  const int64_t share = q_heads / kv_heads;
  if (share > kTile || tokens < 1 || rows < 1) return 1;
  const int64_t per = query_tiles(tokens, rows, share) * (kTile / share);
  int64_t blocks = ceil_div(tokens, per);  // there are at least so many, or as many as rows with tokens
  if (blocks < (rows < tokens ? rows : tokens)) blocks = rows < tokens ? rows : tokens;
  int64_t keys = width * page;
  if (window > 0 && window < keys && sinks < keys && window + sinks + per < keys) keys = window + sinks + per;
  int64_t n = ceil_div(ceil_div(keys, kTile), 2);
  if (n > 148 / (blocks * kv_heads)) n = 148 / (blocks * kv_heads);
  return static_cast<int>(n < 1 ? 1 : n);
}

template <typename T, int DP, int NQ>
int run(const AttnArgs &a, cudaStream_t s) {
  using C = Cfg<DP, NQ>;
  const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  WindowArgs w;
  w.a = a;
  w.share = a.q_heads / a.kv_heads;
  w.tokens_per_tile = kTile / w.share;
  const int page = 1 << a.page_shift;
  w.granule = page < kTile ? page : kTile;
  w.wait_ns = pipeline_wait_ns();
  w.error = device_error_flag();
  if (!w.error) return fail(QS_ERR_CUDA, "attention (window): no device error flag");
  CUtensorMap qmap, kmap, vmap;
  {
    const int64_t dims[3] = {a.dim, a.q_heads, a.tokens}, st[2] = {a.q_head, a.q_token};
    const int box[3] = {64, w.share, w.tokens_per_tile};
    const int e = encode_16bit_map(&qmap, a.q, bf16, 3, dims, st, box);
    if (e) return e;
  }
  for (int i = 0; i < 2; ++i) {
    const int64_t *str = i ? a.vs : a.ks;
    const int64_t dims[4] = {a.dim, page, a.kv_heads, a.pages}, st[3] = {str[2], str[1], str[0]};
    const int box[4] = {64, w.granule, 1, 1};
    const int e = encode_16bit_map(i ? &vmap : &kmap, i ? a.v : a.k, bf16, 4, dims, st, box);
    if (e) return e;
  }
  auto kern = attn_window_kernel<T, DP, NQ>;
  static std::atomic<uint64_t> allowed{0};
  int st = allow_smem("attention (window)", kern, C::smem, allowed);
  if (st) return st;
  const int64_t per = static_cast<int64_t>(NQ) * w.tokens_per_tile;
  const int64_t rows = a.tokens * a.q_heads;
  w.splits = splits_for(a.tokens, a.rows, a.q_heads, a.kv_heads, page, a.width, a.window, a.sinks);
  w.part_o = static_cast<float *>(a.ws);
  w.part_ml = reinterpret_cast<float2 *>(w.part_o + w.splits * rows * DP);
  const int64_t most_rows = a.rows < a.tokens ? a.rows : a.tokens;  // that have a token
  const dim3 grid(static_cast<unsigned>(ceil_div(a.tokens, per) + most_rows), a.kv_heads, w.splits);
  st = launch_pdl("attention (window)", kern, grid, dim3(C::threads), C::smem, s, qmap, kmap, vmap, w);
  if (st || w.splits == 1) return st;
  return launch_pdl("attention (window, join)", window_join_kernel<T, DP>, dim3(static_cast<unsigned>(ceil_div(rows, 8))),
                    dim3(256), 0, s, w);
}

}  // namespace

int64_t attn_window_workspace_bytes(int64_t tokens, int64_t rows, int64_t q_heads, int64_t kv_heads, int64_t dim,
                                    int64_t page, int64_t width, int64_t window, int64_t sinks) {
  const int64_t splits = splits_for(tokens, rows, q_heads, kv_heads, page, width, window, sinks);
  return splits == 1 ? 0 : splits * tokens * q_heads * ((dim <= 64 ? 64 : 128) + 2) * 4;
}

template <typename T>
int run_type(const AttnArgs &a, cudaStream_t s) {
  const bool one = query_tiles(a.tokens, a.rows, a.q_heads / a.kv_heads) == 1;
  if (a.dim <= 64) return one ? run<T, 64, 1>(a, s) : run<T, 64, 2>(a, s);
  return one ? run<T, 128, 1>(a, s) : run<T, 128, 2>(a, s);
}

int launch_attn_window(const AttnArgs &a, cudaStream_t s) {
  return a.dtype == QS_F16 ? run_type<__half>(a, s) : run_type<__nv_bfloat16>(a, s);
}

}  // namespace qs
