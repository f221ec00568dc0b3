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
// The maximum that the weights refer to is renewed, and O rescaled, only when it has
// grown by more than 2^8: until then weights up to 2^8 are exact in the float32 sum
// and lose nothing in the 16-bit ones, and most tiles rescale nothing.
//
// Warps: 0 loads, 1 issues the products (2 and 3 only fill their warpgroup), then four
// per query tile for the softmax, to which the first four leave most of the registers.
#include <cuda.h>

#include <cmath>

#include "qs_attn.cuh"
#include "qs_sm100.cuh"

namespace qs {
namespace {

constexpr int kTile = 128;            // query rows of a tile, keys of a tile
constexpr int kHalf = kTile * 128;    // bytes of 128 rows of 64 values
constexpr uint64_t kDrainNs = kDefaultWaitNs;

template <int DP, int NQ>
struct Cfg {
  static constexpr int halves = DP / 64;
  static constexpr int tile_bytes = halves * kHalf;
  static constexpr int stages = (224 * 1024 - NQ * tile_bytes) / tile_bytes > 8 ? 8 : (224 * 1024 - NQ * tile_bytes) / tile_bytes;
  static constexpr int threads = 128 + NQ * 128;
  static constexpr int tmem_cols = NQ * (kTile + DP) <= 256 ? 256 : 512;
  static constexpr int bars = 1 + 3 * stages + 3 * NQ + 1;
  static constexpr int smem = (NQ + stages) * tile_bytes + bars * 8 + 16 + 1024;
};

struct WindowArgs {
  AttnArgs a;
  int share, tokens_per_tile, granule;  // granule: keys of a load box
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
__device__ __forceinline__ void tmem_st_16(uint32_t addr, const uint32_t *v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15};" ::"r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

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

// What a CTA works on.
struct Job {
  int row;             // -1: none
  int q0, q1;          // the row's tokens in q
  int t0;              // first token of this CTA (in q)
  int pos0;            // its place in the row
  int keys;            // keys that any token of the CTA sees end before this
  int sink_tiles;      // key tiles from 0
  int from, tiles;     // first key after them, tiles in all
};

// Registers per thread: 168 at launch (65536 / 384, in eights); the sum over the
// warpgroups stays 3 x 168.
template <int N>
__device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

template <typename T, int DP, int NQ>
__global__ void __launch_bounds__(Cfg<DP, NQ>::threads, 1)
attn_window_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap, const WindowArgs w) {
  using C = Cfg<DP, NQ>;
  constexpr int S = C::stages;
  extern __shared__ uint8_t dsm[];
  __shared__ Job job_s;
  __shared__ volatile int absent;  // a page among the keys is missing: set before its tile's loads
  const AttnArgs &a = w.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t *base = dsm + ((1024u - (smem_u32(dsm) & 1023u)) & 1023u);
  const uint32_t q_sm = smem_u32(base), ring = q_sm + NQ * C::tile_bytes;
  const uint32_t bar0 = ring + S * C::tile_bytes;
  const uint32_t q_full = bar0;
  auto full = [&](int s) { return bar0 + 8u * (1 + s); };
  auto empty = [&](int s) { return bar0 + 8u * (1 + S + s); };
  auto landed = [&](int s) { return bar0 + 8u * (1 + 2 * S + s); };  // loads of a tile that is then cleared in part
  auto s_full = [&](int t) { return bar0 + 8u * (1 + 3 * S + t); };
  auto p_full = [&](int t) { return bar0 + 8u * (1 + 3 * S + NQ + t); };
  auto o_full = [&](int t) { return bar0 + 8u * (1 + 3 * S + 2 * NQ + t); };
  const uint32_t drain = bar0 + 8u * (1 + 3 * S + 3 * NQ);
  uint32_t *holder = reinterpret_cast<uint32_t *>(base + (NQ + S) * C::tile_bytes + C::bars * 8);

  if (tid == 0) {
    absent = 0;
    sm100::mbar_init(q_full, 1);
    for (int s = 0; s < S; ++s) {
      sm100::mbar_init(full(s), 1);
      sm100::mbar_init(empty(s), 1);
      sm100::mbar_init(landed(s), 1);
    }
    for (int t = 0; t < NQ; ++t) {
      sm100::mbar_init(s_full(t), 1);
      sm100::mbar_init(p_full(t), 128);
      sm100::mbar_init(o_full(t), 1);
    }
    sm100::mbar_init(drain, 1);
    sm100::fence_barrier_init();
  }
  if (warp == 1) sm100::tmem_alloc(smem_u32(holder), C::tmem_cols);
  pdl_wait();
  pdl_launch_dependents();

  // ---- which tokens: CTAs deal the rows' tiles in row order, a row's last tile (the
  // most keys) first
  const int per = NQ * w.tokens_per_tile;
  const int total_tokens = static_cast<int>(a.tokens);
  if (warp == 0) {
    int want = blockIdx.x;
    Job j;
    j.row = -1;
    j.q0 = j.q1 = j.t0 = 0;
    int end = 0;
    for (int r0 = 0; r0 < a.rows && j.row < 0; r0 += 32) {
      const int r = r0 + lane;
      int q0 = 0, q1 = 0, n = 0;
      if (r < a.rows) {
        q0 = clampi(a.cu[r], 0, total_tokens);
        q1 = clampi(a.cu[r + 1], q0, total_tokens);
        n = (q1 - q0 + per - 1) / per;
      }
      int x = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      const bool mine = want >= x - n && want < x;
      const uint32_t who = __ballot_sync(0xffffffffu, mine);
      end = max(end, __reduce_max_sync(0xffffffffu, q1));
      if (who) {
        const int src = __ffs(who) - 1;
        j.row = r0 + src;
        j.q0 = __shfl_sync(0xffffffffu, q0, src);
        j.q1 = __shfl_sync(0xffffffffu, q1, src);
        const int local = __shfl_sync(0xffffffffu, want - (x - n), src), all = __shfl_sync(0xffffffffu, n, src);
        j.t0 = j.q0 + (all - 1 - local) * per;
      } else {
        want -= __shfl_sync(0xffffffffu, x, 31);
      }
    }
    if (j.row >= 0) {
      const int length = max(0, a.lengths[j.row]);
      const int cap = static_cast<int>(min(static_cast<int64_t>(a.width) << a.page_shift, static_cast<int64_t>(0x7ffffff0)));
      const int back = length - (j.q1 - j.q0);
      j.pos0 = back + (j.t0 - j.q0);
      const int last = back + min(j.q1, j.t0 + per) - 1 - j.q0;
      j.keys = clampi(last + 1, 0, min(length, cap));
      const int lo = w.a.window > 0 && j.pos0 + 1 > a.window ? static_cast<int>(j.pos0 + 1 - a.window) : 0;
      const int sinks = static_cast<int>(min(static_cast<int64_t>(min(lo, j.keys)), a.sinks));
      j.sink_tiles = (sinks + kTile - 1) / kTile;
      j.from = max(lo / w.granule * w.granule, j.sink_tiles * kTile);
      j.tiles = j.sink_tiles + max(0, (j.keys - j.from + kTile - 1) / kTile);
    } else {  // a CTA without a tile clears its share of the tokens that belong to no row
      j.t0 = end + want * per;
      j.tiles = 0;
    }
    if (lane == 0) job_s = j;
  }
  sm100::tc_fence_before_sync();
  __syncthreads();
  sm100::tc_fence_after_sync();
  const uint32_t tmem = *holder;
  const Job j = job_s;
  const int kvh = blockIdx.y, n = j.tiles;
  auto key_of_tile = [&](int i) { return i < j.sink_tiles ? i * kTile : j.from + (i - j.sink_tiles) * kTile; };

  if (n == 0) {
    const int end = j.row >= 0 ? min(j.q1, j.t0 + per) : min(total_tokens, j.t0 + per);
    const int count = max(0, end - j.t0) * w.share;
    for (int i = tid; i < count * a.dim; i += C::threads) {
      const int64_t at = static_cast<int64_t>(j.t0 + i / a.dim / w.share) * a.q_heads + kvh * w.share + i / a.dim % w.share;
      store1(static_cast<T *>(a.out) + at * a.dim + i % a.dim, 0.f);
      if (i % a.dim == 0 && a.lse) a.lse[at] = -INFINITY;
    }
  } else if (warp < 4) {
    if (NQ == 2) registers_down<72>();
    if (warp == 0) {
    // ---- loads: Q once, then K and V tiles through one ring.  Lane b takes box b.
    const int boxes = kTile / w.granule, mask = (1 << a.page_shift) - 1;
    if (lane == 0) {
      const int bytes = C::halves * 128 * w.share * w.tokens_per_tile;
      sm100::mbar_arrive_expect_tx(q_full, NQ * bytes);
      for (int t = 0; t < NQ; ++t)
        for (int h = 0; h < C::halves; ++h)
          tma_load_3d(q_sm + t * C::tile_bytes + h * kHalf, &qmap, h * 64, kvh * w.share,
                      j.t0 + t * w.tokens_per_tile, q_full);
    }
    const int *table = a.table + static_cast<int64_t>(j.row) * a.width;
    auto page_at = [&](int i) {  // lane b: the page of box b of tile i, -1 where there is none
      const int k = key_of_tile(i) + lane * w.granule;
      if (i >= n || lane >= boxes || k >= j.keys) return -1;
      const int p = table[k >> a.page_shift];
      return p >= 0 && p < a.pages ? p : -1;
    };
    int issued = 0;
    uint32_t landed_phase = 0;
    int next_page = page_at(0);
    bool ok = true;
    for (int i = 0; i < n && ok; ++i) {
      const int page = next_page;
      next_page = page_at(i + 1);
      const int k0 = key_of_tile(i), k = k0 + lane * w.granule;
      const uint32_t have = __ballot_sync(0xffffffffu, page >= 0);
      const int bytes = __popc(have) * w.granule * 128 * C::halves;
      if (__any_sync(0xffffffffu, page < 0 && lane < boxes && k < j.keys) && lane == 0) absent = 1;
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
            tma_load_4d(dst + h * kHalf + lane * w.granule * 128, kv ? &vmap : &kmap, h * 64, k & mask, kvh, page, bar);
        ++issued;
        if (clear) {
          ok = sm100::mbar_wait_warp(bar, (landed_phase >> s) & 1, w.wait_ns);
          landed_phase ^= 1u << s;
          for (int r = lane; r < kTile; r += 32) {
            const int p = __shfl_sync(0xffffffffu, page, r / w.granule);
            if (p < 0 || k0 + r >= j.keys)
              for (int h = 0; h < C::halves; ++h)
                for (int c = 0; c < 8; ++c)
                  asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(dst + h * kHalf + r * 128 + c * 16), "r"(0)
                               : "memory");
          }
          sm100::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) sm100::mbar_arrive(full(s));
        }
      }
      if (!ok) *w.error = 1;
    }
    // wind down: every load must have landed before the CTA exits
    if (lane == 0) {
      if (!sm100::mbar_wait_bounded(q_full, 0, kDrainNs)) *w.error = 1;
      for (int x = issued > S ? issued - S : 0; x < issued; ++x)
        if (!sm100::mbar_wait_bounded(full(x % S), (x / S) & 1, kDrainNs)) *w.error = 1;
    }
    } else if (warp == 1) {
    // ---- products
    if (lane == 0) {
      constexpr uint32_t id_s = idesc_of<T>(kTile, false), id_o = idesc_of<T>(DP, true);
      auto stage_of = [&](int x) { return ring + (x % S) * C::tile_bytes; };
      auto wait_tile = [&](int x) { return sm100::mbar_wait_bounded(full(x % S), (x / S) & 1, w.wait_ns); };
      auto scores = [&](int t, int x) {  // S of query tile t over the keys in ring place x
        const uint32_t qa = q_sm + t * C::tile_bytes, kb = stage_of(x);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const uint32_t off = (k / 4) * kHalf + (k % 4) * 32;
          sm100::umma_f16(tmem + t * kTile, sm100::sw128_kmajor_desc(qa + off), sm100::sw128_kmajor_desc(kb + off), id_s,
                          k != 0);
        }
        sm100::umma_commit(s_full(t));
      };
      bool ok = sm100::mbar_wait_bounded(q_full, 0, w.wait_ns) && wait_tile(0);
      if (ok) {
        sm100::tc_fence_after_sync();
        for (int t = 0; t < NQ; ++t) scores(t, 0);
        sm100::umma_commit(empty(0));
      }
      for (int i = 0; i < n && ok; ++i) {
        ok = wait_tile(2 * i + 1);
        for (int t = 0; t < NQ && ok; ++t) {
          ok = sm100::mbar_wait_bounded(p_full(t), i & 1, w.wait_ns);
          if (!ok) break;
          sm100::tc_fence_after_sync();
          const uint64_t vb = sw128_mnmajor_desc(stage_of(2 * i + 1));
#pragma unroll
          for (int k = 0; k < kTile / 16; ++k)
            umma_ts(tmem + NQ * kTile + t * DP, tmem + t * kTile + k * 8, vb + k * (16 * 128 >> 4), id_o, (i | k) != 0);
          if (i + 1 < n) {
            if (t == 0) ok = wait_tile(2 * i + 2);
            if (!ok) break;
            sm100::tc_fence_after_sync();
            scores(t, 2 * i + 2);
          } else {
            sm100::umma_commit(o_full(t));
          }
        }
        if (!ok) break;
        sm100::umma_commit(empty((2 * i + 1) % S));
        if (i + 1 < n) sm100::umma_commit(empty((2 * i + 2) % S));
      }
      if (!ok) *w.error = 1;
      sm100::umma_commit(drain);
      if (!sm100::mbar_wait_bounded(drain, 0, kDrainNs)) *w.error = 1;
    }
    }
  } else {
    if (NQ == 2) registers_up<216>();
    // ---- softmax: one thread per query row
    const int t = (warp - 4) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_at = tmem + lanes + t * kTile, o_at = tmem + lanes + NQ * kTile + t * DP;
    const int tok = r / w.share, token = j.t0 + t * w.tokens_per_tile + tok;
    const bool real = tok < w.tokens_per_tile && token < j.q1;
    const int pos = j.pos0 + t * w.tokens_per_tile + tok;
    // keys seen: k <= pos, and k > pos - window or k < sinks
    const int pos_first = j.pos0 + t * w.tokens_per_tile, pos_last = pos_first + w.tokens_per_tile - 1;
    const int64_t win = a.window > 0 ? a.window : (int64_t(1) << 40);
    const int low = static_cast<int>(max(static_cast<int64_t>(-1), pos - win));  // keys above it are recent
    const int64_t low_last = pos_last - win;
    const int sinks = static_cast<int>(min(a.sinks, static_cast<int64_t>(0x7fffffff)));
    const float scale2 = a.scale * kLog2e;
    float m = -INFINITY, l = 0.f;  // m in the units of S
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      ok = sm100::mbar_wait_warp(s_full(t), i & 1, w.wait_ns);
      if (!ok) break;
      sm100::tc_fence_after_sync();
      uint32_t raw[kTile];
#pragma unroll
      for (int c = 0; c < kTile; c += 32) tmem_ld_32(s_at + c, raw + c);
      sm100::tmem_ld_wait();
      float *s = reinterpret_cast<float *>(raw);
      const int k0 = key_of_tile(i);
      const bool plain = k0 + kTile - 1 <= pos_first && (k0 > low_last || k0 + kTile <= sinks) && k0 + kTile <= j.keys;
      const bool gaps = absent != 0;
      if (!plain || gaps) {
#pragma unroll
        for (int c = 0; c < kTile; ++c) {
          const int k = k0 + c;
          if (!(k <= pos && (k > low || k < sinks))) s[c] = -INFINITY;
        }
        if (gaps) {
          const int *table = a.table + static_cast<int64_t>(j.row) * a.width;
          for (int b = 0; b < kTile / w.granule; ++b) {
            const int k = k0 + b * w.granule;
            const int p = k < j.keys ? table[k >> a.page_shift] : 0;
            if (p < 0 || p >= a.pages) {
#pragma unroll
              for (int c = 0; c < kTile; ++c)
                if (c / w.granule == b) s[c] = -INFINITY;
            }
          }
        }
      }
      float tops[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int c = 4; c < kTile; c += 8)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          tops[x] = fmaxf(fmaxf(tops[x], s[c + x]), c + 4 + x < kTile ? s[c + 4 + x] : s[c + x]);
      const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
      const float grown = (top - m) * scale2;
      const bool renew = m == -INFINITY ? top != -INFINITY : grown > 8.f;
      if (__any_sync(0xffffffffu, renew)) {
        const float mn = renew ? fmaxf(m, top) : m;
        const float f = m == mn ? 1.f : ex2((m - mn) * scale2);
        if (i > 0) {
#pragma unroll
          for (int c = 0; c < DP; c += 32) {
            uint32_t o[32];
            tmem_ld_32(o_at + c, o);
            sm100::tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
            tmem_st_32(o_at + c, o);
          }
        }
        l *= f;
        m = mn;
      }
      const float mb = m == -INFINITY ? 0.f : m * scale2;
      const uint64_t scale_2 = pack2(scale2, scale2), mb_2 = pack2(-mb, -mb);
      uint64_t sums[2] = {0, 0};
#pragma unroll
      for (int c = 0; c < kTile; c += 32) {
#pragma unroll
        for (int x = 0; x < 32; x += 2) {
          const float2 e = unpack2(fma2(pack2(s[c + x], s[c + x + 1]), scale_2, mb_2));
          const float p0 = ex2(e.x), p1 = ex2(e.y);
          sums[(x >> 1) & 1] = add2(sums[(x >> 1) & 1], pack2(p0, p1));
          split16<T>(p0, p1, raw[(c + x) / 2]);
        }
        tmem_st_16(s_at + c / 2, raw + c / 2);
      }
      const float2 sum = unpack2(add2(sums[0], sums[1]));
      l += sum.x + sum.y;
      tmem_st_wait();
      sm100::tc_fence_before_sync();
      sm100::mbar_arrive(p_full(t));
    }
    if (ok && sm100::mbar_wait_warp(o_full(t), 0, w.wait_ns)) {
      sm100::tc_fence_after_sync();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int64_t at = static_cast<int64_t>(token) * a.q_heads + kvh * w.share + r % w.share;
      T *out = static_cast<T *>(a.out) + at * a.dim;
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
        uint32_t o[32];
        tmem_ld_32(o_at + c, o);
        sm100::tmem_ld_wait();
        if (real) {
#pragma unroll
          for (int x = 0; x < 32; x += 8) {
            if (c + x >= a.dim) continue;
            uint32_t p[4];
#pragma unroll
            for (int y = 0; y < 4; ++y)
              split16<T>(__uint_as_float(o[x + 2 * y]) * inv, __uint_as_float(o[x + 2 * y + 1]) * inv, p[y]);
            *reinterpret_cast<uint4 *>(out + c + x) = make_uint4(p[0], p[1], p[2], p[3]);
          }
        }
      }
      if (real && a.lse) a.lse[at] = l == 0.f ? -INFINITY : (m == -INFINITY ? 0.f : m * scale2 * kLn2) + logf(l);
    } else {
      *w.error = 1;
    }
  }
  sm100::tc_fence_before_sync();
  __syncthreads();
  sm100::tc_fence_after_sync();
  if (warp == 1) sm100::tmem_dealloc(tmem, C::tmem_cols);
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
  static const cudaError_t attr = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::smem);
  if (attr != cudaSuccess) return fail(QS_ERR_CUDA, "attention (window): %s", cudaGetErrorString(attr));
  const int64_t per = static_cast<int64_t>(NQ) * w.tokens_per_tile;
  const dim3 grid(static_cast<unsigned>(ceil_div(a.tokens, per) + a.rows), a.kv_heads);
  return launch_pdl("attention (window)", kern, grid, dim3(C::threads), C::smem, s, qmap, kmap, vmap, w);
}

}  // namespace

int64_t attn_window_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

int launch_attn_window(const AttnArgs &a, cudaStream_t s) {
  if (a.dim <= 64) return a.dtype == QS_F16 ? run<__half, 64, 2>(a, s) : run<__nv_bfloat16, 64, 2>(a, s);
  return a.dtype == QS_F16 ? run<__half, 128, 2>(a, s) : run<__nv_bfloat16, 128, 2>(a, s);
}

}  // namespace qs
