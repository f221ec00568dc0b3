// Internal launchers shared between the translation units of the library.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/quipsharp_b200.h"

struct CUtensorMap_st;  // CUtensorMap (cuda.h)

namespace qs {

// qs_decode.cu
int launch_decode(int kind, const void *codes, int code_dtype, int64_t count, float *out,
                  cudaStream_t s);
int launch_rvq_decode(int stages, const int *kinds, const void *const *codes, int code_dtype,
                      const float *stage_scales, int64_t count, float *out, cudaStream_t s);
int launch_dequantize_linear(const int16_t *codes, int stages, const int *kinds,
                             const float *stage_scales, const float *layer_scale, int64_t m,
                             int64_t n, float *out, cudaStream_t s);

// qs_transform.cu
int launch_fwht(const void *x, int64_t ld_x, void *y, int64_t ld_y, int dtype, int64_t rows,
                int64_t n, const float *pre, const float *post, cudaStream_t s);
int launch_rfft(int inverse, const void *x, int64_t ld_x, void *y, int64_t ld_y, int dtype,
                int64_t rows, int64_t n, const void *phase, cudaStream_t s);
int64_t linear_input_bytes(int64_t batch, int64_t n);
int launch_linear_input(const void *x, int x_dtype, int64_t batch, int64_t n, int transform,
                        const float *sv, const void *phase_v, void *x2ws, float *y1,
                        int64_t m_local, cudaStream_t s);
struct XPeerGather;
struct TpPush;
int launch_linear_output(float *y1, int64_t ld_y1, int64_t shards, int64_t batch, int64_t m,
                         int transform, const float *su, const void *phase_u, const float *bias,
                         void *y, int y_dtype, cudaStream_t s, const XPeerGather *pg = nullptr);
int check_fft_size(int64_t n_complex);
int check_fwht_size(int64_t n);

// qs_xform2.cu: two-pass RFFT of the linear input / output steps
bool two_pass_rfft(int64_t n_complex, int64_t rows, int *P, int *lgN1);
int64_t two_pass_input_scratch_bytes(int64_t batch, int64_t n);
int launch_two_pass_input(const void *x, int dtype, int64_t batch, int64_t n, const float2 *phase, float scale,
                          __half *x2h, float *rowscale, int n_pad, void *scratch, float *y1, int64_t m_local,
                          cudaStream_t s);
int launch_two_pass_output(float *y1, int64_t batch, int64_t m, const float2 *phase, const float *bias, float scale,
                           void *y, int dtype, cudaStream_t s);

// qs_xsmall.cu: decode-batch FWHT row kernels of the linear input / output steps
constexpr int64_t kSmallRhtMaxRows = 32;
bool small_rht_ok(int64_t n, int64_t rows);
int launch_small_input_rht(const void *x, int dtype, int64_t rows, int64_t n, const float *sv, float scale,
                           __half *x2h, float *rowscale, int n_pad, float *y1, int64_t m_local, cudaStream_t s);
int launch_small_output_rht(const float *y1, int64_t ld_y1, int64_t shards, int64_t batch, int64_t m,
                            const float *su, const float *bias, float scale, void *y, int y_dtype,
                            const XPeerGather *pg, cudaStream_t s);
bool small_rfft_ok(int64_t n_complex, int64_t rows);
int launch_small_input_rfft(const void *x, int dtype, int64_t rows, int64_t n, const float2 *phase, float scale,
                            __half *x2h, float *rowscale, int n_pad, float *y1, int64_t m_local, cudaStream_t s);
int launch_small_output_rfft(const float *y1, int64_t ld_y1, int64_t shards, int64_t batch, int64_t m,
                             const float2 *phase, const float *bias, float scale, void *y, int y_dtype,
                             const XPeerGather *pg, cudaStream_t s);

// qs_fit.cu: stage-scale sweeps of RVQ codebook construction
constexpr int kFitMaxStages = 2;
constexpr int kFitMaxCandidates = 128;
int64_t fit_workspace_bytes(int64_t samples, int ncand);
int launch_fit_sweep(const float *x, int64_t samples, int nprev, const int *prev_kinds, const float *prev_scales,
                     int rvq, int nst, const int *kinds, const float *stage_scales, const float *candidates,
                     int ncand, void *workspace, double *mse, int *best, cudaStream_t s);

// qs_tp.cu: column-sharded tensor parallelism over peer memory
int ipc_export(const void *ptr, void *handle, int64_t *offset);
int ipc_import(const void *handle, int64_t offset, void **ptr);
int ipc_close(void *ptr, int64_t offset);
int64_t tp_workspace_bytes(int64_t batch, int64_t n, int64_t m_local);
int launch_tp_push(const qs_tp_peers *pe, const float *y1, int64_t batch, int64_t m_local, cudaStream_t s);
int launch_matmul_tp(const void *x2ws, int64_t batch, int64_t n, int64_t m_local, const void *packed, int stages,
                     const int *kinds, const float *stage_scales, const float *layer_scale, float *y1,
                     const qs_tp_peers *pe, cudaStream_t s);
int launch_output_peers(const qs_tp_peers *pe, int64_t batch, int64_t m, int transform, const float *su,
                        const void *phase_u, const float *bias, void *y, int y_dtype, cudaStream_t s);
int launch_linear_fwd_tp(const void *x, int x_dtype, int64_t batch, int64_t n, int64_t m, const void *packed,
                         int stages, const int *kinds, const float *stage_scales, const float *layer_scale,
                         int transform, const float *su, const float *sv, const void *phase_u, const void *phase_v,
                         const float *bias, void *y, void *workspace, const qs_tp_peers *pe, cudaStream_t s);

// qs_pack.cu
int launch_pack(const int16_t *codes, int stages, const int *kinds, int64_t m, int64_t n,
                void *packed, cudaStream_t s);

// qs_gemv.cu: fused decode + matmul; batches below kTcMinBatch run the
// decode-regime kernel of this file, larger ones launch_matmul_tc.  push
// (decode batches only): after a grid barrier the CTAs push y1 to every rank.
int launch_matmul(const void *x2ws, int64_t batch, int64_t n, int64_t m, const void *packed,
                  int stages, const int *kinds, const float *stage_scales,
                  const float *layer_scale, float *y1, cudaStream_t s, const TpPush *push = nullptr);

// qs_gemm_tc.cu
int launch_matmul_tc(const void *x2ws, int64_t batch, int64_t n, int64_t m, const void *packed, int stages,
                     const int *kinds, const float *stage_scales, const float *layer_scale, float *y1,
                     cudaStream_t s);
int device_status(cudaStream_t s);
// Device address (current device) of the error flag qs_device_status reports.
int *device_error_flag();
// 2-D tensor map over fp16 rows (rows x n_pad, row stride n_pad elements) with
// a box of box_x elements x box_y rows; 128-byte swizzle or none.
int encode_fp16_rows_map(::CUtensorMap_st *map, const void *x2h, int64_t n_pad, int64_t rows, int box_x, int box_y,
                         bool swizzle128);
// Tensor map over 16-bit values, up to 5 dimensions (innermost first; strides in
// elements of all but the innermost), 128-byte swizzle, zeros outside.
int encode_16bit_map(::CUtensorMap_st *map, const void *base, bool bf16, int rank, const int64_t *dims,
                     const int64_t *strides, const int *box);
// Limit (ns) of every bounded wait between the warps of a pipelined kernel
// (mbarrier waits); a wait that runs out sets the device error flag.  Drains of
// a CTA's own asynchronous copies and tensor-core work keep a fixed 4 s limit.
constexpr uint64_t kDefaultWaitNs = 4000000000ull;
uint64_t pipeline_wait_ns();
void set_pipeline_wait_ns(uint64_t ns);
// Batches of at least this many tokens use the tcgen05 GEMM (128 x 256 tiles,
// decoded weights in shared memory); smaller ones the mma.sync decode-regime
// kernel (weights decoded in registers, passes of 8 or 16 tokens).
constexpr int64_t kTcMinBatch = 33;

// qs_cache.cu: pages of a key-value cache
constexpr int kCacheErrPages = 1;   // a row found no free page, or outgrew its table row
constexpr int kCacheErrParent = 2;  // a parent outside [-1, rows), or a negative token count
constexpr int kCacheMaxRows = 8192;
int64_t cache_workspace_bytes(int64_t rows, int64_t pages);
int launch_cache_fork(const qs_kv_pool &pool, int rows, int width, const int *table, const int *lengths,
                      const int *refcount, const int *parents, int *table_out, int *lengths_out, int *refcount_out,
                      void *ws, cudaStream_t s);
int launch_cache_compact(const qs_kv_pool &pool, int rows, int width, const int *table, const int *lengths,
                         const int *refcount, int *table_out, int *refcount_out, int *used_out, void *ws,
                         cudaStream_t s);
int launch_cache_extend(int64_t page, int64_t pages, int rows, int width, const int *table, const int *lengths,
                        const int *refcount, const int *add, int *table_out, int *lengths_out, int *refcount_out,
                        void *ws, cudaStream_t s);
int launch_cache_write(const qs_kv_pool &pool, int rows, int width, const int *table, const int *lengths,
                       const int *cu, const void *k, int64_t k_token, int64_t k_head, const void *v, int64_t v_token,
                       int64_t v_head, int64_t tokens, cudaStream_t s);
// Reads and clears one of the kCacheErr bits raised on the device (synchronises s).
int take_cache_error(int *bit, cudaStream_t s);
int device_sms();  // of the current device

// Arguments of attention over one layer of the cache (strides in elements).
struct AttnArgs {
  const void *q;
  int64_t q_token, q_head;
  const void *k, *v;
  int64_t ks[3], vs[3];  // page, head, token
  int dtype, dim, q_heads, kv_heads, pages, page_shift;
  int rows, width;
  int64_t tokens;
  const int *table, *lengths, *cu;
  float scale;
  int64_t window, sinks;  // window 0: none
  void *out;
  float *lse;
  void *ws;
};
// qs_attn_decode.cu
int64_t attn_decode_workspace_bytes(int64_t rows, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t page,
                                    int64_t width, int64_t window, int64_t sinks);
int launch_attn_decode(const AttnArgs &a, cudaStream_t s);
// qs_attn_window.cu
int64_t attn_window_workspace_bytes(int64_t tokens, int64_t rows, int64_t q_heads, int64_t kv_heads, int64_t dim,
                                    int64_t page, int64_t width, int64_t window, int64_t sinks);
int launch_attn_window(const AttnArgs &a, cudaStream_t s);

// qs_beam.cu
constexpr int kBeamMaxN = 64;
constexpr int kBeamMaxBeams = 64;
int64_t beam_workspace_bytes(int64_t batch, int64_t beams, int64_t vocab, int64_t n);
int launch_beam_select(const void *logits, int dtype, int64_t batch_stride, int64_t beam_stride, int64_t batch,
                       int64_t beams, int64_t vocab, const float *scores, const uint8_t *finished, int n, int pad,
                       float *scores_out, int *parents_out, int *tokens_out, void *ws, cudaStream_t s);

}  // namespace qs
