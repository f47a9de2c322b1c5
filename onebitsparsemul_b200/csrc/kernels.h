// Launchers of the CUDA kernels behind the C ABI (internal header).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace ob {

// Multiprocessors of the current device (cached per device; the dispatchers size their grids by it).
int sm_count();

// K1 (pack.cu)
// apply_mask (fp16 only): the 2:4 magnitude mask is applied in the same pass; masked (nullable) receives the masked weights
cudaError_t launch_pack(const void* dense, int dense_dtype, int64_t m, int64_t k, void* sparse,
                        void* bits_ref, void* meta_ref, int dialect, void* bits_tile, void* meta_tile,
                        bool apply_mask, void* masked, cudaStream_t stream);
// 2:4 magnitude mask (mask.cu)
cudaError_t launch_mask24(const void* dense_f16, int64_t count, void* masked_f16, void* mask_u8,
                          cudaStream_t stream);
// K4 (relayout.cu)
cudaError_t launch_relayout(const void* bits_ref, const void* meta_ref, int dialect, int64_t m, int64_t k,
                            void* bits_tile, void* meta_tile, cudaStream_t stream);
cudaError_t launch_tile_to_dense(const void* bits_tile, const void* meta_tile, const void* scale, int64_t m,
                                 int64_t k, void* dense, cudaStream_t stream);
// plain one-thread-per-output kernel on the reference orders (gemm_simple.cu)
cudaError_t launch_gemm_simple(const void* bits_ref, const void* meta_ref, int dialect, const void* scale,
                               const void* b, void* d, int64_t m, int64_t n, int64_t k, int out_type,
                               cudaStream_t stream);
// K3: decode kernel, n small (gemm_decode.cu). tile-ordered operands. fresh_weights: the weight buffers were
// written by the kernel launched just before on the same stream (the kernel then loads nothing before that one is done).
cudaError_t launch_gemm_decode(const void* bits_tile, const void* meta_tile, const void* scale, const void* b,
                               void* d, int64_t m, int64_t n, int64_t k, int out_type, bool fresh_weights,
                               cudaStream_t stream);
// K2: tcgen05 kernel (gemm_prefill_sm100.cu). tile-ordered operands; n % 8 == 0.
// status: device word that receives a non-zero code if a bounded wait inside the kernel gave up.
cudaError_t launch_gemm_prefill(const void* bits_tile, const void* meta_tile, const void* scale, const void* b,
                                void* d, int64_t m, int64_t n, int64_t k, int out_type, int* status,
                                cudaStream_t stream);
bool prefill_supported(int64_t m, int64_t n, int64_t k);
// token-major forms (x (n, k), y (n, m), optional bias (m)): the nn.Linear convention
cudaError_t launch_gemm_prefill_tokens(const void* bits_tile, const void* meta_tile, const void* scale, const void* bias,
                                       const void* x, void* y, int64_t m, int64_t n, int64_t k, int out_type, int* status,
                                       cudaStream_t stream);
bool prefill_tokens_supported(int64_t m, int64_t n, int64_t k);
// K2 persistent pair kernel with several destinations: the fp16 result goes to d and to n_extra (<= 7) more
// buffers of the same shape (any address this device can store to, e.g. peer GPUs' memory).
cudaError_t launch_gemm_prefill_scatter(const void* bits_tile, const void* meta_tile, const void* scale, const void* b,
                                        void* d, void* const* extra_dst, int n_extra, int64_t m, int64_t n, int64_t k,
                                        int* status, cudaStream_t stream);
bool prefill_scatter_supported(int64_t m, int64_t n, int64_t k, const void* d);
cudaError_t launch_gemm_decode_tokens(const void* bits_tile, const void* meta_tile, const void* scale, const void* bias,
                                      const void* x, void* y, int64_t m, int64_t n, int64_t k, int out_type,
                                      bool fresh_weights, cudaStream_t stream);
// Reads and clears the decode kernel's bounded-wait status on the current device (0 = nothing gave up).
cudaError_t read_decode_status(int* out);
// K3, tensor-memory form (gemm_decode_sm100.cu): the few-token kernel on tcgen05.mma.sp with a 128 x 16 accumulator.
// Same operands as the two launchers above; token_major selects x (n, k) / y (n, m).
cudaError_t launch_gemm_fewtok(const void* bits_tile, const void* meta_tile, const void* scale, const void* bias,
                               const void* b, void* d, int64_t m, int64_t n, int64_t k, int out_type, bool token_major,
                               bool fresh_weights, cudaStream_t stream);
cudaError_t read_fewtok_status(int* out);

// ---- the operators between the linear layers of a decoder block ----
// residual add and norms (norm.cu); strides in elements from row to row, gate_stride 0 = one gate row for all rows
cudaError_t launch_residual_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, bool residual_f32,
                                 const void* gate, int64_t gate_stride, const void* post_weight, const void* weight, void* y,
                                 int64_t y_stride, void* h, int64_t h_stride, int64_t rows, int64_t hidden, float residual_scale,
                                 float eps, bool bf16, cudaStream_t stream);
// rotary positions and cache append (rotary_append.cu); _ts / _hs: elements from one token / head to the next
cudaError_t launch_rotary(const void* x, int64_t x_ts, int64_t x_hs, void* y, int64_t y_ts, int64_t y_hs, const void* positions,
                          bool positions_i64, const double* inv_freq, int rotary_dim, bool interleaved, float magnitude, int64_t tokens,
                          int64_t heads, int64_t head_dim, bool bf16, cudaStream_t stream);
struct CacheAppendCall {
  const void *k, *v, *q;
  void* q_out;
  int64_t k_ts, k_hs, v_ts, v_hs, q_ts, q_hs, qo_ts, qo_hs;
  const double* inv_freq;
  int rotary_dim;              // 0: nothing is turned
  bool interleaved;
  float magnitude;
  void *k_pages, *v_pages;
  float *k_scale, *v_scale;
  int64_t pages;
  const int *q_start, *kv_len, *table;
  int64_t table_stride, table_width, tokens, seqs, heads, kv_heads, head_dim;
  bool bf16;
  int64_t max_new;             // the caller's bound of a sequence's new tokens: it picks the kernels, results are right whatever it is
};
cudaError_t launch_cache_append(const CacheAppendCall& c, cudaStream_t stream);
cudaError_t read_append_status(int* batch);           // the readers clear the words
// attention over the cache (cache_attend.cu)
struct CacheAttendCall {
  const void* q;
  void* out;
  int64_t q_ts, q_hs, o_ts, o_hs;
  const void *k_pages, *v_pages;
  const float *k_scale, *v_scale;
  int64_t pages;
  const int *q_start, *kv_len, *table;
  int64_t table_stride, table_width, tokens, seqs, heads, kv_heads, head_dim;
  int64_t max_new;             // the caller's bound of a sequence's new tokens: it picks the kernel, results are right whatever it is
  float scale;
  bool causal, bf16;
  int few_rows;                // sequences with at most this many query rows per cache head are one kernel's, the others the other's
};
int64_t cache_attend_workspace(const CacheAttendCall& c);
cudaError_t launch_cache_attend(const CacheAttendCall& c, void* workspace, cudaStream_t stream);
cudaError_t read_attend_status(int* wait, int* batch);
cudaError_t read_attend_many_status(int* wait, int* batch);

}  // namespace ob
