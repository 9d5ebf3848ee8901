/*
 * neso_b200.h — C ABI of the Neso B200 kernel library (sm_100a).
 *
 * Every kernel that Neso compiles and benchmarks is exported here under the
 * reference kernel's name, with the reference's arguments in the reference's
 * order. The rule that turns a reference launch into a call is uniform:
 *
 *   neso_<kernel>(<runtime args in reference order>,
 *                 <the reference kernel's constexpr parameters, as int32>,
 *                 grid_x, grid_y, grid_z,      // the reference launch grid
 *                 stream)                      // cudaStream_t, NULL = legacy
 *
 * The reference grid is validated against the problem it implies (a mismatch
 * returns NESO_ERR_GRID); the kernels then launch their own B200 grid. The
 * caller owns every buffer; pointers are device pointers. All calls are
 * asynchronous on `stream`, thread-safe and never abort: they return a status
 * code, and neso_last_error_string() gives the thread's last message.
 *
 * Extended entry points (neso_fa2_*, neso_*_mnk, neso_w4a16_*) cover the
 * multi-head, causal, relative-position-table and packed-int4 variants that
 * have no reference kernel; each says so.
 */
#ifndef NESO_B200_H
#define NESO_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define NESO_API __attribute__((visibility("default")))
#else
#define NESO_API
#endif

/* A CUDA stream (cudaStream_t / CUstream). NULL selects the legacy stream. */
typedef void* neso_stream_t;

/* Status codes. The reference raises RuntimeError on Metal pipeline/command
 * buffer failures (src/neso/backend/driver.py:138-176, :314-317); these are the
 * C equivalents. */
#define NESO_OK 0
#define NESO_ERR_INVALID_ARG (-1)    /* null pointer, negative size, bad constexpr */
#define NESO_ERR_MISALIGNED (-2)     /* pointer/stride alignment the kernel needs */
#define NESO_ERR_UNSUPPORTED (-3)    /* shape or layout this kernel does not implement */
#define NESO_ERR_GRID (-4)           /* reference grid inconsistent with the problem */
#define NESO_ERR_LAUNCH (-5)         /* CUDA runtime / driver error */
#define NESO_ERR_DEVICE_TIMEOUT (-6) /* a bounded device-side wait expired */
#define NESO_ERR_NO_DEVICE (-7)

/* Element types of the entry points that take more than one. */
#define NESO_F16 0
#define NESO_BF16 1
#define NESO_F32 2

/* ------------------------------------------------------------- runtime -- */
NESO_API const char* neso_last_error_string(void);
NESO_API int neso_version(void);
/* Select the CUDA device used by subsequent calls from this thread. */
NESO_API int neso_set_device(int device);
/* Synchronise `device` and read its status word: *code is 0 when no device
 * wait has timed out since the last neso_clear_device_status(). Returns
 * NESO_ERR_DEVICE_TIMEOUT when *code is non-zero. `where`, `block`, `thread`
 * (any may be NULL) locate the first failing wait. */
NESO_API int neso_device_status(int device, int* code, int* where, int* block, int* thread);
NESO_API int neso_clear_device_status(int device);
/* Self-test of the bounded-wait machinery: launches one CTA that waits on an
 * mbarrier nothing arrives at, with a budget of `budget_us` microseconds, and
 * returns the status the kernel reported (NESO_ERR_DEVICE_TIMEOUT expected). */
NESO_API int neso_selftest_wait_timeout(int budget_us, neso_stream_t stream);
/* JSON launch metadata for a kernel name, same keys as the reference's
 * AOTResult.to_metadata() (src/neso/aot_compile.py:108-117). NULL if unknown. */
NESO_API const char* neso_kernel_metadata(const char* kernel_name);

/* ---------------------------------------------------------- elementwise -- */
/* windows/kernels.py:7-15  vector_add(x, y, output, n_elements, BLOCK_SIZE)
 * (== tests/test_aot.py:17-28 add_kernel). Reference grid: (cdiv(n, BLOCK_SIZE), 1, 1).
 * fp32; output[i] = x[i] + y[i] for i < n_elements. */
NESO_API int neso_vector_add(const float* x, const float* y, float* output, int32_t n_elements, int32_t BLOCK_SIZE,
                    uint32_t grid_x, uint32_t grid_y, uint32_t grid_z, neso_stream_t stream);
/* tests/test_aot.py:17-28 add_kernel(x_ptr, y_ptr, z_ptr, n_elements, BLOCK_SIZE). */
NESO_API int neso_add_kernel(const float* x_ptr, const float* y_ptr, float* z_ptr, int32_t n_elements, int32_t BLOCK_SIZE,
                    uint32_t grid_x, uint32_t grid_y, uint32_t grid_z, neso_stream_t stream);
/* windows/kernels.py:18-22  scale(x, output, factor, n_elements, BLOCK_SIZE).
 * output[i] = x[i] * factor. */
NESO_API int neso_scale(const float* x, float* output, float factor, int32_t n_elements, int32_t BLOCK_SIZE,
               uint32_t grid_x, uint32_t grid_y, uint32_t grid_z, neso_stream_t stream);

/* ----------------------------------------- LLM building blocks (rowops) -- */
/* tests/test_advanced12.py:104-120  rmsnorm_kernel(x_ptr, weight_ptr, out_ptr,
 *   row_stride, n_cols, eps, BLOCK_SIZE). Reference grid: (M, 1, 1), one row per
 *   program: out = x / sqrt(sum(x^2) / n_cols + eps) * w over the first
 *   min(BLOCK_SIZE, n_cols) columns of each row. fp32. */
NESO_API int neso_rmsnorm_kernel(const float* x_ptr, const float* weight_ptr, float* out_ptr, int32_t row_stride,
                        int32_t n_cols, float eps, int32_t BLOCK_SIZE, uint32_t grid_x, uint32_t grid_y,
                        uint32_t grid_z, neso_stream_t stream);
/* tests/test_advanced12.py:135-153  residual_rmsnorm_kernel(x_ptr, residual_ptr,
 *   weight_ptr, out_ptr, row_stride, n_cols, eps, BLOCK_SIZE): RMSNorm of
 *   h = x + residual. Reference grid: (M, 1, 1). */
NESO_API int neso_residual_rmsnorm_kernel(const float* x_ptr, const float* residual_ptr, const float* weight_ptr,
                                 float* out_ptr, int32_t row_stride, int32_t n_cols, float eps, int32_t BLOCK_SIZE,
                                 uint32_t grid_x, uint32_t grid_y, uint32_t grid_z, neso_stream_t stream);
/* tests/test_advanced12.py:156-176  rope_kernel(x_ptr, cos_ptr, sin_ptr, out_ptr,
 *   seq_len, head_dim, BLOCK_D). x, out [seq_len, head_dim], cos/sin
 *   [seq_len, head_dim/2]; rotates pairs (d, d + head_dim/2) for
 *   d < min(BLOCK_D, head_dim/2). Reference grid: (seq_len, 1, 1). */
NESO_API int neso_rope_kernel(const float* x_ptr, const float* cos_ptr, const float* sin_ptr, float* out_ptr,
                     int32_t seq_len, int32_t head_dim, int32_t BLOCK_D, uint32_t grid_x, uint32_t grid_y,
                     uint32_t grid_z, neso_stream_t stream);
/* tests/test_advanced12.py:123-132  silu_kernel(x_ptr, out_ptr, n, BLOCK):
 *   out = x * sigmoid(x). Reference grid: (cdiv(n, BLOCK), 1, 1). */
NESO_API int neso_silu_kernel(const float* x_ptr, float* out_ptr, int32_t n, int32_t BLOCK, uint32_t grid_x,
                     uint32_t grid_y, uint32_t grid_z, neso_stream_t stream);
/* tests/test_triton_jit.py:55-70  softmax_kernel(output_ptr, input_ptr,
 *   input_row_stride, output_row_stride, n_cols, BLOCK_SIZE): row-wise softmax
 *   over the first min(BLOCK_SIZE, n_cols) columns. Reference grid: (M, 1, 1). */
NESO_API int neso_softmax_kernel(float* output_ptr, const float* input_ptr, int32_t input_row_stride,
                        int32_t output_row_stride, int32_t n_cols, int32_t BLOCK_SIZE, uint32_t grid_x,
                        uint32_t grid_y, uint32_t grid_z, neso_stream_t stream);
/* tests/test_advanced12.py:54-67  per_channel_dequant_kernel(x_int8_ptr,
 *   scale_ptr, zero_ptr, out_ptr, n_rows, n_cols, BLOCK_M, BLOCK_N):
 *   out = (x - zero[col]) * scale[col]; x held as int32 (the reference test
 *   passes int32, :222). Reference grid: (cdiv(n_rows, BLOCK_M), cdiv(n_cols, BLOCK_N), 1). */
NESO_API int neso_per_channel_dequant_kernel(const int32_t* x_int8_ptr, const float* scale_ptr, const float* zero_ptr,
                                    float* out_ptr, int32_t n_rows, int32_t n_cols, int32_t BLOCK_M, int32_t BLOCK_N,
                                    uint32_t grid_x, uint32_t grid_y, uint32_t grid_z, neso_stream_t stream);
/* tests/test_advanced12.py:69-84  grouped_dequant_kernel(x_int8_ptr, scale_ptr,
 *   zero_ptr, out_ptr, n, group_size, BLOCK): out[i] = (x[i] - zero[i / gs]) *
 *   scale[i / gs]; x held as int32. Reference grid: (cdiv(n, BLOCK), 1, 1). */
NESO_API int neso_grouped_dequant_kernel(const int32_t* x_int8_ptr, const float* scale_ptr, const float* zero_ptr,
                                float* out_ptr, int32_t n, int32_t group_size, int32_t BLOCK, uint32_t grid_x,
                                uint32_t grid_y, uint32_t grid_z, neso_stream_t stream);
/* tests/test_advanced12.py:87-101  quantize_kernel(x_ptr, scale_ptr, out_ptr, n,
 *   BLOCK): q = x / scale[0], rounded as q +/- 0.5 truncated toward zero,
 *   clamped to [-128, 127], stored as int32. Reference grid: (cdiv(n, BLOCK), 1, 1). */
NESO_API int neso_quantize_kernel(const float* x_ptr, const float* scale_ptr, int32_t* out_ptr, int32_t n, int32_t BLOCK,
                         uint32_t grid_x, uint32_t grid_y, uint32_t grid_z, neso_stream_t stream);

/* ------------------------------------------------------ flash attention -- */
/* tests/test_flash_attention.py:149-152
 *   flash_attention_fwd(Q, K, V, O, N, stride_qo, stride_kv, scale), constexpr d.
 * Single head. Q, K, V fp16 [N, d] with row strides stride_qo / stride_kv
 * (elements), O fp32 [N, d] with row stride stride_qo. HEAD_DIM = d in {64, 128}.
 * Reference grid: (N / BM, 1, 1) with the reference's BM (a power of two in
 * [8, 128]); N must be a multiple of that BM, as in the reference. */
NESO_API int neso_flash_attention_fwd(const void* Q, const void* K, const void* V, float* O, int32_t N, int32_t stride_qo,
                             int32_t stride_kv, float scale, int32_t HEAD_DIM, uint32_t grid_x, uint32_t grid_y,
                             uint32_t grid_z, neso_stream_t stream);

/* tests/test_rel_pos_fa2.py:157-162
 *   rel_pos_fa2_fwd(Q, K, V, bias, O, T, stride, scale, stride_h, bias_stride_h).
 * Multi-head; Q, K, V, bias and O are fp16. Q/K/V/O are [nh, T, d] (row stride
 * `stride`, head stride `stride_h`), bias is a dense [nh, T, T] table (head
 * stride bias_stride_h, row stride T); scores = (Q K^T + bias) * scale
 * (tests/test_rel_pos_fa2.py:202-206). Reference grid: (T / BM, nh, 1). */
NESO_API int neso_rel_pos_fa2_fwd(const void* Q, const void* K, const void* V, const void* bias, void* O, int32_t T,
                         int32_t stride, float scale, int32_t stride_h, int32_t bias_stride_h, int32_t HEAD_DIM,
                         uint32_t grid_x, uint32_t grid_y, uint32_t grid_z, neso_stream_t stream);

/* The hand-written MSL FA2 kernels of the reference's benchmarks:
 *   bench/bench_flash_attention.py:142-149      flash_attention_fwd
 *   bench/bench_flash_attention_opt.py:145-152  flash_attention_opt
 *   bench/bench_fa2_d128.py:116-123             flash_attention_d128
 * each (Q, K, V, O, N, d_head, scale) with Q, K, V, O single-head [N, d]
 * contiguous in one io_type: fp16 when use_half = 1, fp32 when use_half = 0.
 * Constexprs are the MSL generator's parameters (BM, BN, d, THREADS,
 * use_half); d_head must equal d (64 or 128; 128 for flash_attention_d128).
 * Reference grid: (N / BM, 1, 1) with N a multiple of BM; THREADS (1024 in
 * the reference) is accepted and ignored. fp32 operands are rounded to fp16
 * for the tensor cores (the stream's input workspace holds the copies); O is
 * written in io_type. The MSL flash_attention_fwd is exported with an _msl
 * suffix because the TTIR kernel of the same name is exported above. */
NESO_API int neso_flash_attention_fwd_msl(const void* Q, const void* K, const void* V, void* O, int32_t N,
                                          int32_t d_head, float scale, int32_t BM, int32_t BN, int32_t d,
                                          int32_t THREADS, int32_t use_half, uint32_t grid_x, uint32_t grid_y,
                                          uint32_t grid_z, neso_stream_t stream);
NESO_API int neso_flash_attention_opt(const void* Q, const void* K, const void* V, void* O, int32_t N, int32_t d_head,
                                      float scale, int32_t BM, int32_t BN, int32_t d, int32_t THREADS,
                                      int32_t use_half, uint32_t grid_x, uint32_t grid_y, uint32_t grid_z,
                                      neso_stream_t stream);
NESO_API int neso_flash_attention_d128(const void* Q, const void* K, const void* V, void* O, int32_t N,
                                       int32_t d_head, float scale, int32_t BM, int32_t BN, int32_t d,
                                       int32_t THREADS, int32_t use_half, uint32_t grid_x, uint32_t grid_y,
                                       uint32_t grid_z, neso_stream_t stream);

/* Extension (no reference kernel): multi-head FA2 forward over contiguous
 * [B, H, S, D] fp16 Q/K/V with fp32 O [B, H, S, D]. D in {64, 128}, any S >= 1.
 * causal != 0 masks keys j > i. */
NESO_API int neso_fa2_fwd(const void* Q, const void* K, const void* V, float* O, int32_t B, int32_t H, int32_t S, int32_t D,
                 float scale, int32_t causal, neso_stream_t stream);

/* Extension (no reference kernel; nearest is tests/test_rel_pos_fa2.py, whose
 * index is T-1-i+j on a dense table): logits s_ij = (q_i . k_j) * scale +
 * table[h, i - j + S - 1] with an fp32 table [H, 2S - 1]; fp32 O [B, H, S, D]. */
NESO_API int neso_fa2_fwd_relpos_table(const void* Q, const void* K, const void* V, const float* table, float* O, int32_t B,
                              int32_t H, int32_t S, int32_t D, float scale, int32_t causal, neso_stream_t stream);

/* --------------------------------------------------------------- matmul -- */
/* tests/test_aot.py:70-99 (tests/test_triton_jit.py:229-254 for the fp32-C form)
 *   matmul_kernel(a, b, c, M, N, K, stride_am, stride_ak, stride_bk, stride_bn,
 *                 stride_cm, stride_cn, BLOCK_M, BLOCK_N, BLOCK_K)
 * a fp16 [M, K], b fp16 [K, N], c fp32 [M, N]; fp32 accumulation. Unit inner
 * strides (stride_ak = stride_bn = stride_cn = 1), row strides multiples of 8.
 * Reference grid: (cdiv(M, BLOCK_M), cdiv(N, BLOCK_N), 1). */
NESO_API int neso_matmul_kernel(const void* a, const void* b, float* c, int32_t M, int32_t N, int32_t K, int32_t stride_am,
                       int32_t stride_ak, int32_t stride_bk, int32_t stride_bn, int32_t stride_cm, int32_t stride_cn,
                       int32_t BLOCK_M, int32_t BLOCK_N, int32_t BLOCK_K, uint32_t grid_x, uint32_t grid_y,
                       uint32_t grid_z, neso_stream_t stream);

/* bench/bench_matmul.py:79-81 (TTIR) / bench/bench_matmul_opt.py:129-139 (MSL)
 *   matmul_kernel(a, b, c, K, stride_am, stride_bk, stride_cm), constexpr BM, BN.
 * No M/N arguments: M = grid_x * BM, N = grid_y * BN (the reference has no masks). */
NESO_API int neso_matmul_tiled(const void* a, const void* b, float* c, int32_t K, int32_t stride_am, int32_t stride_bk,
                      int32_t stride_cm, int32_t BM, int32_t BN, uint32_t grid_x, uint32_t grid_y, uint32_t grid_z,
                      neso_stream_t stream);

/* ------------------------------------------------------ quantized matmul -- */
/* tests/test_quantized_matmul.py:67-167
 *   w8a16_matmul(A, B, C, K, stride_am, stride_bk, stride_cm), constexpr BM, BN, BK.
 * A fp16 [M, K], B int8 [K, N], C fp32 [M, N]; C = A . f16(B).
 * M = grid_x * BM, N = grid_y * BN (no masks in the reference). */
NESO_API int neso_w8a16_matmul(const void* A, const int8_t* B, float* C, int32_t K, int32_t stride_am, int32_t stride_bk,
                      int32_t stride_cm, int32_t BM, int32_t BN, int32_t BK, uint32_t grid_x, uint32_t grid_y,
                      uint32_t grid_z, neso_stream_t stream);

/* tests/test_quantized_matmul.py:181-283
 *   w8a16_scaled_matmul(A, B, C, scale, K, stride_am, stride_bk, stride_cm)
 * C[m, n] = (sum_k A[m, k] * B[k, n]) * f32(scale[n]); scale fp16 [N]. */
NESO_API int neso_w8a16_scaled_matmul(const void* A, const int8_t* B, float* C, const void* scale, int32_t K,
                             int32_t stride_am, int32_t stride_bk, int32_t stride_cm, int32_t BM, int32_t BN,
                             int32_t BK, uint32_t grid_x, uint32_t grid_y, uint32_t grid_z, neso_stream_t stream);

/* tests/test_advanced12.py:19-48
 *   w8a16_matmul_kernel(a_ptr, b_int8_ptr, c_ptr, scale_ptr, M, N, K,
 *                       stride_am, stride_ak, stride_bk, stride_bn,
 *                       stride_cm, stride_cn, BLOCK_M, BLOCK_N, BLOCK_K)
 * a fp16 [M, K], b int8 [K, N], c fp32 [M, N], scale_ptr one fp32 value:
 * c = (a . f16(b)) * scale_ptr[0], fp32 accumulation. Unit inner strides,
 * stride_am a multiple of 8, stride_bk a multiple of 16. Reference grid:
 * (cdiv(M, BLOCK_M), cdiv(N, BLOCK_N), 1). */
NESO_API int neso_w8a16_matmul_kernel(const void* a_ptr, const int8_t* b_int8_ptr, float* c_ptr,
                                      const float* scale_ptr, int32_t M, int32_t N, int32_t K, int32_t stride_am,
                                      int32_t stride_ak, int32_t stride_bk, int32_t stride_bn, int32_t stride_cm,
                                      int32_t stride_cn, int32_t BLOCK_M, int32_t BLOCK_N, int32_t BLOCK_K,
                                      uint32_t grid_x, uint32_t grid_y, uint32_t grid_z, neso_stream_t stream);
/* The same kernel with b held in an int32 tensor, as the reference's test
 * passes it (tests/test_advanced12.py:184-186): values in [-128, 127]
 * (others saturate), stride_bk in int32 elements, N a multiple of 16. The
 * weights are narrowed to int8 in the stream's input workspace first. */
NESO_API int neso_w8a16_matmul_kernel_i32(const void* a_ptr, const int32_t* b_int8_ptr, float* c_ptr,
                                          const float* scale_ptr, int32_t M, int32_t N, int32_t K, int32_t stride_am,
                                          int32_t stride_ak, int32_t stride_bk, int32_t stride_bn,
                                          int32_t stride_cm, int32_t stride_cn, int32_t BLOCK_M, int32_t BLOCK_N,
                                          int32_t BLOCK_K, uint32_t grid_x, uint32_t grid_y, uint32_t grid_z,
                                          neso_stream_t stream);

/* Extension with explicit sizes (any M >= 1): Y fp32 [M, N] = X fp16 [M, K] .
 * (W int8 [K, N] * scale fp16 [N]); scale may be NULL (unscaled W8A16).
 * Row-major, contiguous. N and K multiples of 16. */
NESO_API int neso_w8a16_matmul_mnk(const void* X, const int8_t* W, const void* scale, float* Y, int32_t M, int32_t N,
                          int32_t K, neso_stream_t stream);

/* Extension (no reference kernel; group semantics follow the grouped dequant
 * of tests/test_advanced12.py:69-84): packed int4, group 128, symmetric.
 * Wq uint8 [K/2, N]: byte (k/2, n) holds k even in bits 0-3 and k odd in bits
 * 4-7, two's-complement nibbles in [-8, 7]; scales fp16 [K/128, N].
 * Y fp32 [M, N] = sum_g scales[g, n] * sum_{k in g} X[m, k] * q[k, n].
 * K a multiple of 128, N a multiple of 16. */
NESO_API int neso_w4a16_g128_matmul(const void* X, const uint8_t* Wq, const void* scales, float* Y, int32_t M, int32_t N,
                           int32_t K, neso_stream_t stream);

/* No counterpart in the reference: an allocation-free form of
 * neso_w8a16_matmul_mnk for callers that cannot call cudaMalloc (for example
 * code running inside a host allocator callback, a pre-reserved memory pool
 * manager, or an environment whose device memory is fully budgeted before
 * launch). Same arguments and result (K = 0 writes zeros). It always runs the
 * tensor-core kernel (decode batches of M <= 4 do not take the GEMV path,
 * which keeps per-launch counters in allocated memory). Its split-K scratch is
 * a fixed array of 2^20 floats (4 MiB) compiled into the library, which every
 * GPU that loads the library keeps until the process exits; the K split is
 * chosen among those whose partial sums (splits x M x N floats) fit it, down
 * to no split at all, so no problem is refused for want of scratch. The first
 * call on a device resolves the array's address and should come before any
 * stream capture. All calls on a device share the array: calls that overlap
 * on the GPU (different streams, or concurrent host threads) race and must be
 * serialised by the caller. A timed-out device wait inside it is reported by
 * neso_device_status until neso_clear_device_status. */
NESO_API int neso_w8a16_matmul_mnk_noalloc(const void* X, const int8_t* W, const void* scale, float* Y, int32_t M,
                                           int32_t N, int32_t K, neso_stream_t stream);

/* ------------------------------------- one decoding step, paged cache -- */
/* Extensions (no reference kernel): what a decoding loop runs next to the
 * GEMV-shaped quantized matmuls. Keys and values live in pages: a cache holds
 * [num_pages, Hkv, page_size, D] 16-bit elements, addressed through a page,
 * head and token stride (elements; D is contiguous, everything else any
 * multiple of 8), so views of other orders or of a joint K/V buffer work. A
 * sequence's token t lies in page block_tables[b][t / page_size], row
 * t % page_size. Lengths, tables, positions and slots are device data: no call
 * reads them on the host, and a captured graph follows them. `workspace` is
 * the caller's and belongs to the call until it has run; calls that may
 * overlap need one each. */

/* Rotate q and k of N new tokens and write k and v to the cache.
 *   pair d < half of token n turns by row positions[a][n] of cos/sin
 *   [table_rows, half], where a is the axis whose section holds d (sections:
 *   `axes` host ints that add up to half; NULL for one axis):
 *     y[d] = x[d] cos - x[d + half] sin,  y[d + half] = x[d] sin + x[d + half] cos
 *   computed in fp32 and rounded once; elements from 2 * half on are copied.
 * q [N, Hq, D], k, v [N, Hkv, D] with token and head strides; q_out [N, Hq, D]
 * contiguous (may be q itself when q is contiguous). slots[n] is token n's
 * place, page * page_size + row. A slot outside the cache marks padding: such
 * a token is not cached and its row of q_out is zero. A position outside the
 * table turns to NaN. Slots of one call have to differ from each other. */
NESO_API int neso_rope_paged_append(const void* q, const void* k, const void* v, const float* cos, const float* sin,
                                    const int32_t* positions, const int64_t* slots, void* q_out, void* k_cache,
                                    void* v_cache, int32_t dtype, int32_t N, int32_t Hq, int32_t Hkv, int32_t D,
                                    int32_t half, int32_t table_rows, int32_t axes, const int32_t* sections,
                                    int64_t q_stride_n, int64_t q_stride_h, int64_t k_stride_n, int64_t k_stride_h,
                                    int64_t v_stride_n, int64_t v_stride_h, int32_t num_pages, int32_t page_size,
                                    int64_t kc_stride_page, int64_t kc_stride_head, int64_t kc_stride_token,
                                    int64_t vc_stride_page, int64_t vc_stride_head, int64_t vc_stride_token,
                                    neso_stream_t stream);

/* Attention of one query token per sequence, q [B, Hq, D], over the cached
 * tokens t < seq_lens[b] (the new one included); query head h reads kv head
 * h / (Hq / Hkv). D in {64, 128}.
 *   s = scale q.k;  s = softcap tanh(s / softcap) if softcap > 0;
 *   s += slopes[h] (t - (len - 1)) if slopes;  t > len - 1 - window if window > 0
 *   out [B, Hq, D] = softmax(s) v, in q's type.
 * With weights_in/weights_out (fp32 [B, Hkv, tokens], may be one buffer; tokens:
 * at least the longest clamped length, only t < seq_lens[b] is touched),
 * weights_out[b, kv, t] = weights_in[b, kv, t] + the sum of the softmax
 * weights of the kv head's query heads, for t < seq_lens[b]; the rest is left.
 * A length is clamped to [0, table_width * page_size]; tokens of a page
 * outside [0, num_pages) are left out, as is one whose score is -inf; with no
 * token left the row is zero. Distances (slopes, window) count cached tokens:
 * after neso_kv_evict has closed the gaps, they are distances in the trimmed
 * cache, not between the positions that the keys were rotated by. */
NESO_API int neso_paged_attention(const void* q, const void* k_cache, const void* v_cache,
                                  const int32_t* block_tables, const int32_t* seq_lens, const float* slopes,
                                  const float* weights_in, float* weights_out, void* out, void* workspace,
                                  int64_t workspace_bytes, int32_t dtype, int32_t B, int32_t Hq, int32_t Hkv,
                                  int32_t D, float scale, float softcap, int32_t window, int64_t q_stride_b,
                                  int64_t q_stride_h, int32_t num_pages, int32_t page_size, int64_t k_stride_page,
                                  int64_t k_stride_head, int64_t k_stride_token, int64_t v_stride_page,
                                  int64_t v_stride_head, int64_t v_stride_token, int32_t table_width,
                                  int64_t table_stride, int64_t win_stride_b, int64_t win_stride_h,
                                  int64_t wout_stride_b, int64_t wout_stride_h, neso_stream_t stream);
/* Bytes of workspace that neso_paged_attention needs on the current device (0:
 * none, workspace may be NULL); negative (a status code) for arguments that it would refuse. */
NESO_API int64_t neso_paged_attention_workspace(int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t table_width,
                                                int32_t page_size, int32_t with_weights);

/* Trim every sequence to at most `budget` (1 to 2^30) tokens per kv head: the first
 * `sink`, the last `recent` and, of those between, the ones with the largest
 * weight (ties: the lower index; NaN counts as largest) are kept, in order,
 * and moved to tokens 0, 1, ... under out_tables. kept [B, Hkv, budget] gets
 * their old indexes (-1 behind the last), new_lens[b] = min(len, budget)
 * (a buffer other than seq_lens).
 * Rows of weights_in hold table_width * page_size floats, whatever the lengths
 * are: all of them may be read. weights_out gets the kept weights and zero up to
 * the old length; it may be weights_in. out_tables may be the pointer block_tables (in
 * place). Otherwise each of its pages either lies where block_tables has it (a copy
 * of the table, or one that keeps some pages: such a sequence moves in order, by one
 * CTA per kv head) or does not occur in block_tables. Two sequences share no page. Kept tokens past the out table's end, and tokens
 * on a page outside [0, num_pages), are not moved. 16-bit elements; D a
 * multiple of 8, at most 256. */
NESO_API int neso_kv_evict(void* k_cache, void* v_cache, const int32_t* block_tables, const int32_t* out_tables,
                           const int32_t* seq_lens, const float* weights_in, float* weights_out, int32_t* kept,
                           int32_t* new_lens, int32_t B, int32_t Hkv, int32_t D, int32_t budget, int32_t recent,
                           int32_t sink, int32_t num_pages, int32_t page_size, int64_t k_stride_page,
                           int64_t k_stride_head, int64_t k_stride_token, int64_t v_stride_page,
                           int64_t v_stride_head, int64_t v_stride_token, int32_t table_width, int64_t table_stride,
                           int32_t out_width, int64_t out_stride, int64_t win_stride_b, int64_t win_stride_h,
                           int64_t wout_stride_b, int64_t wout_stride_h, neso_stream_t stream);

/* Logits of the next token, row by row (fp32 arithmetic, one rounding):
 *   x = logits[b, v]
 *   x = x > 0 ? x / repetition[b] : x * repetition[b]   if v is in the history
 *   x -= frequency[b] * n + presence[b] * (n > 0)        n: times v was generated
 *   x += bias[b, i] for each i with bias_ids[b, i] == v, in order
 *   out[b, v] = -inf unless bit v % 32 of mask[b, v / 32] is set
 * history [B, T] holds history_lens[b] token ids, the first prompt_lens[b] of
 * them the prompt (counted for repetition only); ids outside [0, V) are
 * skipped, lengths clamped to [0, T]. Any of history (with its lengths),
 * prompt_lens (none: all generated), repetition, frequency, presence,
 * bias_ids (with bias) and mask may be NULL. out may be logits itself. */
NESO_API int neso_process_logits(const void* logits, void* out, int32_t dtype, int32_t B, int32_t V,
                                 int64_t logits_stride, int64_t out_stride, const int32_t* history,
                                 const int32_t* history_lens, const int32_t* prompt_lens, int32_t T,
                                 int64_t history_stride, const float* repetition, const float* frequency,
                                 const float* presence, const int32_t* bias_ids, const float* bias, int32_t num_bias,
                                 const int32_t* mask, int64_t mask_stride, neso_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* NESO_B200_H */
