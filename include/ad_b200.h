/* libad_b200 -- C ABI of the B200 CUDA device backend.
 *
 * The reference (Eshaancoding/ad) reaches its GPU through per-backend Python
 * helpers over ctypes bindings of libOpenCL / libcuda+libnvrtc.  This library
 * is the single native boundary that replaces those helpers; the Python device
 * class (ad_b200.device.CudaB200Device) binds it with ctypes.  Each
 * declaration names the reference interface it replaces (path:line within the
 * reference project).
 *
 * Conventions: every function returns 0 on success, non-zero on failure with
 * a message in ad_last_error() (thread-local).  Device addresses are uint64_t.
 * Streams are small integers indexing the context's stream table
 * (0 = compute, 1 = host-to-device copies, 2 = device-to-host copies, 3 = comm).
 */
#ifndef AD_B200_H
#define AD_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define AD_B200_ABI_VERSION 1

typedef struct ad_ctx ad_ctx;
typedef struct ad_kernel ad_kernel;
typedef struct ad_graph ad_graph;

int ad_version(void);
/* cl_helper.py:23-26 check(), cuda_helper.py:14-15 check(): error reporting */
const char* ad_last_error(void);

/* cl_helper.py get_platforms/get_devices/initialize_context/create_command_queue
 * (opencl/device.py:10-44); cuda/device.py:8-19 (cuInit/cuCtxCreate, device 0) */
int ad_device_count(int* n);
int ad_init(int device, int n_streams, ad_ctx** out);
/* opencl/device.py:132-146 __del__ (free_queue/free_context/free_device) */
int ad_destroy(ad_ctx* ctx);
int ad_device_info(ad_ctx* ctx, int* sm_count, int* smem_optin, size_t* free_bytes,
                   size_t* total_bytes);

/* cl_helper.py:151-170 init_buffer; cuda_helper.py:80-84 (cuMemAlloc).  The
 * Python device makes ONE allocation (the arena) and sub-allocates it. */
int ad_malloc(ad_ctx* ctx, size_t bytes, uint64_t* dptr);
/* cl_helper.py free_buffer (opencl/device.py:134-136) */
int ad_free(ad_ctx* ctx, uint64_t dptr);
int ad_memset(ad_ctx* ctx, uint64_t dptr, int value, size_t bytes, int stream);

/* Pinned staging for Feeder/Receiver (the reference copies from pageable numpy
 * memory: cl_helper.py:304-332, cuda_helper.py:86-126) */
int ad_pinned_alloc(size_t bytes, void** p);
int ad_pinned_free(void* p);
/* cl_helper.py:304-332 write_buffer; cuda_helper.py:113-126 (cuMemcpyHtoD at kres offset) */
int ad_h2d(ad_ctx* ctx, uint64_t dst, const void* src, size_t bytes, int stream);
/* cl_helper.py:262-302 read_buffers; cuda_helper.py:86-111 (cuMemcpyDtoH) */
int ad_d2h(ad_ctx* ctx, void* dst, uint64_t src, size_t bytes, int stream);
int ad_d2d(ad_ctx* ctx, uint64_t dst, uint64_t src, size_t bytes, int stream);
/* cl_helper.py:304-332 write_buffer / cuda_helper.py:113-126 with the numpy
 * array's own (pageable) memory as source: staged through a ring of pinned
 * buffers, host copies on a few threads overlapped with the DMA.  Returns once
 * `src` may be reused; the device copy completes in stream order. */
int ad_h2d_pageable(ad_ctx* ctx, uint64_t dst, const void* src, size_t bytes, int stream);
/* cl_helper.py:262-302 read_buffers / cuda_helper.py:86-111 into a pageable
 * (freshly allocated numpy) destination; returns when `dst` holds the data. */
int ad_d2h_pageable(ad_ctx* ctx, void* dst, uint64_t src, size_t bytes, int stream);
/* Host memcpy on the library's copy threads (numpy -> pinned Feeder staging;
 * the reference copies with numpy, cl_helper.py:318-322). */
int ad_host_copy(void* dst, const void* src, size_t bytes);
/* cl_helper.py:457 waitAll (clFinish) */
int ad_stream_sync(ad_ctx* ctx, int stream);
int ad_sync(ad_ctx* ctx);

/* Events: stream ordering between the copy and compute streams, and timing.
 * (The reference has none; its queue-profiling flag is commented out at
 * cl_helper.py:133.) */
int ad_event_create(ad_ctx* ctx, int timing, void** ev);
int ad_event_destroy(void* ev);
int ad_event_record(ad_ctx* ctx, void* ev, int stream);
int ad_stream_wait_event(ad_ctx* ctx, int stream, void* ev);
int ad_event_sync(void* ev);
int ad_event_elapsed_ms(void* start, void* end, float* ms);

/* cl_helper.py:357-384 build_kernel (clCreateProgramWithSource/clBuildProgram);
 * cuda_helper.py:144-198 (nvrtcCompileProgram -> PTX -> cuModuleLoadData).
 * Here NVRTC compiles straight to an sm_100a cubin (no PTX is produced).
 * The returned cubin is malloc'ed; release it with ad_free_host. */
int ad_compile_cubin(const char* src, const char* name, const char* const* opts, int n_opts,
                     void** cubin, size_t* cubin_size, char* log, size_t log_len);
void ad_free_host(void* p);
/* cuda_helper.py:188-198 (cuModuleLoadData + cuModuleGetFunction) */
int ad_load_kernel(ad_ctx* ctx, const void* cubin, const char* fn_name, ad_kernel** out);
/* cl_helper.py free_kernel (opencl/device.py:138-141) */
int ad_kernel_free(ad_kernel* k);
int ad_kernel_set_smem(ad_kernel* k, int bytes);
int ad_kernel_attr(ad_kernel* k, int* regs, int* static_smem, int* max_threads);
/* cl_helper.py:445-455 clEnqueueNDRangeKernel; cuda_helper.py:210-222 cuLaunchKernel.
 * `args` is the usual array of pointers to each kernel parameter. */
int ad_launch(ad_ctx* ctx, ad_kernel* k, unsigned gx, unsigned gy, unsigned gz, unsigned bx,
              unsigned by, unsigned bz, unsigned smem, void** args, int stream);
int ad_check(ad_ctx* ctx);

/* TMA descriptor (CUtensorMap, 128 bytes) for a 2-D row-major tensor; used by
 * the dot-product kernels.  No reference counterpart (the reference's dot
 * product is a scalar loop: opencl/kernels/dotprod.py:7-43). */
int ad_tmap_2d(uint64_t base, uint64_t rows, uint64_t cols, uint64_t row_stride_bytes,
               uint32_t box_rows, uint32_t box_cols, int elem_bytes, int swizzle_bytes,
               void* out128);

/* CUDA-graph capture/replay of a ForNode body.  Replaces the Python replay
 * loop of opencl/device.py:114-124 (`for _ in cmd.r: self._run_proc(...)`). */
int ad_graph_begin(ad_ctx* ctx, int stream);
int ad_graph_end(ad_ctx* ctx, int stream, ad_graph** out);
int ad_graph_launch(ad_ctx* ctx, ad_graph* g, int stream);
int ad_graph_destroy(ad_graph* g);

/* NCCL data-parallel gradient all-reduce.  No reference counterpart: the
 * reference has no multi-device code (TODO.md:68-69 lists it as future work).
 * Init is non-blocking and polled against timeout_s; on timeout or error the
 * communicator is aborted and an error returned. */
int ad_nccl_unique_id(void* out128);
int ad_nccl_init(ad_ctx* ctx, int rank, int world, const void* uid128, double timeout_s);
int ad_allreduce_f32(ad_ctx* ctx, uint64_t send, uint64_t recv, size_t count, int op_max,
                     int stream);
int ad_nccl_abort(ad_ctx* ctx);

/* Gradient all-reduce over peer memory (no reference counterpart: the
 * reference has no multi-device code).  ad_peer_init maps every rank's
 * registered region (one cudaMalloc allocation starting at `base`: the
 * device's arena) into every other rank over CUDA IPC, exchanging the handles
 * with one NCCL all-gather (call it on all ranks after ad_nccl_init).
 * ad_peer_allreduce_f32 sums `count` floats at `ptr` (inside the region,
 * 16-byte aligned, count % 4 == 0) over all ranks in place with one kernel:
 * reduce-scatter + all-gather through NVLink loads and stores, ranks meeting
 * at flag barriers.  `op` (0..63) names the call site: each site's calls must
 * come in the same order on every rank.  A barrier that waits more than 2 s
 * writes 7 to the int at `err` (device address) and the kernel returns.
 * ad_peer_close unmaps (also done by ad_destroy). */
int ad_peer_init(ad_ctx* ctx, uint64_t base, size_t bytes);
int ad_peer_allreduce_f32(ad_ctx* ctx, uint64_t ptr, size_t count, int op, int stream, uint64_t err);
int ad_peer_close(ad_ctx* ctx);

/* cudaProfilerStart (on != 0) / cudaProfilerStop: brackets the launches a
 * profiler started with "--profile-from-start off" captures.  No reference
 * counterpart (measurement only). */
int ad_profiler_range(int on);

/* C = A @ B (b_is_nk = 0: B is K x N row-major) or C = A @ B^T (b_is_nk = 1:
 * B is N x K row-major); A is M x K row-major, C is M x N row-major, all fp32
 * device pointers; 3xTF32 on tcgen05.  No counterpart in the reference: this
 * entry point exists for callers that cannot allocate device memory.  It
 * allocates nothing: its split-operand scratch is a fixed 32 MiB device array
 * inside this library, so problems needing more than 8*(Mp+Np)*Kp + 256 bytes
 * of it (Mp = M rounded up to 128, Np = N to 256, Kp = K to 32) are rejected.
 * All calls share that array: calls that overlap on one GPU race.  The first
 * call on each device resolves the array's address (cudaGetSymbolAddress), so
 * make it before any stream capture.  `stream` is a cudaStream_t (NULL = the
 * legacy default stream); the call returns after its work has finished.
 * The resolved address is kept for the life of the process: do not call this
 * on a device after cudaDeviceReset. */
int ad_dot_tf32x3_noalloc(const float* A, const float* B, float* C, int M, int N, int K,
                          int b_is_nk, void* stream);

/* ---- Operators of language models (no reference counterpart: the reference
 * composes such steps from its elementwise, reduce and dot nodes) ------------
 *
 * They work on the caller's device memory (addresses are multiples of the
 * elements' size), allocate nothing, launch on
 * `stream` (a cudaStream_t; NULL = the legacy default stream) and return
 * without waiting.  `device`: the device that the memory and the stream belong
 * to, or -1 for the current one.  Element types are AD_F32, AD_BF16, AD_F16;
 * strides count elements, not bytes, and a row's elements are adjacent.  Sums
 * are held in 32 bits or more and results do not depend on scheduling.
 * Results may not overlap operands unless a call allows it. */
#define AD_F32 0
#define AD_BF16 1
#define AD_F16 2

/* Rotary positions of queries and keys (k_heads or q_heads may be 0).
 * Operands are [sequences][tokens][heads][dim] with the strides of the first
 * three axes; results may be their operands.  The first `rotary` elements of a
 * head are rotary / 2 pairs: (x[i], x[i + rotary/2]) with layout 0,
 * (x[2i], x[2i+1]) with layout 1; pair (u, v) becomes (u c - v s, v c + u s)
 * with c, s from row positions[token] of the [table_rows][rotary / 2] tables
 * (s negated when `inverse`: also the gradient).  A position outside the
 * tables (of 0 rows, too) makes NaNs.  Positions are of 64 bits when pos64, else of 32. */
int ad_rotary(int device, int dtype, const void* q, const int64_t* q_strides, void* q_out,
              const int64_t* q_out_strides, int q_heads, const void* k, const int64_t* k_strides,
              void* k_out, const int64_t* k_out_strides, int k_heads, int64_t sequences,
              int64_t tokens, int dim, int rotary, int layout, int inverse, const float* cos,
              const float* sin, int64_t table_rows, const void* positions, int pos64,
              int64_t pos_seq_stride, int64_t pos_tok_stride, void* stream);

/* Norms around a block with its gate and the scaled residual sum:
 *   u = norm(z) wa + ba (u = z when wa is NULL),
 *   h = scale x + act(gate) u (h = scale x + u when gate is NULL),
 *   y = norm(h) wb + bb (no y when wb is NULL).
 * kind 0: v / sqrt(mean v^2 + eps); 1: LayerNorm.  act is the sigmoid when
 * gate_sigmoid, else the identity.  Gate row r belongs to the rows
 * [r rows_per_gate, (r + 1) rows_per_gate).  Weights and biases are of type
 * wtype: AD_F32 or dtype.  stats: rows * 4 floats (16-byte aligned) for the
 * gradient.  h may be x or z, y may be the other one. */
int ad_block_norm(int device, int dtype, int wtype, int kind, const void* x, int64_t ldx,
                  const void* z, int64_t ldz, const void* gate, int64_t ldg,
                  int64_t rows_per_gate, int gate_sigmoid, const void* wa, const void* ba,
                  const void* wb, const void* bb, float scale, float eps, int64_t rows, int width,
                  void* h, int64_t ldh, void* y, int64_t ldy, float* stats, void* stream);
/* Bytes of workspace that ad_block_norm_grad needs; rows_per_gate 0: no gate. */
int ad_block_norm_grad_workspace(int device, int64_t rows, int width, int64_t rows_per_gate,
                                 size_t* bytes);
/* The gradients of ad_block_norm's operands from those of h and y: dx, dz, the
 * gate's (of its shape) and, of type wtype, the weights' and biases'.  With no
 * rows those of the weights and biases are zeros; how many rows the gate has is
 * not known then, and its gradient is left to ad_clear_rows. */
int ad_block_norm_grad(int device, int dtype, int wtype, int kind, const void* dh, int64_t lddh,
                       const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* z,
                       int64_t ldz, const void* gate, int64_t ldg, int64_t rows_per_gate,
                       int gate_sigmoid, const void* wa, const void* ba, const void* wb,
                       const void* bb, float scale, const float* stats, int64_t rows, int width,
                       void* dx, int64_t lddx, void* dz, int64_t lddz, void* dgate, int64_t lddg,
                       void* dwa, void* dba, void* dwb, void* dbb, void* workspace,
                       size_t workspace_bytes, void* stream);
/* Zeros in `rows` rows of row_bytes bytes, row_stride bytes apart. */
int ad_clear_rows(int device, void* p, int64_t row_stride, int64_t row_bytes, int64_t rows,
                  void* stream);

/* Of each row of scale * logits: the log probability of its token (0 for a
 * negative token, NaN for one past the vocabulary), the entropy of its
 * distribution, and the `top` (at most 32) most likely tokens with their log
 * probabilities, the lower index first among equal logits (-1 where fewer than
 * `top` logits are numbers).  Tokens are of 64 bits when tok64, else of 32.
 * stats: rows * 4 floats (16-byte aligned): the largest logit, the sum of
 * exp(scale (x - largest)) but for the rounding of scale times the largest, which
 * the gradient knows (0: a row of -inf alone), the entropy, the log of the sum of
 * exp(scale x). */
int ad_token_logprobs(int device, int dtype, const void* logits, int64_t ld, int64_t rows,
                      int64_t vocab, const void* tokens, int tok64, float scale, int top,
                      float* logp, float* entropy, float* stats, float* top_logp,
                      int64_t* top_index, void* stream);
/* The gradient of the logits from g_logp and g_entropy (rows floats each; NULL:
 * zeros).  `grad` may be the logits themselves. */
int ad_token_logprobs_grad(int device, int dtype, const void* logits, int64_t ld, int64_t rows,
                           int64_t vocab, const void* tokens, int tok64, float scale,
                           const float* stats, const float* g_logp, const float* g_entropy,
                           void* grad, int64_t ld_grad, void* stream);

/* Newton-Schulz orthogonalisation of `count` matrices G of rows x cols:
 * X = G / (|G|_F + eps), then `steps` (0 to 32) times X = a X + (b A + c A A) X
 * with A = X X^T and three coefficients a, b, c a step (host memory), from the
 * side with fewer rows.  Any strides; the result must not overlap G.  Products
 * take operands of 11 bits and accumulate in 32: the result is within about
 * 1e-3 (norm-wise) of the exact iteration.  Coefficients that let a singular
 * value grow past 1024 are refused.  A zero matrix gives zeros, whatever eps is,
 * one with NaN or infinity NaNs.  Blocks wait for one another inside the one cooperative
 * kernel; a wait that runs out (2 s) leaves NaNs in the result.  The workspace
 * is 256-byte aligned. */
int ad_orthogonalize_workspace(int64_t count, int64_t rows, int64_t cols, size_t* bytes);
int ad_orthogonalize(int device, int dtype, const void* g, int64_t count, int64_t rows,
                     int64_t cols, int64_t batch_stride, int64_t row_stride, int64_t col_stride,
                     int steps, const float* coefficients, float eps, int out_dtype, void* out,
                     int64_t out_batch_stride, int64_t out_row_stride, int64_t out_col_stride,
                     void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* AD_B200_H */
