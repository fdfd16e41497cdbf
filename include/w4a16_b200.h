/*
 * w4a16_b200.h -- C ABI of the sm_100a (B200) W4A16 fused dequant-GEMM library.
 *
 * Plain C: raw device pointers, 64-bit sizes and an opaque stream handle (a
 * cudaStream_t passed as void*; NULL means the legacy default stream). No
 * torch or C++ types cross this boundary and no exception escapes it: every
 * entry point returns 0 on success or a negative W4A16_* status, and
 * w4a16_strerror() turns a status into text. All launches are asynchronous
 * on the given stream; nothing here allocates device memory or synchronises
 * (scratch memory, where a kernel needs it, is passed in by the caller) except
 * the peer-to-peer buffer helpers w4a16_p2p_*, which set up the multi-GPU path.
 *
 * Data format (the reference's, unchanged): W is [K, N] (K = in_features),
 * quantised in groups of G consecutive K-rows per column.
 *   qweight int32 [K/8, N]  row k = 8i+j of column n in bits [4j, 4j+4) of qweight[i, n]
 *   scales  fp16  [K/G, N]
 *   zeros   fp16  [K/G, N]  integer zero-points (0..15 as produced by w4a16_quantize)
 * All tensors are row-major and dense unless a leading dimension is given.
 */
#ifndef W4A16_B200_H_
#define W4A16_B200_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes. */
#define W4A16_OK                 0
#define W4A16_ERR_INVALID       -1  /* bad size, group size or null pointer */
#define W4A16_ERR_ALIGNMENT     -2  /* pointer/stride alignment a kernel needs is missing */
#define W4A16_ERR_LAUNCH        -3  /* the CUDA launch itself failed */
#define W4A16_ERR_DEVICE        -4  /* device is not sm_100 or cannot be queried */
#define W4A16_ERR_TIMEOUT       -5  /* a kernel's bounded wait expired (sticky device flag) */
#define W4A16_ERR_WORKSPACE     -6  /* workspace missing, too small or misaligned */
#define W4A16_ERR_INDEX         -8  /* an index read from device memory was out of range (sticky flag) */

/* Input dtypes accepted by w4a16_quantize. */
#define W4A16_DTYPE_F16  0
#define W4A16_DTYPE_F32  1
#define W4A16_DTYPE_BF16 2

/* Library version, major*10000 + minor*100 + patch. */
int w4a16_version(void);

/* Human-readable text for a status code; never NULL. */
const char* w4a16_strerror(int status);

/*
 * Fused GEMM: y[m, n] = sum_k x[m, k] * dequant(qweight, scales, zeros)[k, n]
 * accumulated in fp32, rounded to fp16, then (if bias != NULL) y + bias[n]
 * rounded to fp16 again.
 *
 * Replaces the reference's w4a16_matmul (w4a16-kernel/src/w4a16/triton_kernel.py:131-200)
 * and its CUDA twin w4a16_gemm_cuda (w4a16-kernel/src/w4a16/cuda/w4a16_gemm.cu:76-115);
 * the bias add is the one W4A16Linear.forward does afterwards (linear.py:90-91).
 *
 * x: fp16 [M, K] dense. y: fp16, row m at y + m*ldy (ldy >= N), so a caller
 * can write one column shard of a wider output. Requirements (the reference's
 * assertions, triton_kernel.py:153-182): K % 8 == 0, K % group_size == 0,
 * group_size % 64 == 0. M == 0 or N == 0 is a no-op.
 * Routing: M <= 32 runs the memory-bound decode kernel, larger M the tcgen05
 * tensor-core kernel (which needs N % 8 == 0; other N fall back to decode
 * launches over 32-row slices of x).
 *
 * workspace: device scratch of at least w4a16_gemm_workspace_size() bytes,
 * 256-byte aligned, ZEROED before its first use. The decode kernel passes the
 * partial sums of column strips shared by two or more CTAs through its first
 * W4A16_NOALLOC_SCRATCH_BYTES (tagged 64-bit words) and leaves them zero again;
 * the tensor-memory-operand prefill kernel, when it splits K, keeps arrival
 * counters (left zero) and fp32 partial tiles past that offset. So one zeroed
 * buffer serves every later call on the same stream, whatever the shape;
 * launches that may run concurrently need separate workspaces, and a graph
 * capture needs one of its own, zeroed inside the graph. A prefill call
 * given less workspace than the query returned runs without splitting K. (A
 * launch abandoned on W4A16_ERR_TIMEOUT can leave words set: zero the buffer
 * again before reusing it.) May be NULL when the size query returned 0.
 */
int w4a16_gemm(const void* x, const int32_t* qweight, const void* scales,
               const void* zeros, const void* bias, void* y,
               int64_t M, int64_t N, int64_t K, int64_t group_size,
               int64_t ldy, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * w4a16_gemm with an fp32 output and no rounding (and no bias): the partial
 * sums of a K-sharded (row-parallel) layer, summed across GPUs before the one
 * final fp16 rounding, so a sharded layer matches the unsharded result.
 * y: fp32, row m at y + m*ldy. Same requirements and workspace as w4a16_gemm.
 * No reference counterpart: the reference has no multi-GPU path.
 */
int w4a16_gemm_f32(const void* x, const int32_t* qweight, const void* scales,
                   const void* zeros, float* y, int64_t M, int64_t N, int64_t K,
                   int64_t group_size, int64_t ldy, void* workspace,
                   int64_t workspace_bytes, void* stream);

/*
 * SwiGLU of a fused gate/up projection: h[m, n] = silu(g) * u with
 * g = gate_up[m, n] and u = gate_up[m, N + n] (fp16 in, fp32 math, one fp16
 * rounding). gate_up rows have pitch ld_in >= 2N, h rows pitch ld_out >= N.
 * No reference counterpart: it joins the projections of the MLP block the
 * benchmark configuration names.
 */
int w4a16_swiglu(const void* gate_up, void* h, int64_t M, int64_t N, int64_t ld_in,
                 int64_t ld_out, void* stream);

/*
 * The gate/up projection of an MLP block fused with its SwiGLU: the GEMM's epilogue
 * writes h[m, j] = fp16(silu(g) * u) (fp32 math on the fp16-rounded g and u, one
 * rounding: the same values as w4a16_gemm followed by w4a16_swiglu) instead of the
 * [M, N] gate/up output. The weight's N columns hold the gate and up projections
 * interleaved in blocks of 16: columns 32b .. 32b+15 are gate columns 16b .. 16b+15
 * and columns 32b+16 .. 32b+31 the matching up columns, so output column j reads
 * weight columns 32(j/16) + j%16 and that + 16. h: fp16 [M, N/2], row pitch ldh >= N/2.
 * N % 32 == 0; x, qweight, scales, zeros 16-byte aligned (W4A16_ERR_ALIGNMENT
 * otherwise); the other requirements and the workspace are w4a16_gemm's. No reference
 * counterpart: it removes the [M, N] round trip between the projections of the MLP
 * block the benchmark configuration names.
 */
int w4a16_gemm_swiglu(const void* x, const int32_t* qweight, const void* scales,
                      const void* zeros, void* h, int64_t M, int64_t N, int64_t K,
                      int64_t group_size, int64_t ldh, void* workspace,
                      int64_t workspace_bytes, void* stream);

/*
 * Option bits of w4a16_gemm_ex.
 *   W4A16_FLAG_KERNEL_ORDER  qweight holds the kernel nibble order written by
 *                            w4a16_repack instead of the reference's
 *   W4A16_FLAG_SWIGLU        the w4a16_gemm_swiglu epilogue (y is h [M, N/2])
 *   W4A16_FLAG_F32_OUT       the w4a16_gemm_f32 output (fp32, unrounded, no bias)
 *   W4A16_FLAG_BF16_OUT      y (and bias) bf16: the fp32 sums rounded to bf16, then
 *                            y + bias rounded again (for bf16 models, whose
 *                            activations w4a16_convert takes to fp16 first)
 */
#define W4A16_FLAG_KERNEL_ORDER 1u
#define W4A16_FLAG_SWIGLU       2u
#define W4A16_FLAG_F32_OUT      4u
#define W4A16_FLAG_BF16_OUT     8u

/*
 * w4a16_gemm with option bits (above): one entry point for the plain, SwiGLU and
 * fp32-output GEMMs over either nibble order. SWIGLU excludes F32_OUT, BF16_OUT and a
 * bias; F32_OUT excludes BF16_OUT and a bias;
 * KERNEL_ORDER and SWIGLU need N % 8 == 0 and 16-byte-aligned x, qweight, scales and
 * zeros (W4A16_ERR_ALIGNMENT otherwise). Unknown bits: W4A16_ERR_INVALID. No
 * reference counterpart (w4a16_gemm is the reference's operator).
 */
int w4a16_gemm_ex(const void* x, const int32_t* qweight, const void* scales,
                  const void* zeros, const void* bias, void* y, int64_t M, int64_t N,
                  int64_t K, int64_t group_size, int64_t ldy, uint32_t flags,
                  void* workspace, int64_t workspace_bytes, void* stream);

/*
 * dst[i] = src[i] rounded to dst's type, n elements; src fp16, fp32 or bf16, dst fp16
 * or bf16 (W4A16_DTYPE_*). For bf16 activations: bf16 -> fp16 is exact for |x| in
 * [2^-14, 65504] (and 0), so the fp16 GEMM computes the bf16 product unchanged
 * there. No reference counterpart (the reference takes fp16 activations only).
 */
int w4a16_convert(const void* src, int src_dtype, void* dst, int dst_dtype, int64_t n,
                  void* stream);

/*
 * Offline repack of qweight [K/8, N] between the reference's nibble order (row 8i+j in
 * nibble j of word [i, n], w4a16-kernel/src/w4a16/quant.py:45-70) and the kernel order
 * (rows k0, k2, k4, k6, k1, k3, k5, k7 in nibbles 0..7): to_kernel_order != 0 converts
 * reference -> kernel, 0 converts back. Elementwise; out may equal qweight. In the
 * kernel order the GEMMs extract a word's consecutive row pairs with one shift and four
 * masks (W4A16_FLAG_KERNEL_ORDER). No reference counterpart: a load-time layout, the
 * stored (state_dict) format stays the reference's.
 */
int w4a16_repack(const int32_t* qweight, int32_t* out, int64_t K, int64_t N,
                 int to_kernel_order, void* stream);

/*
 * dst = src, `bytes` bytes (a multiple of 16; both 16-byte aligned), as a kernel on
 * `stream` that chains with the GEMM launches around it under programmatic
 * dependent launch. No reference counterpart: it stages a step's inputs in (or its
 * outputs out) inside a CUDA-graph-captured serving loop, where a memory-copy node
 * before a GEMM would make that GEMM wait for its predecessor's completion instead
 * of overlapping the predecessor's tail. Either pointer may be device memory or
 * pinned host memory mapped into the device's address space (W4A16_ERR_INVALID
 * otherwise). src_ready != 0 promises that no earlier kernel on the stream writes
 * src (e.g. inputs the host wrote into pinned memory): the kernel then reads src
 * while the previous kernel still runs. dst is written only after the previous
 * kernel completes, and the copy completes after it.
 */
int w4a16_stage(const void* src, void* dst, int64_t bytes, int src_ready, void* stream);

/*
 * w4a16_gemm_ex on host-resident activations: x_host [M, K] fp16 is staged into the
 * device buffer x_dev, the GEMM writes the device buffer y_dev [M, n] (n = N, or N/2
 * with W4A16_FLAG_SWIGLU; fp32 with W4A16_FLAG_F32_OUT, bf16 with
 * W4A16_FLAG_BF16_OUT, else fp16), and y_dev is staged out to y_host: kernels on
 * `stream` chained under programmatic dependent launch (no copy-engine transfers
 * between them), so an eager loop of calls keeps the GEMM's start overlapped with
 * its predecessor. Up to 32 tokens the GEMM writes y_host directly (y_dev unused). x_host and y_host must be pinned host memory
 * mapped into the device's address space (W4A16_ERR_INVALID otherwise); all four
 * buffers 16-byte aligned, M*K*2 and the y bytes multiples of 16
 * (W4A16_ERR_ALIGNMENT). y_host holds the result once the stream has completed.
 * x_dev/y_dev may be reused by the next call on the same stream. No reference
 * counterpart (the reference's GEMM takes device tensors).
 */
int w4a16_gemm_host(const void* x_host, const int32_t* qweight, const void* scales, const void* zeros,
                    const void* bias, void* y_host, int64_t M, int64_t N, int64_t K, int64_t group_size,
                    uint32_t flags, void* x_dev, void* y_dev, void* workspace, int64_t workspace_bytes,
                    void* stream);

/*
 * Bytes of workspace w4a16_gemm needs for this shape on the current device
 * (0 for shapes whose kernels need none: N % 8 != 0, or a prefill shape run
 * without splitting K). Shapes that route to the decode or prefill kernels need
 * the device (its SM count); on a machine without one the query returns
 * W4A16_ERR_DEVICE. No reference counterpart: the reference's kernels never
 * split K across thread blocks.
 */
int w4a16_gemm_workspace_size(int64_t M, int64_t N, int64_t K, int64_t group_size,
                              int64_t* bytes_out);

/*
 * Group-wise asymmetric uint4 quantisation + packing of w [K, N] (dtype one of
 * W4A16_DTYPE_*), bit-exact with the reference's quantize_weight
 * (w4a16-kernel/src/w4a16/quant.py:101-144): fp32 scale (max-min)/15 (1 when
 * not > 0), zero = clamp(rint(-min/scale), 0, 15), q = clamp(rint(w/scale) + zero, 0, 15).
 * Requirements: K % 8 == 0, K % group_size == 0, group_size >= 1.
 * Non-finite weights produce unspecified codes; the caller rejects them first.
 */
int w4a16_quantize(const void* w, int w_dtype, int32_t* qweight, void* scales,
                   void* zeros, int64_t K, int64_t N, int64_t group_size,
                   void* stream);

/*
 * w4a16_quantize with option bits. W4A16_QUANT_SYMMETRIC: symmetric codes, the
 * layout GPTQ-style checkpoints use with sym=True -- per (group, column) zero = 8 and
 * scale = 2 * max|w| / 15 in fp32 (1 when not > 0), q = clamp(rint(w / scale) + 8,
 * 0, 15) -- stored in the same qweight / scales / zeros format, so every GEMM entry
 * point takes it unchanged. No reference counterpart (the reference quantises
 * asymmetrically only). Unknown bits: W4A16_ERR_INVALID.
 */
#define W4A16_QUANT_SYMMETRIC 1u
int w4a16_quantize_ex(const void* w, int w_dtype, int32_t* qweight, void* scales,
                      void* zeros, int64_t K, int64_t N, int64_t group_size,
                      uint32_t flags, void* stream);

/*
 * Pack int32 codes q [K, N] (each in 0..15) into qweight [K/8, N]
 * (w4a16-kernel/src/w4a16/quant.py:45-70). Codes are masked with 0xF; the
 * range check the reference asserts stays with the caller. K % 8 == 0.
 */
int w4a16_pack_int4(const int32_t* q, int32_t* qweight, int64_t K, int64_t N,
                    void* stream);

/* Inverse of w4a16_pack_int4: qweight [K/8, N] -> q [K, N] in 0..15
 * (w4a16-kernel/src/w4a16/quant.py:73-95). */
int w4a16_unpack_int4(const int32_t* qweight, int32_t* q, int64_t K, int64_t N,
                      void* stream);

/* w[k, n] = fp16(fp16(q - z) * s) for the group of row k, fp16 [K, N]
 * (w4a16-kernel/src/w4a16/quant.py:147-178). K % group_size == 0, K % 8 == 0. */
int w4a16_dequantize(const int32_t* qweight, const void* scales, const void* zeros,
                     void* w, int64_t K, int64_t N, int64_t group_size,
                     void* stream);

/*
 * Read and clear the device's sticky error flags for the current device
 * (bit 0: a bounded wait in a GEMM kernel ran out of its time budget and the
 * kernel abandoned its tile; bit 1: a position, slot, page id or row that a kernel
 * of the cache read from device memory was out of range, and was skipped or read as
 * index 0). Synchronises the given stream.
 * Returns W4A16_OK when no flag was set, W4A16_ERR_INDEX when bit 1 alone was,
 * W4A16_ERR_TIMEOUT when bit 0 was; in that last case it also zeroes this device's w4a16_gemm_noalloc scratch array (if
 * it has been set up) on `stream` and synchronises again, since its callers
 * cannot clear it themselves. Results of the launches since the last check are
 * unspecified after a timeout. Caller-owned workspaces and peer buffers may
 * hold stale words too: zero them (w4a16_reset_scratch) before reusing them.
 * No reference counterpart: the reference's kernels have no bounded waits.
 */
int w4a16_check_device_errors(void* stream, uint32_t* flags_out);

/*
 * Time budget, in nanoseconds, of every bounded wait in the kernels launched
 * after this call (process-wide; 0 restores the default of 4 s; otherwise
 * 1 ms <= ns <= 600 s, else W4A16_ERR_INVALID). Each launch carries the budget
 * as a kernel parameter, so launches already queued or captured in a CUDA graph
 * keep theirs. A shorter budget lets a caller (or a test) detect a lost peer
 * sooner; legitimate waits last microseconds to milliseconds. The waits that
 * keep a kernel from exiting with copies or MMAs in flight always use 4 s.
 * No reference counterpart.
 */
int w4a16_set_wait_budget_ns(int64_t ns);

/*
 * Prefill kernel (M > 32 tokens) selection, process-wide, for the launches after
 * this call. W4A16_PREFILL_AUTO (the default) picks per shape between the kernel
 * whose dequantised weights are the shared-memory B operand of tcgen05.mma
 * (W4A16_PREFILL_SMEM_B) and the one whose dequantised weights are the
 * tensor-memory A operand (W4A16_PREFILL_TMEM_A), by a cost model measured on
 * B200. Forcing one exists for tests and tuning; both give results within the
 * GEMM tolerance of each other (the same fp16 weights, fp32 sums in another order).
 * Anything else returns W4A16_ERR_INVALID. No reference counterpart.
 */
#define W4A16_PREFILL_AUTO 0
#define W4A16_PREFILL_SMEM_B 1
#define W4A16_PREFILL_TMEM_A 2
int w4a16_set_prefill_kernel(int which);
/* The prefill kernel (W4A16_PREFILL_SMEM_B or _TMEM_A) the current selection gives an
 * M x N x K GEMM with N % 8 == 0 on the current device, or W4A16_PREFILL_AUTO when M <= 32
 * (decode). For reports and tests; no reference counterpart. */
int w4a16_prefill_choice(int64_t M, int64_t N, int64_t K, int* which);
/* The plan the cost model makes for an M x N x K GEMM (K % 64 == 0) on a GPU with num_sms
 * SMs, under the current selection, without touching a device: *which as in
 * w4a16_prefill_choice; for the tensor-memory-operand kernel *tokens_per_tile (its tile
 * height, 64..192) and *splits (K split over that many CTAs for the tiles it splits: every
 * tile when the tiles do not fill one wave, else the last wave's; 1: none), else 0 and 1.
 * A launch splits K only when it is given the workspace the size query returns. For reports
 * and tests; no reference counterpart. */
int w4a16_prefill_plan(int64_t M, int64_t N, int64_t K, int num_sms, int* which, int* tokens_per_tile,
                       int* splits);

/*
 * Which CUDA graph capture `stream` is part of: a number of its own for each, 0 when it is not capturing. A workspace
 * whose zeroing was captured is not zero until the graph runs, and one that a graph uses must not serve launches
 * outside it at the same time: give each capture a workspace of its own, zeroed inside it.
 */
int w4a16_stream_capture_id(void* stream, uint64_t* id_out);

/*
 * After W4A16_ERR_TIMEOUT: zero `workspace_bytes` of a caller's GEMM workspace
 * (when `workspace` is not NULL) and this device's w4a16_gemm_noalloc scratch
 * array (when set up), asynchronously on `stream`; allocates nothing. The next
 * GEMM on that stream then starts from clean scratch. No reference counterpart.
 */
int w4a16_reset_scratch(void* workspace, int64_t workspace_bytes, void* stream);

/*
 * w4a16_gemm without a workspace argument and without allocating anything.
 * No counterpart in the reference (its kernels need no scratch at all).
 *
 * For callers that cannot allocate device memory at call time: a C or FFI
 * host with no device allocator of its own, an engine whose memory planner
 * has already handed out all device memory, or a plugin interface whose
 * launch call passes no scratch buffer. The decode kernel's scratch (the
 * partial sums of shared column strips) lives instead in one static device
 * array inside this library, W4A16_NOALLOC_SCRATCH_BYTES per device, whose
 * address the library looks up once per device. Shapes whose decode launch
 * would need more than that return W4A16_ERR_SCRATCH_LIMIT (on a 148-SM B200
 * every shape fits: the need is CTAs * M-tiles * 8 KiB, at most 148 * 4 *
 * 8 KiB = 4.6 MiB); prefill shapes need no scratch.
 *
 * The first call on each device does the set-up: it looks the array up,
 * zeroes it on `stream` and synchronises that stream. Make that first call
 * before any stream capture; a first call made while `stream` is capturing
 * returns W4A16_ERR_INVALID. The array must be zero whenever a decode launch
 * starts: set-up zeroes it and every completed launch leaves it zero; a launch
 * abandoned on a timeout may leave words set, and w4a16_check_device_errors
 * zeroes the array again when it reports W4A16_ERR_TIMEOUT (as does
 * w4a16_reset_scratch). There is ONE scratch array per device, so calls whose kernels can run
 * at the same time (different streams, threads or processes sharing a
 * context, parallel graph branches) race on it and give wrong results: keep
 * every call on one device ordered, or use w4a16_gemm with a workspace per
 * stream. Arguments, routing and results are those of w4a16_gemm.
 */
#define W4A16_NOALLOC_SCRATCH_BYTES (5 * 1024 * 1024)
#define W4A16_ERR_SCRATCH_LIMIT -7  /* shape needs more than the static scratch */
int w4a16_gemm_noalloc(const void* x, const int32_t* qweight, const void* scales,
                       const void* zeros, const void* bias, void* y,
                       int64_t M, int64_t N, int64_t K, int64_t group_size,
                       int64_t ldy, void* stream);

/*
 * Row-parallel decode GEMM fused with its all-reduce (no counterpart in the
 * reference, which has no multi-GPU path): y = fp16(sum over the `world` ranks of
 * x_r @ dequant(W_r)) [+ bias, rounded again], where each rank holds a K-slice
 * of x and of the weight. One kernel per rank: the CTA that finalises an output
 * element writes its fp32 partial, tagged with the call's epoch in one 64-bit
 * word, into this rank's slot of every rank's peer-to-peer buffer (plain stores
 * over NVLink; no fence, no flag); the last CTAs to finish read their share of
 * the elements in every slot of their own buffer until each word carries the
 * epoch's tag (bounded wait), and sum the slots in rank order into y -- the same
 * values as an fp32 all-reduce of the partials followed by one fp16 rounding.
 *
 * peers: HOST array of `world` buffer addresses as mapped on this GPU (this
 * rank's own buffer at index `rank`), each w4a16_p2p_buffer_bytes(world, slot)
 * bytes, 16-byte aligned, zeroed before first use (w4a16_p2p_alloc does); the
 * addresses are copied into the launch. ctl: this rank's two device int32
 * control words, zeroed before first use. slot >= M * N and even. Every rank
 * must issue the same sequence of calls on one stream (a call's words alternate
 * between two buffer halves by the call count kept in ctl); calls on a buffer
 * must not overlap. Requirements as w4a16_gemm plus M <= 32, N % 8 == 0,
 * 16-byte-aligned inputs, 2 <= world <= 8. The workspace is w4a16_gemm's.
 */
int w4a16_gemm_allreduce(const void* x, const int32_t* qweight, const void* scales,
                         const void* zeros, const void* bias, void* y,
                         int64_t M, int64_t N, int64_t K, int64_t group_size,
                         int64_t ldy, void* workspace, int64_t workspace_bytes,
                         const unsigned long long* peers, int world, int rank,
                         int* ctl, int64_t slot, void* stream);

/*
 * Column-parallel decode GEMM fused with its all-gather (no counterpart in the
 * reference): rank r holds columns [r*N, (r+1)*N) of the weight (and of bias) and
 * every rank receives the whole y = [M, world*N] (row pitch ldy >= world*N): the
 * CTA that finalises an element writes its fp16 value (bias added, rounded as
 * w4a16_gemm does) as a tagged 64-bit word into this rank's slot of every rank's
 * buffer, and the last CTAs to finish copy every rank's slot into y once the tags
 * of this call are in (bounded wait). The same bits as w4a16_gemm on each rank
 * followed by an all-gather of the columns. Peers, ctl, slot (>= M*N), ordering
 * and requirements as w4a16_gemm_allreduce, whose buffers it shares.
 */
int w4a16_gemm_allgather(const void* x, const int32_t* qweight, const void* scales,
                         const void* zeros, const void* bias, void* y,
                         int64_t M, int64_t N, int64_t K, int64_t group_size,
                         int64_t ldy, void* workspace, int64_t workspace_bytes,
                         const unsigned long long* peers, int world, int rank,
                         int* ctl, int64_t slot, void* stream);

/* Bytes of one rank's peer-to-peer buffer for w4a16_gemm_allreduce / _allgather. */
int w4a16_p2p_buffer_bytes(int world, int64_t slot, int64_t* bytes_out);

/* A zeroed device buffer of `bytes` on the current device and its 64-byte CUDA
 * IPC handle (for the peers' w4a16_p2p_open); release with w4a16_p2p_free. */
int w4a16_p2p_alloc(int64_t bytes, void** ptr_out, void* handle_out);

/* Map a peer's buffer from its 64-byte IPC handle; release with w4a16_p2p_close. */
int w4a16_p2p_open(const void* handle, void** ptr_out);
int w4a16_p2p_close(void* ptr);
int w4a16_p2p_free(void* ptr);

/*
 * ---------------------------------------------------------------------------
 * Attention over a 4-bit paged key/value cache (no counterpart in the reference,
 * which ends at the linear layers): what lies between a block's qkv projection and
 * its output projection.
 *
 * A cached value is offset + scale * code, code in 0..15, with one fp16 (scale,
 * offset) pair per token, kv head and group of group_size channels: offset =
 * fp16(min), scale = fp16((max - offset) / 15) (1 when not > 0), code =
 * clamp(rint((x - offset) / scale), 0, 15). Values beyond +-65504 are stored as that;
 * a group with an infinity or NaN in it gets the offset NaN. Sixteen tokens of a head
 * make a block: key codes [16, D/2] bytes (channel 2i in the low nibble of byte i),
 * value codes, key pairs [16, D/group_size, 2] fp16, value pairs. A page is
 * page_size / 16 blocks of each kv head. pool: [layers, pages, kv_heads, page bytes],
 * 16-byte aligned.
 */
typedef struct {
  void* pool;
  int64_t layers, pages; /* pages * page_size below 2^32 */
  int32_t kv_heads;
  int32_t head_dim;      /* 64 or 128 */
  int32_t page_size;     /* tokens, a multiple of 16, at most 4096 */
  int32_t group_size;    /* 64, or head_dim */
} w4a16_kv4_cache;

/* Which sequence holds which pages, in device memory: refs [pages] (how many rows hold
 * a page; 0: free), block_table [rows, width] (page ids, -1: none), kv_lens [rows]. */
typedef struct {
  int32_t *refs, *block_table, *kv_lens;
  int32_t pages, rows, width, page_size;
} w4a16_kv4_tables;

/* Bytes of a page of one kv head. */
int w4a16_kv4_page_bytes(int head_dim, int page_size, int group_size, int64_t* bytes_out);

/*
 * Queries [T, heads, D] and keys [T, kv_heads, D] (fp16 or bf16, channels contiguous, any
 * token and head strides, in elements): RMS norm of each head (x / sqrt(mean(x^2) + eps) *
 * weight; a null weight skips it), then the rotation of the first `rot` channels (a multiple
 * of 8): pairs (i, i + rot/2), or (2i, 2i+1) when interleaved, by the angle whose cosine and
 * sine are cos_sin[position][i] and cos_sin[position][rot/2 + i] (fp32 [max_position, rot], 16-byte
 * aligned).
 * positions: [T] (axes 1), or [3, T] (axes 3): frequencies i < axis0_end turn by the first
 * row's position, i < axis1_end by the second's, the others by the third's. fp32 arithmetic,
 * one rounding. q_out, k_out: dense, 16-byte aligned. weight_dtype: dtype, or fp32.
 */
int w4a16_qk_norm_rope(const void* q, const void* k, int dtype, int64_t T, int heads, int kv_heads, int head_dim,
                       int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride, int64_t k_head_stride,
                       const int64_t* positions, int axes, int axis0_end, int axis1_end, const float* cos_sin,
                       int64_t max_position, int rot, int interleaved, const void* q_weight, const void* k_weight,
                       int weight_dtype, float eps, void* q_out, void* k_out, void* stream);

/*
 * The same, with the keys (normed and rotated, not rounded before) and the values [T, kv_heads, D]
 * quantised into `layer` of the cache instead: token t goes to slots[t] = page * page_size +
 * offset in the page (negative: not cached). No slot may appear twice in one call.
 */
int w4a16_qk_norm_rope_append(const void* q, const void* k, const void* v, int dtype, int64_t T, int heads,
                              int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride,
                              int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                              const int64_t* positions, int axes, int axis0_end, int axis1_end, const float* cos_sin,
                              int64_t max_position, int rot, int interleaved, const void* q_weight,
                              const void* k_weight, int weight_dtype, float eps, void* q_out,
                              const w4a16_kv4_cache* cache, int64_t layer, const int64_t* slots, void* stream);

/* Cached tokens back in 16 bits: out [2, n, kv_heads, D] (fp16 or bf16; keys, then values) of the
 * tokens in slots [n]; a negative slot gives zeros. */
int w4a16_kv4_gather(const w4a16_kv4_cache* cache, int64_t layer, const int64_t* slots, int64_t n, void* out, int dtype,
                     void* stream);

/*
 * Attention of new tokens over the cache: q [T, heads, D] (fp16 or bf16, 16-byte aligned, strides
 * multiples of 8 elements), o [T, heads, D] dense, lse [T, heads] fp32 or null (natural log-sum-exp
 * of the scaled scores). Query head h reads kv head h / (heads / kv_heads). Sequence b has kv_lens[b]
 * cached tokens, the new ones (already appended) among them, in the pages block_table[b, :] (entries
 * beyond its length are not read); its queries are q[cu_q[b] : cu_q[b + 1]], or T / seqs each when
 * cu_q is null, the last of which stands at position kv_lens[b] - 1. A query sees the tokens up to its
 * own position, or the last `window` of those when window > 0; one that sees none (a length of 0)
 * gives zeros and lse = -inf, and so do queries before cu_q[0] and from cu_q[seqs] on. max_q: at least the longest sequence's queries (ignored when cu_q is
 * null). workspace: w4a16_kv4_attention_workspace_size bytes, 256-byte aligned, ZEROED before its
 * first use and left ready for the next call on the same stream; calls that may run at the same time
 * need one each, and so does each graph capture (zeroed inside it). Only its first 65536 bytes have to be zero.
 */
int w4a16_kv4_attention(const void* q, int dtype, int64_t T, int heads, int64_t q_token_stride, int64_t q_head_stride,
                        const w4a16_kv4_cache* cache, int64_t layer, const int32_t* block_table, int64_t table_width,
                        const int32_t* kv_lens, const int32_t* cu_q, int64_t seqs, int64_t max_q, float scale,
                        int window, void* o, float* lse, void* workspace, int64_t workspace_bytes, void* stream);
/* The same with a window that does not hide a sequence's first `sinks` tokens: a query sees the tokens t up to
 * its own position with t > position - window or t < sinks. Without a window (0) sinks say nothing. */
int w4a16_kv4_attention_sinks(const void* q, int dtype, int64_t T, int heads, int64_t q_token_stride,
                              int64_t q_head_stride, const w4a16_kv4_cache* cache, int64_t layer,
                              const int32_t* block_table, int64_t table_width, const int32_t* kv_lens,
                              const int32_t* cu_q, int64_t seqs, int64_t max_q, float scale, int window, int sinks,
                              void* o, float* lse, void* workspace, int64_t workspace_bytes, void* stream);
int w4a16_kv4_attention_workspace_size(const w4a16_kv4_cache* cache, int64_t T, int heads, int64_t seqs, int64_t max_q,
                                       int64_t* bytes_out);

/*
 * The attention weight that cached tokens collect: after[b, kv head, t] = what the token had, before[b, kv head, t]
 * (nothing where it is new, t >= kv_lens[b] - queries), plus the sum over the sequence's queries and the kv head's
 * query heads that see it of exp(scale q . k - lse). q .. sinks as in w4a16_kv4_attention_sinks, lse [T, heads] what that
 * call gave (a query of -inf gives nothing; every other one counts, a draft's too that is rejected later). before and
 * after, fp32: entry (sequence, kv head, token) at two strides, tokens contiguous, `capacity` of them; the two are the
 * same, or share no memory (else refused, as are entries of `after` that do). What lies behind a sequence's length is not
 * written; a sequence longer than `capacity` is left out (index flag). workspace: 256-byte aligned, any contents; calls
 * that may run at the same time need one each.
 */
int w4a16_kv4_attention_weights(const void* q, int dtype, int64_t T, int heads, int64_t q_token_stride,
                                int64_t q_head_stride, const w4a16_kv4_cache* cache, int64_t layer,
                                const int32_t* block_table, int64_t table_width, const int32_t* kv_lens,
                                const int32_t* cu_q, int64_t seqs, int64_t max_q, float scale, int window, int sinks,
                                const float* lse, const float* before, int64_t before_seq_stride,
                                int64_t before_head_stride, float* after, int64_t after_seq_stride,
                                int64_t after_head_stride, int64_t capacity, void* workspace, int64_t workspace_bytes,
                                void* stream);
int w4a16_kv4_attention_weights_workspace_size(const w4a16_kv4_cache* cache, int64_t T, int heads, int64_t seqs,
                                               int64_t max_q, int64_t capacity, int64_t* bytes_out);

/* Page src[i] copied to page dst[i] in every layer (pairs with a negative entry are skipped). A page
 * that is some pair's dst must be no other pair's src or dst. */
int w4a16_kv4_copy_pages(const w4a16_kv4_cache* cache, const int32_t* src, const int32_t* dst, int64_t n, void* stream);

/* Row rows[i] gets free pages (the lowest ids, in the order of the requests) up to lens[i] tokens, and
 * kv_lens[rows[i]] = lens[i]. ok[i] = 1; 0, with the row unchanged, where the free pages do not reach
 * that far down the list, the table is too narrow or lens[i] is less than the row holds. Pages that a row
 * has beyond its length (kv_lens was lowered) are used before free ones. No row twice.
 * scratch: n + 1 ints. */
int w4a16_kv4_reserve(const w4a16_kv4_tables* tables, const int32_t* rows, const int32_t* lens, int64_t n, int32_t* ok,
                      int32_t* scratch, void* stream);

/* Child row children[i] becomes a copy of sequence parents[i]: full pages are shared (refs + 1), a partly
 * filled last page is copied, in every layer, into the lowest free page. ok[i] = 0 (and an empty child)
 * where no page is free. Children hold no pages before, appear once, and are no parents. Writes the
 * tables `out` (which may be `in`). scratch: 2 n ints. */
int w4a16_kv4_fork(const w4a16_kv4_cache* cache, const w4a16_kv4_tables* in, const w4a16_kv4_tables* out,
                   const int32_t* parents, const int32_t* children, int64_t n, int32_t* ok, int32_t* scratch,
                   void* stream);

/* The rows give their pages back (refs - 1) and are empty. Writes `out` (which may be `in`). */
int w4a16_kv4_release(const w4a16_kv4_tables* in, const w4a16_kv4_tables* out, const int32_t* rows, int64_t n,
                      void* stream);

/* Rows rows[i] that hold more than `keep` tokens keep `keep` of them, in each layer and kv head on its own: the
 * first `sinks`, the last `recent`, and of the others those with the largest weights (equal ones: the lowest
 * positions; NaN: below every number), in their order, moved into fresh pages (the lowest free ids, in the order
 * of the requests; a page that other rows share stays as it is); the row's other pages are given back and kv_lens[rows[i]]
 * = keep. weights, fp32: entry (layer, row, head, token) at the three strides, `capacity` tokens contiguous; the
 * kept tokens' weights go to kept [.., keep), which is weights or shares no memory with it. ok[i] = 1; 0, with the row unchanged, where
 * the free pages do not reach that far down the list, where the row was named before, or (index flag) where it is out of
 * range or longer than `capacity`. n is at most 2^20, and n rows' pages (of `keep` tokens each) at most 2^31 - 1. Writes
 * the tables `out` (which may be `in`). scratch: w4a16_kv4_evict_scratch_ints ints. */
int w4a16_kv4_evict(const w4a16_kv4_cache* cache, const w4a16_kv4_tables* in, const w4a16_kv4_tables* out,
                    const float* weights, int64_t w_layer_stride, int64_t w_row_stride, int64_t w_head_stride, float* kept,
                    int64_t k_layer_stride, int64_t k_row_stride, int64_t k_head_stride, int64_t capacity,
                    const int32_t* rows, int64_t n, int keep, int sinks, int recent, int32_t* ok, int32_t* scratch,
                    void* stream);
int w4a16_kv4_evict_scratch_ints(const w4a16_kv4_tables* in, int64_t n, int keep, int64_t* ints_out);

/* With c pages in use, the i-th page in use with an id >= c moves to the i-th free page with an id < c, in
 * every layer, and refs and block_table follow. Writes `out` (which may be `in`). scratch: 2 * pages + 1 ints. */
int w4a16_kv4_compact(const w4a16_kv4_cache* cache, const w4a16_kv4_tables* in, const w4a16_kv4_tables* out,
                      int32_t* scratch, void* stream);

/*
 * Verification of drafted tokens (no counterpart in the reference). target [seqs, drafts + 1, vocab] and draft
 * [seqs, drafts, vocab] (null: drafts without probabilities, 1 each) hold probabilities in fp32, fp16 or bf16,
 * the last axis contiguous, strides in elements; tokens [seqs, drafts]; uniforms [seqs, drafts + 1] in [0, 1);
 * counts [seqs] or null: how many of its drafts a sequence has. Draft i is accepted while uniforms[i] * q < p. out
 * [seqs, drafts + 1]: the a accepted ones, the token drawn behind them, -1 from there on; accepted [seqs]: a. The
 * token is the first v at which the running sum of r (within 2^-45 + vocab 2^-64 of the whole) exceeds uniforms[drafts]
 * times its whole: r = max(target[a] - draft[a], 0), or target[a] where all drafts were accepted or r is nothing;
 * -1 where that is nothing too. Differences that are not finite count as nothing. kv_lens (or null): entry rows[b] of n_lens (b where rows is
 * null) is lowered by the sequence's rejected drafts. A token, count or row out of range raises the index flag: the
 * draft is rejected, the count cut to 0..drafts, the length left as it is.
 */
int w4a16_verify_drafts(const void* target, int64_t t_seq_stride, int64_t t_row_stride, const void* draft,
                        int64_t d_seq_stride, int64_t d_row_stride, int dtype, int64_t seqs, int drafts, int64_t vocab,
                        const int64_t* tokens, const float* uniforms, const int32_t* counts, int32_t* kv_lens,
                        const int32_t* rows, int64_t n_lens, int64_t* out, int32_t* accepted, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* W4A16_B200_H_ */
