/*
 * nedo_gpu.h -- C ABI of the B200 (sm_100a) matvec library, libnedo_gpu.so.
 *
 * This is the boundary that replaces the CPU hot path of nedo.cpp:
 *
 *   void nedo::kernels::matvec(const TensorInfo& t, std::span<const std::byte> bytes,
 *                              const float* x, float* y);                 kernels.hpp:20
 *   void nedo::kernels::embedding_row(const TensorInfo& t, std::span<const std::byte> bytes,
 *                                     uint32_t row, float* out);          kernels.hpp:21
 *
 * (paths relative to the nedo.cpp project: include/nedo/kernels.hpp,
 * src/kernels.cpp:162-176).  The C++ forwarding layer in
 * nedo.cpp_b200/cpp/nedo_kernels_cuda.cpp keeps those two signatures and calls
 * the host-pointer entry points below, so src/model.cpp and src/pybind.cpp
 * link unchanged.
 *
 * Conventions
 *   - `type` is the GGUF tensor type code (include/nedo/gguf.hpp:18-19):
 *     NEDO_GPU_F16 = 1, NEDO_GPU_Q4_0 = 2, NEDO_GPU_Q8_0 = 8.
 *   - A weight is `rows` rows of `cols` elements, rows contiguous; `cols` is
 *     the contiguous GGUF dimension (TensorInfo::shape[0]) and `rows` is
 *     TensorInfo::shape[1].  Row size follows tensor_nbytes
 *     (src/gguf.cpp:106-114): F16 2*cols, Q4_0 18*cols/32, Q8_0 34*cols/32.
 *   - Activations and outputs are fp32.  Batched calls use x[batch][cols] and
 *     y[batch][rows].
 *   - Every function returns 0 on success or an NEDO_GPU_ERR_* code, never
 *     throws, and leaves a message for nedo_gpu_last_error() (per thread).
 *   - `stream` is a cudaStream_t passed as void* (NULL = legacy default
 *     stream).  Pointers named *_dev must be device memory on the current
 *     CUDA device; *_host pointers are ordinary host memory.
 */
#ifndef NEDO_GPU_H
#define NEDO_GPU_H

#include <stdint.h>

#if defined(__GNUC__)
#define NEDO_GPU_API __attribute__((visibility("default")))
#else
#define NEDO_GPU_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

enum {
    NEDO_GPU_F16 = 1,
    NEDO_GPU_Q4_0 = 2,
    NEDO_GPU_Q8_0 = 8
};

enum {
    NEDO_GPU_OK = 0,
    NEDO_GPU_ERR_TYPE = 1,    /* type not supported by this entry point          */
    NEDO_GPU_ERR_ALIGN = 2,   /* Q4_0/Q8_0 column count not a multiple of 32      */
    NEDO_GPU_ERR_ROW = 3,     /* embedding row out of range                        */
    NEDO_GPU_ERR_ARG = 4,     /* null pointer, size mismatch, unsupported size     */
    NEDO_GPU_ERR_CUDA = 5,    /* CUDA runtime error (message names the call)       */
    NEDO_GPU_ERR_DEVICE = 6,  /* a kernel gave up on a bounded wait                */
    NEDO_GPU_ERR_NOMEM = 7    /* device or pinned allocation failed                */
};

/* Library version: major*10000 + minor*100 + patch. */
NEDO_GPU_API int nedo_gpu_version(void);

/* Programmatic dependent launch for the device entry points (process-wide,
 * off by default).  When on, a matvec kernel starts streaming its weight
 * while the previous kernel on the same stream is still running and reads x
 * only once that kernel has completed.  Contract: the weight must not be
 * written by the kernel launched immediately before on that stream (GGUF
 * weights are immutable).  Returns the previous setting. */
NEDO_GPU_API int nedo_gpu_set_pdl(int enable);

/* Batched calls on the exact kernels only (process-wide, off by default).
 * By default a batch of 16 or more Q8_0/Q4_0 vectors (4 or more for F16) with
 * rows of at least 1024 elements -- unless it is at most 32 vectors and one
 * launch of the exact multi-vector int8 kernel takes it whole (small
 * matrices) -- runs one tcgen05 GEMM on fp16 operands: x
 * and d*q are each rounded to fp16 once (relative error <= 2^-11 per
 * factor), products and sums are fp32.  Its worst-case error is therefore
 * about 2^-10 * sum_i |w_i x_i| per output, ten times the reference
 * tolerance of 1e-4 * sum_i |w_i x_i|, reached only when the rounding errors
 * of a row share one sign (e.g. a constant positive x against same-sign
 * weights); on independent inputs they cancel and the results stay within
 * the tolerance (tested at every benchmark shape).  When enabled, batches run
 * the int8 tensor-pipe kernels (exact integer block dots, x carried with 28
 * significant bits; up to 32 vectors per weight pass) or, for F16, one
 * streaming pass per vector: within the tolerance by bound.  Returns the
 * previous setting.  No reference counterpart. */
NEDO_GPU_API int nedo_gpu_set_exact_batches(int enable);

/* Message of the last failing call on this thread ("" if none). */
NEDO_GPU_API const char* nedo_gpu_last_error(void);

/* Bound of every spin-wait of the kernels on the current device, in
 * nanoseconds (0 restores the default of 2 s).  A wait that runs out makes
 * its kernel wind down and record the failure, which the next
 * nedo_gpu_status / host call reports as NEDO_GPU_ERR_DEVICE; the device stays
 * usable.  No reference counterpart (the reference has no device waits). */
NEDO_GPU_API int nedo_gpu_set_wait_limit_ns(uint64_t ns);

/* ---------------------------------------------------------------------------
 * Host-pointer entry points: drop-in semantics of the reference.
 *
 * Synchronous: the result is in y_host/out_host on return, like the CPU
 * kernel.  The weight bytes are uploaded to the device on first use (through
 * pinned bounce buffers) and kept resident, keyed by (w_host, w_bytes) and a
 * content fingerprint (first and last 4 KB plus 64 samples, checked on every
 * call) -- the reference passes spans into a GGUF mmap that stay valid and
 * unchanged for the model's lifetime (src/gguf.cpp:139).  A buffer freed and
 * reused at the same address with other bytes is uploaded again.  A caller
 * that rewrites a weight buffer in place where the fingerprint does not look
 * must call nedo_gpu_weight_evict() first.  Calls are serialised per device.
 * ------------------------------------------------------------------------- */

/* Replaces nedo::kernels::matvec (src/kernels.cpp:162-169):
 *   y_host[r] = sum_i dequant(w)[r][i] * x_host[i], r < rows.
 * Errors mirror the reference: a Q4_0/Q8_0 column count that is not a
 * multiple of 32 ("... elements not block aligned", src/gguf.cpp:109-110),
 * an unsupported type ("matvec tensor type not supported", src/kernels.cpp:168).
 * w_bytes must be at least rows * row_bytes. */
NEDO_GPU_API int nedo_gpu_matvec(uint32_t type, uint64_t rows, uint64_t cols, const void* w_host, uint64_t w_bytes,
                    const float* x_host, float* y_host);

/* `batch` calls of nedo_gpu_matvec over one weight in one call:
 * y_host[b][r] = dot(row r, x_host[b]), b < batch (x_host [batch][cols],
 * y_host [batch][rows]).  Replaces the reference's prompt loop, one matvec per
 * token for every weight (src/model.cpp:262-266, the forward lambda at
 * :212-260), with one pass over the weight; the kernel choice is that of
 * nedo_gpu_matvec_dev with the same batch.  Errors as nedo_gpu_matvec. */
NEDO_GPU_API int nedo_gpu_matvec_batch(uint32_t type, uint64_t rows, uint64_t cols, const void* w_host,
                                       uint64_t w_bytes, const float* x_host, float* y_host, uint32_t batch);

/* Replaces nedo::kernels::embedding_row (src/kernels.cpp:170-176): writes the
 * dequantised row `row` (cols floats) to out_host, bit-identical to the
 * reference.  row >= rows -> NEDO_GPU_ERR_ROW ("bad embedding row"). */
NEDO_GPU_API int nedo_gpu_embedding_row(uint32_t type, uint64_t rows, uint64_t cols, const void* w_host, uint64_t w_bytes,
                           uint32_t row, float* out_host);

/* Upload (or find) the resident device copy of a host weight buffer.
 * *w_dev_out receives the device pointer (valid until evicted). */
NEDO_GPU_API int nedo_gpu_weight_upload(const void* w_host, uint64_t w_bytes, const void** w_dev_out);
/* Drop the resident copy of w_host (no-op if absent). */
NEDO_GPU_API int nedo_gpu_weight_evict(const void* w_host);
/* Drop every resident weight on every device this library touched, and free
 * the batched-call buffers that larger calls replaced (a CUDA graph captured
 * with one of those is invalid afterwards). */
NEDO_GPU_API int nedo_gpu_cache_clear(void);

/* ---------------------------------------------------------------------------
 * Device-pointer entry points (asynchronous on `stream`).
 * ------------------------------------------------------------------------- */

/* The matvec of nedo_gpu_matvec on device buffers, for `batch` activation
 * vectors: y_dev[b][r] = dot(row r, x_dev[b]), b < batch.  batch == 1 is the
 * decode path (src/model.cpp:217-259); batch > 1 replaces `batch` serial
 * calls over the same weight, which is how the reference processes a prompt
 * (src/model.cpp:262-266).  Q8_0/Q4_0 batches of 2 to 15 vectors, and of up
 * to 32 that one launch takes whole, run the exact multi-vector int8 kernel
 * (each weight tile read once per launch for all its vectors).  Otherwise,
 * for rows of at least 1024 elements, from 16 vectors on (4 for F16 weights)
 * the batch runs as one tensor-core GEMM with x and the dequantised weight
 * rounded to fp16 (fp32 accumulation).  The GEMM calls
 * calls use two per-device buffers (an fp16 copy of x and, for few row tiles,
 * a split-K workspace), allocated by the first call that needs them and grown
 * by a larger one.  A grown-out buffer stays allocated until
 * nedo_gpu_cache_clear, so a CUDA graph captured earlier keeps working.  To
 * capture such a call in a graph, size the buffers first, outside capture,
 * with nedo_gpu_reserve (or one eager call of the largest shape): a call that
 * has to allocate cannot be captured.  Calls on one device share the buffers:
 * serialise calls that may overlap (other streams, other threads). */
NEDO_GPU_API int nedo_gpu_matvec_dev(uint32_t type, uint64_t rows, uint64_t cols, const void* w_dev, const float* x_dev,
                        float* y_dev, uint32_t batch, void* stream);

/* Size the per-device buffers of a batched nedo_gpu_matvec_dev call of this
 * shape (no-op for shapes that need none), so that the call itself allocates
 * nothing and can be captured in a CUDA graph.  Call outside stream capture.
 * No reference counterpart. */
NEDO_GPU_API int nedo_gpu_reserve(uint32_t type, uint64_t rows, uint64_t cols, uint32_t batch);

/* matvec followed by the greedy pick of the LM head (std::max_element over
 * the logits, src/model.cpp:36: first index of the maximum), fused into the
 * matvec kernel where the shape allows.  y_dev receives the logits;
 * index_dev (int64) the argmax; value_dev (may be NULL) its value.  Uses a
 * per-device scratch area: calls that overlap on the GPU must not share a
 * device. */
NEDO_GPU_API int nedo_gpu_matvec_argmax_dev(uint32_t type, uint64_t rows, uint64_t cols, const void* w_dev, const float* x_dev,
                               float* y_dev, int64_t* index_dev, float* value_dev, void* stream);

/* argmax of an fp32 vector in device memory (first index of the maximum).
 * NaN behaves as in std::max_element: a NaN never wins, except that a NaN at
 * index 0 makes the result 0 (every comparison with it is false); this holds
 * for every argmax entry point. */
NEDO_GPU_API int nedo_gpu_argmax_dev(const float* v_dev, uint64_t n, int64_t* index_dev, float* value_dev, void* stream);

/* nedo_gpu_argmax_dev without any allocation: the same kernel and result,
 * with its per-CTA candidates and completion counter in a fixed 8448-byte
 * __device__ array of the library (room for 1024 CTAs; a launch needing more
 * returns NEDO_GPU_ERR_ARG) instead of the per-device scratch that the other
 * entry points allocate on first use.  No reference counterpart: the
 * reference picks the token on the host (std::max_element, src/model.cpp:36).
 * The first call on a device resolves the array's address; make it outside
 * stream capture.  Calls that may overlap on one device (other streams, other
 * threads) share the array and race: serialise them. */
NEDO_GPU_API int nedo_gpu_argmax_dev_noalloc(const float* v_dev, uint64_t n, int64_t* index_dev, float* value_dev,
                                void* stream);

/* The k largest elements of an fp32 vector in device memory, largest first
 * (equal values: smaller index first; NaN never ahead of a number):
 * ids_dev[0..k) (uint32) and vals_dev[0..k) (may be NULL).  1 <= k <= 256 and
 * k <= n.  This is the candidate selection of the reference's sampler
 * (sample_token, src/model.cpp:38-44: nth_element + sort by logit), done where
 * the logits are.  Uses a per-device scratch area: calls that overlap on the
 * GPU must not share a device. */
NEDO_GPU_API int nedo_gpu_topk_dev(const float* v_dev, uint64_t n, uint32_t k, uint32_t* ids_dev, float* vals_dev,
                                   void* stream);

/* Host-pointer LM head (the matvec of src/model.cpp:259, nedo_gpu_matvec's
 * residency and errors) followed by the top k logits (nedo_gpu_topk_dev), with
 * only the k (id, logit) pairs copied back instead of all `rows` logits:
 * ids_host[0..k), vals_host[0..k) (may be NULL).  1 <= k <= min(rows, 256). */
NEDO_GPU_API int nedo_gpu_lm_head_topk(uint32_t type, uint64_t rows, uint64_t cols, const void* w_host,
                                       uint64_t w_bytes, const float* x_host, uint32_t k, uint32_t* ids_host,
                                       float* vals_host);

/* Host-pointer LM head with the greedy pick (src/model.cpp:36, std::max_element
 * semantics as nedo_gpu_argmax_dev), fused into the matvec where the shape
 * allows: *index_host, *value_host (may be NULL); no logits are copied back. */
NEDO_GPU_API int nedo_gpu_lm_head_argmax(uint32_t type, uint64_t rows, uint64_t cols, const void* w_host,
                                         uint64_t w_bytes, const float* x_host, int64_t* index_host,
                                         float* value_host);

/* Row-sharded matvec with the all-gather of y fused into it (one process
 * per GPU; rows are independent, src/kernels.cpp:166-168).  Computes this
 * rank's rows into y_dev like nedo_gpu_matvec_dev and also stores each row at
 * peer_y[k] + row_offset + r on every peer k (peer device addresses, e.g. from
 * CUDA IPC or symmetric memory, reachable over NVLink), then adds 1 per CTA to
 * each peer's 32-bit word peer_signal[k].  Q8_0 / Q4_0 shapes of the int8
 * tensor-pipe kernel only (plan_info path 4); at most 7 peers.  A receiver
 * calls nedo_gpu_allgather_wait_dev before reading the gathered y.  No
 * reference counterpart: the reference runs on one CPU. */
NEDO_GPU_API int nedo_gpu_matvec_allgather_dev(uint32_t type, uint64_t rows, uint64_t cols, const void* w_dev,
                                  const float* x_dev, float* y_dev, const uint64_t* peer_y,
                                  const uint64_t* peer_signal, uint32_t npeers, uint64_t row_offset, void* stream);

/* Wait on `stream` (one GPU thread, bounded by nedo_gpu_set_wait_limit_ns, 2 s
 * by default; a timeout sets the status word read by nedo_gpu_status) until
 * *signal_dev has advanced by `increment` (peers x CTAs of their launches)
 * past *expected_dev, then advance *expected_dev by `increment` -- also after
 * a timeout, so that signals of a late step are never counted for the next
 * one.  After NEDO_GPU_ERR_DEVICE the gathered rows of that step are invalid;
 * later steps are correct once the late peer has caught up.  Both words start
 * at zero; the caller keeps them per receiving buffer. */
NEDO_GPU_API int nedo_gpu_allgather_wait_dev(uint32_t* signal_dev, uint32_t* expected_dev, uint32_t increment,
                                void* stream);

/* embedding_row for rows [row_begin, row_begin + row_count) into
 * out_dev[row_count][cols]; bit-identical to the reference. */
NEDO_GPU_API int nedo_gpu_dequant_rows_dev(uint32_t type, uint64_t rows, uint64_t cols, const void* w_dev, uint64_t row_begin,
                              uint64_t row_count, float* out_dev, void* stream);

/* Wait for `stream`, then report (and clear) device-side failures recorded
 * by kernels on the current device since the last check. */
NEDO_GPU_API int nedo_gpu_status(void* stream);

/* Describe the kernel choice for a shape: out[0] = path (1 streaming CUDA-core,
 * 2 generic, 3 batched streaming (one launch per vector), 4 int8 tensor-pipe
 * matvec, 5 tcgen05 GEMM over the batch), out[1] grid,
 * out[2] threads, out[3] dynamic shared bytes, out[4] rows per tile,
 * out[5] ring slots (path 5: K splits per tile, > 1 adding a fold kernel),
 * out[6] slot bytes, out[7] warps per CTA (compute warps for path 4),
 * out[8] (when n > 8) kernels one call launches.  Path 4 with several vectors
 * describes the first launch.  n = capacity of out (>= 8). */
NEDO_GPU_API int nedo_gpu_plan_info(uint32_t type, uint64_t rows, uint64_t cols, uint32_t batch, uint32_t* out, int n);

/* ---- Device-resident decode forward pass -------------------------------
 *
 * Replaces the `forward` step of NedoModel::generate_ids (src/model.cpp:212-260):
 * embedding row, then per layer RMSNorm, q/k/v projections, RoPE, the KV-cache
 * write, attention over the sliding window, the output projection and residual,
 * RMSNorm, gate/up projections, SiLU gate (with the MorphFFN masking of the
 * trailing layers, :196-209), the down projection and residual; then the final
 * RMSNorm and the LM-head matvec.  Weights and the fp32 KV cache stay on the
 * device; one call runs the whole pass as one CUDA graph (captured on the first
 * call, the token and position read from device memory) and returns the greedy
 * pick and, on request, the logits.
 *
 * The configuration mirrors ModelConfig (include/nedo/model.hpp:12-16). */
typedef struct {
    uint32_t vocab, dim, layers, heads, kv_heads, head_dim, ffn, context, sliding;
    uint32_t morph_layers, morph_shared, morph_root, morph_suffix;
    float rms_eps, rope_theta;
} nedo_gpu_decoder_config;

/* One GGUF tensor: TensorInfo's type and shape (contiguous dimension first)
 * and a host view of its bytes (e.g. GgufFile::bytes, src/gguf.cpp:139). */
typedef struct {
    uint32_t type;
    uint32_t ndims;
    uint64_t shape[2];
    const void* data;
    uint64_t nbytes;
} nedo_gpu_tensor_view;

/* Tensor order of nedo_gpu_decoder_create:
 *   [0] token_embd (F16 / Q8_0 / Q4_0), [1] output_norm (F32 / F16),
 *   [2] output (F16 / Q8_0 / Q4_0; data NULL: the head is token_embd),
 *   [3] blk.0.ffn_gate_tid2eid, the MorphFFN routing table (F32 [2, vocab];
 *       data NULL: none),
 *   then 9 per layer: attn_norm, attn_q, attn_k, attn_v, attn_output, ffn_norm,
 *   ffn_gate, ffn_up, ffn_down (norms F32 / F16, projections F16 / Q8_0 / Q4_0;
 *   q, k, v of one type, gate and up of one type).
 * Shape and type checks follow the reference: "invalid GQA dimensions"
 * (heads % kv_heads, dim == heads * head_dim), "context_length is zero",
 * "MorphFFN widths do not sum to feed_forward_length", and every tensor's
 * shape against the configuration.  The weights are copied to the device; the
 * host views may be released afterwards. */
typedef struct nedo_gpu_decoder nedo_gpu_decoder;
NEDO_GPU_API int nedo_gpu_decoder_create(const nedo_gpu_decoder_config* cfg, const nedo_gpu_tensor_view* tensors,
                                         uint64_t ntensors, nedo_gpu_decoder** out);

/* One forward pass for `token` at position `pos` (positions from 0, one per
 * call, as generate_ids: the KV-cache slot is pos % window with window =
 * min(sliding ? sliding : context, context)).  *argmax_out (if non-null) gets
 * the greedy pick (std::max_element semantics: first index of the maximum);
 * logits_host (if non-null) gets the vocab logits.  token >= vocab
 * ("prompt token id out of range") and pos >= context are NEDO_GPU_ERR_ARG. */
NEDO_GPU_API int nedo_gpu_decoder_forward(nedo_gpu_decoder* d, uint32_t token, uint64_t pos, float* logits_host,
                                          uint32_t* argmax_out);

/* Greedy generation with the loop on the device: n passes, the first for
 * `token` at `pos`, each next pass fed the previous pass's greedy pick; the
 * picks go to ids_host[0..n) (ids_host[k] is the pick of pass k).  Equivalent
 * to n forward calls with temperature-0 sampling between them
 * (src/model.cpp:271-279) but without a host round trip per token: the n
 * passes are launched back to back and the ids read once.  The eos id does
 * not stop the device loop (the caller truncates at it); pos + n <= context. */
NEDO_GPU_API int nedo_gpu_decoder_generate(nedo_gpu_decoder* d, uint32_t token, uint64_t pos, uint32_t n,
                                           uint32_t* ids_host);

/* Run the passes on `stream` (a cudaStream_t; NULL returns to the decoder's
 * own stream).  The captured graphs are dropped and captured again on the
 * next calls.  Every forward call still waits for its pass to finish. */
NEDO_GPU_API int nedo_gpu_decoder_set_stream(nedo_gpu_decoder* d, void* stream);

/* The logits of the last forward pass in device memory (valid until the next
 * call), for the sampler entry points (nedo_gpu_topk_dev). */
NEDO_GPU_API int nedo_gpu_decoder_logits_dev(nedo_gpu_decoder* d, const float** logits_dev);

/* Zero the KV cache (a new sequence starts at pos 0 either way). */
NEDO_GPU_API int nedo_gpu_decoder_reset(nedo_gpu_decoder* d);

/* Free the decoder's device memory and graphs (NULL is a no-op). */
NEDO_GPU_API void nedo_gpu_decoder_destroy(nedo_gpu_decoder* d);

/* ---- Paged key/value cache of many sequences ----------------------------
 *
 * Device entry points for serving a batch of sequences: a cache of pages that a
 * page table deals out to the sequences, the append that fills it, and the
 * attention that reads it.  They stand next to nedo_gpu_matvec_dev (batch > 1)
 * as its single-sequence counterparts inside nedo_gpu_decoder stand next to the
 * matvec: q|k|v of a batch comes from one nedo_gpu_matvec_dev, goes through
 * nedo_gpu_kv_append_dev, and the attention output goes into the output
 * projection.  The arithmetic is that of src/model.cpp:218-247 and
 * src/kernels.cpp:93-105 per sequence, but for the rotation's angles: append forms
 * them in 64 bits, the decode pass in 32 as the reference does, so at far positions
 * p the keys differ by a turn of up to p * 2^-24 radians, and a cache is continued by
 * the one that began it.  Pages, ragged batches, shared prefixes and page selection
 * have no reference counterpart.
 *
 * All of them are asynchronous on `stream`, allocate nothing and keep nothing
 * between calls, so they can be captured in CUDA graphs and may run at the same
 * time on several streams (each call with a workspace of its own; captured graphs
 * that may overlap too).  The library's first call on a device allocates its state
 * there: make it outside a capture.  Buffers are 16-byte aligned memory of the
 * current device (lists of uint32: 4-byte).  Results repeat bit for bit.
 *
 * Token row t of sequence s (q_start[s] <= t < q_start[s+1]) stands at position
 * kv_len[s] - (q_start[s+1] - t).  A row whose position is negative -- its
 * sequence has fewer cached tokens than rows, e.g. an unused slot of a padded
 * batch with kv_len 0 -- is padding: append writes nothing for it, attention
 * gives it zeros.  Rows from q_start[seqs] on belong to no sequence; their
 * outputs are left as they were.
 *
 * Lengths and page ids are read from device memory.  A sequence whose values are
 * out of range (rows beyond `tokens` or `max_q_len`, more than `max_kv_len`
 * cached tokens, decreasing q_start) is left out, a page id of num_pages or more
 * counts as a page without keys, and either is reported by nedo_gpu_status as
 * NEDO_GPU_ERR_DEVICE. */
typedef struct {
    uint32_t type;       /* 0 (F32), NEDO_GPU_F16 or NEDO_GPU_Q4_0 (see below)            */
    uint32_t kv_heads;
    uint32_t head_dim;   /* a multiple of 8 (Q4_0: of 32), at most 256                   */
    uint32_t page_size;  /* tokens per page: 16, 32, 64, 128 or 256                      */
    uint64_t num_pages;  /* num_pages * kv_heads below 2^31                              */
    void* k;             /* [num_pages][kv_heads][page_size][head_dim]                   */
    void* v;             /* [num_pages][kv_heads][page_size][head_dim]                   */
    void* bounds;        /* [num_pages][kv_heads][2][head_dim], in `type` (Q4_0: in F16): the
                            smallest and the largest value of each channel of the page's keys,
                            as nedo_gpu_kv_append_dev keeps them (NULL: not kept;
                            nedo_gpu_block_select_dev needs it)                            */
} nedo_gpu_kv_cache;

typedef struct {
    uint32_t seqs;               /* sequences                                            */
    uint32_t tokens;             /* rows of the q, qkv and output buffers                */
    uint32_t max_q_len;          /* no sequence has more rows (a bound, at least 1; shapes the
                                    launch)                                               */
    uint32_t max_kv_len;         /* no sequence has more cached tokens (a bound)          */
    uint32_t max_pages;          /* row length of page_table                             */
    uint32_t shared_pages;       /* paged attention: the first shared_pages entries of every
                                    row of page_table are the same pages (0: none shared);
                                    they are read from the first row, used or not         */
    const uint32_t* q_start;     /* device, [seqs + 1]: first token row of each sequence  */
    const uint32_t* kv_len;      /* device, [seqs]: cached tokens, this call's included   */
    const uint32_t* page_table;  /* device, [seqs][max_pages]; entries behind a sequence's
                                    last page, or in front of its window, are not read    */
} nedo_gpu_kv_batch;

/* A cache of type NEDO_GPU_Q4_0 holds 4-bit numbers: 18 bytes for 32 channels of a token,
 * as in a GGUF tensor, with the same meaning, value = d * (n - 8) for n in 0..15 and an fp16
 * scale d, but laid out by pages: k and v are
 * [num_pages][kv_heads][page_size * head_dim / 32 * 18 bytes], of which the first
 * page_size * head_dim / 2 are the numbers, [page_size][head_dim / 8] words of 32 bits
 * (channel 8 w + j of a token: the four bits from bit 2 j on of word w for an even j, from
 * bit 14 + 2 j for an odd one), and the rest the scales, [head_dim / 32][page_size].  Append
 * makes a block of 32 channels so, in 64 bits and without other rounding:
 *   x: its number of largest magnitude (the negative one where both signs have it);
 *   d = -x / 8 to the nearest number of eight significant bits (equally near: the even one), in
 *       steps of no less than 2^-24, its magnitude at most 8160;
 *   n = floor(value / d + 8.5), at least 0 and at most 15; 8 where d is 0.
 * A block with a number that is not finite gets the scale NaN: all its values are NaN.  With
 * such scales every value is an F16 number; with others a caller may have put there (d as
 * GGUF's quantiser rounds it), it is the product rounded to F16. */

/* The new tokens of a batch: rotates queries and keys to their positions and
 * writes keys and values into the cache.  qkv_dev holds `tokens` rows of
 * heads * head_dim query, kv_heads * head_dim key and as many value elements (the
 * decoder's q|k|v layout; an F16 cache gets them rounded to nearest, above 65504 as
 * infinities); the rotated queries go to q_out_dev
 * [tokens][heads][head_dim], which must not overlap qkv_dev.  Channels i and
 * i + head_dim/2 turn by position * rope_theta^(-2i/head_dim), the angle in 64
 * bits; rope_theta 0: no rotation.  With cache->bounds, the channel bounds of every
 * page written are brought up to date: the range of the keys stored since the
 * page's first slot was last written (NaN keys left out), those included that have been
 * written over since, as rejected drafts are, or that lie behind a length taken back. */
NEDO_GPU_API int nedo_gpu_kv_append_dev(const nedo_gpu_kv_cache* cache, const nedo_gpu_kv_batch* batch,
                                        uint32_t heads, const float* qkv_dev, float rope_theta, float* q_out_dev,
                                        void* stream);

/* The keys (rotated) and values that the cache holds for a batch's token rows, in 32 bits:
 * k_out_dev and v_out_dev [tokens][kv_heads][head_dim], which overlap neither each other nor
 * anything that is read; for moving sequences to other pages or another type of cache (kv_append
 * with rope_theta 0 takes them), and for looking at them.  Padding rows get zeros, and so do those
 * on a page id of num_pages or more; rows of no sequence are left as they were. */
NEDO_GPU_API int nedo_gpu_kv_read_dev(const nedo_gpu_kv_cache* cache, const nedo_gpu_kv_batch* batch, float* k_out_dev,
                                      float* v_out_dev, void* stream);

/* Bytes of workspace that nedo_gpu_paged_attention_dev needs for these sizes
 * (possibly 0).  Reads no device memory and needs no device. */
NEDO_GPU_API int nedo_gpu_paged_attention_workspace(const nedo_gpu_kv_cache* cache, const nedo_gpu_kv_batch* batch,
                                                    uint32_t heads, uint32_t window, uint64_t* bytes);

/* Attention of every query row over its sequence's cached tokens, itself
 * included: q_dev and out_dev [tokens][heads][head_dim] (not overlapping),
 *   out = sum_j softmax_j(scale * q.k_j) v_j,  max(0, p - window + 1) <= j <= p
 * for a row at position p (window 0: all).  With shared_pages > 0 the keys of the
 * shared prefix are read once for the whole batch.  Sums and softmax statistics
 * are kept in 32 bits.  The factors of the tensor cores' products -- queries and
 * softmax weights, and the keys and values of an F32 cache where a sequence (or, over a
 * shared prefix, the batch) has more than 16 rows, tokens times heads per KV head -- keep
 * 22 bits down to 2^-27 of the largest number they share a scale with (a row's query
 * channels; a row's weights; 32 or 64 neighbouring keys or values), and 2^-49 of that
 * below.  Fewer rows on an F32 cache are computed in 32 bits throughout.
 *
 * Infinities (an F16 cache holds what is above 65504 as one) count as they do in the
 * formula: a key whose score is -infinity has no weight, one whose score is +infinity
 * makes its rows NaN, and an infinite value gives that infinity to its channel of every
 * row that sees it, or NaN where its weight is below 2^-126 of the row's largest.  Rows
 * whose sums are not finite are formed twice on F16 and Q4_0 caches, the second time key by
 * key: right, but slow. */
NEDO_GPU_API int nedo_gpu_paged_attention_dev(const nedo_gpu_kv_cache* cache, const nedo_gpu_kv_batch* batch,
                                              uint32_t heads, const float* q_dev, float* out_dev, float scale,
                                              uint32_t window, void* workspace_dev, uint64_t workspace_bytes,
                                              void* stream);

/* For every query row and KV head, the `picks` (1..1024) pages whose keys can
 * score highest: blocks_dev [tokens][kv_heads][picks] receives logical page
 * numbers (indexes into the sequence's row of page_table) in ascending order,
 * 0xFFFFFFFF behind the last.  The page of the row's own position is always among
 * them; the others, of those before it, by
 *   score = sum_d (hi_d * sum_g max(q_gd, 0) + lo_d * sum_g min(q_gd, 0))
 * with the page's bounds lo, hi and the KV head's query heads g, summed in 64 bits
 * (equal scores: the lower page; NaN last).  At most 16384 pages per sequence. */
NEDO_GPU_API int nedo_gpu_block_select_dev(const nedo_gpu_kv_cache* cache, const nedo_gpu_kv_batch* batch,
                                           uint32_t heads, const float* q_dev, uint32_t picks, uint32_t* blocks_dev,
                                           void* stream);

/* Bytes of workspace that nedo_gpu_block_attention_dev needs for these sizes. */
NEDO_GPU_API int nedo_gpu_block_attention_workspace(const nedo_gpu_kv_cache* cache, const nedo_gpu_kv_batch* batch,
                                                    uint32_t heads, uint32_t picks, uint64_t* bytes);

/* Attention of every query row over the cached tokens, up to itself, of the pages
 * listed for it and the KV head (blocks_dev as nedo_gpu_block_select_dev writes
 * it; shared_pages is not used).  An entry counts when it is above every entry
 * before it and not beyond the row's own page; others are passed over. */
NEDO_GPU_API int nedo_gpu_block_attention_dev(const nedo_gpu_kv_cache* cache, const nedo_gpu_kv_batch* batch,
                                              uint32_t heads, const float* q_dev, const uint32_t* blocks_dev,
                                              uint32_t picks, float* out_dev, float scale, void* workspace_dev,
                                              uint64_t workspace_bytes, void* stream);

/* ---- Drafted tokens ------------------------------------------------------
 *
 * The sampling step of a batch whose sequences try several tokens at a time: somebody -- a
 * smaller model, a table of earlier text -- has drafted the next tokens of a sequence, one pass
 * over the sequence's last token and its drafts has given the target's logits behind each of
 * them (paged attention takes the rows of a sequence together), and this call says how many of
 * the drafts stand and which token follows.  With random numbers that are uniform and
 * independent, the tokens are distributed as if each had been sampled from the target.  Without
 * drafts (one row per sequence) it samples a token for each.  The reference samples one token of
 * one sequence on the host (sample_token, src/model.cpp:31-53).
 *
 * Row i of sequence s (row_start[s] + i, i below its n rows) has the target's logits behind the
 * sequence's i-th draft, row 0 those behind what was there before.  draft_ids[row] is the token drafted
 * to follow the row; that of a sequence's last row is not read. */
typedef struct {
    uint32_t seqs;
    uint32_t rows;              /* of logits, draft_ids, draft_probs, accept_u and ids           */
    uint32_t max_rows;          /* no sequence has more rows (1..256)                             */
    uint32_t vocab;
    const uint32_t* row_start;  /* device, [seqs + 1]: first row of each sequence                 */
    const float* logits;        /* device, [rows][vocab]                                          */
    const uint32_t* draft_ids;  /* device, [rows]; may be NULL where max_rows is 1                */
    const float* draft_probs;   /* device, [rows][vocab]: the probabilities that a row's draft was drawn
                                   from; NULL: drafts that were certain                           */
    const float* accept_u;      /* device, [rows]: numbers in [0, 1); may be NULL where max_rows is 1 or the
                                   temperature 0                                                  */
    const float* sample_u;      /* device, [seqs]: numbers in [0, 1); may be NULL for temperature 0 */
} nedo_gpu_drafts;

/* Bytes of workspace that nedo_gpu_verify_drafts_dev needs for these sizes.  Reads no device memory. */
NEDO_GPU_API int nedo_gpu_verify_drafts_workspace(const nedo_gpu_drafts* drafts, uint64_t* bytes);

/* accepted_dev [seqs]: how many of a sequence's drafts stand; ids_dev [rows]: they, the token
 * that follows, and 0xFFFFFFFF behind it.  With p = softmax(logits / temperature) and q the draft's
 * probabilities (1 for a certain draft), a draft x of a row stands where all before it do and
 *   accept_u * q(x) < p(x),
 * and the following token is drawn from max(p - q, 0) of the row of the first draft that does
 * not stand (from p, where that leaves nothing), or from p of the last row: the first token at
 * which the running sum passes sample_u times the whole sum.  Temperature 0: a draft stands where
 * it is the first of the largest logits, which is also the token that follows.  Other
 * temperatures: 1e-6 to 1e6.
 *
 * NaN logits count as minus infinity, infinite ones as the largest number; a row of nothing but
 * minus infinity gives no token (0xFFFFFFFF), and no draft stands on it.  NaN and negative draft
 * probabilities count as 0.  The decisions are those of 64-bit arithmetic, in which tokens below
 * 2^-500 of a row's largest have no weight: sums in 32 bits decide only where their error cannot.
 *
 * A sequence whose rows are out of range (decreasing, beyond `rows`, more than max_rows) is left
 * out, a draft that is no token (vocab or more) does not stand, and either is reported by
 * nedo_gpu_status.  Rows of no sequence are left as they were.  Asynchronous on `stream`, without
 * allocations; calls that overlap need workspaces of their own.  logits, draft_probs and the
 * workspace are 16-byte aligned; the results and the workspace overlap neither each other nor anything
 * that is read. */
NEDO_GPU_API int nedo_gpu_verify_drafts_dev(const nedo_gpu_drafts* drafts, float temperature, uint32_t* accepted_dev,
                                            uint32_t* ids_dev, void* workspace_dev, uint64_t workspace_bytes,
                                            void* stream);

#ifdef __cplusplus
}
#endif
#endif /* NEDO_GPU_H */
