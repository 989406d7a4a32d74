/*
 * rq.h -- C ABI of librq, the B200 (sm_100a) quantized-linear and sparse-MoE
 * library behind rustyllm's q4_kernel / StreamingLlamaQuantized /
 * StreamingMixtral APIs.
 *
 * Conventions
 *   - Every entry point returns int: RQ_OK (0) on success, otherwise an
 *     RQ_ERR_* code; rq_last_error() then returns a thread-local message.
 *     This maps onto the reference's `Error::Msg(String)` (src/error.rs:4-29)
 *     the way q4_kernel.rs:90-107 builds its messages.  Nothing aborts.
 *   - Weights are GGML block bytes exactly as they sit in a GGUF tensor
 *     (Q4_0 = 18-byte blocks of 32, Q4_K = 144-byte super-blocks of 256,
 *     Q3_K = 110-byte super-blocks of 256; also Q8_0 = 34 / 32, Q6_K = 210,
 *     Q5_K = 176 and Q2_K = 84 bytes per 256), row-major [out][in/block].
 *     The library copies them to the GPU and owns the device copy.
 *   - `stream` is a cudaStream_t passed as void* (NULL = legacy stream).
 *   - Activation pointers (x, y) may be host or device memory.  Page-locked
 *     host memory (cudaHostAlloc / cudaHostRegister) is used in place: the
 *     kernels read x and write y over the bus.  Pageable host memory is
 *     staged through device memory.  With any host pointer the call returns
 *     with y filled and x no longer read; with device pointers only it is
 *     asynchronous on `stream`.
 *   - One rq_ctx per device; calls on one ctx are serialised by the caller
 *     (the reference's single-writer generate loop,
 *     src/streaming_quantized.rs:345-351).  Weight handles are read-only
 *     during forward calls and may be shared between threads.
 */
#ifndef RQ_H
#define RQ_H

#include <stddef.h>
#include <stdint.h>

#if defined(_WIN32)
#define RQ_API
#else
#define RQ_API __attribute__((visibility("default")))
#endif

#ifdef __cplusplus
extern "C" {
#endif

typedef struct rq_ctx rq_ctx;
typedef struct rq_weight rq_weight;
typedef struct rq_moe rq_moe;

enum rq_status {
    RQ_OK = 0,
    RQ_ERR_INVALID = 1,     /* bad argument, shape or type */
    RQ_ERR_CUDA = 2,        /* CUDA runtime error */
    RQ_ERR_UNSUPPORTED = 3, /* valid request the library does not implement */
    RQ_ERR_OOM = 4,         /* device allocation failed */
    RQ_ERR_TIMEOUT = 5,     /* a bounded device or host wait gave up */
    RQ_ERR_NCCL = 6         /* collective failed */
};

/* GGML type ids (ggml_type / candle GgmlDType numbering). */
enum rq_ggml_type { RQ_Q4_0 = 2, RQ_Q8_0 = 8, RQ_Q2_K = 10, RQ_Q3_K = 11, RQ_Q4_K = 12, RQ_Q5_K = 13, RQ_Q6_K = 14 };

/* ---------------------------------------------------------------- context */

/* Create a context on CUDA device `device`.  Replaces the implicit candle
 * Device::Cuda(n) of src/inference.rs:56-70. */
RQ_API int rq_init(int device, rq_ctx** out);
RQ_API int rq_destroy(rq_ctx* ctx);

/* Copy the calling thread's last error message into buf (NUL-terminated,
 * truncated to n).  Returns the full message length. */
RQ_API int rq_last_error(char* buf, size_t n);

/* Synchronise the context's device and report whether a bounded wait
 * (mbarrier or peer flag, ~1 s) inside a kernel of an asynchronous call on
 * this context -- or of rq_linear_noalloc on this device -- gave up since the
 * last check: RQ_ERR_TIMEOUT (record cleared; the outputs of those calls are
 * incomplete), else RQ_OK.  Calls with host buffers check this themselves
 * before they return.  No reference counterpart (candle's CPU kernels cannot
 * time out). */
RQ_API int rq_ctx_status(rq_ctx* ctx);

/* "rq <version> sm_100a" */
RQ_API const char* rq_version(void);

/* Bytes / elements per GGML block; 0 for an unknown type. */
RQ_API size_t rq_block_bytes(int ggml_type);
RQ_API int rq_block_elems(int ggml_type);

/* ---------------------------------------------------------------- weights */

/* Upload GGML blocks [out][in/block] (host or device pointer, nbytes must be
 * exactly out*in/block*block_bytes).  Replaces QMatMul::from_arc over a
 * GgufLayer tensor (src/streaming_quantized.rs:63-70) and
 * ParallelQ4Linear::from_qtensor (src/q4_kernel.rs:89-171); in must be a
 * multiple of the block size (src/q4_kernel.rs:104-108). */
RQ_API int rq_weight_upload(rq_ctx* ctx, int ggml_type, const void* blocks, size_t nbytes,
                     int64_t out, int64_t in, rq_weight** w);

/* Quantize an f32 matrix [out][in] that is already on this device straight
 * into a device weight (no host round trip); the call returns once the
 * weight is written.  Q4_0 follows the rule of
 * src/q4_kernel.rs:137-163, Q8_0 GGML's rounding rule; the K-types use
 * librq's deterministic quantizers
 * (the counterpart of candle's QTensor::quantize, src/quantize.rs:131). */
RQ_API int rq_weight_quantize(rq_ctx* ctx, int ggml_type, const float* w_dev, int64_t out, int64_t in,
                       rq_weight** w, void* stream);

/* Copy a device weight back as GGML blocks into host memory. */
RQ_API int rq_weight_download(rq_ctx* ctx, const rq_weight* w, void* blocks_host, size_t nbytes);

RQ_API int rq_weight_free(rq_ctx* ctx, rq_weight* w);

/* Any of the out-pointers may be NULL.  device_bytes counts the library's
 * device copy: the GGML byte count, plus 2 pad bytes per Q6_K super-block;
 * Q3_K is held expanded (4-bit values and int8 scales, 148 bytes per
 * 110-byte super-block) so that its matvec is not bound by unpacking. */
RQ_API int rq_weight_info(const rq_weight* w, int* ggml_type, int64_t* out, int64_t* in,
                   size_t* device_bytes);

/* y[out][in] = dequantized weight in f32, bit-identical to GGML's dequant
 * (QTensor::dequantize, used at src/q4_kernel.rs:120-122). */
RQ_API int rq_dequantize(rq_ctx* ctx, const rq_weight* w, float* y, void* stream);

/* ----------------------------------------------------------------- linear */

/* y[M][out] = x[M][in] * W^T in f32.  Replaces QMatMul::forward
 * (src/streaming_quantized.rs:201-203,256,277-278) and
 * ParallelQ4Linear::forward (src/q4_kernel.rs:183-256).  M=1 is the decode
 * matvec; M=K+1 the speculative verify (examples/spec_decode_70b.rs:238);
 * larger M the prefill (src/streaming_quantized.rs:569-575). */
RQ_API int rq_linear(rq_ctx* ctx, const rq_weight* w, const float* x, float* y, int64_t M,
              void* stream);

/* n (1..8) independent decode matvecs y_i[1][out_i] = x_i[1][in] * W_i^T in
 * one launch, for weights of the same type and in_features -- the q/k/v
 * projections of QAttn::forward (src/streaming_quantized.rs:201-203) or the
 * gate/up projections of QMlp::forward (:277), which read the same x.  The
 * weights are streamed back to back without a pipeline drain between them;
 * x_i may alias one another.  x and y must be device memory on the context's
 * device.  Results equal n rq_linear calls with M = 1. */
RQ_API int rq_linear_batch(rq_ctx* ctx, int n, const rq_weight* const* w, const float* const* x,
                           float* const* y, void* stream);

/* A prefetch hint, no reference counterpart: the next M=1 pipeline launch
 * of rq_linear / rq_linear_batch / rq_linear_allreduce on this context
 * prefetches into L2, after its last weight copy, the first rows of these n
 * (<= 3, of one type and in_features) weights -- the weights the caller
 * multiplies next, as a layer loop knows them -- so HBM keeps streaming
 * through the launch gap.  Consumed by that launch; n = 0 clears it.  No
 * effect on results; captured into CUDA graphs like the launch itself. */
RQ_API int rq_linear_prefetch_hint(rq_ctx* ctx, int n, const rq_weight* const* w);

/* Row-parallel linear under tensor parallelism: y[M][out] = the sum over
 * the ranks of x_r[M][in] * W_r^T, where W_r is this rank's column slice of
 * the weight (the o_proj / down_proj shard) and x_r its slice of the input;
 * every rank calls with the same M and gets the same y bits.  At M = 1 the
 * all-reduce runs inside the matvec kernel: each CTA stores its rows of the
 * partial product straight into every peer's NVLink exchange buffer and sums
 * the W slots in rank order once the peers have flagged theirs; otherwise
 * (or with RQ_TP_FUSED=0) the partial product is all-reduced by a separate
 * kernel (NCCL above 512 K elements).  x and y are device memory;
 * asynchronous on `stream`; needs rq_tp_init.  No reference counterpart (the
 * reference runs on one device). */
RQ_API int rq_linear_allreduce(rq_ctx* ctx, const rq_weight* w, const float* x, float* y, int64_t M,
                               void* stream);

/* rq_linear for callers that cannot allocate device memory.  No counterpart
 * in the reference.
 *
 * rq_linear stages activations in a workspace it grows with cudaMalloc.
 * Callers whose device memory is owned by someone else (a serving engine
 * that reserves nearly all HBM up front, a framework allocator such as
 * candle's CUDA device) or whose decode loop cannot afford a cudaMalloc
 * that may synchronise the device use this entry point instead: it calls no
 * cudaMalloc, cudaFree or other allocating routine.  Its staging area is a
 * static 2 MiB device array that every GPU loading librq holds until exit.
 *
 *   - x [M][in] and y [M][out] must be device memory on w's device;
 *   - M * in is limited by the 2 MiB array at 3.5 bytes per element (plus
 *     alignment; e.g. M <= 20 at in = 28672, M <= 73 at in = 8192); larger
 *     requests fail with RQ_ERR_INVALID and a message;
 *   - every row runs the M=1 matvec kernels, so results match rq_linear's
 *     within the linear parity tolerance (relative L2 <= 1e-4; the same
 *     kernels at M = 1, while from M = 2 rq_linear takes its tensor-core
 *     kernels where the weight's type and shape allow); weights with no
 *     M=1 pipeline shape --
 *     Q8_0 / Q5_K with in not a multiple of 256, Q6_K / Q2_K with in not a
 *     multiple of 1024, any type with in > 30720 other than Q4_0 / Q4_K /
 *     Q3_K -- return RQ_ERR_UNSUPPORTED;
 *   - the first call on a device resolves the array's device address
 *     (cudaGetSymbolAddress): make that first call before any stream
 *     capture;
 *   - all calls on a device share the one array, which keeps the last
 *     call's contents: calls that overlap on the GPU (other streams,
 *     threads) race on it, so serialise them;
 *   - the call is asynchronous on `stream`; a bounded kernel wait that gave
 *     up inside it is reported by rq_ctx_status on a context of that device. */
RQ_API int rq_linear_noalloc(const rq_weight* w, const float* x, float* y, int64_t M,
                             void* stream);

/* -------------------------------------------------------- tensor parallel */

/* One process per GPU.  Rank 0 creates an id (rq_tp_unique_id, >= 128
 * bytes), the host side distributes it (e.g. over torch.distributed), and
 * every rank calls rq_tp_init on its context.  Initialisation is bounded by
 * timeout_ms: a rank that never joins yields RQ_ERR_TIMEOUT on the others
 * (the communicator is aborted), never a hang.  No reference counterpart:
 * the reference is single-device (the build's TP splits the QAttn / QMlp
 * linears column- and row-parallel and joins them with all-reduces). */
RQ_API int rq_tp_unique_id(void* id_out, size_t n);
RQ_API int rq_tp_init(rq_ctx* ctx, int world, int rank, const void* id, int timeout_ms);
/* out[n] = sum over ranks of in[n] (f32), asynchronous on stream. */
RQ_API int rq_tp_allreduce_f32(rq_ctx* ctx, const float* in, float* out, int64_t n, void* stream);
/* RQ_OK while the communicator is healthy, RQ_ERR_NCCL after an async error. */
RQ_API int rq_tp_status(rq_ctx* ctx);
RQ_API int rq_tp_finalize(rq_ctx* ctx);

/* ------------------------------------------------------------- sparse MoE */

/* Mixtral SparseMoe (src/streaming_mixtral.rs:259-319) with quantized
 * experts: router weight f32 [E][hidden] (host or device; copied and rounded
 * to F16 as ParallelLinear::new does, src/parallel_linear.rs:128-131), expert
 * weights w1 = gate [ffn][hidden], w3 = up [ffn][hidden], w2 = down
 * [hidden][ffn] (borrowed: they must outlive the layer).  E <= 32.  Under a
 * communicator (rq_tp_init, world W > 1) the experts of other ranks (e % W
 * != rank) may be NULL: the layer then runs expert-parallel only. */
RQ_API int rq_moe_create(rq_ctx* ctx, int n_experts, int top_k, int64_t hidden, int64_t ffn,
                         const float* router_w, const rq_weight* const* w1,
                         const rq_weight* const* w3, const rq_weight* const* w2, rq_moe** out);
RQ_API int rq_moe_free(rq_moe* m);
/* y[T][hidden] = SparseMoe::forward(x[T][hidden]) (:280-319): router,
 * softmax, top-k with renormalised weights (ties to the lower expert index),
 * per-expert token buckets in ascending token order, SwiGLU experts, combine
 * in ascending expert order.  x, y host or device.  expert_ids_out [T][k]
 * (rank order) and perm_out [T*k] (tokens of expert 0, then expert 1, ...)
 * are optional host outputs.  With T < 4 (decode and speculative-verify
 * batches) no expert segment reaches the tensor-core kernels, so routing,
 * permutation and the expert products stay on the device: with device x /
 * y and no routing outputs the call is asynchronous on `stream` and can be
 * captured in a CUDA graph (after one call at that T outside capture, which
 * sizes the layer's buffers).  From T = 4 on, the per-expert token counts
 * are read back to the host once (the reference reads its whole routing
 * table there, :284-286) to pick each segment's kernel. */
/* Forwards of up to max_tokens tokens plan on the device (default and
 * minimum 3): every routing slot becomes one M=1 matvec job whose expert
 * the kernel reads from the routing table -- no host synchronisation,
 * asynchronous and graph-capturable at that T, slower than the host plan
 * from about 4 tokens (each slot streams its expert's weights). */
RQ_API int rq_moe_set_device_plan(rq_moe* m, int64_t max_tokens);

RQ_API int rq_moe_forward(rq_ctx* ctx, rq_moe* m, const float* x, float* y, int64_t T,
                          int32_t* expert_ids_out, int32_t* perm_out, void* stream);
/* Expert-parallel forward over the communicator of ctx: expert e lives on
 * rank e % W.  Each rank passes its own T tokens (T may differ per rank, 0
 * included; every rank must call).  Routing is local; the token rows go to
 * their experts' ranks and the expert outputs come back through NCCL
 * all-to-alls (ncclSend/ncclRecv), and each rank combines its own tokens in
 * ascending expert order.  y, expert_ids_out and perm_out as for
 * rq_moe_forward, for the local tokens; y equals rq_moe_forward on the same
 * tokens bit for bit. */
RQ_API int rq_moe_forward_ep(rq_ctx* ctx, rq_moe* m, const float* x, float* y, int64_t T,
                             int32_t* expert_ids_out, int32_t* perm_out, void* stream);

/* -------------------------------------------------------- Llama decode loop */

/* The quantized Llama forward of StreamingLlamaQuantized with every layer
 * resident on the GPU (src/streaming_quantized.rs:611-729, QBlock
 * :282-318), a per-layer f32 KV cache (QuantStreamCache :93-152) and the
 * greedy step of generate (:539-593).  Config mirrors candle's llama Config
 * fields the block uses (global sizes).  With a tensor-parallel communicator
 * on the context (world W, rank r), each rank holds shard r of every layer:
 * q/k/v/gate/up rows (heads r*n_heads/W.., kv heads r*n_kv_heads/W..,
 * intermediate rows r*intermediate/W..), the matching o/down columns, and
 * lm_head rows r*vocab/W..; the embedding and norms are replicated. */
typedef struct rq_llama rq_llama;
typedef struct rq_llama_config {
    int64_t hidden, intermediate, n_heads, n_kv_heads, head_dim, n_layers, vocab;
    int64_t max_seq;          /* KV cache capacity in positions */
    int64_t max_batch_tokens; /* most tokens per rq_llama_forward (prompt chunk) */
    float rms_eps, rope_theta;
} rq_llama_config;

RQ_API int rq_llama_create(rq_ctx* ctx, const rq_llama_config* cfg, rq_llama** out);
RQ_API int rq_llama_free(rq_llama* m);
/* Layer weights q,k,v,o,gate,up,down (this rank's shards; borrowed: they
 * must outlive m) and the two RmsNorm weights (f32 [hidden], host or device,
 * copied).  Replaces QBlock::load (src/streaming_quantized.rs:290-303). */
RQ_API int rq_llama_set_layer(rq_llama* m, int64_t layer, const rq_weight* const* w7,
                              const float* rms1, const float* rms2);
/* Norms of q and k per head before the rotation (eps = rms_eps), for models
 * that have them: f32 [head_dim] each, host or device, copied.  The one-launch
 * step (rq_llama_set_fused) is not used then.  No reference counterpart. */
RQ_API int rq_llama_set_qk_norm(rq_llama* m, int64_t layer, const float* q_weight, const float* k_weight);
/* Holds the model's cache in 4 bits and in pages of page_size positions (see
 * rq_kv4_create: head_dim 32, 64, 96 or 128) in place of the f32 cache, which
 * is freed: 4.5 / 32 of its memory.  Starts empty, so call it before the first
 * forward; pages come from one ring as the position grows and go back when it
 * is moved (rq_llama_truncate, a forward's index_pos).  The one-launch step is
 * not used then.  No reference counterpart. */
RQ_API int rq_llama_use_kv4(rq_llama* m, int page_size);
/* The keys (rotated) and values that the 4-bit cache of a layer holds at
 * positions pos .. pos + n - 1: f32 [n][n_kv_heads][head_dim] (this rank's
 * heads), host or device.  Synchronous. */
RQ_API int rq_llama_read_kv4(rq_llama* m, int64_t layer, int64_t pos, int64_t n, float* k, float* v);
/* F16 [vocab][hidden] token embedding (model.embed_tokens.weight). */
RQ_API int rq_llama_set_embedding(rq_llama* m, const uint16_t* embed_f16);
/* Final RmsNorm weight (f32 [hidden]) and F16 lm_head rows of this rank
 * ([vocab/W][hidden]). */
RQ_API int rq_llama_set_head(rq_llama* m, const float* ln_f, const uint16_t* lm_head_f16);
/* forward(input_ids, index_pos) of src/streaming_quantized.rs:622-633 over T
 * host tokens at positions index_pos..index_pos+T-1: logits (host or device
 * [vocab], may be NULL; single rank only) of the last position and the
 * greedy next token (may be NULL).  Synchronous.  Leaves the next token and position on the device
 * for rq_llama_decode_step. */
RQ_API int rq_llama_forward(rq_llama* m, const int32_t* tokens, int64_t T, int64_t index_pos,
                            float* logits, int32_t* next_token, void* stream);
/* One greedy decode step entirely on the device (token and position read
 * from and written to device memory), so it can be captured in a CUDA graph
 * and replayed; each step appends its token to the device token list.  By
 * default a chain of per-layer kernels; rq_llama_set_fused(m, 1) makes the
 * step (one GPU, one weight type) a single persistent launch that streams the
 * weights through grid-wide phases and computes the same bits. */
/* The verify forward of speculative decoding (forward_all,
 * src/streaming_quantized.rs:611-620): T tokens at index_pos through every
 * layer, then the final norm and lm_head at EVERY position; argmax[T] (host
 * or device) receives each position's greedy token and logits[T][vocab]
 * (optional, one GPU only) the logits.  Like rq_llama_forward it leaves the
 * KV cache at index_pos + T and the last position's token as the next
 * input; rq_llama_truncate rolls back rejected positions. */
RQ_API int rq_llama_forward_all(rq_llama* m, const int32_t* tokens, int64_t T, int64_t index_pos, float* logits,
                                int32_t* argmax, void* stream);
RQ_API int rq_llama_decode_step(rq_llama* m, void* stream);
RQ_API int rq_llama_set_fused(rq_llama* m, int enable);
/* RQ_ERR_TIMEOUT (and clears it) when a bounded wait inside a kernel of the
 * model (a decode step, the one-launch step, a forward) gave up since the
 * last call; synchronous.  rq_llama_forward / _forward_all check it before
 * they return. */
RQ_API int rq_llama_status(rq_llama* m);
/* Tokens appended since the last reset (count may exceed cap), and the
 * current position.  Synchronous. */
RQ_API int rq_llama_tokens(rq_llama* m, int32_t* out, int64_t cap, int64_t* count,
                           int64_t* position);
RQ_API int rq_llama_reset_tokens(rq_llama* m);
/* QuantStreamCache::truncate / truncate_caches
 * (src/streaming_quantized.rs:131-141,603-609): roll the KV length back. */
RQ_API int rq_llama_truncate(rq_llama* m, int64_t new_len);

/* ------------------------------------------------- paged serving operators */

/* No counterpart in the reference, whose cache is one contiguous f32 buffer
 * per layer and sequence (QuantStreamCache, src/streaming_quantized.rs:93-152).
 * All pointers of this section are device memory on the context's device
 * unless a comment says host; every call is asynchronous on `stream`, reads
 * nothing back, allocates nothing and can be captured in a CUDA graph.  Sizes
 * that a kernel reads from device memory (lengths, offsets, slots, table
 * entries) are checked on the device: an index outside its range is skipped,
 * as each comment says, never followed. */

/* Element types of q, k, v, probabilities and outputs. */
enum rq_dtype { RQ_F32 = 0, RQ_F16 = 1, RQ_BF16 = 2 };

/* A paged key/value cache of one layer, held in 4 bits: n_pages pages of
 * page_size positions (a multiple of 16, at most 4096; n_pages * page_size <
 * 2^31) of n_kv_heads heads, head_dim 32, 64, 96 or 128.  Blocks of 32
 * elements of a head's row: d = f16(m / -8) with m the element of largest
 * magnitude (the first of equals; d saturates at 65504), code = the nearest
 * multiple of d in 0..15 (ties up), value (code - 8) * d: 4.5 bits an
 * element.  A NaN makes its block NaN.  Position `off` of page `p` is slot p *
 * page_size + off.  Positions never written read as zeros. */
typedef struct rq_kv4 rq_kv4;
RQ_API int rq_kv4_create(rq_ctx* ctx, int64_t n_pages, int page_size, int n_kv_heads, int head_dim, rq_kv4** out);
RQ_API int rq_kv4_free(rq_kv4* c);
/* Any of the out-pointers may be NULL. */
RQ_API int rq_kv4_info(const rq_kv4* c, int64_t* n_pages, int* page_size, int* n_kv_heads, int* head_dim,
                       size_t* device_bytes);
/* Quantizes the keys and values of n tokens into slots[n]; a slot outside
 * the cache (-1: padding) is skipped.  k and v are [n][n_kv_heads][head_dim]
 * with the given strides of token and head in elements (host array of two),
 * elements contiguous.  The slots of one call must differ. */
RQ_API int rq_kv4_append(rq_kv4* c, int dtype, const void* k, const int64_t k_stride[2], const void* v,
                         const int64_t v_stride[2], const int32_t* slots, int64_t n, void* stream);
/* k, v [n][n_kv_heads][head_dim] = the values held in slots[n] (zeros for a
 * slot outside the cache). */
RQ_API int rq_kv4_read(rq_kv4* c, const int32_t* slots, int64_t n, int dtype, void* k, void* v, void* stream);

/* Attention of the newest tokens of `batch` sequences over the cache.
 * Sequence b holds kv_lens[b] positions, its newest tokens (already appended)
 * among them; position j lives in page block_table[b * table_stride + j /
 * page_size].  Its n queries are the rows cu_q[b] .. cu_q[b + 1] - 1 of q
 * (n <= max_q; cu_q NULL: row b, n = 1; of more, the rows behind the first
 * max_q are left as they were), query i at position kv_lens[b] - n +
 * i; it sees the positions j <= its own and, with window > 0, j > its own -
 * window.  out row = softmax_j(scale * q . k_j) v over the seen positions, in
 * f32 sums; query head h reads kv head h / (n_heads / n_kv_heads).  f32 and f16
 * queries take the cache's values exactly, whatever other positions hold (where a
 * head's row has blocks whose scales differ by more than 2^14, the smaller ones
 * to 2^-25 of the largest); more than 16 bf16 rows (queries times
 * heads) a kv head take them rounded to f16, where a value below 2^-26 of the
 * largest of its 32 positions keeps fewer bits.  A query
 * that sees nothing gets zeros.  Positions behind table_width * page_size or
 * on a page outside the cache are not seen.  Rows of q and out that belong to
 * no sequence (or lie at or behind n_tokens) are left as they were.  out may
 * be q, otherwise the two must not overlap; rows of out that overlap one
 * another are refused.  max_len (> 0): an upper bound of kv_lens that only guides how the
 * work is split (0: table_width * page_size).  One form serves the whole
 * call, chosen by max_q: single tokens on long caches are faster in a call of
 * their own than among prompts.  `workspace` holds at least
 * rq_kv4_attention_workspace bytes, used by this call alone until it is done
 * (two captured graphs that may run at once need one each). */
typedef struct rq_kv4_query {
    int dtype;
    const void* q;        /* [n_tokens][n_heads][head_dim] */
    int64_t q_stride[2];  /* token, head; elements */
    void* out;
    int64_t out_stride[2];
    int64_t n_tokens, n_heads, batch, max_q;
    const int32_t* cu_q;        /* [batch + 1] or NULL */
    const int32_t* kv_lens;     /* [batch] */
    const int32_t* block_table; /* [batch][table_width] */
    int64_t table_stride, table_width, max_len, window;
    float scale;
    void* workspace;
    size_t workspace_bytes;
} rq_kv4_query;
RQ_API int rq_kv4_attention_workspace(const rq_kv4* c, const rq_kv4_query* a, size_t* bytes);
RQ_API int rq_kv4_attention(rq_kv4* c, const rq_kv4_query* a, void* stream);

/* Per head of q and k: y = x / sqrt(mean(x^2) + eps) * weight (a NULL weight:
 * y = x), then the first rot_dim elements rotated by the angles of the
 * token's position (interleaved 0: element i with i + rot_dim / 2; 1: element
 * 2i with 2i + 1).  cos, sin: f32 [max_pos][rot_dim / 2].  Computed in f32,
 * rounded once.  A token whose position lies outside 0..max_pos-1 (-1:
 * padding) leaves its output rows as they were.  q_out may be q and k_out may
 * be k; otherwise outputs and inputs must not overlap, and rows of an output
 * that overlap one another are refused.  n_heads or n_kv_heads
 * may be 0.  head_dim even, at most 256. */
typedef struct rq_qk_rope {
    int dtype;
    int64_t n_tokens, n_heads, n_kv_heads, head_dim, rot_dim;
    int interleaved;
    const void* q;
    int64_t q_stride[2]; /* token, head; elements */
    void* q_out;
    int64_t q_out_stride[2];
    const void* k;
    int64_t k_stride[2];
    void* k_out;
    int64_t k_out_stride[2];
    const float* q_weight; /* [head_dim] or NULL */
    const float* k_weight;
    float eps;
    const float* cos;
    const float* sin;
    int64_t max_pos;
    const int32_t* positions; /* [n_tokens] */
} rq_qk_rope;
RQ_API int rq_qk_norm_rope(rq_ctx* ctx, const rq_qk_rope* a, void* stream);
/* The same in one launch with the append: the normalised, rotated k (k_out is
 * not used) and v go to `slots` of the cache as rq_kv4_append would put them.
 * A token whose position lies outside the tables is not appended either. */
RQ_API int rq_qk_norm_rope_append(rq_kv4* c, const rq_qk_rope* a, const void* v, const int64_t v_stride[2],
                                  const int32_t* slots, void* stream);

/* Page bookkeeping of `batch` sequences, on the device.  The free pages are a
 * ring of n_pages entries with state {head, free, short}: ring[(head + i) %
 * n_pages], i < free.  extend: sequence b holds ctx_lens[b] positions in its
 * first ceil(ctx_lens[b] / page_size) table entries and gets new_lens[b]
 * more; the pages that these need are taken from the ring in the order of the
 * sequences and written into the table.  Outputs: kv_lens[b] = ctx_lens[b] +
 * new_lens[b] (may be ctx_lens), cu_new[batch + 1] the offsets of the new
 * tokens, and for each of n_tokens rows (n_tokens >= the sum of new_lens; the
 * rest is padding) its position and slot, -1 and -1 for padding.  Where the
 * ring holds too few pages, `short` counts the missing ones and their table
 * entries and slots are -1; a token behind the table's width gets slot -1.
 * state_out may be state_in.  Negative lengths count as 0. */
RQ_API int rq_pages_extend(rq_ctx* ctx, int64_t batch, int page_size, const int32_t* ctx_lens, const int32_t* new_lens,
                           int32_t* table, int64_t table_stride, int64_t table_width, const int32_t* ring,
                           int64_t n_pages, const int32_t* state_in, int32_t* state_out, int32_t* kv_lens,
                           int32_t* cu_new, int32_t* positions, int32_t* slots, int64_t n_tokens, void* stream);
/* Gives back the pages of sequence b behind its first keep_lens[b] positions
 * (of held_lens[b]): their table entries become -1 and the pages join the end
 * of the ring, in the order of the sequences.  state {head, free, short}
 * updated in place. */
RQ_API int rq_pages_release(rq_ctx* ctx, int64_t batch, int page_size, const int32_t* held_lens,
                            const int32_t* keep_lens, int32_t* table, int64_t table_stride, int64_t table_width,
                            int32_t* ring, int64_t n_pages, int32_t* state, void* stream);

/* Verification of drafted tokens (the sampled counterpart of the greedy
 * accept of examples/spec_decode_70b.rs:262-283).  For sequence b with n =
 * n_drafts[b] drafts (NULL: max_drafts): p row i (i = 0..n) are the target's
 * probabilities after i accepted drafts, q row i (i < n) those the i-th draft
 * was drawn from (q NULL: the draft was certain).  Draft i is accepted while
 * u[b][i] * q_i(draft) < p_i(draft).  Then one token is drawn by r[b] in
 * [0, 1): after a rejection at row i from max(p_i - q_i, 0) (from p_i where
 * that has no mass), otherwise from p_n: the first j whose running sum of
 * weights exceeds r * their total.  Sums and products in 64 bits.  NaN and
 * negative probabilities count as 0, infinite ones as the largest finite
 * value, an r outside [0, 1) as the nearest inside; a row without mass draws
 * -1; a draft outside the vocabulary is rejected.  tokens[b] [max_drafts + 1] = the
 * accepted drafts, the drawn token, then -1; accepted[b] their number.
 * p [batch][max_drafts + 1][vocab] and q [batch][max_drafts][vocab] with
 * strides of sequence and row in elements; drafts, u [batch][max_drafts]. */
RQ_API int rq_spec_verify(rq_ctx* ctx, int dtype, const void* p, const int64_t p_stride[2], const void* q,
                          const int64_t q_stride[2], const int32_t* drafts, const int32_t* n_drafts, const float* u,
                          const float* r, int64_t batch, int64_t max_drafts, int64_t vocab, int32_t* tokens,
                          int32_t* accepted, void* stream);

/* ------------------------------------------------------------------- GGUF */

/* A GGUF file read into host memory once (one sequential read, as
 * GgufLayer::open does, src/streaming_quantized.rs:42-61) and parsed:
 * versions 2 and 3, metadata skipped except general.alignment, tensor infos
 * bounds-checked against the file.  The format candle's gguf_file::write
 * emits for the reference's shards (src/quantize.rs:146-150). */
typedef struct rq_gguf rq_gguf;
RQ_API int rq_gguf_open(const char* path, rq_gguf** out);
/* the same from a caller-held buffer (copied), e.g. GgufLayer.buffer */
RQ_API int rq_gguf_open_memory(const void* data, size_t nbytes, rq_gguf** out);
RQ_API int rq_gguf_free(rq_gguf* f);
RQ_API int rq_gguf_tensor_count(const rq_gguf* f, int64_t* count);
/* index of a tensor by name (RQ_ERR_INVALID and index -1 when absent) */
RQ_API int rq_gguf_find(const rq_gguf* f, const char* name, int64_t* index);
/* name (NUL-terminated, truncated to name_cap), ggml type, n_dims, dims[4]
 * innermost first (a [out, in] matrix is {in, out, 1, 1}), offset of the
 * data in the file and its size (0 for an unknown type); NULL outputs are
 * skipped */
RQ_API int rq_gguf_tensor_info(const rq_gguf* f, int64_t index, char* name, size_t name_cap, int* ggml_type,
                               int* n_dims, int64_t* dims, uint64_t* file_offset, uint64_t* nbytes);
/* pointer to a tensor's bytes inside the file buffer (valid until free) */
RQ_API int rq_gguf_tensor_data(const rq_gguf* f, int64_t index, const void** data, uint64_t* nbytes);
/* the first `count` elements of an F32 / F16 / BF16 tensor as f32 (norms,
 * GgufLayer::tensor's dequantize, src/streaming_quantized.rs:74-83) */
RQ_API int rq_gguf_read_f32(const rq_gguf* f, const char* name, float* out, int64_t count);
/* Upload rows [row0, row0+rows) x columns [col0, col0+cols) of a 2-D Q4_0 /
 * Q4_K / Q3_K tensor (rows or cols < 0: to the end; columns on block
 * boundaries): GgufLayer::qmatmul (src/streaming_quantized.rs:63-70) with
 * the tensor-parallel shard taken on the host. */
RQ_API int rq_weight_upload_gguf(rq_ctx* ctx, const rq_gguf* f, const char* name, int64_t row0, int64_t rows,
                                 int64_t col0, int64_t cols, rq_weight** out);
/* Load a shard directory as StreamingLlamaQuantized::from_pretrained reads
 * it (src/streaming_quantized.rs:451-501): model.layers.<l>.gguf for every
 * layer (model.layers.<l>.self_attn.{q,k,v,o}_proj.weight,
 * .mlp.{gate,up,down}_proj.weight, .input_layernorm.weight,
 * .post_attention_layernorm.weight), model.embed_tokens.gguf,
 * model.norm.gguf and lm_head.gguf (absent: the head is the embedding).
 * Under tensor parallelism each rank uploads its own shards.  The model
 * owns the weights it uploads. */
RQ_API int rq_llama_load_gguf_dir(rq_llama* m, const char* dir);

#ifdef __cplusplus
}
#endif
#endif /* RQ_H */
