/*
 * llmi_hip.h -- C ABI of the MI355X (gfx950) quantized-weight path.
 *
 * Every entry point replaces one function of llm-inference-cpp's
 * quantized-weight path; the reference interface each one stands in for is
 * cited beside it (paths relative to the reference repository root).  Plain
 * pointers and sizes only: host pointers unless the name ends in _dev, in
 * which case the pointers are device pointers and the work is queued on
 * `stream` (a hipStream_t; NULL means the library's own stream) without a
 * host synchronisation.
 *
 * Errors: every function returns LLMI_OK (0) or a non-zero LLMI_ERR_* code
 * and leaves a message for llmi_hip_last_error() on the calling thread.  The
 * reference's quant functions have no error channel (they return void and
 * assume valid shapes); here bad shapes, unsupported types and HIP failures
 * are reported instead of being undefined behaviour.
 *
 * Threading: like the reference (include/llmi/util/thread_pool.hpp:18-21,
 * src/server/server.cpp:44-49) calls are not reentrant; serialise them.
 */
#ifndef LLMI_HIP_H
#define LLMI_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
  LLMI_OK = 0,
  LLMI_ERR_ARG = 1,   /* bad shape, type, pointer or token id */
  LLMI_ERR_HIP = 2,   /* HIP runtime failure (allocation, launch, copy) */
  LLMI_ERR_STATE = 3, /* not initialised, cache full, cache from another model */
};

/* Weight storage types; the values of llmi::quant::Type
 * (include/llmi/model/quant.hpp:17). */
enum { LLMI_TYPE_F32 = 0, LLMI_TYPE_Q8_0 = 1, LLMI_TYPE_Q4_0 = 2 };

/* Weights per quantization block (include/llmi/model/quant.hpp:15). */
#define LLMI_BLOCK_SIZE 32

/* GGUF tensor types accepted by llmi_hip_weight_from_gguf: the values of
 * llmi::gguf::TensorType (include/llmi/model/gguf.hpp:26-34). */
enum { LLMI_GGUF_Q4_0 = 2, LLMI_GGUF_Q8_0 = 8 };

/* Model hyper-parameters: the fields of llmi::ModelConfig
 * (include/llmi/model/model.hpp:21-36) that the forward pass reads.
 * head_dim = hidden_size / num_heads (src/model/model.cpp:100-105). */
typedef struct llmi_model_config {
  int32_t arch; /* 0 = Llama, 1 = Qwen2 (model.hpp:16) */
  uint32_t vocab_size;
  uint32_t hidden_size;
  uint32_t intermediate_size;
  uint32_t num_layers;
  uint32_t num_heads;
  uint32_t num_kv_heads;
  uint32_t max_position_embeddings;
  double rms_norm_eps;
  double rope_theta;
  int32_t tie_word_embeddings;
  int32_t qkv_bias;
} llmi_model_config;

typedef struct llmi_hip_weight llmi_hip_weight; /* device-resident packed matrix */

/* ----------------------------------------------------------------- runtime */

/* Selects the GPU and creates the library stream.  Must precede every other
 * call except llmi_hip_last_error and llmi_hip_version. */
int llmi_hip_init(int device);
/* Releases the library stream.  Weights stay valid until freed. */
int llmi_hip_shutdown(void);
const char* llmi_hip_last_error(void);
const char* llmi_hip_version(void);
/* The library's stream (hipStream_t), for callers that queue their own work. */
void* llmi_hip_stream(void);
int llmi_hip_synchronize(void);

/* Plain device memory and copies, for callers without an allocator of
 * their own (tests, bench.py).  Copies are synchronous. */
int llmi_hip_malloc(void** ptr, size_t bytes);
int llmi_hip_free(void* ptr);
int llmi_hip_memcpy_h2d(void* dst_dev, const void* src, size_t bytes);
int llmi_hip_memcpy_d2h(void* dst, const void* src_dev, size_t bytes);
/* Device-to-device copy queued on `stream` (a plain copy kernel). */
int llmi_hip_memcpy_d2d(void* dst_dev, const void* src_dev, size_t bytes, void* stream);
int llmi_hip_memset_dev(void* dst_dev, int value, size_t bytes);

/* HIP events on `stream` (NULL = library stream), for kernel timing. */
int llmi_hip_event_create(void** ev);
int llmi_hip_event_destroy(void* ev);
int llmi_hip_event_record(void* ev, void* stream);
int llmi_hip_event_elapsed_ms(void* start, void* stop, float* ms);

/* Captures the work queued on the library stream between begin and end into
 * a HIP graph (hipStreamBeginCapture / hipGraphInstantiate), for callers
 * that replay a fixed sequence of _dev calls (a decode step, a benchmark
 * pass) without per-launch host overhead.  Only _dev entry points may be
 * called while capturing; the captured kernels allocate and clear nothing. */
int llmi_hip_graph_begin(void);
int llmi_hip_graph_end(void** graph);
int llmi_hip_graph_launch(void* graph);
int llmi_hip_graph_destroy(void* graph);

/* Fills dst_dev[i] = float32(mean + std * z_{offset+i}) from the deterministic
 * "synth-v1" stream `seed` (the same values llm-inference-cpp_amd/synth.py
 * produces on the host).  Test and benchmark input generation only. */
int llmi_hip_synth_normal_dev(float* dst_dev, size_t n, uint64_t seed, uint64_t offset, double mean, double stdev,
                              void* stream);

/* ------------------------------------------------------- block quantizer */

/* Bytes of packed codes per row: in (Q8_0) or ceil(in/2) (Q4_0)
 * (src/model/quant.cpp:18-20). */
size_t llmi_hip_row_bytes(size_t in, int type);

/* Replaces llmi::quant::quantize (include/llmi/model/quant.hpp:51,
 * src/model/quant.cpp:36-102), computed on the GPU.  w is the out x in
 * row-major fp32 matrix; data (out * row_bytes) and scales
 * (out * ceil(in/32)) receive the reference's planar layout
 * (QuantizedMatrix::data / ::scales, quant.hpp:38-48), bit-exact. */
int llmi_hip_quantize(const float* w, size_t out, size_t in, int type, uint8_t* data, float* scales);
int llmi_hip_quantize_dev(const float* w_dev, size_t out, size_t in, int type, uint8_t* data_dev, float* scales_dev,
                          void* stream);

/* ------------------------------------------------ device-resident weights */

/* Uploads a QuantizedMatrix (planar data + scales, as produced by
 * quant::quantize) and re-lays it out for the GPU kernels.  Stands in for the
 * storage of llmi::Weight (include/llmi/model/weight.hpp:18-39,
 * src/model/weight.cpp:16-22). */
int llmi_hip_weight_upload(const uint8_t* data, const float* scales, size_t out, size_t in, int type,
                           llmi_hip_weight** weight);
/* Weight::quantized (src/model/weight.cpp:16-22): quantizes an fp32 matrix on
 * the GPU straight into the device layout.  w is a host pointer.  With
 * LLMI_TYPE_F32 the matrix is kept as fp32 (Weight::from_float,
 * weight.cpp:9-14) and products run kernels::matmul (kernels.cpp:97-113):
 * y = dot(x_r, w_o) + bias with the reference's dot arithmetic, bit-exact. */
int llmi_hip_weight_quantize(const float* w, size_t out, size_t in, int type, llmi_hip_weight** weight);
int llmi_hip_weight_quantize_dev(const float* w_dev, size_t out, size_t in, int type, llmi_hip_weight** weight);
int llmi_hip_weight_free(llmi_hip_weight* weight);
/* Replaces llmi::gguf::to_quantized (include/llmi/model/gguf.hpp:184,
 * src/model/gguf.cpp:577-640) followed by the upload: `blocks` (host) is a
 * GGUF tensor's raw data, nbytes long, out rows of in/32 ggml blocks
 * ({fp16 d; codes}, 34 bytes for Q8_0, 18 for Q4_0).  The device converts
 * each block into the layout llmi_hip_weight_upload produces from the
 * reference's own QuantizedMatrix (fp16 scale -> fp32 exactly; Q4_0's
 * halves-of-the-block nibble pairing re-packed into neighbour pairs), so
 * downloading the result gives to_quantized's data and scales bit for bit.
 * Fails (LLMI_ERR_ARG) where to_quantized fails: a type other than Q8_0 /
 * Q4_0, an empty shape, in not a multiple of 32, or nbytes not matching the
 * shape. */
int llmi_hip_weight_from_gguf(const void* blocks, size_t nbytes, size_t out, size_t in, int gguf_type,
                              llmi_hip_weight** weight);
/* Copies the weight back into the reference's planar layout (an fp32 weight:
 * its out x in floats into data, scales untouched). */
int llmi_hip_weight_download(const llmi_hip_weight* weight, uint8_t* data, float* scales);
/* Shape/type queries; byte_size is QuantizedMatrix::byte_size
 * (quant.hpp:47): packed code bytes + 4 * number of scales. */
int llmi_hip_weight_info(const llmi_hip_weight* weight, size_t* out, size_t* in, int* type, size_t* byte_size);
/* Device footprint of the re-laid-out matrix (codes + scales, with padding). */
size_t llmi_hip_weight_device_bytes(const llmi_hip_weight* weight);

/* Replaces llmi::quant::dequantize_row (quant.hpp:54, quant.cpp:104-117) and
 * the embedding gather Weight::row (weight.cpp:39-45): dst[k] =
 * code[row][k] * scale[row][k/32], one rounding, bit-exact. */
int llmi_hip_dequantize_row(const llmi_hip_weight* weight, size_t row, float* dst);
/* Gathers rows ids_dev[0..n) into dst_dev (n x in).  Ids must be in range. */
int llmi_hip_dequantize_rows_dev(const llmi_hip_weight* weight, const int32_t* ids_dev, size_t n, float* dst_dev,
                                 void* stream);

/* Replaces llmi::quant::matmul (quant.hpp:64-65, quant.cpp:119-153) and
 * Weight::matmul (weight.cpp:30-37): y[r*out + o] = sum_i x[r*in + i] *
 * dequantized(w[o][i]) (+ bias[o]), for r < rows.  The arithmetic is the
 * reference's, operation for operation (per 32-block a fused chain over the
 * block, then a fused chain over the blocks, then + bias), so y is bit-exact.
 * in and out must equal the weight's shape; bias may be NULL.
 * llmi_hip_matmul takes host pointers and returns with y complete. */
int llmi_hip_matmul(const llmi_hip_weight* weight, const float* x, size_t rows, size_t in, size_t out,
                    const float* bias, float* y);
int llmi_hip_matmul_dev(const llmi_hip_weight* weight, const float* x_dev, size_t rows, const float* bias_dev,
                        float* y_dev, void* stream);

/* A fixed list of independent products launched as ONE kernel: for each i,
 * y_dev[i] = quant::matmul(x_dev[i], rows[i], w[i]) (+ bias_dev[i]) exactly
 * as llmi_hip_matmul_dev would compute it (quant.cpp:119-153, bit-identical),
 * for callers that issue many small matmuls back to back (the per-layer
 * Weight::matmul calls of transformer.cpp:245-304 when their inputs are
 * ready together).  rows[i] is 1..8 (NULL: all 1); bias_dev may be NULL (no
 * biases) or hold NULL entries.  Every weight must have in <= ~10k.  The
 * group keeps the pointers, not the data: launch it whenever the inputs are
 * in place.  Products must not write memory another product of the group
 * reads.  llmi_hip_group_launch queues the kernel on `stream` (capturable in
 * a graph). */
typedef struct llmi_hip_group llmi_hip_group;
int llmi_hip_group_create(const llmi_hip_weight* const* w, const float* const* x_dev, const size_t* rows,
                          const float* const* bias_dev, float* const* y_dev, size_t count, llmi_hip_group** out);
int llmi_hip_group_launch(const llmi_hip_group* group, void* stream);
void llmi_hip_group_free(llmi_hip_group* group);

/* Tolerance mode, Q4_0: quant::matmul (quant.cpp:119-153) for batch 1..8
 * with the products summed on the matrix cores in another order than the
 * reference's chains.  NOT bit-exact: |y - y_ref| <= 1e-4 * max|y_ref| (the
 * fp32-accumulate tolerance of the path's contract; measured ~1e-6), with
 * finite x below ~3e38.  The codes enter as exact bf16 values, x as two bf16
 * parts (16 significant bits), sums in fp32.  Same arguments and meaning as
 * llmi_hip_matmul_dev (rows 1..8, in <= ~14k); llmi_hip_tol_group_* run a
 * list of such products as one launch, as llmi_hip_group_* do for the exact
 * kernel.  The exact
 * entry points stay the default everywhere: the model's decode and the
 * reference-signature layer never take this one. */
typedef struct llmi_hip_tol_group llmi_hip_tol_group;
int llmi_hip_matmul_tol_dev(const llmi_hip_weight* weight, const float* x_dev, size_t rows, const float* bias_dev,
                            float* y_dev, void* stream);
int llmi_hip_tol_group_create(const llmi_hip_weight* const* w, const float* const* x_dev, const size_t* rows,
                              const float* const* bias_dev, float* const* y_dev, size_t count,
                              llmi_hip_tol_group** out);
int llmi_hip_tol_group_launch(const llmi_hip_tol_group* group, void* stream);
void llmi_hip_tol_group_free(llmi_hip_tol_group* group);

/* Prefill GEMM on the matrix cores: quant::matmul (quant.cpp:119-153) as the
 * reference's prefill calls it with rows = T tokens (transformer.cpp:245-291),
 * computed with x and the dequantized weights rounded to bf16 and fp32
 * accumulation (bf16 MFMA).  NOT bit-exact: |y - y_ref| <= 2e-2 * max|y_ref|
 * (typically ~1e-3).  Use llmi_hip_matmul_dev where the reference's exact
 * results are needed.  Any rows >= 1; efficient for rows >= 64.
 * llmi_hip_gemm_group_* run a list of such products as one launch (per
 * weight type), e.g. the q/k/v or gate/up products of a layer.  A launch of
 * fewer than 256 output tiles (128 x 256) splits the K of products with
 * more than 1536 inputs over several workgroups and sums their fp32 partials
 * in a second kernel, so a product's results can differ in the last bits
 * between a launch that splits it and one that does not. */
int llmi_hip_matmul_mfma_dev(const llmi_hip_weight* weight, const float* x_dev, size_t rows, const float* bias_dev,
                             float* y_dev, void* stream);
/* llmi_hip_matmul_mfma_dev for callers that cannot allocate device memory
 * (code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  No counterpart in the reference.  Same kernels and results,
 * bit for bit; the GEMM's scratch -- the bf16 copy of x and, for a product
 * whose K is split over several workgroups (more than 1536 inputs on fewer
 * than 256 output tiles of 128 x 256, as llmi_hip_matmul_mfma_dev splits
 * it), its fp32 partial sums -- lives in a
 * fixed per-GPU array set up by llmi_hip_init instead of a buffer the
 * library grows, so the call makes no allocation.  Limit: 2 * rows * (in
 * rounded up to 64), rounded up to 256, plus 4 * rows * out * kchunks when K
 * is split, at most LLMI_MFMA_NOALLOC_SCRATCH_BYTES (LLMI_ERR_ARG beyond).
 * With nk = ceil(in / 64) and tiles = ceil(rows / 128) * ceil(out / 256), K
 * is split when nk > 24, tiles < 256 and k = min(256 / tiles, nk / 8)
 * (integer quotients) is at least 2, into kchunks = ceil(nk / ceil(nk / k))
 * chunks; e.g. 512 rows of 896 x 4864 take 9 chunks and need 21.5 MB.  Calls
 * that overlap on one GPU (e.g. on two streams) share that array and race. */
#define LLMI_MFMA_NOALLOC_SCRATCH_BYTES 33554432
int llmi_hip_matmul_mfma_noalloc_dev(const llmi_hip_weight* weight, const float* x_dev, size_t rows,
                                     const float* bias_dev, float* y_dev, void* stream);
typedef struct llmi_hip_gemm_group llmi_hip_gemm_group;
int llmi_hip_gemm_group_create(const llmi_hip_weight* const* w, const float* const* x_dev, const size_t* rows,
                               const float* const* bias_dev, float* const* y_dev, size_t count,
                               llmi_hip_gemm_group** out);
int llmi_hip_gemm_group_launch(const llmi_hip_gemm_group* group, void* stream);
void llmi_hip_gemm_group_free(llmi_hip_gemm_group* group);

/* ------------------------------------------------- glue kernels (device) */
/* Device counterparts of llmi::kernels (include/llmi/model/kernels.hpp:13-32)
 * and llmi::argmax (transformer.hpp:120), bit-identical to the reference.
 * All pointers are device pointers. */

/* kernels::dot (kernels.cpp:41-95, the AVX2 build's summation order):
 * out[i] = dot(a, b, lens[i]) for i < count. */
int llmi_hip_dot_dev(const float* a, const float* b, const int32_t* lens, size_t count, float* out, void* stream);
/* kernels::rmsnorm (kernels.cpp:115-120) on each of `rows` rows of length n. */
int llmi_hip_rmsnorm_dev(const float* x, const float* w, size_t rows, size_t n, float eps, float* y, void* stream);
/* kernels::softmax (kernels.cpp:136-146), in place on each row. */
int llmi_hip_softmax_dev(float* x, size_t rows, size_t n, void* stream);
/* kernels::silu (kernels.cpp:148), in place. */
int llmi_hip_silu_dev(float* x, size_t n, void* stream);
/* argmax (transformer.cpp:22-24): index of the first maximum of x[0..n). */
int llmi_hip_argmax_dev(const float* x, size_t n, int32_t* out, void* stream);

/* ------------------------------------- paged 8-bit key/value cache (device) */
/* A key/value cache for many sequences at once, beside the fp32 cache of one
 * sequence that the model calls below keep.  No counterpart in the reference
 * (its KVCache holds one sequence in fp32, include/llmi/model/transformer.hpp:
 * 29-45).  The cache of one transformer layer is a pool of pages; a page holds
 * page_tokens positions of every key/value head as int8 codes, in blocks of
 * LLMI_KV8_BLOCK positions with one fp32 scale per block and head, for keys
 * and for values apart:
 *   value = code * scale, scale = float(amax / 127), amax = the largest |value|
 *   of the block and head, code = the exact value / scale rounded to the
 *   nearest integer, ties to even, clamped to -127..127 (scale 0: code 0).
 * A block that is not full is quantized as a whole at every append, from the
 * fp32 rows in `open`: codes depend on the values alone, not on how they were
 * split into calls, and each value is rounded once.  An inf or NaN makes its
 * block's scale inf or NaN and its codes 0, so that every value of the block
 * reads back as NaN.
 *
 * Layouts (device memory of the caller, llmi_hip_kv8_sizes gives the sizes;
 * 16-byte aligned; nothing has to be cleared beforehand):
 *   k       [pages][kv_heads][page_tokens/16][head_dim/16][16 positions][16 dims]
 *   v       [pages][kv_heads][page_tokens/16][head_dim/16][16 dims][16 positions]
 *   scales  [pages][kv_heads][page_tokens/16][2]   (the keys', the values')
 *   open    [slots][kv_heads][2][2][16][head_dim]  block parity, then k / v:
 *           the fp32 rows of the last block of each parity that the appends
 *           under a slot wrote (of a call's blocks, the last two).
 * Which pages a sequence has is the caller's: page p of its table holds
 * positions p * page_tokens ...  Full pages may be shared by sequences. */
#define LLMI_KV8_BLOCK 16
typedef struct llmi_kv8_shape {
  uint32_t heads;       /* query heads, a multiple of kv_heads */
  uint32_t kv_heads;
  uint32_t head_dim;    /* a multiple of 32, 32..256 */
  uint32_t page_tokens; /* positions per page, a multiple of 16, at most 65536 */
  uint32_t pages;       /* pages of the pool */
  uint32_t slots;       /* sequences that `open` has room for */
} llmi_kv8_shape;
typedef struct llmi_kv8_layer { /* one layer's cache */
  int8_t* k;
  int8_t* v;
  float* scales;
  float* open;
} llmi_kv8_layer;
/* Bytes of k (and of v), floats of scales and of open.  Needs no GPU. */
int llmi_hip_kv8_sizes(const llmi_kv8_shape* shape, size_t* code_bytes, size_t* scale_floats, size_t* open_floats);

/* A batch: sequence i brings counts[i] >= 0 new tokens at positions starts[i],
 * starts[i] + 1, ...; its pages are tables[i * table_stride ...], enough for
 * starts[i] + counts[i] positions; slots[i] is its place in `open`.  Token
 * rows are ragged: the tokens of sequence 0, then those of sequence 1, ...
 * All arrays are host memory, read before the call returns.
 * A plan holds a batch's work lists on the device and the attention's
 * workspace, and serves every layer of the same shape.  It is created for at
 * most max_seqs sequences, max_tokens tokens (x heads / kv_heads up to 2^30)
 * and max_pages page entries in all (0: shape->pages); plan_set replaces the
 * batch.
 * plan_set queues one copy on `stream`; the calls below that use the plan
 * follow on that stream.  Launches captured into a graph work on whatever
 * batch is set when they are replayed, in buffers with room for its tokens
 * (plan_set itself is not captured: LLMI_ERR_STATE; after a captured append
 * it takes only batches that can be appended, within that call's rotation
 * tables; after a captured attention only batches with work of the kinds that
 * it was captured for: single tokens or drafts of up to as many rows (tokens
 * x heads / kv_heads, up to 64 a sequence) as were set then, and longer pieces
 * if there were any; a graph captured with an empty batch serves every kind).
 * Launches of one plan must not overlap; two streams or two graphs that run at
 * once need a plan each.
 * Refused (LLMI_ERR_ARG): a slot or page out of range, a negative start or
 * count, a table too short, more than the plan was created for.
 * llmi_hip_kv8_check makes the same checks, without limits of a plan, and
 * those of an append: it needs no GPU. */
typedef struct llmi_hip_kv8_plan llmi_hip_kv8_plan;
int llmi_hip_kv8_check(const llmi_kv8_shape* shape, size_t seqs, const int32_t* slots, const int32_t* starts,
                       const int32_t* counts, const int32_t* tables, size_t table_stride);
int llmi_hip_kv8_plan_create(const llmi_kv8_shape* shape, size_t max_seqs, size_t max_tokens, size_t max_pages,
                             llmi_hip_kv8_plan** plan);
int llmi_hip_kv8_plan_set(llmi_hip_kv8_plan* plan, size_t seqs, const int32_t* slots, const int32_t* starts,
                          const int32_t* counts, const int32_t* tables, size_t table_stride, void* stream);
int llmi_hip_kv8_plan_free(llmi_hip_kv8_plan* plan);

/* Appends the batch's tokens.  q [tokens][heads][head_dim], k and v [tokens]
 * [kv_heads][head_dim], with strides (in floats) from token to token, at
 * least a row's length.  For every head of q and k:
 *   x <- x * w / sqrt(mean(x^2) + eps)     with q_norm / k_norm = w (head_dim
 *                                          floats; both or neither NULL)
 *   (x[i], x[i + d/2]) <- rotation by (cos, sin)[position][i]  with cos_t and
 *                                          sin_t [positions][head_dim / 2];
 *                                          both NULL: none
 * in 64 bits, rounded once to fp32.  q goes to q_out (q_out == q with equal
 * strides: in place); q NULL leaves q out (q_out is not touched).  k and v go
 * to the cache.  A sequence's start is its length so far, a position that it
 * is taken back to, to be written again from there, or a whole number of
 * blocks (pages shared with another sequence before it).  The rows before a
 * start that is not a whole number of blocks come from `open`, so its block
 * must be the last one of its parity (odd or even) that appends under the
 * slot have written: the sequence's last block and, unless a block of its
 * parity was written since, the one before it.  A sequence of 40 positions
 * (blocks 0 to 2) may go back to 16 or any later position; gone back to 20
 * and written to 21, into block 1 again, but not inside block 0, whose rows
 * block 2 has replaced (0 itself is allowed).  Nothing checks that here,
 * `open` being the caller's: such a start quantizes rows of another block.
 * (llmi_hip_model_forward_kv8 refuses it.)
 * LLMI_ERR_ARG: NULL pointers, strides too short, tables of fewer positions
 * than the batch has; LLMI_ERR_STATE: no batch set, or a batch that cannot be
 * appended (set without slots, two sequences with one slot, a page for new
 * tokens that appears twice). */
int llmi_hip_kv8_append_dev(const llmi_hip_kv8_plan* plan, const llmi_kv8_layer* layer, const float* q,
                            size_t q_stride, const float* k, size_t k_stride, const float* v, size_t v_stride,
                            const float* q_norm, const float* k_norm, float eps, const float* cos_t,
                            const float* sin_t, size_t positions, float* q_out, size_t q_out_stride, void* stream);
/* Causal attention of the batch's tokens over their sequences: token row t of
 * head h at position p,
 *   out[t][h] = sum_{j <= p} softmax_j(scale * q[t][h] . key_j) value_j
 * with the keys and values of head h / (heads / kv_heads), as the cache holds
 * them (the batch's own tokens have been appended before).  q and out [tokens]
 * [heads][head_dim] with strides as above; out may be q.  Sums and the
 * softmax in fp32, q carried to 22 bits or more of its row's largest, the
 * weights (times the value scales) to 22 bits or more of their row's largest;
 * results do not depend on the order in which workgroups run.  The sum of
 * weights in [0, 1] times values is taken in fp32 before its division: values
 * of more than 2^127 / positions may give inf, and results below 2^-120 have
 * fewer bits.  inf or NaN in a row of q, or in
 * a block that it sees, gives NaN for that row and head alone. */
int llmi_hip_kv8_attention_dev(const llmi_hip_kv8_plan* plan, const llmi_kv8_layer* layer, const float* q,
                               size_t q_stride, float scale, float* out, size_t out_stride, void* stream);
/* The cached keys and values of the batch's positions, code * scale, as fp32
 * rows [tokens][kv_heads][head_dim] (k or v NULL: left out). */
int llmi_hip_kv8_read_dev(const llmi_hip_kv8_plan* plan, const llmi_kv8_layer* layer, float* k, size_t k_stride,
                          float* v, size_t v_stride, void* stream);

/* ------------------------------------------------ layers of experts (device) */
/* A mixture-of-experts layer over quantized weights: a router that chooses
 * top_k of the experts for every token, products whose matrix is the chosen
 * expert's, and the whole gated MLP with its weighted sum.  No counterpart in
 * the reference, whose decoder is dense (src/model/transformer.cpp:286-292).
 * The choices stay on the device: nothing here waits for it or copies to the
 * host, and every _dev call can be captured into a graph and replayed with
 * other choices.
 *
 * Router.  Of each token's logits [tokens][experts] (stride floats apart) the
 * top_k largest are chosen, in falling order, equal ones by the lower index;
 *   p[t][e] = exp(logit - max) / sum over all experts of exp(logit - max)
 *   weights[t][j] = scale * p of the j-th choice, or with renormalise
 *                   scale * p / (the sum of p over the token's choices)
 * in fp32.  A logit of -inf or NaN (an expert that is switched off) counts as
 * p = 0 and is never chosen: where fewer than top_k are left the remaining
 * ids are -1 and their weights 0.  Logits of +inf share the weight equally.
 * ids and weights [tokens][top_k].  LLMI_ERR_ARG: more than 1024 experts, a
 * top_k above 64 or the number of experts, a stride below it, more than 2^24
 * tokens, a scale that is not finite, ids, weights and logits that overlap. */
int llmi_hip_moe_route_dev(const float* logits, size_t stride, size_t tokens, size_t experts, size_t top_k,
                           int renormalise, float scale, int32_t* ids, float* weights, void* stream);

/* The matrices [out][in] of `count` experts (at most 4096; in and out at most
 * 2^18), of one type (Q8_0 or Q4_0), laid out for the products below.  The
 * same codes and scales as llmi_hip_weight holds, copied: the sources may be
 * freed afterwards.  From weights of one shape and type (loaded in any of the
 * ways above), or from planar device memory, one expert after the other as
 * llmi_hip_quantize_dev writes them ([count][out] rows of row_bytes codes,
 * [count][out][ceil(in / 32)] scales), which has to be complete before the
 * call; both return when the copy is done.  Scales are finite and at most 2^80
 * in magnitude: a block's sum meets its scale before its row's power of two. */
typedef struct llmi_hip_experts llmi_hip_experts;
int llmi_hip_experts_create(const llmi_hip_weight* const* weights, size_t count, llmi_hip_experts** experts);
int llmi_hip_experts_upload_dev(const uint8_t* data_dev, const float* scales_dev, size_t count, size_t out, size_t in,
                                int type, llmi_hip_experts** experts);
int llmi_hip_experts_free(llmi_hip_experts* experts);

/* Products grouped by expert: for every slot s < slots with expert ids[s],
 *   y[s] = W x[s / per_row]     W = expert ids[s]'s matrix
 * x [ceil(slots / per_row)][in] and y [slots][out], rows x_stride and y_stride
 * floats apart.  With a router's ids [tokens][top_k]: slots = tokens * top_k,
 * and per_row = top_k for x of one row a token, 1 for one a slot.  Slots whose
 * id is not 0 .. count - 1 (padding tokens, -1) leave their row of y as it was.
 * per_row may be any number from 1 on (more than slots: one row for all).
 * Sums in fp32, x carried to 22 bits of each element (or 39 of its row's
 * largest); not llmi_hip_matmul_dev's order of additions, so not its bits.  A
 * row's result depends on that row, its expert and the call's sizes alone,
 * never on the other rows or on the order in which workgroups run.  inf or NaN
 * in a row of x gives inf or NaN in that row's results alone.
 * work: device memory of at least the bytes that _bytes gives, 16-byte
 * aligned; nothing has to be cleared, and nothing is kept in it from call to
 * call.  Calls that may run at the same time (two streams, two graphs) need a
 * workspace each; graphs that run one after the other may share one.
 * y must not overlap x or ids, nor the workspace any of them; columns of one
 * array, rows between each other's, are apart.  LLMI_ERR_ARG: more than 2^24
 * slots, strides too short, an overlap, a workspace too small, NULL pointers. */
int llmi_hip_moe_matmul_bytes(const llmi_hip_experts* experts, size_t slots, size_t per_row, size_t* bytes);
int llmi_hip_moe_matmul_dev(const llmi_hip_experts* experts, const int32_t* ids, size_t slots, size_t per_row,
                            const float* x, size_t x_stride, float* y, size_t y_stride, void* work, size_t work_bytes,
                            void* stream);

/* The gated MLP of the chosen experts (the decoder's, transformer.cpp:286-292,
 * with each token's own matrices):
 *   y[t] = residual[t] + sum over j < top_k of weights[t][j] *
 *          down_e( silu(gate_e x[t]) * (up_e x[t]) ),   e = ids[t][j]
 * the sum in fp32, in the order of j (of up to two tokens in the order of the
 * experts' first slots, inputs and experts in one sum, so that the other token's
 * choices may change its last bits).  h = silu(..) * (..) is carried like x.
 * gate and up of one shape and type, down of either type.  x [tokens][in],
 * residual (NULL: 0) and y [tokens][down's out], rows their strides apart; y may
 * be residual (with its stride), otherwise they must be apart, and may be x or
 * overlap it.  A choice
 * whose id is not an expert's adds nothing, whatever its weight.  Everything
 * else as for llmi_hip_moe_matmul_dev. */
int llmi_hip_moe_mlp_bytes(const llmi_hip_experts* gate, const llmi_hip_experts* down, size_t tokens, size_t top_k,
                           size_t* bytes);
int llmi_hip_moe_mlp_dev(const llmi_hip_experts* gate, const llmi_hip_experts* up, const llmi_hip_experts* down,
                         const int32_t* ids, const float* weights, size_t tokens, size_t top_k, const float* x,
                         size_t x_stride, const float* residual, size_t residual_stride, float* y, size_t y_stride,
                         void* work, size_t work_bytes, void* stream);

/* ------------------------------------------------------------- the model */

typedef struct llmi_hip_model llmi_hip_model; /* device-resident quantized decoder */
typedef struct llmi_hip_cache llmi_hip_cache; /* device KV cache of one sequence */

/* Replaces llmi::Transformer::load(model, F32 | Q8_0 | Q4_0)
 * (include/llmi/model/transformer.hpp:58, src/model/transformer.cpp:26-67):
 * quantizes every matrix (embedding, q/k/v/o, gate/up/down, untied lm_head)
 * on the GPU, or keeps them fp32 with LLMI_TYPE_F32; RMSNorm weights and
 * q/k/v biases stay fp32.  `tensors` holds
 * one fp32 array per tensor in the reference's expected_tensors() order
 * (src/model/model.cpp:135-162): embed; per layer input_layernorm, q, k, v,
 * [q_bias, k_bias, v_bias], o, post_attention_layernorm, gate, up, down;
 * final norm; [lm_head when untied].  _dev: the arrays are device pointers. */
int llmi_hip_model_create(const llmi_model_config* cfg, const float* const* tensors, int type, llmi_hip_model** model);
int llmi_hip_model_create_dev(const llmi_model_config* cfg, const float* const* tensors_dev, int type,
                              llmi_hip_model** model);
int llmi_hip_model_free(llmi_hip_model* model);
/* Transformer::weight_bytes (transformer.cpp:69-76). */
size_t llmi_hip_model_weight_bytes(const llmi_hip_model* model);

/* Transformer::new_cache (transformer.cpp:182-190): capacity
 * min(max_len, max_position_embeddings) positions, head-major fp32 K/V. */
int llmi_hip_model_new_cache(llmi_hip_model* model, size_t max_len, llmi_hip_cache** cache);
int llmi_hip_cache_free(llmi_hip_cache* cache);
/* KVCache::length / capacity / reset (transformer.hpp:29-45). */
size_t llmi_hip_cache_length(const llmi_hip_cache* cache);
size_t llmi_hip_cache_capacity(const llmi_hip_cache* cache);
int llmi_hip_cache_reset(llmi_hip_cache* cache);

/* Transformer::forward_cached (transformer.cpp:192-306): runs `n` new tokens
 * through the model, appends their K/V to `cache`, and writes the logits of
 * the last token (vocab floats) or of every new token (n x vocab) when
 * all_positions is set.  Bit-identical to the reference's logits.  Errors
 * (no tokens, id out of range, cache full or from another model) carry the
 * reference's messages. */
int llmi_hip_model_forward_cached(llmi_hip_model* model, llmi_hip_cache* cache, const int32_t* tokens, size_t n,
                                  int all_positions, float* logits);
/* forward_cached filling the reference's ForwardTrace (transformer.hpp:14-19,
 * transformer.cpp:218-221, :294, :299): states (host, NULL to skip) receives
 * (num_layers + 2) x n x hidden_size floats -- the token embeddings, the
 * output of every layer, then the final RMSNorm of every new token. */
int llmi_hip_model_forward_cached_trace(llmi_hip_model* model, llmi_hip_cache* cache, const int32_t* tokens,
                                        size_t n, int all_positions, float* logits, float* states);

/* Transformer::forward (transformer.cpp:78-166): the whole sequence without a
 * caller's cache (the model's own is reused and reset), logits of the last
 * token or of every token; states as for forward_cached_trace (NULL to
 * skip).  Bit-identical to forward_cached on a fresh cache, as the
 * reference's own test holds (tests/transformer_test.cpp:322-339); errors
 * carry forward's messages ("forward: ..."). */
int llmi_hip_model_forward(llmi_hip_model* model, const int32_t* tokens, size_t n, int all_positions, float* logits,
                           float* states);

/* Several sequences through the model at once, over a paged 8-bit cache (the
 * section above): a server's step, with sequences that decode and sequences
 * whose prompt (or a piece of it) is run side by side.  No counterpart in the
 * reference, whose server runs one request after the other
 * (src/server/server.cpp:44-49).
 * new_kv8_cache allocates every layer's pages: `pages` of page_tokens
 * positions (a multiple of 16), places for `slots` sequences, steps of at
 * most max_tokens tokens (and 65535).  The model's head size must be a multiple of 32 up
 * to 256.  Which pages a sequence has is the caller's; free the cache before
 * the model.
 * forward_kv8: sequence i's counts[i] new tokens (tokens: those of sequence 0,
 * then 1, ...) at positions starts[i] .., as llmi_hip_kv8_plan_set takes them
 * and llmi_hip_kv8_check allows them; logits receives vocab floats for the
 * last new token of each sequence that has any.  The linear layers are the
 * exact ones; keys and values are held in 8 bits, so logits are not the
 * reference's: they differ by what rounding them to 1/254 of their block's
 * largest does.  Errors: LLMI_ERR_ARG for a batch, token id or token count
 * that is refused (nothing has run then), LLMI_ERR_STATE for a cache of
 * another model, positions past the context, or a start inside a block whose
 * earlier rows are not held under the sequence's slot (llmi_hip_kv8_append_dev
 * says which are; after a step that failed on its way, none). */
typedef struct llmi_hip_kv8_cache llmi_hip_kv8_cache;
int llmi_hip_model_new_kv8_cache(llmi_hip_model* model, size_t pages, size_t page_tokens, size_t slots,
                                 size_t max_tokens, llmi_hip_kv8_cache** cache);
int llmi_hip_kv8_cache_free(llmi_hip_kv8_cache* cache);
int llmi_hip_model_forward_kv8(llmi_hip_model* model, llmi_hip_kv8_cache* cache, size_t seqs, const int32_t* slots,
                               const int32_t* starts, const int32_t* counts, const int32_t* tables,
                               size_t table_stride, const int32_t* tokens, float* logits);

/* Transformer::generate_greedy_cached (transformer.cpp:308-327): prefill,
 * then up to max_new greedy tokens (first maximum), stopping after a token in
 * stop_ids.  Writes *n_ids ids to `ids` (room for max_new). */
int llmi_hip_model_generate_greedy(llmi_hip_model* model, const int32_t* prompt, size_t n, size_t max_new,
                                   const int32_t* stop_ids, size_t n_stop, int32_t* ids, size_t* n_ids);
/* The scoring loop of llmi-perplexity on one chunk
 * (apps/llmi-perplexity/main.cpp:146-168): Transformer::forward(chunk,
 * all_positions = true) (transformer.cpp:78-166; here through a fresh cache,
 * bit-identical by the reference's own test), then for every position t in
 * [t_start, n - 1): nll[t - t_start] = -(logit_t[chunk[t + 1]] - lse_t),
 * lse_t = log(sum_v exp(double(logit_t[v] - max_t))) + max_t.  The caller
 * sums nll in order, as the app does.  Positions before t_start are still
 * run (they are the later positions' context) but not scored.  mode:
 *   LLMI_SCORE_EXACT      the reference's arithmetic throughout (logits bit-
 *                         identical; the double sum is taken as a tree, so
 *                         nll agrees to ~1e-15 relative);
 *   LLMI_SCORE_MFMA_HEAD  the lm_head on the bf16-MFMA GEMM (logits within
 *                         2e-2 of max|logit|, so each nll within 4e-2 of it);
 *   LLMI_SCORE_MFMA       every linear layer and the lm_head on the bf16-MFMA
 *                         GEMM (the fast perplexity path; not bit-exact). */
enum { LLMI_SCORE_EXACT = 0, LLMI_SCORE_MFMA_HEAD = 1, LLMI_SCORE_MFMA = 2 };
int llmi_hip_model_chunk_nll(llmi_hip_model* model, const int32_t* tokens, size_t n, size_t t_start, int mode,
                             double* nll);
/* ---------------------------------------------------------- token sampling */

/* SamplingConfig (include/llmi/model/sampling.hpp:20-24). */
typedef struct llmi_hip_sampling {
  float temperature; /* <= 0: the first maximum, nothing drawn (sampling.cpp:61) */
  size_t top_k;      /* 0 (or > n): no top-k filter */
  float top_p;       /* >= 1: no nucleus filter */
} llmi_hip_sampling;

/* llmi::sample (include/llmi/model/sampling.hpp:39, src/model/sampling.cpp:
 * 60-77) with its random number given: `target` is the number sample() draws
 * from the caller's generator, std::uniform_real_distribution<double>(0, 1)
 * on std::mt19937_64, once per call when temperature > 0 (no draw, and
 * `target` unused, otherwise).  *id is the reference's index for the same
 * logits, configuration and draw, bit for bit.  Logits may be -inf (masked
 * entries); NaN, or +inf after the division by temperature, are rejected
 * (LLMI_ERR_ARG: the reference's ranking is undefined there); every entry
 * -inf gives index 0, as the reference's fallback to argmax does.
 * _dev: logits in device memory, queued on `stream` (NULL = the library's),
 * synchronous (the index returns to the host).  n >= 1. */
int llmi_hip_sample(const float* logits, size_t n, const llmi_hip_sampling* cfg, double target, int32_t* id);
int llmi_hip_sample_dev(const float* logits, size_t n, const llmi_hip_sampling* cfg, double target, int32_t* id,
                        void* stream);
/* llmi::sampling_probabilities (sampling.hpp:32, sampling.cpp:11-58): the
 * filtered, renormalised distribution (host pointers), bit for bit. */
int llmi_hip_sampling_probabilities(const float* logits, size_t n, const llmi_hip_sampling* cfg, float* probs);
/* Testing aids, no counterpart in the reference: force every double sum of a
 * sample call onto its sequential pass (same results, slower), and report
 * which sums of the last call took the sequential pass (bit 0 softmax sum,
 * 1 top-p sum, 2 running sum of the draw, 3 renormalisation sum, 4 all of
 * the top-p sum, renormalisation sum and draw over the top-k select's
 * k <= 64 ranked values, which always run sequentially). */
int llmi_hip_sampling_set_exact_only(int on);
int llmi_hip_sampling_last_paths(int* paths);

/* One serving step on the device: forward_cached of `tokens` (transformer.cpp:
 * 192-306) and sample() on the last position's logits, which never leave HBM
 * (the loop of src/server/server.cpp:109-195 and llmi-chat, one call per
 * token).  `target` as for llmi_hip_sample. */
int llmi_hip_model_forward_sample(llmi_hip_model* model, llmi_hip_cache* cache, const int32_t* tokens, size_t n,
                                  const llmi_hip_sampling* cfg, double target, int32_t* id);
/* generate_greedy_cached with sample() in place of argmax: prefill, then up to
 * max_new sampled tokens, targets[i] being the draw of step i (room for
 * max_new; the caller draws them from its generator in order), stopping after
 * a token in stop_ids.  Timing as for generate_greedy (last_timing). */
int llmi_hip_model_generate_sampled(llmi_hip_model* model, const int32_t* prompt, size_t n, size_t max_new,
                                    const llmi_hip_sampling* cfg, const double* targets, const int32_t* stop_ids,
                                    size_t n_stop, int32_t* ids, size_t* n_ids);

/* GPU time of the last generate_greedy / generate_sampled call: the prompt
 * prefill and the decode loop (HIP events; the reference's llmi-generate --json reports the
 * same split as wall-clock seconds, apps/llmi-generate/main.cpp:329-345). */
int llmi_hip_model_last_timing(const llmi_hip_model* model, double* prefill_ms, double* decode_ms);

/* Of the last generate_sampled call: how many of its steps were redrawn with
 * a host read-back of their own.  With temperature > 0 the steps are queued
 * on the device in windows and read back once per window; a queued draw that
 * its bounds leave undecided (a target on a running sum) sends the run back
 * to that step, which is redrawn exactly before queueing resumes.  0 when
 * every step ran queued.  Diagnostic: no counterpart in the reference. */
int llmi_hip_model_last_redraws(const llmi_hip_model* model, size_t* steps);

/* The arithmetic of the model's one-token decode steps (forward_cached with
 * one token, generate_greedy / generate_sampled after the prompt).
 * LLMI_DECODE_EXACT (the default): the reference's operations in its order,
 * logits bit-identical to transformer.cpp:192-306.  LLMI_DECODE_TOLERANCE:
 * attention split over position chunks (at most 16 per head), each chunk's
 * softmax taken against its own maximum with the hardware exponential, the
 * chunks merged in the o_proj product's staging, and every matmul split
 * over K into one-wavefront workgroups whose partial sums meet by atomic
 * adds; logits within the path's floating-point tolerance of the exact
 * ones, neither bit-identical nor reproducible bit for bit.  Applies to
 * head_dim 64 / 128 with at most 16 query heads per KV head and row counts
 * of q, k, v, gate and up that are multiples of 64 (other models keep the
 * exact step); the prompt's prefill is exact in both modes.
 * No counterpart in the reference (whose decode is exact by construction):
 * a speed option for callers that accept the tolerance. */
enum { LLMI_DECODE_EXACT = 0, LLMI_DECODE_TOLERANCE = 1 };
int llmi_hip_model_set_decode_mode(llmi_hip_model* model, int mode);

/* Whether generate_greedy replays its tolerance-mode steps (no stop ids, at
 * least 8 new tokens) from one captured HIP graph -- the step's positions
 * and output slot read from device memory, one host launch per token
 * instead of ~5 per layer -- (enable != 0, the default) or launches every
 * kernel of every step (0; e.g. under profilers that do not follow graphs).
 * The same kernels and results either way.  No counterpart in the
 * reference: a launch-overhead option. */
int llmi_hip_model_set_decode_graph(llmi_hip_model* model, int enable);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* LLMI_HIP_H */
