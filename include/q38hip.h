/* libq38hip: MI355X (gfx950) kernels for the Qwen3.8 decode hot path.
 *
 * C ABI only: plain pointers and sizes.  Two families of entry points, and
 * two library extensions (sections 3 and 4):
 *
 *  1. Drop-in replacements for the reference kernel ABI
 *     (include/qwen38/qwen38_quant.h:20-49 of shyringo/qwen3.8-27b-in-c):
 *     same names, same argument meaning, same 1/0 return convention.  They
 *     take HOST pointers, stage them through HBM and run the HIP kernels.
 *
 *  2. Device-resident variants (q38hip_*): every pointer, including
 *     tensor->data, is a device pointer; work is enqueued on `stream`
 *     (a hipStream_t; NULL means the legacy default stream) and the call
 *     returns without synchronising.  Return 1 on success, 0 on an argument
 *     error (message via q38hip_last_error()).
 *
 * Results are bit-identical to the reference's x86 AVX2 CPU kernels on the
 * same inputs: integer block sums exactly, fp32 outputs in the reference's
 * lane order.
 */
#ifndef Q38HIP_H
#define Q38HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Layout-compatible with Q38Q8KBlock (include/qwen38/qwen38_quant.h:14-18). */
#define Q38_Q8_K_BLOCK_SIZE 256
typedef struct {
    float scale;
    int8_t quants[Q38_Q8_K_BLOCK_SIZE];
    int16_t sums[Q38_Q8_K_BLOCK_SIZE / 16];
} Q38Q8KBlock;

/* Layout-compatible with Q38GGUFString / Q38GGUFTensor
 * (include/qwen38/qwen38_gguf.h:57-77).  shape[0] = input width,
 * shape[1] = output rows, type = GGML type id (Q4_K 12, Q6_K 14, IQ1_M 29). */
typedef struct {
    const char *data;
    uint64_t length;
} Q38GGUFString;

typedef struct {
    Q38GGUFString name;
    uint32_t n_dims;
    uint64_t shape[8];
    uint32_t type;
    uint64_t offset;
    uint64_t nbytes;
    const uint8_t *data;
    void *iq1_s_repack;
} Q38GGUFTensor;

/* Layout-compatible with Q38GGUFMeta / Q38GGUF
 * (include/qwen38/qwen38_gguf.h:59-90): the reference's mapped GGUF file,
 * which q38_prepare_iq1_s_repacks takes. */
typedef struct {
    Q38GGUFString key;
    uint32_t type;
    uint32_t array_type;
    uint64_t count;
    const uint8_t *data;
    uint64_t data_size;
} Q38GGUFMeta;

typedef struct {
    int fd;
    const uint8_t *mapping;
    uint64_t mapping_size;
    uint32_t version;
    uint32_t alignment;
    uint64_t data_offset;
    uint64_t tensor_count;
    uint64_t metadata_count;
    Q38GGUFTensor *tensors;
    Q38GGUFMeta *metadata;
} Q38GGUF;

/* ---- 1. reference kernel ABI, host pointers ------------------------------ */

/* replaces q38_f16_to_f32, include/qwen38/qwen38_quant.h:20 */
float q38_f16_to_f32(uint16_t value);

/* replaces q38_quantize_q8_k, include/qwen38/qwen38_quant.h:24-25 */
int q38_quantize_q8_k(Q38Q8KBlock *output, const float *input,
                      uint64_t length);

/* replaces q38_tensor_row_f32, include/qwen38/qwen38_quant.h:27-28: row
 * `row` as fp32 (F32 copied, F16 / BF16 converted, Q8_0, IQ4_NL and
 * Q2_K..Q6_K decoded; other types give NaN, as in the reference) */
int q38_tensor_row_f32(float *output, const Q38GGUFTensor *tensor,
                       uint64_t row);

/* replaces q38_tensor_dot_row_f32, include/qwen38/qwen38_quant.h:30-31:
 * one row's float dot; returns 1 only for a finite result */
int q38_tensor_dot_row_f32(float *output, const float *input,
                           const Q38GGUFTensor *tensor, uint64_t row);

/* replaces q38_tensor_gemv_f32, include/qwen38/qwen38_quant.h:34-35: fp32
 * input (F32, F16, BF16, Q8_0, IQ4_NL, Q2_K..Q6_K; NaN rows for the other
 * types, as in the reference) */
int q38_tensor_gemv_f32(float *output, const float *input,
                        const Q38GGUFTensor *tensor);

/* replaces q38_tensor_gemm_f32, include/qwen38/qwen38_quant.h:44-46;
 * batch-major output, any batch_size >= 1 */
int q38_tensor_gemm_f32(float *output, const float *input,
                        uint32_t batch_size, uint64_t input_length,
                        const Q38GGUFTensor *tensor);

/* replaces q38_tensor_gemv_q8_k, include/qwen38/qwen38_quant.h:38-40
 * (every Q8_K-path format: Q2_K, Q3_K, Q4_K, Q5_K, Q6_K, IQ1_S, IQ1_M,
 * IQ2_XXS, IQ2_XS, IQ2_S, IQ3_XXS, IQ3_S, IQ4_NL, IQ4_XS) */
int q38_tensor_gemv_q8_k(float *output, const Q38Q8KBlock *input,
                         uint64_t input_length,
                         const Q38GGUFTensor *tensor);

/* replaces q38_tensor_gemm_q8_k, include/qwen38/qwen38_quant.h:48-50;
 * output is batch-major, output[token * rows + row]; any batch_size >= 1 */
int q38_tensor_gemm_q8_k(float *output, const Q38Q8KBlock *input,
                         uint32_t batch_size, uint64_t input_length,
                         const Q38GGUFTensor *tensor);

/* replace q38_prepare_iq1_s_repacks / q38_release_iq1_s_repacks,
 * include/qwen38/qwen38_quant.h:54-55 (argument: the caller's Q38GGUF).
 * The GPU kernels read IQ1_S blocks as stored, so no view is built:
 * prepare returns 1 for a non-NULL argument and changes nothing. */
int q38_prepare_iq1_s_repacks(Q38GGUF *gguf);
void q38_release_iq1_s_repacks(Q38GGUF *gguf);

/* ---- 2. device-resident variants ---------------------------------------- */

/* Device form of q38_quantize_q8_k (src/qwen38/qwen38_quant.c:50-88):
 * `rows` independent fp32 rows of `length` elements each. */
int q38hip_quantize_q8_k(Q38Q8KBlock *output, const float *input,
                         uint64_t length, uint32_t rows, void *stream);

/* Device form of q38_tensor_gemm_q8_k (src/qwen38/qwen38_quant.c:2950-3169);
 * batch_size = 1 is q38_tensor_gemv_q8_k (:2833-2922).  Any batch_size >= 1:
 * up to 8 tokens and prompt batches take one launch; shapes without a prompt
 * kernel run as consecutive launches of up to 8 tokens (every token's outputs
 * are independent of the rest of the batch, so the bits are the same). */
int q38hip_gemm_q8_k(float *output, const Q38Q8KBlock *input,
                     uint32_t batch_size, uint64_t input_length,
                     const Q38GGUFTensor *tensor, void *stream);

/* Device form of q38_tensor_gemm_f32 (src/qwen38/qwen38_quant.c:2924-2948):
 * input is batch_size rows of input_length fp32 values; batch_size = 1 is
 * q38_tensor_gemv_f32 (:2812-2831).  Each output is the row's single fmaf
 * chain in the reference's element order (q38_dot_row, :2768-2810). */
int q38hip_gemm_f32(float *output, const float *input, uint32_t batch_size,
                    uint64_t input_length, const Q38GGUFTensor *tensor,
                    void *stream);

/* Device form of q38_tensor_row_f32 (src/qwen38/qwen38_quant.c:3185-3223)
 * for rows first_row .. first_row + row_count - 1: output[r * width + e]. */
int q38hip_row_f32(float *output, const Q38GGUFTensor *tensor,
                   uint64_t first_row, uint32_t row_count, void *stream);

/* Row-wise first-maximum index (q38_argmax, src/qwen38/qwen38_model.c:
 * 1228-1239) of `rows` rows of `count` floats; index_out[rows].  Partial
 * maxima go to a per-device scratch buffer that the library grows on demand
 * (after synchronising the device): calls that overlap on one device race. */
int q38hip_argmax(uint32_t *index_out, const float *values, uint32_t count,
                  uint32_t rows, void *stream);

/* No counterpart in the reference: q38hip_argmax for callers that cannot
 * allocate device memory (code under HIP graph capture, serving loops or
 * harnesses that forbid hipMalloc).  It allocates nothing: the partial
 * maxima go to a fixed 64 KiB array in the library's device memory instead
 * of the growable scratch, so ceil(count / 4096) * rows must be at most 8192
 * (248320-wide rows: up to 134 rows); larger calls return 0 with a message.
 * Every call on one device shares that array, so calls that overlap on one
 * device (on any streams) race.  Results are those of q38hip_argmax. */
int q38hip_argmax_noalloc(uint32_t *index_out, const float *values, uint32_t count,
                          uint32_t rows, void *stream);

/* Device form of q38_sample (src/qwen38/qwen38_sampler.c:51-119): the
 * token drawn from `logits` (vocabulary_size floats, device memory) into
 * *token (a device word).  The sampler's fields
 * (include/qwen38/qwen38_sampler.h:10-18) come as arguments: *state is the
 * xorshift64* state in HOST memory, read at the call and advanced before it
 * returns exactly as q38_sample advances it (one step when temperature > 0
 * and top_k > 1, none otherwise); presence, when not NULL, is presence_size
 * bytes of DEVICE memory (nonzero = token observed).  Token and state are
 * those of q38_sample on the same logits, bit for bit, NaN and infinite
 * logits included.  Limits: vocabulary_size <= 2^20 and, when sampling,
 * min(top_k, vocabulary_size) <= 1024; beyond them the call returns 0 with
 * a message.  Working memory is a per-device buffer (2 MiB, allocated on
 * the first call on a device): calls that overlap on one device race. */
int q38hip_sample(uint32_t *token, uint64_t *state, const float *logits, uint32_t vocabulary_size,
                  float temperature, float top_p, float presence_penalty, uint32_t top_k,
                  const uint8_t *presence, uint32_t presence_size, void *stream);

/* Greedy acceptance of a verify batch (src/qwen38/qwen38_model.c:1662-1702):
 * targets[rows] are the per-row argmaxes, drafts[rows] the draft ids.
 * result[0] = consumed, result[1] = matched, result[2] = next,
 * result[3 .. 3+consumed) = accepted tokens.  result needs rows + 3 words. */
int q38hip_accept(uint32_t *result, const uint32_t *targets,
                  const uint32_t *drafts, uint32_t rows, void *stream);

/* Library extension (no counterpart in the reference): the 16-row tiled
 * layout of a Q4_K matrix that the model engine keeps beside the GGUF
 * layout for its GEMVs and GEMMs.  Tile k holds rows 16k..16k+15 as
 * [block][row][144 bytes]; the last tile is zero-padded.
 * q38hip_tiled_q4k_bytes: size of the tiled copy of `rows` rows of
 * `input_length` elements.  q38hip_repack_q4k_tiles: write it from the
 * row-major matrix (both in device memory). */
uint64_t q38hip_tiled_q4k_bytes(uint32_t rows, uint64_t input_length);
int q38hip_repack_q4k_tiles(void *tiled, const void *q4k_rows, uint32_t rows,
                            uint64_t input_length, void *stream);

/* q38hip_gemm_q8_k over a tiled Q4_K copy: output[t * rows + r] for
 * t < batch_size (at least 1: one launch for one token or a prefill batch,
 * else launches of 2..8 tokens), input_length 5120, 6144, 10240 or 17408.
 * The results are those of q38hip_gemm_q8_k bit for bit. */
int q38hip_gemm_q8_k_tiled(float *output, const Q38Q8KBlock *input,
                           uint32_t batch_size, uint64_t input_length,
                           const void *tiled, uint32_t rows, void *stream);

/* Library extension: the same 16-row tiled copy for IQ1_M
 * ([tile = row / 16][block][row % 16][56 bytes], rows past the last zero),
 * which the engine keeps beside the row-major blocks.
 * q38hip_tiled_iq1m_bytes: its size (0 for a bad shape);
 * q38hip_repack_iq1m_tiles: write it from the row-major matrix (both in
 * device memory, the copy 8-byte aligned); q38hip_gemm_q8_k_iq1m_tiled:
 * q38hip_gemm_q8_k over it for batch_size 1..8 (output[t * rows + r]),
 * input_length 5120, 6144, 10240 or 17408, bit for bit q38hip_gemm_q8_k's
 * results. */
uint64_t q38hip_tiled_iq1m_bytes(uint32_t rows, uint64_t input_length);
int q38hip_repack_iq1m_tiles(void *tiled, const void *iq1m_rows, uint32_t rows,
                             uint64_t input_length, void *stream);
int q38hip_gemm_q8_k_iq1m_tiled(float *output, const Q38Q8KBlock *input,
                                uint32_t batch_size, uint64_t input_length,
                                const void *tiled, uint32_t rows, void *stream);

/* Library extension: the full-attention decode core of one layer on the
 * device, for kernel-level use and tests.  It is the reference's static
 * q38_full_core (src/qwen38/qwen38_model.c:816-885) for `rows` consecutive
 * positions position .. position + rows - 1, row t seeing positions
 * 0 .. position + t (q38_batch_full_attention, :1089-1119): per-head RMS
 * norms of q and k (q_norm, k_norm: 256 floats), RoPE, the K/V cache write
 * of each row, scores, softmax and the sigmoid-gated output.
 *   q_and_gate: row t at t * in_stride floats, 24 heads x (256 q | 256 gate);
 *   key, value: row t at t * in_stride floats, 1024 each;
 *   key_cache: [context_length][1024] fp32 (one layer); value_cache:
 *     channel-major [1024][pitch] fp32 with pitch = context_length rounded
 *     up to a multiple of 32 (position p of channel e at e * pitch + p);
 *     positions before `position` already filled, positions position ..
 *     position + rows - 1 are written;
 *   attention: [rows][6144] gated output; attention_q8k (optional, may be
 *     NULL): its Q8_K blocks [rows][24], the input of the output projection.
 * All pointers are device pointers.  position + rows <= context_length <= 524256.
 * Allocates and frees its working buffers (the RoPE table of the context,
 * the scores) and synchronises `stream` before returning. */
int q38hip_attention_rows(float *attention, Q38Q8KBlock *attention_q8k, const float *q_and_gate,
                          const float *key, const float *value, uint64_t in_stride,
                          const float *q_norm, const float *k_norm, float *key_cache,
                          float *value_cache, uint32_t context_length, uint32_t position,
                          uint32_t rows, void *stream);

/* ---- 3. paged 8-bit key/value cache ---------------------------------------
 *
 * Library extension (no counterpart in the reference, whose cache is fp32 and
 * belongs to one sequence): keys and values of many sequences as 8-bit codes
 * in pages that sequences can share.  Everything lives in device memory that
 * the caller owns and describes by a Q38KVPages; the calls enqueue on
 * `stream` (of the current device, the cache's), allocate nothing, read nothing
 * back and can be captured into a HIP graph.  Calls on one cache have to be
 * ordered (one stream, or events).
 *
 *   data    [layers][pages][2][kv_heads][page_tokens * head_dim] codes, 16-byte
 *           aligned: keys (half 0) are [token][channel], values (half 1)
 *           [channel][token]
 *   scales  [layers][pages][2][kv_heads] powers of two; a code c stands for
 *           c * scale (int8: -127 .. 127; e4m3: OCP float8, up to 448)
 *   refs    [pages]: the sequences that a page belongs to; 0 is a free page
 *   tables  [sequences][table_entries]: page of tokens entry * page_tokens ..;
 *           -1 behind a sequence's last page
 *   lengths [sequences]: tokens
 *   status  [1]: Q38_KV_* bits that calls set (never clear) for what they find
 *           in device memory; a host program reads it when it likes
 *
 * page_tokens is 16, 32, 64 or 128, head_dim 64, 128 or 256, table_entries *
 * page_tokens below 2^31.  A page serves all layers.  All ids are 32-bit words
 * in device memory.  Ids and pages outside the cache are never followed: they
 * set a status bit, and what they stand for holds no tokens.  (Append alone
 * leaves the rows of a bad id out without a bit: the extend call before it and
 * the attention call behind it report the id.) */
enum { Q38_KV_INT8 = 0, Q38_KV_E4M3 = 1 };
enum {
    Q38_KV_BAD_SEQUENCE = 1,   /* an id outside the cache; extend: twice in a call, or fewer than 0 rows; fork: a child as parent */
    Q38_KV_POOL_FULL = 2,      /* extend: fewer free pages than asked for; nothing was done */
    Q38_KV_TABLE_FULL = 4,     /* extend: longer than a table holds; nothing was done */
    Q38_KV_BAD_PAGE = 8,       /* a page outside the pool */
    Q38_KV_NOT_EMPTY = 16,     /* fork: the child holds tokens; that pair was left out */
    Q38_KV_BAD_ROWS = 32       /* append, attention: row_starts that decrease; nothing was done */
};
typedef struct {
    uint8_t *data;
    float *scales;
    int32_t *refs;
    int32_t *tables;
    int32_t *lengths;
    int32_t *status;
    uint32_t layers, pages, page_tokens, kv_heads, head_dim, sequences, table_entries, type;
} Q38KVPages;

/* An empty cache: every page free, every table -1, lengths and status 0. */
int q38hip_kv_reset(const Q38KVPages *cache, void *stream);

/* Bytes of the workspace that extend and compact take (16-byte aligned device
 * memory, one call at a time); 0 for a bad cache. */
uint64_t q38hip_kv_workspace_bytes(const Q38KVPages *cache);

/* sequences[i] grows by rows[i] tokens (count <= 1024, distinct ids): its
 * table gets the pages, lowest free page first in the order of the items, and
 * its length the sum.  A partly filled last page that other sequences share,
 * after the items before i took their copies, is copied in all layers first,
 * so what append writes is the sequence's own.  All items or none: see the
 * status bits. */
int q38hip_kv_extend(const Q38KVPages *cache, const int32_t *sequences, const int32_t *rows, uint32_t count,
                     void *workspace, void *stream);

/* Sequence children[i], which has to be empty, becomes the first lengths[i]
 * tokens of parents[i] (all of them where lengths is NULL) and shares their
 * pages.  Children (count <= 65536) are distinct and none is a parent in the
 * same call. */
int q38hip_kv_fork(const Q38KVPages *cache, const int32_t *parents, const int32_t *children, const int32_t *lengths,
                   uint32_t count, void *stream);

/* sequences[i] keeps its first lengths[i] tokens (0: it is freed; more than it
 * has: unchanged); pages that no sequence holds any more are free. */
int q38hip_kv_truncate(const Q38KVPages *cache, const int32_t *sequences, const int32_t *lengths, uint32_t count,
                       void *stream);

/* The pages in use move to the front of the pool, in place: with n in use, the
 * j-th of them at or above n goes to the j-th free page below n.  The first
 * two words of the workspace then hold the number of moves and n. */
int q38hip_kv_compact(const Q38KVPages *cache, void *workspace, void *stream);

/* Pages sources[i] to pages targets[i], codes and scales of all layers
 * (a negative id: no copy); a target is no other pair's source or target. */
int q38hip_kv_copy(const Q38KVPages *cache, const int32_t *sources, const int32_t *targets, uint32_t count,
                   void *stream);

/* Rows of the attention calls: sequences[i] owns rows row_starts[i] ..
 * row_starts[i + 1] - 1 of total_rows (device words, non-decreasing), or
 * total_rows / count rows each where row_starts is NULL.  They are the last
 * rows of the sequence's tokens: row t of r stands at position
 * length - r + t.  Rows that no sequence owns are neither read nor written.
 * type is the GGML id of the rows: F32 0, F16 1, BF16 30.  What a launch cannot
 * hold is refused: from about 2^21 sequences to an append on, 2^24 to the others. */

/* Quantises the rows' keys and values ([kv_heads][head_dim], rows row_stride
 * elements apart) into the pages of one layer.  Per page, head and half: with
 * a the largest magnitude among its new tokens and k >= -100 the least with a
 * <= M 2^k (M = 127 or 448), the scale becomes 2^k where the page holds no
 * older token, else the larger of 2^k and what it was, and older codes are
 * rounded to a scale that grew; new codes are value / scale, rounded to
 * nearest, ties to even.  A value that is not finite makes the scale NaN.  The
 * sequences of a call are distinct, and the pages that their rows fall into
 * theirs alone, as extend leaves them. */
int q38hip_kv_append(const Q38KVPages *cache, uint32_t layer, const void *key, const void *value, uint32_t type,
                     uint64_t row_stride, const int32_t *sequences, const int32_t *row_starts, uint32_t count,
                     uint32_t total_rows, void *stream);

/* Causal attention of the rows' queries over their sequences' tokens in one
 * layer: output[row][head] = sum softmax(scale q.k) v over positions 0 ..
 * length - r + t, times sigmoid(gate) where gate is not NULL; zeros for a row
 * that sees nothing.  Query head h reads key/value head h / (heads /
 * kv_heads).  Head h of a row begins at row * query_row_stride + h *
 * query_head_stride elements of query and of gate; output rows are
 * output_row_stride elements apart, heads head_dim.  Sums, maxima and totals are
 * in fp32.  In the products queries of fp32 rows keep 22 bits, and a weight times
 * its page's value scale 11 (16-bit rows) or 22 (fp32 rows), or 2^-31 of the
 * largest where that is more: a page whose values count that little is left out,
 * in channels too where the pages that count hold zeros.
 * q38hip_kv_attention_workspace_bytes: device memory for the call (16-byte
 * aligned; 0: none needed, or a bad call). */
uint64_t q38hip_kv_attention_workspace_bytes(const Q38KVPages *cache, uint32_t type, uint32_t heads, uint32_t count,
                                             uint32_t total_rows);
int q38hip_kv_attention(const Q38KVPages *cache, uint32_t layer, void *output, const void *query, const void *gate,
                        uint32_t type, uint32_t heads, uint64_t query_row_stride, uint64_t query_head_stride,
                        uint64_t output_row_stride, float scale, const int32_t *sequences, const int32_t *row_starts,
                        uint32_t count, uint32_t total_rows, void *workspace, void *stream);

/* ---- 4. operators of a decoder layer --------------------------------------
 *
 * Library extension (no counterpart in the reference, whose engine does these
 * in fp32, in its own order, for one model): for programs that bring their own
 * model to the paged cache.  Every pointer is a device pointer; the calls
 * enqueue on `stream` (of the current device, which holds the tensors),
 * allocate nothing, read nothing back, keep nothing from one call to the next
 * and can be captured into a HIP graph.  Calls do not share memory that the
 * caller does not share between them.  Rows, widths and counts are at least 1.
 *
 * type is the GGML id of elements: F32 0, F16 1, BF16 30.  Sums, means and
 * totals are in fp32 or more; a result is rounded once, to its type, ties to
 * even.  Strides are in elements; elements of a row (of a head) are contiguous.
 * Any alignment of elements is taken; 16-byte aligned rows are faster.
 * Outputs overlap no inputs except where said, and no output's rows overlap.
 *
 * Rows in 8 bits: codes [rows][width], e4m3 (OCP float8), and scales
 * [rows][pitch] with one byte e for each 128 neighbours of a row (the last
 * ones of a row may be fewer): a code c stands for c * 2^(e - 127).  pitch is
 * the number of blocks rounded up to a multiple of 4; bytes behind the last
 * block are 0.  With a the block's largest magnitude, e - 127 is the least k >=
 * -100 with a <= 448 * 2^k, so dividing by the scale is exact and a code is one
 * rounding.  A block that holds a value that is not finite has scale 255 (NaN) and codes
 * 0x7f (NaN). */

/* bytes between the scales of two rows of `width` elements; 0 for width 0 or above 2^24 */
uint32_t q38hip_e4m3_scale_pitch(uint64_t width);

/* Rows into 8 bits: x, or x * silu(gate) where gate is not NULL (gate / (1 +
 * e^-gate), the middle of a SwiGLU).  width up to 2^24, rows * ceil(width /
 * 2048) below 2^24. */
int q38hip_quantize_e4m3(uint8_t *codes, uint8_t *scales, const void *x, uint64_t x_row_stride, const void *gate,
                         uint64_t gate_row_stride, uint32_t type, uint64_t width, uint32_t rows, void *stream);

/* Root-mean-square norm of rows: t = x, or x + addend rounded to `type` and
 * stored in total where addend is not NULL; y = t / sqrt(mean(t^2) + eps) *
 * (weight + weight_offset).  y goes to output, in `type`, where that is not
 * NULL, and to codes and scales where those are not NULL; one of them at least.
 * weight has `width` elements of weight_type.  total may be x or addend itself
 * (same pointer and stride), output x or addend, total not output.  width up to
 * 2^24, rows below 2^24, with widths above 8192 below 2^22; 2^40 elements. */
int q38hip_rms_norm(void *output, uint64_t output_row_stride, uint8_t *codes, uint8_t *scales, void *total,
                    uint64_t total_row_stride, const void *x, uint64_t x_row_stride, const void *addend,
                    uint64_t addend_row_stride, uint32_t type, const void *weight, uint32_t weight_type,
                    float weight_offset, float eps, uint64_t width, uint32_t rows, void *stream);

/* Rows in 8 bits times a matrix in e4m3: output[t][r] = sum over blocks b of
 * 2^(scales[t][b] - 127) * weight_scales[r / 128][b] * (the block's products of
 * codes[t] and weight[r]), for t < batch_size, r < rows.  weight is
 * [rows][input_length] codes, weight_scales [ceil(rows / 128)][blocks] floats;
 * input_length is a multiple of 16, codes and weight 16-byte aligned, scales 4.
 * output is of `type`, rows output_row_stride elements apart.  Products of codes are
 * exact and their sums in fp32; for 16-bit outputs the matrix unit adds a block's
 * products at 13 bits below the largest of them (about 3e-5 of the result's norm).
 * A block's part is formed in fp32: for F32 outputs what of 2^(scales - 127) is
 * beyond 2^-100 or 2^100 goes to weight_scales first, the rest to the products;
 * for 16-bit ones all of it goes to the block's sum of products (2^-18 to 2^25 in
 * size).  What leaves fp32's normal range on the way is infinite (NaN where the block's
 * sum is 0), or 0 or has fewer bits.
 * batch_size, input_length and rows up to 2^24, 2^36 outputs.
 * q38hip_gemm_e4m3_workspace_bytes: device memory for the call, 16-byte aligned
 * (0: none needed, or a bad call). */
uint64_t q38hip_gemm_e4m3_workspace_bytes(uint32_t batch_size, uint64_t input_length, uint32_t rows);
int q38hip_gemm_e4m3(void *output, uint32_t type, uint64_t output_row_stride, const uint8_t *codes,
                     const uint8_t *scales, uint32_t batch_size, uint64_t input_length, const uint8_t *weight,
                     const float *weight_scales, uint32_t rows, void *workspace, void *stream);

/* Rotary positions: in each head of each row, pair i of `pairs` is turned by
 * positions[row] * frequencies[i] radians and multiplied by magnitude: (a, b)
 * becomes magnitude * (a cos - b sin, b cos + a sin).  The pair is channels
 * 2i and 2i + 1 where interleaved is not 0, else i and i + pairs; channels from
 * 2 * pairs on are copied.  Angles and their sines and cosines are formed in fp64, so
 * far positions keep the accuracy of near ones.  output may be x itself (same pointer and strides).
 * 2 * pairs <= head_dim <= 1024, heads * head_dim <= 2^20, rows below 2^24. */
int q38hip_rotary(void *output, uint64_t output_row_stride, uint64_t output_head_stride, const void *x,
                  uint64_t x_row_stride, uint64_t x_head_stride, uint32_t type, uint32_t rows, uint32_t heads,
                  uint32_t head_dim, const int32_t *positions, const float *frequencies, uint32_t pairs,
                  int interleaved, float magnitude, void *stream);

/* Causal attention of whole prompts, packed: sequence i of count owns rows
 * row_starts[i] .. row_starts[i + 1] - 1 of total_rows (device words,
 * non-decreasing).  output[row][head] = sum softmax(scale q.k) v over the rows
 * of its sequence up to itself, times sigmoid(gate) where gate is not NULL.
 * What other sequences and later rows hold, NaN included, has no part in it.
 * Calls with values or keys that are not finite take longer: 3 to 8 times where
 * many rows see them, and the up to 64 rows before such a one are formed one by one
 * (0.3 ms each at 4096 tokens of 24 heads of 256), as all rows are that see infinite
 * keys, or infinite values of F16 (up to 60 times as long).
 * Rows that no sequence owns are not written.  Where row_starts decrease, what
 * is written to rows of the output is unspecified.  Query head h reads
 * key/value head h / (heads / kv_heads).  Head h of a row begins at row *
 * query_row_stride + h * query_head_stride elements of query and of gate;
 * rows of key, value and output are their strides apart, heads head_dim, which
 * is 64, 128 or 256, of at most 65535 heads; up to 2^24 rows and sequences,
 * total_rows * heads up to 2^30, scale up to 2^127.  Scores, statistics and sums are in
 * fp32; in the second product the weights of 16-bit rows have 8 (BF16) or 11 (F16)
 * bits, those of F16 below 2^-9 of the largest weight of the same 32 or 64 keys
 * fewer (they are off by up to 2^-20 of that one). */
int q38hip_prompt_attention(void *output, uint64_t output_row_stride, const void *query, const void *gate,
                            uint64_t query_row_stride, uint64_t query_head_stride, const void *key,
                            uint64_t key_row_stride, const void *value, uint64_t value_row_stride, uint32_t type,
                            uint32_t heads, uint32_t kv_heads, uint32_t head_dim, float scale,
                            const int32_t *row_starts, uint32_t count, uint32_t total_rows, void *stream);

/* Last argument error of the calling thread ("" when none). */
const char *q38hip_last_error(void);

/* Synchronise the device; returns 1 when no HIP error is pending. */
int q38hip_synchronize(void);

#ifdef __cplusplus
}
#endif

#endif
