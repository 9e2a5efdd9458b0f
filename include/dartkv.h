/*
 * dartkv.h — C ABI of the MI355X-native DartKV compressed-KV path.
 *
 * libdartkv_hip.so exports these functions.  Every pointer is a device pointer
 * unless stated otherwise.  Every call enqueues work on the given HIP stream
 * (a hipStream_t passed as void*, NULL = default stream), returns immediately,
 * and returns DKV_OK (0) or an error code.  On error, dkv_last_error() returns a
 * thread-local message.  Nothing here allocates device memory: callers pass
 * outputs and workspace.  A call's launches pass records through its workspace, so
 * one workspace serves the calls of one host thread on one stream.
 *
 * Element types (the *_dtype arguments) use DKV_DTYPE_*.  Sources, outputs,
 * caches and queries may be float64, float32, float16 or bfloat16 (the page
 * kernels of dkv_decode_attention take bf16 / fp16 caches; everything else
 * takes all four).  As in the reference, quantization runs in the source
 * dtype: a float64 source in IEEE double with eps 1e-6, its float64 scale and
 * minimum converted to a 16-bit metadata dtype through float32, as torch does.
 *
 * Layouts are the reference's tensor layouts (reference src/dart/quantization.py,
 * src/dart/mixed.py), so a reference-side binding can hand over the storage
 * of its QuantizedTensor / MixedQuantizedKey fields unchanged.
 */
#ifndef DARTKV_H
#define DARTKV_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DKV_DTYPE_F32 0
#define DKV_DTYPE_F16 1
#define DKV_DTYPE_BF16 2
#define DKV_DTYPE_F64 3

#define DKV_OK 0
#define DKV_ERR_INVALID 1     /* bad shape / argument (Python: ValueError)     */
#define DKV_ERR_UNSUPPORTED 2 /* valid but not implemented here (ValueError)   */
#define DKV_ERR_DTYPE 3       /* bad element type (Python: TypeError)          */
#define DKV_ERR_HIP 4         /* HIP runtime failure (Python: RuntimeError)     */

#define DKV_KEY_DENSE 0
#define DKV_KEY_UNIFORM 1
#define DKV_KEY_MIXED 2
#define DKV_VALUE_DENSE 0
#define DKV_VALUE_UNIFORM 1

#define DKV_SELECT_MAGNITUDE 0
#define DKV_SELECT_VARIANCE 1
#define DKV_SELECT_GIVEN 2 /* caller supplies per-head indices ("random" strategy) */

/* Thread-local description of the last error on this thread. */
const char* dkv_last_error(void);

/* ABI version (17); bumps when a struct or an entry point below changes. */
int dkv_abi_version(void);

/*
 * Uniform group quantization of `rows` rows of `n` elements each, groups of
 * `group` consecutive elements, last group padded by repeating the row's last
 * element.  Element (r, i) of the source is at src[r * row_stride + i * elem_stride].
 *
 * Outputs (contiguous): values[rows][packed_bytes] with element i of a row at
 * byte i / (8/bits), bits [(i % (8/bits)) * bits, ...) (LSB first);
 * scale[rows][groups], zero[rows][groups] in meta_dtype.
 *
 * Replaces reference src/dart/quantization.py:134-204 (`quantize`, after its
 * movedim to the last axis) and :213-223 (`quantize_axis`); the cache calls it
 * for value pages (src/dart/cache.py:505-512).
 */
int dkv_quantize_rows(const void* src, int src_dtype, int64_t rows, int64_t n,
                      int64_t row_stride, int64_t elem_stride, int bits, int64_t group,
                      uint8_t* values, void* scale, void* zero, int meta_dtype, void* stream);

/*
 * dkv_quantize_rows over `blocks` blocks of `block_rows` rows each, the form a
 * token slice of a [B, H, T, D] tensor takes: row r = blk * block_rows + i
 * (0 <= i < block_rows) starts at src[blk * block_stride + i * row_stride] and
 * its elements are contiguous.  Outputs are laid out as for dkv_quantize_rows
 * with rows = blocks * block_rows, so the result equals dkv_quantize_rows on
 * the contiguous copy of the slice without making that copy.
 *
 * Replaces the same reference code as dkv_quantize_rows: the cache quantizes
 * value pages cut out of the appended tensor along tokens
 * (src/dart/cache.py:505-512, src/dart/quantization.py:134-204).
 */
int dkv_quantize_row_blocks(const void* src, int src_dtype, int64_t blocks, int64_t block_stride,
                            int64_t block_rows, int64_t n, int64_t row_stride, int bits, int64_t group,
                            uint8_t* values, void* scale, void* zero, int meta_dtype, void* stream);

/*
 * Value rows for dkv_quantize_key_pages to quantize in the same call, with the
 * meaning of dkv_quantize_row_blocks's arguments: `blocks` blocks of
 * `block_rows` rows of `n` contiguous elements, row r = blk * block_rows + i at
 * src[blk * block_stride + i * row_stride]; outputs laid out as for
 * dkv_quantize_rows.
 */
typedef struct dkv_value_rows_args {
  const void* src;
  int64_t src_dtype;
  int64_t blocks, block_stride, block_rows, n, row_stride;
  int64_t bits, group;
  uint8_t* values;
  void* scale;
  void* zero;
  int64_t meta_dtype;
  /* Optional (NULL: no check): a uint32 the device can write (device memory,
   * or pinned host memory, read after a stream synchronization without a
   * copy) set to 1 when a group holds a NaN or an infinity (the reference
   * raises ValueError for such inputs, src/dart/quantization.py:159-160);
   * never cleared by the library. */
  uint32_t* nonfinite;
  /* Output placement: source row blk * block_rows + i goes to output row
   * blk * out_block_rows + out_row0 + i (out_block_rows 0: block_rows, the
   * contiguous layout), so a caller can quantize new token rows straight into
   * a [B][H][capacity][...] store at token offset out_row0. */
  int64_t out_block_rows, out_row0;
} dkv_value_rows_args;

/*
 * dkv_quantize_row_blocks described by a dkv_value_rows_args, with its
 * optional non-finite flag: the form the cache uses for value pages that are
 * quantized without keys (reference src/dart/cache.py:457-470 and :505-512,
 * quantize at src/dart/quantization.py:134-204).
 */
int dkv_quantize_value_rows(const dkv_value_rows_args* args, void* stream);

/*
 * Key quantization along tokens for `n_pages` pages of `page_tokens` tokens.
 * Source keys are [B, H, T, D]; page p covers tokens
 * [p * page_tokens, (p + 1) * page_tokens) of `src`, element (b, h, t, d) at
 * src[b*sb + h*sh + t*st + d*sd].
 *
 * key_mode DKV_KEY_MIXED (Dart promotion, reference src/dart/mixed.py:166-244,
 * channel choice :119-163): per page, fields laid out as the reference's
 *   low   [B][H][D][G][nb]  uint8, nb = ceil(group/4)
 *   high  [B][H][K][G][nb]  uint8 (upper 2 bits of promoted channels, top-k order)
 *   idx   [B][H][K]         int32
 *   scale [B][H][D][G], zero [B][H][D][G] in meta_dtype
 * with G = ceil(page_tokens / group) and K = `promoted`.  `selection` picks the
 * channel score (DKV_SELECT_*); DKV_SELECT_GIVEN reads given_idx[H][K].
 *
 * key_mode DKV_KEY_UNIFORM (reference src/dart/quantization.py:213-223 with
 * axis=-2, as src/dart/cache.py:497-502 calls it):
 *   low   [B][H][D][pk]     uint8 codes of the padded token axis, pk = ceil(G*group / (8/bits))
 *   scale [B][H][D][G], zero [B][H][D][G]
 * (high and idx unused).
 *
 * Page p's fields start at field + p * field_page_stride (strides in bytes).
 * Replaces reference src/dart/cache.py:481-503 (`_quantize_key_pages`).
 */
struct dkv_copy_block; /* defined with dkv_copy_token_blocks below */

typedef struct dkv_key_pages_args {
  const void* src;
  int64_t src_dtype;
  int64_t B, H, D, page_tokens, n_pages;
  int64_t sb, sh, st, sd; /* element strides of the source */
  int64_t key_mode, bits, group, promoted, selection;
  const int32_t* given_idx;
  int64_t meta_dtype;
  uint8_t* low;
  int64_t low_page_stride;
  uint8_t* high;
  int64_t high_page_stride;
  int32_t* idx;
  int64_t idx_page_stride;
  void* scale;
  int64_t scale_page_stride;
  void* zero;
  int64_t zero_page_stride;
  /* Optional (NULL: keys only): the value rows of the same tokens, quantized
   * by this call too.  The reference quantizes a page's keys and its values
   * one after the other (src/dart/cache.py:472-479); given both, the library
   * runs the value kernel alongside the key path's serial channel selection. */
  const dkv_value_rows_args* values;
  /* Optional (NULL: no check): a uint32 the device can write (as in
   * dkv_value_rows_args) set to 1 when a key group holds a NaN or an
   * infinity (reference src/dart/mixed.py:187-188 and
   * src/dart/quantization.py:159-160 raise ValueError); never cleared. */
  uint32_t* nonfinite;
  /* Optional (n_copies 0: none): up to DKV_COPY_MAX_BLOCKS dense token-row
   * copies, with the meaning dkv_copy_token_blocks gives them, made by this
   * call too.  An append keeps its sink tokens and its held tail dense next
   * to the pages it quantizes (reference src/dart/cache.py:183-185 and
   * :417-418, :451-467); given here, the library runs them inside a quantize
   * launch where one has room for them. */
  const struct dkv_copy_block* copies;
  int64_t n_copies;
} dkv_key_pages_args;

int dkv_quantize_key_pages(const dkv_key_pages_args* args, void* stream);

/*
 * Copy the token rows of up to DKV_COPY_MAX_BLOCKS dense blocks in one
 * launch: block j sets dst[b][h][t] = src[b][h][t] (row_bytes bytes) for
 * b < B, h < H, t < T; the strides are in bytes, and a block's source and
 * destination must not overlap.  Blocks of zero rows are skipped.  This is
 * how an append keeps its dense tokens: reference src/dart/cache.py:183-185
 * (the sink tokens' clone) and :417-418, :451-467 (the pending tail's clone).
 */
#define DKV_COPY_MAX_BLOCKS 8

typedef struct dkv_copy_block {
  const void* src;
  void* dst;
  int64_t B, H, T, row_bytes;
  int64_t src_sb, src_sh, src_st;
  int64_t dst_sb, dst_sh, dst_st;
} dkv_copy_block;

int dkv_copy_token_blocks(const dkv_copy_block* blocks, int64_t n_blocks, void* stream);

/*
 * Dequantize `rows` rows produced by dkv_quantize_rows (same layout) into
 * out[r * out_row_stride + i] (i < n) in out_dtype, with the reference's
 * rounding chain: out = to_out(meta(meta(code * scale) + zero)).
 * Replaces reference src/dart/quantization.py:96-109 and the uniform kernels of
 * src/dart/triton_ops.py:32-110.
 */
int dkv_dequantize_rows(const uint8_t* values, const void* scale, const void* zero, int meta_dtype,
                        int64_t rows, int64_t n, int bits, int64_t group, void* out, int out_dtype,
                        int64_t out_row_stride, void* stream);

/*
 * Dequantize mixed keys (layout of dkv_quantize_key_pages, one page of
 * `tokens` tokens) to out[B][H][tokens][D] in out_dtype.
 * Replaces reference src/dart/mixed.py:72-94 and src/dart/triton_ops.py:113-201.
 */
int dkv_dequantize_mixed(const uint8_t* low, const uint8_t* high, const int32_t* idx, const void* scale,
                         const void* zero, int meta_dtype, int64_t B, int64_t H, int64_t D, int64_t tokens,
                         int64_t group, int64_t promoted, void* out, int out_dtype, void* stream);

/*
 * One cache segment (a page, a dense sink piece, the dense pending tail) as
 * the decode kernel sees it.  Field addresses are device addresses; *_bh are
 * strides, in elements of that field, between consecutive (batch, kv-head)
 * blocks.  Inside a block the layouts are those of dkv_quantize_key_pages /
 * dkv_quantize_rows, and a dense block is [tokens][D] with row stride D.
 *   key[0]: dense values | uniform codes | mixed low codes
 *   key[1]: mixed high codes      key[2]: mixed channel indices (int32)
 *   key[3]: scale                 key[4]: zero
 *   value[0]: dense values | codes   value[1]: scale   value[2]: zero
 */
typedef struct dkv_segment {
  int32_t tokens;
  int32_t key_kind;   /* DKV_KEY_*   */
  int32_t value_kind; /* DKV_VALUE_* */
  int32_t key_bits;
  int32_t key_group;
  int32_t promoted;
  int32_t value_bits;
  int32_t value_group;
  uint64_t key[5];
  int64_t key_bh[5];
  uint64_t value[3];
  int64_t value_bh[3];
} dkv_segment;

/*
 * Single-token GQA decode attention over a packed cache: query [B][Hq][D]
 * (element (b,h,d) at query[b*q_sb + h*q_sh + d]) attends to every token of
 * segments[0..n_segments) (device array, in sequence order) and, when
 * tail.tokens > 0, to `tail` (passed by value, last in sequence).  Query head h
 * uses KV head h / (Hq/Hkv).  Logits are (q . k) * scale in fp32 with an online
 * softmax; K and V are dequantized with the reference's rounding chain.
 *
 * Work is split over contiguous segment ranges per (batch, kv head); partial
 * (max, sum, acc[D]) go to `workspace` (dkv_decode_workspace_bytes bytes for
 * n_splits + fast_splits records) and a merge pass writes out[b][h][d]
 * (out_sb, out_sh strides, q dtype) and, if out_f32 != NULL, the fp32 result
 * before the final cast to out_f32[(b*Hq + h)*D + d].
 *
 * Fast page path: when fast_count > 0, descriptor entries
 * [fast_first, fast_first + fast_count) must all be full 128-token pages with
 * head_dim 128, Dart keys with fast_promoted promoted channels (a multiple of
 * 16, at most 64, one key group per page), 2-bit values in groups of
 * fast_value_group channels (a multiple of 16 dividing 128), fp16 metadata and a
 * bf16 or fp16 cache, every field 16-byte aligned, and Hq / Hkv of 1, 2, 4,
 * 8 or 16; the caller guarantees this (except the head ratio, which is checked).
 * Those pages are processed by the MFMA page kernel (16 rows, and uniform runs
 * that it is faster on: the tile kernel)
 * over `fast_splits` splits; the other entries and the tail by the tile or
 * general kernel over `n_splits` splits.
 * With fast_promoted == 0 the run is instead uniform pages: keys quantized
 * with fast_key_bits bits along the tokens (one key group per page), values
 * with fast_value_bits bits along the channels in groups of fast_value_group
 * (2, 4 or 8 bits each), split over half pages (fast_splits at most
 * 2 * fast_count), also with Hq / Hkv of 1, 2, 4 or 8.  For Dart pages
 * fast_key_bits and fast_value_bits are 0 or 2.
 *
 * Dense rest: when rest_dense_tokens > 0 the caller guarantees that every entry
 * outside the fast range and the tail are dense segments in the cache dtype
 * (bf16 or fp16) with 16-byte aligned rows and at most rest_dense_tokens
 * tokens each; then one wave per 32-token chunk handles them (head_dim 128, at
 * most 8 query heads per KV head, 16 beside a Dart run, n_splits = number of those segments *
 * ceil(rest_dense_tokens / 32)).
 *
 * Checked guarantees: when segments_host is not NULL it holds the same
 * n_segments descriptors in host memory, and every entry of the fast range and,
 * with rest_dense_tokens > 0, every other entry is checked against the rules
 * above (DKV_ERR_INVALID naming the entry); the tail is always checked.
 * Without a host copy the caller guarantees them, and a non-page segment the
 * dense kernel cannot read makes the result NaN instead of wrong.
 *
 * Query range: the page kernels compute with fp16 operands; each split scales
 * its query heads by a power of two that brings the largest |q| into
 * [2^14, 2^15) and takes the inverse power into the logit scale (exact), so any
 * finite query works, and queries in fp16's normal range give the same bits as
 * without the scaling.
 *
 * Timing: fast_events[0] / [1], when not NULL, are hipEvent_t handles recorded
 * on `stream` right before and right after the page kernel's launch.
 *
 * Replayable launches: when tail_tokens_dev is not NULL, the kernels read the
 * tail's token count from that device int64 when they run, clamped to
 * [0, tail.tokens]; tail.tokens then gives the tail's capacity (and sizes the
 * splits).  A caller that captures these launches in a graph and appends to
 * the tail on the device between replays keeps the count there.
 *
 * Replaces reference src/dart/fused_attention.py:654-771
 * (`fused_dart_attention`, one query token) and, for one query token,
 * src/dart/attention.py:32-87 (`streamed_dart_attention`).
 */
typedef struct dkv_decode_args {
  const void* query;
  int64_t q_dtype, q_sb, q_sh;
  void* out;
  int64_t out_sb, out_sh;
  float* out_f32;
  const dkv_segment* segments;
  int64_t n_segments;
  dkv_segment tail;
  int64_t B, Hq, Hkv, D;
  int64_t cache_dtype, meta_dtype;
  double scale;
  int64_t n_splits;
  void* workspace;
  int64_t workspace_bytes;
  int64_t fast_first, fast_count, fast_promoted, fast_value_group, fast_splits;
  int64_t rest_dense_tokens;
  void* fast_events[2];
  const int64_t* tail_tokens_dev;
  int64_t fast_key_bits, fast_value_bits;
  const dkv_segment* segments_host;
} dkv_decode_args;

/*
 * A cache's contents as dense tensors: every segment dequantized (or copied)
 * to its tokens of keys and values, both [B][H][tokens][D] in `dtype` (the
 * cache's; dense segments hold it).  `chunks` is a device array of n_chunks
 * triples (segment index, first token, output token): tokens [first, min(first
 * + 128, segment tokens)) of that segment go to output tokens [output token,
 * ...); first is a multiple of 128.  The tail (by value, tokens 0: none) goes
 * to output tokens from tail_start.  D up to 16384.
 *
 * Replaces reference src/dart/cache.py:192-204 (`get`), which dequantizes and
 * concatenates segment by segment (src/dart/quantization.py:96-109,
 * src/dart/mixed.py:72-94).
 */
typedef struct dkv_materialize_args {
  const dkv_segment* segments;
  const int32_t* chunks;
  int64_t n_chunks;
  dkv_segment tail;
  int64_t tail_start;
  int64_t B, H, D, tokens;
  int64_t dtype, meta_dtype;
  void* keys;
  void* values;
} dkv_materialize_args;

int dkv_materialize(const dkv_materialize_args* args, void* stream);

/*
 * Decode-step preparation for the Qwen3 adapter, one new token per sequence:
 * qkv[b] holds the projected query heads, key heads and value heads of
 * sequence b (Hq + 2 Hkv rows of D = 128 elements, row stride qkv_sb elements,
 * cache dtype bf16 or fp16).  Query and key heads get RMSNorm (fp32 x *
 * rsqrt(mean(x^2) + eps), rounded, times q_weight / k_weight[D], rounded) and
 * the rotary embedding (x*cos + rotate_half(x)*sin, each product and the sum
 * rounded; cos, sin [D] for this token's position).  Queries go to
 * q_out[B][Hq][D]; keys and values to tail_key / tail_value[B][Hkv][cap][D] at
 * token index *tail_pos (a device int64, read when the kernel runs; positions
 * outside [0, cap) write nothing).  *tail_pos itself is not changed.
 *
 * Replaces, for one query token, the Transformers Qwen3 q_norm / k_norm and
 * apply_rotary_pos_emb calls of reference src/dart/integrations/qwen3.py:48-53
 * and the append of the new key/value in src/dart/integrations/huggingface.py:68.
 */
typedef struct dkv_decode_prep_args {
  const void* qkv;
  int64_t qkv_sb;
  const void* q_weight;
  const void* k_weight;
  double eps;
  const void* cos;
  const void* sin;
  void* q_out;
  void* tail_key;
  void* tail_value;
  const int64_t* tail_pos;
  int64_t B, Hq, Hkv, D, cap, dtype;
} dkv_decode_prep_args;

int dkv_decode_prep(const dkv_decode_prep_args* args, void* stream);

int64_t dkv_decode_workspace_bytes(int64_t B, int64_t Hq, int64_t D, int64_t n_splits);

/*
 * The kernels dkv_decode_attention would run a call on (host only; device
 * pointers, workspace and n_splits need not be set): `run` for the page run,
 * `rest` for the other entries and the tail, and the number of pieces the
 * rest's work comes in (more splits than that leave some empty).
 */
#define DKV_KERNEL_NONE 0
#define DKV_KERNEL_PAGES 1   /* the page kernels */
#define DKV_KERNEL_TILES 2   /* the tile kernel */
#define DKV_KERNEL_DENSE 3   /* the dense chunks */
#define DKV_KERNEL_GENERAL 4 /* the general kernel */
typedef struct dkv_decode_kernels {
  int64_t run, rest, rest_units;
} dkv_decode_kernels;

int dkv_decode_route(const dkv_decode_args* args, dkv_decode_kernels* out);

int dkv_decode_attention(const dkv_decode_args* args, void* stream);

/*
 * dkv_decode_attention without a caller workspace and without any device
 * allocation: the split records go to a static device array of
 * dkv_decode_scratch_bytes() bytes (32 MiB) that the library holds on each
 * GPU it runs on until the process ends.  args->workspace and
 * args->workspace_bytes are ignored; every other argument means what it means
 * for dkv_decode_attention.  A call whose records
 * (dkv_decode_workspace_bytes of its splits) exceed the scratch returns
 * DKV_ERR_INVALID.  Calls that overlap on one GPU (several streams or host
 * threads) share the array and race; callers serialize them.
 *
 * No counterpart in the reference: it is for callers that cannot allocate
 * device memory (code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc).
 */
int dkv_decode_attention_noalloc(const dkv_decode_args* args, void* stream);
int64_t dkv_decode_scratch_bytes(void);

/*
 * Attention over whole prompts: query [.., Hq, D], keys and values [.., Hkv, D]
 * in bf16 or fp16, element (b, t, h, d) at base[b * sb + t * st + h * sh + d].
 * Query head h uses KV head h / (Hq / Hkv); out = softmax(scale q.k) v in fp32
 * statistics and accumulators, out in the same dtype.
 *
 * Without starts: `requests` sequences of q_tokens query and k_tokens key
 * tokens each (a batch).  With q_starts and k_starts (device int32
 * [requests + 1], ascending): packed sequences, request r's query tokens at
 * rows [q_starts[r], q_starts[r + 1]) of q_tokens, its keys likewise; sb is
 * not used.  Starts outside the tensors are clamped to them.  fill: output rows
 * behind q_starts[requests] and before q_starts[0] become 0 (0: they are left as
 * they were).
 *
 * causal: the last query token sees all nk keys, token i of nq the first
 * i + 1 + nk - nq.  A row that sees no key is 0.  scale from 1e-37 to 1e30 (not
 * included).  D a multiple of 8 up to 256;
 * rows 16-byte aligned (out: 8).  Forward only.  workspace (16-byte aligned):
 * dkv_prompt_attention_workspace_bytes of the same arguments (pointers apart
 * from whether there are starts are not looked at), 0 where the keys are not
 * split; its contents need not be kept.
 *
 * No counterpart in the reference, whose prefill runs the model's attention
 * backend (src/dart/integrations/qwen3.py:85-97).
 */
typedef struct dkv_prompt_attention_args {
  const void* query;
  const void* keys;
  const void* values;
  void* out;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh, o_sb, o_st, o_sh;
  const int32_t* q_starts;
  const int32_t* k_starts;
  int64_t requests, Hq, Hkv, D, q_tokens, k_tokens;
  int64_t dtype;
  double scale;
  int64_t causal, fill;
  void* workspace;
  int64_t workspace_bytes;
} dkv_prompt_attention_args;

int64_t dkv_prompt_attention_workspace_bytes(const dkv_prompt_attention_args* args);
int dkv_prompt_attention(const dkv_prompt_attention_args* args, void* stream);

/*
 * A block cache: requests of different lengths whose keys and values lie in
 * blocks of block_size tokens (16, 32, 64, 128 or 256), found through a table
 * (no counterpart in the reference, whose sequences all have one length).
 * Device state, all int32:
 *   table   [requests][max_blocks]: a request's blocks in order, -1 behind them
 *   lengths [requests]: tokens of each request
 *   free    [blocks]: free[0 .. state[0]) is the stack of free blocks
 *   state   [4]: free blocks, status, the ticket of a running call, 0
 *
 * dkv_reserve_blocks gives request r tokens[r] new tokens behind its lengths[r]
 * and the blocks they need, from the top of the stack in the requests' order.
 * slots [total] (int64, 16-byte aligned) becomes block * block_size + offset of
 * every new token, packed in the requests' order, and -1 behind the last; starts
 * [requests + 1] their first places; positions [total] (int32, 16-byte aligned,
 * optional) their places within the requests, -1 where slots are.  Stack entries that are taken become -1.
 * dkv_release_blocks drops the last tokens[r] of each request (all of them when
 * tokens is NULL, or more than it has) and returns the blocks that no token is
 * left in; it undoes a reserve of the same counts exactly (a block that keeps
 * tokens keeps its scale).
 *
 * A call that cannot be met changes nothing but the status, where it sets 1
 * (too few free blocks), 2 (a request needs more than max_blocks), 4 (a
 * negative count) or 8 (more new tokens than total); a reserve's slots are
 * then -1 and its starts 0.  Calls on one state run in order: two streams must
 * not run them at once.  At most 8,190 requests.
 *
 * shares [blocks] (int32, optional): how many requests beside one hold each block
 * (dkv_fork_blocks); 0 for a free one.  With it,
 *   - dkv_reserve_blocks gives a request that gets tokens in a block others hold a
 *     copy of that block, a new one from the stack before the request's other new
 *     blocks; of the writers in one call that are all of a block's holders, the last
 *     keeps it.  copies [requests][3] lists what dkv_copy_blocks has to copy before
 *     the tokens are appended: block, its copy, tokens; (-1, -1, -1) behind the last.
 *     (A block is known by the token behind the request's last: a request whose last
 *     block is full writes to a new one.)
 *   - dkv_release_blocks returns the blocks that no request holds any more, the
 *     lowest number on top of the stack, and leaves a request alone (status 2) whose
 *     length is more than max_blocks blocks hold; workspace:
 *     dkv_share_workspace_bytes.
 */
typedef struct dkv_block_tables_args {
  int32_t* table;
  int32_t* lengths;
  int32_t* free;
  int32_t* state;
  const int32_t* tokens;
  int64_t* slots;
  int32_t* starts;
  int64_t total, requests, max_blocks, blocks, block_size;
  int32_t* shares;
  int32_t* copies;
  const int32_t* sources;
  int32_t* positions;
  void* workspace;
  int64_t workspace_bytes;
} dkv_block_tables_args;

int dkv_reserve_blocks(const dkv_block_tables_args* args, void* stream);
int dkv_release_blocks(const dkv_block_tables_args* args, void* stream);

/*
 * dkv_fork_blocks: request r with sources[r] >= 0 becomes a copy of what request
 * sources[r] was before the call, of its first tokens[r] tokens (tokens NULL, or more
 * than it has: all), all requests at once; -1 leaves it as it is.  Blocks are not
 * copied but held by both (shares, required); what no request holds any more returns to
 * the stack, the lowest number on top.  A request whose source is not one, or whose
 * count is negative, stays as it was (status 16 or 4).  Uses table, lengths, free,
 * state, shares, sources, tokens and workspace.
 *
 * dkv_compact_blocks: the blocks in use move to the lowest numbers, so that the free
 * ones are the highest: with n in use, the used ones from n on go to the free ones below
 * n, both in ascending order.  Tables and shares follow, the stack has the lowest
 * number on top; copies [blocks / 2][3] lists (block, its new number, block_size) for
 * dkv_copy_blocks, (-1, -1, -1) behind the last.  shares may be NULL.  A state whose stack
 * is not one (its count or entries outside the blocks) is left alone (status 1).
 *
 * dkv_share_workspace_bytes: the workspace (16-byte aligned, its contents need not be
 * kept) of a dkv_fork_blocks, a dkv_compact_blocks or a dkv_release_blocks with shares.
 */
int64_t dkv_share_workspace_bytes(const dkv_block_tables_args* args);
int dkv_fork_blocks(const dkv_block_tables_args* args, void* stream);
int dkv_compact_blocks(const dkv_block_tables_args* args, void* stream);

/*
 * The first copies[i][2] tokens of block copies[i][0], and its scales, to block
 * copies[i][1], for each of `count` entries, in each of `layers` layers: key_codes,
 * value_codes [layers][blocks][H][block_size][D] and key_scale, value_scale
 * [layers][blocks][H], each with its stride between layers (elements).  Entries with a
 * number outside the blocks are skipped.  No target may be another entry's source or
 * target.  D a multiple of 16 up to 512.
 */
typedef struct dkv_copy_blocks_args {
  const int32_t* copies;
  int64_t count, layers, blocks, H, block_size, D;
  uint8_t* key_codes;
  uint8_t* value_codes;
  float* key_scale;
  float* value_scale;
  int64_t key_stride, value_stride, key_scale_stride, value_scale_stride;
} dkv_copy_blocks_args;

int dkv_copy_blocks(const dkv_copy_blocks_args* args, void* stream);

/*
 * New keys and values [tokens][H][D] (bf16, fp16 or fp32; element (t, h, d) at
 * base[t * st + h * sh + d], rows 16-byte aligned) into the e4m3 blocks
 * key_codes, value_codes [blocks][H][block_size][D] with one float scale per
 * block and head, key_scale, value_scale [blocks][H], at `slots` as
 * dkv_reserve_blocks gives them (each slot once, a block's slots next to each
 * other and ascending; a slot outside the blocks writes nothing).  The scale is
 * 2^e with the least e in [-120, 121] that brings the largest magnitude of the
 * block's tokens so far to at most 448 (-120 for zeros); codes are value /
 * scale rounded half to even.  A token at offset 0 begins its block anew; when
 * later tokens raise the scale, the codes before them are rounded to it.
 * A NaN or an infinity becomes e4m3's NaN, does not count for the scale, and
 * sets *nonfinite (optional) to 1.  D a multiple of 16 up to 512.
 */
typedef struct dkv_append_blocks_args {
  const void* keys;
  const void* values;
  int64_t dtype, k_st, k_sh, v_st, v_sh;
  const int64_t* slots;
  int64_t tokens, H, D, blocks, block_size;
  uint8_t* key_codes;
  uint8_t* value_codes;
  float* key_scale;
  float* value_scale;
  uint32_t* nonfinite;
} dkv_append_blocks_args;

int dkv_append_blocks(const dkv_append_blocks_args* args, void* stream);

/*
 * Attention of each request's newest tokens over its blocks: query [tokens][Hq][D]
 * (bf16 or fp16), request r's at rows [starts[r], starts[r + 1]) (starts NULL:
 * one token each), the last of them at position lengths[r] - 1, so token i of n
 * sees the first lengths[r] - n + 1 + i keys.  A row that sees no key is 0.
 * fill: rows behind starts[requests] and before starts[0] become 0 (0: they are
 * left as they were).
 * max_tokens: no request has more new tokens (the rows of a request that has
 * more are undefined).  Scales are powers of two, as dkv_append_blocks writes
 * them; others give undefined results.  Bytes of blocks behind a request's
 * length are not used; a table entry outside [0, blocks) makes the rows that see
 * it NaN.  scale from 1e-37 to 1e30 (not included).  D a multiple of 16 up to
 * 256.  workspace (16-byte aligned): dkv_block_attention_workspace_bytes of the
 * same arguments (pointers are not looked at); its contents need not be kept.
 */
typedef struct dkv_block_attention_args {
  const void* query;
  void* out;
  int64_t dtype, q_st, q_sh, o_st, o_sh;
  int64_t tokens;
  const int32_t* starts;
  const int32_t* table;
  const int32_t* lengths;
  int64_t requests, max_blocks, blocks, block_size;
  const uint8_t* key_codes;
  const uint8_t* value_codes;
  const float* key_scale;
  const float* value_scale;
  int64_t Hq, Hkv, D;
  double scale;
  int64_t max_tokens, fill;
  void* workspace;
  int64_t workspace_bytes;
} dkv_block_attention_args;

int64_t dkv_block_attention_workspace_bytes(const dkv_block_attention_args* args);
int dkv_block_attention(const dkv_block_attention_args* args, void* stream);

/*
 * RMS norm of each query and key head and its rotation by the token's position:
 * x r w with r = 1 / sqrt(mean(x^2) + eps) over the head's D channels (a NULL weight:
 * no norm), then of the first 2 * half channels the pairs (i, i + half), or with
 * interleaved (2 i, 2 i + 1), turn: a' = a cos_i - b sin_i, b' = b cos_i + a sin_i.
 * fp32 between the load and one rounding.
 *
 * query, keys and the outputs have bf16, fp16 or fp32 element (b, t, h, d) at
 * base[b * sb + t * st + h * sh + d], rows of D (a multiple of 8 up to 256) and weights
 * [D] 16-byte aligned.  cos, sin: rows of half angles.  positions NULL: token (b, t)'s at
 * b * c_sb + t * c_st; else int32 (wide_positions: int64) [batch * tokens], the rows of a
 * table of table_rows rows; a position behind it makes the turned channels NaN, a negative
 * one is of no token: its rows are 0 and have no part in the gradients.  Rows of
 * cos and sin start at multiples of 16 bytes where half is a multiple of 8 (of two
 * elements where it is even).
 *
 * The backward call takes the gradients of the outputs as q_grad, k_grad, and writes
 * those of the inputs to q_out, k_out, and of the weights to q_weight_grad, k_weight_grad
 * (weight_dtype; NULL: not wanted).  Sums are made in one order, whatever runs beside.
 * Calls of no tokens launch nothing and write nothing, no weights' gradients either.
 * workspace (16-byte aligned): dkv_rotate_heads_backward_workspace_bytes, where a
 * weight's gradient is wanted.
 *
 * Beside dkv_decode_prep, which does this for one layout of one new token of each
 * sequence and rounds after each step as the Transformers modules do (reference
 * src/dart/integrations/qwen3.py:48-53).
 */
typedef struct dkv_rotate_heads_args {
  const void* query;
  const void* keys;
  void* q_out;
  void* k_out;
  const void* q_grad;
  const void* k_grad;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, qo_sb, qo_st, qo_sh, ko_sb, ko_st, ko_sh;
  int64_t qg_sb, qg_st, qg_sh, kg_sb, kg_st, kg_sh;
  const void* q_weight;
  const void* k_weight;
  void* q_weight_grad;
  void* k_weight_grad;
  const void* cos;
  const void* sin;
  const void* positions;
  int64_t c_sb, c_st, table_rows, wide_positions;
  int64_t batch, tokens, Hq, Hkv, D, half, interleaved;
  int64_t dtype, weight_dtype, angle_dtype;
  double eps;
  void* workspace;
  int64_t workspace_bytes;
} dkv_rotate_heads_args;

int dkv_rotate_heads(const dkv_rotate_heads_args* args, void* stream);
int64_t dkv_rotate_heads_backward_workspace_bytes(const dkv_rotate_heads_args* args);
int dkv_rotate_heads_backward(const dkv_rotate_heads_args* args, void* stream);

/*
 * dkv_append_blocks of keys that are normed and turned on their way (rounded to their
 * type, then to codes), and their queries, in one launch: of `rotation` it takes query,
 * q_out and their strides, Hq, weights, angles, positions (required), half (a multiple of
 * 8), eps and interleaved; batch is 1, and tokens, Hkv (args->H), D and dtype are the same
 * in both.  keys and k_out of `rotation` are not used.
 */
int dkv_append_rotated_blocks(const dkv_append_blocks_args* args, const dkv_rotate_heads_args* rotation, void* stream);

/*
 * For each of `rows` rows of `vocab` logits (bf16, fp16 or fp32, `stride` elements
 * apart): logprobs, the log probability of tokens[row] (int32; wide_tokens: int64; 0 for
 * a negative one, NaN for one of vocab or more); entropy, in nats; and with top > 0 (up to
 * 64) the most likely alternatives, top_tokens and top_logprobs [rows][top], in
 * descending order, the lower number first among equals.
 *
 * -inf is a logit of probability 0.  A row of nothing else has log probabilities -inf and
 * entropy 0 (and a gradient of 0).  A NaN or an infinity makes the row's log
 * probabilities and entropy NaN; NaN logits are no alternatives (where too few others are,
 * top_tokens are -1).
 *
 * stats [rows][2] (optional): a reference m and log2 of the sum of e^(x - m) over the
 * row, which the backward call needs.  m depends on how the row is read and is not its
 * maximum; m + ln(2) log2(sum) is the logarithm of the sum of e^x.  workspace (16-byte aligned): dkv_token_logprobs_workspace_bytes.
 *
 * The backward call writes the gradient of the logits to grads.out (rows `stride` apart)
 * from those of logprobs, entropy and top_logprobs (NULL: 0); of args it reads logits,
 * tokens, stats, entropy and top_tokens.  No counterpart in the reference.
 */
typedef struct dkv_token_logprobs_args {
  const void* logits;
  const void* tokens;
  float* logprobs;
  float* entropy;
  float* stats;
  float* top_logprobs;
  int64_t* top_tokens;
  int64_t stride, rows, vocab, top, dtype, wide_tokens;
  void* workspace;
  int64_t workspace_bytes;
} dkv_token_logprobs_args;

typedef struct dkv_token_logprobs_grads {
  const float* logprobs;
  const float* entropy;
  const float* top_logprobs;
  void* out;
  int64_t stride;
} dkv_token_logprobs_grads;

int64_t dkv_token_logprobs_workspace_bytes(const dkv_token_logprobs_args* args);
int dkv_token_logprobs(const dkv_token_logprobs_args* args, void* stream);
int dkv_token_logprobs_backward(const dkv_token_logprobs_args* args, const dkv_token_logprobs_grads* grads,
                                void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DARTKV_H */
