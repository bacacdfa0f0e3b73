/* C ABI of the MI355X (gfx950) static INT8 KV-cache kernels.
 *
 * Every entry point takes plain device pointers, element strides (int64) and a hipStream_t passed
 * as void*. Nothing here allocates device memory or synchronises the host: each call validates its
 * arguments, enqueues its kernels on `stream` and returns 0, or returns a nonzero KVQ_ERR_* code
 * without launching anything; kvq_last_error() then describes the failure (thread-local string).
 *
 * Layout conventions (all strides in elements of the pointed-to type):
 *   key/value      bf16  [T, H, D]       strides (st, sh, 1)
 *   k/v cache      int8  [nb, bs, H, D]  strides (sb, sn, sh, 1) -- vLLM's interleaved
 *                                         [nb, H, bs, 2D] view or separate caches alike
 *   q / out        bf16  [T, Hq, D]      strides (st, sh, 1)
 *   slot_mapping   int64 [n], -1 = padding (skipped)
 *   cu_seqlens_q   int32 [B + 1], seq_lens int32 [B], block_table int32 [B, W] (row stride)
 *   k/v scales     fp32  [Hkv, D] (per channel) or [Hkv, 1] (per head), contiguous; k_mu fp32 [Hkv, D]
 * head_dim D is 64 or 128; block_size a power of two >= 16. Base pointers of bf16 / int8 rows must be
 * 16-byte aligned and their row strides multiples of 16 bytes (vLLM's views satisfy this).
 * Page ids read from a block table outside [0, num_blocks) are replaced by page 0 inside the kernels,
 * so a malformed table yields garbage rows rather than a memory fault (the reference leaves this
 * undefined; its KVQ_DEBUG host check, mirrored in kvq/cuda_kernels.py, reports such tables).
 */
#ifndef KVQ_INT8_H
#define KVQ_INT8_H

#include <stdint.h>

/* The version of these entry points' signatures (kvq_abi_version): changes with any of them. */
#define KVQ_ABI_VERSION 16

#ifdef __cplusplus
extern "C" {
#endif

enum {
  KVQ_OK = 0,
  KVQ_ERR_ARG = 1,     /* shape / layout / value rejected before launch */
  KVQ_ERR_LAUNCH = 2,  /* the HIP runtime reported an error for the launch */
};

/* Fused quantize + reshape_and_cache.
 * Replaces the pybind op quant_cache (reference kvq/cuda/int8_kv.cu:554-575, kernel :55-84), bound
 * as kvq/cuda_kernels.py:42-44 quant_reshape_and_cache.
 *   kc[slot / bs, slot % bs, h, d] = sat127(rint(fl((f32(key[t,h,d]) - k_mu[h,d]) / k_scale)))
 *   vc[...]                        = sat127(rint(fl(f32(value[t,h,d]) / v_scale)))
 * for t < n_tokens whose slot is in [0, num_blocks * block_size); other slots are skipped.
 * k_scale_cols / v_scale_cols: D (per channel) or 1 (per head). head_dim 64 or 128; rows, strides
 * and the per-channel tables / k_mu 16-byte aligned. Any head count when num_heads * head_dim is a
 * multiple of 512 and the key / value extents and a cache row's head span are below 2 GiB (the
 * wavefront-per-token kernel); otherwise num_heads * head_dim <= 2048. Stream-ordered, allocates
 * nothing. */
int kvq_quant_cache(const void* key, int64_t key_st, int64_t key_sh, const void* value, int64_t val_st,
                    int64_t val_sh, int8_t* k_cache, int64_t kc_sb, int64_t kc_sn, int64_t kc_sh, int8_t* v_cache,
                    int64_t vc_sb, int64_t vc_sn, int64_t vc_sh, const int64_t* slot_mapping, int64_t n_tokens,
                    int64_t num_heads, int64_t head_dim, int64_t num_blocks, int64_t block_size,
                    const float* k_scale, int64_t k_scale_cols, const float* v_scale, int64_t v_scale_cols,
                    const float* k_mu, void* stream);

/* Standalone q quantization (k scale folded in).
 * Replaces the pybind op quant_q (reference kvq/cuda/int8_kv.cu:577-598, kernel :89-111), bound as
 * kvq/cuda_kernels.py:47-48. x = f32(q[t,h,:]) * k_scale[h / G, :] when k_scale_cols == D (a per-head
 * K scale is not folded); one scale s = max(amax_group / 127, 1e-8) per `group` channels (128 or 32,
 * D = 128); q_i8 = sat127(rint(fl(x / s))). Outputs: q_i8 contiguous [T, Hq, 128], q_scale contiguous
 * [T, Hq, 128 / group]. */
int kvq_quant_q(const void* q, int64_t q_st, int64_t q_sh, int64_t num_tokens, int64_t num_q_heads,
                int64_t head_dim, const float* k_scale, int64_t num_kv_heads, int64_t k_scale_cols,
                int64_t group, int8_t* q_i8, float* q_scale, void* stream);

/* INT8 paged attention for requests with 1 <= q_len <= qmax (decode, spec-decode verification),
 * implementation B of the reference (kvq/int8_ref.py:108-143 with p_tile = 32).
 * Replaces the pybind op int8_decode_attention (reference kvq/cuda/int8_kv.cu:600-648, kernels
 * :168-463 and :472-503), bound as kvq/cuda_kernels.py:51-58 decode_attention.
 * Requests with q_len == 0 or q_len > qmax are skipped (their out rows untouched).
 * Work is split stream-K: the batch is one line of units -- request by request, kv head by kv head,
 * group of up to four 16-row tiles of (token, q head) rows, then 32-key tile -- and each of about
 * target_waves / w workgroups of w <= 4 wavefronts (target_waves 0 = as many wavefronts as the chosen
 * kernel keeps resident on the device) takes an equal contiguous range of it; the wavefronts of a workgroup split a range by row
 * tile and, for short queries, by interleaved key tiles merged in LDS. A (request, kv head, row
 * group) that one workgroup covers whole writes out directly; one that is cut writes fp32 pieces to
 * segm_out [T, Hq, S, D] and segm_max / segm_sum [T, Hq, S] (element (t, h, s) at
 * t * seg_st + h * seg_sh + s, segm_out at that index * D + d), which a second kernel merges.
 * num_splits (<= 64) is S, the most pieces the buffers hold: no segment is cut into more.
 * num_splits == 1 (the reference's single pass without split buffers, int8_kv.cu:612-613): nothing
 * is cut and segm_* may be NULL -- each (request, kv head, row group) runs whole in the workgroup
 * whose range it starts in, its keys split over the workgroup's wavefronts and merged in LDS; one
 * kernel, no second launch. The split buffers are scratch of the call: their contents are internal
 * (segm_sum carries the piece count in its sign), as the reference's. */
int kvq_int8_decode_attention(const void* q, int64_t q_st, int64_t q_sh, const int8_t* k_cache, int64_t k_sb,
                              int64_t k_sn, int64_t k_sh, const int8_t* v_cache, int64_t v_sb, int64_t v_sn,
                              int64_t v_sh, int64_t num_blocks, int64_t block_size, int64_t num_kv_heads,
                              int64_t head_dim, void* out,
                              int64_t o_st, int64_t o_sh, const int32_t* cu_seqlens_q, const int32_t* seq_lens,
                              const int32_t* block_table, int64_t bt_stride, int64_t num_seqs, int64_t num_q_heads,
                              const float* k_scale, int64_t k_scale_cols, const float* v_scale,
                              int64_t v_scale_cols, double softmax_scale, float* segm_out, float* segm_max,
                              float* segm_sum, int64_t seg_st, int64_t seg_sh, int64_t num_splits,
                              int64_t target_waves, int64_t max_query_len, int64_t qmax, void* stream);

/* kvq_int8_decode_attention with two additions to the reference's operator, bound by
 * kvq/cuda_kernels.py decode_attention / paged_attention (q_group=, and split buffers of fewer rows):
 *  - q_group: head_dim is kvq_int8_decode_attention's one q scale per (token, q head); 32 quantizes q
 *    with one scale per 32 channels and sums the groups' scaled integer dots in fp32 -- the reference's
 *    numerics configurations B_channel_qgroup32 / B_channel_smooth_qgroup32 (q_gran "group32",
 *    kvq/int8_ref.py:120-129), which its CUDA kernel does not implement (kvq/vllm_int8/backend.py:125-128
 *    rejects them).
 *  - segm_rows: the split buffers' token rows. The reference indexes them by token and so needs a row
 *    for every token of q (int8_kv.cu:612-620); here a request whose tokens do not all lie in
 *    [0, segm_rows) is never cut (it runs whole, written directly), so a caller may pass buffers sized
 *    for its short requests only -- e.g. for a batch that puts them first -- and still have the longest
 *    of those cut across workgroups. segm_rows >= T is kvq_int8_decode_attention.
 * Other arguments and results as kvq_int8_decode_attention. */
int kvq_int8_decode_attention_ex(const void* q, int64_t q_st, int64_t q_sh, const int8_t* k_cache, int64_t k_sb,
                                 int64_t k_sn, int64_t k_sh, const int8_t* v_cache, int64_t v_sb, int64_t v_sn,
                                 int64_t v_sh, int64_t num_blocks, int64_t block_size, int64_t num_kv_heads,
                                 int64_t head_dim, void* out, int64_t o_st, int64_t o_sh, const int32_t* cu_seqlens_q,
                                 const int32_t* seq_lens, const int32_t* block_table, int64_t bt_stride,
                                 int64_t num_seqs, int64_t num_q_heads, const float* k_scale, int64_t k_scale_cols,
                                 const float* v_scale, int64_t v_scale_cols, double softmax_scale, float* segm_out,
                                 float* segm_max, float* segm_sum, int64_t seg_st, int64_t seg_sh, int64_t num_splits,
                                 int64_t segm_rows, int64_t target_waves, int64_t max_query_len, int64_t qmax,
                                 int64_t q_group, void* stream);

/* kvq_int8_decode_attention without split buffers from the caller and without any allocation: no
 * counterpart in the reference. For callers that cannot allocate device memory around the call (code
 * under HIP graph capture, tight serving loops, harnesses that forbid hipMalloc). Same arguments and
 * results as kvq_int8_decode_attention with num_splits pieces, except that the split partials live in
 * a device array of the library (kvq_noalloc_scratch_bytes() bytes, 64 MiB, per GPU, held until the
 * process ends) instead of segm_out / segm_max / segm_sum; num_tokens (rows of q / out) sizes them.
 * Rejected (KVQ_ERR_ARG) when num_tokens * num_q_heads * num_splits * (head_dim + 2) * 4 bytes exceed
 * that array; num_splits == 1 uses none of it. Calls on one GPU share the array: calls that overlap
 * on one GPU (concurrent streams or threads) race and must be serialised by the caller. */
int kvq_int8_decode_attention_noalloc(const void* q, int64_t q_st, int64_t q_sh, int64_t num_tokens,
                                      const int8_t* k_cache, int64_t k_sb, int64_t k_sn, int64_t k_sh,
                                      const int8_t* v_cache, int64_t v_sb, int64_t v_sn, int64_t v_sh,
                                      int64_t num_blocks, int64_t block_size, int64_t num_kv_heads, int64_t head_dim,
                                      void* out, int64_t o_st, int64_t o_sh, const int32_t* cu_seqlens_q,
                                      const int32_t* seq_lens, const int32_t* block_table, int64_t bt_stride,
                                      int64_t num_seqs, int64_t num_q_heads, const float* k_scale,
                                      int64_t k_scale_cols, const float* v_scale, int64_t v_scale_cols,
                                      double softmax_scale, int64_t num_splits, int64_t target_waves,
                                      int64_t max_query_len, int64_t qmax, void* stream);

/* Size in bytes of the device array kvq_int8_decode_attention_noalloc keeps its split partials in. */
int kvq_noalloc_scratch_bytes(void);

/* Dequantize pages of the INT8 cache into a contiguous bf16 cache [P, bs, H, D] (long-query path).
 * Replaces the pybind op dequant_pages (reference kvq/cuda/int8_kv.cu:650-672, kernel :505-542),
 * called from kvq/cuda_kernels.py:120-122. Output page p is page src_j[p] of request src_req[p]:
 * physical page block_table[src_req[p] * bt_stride + src_j[p]]. ko = bf16_rne(f32(k_i8) * k_scale)
 * (K keeps k - mu), vo likewise. */
int kvq_dequant_pages(const int8_t* k_cache, int64_t k_sb, int64_t k_sn, int64_t k_sh, const int8_t* v_cache,
                      int64_t v_sb, int64_t v_sn, int64_t v_sh, int64_t num_blocks, int64_t block_size, int64_t num_heads,
                      int64_t head_dim, void* k_out, void* v_out, const int32_t* block_table, int64_t bt_stride,
                      const int32_t* src_req, const int32_t* src_j, int64_t num_pages, const float* k_scale,
                      int64_t k_scale_cols, const float* v_scale, int64_t v_scale_cols, void* stream);

/* bf16 paged prefill attention over the temporary cache that kvq_dequant_pages fills: the consumer
 * the reference delegates to vLLM's FlashAttention (kvq/cuda_kernels.py:128-130,
 * flash_attn_varlen_func(q, kt, vt, out, cu_seqlens_q, seqused_k, ..., causal=True,
 * block_table=plan.block_table)); no pybind counterpart. For the rows listed by the work list
 * (tile_req[i], tile_row[i]): rows_per_tile (= kvq_prefill_rows_per_tile()) rows (token, q head) =
 * (r / G, r % G) of request tile_req[i] from row tile_row[i] on, every kv head;
 * o = softmax(q k^T * softmax_scale) v over keys
 * j <= seq_lens[req] - q_len + t (bottom-right causal), fp32 softmax and accumulation, P rounded to
 * bf16 for the PV product. Caches: bf16 [num_blocks, block_size, H, D] views, element strides; key j
 * of request r is slot j % block_size of page block_table[r * bt_stride + j / block_size].
 * Rows not in the work list are not written. */
int kvq_paged_prefill_attention(const void* q, int64_t q_st, int64_t q_sh, const void* k_cache, int64_t k_sb,
                                int64_t k_sn, int64_t k_sh, const void* v_cache, int64_t v_sb, int64_t v_sn,
                                int64_t v_sh, int64_t num_blocks, int64_t block_size, int64_t num_kv_heads,
                                int64_t head_dim, void* out, int64_t o_st, int64_t o_sh,
                                const int32_t* cu_seqlens_q, const int32_t* seq_lens, const int32_t* block_table,
                                int64_t bt_stride, int64_t num_q_heads, const int32_t* tile_req,
                                const int32_t* tile_row, int64_t num_tiles, int64_t rows_per_tile,
                                double softmax_scale, void* stream);

/* The same attention read straight from the INT8 pages, in place of kvq_dequant_pages followed by
 * kvq_paged_prefill_attention -- no temporary bf16 cache. No counterpart in the reference, which always
 * dequantizes first (kvq/cuda_kernels.py:106-131). Caches: int8 [num_blocks, block_size, H, D] views
 * with byte strides (multiples of 16) and block_table the requests' own pages, as
 * kvq_int8_decode_attention takes them; k_scale / v_scale as kvq_dequant_pages takes them
 * (k_scale_cols 1 or head_dim). Work list and rows as kvq_paged_prefill_attention. fold_scales 0: K and
 * V converted as kvq_dequant_pages converts them, output bit-identical to that pair's; 1: the codes
 * converted exactly, k_scale folded into q (bf16(q x k_scale)) and v_scale applied to the fp32 output
 * (faster; not bit-identical). */
int kvq_int8_prefill_attention(const void* q, int64_t q_st, int64_t q_sh, const int8_t* k_cache, int64_t k_sb,
                               int64_t k_sn, int64_t k_sh, const int8_t* v_cache, int64_t v_sb, int64_t v_sn,
                               int64_t v_sh, int64_t num_blocks, int64_t block_size, int64_t num_kv_heads,
                               int64_t head_dim, void* out, int64_t o_st, int64_t o_sh,
                               const int32_t* cu_seqlens_q, const int32_t* seq_lens, const int32_t* block_table,
                               int64_t bt_stride, int64_t num_q_heads, const int32_t* tile_req,
                               const int32_t* tile_row, int64_t num_tiles, int64_t rows_per_tile,
                               double softmax_scale, const float* k_scale, int64_t k_scale_cols,
                               const float* v_scale, int64_t v_scale_cols, int64_t fold_scales, void* stream);

/* kvq_paged_prefill_attention / kvq_int8_prefill_attention with a split work list: several entries may share a
 * request and first row, each reading one piece of the rows' key tiles (32 keys), so that few rows over many
 * keys fill the chip. No counterpart in the reference. Entry i is piece (tile_piece[i] & 0xffff) of
 * (tile_piece[i] >> 16) equal shares (1 .. kvq_prefill_max_parts()) of the tiles the lengths on the device give;
 * an entry that is its rows' only piece writes out and ignores tile_slot. The others leave fp32 partials in slot
 * tile_slot[i] of part_out [slots, Hkv, rows_per_tile, D] and part_ml [slots, Hkv, rows_per_tile, 2], and a second
 * kernel merges them: merge [num_merge, 4] int32 lists (request, first row, slot of piece 0, pieces), pieces in
 * consecutive slots; every cut (request, first row) once. merge and both buffers 16-byte aligned; the buffers are
 * scratch of the call. tile_piece NULL: the calls above. */
int kvq_paged_prefill_attention_ex(const void* q, int64_t q_st, int64_t q_sh, const void* k_cache, int64_t k_sb,
                                   int64_t k_sn, int64_t k_sh, const void* v_cache, int64_t v_sb, int64_t v_sn,
                                   int64_t v_sh, int64_t num_blocks, int64_t block_size, int64_t num_kv_heads,
                                   int64_t head_dim, void* out, int64_t o_st, int64_t o_sh,
                                   const int32_t* cu_seqlens_q, const int32_t* seq_lens, const int32_t* block_table,
                                   int64_t bt_stride, int64_t num_q_heads, const int32_t* tile_req,
                                   const int32_t* tile_row, int64_t num_tiles, int64_t rows_per_tile,
                                   double softmax_scale, const int32_t* tile_piece, const int32_t* tile_slot,
                                   const int32_t* merge, int64_t num_merge, float* part_out, float* part_ml,
                                   void* stream);
int kvq_int8_prefill_attention_ex(const void* q, int64_t q_st, int64_t q_sh, const int8_t* k_cache, int64_t k_sb,
                                  int64_t k_sn, int64_t k_sh, const int8_t* v_cache, int64_t v_sb, int64_t v_sn,
                                  int64_t v_sh, int64_t num_blocks, int64_t block_size, int64_t num_kv_heads,
                                  int64_t head_dim, void* out, int64_t o_st, int64_t o_sh,
                                  const int32_t* cu_seqlens_q, const int32_t* seq_lens, const int32_t* block_table,
                                  int64_t bt_stride, int64_t num_q_heads, const int32_t* tile_req,
                                  const int32_t* tile_row, int64_t num_tiles, int64_t rows_per_tile,
                                  double softmax_scale, const float* k_scale, int64_t k_scale_cols,
                                  const float* v_scale, int64_t v_scale_cols, int64_t fold_scales,
                                  const int32_t* tile_piece, const int32_t* tile_slot, const int32_t* merge,
                                  int64_t num_merge, float* part_out, float* part_ml, void* stream);

/* Most pieces a split work list may cut an entry's keys into. No counterpart in the reference. */
int kvq_prefill_max_parts(void);

/* Rows per work-list entry of kvq_paged_prefill_attention. No counterpart in the reference. */
int kvq_prefill_rows_per_tile(void);

/* Instrumentation, no counterpart in the reference: when set (non-NULL hipEvent_t handles), the next
 * kvq_int8_decode_attention call on this thread records `start` on its stream right before the
 * attention kernel and `stop` right after it (before the split merge), then forgets the pair. Lets a
 * benchmark time the attention kernel alone with events. Returns 0. */
int kvq_set_attention_events(void* start, void* stop);

/* Instrumentation, no counterpart in the reference: reads `bytes` bytes at `data` (16-byte aligned, a
 * multiple of 16) once with `workgroups` workgroups of 256 lanes (each streaming a contiguous share,
 * non-temporal loads) and writes each lane's XOR of the 32-bit words it read to out[workgroups * 256]. Timing it gives the
 * streaming-read rate HBM sustains on the device, the ceiling bench.py reports beside the attention
 * kernel. Stream-ordered, allocates nothing. */
int kvq_stream_read(const void* data, int64_t bytes, uint32_t* out, int64_t workgroups, void* stream);

/* Dense-bf16 MFMA probe, no counterpart in the reference: `workgroups` x 4 wavefronts each run 8
 * independent chains of 16x16x32 bf16 MFMAs for `iters` rounds (a multiple of 4) on operands from `data`
 * (16 KB of bf16, 16-byte aligned), storing one float per thread in `out` (workgroups x 256). FLOP per
 * launch: workgroups x 4 x iters x 8 x 16,384. bench.py times it for the bf16 rate the card sustains
 * under its power limit, the ceiling beside the prefill kernel's. */
int kvq_mfma_probe(const void* data, int64_t iters, float* out, int64_t workgroups, void* stream);

/* Instrumentation, no counterpart in the reference: reads `read_bytes` at `src` and writes `write_bytes`
 * at `dst` once, in order, with `workgroups` workgroups of 256 lanes (each a contiguous share of both,
 * the two streams interleaved in the fixed ratio of their sizes; non-temporal loads and stores; the
 * written values depend on what was read). The sizes are multiples of 16 bytes in the ratio 2 : 1,
 * 1 : 1 or 1 : 2 (KVQ_ERR_ARG otherwise). Timing it at a kernel's byte mix -- 2 : 1 for
 * kvq_quant_cache, 1 : 2 for kvq_dequant_pages -- gives the cost of a plain stream of those bytes on
 * the device: the floor bench.py reports beside those kernels. Stream-ordered, allocates nothing. */
int kvq_stream_rw(const void* src, int64_t read_bytes, void* dst, int64_t write_bytes, int64_t workgroups,
                  void* stream);

/* Instrumentation, no counterpart in the reference: the memory traffic of kvq_quant_cache without its
 * arithmetic. Reads the key and value rows [T, H, D] bf16 (heads contiguous) of the tokens whose slot is
 * in [0, num_blocks * block_size) and writes one byte per element (the bf16's high byte) to both caches'
 * rows (slot / block_size, slot % block_size, head) -- caches of strides c_sb, c_sn, c_sh bytes (the K
 * and V views of one layout share them). Timed beside kvq_quant_cache it gives the floor of a stream of
 * those bytes scattered by slot. Stream-ordered, allocates nothing. */
int kvq_stream_scatter(const void* key, int64_t key_st, int64_t key_sh, const void* value, int64_t val_st,
                       int64_t val_sh, int8_t* k_cache, int8_t* v_cache, int64_t c_sb, int64_t c_sn, int64_t c_sh,
                       const int64_t* slot_mapping, int64_t n_tokens, int64_t num_heads, int64_t head_dim,
                       int64_t num_blocks, int64_t block_size, void* stream);

/* ---- Block-scaled INT8 cache: no calibrated scales, no counterpart in the reference ----
 * A block is `group` consecutive positions of a page (group = 16, 32, 64 or 128, at most block_size; block b of a page
 * is its slots b group .. + group - 1). Each (page, kv head, block) has one fp32 scale for K and one for V: at
 * page * s_sb + head * s_sh + b * s_sg floats of k_scale / v_scale (the same strides for both). A cached value is
 * code * scale. Caches, tables and lengths as above (16-byte aligned rows; head_dim 64 or 128). */

/* Quantize a step's new tokens into their blocks: request r's tokens cu_seqlens_q[r] .. cu_seqlens_q[r + 1] - 1 of key /
 * value are its last positions (up to seq_lens[r] - 1), in pages of its row of block_table. For each block touched and
 * head, over the block's new values x, with s_old the block's scale if it holds earlier positions of the request, else 0:
 *   s = max(s_old, fl(max |x| / 127), 1e-8)   (finite x; an infinite one saturates, a NaN's code is any)
 *   new slots sat127(rint(fl(x / s))), the request's earlier slots of the block rint(fl(code * fl(s_old / s))) if s > s_old
 * Other slots and scales stay as they are. A page id outside [0, num_blocks) and a token at a negative position
 * (seq_lens[r] < its tokens) are skipped, as are tokens from num_tokens on (the rows key / value hold). The pages that
 * a call writes must belong to one request each. Stream-ordered, allocates nothing, bit-reproducible. */
int kvq_quant_block_cache(const void* key, int64_t key_st, int64_t key_sh, const void* value, int64_t val_st,
                          int64_t val_sh, int64_t num_tokens, int8_t* k_cache, int64_t kc_sb, int64_t kc_sn,
                          int64_t kc_sh, int8_t* v_cache, int64_t vc_sb, int64_t vc_sn, int64_t vc_sh,
                          int64_t num_blocks, int64_t block_size, int64_t num_heads, int64_t head_dim, float* k_scale,
                          float* v_scale, int64_t s_sb, int64_t s_sh, int64_t s_sg, int64_t group,
                          const int32_t* cu_seqlens_q, const int32_t* seq_lens, const int32_t* block_table,
                          int64_t bt_stride, int64_t num_seqs, void* stream);

/* Read ranges of keys back: positions starts[r] .. of request r become rows cu_seqlens_k[r] .. cu_seqlens_k[r + 1] - 1
 * of k_out / v_out (bf16 [num_rows, H, D], strides (st, sh, 1)): bf16_rne(code * scale). Rows past cu_seqlens_k's last
 * entry are left as they were, rows from num_rows on are not written, a negative start reads nothing. */
int kvq_read_block_cache(const int8_t* k_cache, int64_t kc_sb, int64_t kc_sn, int64_t kc_sh, const int8_t* v_cache,
                         int64_t vc_sb, int64_t vc_sn, int64_t vc_sh, int64_t num_blocks, int64_t block_size,
                         int64_t num_heads, int64_t head_dim, const float* k_scale, const float* v_scale, int64_t s_sb,
                         int64_t s_sh, int64_t s_sg, int64_t group, const int32_t* starts, const int32_t* cu_seqlens_k,
                         const int32_t* block_table, int64_t bt_stride, int64_t num_seqs, void* k_out, int64_t ko_st,
                         int64_t ko_sh, void* v_out, int64_t vo_st, int64_t vo_sh, int64_t num_rows, void* stream);

/* Attention over a block-scaled cache for requests with 1 <= q_len <= qmax:
 *   o = softmax(q . (k_code * k_scale) * softmax_scale) (v_code * v_scale),  bottom-right causal, bf16 q and out;
 * a row that sees no key is zero, another whose q holds a NaN or an infinity is NaN; softmax_scale from 1e-16 to 1e16. The
 * codes are exact, a V scale counts as at least 2^-70 (the write's least is 1e-8). Rounded: each channel of q to a multiple of
 * its row's largest / 16,256; the weights to 2^-14 of each where at most 16 (token, q head) rows share a kv head, and by
 * attn_rules.h up to 32, else to bf16 (2^-8 of each). Rows, skipped requests, split buffers and the other arguments as
 * kvq_int8_decode_attention_ex (segm_sum's last piece is marked by its sign). */
int kvq_block_decode_attention(const void* q, int64_t q_st, int64_t q_sh, const int8_t* k_cache, int64_t k_sb,
                               int64_t k_sn, int64_t k_sh, const int8_t* v_cache, int64_t v_sb, int64_t v_sn,
                               int64_t v_sh, int64_t num_blocks, int64_t block_size, int64_t num_kv_heads,
                               int64_t head_dim, const float* k_scale, const float* v_scale, int64_t s_sb, int64_t s_sh,
                               int64_t s_sg, int64_t group, void* out, int64_t o_st, int64_t o_sh,
                               const int32_t* cu_seqlens_q, const int32_t* seq_lens, const int32_t* block_table,
                               int64_t bt_stride, int64_t num_seqs, int64_t num_q_heads, double softmax_scale,
                               float* segm_out, float* segm_max, float* segm_sum, int64_t seg_st, int64_t seg_sh,
                               int64_t num_splits, int64_t segm_rows, int64_t target_waves, int64_t max_query_len,
                               int64_t qmax, void* stream);

/* Pages' codes as bf16 (exact) in a contiguous temporary cache [num_pages, bs, H, D], pages as kvq_dequant_pages takes
 * them, and in scales_out [H, num_pages * bs / 16, 4] what the prefill below needs of each 16 slots' scales. */
int kvq_block_codes(const int8_t* k_cache, int64_t k_sb, int64_t k_sn, int64_t k_sh, const int8_t* v_cache, int64_t v_sb,
                    int64_t v_sn, int64_t v_sh, int64_t num_blocks, int64_t block_size, int64_t num_heads, int64_t head_dim,
                    const float* k_scale, const float* v_scale, int64_t s_sb, int64_t s_sh, int64_t s_sg, int64_t group,
                    void* k_out, void* v_out, float* scales_out, const int32_t* block_table, int64_t bt_stride,
                    const int32_t* src_req, const int32_t* src_j, int64_t num_pages, void* stream);

/* The same attention for the rows of a work list, as kvq_int8_prefill_attention_ex takes it (tile_piece NULL: every
 * entry reads all of its rows' keys). k_codes / v_codes / code_scales: the requests' pages as kvq_block_codes leaves them
 * (num_pages of them, codes_table [num_seqs, ..] with row stride ct_stride in place of block_table), read instead of the
 * int8 pages, whose conversion in the kernel costs more where many rows read each key; q is then taken as it is. NULL: the
 * int8 pages. Weights are rounded to bf16 either way. */
int kvq_block_prefill_attention(const void* q, int64_t q_st, int64_t q_sh, const int8_t* k_cache, int64_t k_sb,
                                int64_t k_sn, int64_t k_sh, const int8_t* v_cache, int64_t v_sb, int64_t v_sn,
                                int64_t v_sh, int64_t num_blocks, int64_t block_size, int64_t num_kv_heads,
                                int64_t head_dim, const float* k_scale, const float* v_scale, int64_t s_sb, int64_t s_sh,
                                int64_t s_sg, int64_t group, void* out, int64_t o_st, int64_t o_sh,
                                const int32_t* cu_seqlens_q, const int32_t* seq_lens, const int32_t* block_table,
                                int64_t bt_stride, int64_t num_q_heads, const int32_t* tile_req, const int32_t* tile_row,
                                int64_t num_tiles, int64_t rows_per_tile, double softmax_scale, const int32_t* tile_piece,
                                const int32_t* tile_slot, const int32_t* merge, int64_t num_merge, float* part_out,
                                float* part_ml, const void* k_codes, const void* v_codes, const float* code_scales,
                                int64_t num_pages, const int32_t* codes_table, int64_t ct_stride, void* stream);

/* ---- 4-bit cache, no counterpart in the reference ----
 * A cached value is an e2m1 code (0, 1/2, 1, 3/2, 2, 3, 4, 6 or their negatives) times 2^(byte - 127), one exponent byte for
 * each 32 channels of a row (page, slot, head), K's and V's apart. Caches are bytes [nb, bs, H, D / 2], strides (sb, sn, sh, 1)
 * in bytes, multiples of 16, pages below 4 GiB apart, channel 2 c in the low half of byte c; exponent bytes k_scale / v_scale
 * [nb, H, bs, D / 32], strides (s_sb, s_sh, D / 32, 1), 16-byte aligned as well. Tables and lengths as above; head_dim 64 or
 * 128. An exponent byte that the write does not make (above 252: 255 would be no number) may give any value for its own row and for
 * the query rows that see it, and counts nowhere else. */

/* Quantize rows into slots: for t < num_tokens whose slot is in [0, nb * bs), others are skipped. Of a group's 32 values x, with
 * top = max |x| (finite x):  e = floor(log2 top) - 2, one more where top 2^-e > 7, from -100 to 125; byte e + 127; codes the
 * nearest of x 2^-e, ties to the even code, at most 6 (infinities too); a NaN is 0. A slot occurs once. Bit-reproducible. */
int kvq_quant_fp4_cache(const void* key, int64_t key_st, int64_t key_sh, const void* value, int64_t val_st, int64_t val_sh,
                        uint8_t* k_cache, int64_t kc_sb, int64_t kc_sn, int64_t kc_sh, uint8_t* v_cache, int64_t vc_sb,
                        int64_t vc_sn, int64_t vc_sh, int64_t num_blocks, int64_t block_size, int64_t num_heads,
                        int64_t head_dim, uint8_t* k_scale, uint8_t* v_scale, int64_t s_sb, int64_t s_sh,
                        const int64_t* slot_mapping, int64_t num_tokens, void* stream);

/* Read ranges of keys back as bf16 (exact), with kvq_read_block_cache's ranges and rows. */
int kvq_read_fp4_cache(const uint8_t* k_cache, int64_t kc_sb, int64_t kc_sn, int64_t kc_sh, const uint8_t* v_cache,
                       int64_t vc_sb, int64_t vc_sn, int64_t vc_sh, int64_t num_blocks, int64_t block_size, int64_t num_heads,
                       int64_t head_dim, const uint8_t* k_scale, const uint8_t* v_scale, int64_t s_sb, int64_t s_sh,
                       const int32_t* starts, const int32_t* cu_seqlens_k, const int32_t* block_table, int64_t bt_stride,
                       int64_t num_seqs, void* k_out, int64_t ko_st, int64_t ko_sh, void* v_out, int64_t vo_st, int64_t vo_sh,
                       int64_t num_rows, void* stream);

/* Pages as bf16 (exact) in a contiguous temporary cache [num_pages, bs, H, D], pages as kvq_dequant_pages takes them, and in
 * scales_out [H, num_pages * bs / 16, 4] the table that the prefill below reads beside them. */
int kvq_fp4_pages(const uint8_t* k_cache, int64_t kc_sb, int64_t kc_sn, int64_t kc_sh, const uint8_t* v_cache, int64_t vc_sb,
                  int64_t vc_sn, int64_t vc_sh, int64_t num_blocks, int64_t block_size, int64_t num_heads, int64_t head_dim,
                  const uint8_t* k_scale, const uint8_t* v_scale, int64_t s_sb, int64_t s_sh, void* k_out, void* v_out,
                  float* scales_out, const int32_t* block_table, int64_t bt_stride, const int32_t* src_req,
                  const int32_t* src_j, int64_t num_pages, void* stream);

/* The attention below for the rows of a work list, as kvq_paged_prefill_attention_ex takes it (tile_piece NULL: every entry
 * reads all of its rows' keys), over pages that kvq_fp4_pages left (pages_table [num_seqs, ..], row stride pt_stride), with the
 * same q and weights. */
int kvq_fp4_prefill_attention(const void* q, int64_t q_st, int64_t q_sh, const void* k_pages, const void* v_pages,
                              const float* page_scales, int64_t num_pages, int64_t block_size, int64_t num_kv_heads,
                              int64_t head_dim, void* out, int64_t o_st, int64_t o_sh, const int32_t* cu_seqlens_q,
                              const int32_t* seq_lens, const int32_t* pages_table, int64_t pt_stride, int64_t num_q_heads,
                              const int32_t* tile_req, const int32_t* tile_row, int64_t num_tiles, int64_t rows_per_tile,
                              double softmax_scale, const int32_t* tile_piece, const int32_t* tile_slot, const int32_t* merge,
                              int64_t num_merge, float* part_out, float* part_ml, void* stream);

/* Attention over a 4-bit cache for requests with 1 <= q_len <= qmax: o = softmax(q k^T softmax_scale) v, bottom-right causal,
 * bf16 q and out; a row that sees no key is zero, another whose q holds a NaN or an infinity is NaN. Cached values are exact.
 * Rounded: the weights, to a sum of two bf16 (2^-14 of each). lse (fp32 [T, Hq], row stride lse_st, or NULL): the rows' natural
 * log-sum-exp, -inf where no key is seen. softmax_scale from 1e-16 to 1e16. K's and V's page and slot strides are the same.
 * max_query_len picks the launch: requests with more tokens, up to qmax, are served too. Rows, skipped requests, split buffers
 * and the other arguments as kvq_block_decode_attention. */
int kvq_fp4_decode_attention(const void* q, int64_t q_st, int64_t q_sh, const uint8_t* k_cache, int64_t k_sb, int64_t k_sn,
                             int64_t k_sh, const uint8_t* v_cache, int64_t v_sb, int64_t v_sn, int64_t v_sh,
                             int64_t num_blocks, int64_t block_size, int64_t num_kv_heads, int64_t head_dim,
                             const uint8_t* k_scale, const uint8_t* v_scale, int64_t s_sb, int64_t s_sh, void* out,
                             int64_t o_st, int64_t o_sh, const int32_t* cu_seqlens_q, const int32_t* seq_lens,
                             const int32_t* block_table, int64_t bt_stride, int64_t num_seqs, int64_t num_q_heads,
                             double softmax_scale, float* segm_out, float* segm_max, float* segm_sum, int64_t seg_st,
                             int64_t seg_sh, int64_t num_splits, int64_t segm_rows, float* lse, int64_t lse_st,
                             int64_t target_waves, int64_t max_query_len, int64_t qmax, void* stream);

/* Add the attention weights of a step's rows to running sums: for requests with 1 <= q_len <= qmax and j < w_cols,
 *   weights[r, h, j] += sum over r's tokens and h's q heads that see key j of exp(q . k_j softmax_scale - lse)
 * weights fp32 [B, Hkv, w_cols], strides (w_sr, w_sh, 1); lse as kvq_fp4_decode_attention leaves it, rows whose lse is not
 * finite add nothing. Row r of weights belongs to request r alone, and no two rows overlap. Bit-reproducible. */
int kvq_fp4_key_weights(const void* q, int64_t q_st, int64_t q_sh, const uint8_t* k_cache, int64_t k_sb, int64_t k_sn,
                        int64_t k_sh, int64_t num_blocks, int64_t block_size, int64_t num_kv_heads, int64_t head_dim,
                        const uint8_t* k_scale, int64_t s_sb, int64_t s_sh, const float* lse, int64_t lse_st, float* weights,
                        int64_t w_sr, int64_t w_sh, int64_t w_cols, const int32_t* cu_seqlens_q, const int32_t* seq_lens,
                        const int32_t* block_table, int64_t bt_stride, int64_t num_seqs, int64_t num_q_heads,
                        double softmax_scale, int64_t max_query_len, int64_t qmax, void* stream);

/* Evict: of request r's n = seq_lens[r] keys (at most its bt_cols pages' slots), each kv head keeps m = keep[r] (at most
 * kept_cols, at least 0): the last min(recent, m) and, of those before, the ones of the largest weights (ties to the lowest
 * position, a NaN the largest; 0 from w_cols on). Their rows move to positions 0 .. m - 1 in order, their weights with them;
 * weights[r, h, m .. n - 1] become 0. kept[r, h, i] (int32, strides (kp_sr, kp_sh, 1)): the position that row i held before;
 * new_lens[r] = min(n, m); new_lens may be seq_lens or keep itself (one launch more), and overlaps them in no other way. Where
 * n <= m nothing moves (kept[r, h, i] = i). Entries of kept from new_lens[r] on and cache rows from there on are left as they are.
 * Rows (r, h) of weights do not overlap, nor do kept's. The pages of a call's requests must be theirs alone. Page ids outside
 * [0, nb) read as page 0, and are not written. A table has at most 2^28 slots (bt_cols * block_size). Bit-reproducible. */
int kvq_fp4_evict(uint8_t* k_cache, int64_t k_sb, int64_t k_sn, int64_t k_sh, uint8_t* v_cache, int64_t v_sb, int64_t v_sn,
                  int64_t v_sh, int64_t num_blocks, int64_t block_size, int64_t num_heads, int64_t head_dim, uint8_t* k_scale,
                  uint8_t* v_scale, int64_t s_sb, int64_t s_sh, float* weights, int64_t w_sr, int64_t w_sh, int64_t w_cols,
                  const int32_t* seq_lens, const int32_t* keep, int64_t recent, const int32_t* block_table, int64_t bt_stride,
                  int64_t bt_cols, int64_t num_seqs, int32_t* kept, int64_t kp_sr, int64_t kp_sh, int64_t kept_cols,
                  int32_t* new_lens, void* stream);

/* RMS norm of each head's query and key rows and their rotation by position, for t < num_tokens and positions[t] in
 * [0, num_positions) (other tokens' output rows are left as they are):
 *   y = x / sqrt(mean(x^2) + eps) * weight;   (a, b) -> (a cos - b sin, b cos + a sin)
 * for the pairs of the first rotary_dim channels: (i, i + rotary_dim / 2), or (2 i, 2 i + 1) where interleaved. q / k and their
 * outputs bf16 [T, H, D], strides (st, sh, 1), an output may be its input; positions int32 or int64 (position_bits); table
 * [num_positions, rotary_dim] (row stride t_st) fp32 or bf16: rotary_dim / 2 cosines, then as many sines; weights [D] fp32 or
 * bf16, both NULL: no norm. fp32 throughout, the sum of a row's squares too (values within 2^-60 .. 2^60, smaller ones where eps
 * is not 0), one rounding. rotary_dim a multiple of 16. No counterpart in the reference. */
int kvq_norm_rope(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh, void* q_out,
                  int64_t qo_st, int64_t qo_sh, void* k_out, int64_t ko_st, int64_t ko_sh, int64_t num_tokens,
                  int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, const void* positions, int64_t position_bits,
                  const void* table, int64_t t_st, int64_t num_positions, int64_t rotary_dim, int64_t table_bf16,
                  const void* q_weight, const void* k_weight, int64_t weight_bf16, double eps, int64_t interleaved,
                  void* stream);

/* Text of the last error on this thread ("" if none). */
const char* kvq_last_error(void);

/* ABI version of this library (bumped on any signature change or new entry point). */
int kvq_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* KVQ_INT8_H */
