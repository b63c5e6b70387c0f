/* tq4_kv8.h -- C ABI of the 8-bit paged KV cache: the page plan of a serving
 * step, the cache writer and the attention over it.
 *
 * The third cache format beside the 4-bit ones of tq4.h and tq4_kv4fp8.h, for
 * models that 4 bits cost too much: no rotation, one byte an element, one
 * scale for each page and head. No reference counterpart.
 *
 * CACHE (d = head_size, H = num_kv_heads, S = block_size, P = num_blocks):
 *   key    byte ((page*H + head)*S + token)*d + channel                token-major
 *   value  byte ((page*H + head)*S)*d + (token/16)*16*d + channel*16 + token%16
 *                                          strips of 16 tokens, channel-major
 *   scale  float (plane*P + page)*H + head           plane 0 key, 1 value
 *   code   TQ4_KV8_FP8: OCP FP8 e4m3 (largest 448); TQ4_KV8_INT8: signed,
 *          two's complement (largest 127); stored value = code * scale.
 * Scales are positive finite floats; the writer makes powers of two from 2^-100
 * on, up to 2^120 (FP8) and 2^122 (INT8), which hold the largest BF16 value. The
 * attention reads a scale outside [2^-100, 2^122] as the nearer end.
 *
 * Supported shapes: head_size in {64, 128, 256}; block_size a multiple of 16,
 * at most 1024; GQA group num_heads / num_kv_heads in [1, 16]. Caches, activations and
 * outputs are 16-byte aligned, token strides (elements) multiples of 8
 * (TQ4_ERR_ALIGNMENT).
 *
 * STATUS: 0 or a negative TQ4_ERR_* code (tq4.h); nothing is launched when an
 * argument is refused. Nothing is allocated, synchronised or thrown.
 */
#ifndef TQ4_KV8_H
#define TQ4_KV8_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TQ4_KV8_FP8 0  /* code types */
#define TQ4_KV8_INT8 1

/* ----------------------------------------------------------------------
 * The page plan of a step: block tables, slot map and positions of
 * num_requests requests from their lengths, on the device.
 *
 * Per request b, c = context_lens[b] (held in [0, max_blocks_per_seq * S]) and
 * n = query_lens[b] new tokens (negative: 0). cu_seqlens[b] = n_0 + .. +
 * n_(b-1) (num_requests + 1 entries, saturating at 2^31 - 1): the tokens of b
 * are rows [cu_seqlens[b], cu_seqlens[b+1]) of the step's activations.
 * The pool's free pages are a ring: free_pages[num_blocks], free_state = {head,
 * count}; free page k is free_pages[(head + k) % num_blocks].
 *   1. A request with release[b] != 0 (release may be NULL: none) gives its
 *      ceil(c/S) pages back, in request order, to the ring's end, and its
 *      context becomes empty. Pages given back serve the next call on; a page
 *      that would not fit into the ring (more pages than the pool has) is
 *      dropped. All ceil(c/S) entries have to name pages, as the ring's free
 *      entries have to: one that names none is counted and handed on like a
 *      page, and the rows that a later request is granted in it have slot -1. A
 *      caller that takes pages out of a request's table gives the others back
 *      itself, or shortens the context to those in front, before it releases it.
 *   2. In request order, b needs w = ceil((c + n)/S) - ceil(c/S) pages. It is
 *      granted when its context fits the table and its rows fit max_tokens,
 *      and w is 0 or the pages needed up to and with it, by requests that fit,
 *      are free. Pages leave the ring's head in request order into
 *      block_tables[b].
 *   3. granted[b] = n or 0; new_context_lens[b] = c + n or c; slot_mapping of a
 *      granted token = page * S + offset and positions (may be NULL) its place
 *      in its sequence; every other row up to max_tokens has slot -1 and
 *      position 0, as has a token whose block-table entry names no page.
 *      new_free_state = {head, count} after the call.
 * new_context_lens may be context_lens and new_free_state free_state; no other
 * two buffers may overlap. Table entries that are not opened stay as they are.
 * num_blocks * block_size <= 2^31 and num_requests * max_blocks_per_seq < 2^31
 * (TQ4_ERR_RANGE).
 * slot_mapping may be NULL when max_tokens is 0.
 * workspace: tq4_paged_plan_workspace_bytes(num_requests) bytes, 16-byte
 * aligned, any contents; calls that overlap in time need their own. */
size_t tq4_paged_plan_workspace_bytes(uint32_t num_requests);

int tq4_paged_plan(void* stream, const int32_t* context_lens, const int32_t* query_lens,
                   const int32_t* release, int32_t* block_tables, int32_t* free_pages,
                   const int32_t* free_state, int32_t* slot_mapping, int32_t* positions,
                   int32_t* cu_seqlens, int32_t* granted, int32_t* new_context_lens,
                   int32_t* new_free_state, void* workspace, size_t workspace_bytes,
                   uint32_t num_requests, uint32_t max_blocks_per_seq, uint32_t block_size,
                   uint32_t num_blocks, uint32_t max_tokens);

/* ----------------------------------------------------------------------
 * The writer: num_tokens rows of keys and values (element_type 0 FP16, 1 BF16;
 * [num_kv_heads][d] contiguous, rows key_stride / value_stride elements apart)
 * into the cache at slot_mapping[t] = page * S + offset. A negative slot or one
 * past the pool writes nothing.
 * Per (page, head, plane) that the call writes:
 *   need  = the least 2^e >= 2^-100 with amax <= C * 2^e, amax the largest
 *           finite |x| of the rows that it writes there, C = 448 or 127;
 *   old   = the page's scale; 0 when the call writes the page's offset 0 (it
 *           opens the page: what the page held is given up) or when the scale
 *           is no positive finite number;
 *   scale = max(old, need). Where it grew in a page that was not opened, the
 *           codes that the page holds become RN(code * (old / scale));
 *   code  = RN(x * (1 / scale)), to nearest even, saturated; +inf and NaN give
 *           the largest code, -inf the smallest.
 * The rows of one page stand together: consecutive rows t, in any order of
 * offsets; of two rows for one slot the later one is written, the other counts
 * for nothing. Rows of one page in
 * two places of a call leave that page's codes and scale undefined (no other
 * page's). num_kv_heads <= 8192, num_tokens * num_kv_heads <= 2^26
 * (TQ4_ERR_RANGE). */
int tq4_kv8_reshape_and_cache(void* stream, int element_type, int code_type, const void* key,
                              const void* value, void* key_cache, void* value_cache,
                              float* scale_cache, const int32_t* slot_mapping,
                              uint64_t key_stride, uint64_t value_stride, uint32_t num_tokens,
                              uint32_t num_kv_heads, uint32_t head_size, uint32_t block_size,
                              uint32_t num_blocks);

/* ----------------------------------------------------------------------
 * Attention over the cache: out = softmax(scale * q . k) v per row, q
 * [rows][num_heads][d] (element_type; rows q_stride elements apart), out the
 * same shape, contiguous; q head j reads kv head j / (num_heads /
 * num_kv_heads). block_tables [num_seqs][max_blocks_per_seq]; context_lens
 * [num_seqs] (held in [0, max_blocks_per_seq * S]). A token whose table entry
 * names no page, past its context, or behind what a causal row sees contributes
 * nothing, whatever its bytes are (a NaN code of another writer's among them); a
 * row that sees no token is 0.
 *
 * The decode: one row a sequence (row b = sequence b).
 * num_splits, at most TQ4_KV8_MAX_SPLITS: the parts that each sequence's tokens
 * are cut into, joined by a second kernel. A row's bits then depend on its own
 * sequence and num_splits alone. 0 = auto, from the shapes: parts, or (long
 * tables of many sequences) the batch's tokens in equal shares, whose cuts, and
 * so the last bits of a row, move with the other sequences' lengths. A call's
 * results are the same every time. workspace: tq4_kv8_decode_workspace_bytes
 * bytes (0: none needed) for the same num_splits, 16-byte aligned, any contents;
 * calls that overlap in time need their own (TQ4_ERR_WORKSPACE).
 * num_seqs * splits < 2^24; rows * num_heads < 2^24, or 2^22 where the join has
 * many records a row (more than 32 splits, or few sequences in shares);
 * max_blocks_per_seq * block_size < 2^31; in shares num_seqs * num_kv_heads *
 * (tokens of a table, in 64s) <= 0xff000000 (TQ4_ERR_RANGE). */
#define TQ4_KV8_MAX_SPLITS 256u
size_t tq4_kv8_decode_workspace_bytes(uint32_t num_seqs, uint32_t num_heads,
                                      uint32_t num_kv_heads, uint32_t head_size,
                                      uint32_t block_size, uint32_t max_blocks_per_seq,
                                      uint32_t num_splits);

int tq4_kv8_paged_decode(void* stream, int element_type, int code_type, const void* q,
                         const void* key_cache, const void* value_cache,
                         const float* scale_cache, const int32_t* block_tables,
                         const int32_t* context_lens, void* workspace, size_t workspace_bytes,
                         void* out, uint64_t q_stride, uint32_t num_seqs, uint32_t num_heads,
                         uint32_t num_kv_heads, uint32_t head_size, uint32_t block_size,
                         uint32_t num_blocks, uint32_t max_blocks_per_seq, uint32_t num_splits,
                         float scale);

/* Several rows a sequence (prompt chunks, drafted tokens, cross attention):
 * sequence b has rows [cu_seqlens[b], cu_seqlens[b+1]) of num_rows, at most
 * max_query_len of them. causal: row i of n sees the tokens up to
 * context_len - n + i, its own the last (the chunk's keys and values are in the
 * cache already); otherwise every token of the context. Rows outside the
 * sequences' ranges, past num_rows or past max_query_len are left as they are.
 * workspace: tq4_kv8_prefill_workspace_bytes, as above. */
size_t tq4_kv8_prefill_workspace_bytes(uint32_t num_rows, uint32_t num_seqs, uint32_t num_heads,
                                       uint32_t num_kv_heads, uint32_t head_size,
                                       uint32_t block_size, uint32_t max_blocks_per_seq,
                                       uint32_t max_query_len);

int tq4_kv8_paged_prefill(void* stream, int element_type, int code_type, const void* q,
                          const void* key_cache, const void* value_cache,
                          const float* scale_cache, const int32_t* block_tables,
                          const int32_t* context_lens, const int32_t* cu_seqlens,
                          void* workspace, size_t workspace_bytes, void* out, uint64_t q_stride,
                          uint32_t num_rows, uint32_t num_seqs, uint32_t num_heads,
                          uint32_t num_kv_heads, uint32_t head_size, uint32_t block_size,
                          uint32_t num_blocks, uint32_t max_blocks_per_seq,
                          uint32_t max_query_len, int causal, float scale);

#ifdef __cplusplus
}
#endif
#endif
