/*
 * cie_paged_attention.h — C ABI of the MI355X (gfx950) paged-KV GQA attention
 * hot path: KV append, split-KV decode (load + merge) and the varlen mixed
 * (chunked prefill + decode) causal kernel.
 *
 * Conventions shared by every entry point
 * ---------------------------------------
 *  - Every pointer is a device pointer owned by the caller.  Nothing here
 *    allocates, frees or synchronises; kernels are enqueued on `stream`
 *    (a hipStream_t passed as void*; NULL = the null stream), so the calls are
 *    safe under hipGraph stream capture.
 *  - fp16 tensors are IEEE binary16.  Index tensors are int64, the dtype the
 *    reference uses for lens / slot ids / block tables / cu_seqlens.
 *  - KV pool layout is the reference's (n_pages, H_kv, page_size, D) with the
 *    last two dims dense (stride(3) == 1, stride(2) == D); the page and head
 *    strides are passed explicitly (in elements).
 *  - The block table is (n_slots, bt_stride) int64; only the first bt_width
 *    entries of a row are valid logical pages.
 *  - `err` (nullable) is an int32 device word.  Kernels never fault on a bad
 *    index: an out-of-range page id, slot id or length is clamped / skipped and
 *    the matching CIE_ERRBIT_* bit is OR-ed into *err.
 *  - Return value: 0 on success, a negative CIE_E* code for an argument error
 *    detected on the host (nothing is launched), or a positive hipError_t from
 *    the launch.
 */
#ifndef CIE_PAGED_ATTENTION_H
#define CIE_PAGED_ATTENTION_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CIE_OK 0
#define CIE_EINVAL (-1)      /* inconsistent sizes / strides / null pointer      */
#define CIE_EUNSUPPORTED (-2) /* shape outside what the kernels are built for   */
#define CIE_ESCRATCH (-3)     /* problem larger than the static scratch of an
                                 allocation-free entry point                     */

#define CIE_ERRBIT_PAGE 1     /* page id outside [0, n_pages)                    */
#define CIE_ERRBIT_LEN 2      /* length beyond the block-table row capacity      */
#define CIE_ERRBIT_OFFSET 4   /* in-page offset outside [0, page_size)           */
#define CIE_ERRBIT_SPLIT 8    /* a split-arrival counter held a stale value at the
                                 start of the call (see `counters` below)        */
#define CIE_ERRBIT_PLAN 16    /* a planned call whose plan was made for another
                                 batch shape or partials budget (the call wrote
                                 nothing), or a batch with more work items than
                                 its plan holds (cie_mixed_plan)                  */
#define CIE_ERRBIT_FREE 32    /* a free list with too few pages (or too many given
                                 back), or a slot that comes twice in the call    */
#define CIE_ERRBIT_ADAPTER 64 /* adapter id at or past the number of adapters     */

/* Element types of the entry points that take one. */
#define CIE_F16 0
#define CIE_BF16 1
#define CIE_F32 2

/* Version of this ABI (bumped on any signature change). */
int cie_abi_version(void);

/* Human-readable name of a CIE_E* / hipError_t status. */
const char* cie_status_string(int status);

/*
 * Decode KV append: for each sequence b, pos = lens[slot_ids[b]],
 *   k_pool[block_table[slot, pos / page_size], h, pos % page_size, :] = k_new[b, h, :]
 * (same for V).  Bit-exact fp16 copy.
 * Replaces KVStorage.decode_update (kv_cache/storage.py:87-122): the torch
 * gather of lens / block_table plus two index_put_ scatters.
 * k_new / v_new are (B, H_kv, D) views with their own token and head strides
 * (elements); the last dim must be dense.
 */
int cie_kv_append_decode(void* k_pool, void* v_pool,
                         const void* k_new, const void* v_new,
                         int64_t k_tok_stride, int64_t k_head_stride,
                         int64_t v_tok_stride, int64_t v_head_stride,
                         const int64_t* slot_ids, const int64_t* lens,
                         const int64_t* block_table,
                         int64_t B, int64_t H_kv, int64_t page_size, int64_t D,
                         int64_t n_pages, int64_t pool_page_stride,
                         int64_t pool_head_stride, int64_t bt_stride,
                         int64_t bt_width, int64_t n_slots,
                         int32_t* err, void* stream);

/*
 * Token-mode (mixed) KV append: for each packed token t < T,
 *   k_pool[pages[t], h, offsets[t], :] = k_new[t, h, :]   (same for V).
 * Replaces KVStorage.mixed_update (kv_cache/storage.py:62-85).
 */
int cie_kv_append_tokens(void* k_pool, void* v_pool,
                         const void* k_new, const void* v_new,
                         int64_t k_tok_stride, int64_t k_head_stride,
                         int64_t v_tok_stride, int64_t v_head_stride,
                         const int64_t* pages, const int64_t* offsets,
                         int64_t T, int64_t H_kv, int64_t page_size, int64_t D,
                         int64_t n_pages, int64_t pool_page_stride,
                         int64_t pool_head_stride, int32_t* err, void* stream);

/*
 * Split-KV paged GQA decode, one query token per sequence:
 *   o[b, h, :] = softmax(q[b, h, :] . K_b^T * D^-0.5) . V_b
 * over the first lens[b] tokens of slot slot_ids[b]'s pages, kv head h / G.
 * lens[b] == 0 gives o = 0.  One kernel launch: the KV splits, and the
 * log-sum-exp merge done by the last workgroup of each (sequence, kv head).
 * Replaces decode_gqa_attention (attn/core.py:13-66), i.e. the Triton
 * decode_gqa_attention_kernel_load (kernels/decode_attention.py:12-179) and
 * decode_attention_kernel_merge (kernels/decode_attention.py:182-272).
 *   q, o       : (B, H_q, D) dense fp16, 16-byte aligned
 *   lens       : (B,) attended lengths (the reference passes lens[slot] + 1)
 *   n_splits   : KV splits per (sequence, kv head) — the reference's
 *                `num_programs`
 *                (1 <= n_splits <= cie_paged_decode_max_splits())
 *   partials   : cie_paged_decode_partials_bytes(B, H_q, D, n_splits) bytes,
 *                16-byte aligned, any contents: the splits' softmax state
 *   counters   : 2 * B * H_kv int32, 16-byte aligned: one arrival word per
 *                (sequence, kv head), then one stale word per (sequence, kv
 *                head).  They must be zero before the call and every
 *                completed call leaves them zero, so one zeroed buffer serves
 *                any number of stream-ordered calls.  Calls that can overlap
 *                in time must not share counters or partials.  A call that
 *                finds an arrival word outside [0, n_splits) raises
 *                CIE_ERRBIT_SPLIT (its o is then not valid); when every split
 *                of a (sequence, kv head) finds it stale, the call also puts
 *                both words back to zero.  A stale value inside [0, n_splits)
 *                cannot be told apart from live arrivals and may survive the
 *                call, so after CIE_ERRBIT_SPLIT the caller zeroes the
 *                counters before the next call.
 *   partials and counters may be NULL when n_splits == 1.
 */
int64_t cie_paged_decode_partials_bytes(int64_t B, int64_t H_q, int64_t D,
                                        int64_t n_splits);
int cie_paged_decode_max_splits(void);
int cie_paged_decode(void* o, const void* q,
                     const void* k_pool, const void* v_pool,
                     const int64_t* lens, const int64_t* slot_ids,
                     const int64_t* block_table,
                     void* partials, int32_t* counters,
                     int64_t B, int64_t H_q, int64_t H_kv, int64_t D,
                     int64_t page_size, int64_t n_pages,
                     int64_t pool_page_stride, int64_t pool_head_stride,
                     int64_t bt_stride, int64_t bt_width, int64_t n_slots,
                     int64_t n_splits, int32_t* err, void* stream);

/*
 * Decode step with the KV append fused in, one launch: for each sequence b,
 * pos = lens[slot_ids[b]] (the pool's prior length per slot, (n_slots,)),
 * the new K/V rows k_new[b] / v_new[b] are written to
 * (block_table[slot, pos / page_size], pos % page_size) bit-exactly, and o is
 * the decode attention over the pos + 1 tokens that then exist.
 * Equivalent to KVStorage.decode_update (kv_cache/storage.py:87-122) followed
 * by gqa_decode_attention with lens[slot] + 1 (attn/core.py:200-215).
 * partials / counters as for cie_paged_decode.
 */
int cie_paged_decode_append(void* o, const void* q, void* k_pool, void* v_pool,
                            const void* k_new, const void* v_new,
                            int64_t k_tok_stride, int64_t k_head_stride,
                            int64_t v_tok_stride, int64_t v_head_stride,
                            const int64_t* lens, const int64_t* slot_ids,
                            const int64_t* block_table, void* partials,
                            int32_t* counters,
                            int64_t B, int64_t H_q, int64_t H_kv, int64_t D,
                            int64_t page_size, int64_t n_pages,
                            int64_t pool_page_stride, int64_t pool_head_stride,
                            int64_t bt_stride, int64_t bt_width,
                            int64_t n_slots, int64_t n_splits, int32_t* err,
                            void* stream);

/*
 * Planned decode.  The slot ids, lengths and block-table rows a decode step
 * reads are the same for every layer of the step (KVStorage advances the
 * lengths after the last layer), so a step can make a plan once and run each
 * layer's decode from it:
 *   cie_paged_decode_plan       once per step: each sequence's attended
 *                               length (append = 1: lens is (n_slots,) prior
 *                               lengths, attended = lens[slot] + 1, as
 *                               cie_paged_decode_append; append = 0: lens is
 *                               (B,) attended lengths, as cie_paged_decode),
 *                               its splits (balanced by length over the
 *                               n_workgroups of the grid) and each workgroup's
 *                               page ids, into `plan`
 *                               (cie_paged_decode_plan_bytes(n_workgroups)
 *                               bytes, 16-byte aligned, any contents).  Index
 *                               errors are reported here (CIE_ERRBIT_*).
 *   cie_paged_decode_planned,   per layer: the same results as
 *   cie_paged_decode_append_planned,   cie_paged_decode / _append / _qkv_rope
 *   cie_paged_decode_qkv_rope_planned  on the plan's sequences, but the
 *                               launch reads one descriptor and its page ids
 *                               instead of the slot id, then the block table
 *                               and the length: one memory round trip less
 *                               before its first K/V loads.
 * The plan must be made with the same append mode, block table and lengths
 * as the layers' calls, and n_workgroups must be the same for all of them.
 * n_workgroups = cie_paged_decode_plan_workgroups(B, H_kv, n_splits):
 * B * H_kv * n_splits, or with n_splits = 0 the library's default (about
 * one workgroup per CU, two where B * H_kv is more than the CUs, and one per
 * (sequence, kv head) where it is more than twice as many); it must lie
 * in [B * H_kv, B * H_kv * cie_paged_decode_max_splits()] and be a multiple
 * of H_kv.  Equal lengths give every (sequence, kv head) as many splits as
 * fit, n_workgroups / (B * H_kv) rounded down, but none of fewer than 4
 * 16-key tiles (48 or 64 under the default of two workgroups per CU); unequal
 * ones give longer sequences more.  partials:
 * cie_paged_decode_planned_partials_bytes(n_workgroups, H_q, H_kv, D);
 * counters: 2 * B * H_kv words as for cie_paged_decode.  B <= 1024.
 * Replaces decode_gqa_attention (attn/core.py:13-66) and its grid
 * (P, H_kv, B) (attn/core.py:37) for every layer of a decode step.
 */
int64_t cie_paged_decode_plan_workgroups(int64_t B, int64_t H_kv, int64_t n_splits);
int64_t cie_paged_decode_plan_bytes(int64_t n_workgroups);
int64_t cie_paged_decode_planned_partials_bytes(int64_t n_workgroups, int64_t H_q, int64_t H_kv,
                                                int64_t D);
int cie_paged_decode_plan(void* plan, const int64_t* lens, const int64_t* slot_ids,
                          const int64_t* block_table, int64_t B, int64_t H_kv,
                          int64_t page_size, int64_t n_pages, int64_t bt_stride,
                          int64_t bt_width, int64_t n_slots, int64_t append,
                          int64_t n_workgroups, int32_t* err, void* stream);
int cie_paged_decode_planned(void* o, const void* q, const void* k_pool, const void* v_pool,
                             const int32_t* plan, const int64_t* block_table, void* partials,
                             int32_t* counters, int64_t B, int64_t H_q, int64_t H_kv, int64_t D,
                             int64_t page_size, int64_t n_pages, int64_t pool_page_stride,
                             int64_t pool_head_stride, int64_t bt_stride, int64_t bt_width,
                             int64_t n_workgroups, int32_t* err, void* stream);
int cie_paged_decode_append_planned(void* o, const void* q, void* k_pool, void* v_pool,
                                    const void* k_new, const void* v_new,
                                    int64_t k_tok_stride, int64_t k_head_stride,
                                    int64_t v_tok_stride, int64_t v_head_stride,
                                    const int32_t* plan, const int64_t* block_table,
                                    void* partials, int32_t* counters,
                                    int64_t B, int64_t H_q, int64_t H_kv, int64_t D,
                                    int64_t page_size, int64_t n_pages,
                                    int64_t pool_page_stride, int64_t pool_head_stride,
                                    int64_t bt_stride, int64_t bt_width, int64_t n_workgroups,
                                    int32_t* err, void* stream);
int cie_paged_decode_qkv_rope_planned(void* o, const void* qkv, int64_t qkv_row_stride,
                                      const void* cos, const void* sin, int64_t cs_row_stride,
                                      void* k_pool, void* v_pool, const int32_t* plan,
                                      const int64_t* block_table, void* partials,
                                      int32_t* counters, int64_t B, int64_t H_q, int64_t H_kv,
                                      int64_t D, int64_t page_size, int64_t n_pages,
                                      int64_t pool_page_stride, int64_t pool_head_stride,
                                      int64_t bt_stride, int64_t bt_width, int64_t n_workgroups,
                                      int32_t* err, void* stream);

/*
 * Allocation-free form of cie_paged_decode_append.  No counterpart in the
 * reference: it is for callers that cannot allocate device memory (code under
 * hipGraph stream capture, tight serving loops, harnesses that forbid
 * hipMalloc).  Same arguments and result as cie_paged_decode_append without
 * `partials` / `counters`: those live in a static device array of this
 * library (4 MiB of split partials plus 16,384 counter words, one copy per
 * GPU, held until the process ends).  The counters are zeroed by a fill
 * kernel on `stream` at the first call on a device and left zero by every
 * completed call.  A call with n_splits > 1 whose partials
 * (cie_paged_decode_partials_bytes) exceed 4 MiB or with 2 * B * H_kv > 16384
 * returns CIE_ESCRATCH and launches nothing (a one-split call uses no
 * scratch).  cie_paged_decode_noalloc_limit(H_q, H_kv, D, n_splits) gives the
 * largest B this entry point accepts (the scratch bounds, and the kernel's
 * B <= 65535), or -1 for arguments no call accepts (n_splits outside
 * [1, cie_paged_decode_max_splits()], H_q not a multiple of H_kv).  Every
 * call on one GPU shares the array: calls that can overlap in time on one
 * GPU (different streams) race and must not be made.
 */
int64_t cie_paged_decode_noalloc_limit(int64_t H_q, int64_t H_kv, int64_t D, int64_t n_splits);
int cie_paged_decode_append_noalloc(void* o, const void* q, void* k_pool, void* v_pool,
                                    const void* k_new, const void* v_new,
                                    int64_t k_tok_stride, int64_t k_head_stride,
                                    int64_t v_tok_stride, int64_t v_head_stride,
                                    const int64_t* lens, const int64_t* slot_ids,
                                    const int64_t* block_table,
                                    int64_t B, int64_t H_q, int64_t H_kv, int64_t D,
                                    int64_t page_size, int64_t n_pages,
                                    int64_t pool_page_stride, int64_t pool_head_stride,
                                    int64_t bt_stride, int64_t bt_width,
                                    int64_t n_slots, int64_t n_splits, int32_t* err,
                                    void* stream);

/*
 * Decode step from the fused QKV projection, RoPE and KV append fused in, one
 * launch.  Row b of qkv (qkv_row_stride elements apart, 16-byte aligned)
 * holds q (H_q heads), then k (H_kv), then v (H_kv), D each; cos / sin rows b
 * (cs_row_stride apart) are the new token's rotary tables.  q and k are
 * rotated in registers as transformers' apply_rotary_pos_emb does
 * (x*cos + rotate_half(x)*sin, computed in fp32, rounded once to fp16), the
 * rotated k and v rows are appended at pos = lens[slot_ids[b]], and o is the
 * decode attention of the rotated q over the pos + 1 tokens.
 * Replaces the decode branch of TritonQwen2Attention.forward
 * (attn/core.py:181-215): the QKV split, apply_rotary_pos_emb,
 * KVStorage.decode_update and gqa_decode_attention.  Other arguments as for
 * cie_paged_decode_append.
 */
int cie_paged_decode_qkv_rope(void* o, const void* qkv, int64_t qkv_row_stride,
                              const void* cos, const void* sin, int64_t cs_row_stride,
                              void* k_pool, void* v_pool,
                              const int64_t* lens, const int64_t* slot_ids,
                              const int64_t* block_table, void* partials,
                              int32_t* counters,
                              int64_t B, int64_t H_q, int64_t H_kv, int64_t D,
                              int64_t page_size, int64_t n_pages,
                              int64_t pool_page_stride, int64_t pool_head_stride,
                              int64_t bt_stride, int64_t bt_width, int64_t n_slots,
                              int64_t n_splits, int32_t* err, void* stream);

/*
 * Token-mode append from the fused QKV projection, with RoPE: for each packed
 * token t < T (row t of qkv, layout as for cie_paged_decode_qkv_rope; cos /
 * sin row t), the rotated q heads go to q_out (T, H_q, D) dense, and the
 * rotated k and the v rows to (pages[t], head, offsets[t]) of the pools.
 * Replaces the mixed branch's QKV split, apply_rotary_pos_emb and
 * KVStorage.mixed_update (attn/core.py:181-198, 226-229;
 * kv_cache/storage.py:62-85).  D must be a multiple of 16; every pointer
 * 16-byte aligned.
 */
int cie_kv_append_tokens_qkv_rope(void* q_out, void* k_pool, void* v_pool,
                                  const void* qkv, int64_t qkv_row_stride,
                                  const void* cos, const void* sin,
                                  int64_t cs_row_stride,
                                  const int64_t* pages, const int64_t* offsets,
                                  int64_t T, int64_t H_q, int64_t H_kv,
                                  int64_t page_size, int64_t D, int64_t n_pages,
                                  int64_t pool_page_stride,
                                  int64_t pool_head_stride, int32_t* err,
                                  void* stream);

/*
 * Varlen causal GQA attention over the paged pool for a packed batch of
 * chunked-prefill and decode sequences.  Sequence b owns query rows
 * [cu_seqlens[b], cu_seqlens[b+1]); its row i sits at absolute position
 * kv_lens[b] + i and attends keys [0, kv_lens[b] + i] of slot slot_ids[b].
 * Rows outside every sequence are not written.  An Inf or NaN in a key's V row
 * reaches the rows that attend the key, and may reach the rows before them in
 * the same 16 rows of the sequence (rows 16 * i .. 16 * i + 15); no others.
 * Replaces mixed_gqa_attention (attn/core.py:69-111), i.e. the Triton
 * mixed_gqa_attention_kernel (kernels/prefill_attention.py:10-198).
 *   q, o       : (total_T, H_q, D) dense fp16
 *   max_seqlen : upper bound on every sequence's query length (the
 *                reference's metadata token-count bucket); rows past it are
 *                not computed (CIE_ERRBIT_LEN).  B <= 1024 (its plan
 *                tables live in LDS: a batch that would take a workgroup
 *                past the device's LDS limit gets CIE_EUNSUPPORTED).
 *   partials, partials_bytes : a 16-byte aligned buffer of any contents
 *                (per-chunk softmax state of the tiles the call splits over
 *                several workgroups); its size is a budget, not a bound the
 *                call checks against the batch.  Sequences whose split
 *                tiles' rows (rows x H_q x chunks of each split tile) fit
 *                the budget, in sequence order, are split; the rest run
 *                unsplit — same results, longer critical path.  A row takes
 *                4 * (D + 2) bytes; the budget caps at 2,097,088 rows.
 *                cie_mixed_partials_bytes(total_T, H_q, D) is the default:
 *                per q head, the larger of 2 rows per token and 16 rows (a
 *                decode row's most chunks) for each of the first 64 tokens
 *                (about 7.8 MB for 1,052 tokens, 14 heads, D = 64; 3.8 MB
 *                at most below 512 tokens); partials may be NULL with
 *                partials_bytes = 0 (nothing splits).  Launches of many rows
 *                run wide query tiles, which split long prefixes over more
 *                workgroups: cie_mixed_default_partials_bytes is the same
 *                number for the others, and at least 8 rows for each of a
 *                wide launch's first 2,048 tokens (D = 128: 1,024).
 *   counters   : cie_mixed_counters(B, H_kv, max_seqlen) int32, 16-byte
 *                aligned, zero before the call and left zero by it (an
 *                arrival word and a stale word per query tile and column
 *                group, with CIE_ERRBIT_SPLIT as for cie_paged_decode; the
 *                same buffer can serve cie_paged_decode, calls being
 *                stream-ordered)
 */
int64_t cie_mixed_partials_bytes(int64_t total_T, int64_t H_q, int64_t D);
int64_t cie_mixed_default_partials_bytes(int64_t total_T, int64_t max_seqlen, int64_t H_q,
                                         int64_t H_kv, int64_t D);
int64_t cie_mixed_counters(int64_t B, int64_t H_kv, int64_t max_seqlen);
int cie_mixed_attention(void* o, const void* q,
                        const void* k_pool, const void* v_pool,
                        const int64_t* cu_seqlens, const int64_t* kv_lens,
                        const int64_t* slot_ids, const int64_t* block_table,
                        void* partials, int64_t partials_bytes, int32_t* counters,
                        int64_t B, int64_t total_T, int64_t max_seqlen,
                        int64_t H_q, int64_t H_kv, int64_t D,
                        int64_t page_size, int64_t n_pages,
                        int64_t pool_page_stride, int64_t pool_head_stride,
                        int64_t bt_stride, int64_t bt_width, int64_t n_slots,
                        int32_t* err, void* stream);

/*
 * Planned mixed attention: one plan per mixed step.  The batch's sequences
 * (cu_seqlens, kv_lens, slot_ids) are the same for every layer of a step, as
 * the reference's AttentionMetadata is built once per step
 * (attn/metadata.py:3-55) and every layer's mixed_gqa_attention reads it
 * (attn/core.py:69-111).  cie_mixed_plan runs the plan each launch of
 * cie_mixed_attention makes for itself — the work items, their order and
 * the sequences' partial bases — once, into `plan`; each layer's
 * cie_mixed_attention_planned then reads its items' descriptors in one
 * memory round trip instead of loading the sequence tables and planning.
 * The results equal cie_mixed_attention's bit for bit.
 *   plan          : cie_mixed_plan_bytes(B, total_T) bytes, 16-byte aligned;
 *                   valid for the batch (cu_seqlens, kv_lens, slot_ids),
 *                   shape and partials_bytes it was made with.  A planned
 *                   call whose B, max_seqlen's query tiles, H_q, H_kv or
 *                   partials budget differ from the plan's, or whose total_T
 *                   or max_seqlen makes items of another kind (wide ones from
 *                   a number of rows on), writes nothing
 *                   and raises CIE_ERRBIT_PLAN.  A batch with more items than
 *                   the plan holds (only sequences that overlap in
 *                   cu_seqlens can have them) gets an empty plan and
 *                   CIE_ERRBIT_PLAN.  Rows past max_seqlen are reported
 *                   (CIE_ERRBIT_LEN) by cie_mixed_plan.
 *   other arguments as for cie_mixed_attention.
 */
int64_t cie_mixed_plan_bytes(int64_t B, int64_t total_T);
int cie_mixed_plan(int32_t* plan, int64_t plan_bytes,
                   const int64_t* cu_seqlens, const int64_t* kv_lens, const int64_t* slot_ids,
                   int64_t B, int64_t total_T, int64_t max_seqlen,
                   int64_t H_q, int64_t H_kv, int64_t D, int64_t page_size,
                   int64_t bt_width, int64_t n_slots, int64_t partials_bytes,
                   int32_t* err, void* stream);
int cie_mixed_attention_planned(void* o, const void* q,
                                const void* k_pool, const void* v_pool,
                                const int32_t* plan, int64_t plan_bytes,
                                const int64_t* block_table,
                                void* partials, int64_t partials_bytes, int32_t* counters,
                                int64_t B, int64_t total_T, int64_t max_seqlen,
                                int64_t H_q, int64_t H_kv, int64_t D,
                                int64_t page_size, int64_t n_pages,
                                int64_t pool_page_stride, int64_t pool_head_stride,
                                int64_t bt_stride, int64_t bt_width, int64_t n_slots,
                                int32_t* err, void* stream);

/*
 * The 8-bit cache: K and V rows in e4m3 (OCP: finite, largest 448), with a
 * power-of-two scale for each block of 16 tokens, kv head and K / V.
 *   pools      : (n_pages, H_kv, page_size, D) bytes, last two dims dense, 16-byte
 *                aligned, page and head strides multiples of 16 (in elements);
 *                page_size a multiple of 16, D 64 or 128
 *   scales     : (n_pages, H_kv, page_size / 16, 2) dense fp32, 16-byte aligned;
 *                [..., 0] K's and [..., 1] V's, 2^e with -15 <= e <= 8, written by the
 *                appends.  A held value is byte * 2^e, always an fp16 value.
 * A block's e is the least with amax <= 448 * 2^e over the rows written since its
 * row 0 last was: writing row 0 starts the block anew (the bytes of its other rows
 * then mean nothing until written), writing another row keeps the others, rounded
 * again where e grows.  Values are rounded to nearest even; beyond +-61440 (240 *
 * 2^8; infinities too) they are held as that; NaN is held as NaN and not in amax.
 * Nothing else is shared with the fp16 pools' entry points: strides, indices, err,
 * counters and partials behave as theirs do.  No call allocates or synchronises.
 *
 * Append, as cie_kv_append_decode / _tokens / _tokens_qkv_rope:
 *  - decode: slots other than padding must not share the page they append to; of a
 *    slot that comes several times in the batch the last row is written.
 *  - tokens: (pages[t], offsets[t]) in any order; of an index that comes several
 *    times the last token is written.  Bad indices are skipped and reported.
 * Read back: k_out / v_out (T, H_kv, D) dense fp16 = the values of the rows
 * (pages[t], offsets[t]), exactly; zeros (and a report) for a bad index.
 */
int cie_q8_append_decode(void* k_pool, void* v_pool, void* scales,
                         const void* k_new, const void* v_new,
                         int64_t k_tok_stride, int64_t k_head_stride,
                         int64_t v_tok_stride, int64_t v_head_stride,
                         const int64_t* slot_ids, const int64_t* lens,
                         const int64_t* block_table, int64_t B, int64_t H_kv,
                         int64_t page_size, int64_t D, int64_t n_pages,
                         int64_t pool_page_stride, int64_t pool_head_stride,
                         int64_t bt_stride, int64_t bt_width, int64_t n_slots,
                         int32_t* err, void* stream);
int cie_q8_append_tokens(void* k_pool, void* v_pool, void* scales,
                         const void* k_new, const void* v_new,
                         int64_t k_tok_stride, int64_t k_head_stride,
                         int64_t v_tok_stride, int64_t v_head_stride,
                         const int64_t* pages, const int64_t* offsets, int64_t T,
                         int64_t H_kv, int64_t page_size, int64_t D, int64_t n_pages,
                         int64_t pool_page_stride, int64_t pool_head_stride,
                         int32_t* err, void* stream);
int cie_q8_append_tokens_qkv_rope(void* q_out, void* k_pool, void* v_pool, void* scales,
                                  const void* qkv, int64_t qkv_row_stride,
                                  const void* cos, const void* sin, int64_t cs_row_stride,
                                  const int64_t* pages, const int64_t* offsets, int64_t T,
                                  int64_t H_q, int64_t H_kv, int64_t page_size, int64_t D,
                                  int64_t n_pages, int64_t pool_page_stride,
                                  int64_t pool_head_stride, int32_t* err, void* stream);
int cie_q8_read_tokens(void* k_out, void* v_out, const void* k_pool, const void* v_pool,
                       const void* scales, const int64_t* pages, const int64_t* offsets,
                       int64_t T, int64_t H_kv, int64_t page_size, int64_t D,
                       int64_t n_pages, int64_t pool_page_stride,
                       int64_t pool_head_stride, int32_t* err, void* stream);

/*
 * Decode over the 8-bit cache, as cie_paged_decode / _append / _qkv_rope, one launch.
 * plan: NULL, with n_splits splits per (sequence, kv head), or a step's
 * cie_paged_decode_plan (same append mode; lens and slot_ids are then not read), with
 * n_splits its n_workgroups; a plan that does not fit the call (made in the other
 * append mode, for more sequences, heads, slots or pages, or split where the call has
 * no partials) is not followed and raises CIE_ERRBIT_PLAN, or CIE_ERRBIT_PAGE for its
 * pages; of a plan for fewer sequences or heads the others are left as they are, and
 * CIE_ERRBIT_PLAN raised.  (Its lengths, page size and block table are the caller's to
 * keep the same.)  partials:
 * cie_paged_decode_planned_partials_bytes(workgroups, H_q, H_kv, D), workgroups =
 * B * H_kv * n_splits or the plan's; counters: 2 * B * H_kv words; both may be NULL
 * where workgroups == B * H_kv.  The appending forms leave the same bytes and scales
 * as cie_q8_append_decode, and attend them.  n_pages < 2^31.
 */
int cie_q8_decode(void* o, const void* q, const void* k_pool, const void* v_pool,
                  const void* scales, const int64_t* lens, const int64_t* slot_ids,
                  const int64_t* block_table, const int32_t* plan,
                  void* partials, int32_t* counters,
                  int64_t B, int64_t H_q, int64_t H_kv, int64_t D, int64_t page_size,
                  int64_t n_pages, int64_t pool_page_stride, int64_t pool_head_stride,
                  int64_t bt_stride, int64_t bt_width, int64_t n_slots,
                  int64_t n_splits, int32_t* err, void* stream);
int cie_q8_decode_append(void* o, const void* q, void* k_pool, void* v_pool, void* scales,
                         const void* k_new, const void* v_new,
                         int64_t k_tok_stride, int64_t k_head_stride,
                         int64_t v_tok_stride, int64_t v_head_stride,
                         const int64_t* lens, const int64_t* slot_ids,
                         const int64_t* block_table, const int32_t* plan,
                         void* partials, int32_t* counters,
                         int64_t B, int64_t H_q, int64_t H_kv, int64_t D, int64_t page_size,
                         int64_t n_pages, int64_t pool_page_stride, int64_t pool_head_stride,
                         int64_t bt_stride, int64_t bt_width, int64_t n_slots,
                         int64_t n_splits, int32_t* err, void* stream);
int cie_q8_decode_qkv_rope(void* o, const void* qkv, int64_t qkv_row_stride,
                           const void* cos, const void* sin, int64_t cs_row_stride,
                           void* k_pool, void* v_pool, void* scales,
                           const int64_t* lens, const int64_t* slot_ids,
                           const int64_t* block_table, const int32_t* plan,
                           void* partials, int32_t* counters,
                           int64_t B, int64_t H_q, int64_t H_kv, int64_t D, int64_t page_size,
                           int64_t n_pages, int64_t pool_page_stride, int64_t pool_head_stride,
                           int64_t bt_stride, int64_t bt_width, int64_t n_slots,
                           int64_t n_splits, int32_t* err, void* stream);

/*
 * Varlen causal attention over the 8-bit cache, as cie_mixed_attention, from a plan:
 *   cie_q8_mixed_plan   once per step: the work items of its sequences, into `plan`
 *                       (cie_q8_mixed_plan_bytes bytes, 16-byte aligned, any
 *                       contents).  Index errors, and rows at or past max_seqlen
 *                       (not computed), are reported here.
 *   cie_q8_mixed        per layer.  A plan made for other sizes (B, total_T, heads,
 *                       D, page_size, block table) writes nothing and raises
 *                       CIE_ERRBIT_PLAN.  Where cu_seqlens decreases anywhere,
 *                       nothing of the batch is computed (CIE_ERRBIT_PAGE).
 * A NaN in a key's K or V row reaches the rows that attend the key, and no others.
 * partials: cie_q8_mixed_partials_bytes bytes, 16-byte aligned; counters:
 * cie_q8_mixed_counters() words, zero before the call and after it.
 * B <= 2048, H_q / H_kv <= 16, total_T <= 2^24.
 */
int64_t cie_q8_mixed_plan_bytes(int64_t B, int64_t total_T, int64_t H_q, int64_t H_kv);
int64_t cie_q8_mixed_partials_bytes(int64_t total_T, int64_t H_q, int64_t D);
int64_t cie_q8_mixed_counters(void);
int cie_q8_mixed_plan(int32_t* plan, int64_t plan_bytes,
                      const int64_t* cu_seqlens, const int64_t* kv_lens, const int64_t* slot_ids,
                      int64_t B, int64_t total_T, int64_t max_seqlen,
                      int64_t H_q, int64_t H_kv, int64_t D, int64_t page_size,
                      int64_t bt_width, int64_t n_slots, int32_t* err, void* stream);
int cie_q8_mixed(void* o, const void* q, const void* k_pool, const void* v_pool,
                 const void* scales, const int32_t* plan, int64_t plan_bytes,
                 const int64_t* block_table, void* partials, int64_t partials_bytes,
                 int32_t* counters, int64_t B, int64_t total_T,
                 int64_t H_q, int64_t H_kv, int64_t D, int64_t page_size, int64_t n_pages,
                 int64_t pool_page_stride, int64_t pool_head_stride,
                 int64_t bt_stride, int64_t bt_width, int64_t n_slots,
                 int32_t* err, void* stream);

/*
 * Block tables and slot maps from request lengths.  Sequence b is slot
 * slot_ids[b], holds lens[slot] tokens (lens (n_slots,)) and has new_tokens[b] new
 * ones, packed one sequence after another:
 *   cu_seqlens[b + 1] = cu_seqlens[b] + new_tokens[b]              (B + 1 words)
 *   row t of sequence b: slots[t] = slot, positions[t] = lens[slot] + t - cu[b],
 *     pages[t] = block_table[slot, position / page_size],
 *     offsets[t] = position % page_size                            (T words each)
 * Rows behind the last sequence get zeros (slot 0 and page 0: the padding rows').
 * Beside the reference's AttentionMetadata and its mixed step's index recipe
 * (attn/metadata.py:3-55, scheduler/mixed_module.py:99-132).
 *
 * free_list (nullable): n_pages + 2 words: the count of free pages, a word of the
 * kernels' own (0), and the free pages, the next one last.  With it, each sequence
 * of a slot other than 0 first gets the pages that its new tokens need, in the
 * order of the sequences and of their positions: into block_table, and out of the
 * list.  If the list has too few, or a slot comes twice among sequences with new
 * tokens, no sequence gets any (CIE_ERRBIT_FREE).  Rows whose page the sequence has
 * not got are mapped to page 0.
 * A bad slot id: its rows are padding rows (CIE_ERRBIT_PAGE).  A position past the
 * table's row: page 0, offset 0, and no new pages for its sequence; rows past T are
 * dropped, negative counts are 0 (CIE_ERRBIT_LEN).  Page ids are not checked, but
 * for those of the list (CIE_ERRBIT_PAGE, page 0 in their place).
 * lens is not advanced.  B <= 2048, T <= 2^24, n_pages and bt_width <= 2^24,
 * page_size <= 2^30.
 */
int cie_step_maps(int64_t* cu_seqlens, int64_t* slots, int64_t* positions, int64_t* pages,
                  int64_t* offsets, const int64_t* slot_ids, const int64_t* new_tokens,
                  const int64_t* lens, int64_t* block_table, int64_t* free_list,
                  int64_t B, int64_t T, int64_t page_size, int64_t n_pages,
                  int64_t bt_stride, int64_t bt_width, int64_t n_slots,
                  int32_t* err, void* stream);

/*
 * Gives pages back: sequence b keeps keep[b] tokens (NULL: none) of the held[b]
 * whose pages it has (NULL: lens[slot]; held >= lens[slot], as after cie_step_maps
 * and before lens is advanced).  Its pages past the kept tokens go back to the list, in the reverse
 * of the order in which cie_step_maps hands pages out, their table entries become
 * 0, and lens[slot] = keep[b].  Slot 0 is left as it is.
 * A slot that comes twice, or a list that has no room for the pages: nothing is
 * done (CIE_ERRBIT_FREE).  A bad slot id (CIE_ERRBIT_PAGE) or lengths that are not
 * 0 <= keep <= held <= the table's row, lens[slot] <= held (CIE_ERRBIT_LEN): that
 * sequence is left as it is.  Table entries of 0 hold no page, as after a
 * cie_step_maps whose pages the list did not have: they are not given back
 * (CIE_ERRBIT_PAGE).  A page id outside the pool goes into the list as page 0
 * (CIE_ERRBIT_PAGE, here and where it is handed out).  Sizes as cie_step_maps.
 */
int cie_release_pages(int64_t* free_list, const int64_t* slot_ids, int64_t* lens,
                      int64_t* block_table, const int64_t* keep, const int64_t* held,
                      int64_t B, int64_t page_size, int64_t n_pages,
                      int64_t bt_stride, int64_t bt_width, int64_t n_slots,
                      int32_t* err, void* stream);

/*
 * Rotary positions.  Pair i of a head's first rot dims, (x, y), becomes
 *   scale * (x cos a - y sin a, y cos a + x sin a),  a = positions[t] * freqs[i]
 * with freqs[i] in radians a position (rot / 2 doubles).  Pairs are dims
 * (i, i + rot / 2), or (2i, 2i + 1) where interleaved; dims from rot on are copied.
 * Angles are computed in fp64 (for 16-bit types their cos and sin in fp32), products
 * and sums in fp32, outputs rounded once.
 * Beside apply_rotary_pos_emb of the reference's layer (attn/core.py:193-198).
 *   cie_rotary         q (T, H_q, D) and k (T, H_kv, D) views, their own token and
 *                      head strides (elements), dims dense; either may have no
 *                      heads.  Outputs dense, and not in the inputs' memory.
 *   cie_kv_append_tokens_qkv_rotary
 *                      from rows of the fused QKV projection, as
 *                      cie_kv_append_tokens_qkv_rope: q into q_out, k and v into
 *                      the pools (16-bit types).
 *   cie_rotary_tables  scale * cos a and scale * sin a for each of rot dims,
 *                      (T, rot) each.
 * dtype: CIE_F16, CIE_BF16 or CIE_F32, of inputs and outputs.  rot, D even.
 */
int cie_rotary(void* q_out, void* k_out, const void* q, const void* k,
               int64_t q_tok_stride, int64_t q_head_stride,
               int64_t k_tok_stride, int64_t k_head_stride,
               const int64_t* positions, const double* freqs, double scale,
               int64_t T, int64_t H_q, int64_t H_kv, int64_t D, int64_t rot,
               int interleaved, int dtype, void* stream);
int cie_kv_append_tokens_qkv_rotary(void* q_out, void* k_pool, void* v_pool, const void* qkv,
                                    int64_t qkv_row_stride, const int64_t* positions,
                                    const double* freqs, double scale,
                                    const int64_t* pages, const int64_t* offsets,
                                    int64_t T, int64_t H_q, int64_t H_kv, int64_t page_size,
                                    int64_t D, int64_t n_pages, int64_t pool_page_stride,
                                    int64_t pool_head_stride, int64_t rot, int interleaved,
                                    int dtype, int32_t* err, void* stream);
int cie_rotary_tables(void* cos, void* sin, const int64_t* positions, const double* freqs,
                      double scale, int64_t T, int64_t rot, int interleaved, int dtype,
                      void* stream);

/*
 * Low-rank adapters of many requests beside a shared projection:
 *   y[t, s] += scales[i] * B[i, s] (A[i, s] x[t]),   i = the adapter of row t,
 * for each slice s of y's columns, in place.  a (N, n_slices, R, d_in) and b
 * (N, d_out, R) dense, d_out the slices' widths together; scales (N) float;
 * ranks (N) int32: adapter i has ranks[i] <= R rows of rank, and zeros behind them
 * in a and b.  Rows without an adapter, and rows behind T, are left as they are.
 * A x is summed in fp32 and enters the second product as two values of float16 (22
 * bits, or 2^-39 of the row's largest in its slice where that is more) or three of
 * bfloat16 (all 24), that one summed in fp32 and added to y in fp32:
 * one rounding to the element type at the end.
 *   cie_adapter_plan   once per step: which rows share an adapter, into `plan`
 *                      (cie_adapter_plan_bytes(T, N) bytes, 16-byte aligned, any
 *                      contents).  Row t has adapter slot_adapters[row_slots[t]]
 *                      (row_slots NULL: slot_adapters[t]); a negative one is none, as
 *                      is a bad slot (CIE_ERRBIT_PAGE) or one >= N (CIE_ERRBIT_ADAPTER).
 *   cie_adapter_add    per projection.  A plan made for other T or N: nothing is
 *                      written, CIE_ERRBIT_PLAN.
 * slice_widths: n_slices (<= 4) host values.  R a multiple of 16, R <= 128;
 * N <= 1024, T <= 2^24; dtype CIE_F16 or CIE_BF16; x and y rows are dense, with
 * their own row strides (elements), x not in y's memory.
 */
int64_t cie_adapter_plan_bytes(int64_t T, int64_t N);
int cie_adapter_plan(int32_t* plan, int64_t plan_bytes, const int64_t* row_slots,
                     const int64_t* slot_adapters, int64_t T, int64_t n_slots, int64_t N,
                     int32_t* err, void* stream);
int cie_adapter_add(void* y, int64_t y_row_stride, const void* x, int64_t x_row_stride,
                    const void* a, const void* b, const float* scales, const int32_t* ranks,
                    const int32_t* plan, int64_t plan_bytes, int64_t T, int64_t N, int64_t R,
                    int64_t d_in, const int64_t* slice_widths, int64_t n_slices,
                    int dtype, int32_t* err, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* CIE_PAGED_ATTENTION_H */
