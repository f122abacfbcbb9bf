/*
 * dsa_b200.h -- C ABI of the B200 (sm_100a) DSA decode kernels.
 *
 * Two operators, both destination-passing style (the caller owns inputs,
 * outputs and the scratch workspace; nothing here allocates device memory):
 *
 *   dsa_indexer_run    -- FP8 lightning indexer + top-2048 select.
 *     Replaces the reference entry point
 *       run(q_index_fp8, k_index_cache_fp8, weights, seq_lens, block_table,
 *           topk_indices)
 *     at dsa_indexer/solution/triton/kernel.py:364-436 and its host driver
 *     dsa_topk_run_ms (kernel.py:190-319).
 *
 *   dsa_attention_run  -- sparse MLA attention over the selected slots.
 *     Replaces the reference entry point
 *       run(q_nope, q_pe, ckv_cache, kpe_cache, sparse_indices, sm_scale,
 *           output, lse)
 *     at dsa_attention/solution/triton/kernel.py:240-252 and its host driver
 *     dsa_sparse_attention (kernel.py:174-218).
 *
 * All pointers are device pointers except where stated; all launches go to
 * `stream` (a cudaStream_t passed as void*), so calls are CUDA-graph
 * capturable.  No call synchronises the device or reads device memory on the
 * host (unlike the reference indexer, which reads seq_lens on the host at
 * kernel.py:375).
 *
 * Every function returns a dsa_status (0 == DSA_OK).  Argument errors are
 * detected on the host before anything is launched.  Data-dependent errors
 * (a page id outside the pool, a seq_len larger than the block table, a
 * sparse index outside the cache, a bounded wait that ran out) are recorded
 * by the kernels as bits of a sticky 32-bit word at the start of the
 * workspace; dsa_read_device_status() reads and optionally clears it.
 */
#ifndef DSA_B200_H_
#define DSA_B200_H_

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define DSA_API __attribute__((visibility("default")))
#else
#define DSA_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes (host side) ---------------------------------------- */
#define DSA_OK                       0
#define DSA_ERR_INVALID_ARGUMENT     1
#define DSA_ERR_MISALIGNED           2
#define DSA_ERR_WORKSPACE_TOO_SMALL  3
#define DSA_ERR_CUDA                 4
#define DSA_ERR_UNSUPPORTED_DEVICE   5
#define DSA_ERR_TENSOR_MAP           6
#define DSA_ERR_OVERLAP              7

/* ---- sticky device status bits (first uint32 of each workspace) ------ */
#define DSA_DEV_BAD_SEQ_LEN   0x1u  /* seq_len < 0 or > max_pages*64; clamped   */
#define DSA_DEV_BAD_PAGE      0x2u  /* block_table entry outside [0, num_pages) */
#define DSA_DEV_BAD_INDEX     0x4u  /* sparse index outside [-1, num_slots)     */
#define DSA_DEV_WAIT_TIMEOUT  0x8u  /* a bounded pipeline wait gave up          */
#define DSA_DEV_STALE_WORKSPACE 0x10u /* workspace contents did not match: a merge */
                                      /* counter not zero on entry, or an indexer */
                                      /* histogram not matching its scores        */

/* Shape constants of the two contest definitions
 * dsa_topk_indexer_fp8_h64_d128_topk2048_ps64 and
 * dsa_sparse_attention_h16_ckv512_kpe64_topk2048_ps64. */
#define DSA_PAGE_SIZE        64
#define DSA_INDEX_HEADS      64
#define DSA_INDEX_DIM        128
#define DSA_INDEX_PAGE_BYTES 8448  /* 64*128 fp8 + 64 fp32 scales (kernel.py:80) */
#define DSA_TOPK             2048
#define DSA_ATTN_HEADS       16
#define DSA_CKV_DIM          512
#define DSA_KPE_DIM          64
/* A page of the 8-bit latent cache: 64 x 512 e4m3 codes (ckv), then 64 x 64 bf16
 * (kpe), then 64 fp32 scales, one for each token: a latent is code * scale. */
#define DSA_LATENT_PAGE_BYTES 41216

/* Version of this ABI (bumped on any signature change). */
DSA_API int dsa_b200_abi_version(void);

/* Human-readable text for a dsa_status value; never NULL. */
DSA_API const char* dsa_b200_status_string(int status);

/* Bytes of device workspace dsa_indexer_run needs for this batch and block
 * table width: a 256-byte header, 32 KiB of per-request ready counters
 * (the score kernel counts each request's scored tiles there and the top-k
 * select of that request starts once they are all counted; the counters
 * carry over from call to call and are never reset), a [batch, 2048] uint32
 * radix histogram (cleared by the call itself, on its stream, before the
 * scores are added) and [batch, max_pages*64] fp32 score rows.  Zero-fill a
 * workspace once before its first use, so that the status word in its
 * header starts clear and the ready counters start consistent. */
DSA_API size_t dsa_indexer_workspace_bytes(int32_t batch, int32_t max_pages);

/* FP8 lightning indexer, decode (one query token per request).
 *
 *   q_index_fp8       [batch, 64, 128] float8_e4m3fn, contiguous
 *   k_index_cache_fp8 num_pages pages of 8448 bytes: 64x128 fp8 then 64 fp32
 *                     scales (the [num_pages, 64, 1, 132] uint8 cache viewed
 *                     as bytes), 16-byte aligned
 *   weights           [batch, 64] fp32
 *   seq_lens          [batch] int32 (device memory; never read on the host)
 *   block_table       [batch, max_pages] int32
 *   topk_indices      [batch, 2048] int32 output: global slot ids
 *                     block_table[b, t/64]*64 + t%64 of the top-min(L,2048)
 *                     tokens, score descending, ties by lower token index,
 *                     then -1 padding.
 *
 * Mirrors dsa_indexer/solution/triton/kernel.py:364 (argument order and
 * meaning), plus the sizes a C caller must pass explicitly. */
DSA_API int dsa_indexer_run(const void* q_index_fp8, const void* k_index_cache_fp8,
                    int64_t num_pages, const float* weights,
                    const int32_t* seq_lens, const int32_t* block_table,
                    int32_t batch, int32_t max_pages, int32_t* topk_indices,
                    void* workspace, size_t workspace_bytes, void* stream);

/* Bytes of device workspace dsa_attention_run needs for num_tokens queries
 * on this device: a 256-byte header, two split-softmax partial records per
 * CTA (a token segment's O in fp32 and its per-head max and sum, 32.1 KiB
 * each) and two merge counters per token, placed at the end of the
 * workspace.  Zero-fill a workspace once before its first use (status word
 * and counters start at zero) and pass the same workspace_bytes to every
 * call on it.  Every call leaves the counters at zero again, including one
 * that gave up on a bounded wait (DSA_DEV_WAIT_TIMEOUT).  A counter found
 * non-zero on entry (the workspace was changed from outside, or two calls on
 * it overlapped) is reported as DSA_DEV_STALE_WORKSPACE by this and every
 * later call until the workspace is zero-filled again. */
DSA_API size_t dsa_attention_workspace_bytes(int32_t num_tokens);

/* Sparse MLA attention, one query token per row of sparse_indices.
 * Launched with programmatic stream serialization: it may be scheduled while
 * the previous kernel on `stream` drains, and touches global memory only
 * after that kernel has completed.
 *
 *   q_nope          [num_tokens, 16, 512] bf16
 *   q_pe            [num_tokens, 16, 64]  bf16
 *   ckv_cache       num_slots rows of 512 bf16 ([pages, 64, 512] flattened)
 *   kpe_cache       num_slots rows of 64 bf16  ([pages, 64, 64] flattened)
 *   sparse_indices  [num_tokens, 2048] int32 global slot ids, -1 = padding
 *   output          [num_tokens, 16, 512] bf16
 *   lse             [num_tokens, 16] fp32, base-2 log-sum-exp of the scaled
 *                   logits; -inf (and output 0) for a row with no valid index
 *
 * Mirrors dsa_attention/solution/triton/kernel.py:241 (argument order and
 * meaning), plus the sizes a C caller must pass explicitly. */
DSA_API int dsa_attention_run(const void* q_nope, const void* q_pe,
                      const void* ckv_cache, const void* kpe_cache,
                      int64_t num_slots, const int32_t* sparse_indices,
                      int32_t num_tokens, float sm_scale,
                      void* output, float* lse,
                      void* workspace, size_t workspace_bytes, void* stream);

/* Size of the scratch array compiled into the library for
 * dsa_indexer_run_noalloc: the 256-byte header, the per-request ready
 * counters (32 KiB), 64 radix histograms and 1,048,576 fp32 score slots
 * (4.5 MiB per GPU that loads the library). */
#define DSA_NOALLOC_SCRATCH_BYTES (256u + 32768u + 64u * 2048u * 4u + 1048576u * 4u)

/* dsa_indexer_run without a workspace argument, for callers that cannot
 * allocate device memory when they call: hosts that reach this library
 * through C / JNI / FFI while another allocator owns the device memory, and
 * serving loops that allow no cudaMalloc after warm-up.  Scratch comes from
 * a fixed array inside the library (DSA_NOALLOC_SCRATCH_BYTES), so the
 * problem must fit: dsa_indexer_workspace_bytes(batch, max_pages) may not
 * exceed it (e.g. 64 requests x 256 pages, or 8 requests x 2048 pages);
 * otherwise the call returns DSA_ERR_WORKSPACE_TOO_SMALL before touching the
 * device.  Nothing is allocated or freed.
 *   - The first call on a device looks up the array's device address, so
 *     make it before capturing any stream.
 *   - All calls share the one array: calls whose work overlaps on the GPU
 *     (other streams, other threads) race and corrupt each other's results.
 *   - Data-dependent device errors are recorded in the array's status word,
 *     which this entry point gives no way to read; use dsa_indexer_run when
 *     they must be observed.
 * Arguments have the meaning of dsa_indexer_run.  No counterpart in the
 * reference, which always allocates its scratch through PyTorch. */
DSA_API int dsa_indexer_run_noalloc(const void* q_index_fp8, const void* k_index_cache_fp8,
                                    int64_t num_pages, const float* weights,
                                    const int32_t* seq_lens, const int32_t* block_table,
                                    int32_t batch, int32_t max_pages, int32_t* topk_indices,
                                    void* stream);

/* Bytes of device workspace dsa_indexer_prefill_run needs: a 256-byte header,
 * a [num_rows, 2048] uint32 radix histogram (cleared by the call), [num_rows,
 * max_pages*64] fp32 score rows and the row-group plan (about
 * (num_rows + 3*num_requests)/4 groups of 16 bytes, plus 4 bytes per row and
 * per request).  Zero-fill it once before its first use. */
DSA_API size_t dsa_indexer_prefill_workspace_bytes(int32_t num_rows, int32_t num_requests,
                                                   int32_t max_pages);

/* FP8 lightning indexer for many query rows per request (prefill, chunked
 * prefill, speculative rows): row t of request r is the decode problem
 * (q[t], weights[t], seq_lens[t], block_table[r]).
 *
 *   q_index_fp8       [num_rows, 64, 128] float8_e4m3fn, 16-byte aligned
 *   k_index_cache_fp8 as for dsa_indexer_run
 *   weights           [num_rows, 64] fp32, 16-byte aligned
 *   seq_lens          [num_rows] int32: tokens row t sees (causal rows of a
 *                     prefill chunk see growing prefixes)
 *   block_table       [num_requests, max_pages] int32
 *   cu_seqlens_q      [num_requests + 1] int32: request r owns rows
 *                     [cu_seqlens_q[r], cu_seqlens_q[r+1]); 0 and num_rows
 *                     at the ends (a violation sets DSA_DEV_BAD_SEQ_LEN)
 *   topk_indices      [num_rows, 2048] int32 output, as for dsa_indexer_run
 *
 * Rows are scored four at a time per request as one FP8 tensor-core GEMM
 * (N = 4 rows x 64 heads), so each 128-token K tile is read once per four
 * rows.  With cu_seqlens_q = 0..num_rows it computes exactly what
 * dsa_indexer_run computes.  No counterpart in the reference, whose indexer
 * definition is decode-only (one query per request). */
DSA_API int dsa_indexer_prefill_run(const void* q_index_fp8, const void* k_index_cache_fp8,
                                    int64_t num_pages, const float* weights,
                                    const int32_t* seq_lens, const int32_t* block_table,
                                    const int32_t* cu_seqlens_q, int32_t num_rows,
                                    int32_t num_requests, int32_t max_pages,
                                    int32_t* topk_indices, void* workspace, size_t workspace_bytes,
                                    void* stream);

/* Quantises new indexer keys into the paged FP8 K cache (the step before
 * dsa_indexer_run in a serving loop).
 *
 *   k                  [num_tokens, 128] bf16, 8-byte aligned
 *   slot_mapping       [num_tokens] int64 global slot ids (page*64 + token);
 *                      negative = padding, skipped
 *   k_index_cache_fp8  num_pages pages of 8448 bytes (the layout
 *                      dsa_indexer_run reads), 16-byte aligned
 *   ue8m0              non-zero: round each scale up to a power of two
 *   status             optional device word (NULL = none): DSA_DEV_BAD_INDEX
 *                      is OR-ed in for a slot >= num_pages*64 (not written)
 *
 * Per token: scale = max(1e-4, max|k|)/448 (ue8m0: 2^ceil(log2 scale)),
 * fp8 = e4m3(k/scale) round-to-nearest-even, stored at the token's row and
 * scale slot.  The reference only defines the page layout
 * (dsa_indexer/solution/triton/kernel.py:80,120-124); the arithmetic is the
 * published vLLM indexer cache writer (indexer_k_quant_and_cache). */
DSA_API int dsa_index_cache_write(const void* k, const int64_t* slot_mapping, int32_t num_tokens,
                                  void* k_index_cache_fp8, int64_t num_pages, int32_t ue8m0,
                                  uint32_t* status, void* stream);

/* Bytes of device workspace dsa_tree_attention_run needs on this device, the
 * same for every call: a 256-byte header, two fp32 records of 64 rows per SM
 * (39 MB in all) for contexts that several SMs share, and the call's list of
 * row groups (2.6 MB).  Zero-fill it once (its status word); nothing else in
 * it carries over from call to call.  Calls that may overlap on the device
 * need a workspace each; threads may call with one workspace on one stream. */
DSA_API size_t dsa_tree_attention_workspace_bytes(void);

/* Attention of a tree of drafted tokens over the paged ckv / kpe cache
 * (speculative decoding; one draft per request is plain dense decoding).
 * Request r has prefix_lens[r] cached tokens and the drafts
 * cu_drafts[r] .. cu_drafts[r+1]-1, whose ckv / kpe rows lie in the cache
 * behind the prefix (position prefix + j for its j-th draft).  A draft sees
 * the whole prefix and those drafts of its request whose bits its mask has.
 * Equal to indexer and sparse attention where a draft sees at most 2048 tokens.
 *
 *   q_nope        [num_drafts, num_heads, 512] bf16, contiguous
 *   q_pe          [num_drafts, num_heads, 64] bf16, contiguous
 *   ckv_cache     num_pages pages of 64 rows of 512 bf16; pages lie
 *                 ckv_page_bytes apart and a page's rows ckv_row_bytes
 *                 (multiples of 16: ckv and kpe may be slices of one cache)
 *   kpe_cache     the same with rows of 64 bf16
 *   prefix_lens   [num_requests] int32
 *   block_table   [num_requests, max_pages] int32
 *   cu_drafts     [num_requests + 1] int32; rows outside of
 *                 [cu_drafts[0], cu_drafts[num_requests]) are left as they are
 *   tree_mask     [num_drafts, mask_words] int64: bit j & 63 of word j / 64
 *                 is set if the draft sees its request's j-th draft (itself
 *                 and its ancestors, as a rule); 64 * mask_words drafts a
 *                 request at most; bits of drafts that the request does not
 *                 have are ignored
 *   output        [num_drafts, num_heads, 512] bf16; may be q_nope itself
 *   lse           [num_drafts, num_heads] fp32, base-2 log-sum-exp of the
 *                 scaled logits; a row that sees nothing has -inf, output 0
 *
 * Outputs that share memory with anything else: DSA_ERR_OVERLAP.
 * 1 <= num_heads <= 128; num_drafts * num_heads <= 2^24, num_requests <= 65536
 * and (num_drafts * num_heads / 64 + num_requests) * (max_pages + 3) <= 2^30.
 * Masked cache rows may hold anything; whether a visible row with a logit of
 * -inf adds 0 times its infinite values or nothing is not defined.  Data-dependent
 * errors: lengths that do not fit the table (clamped), drafts that do not fit
 * cu_drafts or the mask (left out), a cu_drafts that decreases (the call then
 * writes no row): DSA_DEV_BAD_SEQ_LEN; page ids outside the pool (their tokens
 * are masked): DSA_DEV_BAD_PAGE. */
DSA_API int dsa_tree_attention_run(const void* q_nope, const void* q_pe, const void* ckv_cache,
                                   int64_t ckv_page_bytes, int64_t ckv_row_bytes,
                                   const void* kpe_cache, int64_t kpe_page_bytes,
                                   int64_t kpe_row_bytes, int64_t num_pages,
                                   const int32_t* prefix_lens, const int32_t* block_table,
                                   const int32_t* cu_drafts, const int64_t* tree_mask,
                                   int32_t num_requests, int32_t num_drafts, int32_t num_heads,
                                   int32_t max_pages, int32_t mask_words, float sm_scale,
                                   void* output, float* lse, void* workspace,
                                   size_t workspace_bytes, void* stream);

/* Accumulates the attention weight that each cached token got from the rows
 * of a dsa_tree_attention_run with the same arguments:
 *   acc_out[r, k] = acc[r, k] + sum over drafts i of r, heads h that see k of
 *                   2^(scaled logit - lse[i, h])
 * for every position k < max_pages * 64 (+ 0 behind a request's tokens).
 *
 *   lse           [num_drafts, num_heads] fp32, as the attention gave it; a
 *                 row with -inf adds nothing (so rows of rejected drafts are
 *                 kept out; leaving them out of the arguments would move the
 *                 positions of the drafts behind them)
 *   acc           [num_requests, max_pages * 64] fp32, rows acc_stride apart
 *   acc_out       likewise; may be acc itself, else it shares memory with no
 *                 other argument (DSA_ERR_OVERLAP)
 *
 * The sums run in a fixed order (no atomics).  The workspace holds only the
 * status word (256 bytes). */
DSA_API int dsa_tree_weights_run(const void* q_nope, const void* q_pe, const void* ckv_cache,
                                 int64_t ckv_page_bytes, int64_t ckv_row_bytes,
                                 const void* kpe_cache, int64_t kpe_page_bytes,
                                 int64_t kpe_row_bytes, int64_t num_pages,
                                 const int32_t* prefix_lens, const int32_t* block_table,
                                 const int32_t* cu_drafts, const int64_t* tree_mask,
                                 int32_t num_requests, int32_t num_drafts, int32_t num_heads,
                                 int32_t max_pages, int32_t mask_words, float sm_scale,
                                 const float* lse, const float* acc, int64_t acc_stride,
                                 float* acc_out, int64_t acc_out_stride, void* workspace,
                                 size_t workspace_bytes, void* stream);

/* Evicts tokens by accumulated attention weight and moves what is kept to new
 * pages.  Request r has seq_lens[r] tokens.  If they are more than `budget`,
 * its first num_sink and last num_recent tokens are kept, and of those between
 * them the ones of largest acc (equal: the earlier; NaN is largest), `budget`
 * in all; else all are kept.  The order of the kept tokens stays.
 *
 *   acc               [num_requests, max_pages * 64] fp32, rows acc_stride apart
 *   seq_lens          [num_requests] int32
 *   block_table       [num_requests, max_pages] int32
 *   new_block_table   [num_requests, new_max_pages] int32, budget <=
 *                     64 * new_max_pages: pages of the same pool that no
 *                     request's block_table row uses (several requests may
 *                     share pages to move from: nothing there is changed)
 *   ckv_cache, kpe_cache  as for dsa_tree_attention_run, written in place
 *   k_index_cache_fp8 num_pages pages of 8448 bytes, or NULL
 *   keep              [num_requests, budget] int32: the kept positions,
 *                     ascending, then -1
 *   new_seq_lens      [num_requests] int32; may be seq_lens itself
 *   new_acc           [num_requests, new_max_pages * 64] fp32, rows
 *                     new_acc_stride apart: acc of the kept tokens, then 0
 *
 * Token keep[r, i] becomes token i of the new table's row.  keep, new_seq_lens
 * and new_acc share memory neither with one another nor with acc, the tables
 * or (but for new_seq_lens in place) seq_lens: DSA_ERR_OVERLAP.  Data-dependent
 * errors: a seq_len outside [0, max_pages * 64] (clamped):
 * DSA_DEV_BAD_SEQ_LEN; a page outside the pool (its tokens are not moved):
 * DSA_DEV_BAD_PAGE.  The workspace holds only the status word (256 bytes). */
DSA_API int dsa_cache_evict_run(const float* acc, int64_t acc_stride, const int32_t* seq_lens,
                                const int32_t* block_table, const int32_t* new_block_table,
                                int32_t num_requests, int32_t max_pages, int32_t new_max_pages,
                                void* ckv_cache, int64_t ckv_page_bytes, int64_t ckv_row_bytes,
                                void* kpe_cache, int64_t kpe_page_bytes, int64_t kpe_row_bytes,
                                void* k_index_cache_fp8, int64_t num_pages, int32_t budget,
                                int32_t num_sink, int32_t num_recent, int32_t* keep,
                                int32_t* new_seq_lens, float* new_acc, int64_t new_acc_stride,
                                void* workspace, size_t workspace_bytes, void* stream);

/* Writes new tokens into the paged latent cache in 8 bits, with the latent's norm
 * and the rotation of the position part in the same pass.  With c the first 512
 * and e the last 64 values of a token's row:
 *   t = c * norm_weight,  r = 1 / sqrt(mean(c^2) + eps),  M = max |t|
 *   codes = e4m3(448 t / M) to nearest even,  scale = r M / 448
 *   e: (a, b) -> (a cos - b sin, b cos + a sin) for its 32 pairs
 *
 *   kv             num_tokens rows of 576 bf16, kv_row_bytes apart (a multiple of
 *                  16, the base 16-byte aligned)
 *   slot_mapping   [num_tokens] int64 global slot ids (page * 64 + token);
 *                  negative: padding, skipped.  What a slot holds that is given
 *                  twice in one call is not defined.
 *   norm_weight    [512] bf16, 16-byte aligned; NULL: no norm (t = c, r = 1)
 *   positions      [num_tokens] int64, with cos_sin [max_positions, 64] fp32: 32
 *                  cosines, then 32 sines of a position's angles; both NULL: no
 *                  rotation
 *   interleaved    non-zero: the pairs are (2 i, 2 i + 1); zero: (i, i + 32)
 *   latent_cache   num_pages pages of DSA_LATENT_PAGE_BYTES, 16-byte aligned
 *   status         optional device word (NULL: none): DSA_DEV_BAD_INDEX is OR-ed
 *                  in for a slot >= num_pages * 64 or a position outside of the
 *                  table; such a token is not written
 *
 * A row with an infinity or NaN in its latent, or whose scale would be above the
 * largest fp32 number, is stored as NaN throughout, one whose scale would be below
 * 2^-126 as zeros; both have the scale 1.  A cache that shares memory with an input:
 * DSA_ERR_OVERLAP. */
DSA_API int dsa_latent_cache_write(const void* kv, int64_t kv_row_bytes, const int64_t* slot_mapping,
                                   int32_t num_tokens, const void* norm_weight, float eps,
                                   const int64_t* positions, const float* cos_sin, int64_t max_positions,
                                   int32_t interleaved, void* latent_cache, int64_t num_pages,
                                   uint32_t* status, void* stream);

/* Reads ranges of cached tokens back: row cu_rows[r] + i becomes the token at
 * position starts[r] + i of request r, ckv as bf16(code * scale), kpe as it is.
 *
 *   block_table    [num_requests, max_pages] int32
 *   starts         [num_requests] int32
 *   cu_rows        [num_requests + 1] int32, ascending; rows outside of
 *                  [cu_rows[0], cu_rows[num_requests]) are left as they are
 *   ckv, kpe       num_rows rows of 512 and 64 bf16, 16-byte aligned and
 *                  multiples of 16 bytes apart (they may be columns of one buffer)
 *   status         device word: DSA_DEV_BAD_SEQ_LEN for a position outside of the
 *                  table, DSA_DEV_BAD_PAGE for a page outside of the pool; such a
 *                  row is written as zeros
 *
 * Outputs that share memory with anything else: DSA_ERR_OVERLAP. */
DSA_API int dsa_latent_cache_read(const void* latent_cache, int64_t num_pages,
                                  const int32_t* block_table, const int32_t* starts,
                                  const int32_t* cu_rows, int32_t num_requests, int32_t max_pages,
                                  int32_t num_rows, void* ckv, int64_t ckv_row_bytes, void* kpe,
                                  int64_t kpe_row_bytes, uint32_t* status, void* stream);

/* Bytes of device workspace the two calls below need on this device, the same for
 * every call: a 256-byte header, two fp32 records of 32 rows per SM (19 MB) and the
 * call's list of row groups (9 MB).  Zero-fill it once (its status word); nothing
 * else in it carries over.  Calls that may overlap on the device need a workspace
 * each; threads may call with one workspace on one stream. */
DSA_API size_t dsa_latent_attention_workspace_bytes(void);

/* Attention over everything a request has in the latent cache in 8 bits: of single
 * tokens (decoding), or of the last rows of each request (chains of drafts, whose
 * own tokens are in the cache), each of which sees the tokens up to its own.
 *
 *   q_nope         [num_rows, num_heads, 512] bf16, contiguous
 *   q_pe           [num_rows, num_heads, 64] bf16, contiguous
 *   latent_cache   num_pages pages of DSA_LATENT_PAGE_BYTES
 *   seq_lens       [num_requests] int32: cached tokens, the rows' own among them
 *   block_table    [num_requests, max_pages] int32
 *   cu_rows        [num_requests + 1] int32: request r has the rows cu_rows[r] ..
 *                  cu_rows[r+1]-1; row j of n sees seq_lens[r] - n + 1 + j tokens.
 *                  Rows outside of [cu_rows[0], cu_rows[num_requests]) are left as
 *                  they are.  NULL: row r is request r's only one
 *   output         [num_rows, num_heads, 512] bf16; may be q_nope itself
 *   lse            [num_rows, num_heads] fp32, base-2 log-sum-exp of the scaled
 *                  logits; a row that sees nothing has -inf, output 0
 *
 * 1 <= num_heads <= 128; num_rows * num_heads <= 2^24, num_requests <= 65536 and
 * (num_rows * num_heads / 16 + num_requests) * (max_pages / 2 + 4) <= 2^30.  Tokens
 * that no row sees may hold anything; a visible one with NaN makes the output NaN.
 * Values of q_nope are exact from 2^-13 of their row's largest up, smaller ones to
 * 2^-21 of that; weights times scales to 2^-14 of each and 2^-28 of the row's largest.
 * Where scales of one request differ by 2^60 and more, tokens of the small ones may
 * count as zeros.
 * Outputs that share memory with anything else: DSA_ERR_OVERLAP.  Data-dependent
 * errors: lengths that do not fit the table (clamped), cu_rows that do not fit
 * (the request is left out; decreasing: the call writes no row): DSA_DEV_BAD_SEQ_LEN;
 * page ids outside the pool (their tokens are masked): DSA_DEV_BAD_PAGE. */
DSA_API int dsa_latent_attention_run(const void* q_nope, const void* q_pe, const void* latent_cache,
                                     int64_t num_pages, const int32_t* seq_lens,
                                     const int32_t* block_table, const int32_t* cu_rows,
                                     int32_t num_requests, int32_t num_rows, int32_t num_heads,
                                     int32_t max_pages, float sm_scale, void* output, float* lse,
                                     void* workspace, size_t workspace_bytes, void* stream);

/* The same over selected slots (as dsa_attention_run, of the cache in 8 bits).
 *
 *   sparse_indices [num_rows, topk] int32 slots, -1: none; topk <= 65536.  A slot
 *                  that is given twice counts twice.
 *
 * num_rows * ceil(num_heads / 16) <= 2^20.
 * Indices outside of [-1, num_pages * 64): DSA_DEV_BAD_INDEX, taken as -1. */
DSA_API int dsa_latent_sparse_attention_run(const void* q_nope, const void* q_pe,
                                            const void* latent_cache, int64_t num_pages,
                                            const int32_t* sparse_indices, int32_t num_rows,
                                            int32_t num_heads, int32_t topk, float sm_scale,
                                            void* output, float* lse, void* workspace,
                                            size_t workspace_bytes, void* stream);

/* Verifies drafted tokens against the target's probabilities, from given random
 * numbers, and draws the token that follows.  Request r has the rows
 * cu_drafts[r] .. cu_drafts[r+1]-1: its last certain token, then drafts, a tree by
 * their parents.  From row 0 on, the children of a row are looked at in their
 * order; child x is accepted with probability min(1, p'(x) / q(x)), p' being the
 * target's distribution after the row, from which each rejection takes q away:
 *   c = 0, R = 1;  accepted: u q(x) R < max(p(x) - c q(x), 0)
 *   rejected:      c += R, R = sum max(p - c q, 0)
 * The walk goes on at an accepted row.  Where it ends, the next token is the first
 * whose running sum of max(p - c q, 0) exceeds sample_u of the whole (of p, if the
 * whole is 0; -1 if that is 0 too, or if either holds NaN: q's counts once something
 * was rejected).  Probabilities are 0, of either sign, or more.  All in 64 bits.
 *
 *   target_probs   num_rows rows of vocab fp32, target_stride values apart: the
 *                  target's distribution after each row
 *   draft_probs    likewise: what the children of each row were drawn from; NULL:
 *                  q is 1 at the drafted token, a rejected x is struck out of p
 *   draft_tokens   [num_rows] int32 (row 0's is not read)
 *   parents        [num_rows] int32, in the request; below the row's own place
 *   cu_drafts      [num_requests + 1] int32
 *   accept_u       [num_rows] fp32, sample_u [num_requests] fp32, in [0, 1)
 *   path           [num_requests, path_width] int32: the accepted rows' places in
 *                  the request, then -1; the walk ends when it is full
 *   num_accepted   [num_requests] int32
 *   next_token     [num_requests] int32
 *   status         device word: DSA_DEV_BAD_SEQ_LEN for cu_drafts that do not fit (the
 *                  request is taken as empty) and requests of over 4096 rows (cut
 *                  off there), DSA_DEV_BAD_INDEX for tokens outside of the vocabulary
 *                  (never accepted)
 *
 * num_rows <= 2^24, num_requests <= 65536, vocab <= 2^28, path_width <= 65536.
 * Outputs that share memory with anything else: DSA_ERR_OVERLAP. */
DSA_API int dsa_verify_run(const float* target_probs, int64_t target_stride, const float* draft_probs,
                           int64_t draft_stride, const int32_t* draft_tokens, const int32_t* parents,
                           const int32_t* cu_drafts, const float* accept_u, const float* sample_u,
                           int32_t num_requests, int32_t num_rows, int32_t vocab, int32_t path_width,
                           int32_t* path, int32_t* num_accepted, int32_t* next_token,
                           uint32_t* status, void* stream);

/* Copies the sticky device status word of `workspace` to *status_out
 * (synchronising `stream`), and zeroes it when `clear` is non-zero.
 * No counterpart in the reference, which has no error channel
 * (errors there surface as Python exceptions, FAQ.md:238-240). */
DSA_API int dsa_read_device_status(void* workspace, uint32_t* status_out, int clear,
                           void* stream);

/* ---- test hook ---------------------------------------------------------
 * Arms one fault for the next call of the operator it names, made by any
 * thread of this process (the call consumes it).
 * DSA_TEST_SKIP_ARRIVAL, for the next dsa_attention_run: makes,
 * in every CTA, the producers of its second tile issue no copy and no
 * arrival for it, and every bounded wait of that launch gives up after
 * `wait_limit_ns` instead of 2 s.  The launch then ends with
 * DSA_DEV_WAIT_TIMEOUT set and its output void; every wait stays bounded and
 * the workspace's merge counters are left at zero, so the next call is
 * exact.  kind DSA_TEST_NONE disarms every armed fault.  For tests of the
 * failure path only; no counterpart in the reference. */
#define DSA_TEST_NONE         0
#define DSA_TEST_SKIP_ARRIVAL 1
/* DSA_TEST_SKIP_READY, for the next dsa_indexer_run (the no-allocation entry
 * point included): the score kernel publishes no ready count for request 0,
 * and the select's wait for a request's ready count gives up after
 * `wait_limit_ns` instead of 2 s.  The call ends with DSA_DEV_WAIT_TIMEOUT set
 * and row 0 written as all -1; the other rows are exact, and the select
 * resynchronises request 0's consumed count with its scored count, so the
 * next call is exact. */
#define DSA_TEST_SKIP_READY   2
DSA_API int dsa_b200_test_inject(int kind, uint64_t wait_limit_ns);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* DSA_B200_H_ */
