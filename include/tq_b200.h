/*
 * libtq_b200 — C ABI of the TurboQuant hot paths for NVIDIA B200 (sm_100a).
 *
 * Conventions (the launcher style of the reference's native library,
 * turboquant/kernels/fp4_pa_v9.hip:177-197 as called from
 * turboquant/integration/tq_fp4_backend.py:274-295): C linkage, raw device
 * pointers, plain ints and floats, the stream last.  Unlike the reference's
 * `void` launchers every function returns a status: 0 on success, a negative
 * TQ_ERR_* otherwise.  Nothing here allocates, synchronises or keeps global
 * state unless its comment says so; the caller owns every buffer, including
 * the split-K workspace, so the calls can be captured in CUDA graphs.
 *
 * All tensors are contiguous in their last dimension; head_dim is 128.
 * "rotated space" means multiplied by the normalised 128x128 Walsh-Hadamard
 * matrix of turboquant/core/rotation.py:28-44.
 */
#ifndef TQ_B200_H_
#define TQ_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct CUstream_st* tq_stream_t; /* same type as cudaStream_t */

#define TQ_OK 0
#define TQ_ERR_ARG (-1)         /* null pointer, negative size, bad stride or alignment */
#define TQ_ERR_UNSUPPORTED (-2) /* bit width / block size / group size outside what is built */
#define TQ_ERR_LAUNCH (-3)      /* the CUDA runtime rejected the launch */
#define TQ_ERR_WORKSPACE (-4)   /* caller-provided workspace too small */

#define TQ_DTYPE_F16 0
#define TQ_DTYPE_BF16 1
#define TQ_DTYPE_F32 2

/* Flags that may be OR-ed into the io_dtype argument of tq_decode_paged / tq_decode_paged_static. */
#define TQ_IO_ROTATE_Q 0x100     /* q_rot is given in ORIGINAL space: the kernel rotates it (q' = q H) while loading;
                                    q_proj must be NULL */
#define TQ_IO_DEROTATE_OUT 0x200 /* write out in original space (out H), as the reference's rotate_output does */
#define TQ_IO_TCGEN05 0x400      /* run the tensor-memory (tcgen05) variant of the decode kernel where it exists: 2- and
                                    3-bit codebooks without Sparse-V; other formats ignore the flag.  Slower than the
                                    default kernel on this hardware.  The query heads of a group share one scale: held to
                                    3e-3 + 1.5e-2 |ref| for heads of like size; a head whose query is far smaller than
                                    another one's of its group loses precision. */

/* Bits set by kernels in the optional device-side status word. */
#define TQ_COMPRESS_TCGEN05 2 /* flag in tq_compress_paged's `prerotated` argument, see there */

#define TQ_STATUS_BAD_BLOCK 1 /* a block-table entry was outside [0, num_blocks) and was clamped */
#define TQ_STATUS_TIMEOUT 2   /* a bounded wait on an async copy ran out */
#define TQ_STATUS_BAD_SLOT 4  /* a slot index was >= num_blocks * block_size and was skipped */
#define TQ_STATUS_BAD_POSITION 8 /* a position was outside the rotary table and was clamped */
#define TQ_STATUS_NO_BLOCKS 16   /* a request got no slots: the free blocks were used up */
#define TQ_STATUS_TOO_LONG 32    /* a request's rows, blocks or queries exceed what the call's tensors hold; it was cut or left out */

/* Library version, (major << 16) | minor.  Host only. */
int tq_version(void);

/* Bytes of one 16-token page of the paged cache for a format, or a negative
 * status.  The cache tensor is uint8 [num_blocks, num_kv_heads,
 * block_size / 16 * page_bytes]; this replaces the fixed 68-byte slot of
 * TurboQuantFP4Backend.get_kv_cache_shape
 * (turboquant/integration/tq_fp4_backend.py:699-722).  Host only. */
int tq_page_bytes(int k_bits, int v_bits, int use_qjl);

/* KV compression into the paged cache: rotation (fast WHT, skipped when
 * `prerotated`), norm, Lloyd-Max bucketize, residual signs and norm (K only,
 * when use_qjl), bit-packing, scatter by slot.  One launch handles K and V.
 *
 * Replaces the cache-update step the reference does with torch ops,
 * turbo4_fp8_compress_and_scatter (turboquant/integration/vllm_backend.py:
 * 179-230) / TurboQuantFP4Impl.do_kv_cache_update
 * (turboquant/integration/tq_fp4_backend.py:456-484), with the arithmetic of
 * polarquant_compress (turboquant/core/quantizer.py:141-173) and the packed
 * fields of compress_k / compress_v (turboquant/kernels/packed_compress.py:
 * 157-177, 226-240).
 *
 * key, value: [n_tokens, n_kv_heads, 128] of in_dtype with element strides
 * (stride_token, stride_head); the 128 values of a head are contiguous and
 * 16-byte aligned.  slot_mapping: int64 [n_tokens]; negative slots are
 * clamped to 0 as the reference does (vllm_backend.py:224); slots beyond the
 * cache are skipped and flagged in *status.  centroids: fp32 [2^bits],
 * boundaries: fp32 [2^bits - 1], ascending, on the device.  status: optional
 * device int32, OR-ed with TQ_STATUS_* bits; may be NULL.
 *
 * The fast path (tensor-core rotation, table-driven bucketize) needs
 * neighbouring boundaries to be more than 1/64 apart - true of the Lloyd-Max
 * codebooks for 128 dims at 2, 3 and 4 bits; other codebooks are handled by a
 * slower generic path with the same results.  A vector that contains a NaN or
 * an infinity gets the indices of a zero vector and a non-finite norm.  The
 * first call on a device sets a function attribute (shared-memory size) and
 * should be made before any stream capture.
 *
 * prerotated: 0 = rotate here, 1 = the rows are already rotated; OR-ed with
 * TQ_COMPRESS_TCGEN05 the rotation of fp16 / bf16 rows of a large launch runs as
 * one 128 x 128 x 128 tcgen05 product per 128 rows with one thread per vector
 * afterwards (an opt-in variant: same results within the rotation allowance,
 * about 15 % slower than the default kernel on this hardware). */
int tq_compress_paged(const void* key, const void* value, int in_dtype,
                      int64_t k_stride_token, int64_t k_stride_head,
                      int64_t v_stride_token, int64_t v_stride_head,
                      void* cache, int64_t num_blocks, int block_size,
                      const int64_t* slot_mapping,
                      const float* k_centroids, const float* k_boundaries,
                      const float* v_centroids, const float* v_boundaries,
                      int n_tokens, int n_kv_heads, int k_bits, int v_bits,
                      int use_qjl, int prerotated, int32_t* status, tq_stream_t stream);

/* Pages of one (sequence, kv head) that a split-K chunk covers when the
 * caller passes chunk_pages = 0 to tq_decode_paged.  Host only. */
int tq_decode_auto_chunk_pages(int num_seqs, int num_kv_heads, int num_q_heads, int max_pages_per_seq);

/* Bytes of split-K workspace tq_decode_paged needs.  Host only. */
int64_t tq_decode_workspace_bytes(int num_seqs, int num_q_heads, int num_kv_heads,
                                  int max_pages_per_seq, int chunk_pages);

/* Bytes of workspace with which tq_decode_paged(chunk_pages = 0) runs the kernel that suits the shape best: at least
 * tq_decode_workspace_bytes(...), with which it runs the chunked kernel; 11 MB where the persistent kernel is the better
 * one.  The two kernels add in another order: with a workspace between the two sizes the last bits differ.  Host only. */
int64_t tq_decode_auto_workspace_bytes(int num_seqs, int num_q_heads, int num_kv_heads, int max_pages_per_seq);

/* Asymmetric packed paged decode attention with GQA and split-K, one query
 * token per sequence.  Replaces _tq_v12_sparse_v_kernel / _tq_v11_single_kernel
 * (turboquant/kernels/sparse_v.py:26-159, 164-261) and, for the score
 * estimator with the QJL sign term, _packed_attn_v7 + _splitk_reduce
 * (turboquant/kernels/packed_attention.py:76-227); it is called where the
 * reference calls launch_fp4_pa_v9 (turboquant/integration/tq_fp4_backend.py:
 * 274-295).
 *
 * out, q_rot, q_proj: [num_seqs, num_q_heads, 128] of io_dtype (fp16 or
 * bf16, optionally OR-ed with TQ_IO_ROTATE_Q / TQ_IO_DEROTATE_OUT to fuse the two
 * rotations of TurboQuantFP8State.rotate_query / rotate_output,
 * turboquant/integration/vllm_backend.py:158-176, into this call); q_rot is the query in rotated space, q_proj = S q_rot (pass q_rot,
 * or NULL, when S = I).  score = sm_scale * (k_norm <q_rot, c[k_idx]> +
 * corr_scale * k_rnorm <q_proj, signs>); out = softmax(score) applied to
 * v_norm * c_v[v_idx], in rotated space.  Query head h reads kv head
 * h / (num_q_heads / num_kv_heads).  sparse_thresh > 0 enables the Sparse-V
 * rule (a 16-token V page is not fetched when every softmax weight in it, for
 * every query head of the group, is <= sparse_thresh relative to the running
 * maximum); <= 0 disables it.  block_tables: int32 [num_seqs, bt_stride];
 * seq_lens: int32 [num_seqs].  workspace: 16-byte
 * aligned, this call's own until its kernels are done; tq_decode_auto_workspace_bytes(...)
 * bytes with chunk_pages = 0 (tq_decode_workspace_bytes(...) are enough, for the
 * chunked kernel), tq_decode_workspace_bytes(...) with a chunk_pages.  skip_stats:
 * optional device uint32[2] = {V pages visited, V pages skipped}, accumulated
 * with atomics when non-NULL.  Sequences of length 0 produce zeros. */
int tq_decode_paged(void* out, const void* q_rot, const void* q_proj, int io_dtype,
                    const void* cache, int64_t num_blocks, int block_size,
                    const int32_t* block_tables, int64_t bt_stride, const int32_t* seq_lens,
                    const float* k_centroids, const float* v_centroids,
                    float sm_scale, float corr_scale, float sparse_thresh,
                    void* workspace, int64_t workspace_bytes,
                    int32_t* status, uint32_t* skip_stats,
                    int num_seqs, int num_q_heads, int num_kv_heads, int max_pages_per_seq,
                    int k_bits, int v_bits, int use_qjl, int chunk_pages, tq_stream_t stream);

#define TQ_DECODE_STATIC_SCRATCH_BYTES (16 * 1024 * 1024)

/* tq_decode_paged for callers that cannot provide a workspace.  It has no
 * counterpart in the reference.  Meant for hosts that cannot allocate device
 * memory themselves: a server that gave all free HBM to its KV-cache pool at
 * start-up, so any later allocation fails, or a foreign-language binding that
 * only passes on pointers it received.  Same arguments as tq_decode_paged
 * without workspace / workspace_bytes; the split-K partials go to a fixed
 * 16 MiB array that is part of the library image (the chunked kernel runs, also
 * with chunk_pages = 0; every GPU that loads the
 * library holds those 16 MiB until the process exits).  Problems that need
 * more (tq_decode_workspace_bytes(...) > TQ_DECODE_STATIC_SCRATCH_BYTES)
 * are refused with TQ_ERR_WORKSPACE before anything is launched: pass a
 * larger chunk_pages or use tq_decode_paged.  The function calls no
 * allocation routine.  The first call on each device looks up the device
 * address of the array (cudaGetSymbolAddress) and remembers it; make that
 * first call during set-up, before any stream capture begins.  All calls on
 * a device share the one array, which keeps whatever the last call left in it
 * (nothing in it needs clearing: each call writes every partial it later
 * reads); two calls whose kernels overlap on the GPU, e.g. on different
 * streams, race on it and must be serialised by the caller. */
int tq_decode_paged_static(void* out, const void* q_rot, const void* q_proj, int io_dtype,
                           const void* cache, int64_t num_blocks, int block_size,
                           const int32_t* block_tables, int64_t bt_stride, const int32_t* seq_lens,
                           const float* k_centroids, const float* v_centroids,
                           float sm_scale, float corr_scale, float sparse_thresh,
                           int32_t* status, uint32_t* skip_stats,
                           int num_seqs, int num_q_heads, int num_kv_heads, int max_pages_per_seq,
                           int k_bits, int v_bits, int use_qjl, int chunk_pages, tq_stream_t stream);

/* Fast Walsh-Hadamard rotation of n rows of 128 values: out = scale * (in @ H).
 * Used for q' = q H before decode and out = o H after it, the two matmuls of
 * TurboQuantFP8State.rotate_query / rotate_output
 * (turboquant/integration/vllm_backend.py:158-176).  in and out may alias. */
int tq_wht_rows(const void* in, void* out, int dtype, int64_t n_rows, float scale, tq_stream_t stream);

/* Contiguous packed K compression, the output format of compress_k /
 * compress_k_permuted (turboquant/kernels/packed_compress.py:157-177,
 * 219-223): k_idx uint8 [n, 16*bits] (2-bit: 4 per byte LSB first; 4-bit: low
 * nibble first; 3-bit: little-endian bit stream as decoded at
 * turboquant/kernels/sparse_v.py:57-60), k_signs uint8 [n, 16] (sequential,
 * or in the stride-4 order of permute_signs_for_chunked,
 * packed_compress.py:180-216, when permute_signs), k_rnorm and k_norm fp16 [n].
 * Arithmetic as turboquant/core/quantizer.py:141-173.  More than 32768 rows
 * take the persistent table-driven kernel (as tq_compress_paged: on already
 * rotated rows the indices and signs are the reference's bit for bit, with
 * the rotation done here at most 1e-4 of the coordinates differ by one
 * centroid); smaller launches take the binary-search kernel. */
int tq_compress_k(const void* K, int in_dtype, int64_t n, const float* centroids, const float* boundaries,
                  int bits, int prerotated, int permute_signs,
                  uint8_t* k_idx, uint8_t* k_signs, void* k_rnorm, void* k_norm, tq_stream_t stream);

/* Contiguous packed V compression, compress_v (packed_compress.py:226-240):
 * v_idx uint8 [n, 16*bits], v_norm fp16 [n]. */
int tq_compress_v(const void* V, int in_dtype, int64_t n, const float* boundaries, int bits, int prerotated,
                  uint8_t* v_idx, void* v_norm, tq_stream_t stream);

/* polarquant_compress (turboquant/core/quantizer.py:111-183) with unpacked
 * outputs: indices int64 [n,128], norms fp32 [n], k_mse_rot fp32 [n,128] and,
 * when use_qjl, signs fp32 (+-1) [n,128] and rnorm fp32 [n]. */
int tq_polarquant_compress(const void* x, int in_dtype, int64_t n, const float* centroids,
                           const float* boundaries, int bits, int use_qjl, int prerotated,
                           int64_t* indices, float* norms, float* k_mse_rot, float* signs, float* rnorm,
                           tq_stream_t stream);

/* Bytes of workspace tq_packed_attention needs for a split count, 0 (which shares the steps of all rows) included.  With
 * num_splits = 0 and less than that, but enough for tq_packed_attention_auto_splits parts a row, it runs those.  Host only. */
int64_t tq_packed_attention_workspace_bytes(int BH, int num_splits);

/* About how many CTAs share a row when num_splits = 0; replaces the MI355X
 * tuning table of _get_config (packed_attention.py:236-267).  Host only. */
int tq_packed_attention_auto_splits(int BH, int Sk);

/* packed_attention (turboquant/kernels/packed_attention.py:290-344):
 * contiguous [BH, Sk, ...] packed K/V, one query row per BH, split-K partial
 * kernel plus merge.  Q, Q_proj fp16 [BH,128]; k_idx/v_idx uint8
 * [BH,Sk,16*bits]; k_signs_perm uint8 [BH,Sk,16] in stride-4 order; norms fp16
 * [BH,Sk]; centroids fp32 [2^bits]; out fp16 [BH,128] in rotated space.  Q, k_idx,
 * k_signs_perm, v_idx and workspace start on 16 bytes. */
int tq_packed_attention(const void* Q, const void* Q_proj, const uint8_t* k_idx, const uint8_t* k_signs_perm,
                        const void* k_rnorm, const void* k_norm, const uint8_t* v_idx, const void* v_norm,
                        const float* centroids, float corr_scale, int BH, int Sk, int bits, int num_splits,
                        void* workspace, int64_t workspace_bytes, void* out, tq_stream_t stream);

/* Rotary positions of query and key heads, out of place or in place (q_out = q,
 * k_out = k; other overlaps are not allowed).  q, q_out: [rows, num_q_heads,
 * head_dim], k, k_out: [rows, num_kv_heads, head_dim] of dtype; strides: 8
 * element strides, (row, head) of q, k, q_out, k_out.  Values 0 .. rotary_dim
 * of each head are turned, the rest copied: pairs (i, i + rotary_dim / 2), or
 * (2i, 2i + 1) when interleaved; inverse turns back (the gradient of the turn).
 * table: fp32 [table_rows, rotary_dim], cosines then sines of the
 * rotary_dim / 2 angles of a position; positions: int64 (wide_positions) or
 * int32 [rows], clamped to the table with TQ_STATUS_BAD_POSITION.  Interleaved
 * pairs start on their own size. */
int tq_rotary(const void* q, const void* k, void* q_out, void* k_out, int dtype, const int64_t* strides,
              const void* positions, int wide_positions, const float* table, int64_t table_rows, int64_t rows,
              int num_q_heads, int num_kv_heads, int head_dim, int rotary_dim, int interleaved, int inverse,
              int32_t* status, tq_stream_t stream);

/* Bytes of one 16-token page of the 8-bit cache: e4m3 codes of K [16][head_dim],
 * of V [16][head_dim], the fp32 scales of K and V, 24 unused bytes; negative
 * for a head_dim other than 64 and 128.  The cache is uint8 [num_blocks,
 * num_kv_heads, block_size / 16 * page_bytes], as the packed one.  Host only. */
int tq_cache8_page_bytes(int head_dim);

/* New K/V rows into the 8-bit cache.  A scale is 2^e with the smallest e >= -100
 * for which no finite value of the page's rows is above 448 * 2^e; a code is
 * the e4m3 value nearest to x / scale (ties to even; infinities saturate, a NaN
 * stays one).  A page whose first slot is among the rows is begun anew: its
 * scale comes from these rows alone.  Otherwise the page keeps the larger of
 * its scale and theirs, and the codes before them are rescaled when it grows
 * (exact, but for codes that become subnormal).  Codes behind the last row
 * written are left as they were.
 *
 * key, value: as in tq_compress_paged, with head_dim 64 or 128; rows, heads
 * and the cache start on 16 bytes.  slot_mapping: int64 [n_tokens]; negative
 * slots are skipped, slots beyond the cache are skipped and flagged.  Rows of
 * one page stand next to one another in ascending order, as sequences bring
 * them; if a call names a page in two places, or a slot twice, that page's
 * content is not specified. */
int tq_quantize8_paged(const void* key, const void* value, int in_dtype, int64_t k_stride_token, int64_t k_stride_head,
                       int64_t v_stride_token, int64_t v_stride_head, void* cache, int64_t num_blocks, int block_size,
                       const int64_t* slot_mapping, int64_t n_tokens, int n_kv_heads, int head_dim, int32_t* status,
                       tq_stream_t stream);

/* Bytes of workspace tq_attend8_paged needs.  Host only. */
int64_t tq_attend8_workspace_bytes(int64_t num_rows, int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                                   int max_queries, int max_pages_per_seq);

/* Attention over the 8-bit cache, causal at the end of each sequence.  out, q:
 * [num_rows, num_q_heads, head_dim] of io_dtype (fp16 or bf16), 16-byte aligned.
 * Rows query_start_loc[i] .. query_start_loc[i + 1] (int32 [num_seqs + 1],
 * ascending) are the last tokens of sequence i, whose seq_lens[i] tokens, these
 * included, are in the cache; query_start_loc = NULL: row i is sequence i's
 * only one.  Row j of n sees the first seq_lens[i] - n + j + 1 tokens; one that
 * sees none becomes zeros.  max_queries: at least the most rows of a sequence
 * (the ones beyond are left out and flagged, the others served as if they were
 * all).  Rows that are left out or that no sequence has - before the first one,
 * behind the last one - are left as they were, or become zeros when zero_rest.
 * block_tables,
 * bt_stride, seq_lens, max_pages_per_seq, workspace, status: as in
 * tq_decode_paged. */
int tq_attend8_paged(void* out, const void* q, int io_dtype, const void* cache, int64_t num_blocks, int block_size,
                     const int32_t* block_tables, int64_t bt_stride, const int32_t* seq_lens, const int32_t* query_start_loc,
                     float sm_scale, void* workspace, int64_t workspace_bytes, int32_t* status, int64_t num_rows,
                     int num_seqs, int num_q_heads, int num_kv_heads, int head_dim, int max_queries,
                     int max_pages_per_seq, int zero_rest, tq_stream_t stream);

/* Step tables from the requests' lengths.  Request i has context_lens[i] tokens
 * in the cache, in the first ceil(context / block_size) blocks of row i of
 * block_tables, and brings query_lens[i] new ones (negative counts as 0).  The
 * blocks it lacks come from the top of the stack free_blocks[0 ..
 * *free_count) in the order of the requests and are written into its row of
 * block_tables.  Out: slot_mapping and positions (int64 [num_rows]) of the new
 * tokens, request after request; seq_lens[i] = context + query;
 * query_start_loc (int32 [num_requests + 1]); *new_free_count, the height of the
 * stack afterwards.  free_blocks and *free_count are not changed, so that a
 * repeated call gives the same tables.  Rows behind the last request get slot
 * -1 and position 0.  A request for which the blocks do not suffice
 * (TQ_STATUS_NO_BLOCKS), or whose rows or blocks do not fit num_rows or
 * table_width (TQ_STATUS_TOO_LONG), takes none: its rows get slot -1, its
 * seq_lens entry stays the context.  No output may overlap an input. */
int tq_plan_step(const int32_t* query_lens, const int32_t* context_lens, int32_t* block_tables, int64_t bt_stride,
                 const int32_t* free_blocks, const int32_t* free_count, int64_t* slot_mapping, int64_t* positions,
                 int32_t* seq_lens, int32_t* query_start_loc, int32_t* new_free_count, int32_t* status,
                 int64_t num_requests, int64_t table_width, int64_t num_free, int block_size, int64_t num_rows,
                 tq_stream_t stream);

/* The blocks of the requests with ended[i] != 0 (the first ceil(context /
 * block_size) of their rows) go onto the stack, request after request:
 * free_blocks[*free_count ..); *new_free_count is its new height and
 * new_context_lens[i] 0 for them, context_lens[i] for the others.  *free_count
 * is not changed.  What exceeds the stack's num_free places is dropped and
 * flagged (TQ_STATUS_TOO_LONG). */
int tq_release_blocks(const uint8_t* ended, const int32_t* context_lens, const int32_t* block_tables, int64_t bt_stride,
                      int32_t* free_blocks, const int32_t* free_count, int32_t* new_context_lens, int32_t* new_free_count,
                      int32_t* status, int64_t num_requests, int64_t table_width, int64_t num_free, int block_size,
                      tq_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* TQ_B200_H_ */
