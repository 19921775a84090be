/*
 * dsa_chunk.h - C ABI of the operators on a chunk of new tokens in libdsa_mla.so:
 * norms of queries and keys with the position rotation (dsa_qk_norm_rope), the
 * write of latent rows and index keys into the paged caches (dsa_kv_append), and
 * dense attention of the chunk's tokens over the paged latent cache
 * (dsa_mla_chunk).  They fill and read the caches that dsa_mla_decode,
 * dsa_mla_prefill and dsa_indexer_scores use; where a context is no longer than
 * the top-k, every position is selected and dsa_mla_chunk takes the place of the
 * scorer, the selection and the sparse attention.
 *
 * The reference has none of them: its callers write the caches
 * (opus_attn/dsa_v32/README.md:99) and pass rotated queries.
 *
 * The chunk.  Sequence b of B brings tokens q_indptr[b] .. q_indptr[b + 1] - 1 of
 * the T rows of a call (q_indptr int32 [B + 1], ascending) and is seq_lens[b]
 * long with them: with n_b = q_indptr[b + 1] - q_indptr[b], token t is position
 *     p = seq_lens[b] - n_b + (t - q_indptr[b]).
 * Rows before q_indptr[0] or from q_indptr[B] on belong to no sequence: nothing
 * is computed or written for them, so a batch may be padded.  A sequence may bring no token.
 *
 * Pages.  Position p of sequence b lies in cache row
 *     block_table[b * block_table_stride + p / block_size] * block_size
 *         + p % block_size                        (block_table != NULL)
 *     b * kv_batch_stride + p                     (block_table == NULL)
 * if 0 <= p < table_blocks * block_size (paged) or, with kv_batch_stride > 0,
 * p < kv_batch_stride (flat), and if that row lies inside the cache.  A position
 * without a row is neither read nor written.
 *
 * Conventions (pointers, strides in elements, streams, errors) as in dsa_mla.h.
 * No entry allocates or synchronises, all may be captured into a graph, and
 * calls on distinct streams may run at once if they do not write the same rows
 * or share a workspace.  All sums are fp32 and every output is rounded once.
 */
#ifndef DSA_CHUNK_H_
#define DSA_CHUNK_H_

#include <stddef.h>
#include <stdint.h>

#include "dsa_mla.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
    DSA_NORM_NONE = 0,
    DSA_NORM_RMS = 1,          /* x / sqrt(mean(x^2) + eps) */
    DSA_NORM_LAYER = 2         /* (x - mean(x)) / sqrt(var(x) + eps) */
} dsa_norm;

typedef enum {
    DSA_ROPE_NONE = 0,
    DSA_ROPE_INTERLEAVED = 1,  /* pair i of the 64 rotated values: (2 i, 2 i + 1) */
    DSA_ROPE_HALVES = 2        /* pair i: (i, i + 32) */
} dsa_rope;

/* Rows of a stream: bf16 x [T, H, D] and out [T, H, D], last dim dense.  out may
 * be x itself (same pointer and strides).  Rows of out that overlap one another, x
 * otherwise, or the other stream's x or out are refused (DSA_ERR_BAD_STRIDE), and so
 * are two that lie among one another with different strides: slices of one buffer
 * need the same stride_t and, with several heads each that take turns, stride_h.
 * weight and bias (fp32 [norm_dim]; either may be NULL) follow the norm; they
 * must be NULL without one.  H == 0: no such stream. */
typedef struct {
    const void* x;
    int64_t stride_t, stride_h;
    void* out;
    int64_t out_stride_t, out_stride_h;
    const float* weight;
    const float* bias;
    int32_t H;
    int32_t norm;              /* dsa_norm */
} dsa_norm_rope_rows;

/*
 * Norms of queries and keys for each head, with the position rotation in the
 * same pass.  Each row's values 0 .. norm_dim - 1 go through its stream's norm,
 * then values rot_off .. rot_off + 63 are rotated by the row's position:
 *     (a, b) -> (a cos_i - b sin_i, b cos_i + a sin_i)   for pair i < 32,
 * sin negated when inverse != 0 (an attention output whose values carry the
 * rotation is turned back this way).
 * cos_sin  : fp32 [n_pos, 64] dense, row p = 32 cosines then 32 sines.  A token
 *            whose position lies outside [0, n_pos) gets NaN rotated values.
 * positions: int32 [T]; NULL: the chunk's (q_indptr, seq_lens, B), rows of no
 *            sequence then being left as they were.
 * D        : 128 (index vectors), 512 (V4 rows) or 576 (latent rows)
 * norm_dim : a multiple of 8, 8 .. min(D, 512)
 * rot_off  : a multiple of 64, 0 .. D - 64
 * Alignment: x, out, cos_sin, weight and bias 16 bytes, strides multiples of 8.
 * Limit: T x (ceil(q.H / g) + ceil(k.H / g)) at most 2^26 - 4, with g = 16 for
 * D = 128, else 8.
 */
typedef struct {
    dsa_norm_rope_rows q, k;
    const float* cos_sin;      /* may be NULL with DSA_ROPE_NONE */
    int64_t n_pos;
    const int32_t* positions;
    const int32_t* q_indptr;
    const int32_t* seq_lens;
    int32_t T, B;
    int32_t D, norm_dim, rot_off;
    int32_t rope;              /* dsa_rope */
    int32_t inverse;
    float eps;
} dsa_qk_norm_rope_args;

int dsa_qk_norm_rope(const dsa_qk_norm_rope_args* args, void* stream);

/*
 * Append a chunk's latent rows and index keys to their paged caches.
 * kv       : bf16 [T, 576] (DSA_KV_BF16, DSA_KV_FP8_656, DSA_KV_MXFP8) or
 *            [T, 512] (DSA_KV_BF16_D512, DSA_KV_MXFP8_V4); NULL: no latent rows.
 *            norm (NONE or RMS, weight fp32 [512] or NULL) covers values 0..511,
 *            then the last 64 values are rotated (rope) by the token's position.
 * cache    : the rows of kv_format, cache_rows of them:
 *            DSA_KV_BF16, DSA_KV_BF16_D512: bf16 rows
 *            DSA_KV_FP8_656: 656-byte rows, scale = amax / 448 per 128 values
 *              (IEEE division), code = e4m3fn(x / scale) as dsa_kv_quantize_fp8
 *              gives them (with no norm and no rotation: the same bytes)
 *            DSA_KV_MXFP8: cache = 512 codes, cache_scale = 16 E8M0 bytes,
 *              cache_rope = 64 bf16 values
 *            DSA_KV_MXFP8_V4: cache = 448 codes, then 14 E8M0 bytes (the row's
 *              other bytes stay as they were), cache_rope = 64 bf16 values
 *            E8M0: per 32 values the least power of two 2^e >= amax / 448, e at
 *            least -126 (e = 0 for 32 zeros), byte e + 127.
 *            A NaN value becomes a NaN code in every format, also where its group
 *            holds nothing else (scale 0, or E8M0 127).  Row strides in elements of
 *            each stream (bytes for codes and scales); 0 = dense.
 * index_k  : bf16 [T, 128]; NULL: no index keys.  index_norm over all 128
 *            values, then the first 64 rotated (index_rope), written as bf16 to
 *            the token's row of index_cache (the same row number).
 * cos_sin  : as in dsa_qk_norm_rope.  The rotated values of a token at or past
 *            n_pos are NaN.
 * T, with index keys T + ceil(T / 4), is at most 2^26 - 4.
 * A call must not name one cache row twice.  Flat caches of several sequences
 * need kv_batch_stride > 0.
 * Alignment: 16 bytes for pointers to rows, cos_sin, weights and biases; bf16
 * strides multiples of 8, byte strides of 16.
 */
typedef struct {
    const void* kv;
    int64_t kv_stride_t;
    const float* weight;
    void* cache;
    void* cache_scale;
    void* cache_rope;
    int64_t cache_rows;
    int64_t stride_row, scale_stride_row, rope_stride_row;   /* 0 = dense */
    int32_t kv_format;
    int32_t norm, rope;

    int32_t index_norm, index_rope;
    const void* index_k;
    int64_t index_stride_t;
    const float* index_weight;
    const float* index_bias;
    void* index_cache;
    int64_t index_rows, index_stride_row;                    /* 0 = dense */

    const float* cos_sin;
    int64_t n_pos;
    const int32_t* q_indptr;
    const int32_t* seq_lens;
    const int32_t* block_table;
    int64_t block_table_stride;
    int32_t table_blocks, block_size;
    int64_t kv_batch_stride;
    int32_t T, B;
    float eps, index_eps;
} dsa_kv_append_args;

int dsa_kv_append(const dsa_kv_append_args* args, void* stream);

/*
 * Dense attention of a chunk's tokens over the paged latent cache.
 *     s_j = (q[t, h] . k_j) * sm_scale
 *     O   = sum_j exp(s_j) k_j[0:512] / sum_j exp(s_j),  LSE = ln sum_j exp(s_j)
 * over the positions j of the token's sequence with a row in the cache,
 * 0 <= j < seq_lens[b] and, when causal != 0, j <= p (the token's own position).
 * A token with none gets O = 0 and LSE = +inf.  A NaN or infinity in a row reaches
 * the tokens that attend it and no others.  sm_scale must be positive and finite.
 * q        : bf16 [T, H, 576] addressed by q_stride_{t,h}
 * kv_cache : kv_format DSA_KV_BF16 or DSA_KV_FP8_656, rows kv_stride_row
 *            elements apart (0 = dense), kv_total_rows below 2^31
 * out      : bf16 [T, H, 512] addressed by o_stride_{t,h}
 * lse      : fp32 [T, H] dense (may be NULL)
 * max_kv_len: an upper bound of seq_lens (the host cannot read them; it sizes
 *            the split).  A token of a longer sequence is not cut silently: its
 *            O and LSE are NaN.
 * num_splits: 0 = automatic, or 1 .. DSA_MLA_MAX_SPLITS parts of max_kv_len
 *            positions (rounded up to whole tiles of 32), whose fp32 partials
 *            (workspace: num_splits x T x H x 513 floats and 16 bytes) a combine
 *            merges.  Automatic: whether to split by the call's sizes, and up to
 *            64 sequences the size of a split by their lengths, on the device
 *            (dsa_mla_chunk_num_splits: the most that one sequence has).  Of more
 *            sequences a split is an even part of max_kv_len, which should then be
 *            near their lengths: with a bound far above them most parts are empty.
 * Scores and sums are fp32.  Probabilities are rounded to 16 bits for the
 * product with V (bf16; fp16 for DSA_KV_FP8_656, where those below fp16's normal
 * range are off by at most 2^-10 of the largest |V| together, up to 2^28 positions
 * a split).  656-byte rows: scores use
 * their exact values; V is rounded to fp16 (its scale's mantissa first), and
 * every scale must lie in [0, 128), a token that attends a row with another
 * scale getting NaN, as in dsa_mla.h.
 * Limits: T x H + 32 B at most 2^29 - 32 (split calls: T x H at most 2^26 - 4),
 * kv_total_rows and block_size x table_blocks below 2^31, max_kv_len at most
 * DSA_MLA_MAX_LIST; beyond them DSA_ERR_BAD_SHAPE.
 * Alignment: q and kv_cache 16 bytes, out 8; q's strides multiples of 8, out's of
 * 4, cache rows of 16 bytes and below 4 GiB.  Rows of out that overlap one another
 * are refused (DSA_ERR_BAD_STRIDE); out must not overlap the cache, q, or lse.
 * The split and so the last bits depend on the call's sizes and, with
 * num_splits = 0, on the lengths of all its sequences; one call repeats its bits.
 */
typedef struct {
    const void* q;
    int64_t q_stride_t, q_stride_h;
    const int32_t* q_indptr;
    const int32_t* seq_lens;
    const void* kv_cache;
    int64_t kv_total_rows;
    int64_t kv_stride_row;       /* 0 = dense rows */
    int32_t kv_format;
    int32_t block_size;
    const int32_t* block_table;
    int64_t block_table_stride;
    int64_t kv_batch_stride;
    void* out;
    int64_t o_stride_t, o_stride_h;
    float* lse;
    int32_t table_blocks;
    int32_t T, B, H;
    int32_t causal;
    int32_t max_kv_len;
    int32_t num_splits;          /* 0 = automatic */
    float sm_scale;
} dsa_mla_chunk_args;

/* Workspace bytes dsa_mla_chunk needs (0 when it runs unsplit), and its split count. */
int dsa_mla_chunk_workspace_size(const dsa_mla_chunk_args* args, size_t* bytes);
int dsa_mla_chunk_num_splits(const dsa_mla_chunk_args* args, int32_t* num_splits);
int dsa_mla_chunk(const dsa_mla_chunk_args* args, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DSA_CHUNK_H_ */
