/*
 * cfi_serve.h -- operators for serving many sequences at once: a key-value cache in pages (f16 or
 * quantised to Q8_0 as it is written), the attention of a batch's new tokens over it, the attention
 * of packed prompts of different lengths, and sampling.
 *
 * No counterpart in cuda-for-intel, whose host application keeps one contiguous f16 cache, masks
 * its prompts and samples on the CPU.  All pointers are device pointers unless said otherwise,
 * `stream` is a cudaStream_t, and each function returns 0 or a CUDA error code: cudaErrorInvalidValue,
 * before anything is launched, for arguments outside what is documented here.  Nothing is
 * allocated but per-stream scratch, which grows outside stream capture only (run the largest
 * call once before capturing).  Lengths, page tables, slots and sampling settings are read from
 * device memory by the kernels: a captured graph can be replayed with new ones.
 *
 * Types are ggml's ids: 0 F32, 1 F16, 8 Q8_0.
 */
#ifndef CFI_SERVE_H
#define CFI_SERVE_H
#include <stddef.h>
#include <stdint.h>

#ifndef CFI_API
#define CFI_API __attribute__((visibility("default")))
#endif

#ifdef __cplusplus
extern "C" {
#endif

/*
 * A paged cache: two pools (K and V) of n_pages pages, 16-byte aligned.  A page holds page_size
 * positions (a power of two, 16 to 256) of every kv head; slot s is position s % page_size of page
 * s / page_size.  A pool is [page][kv head][region], one region being
 *   F16:  page_size x head_dim f16;
 *   Q8_0: page_size x head_dim int8, then page_size x head_dim/32 f16 scales -- ggml's Q8_0 values
 *         (blocks of 32, q * scale) with quants and scales apart, so that both are read in
 *         16-byte pieces.
 * head_dim 64 or 128.  Which sequence owns which page is the caller's page table.
 */
typedef struct {
    void *k, *v;
    int type; /* 1 F16 or 8 Q8_0 */
    int n_pages, page_size, n_kv_head, head_dim;
} CfiPagedCache;

/* Bytes of one page of one pool; 0 for a description outside the above (k and v are not looked at). */
CFI_API size_t cfi_paged_page_bytes(const CfiPagedCache *cache);

/* Row t of k and v ([token][kv head][dim], src_type 0 F32 or 1 F16, row strides in values, a
 * multiple of 8, heads contiguous, 16-byte aligned) is written to slot slots[t], for all kv heads.
 * A slot outside [0, n_pages * page_size) stores nothing.  Two rows with the same slot: which one
 * remains is undefined.
 * Q8_0, per 32 values: d = max|x| / 127, q = x * (1/d) rounded to nearest even, scale f16(d); a block
 * with an infinity or a NaN, or whose d passes f16 (8.3e6 and more), has no finite scale and touches no other block: it
 * reads back as NaN, past f16 alone as NaN or infinities. */
CFI_API int cfi_paged_kv_store(const CfiPagedCache *cache, const void *k, const void *v, int src_type,
                               long long k_stride, long long v_stride, const int64_t *slots, int n_tokens, void *stream);

/* The reverse: row t of k and v ([token][kv head][dim] f16, row strides as above) = slot slots[t],
 * dequantised; zeros where the slot is outside the pool.  Reading a context back gives
 * cfi_packed_attention its earlier keys. */
CFI_API int cfi_paged_kv_load(const CfiPagedCache *cache, const int64_t *slots, void *k, void *v, long long k_stride,
                              long long v_stride, int n_tokens, void *stream);

/*
 * Attention of one new token for each of n_seq sequences over its pages: for query head h of
 * sequence s, with kv head h / (n_head / n_kv_head),
 *   out[s][h] = sum_{j < lens[s]} softmax_j(scale * q[s][h] . K[j]) V[j],
 * position j being slot table[s * max_pages + j / page_size] * page_size + j % page_size.  lens[s]
 * (the new token's own row, stored before, included) is cut to max_pages * page_size; a length of
 * zero or less gives zeros.  A page id outside the pool is read as the nearest page inside.  What
 * lies in a page past the length never matters, whatever it holds.
 * q and out: [sequence][head][dim], types 0 F32 or 1 F16, row strides in values (q's a multiple of
 * 8), 16-byte aligned; scale > 0.  Sums and maxima are in 32 bits and the operands of the products with
 * K and V carry 22 bits, a query's values no bits below 2^-38 of their head's largest and a weight (Q8_0: times its
 * scale of V) none below 2^-39 of the largest: the results are those of 32-bit arithmetic on the cached values, as
 * long as the scores are within the range of f32.
 * A NaN makes NaN of what the formula takes it into and of nothing else: in q its head's outputs, in a row of K within
 * the length those of its kv head's query heads, in V the same dims of them.  An infinity there makes of these NaN
 * or what the formula gives.  Bounds: n_seq 65535, and n_seq * n_kv_head * ceil(n_head / n_kv_head / 8) *
 * (max_pages * page_size + 80) below 2^35.
 */
CFI_API int cfi_paged_attention(const CfiPagedCache *cache, const void *q, int q_type, long long q_stride, void *out,
                                int out_type, long long out_stride, const int32_t *table, int max_pages,
                                const int32_t *lens, int n_seq, int n_head, float scale, void *stream);

/*
 * Attention of packed sequences: sequence s has the queries cu_q[s] .. cu_q[s+1] and the keys
 * cu_kv[s] .. cu_kv[s+1] (device arrays of n_seq + 1, ascending from 0, ends at most n_q and n_kv;
 * a query range that leaves [0, n_q) or a key range that leaves [0, n_kv) is cut to it).
 * causal: the last query sees all keys, query i of nq the keys j <= i + (nk - nq) -- with nk > nq
 * the first keys are an earlier context; a query that sees no key gives zeros.  causal 0: every
 * query sees all the sequence's keys.  Rows of out past cu_q[n_seq] are left as they are.
 * q, out: [token][head][dim], k, v: [token][kv head][dim]; q, k, v f16, out F32 or F16; row strides
 * in values, multiples of 8, heads contiguous, 16-byte aligned; n_head / n_kv_head at most 128;
 * head_dim 64 or 128; scale > 0.  Products are of f16 values (the softmax weights rounded to f16 too) with
 * 32-bit sums.  What a key holds that a query does not see never matters to it, whatever it is; a NaN or an infinity in V reaches
 * the same dims of the queries that see it (and costs their tiles a slow second pass).
 */
typedef struct {
    const void *q, *k, *v;
    void *out;
    const int32_t *cu_q, *cu_kv;
    long long q_stride, k_stride, v_stride, out_stride;
    int n_seq, n_q, n_kv, n_head, n_kv_head, head_dim, out_type, causal;
    float scale;
} CfiPackedAttention;
CFI_API int cfi_packed_attention(const CfiPackedAttention *a, void *stream);

/*
 * One token for each of n_rows rows of n_vocab logits (row stride in values), from the uniform
 * number u[row] in [0, 1).  In order:
 *   z = logit / temperature[row] (of any size: where the largest passes f32, it and its equals have all the weight);
 *     temperature <= 0 takes the largest logit;
 *   top_k[row] > 0 keeps the top_k largest;
 *   top_p[row] < 1 keeps, of those in falling order, the shortest run whose weight reaches top_p of
 *     theirs (a token stays when the weight before it is less);
 *   min_p[row] > 0 keeps what has at least min_p times the largest's weight.
 * The largest always stays; among equal logits the lower index comes first.  token[row] is the
 * first kept index, in index order, whose running weight exceeds u times the kept weight.  A weight is
 * exp(z - max), cut to a whole multiple of 2^-40: the sums are of whole numbers, so that the
 * token does not depend on the order of summation, the batch or the launch.
 * temperature, top_k, top_p, min_p may each be NULL: 1, off, off, off.  logprob (may be NULL): the
 * log of the token's share of the kept weight.  -inf and NaN logits are never taken (+inf is the
 * largest); a row of nothing else gives token -1 and logprob -inf.  n_vocab at most 400000.
 */
CFI_API int cfi_sample(const float *logits, long long row_stride, int n_rows, int n_vocab, const float *temperature,
                       const int32_t *top_k, const float *top_p, const float *min_p, const float *u, int32_t *token,
                       float *logprob, void *stream);

#ifdef __cplusplus
}
#endif
#endif
