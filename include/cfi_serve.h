/*
 * cfi_serve.h -- operators for serving many sequences at once: a key-value cache in pages (f16, or
 * quantised to Q8_0 or Q4_1 as it is written), page tables and slots made on the device, the rows'
 * norm and rotation on their way into the cache, the attention of a batch's new tokens over it, the
 * attention of packed prompts of different lengths, and sampling.
 *
 * No counterpart in cuda-for-intel, whose host application keeps one contiguous f16 cache, masks
 * its prompts and samples on the CPU.  All pointers are device pointers unless said otherwise,
 * `stream` is a cudaStream_t, and each function returns 0 or a CUDA error code: cudaErrorInvalidValue,
 * before anything is launched, for arguments outside what is documented here.  Nothing is
 * allocated but per-stream scratch, which grows outside stream capture only (run the largest
 * call once before capturing).  A captured graph keeps the scratch of the stream that it was captured on: graphs that were captured on
 * one stream, and what else runs on that stream, do not run at the same time.  Lengths, page tables, slots and sampling settings are read from
 * device memory by the kernels: a captured graph can be replayed with new ones.
 *
 * Types are ggml's ids: 0 F32, 1 F16, 3 Q4_1, 8 Q8_0.
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
 *         16-byte pieces;
 *   Q4_1: page_size / 16 tiles of 16 positions, each 16 rows of head_dim/2 bytes of nibbles, then 16 rows
 *         of head_dim/32 f16 scales and head_dim/32 f16 minima -- ggml's Q4_1 values (blocks of 32,
 *         q * scale + minimum) in the order in which the attention reads them.  With b a block and the
 *         lower dim of two in a byte's lower nibble: a row of K is 4 groups, group c holding dims
 *         32 b + 8 c .. + 7 of each b in turn (4 bytes a block); a row of V is 8 groups, group g holding
 *         dims 32 b + 4 g .. + 3 of each b (2 bytes a block), and with head_dim 128 group g lies at
 *         place g ^ 4 in the rows 2, 3, 6, 7, 10, 11, 14 and 15 of a tile.
 * head_dim 64 or 128.  Which sequence owns which page is the caller's page table (cfi_paged_place
 * makes one on the device).
 */
typedef struct {
    void *k, *v;
    int type; /* 1 F16, 3 Q4_1 or 8 Q8_0 */
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
 * reads back as NaN, past f16 alone as NaN or infinities.
 * Q4_1, per 32 values: d = (max - min) / 15, q = (x - min) / d rounded to nearest, halves up (0 where d is 0), scale f16(d),
 * minimum f16(min): quotient and d are rounded from their exact values.  A block with an infinity or a NaN, or whose d or min
 * passes f16, reads back as NaN and touches no other block. */
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
 * K and V carry 22 bits, a query's values no bits below 2^-38 (Q4_1: 2^-30) of their head's largest and a weight (Q8_0 and
 * Q4_1: times its scale of V) none below 2^-39 of the largest (Q4_1: scales below 2^-15 count as that): the results are those of
 * 32-bit arithmetic on the cached values, as long as the scores are within the range of f32.  (Q4_1: of the scaled whole numbers and
 * the minima, which are summed apart; the minima of K meet the sums of a query's values over each block, of which 22 bits are kept.)
 * A NaN makes NaN of what the formula takes it into and of nothing else: in q its head's outputs, in a row of K within
 * the length those of its kv head's query heads, in V the same dims of them.  An infinity there makes of these NaN
 * or what the formula gives.  Bounds: n_seq 65535, and n_seq * n_kv_head * ceil(n_head / n_kv_head / 8) *
 * (max_pages * page_size + 80) below 2^35.
 */
CFI_API int cfi_paged_attention(const CfiPagedCache *cache, const void *q, int q_type, long long q_stride, void *out,
                                int out_type, long long out_stride, const int32_t *table, int max_pages,
                                const int32_t *lens, int n_seq, int n_head, float scale, void *stream);

/*
 * The rows of a stacked or separate product on their way into the attention: each head of q and k gets its
 * bias, a norm and the rotation, v its bias, in one pass.  Per token t and head, in 32 bits:
 *   x = row + bias;
 *   x = x / sqrt(mean(x^2) + eps) * norm        (q_norm and k_norm: head_dim weights each; NULL: no norm);
 *   for i < n_rot / 2: (x[i], x[i + n_rot/2]) turned by the angle
 *     pos[t] * freq_scale * freq_base^(-2 i / n_rot) / freq_factors[i]    (freq_factors NULL: ones);
 *   what lies at n_rot and behind is not turned.
 * The angle is formed modulo a turn in 64 bits and rounded once to 32.  With theta the pair's angle at position 1, up to 2^24 rad, it is
 * off, before its sine and cosine, by 1e-7 rad and |pos| * max(1, |theta|) * 2^-53 rad at most; with freq_factors, which are part of
 * theta, by 1e-7 rad and |pos| * max(1, |theta|) * 2^-45 rad.
 * q_out, k_out and v_out get the rows (F32 or F16); with `cache` the rows of k and v also go to its slots, as
 * cfi_paged_kv_store would put them there (from 32 bits).  A slot outside the pool stores nothing.
 * q: n_head heads, k and v: n_kv_head; in_type, q_out_type, kv_out_type 0 F32 or 1 F16; biases and norms F32;
 * [token][head][dim] with row strides in values, multiples of 8, heads contiguous, rows, biases and norms 16-byte aligned.
 * head_dim 64 or 128 (a cache's has to be the same, and its n_kv_head); n_rot a multiple of 8 up to head_dim, 0 for no rotation
 * (pos is not looked at then); eps >= 0, freq_base > 0, freq_scale finite, freq_factors not 0.
 * k, v, biases, norms, k_out, v_out and cache may be NULL each: k_out needs k, v_out needs v, the cache both and slots; k
 * without k_out and cache, or v without v_out and cache, is refused.  n_tokens times all heads below 2^31.  An output may be its
 * input in place, with the same type and stride.
 */
typedef struct {
    const void *q, *k, *v;
    const float *q_bias, *k_bias, *v_bias, *q_norm, *k_norm, *freq_factors;
    const int32_t *pos;
    void *q_out, *k_out, *v_out;
    const int64_t *slots;
    long long q_stride, k_stride, v_stride, q_out_stride, k_out_stride, v_out_stride;
    int n_tokens, n_head, n_kv_head, head_dim, n_rot, in_type, q_out_type, kv_out_type;
    float eps, freq_base, freq_scale;
} CfiNormRope;
CFI_API int cfi_norm_rope(const CfiNormRope *a, const CfiPagedCache *cache, void *stream);

/*
 * Page tables on the device.  Row r of `table` lists the pages of a sequence that holds cached[r] positions
 * (ceil(cached[r] / page_size) of them); free_pages[0 .. n_free[0]) is a stack of the pages that nobody has.  The
 * caller fills them once; the calls below keep them, on the device alone, so that a captured step goes on by itself.
 */
typedef struct {
    int32_t *table;      /* [n_rows][max_pages] */
    int32_t *cached;     /* [n_rows] */
    int32_t *free_pages; /* [n_pages], of which the first n_free[0] count */
    int32_t *n_free;     /* [1] */
    int n_rows, max_pages, page_size, n_pages; /* n_rows up to 65536; page_size a power of two, 16 to 256 */
} CfiPageTable;

/* What the calls write to status[0]. */
enum {
    CFI_PLACED = 0,
    CFI_PLACE_BAD_ROW = 1,  /* a row outside [0, n_rows), one that occurs twice, or a negative count */
    CFI_PLACE_TOO_LONG = 2, /* a sequence would not fit max_pages, or the batch's positions pass 2^31 */
    CFI_PLACE_NO_ROOM = 3,  /* more new tokens than max_new, or more positions than max_context */
    CFI_PLACE_NO_PAGES = 4  /* the stack holds less pages than are needed (cfi_paged_trim: more would be free than there are) */
};

/*
 * The batch's sequences rows[0 .. n_seq) get n_new[s] >= 0 tokens each behind what they hold.  The pages that this takes
 * come from the top of the stack, in the order of the batch and of the positions.  Written, for what the kernels of
 * a step or of packed prompts read:
 *   lens[s] and batch_table[s][0 .. pages): positions after the call and the pages that hold them (the rest of a row of
 *     max_pages is left as it is);
 *   cu_q, cu_kv (n_seq + 1): where each sequence's new tokens and positions begin among the packed ones;
 *   slots, positions (max_new): of each new token; behind the last one -1 and 0;
 *   context (max_context; may be NULL): the slots of all positions of all sequences; behind the last one -1;
 *   table, cached, n_free: the new state.
 * All or nothing: where the batch cannot be placed, status[0] says why (the least of the codes that apply), the state stays as it
 * was, lens, cu_q, cu_kv and positions are 0 and slots and context -1, so that a step captured behind the call stores nothing.
 * n_seq up to 8192; rows and n_new are read on the device.  Calls on one page table have to be ordered, as by one stream.
 */
typedef struct {
    const int32_t *rows, *n_new;
    int32_t *lens, *batch_table, *cu_q, *cu_kv, *positions, *status;
    int64_t *slots, *context;
    int n_seq, max_new, max_context;
} CfiPagedPlace;
CFI_API int cfi_paged_place(const CfiPageTable *t, const CfiPagedPlace *a, void *stream);

/* The sequences rows[0 .. n_seq) keep their first keep[s] positions (all, where they hold no more; none, where keep[s] is
 * negative), and the pages behind those go back to the stack: drafted tokens that were not taken, or, with 0, a sequence that is
 * done.  The last page of the last sequence goes first, so that what follows a cfi_paged_place of the same rows undoes it.  Rows of
 * the table are left as they are.  status as above; nothing is done where it is not 0. */
CFI_API int cfi_paged_trim(const CfiPageTable *t, const int32_t *rows, const int32_t *keep, int n_seq, int32_t *status, void *stream);

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
