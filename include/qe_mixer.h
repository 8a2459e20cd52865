/* qe_mixer.h -- C ABI of the token mixers beside the MoE block (qe_moe.h), on MI355X (gfx950).
 *
 * A layer of the model is a token mixer and then the MoE block.  This header
 * holds the mixers' cores, without the projections around them:
 *   qe_attn_*   rotary positions, a paged key-value cache, and causal
 *               attention over it, of packed prompts and of single tokens
 *               (the place of rope_kv, attn_block and the decode attention,
 *               engine/qe.cpp:1406-1453, :1873-1954, :2313-2465, and of
 *               flash_prefill, :438-678);
 *   qe_delta_*  the gated delta rule, of packed prompts and of single tokens
 *               (the place of dn_recurrent, engine/qe.cpp:1328-1405, and of
 *               decode's delta step, :2272-2312).
 *
 * Conventions, as in qe_moe.h: plain pointers and sizes, tensors in device
 * memory of the context's device, `stream` a hipStream_t of that device (NULL
 * = its default stream).  Calls enqueue work on `stream`, allocate nothing and
 * return without a host sync; they can be captured into a HIP graph.  A call
 * that would take more threads than a launch has (2^32) is refused.  A
 * context is used by one host thread at a time, and calls on one context that
 * could overlap (other streams, two graphs replayed at once) race on its
 * scratch, and may leave it unusable: give each its own context.  Entry points return 0 or a negative
 * QE_ERR_* code (qe_moe.h), and qe_moe_last_error() describes the calling
 * thread's last failure.  The calling thread's current device is left as it
 * was.  What a call writes may overlap what else it uses only where that is
 * said below.
 *
 * What stands in device memory (lengths, page tables, slots) is checked by the
 * kernels: a bad value makes no access out of bounds, its sequence's outputs
 * are zeros (with offsets outside the call's tokens those rows that are the
 * call's; qe_attn_append leaves the token out: nothing of it is written),
 * and the context remembers it.  The next call on the context
 * that looks returns QE_ERR_STATE for it, once, without doing its own work:
 * every entry point looks at entry without synchronising, qe_attn_check and
 * qe_delta_check after synchronising `stream`.
 */
#ifndef QE_MIXER_H
#define QE_MIXER_H
#include "qe_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of activations and caches. */
#define QE_F32 0
#define QE_F16 1
#define QE_BF16 2

/* ---- attention over a paged key-value cache ------------------------------ */

#define QE_ATTN_GROUP_MAX 16 /* query heads per key-value head */

typedef struct {
    int q_heads, kv_heads; /* query head h reads key-value head h / (q_heads / kv_heads); at most QE_ATTN_GROUP_MAX share one */
    int head_dim;          /* 64, 128 or 256 */
    int page;              /* positions of a page: 16, 32, 64, 128 or 256 */
    int type;              /* QE_F16 or QE_BF16: of the cache, of attention's q and out */
    float scale;           /* of the scores, > 0; 0 = 1 / sqrt(head_dim) */
    int rotary;            /* leading elements of a head that rotate: a multiple of 16, at most head_dim, 0 = none */
    double theta;          /* base of the rotation: pair i turns by position * theta^(-2 i / rotary); > 1 if rotary > 0 */
    int sections[3];       /* rotated pairs of each axis (time, height, width), together rotary / 2; one axis: {rotary / 2, 0, 0} */
    int interleaved;       /* 0: the axes' pairs stand one axis after the other.  1: they take turns: pair i is the height's
                              if i % 3 == 1 and i < 3 sections[1], the width's if i % 3 == 2 and i < 3 sections[2],
                              else the time's (of rotary / 2 pairs in all; sections[1] and [2] must fit) */
} qe_attn_desc;

typedef struct qe_attn_ctx qe_attn_ctx;

/* Create a context on `device`: scratch of a fixed size (35, 68 or 135 MB with
 * heads of 64, 128 or 256) for the partial results of calls that split a
 * sequence's length; half of it is for prompts over an 8-bit cache alone. */
int qe_attn_create(int device, const qe_attn_desc *desc, qe_attn_ctx **out);
int qe_attn_destroy(qe_attn_ctx *ctx);

/* A cache is two arrays of `n_pages` pages in device memory, k and v, each page
 * [kv_heads][page][head_dim] of the context's type, 16-byte aligned.  Position
 * p of a sequence is row p % page of the page that its table row names at
 * p / page.  Rows at and behind a sequence's kv_len are never used, whatever
 * they hold. */
typedef struct {
    void *k, *v;
    int64_t n_pages; /* 1 .. 2^31 - 1 */
} qe_kv_cache;

/* The sequences of a call.  cu_q, kv_len and table are device memory, read when
 * the work runs.  Sequence i's new tokens are rows cu_q[i] .. cu_q[i+1] - 1 of
 * q, k, v and out (0 <= cu_q[0] <= ... <= cu_q[n_seqs] <= n_tokens); they are
 * the last of its kv_len[i] positions.  kv_len counts them.  Rows of out that
 * belong to no sequence are left as they were.  Where offsets fall, which is
 * reported, qe_attn_prompt's rows may hold anything, and qe_attn_append leaves
 * out the tokens of the sequences beside them. */
typedef struct {
    int n_seqs;            /* 1 .. 65535 */
    int n_tokens;          /* rows given; 0 .. 2^24 - 1 */
    const int32_t *cu_q;   /* [n_seqs + 1]; NULL: one token per sequence (n_tokens == n_seqs) */
    const int32_t *kv_len; /* [n_seqs], each 0 .. max_pages * page */
    const int32_t *table;  /* page ids, sequence i's at table + i * table_stride */
    int table_stride;      /* >= max_pages */
    int max_pages;         /* columns of the table, >= 1; max_pages * page <= 2^30 */
    int max_len;           /* the longest kv_len as far as the host knows, for choosing how a call is split (results do
                              not depend on it but for rounding); 0 = max_pages * page */
} qe_attn_batch;

/* Rotary positions and cache write: q's rows rotated into q_out, k's rows
 * rotated and v's as they are into the cache at their positions.  q, k and v are
 * of in_type (QE_F32 or the context's type), token t's heads at base + t *
 * stride elements, contiguous; q_out is of the context's type.  pos: int32
 * [n_axes][n_tokens], n_axes = 3 if sections name more than one axis, else 1;
 * NULL = the position in the sequence, on every axis.  Angles are computed in
 * 64 bits.  q and q_out may both be NULL (keys and values only); q_out may be q
 * if in_type is the context's type and the strides are equal.  Pointers are
 * 16-byte aligned and strides multiples of 16 bytes.  A token before its
 * sequence's first position (cu_q gives more tokens than kv_len) writes nothing
 * to the cache; its q is rotated by pos or by its negative position.  A row of a
 * page that two tokens of the call write may hold parts of both. */
int qe_attn_append(qe_attn_ctx *ctx, const qe_attn_batch *batch, const qe_kv_cache *cache, int in_type, const void *q,
                   int64_t q_stride, const void *k, int64_t k_stride, const void *v, int64_t v_stride, const int32_t *pos,
                   void *q_out, int64_t q_out_stride, void *stream);

/* Causal attention of a call's packed prompts (batch->cu_q is not NULL): out =
 * softmax(scale q K^T) V for each row, over the positions of its sequence up
 * to its own.  A row with none (cu_q gives more tokens than kv_len) is zeros.  q and out are of the context's type, strides
 * in elements, 16-byte aligned; out may be q (equal strides).  Scores, softmax
 * and sums are in 32 bits; probabilities are rounded to the context's type for
 * the product with V (fp16: below 2^-21 of a row's greatest, 2^-29 for single
 * tokens, to fixed steps).  A V element that is infinite or NaN reaches the rows
 * that attend to its position, and no others.  The last sequence's last rows are
 * started first: a packed call is fastest with its longest sequences last. */
int qe_attn_prompt(qe_attn_ctx *ctx, const qe_attn_batch *batch, const qe_kv_cache *cache, const void *q, int64_t q_stride,
                   void *out, int64_t out_stride, void *stream);

/* The same for one new token per sequence: batch->cu_q is NULL.  A long
 * sequence's length is split over workgroups and their results joined. */
int qe_attn_decode(qe_attn_ctx *ctx, const qe_attn_batch *batch, const qe_kv_cache *cache, const void *q, int64_t q_stride,
                   void *out, int64_t out_stride, void *stream);

/* ---- norms with the rotation, and an 8-bit cache ---------------------------- */

/* Norms of q's and k's heads before the rotation: x <- x / sqrt(mean(x^2) +
 * eps) * weight, in 32 bits.  Weights are device memory, fp32 [head_dim],
 * 16-byte aligned, the same for all heads; NULL: q (or k) is not normed.
 * eps is 1e-30 or more.  A head whose squares sum beyond the range of 32 bits is NaN. */
typedef struct {
    const float *q_weight, *k_weight;
    float eps;
} qe_attn_norm;

/* qe_attn_append with norms: q and k are normed and then rotated, v is as it is. */
int qe_attn_append_normed(qe_attn_ctx *ctx, const qe_attn_batch *batch, const qe_kv_cache *cache, const qe_attn_norm *norm, int in_type,
                          const void *q, int64_t q_stride, const void *k, int64_t k_stride, const void *v, int64_t v_stride,
                          const int32_t *pos, void *q_out, int64_t q_out_stride, void *stream);

/* Element types of an 8-bit cache: integers -127 .. 127, and floating point of
 * 4 exponent bits (bias 7) and 3 more (448 is the greatest, no infinities). */
#define QE_I8 3
#define QE_F8 4

/* An 8-bit cache: pages as in qe_kv_cache, [kv_heads][page][head_dim] codes of
 * one byte, and a scale for each of their rows, [n_pages][kv_heads][page]: an
 * element is code times scale.  All are 16-byte aligned.  (QE_F8: a code that is NaN is no
 * value of a cache; where a position has one, its sequence's outputs may be NaN.) */
typedef struct {
    void *k, *v;
    float *k_scale, *v_scale;
    int64_t n_pages; /* 1 .. 2^31 - 1 */
    int type;        /* QE_I8 or QE_F8 */
} qe_kv_cache8;

/* qe_attn_append to an 8-bit cache, with norms (norm may be NULL: none).  A row
 * x of k or v has the scale max |x| / 127 (QE_F8: / 448) and the codes x /
 * scale, rounded to nearest, in 32 bits: x is not rounded to 16 bits before.  A
 * row whose greatest is below 2^-100 has the scale 0; one with an element that
 * is not finite has the scale NaN, and all of its elements are NaN. */
int qe_attn_append8(qe_attn_ctx *ctx, const qe_attn_batch *batch, const qe_kv_cache8 *cache, const qe_attn_norm *norm, int in_type,
                    const void *q, int64_t q_stride, const void *k, int64_t k_stride, const void *v, int64_t v_stride,
                    const int32_t *pos, void *q_out, int64_t q_out_stride, void *stream);

/* The inverse: the keys and values that an 8-bit cache holds for the positions
 * of the call's tokens, rounded to the context's type, in rows of kv_heads *
 * head_dim (either of k and v may be NULL).  With cu_q the sums of kv_len all of
 * a batch's positions are read.  A token before its sequence's first position,
 * one whose length or page is bad, and one beside offsets that fall has rows of
 * zeros; rows of no sequence are left as they were. */
int qe_attn_read8(qe_attn_ctx *ctx, const qe_attn_batch *batch, const qe_kv_cache8 *cache, void *k, int64_t k_stride, void *v, int64_t v_stride,
                  void *stream);

/* qe_attn_prompt and qe_attn_decode over an 8-bit cache.  Products are as exact
 * as with a 16-bit cache, since codes are numbers of both 16-bit types; a key's
 * scale multiplies its score and a value's its probability, which is then, in
 * prompts, rounded to the context's type (fp16: to fixed steps below 2^-19 of
 * a row's greatest probability and the greatest scale of the positions that it
 * attends to), and for single tokens taken as two numbers of it.  A scale that is
 * not finite reaches the rows that attend to its position, and no others.  Of up to 64
 * sequences the longest are started first, in whatever order they are given. */
int qe_attn_prompt8(qe_attn_ctx *ctx, const qe_attn_batch *batch, const qe_kv_cache8 *cache, const void *q, int64_t q_stride, void *out,
                    int64_t out_stride, void *stream);
int qe_attn_decode8(qe_attn_ctx *ctx, const qe_attn_batch *batch, const qe_kv_cache8 *cache, const void *q, int64_t q_stride, void *out,
                    int64_t out_stride, void *stream);

/* ---- sequences that share their beginnings ----------------------------------- */

/* Groups of a call's sequences.  Group g's are seqs[g] .. seqs[g+1] - 1 (0 <=
 * seqs[0] <= ... <= seqs[n_groups] <= n_seqs); their first prefix[g] positions
 * are the same, and stand in the pages of the group's first sequence.  kv_len
 * counts them.  Of another sequence's table the entries of pages that lie wholly
 * before position prefix[g] are not used, and of the page that the position lies in
 * only the rows from it on.  A sequence of no group has all positions to itself.
 * Where a prefix is out of range (0 .. max_pages * page), a group's offsets
 * leave the call's sequences, or a sequence is shorter than its group's prefix,
 * those sequences' outputs are zeros; where offsets fall, the call's outputs may
 * hold anything.  Either is reported as a bad length. */
typedef struct {
    int n_groups;          /* 1 .. 65535 */
    const int32_t *seqs;   /* device [n_groups + 1] */
    const int32_t *prefix; /* device [n_groups] */
    int max_prefix;        /* the greatest prefix as far as the host knows, for choosing splits (results do not depend on it but
                              for rounding): its difference from batch->max_len is what sequences are expected to have to
                              themselves, and some may have more; 0 = not known */
} qe_attn_shared;

/* qe_attn_decode and qe_attn_decode8 of such sequences: a group's shared keys and
 * values are read once for all of its queries.  The results are those of the
 * plain calls on tables whose first entries are the shared pages, but for
 * rounding (fp16: probabilities below 2^-21 of a row's greatest to fixed steps;
 * over an 8-bit cache those of the shared positions are rounded as in prompts).
 * A bad page among the shared ones makes zeros of all of its
 * group's outputs. */
int qe_attn_decode_shared(qe_attn_ctx *ctx, const qe_attn_batch *batch, const qe_attn_shared *shared, const qe_kv_cache *cache, const void *q,
                          int64_t q_stride, void *out, int64_t out_stride, void *stream);
int qe_attn_decode8_shared(qe_attn_ctx *ctx, const qe_attn_batch *batch, const qe_attn_shared *shared, const qe_kv_cache8 *cache,
                           const void *q, int64_t q_stride, void *out, int64_t out_stride, void *stream);

/* Synchronise `stream` and report a bad length or page that a kernel met. */
int qe_attn_check(qe_attn_ctx *ctx, void *stream);

/* ---- gated delta rule ------------------------------------------------------ */

typedef struct {
    int k_heads, v_heads; /* value head h goes with key head h / (v_heads / k_heads) */
    int dim_k, dim_v;     /* 64 or 128 each */
    int type;             /* of q, k, v and out: QE_F32, QE_F16 or QE_BF16 */
    int l2norm;           /* 1: q and k rows are divided by sqrt(sum of squares + 1e-6) first */
    float scale;          /* of q; 0 = 1 / sqrt(dim_k) */
    int t_max;            /* largest n_tokens of qe_delta_prompt, 1 .. 2^20 */
    int seqs_max;         /* largest n_seqs of a call, 1 .. 65535 */
} qe_delta_desc;

typedef struct qe_delta_ctx qe_delta_ctx;

/* Create a context on `device`.  Scratch, for every 64 tokens of t_max and
 * every sequence of seqs_max: 49 KiB per value head, and per key head 768 bytes
 * of dim_k for fp32 (96 KiB of 128), 512 for fp16, none for bf16. */
int qe_delta_create(int device, const qe_delta_desc *desc, qe_delta_ctx **out);
int qe_delta_destroy(qe_delta_ctx *ctx);

/* Tensors of a call.  For every value head and token t of a sequence, with S
 * its state [dim_k][dim_v] (fp32):
 *   S <- exp(g_t) S;  u = beta_t (v_t - S^T k_t);  S <- S + k_t u^T;  out_t = scale S^T q_t.
 * States live in a pool of n_slots, each [v_heads][dim_k][dim_v].  Sequence i
 * starts from slot slots_in[i] (-1: zeros) and leaves its last state in
 * slots_out[i] (-1: nowhere).  A sequence may leave its state in the slot it
 * started from, and several may start from one slot; a slot that a sequence
 * writes may not be read or written by another in the same call.  A sequence
 * that would write a slot another one reads, or one that an earlier one
 * writes, is not computed: its outputs are zeros, its slot stays as it was, and
 * the context remembers it.  So is one with a slot outside the pool.  A sequence
 * without tokens passes its state on as it is.  Tokens are causal: a q, k, v,
 * g or beta that is infinite or NaN reaches no token before its own and no
 * other sequence.  A key whose sum of squares passes the range of 32 bits (a
 * length of 1.8e19) counts as not finite, and with l2norm so does a query.  Where
 * the rule itself leaves the range of 32 bits (g above 0 for long, or keys much
 * longer than one without l2norm), other tokens of the same 64 may be NaN, too. */
typedef struct {
    int n_seqs, n_tokens;
    const void *q, *k, *v;    /* [n_tokens] rows of k_heads * dim_k, k_heads * dim_k, v_heads * dim_v, of the context's type */
    int64_t q_stride, k_stride, v_stride; /* elements from token to token */
    const float *g, *beta;    /* [n_tokens][v_heads], contiguous; g is the log of the decay (below -1e4 counts as -1e4) */
    float *pool;              /* 16-byte aligned */
    int64_t n_slots;
    const int32_t *slots_in, *slots_out; /* device [n_seqs] */
    void *out;                /* [n_tokens] rows of v_heads * dim_v */
    int64_t out_stride;
} qe_delta_args;

/* Packed prompts: sequence i's tokens are rows cu[i] .. cu[i+1] - 1 (device
 * int32 [n_seqs + 1], 0 <= cu[0] <= ... <= cu[n_seqs] <= n_tokens); other rows
 * of out are left as they were.  Where offsets fall, which is reported, the
 * call's rows and the states it leaves may hold anything. */
int qe_delta_prompt(qe_delta_ctx *ctx, const qe_delta_args *args, const int32_t *cu, void *stream);

/* One token per sequence: n_tokens == n_seqs, row i is sequence i's.
 * A sequence whose slots are both -1 is computed from zeros and kept nowhere. */
int qe_delta_decode(qe_delta_ctx *ctx, const qe_delta_args *args, void *stream);

/* Synchronise `stream` and report a bad slot or length that a kernel met. */
int qe_delta_check(qe_delta_ctx *ctx, void *stream);

#ifdef __cplusplus
}
#endif
#endif
