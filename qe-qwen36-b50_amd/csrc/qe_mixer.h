// Internal declarations of the token mixers (include/qe_mixer.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/qe_mixer.h"
#include "qe_mixer_plan.h"

// What a kernel of a context reports: 0 or one of these in the context's host-mapped word.
enum : unsigned { QE_BAD_LENGTH = 1, QE_BAD_PAGE = 2, QE_BAD_SLOT = 3, QE_BAD_SHARED_SLOT = 4 };

struct QeAttnArgs {
    const void *q;
    void *out;
    const void *kc, *vc;
    int64_t q_stride, out_stride; // elements
    const int32_t *cu, *kv_len, *table;
    int n_seqs, n_tokens, table_stride, max_pages;
    int q_heads, kv_heads, group, page_log2;
    unsigned n_pages;
    float scale_log2; // scale * log2(e)
    int splits, tiles; // workgroups for a sequence (decode) or tile of rows (prompt) and key-value head
    int steps;         // decode: see qe_attn_decode_plan
    bool once;         // decode: see qe_attn_decode_once
    float *part_o;   // partial results: [item][split][row][head_dim], unnormalised
    float2 *part_ml; // [item][split][row] (decode: of 16): running maximum and sum; decode: sum < 0: the split met a bad page
    unsigned long long *arrived; // per sequence and key-value head, 0 between calls: decode's workgroups that are done; 16 bytes of zeros behind the last
    unsigned *err;
};

struct QeAppendArgs {
    const void *q, *k, *v;
    void *q_out, *kc, *vc;
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    const int32_t *pos, *cu, *kv_len, *table;
    const double *turns; // of each pair and position: theta^(-2 i / rotary) / (2 pi)
    const uint8_t *axis; // of each pair
    int n_axes, n_seqs, n_tokens, table_stride, max_pages;
    int q_heads, kv_heads, head_dim, page_log2, rotary;
    unsigned n_pages;
    unsigned *err;
};

// Norms, and an 8-bit cache: `a` with kc and vc codes (or 16-bit elements).
struct QeAppend8Args {
    QeAppendArgs a;
    const float *wq, *wk; // norms' weights, or null
    float eps;
    float *ks, *vs; // scales
};
struct QeRead8Args {
    const void *kc, *vc;
    const float *ks, *vs;
    void *k, *v;
    int64_t k_stride, v_stride;
    const int32_t *cu, *kv_len, *table;
    int n_seqs, n_tokens, table_stride, max_pages, kv_heads, head_dim, page_log2;
    unsigned n_pages;
    unsigned *err;
};

// Attention over an 8-bit cache: `a` with kc and vc codes.
struct QeAttn8Args {
    QeAttnArgs a;
    const float *ks, *vs; // scales
    bool spread;          // prompts: all tiles' first splits before their second ones (qe_attn_prompt8_blind)
};

// Sequences that share beginnings: `x` with kc, vc and, of an 8-bit cache, scales; x.a.splits and x.a.steps of their own
// positions, x.a.tiles of QE_ATTN_SHARED_BM rows.
struct QeSharedArgs {
    QeAttn8Args x;
    const int32_t *seqs, *prefix; // [n_groups + 1], [n_groups]
    int n_groups, psplits;
    int seq0, seq1; // of this launch
};

#define QE_CACHE16 0 /* a cache of the context's type, beside QE_I8 and QE_F8 */
hipError_t qe_launch_attn_prompt8(const QeAttn8Args &a, int head_dim, int type, int cache_type, int bm, bool halves, hipStream_t st);
hipError_t qe_launch_attn_decode8(const QeAttn8Args &a, int head_dim, int type, int cache_type, hipStream_t st);
hipError_t qe_launch_attn_shared(const QeSharedArgs &a, int head_dim, int type, int cache_type, hipStream_t st);
hipError_t qe_launch_append8(const QeAppend8Args &a, int in_type, int type, int cache_type, hipStream_t st);
hipError_t qe_launch_read8(const QeRead8Args &a, int type, int cache_type, hipStream_t st);
hipError_t qe_launch_append(const QeAppendArgs &a, int in_type, int type, hipStream_t st);
hipError_t qe_launch_attn_decode(const QeAttnArgs &a, int head_dim, int type, hipStream_t st);
hipError_t qe_launch_attn_prompt(const QeAttnArgs &a, int head_dim, int type, int bm, hipStream_t st);

struct QeDeltaArgs {
    const void *q, *k, *v;
    void *out;
    int64_t q_stride, k_stride, v_stride, out_stride;
    const float *g, *beta;
    float *pool;
    int64_t n_slots;
    const int32_t *slots_in, *slots_out, *cu;
    int n_seqs, n_tokens, k_heads, v_heads, group;
    int l2norm;
    int heads; // prompt: see qe_delta_heads
    float scale;
    float *ws;           // [chunk][v_head][QE_DELTA_WS]: see qe_delta.hip
    short *ws_kq;        // [chunk][k_head][K, Q][plane][64][dim_k], for types of more than one plane
    unsigned char *skip; // [n_seqs]: a sequence whose slots are bad
    unsigned *err;
};

hipError_t qe_launch_delta_prompt(const QeDeltaArgs &a, int dim_k, int dim_v, int type, hipStream_t st);
hipError_t qe_launch_delta_decode(const QeDeltaArgs &a, int dim_k, int dim_v, int type, hipStream_t st);

int qe_fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
