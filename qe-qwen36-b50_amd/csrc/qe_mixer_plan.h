// How a call of the token mixers is cut into workgroups, and which values from device
// memory are used.  Plain C++ that the launchers, the kernels and the CPU tests share.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define QE_MIX_HD __host__ __device__ __forceinline__
#else
#define QE_MIX_HD static inline
#endif

// A launch has less than 2^32 threads.
QE_MIX_HD bool qe_fits_launch(int64_t workgroups, int threads) { return workgroups < ((int64_t)1 << 32) / threads; }

// ---- attention ----------------------------------------------------------------
#define QE_ATTN_SUB 16     /* keys that share one page lookup: the smallest page */
#define QE_ATTN_TILE 32    /* keys of a decode wave's step */
#define QE_ATTN_WGS 512    /* workgroups a prompt call is split up to: two for each of the 256 CUs */
#define QE_ATTN_DECODE_WGS 2048 /* and a decode call at most */
#define QE_ATTN_DECODE_SPLITS 1024
#define QE_ATTN_JOIN 16    /* splits that the last workgroup of a decode call joins itself; more: a launch of its own */

// A decode call gives a workgroup `steps` steps of QE_ATTN_TILE keys of one sequence and key-value
// head, the same for all sequences, so that a ragged batch is even: `splits` workgroups are
// launched for each, enough for max_len, and those behind a sequence's end do nothing.
// One sequence: as many workgroups as the GPU holds at once, two or three a CU (LDS; a round of at most
// 512 takes 37 us over 100,000 keys of two heads of 256, 696 take 40), of at least two steps.
// Several, which may differ in length: up to 2048, but of at least eight steps where that
// many fill the GPU.  units = n_seqs * kv_heads.
QE_MIX_HD void qe_attn_decode_plan(int64_t n_seqs, int64_t kv_heads, int head_dim, int64_t max_len, int *steps, int *splits) {
    const int64_t tiles = (max_len + QE_ATTN_TILE - 1) / QE_ATTN_TILE, units = n_seqs * kv_heads, total = tiles * units;
    const int64_t round = head_dim == 256 ? 512 : 768, once = (total + round - 1) / round;
    int64_t per = once;
    if (n_seqs > 1) {
        per = (total + QE_ATTN_DECODE_WGS - 1) / QE_ATTN_DECODE_WGS;
        if (per < 8) per = once < 8 ? once : 8;
    }
    if (per > tiles) per = tiles; // one workgroup for each
    if (per < 2) per = 2;
    if (per < (tiles + QE_ATTN_DECODE_SPLITS - 1) / QE_ATTN_DECODE_SPLITS) per = (tiles + QE_ATTN_DECODE_SPLITS - 1) / QE_ATTN_DECODE_SPLITS;
    int64_t s = (tiles + per - 1) / per;
    if (s < 1 || units >= QE_ATTN_DECODE_WGS) s = 1;
    *steps = (int)per;
    *splits = (int)s;
}
// Steps of a sequence of `len` keys in each of its workgroups (more than planned where the host's max_len was short
// of it), and how many of those have any.
QE_MIX_HD int qe_attn_decode_steps(int len, int steps, int splits) {
    const int tiles = (len + QE_ATTN_TILE - 1) / QE_ATTN_TILE, need = (tiles + splits - 1) / splits;
    return need > steps ? need : steps;
}
QE_MIX_HD int qe_attn_decode_active(int len, int steps) { return ((len + QE_ATTN_TILE - 1) / QE_ATTN_TILE + steps - 1) / steps; }
// Whether a decode call's keys and values exceed the eight L2s of 4 MB and pass through them (per call, on data of ten
// layers in turn: 8 x 2000 keys of 8 heads of 128, 65 MB, 20.2 -> 19.1 us; 100,000 keys of 2 of 256, 205 MB, 45.4 -> 42.5; but
// 8000 of these, 16 MB, 12.8 -> 13.6, which stay).
QE_MIX_HD bool qe_attn_decode_once(int64_t n_seqs, int64_t kv_heads, int head_dim, int64_t max_len) {
    return n_seqs * kv_heads * head_dim * 4 >= ((int64_t)32 << 20) / (max_len > 0 ? max_len : 1);
}
// Partial results that a decode call can need: with more than one split units < QE_ATTN_DECODE_WGS, and
// units * splits < QE_ATTN_DECODE_WGS + units.
#define QE_ATTN_PART_WGS (2 * QE_ATTN_DECODE_WGS)

// Query rows of a prompt call are its tokens times the heads that share a key-value head,
// and a workgroup takes `bm` of one sequence.  Tile numbers are handed out so that the
// launch needs no lengths from the device: sequence i's tiles start at first(i) =
// cu[i] * group / bm + i, and since floor(a + b) + 1 >= floor(a) + ceil(b) they end before
// first(i + 1).  Numbers between are of no sequence and do nothing.
QE_MIX_HD int qe_attn_first_tile(int cu, int i, int group, int bm) { return (int)((int64_t)cu * group / bm) + i; }
QE_MIX_HD int qe_attn_max_tiles(int n_tokens, int n_seqs, int group, int bm) {
    return (int)((int64_t)n_tokens * group / bm) + n_seqs;
}

// Rows of a prompt workgroup.  With heads of 256 and 64 keys a step its K and V tiles fill a CU's LDS, so eight
// waves are the way to two waves a SIMD; calls with too few rows for that, and smaller heads, take four.
QE_MIX_HD int qe_attn_prompt_rows(int n_tokens, int n_seqs, int group, int kv_heads, int head_dim) {
    return head_dim == 256 && (int64_t)qe_attn_max_tiles(n_tokens, n_seqs, group, 256) * kv_heads >= 256 ? 256 : 128;
}

// Splits of a prompt call's keys: two workgroups for each CU, of at least 256 keys; above 128 tiles none.  Where the tiles
// fill the GPU a split only adds the join: 528 tiles take 47 us a call, and 78 in two splits.  From 129 to 255 tiles, which
// leave half of the places empty, it is right over short keys (900 tokens of 32 and 8 heads of 128: 34 us, 45 in two
// splits; 1200 of 24 and 8 heads of 64: 31, 39) and wrong over long ones (2000 tokens of 16 and 2 heads of 256: 92 us, 84 in
// two; 16 x 4 after 8000 with heads of 128: 165, 123 in three; 600 after 20,000: 404, 260).
QE_MIX_HD int qe_attn_prompt_splits(int64_t tiles, int64_t max_len) {
    if (tiles > 128) return 1;
    const int64_t most = (max_len + 255) / 256, want = QE_ATTN_WGS / tiles;
    const int64_t s = want < most ? want : most;
    return s < 1 ? 1 : (int)s;
}

// The part [*lo, *hi) of n steps that split s of `splits` takes.
QE_MIX_HD void qe_split_range(int n, int splits, int s, int *lo, int *hi) {
    const int per = (n + splits - 1) / splits;
    const int64_t a = (int64_t)s * per, b = a + per;
    *lo = a < n ? (int)a : n;
    *hi = b < n ? (int)b : n;
}

// A length or offset from device memory that is outside lo .. hi becomes `other`, and *bad is set.
QE_MIX_HD int qe_checked(int v, int lo, int hi, int other, unsigned *bad) {
    if (v < lo || v > hi) {
        *bad = 1;
        return other;
    }
    return v;
}

// Whether a sequence's offsets are not: below 0, falling, or behind the call's tokens.
QE_MIX_HD bool qe_bad_offsets(int cu0, int cu1, int n_tokens) { return cu0 < 0 || cu1 < cu0 || cu1 > n_tokens; }
QE_MIX_HD int qe_clamped(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
// The sequence's rows [*begin, *end) among the call's, whatever its offsets are; *bad is set where they are not.
QE_MIX_HD void qe_rows_of(int cu0, int cu1, int n_tokens, int *begin, int *end, unsigned *bad) {
    *begin = qe_clamped(cu0, 0, n_tokens);
    *end = qe_clamped(cu1, *begin, n_tokens);
    if (qe_bad_offsets(cu0, cu1, n_tokens)) *bad = 1;
}

// ---- gated delta rule ------------------------------------------------------------
#define QE_DELTA_C 64                     /* tokens of a chunk */
#define QE_DELTA_WS (6 * 64 * 64 / 2 + 4 * 64) /* floats kept per chunk and value head: six planes of 16 bits, four vectors */

// Chunk numbers are handed out as a prompt's tiles are: sequence i's start at first(i).
QE_MIX_HD int qe_delta_first_chunk(int cu, int i) { return cu / QE_DELTA_C + i; }
// 16-bit planes that keys and queries are cut into and kept as; bf16 ones are one as they stand.
QE_MIX_HD int qe_delta_kept_planes(int bytes, int is_bf16) { return is_bf16 ? 0 : bytes == 4 ? 3 : 2; }
// Value heads of a workgroup that makes a chunk's matrices: all of the key head's, which share the products of keys and
// queries, unless a workgroup for each is no more than the GPU holds at once, three a CU (one bf16 chunk of 16 and 32
// heads: 10 us, and 15 with two heads a workgroup).
QE_MIX_HD int qe_delta_heads(int64_t chunks, int v_heads, int group) { return chunks * v_heads <= 768 ? 1 : group; }
QE_MIX_HD int qe_delta_max_chunks(int n_tokens, int n_seqs) { return n_tokens / QE_DELTA_C + n_seqs; }

// Whether sequence i of a call may be computed: its slots are in the pool (or -1), and nobody
// else reads the slot it writes, and no earlier one writes it.  0, or what is wrong: the two
// values below.  Of the sequences that are computed no two touch a slot that one of them
// writes: a later writer of the same slot is refused, and so is the writer of a slot that
// any other sequence reads.
#define QE_SLOT_OUTSIDE 1
#define QE_SLOT_SHARED 2
QE_MIX_HD int qe_slot_pair(int64_t n_slots, int in_i, int out_i) {
    return in_i < -1 || in_i >= n_slots || out_i < -1 || out_i >= n_slots ? QE_SLOT_OUTSIDE : 0;
}
QE_MIX_HD int qe_slot_conflict(int i, int out_i, int j, int in_j, int out_j) {
    return out_i >= 0 && j != i && (in_j == out_i || (j < i && out_j == out_i)) ? QE_SLOT_SHARED : 0;
}
