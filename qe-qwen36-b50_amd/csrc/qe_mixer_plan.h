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
// `round`: the workgroups that the GPU holds at once; `least`: steps of one where there are several sequences.
QE_MIX_HD void qe_attn_decode_cut(int64_t n_seqs, int64_t kv_heads, int round, int least, int64_t max_len, int *steps, int *splits) {
    const int64_t tiles = (max_len + QE_ATTN_TILE - 1) / QE_ATTN_TILE, units = n_seqs * kv_heads, total = tiles * units;
    const int64_t once = (total + round - 1) / round;
    int64_t per = once;
    if (n_seqs > 1) {
        per = (total + QE_ATTN_DECODE_WGS - 1) / QE_ATTN_DECODE_WGS;
        if (per < least) per = once < least ? once : least;
    }
    if (per > tiles) per = tiles; // one workgroup for each
    if (per < 2) per = 2;
    if (per < (tiles + QE_ATTN_DECODE_SPLITS - 1) / QE_ATTN_DECODE_SPLITS) per = (tiles + QE_ATTN_DECODE_SPLITS - 1) / QE_ATTN_DECODE_SPLITS;
    int64_t s = (tiles + per - 1) / per;
    if (s < 1 || units >= QE_ATTN_DECODE_WGS) s = 1;
    *steps = (int)per;
    *splits = (int)s;
}
QE_MIX_HD void qe_attn_decode_plan(int64_t n_seqs, int64_t kv_heads, int head_dim, int64_t max_len, int *steps, int *splits) {
    qe_attn_decode_cut(n_seqs, kv_heads, head_dim == 256 ? 512 : 768, 8, max_len, steps, splits);
}
// Over an 8-bit cache at least six steps (24 ragged sequences up to 8095 keys, 2 heads of 256: 32.5 us a call, 39.8 with
// eight, 32.5 with four; 8 x 8000: 24.9, 22.1 and 25.9).  Fewer and longer ones, so that the last workgroup joins all
// 16, are 5 to 10 % faster for sequences of one length, and a third slower where they differ much.
QE_MIX_HD void qe_attn_decode8_plan(int64_t n_seqs, int64_t kv_heads, int64_t max_len, int *steps, int *splits) {
    qe_attn_decode_cut(n_seqs, kv_heads, 512, 6, max_len, steps, splits);
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

// Whether a prompt workgroup over an 8-bit cache has eight waves, four for a tile's even steps and four for its odd ones, which join
// in LDS.  A wave alone on its SIMD takes 1.9 us for a step of 64 keys and heads of 128, two side by side 2.5: where a CU has one
// workgroup for most of the time, since tiles are few or unequal, eight waves take less.  Microseconds a call, int8, 32 / 8 heads
// of 128 unless other heads are named:
//   129 to 256 tiles and more than 4 steps: 900 tokens 28 (two splits 40); 3 x 300 after 1500 47 (splits 73); 1100 of 16 / 16 heads
//     of 64 24 (36).  Up to 128 tiles splits are as good (300 after 1000 30, 35 with eight waves);
//   257 to 512 tiles and at least 16 steps: 1500 tokens 40 (four waves 49); 200, 333 and 967 after 0, 1700 and 0 54 (65); but equal
//     tiles, 4 x 400 after 2000, 108 (97).  With less steps the join is what they save: 6 x 256 after 256 36 (30);
//   from 64 steps on a long tile among short ones needs splits: 256 and 800 after 4500 and 0 104 (splits 65);
//   tiles that fill the GPU: 8000 tokens 702 (625);  heads of 256, whose join is 128 KB: 1000 tokens of 16 / 2 54 (44).
QE_MIX_HD bool qe_attn_prompt8_halves(int64_t tiles, int bn, int64_t max_len) {
    const int64_t longest = (max_len + bn - 1) / bn;
    return bn == 64 && longest < 64 && (tiles <= 256 ? tiles > 128 && longest > 4 : tiles <= 512 && longest >= 16);
}
// A prompt call over an 8-bit cache splits a tile's keys by how many it has, so that a long tile among short ones is cut and these
// are not: `steps` steps a workgroup, at most `splits` for a tile and key-value head, as many as there is scratch for.
// Workgroups that a tile has no use for end at once, and one that has all of a tile's keys writes its rows itself.  At
// least eight steps, and as many as let twice the places of the GPU hold all tiles if each were as long as the longest (32 / 8 heads
// of 128, int8: 600 tokens after 20,000 326 us with 1.5 times, 290 with twice and with three times, 545 without; 50, 700 and 20
// after 5000, 0 and 19,000 of 24 / 8 heads of 64 93, 84 and 84, 377 without).  Where tiles fill half of the places and none has 40
// steps the join costs as much as it saves (4 x 400 after 2000 103 us without, 122 with; 1500 tokens 53 and 65).
// Partial results are of whole tiles, and there is room for 131,072 rows of them, twice what the other calls need: a long tile among short
// ones is cut into as many splits as there are for all.  (int8; with 65,536 rows: 256 and 800 after 4500 and 0 67 -> 135 us, 100 and 400
// after 30,000 and 1000 of 16 / 2 heads of 256 120 -> 222, 300 and 900 after 20,000 and 0 207 -> 552, 1500 after 10,000 of 24 / 8 of 64 205 -> 298,
// but 600 after 20,000 288 -> 285, 300 after 8000 81 -> 74, 800 after 30,000 of 16 / 2 of 256 463 -> 451; 98,304 are between or worse.)
#define QE_ATTN_PROMPT8_ROWS 131072
QE_MIX_HD void qe_attn_prompt8_plan(int64_t tiles, int bm, int bn, int64_t max_len, int *steps, int *splits) {
    const int64_t longest = (max_len + bn - 1) / bn, places = bm == 256 ? 256 : 512, room = QE_ATTN_PROMPT8_ROWS / (tiles * bm);
    int64_t per = (longest * tiles + 2 * places - 1) / (2 * places);
    if (per > longest) per = longest;
    if (per < 8) per = 8;
    int64_t s = (longest + per - 1) / per;
    if (s > room) s = room;
    if (s < 1 || (2 * tiles > places && longest < 40) || qe_attn_prompt8_halves(tiles, bn, max_len)) s = 1;
    *steps = (int)per;
    *splits = (int)s;
}
// The same where the host says nothing of the lengths, and a table may have room for far more than any sequence has: planned as if the
// call's tokens were all that there is, with splits (of at least 40 steps where tiles alone fill the places) for tiles that turn out to have more
// steps, as long as these are 1024 workgroups.  All tiles' first splits are begun before the second ones, which may all have none.  (Tables of
// 262,144 positions, int8, 32 / 8 heads of 128, us a call with lengths stated, without, and without as if all were as long as the table: 900
// tokens 28, 30, 56; 1000 of 16 / 2 heads of 256 44, 43, 104; 200, 333 and 967 after 0, 1700 and 0 51, 54, 70; 300 after 1000 29, 32, 59;
// 600 after 20,000 285, 325, 796; 256 and 800 after 4500 and 0 67, 85, 138; 30 after 10,000 of 16 / 2 of 256 34, 33, 85.)
// Whether a workgroup has eight waves.
QE_MIX_HD bool qe_attn_prompt8_blind(int64_t tiles, int bm, int bn, int64_t n_tokens, int64_t max_len, int *steps, int *splits) {
    const int64_t likely = n_tokens < max_len ? n_tokens : max_len;
    const bool halves = qe_attn_prompt8_halves(tiles, bn, likely);
    qe_attn_prompt8_plan(tiles, bm, bn, likely, steps, splits);
    if ((halves || 2 * tiles > (bm == 256 ? 256 : 512)) && *steps < 40) *steps = 40;
    const int64_t longest = (max_len + bn - 1) / bn, room = QE_ATTN_PROMPT8_ROWS / (tiles * bm), most = 1024 / tiles;
    int64_t s = (longest + *steps - 1) / *steps;
    if (s > room) s = room;
    if (s > most) s = most;
    if (s > *splits) *splits = (int)s;
    return halves;
}
// Steps of `bn` keys of the tile of rows from row0 on, up to the place of its last row.  (The sequence's rows are tokens begin ..
// end - 1 times `group`, and its last position is the last token's.)
QE_MIX_HD int qe_attn_tile_steps(int len, int begin, int end, int row0, int group, int bm, int bn) {
    const int n_rows = (end - begin) * group, last = (row0 + bm < n_rows ? row0 + bm - 1 : n_rows - 1) / group, keys = len - (end - begin) + last + 1;
    return keys > 0 ? (keys + bn - 1) / bn : 0;
}
QE_MIX_HD int qe_attn_tile_splits(int n, int steps, int splits) {
    const int s = (n + steps - 1) / steps;
    return s < 1 ? 1 : s < splits ? s : splits;
}

// A call of single tokens whose sequences share beginnings: `psplits` workgroups for every 128 rows of a group's queries and
// key-value head over the shared keys, and `splits` of `steps` steps for a sequence's own (qe_attn_decode_cut).
// A split of the shared keys costs its partial results, and saves the others time: P splits take about a prefix / P + b rows
// P, which is least where P^2 is a / b times prefix / rows.  With a / b = 40, at least 64 keys, and at most one workgroup a CU if all
// sequences are one group's, 32 sequences of 16 heads of 256 behind 8000 take 34 us a call (36 with 60, 39 with 100), 8 behind 16,000 30 (29, 29).
// Each group has tiles of its own, so that several have more workgroups than that.  Counting them, with as many workgroups as the GPU holds at
// once, is right where groups are alike (32 of two behind 2000, 16 / 2 heads of 256, 33 us for 40; of 32 / 8 of 128 56 for 64) and far off where one
// is large and others share little (8 sequences behind 20,000 beside 50 of their own 201 us for 62; 32 behind 8000 beside 32, 32 / 8 of 128, 122 for 44).
// A sequence's own positions: at least twelve steps a workgroup, or as few as make 768 workgroups if all are as long as the longest.
// (32 sequences of 16 / 2 heads of 256 with up to 1500 of their own: 31.8 us a call, 33.4 with 512, 37.9 with 1024; 50 of 8 / 1 with up to
// 1000: 25.9, 27.0, 26.4.  At least eight steps: 64 of 32 / 8 heads of 128 with up to 1000 46.9 for 42.2, but 40 of 24 / 8 of 64 with up to
// 1500 26.7 for 29.1.)
// That is planned for max_own, the longest own part as far as the hints tell: the difference of the longest length and the longest prefix, or,
// where not both are stated, 0 (not known: eight steps a workgroup).  It may be wrong, for a sequence behind a shorter prefix or of no group
// may have far more of its own: there are workgroups for up to max_len positions, of at least as many steps, as long as these are 1024 in
// all, and those that a sequence has no use for end at once.  They come last in the launch.  (One of 30,000 positions beside eight that have ten each
// behind 30,000, 16 / 2 heads of 256: 37 us a call, 440 with workgroups for max_own alone; four of 2000 beside ten behind 16,000: 30, 43.  32
// behind 8000 without a hint: 30, 47, and 31 with hints either way; with 2048 workgroups 31.5, and 44 where those without keys come among the others.)
// Each leaves partial results, psplits + splits for a row of n_seqs * q_heads, which have room for QE_ATTN_SHARED_ROWS.  At
// most 2^15 rows are in a launch (qe_attn_shared_seqs), so that each has room for two.
#define QE_ATTN_SHARED_ROWS 65536
#define QE_ATTN_SHARED_BM 128 /* rows of a workgroup */
QE_MIX_HD int qe_attn_shared_seqs(int n_seqs, int q_heads) {
    const int most = QE_ATTN_SHARED_ROWS / 2 / q_heads;
    return n_seqs < most ? n_seqs : most;
}
QE_MIX_HD void qe_attn_shared_plan(int n_seqs, int q_heads, int kv_heads, int64_t max_prefix, int64_t max_own, int *psplits, int *steps, int *splits,
                                    int64_t max_len = 0) {
    const int64_t rows = (int64_t)n_seqs * q_heads, room = QE_ATTN_SHARED_ROWS / rows;
    *steps = 8, *splits = 1;
    if (max_own > 0) qe_attn_decode_cut(n_seqs, kv_heads, 768, 12, max_own, steps, splits);
    const int64_t longest = (max_len + (int64_t)QE_ATTN_TILE * *steps - 1) / ((int64_t)QE_ATTN_TILE * *steps), most_wgs = 1024 / ((int64_t)n_seqs * kv_heads);
    const int64_t more = longest < most_wgs ? longest : most_wgs;
    if (more > *splits) *splits = (int)more;
    if (*splits > (room + 1) / 2) *splits = (int)((room + 1) / 2);
    const int64_t tiles = ((int64_t)n_seqs * (q_heads / kv_heads) + QE_ATTN_SHARED_BM - 1) / QE_ATTN_SHARED_BM * kv_heads;
    const int64_t most = (max_prefix + 63) / 64, fill = (256 + tiles - 1) / tiles;
    int64_t s = 1;
    while (s * s * rows < 40 * max_prefix && s < most && s < fill) ++s;
    if (s > room - *splits) s = room - *splits;
    *psplits = s < 1 ? 1 : (int)s;
}
// Steps of `step` keys of a shared beginning in each of its splits, and how many of those have any.
QE_MIX_HD int qe_attn_shared_per(int prefix, int step, int psplits) { return ((prefix + step - 1) / step + psplits - 1) / psplits; }
QE_MIX_HD int qe_attn_shared_active(int prefix, int step, int psplits) {
    const int per = qe_attn_shared_per(prefix, step, psplits);
    return per ? ((prefix + step - 1) / step + per - 1) / per : 0;
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
