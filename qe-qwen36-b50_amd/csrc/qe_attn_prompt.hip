// Causal attention of packed prompts over a paged cache.
//
// A workgroup takes 32 query rows for each of its waves, of one sequence and one key-value head
// (its tokens times the heads that share the key-value head, so that no key is read for one
// head alone), and steps through the keys 64 (or 32, below) at a time.  Per
// step S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16: a lane's column is one query
// row, so maximum, sum and rescaling are per lane (plus one exchange between the wave's
// halves), and the registers that hold S^T's rows are, once rounded, the second product's
// operand as they stand: its k runs over the keys in the order in which they lie there, and
// V^T is read from LDS in that order by transposing reads.
//
// K and V tiles reach LDS by direct loads into one of two buffers while the other is
// worked on.  16-byte chunks are permuted within their rows at the source (LDS rows
// are contiguous for direct loads): K's by row % 8, so that the eight rows of a read's
// phase lie in different banks, V's 64-byte units by row % 4.
//
// Scores, maxima and sums are in 32 bits; probabilities are rounded to the cache's type for the
// second product (exponent_base).  A row's maximum is raised only where a score exceeds it by 2^8, so that O is seldom rescaled.
// Long prompts are bound by the matrix cores, whose issue the exponentials share: 8192 tokens of 16 heads of 256 (550
// GFLOP), bf16, 557 us on average of 30 in a row, under which the clock falls, and 511 at least: 990 and 1080 TFLOP/s where a
// large library product reaches 1219.  Five
// prompts of 1999 tokens, 32 heads of 128, fp16: 38 us, the longest row blocks' 18 steps in turn.
// 100 tokens: 13 us, latency (lengths, pages, four steps, the output), much of it the code's first way through the
// instruction cache: a workgroup whose code was three times as long, in steps of 64 keys with 512 registers, took 15.
#include "qe_attn_rows.h"

// Four waves with heads of up to 128, and two or more workgroups on a CU.  With heads of 256 the tiles fill a CU's LDS, so
// eight waves are the way to two waves a SIMD, and o and q leave registers for 32 keys' scores at a time, not 64; a call
// too small for eight takes four, in steps of 32 keys, so that two workgroups share a CU there, too.  (Measured and not kept: the next tile's scores made among this
// one's exponentials, 10 % slower over 4096 tokens of heads of 64 and 128; the second four waves half a tile behind the
// first, 8 % slower over 8192 of 256; 64 rows a wave, whose 512 registers do not hold them.)
template <bool BF, int DH, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void k_attn_prompt(const QeAttnArgs a) {
    constexpr int BM = 32 * WAVES, BN = DH == 256 && WAVES == 4 ? 32 : 64, PART = BN / WAVES;
    // two buffers, variables of their own: else the compiler has every LDS read wait for the direct loads in flight
    __shared__ __align__(16) short k_a[BN * DH], v_a[BN * DH], k_b[BN * DH], v_b[BN * DH];
    // rows with an infinity or a NaN in V, of the tiles that some rows attend to in part: from `clear` on, BM tokens at most
    __shared__ unsigned long long odd_rows[BM / BN + 2];
    __shared__ int lost_s[WAVES]; // a wave met a page that is none
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int split = blockIdx.x % a.splits, kvh = blockIdx.x / a.splits % a.kv_heads;
    // A sequence's late rows have more keys: first.  (So are the last sequence's, whatever its length: 31 prompts of 32 heads of
    // 128, one of 1500 tokens and the others of 30, take 44 us with the long one last and 50 with it first.)
    const int tile = a.tiles - 1 - blockIdx.x / a.splits / a.kv_heads;
    // Workgroup i looks at sequence i's offsets, for the report: where they fall, a sequence may have no tile below.  (There
    // are more workgroups than sequences; the others look at the last one's, so that no branch has its own wait for the loads.)
    const int mine = blockIdx.x < (unsigned)a.n_seqs ? blockIdx.x : a.n_seqs - 1;
    const int mine0 = scalar_load(a.cu + mine), mine1 = scalar_load(a.cu + mine + 1);
    int seq = 0;
    for (int hi = a.n_seqs; hi - seq > 1;) { // the last sequence whose first tile is not behind this one
        const int mid = (seq + hi) >> 1;
        if (qe_attn_first_tile(qe_clamped(scalar_load(a.cu + mid), 0, a.n_tokens), mid, a.group, BM) <= tile) seq = mid;
        else hi = mid;
    }
    const int cu0 = scalar_load(a.cu + seq), cu1 = scalar_load(a.cu + seq + 1), kv = scalar_load(a.kv_len + seq);
    unsigned bad_len = 0;
    int begin, end;
    qe_rows_of(cu0, cu1, a.n_tokens, &begin, &end, &bad_len);
    const int local = tile - qe_attn_first_tile(begin, seq, a.group, BM);
    int len = qe_checked(kv, 0, a.max_pages << a.page_log2, 0, &bad_len);
    if (bad_len) len = 0; // no row has a position: zeros
    if ((bad_len || qe_bad_offsets(mine0, mine1, a.n_tokens)) && tid == 0) report(a.err, QE_BAD_LENGTH);
    const int n_rows = (end - begin) * a.group;
    if (local < 0 || (int64_t)local * BM >= n_rows) return; // uniform: no row of the sequence
    const int row0 = local * BM, first = len - (end - begin); // first: position of the sequence's first row
    const int32_t *table = a.table + (size_t)seq * a.table_stride;

    // keys of the tile: up to its last row's place; below `clear` every row attends to every key
    const int last_tok = (row0 + BM < n_rows ? row0 + BM - 1 : n_rows - 1) / a.group;
    const int keys = first + last_tok + 1, clear = first + row0 / a.group + 1 > 0 ? first + row0 / a.group + 1 : 0;
    // the same for the wave
    const int wave_row = row0 + wave * 32, wave_end = wave_row + 32 < n_rows ? wave_row + 32 : n_rows;
    const int wave_keys = wave_row < n_rows ? first + (wave_end - 1) / a.group + 1 : 0, wave_clear = first + wave_row / a.group + 1;
    int lo, hi;
    qe_split_range(keys > 0 ? (keys + BN - 1) / BN : 0, a.splits, split, &lo, &hi);

    int page = 0; // of the wave's part of the next tile
    if (lo < hi) {
        page = page_of<BN, WAVES>(a, table, lo * BN, len, wave);
        load_part<DH, BN, WAVES, true>(a, page, kvh, lo * BN, len, wave, k_a);
        load_part<DH, BN, WAVES, false>(a, page, kvh, lo * BN, len, wave, v_a);
        page = page_of<BN, WAVES>(a, table, (lo + 1) * BN, len, wave);
    }
    Rows<BF, DH> w;
    {
        const int row = wave_row + (tid & 31), h = tid >> 5 & 1;
        const bool there = row < n_rows;
        const int tok = there ? row / a.group : 0, head = kvh * a.group + (there ? row - tok * a.group : 0);
        w.place = there ? first + tok : -1;
        const short *q = (const short *)a.q + (size_t)(begin + tok) * a.q_stride + (size_t)head * DH + h * 8;
#pragma unroll
        for (int s = 0; s < DH / 16; ++s) w.q[s] = there ? *(const qe_s8 *)(q + s * 16) : qe_s8{};
        w.m = -INFINITY;
        w.l = 0;
#pragma unroll
        for (int d = 0; d < DH / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) w.o[d][i] = 0;
    }
    if (tid < BM / BN + 2) odd_rows[tid] = 0;
    const int lost = __any(lo < hi ? lost_pages<64 * WAVES>(a, table, (len + (1 << a.page_log2) - 1) >> a.page_log2, tid) : 0);
    if ((tid & 63) == 0) lost_s[wave] = lost;
    lds_barrier(); // for odd_rows, too: the first tile's marks come before its own barrier
    int any = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) any |= lost_s[i];
    if (__builtin_amdgcn_readfirstlane(any)) {
        if (tid == 0) report(a.err, QE_BAD_PAGE);
        hi = lo; // no key: zeros
        __builtin_amdgcn_s_waitcnt(0x0f70); // nothing reads what is on its way to LDS, but it lands before the workgroup ends
    }

    // The wave's direct loads have landed.  A probability of 0 times an infinity or NaN is NaN: in its part of V's tile t rows
    // behind the end become zeros, and so do elements that are not finite, which are added in the end for the rows
    // that attend to them.
    auto arrived = [&](int t, short *v_lds) {
        __builtin_amdgcn_s_waitcnt(0x0f70);
        const int k0 = t * BN;
        if (k0 + BN > clear)
            for (int i = lane_now(); i < PART * (DH / 8); i += 64) {
                const int row = wave * PART + i / (DH / 8);
                short *at = v_lds + wave * PART * DH + i * 8;
                qe_s8 x = *(const qe_s8 *)at;
                if (k0 + row >= len) {
                    *(qe_s8 *)at = qe_s8{};
                } else {
                    constexpr int top = BF ? 0x7f80 : 0x7c00;
                    bool odd = false;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if ((x[j] & top) == top) x[j] = 0, odd = true;
                    if (odd) {
                        *(qe_s8 *)at = x;
                        atomicOr(&odd_rows[t - clear / BN], 1ull << row);
                    }
                }
            }
    };
    auto work = [&](int t, const short *k_lds, short *v_lds, short *k_next, short *v_next) {
        arrived(t, v_lds);
        lds_barrier(); // the others' loads, too, and no wave reads the other buffers any more
        const int k0 = t * BN;
        if (t + 1 < hi) {
            load_part<DH, BN, WAVES, true>(a, page, kvh, k0 + BN, len, wave, k_next);
            load_part<DH, BN, WAVES, false>(a, page, kvh, k0 + BN, len, wave, v_next);
        }
        page = page_of<BN, WAVES>(a, table, k0 + 2 * BN, len, wave); // looked up a step before it is needed
        if (k0 >= wave_keys) return;
        constexpr int KB = DH == 256 ? 1 : 2;
#pragma unroll
        for (int b = 0; b < BN / 32; b += KB) {
            Scores<KB> s;
            w.scores(k_lds, b, s);
            schedule<4, KB * DH / 16, 1>();
            if (k0 + BN > wave_clear) s.mask(w.place - k0 - b * 32 - 4 * (lane_now() >> 5));
            w.raise(s.top() * a.scale_log2);
            Probs<KB> p;
            w.exponentials(a.scale_log2, s, p);
            w.values(v_lds, b, p);
            schedule<3, KB * DH / 16, 2>();
        }
    };
    for (int t = lo; t < hi; t += 2) {
        work(t, k_a, v_a, k_b, v_b);
        if (t + 1 < hi) work(t + 1, k_b, v_b, k_a, v_a);
    }
    lds_barrier(); // all marks are made
    const int h = lane_now() >> 5;
    for (int t = clear / BN; t < hi; ++t) {
        unsigned long long odd = t >= lo ? odd_rows[t - clear / BN] : 0;
        while (odd) { // uniform, and empty but for values that are not finite
            const int key = t * BN + __ffsll(odd) - 1;
            odd &= odd - 1;
            unsigned known = 0;
            const size_t at = sub_row(a, table, kvh, __builtin_amdgcn_readfirstlane(key) & ~15, &known) + (key & 15);
            const short *v = (const short *)a.vc + at * DH + 4 * h;
            if (key <= w.place)
#pragma unroll
                for (int d = 0; d < DH / 32; ++d)
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const qe_s4 x = *(const qe_s4 *)(v + d * 32 + 2 * i);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float y = from16<BF>(x[j]);
                            if (!__builtin_isfinite(y)) w.o[d][i + j] += y;
                        }
                        asm volatile("" ::: "memory"); // not all of the row in registers at once
                    }
        }
    }
    w.template finish<BM>(a, begin, n_rows, row0, wave_row, tile, kvh, split, a.splits == 1);
}

template <bool BF, int DH, int WAVES>
static hipError_t launch_waves(const QeAttnArgs &a, hipStream_t st) {
    k_attn_prompt<BF, DH, WAVES><<<dim3((unsigned)(a.tiles * a.kv_heads * a.splits)), dim3(64 * WAVES), 0, st>>>(a);
    launch_prompt_join<BF, DH, 32 * WAVES>(a, st);
    return hipGetLastError();
}
template <bool BF, int DH>
static hipError_t launch_prompt(const QeAttnArgs &a, int bm, hipStream_t st) {
    if constexpr (DH == 256)
        if (bm == 256) return launch_waves<BF, DH, 8>(a, st);
    return launch_waves<BF, DH, 4>(a, st);
}

hipError_t qe_launch_attn_prompt(const QeAttnArgs &a, int head_dim, int type, int bm, hipStream_t st) {
    if (type == QE_BF16)
        return head_dim == 64    ? launch_prompt<true, 64>(a, bm, st)
               : head_dim == 128 ? launch_prompt<true, 128>(a, bm, st)
                                 : launch_prompt<true, 256>(a, bm, st);
    return head_dim == 64    ? launch_prompt<false, 64>(a, bm, st)
           : head_dim == 128 ? launch_prompt<false, 128>(a, bm, st)
                             : launch_prompt<false, 256>(a, bm, st);
}
