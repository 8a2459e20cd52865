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
#include "qe_mixer_device.h"

__device__ __forceinline__ int k_swz(int row) { return row & 7; }
template <int DH>
__device__ __forceinline__ int v_swz(int row) {
    return DH == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2;
}

// The lane's number, made where it is needed: kept, and what follows from it, it would take registers that the loop over
// the tiles does not have, and reloads of spilled ones wait for the direct loads in flight.
__device__ __forceinline__ int lane_now() {
    int lane;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
    return lane;
}

// The page of a wave's part of the tile of BN keys from position k0 on: all of the part's rows lie in one.
// Rows behind the end may lie in none, then any of the sequence's do (their probabilities are zero).
template <int BN, int WAVES>
__device__ __forceinline__ int page_of(const QeAttnArgs &a, const int32_t *table, int k0, int len, int wave) {
    const int sub = k0 + wave * (BN / WAVES);
    return scalar_load(table + ((sub < len ? sub : len - 1) >> a.page_log2));
}
// The part's rows of K or V to LDS.
template <int DH, int BN, int WAVES, bool IS_K>
__device__ __forceinline__ void load_part(const QeAttnArgs &a, int page, int kvh, int k0, int len, int wave, short *lds) {
    constexpr int CH = DH / 8, ROWS = 64 / CH, PART = BN / WAVES; // chunks of a row, rows of one direct load, rows of a wave
    const int sub = k0 + wave * PART, at = sub < len ? sub : (len - 1) & -PART;
    unsigned known = 0; // that a page is none: lost_pages
    const size_t r0 = page_row(a, page, kvh, at, &known);
    const char *from = (const char *)(IS_K ? a.kc : a.vc) + r0 * DH * 2;
    // A uniform address and a 32-bit offset: a later row's permutation differs from the first load's by a constant.
    const int lane = lane_now(), row = lane / CH, c = lane % CH;
    const unsigned off = row * DH * 2 + ((c ^ (IS_K ? k_swz(row) : v_swz<DH>(row))) << 4);
#pragma unroll
    for (int i = 0; i < PART / ROWS; ++i)
        load_lds16_from(from, PART * DH * 2, off ^ ((IS_K ? k_swz(i * ROWS) : v_swz<DH>(i * ROWS)) << 4), i * 1024, lds + (wave * PART + i * ROWS) * DH);
}

// Whether one of the `n` pages of a sequence is none of the cache's: of the thread's share of them.  Each workgroup
// looks at all, since the rows of all are zeros then; four at a time, the last again behind the end.
template <int THREADS>
__device__ __forceinline__ int lost_pages(const QeAttnArgs &a, const int32_t *table, int n, int tid) {
    int lost = 0;
    for (int i = tid; i < n; i += 4 * THREADS) {
        unsigned p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = table[i + j * THREADS < n ? i + j * THREADS : n - 1];
#pragma unroll
        for (int j = 0; j < 4; ++j) lost |= p[j] >= a.n_pages;
    }
    return lost;
}

__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
// the larger of the values of lanes l and l ^ 32
__device__ __forceinline__ float max_halves(float x) {
    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}

// The order of N matrix products that take READS LDS reads each: the reads of AHEAD of them first, then those of one for
// each product.  Left alone, the scheduler reads, waits and multiplies in turn.
template <int AHEAD, int N, int READS>
__device__ __forceinline__ void schedule() {
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * READS, 0);
#pragma unroll
    for (int i = 0; i < N - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
}

// A wave's 32 query rows, lane r of either half row r, and their scores of KB blocks of 32 keys.
template <int KB>
struct Scores {
    qe_f16v s[KB]; // S^T

    // keys behind `limit`, counted from the lane's first, are not attended to
    __device__ __forceinline__ void mask(int limit) {
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (b * 32 + 8 * (i / 4) + i % 4 > limit) s[b][i] = -INFINITY;
    }
    __device__ __forceinline__ float top() const { // of the row
        float t = s[0][0];
#pragma unroll
        for (int i = 1; i < 15; i += 2) t = max3(t, s[0][i], s[0][i + 1]);
        t = max3(t, s[0][15], s[KB - 1][0]);
        if constexpr (KB == 2) {
#pragma unroll
            for (int i = 1; i < 15; i += 2) t = max3(t, s[1][i], s[1][i + 1]);
            t = fmaxf(t, s[1][15]);
        }
        return max_halves(t);
    }
};
template <int KB>
struct Probs {
    union {
        unsigned u[4];
        qe_s8 v;
    } p[KB][2]; // 16 keys each, as the second product's operand
};

template <bool BF, int DH>
struct Rows {
    static constexpr int LAG = 8;
    qe_f16v o[DH / 32]; // O^T
    qe_s8 q[DH / 16];
    float m, l; // running maximum of the scores (scaled, in powers of two) and sum
    int place;  // position of the lane's query; below 0 where it attends to nothing

    // S^T = K Q^T of KB blocks from block b0 of the tile on.  Chunk 2 st + h of K's row r is permuted by the row's low
    // bits, so the four st of a 128-byte block are one address with constants exclusive-or'ed in.
    template <int KB>
    __device__ __forceinline__ void scores(const short *k_lds, int b0, Scores<KB> &x) const {
        const int lane = lane_now(), r = lane & 31, h = lane >> 5;
        const unsigned ka = r * DH * 2 + ((h ^ k_swz(r)) << 4);
#pragma unroll
        for (int b = 0; b < KB; ++b) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x.s[b][i] = 0;
#pragma unroll
            for (int st = 0; st < DH / 16; ++st)
                x.s[b] = mfma32<BF>(*(const qe_s8 *)((const char *)k_lds + ((ka ^ (st & 3) << 5) + (b0 + b) * 64 * DH + (st >> 2) * 128)), q[st], x.s[b]);
        }
    }
    // The maximum that is subtracted only has to keep the powers of two in range: it follows the true one
    // when that has grown by more than 2^8, which after the first keys is rare.
    __device__ __forceinline__ void raise(float top) {
        if (__any(top > m + (float)LAG)) {
            const float mn = fmaxf(m, top), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            if (__any(m != -INFINITY)) // else nothing is summed yet
#pragma unroll
                for (int d = 0; d < DH / 32; ++d) o[d] *= f;
            l *= f;
            m = mn;
        }
    }
    template <int KB>
    __device__ __forceinline__ void exponentials(float scale, const Scores<KB> &x, Probs<KB> &p) {
        const float base = exponent_base<BF, LAG>(m);
        float sum[2] = {0, 0};
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float y = __builtin_amdgcn_exp2f(fmaf(x.s[b][i], scale, base));
                const float z = __builtin_amdgcn_exp2f(fmaf(x.s[b][i + 1], scale, base));
                sum[0] += y;
                sum[1] += z;
                p.p[b][i / 8].u[i % 8 / 2] = pack2<BF>(y, z);
            }
        l += sum[0] + sum[1];
    }
    // O^T += V^T P^T.  The 64-byte units d of the row that a lane addresses in a transposing read are one address with
    // constants, too.
    template <int KB>
    __device__ __forceinline__ void values(const short *v_lds, int b0, const Probs<KB> &p) {
        const int lane = lane_now(), h = lane >> 5, tr = (lane & 15) >> 2, el = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
        const unsigned va = (4 * h + tr) * DH * 2 + (((el >> 3) ^ v_swz<DH>(tr)) << 4) + (el & 7) * 2;
#pragma unroll
        for (int ks = 0; ks < 2 * KB; ++ks)
#pragma unroll
            for (int d = 0; d < DH / 32; ++d) {
                const unsigned vp = (va ^ (d & 3) << 6) + (b0 * 2 + ks) * 32 * DH + (d >> 2) * 256;
                const qe_s4 x = lds_tr((const short *)((const char *)v_lds + vp)), y = lds_tr((const short *)((const char *)v_lds + (vp + 16 * DH))); // 8 rows on the permutation is the same
                o[d] = mfma32<BF>(qe_s8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]}, p.p[ks / 2][ks % 2].v, o[d]);
            }
    }
};

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
    const int lane = lane_now(), r = lane & 31, h = lane >> 5;
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
    const float l = w.l + __shfl_xor(w.l, 32);
    const int row = wave_row + r;
    if (a.splits == 1) {
        if (row >= n_rows) return;
        const int tok = row / a.group, head = kvh * a.group + row - tok * a.group;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        short *out = (short *)a.out + (size_t)(begin + tok) * a.out_stride + (size_t)head * DH;
#pragma unroll
        for (int d = 0; d < DH / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                uint2 x;
                x.x = pack2<BF>(w.o[d][i] * inv, w.o[d][i + 1] * inv);
                x.y = pack2<BF>(w.o[d][i + 2] * inv, w.o[d][i + 3] * inv);
                *(uint2 *)(out + d * 32 + 2 * i + 4 * h) = x;
            }
    } else {
        const size_t at = (((size_t)tile * a.kv_heads + kvh) * a.splits + split) * BM + row - row0;
#pragma unroll
        for (int d = 0; d < DH / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *(qe_f4 *)(a.part_o + at * DH + d * 32 + 2 * i + 4 * h) = qe_f4{w.o[d][i], w.o[d][i + 1], w.o[d][i + 2], w.o[d][i + 3]};
        if (h == 0) a.part_ml[at] = make_float2(w.m, l);
    }
}

// The splits' results joined, W waves per query row: one, but for few rows over more than 8 splits a workgroup's four, each
// over every fourth split.  (The call with one wave a row and with four, of 16 and 2 heads of 256: 30 tokens after 10,000, 40
// splits, 50 and 39 us, but 1000 tokens, 4 splits, 50 and 58; of 32 and 8 heads of 128: 64 after 5200, 21 splits, 42 and 36,
// but 200 after 4000, 9 splits, 45 and 50.)
template <bool BF, int DH, int BM, int W>
__global__ __launch_bounds__(256) void k_attn_prompt_join(const QeAttnArgs a) {
    constexpr int E = DH / 64;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, item = blockIdx.x / (BM * W / 4);
    const int in_tile = blockIdx.x % (BM * W / 4) * (4 / W) + wave / W, tile = item / a.kv_heads, kvh = item % a.kv_heads;
    int seq = 0;
    for (int hi = a.n_seqs; hi - seq > 1;) {
        const int mid = (seq + hi) >> 1;
        if (qe_attn_first_tile(qe_clamped(scalar_load(a.cu + mid), 0, a.n_tokens), mid, a.group, BM) <= tile) seq = mid;
        else hi = mid;
    }
    unsigned bad = 0;
    int begin, end;
    qe_rows_of(scalar_load(a.cu + seq), scalar_load(a.cu + seq + 1), a.n_tokens, &begin, &end, &bad);
    const int local = tile - qe_attn_first_tile(begin, seq, a.group, BM);
    const int64_t row = (int64_t)local * BM + in_tile;
    // (of one row or of none with four waves a row: uniform there)
    if (local < 0 || row >= (int64_t)(end - begin) * a.group) return;
    const size_t at = ((size_t)tile * a.kv_heads + kvh) * a.splits * BM + in_tile;
    float m = -INFINITY;
    for (int s = lane; s < a.splits; s += 64) m = fmaxf(m, a.part_ml[at + (size_t)s * BM].x);
    for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
    float sum = 0, o[E];
    for (int e = 0; e < E; ++e) o[e] = 0;
#pragma unroll 4
    for (int s = wave % W; s < a.splits; s += W) {
        const float2 x = a.part_ml[at + (size_t)s * BM];
        float y[E];
        for (int e = 0; e < E; ++e) y[e] = a.part_o[(at + (size_t)s * BM) * DH + e * 64 + lane];
        const float f = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.x - m);
        if (x.y == 0.f) continue; // no key of that split
        sum += f * x.y;
        for (int e = 0; e < E; ++e) o[e] += f * y[e];
    }
    if constexpr (W == 4) {
        __shared__ float o_s[4][DH], sum_s[4];
        for (int e = 0; e < E; ++e) o_s[wave][e * 64 + lane] = o[e];
        if (lane == 0) sum_s[wave] = sum;
        __syncthreads();
        if (wave) return;
        sum = (sum_s[0] + sum_s[1]) + (sum_s[2] + sum_s[3]);
        for (int e = 0; e < E; ++e)
            o[e] = (o_s[0][e * 64 + lane] + o_s[1][e * 64 + lane]) + (o_s[2][e * 64 + lane] + o_s[3][e * 64 + lane]);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int tok = (int)(row / a.group), head = kvh * a.group + (int)(row - (int64_t)tok * a.group);
    short *out = (short *)a.out + (size_t)(begin + tok) * a.out_stride + (size_t)head * DH;
    for (int e = 0; e < E; ++e) out[e * 64 + lane] = (short)pack2<BF>(o[e] * inv, 0.f);
}

template <bool BF, int DH, int WAVES>
static hipError_t launch_waves(const QeAttnArgs &a, hipStream_t st) {
    k_attn_prompt<BF, DH, WAVES><<<dim3((unsigned)(a.tiles * a.kv_heads * a.splits)), dim3(64 * WAVES), 0, st>>>(a);
    const unsigned rows = (unsigned)(a.tiles * a.kv_heads) * (32 * WAVES);
    if (a.splits > 8 && rows <= 4096) k_attn_prompt_join<BF, DH, 32 * WAVES, 4><<<dim3(rows), dim3(256), 0, st>>>(a);
    else if (a.splits > 1) k_attn_prompt_join<BF, DH, 32 * WAVES, 1><<<dim3(rows / 4), dim3(256), 0, st>>>(a);
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
