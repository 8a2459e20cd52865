// Causal attention of packed prompts over an 8-bit paged cache.
//
// As k_attn_prompt (qe_attn_prompt.hip), whose products, softmax and split of the work these are: 32 query rows a wave, S^T = K
// Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16 from tiles in LDS.  The tiles hold the codes as 16-bit numbers, exactly: each
// wave loads its part of the next tile's codes while this one is worked on, turns them to 16 bits when its work is done,
// and writes them to the other of two buffers, so that a code is turned once for all rows of a workgroup.  With heads of 256
// the registers are full: there the codes wait in a few KB of LDS, by direct loads.  A key's scale multiplies its scores and a
// value's its probabilities (in fp16 in units of theirs: RowUnits), from one register: lane n of 16 has the scale of the n-th
// of the 16 keys in the lane's registers.  Where tiles are few, eight waves share a tile's rows, four for the even steps and four for
// the odd ones (HALVES, qe_attn_prompt8_halves), and join their sums in LDS.
#include "qe_attn_stage8.h"

//
// Bound by the matrix cores and by the vector instructions beside them, which turn codes, apply scales and make exponentials: 8192
// tokens of 16 / 2 heads of 256, e4m3, take 545 to 575 us a pass, 960 to 1010 TFLOP/s (16-bit tiles, which come by direct loads: 480 to 515); 8000 of
// 32 / 8 of 128 590 to 635 us, 820 to 880 TFLOP/s.  (Cards and runs differ by so much; figures that are set against each other, here and below, are of one
// run.)  Packed prompts of 200, 333 and 967 tokens after 0, 1700 and 0 take 54: the longest tiles' 32 steps, on a GPU half
// full.  Eight waves and 256 rows for heads of 128: 8000 tokens 613 us for 635, but 5000 of 14 / 2 185 for 158.
template <bool BF, int DH, int CT, int WAVES, int HALVES>
__global__ __launch_bounds__(64 * WAVES * HALVES, 2) void k_attn_prompt8(const QeAttn8Args x) {
    const QeAttnArgs &a = x.a;
    typedef Stage<CT, BF, DH, WAVES> ST;
    constexpr int BM = 32 * WAVES, BN = ST::BN, KB = DH == 256 ? 1 : 2;
    static_assert(BN == 32 * KB, "a tile is a step");
    __shared__ __align__(16) short k_a[HALVES][BN * DH], v_a[HALVES][BN * DH], k_b[HALVES][BN * DH], v_b[HALVES][BN * DH];
    __shared__ __align__(16) uint8_t raw_s[ST::RAW ? WAVES * HALVES * ST::RAW : 16];
    __shared__ float s_a[HALVES][2][BN], s_b[HALVES][2][BN];
    const int tid = threadIdx.x, thread_wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = HALVES == 1 ? 0 : thread_wave / WAVES, wave = thread_wave - half * WAVES;
    const int beside = x.spread ? 1 : a.splits; // splits of a tile that are begun one after the other
    const int split = blockIdx.x % beside + blockIdx.y, kvh = blockIdx.x / beside % a.kv_heads;
    const int rank = blockIdx.x / beside / a.kv_heads; // of the workgroup's tile, in the order in which they are begun
    // workgroup i looks at sequence i's offsets, for the report: where they fall, a sequence may have no tile below
    const int mine = blockIdx.x < (unsigned)a.n_seqs ? blockIdx.x : a.n_seqs - 1;
    const int mine0 = scalar_load(a.cu + mine), mine1 = scalar_load(a.cu + mine + 1);
    int cu0, cu1, kv, seq, local;
    // The longest sequence's last rows first, from a sequence for each lane and the tiles of all longer ones: 200, 333 and 967 tokens after 0, 1700 and 0 take 54 us
    // in place of 62, and 500, 60, 40, 20, 300 and 1000 after 0, 9000, 0, 3000, 0 and 0 of 16 / 2 heads of 256 133 in place of 170.
    if (a.n_seqs <= 64) {
        const int lane = lane_now(), i = lane < a.n_seqs ? lane : a.n_seqs - 1;
        const int c0 = a.cu[i], c1 = a.cu[i + 1], length = a.kv_len[i];
        unsigned any = 0;
        int begin, end, before = 0;
        qe_rows_of(c0, c1, a.n_tokens, &begin, &end, &any);
        const int n = ((end - begin) * a.group + BM - 1) / BM;
        for (int j = 0; j < a.n_seqs; ++j) {
            const int other = __builtin_amdgcn_readlane(length, j);
            before += other > length || (other == length && j < lane) ? __builtin_amdgcn_readlane(n, j) : 0;
        }
        const uint64_t here = __ballot(lane < a.n_seqs && rank >= before && rank < before + n);
        seq = here ? __builtin_ctzll(here) : 0;
        cu0 = __builtin_amdgcn_readlane(c0, seq), cu1 = __builtin_amdgcn_readlane(c1, seq), kv = __builtin_amdgcn_readlane(length, seq);
        local = here ? __builtin_amdgcn_readlane(before + n, seq) - 1 - rank : -1;
    } else { // the last sequence's last rows first
        const int place = a.tiles - 1 - rank;
        seq = 0;
        for (int hi = a.n_seqs; hi - seq > 1;) { // the last sequence whose first tile is not behind this one
            const int mid = (seq + hi) >> 1;
            if (qe_attn_first_tile(qe_clamped(scalar_load(a.cu + mid), 0, a.n_tokens), mid, a.group, BM) <= place) seq = mid;
            else hi = mid;
        }
        cu0 = scalar_load(a.cu + seq), cu1 = scalar_load(a.cu + seq + 1), kv = scalar_load(a.kv_len + seq);
        local = place - qe_attn_first_tile(qe_clamped(cu0, 0, a.n_tokens), seq, a.group, BM);
    }
    unsigned bad_len = 0;
    int begin, end;
    qe_rows_of(cu0, cu1, a.n_tokens, &begin, &end, &bad_len);
    const int tile = qe_attn_first_tile(begin, seq, a.group, BM) + local;
    int len = qe_checked(kv, 0, a.max_pages << a.page_log2, 0, &bad_len);
    if (bad_len) len = 0; // no row has a position: zeros
    if ((bad_len || qe_bad_offsets(mine0, mine1, a.n_tokens)) && tid == 0) report(a.err, QE_BAD_LENGTH);
    const int n_rows = (end - begin) * a.group;
    if (local < 0 || (int64_t)local * BM >= n_rows) return; // uniform: no row of the sequence
    const int row0 = local * BM, first = len - (end - begin); // first: position of the sequence's first row
    const int32_t *table = a.table + (size_t)seq * a.table_stride;

    const int wave_row = row0 + wave * 32, wave_end = wave_row + 32 < n_rows ? wave_row + 32 : n_rows;
    const int wave_keys = wave_row < n_rows ? first + (wave_end - 1) / a.group + 1 : 0, wave_clear = first + wave_row / a.group + 1;
    const int steps = qe_attn_tile_steps(len, begin, end, row0, a.group, BM, BN), splits = qe_attn_tile_splits(steps, a.steps, a.splits);
    if (split >= splits) return;
    int lo, hi;
    qe_split_range(steps, splits, split, &lo, &hi);

    ST stage;
    uint8_t *raw = raw_s + thread_wave * ST::RAW;
    int page = 0; // of the wave's part of the tile after the one that is loaded
    const int t0 = lo + half; // the half's first step
    if (t0 < hi) {
        page = page_of<BN, WAVES>(a, table, t0 * BN, len, wave);
        stage.issue(x, page, kvh, t0 * BN, len, wave, raw);
        page = page_of<BN, WAVES>(a, table, (t0 + HALVES) * BN, len, wave);
    }
    Rows<BF, DH> w;
    RowUnits<BF> units;
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
    if (lo < hi) {
        const int lost = lost_pages<64 * WAVES * HALVES>(a, table, (len + (1 << a.page_log2) - 1) >> a.page_log2, tid);
        if (__syncthreads_or(lost)) { // (it waits for what is on its way to LDS, too)
            if (tid == 0) report(a.err, QE_BAD_PAGE);
            hi = lo; // no key: zeros
        }
    }
    // Q and the first tile have come, on every way to the loop: else the compiler has each step wait for Q, and with it for the
    // loads in flight.
    __builtin_amdgcn_s_waitcnt(0x0f70);
    if (t0 < hi) {
        stage.land(t0 * BN, len, wave, raw, k_a[half], v_a[half], s_a[half][0], s_a[half][1]);
        if (t0 + HALVES < hi) stage.issue(x, page, kvh, (t0 + HALVES) * BN, len, wave, raw);
        page = page_of<BN, WAVES>(a, table, (t0 + 2 * HALVES) * BN, len, wave);
    }
    const bool few = n_rows < BM && steps <= 8; // few rows of few keys: sum_rounded
    auto work = [&](int t, const short *k_lds, const short *v_lds, const float (*s_lds)[BN], short *k_next, short *v_next, float (*s_next)[BN]) {
        lds_barrier(); // the tile is there, and no wave reads the other buffers any more
        const int k0 = t * BN;
        if ((HALVES == 1 || t < hi) && k0 < wave_keys) {
            const int lane = lane_now(), at = 8 * (lane >> 2 & 3) + 4 * (lane >> 5) + (lane & 3);
            Scores<KB> s;
            w.scores(k_lds, 0, s);
            schedule<4, KB * DH / 16, 1>();
#pragma unroll
            for (int b = 0; b < KB; ++b) scaled(s.s[b], s_lds[0][b * 32 + at]);
            const bool cut = k0 + BN > wave_clear;
            // The last key that the row attends to, counted from the lane's first; made anew in each branch, since of one number the
            // compiler makes all comparisons in every step (637 us for 614 at 8000 tokens).
            auto limit = [&] {
                int x = w.place - k0 - 4 * (lane >> 5);
                asm volatile("" : "+v"(x));
                return x;
            };
            if (cut) s.mask(limit());
            w.raise(s.top() * a.scale_log2);
            if constexpr (!BF) {
                unsigned top = 0;
                if (cut) {
                    const int last = limit();
#pragma unroll
                    for (int b = 0; b < KB; ++b) top = max(top, greatest_seen(size_bits(s_lds[1][b * 32 + at]), b, last));
                    const auto halves = __builtin_amdgcn_permlane32_swap(top, top, false, false);
                    top = max(halves[0], halves[1]);
                } else {
                    top = greatest(size_bits(s_lds[1][lane & (BN - 1)]));
                }
                units.raise(top, w);
            }
            Probs<KB> p;
            w.weigh(a.scale_log2, BF ? 0.f : units.log2, s);
#pragma unroll
            for (int b = 0; b < KB; ++b) scaled(s.s[b], s_lds[1][b * 32 + at]);
            if (cut) s.clear(limit()); // a scale that is not finite reaches the rows that attend to its position
            s.template pack<BF>(p);
            if (few || (cut && k0 == 0)) // (in all cut tiles it would cost 4 to 8 % of 1000 tokens, for few rows of many keys 13 %)
                sum_rounded(w.l, s, p, s_lds[1] + at, units);
            w.values(v_lds, 0, p);
            schedule<3, KB * DH / 16, 2>();
        }
        if (t + HALVES < hi) {
            stage.land(k0 + HALVES * BN, len, wave, raw, k_next, v_next, s_next[0], s_next[1]);
            if (t + 2 * HALVES < hi) stage.issue(x, page, kvh, k0 + 2 * HALVES * BN, len, wave, raw);
            page = page_of<BN, WAVES>(a, table, k0 + 3 * HALVES * BN, len, wave);
        }
    };
    for (int t = lo; t < hi; t += 2 * HALVES) { // both halves pass all barriers
        work(t + half, k_a[half], v_a[half], s_a[half], k_b[half], v_b[half], s_b[half]);
        if (t + HALVES < hi) work(t + HALVES + half, k_b[half], v_b[half], s_b[half], k_a[half], v_a[half], s_a[half]);
    }
    if constexpr (!BF) w.times(units.unit());
    if constexpr (HALVES == 2) { // the second half's sums, through the tiles' LDS
        constexpr int LOT = 64 * WAVES * 16, LOTS = HALVES * BN * DH / 2 / LOT; // floats of 32 columns; these that an array has room for
        static_assert(LOTS >= 1 && 4 * LOTS * 32 >= DH, "room for all columns");
        __shared__ float ml_s[2][64 * WAVES];
        float *const room[4] = {(float *)k_a, (float *)v_a, (float *)k_b, (float *)v_b};
        const int at = wave * 64 + (tid & 63);
        lds_barrier(); // no wave reads a tile any more
        if (half) {
#pragma unroll
            for (int d = 0; d < DH / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) room[d / LOTS][d % LOTS * LOT + i * 64 * WAVES + at] = w.o[d][i];
            ml_s[0][at] = w.m;
            ml_s[1][at] = w.l;
        }
        lds_barrier();
        if (half) return;
        const float m1 = ml_s[0][at], m = fmaxf(w.m, m1);
        const float f0 = w.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w.m - m), f1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - m);
        w.l = w.l * f0 + ml_s[1][at] * f1;
        w.m = m;
#pragma unroll
        for (int d = 0; d < DH / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) w.o[d][i] = w.o[d][i] * f0 + room[d / LOTS][d % LOTS * LOT + i * 64 * WAVES + at] * f1;
    }
    w.template finish<BM>(a, begin, n_rows, row0, wave_row, tile, kvh, split, splits == 1);
}

// The splits' results joined, of the tiles that have several: a workgroup for ROWS of a tile's rows and a key-value head, each wave
// one row after the other, all of a row's reads (and the next rows') in flight.
template <bool BF, int DH, int BM, int BN, int ROWS>
__global__ __launch_bounds__(256) void k_attn_prompt8_join(const QeAttnArgs a) {
    constexpr int E = DH / 64;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, item = blockIdx.x / (BM / ROWS), tile = item / a.kv_heads, kvh = item % a.kv_heads;
    int seq = 0;
    for (int hi = a.n_seqs; hi - seq > 1;) {
        const int mid = (seq + hi) >> 1;
        if (qe_attn_first_tile(qe_clamped(scalar_load(a.cu + mid), 0, a.n_tokens), mid, a.group, BM) <= tile) seq = mid;
        else hi = mid;
    }
    unsigned bad = 0;
    int begin, end;
    qe_rows_of(scalar_load(a.cu + seq), scalar_load(a.cu + seq + 1), a.n_tokens, &begin, &end, &bad);
    const int len = qe_checked(scalar_load(a.kv_len + seq), 0, a.max_pages << a.page_log2, 0, &bad);
    const int local = tile - qe_attn_first_tile(begin, seq, a.group, BM), n_rows = (end - begin) * a.group;
    if (local < 0 || (int64_t)local * BM >= n_rows) return;
    const int splits = qe_attn_tile_splits(qe_attn_tile_steps(bad ? 0 : len, begin, end, local * BM, a.group, BM, BN), a.steps, a.splits);
    if (splits <= 1) return; // its one workgroup has written the rows
    const size_t at0 = ((size_t)tile * a.kv_heads + kvh) * a.splits * BM;
    const int first = blockIdx.x % (BM / ROWS) * ROWS, left = n_rows - local * BM - first;
#pragma unroll 2
    for (int r = wave; r < ROWS; r += 4) {
        if (r >= left) return;
        const size_t at = at0 + first + r;
        float m = -INFINITY, sum = 0, o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = 0;
        for (int s = lane; s < splits; s += 64) m = fmaxf(m, a.part_ml[at + (size_t)s * BM].x);
        for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
#pragma unroll 4
        for (int s = 0; s < splits; ++s) {
            const float2 x = a.part_ml[at + (size_t)s * BM];
            float y[E];
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = a.part_o[(at + (size_t)s * BM) * DH + e * 64 + lane];
            const float f = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.x - m);
            const bool any = x.y != 0.f; // else no key of that split
            sum += any ? f * x.y : 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += any ? f * y[e] : 0.f;
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int row = local * BM + first + r, tok = row / a.group, head = kvh * a.group + row - tok * a.group;
        short *out = (short *)a.out + (size_t)(begin + tok) * a.out_stride + (size_t)head * DH;
#pragma unroll
        for (int e = 0; e < E; ++e) out[e * 64 + lane] = (short)pack2<BF>(o[e] * inv, 0.f);
    }
}

template <bool BF, int DH, int CT, int WAVES, int HALVES>
static hipError_t launch_waves8(const QeAttn8Args &x, hipStream_t st) {
    constexpr int BM = 32 * WAVES, BN = Stage<CT, BF, DH, WAVES>::BN;
    const unsigned items = (unsigned)(x.a.tiles * x.a.kv_heads);
    k_attn_prompt8<BF, DH, CT, WAVES, HALVES><<<x.spread ? dim3(items, x.a.splits) : dim3(items * x.a.splits), dim3(64 * WAVES * HALVES), 0, st>>>(x);
    // few tiles: fewer rows a workgroup
    if (x.a.splits > 1 && items >= 128) k_attn_prompt8_join<BF, DH, BM, BN, 32><<<dim3(items * (BM / 32)), dim3(256), 0, st>>>(x.a);
    else if (x.a.splits > 1) k_attn_prompt8_join<BF, DH, BM, BN, 4><<<dim3(items * (BM / 4)), dim3(256), 0, st>>>(x.a);
    return hipGetLastError();
}
template <bool BF, int CT>
static hipError_t launch_prompt8(const QeAttn8Args &x, int head_dim, int bm, bool halves, hipStream_t st) {
    if (head_dim == 64) return halves ? launch_waves8<BF, 64, CT, 4, 2>(x, st) : launch_waves8<BF, 64, CT, 4, 1>(x, st);
    if (head_dim == 128) return halves ? launch_waves8<BF, 128, CT, 4, 2>(x, st) : launch_waves8<BF, 128, CT, 4, 1>(x, st);
    if (bm == 256) return launch_waves8<BF, 256, CT, 8, 1>(x, st);
    return launch_waves8<BF, 256, CT, 4, 1>(x, st);
}

hipError_t qe_launch_attn_prompt8(const QeAttn8Args &x, int head_dim, int type, int cache_type, int bm, bool halves, hipStream_t st) {
    if (type == QE_BF16) return cache_type == QE_I8 ? launch_prompt8<true, QE_I8>(x, head_dim, bm, halves, st) : launch_prompt8<true, QE_F8>(x, head_dim, bm, halves, st);
    return cache_type == QE_I8 ? launch_prompt8<false, QE_I8>(x, head_dim, bm, halves, st) : launch_prompt8<false, QE_F8>(x, head_dim, bm, halves, st);
}
