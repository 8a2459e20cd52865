// Attention of single tokens whose sequences share their beginnings: a shared key and value is read once for all rows of its
// group, not once a sequence.
//
// Three launches.  k_shared_prefix: 128 rows of a group (its sequences' heads of one key-value head) over a split of the shared
// positions, by the products of a prompt (qe_attn_rows.h) without a causal mask.  k_shared_own: a sequence's own positions, by
// those of k_attn_decode.  Both leave unnormalised partial results with their maximum and sum, in 32 bits, and k_shared_join
// joins a row's.  Positions are read through the table of the group's first sequence below the group's length, and
// through a sequence's own from there on.
#include "qe_attn_stage8.h"

// ---- groups --------------------------------------------------------------------------------------------
// Sequence seq's group: its first sequence and how many positions are shared (0: it is of no group).  False where the offsets
// at that place are none, or the length is out of range.
__device__ __forceinline__ bool group_of(const QeSharedArgs &y, int seq, int *first, int *shared) {
    const QeAttnArgs &a = y.x.a;
    int lo = 0;
    for (int hi = y.n_groups; hi - lo > 1;) {
        const int mid = (lo + hi) >> 1;
        if (scalar_load(y.seqs + mid) <= seq) lo = mid;
        else hi = mid;
    }
    const int before = scalar_load(y.seqs + (lo ? lo - 1 : 0)), begin = scalar_load(y.seqs + lo), end = scalar_load(y.seqs + lo + 1);
    const int after = scalar_load(y.seqs + (lo + 2 <= y.n_groups ? lo + 2 : y.n_groups)), n = scalar_load(y.prefix + lo);
    *first = begin;
    *shared = 0;
    if (before > begin || end > after || qe_bad_offsets(begin, end, a.n_seqs)) return false;
    if (seq < begin || seq >= end) return true;
    if (n < 0 || n > a.max_pages << a.page_log2) return false;
    *shared = n;
    return true;
}
// A sequence's own positions [*start, *len); false (and none) where its length, or its group, is bad.
__device__ __forceinline__ bool own_positions(const QeSharedArgs &y, int seq, int *start, int *len) {
    const QeAttnArgs &a = y.x.a;
    int first;
    *len = scalar_load(a.kv_len + seq);
    const bool known = group_of(y, seq, &first, start);
    if (known && *len >= *start && *len <= a.max_pages << a.page_log2) return true;
    *len = *start = 0;
    return false;
}
// 32-key steps from the one that start lies in on
__device__ __forceinline__ int own_length(int start, int len) { return len > start ? len - (start & -QE_ATTN_TILE) : 0; }

template <int DH>
constexpr int shared_step() { return DH == 256 ? 32 : 64; } // keys of a prefix workgroup's step

// A partial result's place: those of a row are together, the prefix's first.
__device__ __forceinline__ size_t part_of(const QeSharedArgs &y, int seq, int head, int split) {
    return ((size_t)(seq - y.seq0) * y.x.a.q_heads + head) * (y.psplits + y.x.a.splits) + split;
}

// ---- the shared positions ---------------------------------------------------------------------------------
template <bool BF, int DH, int CT>
__global__ __launch_bounds__(256, 2) void k_shared_prefix(const QeSharedArgs y) {
    const QeAttnArgs &a = y.x.a;
    constexpr bool CODES = CT != QE_CACHE16;
    typedef Stage<CODES ? CT : QE_I8, BF, DH, 4> ST;
    constexpr int BM = QE_ATTN_SHARED_BM, BN = shared_step<DH>(), KB = BN / 32, PART = BN / 4;
    static_assert(ST::BN == BN, "a stage is a step");
    __shared__ __align__(16) short k_a[BN * DH], v_a[BN * DH], k_b[BN * DH], v_b[BN * DH];
    __shared__ __align__(16) uint8_t raw_s[CODES && ST::WAIT_IN_LDS ? 2 * BN * DH : 16];
    __shared__ float s_a[2][BN], s_b[2][BN];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int split = blockIdx.x % y.psplits, kvh = blockIdx.x / y.psplits % a.kv_heads, tile = blockIdx.x / y.psplits / a.kv_heads;
    // the group: the last one whose first tile is not behind this one, among this launch's sequences
    int g = 0;
    for (int hi = y.n_groups; hi - g > 1;) {
        const int mid = (g + hi) >> 1;
        if (qe_attn_first_tile(qe_clamped(scalar_load(y.seqs + mid), y.seq0, y.seq1) - y.seq0, mid, a.group, BM) <= tile) g = mid;
        else hi = mid;
    }
    const int g0 = scalar_load(y.seqs + g), g1 = scalar_load(y.seqs + g + 1), len = scalar_load(y.prefix + g);
    if (qe_bad_offsets(g0, g1, a.n_seqs) || len <= 0 || len > a.max_pages << a.page_log2) return; // k_shared_join reports it
    const int begin = qe_clamped(g0, y.seq0, y.seq1), end = qe_clamped(g1, y.seq0, y.seq1);
    const int row0 = (tile - qe_attn_first_tile(begin - y.seq0, g, a.group, BM)) * BM, n_rows = (end - begin) * a.group;
    const int per = qe_attn_shared_per(len, BN, y.psplits), lo = split * per, steps = (len + BN - 1) / BN, hi = lo + per < steps ? lo + per : steps;
    if (row0 < 0 || row0 >= n_rows || lo >= hi) return; // uniform
    const int32_t *table = a.table + (size_t)g0 * a.table_stride;
    const int wave_row = row0 + wave * 32, row = wave_row + (tid & 31);
    const bool there = row < n_rows;
    const int seq = begin + (there ? row / a.group : 0), head = kvh * a.group + (there ? row % a.group : 0);

    unsigned bad = 0; // a page of the wave's that is none
    ST stage;
    uint8_t *raw = raw_s + (CODES && ST::WAIT_IN_LDS ? wave * (2 * PART * DH) : 0);
    auto load = [&](int t, short *k_lds, short *v_lds) { // the wave's part of tile t
        const int k0 = t * BN, page = page_of<BN, 4>(a, table, k0, len, wave);
        bad |= (unsigned)page >= a.n_pages;
        if constexpr (CODES) {
            stage.issue(y.x, page, kvh, k0, len, wave, raw);
        } else {
            load_part<DH, BN, 4, true>(a, page, kvh, k0, len, wave, k_lds);
            load_part<DH, BN, 4, false>(a, page, kvh, k0, len, wave, v_lds);
        }
    };
    load(lo, k_a, v_a);
    Rows<BF, DH> w;
    Units units;
    {
        const short *q = (const short *)a.q + (size_t)seq * a.q_stride + (size_t)head * DH + (tid >> 5 & 1) * 8;
#pragma unroll
        for (int s = 0; s < DH / 16; ++s) w.q[s] = there ? *(const qe_s8 *)(q + s * 16) : qe_s8{};
        w.m = -INFINITY;
        w.l = 0;
#pragma unroll
        for (int d = 0; d < DH / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) w.o[d][i] = 0;
    }
    if constexpr (CODES) {
        stage.land(lo * BN, len, wave, raw, k_a, v_a, s_a[0], s_a[1]);
        if (lo + 1 < hi) load(lo + 1, nullptr, nullptr);
    }
    auto work = [&](int t, const short *k_lds, short *v_lds, const float (*s_lds)[BN], short *k_next, short *v_next, float (*s_next)[BN]) {
        const int k0 = t * BN;
        if constexpr (!CODES) {
            __builtin_amdgcn_s_waitcnt(0x0f70);
            if (k0 + BN > len) // rows behind the end hold anything: a probability of 0 times NaN is NaN
                for (int i = lane_now(); i < PART * (DH / 8); i += 64)
                    if (k0 + wave * PART + i / (DH / 8) >= len) *(qe_s8 *)(v_lds + wave * PART * DH + i * 8) = qe_s8{};
        }
        lds_barrier(); // the tile is there, and no wave reads the other buffers any more
        if (!CODES && t + 1 < hi) load(t + 1, k_next, v_next);
        if (wave_row < n_rows) {
            const int lane = lane_now(), at = 8 * (lane >> 2 & 3) + 4 * (lane >> 5) + (lane & 3);
            Scores<KB> s;
            w.scores(k_lds, 0, s);
            schedule<4, KB * DH / 16, 1>();
            if constexpr (CODES)
#pragma unroll
                for (int b = 0; b < KB; ++b) scaled(s.s[b], s_lds[0][b * 32 + at]);
            if (k0 + BN > len) s.mask(len - 1 - k0 - 4 * (lane >> 5));
            w.raise(s.top() * a.scale_log2);
            Probs<KB> p;
            if constexpr (CODES) {
                if constexpr (!BF) w.times(units.raise(s_lds[1][lane & (BN - 1)]));
                w.weigh(a.scale_log2, s);
#pragma unroll
                for (int b = 0; b < KB; ++b) scaled(s.s[b], BF ? s_lds[1][b * 32 + at] : s_lds[1][b * 32 + at] * units.inverse);
                s.template pack<BF>(p);
            } else {
                w.exponentials(a.scale_log2, s, p);
            }
            w.values(v_lds, 0, p);
            schedule<3, KB * DH / 16, 2>();
        }
        if constexpr (CODES)
            if (t + 1 < hi) {
                stage.land(k0 + BN, len, wave, raw, k_next, v_next, s_next[0], s_next[1]);
                if (t + 2 < hi) load(t + 2, nullptr, nullptr);
            }
    };
    for (int t = lo; t < hi; t += 2) {
        work(t, k_a, v_a, s_a, k_b, v_b, s_b);
        if (t + 1 < hi) work(t + 1, k_b, v_b, s_b, k_a, v_a, s_a);
    }
    if constexpr (CODES && !BF) w.times(units.unit);
    bad = __syncthreads_or(bad);
    if (bad && tid == 0) report(a.err, QE_BAD_PAGE);
    const float sum = w.l + __shfl_xor(w.l, 32);
    if (!there) return;
    const int h = lane_now() >> 5;
    const size_t at = part_of(y, seq, head, split);
#pragma unroll
    for (int d = 0; d < DH / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            *(qe_f4 *)(a.part_o + at * DH + d * 32 + 2 * i + 4 * h) = qe_f4{w.o[d][i], w.o[d][i + 1], w.o[d][i + 2], w.o[d][i + 3]};
    if (h == 0) a.part_ml[at] = make_float2(w.m, bad ? -1.f : sum);
}

// ---- a sequence's own positions -----------------------------------------------------------------------------
// As k_attn_decode and k_attn_decode8, from a position on that may lie within a step.
template <bool BF, int DH, int CT>
__global__ __launch_bounds__(256, DH == 256 ? 2 : 3) void k_shared_own(const QeSharedArgs y) {
    const QeAttnArgs &a = y.x.a;
    constexpr bool CODES = CT != QE_CACHE16;
    constexpr int SIZE = CODES ? 1 : 2;                // bytes of an element
    constexpr int CH = DH * SIZE / 16, ROWS = 64 / CH; // 16-byte chunks of a row, rows of one direct load
    constexpr int KL = DH * SIZE / 64, DB = DH / 16;
    constexpr int LDS = QE_ATTN_TILE * DH; // shorts of a wave: room for 16 heads x DH floats
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    __shared__ __align__(16) short lds[4][LDS];
    __shared__ float2 ml[4][16];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, col = lane & 15, c = lane >> 4;
    const int split = blockIdx.x % a.splits, item = blockIdx.x / a.splits, seq = y.seq0 + item / a.kv_heads, kvh = item % a.kv_heads;
    const short *q = (const short *)a.q + (size_t)seq * a.q_stride + ((size_t)kvh * a.group + col) * DH;
    qe_s8 qf[DH / 32]; // in the order of the codes (k_attn_decode8), or of K
#pragma unroll
    for (int s = 0; s < DH / 32; ++s) qf[s] = col < a.group ? *(const qe_s8 *)(q + (CODES ? s / 2 * 64 + c * 16 + s % 2 * 8 : s * 32 + c * 8)) : qe_s8{};
    int start, len;
    own_positions(y, seq, &start, &len);
    const int own = own_length(start, len), base0 = start & -QE_ATTN_TILE;
    const int steps = qe_attn_decode_steps(own, a.steps, a.splits);
    if (split >= qe_attn_decode_active(own, steps)) return;
    const int32_t *table = a.table + (size_t)seq * a.table_stride;
    const int tiles = (own + QE_ATTN_TILE - 1) / QE_ATTN_TILE, lo = split * steps, hi = lo + steps < tiles ? lo + steps : tiles;
    unsigned bad = 0;
    qe_f4 acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = qe_f4{0, 0, 0, 0};
    float m = -INFINITY, l = 0;
    Units units;
    uint8_t *vb = (uint8_t *)lds[wave];
    const int tr_key = CODES ? 4 * c + (col >> 1 & 3) + (col & 8) * 2 : 4 * c + (col >> 2);
    auto swz = [](int r) { return CODES ? swz8<DH>(r) : v_swz<DH>(r); };
    for (int t = lo + wave; t < hi; t += 4) {
        const int k0 = base0 + t * QE_ATTN_TILE;
        // 16 positions that all lie before the first, or behind the last, may have no page: any of the sequence's own does
        const int p0 = k0 + 16 > start ? k0 : start & -16, p1 = k0 + 16 < len ? k0 + 16 : p0;
        const size_t r0 = sub_row(a, table, kvh, p0, &bad), r1 = sub_row(a, table, kvh, p1, &bad);
        const uint8_t *kp0 = (const uint8_t *)a.kc + (r0 + col) * DH * SIZE + c * 16, *kp1 = (const uint8_t *)a.kc + (r1 + col) * DH * SIZE + c * 16;
        u4 kr[2][KL];
#pragma unroll
        for (int s = 0; s < KL; ++s) kr[0][s] = *(const u4 *)(kp0 + s * 64);
#pragma unroll
        for (int s = 0; s < KL; ++s) kr[1][s] = *(const u4 *)(kp1 + s * 64);
        float ks = 0, vs = 0;
        if constexpr (CODES) {
            const size_t sr = (col & 4 ? r1 : r0) + 4 * c + (col & 3);
            ks = y.x.ks[sr], vs = y.x.vs[sr];
        }
#pragma unroll
        for (int i = 0; i < QE_ATTN_TILE / ROWS; ++i) {
            const int row = i * ROWS + lane / CH, ch = (lane % CH) ^ swz(row);
            load_lds16_from((const uint8_t *)a.vc + (i * ROWS < 16 ? r0 : r1) * DH * SIZE, 16 * DH * SIZE, (row & 15) * DH * SIZE + ch * 16, 0, vb + i * 1024);
        }
        __builtin_amdgcn_sched_barrier(0); // all loads are under way before the first is waited for
        qe_f4 s[2] = {qe_f4{0, 0, 0, 0}, qe_f4{0, 0, 0, 0}};
#pragma unroll
        for (int st = 0; st < KL; ++st) {
            if constexpr (CODES) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    s[0] = mfma16<BF>(elements_of<CT, BF>(kr[0][st][2 * h], kr[0][st][2 * h + 1]), qf[2 * st + h], s[0]);
                    s[1] = mfma16<BF>(elements_of<CT, BF>(kr[1][st][2 * h], kr[1][st][2 * h + 1]), qf[2 * st + h], s[1]);
                }
            } else {
                s[0] = mfma16<BF>(__builtin_bit_cast(qe_s8, kr[0][st]), qf[st], s[0]);
                s[1] = mfma16<BF>(__builtin_bit_cast(qe_s8, kr[1][st]), qf[st], s[1]);
            }
        }
        if constexpr (CODES) {
            s[0] = qe_f4{s[0][0] * of_lane<0>(ks), s[0][1] * of_lane<1>(ks), s[0][2] * of_lane<2>(ks), s[0][3] * of_lane<3>(ks)};
            s[1] = qe_f4{s[1][0] * of_lane<4>(ks), s[1][1] * of_lane<5>(ks), s[1][2] * of_lane<6>(ks), s[1][3] * of_lane<7>(ks)};
        }
        const bool cut = k0 < start || k0 + QE_ATTN_TILE > len;
        auto outside = [&](int key) { return k0 + key < start || k0 + key >= len; };
        if (cut) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (outside(4 * c + i)) s[0][i] = -INFINITY;
                if (outside(16 + 4 * c + i)) s[1][i] = -INFINITY;
            }
        }
        float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                          fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        if (__any(top > m)) {
            const float mn = fmaxf(m, top), f = m == -INFINITY ? 0.f : exp2f((m - mn) * a.scale_log2);
#pragma unroll
            for (int d = 0; d < DB; ++d) acc[d] *= f;
            l *= f;
            m = mn;
        }
        if constexpr (CODES && !BF) {
            const float f = units.raise(cut && outside((col & 4 ? 16 : 0) + 4 * c + (col & 3)) ? 0.f : vs);
            if (f != 1.f)
#pragma unroll
                for (int d = 0; d < DB; ++d) acc[d] *= f;
            vs *= units.inverse;
        }
        const float base = exponent_base<BF, Rows<BF, DH>::LAG>(m * a.scale_log2); // as large as the prefix's are kept
        float p[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            p[i] = __builtin_amdgcn_exp2f(fmaf(s[0][i], a.scale_log2, base));
            p[4 + i] = __builtin_amdgcn_exp2f(fmaf(s[1][i], a.scale_log2, base));
        }
        l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        if constexpr (CODES) {
            p[0] *= of_lane<0>(vs), p[1] *= of_lane<1>(vs), p[2] *= of_lane<2>(vs), p[3] *= of_lane<3>(vs);
            p[4] *= of_lane<4>(vs), p[5] *= of_lane<5>(vs), p[6] *= of_lane<6>(vs), p[7] *= of_lane<7>(vs);
            if (cut) { // a scale there may be anything
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (outside(4 * c + i)) p[i] = 0;
                    if (outside(16 + 4 * c + i)) p[4 + i] = 0;
                }
            }
        }
        union {
            unsigned u[4];
            qe_s8 v;
        } pf;
#pragma unroll
        for (int i = 0; i < 4; ++i) pf.u[i] = pack2<BF>(p[2 * i], p[2 * i + 1]);
        __builtin_amdgcn_s_waitcnt(0x0f70); // the direct loads have landed (vmcnt 0)
        if (CT != QE_I8 && cut) {            // V there may be anything: a probability of 0 times NaN is NaN
            for (int i = lane; i < QE_ATTN_TILE * CH; i += 64)
                if (outside(i / CH)) *(uint4 *)(vb + i * 16) = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            if constexpr (CODES) {
                const uint2 v = lds_tr8(vb + tr_key * DH + ((d ^ swz(tr_key)) << 4) + (col & 1) * 8);
                acc[d] = mfma16<BF>(elements_of<CT, BF>(v.x, v.y), pf.v, acc[d]);
            } else {
                const int el = d * 16 + (col & 3) * 4, at = (((el >> 3) ^ swz(tr_key)) << 3) + (el & 7); // 16 rows on the permutation is the same
                const qe_s4 x = lds_tr((const short *)vb + tr_key * DH + at), z = lds_tr((const short *)vb + (tr_key + 16) * DH + at);
                acc[d] = mfma16<BF>(qe_s8{x[0], x[1], x[2], x[3], z[0], z[1], z[2], z[3]}, pf.v, acc[d]);
            }
        }
    }
    if constexpr (CODES && !BF)
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] *= units.unit;
    // the four waves' results joined (as in finish_decode), and left as a partial one
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (lane < 16) ml[wave][lane] = make_float2(m, l);
    float *o = (float *)lds[wave];
#pragma unroll
    for (int d = 0; d < DB; ++d) *(qe_f4 *)(o + col * DH + ((d * 4 + c) ^ col) * 4) = acc[d];
    bad = __syncthreads_or(bad);
    if (bad && tid == 0) report(a.err, QE_BAD_PAGE);
    for (int i = tid; i < a.group * (DH / 4); i += 256) {
        const int h = i / (DH / 4), d = i % (DH / 4) * 4;
        float top = ml[0][h].x;
#pragma unroll
        for (int w = 1; w < 4; ++w) top = fmaxf(top, ml[w][h].x);
        float sum = 0;
        qe_f4 r = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float2 x = ml[w][h];
            const float f = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((x.x - top) * a.scale_log2);
            const qe_f4 v = *(const qe_f4 *)((const float *)lds[w] + h * DH + ((d / 4) ^ h) * 4);
            const bool any = x.y != 0.f; // else a wave without keys
            sum += any ? f * x.y : 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] += any ? f * v[j] : 0.f;
        }
        const size_t at = part_of(y, seq, kvh * a.group + h, y.psplits + split);
        *(qe_f4 *)(a.part_o + at * DH + d) = r;
        if (d == 0) a.part_ml[at] = make_float2(top * a.scale_log2, bad ? -1.f : sum);
    }
}

// ---- a row's partial results joined: a wave a row -----------------------------------------------------------
template <bool BF, int DH>
__global__ __launch_bounds__(256) void k_shared_join(const QeSharedArgs y) {
    const QeAttnArgs &a = y.x.a;
    constexpr int E = DH / 64;
    // all groups' offsets are looked at, for the report: those that are wrong may hold no sequence
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < y.n_groups; i += (int64_t)gridDim.x * 256)
        if (qe_bad_offsets(y.seqs[i], y.seqs[i + 1], a.n_seqs) || y.prefix[i] < 0 || y.prefix[i] > a.max_pages << a.page_log2) report(a.err, QE_BAD_LENGTH);
    const int lane = threadIdx.x & 63, row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (row >= (y.seq1 - y.seq0) * a.q_heads) return;
    const int seq = y.seq0 + row / a.q_heads, head = row % a.q_heads;
    int start, len;
    const bool good = own_positions(y, seq, &start, &len);
    if (!good && lane == 0) report(a.err, QE_BAD_LENGTH);
    const int own = own_length(start, len), np = qe_attn_shared_active(start, shared_step<DH>(), y.psplits);
    const int n = np + qe_attn_decode_active(own, qe_attn_decode_steps(own, a.steps, a.splits));
    const size_t at = part_of(y, seq, head, 0);
    const int gap = y.psplits - np; // places of splits without keys
    float m = -INFINITY;
    bool bad = false;
    for (int s = lane; s < n; s += 64) {
        const float2 x = a.part_ml[at + s + (s < np ? 0 : gap)];
        m = fmaxf(m, x.x);
        bad |= x.y < 0.f;
    }
    for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
    bad = __any(bad);
    float sum = 0, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0;
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
        const size_t i = at + s + (s < np ? 0 : gap);
        const float2 x = a.part_ml[i];
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = a.part_o[i * DH + e * 64 + lane];
        const float f = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.x - m);
        if (x.y == 0.f) continue;
        sum += f * x.y;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += f * v[e];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    short *out = (short *)a.out + (size_t)seq * a.out_stride + (size_t)head * DH;
#pragma unroll
    for (int e = 0; e < E; ++e) out[e * 64 + lane] = bad ? 0 : (short)pack2<BF>(o[e] * inv, 0.f);
}

template <bool BF, int DH, int CT>
static hipError_t launch_shared(const QeSharedArgs &y, hipStream_t st) {
    const QeAttnArgs &a = y.x.a;
    const int n = y.seq1 - y.seq0;
    k_shared_prefix<BF, DH, CT><<<dim3((unsigned)(a.tiles * a.kv_heads * y.psplits)), dim3(256), 0, st>>>(y);
    k_shared_own<BF, DH, CT><<<dim3((unsigned)(n * a.kv_heads * a.splits)), dim3(256), 0, st>>>(y);
    k_shared_join<BF, DH><<<dim3((unsigned)((n * a.q_heads + 3) / 4)), dim3(256), 0, st>>>(y);
    return hipGetLastError();
}
template <bool BF, int CT>
static hipError_t launch_shared(const QeSharedArgs &y, int head_dim, hipStream_t st) {
    return head_dim == 64 ? launch_shared<BF, 64, CT>(y, st) : head_dim == 128 ? launch_shared<BF, 128, CT>(y, st) : launch_shared<BF, 256, CT>(y, st);
}
template <bool BF>
static hipError_t launch_shared(const QeSharedArgs &y, int head_dim, int cache_type, hipStream_t st) {
    if (cache_type == QE_I8) return launch_shared<BF, QE_I8>(y, head_dim, st);
    return cache_type == QE_F8 ? launch_shared<BF, QE_F8>(y, head_dim, st) : launch_shared<BF, QE_CACHE16>(y, head_dim, st);
}
hipError_t qe_launch_attn_shared(const QeSharedArgs &y, int head_dim, int type, int cache_type, hipStream_t st) {
    return type == QE_BF16 ? launch_shared<true>(y, head_dim, cache_type, st) : launch_shared<false>(y, head_dim, cache_type, st);
}
