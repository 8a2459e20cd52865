// Attention of single tokens whose sequences share their beginnings: a shared key and value is read once for all rows of its
// group, not once a sequence.
//
// One launch for all keys, whose workgroups are of two kinds, and one for the join.  Prefix workgroups take 128 rows of a group
// (its sequences' heads of one key-value head) over a split of the shared positions, by the products of a prompt
// (qe_attn_rows.h) without a causal mask; the others a sequence's own positions, by those of k_attn_decode.  Both leave
// unnormalised partial results with their maximum and sum, in 32 bits, and k_shared_join joins a row's.  Positions are read
// through the table of the group's first sequence below the group's length, and through a sequence's own from there on.
//
// A shared key has 2 group n flops for a byte or two (n sequences), so that the prefix is bound by its products from some hundred rows
// on, and the own positions by memory.  Neither fills the GPU for long: 32 sequences behind 8000 positions, 16 / 2 heads of 256 in bf16, take
// 26 us and 6 for the join, where their 69 MB take 14 and the sequences alone would read 577; 64 in three groups, 32 / 8 of 128, e4m3, 36
// and 7 (90 MB); four behind 1000, int8, 8 and 4.  Launches of their own for the two kinds of work: 60 us for 34.
#include "qe_attn_keys.h"
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
// from the step on that start lies in
__device__ __forceinline__ int own_length(int start, int len) { return len > start ? len - (start & -QE_ATTN_TILE) : 0; }

template <int DH>
constexpr int shared_step() { return DH == 256 ? 32 : 64; } // keys of a prefix workgroup's step

// A partial result's place: those of a row are together, the prefix's first.
__device__ __forceinline__ size_t part_of(const QeSharedArgs &y, int seq, int head, int split) {
    return ((size_t)(seq - y.seq0) * y.x.a.q_heads + head) * (y.psplits + y.x.a.splits) + split;
}

// ---- the shared positions ---------------------------------------------------------------------------------
template <bool BF, int DH, int CT>
__device__ __forceinline__ void shared_prefix(const QeSharedArgs &y, int tile, int kvh, int split, short *k_a, short *v_a, short *k_b, short *v_b,
                                              uint8_t *raw_s, float (*s_a)[shared_step<DH>()], float (*s_b)[shared_step<DH>()]) {
    const QeAttnArgs &a = y.x.a;
    constexpr bool CODES = CT != QE_CACHE16;
    typedef Stage<CODES ? CT : QE_I8, BF, DH, 4> ST;
    constexpr int BM = QE_ATTN_SHARED_BM, BN = shared_step<DH>(), KB = BN / 32, PART = BN / 4;
    static_assert(ST::BN == BN, "a stage is a step");
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
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
    uint8_t *raw = raw_s + (CODES ? wave * ST::RAW : 0);
    // pages of the wave's parts of 64 tiles, a lane each, looked up together
    int pages = 0, pages_lo = lo - 64;
    auto load = [&](int t, short *k_lds, short *v_lds) { // the wave's part of tile t
        if (t >= pages_lo + 64) {
            pages_lo = t;
            const int at = (t + lane_now()) * BN + wave * PART;
            pages = table[(at < len ? at : len - 1) >> a.page_log2];
        }
        const int k0 = t * BN, page = __builtin_amdgcn_readlane(pages, t - pages_lo);
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
    RowUnits<BF> units;
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
    // Q and the first tile have come: else the compiler has each step wait for Q, and with it for the loads in flight
    __builtin_amdgcn_s_waitcnt(0x0f70);
    if constexpr (CODES) {
        stage.land(lo * BN, len, wave, raw, k_a, v_a, s_a[0], s_a[1]);
        if (lo + 1 < hi) load(lo + 1, nullptr, nullptr);
    }
    const bool few = n_rows < BM; // sum_rounded
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
                if constexpr (!BF) units.raise(greatest(size_bits(s_lds[1][lane & (BN - 1)])), w);
                w.weigh(a.scale_log2, BF ? 0.f : units.log2, s);
#pragma unroll
                for (int b = 0; b < KB; ++b) scaled(s.s[b], s_lds[1][b * 32 + at]);
                s.template pack<BF>(p);
                if (few) sum_rounded(w.l, s, p, s_lds[1] + at, units);
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
    if constexpr (CODES && !BF) w.times(units.unit());
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
// buf_a, buf_b: a wave's LDS, for its steps; row(w, h): DH floats of LDS for wave w's head h.
template <bool BF, int DH, int CT, bool AHEAD, typename ROW>
__device__ __forceinline__ void shared_own(const QeSharedArgs &y, int item, int split, uint8_t *buf_a, uint8_t *buf_b, const ROW &row, float2 (*ml)[16]) {
    const QeAttnArgs &a = y.x.a;
    typedef KeyWave<BF, DH, CT, Rows<BF, DH>::LAG, false> Wave; // probabilities as large as the prefix's are kept
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, col = lane & 15, c = lane >> 4;
    const int seq = y.seq0 + item / a.kv_heads, kvh = item % a.kv_heads;
    Wave w;
    w.begin(a, seq, kvh, lane);
    int start, len;
    own_positions(y, seq, &start, &len);
    const int own = own_length(start, len), base = start & -Wave::TILE;
    const int steps = qe_attn_decode_steps(own, a.steps, a.splits);
    if (split >= qe_attn_decode_active(own, steps)) return;
    const int32_t *table = a.table + (size_t)seq * a.table_stride;
    const int tiles = (len - base + Wave::TILE - 1) / Wave::TILE, lo = split * steps + wave, hi = split * steps + steps < tiles ? split * steps + steps : tiles;
    typename Wave::Pages pages = {};
    if (lo < hi) pages = Wave::look_up(a, table, base + lo * Wave::TILE, start, len);
    if constexpr (AHEAD) run_steps_ahead(w, a, y.x.ks, y.x.vs, table, kvh, base, start, len, lo, hi, pages, buf_a, buf_b);
    else run_steps(w, a, y.x.ks, y.x.vs, table, kvh, base, start, len, lo, hi, pages, buf_a);
    w.end();
    // the four waves' results joined (as in finish_decode), and left as a partial one
    float l = w.l;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (lane < 16) ml[wave][lane] = make_float2(w.m, l);
    float *o = row(wave, col);
#pragma unroll
    for (int d = 0; d < DH / 16; ++d) *(qe_f4 *)(o + ((d * 4 + c) ^ col) * 4) = w.acc[d];
    const int bad = __syncthreads_or(w.bad);
    if (bad && tid == 0) report(a.err, QE_BAD_PAGE);
    for (int i = tid; i < a.group * (DH / 4); i += 256) {
        const int h = i / (DH / 4), d = i % (DH / 4) * 4;
        float top = ml[0][h].x;
#pragma unroll
        for (int v = 1; v < 4; ++v) top = fmaxf(top, ml[v][h].x);
        float sum = 0;
        qe_f4 r = {0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float2 x = ml[u][h];
            const float f = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((x.x - top) * a.scale_log2);
            const qe_f4 v = *(const qe_f4 *)(row(u, h) + ((d / 4) ^ h) * 4);
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

// Prefix workgroups come first, since they are the longest; those of the same keys, one for each 128 rows, go to one XCD, whose
// L2 has the keys from the first one's reading on (workgroups go to the eight in turn).
template <bool BF, int DH, int CT>
__global__ __launch_bounds__(256, 2) void k_shared(const QeSharedArgs y) {
    const QeAttnArgs &a = y.x.a;
    constexpr int BN = shared_step<DH>();
    constexpr bool CODES = CT != QE_CACHE16;
    __shared__ __align__(16) short k_a[BN * DH], v_a[BN * DH], k_b[BN * DH], v_b[BN * DH];
    __shared__ __align__(16) uint8_t raw_s[CODES && DH == 256 ? 4 * Stage<QE_I8, BF, DH, 4>::RAW : 16];
    __shared__ __align__(16) float s_a[2][BN], s_b[2][BN];
    const int units = y.psplits * a.kv_heads, prefix = (units + 7) / 8 * 8 * a.tiles;
    if ((int)blockIdx.x < prefix) {
        const int unit = blockIdx.x / 8 / a.tiles * 8 + blockIdx.x % 8;
        if (unit < units) shared_prefix<BF, DH, CT>(y, blockIdx.x / 8 % a.tiles, unit / y.psplits, unit % y.psplits, k_a, v_a, k_b, v_b, raw_s, s_a, s_b);
    } else {
        static_assert(sizeof k_a >= 64 * DH, "room for a wave's values of a step, and its results");
        __shared__ float2 ml[4][16];
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), at = blockIdx.x - prefix;
        // a wave's own: two, for the values of a step each (of 16 bits and heads of 256 one)
        constexpr bool AHEAD = DH < 256; // (with 256 registers spill, and buffers of 16 bits would not fit)
        auto buffer = [&](int w, int second) {
            if (!AHEAD) return (uint8_t *)(w < 2 ? w == 0 ? k_a : v_a : w == 2 ? k_b : v_b);
            return (uint8_t *)(second ? w < 2 ? k_b : v_b : w < 2 ? k_a : v_a) + (w & 1) * (sizeof k_a / 2);
        };
        static_assert(!AHEAD || sizeof k_a / 2 >= 64 * DH, "room in one of two for sixteen heads' results");
        auto row = [&](int w, int h) { return (float *)buffer(w, 0) + h * DH; };
        // all sequences' first splits, then their second ones: those that have no keys end the launch
        const int items = (y.seq1 - y.seq0) * a.kv_heads;
        shared_own<BF, DH, CT, AHEAD>(y, at % items, at / items, buffer(wave, 0), buffer(wave, 1), row, ml);
    }
}

// ---- a row's partial results joined: a workgroup a row, its four waves every fourth split -------------------------
// (6 us, of which most is the launch and the look-ups.  Measured and not kept: sixteen waves a row where there are few rows and many
// splits; the first 32 results read while it is looked up which there are.)
template <bool BF, int DH>
__global__ __launch_bounds__(256) void k_shared_join(const QeSharedArgs y) {
    const QeAttnArgs &a = y.x.a;
    constexpr int E = DH / 64;
    // all groups' offsets are looked at, for the report: those that are wrong may hold no sequence
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < y.n_groups; i += (int64_t)gridDim.x * 256)
        if (qe_bad_offsets(y.seqs[i], y.seqs[i + 1], a.n_seqs) || y.prefix[i] < 0 || y.prefix[i] > a.max_pages << a.page_log2) report(a.err, QE_BAD_LENGTH);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, seq = y.seq0 + blockIdx.x / a.q_heads, head = blockIdx.x % a.q_heads;
    int start, len;
    const bool good = own_positions(y, seq, &start, &len);
    if (!good && threadIdx.x == 0) report(a.err, QE_BAD_LENGTH);
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
    for (int s = wave; s < n; s += 4) {
        const size_t i = at + s + (s < np ? 0 : gap);
        const float2 x = a.part_ml[i];
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = a.part_o[i * DH + e * 64 + lane];
        const float f = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.x - m);
        const bool any = x.y != 0.f; // else no key
        sum += any ? f * x.y : 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += any ? f * v[e] : 0.f;
    }
    __shared__ float o_s[4][DH], sum_s[4];
#pragma unroll
    for (int e = 0; e < E; ++e) o_s[wave][e * 64 + lane] = o[e];
    if (lane == 0) sum_s[wave] = sum;
    __syncthreads();
    if (wave) return;
    sum = (sum_s[0] + sum_s[1]) + (sum_s[2] + sum_s[3]);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    short *out = (short *)a.out + (size_t)seq * a.out_stride + (size_t)head * DH;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float r = (o_s[0][e * 64 + lane] + o_s[1][e * 64 + lane]) + (o_s[2][e * 64 + lane] + o_s[3][e * 64 + lane]);
        out[e * 64 + lane] = bad ? 0 : (short)pack2<BF>(r * inv, 0.f);
    }
}

template <bool BF, int DH, int CT>
static hipError_t launch_shared(const QeSharedArgs &y, hipStream_t st) {
    const QeAttnArgs &a = y.x.a;
    const unsigned n = y.seq1 - y.seq0, prefix = (unsigned)(y.psplits * a.kv_heads + 7) / 8 * 8 * a.tiles;
    k_shared<BF, DH, CT><<<dim3(prefix + n * a.kv_heads * a.splits), dim3(256), 0, st>>>(y);
    k_shared_join<BF, DH><<<dim3(n * a.q_heads), dim3(256), 0, st>>>(y);
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
