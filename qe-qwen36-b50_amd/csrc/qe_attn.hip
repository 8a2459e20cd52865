// Rotary positions with the cache write, and attention of single tokens over a paged cache.
#include "qe_mixer_device.h"

// ---------------------------------------------------------------------------
// Rotary positions and cache write, a workgroup per token.
// Pair (i, i + rotary/2) turns by pos * theta^(-2 i / rotary).  The angle is taken in turns
// in 64 bits (a position of 2^18 times a pair's 24-bit rate would leave 2^-6 of a turn in
// 32) and only the fraction goes to the 32-bit sine and cosine; they are made once per token
// and pair, in LDS, for all of its heads.  A work item is 16 elements of a head: 8 pairs,
// or 16 elements behind the rotated ones.  Bound by memory: q, k and v read and written.  8192
// tokens of 32 + 2 x 8 heads of 128, fp16, 201 MB: 31 us, 6.4 TB/s (a large copy here reaches 5.1; part of
// it stays in the last-level cache); of 16 + 2 x 2 heads of 256 from fp32 to bf16, 252 MB: 39 us.  8 tokens: 4 us, of
// which most is the launch.  Stores that pass the caches by save 2 of 40 us between calls on other data, and cost the
// attention that follows, which reads these rows, more.
// ---------------------------------------------------------------------------
template <typename IN>
__device__ __forceinline__ void load8(const IN *p, float *x) {
    if constexpr (sizeof(IN) == 4) {
        const qe_f4 a = *(const qe_f4 *)p, b = *(const qe_f4 *)(p + 4);
        for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
    } else {
        const auto a = *(const __attribute__((ext_vector_type(8))) IN *)p;
        for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
    }
}
template <typename OUT>
__device__ __forceinline__ void store8(OUT *p, const float *x) {
    __attribute__((ext_vector_type(8))) OUT a;
    for (int i = 0; i < 8; ++i) a[i] = (OUT)x[i];
    *(__attribute__((ext_vector_type(8))) OUT *)p = a;
}

template <typename IN, typename OUT>
__global__ __launch_bounds__(256) void k_append(const QeAppendArgs a) {
    __shared__ float2 cs[128];
    const int t = blockIdx.x, tid = threadIdx.x, half = a.rotary / 2;
    if (a.cu && (int64_t)t * 256 < a.n_seqs) // all sequences' offsets, for the report: those that are wrong may hold no token
        for (int64_t i = (int64_t)t * 256 + tid; i < a.n_seqs; i += (int64_t)gridDim.x * 256)
            if (qe_bad_offsets(a.cu[i], a.cu[i + 1], a.n_tokens)) report(a.err, QE_BAD_LENGTH);
    // the token's sequence, the last whose first row is not behind t, and its row in the cache: by every wave for itself, through
    // the scalar cache, with no barrier
    int seq = t, end = t + 1;
    bool known = true;
    if (a.cu) {
        int lo = 0, hi = a.n_seqs; // cu[lo] <= t < cu[hi], as far as cu rises
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (scalar_load(a.cu + mid) <= t) lo = mid;
            else hi = mid;
        }
        // next to offsets that fall, it is not known whose the token is
        const int before = scalar_load(a.cu + (lo ? lo - 1 : 0)), begin = scalar_load(a.cu + lo), after = scalar_load(a.cu + (lo + 2 <= a.n_seqs ? lo + 2 : a.n_seqs));
        end = scalar_load(a.cu + lo + 1);
        known = before <= begin && end <= after && !qe_bad_offsets(begin, end, a.n_tokens);
        if (t < begin || t >= end) return; // of no sequence
        seq = lo;
    }
    unsigned bad = 0;
    const int len = qe_checked(scalar_load(a.kv_len + seq), 0, a.max_pages << a.page_log2, -1, &bad), place = len - end + t;
    if (!known || bad) {
        if (tid == 0) report(a.err, QE_BAD_LENGTH);
        return;
    }
    long row = -1; // a token before the sequence's first position has none
    if (place >= 0) {
        const unsigned p = (unsigned)scalar_load(a.table + (size_t)seq * a.table_stride + (place >> a.page_log2));
        if (p >= a.n_pages) {
            if (tid == 0) report(a.err, QE_BAD_PAGE);
            return;
        }
        row = ((long)p * a.kv_heads << a.page_log2) + (place & ((1 << a.page_log2) - 1));
    }
    if (tid < half) {
        const int pos = a.pos ? a.pos[(size_t)(a.n_axes > 1 ? a.axis[tid] : 0) * a.n_tokens + t] : place;
        const double turn = (double)pos * a.turns[tid];
        float s, c;
        sincospif((float)(2.0 * (turn - rint(turn))), &s, &c);
        cs[tid] = make_float2(c, s);
    }
    __syncthreads();
    const int per = a.head_dim / 16; // items of a head
    const int n_q = a.q ? a.q_heads * per : 0, n_k = a.kv_heads * per;
    for (int it = tid; it < n_q + 2 * n_k; it += 256) {
        const int kind = it < n_q ? 0 : it < n_q + n_k ? 1 : 2, j = it - (kind == 0 ? 0 : kind == 1 ? n_q : n_q + n_k);
        if (kind && row < 0) break;
        const int head = j / per, c = j - head * per;
        const bool turned = kind < 2 && c * 16 < a.rotary;
        const int e0 = turned ? c * 8 : c * 16, e1 = turned ? half + c * 8 : c * 16 + 8;
        const IN *src = kind == 0   ? (const IN *)a.q + (size_t)t * a.q_stride
                        : kind == 1 ? (const IN *)a.k + (size_t)t * a.k_stride
                                    : (const IN *)a.v + (size_t)t * a.v_stride;
        src += (size_t)head * a.head_dim;
        float x[8], y[8];
        load8(src + e0, x);
        load8(src + e1, y);
        if (turned)
            for (int i = 0; i < 8; ++i) {
                const float2 r = cs[e0 + i];
                const float u = x[i], w = y[i];
                x[i] = fmaf(u, r.x, -(w * r.y));
                y[i] = fmaf(w, r.x, u * r.y);
            }
        OUT *dst = kind == 0 ? (OUT *)a.q_out + (size_t)t * a.q_out_stride + (size_t)head * a.head_dim
                             : (OUT *)(kind == 1 ? a.kc : a.vc) + (row + ((long)head << a.page_log2)) * a.head_dim;
        store8(dst + e0, x);
        store8(dst + e1, y);
    }
}

hipError_t qe_launch_append(const QeAppendArgs &a, int in_type, int type, hipStream_t st) {
    if (a.n_tokens == 0) return hipSuccess;
    const dim3 g(a.n_tokens), b(256);
    if (type == QE_BF16) {
        if (in_type == QE_F32) k_append<float, __bf16><<<g, b, 0, st>>>(a);
        else k_append<__bf16, __bf16><<<g, b, 0, st>>>(a);
    } else {
        if (in_type == QE_F32) k_append<float, _Float16><<<g, b, 0, st>>>(a);
        else k_append<_Float16, _Float16><<<g, b, 0, st>>>(a);
    }
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Decode: a workgroup per (sequence, key-value head, split of its length), its four waves
// each over their own 32-key steps, no barrier before the end.
//
// The heads that share a key-value head are the columns of both products, so every key and
// value is read once: S^T = K Q^T (16 keys x 16 heads per matrix product, K rows straight
// from memory to the operand registers) and O^T += V^T P^T.  S^T leaves 4 consecutive keys of
// a lane's column in its registers; two such groups are the 8 k of the second product's
// operand, and V^T is read from LDS with the transposing read in that same order of keys, so
// probabilities never cross lanes.  V reaches LDS by direct loads, its 64-byte units
// permuted by row so that the four rows of a transposing read hit different banks.
// Running maximum and sum in 32 bits per head; O is rescaled only when a maximum grew.  Probabilities are
// rounded to the cache's type for the second product (exponent_base; their sum is of the unrounded ones).
// Long lengths are bound by memory: one sequence of 100,000 keys, two key-value heads of 256, bf16, 205 MB:
// 37 us, 5.5 TB/s, and 5 for the join; 24 sequences of 38 to 8,095 keys, eight heads of 128, fp16, 339 MB: 70 us,
// 4.8 TB/s.  Short ones by latency: 700 keys take 10 us (length and page, keys and values, the exchange through
// memory, the join), where a launch that does nothing takes 2.
// ---------------------------------------------------------------------------
template <int DH>
__device__ __forceinline__ int v_swizzle(int row) { // of the 16-byte chunk index
    return DH == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2;
}

template <bool BF, int DH, bool ONCE>
__global__ __launch_bounds__(256, 2) void k_attn_decode(const QeAttnArgs a) {
    constexpr int CH = DH / 8;       // 16-byte chunks of a row
    constexpr int ROWS = 64 / CH;    // rows of one direct load
    constexpr int KS = DH / 32, DB = DH / 16;
    __shared__ __align__(16) short v_lds[4][QE_ATTN_TILE * DH];
    __shared__ float2 ml[4][16];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, col = lane & 15, c = lane >> 4;
    // Workgroups go to the eight XCDs in turn.  Where the last one joins (below), a sequence's and head's all go to
    // one, whose L2 then has their results; else any order does.
    const bool near = a.splits > 1 && a.splits <= QE_ATTN_JOIN;
    const int at = near ? blockIdx.x / 8 : blockIdx.x, split = at % a.splits, item = near ? at / a.splits * 8 + blockIdx.x % 8 : at / a.splits;
    if (item >= a.n_seqs * a.kv_heads) return;
    const int seq = item / a.kv_heads, kvh = item % a.kv_heads;
    unsigned bad_len = 0, bad = 0;
    // the wave's first page, looked up along with the length, as it is if the length is no longer than the host believed
    const unsigned first = ((unsigned)split * a.steps + wave) * QE_ATTN_TILE, cap = a.max_pages - 1;
    const unsigned guess0 = first >> a.page_log2 < cap ? first >> a.page_log2 : cap, guess1 = (first + 16) >> a.page_log2 < cap ? (first + 16) >> a.page_log2 : cap;
    int page0 = scalar_load(a.table + (size_t)seq * a.table_stride + guess0), page1 = scalar_load(a.table + (size_t)seq * a.table_stride + guess1);
    const short *q = (const short *)a.q + (size_t)seq * a.q_stride + ((size_t)kvh * a.group + col) * DH + c * 8;
    qe_s8 qf[KS];
    for (int s = 0; s < KS; ++s) qf[s] = col < a.group ? *(const qe_s8 *)(q + s * 32) : qe_s8{};
    const int len = qe_checked(scalar_load(a.kv_len + seq), 0, a.max_pages << a.page_log2, 0, &bad_len);
    const int32_t *table = a.table + (size_t)seq * a.table_stride;
    const size_t G = a.group;
    const int steps = qe_attn_decode_steps(len, a.steps, a.splits), active = qe_attn_decode_active(len, steps);
    if (split >= (active > 1 ? active : 1)) return; // a sequence without keys is the first workgroup's, which writes zeros

    const int tiles = (len + QE_ATTN_TILE - 1) / QE_ATTN_TILE, lo = split * steps, hi = lo + steps < tiles ? lo + steps : tiles;
    qe_f4 acc[DB];
    for (int d = 0; d < DB; ++d) acc[d] = qe_f4{0, 0, 0, 0};
    float m = -INFINITY, l = 0;
    short *vb = v_lds[wave];
    // keys and values of a call that exceed the L2s pass through them (qe_attn_decode_once)
    auto load_k = [](const short *p) { return ONCE ? __builtin_nontemporal_load((const qe_s8 *)p) : *(const qe_s8 *)p; };
    const int tr_row = col >> 2, tr_el = (col & 3) * 4; // of a transposing read
    for (int t = lo + wave; t < hi; t += 4) {
        const int k0 = t * QE_ATTN_TILE;
        // the 16 positions from k0 + 16 on may be behind the end: any page of the sequence does
        if (t != lo + wave || steps != a.steps) {
            page0 = scalar_load(table + (k0 >> a.page_log2));
            if (k0 + 16 < len) page1 = scalar_load(table + ((k0 + 16) >> a.page_log2));
        }
        const size_t r0 = page_row(a, page0, kvh, k0, &bad);
        const size_t r1 = k0 + 16 < len ? page_row(a, page1, kvh, k0 + 16, &bad) : r0;
        qe_s8 kf[2][KS];
        const short *kp0 = (const short *)a.kc + (r0 + col) * DH + c * 8, *kp1 = (const short *)a.kc + (r1 + col) * DH + c * 8;
#pragma unroll
        for (int s = 0; s < KS; ++s) kf[0][s] = load_k(kp0 + s * 32);
#pragma unroll
        for (int s = 0; s < KS; ++s) kf[1][s] = load_k(kp1 + s * 32);
#pragma unroll
        for (int i = 0; i < QE_ATTN_TILE / ROWS; ++i) {
            const int row = i * ROWS + lane / CH, ch = (lane % CH) ^ v_swizzle<DH>(row);
            load_lds16_from<ONCE>((const short *)a.vc + (i * ROWS < 16 ? r0 : r1) * DH, 32 * DH, ((row & 15) * DH + ch * 8) * 2, 0, vb + i * 512);
        }
        __builtin_amdgcn_sched_barrier(0); // all loads are under way before the first is waited for
        qe_f4 s[2] = {qe_f4{0, 0, 0, 0}, qe_f4{0, 0, 0, 0}};
#pragma unroll
        for (int st = 0; st < KS; ++st) {
            s[0] = mfma16<BF>(kf[0][st], qf[st], s[0]);
            s[1] = mfma16<BF>(kf[1][st], qf[st], s[1]);
        }
        if (k0 + QE_ATTN_TILE > len) {
            for (int i = 0; i < 4; ++i) {
                if (k0 + 4 * c + i >= len) s[0][i] = -INFINITY;
                if (k0 + 16 + 4 * c + i >= len) s[1][i] = -INFINITY;
            }
        }
        float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                          fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        if (__any(top > m)) {
            const float mn = fmaxf(m, top), f = m == -INFINITY ? 0.f : exp2f((m - mn) * a.scale_log2);
            for (int d = 0; d < DB; ++d) acc[d] *= f;
            l *= f;
            m = mn;
        }
        const float base = exponent_base<BF, 0>(m * a.scale_log2);
        float p[8];
        for (int i = 0; i < 4; ++i) {
            p[i] = __builtin_amdgcn_exp2f(fmaf(s[0][i], a.scale_log2, base));
            p[4 + i] = __builtin_amdgcn_exp2f(fmaf(s[1][i], a.scale_log2, base));
        }
        l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        union {
            unsigned u[4];
            qe_s8 v;
        } pf;
        for (int i = 0; i < 4; ++i) pf.u[i] = pack2<BF>(p[2 * i], p[2 * i + 1]);
        __builtin_amdgcn_s_waitcnt(0x0f70); // the direct loads have landed (vmcnt 0)
        if (k0 + QE_ATTN_TILE > len) {       // rows behind the end hold anything: a probability of 0 times NaN is NaN
            for (int i = lane; i < QE_ATTN_TILE * CH; i += 64)
                if (k0 + i / CH >= len) *(qe_s8 *)(vb + i * 8) = qe_s8{};
        }
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            const int ra = 4 * c + tr_row, rb = ra + 16;
            const int el = d * 16 + tr_el;
            const qe_s4 x = lds_tr(vb + ra * DH + (((el >> 3) ^ v_swizzle<DH>(ra)) << 3) + (el & 7));
            const qe_s4 y = lds_tr(vb + rb * DH + (((el >> 3) ^ v_swizzle<DH>(rb)) << 3) + (el & 7));
            acc[d] = mfma16<BF>(qe_s8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]}, pf.v, acc[d]);
        }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (lane < 16) ml[wave][lane] = make_float2(m, l);
    // the waves' results through LDS (a wave's own V buffer holds 16 heads x DH floats)
    float *o = (float *)vb;
    for (int d = 0; d < DB; ++d) *(qe_f4 *)(o + col * DH + ((d * 4 + c) ^ col) * 4) = acc[d]; // 16-byte units permuted by row: rows lie in the same banks
    bad = __syncthreads_or(bad) ? 1 : 0;
    if (tid == 0 && (bad | bad_len)) report(a.err, bad ? QE_BAD_PAGE : QE_BAD_LENGTH);
    for (int i = tid; i < a.group * (DH / 4); i += 256) {
        const int h = i / (DH / 4), d = i % (DH / 4) * 4;
        float top = ml[0][h].x;
        for (int w = 1; w < 4; ++w) top = fmaxf(top, ml[w][h].x);
        float sum = 0;
        qe_f4 r = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; ++w) { // no branches: each would wait for the LDS anew
            const float2 x = ml[w][h];
            const float f = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((x.x - top) * a.scale_log2);
            const qe_f4 y = *(const qe_f4 *)((const float *)v_lds[w] + h * DH + ((d / 4) ^ h) * 4);
            const bool any = x.y != 0.f; // else a wave without keys
            sum += any ? f * x.y : 0.f;
            for (int j = 0; j < 4; ++j) r[j] += any ? f * y[j] : 0.f;
        }
        if (active <= 1) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            r *= inv;
            if (bad) r = qe_f4{0, 0, 0, 0};
            uint2 w;
            w.x = pack2<BF>(r[0], r[1]);
            w.y = pack2<BF>(r[2], r[3]);
            *(uint2 *)((short *)a.out + (size_t)seq * a.out_stride + ((size_t)kvh * G + h) * DH + d) = w;
        } else {
            const size_t part = (size_t)item * a.splits + split, row = part * G + h;
            float2 *to_ml = a.part_ml + part * QE_ATTN_GROUP_MAX + h;
            if (a.splits <= QE_ATTN_JOIN) {
                store_through(a.part_o + row * DH + d, qe_f2{r[0], r[1]});
                store_through(a.part_o + row * DH + d + 2, qe_f2{r[2], r[3]});
                if (d == 0) store_through((float *)to_ml, qe_f2{top, bad ? -1.f : sum});
            } else {
                *(qe_f4 *)(a.part_o + row * DH + d) = r;
                if (d == 0) *to_ml = make_float2(top, bad ? -1.f : sum);
            }
        }
    }
    if (active <= 1 || a.splits > QE_ATTN_JOIN) return;
    // Few splits: the workgroup that is the last of its sequence and key-value head to arrive joins them.  Results
    // are written through to, and read from, where all XCDs see the same; a workgroup counts itself when its own
    // stores are acknowledged.  The last one sets the count back for the next call.
    // The count's low 8 bits are all workgroups', then 7 for those of each XCD.
    __shared__ unsigned long long count_s;
    const unsigned xcd = xcd_id();
    const unsigned long long one = 1ull + (1ull << (8 + 7 * xcd));
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __syncthreads();
    if (tid == 0) count_s = __hip_atomic_fetch_add(a.arrived + item, one, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + one;
    __syncthreads();
    const unsigned long long count = count_s;
    if ((count & 255) != (unsigned)active) return;
    if (tid == 0) __hip_atomic_store(a.arrived + item, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const size_t row0 = (size_t)item * a.splits * G;
    // All on this XCD, as the order of launch has it: their results are in its L2, and are read as usual (they were not
    // before in this launch, so no older copy is nearer).  Else from behind the L2s.
    const bool near_all = (count >> (8 + 7 * xcd) & 127) == (unsigned)active;
    float2 *all_ml = (float2 *)v_lds[0]; // [split][16]
    float *sums = (float *)(all_ml + QE_ATTN_JOIN * 16), *weight = sums + 16; // [split][16]
    float2 mine = make_float2(-INFINITY, 0.f);
    if (tid < active * 16 && (tid & 15) < a.group) { // a split's 16 are a cache line of their own
        const float2 *p = a.part_ml + (size_t)item * a.splits * QE_ATTN_GROUP_MAX + tid;
        if (near_all) {
            mine = *p;
        } else {
            const qe_f2 x = load_through((const float *)p);
            mine = make_float2(x[0], x[1]);
        }
    }
    all_ml[tid] = mine;
    __syncthreads();
    if (tid < a.group) {
        float top = -INFINITY, sum = 0;
        bool none = false;
        float2 x[QE_ATTN_JOIN];
#pragma unroll
        for (int s = 0; s < QE_ATTN_JOIN; ++s) x[s] = all_ml[s * 16 + tid];
#pragma unroll
        for (int s = 0; s < QE_ATTN_JOIN; ++s) top = fmaxf(top, x[s].x), none |= x[s].y < 0.f;
#pragma unroll
        for (int s = 0; s < QE_ATTN_JOIN; ++s) {
            const bool any = x[s].y != 0.f;
            const float f = x[s].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((x[s].x - top) * a.scale_log2);
            sum += any ? f * x[s].y : 0.f;
            weight[s * 16 + tid] = any ? f : 0.f; // a split without sum has left zeros
        }
        sums[tid] = none ? -1.f : sum;
    }
    __syncthreads();
    // a thread's 16 bytes of a row, all splits' in flight
    const int n = a.group * (DH / 4);
    const float *none = (const float *)(a.arrived + QE_ATTN_DECODE_WGS);
    for (int i = tid; i < n; i += 256) {
        const int h = i / (DH / 4), d = i % (DH / 4) * 4;
        const float *p = a.part_o + (row0 + h) * DH + d;
        qe_f4 o[QE_ATTN_JOIN];
#pragma unroll
        for (int g = 0; g < QE_ATTN_JOIN; g += 4) {
            if (g >= active) { // uniform
                o[g] = o[g + 1] = o[g + 2] = o[g + 3] = qe_f4{0, 0, 0, 0};
                continue;
            }
#pragma unroll
            for (int s = g; s < g + 4; ++s) {
                const float *at = s < active ? p + s * G * DH : none; // behind the last zeros
                if (near_all) {
                    o[s] = *(const qe_f4 *)at;
                } else {
                    const qe_f2 x = load_through(at), y = load_through(at + 2);
                    o[s] = qe_f4{x[0], x[1], y[0], y[1]};
                }
            }
        }
        float f[QE_ATTN_JOIN];
#pragma unroll
        for (int s = 0; s < QE_ATTN_JOIN; ++s) f[s] = weight[s * 16 + h]; // (as above: no branches around LDS reads)
        qe_f4 r = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < QE_ATTN_JOIN; ++s)
            for (int j = 0; j < 4; ++j) r[j] = fmaf(f[s], o[s][j], r[j]);
        const float sum = sums[h];
        r *= sum == 0.f ? 0.f : 1.f / sum;
        if (sum < 0.f) r = qe_f4{0, 0, 0, 0};
        uint2 w;
        w.x = pack2<BF>(r[0], r[1]);
        w.y = pack2<BF>(r[2], r[3]);
        *(uint2 *)((short *)a.out + (size_t)seq * a.out_stride + ((size_t)kvh * G + h) * DH + d) = w;
    }
}

// ---------------------------------------------------------------------------
// Many splits' results joined: o = sum 2^(m_s - m) o_s / sum 2^(m_s - m) l_s.  A workgroup of
// 1024 threads for 64 elements of a row, 16 threads for them and 64 groups over the splits: a
// read of a few hundred partial rows is latency, so all of it is in flight at once.  (256 splits of
// 16 rows of 256, 4 MB: 27 us by a workgroup of 256 threads a row, 10 by four a row.)
// ---------------------------------------------------------------------------
template <bool BF, int DH>
__global__ __launch_bounds__(1024) void k_attn_join(const QeAttnArgs a) {
    static_assert(QE_ATTN_DECODE_SPLITS <= 1024, "a thread looks at one split's maximum");
    __shared__ float w_s[1024], red[16], red2[16];
    __shared__ __align__(16) qe_f4 o_s[256];
    const int tid = threadIdx.x, part = blockIdx.x % (DH / 64), head = blockIdx.x / (DH / 64) % a.q_heads, seq = blockIdx.x / (DH / 64) / a.q_heads;
    const int kvh = head / a.group, h = head % a.group;
    unsigned bad_len = 0;
    const int len = qe_checked(scalar_load(a.kv_len + seq), 0, a.max_pages << a.page_log2, 0, &bad_len);
    const int active = qe_attn_decode_active(len, qe_attn_decode_steps(len, a.steps, a.splits));
    if (active <= 1) return; // its one workgroup has written the row
    const size_t row0 = ((size_t)seq * a.kv_heads + kvh) * a.splits * a.group + h;
    const int d = part * 64 + tid % 16 * 4;
    const float2 x = tid < active ? a.part_ml[(((size_t)seq * a.kv_heads + kvh) * a.splits + tid) * QE_ATTN_GROUP_MAX + h] : make_float2(-INFINITY, 0.f);
    qe_f4 o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) { // the first 256 splits; behind the last the first again, unused
        const int s = tid / 16 + 64 * k;
        o[k] = *(const qe_f4 *)(a.part_o + (row0 + (size_t)(s < active ? s : 0) * a.group) * DH + d);
    }
    float m = x.x;
    for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
    if ((tid & 63) == 0) red[tid >> 6] = m;
    const int bad = __syncthreads_or(x.y < 0.f);
    m = red[0];
    for (int k = 1; k < 16; ++k) m = fmaxf(m, red[k]);
    const float f = x.y == 0.f || x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((x.x - m) * a.scale_log2);
    w_s[tid] = x.y == 0.f ? -1.f : f; // -1: nothing of that split is used
    float sum = x.y == 0.f ? 0.f : f * x.y;
    for (int k = 32; k; k >>= 1) sum += __shfl_xor(sum, k);
    if ((tid & 63) == 0) red2[tid >> 6] = sum;
    __syncthreads();
    sum = 0;
    for (int k = 0; k < 16; ++k) sum += red2[k];
    qe_f4 r = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int s = tid / 16 + 64 * k;
        const float w = s < active ? w_s[s] : -1.f;
        if (w >= 0.f || w != w) r += w * o[k];
    }
    for (int s = tid / 16 + 256; s < active; s += 64) {
        const float w = w_s[s];
        const qe_f4 y = *(const qe_f4 *)(a.part_o + (row0 + (size_t)s * a.group) * DH + d);
        if (w >= 0.f || w != w) r += w * y;
    }
    for (int k = 16; k < 64; k <<= 1) // the wave's four groups
        for (int j = 0; j < 4; ++j) r[j] += __shfl_xor(r[j], k);
    if ((tid & 63) < 16) o_s[(tid >> 6) * 16 + tid % 16] = r;
    __syncthreads();
    if (tid < 16) {
        for (int g = 1; g < 16; ++g) r += o_s[g * 16 + tid];
        r *= sum == 0.f ? 0.f : 1.f / sum;
        if (bad) r = qe_f4{0, 0, 0, 0};
        uint2 w;
        w.x = pack2<BF>(r[0], r[1]);
        w.y = pack2<BF>(r[2], r[3]);
        *(uint2 *)((short *)a.out + (size_t)seq * a.out_stride + (size_t)head * DH + d) = w;
    }
}

template <bool BF, int DH>
static hipError_t launch_decode(const QeAttnArgs &a, hipStream_t st) {
    const unsigned units = (unsigned)(a.n_seqs * a.kv_heads), whole = a.splits > 1 && a.splits <= QE_ATTN_JOIN ? (units + 7) / 8 * 8 : units;
    if (a.once) k_attn_decode<BF, DH, true><<<dim3(whole * a.splits), dim3(256), 0, st>>>(a);
    else k_attn_decode<BF, DH, false><<<dim3(whole * a.splits), dim3(256), 0, st>>>(a);
    if (a.splits > QE_ATTN_JOIN) k_attn_join<BF, DH><<<dim3((unsigned)(a.n_seqs * a.q_heads * (DH / 64))), dim3(1024), 0, st>>>(a);
    return hipGetLastError();
}

hipError_t qe_launch_attn_decode(const QeAttnArgs &a, int head_dim, int type, hipStream_t st) {
    if (type == QE_BF16)
        return head_dim == 64 ? launch_decode<true, 64>(a, st) : head_dim == 128 ? launch_decode<true, 128>(a, st) : launch_decode<true, 256>(a, st);
    return head_dim == 64 ? launch_decode<false, 64>(a, st) : head_dim == 128 ? launch_decode<false, 128>(a, st) : launch_decode<false, 256>(a, st);
}
