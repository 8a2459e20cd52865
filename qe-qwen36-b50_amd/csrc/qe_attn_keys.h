// A wave's part of single-token attention over some of a sequence's keys, of a cache of 8 bits, or of 16.
#pragma once
#include "qe_attn_rows.h"

// The heads that share a key-value head are the columns of S^T = K Q^T and O^T += V^T P^T (v_mfma_f32_16x16x32), so every key and
// value is read once, and probabilities never cross lanes: as in k_attn_decode.
//
// Codes are turned to 16 bits in registers, exactly, right before the products; what memory and LDS carry are bytes.  A lane
// loads 16 codes of a key at once: the products' k may run over a head's elements in any order, so its first 8 belong to one
// product and its last 8 to the next, and Q is loaded in that order.  V reaches LDS by direct loads as it is, and V^T leaves it by
// transposing reads of bytes; its 16-byte chunks are permuted by row so that the 16 rows that half a wave reads lie in
// different banks.  A key's scale multiplies its scores, a value's its probabilities, each from one register: lane n of
// 16 has the scale of their n-th key, which the multiplication takes from there.  A probability times its value's scale is two numbers
// of the context's type for the second product, the rounded one and what that leaves (fp16: Units): rounded once, the greatest one's error
// would be all of a row's with few keys, and as large as the result's own rounding.  It costs 1 to 2 % of a call (heads of 64: 6 to 9 %), and
// halves the squared error.
//
// A step is 32 keys.  LAG: exponent_base.
template <bool BF, int DH, int CT, int LAG, bool ONCE>
struct KeyWave {
    static constexpr bool CODES = CT != QE_CACHE16;
    static constexpr int SIZE = CODES ? 1 : 2;                // bytes of an element
    static constexpr int NB = 2, TILE = NB * 16;              // blocks of 16 keys in a step
    static constexpr int CH = DH * SIZE / 16, ROWS = 64 / CH; // 16-byte chunks of a row, rows of one direct load
    static constexpr int KL = DH * SIZE / 64, DB = DH / 16;
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    typedef int Pages __attribute__((ext_vector_type(NB)));

    qe_s8 q[DH / 32]; // of head `col`; in the order of the codes, or of K
    qe_f4 acc[DB];    // O^T
    float m, l;       // running maximum of the scores (as they are) and sum, of the lane's keys
    unsigned bad;     // met a page that is none
    Units units;

    __device__ __forceinline__ void begin(const QeAttnArgs &a, int seq, int kvh, int lane) {
        const int col = lane & 15, c = lane >> 4;
        const short *p = (const short *)a.q + (size_t)seq * a.q_stride + ((size_t)kvh * a.group + col) * DH;
#pragma unroll
        for (int s = 0; s < DH / 32; ++s) q[s] = col < a.group ? *(const qe_s8 *)(p + (CODES ? s / 2 * 64 + c * 16 + s % 2 * 8 : s * 32 + c * 8)) : qe_s8{};
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] = qe_f4{0, 0, 0, 0};
        m = -INFINITY, l = 0;
        bad = 0;
    }
    // 16 positions that all lie before the first, or behind the last, may have no page: others of the step do.
    static __device__ __forceinline__ int place_of(int k0, int b, int start, int len) {
        const int p = k0 + 16 * b, first = start & -16;
        return p < first ? first : p < len ? p : k0 < first ? first : k0;
    }
    static __device__ __forceinline__ Pages look_up(const QeAttnArgs &a, const int32_t *table, int k0, int start, int len) {
        Pages pages;
#pragma unroll
        for (int b = 0; b < NB; ++b) pages[b] = scalar_load(table + (place_of(k0, b, start, len) >> a.page_log2));
        return pages;
    }
    // A step's keys and scales on their way, and its values on theirs to LDS of this wave's (TILE * DH * SIZE bytes).
    struct Step {
        u4 k[NB][KL];
        float ks[NB / 2], vs[NB / 2];
    };
    static constexpr int LOADS = NB * KL + (CODES ? NB : 0) + TILE / ROWS; // of a step
    // The step of keys from k0 on, of which those in [start, len) count, in the pages given.
    __device__ __forceinline__ void issue(const QeAttnArgs &a, const float *k_scale, const float *v_scale, int kvh, int k0, int start, int len, const Pages pages,
                                          uint8_t *vb, Step &x) {
        const int lane = lane_now(), col = lane & 15, c = lane >> 4;
        auto load16 = [](const void *p) { return ONCE ? __builtin_nontemporal_load((const u4 *)p) : *(const u4 *)p; };
        size_t r[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) r[b] = page_row(a, pages[b], kvh, place_of(k0, b, start, len), &bad);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int s = 0; s < KL; ++s) x.k[b][s] = load16((const uint8_t *)a.kc + (r[b] + col) * DH * SIZE + c * 16 + s * 64);
        if constexpr (CODES)
#pragma unroll
            for (int j = 0; j < NB / 2; ++j) {
                const size_t even = r[2 * j], odd = r[2 * j + 1], sr = (col & 4 ? odd : even) + 4 * c + (col & 3);
                x.ks[j] = k_scale[sr], x.vs[j] = v_scale[sr];
            }
        auto swz = [](int row) { return CODES ? swz8<DH>(row) : v_swz<DH>(row); };
#pragma unroll
        for (int i = 0; i < TILE / ROWS; ++i) {
            const int row = i * ROWS + lane / CH, ch = (lane % CH) ^ swz(row);
            load_lds16_from<ONCE>((const uint8_t *)a.vc + r[i * ROWS / 16] * DH * SIZE, 16 * DH * SIZE, (row & 15) * DH * SIZE + ch * 16, 0, vb + i * 1024);
        }
        __builtin_amdgcn_sched_barrier(0); // all loads are under way before the first is waited for
    }
    // The step that `x` and vb hold, or will.  MORE: another one was issued after it.
    template <bool MORE>
    __device__ __forceinline__ void work(const QeAttnArgs &a, int k0, int start, int len, uint8_t *vb, Step &x) {
        const int lane = lane_now(), col = lane & 15, c = lane >> 4;
        auto swz = [](int row) { return CODES ? swz8<DH>(row) : v_swz<DH>(row); };
        qe_f4 s[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) s[b] = qe_f4{0, 0, 0, 0};
#pragma unroll
        for (int st = 0; st < KL; ++st)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if constexpr (CODES) {
                    s[b] = mfma16<BF>(elements_of<CT, BF>(x.k[b][st][0], x.k[b][st][1]), q[2 * st], s[b]);
                    s[b] = mfma16<BF>(elements_of<CT, BF>(x.k[b][st][2], x.k[b][st][3]), q[2 * st + 1], s[b]);
                } else {
                    s[b] = mfma16<BF>(__builtin_bit_cast(qe_s8, x.k[b][st]), q[st], s[b]);
                }
            }
        if constexpr (CODES)
#pragma unroll
            for (int j = 0; j < NB / 2; ++j) {
                s[2 * j] = by_scale<0>(s[2 * j], x.ks[j]);
                s[2 * j + 1] = by_scale<4>(s[2 * j + 1], x.ks[j]);
            }
        const bool cut = k0 < start || k0 + TILE > len;
        auto outside = [&](int key) { return k0 + key < start || k0 + key >= len; };
        if (cut)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (outside(16 * b + 4 * c + i)) s[b][i] = -INFINITY;
        float top = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
#pragma unroll
        for (int b = 1; b < NB; ++b) top = fmaxf(top, fmaxf(fmaxf(s[b][0], s[b][1]), fmaxf(s[b][2], s[b][3])));
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
            float most = 0;
#pragma unroll
            for (int j = 0; j < NB / 2; ++j) {
                const float v = fabsf(x.vs[j]);
                if (!(cut && outside(32 * j + (col & 4 ? 16 : 0) + 4 * c + (col & 3))) && v < INFINITY) most = fmaxf(most, v);
            }
            const float f = units.raise(most);
            if (f != 1.f)
#pragma unroll
                for (int d = 0; d < DB; ++d) acc[d] *= f;
#pragma unroll
            for (int j = 0; j < NB / 2; ++j) x.vs[j] *= units.inverse;
        }
        const float base = exponent_base<BF, LAG>(m * a.scale_log2);
        qe_s8 pf[NB / 2], rest[NB / 2]; // rest: what the rounding to 16 bits leaves of a probability times its value's scale
#pragma unroll
        for (int j = 0; j < NB / 2; ++j) {
            qe_f4 p = exponentials(s[2 * j], a.scale_log2, base), z = exponentials(s[2 * j + 1], a.scale_log2, base);
            l += ((p[0] + p[1]) + (p[2] + p[3])) + ((z[0] + z[1]) + (z[2] + z[3]));
            if constexpr (CODES) {
                p = by_scale<0>(p, x.vs[j]);
                z = by_scale<4>(z, x.vs[j]);
                if (cut) // a scale there may be anything
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        p[i] = outside(32 * j + 4 * c + i) ? 0.f : p[i];
                        z[i] = outside(32 * j + 16 + 4 * c + i) ? 0.f : z[i];
                    }
            }
            pf[j] = __builtin_bit_cast(qe_s8, u4{pack2<BF>(p[0], p[1]), pack2<BF>(p[2], p[3]), pack2<BF>(z[0], z[1]), pack2<BF>(z[2], z[3])});
            if constexpr (CODES) {
                auto left = [](unsigned hi, float a, float b) {
                    const float2 x = rest_of<BF>(hi, a, b);
                    return pack2<BF>(x.x, x.y);
                };
                const u4 hi = __builtin_bit_cast(u4, pf[j]);
                rest[j] = __builtin_bit_cast(qe_s8, u4{left(hi[0], p[0], p[1]), left(hi[1], p[2], p[3]), left(hi[2], z[0], z[1]), left(hi[3], z[2], z[3])});
            }
        }
        constexpr int LATER = MORE ? LOADS : 0;
        __builtin_amdgcn_s_waitcnt(0x0f70 | (LATER & 15) | LATER >> 4 << 14); // its direct loads have landed (vmcnt LATER)
        if (CT != QE_I8 && cut)              // V there may be anything: a probability of 0 times NaN is NaN
            for (int i = lane; i < TILE * CH; i += 64)
                if (outside(i / CH)) *(uint4 *)(vb + i * 16) = make_uint4(0, 0, 0, 0);
        // the lane's row of a transposing read: of bytes one of its group's eight keys, of 16 bits one of four
        const int key = CODES ? 4 * c + (col >> 1 & 3) + (col & 8) * 2 : 4 * c + (col >> 2);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int j = 0; j < NB / 2; ++j) { // 16 rows on, and 32, the permutation is the same but for bits that key has
                if constexpr (CODES) {
                    const uint2 v = lds_tr8(vb + (key + 32 * j) * DH + ((d ^ swz(key)) << 4) + (col & 1) * 8);
                    const qe_s8 y = elements_of<CT, BF>(v.x, v.y);
                    acc[d] = mfma16<BF>(y, rest[j], mfma16<BF>(y, pf[j], acc[d]));
                } else {
                    const int el = d * 16 + (col & 3) * 4, at = (((el >> 3) ^ swz(key)) << 3) + (el & 7);
                    const qe_s4 x = lds_tr((const short *)vb + key * DH + at), z = lds_tr((const short *)vb + (key + 16) * DH + at);
                    acc[d] = mfma16<BF>(qe_s8{x[0], x[1], x[2], x[3], z[0], z[1], z[2], z[3]}, pf[j], acc[d]);
                }
            }
    }
    __device__ __forceinline__ void end() {
        if constexpr (CODES && !BF)
#pragma unroll
            for (int d = 0; d < DB; ++d) acc[d] *= units.unit;
    }
    static __device__ __forceinline__ qe_f4 exponentials(qe_f4 x, float scale, float base) {
        return qe_f4{__builtin_amdgcn_exp2f(fmaf(x[0], scale, base)), __builtin_amdgcn_exp2f(fmaf(x[1], scale, base)),
                     __builtin_amdgcn_exp2f(fmaf(x[2], scale, base)), __builtin_amdgcn_exp2f(fmaf(x[3], scale, base))};
    }
    template <int I>
    static __device__ __forceinline__ qe_f4 by_scale(qe_f4 x, float s) {
        return qe_f4{x[0] * of_lane<I>(s), x[1] * of_lane<I + 1>(s), x[2] * of_lane<I + 2>(s), x[3] * of_lane<I + 3>(s)};
    }
};

// A wave's steps from t on, every fourth one up to `hi`, of keys counted from `base` (a multiple of the step's).  `pages` are the
// first one's.  (In k_attn_decode8 these; issuing the next step before this one's work took it from 42 to 47 us for 24 ragged
// sequences of 8 heads of 128, since fewer waves fit; steps of 64 keys, to 48.)
template <typename WAVE>
__device__ __forceinline__ void run_steps(WAVE &w, const QeAttnArgs &a, const float *ks, const float *vs, const int32_t *table, int kvh, int base, int start, int len,
                                          int t, int hi, typename WAVE::Pages pages, uint8_t *vb) {
    for (; t < hi; t += 4) {
        typename WAVE::Step x;
        const int k0 = base + t * WAVE::TILE;
        w.issue(a, ks, vs, kvh, k0, start, len, pages, vb, x);
        if (t + 4 < hi) pages = WAVE::look_up(a, table, k0 + 4 * WAVE::TILE, start, len);
        w.template work<false>(a, k0, start, len, vb, x);
    }
}
// The same with the next step on its way to the other of two buffers while one is worked on, where registers are there anyway.
// (The buffers are in variables of their own: else the compiler has LDS reads wait for all direct loads in flight.)
template <typename WAVE>
__device__ __forceinline__ void run_steps_ahead(WAVE &w, const QeAttnArgs &a, const float *ks, const float *vs, const int32_t *table, int kvh, int base, int start,
                                                int len, int t, int hi, typename WAVE::Pages pages, uint8_t *buf_a, uint8_t *buf_b) {
    constexpr int TILE = WAVE::TILE;
    if (t >= hi) return;
    typename WAVE::Step x, y;
    auto pages_of = [&](int i) { return WAVE::look_up(a, table, base + (i < hi ? i : t) * TILE, start, len); };
    w.issue(a, ks, vs, kvh, base + t * TILE, start, len, pages, buf_a, x);
    pages = pages_of(t + 4);
    for (; t + 4 < hi; t += 8) {
        w.issue(a, ks, vs, kvh, base + (t + 4) * TILE, start, len, pages, buf_b, y);
        pages = pages_of(t + 8);
        w.template work<true>(a, base + t * TILE, start, len, buf_a, x);
        if (t + 8 >= hi) {
            w.template work<false>(a, base + (t + 4) * TILE, start, len, buf_b, y);
            return;
        }
        w.issue(a, ks, vs, kvh, base + (t + 8) * TILE, start, len, pages, buf_a, x);
        pages = pages_of(t + 12);
        w.template work<true>(a, base + (t + 4) * TILE, start, len, buf_b, y);
    }
    w.template work<false>(a, base + t * TILE, start, len, buf_a, x);
}
