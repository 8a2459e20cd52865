// Tiles of an 8-bit cache as 16-bit numbers in LDS, and their scales.
#pragma once
#include "qe_attn_rows.h"

// A wave's part of a tile of BN keys on its way: as codes in registers, or (heads of 256, whose rows fill the registers) in LDS
// that only this wave uses.
template <int CT, bool BF, int DH, int WAVES>
struct Stage {
    static constexpr int BN = DH == 256 ? 32 : 64, PART = BN / WAVES, NL = PART * DH / 1024; // 16-byte loads of a lane
    static constexpr int CH = DH / 16;                                                       // chunks of a row
    // of heads of 256: V, and with eight waves K, too (with four, two workgroups fit a CU's LDS only without)
    static constexpr bool V_IN_LDS = DH == 256, K_IN_LDS = DH == 256 && WAVES == 8;
    static constexpr int RAW = (V_IN_LDS + K_IN_LDS) * PART * DH; // bytes of LDS a wave
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    u4 k[K_IN_LDS ? 1 : NL], v[V_IN_LDS ? 1 : NL];
    float ks, vs; // lane n: the scales of the part's key n % PART

    // The codes of the wave's part of the tile of BN keys from k0 on.
    __device__ __forceinline__ void issue(const QeAttn8Args &x, int page, int kvh, int k0, int len, int wave, uint8_t *raw) {
        const int sub = k0 + wave * PART, at = sub < len ? sub : (len - 1) & -PART;
        unsigned known = 0; // that a page is none: lost_pages
        const size_t r0 = page_row(x.a, page, kvh, at, &known);
        const unsigned lane = lane_now(), n = lane % PART;
        ks = (x.ks + r0)[n];
        vs = (x.vs + r0)[n];
        const uint8_t *kp = (const uint8_t *)x.a.kc + r0 * DH, *vp = (const uint8_t *)x.a.vc + r0 * DH;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            if constexpr (K_IN_LDS) load_lds16_from(kp, PART * DH, lane * 16, i * 1024, raw + (NL + i) * 1024);
            else k[i] = *(const u4 *)(kp + i * 1024 + lane * 16);
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            if constexpr (V_IN_LDS) load_lds16_from(vp, PART * DH, lane * 16, i * 1024, raw + i * 1024);
            else v[i] = *(const u4 *)(vp + i * 1024 + lane * 16);
        }
    }
    // A load's registers, not looked at before this place: the compiler would begin to take codes apart where they are loaded,
    // and wait for them there.
    static __device__ __forceinline__ u4 come(u4 x) {
        asm volatile("" : "+v"(x));
        return x;
    }
    // They have come: to the tiles, as 16-bit numbers.  Behind the end, where codes and scales may be anything, zeros.
    __device__ __forceinline__ void land(int k0, int len, int wave, const uint8_t *raw, short *k_lds, short *v_lds, float *ks_lds, float *vs_lds) {
        if constexpr (V_IN_LDS) __builtin_amdgcn_s_waitcnt(0x0f70);
        const unsigned lane = lane_now(), n = lane % PART;
        // Lanes 0 .. PART - 1 write the part's keys' scales, the next PART its values', the others again what these did.
        const bool of_v = lane / PART & 1;
        (of_v ? vs_lds : ks_lds)[wave * PART + n] = k0 + wave * PART + (int)n < len ? (of_v ? vs : ks) : 0.f;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            u4 a, b;
            if constexpr (K_IN_LDS) a = *(const u4 *)(raw + (NL + i) * 1024 + lane * 16);
            else a = come(k[i]);
            if constexpr (V_IN_LDS) b = *(const u4 *)(raw + i * 1024 + lane * 16);
            else b = come(v[i]);
            const int row = wave * PART + i * (64 / CH) + lane / CH;
            if (CT == QE_F8 && k0 + BN > len) { // uniform
                if (k0 + row >= len) a = b = u4{0, 0, 0, 0};
            }
            // a lane's two chunks: of K neighbours but for the permutation, of V side by side
            char *kr = (char *)k_lds + row * DH * 2, *vr = (char *)v_lds + row * DH * 2;
            const unsigned ko = (lane % CH * 2 ^ k_swz(row)) << 4, vo = (lane % CH * 2 ^ v_swz<DH>(row)) << 4;
            *(qe_s8 *)(kr + ko) = elements_of<CT, BF>(a[0], a[1]);
            *(qe_s8 *)(kr + (ko ^ 16)) = elements_of<CT, BF>(a[2], a[3]);
            *(qe_s8 *)(vr + vo) = elements_of<CT, BF>(b[0], b[1]);
            *(qe_s8 *)(vr + vo + 16) = elements_of<CT, BF>(b[2], b[3]);
        }
    }
};

// x[i] times lane i's scale, of each 16 lanes
template <int I = 0>
__device__ __forceinline__ void scaled(qe_f16v &x, float s) {
    if constexpr (I < 16) {
        x[I] *= of_lane<I>(s);
        scaled<I + 1>(x, s);
    }
}
// Units (qe_mixer_device.h) of a block's rows, a lane's row for itself: a value behind a row's causal limit may be far greater than all
// of the row's own, and is nothing to it.  Where all rows see all of a tile's keys they are raised by its greatest scale, in the tiles that
// the causal limit cuts each by its own keys', which with the per-lane comparison costs fp16 prompts 0.5 to 2.5 % (8000 tokens of 32 / 8
// heads of 128 631 -> 637 us, packed ones 52.0 -> 52.9).  The probabilities and their sum count units, too, by the exponent that makes
// them; units are powers of two, so that no rounding changes.
template <bool BF>
struct RowUnits {
    static constexpr int LEAST = 127 - 60; // (of a scale below 2^-60 nothing is left in fp16)
    unsigned bits = (unsigned)LEAST << 23; // of the unit
    float log2 = LEAST - 127;
    // top: size_bits of the greatest scale that the row attends to in a tile.
    template <typename ROWS>
    __device__ __forceinline__ void raise(unsigned top, ROWS &rows) {
        const bool above = top > bits;
        if (__any(above)) {
            const int was = bits >> 23, next = min((int)(top >> 23) + 2, 227), now = above ? next : was;
            bits = (unsigned)now << 23;
            log2 = now - 127;
            rows.times(__builtin_ldexpf(1.f, was - now));
        }
    }
    __device__ __forceinline__ float unit() const { return __uint_as_float(bits); }
};
// Of a lane's 16 keys in Scores::s[b], which are those up to `limit`, the greatest scale's size_bits; `top` holds theirs, a key a lane.
template <int I = 0>
__device__ __forceinline__ unsigned greatest_seen(unsigned top, int b, int limit) {
    if constexpr (I < 16) {
        const unsigned x = (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x150 + I, 0xf, 0xf, true);
        return max(b * 32 + 8 * (I / 4) + I % 4 > limit ? 0 : x, greatest_seen<I + 1>(top, b, limit));
    }
    return 0;
}

// The sum of the probabilities as they are rounded, in place of as they were: x are they times their values' scales s, p is x rounded.
// A row's weights then sum to 1, and where one probability is nearly all, its rounding is in both and none of it in the result; a row
// of one key is its value: weights w with roundings e of u at most leave a result o the sum of e w (v - o), in place of e w v.  That is u (sum w |v| +
// |o|) at most, more than u sum w |v| where little of a row's weight is on its values and the rest on zeros, and as a rule less.  (Over many
// rows with many keys it changes little.)  Scales far below the greatest, whose products may be
// too small for the type, are left out: in fp16 those below 2^-6 of the row's unit.
template <bool BF, int I = 0, int KB>
__device__ __forceinline__ void sum_rounded(float &l, const Scores<KB> &x, const Probs<KB> &p, int b, float inverse, float most) {
    if constexpr (I < 16) {
        const float2 r = rest_of<BF>(p.p[b][I / 8].u[I % 8 / 2], x.s[b][I], x.s[b][I + 1]);
        auto below = [&](float y) { return BF || fabsf(y) < most ? y : 0.f; };
        l = fmaf(-r.x, below(of_lane<I>(inverse)), fmaf(-r.y, below(of_lane<I + 1>(inverse)), l));
        sum_rounded<BF, I + 2>(l, x, p, b, inverse, most);
    }
}
template <bool BF, int KB>
__device__ __forceinline__ void sum_rounded(float &l, const Scores<KB> &x, const Probs<KB> &p, const float *scales, RowUnits<BF> units) {
    const float most = BF ? 0.f : __uint_as_float(((127u + 6 + 127) << 23) - units.bits); // 2^6 over the unit
#pragma unroll
    for (int b = 0; b < KB; ++b) {
        const float s = scales[b * 32];
        sum_rounded<BF>(l, x, p, b, BF && !(s > 0x1p-60f) ? 0.f : __builtin_amdgcn_rcpf(s), most);
    }
}
