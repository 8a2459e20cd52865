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
    float scale; // lanes 0 .. PART - 1: of the part's keys, 32 .. 32 + PART - 1: of its values

    // The codes of the wave's part of the tile of BN keys from k0 on.
    __device__ __forceinline__ void issue(const QeAttn8Args &x, int page, int kvh, int k0, int len, int wave, uint8_t *raw) {
        const int sub = k0 + wave * PART, at = sub < len ? sub : (len - 1) & -PART;
        unsigned known = 0; // that a page is none: lost_pages
        const size_t r0 = page_row(x.a, page, kvh, at, &known);
        const int lane = lane_now(), n = lane & 31;
        scale = (lane < 32 ? x.ks : x.vs)[r0 + (n < PART ? n : 0)];
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
    // They have come: to the tiles, as 16-bit numbers.  Behind the end, where codes and scales may be anything, zeros.
    __device__ __forceinline__ void land(int k0, int len, int wave, const uint8_t *raw, short *k_lds, short *v_lds, float *ks, float *vs) {
        if constexpr (V_IN_LDS) __builtin_amdgcn_s_waitcnt(0x0f70);
        const int lane = lane_now(), n = lane & 31;
        const bool cut = k0 + BN > len;
        if (n < PART) (lane < 32 ? ks : vs)[wave * PART + n] = cut && k0 + wave * PART + n >= len ? 0.f : scale;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int row = wave * PART + i * (64 / CH) + lane / CH, c = lane % CH * 2;
            u4 a, b;
            if constexpr (K_IN_LDS) a = *(const u4 *)(raw + (NL + i) * 1024 + lane * 16);
            else a = k[i];
            if constexpr (V_IN_LDS) b = *(const u4 *)(raw + i * 1024 + lane * 16);
            else b = v[i];
            if (CT == QE_F8 && cut && k0 + row >= len) a = b = u4{0, 0, 0, 0};
            short *kr = k_lds + row * DH, *vr = v_lds + row * DH;
            *(qe_s8 *)(kr + ((c ^ k_swz(row)) << 3)) = elements_of<CT, BF>(a[0], a[1]);
            *(qe_s8 *)(kr + (((c + 1) ^ k_swz(row)) << 3)) = elements_of<CT, BF>(a[2], a[3]);
            *(qe_s8 *)(vr + ((c ^ v_swz<DH>(row)) << 3)) = elements_of<CT, BF>(b[0], b[1]);
            *(qe_s8 *)(vr + (((c + 1) ^ v_swz<DH>(row)) << 3)) = elements_of<CT, BF>(b[2], b[3]);
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
