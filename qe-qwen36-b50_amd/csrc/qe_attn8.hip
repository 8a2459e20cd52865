// Attention of single tokens over an 8-bit paged cache.
#include "qe_attn_decode.h"

// ---------------------------------------------------------------------------
// As k_attn_decode: a workgroup per (sequence, key-value head, split of its length), its four waves each over their own
// 32-key steps, the heads that share a key-value head as columns of S^T = K Q^T and O^T += V^T P^T.
//
// Codes are turned to 16 bits in registers, exactly, right before the products; what memory and LDS carry are bytes.  A lane
// loads 16 codes of a key at once: the products' k may run over a head's elements in any order, so its first 8 belong to one
// product and its last 8 to the next, and Q is loaded in that order.  V reaches LDS by direct loads as it is, and V^T leaves it by
// transposing reads of bytes; its 16-byte chunks are permuted by row so that the 16 rows that half a wave reads lie in
// different banks.  A key's scale multiplies its scores, a value's its probabilities, each from one register: lane n of
// 16 has the scale of their n-th key, which the multiplication takes from there.
// Probabilities, times their values' scales, are rounded to the context's type for the second product (fp16: Units).
// ---------------------------------------------------------------------------
template <bool BF, int DH, int CT, bool ONCE>
__global__ __launch_bounds__(256, DH == 256 ? 2 : DH == 128 ? 3 : 4) void k_attn_decode8(const QeAttn8Args x) {
    const QeAttnArgs &a = x.a;
    constexpr int CH = DH / 16;    // 16-byte chunks of a row
    constexpr int ROWS = 64 / CH;  // rows of one direct load
    constexpr int KL = DH / 64, DB = DH / 16;
    constexpr int LDS = QE_ATTN_TILE * DH;     // bytes of a wave's V, and half of what its results take
    __shared__ __align__(16) short lds[4][LDS];
    __shared__ float2 ml[4][16];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, col = lane & 15, c = lane >> 4;
    // Workgroups go to the eight XCDs in turn: where the last one joins, a sequence's and head's all go to one.
    const bool near = a.splits > 1 && a.splits <= QE_ATTN_JOIN;
    const int at = near ? blockIdx.x / 8 : blockIdx.x, split = at % a.splits, item = near ? at / a.splits * 8 + blockIdx.x % 8 : at / a.splits;
    if (item >= a.n_seqs * a.kv_heads) return;
    const int seq = item / a.kv_heads, kvh = item % a.kv_heads;
    unsigned bad_len = 0, bad = 0;
    const int32_t *table = a.table + (size_t)seq * a.table_stride;
    // the wave's first page, looked up along with the length, as it is if the length is no longer than the host believed
    const unsigned first = ((unsigned)split * a.steps + wave) * QE_ATTN_TILE, cap = a.max_pages - 1;
    const unsigned guess0 = first >> a.page_log2 < cap ? first >> a.page_log2 : cap, guess1 = (first + 16) >> a.page_log2 < cap ? (first + 16) >> a.page_log2 : cap;
    int page0 = scalar_load(table + guess0), page1 = scalar_load(table + guess1);
    const short *q = (const short *)a.q + (size_t)seq * a.q_stride + ((size_t)kvh * a.group + col) * DH + c * 16;
    qe_s8 qf[2 * KL];
#pragma unroll
    for (int s = 0; s < 2 * KL; ++s) qf[s] = col < a.group ? *(const qe_s8 *)(q + s / 2 * 64 + s % 2 * 8) : qe_s8{};
    const int len = qe_checked(scalar_load(a.kv_len + seq), 0, a.max_pages << a.page_log2, 0, &bad_len);
    const int steps = qe_attn_decode_steps(len, a.steps, a.splits), active = qe_attn_decode_active(len, steps);
    if (split >= (active > 1 ? active : 1)) return; // a sequence without keys is the first workgroup's, which writes zeros

    const int tiles = (len + QE_ATTN_TILE - 1) / QE_ATTN_TILE, lo = split * steps, hi = lo + steps < tiles ? lo + steps : tiles;
    qe_f4 acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = qe_f4{0, 0, 0, 0};
    float m = -INFINITY, l = 0;
    Units units;
    uint8_t *vb = (uint8_t *)lds[wave];
    auto load16 = [](const void *p) {
        typedef unsigned u4 __attribute__((ext_vector_type(4)));
        return ONCE ? __builtin_nontemporal_load((const u4 *)p) : *(const u4 *)p;
    };
    // the lane's row of a transposing read, one of its group's eight keys, and its half of the 16 columns
    const int tr_key = 4 * c + (col >> 1 & 3) + (col & 8) * 2;
    const uint8_t *tr = vb + tr_key * DH + (col & 1) * 8;
    for (int t = lo + wave; t < hi; t += 4) {
        const int k0 = t * QE_ATTN_TILE;
        // the 16 positions from k0 + 16 on may be behind the end: any page of the sequence does
        if (t != lo + wave || steps != a.steps) {
            page0 = scalar_load(table + (k0 >> a.page_log2));
            if (k0 + 16 < len) page1 = scalar_load(table + ((k0 + 16) >> a.page_log2));
        }
        const size_t r0 = page_row(a, page0, kvh, k0, &bad);
        const size_t r1 = k0 + 16 < len ? page_row(a, page1, kvh, k0 + 16, &bad) : r0;
        const uint8_t *kp0 = (const uint8_t *)a.kc + (r0 + col) * DH + c * 16, *kp1 = (const uint8_t *)a.kc + (r1 + col) * DH + c * 16;
        decltype(load16(kp0)) kr[2][KL];
#pragma unroll
        for (int s = 0; s < KL; ++s) kr[0][s] = load16(kp0 + s * 64);
#pragma unroll
        for (int s = 0; s < KL; ++s) kr[1][s] = load16(kp1 + s * 64);
        const size_t sr = (col & 4 ? r1 : r0) + 4 * c + (col & 3);
        const float ks = x.ks[sr];
        float vs = x.vs[sr];
#pragma unroll
        for (int i = 0; i < QE_ATTN_TILE / ROWS; ++i) {
            const int row = i * ROWS + lane / CH, ch = (lane % CH) ^ swz8<DH>(row);
            load_lds16_from<ONCE>((const uint8_t *)a.vc + (i * ROWS < 16 ? r0 : r1) * DH, 16 * DH, (row & 15) * DH + ch * 16, 0, vb + i * 1024);
        }
        __builtin_amdgcn_sched_barrier(0); // all loads are under way before the first is waited for
        qe_f4 s[2] = {qe_f4{0, 0, 0, 0}, qe_f4{0, 0, 0, 0}};
#pragma unroll
        for (int st = 0; st < KL; ++st)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                s[0] = mfma16<BF>(elements_of<CT, BF>(kr[0][st][2 * h], kr[0][st][2 * h + 1]), qf[2 * st + h], s[0]);
                s[1] = mfma16<BF>(elements_of<CT, BF>(kr[1][st][2 * h], kr[1][st][2 * h + 1]), qf[2 * st + h], s[1]);
            }
        s[0] = qe_f4{s[0][0] * of_lane<0>(ks), s[0][1] * of_lane<1>(ks), s[0][2] * of_lane<2>(ks), s[0][3] * of_lane<3>(ks)};
        s[1] = qe_f4{s[1][0] * of_lane<4>(ks), s[1][1] * of_lane<5>(ks), s[1][2] * of_lane<6>(ks), s[1][3] * of_lane<7>(ks)};
        const bool cut = k0 + QE_ATTN_TILE > len;
        if (cut) {
#pragma unroll
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
#pragma unroll
            for (int d = 0; d < DB; ++d) acc[d] *= f;
            l *= f;
            m = mn;
        }
        if constexpr (!BF) {
            const float f = units.raise(!cut || (col & 4 ? k0 + 16 : k0) + 4 * c + (col & 3) < len ? vs : 0.f);
            if (f != 1.f)
#pragma unroll
                for (int d = 0; d < DB; ++d) acc[d] *= f;
            vs *= units.inverse;
        }
        const float base = exponent_base<BF, 0>(m * a.scale_log2);
        float p[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            p[i] = __builtin_amdgcn_exp2f(fmaf(s[0][i], a.scale_log2, base));
            p[4 + i] = __builtin_amdgcn_exp2f(fmaf(s[1][i], a.scale_log2, base));
        }
        l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        float w[8] = {p[0] * of_lane<0>(vs), p[1] * of_lane<1>(vs), p[2] * of_lane<2>(vs), p[3] * of_lane<3>(vs),
                      p[4] * of_lane<4>(vs), p[5] * of_lane<5>(vs), p[6] * of_lane<6>(vs), p[7] * of_lane<7>(vs)};
        if (cut) { // a scale behind the end may be anything
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (k0 + 4 * c + i >= len) w[i] = 0;
                if (k0 + 16 + 4 * c + i >= len) w[4 + i] = 0;
            }
        }
        union {
            unsigned u[4];
            qe_s8 v;
        } pf;
#pragma unroll
        for (int i = 0; i < 4; ++i) pf.u[i] = pack2<BF>(w[2 * i], w[2 * i + 1]);
        __builtin_amdgcn_s_waitcnt(0x0f70); // the direct loads have landed (vmcnt 0)
        if (CT == QE_F8 && cut) {            // codes behind the end may be NaN: a probability of 0 times NaN is NaN
            for (int i = lane; i < QE_ATTN_TILE * CH; i += 64)
                if (k0 + i / CH >= len) *(uint4 *)(vb + i * 16) = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            const uint2 v = lds_tr8(tr + ((d ^ swz8<DH>(tr_key)) << 4));
            acc[d] = mfma16<BF>(elements_of<CT, BF>(v.x, v.y), pf.v, acc[d]);
        }
    }
    if constexpr (!BF)
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] *= units.unit;
    finish_decode<BF, DH>(a, item, split, active, acc, m, l, bad, bad_len, &lds[0][0], LDS, ml);
}

template <bool BF, int DH, int CT>
static hipError_t launch_decode8(const QeAttn8Args &x, hipStream_t st) {
    const QeAttnArgs &a = x.a;
    const unsigned units = (unsigned)(a.n_seqs * a.kv_heads), whole = a.splits > 1 && a.splits <= QE_ATTN_JOIN ? (units + 7) / 8 * 8 : units;
    if (a.once) k_attn_decode8<BF, DH, CT, true><<<dim3(whole * a.splits), dim3(256), 0, st>>>(x);
    else k_attn_decode8<BF, DH, CT, false><<<dim3(whole * a.splits), dim3(256), 0, st>>>(x);
    if (a.splits > QE_ATTN_JOIN) k_attn_join<BF, DH><<<dim3((unsigned)(a.n_seqs * a.q_heads * (DH / 64))), dim3(1024), 0, st>>>(a);
    return hipGetLastError();
}
template <bool BF, int CT>
static hipError_t launch_decode8(const QeAttn8Args &x, int head_dim, hipStream_t st) {
    return head_dim == 64 ? launch_decode8<BF, 64, CT>(x, st) : head_dim == 128 ? launch_decode8<BF, 128, CT>(x, st) : launch_decode8<BF, 256, CT>(x, st);
}

hipError_t qe_launch_attn_decode8(const QeAttn8Args &x, int head_dim, int type, int cache_type, hipStream_t st) {
    if (type == QE_BF16) return cache_type == QE_I8 ? launch_decode8<true, QE_I8>(x, head_dim, st) : launch_decode8<true, QE_F8>(x, head_dim, st);
    return cache_type == QE_I8 ? launch_decode8<false, QE_I8>(x, head_dim, st) : launch_decode8<false, QE_F8>(x, head_dim, st);
}
