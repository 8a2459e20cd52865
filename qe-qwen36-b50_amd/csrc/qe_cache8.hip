// Norms, rotary positions and the write to a cache of 16 or 8 bits in one pass, and an 8-bit cache read back.
#include "qe_mixer_device.h"

// ---------------------------------------------------------------------------
// A workgroup per token, work items of 16 elements of a head as in k_append: 8 rotated pairs (i, i + rotary / 2), or 16
// elements behind them.  A head's items are 4, 8 or 16 lanes of one wave, so that its sum of squares and its greatest
// element are a few exchanges between lanes, and everything stays in registers from the load to the codes:
//   y = x / sqrt(mean(x^2) + eps) w, rotated;  scale = max |y| / 127 or / 448;  codes = y / scale, to nearest.
// The greatest is found among the bits without sign, where what is not finite is greater than all else.
//
// Bound by memory: 8000 tokens of 32 + 2 x 8 heads of 128, fp16 to e4m3, are 181 MB and take 39 to 40 us, 4.5 to 4.7 TB/s (a large copy reaches
// 5.0); 2000 tokens of 16 + 2 x 2 heads of 256 with norms, bf16 to 16 bits, 41 MB, 12 us.  Eight single tokens take 4.9 us, a launch and one round trip each for length, page and
// data.  A thread for each item, up to 512 a token, is slower than turns of 256 (42 us for 8000 tokens).
// ---------------------------------------------------------------------------
template <typename IN>
__device__ __forceinline__ void load8(const IN *p, float *x) {
    if constexpr (sizeof(IN) == 4) {
        const qe_f4 a = *(const qe_f4 *)p, b = *(const qe_f4 *)(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
    } else {
        const auto a = *(const __attribute__((ext_vector_type(8))) IN *)p;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
    }
}

// (Six instructions an element cost 1 to 2 % of a call whose tokens come from memory, 7 % of one of 5000 tokens of heads of 64 in the caches; the
// compiler's division 4 and 20 %.)
// x / s as 32 bits have it, for s in [1, 2) and its reciprocal to nearest: next to a border between two codes the product with a
// reciprocal would give the other one.  One correction by the remainder, which fmaf has exactly, makes the quotient one of the two floats next to
// x / s; a second rounds it to nearest (P. Markstein, Computation of elementary functions on the IBM RISC System/6000, 1990).
__device__ __forceinline__ float over(float x, float s, float inv) {
    float q = x * inv;
    q = fmaf(fmaf(-q, s, x), inv, q);
    return fmaf(fmaf(-q, s, x), inv, q);
}
// 8 values over their row's scale to codes
template <int CT>
__device__ __forceinline__ uint2 codes8(const float *x, float scale) {
    // both by a power of two that brings the scale to [1, 2), so that no remainder is too small for 32 bits
    const float up = __uint_as_float((254u << 23) - (__float_as_uint(scale) & 0x7f800000u)), s = scale * up, inv = 1.f / s;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = over(x[i] * up, s, inv);
    unsigned w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (CT == QE_I8) {
            // added to 1.5 2^23, a number's last bits are its nearest integer
            unsigned b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(y[4 * h + i] + 12582912.f);
            w[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400), 0x05040100);
        } else {
            int v = 0;
            v = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], v, false);
            v = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], v, true);
            w[h] = (unsigned)v;
        }
    }
    return make_uint2(w[0], w[1]);
}

// A value joined over the N lanes (4, 8 or 16, aligned) of a head.  Once four lanes agree, mirroring eight (and then sixteen)
// brings each the other four's (and eight's).
template <int CTRL>
__device__ __forceinline__ unsigned lanes(unsigned x) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true); }
template <int N>
__device__ __forceinline__ float sum_over(float x) {
    x += __uint_as_float(lanes<0xb1>(__float_as_uint(x)));
    x += __uint_as_float(lanes<0x4e>(__float_as_uint(x)));
    if (N > 4) x += __uint_as_float(lanes<0x141>(__float_as_uint(x)));
    if (N > 8) x += __uint_as_float(lanes<0x140>(__float_as_uint(x)));
    return x;
}
template <int N>
__device__ __forceinline__ unsigned max_over(unsigned x) {
    x = max(x, lanes<0xb1>(x));
    x = max(x, lanes<0x4e>(x));
    if (N > 4) x = max(x, lanes<0x141>(x));
    if (N > 8) x = max(x, lanes<0x140>(x));
    return x;
}

// a work item of a token: 16 elements of a head, in two runs of 8
template <typename IN, int DH>
struct Item {
    int kind, head, c, e0, e1; // kind: 0 q, 1 k, 2 v
    bool turned;
    const IN *src;
    __device__ __forceinline__ Item(const QeAppendArgs &a, int t, int it) {
        constexpr int PER = DH / 16;
        const int n_q = a.q ? a.q_heads * PER : 0, n_k = a.kv_heads * PER;
        kind = it < n_q ? 0 : it < n_q + n_k ? 1 : 2;
        const int j = it - (kind == 0 ? 0 : kind == 1 ? n_q : n_q + n_k);
        head = j / PER, c = j % PER;
        turned = kind < 2 && c * 16 < a.rotary;
        e0 = turned ? c * 8 : c * 16, e1 = turned ? a.rotary / 2 + c * 8 : c * 16 + 8;
        src = (kind == 0 ? (const IN *)a.q + (size_t)t * a.q_stride : kind == 1 ? (const IN *)a.k + (size_t)t * a.k_stride : (const IN *)a.v + (size_t)t * a.v_stride) + head * DH;
    }
};

template <typename IN, typename OUT, int CT, int DH>
__global__ __launch_bounds__(256) void k_append8(const QeAppend8Args x) {
    typedef __attribute__((ext_vector_type(8))) OUT OUT8;
    constexpr int PER = DH / 16; // items of a head
    const QeAppendArgs &a = x.a;
    __shared__ float2 cs[128];
    const int t = blockIdx.x, tid = threadIdx.x, n = ((a.q ? a.q_heads : 0) + 2 * a.kv_heads) * PER;
    float u[16];
    if (tid < n) { // the first item's elements, on their way while the token's place is looked up
        const Item<IN, DH> m(a, t, tid);
        load8(m.src + m.e0, u);
        load8(m.src + m.e1, u + 8);
    }
    report_offsets(a);
    QeToken at;
    if (!token_place(a, t, tid == 0, at)) return;
    if (tid < a.rotary / 2) {
        const int pos = a.pos ? a.pos[(size_t)(a.n_axes > 1 ? a.axis[tid] : 0) * a.n_tokens + t] : at.place;
        const double turn = (double)pos * a.turns[tid];
        float s, c;
        sincospif((float)(2.0 * (turn - rint(turn))), &s, &c);
        cs[tid] = make_float2(c, s);
    }
    __syncthreads();
    for (int it = tid; it < n; it += 256) {
        const Item<IN, DH> m(a, t, it);
        if (m.kind && at.row < 0) break;
        if (it != tid) {
            load8(m.src + m.e0, u);
            load8(m.src + m.e1, u + 8);
        }
        const float *w = m.kind == 0 ? x.wq : m.kind == 1 ? x.wk : nullptr;
        if (w) {
            float sum = 0, wt[16];
            load8(w + m.e0, wt);
            load8(w + m.e1, wt + 8);
#pragma unroll
            for (int i = 0; i < 16; ++i) sum = fmaf(u[i], u[i], sum);
            sum = sum_over<PER>(sum);
            const float r = sum < INFINITY ? __builtin_amdgcn_rsqf(fmaf(sum, 1.f / DH, x.eps)) : NAN; // to 2^-23
#pragma unroll
            for (int i = 0; i < 16; ++i) u[i] = u[i] * r * wt[i];
        }
        if (m.turned)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 r = cs[m.e0 + i];
                const float p = u[i], q = u[8 + i];
                u[i] = fmaf(p, r.x, -(q * r.y));
                u[8 + i] = fmaf(q, r.x, p * r.y);
            }
        const size_t row = (size_t)(at.row + ((long)m.head << a.page_log2));
        if (CT == QE_CACHE16 || m.kind == 0) { // 16 bits
            OUT *dst = m.kind == 0 ? (OUT *)a.q_out + (size_t)t * a.q_out_stride + (size_t)m.head * DH : (OUT *)(m.kind == 1 ? a.kc : a.vc) + row * DH;
            OUT8 lo, hi;
#pragma unroll
            for (int i = 0; i < 8; ++i) lo[i] = (OUT)u[i], hi[i] = (OUT)u[8 + i];
            *(OUT8 *)(dst + m.e0) = lo;
            *(OUT8 *)(dst + m.e1) = hi;
        } else {
            unsigned top = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(u[i]) & 0x7fffffffu);
            top = max_over<PER>(top);
            float scale = __uint_as_float(top) / (CT == QE_I8 ? 127.f : 448.f);
            uint2 lo = make_uint2(0, 0), hi = lo;
            if (top < 0x0d800000u) { // below 2^-100
                scale = 0;
            } else if (top >= 0x7f800000u) {
                scale = NAN;
            } else {
                lo = codes8<CT>(u, scale);
                hi = codes8<CT>(u + 8, scale);
            }
            uint8_t *dst = (uint8_t *)(m.kind == 1 ? a.kc : a.vc) + row * DH;
            *(uint2 *)(dst + m.e0) = lo;
            *(uint2 *)(dst + m.e1) = hi;
            if (m.c == 0) (m.kind == 1 ? x.ks : x.vs)[row] = scale;
        }
    }
}

template <typename IN, typename OUT, int CT>
static hipError_t launch_append8(const QeAppend8Args &a, hipStream_t st) {
    const dim3 g(a.a.n_tokens), b(256);
    if (a.a.head_dim == 64) k_append8<IN, OUT, CT, 64><<<g, b, 0, st>>>(a);
    else if (a.a.head_dim == 128) k_append8<IN, OUT, CT, 128><<<g, b, 0, st>>>(a);
    else k_append8<IN, OUT, CT, 256><<<g, b, 0, st>>>(a);
    return hipGetLastError();
}
template <typename IN, typename OUT>
static hipError_t launch_append8(const QeAppend8Args &a, int cache_type, hipStream_t st) {
    if (cache_type == QE_I8) return launch_append8<IN, OUT, QE_I8>(a, st);
    return cache_type == QE_F8 ? launch_append8<IN, OUT, QE_F8>(a, st) : launch_append8<IN, OUT, QE_CACHE16>(a, st);
}
hipError_t qe_launch_append8(const QeAppend8Args &a, int in_type, int type, int cache_type, hipStream_t st) {
    if (a.a.n_tokens == 0) return hipSuccess;
    if (type == QE_BF16) return in_type == QE_F32 ? launch_append8<float, __bf16>(a, cache_type, st) : launch_append8<__bf16, __bf16>(a, cache_type, st);
    return in_type == QE_F32 ? launch_append8<float, _Float16>(a, cache_type, st) : launch_append8<_Float16, _Float16>(a, cache_type, st);
}

// ---------------------------------------------------------------------------
// An 8-bit cache read back: a wave per token, 16 codes a lane and turn.  y = code times scale, rounded to 32 bits and then to 16.
// Bound by memory: 18,178 positions of 8 heads of 128, e4m3 to fp16, are 113 MB and take 26 us, 4.3 TB/s.  Two or four tokens a wave: 31 and
// 32 us (with ordinary stores, when one took 29).
// ---------------------------------------------------------------------------
template <bool BF, int CT>
__global__ __launch_bounds__(256) void k_read8(const QeRead8Args a) {
    report_offsets(a);
    const int t = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), lane = threadIdx.x & 63;
    if (t >= a.n_tokens) return;
    QeToken at;
    const bool known = token_place(a, t, lane == 0, at);
    if (!known && !at.in_call) return;
    const bool there = known && at.row >= 0;
    const int per = a.head_dim / 16, n = a.kv_heads * per;
    for (int it = lane; it < 2 * n; it += 64) {
        const bool is_k = it < n;
        const int j = is_k ? it : it - n, head = j / per, c = j - head * per;
        short *dst = is_k ? (short *)a.k + (size_t)t * a.k_stride : (short *)a.v + (size_t)t * a.v_stride;
        if (!(is_k ? a.k : a.v)) continue;
        dst += head * a.head_dim + c * 16;
        uint4 o[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if (there) {
            const size_t row = (size_t)(at.row + ((long)head << a.page_log2));
            const uint4 x = *(const uint4 *)((const uint8_t *)(is_k ? a.kc : a.vc) + row * a.head_dim + c * 16);
            const float s = (is_k ? a.ks : a.vs)[row];
            const unsigned w[4] = {x.x, x.y, x.z, x.w};
            unsigned r[8];
            for (int i = 0; i < 4; ++i) {
                float y[4];
                floats_of<CT>(w[i], y);
                r[2 * i] = pack2<BF>(y[0] * s, y[1] * s);
                r[2 * i + 1] = pack2<BF>(y[2] * s, y[3] * s);
            }
            o[0] = make_uint4(r[0], r[1], r[2], r[3]);
            o[1] = make_uint4(r[4], r[5], r[6], r[7]);
        }
        // (past the caches: 18,178 positions 28.8 -> 25.5 us)
        typedef unsigned u4 __attribute__((ext_vector_type(4)));
        __builtin_nontemporal_store(u4{o[0].x, o[0].y, o[0].z, o[0].w}, (u4 *)dst);
        __builtin_nontemporal_store(u4{o[1].x, o[1].y, o[1].z, o[1].w}, (u4 *)(dst + 8));
    }
}

hipError_t qe_launch_read8(const QeRead8Args &a, int type, int cache_type, hipStream_t st) {
    if (a.n_tokens == 0) return hipSuccess;
    const dim3 g((a.n_tokens + 3) / 4), b(256);
    if (type == QE_BF16) {
        if (cache_type == QE_I8) k_read8<true, QE_I8><<<g, b, 0, st>>>(a);
        else k_read8<true, QE_F8><<<g, b, 0, st>>>(a);
    } else {
        if (cache_type == QE_I8) k_read8<false, QE_I8><<<g, b, 0, st>>>(a);
        else k_read8<false, QE_F8><<<g, b, 0, st>>>(a);
    }
    return hipGetLastError();
}
