// The end of a single-token attention workgroup, and the join of many splits' results: the same for caches of 16 and of 8 bits.
#pragma once
#include "qe_mixer_device.h"

// Four waves' results (acc: O^T, column the head; m, l: running maximum and sum of the lane's keys) of split `split` of
// sequence and key-value head `item`: joined, and written where there is one active split, else left as a partial result,
// which with few splits the last workgroup to arrive joins.  row(w, h): DH floats of LDS for wave w's head h, of HEADS at a time;
// lds: some of it, 4 KB.
template <bool BF, int DH, int HEADS, typename ROW>
__device__ __forceinline__ void finish_decode(const QeAttnArgs &a, int item, int split, int active, const qe_f4 *acc, float m, float l, unsigned bad,
                                              unsigned bad_len, const ROW &row, void *lds, float2 (*ml)[16]) {
    constexpr int DB = DH / 16;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, col = lane & 15, c = lane >> 4;
    const int seq = item / a.kv_heads, kvh = item % a.kv_heads;
    const size_t G = a.group;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (lane < 16) ml[wave][lane] = make_float2(m, l);
#pragma unroll
    for (int h0 = 0; h0 < 16; h0 += HEADS) {
        if (h0 && h0 >= a.group) break;
        // the waves' results through LDS
        if (h0) __syncthreads();
        if (HEADS == 16 || col / HEADS == h0 / HEADS) {
            float *o = row(wave, col - h0);
            for (int d = 0; d < DB; ++d) *(qe_f4 *)(o + ((d * 4 + c) ^ col) * 4) = acc[d]; // 16-byte units permuted by row: rows lie in the same banks
        }
        if (h0) {
            __syncthreads();
        } else {
            bad = __syncthreads_or(bad) ? 1 : 0;
            if (tid == 0 && (bad | bad_len)) report(a.err, bad ? QE_BAD_PAGE : QE_BAD_LENGTH);
        }
        const int heads = a.group - h0 < HEADS ? a.group - h0 : HEADS;
        for (int i = tid; i < heads * (DH / 4); i += 256) {
            const int h = h0 + i / (DH / 4), d = i % (DH / 4) * 4;
            float top = ml[0][h].x;
            for (int w = 1; w < 4; ++w) top = fmaxf(top, ml[w][h].x);
            float sum = 0;
            qe_f4 r = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < 4; ++w) { // no branches: each would wait for the LDS anew
                const float2 x = ml[w][h];
                const float f = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((x.x - top) * a.scale_log2);
                const qe_f4 y = *(const qe_f4 *)(row(w, h - h0) + ((d / 4) ^ h) * 4);
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
                const size_t part = (size_t)item * a.splits + split, place = part * G + h;
                float2 *to_ml = a.part_ml + part * QE_ATTN_GROUP_MAX + h;
                if (a.splits <= QE_ATTN_JOIN) {
                    store_through(a.part_o + place * DH + d, qe_f2{r[0], r[1]});
                    store_through(a.part_o + place * DH + d + 2, qe_f2{r[2], r[3]});
                    if (d == 0) store_through((float *)to_ml, qe_f2{top, bad ? -1.f : sum});
                } else {
                    *(qe_f4 *)(a.part_o + place * DH + d) = r;
                    if (d == 0) *to_ml = make_float2(top, bad ? -1.f : sum);
                }
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
    float2 *all_ml = (float2 *)lds; // [split][16]
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
