// Attention of blocks of query rows on v_mfma_f32_32x32x16: the tiles' layout in LDS, a wave's 32 rows, the join of splits.
// For caches of 16 bits (qe_attn_prompt.hip) and of 8 (qe_attn_prompt8.hip).
#pragma once
#include "qe_mixer_device.h"

__device__ __forceinline__ int k_swz(int row) { return row & 7; }
template <int DH>
__device__ __forceinline__ int v_swz(int row) {
    return DH == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2;
}

// The lane's number, made where it is needed: kept, and what follows from it, it would take registers that the loop over
// the tiles does not have, and reloads of spilled ones wait for the direct loads in flight.
__device__ __forceinline__ int lane_now() {
    int lane;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
    return lane;
}

// The page of a wave's part of the tile of BN keys from position k0 on: all of the part's rows lie in one.
// Rows behind the end may lie in none, then any of the sequence's do (their probabilities are zero).
template <int BN, int WAVES>
__device__ __forceinline__ int page_of(const QeAttnArgs &a, const int32_t *table, int k0, int len, int wave) {
    const int sub = k0 + wave * (BN / WAVES);
    return scalar_load(table + ((sub < len ? sub : len - 1) >> a.page_log2));
}
// The part's rows of K or V to LDS.
template <int DH, int BN, int WAVES, bool IS_K>
__device__ __forceinline__ void load_part(const QeAttnArgs &a, int page, int kvh, int k0, int len, int wave, short *lds) {
    constexpr int CH = DH / 8, ROWS = 64 / CH, PART = BN / WAVES; // chunks of a row, rows of one direct load, rows of a wave
    const int sub = k0 + wave * PART, at = sub < len ? sub : (len - 1) & -PART;
    unsigned known = 0; // that a page is none: lost_pages
    const size_t r0 = page_row(a, page, kvh, at, &known);
    const char *from = (const char *)(IS_K ? a.kc : a.vc) + r0 * DH * 2;
    // A uniform address and a 32-bit offset: a later row's permutation differs from the first load's by a constant.
    const int lane = lane_now(), row = lane / CH, c = lane % CH;
    const unsigned off = row * DH * 2 + ((c ^ (IS_K ? k_swz(row) : v_swz<DH>(row))) << 4);
#pragma unroll
    for (int i = 0; i < PART / ROWS; ++i)
        load_lds16_from(from, PART * DH * 2, off ^ ((IS_K ? k_swz(i * ROWS) : v_swz<DH>(i * ROWS)) << 4), i * 1024, lds + (wave * PART + i * ROWS) * DH);
}

// Whether one of the `n` pages of a sequence is none of the cache's: of the thread's share of them.  Each workgroup
// looks at all, since the rows of all are zeros then; four at a time, the last again behind the end.
template <int THREADS>
__device__ __forceinline__ int lost_pages(const QeAttnArgs &a, const int32_t *table, int n, int tid) {
    int lost = 0;
    for (int i = tid; i < n; i += 4 * THREADS) {
        unsigned p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = table[i + j * THREADS < n ? i + j * THREADS : n - 1];
#pragma unroll
        for (int j = 0; j < 4; ++j) lost |= p[j] >= a.n_pages;
    }
    return lost;
}

__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
// the larger of the values of lanes l and l ^ 32
__device__ __forceinline__ float max_halves(float x) {
    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}

// The order of N matrix products that take READS LDS reads each: the reads of AHEAD of them first, then those of one for
// each product.  Left alone, the scheduler reads, waits and multiplies in turn.
template <int AHEAD, int N, int READS>
__device__ __forceinline__ void schedule() {
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * READS, 0);
#pragma unroll
    for (int i = 0; i < N - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
}

template <int KB>
struct Probs {
    union {
        unsigned u[4];
        qe_s8 v;
    } p[KB][2]; // 16 keys each, as the second product's operand
};

// A wave's 32 query rows, lane r of either half row r, and their scores of KB blocks of 32 keys.
template <int KB>
struct Scores {
    qe_f16v s[KB]; // S^T

    // keys behind `limit`, counted from the lane's first, are not attended to
    __device__ __forceinline__ void mask(int limit) {
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (b * 32 + 8 * (i / 4) + i % 4 > limit) s[b][i] = -INFINITY;
    }
    // probabilities: 0 there
    __device__ __forceinline__ void clear(int limit) {
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (b * 32 + 8 * (i / 4) + i % 4 > limit) s[b][i] = 0;
    }
    template <bool BF>
    __device__ __forceinline__ void pack(Probs<KB> &p) const {
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 16; i += 2) p.p[b][i / 8].u[i % 8 / 2] = pack2<BF>(s[b][i], s[b][i + 1]);
    }
    __device__ __forceinline__ float top() const { // of the row
        float t = s[0][0];
#pragma unroll
        for (int i = 1; i < 15; i += 2) t = max3(t, s[0][i], s[0][i + 1]);
        t = max3(t, s[0][15], s[KB - 1][0]);
        if constexpr (KB == 2) {
#pragma unroll
            for (int i = 1; i < 15; i += 2) t = max3(t, s[1][i], s[1][i + 1]);
            t = fmaxf(t, s[1][15]);
        }
        return max_halves(t);
    }
};
template <bool BF, int DH>
struct Rows {
    static constexpr int LAG = 8;
    qe_f16v o[DH / 32]; // O^T
    qe_s8 q[DH / 16];
    float m, l; // running maximum of the scores (scaled, in powers of two) and sum
    int place;  // position of the lane's query; below 0 where it attends to nothing

    // S^T = K Q^T of KB blocks from block b0 of the tile on.  Chunk 2 st + h of K's row r is permuted by the row's low
    // bits, so the four st of a 128-byte block are one address with constants exclusive-or'ed in.
    template <int KB>
    __device__ __forceinline__ void scores(const short *k_lds, int b0, Scores<KB> &x) const {
        const int lane = lane_now(), r = lane & 31, h = lane >> 5;
        const unsigned ka = r * DH * 2 + ((h ^ k_swz(r)) << 4);
#pragma unroll
        for (int b = 0; b < KB; ++b) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x.s[b][i] = 0;
#pragma unroll
            for (int st = 0; st < DH / 16; ++st)
                x.s[b] = mfma32<BF>(*(const qe_s8 *)((const char *)k_lds + ((ka ^ (st & 3) << 5) + (b0 + b) * 64 * DH + (st >> 2) * 128)), q[st], x.s[b]);
        }
    }
    // The maximum that is subtracted only has to keep the powers of two in range: it follows the true one
    // when that has grown by more than 2^8, which after the first keys is rare.
    __device__ __forceinline__ void raise(float top) {
        if (__any(top > m + (float)LAG)) {
            const float mn = fmaxf(m, top), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            if (__any(m != -INFINITY)) // else nothing is summed yet
#pragma unroll
                for (int d = 0; d < DH / 32; ++d) o[d] *= f;
            l *= f;
            m = mn;
        }
    }
    template <int KB>
    __device__ __forceinline__ void exponentials(float scale, const Scores<KB> &x, Probs<KB> &p) {
        const float base = exponent_base<BF, LAG>(m);
        float sum[2] = {0, 0};
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float y = __builtin_amdgcn_exp2f(fmaf(x.s[b][i], scale, base));
                const float z = __builtin_amdgcn_exp2f(fmaf(x.s[b][i + 1], scale, base));
                sum[0] += y;
                sum[1] += z;
                p.p[b][i / 8].u[i % 8 / 2] = pack2<BF>(y, z);
            }
        l += sum[0] + sum[1];
    }
    // the sums count other units: RowUnits
    __device__ __forceinline__ void times(float f) {
#pragma unroll
        for (int d = 0; d < DH / 32; ++d) o[d] *= f;
        l *= f;
    }
    // the scores become probabilities, not rounded yet; in units of 2^unit
    template <int KB>
    __device__ __forceinline__ void weigh(float scale, float unit, Scores<KB> &x) {
        const float base = exponent_base<BF, LAG>(m) - unit;
        float sum[2] = {0, 0};
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                x.s[b][i] = __builtin_amdgcn_exp2f(fmaf(x.s[b][i], scale, base));
                sum[i & 1] += x.s[b][i];
            }
        l += sum[0] + sum[1];
    }
    // O^T += V^T P^T.  The 64-byte units d of the row that a lane addresses in a transposing read are one address with
    // constants, too.
    template <int KB>
    __device__ __forceinline__ void values(const short *v_lds, int b0, const Probs<KB> &p) {
        const int lane = lane_now(), h = lane >> 5, tr = (lane & 15) >> 2, el = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
        const unsigned va = (4 * h + tr) * DH * 2 + (((el >> 3) ^ v_swz<DH>(tr)) << 4) + (el & 7) * 2;
#pragma unroll
        for (int ks = 0; ks < 2 * KB; ++ks)
#pragma unroll
            for (int d = 0; d < DH / 32; ++d) {
                const unsigned vp = (va ^ (d & 3) << 6) + (b0 * 2 + ks) * 32 * DH + (d >> 2) * 256;
                const qe_s4 x = lds_tr((const short *)((const char *)v_lds + vp)), y = lds_tr((const short *)((const char *)v_lds + (vp + 16 * DH))); // 8 rows on the permutation is the same
                o[d] = mfma32<BF>(qe_s8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]}, p.p[ks / 2][ks % 2].v, o[d]);
            }
    }
    // The rows to `out` (direct), or as a split's partial results.
    template <int BM>
    __device__ __forceinline__ void finish(const QeAttnArgs &a, int begin, int n_rows, int row0, int wave_row, int tile, int kvh, int split, bool direct) const {
        const int lane = lane_now(), r = lane & 31, h = lane >> 5;
        const float sum = l + __shfl_xor(l, 32);
        const int row = wave_row + r;
        if (direct) {
            if (row >= n_rows) return;
            const int tok = row / a.group, head = kvh * a.group + row - tok * a.group;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            short *out = (short *)a.out + (size_t)(begin + tok) * a.out_stride + (size_t)head * DH;
#pragma unroll
            for (int d = 0; d < DH / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    uint2 x;
                    x.x = pack2<BF>(o[d][i] * inv, o[d][i + 1] * inv);
                    x.y = pack2<BF>(o[d][i + 2] * inv, o[d][i + 3] * inv);
                    *(uint2 *)(out + d * 32 + 2 * i + 4 * h) = x;
                }
        } else {
            const size_t at = (((size_t)tile * a.kv_heads + kvh) * a.splits + split) * BM + row - row0;
#pragma unroll
            for (int d = 0; d < DH / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *(qe_f4 *)(a.part_o + at * DH + d * 32 + 2 * i + 4 * h) = qe_f4{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
            if (h == 0) a.part_ml[at] = make_float2(m, sum);
        }
    }
};

// The splits' results joined, W waves per query row: one, but for few rows over more than 8 splits a workgroup's four, each
// over every fourth split.  (The call with one wave a row and with four, of 16 and 2 heads of 256: 30 tokens after 10,000, 40
// splits, 50 and 39 us, but 1000 tokens, 4 splits, 50 and 58; of 32 and 8 heads of 128: 64 after 5200, 21 splits, 42 and 36,
// but 200 after 4000, 9 splits, 45 and 50.)
template <bool BF, int DH, int BM, int W>
__global__ __launch_bounds__(256) void k_attn_prompt_join(const QeAttnArgs a) {
    constexpr int E = DH / 64;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, item = blockIdx.x / (BM * W / 4);
    const int in_tile = blockIdx.x % (BM * W / 4) * (4 / W) + wave / W, tile = item / a.kv_heads, kvh = item % a.kv_heads;
    int seq = 0;
    for (int hi = a.n_seqs; hi - seq > 1;) {
        const int mid = (seq + hi) >> 1;
        if (qe_attn_first_tile(qe_clamped(scalar_load(a.cu + mid), 0, a.n_tokens), mid, a.group, BM) <= tile) seq = mid;
        else hi = mid;
    }
    unsigned bad = 0;
    int begin, end;
    qe_rows_of(scalar_load(a.cu + seq), scalar_load(a.cu + seq + 1), a.n_tokens, &begin, &end, &bad);
    const int local = tile - qe_attn_first_tile(begin, seq, a.group, BM);
    const int64_t row = (int64_t)local * BM + in_tile;
    // (of one row or of none with four waves a row: uniform there)
    if (local < 0 || row >= (int64_t)(end - begin) * a.group) return;
    const size_t at = ((size_t)tile * a.kv_heads + kvh) * a.splits * BM + in_tile;
    float m = -INFINITY;
    for (int s = lane; s < a.splits; s += 64) m = fmaxf(m, a.part_ml[at + (size_t)s * BM].x);
    for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
    float sum = 0, o[E];
    for (int e = 0; e < E; ++e) o[e] = 0;
#pragma unroll 4
    for (int s = wave % W; s < a.splits; s += W) {
        const float2 x = a.part_ml[at + (size_t)s * BM];
        float y[E];
        for (int e = 0; e < E; ++e) y[e] = a.part_o[(at + (size_t)s * BM) * DH + e * 64 + lane];
        const float f = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.x - m);
        if (x.y == 0.f) continue; // no key of that split
        sum += f * x.y;
        for (int e = 0; e < E; ++e) o[e] += f * y[e];
    }
    if constexpr (W == 4) {
        __shared__ float o_s[4][DH], sum_s[4];
        for (int e = 0; e < E; ++e) o_s[wave][e * 64 + lane] = o[e];
        if (lane == 0) sum_s[wave] = sum;
        __syncthreads();
        if (wave) return;
        sum = (sum_s[0] + sum_s[1]) + (sum_s[2] + sum_s[3]);
        for (int e = 0; e < E; ++e)
            o[e] = (o_s[0][e * 64 + lane] + o_s[1][e * 64 + lane]) + (o_s[2][e * 64 + lane] + o_s[3][e * 64 + lane]);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int tok = (int)(row / a.group), head = kvh * a.group + (int)(row - (int64_t)tok * a.group);
    short *out = (short *)a.out + (size_t)(begin + tok) * a.out_stride + (size_t)head * DH;
    for (int e = 0; e < E; ++e) out[e * 64 + lane] = (short)pack2<BF>(o[e] * inv, 0.f);
}

template <bool BF, int DH, int BM>
static void launch_prompt_join(const QeAttnArgs &a, hipStream_t st) {
    const unsigned rows = (unsigned)(a.tiles * a.kv_heads) * BM;
    if (a.splits > 8 && rows <= 4096) k_attn_prompt_join<BF, DH, BM, 4><<<dim3(rows), dim3(256), 0, st>>>(a);
    else if (a.splits > 1) k_attn_prompt_join<BF, DH, BM, 1><<<dim3(rows / 4), dim3(256), 0, st>>>(a);
}
