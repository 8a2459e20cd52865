// Causal attention of packed prompts over a paged cache.
//
// A workgroup takes 32 query rows for each of its waves, of one sequence and one key-value head
// (its tokens times the heads that share the key-value head, so that no key is read for one
// head alone), and steps through the keys 64 at a time.  Per
// step S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16: a lane's column is one query
// row, so maximum, sum and rescaling are per lane (plus one exchange between the wave's
// halves), and the registers that hold S^T's rows are, once rounded, the second product's
// operand as they stand: its k runs over the keys in the order in which they lie there, and
// V^T is read from LDS in that order by transposing reads.
//
// K and V tiles reach LDS by direct loads into one of two buffers while the other is
// worked on.  16-byte chunks are permuted within their rows at the source (LDS rows
// are contiguous for direct loads): K's by row % 8, so that the eight rows of a read's
// phase lie in different banks, V's 64-byte units by row % 4.
#include "qe_mixer_device.h"

#define BN QE_ATTN_BN

template <int DH>
__device__ __forceinline__ int k_swz(int row) {
    return row & 7;
}
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
template <int WAVES>
__device__ __forceinline__ int page_of(const QeAttnArgs &a, const int32_t *table, int k0, int len, int wave) {
    const int sub = k0 + wave * (BN / WAVES);
    return *(const __attribute__((address_space(4))) int32_t *)(uintptr_t)(table + ((sub < len ? sub : len - 1) >> a.page_log2));
}
// K and V of the part to LDS.
template <int DH, int WAVES>
__device__ __forceinline__ void load_tile(const QeAttnArgs &a, int page, int kvh, int k0, int len, int wave, short *k_lds,
                                          short *v_lds, unsigned *bad) {
    constexpr int CH = DH / 8, ROWS = 64 / CH, PART = BN / WAVES; // chunks of a row, rows of one direct load, rows of a wave
    const int sub = k0 + wave * PART, at = sub < len ? sub : (len - 1) & -PART;
    unsigned p = (unsigned)page;
    if (p >= a.n_pages) *bad = 1, p = 0;
    const size_t r0 = (((size_t)p * a.kv_heads + kvh) << a.page_log2) + (at & ((1 << a.page_log2) - 1));
    const char *kc = (const char *)a.kc + r0 * DH * 2, *vc = (const char *)a.vc + r0 * DH * 2;
    // A uniform address and a 32-bit offset: a later row's permutation differs from the first load's by a constant.
    const int lane = lane_now(), row = lane / CH, c = lane % CH;
    const unsigned k_off = row * DH * 2 + ((c ^ k_swz<DH>(row)) << 4), v_off = row * DH * 2 + ((c ^ v_swz<DH>(row)) << 4);
#pragma unroll
    for (int i = 0; i < PART / ROWS; ++i) {
        load_lds16(kc + i * 1024 + (k_off ^ (k_swz<DH>(i * ROWS) << 4)), k_lds + (wave * PART + i * ROWS) * DH);
        load_lds16(vc + i * 1024 + (v_off ^ (v_swz<DH>(i * ROWS) << 4)), v_lds + (wave * PART + i * ROWS) * DH);
    }
}

__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

// Order of a block's `n` operands of `reads` LDS reads and `products` matrix products each: `ahead` operands read first.
template <int AHEAD, int N, int READS, int PRODUCTS>
__device__ __forceinline__ void schedule() {
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * READS, 0);
#pragma unroll
    for (int i = 0; i < N - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, AHEAD * PRODUCTS, 0);
}

// A wave's query rows, 32 NB of them: column r of block n is row 32 n + r.
template <bool BF, int DH, int NB>
struct Rows {
    qe_f16v o[NB][DH / 32]; // O^T
    qe_s8 q[NB][DH / 16];
    float m[NB], l[NB]; // running maximum of the scores (scaled, in powers of two) and sum
    int place[NB];      // position of the lane's query; below 0 where it attends to nothing

    __device__ __forceinline__ void step(const QeAttnArgs &a, const short *k_lds, const short *v_lds, int k0, bool masked) {
        const int lane = lane_now(), r = lane & 31, h = lane >> 5;
        // Byte addresses in LDS.  K: chunk 2 st + h of row r is permuted by the row's low bits, so the four st of a
        // 128-byte block are one address with constants exclusive-or'ed in.  V: so are the 64-byte units d of the
        // row that a lane addresses in a transposing read.
        const int tr = (lane & 15) >> 2, el = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
        const unsigned ka = r * DH * 2 + ((h ^ k_swz<DH>(r)) << 4);
        const unsigned va = (4 * h + tr) * DH * 2 + (((el >> 3) ^ v_swz<DH>(tr)) << 4) + (el & 7) * 2;
        // Key blocks of 32 whose scores are held together: two, or one where o and q leave no registers for more.
        constexpr int KB = DH == 256 ? 1 : 2;
#pragma unroll
        for (int b0 = 0; b0 < 2; b0 += KB) {
            qe_f16v s[NB][KB];
#pragma unroll
            for (int b = 0; b < KB; ++b) {
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[n][b][i] = 0;
#pragma unroll
                for (int st = 0; st < DH / 16; ++st) {
                    const qe_s8 kf = *(const qe_s8 *)((const char *)k_lds + ((ka ^ (st & 3) << 5) + (b0 + b) * 64 * DH + (st >> 2) * 128));
#pragma unroll
                    for (int n = 0; n < NB; ++n) s[n][b] = mfma32<BF>(kf, q[n][st], s[n][b]);
                }
            }
            // The matrix products take the LDS reads as they come: four in flight (and in the second product three pairs),
            // then one more for each product.  Left alone, the scheduler reads, waits and multiplies in turn.
            schedule<4, KB * DH / 16, 1, NB>();
            union {
                unsigned u[4];
                qe_s8 v;
            } p[NB][KB][2];
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                if (masked) {
                    const int limit = place[n] - k0 - 4 * h - b0 * 32; // the last key that the row attends to, counted from the lane's first
#pragma unroll
                    for (int b = 0; b < KB; ++b)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (b * 32 + 8 * (i / 4) + i % 4 > limit) s[n][b][i] = -INFINITY;
                }
                float top = s[n][0][0];
#pragma unroll
                for (int i = 1; i < 15; i += 2) top = max3(top, s[n][0][i], s[n][0][i + 1]);
                top = max3(top, s[n][0][15], s[n][KB - 1][0]);
                if constexpr (KB == 2) {
#pragma unroll
                    for (int i = 1; i < 15; i += 2) top = max3(top, s[n][1][i], s[n][1][i + 1]);
                    top = fmaxf(top, s[n][1][15]);
                }
                top = fmaxf(top, __shfl_xor(top, 32)) * a.scale_log2;
                // The maximum that is subtracted only has to keep the powers of two in range: it follows the true one
                // when that has grown by more than 2^8, which after the first keys is rare.
                if (__any(top > m[n] + 8.f)) {
                    const float mn = fmaxf(m[n], top), f = m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[n] - mn);
#pragma unroll
                    for (int d = 0; d < DH / 32; ++d) o[n][d] *= f;
                    l[n] *= f;
                    m[n] = mn;
                }
                const float base = m[n] == -INFINITY ? 0.f : -m[n];
                float sum = 0;
#pragma unroll
                for (int b = 0; b < KB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const float x = __builtin_amdgcn_exp2f(fmaf(s[n][b][i], a.scale_log2, base));
                        const float y = __builtin_amdgcn_exp2f(fmaf(s[n][b][i + 1], a.scale_log2, base));
                        sum += x + y;
                        p[n][b][i / 8].u[i % 8 / 2] = pack2<BF>(x, y);
                    }
                l[n] += sum;
            }
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                    for (int d = 0; d < DH / 32; ++d) {
                        const unsigned vp = (va ^ (d & 3) << 6) + ((b0 + b) * 2 + ks) * 32 * DH + (d >> 2) * 256;
                        const qe_s4 x = lds_tr((const short *)((const char *)v_lds + vp)), y = lds_tr((const short *)((const char *)v_lds + (vp + 16 * DH))); // 8 rows on the permutation is the same
                        const qe_s8 vf = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
#pragma unroll
                        for (int n = 0; n < NB; ++n) o[n][d] = mfma32<BF>(vf, p[n][b][ks].v, o[n][d]);
                    }
            schedule<3, KB * 2 * DH / 32, 2, NB>();
        }
    }
};

template <bool BF, int DH, int WAVES, int NB>
__global__ __launch_bounds__(64 * WAVES, NB == 2 && DH == 256 ? 1 : 2) void k_attn_prompt(const QeAttnArgs a) {
    constexpr int BM = 32 * WAVES * NB, THREADS = 64 * WAVES;
    // two buffers, variables of their own: else the compiler has every LDS read wait for the direct loads in flight
    __shared__ __align__(16) short k_a[BN * DH], v_a[BN * DH], k_b[BN * DH], v_b[BN * DH];
    // rows with an infinity or a NaN in V, of the tiles that some rows attend to in part: from `clear` on, BM tokens at most
    __shared__ unsigned long long odd_rows[BM / BN + 2];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int split = blockIdx.x % a.splits, kvh = blockIdx.x / a.splits % a.kv_heads;
    const int tile = a.tiles - 1 - blockIdx.x / a.splits / a.kv_heads; // late rows have more keys: first
    int seq = 0;
    for (int hi = a.n_seqs; hi - seq > 1;) { // the last sequence whose first tile is not behind this one
        const int mid = (seq + hi) >> 1;
        if (qe_attn_first_tile(a.cu[mid], mid, a.group, BM) <= tile) seq = mid;
        else hi = mid;
    }
    const int local = tile - qe_attn_first_tile(a.cu[seq], seq, a.group, BM);
    unsigned bad_len = 0, bad = 0;
    const int begin = qe_checked(a.cu[seq], 0, a.n_tokens, 0, &bad_len);
    const int end = qe_checked(a.cu[seq + 1], begin, a.n_tokens, begin, &bad_len);
    const int len = qe_checked(a.kv_len[seq], 0, a.max_pages << a.page_log2, 0, &bad_len);
    if (bad_len && tid == 0) report(a.err, QE_BAD_LENGTH);
    const int n_rows = (end - begin) * a.group;
    if (local < 0 || (int64_t)local * BM >= n_rows) return; // uniform: no row of the sequence
    const int row0 = local * BM, first = len - (end - begin); // first: position of the sequence's first row
    const int32_t *table = a.table + (size_t)seq * a.table_stride;

    Rows<BF, DH, NB> w;
    const int wave_row = row0 + wave * 32 * NB;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const int row = wave_row + n * 32 + (tid & 31), h = tid >> 5 & 1;
        const bool there = row < n_rows;
        const int tok = there ? row / a.group : 0, head = kvh * a.group + (there ? row - tok * a.group : 0);
        w.place[n] = there ? first + tok : -1;
        const short *q = (const short *)a.q + (size_t)(begin + tok) * a.q_stride + (size_t)head * DH + h * 8;
#pragma unroll
        for (int s = 0; s < DH / 16; ++s) w.q[n][s] = there ? *(const qe_s8 *)(q + s * 16) : qe_s8{};
        w.m[n] = -INFINITY;
        w.l[n] = 0;
#pragma unroll
        for (int d = 0; d < DH / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) w.o[n][d][i] = 0;
    }
    // keys of the tile: up to its last row's place; below `clear` every row attends to every key
    const int last_tok = (row0 + BM < n_rows ? row0 + BM - 1 : n_rows - 1) / a.group;
    const int keys = first + last_tok + 1, clear = first + row0 / a.group + 1 > 0 ? first + row0 / a.group + 1 : 0;
    // the same for the wave
    const int wave_end = wave_row + 32 * NB < n_rows ? wave_row + 32 * NB : n_rows;
    const int wave_keys = wave_row < n_rows ? first + (wave_end - 1) / a.group + 1 : 0, wave_clear = first + wave_row / a.group + 1;
    int lo, hi;
    qe_split_range(keys > 0 ? (keys + BN - 1) / BN : 0, a.splits, split, &lo, &hi);

    int page = 0; // of the wave's part of the next tile
    auto work = [&](const short *k_lds, short *v_lds, short *k_next, short *v_next, int t) {
        __builtin_amdgcn_s_waitcnt(0x0f70); // this wave's direct loads have landed,
        lds_barrier();                      // the others' too, and no wave reads the other buffers any more
        const int k0 = t * BN;
        if (t + 1 < hi) load_tile<DH, WAVES>(a, page, kvh, k0 + BN, len, wave, k_next, v_next, &bad);
        page = page_of<WAVES>(a, table, k0 + 2 * BN, len, wave); // looked up a step before it is needed
        const bool masked = k0 + BN > clear;
        if (masked) {
            // A probability of 0 times an infinity or NaN is NaN: rows behind the end become zeros, and
            // so do elements that are not finite, which are added in the end for the rows that attend to them.
            for (int i = wave * 64 + lane_now(); i < BN * (DH / 8); i += THREADS) {
                const int row = i / (DH / 8);
                qe_s8 x = *(const qe_s8 *)(v_lds + i * 8);
                if (k0 + row >= len) {
                    *(qe_s8 *)(v_lds + i * 8) = qe_s8{};
                } else {
                    constexpr int top = BF ? 0x7f80 : 0x7c00;
                    bool odd = false;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if ((x[j] & top) == top) x[j] = 0, odd = true;
                    if (odd) {
                        *(qe_s8 *)(v_lds + i * 8) = x;
                        atomicOr(&odd_rows[t - clear / BN], 1ull << row);
                    }
                }
            }
            lds_barrier();
        }
        if (k0 < wave_keys) w.step(a, k_lds, v_lds, k0, k0 + BN > wave_clear);
    };
    if (tid < BM / BN + 2) odd_rows[tid] = 0; // a barrier before the first tile's
    if (lo < hi) {
        load_tile<DH, WAVES>(a, page_of<WAVES>(a, table, lo * BN, len, wave), kvh, lo * BN, len, wave, k_a, v_a, &bad);
        page = page_of<WAVES>(a, table, (lo + 1) * BN, len, wave);
    }
    for (int t = lo; t < hi; t += 2) {
        work(k_a, v_a, k_b, v_b, t);
        if (t + 1 < hi) work(k_b, v_b, k_a, v_a, t + 1);
    }
    if (bad && (tid & 63) == 0) report(a.err, QE_BAD_PAGE);
    const bool void_rows = __syncthreads_or(bad);
    const int lane = lane_now(), r = lane & 31, h = lane >> 5;
    for (int t = clear / BN; t < hi; ++t) {
        unsigned long long odd = t >= lo ? odd_rows[t - clear / BN] : 0;
        while (odd) { // uniform, and empty but for values that are not finite
            const int key = t * BN + __ffsll(odd) - 1;
            odd &= odd - 1;
            const size_t at = sub_row(a, table, kvh, key & ~15, &bad) + (key & 15);
            const short *v = (const short *)a.vc + at * DH + 4 * h;
#pragma unroll
            for (int n = 0; n < NB; ++n)
                if (key <= w.place[n])
#pragma unroll
                    for (int d = 0; d < DH / 32; ++d)
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const qe_s4 x = *(const qe_s4 *)(v + d * 32 + 2 * i);
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float y = from16<BF>(x[j]);
                                if (!__builtin_isfinite(y)) w.o[n][d][i + j] += y;
                            }
                            asm volatile("" ::: "memory"); // not all of the row in registers at once
                        }
        }
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const float l = w.l[n] + __shfl_xor(w.l[n], 32);
        const int row = wave_row + n * 32 + r;
        if (a.splits == 1) {
            if (row < n_rows) {
                const int tok = row / a.group, head = kvh * a.group + row - tok * a.group;
                const float inv = l == 0.f ? 0.f : 1.f / l;
                short *out = (short *)a.out + (size_t)(begin + tok) * a.out_stride + (size_t)head * DH;
#pragma unroll
                for (int d = 0; d < DH / 32; ++d)
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        uint2 x;
                        x.x = pack2<BF>(w.o[n][d][i] * inv, w.o[n][d][i + 1] * inv);
                        x.y = pack2<BF>(w.o[n][d][i + 2] * inv, w.o[n][d][i + 3] * inv);
                        if (void_rows) x = make_uint2(0, 0);
                        *(uint2 *)(out + d * 32 + 2 * i + 4 * h) = x;
                    }
            }
        } else {
            const size_t at = (((size_t)tile * a.kv_heads + kvh) * a.splits + split) * BM + row - row0;
#pragma unroll
            for (int d = 0; d < DH / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *(qe_f4 *)(a.part_o + at * DH + d * 32 + 2 * i + 4 * h) = qe_f4{w.o[n][d][i], w.o[n][d][i + 1], w.o[n][d][i + 2], w.o[n][d][i + 3]};
            if (h == 0) a.part_ml[at] = make_float2(w.m[n], void_rows ? -1.f : l);
        }
    }
}

// The splits' results joined, a wave per query row.
template <bool BF, int DH, int BM>
__global__ __launch_bounds__(256) void k_attn_prompt_join(const QeAttnArgs a) {
    constexpr int E = DH / 64;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int in_tile = blockIdx.x % (BM / 4) * 4 + wave, tile = blockIdx.x / (BM / 4) / a.kv_heads, kvh = blockIdx.x / (BM / 4) % a.kv_heads;
    int lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (qe_attn_first_tile(a.cu[mid], mid, a.group, BM) <= tile) lo = mid;
        else hi = mid;
    }
    unsigned bad = 0;
    const int begin = qe_checked(a.cu[lo], 0, a.n_tokens, 0, &bad), end = qe_checked(a.cu[lo + 1], begin, a.n_tokens, begin, &bad);
    const int local = tile - qe_attn_first_tile(a.cu[lo], lo, a.group, BM);
    const int64_t row = (int64_t)local * BM + in_tile;
    if (local < 0 || row >= (int64_t)(end - begin) * a.group) return;
    const size_t at = ((size_t)tile * a.kv_heads + kvh) * a.splits * BM + in_tile;
    float m = -INFINITY;
    bool none = false;
    for (int s = 0; s < a.splits; ++s) {
        const float2 x = a.part_ml[at + (size_t)s * BM];
        m = fmaxf(m, x.x);
        none |= x.y < 0.f;
    }
    float sum = 0, o[E];
    for (int e = 0; e < E; ++e) o[e] = 0;
    for (int s = 0; s < a.splits; ++s) {
        const float2 x = a.part_ml[at + (size_t)s * BM];
        if (x.y == 0.f) continue; // no key of that split
        const float f = x.x == -INFINITY ? 0.f : exp2f(x.x - m);
        sum += f * x.y;
        for (int e = 0; e < E; ++e) o[e] += f * a.part_o[(at + (size_t)s * BM) * DH + e * 64 + lane];
    }
    const float inv = none || sum == 0.f ? 0.f : 1.f / sum;
    const int tok = (int)(row / a.group), head = kvh * a.group + (int)(row - (int64_t)tok * a.group);
    short *out = (short *)a.out + (size_t)(begin + tok) * a.out_stride + (size_t)head * DH;
    for (int e = 0; e < E; ++e) out[e * 64 + lane] = (short)pack2<BF>(none ? 0.f : o[e] * inv, 0.f);
}

template <bool BF, int DH, int WAVES, int NB>
static hipError_t launch_waves(const QeAttnArgs &a, hipStream_t st) {
    k_attn_prompt<BF, DH, WAVES, NB><<<dim3((unsigned)(a.tiles * a.kv_heads * a.splits)), dim3(64 * WAVES), 0, st>>>(a);
    if (a.splits > 1)
        k_attn_prompt_join<BF, DH, 32 * WAVES * NB><<<dim3((unsigned)(a.tiles * a.kv_heads * (8 * WAVES * NB))), dim3(256), 0, st>>>(a);
    return hipGetLastError();
}
template <bool BF, int DH>
static hipError_t launch_prompt(const QeAttnArgs &a, int bm, hipStream_t st) {
    if constexpr (DH == 256)
        if (bm == 256) return launch_waves<BF, DH, 8, 1>(a, st);
    return launch_waves<BF, DH, 4, 1>(a, st);
}

hipError_t qe_launch_attn_prompt(const QeAttnArgs &a, int head_dim, int type, int bm, hipStream_t st) {
    if (type == QE_BF16)
        return head_dim == 64    ? launch_prompt<true, 64>(a, bm, st)
               : head_dim == 128 ? launch_prompt<true, 128>(a, bm, st)
                                 : launch_prompt<true, 256>(a, bm, st);
    return head_dim == 64    ? launch_prompt<false, 64>(a, bm, st)
           : head_dim == 128 ? launch_prompt<false, 128>(a, bm, st)
                             : launch_prompt<false, 256>(a, bm, st);
}
