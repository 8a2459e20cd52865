// Attention of single tokens over an 8-bit paged cache.
#include "qe_attn_decode.h"
#include "qe_attn_keys.h"

// ---------------------------------------------------------------------------
// As k_attn_decode: a workgroup per (sequence, key-value head, split of its length), its four waves each over their own steps
// (KeyWave), no barrier before the end.
//
// Bound by memory where lengths are long: 24 ragged sequences of up to 8,095 keys, 8 heads of 128 of e4m3, are 175 MB and take 42 us, 4.2 TB/s
// (the longest sequences' last steps find half of the GPU done).  900 keys of one sequence, 2 heads of 256, take 10 us: length and page, keys and
// values, the exchange and the join, one after the other.  Steps of 64 keys in place of 32: 48 us for 42.
// ---------------------------------------------------------------------------
template <bool BF, int DH, int CT, bool ONCE>
__global__ __launch_bounds__(256, DH == 64 ? 4 : 3) void k_attn_decode8(const QeAttn8Args x) {
    const QeAttnArgs &a = x.a;
    typedef KeyWave<BF, DH, CT, 0, ONCE> Wave;
    constexpr int HEADS = DH == 256 ? 8 : 16; // of results in LDS at a time: with 16 of 256 two workgroups fit a CU, else three
    __shared__ __align__(16) short lds[4][HEADS * DH * 2];
    __shared__ float2 ml[4][16];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    // Workgroups go to the eight XCDs in turn: where the last one joins, a sequence's and head's all go to one.
    const bool near = a.splits > 1 && a.splits <= QE_ATTN_JOIN;
    const int at = near ? blockIdx.x / 8 : blockIdx.x, split = at % a.splits, item = near ? at / a.splits * 8 + blockIdx.x % 8 : at / a.splits;
    if (item >= a.n_seqs * a.kv_heads) return;
    const int seq = item / a.kv_heads, kvh = item % a.kv_heads;
    unsigned bad_len = 0;
    const int32_t *table = a.table + (size_t)seq * a.table_stride;
    // the wave's first pages, looked up along with the length, as it is if the length is no longer than the host believed
    const unsigned first = ((unsigned)split * a.steps + wave) * Wave::TILE, cap = a.max_pages - 1;
    typename Wave::Pages pages;
#pragma unroll
    for (int b = 0; b < Wave::NB; ++b) pages[b] = scalar_load(table + ((first + 16 * b) >> a.page_log2 < cap ? (first + 16 * b) >> a.page_log2 : cap));
    Wave w;
    w.begin(a, seq, kvh, lane);
    const int len = qe_checked(scalar_load(a.kv_len + seq), 0, a.max_pages << a.page_log2, 0, &bad_len);
    const int steps = qe_attn_decode_steps(len, a.steps, a.splits), active = qe_attn_decode_active(len, steps);
    if (split >= (active > 1 ? active : 1)) return; // a sequence without keys is the first workgroup's, which writes zeros

    const int tiles = (len + Wave::TILE - 1) / Wave::TILE, lo = split * steps + wave, hi = split * steps + steps < tiles ? split * steps + steps : tiles;
    if (lo < hi) {
        if (steps != a.steps) pages = Wave::look_up(a, table, lo * Wave::TILE, 0, len);
        else if (lo * Wave::TILE + 16 >= len) pages[1] = pages[0]; // behind the end any page of the step's
    }
    run_steps(w, a, x.ks, x.vs, table, kvh, 0, 0, len, lo, hi, pages, (uint8_t *)lds[wave]);
    w.end();
    finish_decode<BF, DH, HEADS>(a, item, split, active, w.acc, w.m, w.l, w.bad, bad_len, [&](int v, int h) { return (float *)lds[v] + h * DH; }, lds[0], ml);
}

// Many splits' results of several sequences joined: a workgroup a row, its four waves every fourth split.  (k_attn_join, which has
// all reads of a row in flight at once, is for one long sequence's few rows: 24 ragged ones, 16 heads of 256, 32 splits: 52 us a
// call with it, 40 with this.)
template <bool BF, int DH>
__global__ __launch_bounds__(256) void k_attn_join_rows(const QeAttnArgs a) {
    constexpr int E = DH / 64;
    __shared__ float o_s[4][DH], sum_s[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, seq = blockIdx.x / a.q_heads, head = blockIdx.x % a.q_heads, kvh = head / a.group, h = head % a.group;
    unsigned bad_len = 0;
    const int len = qe_checked(scalar_load(a.kv_len + seq), 0, a.max_pages << a.page_log2, 0, &bad_len);
    const int n = qe_attn_decode_active(len, qe_attn_decode_steps(len, a.steps, a.splits));
    if (n <= 1) return; // its one workgroup has written the row
    const size_t at = ((size_t)seq * a.kv_heads + kvh) * a.splits;
    float m = -INFINITY;
    bool bad = false;
    for (int s = lane; s < n; s += 64) {
        const float2 x = a.part_ml[(at + s) * QE_ATTN_GROUP_MAX + h];
        m = fmaxf(m, x.x);
        bad |= x.y < 0.f;
    }
    for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
    bad = __any(bad);
    float sum = 0, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0;
#pragma unroll 8
    for (int s = wave; s < n; s += 4) {
        const float2 x = a.part_ml[(at + s) * QE_ATTN_GROUP_MAX + h];
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = a.part_o[((at + s) * a.group + h) * DH + e * 64 + lane];
        const float f = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((x.x - m) * a.scale_log2);
        const bool any = x.y != 0.f; // else no key
        sum += any ? f * x.y : 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += any ? f * v[e] : 0.f;
    }
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
static hipError_t launch_decode8(const QeAttn8Args &x, hipStream_t st) {
    const QeAttnArgs &a = x.a;
    const unsigned units = (unsigned)(a.n_seqs * a.kv_heads), whole = a.splits > 1 && a.splits <= QE_ATTN_JOIN ? (units + 7) / 8 * 8 : units;
    if (a.once) k_attn_decode8<BF, DH, CT, true><<<dim3(whole * a.splits), dim3(256), 0, st>>>(x);
    else k_attn_decode8<BF, DH, CT, false><<<dim3(whole * a.splits), dim3(256), 0, st>>>(x);
    if (a.splits > QE_ATTN_JOIN && a.n_seqs > 1) k_attn_join_rows<BF, DH><<<dim3((unsigned)(a.n_seqs * a.q_heads)), dim3(256), 0, st>>>(a);
    else if (a.splits > QE_ATTN_JOIN) k_attn_join<BF, DH><<<dim3((unsigned)(a.n_seqs * a.q_heads * (DH / 64))), dim3(1024), 0, st>>>(a);
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
