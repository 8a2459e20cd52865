// The gated delta rule.  For each value head and token, S its state [dim_k][dim_v]:
//   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = scale S^T q.
//
// Single tokens: qe_delta_decode's kernel, bound by reading and writing the states.
//
// Prompts, in chunks of 64 tokens.  With b the running sum of g in the chunk, S its state
// before it and fade_ij = e^(b_i - b_j), substituting the recurrence into itself gives
//   u_i + sum_{j<i} beta_i fade_ij (k_i . k_j) u_j = beta_i (v_i - e^(b_i) S^T k_i),
// a unit lower triangular system whose matrix I + A depends on no state.  So
//   U = (I + A)^-1 diag(beta) (V - diag(e^b) K S),
//   O = diag(e^b) Q S + M U,   M_ij = fade_ij (q_i . k_j) for j <= i,
//   S' = e^(b_last) S + sum_i e^(b_last - b_i) k_i u_i^T.
// k_delta_chunks makes T = (I + A)^-1 diag(beta) and M of every chunk and head at once;
// k_delta_scan then walks a sequence's chunks with the state in registers, a workgroup per
// (sequence, value head, 16 columns of the state).
//
// State and sums are in 32 bits, b in 64 (a difference of two long sums).  Products run on the bf16
// matrix cores at 32-bit precision: an operand is cut into planes of 8 significant bits, x = x0 + x1
// + x2 (bf16 inputs are one plane, fp16 two, fp32 three), and of the planes' products, each exact
// and summed in 32 bits, those down to 2^-16 of the largest are taken; what is left out is
// a rounding of 32 bits.  Six such products of 16x16x32 take 96 cycles where v_mfma_f32_16x16x4
// takes 256 (bf16 inputs: three products, 48).  Results in 16 bits need two planes less
// exactly: see NO below.
#include "qe_mixer_device.h"

template <typename T>
__device__ __forceinline__ qe_f4 load4(const T *p) {
    if constexpr (sizeof(T) == 4) {
        return *(const qe_f4 *)p;
    } else {
        const auto x = *(const __attribute__((ext_vector_type(4))) T *)p;
        return qe_f4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
    }
}

// v_mfma_f32_16x16x4: A lane l supplies row l % 16, k = l / 16; B column l % 16; D as mfma16.
// With operands read 4 floats at a time, product j of a group of 16 k takes k = 4 (l / 16) + j
// from both sides, and a D result is a B operand as it stands.
__device__ __forceinline__ qe_f4 mma4(qe_f4 a, qe_f4 b, qe_f4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

// What a key or query with this sum of squares is multiplied by.  Where the sum passes 32 bits it is not known: NaN, in prompts
// and single steps alike (1 / sqrt(inf) would make a silent zero of the row).
__device__ __forceinline__ float norm_factor(float squares, bool l2norm) {
    return !__builtin_isfinite(squares) ? NAN : l2norm ? 1.f / sqrtf(squares + 1e-6f) : 1.f;
}

__device__ __forceinline__ float log_decay(float g) { return g < -1e4f ? -1e4f : g; } // e^-1e4 is 0; a NaN stays

// Planes of a type's values, and planes that the product for the outputs takes of S, M and U.
template <typename T>
constexpr int planes_of() { return sizeof(T) == 4 ? 3 : __is_same(T, __bf16) ? 1 : 2; }

__device__ __forceinline__ short bf16_bits(float x) { return __builtin_bit_cast(short, (__bf16)x); }
// the next plane of x, which is taken off it
__device__ __forceinline__ short next_plane(float &x) {
    const __bf16 h = (__bf16)x;
    x -= (float)h;
    return __builtin_bit_cast(short, h);
}
// 4 values to N planes, `apart` elements from each other.  Planes are cut off here, not rounded
// (8 bits of 24 each): half the instructions, in the chain that bounds a prompt.  The matrices
// that they meet are rounded, so what is left out of a product has no sign of its own.
template <int N>
__device__ __forceinline__ void put4(short *p, int apart, qe_f4 x) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        unsigned u[4];
        for (int j = 0; j < 4; ++j) u[j] = __float_as_uint(x[j]);
        uint2 h;
        h.x = __builtin_amdgcn_perm(u[1], u[0], 0x07060302);
        h.y = __builtin_amdgcn_perm(u[3], u[2], 0x07060302);
        *(uint2 *)(p + i * apart) = h;
        if (i + 1 < N)
            for (int j = 0; j < 4; ++j) x[j] -= __uint_as_float(u[j] & 0xffff0000u);
    }
}
// Products of planes i of a and j of b with i + j <= LIM, summed apart by size: the sums of many
// small ones are then as exact as the large one's, and the chains overlap.
template <int NA, int NB, int LIM>
__device__ __forceinline__ void mul_planes(const qe_s8 *a, const qe_s8 *b, qe_f4 *acc) {
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
            if (i + j <= LIM) acc[i + j] = mfma16<true>(a[i], b[j], acc[i + j]);
}

// ---------------------------------------------------------------------------
// Which sequences of a call are computed (rules in qe_mixer_plan.h).
// ---------------------------------------------------------------------------
// Up to 256 sequences: by every workgroup of its own sequence, else by a launch before.
__device__ __forceinline__ int slots_of(const QeDeltaArgs &a, int seq, int in_i, int out_i) { // what is wrong; workgroup-uniform
    if (a.skip) return a.skip[seq];
    int what = qe_slot_pair(a.n_slots, in_i, out_i);
    if (a.n_seqs > 1) {
        const int j = threadIdx.x;
        if (__syncthreads_or(j < a.n_seqs ? qe_slot_conflict(seq, out_i, j, a.slots_in[j], a.slots_out[j]) : 0) && !what) what = QE_SLOT_SHARED;
    }
    return what;
}
__device__ __forceinline__ void report_slots(const QeDeltaArgs &a, int what) {
    if (threadIdx.x == 0 && what && !a.skip) report(a.err, what == QE_SLOT_OUTSIDE ? QE_BAD_SLOT : QE_BAD_SHARED_SLOT);
}
__global__ __launch_bounds__(256) void k_delta_slots(const QeDeltaArgs a) {
    const int i = blockIdx.x;
    const int in_i = a.slots_in[i], out_i = a.slots_out[i];
    int what = qe_slot_pair(a.n_slots, in_i, out_i);
    int shared = 0;
    for (int j = threadIdx.x; j < a.n_seqs; j += 256) shared |= qe_slot_conflict(i, out_i, j, a.slots_in[j], a.slots_out[j]);
    shared = __syncthreads_or(shared);
    if (threadIdx.x == 0) {
        if (!what && shared) what = QE_SLOT_SHARED;
        a.skip[i] = (unsigned char)what;
        if (what) report(a.err, what == QE_SLOT_OUTSIDE ? QE_BAD_SLOT : QE_BAD_SHARED_SLOT);
    }
}

// ---------------------------------------------------------------------------
// One token per sequence: a workgroup per (sequence, value head, 32 columns of its state),
// a thread 4 columns of DK / 32 rows.  S^T k and S^T q are summed in the one pass over the old
// state that it needs (S'^T q = e^g S^T q + (k . q) u), so the state is read once, kept
// in registers and written once.  Bound by memory: 64 sequences of 32 heads of 128 x 128, 270 MB: 51 us,
// 5.3 TB/s (a large copy reaches 5.1).  One sequence: 5 us, latency.  States pass the caches by: until the next
// token the other layers' come through them.  Per call on states of many layers in turn: 16 sequences 19.2 -> 13.5 us, 64
// 58.9 -> 53.5; on the same states over and over 15.1 -> 12.7 and 47.7 -> 50.7.
// ---------------------------------------------------------------------------
template <typename IN, int DK, int DV>
__global__ __launch_bounds__(256) void k_delta_decode(const QeDeltaArgs a) {
    constexpr int ROWS = DK / 32;
    __shared__ float qk[2][DK];
    __shared__ float part[4][3];
    __shared__ __align__(16) qe_f4 red[4][2][8];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int slice = blockIdx.x % (DV / 32), head = blockIdx.x / (DV / 32) % a.v_heads, seq = blockIdx.x / (DV / 32) / a.v_heads;
    const int kh = head / a.group, col = slice * 32 + (tid & 7) * 4, row = tid >> 3;
    IN *out = (IN *)a.out + (size_t)seq * a.out_stride + (size_t)head * DV;
    const int in_i = a.slots_in[seq], out_i = a.slots_out[seq];
    const int what = slots_of(a, seq, in_i, out_i);
    report_slots(a, what);
    if (what) {
        if (tid < 32) out[slice * 32 + tid] = (IN)0.f;
        return;
    }
    qe_f4 s[ROWS];
    const float *from = a.pool + ((size_t)(in_i < 0 ? 0 : in_i) * a.v_heads + head) * DK * DV;
    for (int i = 0; i < ROWS; ++i) s[i] = in_i < 0 ? qe_f4{0, 0, 0, 0} : __builtin_nontemporal_load((const qe_f4 *)(from + (size_t)(row + 32 * i) * DV + col));

    float x = 0, y = 0;
    if (tid < DK) {
        x = (float)((const IN *)a.q)[(size_t)seq * a.q_stride + (size_t)kh * DK + tid];
        y = (float)((const IN *)a.k)[(size_t)seq * a.k_stride + (size_t)kh * DK + tid];
        qk[0][tid] = x;
        qk[1][tid] = y;
    }
    float xx = x * x, yy = y * y, xy = x * y;
    for (int d = 32; d; d >>= 1) xx += __shfl_xor(xx, d), yy += __shfl_xor(yy, d), xy += __shfl_xor(xy, d);
    if (lane == 0) part[wave][0] = xx, part[wave][1] = yy, part[wave][2] = xy;
    const float e = expf(log_decay(a.g[(size_t)seq * a.v_heads + head])), beta = a.beta[(size_t)seq * a.v_heads + head];
    const qe_f4 v = load4((const IN *)a.v + (size_t)seq * a.v_stride + (size_t)head * DV + col);
    __syncthreads();
    xx = (part[0][0] + part[1][0]) + (part[2][0] + part[3][0]);
    yy = (part[0][1] + part[1][1]) + (part[2][1] + part[3][1]);
    xy = (part[0][2] + part[1][2]) + (part[2][2] + part[3][2]);
    const float rq = (a.l2norm ? norm_factor(xx, true) : 1.f) * a.scale, rk = norm_factor(yy, a.l2norm);
    qe_f4 sk = {0, 0, 0, 0}, sq = {0, 0, 0, 0};
    for (int i = 0; i < ROWS; ++i) {
        s[i] *= e;
        sq += s[i] * qk[0][row + 32 * i];
        sk += s[i] * qk[1][row + 32 * i];
    }
    for (int d = 8; d < 64; d <<= 1)
        for (int c = 0; c < 4; ++c) sk[c] += __shfl_xor(sk[c], d), sq[c] += __shfl_xor(sq[c], d);
    if (lane < 8) red[wave][0][lane] = sk, red[wave][1][lane] = sq;
    __syncthreads();
    sk = (red[0][0][tid & 7] + red[1][0][tid & 7]) + (red[2][0][tid & 7] + red[3][0][tid & 7]);
    const qe_f4 u = beta * (v - rk * sk);
    if (out_i >= 0) {
        float *to = a.pool + ((size_t)out_i * a.v_heads + head) * DK * DV;
        for (int i = 0; i < ROWS; ++i) __builtin_nontemporal_store(s[i] + (rk * qk[1][row + 32 * i]) * u, (qe_f4 *)(to + (size_t)(row + 32 * i) * DV + col));
    }
    if (tid < 8) {
        sq = (red[0][1][tid] + red[1][1][tid]) + (red[2][1][tid] + red[3][1][tid]);
        const qe_f4 o = rq * (sq + (rk * xy) * u);
        for (int c = 0; c < 4; ++c) out[col + c] = (IN)o[c];
    }
}

// ---------------------------------------------------------------------------
// T and M of every chunk, a workgroup per (chunk, key head).  K K^T and Q K^T are shared by the
// key head's value heads.  Wave w has rows 16 w .. + 15.  The inverse of I + A by blocks of
// 16, in 32 bits: the diagonal ones by substitution, a lane per column; then by distance
// from the diagonal T_ij = -T_ii sum_k A_ik T_kj.
// Workspace of a chunk and value head, as k_delta_scan's waves load it: T's planes and M's, each
// [wave][32 columns][plane][lane][8] (columns that lie above the diagonal for all of a wave's rows
// are not written), then per token e^b / |k|, scale e^b / |q|, e^(b_last - b) / |k|, and
// e^(b_last).  fp16 and fp32 keys and queries are cut into planes here too, for a chunk and key
// head: K [plane][64][DK] as it lies in LDS, Q [wave][32 of DK][plane][lane][8].
// 8192 bf16 tokens of 16 key and 32 value heads of 128: 68 us (fp16 93, fp32 131), against 52 for its reads and writes at a large copy's
// rate; the rest is the barriers between a head's short steps.
// ---------------------------------------------------------------------------
template <int DK>
__device__ __forceinline__ int key_swz(int row) { // of the 16-byte chunk index: 8 rows' pairs of chunks in different banks
    return DK == 64 ? ((row >> 1) & 3) << 1 : (row & 7) << 1;
}

template <typename IN>
__device__ __forceinline__ void load8_planes(const IN *p, bool there, qe_s8 *h, float &square) {
    constexpr int NP = planes_of<IN>();
    float x[8];
    if constexpr (sizeof(IN) == 4) {
        const qe_f4 a = there ? *(const qe_f4 *)p : qe_f4{0, 0, 0, 0}, b = there ? *(const qe_f4 *)(p + 4) : qe_f4{0, 0, 0, 0};
        for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
    } else {
        const qe_s8 a = there ? *(const qe_s8 *)p : qe_s8{};
        for (int i = 0; i < 8; ++i) x[i] = from16<__is_same(IN, __bf16)>(a[i]);
        if constexpr (NP == 1) h[0] = a;
    }
    for (int i = 0; i < 8; ++i) square += x[i] * x[i];
    if constexpr (NP > 1)
        for (int n = 0; n < NP; ++n)
            for (int i = 0; i < 8; ++i) h[n][i] = next_plane(x[i]);
}

// (Three workgroups a CU, as the LDS allows: 1999 fp32 tokens of 16 and 32 heads of 128 take 38 us, with two 46, although
// the 168 registers of three spill 14 there, in no other type or size.  One chunk: 10 us, its steps' latency.)
template <typename IN, int DK>
__global__ __launch_bounds__(256, 3) void k_delta_chunks(const QeDeltaArgs a) {
    constexpr int LD = 68, KS = DK / 32, NP = planes_of<IN>(), NO = sizeof(IN) == 4 ? 3 : 2;
    // K's planes as they are in k_delta_scan's LDS, then the heads' matrices
    constexpr int K_BYTES = NP * 64 * DK * 2, M_BYTES = 3 * 64 * LD * 4;
    __shared__ __align__(16) char lds[K_BYTES > M_BYTES ? K_BYTES : M_BYTES];
    short *k_s = (short *)lds;
    float *A = (float *)lds, *T = A + 64 * LD, *M = T + 64 * LD;
    __shared__ double b_s[64]; // in powers of two, as the hardware's exponential takes them
    __shared__ float kk_s[64], rk_s[64], rq_s[64], beta_s[64];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 15, c = lane >> 4;
    const int parts = a.v_heads / a.heads, chunk = blockIdx.x / parts, head0 = blockIdx.x % parts * a.heads, kh = head0 / a.group;
    int seq = 0;
    for (int hi = a.n_seqs; hi - seq > 1;) {
        const int mid = (seq + hi) >> 1;
        if (qe_delta_first_chunk(a.cu[mid], mid) <= chunk) seq = mid;
        else hi = mid;
    }
    unsigned bad = 0;
    int begin, end;
    qe_rows_of(scalar_load(a.cu + seq), scalar_load(a.cu + seq + 1), a.n_tokens, &begin, &end, &bad);
    const int64_t local = chunk - qe_delta_first_chunk(begin, seq);
    if (bad || local < 0 || local * QE_DELTA_C >= end - begin) return; // uniform
    const int t0 = begin + (int)local * QE_DELTA_C, n = end - t0 < QE_DELTA_C ? end - t0 : QE_DELTA_C;

    const IN *q = (const IN *)a.q + (size_t)kh * DK + 8 * c, *k = (const IN *)a.k + (size_t)kh * DK + 8 * c;
    const int row = 16 * wave + r;
    // the next head's, loaded a head ahead (the first's too, unless fp32's planes need the registers); behind the end the
    // last token's, unused
    const size_t gate = (size_t)(t0 + (lane < n ? lane : n - 1)) * a.v_heads + head0;
    float g_next = 0, beta_next = 0;
    if constexpr (NP < 3) g_next = a.g[gate], beta_next = a.beta[gate];
    qe_f4 gk[4], gq[4]; // K K^T and Q K^T, blocks 0 .. wave of the wave's rows
    {
        qe_s8 kr[KS][NP], qr[KS][NP];
        float kk = 0, qq = 0;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            load8_planes(k + (size_t)(t0 + row) * a.k_stride + 32 * s, row < n, kr[s], kk);
            load8_planes(q + (size_t)(t0 + row) * a.q_stride + 32 * s, row < n, qr[s], qq);
            for (int i = 0; i < NP; ++i) {
                const int at = (i * 64 + row) * DK + (((4 * s + c) ^ key_swz<DK>(row)) << 3);
                *(qe_s8 *)(k_s + at) = kr[s][i];
                if constexpr (NP > 1) { // (every workgroup of the key head writes the same)
                    short *ws = a.ws_kq + ((size_t)chunk * a.k_heads + kh) * 2 * NP * 64 * DK;
                    *(qe_s8 *)(ws + at) = kr[s][i];
                    *(qe_s8 *)(ws + NP * 64 * DK + ((wave * KS + s) * NP + i) * 512 + lane * 8) = qr[s][i];
                }
            }
        }
        kk += __shfl_xor(kk, 16), qq += __shfl_xor(qq, 16);
        kk += __shfl_xor(kk, 32), qq += __shfl_xor(qq, 32);
        if (lane < 16) {
            kk_s[row] = kk;
            // rows behind the end stand for the last token's in k_delta_scan: factors of 0 keep them from overflowing
            rk_s[row] = row >= n ? 0.f : norm_factor(kk, a.l2norm);
            rq_s[row] = row >= n ? 0.f : (a.l2norm ? norm_factor(qq, true) : 1.f) * a.scale;
        }
        __syncthreads();
#pragma unroll
        for (int cb = 0; cb < 4; ++cb) {
            if (cb > wave) continue;
            const int col = 16 * cb + r;
            qe_f4 k3[3] = {}, q3[3] = {};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                qe_s8 kb[NP];
                for (int i = 0; i < NP; ++i) kb[i] = *(const qe_s8 *)(k_s + (i * 64 + col) * DK + (((4 * s + c) ^ key_swz<DK>(col)) << 3));
                mul_planes<NP, NP, 2>(kr[s], kb, k3);
                mul_planes<NP, NP, 2>(qr[s], kb, q3);
            }
            gk[cb] = k3[0] + (k3[1] + k3[2]);
            gq[cb] = q3[0] + (q3[1] + q3[2]);
        }
    }
    if constexpr (NP == 3) g_next = a.g[gate], beta_next = a.beta[gate];
    for (int gi = 0; gi < a.heads; ++gi) {
        const int head = head0 + gi;
        float *ws = a.ws + ((size_t)chunk * a.v_heads + head) * QE_DELTA_WS, *factors = ws + QE_DELTA_WS - 256;
        double b = lane < n ? (double)log_decay(g_next) * 1.4426950408889634 : 0.0;
        float beta = lane < n ? beta_next : 0.f;
        if (gi + 1 < a.heads) g_next = a.g[gate + gi + 1], beta_next = a.beta[gate + gi + 1];
        for (int d = 1; d < 64; d <<= 1) {
            const double up = __shfl_up(b, d);
            if (lane >= d) b += up;
        }
        __syncthreads(); // rk_s and rq_s are written, K is read; the last head's b_s, beta_s, T and M are read
        // A product of 0 and an infinity or NaN is NaN, and in a block above the diagonal's zeros it would
        // reach tokens before its own.  So from the first token whose key, gate or decay is not finite on
        // (what comes after it is not finite either) the matrices are zeros and the factors NaN.
        const bool finite = __builtin_isfinite(b) && __builtin_isfinite(beta) && __builtin_isfinite(kk_s[lane]);
        const unsigned long long odd = __ballot(!finite);
        const int fine = odd ? __ffsll(odd) - 1 : 64; // tokens before it
        if (lane >= fine) beta = 0.f;
        if (wave == 0) {
            b_s[lane] = b;
            beta_s[lane] = beta;
        }
        if (wave == 1) {
            const double last = __shfl(b, 63);
            const float e = __builtin_amdgcn_exp2f((float)b), none = lane < fine ? 0.f : NAN;
            factors[lane] = e * rk_s[lane] + none;
            factors[64 + lane] = e * rq_s[lane] + none;
            factors[128 + lane] = __builtin_amdgcn_exp2f((float)(last - b)) * rk_s[lane] + (fine < 64 ? NAN : 0.f);
            if (lane == 0) factors[192] = __builtin_amdgcn_exp2f((float)last) + (fine < 64 ? NAN : 0.f);
        }
        __syncthreads();
        double b_i[4], b_j[4]; // all read at once, and values that are not wanted dropped after: no branches around LDS reads
        float q_i[4], k_i[4], k_j[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int ri = 16 * wave + 4 * c + i, cj = 16 * i + r;
            b_i[i] = b_s[ri], b_j[i] = b_s[cj];
            q_i[i] = rq_s[ri], k_i[i] = rk_s[ri] * beta_s[ri], k_j[i] = rk_s[cj];
        }
#pragma unroll
        for (int cb = 0; cb < 4; ++cb) {
            if (cb > (wave | 1)) continue; // and zeros to the right of the diagonal in its 32 columns
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int ri = 16 * wave + 4 * c + i, cj = 16 * cb + r;
                const bool in = cb <= wave && cj <= ri && ri < fine;
                const float fade = __builtin_amdgcn_exp2f((float)(b_i[i] - b_j[cb])) * k_j[cb];
                const float m = gq[cb][i] * fade * q_i[i], x = gk[cb][i] * fade * k_i[i];
                M[ri * LD + cj] = in ? m : 0.f;
                A[ri * LD + cj] = in && cj < ri ? x : 0.f;
                if (cb > wave) T[ri * LD + cj] = 0.f;
            }
        }
        __syncthreads();
        {
            float x[16];
            const float *d = A + 16 * wave * LD + 16 * wave;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                x[i] = i == r ? 1.f : 0.f;
#pragma unroll
                for (int j = 0; j < i; ++j) x[i] = fmaf(-d[i * LD + j], x[j], x[i]);
            }
            if (lane < 16)
#pragma unroll
                for (int i = 0; i < 16; ++i) T[(16 * wave + i) * LD + 16 * wave + r] = x[i];
        }
        for (int d = 1; d < 4; ++d) {
            __syncthreads();
            if (wave >= d) {
                const int jb = wave - d;
                qe_f4 in = {0, 0, 0, 0}, to = {0, 0, 0, 0};
                for (int kb = jb; kb < wave; ++kb) {
                    qe_f4 t;
                    for (int j = 0; j < 4; ++j) t[j] = T[(16 * kb + 4 * c + j) * LD + 16 * jb + r];
                    in = mma4(*(const qe_f4 *)(A + (16 * wave + r) * LD + 16 * kb + 4 * c), t, in);
                }
                to = mma4(*(const qe_f4 *)(T + (16 * wave + r) * LD + 16 * wave + 4 * c), in, to);
                for (int i = 0; i < 4; ++i) T[(16 * wave + 4 * c + i) * LD + 16 * jb + r] = -to[i];
            }
        }
        __syncthreads();
        // 8 columns of a row at a time to the planes: wave w has rows 16 w .. + 15, in steps of 8
        for (int i = 0; i < 2; ++i) {
            const int ri = 16 * wave + 8 * i + (lane >> 3), cj = (lane & 7) * 8;
            if (cj / 32 > wave / 2) continue;
            float t[8], m[8];
            for (int j = 0; j < 8; ++j) {
                t[j] = T[ri * LD + cj + j] * beta_s[cj + j];
                m[j] = M[ri * LD + cj + j];
            }
            // the lane (cj % 32) / 8 * 16 + ri % 16 of the wave's operand for columns 32 (cj / 32) .. + 31
            short *to = (short *)ws + (wave * 2 + cj / 32) * 3 * 512 + ((cj % 32) / 8 * 16 + ri % 16) * 8;
            for (int p = 0; p < 3; ++p) {
                qe_s8 h;
                for (int j = 0; j < 8; ++j) h[j] = next_plane(t[j]);
                *(qe_s8 *)(to + p * 512) = h;
            }
            for (int p = 0; p < NO; ++p) {
                qe_s8 h;
                for (int j = 0; j < 8; ++j) h[j] = next_plane(m[j]);
                *(qe_s8 *)(to + 4 * 6 * 512 + p * 512) = h;
            }
        }
    }
}

// ---------------------------------------------------------------------------
// The walk over a sequence's chunks, 16 columns of a value head's state: a workgroup of eight
// waves.  The state's next value hangs on three products one after the other (K S, T times
// what is left of V, K^T U), so waves 0 .. 3 do little else, 16 rows of the chunk and DK / 4
// of the state each, and waves 4 .. 7 make the outputs of 16 rows each beside them.
// What waves exchange (S, V - .. K S, U) goes through LDS as planes, transposed [column][row]: a
// result's registers are 4 consecutive rows of its column, an operand's 8.  K lies in LDS in
// two buffers, the next chunk's loaded directly while this one's is used: its rows are
// the first product's operand, and transposing reads give the third's.
// What bounds it: the chain of products, exchanges and barriers of a chunk, one chain wave on
// each SIMD (a sequence of 32 heads in 8 slices is a workgroup for each of the 256 CUs).  A load stalls the wave that issues it
// while the CU's 64 bytes a cycle are taken (some 65 KiB a chunk), so the loads are few and
// wide, and spread over the waves and over the chunk.  8192 bf16 tokens of 32 heads of 128 x 128: 240 us on
// average of 30 in a row, 223 at least (fp16 303, fp32 418), 1.8 a chunk: of some 3,800 cycles K S takes 550, what is left
// of V to LDS 400, T times it 280, U to LDS 500, the state's update and S to LDS 1,150, the rest is barriers.  1999 fp32
// tokens of three prompts: 90 us.
// ---------------------------------------------------------------------------
// Where the LDS holds two workgroups (bf16, and fp16 keys of 64), 128 registers let it, and the bound keeps it so: sequences
// side by side overlap (16 of 500 tokens, bf16: 354 us the call with one a CU, 300 with two; one of 8192 has one a CU anyhow).
template <typename IN, int DK, int DV>
__global__ __launch_bounds__(512, sizeof(IN) == 2 && (DK == 64 || __is_same(IN, __bf16)) ? 4 : 2) void k_delta_scan(const QeDeltaArgs a) {
    constexpr int KS = DK / 32, SB = DK / 64, LS = DK + 8, LT = 72, NP = planes_of<IN>(), NO = sizeof(IN) == 4 ? 3 : 2;
    constexpr int SL = DV / 16, VL = 16 / sizeof(IN); // elements of V in 16 bytes
    // what is loaded ahead has two buffers, variables of their own: else the compiler has every LDS read wait for
    // the direct loads in flight
    __shared__ __align__(16) short k_even[NP * 64 * DK], k_odd[NP * 64 * DK];
    constexpr int VW = 64 * VL; // elements of V that a wave loads: its 16 rows, in 16 bits twice
    __shared__ __align__(16) IN v_even[4 * VW], v_odd[4 * VW];
    __shared__ __align__(16) float f_even[4 * 256], f_odd[4 * 256]; // the factors, a copy for each wave
    __shared__ __align__(16) short s_p[3 * 16 * LS], r_p[3 * 16 * LT], u_p[NO * 16 * LT], w_p[3 * 16 * LT];
    __shared__ int odd_s[2][16]; // of each column: the chunk's first token with a value that is not finite, or 64
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane((tid >> 6) & 3), lane = tid & 63, r = lane & 15, c = lane >> 4;
    const bool chain = tid < 256;
    const int seq = blockIdx.x / (SL * a.v_heads), at = blockIdx.x - seq * SL * a.v_heads;
    // Workgroups go to the eight XCDs in turn: a head's slices, which read the same K, Q, T and M, to one L2.
    const bool eights = a.v_heads % 8 == 0;
    const int slice = eights ? at / 8 % SL : at % SL, head = eights ? at / (8 * SL) * 8 + at % 8 : at / SL;
    const int kh = head / a.group, col = slice * 16 + r;
    unsigned bad = 0;
    int begin, end;
    qe_rows_of(a.cu[seq], a.cu[seq + 1], a.n_tokens, &begin, &end, &bad);
    if (bad && tid == 0) report(a.err, QE_BAD_LENGTH);
    const int in_i = a.slots_in[seq], out_i = a.slots_out[seq], what = slots_of(a, seq, in_i, out_i);
    report_slots(a, what);
    if (bad || what) {
        for (int t = begin + (tid >> 4); t < end; t += 32) ((IN *)a.out)[(size_t)t * a.out_stride + (size_t)head * DV + slice * 16 + (tid & 15)] = (IN)0.f;
        return;
    }
    const int chunk0 = qe_delta_first_chunk(begin, seq), row = 16 * wave + r, kb = wave / 2; // kb: the last 32 columns that the wave's rows reach
    const short *ws = (const short *)(a.ws + ((size_t)chunk0 * a.v_heads + head) * QE_DELTA_WS);
    const size_t ws_step = (size_t)a.v_heads * QE_DELTA_WS * 2;
    const short *kq = NP == 1 ? nullptr : a.ws_kq + ((size_t)chunk0 * a.k_heads + kh) * 2 * NP * 64 * DK;
    const size_t kq_step = (size_t)a.k_heads * 2 * NP * 64 * DK;
    if (tid < 32) odd_s[tid >> 4][tid & 15] = 64;
    // Loads run one chunk ahead, without branches: what a wave may leave in flight is counted, and where a branch
    // makes the count uncertain the compiler waits for loads just issued.  So behind the last chunk they take it
    // again, and waves whose rows of T and M are short load their unwritten half as well.  Rows behind the
    // sequence's end are its last one's: T's columns and rows are zeros there.
    if (chain) {
        // As in k_delta_chunks, what is not finite must not meet the zeros above the diagonal: it becomes
        // 0, and its column's outputs from that token on, and its state, NaN.
        auto cleared = [&](qe_f4 x, int p) {
            bool odd = false;
            for (int j = 0; j < 4; ++j) odd |= !__builtin_isfinite(x[j]);
            if (__any(odd)) {
                for (int j = 0; j < 4; ++j)
                    if (!__builtin_isfinite(x[j])) {
                        x[j] = 0.f;
                        atomicMin(&odd_s[p][r], 16 * wave + 4 * c + j);
                    }
            }
            return x;
        };
        qe_f4 S[SB];
        for (int i = 0; i < SB; ++i)
            for (int j = 0; j < 4; ++j)
                S[i][j] = in_i < 0 ? 0.f : a.pool[(((size_t)in_i * a.v_heads + head) * DK + 16 * (wave * SB + i) + 4 * c + j) * DV + col];
        qe_s8 tf[2][3];
        auto load = [&](const short *w) {
            for (int p = 0; p < 3; ++p) {
                tf[0][p] = *(const qe_s8 *)(w + wave * 6 * 512 + p * 512 + lane * 8);
                tf[1][p] = *(const qe_s8 *)(w + wave * 6 * 512 + 3 * 512 + p * 512 + lane * 8);
            }
        };
        auto step = [&](const int par, const short *k_s, const IN *v_s, const float *f_s, int t0) {
            lds_barrier();
            qe_f4 x[3] = {};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                qe_s8 kf[NP], sf[3];
                for (int p = 0; p < NP; ++p) kf[p] = *(const qe_s8 *)(k_s + (p * 64 + row) * DK + (((4 * s + c) ^ key_swz<DK>(row)) << 3));
                for (int p = 0; p < 3; ++p) sf[p] = *(const qe_s8 *)(s_p + (p * 16 + r) * LS + 32 * s + 8 * c);
                mul_planes<NP, 3, 2>(kf, sf, x);
            }
            qe_s8 kt[SB][2][NP]; // K^T for the last product
#pragma unroll
            for (int i = 0; i < SB; ++i)
                for (int s = 0; s < 2; ++s)
                    for (int p = 0; p < NP; ++p) {
                        const int ra = 32 * s + 4 * c + (r >> 2), el = 16 * (wave * SB + i) + (r & 3) * 4;
                        const short *at = k_s + (p * 64 + ra) * DK + (((el >> 3) ^ key_swz<DK>(ra)) << 3) + (el & 7);
                        const qe_s4 lo = lds_tr(at), hi = lds_tr(at + 16 * DK); // 16 rows on the permutation is the same
                        kt[i][s][p] = qe_s8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                    }
            qe_f4 v;
            if constexpr (sizeof(IN) == 2) {
                const qe_s4 h = lds_tr((const short *)v_s + wave * VW + (4 * c + (r >> 2)) * 16 + (r & 3) * 4);
                for (int j = 0; j < 4; ++j) v[j] = from16<__is_same(IN, __bf16)>(h[j]);
            } else {
                for (int j = 0; j < 4; ++j) v[j] = v_s[wave * VW + (4 * c + j) * 16 + r];
            }
            const float *f = f_s + 256 * wave;
            const qe_f4 cx = *(const qe_f4 *)(f + 16 * wave + 4 * c), cu = *(const qe_f4 *)(f + 128 + 16 * wave + 4 * c);
            const float last = f[192];
            put4<3>(r_p + r * LT + 16 * wave + 4 * c, 16 * LT, cleared(v - cx * (x[0] + (x[1] + x[2])), par));
            lds_barrier();
            qe_f4 u3[3] = {};
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (s > kb) continue;
                qe_s8 rf[3];
                for (int p = 0; p < 3; ++p) rf[p] = *(const qe_s8 *)(r_p + (p * 16 + r) * LT + 32 * s + 8 * c);
                mul_planes<3, 3, 2>(tf[s], rf, u3);
            }
            const qe_f4 u = cleared(u3[0] + (u3[1] + u3[2]), par);
            put4<3>(w_p + r * LT + 16 * wave + 4 * c, 16 * LT, u * cu);
            put4<NO>(u_p + r * LT + 16 * wave + 4 * c, 16 * LT, u);
            ws += (t0 + QE_DELTA_C < end) * ws_step;
            load(ws);
            lds_barrier();
            const int spoilt = odd_s[par][r];
            if (tid < 16) odd_s[par ^ 1][tid] = 64; // last read a chunk ago, next written in the next
            qe_s8 wf[2][3];
#pragma unroll
            for (int s = 0; s < 2; ++s)
                for (int p = 0; p < 3; ++p) {
                    const short *at = w_p + (p * 16 + r) * LT + 32 * s + 4 * c;
                    const qe_s4 lo = *(const qe_s4 *)at, hi = *(const qe_s4 *)(at + 16);
                    wf[s][p] = qe_s8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                }
#pragma unroll
            for (int i = 0; i < SB; ++i) {
                qe_f4 d[3] = {};
#pragma unroll
                for (int s = 0; s < 2; ++s) mul_planes<NP, 3, 2>(kt[i][s], wf[s], d);
                S[i] = S[i] * (spoilt < 64 ? NAN : last) + (d[0] + (d[1] + d[2]));
                put4<3>(s_p + r * LS + 16 * (wave * SB + i) + 4 * c, 16 * LS, S[i]);
            }
        };
        for (int i = 0; i < SB; ++i) put4<3>(s_p + r * LS + 16 * (wave * SB + i) + 4 * c, 16 * LS, S[i]);
        if (begin < end) load(ws);
        for (int t0 = begin; t0 < end; t0 += 2 * QE_DELTA_C) {
            step(0, k_even, v_even, f_even, t0);
            if (t0 + QE_DELTA_C < end) step(1, k_odd, v_odd, f_odd, t0 + QE_DELTA_C);
        }
        if (out_i >= 0)
            for (int i = 0; i < SB; ++i)
                for (int j = 0; j < 4; ++j) a.pool[(((size_t)out_i * a.v_heads + head) * DK + 16 * (wave * SB + i) + 4 * c + j) * DV + col] = S[i][j];
    } else {
        qe_s8 q_even[KS][NP], q_odd[KS][NP], mf[2][NO];
        auto load_k = [&](int t0, const short *from, short *to) {
            constexpr int ROWS = 512 / DK; // of one direct load
#pragma unroll
            for (int i = 0; i < NP * 16 / ROWS; ++i) {
                const int p = i / (16 / ROWS), rr = wave * 16 + i % (16 / ROWS) * ROWS, mine = rr + lane / (DK / 8), ch = (lane % (DK / 8)) ^ key_swz<DK>(mine);
                const short *src = NP == 1 ? (const short *)a.k + (size_t)(t0 + mine < end ? t0 + mine : end - 1) * a.k_stride + (size_t)kh * DK + ch * 8
                                           : from + (p * 64 + rr) * DK + lane * 8;
                load_lds16(src, to + (p * 64 + rr) * DK);
            }
        };
        auto load_v = [&](int t0, const short *w, IN *v_to, float *f_to) {
            constexpr int PER = 16 / VL; // lanes of a row
            const int t = t0 + 16 * wave + lane / PER % 16;
            load_lds16((const IN *)a.v + (size_t)(t < end ? t : end - 1) * a.v_stride + (size_t)head * DV + slice * 16 + lane % PER * VL, v_to + wave * VW);
            load_lds16((const float *)w + QE_DELTA_WS - 256 + lane * 4, f_to + wave * 256);
        };
        auto load_q = [&](int t0, const short *from, qe_s8 (*qf)[NP]) {
            const short *q = (const short *)a.q + (size_t)(t0 + row < end ? t0 + row : end - 1) * a.q_stride + (size_t)kh * DK + 8 * c;
            for (int s = 0; s < KS; ++s)
                for (int p = 0; p < NP; ++p)
                    qf[s][p] = *(const qe_s8 *)(NP == 1 ? q + 32 * s : from + NP * 64 * DK + ((wave * KS + s) * NP + p) * 512 + lane * 8);
        };
        auto load_m = [&](const short *w) {
            for (int p = 0; p < NO; ++p) {
                mf[0][p] = *(const qe_s8 *)(w + 4 * 6 * 512 + wave * 6 * 512 + p * 512 + lane * 8);
                mf[1][p] = *(const qe_s8 *)(w + 4 * 6 * 512 + wave * 6 * 512 + 3 * 512 + p * 512 + lane * 8);
            }
        };
        IN *out = (IN *)a.out + (size_t)(begin + 16 * wave + 4 * c) * a.out_stride + (size_t)head * DV + col; // the first of the lane's four rows
        auto step = [&](const int par, const bool whole, const float *f_s, short *k_next, IN *v_next, float *f_next, const qe_s8 (*qf)[NP], qe_s8 (*q_next)[NP], int t0) {
            const int ahead = t0 + QE_DELTA_C < end;
            kq += ahead * kq_step, ws += ahead * ws_step;
            // K, V and the factors have landed, and Q: younger than the direct loads are those of Q, then of M, then the last
            // chunk's four stores.  (A register that is still to be loaded when it is used makes the compiler wait for
            // the direct loads in flight as well: so Q is here before the next ones begin, and M's come long before its use.)
            constexpr int younger = 2 * NO + (KS * NP < 4 ? KS * NP : 4);
            __builtin_amdgcn_s_waitcnt(0x0f70 | (younger & 15) | (younger >> 4) << 14);
            lds_barrier();
            // The chain's waves now read all of S, which takes the LDS's bandwidth; these issue loads meanwhile,
            // and read S while the chain is at its next product.
            load_v(t0 + ahead * QE_DELTA_C, ws, v_next, f_next);
            load_k(t0 + ahead * QE_DELTA_C, kq, k_next);
            asm volatile("" ::: "memory"); // the count above needs Q's loads behind the direct ones
            load_q(t0 + ahead * QE_DELTA_C, kq, q_next);
            lds_barrier();
            qe_f4 x[3] = {};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                qe_s8 sf[NO];
                for (int p = 0; p < NO; ++p) sf[p] = *(const qe_s8 *)(s_p + (p * 16 + r) * LS + 32 * s + 8 * c);
                mul_planes<NP, NO, NO - 1>(qf[s], sf, x);
                if (s & 1) __builtin_amdgcn_sched_barrier(0); // all of S read at once would take more than 128 registers
            }
            qe_f4 o = *(const qe_f4 *)(f_s + 256 * wave + 64 + 16 * wave + 4 * c) * (x[0] + (x[1] + x[2]));
            lds_barrier();
            const int spoilt = odd_s[par][r];
            qe_f4 y[3] = {};
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (s > kb) continue;
                qe_s8 uf[NO];
                for (int p = 0; p < NO; ++p) uf[p] = *(const qe_s8 *)(u_p + (p * 16 + r) * LT + 32 * s + 8 * c);
                mul_planes<NO, NO, NO - 1>(mf[s], uf, y);
            }
            load_m(ws);
            o += y[0] + (y[1] + y[2]);
            for (int j = 0; j < 4; ++j) {
                const int t = 16 * wave + 4 * c + j;
                if (whole || t0 + t < end) out[j * a.out_stride] = (IN)(t < spoilt ? o[j] : NAN);
            }
            out += QE_DELTA_C * a.out_stride;
        };
        if (begin < end) {
            load_v(begin, ws, v_even, f_even);
            load_k(begin, kq, k_even);
            load_q(begin, kq, q_even);
            load_m(ws);
            __builtin_amdgcn_s_waitcnt(0x0f70); // in whatever order they were issued here
        }
        int t0 = begin;
        for (; t0 + 2 * QE_DELTA_C <= end; t0 += 2 * QE_DELTA_C) {
            step(0, true, f_even, k_odd, v_odd, f_odd, q_even, q_odd, t0);
            step(1, true, f_odd, k_even, v_even, f_even, q_odd, q_even, t0 + QE_DELTA_C);
        }
        if (t0 < end) step(0, false, f_even, k_odd, v_odd, f_odd, q_even, q_odd, t0);
        if (t0 + QE_DELTA_C < end) step(1, false, f_odd, k_even, v_even, f_even, q_odd, q_even, t0 + QE_DELTA_C);
    }
}

template <typename IN, int DK, int DV>
static hipError_t prompt(QeDeltaArgs a, hipStream_t st) {
    const unsigned chunks = (unsigned)qe_delta_max_chunks(a.n_tokens, a.n_seqs);
    if (a.n_seqs <= 256) a.skip = nullptr;
    else k_delta_slots<<<dim3((unsigned)a.n_seqs), dim3(256), 0, st>>>(a);
    a.heads = qe_delta_heads(chunks, a.v_heads, a.group);
    k_delta_chunks<IN, DK><<<dim3(chunks * (a.v_heads / a.heads)), dim3(256), 0, st>>>(a);
    k_delta_scan<IN, DK, DV><<<dim3((unsigned)a.n_seqs * a.v_heads * (DV / 16)), dim3(512), 0, st>>>(a);
    return hipGetLastError();
}
template <typename IN, int DK, int DV>
static hipError_t decode(QeDeltaArgs a, hipStream_t st) {
    if (a.n_seqs <= 256) a.skip = nullptr;
    else k_delta_slots<<<dim3((unsigned)a.n_seqs), dim3(256), 0, st>>>(a);
    k_delta_decode<IN, DK, DV><<<dim3((unsigned)a.n_seqs * a.v_heads * (DV / 32)), dim3(256), 0, st>>>(a);
    return hipGetLastError();
}
template <typename IN, int DK, int DV>
static hipError_t either(const QeDeltaArgs &a, bool one, hipStream_t st) {
    return one ? decode<IN, DK, DV>(a, st) : prompt<IN, DK, DV>(a, st);
}
template <typename IN>
static hipError_t by_dims(const QeDeltaArgs &a, int dk, int dv, bool one, hipStream_t st) {
    if (dk == 64) return dv == 64 ? either<IN, 64, 64>(a, one, st) : either<IN, 64, 128>(a, one, st);
    return dv == 64 ? either<IN, 128, 64>(a, one, st) : either<IN, 128, 128>(a, one, st);
}
static hipError_t by_type(const QeDeltaArgs &a, int dk, int dv, int type, bool one, hipStream_t st) {
    return type == QE_F32 ? by_dims<float>(a, dk, dv, one, st) : type == QE_F16 ? by_dims<_Float16>(a, dk, dv, one, st) : by_dims<__bf16>(a, dk, dv, one, st);
}
hipError_t qe_launch_delta_prompt(const QeDeltaArgs &a, int dk, int dv, int type, hipStream_t st) { return by_type(a, dk, dv, type, false, st); }
hipError_t qe_launch_delta_decode(const QeDeltaArgs &a, int dk, int dv, int type, hipStream_t st) { return by_type(a, dk, dv, type, true, st); }
