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
// State, sums and products are in 32 bits, b in 64 (a difference of two long sums).
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

__device__ __forceinline__ float log_decay(float g) { return g < -1e4f ? -1e4f : g; } // e^-1e4 is 0; a NaN stays

// ---------------------------------------------------------------------------
// Which sequences of a call are computed (rules in qe_mixer_plan.h).
// ---------------------------------------------------------------------------
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
// in registers and written once.
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
    int what = qe_slot_pair(a.n_slots, in_i, out_i);
    if (a.n_seqs > 1) {
        int shared = 0;
        if (a.skip) what = a.skip[seq];
        else {
            if (tid < a.n_seqs) shared = qe_slot_conflict(seq, out_i, tid, a.slots_in[tid], a.slots_out[tid]);
            if (__syncthreads_or(shared) && !what) what = QE_SLOT_SHARED;
        }
    }
    if (what) {
        if (tid < 32) out[slice * 32 + tid] = (IN)0.f;
        if (tid == 0 && !a.skip) report(a.err, what == QE_SLOT_OUTSIDE ? QE_BAD_SLOT : QE_BAD_SHARED_SLOT);
        return;
    }
    qe_f4 s[ROWS];
    const float *from = a.pool + ((size_t)(in_i < 0 ? 0 : in_i) * a.v_heads + head) * DK * DV;
    for (int i = 0; i < ROWS; ++i) s[i] = in_i < 0 ? qe_f4{0, 0, 0, 0} : *(const qe_f4 *)(from + (size_t)(row + 32 * i) * DV + col);

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
    const float rq = (a.l2norm ? 1.f / sqrtf(xx + 1e-6f) : 1.f) * a.scale, rk = a.l2norm ? 1.f / sqrtf(yy + 1e-6f) : 1.f;
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
        for (int i = 0; i < ROWS; ++i) *(qe_f4 *)(to + (size_t)(row + 32 * i) * DV + col) = s[i] + (rk * qk[1][row + 32 * i]) * u;
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
// 16: the diagonal ones by substitution, a lane per column; then by distance from the
// diagonal T_ij = -T_ii sum_k A_ik T_kj.
// Workspace of a chunk and value head: T [64][64], M [64][64] (blocks above the diagonal are not
// written), then per token e^b / |k|, scale e^b / |q|, e^(b_last - b) / |k|, and e^(b_last).
// ---------------------------------------------------------------------------
template <typename IN, int DK>
__global__ __launch_bounds__(256) void k_delta_chunks(const QeDeltaArgs a) {
    constexpr int LD = 68, KS = DK / 16;
    __shared__ __align__(16) float A[64 * LD], T[64 * LD];
    __shared__ double b_s[64];
    __shared__ float kk_s[64], rk_s[64], rq_s[64], beta_s[64];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 15, c = lane >> 4;
    const int chunk = blockIdx.x / a.k_heads, kh = blockIdx.x % a.k_heads;
    int seq = 0;
    for (int hi = a.n_seqs; hi - seq > 1;) {
        const int mid = (seq + hi) >> 1;
        if (qe_delta_first_chunk(a.cu[mid], mid) <= chunk) seq = mid;
        else hi = mid;
    }
    unsigned bad = 0;
    const int begin = qe_checked(a.cu[seq], 0, a.n_tokens, 0, &bad), end = qe_checked(a.cu[seq + 1], begin, a.n_tokens, begin, &bad);
    const int64_t local = chunk - qe_delta_first_chunk(a.cu[seq], seq);
    if (bad || a.skip[seq] || local < 0 || local * QE_DELTA_C >= end - begin) return; // uniform
    const int t0 = begin + (int)local * QE_DELTA_C, n = end - t0 < QE_DELTA_C ? end - t0 : QE_DELTA_C;

    const IN *q = (const IN *)a.q + (size_t)kh * DK + 4 * c, *k = (const IN *)a.k + (size_t)kh * DK + 4 * c;
    const int row = 16 * wave + r;
    qe_f4 kr[KS], qr[KS];
    float kk = 0, qq = 0;
    for (int s = 0; s < KS; ++s) {
        kr[s] = row < n ? load4(k + (size_t)(t0 + row) * a.k_stride + 16 * s) : qe_f4{0, 0, 0, 0};
        qr[s] = row < n ? load4(q + (size_t)(t0 + row) * a.q_stride + 16 * s) : qe_f4{0, 0, 0, 0};
        for (int j = 0; j < 4; ++j) kk += kr[s][j] * kr[s][j], qq += qr[s][j] * qr[s][j];
    }
    kk += __shfl_xor(kk, 16), qq += __shfl_xor(qq, 16);
    kk += __shfl_xor(kk, 32), qq += __shfl_xor(qq, 32);
    if (lane < 16) {
        kk_s[row] = kk;
        rk_s[row] = a.l2norm ? 1.f / sqrtf(kk + 1e-6f) : 1.f;
        rq_s[row] = (a.l2norm ? 1.f / sqrtf(qq + 1e-6f) : 1.f) * a.scale;
    }
    qe_f4 gk[4], gq[4]; // K K^T and Q K^T, blocks 0 .. wave of the wave's rows
#pragma unroll
    for (int cb = 0; cb < 4; ++cb) {
        gk[cb] = gq[cb] = qe_f4{0, 0, 0, 0};
        if (cb > wave) continue;
        const int col = 16 * cb + r;
        for (int s = 0; s < KS; ++s) {
            const qe_f4 kb = col < n ? load4(k + (size_t)(t0 + col) * a.k_stride + 16 * s) : qe_f4{0, 0, 0, 0};
            gk[cb] = mma4(kr[s], kb, gk[cb]);
            gq[cb] = mma4(qr[s], kb, gq[cb]);
        }
    }
    for (int gi = 0; gi < a.group; ++gi) {
        const int head = kh * a.group + gi;
        float *ws = a.ws + ((size_t)chunk * a.v_heads + head) * QE_DELTA_WS;
        double b = lane < n ? (double)log_decay(a.g[(size_t)(t0 + lane) * a.v_heads + head]) : 0.0;
        for (int d = 1; d < 64; d <<= 1) {
            const double up = __shfl_up(b, d);
            if (lane >= d) b += up;
        }
        float beta = lane < n ? a.beta[(size_t)(t0 + lane) * a.v_heads + head] : 0.f;
        __syncthreads(); // rk_s and rq_s are written, the last head's b_s, beta_s, A and T are read
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
            const float e = expf((float)b), none = lane < fine ? 0.f : NAN;
            ws[2 * 4096 + lane] = e * rk_s[lane] + none;
            ws[2 * 4096 + 64 + lane] = e * rq_s[lane] + none;
            ws[2 * 4096 + 128 + lane] = expf((float)(last - b)) * rk_s[lane] + (fine < 64 ? NAN : 0.f);
            if (lane == 0) ws[2 * 4096 + 192] = expf((float)last) + (fine < 64 ? NAN : 0.f);
        }
        __syncthreads();
#pragma unroll
        for (int cb = 0; cb < 4; ++cb) {
            if (cb > wave) continue;
            for (int i = 0; i < 4; ++i) {
                const int ri = 16 * wave + 4 * c + i, cj = 16 * cb + r;
                const bool in = cj <= ri && ri < fine;
                const float fade = in ? expf((float)(b_s[ri] - b_s[cj])) * rk_s[cj] : 0.f;
                ws[4096 + ri * 64 + cj] = in ? gq[cb][i] * fade * rq_s[ri] : 0.f;
                A[ri * LD + cj] = in && cj < ri ? gk[cb][i] * fade * (rk_s[ri] * beta_s[ri]) : 0.f;
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
        for (int i = 0; i < 4; ++i) {
            const int ri = 16 * wave + 4 * i + c, cj = 4 * r;
            if (cj / 16 > wave) continue;
            qe_f4 t = *(const qe_f4 *)(T + ri * LD + cj);
            for (int j = 0; j < 4; ++j) t[j] *= beta_s[cj + j];
            *(qe_f4 *)(ws + ri * 64 + cj) = t;
        }
    }
}

// ---------------------------------------------------------------------------
// The walk over a sequence's chunks, 16 columns of a value head's state.  Wave w computes
// rows 16 w .. + 15 of K S, Q S, U and O, and keeps rows DK / 4 w .. of the state.  What the
// waves exchange (S, V - .. K S, U) goes through LDS transposed, [column][row], so that the
// registers of a result are written, and an operand's read, 4 floats at a time.
// ---------------------------------------------------------------------------
template <typename IN, int DK, int DV>
__global__ __launch_bounds__(256) void k_delta_scan(const QeDeltaArgs a) {
    constexpr int KS = DK / 16, SB = DK / 64, LK = DK + 4, LT = 68;
    __shared__ __align__(16) float k_s[2][64 * LK], s_t[16 * LK], r_t[16 * LT], u_t[16 * LT];
    __shared__ int odd_s[2][16]; // of each column: the chunk's first token with a value that is not finite, or 64
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 15, c = lane >> 4;
    const int slice = blockIdx.x % (DV / 16), head = blockIdx.x / (DV / 16) % a.v_heads, seq = blockIdx.x / (DV / 16) / a.v_heads;
    const int kh = head / a.group, col = slice * 16 + r;
    unsigned bad = 0;
    const int begin = qe_checked(a.cu[seq], 0, a.n_tokens, 0, &bad), end = qe_checked(a.cu[seq + 1], begin, a.n_tokens, begin, &bad);
    if (bad && tid == 0) report(a.err, QE_BAD_LENGTH);
    if (bad | a.skip[seq]) {
        for (int t = begin + (tid >> 4); t < end; t += 16) ((IN *)a.out)[(size_t)t * a.out_stride + (size_t)head * DV + slice * 16 + (tid & 15)] = (IN)0.f;
        return;
    }
    const int in_i = a.slots_in[seq], out_i = a.slots_out[seq];
    qe_f4 S[SB];
    for (int i = 0; i < SB; ++i)
        for (int j = 0; j < 4; ++j)
            S[i][j] = in_i < 0 ? 0.f : a.pool[(((size_t)in_i * a.v_heads + head) * DK + 16 * (wave * SB + i) + 4 * c + j) * DV + col];

    const IN *q = (const IN *)a.q + (size_t)kh * DK + 4 * c, *k = (const IN *)a.k + (size_t)kh * DK + 4 * c;
    const float *ws = a.ws + ((size_t)qe_delta_first_chunk(a.cu[seq], seq) * a.v_heads + head) * QE_DELTA_WS;
    int par = 0;
    if (tid < 32) odd_s[tid >> 4][tid & 15] = 64;
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
    for (int t0 = begin; t0 < end; t0 += QE_DELTA_C, ws += (size_t)a.v_heads * QE_DELTA_WS, par ^= 1) {
        const int n = end - t0 < QE_DELTA_C ? end - t0 : QE_DELTA_C, row = 16 * wave + r;
        qe_f4 kr[KS], qr[KS], tr[4], mr[4], v;
        for (int s = 0; s < KS; ++s) {
            kr[s] = row < n ? load4(k + (size_t)(t0 + row) * a.k_stride + 16 * s) : qe_f4{0, 0, 0, 0};
            qr[s] = row < n ? load4(q + (size_t)(t0 + row) * a.q_stride + 16 * s) : qe_f4{0, 0, 0, 0};
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            if (s > wave) continue;
            tr[s] = *(const qe_f4 *)(ws + row * 64 + 16 * s + 4 * c);
            mr[s] = *(const qe_f4 *)(ws + 4096 + row * 64 + 16 * s + 4 * c);
        }
        for (int j = 0; j < 4; ++j) {
            const int t = 16 * wave + 4 * c + j;
            v[j] = t < n ? (float)((const IN *)a.v)[(size_t)(t0 + t) * a.v_stride + (size_t)head * DV + col] : 0.f;
        }
        const qe_f4 cx = *(const qe_f4 *)(ws + 2 * 4096 + 16 * wave + 4 * c), cq = *(const qe_f4 *)(ws + 2 * 4096 + 64 + 16 * wave + 4 * c);
        const float last = ws[2 * 4096 + 192];
        for (int i = 0; i < SB; ++i) *(qe_f4 *)(s_t + r * LK + 16 * (wave * SB + i) + 4 * c) = S[i];
        for (int s = 0; s < KS; ++s) *(qe_f4 *)(k_s[par] + row * LK + 16 * s + 4 * c) = kr[s];
        __syncthreads();
        qe_f4 ks = {0, 0, 0, 0}, qs = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const qe_f4 b = *(const qe_f4 *)(s_t + r * LK + 16 * s + 4 * c);
            ks = mma4(kr[s], b, ks);
            qs = mma4(qr[s], b, qs);
        }
        *(qe_f4 *)(r_t + r * LT + 16 * wave + 4 * c) = cleared(v - cx * ks, par);
        __syncthreads();
        qe_f4 u = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < 4; ++s)
            if (s <= wave) u = mma4(tr[s], *(const qe_f4 *)(r_t + r * LT + 16 * s + 4 * c), u);
        *(qe_f4 *)(u_t + r * LT + 16 * wave + 4 * c) = cleared(u, par);
        __syncthreads();
        const int odd = odd_s[par][r];
        if (tid < 16) odd_s[par ^ 1][tid] = 64; // last read a chunk ago, next written in the next
        qe_f4 o = cq * qs, us[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            us[s] = *(const qe_f4 *)(u_t + r * LT + 16 * s + 4 * c);
            if (s <= wave) o = mma4(mr[s], us[s], o);
            us[s] *= *(const qe_f4 *)(ws + 2 * 4096 + 128 + 16 * s + 4 * c);
        }
        for (int j = 0; j < 4; ++j) {
            const int t = 16 * wave + 4 * c + j;
            if (t < n) ((IN *)a.out)[(size_t)(t0 + t) * a.out_stride + (size_t)head * DV + col] = (IN)(t < odd ? o[j] : NAN);
        }
#pragma unroll
        for (int i = 0; i < SB; ++i) {
            S[i] *= odd < 64 ? NAN : last;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                qe_f4 kt;
                for (int j = 0; j < 4; ++j) kt[j] = k_s[par][(16 * s + 4 * c + j) * LK + 16 * (wave * SB + i) + r];
                S[i] = mma4(kt, us[s], S[i]);
            }
        }
    }
    if (out_i >= 0)
        for (int i = 0; i < SB; ++i)
            for (int j = 0; j < 4; ++j) a.pool[(((size_t)out_i * a.v_heads + head) * DK + 16 * (wave * SB + i) + 4 * c + j) * DV + col] = S[i][j];
}

template <typename IN, int DK, int DV>
static hipError_t prompt(const QeDeltaArgs &a, hipStream_t st) {
    const unsigned chunks = (unsigned)qe_delta_max_chunks(a.n_tokens, a.n_seqs);
    k_delta_slots<<<dim3((unsigned)a.n_seqs), dim3(256), 0, st>>>(a);
    k_delta_chunks<IN, DK><<<dim3(chunks * a.k_heads), dim3(256), 0, st>>>(a);
    k_delta_scan<IN, DK, DV><<<dim3((unsigned)a.n_seqs * a.v_heads * (DV / 16)), dim3(256), 0, st>>>(a);
    return hipGetLastError();
}
template <typename IN, int DK, int DV>
static hipError_t decode(QeDeltaArgs a, hipStream_t st) {
    if (a.n_seqs <= 256) a.skip = nullptr; // every workgroup looks at all slots itself
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
