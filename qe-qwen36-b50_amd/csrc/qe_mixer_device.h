// Device helpers of the token mixers: 16-bit types on the matrix cores, page lookups.
#pragma once
#include "qe_mixer.h"

typedef float qe_f2 __attribute__((ext_vector_type(2)));
typedef float qe_f4 __attribute__((ext_vector_type(4)));
typedef float qe_f16v __attribute__((ext_vector_type(16)));
typedef short qe_s4 __attribute__((ext_vector_type(4)));
typedef short qe_s8 __attribute__((ext_vector_type(8)));
typedef __bf16 qe_b8 __attribute__((ext_vector_type(8)));
typedef _Float16 qe_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 qe_b2 __attribute__((ext_vector_type(2)));
typedef _Float16 qe_h2 __attribute__((ext_vector_type(2)));

#define QE_LDS(T, p) ((__attribute__((address_space(3))) T *)(p))
#define QE_GLOBAL(T, p) ((const __attribute__((address_space(1))) T *)(p))

// v_mfma_f32_16x16x32: A lane l supplies row l % 16, k = 8 (l / 16) .. + 7; B the same of
// column l % 16; D has column l % 16, rows 4 (l / 16) .. + 3.
// v_mfma_f32_32x32x16: A row l % 32, k = 8 (l / 32) .. + 7; D column l % 32, register i holds
// row 8 (i / 4) + 4 (l / 32) + i % 4.
template <bool BF>
__device__ __forceinline__ qe_f4 mfma16(qe_s8 a, qe_s8 b, qe_f4 c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(qe_b8, a), __builtin_bit_cast(qe_b8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(qe_h8, a), __builtin_bit_cast(qe_h8, b), c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ qe_f16v mfma32(qe_s8 a, qe_s8 b, qe_f16v c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(qe_b8, a), __builtin_bit_cast(qe_b8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(qe_h8, a), __builtin_bit_cast(qe_h8, b), c, 0, 0, 0);
}

// two floats to the 16-bit type, to nearest even
template <bool BF>
__device__ __forceinline__ unsigned pack2(float a, float b) {
    if constexpr (BF)
        return __builtin_bit_cast(unsigned, qe_b2{(__bf16)a, (__bf16)b});
    else
        return __builtin_bit_cast(unsigned, qe_h2{(_Float16)a, (_Float16)b});
}
template <bool BF>
__device__ __forceinline__ float from16(short x) {
    if constexpr (BF)
        return __uint_as_float((unsigned)(unsigned short)x << 16);
    else
        return (float)__builtin_bit_cast(_Float16, x);
}
// what pack2's rounding leaves of them, in 32 bits
template <bool BF>
__device__ __forceinline__ float2 rest_of(unsigned packed, float a, float b) {
    return make_float2(a - from16<BF>((short)packed), b - from16<BF>((short)(packed >> 16)));
}

// Probabilities, rounded to the cache's type for the product with V, are kept 2^UP times as large where the type is fp16,
// and so is their sum: fp16 has fixed steps below 2^-14 and nothing below 2^-25, and of 2^20 keys at 2^-25.1 of the
// greatest, 2.8 % of a row's weight, none would count.  2^15, fp16's greatest power of two, is the most they reach:
// where the subtracted maximum may lag behind the true one by 2^LAG, UP is 15 - LAG.
template <bool BF, int LAG>
__device__ __forceinline__ float exponent_base(float m) { return m == -INFINITY ? 0.f : (BF ? 0.f : 15.f - LAG) - m; }

// Transposing LDS read: of each 16 lanes, lane l addresses 4 elements of row l / 4 (columns
// 4 (l % 4) .. + 3) and gets column l of the four rows.
__device__ __forceinline__ qe_s4 lds_tr(const short *p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) qe_s4 *)p);
}
// 64 lanes x 16 bytes from global memory straight to LDS: lane l's land at dst + 16 l
__device__ __forceinline__ void load_lds16(const void *src, void *dst) {
    __builtin_amdgcn_global_load_lds(QE_GLOBAL(void, src), QE_LDS(void, dst), 16, 0, 0);
}
// The same as buffer loads: `at` bytes per lane and `more` for all behind a uniform `src`, of which `bytes` may be read.
// The compiler takes global_load_lds for one that may read LDS as well, and while one is in flight waits for all LDS reads,
// or for all loads, where it needs the first.  (ONCE: the data is not expected to be read again soon, and need not stay in
// the caches.)
template <bool ONCE = false>
__device__ __forceinline__ void load_lds16_from(const void *src, int bytes, unsigned at, unsigned more, void *dst) {
    __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc((void *)src, 0, bytes, 0x00027000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, QE_LDS(void, dst), 16, at, more, 0, ONCE ? 2 : 0);
}

// A workgroup's barrier for what it exchanges through LDS.  __syncthreads() would also wait for
// all global loads and direct loads in flight, which here are meant for later.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// 8 bytes to and from where all XCDs see the same, past their L2s
__device__ __forceinline__ void store_through(float *p, qe_f2 x) {
    __hip_atomic_store((unsigned long long *)p, __builtin_bit_cast(unsigned long long, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ qe_f2 load_through(const float *p) {
    return __builtin_bit_cast(qe_f2, __hip_atomic_load((const unsigned long long *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

__device__ __forceinline__ void report(unsigned *err, unsigned what) {
    __hip_atomic_store(err, what, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// a word of memory that no kernel in flight writes, at a wave-uniform address, through the scalar cache
__device__ __forceinline__ int scalar_load(const int32_t *p) { return *(const __attribute__((address_space(4))) int32_t *)(uintptr_t)p; }
__device__ __forceinline__ unsigned xcd_id() { return __builtin_amdgcn_s_getreg(20 | 3 << 11) & 7; } // HW_REG_XCC_ID, 4 bits

// First row of the 16 positions from pos16 (a multiple of 16) on, of one key-value head, in their page.
// A page id outside the cache becomes page 0 and sets *bad.
__device__ __forceinline__ size_t page_row(const QeAttnArgs &a, int page, int kvh, int pos16, unsigned *bad) {
    unsigned p = (unsigned)page;
    if (p >= a.n_pages) *bad = 1, p = 0;
    return (((size_t)p * a.kv_heads + kvh) << a.page_log2) + (pos16 & ((1 << a.page_log2) - 1));
}
// the same, with the page looked up
__device__ __forceinline__ size_t sub_row(const QeAttnArgs &a, const int32_t *table, int kvh, int pos16, unsigned *bad) {
    return page_row(a, scalar_load(table + (pos16 >> a.page_log2)), kvh, pos16, bad);
}

// ---- a token of an append or read: its sequence, and its row in the cache --------------------------------
struct QeToken {
    int place;    // position in its sequence; below 0: before the first
    long row;     // of key-value head 0 among all rows of the cache; -1 where place is below 0
    bool in_call; // of a sequence, as far as is known
};
// All sequences' offsets are looked at, for the report: those that are wrong may hold no token.  (Workgroups of 256 threads.)
template <typename ARGS>
__device__ __forceinline__ void report_offsets(const ARGS &a) {
    if (a.cu && (int64_t)blockIdx.x * 256 < a.n_seqs)
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.n_seqs; i += (int64_t)gridDim.x * 256)
            if (qe_bad_offsets(a.cu[i], a.cu[i + 1], a.n_tokens)) report(a.err, QE_BAD_LENGTH);
}
// Token t's, by every wave for itself, through the scalar cache, with no barrier.  False: it has none; `teller` reports why.
template <typename ARGS>
__device__ __forceinline__ bool token_place(const ARGS &a, int t, bool teller, QeToken &x) {
    // the last sequence whose first row is not behind t
    int seq = t, end = t + 1;
    bool known = true;
    x.in_call = true;
    if (a.cu) {
        int lo = 0, hi = a.n_seqs; // cu[lo] <= t < cu[hi], as far as cu rises
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (scalar_load(a.cu + mid) <= t) lo = mid;
            else hi = mid;
        }
        // next to offsets that fall, it is not known whose the token is
        const int before = scalar_load(a.cu + (lo ? lo - 1 : 0)), begin = scalar_load(a.cu + lo), after = scalar_load(a.cu + (lo + 2 <= a.n_seqs ? lo + 2 : a.n_seqs));
        end = scalar_load(a.cu + lo + 1);
        known = before <= begin && end <= after && !qe_bad_offsets(begin, end, a.n_tokens);
        if (t < begin || t >= end) { // of no sequence
            x.in_call = false;
            return false;
        }
        seq = lo;
    }
    unsigned bad = 0;
    const int len = qe_checked(scalar_load(a.kv_len + seq), 0, a.max_pages << a.page_log2, -1, &bad);
    x.place = len - end + t;
    x.row = -1;
    if (!known || bad) {
        if (teller) report(a.err, QE_BAD_LENGTH);
        return false;
    }
    if (x.place >= 0) {
        const unsigned p = (unsigned)scalar_load(a.table + (size_t)seq * a.table_stride + (x.place >> a.page_log2));
        if (p >= a.n_pages) {
            if (teller) report(a.err, QE_BAD_PAGE);
            return false;
        }
        x.row = ((long)p * a.kv_heads << a.page_log2) + (x.place & ((1 << a.page_log2) - 1));
    }
    return true;
}

// ---- codes of 8 bits ------------------------------------------------------------------------------------
// a word's four codes in 32 bits
template <int CT>
__device__ __forceinline__ void floats_of(unsigned w, float *y) {
    if constexpr (CT == QE_I8) {
        for (int i = 0; i < 4; ++i) y[i] = (float)(signed char)(w >> (8 * i));
    } else {
        const qe_f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        y[0] = a[0], y[1] = a[1], y[2] = b[0], y[3] = b[1];
    }
}

// eight codes as the matrix cores' 16-bit type; exact, a code has at most 8 bits
template <int CT, bool BF>
__device__ __forceinline__ qe_s8 elements_of(unsigned lo, unsigned hi) {
    unsigned r[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const unsigned w = h ? hi : lo;
        if constexpr (CT == QE_F8 && BF) {
            r[2 * h] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
            r[2 * h + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true));
        } else if constexpr (CT == QE_F8) {
            r[2 * h] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
            r[2 * h + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true));
        } else if constexpr (BF) {
            float y[4];
            floats_of<QE_I8>(w, y);
            r[2 * h] = pack2<true>(y[0], y[1]);
            r[2 * h + 1] = pack2<true>(y[2], y[3]);
        } else { // 1024 + (code + 128), by a byte before it, less 1152
            const unsigned u = w ^ 0x80808080u;
            const qe_h2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
            r[2 * h] = __builtin_bit_cast(unsigned, __builtin_bit_cast(qe_h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off);
            r[2 * h + 1] = __builtin_bit_cast(unsigned, __builtin_bit_cast(qe_h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off);
        }
    }
    return __builtin_bit_cast(qe_s8, make_uint4(r[0], r[1], r[2], r[3]));
}
// Lane I of each 16's value, to all of them: the compiler makes it an operand of the instruction that uses it.
template <int I>
__device__ __forceinline__ float of_lane(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x150 + I, 0xf, 0xf, true));
}
// A scale's bits without sign, in the order of their sizes; none of one that is not finite, which reaches the rows that attend to it
// without this.
__device__ __forceinline__ unsigned size_bits(float scale) {
    const unsigned x = __float_as_uint(scale) & 0x7fffffffu;
    return x >= 0x7f800000u ? 0 : x;
}
// The greatest over all lanes.
__device__ __forceinline__ unsigned greatest(unsigned top) {
    top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0xb1, 0xf, 0xf, true));
    top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x4e, 0xf, 0xf, true));
    top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x141, 0xf, 0xf, true));
    top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x140, 0xf, 0xf, true));
    const auto a = __builtin_amdgcn_permlane16_swap(top, top, false, false);
    top = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(top, top, false, false);
    return __builtin_amdgcn_readfirstlane(max(b[0], b[1]));
}
// The value scales of an 8-bit cache as fp16 probabilities can take them: a probability times a scale has no bounded range, but
// times scale / unit it has, where unit is a power of two that is above all scales so far.  The sums with V count units; they are
// brought to a new one where a tile has a greater scale.  (bf16 has the range of 32 bits and needs none.)
struct Units {
    float unit = 0, inverse = 0;
    // `scale`, over all lanes: a tile's; those of fewer lanes are in others, too.  What sums so far are to be multiplied by.
    __device__ __forceinline__ float raise(float scale) {
        const unsigned bits = greatest(size_bits(scale));
        if (__uint_as_float(bits) <= unit) return 1.f;
        // two to four times the greatest, so that it seldom changes; within 2^-100 .. 2^100
        unsigned e = (bits >> 23) + 2;
        e = e < 27 ? 27 : e > 227 ? 227 : e;
        const float was = unit, next = __uint_as_float(e << 23);
        if (next <= was) return 1.f;
        unit = next;
        inverse = __uint_as_float((254 - e) << 23);
        return was * inverse;
    }
};
// Transposing LDS read of bytes: of each 16 lanes, lane l addresses 8 bytes of row l / 2 (columns 8 (l % 2) .. + 7) and gets
// column l of the eight rows.
__device__ __forceinline__ uint2 lds_tr8(const uint8_t *p) {
    typedef int i2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i2 *)p));
}
// Permutation of a row's 16-byte chunks of codes in LDS: the 16 rows that half a wave reads with lds_tr8 lie in different banks.
template <int DH>
__device__ __forceinline__ int swz8(int row) { // of the 16-byte chunk index
    return DH == 256 ? (row & 7) | (row >> 4 & 1) << 3 : DH == 128 ? (row >> 1 & 3) | (row >> 4 & 1) << 2 : (row >> 2 & 1) | (row >> 4 & 1) << 1;
}
