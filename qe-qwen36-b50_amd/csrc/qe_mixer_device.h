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
