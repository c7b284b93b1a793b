// attn_mfma.h -- what the matrix kernels of the attention share: vector types,
// products, copies to LDS, swizzles, the sequence of a unit of rows.
#pragma once

#include "attn.h"
#include "tkv_reduce.h"

namespace tkv {
namespace attn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Vec {  // 16 bytes
    static constexpr int N = 16 / sizeof(T);
    typedef T type __attribute__((ext_vector_type(N)));
};

__device__ __forceinline__ f32x4 mfma16(Vec<__bf16>::type a, Vec<__bf16>::type b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(Vec<_Float16>::type a, Vec<_Float16>::type b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(bf16x4 a, bf16x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a),
                                                     __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(f16x4 a, f16x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(Vec<__bf16>::type a, Vec<__bf16>::type b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(Vec<_Float16>::type a, Vec<_Float16>::type b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// 16 bytes per lane from global memory to LDS at `dst` (wave-uniform) + 16 lane.
// In asm, since the compiler would put a wait for every copy in flight before
// each LDS read it cannot tell apart from the copy's destination; the waits
// here are the callers' own (wait_vm below, before a barrier).  No register is
// written but m0, which is named as clobbered, so that the compiler carries no value
// of its own in it across the copy (it warns of any reserved register there); the
// s_nop is the wait state between a scalar write of m0 and the copy that uses it.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy16_to_lds(const void* src, unsigned dst) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                 :
                 : "v"(src), "s"(dst)
                 : "memory", "m0");
}
// The same from a wave-uniform base and a byte offset per lane.
__device__ __forceinline__ void copy16_to_lds(const char* base, uint32_t offset, unsigned dst) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :
                 : "v"(offset), "s"(base), "s"(dst)
                 : "memory", "m0");
}
// 4 bytes per lane, to `dst` + 4 lane.
__device__ __forceinline__ void copy4_to_lds(const void* src, unsigned dst) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
                 :
                 : "v"(src), "s"(dst)
                 : "memory", "m0");
}
#pragma clang diagnostic pop
// Waits until at most N of the wave's memory operations are in flight.
template <int N>
__device__ __forceinline__ void wait_vm_but() {
    static_assert(N >= 0 && N < 64, "vmcnt");
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
__device__ __forceinline__ unsigned lds_at(const void* p) {
    return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ const char* uniform(const char* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    return reinterpret_cast<const char*>((uint64_t)(uint32_t)uniform((int)v) |
                                         (uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32);
}
// A wave-uniform element of read-only memory, through the scalar cache.
__device__ __forceinline__ int load_uniform(const int32_t* p) {
    return *(const __attribute__((address_space(4))) int32_t*)p;
}

// The other half's value: lanes l and l + 32 exchange.
__device__ __forceinline__ float other_half(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(threadIdx.x & 32 ? r[0] : r[1]);
}

// The same between 16-lane rows: lanes l and l ^ 16.
__device__ __forceinline__ float other_row(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(threadIdx.x & 16 ? r[0] : r[1]);
}

// LDS rows of CPR 16-byte chunks.  Key rows are read 16 lanes = 16 rows at one
// chunk at a time: the chunk is XORed so that the 16 land in different banks.
template <int CPR>
__device__ __forceinline__ int swz_k(int row) {
    if constexpr (CPR % 16 == 0) return row & 15;
    else if constexpr (CPR % 8 == 0) return (row >> 1) & 7;
    else if constexpr (CPR % 4 == 0) return (row >> 2) & 3;
    else return (row >> 3) & 1;
}
// Value rows are read four rows (16-bit types; two rows 4 apart for f32) at a
// 64-byte (128-byte) window at a time: the window is XORed.
template <int CPR, int SIZE>
__device__ __forceinline__ int swz_v(int row) {
    if constexpr (SIZE == 4) return CPR % 16 == 0 ? ((row >> 2) & 1) << 3 : 0;
    else if constexpr (CPR % 16 == 0) return (row & 3) << 2;
    else if constexpr (CPR % 8 == 0) return ((row >> 1) & 1) << 2;
    else return 0;
}

enum { KV_PACKED = 0, KV_PAGED = 1, KV_I8 = 2 };

// Sequence of a unit of ROWS query rows, and the sequence's first unit: sequence
// i's units begin at floor(cu[i] g / ROWS) + i, which leaves each sequence room
// for all of its rows (and up to one unit without any).  Lanes look at 64
// sequences at a time: the last one that begins at or before the unit.  -1 for a
// unit before the first sequence's: its rows are nobody's, and taking the first
// sequence's again would write them from two workgroups, the second of which
// could read queries that the first had stored its outputs over.
template <bool PAGED, int ROWS>
__device__ __forceinline__ int tile_seq(const AttnArgs& a, int unit, int* first) {
    const int lane = threadIdx.x & 63;
    int found = -1, begin = 0;
    for (int b = 0; b < a.seqs; b += 64) {
        const int i = b + lane;
        int at = 0x7fffffff;
        if (i < a.seqs) {
            const int q0 = (PAGED && !a.cu_q) ? i : clamp_to(a.cu_q[i], a.tokens);
            at = (int)((int64_t)q0 * a.g / ROWS) + i;
        }
        const unsigned long long before = __ballot(at <= unit);
        if (!before) break;
        const int last = 63 - __builtin_clzll(before);
        found = b + last;
        begin = __shfl(at, last);
        if (last < 63) break;
    }
    *first = uniform(begin);
    return uniform(found);
}

// f16 weights are exp2(a - m + 7): with the 2^8 that the maximum may lag, up to
// 2^15, below f16's largest.  The top one of a row is at least 2^7, so f16's
// smallest step rounds weights down to 2^-21 of it to 11 bits and drops none
// above 2^-32 of it (at exp2(a - m), 2^-25: 131071 keys just below that are 2^-8 of
// the sum).  (m - kLift, l, O) is what the joins of waves and splits get.
template <typename T, bool SCALED>
constexpr float kLift = std::is_same<T, _Float16>::value && !SCALED ? 7.0f : 0.0f;

// f16 weights over an int8 cache: each weight is multiplied by its value's scale,
// and the products reach over more octaves than f16 has, so they are taken, and O
// is kept, in units of a power of two.  The unit follows the row's largest product
// so far, `top`, in the weights' present base (never the scales alone: a key of no
// weight may have any).  It is raised at once, to 2^14 below the product, and
// lowered once that is over 2^8 too high: a product is off by 2^-11 of itself or
// 2^-31 of the largest.  0 while every product is.
__device__ __forceinline__ float product_unit(float unit, float top) {
    const int e = (int)(__float_as_uint(top) >> 23);  // top >= 0; 255: not finite
    if (top == 0.0f || e == 255) return unit;
    const float u = __uint_as_float((unsigned)max(e - 14, 27) << 23);  // 2^-100 at least
    return u > unit || u < unit * 0x1p-8f ? fmaxf(u, unit * 0x1p-100f) : unit;
}
// 1 / unit (2^127 for 0).
__device__ __forceinline__ float inverse_unit(float unit) {
    return __uint_as_float((254u << 23) - __float_as_uint(unit));
}

// Partial sums of a split, written where the unit's last workgroup, on whatever
// XCD, reads them (agent scope: past this XCD's L2; see arrive_last).  8 bytes is
// the widest such access, so sums are laid out for lanes to be 8 bytes apart: a
// wave writes and reads whole lines.  (16 bytes apart, in rows of the output, the
// same traffic took twice as long as the whole attention of 8 x 1024 tokens.)
typedef unsigned long long u64;
__device__ __forceinline__ void put_sum(u64* p, float x, float y) {
    __hip_atomic_store(p, (u64)__float_as_uint(x) | ((u64)__float_as_uint(y) << 32), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get_sum(const u64* p) {
    const u64 w = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((unsigned)w), __uint_as_float((unsigned)(w >> 32)));
}

// Four elements of an output row.
template <typename T>
__device__ __forceinline__ void put_out4(const AttnArgs& a, int64_t token, int head, int e, f32x4 y) {
    const int64_t at = token * a.o_st + (int64_t)head * a.o_sh + e;
    if (sizeof(T) == 4 || a.out_f32) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + at) = y;
    } else {
        typedef T T4 __attribute__((ext_vector_type(4)));
        T4 z;
#pragma unroll
        for (int j = 0; j < 4; j++) z[j] = (T)y[j];
        *reinterpret_cast<T4*>(static_cast<T*>(a.out) + at) = z;
    }
}

// An output row from the sums of attend_row, by one wave.
template <typename T>
__device__ __forceinline__ void put_row(const AttnArgs& a, int64_t token, int head, float l, const float (&acc)[4]) {
    const int lane = threadIdx.x & 63;
    const int64_t at = token * a.o_st + (int64_t)head * a.o_sh;
    for (int e = 0; e < 4; e++) {
        const int x = lane + 64 * e;
        if (x >= a.d) continue;
        const float y = l == 0.0f ? 0.0f : acc[e] / l;
        if (a.out_f32) static_cast<float*>(a.out)[at + x] = y;
        else static_cast<T*>(a.out)[at + x] = from_f32<T>(y);
    }
}

}  // namespace attn
}  // namespace tkv
