// gnr_int8.h -- what gnr_quant.hip (8-bit rows: quantise, cache write, cache read) and gnr_int8.hip (their product) share.
//
// A ROW is the channel vector of one pixel (or one token): K signed bytes, contiguous, and ONE fp32 scale:
//     a = max(max_k |x_k|, 2^-100)      scale = a / 127      q_k = rint(fl32(x_k * fl32(127 / a)))
// The two roundings to fp32 belong to the definition (a value on the border between two steps has one answer).  |q| <= 127:
// x_k / a <= 1 and 127 * (1 + 2^-23) still rounds to 127.  The floor 2^-100 keeps 127 / a finite; an all-zero row has q = 0.
// A row that holds an Inf or a NaN gets q = 0 and scale = NaN: it reads back as NaN, in products too.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/gnr.h"

namespace gnr {
int fail(const char* fmt, ...);

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float fv4 __attribute__((ext_vector_type(4)));

constexpr unsigned ROW_FLOOR_BITS = 0x0d800000u;        // 2^-100

// Elements of 16 consecutive bytes.  The pointers need the element's own alignment only: gfx950 loads and stores 16 bytes
// at any address (rows of 129 halves or 387 floats start anywhere), so no path is split on alignment.
template <typename T> struct Vec {
    static constexpr int N = 16 / sizeof(T);
    T v[N];
};
template <typename T> __device__ __forceinline__ Vec<T> load_vec(const T* p) {
    Vec<T> r;
    __builtin_memcpy(&r, p, 16);
    return r;
}
// n < N elements (none for n <= 0), the rest 0
template <typename T> __device__ __forceinline__ Vec<T> load_part(const T* p, int n) {
    if (n >= Vec<T>::N) return load_vec(p);
    Vec<T> r;
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i) r.v[i] = i < n ? p[i] : (T)0.0f;
    return r;
}
constexpr long CACHES = 256L << 20;                      // bytes behind the L2s
// STREAM: a result that exceeds the caches goes past them (gnr_quant.hip, read_maps_kernel on rows that the caches hold: 112 -> 51 us)
template <bool STREAM = false, typename T> __device__ __forceinline__ void store_part(T* p, const Vec<T>& r, int n) {
    if (n >= Vec<T>::N) {
        if constexpr (STREAM) {
            typedef int any4 __attribute__((ext_vector_type(4), aligned(1)));
            __builtin_nontemporal_store(__builtin_bit_cast(any4, r), (any4*)p);
        } else {
            __builtin_memcpy(p, &r, 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < Vec<T>::N; ++i)
            if (i < n) p[i] = r.v[i];
    }
}

// 16 bytes of elements kept as four words between the row maximum and the quantisation (16-bit elements stay packed: unpacked, a
// thread's share of a row would be twice the registers).  The maximum works on the words: without the sign bits they are ordered
// like |x|, with Inf and NaN on top.
struct Raw16 {
    unsigned w[4];
};
template <typename T> __device__ __forceinline__ Raw16 load_raw(const T* p, int n) {          // n >= 1 elements, the rest 0
    Raw16 r = {};
    if (n >= Vec<T>::N) __builtin_memcpy(&r, p, 16);
    else
#pragma unroll
        for (int i = 0; i < Vec<T>::N; ++i)
            if (i < n) {
                if constexpr (sizeof(T) == 4) r.w[i] = __builtin_bit_cast(unsigned, p[i]);
                else r.w[i >> 1] |= (unsigned)__builtin_bit_cast(unsigned short, p[i]) << 16 * (i & 1);
            }
    return r;
}
template <typename T> __device__ __forceinline__ unsigned max_bits(unsigned a, unsigned w) {
    if constexpr (sizeof(T) == 4) {
        w &= 0x7fffffffu;
        return w > a ? w : a;
    } else {
        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, w & 0x7fff7fffu)));
    }
}
template <typename T> __device__ __forceinline__ float raw_value(const unsigned (&w)[4], int v) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[v]);
    else return (float)__builtin_bit_cast(T, (unsigned short)(w[v >> 1] >> 16 * (v & 1)));
}

// the row's scale and its reciprocal step from the bits of its largest |x|; a row with an Inf / NaN: per = 0, scale = NaN
__device__ __forceinline__ void row_scale(unsigned a_bits, float& scale, float& per) {
    const bool bad = a_bits >= 0x7f800000u;
    const float a = __uint_as_float(a_bits > ROW_FLOOR_BITS ? a_bits : ROW_FLOOR_BITS);
    scale = bad ? __uint_as_float(0x7fc00000u) : a / 127.0f;
    per = bad ? 0.0f : 127.0f / a;
}
// per == 0 marks a bad row: its values may be Inf / NaN, whose product is NaN -> q = 0
__device__ __forceinline__ int row_step(float x, float per) { return per == 0.0f ? 0 : (int)rintf(x * per); }
__device__ __forceinline__ unsigned pack4(int a, int b, int c, int d) {
    return (unsigned)(a & 255) | (unsigned)(b & 255) << 8 | (unsigned)(c & 255) << 16 | (unsigned)d << 24;
}

// Where row `i` of a slot list lives.  slots == NULL: i itself.  A negative slot is padding (an empty row), a slot beyond the
// cache a mistake: neither is addressed, the caller gets base 0 and the scale that stands for it (0 / NaN).
struct SlotRef {
    long slot;
    int state;        // 0: in the cache; 1: padding; 2: out of range
};
__device__ __forceinline__ SlotRef slot_of(const int64_t* slots, long n_slots, long i) {
    if (!slots) return SlotRef{i, 0};
    const long s = slots[i];
    return s < 0 ? SlotRef{0, 1} : (s >= n_slots ? SlotRef{0, 2} : SlotRef{s, 0});
}

// Workgroups go round robin over the 8 XCDs: block i works on tile (i % 8) (n / 8) + i / 8, so that one XCD walks neighbouring tiles
__device__ __forceinline__ unsigned xcd_block(unsigned n) {
    const unsigned per = n >> 3;
    return blockIdx.x < per * 8 ? (blockIdx.x & 7) * per + (blockIdx.x >> 3) : blockIdx.x;
}

// A grid counts its threads in 32 bits; a larger one is cut off without an error
inline int check_grid(const char* what, long blocks, long threads) {
    return blocks * threads < (1L << 32) ? 0 : fail("%s: %ld workgroups of %ld threads exceed one launch", what, blocks, threads);
}
int launch_quantize(const GnrRowsProblem& p, hipStream_t st);        // defined in gnr_quant.hip; 0 == enqueued
}  // namespace gnr
