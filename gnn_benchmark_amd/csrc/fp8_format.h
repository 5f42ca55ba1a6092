// The 8-bit format of the training operators (include/gnn_train.h): e4m3 codes in blocks of 128 with a power-of-two
// scale per block, and the loads and stores of fp32 / bf16 rows that its producers share.
#pragma once

#include "common.h"
#include "gnn_train.h"

namespace gnnagg {

constexpr int kBlock8 = 128;              // values under one scale
constexpr int kMinExp8 = -126, kMaxExp8 = 120;
constexpr float kFloatMax = 3.402823466e38f;

inline int64_t pad128(int64_t n) { return (n + kBlock8 - 1) / kBlock8 * kBlock8; }

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
struct bf16_t {                           // storage of one bf16 value
    unsigned short bits;
};

__device__ __forceinline__ float bf16_value(unsigned short b) { return __uint_as_float((uint32_t)b << 16); }

// 2^e, -126 <= e <= 127
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Smallest e with top * 2^-e <= 448 = 1.75 * 2^8, inside the format's range; top finite and >= 0.
__device__ __forceinline__ int block_exponent(float top) {
    const uint32_t u = __float_as_uint(top);
    const int p = (int)(u >> 23) - 127;   // (a subnormal top lands below the range either way)
    const int e = p - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < kMinExp8 ? kMinExp8 : (e > kMaxExp8 ? kMaxExp8 : e);
}

__device__ __forceinline__ float finite_magnitude(float x) {
    const float a = __builtin_fabsf(x);
    return a <= kFloatMax ? a : 0.0f;     // 0 for infinities and NaN
}
__device__ __forceinline__ float finite_magnitude(const f32x4 v) {
    return fmaxf(fmaxf(finite_magnitude(v.x), finite_magnitude(v.y)),
                 fmaxf(finite_magnitude(v.z), finite_magnitude(v.w)));
}

// an infinity becomes NaN, so that the conversion's own treatment of it does not matter
__device__ __forceinline__ float nan_unless_finite(float x) {
    return __builtin_fabsf(x) <= kFloatMax ? x : __builtin_nanf("");
}

// four values scaled by inv = 2^-e (|v * inv| <= 448) -> four codes, the first in the lowest byte
__device__ __forceinline__ uint32_t encode4(const f32x4 v, float inv) {
    uint32_t r = 0;
    r = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(nan_unless_finite(v.x) * inv, nan_unless_finite(v.y) * inv, (int)r, false);
    r = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(nan_unless_finite(v.z) * inv, nan_unless_finite(v.w) * inv, (int)r, true);
    return r;
}

__device__ __forceinline__ f32x4 decode4(uint32_t c) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false);
    const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    return f32x4{lo.x, lo.y, hi.x, hi.y};
}

// the largest of 32 neighbouring lanes' words, in all of them
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    // (turned by 1, 2, 4 and 8 lanes inside sixteen, then the sixteens exchanged: on the vector unit, LDS takes no part)
    const auto larger = [](uint32_t a, int b) { return (uint32_t)b > a ? (uint32_t)b : a; };
    v = larger(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
    v = larger(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
    v = larger(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
    v = larger(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));
    const auto pair = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return pair[0] > pair[1] ? pair[0] : pair[1];
}

// Four consecutive values of a row of `width`, the first at column c, as they lie in memory (load4_raw: nothing waits for
// them before widen) or in fp32.  VEC: the row is aligned for one wide load and width % 4 == 0.  Columns past the width
// read as zero.
__device__ __forceinline__ f32x4 widen(const f32x4 v) { return v; }
__device__ __forceinline__ f32x4 widen(const u16x4 u) {
    return f32x4{bf16_value(u.x), bf16_value(u.y), bf16_value(u.z), bf16_value(u.w)};
}
// (I: int where the width allows; comparisons of 64 bits are what a narrow row's time goes into.)
template <bool VEC, typename I>
__device__ __forceinline__ f32x4 load4_raw(const float *row, I c, I width) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (VEC) {
        if (c < width) v = *reinterpret_cast<const f32x4 *>(row + c);
    } else if (width > 0) {  // four loads in bounds, what they read past the width replaced: no branch between them
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = row[c + j < width ? c + j : width - 1];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = c + j < width ? v[j] : 0.0f;
    }
    return v;
}
template <bool VEC, typename I>
__device__ __forceinline__ u16x4 load4_raw(const bf16_t *row, I c, I width) {
    u16x4 v = {0, 0, 0, 0};
    if (VEC) {
        if (c < width) v = *reinterpret_cast<const u16x4 *>(row + c);
    } else if (width > 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = row[c + j < width ? c + j : width - 1].bits;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = c + j < width ? v[j] : (unsigned short)0;
    }
    return v;
}
template <bool VEC, typename T, typename I>
__device__ __forceinline__ f32x4 load4(const T *row, I c, I width) {
    return widen(load4_raw<VEC>(row, c, width));
}
template <typename T>
struct RawOf;
template <>
struct RawOf<float> {
    typedef f32x4 type;
};
template <>
struct RawOf<bf16_t> {
    typedef u16x4 type;
};

// two fp32 values -> two bf16 in one word (round to nearest even, the hardware's conversion)
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    union {
        bf16x2_t h;
        uint32_t u;
    } x;
    x.h = __builtin_convertvector(f32x2{a, b}, bf16x2_t);
    return x.u;
}

template <bool VEC, typename I>
__device__ __forceinline__ void store4(float *row, I c, I width, const f32x4 v) {
    if (VEC) {
        if (c < width) *reinterpret_cast<f32x4 *>(row + c) = v;
    } else {
        if (c + 0 < width) row[c + 0] = v.x;
        if (c + 1 < width) row[c + 1] = v.y;
        if (c + 2 < width) row[c + 2] = v.z;
        if (c + 3 < width) row[c + 3] = v.w;
    }
}
template <bool VEC, typename I>
__device__ __forceinline__ void store4(bf16_t *row, I c, I width, const f32x4 v) {
    const uint32_t lo = bf16_pair(v.x, v.y), hi = bf16_pair(v.z, v.w);
    if (VEC) {
        if (c < width) *reinterpret_cast<uint2 *>(row + c) = uint2{lo, hi};
    } else {
        if (c + 0 < width) row[c + 0].bits = (unsigned short)lo;
        if (c + 1 < width) row[c + 1].bits = (unsigned short)(lo >> 16);
        if (c + 2 < width) row[c + 2].bits = (unsigned short)hi;
        if (c + 3 < width) row[c + 3].bits = (unsigned short)(hi >> 16);
    }
}

// what store4 leaves in memory, as fp32
__device__ __forceinline__ f32x4 rounded(const float *, const f32x4 v) { return v; }
__device__ __forceinline__ f32x4 rounded(const bf16_t *, const f32x4 v) {
    const uint32_t lo = bf16_pair(v.x, v.y), hi = bf16_pair(v.z, v.w);
    return f32x4{bf16_value((unsigned short)lo), bf16_value((unsigned short)(lo >> 16)), bf16_value((unsigned short)hi),
                 bf16_value((unsigned short)(hi >> 16))};
}

// A barrier for what the block's threads wrote to LDS.  __syncthreads() also waits for every load from memory still on its
// way to registers, which takes the point out of asking for them early.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Keeps an address that is the same for the whole wave in scalar registers.  (Said to be global memory's on the way through:
// behind the asm the compiler would not know, and a flat load also counts as an LDS access, which every barrier waits for.)
template <typename T>
__device__ __forceinline__ const T *scalar(const T *p) {
    const __attribute__((address_space(1))) T *global = (const __attribute__((address_space(1))) T *)p;
    asm volatile("" : "+s"(global));
    return (const T *)global;
}

// host: may rows at p with this stride and width be moved four values at a time?
inline bool vec4_rows(const void *p, int64_t stride, int64_t width, int dtype) {
    const uintptr_t bytes = dtype == GNNAGG_F32 ? 16 : 8;
    return !p || (width % 4 == 0 && stride % 4 == 0 && reinterpret_cast<uintptr_t>(p) % bytes == 0);
}
inline bool known_dtype(int dtype) { return dtype == GNNAGG_F32 || dtype == GNNAGG_BF16; }

// out[c] = sum over b < blocks of partial[b][c], in a fixed order (rmsnorm.hip)
int launch_column_reduce(const float *partial, int64_t blocks, int64_t width, float *out, hipStream_t stream);

}  // namespace gnnagg
