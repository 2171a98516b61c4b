// Eight consecutive elements of a 32- or 16-bit type a lane: loads, stores and conversions for the token and activation kernels.
#pragma once
#include "common.h"

typedef uint32_t u32;
constexpr int kVec = 8;

typedef u32 u32x4 __attribute__((ext_vector_type(4)));
template <typename T> struct Raw8;
template <> struct Raw8<float> { u32x4 a, b; };
template <> struct Raw8<__bf16> { u32x4 a; };
template <> struct Raw8<_Float16> { u32x4 a; };
// rows of an odd vocabulary start at any element: the type says so, the hardware takes unaligned 16-byte accesses
typedef u32x4 u32x4_any __attribute__((aligned(2)));

__device__ __forceinline__ void unpack8(const Raw8<float> &r, float *z) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const u32 a = r.a[i], b = r.b[i];  // (a bit_cast of a vector's element itself reads element 0)
        z[i] = __builtin_bit_cast(float, a);
        z[4 + i] = __builtin_bit_cast(float, b);
    }
}
__device__ __forceinline__ void unpack8(const Raw8<__bf16> &r, float *z) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        z[2 * i] = __builtin_bit_cast(float, r.a[i] << 16);
        z[2 * i + 1] = __builtin_bit_cast(float, r.a[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack8(const Raw8<_Float16> &r, float *z) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const u32 a = r.a[i];
        const h2 v = __builtin_bit_cast(h2, a);
        z[2 * i] = (float)v[0];
        z[2 * i + 1] = (float)v[1];
    }
}
template <typename T>
__device__ __forceinline__ u32 pack2(float a, float b) {  // one rounding to nearest even: the result's type
    typedef T t2 __attribute__((ext_vector_type(2)));
    const t2 v = {(T)a, (T)b};
    return __builtin_bit_cast(u32, v);
}
template <typename T>
__device__ __forceinline__ void load8(const T *p, int n, Raw8<T> &r) {
    if (n >= kVec) {
        r.a = *(const u32x4_any *)p;
        if constexpr (sizeof(T) == 4) r.b = *((const u32x4_any *)p + 1);
    } else {  // the row's last lane
        T t[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) t[i] = i < n ? p[i] : (T)0.0f;
        r = __builtin_bit_cast(Raw8<T>, t);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T *p, int n, const float *z) {
    if (n >= kVec) {
        if constexpr (sizeof(T) == 4) {
            u32x4 a, b;
#pragma unroll
            for (int i = 0; i < 4; ++i) { a[i] = __builtin_bit_cast(u32, z[i]); b[i] = __builtin_bit_cast(u32, z[4 + i]); }
            *(u32x4_any *)p = a;
            *((u32x4_any *)p + 1) = b;
        } else {
            u32x4 a;
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = pack2<T>(z[2 * i], z[2 * i + 1]);
            *(u32x4_any *)p = a;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
            if (i < n) p[i] = (T)z[i];
    }
}

template <bool B>
struct Bool { static constexpr bool value = B; };  // a condition of a generic lambda's

__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, dpp_mov<0xB1>(x));
    x = fmaxf(x, dpp_mov<0x4E>(x));
    x = fmaxf(x, dpp_mov<0x141>(x));
    x = fmaxf(x, dpp_mov<0x140>(x));
    return fmaxf(fmaxf(read_lane(x, 0), read_lane(x, 16)), fmaxf(read_lane(x, 32), read_lane(x, 48)));
}
__device__ __forceinline__ float wave_sum(float x) {
    x += dpp_mov<0xB1>(x);
    x += dpp_mov<0x4E>(x);
    x += dpp_mov<0x141>(x);
    x += dpp_mov<0x140>(x);
    return (read_lane(x, 0) + read_lane(x, 16)) + (read_lane(x, 32) + read_lane(x, 48));
}
