// A row of values spread over the lanes of one wave or of a workgroup: lane t
// of T holds elements [8 (t + c T), +8) for c < NV, as f32.
#pragma once
#include "common.hpp"

namespace pkx {

// Eight elements in one access at whatever alignment the element type has: gfx9
// global accesses of 16 bytes need none.
typedef half8v half8u __attribute__((aligned(2)));
typedef float4v float4u __attribute__((aligned(4)));
typedef int2v int2u __attribute__((aligned(1)));

__device__ __forceinline__ void load8u(float (&v)[8], const f16* p) {
    const half8v a = *(const half8u*)p;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)a[e];
}
__device__ __forceinline__ void load8u(float (&v)[8], const float* p) {
    const float4v a = *(const float4u*)p, b = *(const float4u*)(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[4 + e] = b[e]; }
}
__device__ __forceinline__ void store8u(f16* p, const float (&v)[8]) {
    half8v a;
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = (f16)v[e];
    *(half8u*)p = a;
}
__device__ __forceinline__ void store8u(float* p, const float (&v)[8]) {
    float4v a, b;
#pragma unroll
    for (int e = 0; e < 4; ++e) { a[e] = v[e]; b[e] = v[4 + e]; }
    *(float4u*)p = a;
    *(float4u*)(p + 4) = b;
}

// Elements [i, i + 8) of a row of d; those past its end are 0 and are not read.
template <typename T> __device__ __forceinline__ void load_row8(float (&v)[8], const T* row, int i, int d) {
    if (i + 8 <= d) {
        load8u(v, row + i);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = i + e < d ? (float)row[i + e] : 0.f;
}
template <typename T> __device__ __forceinline__ void store_row8(T* row, const float (&v)[8], int i, int d) {
    if (i + 8 <= d) {
        store8u(row + i, v);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (i + e < d) row[i + e] = (T)v[e];
}

__device__ __forceinline__ double readlane_f64(double v, int lane) {
    const long long b = __builtin_bit_cast(long long, v);
    const unsigned lo = __builtin_amdgcn_readlane((int)b, lane), hi = __builtin_amdgcn_readlane((int)(b >> 32), lane);
    return __builtin_bit_cast(double, (long long)((unsigned long long)hi << 32 | lo));
}
template <int CTRL> __device__ __forceinline__ double dpp_get_f64(double v) {
    const long long b = __builtin_bit_cast(long long, v);
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, 0xF, 0xF, false);
    const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (long long)((unsigned long long)hi << 32 | lo));
}
// Sum over a whole wave, every lane active and receiving it.
__device__ __forceinline__ double wave_sum_f64(double v) {
    v += dpp_get_f64<0xB1>(v);
    v += dpp_get_f64<0x4E>(v);
    v += dpp_get_f64<0x141>(v);
    v += dpp_get_f64<0x140>(v);
    return (readlane_f64(v, 0) + readlane_f64(v, 16)) + (readlane_f64(v, 32) + readlane_f64(v, 48));
}
__device__ __forceinline__ float wave_max_full(float v) {
    v = fmaxf(v, dpp_get<0xB1>(v));
    v = fmaxf(v, dpp_get<0x4E>(v));
    v = fmaxf(v, dpp_get<0x141>(v));
    v = fmaxf(v, dpp_get<0x140>(v));
    const int b = __builtin_bit_cast(int, v);
    const float r0 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 0));
    const float r1 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 16));
    const float r2 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 32));
    const float r3 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 48));
    return fmaxf(fmaxf(r0, r1), fmaxf(r2, r3));
}

// The largest finite magnitude among v and top.
__device__ __forceinline__ float finite_max8(const float (&v)[8], float top) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float a = fabsf(v[e]);
        top = a <= 3.402823466e38f ? fmaxf(top, a) : top;
    }
    return top;
}
// clamp(round(x / s), -127, 127), ties to even; NaN is held as 0, 0 where the scale is 0.
__device__ __forceinline__ int2v quantised8(const float (&v)[8], float s) {
    int2v w = {};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float r = s != 0.f ? rintf(v[e] / s) : 0.f;
        r = r != r ? 0.f : fminf(fmaxf(r, -127.f), 127.f);
        w[e >> 2] |= (int)((unsigned)((int)r & 0xFF) << (8 * (e & 3)));
    }
    return w;
}
__device__ __forceinline__ void store_bytes8(int8_t* row, int2v w, int i, int d) {
    if (i + 8 <= d) {
        *(int2u*)(row + i) = w;
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (i + e < d) row[i + e] = (int8_t)(w[e >> 2] >> (8 * (e & 3)));
}

}  // namespace pkx
