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
// Stores past the caches next to the units: what these kernels write they do not read again, and lines kept for it push out
// what they do (4 x 8192 tokens turned 49.3 -> 44.3 us, 2000 x 1024 normed 8.6 -> 7.6; loads past them cost a quarter more).
__device__ __forceinline__ void store8u(f16* p, const float (&v)[8]) {
    half8v a;
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = (f16)v[e];
    __builtin_nontemporal_store(a, (half8u*)p);
}
__device__ __forceinline__ void store8u(float* p, const float (&v)[8]) {
    float4v a, b;
#pragma unroll
    for (int e = 0; e < 4; ++e) { a[e] = v[e]; b[e] = v[4 + e]; }
    __builtin_nontemporal_store(a, (float4u*)p);
    __builtin_nontemporal_store(b, (float4u*)(p + 4));
}

// Elements [i, i + 8) of a row of d; those past its end are 0 and are not read.  d may be all that an int holds.
template <typename T> __device__ __forceinline__ void load_row8(float (&v)[8], const T* row, int i, int d) {
    if (i <= d - 8) {
        load8u(v, row + i);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if (i >= d) return;
    T a[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = row[i + e < d ? i + e : d - 1];       // the last one again: no branch for each
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = i + e < d ? (float)a[e] : 0.f;
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

// The same in pieces of four.
template <typename T> __device__ __forceinline__ void load_row4(float* v, const T* row, int i, int d) {
    typedef T vec __attribute__((ext_vector_type(4)));
    typedef vec vecu __attribute__((aligned(sizeof(T))));
    if (i + 4 <= d) {
        const vec a = *(const vecu*)(row + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)a[e];
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = i + e < d ? (float)row[i + e] : 0.f;
}
template <typename T> __device__ __forceinline__ void store_row4(T* row, const float* v, int i, int d) {
    typedef T vec __attribute__((ext_vector_type(4)));
    typedef vec vecu __attribute__((aligned(sizeof(T))));
    if (i + 4 <= d) {
        vec a;
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = (T)v[e];
        __builtin_nontemporal_store(a, (vecu*)(row + i));
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
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
// Sum over the T = 16, 32 or 64 lanes that share a row, all of them active and receiving it (other rows' lanes need not be).
template <int T> __device__ __forceinline__ double lanes_sum_f64(double v) {
    v += dpp_get_f64<0xB1>(v);
    v += dpp_get_f64<0x4E>(v);
    v += dpp_get_f64<0x141>(v);
    v += dpp_get_f64<0x140>(v);
    if constexpr (T == 16) return v;
    const double a = readlane_f64(v, 0) + readlane_f64(v, 16), b = readlane_f64(v, 32) + readlane_f64(v, 48);
    return T == 64 ? a + b : (threadIdx.x & 32) ? b : a;
}
template <int T> __device__ __forceinline__ float lanes_max(float v) {
    v = fmaxf(v, dpp_get<0xB1>(v));
    v = fmaxf(v, dpp_get<0x4E>(v));
    v = fmaxf(v, dpp_get<0x141>(v));
    v = fmaxf(v, dpp_get<0x140>(v));
    if constexpr (T == 16) return v;
    const int b = __builtin_bit_cast(int, v);
    const float r0 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 0));
    const float r1 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 16));
    const float r2 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 32));
    const float r3 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 48));
    if constexpr (T == 32) return (threadIdx.x & 32) ? fmaxf(r2, r3) : fmaxf(r0, r1);
    return fmaxf(fmaxf(r0, r1), fmaxf(r2, r3));
}

// The largest magnitude of a row, and whether it holds an infinity or a NaN: `odd` is 0 times every value, NaN then.
struct RowMax {
    float top = 0.f, odd = 0.f;
    __device__ __forceinline__ void add(const float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            top = fmaxf(top, fabsf(v[e]));
            odd = fmaf(v[e], 0.f, odd);
        }
    }
};
// The largest finite magnitude among v and top.
__device__ __forceinline__ float finite_max8(const float (&v)[8], float top) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float a = fabsf(v[e]);
        top = a <= 3.402823466e38f ? fmaxf(top, a) : top;
    }
    return top;
}

struct RowTop { float top; bool plain; };    // the largest finite magnitude of a row; whether all of it is finite
// Of the NV x 8 values a lane, T lanes to the row: part [T / 64] joins the waves of a row, whose sign bits mark the odd ones.
template <int T, int NV> __device__ __forceinline__ RowTop row_top(const float (&v)[NV][8], float* part) {
    RowMax seen;
#pragma unroll
    for (int k = 0; k < NV; ++k) seen.add(v[k]);
    uint64_t odd = __ballot(seen.odd != 0.f);
    if constexpr (T < 64) odd = odd >> (threadIdx.x & 63 & ~(T - 1)) & ((1ull << T) - 1);
    RowTop o{seen.top, odd == 0};
    if (!o.plain) {
        o.top = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) o.top = finite_max8(v[k], o.top);
    }
    o.top = lanes_max<T < 64 ? T : 64>(o.top);
    if constexpr (T > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x % T >> 6] = o.plain ? o.top : -o.top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < T / 64; ++i) {
            o.plain &= __builtin_bit_cast(int, part[i]) >= 0;
            o.top = fmaxf(o.top, fabsf(part[i]));
        }
    }
    return o;
}

// Rows held in 8 bits: q = clamp(round(x / s), -127, 127) with the division one correctly rounded f32
// operation, ties to even; NaN is held as 0, everything as 0 where the scale is 0.
//
// The division by r = RN(1 / s): q0 = x r is within 2 units in the last place, each step q + (x - q s) r (the
// remainder exact) squares that, and after two the quotient is the correctly rounded
// one (Markstein's theorem; s of an all-ones significand excepted).  5 operations instead of about
// 20: 16384 x 4096 f16 37 us, 52-62 with divisions.  Rows with an infinity or a NaN, and scales
// whose remainders might be subnormal, are divided outright.  A finite |x / s| is at most 127 (1 + 2^-23), so that adding
// 1.5 2^23 rounds it to an integer whose byte is the lowest of the sum.
struct RowQuantiser {
    float s, r;
    bool fast;
    __device__ __forceinline__ RowQuantiser(float scale, bool plain) : s(scale) {
        const uint32_t b = __builtin_bit_cast(uint32_t, s);
        fast = plain && s > 1e-25f && s < 1e25f && (b & 0x7FFFFF) != 0x7FFFFF;
        r = fast ? 1.0f / s : 0.f;
    }
    __device__ __forceinline__ int2v operator()(const float (&v)[8]) const {
        int2v w = {};
        if (fast) {
            uint32_t u[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float q = v[e] * r;
                q = fmaf(fmaf(-q, s, v[e]), r, q);
                q = fmaf(fmaf(-q, s, v[e]), r, q);
                u[e] = __builtin_bit_cast(uint32_t, q + 12582912.f);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t a = __builtin_amdgcn_perm(u[4 * h + 1], u[4 * h], 0x0c0c0400u);
                const uint32_t b = __builtin_amdgcn_perm(u[4 * h + 3], u[4 * h + 2], 0x04000c0cu);
                w[h] = (int)(a | b);
            }
            return w;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float q = s != 0.f ? rintf(v[e] / s) : 0.f;
            q = q != q ? 0.f : fminf(fmaxf(q, -127.f), 127.f);
            w[e >> 2] |= (int)((unsigned)((int)q & 0xFF) << (8 * (e & 3)));
        }
        return w;
    }
};
__device__ __forceinline__ void store_bytes8(int8_t* row, int2v w, int i, int d) {
    if (i <= d - 8) {
        *(int2u*)(row + i) = w;
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (i + e < d) row[i + e] = (int8_t)(w[e >> 2] >> (8 * (e & 3)));
}

__device__ __forceinline__ void store_bytes4(int8_t* row, int w, int i, int d) {
    typedef int int1u __attribute__((aligned(1)));
    if (i + 4 <= d) {
        *(int1u*)(row + i) = w;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (i + e < d) row[i + e] = (int8_t)(w >> (8 * e));
}

}  // namespace pkx
