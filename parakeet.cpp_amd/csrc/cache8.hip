// The 8-bit key/value cache: clearing slots, appending tokens and reading them back.
//
// A block is 32 tokens of one slot and head; its scale is s = max |x| / 127
// over the values appended to it so far, and a value is held as
// clamp(round(x / s), -127, 127) (round to nearest, ties to even).  A new token
// with larger values raises the scale to s' and the block's earlier integers
// become round(q * (s / s')).  Every step is one correctly rounded f32
// operation (no contraction in this file), so the integers are reproducible.
// NaN is held as 0 and an infinity as +-127; neither takes part in the maximum.
#pragma clang fp contract(off)

#include "decoder.hpp"

namespace pkx {
namespace {

__device__ __forceinline__ int2v pack_bytes(const int (&q)[8]) {
    int2v w;
#pragma unroll
    for (int h = 0; h < 2; ++h)
        w[h] = (q[4 * h] & 0xFF) | (q[4 * h + 1] & 0xFF) << 8 | (q[4 * h + 2] & 0xFF) << 16 | (int)((unsigned)q[4 * h + 3] << 24);
    return w;
}
__device__ __forceinline__ int2v quantised(const float (&x)[8], float s) {
    int q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float v = s != 0.f ? rintf(x[e] / s) : 0.f;
        v = v != v ? 0.f : fminf(fmaxf(v, -127.f), 127.f);
        q[e] = (int)v;
    }
    return pack_bytes(q);
}
__device__ __forceinline__ int2v rescaled(int2v old, float ratio) {
    int q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = (int)rintf((float)(int8_t)(old[e >> 2] >> (8 * (e & 3))) * ratio);
    return pack_bytes(q);
}
// eight values from element o on, and the largest of their magnitudes that are finite and of top
template <bool F32> __device__ __forceinline__ float load8(float (&x)[8], const void* base, int64_t o, float top) {
    if constexpr (F32) {
        const float4v a = *(const float4v*)((const float*)base + o), b = *(const float4v*)((const float*)base + o + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) { x[e] = a[e]; x[4 + e] = b[e]; }
    } else {
        const half8v a = *(const half8v*)((const f16*)base + o);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)a[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float a = fabsf(x[e]);
        top = a <= 3.402823466e38f ? fmaxf(top, a) : top;
    }
    return top;
}

// One workgroup per (block of 32 tokens, head, keys or values, row).  Thread t
// holds dimensions [8 (t % n8), +8) of the block's tokens t / n8 + k * (256 / n8),
// n8 = dk / 8: at most 32 values, read once, kept in registers between the
// maximum and the quantisation.  The earlier tokens of a first block are read only
// where its scale rises (read ahead in every call: 4.7 us became 5.0 and 7.1 became
// 8.2).  8 rows x 200 tokens x 8 heads x 64, f32: 5.3 us, 6.6 MB read and 1.6 written:
// latency and a launch.
template <bool F32> __global__ __launch_bounds__(256) void cache8_append_kernel(CacheAppendParams p, int blocks) {
    const int t = threadIdx.x, kh = blockIdx.y, r = udiv_small(blockIdx.x, blocks), bi = blockIdx.x - r * blocks;
    const bool values = blockIdx.z != 0;
    const int start = p.start[r], slot = p.slot ? p.slot[r] : r;
    int n = p.count ? p.count[r] : p.n_new;
    n = n < 0 ? 0 : n > p.n_new ? p.n_new : n;
    if (start < 0 || start >= p.c.cap || (unsigned)slot >= (unsigned)p.c.n_slots) return;
    const int end = n < p.c.cap - start ? start + n : p.c.cap;     // tokens past the capacity are dropped
    const int blk = start / kCacheBlock + bi, t0 = blk * kCacheBlock;
    const int lo = start > t0 ? start : t0, hi = end < t0 + kCacheBlock ? end : t0 + kCacheBlock;
    if (lo >= hi) return;
    __shared__ float part[4];
    __shared__ int taken;
    // of rows that name the same slot the first is appended
    if (p.slot) {
        if (t == 0) taken = 0;
        __syncthreads();
        for (int j = t; j < r; j += 256)
            if (p.slot[j] == slot) taken = 1;
        __syncthreads();
        if (taken) return;
    }
    if (p.table && kh == 0 && !values)
        for (int j = lo + t; j < hi; j += 256) p.table[r * p.table_ld + j] = slot;

    const int dk = p.c.dk, n8 = dk / 8, step = 256 / n8, d = 8 * (t % n8), mine = t / n8;
    const bool on = mine < step;         // 256 is no multiple of n8 for some widths
    const int64_t src = values ? r * p.v_row + kh * p.v_head : r * p.k_row + kh * p.k_head;
    const int64_t tok = values ? p.v_tok : p.k_tok;
    const void* base = values ? p.v : p.k;
    const int64_t head = (int64_t)slot * p.c.Hkv + kh;
    int8_t* dst = (values ? p.c.v : p.c.k) + head * p.c.cap * dk;
    float* sc = (values ? p.c.v_scale : p.c.k_scale) + head * (p.c.cap / kCacheBlock) + blk;

    float x[4][8], top = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int at = t0 + mine + k * step;
        const bool in = on && at >= lo && at < hi;     // tokens past the block are >= hi
#pragma unroll
        for (int e = 0; e < 8; ++e) x[k][e] = 0.f;
        if (in) {
            top = load8<F32>(x[k], base, src + (at - start) * tok + d, top);
        }
    }
    top = wave_max(top);
    if ((t & 63) == 0) part[t >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    const float before = lo > t0 ? *sc : 0.f;          // a block that starts here holds nothing yet
    const float s = fmaxf(before, top / 127.0f);
    const float ratio = s != 0.f ? before / s : 0.f;
    __syncthreads();                                   // every thread has the old scale
    if (t == 0) *sc = s;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int at = t0 + mine + k * step;
        if (!on || at >= hi) continue;
        int8_t* y = dst + (int64_t)at * dk + d;
        if (at >= lo) *(int2v*)y = quantised(x[k], s);
        else if (ratio != 1.0f) *(int2v*)y = rescaled(*(const int2v*)y, ratio);
    }
}

// One new token a row, the step of a decoder: a wave per (row, head, keys or
// values), so that the prologue, which is most of it, runs once.  Every group of
// n8 lanes has the token; where the scale rises the groups share out the block's
// earlier tokens.  128 rows x 8 heads x 64: 4.3 us, on the kernel above 6.7; 1 row 3.7
// and 3.9.
template <bool F32> __global__ __launch_bounds__(256) void cache8_append_one_kernel(CacheAppendParams p, int units) {
    const int unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (unit >= units) return;
    const bool values = unit & 1;
    const int rh = unit >> 1, r = __builtin_amdgcn_readfirstlane(udiv_small(rh, p.c.Hkv)), kh = rh - r * p.c.Hkv;
    const int start = p.start[r], slot = p.slot ? p.slot[r] : r;
    if ((p.count && p.count[r] <= 0) || start < 0 || start >= p.c.cap || (unsigned)slot >= (unsigned)p.c.n_slots) return;
    // of rows that name the same slot the first is appended
    if (p.slot) {
        bool taken = false;
        for (int j = lane; j < r; j += 64) taken |= p.slot[j] == slot;
        if (__ballot(taken)) return;
    }
    if (p.table && kh == 0 && !values && lane == 0) p.table[r * p.table_ld + start] = slot;

    const int dk = p.c.dk, n8 = dk / 8, step = udiv_small(64, n8), mine = udiv_small(lane, n8), d = 8 * (lane - mine * n8);
    const int64_t src = values ? r * p.v_row + kh * p.v_head : r * p.k_row + kh * p.k_head;
    const int64_t head = (int64_t)slot * p.c.Hkv + kh;
    const int blk = start / kCacheBlock, first = blk * kCacheBlock;
    int8_t* dst = (values ? p.c.v : p.c.k) + head * p.c.cap * dk + d;
    float* sc = (values ? p.c.v_scale : p.c.k_scale) + head * (p.c.cap / kCacheBlock) + blk;
    const float before = start > first ? *sc : 0.f;          // a block that starts here holds nothing yet
    float x[8];
    const float top = wave_max(load8<F32>(x, values ? p.v : p.k, src + d, 0.f));
    const float s = fmaxf(before, top / 127.0f);
    const float ratio = s != 0.f ? before / s : 0.f;
    if (lane == 0) *sc = s;
    if (mine == 0) *(int2v*)(dst + (int64_t)start * dk) = quantised(x, s);
    if (ratio == 1.0f || mine >= step) return;               // 64 is no multiple of n8 for some widths
    for (int at = first + mine; at < start; at += 4 * step) {
        int2v old[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) old[k] = *(const int2v*)(dst + (int64_t)(at + k * step < start ? at + k * step : at) * dk);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (at + k * step < start) *(int2v*)(dst + (int64_t)(at + k * step) * dk) = rescaled(old[k], ratio);
    }
}

// The scales of a slot, 8 bytes for 64 x d_head held: a launch and little else, once a sequence.
__global__ __launch_bounds__(256) void cache8_clear_kernel(Cache8 c, const int* slots) {
    const int r = blockIdx.x, slot = slots ? slots[r] : r;
    if ((unsigned)slot >= (unsigned)c.n_slots) return;
    const int64_t n = (int64_t)c.Hkv * (c.cap / kCacheBlock), step = (int64_t)gridDim.y * 256;
    for (int64_t i = (int64_t)blockIdx.y * 256 + threadIdx.x; i < n; i += step) {
        c.k_scale[slot * n + i] = 0.f;
        c.v_scale[slot * n + i] = 0.f;
    }
}

// Eight values of K and V per thread: tokens start[r] .. + n of row r's slot as q * scale.
// Bound by what it writes, 4 bytes a value: 128 rows x 32 tokens x 8 heads x 64, 16.8 MB,
// 7.2 us.
__global__ __launch_bounds__(256) void cache8_read_kernel(CacheReadParams p, int per, int chunks) {
    const int n8 = p.c.dk / 8, r = udiv_small(blockIdx.x, chunks);
    const unsigned in = (blockIdx.x - r * chunks) * 256 + threadIdx.x;
    if (in >= (unsigned)per) return;
    const unsigned hk = in / n8, i = hk / p.c.Hkv;
    const int d = 8 * (in - hk * n8), kh = hk - i * p.c.Hkv;
    const int64_t at = (int64_t)p.start[r] + i, out = ((int64_t)r * per + in) * 8;
    const int slot = p.slot ? p.slot[r] : r;
    const bool live = at >= 0 && at < p.c.cap && (unsigned)slot < (unsigned)p.c.n_slots;
    const int64_t head = live ? (int64_t)slot * p.c.Hkv + kh : 0, tk = live ? at : 0;
    int2v w[2] = {};
    float s[2] = {};
#pragma unroll
    for (int z = 0; z < 2; ++z)
        if (live && (z ? p.v : p.k)) {
            w[z] = *(const int2v*)((z ? p.c.v : p.c.k) + (head * p.c.cap + tk) * p.c.dk + d);
            s[z] = (z ? p.c.v_scale : p.c.k_scale)[head * (p.c.cap / kCacheBlock) + tk / kCacheBlock];
        }
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        float* y = z ? p.v : p.k;
        if (!y) continue;
        float4v a, b;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            a[e] = live ? (float)(int8_t)(w[z][0] >> (8 * e)) * s[z] : 0.f;
            b[e] = live ? (float)(int8_t)(w[z][1] >> (8 * e)) * s[z] : 0.f;
        }
        *(float4v*)(y + out) = a;
        *(float4v*)(y + out + 4) = b;
    }
}

}  // namespace

void launch_cache8_clear(const Cache8& c, int rows, const int* slot, hipStream_t s) {
    if (rows == 0) return;
    const int64_t pieces = ((int64_t)c.Hkv * (c.cap / kCacheBlock) + 1023) / 1024;     // four scales a thread
    launch(cache8_clear_kernel, dim3((unsigned)rows, (unsigned)(pieces < 64 ? pieces : 64)), dim3(256), 0, s, c, slot);
}

void launch_cache8_append(const CacheAppendParams& p, hipStream_t s) {
    if (p.R == 0 || p.n_new == 0) return;
    const int64_t blocks = ((int64_t)p.n_new + kCacheBlock - 2) / kCacheBlock + 1;     // wherever the first token falls in its block
    const int64_t x = p.R * blocks;
    require(x < (1 << 22) && p.c.Hkv <= 65535, "cache append: at most 2^22 blocks of 32 tokens in one call");
    if (p.n_new == 1 && (double)p.R * p.c.Hkv < (double)(1 << 21)) {
        const int units = 2 * p.R * p.c.Hkv;
        launch(p.f32 ? cache8_append_one_kernel<true> : cache8_append_one_kernel<false>, dim3((units + 3) / 4), dim3(256), 0, s, p, units);
        return;
    }
    const dim3 grid((unsigned)x, p.c.Hkv, 2);
    if (p.f32) launch(cache8_append_kernel<true>, grid, dim3(256), 0, s, p, (int)blocks);
    else launch(cache8_append_kernel<false>, grid, dim3(256), 0, s, p, (int)blocks);
}

void launch_cache8_read(const CacheReadParams& p, hipStream_t s) {
    if (p.R == 0 || p.n == 0 || (!p.k && !p.v)) return;
    // (in f64: no product of the sizes that a call may name wraps)
    require((double)p.R * p.n * p.c.Hkv < (double)(1 << 30), "cache read: at most 2^30 rows of d_head values in one call");
    const int64_t per = (int64_t)p.n * p.c.Hkv * (p.c.dk / 8), chunks = (per + 255) / 256;
    require(p.R * chunks < (1 << 22), "cache read: at most 2^33 values in one call");
    launch(cache8_read_kernel, dim3((unsigned)(p.R * chunks)), dim3(256), 0, s, p, (int)per, (int)chunks);
}

}  // namespace pkx
