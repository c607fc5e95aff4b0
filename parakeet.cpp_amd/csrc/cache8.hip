// The 8-bit key/value cache: appending tokens and reading them back.
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

// One workgroup per (block of 32 tokens, head, keys or values, row).  Thread t
// holds dimensions [8 (t % n8), +8) of the block's tokens t / n8 + k * (256 / n8),
// n8 = dk / 8: at most 32 values, read once, kept in registers between the
// maximum and the quantisation.
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
            const int64_t o = src + (at - start) * tok + d;
            if constexpr (F32) {
                const float4v a = *(const float4v*)((const float*)base + o), b = *(const float4v*)((const float*)base + o + 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) { x[k][e] = a[e]; x[k][4 + e] = b[e]; }
            } else {
                const half8v a = *(const half8v*)((const f16*)base + o);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[k][e] = (float)a[e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float a = fabsf(x[k][e]);
                top = a <= 3.402823466e38f ? fmaxf(top, a) : top;
            }
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
        int q[8];
        if (at >= lo) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float v = s != 0.f ? rintf(x[k][e] / s) : 0.f;
                v = v != v ? 0.f : fminf(fmaxf(v, -127.f), 127.f);
                q[e] = (int)v;
            }
        } else {
            if (ratio == 1.0f) continue;
            const int2v old = *(const int2v*)y;
#pragma unroll
            for (int e = 0; e < 8; ++e) q[e] = (int)rintf((float)(int8_t)(old[e >> 2] >> (8 * (e & 3))) * ratio);
        }
        int2v w;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            w[h] = (q[4 * h] & 0xFF) | (q[4 * h + 1] & 0xFF) << 8 | (q[4 * h + 2] & 0xFF) << 16 | (int)((unsigned)q[4 * h + 3] << 24);
        *(int2v*)y = w;
    }
}

// Eight values of K and V per thread: tokens start[r] .. + n of row r's slot as q * scale.
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

void launch_cache8_append(const CacheAppendParams& p, hipStream_t s) {
    if (p.R == 0 || p.n_new == 0) return;
    const int64_t blocks = ((int64_t)p.n_new + kCacheBlock - 2) / kCacheBlock + 1;     // wherever the first token falls in its block
    const int64_t x = p.R * blocks;
    require(x < (1 << 22) && p.c.Hkv <= 65535, "cache append: at most 2^22 blocks of 32 tokens in one call");
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
