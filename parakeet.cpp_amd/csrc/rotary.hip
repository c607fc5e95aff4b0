// Rotary positions: the pair (a, b) of frequency f at position p becomes
//   (a cos t - b sin t, b cos t + a sin t) mult,  t = p f,
// with pairs of neighbours (2 j, 2 j + 1) or of the halves (j, j + rot / 2) of the first
// rot dimensions; the others stay as they are.
// Bytes bound: every element is read and written once.
#pragma clang fp contract(off)

#include "block.hpp"
#include "rows.hpp"

namespace pkx {
namespace {

// cos and sin of 2 pi x: x reduced in f64 to the nearest quarter turn, where the
// remainder u (at most an eighth of a turn) loses nothing but its rounding to f32, then the
// Taylor series of both about 0 in v = 2 pi u: their first terms left out are
// below 2 10^-9 (sine, relative) and 5 10^-10 (cosine).
__device__ __forceinline__ float2v cos_sin_turns(double x) {
    const double q = rint(4.0 * x);
    const float v = (float)((x - 0.25 * q) * 6.283185307179586476925);
    const float z = v * v;
    float s = 2.7557319e-6f;
    s = fmaf(s, z, -1.98412698e-4f);
    s = fmaf(s, z, 8.33333333e-3f);
    s = fmaf(s, z, -1.66666667e-1f);
    s = fmaf(s * z, v, v);
    float c = -2.7557319e-7f;
    c = fmaf(c, z, 2.48015873e-5f);
    c = fmaf(c, z, -1.38888889e-3f);
    c = fmaf(c, z, 4.16666667e-2f);
    c = fmaf(c, z, -0.5f);
    c = fmaf(c, z, 1.0f);
    const int k = (int)(q - 4.0 * floor(0.25 * q));            // quarter turns, 0..3
    const float a = k & 1 ? s : c, b = k & 1 ? c : s;
    return float2v{(k == 1 || k == 2) ? -a : a, k >= 2 ? -b : b};
}

// One workgroup per TOK tokens of a row: their angles once into LDS, then all heads.
// An item is up to eight pairs of a head, or eight of its other dimensions.
template <typename ET, int TOK> __global__ __launch_bounds__(256) void rotary_kernel(RotaryParams p, int groups) {
    extern __shared__ float2v turn[];        // [TOK][rot / 2]
    const int r = udiv_small(blockIdx.x, groups), i0 = (blockIdx.x - r * groups) * TOK;
    int n = p.count ? p.count[r] : p.n;
    n = n > p.n ? p.n : n;
    if (i0 >= n) return;
    const int toks = n - i0 < TOK ? n - i0 : TOK, pairs = p.rot / 2;
    const int64_t first = p.start ? p.start[r] : 0;
    for (int j = threadIdx.x; j < toks * pairs; j += 256) {
        const int i = udiv_small(j, pairs), f = j - i * pairs;
        const int64_t at = p.pos ? p.pos[r * p.pos_row + i0 + i] : first + i0 + i;
        const float2v cs = cos_sin_turns((double)at * p.freq[f] * 0.159154943091895335769);
        turn[j] = float2v{cs[0] * p.mult, cs[1] * p.mult};
    }
    __syncthreads();
    const int turned = (pairs + 7) / 8, rest = p.dk - p.rot, items = turned + (rest + 7) / 8;
    for (int z = 0; z < p.parts; ++z) {
        const RotaryPart& a = p.part[z];
        const bool copy = a.src != a.dst;
        const int per = a.heads * items, all = toks * per;
        for (int j = threadIdx.x; j < all; j += 256) {
            const int i = udiv_small(j, per), hi = j - i * per, h = udiv_small(hi, items), it = hi - h * items;
            const ET* src = (const ET*)a.src + r * a.s_row + (int64_t)(i0 + i) * a.s_tok + h * a.s_head;
            ET* dst = (ET*)a.dst + r * a.d_row + (int64_t)(i0 + i) * a.d_tok + h * a.d_head;
            if (it >= turned) {
                if (!copy) continue;
                float v[8];
                load_row8(v, src + p.rot, 8 * (it - turned), rest);
                store_row8(dst + p.rot, v, 8 * (it - turned), rest);
                continue;
            }
            const int f = 8 * it;
            float u[8], v[8], x[8], y[8];
            if (p.interleaved) {             // pairs f .. f + 8: elements 2 f .. 2 f + 16
                load_row8(u, src, 2 * f, p.rot);
                load_row8(v, src, 2 * f + 8, p.rot);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = u[2 * e]; y[e] = u[2 * e + 1];
                    x[4 + e] = v[2 * e]; y[4 + e] = v[2 * e + 1];
                }
            } else {
                load_row8(x, src, f, pairs);
                load_row8(y, src + pairs, f, pairs);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float2v cs = f + e < pairs ? turn[i * pairs + f + e] : float2v{0.f, 0.f};
                const float s = x[e] * cs[0] - y[e] * cs[1], t = y[e] * cs[0] + x[e] * cs[1];
                x[e] = s;
                y[e] = t;
            }
            if (p.interleaved) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    u[2 * e] = x[e]; u[2 * e + 1] = y[e];
                    v[2 * e] = x[4 + e]; v[2 * e + 1] = y[4 + e];
                }
                store_row8(dst, u, 2 * f, p.rot);
                store_row8(dst, v, 2 * f + 8, p.rot);
            } else {
                store_row8(dst, x, f, pairs);
                store_row8(dst + pairs, y, f, pairs);
            }
        }
    }
}

}  // namespace

void launch_rotary(const RotaryParams& p, hipStream_t s) {
    if (p.R == 0 || p.n == 0 || p.parts == 0) return;
    constexpr int kTok = 4;
    const int groups = p.n == 1 ? 1 : cdiv(p.n, kTok);
    require((double)p.R * groups < (double)(1 << 22), "rotary: too many tokens for one call");
    if (p.n == 1) launch(p.f32 ? rotary_kernel<float, 1> : rotary_kernel<f16, 1>, dim3(p.R), dim3(256), p.rot / 2 * 8, s, p, 1);
    else launch(p.f32 ? rotary_kernel<float, kTok> : rotary_kernel<f16, kTok>, dim3(p.R * groups), dim3(256), kTok * p.rot / 2 * 8, s, p, groups);
}

}  // namespace pkx
