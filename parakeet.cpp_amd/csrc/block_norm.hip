// Norm of a block's output, gate, residual sum and the next block's norm in one
// pass over the row:
//   u = post(y), x' = x + alpha g u, h = pre(x').
// Bytes bound: x, y and the gate are read once, x' and h written once, the row
// stays in registers in between.
//
// Moments are summed in f64 about the row's first element c: with s = sum (v - c)
// and t = sum (v - c)^2, mean = c + s / d and var = t / d - (s / d)^2.  c belongs
// to the row, so (mean - c)^2 <= d var and the difference loses at most log2(d + 1)
// of 53 bits, whatever the mean; and no f32 square overflows.  One reduction
// gives both moments.  f64 sums run at the rate of f32 ones here and hide behind the
// row's bytes.
#pragma clang fp contract(off)

#include "block.hpp"
#include "rows.hpp"

namespace pkx {
namespace {

struct Moments { double s, t; };

// Sums over the T lanes that share a row.
template <int T> __device__ __forceinline__ Moments row_sum(Moments m, double (&part)[2 * (T / 64)]) {
    m.s = wave_sum_f64(m.s);
    m.t = wave_sum_f64(m.t);
    if constexpr (T > 64) {
        const int w = threadIdx.x >> 6;
        __syncthreads();                     // the last sums have been read
        if ((threadIdx.x & 63) == 0) {
            part[2 * w] = m.s;
            part[2 * w + 1] = m.t;
        }
        __syncthreads();
        m = {0, 0};
#pragma unroll
        for (int i = 0; i < T / 64; ++i) {
            m.s += part[2 * i];
            m.t += part[2 * i + 1];
        }
    }
    return m;
}

// v becomes its norm: LayerNorm or RMS, times w, plus b (either may be missing).
template <int T, int NV>
__device__ __forceinline__ void normalise(float (&v)[NV][8], int kind, const float* w, const float* b, float eps, float first, int t,
                                          int d, double inv_d, double (&part)[2 * (T / 64)]) {
    const bool layer = kind == NORM_LAYER;
    const double c = layer ? (double)first : 0.0;
    Moments m = {0, 0};
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int i = 8 * (t + k * T) + e;
            const double x = i < d ? (double)v[k][e] - c : 0.0;
            m.s += x;
            m.t = fma(x, x, m.t);
        }
    m = row_sum<T>(m, part);
    const double mu = layer ? m.s * inv_d : 0.0;
    const double var = m.t * inv_d - mu * mu + (double)eps;
    // 1 / sqrt(var): v_rsq_f64 is good to 2^-24 or so, a Newton step squares that
    double r = __builtin_amdgcn_rsq(var);
    r = r * (1.5 - 0.5 * var * r * r);
    const float inv = (float)r;
    const double mean = c + mu;
    const float hi = (float)mean, lo = (float)(mean - hi);     // v - mean exactly where v is near it
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int i = 8 * (t + k * T);
        if (i >= d) continue;
        float ww[8], bb[8];
        if (w) load_row8(ww, w, i, d);
        if (b) load_row8(bb, b, i, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float x = layer ? (v[k][e] - hi) - lo : v[k][e];
            x *= inv;
            if (w) x *= ww[e];
            if (b) x += bb[e];
            v[k][e] = x;
        }
    }
}

// One row to T lanes: a wave up to 2048 channels, a workgroup beyond.
template <typename ET, typename XT, bool I8, int T, int NV>
__global__ __launch_bounds__(T < 256 ? 256 : T) void block_norm_kernel(BlockNormParams p) {
    constexpr int kRows = T < 256 ? 256 / T : 1;
    __shared__ double part[kRows][2 * (T / 64)];
    __shared__ float top_part[T / 64];
    const int t = threadIdx.x % T, d = p.d;
    const int mine = kRows > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / T) : 0;
    const int64_t r = (int64_t)blockIdx.x * kRows + mine;
    if (r >= p.rows) return;                 // whole waves; T > 64 has one row to a workgroup
    double (&ps)[2 * (T / 64)] = part[mine];

    const XT* xr = (const XT*)p.x + r * p.x_row;
    const ET* yr = (const ET*)p.y + r * p.y_row;
    float x[NV][8], y[NV][8];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int i = 8 * (t + k * T);
        if (p.x) load_row8(x[k], xr, i, d);
        if (p.y) load_row8(y[k], yr, i, d);
    }
    if (p.y) {
        if (p.post != NORM_NONE) normalise<T, NV>(y, p.post, p.post_w, p.post_b, p.post_eps, (float)yr[0], t, d, p.inv_d, ps);
        const ET* gr = (const ET*)p.gate + (p.gate ? (r / p.rows_per_gate) * p.gate_row : 0);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int i = 8 * (t + k * T);
            if (p.gate) {
                float g[8];
                load_row8(g, gr, i, d);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (p.sigmoid) g[e] = 1.0f / (1.0f + expf(-g[e]));
                    y[k][e] *= g[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) x[k][e] = p.x ? x[k][e] + p.alpha * y[k][e] : p.alpha * y[k][e];
        }
    }
    // the first element of x', for every lane
    float first = 0.f;
    if (p.pre == NORM_LAYER) {
        if constexpr (T == 64) first = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x[0][0]), 0));
        else {
            __shared__ float x0;
            if (t == 0) x0 = x[0][0];
            __syncthreads();
            first = x0;
        }
    }
    if (p.x_out) {
        XT* o = (XT*)p.x_out + r * p.x_out_row;
#pragma unroll
        for (int k = 0; k < NV; ++k) store_row8(o, x[k], 8 * (t + k * T), d);
    }
    if (!p.h) return;
    if (p.pre != NORM_NONE) normalise<T, NV>(x, p.pre, p.pre_w, p.pre_b, p.pre_eps, first, t, d, p.inv_d, ps);
    if constexpr (I8) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (8 * (t + k * T) + e >= d) x[k][e] = 0.f;    // weights and biases are not read there
        const RowTop top = row_top<T, NV>(x, top_part);
        const float s = top.top / 127.0f;
        if (t == 0) p.h_scale[r] = s;
        const RowQuantiser held(s, top.plain);
        int8_t* o = (int8_t*)p.h + r * p.h_row;
#pragma unroll
        for (int k = 0; k < NV; ++k) store_bytes8(o, held(x[k]), 8 * (t + k * T), d);
    } else {
        ET* o = (ET*)p.h + r * p.h_row;
#pragma unroll
        for (int k = 0; k < NV; ++k) store_row8(o, x[k], 8 * (t + k * T), d);
    }
}

template <typename ET, typename XT, bool I8> void launch_typed(const BlockNormParams& p, hipStream_t s) {
    const unsigned rows = (unsigned)p.rows;
    if (p.d <= 512) launch(block_norm_kernel<ET, XT, I8, 64, 1>, dim3((rows + 3) / 4), dim3(256), 0, s, p);
    else if (p.d <= 1024) launch(block_norm_kernel<ET, XT, I8, 64, 2>, dim3((rows + 3) / 4), dim3(256), 0, s, p);
    else if (p.d <= 2048) launch(block_norm_kernel<ET, XT, I8, 256, 1>, dim3(rows), dim3(256), 0, s, p);
    else if (p.d <= 4096) launch(block_norm_kernel<ET, XT, I8, 256, 2>, dim3(rows), dim3(256), 0, s, p);
    else if (p.d <= 8192) launch(block_norm_kernel<ET, XT, I8, 1024, 1>, dim3(rows), dim3(1024), 0, s, p);
    else launch(block_norm_kernel<ET, XT, I8, 1024, 2>, dim3(rows), dim3(1024), 0, s, p);
}

}  // namespace

void launch_block_norm(BlockNormParams p, hipStream_t s) {
    if (p.rows == 0) return;
    p.inv_d = 1.0 / p.d;
    if (p.f32) p.h_i8 ? launch_typed<float, float, true>(p, s) : launch_typed<float, float, false>(p, s);
    else if (p.x_f32) p.h_i8 ? launch_typed<f16, float, true>(p, s) : launch_typed<f16, float, false>(p, s);
    else p.h_i8 ? launch_typed<f16, f16, true>(p, s) : launch_typed<f16, f16, false>(p, s);
}

}  // namespace pkx
