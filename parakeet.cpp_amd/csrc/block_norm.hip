// Norm of a block's output, gate, residual sum and the next block's norm in one
// pass over the row:
//   u = post(y), x' = x + alpha g u, h = pre(x').
// Bytes bound: x, y and the gate are read once, x' and h written once, the row
// stays in registers in between.  8192 x 4090 f32 with a gate row for each (670 MB): 121 us,
// 5.5 TB/s.  2000 x 1024 f16 with an f32 stream (25 MB): 7.6 us, 3.2 TB/s, where a copy of them takes
// 4.1: a row's vectors are asked for one behind the other (each is converted to f32 where it is loaded), and its second norm's weights wait
// for x's stores.
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
template <int T> constexpr int kWaves = T > 64 ? T / 64 : 1;     // of a row

// Sums over the T lanes that share a row.
template <int T> __device__ __forceinline__ Moments row_sum(Moments m, double (&part)[2 * kWaves<T>]) {
    m.s = lanes_sum_f64<T < 64 ? T : 64>(m.s);
    m.t = lanes_sum_f64<T < 64 ? T : 64>(m.t);
    if constexpr (T > 64) {
        const int w = threadIdx.x % T >> 6;
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

// Element e of a lane's k-th eight: eight in a row (RUN) for f16 operands; two pieces of four for f32 ones, each next to the
// neighbouring lanes', so that a store fills whole lines (8192 x 4090: 133 -> 123 us, 8% fewer bytes written; with an f16 operand
// pieces of 8 bytes cost more than that, 2000 x 1024 7.6 and 8.1).
template <int T, int RUN> __device__ __forceinline__ int place(int t, int k, int e) {
    return RUN == 8 ? 8 * (t + k * T) + e : 4 * (t + (2 * k + (e >> 2)) * T) + (e & 3);
}
template <int T, int RUN, typename S> __device__ __forceinline__ void get(float (&v)[8], const S* p, int t, int k, int d) {
    if constexpr (RUN == 8) load_row8(v, p, place<T, 8>(t, k, 0), d);
    else {
        load_row4(v, p, place<T, 4>(t, k, 0), d);
        load_row4(v + 4, p, place<T, 4>(t, k, 4), d);
    }
}
template <int T, int RUN, typename S> __device__ __forceinline__ void put(S* p, const float (&v)[8], int t, int k, int d) {
    if constexpr (RUN == 8) store_row8(p, v, place<T, 8>(t, k, 0), d);
    else {
        store_row4(p, v, place<T, 4>(t, k, 0), d);
        store_row4(p, v + 4, place<T, 4>(t, k, 4), d);
    }
}

// A lane's part of a vector of d, asked for before it is needed.
template <int T, int NV, int RUN> struct Part {
    float v[NV][8];
    bool there = false;
    template <typename S> __device__ __forceinline__ void ask(const S* p, int t, int d) {
        there = p != nullptr;
        if (there)
#pragma unroll
            for (int k = 0; k < NV; ++k) get<T, RUN>(v[k], p, t, k, d);
    }
};

// v becomes its norm: LayerNorm or RMS, times w, plus b (either may be missing).
template <int T, int NV, int RUN>
__device__ __forceinline__ void normalise(float (&v)[NV][8], int kind, const Part<T, NV, RUN>& w, const Part<T, NV, RUN>& b, float eps, float first, int t,
                                          int d, double inv_d, double (&part)[2 * kWaves<T>]) {
    const bool layer = kind == NORM_LAYER;
    Moments m = {0, 0};
    if (layer) {
        const double c = (double)first;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (place<T, RUN>(t, k, 7) >= d)      // what lies past the row's end adds nothing
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (place<T, RUN>(t, k, e) >= d) v[k][e] = first;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double x = (double)v[k][e] - c;
                m.s += x;
                m.t = fma(x, x, m.t);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (place<T, RUN>(t, k, 7) >= d)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (place<T, RUN>(t, k, e) >= d) v[k][e] = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) m.t = fma((double)v[k][e], (double)v[k][e], m.t);
        }
    }
    m = row_sum<T>(m, part);
    const double mu = layer ? m.s * inv_d : 0.0;
    const double var = m.t * inv_d - mu * mu + (double)eps;
    // 1 / sqrt(var): v_rsq_f64 is good to 2^-24 or so, a Newton step squares that
    const double r = __builtin_amdgcn_rsq(var);
    float inv = (float)(r * (1.5 - 0.5 * var * r * r));
    double mean = (double)first + mu;
    // Where v - mean, what f32 leaves of the mean or 1 / sqrt(var) would pass f32's normal numbers the row is taken times a power of
    // two (a deviation below 2^-100 that is not 0 leaves values below 2^-69); the step makes NaN of an infinite variance's root,
    // whose reciprocal is 0.  One test, of the exponent (2000 x 1024 7.62 us; without any 7.51, with
    // three of var 7.67).
    constexpr uint32_t kLow = (1023 - 200) << 20, kHigh = (1023 + 240) << 20;
    if ((uint32_t)(__builtin_bit_cast(uint64_t, var) >> 32) - kLow >= kHigh - kLow) {
        const bool large = var >= 0x1p240;
        const float by = large ? 0.25f : 0x1p100f;
        inv = var < __builtin_inf() ? (float)(r * (1.5 - 0.5 * var * r * r) * (large ? 4 : 0x1p-100)) : (float)r;
        mean *= (double)by;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[k][e] *= by;
    }
    if (layer) {
        const float hi = (float)mean, lo = (float)(mean - hi);     // v - mean exactly where v is near it
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[k][e] = (v[k][e] - hi) - lo;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[k][e] *= inv;
    if (w.there)
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[k][e] *= w.v[k][e];
    if (b.there)
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[k][e] += b.v[k][e];
}

// One row to T lanes: a quarter of a wave up to 128 channels, half of one up to 256, a wave up to 512, two up to 1024, a
// workgroup beyond.
template <typename ET, typename XT, bool I8, int T, int NV, bool EARLY>
__global__ __launch_bounds__(T < 256 ? 256 : T) void block_norm_kernel(BlockNormParams p) {
    constexpr int kRows = T < 256 ? 256 / T : 1, RUN = sizeof(ET) == 2 ? 8 : 4;
    __shared__ double part[kRows][2 * kWaves<T>];
    __shared__ float top_part[kRows][kWaves<T>], x0[kRows];
    const int t = threadIdx.x % T, d = p.d;
    const int mine = kRows == 1 ? 0 : T < 64 ? threadIdx.x / T : __builtin_amdgcn_readfirstlane(threadIdx.x / T);
    const int r = blockIdx.x * kRows + mine;
    if (r >= p.rows) return;                 // all lanes of a row; whole waves where there are barriers, which wait for them no more
    double (&ps)[2 * kWaves<T>] = part[mine];

    // EARLY: everything that the row needs is asked for at once, which is what a few rows wait for (the kernel
    // alone, 1 x 4096 4.5 us, 4.8 with each vector read where it is used); many rows need the registers for more rows at a time
    // (1000 x 4096 13.7 us, early 15.3; 8192 x 4090 f32 121 and 141)
    const XT* xr = p.x ? (const XT*)p.x + r * p.x_row : nullptr;
    const ET* yr = p.y ? (const ET*)p.y + r * p.y_row : nullptr;
    const ET* gr = p.gate ? (const ET*)p.gate + udiv_small(r, p.rows_per_gate) * p.gate_row : nullptr;
    Part<T, NV, RUN> x, y, gate, post_w, post_b, pre_w, pre_b;
    y.ask(yr, t, d);
    const float first_y = p.post == NORM_LAYER ? (float)yr[0] : 0.f;
    x.ask(xr, t, d);
    if (EARLY) {
        gate.ask(gr, t, d);
        post_w.ask(p.post_w, t, d);
        post_b.ask(p.post_b, t, d);
        pre_w.ask(p.pre_w, t, d);
        pre_b.ask(p.pre_b, t, d);
    }
    if (y.there) {
        if (!EARLY) {
            post_w.ask(p.post_w, t, d);
            post_b.ask(p.post_b, t, d);
        }
        if (p.post != NORM_NONE) normalise<T, NV, RUN>(y.v, p.post, post_w, post_b, p.post_eps, first_y, t, d, p.inv_d, ps);
        if (!EARLY) gate.ask(gr, t, d);
        if (gate.there) {
            if (p.sigmoid)
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int e = 0; e < 8; ++e) gate.v[k][e] = 1.0f / (1.0f + expf(-gate.v[k][e]));
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) y.v[k][e] *= gate.v[k][e];
        }
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) x.v[k][e] = x.there ? x.v[k][e] + p.alpha * y.v[k][e] : p.alpha * y.v[k][e];
    }
    // the first element of x', for every lane
    float first = 0.f;
    if (p.pre == NORM_LAYER) {
        if constexpr (T < 64) first = __shfl(x.v[0][0], 0, T);
        else if constexpr (T == 64) first = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x.v[0][0]), 0));
        else {
            if (t == 0) x0[mine] = x.v[0][0];
            __syncthreads();
            first = x0[mine];
        }
    }
    if (p.x_out) {
        XT* o = (XT*)p.x_out + r * p.x_out_row;
#pragma unroll
        for (int k = 0; k < NV; ++k) put<T, RUN>(o, x.v[k], t, k, d);
    }
    if (!p.h) return;
    if (!EARLY) {
        pre_w.ask(p.pre_w, t, d);
        pre_b.ask(p.pre_b, t, d);
    }
    if (p.pre != NORM_NONE) normalise<T, NV, RUN>(x.v, p.pre, pre_w, pre_b, p.pre_eps, first, t, d, p.inv_d, ps);
    if constexpr (I8) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (place<T, RUN>(t, k, e) >= d) x.v[k][e] = 0.f;    // weights and biases are not read there
        const RowTop top = row_top<T, NV>(x.v, top_part[mine]);
        const float s = top.top / 127.0f;
        if (t == 0) p.h_scale[r] = s;
        const RowQuantiser held(s, top.plain);
        int8_t* o = (int8_t*)p.h + r * p.h_row;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int2v q = held(x.v[k]);
            if constexpr (RUN == 8) store_bytes8(o, q, place<T, 8>(t, k, 0), d);
            else {
                store_bytes4(o, q[0], place<T, 4>(t, k, 0), d);
                store_bytes4(o, q[1], place<T, 4>(t, k, 4), d);
            }
        }
    } else {
        ET* o = (ET*)p.h + r * p.h_row;
#pragma unroll
        for (int k = 0; k < NV; ++k) put<T, RUN>(o, x.v[k], t, k, d);
    }
}

template <typename ET, typename XT, bool I8, int T, int NV, bool EARLY> void launch_rows(const BlockNormParams& p, hipStream_t s) {
    constexpr int kRows = T < 256 ? 256 / T : 1;
    launch(block_norm_kernel<ET, XT, I8, T, NV, EARLY>, dim3((unsigned)((p.rows + kRows - 1) / kRows)), dim3(T * kRows), 0, s, p);
}
// Early up to four waves a CU (512 x 1024, one block's two norms: 5.1 and 5.3 us; 2000 x 1024: 9.1 and 8.5).
template <typename ET, typename XT, bool I8, int T, int NV> void launch_width(const BlockNormParams& p, hipStream_t s) {
    constexpr bool fits = NV <= 2;           // the widest rows' weights would not fit the registers
    if (fits && p.rows * T <= 64 * 1024) launch_rows<ET, XT, I8, T, NV, fits>(p, s);
    else launch_rows<ET, XT, I8, T, NV, false>(p, s);
}
// Narrow rows, a head's for instance, share a wave.  Residual and RMS norm of f16 operands, a stream in f16 / in f32: 32000 x 128
// 7.4 / 10.3 us, a wave to each 18.4 / 18.4; 32000 x 256 12.2 / 17.1 and 18.8 / 21.7.
// Wide ones have eight waves (4000 x 8192 f16 113 us, 1000 x 16384 42; 16 waves 143 and 44); up to 4096 channels only while there are
// few rows (1 x 3752 5.7 us, four waves 6.4; 8192 x 4090 f32 133 and 121).
template <typename ET, typename XT, bool I8> void launch_typed(const BlockNormParams& p, hipStream_t s) {
    if (p.d <= 128) launch_width<ET, XT, I8, 16, 1>(p, s);
    else if (p.d <= 256) launch_width<ET, XT, I8, 32, 1>(p, s);
    else if (p.d <= 512) launch_width<ET, XT, I8, 64, 1>(p, s);
    else if (p.d <= 1024) launch_width<ET, XT, I8, 128, 1>(p, s);
    else if (p.d <= 2048) launch_width<ET, XT, I8, 256, 1>(p, s);
    else if (p.d <= 4096) p.rows <= 256 ? launch_width<ET, XT, I8, 512, 1>(p, s) : launch_rows<ET, XT, I8, 256, 2, false>(p, s);     // past four waves a CU
    else if (p.d <= 8192) launch_width<ET, XT, I8, 512, 2>(p, s);
    else launch_width<ET, XT, I8, 512, 4>(p, s);
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
