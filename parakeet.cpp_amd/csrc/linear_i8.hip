// Products of 8-bit tokens and 8-bit weights, a scale for each token and each
// output channel:
//   y[m][n] = add[m][n] + alpha act(xs[m] ws[n] sum_k x[m][k] w[n][k] + bias[n]).
// Sums are exact in i32 (K up to 2^17: 127 * 127 * 2^17 < 2^31); everything after them is f32.
//
// The weights are the A operand of the matrix instructions and the tokens the B
// operand, so that a lane ends with one token and consecutive channels.  Their
// layout (block.hpp) is that of the fragments: a wave's load is 1 KB in a row.
// Slot i of a block's 32 holds channel tail_col(i), which leaves a lane of the
// 32 x 32 form with 16 consecutive channels and one of the 16 x 16 form with 4.
#include "block.hpp"
#include "rows.hpp"

namespace pkx {
namespace {

typedef int int16v __attribute__((ext_vector_type(16)));

// ---- quantising rows -------------------------------------------------------
// s = max |x| / 127 over the finite values, x held as clamp(round(x / s), -127, 127), each step one f32 operation.
// A row is read once and kept in registers up to 8 T NV values; longer rows are read twice.
template <typename ET, int T, int NV> __global__ __launch_bounds__(T < 256 ? 256 : T) void quantize_rows_kernel(QuantizeRowsParams p) {
    constexpr int kRows = T < 256 ? 256 / T : 1;
    __shared__ float part[T / 64];
    const int t = threadIdx.x % T, d = p.d;
    const int64_t r = (int64_t)blockIdx.x * kRows + (kRows > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / T) : 0);
    if (r >= p.rows) return;
    const ET* x = (const ET*)p.x + r * p.x_row;
    float v[NV][8], top = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        load_row8(v[k], x, 8 * (t + k * T), d);
        top = finite_max8(v[k], top);
    }
    for (int i = 8 * (t + NV * T); i < d; i += 8 * T) {
        float w[8];
        load_row8(w, x, i, d);
        top = finite_max8(w, top);
    }
    top = wave_max_full(top);
    if constexpr (T > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < T / 64; ++i) top = fmaxf(top, part[i]);
    }
    const float s = top / 127.0f;
    if (t == 0) p.scale[r] = s;
    int8_t* q = p.q + r * p.q_row;
#pragma unroll
    for (int k = 0; k < NV; ++k) store_bytes8(q, quantised8(v[k], s), 8 * (t + k * T), d);
    for (int i = 8 * (t + NV * T); i < d; i += 8 * T) {
        float w[8];
        load_row8(w, x, i, d);
        store_bytes8(q, quantised8(w, s), i, d);
    }
}

template <typename ET> void launch_quantize_typed(const QuantizeRowsParams& p, hipStream_t s) {
    const unsigned rows = (unsigned)p.rows;
    if (p.d <= 512) launch(quantize_rows_kernel<ET, 64, 1>, dim3((rows + 3) / 4), dim3(256), 0, s, p);
    else if (p.d <= 2048) launch(quantize_rows_kernel<ET, 256, 1>, dim3(rows), dim3(256), 0, s, p);
    else if (p.d <= 4096) launch(quantize_rows_kernel<ET, 256, 2>, dim3(rows), dim3(256), 0, s, p);
    else launch(quantize_rows_kernel<ET, 1024, 2>, dim3(rows), dim3(1024), 0, s, p);
}

// ---- weights ---------------------------------------------------------------
// A thread per 16 bytes of the layout.
__global__ __launch_bounds__(256) void i8_pack_kernel(const int8_t* w, int64_t w_row, int N, int K, int kblocks, int64_t pieces, int8_t* out) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= pieces) return;
    const int slot = (int)(at & 31), group = (int)(at >> 5 & 3);
    const int64_t block = at >> 7;
    const int nb = (int)(block / kblocks), kb = (int)(block - (int64_t)nb * kblocks);
    const int n = nb * kI8ColBlock + tail_col(slot), k0 = kb * kI8DepthBlock + 16 * group;
    int4v v = {};
    for (int e = 0; e < 16; ++e)
        if (n < N && k0 + e < K) v[e >> 2] |= (int)((unsigned)(w[n * w_row + k0 + e] & 0xFF) << (8 * (e & 3)));
    *(int4v*)(out + at * 16) = v;
}

// ---- epilogue --------------------------------------------------------------
// CNT channels from n0 on of token m.
template <typename YT, int CNT>
__device__ __forceinline__ void finish(const LinearI8Params& p, const int* acc, int m, int n0, float xs) {
    const int64_t row = (int64_t)m;
    YT* y = (YT*)p.y + row * p.y_row + n0;
    const YT* add = p.add ? (const YT*)p.add + row * p.add_row + n0 : nullptr;
    typedef YT vec __attribute__((ext_vector_type(CNT)));
    typedef vec vecu __attribute__((aligned(sizeof(YT))));
    typedef float fvec __attribute__((ext_vector_type(CNT)));
    typedef fvec fvecu __attribute__((aligned(4)));
    if (n0 + CNT <= p.N) {
        const fvec ws = *(const fvecu*)(p.w_scale + n0);
        fvec b = {};
        if (p.bias) b = *(const fvecu*)(p.bias + n0);
        vec a = {};
        if (add) a = *(const vecu*)add;
        vec o;
#pragma unroll
        for (int e = 0; e < CNT; ++e) {
            float v = (float)acc[e] * (xs * ws[e]);
            if (p.bias) v += b[e];
            if (p.silu) v = v / (1.0f + expf(-v));
            v *= p.alpha;
            if (add) v += (float)a[e];
            o[e] = (YT)v;
        }
        *(vecu*)y = o;
        return;
    }
#pragma unroll
    for (int e = 0; e < CNT; ++e) {
        if (n0 + e >= p.N) break;
        float v = (float)acc[e] * (xs * p.w_scale[n0 + e]);
        if (p.bias) v += p.bias[n0 + e];
        if (p.silu) v = v / (1.0f + expf(-v));
        v *= p.alpha;
        if (add) v += (float)add[e];
        y[e] = (YT)v;
    }
}

// ---- few tokens ------------------------------------------------------------
// 16 channels x 16 MT tokens to a workgroup, K shared out over its waves block by
// block (a wave reads 1 KB of weights and MT KB of tokens per step, straight into
// the fragments) and the partial sums joined through LDS.
template <typename YT, int MT, int W> __global__ __launch_bounds__(W * 64) void i8_rows_kernel(LinearI8Params p, int mtiles) {
    __shared__ int4v part[W][MT][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int unit = blockIdx.x, nh = udiv_small(unit, mtiles), m0 = (unit - nh * mtiles) * 16 * MT;
    const int kblocks = (p.K + kI8DepthPad - 1) / kI8DepthPad * (kI8DepthPad / kI8DepthBlock);
    const int8_t* wp = (const int8_t*)p.w + (int64_t)(nh >> 1) * kblocks * 2048;
    const __amdgpu_buffer_rsrc_t rw = make_rsrc(wp, (int64_t)kblocks * 2048);
    const int k16 = (p.K + 15) & ~15, rows = p.M - m0 < 16 * MT ? p.M - m0 : 16 * MT;
    const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.x + (int64_t)m0 * p.x_row, (int64_t)(rows - 1) * p.x_row + k16);
    const uint32_t wo = ((lane >> 4) * 32 + 16 * (nh & 1) + (lane & 15)) * 16;
    const uint32_t xo = (uint32_t)((lane & 15) * p.x_row + 16 * (lane >> 4));
    int4v acc[MT] = {};
    for (int kb = w; kb < kblocks; kb += W) {
        const int4v a = __builtin_amdgcn_raw_buffer_load_b128(rw, wo, kb * 2048, 0);
        int4v b[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) b[i] = __builtin_amdgcn_raw_buffer_load_b128(rx, xo + (uint32_t)(16 * i * p.x_row) + kb * 64, 0, 0);
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b[i], acc[i], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) part[w][i][lane] = acc[i];
    __syncthreads();
    for (int i = w; i < MT; i += W) {
        int4v s = part[0][i][lane];
#pragma unroll
        for (int j = 1; j < W; ++j) s += part[j][i][lane];
        const int m = m0 + 16 * i + (lane & 15), g = lane >> 4, h = nh & 1;
        // slots 16 h + 4 g + r of the block are these four channels
        const int n0 = (nh >> 1) * kI8ColBlock + 16 * (g & 1) + 4 * (2 * h + (g >> 1));
        if (m < p.M && n0 < p.N) finish<YT, 4>(p, (const int*)&s, m, n0, p.x_scale[m]);
    }
}

// ---- many tokens -----------------------------------------------------------
// WM x WN waves of TM x TN tiles of 32 tokens x 32 channels.  Tokens go through
// LDS (rows of 128 bytes, their 16-byte pieces permuted by the row so that the
// reads of a tile fall into different banks), weights straight into the fragments.
template <typename YT, int WM, int WN, int TM, int TN>
__global__ __launch_bounds__(WM * WN * 64) void i8_tile_kernel(LinearI8Params p, int mtiles, int ntiles) {
    constexpr int W = WM * WN, BM = 32 * WM * TM, BN = 32 * WN * TN, ROWS = BM / 8 / W;   // DMA instructions of a wave per slab
    static_assert(BM / 8 % W == 0, "rows of a slab go evenly over the waves");
    __shared__ __align__(16) uint8_t slab[2][BM * 128];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wid % WM, wn = wid / WM;
    const int tile = xcd_tile(blockIdx.x, mtiles * ntiles);
    const int tn = tile / mtiles, m0 = (tile - tn * mtiles) * BM, n0 = tn * BN;
    const int slabs = (p.K + kI8DepthPad - 1) / kI8DepthPad, kblocks = 2 * slabs;
    const int k16 = (p.K + 15) & ~15, rows = p.M - m0 < BM ? p.M - m0 : BM;
    const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.x + (int64_t)m0 * p.x_row, (int64_t)(rows - 1) * p.x_row + k16);
    const int nblocks = (p.N + 31) / 32, b0 = n0 / 32, nb = nblocks - b0 < BN / 32 ? nblocks - b0 : BN / 32;
    const __amdgpu_buffer_rsrc_t rw = make_rsrc((const int8_t*)p.w + (int64_t)b0 * kblocks * 2048, (int64_t)nb * kblocks * 2048);

    uint32_t xo[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = (wid * ROWS + i) * 8 + (lane >> 3);
        xo[i] = (uint32_t)(r * p.x_row + 16 * ((lane & 7) ^ (r & 7)));
    }
    uint32_t wo[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) wo[j] = (uint32_t)((wn * TN + j) * kblocks * 2048 + lane * 16);
    const uint8_t* arow[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) arow[b] = slab[b] + (wm * TM * 32 + (lane & 31)) * 128;
    const int half = lane >> 5, sw = lane & 7;

    int16v acc[TM][TN] = {};
    int4v wf[2][4][TN];
    auto fetch = [&](int k, int b) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) lds_dma16(rx, slab[b] + (wid * ROWS + i) * 1024, xo[i], k * 128);
    };
    auto fetch_w = [&](int k, int4v (&f)[4][TN]) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int j = 0; j < TN; ++j) f[q][j] = __builtin_amdgcn_raw_buffer_load_b128(rw, wo[j] + q * 1024, k * 4096, 0);
    };
    auto step = [&](int k, int b) {
        wait_vmcnt<0>();
        __syncthreads();
        if (k + 1 < slabs) {
            fetch(k + 1, b ^ 1);
            fetch_w(k + 1, wf[b ^ 1]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            int4v xf[TM];
#pragma unroll
            for (int i = 0; i < TM; ++i) xf[i] = *(const int4v*)(arow[b] + i * 32 * 128 + 16 * ((2 * q + half) ^ sw));
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[b][q][j], xf[i], acc[i][j], 0, 0, 0);
        }
    };
    fetch(0, 0);
    fetch_w(0, wf[0]);
    int k = 0;
    for (; k + 1 < slabs; k += 2) {
        step(k, 0);
        step(k + 1, 1);
    }
    if (k < slabs) step(k, 0);

#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int m = m0 + (wm * TM + i) * 32 + (lane & 31);
        if (m >= p.M) continue;
        const float xs = p.x_scale[m];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int n = n0 + (wn * TN + j) * 32 + 16 * half;
            if (n < p.N) finish<YT, 16>(p, (const int*)&acc[i][j], m, n, xs);
        }
    }
}

template <typename YT> void launch_typed(const LinearI8Params& p, hipStream_t s) {
    if (p.M <= 64) {
        const int mt = p.M <= 16 ? 1 : 2, mtiles = cdiv(p.M, 16 * mt), units = 2 * cdiv(p.N, 32) * mtiles;
        if (mt == 1) launch(i8_rows_kernel<YT, 1, 8>, dim3(units), dim3(512), 0, s, p, mtiles);
        else launch(i8_rows_kernel<YT, 2, 8>, dim3(units), dim3(512), 0, s, p, mtiles);
        return;
    }
    if ((int64_t)cdiv(p.M, 256) * cdiv(p.N, 256) >= 200) {
        const int mt = cdiv(p.M, 256), nt = cdiv(p.N, 256);
        launch(i8_tile_kernel<YT, 2, 4, 4, 2>, dim3(mt * nt), dim3(512), 0, s, p, mt, nt);
        return;
    }
    const int mt = cdiv(p.M, 128), nt = cdiv(p.N, 128);
    launch(i8_tile_kernel<YT, 2, 2, 2, 2>, dim3(mt * nt), dim3(256), 0, s, p, mt, nt);
}

}  // namespace

void launch_quantize_rows(const QuantizeRowsParams& p, hipStream_t s) {
    if (p.rows == 0) return;
    p.f32 ? launch_quantize_typed<float>(p, s) : launch_quantize_typed<f16>(p, s);
}
void launch_i8_weight_pack(const int8_t* w, int64_t w_row, int N, int K, void* packed, hipStream_t s) {
    const int64_t pieces = i8_weight_bytes(N, K) / 16;
    if (pieces == 0) return;
    const int kblocks = (K + kI8DepthPad - 1) / kI8DepthPad * (kI8DepthPad / kI8DepthBlock);
    launch(i8_pack_kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, s, w, w_row, N, K, kblocks, pieces, (int8_t*)packed);
}
void launch_linear_i8(const LinearI8Params& p, hipStream_t s) {
    if (p.M == 0 || p.N == 0) return;
    p.y_f32 ? launch_typed<float>(p, s) : launch_typed<f16>(p, s);
}

}  // namespace pkx
