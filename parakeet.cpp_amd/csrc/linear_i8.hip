// Products of 8-bit tokens and 8-bit weights, a scale for each token and each
// output channel:
//   y[m][n] = add[m][n] + alpha act(xs[m] ws[n] sum_k x[m][k] w[n][k] + bias[n]).
// Sums are exact in i32 (128 * 128 * K < 2^31 for K below 2^17); everything after them is f32.
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
// A row is read once and kept in registers up to 8 T NV values; longer rows are read twice, counted in 64 bits (a lane's last step may end past
// 2^31).  16384 x 4096 f16 (201 MB): 37 us,
// 5.4 TB/s.
template <typename ET, int T, int NV> __global__ __launch_bounds__(T < 256 ? 256 : T) void quantize_rows_kernel(QuantizeRowsParams p) {
    constexpr int kRows = T < 256 ? 256 / T : 1;
    __shared__ float part[kRows][T / 64], more[T / 64];
    const int t = threadIdx.x % T, d = p.d;
    const int mine = kRows > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / T) : 0;
    const int64_t r = (int64_t)blockIdx.x * kRows + mine;
    if (r >= p.rows) return;
    const ET* x = (const ET*)p.x + r * p.x_row;
    float v[NV][8];
#pragma unroll
    for (int k = 0; k < NV; ++k) load_row8(v[k], x, 8 * (t + k * T), d);
    RowTop top = row_top<T, NV>(v, part[mine]);
    const bool longer = d > 8 * T * NV;
    if (longer) {                            // only the longest rows' kernel: T > 64
        float w[1][8] = {}, m = 0.f;
        bool plain = true;
        for (int64_t i = 8 * (t + NV * T); i < d; i += 8 * T) {
            RowMax seen;
            load_row8(w[0], x, (int)i, d);
            seen.add(w[0]);
            plain &= seen.odd == 0.f;
            m = finite_max8(w[0], m);
        }
        w[0][0] = m;
#pragma unroll
        for (int e = 1; e < 8; ++e) w[0][e] = 0.f;
        const RowTop rest = row_top<T, 1>(w, more);
        top.top = fmaxf(top.top, rest.top);
        top.plain &= __syncthreads_and(plain);
    }
    const float s = top.top / 127.0f;
    if (t == 0) p.scale[r] = s;
    const RowQuantiser held(s, top.plain);
    int8_t* q = p.q + r * p.q_row;
#pragma unroll
    for (int k = 0; k < NV; ++k) store_bytes8(q, held(v[k]), 8 * (t + k * T), d);
    if (longer)
        for (int64_t i = 8 * (t + NV * T); i < d; i += 8 * T) {
            float w[8];
            load_row8(w, x, (int)i, d);
            store_bytes8(q, held(w), (int)i, d);
        }
}

// 4000 x 8192 f16 on 8 waves a row 16.7 us, on 16 25.6; 100 x 50000 11.8 and 9.4.
template <typename ET> void launch_quantize_typed(const QuantizeRowsParams& p, hipStream_t s) {
    const unsigned rows = (unsigned)p.rows;
    if (p.d <= 512) launch(quantize_rows_kernel<ET, 64, 1>, dim3((rows + 3) / 4), dim3(256), 0, s, p);
    else if (p.d <= 1024) launch(quantize_rows_kernel<ET, 128, 1>, dim3((rows + 1) / 2), dim3(256), 0, s, p);
    else if (p.d <= 2048) launch(quantize_rows_kernel<ET, 256, 1>, dim3(rows), dim3(256), 0, s, p);
    else if (p.d <= 4096) launch(quantize_rows_kernel<ET, 256, 2>, dim3(rows), dim3(256), 0, s, p);
    else if (p.d <= 8192) launch(quantize_rows_kernel<ET, 512, 2>, dim3(rows), dim3(512), 0, s, p);
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
    typedef int4v int4u __attribute__((aligned(1)));
    if (n < N && k0 + 16 <= K) v = *(const int4u*)(w + n * w_row + k0);
    else
        for (int e = 0; e < 16; ++e)
            if (n < N && k0 + e < K) v[e >> 2] |= (int)((unsigned)(w[n * w_row + k0 + e] & 0xFF) << (8 * (e & 3)));
    *(int4v*)(out + at * 16) = v;
}

// ---- epilogue --------------------------------------------------------------
// v / (1 + e^-v).  e^-v as 2^t (1 + r ln 2) with t = -v log2 e in f32 and r what its rounding left; the
// reciprocal of 1 + e^-v to half a step by a Newton step.  About 10 instructions where expf
// and a division take 35.
// An f16 result takes the bare exponential and reciprocal (|v| 2^-23 relative, far below its 2^-11):
// 2000 x 4096 outputs 1.2 us less.
template <typename YT> __device__ __forceinline__ float silu_of(float v) {
#pragma clang fp contract(off)               // t - 64 of the rounded t
    if constexpr (sizeof(YT) == 2) return silu_dev(v);
    const float t = v * -1.4426950408889634f;
    const float r = fmaf(v, -1.925963033500e-8f, fmaf(v, -1.4426950408889634f, -t));   // log2 e less its f32
    // times 2^-64 from e^-v = 2^60 on, where v e^v may be a normal number though e^-v is past all that f32 holds, or its reciprocal below the
    // normal numbers (which the hardware makes 0); t - 64 is exact there
    const bool far = t > 60.f;
    const float by = far ? 0x1p-64f : 1.0f;
    float e = __builtin_amdgcn_exp2f(far ? t - 64.f : t);
    e = fabsf(t) < 192.f ? fmaf(e, r * 0.69314718056f, e) : e;     // else 0, or past everything even so
    const float d = by + e;
    float q = __builtin_amdgcn_rcpf(d);
    q = d <= 3.402823466e38f ? fmaf(fmaf(-d, q, 1.0f), q, q) : q;
    return v * by * q;
}

// What a lane needs of CNT channels from n0 < N on, for any number of tokens.  STREAM: y is written past the caches next to the
// units, which keep tokens and weights for the tiles that follow (2000 x 4096 x 1024 16.4 -> 14.0 us), where its rows are whole lines:
// else those caches join what two lanes write of a line (7662 x 4426 x 64 25 us, past them 38).
template <typename YT, int CNT, bool STREAM> struct Channels {
    typedef YT vec __attribute__((ext_vector_type(CNT)));
    typedef vec vecu __attribute__((aligned(sizeof(YT))));
    typedef float fvec __attribute__((ext_vector_type(CNT)));
    typedef fvec fvecu __attribute__((aligned(4)));
    typedef int ivec __attribute__((ext_vector_type(CNT)));
    fvec ws, b = {};
    int n0;
    bool whole;

    __device__ __forceinline__ Channels(const LinearI8Params& p, int n) : n0(n), whole(n + CNT <= p.N) {
        if (whole) {
            ws = *(const fvecu*)(p.w_scale + n0);
            if (p.bias) b = *(const fvecu*)(p.bias + n0);
        } else {
#pragma unroll
            for (int e = 0; e < CNT; ++e) {
                const int at = n0 + e < p.N ? n0 + e : n0;
                ws[e] = p.w_scale[at];
                if (p.bias) b[e] = p.bias[at];
            }
        }
    }
    __device__ __forceinline__ void store(const LinearI8Params& p, ivec acc, int m, float xs) const {
        YT* y = (YT*)p.y + (int64_t)m * p.y_row + n0;
        const YT* add = p.add ? (const YT*)p.add + (int64_t)m * p.add_row + n0 : nullptr;
        vec a = {};
        if (add) {
            if (whole) a = *(const vecu*)add;
            else
#pragma unroll
                for (int e = 0; e < CNT; ++e)
                    if (n0 + e < p.N) a[e] = add[e];
        }
        float v[CNT];
#pragma unroll
        for (int e = 0; e < CNT; ++e) v[e] = (float)acc[e] * (xs * ws[e]) + b[e];
        if (p.silu)
#pragma unroll
            for (int e = 0; e < CNT; ++e) v[e] = silu_of<YT>(v[e]);
        if (p.alpha != 1.0f)
#pragma unroll
            for (int e = 0; e < CNT; ++e) v[e] *= p.alpha;
        if (add)
#pragma unroll
            for (int e = 0; e < CNT; ++e) v[e] += (float)a[e];
        vec o;
#pragma unroll
        for (int e = 0; e < CNT; ++e) o[e] = (YT)v[e];
        if (whole && STREAM && p.lines) __builtin_nontemporal_store(o, (vecu*)y);
        else if (whole) *(vecu*)y = o;
        else
#pragma unroll
            for (int e = 0; e < CNT; ++e)
                if (n0 + e < p.N) y[e] = o[e];
    }
};

// ---- few tokens ------------------------------------------------------------
// 16 channels x 16 tokens to a workgroup, K shared out over its eight waves block by
// block (a wave reads 1 KB of weights and 1 KB of tokens per block, straight into
// the fragments, four blocks at a time) and the partial sums joined through LDS.
// 64 tokens to a workgroup read the weights once instead of four times, but are fewer workgroups: 64 x 1024 x 4096
// 9.7 us instead of 4.8 (64 of them; with more channels, and so more workgroups, it was not measured).  1 x 8192 x 8192: 11.2 us, 67 MB at 6 TB/s.
constexpr int kRowWaves = 8;
template <typename YT>
__device__ __forceinline__ void rows_finish(const LinearI8Params& p, int4v acc, int4v (&part)[kRowWaves][64], int nh, int m0, const float* xs) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    part[w][lane] = acc;
    __syncthreads();
    // slots 16 h + 4 g + r of the block are these four channels
    const int g = lane >> 4, h = nh & 1, n0 = (nh >> 1) * kI8ColBlock + 16 * (g & 1) + 4 * (2 * h + (g >> 1));
    const int m = m0 + (lane & 15);
    if (w != 0 || m >= p.M || n0 >= p.N) return;
    const Channels<YT, 4, false> ch(p, n0);
    int4v s = part[0][lane];
#pragma unroll
    for (int j = 1; j < kRowWaves; ++j) s += part[j][lane];
    ch.store(p, s, m, xs[m - m0]);
}

template <typename YT> __global__ __launch_bounds__(kRowWaves * 64) void i8_rows_kernel(LinearI8Params p, int mtiles) {
    constexpr int W = kRowWaves, U = 4;
    __shared__ int4v part[W][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int unit = xcd_tile(blockIdx.x, gridDim.x), nh = udiv_small(unit, mtiles), m0 = (unit - nh * mtiles) * 16;     // an XCD reads few weights
    const int kblocks = (p.K + kI8DepthPad - 1) / kI8DepthPad * (kI8DepthPad / kI8DepthBlock);
    const __amdgpu_buffer_rsrc_t rw = make_rsrc((const int8_t*)p.w + (int64_t)(nh >> 1) * kblocks * 2048, (int64_t)kblocks * 2048);
    const int k16 = (p.K + 15) & ~15, rows = p.M - m0 < 16 ? p.M - m0 : 16;
    const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.x + (int64_t)m0 * p.x_row, (int64_t)(rows - 1) * p.x_row + k16);
    const uint32_t wo = ((lane >> 4) * 32 + 16 * (nh & 1) + (lane & 15)) * 16;
    const uint32_t xo = (uint32_t)((lane & 15) * p.x_row + 16 * (lane >> 4));
    int4v acc = {};
    for (int k0 = w; k0 < kblocks; k0 += U * W) {
        int4v a[U], b[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {        // blocks past the last: zeros, and no token read
            const int kb = k0 + u * W;
            a[u] = __builtin_amdgcn_raw_buffer_load_b128(rw, kb < kblocks ? wo + kb * 2048 : OOB, 0, 0);
            b[u] = __builtin_amdgcn_raw_buffer_load_b128(rx, kb < kblocks ? xo + kb * 64 : OOB, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u], b[u], acc, 0, 0, 0);
    }
    rows_finish<YT>(p, acc, part, nh, m0, p.x_scale + m0);
}

// Few tokens as they come, quantised by every workgroup for itself: one launch instead of two where that costs less than
// a launch.  Each wave asks for its first blocks of weights, then the rows are shared out: `wpr` waves to a row, up
// to 8 x 64 x NV values a wave, held in LDS in rows 16 bytes apart in banks.  1 x 4096 x 1024: 3.7 us, in two launches
// 5.2; 16 x 4096 x 1024 5.0 and 5.6; 16 x 4096 x 2048 7.1 and 5.9, so up to 2^14 values.  More tokens than 16 while the
// workgroups are one round of the chip: 64 x 1024 x 1024 5.4 and 5.7, 64 x 4096 x 256 8.1 and 6.2.
template <typename YT, typename XT, int NV> __global__ __launch_bounds__(512) void i8_rows_fused_kernel(LinearI8Params p, const XT* x, int64_t x_row, int wpr, int mtiles) {
    constexpr int W = kRowWaves, U = 8;
    extern __shared__ __align__(16) uint8_t held[];          // [rows][kpad + 16]
    __shared__ int4v part[W][64];
    __shared__ float tops[W], scale[16];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int unit = xcd_tile(blockIdx.x, gridDim.x), nh = udiv_small(unit, mtiles), m0 = (unit - nh * mtiles) * 16;
    const int rows = p.M - m0 < 16 ? p.M - m0 : 16;
    x += m0 * x_row;
    const int kpad = (p.K + kI8DepthPad - 1) / kI8DepthPad * kI8DepthPad, kblocks = kpad / kI8DepthBlock, ld = kpad + 16;
    const __amdgpu_buffer_rsrc_t rw = make_rsrc((const int8_t*)p.w + (int64_t)(nh >> 1) * kblocks * 2048, (int64_t)kblocks * 2048);
    const uint32_t wo = ((lane >> 4) * 32 + 16 * (nh & 1) + (lane & 15)) * 16;
    int4v a[U];
#pragma unroll
    for (int u = 0; u < U; ++u) a[u] = __builtin_amdgcn_raw_buffer_load_b128(rw, w + u * W < kblocks ? wo + (w + u * W) * 2048 : OOB, 0, 0);

    const int slots = W / wpr, sub = w % wpr;
    auto load = [&](int r, float (&v)[NV][8]) {
#pragma unroll
        for (int k = 0; k < NV; ++k) load_row8(v[k], x + r * x_row, 8 * (lane + 64 * (sub + wpr * k)), p.K);
    };
    auto hold = [&](int r, const float (&v)[NV][8], RowTop top) {
        const float s = top.top / 127.0f;
        if (lane == 0 && sub == 0) scale[r] = s;
        const RowQuantiser q(s, top.plain);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int at = 8 * (lane + 64 * (sub + wpr * k));
            if (at < kpad) *(int2v*)(held + r * ld + at) = q(v[k]);      // zeros past K
        }
    };
    if (wpr == 1) {
        for (int r = w; r < rows; r += slots) {
            float v[NV][8];
            load(r, v);
            hold(r, v, row_top<64, NV>(v, nullptr));
        }
    } else {                                 // one row at most to a wave
        const int r = w / wpr;
        float v[NV][8] = {};
        if (r < rows) load(r, v);
        RowTop top = row_top<64, NV>(v, nullptr);
        if (lane == 0) tops[w] = top.plain ? top.top : -top.top;
        __syncthreads();
        for (int i = 0; i < wpr; ++i) {
            const float o = tops[w - sub + i];
            top.plain &= __builtin_bit_cast(int, o) >= 0;
            top.top = fmaxf(top.top, fabsf(o));
        }
        if (r < rows) hold(r, v, top);
    }
    __syncthreads();
    const int row = (lane & 15) < rows ? lane & 15 : rows - 1;         // tokens past the last give sums that nobody reads
    const uint8_t* xr = held + row * ld + 16 * (lane >> 4);
    int4v acc = {};
    for (int k0 = w; k0 < kblocks; k0 += U * W) {
        if (k0 > w)
#pragma unroll
            for (int u = 0; u < U; ++u) a[u] = __builtin_amdgcn_raw_buffer_load_b128(rw, k0 + u * W < kblocks ? wo + (k0 + u * W) * 2048 : OOB, 0, 0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k0 + u * W >= kblocks) break;
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u], *(const int4v*)(xr + (k0 + u * W) * 64), acc, 0, 0, 0);
        }
    }
    rows_finish<YT>(p, acc, part, nh, m0, scale);
}

// ---- many tokens -----------------------------------------------------------
// Four waves side by side, each TM x TN tiles of 32 tokens x 32 channels.  Tokens go through
// LDS (rows of 128 bytes, their 16-byte pieces permuted by the row so that the
// reads of a tile fall into different banks), weights straight into the fragments.
//
// Slab k (128 inputs) is computed in step k.  Its weights were asked for in step k - WD + 1, its tokens, by loads
// straight into LDS, in step k - WD - 1, and waited for by every wave before the barrier that opens step
// k - 1; so the first fragments of step k are read during step k - 1 and no wave
// waits for LDS after a barrier.  Small tiles, whose products of a quarter slab are over before LDS
// answers, have read the whole of slab k by then (AHEAD).  Step k fills the stage that is free: slab k's, read
// ahead, or else slab k - 1's.
// A barrier of the workgroup's waves behind their own LDS reads and all but the last N of their vector-memory
// operations; no memory operation passes it.
template <int N> __device__ __forceinline__ void join() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (0x7 << 4));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <typename YT, int TM, int TN>
__global__ __launch_bounds__(256, 2) void i8_tile_kernel(LinearI8Params p, int mtiles, int ntiles) {
    constexpr int W = 4, BM = 32 * TM, BN = 32 * W * TN, ROWS = BM / 8 / W;   // DMA instructions of a wave per slab
    constexpr bool AHEAD = TM * TN <= 4;
    // weights of two slabs in turn; of four: no faster (512 x 4096 x 4096 on 64 x 128 tiles 15.9 and 15.8 us), more registers
    constexpr int WD = 2, ST = AHEAD ? WD + 1 : WD + 2, STAGE = BM * 128;    // ST stages of tokens
    static_assert(BM / 8 % W == 0, "rows of a slab go evenly over the waves");
    constexpr int SUMS = W * 32 * TN * 128;      // 32 tokens' sums of every wave, at the end
    __shared__ __align__(16) uint8_t slab[ST * STAGE > SUMS ? ST * STAGE : SUMS];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // an XCD's tiles are neighbours: eight rows of tiles at a time, column by column (8192^3 on
    // tiles of 256 x 256: 482 us; one row at a time 563, 16 rows 565, 32 rows 603)
    constexpr int group = 8;
    const int tile = xcd_tile(blockIdx.x, mtiles * ntiles);
    const int g = tile / (group * ntiles), in = tile - g * group * ntiles;
    const int gm = mtiles - g * group < group ? mtiles - g * group : group;
    const int tn = in / gm, m0 = (g * group + in - tn * gm) * BM, n0 = tn * BN;
    const int slabs = (p.K + kI8DepthPad - 1) / kI8DepthPad, kblocks = 2 * slabs;
    const int k16 = (p.K + 15) & ~15, rows = p.M - m0 < BM ? p.M - m0 : BM;
    const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.x + (int64_t)m0 * p.x_row, (int64_t)(rows - 1) * p.x_row + k16);
    const int nblocks = (p.N + 31) / 32, b0 = n0 / 32, nb = nblocks - b0 < BN / 32 ? nblocks - b0 : BN / 32;
    const __amdgpu_buffer_rsrc_t rw = make_rsrc((const int8_t*)p.w + (int64_t)b0 * kblocks * 2048, (int64_t)nb * kblocks * 2048);

    uint32_t xo[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = (wid * ROWS + i) * 8 + (lane >> 3);
        xo[i] = (uint32_t)(r * p.x_row + 16 * ((lane & 7) ^ (r >> 1 & 7)));
    }
    uint32_t wo[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) wo[j] = (uint32_t)((wid * TN + j) * kblocks * 2048 + lane * 16);
    uint32_t ao[4];                          // a lane's pieces of a stage, tile 0
#pragma unroll
    for (int q = 0; q < 4; ++q) ao[q] = (uint32_t)((lane & 31) * 128 + 16 * ((2 * q + (lane >> 5)) ^ (lane >> 1 & 7)));

    int16v acc[TM][TN] = {};
    int4v wf[WD][4][TN], xf[2][AHEAD ? 4 : 1][TM];
    // past the last slab nothing is read: a resource of no bytes, so that every step issues the same loads
    const __amdgpu_buffer_rsrc_t none = make_rsrc(p.w, 0);
    auto fetch = [&](int k, int stage, int i) {      // a wave's i-th 1 KB of slab k
        // the whole offset in the lane's part: only that is held against the end of the tokens
        lds_dma16(k < slabs ? rx : none, slab + stage * STAGE + (wid * ROWS + i) * 1024, xo[i] + k * 128, 0);
    };
    auto fetch_w = [&](int k, int q, int4v (&f)[4][TN]) {
        const __amdgpu_buffer_rsrc_t r = k < slabs ? rw : none;
#pragma unroll
        for (int j = 0; j < TN; ++j) f[q][j] = __builtin_amdgcn_raw_buffer_load_b128(r, wo[j] + q * 1024, k * 4096, 0);
    };
    auto read = [&](int stage, int q, int4v (&f)[TM]) {
        const uint8_t* st = slab + stage * STAGE;
#pragma unroll
        for (int i = 0; i < TM; ++i) f[i] = *(const int4v*)(st + ao[q] + i * 32 * 128);
    };
    int stage = 0;                           // slab k's
    auto step = [&](int k, int u, int4v (&w)[4][TN], int4v (&next)[4][TN]) {     // u: k modulo WD
        // slab k + 1 is there; what the last WD - 1 steps asked for may still be on its way
        join<(WD - 1) * (ROWS + 4 * TN)>();
        const int after = stage == ST - 1 ? 0 : stage + 1, before = stage == 0 ? ST - 1 : stage - 1;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (AHEAD) read(after, q, xf[(u + 1) & 1][q]);
            else if (q < 3) read(stage, q + 1, xf[(q + 1) & 1][0]);
            else read(after, 0, xf[0][0]);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                // loads in the middle of the products, a few at a time: in one burst they fill the queue and hold up what is behind them
                if (i == TM / 2) {
                    __builtin_amdgcn_sched_barrier(0);
                    fetch_w(k + WD - 1, q, next);
#pragma unroll
                    for (int d = q * ROWS / 4; d < (q + 1) * ROWS / 4; ++d) fetch(k + WD + 1, AHEAD ? stage : before, d);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[q][j], AHEAD ? xf[u & 1][q][i] : xf[q & 1][0][i], acc[i][j], 0, 0, 0);
            }
        }
        stage = after;
    };
    // in the order in which the steps before the first would have issued them, so that step 0's count holds
#pragma unroll
    for (int k = 0; k < WD + 1; ++k) {
        if (k >= 2)
#pragma unroll
            for (int q = 0; q < 4; ++q) fetch_w(k - 2, q, wf[k - 2]);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) fetch(k, k, i);
    }
    join<(WD - 1) * (ROWS + 4 * TN) + ROWS>();
#pragma unroll
    for (int q = 0; q < (AHEAD ? 4 : 1); ++q) read(0, q, xf[0][q]);
    for (int k = 0; k < slabs; k += WD) {
#pragma unroll
        for (int u = 0; u < WD; ++u)
            if (k + u < slabs) step(k + u, u, wf[u], wf[(u + WD - 1) % WD]);
    }

    // A wave's sums pass through LDS (32 tokens at a time, their 16-byte pieces permuted by the row), so that
    // neighbouring lanes write neighbouring pieces of a row: as the matrix instructions leave them a store would touch 64
    // half lines (2000 x 4096 outputs took 6 us that way, a fill of their 16 MB 4.9).
    constexpr int E = 16 / sizeof(YT), PER = 32 * TN / E, STEP = 64 / PER, PIECES = 8 * TN;
    join<0>();
    auto swizzle = [](int r) { return TN == 1 ? r >> 1 & 7 : r & (PIECES - 1); };   // 16 rows' pieces in 64 banks
    uint8_t* own = slab + wid * 32 * TN * 128;
    const int n = n0 + wid * TN * 32 + E * (lane % PER);
    if (n0 + wid * TN * 32 >= p.N) return;
    const Channels<YT, E, true> ch(p, n < p.N ? n : p.N - 1);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int r0 = lane & 31;
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int piece = 8 * j + 4 * (lane >> 5) + g;
                *(int4v*)(own + r0 * TN * 128 + 16 * (piece ^ swizzle(r0))) = int4v{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
            }
#pragma unroll
        for (int r1 = 0; r1 < 32; r1 += STEP) {
            const int r = r1 + lane / PER, m = m0 + i * 32 + r;
            typename Channels<YT, E, true>::ivec v;
#pragma unroll
            for (int h = 0; h < E / 4; ++h) {
                const int4v c = *(const int4v*)(own + r * TN * 128 + 16 * (((E / 4) * (lane % PER) + h) ^ swizzle(r)));
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * h + e] = c[e];
            }
            if (m < p.M && n < p.N) ch.store(p, v, m, p.x_scale[m]);
        }
    }
}

template <typename YT, int TM, int TN> void launch_tiles(LinearI8Params p, hipStream_t s) {
    p.lines = ((uintptr_t)p.y | (uintptr_t)(p.y_row * (int64_t)sizeof(YT))) % 64 == 0;
    const int mt = cdiv(p.M, 32 * TM), nt = cdiv(p.N, 128 * TN);
    launch(i8_tile_kernel<YT, TM, TN>, dim3(mt * nt), dim3(256), 0, s, p, mt, nt);
}

// The form of the least estimated time: a start and, for each round of workgroups that the chip holds, an end and the
// 1024s of K.  Fitted to products run back to back (0.15 s: the card's clock is then 1.6 GHz for the large ones), us:
//                              16 x 16   32 x 128   64 x 128   64 x 256   128 x 256
//      64 x  1024 x 4096          4.3       7.9        9.4       14.8        24.9
//     128 x  4096 x 4096         19.6       8.1        9.5       15.0        27.4
//     200 x  1024 x 1024          5.2       4.5        5.4        8.0        13.3
//     512 x  4096 x 4096         72        16.7       14.9       18.2        29.6
//    1000 x  4096 x 1024                    9.4        8.1        8.9        13.5
//    2000 x  4096 x 1024                   18.9       14.8       13.9        15.1    (256 x 256, eight waves: 17.9)
//    2000 x  4096 x 4096                   57.7       44.9       37.3        35.7                            42.1
//   16384 x  4096 x 4096                  443        319        278         237                             245
//    8192 x  8192 x 8192                  888        619        532         445                             450
// Over 63 shapes that it was fitted to the form taken is 0.4% slower than the best one on the mean (12% at most), over 40 others 2.8%
// (26%: 1901 x 8099 x 426; 21%: 7384 x 831 x 4723).  None has weights above 18 MB, and the estimate knows neither their bytes nor that a
// unit's second tile is a whole one: it says 13.8 us of 64 x 8192 x 8192, which takes 21.5, and 20.9 of 4223 x 1024 x 4096, 30.4.
LinearI8Tile least_tile(int M, int N, int K) {
    const float depth = K / 1024.0f;
    const auto rounds = [&](int bm, int bn, float held) { return (float)cdiv(M, bm) * cdiv(N, bn) / held; };
    const auto least = [](float r, float most) { return r > most ? r : most; };    // fewer workgroups take no less
    const float units = rounds(16, 16, 256), rows = 2.65f + least(units, 0.85f) * (0.34f + 0.43f * depth);
    // a launch holds fewer than 2^32 threads; 2^36 results are fewer than that on the larger tiles
    const bool small = (int64_t)cdiv(M, 32) * cdiv(N, 128) < 1 << 24;
    const float t32 = small ? 3.15f + least(rounds(32, 128, 256), 0.76f) * (0.22f + 1.72f * depth) : __builtin_inff();
    const float t64 = 3.74f + least(rounds(64, 128, 256), 0.77f) * (0.74f + 2.07f * depth);
    const float wide64 = 4.26f + least(rounds(64, 256, 512), 0.4f) * (3.33f + 7.24f * depth);
    const float wide128 = 5.98f + least(rounds(128, 256, 512), 0.45f) * (4.66f + 13.87f * depth);
    const float best = fminf(fminf(t32, t64), fminf(wide64, wide128));
    if (rows < best && units * 256 < (float)(1 << 21)) return {16, 16, 2 * (int64_t)cdiv(N, 32) * cdiv(M, 16)};
    const auto tile = [&](int bm, int bn) { return LinearI8Tile{bm, bn, (int64_t)cdiv(M, bm) * cdiv(N, bn)}; };
    return wide128 == best ? tile(128, 256) : wide64 == best ? tile(64, 256) : t64 == best ? tile(64, 128) : tile(32, 128);
}
template <typename YT> void launch_typed(const LinearI8Params& p, hipStream_t s) {
    const LinearI8Tile t = least_tile(p.M, p.N, p.K);
    if (t.tokens == 16) launch(i8_rows_kernel<YT>, dim3((unsigned)t.workgroups), dim3(512), 0, s, p, cdiv(p.M, 16));
    else if (t.tokens == 128) launch_tiles<YT, 4, 2>(p, s);
    else if (t.channels == 256) launch_tiles<YT, 2, 2>(p, s);
    else if (t.tokens == 64) launch_tiles<YT, 2, 1>(p, s);
    else launch_tiles<YT, 1, 1>(p, s);
}

// Waves to a row of the fused form: all eight for one token, one from five tokens on.
int fused_waves(int M) { return M == 1 ? 8 : M == 2 ? 4 : M <= 4 ? 2 : 1; }

template <typename YT, typename XT> void launch_fused(const LinearI8Params& p, const QuantizeRowsParams& q, hipStream_t s) {
    const int wpr = fused_waves(p.M), kpad = cdiv(p.K, kI8DepthPad) * kI8DepthPad, mtiles = cdiv(p.M, 16);
    const uint32_t lds = (p.M < 16 ? p.M : 16) * (kpad + 16);
    const int per = cdiv(kpad, 512 * wpr);
    const dim3 grid(2 * cdiv(p.N, 32) * mtiles);
    if (per <= 1) launch(i8_rows_fused_kernel<YT, XT, 1>, grid, dim3(512), lds, s, p, (const XT*)q.x, q.x_row, wpr, mtiles);
    else if (per <= 2) launch(i8_rows_fused_kernel<YT, XT, 2>, grid, dim3(512), lds, s, p, (const XT*)q.x, q.x_row, wpr, mtiles);
    else launch(i8_rows_fused_kernel<YT, XT, 4>, grid, dim3(512), lds, s, p, (const XT*)q.x, q.x_row, wpr, mtiles);
}

}  // namespace

LinearI8Tile linear_i8_tile(int M, int N, int K, bool i8) {
    if (M == 0 || N == 0) return {0, 0, 0};
    if (!i8 && linear_i8_fused(M, N, K)) return {16, 16, 2 * (int64_t)cdiv(N, 32) * cdiv(M, 16)};
    return least_tile(M, N, K);
}
bool linear_i8_fused(int M, int N, int K) {
    const int kpad = cdiv(K, kI8DepthPad) * kI8DepthPad, rows = M < 16 ? M : 16;
    if (kpad > 4 * 512 * fused_waves(M) || rows * kpad > 16384) return false;
    return M <= 16 || (double)cdiv(N, 32) * 2 * cdiv(M, 16) <= 256;
}
void launch_linear_i8_fused(const LinearI8Params& p, const QuantizeRowsParams& q, hipStream_t s) {
    if (p.M == 0 || p.N == 0) return;
    if (p.y_f32) q.f32 ? launch_fused<float, float>(p, q, s) : launch_fused<float, f16>(p, q, s);
    else q.f32 ? launch_fused<f16, float>(p, q, s) : launch_fused<f16, f16>(p, q, s);
}

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
