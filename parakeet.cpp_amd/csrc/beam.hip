// Beam search: the W best of an item's W x V candidates, and the reordering of
// the beams' states by their parents.
//
// Candidate (w, v) has the score c = score[w] + (x[w][v] - lse[w]),
// lse = log sum exp x[w], and a finished beam has the one candidate (end,
// score).  Beams compete with each other through lse, so the sums of the
// exponentials and everything after them are in f64 (the terms are f32
// exponentials of an argument with 2^-40 relative error: their errors are
// independent and average out to about 1e-8 of lse).  Within a beam the order
// of the candidates is that of the logits, so a beam's W largest logits are
// all that can win.
//
// select_rows: one wave per chunk of a row, the chunk in registers: maximum,
// sum of exp(x - maximum), and its W largest logits in W rounds of a wave-wide
// maximum (ties: lowest index).  select_item: one wave per item: lse of each
// beam, then W rounds of a maximum over the heads of all lists.
#include "decoder.hpp"

namespace pkx {
namespace {

constexpr int kPer = 32, kChunk = 64 * kPer;    // logits per lane and per wave

// float -> unsigned with the same order; NaN below everything, -0 as +0
__device__ __forceinline__ uint32_t order_bits(float x) {
    x += 0.0f;
    const uint32_t u = __float_as_uint(x);
    return x != x ? 0u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t w = __shfl_xor(v, o, 64);
        v = v > w ? v : w;
    }
    return v;
}
__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

struct ChunkStat { float max; float pad; double sum; };     // NaN sum: a NaN or +inf logit
struct SelectWork {
    ChunkStat* stat;      // [B W][chunks]
    float* val;           // [B W][chunks][W]
    int* idx;             // [B W][chunks][W], -1 past a list's end
    int chunks;
};

// e^d for d <= 0: 2^(d log2 e) with the product's rounding error carried along
__device__ __forceinline__ float exp_below(float d) {
    d = fmaxf(d, -200.0f);       // 0 from there on
    const float t = d * 1.4426950408889634f;
    const float lo = fmaf(d, 1.4426950408889634f, -t) + d * 1.925963033500e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, lo * 0.6931471805599453f, e);
}

template <bool F32> __global__ __launch_bounds__(256) void select_rows_kernel(BeamSelectParams p, SelectWork ws) {
    const int lane = threadIdx.x & 63;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), rows = (int64_t)p.B * p.W;
    if (unit >= rows * ws.chunks) return;
    const int64_t row = unit / ws.chunks;
    const int base = (int)(unit - row * ws.chunks) * kChunk;
    if (p.done && p.done[row]) return;                       // its one candidate needs no logits
    const int n = p.V - base < kChunk ? p.V - base : kChunk;
    uint32_t key[kPer];
    float mx = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int at = i * 64 + lane;
        float x = 0.f;
        if (at < n) {
            if constexpr (F32) x = ((const float*)p.logits)[row * p.row + base + at];
            else x = (float)((const f16*)p.logits)[row * p.row + base + at];
            bad |= x != x || x == INFINITY;
            mx = fmaxf(mx, x);
        }
        key[i] = at < n ? order_bits(x) : 0u;                // 0: no logit here (or NaN)
    }
    mx = wave_max(mx);
    double sum = 0.0;
    if (mx != -INFINITY) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const float x = order_value(key[i]);
            if (key[i] != 0u) sum += (double)exp_below(x - mx);
        }
    }
    sum = wave_sum_f64(sum);
    if (__ballot(bad)) sum = __builtin_nan("");
    if (lane == 0) ws.stat[unit] = ChunkStat{mx, 0.f, sum};
    float* val = ws.val + unit * p.W;
    int* idx = ws.idx + unit * p.W;
    uint32_t best = 0;
    int where = 0;
    auto rescan = [&] {
        best = 0;
        where = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (key[i] > best) {
                best = key[i];
                where = i;
            }
    };
    rescan();
    for (int k = 0; k < p.W; ++k) {
        const uint32_t top = wave_max_u32(best);
        if (top == 0u) {
            for (int j = k + lane; j < p.W; j += 64) idx[j] = -1;
            break;
        }
        // lowest index of the largest: lowest i, then lowest lane
        int at = best == top ? where * 64 + lane : 0x7fffffff;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const int w = __shfl_xor(at, o, 64);
            at = at < w ? at : w;
        }
        if (lane == 0) {
            val[k] = order_value(top);
            idx[k] = base + at;
        }
        if (lane == (at & 63)) {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (i == (at >> 6)) key[i] = 0u;
            rescan();
        }
    }
}

// candidate a = w V + v of score ca ranks before b (-1: none)
__device__ __forceinline__ bool before(double ca, int64_t a, double cb, int64_t b) {
    return a >= 0 && (b < 0 || ca > cb || (ca == cb && a < b));
}

__global__ __launch_bounds__(64) void select_item_kernel(BeamSelectParams p, SelectWork ws) {
    const int lane = threadIdx.x, b = blockIdx.x, W = p.W, lists = W * ws.chunks;
    __shared__ double lse[kMaxBeams], score[kMaxBeams];
    __shared__ int kind[kMaxBeams];            // 0: its lists, 1: finished, 2: no finite score
    extern __shared__ int head[];              // [lists]
    for (int w = 0; w < W; ++w) {
        const int64_t row = (int64_t)b * W + w;
        const float sc = p.scores[row];
        const bool fin = p.done && p.done[row];
        double z = 0.0;
        if (!fin) {
            float mx = -INFINITY;
            for (int i = lane; i < ws.chunks; i += 64) mx = fmaxf(mx, ws.stat[row * ws.chunks + i].max);
            mx = wave_max(mx);
            double s = 0.0;
            for (int i = lane; i < ws.chunks; i += 64) {
                const ChunkStat st = ws.stat[row * ws.chunks + i];
                if (st.max != -INFINITY || st.sum != 0.0) s += st.sum * exp((double)st.max - (double)mx);
            }
            z = (double)mx + log(wave_sum_f64(s));
        }
        if (lane == 0) {
            const bool dead = !(sc < INFINITY) || sc == -INFINITY || !(z < 1e300 && z > -1e300);
            score[w] = !(sc < INFINITY) ? -INFINITY : (double)sc;
            lse[w] = z;
            kind[w] = fin ? 1 : dead ? 2 : 0;
        }
    }
    for (int i = lane; i < lists; i += 64) head[i] = 0;
    __syncthreads();
    for (int k = 0; k < W; ++k) {
        double bc = 0.0;
        int64_t ba = -1;
        int bl = -1;
        for (int i = lane; i < lists; i += 64) {
            const int w = i / ws.chunks, h = head[i], first = i - w * ws.chunks == 0;
            if (h >= W) continue;
            double c;
            int64_t at;
            if (kind[w] == 1) {
                if (!first || h) continue;
                c = score[w];
                at = (int64_t)w * p.V + p.end_id;
            } else if (kind[w] == 2) {             // every candidate is -inf: in order of the index
                if (!first || h >= p.V) continue;
                c = -INFINITY;
                at = (int64_t)w * p.V + h;
            } else {
                const int64_t o = ((int64_t)b * lists + i) * W + h;
                if (ws.idx[o] < 0) continue;
                c = score[w] + ((double)ws.val[o] - lse[w]);
                at = (int64_t)w * p.V + ws.idx[o];
            }
            if (before(c, at, bc, ba)) {
                bc = c;
                ba = at;
                bl = i;
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const double c = __shfl_xor(bc, o, 64);
            const int64_t a = __shfl_xor(ba, o, 64);
            const int l = __shfl_xor(bl, o, 64);
            if (before(c, a, bc, ba)) {
                bc = c;
                ba = a;
                bl = l;
            }
        }
        if (lane == 0) {
            const int w = (int)(ba / p.V), v = (int)(ba - (int64_t)w * p.V);
            const int64_t o = (int64_t)b * W + k;
            p.parent[o] = w;
            p.token[o] = v;
            p.new_scores[o] = (float)bc;
            if (p.new_done) p.new_done[o] = (kind[w] == 1 || v == p.end_id) ? 1 : 0;
            head[bl] += 1;
        }
        __syncthreads();
    }
}

struct ReorderParams {
    const int* parent;
    int64_t rows;
    int W, n;
    BeamState st[kMaxBeamStates];
    int width[kMaxBeamStates];       // bytes a thread moves at a time
};

__global__ __launch_bounds__(256) void reorder_kernel(ReorderParams p) {
    const BeamState& s = p.st[blockIdx.y];
    const int width = p.width[blockIdx.y];
    const int64_t row = blockIdx.x, item = row / p.W;
    const int from = p.parent[row];
    if ((unsigned)from >= (unsigned)p.W) return;             // left as it was
    const uint8_t* x = s.src + (item * p.W + from) * s.src_row;
    uint8_t* y = s.dst + row * s.dst_row;
    const int64_t first = (int64_t)blockIdx.z * 256 + threadIdx.x, step = (int64_t)gridDim.z * 256;
    if (width == 16) {
        for (int64_t i = first; i < s.bytes / 16; i += step) ((int4v*)y)[i] = ((const int4v*)x)[i];
    } else if (width == 4) {
        for (int64_t i = first; i < s.bytes / 4; i += step) ((int*)y)[i] = ((const int*)x)[i];
    } else {
        for (int64_t i = first; i < s.bytes; i += step) y[i] = x[i];
    }
}

size_t up16(size_t n) { return (n + 15) / 16 * 16; }

}  // namespace

size_t beam_select_workspace(const BeamSelectParams& p) {
    const size_t lists = (size_t)p.B * p.W * cdiv(p.V, kChunk);
    return lists * sizeof(ChunkStat) + up16(lists * p.W * sizeof(float)) + lists * p.W * sizeof(int);
}

void launch_beam_select(const BeamSelectParams& p, void* ws, size_t ws_bytes, hipStream_t s) {
    if (p.B == 0) return;
    const size_t need = beam_select_workspace(p);
    require(ws && ws_bytes >= need, "beam select: the workspace is smaller than its size query says");
    SelectWork w;
    w.chunks = cdiv(p.V, kChunk);
    const size_t lists = (size_t)p.B * p.W * w.chunks;
    require(lists < ((size_t)1 << 25) && (size_t)p.W * w.chunks <= 12288, "beam select: too many beams and words for one call");
    w.stat = (ChunkStat*)ws;
    w.val = (float*)((char*)ws + lists * sizeof(ChunkStat));
    w.idx = (int*)((char*)w.val + up16(lists * p.W * sizeof(float)));
    const dim3 grid((unsigned)((lists + 3) / 4));
    if (p.f32) launch(select_rows_kernel<true>, grid, dim3(256), 0, s, p, w);
    else launch(select_rows_kernel<false>, grid, dim3(256), 0, s, p, w);
    launch(select_item_kernel, dim3(p.B), dim3(64), (uint32_t)(p.W * w.chunks * sizeof(int)), s, p, w);
}

void launch_beam_reorder(const int* parent, int B, int W, const BeamState* states, int n, hipStream_t s) {
    if (B == 0 || n == 0) return;
    ReorderParams p = {};
    p.parent = parent;
    p.rows = (int64_t)B * W;
    p.W = W;
    int64_t most = 0;
    for (int i = 0; i < n; ++i) {
        if (states[i].bytes == 0) continue;
        const uintptr_t bits = (uintptr_t)states[i].src | (uintptr_t)states[i].dst | (uintptr_t)states[i].src_row |
                               (uintptr_t)states[i].dst_row | (uintptr_t)states[i].bytes;
        p.st[p.n] = states[i];
        p.width[p.n] = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
        const int64_t units = states[i].bytes / p.width[p.n];
        most = units > most ? units : most;
        ++p.n;
    }
    if (p.n == 0) return;
    require(p.rows < (1 << 23), "beam reorder: too many rows for one call");
    int64_t z = (most + 1023) / 1024;                        // four pieces a thread
    z = z > 64 ? 64 : z;
    launch(reorder_kernel, dim3((unsigned)p.rows, p.n, (unsigned)z), dim3(256), 0, s, p);
}

}  // namespace pkx
