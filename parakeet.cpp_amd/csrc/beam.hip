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
// The W largest of many values: with the values in 64 groups, the W-th largest
// of the groups' maxima bounds the W-th largest value from below, and only a few
// values more than W reach it.  The bound is found bit by bit on an
// order-preserving integer (a ballot and a count per bit, its top 20 bits: a lower
// bound is all that is wanted); the values that reach it go to a list in LDS and
// are ranked there by counting.  Where more reach it than the list holds (ties),
// W rounds of a maximum over the workgroup take over.  (W rounds for every call
// instead of the bound: 25.1, 41.1 and 145 us for the calls below.)
//
// Few words (all of an item in one workgroup's registers): select_small, one
// launch.  Otherwise select_rows, a workgroup per row or chunk of one, writes
// the chunk's maximum, sum and list; select_item, a workgroup per item, forms
// the scores and ranks them.
//
// Measured, with the reordering of the states, us: 1 item x 4 beams x 1025 words
// (f32) 9.1, 16 x 8 x 8193 (f16) 13.8, 32 x 16 x 32769 (f32) 29.2.  A launch that
// does nothing takes 2.5 to 3, so the first two are launches and dependent steps; the
// last reads its 67 MB of logits at 3.7 TB/s in 18 (a copy reaches 5.1).
#include "decoder.hpp"

namespace pkx {
namespace {

constexpr int kPer = 32, kSmallPer = 16, kFew = 8;      // logits a lane holds: of a chunk, of an item, of a short row
constexpr int kRowThreads = 256, kChunk = kRowThreads * kPer;
constexpr int kSmallThreads = 1024, kItemThreads = 1024;
constexpr int kList = 128;                      // candidates of a chunk
constexpr int kHits = 1024;                     // candidates of an item that are ranked

// float -> unsigned with the same order; NaN below everything, -0 as +0
__device__ __forceinline__ uint32_t order_bits(float x) {
    x += 0.0f;
    const uint32_t u = __float_as_uint(x);
    return x != x ? 0u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
// the least float whose order_bits reach k
__device__ __forceinline__ float order_value(uint32_t k) {
    return k < 0x00800000u ? -INFINITY : __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

template <int CTRL> __device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
template <int CTRL> __device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)dpp_u32<CTRL>((uint32_t)(u >> 32)) << 32 | dpp_u32<CTRL>((uint32_t)u));
}
// over the whole wave, every lane receiving the result: DPP within 16 lanes,
// then lane swaps between the rows
__device__ __forceinline__ float wave_max_dpp(float v) {
    v = fmaxf(v, dpp_get<0xB1>(v));
    v = fmaxf(v, dpp_get<0x4E>(v));
    v = fmaxf(v, dpp_get<0x141>(v));
    v = fmaxf(v, dpp_get<0x140>(v));
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ double row16_sum_f64(double v) {
    v += dpp_f64<0xB1>(v);
    v += dpp_f64<0x4E>(v);
    v += dpp_f64<0x141>(v);
    v += dpp_f64<0x140>(v);
    return v;
}
__device__ __forceinline__ double wave_sum_f64(double v) {
    v = row16_sum_f64(v);
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

struct ChunkStat { float max; int n; double sum; };     // n: candidates listed; NaN sum: a NaN or +inf logit
struct Entry { uint32_t key; int v; };                  // order_bits of the logit, the word
struct SelectWork {
    ChunkStat* stat;      // [B W][chunks]
    Entry* list;          // [B W][chunks][kList]
    int chunks, len;      // len: logits of a chunk
};

// e^d for d <= 0: 2^(d log2 e) with the product's rounding error carried along
__device__ __forceinline__ float exp_below(float d) {
    d = fmaxf(d, -200.0f);       // 0 from there on
    const float t = d * 1.4426950408889634f;
    const float lo = fmaf(d, 1.4426950408889634f, -t) + d * 1.925963033500e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, lo * 0.6931471805599453f, e);
}

// n logits of a row over `threads` threads, VEC adjacent ones a thread and step:
// 16 bytes (rows of odd length are aligned to their elements only), or one where
// that leaves threads without any (f16, 4 beams x 1025 words: 8.0 us with 16 bytes, 6.4
// with one; 16 x 8 x 700: 9.1 and 7.8).  PER registers, used or not, are what a
// short row costs (4 x 1025, f32: 7.2 us with 32, 6.4 with 8).  Register i of thread t is
// logit word(i), -inf where there is none.  The thread whose piece the row's
// end cuts reads the row's last 16 bytes instead and leaves out what its
// neighbour has, so that no load waits on a branch.
template <bool F32, int VEC, int PER> struct RowRegs {
    static constexpr int G = PER / VEC;
    float x[PER];
    int n, o0, step, groups, last;
    __device__ __forceinline__ int piece(int g) const { return o0 + g * step; }
    __device__ __forceinline__ int cut(int g) const { return piece(g) < last ? piece(g) : last; }
    __device__ __forceinline__ int word(int i) const { return cut(i / VEC) + i % VEC; }
    __device__ __forceinline__ bool has(int i) const { return word(i) >= piece(i / VEC) && word(i) < n; }
    __device__ __forceinline__ bool any() const { return o0 < n; }
    __device__ __forceinline__ void load(const void* logits, int64_t first, int n_, int t, int threads) {
        typedef int words4 __attribute__((ext_vector_type(4), aligned(4)));
        typedef int words2 __attribute__((ext_vector_type(4), aligned(2)));
        using words = std::conditional_t<F32, words4, words2>;
        n = n_;
        o0 = t * VEC;
        step = threads * VEC;
        last = __builtin_amdgcn_readfirstlane(n > VEC ? n - VEC : 0);
        const int left = n - __builtin_amdgcn_readfirstlane(o0);
        groups = left > 0 ? (left + step - 1) / step : 0;        // steps that reach any of the wave's lanes
        // steps past the row's end read its last piece again
        if constexpr (VEC == 1) {
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int64_t o = first + cut(g);
                const float v = F32 ? ((const float*)logits)[o] : (float)((const f16*)logits)[o];
                x[g] = has(g) ? v : -INFINITY;
            }
        } else {
            int4v raw[G];
#pragma unroll
            for (int g = 0; g < G; ++g) raw[g] = *(const words*)((const uint8_t*)logits + (first + cut(g)) * (F32 ? 4 : 2));
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int g = i / VEC, e = i % VEC;
                float v;
                if constexpr (F32) v = __int_as_float(raw[g][e]);
                else v = (float)__builtin_bit_cast(f16, (uint16_t)((uint32_t)raw[g][e / 2] >> (16 * (e & 1))));
                x[i] = has(i) ? v : -INFINITY;
            }
        }
    }
    __device__ __forceinline__ float max() const {
        float m = x[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) m = fmaxf(m, x[i]);
        return m;
    }
    // sum of e^(x - m) for a maximum m over these and other lanes, NaN where a logit is NaN or +inf
    __device__ __forceinline__ double sum(float m) const {
        double s = 0.0;
        bool bad = false;
        if (m == -INFINITY) m = 0.f;
        steps([&](int i) {
            bad |= !(x[i] < INFINITY);
            s += (double)exp_below(x[i] - m);
        });
        return bad ? __builtin_nan("") : s;
    }
    template <typename F> __device__ __forceinline__ void each(F&& f) const {
        steps([&](int i) {
            if (has(i)) f(x[i], word(i));
        });
    }
    // f(register) for the registers of the steps that reach the wave, unrolled whatever f is
    template <typename F> __device__ __forceinline__ void steps(F&& f) const {
        int n_steps = __builtin_amdgcn_readfirstlane(groups);
        asm volatile("" : "+s"(n_steps));       // else the compiler copies what follows for every number of steps
        step_from<0>(n_steps, f);
    }
    template <int S, typename F> __device__ __forceinline__ void step_from(int n_steps, F& f) const {
        if constexpr (S < G) {
            if (S >= n_steps) return;
#pragma unroll
            for (int e = 0; e < VEC; ++e) f(S * VEC + e);
            step_from<S + 1>(n_steps, f);
        }
    }
};

// the largest T (of 20 bits) that W lanes' keys reach, at least 1
__device__ __forceinline__ uint32_t reach_of(uint32_t key, int W) {
    uint32_t T = 0;
#pragma unroll
    for (int bit = 31; bit >= 12; --bit) {
        const uint32_t c = T | (1u << bit);
        if (__popcll(__ballot(key >= c)) >= W) T = c;
    }
    return T ? T : 1u;
}

// ... with every thread's best key in LDS, folded to 64 groups (the same in every wave)
template <int WAVES> __device__ __forceinline__ uint32_t reach_of_block(const uint32_t* keys, int W) {
    uint32_t k = keys[threadIdx.x & 63];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
        const uint32_t o = keys[i * 64 + (threadIdx.x & 63)];
        k = o > k ? o : k;
    }
    return reach_of(k, W);
}

// Candidates rank by score, then by beam, then by `in`: the logit's order bits
// and the complement of the word (a beam's own order).
struct Cand {
    double c;
    uint64_t in;       // 0: none
    int w;
};
__device__ __forceinline__ uint64_t in_beam(uint32_t key, int v) { return (uint64_t)key << 32 | (uint32_t)~v; }
__device__ __forceinline__ bool before(const Cand& a, const Cand& b) {
    if (a.in == 0 || b.in == 0) return a.in != 0;
    return a.c > b.c || (a.c == b.c && (a.w < b.w || (a.w == b.w && a.in > b.in)));
}
__device__ __forceinline__ uint64_t shfl_xor_u64(uint64_t v, int o) {
    return (uint64_t)__shfl_xor((uint32_t)(v >> 32), o, 64) << 32 | __shfl_xor((uint32_t)v, o, 64);
}
template <int WAVES> __device__ Cand block_best(Cand a, Cand* part) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const Cand b = {__shfl_xor(a.c, o, 64), shfl_xor_u64(a.in, o), __shfl_xor(a.w, o, 64)};
        if (before(b, a)) a = b;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = a;
    __syncthreads();
    a = part[0];
    for (int i = 1; i < WAVES; ++i)
        if (before(part[i], a)) a = part[i];
    return a;
}

enum BeamKind : int { BEAM_LIVE = 0, BEAM_DONE = 1, BEAM_DEAD = 2 };    // dead: no candidate above -inf
struct Hits {
    double c[kHits];
    uint64_t in[kHits];
    uint8_t w[kHits];
    int n;
};
__device__ __forceinline__ void put_out(const BeamSelectParams& p, int b, int rank, const Cand& x, int kind) {
    const int64_t o = (int64_t)b * p.W + rank;
    const int v = (int)~(uint32_t)x.in;
    p.parent[o] = x.w;
    p.token[o] = v;
    p.new_scores[o] = (float)x.c;
    if (p.new_done) p.new_done[o] = (kind == BEAM_DONE || v == p.end_id) ? 1 : 0;
}
__device__ __forceinline__ void add_hit(Hits& h, const Cand& x) {
    const int at = atomicAdd(&h.n, 1);      // the ranking does not go by the place
    if (at < kHits) {
        h.c[at] = x.c;
        h.in[at] = x.in;
        h.w[at] = (uint8_t)x.w;
    }
}
// every candidate of the list counts those before it (at least W are listed), 16 lanes a candidate
__device__ __forceinline__ void rank_hits(const BeamSelectParams& p, int b, const Hits& h, const uint8_t* kind) {
    const int n = h.n, l = threadIdx.x & 15;
    for (int i0 = 0; i0 < n; i0 += (int)blockDim.x / 16) {
        const int i = i0 + (threadIdx.x >> 4), at = i < n ? i : n - 1;
        const Cand x = {h.c[at], h.in[at], h.w[at]};
        int rank = 0;
        for (int j = l; j < n; j += 16) rank += before(Cand{h.c[j], h.in[j], h.w[j]}, x) ? 1 : 0;
        rank += (int)dpp_u32<0xB1>((uint32_t)rank);
        rank += (int)dpp_u32<0x4E>((uint32_t)rank);
        rank += (int)dpp_u32<0x141>((uint32_t)rank);
        rank += (int)dpp_u32<0x140>((uint32_t)rank);
        if (l == 0 && i < n && rank < p.W) put_out(p, b, rank, x, kind[x.w]);
    }
}

__device__ __forceinline__ double beam_score(const BeamSelectParams& p, int64_t row) {
    const float s = p.scores[row];
    return s < INFINITY ? (double)s : -INFINITY;         // NaN and +inf count as -inf
}
__device__ __forceinline__ bool is_dead(double score, double lse) { return score == -INFINITY || !(lse < 1e300 && lse > -1e300); }

// One workgroup per item, all its logits in registers: `per` waves a beam.
template <bool F32, int VEC, int PER> __global__ __launch_bounds__(kSmallThreads) void select_small_kernel(BeamSelectParams p, int per) {
    __shared__ Hits hits;
    __shared__ float smax[16];
    __shared__ double ssum[16];
    __shared__ uint32_t keys[kSmallThreads];
    __shared__ uint8_t kinds[kMaxBeams];
    __shared__ uint64_t limit[kMaxBeams];
    __shared__ Cand part[16];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, b = blockIdx.x;
    const int w = wave / per, first = w * per, t = threadIdx.x - first * 64, threads = per * 64;
    const bool on = w < p.W;
    const int64_t row = (int64_t)b * p.W + (on ? w : 0);
    RowRegs<F32, VEC, PER> r;
    r.load(p.logits, row * p.row, on ? p.V : 0, t, threads);       // a finished beam's too: nothing waits on done
    const bool fin = on && p.done && p.done[row];
    const double score = beam_score(p, row);
    const float lane_max = r.max();
    const float wm = wave_max_dpp(lane_max);
    const double sum = wave_sum_f64(r.sum(wm));
    if (lane == 0) {
        smax[wave] = wm;
        ssum[wave] = sum;
    }
    if (threadIdx.x == 0) hits.n = 0;
    __syncthreads();
    // lane i < per joins wave i of the beam
    const float om = on && lane < per ? smax[first + lane] : -INFINITY;
    const float m = wave_max_dpp(om);
    const double os = on && lane < per ? ssum[first + lane] : 0.0;
    const double s = wave_sum_f64(om == m ? os : os * exp((double)om - (double)m));
    const double lse = (double)m + log(s);
    const int kind = fin ? BEAM_DONE : is_dead(score, lse) ? BEAM_DEAD : BEAM_LIVE;
    if (on && t == 0) kinds[w] = (uint8_t)kind;
    // a dead beam's words have equal keys: they rank by the word
    auto key_of = [&](float x) { return kind == BEAM_DEAD ? 1u : order_bits(x); };
    auto score_of = [&](float x) { return kind == BEAM_DEAD ? -INFINITY : score + ((double)x - lse); };
    uint32_t best = 0;
    if (fin) best = t == 0 ? order_bits((float)score) : 0u;
    else if (r.any()) best = order_bits((float)score_of(lane_max));
    keys[threadIdx.x] = best;
    __syncthreads();
    const uint32_t R = reach_of_block<16>(keys, p.W);
    if (best >= R) {
        if (fin) {
            add_hit(hits, Cand{score, in_beam(~0u, p.end_id), w});
        } else {
            r.each([&](float x, int v) {
                const double c = score_of(x);
                if (order_bits((float)c) >= R) add_hit(hits, Cand{c, in_beam(key_of(x), v), w});
            });
        }
    }
    __syncthreads();
    if (hits.n <= kHits) {
        rank_hits(p, b, hits, kinds);
        return;
    }
    if (threadIdx.x < p.W) limit[threadIdx.x] = ~0ull;
    __syncthreads();
    for (int k = 0; k < p.W; ++k) {
        Cand x = {0.0, 0, w};
        if (fin && t == 0) x = Cand{score, in_beam(~0u, p.end_id), w};
        if (on && !fin) {
            float xv = 0.f;
            const uint64_t most = limit[w];
            r.each([&](float v, int word) {
                asm volatile("" : "+v"(v));     // formed anew each round, not kept for all registers
                const uint64_t in = in_beam(key_of(v), word);
                if (in < most && in > x.in) {
                    x.in = in;
                    xv = v;
                }
            });
            x.c = score_of(xv);
        }
        if (on && x.in >= limit[w]) x.in = 0;
        const Cand top = block_best<16>(x, part);
        if (threadIdx.x == 0) {
            put_out(p, b, k, top, kinds[top.w]);
            limit[top.w] = top.in;
        }
        __syncthreads();
    }
}

// One workgroup per chunk of a row: its maximum, sum and candidates.  Chunks of up
// to 8192 logits, read once, all loads in flight at once; 512 rows of 32769 f32 take
// 17.9 us, two thirds of it VALU issue (an exponential and an f64 sum per logit).
template <bool F32, int VEC, int PER> __global__ __launch_bounds__(kRowThreads) void select_rows_kernel(BeamSelectParams p, SelectWork ws) {
    __shared__ float smax[4];
    __shared__ double ssum[4];
    __shared__ uint32_t keys[kRowThreads];
    __shared__ int count;
    __shared__ Cand part[4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, t = threadIdx.x;
    const int64_t unit = xcd_tile(blockIdx.x, gridDim.x), row = unit / ws.chunks;
    if (p.done && p.done[row]) return;                       // its one candidate needs no logits
    const int base = (int)(unit - row * ws.chunks) * ws.len;
    const int n = p.V - base < ws.len ? p.V - base : ws.len;
    RowRegs<F32, VEC, PER> r;
    r.load(p.logits, row * p.row + base, n, t, kRowThreads);
    const float lane_max = r.max();
    const float wm = wave_max_dpp(lane_max);
    const uint32_t best = r.any() ? order_bits(lane_max) : 0u;
    keys[t] = best;
    if (lane == 0) smax[wave] = wm;
    if (t == 0) count = 0;
    __syncthreads();
    const float m = fmaxf(fmaxf(smax[0], smax[1]), fmaxf(smax[2], smax[3]));
    const uint32_t R = reach_of_block<4>(keys, p.W);
    const double sum = wave_sum_f64(r.sum(m));
    if (lane == 0) ssum[wave] = sum;
    Entry* list = ws.list + unit * kList;
    if (best >= R) {
        const float least = order_value(R);
        r.each([&](float x, int v) {
            if (!(x >= least)) return;
            const int at = atomicAdd(&count, 1);
            if (at < kList) list[at] = Entry{order_bits(x), base + v};
        });
    }
    __syncthreads();
    int listed = count;
    if (listed > kList) {      // too many ties: the W best one by one
        uint64_t limit = ~0ull;
        listed = p.W < n ? p.W : n;
        for (int k = 0; k < listed; ++k) {
            Cand x = {0.0, 0, 0};
            r.each([&](float v, int word) {
                asm volatile("" : "+v"(v));     // formed anew each round, not kept for all registers
                const uint64_t in = in_beam(order_bits(v), word);
                if (in < limit && in > x.in) x.in = in;
            });
            limit = block_best<4>(x, part).in;
            if (t == 0) list[k] = Entry{(uint32_t)(limit >> 32), base + (int)~(uint32_t)limit};
        }
    }
    if (t == 0) ws.stat[unit] = ChunkStat{m, listed, (ssum[0] + ssum[1]) + (ssum[2] + ssum[3])};
}

// One workgroup per item over its chunks' lists: a chain of dependent steps (statistics,
// f64 exponentials and a logarithm, bound, ranking) of 6.6 us for 8 beams x 2 chunks, 8.9
// for 16 x 5, however many items there are up to the chip's 256 CUs.
__global__ __launch_bounds__(kItemThreads) void select_item_kernel(BeamSelectParams p, SelectWork ws) {
    constexpr int WAVES = kItemThreads / 64;
    __shared__ Hits hits;
    __shared__ double lse[kMaxBeams], score[kMaxBeams];
    __shared__ uint32_t keys[kItemThreads];
    __shared__ uint8_t kinds[kMaxBeams];
    __shared__ uint64_t limit[kMaxBeams];
    __shared__ Cand part[WAVES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, b = blockIdx.x, W = p.W, lists = W * ws.chunks;
    const ChunkStat* stat = ws.stat + (int64_t)b * lists;
    const Entry* list = ws.list + (int64_t)b * lists * kList;
    // the first entries of the wave's first kHeld lists, in flight while the sums are joined
    constexpr int kHeld = 8;
    Entry held[kHeld];
    int len[kHeld];
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        const int i = wave + k * WAVES;
        held[k] = Entry{0, 0};
        len[k] = 0;
        if (i < lists) {
            held[k] = list[(int64_t)i * kList + lane];  // past the list's end: anything, not used
            len[k] = stat[i].n;
        }
    }
    {   // 16 lanes a beam
        const int w = threadIdx.x >> 4, l = threadIdx.x & 15;
        const int64_t row = (int64_t)b * W + w;
        const bool fin = w < W && p.done && p.done[row];
        const bool read = w < W;       // (a finished beam's are anything, and not used)
        float m = -INFINITY;
        double s = 0.0;
        // the running maximum and sum over the lane's chunks, then over the lanes
        for (int i = l; read && i < ws.chunks; i += 16) {
            const ChunkStat x = stat[w * ws.chunks + i];
            const float hi = fmaxf(m, x.max);
            if (hi != -INFINITY) s = s * exp((double)m - (double)hi) + x.sum * exp((double)x.max - (double)hi);
            else s += x.sum;
            m = hi;
        }
        float g = m;
        g = fmaxf(g, dpp_get<0xB1>(g));
        g = fmaxf(g, dpp_get<0x4E>(g));
        g = fmaxf(g, dpp_get<0x141>(g));
        g = fmaxf(g, dpp_get<0x140>(g));
        s = row16_sum_f64(g != -INFINITY ? s * exp((double)m - (double)g) : s);
        if (l == 0 && w < W) {
            const double sc = beam_score(p, row), z = (double)g + log(s);
            score[w] = sc;
            lse[w] = z;
            kinds[w] = (uint8_t)(fin ? BEAM_DONE : is_dead(sc, z) ? BEAM_DEAD : BEAM_LIVE);
            limit[w] = ~0ull;
        }
    }
    if (threadIdx.x == 0) hits.n = 0;
    __syncthreads();
    // the held lists' candidates, in registers; their second 64 entries, the
    // other lists and the beams without lists are formed when asked for
    Cand mine[kHeld];
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        const int i = wave + k * WAVES;
        mine[k] = Cand{0.0, 0, 0};
        if (i >= lists) continue;
        const int w = udiv_small(i, ws.chunks);
        len[k] = kinds[w] == BEAM_LIVE ? len[k] : 0;
        mine[k] = Cand{score[w] + ((double)order_value(held[k].key) - lse[w]), lane < len[k] ? in_beam(held[k].key, held[k].v) : 0, w};
    }
    // calls f with every candidate of this thread
    auto each = [&](auto&& f) {
        auto listed = [&](int i, int w, int j) {
            const Entry e = list[(int64_t)i * kList + j];
            f(Cand{score[w] + ((double)order_value(e.key) - lse[w]), in_beam(e.key, e.v), w});
        };
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            if (mine[k].in) f(mine[k]);
            if (lane + 64 < len[k]) listed(wave + k * WAVES, mine[k].w, lane + 64);
        }
        for (int i = wave + kHeld * WAVES; i < lists; i += WAVES) {
            const int w = udiv_small(i, ws.chunks);
            if (kinds[w] != BEAM_LIVE) continue;
            const int n = stat[i].n;
            for (int j = lane; j < n; j += 64) listed(i, w, j);
        }
        for (int w = wave; w < W; w += WAVES) {
            if (kinds[w] == BEAM_DONE && lane == 0) f(Cand{score[w], in_beam(~0u, p.end_id), w});
            if (kinds[w] == BEAM_DEAD && lane < W && lane < p.V) f(Cand{-INFINITY, in_beam(1u, lane), w});
        }
    };
    uint32_t best = 0;
    each([&](const Cand& x) {
        const uint32_t k = order_bits((float)x.c);
        best = k > best ? k : best;
    });
    keys[threadIdx.x] = best;
    __syncthreads();
    const uint32_t R = reach_of_block<WAVES>(keys, W);
    each([&](const Cand& x) {
        if (order_bits((float)x.c) >= R) add_hit(hits, x);
    });
    __syncthreads();
    if (hits.n <= kHits) {
        rank_hits(p, b, hits, kinds);
        return;
    }
    for (int k = 0; k < W; ++k) {
        Cand x = {0.0, 0, 0};
        each([&](const Cand& y) {
            if (y.in < limit[y.w] && before(y, x)) x = y;
        });
        const Cand best_of = block_best<WAVES>(x, part);
        if (threadIdx.x == 0) {
            put_out(p, b, k, best_of, kinds[best_of.w]);
            limit[best_of.w] = best_of.in;
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

// All states in one launch: rows x states x pieces.  4 states of 2560 bytes x 128 rows
// 2.9 us, near an empty launch.
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

// waves a beam where an item fits one workgroup's registers, 0 where it does not.
// One launch against two, us: 1 item x 4 beams x 1025 words 6.4 and 8.6, 16 x 4 x 4096
// 9.4 and 10.8, 16 x 16 x 1024 11.2 and 11.8; with 32 logits a lane 16 x 4 x 8192 took
// 13.8 and 11.6, so 16 is the limit.
int small_waves(const BeamSelectParams& p) {
    if (p.W > 16) return 0;
    const int per = 16 / p.W;
    return p.V <= per * 64 * kSmallPer ? per : 0;
}

SelectWork select_work(const BeamSelectParams& p) {
    SelectWork w = {};
    w.chunks = cdiv(p.V, kChunk);
    w.len = (cdiv(p.V, w.chunks) + 7) / 8 * 8;       // about equal chunks
    return w;
}

}  // namespace

size_t beam_select_workspace(const BeamSelectParams& p) {
    if (p.B == 0 || small_waves(p)) return 0;
    return (size_t)p.B * p.W * select_work(p).chunks * (sizeof(ChunkStat) + kList * sizeof(Entry));
}

void launch_beam_select(const BeamSelectParams& p, void* ws, size_t ws_bytes, hipStream_t s) {
    if (p.B == 0) return;
    const int wide = p.f32 ? 4 : 8;
    require(p.B < (1 << 22), "beam select: at most 2^22 items in one call");
    if (const int per = small_waves(p)) {
        const int threads = per * 64;
        auto* k = p.V < threads * wide ? (p.f32 ? select_small_kernel<true, 1, kFew> : select_small_kernel<false, 1, kFew>)
                  : !p.f32             ? select_small_kernel<false, 8, kSmallPer>
                                       : p.V <= threads * kFew ? select_small_kernel<true, 4, kFew> : select_small_kernel<true, 4, kSmallPer>;
        launch(k, dim3(p.B), dim3(kSmallThreads), 0, s, p, per);
        return;
    }
    const size_t need = beam_select_workspace(p);
    require(ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= need,
            "beam select: the workspace is smaller than its size query says, or not 16-byte aligned");
    SelectWork w = select_work(p);
    const size_t lists = (size_t)p.B * p.W * w.chunks;
    require(lists < ((size_t)1 << 23), "beam select: too many beams and words for one call");
    w.stat = (ChunkStat*)ws;
    w.list = (Entry*)((char*)ws + lists * sizeof(ChunkStat));
    auto* k = p.V < kRowThreads * wide ? (p.f32 ? select_rows_kernel<true, 1, kFew> : select_rows_kernel<false, 1, kFew>)
              : !p.f32                 ? select_rows_kernel<false, 8, kPer>
                                       : w.len <= kRowThreads * kFew ? select_rows_kernel<true, 4, kFew> : select_rows_kernel<true, 4, kPer>;
    launch(k, dim3((unsigned)lists), dim3(kRowThreads), 0, s, p, w);
    launch(select_item_kernel, dim3(p.B), dim3(kItemThreads), 0, s, p, w);
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
    int64_t z = (most + 1023) / 1024;                        // four pieces a thread
    z = z > 64 ? 64 : z;
    launch(reorder_kernel, dim3((unsigned)p.rows, p.n, (unsigned)z), dim3(256), 0, s, p);
}

}  // namespace pkx
