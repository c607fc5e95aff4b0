// Attention of a decoder's queries to keys of another length: encoder states
// in f16 or f32, or an 8-bit cache (int8 with a scale for each 32 tokens and
// head).  One pass over the keys with the running maximum m and sum l of the
// softmax: for a tile of keys, m' = max(m, max s), a = 2^(m - m'),
// p = 2^(s - m'), l = a l + sum p, O = a O + p V; out = O / l, zeros where no
// key was attended (l = 0).  s is in log2 units (log2 e folded into the scale).
//
// Everything stays in registers.  Both products are formed transposed on
// 16-row matrix instructions, so that a lane's column is one query:
// S^T = K Q^T leaves lane (c, g) (c = lane % 16, g = lane / 16) the scores of
// query c with keys 4g + e and 16 + 4g + e of a 32-key tile, which is already
// the B operand of O^T = V^T P^T when that product's contraction index (g, i)
// stands for key 4g + i (i < 4) or 16 + 4g + i - 4.  Its A operand wants eight
// keys of one dimension per lane while V is stored by key, so each lane loads
// dimensions [c D/16, (c+1) D/16) of its eight keys (the 16 lanes of a group
// read one whole row) and pairs of rows are interleaved with v_perm: row c of
// the j-th product is dimension c D/16 + j, and a lane ends with runs of D/16
// consecutive output dimensions.  No LDS but for joining waves.
//
// A workgroup is four waves with a share of the keys each, joined in LDS at the
// end.  Where a call has few rows the keys are also split over workgroups, each
// writing its unnormalised O and (m, l), and dec_join_kernel joins them.
//
// 8-bit keys: the int8 go through v_perm into f16 mantissas
// (0x6400 | (b ^ 0x80) = 1024 + b + 128, minus 1152: exact), the scale of a
// block multiplies the scores and the tile's P V product in f32.  With f32
// queries, q and p are split into two f16 terms of 22 bits together, so the
// int8 products keep f32's accuracy at twice the matrix instructions (the f32 ones
// have a sixteenth of the f16 ones' rate).
//
// Measured, us (a copy moves 5.1 TB/s, a launch that does nothing takes 2.5 to 3):
//   f16 1 row x 8 heads x 64, 125 keys                     4.4   launch, dependent loads
//   f16 16 x 4 rows x 8 heads x 128, up to 375 keys        7.8   15 MB at 2.0 TB/s; latency
//   f16 4 x 8 rows x 16 (8) heads x 64, 3750 keys         10.0 + 3.9 to join: 31 MB, 3.1 TB/s
//   f32 3 x 37 rows x 8 heads x 64, up to 211 keys         8.0   latency, matrix pipe
//   int8 128 beams x 8 heads x 64, up to 448 keys, table  14.3   VALU issue 68%
//   int8 4 rows x 16 (4) heads x 128, up to 32768 keys    23.4 + 4.7 to join: 92 MB, 3.9 TB/s
//   int8, f32 8 x 200 rows x 8 heads x 64, up to 1025     19.0   VALU issue 65%: conversions
#include "decoder.hpp"

namespace pkx {
namespace {

constexpr double kLog2e = 1.4426950408889634;
constexpr float kNoMax = -3.0e38f;   // below every score: m - m' is finite from the start

__device__ __forceinline__ float xgroup_max(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float xgroup_sum(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// v_max3_f32 as it is: the compiler puts a canonicalising v_max before every
// fmaxf of a matrix product's result.  It keeps no waits around inline assembly
// either: matrix products go through settled() first, and what comes out through an
// ordinary instruction before a lane swap reads it.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ float max8(float4v x, float4v y) {
    return max3(max3(x[0], x[1], x[2]), max3(x[3], y[0], y[1]), max3(y[2], y[3], y[3]));
}
// 20 wait states, enough for the longest matrix instruction's result (19)
__device__ __forceinline__ void settled(float4v (&s)[2][4]) {
    asm("s_nop 15\n\ts_nop 3"
        : "+v"(s[0][0]), "+v"(s[0][1]), "+v"(s[0][2]), "+v"(s[0][3]), "+v"(s[1][0]), "+v"(s[1][1]), "+v"(s[1][2]), "+v"(s[1][3]));
}

// bits 0 .. n - 1
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

// x / d for scalars below 2^22
__device__ __forceinline__ int uniform_div(int x, int d) { return __builtin_amdgcn_readfirstlane(udiv_small(x, d)); }

// int8 pairs spread to the low bytes of two halves -> f16
__device__ __forceinline__ uint32_t i8_pair_f16(uint32_t spread) {
    const half2v h = __builtin_bit_cast(half2v, spread ^ 0x64806480u) + (half2v){(f16)-1152.0f, (f16)-1152.0f};
    return __builtin_bit_cast(uint32_t, h);
}

template <int N> __device__ __forceinline__ void load_words(uint32_t (&d)[N], const uint8_t* p) {
    if constexpr (N == 1) {
        d[0] = *(const uint32_t*)p;
    } else if constexpr (N == 2) {
        const int2v t = *(const int2v*)p;
        d[0] = t[0]; d[1] = t[1];
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const int4v t = *(const int4v*)(p + 4 * i);
            d[i] = t[0]; d[i + 1] = t[1]; d[i + 2] = t[2]; d[i + 3] = t[3];
        }
    }
}

// Registers of a 32-key tile: key tiles kt = 0, 1 of 16 keys (lane c's row),
// and the lane's eight value rows.
template <int KV, int D> struct Tile {
    static constexpr int ES = KV == KV_F16 ? 2 : KV == KV_F32 ? 4 : 1;
    static constexpr int NK = D * ES / 16;                        // dwords of a lane's quarter of a key row
    static constexpr int NV = D * ES / 64 > 0 ? D * ES / 64 : 1;  // dwords of its sixteenth of a value row
    uint32_t k[2][NK];
    uint32_t v[8][NV];
    float ks, vs;    // scales of the block, or (table) of key lane % 32
    int ok;          // key lane % 32 is attended
};

// byte offset in a key row of the n-th 16-byte (or narrower) piece of group g
template <int KV, int D> __device__ __forceinline__ int key_piece(int n, int g) {
    if constexpr (KV == KV_I8 && D == 32) return 8 * g;
    return 64 * n + 16 * g;
}
// dimension of element x of group g's fragment of contraction step s (32 deep)
template <int KV, int D> __device__ __forceinline__ int key_dim(int s, int g) {
    if constexpr (KV == KV_I8 && D > 32) return 64 * (s >> 1) + 16 * g + 8 * (s & 1);
    return 32 * s + 8 * g;
}

struct KeySource {
    const uint8_t *k, *v;        // item and head
    uint32_t k_row, v_row;       // bytes between keys
    const float *ks, *vs;
    const uint8_t* mask;
    int T, k_bytes;
    uint32_t v_at;               // the lane's first value row and dimension, from a tile's first row
    uint32_t k_at[8];            // its pieces of key row c
    // table
    const int* table;
    int n_slots;
    int64_t k_slot, s_slot;      // bytes and scales between slots (keys and values alike)
    bool far;                    // a slot's offset may not fit 32 bits
    uint32_t span;               // otherwise: bytes from k (and v) to the last slot's end
};

// A buffer resource of one step's rows, built from scalars.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t step_rsrc(const uint8_t* base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, (int)bytes, 0x00020000);
}

// n dwords at a byte offset.  All of it goes into the per-lane offset, which is
// what the range check compares with the resource's size (a scalar offset is
// subtracted from the size first, and a larger one would wrap).
template <int N, typename R> __device__ __forceinline__ void buffer_words(uint32_t (&d)[N], R r, uint32_t at) {
    if constexpr (N == 1) {
        d[0] = __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0);
    } else if constexpr (N == 2) {
        const int2v x = __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0);
        d[0] = x[0]; d[1] = x[1];
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const int4v x = __builtin_amdgcn_raw_buffer_load_b128(r, at + 4 * i, 0, 0);
            d[i] = x[0]; d[i + 1] = x[1]; d[i + 2] = x[2]; d[i + 3] = x[3];
        }
    }
}

// The rows of a tile come through a buffer resource of exactly the tile's valid
// rows, built from scalars: offsets are the same in every tile, and rows past the
// last key read as zeros.
template <int KV, int D>
__device__ __forceinline__ void load_tile(Tile<KV, D>& t, const KeySource& s, int t0, int lane) {
    using TL = Tile<KV, D>;
    const int last = s.T - 1, tb = t0 < last ? t0 : last;          // tiles past the end read the last key again
    const int left = last - tb, rows = left < 31 ? left : 31, mine = lane & 31;
    bool ok = t0 + mine < s.T;
    if (s.mask) ok = ok && s.mask[tb + (mine < left ? mine : left)] != 0;
    t.ok = ok;
    if constexpr (KV == KV_I8) {
        t.ks = s.ks[tb / kCacheBlock];
        t.vs = s.vs[tb / kCacheBlock];
    }
    const auto kr = step_rsrc(s.k + (int64_t)tb * s.k_row, rows * s.k_row + s.k_bytes);
    const auto vr = step_rsrc(s.v + (int64_t)tb * s.v_row, rows * s.v_row + s.k_bytes);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
        constexpr int N = TL::NK == 2 ? 2 : 4;
#pragma unroll
        for (int n = 0; n < TL::NK / N; ++n) {
            uint32_t d[N];
            buffer_words(d, kr, s.k_at[n] + 16 * kt * s.k_row);
#pragma unroll
            for (int i = 0; i < N; ++i) t.k[kt][N * n + i] = d[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t at = s.v_at + (i < 4 ? i : 12 + i) * s.v_row;
        if constexpr (KV == KV_I8 && D == 32) t.v[i][0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(vr, at, 0, 0);
        else buffer_words(t.v[i], vr, at);
    }
}

// The same with every key's slot from the table: lane l (mod 32) forms key l's
// offset, the lanes that read its row fetch it from there.
template <int D> __device__ __forceinline__ void load_tile_by_table(Tile<KV_I8, D>& t, const KeySource& s, int t0, int slot, int lane) {
    using TL = Tile<KV_I8, D>;
    const int c = lane & 15, g = lane >> 4, last = s.T - 1, tb = t0 < last ? t0 : last;
    const int left = last - tb, mine = lane & 31, row = mine < left ? mine : left;
    const bool in = (unsigned)slot < (unsigned)s.n_slots;
    t.ok = t0 + mine < s.T && in;
    slot = in ? slot : 0;
    t.ks = s.ks[slot * s.s_slot + tb / kCacheBlock];
    t.vs = s.vs[slot * s.s_slot + tb / kCacheBlock];
    if (!s.far) {        // through resources of all slots, offsets of 32 bits
        const uint32_t mine_at = (uint32_t)slot * (uint32_t)s.k_slot + (tb + row) * s.k_row;
        const auto kr = step_rsrc(s.k, s.span), vr = step_rsrc(s.v, s.span);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            constexpr int N = TL::NK == 2 ? 2 : 4;
            const uint32_t at = (uint32_t)__shfl((int)mine_at, 16 * kt + c, 64);
#pragma unroll
            for (int n = 0; n < TL::NK / N; ++n) {
                uint32_t d[N];
                buffer_words(d, kr, at + s.k_at[n]);
#pragma unroll
                for (int i = 0; i < N; ++i) t.k[kt][N * n + i] = d[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t at = (uint32_t)__shfl((int)mine_at, (i < 4 ? 0 : 12) + 4 * g + i, 64) + s.v_at;
            if constexpr (D == 32) t.v[i][0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(vr, at, 0, 0);
            else buffer_words(t.v[i], vr, at);
        }
        return;
    }
    const int64_t mine_at = slot * s.k_slot + (int64_t)(tb + row) * s.k_row;
    auto from = [&](int r) {
        return (int64_t)((uint64_t)(uint32_t)__shfl((int)(mine_at >> 32), r, 64) << 32 | (uint32_t)__shfl((int)mine_at, r, 64));
    };
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
        constexpr int N = TL::NK == 2 ? 2 : 4;
        const uint8_t* x = s.k + from(16 * kt + c);
#pragma unroll
        for (int n = 0; n < TL::NK / N; ++n) {
            uint32_t d[N];
            load_words(d, x + s.k_at[n]);
#pragma unroll
            for (int i = 0; i < N; ++i) t.k[kt][N * n + i] = d[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint8_t* x = s.v + from((i < 4 ? 0 : 12) + 4 * g + i) + s.v_at;
        if constexpr (D == 32) t.v[i][0] = *(const uint16_t*)x;
        else load_words(t.v[i], x);
    }
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const half2v h = {(f16)a, (f16)b};
    return __builtin_bit_cast(uint32_t, h);
}
// Two values as pairs of f16 terms: what the rounding leaves is exact in f32.  The first
// terms are formed twice, and once from a product fused into the conversion they could
// differ by one of their steps, so either they are taken from their register (fewer
// instructions: 8 prompts of 200 rows 18.6 us, so 17.6) or the values are (fewer
// registers, where all are in use).
template <bool VALUES> __device__ __forceinline__ void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
    if constexpr (VALUES) asm("" : "+v"(a), "+v"(b));
    hi = pack_f16(a, b);
    if constexpr (!VALUES) asm("" : "+v"(hi));
    const half2v h = __builtin_bit_cast(half2v, hi);
    lo = pack_f16(fmaf((float)h[0], -1.0f, a), fmaf((float)h[1], -1.0f, b));
}

// Row m of an item and key head as lane group g's fragments (LAYOUT: the kind
// of keys whose order of dimensions they meet); returns its query index.  Rows past the queries are zeros.
template <int KV, bool QF32, int D, int LAYOUT, int NQ>
__device__ __forceinline__ int load_query(const DecAttnParams& p, int m, int b, int kh, int cnt, int g, uint32_t (&q)[NQ], float& qf, float& qf_lo) {
    const int i = udiv_small(m, p.G), h = kh * p.G + (m - i * p.G);
    const bool live = i < cnt;
    // rows past the queries and pieces past the head's dimensions read another
    // row's or piece instead and become zeros: the loads wait on no branch
    const int64_t at = b * p.q_item + (live ? i * p.q_row : 0) + h * p.q_head;
    qf = p.scale;
    qf_lo = p.scale_lo;
    if constexpr (KV == KV_F32) {
        float4v x[D / 16];
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
            const int d = 16 * n + 4 * g;
            x[n] = *(const float4v*)((const float*)p.q + at + (d < p.dk ? d : 0));
        }
#pragma unroll
        for (int n = 0; n < D / 16; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) q[4 * n + e] = live && 16 * n + 4 * g < p.dk ? __float_as_uint(x[n][e]) : 0u;
    } else if constexpr (!QF32) {
        int4v x[D / 32];
#pragma unroll
        for (int n = 0; n < D / 32; ++n) {
            const int d = key_dim<LAYOUT, D>(n, g);
            x[n] = *(const int4v*)((const f16*)p.q + at + (d < p.dk ? d : 0));
        }
#pragma unroll
        for (int n = 0; n < D / 32; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) q[4 * n + e] = live && key_dim<LAYOUT, D>(n, g) < p.dk ? x[n][e] : 0;
    } else {
        // q = (hi + lo) / f with f the power of two that takes the row's
        // largest value to [2^13, 2^14): hi has 11 bits, lo the next 11, so
        // that at most 2^-23 of a value is dropped, or 2^-38 of the
        // largest where lo is subnormal
        float4v y[D / 32][2];
#pragma unroll
        for (int n = 0; n < D / 32; ++n) {
            const int d = key_dim<LAYOUT, D>(n, g);
            const float* src = (const float*)p.q + at + (d < p.dk ? d : 0);
            y[n][0] = *(const float4v*)src;
            y[n][1] = *(const float4v*)(src + 4);
        }
        float x[D / 32][8], top = 0.f;
#pragma unroll
        for (int n = 0; n < D / 32; ++n) {
            const bool in = live && key_dim<LAYOUT, D>(n, g) < p.dk;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[n][e] = in ? y[n][e >> 2][e & 3] : 0.f;
                top = fmaxf(top, fabsf(x[n][e]));
            }
        }
        top = xgroup_max(top);
        int ex = 0;
        (void)frexpf(top, &ex);                        // top = [1/2, 1) 2^ex
        ex = ex < -100 ? -100 : ex;
        const float f = ldexpf(1.0f, 14 - ex);
        qf *= ldexpf(1.0f, ex - 14);
        qf_lo *= ldexpf(1.0f, ex - 14);
#pragma unroll
        for (int n = 0; n < D / 32; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) split_f16<false>(x[n][2 * e] * f, x[n][2 * e + 1] * f, q[4 * n + e], q[D / 8 + 4 * n + e]);
    }
    return i;
}

// scores of a 16-key tile (c: keys 4g + e of query lane % 16)
template <int KV, int D, bool QF32, int NQ>
__device__ __forceinline__ float4v tile_scores(const uint32_t (&k)[Tile<KV, D>::NK], const uint32_t (&q)[NQ]) {
    float4v acc = {0.f, 0.f, 0.f, 0.f};
    if constexpr (KV == KV_F32) {      // two sums of half the length, for their rounding
        float4v odd = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < D / 4; i += 2) {
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[i]), __uint_as_float(q[i]), acc, 0, 0, 0);
            odd = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[i + 1]), __uint_as_float(q[i + 1]), odd, 0, 0, 0);
        }
        acc += odd;
    } else {
        // (the second terms' products first: the sum is rounded at its full size in
        // those of the first only)
        half8v a[D / 32];
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            int4v w;
            if constexpr (KV == KV_F16) {
                w = (int4v){(int)k[4 * s], (int)k[4 * s + 1], (int)k[4 * s + 2], (int)k[4 * s + 3]};
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    w[2 * h] = i8_pair_f16(__builtin_amdgcn_perm(0, k[2 * s + h], 0x0c010c00));
                    w[2 * h + 1] = i8_pair_f16(__builtin_amdgcn_perm(0, k[2 * s + h], 0x0c030c02));
                }
            }
            a[s] = __builtin_bit_cast(half8v, w);
        }
#pragma unroll
        for (int part = KV == KV_I8 && QF32 ? 1 : 0; part >= 0; --part)
#pragma unroll
            for (int s = 0; s < D / 32; ++s) {
                const int o = part * (D / 8) + 4 * s;
                const int4v b = {(int)q[o], (int)q[o + 1], (int)q[o + 2], (int)q[o + 3]};
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[s], __builtin_bit_cast(half8v, b), acc, 0, 0, 0);
            }
    }
    return acc;
}

// A operand of the j-th value product: eight keys of dimension c D/16 + j
template <int KV, int D> __device__ __forceinline__ half8v value_frag(const uint32_t (&v)[8][Tile<KV, D>::NV], int j) {
    int4v a;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (KV == KV_F16) {
            a[i] = __builtin_amdgcn_perm(v[2 * i + 1][j >> 1], v[2 * i][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
        } else {
            const uint32_t b = j & 3;
            a[i] = i8_pair_f16(__builtin_amdgcn_perm(v[2 * i + 1][j >> 2], v[2 * i][j >> 2], 0x0c040c00u | b | (b << 16)));
        }
    }
    return __builtin_bit_cast(half8v, a);
}

// Block -> work.  Block n runs on XCD n % 8.  The row tiles of one split, item
// and key head read the same keys and stay on one XCD; eight neighbouring ones of
// these go to the eight XCDs, each eight turned by one against the last, so that no
// XCD gets all of a long item or of a split that most items do not reach (whole
// items to an XCD: 8 prompts of 200 rows on up to 1025 tokens, f32, 22.8 us; so
// 18.4).  The last ones, where they are no multiple of 8, are spread over the XCDs.
// With a table neighbouring items share keys, and each XCD takes a range of them.
template <bool TABLE>
__device__ __forceinline__ void work_of(int bid, const DecAttnParams& p, int mt, int& b, int& kh, int& split, int& mtile) {
    const int units = p.B * p.Hkv, total = units * p.splits, even = (total >> 3) * 8 * mt;
    int u;
    if (TABLE || bid >= even) {
        const int at = TABLE ? xcd_tile(bid, total * mt) : bid;
        u = uniform_div(at, mt);
        mtile = at - u * mt;
    } else {
        const int loc = bid >> 3, r = uniform_div(loc, mt);
        u = r * 8 + ((bid + r) & 7);
        mtile = loc - r * mt;
    }
    split = uniform_div(u, units);
    u -= split * units;
    b = uniform_div(u, p.Hkv);
    kh = u - b * p.Hkv;
}

// Workgroups to a CU: as many as the registers allow without spilling (f32,
// d_head 128, 54 rows x 334 keys x 56 heads: 25.4 us at one, 22.1 at two (20.3 by now); f32, 64: one
// more than three spills, 18.1 -> 19.4).
constexpr int attn_wgs(int kv, int d) { return d > 64 ? 2 : kv == KV_F32 && d > 32 ? 3 : 4; }

template <int KV, bool QF32, int D, bool TABLE>
__global__ __launch_bounds__(256, attn_wgs(KV, D)) void dec_attn_kernel(DecAttnParams p) {
    using TL = Tile<KV, D>;
    constexpr bool SPLIT = KV == KV_I8 && QF32;            // q and p as two f16 terms
    constexpr int NQ = KV == KV_F32 ? D / 4 : SPLIT ? D / 4 : D / 8;
    constexpr int NJ = D / 16, WK = 4, ROWS = 16;
    const int lane = threadIdx.x & 63, wk = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int M = p.n_q * p.G, mt = (M + ROWS - 1) / ROWS;
    int b, kh, split, mtile;
    work_of<TABLE>(blockIdx.x, p, mt, b, kh, split, mtile);

    int T = p.k_len ? p.k_len[b] : p.n_k;
    T = T < 0 ? 0 : T > p.n_k ? p.n_k : T;
    int cnt = p.q_len ? p.q_len[b] : p.n_q;
    cnt = cnt < 0 ? 0 : cnt > p.n_q ? p.n_q : cnt;
    if (uniform_div(mtile * ROWS, p.G) >= cnt) return;                 // no row of this tile is asked for
    const int m0 = mtile * ROWS;
    KeySource s = {};
    s.k_row = (uint32_t)p.k_row * TL::ES;
    s.v_row = (uint32_t)p.v_row * TL::ES;
    s.k_bytes = p.dk * TL::ES;
    if constexpr (KV == KV_I8) {
        int sl = TABLE ? 0 : p.slot ? p.slot[b] : b;
        if ((unsigned)sl >= (unsigned)p.n_slots) {
            sl = 0;
            T = 0;
        }
        s.s_slot = (int64_t)p.Hkv * p.n_blocks;
        s.k = (const uint8_t*)p.k + sl * p.k_item + kh * p.k_head;
        s.v = (const uint8_t*)p.v + sl * p.v_item + kh * p.v_head;
        s.ks = p.k_scale + sl * s.s_slot + (int64_t)kh * p.n_blocks;
        s.vs = p.v_scale + sl * s.s_slot + (int64_t)kh * p.n_blocks;
        if constexpr (TABLE) {
            s.table = p.table + b * p.table_ld;
            s.n_slots = p.n_slots;
            s.k_slot = p.k_item;
            s.far = p.n_slots * p.k_item > 0x7fffffffll;
            s.span = (uint32_t)(p.n_slots * p.k_item - kh * p.k_head);
        }
    } else {
        s.k = (const uint8_t*)p.k + (b * p.k_item + kh * p.k_head) * TL::ES;
        s.v = (const uint8_t*)p.v + (b * p.v_item + kh * p.v_head) * TL::ES;
        s.mask = p.mask ? p.mask + b * p.mask_item : nullptr;
    }
    s.T = T;
    // pieces past the head's dimensions read its first again (their queries are
    // zero; their output is not stored); with the table the row comes separately
#pragma unroll
    for (int n = 0; n < (TL::NK + 3) / 4; ++n) {
        const int o = key_piece<KV, D>(n, g);
        s.k_at[n] = (TABLE ? 0 : c * s.k_row) + (o < s.k_bytes ? o : 0);
    }
    s.v_at = (TABLE ? 0 : 4 * g * s.v_row) + (c * NJ < p.dk ? c * NJ : 0) * TL::ES;

    // queries: B operand, column c = row m0 + c
    uint32_t q[NQ];
    float qf, qf_lo;     // factor of the scores, what its rounding left
    const int qi = load_query<KV, QF32, D, KV>(p, m0 + c, b, kh, cnt, g, q, qf, qf_lo);
    const int lim = p.causal ? T - cnt + qi + 1 : T;       // keys below it are seen

    float4v o[NJ];
    float m = kNoMax, l = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j] = (float4v){0.f, 0.f, 0.f, 0.f};

    // keys of this wave: every WK-th tile of the workgroup's share, up to the
    // last that one of its rows sees
    int hi = T, all = T;         // (all: keys that every row sees)
    if (p.causal) {
        const int mi = uniform_div(m0 + ROWS - 1, p.G), il = mi < cnt ? mi : cnt - 1;
        hi = T - cnt + il + 1 < T ? T - cnt + il + 1 : T;
        all = T - cnt + uniform_div(m0, p.G) + 1;
    }
    const int k0 = split * p.split_keys;
    const int64_t ke = (int64_t)k0 + p.split_keys;
    const int k1 = ke < hi ? (int)ke : hi;
    constexpr int STEP = 32 * WK;

    auto compute = [&](Tile<KV, D>& t, int t0) {
        const uint32_t keep = (uint32_t)__ballot(t.ok);
        if (keep == 0) return;
        const bool whole = keep == 0xffffffffu;
        if (!whole) {      // what stands in the value rows of keys left out may be anything
            const uint32_t bits = ((keep >> (4 * g)) & 0xF) | (((keep >> (16 + 4 * g)) & 0xF) << 4);
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int w = 0; w < TL::NV; ++w) t.v[i][w] = (bits >> i) & 1 ? t.v[i][w] : 0;
        }
        float ks8[8], vs8[8];
        if constexpr (TABLE) {
            const float kept_vs = t.ok ? t.vs : 0.f;       // (of a key left out: anything, NaN too)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = (i < 4 ? 0 : 12) + 4 * g + i;
                ks8[i] = __shfl(t.ks, r, 64);
                vs8[i] = __shfl(kept_vs, r, 64);
            }
        }
        float vf = 1.0f, pf[8];
        uint32_t ph[4], pl[4];
        const float4v s0 = tile_scores<KV, D, QF32, NQ>(t.k[0], q);
        const float4v s1 = tile_scores<KV, D, QF32, NQ>(t.k[1], q);
        // f32: the factor f of a score in two terms, and a weight's exponent s f - max
        // rounded as a whole, since an error of 2^-24 of a score of 17 is one of 7e-7 of
        // its weight (with the table, where every key has a factor of its own, neither: 128
        // beams x 8 heads x 64 took 19.4 us instead of 15.0)
        float sv[8], fe[8], fl[8], sc[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            sv[e] = e < 4 ? s0[e & 3] : s1[e & 3];
            const float ks = TABLE ? ks8[e] : KV == KV_I8 ? t.ks : 1.0f;
            fe[e] = KV == KV_I8 ? qf * ks : qf;
            if constexpr (QF32 && !TABLE) fl[e] = KV == KV_I8 ? fmaf(qf_lo, ks, fmaf(qf, ks, -fe[e])) : qf_lo;
            sc[e] = sv[e] * fe[e];
        }
        const bool cut = !whole || t0 + 32 > all;
        const uint32_t see = keep >> (4 * g) & low_bits(lim - t0 - 4 * g);
        auto leave_out = [&](float (&x)[8]) {
            if (cut) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (!(see & (1u << (e < 4 ? e : 12 + e)))) x[e] = -INFINITY;
            }
        };
        leave_out(sc);
        const float top = max8((float4v){sc[0], sc[1], sc[2], sc[3]}, (float4v){sc[4], sc[5], sc[6], sc[7]});
        const float mx = xgroup_max(fmaxf(m, top));
        const float alpha = __builtin_amdgcn_exp2f(m - mx);
        m = mx;
        if constexpr (QF32 && !TABLE) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sc[e] = fmaf(sv[e], fl[e], fmaf(sv[e], fe[e], -mx));
            leave_out(sc);
        } else {
            // weights, and so l and O, are 2^14 p where they go to f16 alone: down to
            // 2^-28 of the largest they keep its 11 bits, then 2^-39 of it
#pragma unroll
            for (int e = 0; e < 8; ++e) sc[e] -= QF32 ? mx : mx - 14.0f;
        }
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            pf[e] = __builtin_amdgcn_exp2f(sc[e]);
            sum += pf[e];
        }
        l = l * alpha + sum;
        if constexpr (KV == KV_I8) {
            if constexpr (TABLE) {
                // weights p vs of keys with different scales: their largest becomes
                // 2^14, so that f16 keeps it exactly whatever the scales (a power of two instead
                // doubled the error of outputs that one key decides; the reciprocal's last
                // bit is one of 2^-23).  A largest below 2^-110 is as good as none, and its
                // reciprocal would not be finite
#pragma unroll
                for (int e = 0; e < 8; ++e) pf[e] *= vs8[e];
                float top = max8((float4v){pf[0], pf[1], pf[2], pf[3]}, (float4v){pf[4], pf[5], pf[6], pf[7]});
                top = xgroup_max(fmaxf(top, 0x1p-110f));
                const float inv = __builtin_amdgcn_rcpf(top) * 0x1p14f;
#pragma unroll
                for (int e = 0; e < 8; ++e) pf[e] *= inv;
                vf = top * 0x1p-14f;
            } else {
                vf = SPLIT ? t.vs * 0x1p-14f : t.vs;
            }
        }
        if constexpr (SPLIT) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float up = TABLE ? 1.0f : 0x1p14f;
                split_f16<false>(pf[2 * e] * up, pf[2 * e + 1] * up, ph[e], pl[e]);
            }
        } else if constexpr (KV != KV_F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) ph[e] = pack_f16(pf[2 * e], pf[2 * e + 1]);
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if constexpr (KV == KV_F32) {
                float4v acc = o[j] * alpha;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(t.v[i][j]), pf[i], acc, 0, 0, 0);
                o[j] = acc;
            } else {
                const half8v a = value_frag<KV, D>(t.v, j);
                const int4v bi = {(int)ph[0], (int)ph[1], (int)ph[2], (int)ph[3]};
                float4v acc = o[j] * alpha;
                if constexpr (KV == KV_F16) {
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, __builtin_bit_cast(half8v, bi), acc, 0, 0, 0);
                } else {
                    float4v blk = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, __builtin_bit_cast(half8v, bi),
                                                                        (float4v){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                    if constexpr (SPLIT) {
                        const int4v bl = {(int)pl[0], (int)pl[1], (int)pl[2], (int)pl[3]};
                        blk = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, __builtin_bit_cast(half8v, bl), blk, 0, 0, 0);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[e] = fmaf(vf, blk[e], acc[e]);
                }
                o[j] = acc;
            }
        }
    };

    if (k0 + 32 * wk < k1) {
        int t0 = k0 + 32 * wk;
        if constexpr (KV == KV_F32) {      // (a second tile in flight gained nothing, eight key shares lost 10 to 40%)
            for (; t0 < k1; t0 += STEP) {
                Tile<KV, D> a;
                load_tile<KV, D>(a, s, t0, lane);
                compute(a, t0);
            }
        } else {
            // the next tile's loads are in flight while a tile is computed,
            // the table's entries one tile further ahead
            Tile<KV, D> a, bt;
            int e = 0;
            auto load = [&](Tile<KV, D>& t, int at) {
                if constexpr (TABLE) {
                    const int slot = e, next = at + STEP + (lane & 31);
                    e = s.table[next < T ? next : T - 1];
                    load_tile_by_table<D>(t, s, at, slot, lane);
                } else {
                    load_tile<KV, D>(t, s, at, lane);
                }
            };
            if constexpr (TABLE) {
                const int at = t0 + (lane & 31);
                e = s.table[at < T ? at : T - 1];
            }
            load(a, t0);
            while (true) {
                load(bt, t0 + STEP);
                compute(a, t0);
                t0 += STEP;
                if (t0 >= k1) break;
                load(a, t0 + STEP);
                compute(bt, t0);
                t0 += STEP;
                if (t0 >= k1) break;
            }
        }
    }

    l = xgroup_sum(l);       // a lane's sum covers its own keys

    // lane (c, g) stores row c, dimensions (4g + e) NJ .. + NJ
    auto store = [&](int e, const float* x, float ml, float ll) {
        const int mr = m0 + c, i = udiv_small(mr, p.G), h = kh * p.G + (mr - i * p.G), d = (4 * g + e) * NJ;
        if (i >= cnt || d >= p.dk) return;
        if (p.splits > 1) {
            const int64_t at = ((int64_t)(b * p.Hkv + kh) * M + mr) * p.splits + split;
            if (d == 0) p.part_ml[at] = float2{ml, ll};
            if (ll != 0.f) {
                float* y = p.part_o + at * p.dk + d;
#pragma unroll
                for (int j = 0; j < NJ; j += 2) *(float2v*)(y + j) = (float2v){x[j], x[j + 1]};
            }
            return;
        }
        const float inv = ll != 0.f ? 1.0f / ll : 0.f;
        const int64_t at = b * p.o_item + i * p.o_row + h * p.o_head + d;
        if constexpr (QF32) {
            float* y = (float*)p.out + at;
#pragma unroll
            for (int j = 0; j < NJ; j += 2) *(float2v*)(y + j) = (float2v){x[j] * inv, x[j + 1] * inv};
        } else {
            uint32_t w[NJ / 2];
#pragma unroll
            for (int j = 0; j < NJ; j += 2) w[j / 2] = pack_f16(x[j] * inv, x[j + 1] * inv);
            f16* y = (f16*)p.out + at;
            if constexpr (NJ == 8) *(int4v*)y = (int4v){(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
            else if constexpr (NJ == 4) *(int2v*)y = (int2v){(int)w[0], (int)w[1]};
            else *(uint32_t*)y = w[0];
        }
    };
    // the key shares, brought to a common maximum: wave e adds and stores
    // accumulator register e of all four, in wave order
    __shared__ float sml[2][WK][16];
    __shared__ float so[WK][4][NJ][64];
    if (g == 0) {
        sml[0][wk][c] = m;
        sml[1][wk][c] = l;
    }
    __syncthreads();
    float mm = sml[0][0][c], ll = 0.f;
#pragma unroll
    for (int w = 1; w < WK; ++w) mm = fmaxf(mm, sml[0][w][c]);
#pragma unroll
    for (int w = 0; w < WK; ++w) ll += sml[1][w][c] * __builtin_amdgcn_exp2f(sml[0][w][c] - mm);
    const float fw = __builtin_amdgcn_exp2f(m - mm);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) so[wk][e][j][lane] = o[j][e] * fw;
    __syncthreads();
    float x[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        x[j] = so[0][wk][j][lane];
#pragma unroll
        for (int w = 1; w < WK; ++w) x[j] += so[w][wk][j][lane];
    }
    store(wk, x, mm, ll);
}

// Exponent field of the power of two at or above a finite scale x >= 0, 0 for none.
__device__ __forceinline__ int scale_exponent(float x) {
    const uint32_t u = (uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(x));
    const int e = (int)((u + 0x7fffffu) >> 23);
    return u == 0 ? 0 : e < 1 ? 1 : e > 254 ? 254 : e;
}

// Many query rows against the same keys: 128 rows a workgroup, 32 a wave, the
// keys in steps of 64 through LDS, where every wave reads them.  8-bit keys
// become f16 on the way in, once for the workgroup.  The value rows are turned
// there too: a thread loads 8 keys x D/32 dimensions and writes, per dimension,
// its 8 keys as one 16-byte piece, in the order in which the value product's
// operand wants them.  The next step's rows are loaded to registers while a
// step is computed.  LDS rows of 16-byte pieces are permuted (piece ^ a number
// from the row) so that the 16 rows of an operand read fall on different banks
// (64 of 4 bytes here: with a permutation that repeats after 8 rows the reads of
// 256-byte rows took twice as long).
//
// Weights go to f16 as 2^14 p: 2^14 keeps small ones out of f16's subnormals, and rides
// in the exponent.  With 8-bit keys the accumulator's unit is the block's value scale,
// whatever scales other blocks have that a row does not see or has no weight for.
// f16: it changes from block to block, along with the running maximum before a step's first block and
// by a product of its own between the two (2% of the time; the ratio of the scales in the
// weights instead cost a dominating weight, else exact, its rounding: 6 x 150 rows x 32
// heads x 128, 1100 tokens were off by 2.7e-4 of their size, so by 2.33e-4; the rounding of the output is 2.07e-4).
// f32: the unit is the power of two at or above the larger scale of a step's two blocks,
// so that it changes without a rounding and a weight's two terms carry r = scale / unit;
// blocks more than 2^6 apart are taken one after the other, so r is at least 2^-7 and the terms
// keep 22 bits of a weight down to 2^-9 of the largest, 11 of it down to 2^-21.
// (The unit stays above 2^-72 of its largest so far, for the accumulator's range; r goes below that only from there on.)
//
// f16, 16 x 448 rows x 8 heads x 128, 750 keys: 42.6 us alone, 38.2 in a stream of
// such calls (575 TFLOP/s; a large product of the library reaches 1071), 118 on
// dec_attn_kernel.  VALU issue 49%, matrix pipe 30%, LDS 30%: a wave's softmax stands
// between its products, and 226 registers leave two waves a SIMD to overlap them.
// Tried: 16 rows a wave and eight waves (57 us), two LDS buffers (44.4).
template <int KV, bool QF32, int D, bool CAUSAL>
__global__ __launch_bounds__(256, 2) void dec_tile_kernel(DecAttnParams p) {
    constexpr int QT = 2, NW = 4, ROWS = 16 * QT * NW, KT = 64;
    constexpr bool SPLIT = KV == KV_I8 && QF32, RIDES = KV == KV_I8 && !QF32;
    constexpr int ES = KV == KV_F16 ? 2 : 1, NQ = SPLIT ? D / 4 : D / 8, NJ = D / 16;
    constexpr int PIECES = D * ES / 16, KP = KT * PIECES / 256;     // 16-byte pieces of a key row; of a thread
    constexpr int DV = D / 32;                                      // value dimensions of a thread
    constexpr int KC = D / 8;                                       // 16-byte pieces of a key row in LDS
    constexpr int JB = NJ < 4 ? NJ : 4;                             // value products in flight
    __shared__ __align__(16) f16 sk[KT * D];
    __shared__ __align__(16) f16 sv[D * KT];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), c = lane & 15, g = lane >> 4;
    const int M = p.n_q * p.G, mt = (M + ROWS - 1) / ROWS;
    int b, kh, split, mtile;
    work_of<false>(blockIdx.x, p, mt, b, kh, split, mtile);
    int T = p.k_len ? p.k_len[b] : p.n_k;
    T = T < 0 ? 0 : T > p.n_k ? p.n_k : T;
    int cnt = p.q_len ? p.q_len[b] : p.n_q;
    cnt = cnt < 0 ? 0 : cnt > p.n_q ? p.n_q : cnt;
    if (uniform_div(mtile * ROWS, p.G) >= cnt) return;                 // no row of this tile is asked for
    const int m0 = mtile * ROWS + wave * 16 * QT;
    const uint8_t *kb, *vb;
    const float *ksc = nullptr, *vsc = nullptr;
    const uint8_t* mask = nullptr;
    if constexpr (KV == KV_I8) {
        int sl = p.slot ? p.slot[b] : b;
        if ((unsigned)sl >= (unsigned)p.n_slots) {
            sl = 0;
            T = 0;
        }
        kb = (const uint8_t*)p.k + sl * p.k_item + kh * p.k_head;
        vb = (const uint8_t*)p.v + sl * p.v_item + kh * p.v_head;
        ksc = p.k_scale + ((int64_t)sl * p.Hkv + kh) * p.n_blocks;
        vsc = p.v_scale + ((int64_t)sl * p.Hkv + kh) * p.n_blocks;
    } else {
        kb = (const uint8_t*)p.k + (b * p.k_item + kh * p.k_head) * ES;
        vb = (const uint8_t*)p.v + (b * p.v_item + kh * p.v_head) * ES;
        mask = p.mask ? p.mask + b * p.mask_item : nullptr;
    }
    const uint32_t k_row = (uint32_t)p.k_row * ES, v_row = (uint32_t)p.v_row * ES;

    uint32_t q[QT][NQ];
    float qf[QT], qf_lo[QT];     // factor of the scores, what its rounding left
    int lim[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int i = load_query<KV, QF32, D, KV_F16>(p, m0 + 16 * qt + c, b, kh, cnt, g, q[qt], qf[qt], qf_lo[qt]);
        lim[qt] = CAUSAL ? T - cnt + i + 1 : T;
        if (p.scale < 0.f) {       // the factor is not negative: maxima are taken before it
            qf[qt] = -qf[qt];
            qf_lo[qt] = -qf_lo[qt];
#pragma unroll
            for (int n = 0; n < NQ; ++n) q[qt][n] ^= 0x80008000u;
        }
    }
    // keys that one of the rows of the workgroup, of the wave sees; keys that all of the wave's see
    auto seen = [&](int m) {
        const int i = uniform_div(m, p.G);
        return CAUSAL ? T - cnt + (i < cnt ? i : cnt - 1) + 1 : T;
    };
    const int hi = seen(mtile * ROWS + ROWS - 1), hi_wave = seen(m0 + 16 * QT - 1), all_wave = seen(m0);
    const int k0 = split * p.split_keys;
    const int64_t ke = (int64_t)k0 + p.split_keys;
    const int k1 = ke < hi ? (int)ke : hi;

    float4v o[QT][NJ];
    float m[QT], l[QT];
    // the accumulator's unit (0: no value yet) and its largest; f32: their exponent fields
    float unit = 0.f, unit_top = 0.f;
    int unit_e = 0, top_e = 0;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        m[qt] = kNoMax;
        l[qt] = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[qt][j] = (float4v){0.f, 0.f, 0.f, 0.f};
    }

    // the step in flight
    uint32_t kr[KP][4], vr[8][DV * ES > 4 ? DV * ES / 4 : 1];
    uint32_t mr8 = 1;
    float ksr[2] = {1.f, 1.f}, vsr[2] = {1.f, 1.f};
    const int oct = t >> 5, d0 = (t & 31) * DV;            // value work: keys of octet oct, dimensions d0 .. d0 + DV
    const int v_key = 32 * (oct >> 2) + 4 * (oct & 3);
    const uint32_t v_at = (uint32_t)v_key * v_row + (d0 < p.dk ? d0 : 0) * ES;
    constexpr int KSTEP = 256 / PIECES;                    // key work: piece k_ch of keys k_key + n KSTEP
    const int k_key = t / PIECES, k_ch = t % PIECES;
    const uint32_t k_at = (uint32_t)k_key * k_row + (16 * k_ch < p.dk * ES ? 16 * k_ch : 0);
    // LDS addresses that differ in more than a constant (see stage for the permutation)
    auto key_turn = [](int key) { return KC == 16 ? key & 15 : KC == 8 ? (key >> 1) & 7 : (key >> 2) & 3; };
    int ka[D / 32], va[2][2];
#pragma unroll
    for (int n = 0; n < D / 32; ++n) ka[n] = c * D + 8 * ((4 * n + g) ^ key_turn(c));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) va[h][i] = c * KT + 8 * ((4 * h + g) ^ (c & 7) ^ (c >> 3) ^ (2 * i));
    }
    auto load = [&](int t0) {
        const int left = T - 1 - t0;                       // t0 < T
        if (mask) mr8 = mask[t0 + (lane < left ? lane : left)];
        if constexpr (KV == KV_I8) {
            const int blk = t0 / kCacheBlock, last = (T - 1) / kCacheBlock;
            ksr[0] = ksc[blk];
            vsr[0] = vsc[blk];
            ksr[1] = ksc[blk < last ? blk + 1 : blk];
            vsr[1] = vsc[blk < last ? blk + 1 : blk];
        }
        // rows past the last key are out of the resources' range: zeros
        const int rows = left < KT - 1 ? left : KT - 1;
        const auto kt = step_rsrc(kb + (int64_t)t0 * k_row, rows * k_row + p.dk * ES);
        const auto vt = step_rsrc(vb + (int64_t)t0 * v_row, rows * v_row + p.dk * ES);
#pragma unroll
        for (int n = 0; n < KP; ++n) buffer_words(kr[n], kt, k_at + n * KSTEP * k_row);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t at = v_at + (i < 4 ? i : 12 + i) * v_row;
            if constexpr (DV * ES == 2) vr[i][0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(vt, at, 0, 0);
            else buffer_words(vr[i], vt, at);
        }
    };
    auto stage = [&](uint64_t keep) {
#pragma unroll
        for (int n = 0; n < KP; ++n) {
            const int key = k_key + n * KSTEP, ch = k_ch, x = key_turn(k_key);    // KSTEP % 16 = 0
            f16* row = sk + key * D;
            if constexpr (KV == KV_F16) {
                *(int4v*)(row + 8 * (ch ^ x)) = (int4v){(int)kr[n][0], (int)kr[n][1], (int)kr[n][2], (int)kr[n][3]};
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    int4v w;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        w[2 * e] = i8_pair_f16(__builtin_amdgcn_perm(0, kr[n][2 * h + e], 0x0c010c00));
                        w[2 * e + 1] = i8_pair_f16(__builtin_amdgcn_perm(0, kr[n][2 * h + e], 0x0c030c02));
                    }
                    *(int4v*)(row + 8 * ((2 * ch + h) ^ x)) = w;
                }
            }
        }
        if (keep != ~0ull) {       // what stands in the value rows of keys left out may be anything
            const uint32_t half = (uint32_t)(keep >> (32 * (oct >> 2))), at = 4 * (oct & 3);
            const uint32_t bits = ((half >> at) & 0xF) | (((half >> (16 + at)) & 0xF) << 4);
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (uint32_t& w : vr[i]) w = (bits >> i) & 1 ? w : 0;
        }
#pragma unroll
        for (int j = 0; j < DV; ++j) {
            const int d = d0 + j, f = (d & 7) ^ ((d >> 3) & 3);
            int4v w;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (KV == KV_F16) {
                    w[i] = __builtin_amdgcn_perm(vr[2 * i + 1][j >> 1], vr[2 * i][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
                } else {
                    const uint32_t e = j & 3;
                    w[i] = i8_pair_f16(__builtin_amdgcn_perm(vr[2 * i + 1][j >> 2], vr[2 * i][j >> 2], 0x0c040c00u | e | (e << 16)));
                }
            }
            *(int4v*)(sv + d * KT + 8 * (oct ^ f)) = w;
        }
    };
    auto compute = [&](int t0, uint64_t keep, const float (&ks)[2], const float (&vs)[2]) {
        // (a wave that feeds the matrix pipe goes before one at its softmax: 2 to 5% in f16)
        if constexpr (KV == KV_F16) __builtin_amdgcn_s_setprio(1);
        float4v s[QT][4];
        // consecutive products go to different accumulators
#pragma unroll
        for (int n = 0; n < D / 32; ++n) {
            half8v a[4];
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) a[kt] = *(const half8v*)(sk + ka[n] + 16 * kt * D);
#pragma unroll
            for (int part = 0; part < (SPLIT ? 2 : 1); ++part)
#pragma unroll
                for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                    for (int qt = 0; qt < QT; ++qt) {
                        const int o = part * (D / 8) + 4 * n;
                        const int4v bq = {(int)q[qt][o], (int)q[qt][o + 1], (int)q[qt][o + 2], (int)q[qt][o + 3]};
                        const float4v from = n == 0 && part == 0 ? (float4v){0.f, 0.f, 0.f, 0.f} : s[qt][kt];
                        s[qt][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[kt], __builtin_bit_cast(half8v, bq), from, 0, 0, 0);
                    }
        }
        if constexpr (KV == KV_F16) __builtin_amdgcn_s_setprio(0);
        settled(s);
        const bool cut = keep != ~0ull || t0 + KT > all_wave;
        float rv[2] = {1.f, 1.f}, ri[2] = {1.f, 1.f}, rl[2] = {0.f, 0.f}, grow = 1.f, grow2 = 1.f;
        if constexpr (RIDES) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // (a block of zeros: a factor that leaves nothing in f16 but the weights' sum in f32)
                const float to = vs[h] > 0.f ? fmaxf(fmaxf(vs[h], unit_top * 0x1p-72f), 0x1p-126f) : unit;
                const float inv = __builtin_amdgcn_rcpf(to), r = vs[h] > 0.f ? fmaxf(vs[h] * inv, 0x1p-60f) : 0x1p-60f;
                (h == 0 ? grow : grow2) = to > 0.f ? unit * inv : 1.f;
                unit = to;
                unit_top = fmaxf(unit_top, to);
                ri[h] = __builtin_amdgcn_rcpf(r);
                rl[h] = __builtin_amdgcn_logf(r);
            }
        } else if constexpr (KV == KV_I8) {
            const int e0 = scale_exponent(vs[0]), e1 = scale_exponent(vs[1]), e = e0 > e1 ? e0 : e1;
            if (e != 0) {
                top_e = e > top_e ? e : top_e;
                const int to = e > top_e - 72 ? e : top_e - 72;
                grow = ldexpf(1.0f, unit_e - to);
                unit_e = to;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                rv[h] = fmaxf(ldexpf(vs[h], 127 - unit_e), 0x1p-60f) * 0x1p14f;
            }
        }
        uint32_t ph[QT][2][4], pl[QT][2][4];
        float alpha[QT];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            // (not zero, as for a block of zeros: -inf stays -inf)
            float f[2], fl[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                f[h] = KV == KV_I8 ? qf[qt] * ks[h] : qf[qt];
                if constexpr (SPLIT) {
                    // in two terms, as in dec_attn_kernel, the first rounded down: the second is
                    // not negative then, nor zero, and -inf stays -inf
                    const bool above = fmaf(qf_lo[qt], ks[h], fmaf(qf[qt], ks[h], -f[h])) < 0.f;
                    f[h] = __uint_as_float(__float_as_uint(f[h]) - (above ? 1 : 0));
                    fl[h] = fmaxf(fmaf(qf_lo[qt], ks[h], fmaf(qf[qt], ks[h], -f[h])), 0x1p-126f);
                }
                f[h] = fmaxf(f[h], 1e-37f);
            }
            if (cut) {
                const int below = lim[qt] - t0 - 4 * g;
                const uint32_t see[2] = {(uint32_t)keep >> (4 * g) & low_bits(below), (uint32_t)(keep >> 32) >> (4 * g) & low_bits(below - 32)};
#pragma unroll
                for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(see[kt >> 1] & (1u << (16 * (kt & 1) + e)))) s[qt][kt][e] = -INFINITY;
            }
            float mx = m[qt];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                mx = fmaxf(mx, max8(s[qt][2 * h], s[qt][2 * h + 1]) * f[h]);
            }
            mx = fmaxf(m[qt], xgroup_max(mx));
            alpha[qt] = __builtin_amdgcn_exp2f(m[qt] - mx) * grow;
            l[qt] *= __builtin_amdgcn_exp2f(m[qt] - mx);
            m[qt] = mx;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float off = SPLIT ? -mx : 14.0f - mx + (RIDES ? rl[h] : 0.f);
                float pf[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = s[qt][2 * h + (e >> 2)][e & 3];
                    float y = fmaf(x, f[h], off);
                    if constexpr (SPLIT) y = fmaf(x, fl[h], y);
                    pf[e] = __builtin_amdgcn_exp2f(y);
                }
                const float sum = ((pf[0] + pf[1]) + (pf[2] + pf[3])) + ((pf[4] + pf[5]) + (pf[6] + pf[7]));
                l[qt] = RIDES ? fmaf(sum, ri[h], l[qt]) : l[qt] + sum;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (SPLIT) split_f16<true>(pf[2 * e] * rv[h], pf[2 * e + 1] * rv[h], ph[qt][h][e], pl[qt][h][e]);
                    else ph[qt][h][e] = pack_f16(pf[2 * e], pf[2 * e + 1]);
                }
            }
        }
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
#pragma unroll
            for (int j = 0; j < NJ; ++j) o[qt][j] *= alpha[qt];
        if constexpr (KV == KV_F16) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j0 = 0; j0 < NJ; j0 += JB) {
                half8v a[JB];
#pragma unroll
                for (int j = 0; j < JB; ++j) a[j] = *(const half8v*)(sv + va[h][(j0 + j) & 1] + 16 * (j0 + j) * KT);
                if constexpr (RIDES) {
                    if (h == 1) {
#pragma unroll
                        for (int qt = 0; qt < QT; ++qt)
#pragma unroll
                            for (int j = 0; j < JB; ++j) o[qt][j0 + j] *= grow2;
                    }
                }
#pragma unroll
                for (int part = 0; part < (SPLIT ? 2 : 1); ++part)
#pragma unroll
                    for (int j = 0; j < JB; ++j)
#pragma unroll
                        for (int qt = 0; qt < QT; ++qt) {
                            const uint32_t(&w)[4] = part ? pl[qt][h] : ph[qt][h];
                            const int4v bp = {(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
                            o[qt][j0 + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[j], __builtin_bit_cast(half8v, bp), o[qt][j0 + j], 0, 0, 0);
                        }
            }
        if constexpr (KV == KV_F16) __builtin_amdgcn_s_setprio(0);
    };

    if (k0 < k1) load(k0);
    bool second = false;       // the second half of a step whose blocks' scales are far apart: loaded and staged again
    for (int t0 = k0; t0 < k1;) {
        uint64_t keep = __ballot(t0 + lane < T && mr8 != 0);           // the same in every wave
        const float ks[2] = {ksr[0], ksr[1]};
        float vs[2] = {vsr[0], vsr[1]};
        stage(keep);
        __syncthreads();
        int next = t0 + KT;
        if constexpr (SPLIT) {
            const int e0 = scale_exponent(vs[0]), e1 = scale_exponent(vs[1]);
            if (e0 != 0 && e1 != 0 && (e0 > e1 + 6 || e1 > e0 + 6)) {
                keep &= second ? 0xffffffff00000000ull : 0xffffffffull;
                vs[0] = vs[1] = second ? vs[1] : vs[0];
                second = !second;
                next = second ? t0 : next;
            }
        }
        if (next < k1) load(next);
        if (!CAUSAL || t0 < hi_wave) compute(t0, keep, ks, vs);
        __syncthreads();
        t0 = next;
    }

#pragma unroll
    for (int qt = 0; qt < QT; ++qt) l[qt] = xgroup_sum(l[qt]);
    // lane (c, g) has row c's dimensions 16 j + 4 g .. + 4
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const float ll = l[qt];
        const int mr = m0 + 16 * qt + c, i = udiv_small(mr, p.G), h = kh * p.G + (mr - i * p.G);
        if (i >= cnt) continue;
        const float out_unit = SPLIT ? ldexpf(unit_e != 0 ? 1.0f : 0.f, unit_e - 141) : RIDES ? unit : 1.0f;
        if (p.splits > 1) {
            const int64_t at = ((int64_t)(b * p.Hkv + kh) * M + mr) * p.splits + split;
            if (g == 0) p.part_ml[at] = float2{m[qt], ll};
            if (ll == 0.f) continue;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                if (16 * j + 4 * g < p.dk) *(float4v*)(p.part_o + at * p.dk + 16 * j + 4 * g) = o[qt][j] * out_unit;
            continue;
        }
        const float f = ll != 0.f ? out_unit / ll : 0.f;
        const int64_t at = b * p.o_item + i * p.o_row + h * p.o_head + 4 * g;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if (16 * j + 4 * g >= p.dk) continue;
            const float4v x = o[qt][j] * f;
            if constexpr (QF32) *(float4v*)((float*)p.out + at + 16 * j) = x;
            else *(int2v*)((f16*)p.out + at + 16 * j) = (int2v){(int)pack_f16(x[0], x[1]), (int)pack_f16(x[2], x[3])};
        }
    }
}

// Joins the splits' (m, l, O), at most 64 of them.  Few rows: a workgroup a row,
// lane s of every wave with split s's factor 2^(m_s - max m); wave w adds splits
// w, w + 4, ... in that order, two dimensions a lane, and the four sums are added
// in wave order.
template <bool F32> __global__ __launch_bounds__(256) void dec_join_kernel(DecAttnParams p) {
    __shared__ float so[4][128];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, M = p.n_q * p.G, d = 2 * lane;
    const int row = blockIdx.x, unit = uniform_div(row, M), mr = row - unit * M;
    const int b = uniform_div(unit, p.Hkv), kh = unit - b * p.Hkv, i = uniform_div(mr, p.G), h = kh * p.G + (mr - i * p.G);
    const float2 ml = lane < p.splits ? p.part_ml[(int64_t)row * p.splits + lane] : float2{kNoMax, 0.f};
    if (i >= (p.q_len ? p.q_len[b] : p.n_q)) return;
    const float mm = wave_max(ml.x);
    // a split without a key (l = 0) has not written its O
    const float f = ml.y != 0.f ? __builtin_amdgcn_exp2f(ml.x - mm) : 0.f;
    const float l = wave_sum(ml.y * f);
    float x0 = 0.f, x1 = 0.f;
    if (d < p.dk) {
        const float* src = p.part_o + (int64_t)row * p.splits * p.dk + d;
        for (int s0 = wave; s0 < p.splits; s0 += 16) {
            float2v o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int s = s0 + 4 * k;
                o[k] = *(const float2v*)(src + (int64_t)(s < p.splits ? s : s0) * p.dk);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int s = s0 + 4 * k;
                const float fs = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), s & 63));
                const bool add = s < p.splits && fs != 0.f;
                x0 += add ? o[k][0] * fs : 0.f;
                x1 += add ? o[k][1] * fs : 0.f;
            }
        }
    }
    so[wave][d] = x0;
    so[wave][d + 1] = x1;
    __syncthreads();
    if (wave != 0 || d >= p.dk) return;
    x0 = (so[0][d] + so[1][d]) + (so[2][d] + so[3][d]);
    x1 = (so[0][d + 1] + so[1][d + 1]) + (so[2][d + 1] + so[3][d + 1]);
    const float inv = l != 0.f ? 1.0f / l : 0.f;
    const int64_t at = b * p.o_item + i * p.o_row + h * p.o_head + d;
    if constexpr (F32) *(float2v*)((float*)p.out + at) = (float2v){x0 * inv, x1 * inv};
    else *(uint32_t*)((f16*)p.out + at) = pack_f16(x0 * inv, x1 * inv);
}

// Many rows (and so few splits): four dimensions a thread, dk / 4 threads a row,
// the splits in order, four at a time.
template <bool F32> __global__ __launch_bounds__(256) void dec_join_rows_kernel(DecAttnParams p, int rows) {
    const int per = p.dk >> 2, M = p.n_q * p.G, tr = udiv_small(threadIdx.x, per), d = 4 * (threadIdx.x - tr * per);
    const int rpb = uniform_div(256, per), row = blockIdx.x * rpb + tr;
    if (tr >= rpb || row >= rows) return;
    const int unit = udiv_small(row, M), mr = row - unit * M, b = udiv_small(unit, p.Hkv), kh = unit - b * p.Hkv;
    const int i = udiv_small(mr, p.G), h = kh * p.G + (mr - i * p.G);
    if (i >= (p.q_len ? p.q_len[b] : p.n_q)) return;
    const float2* ml = p.part_ml + (int64_t)row * p.splits;
    const float* src = p.part_o + (int64_t)row * p.splits * p.dk + d;
    float m = kNoMax, l = 0.f;
    float4v x = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < p.splits; s0 += 4) {
        float2 v[4];
        float4v o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int s = s0 + k < p.splits ? s0 + k : s0;
            v[k] = ml[s];
            o[k] = *(const float4v*)(src + (int64_t)s * p.dk);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (s0 + k >= p.splits || v[k].y == 0.f) continue;     // (O of a split without a key is not written)
            const float hi = fmaxf(m, v[k].x), fo = __builtin_amdgcn_exp2f(m - hi), fn = __builtin_amdgcn_exp2f(v[k].x - hi);
            m = hi;
            l = l * fo + v[k].y * fn;
            x = x * fo + o[k] * fn;
        }
    }
    x *= l != 0.f ? 1.0f / l : 0.f;
    const int64_t at = b * p.o_item + i * p.o_row + h * p.o_head + d;
    if constexpr (F32) *(float4v*)((float*)p.out + at) = x;
    else *(int2v*)((f16*)p.out + at) = (int2v){(int)pack_f16(x[0], x[1]), (int)pack_f16(x[2], x[3])};
}

// Rows a workgroup takes and how many ways the keys are split over workgroups.
struct Shape { bool wide; int rows, mt, splits, keys; };
Shape split_shape(const DecAttnParams& p, bool wide) {
    Shape s;
    const int64_t M = (int64_t)p.n_q * p.G, units = (int64_t)p.B * p.Hkv;
    const int tiles = cdiv(p.n_k > 0 ? p.n_k : 1, 32);
    s.wide = wide;
    s.rows = wide ? 128 : 16;
    s.mt = cdiv(M, s.rows);
    const int64_t wgs = units * s.mt;
    int64_t want = wgs >= 512 ? 1 : 512 / wgs;             // about two workgroups per CU
    if (want > 64) want = 64;
    // whole rounds of the four key shares, or steps of dec_tile_kernel.  A split
    // costs its partial sums and the join's launch, so it takes at least four
    // rounds (of about 0.5 us; f32 heads above 64 one round, of 2 us) or eight steps
    // (1 us), four where there are few rows to join
    int per = (cdiv(tiles, want) + 3) / 4 * 4;
    const int least = p.kv == KV_F32 && p.dk > 64 ? 4 : wide && units * M <= 1024 ? 8 : 16;
    if (per < least) per = least;
    s.splits = cdiv(tiles, per);
    s.keys = per * 32;
    return s;
}
Shape attn_shape(const DecAttnParams& p) {
    // dec_tile_kernel's rows share what they read and convert, but its time goes by
    // the steps of a workgroup, however few workgroups there are and rows they have.
    // By tiles of 16 rows x 32 keys, 16 of them a full step, f16:
    //   tiles  steps x rounds   16-row form   128-row form, us
    //    3328        2               8.7           7.0    (d_head 64: 8 items x 8 heads x 200 rows, 128 keys)
    //    6656        4              11.7           9.3    (256 keys)
    //    6144        6               9.0          12.0    (16 x 8 x 64 rows, 375 keys)
    //    9984        6              22.1          17.7    (d_head 128: 8 x 8 x 200 rows, 375 keys)
    //    4608        8              11.8          20.2    (4 x 8 x 130 rows, 500 keys)
    // 8-bit keys (where rows see part of the keys and lengths differ): with d_head 64
    // no gain in most (37.6 against 44.1 at 112896 tiles, 119 against 120 at 448000).  With
    // 128 dimensions, f16, by tiles alone:
    //   27456  24.5  30.1  (8 x 8 x 200 rows, 1025 keys)      61440  39.0  40.4  (4 x 16 x 256, 1920)
    //   32256  24.9  28.9  (4 x 16 x 128, 2000)               64512  44.8  41.3  (2 x 16 x 512, 2000)
    //   36864  32.8  30.7  (32 x 8 x 130, 512)                67200  48.4  48.3  (6 x 32 x 150, 1100)
    //   54912  39.5  39.8  (8 x 16 x 200, 1025)              141056   100  65.5  (2 x 64 x 600, 900)
    // Even at the bound; away from its middle it misses full rounds of full tiles (50176:
    // 53.3 30.3, 8 x 16 x 448 rows, 448 keys) and takes tiles that are half empty (65536: 44.5
    // 50.0, 16 x 32 x 64, 1000).  f32 the same within 10% (67200: 61.8 66.0; 141056: 135 92.2).
    // (Rounds are of the chip's 256 CUs, written in: the workspace can be asked for without a device.)
    const int64_t M = (int64_t)p.n_q * p.G;
    if (p.kv == KV_F32 || p.table || M < 64) return split_shape(p, false);
    const Shape wide = split_shape(p, true);
    const int64_t units = (int64_t)p.B * p.Hkv, tiles = units * cdiv(M, 16) * cdiv(p.n_k, 32);
    const int64_t steps = (int64_t)(p.n_k < wide.keys ? cdiv(p.n_k, 64) : wide.keys / 64) * cdiv(units * wide.mt * wide.splits, 256);
    return (p.kv == KV_F16 ? steps > 0 && tiles >= 1500 * steps : p.dk > 64 && tiles >= 60000) ? wide : split_shape(p, false);
}

template <int KV, bool QF32, int D, bool TABLE> void launch_shape(const DecAttnParams& p, const Shape& sh, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)p.B * p.Hkv * sh.mt * sh.splits));
    if constexpr (KV == KV_F16 || (KV == KV_I8 && D > 64 && !TABLE))
        if (sh.wide) {
            if (p.causal && KV == KV_I8) launch(dec_tile_kernel<KV, QF32, D, KV == KV_I8>, grid, dim3(256), 0, s, p);
            else launch(dec_tile_kernel<KV, QF32, D, false>, grid, dim3(256), 0, s, p);
            return;
        }
    launch(dec_attn_kernel<KV, QF32, D, TABLE>, grid, dim3(256), 0, s, p);
}
// Head widths above 64 take 128's registers and matrix instructions.  us at 64, 80, 96, 128:
//   f16 16 x 4 rows x 8 heads, 375 keys            6.0   8.0   8.2   8.1
//   f16 16 x 448 rows x 8 heads, 750 keys         27.6  38.9  39.6  40.2
//   f32 8 x 54 rows x 8 heads, 334 keys            9.5  18.4  18.3  18.6
//   int8 4 rows x 16 (4) heads, 32768 keys        16.4  21.9  22.5  27.3
//   int8 128 beams x 8 heads, 448 keys, table     13.5  22.0  22.2  22.7
//   int8, f32 8 x 200 rows x 8 heads, 1025 keys   18.1  30.0  30.3  31.6
template <int KV, bool QF32, bool TABLE> void launch_width(const DecAttnParams& p, const Shape& sh, hipStream_t s) {
    if (p.dk <= 32) launch_shape<KV, QF32, 32, TABLE>(p, sh, s);
    else if (p.dk <= 64) launch_shape<KV, QF32, 64, TABLE>(p, sh, s);
    else launch_shape<KV, QF32, 128, TABLE>(p, sh, s);
}

}  // namespace

size_t dec_attention_workspace(const DecAttnParams& p) {
    if (p.B == 0 || p.n_q == 0) return 0;
    const Shape sh = attn_shape(p);
    if (sh.splits == 1) return 0;
    const size_t parts = (size_t)p.B * p.Hkv * p.n_q * p.G * sh.splits;
    return parts * (sizeof(float2) + (size_t)p.dk * sizeof(float));
}

void launch_dec_attention(DecAttnParams p, void* ws, size_t ws_bytes, hipStream_t s) {
    if (p.B == 0 || p.n_q == 0) return;
    const Shape sh = attn_shape(p);
    const size_t need = dec_attention_workspace(p);
    require(need == 0 || (ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= need),
            "attention: the workspace is smaller than its size query says, or not 16-byte aligned");
    const double scale = (double)p.scale * kLog2e;
    p.scale = (float)scale;
    p.scale_lo = (float)(scale - p.scale);
    p.splits = sh.splits;
    p.split_keys = sh.keys;
    if (need) {
        const size_t parts = (size_t)p.B * p.Hkv * p.n_q * p.G * sh.splits;
        p.part_o = (float*)ws;
        p.part_ml = (float2*)(p.part_o + parts * p.dk);
    }
    if (p.kv == KV_F16) launch_width<KV_F16, false, false>(p, sh, s);
    else if (p.kv == KV_F32) launch_width<KV_F32, true, false>(p, sh, s);
    else if (p.q_f32) p.table ? launch_width<KV_I8, true, true>(p, sh, s) : launch_width<KV_I8, true, false>(p, sh, s);
    else p.table ? launch_width<KV_I8, false, true>(p, sh, s) : launch_width<KV_I8, false, false>(p, sh, s);
    if (sh.splits > 1) {
        const int64_t rows = (int64_t)p.B * p.Hkv * p.n_q * p.G;
        // threads by the row leave the chip short of them: 64 rows x 29 splits 9.1 us, by
        // the workgroup 4.7; 2048 x 15 4.8 and 4.8; 12800 x 3 5.0 and 7.5
        if (rows <= 1024) {
            auto* k = p.q_f32 ? dec_join_kernel<true> : dec_join_kernel<false>;
            launch(k, dim3((unsigned)rows), dim3(256), 0, s, p);
        } else {
            const int rpb = 256 / (p.dk / 4);
            auto* k = p.q_f32 ? dec_join_rows_kernel<true> : dec_join_rows_kernel<false>;
            launch(k, dim3((unsigned)((rows + rpb - 1) / rpb)), dim3(256), 0, s, p, (int)rows);
        }
    }
}

}  // namespace pkx
