// Rules on a row of logits before a selection: with c the times that word v is
// among the row's last tokens,
//   x = c ? (x > 0 ? x / repetition : x repetition) - presence - frequency c : x
//   x = x + bias[v];  -inf where the mask's bit of v is 0.
// Bytes bound: logits read and written once; the counts of a tile of words are kept in LDS.
#pragma clang fp contract(off)

#include "block.hpp"
#include "rows.hpp"

namespace pkx {
namespace {

// E elements in one access at the element type's alignment.
template <typename T, int E> struct Piece {
    typedef T vec __attribute__((ext_vector_type(E)));
    typedef vec vecu __attribute__((aligned(sizeof(T))));
};

// One workgroup per row and tile of at most WORDS words (`width`, a multiple of 32).  The chain is length, table, tokens,
// counts; logits, biases and mask are asked for behind the table's entries and used when the counts are there, and no
// barrier waits for them (__syncthreads() waits for LDS alone).  What V leaves past whole pieces of 16 bytes goes to one thread
// a word.  A row's tiles, and the beams that share its history, run on one XCD, whose L2 then reads a history and a bias row once:
// 512 rows x 32769 f32, the last 1024 of 4096 tokens, 27.2 us (34.8 with the tiles dealt over the XCDs; 4.9 TB/s of logits read and
// written, a copy's rate).
constexpr int kRuleThreads = 512;
template <typename ET, int WORDS> __global__ __launch_bounds__(kRuleThreads) void logit_rules_kernel(LogitRulesParams p, int tiles, int width) {
    constexpr int T = kRuleThreads, E = 16 / sizeof(ET), NV = WORDS / (T * E);     // neighbouring lanes', neighbouring pieces
    constexpr int U = 4;                     // positions a thread has under way
    typedef typename Piece<ET, E>::vec vec;
    typedef typename Piece<ET, E>::vecu vecu;
    typedef typename Piece<float, E>::vec fvec;
    typedef typename Piece<float, E>::vecu fvecu;
    __shared__ __align__(16) uint32_t times[WORDS];
    const int unit = xcd_tile(blockIdx.x, gridDim.x), r = udiv_small(unit, tiles), t = threadIdx.x;
    const int v0 = (unit - r * tiles) * width, words = p.V - v0 < width ? p.V - v0 : width;
    const int whole = words & ~(E - 1), rest = words - whole;
    const bool count = p.tokens != nullptr;
    int from = 0, n = 0, mine = r;
    if (count) {
        n = p.len[r];
        n = n < 0 ? 0 : n > p.cap ? p.cap : n;
        from = p.window > 0 && n > p.window ? n - p.window : 0;
        mine = p.slot ? p.slot[r] : r;
    }
    int slot[U];
    auto slots = [&](int i0) {
        if (p.table) {
#pragma unroll
            for (int u = 0; u < U; ++u) slot[u] = i0 + u * T < n ? p.table[r * p.table_row + i0 + u * T] : -1;
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) slot[u] = i0 + u * T < n ? mine : -1;
        }
    };
    slots(from + t);

    int bi = p.bias ? (p.bias_index ? p.bias_index[r] : r) : -1;
    if ((unsigned)bi >= (unsigned)p.n_bias) bi = -1;
    int mi = p.mask ? (p.mask_index ? p.mask_index[r] : r) : -1;
    if ((unsigned)mi >= (unsigned)p.n_mask) mi = -1;
    const ET* x = (const ET*)p.x + r * p.x_row + v0;
    ET* o = (ET*)p.out + r * p.out_row + v0;
    const float* b = p.bias + (bi >= 0 ? bi * p.bias_row + v0 : 0);
    const uint32_t* m = p.mask + (mi >= 0 ? mi * p.mask_row + v0 / 32 : 0);
    vec v[NV];
    fvec bias[NV];
    uint32_t bits[NV];
    ET last = (ET)0.f;
    float last_bias = 0.f;
    uint32_t last_bits = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if (E * (t + k * T) < whole) v[k] = *(const vecu*)(x + E * (t + k * T));
    if (t < rest) last = x[whole + t];
    if (bi >= 0) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (E * (t + k * T) < whole) bias[k] = *(const fvecu*)(b + E * (t + k * T));
        if (t < rest) last_bias = b[whole + t];
    }
    if (mi >= 0) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (E * (t + k * T) < whole) bits[k] = m[E * (t + k * T) / 32];
        if (t < rest) last_bits = m[(whole + t) / 32];
    }
    const float rep = p.repetition ? p.repetition[r] : 1.f, pres = p.presence ? p.presence[r] : 0.f;
    const float freq = p.frequency ? p.frequency[r] : 0.f;
    if (count) {
#pragma unroll
        for (int k = 0; k < WORDS / (4 * T); ++k) *(int4v*)(times + 4 * (t + k * T)) = int4v{0, 0, 0, 0};
        __syncthreads();
        for (int i0 = from + t; i0 < n;) {
            int word[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                word[u] = (unsigned)slot[u] < (unsigned)p.n_slots ? p.tokens[(int64_t)slot[u] * p.cap + i0 + u * T] : -1;
            i0 += U * T;
            if (i0 < n) slots(i0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const unsigned w = (unsigned)word[u] - (unsigned)v0;
                if (word[u] >= 0 && w < (unsigned)words) atomicAdd(&times[w], 1u);
            }
        }
        __syncthreads();
    }
    auto ruled = [&](float y, uint32_t c, float add, bool keep) {
        if (c) y = (y > 0.f ? y / rep : y * rep) - pres - freq * (float)c;
        if (bi >= 0) y += add;
        return mi < 0 || keep ? y : -__builtin_inff();
    };
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int i = E * (t + k * T);
        if (i >= whole) continue;
        uint32_t c[E] = {};
        if (count)
#pragma unroll
            for (int e = 0; e < E; e += 4) *(int4v*)(c + e) = *(const int4v*)(times + i + e);
        vec y;
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = (ET)ruled((float)v[k][e], c[e], bias[k][e], bits[k] >> (i % 32 + e) & 1);
        __builtin_nontemporal_store(y, (vecu*)(o + i));
    }
    if (t < rest) o[whole + t] = (ET)ruled((float)last, count ? times[whole + t] : 0u, last_bias, last_bits >> ((whole + t) % 32) & 1);
}

// Tiles of 4096 words while they all are on the chip at once (8 x 262144 f32: 6.8 us, of 8192 words 8.1), then of 8192, which
// go through the histories half as often (512 x 32769 f32 with all of 4096 tokens: 34.1 us, of 4096 words 38.6).
template <typename ET, int WORDS> void launch_tiles(const LogitRulesParams& p, hipStream_t s) {
    const int tiles = cdiv(p.V, WORDS), width = cdiv(cdiv(p.V, tiles), 32) * 32;        // of one width, not full ones and a rest
    require((double)p.R * tiles < (double)(1 << 22), "logit rules: too many rows for one call");
    launch(logit_rules_kernel<ET, WORDS>, dim3(p.R * tiles), dim3(kRuleThreads), 0, s, p, tiles, width);
}
template <typename ET> void launch_typed(const LogitRulesParams& p, hipStream_t s) {
    if ((int64_t)p.R * cdiv(p.V, 4096) <= 1024) launch_tiles<ET, 4096>(p, s);
    else launch_tiles<ET, 8192>(p, s);
}

}  // namespace

void launch_logit_rules(const LogitRulesParams& p, hipStream_t s) {
    if (p.R == 0 || p.V == 0) return;
    p.f32 ? launch_typed<float>(p, s) : launch_typed<f16>(p, s);
}

}  // namespace pkx
