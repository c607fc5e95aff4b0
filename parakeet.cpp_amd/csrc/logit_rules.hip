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

// One workgroup per row and TILE words: it counts the row's tokens among them, then passes over the logits.
template <typename ET, int TILE> __global__ __launch_bounds__(512) void logit_rules_kernel(LogitRulesParams p, int tiles) {
    __shared__ uint32_t times[TILE];
    const int r = udiv_small(blockIdx.x, tiles), t = threadIdx.x;
    const int v0 = (blockIdx.x - r * tiles) * TILE, words = p.V - v0 < TILE ? p.V - v0 : TILE;
    const bool count = p.tokens != nullptr;
    if (count) {
        for (int i = t; i < TILE; i += 512) times[i] = 0;
        __syncthreads();
        int n = p.len[r];
        n = n < 0 ? 0 : n > p.cap ? p.cap : n;
        const int from = p.window > 0 && n > p.window ? n - p.window : 0;
        const int mine = p.slot ? p.slot[r] : r;
        for (int i = from + t; i < n; i += 512) {
            const int slot = p.table ? p.table[r * p.table_row + i] : mine;
            if ((unsigned)slot >= (unsigned)p.n_slots) continue;
            const unsigned w = (unsigned)p.tokens[(int64_t)slot * p.cap + i] - (unsigned)v0;
            if (w < (unsigned)words) atomicAdd(&times[w], 1u);
        }
        __syncthreads();
    }
    const float rep = p.repetition ? p.repetition[r] : 1.f, pres = p.presence ? p.presence[r] : 0.f;
    const float freq = p.frequency ? p.frequency[r] : 0.f;
    int bi = p.bias ? (p.bias_index ? p.bias_index[r] : r) : -1;
    if ((unsigned)bi >= (unsigned)p.n_bias) bi = -1;
    int mi = p.mask ? (p.mask_index ? p.mask_index[r] : r) : -1;
    if ((unsigned)mi >= (unsigned)p.n_mask) mi = -1;
    const ET* x = (const ET*)p.x + r * p.x_row + v0;
    ET* o = (ET*)p.out + r * p.out_row + v0;
    const float* b = p.bias + (bi >= 0 ? bi * p.bias_row + v0 : 0);
    const uint32_t* m = p.mask + (mi >= 0 ? mi * p.mask_row + v0 / 32 : 0);
    for (int i = 8 * t; i < words; i += 8 * 512) {
        float v[8];
        load_row8(v, x, i, words);
        if (count) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t c = times[i + e];
                if (c) v[e] = (v[e] > 0.f ? v[e] / rep : v[e] * rep) - pres - freq * (float)c;
            }
        }
        if (bi >= 0) {
            float bb[8];
            load_row8(bb, b, i, words);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += bb[e];
        }
        if (mi >= 0) {
            const uint32_t bits = m[i / 32] >> (i % 32);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (!(bits >> e & 1)) v[e] = -__builtin_inff();
        }
        store_row8(o, v, i, words);
    }
}

}  // namespace

void launch_logit_rules(const LogitRulesParams& p, hipStream_t s) {
    if (p.R == 0 || p.V == 0) return;
    constexpr int kTile = 8192;
    const int tiles = cdiv(p.V, kTile);
    require((double)p.R * tiles < (double)(1 << 22), "logit rules: too many rows for one call");
    launch(p.f32 ? logit_rules_kernel<float, kTile> : logit_rules_kernel<f16, kTile>, dim3(p.R * tiles), dim3(512), 0, s, p, tiles);
}

}  // namespace pkx
