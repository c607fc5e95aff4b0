// Rotary positions: the pair (a, b) of frequency f at position p becomes
//   (a cos t - b sin t, b cos t + a sin t) mult,  t = p f,
// with pairs of neighbours (2 j, 2 j + 1) or of the halves (j, j + rot / 2) of the first
// rot dimensions; the others stay as they are.
// Bytes bound: every element is read and written once.  4 x 8192 ragged tokens x 20 heads x 128 f16 (235 MB): 44 us,
// 5.3 TB/s, where a copy of 1 GiB reaches 5.1.
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

// One workgroup per `tok` tokens of a row and part (blockIdx.y): their angles once into LDS, then the part's heads, IT items a
// thread at a time.  An item is E elements of a head, 16 bytes (pairs of neighbours, or elements past rot), or E pairs of
// halves; the first ones are asked for before the angles are formed.  WHOLE: every item is, so nothing looks for an end.
template <typename ET, bool INTER, bool WHOLE, int E, int IT>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryParams p, int most) {
    extern __shared__ float2v turn[];        // [tok][rot / 2]
    const RotaryPart q = p.part[blockIdx.y];
    const int r = udiv_small(blockIdx.x, most), block = blockIdx.x - r * most;
    if (block >= q.blocks) return;           // another part, of fewer tokens a block, has more; past them i0 would pass 32 bits
    const int i0 = block * q.tok;
    int n = p.count ? p.count[r] : p.n;
    n = n > p.n ? p.n : n;
    if (i0 >= n) return;
    const int toks = n - i0 < q.tok ? n - i0 : q.tok, pairs = p.rot / 2, rest = p.dk - p.rot;
    const int turned = INTER ? (p.rot + E - 1) / E : (pairs + E - 1) / E, items = turned + (rest + E - 1) / E, per = q.heads * items;
    const int all = toks * per;
    const ET* from = (const ET*)q.src + r * q.s_row + i0 * q.s_tok;
    ET* to = (ET*)q.dst + r * q.d_row + i0 * q.d_tok;

    auto get = [](float (&v)[E], const ET* row, int i, int d) {
        if constexpr (E == 8) load_row8(v, row, i, WHOLE ? i + 8 : d);
        else load_row4(v, row, i, WHOLE ? i + 4 : d);
    };
    auto put = [](ET* row, const float (&v)[E], int i, int d) {
        if constexpr (E == 8) store_row8(row, v, i, WHOLE ? i + 8 : d);
        else store_row4(row, v, i, WHOLE ? i + 4 : d);
    };
    // at: an item's first pair, or -1 - its first element past rot; whole elements and pairs beyond a head's end are zeros
    float a[IT][E], b[IT][E] = {};
    const ET* src[IT];
    ET* dst[IT];
    int at[IT], tok[IT];
    auto load = [&](int j0) {
#pragma unroll
        for (int u = 0; u < IT; ++u) {
            const int j = j0 + 256 * u < all ? j0 + 256 * u : 0;
            tok[u] = udiv_small(j, per);
            const int hi = j - tok[u] * per, h = udiv_small(hi, items), it = hi - h * items;
            src[u] = from + tok[u] * q.s_tok + h * q.s_head;
            dst[u] = to + tok[u] * q.d_tok + h * q.d_head;
            at[u] = it >= turned ? -1 - E * (it - turned) : INTER ? E / 2 * it : E * it;
            if (j0 + 256 * u >= all) dst[u] = nullptr;
            const bool other = at[u] < 0;
            if (other && src[u] == dst[u]) dst[u] = nullptr;
            // what an item reads past its end is the same head's and goes nowhere; only the head's end is looked for
            get(a[u], src[u] + (other ? p.rot : 0), other ? -1 - at[u] : INTER ? 2 * at[u] : at[u], other ? rest : p.dk);
            if (!INTER && !other) get(b[u], src[u] + pairs, at[u], p.dk - pairs);
        }
    };
    auto turn_and_store = [&]() {
#pragma unroll
        for (int u = 0; u < IT; ++u) {
            if (!dst[u]) continue;
            const bool other = at[u] < 0;
            const float2v* cs = turn + tok[u] * pairs + (other ? 0 : at[u]);
            float o[E], o2[E];
#pragma unroll
            for (int e = 0; e < (INTER ? E / 2 : E); ++e) {
                const float2v c = (WHOLE ? !other : !other && at[u] + e < pairs) ? cs[e] : float2v{0.f, 0.f};
                const float v = INTER ? a[u][2 * (e % (E / 2))] : a[u][e], w = INTER ? a[u][2 * (e % (E / 2)) + 1] : b[u][e];
                const float x = v * c[0] - w * c[1], y = w * c[0] + v * c[1];
                if (INTER) {
                    o[2 * (e % (E / 2))] = other ? v : x;
                    o[2 * (e % (E / 2)) + 1] = other ? w : y;
                } else {
                    o[e] = other ? v : x;
                    o2[e] = y;
                }
            }
            put(dst[u] + (other ? p.rot : 0), o, other ? -1 - at[u] : INTER ? 2 * at[u] : at[u], other ? rest : INTER ? p.rot : pairs);
            if (!INTER && !other) put(dst[u] + pairs, o2, at[u], pairs);
        }
    };

    load(threadIdx.x);
    const int64_t first = p.start ? p.start[r] : 0;
    for (int j = threadIdx.x; j < toks * pairs; j += 256) {
        const int i = udiv_small(j, pairs), f = j - i * pairs;
        const int64_t where = p.pos ? p.pos[r * p.pos_row + i0 + i] : first + i0 + i;
        const float2v cs = cos_sin_turns((double)where * p.freq[f] * 0.159154943091895335769);
        turn[j] = float2v{cs[0] * p.mult, cs[1] * p.mult};
    }
    __syncthreads();
    for (int j = threadIdx.x;;) {
        turn_and_store();
        j += 256 * IT;
        if (j >= all) break;
        load(j);
    }
}

template <typename ET, bool INTER, bool WHOLE, int E, int IT> void launch_typed(RotaryParams p, hipStream_t s) {
    const int pairs = p.rot / 2, items = cdiv(INTER ? p.rot : pairs, E) + cdiv(p.dk - p.rot, E);
    int most = 1, lds = 0;
    for (int z = 0; z < p.parts; ++z) {      // as many tokens as give every thread its IT items, within 32 KB of angles
        int tok = 256 * IT / (p.part[z].heads * items);
        if (tok * pairs > 4096) tok = 4096 / pairs;
        tok = tok < 1 ? 1 : tok > p.n ? p.n : tok;
        p.part[z].tok = tok;
        p.part[z].blocks = cdiv(p.n, tok);
        most = p.part[z].blocks > most ? p.part[z].blocks : most;
        lds = tok * pairs * 8 > lds ? tok * pairs * 8 : lds;
    }
    require((double)p.R * most < (double)(1 << 22), "rotary: too many tokens for one call");
    launch(rotary_kernel<ET, INTER, WHOLE, E, IT>, dim3(p.R * most, p.parts), dim3(256), lds, s, p, most);
}
// Items of 16 bytes where head and pairs divide into them, of 8 for f16 where not, and of four elements with ends looked for in
// any other case (4 x 4096 tokens x 20 heads x 80, 20 pairs of halves: 8 bytes 26.1 us, 16 with ends 37.8; 10 pairs, with ends, 48).
template <typename ET, bool INTER> void launch_items(const RotaryParams& p, hipStream_t s) {
    constexpr int E = 16 / sizeof(ET), IT = INTER ? 4 : 2;
    const int unit = INTER ? p.rot : p.rot / 2, rest = p.dk - p.rot;
    if (unit % E == 0 && rest % E == 0) launch_typed<ET, INTER, true, E, IT>(p, s);
    else if (unit % 4 == 0 && rest % 4 == 0) launch_typed<ET, INTER, true, 4, IT>(p, s);
    else launch_typed<ET, INTER, false, 4, 2>(p, s);
}

}  // namespace

void launch_rotary(const RotaryParams& p, hipStream_t s) {
    if (p.R == 0 || p.n == 0 || p.parts == 0) return;
    if (p.f32) p.interleaved ? launch_items<float, true>(p, s) : launch_items<float, false>(p, s);
    else p.interleaved ? launch_items<f16, true>(p, s) : launch_items<f16, false>(p, s);
}

}  // namespace pkx
