// Operators around an attention decoder's attention: norms with residual and
// gate, 8-bit products, rotary positions, rules on logits.
#pragma once
#include "common.hpp"

namespace pkx {

enum NormKind : int { NORM_NONE = 0, NORM_LAYER = 1, NORM_RMS = 2 };

struct BlockNormParams {
    bool f32 = false, x_f32 = true;      // y, gate and h; x and x_out
    bool h_i8 = false;                   // h in 8 bits with a scale a row
    int64_t rows = 0;
    int d = 0;
    double inv_d = 0;                    // 1 / d, set by the launch
    const void* x = nullptr;  int64_t x_row = 0;
    const void* y = nullptr;  int64_t y_row = 0;
    const void* gate = nullptr;  int64_t gate_row = 0;
    int rows_per_gate = 1, sigmoid = 0;
    int post = NORM_NONE, pre = NORM_NONE;
    const float *post_w = nullptr, *post_b = nullptr, *pre_w = nullptr, *pre_b = nullptr;
    float post_eps = 0.f, pre_eps = 0.f, alpha = 1.f;
    void* x_out = nullptr;  int64_t x_out_row = 0;
    void* h = nullptr;  int64_t h_row = 0;
    float* h_scale = nullptr;
};
constexpr int kMaxNormWidth = 16384;
void launch_block_norm(BlockNormParams p, hipStream_t s);

struct QuantizeRowsParams {
    bool f32 = false;
    int64_t rows = 0;
    int d = 0;
    const void* x = nullptr;  int64_t x_row = 0;
    int8_t* q = nullptr;  int64_t q_row = 0;
    float* scale = nullptr;
};
void launch_quantize_rows(const QuantizeRowsParams& p, hipStream_t s);

// Weights of an 8-bit product, laid out in blocks of 32 output channels x 64
// inputs (2 KB): [N / 32][K / 64][4 groups of 16 inputs][32 channels][16 bytes],
// zeros past the last channel and input, K padded to 128.
constexpr int kI8ColBlock = 32, kI8DepthBlock = 64, kI8DepthPad = 128;
inline int64_t i8_weight_bytes(int64_t N, int64_t K) {
    return (N + kI8ColBlock - 1) / kI8ColBlock * kI8ColBlock * ((K + kI8DepthPad - 1) / kI8DepthPad * kI8DepthPad);
}
void launch_i8_weight_pack(const int8_t* w, int64_t w_row, int N, int K, void* packed, hipStream_t s);

struct LinearI8Params {
    int M = 0, N = 0, K = 0;
    const int8_t* x = nullptr;  int64_t x_row = 0;
    const float* x_scale = nullptr;
    const void* w = nullptr;
    const float* w_scale = nullptr;
    const float* bias = nullptr;
    int silu = 0;
    float alpha = 1.f;
    bool y_f32 = false;
    const void* add = nullptr;  int64_t add_row = 0;
    void* y = nullptr;  int64_t y_row = 0;
    bool lines = false;                  // y's rows begin at multiples of 64 bytes, set by the launch
};
void launch_linear_i8(const LinearI8Params& p, hipStream_t s);
// The same from rows as they come, in one launch, for the few and short ones that linear_i8_fused() names.
bool linear_i8_fused(int M, int N, int K);
void launch_linear_i8_fused(const LinearI8Params& p, const QuantizeRowsParams& q, hipStream_t s);
// What a workgroup of a call takes, and how many there are (16 x 16 on 512 threads, the others on 256).
struct LinearI8Tile {
    int tokens, channels;
    int64_t workgroups;
};
LinearI8Tile linear_i8_tile(int M, int N, int K, bool i8);

constexpr int kRotaryParts = 4, kMaxRotaryWidth = 512;
struct RotaryPart {
    const void* src;  int64_t s_row, s_tok, s_head;
    void* dst;        int64_t d_row, d_tok, d_head;
    int heads;
    int tok = 1, blocks = 1;              // tokens of a workgroup, workgroups of a row: set by the launch
};
struct RotaryParams {
    bool f32 = false;
    int R = 0, n = 0, dk = 0, rot = 0, interleaved = 0, parts = 0;
    float mult = 1.f;
    const double* freq = nullptr;         // [rot / 2] radians a position
    const int* start = nullptr;           // [R], NULL: 0
    const int* pos = nullptr;  int64_t pos_row = 0;   // [R][n], NULL: start + i
    const int* count = nullptr;           // [R], NULL: n
    RotaryPart part[kRotaryParts];
};
void launch_rotary(const RotaryParams& p, hipStream_t s);

struct LogitRulesParams {
    bool f32 = false;
    int R = 0, V = 0, cap = 0, n_slots = 0, window = 0;
    const void* x = nullptr;  int64_t x_row = 0;
    void* out = nullptr;      int64_t out_row = 0;
    const int* tokens = nullptr;          // [n_slots][cap]
    const int *len = nullptr, *slot = nullptr, *table = nullptr;  int64_t table_row = 0;
    const float *repetition = nullptr, *presence = nullptr, *frequency = nullptr;   // [R]
    const float* bias = nullptr;  int64_t bias_row = 0;  int n_bias = 0;  const int* bias_index = nullptr;
    const uint32_t* mask = nullptr;  int64_t mask_row = 0;  int n_mask = 0;  const int* mask_index = nullptr;
};
void launch_logit_rules(const LogitRulesParams& p, hipStream_t s);

}  // namespace pkx
