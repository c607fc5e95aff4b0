// Operators of an attention decoder: cross attention to encoder states,
// attention over an 8-bit key/value cache, beam selection and reordering.
#pragma once
#include "common.hpp"

namespace pkx {

constexpr int kCacheBlock = 32;   // tokens that share a scale in the 8-bit cache

enum KvKind : int { KV_F16 = 0, KV_F32 = 1, KV_I8 = 2 };

// Query rows of one item and key head: m = i * G + g for query i and head
// kh * G + g.  Strides in elements; the head dimension is contiguous.
struct DecAttnParams {
    int kv = KV_F16;
    bool q_f32 = false;
    const void* q = nullptr;  int64_t q_item = 0, q_row = 0, q_head = 0;
    const void* k = nullptr;  int64_t k_item = 0, k_row = 0, k_head = 0;
    const void* v = nullptr;  int64_t v_item = 0, v_row = 0, v_head = 0;
    void* out = nullptr;      int64_t o_item = 0, o_row = 0, o_head = 0;
    // 8-bit cache: item b's keys are slot[b]'s, or position t's table[b][t]'s
    const float* k_scale = nullptr;
    const float* v_scale = nullptr;
    const int* slot = nullptr;
    const int* table = nullptr;  int64_t table_ld = 0;
    int n_slots = 0, n_blocks = 0;
    const int* q_len = nullptr;               // [B] query rows of an item, NULL: n_q
    const int* k_len = nullptr;               // [B] keys of an item, NULL: n_k
    const uint8_t* mask = nullptr;  int64_t mask_item = 0;   // [B][n_k], 0: the key is not attended
    int B = 0, n_q = 0, n_k = 0, Hkv = 0, G = 1, dk = 0;
    int causal = 0;      // query i of n sees keys t <= len - n + i
    float scale = 1.0f, scale_lo = 0.0f;      // in launches: scale log2 e, what its rounding left
    int splits = 1, split_keys = 0;
    float* part_o = nullptr;      // [row][split][D]
    float2* part_ml = nullptr;    // [row][split] {running maximum (log2 units), sum}
};
// Bytes of workspace that launch_dec_attention needs for these sizes.
size_t dec_attention_workspace(const DecAttnParams& p);
void launch_dec_attention(DecAttnParams p, void* ws, size_t ws_bytes, hipStream_t s);

struct Cache8 {
    int n_slots = 0, Hkv = 0, dk = 0, cap = 0;
    int8_t *k = nullptr, *v = nullptr;
    float *k_scale = nullptr, *v_scale = nullptr;
};
// The scales of row r's slot (slot NULL: slot r) become 0.
void launch_cache8_clear(const Cache8& c, int rows, const int* slot, hipStream_t s);

struct CacheAppendParams {
    Cache8 c;
    bool f32 = false;
    const void* k = nullptr;  int64_t k_row = 0, k_tok = 0, k_head = 0;
    const void* v = nullptr;  int64_t v_row = 0, v_tok = 0, v_head = 0;
    const int *slot = nullptr, *start = nullptr, *count = nullptr;
    int* table = nullptr;  int64_t table_ld = 0;
    int R = 0, n_new = 0;
};
void launch_cache8_append(const CacheAppendParams& p, hipStream_t s);
struct CacheReadParams {
    Cache8 c;
    const int *slot = nullptr, *start = nullptr;
    float *k = nullptr, *v = nullptr;   // [R][n][Hkv][dk]
    int R = 0, n = 0;
};
void launch_cache8_read(const CacheReadParams& p, hipStream_t s);

struct BeamSelectParams {
    bool f32 = false;
    int B = 0, W = 0, V = 0, end_id = -1;
    const void* logits = nullptr;  int64_t row = 0;   // elements between rows
    const float* scores = nullptr;
    const uint8_t* done = nullptr;
    int *parent = nullptr, *token = nullptr;
    float* new_scores = nullptr;
    uint8_t* new_done = nullptr;
};
constexpr int kMaxBeams = 32;
size_t beam_select_workspace(const BeamSelectParams& p);
void launch_beam_select(const BeamSelectParams& p, void* ws, size_t ws_bytes, hipStream_t s);

constexpr int kMaxBeamStates = 32;
struct BeamState {
    const uint8_t* src;
    uint8_t* dst;
    int64_t src_row, dst_row, bytes;
};
void launch_beam_reorder(const int* parent, int B, int W, const BeamState* states, int n, hipStream_t s);

}  // namespace pkx
