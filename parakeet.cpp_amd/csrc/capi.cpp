// extern "C" boundary (include/pkx.h).  Every entry point catches all C++
// exceptions and reports them through a thread-local last-error string, the
// same no-throw convention as the reference C API (src/parakeet_capi.cpp:207-225).
#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>
#include <string>
#include <utility>
#include <vector>

#include "../../include/pkx.h"
#include "block.hpp"
#include "decoder.hpp"
#include "mel.hpp"
#include "model.hpp"
#include "quantize.hpp"

struct pkx_mel {
    std::unique_ptr<pkx::MelFront> impl;
};

struct pkx_model {
    pkx_config cfg;
    int precision;
    std::unique_ptr<pkx::Model> impl;
};

struct pkx_streaming {
    pkx::Model* model;
    std::unique_ptr<pkx::StreamState> st;
};

// Fixed device scratch of pkx_tdt_joint_argmax_noalloc: one copy per GPU,
// held until the process ends.  Host code never passes the symbol's name as an
// address (it is a host-side stand-in there); joint_scratch() finds each GPU's
// copy with hipGetSymbolAddress (at model set-up, with the model's device
// current) and that address is used from then on.
static __device__ __align__(256) float scratch[PKX_JOINT_NOALLOC_MAX_FLOATS];

namespace {
thread_local std::string g_last_error;

template <typename F>
int guarded(F&& f) {
    try {
        f();
        g_last_error.clear();
        return 0;
    } catch (const std::exception& e) {
        g_last_error = e.what();
    } catch (...) {
        g_last_error = "unknown error";
    }
    pkx::tl_launch_hook = nullptr;   // a failed call may leave a profiled region open
    return 1;
}

hipStream_t st(void* s) { return (hipStream_t)s; }

constexpr int kMaxDevices = 64;

// Device address of this GPU's copy of `scratch` (below the namespace), looked
// up with hipGetSymbolAddress once per device with that device current.

float* joint_scratch() {
    static std::mutex mu;
    static float* ptr[kMaxDevices] = {};
    int dev = 0;
    PKX_HIP(hipGetDevice(&dev));
    if (dev < 0 || dev >= kMaxDevices) throw std::invalid_argument("device index out of range");
    std::lock_guard<std::mutex> lock(mu);
    if (!ptr[dev]) {
        void* p = nullptr;
        PKX_HIP(hipGetSymbolAddress(&p, HIP_SYMBOL(scratch)));
        // the code objects of the kernels the entry point launches, loaded now
        // rather than at its first launch
        pkx::gemm_module_ready();
        pkx::elementwise_module_ready();
        ptr[dev] = (float*)p;
    }
    return ptr[dev];
}

void need(bool ok, const char* what) {
    if (!ok) throw std::invalid_argument(what);
}

pkx::ModelConfig to_internal(const pkx_config& c) {
    pkx::ModelConfig m;
    m.d_model = c.d_model;
    m.n_layers = c.n_layers;
    m.n_heads = c.n_heads;
    m.ff_dim = c.ff_dim;
    m.conv_kernel = c.conv_kernel;
    m.n_mels = c.n_mels;
    m.sub_channels = c.sub_channels;
    m.xscaling = c.xscaling;
    m.vocab_size = c.vocab_size;
    m.n_durations = c.n_durations;
    m.conv_ln = c.conv_ln;
    m.causal_sub = c.causal_sub;
    m.conv_causal = c.conv_causal;
    m.att_limited = c.att_limited;
    m.att_left = c.att_left;
    m.att_right = c.att_right;
    m.stream_chunk_first = c.stream_chunk_first;
    m.stream_chunk = c.stream_chunk;
    m.stream_pre_cache = c.stream_pre_cache;
    m.stream_cache_len = c.stream_cache_len;
    m.stream_valid_out_len = c.stream_valid_out_len;
    m.stream_drop_extra = c.stream_drop_extra;
    return m;
}

pkx_config to_public(const pkx::ModelConfig& m) {
    pkx_config c;
    c.d_model = m.d_model;
    c.n_layers = m.n_layers;
    c.n_heads = m.n_heads;
    c.ff_dim = m.ff_dim;
    c.conv_kernel = m.conv_kernel;
    c.n_mels = m.n_mels;
    c.sub_channels = m.sub_channels;
    c.xscaling = m.xscaling;
    c.vocab_size = m.vocab_size;
    c.n_durations = m.n_durations;
    c.conv_ln = m.conv_ln;
    c.causal_sub = m.causal_sub;
    c.conv_causal = m.conv_causal;
    c.att_limited = m.att_limited;
    c.att_left = m.att_left;
    c.att_right = m.att_right;
    c.stream_chunk_first = m.stream_chunk_first;
    c.stream_chunk = m.stream_chunk;
    c.stream_pre_cache = m.stream_pre_cache;
    c.stream_cache_len = m.stream_cache_len;
    c.stream_valid_out_len = m.stream_valid_out_len;
    c.stream_drop_extra = m.stream_drop_extra;
    return c;
}

// A stream of another device than the current one: the launch would go astray.
void need_device(hipStream_t s) {
    if (!s) return;
    int cur = 0;
    hipDevice_t dev = 0;
    PKX_HIP(hipGetDevice(&cur));
    PKX_HIP(hipStreamGetDevice(s, &dev));
    need(dev == cur, "the stream belongs to another device than the current one");
}

bool is_f32(int type, const char* what) {
    need(type == PKX_TYPE_F32 || type == PKX_TYPE_F16, what);
    return type == PKX_TYPE_F32;
}

// Rows of an output that do not run into each other: each stride at least what the
// smaller ones span.
void need_apart(int64_t a, int64_t na, int64_t b, int64_t nb, int64_t c, int64_t nc, int64_t row, const char* what) {
    std::pair<int64_t, int64_t> dim[3] = {{a, na}, {b, nb}, {c, nc}};
    std::sort(dim, dim + 3);
    double span = (double)row;
    for (const auto& [stride, n] : dim) {
        if (n <= 1) continue;
        need((double)stride >= span, what);
        span += (double)stride * (double)(n - 1);
    }
}

// What the kernels' 32-bit indexes hold; in f64, where no product of sizes wraps.
void need_rows(int items, int n_q, int heads) {
    need((double)items * n_q * heads < (double)(1 << 22), "attention: at most 2^22 rows x heads in one call");
}

// A strided operand read or written in 16-byte pieces.
void need_view(const void* p, int64_t a, int64_t b, int64_t c, bool f32, const char* what) {
    const int64_t unit = f32 ? 4 : 8;
    need(p != nullptr && (uintptr_t)p % 16 == 0, what);
    need(a >= 0 && b >= 0 && c >= 0 && a % unit == 0 && b % unit == 0 && c % unit == 0, what);
}

pkx::DecAttnParams cross_params(const pkx_cross_attn* a) {
    need(a, "null argument");
    const bool f32 = is_f32(a->type, "cross attention: type must be PKX_TYPE_F32 or PKX_TYPE_F16");
    need(a->n_items >= 0 && a->n_q >= 0 && a->n_k >= 0, "cross attention: negative size");
    need(a->n_k <= (1 << 30), "cross attention: more than 2^30 keys");
    need(a->n_heads >= 1 && a->n_kv_heads >= 1 && a->n_heads % a->n_kv_heads == 0,
         "cross attention: n_heads must be a multiple of n_kv_heads");
    need(a->d_head >= 8 && a->d_head <= 128 && a->d_head % 8 == 0, "cross attention: d_head must be a multiple of 8 up to 128");
    pkx::DecAttnParams p;
    p.kv = f32 ? pkx::KV_F32 : pkx::KV_F16;
    p.q_f32 = f32;
    p.B = a->n_items;
    p.n_q = a->n_q;
    p.n_k = a->n_k;
    p.Hkv = a->n_kv_heads;
    p.G = a->n_heads / a->n_kv_heads;
    p.dk = a->d_head;
    need_rows(a->n_items, a->n_q, a->n_heads);
    need(std::isfinite(a->scale * 2.0f), "cross attention: scale is not finite");
    need(!a->k_mask || a->k_mask_item >= 0, "cross attention: negative stride of k_mask");
    p.scale = a->scale;
    p.q = a->q; p.q_item = a->q_item; p.q_row = a->q_row; p.q_head = a->q_head;
    p.k = a->k; p.k_item = a->k_item; p.k_row = a->k_row; p.k_head = a->k_head;
    p.v = a->v; p.v_item = a->v_item; p.v_row = a->v_row; p.v_head = a->v_head;
    p.out = a->out; p.o_item = a->out_item; p.o_row = a->out_row; p.o_head = a->out_head;
    p.q_len = a->q_len;
    p.k_len = a->k_len;
    p.mask = a->k_mask;
    p.mask_item = a->k_mask_item;
    return p;
}

pkx::Cache8 cache_params(const pkx_cache8* c) {
    need(c, "null argument");
    need(c->n_slots >= 1 && c->n_kv_heads >= 1, "8-bit cache: no slots or heads");
    need(c->d_head >= 16 && c->d_head <= 128 && c->d_head % 16 == 0, "8-bit cache: d_head must be a multiple of 16 up to 128");
    need(c->capacity >= PKX_CACHE8_BLOCK && c->capacity % PKX_CACHE8_BLOCK == 0 && c->capacity <= (1 << 30),
         "8-bit cache: capacity must be a multiple of PKX_CACHE8_BLOCK up to 2^30");
    need(c->k && c->v && c->k_scale && c->v_scale, "8-bit cache: null buffer");
    need(((uintptr_t)c->k | (uintptr_t)c->v) % 16 == 0 && ((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) % 4 == 0,
         "8-bit cache: k and v must be 16-byte aligned");
    pkx::Cache8 o;
    o.n_slots = c->n_slots;
    o.Hkv = c->n_kv_heads;
    o.dk = c->d_head;
    o.cap = c->capacity;
    o.k = c->k;
    o.v = c->v;
    o.k_scale = c->k_scale;
    o.v_scale = c->v_scale;
    return o;
}

pkx::DecAttnParams cache_attn_params(const pkx_cache8* c, const pkx_cache8_attn* a) {
    const pkx::Cache8 o = cache_params(c);
    need(a, "null argument");
    pkx::DecAttnParams p;
    p.kv = pkx::KV_I8;
    p.q_f32 = is_f32(a->type, "cache attention: type must be PKX_TYPE_F32 or PKX_TYPE_F16");
    need(a->n_rows >= 0 && a->n_q >= 0, "cache attention: negative size");
    need(a->n_heads >= 1 && a->n_heads % o.Hkv == 0, "cache attention: n_heads must be a multiple of the cache's heads");
    need(a->max_len >= 0, "cache attention: negative max_len");
    p.B = a->n_rows;
    p.n_q = a->n_q;
    p.n_k = a->max_len > 0 && a->max_len < o.cap ? a->max_len : o.cap;
    p.Hkv = o.Hkv;
    p.G = a->n_heads / o.Hkv;
    p.dk = o.dk;
    need_rows(a->n_rows, a->n_q, a->n_heads);
    need(std::isfinite(a->scale * 2.0f), "cache attention: scale is not finite");
    p.scale = a->scale;
    p.causal = a->causal != 0;
    p.q = a->q; p.q_item = a->q_row; p.q_row = a->q_tok; p.q_head = a->q_head;
    p.out = a->out; p.o_item = a->out_row; p.o_row = a->out_tok; p.o_head = a->out_head;
    p.k = o.k;
    p.v = o.v;
    p.k_item = p.v_item = (int64_t)o.Hkv * o.cap * o.dk;
    p.k_head = p.v_head = (int64_t)o.cap * o.dk;
    p.k_row = p.v_row = o.dk;
    p.k_scale = o.k_scale;
    p.v_scale = o.v_scale;
    p.n_slots = o.n_slots;
    p.n_blocks = o.cap / PKX_CACHE8_BLOCK;
    p.slot = a->slot;
    p.table = a->table;
    p.table_ld = a->table_row;
    p.k_len = a->len;
    p.q_len = a->q_len;
    return p;
}

pkx::BeamSelectParams beam_params(const pkx_beam_select_args* a) {
    need(a, "null argument");
    pkx::BeamSelectParams p;
    p.f32 = is_f32(a->type, "beam select: type must be PKX_TYPE_F32 or PKX_TYPE_F16");
    need(a->n_items >= 0 && a->n_beams >= 1 && a->n_beams <= pkx::kMaxBeams, "beam select: n_beams must be 1 to 32");
    need(a->vocab <= (1 << 22), "beam select: a vocabulary of at most 2^22 words");
    need(a->vocab >= 1 && a->end_id >= -1 && a->end_id < a->vocab, "beam select: end_id must be -1 or a word of the vocabulary");
    need(!a->done || a->end_id >= 0, "beam select: finished beams need an end_id");
    p.B = a->n_items;
    p.W = a->n_beams;
    p.V = a->vocab;
    p.end_id = a->end_id;
    p.logits = a->logits;
    p.row = a->logits_row;
    p.scores = a->scores;
    p.done = a->done;
    p.parent = a->parent;
    p.token = a->token;
    p.new_scores = a->new_scores;
    p.new_done = a->new_done;
    return p;
}
// A strided operand as the bytes it touches: `row` adjacent ones at every multiple of each dimension's stride.
struct Span {
    uintptr_t at;
    int64_t row;
    std::pair<int64_t, int64_t> dim[3];   // stride in bytes, count; largest stride first
    int dims = 0;

    Span(const void* p, int64_t bytes, std::initializer_list<std::pair<int64_t, int64_t>> all) : at((uintptr_t)p), row(bytes) {
        for (const auto& d : all)
            if (d.second > 1) dim[dims++] = d;
        std::sort(dim, dim + dims, [](const auto& a, const auto& b) { return a.first > b.first; });
    }
    double bytes(int from = 0) const {    // from the first byte to the last, of the dimensions from `from` on
        double n = (double)row;
        for (int i = from; i < dims; ++i) n += (double)dim[i].first * (double)(dim[i].second - 1);
        return n;
    }
};

// Whether two operands have no byte in common, as far as their strides say it: one ends before the other begins, or their
// largest strides are the same and within one period (two column ranges of the same rows) they lie apart.
bool apart(const Span& a, const Span& b) {
    if (a.at > b.at) return apart(b, a);
    if ((double)(b.at - a.at) >= a.bytes()) return true;
    uint64_t from = b.at - a.at;
    for (int i = 0; i < a.dims && i < b.dims; ++i) {
        if (a.dim[i].first != b.dim[i].first || a.dim[i].first <= 0) return false;
        const double period = (double)a.dim[i].first, na = a.bytes(i + 1), nb = b.bytes(i + 1);
        // b's place in a's period; neither may run into the next one
        from %= (uint64_t)a.dim[i].first;
        if (na > period || (double)from + nb > period) return false;
        if ((double)from >= na) return true;
    }
    return false;
}
bool same(const Span& a, const Span& b) {
    if (a.at != b.at || a.row != b.row || a.dims != b.dims) return false;
    return std::equal(a.dim, a.dim + a.dims, b.dim);
}

// Rows of n elements of e bytes, `count` of them `stride` elements apart.
Span rows_of(const void* p, int64_t n, int64_t e, int64_t stride, int64_t count) { return Span(p, n * e, {{stride * e, count}}); }

// Addresses and extents that 64-bit byte arithmetic holds.
void need_rows_of(const void* p, int e, int64_t stride, int64_t count, int64_t least, const char* what) {
    need(p && (uintptr_t)p % e == 0 && (stride >= least || (count <= 1 && stride >= 0)), what);
    need((double)stride * (double)count * e < 0x1p62, what);
}

void need_i8_weight(int n_out, int n_in) {
    need(n_out >= 0 && n_out < (1 << 22) && n_in >= 1 && n_in <= PKX_I8_MAX_DEPTH, "8-bit weights: n_out below 2^22 and n_in 1 to PKX_I8_MAX_DEPTH");
    need(pkx::i8_weight_bytes(n_out, n_in) < (int64_t(1) << 35), "8-bit weights: 32 GiB or more");
}
pkx::LinearI8Params linear_i8_params(const pkx_linear_i8_args* a) {
    need(a, "null argument");
    pkx::LinearI8Params p;
    p.y_f32 = is_f32(a->type, "8-bit linear: type must be PKX_TYPE_F32 or PKX_TYPE_F16");
    need(a->x_type == PKX_TYPE_I8 || a->x_type == PKX_TYPE_F32 || a->x_type == PKX_TYPE_F16,
         "8-bit linear: x_type must be PKX_TYPE_I8, PKX_TYPE_F32 or PKX_TYPE_F16");
    need(a->n_rows >= 0 && a->n_out >= 0 && a->n_in >= 1 && a->n_in <= PKX_I8_MAX_DEPTH,
         "8-bit linear: negative size, or n_in outside 1 to PKX_I8_MAX_DEPTH");
    need(a->n_rows < (1 << 22) && a->n_out < (1 << 22) && (double)a->n_rows * a->n_out < 0x1p36,
         "8-bit linear: n_rows and n_out below 2^22, and 2^36 outputs in one call");
    need(a->act == PKX_ACT_NONE || a->act == PKX_ACT_SILU, "8-bit linear: act must be PKX_ACT_NONE or PKX_ACT_SILU");
    need(std::isfinite(a->alpha), "8-bit linear: alpha is not finite");
    p.M = a->n_rows;
    p.N = a->n_out;
    p.K = a->n_in;
    p.w = a->w;
    p.w_scale = a->w_scale;
    p.bias = a->bias;
    p.silu = a->act == PKX_ACT_SILU;
    p.alpha = a->alpha;
    p.add = a->add;
    p.add_row = a->add_row;
    p.y = a->y;
    p.y_row = a->y_row;
    return p;
}
// Quantised tokens in the workspace: rows of whole 16 bytes, then their scales.
int64_t i8_row(const pkx_linear_i8_args* a) { return ((int64_t)a->n_in + 15) / 16 * 16; }
size_t i8_workspace(const pkx_linear_i8_args* a) {
    return a->x_type == PKX_TYPE_I8 || a->n_rows == 0 || a->n_out == 0 || pkx::linear_i8_fused(a->n_rows, a->n_out, a->n_in) ? 0 : (size_t)a->n_rows * (i8_row(a) + 4);
}
// Every element where it was: a stride counts where its dimension has more than one.
bool in_place(const pkx::RotaryPart& p, int64_t rows, int64_t toks) {
    return p.src == p.dst && (rows <= 1 || p.s_row == p.d_row) && (toks <= 1 || p.s_tok == p.d_tok) && (p.heads <= 1 || p.s_head == p.d_head);
}
pkx::QuantizeRowsParams quantize_rows_params(int type, const void* x, int64_t x_row, int64_t n_rows, int n) {
    pkx::QuantizeRowsParams p;
    p.f32 = is_f32(type, "quantise rows: type must be PKX_TYPE_F32 or PKX_TYPE_F16");
    need(n_rows >= 0 && n_rows < (1 << 22) && n >= 0, "quantise rows: negative size, or 2^22 rows");
    if (n_rows > 0) need_rows_of(x, p.f32 ? 4 : 2, x_row, n_rows, 0, "quantise rows: x is null, misaligned or of a negative stride");
    p.rows = n_rows;
    p.d = n;
    p.x = x;
    p.x_row = x_row;
    return p;
}
}  // namespace

extern "C" {

int pkx_abi_version(void) { return PKX_ABI_VERSION; }
const char* pkx_last_error(void) { return g_last_error.c_str(); }

int pkx_device_count(int* n) {
    return guarded([&] { need(n, "null n"); PKX_HIP(hipGetDeviceCount(n)); });
}
int pkx_malloc(void** dev, size_t bytes) {
    return guarded([&] { need(dev, "null out"); PKX_HIP(hipMalloc(dev, bytes ? bytes : 16)); });
}
int pkx_free(void* dev) {
    return guarded([&] { if (dev) PKX_HIP(hipFree(dev)); });
}
int pkx_mem_info(size_t* free_bytes, size_t* total_bytes) {
    return guarded([&] {
        need(free_bytes && total_bytes, "null out");
        PKX_HIP(hipMemGetInfo(free_bytes, total_bytes));
    });
}
int pkx_memcpy_h2d(void* dst, const void* src, size_t bytes, void* s) {
    return guarded([&] {
        PKX_HIP(hipMemcpyAsync(dst, src, bytes, hipMemcpyHostToDevice, st(s)));
        PKX_HIP(hipStreamSynchronize(st(s)));
    });
}
int pkx_memcpy_d2h(void* dst, const void* src, size_t bytes, void* s) {
    return guarded([&] {
        PKX_HIP(hipMemcpyAsync(dst, src, bytes, hipMemcpyDeviceToHost, st(s)));
        PKX_HIP(hipStreamSynchronize(st(s)));
    });
}
int pkx_memcpy_d2d(void* dst, const void* src, size_t bytes, void* s) {
    return guarded([&] { PKX_HIP(hipMemcpyAsync(dst, src, bytes, hipMemcpyDeviceToDevice, st(s))); });
}
int pkx_stream_create(void** s) {
    return guarded([&] {
        need(s, "null out");
        hipStream_t h;
        PKX_HIP(hipStreamCreateWithFlags(&h, hipStreamNonBlocking));
        *s = h;
    });
}
int pkx_stream_destroy(void* s) {
    return guarded([&] { if (s) PKX_HIP(hipStreamDestroy(st(s))); });
}
int pkx_stream_synchronize(void* s) {
    return guarded([&] { PKX_HIP(hipStreamSynchronize(st(s))); });
}
int pkx_event_create(void** e) {
    return guarded([&] {
        need(e, "null out");
        hipEvent_t h;
        PKX_HIP(hipEventCreate(&h));
        *e = h;
    });
}
int pkx_event_destroy(void* e) {
    return guarded([&] { if (e) PKX_HIP(hipEventDestroy((hipEvent_t)e)); });
}
int pkx_event_record(void* e, void* s) {
    return guarded([&] { PKX_HIP(hipEventRecord((hipEvent_t)e, st(s))); });
}
int pkx_event_elapsed_ms(float* ms, void* a, void* b) {
    return guarded([&] {
        need(ms && a && b, "null argument");
        PKX_HIP(hipEventSynchronize((hipEvent_t)b));
        PKX_HIP(hipEventElapsedTime(ms, (hipEvent_t)a, (hipEvent_t)b));
    });
}

int pkx_model_load_gguf(const char* path, int precision, pkx_model** out) {
    return guarded([&] {
        need(path && out, "null argument");
        *out = nullptr;
        std::unique_ptr<pkx::Model> impl = pkx::load_gguf(path, precision);
        (void)joint_scratch();   // set-up: this GPU's scratch address (see pkx_model_finalize)
        pkx_model* m = new pkx_model;
        m->cfg = to_public(impl->config());
        m->precision = impl->precision();
        m->impl = std::move(impl);
        *out = m;
    });
}

int pkx_gguf_read_kv(const char* path, pkx_gguf_kv_fn fn, void* user) {
    return guarded([&] {
        need(path && fn, "null argument");
        std::vector<pkx_gguf_str> tmp;
        pkx::read_gguf_kv(path, [&](const std::string& key, int type, int et, uint64_t n, const void* raw,
                                    const std::vector<std::string>* strs) {
            if (strs) {
                tmp.resize(strs->size());
                for (size_t i = 0; i < strs->size(); ++i) tmp[i] = pkx_gguf_str{(*strs)[i].data(), (*strs)[i].size()};
                fn(user, key.c_str(), type, et, n, tmp.data());
            } else {
                fn(user, key.c_str(), type, et, n, raw);
            }
        });
    });
}

int pkx_model_create(const pkx_config* cfg, int precision, pkx_model** out) {
    return guarded([&] {
        need(cfg && out, "null argument");
        need(precision >= -1 && precision <= 1, "precision must be PKX_PREC_AUTO/F32/F16");
        *out = nullptr;
        pkx_model* m = new pkx_model;
        m->cfg = *cfg;
        m->precision = precision;
        try {
            m->impl.reset(new pkx::Model(to_internal(*cfg), precision));
        } catch (...) {
            delete m;
            throw;
        }
        *out = m;
    });
}

int pkx_model_set_tensor(pkx_model* m, const char* name, int gtype, int n_dims, const int64_t* ne,
                         const void* data, size_t nbytes) {
    return guarded([&] {
        need(m && name && ne && data, "null argument");
        m->impl->set_tensor(name, gtype, n_dims, ne, data, nbytes);
    });
}

int pkx_model_finalize(pkx_model* m) {
    return guarded([&] {
        need(m, "null model");
        m->impl->finalize();
        m->precision = m->impl->precision();
        // Set-up of pkx_tdt_joint_argmax_noalloc on this GPU: the symbol lookup
        // (the first one on a device materialises the array's storage) happens
        // here, so that entry point itself takes no device memory.
        (void)joint_scratch();
    });
}

int pkx_model_free(pkx_model* m) {
    return guarded([&] { delete m; });
}

int pkx_model_info(pkx_model* m, pkx_config* cfg, int* precision, int* has_ctc, int* has_joint) {
    return guarded([&] {
        need(m, "null model");
        if (cfg) *cfg = to_public(m->impl->config());
        if (precision) *precision = m->impl->precision();
        if (has_ctc) *has_ctc = m->impl->has_ctc() ? 1 : 0;
        if (has_joint) *has_joint = m->impl->has_joint() ? 1 : 0;
    });
}

int pkx_subsampled_len(int T) { return pkx::subsampled_len(T); }
int pkx_valid_out_len(int T, int in_valid) { return pkx::valid_out_len(T, in_valid); }

int pkx_encoder_forward(pkx_model* m, const float* mel, int B, int T_max, const int* valid_T, int mask_mode,
                        float* out, int* T_out, int* valid_out, float* capture, void* s) {
    return guarded([&] {
        need(m && mel && out, "null argument");
        need(mask_mode == PKX_MASK_BATCHED || mask_mode == PKX_MASK_SCALAR, "bad mask_mode");
        const int Tp = m->impl->encoder_forward(mel, B, T_max, valid_T, mask_mode == PKX_MASK_BATCHED, out,
                                                valid_out, capture, st(s));
        if (T_out) *T_out = Tp;
    });
}

int pkx_compact_channels_first(const float* x, int B, int T, int D, const int* valid, const int64_t* offs,
                               float* out, void* s) {
    return guarded([&] {
        need(x && valid && offs && out, "null argument");
        pkx::launch_compact_channels_first(x, B, T, D, valid, offs, out, st(s));
    });
}

int pkx_subsampling_forward(pkx_model* m, const float* mel, int B, int T_max, const int* valid_T, int mask_mode,
                            float* out, int* T_out, int* valid_out, void* s) {
    return guarded([&] {
        need(m && mel && out, "null argument");
        const int base = mask_mode & ~PKX_MASK_WHOLE_FRAMES;
        need(base == PKX_MASK_BATCHED || base == PKX_MASK_SCALAR, "bad mask_mode");
        const int Tp = m->impl->subsampling_forward(mel, B, T_max, valid_T, base == PKX_MASK_BATCHED, out,
                                                    valid_out, st(s), false,
                                                    (mask_mode & PKX_MASK_WHOLE_FRAMES) != 0);
        if (T_out) *T_out = Tp;
    });
}

int pkx_conformer_layer_forward(pkx_model* m, int layer, const float* x, int B, int T, const int* valid,
                                const float* pos_emb, float* out, float* conv_out, void* s) {
    return guarded([&] {
        need(m && x && out, "null argument");
        m->impl->conformer_layer_forward(layer, x, B, T, valid, pos_emb, out, conv_out, st(s));
    });
}

int pkx_relpos_attention_forward(pkx_model* m, int layer, const float* x, int B, int T, const int* valid,
                                 const float* pos_emb, float* out, void* s) {
    return guarded([&] {
        need(m && x && out, "null argument");
        m->impl->relpos_attention_forward(layer, x, B, T, valid, pos_emb, out, st(s));
    });
}

int pkx_conv_module_forward(pkx_model* m, int layer, const float* c, int B, int T, const int* valid,
                            float* out, void* s) {
    return guarded([&] {
        need(m && c && out, "null argument");
        m->impl->conv_module_forward(layer, c, B, T, valid, out, st(s));
    });
}

int pkx_ctc_forward(pkx_model* m, const float* enc, int64_t M, float* logprobs, int32_t* argmax, void* s) {
    return guarded([&] {
        need(m && enc && logprobs && argmax, "null argument");
        m->impl->ctc_forward(enc, M, logprobs, argmax, st(s));
    });
}

int pkx_tdt_joint_argmax(pkx_model* m, const float* enc, int64_t M, const float* g, float* logits, int32_t* tok,
                         int32_t* dur, void* s) {
    return guarded([&] {
        need(m && enc && g && logits && tok && dur, "null argument");
        m->impl->tdt_joint_argmax(enc, M, g, logits, tok, dur, st(s));
    });
}

int pkx_tdt_joint_argmax_noalloc(pkx_model* m, const float* enc, int64_t M, const float* g, float* logits,
                                 int32_t* tok, int32_t* dur, void* s) {
    return guarded([&] {
        need(m && enc && g && logits && tok && dur, "null argument");
        need(m->impl->has_joint(), "model has no TDT joint");
        const int64_t Hj = m->impl->joint_hidden();
        need(M >= 1, "joint: no frames");
        // scratch layout: pp [Hj] at 0, hid [M][Hj] from the next 256-byte boundary
        const int64_t hid_off = (Hj + 63) / 64 * 64;
        need(M <= ((int64_t)PKX_JOINT_NOALLOC_MAX_FLOATS - hid_off) / Hj,
             "pkx_tdt_joint_argmax_noalloc: M frames need more than the fixed scratch array of "
             "PKX_JOINT_NOALLOC_MAX_FLOATS floats (at most (PKX_JOINT_NOALLOC_MAX_FLOATS - joint_hidden) / "
             "joint_hidden frames); use pkx_tdt_joint_argmax");
        float* sc = joint_scratch();
        m->impl->tdt_joint_argmax_in(enc, M, g, logits, tok, dur, sc, sc + hid_off, st(s));
    });
}

int pkx_dequantize(int gtype, const void* src, float* dst, int64_t n, void* s) {
    return guarded([&] {
        need(src && dst, "null argument");
        pkx::launch_dequantize(gtype, src, dst, n, st(s));
    });
}

int pkx_linear(int precision, int gtype, int N, int K, const void* host_w, size_t nbytes, const float* bias,
               const float* x, int64_t M, float* y, void* s) {
    return guarded([&] {
        need(host_w && x && y, "null argument");
        need(precision == PKX_PREC_F32 || precision == PKX_PREC_F16, "precision must be F32 or F16");
        pkx::HostTensor t;
        t.gtype = gtype;
        t.n_dims = 2;
        t.ne[0] = K;
        t.ne[1] = N;
        t.bytes.assign((const uint8_t*)host_w, (const uint8_t*)host_w + nbytes);
        pkx::linear_raw((pkx::Precision)precision, t, N, K, bias, x, M, y, st(s));
    });
}

int pkx_linear_residual(int precision, int gtype, int N, int K, const void* host_w, size_t nbytes, const float* bias,
                        const float* x, int64_t M, float alpha, float* y, void* s) {
    return guarded([&] {
        need(host_w && x && y, "null argument");
        need(precision == PKX_PREC_F32 || precision == PKX_PREC_F16, "precision must be F32 or F16");
        pkx::HostTensor t;
        t.gtype = gtype;
        t.n_dims = 2;
        t.ne[0] = K;
        t.ne[1] = N;
        t.bytes.assign((const uint8_t*)host_w, (const uint8_t*)host_w + nbytes);
        pkx::linear_raw((pkx::Precision)precision, t, N, K, bias, x, M, y, st(s), true, alpha);
    });
}

int pkx_layernorm(const float* x, const float* g, const float* b, float* y, int64_t M, int D, float eps,
                  void* s) {
    return guarded([&] {
        need(x && g && b && y, "null argument");
        pkx::LnParams p;
        p.x = x;
        p.g = g;
        p.b = b;
        p.y = y;
        p.M = M;
        p.D = D;
        p.eps = eps;
        pkx::launch_layernorm(pkx::PREC_F32, p, st(s));
    });
}

int pkx_rel_pos_encoding(int T, int D, float* out, void* s) {
    return guarded([&] {
        need(out && T > 0 && D > 0, "bad argument");
        pkx::launch_rel_pos_encoding(pkx::PREC_F32, out, T, D, st(s));
    });
}

int pkx_model_set_profiling(pkx_model* m, unsigned family_mask, int stride) {
    return guarded([&] {
        need(m, "null model");
        m->impl->set_profiling(family_mask, stride);
    });
}

int pkx_model_profile_read(pkx_model* m, double* ms, int64_t* launches) {
    return guarded([&] {
        need(m, "null model");
        m->impl->profile_read(ms, launches);
    });
}

int pkx_transducer_greedy(pkx_model* m, const float* enc, int B, int T_max, const int* T_valid,
                          const int32_t* durations, int n_durations, int blank_id, int max_symbols, int cap,
                          int32_t* ids, int32_t* frames, float* conf, int32_t* span, int* counts, void* s) {
    return guarded([&] {
        need(m && enc, "null argument");
        m->impl->transducer_greedy(enc, B, T_max, T_valid, durations, n_durations, blank_id, max_symbols, cap, ids,
                                   frames, conf, span, counts, st(s));
    });
}
int pkx_streaming_create(pkx_model* m, int n_streams, int max_window, void* s, pkx_streaming** out) {
    return guarded([&] {
        need(m && out, "null argument");
        *out = nullptr;
        std::unique_ptr<pkx_streaming> h(new pkx_streaming);
        h->model = m->impl.get();
        h->st = h->model->stream_create(n_streams, max_window, st(s));
        *out = h.release();
    });
}
int pkx_streaming_free(pkx_streaming* h) {
    return guarded([&] { delete h; });
}
int pkx_streaming_reset(pkx_streaming* h, void* s) {
    return guarded([&] {
        need(h, "null argument");
        h->model->stream_reset(*h->st, st(s));
    });
}
int pkx_streaming_info(const pkx_streaming* h, int* chunk_first, int* chunk, int* pre_cache, int* valid_out_len,
                       int* step) {
    return guarded([&] {
        need(h, "null argument");
        const pkx::ModelConfig& c = h->model->config();
        if (chunk_first) *chunk_first = c.stream_chunk_first;
        if (chunk) *chunk = c.stream_chunk;
        if (pre_cache) *pre_cache = c.stream_pre_cache;
        if (valid_out_len) *valid_out_len = c.stream_valid_out_len;
        if (step) *step = h->st->step;
    });
}
int pkx_streaming_chunk_len(const pkx_streaming* h, int n) { return h ? h->model->stream_chunk_len(*h->st, n) : -1; }
int pkx_streaming_step(pkx_streaming* h, const float* mel, int n, int is_last, float* out, int* n_valid, void* s) {
    return guarded([&] {
        need(h && mel && out && n_valid, "null argument");
        *n_valid = h->model->stream_step(*h->st, mel, n, is_last != 0, out, st(s));
    });
}
int pkx_mel_create(const pkx_mel_config* cfg, const float* window, int window_len, const float* fb,
                   pkx_mel** out) {
    return guarded([&] {
        need(cfg && out && window && fb, "null argument");
        *out = nullptr;
        pkx::MelConfig c;
        c.n_fft = cfg->n_fft;
        c.win_length = window_len;
        c.hop = cfg->hop_length;
        c.n_mels = cfg->n_mels;
        c.per_feature = cfg->per_feature ? 1 : 0;
        c.preemph = cfg->preemph;
        c.mag_power = cfg->mag_power;
        c.log_guard = cfg->log_zero_guard;
        std::unique_ptr<pkx_mel> h(new pkx_mel);
        h->impl.reset(new pkx::MelFront(c, window, window_len, fb));
        *out = h.release();
    });
}
int pkx_mel_load_gguf(const char* path, pkx_mel** out) {
    return guarded([&] {
        need(path && out, "null argument");
        *out = nullptr;
        pkx::MelConfig c;
        std::vector<float> window, fb;
        pkx::load_mel_gguf(path, c, window, fb);
        std::unique_ptr<pkx_mel> h(new pkx_mel);
        h->impl.reset(new pkx::MelFront(c, window.data(), (int)window.size(), fb.data()));
        *out = h.release();
    });
}
int pkx_mel_free(pkx_mel* m) {
    return guarded([&] { delete m; });
}
int pkx_mel_info(const pkx_mel* m, pkx_mel_config* cfg) {
    return guarded([&] {
        need(m && cfg, "null argument");
        const pkx::MelConfig& c = m->impl->config();
        cfg->n_fft = c.n_fft;
        cfg->win_length = c.win_length;
        cfg->hop_length = c.hop;
        cfg->n_mels = c.n_mels;
        cfg->per_feature = c.per_feature;
        cfg->preemph = c.preemph;
        cfg->mag_power = c.mag_power;
        cfg->log_zero_guard = c.log_guard;
    });
}
int pkx_mel_frames(const pkx_mel* m, int n_samples) { return m ? m->impl->frames(n_samples) : -1; }
int pkx_mel_forward(pkx_mel* m, const float* pcm, int B, int64_t S_stride, const int* n_samples, float* mel,
                    int T_max, int* T_out, void* s) {
    return guarded([&] {
        need(m != nullptr, "null mel handle");
        m->impl->forward(pcm, B, S_stride, n_samples, mel, T_max, T_out, st(s));
    });
}

int pkx_quantize(int gtype, const float* src, void* dst, int64_t n_rows, int64_t n_per_row, void* s) {
    return guarded([&] {
        need(src && dst, "null buffer");
        pkx::quantize_rows(gtype, src, dst, n_rows, n_per_row, st(s));
    });
}
int pkx_quantize_gguf(const char* in_path, const char* out_path, int gtype, int* n_quantized, int* n_kept,
                      int* n_skipped) {
    return guarded([&] {
        need(in_path && out_path, "null path");
        const pkx::QuantizeCounts c = pkx::quantize_gguf(in_path, out_path, gtype);
        if (n_quantized) *n_quantized = c.quantized;
        if (n_kept) *n_kept = c.kept;
        if (n_skipped) *n_skipped = c.skipped;
    });
}

int pkx_cross_attention_workspace(const pkx_cross_attn* a, size_t* bytes) {
    return guarded([&] {
        need(bytes, "null argument");
        *bytes = pkx::dec_attention_workspace(cross_params(a));
    });
}
int pkx_cross_attention(const pkx_cross_attn* a, void* ws, size_t ws_bytes, void* s) {
    return guarded([&] {
        const pkx::DecAttnParams p = cross_params(a);
        if (p.B == 0 || p.n_q == 0) return;
        need_view(p.q, p.q_item, p.q_row, p.q_head, p.q_f32, "cross attention: q must be 16-byte aligned with strides of whole 16 bytes");
        need_view(p.out, p.o_item, p.o_row, p.o_head, p.q_f32, "cross attention: out must be 16-byte aligned with strides of whole 16 bytes");
        need_apart(p.o_item, p.B, p.o_row, p.n_q, p.o_head, a->n_heads, p.dk, "cross attention: rows of out overlap");
        if (p.n_k > 0) {
            need_view(p.k, p.k_item, p.k_row, p.k_head, p.q_f32, "cross attention: k must be 16-byte aligned with strides of whole 16 bytes");
            need_view(p.v, p.v_item, p.v_row, p.v_head, p.q_f32, "cross attention: v must be 16-byte aligned with strides of whole 16 bytes");
            need(p.k_row < (1 << 22) && p.v_row < (1 << 22), "cross attention: key rows must be less than 2^22 elements apart");
        }
        need_device(st(s));
        pkx::launch_dec_attention(p, ws, ws_bytes, st(s));
    });
}

int pkx_cache8_clear(const pkx_cache8* c, int n_rows, const int32_t* slot, void* s) {
    return guarded([&] {
        const pkx::Cache8 o = cache_params(c);
        need(n_rows >= 0, "cache clear: negative size");
        need(slot || n_rows <= o.n_slots, "cache clear: more rows than slots");
        need_device(st(s));
        pkx::launch_cache8_clear(o, n_rows, slot, st(s));
    });
}
int pkx_cache8_append(const pkx_cache8* c, const pkx_cache8_tokens* t, void* s) {
    return guarded([&] {
        pkx::CacheAppendParams p;
        p.c = cache_params(c);
        need(t, "null argument");
        p.f32 = is_f32(t->type, "cache append: type must be PKX_TYPE_F32 or PKX_TYPE_F16");
        need(t->n_rows >= 0 && t->n_new >= 0, "cache append: negative size");
        if (t->n_rows == 0 || t->n_new == 0) return;
        need_view(t->k, t->k_row, t->k_tok, t->k_head, p.f32, "cache append: k must be 16-byte aligned with strides of whole 16 bytes");
        need_view(t->v, t->v_row, t->v_tok, t->v_head, p.f32, "cache append: v must be 16-byte aligned with strides of whole 16 bytes");
        need(t->start, "cache append: null start");
        need(t->slot || t->n_rows <= c->n_slots, "cache append: more rows than slots");
        need(!t->table || t->table_row >= c->capacity, "cache append: table rows are shorter than the capacity");
        p.k = t->k; p.k_row = t->k_row; p.k_tok = t->k_tok; p.k_head = t->k_head;
        p.v = t->v; p.v_row = t->v_row; p.v_tok = t->v_tok; p.v_head = t->v_head;
        p.slot = t->slot;
        p.start = t->start;
        p.count = t->count;
        p.table = t->table;
        p.table_ld = t->table_row;
        p.R = t->n_rows;
        p.n_new = t->n_new;
        need_device(st(s));
        pkx::launch_cache8_append(p, st(s));
    });
}
int pkx_cache8_read(const pkx_cache8* c, int n_rows, int n, const int32_t* slot, const int32_t* start, float* k_out,
                    float* v_out, void* s) {
    return guarded([&] {
        pkx::CacheReadParams p;
        p.c = cache_params(c);
        need(n_rows >= 0 && n >= 0, "cache read: negative size");
        if (n_rows == 0 || n == 0) return;
        need(start && ((uintptr_t)k_out | (uintptr_t)v_out) % 16 == 0, "cache read: null start, or outputs not 16-byte aligned");
        p.slot = slot;
        p.start = start;
        p.k = k_out;
        p.v = v_out;
        p.R = n_rows;
        p.n = n;
        need_device(st(s));
        pkx::launch_cache8_read(p, st(s));
    });
}
int pkx_cache8_attention_workspace(const pkx_cache8* c, const pkx_cache8_attn* a, size_t* bytes) {
    return guarded([&] {
        need(bytes, "null argument");
        *bytes = pkx::dec_attention_workspace(cache_attn_params(c, a));
    });
}
int pkx_cache8_attention(const pkx_cache8* c, const pkx_cache8_attn* a, void* ws, size_t ws_bytes, void* s) {
    return guarded([&] {
        const pkx::DecAttnParams p = cache_attn_params(c, a);
        if (p.B == 0 || p.n_q == 0) return;
        need_view(p.q, p.q_item, p.q_row, p.q_head, p.q_f32, "cache attention: q must be 16-byte aligned with strides of whole 16 bytes");
        need_view(p.out, p.o_item, p.o_row, p.o_head, p.q_f32, "cache attention: out must be 16-byte aligned with strides of whole 16 bytes");
        need_apart(p.o_item, p.B, p.o_row, p.n_q, p.o_head, a->n_heads, p.dk, "cache attention: rows of out overlap");
        need(p.k_len, "cache attention: null len");
        need(p.slot || p.table || p.B <= p.n_slots, "cache attention: more rows than slots");
        need(!p.table || p.table_ld >= p.n_k, "cache attention: table rows are shorter than max_len");
        need_device(st(s));
        pkx::launch_dec_attention(p, ws, ws_bytes, st(s));
    });
}

int pkx_beam_select_workspace(const pkx_beam_select_args* a, size_t* bytes) {
    return guarded([&] {
        need(bytes, "null argument");
        *bytes = pkx::beam_select_workspace(beam_params(a));
    });
}
int pkx_beam_select(const pkx_beam_select_args* a, void* ws, size_t ws_bytes, void* s) {
    return guarded([&] {
        const pkx::BeamSelectParams p = beam_params(a);
        if (p.B == 0) return;
        need(p.logits && p.scores && p.parent && p.token && p.new_scores, "beam select: null buffer");
        need((uintptr_t)p.logits % (p.f32 ? 4 : 2) == 0 && p.row >= 0, "beam select: misaligned logits or a negative row stride");
        need((uintptr_t)ws % 16 == 0, "beam select: the workspace must be 16-byte aligned");
        need_device(st(s));
        pkx::launch_beam_select(p, ws, ws_bytes, st(s));
    });
}
int pkx_beam_reorder(const int32_t* parent, int n_items, int n_beams, const pkx_beam_state* states, int n_states, void* s) {
    return guarded([&] {
        need(n_items >= 0 && n_beams >= 1, "beam reorder: bad size");
        need(n_states >= 0 && n_states <= pkx::kMaxBeamStates, "beam reorder: at most PKX_BEAM_MAX_STATES states");
        if (n_items == 0 || n_states == 0) return;
        need(parent && states, "null argument");
        need((double)n_items * n_beams < (double)(1 << 23), "beam reorder: too many rows for one call");
        pkx::BeamState p[pkx::kMaxBeamStates];
        const int64_t rows = (int64_t)n_items * n_beams;
        for (int i = 0; i < n_states; ++i) {
            const pkx_beam_state& x = states[i];
            need(x.bytes >= 0 && (x.src_row >= x.bytes || x.src_row == 0) && x.dst_row >= x.bytes,
                 "beam reorder: row strides must be at least the row's bytes");
            // (no span below wraps then, whichever state comes first)
            need((double)rows * (double)std::max({x.src_row, x.dst_row, x.bytes}) < 0x1p62, "beam reorder: rows past the address space");
        }
        for (int i = 0; i < n_states; ++i) {
            const pkx_beam_state& x = states[i];
            if (x.bytes > 0) {
                need(x.src && x.dst, "beam reorder: null state");
                const uintptr_t b = (uintptr_t)x.dst, be = b + (rows - 1) * x.dst_row + x.bytes;
                const uintptr_t pa = (uintptr_t)parent, pe = pa + rows * sizeof(int32_t);
                need(pe <= b || be <= pa, "beam reorder: parent overlaps a destination");
                for (int j = 0; j < n_states; ++j) {
                    const uintptr_t a = (uintptr_t)states[j].src, ae = a + (rows - 1) * states[j].src_row + states[j].bytes;
                    need(states[j].bytes <= 0 || ae <= b || be <= a, "beam reorder: a source overlaps a destination");
                }
            }
            p[i] = pkx::BeamState{(const uint8_t*)x.src, (uint8_t*)x.dst, x.src_row, x.dst_row, x.bytes};
        }
        need_device(st(s));
        pkx::launch_beam_reorder(parent, n_items, n_beams, p, n_states, st(s));
    });
}

int pkx_block_norm(const pkx_block_norm_args* a, void* s) {
    return guarded([&] {
        need(a, "null argument");
        pkx::BlockNormParams p;
        p.f32 = is_f32(a->type, "block norm: type must be PKX_TYPE_F32 or PKX_TYPE_F16");
        p.x_f32 = is_f32(a->x_type, "block norm: x_type must be PKX_TYPE_F32 or PKX_TYPE_F16");
        need(p.x_f32 || !p.f32, "block norm: an f16 x goes with f16 y, gate and h");
        need(a->n_rows >= 0 && a->n_rows < (1 << 22), "block norm: negative size, or 2^22 rows");
        need(a->d >= 1 && a->d <= PKX_NORM_MAX_WIDTH, "block norm: d must be 1 to PKX_NORM_MAX_WIDTH");
        for (int kind : {a->post, a->pre})
            need(kind == PKX_NORM_NONE || kind == PKX_NORM_LAYER || kind == PKX_NORM_RMS, "block norm: post and pre must be PKX_NORM_*");
        need(a->gate_fn == PKX_GATE_LINEAR || a->gate_fn == PKX_GATE_SIGMOID, "block norm: gate_fn must be PKX_GATE_*");
        need(a->post_eps >= 0 && a->pre_eps >= 0 && std::isfinite(a->post_eps) && std::isfinite(a->pre_eps),
             "block norm: eps must be finite and not negative");
        need(std::isfinite(a->alpha), "block norm: alpha is not finite");
        need(a->x || a->y, "block norm: neither x nor y");
        need(a->x_out || a->h, "block norm: neither x_out nor h");
        need(!a->gate || (a->y && a->rows_per_gate >= 1), "block norm: a gate needs y, and rows_per_gate of at least 1");
        need(a->post == PKX_NORM_NONE ? !a->post_w && !a->post_b : a->y != nullptr, "block norm: post without y, or weights without post");
        need(a->pre == PKX_NORM_NONE ? !a->pre_w && !a->pre_b : a->h != nullptr, "block norm: pre without h, or weights without pre");
        need(!a->h_i8 || (a->h && a->h_scale), "block norm: 8 bits without h or h_scale");
        if (a->n_rows == 0) return;
        const int e = p.f32 ? 4 : 2, ex = p.x_f32 ? 4 : 2, eh = a->h_i8 ? 1 : e;
        const int64_t rows = a->n_rows, d = a->d, gates = a->gate ? (rows - 1) / a->rows_per_gate + 1 : 0;
        if (a->x) need_rows_of(a->x, ex, a->x_row, rows, 0, "block norm: x is misaligned or of a negative stride");
        if (a->y) need_rows_of(a->y, e, a->y_row, rows, 0, "block norm: y is misaligned or of a negative stride");
        if (a->gate) need_rows_of(a->gate, e, a->gate_row, gates, 0, "block norm: gate is misaligned or of a negative stride");
        if (a->x_out) need_rows_of(a->x_out, ex, a->x_out_row, rows, d, "block norm: x_out is misaligned, or its rows overlap");
        if (a->h) need_rows_of(a->h, eh, a->h_row, rows, d, "block norm: h is misaligned, or its rows overlap");
        const Span none(nullptr, 0, {});
        const Span x = a->x ? rows_of(a->x, d, ex, a->x_row, rows) : none, y = a->y ? rows_of(a->y, d, e, a->y_row, rows) : none;
        const Span g = a->gate ? rows_of(a->gate, d, e, a->gate_row, gates) : none;
        const Span o = a->x_out ? rows_of(a->x_out, d, ex, a->x_out_row, rows) : none;
        const Span h = a->h ? rows_of(a->h, d, eh, a->h_row, rows) : none;
        const Span hs = a->h_i8 ? rows_of(a->h_scale, 1, 4, 1, rows) : none;
        for (const Span* w : {&o, &h, &hs}) {
            if (!w->at) continue;
            for (const Span* in : {&x, &y, &g})
                need(!in->at || apart(*w, *in) || (w == &o && in == &x && same(o, x)) || (w == &h && in == &y && same(h, y) && !a->h_i8),
                     "block norm: an output overlaps an input");
            for (const float* v : {a->post_w, a->post_b, a->pre_w, a->pre_b})
                need(!v || apart(*w, Span(v, 4 * d, {})), "block norm: an output overlaps a weight");
            for (const Span* w2 : {&o, &h, &hs}) need(w == w2 || !w2->at || apart(*w, *w2), "block norm: the outputs overlap");
        }
        p.h_i8 = a->h_i8 != 0;
        p.rows = rows;
        p.d = a->d;
        p.x = a->x; p.x_row = a->x_row;
        p.y = a->y; p.y_row = a->y_row;
        p.gate = a->gate; p.gate_row = a->gate_row;
        p.rows_per_gate = a->gate && a->rows_per_gate < rows ? (int)a->rows_per_gate : (int)rows;
        p.sigmoid = a->gate_fn == PKX_GATE_SIGMOID;
        p.post = a->post;
        p.pre = a->pre;
        p.post_w = a->post_w; p.post_b = a->post_b; p.post_eps = a->post_eps;
        p.pre_w = a->pre_w; p.pre_b = a->pre_b; p.pre_eps = a->pre_eps;
        p.alpha = a->alpha;
        p.x_out = a->x_out; p.x_out_row = a->x_out_row;
        p.h = a->h; p.h_row = a->h_row;
        p.h_scale = a->h_scale;
        need_device(st(s));
        pkx::launch_block_norm(p, st(s));
    });
}

int pkx_quantize_rows(int type, const void* x, int64_t x_row, int64_t n_rows, int n, int8_t* q, int64_t q_row, float* scale, void* s) {
    return guarded([&] {
        pkx::QuantizeRowsParams p = quantize_rows_params(type, x, x_row, n_rows, n);
        if (n_rows == 0) return;
        need_rows_of(q, 1, q_row, n_rows, n, "quantise rows: q is null, or its rows overlap");
        need(scale && (uintptr_t)scale % 4 == 0, "quantise rows: scale is null or misaligned");
        const Span in = rows_of(x, n, p.f32 ? 4 : 2, x_row, n_rows), out = rows_of(q, n, 1, q_row, n_rows), sc = rows_of(scale, 1, 4, 1, n_rows);
        need(apart(in, out) && apart(in, sc) && apart(out, sc), "quantise rows: an output overlaps x or the other one");
        p.q = q;
        p.q_row = q_row;
        p.scale = scale;
        need_device(st(s));
        pkx::launch_quantize_rows(p, st(s));
    });
}

int pkx_i8_weight_bytes(int n_out, int n_in, size_t* bytes) {
    return guarded([&] {
        need(bytes, "null argument");
        need_i8_weight(n_out, n_in);
        *bytes = (size_t)pkx::i8_weight_bytes(n_out, n_in);
    });
}
int pkx_i8_weight_pack(const int8_t* w, int64_t w_row, int n_out, int n_in, void* packed, void* s) {
    return guarded([&] {
        need_i8_weight(n_out, n_in);
        if (n_out == 0) return;
        need_rows_of(w, 1, w_row, n_out, 0, "8-bit weights: w is null or of a negative stride");
        need(packed && (uintptr_t)packed % 16 == 0, "8-bit weights: packed is null or not 16-byte aligned");
        need(apart(rows_of(w, n_in, 1, w_row, n_out), Span(packed, pkx::i8_weight_bytes(n_out, n_in), {})), "8-bit weights: packed overlaps w");
        need_device(st(s));
        pkx::launch_i8_weight_pack(w, w_row, n_out, n_in, packed, st(s));
    });
}

int pkx_linear_i8_workspace(const pkx_linear_i8_args* a, size_t* bytes) {
    return guarded([&] {
        need(bytes, "null argument");
        linear_i8_params(a);
        *bytes = i8_workspace(a);
    });
}
int pkx_linear_i8_tile(const pkx_linear_i8_args* a, int* tokens, int* channels, int64_t* workgroups) {
    return guarded([&] {
        need(tokens && channels && workgroups, "null argument");
        const pkx::LinearI8Params p = linear_i8_params(a);
        const pkx::LinearI8Tile t = pkx::linear_i8_tile(p.M, p.N, p.K, a->x_type == PKX_TYPE_I8);
        *tokens = t.tokens;
        *channels = t.channels;
        *workgroups = t.workgroups;
    });
}
int pkx_linear_i8(const pkx_linear_i8_args* a, void* ws, size_t ws_bytes, void* s) {
    return guarded([&] {
        pkx::LinearI8Params p = linear_i8_params(a);
        if (p.M == 0 || p.N == 0) return;
        const int e = p.y_f32 ? 4 : 2;
        const int64_t M = p.M, N = p.N, K = p.K;
        need(p.w && (uintptr_t)p.w % 16 == 0, "8-bit linear: w is null or not 16-byte aligned");
        need(p.w_scale && (uintptr_t)p.w_scale % 4 == 0 && (uintptr_t)p.bias % 4 == 0, "8-bit linear: w_scale is null, or it or bias misaligned");
        need_rows_of(p.y, e, p.y_row, M, N, "8-bit linear: y is null or misaligned, or its rows overlap");
        if (p.add) need_rows_of(p.add, e, p.add_row, M, 0, "8-bit linear: add is misaligned or of a negative stride");
        const Span y = rows_of(p.y, N, e, p.y_row, M);
        if (p.add) {
            const Span add = rows_of(p.add, N, e, p.add_row, M);
            need(apart(y, add) || same(y, add), "8-bit linear: y overlaps add without being it");
        }
        need(apart(y, Span(p.w, pkx::i8_weight_bytes(N, K), {})) && apart(y, Span(p.w_scale, 4 * N, {})) &&
                 (!p.bias || apart(y, Span(p.bias, 4 * N, {}))), "8-bit linear: y overlaps the weights, their scales or the bias");
        if (a->x_type == PKX_TYPE_I8) {
            need_rows_of(a->x, 16, a->x_row, M, K, "8-bit linear: x is null, not 16-byte aligned or of rows shorter than n_in");
            need(a->x_row % 16 == 0 && a->x_row >= K && a->x_row < (1 << 22), "8-bit linear: x_row must be a multiple of 16, at least n_in and below 2^22");
            need(a->x_scale && (uintptr_t)a->x_scale % 4 == 0, "8-bit linear: x_scale is null or misaligned");
            need(apart(y, rows_of(a->x, i8_row(a), 1, a->x_row, M)) && apart(y, Span(a->x_scale, 4 * M, {})), "8-bit linear: y overlaps x or its scales");
            p.x = (const int8_t*)a->x;
            p.x_row = a->x_row;
            p.x_scale = a->x_scale;
            need_device(st(s));
            pkx::launch_linear_i8(p, st(s));
            return;
        }
        need(!a->x_scale, "8-bit linear: x_scale goes with PKX_TYPE_I8");
        pkx::QuantizeRowsParams q = quantize_rows_params(a->x_type, a->x, a->x_row, M, a->n_in);
        need(apart(y, rows_of(a->x, K, q.f32 ? 4 : 2, a->x_row, M)), "8-bit linear: y overlaps x");
        if (pkx::linear_i8_fused(p.M, p.N, p.K)) {
            need_device(st(s));
            pkx::launch_linear_i8_fused(p, q, st(s));
            return;
        }
        need(ws && (uintptr_t)ws % 16 == 0, "8-bit linear: the workspace is null or not 16-byte aligned");
        need(ws_bytes >= i8_workspace(a), "8-bit linear: the workspace is too small");
        q.q = (int8_t*)ws;
        q.q_row = i8_row(a);
        q.scale = (float*)((char*)ws + M * q.q_row);
        p.x = q.q;
        p.x_row = q.q_row;
        p.x_scale = q.scale;
        need_device(st(s));
        pkx::launch_quantize_rows(q, st(s));
        pkx::launch_linear_i8(p, st(s));
    });
}

int pkx_rotary(const pkx_rotary_args* a, void* s) {
    return guarded([&] {
        need(a, "null argument");
        pkx::RotaryParams p;
        p.f32 = is_f32(a->type, "rotary: type must be PKX_TYPE_F32 or PKX_TYPE_F16");
        need(a->n_rows >= 0 && a->n_tok >= 0, "rotary: negative size");
        need(a->d_head >= 1 && a->d_head <= pkx::kMaxRotaryWidth, "rotary: d_head must be 1 to 512");
        need(a->rot >= 0 && a->rot % 2 == 0 && a->rot <= a->d_head, "rotary: rot must be even and at most d_head");
        need(a->n_parts >= 0 && a->n_parts <= PKX_ROTARY_MAX_PARTS, "rotary: at most PKX_ROTARY_MAX_PARTS parts");
        need(std::isfinite(a->mult), "rotary: mult is not finite");
        need(!a->pos || a->pos_row >= 0, "rotary: negative stride of pos");
        for (int i = 0; i < a->n_parts; ++i) need(a->part[i].n_heads >= 0 && a->part[i].n_heads <= 4096, "rotary: a part has 0 to 4096 heads");
        if (a->n_rows == 0 || a->n_tok == 0) return;
        need(a->freq && (uintptr_t)a->freq % 8 == 0, "rotary: freq is null or misaligned");
        const int e = p.f32 ? 4 : 2;
        const int64_t R = a->n_rows, n = a->n_tok;
        std::vector<Span> src, dst;
        for (int i = 0; i < a->n_parts; ++i) {
            const pkx_rotary_part& x = a->part[i];
            if (x.n_heads == 0) continue;
            need(x.src && x.dst && ((uintptr_t)x.src | (uintptr_t)x.dst) % e == 0, "rotary: a part's src or dst is null or misaligned");
            need(x.src_row >= 0 && x.src_tok >= 0 && x.src_head >= 0 && x.dst_row >= 0 && x.dst_tok >= 0 && x.dst_head >= 0, "rotary: negative stride");
            need_apart(x.dst_row, R, x.dst_tok, n, x.dst_head, x.n_heads, a->d_head, "rotary: rows of a dst overlap");
            src.emplace_back(x.src, (int64_t)a->d_head * e, std::initializer_list<std::pair<int64_t, int64_t>>{{x.src_row * e, R}, {x.src_tok * e, n}, {x.src_head * e, x.n_heads}});
            dst.emplace_back(x.dst, (int64_t)a->d_head * e, std::initializer_list<std::pair<int64_t, int64_t>>{{x.dst_row * e, R}, {x.dst_tok * e, n}, {x.dst_head * e, x.n_heads}});
            need(src.back().bytes() < 0x1p62 && dst.back().bytes() < 0x1p62, "rotary: strides past the address space");
            pkx::RotaryPart& o = p.part[p.parts++];
            o = pkx::RotaryPart{x.src, x.src_row, x.src_tok, x.src_head, x.dst, x.dst_row, x.dst_tok, x.dst_head, x.n_heads};
        }
        for (size_t i = 0; i < dst.size(); ++i) {
            for (size_t j = 0; j < dst.size(); ++j) {
                need(apart(dst[i], src[j]) || (i == j && in_place(p.part[i], R, n)), "rotary: a dst overlaps a src without being its own");
                need(i == j || apart(dst[i], dst[j]), "rotary: two dsts overlap");
            }
            need(a->rot == 0 || apart(dst[i], Span(a->freq, 4 * (int64_t)a->rot, {})), "rotary: a dst overlaps freq");
            need((!a->start || apart(dst[i], Span(a->start, 4 * R, {}))) && (!a->count || apart(dst[i], Span(a->count, 4 * R, {}))) &&
                     (!a->pos || apart(dst[i], rows_of(a->pos, n, 4, a->pos_row, R))), "rotary: a dst overlaps start, pos or count");
        }
        p.R = a->n_rows;
        p.n = a->n_tok;
        p.dk = a->d_head;
        p.rot = a->rot;
        p.interleaved = a->interleaved != 0;
        p.mult = a->mult;
        p.freq = a->freq;
        p.start = a->start;
        p.pos = a->pos;
        p.pos_row = a->pos_row;
        p.count = a->count;
        need_device(st(s));
        pkx::launch_rotary(p, st(s));
    });
}
int pkx_rotary_frequencies(double base, int rot, double factor, double context, double low, double high, double* freq) {
    return guarded([&] {
        need(freq, "null argument");
        need(rot >= 0 && rot % 2 == 0 && rot <= pkx::kMaxRotaryWidth, "rotary: rot must be even and at most 512");
        need(base > 0 && std::isfinite(base) && factor > 0 && std::isfinite(factor), "rotary: base and factor must be positive and finite");
        need(context >= 0 && std::isfinite(context) && (context == 0 || (high > low && std::isfinite(high - low))), "rotary: context must not be negative, and high above low");
        for (int j = 0; j < rot / 2; ++j) {
            const double f = std::pow(base, -2.0 * j / rot);
            double keep = 0;
            if (context > 0) keep = std::min(1.0, std::max(0.0, (context * f / (2 * M_PI) - low) / (high - low)));
            freq[j] = f * (keep + (1 - keep) / factor);
        }
    });
}

int pkx_logit_rules(const pkx_logit_rules_args* a, void* s) {
    return guarded([&] {
        need(a, "null argument");
        pkx::LogitRulesParams p;
        p.f32 = is_f32(a->type, "logit rules: type must be PKX_TYPE_F32 or PKX_TYPE_F16");
        need(a->n_rows >= 0 && a->vocab >= 0 && a->window >= 0, "logit rules: negative size");
        need(a->vocab <= (1 << 22), "logit rules: a vocabulary of at most 2^22 words");
        if (a->n_rows == 0 || a->vocab == 0) return;
        const int e = p.f32 ? 4 : 2;
        const int64_t R = a->n_rows, V = a->vocab;
        need_rows_of(a->logits, e, a->logits_row, R, 0, "logit rules: logits are null, misaligned or of a negative stride");
        need_rows_of(a->out, e, a->out_row, R, V, "logit rules: out is null or misaligned, or its rows overlap");
        const Span in = rows_of(a->logits, V, e, a->logits_row, R), out = rows_of(a->out, V, e, a->out_row, R);
        need(same(in, out) || apart(in, out), "logit rules: out overlaps logits without being them");
        if (a->tokens) {
            need(a->n_slots >= 1 && a->capacity >= 0 && a->capacity <= (1 << 30), "logit rules: no slots, or a capacity that is negative or above 2^30");
            need((double)a->n_slots * a->capacity < 0x1p60 && a->table_row >= 0 && (double)a->table_row * R < 0x1p60, "logit rules: tokens or table past the address space");
            need(a->len, "logit rules: null len");
            need(a->slot || a->table || R <= a->n_slots, "logit rules: more rows than slots");
            need(!a->table || a->table_row >= a->capacity, "logit rules: table rows are shorter than the capacity");
            need(apart(out, Span(a->tokens, 4 * (int64_t)a->n_slots * a->capacity, {})) && apart(out, Span(a->len, 4 * R, {})) &&
                     (!a->slot || apart(out, Span(a->slot, 4 * R, {}))) && (!a->table || apart(out, rows_of(a->table, a->capacity, 4, a->table_row, R))),
                 "logit rules: out overlaps the tokens, their lengths, slots or table");
            p.tokens = a->tokens;
            p.n_slots = a->n_slots;
            p.cap = a->capacity;
            p.len = a->len;
            p.slot = a->slot;
            p.table = a->table;
            p.table_row = a->table_row;
            p.window = a->window;
            p.repetition = a->repetition;
            p.presence = a->presence;
            p.frequency = a->frequency;
            for (const float* v : {a->repetition, a->presence, a->frequency})
                need(!v || apart(out, Span(v, 4 * R, {})), "logit rules: out overlaps a penalty");
        }
        if (a->bias) {
            need(a->n_bias >= 0 && (uintptr_t)a->bias % 4 == 0 && a->bias_row >= 0 && (double)a->bias_row * a->n_bias < 0x1p60, "logit rules: bias is misaligned, or of a negative count or stride");
            need(a->n_bias == 0 || apart(out, rows_of(a->bias, V, 4, a->bias_row, a->n_bias)), "logit rules: out overlaps bias");
            need(!a->bias_index || apart(out, Span(a->bias_index, 4 * R, {})), "logit rules: out overlaps bias_index");
            p.bias = a->bias;
            p.bias_row = a->bias_row;
            p.n_bias = a->n_bias;
            p.bias_index = a->bias_index;
        }
        if (a->mask) {
            need(a->n_mask >= 0 && (uintptr_t)a->mask % 4 == 0 && a->mask_row >= 0 && (double)a->mask_row * a->n_mask < 0x1p60, "logit rules: mask is misaligned, or of a negative count or stride");
            need(a->n_mask == 0 || apart(out, rows_of(a->mask, (V + 31) / 32, 4, a->mask_row, a->n_mask)), "logit rules: out overlaps mask");
            need(!a->mask_index || apart(out, Span(a->mask_index, 4 * R, {})), "logit rules: out overlaps mask_index");
            p.mask = a->mask;
            p.mask_row = a->mask_row;
            p.n_mask = a->n_mask;
            p.mask_index = a->mask_index;
        }
        p.R = a->n_rows;
        p.V = a->vocab;
        p.x = a->logits;
        p.x_row = a->logits_row;
        p.out = a->out;
        p.out_row = a->out_row;
        need_device(st(s));
        pkx::launch_logit_rules(p, st(s));
    });
}

}  // extern "C"
