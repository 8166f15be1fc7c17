// C entries of the operators on a caller's own device memory
// (include/mtb_decoder.h): argument checks, the device of the memory, launch.
#include "../../include/mtb_decoder.h"
#include "ops.hpp"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <string>

using namespace mtb;

extern "C" __attribute__((visibility("hidden"))) void mtb_set_global_error(const char* text);

namespace {

static_assert(int(MTB_T_F32) == OP_F32 && int(MTB_T_F16) == OP_F16 && int(MTB_T_BF16) == OP_BF16, "one set of type codes");
static_assert(int(MTB_BAD_PAGE) == BAD_PAGE && int(MTB_BAD_LEN) == BAD_LEN && int(MTB_BAD_TOKENS) == BAD_TOKENS && int(MTB_BAD_WAIT) == BAD_WAIT,
              "one set of bits");
static_assert((long long)MTB_ATTENTION_WORKSPACE == kAttnWorkspace, "the header's size is the kernels'");

std::atomic<int> g_stall{0};  // calls that are to stall (mtb_debug_stall_attention)

int fail(int code, const std::string& text) {
    mtb_set_global_error(text.c_str());
    return code;
}

// An exception (a string that finds no memory) ends at the C boundary.
template <class F>
int guarded(F&& f) {
    try {
        return f();
    } catch (...) {
        mtb_set_global_error("unknown error");
        return -1;
    }
}

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
template <class... P>
bool words(const P*... p) { return (aligned(p, 4) && ...); }

// Makes the device that owns `p` current; the caller's comes back at the end.
struct OnDevice {
    int saved = -1, device = -1;
    int enter(const char* what, const void* p) {
        cudaPointerAttributes at{};
        const cudaError_t e = cudaPointerGetAttributes(&at, p);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return fail(-1, std::string(what) + ": " + cudaGetErrorString(e));
        }
        if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
            return fail(-1, std::string(what) + ": not device memory");
        device = at.device;
        if (cudaGetDevice(&saved) != cudaSuccess) saved = -1;
        if (saved != device && cudaSetDevice(device) != cudaSuccess) return fail(-1, "cudaSetDevice failed");
        return 0;
    }
    ~OnDevice() {
        if (saved >= 0 && saved != device && device >= 0) cudaSetDevice(saved);
    }
};

int launched(const char* what, cudaError_t e) {
    if (e == cudaSuccess) return 0;
    return fail(-1, std::string(what) + ": " + cudaGetErrorString(e));
}

// The view, checked: 0, or the error's code.
int view_of(const char* what, const mtb_paged_cache* c, PagedView* out) {
    const std::string w(what);
    if (!c) return fail(-1, w + ": null cache");
    if (c->n_seq < 0) return fail(-2, w + ": n_seq must not be negative");
    if (c->n_seq > 0 && (!c->k || !c->v || !c->page_table || !c->kv_len)) return fail(-1, w + ": null pointer in the cache");
    if (c->type != MTB_T_F16 && c->type != MTB_T_BF16) return fail(-2, w + ": the cache's type is f16 or bf16");
    if (c->head_dim != 64 && c->head_dim != 128) return fail(-2, w + ": head_dim must be 64 or 128");
    if (c->n_kv_heads < 1 || c->n_kv_heads > 65535) return fail(-2, w + ": n_kv_heads must be in [1, 65535]");
    if (c->n_pages < 1 || c->table_stride < 1) return fail(-2, w + ": n_pages and table_stride must be positive");
    if (c->table_stride > (1 << 24)) return fail(-2, w + ": table_stride must be at most 2^24 (positions are int32)");
    if (c->n_seq > 65535) return fail(-2, w + ": n_seq must be at most 65535");
    if (int64_t(c->n_seq) * c->n_kv_heads > (1 << 24)) return fail(-2, w + ": n_seq * n_kv_heads must be at most 2^24");
    if (!aligned(c->k, 16) || !aligned(c->v, 16)) return fail(-2, w + ": k and v must be 16-byte aligned");
    if (!words(c->page_table, c->kv_len, c->position, c->weight, c->status)) return fail(-2, w + ": a pointer is not aligned to its elements");
    const int64_t block = int64_t(kPage) * c->head_dim;
    if (c->head_stride % 8 || c->page_stride % 8 || c->head_stride < block || c->page_stride < block)
        return fail(-2, w + ": the cache's strides must be multiples of 8 elements that hold a page's rows");
    // Tensor maps take strides below 2^40 bytes.
    if (c->head_stride >= (1ll << 38) || c->page_stride >= (1ll << 38)) return fail(-2, w + ": a cache stride is too large");
    *out = PagedView{static_cast<char*>(c->k), static_cast<char*>(c->v), c->type, c->head_dim, c->n_kv_heads, c->n_pages,
                     c->page_stride, c->head_stride, c->page_table, c->table_stride, c->n_seq, c->kv_len, c->position,
                     c->weight, c->status};
    return 0;
}

int heads_of(const std::string& w, int n_heads, int n_kv) {
    if (n_heads < 1 || n_heads % n_kv) return fail(-2, w + ": n_heads must be a multiple of n_kv_heads");
    if (n_heads / n_kv > kMaxGroup) return fail(-2, w + ": at most 64 query heads for each KV head");
    return 0;
}

int attention_args(const char* what, const mtb_paged_cache* cache, const int32_t* cu, int n_tokens, int max_tokens,
                   const void* q, int64_t q_stride, int n_heads, float scale, AttnArgs* a) {
    const std::string w(what);
    if (const int rc = view_of(what, cache, &a->c)) return rc;
    if (n_tokens < 0) return fail(-2, w + ": n_tokens must not be negative");
    if (const int rc = heads_of(w, n_heads, cache->n_kv_heads)) return rc;
    // Rows and their tiles are counted in int32.
    if (int64_t(n_tokens) * (n_heads / cache->n_kv_heads) > (1 << 30)) return fail(-2, w + ": n_tokens * n_heads / n_kv_heads must be at most 2^30");
    if (n_tokens == 0 || cache->n_seq == 0) return 0;
    if (!cu || !q) return fail(-1, w + ": null pointer");
    if (!aligned(q, 16) || q_stride % 8 || q_stride < int64_t(n_heads) * cache->head_dim || q_stride >= (1ll << 38))
        return fail(-2, w + ": q must be 16-byte aligned, its stride a multiple of 8 elements that holds a token's rows");
    if (!words(cu)) return fail(-2, w + ": a pointer is not aligned to its elements");
    if (!std::isfinite(scale)) return fail(-2, w + ": scale must be finite");
    a->cu = cu;
    a->n_tokens = n_tokens;
    a->max_tokens = max_tokens <= 0 || max_tokens > n_tokens ? n_tokens : max_tokens;
    a->q = static_cast<const char*>(q);
    a->q_stride = q_stride;
    a->n_heads = n_heads;
    a->scale = scale;
    a->G = n_heads / cache->n_kv_heads;
    a->by_G = FastDiv::of(a->G);
    for (int left = g_stall.load(); left > 0;)
        if (g_stall.compare_exchange_weak(left, left - 1)) a->c.n_seq = left = 0;
    return 0;
}

}  // namespace

extern "C" {

int mtb_rope_frequencies(int rotary_dim, double base, int kind, double factor, double original_len, double fast,
                         double slow, double* inv_freq, float* out_factor) {
    return guarded([&]() -> int {
        if (rotary_dim < 0 || rotary_dim % 2 || rotary_dim > 128) return fail(-2, "rope_frequencies: rotary_dim must be even, in [0, 128]");
        if ((rotary_dim && !inv_freq) || !out_factor) return fail(-1, "rope_frequencies: null argument");
        if (!(base > 0) || !std::isfinite(base)) return fail(-2, "rope_frequencies: base must be positive");
        if (kind < MTB_ROPE_PLAIN || kind > MTB_ROPE_BANDS) return fail(-2, "rope_frequencies: unknown scaling");
        const bool blend = kind == MTB_ROPE_YARN || kind == MTB_ROPE_BANDS;
        if (kind != MTB_ROPE_PLAIN && (!(factor >= 1) || !std::isfinite(factor)))
            return fail(-2, "rope_frequencies: factor must be at least 1");
        if (blend && (!(original_len > 0) || !(slow > 0) || !(fast > slow) || !std::isfinite(original_len) || !std::isfinite(fast)))
            return fail(-2, "rope_frequencies: original_len > 0 and fast > slow > 0 are wanted");
        if (kind == MTB_ROPE_YARN && !(base > 1)) return fail(-2, "rope_frequencies: base must be above 1");
        const int half = rotary_dim / 2;
        const double pi2 = 6.283185307179586476925;
        if (kind == MTB_ROPE_NTK && rotary_dim > 2) base *= std::pow(factor, double(rotary_dim) / (rotary_dim - 2));
        // The pair index at which a pair turns `t` times over original_len.
        auto pair_at = [&](double t) { return rotary_dim * std::log(original_len / (t * pi2)) / (2 * std::log(base)); };
        double low = 0, high = 0;
        if (kind == MTB_ROPE_YARN) {
            low = std::max(std::floor(pair_at(fast)), 0.0);
            high = std::min(std::ceil(pair_at(slow)), rotary_dim - 1.0);
            if (high <= low) high = low + 0.001;
        }
        for (int j = 0; j < half; ++j) {
            const double f = std::pow(base, -2.0 * j / rotary_dim);
            double keep = 1;  // share of the plain frequency
            if (kind == MTB_ROPE_LINEAR) keep = 0;
            if (kind == MTB_ROPE_YARN) keep = 1 - std::min(std::max((j - low) / (high - low), 0.0), 1.0);
            if (kind == MTB_ROPE_BANDS) keep = std::min(std::max((original_len * f / pi2 - slow) / (fast - slow), 0.0), 1.0);
            inv_freq[j] = kind == MTB_ROPE_PLAIN || kind == MTB_ROPE_NTK ? f : f * keep + f / factor * (1 - keep);
        }
        *out_factor = kind == MTB_ROPE_YARN ? float(0.1 * std::log(factor) + 1.0) : 1.0f;
        return 0;
    });
}

int mtb_rope_append(const mtb_paged_cache* cache, const int32_t* cu_tokens, int n_tokens, const int32_t* positions,
                    int in_type, const void* q, int64_t q_stride, int n_heads, const void* k, int64_t k_stride,
                    const void* v, int64_t v_stride, const double* inv_freq, int rotary_dim, int interleaved,
                    float factor, void* q_out, int64_t q_out_stride, void* stream) {
    return guarded([&]() -> int {
        const std::string w("rope_append");
        RopeArgs a{};
        if (const int rc = view_of("rope_append", cache, &a.c)) return rc;
        if (n_tokens < 0) return fail(-2, w + ": n_tokens must not be negative");
        if (n_heads < 1 || n_heads > 65535) return fail(-2, w + ": n_heads must be in [1, 65535]");
        if (in_type != MTB_T_F32 && in_type != cache->type) return fail(-2, w + ": q, k and v are f32 or of the cache's type");
        const int D = cache->head_dim;
        if (rotary_dim < 0 || rotary_dim > D || rotary_dim % 2) return fail(-2, w + ": rotary_dim must be even, in [0, head_dim]");
        if (q_stride < int64_t(n_heads) * D || q_out_stride < int64_t(n_heads) * D || k_stride < int64_t(cache->n_kv_heads) * D ||
            v_stride < int64_t(cache->n_kv_heads) * D)
            return fail(-2, w + ": a stride is shorter than a token's rows");
        if (n_tokens == 0 || cache->n_seq == 0) return 0;
        if (!cu_tokens || !positions || !q || !k || !v || !q_out || (rotary_dim && !inv_freq)) return fail(-1, w + ": null pointer");
        const size_t in_size = in_type == MTB_T_F32 ? 4 : 2;
        if (!aligned(q, in_size) || !aligned(k, in_size) || !aligned(v, in_size) || !aligned(q_out, 2) || !aligned(inv_freq, 8) ||
            !words(cu_tokens, positions))
            return fail(-2, w + ": a pointer is not aligned to its elements");
        if (q == q_out && (in_type != cache->type || q_stride != q_out_stride))
            return fail(-2, w + ": q_out may be q only in the same type, with the same stride");
        a.cu = cu_tokens;
        a.n_tokens = n_tokens;
        a.positions = positions;
        a.in_type = in_type;
        a.q = static_cast<const char*>(q);
        a.k = static_cast<const char*>(k);
        a.v = static_cast<const char*>(v);
        a.q_stride = q_stride;
        a.k_stride = k_stride;
        a.v_stride = v_stride;
        a.out_stride = q_out_stride;
        a.n_heads = n_heads;
        a.inv_freq = inv_freq;
        a.rotary = rotary_dim;
        a.interleaved = interleaved != 0;
        a.factor = factor;
        a.out = static_cast<char*>(q_out);
        OnDevice on;
        if (const int rc = on.enter("rope_append", cache->k)) return rc;
        return launched("rope_append", launch_rope_append(a, static_cast<cudaStream_t>(stream)));
    });
}

int mtb_paged_attention(const mtb_paged_cache* cache, const int32_t* cu_tokens, int n_tokens, int max_tokens,
                        const void* q, int64_t q_stride, int n_heads, float scale, void* out, int64_t out_stride,
                        float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        const std::string w("paged_attention");
        AttnArgs a{};
        if (const int rc = attention_args("paged_attention", cache, cu_tokens, n_tokens, max_tokens, q, q_stride, n_heads, scale, &a)) return rc;
        if (n_tokens == 0 || cache->n_seq == 0) return 0;
        if (!out || !workspace) return fail(-1, w + ": null pointer");
        if (!aligned(out, 16) || out_stride % 8 || out_stride < int64_t(n_heads) * cache->head_dim)
            return fail(-2, w + ": out must be 16-byte aligned, its stride a multiple of 8 elements that holds a token's rows");
        if (!words(lse)) return fail(-2, w + ": a pointer is not aligned to its elements");
        if (workspace_bytes < size_t(kAttnWorkspace) || !aligned(workspace, 256))
            return fail(-2, w + ": the workspace must have MTB_ATTENTION_WORKSPACE bytes, 256-byte aligned");
        a.out = static_cast<char*>(out);
        a.out_stride = out_stride;
        a.lse = lse;
        a.workspace = static_cast<char*>(workspace);
        OnDevice on;
        if (const int rc = on.enter("paged_attention", cache->k)) return rc;
        return launched("paged_attention", launch_paged_attention(a, static_cast<cudaStream_t>(stream)));
    });
}

int mtb_attention_weights(const mtb_paged_cache* cache, const int32_t* cu_tokens, int n_tokens, int max_tokens,
                          const void* q, int64_t q_stride, int n_heads, float scale, const float* lse, float decay,
                          void* stream) {
    return guarded([&]() -> int {
        const std::string w("attention_weights");
        AttnArgs a{};
        if (const int rc = attention_args("attention_weights", cache, cu_tokens, n_tokens, max_tokens, q, q_stride, n_heads, scale, &a)) return rc;
        if (n_tokens == 0 || cache->n_seq == 0) return 0;
        if (!lse || !cache->weight) return fail(-1, w + ": null pointer (lse and the cache's weight are needed)");
        if (!words(lse)) return fail(-2, w + ": a pointer is not aligned to its elements");
        if (!std::isfinite(decay)) return fail(-2, w + ": decay must be finite");
        a.lse = const_cast<float*>(lse);
        a.decay = decay;
        OnDevice on;
        if (const int rc = on.enter("attention_weights", cache->k)) return rc;
        return launched("attention_weights", launch_attention_weights(a, static_cast<cudaStream_t>(stream)));
    });
}

void mtb_debug_stall_attention(int n) { g_stall.store(n > 0 ? n : 0); }

int64_t mtb_cache_evict_workspace(int n_seq, int n_kv_heads, int table_stride) {
    if (n_seq < 0 || n_seq > 65535 || n_kv_heads < 1 || n_kv_heads > 65535 || int64_t(n_seq) * n_kv_heads > (1 << 24) || table_stride < 1 ||
        table_stride > (1 << 24))
        return -2;
    return evict_workspace(n_seq, n_kv_heads, table_stride);
}

int mtb_cache_evict(const mtb_paged_cache* cache, int keep, int sinks, int recent, int32_t* new_len, void* workspace,
                    size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        const std::string w("cache_evict");
        EvictArgs a{};
        if (const int rc = view_of("cache_evict", cache, &a.c)) return rc;
        if (keep < 0 || sinks < 0 || recent < 0 || int64_t(sinks) + recent > keep)
            return fail(-2, w + ": sinks + recent must be in [0, keep]");
        if (cache->n_pages > (1 << 25)) return fail(-2, w + ": n_pages must be at most 2^25 (rows of the pool are counted in int32)");
        if (cache->n_seq == 0) return 0;
        if (!cache->position || !cache->weight || !new_len || !workspace)
            return fail(-1, w + ": null pointer (the cache's position and weight are needed)");
        if (!words(new_len)) return fail(-2, w + ": a pointer is not aligned to its elements");
        if (int64_t(workspace_bytes) < evict_workspace(cache->n_seq, cache->n_kv_heads, cache->table_stride) || !aligned(workspace, 16))
            return fail(-2, w + ": the workspace must have mtb_cache_evict_workspace bytes, 16-byte aligned");
        a.keep = keep;
        a.sinks = sinks;
        a.recent = recent;
        a.new_len = new_len;
        a.workspace = static_cast<char*>(workspace);
        OnDevice on;
        if (const int rc = on.enter("cache_evict", cache->k)) return rc;
        return launched("cache_evict", launch_cache_evict(a, static_cast<cudaStream_t>(stream)));
    });
}

int mtb_logits_process(const void* logits, int type, int rows, int vocab, int64_t stride,
                       const mtb_logits_params* params, void* out, int64_t out_stride, int32_t* choice, void* stream) {
    return guarded([&]() -> int {
        const std::string w("logits_process");
        if (type != MTB_T_F32 && type != MTB_T_F16 && type != MTB_T_BF16) return fail(-2, w + ": unknown type");
        // Ids and places in the lists are counted in int32, with steps beyond the end.
        if (rows < 0 || vocab < 1 || vocab > (1 << 30)) return fail(-2, w + ": rows must not be negative, vocab in [1, 2^30]");
        if (stride < vocab || (out && out_stride < vocab)) return fail(-2, w + ": a stride is shorter than a row");
        if (!out && !choice) return fail(-1, w + ": out and choice are both null");
        const mtb_logits_params none{};
        const mtb_logits_params& p = params ? *params : none;
        const bool penal = p.repetition || p.presence || p.frequency;
        if (penal && (!p.history || !p.history_begin || !p.history_end)) return fail(-1, w + ": penalties need the history and its bounds");
        if ((p.bias_ids || p.bias_values) && (!p.bias_ids || !p.bias_values || !p.bias_begin || !p.bias_end))
            return fail(-1, w + ": biases need ids, values and bounds");
        if (p.mask && p.mask_stride < (vocab + 31) / 32) return fail(-2, w + ": mask_stride is shorter than a mask row");
        if (p.history_len < 0 || p.bias_len < 0 || p.mask_rows < 0) return fail(-2, w + ": a length must not be negative");
        if (p.history_len > (1 << 30) || p.bias_len > (1 << 30)) return fail(-2, w + ": a list has at most 2^30 entries");
        if (rows > (1 << 26)) return fail(-2, w + ": rows must be at most 2^26");
        if (rows == 0) return 0;
        if (!logits) return fail(-1, w + ": null pointer");
        const size_t size = type == MTB_T_F32 ? 4 : 2;
        if (!aligned(logits, size) || (out && !aligned(out, size)) ||
            !words(choice, p.history, p.history_begin, p.history_end, p.repetition, p.presence, p.frequency, p.bias_ids, p.bias_values, p.bias_begin,
                   p.bias_end, p.mask, p.mask_row))
            return fail(-2, w + ": a pointer is not aligned to its elements");
        if (out == logits && stride != out_stride) return fail(-2, w + ": in place, both strides are the same");
        LogitsArgs a{};
        a.x = static_cast<const char*>(logits);
        a.y = static_cast<char*>(out);
        a.type = type;
        a.rows = rows;
        a.vocab = vocab;
        a.x_stride = stride;
        a.y_stride = out_stride;
        if (penal) {
            a.hist = p.history;
            a.hist_begin = p.history_begin;
            a.hist_end = p.history_end;
            a.rep = p.repetition;
            a.pres = p.presence;
            a.freq = p.frequency;
        }
        a.hist_len = int(p.history_len);
        a.bias_len = int(p.bias_len);
        a.mask_rows = p.mask_rows;
        a.bias_ids = p.bias_ids;
        a.bias_val = p.bias_values;
        a.bias_begin = p.bias_begin;
        a.bias_end = p.bias_end;
        a.mask = p.mask;
        a.mask_stride = p.mask_stride;
        a.mask_row = p.mask_row;
        a.choice = choice;
        OnDevice on;
        if (const int rc = on.enter("logits_process", logits)) return rc;
        return launched("logits_process", launch_logits_process(a, static_cast<cudaStream_t>(stream)));
    });
}

}  // extern "C"
