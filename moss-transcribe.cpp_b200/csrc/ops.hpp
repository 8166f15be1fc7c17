// Operators on a caller's own device memory: what the C entries (ops_api.cu)
// hand to the kernels (ops_cache.cu, ops_attention.cu, ops_logits.cu).
#pragma once

#include "mtb_internal.hpp"

namespace mtb {

enum OpType : int { OP_F32 = 0, OP_F16 = 1, OP_BF16 = 2 };
enum OpStatus : int { BAD_PAGE = 1, BAD_LEN = 2, BAD_TOKENS = 4, BAD_WAIT = 8 };

constexpr int kMaxGroup = 64;  // query heads per KV head

// mtb_paged_cache as the kernels take it.
struct PagedView {
    char* k;
    char* v;
    int type, head_dim, n_kv, n_pages;
    long long page_stride, head_stride;  // elements
    const int* table;
    int table_stride, n_seq;
    const int* kv_len;
    int* position;
    float* weight;
    int* status;
};

struct RopeArgs {
    PagedView c;
    const int* cu;
    int n_tokens;
    const int* positions;
    int in_type;
    const char *q, *k, *v;
    long long q_stride, k_stride, v_stride, out_stride;
    int n_heads;
    const double* inv_freq;
    int rotary, interleaved;
    float factor;
    char* out;
};

// n / d for n < 2^31, without a division on the device: the high word of
// n * m, m = ceil(2^(32 + s) / d), shifted by s (d <= 2^(s + 1)).
struct FastDiv {
    uint32_t m;
    int s;
    static FastDiv of(int d) {
        FastDiv f{0, 0};
        while ((2ll << f.s) < d) ++f.s;
        f.m = d == 1 ? 0 : uint32_t(((1ull << (32 + f.s)) + d - 1) / d);
        return f;
    }
#ifdef __CUDACC__
    __device__ __forceinline__ int operator()(int n) const { return m ? int(__umulhi(uint32_t(n), m) >> s) : n; }
#endif
};

struct AttnArgs {
    PagedView c;
    const int* cu;
    int n_tokens, max_tokens;
    const char* q;
    long long q_stride;
    int n_heads;
    float scale;
    char* out;
    long long out_stride;
    float* lse;        // written by the attention, read by the weights
    float decay;       // weights only
    char* workspace;
    int G, per;         // query heads per KV head, new tokens per tile
    FastDiv by_G, by_per;
};

struct EvictArgs {
    PagedView c;
    int keep, sinks, recent;
    int* new_len;
    char* workspace;
};

struct LogitsArgs {
    const char* x;
    char* y;
    int type, rows, vocab;
    long long x_stride, y_stride;  // elements
    const int *hist, *hist_begin, *hist_end;
    const float *rep, *pres, *freq;
    const int* bias_ids;
    const float* bias_val;
    const int *bias_begin, *bias_end;
    const uint32_t* mask;
    long long mask_stride;
    const int* mask_row;
    int hist_len, bias_len, mask_rows;
    int* choice;
};

// Each returns the launch's error.  The device of the memory is current.
cudaError_t launch_rope_append(const RopeArgs& a, cudaStream_t s);
cudaError_t launch_paged_attention(const AttnArgs& a, cudaStream_t s);
cudaError_t launch_attention_weights(const AttnArgs& a, cudaStream_t s);
cudaError_t launch_cache_evict(const EvictArgs& a, cudaStream_t s);
cudaError_t launch_logits_process(const LogitsArgs& a, cudaStream_t s);

// Workspace bytes of the eviction: per (sequence, KV head) a 256-byte head and
// two lists of at most half the table's positions.
constexpr long long evict_workspace(long long n_seq, long long n_kv, long long table_stride) {
    return n_seq * n_kv * (256 + table_stride * kPage * 4);
}
constexpr long long kAttnWorkspace = 64ll << 20;

}  // namespace mtb
