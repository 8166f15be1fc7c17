// mtb_paged_attention and mtb_attention_weights.
//
// One CTA per (token, head), the cache in chunks of 128 slots: a thread forms
// one slot's score, the chunk's maximum and sum rescale the running ones
// (softmax in one pass), then a thread owns one dim of the row and adds the chunk's V.
#include "ops_common.cuh"

#include <algorithm>

namespace mtb {
namespace {

using namespace ops;

constexpr int kSimpleThreads = 128;

template <class T>
__global__ void __launch_bounds__(kSimpleThreads) k_attention_simple(AttnArgs a) {
    __shared__ float s_q[128], s_p[kSimpleThreads], s_red[4];
    const PagedView& c = a.c;
    const int t = blockIdx.x, h = blockIdx.y, D = c.head_dim, g = h / (a.n_heads / c.n_kv);
    const int seq = seq_of_token(a.cu, c.n_seq, t);
    if (seq < 0) return;
    const int2 tok = seq_tokens(c, a.cu, a.n_tokens, seq);
    if (t - tok.x >= tok.y) return;
    const int len = seq_len(c, seq);
    const int sees = len - tok.y + (t - tok.x) + 1;
    if (len < tok.y && threadIdx.x == 0) flag(c, BAD_LEN);
    const T* q = reinterpret_cast<const T*>(a.q) + t * a.q_stride + (long long)h * D;
    if (threadIdx.x < D) s_q[threadIdx.x] = to_f32<T>(q[threadIdx.x]);
    __syncthreads();
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (int j0 = 0; j0 < sees; j0 += kSimpleThreads) {
        const int j = j0 + threadIdx.x;
        float s = -INFINITY;
        if (j < sees) {
            const int page = page_of(c, seq, j / kPage);
            if (page >= 0) {
                const T* k = reinterpret_cast<const T*>(c.k) + page * c.page_stride + g * c.head_stride + (long long)(j % kPage) * D;
                s = 0.f;
                for (int d = 0; d < D; ++d) s = fmaf(s_q[d], to_f32<T>(k[d]), s);
                s *= a.scale;
            }
        }
        float mx = s;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
        const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.f : mn;
        const float p = expf(s - base), keep = expf(m - base);
        s_p[threadIdx.x] = p;
        __syncthreads();
        o *= keep;
        l *= keep;
        m = mn;
        for (int i = 0; i < min(kSimpleThreads, sees - j0); ++i) {
            l += s_p[i];
            if (threadIdx.x < D && s_p[i] != 0.f) {
                const int page = c.table[(long long)seq * c.table_stride + (j0 + i) / kPage];
                const T* v = reinterpret_cast<const T*>(c.v) + page * c.page_stride + g * c.head_stride + (long long)((j0 + i) % kPage) * D;
                o = fmaf(s_p[i], to_f32<T>(v[threadIdx.x]), o);
            }
        }
        __syncthreads();
    }
    T* out = reinterpret_cast<T*>(a.out) + t * a.out_stride + (long long)h * D;
    if (threadIdx.x < D) out[threadIdx.x] = from_f32<T>(l == 0.f ? 0.f : o / l);
    if (threadIdx.x == 0 && a.lse) a.lse[(long long)t * a.n_heads + h] = l == 0.f ? -INFINITY : m + logf(l);
}

// One CTA of 64 threads per (sequence, KV head, page): a thread owns a slot.
template <class T>
__global__ void __launch_bounds__(kPage) k_weights_simple(AttnArgs a, int pages) {
    __shared__ float s_q[128];
    const PagedView& c = a.c;
    const int seq = blockIdx.x / pages, p = blockIdx.x % pages, g = blockIdx.y, D = c.head_dim, G = a.n_heads / c.n_kv;
    const int2 tok = seq_tokens(c, a.cu, a.n_tokens, seq);
    const int len = seq_len(c, seq);
    if (tok.y == 0 || p * kPage >= len) return;
    const int page = page_of(c, seq, p);
    if (page < 0) return;
    const int slot = p * kPage + threadIdx.x;
    const T* k = reinterpret_cast<const T*>(c.k) + page * c.page_stride + g * c.head_stride + (long long)threadIdx.x * D;
    float w = 0.f;
    for (int i = max(0, p * kPage - (len - tok.y)); i < tok.y; ++i)
        for (int h = g * G; h < (g + 1) * G; ++h) {
            __syncthreads();
            const T* q = reinterpret_cast<const T*>(a.q) + (tok.x + i) * a.q_stride + (long long)h * D;
            for (int d = threadIdx.x; d < D; d += kPage) s_q[d] = to_f32<T>(q[d]);
            __syncthreads();
            if (slot > len - tok.y + i) continue;
            float s = 0.f;
            for (int d = 0; d < D; ++d) s = fmaf(s_q[d], to_f32<T>(k[d]), s);
            w += expf(s * a.scale - a.lse[(long long)(tok.x + i) * a.n_heads + h]);
        }
    if (slot < len) {
        float* at = c.weight + ((long long)page * c.n_kv + g) * kPage + threadIdx.x;
        *at = a.decay == 0.f ? w : fmaf(a.decay, *at, w);
    }
}

}  // namespace

cudaError_t launch_paged_attention(const AttnArgs& a, cudaStream_t s) {
    const dim3 grid(a.n_tokens, a.n_heads);
    if (a.c.type == OP_F16) k_attention_simple<__half><<<grid, kSimpleThreads, 0, s>>>(a);
    else k_attention_simple<__nv_bfloat16><<<grid, kSimpleThreads, 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_attention_weights(const AttnArgs& a, cudaStream_t s) {
    const dim3 grid(a.c.n_seq * a.c.table_stride, a.c.n_kv);
    if (a.c.type == OP_F16) k_weights_simple<__half><<<grid, kPage, 0, s>>>(a, a.c.table_stride);
    else k_weights_simple<__nv_bfloat16><<<grid, kPage, 0, s>>>(a, a.c.table_stride);
    return cudaGetLastError();
}

}  // namespace mtb
