// mtb_logits_process: penalties for repeated tokens, biases and grammar masks
// on logits rows, with the greedy choice.
//
// Bound: bytes (each logit read and written once; one row of 152 k values: latency).
// A cluster of 8 CTAs takes a row, each an eighth of the vocabulary in slices
// of at most 8192 ids.  What touches few ids is put in shared memory first: a
// bitmap of the ids in the row's history or biases, their counts and the index
// of their last bias.  Only touched ids read those, so only they need be
// cleared.  The row's choice joins the CTAs' over distributed shared memory:
// no workspace, no atomics on values, and an order that does not matter
// (largest value, then lowest id).
#include "ops_common.cuh"

#include <algorithm>
#include <cooperative_groups.h>

namespace mtb {
namespace {

using namespace ops;
namespace cg = cooperative_groups;

constexpr int kLogitsCluster = 8;
constexpr int kLogitsThreads = 512;
constexpr int kLogitsSlice = 8192;
constexpr int kLogitsSmem = kLogitsSlice / 8 + kLogitsSlice * 8;

struct Best {
    float v;
    int i;
};
__device__ __forceinline__ Best better(Best a, Best b) { return b.v > a.v || (b.v == a.v && b.i >= 0 && b.i < a.i) ? b : a; }

template <class T, bool kVec>
__global__ void __cluster_dims__(kLogitsCluster, 1, 1) __launch_bounds__(kLogitsThreads) k_logits(LogitsArgs a) {
    extern __shared__ unsigned s_touched[];                                  // [slice / 32]
    int* s_count = reinterpret_cast<int*>(s_touched + kLogitsSlice / 32);    // [slice]
    int* s_bias = s_count + kLogitsSlice;                                    // [slice] index of the last entry, or -1
    __shared__ Best s_best[kLogitsThreads / 32];
    __shared__ Best s_cta;
    const int row = blockIdx.x / kLogitsCluster, part = blockIdx.x % kLogitsCluster;
    // The CTA's ids: whole mask words and whole 16-byte accesses.
    const int share = ((a.vocab + kLogitsCluster - 1) / kLogitsCluster + 31) / 32 * 32;
    const int first = min((long long)a.vocab, (long long)part * share), last = min((long long)a.vocab, (long long)first + share);
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
    T* y = a.y ? reinterpret_cast<T*>(a.y) + row * a.y_stride : nullptr;
    const int h0 = a.hist ? max(a.hist_begin[row], 0) : 0, h1 = a.hist ? min(a.hist_end[row], a.hist_len) : 0;
    const int b0 = a.bias_ids ? max(a.bias_begin[row], 0) : 0, b1 = a.bias_ids ? min(a.bias_end[row], a.bias_len) : 0;
    const bool has_rep = a.rep, has_freq = a.freq, has_pres = a.pres;
    const float rep = has_rep ? a.rep[row] : 1.f, freq = has_freq ? a.freq[row] : 0.f, pres = has_pres ? a.pres[row] : 0.f;
    const int mask_row = !a.mask ? -1 : a.mask_row ? a.mask_row[row] : row;
    const unsigned* mask = mask_row < 0 || mask_row >= a.mask_rows ? nullptr : a.mask + mask_row * a.mask_stride;
    Best best{-INFINITY, -1};
    for (int s0 = first; s0 < last; s0 += kLogitsSlice) {
        const int n = min(kLogitsSlice, last - s0);
        for (int i = threadIdx.x; i < (n + 31) / 32; i += kLogitsThreads) s_touched[i] = 0u;
        __syncthreads();
        const bool few = h1 > h0 || b1 > b0;
        if (few) {
            for (int i = h0 + threadIdx.x; i < h1; i += kLogitsThreads) {
                const int id = a.hist[i] - s0;
                if (a.hist[i] >= 0 && (unsigned)id < (unsigned)n) {
                    atomicOr(&s_touched[id >> 5], 1u << (id & 31));
                    s_count[id] = 0;
                    s_bias[id] = -1;
                }
            }
            for (int i = b0 + threadIdx.x; i < b1; i += kLogitsThreads) {
                const int id = a.bias_ids[i] - s0;
                if (a.bias_ids[i] >= 0 && (unsigned)id < (unsigned)n) {
                    atomicOr(&s_touched[id >> 5], 1u << (id & 31));
                    s_count[id] = 0;
                    s_bias[id] = -1;
                }
            }
            __syncthreads();
            for (int i = h0 + threadIdx.x; i < h1; i += kLogitsThreads) {
                const int id = a.hist[i] - s0;
                if (a.hist[i] >= 0 && (unsigned)id < (unsigned)n) atomicAdd(&s_count[id], 1);
            }
            for (int i = b0 + threadIdx.x; i < b1; i += kLogitsThreads) {
                const int id = a.bias_ids[i] - s0;
                if (a.bias_ids[i] >= 0 && (unsigned)id < (unsigned)n) atomicMax(&s_bias[id], i);
            }
            __syncthreads();
        }
        auto one = [&](float v, int id, unsigned touched, unsigned allowed) {
            if (touched) {
                const int cnt = s_count[id], bi = s_bias[id];
                if (cnt > 0) {
                    if (has_rep) v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
                    if (has_freq) v = __fsub_rn(v, __fmul_rn(freq, (float)cnt));
                    if (has_pres) v = __fsub_rn(v, pres);
                }
                if (bi >= 0) v = __fadd_rn(v, a.bias_val[bi]);
            }
            if (!allowed) v = -INFINITY;
            if (v > best.v) best = Best{v, s0 + id};
            return v;
        };
        constexpr int per = kVec ? 16 / sizeof(T) : 1;
        for (int i = threadIdx.x * per; i < n; i += kLogitsThreads * per) {
            const unsigned touched = s_touched[i >> 5] >> (i & 31);
            const unsigned allowed = mask ? mask[(s0 + i) >> 5] >> (i & 31) : 0xffffffffu;
            if (kVec && i + per <= n) {
                float v[per];
                if constexpr (kVec) load_vec<T, per>(x + s0 + i, v);
#pragma unroll
                for (int e = 0; e < per; ++e) v[e] = one(v[e], i + e, (touched >> e) & 1u, (allowed >> e) & 1u);
                if constexpr (kVec)
                    if (y) store_vec<T, per>(y + s0 + i, v);
            } else {
                for (int e = 0; e < per && i + e < n; ++e) {
                    const float v = one(to_f32<T>(x[s0 + i + e]), i + e, (touched >> e) & 1u, (allowed >> e) & 1u);
                    if (y) y[s0 + i + e] = from_f32<T>(v);
                }
            }
        }
        __syncthreads();
    }
    if (!a.choice) return;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o)});
    if ((threadIdx.x & 31) == 0) s_best[threadIdx.x >> 5] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kLogitsThreads / 32; ++w) best = better(best, s_best[w]);
        s_cta = best;
    }
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (part == 0 && threadIdx.x == 0) {
        for (int r = 1; r < kLogitsCluster; ++r) best = better(best, *cluster.map_shared_rank(&s_cta, r));
        a.choice[row] = best.i;
    }
    cluster.sync();
}

template <class T>
cudaError_t logits_typed(const LogitsArgs& a, cudaStream_t s) {
    constexpr int per = 16 / sizeof(T);
    auto ok = [](const void* p, long long stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % per == 0; };
    const bool vec = ok(a.x, a.x_stride) && (!a.y || ok(a.y, a.y_stride));
    auto go = [&](auto kernel) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kLogitsSmem);
        if (e != cudaSuccess) return e;
        kernel<<<a.rows * kLogitsCluster, kLogitsThreads, kLogitsSmem, s>>>(a);
        return cudaGetLastError();
    };
    return vec ? go(k_logits<T, true>) : go(k_logits<T, false>);
}

}  // namespace

cudaError_t launch_logits_process(const LogitsArgs& a, cudaStream_t s) {
    if (a.type == OP_F32) return logits_typed<float>(a, s);
    return a.type == OP_F16 ? logits_typed<__half>(a, s) : logits_typed<__nv_bfloat16>(a, s);
}

}  // namespace mtb
