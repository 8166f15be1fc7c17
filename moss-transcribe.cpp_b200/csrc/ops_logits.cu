// mtb_logits_process: penalties for repeated tokens, biases and grammar masks
// on logits rows, with the greedy choice.
//
// Bound: bytes (each logit read and written once; one row of 152 k values: latency).
// A cluster takes a row, 8 CTAs (16 while there are few rows), each an equal
// share of the vocabulary in slices of at most 19456 ids.  A slice has a word of
// shared memory for each id: its count in the row's history in the low half, its
// last bias entry + 1 in the high half (histories or bias lists of 65535 or more
// take two words an id).  All CTAs of the row read its whole history and keep what is theirs; the
// first logits are on their way meanwhile.  Two CTAs to an SM, so that one streams while
// the other counts.  The row's choice joins the CTAs' over distributed shared
// memory: no workspace, no atomics on values, and an order that does not matter
// (largest value, then lowest id).
#include "ops_common.cuh"

#include <algorithm>
#include <cooperative_groups.h>
#include <type_traits>

namespace mtb {
namespace {

using namespace ops;
namespace cg = cooperative_groups;

constexpr int kLogitsThreads = 512;
constexpr int kLogitsSlice = 19456;
constexpr int kLogitsSmem = kLogitsSlice * 4;
constexpr int kLogitsBatch = 4;  // 16-byte loads of a thread in flight

struct Best {
    float v;
    int i;
};
__device__ __forceinline__ Best better(Best a, Best b) { return b.v > a.v || (b.v == a.v && b.i >= 0 && b.i < a.i) ? b : a; }

template <class T, bool kVec>
__global__ void __launch_bounds__(kLogitsThreads, 2) k_logits(const __grid_constant__ LogitsArgs a, int width) {
    constexpr int per = kVec ? 16 / sizeof(T) : 1;
    using Raw = typename std::conditional<kVec, uint4, T>::type;
    extern __shared__ __align__(16) unsigned s_word[];
    __shared__ Best s_best[kLogitsThreads / 32];
    __shared__ Best s_cta;
    const int row = blockIdx.x / width, part = blockIdx.x % width;
    // The CTA's ids: whole mask words and whole 16-byte accesses.
    const int share = ((a.vocab + width - 1) / width + 31) / 32 * 32;
    const int first = (int)min((long long)a.vocab, (long long)part * share), last = (int)min((long long)a.vocab, (long long)first + share);
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
    T* y = a.y ? reinterpret_cast<T*>(a.y) + row * a.y_stride : nullptr;
    const int h0 = a.hist ? max(a.hist_begin[row], 0) : 0, h1 = a.hist ? min(a.hist_end[row], a.hist_len) : 0;
    const int b0 = a.bias_ids ? max(a.bias_begin[row], 0) : 0, b1 = a.bias_ids ? min(a.bias_end[row], a.bias_len) : 0;
    const bool has_rep = a.rep, has_freq = a.freq, has_pres = a.pres;
    const float rep = has_rep ? a.rep[row] : 1.f, freq = has_freq ? a.freq[row] : 0.f, pres = has_pres ? a.pres[row] : 0.f;
    const int mask_row = !a.mask ? -1 : a.mask_row ? a.mask_row[row] : row;
    const unsigned* mask = mask_row < 0 || mask_row >= a.mask_rows ? nullptr : a.mask + mask_row * a.mask_stride;
    const bool few = h1 > h0 || b1 > b0;
    const bool wide = h1 - h0 > 65535 || b1 - b0 > 65534;
    const int slice = wide ? kLogitsSlice / 2 : kLogitsSlice;
    unsigned* s_more = s_word + kLogitsSlice / 2;  // wide: the bias entries
    Best best{-INFINITY, -1};
    for (int s0 = first; s0 < last; s0 += slice) {
        const int n = min(slice, last - s0);
        Raw raw[kLogitsBatch];
        auto fetch = [&](int i0) {
#pragma unroll
            for (int u = 0; u < kLogitsBatch; ++u) {
                const int i = i0 + u * kLogitsThreads * per;
                if (i + per <= n) raw[u] = *reinterpret_cast<const Raw*>(x + s0 + i);
            }
        };
        fetch(threadIdx.x * per);
        if (few) {
            const int words = wide ? kLogitsSlice : (n + 3) / 4 * 4;
            for (int i = threadIdx.x * 4; i < words; i += kLogitsThreads * 4) *reinterpret_cast<uint4*>(s_word + i) = make_uint4(0, 0, 0, 0);
            __syncthreads();
            for (int i = b0 + threadIdx.x; i < b1; i += kLogitsThreads) {
                const int id = a.bias_ids[i], at = id - s0;
                if (id >= 0 && (unsigned)at < (unsigned)n) {
                    if (wide) atomicMax(&s_more[at], (unsigned)(i - b0) + 1u);
                    else atomicMax(&s_word[at], ((unsigned)(i - b0) + 1u) << 16);
                }
            }
            if (b1 > b0 && h1 > h0) __syncthreads();  // counts are added below the bias entries
#pragma unroll 4
            for (int i = h0 + threadIdx.x; i < h1; i += kLogitsThreads) {
                const int id = a.hist[i], at = id - s0;
                if (id >= 0 && (unsigned)at < (unsigned)n) atomicAdd(&s_word[at], 1u);
            }
            __syncthreads();
        }
        auto one = [&](float v, int i, unsigned word, unsigned allowed) {
            const unsigned more = wide && few ? s_more[i] : 0u;
            if (word | more) {
                const int cnt = wide ? word : word & 0xffffu, bi = (int)(wide ? more : word >> 16) - 1;
                if (cnt > 0) {
                    if (has_rep) v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
                    if (has_freq) v = __fsub_rn(v, __fmul_rn(freq, (float)cnt));
                    if (has_pres) v = __fsub_rn(v, pres);
                }
                if (bi >= 0) v = __fadd_rn(v, a.bias_val[b0 + bi]);
            }
            if (!allowed) v = -INFINITY;
            if (v > best.v) best = Best{v, s0 + i};
            return v;
        };
        for (int i0 = threadIdx.x * per; i0 < n; i0 += kLogitsBatch * kLogitsThreads * per) {
#pragma unroll
            for (int u = 0; u < kLogitsBatch; ++u) {
                const int i = i0 + u * kLogitsThreads * per;
                if (i >= n) break;
                const unsigned allowed = mask ? mask[(s0 + i) >> 5] >> (i & 31) : 0xffffffffu;
                if (i + per <= n) {
                    if constexpr (kVec) {
                        const T* t = reinterpret_cast<const T*>(&raw[u]);
                        float v[per];
#pragma unroll
                        for (int e = 0; e < per; e += 4) {
                            const uint4 w = few ? *reinterpret_cast<const uint4*>(s_word + i + e) : make_uint4(0, 0, 0, 0);
                            v[e] = one(to_f32<T>(t[e]), i + e, w.x, (allowed >> e) & 1u);
                            v[e + 1] = one(to_f32<T>(t[e + 1]), i + e + 1, w.y, (allowed >> (e + 1)) & 1u);
                            v[e + 2] = one(to_f32<T>(t[e + 2]), i + e + 2, w.z, (allowed >> (e + 2)) & 1u);
                            v[e + 3] = one(to_f32<T>(t[e + 3]), i + e + 3, w.w, (allowed >> (e + 3)) & 1u);
                        }
                        if (y) store_vec<T, per>(y + s0 + i, v);
                    } else {
                        const float v = one(to_f32<T>(raw[u]), i, few ? s_word[i] : 0u, allowed & 1u);
                        if (y) y[s0 + i] = from_f32<T>(v);
                    }
                } else {  // the row's last few ids
                    for (int e = 0; i + e < n; ++e) {
                        const float v = one(to_f32<T>(x[s0 + i + e]), i + e, few ? s_word[i + e] : 0u, (allowed >> e) & 1u);
                        if (y) y[s0 + i + e] = from_f32<T>(v);
                    }
                }
            }
            fetch(i0 + kLogitsBatch * kLogitsThreads * per);
        }
        if (s0 + slice < last) __syncthreads();  // the words are used again
    }
    if (!a.choice) return;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o)});
    if ((threadIdx.x & 31) == 0) s_best[threadIdx.x >> 5] = best;
    __syncthreads();
    if (threadIdx.x < 32) {
        best = threadIdx.x < kLogitsThreads / 32 ? s_best[threadIdx.x] : Best{-INFINITY, -1};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o)});
        if (threadIdx.x == 0) s_cta = best;
    }
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (part == 0 && threadIdx.x < 32) {
        best = (int)threadIdx.x < width ? *cluster.map_shared_rank(&s_cta, threadIdx.x) : Best{-INFINITY, -1};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o)});
        if (threadIdx.x == 0) a.choice[row] = best.i;
    }
    cluster.sync();
}

template <class T, bool kVec>
cudaError_t logits_launch(const LogitsArgs& a, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    auto* kernel = k_logits<T, kVec>;
    cudaError_t e = allow_smem(kernel, kLogitsSmem, &done, true);
    if (e != cudaSuccess) return e;
    // 16 CTAs a row while that leaves SMs without work (two CTAs fit each).
    const int width = a.rows <= 148 * 2 / 16 && a.vocab >= 16 * 1024 ? 16 : 8;
    const int share = ((a.vocab + width - 1) / width + 31) / 32 * 32;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(a.rows * width);
    c.blockDim = dim3(kLogitsThreads);
    // Two words an id only in a full table: the device decides.
    c.dynamicSmemBytes = share * 2 > kLogitsSlice || a.hist_len > 65535 || a.bias_len > 65534 ? kLogitsSmem : std::max(share * 4, 16);
    c.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)width, 1, 1};
    c.attrs = at;
    c.numAttrs = 1;
    e = cudaLaunchKernelEx(&c, kernel, a, width);
    return e != cudaSuccess ? e : cudaGetLastError();
}

template <class T>
cudaError_t logits_typed(const LogitsArgs& a, cudaStream_t s) {
    constexpr int per = 16 / sizeof(T);
    auto ok = [](const void* p, long long stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % per == 0; };
    const bool vec = ok(a.x, a.x_stride) && (!a.y || ok(a.y, a.y_stride));
    return vec ? logits_launch<T, true>(a, s) : logits_launch<T, false>(a, s);
}

}  // namespace

cudaError_t launch_logits_process(const LogitsArgs& a, cudaStream_t s) {
    if (a.type == OP_F32) return logits_typed<float>(a, s);
    return a.type == OP_F16 ? logits_typed<__half>(a, s) : logits_typed<__nv_bfloat16>(a, s);
}

}  // namespace mtb
