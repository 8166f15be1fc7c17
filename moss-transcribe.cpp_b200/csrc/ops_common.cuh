// Device helpers shared by the operators on a caller's own memory.
#pragma once

#include "ops.hpp"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

namespace mtb {
namespace ops {

__device__ __forceinline__ void flag(const PagedView& c, int bit) {
    if (c.status) atomicOr(c.status, bit);
}

// Positions that sequence s holds, inside its row of the page table.
__device__ __forceinline__ int seq_len(const PagedView& c, int s) {
    const int n = c.kv_len[s];
    const long long most = (long long)c.table_stride * kPage;
    if (n < 0 || n > most) {
        flag(c, BAD_LEN);
        return n < 0 ? 0 : (int)most;
    }
    return n;
}

// First new token of sequence s and their number (0 for a bad pair of bounds).
__device__ __forceinline__ int2 seq_tokens(const PagedView& c, const int* cu, int n_tokens, int s) {
    const int b = cu[s], e = cu[s + 1];
    if (b < 0 || e < b || e > n_tokens) {
        flag(c, BAD_TOKENS);
        return make_int2(0, 0);
    }
    return make_int2(b, e - b);
}

// The sequence that token t belongs to, -1 if none: the last s with cu[s] <= t.
__device__ __forceinline__ int seq_of_token(const int* cu, int n_seq, int t) {
    int lo = 0, hi = n_seq;  // cu[lo] <= t < cu[hi], as far as cu ascends
    if (t < cu[0] || t >= cu[n_seq]) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Page of positions [64 p, 64 p + 64) of sequence s, -1 if its entry is bad.
__device__ __forceinline__ int page_of(const PagedView& c, int s, int p) {
    const int id = c.table[(long long)s * c.table_stride + p];
    if ((unsigned)id >= (unsigned)c.n_pages) {
        flag(c, BAD_PAGE);
        return -1;
    }
    return id;
}

template <class T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N values between memory and f32 registers, 16 bytes an access.
template <class T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[N]) {
    constexpr int per = 16 / sizeof(T);
    static_assert(N % per == 0, "whole 16-byte accesses");
#pragma unroll
    for (int i = 0; i < N / per; ++i) {
        const uint4 u = *reinterpret_cast<const uint4*>(p + i * per);
        const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int j = 0; j < per; ++j) x[i * per + j] = to_f32<T>(t[j]);
    }
}
template <class T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[N]) {
    constexpr int per = 16 / sizeof(T);
    static_assert(N % per == 0, "whole 16-byte accesses");
#pragma unroll
    for (int i = 0; i < N / per; ++i) {
        uint4 u;
        T* t = reinterpret_cast<T*>(&u);
#pragma unroll
        for (int j = 0; j < per; ++j) t[j] = from_f32<T>(x[i * per + j]);
        *reinterpret_cast<uint4*>(p + i * per) = u;
    }
}

// Lets a kernel have that much dynamic shared memory, once on each device.
template <class K>
cudaError_t allow_smem(K* kernel, int bytes, std::atomic<uint64_t>* done, bool wide_clusters = false) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (device & 63);
    if (done->load(std::memory_order_relaxed) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && wide_clusters) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) done->fetch_or(bit, std::memory_order_relaxed);
    return e;
}

}  // namespace ops
}  // namespace mtb
