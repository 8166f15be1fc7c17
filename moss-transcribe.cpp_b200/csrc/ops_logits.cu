// mtb_logits_process: penalties for repeated tokens, biases and grammar masks
// on logits rows, with the greedy choice.
//
// Bound: bytes (each logit read and written once; one row of 152 k values: latency).
// A cluster takes a row, 8 CTAs (16 while there are few rows).  The vocabulary goes
// round the CTAs in runs of 1024 ids, since histories crowd at low ids, in slices of at most 19 runs a
// CTA.  A slice has a word of shared memory for each id: its count in the row's history in
// the low half, its last bias entry + 1 in the high half (histories or bias lists
// of 65535 or more take two words an id).  All CTAs of the row read its whole
// history and keep what is theirs.  Then the logits stream through, untouched ids for the
// choice, masked ones to -inf; and then each touched id is done over, by whoever of
// the history's threads first takes its word away: penalties and biases are a few
// thousand ids, and cost the stream no branch.  Two CTAs to an SM, so that one
// streams while the other counts.  The row's choice joins the CTAs' in the first one's shared
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
constexpr int kLogitsRun = 1024;
constexpr int kLogitsSlice = 19 * kLogitsRun;
constexpr int kLogitsSmem = kLogitsSlice * 4;
constexpr int kLogitsBatch = 4;  // 16-byte loads of a thread in flight
constexpr int kLogitsHeld = 8;   // history ids a thread reads ahead

struct Best {
    float v;
    int i;
};
__device__ __forceinline__ Best better(Best a, Best b) { return b.v > a.v || (b.v == a.v && b.i >= 0 && b.i < a.i) ? b : a; }

// width = 1 << log_width CTAs a row.
template <class T, bool kVec>
__global__ void __launch_bounds__(kLogitsThreads, 2) k_logits(const __grid_constant__ LogitsArgs a, int log_width) {
    constexpr int per = kVec ? 16 / sizeof(T) : 1;
    using Raw = typename std::conditional<kVec, uint4, T>::type;
    extern __shared__ __align__(16) unsigned s_word[];
    __shared__ Best s_best[kLogitsThreads / 32];
    __shared__ Best s_row[16];
    __shared__ __align__(8) uint64_t s_done;
    const int width = 1 << log_width, row = blockIdx.x >> log_width, part = blockIdx.x & (width - 1);
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t done = (uint32_t)__cvta_generic_to_shared(&s_done);
    if (threadIdx.x == 0) {
        asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(done), "r"(width) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // waited for where the choice is joined
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
    T* y = a.y ? reinterpret_cast<T*>(a.y) + row * a.y_stride : nullptr;
    const int h0 = a.hist ? max(a.hist_begin[row], 0) : 0, h1 = a.hist ? min(a.hist_end[row], a.hist_len) : 0;
    const int b0 = a.bias_ids ? max(a.bias_begin[row], 0) : 0, b1 = a.bias_ids ? min(a.bias_end[row], a.bias_len) : 0;
    const int mask_row = !a.mask ? -1 : a.mask_row ? a.mask_row[row] : row;
    const unsigned* mask = mask_row < 0 || mask_row >= a.mask_rows ? nullptr : a.mask + mask_row * a.mask_stride;
    const bool few = h1 > h0 || b1 > b0;
    const bool wide = h1 - h0 > 65535 || b1 - b0 > 65534;
    // Places of the CTA's ids, in order: place i is id ((i / run) width + part) run + i % run.
    const int slice = wide ? kLogitsSlice / 2 / kLogitsRun * kLogitsRun : kLogitsSlice;
    const int runs = (a.vocab + kLogitsRun - 1) / kLogitsRun;
    const int places = (runs - part + width - 1) / width * kLogitsRun;  // the last run may be short
    unsigned* s_more = s_word + slice;                                  // wide: the bias entries
    auto id_of = [&](int place) { return (((place / kLogitsRun) << log_width) + part) * kLogitsRun + place % kLogitsRun; };
    // Whether an id is the CTA's, and its place.
    auto place_of = [&](int id, int* place) {
        const int run = id / kLogitsRun;
        *place = (run >> log_width) * kLogitsRun + id % kLogitsRun;
        return (unsigned)id < (unsigned)a.vocab && (run & (width - 1)) == part;
    };
    Best best{-INFINITY, -1};
    for (int s0 = 0; s0 < places; s0 += slice) {
        const int n = min(slice, places - s0);
        Raw raw[kLogitsBatch];
        auto fetch = [&](int i0) {
#pragma unroll
            for (int u = 0; u < kLogitsBatch; ++u) {
                const int i = i0 + u * kLogitsThreads * per;
                if (i < n) {
                    const int id = id_of(s0 + i);
                    if (id + per <= a.vocab) raw[u] = *reinterpret_cast<const Raw*>(x + id);
                }
            }
        };
        fetch(threadIdx.x * per);
        int held[kLogitsHeld];
        if (few) {
#pragma unroll
            for (int k = 0; k < kLogitsHeld; ++k) {
                const int i = h0 + threadIdx.x + k * kLogitsThreads;
                held[k] = i < h1 ? a.hist[i] : -1;
            }
            const int words = wide ? 2 * slice : n;
            for (int i = threadIdx.x * 4; i < words; i += kLogitsThreads * 4) *reinterpret_cast<uint4*>(s_word + i) = make_uint4(0, 0, 0, 0);
            __syncthreads();
            for (int i = b0 + threadIdx.x; i < b1; i += kLogitsThreads) {
                int at;
                if (place_of(a.bias_ids[i], &at) && (unsigned)(at -= s0) < (unsigned)n) {
                    if (wide) atomicMax(&s_more[at], (unsigned)(i - b0) + 1u);
                    else atomicMax(&s_word[at], ((unsigned)(i - b0) + 1u) << 16);
                }
            }
            if (b1 > b0 && h1 > h0) __syncthreads();  // counts are added below the bias entries
            auto count = [&](int id) {
                int at;
                if (place_of(id, &at) && (unsigned)(at -= s0) < (unsigned)n) atomicAdd(&s_word[at], 1u);
            };
#pragma unroll
            for (int k = 0; k < kLogitsHeld; ++k) count(held[k]);
            for (int i = h0 + threadIdx.x + kLogitsHeld * kLogitsThreads; i < h1; i += kLogitsThreads) count(a.hist[i]);
            __syncthreads();
        }
        for (int i0 = threadIdx.x * per; i0 < n; i0 += kLogitsBatch * kLogitsThreads * per) {
#pragma unroll
            for (int u = 0; u < kLogitsBatch; ++u) {
                const int i = i0 + u * kLogitsThreads * per, id = id_of(s0 + i);
                if (i >= n || id >= a.vocab) break;
                const unsigned allowed = mask ? mask[id >> 5] >> (id & 31) : 0xffffffffu;
                auto one = [&](float v, int e, unsigned touched) {
                    if (!((allowed >> e) & 1u)) v = -INFINITY;
                    if (!touched && v > best.v) best = Best{v, id + e};
                    return v;
                };
                if (id + per <= a.vocab) {
                    if constexpr (kVec) {
                        const T* t = reinterpret_cast<const T*>(&raw[u]);
                        float v[per];
#pragma unroll
                        for (int e = 0; e < per; e += 4) {
                            uint4 w = make_uint4(0, 0, 0, 0);
                            if (few) {
                                w = *reinterpret_cast<const uint4*>(s_word + i + e);
                                if (wide) {
                                    const uint4 m = *reinterpret_cast<const uint4*>(s_more + i + e);
                                    w.x |= m.x, w.y |= m.y, w.z |= m.z, w.w |= m.w;
                                }
                            }
                            v[e] = one(to_f32<T>(t[e]), e, w.x);
                            v[e + 1] = one(to_f32<T>(t[e + 1]), e + 1, w.y);
                            v[e + 2] = one(to_f32<T>(t[e + 2]), e + 2, w.z);
                            v[e + 3] = one(to_f32<T>(t[e + 3]), e + 3, w.w);
                        }
                        if (y) store_vec<T, per>(y + id, v);
                    } else {
                        const float v = one(to_f32<T>(raw[u]), 0, few ? s_word[i] | (wide ? s_more[i] : 0u) : 0u);
                        if (y) y[id] = from_f32<T>(v);
                    }
                } else {  // the row's last few ids
                    for (int e = 0; id + e < a.vocab; ++e) {
                        const float v = one(to_f32<T>(x[id + e]), e, few ? s_word[i + e] | (wide ? s_more[i + e] : 0u) : 0u);
                        if (y) y[id + e] = from_f32<T>(v);
                    }
                }
            }
            fetch(i0 + kLogitsBatch * kLogitsThreads * per);
        }
        if (few) {
            __syncthreads();  // the words have been read, the ids written
            const bool has_rep = a.rep, has_freq = a.freq, has_pres = a.pres;
            const float rep = has_rep ? a.rep[row] : 1.f, freq = has_freq ? a.freq[row] : 0.f, pres = has_pres ? a.pres[row] : 0.f;
            auto redo = [&](int id, bool from_history) {
                int at;
                if (!place_of(id, &at) || (unsigned)(at -= s0) >= (unsigned)n) return;
                // Who takes the word takes the id; of two words, the count's first.
                const unsigned word = atomicExch(&s_word[at], 0u);
                if (word == 0u && !(wide && !from_history)) return;
                const unsigned more = wide ? atomicExch(&s_more[at], 0u) : 0u;
                if ((word | more) == 0u) return;
                const int cnt = wide ? word : word & 0xffffu, bi = (int)(wide ? more : word >> 16) - 1;
                float v = to_f32<T>(x[id]);
                if (cnt > 0) {
                    if (has_rep) v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
                    if (has_freq) v = __fsub_rn(v, __fmul_rn(freq, (float)cnt));
                    if (has_pres) v = __fsub_rn(v, pres);
                }
                if (bi >= 0) v = __fadd_rn(v, a.bias_val[b0 + bi]);
                if (mask && !((mask[id >> 5] >> (id & 31)) & 1u)) v = -INFINITY;
                if (v > best.v || (v == best.v && id < best.i)) best = Best{v, id};
                if (y) y[id] = from_f32<T>(v);
            };
#pragma unroll 1
            for (int i = h0 + threadIdx.x; i < h1; i += kLogitsThreads) redo(a.hist[i], true);
            if (wide) __syncthreads();  // an id with both has gone with its count
#pragma unroll 1
            for (int i = b0 + threadIdx.x; i < b1; i += kLogitsThreads) redo(a.bias_ids[i], false);
            if (s0 + slice < places) __syncthreads();  // the words are used again
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o)});
    if ((threadIdx.x & 31) == 0) s_best[threadIdx.x >> 5] = best;
    __syncthreads();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all CTAs have begun
    if (!a.choice || threadIdx.x >= 32) return;
    best = threadIdx.x < kLogitsThreads / 32 ? s_best[threadIdx.x] : Best{-INFINITY, -1};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o)});
    if (threadIdx.x == 0) {
        // Into the first CTA's memory; it alone stays until all have come.
        *cluster.map_shared_rank(&s_row[part], 0) = best;
        uint32_t there;
        asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(there) : "r"(done));
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(there) : "memory");
    }
    if (part) return;
    bool ok = false;
    for (int left = 1 << 22; !ok && left > 0; --left) {
        uint32_t is;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], 0;\n selp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(is)
                     : "r"(done)
                     : "memory");
        ok = is;
    }
    best = ok && (int)threadIdx.x < width ? s_row[threadIdx.x] : Best{-INFINITY, -1};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o)});
    if (threadIdx.x == 0) a.choice[row] = best.i;
}

template <class T, bool kVec>
cudaError_t logits_launch(const LogitsArgs& a, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    auto* kernel = k_logits<T, kVec>;
    cudaError_t e = allow_smem(kernel, kLogitsSmem, &done, true);
    if (e != cudaSuccess) return e;
    // 16 CTAs a row while that leaves SMs without work (two CTAs fit each).
    const int log_width = a.rows <= 148 * 2 / 16 && a.vocab > 8 * kLogitsRun ? 4 : 3, width = 1 << log_width;
    const int places = ((a.vocab + kLogitsRun - 1) / kLogitsRun + width - 1) / width * kLogitsRun;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(a.rows * width);
    c.blockDim = dim3(kLogitsThreads);
    // Rows that may need two words an id take the whole table.
    c.dynamicSmemBytes = a.hist_len > 65535 || a.bias_len > 65534 ? kLogitsSmem : std::min(places * 4, kLogitsSmem);
    c.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)width, 1, 1};
    c.attrs = at;
    c.numAttrs = 1;
    e = cudaLaunchKernelEx(&c, kernel, a, log_width);
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
