// mtb_logits_process: penalties for repeated tokens, biases and grammar masks
// on logits rows, with the greedy choice.
//
// Bound: bytes (each logit read and written once; one row of 152 k values: latency).
// A cluster takes a row, 8 CTAs (16 while there are few rows).  The vocabulary goes
// round the CTAs in runs of 1024 ids, since histories crowd at low ids, in slices of at most 19 runs a
// CTA.  A slice has a word of shared memory for each id: its count in the row's history in
// the low half, its last bias entry + 1 in the high half (histories or bias lists
// of 65535 or more take two words an id).  All CTAs of the row read its whole
// history and keep what is theirs; who touches an id first puts it on a list.  Then the logits
// stream through, untouched ids for the choice, masked ones to -inf; and then the listed
// ids are done over: penalties and biases are a few
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
constexpr int kLogitsList = 8192;  // touched ids of a slice; of more, all its words are looked at
constexpr int kLogitsBatch = 4;    // 16-byte loads of a thread in flight
constexpr int kLogitsHeld = 8;     // history ids a thread reads ahead

struct Best {
    float v;
    int i;
};
__device__ __forceinline__ Best better(Best a, Best b) { return b.v > a.v || (b.v == a.v && b.i >= 0 && b.i < a.i) ? b : a; }

// A CTA's share of a row.
struct Share {
    int row, part, log_width;
    int h0, h1, b0, b1;
    const unsigned* mask;
};

template <class T, bool kVec, bool kWide>
__device__ __forceinline__ Best logits_share(const LogitsArgs& a, const Share& sh, unsigned* s_word, unsigned short* s_list, int* s_listed) {
    constexpr int per = kVec ? 16 / sizeof(T) : 1;
    constexpr int slice = kWide ? kLogitsSlice / 2 / kLogitsRun * kLogitsRun : kLogitsSlice;
    using Raw = typename std::conditional<kVec, uint4, T>::type;
    const T* x = reinterpret_cast<const T*>(a.x) + sh.row * a.x_stride;
    T* y = a.y ? reinterpret_cast<T*>(a.y) + sh.row * a.y_stride : nullptr;
    const int width = 1 << sh.log_width;
    const bool few = sh.h1 > sh.h0 || sh.b1 > sh.b0;
    // Places of the CTA's ids, in order: place i is id ((i / run) width + part) run + i % run.
    const int runs = (a.vocab + kLogitsRun - 1) / kLogitsRun;
    const int places = (runs - sh.part + width - 1) / width * kLogitsRun;  // the last run may be short
    unsigned* s_more = s_word + slice;                                     // wide: the bias entries
    auto id_of = [&](int place) { return (((place / kLogitsRun) << sh.log_width) + sh.part) * kLogitsRun + place % kLogitsRun; };
    // An id's place in the slice, negative if it is not there.
    auto place_of = [&](int id, int s0, int n) {
        const int run = id / kLogitsRun, at = (run >> sh.log_width) * kLogitsRun + id % kLogitsRun - s0;
        return (unsigned)id < (unsigned)a.vocab && (run & (width - 1)) == sh.part && (unsigned)at < (unsigned)n ? at : -1;
    };
    Best best{-INFINITY, -1};
    for (int s0 = 0; s0 < places; s0 += slice) {
        const int n = min(slice, places - s0);
        Raw raw[kLogitsBatch];
        auto fetch = [&](int i0) {
#pragma unroll
            for (int u = 0; u < kLogitsBatch; ++u) {
                const int i = i0 + u * kLogitsThreads * per, id = id_of(s0 + i);
                if (i < n && id + per <= a.vocab) raw[u] = *reinterpret_cast<const Raw*>(x + id);
            }
        };
        fetch(threadIdx.x * per);
        if (few) {
            int held[kLogitsHeld];
#pragma unroll
            for (int k = 0; k < kLogitsHeld; ++k) {
                const int i = sh.h0 + threadIdx.x + k * kLogitsThreads;
                held[k] = i < sh.h1 ? a.hist[i] : -1;
            }
            for (int i = threadIdx.x * 4; i < (kWide ? 2 * slice : n); i += kLogitsThreads * 4)
                *reinterpret_cast<uint4*>(s_word + i) = make_uint4(0, 0, 0, 0);
            if (threadIdx.x == 0) *s_listed = 0;
            __syncthreads();
            auto list = [&](int at) {
                const int k = atomicAdd(s_listed, 1);
                if (k < kLogitsList) s_list[k] = (unsigned short)at;
            };
#pragma unroll 1
            for (int i = sh.b0 + threadIdx.x; i < sh.b1; i += kLogitsThreads) {
                const int at = place_of(a.bias_ids[i], s0, n);
                if (at < 0) continue;
                const unsigned entry = (unsigned)(i - sh.b0) + 1u;
                if (atomicMax(kWide ? &s_more[at] : &s_word[at], kWide ? entry : entry << 16) == 0u) list(at);
            }
            if (sh.b1 > sh.b0 && sh.h1 > sh.h0) __syncthreads();  // counts are added below the bias entries
            auto count = [&](int id) {
                const int at = place_of(id, s0, n);
                if (at >= 0 && atomicAdd(&s_word[at], 1u) == 0u && (!kWide || s_more[at] == 0u)) list(at);
            };
#pragma unroll
            for (int k = 0; k < kLogitsHeld; ++k) count(held[k]);
#pragma unroll 1
            for (int i = sh.h0 + threadIdx.x + kLogitsHeld * kLogitsThreads; i < sh.h1; i += kLogitsThreads) count(a.hist[i]);
            __syncthreads();
        }
        auto touched = [&](int i) { return few && (s_word[i] | (kWide ? s_more[i] : 0u)) != 0u; };
#pragma unroll 1
        for (int i0 = threadIdx.x * per; i0 < n; i0 += kLogitsBatch * kLogitsThreads * per) {
#pragma unroll
            for (int u = 0; u < kLogitsBatch; ++u) {
                const int i = i0 + u * kLogitsThreads * per, id = id_of(s0 + i);
                if (i >= n || id >= a.vocab) break;
                if (id + per <= a.vocab) {
                    const T* t = reinterpret_cast<const T*>(&raw[u]);
                    float v[per], w[per];  // w: what may be chosen
#pragma unroll
                    for (int e = 0; e < per; ++e) v[e] = to_f32<T>(t[e]);
                    if (sh.mask) {
                        const unsigned allowed = sh.mask[id >> 5] >> (id & 31);
#pragma unroll
                        for (int e = 0; e < per; ++e)
                            if (!((allowed >> e) & 1u)) v[e] = -INFINITY;
                    }
#pragma unroll
                    for (int e = 0; e < per; ++e) w[e] = v[e];
                    if (few) {
                        if constexpr (kVec) {
#pragma unroll
                            for (int e = 0; e < per; e += 4) {
                                uint4 k = *reinterpret_cast<const uint4*>(s_word + i + e);
                                if (kWide) {
                                    const uint4 m = *reinterpret_cast<const uint4*>(s_more + i + e);
                                    k.x |= m.x, k.y |= m.y, k.z |= m.z, k.w |= m.w;
                                }
                                if (k.x) w[e] = -INFINITY;
                                if (k.y) w[e + 1] = -INFINITY;
                                if (k.z) w[e + 2] = -INFINITY;
                                if (k.w) w[e + 3] = -INFINITY;
                            }
                        } else if (touched(i)) {
                            w[0] = -INFINITY;
                        }
                    }
                    float top = w[0];
#pragma unroll
                    for (int e = 1; e < per; ++e) top = fmaxf(top, w[e]);
                    if (top > best.v) {  // seldom, once some have been seen
                        int at = per - 1;
#pragma unroll
                        for (int e = per - 2; e >= 0; --e)
                            if (w[e] == top) at = e;
                        best = Best{top, id + at};
                    }
                    if (y) {
                        if constexpr (kVec) store_vec<T, per>(y + id, v);
                        else y[id] = from_f32<T>(v[0]);
                    }
                } else {  // the row's last few ids
#pragma unroll 1
                    for (int e = 0; id + e < a.vocab; ++e) {
                        float v = to_f32<T>(x[id + e]);
                        if (sh.mask && !((sh.mask[(id + e) >> 5] >> ((id + e) & 31)) & 1u)) v = -INFINITY;
                        if (!touched(i + e) && v > best.v) best = Best{v, id + e};
                        if (y) y[id + e] = from_f32<T>(v);
                    }
                }
            }
            fetch(i0 + kLogitsBatch * kLogitsThreads * per);
        }
        if (few) {
            __syncthreads();  // the ids have been written
            const bool has_rep = a.rep, has_freq = a.freq, has_pres = a.pres;
            const float rep = has_rep ? a.rep[sh.row] : 1.f, freq = has_freq ? a.freq[sh.row] : 0.f, pres = has_pres ? a.pres[sh.row] : 0.f;
            const int listed = *s_listed;
            const bool all = listed > kLogitsList;
#pragma unroll 1
            for (int k = threadIdx.x; k < (all ? n : listed); k += kLogitsThreads) {
                const int at = all ? k : s_list[k];
                const unsigned word = s_word[at], more = kWide ? s_more[at] : 0u;
                if ((word | more) == 0u) continue;
                const int id = id_of(s0 + at);
                const int cnt = kWide ? word : word & 0xffffu, bi = (int)(kWide ? more : word >> 16) - 1;
                float v = to_f32<T>(x[id]);
                if (cnt > 0) {
                    if (has_rep) v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
                    if (has_freq) v = __fsub_rn(v, __fmul_rn(freq, (float)cnt));
                    if (has_pres) v = __fsub_rn(v, pres);
                }
                if (bi >= 0) v = __fadd_rn(v, a.bias_val[sh.b0 + bi]);
                if (sh.mask && !((sh.mask[id >> 5] >> (id & 31)) & 1u)) v = -INFINITY;
                if (v > best.v || (v == best.v && id < best.i)) best = Best{v, id};
                if (y) y[id] = from_f32<T>(v);
            }
            if (s0 + slice < places) __syncthreads();  // words and list are used again
        }
    }
    return best;
}

// 1 << log_width CTAs a row; table: bytes of the words.
template <class T, bool kVec>
__global__ void __launch_bounds__(kLogitsThreads, 2) k_logits(const __grid_constant__ LogitsArgs a, int log_width, int table) {
    extern __shared__ __align__(16) unsigned s_word[];
    unsigned short* s_list = reinterpret_cast<unsigned short*>(reinterpret_cast<char*>(s_word) + table);
    __shared__ Best s_best[kLogitsThreads / 32];
    __shared__ Best s_row[16];
    __shared__ __align__(8) uint64_t s_done;
    __shared__ int s_listed;
    const int width = 1 << log_width, row = blockIdx.x >> log_width, part = blockIdx.x & (width - 1);
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t done = (uint32_t)__cvta_generic_to_shared(&s_done);
    if (threadIdx.x == 0) {
        asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(done), "r"(width) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // waited for where the choice is joined
    Share sh{row, part, log_width, 0, 0, 0, 0, nullptr};
    if (a.hist) sh.h0 = max(a.hist_begin[row], 0), sh.h1 = min(a.hist_end[row], a.hist_len);
    if (a.bias_ids) sh.b0 = max(a.bias_begin[row], 0), sh.b1 = min(a.bias_end[row], a.bias_len);
    if (a.mask) {
        const int m = a.mask_row ? a.mask_row[row] : row;
        if (m >= 0 && m < a.mask_rows) sh.mask = a.mask + m * a.mask_stride;
    }
    Best best = sh.h1 - sh.h0 > 65535 || sh.b1 - sh.b0 > 65534 ? logits_share<T, kVec, true>(a, sh, s_word, s_list, &s_listed)
                                                               : logits_share<T, kVec, false>(a, sh, s_word, s_list, &s_listed);
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
    cudaError_t e = allow_smem(kernel, kLogitsSlice * 4 + kLogitsList * 2, &done, true);
    if (e != cudaSuccess) return e;
    // 16 CTAs a row while that leaves SMs without work (two CTAs fit each).
    const int log_width = a.rows <= 148 * 2 / 16 && a.vocab > 8 * kLogitsRun ? 4 : 3, width = 1 << log_width;
    const int places = ((a.vocab + kLogitsRun - 1) / kLogitsRun + width - 1) / width * kLogitsRun;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(a.rows * width);
    c.blockDim = dim3(kLogitsThreads);
    // Rows that may need two words an id take the whole table.
    const int words = a.hist_len > 65535 || a.bias_len > 65534 ? kLogitsSlice : std::min(places, kLogitsSlice);
    const int table = a.hist || a.bias_ids ? words * 4 : 0;
    c.dynamicSmemBytes = table ? table + kLogitsList * 2 : 0;
    c.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)width, 1, 1};
    c.attrs = at;
    c.numAttrs = 1;
    e = cudaLaunchKernelEx(&c, kernel, a, log_width, table);
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
