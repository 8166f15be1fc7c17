// mtb_logits_process: penalties for repeated tokens, biases and grammar masks
// on logits rows, with the greedy choice.
//
// Bound: bytes (each logit read and written once); one row of 152 k values: latency.
// A row belongs to 1 to 16 CTAs, as many as fill the SMs (one from 128 rows on: two
// CTAs to an SM, each a row; clusters of more take longer to place than they save).
// The vocabulary goes round a row's CTAs in runs of 1024 ids, since histories crowd at
// low ids.  What touches few ids is set apart: a hash table in shared memory takes the ids of
// the row's history and biases that are the CTA's, with their counts (low half of a
// word) and last bias entry + 1 (high half), and a bitmap says which ids it has.  The
// table's words then become the ids' new values.  The logits stream through once: masked ones to
// -inf, those of the bitmap from the table (writing them behind the stream instead cost 256 rows
// with 4096 ids of history 35 us in sectors written twice, and penalties within the
// stream as much in divergence).  Lists of more than 6144
// entries, or shares of more than 262144 ids, go in slices of 8192 ids with two words each
// instead.  The row's choice joins the CTAs' in the first one's shared
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
constexpr int kTableSlots = 8192;         // hash table: ids, then words; or a slice's two words an id
constexpr int kTableMost = 6144;          // entries of history and biases that it takes
constexpr int kShareMost = 32768 * 8;     // ids of the bitmap
constexpr int kTableBytes = kTableSlots * 8;
constexpr int kLogitsBatch = 5;           // 16-byte loads of a thread in flight
constexpr int kLogitsHeld = 8;            // history ids a thread reads ahead

struct Best {
    float v;
    int i;
};
__device__ __forceinline__ Best better(Best a, Best b) { return b.v > a.v || (b.v == a.v && b.i >= 0 && b.i < a.i) ? b : a; }
__device__ __forceinline__ Best warp_best(Best b) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) b = better(b, Best{__shfl_xor_sync(0xffffffffu, b.v, o), __shfl_xor_sync(0xffffffffu, b.i, o)});
    return b;
}

// A CTA's share of a row.  Places of its ids, in order: place i is id
// ((i / run) width + part) run + i % run.
struct Share {
    int row, part, log_width;
    int places;  // the last run may be short
    int h0, h1, b0, b1;
    const unsigned* mask;
    __device__ __forceinline__ int id_of(int place) const { return (((place / kLogitsRun) << log_width) + part) * kLogitsRun + place % kLogitsRun; }
    // An id's place, negative if it is not the CTA's.
    __device__ __forceinline__ int place_of(int id, int vocab) const {
        const int run = id / kLogitsRun;
        return (unsigned)id < (unsigned)vocab && (run & ((1 << log_width) - 1)) == part ? (run >> log_width) * kLogitsRun + id % kLogitsRun : -1;
    }
};

template <class T, bool kVec>
struct Batch {
    static constexpr int per = kVec ? 16 / sizeof(T) : 1;
    static constexpr int kStep = kLogitsBatch * kLogitsThreads * per;
    using Raw = typename std::conditional<kVec, uint4, T>::type;
    Raw raw[kLogitsBatch];
    unsigned allowed[kLogitsBatch];
    // The thread's vectors from place i0 of the share on.
    __device__ __forceinline__ void fetch(const T* x, const Share& sh, int vocab, int i0) {
#pragma unroll
        for (int u = 0; u < kLogitsBatch; ++u) {
            const int i = i0 + u * kLogitsThreads * per, id = sh.id_of(i);
            if (i < sh.places && id + per <= vocab) raw[u] = *reinterpret_cast<const Raw*>(x + id);
        }
    }
    __device__ __forceinline__ void masks(const Share& sh, int vocab, int i0) {
#pragma unroll
        for (int u = 0; u < kLogitsBatch; ++u) {
            const int i = i0 + u * kLogitsThreads * per, id = sh.id_of(i);
            allowed[u] = sh.mask && i < sh.places && id < vocab ? sh.mask[id >> 5] >> (id & 31) : 0xffffffffu;
        }
    }
};

struct Penalties {
    bool has_rep, has_freq, has_pres;
    float rep, freq, pres;
    const float* bias;
    __device__ __forceinline__ Penalties(const LogitsArgs& a, const Share& sh)
        : has_rep(a.rep), has_freq(a.freq), has_pres(a.pres), rep(a.rep ? a.rep[sh.row] : 1.f), freq(a.freq ? a.freq[sh.row] : 0.f),
          pres(a.pres ? a.pres[sh.row] : 0.f), bias(a.bias_val + sh.b0) {}
    __device__ __forceinline__ float operator()(float v, int count, int entry) const {
        if (count > 0) {
            if (has_rep) v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
            if (has_freq) v = __fsub_rn(v, __fmul_rn(freq, (float)count));
            if (has_pres) v = __fsub_rn(v, pres);
        }
        return entry >= 0 ? __fadd_rn(v, bias[entry]) : v;
    }
};

// Places [s0, s0 + n) through: penalties and biases for those of the bitmap (of the n
// places, or null), as `change` of place and value has them; masks; the choice.  `got`
// holds the first batch.
template <class T, bool kVec, class F>
__device__ __forceinline__ void stream(const LogitsArgs& a, const Share& sh, const T* x, T* y, Batch<T, kVec>& got, int s0, int n,
                                       const unsigned* s_bits, F&& change, Best& best) {
    constexpr int per = Batch<T, kVec>::per;
#pragma unroll 1
    for (int i0 = threadIdx.x * per; i0 < n; i0 += Batch<T, kVec>::kStep) {
#pragma unroll
        for (int u = 0; u < kLogitsBatch; ++u) {
            const int i = i0 + u * kLogitsThreads * per, id = sh.id_of(s0 + i);
            if (i >= n || id >= a.vocab) break;
            const unsigned touched = s_bits ? s_bits[i >> 5] >> (i & 31) : 0u;
            if (id + per <= a.vocab) {
                const T* t = reinterpret_cast<const T*>(&got.raw[u]);
                float v[per];
#pragma unroll
                for (int e = 0; e < per; ++e) v[e] = to_f32<T>(t[e]);
#pragma unroll 1
                for (unsigned bits = touched & got.allowed[u] & ((1u << per) - 1); bits; bits &= bits - 1) {
                    const int at = __ffs(bits) - 1;
                    float w = v[0];
#pragma unroll
                    for (int e = 1; e < per; ++e) w = e == at ? v[e] : w;
                    w = change(i + at, id + at, w);
#pragma unroll
                    for (int e = 0; e < per; ++e) v[e] = e == at ? w : v[e];
                }
                if (sh.mask) {
#pragma unroll
                    for (int e = 0; e < per; ++e)
                        if (!((got.allowed[u] >> e) & 1u)) v[e] = -INFINITY;
                }
                float top = v[0];
#pragma unroll
                for (int e = 1; e < per; ++e) top = fmaxf(top, v[e]);
                if (top > best.v) {  // seldom, once some have been seen
                    int at = per - 1;
#pragma unroll
                    for (int e = per - 2; e >= 0; --e)
                        if (v[e] == top) at = e;
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
                    if ((touched >> e) & 1u) v = change(i + e, id + e, v);
                    if (sh.mask && !((sh.mask[(id + e) >> 5] >> ((id + e) & 31)) & 1u)) v = -INFINITY;
                    if (v > best.v) best = Best{v, id + e};
                    if (y) y[id + e] = from_f32<T>(v);
                }
            }
        }
        if (i0 + Batch<T, kVec>::kStep < n) {
            got.fetch(x, sh, a.vocab, s0 + i0 + Batch<T, kVec>::kStep);
            got.masks(sh, a.vocab, s0 + i0 + Batch<T, kVec>::kStep);
        }
    }
}

// The share with its touched ids in the hash table.
template <class T, bool kVec>
__device__ __forceinline__ Best share_hashed(const LogitsArgs& a, const Share& sh, Batch<T, kVec>& got, unsigned* s_table, unsigned* s_bits) {
    const T* x = reinterpret_cast<const T*>(a.x) + sh.row * a.x_stride;
    T* y = a.y ? reinterpret_cast<T*>(a.y) + sh.row * a.y_stride : nullptr;
    const bool few = sh.h1 > sh.h0 || sh.b1 > sh.b0;
    // Slots: twice the entries at least, a power of two.
    const int entries = sh.h1 - sh.h0 + sh.b1 - sh.b0;
    const int log_slots = min(13, max(9, 33 - __clz(entries | 1))), slots = 1 << log_slots;
    int* s_id = reinterpret_cast<int*>(s_table);
    unsigned* s_word = s_table + slots;
    Best best{-INFINITY, -1};
    got.masks(sh, a.vocab, threadIdx.x * Batch<T, kVec>::per);
    if (few) {
        int held[kLogitsHeld];
#pragma unroll
        for (int k = 0; k < kLogitsHeld; ++k) {
            const int i = sh.h0 + threadIdx.x + k * kLogitsThreads;
            held[k] = i < sh.h1 ? a.hist[i] : -1;
        }
        for (int i = threadIdx.x * 4; i < slots; i += kLogitsThreads * 4) {
            *reinterpret_cast<int4*>(s_id + i) = make_int4(-1, -1, -1, -1);
            *reinterpret_cast<uint4*>(s_word + i) = make_uint4(0, 0, 0, 0);
        }
        for (int i = threadIdx.x; i < sh.places / 32; i += kLogitsThreads) s_bits[i] = 0u;
        __syncthreads();
        // The id's slot, taken if it is new; negative if it is not the CTA's.
        // There are fewer entries than slots: the search ends.
        auto slot_of = [&](int id) {
            const int at = sh.place_of(id, a.vocab);
            if (at < 0) return -1;
            unsigned slot = ((unsigned)id * 2654435769u) >> (32 - log_slots);
#pragma unroll 1
            for (int tries = 0; tries < slots; ++tries) {
                const int had = atomicCAS(&s_id[slot], -1, id);
                if (had == -1) atomicOr(&s_bits[at >> 5], 1u << (at & 31));
                if (had == -1 || had == id) return (int)slot;
                slot = (slot + 1) & (slots - 1);
            }
            return -1;
        };
        if (sh.b1 > sh.b0) {
#pragma unroll 1
            for (int i = sh.b0 + threadIdx.x; i < sh.b1; i += kLogitsThreads) {
                const int slot = slot_of(a.bias_ids[i]);
                if (slot >= 0) atomicMax(&s_word[slot], ((unsigned)(i - sh.b0) + 1u) << 16);
            }
            __syncthreads();  // counts are added below the bias entries
        }
        auto count = [&](int id) {
            const int slot = slot_of(id);
            if (slot >= 0) atomicAdd(&s_word[slot], 1u);
        };
#pragma unroll 1
        for (int k = 0; k < kLogitsHeld; ++k) {
            int id = -1;
#pragma unroll
            for (int j = 0; j < kLogitsHeld; ++j) id = j == k ? held[j] : id;
            if (sh.h0 + threadIdx.x + k * kLogitsThreads < sh.h1) count(id);
        }
#pragma unroll 1
        for (int i = sh.h0 + threadIdx.x + kLogitsHeld * kLogitsThreads; i < sh.h1; i += kLogitsThreads) count(a.hist[i]);
        __syncthreads();
    }
    if (few) {
        const Penalties penalties(a, sh);
#pragma unroll 4
        for (int k = threadIdx.x; k < slots; k += kLogitsThreads) {
            const int id = s_id[k];
            if (id < 0) continue;
            const unsigned word = s_word[k];
            s_word[k] = __float_as_uint(penalties(to_f32<T>(x[id]), word & 0xffffu, (int)(word >> 16) - 1));
        }
        __syncthreads();
    }
    auto change = [&](int, int id, float) {
        unsigned slot = ((unsigned)id * 2654435769u) >> (32 - log_slots);
#pragma unroll 1
        for (int tries = 0; tries < slots && s_id[slot] != id; ++tries) slot = (slot + 1) & (slots - 1);
        return __uint_as_float(s_word[slot]);
    };
    stream<T, kVec>(a, sh, x, y, got, 0, sh.places, few ? s_bits : nullptr, change, best);
    return best;
}

// The share in slices whose ids have a count and a bias entry each.
template <class T, bool kVec>
__device__ __forceinline__ Best share_sliced(const LogitsArgs& a, const Share& sh, Batch<T, kVec>& got, unsigned* s_table, unsigned* s_bits) {
    const T* x = reinterpret_cast<const T*>(a.x) + sh.row * a.x_stride;
    T* y = a.y ? reinterpret_cast<T*>(a.y) + sh.row * a.y_stride : nullptr;
    unsigned *s_count = s_table, *s_entry = s_table + kTableSlots;
    const Penalties penalties(a, sh);
    auto change = [&](int place, int, float v) { return penalties(v, (int)s_count[place], (int)s_entry[place] - 1); };
    Best best{-INFINITY, -1};
    for (int s0 = 0; s0 < sh.places; s0 += kTableSlots) {
        const int n = min(kTableSlots, sh.places - s0);
        for (int i = threadIdx.x * 4; i < 2 * kTableSlots; i += kLogitsThreads * 4) *reinterpret_cast<uint4*>(s_table + i) = make_uint4(0, 0, 0, 0);
        for (int i = threadIdx.x; i < kTableSlots / 32; i += kLogitsThreads) s_bits[i] = 0u;
        __syncthreads();
        auto touch = [&](int id) {
            const int at = sh.place_of(id, a.vocab);
            if (at < s0 || at >= s0 + n) return -1;
            atomicOr(&s_bits[(at - s0) >> 5], 1u << ((at - s0) & 31));
            return at - s0;
        };
#pragma unroll 1
        for (int i = sh.b0 + threadIdx.x; i < sh.b1; i += kLogitsThreads) {
            const int at = touch(a.bias_ids[i]);
            if (at >= 0) atomicMax(&s_entry[at], (unsigned)(i - sh.b0) + 1u);
        }
#pragma unroll 1
        for (int i = sh.h0 + threadIdx.x; i < sh.h1; i += kLogitsThreads) {
            const int at = touch(a.hist[i]);
            if (at >= 0) atomicAdd(&s_count[at], 1u);
        }
        __syncthreads();
        got.fetch(x, sh, a.vocab, s0 + threadIdx.x * Batch<T, kVec>::per);
        got.masks(sh, a.vocab, s0 + threadIdx.x * Batch<T, kVec>::per);
        stream<T, kVec>(a, sh, x, y, got, s0, n, s_bits, change, best);
        __syncthreads();  // the words are used again
    }
    return best;
}

// 1 << log_width CTAs a row.
template <class T, bool kVec>
__global__ void __launch_bounds__(kLogitsThreads, 2) k_logits(const __grid_constant__ LogitsArgs a, int log_width) {
    extern __shared__ __align__(16) unsigned s_table[];
    unsigned* s_bits = s_table + 2 * kTableSlots;
    __shared__ Best s_best[kLogitsThreads / 32];
    __shared__ Best s_row[16];
    __shared__ __align__(8) uint64_t s_done;
    const int width = 1 << log_width, row = blockIdx.x >> log_width, part = blockIdx.x & (width - 1);
    const uint32_t done = (uint32_t)__cvta_generic_to_shared(&s_done);
    if (width > 1) {
        if (threadIdx.x == 0) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(done), "r"(width) : "memory");
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // waited for where the choice is joined
    }
    const int runs = (a.vocab + kLogitsRun - 1) / kLogitsRun;
    Share sh{row, part, log_width, (runs - part + width - 1) / width * kLogitsRun, 0, 0, 0, 0, nullptr};
    Batch<T, kVec> got;
    got.fetch(reinterpret_cast<const T*>(a.x) + row * a.x_stride, sh, a.vocab, threadIdx.x * Batch<T, kVec>::per);
    // Both bounds inside the list: what is added to them below stays below 2^31.
    if (a.hist) sh.h0 = min(max(a.hist_begin[row], 0), a.hist_len), sh.h1 = max(sh.h0, min(a.hist_end[row], a.hist_len));
    if (a.bias_ids) sh.b0 = min(max(a.bias_begin[row], 0), a.bias_len), sh.b1 = max(sh.b0, min(a.bias_end[row], a.bias_len));
    if (a.mask) {
        const int m = a.mask_row ? a.mask_row[row] : row;
        if (m >= 0 && m < a.mask_rows) sh.mask = a.mask + m * a.mask_stride;
    }
    const long long entries = (long long)(sh.h1 - sh.h0) + (sh.b1 - sh.b0);
    Best best = entries > 0 && (entries > kTableMost || sh.places > kShareMost) ? share_sliced<T, kVec>(a, sh, got, s_table, s_bits)
                                                                               : share_hashed<T, kVec>(a, sh, got, s_table, s_bits);
    best = warp_best(best);
    if ((threadIdx.x & 31) == 0) s_best[threadIdx.x >> 5] = best;
    __syncthreads();
    if (width > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all CTAs have begun
    if (!a.choice || threadIdx.x >= 32) return;
    best = warp_best(threadIdx.x < kLogitsThreads / 32 ? s_best[threadIdx.x] : Best{-INFINITY, -1});
    if (width > 1) {
        if (threadIdx.x == 0) {
            // Into the first CTA's memory; it alone stays until all have come.
            *cg::this_cluster().map_shared_rank(&s_row[part], 0) = best;
            uint32_t there;
            asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(there) : "r"(done));
            asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(there) : "memory");
        }
        if (part) return;
        bool ok = false;
#pragma unroll 1
        for (int left = 1 << 22; !ok && left > 0; --left) {
            uint32_t is;
            asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], 0;\n selp.u32 %0, 1, 0, p;\n}\n"
                         : "=r"(is)
                         : "r"(done)
                         : "memory");
            ok = is;
        }
        best = warp_best(ok && (int)threadIdx.x < width ? s_row[threadIdx.x] : Best{-INFINITY, -1});
    }
    if (threadIdx.x == 0) a.choice[row] = best.i;
}

template <class T, bool kVec>
cudaError_t logits_launch(const LogitsArgs& a, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    auto* kernel = k_logits<T, kVec>;
    cudaError_t e = allow_smem(kernel, kTableBytes + kShareMost / 8, &done, true);
    if (e != cudaSuccess) return e;
    const int runs = (a.vocab + kLogitsRun - 1) / kLogitsRun;
    int log_width = 0;
    while (log_width < 4 && (a.rows << (log_width + 1)) <= 256 && (2 << log_width) <= runs) ++log_width;
    const int width = 1 << log_width, places = (runs + width - 1) / width * kLogitsRun;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(a.rows * width);
    c.blockDim = dim3(kLogitsThreads);
    c.dynamicSmemBytes = a.hist || a.bias_ids ? kTableBytes + std::min(std::max(places, kTableSlots), kShareMost) / 8 : 0;
    c.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)width, 1, 1};
    c.attrs = at;
    c.numAttrs = width > 1 ? 1 : 0;
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
