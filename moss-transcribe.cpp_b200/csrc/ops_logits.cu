// mtb_logits_process: penalties for repeated tokens, biases and grammar masks
// on logits rows, with the greedy choice.
//
// Bound: bytes (each logit read and written once); one row of 152 k values: latency (7.5 us).
// 256 f32 rows, half of the ids masked: 55 us without lists (5.7 TB/s, a plain copy 49 us), 85 us
// with 4096 ids of history and 300 biases a row (3.7 TB/s): a CTA forms its lists before its stream starts.
// A row belongs to 1 to 16 CTAs, as many as fill the SMs (one from 129 rows on: two
// CTAs to an SM, each a row; clusters of more take longer to place than they save).
// The vocabulary goes round a row's CTAs in runs of 1024 ids, since histories crowd at
// low ids.  What touches few ids is set apart: a bitmap in shared memory says which of the
// CTA's ids are in the row's history or biases; an id's rank among them (the bits before its
// word, summed once, and those before it in the word) is its place in a list of words, with its count (low
// half) and last bias entry + 1 (high half), and in a list of its new value.  The logits
// stream through once: masked ones to -inf, those of the bitmap from the list (writing them behind the
// stream instead cost 256 rows with 4096 ids of history 35 us in sectors written twice,
// penalties within the stream as much in divergence, a hash table's search there 10 us).
// Lists of more than 6144 entries, or shares of more than 262144 ids, which do not fit beside
// one another at two CTAs to an SM, go in slices of 8192 ids with two words each instead, and each
// slice goes through the lists: 256 rows of 151936 ids 86 us with 6144 entries, 153 with 6145 (8 rows 19 and
// 16: 16 CTAs a row, one or two slices each); 130 rows of 262144 ids 64 us, of 262145 198.  The row's choice joins the CTAs' in the first one's shared
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
constexpr int kTableSlots = 8192;         // ids of a slice, two words each
constexpr int kTableMost = 6144;          // entries of history and biases that the lists by rank take
constexpr int kShareMost = 32768 * 8;     // ids of the bitmap
constexpr int kTableBytes = kTableSlots * 8;
static_assert(kTableMost * 8 + kShareMost / 32 * 2 <= kTableBytes, "words, values and the words' sums of bits in a slice's place");
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
// places, or null), as `change` of a value or `patch` of a vector has them; masks; the
// choice.  `got` holds the first batch.
template <class T, bool kVec, class F, class G>
__device__ __forceinline__ void stream(const LogitsArgs& a, const Share& sh, const T* x, T* y, Batch<T, kVec>& got, int s0, int n,
                                       const unsigned* s_bits, F&& change, G&& patch, Best& best) {
    constexpr int per = Batch<T, kVec>::per;
#pragma unroll 1
    for (int i0 = threadIdx.x * per; i0 < n; i0 += Batch<T, kVec>::kStep) {
#pragma unroll
        for (int u = 0; u < kLogitsBatch; ++u) {
            const int i = i0 + u * kLogitsThreads * per, id = sh.id_of(s0 + i);
            if (i >= n || id >= a.vocab) break;
            const unsigned word = s_bits ? s_bits[i >> 5] : 0u, touched = word >> (i & 31);
            if (id + per <= a.vocab) {
                const T* t = reinterpret_cast<const T*>(&got.raw[u]);
                float v[per];
#pragma unroll
                for (int e = 0; e < per; ++e) v[e] = to_f32<T>(t[e]);
                const unsigned hit = touched & got.allowed[u] & ((1u << per) - 1);
                if (hit) patch(v, word, hit, i, id);
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

// The share with its touched ids in lists by their rank.
template <class T, bool kVec>
__device__ __forceinline__ Best share_ranked(const LogitsArgs& a, const Share& sh, Batch<T, kVec>& got, unsigned* s_table, unsigned* s_bits) {
    __shared__ int s_warp[kLogitsThreads / 32];
    constexpr int per = Batch<T, kVec>::per;
    const T* x = reinterpret_cast<const T*>(a.x) + sh.row * a.x_stride;
    T* y = a.y ? reinterpret_cast<T*>(a.y) + sh.row * a.y_stride : nullptr;
    const bool few = sh.h1 > sh.h0 || sh.b1 > sh.b0;
    unsigned* s_word = s_table;
    float* s_value = reinterpret_cast<float*>(s_table + kTableMost);
    uint16_t* s_before = reinterpret_cast<uint16_t*>(s_table + 2 * kTableMost);
    auto rank = [&](int place) { return s_before[place >> 5] + __popc(s_bits[place >> 5] & ((1u << (place & 31)) - 1)); };
    Best best{-INFINITY, -1};
    got.masks(sh, a.vocab, threadIdx.x * per);
    if (few) {
        int at[kLogitsHeld];  // places of the first ids, negative: not the CTA's
        float value[kLogitsHeld];
#pragma unroll
        for (int k = 0; k < kLogitsHeld; ++k) {
            const int i = sh.h0 + threadIdx.x + k * kLogitsThreads;
            at[k] = i < sh.h1 ? a.hist[i] : -1;
        }
        const int entries = sh.h1 - sh.h0 + sh.b1 - sh.b0, words = sh.places / 32;
        for (int i = threadIdx.x; i < entries; i += kLogitsThreads) s_word[i] = 0u;
        for (int i = threadIdx.x; i < words; i += kLogitsThreads) s_bits[i] = 0u;
#pragma unroll
        for (int k = 0; k < kLogitsHeld; ++k) {
            const int id = at[k];
            at[k] = sh.place_of(id, a.vocab);
            value[k] = at[k] >= 0 ? to_f32<T>(x[id]) : 0.f;
        }
        __syncthreads();
        // Entries behind those that the thread holds, and the biases.
        const int h_rest = sh.h0 + kLogitsHeld * kLogitsThreads;
        auto mark = [&](int place) {
            if (place >= 0) atomicOr(&s_bits[place >> 5], 1u << (place & 31));
        };
#pragma unroll
        for (int k = 0; k < kLogitsHeld; ++k) mark(at[k]);
#pragma unroll 1
        for (int i = h_rest + threadIdx.x; i < sh.h1; i += kLogitsThreads) mark(sh.place_of(a.hist[i], a.vocab));
#pragma unroll 1
        for (int i = sh.b0 + threadIdx.x; i < sh.b1; i += kLogitsThreads) mark(sh.place_of(a.bias_ids[i], a.vocab));
        __syncthreads();
        // Bits before each word: a thread has consecutive words, an odd number (no two lanes of a warp on one bank).
        const int each = (words / kLogitsThreads + 1) | 1;
        const int w0 = min(words, (int)threadIdx.x * each), w1 = min(words, w0 + each), lane = threadIdx.x & 31;
        int sum = 0;
#pragma unroll 1
        for (int i = w0; i < w1; ++i) sum += __popc(s_bits[i]);
        int upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int z = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += z;
        }
        if (lane == 31) s_warp[threadIdx.x >> 5] = upto;
        __syncthreads();
        int before = upto - sum;
#pragma unroll
        for (int w = 0; w < kLogitsThreads / 32; ++w)
            if (w < (int)(threadIdx.x >> 5)) before += s_warp[w];
#pragma unroll 1
        for (int i = w0; i < w1; ++i) {
            s_before[i] = (uint16_t)before;
            before += __popc(s_bits[i]);
        }
        __syncthreads();
        if (sh.b1 > sh.b0) {
#pragma unroll 1
            for (int i = sh.b0 + threadIdx.x; i < sh.b1; i += kLogitsThreads) {
                const int place = sh.place_of(a.bias_ids[i], a.vocab);
                if (place >= 0) atomicMax(&s_word[rank(place)], ((unsigned)(i - sh.b0) + 1u) << 16);
            }
            __syncthreads();  // counts are added below the bias entries
        }
#pragma unroll
        for (int k = 0; k < kLogitsHeld; ++k)
            if (at[k] >= 0) atomicAdd(&s_word[rank(at[k])], 1u);
#pragma unroll 1
        for (int i = h_rest + threadIdx.x; i < sh.h1; i += kLogitsThreads) {
            const int place = sh.place_of(a.hist[i], a.vocab);
            if (place >= 0) atomicAdd(&s_word[rank(place)], 1u);
        }
        __syncthreads();
        // The new values; an id that occurs several times gets the same one each time.
        const Penalties penalties(a, sh);
        auto renew = [&](int place, float v) {
            if (place < 0) return;
            const int r = rank(place);
            s_value[r] = penalties(v, s_word[r] & 0xffffu, (int)(s_word[r] >> 16) - 1);
        };
#pragma unroll 1
        for (int k = 0; k < kLogitsHeld && k * kLogitsThreads < sh.h1 - sh.h0; ++k) {
            int place = -1;
            float v = 0.f;
#pragma unroll
            for (int j = 0; j < kLogitsHeld; ++j)
                if (j == k) place = at[j], v = value[j];
            renew(place, v);
        }
#pragma unroll 1
        for (int i = h_rest + threadIdx.x; i < sh.h1; i += kLogitsThreads) {
            const int id = a.hist[i], place = sh.place_of(id, a.vocab);
            if (place >= 0) renew(place, to_f32<T>(x[id]));
        }
#pragma unroll 1
        for (int i = sh.b0 + threadIdx.x; i < sh.b1; i += kLogitsThreads) {
            const int id = a.bias_ids[i], place = sh.place_of(id, a.vocab);
            if (place >= 0) renew(place, to_f32<T>(x[id]));
        }
        __syncthreads();
    }
    auto change = [&](int place, int, float) { return s_value[rank(place)]; };
    auto patch = [&](float (&v)[per], unsigned word, unsigned hit, int place, int) {
        const int first = s_before[place >> 5] + __popc(word & ((1u << (place & 31)) - 1));
        const unsigned touched = word >> (place & 31);
#pragma unroll
        for (int e = 0; e < per; ++e)
            if ((hit >> e) & 1u) v[e] = s_value[first + __popc(touched & ((1u << e) - 1))];
    };
    stream<T, kVec>(a, sh, x, y, got, 0, sh.places, few ? s_bits : nullptr, change, patch, best);
    return best;
}

// The share in slices whose ids have a count and a bias entry each.
template <class T, bool kVec>
__device__ __forceinline__ Best share_sliced(const LogitsArgs& a, const Share& sh, Batch<T, kVec>& got, unsigned* s_table, unsigned* s_bits) {
    const T* x = reinterpret_cast<const T*>(a.x) + sh.row * a.x_stride;
    T* y = a.y ? reinterpret_cast<T*>(a.y) + sh.row * a.y_stride : nullptr;
    unsigned *s_count = s_table, *s_entry = s_table + kTableSlots;
    const Penalties penalties(a, sh);
    constexpr int per = Batch<T, kVec>::per;
    auto change = [&](int place, int, float v) { return penalties(v, (int)s_count[place], (int)s_entry[place] - 1); };
    auto patch = [&](float (&v)[per], unsigned, unsigned hit, int place, int id) {
#pragma unroll 1
        for (; hit; hit &= hit - 1) {
            const int at = __ffs(hit) - 1;
            float w = v[0];
#pragma unroll
            for (int e = 1; e < per; ++e) w = e == at ? v[e] : w;
            w = change(place + at, id + at, w);
#pragma unroll
            for (int e = 0; e < per; ++e) v[e] = e == at ? w : v[e];
        }
    };
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
        stream<T, kVec>(a, sh, x, y, got, s0, n, s_bits, change, patch, best);
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
    const int width = 1 << log_width, row = blockIdx.x >> log_width, part = blockIdx.x & (width - 1);
    if (width > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // waited for where the choice is joined
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
                                                                               : share_ranked<T, kVec>(a, sh, got, s_table, s_bits);
    best = warp_best(best);
    if ((threadIdx.x & 31) == 0) s_best[threadIdx.x >> 5] = best;
    __syncthreads();
    if (width > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all CTAs have begun
    if (!a.choice) return;
    if (threadIdx.x < 32) {
        best = warp_best(threadIdx.x < kLogitsThreads / 32 ? s_best[threadIdx.x] : Best{-INFINITY, -1});
        // Into the first CTA's memory, which stays until all have come.
        if (width > 1 && threadIdx.x == 0) *cg::this_cluster().map_shared_rank(&s_row[part], 0) = best;
        __syncwarp();
    }
    if (width > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (part || threadIdx.x >= 32) return;
        best = warp_best((int)threadIdx.x < width ? s_row[threadIdx.x] : Best{-INFINITY, -1});
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
