// Rotary positions with the append to a paged cache, and eviction from it.
#include "ops_common.cuh"

#include <algorithm>
#include <climits>
#include <cooperative_groups.h>
#include <cstdint>

namespace mtb {
namespace {

using namespace ops;
namespace cg = cooperative_groups;

// ---- mtb_rope_append ----------------------------------------------------------------------------------------------
//
// Per token: (a, b) -> (a c - b s, b c + a s) for each pair, c and s of
// position * inv_freq[pair].  Far positions lose that angle in f32 (a position
// of 10^6 leaves an error of 0.06), so it is formed and reduced to [-pi, pi] in
// f64; its sine and cosine are f32 (the results have 16 bits).  They depend on
// the token alone, so a CTA forms them once in shared memory for all heads.
// Bound: bytes (q, k, v read and written once): 9730 f32 tokens of 16 + 2 x 8 heads of 128 into
// f16 take 45 us (5.3 TB/s), bf16 ones into bf16 32 us (5.0 TB/s), with position and weight 32.5; a step's few tokens:
// latency (3.4 us).  Half pairs of dims that are no multiple of 16, or other alignments, go a pair or a dim a thread
// with 2-byte accesses: the bf16 tokens take 125 us with 90 dims rotated, 49 with 96.

constexpr int kRopeThreads = 256;
constexpr int kRopeTokens = 4;  // tokens a CTA at most

struct RopeToken {
    int seq, slot, page, position;
};

__device__ __forceinline__ void angle(const RopeArgs& a, int position, int j, float* c, float* s) {
    const double t = (double)position * a.inv_freq[j];
    const double n = rint(t * 0.15915494309189533577);
    double r = fma(-n, 6.283185307179586232, t);
    r = fma(-n, 2.4492935982947064e-16, r);
    float si, co;
    sincosf((float)r, &si, &co);
    *c = co * a.factor;
    *s = si * a.factor;
}

template <class I, class O, bool kVec>
__global__ void __launch_bounds__(kRopeThreads) k_rope_append(RopeArgs a, int per_cta) {
    __shared__ float s_cos[kRopeTokens][64], s_sin[kRopeTokens][64];
    __shared__ RopeToken s_tok[kRopeTokens];
    const PagedView& c = a.c;
    const int t0 = blockIdx.x * per_cta;
    const int half = a.rotary / 2;
    if (threadIdx.x < per_cta) {
        const int t = t0 + threadIdx.x;
        RopeToken r{-1, -1, -1, 0};
        if (t < a.n_tokens) r.seq = seq_of_token(a.cu, c.n_seq, t);
        if (r.seq >= 0) {
            r.position = a.positions[t];
            const int2 tok = seq_tokens(c, a.cu, a.n_tokens, r.seq);
            if (t - tok.x >= tok.y) {  // a bad pair of bounds: not this sequence's token
                r.seq = -1;
            } else {
                const int len = seq_len(c, r.seq);
                r.slot = len - tok.y + (t - tok.x);
                if (r.slot < 0) flag(c, BAD_LEN);
                else r.page = page_of(c, r.seq, r.slot / kPage);
            }
        }
        s_tok[threadIdx.x] = r;
    }
    // Bounds that do not ascend are reported for every sequence, also where no token finds it.
    if (blockIdx.x == 0)
        for (int s = kRopeThreads - 1 - threadIdx.x; s < c.n_seq; s += kRopeThreads) seq_tokens(c, a.cu, a.n_tokens, s);
    for (int i = threadIdx.x; i < per_cta * half; i += kRopeThreads) {
        const int t = t0 + i / half, j = i % half;
        if (t < a.n_tokens) angle(a, a.positions[t], j, &s_cos[i / half][j], &s_sin[i / half][j]);
    }
    __syncthreads();
    const int D = c.head_dim, R = a.rotary;
    const int heads = a.n_heads + 2 * c.n_kv;
    for (int u = 0; u < per_cta; ++u) {
        const RopeToken r = s_tok[u];
        if (r.seq < 0) continue;
        const int t = t0 + u;
        // Source and destination of one head of q, k, v; no destination: nullptr.
        auto place = [&](int h, const I** src, O** dst, bool* turn) {
            if (h < a.n_heads) {
                *src = reinterpret_cast<const I*>(a.q) + t * a.q_stride + (long long)h * D;
                *dst = reinterpret_cast<O*>(a.out) + t * a.out_stride + (long long)h * D;
                *turn = true;
                return;
            }
            const bool is_k = h < a.n_heads + c.n_kv;
            const int g = h - a.n_heads - (is_k ? 0 : c.n_kv);
            *src = is_k ? reinterpret_cast<const I*>(a.k) + t * a.k_stride + (long long)g * D
                        : reinterpret_cast<const I*>(a.v) + t * a.v_stride + (long long)g * D;
            *turn = is_k;
            *dst = r.page < 0 ? nullptr
                              : reinterpret_cast<O*>(is_k ? c.k : c.v) + r.page * c.page_stride + g * c.head_stride +
                                    (long long)(r.slot % kPage) * D;
        };
        const float *co = s_cos[u], *si = s_sin[u];
        if (kVec) {
            // Items of 8 dims; in the half layout an item of the first half of
            // the rotated dims takes its partner 8 along.
            const int chunks = D / 8, pairs = a.interleaved ? 0 : R / 16, items = chunks - pairs;
            for (int i = threadIdx.x; i < heads * items; i += kRopeThreads) {
                const int h = i / items;
                int ch = i % items;
                const I* src;
                O* dst;
                bool turn;
                place(h, &src, &dst, &turn);
                if (!dst) continue;
                float x[8], y[8];
                if (!a.interleaved && ch < pairs) {
                    float z[8];
                    load_vec<I, 8>(src + ch * 8, x);
                    load_vec<I, 8>(src + ch * 8 + R / 2, z);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float cc = turn ? co[ch * 8 + e] : 1.f, ss = turn ? si[ch * 8 + e] : 0.f;
                        y[e] = turn ? __fsub_rn(x[e] * cc, z[e] * ss) : x[e];
                        z[e] = turn ? __fadd_rn(z[e] * cc, x[e] * ss) : z[e];
                    }
                    store_vec<O, 8>(dst + ch * 8, y);
                    store_vec<O, 8>(dst + ch * 8 + R / 2, z);
                    continue;
                }
                if (ch >= pairs) ch += pairs;  // dims behind the rotated ones
                load_vec<I, 8>(src + ch * 8, x);
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const bool on = turn && a.interleaved && ch * 8 + e < R;
                    const int j = on ? (ch * 8 + e) / 2 : 0;
                    y[e] = on ? __fsub_rn(x[e] * co[j], x[e + 1] * si[j]) : x[e];
                    y[e + 1] = on ? __fadd_rn(x[e + 1] * co[j], x[e] * si[j]) : x[e + 1];
                }
                store_vec<O, 8>(dst + ch * 8, y);
            }
        } else {
            // Any alignment, any even R: an item is a pair, or one dim that passes.
            const int items = half + D - R;
            for (int i = threadIdx.x; i < heads * items; i += kRopeThreads) {
                const int h = i / items, j = i % items;
                const I* src;
                O* dst;
                bool turn;
                place(h, &src, &dst, &turn);
                if (!dst) continue;
                if (j >= half) {
                    dst[R + j - half] = from_f32<O>(to_f32<I>(src[R + j - half]));
                    continue;
                }
                const int d0 = a.interleaved ? 2 * j : j, d1 = a.interleaved ? d0 + 1 : j + half;
                const float x = to_f32<I>(src[d0]), z = to_f32<I>(src[d1]);
                dst[d0] = from_f32<O>(turn ? __fsub_rn(x * co[j], z * si[j]) : x);
                dst[d1] = from_f32<O>(turn ? __fadd_rn(z * co[j], x * si[j]) : z);
            }
        }
        if (r.page >= 0)
            for (int g = threadIdx.x; g < c.n_kv; g += kRopeThreads) {
                const long long at = ((long long)r.page * c.n_kv + g) * kPage + r.slot % kPage;
                if (c.position) c.position[at] = r.position;
                if (c.weight) c.weight[at] = 0.f;
            }
    }
}

template <class I, class O>
cudaError_t rope_typed(const RopeArgs& a, cudaStream_t s) {
    // One token a CTA until the GPU's 148 SMs have two each: few tokens then spread over more
    // SMs; beyond that four share the CTA's start and its angles' threads.
    const int per = a.n_tokens < 2 * 148 ? 1 : kRopeTokens;
    const int in16 = 16 / (int)sizeof(I);
    auto ok = [](const void* p, long long stride, int per16) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % per16 == 0;
    };
    const bool vec = ok(a.q, a.q_stride, in16) && ok(a.k, a.k_stride, in16) && ok(a.v, a.v_stride, in16) &&
                     ok(a.out, a.out_stride, 8) && (a.interleaved || a.rotary % 16 == 0);
    const int grid = (a.n_tokens + per - 1) / per;
    if (vec) k_rope_append<I, O, true><<<grid, kRopeThreads, 0, s>>>(a, per);
    else k_rope_append<I, O, false><<<grid, kRopeThreads, 0, s>>>(a, per);
    return cudaGetLastError();
}

// ---- mtb_cache_evict ----------------------------------------------------------------------------------------------
//
// Two kernels.  The first, one cluster per (sequence, KV head): each slot's rank
// as a 32-bit key (protected: all ones; else the weight's bits in ascending
// order; NaN 0), the keep-th largest key by three passes of 11, 11 and 10 bits,
// and lists of the gaps below `keep` and of the kept slots behind it, as rows of the pool.  Ties at
// the threshold go to the lowest slots.  k_evict_rank_regs holds eight slots a
// thread in registers, in as many CTAs as that takes (four SMs for a half-hour
// recording); k_evict_rank, one CTA, takes longer lists and books that are not 16-byte
// aligned.  The second, k_evict_move, copies the listed rows:
// sources lie at or behind `keep`, gaps below it, so no row is both and the
// copies need no order.  Bound: the ranking by latency (three histograms, one after the other: 13 us for one CTA
// a list, 23 us for clusters of four), the copies by bytes in rows of 256 (four recordings of 25000
// cut to 8192: some 180 MB in 42 us, 4.3 TB/s; four rows of a warp in flight and as many CTAs as rows
// want rather than one wave: 72.1 -> 69.5 us in all).

constexpr int kRankThreads = 1024;
constexpr int kRankBins = 2048;
constexpr int kRankKeys = 40960;  // keys kept in shared memory (160 KB); more are formed again in each pass

struct EvictHead {
    int moves, new_len;
};

__device__ __forceinline__ unsigned weight_key(float w) {
    if (isnan(w)) return 0u;
    const unsigned b = __float_as_uint(w + 0.f);  // -0 ranks as 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Exclusive sum over the CTA; *total: the sum of all.
__device__ __forceinline__ int block_scan(int v, int* s_warp, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int y = lane < (int)(blockDim.x >> 5) ? s_warp[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int z = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) y += z;
        }
        s_warp[lane] = y;
    }
    __syncthreads();
    *total = s_warp[(blockDim.x >> 5) - 1];
    const int before = (warp ? s_warp[warp - 1] : 0) + x - v;
    __syncthreads();
    return before;
}

__device__ __forceinline__ int block_max(int v, int* s_warp) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s_warp[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    return v;
}

__global__ void __launch_bounds__(kRankThreads) k_evict_rank(EvictArgs a) {
    extern __shared__ unsigned s_key[];
    __shared__ int s_hist[kRankBins];
    __shared__ int s_warp[32];
    __shared__ int s_pick, s_left, s_bad;
    const PagedView& c = a.c;
    const int seq = blockIdx.x / c.n_kv, h = blockIdx.x % c.n_kv;
    char* ws = a.workspace + evict_workspace(1, 1, c.table_stride) * blockIdx.x;
    EvictHead* head = reinterpret_cast<EvictHead*>(ws);
    int* to = reinterpret_cast<int*>(ws + 256);
    int* from = to + c.table_stride * (kPage / 2);
    const int n = seq_len(c, seq);
    if (threadIdx.x == 0) s_bad = 0;
    __syncthreads();
    if (n > a.keep)
        for (int p = threadIdx.x; p < (n + kPage - 1) / kPage; p += kRankThreads)
            if (page_of(c, seq, p) < 0) s_bad = 1;
    __syncthreads();
    if (n <= a.keep || s_bad) {
        if (threadIdx.x == 0) *head = EvictHead{0, n};
        return;
    }
    const int* table = c.table + (long long)seq * c.table_stride;
    auto at = [&](int i) { return ((long long)table[i / kPage] * c.n_kv + h) * kPage + i % kPage; };
    int newest = INT_MIN;
    for (int i = threadIdx.x; i < n; i += kRankThreads) newest = max(newest, c.position[at(i)]);
    newest = block_max(newest, s_warp);
    auto form = [&](int i) -> unsigned {
        const long long m = at(i);
        const int p = c.position[m];
        if (p < a.sinks || (long long)p > (long long)newest - a.recent) return 0xffffffffu;
        return weight_key(c.weight[m]);
    };
    const bool held = n <= kRankKeys;
    if (held)
        for (int i = threadIdx.x; i < n; i += kRankThreads) s_key[i] = form(i);
    auto key = [&](int i) { return held ? s_key[i] : form(i); };
    // The keep-th largest key: `prefix` its leading bits so far, `left` how
    // many of the keys with that prefix are still to be taken.
    unsigned prefix = 0, known = 0;
    int left = a.keep;
    for (int pass = 0; pass < 3 && left > 0; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const int bins = pass == 2 ? 1024 : 2048;
        for (int i = threadIdx.x; i < kRankBins; i += kRankThreads) s_hist[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kRankThreads) {
            const unsigned k = key(i);
            if ((k & known) == prefix) atomicAdd(&s_hist[(k >> shift) & (bins - 1)], 1);
        }
        __syncthreads();
        // Bins from the top: thread t has bins 2047 - 2t and 2046 - 2t.
        const int b1 = kRankBins - 1 - 2 * threadIdx.x;
        const int c1 = s_hist[b1], c0 = s_hist[b1 - 1];
        int total;
        const int before = block_scan(c1 + c0, s_warp, &total);
        if (before < left && left <= before + c1) {
            s_pick = b1;
            s_left = left - before;
        } else if (before + c1 < left && left <= before + c1 + c0) {
            s_pick = b1 - 1;
            s_left = left - before - c1;
        }
        __syncthreads();
        prefix |= (unsigned)s_pick << shift;
        known |= (unsigned)(bins - 1) << shift;
        left = s_left;
        __syncthreads();
    }
    // keep == 0: nothing stays.  Else keys above prefix stay, and the first
    // `left` of those equal to it, in slot order.  A thread has consecutive
    // slots, an odd number of them (no two lanes of a warp on one bank).
    const int per = (n + kRankThreads - 1) / kRankThreads | 1;
    const int lo = min(n, (int)threadIdx.x * per), hi = min(n, lo + per);
    int ties = 0;
    for (int i = lo; i < hi; ++i) ties += key(i) == prefix;
    int total;
    int tie = block_scan(ties, s_warp, &total);
    const int tie0 = tie;
    auto stays = [&](int i) {
        const unsigned k = key(i);
        return a.keep > 0 && (k > prefix || (k == prefix && tie++ < left));
    };
    int gaps = 0, come = 0;
    for (int i = lo; i < hi; ++i) {
        const bool st = stays(i);
        gaps += !st && i < a.keep;
        come += st && i >= a.keep;
    }
    int moves, same;
    int g = block_scan(gaps, s_warp, &moves);
    int f = block_scan(come, s_warp, &same);
    tie = tie0;
    for (int i = lo; i < hi; ++i) {
        const bool st = stays(i);
        const int row = table[i / kPage] * kPage + i % kPage;
        if (!st && i < a.keep) to[g++] = row;
        if (st && i >= a.keep) from[f++] = row;
    }
    if (threadIdx.x == 0) *head = EvictHead{min(moves, same), a.keep};
}

// Eight slots a thread.  What the cluster's CTAs tell one another (histograms,
// counts) they read from one another's shared memory, behind cluster barriers.
constexpr int kRankEach = 8;
constexpr int kRankCopies = 4;  // of the histogram, by lane: neighbours' weights fall into the same few bins

struct RankShared {
    int hist[kRankCopies][kRankBins];
    int warp[32];
    int sums[kRankBins];
    int newest, bad, ties, gaps, come, pick, left, count;
};

__global__ void __launch_bounds__(kRankThreads) k_evict_rank_regs(EvictArgs a, int width) {
    __shared__ __align__(16) RankShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const PagedView& c = a.c;
    const int list = blockIdx.x / width, part = blockIdx.x % width, seq = list / c.n_kv, h = list % c.n_kv;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    char* ws = a.workspace + evict_workspace(1, 1, c.table_stride) * list;
    EvictHead* head = reinterpret_cast<EvictHead*>(ws);
    int* to = reinterpret_cast<int*>(ws + 256);
    int* from = to + c.table_stride * (kPage / 2);
    const int n = seq_len(c, seq);
    if (n <= a.keep) {
        if (part == 0 && threadIdx.x == 0) *head = EvictHead{0, n};
        return;  // the whole cluster
    }
    const int i0 = (part * kRankThreads + threadIdx.x) * kRankEach;
    const int mine = min(max(n - i0, 0), kRankEach);
    int pos[kRankEach];
    unsigned key[kRankEach];
    int newest = INT_MIN, row0 = 0;  // row0: the first slot's row of the pool
    if (threadIdx.x == 0) sh.bad = 0;
    __syncthreads();
    if (mine > 0) {
        const int page = page_of(c, seq, i0 / kPage);
        row0 = page * kPage + i0 % kPage;
        if (page < 0) {
            sh.bad = 1;
        } else {
            const long long at = ((long long)page * c.n_kv + h) * kPage + i0 % kPage;
            const int4 p0 = *reinterpret_cast<const int4*>(c.position + at), p1 = *reinterpret_cast<const int4*>(c.position + at + 4);
            const float4 w0 = *reinterpret_cast<const float4*>(c.weight + at), w1 = *reinterpret_cast<const float4*>(c.weight + at + 4);
            pos[0] = p0.x, pos[1] = p0.y, pos[2] = p0.z, pos[3] = p0.w, pos[4] = p1.x, pos[5] = p1.y, pos[6] = p1.z, pos[7] = p1.w;
            const float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int e = 0; e < kRankEach; ++e) {
                key[e] = weight_key(w[e]);
                if (e < mine) newest = max(newest, pos[e]);
            }
        }
    }
    newest = block_max(newest, sh.warp);
    if (threadIdx.x == 0) sh.newest = newest;
    cluster.sync();
    int bad = 0;
    for (int r = 0; r < width; ++r) {
        const RankShared* o = cluster.map_shared_rank(&sh, r);
        newest = max(newest, o->newest);
        bad |= o->bad;
    }
    if (bad) {  // the same in all CTAs; a last barrier, for they read one another's
        if (part == 0 && threadIdx.x == 0) *head = EvictHead{0, n};
        cluster.sync();
        return;
    }
#pragma unroll
    for (int e = 0; e < kRankEach; ++e)
        if (e < mine && (pos[e] < a.sinks || (long long)pos[e] > (long long)newest - a.recent)) key[e] = 0xffffffffu;
    unsigned prefix = 0, known = 0;
    int left = a.keep;
    for (int pass = 0; pass < 3 && a.keep > 0; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
        for (int i = threadIdx.x; i < kRankCopies * kRankBins; i += kRankThreads) (&sh.hist[0][0])[i] = 0;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kRankEach; ++e)
            if (e < mine && (key[e] & known) == prefix) atomicAdd(&sh.hist[threadIdx.x % kRankCopies][(key[e] >> shift) & (bins - 1)], 1);
        __syncthreads();
        // Bins from the top: thread t has bins 2047 - 2t and 2046 - 2t; of its CTA, then of all.
        const int b1 = kRankBins - 1 - 2 * threadIdx.x;
        int c1 = 0, c0 = 0;
#pragma unroll
        for (int k = 0; k < kRankCopies; ++k) {
            const int2 x = *reinterpret_cast<const int2*>(&sh.hist[k][b1 - 1]);
            c0 += x.x;
            c1 += x.y;
        }
        if (width > 1) {
            *reinterpret_cast<int2*>(&sh.sums[b1 - 1]) = make_int2(c0, c1);
            cluster.sync();
            c0 = c1 = 0;
#pragma unroll 4
            for (int r = 0; r < width; ++r) {
                const int2 x = *reinterpret_cast<const int2*>(&cluster.map_shared_rank(&sh, r)->sums[b1 - 1]);
                c0 += x.x;
                c1 += x.y;
            }
        }
        int total;
        const int before = block_scan(c1 + c0, sh.warp, &total);
        if (before < left && left <= before + c1) {
            sh.pick = b1;
            sh.left = left - before;
            sh.count = c1;
        } else if (before + c1 < left && left <= before + c1 + c0) {
            sh.pick = b1 - 1;
            sh.left = left - before - c1;
            sh.count = c0;
        }
        if (width > 1) cluster.sync();  // the sums may be written again, the pick be read
        else __syncthreads();
        prefix |= (unsigned)sh.pick << shift;
        known |= (unsigned)(bins - 1) << shift;
        left = sh.left;
        if (left == sh.count) break;  // all of the bin's keys stay: their other bits do not matter
    }
    // Keys above prefix stay, and the first `left` of those equal to it, as far as it is known.
    int ties = 0, total;
#pragma unroll
    for (int e = 0; e < kRankEach; ++e) {
        key[e] &= known;
        ties += e < mine && key[e] == prefix;
    }
    int tie = block_scan(ties, sh.warp, &total);
    if (threadIdx.x == 0) sh.ties = total;
    cluster.sync();
    for (int r = 0; r < part; ++r) tie += cluster.map_shared_rank(&sh, r)->ties;
    unsigned stays = 0;
    int gaps = 0, come = 0;
#pragma unroll
    for (int e = 0; e < kRankEach; ++e) {
        const bool st = e < mine && a.keep > 0 && (key[e] > prefix || (key[e] == prefix && tie++ < left));
        stays |= (unsigned)st << e;
        gaps += e < mine && !st && i0 + e < a.keep;
        come += st && i0 + e >= a.keep;
    }
    int gap_total, come_total;
    int g = block_scan(gaps, sh.warp, &gap_total);
    int f = block_scan(come, sh.warp, &come_total);
    if (threadIdx.x == 0) {
        sh.gaps = gap_total;
        sh.come = come_total;
    }
    cluster.sync();
    int moves = 0;
    for (int r = 0; r < width; ++r) {
        const RankShared* o = cluster.map_shared_rank(&sh, r);
        if (r < part) {
            g += o->gaps;
            f += o->come;
        }
        moves += o->gaps;
    }
#pragma unroll
    for (int e = 0; e < kRankEach; ++e) {
        const bool st = (stays >> e) & 1;
        if (e < mine && !st && i0 + e < a.keep) to[g++] = row0 + e;
        if (st && i0 + e >= a.keep) from[f++] = row0 + e;
    }
    if (part == 0 && threadIdx.x == 0) *head = EvictHead{moves, a.keep};
    cluster.sync();  // nobody leaves while its counts are read
}

constexpr int kMoveThreads = 256;
constexpr int kMoveBatch = 4;  // rows of a warp in flight

__global__ void __launch_bounds__(kMoveThreads) k_evict_move(EvictArgs a, int lists) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // launched while the ranking still runs
    const PagedView& c = a.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per_row = c.head_dim / 8;  // 16-byte pieces of a K or V row
    char* base = lane < per_row ? c.k : c.v;
    const int piece = 16 * (lane % per_row);
    for (int l = blockIdx.y; l < lists; l += gridDim.y) {
        const int seq = l / c.n_kv, h = l % c.n_kv;
        const char* ws = a.workspace + evict_workspace(1, 1, c.table_stride) * l;
        const EvictHead head = *reinterpret_cast<const EvictHead*>(ws);
        const int* to = reinterpret_cast<const int*>(ws + 256);
        const int* from = to + c.table_stride * (kPage / 2);
        if (blockIdx.x == 0 && threadIdx.x == 0 && h == 0) a.new_len[seq] = head.new_len;
        const int step = gridDim.x * (kMoveThreads / 32) * kMoveBatch;
        int i0 = (blockIdx.x * (kMoveThreads / 32) + warp) * kMoveBatch;
        // A lane a row: its places, read one batch ahead.
        int d = 0, f = 0;
        if (lane < kMoveBatch && i0 + lane < head.moves) d = to[i0 + lane], f = from[i0 + lane];
        for (; i0 < head.moves; i0 += step) {
            const int rows = min(kMoveBatch, head.moves - i0);
            const long long od = 2 * ((long long)(d / kPage) * c.page_stride + h * c.head_stride + (long long)(d % kPage) * c.head_dim);
            const long long of = 2 * ((long long)(f / kPage) * c.page_stride + h * c.head_stride + (long long)(f % kPage) * c.head_dim);
            uint4 x[kMoveBatch];
#pragma unroll
            for (int r = 0; r < kMoveBatch; ++r) {
                const long long o = __shfl_sync(0xffffffffu, of, r);
                if (r < rows && lane < 2 * per_row) x[r] = *reinterpret_cast<const uint4*>(base + o + piece);
            }
            if (lane < rows) {
                const long long md = ((long long)(d / kPage) * c.n_kv + h) * kPage + d % kPage, mf = ((long long)(f / kPage) * c.n_kv + h) * kPage + f % kPage;
                const float w = c.weight[mf];
                const int p = c.position[mf];
                c.weight[md] = w;
                c.position[md] = p;
            }
            if (lane < kMoveBatch && i0 + step + lane < head.moves) d = to[i0 + step + lane], f = from[i0 + step + lane];
#pragma unroll
            for (int r = 0; r < kMoveBatch; ++r) {
                const long long o = __shfl_sync(0xffffffffu, od, r);
                if (r < rows && lane < 2 * per_row) *reinterpret_cast<uint4*>(base + o + piece) = x[r];
            }
        }
    }
}

}  // namespace

cudaError_t launch_rope_append(const RopeArgs& a, cudaStream_t s) {
    const bool f32 = a.in_type == OP_F32;
    if (a.c.type == OP_F16)
        return f32 ? rope_typed<float, __half>(a, s) : rope_typed<__half, __half>(a, s);
    return f32 ? rope_typed<float, __nv_bfloat16>(a, s) : rope_typed<__nv_bfloat16, __nv_bfloat16>(a, s);
}

cudaError_t launch_cache_evict(const EvictArgs& a, cudaStream_t s) {
    const int lists = a.c.n_seq * a.c.n_kv;
    const long long most_len = (long long)a.c.table_stride * kPage;
    // As many CTAs a list as its longest needs with eight slots a thread.
    int width = 1;
    while (width < 8 && most_len > (long long)width * kRankThreads * kRankEach) width *= 2;
    const bool regs = most_len <= (long long)width * kRankThreads * kRankEach && reinterpret_cast<uintptr_t>(a.c.position) % 16 == 0 &&
                      reinterpret_cast<uintptr_t>(a.c.weight) % 16 == 0;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    cudaError_t e;
    if (regs) {
        cfg.gridDim = dim3(lists * width);
        cfg.blockDim = dim3(kRankThreads);
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim = {(unsigned)width, 1, 1};
        e = cudaLaunchKernelEx(&cfg, k_evict_rank_regs, a, width);
    } else {
        static std::atomic<uint64_t> done{0};
        if ((e = allow_smem(k_evict_rank, kRankKeys * 4, &done)) != cudaSuccess) return e;
        k_evict_rank<<<lists, kRankThreads, int(std::min<long long>(most_len, kRankKeys)) * 4, s>>>(a);
        e = cudaGetLastError();
    }
    if (e != cudaSuccess) return e;
    const long long most = std::min<long long>(a.keep, most_len / 2);
    const int rows = kMoveThreads / 32 * kMoveBatch;
    const int wide = (int)std::max<long long>(1, std::min<long long>((most + rows - 1) / rows, 1 + 148 * 32 / lists));
    cfg.gridDim = dim3(wide, std::min(lists, 65535));
    cfg.blockDim = dim3(kMoveThreads);
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    e = cudaLaunchKernelEx(&cfg, k_evict_move, a, lists);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace mtb
