// What the attention kernels over a paged cache share: how the work is cut,
// how parts of a row tile are joined, barriers and copies.
//
// Rows: the new tokens of a sequence times the query heads of one KV head,
// row r = (token r / G, head r % G); a tile is some consecutive rows.  Units: a
// tile's visible cache in blocks of slots (at least one).  All units of
// all (sequence, KV head, tile) stand in one line, each tile behind some units for its own cost, and CTA c of g takes the
// c-th of g equal intervals of it, whatever the lengths are.  A tile that lies in
// one interval is finished there.  One that spans several leaves its parts (f32
// sums, row bases and row sums) in the workspace, and whichever CTA comes last
// joins them in the order of the intervals: no order of arrival changes a bit,
// and no CTA waits for another.
#pragma once

#include "ops_common.cuh"

#include <cuda.h>

namespace mtb {
namespace ops {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// ---- barriers and copies -------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t* b, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* b, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}
// Waits are for copies, products or warps of the same CTA.  The longest last as long as
// one CTA's share of a tile (warps that have nothing to do in it): 1.7 us for 128 slots.
constexpr int kWaitTries = 1 << 19;  // two seconds: a try that fails takes 4 us (measured)

// Waits for a phase; false once the wait ran out or another wait of this CTA
// did (`gave_up`, shared memory), so that every role leaves its loop.
__device__ __forceinline__ bool bar_wait(uint64_t* b, unsigned parity, volatile int* gave_up) {
    const uint32_t at = smem_u32(b);
    int left = kWaitTries;
#pragma unroll 1
    for (;;) {
        uint32_t ok;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(ok)
                     : "r"(at), "r"(parity)
                     : "memory");
        if (ok) return true;
        if (*gave_up) return false;
        if (--left == 0) {
            *gave_up = 1;
            return false;
        }
    }
}

// A barrier among some threads of the CTA whose wait is bounded: a role that
// has left its loop leaves nobody waiting for good.
struct SyncPoint {
    uint64_t* bar;
    unsigned phase = 0;
    volatile int* gave_up;
    __device__ __forceinline__ void sync() {  // counts warps
        __syncwarp();
        if ((threadIdx.x & 31) == 0) bar_arrive(bar);
        bar_wait(bar, phase, gave_up);
        phase ^= 1;
    }
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tma_prefetch(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
                 : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
                 : "memory");
}

// ---- tensor memory and its products --------------------------------------------------------------------------------

__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// The barrier gets one arrival when all products that this thread has issued are done.
__device__ __forceinline__ void tc_commit(uint64_t* b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(b)) : "memory");
}

// 32 lanes (the warp's quarter), consecutive columns: a thread has one row.
template <int kAt, int kN>
__device__ __forceinline__ void tmem_ld32(float (&x)[kN], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=f"(x[kAt + 0]), "=f"(x[kAt + 1]), "=f"(x[kAt + 2]), "=f"(x[kAt + 3]), "=f"(x[kAt + 4]), "=f"(x[kAt + 5]), "=f"(x[kAt + 6]), "=f"(x[kAt + 7]), "=f"(x[kAt + 8]), "=f"(x[kAt + 9]), "=f"(x[kAt + 10]), "=f"(x[kAt + 11]), "=f"(x[kAt + 12]), "=f"(x[kAt + 13]), "=f"(x[kAt + 14]), "=f"(x[kAt + 15]), "=f"(x[kAt + 16]), "=f"(x[kAt + 17]), "=f"(x[kAt + 18]), "=f"(x[kAt + 19]), "=f"(x[kAt + 20]), "=f"(x[kAt + 21]), "=f"(x[kAt + 22]), "=f"(x[kAt + 23]), "=f"(x[kAt + 24]), "=f"(x[kAt + 25]), "=f"(x[kAt + 26]), "=f"(x[kAt + 27]), "=f"(x[kAt + 28]), "=f"(x[kAt + 29]), "=f"(x[kAt + 30]), "=f"(x[kAt + 31])
                 : "r"(at));
}
template <int kAt, int kN>
__device__ __forceinline__ void tmem_st32(uint32_t at, const float (&x)[kN]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
                 ::"r"(at), "f"(x[kAt + 0]), "f"(x[kAt + 1]), "f"(x[kAt + 2]), "f"(x[kAt + 3]), "f"(x[kAt + 4]), "f"(x[kAt + 5]), "f"(x[kAt + 6]), "f"(x[kAt + 7]), "f"(x[kAt + 8]), "f"(x[kAt + 9]), "f"(x[kAt + 10]), "f"(x[kAt + 11]), "f"(x[kAt + 12]), "f"(x[kAt + 13]), "f"(x[kAt + 14]), "f"(x[kAt + 15]), "f"(x[kAt + 16]), "f"(x[kAt + 17]), "f"(x[kAt + 18]), "f"(x[kAt + 19]), "f"(x[kAt + 20]), "f"(x[kAt + 21]), "f"(x[kAt + 22]), "f"(x[kAt + 23]), "f"(x[kAt + 24]), "f"(x[kAt + 25]), "f"(x[kAt + 26]), "f"(x[kAt + 27]), "f"(x[kAt + 28]), "f"(x[kAt + 29]), "f"(x[kAt + 30]), "f"(x[kAt + 31])
                 : "memory");
}
template <int kAt, int kN>
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&x)[kN]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(at), "r"(x[kAt + 0]), "r"(x[kAt + 1]), "r"(x[kAt + 2]), "r"(x[kAt + 3]), "r"(x[kAt + 4]), "r"(x[kAt + 5]), "r"(x[kAt + 6]), "r"(x[kAt + 7]), "r"(x[kAt + 8]), "r"(x[kAt + 9]), "r"(x[kAt + 10]), "r"(x[kAt + 11]), "r"(x[kAt + 12]), "r"(x[kAt + 13]), "r"(x[kAt + 14]), "r"(x[kAt + 15])
                 : "memory");
}

// Descriptors of operand tiles of [dims / 64][rows][64 dims], 128-byte swizzle,
// 1024-byte aligned: the low word is the tile's (an offset adds its bytes / 16), the
// high word the layout's.  K-major (products over the dims): 8-row groups 1024 bytes
// apart.  MN-major (over the rows): also 64-dim parts `part` bytes apart.
__device__ __forceinline__ uint32_t desc_lo_k(uint32_t at) { return (at >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_lo_mn(uint32_t at, uint32_t part) { return (at >> 4) | ((part >> 4) << 16); }
constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);

// A value that all lanes have, as one the compiler knows to be uniform: the
// tensor cores' operands are uniform registers, and anything else is moved there
// for each product (measured: 90 clocks an issue instead of the product's 64).
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ bool elect_one() {
    uint32_t is;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(is));
    return is;
}

// f32 sums of 16-bit products, 128 rows x n columns.
constexpr uint32_t kNegateA = 1u << 13;
__device__ __forceinline__ constexpr uint32_t tc_instr(bool bf16, int n, bool b_mn) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t instr, bool add) {
    asm volatile("{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n"
                 ::"r"(d), "r"(a), "r"(b), "r"(instr), "r"((uint32_t)add), "r"(kDescHi)
                 : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t instr, bool add) {
    asm volatile("{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %4, 0;\n mov.b64 db, {%2, %5};\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n"
                 ::"r"(d), "r"(a), "r"(b), "r"(instr), "r"((uint32_t)add), "r"(kDescHi)
                 : "memory");
}

// ---- the line of units ---------------------------------------------------------------------------------------------

constexpr int kMaxCtas = 1024;  // counters that fit the workspace
constexpr int kMaxSms = 160;    // CTAs whose parts fit it

struct SeqWork {
    int len, tok0, n_new;
};

// Tiles hold whole tokens, so that a tile's q is one box: `per` tokens, `rows` =
// per G rows.
struct Geometry {
    int G, per, rows;
    FastDiv by_G, by_per;
    int block;  // slots per block
    int extra;  // units that stand for a tile's own cost (its q, its end) before those of its blocks
};
__device__ __forceinline__ Geometry geometry(const AttnArgs& a, int block, int extra) {
    return Geometry{a.G, a.per, a.per * a.G, a.by_G, a.by_per, block, extra};
}

__device__ __forceinline__ SeqWork seq_work(const AttnArgs& a, int s) {
    const int b = a.cu[s], e = a.cu[s + 1], n = a.c.kv_len[s];  // together: none waits for another
    if (b < 0 || e < b || e > a.n_tokens) {
        flag(a.c, BAD_TOKENS);
        return SeqWork{0, 0, 0};
    }
    const int len = (int)min(max((long long)n, 0ll), (long long)a.c.table_stride * kPage);
    if (e > b && len != n) flag(a.c, BAD_LEN);
    return SeqWork{len, b, e - b};
}

// How a sequence's work under one KV head is cut: tiles, and units of a tile.
struct CutRows {  // the attention: tiles of rows, in blocks of the slots that they see, at least one
    static __device__ __forceinline__ int tiles(const SeqWork& w, const Geometry& ge) { return ge.by_per(w.n_new + ge.per - 1); }
    static __device__ __forceinline__ int units(const SeqWork& w, const Geometry& ge, int tile) {
        const int end = min(w.n_new, (tile + 1) * ge.per);
        return max(1, (w.len - w.n_new + end + ge.block - 1) / ge.block);
    }
};
struct CutPages {  // the weights of few rows: one tile, in blocks of slots
    static __device__ __forceinline__ int tiles(const SeqWork& w, const Geometry&) { return w.n_new > 0 && w.len > 0; }
    static __device__ __forceinline__ int units(const SeqWork& w, const Geometry& ge, int) { return (w.len + ge.block - 1) / ge.block; }
};
struct CutSlots {  // the weights of many: tiles of slots, in tiles of the new tokens that see some of them
    static __device__ __forceinline__ int tiles(const SeqWork& w, const Geometry& ge) {
        return w.n_new > 0 ? (w.len + ge.block - 1) / ge.block : 0;
    }
    static __device__ __forceinline__ int first(const SeqWork& w, const Geometry& ge, int tile) {
        return ge.by_per(max(0, tile * ge.block - (w.len - w.n_new)));
    }
    static __device__ __forceinline__ int units(const SeqWork& w, const Geometry& ge, int tile) {
        return ge.by_per(w.n_new + ge.per - 1) - first(w, ge, tile);
    }
};
// Units of a sequence under one KV head, one sequence a lane: few tiles by
// the lane itself, many by the whole warp.
template <class Cut>
__device__ __forceinline__ long long head_units(const SeqWork& w, const Geometry& ge) {
    const int lane = threadIdx.x & 31;
    const int tiles = Cut::tiles(w, ge);
    long long u = 0;
    if (tiles <= 4)
#pragma unroll 1
        for (int t = 0; t < tiles; ++t) u += Cut::units(w, ge, t) + ge.extra;
#pragma unroll 1
    for (unsigned many = __ballot_sync(0xffffffffu, tiles > 4); many; many &= many - 1) {
        const int from = __ffs(many) - 1;
        const SeqWork x{__shfl_sync(0xffffffffu, w.len, from), 0, __shfl_sync(0xffffffffu, w.n_new, from)};
        const int n = __shfl_sync(0xffffffffu, tiles, from);
        long long sum = 0;
#pragma unroll 1
        for (int t = lane; t < n; t += 32) sum += Cut::units(x, ge, t) + ge.extra;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == from) u = sum;
    }
    return u;
}

// x / z for a quotient below 2^20: values mostly fit 32 bits, and where they do
// not, bit by bit (a call of the 64-bit division would cost the kernels registers).
__device__ __forceinline__ int div_small(long long x, long long z) {
    if (x < (1ll << 32) && z < (1ll << 32)) return (int)((unsigned)x / (unsigned)z);
    int q = 0;
#pragma unroll 1
    for (int bit = 1 << 19; bit; bit >>= 1)
        if ((q | bit) * z <= x) q |= bit;
    return q;
}
// total * b / parts, both below 2^11.
__device__ __forceinline__ long long share_of(long long total, int b, int parts) {
    const unsigned hi = (unsigned)(total >> 20), d = (unsigned)parts;
    const unsigned q1 = hi / d, low = ((hi - q1 * d) << 20) | (unsigned)(total & 0xfffff), q0 = low / d;
    return (((long long)q1 << 20) + q0) * b + (low - q0 * d) * (unsigned)b / d;
}

// The CTA's interval of the line, and where it begins.
struct Line {
    long long total, tiles, lo, hi;
    int ctas;       // CTAs that have an interval
    int seq;        // sequence of unit lo
    long long off;  // of lo in that sequence's units
    long long per;  // that sequence's units under one KV head
    SeqWork work;   // that sequence's
};

// As many CTAs as there are, but fewer where their intervals would be shorter
// than min_units, unless there is a tile for each.  Never more than units: a split
// tile's parts are counted by the intervals it spans, so none of them may be empty.
__device__ __forceinline__ void cut_line(Line* l, int min_units) {
    const long long fit = max(max(1ll, l->tiles), l->total / min_units);
    l->ctas = (int)min(min((long long)gridDim.x, fit), l->total);
    l->lo = l->hi = 0;
    if ((int)blockIdx.x < l->ctas) {
        l->lo = share_of(l->total, blockIdx.x, l->ctas);
        l->hi = share_of(l->total, blockIdx.x + 1, l->ctas);
    }
}

// Up to 32 sequences: one warp by itself.
template <class Cut>
__device__ Line find_line_warp(const AttnArgs& a, const Geometry& ge, int min_units) {
    const int lane = threadIdx.x & 31;
    SeqWork w{0, 0, 0};
    if (lane < a.c.n_seq) {
        w = seq_work(a, lane);
        if (w.n_new > w.len && blockIdx.x == 0) flag(a.c, BAD_LEN);
    }
    const long long per = head_units<Cut>(w, ge), v = per * a.c.n_kv;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    Line l{};
    l.total = __shfl_sync(0xffffffffu, x, 31);
    int tiles = (int)min((long long)Cut::tiles(w, ge) * a.c.n_kv, (long long)kMaxCtas);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    l.tiles = tiles;
    cut_line(&l, min_units);
    const unsigned at = __ballot_sync(0xffffffffu, v > 0 && x - v <= l.lo && l.lo < x);
    l.seq = max(0, __ffs(at) - 1);
    l.off = l.lo - __shfl_sync(0xffffffffu, x - v, l.seq);
    l.per = __shfl_sync(0xffffffffu, per, l.seq);
    l.work = SeqWork{__shfl_sync(0xffffffffu, w.len, l.seq), __shfl_sync(0xffffffffu, w.tok0, l.seq), __shfl_sync(0xffffffffu, w.n_new, l.seq)};
    return l;
}

// Any number: all threads of the CTA; s_scan: one long long a warp + 3.
template <int kThreads, class Cut>
__device__ __noinline__ Line find_line_cta(const AttnArgs& a, const Geometry ge, int min_units, long long* s_scan) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int kWarps = kThreads / 32;
    __shared__ int s_tiles[kWarps];
    int tiles = 0;
    auto units_of = [&](int s, bool first) {
        SeqWork w{0, 0, 0};
        if (s < a.c.n_seq) {
            w = seq_work(a, s);
            if (first && w.n_new > w.len && blockIdx.x == 0) flag(a.c, BAD_LEN);
        }
        if (first) tiles += (int)min((long long)Cut::tiles(w, ge) * a.c.n_kv, (long long)kMaxCtas);
        return head_units<Cut>(w, ge) * a.c.n_kv;
    };
    long long mine = 0, sum = 0;
    for (int s0 = 0; s0 < a.c.n_seq; s0 += kThreads) {
        mine = units_of(s0 + threadIdx.x, true);
        sum += mine;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    }
    if (lane == 0) {
        s_scan[warp] = sum;
        s_tiles[warp] = tiles;
    }
    __syncthreads();
    Line l{};
#pragma unroll 1
    for (int w = 0; w < kWarps; ++w) {
        l.total += s_scan[w];
        l.tiles += s_tiles[w];
    }
    cut_line(&l, min_units);
    long long base = 0;
    for (int s0 = 0; s0 < a.c.n_seq; s0 += kThreads) {
        const long long v = a.c.n_seq <= kThreads ? mine : units_of(s0 + threadIdx.x, false);
        long long x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) s_scan[warp] = x;
        __syncthreads();
        long long before = base;
#pragma unroll 1
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += s_scan[w];
            base += s_scan[w];
        }
        const long long first = before + x - v;
        if (v > 0 && first <= l.lo && l.lo < first + v) {
            s_scan[kWarps] = s0 + threadIdx.x;
            s_scan[kWarps + 1] = l.lo - first;
            s_scan[kWarps + 2] = v / a.c.n_kv;
        }
    }
    __syncthreads();
    l.seq = (int)s_scan[kWarps];
    l.off = s_scan[kWarps + 1];
    l.per = s_scan[kWarps + 2];
    if (l.lo < l.hi) l.work = seq_work(a, l.seq);
    return l;
}

// The interval, for the producer warp; all threads call, and with few
// sequences nobody waits.
template <int kThreads, class Cut>
__device__ __forceinline__ Line find_line(const AttnArgs& a, const Geometry& ge, int min_units, long long* s_scan, bool producer) {
    if (a.c.n_seq > 32) return find_line_cta<kThreads, Cut>(a, ge, min_units, s_scan);
    if (!producer) return Line{};
    return find_line_warp<Cut>(a, ge, min_units);
}

// The CTA whose interval holds unit u.
__device__ __forceinline__ int cta_of(long long total, int ctas, long long u) { return div_small((u + 1) * ctas - 1, total); }

// A CTA's part of one tile: blocks [b0, b1) of its n, with what the roles need
// of its sequence.  n == 0: there are no more parts.
struct Part {
    int seq, head, tile, b0, b1, n;
    int len, tok0, n_new;
    int ctas;  // of the line
    long long u0, total;  // the tile's first block in the line of `total` units
    __device__ int first_cta() const { return cta_of(total, ctas, u0); }
    __device__ int last_cta() const { return cta_of(total, ctas, u0 + n - 1); }
};

// Walks the CTA's interval, one warp.  Whole: a tile goes undivided to the
// interval that holds its first unit.
template <class Cut, bool kWhole = false>
struct Walk {
    const AttnArgs& a;
    const Geometry ge;
    const Line& line;
    long long at;  // next unit
    SeqWork w{};
    int seq, head = 0, tile = 0, block = 0, tiles = 0;

    __device__ Walk(const AttnArgs& args, const Geometry& g, const Line& l) : a(args), ge(g), line(l), at(l.lo), seq(l.seq) {
        if (l.lo >= l.hi) return;
        w = l.work;
        tiles = Cut::tiles(w, ge);
        head = a.c.n_kv == 1 ? 0 : div_small(l.off, l.per);
        long long off = l.off - head * l.per;
        const int lane = threadIdx.x & 31;
        for (;; tile += 32) {  // 32 tiles at a time
            long long x = tile + lane < tiles ? Cut::units(w, ge, tile + lane) + ge.extra : 0;
            const long long v = x;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            const unsigned past = __ballot_sync(0xffffffffu, off < x);
            if (past) {
                const int i = __ffs(past) - 1;
                tile += i;
                block = (int)(off - __shfl_sync(0xffffffffu, x - v, i));
                break;
            }
            off -= __shfl_sync(0xffffffffu, x, 31);
        }
        if (kWhole && block > 0) {
            at += Cut::units(w, ge, tile) + ge.extra - block;
            step();
        }
    }
    __device__ void step() {
        block = 0;
        if (++tile < tiles) return;
        tile = 0;
        if (++head < a.c.n_kv) return;
        head = 0;
        // The next sequence that has tiles: a lane a sequence, since thousands without may lie between.
        const int lane = threadIdx.x & 31;
        while (at < line.hi) {
            if (++seq >= a.c.n_seq) {  // lengths that changed under the kernel
                at = line.hi;
                break;
            }
            const SeqWork x = seq + lane < a.c.n_seq ? seq_work(a, seq + lane) : SeqWork{0, 0, 0};
            const int n = Cut::tiles(x, ge);
            const unsigned some = __ballot_sync(0xffffffffu, n > 0);
            if (!some) {
                seq += 31;
                continue;
            }
            const int from = __ffs(some) - 1;
            seq += from;
            w = SeqWork{__shfl_sync(0xffffffffu, x.len, from), __shfl_sync(0xffffffffu, x.tok0, from), __shfl_sync(0xffffffffu, x.n_new, from)};
            tiles = __shfl_sync(0xffffffffu, n, from);
            break;
        }
    }
    __device__ bool next(Part* p) {
        while (at < line.hi) {
            const int n = Cut::units(w, ge, tile), all = n + ge.extra;
            const int take = kWhole ? all : (int)min((long long)(all - block), line.hi - at);
            const long long u0 = at - block;
            const int b0 = max(0, block - ge.extra), b1 = block + take - ge.extra;
            *p = Part{seq, head, tile, b0, b1, n, w.len, w.tok0, w.n_new, line.ctas, u0 + ge.extra, line.total};
            at += take;
            block += take;
            if (block == all) step();
            if (b1 > 0) return true;  // else the interval ended before the tile's first block
        }
        return false;
    }
};

// The producer warp walks and hands the parts to the other roles' warps
// through a ring in shared memory.
template <int kRing>
struct PartRing {
    Part part[kRing];
    uint64_t full[kRing], taken[kRing];
    __device__ void init(int warps) {
        for (int i = 0; i < kRing; ++i) {
            bar_init(&full[i], 1);
            bar_init(&taken[i], warps);
        }
    }
    // The producer warp, the i-th part; false: the wait for room ran out.  Without sequences (calls that
    // mtb_debug_stall_attention picks; no others are launched) nothing is put, so that the others' waits run out.
    __device__ bool put(unsigned i, const Part& p, volatile int* gave_up) {
        if (i >= kRing && !bar_wait(&taken[i % kRing], (i / kRing - 1) & 1, gave_up)) return false;
        if ((threadIdx.x & 31) == 0) {
            part[i % kRing] = p;
            bar_arrive(&full[i % kRing]);
        }
        __syncwarp();
        return true;
    }
    // A warp; false: there are no more.
    __device__ bool get(unsigned i, Part* p, volatile int* gave_up) {
        if (!bar_wait(&full[i % kRing], (i / kRing) & 1, gave_up)) return false;
        *p = part[i % kRing];
        __syncwarp();
        if ((threadIdx.x & 31) == 0) bar_arrive(&taken[i % kRing]);
        return p->n > 0;
    }
};

// ---- parts in the workspace ----------------------------------------------------------------------------------------

// Counters (one for each CTA that begins a split tile), then two parts for each
// CTA: of the tile that reached into its interval, and of the one that begins
// there.  A part: row bases (log2), row sums, f32 sums of p v.
constexpr size_t kPartsAt = 8192;

template <int kRows, int kD>
__device__ __forceinline__ float* part_at(const AttnArgs& a, int cta, bool begins) {
    return reinterpret_cast<float*>(a.workspace + kPartsAt) + (size_t)(2 * cta + (begins ? 1 : 0)) * (kRows * (kD + 2));
}

// Loads of what other CTAs wrote in this launch: from L2, and kept in order with the barriers.
__device__ __forceinline__ float ld_cg(const float* p) {
    float x;
    asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(x) : "l"(p));
    return x;
}
__device__ __forceinline__ float4 ld_cg4(const float* p) {
    float4 x;
    asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "l"(p));
    return x;
}

template <class T>
__device__ __forceinline__ void store4(T* p, float4 x) {
    uint2 u;
    T* t = reinterpret_cast<T*>(&u);
    t[0] = from_f32<T>(x.x);
    t[1] = from_f32<T>(x.y);
    t[2] = from_f32<T>(x.z);
    t[3] = from_f32<T>(x.w);
    *reinterpret_cast<uint2*>(p) = u;
}

// Where row r of a part's tile goes; false: not a row of the sequence.
__device__ __forceinline__ bool row_place(const Geometry& ge, const Part& p, int r, long long* token, int* head) {
    const int t = ge.by_G(r), tok = p.tile * ge.per + t;
    if (t >= ge.per || tok >= p.n_new) return false;
    *token = p.tok0 + tok;
    *head = p.head * ge.G + r - t * ge.G;
    return true;
}

// Counts a part of a split tile as written; the number of its parts for whom it was
// the last, else 0.  By one thread, between two barriers of the CTA: its release
// covers what the others wrote before the first, its acquire what they read behind the second.
__device__ __forceinline__ int parts_if_last(const AttnArgs& a, const Part& p) {
    const int c0 = p.first_cta(), parts = p.last_cta() - c0 + 1;
    int* count = reinterpret_cast<int*>(a.workspace) + c0;
    int before;
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(count) : "memory");
    if (before != parts - 1) return 0;
    *count = 0;
    return parts;
}

// Joins a split tile's parts, by kWarps warps numbered from 0.  First each row's
// factors, which take the bases' place: few rows a warp each, a lane a part; many
// rows a thread each.  Then the sums: four columns a thread; the loads wait for
// nothing, and go out for eight parts (few rows) or eight rows (many) at a time.
template <class T, int kRows, int kD, int kWarps>
__device__ __forceinline__ void join_parts(const AttnArgs& a, const Geometry& ge, const Part& p, int parts, SyncPoint& all) {
    constexpr bool kFew = kRows <= 32;
    constexpr int kThreads = kWarps * 32, kStep = 2 * kRows * (kD + 2);  // floats from a part to the next; the first is the one that begins the tile
    constexpr int kEach = kFew ? (kMaxSms + 31) / 32 : 1;                 // parts of a lane
    const int rows = min(ge.rows, (p.n_new - p.tile * ge.per) * ge.G);
    const int lane = threadIdx.x & 31;
    float* others = part_at<kRows, kD>(a, p.first_cta(), false);  // part i > 0 at others + i kStep, part 0 half a step behind
    auto at = [&](int c) { return others + (size_t)c * kStep + (c ? 0 : kStep / 2); };
#pragma unroll 1
    for (int r = kFew ? threadIdx.x >> 5 : threadIdx.x; r < rows; r += kFew ? kWarps : kThreads) {
        float m = -INFINITY, sum = 0.f;
        if constexpr (kFew) {
            float mi[kEach], li[kEach];
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                const int c = lane + 32 * k;
                mi[k] = c < parts ? ld_cg(at(c) + r) : -INFINITY;
                li[k] = c < parts ? ld_cg(at(c) + kRows + r) : 0.f;
            }
#pragma unroll
            for (int k = 0; k < kEach; ++k) m = fmaxf(m, mi[k]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                mi[k] = exp2_fast(mi[k] - base);
                sum = __fmaf_rn(mi[k], li[k], sum);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
            for (int k = 0; k < kEach; ++k)
                if (lane + 32 * k < parts) __stcg(at(lane + 32 * k) + r, mi[k] * inv);
        } else {
#pragma unroll 4
            for (int c = 0; c < parts; ++c) m = fmaxf(m, ld_cg(at(c) + r));
            const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 4
            for (int c = 0; c < parts; ++c) sum = __fmaf_rn(exp2_fast(ld_cg(at(c) + r) - base), ld_cg(at(c) + kRows + r), sum);
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll 4
            for (int c = 0; c < parts; ++c) __stcg(at(c) + r, exp2_fast(ld_cg(at(c) + r) - base) * inv);
        }
        long long token;
        int head;
        if ((!kFew || lane == 0) && a.lse && row_place(ge, p, r, &token, &head))
            a.lse[token * a.n_heads + head] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * kLn2;
    }
    all.sync();
    constexpr int kCols = kD / 4, kItems = kFew ? 1 : 8, kParts = kFew ? 8 : 1;
    const int items = rows * kCols;
#pragma unroll 1
    for (int i0 = threadIdx.x; i0 < items; i0 += kItems * kThreads) {
        float4 o[kItems];
#pragma unroll
        for (int u = 0; u < kItems; ++u) o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int c0 = 0; c0 < parts; c0 += kParts) {
            float f[kItems * kParts];
            float4 x[kItems * kParts];
#pragma unroll
            for (int u = 0; u < kItems * kParts; ++u) {
                const int i = i0 + (kFew ? 0 : u * kThreads), c = c0 + (kFew ? u : 0), r = i / kCols;
                f[u] = 0.f;
                x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i < items && c < parts) {
                    f[u] = ld_cg(at(c) + r);
                    x[u] = ld_cg4(at(c) + 2 * kRows + r * kD + i % kCols * 4);
                }
            }
#pragma unroll
            for (int u = 0; u < kItems * kParts; ++u) {
                float4& y = o[kFew ? 0 : u];
                y.x = __fmaf_rn(f[u], x[u].x, y.x);
                y.y = __fmaf_rn(f[u], x[u].y, y.y);
                y.z = __fmaf_rn(f[u], x[u].z, y.z);
                y.w = __fmaf_rn(f[u], x[u].w, y.w);
            }
        }
#pragma unroll
        for (int u = 0; u < kItems; ++u) {
            const int i = i0 + u * kThreads;
            long long token;
            int head;
            if (i < items && row_place(ge, p, i / kCols, &token, &head))
                store4<T>(reinterpret_cast<T*>(a.out) + token * a.out_stride + (long long)head * kD + i % kCols * 4, o[u]);
        }
    }
}

}  // namespace ops
}  // namespace mtb
