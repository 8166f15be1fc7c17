// mtb_paged_attention and mtb_attention_weights.
//
// o = sum_j exp(s_j - lse) v_j with s = scale q.k, one pass over the cache: a
// running base m and sum l of p = exp2(s log2 e - m), the sums of p v rescaled when the
// maximum has grown by more than 8 since m was set (l and the sums are f32).  p is
// rounded to the cache's type for the product with v, as the tensor cores want it (for
// at most 16 rows the rest goes into a second product); l adds it unrounded.  bf16 holds any p as exactly as 1.  fp16 loses bits below 2^-14
// and everything below 2^-25, so m lies 7 below the maximum there: p stays below 2^15,
// and one that is 2^-21 of the largest keeps its bits (a first position that takes
// nearly all of the weight is no rare sight).
#include "ops_attention.cuh"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace mtb {
namespace {

using namespace ops;

// Units that stand for a tile's own cost, and those of a CTA's interval at least.
// Tiles of a chunk: prompts of 1 .. 2048 rows take 73.7 us with 1, 70.0 with 2, 72.5
// with 3.  Few rows: eight ragged sequences 61.0 us with 1, 57.4 with 2, 56.5
// with 4, 56.2 with 6; one token over 408 slots 13.2 us cut at 8 units, 8.3 at 16.
constexpr int kRowsExtra = 4, kRowsMinUnits = 16;    // of 64 slots
constexpr int kTilesExtra = 2, kTilesMinUnits = 4;  // of 128 slots


__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// 2^x on the FMA units, for x in [-125, 127]: x = n + r, r in [-1/2, 1/2], a
// degree-5 polynomial for 2^r (least relative error, 2.1e-7 as evaluated), n added
// to the exponent.  Below -125: 0.
__device__ __forceinline__ float2 exp2_poly(float2 x0) {
    float2 x = x0;
    const float2 shift = make_float2(12582912.f, 12582912.f), back = make_float2(-12582912.f, -12582912.f);
    x.x = fmaxf(x.x, -125.f);
    x.y = fmaxf(x.y, -125.f);
    const float2 t = __fadd2_rn(x, shift);  // the nearest integer, in the low bits
    const float2 n = __fadd2_rn(t, back);
    const float2 r = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
    float2 p = __ffma2_rn(make_float2(0.0013276471f, 0.0013276471f), r, make_float2(0.009675541f, 0.009675541f));
    p = __ffma2_rn(p, r, make_float2(0.05550713f, 0.05550713f));
    p = __ffma2_rn(p, r, make_float2(0.2402212f, 0.2402212f));
    p = __ffma2_rn(p, r, make_float2(0.69314694f, 0.69314694f));
    p = __ffma2_rn(p, r, make_float2(1.0000001f, 1.0000001f));
    p.x = __int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23));
    p.y = __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23));
    p.x = x0.x >= -125.f ? p.x : max_nan(x0.x, 0.f);  // a NaN stays one
    p.y = x0.y >= -125.f ? p.y : max_nan(x0.y, 0.f);
    return p;
}
// How far m lies below the maximum that it was set by.
template <class T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.f : 0.f;

template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// What pack2 left of the two values, packed in turn.
__device__ __forceinline__ float2 unpack2(uint32_t x, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }
__device__ __forceinline__ float2 unpack2(uint32_t x, __nv_bfloat16) { return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)); }
template <class T>
__device__ __forceinline__ uint32_t pack2_rest(uint32_t packed, float lo, float hi) {
    const float2 y = unpack2(packed, T());
    return pack2<T>(lo - y.x, hi - y.y);
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

bool encode(CUtensorMap* map, int type, int rank, void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    static const EncodeFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeFn>(f);
    }();
    const cuuint32_t steps[4] = {1, 1, 1, 1};
    return fn && fn(map, type == OP_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, base, dims, strides, box, steps,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// K or V: (dim, row of the page, KV head, page) in boxes of 64 dims x 64 rows.
bool encode_cache(CUtensorMap* map, const PagedView& c, void* base) {
    const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, kPage, (cuuint64_t)c.n_kv, (cuuint64_t)c.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)c.head_dim * 2, (cuuint64_t)c.head_stride * 2, (cuuint64_t)c.page_stride * 2};
    const cuuint32_t box[4] = {64, kPage, 1, 1};
    return encode(map, c.type, 4, base, dims, strides, box);
}

// q: (dim, head, token) in boxes of 64 dims x one KV head's group x as many whole tokens as the rows hold.
bool encode_q(CUtensorMap* map, const AttnArgs& a, int rows) {
    const int G = a.G;
    const cuuint64_t dims[3] = {(cuuint64_t)a.c.head_dim, (cuuint64_t)a.n_heads, (cuuint64_t)a.n_tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)a.c.head_dim * 2, (cuuint64_t)a.q_stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)(rows / G)};
    return encode(map, a.c.type, 3, const_cast<char*>(a.q), dims, strides, box);
}

// ---- few rows ------------------------------------------------------------------------------------------------------
//
// A step or a verify pass: a tile of 16 or 32 rows, so each K and V byte
// serves few products and the cache's bytes bound the kernel.  One CTA per SM
// walks its interval of 64-slot pages; a producer warp brings a page's K and V
// (TMA boxes of 64 slots x 64 dims, 128-byte swizzle: the ldmatrix reads below
// are free of bank conflicts) into a ring of as many pages as shared memory
// holds, and the next tile's q, across tile borders.  Each of four warps takes 16 of a page's 64
// slots, with a maximum, sum and f32 result of its own (m16n8k16, scores stay in
// registers as the second product's operand), so that no page costs a barrier among them;
// they are joined when the tile's part ends.  16 rows: two such sets of
// four warps take the pages in turn (a page is a chain of dependent steps, two
// chains fill each other's gaps), and what P's rounding to 16 bits left goes into a
// second product: results are then as near as f32 probabilities bring them (bf16, one
// token over 408 slots: 0.0017 relative, the result's own rounding, instead of 0.0028) for 1% of the
// time of heads of 128 (32 sequences 50.1 -> 50.7 us), 6% of heads of 64 (four tokens of 4 x 9000
// slots 20.1 -> 21.3); 32 rows would pay a ninth (45 -> 50 us) and go without.  16 heads of 128 over 8 KV heads: one token over 27000
// slots 26.1 us (4.2 TB/s: the start, the last pages and the join are a third of it), 32 sequences of 2048
// slots 51 us (5.3 TB/s), eight ragged sequences of 1 .. 8 new tokens 57 us (5.3 TB/s).

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <class T>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// MW: 16-row tiles of a warp; WP: sets of four warps, by pages.
template <int kD, int MW, int WP>
struct RowsShape {
    static constexpr int kRows = 16 * MW;
    static constexpr int kWarps = 4 * WP;                      // consumers; they share all rows
    static constexpr int kThreads = (kWarps + 1) * 32;
    static constexpr int kHalf = kPage * 128;                  // bytes of 64 slots x 64 dims
    static constexpr int kStage = 2 * (kD / 64) * kHalf;       // a page's K, then its V
    static constexpr int kQ = kRows * kD * 2;                  // one of two
    static constexpr int kPad = kD + 8;                        // floats of a warp's result row: no two rows on the same banks
    static constexpr int kJoin = kWarps * kRows * kPad * 4;
    static constexpr int kRoom = 227 * 1024 - 1024 - 4096;     // alignment, static
    static constexpr int kFit = (kRoom - 2 * kQ - kJoin) / kStage;
    // A stage always falls to the same set of warps: each waits for every fill
    // of its stages, or a barrier's parity would say nothing.
    static constexpr int kStages = (kFit > 12 ? 12 : kFit) / WP * WP;
    // What P's rounding left goes into a second product, where another set of warps fills its time.
    static constexpr bool kRest = WP > 1;
    static constexpr int kSmem = 1024 + kStages * kStage + 2 * kQ + kJoin;
};
constexpr int kPartRing = 8;

template <class T, int kD, int MW, int WP>
__global__ void __launch_bounds__(RowsShape<kD, MW, WP>::kThreads, 1)
    k_attention_rows(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                     const __grid_constant__ CUtensorMap q_map) {
    using S = RowsShape<kD, MW, WP>;
    constexpr int kParts = kD / 64;  // 64-dim parts of a row
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[S::kStages], empty[S::kStages], q_full[2], q_empty[2], all_bar, read_bar;
    __shared__ PartRing<kPartRing> parts;
    __shared__ int s_page[S::kStages];  // the stage's page, negative: masked
    __shared__ long long s_scan[16];
    __shared__ float s_m[S::kWarps][S::kRows], s_l[S::kWarps][S::kRows];
    __shared__ int s_gave_up, s_last;
    const uint32_t ring = (smem_u32(smem_raw) + 1023) & ~1023u;
    const uint32_t q_at = ring + S::kStages * S::kStage;
    float* join = reinterpret_cast<float*>(smem_raw + (q_at - smem_u32(smem_raw)) + 2 * S::kQ);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.G, per = a.per, live = per * G;  // whole tokens and rows of a tile
    const Geometry ge = geometry(a, kPage, kRowsExtra);
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kStages; ++i) {
            bar_init(&full[i], 1);
            bar_init(&empty[i], 4);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(&q_full[i], 1);
            bar_init(&q_empty[i], S::kWarps);
        }
        bar_init(&all_bar, S::kWarps);
        bar_init(&read_bar, S::kWarps);
        parts.init(S::kWarps);
        s_gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == S::kWarps * 32) {
        tma_prefetch(&k_map);
        tma_prefetch(&v_map);
        tma_prefetch(&q_map);
    }
    __syncthreads();
    const Line line = find_line<S::kThreads, CutRows>(a, ge, kRowsMinUnits, s_scan, warp == S::kWarps);
    Part p;

    if (warp == S::kWarps) {
        // Producer: table entries 32 at a time, one a lane.
        Walk<CutRows> walk(a, ge, line);
        int st = 0, round = 0;
        unsigned turn = 0;
        bool ok = true;
        while (ok && walk.next(&p)) {
            if (!parts.put(turn, p, &s_gave_up)) break;
            const int qb = turn & 1;
            if (turn >= 2 && !bar_wait(&q_empty[qb], ((turn >> 1) - 1) & 1, &s_gave_up)) break;
            if (lane == 0) {
                bar_expect(&q_full[qb], live * kD * 2);
#pragma unroll
                for (int h = 0; h < kParts; ++h)
                    tma_load_3d(q_at + qb * S::kQ + h * (S::kRows * 128), &q_map, h * 64, p.head * G, p.tok0 + p.tile * per, &q_full[qb]);
            }
            ++turn;
            for (int b0 = p.b0; ok && b0 < p.b1; b0 += 32) {
                int mine = -1;
                if (b0 + lane < p.b1 && (long long)(b0 + lane) * kPage < p.len) mine = page_of(a.c, p.seq, b0 + lane);
                for (int b = b0; b < min(p.b1, b0 + 32); ++b) {
                    const int page = __shfl_sync(0xffffffffu, mine, b - b0);
                    if (round > 0 && !bar_wait(&empty[st], (round - 1) & 1, &s_gave_up)) {
                        ok = false;
                        break;
                    }
                    if (lane == 0) {
                        s_page[st] = page;
                        if (page < 0) {
                            bar_arrive(&full[st]);
                        } else {
                            bar_expect(&full[st], S::kStage);
                            const uint32_t dst = ring + st * S::kStage;
#pragma unroll
                            for (int h = 0; h < kParts; ++h)
                                tma_load_4d(dst + h * S::kHalf, &k_map, h * 64, 0, p.head, page, &full[st]);
#pragma unroll
                            for (int h = 0; h < kParts; ++h)
                                tma_load_4d(dst + (kParts + h) * S::kHalf, &v_map, h * 64, 0, p.head, page, &full[st]);
                        }
                    }
                    __syncwarp();
                    if (++st == S::kStages) st = 0, ++round;
                }
            }
        }
        p.n = 0;
        if (a.c.n_seq > 0) parts.put(turn, p, &s_gave_up);
        // No copy is left in flight when the CTA ends: each stage's last fill has landed.
        volatile int none = 0;
        #pragma unroll 1
        for (int i = 0; i < S::kStages; ++i) {
            const int fills = round + (i < st ? 1 : 0);
            if (fills > 0) bar_wait(&full[i], (fills - 1) & 1, &none);
        }
        #pragma unroll 1
        for (int i = 0; i < 2; ++i) {
            const int fills = (turn + 1 - i) / 2;
            if (fills > 0) bar_wait(&q_full[i], (fills - 1) & 1, &none);
        }
        if (lane == 0 && s_gave_up) flag(a.c, BAD_WAIT);
        return;
    }

    const int wp = warp >> 2, sw = warp & 3;
    const float to_log2 = a.scale * kLog2e;
    SyncPoint all{&all_bar, 0, &s_gave_up};
    int st = 0, mine = 0;  // mine: whose turn the stage is
    unsigned phase = 0;
    for (unsigned turn = 0; parts.get(turn, &p, &s_gave_up); ++turn) {
        const int base = p.len - p.n_new;  // the first new token's slot
        const int rows = min(live, p.n_new * G - p.tile * live);
        const int first = p.tile * per;    // the tile's first token
        // Slots that the thread's rows see: [0, base + token(r) + 1); least, most: of the tile's rows.
        int sees[MW][2];
#pragma unroll
        for (int mt = 0; mt < MW; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) sees[mt][e] = base + first + ge.by_G(mt * 16 + e * 8 + lane / 4) + 1;
        const int least = base + first + 1, most = base + min(first + per, p.n_new);
        bool ok = bar_wait(&q_full[turn & 1], (turn >> 1) & 1, &s_gave_up);
        const uint32_t qa = q_at + (turn & 1) * S::kQ;
        uint32_t q[MW == 1 ? kD / 16 : 1][4];
        if constexpr (MW == 1) {
#pragma unroll
            for (int kk = 0; kk < kD / 16; ++kk) {
                const int r = lane & 15, ch = kk * 2 + (lane >> 4);
                ldsm4(q[kk], qa + (ch / 8) * (S::kRows * 128) + r * 128 + (((ch & 7) ^ (r & 7)) * 16));
            }
        }
        float o[MW][kD / 8][4], m[MW][2], l[MW][2];
#pragma unroll
        for (int mt = 0; mt < MW; ++mt) {
#pragma unroll
            for (int n = 0; n < kD / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[mt][n][e] = 0.f;
            m[mt][0] = m[mt][1] = -INFINITY;
            l[mt][0] = l[mt][1] = 0.f;
        }
        for (int b = p.b0; ok && b < p.b1; ++b) {
            const bool here = mine == wp;
            const int at = st;
            const unsigned parity = phase;
            if (++st == S::kStages) st = 0, phase ^= 1;
            if (++mine == WP) mine = 0;
            if (!here) continue;
            if (!bar_wait(&full[at], parity, &s_gave_up)) {
                ok = false;
                break;
            }
            const int s0 = b * kPage + sw * 16;  // the warp's first slot
            if (s_page[at] >= 0 && s0 < most) {
                const uint32_t kb = ring + at * S::kStage, vb = kb + kParts * S::kHalf;
                float s[MW][2][4];
#pragma unroll
                for (int mt = 0; mt < MW; ++mt)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[mt][n][e] = 0.f;
#pragma unroll
                for (int kk = 0; kk < kD / 16; ++kk) {
                    uint32_t kf[4];
                    const int slot = sw * 16 + ((lane >> 4) << 3) + (lane & 7), ch = kk * 2 + ((lane >> 3) & 1);
                    ldsm4(kf, kb + (ch / 8) * S::kHalf + slot * 128 + (((ch & 7) ^ (slot & 7)) * 16));
#pragma unroll
                    for (int mt = 0; mt < MW; ++mt) {
                        uint32_t qf[4];
                        if constexpr (MW == 1) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) qf[e] = q[kk][e];
                        } else {
                            const int r = mt * 16 + (lane & 15), qc = kk * 2 + (lane >> 4);
                            ldsm4(qf, qa + (qc / 8) * (S::kRows * 128) + r * 128 + (((qc & 7) ^ (r & 7)) * 16));
                        }
                        mma16<T>(s[mt][0], qf, kf[0], kf[1]);
                        mma16<T>(s[mt][1], qf, kf[2], kf[3]);
                    }
                }
                uint32_t pa[MW][4], rest[MW][4];
                const bool mask = s0 + 16 > least;
#pragma unroll
                for (int mt = 0; mt < MW; ++mt) {
                    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float x = s[mt][n][e] * to_log2;
                            if (mask && s0 + n * 8 + (lane & 3) * 2 + (e & 1) >= sees[mt][e >> 1]) x = -INFINITY;
                            s[mt][n][e] = x;
                            top[e >> 1] = fmaxf(top[e >> 1], x);
                        }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
                        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
                    }
                    // The base follows only when the maximum has grown by more than 8.
                    const bool grown[2] = {top[0] > m[mt][0] + (8.f + kLift<T>), top[1] > m[mt][1] + (8.f + kLift<T>)};
                    if (__any_sync(0xffffffffu, grown[0] || grown[1])) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float to = grown[e] ? top[e] - kLift<T> : m[mt][e];  // a row goes by its own scores alone
                            const float f = to == -INFINITY ? 1.f : exp2_fast(m[mt][e] - to);
                            m[mt][e] = to;
                            l[mt][e] *= f;
#pragma unroll
                            for (int n = 0; n < kD / 8; ++n) {
                                o[mt][n][2 * e] *= f;
                                o[mt][n][2 * e + 1] *= f;
                            }
                        }
                    }
                    const float b0 = m[mt][0] == -INFINITY ? 0.f : m[mt][0], b1 = m[mt][1] == -INFINITY ? 0.f : m[mt][1];
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[mt][n][e] = exp2_fast(s[mt][n][e] - (e < 2 ? b0 : b1));
                            l[mt][e >> 1] += s[mt][n][e];
                        }
                        pa[mt][2 * n] = pack2<T>(s[mt][n][0], s[mt][n][1]);
                        pa[mt][2 * n + 1] = pack2<T>(s[mt][n][2], s[mt][n][3]);
                        if constexpr (S::kRest) {
                            rest[mt][2 * n] = pack2_rest<T>(pa[mt][2 * n], s[mt][n][0], s[mt][n][1]);
                            rest[mt][2 * n + 1] = pack2_rest<T>(pa[mt][2 * n + 1], s[mt][n][2], s[mt][n][3]);
                        }
                    }
                }
                // V at or behind the sequence's end may hold anything: 0 there, since 0 * NaN is NaN.
                const bool tail = s0 + 16 > p.len;
                uint32_t lo_on = 0xffffffffu, hi_on = 0xffffffffu;
                if (tail) {
                    const int first_slot = s0 + (lane & 3) * 2;
                    lo_on = (first_slot < p.len ? 0xffffu : 0u) | (first_slot + 1 < p.len ? 0xffff0000u : 0u);
                    hi_on = (first_slot + 8 < p.len ? 0xffffu : 0u) | (first_slot + 9 < p.len ? 0xffff0000u : 0u);
                }
                // Two 16-dim columns at a time, so that a result's two products have others between them.
#pragma unroll
                for (int nd = 0; nd < kD / 16; nd += 2) {
                    uint32_t vf[2][4];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int slot = sw * 16 + (lane & 15), ch = (nd + i) * 2 + (lane >> 4);
                        ldsm4t(vf[i], vb + (ch / 8) * S::kHalf + slot * 128 + (((ch & 7) ^ (slot & 7)) * 16));
                        if (tail) {
                            vf[i][0] &= lo_on;
                            vf[i][1] &= hi_on;
                            vf[i][2] &= lo_on;
                            vf[i][3] &= hi_on;
                        }
                    }
#pragma unroll
                    for (int pass = 0; pass < (S::kRest ? 2 : 1); ++pass)
#pragma unroll
                        for (int mt = 0; mt < MW; ++mt)
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                mma16<T>(o[mt][2 * (nd + i)], pass ? rest[mt] : pa[mt], vf[i][0], vf[i][1]);
                                mma16<T>(o[mt][2 * (nd + i) + 1], pass ? rest[mt] : pa[mt], vf[i][2], vf[i][3]);
                            }
                }
            }
            __syncwarp();
            if (lane == 0) bar_arrive(&empty[at]);
        }
        __syncwarp();
        if (lane == 0) bar_arrive(&q_empty[turn & 1]);
        // Every warp leaves its results in shared memory, once all are through with the last tile's.
        if (turn > 0) bar_wait(&read_bar, (turn - 1) & 1, &s_gave_up);
#pragma unroll
        for (int mt = 0; mt < MW; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = mt * 16 + e * 8 + lane / 4;
                l[mt][e] += __shfl_xor_sync(0xffffffffu, l[mt][e], 1);
                l[mt][e] += __shfl_xor_sync(0xffffffffu, l[mt][e], 2);
                if (r >= rows) continue;
                if ((lane & 3) == 0) {
                    s_m[warp][r] = m[mt][e];
                    s_l[warp][r] = l[mt][e];
                }
#pragma unroll
                for (int n = 0; n < kD / 8; ++n)
                    *reinterpret_cast<float2*>(join + (warp * S::kRows + r) * S::kPad + n * 8 + (lane & 3) * 2) =
                        make_float2(o[mt][n][2 * e], o[mt][n][2 * e + 1]);
            }
        all.sync();
        const bool whole = p.b1 - p.b0 == p.n;
        float* part = whole ? nullptr : part_at<S::kRows, kD>(a, blockIdx.x, p.b0 == 0);
#pragma unroll 1
        for (int i = threadIdx.x; ok && i < rows * (kD / 4); i += S::kWarps * 32) {
            const int r = i / (kD / 4), col = i % (kD / 4) * 4;
            float top = -INFINITY, sum = 0.f;
            float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int x = 0; x < S::kWarps; ++x) top = fmaxf(top, s_m[x][r]);
            const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int x = 0; x < S::kWarps; ++x) {
                const float f = exp2_fast(s_m[x][r] - from);
                const float4 y = *reinterpret_cast<const float4*>(join + (x * S::kRows + r) * S::kPad + col);
                sum = __fmaf_rn(s_l[x][r], f, sum);
                z.x = __fmaf_rn(y.x, f, z.x);
                z.y = __fmaf_rn(y.y, f, z.y);
                z.z = __fmaf_rn(y.z, f, z.z);
                z.w = __fmaf_rn(y.w, f, z.w);
            }
            if (whole) {
                long long token;
                int head;
                row_place(ge, p, r, &token, &head);
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                store4<T>(reinterpret_cast<T*>(a.out) + token * a.out_stride + (long long)head * kD + col,
                          make_float4(z.x * inv, z.y * inv, z.z * inv, z.w * inv));
                if (col == 0 && a.lse) a.lse[token * a.n_heads + head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
            } else {
                *reinterpret_cast<float4*>(part + 2 * S::kRows + r * kD + col) = z;
                if (col == 0) {
                    part[r] = top;
                    part[S::kRows + r] = sum;
                }
            }
        }
        __syncwarp();
        if (lane == 0) bar_arrive(&read_bar);
        if (!whole) {
            all.sync();
            if (threadIdx.x == 0) s_last = parts_if_last(a, p);
            all.sync();
            if (s_last) join_parts<T, S::kRows, kD, S::kWarps>(a, ge, p, s_last, all);
        }
    }
    if (lane == 0 && *(volatile int*)&s_gave_up) flag(a.c, BAD_WAIT);  // the producer may have left before
}

// The arguments with a tile of `rows` rows at most.
AttnArgs with_tile(const AttnArgs& a, int rows) {
    AttnArgs b = a;
    b.per = rows / a.G;
    b.by_per = FastDiv::of(b.per);
    return b;
}

template <class T, int kD, int MW, int WP>
cudaError_t launch_rows(const AttnArgs& a, const CUtensorMap& km, const CUtensorMap& vm, int sms, cudaStream_t s) {
    using S = RowsShape<kD, MW, WP>;
    CUtensorMap qm;
    if (!encode_q(&qm, a, S::kRows)) return cudaErrorInvalidValue;
    auto* kernel = k_attention_rows<T, kD, MW, WP>;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(kernel, S::kSmem, &done);
    if (e != cudaSuccess) return e;
    kernel<<<sms, S::kThreads, S::kSmem, s>>>(with_tile(a, S::kRows), km, vm, qm);
    return cudaGetLastError();
}

// ---- many rows -----------------------------------------------------------------------------------------------------
//
// A chunk of new tokens: 256 rows a tile as two halves of 128, blocks of 128
// slots; the products bound the kernel, with the exponentials next to them
// (both take 1024 clocks of an SM for a half's block).  tcgen05 products,
// issued by one thread: S = Q K^T into tensor memory, and O += P V with P
// read from there.  The halves alternate: while a half's four warps (a row a thread,
// so maxima and sums need no other thread) turn S into P, the tensor cores work for the
// other.  P takes the place of S.  A half's products run in order, so S of block
// j + 1 is issued behind P V of block j without a wait, and once S is there O is
// free to be rescaled.  P has 16 bits here: its rounding's rest in a second product too (as
// for few rows) brings bf16 results from 0.0023 .. 0.0020 relative to 0.0017 .. 0.0016, the result's own
// rounding, and takes 437 us for the chunk below, 87 for prompts of 64 dims (70 without).
// 2048 new tokens over 24576 slots, 16 heads of 128: 311 us alone,
// 1.27 PFLOP/s, 76% of what a library product reaches in a burst; for seconds on end 371 us (1.07, 77% of
// what the product holds for seconds; the power limit has the clock at 1.54 GHz); a fresh prompt of 4096 tokens 81 us (0.85 PFLOP/s counting what is
// masked as not done).  A steady block takes 3200 clocks for both halves where the products
// alone take 2048: a half's chain from S over its maximum (450) and exponentials (1540) to P
// and the next S is as long as that.
constexpr int kTileRows2 = 256;
constexpr int kTileBlock = 128;
constexpr int kTileThreads = 384;  // warps 0-3 and 4-7: the halves; 8: products; 9, 10: copies; 11: what has arrived
// Registers: 168 a thread at launch; a half's threads hold a row of 128 scores,
// so the other four warps give theirs up: 256 x 224 + 128 x 56 = 384 x 168.
constexpr int kHalfRegs = 224, kOtherRegs = 56;
constexpr int kTileEntries = 4;    // ring of K and V blocks, in turn
constexpr int kBadRing = 16;       // blocks whose bad-page bits are kept

template <int kD>
struct TileShape {
    static constexpr int kPart = kTileBlock * 128;        // bytes of 128 rows x 64 dims
    static constexpr int kEntry = (kD / 64) * kPart;      // one K or V block, or one half's q
    static constexpr int kSmem = 1024 + (kTileEntries + 2) * kEntry;
};

template <class T, int kD>
__global__ void __launch_bounds__(kTileThreads, 1)
    k_attention_tiles(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                      const __grid_constant__ CUtensorMap q_map) {
    using S = TileShape<kD>;
    constexpr int kParts = kD / 64;
    constexpr bool kBf16 = !std::is_same<T, __half>::value;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[kTileEntries], empty[kTileEntries], q_full[2], q_empty, s_full[2], p_full[2][2], o_full[2], all_bar, drained;
    __shared__ PartRing<kPartRing> parts;
    __shared__ long long s_scan[16];
    __shared__ int s_bad[kBadRing];  // bit 0, 1: the block's pages that are masked
    __shared__ int s_gave_up, s_last;
    __shared__ uint32_t s_tmem;
    const uint32_t ring = (smem_u32(smem_raw) + 1023) & ~1023u;
    const uint32_t q_at = ring + kTileEntries * S::kEntry;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // A half has as many whole tokens as 128 rows hold.
    const int G = a.G, per = a.per / 2, live = per * G;
    const Geometry ge = geometry(a, kTileBlock, kTilesExtra);
    if (threadIdx.x == 0) {
        for (int i = 0; i < kTileEntries; ++i) {
            bar_init(&full[i], 1);
            bar_init(&empty[i], 1);
        }
        for (int h = 0; h < 2; ++h) {
            bar_init(&q_full[h], 1);
            bar_init(&s_full[h], 1);
            bar_init(&p_full[h][0], h == 0 ? 5 : 4);
            bar_init(&p_full[h][1], 4);
            bar_init(&o_full[h], 1);
        }
        bar_init(&q_empty, 1);
        bar_init(&all_bar, 8);
        bar_init(&drained, 1);
        parts.init(11);
        s_gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == 9 * 32) {
        tma_prefetch(&k_map);
        tma_prefetch(&v_map);
        tma_prefetch(&q_map);
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;  // S of the halves at 0 and 128, O at 256 and 384
    const Line line = find_line<kTileThreads, CutRows>(a, ge, kTilesMinUnits, s_scan, warp == 9);

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        Part p;
        if (warp == 9) {
            // K and V blocks, in turn.
            Walk<CutRows> walk(a, ge, line);
            int e = 0, round = 0, slot = 0;
            unsigned turn = 0;
            bool ok = true;
            while (ok && walk.next(&p)) {
                if (!parts.put(turn, p, &s_gave_up)) break;
                ++turn;
                for (int b0 = p.b0; ok && b0 < p.b1; b0 += 16) {
                    // 32 pages, one a lane; no page there: the box past the pool, which reads as 0.
                    const int at = b0 * 2 + lane;
                    int mine = -1;
                    if (at < p.b1 * 2 && (long long)at * kPage < p.len) mine = page_of(a.c, p.seq, at);
                    for (int b = b0; ok && b < min(p.b1, b0 + 16); ++b) {
                        const int pg0 = __shfl_sync(0xffffffffu, mine, 2 * (b - b0)), pg1 = __shfl_sync(0xffffffffu, mine, 2 * (b - b0) + 1);
#pragma unroll
                        for (int kv = 0; kv < 2; ++kv) {
                            if (round > 0 && !bar_wait(&empty[e], (round - 1) & 1, &s_gave_up)) {
                                ok = false;
                                break;
                            }
                            if (lane == 0) {
                                if (kv == 0) s_bad[slot] = (pg0 < 0 ? 1 : 0) | (pg1 < 0 ? 2 : 0);
                                bar_expect(&full[e], S::kEntry);
                                const uint32_t dst = ring + e * S::kEntry;
                                const CUtensorMap* map = kv ? &v_map : &k_map;
#pragma unroll
                                for (int h = 0; h < kParts; ++h) {
                                    tma_load_4d(dst + h * S::kPart, map, h * 64, 0, p.head, pg0 < 0 ? a.c.n_pages : pg0, &full[e]);
                                    tma_load_4d(dst + h * S::kPart + kPage * 128, map, h * 64, 0, p.head, pg1 < 0 ? a.c.n_pages : pg1, &full[e]);
                                }
                            }
                            __syncwarp();
                            if (++e == kTileEntries) e = 0, ++round;
                        }
                        slot = (slot + 1) % kBadRing;
                    }
                }
            }
            p.n = 0;
            if (a.c.n_seq > 0) parts.put(turn, p, &s_gave_up);
            #pragma unroll 1
            for (int i = 0; i < kTileEntries; ++i) {  // every copy has landed before the CTA ends
                const int fills = round + (i < e ? 1 : 0);
                volatile int none = 0;
                if (fills > 0) bar_wait(&full[i], (fills - 1) & 1, &none);
            }
        } else if (warp == 10) {
            // q rows: the next tile's as soon as the last product with this one's is done.
            int fills[2] = {0, 0};
            for (unsigned turn = 0; parts.get(turn, &p, &s_gave_up); ++turn) {
                if (turn > 0 && !bar_wait(&q_empty, (turn - 1) & 1, &s_gave_up)) break;
                const int halves = p.n_new > (2 * p.tile + 1) * per ? 2 : 1;
                for (int h = 0; h < halves; ++h) {
                    if (lane == 0) {
                        bar_expect(&q_full[h], live * kD * 2);
#pragma unroll
                        for (int i = 0; i < kParts; ++i)
                            tma_load_3d(q_at + h * S::kEntry + i * S::kPart, &q_map, i * 64, p.head * G, p.tok0 + (2 * p.tile + h) * per, &q_full[h]);
                    }
                    ++fills[h];
                }
            }
            volatile int none = 0;
            for (int h = 0; h < 2; ++h)
                if (fills[h] > 0) bar_wait(&q_full[h], (fills[h] - 1) & 1, &none);
        } else if (warp == 8) {
            const uint32_t kQk = tc_instr(kBf16, kTileBlock, false) | (a.scale < 0.f ? kNegateA : 0u);
            constexpr uint32_t kPv = tc_instr(kBf16, kD, true);
            const uint32_t t_at = uniform(tmem), q_lo = uniform(desc_lo_k(q_at)), k_lo = uniform(desc_lo_k(ring)),
                           v_lo = uniform(desc_lo_mn(ring, S::kPart));
            int e = 0;
            unsigned phase = 0, q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
            auto qk = [&](int h, int entry) {
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < kD / 16; ++kk) {
                        const uint32_t off = ((kk / 4) * S::kPart + (kk % 4) * 32) / 16;
                        tc_mma_ss(t_at + h * 128, q_lo + h * (S::kEntry / 16) + off, k_lo + entry * (S::kEntry / 16) + off, kQk, kk > 0);
                    }
                    tc_commit(&s_full[h]);
                }
                __syncwarp();
            };
            auto next_entry = [&]() {
                const int at = e;
                if (++e == kTileEntries) e = 0, phase ^= 1;
                return at;
            };
            // A wait that ends early is not looked at: the products then run over what is there, and the call's results are
            // void anyway.  (A vote after each wait cost 45 clocks of the some 250 that queued products hide.)
            for (unsigned turn = 0; __all_sync(0xffffffffu, parts.get(turn, &p, &s_gave_up)); ++turn) {
                const int b0 = uniform(p.b0), b1 = uniform(p.b1);
                const int halves = uniform(p.n_new > (2 * p.tile + 1) * per ? 2 : 1);
                for (int h = 0; h < halves; ++h) {
                    bar_wait(&q_full[h], q_phase[h], &s_gave_up);
                    q_phase[h] ^= 1;
                }
                bar_wait(&full[e], phase, &s_gave_up);
                const int ke = next_entry();
                tc_fence_after();
                qk(0, ke);
                if (halves == 2) qk(1, ke);
                if (elect_one()) {
                    tc_commit(&empty[ke]);
                    if (b1 - b0 == 1) tc_commit(&q_empty);
                }
                __syncwarp();
                for (int b = b0; b < b1; ++b) {
                    const bool more = b + 1 < b1;
                    const int v_at = next_entry(), k_at = more ? next_entry() : 0;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (h >= halves) break;
                        // P comes as three quarters of the block's slots and the last one: the first products hide its making,
                        // and few are left before the next S (halves: 70.8 us for the prompts against 69.8).
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            bar_wait(&p_full[h][g], p_phase[h], &s_gave_up);
                            tc_fence_after();
                            if (elect_one()) {
#pragma unroll
                                for (int kk = g * 6; kk < 6 + 2 * g; ++kk)
                                    tc_mma_ts(t_at + 256 + h * 128, t_at + h * 128 + kk * 8, v_lo + v_at * (S::kEntry / 16) + kk * (2048 / 16),
                                              kPv, b > b0 || kk > 0);
                                if (g == 1 && !more) tc_commit(&o_full[h]);
                            }
                            __syncwarp();
                        }
                        p_phase[h] ^= 1;
                        if (more) qk(h, k_at);
                    }
                    if (elect_one()) {
                        tc_commit(&empty[v_at]);
                        if (more) tc_commit(&empty[k_at]);
                        if (b + 2 == b1) tc_commit(&q_empty);
                    }
                    __syncwarp();
                }
            }
            // Nothing that was issued is left running.
            volatile int none = 0;
            if (elect_one()) tc_commit(&drained);
            __syncwarp();
            bar_wait(&drained, 0, &none);
        } else {
            // A block's V and the next one's K: that they are there counts as part of the first half's P, so the products'
            // warp has one wait for both (two more of its own left the tensor cores idle for 400 clocks a block).
            int e = 0;
            unsigned phase = 0, p_phase = 0;
            bool ok = true;
            auto next_entry = [&](bool wait) {
                if (wait) ok = ok && bar_wait(&full[e], phase, &s_gave_up);
                if (++e == kTileEntries) e = 0, phase ^= 1;
            };
            for (unsigned turn = 0; ok && parts.get(turn, &p, &s_gave_up); ++turn) {
                // The first K: the products' warp waits for it, and may have given it back, and seen it filled again, before
                // this warp comes by.  The others are not given back without this warp's arrival.
                next_entry(false);
                for (int b = p.b0; ok && b < p.b1; ++b) {
                    const int ve = e;
                    next_entry(true);
                    if (ok && (b + 1) * kTileBlock > p.len) {
                        // V at or behind the sequence's end may hold anything: 0 there, since 0 * NaN is NaN.
                        const int from = max(0, p.len - b * kTileBlock);
                        uint8_t* v = smem_raw + (ring - smem_u32(smem_raw)) + ve * S::kEntry;
                        for (int i = lane; i < kParts * (kTileBlock - from) * 8; i += 32) {
                            const int h = i / ((kTileBlock - from) * 8), j = i % ((kTileBlock - from) * 8);
                            *reinterpret_cast<uint4*>(v + h * S::kPart + from * 128 + j * 16) = make_uint4(0, 0, 0, 0);
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    if (b + 1 < p.b1) next_entry(true);
                    __syncwarp();
                    if (lane == 0) bar_arrive(&p_full[0][0]);
                    ok = ok && bar_wait(&p_full[0][0], p_phase, &s_gave_up);  // not twice in one phase
                    p_phase ^= 1;
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kHalfRegs));
        const int half = warp >> 2, in_half = (warp & 3) * 32 + lane;
        const int r = in_half < live ? half * live + in_half : kTileRows2;  // the tile's row, or none
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + lanes + half * 128, t_o = tmem + lanes + 256 + half * 128;
        const float to_log2 = fmaxf(fabsf(a.scale), 1e-37f) * kLog2e;  // above 0: a masked -inf stays -inf
        SyncPoint all{&all_bar, 0, &s_gave_up};
        unsigned s_phase = 0, o_phase = 0;
        int slot = 0;
        Part p;
        for (unsigned turn = 0; parts.get(turn, &p, &s_gave_up); ++turn) {
            const int base = p.len - p.n_new;
            const bool mine = half == 0 || p.n_new > (2 * p.tile + 1) * per;
            const bool whole = p.b1 - p.b0 == p.n;
            if (mine) {
                bool ok = true;
                float m = -INFINITY, l = 0.f;
                const int first = (2 * p.tile + half) * per;  // the half's first token
                const int sees = min(first + ge.by_G(in_half), p.n_new - 1) + base + 1;
                const int least = first + base + 1;           // slots that every row of the half sees
                for (int b = p.b0; b < p.b1; ++b) {
                    if (!bar_wait(&s_full[half], s_phase, &s_gave_up)) {
                        ok = false;
                        break;
                    }
                    s_phase ^= 1;
                    tc_fence_after();
                    float s[128];
                    tmem_ld32<0>(s, t_s);
                    tmem_ld32<32>(s, t_s + 32);
                    tmem_ld32<64>(s, t_s + 64);
                    tmem_ld32<96>(s, t_s + 96);
                    tmem_wait_ld();
                    const int bad = s_bad[slot];
                    slot = (slot + 1) % kBadRing;
                    const int s0 = b * kTileBlock;
                    if (s0 + kTileBlock > least || bad) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int n = sees - s0 - c * 32;  // slots of these 32 that the row sees
                            unsigned on = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1;
                            if ((bad >> (c / 2)) & 1) on = 0u;
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (!((on >> i) & 1)) s[c * 32 + i] = -INFINITY;
                        }
                    }
                    // A NaN is no maximum, but its exponential makes the row's sum NaN.
                    float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                    for (int i = 4; i < 124; i += 8)
#pragma unroll
                        for (int j = 0; j < 4; ++j) top[j] = fmaxf(fmaxf(top[j], s[i + j]), s[i + 4 + j]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) top[j] = fmaxf(top[j], s[124 + j]);
                    top[0] = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                    const float reach = top[0] * to_log2;
                    const bool grown = reach > m + (8.f + kLift<T>);
                    if (__any_sync(0xffffffffu, grown)) {
                        const float to = grown ? reach - kLift<T> : m;  // a row goes by its own scores alone
                        const float f = to == -INFINITY ? 1.f : exp2_fast(m - to);
                        m = to;
                        l *= f;
                        if (b > p.b0) {
#pragma unroll 1
                            for (int c = 0; c < kD / 32; ++c) {
                                float o[32];
                                tmem_ld32<0>(o, t_o + c * 32);
                                tmem_wait_ld();
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] *= f;
                                tmem_st32<0>(t_o + c * 32, o);
                            }
                        }
                    }
                    const float2 by = make_float2(to_log2, to_log2);
                    const float less = m == -INFINITY ? 0.f : -m;
                    const float2 from = make_float2(less, less);
                    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t pk[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            float2 x = __ffma2_rn(make_float2(s[c * 32 + 2 * i], s[c * 32 + 2 * i + 1]), by, from);
                            x.x = exp2_fast(x.x);
                            x.y = exp2_fast(x.y);
                            sum[i & 1] = __fadd2_rn(sum[i & 1], x);
                            pk[i] = pack2<T>(x.x, x.y);
                        }
                        tmem_st16<0>(t_s + c * 16, pk);
                        if (c >= 2) {
                            tmem_wait_st();
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) bar_arrive(&p_full[half][c - 2]);
                        }
                    }
                    l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                }
                long long token = 0;
                int head = 0;
                const bool row = row_place(ge, p, r, &token, &head);
                const float inv = l == 0.f ? 0.f : 1.f / l;
                T* out = reinterpret_cast<T*>(a.out) + token * a.out_stride + (long long)head * kD;
                float* part = whole ? nullptr : part_at<kTileRows2, kD>(a, blockIdx.x, p.b0 == 0);
                if (ok && row && whole && a.lse) a.lse[token * a.n_heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
                if (ok && row && !whole) {
                    part[r] = m;
                    part[kTileRows2 + r] = l;
                    part += 2 * kTileRows2 + r * kD;
                }
                if (ok && bar_wait(&o_full[half], o_phase, &s_gave_up)) {
                    o_phase ^= 1;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < kD / 32; ++c) {
                        float o[32];
                        tmem_ld32<0>(o, t_o + c * 32);
                        tmem_wait_ld();
                        if (!row) continue;
                        if (whole) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float x[8];
#pragma unroll
                                for (int k = 0; k < 8; ++k) x[k] = o[i * 8 + k] * inv;
                                store_vec<T, 8>(out + c * 32 + i * 8, x);
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                *reinterpret_cast<float4*>(part + c * 32 + i * 4) = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                        }
                    }
                }
            } else {
                slot = (slot + p.b1 - p.b0) % kBadRing;
            }
            if (!whole) {
                all.sync();
                if (threadIdx.x == 0) s_last = parts_if_last(a, p);
                all.sync();
                if (s_last) join_parts<T, kTileRows2, kD, 8>(a, ge, p, s_last, all);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && s_gave_up) flag(a.c, BAD_WAIT);
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// A tile is two halves of whole tokens.
AttnArgs two_halves(const AttnArgs& a) {
    AttnArgs b = a;
    b.per = 2 * (128 / a.G);
    b.by_per = FastDiv::of(b.per);
    return b;
}

template <class T, int kD>
cudaError_t launch_tiles(const AttnArgs& a, const CUtensorMap& km, const CUtensorMap& vm, int sms, cudaStream_t s) {
    CUtensorMap qm;
    if (!encode_q(&qm, a, 128)) return cudaErrorInvalidValue;
    auto* kernel = k_attention_tiles<T, kD>;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(kernel, TileShape<kD>::kSmem, &done);
    if (e != cudaSuccess) return e;
    kernel<<<sms, kTileThreads, TileShape<kD>::kSmem, s>>>(two_halves(a), km, vm, qm);
    return cudaGetLastError();
}

// ---- weights, few rows ---------------------------------------------------------------------------------------------
//
// weight[slot] += sum over rows exp2(s - lse log2 e), s formed again: K is read
// a second time (from L2 as far as it still lies there), V is not.  As above, a
// set of four warps takes a page, 16 slots a warp, two sets in turn; a thread adds its rows' probabilities of
// its columns, and eight lanes' sums make a slot's.  All rows of a (sequence, KV head)
// pass over the part's pages 64 at a time, so nothing is joined between CTAs.
// Eight ragged sequences of 1 .. 8 new tokens, 64 .. 27000 slots: 36 us for 154 MB of K, 68 us with
// a decay (the old weights are read where the new ones are written, by the warps that hold the page).
constexpr int kWRows = 64;
constexpr int kWWarps = 8, kWThreads = (kWWarps + 1) * 32;

template <int kD>
struct WRowsShape {
    static constexpr int kStage = (kD / 64) * kPage * 128;
    static constexpr int kQ = kWRows * kD * 2;
    static constexpr int kStages = 10;  // even: a stage falls to one set of warps
    static constexpr int kSmem = 1024 + kStages * kStage + 2 * kQ;
};

template <class T, int kD>
__global__ void __launch_bounds__(kWThreads, 1)
    k_weights_rows(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap q_map) {
    using S = WRowsShape<kD>;
    constexpr int kParts = kD / 64, kHalf = kPage * 128;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[S::kStages], empty[S::kStages], q_full[2], q_empty[2], all_bar;
    __shared__ PartRing<kPartRing> parts;
    __shared__ int s_page[S::kStages];
    __shared__ long long s_scan[16];
    __shared__ float s_lse[2][kWRows];
    __shared__ int s_gave_up;
    const uint32_t ring = (smem_u32(smem_raw) + 1023) & ~1023u;
    const uint32_t q_at = ring + S::kStages * S::kStage;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.G, per = a.per, live = per * G;  // tokens and rows that pass at once
    const Geometry ge = geometry(a, kPage, 1);
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kStages; ++i) {
            bar_init(&full[i], 1);
            bar_init(&empty[i], 4);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(&q_full[i], 1);
            bar_init(&q_empty[i], kWWarps);
        }
        bar_init(&all_bar, kWWarps);
        parts.init(kWWarps);
        s_gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == kWWarps * 32) {
        tma_prefetch(&k_map);
        tma_prefetch(&q_map);
    }
    __syncthreads();
    const Line line = find_line<kWThreads, CutPages>(a, ge, kRowsMinUnits, s_scan, warp == kWWarps);
    Part p;
    if (warp == kWWarps) {
        Walk<CutPages> walk(a, ge, line);
        int st = 0, round = 0;
        unsigned turn = 0, pass = 0;
        bool ok = true;
        while (ok && walk.next(&p)) {
            if (!parts.put(turn, p, &s_gave_up)) break;
            ++turn;
            for (int t0 = 0; ok && t0 < p.n_new; t0 += per) {
                const int qb = pass & 1;
                if (pass >= 2 && !bar_wait(&q_empty[qb], ((pass >> 1) - 1) & 1, &s_gave_up)) {
                    ok = false;
                    break;
                }
#pragma unroll
                for (int i = 0; i < kWRows / 32; ++i) {
                    const int r = i * 32 + lane, tok = t0 + ge.by_G(r);
                    float x = INFINITY;  // exp2(s - inf) = 0: no row, or one that sees nothing
                    if (r < live && tok < p.n_new) {
                        x = a.lse[(long long)(p.tok0 + tok) * a.n_heads + p.head * G + r - ge.by_G(r) * G] * kLog2e;
                        if (x == -INFINITY) x = INFINITY;
                    }
                    s_lse[qb][r] = x;
                }
                __syncwarp();
                if (lane == 0) {
                    bar_expect(&q_full[qb], live * kD * 2);
#pragma unroll
                    for (int h = 0; h < kParts; ++h)
                        tma_load_3d(q_at + qb * S::kQ + h * (kWRows * 128), &q_map, h * 64, p.head * G, p.tok0 + t0, &q_full[qb]);
                }
                ++pass;
                for (int b0 = p.b0; ok && b0 < p.b1; b0 += 32) {
                    const int mine = b0 + lane < p.b1 ? page_of(a.c, p.seq, b0 + lane) : -1;
                    for (int b = b0; b < min(p.b1, b0 + 32); ++b) {
                        const int page = __shfl_sync(0xffffffffu, mine, b - b0);
                        if (round > 0 && !bar_wait(&empty[st], (round - 1) & 1, &s_gave_up)) {
                            ok = false;
                            break;
                        }
                        if (lane == 0) {
                            s_page[st] = page;
                            if (page < 0) {
                                bar_arrive(&full[st]);
                            } else {
                                bar_expect(&full[st], S::kStage);
#pragma unroll
                                for (int h = 0; h < kParts; ++h)
                                    tma_load_4d(ring + st * S::kStage + h * kHalf, &k_map, h * 64, 0, p.head, page, &full[st]);
                            }
                        }
                        __syncwarp();
                        if (++st == S::kStages) st = 0, ++round;
                    }
                }
            }
        }
        p.n = 0;
        if (a.c.n_seq > 0) parts.put(turn, p, &s_gave_up);
        volatile int none = 0;
        #pragma unroll 1
        for (int i = 0; i < S::kStages; ++i) {
            const int fills = round + (i < st ? 1 : 0);
            if (fills > 0) bar_wait(&full[i], (fills - 1) & 1, &none);
        }
        #pragma unroll 1
        for (int i = 0; i < 2; ++i) {
            const int fills = (pass + 1 - i) / 2;
            if (fills > 0) bar_wait(&q_full[i], (fills - 1) & 1, &none);
        }
        if (lane == 0 && s_gave_up) flag(a.c, BAD_WAIT);
        return;
    }
    const int wp = warp >> 2, sw = warp & 3;
    const float to_log2 = a.scale * kLog2e;
    SyncPoint all{&all_bar, 0, &s_gave_up};
    int st = 0, mine = 0;
    unsigned phase = 0, pass = 0;
    bool ok = true;
    for (unsigned turn = 0; ok && parts.get(turn, &p, &s_gave_up); ++turn) {
        const int base = p.len - p.n_new;
        for (int t0 = 0; ok && t0 < p.n_new; t0 += per, ++pass) {
            if (t0 > 0) all.sync();  // another set's warps may have left these slots' sums
            const int qb = pass & 1;
            const int rows = min(per, p.n_new - t0) * G, tiles = (rows + 15) / 16;
            ok = bar_wait(&q_full[qb], (pass >> 1) & 1, &s_gave_up);
            const uint32_t qa = q_at + qb * S::kQ;
            for (int b = p.b0; ok && b < p.b1; ++b) {
                const bool here = mine == wp;
                const int at = st;
                const unsigned parity = phase;
                if (++st == S::kStages) st = 0, phase ^= 1;
                mine ^= 1;
                if (!here) continue;
                if (!bar_wait(&full[at], parity, &s_gave_up)) {
                    ok = false;
                    break;
                }
                const int s0 = b * kPage + sw * 16, page = s_page[at];
                if (page >= 0 && s0 < p.len) {
                    const uint32_t kb = ring + at * S::kStage;
                    uint32_t kf[kD / 16][4];
#pragma unroll
                    for (int kk = 0; kk < kD / 16; ++kk) {
                        const int slot = sw * 16 + ((lane >> 4) << 3) + (lane & 7), ch = kk * 2 + ((lane >> 3) & 1);
                        ldsm4(kf[kk], kb + (ch / 8) * kHalf + slot * 128 + (((ch & 7) ^ (slot & 7)) * 16));
                    }
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
                    for (int mt = 0; mt < tiles; ++mt) {
                        float s[2][4];
#pragma unroll
                        for (int n = 0; n < 2; ++n)
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
                        for (int kk = 0; kk < kD / 16; ++kk) {
                            uint32_t qf[4];
                            const int r = mt * 16 + (lane & 15), qc = kk * 2 + (lane >> 4);
                            ldsm4(qf, qa + (qc / 8) * (kWRows * 128) + r * 128 + (((qc & 7) ^ (r & 7)) * 16));
                            mma16<T>(s[0], qf, kf[kk][0], kf[kk][1]);
                            mma16<T>(s[1], qf, kf[kk][2], kf[kk][3]);
                        }
                        const bool mask = s0 + 16 > base + t0 + ge.by_G(mt * 16) + 1 || mt * 16 + 16 > rows;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int r = mt * 16 + (e >> 1) * 8 + lane / 4;
                            const float less = s_lse[qb][r];
                            const int sees = !mask ? INT_MAX : r < rows ? base + t0 + ge.by_G(r) + 1 : 0;
#pragma unroll
                            for (int n = 0; n < 2; ++n) {
                                const float x = exp2_fast(__fmaf_rn(s[n][e], to_log2, -less));
                                sum[n * 2 + (e & 1)] += s0 + n * 8 + (lane & 3) * 2 + (e & 1) < sees ? x : 0.f;
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 4);
                        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 8);
                        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 16);
                    }
                    if (lane < 4) {
                        float* to = a.c.weight + ((long long)page * a.c.n_kv + p.head) * kPage + sw * 16;
                        const float decay = t0 == 0 ? a.decay : 1.f;  // later rows add to what the first ones left
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int off = (i >> 1) * 8 + lane * 2 + (i & 1);
                            if (s0 + off < p.len) to[off] = decay == 0.f ? sum[i] : __fmaf_rn(decay, to[off], sum[i]);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) bar_arrive(&empty[at]);
            }
            __syncwarp();
            if (lane == 0) bar_arrive(&q_empty[qb]);
        }
    }
    if (lane == 0 && *(volatile int*)&s_gave_up) flag(a.c, BAD_WAIT);
}

// ---- weights, many rows --------------------------------------------------------------------------------------------
//
// S^T = K Q^T: a thread has one slot's scores against 128 rows, so a slot's sum is
// one thread's.  A tile of 256 slots (two halves of 128, four warps each) stays in
// shared memory while the rows that see it stream past, 128 / G whole tokens at a time
// with their log-sums; S is double-buffered in tensor memory, so the products run
// ahead.  The exponentials bound it: one for each product of 128 dims.  2048 new
// tokens over 24576 slots, 16 heads: 255 .. 300 us by the clock that the power limit leaves
// (0.77 .. 0.66 PFLOP/s; for seconds on end 274); 768 tiles on 148 SMs leave a seventh of that idle.  Tiles of 128 slots whose rows the halves take in turn: a
// fresh prompt of 4096 tokens 83 us instead of 115, this chunk 262, 128 rows over 8192 slots 27 instead of 19.
constexpr int kWTileSlots = 256, kWTileRows = 128;
constexpr int kWEntries = 2;  // ring of row tiles
// Of eight pairs of exponentials, those that go to the FMA units (the polynomial
// above) and not to the special function units: the long chunk takes 274 us with none,
// 256 with 1, 255 with 2, 269 with 3, 322 with 4.
constexpr int kPolyOf8 = 2;
constexpr int kWLse = 4;      // ring of their log-sums

template <int kD>
struct WTileShape {
    static constexpr int kPart = 128 * 128;
    static constexpr int kEntry = (kD / 64) * kPart;
    static constexpr int kSmem = 1024 + (4 + kWEntries) * kEntry;  // two tiles of slots (the next one arrives early)
};

template <class T, int kD>
__global__ void __launch_bounds__(kTileThreads, 1)
    k_weights_tiles(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap q_map) {
    using S = WTileShape<kD>;
    constexpr int kParts = kD / 64;
    constexpr bool kBf16 = !std::is_same<T, __half>::value;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t k_full[2], k_empty[2], q_full[kWEntries], q_empty[kWEntries], l_full[kWLse], l_empty[kWLse], s_full[2][2], s_empty[2][2],
        drained;
    __shared__ PartRing<kPartRing> parts;
    __shared__ long long s_scan[16];
    __shared__ __align__(16) float s_less[kWLse][kWTileRows];  // - lse log2 e; -inf adds nothing
    __shared__ int s_sees[kWLse][kWTileRows];                  // slots that the row sees
    __shared__ int s_nan[kWLse];                               // slots that a row sees whose log-sum is NaN
    __shared__ int s_gave_up;
    __shared__ uint32_t s_tmem;
    const uint32_t k_at = (smem_u32(smem_raw) + 1023) & ~1023u;
    const uint32_t q_at = k_at + 4 * S::kEntry;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.G, per = a.per, live = per * G;  // tokens and rows of a row tile
    const Geometry ge = geometry(a, kWTileSlots, 0);
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            bar_init(&k_full[i], 1);
            bar_init(&k_empty[i], 1);
            for (int j = 0; j < 2; ++j) {
                bar_init(&s_full[i][j], 1);
                bar_init(&s_empty[i][j], 4);
            }
        }
        for (int i = 0; i < kWEntries; ++i) {
            bar_init(&q_full[i], 1);
            bar_init(&q_empty[i], 1);
        }
        for (int i = 0; i < kWLse; ++i) {
            bar_init(&l_full[i], 32);
            bar_init(&l_empty[i], 8);
        }
        bar_init(&drained, 1);
        parts.init(10);
        s_gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // Rows past live are never written by a copy: 0, once.
    {
        uint8_t* q = smem_raw + (q_at - smem_u32(smem_raw));
        for (int i = threadIdx.x; i < kWEntries * S::kEntry / 16; i += kTileThreads) reinterpret_cast<uint4*>(q)[i] = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (threadIdx.x == 9 * 32) {
        tma_prefetch(&k_map);
        tma_prefetch(&q_map);
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    const Line line = find_line<kTileThreads, CutSlots>(a, ge, kTilesMinUnits, s_scan, warp == 9);
    Part p;
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == 9) {
            // Copies: a tile of slots, then the row tiles that see it.
            Walk<CutSlots, true> walk(a, ge, line);
            int e = 0, round = 0, kt = 0;
            unsigned turn = 0;
            bool ok = true;
            while (ok && walk.next(&p)) {
                if (!parts.put(turn, p, &s_gave_up)) break;
                ++turn;
                const int kb = kt & 1;
                if (kt >= 2 && !bar_wait(&k_empty[kb], ((kt >> 1) - 1) & 1, &s_gave_up)) break;
                int page = -1;
                if (lane < 4 && (long long)p.tile * kWTileSlots + lane * kPage < p.len) page = page_of(a.c, p.seq, p.tile * 4 + lane);
                if (lane == 0) bar_expect(&k_full[kb], 2 * S::kEntry);
                for (int i = 0; i < 4; ++i) {
                    const int pg = __shfl_sync(0xffffffffu, page, i);
                    if (lane == 0)
#pragma unroll
                        for (int h = 0; h < kParts; ++h)
                            tma_load_4d(k_at + (2 * kb + i / 2) * S::kEntry + h * S::kPart + (i % 2) * kPage * 128, &k_map, h * 64, 0, p.head,
                                        pg < 0 ? a.c.n_pages : pg, &k_full[kb]);
                }
                ++kt;
                const int q0 = CutSlots::first(SeqWork{p.len, 0, p.n_new}, ge, p.tile);
                for (int b = 0; b < p.n; ++b) {
                    if (round > 0 && !bar_wait(&q_empty[e], (round - 1) & 1, &s_gave_up)) {
                        ok = false;
                        break;
                    }
                    if (lane == 0) {
                        bar_expect(&q_full[e], live * kD * 2);
#pragma unroll
                        for (int h = 0; h < kParts; ++h)
                            tma_load_3d(q_at + e * S::kEntry + h * S::kPart, &q_map, h * 64, p.head * G, p.tok0 + (q0 + b) * per, &q_full[e]);
                    }
                    __syncwarp();
                    if (++e == kWEntries) e = 0, ++round;
                }
            }
            p.n = 0;
            if (a.c.n_seq > 0) parts.put(turn, p, &s_gave_up);
            volatile int none = 0;
            #pragma unroll 1
            for (int i = 0; i < kWEntries; ++i) {
                const int fills = round + (i < e ? 1 : 0);
                if (fills > 0) bar_wait(&q_full[i], (fills - 1) & 1, &none);
            }
            #pragma unroll 1
            for (int i = 0; i < 2; ++i) {
                const int fills = (kt + 1 - i) / 2;
                if (fills > 0) bar_wait(&k_full[i], (fills - 1) & 1, &none);
            }
        } else if (warp == 10) {
            // The row tiles' log-sums and limits.
            int e = 0, round = 0;
            bool ok = true;
            for (unsigned turn = 0; ok && parts.get(turn, &p, &s_gave_up); ++turn) {
                const int q0 = CutSlots::first(SeqWork{p.len, 0, p.n_new}, ge, p.tile), base = p.len - p.n_new;
                for (int b = 0; b < p.n; ++b) {
                    if (round > 0 && !bar_wait(&l_empty[e], (round - 1) & 1, &s_gave_up)) {
                        ok = false;
                        break;
                    }
                    unsigned nan = 0;
#pragma unroll
                    for (int i = 0; i < kWTileRows / 32; ++i) {
                        const int r = i * 32 + lane, tok = (q0 + b) * per + ge.by_G(r);
                        float less = 0.f;
                        int sees = 0;
                        if (r < live && tok < p.n_new) {
                            const float x = -a.lse[(long long)(p.tok0 + tok) * a.n_heads + p.head * G + r - ge.by_G(r) * G] * kLog2e;
                            sees = base + tok + 1;
                            // No slot (lse -inf: none at all, or bad pages only) and NaN: -inf, for a masked score's -inf plus
                            // either would be NaN where the row sees nothing.  What a NaN row does see becomes NaN at the end.
                            less = x < INFINITY ? x : -INFINITY;
                            if (isnan(x)) nan = max(nan, (unsigned)max(sees, 0));
                        }
                        s_less[e][r] = less;
                        s_sees[e][r] = sees;
                    }
                    nan = __reduce_max_sync(0xffffffffu, nan);
                    if (lane == 0) s_nan[e] = (int)nan;
                    bar_arrive(&l_full[e]);
                    if (++e == kWLse) e = 0, ++round;
                }
            }
        } else if (warp == 8) {
            const uint32_t kInstr = tc_instr(kBf16, kWTileRows, false) | (a.scale < 0.f ? kNegateA : 0u);
            const uint32_t t_at = uniform(tmem), k_lo = uniform(desc_lo_k(k_at)), q_lo = uniform(desc_lo_k(q_at));
            int e = 0, kt = 0, buf = 0;
            unsigned phase = 0, s_phase = 1;  // the first wait for an empty S passes
            // A wait that ends early is not looked at, as above.
            for (unsigned turn = 0; __all_sync(0xffffffffu, parts.get(turn, &p, &s_gave_up)); ++turn) {
                const int kb = kt & 1, n = uniform(p.n);
                bar_wait(&k_full[kb], (kt >> 1) & 1, &s_gave_up);
                for (int b = 0; b < n; ++b) {
                    bar_wait(&q_full[e], phase, &s_gave_up);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        bar_wait(&s_empty[h][buf], s_phase, &s_gave_up);
                        tc_fence_after();
                        if (elect_one()) {
#pragma unroll
                            for (int kk = 0; kk < kD / 16; ++kk) {
                                const uint32_t off = ((kk / 4) * S::kPart + (kk % 4) * 32) / 16;
                                tc_mma_ss(t_at + (h * 2 + buf) * 128, k_lo + (2 * kb + h) * (S::kEntry / 16) + off,
                                          q_lo + e * (S::kEntry / 16) + off, kInstr, kk > 0);
                            }
                            tc_commit(&s_full[h][buf]);
                        }
                        __syncwarp();
                    }
                    if (elect_one()) tc_commit(&q_empty[e]);
                    __syncwarp();
                    if (++e == kWEntries) e = 0, phase ^= 1;
                    buf ^= 1;
                    if (buf == 0) s_phase ^= 1;
                }
                if (elect_one()) tc_commit(&k_empty[kb]);
                __syncwarp();
                ++kt;
            }
            volatile int none = 0;
            if (elect_one()) tc_commit(&drained);
            __syncwarp();
            bar_wait(&drained, 0, &none);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kHalfRegs));
        const int half = warp >> 2;
        const uint32_t t_s = tmem + ((uint32_t)((warp & 3) * 32) << 16) + half * 256;
        const float to_log2 = fmaxf(fabsf(a.scale), 1e-37f) * kLog2e;  // above 0: a masked -inf stays -inf
        const float2 by = make_float2(to_log2, to_log2);
        int e = 0, buf = 0;
        unsigned phase = 0, s_phase = 0;
        bool ok = true;
        for (unsigned turn = 0; ok && parts.get(turn, &p, &s_gave_up); ++turn) {
            const int q0 = CutSlots::first(SeqWork{p.len, 0, p.n_new}, ge, p.tile);
            const int h0 = p.tile * kWTileSlots + half * 128, slot = h0 + (warp & 3) * 32 + lane;
            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            for (int b = 0; ok && b < p.n; ++b) {
                ok = bar_wait(&s_full[half][buf], s_phase, &s_gave_up) && bar_wait(&l_full[e], phase, &s_gave_up);
                if (!ok) break;
                tc_fence_after();
                const int t0 = (q0 + b) * per;
                // Some row is none, or does not see all of the half's slots.
                const bool mask = live < kWTileRows || t0 + per > p.n_new || h0 + 128 > p.len - p.n_new + t0 + 1;
                float s[128];
                tmem_ld32<0>(s, t_s + buf * 128);
                tmem_ld32<32>(s, t_s + buf * 128 + 32);
                tmem_ld32<64>(s, t_s + buf * 128 + 64);
                tmem_ld32<96>(s, t_s + buf * 128 + 96);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(&s_empty[half][buf]);
                if (mask) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int4 sees = *reinterpret_cast<const int4*>(&s_sees[e][i * 4]);
                        if (slot >= sees.x) s[4 * i] = -INFINITY;
                        if (slot >= sees.y) s[4 * i + 1] = -INFINITY;
                        if (slot >= sees.z) s[4 * i + 2] = -INFINITY;
                        if (slot >= sees.w) s[4 * i + 3] = -INFINITY;
                    }
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float4 less = *reinterpret_cast<const float4*>(&s_less[e][i * 4]);
                    float2 x = __ffma2_rn(make_float2(s[4 * i], s[4 * i + 1]), by, make_float2(less.x, less.y));
                    float2 y = __ffma2_rn(make_float2(s[4 * i + 2], s[4 * i + 3]), by, make_float2(less.z, less.w));
                    if (2 * i % 8 < kPolyOf8) x = exp2_poly(x);
                    else x.x = exp2_fast(x.x), x.y = exp2_fast(x.y);
                    if ((2 * i + 1) % 8 < kPolyOf8) y = exp2_poly(y);
                    else y.x = exp2_fast(y.x), y.y = exp2_fast(y.y);
                    sum[0] = __fadd2_rn(sum[0], x);
                    sum[1] = __fadd2_rn(sum[1], y);
                }
                if (slot < s_nan[e]) sum[0].x = NAN;
                __syncwarp();
                if (lane == 0) bar_arrive(&l_empty[e]);
                if (++e == kWLse) e = 0, phase ^= 1;
                buf ^= 1;
                if (buf == 0) s_phase ^= 1;
            }
            if (ok && slot < p.len) {
                const int page = page_of(a.c, p.seq, slot / kPage);
                if (page >= 0) {
                    float* at = a.c.weight + ((long long)page * a.c.n_kv + p.head) * kPage + slot % kPage;
                    const float x = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                    *at = a.decay == 0.f ? x : __fmaf_rn(a.decay, *at, x);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && s_gave_up) flag(a.c, BAD_WAIT);
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// Up to 64 rows pages stream past the rows, from 65 on rows past the slots.  Measured (16 heads of 128 over 8 KV heads,
// us here and there): 4 x 8192 slots 32 rows 20.9 and 23.0, 48 rows 25.4 and 23.2, 64 rows 30.0 and 23.1; 16 x 8192
// 70.6 and 77.2, 88.8 and 76.0, 110 and 76; 16 x 1024 14.6 and 16.3, 17.2 and 15.9, 19.0 and 15.8.  So the two meet
// near 40 rows; 64 is what a pass of the first kernel holds.
template <class T, int kD>
cudaError_t launch_weights(const AttnArgs& a, const CUtensorMap& km, int sms, cudaStream_t s) {
    const long long rows = (long long)a.max_tokens * a.G;
    CUtensorMap qm;
    if (!encode_q(&qm, a, rows <= kWRows ? kWRows : kWTileRows)) return cudaErrorInvalidValue;
    cudaError_t e;
    if (rows <= kWRows) {
        auto* kernel = k_weights_rows<T, kD>;
        static std::atomic<uint64_t> done{0};
        if ((e = allow_smem(kernel, WRowsShape<kD>::kSmem, &done)) != cudaSuccess) return e;
        kernel<<<sms, kWThreads, WRowsShape<kD>::kSmem, s>>>(with_tile(a, kWRows), km, qm);
    } else {
        auto* kernel = k_weights_tiles<T, kD>;
        static std::atomic<uint64_t> done{0};
        if ((e = allow_smem(kernel, WTileShape<kD>::kSmem, &done)) != cudaSuccess) return e;
        kernel<<<sms, kTileThreads, WTileShape<kD>::kSmem, s>>>(with_tile(a, kWTileRows), km, qm);
    }
    return cudaGetLastError();
}

// One 16-row tile at most, one 32-row tile, or 256-row tiles.  Measured (16 heads of 128 over 8 KV heads, us by each of the
// three): 4 x 8192 slots 16 rows 33.0, 38.7, 37.7, 32 rows 42.4, 44.8, 39.2, 48 rows 58.2, 67.5, 40.8; 16 x 8192 16 rows
// 91, 107, 99, 32 rows 169, 120, 103; 4 x 1024 16 rows 18.8, 24.2, 16.9, 32 rows 18.9, 30.0, 17.8.  So the
// chunks' kernel is ahead of the 32-row tile by an eighth or more there.
template <class T, int kD>
cudaError_t launch_by_rows(const AttnArgs& a, const CUtensorMap& km, const CUtensorMap& vm, int sms, cudaStream_t s) {
    const long long rows = (long long)a.max_tokens * a.G;
    if (rows <= 16) return launch_rows<T, kD, 1, 2>(a, km, vm, sms, s);
    if (rows <= 32) return launch_rows<T, kD, 2, 1>(a, km, vm, sms, s);
    return launch_tiles<T, kD>(a, km, vm, sms, s);
}

int sm_count() {
    static std::atomic<int> known[64];
    int device = 0, n = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return 0;
    if (device < 64 && (n = known[device].load(std::memory_order_relaxed))) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return 0;
    n = std::min(n, kMaxSms);
    if (device < 64) known[device].store(n, std::memory_order_relaxed);
    return n;
}

}  // namespace

template <class F>
cudaError_t by_type(const PagedView& c, F&& f) {
    using D64 = std::integral_constant<int, 64>;
    using D128 = std::integral_constant<int, 128>;
    if (c.type == OP_F16) return c.head_dim == 64 ? f(__half(), D64()) : f(__half(), D128());
    return c.head_dim == 64 ? f(__nv_bfloat16(), D64()) : f(__nv_bfloat16(), D128());
}

cudaError_t launch_paged_attention(const AttnArgs& a, cudaStream_t s) {
    CUtensorMap km, vm;
    const int sms = sm_count();
    if (sms == 0 || !encode_cache(&km, a.c, a.c.k) || !encode_cache(&vm, a.c, a.c.v)) return cudaErrorInvalidValue;
    return by_type(a.c, [&](auto t, auto d) { return launch_by_rows<decltype(t), decltype(d)::value>(a, km, vm, sms, s); });
}

cudaError_t launch_attention_weights(const AttnArgs& a, cudaStream_t s) {
    CUtensorMap km;
    const int sms = sm_count();
    if (sms == 0 || !encode_cache(&km, a.c, a.c.k)) return cudaErrorInvalidValue;
    return by_type(a.c, [&](auto t, auto d) { return launch_weights<decltype(t), decltype(d)::value>(a, km, sms, s); });
}

}  // namespace mtb
