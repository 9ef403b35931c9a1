// Attention over the 8-bit pages for few query tokens: a decode step, or a handful of tokens behind a long cache.
//
//   out[row] = sum_t softmax_t(scale * q[row] . K_t) V_t,     K_t = 2^ek code_k[t],  V_t = 2^ev code_v[t]
//
// A row is a (query token, query head) pair of one kv head; 8 (or 16) of them are the columns of every product, so that a
// page is read once for all heads that share it. A warp takes a page (16 tokens) at a time:
//   scores   S^T[16 tokens x 8 rows]  = codes_k . q^T          mma.m16n8k16, the codes as fp16 (exact) in the A operand
//   weights  2^(S 2^ek f - m)  with a running reference m of each row that follows the maximum in steps
//   values   O^T[dim x 8 rows] += 2^ev (codes_v . P^T)          the same, channels in the A operand's rows
// The score product leaves tokens in rows; P^T as the B operand wants them in the reduction: four 8 x 8 transposes in registers
// (movmatrix). The query is exact in fp16 after a power of two is taken out of each row (fp32 queries: two fp16 parts and two products). P enters as two
// fp16 parts, so that nothing on the way is rounded to fewer than 21 bits: with one part the weight of a token that
// dominates a row would be 2^-12 off, and the products have room for it (the kernel is bound by memory).
//
// Bound: a chunk's 2 * 16 * dim + 16 bytes come once from memory. They come by one bulk copy into a ring of a warp's own (3 chunks ahead, 6 for head size 64), 190 KB in
// flight on an SM; the tensor cores and some 300 issue slots a page and warp run under that. With two groups of eight rows at head size 128 four CTAs an SM take spills of 128 to 160 bytes a
// thread (fp32 queries 432): 16 x 4096 tokens, 16 heads a kv head 51 us, three CTAs without them 57.
//
// Split. A cluster of CTAs has one (sequence, kv head, row tile) triple or, where there are fewer triples than the device has room for clusters, an equal part of
// its pages; the CTAs share those pages and add their sums up through distributed shared memory, each a slice of the rows. Parts of one triple meet in the workspace:
// the last CTA to arrive adds them in order. Nothing depends on timing. (16 sequences around 4096 tokens, 8 kv heads: one flat list of pages cut into equal shares, joined
// in the workspace, took 36.8 us: shares that crossed a border ran twice through the start, and every join cost some 4 us.)

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "byte_cluster.cuh"
#include "byte_layout.cuh"
#include "byte_workspace.cuh"
#include "umma.cuh"

namespace leankv {
namespace bytes {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kFewPages = 8;                       // of a CTA: below, a smaller cluster
constexpr int kPartPages = 16;                     // of a CTA: below, a triple is not cut into parts, nor into two (joining them costs 2 - 3 us)
constexpr int kWavePages = 96;                     // of a CTA where there is more than one wave of them
// A row's reference lies kLift below the largest score seen when it last moved, and moves when a score exceeds it by more than kReach: weights are at most
// 2^15 in fp16, and one of 2^-24 of the largest is still a normal number there. Moving costs the rescaling of all sums.
constexpr float kLift = 10.f, kReach = 15.f;
constexpr float kNoRef = -3.402823466e38f;         // a maximum before any score: below all of them, and finite, so that masked scores give weight 0
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kJoin = 32;                          // parts of a triple that are joined at a time
__host__ __device__ constexpr int stages(int dim) { return dim == 128 ? 3 : 6; }
__host__ __device__ constexpr int row_floats(int dim) { return dim + 4; }               // a row of the warps' sums in shared memory: no bank is met twice
__host__ __device__ constexpr size_t ring_bytes(int dim) { return (size_t)kWarps * stages(dim) * chunk_bytes(dim); }

struct AttnParams {
    const uint8_t* chunks;
    int n_pages, H, B, G, tokens, row_tiles;
    leankv_vectors_t q, out;
    float scale;                                   // softmax scale * log2(e)
    const int32_t* indptr;
    const int32_t* indices;
    const int32_t* last;
    const int32_t* lists;                          // [B][H][n_lists] page ids, or null: every page
    int n_lists;
    int part_pages;                                // a triple of more pages is cut into parts; 0: none is
    int* status;
    unsigned* counters;
    float* partials;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t n) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(n) : "memory");
}
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t n, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(n), "r"(bar)
                 : "memory");
}
// Codes (stored + 128) 0, 1 or 2, 3 of a word as two fp16 numbers: 0x64 in front of a byte is 1024 + byte.
template <int kPair>
__device__ __forceinline__ uint32_t codes_f16(uint32_t w) {
    const uint32_t x = __byte_perm(w, 0x64646464u, kPair == 0 ? 0x4140 : 0x4342);
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

template <typename T>
__device__ __forceinline__ void store4_as(T* to, float4 v) {
    if constexpr (std::is_same<T, float>::value) *reinterpret_cast<float4*>(to) = v;
    else if constexpr (std::is_same<T, bf16>::value) *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
    else *reinterpret_cast<uint2*>(to) = make_uint2(pack_f16(v.x, v.y), pack_f16(v.z, v.w));
}

// kTiles: groups of eight rows.
template <typename T, int D, int kTiles>
__global__ void __launch_bounds__(kThreads, 4) attn_kernel(const AttnParams p) {
    constexpr int kStages = stages(D);
    constexpr uint32_t kChunk = chunk_bytes(D);
    constexpr int kSteps = D / 16;                 // of the score product, and 16-channel tiles of the values'
    constexpr int kRows = 8 * kTiles;
    constexpr int kQParts = std::is_same<T, float>::value ? 2 : 1;
    constexpr int kPitch = row_floats(D);
    extern __shared__ __align__(128) uint8_t s_ring[];
    __shared__ __align__(8) uint64_t s_bar[kWarps][kStages];
    __shared__ int s_first[LEANKV_BYTES_MAX_BATCH + 1];              // parts of the sequences before b, for each (head, row tile)
    __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
    __shared__ float2 s_ml[kRows];                                   // of the CTA
    __shared__ int s_sum[kWarps];
    __shared__ int s_last;
    static_assert((size_t)(kWarps + 1) * kRows * kPitch * 4 <= ring_bytes(D) && (3 * kJoin * kRows + kThreads) * 4 <= ring_bytes(D), "sums lie over the ring");

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < kStages; ++s) umma::bar_init_n(umma::smem_addr(&s_bar[warp][s]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    pdl_begin();

    unsigned rank, ctas;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
    const int unit = blockIdx.x / ctas, HR = p.H * p.row_tiles, rows_all = p.tokens * p.G;

    // ---- the cluster's triple, and its part of the pages ----
    auto held = [&](int b) {                           // pages that sequence b's triples read
        const int n = p.indptr[b + 1] - p.indptr[b];
        return p.lists == nullptr ? n : min(n, p.n_lists);
    };
    int b, hr, part = 0, parts = 1;
    if (p.part_pages == 0) {
        b = unit / HR;
        hr = unit - b * HR;
    } else {
        const int per = (p.B + kThreads - 1) / kThreads, from = min(tid * per, p.B), to = min(from + per, p.B);
        auto parts_of = [&](int i) { return max(1, (held(i) + p.part_pages - 1) / p.part_pages); };
        int sum = 0;
        for (int i = from; i < to; ++i) sum += parts_of(i);
        int incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int add = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += add;
        }
        if (lane == 31) s_sum[warp] = incl;
        __syncthreads();
        int run = incl - sum;
        for (int w = 0; w < warp; ++w) run += s_sum[w];
        for (int i = from; i < to; ++i) {
            s_first[i] = run;
            run += parts_of(i);
        }
        if (to == p.B) s_first[p.B] = run;             // every thread with to = B has the same sum
        __syncthreads();
        if (s_first[p.B] * HR > (int)(gridDim.x / ctas)) {                 // more pages than the caller's bound: parts would be missing
            if (unit == 0 && rank == 0 && tid == 0) atomicOr(p.status, kTooMany);
            return;
        }
        if (unit >= s_first[p.B] * HR) return;         // the whole cluster: the grid was sized for the bound
        b = 0;
        for (int step = 512; step > 0; step >>= 1)
            if (b + step < p.B && s_first[b + step] * HR <= unit) b += step;
        parts = s_first[b + 1] - s_first[b];
        part = unit - s_first[b] * HR;
        hr = part / parts;
        part -= hr * parts;
    }
    const int ip = p.indptr[b], all_pages = p.indptr[b + 1] - ip, length = (all_pages - 1) * kPage + p.last[b];
    const int have = p.lists == nullptr ? all_pages : min(all_pages, p.n_lists);
    const int h = hr / p.row_tiles, row0 = (hr - h * p.row_tiles) * kRows;
    const int32_t* ids = p.lists == nullptr ? p.indices + ip : p.lists + ((long long)b * p.H + h) * p.n_lists;
    auto share = [](int n, int i, int of) { return i * (n / of) + min(i, n % of); };       // the first of n things that the i-th has
    const int part0 = share(have, part, parts), part_n = share(have, part + 1, parts) - part0;
    const int i0 = part0 + share(part_n, (int)rank, (int)ctas), n = part0 + share(part_n, (int)rank + 1, (int)ctas) - i0;
    auto out_row = [&](int r) -> T* {                  // row r of the tile; null where there is none
        const int row = row0 + r;
        if (row >= rows_all) return nullptr;
        const int tok = row / p.G;
        return static_cast<T*>(p.out.data) + b * p.out.seq + (long long)(h * p.G + row - tok * p.G) * p.out.head + tok * p.out.token;
    };
    const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);

    const uint32_t bar0 = umma::smem_addr(&s_bar[warp][0]);
    uint8_t* ring = s_ring + (size_t)warp * kStages * kChunk;
    const uint32_t ring0 = umma::smem_addr(ring);
    bool ok = true;
    const int mine = warp < n ? (n - warp + kWarps - 1) / kWarps : 0;       // pages i0 + warp, + kWarps, ..
    auto page_id = [&](int j) -> int { return j < mine ? ids[i0 + warp + kWarps * j] : 0; };
    int id_now = page_id(lane), id_next = page_id(lane + 32);
    auto copy = [&](int j, int id) {                   // chunk j of the warp
        const unsigned s = (unsigned)j % kStages;
        if (lane == 0) {
            expect_bytes(bar0 + 8 * s, kChunk);
            bulk_copy(ring0 + s * kChunk, p.chunks + ((size_t)((unsigned)id < (unsigned)p.n_pages ? id : 0) * p.H + h) * kChunk, kChunk, bar0 + 8 * s);
        }
    };
    for (int j = 0; j < min(mine, kStages); ++j) copy(j, __shfl_sync(0xffffffffu, id_now, j));

    // ---- queries: B operands, and what the rows' scores are multiplied with ----
    uint32_t qf[kTiles][kQParts][kSteps][2];
    float factor[kTiles][2];
    int limit[kTiles][2];                          // the last position that rows 2t, 2t + 1 see
#pragma unroll
    for (int n8 = 0; n8 < kTiles; ++n8) {
        const int row = row0 + 8 * n8 + g, tok = row / p.G;
        Eight<T> x[D / 64][2];
        const T* src = static_cast<const T*>(p.q.data) + b * p.q.seq + (long long)(h * p.G + row - tok * p.G) * p.q.head + tok * p.q.token + 16 * t;
        uint32_t amax = 0;
#pragma unroll
        for (int hh = 0; hh < D / 64; ++hh)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (row < rows_all) x[hh][e].load(src + 64 * hh + 8 * e);
                else x[hh][e].zero();
#pragma unroll
                for (int k = 0; k < 8; ++k) amax = max(amax, __float_as_uint(x[hh][e].get(k)) & 0x7fffffffu);
            }
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // the largest magnitude is brought to 2^14 .. 2^15; numbers below 2^-38 of it lose places
        const int e2 = std::is_same<T, __half>::value ? 0 : max((int)(amax >> 23) - 127 - 14, -126);
        const float down = power_of_two(-e2);
#pragma unroll
        for (int hh = 0; hh < D / 64; ++hh)
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float a = x[hh][s >> 1].get(4 * (s & 1) + 2 * e) * down, c = x[hh][s >> 1].get(4 * (s & 1) + 2 * e + 1) * down;
                    const uint32_t hi = pack_f16(a, c);
                    qf[n8][0][4 * hh + s][e] = hi;
                    if constexpr (kQParts == 2) {
                        const float2 got = unpack_f16(hi);
                        qf[n8][kQParts - 1][4 * hh + s][e] = pack_f16(a - got.x, c - got.y);
                    }
                }
        const float mult = power_of_two(e2) * p.scale;
        const int lim = length - p.tokens + tok;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            factor[n8][e] = __shfl_sync(0xffffffffu, mult, 8 * t + 4 * e);
            limit[n8][e] = __shfl_sync(0xffffffffu, lim, 8 * t + 4 * e);
        }
    }
    // positions at and below this one are seen by all rows of the tile (rows beyond the last one may see more)
    const int seen_by_all = length - p.tokens + row0 / p.G;

    float o[kTiles][kSteps][4];
    float m[kTiles][2], l[kTiles][2];
#pragma unroll
    for (int n8 = 0; n8 < kTiles; ++n8) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n8][i][e] = 0.f;
        m[n8][0] = m[n8][1] = kNoRef;
        l[n8][0] = l[n8][1] = 0.f;
    }

    for (int j = 0; j < mine; ++j) {
        if (j > 0 && (j & 31) == 0) {
            id_now = id_next;
            id_next = page_id(j + 32 + lane);
        }
        const unsigned s = (unsigned)j % kStages;
        ok = __all_sync(0xffffffffu, umma::bar_wait(bar0 + 8 * s, (unsigned)j / kStages & 1));
        if (!ok) {                                 // those behind it are given the same time, then the rows get NaN
            for (int x = j + 1; x < min(mine, j + kStages); ++x) umma::bar_wait(bar0 + 8 * ((unsigned)x % kStages), (unsigned)x / kStages & 1);
            if (lane == 0) atomicOr(p.status, kTimedOut);
            break;
        }
        const bool bad = (unsigned)__shfl_sync(0xffffffffu, id_now, j & 31) >= (unsigned)p.n_pages;
        const uint8_t* chunk = ring + (size_t)s * kChunk;
        const float2 scales = *reinterpret_cast<const float2*>(chunk + 2 * half_bytes(D));

        float sc[kTiles][4];
#pragma unroll
        for (int n8 = 0; n8 < kTiles; ++n8)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[n8][e] = 0.f;
#pragma unroll
        for (int hh = 0; hh < D / 64; ++hh) {
            const uint4 ka = *reinterpret_cast<const uint4*>(chunk + hh * 1024 + g * 64 + t * 16);
            const uint4 kb = *reinterpret_cast<const uint4*>(chunk + hh * 1024 + (g + 8) * 64 + t * 16);
            const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t a[4] = {codes_f16<0>(wa[k]), codes_f16<0>(wb[k]), codes_f16<1>(wa[k]), codes_f16<1>(wb[k])};
#pragma unroll
                for (int n8 = 0; n8 < kTiles; ++n8)
#pragma unroll
                    for (int part = 0; part < kQParts; ++part) mma_f16(sc[n8], a, qf[n8][part][4 * hh + k][0], qf[n8][part][4 * hh + k][1]);
            }
        }
        // a block with a scale that is no number answers nobody who sees it; its codes are zeros
        const float ks = isnan(scales.y) ? scales.y : scales.x, vs = isnan(scales.y) ? 0.f : scales.y;
        const int i = i0 + warp + kWarps * j;      // of the triple's pages
        // only the last page of a list is cut
        const int first = p.lists == nullptr ? i * kPage : i == have - 1 ? (all_pages - 1) * kPage : 0;
        const bool cut = bad || first + kPage - 1 > seen_by_all;
        uint32_t ph[kTiles][2], pl[kTiles][2];
        bool raise = false;
#pragma unroll
        for (int n8 = 0; n8 < kTiles; ++n8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {          // token g + 8 (e >> 1), row 2t + (e & 1)
                // rounded by itself: fused with the weight's subtraction, its last places would be powers of two of a large score
                sc[n8][e] = __fmul_rn(sc[n8][e], ks * factor[n8][e & 1]);
                if (cut && (bad || first + g + 8 * (e >> 1) > limit[n8][e & 1])) sc[n8][e] = -INFINITY;
                raise |= sc[n8][e] > __fadd_rd(m[n8][e & 1], kReach);          // to nearest, m + 15 is m + 16 for numbers around 2^28, a weight beyond fp16
            }
        }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int n8 = 0; n8 < kTiles; ++n8)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float best = fmaxf(sc[n8][e], sc[n8][e + 2]);
#pragma unroll
                    for (int x = 4; x < 32; x *= 2) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, x));
                    const float now = __fadd_ru(best, -kLift);
                    if (now > m[n8][e]) {
                        const float down = ex2(m[n8][e] - now);
                        m[n8][e] = now;
                        l[n8][e] *= down;
#pragma unroll
                        for (int k = 0; k < kSteps; ++k) {
                            o[n8][k][e] *= down;
                            o[n8][k][e + 2] *= down;
                        }
                    }
                }
        }
#pragma unroll
        for (int n8 = 0; n8 < kTiles; ++n8) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[e] = ex2(sc[n8][e] - m[n8][e & 1]);
                l[n8][e & 1] += w[e];
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t hi = pack_f16(w[2 * e], w[2 * e + 1]);
                const float2 got = unpack_f16(hi);
                ph[n8][e] = transpose8(hi);
                pl[n8][e] = transpose8(pack_f16(w[2 * e] - got.x, w[2 * e + 1] - got.y));
            }
        }
        const uint8_t* values = chunk + half_bytes(D) + lane * 16;
#pragma unroll
        for (int part = 0; part < D / 32; ++part) {
            const uint4 v = *reinterpret_cast<const uint4*>(values + part * 512);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t a[4] = {codes_f16<0>(w[2 * k]), codes_f16<0>(w[2 * k + 1]), codes_f16<1>(w[2 * k]), codes_f16<1>(w[2 * k + 1])};
#pragma unroll
                for (int n8 = 0; n8 < kTiles; ++n8) {
                    float d[4] = {0.f, 0.f, 0.f, 0.f};
                    mma_f16(d, a, pl[n8][0], pl[n8][1]);
                    mma_f16(d, a, ph[n8][0], ph[n8][1]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n8][2 * part + k][e] = fmaf(d[e], vs, o[n8][2 * part + k][e]);
                }
            }
        }
        __syncwarp();
        if (j + kStages < mine) copy(j + kStages, __shfl_sync(0xffffffffu, ((j + kStages) ^ j) & 32 ? id_next : id_now, (j + kStages) & 31));
        if (bad && lane == 0) atomicOr(p.status, kBadPage);
    }

    // ---- the warps' sums, over the ring: first of the CTA, then of the cluster ----
    __syncthreads();                                   // every warp has read its last chunk
    float* sums = reinterpret_cast<float*>(s_ring);
#pragma unroll
    for (int n8 = 0; n8 < kTiles; ++n8)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int x = 4; x < 32; x *= 2) l[n8][e] += __shfl_xor_sync(0xffffffffu, l[n8][e], x);
            const int r = 8 * n8 + 2 * t + e;
            if (g == 0) {
                s_m[warp][r] = m[n8][e];
                s_l[warp][r] = ok ? l[n8][e] : NAN;
            }
            float* to = sums + ((size_t)warp * kRows + r) * kPitch + g;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                to[16 * k] = o[n8][k][e];
                to[16 * k + 8] = o[n8][k][e + 2];
            }
        }
    __syncthreads();
    constexpr int kAll = kRows * (D / 4), kItems = kAll / kThreads;       // four numbers of a row each
    float* shared = sums + (size_t)kWarps * kRows * kPitch;               // the CTA's, for its neighbours
    float* partial = p.partials + (size_t)unit * partial_floats(D, kRows);
    auto finish = [&](int i, float4 v, float top, float sum) {
        const int r = i / (D / 4), d4 = i % (D / 4);
        if (parts > 1) {
            *reinterpret_cast<float4*>(partial + 4 * i) = v;
            if (d4 == 0) *reinterpret_cast<float2*>(partial + (size_t)kRows * D + 2 * r) = make_float2(top, sum);
            return;
        }
        T* to = out_row(r);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        if (to != nullptr) store4_as(to + 4 * d4, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
    };
#pragma unroll
    for (int x = 0; x < kItems; ++x) {
        const int i = tid + x * kThreads, r = i / (D / 4), d4 = i % (D / 4);
        float top = s_m[0][r], sum = 0.f;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s_m[w][r]);
        float4 v = none;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = ex2(s_m[w][r] - top);
            const float4 y = *reinterpret_cast<const float4*>(sums + ((size_t)w * kRows + r) * kPitch + 4 * d4);
            sum = fmaf(s_l[w][r], f, sum);
            v.x = fmaf(y.x, f, v.x), v.y = fmaf(y.y, f, v.y), v.z = fmaf(y.z, f, v.z), v.w = fmaf(y.w, f, v.w);
        }
        if (ctas == 1) {
            finish(i, v, top, sum);
        } else {
            *reinterpret_cast<float4*>(shared + 4 * i) = v;
            if (d4 == 0) s_ml[r] = make_float2(top, sum);
        }
    }
    if (ctas > 1) {
        cluster_sync();
        const uint32_t mine_at = umma::smem_addr(shared), ml_at = umma::smem_addr(s_ml);
        for (int i = tid * (int)ctas + (int)rank; i < kAll; i += kThreads * (int)ctas) {
            const int r = i / (D / 4);
            float2 ml[kMaxCluster];
            float4 y[kMaxCluster];
            float top = kNoRef, sum = 0.f;
#pragma unroll
            for (int c = 0; c < kMaxCluster; ++c) {
                if (c >= (int)ctas) continue;
                ml[c] = peer_f32x2(ml_at + 8 * r, c);
                y[c] = peer_f32x4(mine_at + 16 * i, c);
                top = fmaxf(top, ml[c].x);
            }
            float4 v = none;
#pragma unroll
            for (int c = 0; c < kMaxCluster; ++c) {
                if (c >= (int)ctas) continue;
                const float f = ex2(ml[c].x - top);
                sum = fmaf(ml[c].y, f, sum);
                v.x = fmaf(y[c].x, f, v.x), v.y = fmaf(y[c].y, f, v.y), v.z = fmaf(y[c].z, f, v.z), v.w = fmaf(y[c].w, f, v.w);
            }
            finish(i, v, top, sum);
        }
        cluster_sync();                                // nobody leaves while its sums are read
    }
    if (parts == 1) return;

    // ---- parts of a triple: the last CTA adds them up ----
    __syncthreads();
    const int unit0 = unit - part;
    if (tid == 0) {
        const bool is_last = arrive(p.counters + unit0) == (unsigned)(parts * (int)ctas - 1);
        if (is_last) p.counters[unit0] = 0;
        s_last = is_last;
    }
    __syncthreads();
    if (!s_last) return;
    // kJoin parts at a time: what each counts (a thread a row and part), and their sums; 16 loads of a thread are in flight
    constexpr int kGroups = kThreads / kRows, kEach = kJoin / kGroups, kBatch = 16 / kItems;
    float* s_w = sums;                                 // [kJoin][kRows]: factors, and factors times sums
    float* s_wl = s_w + kJoin * kRows;
    float* s_top = s_wl + kJoin * kRows;               // [kGroups][kRows]
    const int mr = tid % kRows, mg = tid / kRows;
    float4 v[kItems];
    float sum[kItems], top = kNoRef;
#pragma unroll
    for (int x = 0; x < kItems; ++x) v[x] = none, sum[x] = 0.f;
    for (int from = 0; from < parts; from += kJoin) {
        const int here = min(kJoin, parts - from);
        const float* first = p.partials + (size_t)(unit0 + from) * partial_floats(D, kRows);
        auto piece = [&](int c, int x) { return __ldcg(reinterpret_cast<const float4*>(first + (size_t)c * partial_floats(D, kRows)) + tid + x * kThreads); };
        float2 ml[kEach];
        float now = top;
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
            const int c = mg + x * kGroups;
            ml[x] = c < here ? __ldcg(reinterpret_cast<const float2*>(first + (size_t)c * partial_floats(D, kRows) + (size_t)kRows * D) + mr) : make_float2(kNoRef, 0.f);
        }
        float4 y[kBatch][kItems];
#pragma unroll
        for (int c = 0; c < kBatch; ++c)
#pragma unroll
            for (int x = 0; x < kItems; ++x)
                if (c < here) y[c][x] = piece(c, x);
#pragma unroll
        for (int x = 0; x < kEach; ++x) now = fmaxf(now, ml[x].x);
        s_top[mg * kRows + mr] = now;
        __syncthreads();
#pragma unroll
        for (int x = 0; x < kGroups; ++x) now = fmaxf(now, s_top[x * kRows + mr]);
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
            const float f = ex2(ml[x].x - now);
            s_w[(mg + x * kGroups) * kRows + mr] = f;
            s_wl[(mg + x * kGroups) * kRows + mr] = f * ml[x].y;
        }
        __syncthreads();
        if (mg == 0) s_top[mr] = ex2(top - now);       // of the parts before
        top = now;
        __syncthreads();
        auto add = [&](int c, int x, float4 a) {
            const int r = (tid + x * kThreads) / (D / 4);
            const float w = s_w[c * kRows + r];
            sum[x] += s_wl[c * kRows + r];
            v[x].x = fmaf(a.x, w, v[x].x), v[x].y = fmaf(a.y, w, v[x].y), v[x].z = fmaf(a.z, w, v[x].z), v[x].w = fmaf(a.w, w, v[x].w);
        };
#pragma unroll
        for (int x = 0; x < kItems; ++x) {
            const float keep = s_top[(tid + x * kThreads) / (D / 4)];
            sum[x] *= keep, v[x].x *= keep, v[x].y *= keep, v[x].z *= keep, v[x].w *= keep;
        }
#pragma unroll
        for (int c = 0; c < kBatch; ++c)
#pragma unroll
            for (int x = 0; x < kItems; ++x)
                if (c < here) add(c, x, y[c][x]);
        for (int from_c = kBatch; from_c < here; from_c += kBatch) {
#pragma unroll
            for (int c = 0; c < kBatch; ++c)
#pragma unroll
                for (int x = 0; x < kItems; ++x)
                    if (from_c + c < here) y[c][x] = piece(from_c + c, x);
#pragma unroll
            for (int c = 0; c < kBatch; ++c)
#pragma unroll
                for (int x = 0; x < kItems; ++x)
                    if (from_c + c < here) add(from_c + c, x, y[c][x]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < kItems; ++x) {
        const int i = tid + x * kThreads;
        T* to = out_row(i / (D / 4));
        const float inv = sum[x] == 0.f ? 0.f : 1.f / sum[x];
        if (to != nullptr) store4_as(to + 4 * (i % (D / 4)), make_float4(v[x].x * inv, v[x].y * inv, v[x].z * inv, v[x].w * inv));
    }
}

// How a launch is cut: CTAs of a cluster, pages of a part (0: triples are whole), clusters of the grid.
struct Plan {
    int ctas;
    int part_pages;
    long long clusters;
};
// room[i]: clusters of 2^i CTAs that the device holds at once; triples, their longest one's pages, all their pages.
Plan make_plan(const int (&room)[4], long long triples, long long longest, long long total) {
    int i = 0;
    Plan plan;
    if (triples > room[0]) {
        // more than one wave: single CTAs, which start as others end; clusters would wait for all of theirs (256 sequences of 500 tokens, 8 kv heads: 54 us, clusters
        // of two / four 76 / 113; 80 of 4096, of 96 pages each / whole / clusters of two 124 / 133 / 122)
        plan.part_pages = kWavePages;
    } else {
        // as many CTAs of a triple as there is room for, with kFewPages each at least; parts where whole clusters fit more than once
        while (i < 3 && room[i + 1] >= triples && longest > (kFewPages << i)) ++i;
        // long streams in parts: smaller clusters if those fill the device by a tenth more (4 sequences of 32781 tokens: 512 CTAs in clusters of eight
        // 55.4 us, 576 in clusters of two 52.1; one of 16384, 16 pages a CTA: 16.9 and 18.6)
        auto used = [&](int k) { return room[k] / triples * triples << k; };
        if (longest * triples > 64ll * used(i))
            for (int k = i - 1; k >= 0; --k)
                if (10 * used(k) >= 11 * used(i)) i = k;
        const long long most = room[i] / triples, even = (longest + most - 1) / most;
        plan.part_pages = (int)std::max(room[i] > triples ? std::min(even, (total + room[i] - triples - 1) / (room[i] - triples)) : even, (long long)kPartPages << i);
    }
    plan.ctas = 1 << i;
    if (total / plan.part_pages + triples > kMaxParts)
        plan.part_pages = (int)(triples >= kMaxParts ? longest : std::max<long long>(plan.part_pages, total / (kMaxParts - triples) + 1));
    if (longest <= plan.part_pages || (triples <= room[0] && longest <= 2ll * kPartPages << i)) plan.part_pages = 0;
    plan.clusters = plan.part_pages == 0 ? triples : total / plan.part_pages + triples;
    return plan;
}

template <typename T, int D, int kTiles>
int launch(const AttnParams& p, int max_pages_seq, long long total_pages, cudaStream_t st) {
    static std::atomic<unsigned long long> ready{0};             // a bit for each device
    static int rooms[64][4];
    int dev = 0;
    LEANKV_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return LEANKV_ELIMIT;
    constexpr size_t smem = ring_bytes(D);
    if (((ready.load(std::memory_order_acquire) >> dev) & 1ull) == 0) {
        LEANKV_CUDA_TRY(cudaFuncSetAttribute(attn_kernel<T, D, kTiles>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        for (int i = 0; i < 4; ++i) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(1u << i);
            cfg.blockDim = dim3(kThreads);
            cfg.dynamicSmemBytes = smem;
            cudaLaunchAttribute attr;
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = 1u << i, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
            cfg.attrs = &attr, cfg.numAttrs = 1;
            int n = 0;
            LEANKV_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, attn_kernel<T, D, kTiles>, &cfg));
            rooms[dev][i] = std::max(n, 1);
        }
        ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    const long long rows = (long long)p.H * p.row_tiles, longest = p.lists == nullptr ? max_pages_seq : std::min(max_pages_seq, p.n_lists);
    const long long total = std::min(total_pages, p.B * longest) * rows;
    if (p.B * rows > 0x7fffffffll || total > 0x7fffffffll) return LEANKV_ELIMIT;
    const Plan plan = make_plan(rooms[dev], p.B * rows, longest, p.lists == nullptr ? total : p.B * longest * rows);
    if (plan.clusters * plan.ctas > 0x7fffffffll) return LEANKV_ELIMIT;
    AttnParams q = p;
    q.part_pages = plan.part_pages;
    const dim3 grid((unsigned)(plan.clusters * plan.ctas));
    if (plan.ctas == 1) LEANKV_CUDA_TRY(launch_early(attn_kernel<T, D, kTiles>, grid, dim3(kThreads), smem, st, q));
    else LEANKV_CUDA_TRY(launch_cluster_kernel_ex(true, dim3(plan.ctas), attn_kernel<T, D, kTiles>, grid, dim3(kThreads), smem, st, q));
    return LEANKV_OK;
}

template <typename T>
int launch(const AttnParams& p, int dim, int rows, int max_pages_seq, long long total_pages, cudaStream_t st) {
    if (dim == 128) return rows == 8 ? launch<T, 128, 1>(p, max_pages_seq, total_pages, st) : launch<T, 128, 2>(p, max_pages_seq, total_pages, st);
    return rows == 8 ? launch<T, 64, 1>(p, max_pages_seq, total_pages, st) : launch<T, 64, 2>(p, max_pages_seq, total_pages, st);
}

}  // namespace
}  // namespace bytes
}  // namespace leankv

using namespace leankv;

extern "C" size_t leankv_byte_attn_workspace_bytes(void) { return bytes::kWorkspaceBytes; }

extern "C" int leankv_byte_attn(const leankv_byte_attn_t* a, void* stream) {
    if (const int rc = bytes::check_attn(a, bytes::kWorkspaceBytes)) return rc;
    bytes::AttnParams p = {};
    p.chunks = static_cast<const uint8_t*>(a->pool.chunks);
    p.n_pages = a->pool.n_pages, p.H = a->pool.kv_heads, p.B = a->batch, p.G = a->q_heads / a->pool.kv_heads, p.tokens = a->tokens;
    const long long rows_all = (long long)a->tokens * p.G;
    if (rows_all > (1ll << 24)) return LEANKV_ELIMIT;
    const int rows = rows_all <= 8 ? 8 : 16;
    p.row_tiles = (int)((rows_all + rows - 1) / rows);
    p.q = a->q, p.out = a->out;
    p.scale = a->scale * bytes::kLog2e;
    p.indptr = a->kv_indptr, p.indices = a->kv_page_indices, p.last = a->kv_last_page_len;
    p.lists = a->block_pages, p.n_lists = a->n_blocks;
    p.status = static_cast<int*>(a->workspace);
    p.counters = reinterpret_cast<unsigned*>(p.status + bytes::kStatusWords);
    p.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + bytes::kPartialsAt);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->dtype == LEANKV_BYTES_F16 ? bytes::launch<__half>(p, a->pool.dim, rows, a->max_pages_seq, a->total_pages, st)
         : a->dtype == LEANKV_BYTES_BF16 ? bytes::launch<bf16>(p, a->pool.dim, rows, a->max_pages_seq, a->total_pages, st)
                                         : bytes::launch<float>(p, a->pool.dim, rows, a->max_pages_seq, a->total_pages, st);
}

extern "C" int leankv_byte_status(const void* workspace, int* status) {
    if (!workspace || !status) return LEANKV_EINVAL;
    LEANKV_CUDA_TRY(cudaMemcpy(status, workspace, sizeof(int), cudaMemcpyDeviceToHost));
    return LEANKV_OK;
}
