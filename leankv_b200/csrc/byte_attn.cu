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
// Bound: a chunk's 2 * 16 * dim + 16 bytes come once from memory. They come by one bulk copy into a ring of a warp's own (4 to 8 chunks ahead), 190 KB in
// flight on an SM; the tensor cores and some 300 issue slots a page and warp run under that.
//
// Split: all pages of all (sequence, kv head, row tile) triples are one flat list, the grid one wave of CTAs with equal shares. A share is cut at
// the triples' borders; a triple that several CTAs share leaves partial sums in the workspace, and the last CTA to arrive adds
// them up in the CTAs' order, so that results do not depend on timing.

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "byte_layout.cuh"
#include "umma.cuh"

namespace leankv {
namespace bytes {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kCtasPerSm = 3;
constexpr int kMinPages = 8;                       // of a CTA
// A row's reference lies kLift below the largest score seen when it last moved, and moves when a score exceeds it by more than kReach: weights are at most
// 2^15 in fp16, and one of 2^-24 of the largest is still a normal number there. Moving costs the rescaling of all sums.
constexpr float kLift = 10.f, kReach = 15.f;
constexpr float kNoRef = -1.0e30f;                 // a maximum before any score: finite, so that masked scores give weight 0
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kCounters = 4096;
constexpr int kStatusWords = 64;
constexpr int kMaxCtas = 1024;
constexpr int kTimedOut = 1, kBadPage = 2;

__host__ __device__ constexpr int stages(int dim) { return dim == 128 ? 4 : 8; }
__host__ __device__ constexpr int row_floats(int dim) { return dim + 4; }               // a row of the warps' sums in shared memory: no bank is met twice
__host__ __device__ constexpr size_t ring_bytes(int dim) { return (size_t)kWarps * stages(dim) * chunk_bytes(dim); }
__host__ __device__ constexpr size_t partial_floats(int dim, int rows) { return (size_t)rows * (dim + 2); }
constexpr size_t kWorkspaceBytes = 4 * (size_t)kStatusWords + 4 * (size_t)kCounters + 2 * (size_t)kMaxCtas * partial_floats(128, 16) * 4;

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
__global__ void __launch_bounds__(kThreads, kCtasPerSm) attn_kernel(const AttnParams p) {
    constexpr int kStages = stages(D);
    constexpr uint32_t kChunk = chunk_bytes(D);
    constexpr int kSteps = D / 16;                 // of the score product, and 16-channel tiles of the values'
    constexpr int kRows = 8 * kTiles;
    constexpr int kQParts = std::is_same<T, float>::value ? 2 : 1;
    constexpr int kPitch = row_floats(D);
    extern __shared__ __align__(128) uint8_t s_ring[];
    __shared__ __align__(8) uint64_t s_bar[kWarps][kStages];
    __shared__ int s_first[LEANKV_BYTES_MAX_BATCH + 1];              // pages of the sequences before b
    __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
    __shared__ int s_sum[kWarps];
    __shared__ int s_last;
    static_assert((size_t)kWarps * kRows * kPitch * 4 <= ring_bytes(D), "the warps' sums lie over the ring");

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < kStages; ++s) umma::bar_init_n(umma::smem_addr(&s_bar[warp][s]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    pdl_begin();

    // ---- pages of each sequence, added up ----
    const int ip0 = p.indptr[0];
    if (p.lists == nullptr) {
        for (int i = tid; i <= p.B; i += kThreads) s_first[i] = p.indptr[i] - ip0;
    } else {
        const int per = (p.B + kThreads - 1) / kThreads, from = min(tid * per, p.B), to = min(from + per, p.B);
        int sum = 0;
        for (int i = from; i < to; ++i) sum += min(p.indptr[i + 1] - p.indptr[i], p.n_lists);
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
            run += min(p.indptr[i + 1] - p.indptr[i], p.n_lists);
        }
        if (to == p.B) s_first[p.B] = run;             // every thread with to = B has the same sum
    }
    __syncthreads();

    const int HR = p.H * p.row_tiles, rows_all = p.tokens * p.G;
    auto out_row = [&](int b, int hr, int r) -> T* {       // row r of a tile; null where there is none
        const int h = hr / p.row_tiles, row = (hr - h * p.row_tiles) * kRows + r;
        if (row >= rows_all) return nullptr;
        const int tok = row / p.G;
        return static_cast<T*>(p.out.data) + b * p.out.seq + (long long)(h * p.G + row - tok * p.G) * p.out.head + tok * p.out.token;
    };
    const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
        if (s_first[b + 1] > s_first[b]) continue;
        for (int i = tid; i < HR * kRows * (D / 4); i += kThreads) {
            T* to = out_row(b, i / (kRows * (D / 4)), i / (D / 4) % kRows);
            if (to != nullptr) store4_as(to + 4 * (i % (D / 4)), none);
        }
    }

    // ---- this CTA's share of the flat list ----
    const long long F = (long long)s_first[p.B] * HR, triples = (long long)p.B * HR;
    long long C = min((long long)gridDim.x, (F + kMinPages - 1) / kMinPages);
    if (C >= 3 * triples) C -= C % triples;            // equal sequences are cut at their borders
    if ((long long)blockIdx.x >= C) return;
    const long long f_lo = blockIdx.x * F / C, f_hi = (blockIdx.x + 1ll) * F / C;
    auto cta_of = [&](long long f) { return (int)(((f + 1) * C + F - 1) / F) - 1; };

    const uint32_t bar0 = umma::smem_addr(&s_bar[warp][0]);
    uint8_t* ring = s_ring + (size_t)warp * kStages * kChunk;
    const uint32_t ring0 = umma::smem_addr(ring);
    unsigned taken = 0;                                // chunks of this warp so far
    bool ok = true;

    for (long long f = f_lo; f < f_hi;) {
        int b = 0;
        for (int step = 512; step > 0; step >>= 1)
            if (b + step < p.B && (long long)s_first[b + step] * HR <= f) b += step;
        // sequences without pages share their first page's number with the next one: the search ends on the last of them, which has pages
        const int have = s_first[b + 1] - s_first[b];
        const long long in_seq = f - (long long)s_first[b] * HR;
        const int hr = (int)(in_seq / have), i0 = (int)(in_seq - (long long)hr * have);
        const int n = (int)min((long long)(have - i0), f_hi - f);
        const long long triple = f - i0;
        const int h = hr / p.row_tiles, row0 = (hr - h * p.row_tiles) * kRows;
        f += n;

        const int ip = p.indptr[b], all_pages = p.indptr[b + 1] - ip, length = (all_pages - 1) * kPage + p.last[b];
        const int32_t* ids = p.lists == nullptr ? p.indices + ip : p.lists + ((long long)b * p.H + h) * p.n_lists;
        const int mine = ok && warp < n ? (n - warp + kWarps - 1) / kWarps : 0;       // pages i0 + warp, + kWarps, ..
        auto page_id = [&](int j) -> int { return j < mine ? ids[i0 + warp + kWarps * j] : 0; };
        int id_now = page_id(lane), id_next = page_id(lane + 32);
        auto copy = [&](int j, int id) {               // chunk j of the segment
            const unsigned s = (taken + j) % kStages;
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
            const unsigned s = (taken + j) % kStages;
            ok = __all_sync(0xffffffffu, umma::bar_wait(bar0 + 8 * s, (taken + j) / kStages & 1));
            if (!ok) {                                 // those behind it are given the same time, then the rows get NaN
                for (int x = j + 1; x < min(mine, j + kStages); ++x) umma::bar_wait(bar0 + 8 * ((taken + x) % kStages), (taken + x) / kStages & 1);
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
                    sc[n8][e] *= ks * factor[n8][e & 1];
                    if (cut && (bad || first + g + 8 * (e >> 1) > limit[n8][e & 1])) sc[n8][e] = -INFINITY;
                    raise |= sc[n8][e] > m[n8][e & 1] + kReach;
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
                        if (best - kLift > m[n8][e]) {
                            const float down = ex2(m[n8][e] - (best - kLift));
                            m[n8][e] = best - kLift;
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
        taken += mine;

        // ---- the warps' sums, over the ring ----
        __syncthreads();                               // every warp has read its last chunk
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
        const bool whole = n == have;
        float* part = p.partials + (2 * (size_t)blockIdx.x + (i0 > 0 ? 0 : 1)) * partial_floats(D, kRows);
        for (int i = tid; i < kRows * (D / 4); i += kThreads) {
            const int r = i / (D / 4), d4 = i % (D / 4);
            float top = s_m[0][r], sum = 0.f;
#pragma unroll
            for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s_m[w][r]);
            float4 v = none;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float x = ex2(s_m[w][r] - top);
                const float4 y = *reinterpret_cast<const float4*>(sums + ((size_t)w * kRows + r) * kPitch + 4 * d4);
                sum = fmaf(s_l[w][r], x, sum);
                v.x = fmaf(y.x, x, v.x), v.y = fmaf(y.y, x, v.y), v.z = fmaf(y.z, x, v.z), v.w = fmaf(y.w, x, v.w);
            }
            if (whole) {
                T* to = out_row(b, hr, r);
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                if (to != nullptr) store4_as(to + 4 * d4, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
            } else {
                *reinterpret_cast<float4*>(part + (size_t)r * D + 4 * d4) = v;
                if (d4 == 0) *reinterpret_cast<float2*>(part + (size_t)kRows * D + 2 * r) = make_float2(top, sum);
            }
        }
        // generic writes to the ring come before the next copies into it
        umma::fence_operands();
        __syncthreads();
        if (whole) continue;

        // ---- a triple that several CTAs share: the last one adds the shares up ----
        const int c0 = cta_of(triple), c1 = cta_of(triple + have - 1);
        if (tid == 0) {
            const bool is_last = arrive(p.counters + c0) == (unsigned)(c1 - c0);
            if (is_last) p.counters[c0] = 0;
            s_last = is_last;
        }
        __syncthreads();
        if (s_last) {
            auto slot = [&](int c) { return p.partials + (2 * (size_t)c + (triple < c * F / C ? 0 : 1)) * partial_floats(D, kRows); };
            for (int i = tid; i < kRows * (D / 4); i += kThreads) {
                const int r = i / (D / 4), d4 = i % (D / 4);
                float top = kNoRef, sum = 0.f;
                float4 v = none;
#pragma unroll 4
                for (int c = c0; c <= c1; ++c) {
                    const float* from = slot(c);
                    const float pm = ld_cg_f32(from + (size_t)kRows * D + 2 * r), pl = ld_cg_f32(from + (size_t)kRows * D + 2 * r + 1);
                    const float4 y = ld_cg_f32x4(from + (size_t)r * D + 4 * d4);
                    const float now = fmaxf(top, pm), keep = ex2(top - now), x = ex2(pm - now);
                    top = now;
                    sum = fmaf(pl, x, sum * keep);
                    v.x = fmaf(y.x, x, v.x * keep), v.y = fmaf(y.y, x, v.y * keep);
                    v.z = fmaf(y.z, x, v.z * keep), v.w = fmaf(y.w, x, v.w * keep);
                }
                T* to = out_row(b, hr, r);
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                if (to != nullptr) store4_as(to + 4 * d4, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
            }
        }
        __syncthreads();                               // s_last is read
    }
}

template <typename T, int D, int kTiles>
int launch(const AttnParams& p, int max_pages_seq, cudaStream_t st) {
    static std::atomic<unsigned long long> ready{0};             // a bit for each device
    int dev = 0;
    LEANKV_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return LEANKV_ELIMIT;
    constexpr size_t smem = ring_bytes(D);
    if (((ready.load(std::memory_order_acquire) >> dev) & 1ull) == 0) {
        LEANKV_CUDA_TRY(cudaFuncSetAttribute(attn_kernel<T, D, kTiles>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    const long long pages = (long long)p.B * p.H * p.row_tiles * (p.lists == nullptr ? max_pages_seq : std::min(max_pages_seq, p.n_lists));
    const long long grid = std::min<long long>(std::min(kCtasPerSm * sm_count(), kMaxCtas), (pages + kMinPages - 1) / kMinPages);
    LEANKV_CUDA_TRY(launch_early(attn_kernel<T, D, kTiles>, dim3((unsigned)std::max(grid, 1ll)), dim3(kThreads), smem, st, p));
    return LEANKV_OK;
}

template <typename T>
int launch(const AttnParams& p, int dim, int rows, int max_pages_seq, cudaStream_t st) {
    if (dim == 128) return rows == 8 ? launch<T, 128, 1>(p, max_pages_seq, st) : launch<T, 128, 2>(p, max_pages_seq, st);
    return rows == 8 ? launch<T, 64, 1>(p, max_pages_seq, st) : launch<T, 64, 2>(p, max_pages_seq, st);
}

}  // namespace
}  // namespace bytes
}  // namespace leankv

using namespace leankv;

extern "C" size_t leankv_byte_attn_workspace_bytes(void) { return bytes::kWorkspaceBytes; }

extern "C" int leankv_byte_attn(const leankv_byte_pool_t* pool, int dtype, const leankv_vectors_t* q, const leankv_vectors_t* out, int B,
                                int q_heads, int tokens, float scale, const int32_t* kv_indptr, const int32_t* kv_page_indices,
                                const int32_t* kv_last_page_len, int max_pages_seq, const int32_t* block_pages, int n_blocks, void* workspace,
                                size_t workspace_bytes, void* stream) {
    if (!bytes::good_pool(pool) || !bytes::good_type(dtype) || !q || !out || !q->data || !out->data || B <= 0 || tokens <= 0 || q_heads <= 0 ||
        q_heads % pool->kv_heads != 0 || !kv_indptr || !kv_page_indices || !kv_last_page_len || max_pages_seq < 0 ||
        (block_pages != nullptr && (tokens != 1 || n_blocks <= 0)))
        return LEANKV_EINVAL;
    if (B > LEANKV_BYTES_MAX_BATCH || q_heads / pool->kv_heads > LEANKV_BYTES_MAX_GROUP) return LEANKV_ELIMIT;
    if (!bytes::aligned_pool(pool) || !bytes::aligned_vectors(q, dtype, B, q_heads, tokens) ||
        !bytes::aligned_vectors(out, dtype, B, q_heads, tokens) || !aligned16(workspace))
        return LEANKV_EALIGN;
    if (!workspace || workspace_bytes < bytes::kWorkspaceBytes) return LEANKV_EWORKSPACE;
    bytes::AttnParams p = {};
    p.chunks = static_cast<const uint8_t*>(pool->chunks);
    p.n_pages = pool->n_pages, p.H = pool->kv_heads, p.B = B, p.G = q_heads / pool->kv_heads, p.tokens = tokens;
    const long long rows_all = (long long)tokens * p.G;
    if (rows_all > (1ll << 24)) return LEANKV_ELIMIT;
    const int rows = rows_all <= 8 ? 8 : 16;
    p.row_tiles = (int)((rows_all + rows - 1) / rows);
    p.q = *q, p.out = *out;
    p.scale = scale * bytes::kLog2e;
    p.indptr = kv_indptr, p.indices = kv_page_indices, p.last = kv_last_page_len;
    p.lists = block_pages, p.n_lists = n_blocks;
    p.status = static_cast<int*>(workspace);
    p.counters = reinterpret_cast<unsigned*>(p.status + bytes::kStatusWords);
    p.partials = reinterpret_cast<float*>(p.counters + bytes::kCounters);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == LEANKV_BYTES_F16 ? bytes::launch<__half>(p, pool->dim, rows, max_pages_seq, st)
         : dtype == LEANKV_BYTES_BF16 ? bytes::launch<bf16>(p, pool->dim, rows, max_pages_seq, st)
                                      : bytes::launch<float>(p, pool->dim, rows, max_pages_seq, st);
}

extern "C" int leankv_byte_status(const void* workspace, int* status) {
    if (!workspace || !status) return LEANKV_EINVAL;
    LEANKV_CUDA_TRY(cudaMemcpy(status, workspace, sizeof(int), cudaMemcpyDeviceToHost));
    return LEANKV_OK;
}
