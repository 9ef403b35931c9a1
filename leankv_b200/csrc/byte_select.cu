// Which blocks of a long cache a query token reads: a cheap upper bound of its scores for every block, and the best of them.
//
// Bound of a block. For a query row q and any key k of the block, q.k = sum_d q_d k_d <= sum_d max(q_d, 0) max_d + min(q_d, 0) min_d with the
// largest and smallest key of each channel. Summed over the heads of a group that is ONE pair of vectors, P = sum_g max(q_g, 0) and N = sum_g min(q_g, 0),
// against the block's 2 * dim codes. With q rounded to whole numbers (11 bits and a sign, one power of two for the group) everything is a
// whole number: dp2a takes two 16-bit by 8-bit products at a time, sums are exact, and the choice does not depend on any order.
// A record is 2 * dim + 16 bytes against 32 * dim + 16 of the block: the scores read 1/16 of the cache.
//
// score_kernel: a CTA asks for the records of its blocks first and forms P and N while they come; a lane has 16 bytes of a record and its 16 numbers of P
// or N in registers, dim / 8 lanes share a record.
// select_kernel: a CTA has a (sequence, kv head); scores are whole numbers in the scores' order, kept in registers. The border is found in the range between the
// smallest and the largest: 2048 bins, the one that holds the border becomes the next range (scores share their upper bits: bins of the number itself would all
// be hit in one place; counting against three borders a step, 16 steps of a barrier each, took 23 us for 8193 blocks). Mostly two rounds. Positions come from ballots and
// one scan, so that the list ascends.

#include <algorithm>

#include "byte_layout.cuh"

namespace leankv {
namespace bytes {
namespace {

constexpr int kScoreThreads = 128, kScoreWarps = kScoreThreads / 32;
constexpr int kScoreBlocks = 64;                   // of a CTA
constexpr int kPer = 16;                           // scores that a thread keeps in registers
constexpr int kBins = 2048;

struct SelectParams {
    const uint8_t* bounds;
    int H, n_pages, G, max_pages, n_blocks, sinks, recent;
    leankv_vectors_t q;
    const int32_t* indptr;
    const int32_t* indices;
    float* scores;                                 // [B][H][max_pages]
    int32_t* blocks;
    int32_t* block_pages;
};

template <typename T, int D>
__global__ void __launch_bounds__(kScoreThreads) score_kernel(const SelectParams p) {
    constexpr int kLanes = D / 8;                  // of a record
    constexpr int kAtOnce = 32 / kLanes, kOfWarp = kScoreBlocks / kScoreWarps, kLoads = kOfWarp / kAtOnce;
    constexpr int kHeads = LEANKV_BYTES_MAX_GROUP * (D / 8) / kScoreThreads;      // eights of the group's queries that a thread has at most
    __shared__ uint32_t s_amax[kScoreWarps];
    __shared__ __align__(16) short s_int[LEANKV_BYTES_MAX_GROUP][D];
    __shared__ __align__(16) short s_pn[2 * D];
    pdl_begin();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int h = blockIdx.y, b = blockIdx.z;
    const int ip = p.indptr[b], pages = min(p.indptr[b + 1] - ip, p.max_pages);
    if (pages <= p.n_blocks || (int)blockIdx.x * kScoreBlocks >= pages) return;
    int first = blockIdx.x * kScoreBlocks + warp * kOfWarp;

    // ---- queries and records are asked for ----
    const T* q = static_cast<const T*>(p.q.data) + b * p.q.seq + (long long)h * p.G * p.q.head;
    const int eights = p.G * (D / 8);
    Eight<T> x[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        const int at = tid + i * kScoreThreads;
        if (at < eights) x[i].load(q + (at / (D / 8)) * p.q.head + at % (D / 8) * 8);
        else x[i].zero();
    }
    const int part = lane % kLanes, sub = lane / kLanes;
    uint4 c[kLoads];
    float scale[kLoads];
    auto ask = [&] {
        int id = -1;                               // of block first + lane
        if (lane < kOfWarp && first + lane < pages) id = p.indices[ip + first + lane];
        if ((unsigned)id >= (unsigned)p.n_pages) id = -1;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int mine = __shfl_sync(0xffffffffu, id, i * kAtOnce + sub);
            const uint8_t* rec = p.bounds + ((size_t)max(mine, 0) * p.H + h) * bounds_bytes(D);
            c[i] = __ldg(reinterpret_cast<const uint4*>(rec) + part);
            scale[i] = part != 0 ? 0.f : mine < 0 ? -INFINITY : __ldg(reinterpret_cast<const float*>(rec + 2 * D));
        }
    };
    ask();

    // ---- P and N ----
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(x[i].get(e)) & 0x7fffffffu);
    amax = __reduce_max_sync(0xffffffffu, amax);
    if (lane == 0) s_amax[warp] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kScoreWarps; ++w) amax = max(amax, s_amax[w]);
    const bool finite = amax < 0x7f800000u;        // else every score is 0
    const float down = power_of_two(-least_exponent<2047>(min(amax, 0x7f7fffffu)));
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        const int at = tid + i * kScoreThreads;
        if (at >= eights) continue;
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int lo = finite ? __float2int_rn(x[i].get(2 * e) * down) : 0, hi = finite ? __float2int_rn(x[i].get(2 * e + 1) * down) : 0;
            w[e] = ((uint32_t)lo & 0xffffu) | ((uint32_t)hi << 16);
        }
        *reinterpret_cast<uint4*>(&s_int[at / (D / 8)][at % (D / 8) * 8]) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __syncthreads();
    if (tid < D) {
        int up = 0, low = 0;
        for (int g = 0; g < p.G; ++g) {
            const int i = s_int[g][tid];
            up += max(i, 0);
            low += min(i, 0);
        }
        s_pn[tid] = (short)up;
        s_pn[D + tid] = (short)low;
    }
    __syncthreads();
    int pn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) pn[e] = reinterpret_cast<const int*>(s_pn)[8 * part + e];

    float* out = p.scores + ((long long)b * p.H + h) * p.max_pages;
    for (;;) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
            int u = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                u = __dp2a_lo(pn[2 * e], (int)w[e], u);
                u = __dp2a_hi(pn[2 * e + 1], (int)w[e], u);
            }
#pragma unroll
            for (int o = 1; o < kLanes; o *= 2) u += __shfl_xor_sync(0xffffffffu, u, o);
            const int j = first + i * kAtOnce + sub;
            if (part == 0 && j < pages) out[j] = scale[i] == -INFINITY ? -INFINITY : __int2float_rn(u) * scale[i];
        }
        // a launch for sequences of any length has fewer CTAs than the longest would take
        first += (int)gridDim.x * kScoreBlocks;
        if (first >= pages) break;                 // (the whole warp)
        ask();
    }
}

// fp32 numbers as whole numbers in the same order; a product with NaN, which is 0x7fffffff, is the largest of 32 bits.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t x = __float_as_uint(v);
    return x ^ ((x >> 31) ? 0xffffffffu : 0x80000000u);
}

template <int kThreads>
__global__ void __launch_bounds__(kThreads) select_kernel(const SelectParams p) {
    constexpr int kWarps = kThreads / 32, kSlab = kPer * kThreads, kOwn = kBins / kThreads;      // kOwn: bins of a thread
    __shared__ uint32_t s_low[kWarps], s_high[kWarps];
    __shared__ int s_bin[kBins];
    __shared__ int s_part[kWarps];
    __shared__ int s_at, s_above, s_in;
    __shared__ uint32_t s_rank[kPer * kWarps];     // chosen in any case | at the border << 16, of a warp's 32 scores; then those before them
    pdl_begin();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int h = blockIdx.x, b = blockIdx.y;
    const int ip = p.indptr[b], pages = min(p.indptr[b + 1] - ip, p.max_pages);
    const long long pair = (long long)b * p.H + h;
    int32_t* blocks = p.blocks + pair * p.n_blocks;
    int32_t* block_pages = p.block_pages + pair * p.n_blocks;
    if (pages <= p.n_blocks) {
        for (int j = tid; j < p.n_blocks; j += kThreads) {
            blocks[j] = j < pages ? j : -1;
            block_pages[j] = j < pages ? p.indices[ip + j] : 0;
        }
        return;
    }
    const float* scores = p.scores + pair * p.max_pages;
    const int first = p.sinks, last = pages - p.recent;                          // blocks that a score decides on: first .. last - 1
    const int slabs = (pages + kSlab - 1) / kSlab;
    uint32_t key[kPer];
    auto load = [&](int slab) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int j = slab * kSlab + i * kThreads + tid;
            key[i] = j >= first && j < last ? ordered(scores[j]) : 0u;
        }
    };
    auto decided = [&](int slab, int i) {
        const int j = slab * kSlab + i * kThreads + tid;
        return j >= first && j < last;
    };

    // ---- the range of the scores ----
    uint32_t low = 0xffffffffu, high = 0u;
    for (int slab = 0; slab < slabs; ++slab) {
        load(slab);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (decided(slab, i)) low = min(low, key[i]), high = max(high, key[i]);
    }
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    if (lane == 0) s_low[warp] = low, s_high[warp] = high;
    __syncthreads();
    low = __reduce_min_sync(0xffffffffu, s_low[lane % kWarps]);
    high = __reduce_max_sync(0xffffffffu, s_high[lane % kWarps]);

    // ---- the border: all keys above it are chosen, and the first `room` of those that are it ----
    int room = p.n_blocks - p.sinks - p.recent;    // of those in low .. high
    uint32_t border = high;
    if (room > 0) {
        for (;;) {
            const int bits = 32 - __clz((int)(high - low)), shift = bits > 11 ? bits - 11 : 0;
            for (int i = tid; i < kBins; i += kThreads) s_bin[i] = 0;
            __syncthreads();
            for (int slab = 0; slab < slabs; ++slab) {
                if (slabs > 1) load(slab);
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                    if (decided(slab, i) && key[i] >= low && key[i] <= high) atomicAdd(&s_bin[(key[i] - low) >> shift], 1);
            }
            __syncthreads();
            int own[kOwn], sum = 0;                // thread: bins from the top down
#pragma unroll
            for (int i = 0; i < kOwn; ++i) {
                own[i] = s_bin[kBins - 1 - (tid * kOwn + i)];
                sum += own[i];
            }
            int incl = sum;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int add = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += add;
            }
            if (lane == 31) s_part[warp] = incl;
            __syncthreads();
            int above = incl - sum;
            for (int w = 0; w < warp; ++w) above += s_part[w];
#pragma unroll
            for (int i = 0; i < kOwn; ++i) {
                if (above < room && above + own[i] >= room) s_at = kBins - 1 - (tid * kOwn + i), s_above = above, s_in = own[i];
                above += own[i];
            }
            __syncthreads();
            room -= s_above;
            low += (uint32_t)s_at << shift;
            if (shift == 0 || s_in == room) break;
            high = low + min(high - low, (1u << shift) - 1u);          // not beyond the range before: with NaN in it that would end at zero
        }
        border = low;
        // a bin that is chosen whole: everything from its lower end on
        if (s_in == room) border = low - 1u, room = 0;
    }

    // ---- positions ----
    int base = 0, base_at = 0;                     // chosen in any case, and at the border, in earlier slabs
    for (int slab = 0; slab < slabs; ++slab) {
        if (slabs > 1) load(slab);
        uint32_t in[kPer], at[kPer];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int j = slab * kSlab + i * kThreads + tid;
            const bool score = decided(slab, i);
            in[i] = __ballot_sync(0xffffffffu, j < pages && (!score || (p.n_blocks > p.sinks + p.recent && key[i] > border)));
            at[i] = __ballot_sync(0xffffffffu, score && room > 0 && key[i] == border);
            if (lane == 0) s_rank[i * kWarps + warp] = (uint32_t)__popc(in[i]) | (uint32_t)__popc(at[i]) << 16;
        }
        __syncthreads();
        // kPer * kWarps sums, one of a thread at most; counts of a slab stay below 2^16
        constexpr int kSums = kPer * kWarps;
        static_assert(kSums <= kThreads, "one sum of a thread");
        uint32_t mine = tid < kSums ? s_rank[tid] : 0u, incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const uint32_t add = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += add;
        }
        if (lane == 31) s_part[warp] = (int)incl;
        __syncthreads();
        uint32_t before = incl - mine, all = 0;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += (uint32_t)s_part[w];
            all += (uint32_t)s_part[w];
        }
        if (tid < kSums) s_rank[tid] = before;
        __syncthreads();
        const uint32_t lanes = (1u << lane) - 1u;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const bool is_in = in[i] >> lane & 1u, is_at = at[i] >> lane & 1u;
            if (!is_in && !is_at) continue;
            const uint32_t r = s_rank[i * kWarps + warp];
            const int n_in = base + (int)(r & 0xffffu) + __popc(in[i] & lanes), n_at = base_at + (int)(r >> 16) + __popc(at[i] & lanes);
            if (!is_in && n_at >= room) continue;
            const int j = slab * kSlab + i * kThreads + tid, to = n_in + min(n_at, room);
            blocks[to] = j;
            block_pages[to] = p.indices[ip + j];
        }
        base += (int)(all & 0xffffu);
        base_at += (int)(all >> 16);
    }
}

template <typename T, int D>
int launch(const SelectParams& p, int B, cudaStream_t st) {
    if (p.max_pages > p.n_blocks) {
        // as many CTAs as there are turns for, up to four waves of them
        const long long turns = ((long long)p.max_pages + kScoreBlocks - 1) / kScoreBlocks, most = std::max(1ll, 64ll * sm_count() / ((long long)p.H * B));
        LEANKV_CUDA_TRY(launch_early(score_kernel<T, D>, dim3((unsigned)std::min(turns, most), (unsigned)p.H, (unsigned)B), dim3(kScoreThreads), 0, st, p));
    }
    LEANKV_CUDA_TRY(p.max_pages <= 256 * kPer ? launch_early(select_kernel<256>, dim3((unsigned)p.H, (unsigned)B), dim3(256), 0, st, p)
                                              : launch_early(select_kernel<1024>, dim3((unsigned)p.H, (unsigned)B), dim3(1024), 0, st, p));
    return LEANKV_OK;
}

}  // namespace
}  // namespace bytes
}  // namespace leankv

using namespace leankv;

extern "C" int leankv_byte_select(const leankv_byte_select_t* a, void* stream) {
    if (!a || !bytes::good_pool(&a->pool) || !bytes::good_type(a->dtype) || !a->q.data || a->batch <= 0 || a->q_heads <= 0 ||
        a->q_heads % a->pool.kv_heads != 0 || !a->kv_indptr || !a->kv_page_indices || a->max_pages_seq < 0 || a->n_blocks <= 0 || a->sinks < 0 ||
        a->recent < 1 || a->sinks > a->n_blocks - a->recent || !a->blocks || !a->block_pages || !a->scores)
        return LEANKV_EINVAL;
    if (a->batch > LEANKV_BYTES_MAX_BATCH || a->q_heads / a->pool.kv_heads > LEANKV_BYTES_MAX_GROUP || a->pool.kv_heads > 65535) return LEANKV_ELIMIT;
    if (!bytes::aligned_pool(&a->pool) || !bytes::aligned_vectors(&a->q, a->dtype, a->batch, a->q_heads, 1)) return LEANKV_EALIGN;
    bytes::SelectParams p = {};
    p.bounds = static_cast<const uint8_t*>(a->pool.bounds);
    p.H = a->pool.kv_heads, p.n_pages = a->pool.n_pages, p.G = a->q_heads / a->pool.kv_heads;
    p.max_pages = a->max_pages_seq, p.n_blocks = a->n_blocks, p.sinks = a->sinks, p.recent = a->recent;
    p.q = a->q;
    p.indptr = a->kv_indptr, p.indices = a->kv_page_indices;
    p.scores = a->scores, p.blocks = a->blocks, p.block_pages = a->block_pages;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int B = a->batch;
    if (a->pool.dim == 128)
        return a->dtype == LEANKV_BYTES_F16 ? bytes::launch<__half, 128>(p, B, st) : a->dtype == LEANKV_BYTES_BF16 ? bytes::launch<bf16, 128>(p, B, st) : bytes::launch<float, 128>(p, B, st);
    return a->dtype == LEANKV_BYTES_F16 ? bytes::launch<__half, 64>(p, B, st) : a->dtype == LEANKV_BYTES_BF16 ? bytes::launch<bf16, 64>(p, B, st) : bytes::launch<float, 64>(p, B, st);
}
