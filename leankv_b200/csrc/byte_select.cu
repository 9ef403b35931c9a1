// Which blocks of a long cache a query token reads: a cheap upper bound of its scores for every block, and the best of them.
//
// Bound of a block. For a query row q and any key k of the block, q.k = sum_d q_d k_d <= sum_d max(q_d, 0) max_d + min(q_d, 0) min_d with the
// largest and smallest key of each channel. Summed over the heads of a group that is ONE pair of vectors, P = sum_g max(q_g, 0) and N = sum_g min(q_g, 0),
// against the block's 2 * dim codes. With q rounded to whole numbers (11 bits and a sign, one power of two for the group) everything is a
// whole number: dp2a takes two 16-bit by 8-bit products at a time, sums are exact, and the choice does not depend on any order.
// A record is 2 * dim + 16 bytes against 32 * dim + 16 of the block: the scores read 1/16 of the cache.
//
// score_kernel: a lane has 16 bytes of a record and its 16 numbers of P or N in registers; dim / 8 lanes share a record.
// select_kernel: a CTA has a (sequence, kv head); a thread's scores stay in registers as whole numbers in the scores' order, and the border is found from the
// top two bits at a time by counting (three counts a step, one barrier), which knows no worst case: a histogram's atomics meet in one bin, since scores
// share their upper bits. Counting stops when the count is what is wanted. Positions come from one scan.

#include <algorithm>

#include "byte_layout.cuh"

namespace leankv {
namespace bytes {
namespace {

constexpr int kScoreThreads = 128;
constexpr int kScoreBlocks = 64;                   // of a CTA
constexpr int kPer = 16;                           // scores that a thread keeps in registers

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
    __shared__ uint32_t s_amax[kScoreThreads / 32];
    __shared__ __align__(16) short s_pn[2 * D];
    pdl_begin();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int h = blockIdx.y, b = blockIdx.z;
    const int ip = p.indptr[b], pages = min(p.indptr[b + 1] - ip, p.max_pages), first = blockIdx.x * kScoreBlocks;
    if (pages <= p.n_blocks || first >= pages) return;
    const T* q = static_cast<const T*>(p.q.data) + b * p.q.seq + (long long)h * p.G * p.q.head;
    uint32_t amax = 0;
    for (int i = tid; i < p.G * (D / 8); i += kScoreThreads) {
        Eight<T> x;
        x.load(q + (i / (D / 8)) * p.q.head + i % (D / 8) * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(x.get(e)) & 0x7fffffffu);
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    if (lane == 0) s_amax[warp] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kScoreThreads / 32; ++w) amax = max(amax, s_amax[w]);
    const bool finite = amax < 0x7f800000u;        // else every score is 0
    const float down = power_of_two(-least_exponent<2047>(min(amax, 0x7f7fffffu)));
    if (tid < D / 8) {
        int up[8], low[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) up[e] = low[e] = 0;
        for (int g = 0; g < p.G; ++g) {
            Eight<T> x;
            x.load(q + g * p.q.head + 8 * tid);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int i = finite ? __float2int_rn(x.get(e) * down) : 0;
                up[e] += max(i, 0);
                low[e] += min(i, 0);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            s_pn[8 * tid + e] = (short)up[e];
            s_pn[D + 8 * tid + e] = (short)low[e];
        }
    }
    __syncthreads();
    const int part = lane % kLanes, sub = lane / kLanes;
    int pn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) pn[e] = reinterpret_cast<const int*>(s_pn)[8 * part + e];
    constexpr int kAtOnce = 32 / kLanes;
    float* out = p.scores + ((long long)b * p.H + h) * p.max_pages;
#pragma unroll 4
    for (int i = 0; i < kScoreBlocks / (kScoreThreads / 32 * kAtOnce); ++i) {
        const int j = first + (i * (kScoreThreads / 32) + warp) * kAtOnce + sub;
        const int id = j < pages ? p.indices[ip + j] : -1;
        const bool there = (unsigned)id < (unsigned)p.n_pages;
        const uint8_t* rec = p.bounds + ((size_t)(there ? id : 0) * p.H + h) * bounds_bytes(D);
        const uint4 c = __ldg(reinterpret_cast<const uint4*>(rec) + part);
        const float scale = __ldg(reinterpret_cast<const float*>(rec + 2 * D));
        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
        int u = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            u = __dp2a_lo(pn[2 * e], (int)w[e], u);
            u = __dp2a_hi(pn[2 * e + 1], (int)w[e], u);
        }
#pragma unroll
        for (int o = 1; o < kLanes; o *= 2) u += __shfl_xor_sync(0xffffffffu, u, o);
        if (part == 0 && j < pages) out[j] = there ? __int2float_rn(u) * scale : -INFINITY;
    }
}

// fp32 numbers as whole numbers in the same order; NaN (without a sign) above infinity.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t x = __float_as_uint(v);
    return x ^ ((x >> 31) ? 0xffffffffu : 0x80000000u);
}

template <int kThreads>
__global__ void __launch_bounds__(kThreads) select_kernel(const SelectParams p) {
    constexpr int kWarps = kThreads / 32;
    __shared__ int s_count[2][3][kWarps];
    __shared__ long long s_scan[kWarps];
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
    // thread: blocks per * tid .. ; the first kPer in registers (all of them for up to kPer * kThreads blocks). Blocks that are taken or left in any case have the
    // largest and smallest key
    const float* scores = p.scores + pair * p.max_pages;
    const int per = (pages + kThreads - 1) / kThreads, base = tid * per;
    auto key_at = [&](int i) -> uint32_t {         // 0: not there
        const int j = base + i;
        if (i >= per || j >= pages) return 0u;
        if (j < p.sinks || j >= pages - p.recent) return 0xffffffffu;
        return min(max(ordered(scores[j]), 1u), 0xfffffffeu);
    };
    uint32_t key[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) key[i] = key_at(i);
    auto over_all = [&](auto&& f) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) f(i, key[i]);
        for (int i = kPer; i < per; ++i) f(i, key_at(i));
    };
    // the largest border with at least n_blocks keys at or above it
    uint32_t border = 0;
    int step = 0, at_border = pages;
    for (int shift = 30; shift >= 0 && at_border != p.n_blocks; shift -= 2, step ^= 1) {
        int n[3] = {0, 0, 0};
        over_all([&](int, uint32_t k) {
#pragma unroll
            for (uint32_t x = 0; x < 3; ++x) n[x] += k >= border + ((x + 1) << shift) ? 1 : 0;
        });
#pragma unroll
        for (int x = 0; x < 3; ++x) {
            const int sum = __reduce_add_sync(0xffffffffu, n[x]);
            if (lane == 0) s_count[step][x][warp] = sum;
        }
        __syncthreads();
        uint32_t take = 0;
#pragma unroll
        for (int x = 0; x < 3; ++x) {
            int all = lane < kWarps ? s_count[step][x][lane] : 0;
            all = __reduce_add_sync(0xffffffffu, all);
            if (all >= p.n_blocks) {
                take = x + 1;
                at_border = all;
            }
        }
        border += take << shift;
    }
    // all keys above the border, and the first of those at it
    long long mine = 0;                            // above: low half, at: high half
    over_all([&](int, uint32_t k) { mine += k > border ? 1ll : k == border && k != 0u ? 1ll << 32 : 0ll; });
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const long long add = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += add;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    long long before = incl - mine, all = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += s_scan[w];
        all += s_scan[w];
    }
    const int room = p.n_blocks - (int)(all & 0xffffffffll);      // of those at the border
    int above = (int)(before & 0xffffffffll), at = (int)(before >> 32);
    over_all([&](int i, uint32_t k) {
        if (k > border || (k == border && k != 0u && at < room)) {
            const int to = above + min(at, room);
            blocks[to] = base + i;
            block_pages[to] = p.indices[ip + base + i];
        }
        above += k > border ? 1 : 0;
        at += k == border && k != 0u ? 1 : 0;
    });
}

template <typename T, int D>
int launch(const SelectParams& p, int B, cudaStream_t st) {
    if (p.max_pages > p.n_blocks)
        LEANKV_CUDA_TRY(launch_early(score_kernel<T, D>, dim3((unsigned)((p.max_pages + kScoreBlocks - 1) / kScoreBlocks), (unsigned)p.H, (unsigned)B),
                                     dim3(kScoreThreads), 0, st, p));
    LEANKV_CUDA_TRY(p.max_pages <= 256 * kPer ? launch_early(select_kernel<256>, dim3((unsigned)p.H, (unsigned)B), dim3(256), 0, st, p)
                                              : launch_early(select_kernel<1024>, dim3((unsigned)p.H, (unsigned)B), dim3(1024), 0, st, p));
    return LEANKV_OK;
}

}  // namespace
}  // namespace bytes
}  // namespace leankv

using namespace leankv;

extern "C" int leankv_byte_select(const leankv_byte_pool_t* pool, int dtype, const leankv_vectors_t* q, int B, int q_heads, const int32_t* kv_indptr,
                                  const int32_t* kv_page_indices, int max_pages_seq, int n_blocks, int sinks, int recent, int32_t* blocks,
                                  int32_t* block_pages, float* scores, void* stream) {
    if (!bytes::good_pool(pool) || !bytes::good_type(dtype) || !q || !q->data || B <= 0 || q_heads <= 0 || q_heads % pool->kv_heads != 0 ||
        !kv_indptr || !kv_page_indices || max_pages_seq < 0 || n_blocks <= 0 || sinks < 0 || recent < 1 || sinks > n_blocks - recent || !blocks ||
        !block_pages || !scores)
        return LEANKV_EINVAL;
    if (B > LEANKV_BYTES_MAX_BATCH || q_heads / pool->kv_heads > LEANKV_BYTES_MAX_GROUP || pool->kv_heads > 65535) return LEANKV_ELIMIT;
    if (!bytes::aligned_pool(pool) || !bytes::aligned_vectors(q, dtype, B, q_heads, 1)) return LEANKV_EALIGN;
    bytes::SelectParams p = {};
    p.bounds = static_cast<const uint8_t*>(pool->bounds);
    p.H = pool->kv_heads, p.n_pages = pool->n_pages, p.G = q_heads / pool->kv_heads;
    p.max_pages = max_pages_seq, p.n_blocks = n_blocks, p.sinks = sinks, p.recent = recent;
    p.q = *q;
    p.indptr = kv_indptr, p.indices = kv_page_indices;
    p.scores = scores, p.blocks = blocks, p.block_pages = block_pages;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (pool->dim == 128)
        return dtype == LEANKV_BYTES_F16 ? bytes::launch<__half, 128>(p, B, st) : dtype == LEANKV_BYTES_BF16 ? bytes::launch<bf16, 128>(p, B, st) : bytes::launch<float, 128>(p, B, st);
    return dtype == LEANKV_BYTES_F16 ? bytes::launch<__half, 64>(p, B, st) : dtype == LEANKV_BYTES_BF16 ? bytes::launch<bf16, 64>(p, B, st) : bytes::launch<float, 64>(p, B, st);
}
