// Causal attention of a prompt chunk over the 8-bit pages, on tcgen05.
//
// A CTA takes 256 rows of a kv head, two tiles of 128 (query token, query head) pairs, against 128 keys (eight pages) at a time. Both row tiles use the same
// keys and values, so that the codes are turned into fp16 operands once for 256 rows, inside this kernel:
//   warps 8 - 11  pages from memory into registers a whole key tile ahead; code + 128 behind the byte 0x64 is the fp16 number 1152 + code, one
//                 fused multiply-add makes it exact (and scales values); 16-byte (8-byte) stores fill core matrices in order
//   warp 12       S_r = Q_r K^T and O_r += P_r V of both row tiles, one thread issues
//   warp 13       the scales of a key tile: the keys' for the rows, the values' exponents for rows and converting warps
//   warps 14, 15  ask for pages into L2, then wait
//   warps 0 - 7   a thread a row: scores from tensor memory, maximum, weights back over the scores as fp16
// A row's 128 scores stay in registers, which the row warps take from the others (of the launch's 128 each: 192, converting warps 88, the last four 40).
// The row tiles alternate: the products of one run under the exponentials of the other. Tensor memory: S of both (128 columns each), O of both (dim each), for dim 64 weights.
//
// Exactness. Keys enter as their codes (the scale, one number for 16 keys, is multiplied to the scores in fp32), queries in fp16 with a power of two taken out
// of each row. Values enter as code * 2^(e - t), t the largest exponent of the key tile's pages, exactly; the tile's t goes into the weights, which are
// 2^(score - m + t - r) against a row's own references: m for its sum, r for the exponents of the values that count for it. So no row depends on values that it
// does not see, and a row of small ones is as good as any. (One exponent for all pages of the CTA, which was simpler, turned rows of values 2^-25 below a later token's into zeros.) Where the
// pages of a tile are more than kFlat exponents apart, their codes enter as they are and each page's e goes into its weights; such a tile, or one whose t is far from
// the row's r, has its exponentials for sums and outputs apart. There a token counts for r only if one of its codes is not zero (a block's scale may be another token's, one
// that the row does not see), and r comes down to where the outputs are when the weights of a later tile would be far below them. Weights are fp16 (2^-11), with references such that 2^-21 of a row's largest term still
// has all its places (2^-13 under a tile whose exponents are kFlat apart; a row's largest term is its largest weight times that block's scale); their sum is fp32 before that rounding.
//
// Bound: a key tile is 4 x 512 tensor cycles (dim 128) and 2 x 1024 cycles of ex2; operand reads (192 KB) and the converted tiles (64 KB written) take the
// same time of shared memory's 128 bytes a cycle. It takes some 3600: a row tile's rows have 128 scores for 2400 cycles and then nothing for 1250, until the last weights
// are multiplied (400) and the next scores formed over them (580, and 270 on the way); two row tiles are what tensor memory holds, and what one leaves the other does not fill.
// 4096 tokens, 8 kv heads of 4, bf16: 145 us, 948 TFLOP/s; 8192, fp16: 490, 1120; 512 behind 3584: 46; dim 64, 4096: 117. (With one exponent a CTA 140, 479, 48, 118: a warp for the
// scales gives the converting warps back the registers that the rows' second reference takes.)
//
// Long caches behind few rows: a cluster's CTAs share the keys of a block of rows, each leaves its sums in its shared memory, and each joins a part of the rows from there
// (through the workspace and a second kernel: 512 behind 3584 52.4 us). Where a cluster of eight leaves SMs free several clusters share them, and their sums meet in the workspace.

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "byte_cluster.cuh"
#include "byte_layout.cuh"
#include "byte_workspace.cuh"
#include "tile_softmax.cuh"

namespace leankv {
namespace bytes {
namespace {

constexpr int kRowsTile = 128, kTiles = 2;
constexpr int kKeysTile = 128, kPagesTile = kKeysTile / kPage;
constexpr int kRowWarps = 8, kConvWarps = 4, kMmaWarp = kRowWarps + kConvWarps, kScaleWarp = kMmaWarp + 1;
constexpr int kThreads = 512;                         // four warpgroups: registers change hands by warpgroup
constexpr int kPagesWarp = kPagesTile / kConvWarps;
constexpr float kNoRef = -3.402823466e38f;            // a maximum before any score: below all of them, and finite, so that masked scores give weight 0
constexpr float kLift = 7.f, kReach = 15.f;           // the reference of a row is its maximum - kLift when it moves, and moves beyond kReach above it
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kScaleSlots = 4;
constexpr int kFlat = 8;                              // value scales of a key tile share an exponent if theirs are no further apart: each step costs a row's weights a bit of fp16's range
constexpr int kPaged = 1024;                          // on top of a tile's exponent: its pages keep their own
constexpr float kLeap = 24.f;                         // a tile's exponent less a row's r, beyond which r moves for tokens only that hold more than zeros
constexpr float kFar = 60.f, kExact = 4194304.f;      // a tile's exponent against the row's, and a row's reference, up to which one exponential serves outputs and sum
constexpr float kLeast = -1000.f;                     // of r: weights of 2^-1000 and less are none in any type

__host__ __device__ constexpr uint32_t q_bytes(int dim) { return kRowsTile * dim * 2; }
__host__ __device__ constexpr uint32_t k_bytes(int dim) { return kKeysTile * dim * 2; }
constexpr size_t smem_bytes(int dim) { return kTiles * q_bytes(dim) + 4 * k_bytes(dim) + 1024; }

struct PromptParams {
    const uint8_t* chunks;
    int n_pages, H, B, G, tokens, tile_tokens;        // tokens of a row tile
    leankv_vectors_t q, out;
    float scale;                                      // softmax scale * log2(e)
    const int32_t* indptr;
    const int32_t* indices;
    const int32_t* last;
    int first_blocks;                                 // blocks of rows that start together
    int n_splits, ctas;                               // shares of a block's keys; CTAs of a cluster. More shares than that are joined in the workspace
    float* partials;                                  // [block of a kv head][cluster][256 rows][dim + 2]
    unsigned* counters;                               // [block of a kv head][CTA of a cluster], zero between launches
    int* status;
};

enum { kQFull, kKFull = kQFull + 2, kVFull = kKFull + 2, kKFree = kVFull + 2, kVFree = kKFree + 2, kSFull = kVFree + 2, kPHalf = kSFull + 2, kPFull = kPHalf + 2, kSRead = kPFull + 2, kPvDone = kSRead + 2, kBars = kPvDone + 2 };

// Codes of a word's bytes 0, 1 / 2, 3 times s: (1024 + byte) s - 1152 s in one rounding of an exact number.
__device__ __forceinline__ uint32_t codes_times(uint32_t w, uint32_t sel, __half2 s, __half2 off) {
    const uint32_t x = __byte_perm(w, 0x64646464u, sel);
    const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&x), s, off);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// Position c of a page's 16 in the operands: the values' words hold tokens 2t, 2t + 1, 2t + 8, 2t + 9, and keys follow the same order.
__host__ __device__ constexpr int token_at(int c) { return 2 * (c >> 2) + (c & 1) + 8 * ((c >> 1) & 1); }

__device__ __forceinline__ float largest3(uint32_t a, uint32_t b, uint32_t c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
    return d;
}

// kShared: a cluster's CTAs share the keys of a block of rows. A kernel of its own: with both ends in one, and their registers, the row loop of either took 5 to 10 % longer
// (8192 tokens: 523 against 491 us).
template <typename T, int D, bool kShared>
__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(const PromptParams p) {
    extern __shared__ __align__(16) uint8_t s_raw[];
    __shared__ __align__(8) uint64_t s_bar[kBars];
    __shared__ uint32_t s_tmem;
    __shared__ __align__(16) float s_ks[kScaleSlots][kPagesTile];
    __shared__ float s_ve[kScaleSlots][kPagesTile];                   // the values' exponent of each page
    __shared__ __half2 s_times[kScaleSlots][kPagesTile];              // what a page's value codes are multiplied with
    __shared__ float s_tile[kScaleSlots];                             // the largest of a key tile, kPaged more where its pages keep their own
    __shared__ __align__(8) float2 s_ml[kTiles * kRowsTile];          // reference and sum of a row
    __shared__ int s_last;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    uint8_t* base = s_raw + ((1024u - (umma::smem_addr(s_raw) & 1023u)) & 1023u);
    uint8_t* s_q = base;                              // two row tiles
    uint8_t* s_k = s_q + kTiles * q_bytes(D);         // two key tiles
    uint8_t* s_v = s_k + 2 * k_bytes(D);              // two value tiles
    auto bar = [&](int b) { return umma::smem_addr(&s_bar[b]); };
    auto wait2 = [&](int b, int j) { return umma::bar_wait(bar(b + (j & 1)), (uint32_t)((j >> 1) & 1)); };      // pairs by key tile
    auto wait1 = [&](int b, int j) { return umma::bar_wait(bar(b), (uint32_t)(j & 1)); };                       // one for every key tile
    auto all = [&](bool done) { return __all_sync(0xffffffffu, done) != 0; };

    if (tid == 0) {
        for (int b = 0; b < kBars; ++b) {
            const int count = b >= kKFull && b < kVFull ? 32 * (kConvWarps + 1) : b >= kVFull && b < kKFree ? 32 * kConvWarps : b < kKFull || (b >= kPHalf && b < kPvDone) ? kRowsTile : 1;
            umma::bar_init_n(bar(b), count);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // tensor memory behind the wait (a launch ahead may hold some); later launches come when this one ends
    pdl_wait();
    if (warp == kMmaWarp) umma::tmem_alloc_n(umma::smem_addr(&s_tmem), 512);
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    // dim 64 leaves room for weights of their own: the next scores need not wait for the value product (4096 tokens 123 -> 117 us)
    constexpr bool kApart = D == 64;
    constexpr int kPColumns = kApart ? kKeysTile / 2 : kKeysTile;
    const uint32_t tm_s = tmem, tm_o = tmem + kTiles * kKeysTile, tm_p = kApart ? tm_o + kTiles * D : tm_s;

    const int kvh = blockIdx.x % p.H, b = blockIdx.x / p.H, split = kShared ? blockIdx.z : 0;
    const int ip = p.indptr[b], pages = p.indptr[b + 1] - ip;
    const int start = pages > 0 ? (pages - 1) * kPage + p.last[b] - p.tokens : -p.tokens;      // position of the chunk's first token
    const int block = (int)gridDim.y - 1 - (int)blockIdx.y;                                    // the longest first
    const int tok0 = block * kTiles * p.tile_tokens, last_tok = min(tok0 + kTiles * p.tile_tokens, p.tokens) - 1;
    const int n_all = start + last_tok < 0 ? 0 : (start + last_tok) / kKeysTile + 1;
    const int t0 = kShared ? (int)((long long)n_all * split / p.n_splits) : 0, n = kShared ? (int)((long long)n_all * (split + 1) / p.n_splits) - t0 : n_all;
    const int page0 = t0 * kPagesTile;

    bool ok = true;
    const int tile = warp >> 2, row = tid & (kRowsTile - 1);             // of the row threads
    const int tok = tok0 + tile * p.tile_tokens + row / p.G;
    const bool real = warp < kRowWarps && row < p.tile_tokens * p.G && tok < p.tokens;
    const int head = kvh * p.G + row % p.G;
    if (warp >= kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == kMmaWarp) {
            // ---- products ----
            auto scores = [&](int r, int j) {
                if (umma::elect()) {
                    const uint64_t a = umma::desc_k(umma::smem_addr(s_q + r * q_bytes(D)), D / 8), c = umma::desc_k(umma::smem_addr(s_k + (j & 1) * k_bytes(D)), D / 8);
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks)
                        umma::mma_f16_n(tm_s + r * kKeysTile, a + (uint64_t)ks * (2 * umma::kLbo >> 4), c + (uint64_t)ks * (2 * umma::kLbo >> 4), umma::idesc_n(kKeysTile), ks > 0);
                    umma::commit(bar(kSFull + r));
                    if (r == kTiles - 1 && j + 2 < n) umma::commit(bar(kKFree + (j & 1)));
                }
                __syncwarp();
            };
            auto values = [&](int r, int j) {              // both parts of a row tile's weights
                const uint64_t c = umma::desc_k(umma::smem_addr(s_v + (j & 1) * k_bytes(D)), kKeysTile / 8);
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    ok = ok && all(wait1((part == 0 ? kPHalf : kPFull) + r, j));
                    if (!ok) return;
                    umma::fence_after_sync();
                    if (umma::elect()) {
#pragma unroll
                        for (int ks = part * 6; ks < 6 + part * 2; ++ks)
                            umma::mma_f16_ts(tm_o + r * D, tm_p + r * kPColumns + 8 * ks, c + (uint64_t)ks * (2 * umma::kLbo >> 4), umma::idesc_n(D), j > 0 || ks > 0);
                        if (part == 1) {
                            umma::commit(bar(kPvDone + r));
                            if (r == kTiles - 1 && j + 2 < n) umma::commit(bar(kVFree + (j & 1)));
                        }
                    }
                    __syncwarp();
                }
            };
            if (n > 0) ok = all(wait2(kKFull, 0));
            for (int r = 0; r < kTiles && ok && n > 0; ++r) {
                ok = all(wait1(kQFull + r, 0));
                umma::fence_after_sync();
                if (ok) scores(r, 0);
            }
            for (int j = 0; j < n && ok; ++j) {
                for (int r = 0; r < kTiles && ok; ++r) {
                    if constexpr (kApart) {                // as soon as the ones before have been read; then the other row tile's weights
                        if (j + 1 < n) {
                            if (r == 0) ok = all(wait2(kKFull, j + 1));
                            ok = ok && all(wait1(kSRead + r, j));
                            umma::fence_after_sync();
                            if (ok) scores(r, j + 1);
                        }
                        const int vr = 1 - r, vj = j - vr;
                        if (vj < 0 || !ok) continue;
                        if (vr == 0) ok = all(wait2(kVFull, vj));
                        values(vr, vj);
                    } else {
                        if (r == 0) ok = all(wait2(kVFull, j));
                        values(r, j);
                        if (ok && j + 1 < n) {             // its scores go over these weights
                            if (r == 0) ok = all(wait2(kKFull, j + 1));
                            ok = ok && all(wait1(kPvDone + r, j));
                            umma::fence_after_sync();
                            if (ok) scores(r, j + 1);
                        }
                    }
                }
            }
            if (kApart && ok && n > 0) values(1, n - 1);
        } else if (warp == kScaleWarp) {
            // ---- scales: lane i < 2 kPagesTile has the values' (the second eight the keys') of page i % kPagesTile of a key tile ----
            auto scale_of = [&](int j) -> uint32_t {       // as bits; 0: no such page
                const int i = page0 + j * kPagesTile + lane % kPagesTile;
                const int id = lane >= 2 * kPagesTile || j >= n || i >= pages ? -1 : p.indices[ip + i];
                return (unsigned)id >= (unsigned)p.n_pages ? 0u
                     : __ldg(reinterpret_cast<const uint32_t*>(p.chunks + ((size_t)id * p.H + kvh) * chunk_bytes(D) + 2 * half_bytes(D)) + (lane < kPagesTile ? 1 : 0));
            };
            uint32_t scale = scale_of(0);
            for (int j = 0; j < n && ok; ++j) {
                if (j >= 2) ok = all(wait2(kKFree, j - 2));
                if (!ok) break;
                const uint32_t next = scale_of(j + 1);
                // the values' exponents, of pages that are there and hold numbers
                const bool counts = lane < kPagesTile && scale - 1u < 0x7f7fffffu;
                const int e = (int)(scale >> 23) - 127, slot = j & (kScaleSlots - 1);
                const int top = __reduce_max_sync(0xffffffffu, counts ? e : -127);
                const bool flat = top - __reduce_min_sync(0xffffffffu, counts ? e : top) <= kFlat;
                const uint32_t key_scale = __shfl_down_sync(0xffffffffu, scale, kPagesTile);
                if (lane < kPagesTile) {
                    s_ks[slot][lane] = __uint_as_float(scale > 0x7f800000u ? scale : key_scale);
                    s_ve[slot][lane] = counts ? (float)(flat ? top : e) : -1000.f;
                    // 2^(e - top) in fp16, 1 where the pages keep their own; 0 for a scale that is no number (its codes are zeros)
                    s_times[slot][lane] = __half2half2(__ushort_as_half((unsigned short)(!counts ? 0 : flat ? (e - top + 15) << 10 : 0x3c00)));
                    if (lane == 0) s_tile[slot] = (float)(flat ? top : top + kPaged);
                }
                umma::bar_arrive(bar(kKFull + (j & 1)));
                scale = next;
            }
        } else if ((int)blockIdx.y < p.first_blocks) {
            // ---- the CTAs that start together walk the same pages: each asks for a part of them into L2 (4096 tokens of six caches in turn 150 -> 145 us) ----
            constexpr int kAskers = kThreads - 32 * (kScaleWarp + 1);
            const int to = kShared ? min(page0 + n * kPagesTile, pages) : pages;
            for (int i = page0 + blockIdx.y + p.first_blocks * (tid - 32 * (kScaleWarp + 1)); i < to; i += p.first_blocks * kAskers) {
                const int id = p.indices[ip + i];
                if ((unsigned)id < (unsigned)p.n_pages)
                    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.chunks + ((size_t)id * p.H + kvh) * chunk_bytes(D)), "r"(chunk_bytes(D)) : "memory");
            }
        }
    } else if (warp >= kRowWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        // ---- codes to operands: a warp has pages kPagesWarp w .. of every key tile ----
        const int first = (warp - kRowWarps) * kPagesWarp;
        // values: lanes of half a warp have eight channels of the same tokens' half, so that their stores fill a core matrix
        const int g = lane >> 1 & 7, t = 2 * (lane >> 4) + (lane & 1);
        constexpr int kLoads = D / 32;                // 16-byte pieces of a lane, of keys and of values
        uint4 kr[kPagesWarp][kLoads], vr[kPagesWarp][kLoads];
        auto page_of = [&](int j) -> int {            // lane i < kPagesWarp: page id of key tile j, or -1
            const int i = page0 + j * kPagesTile + first + lane;
            if (lane >= kPagesWarp || j >= n || i >= pages) return -1;
            const int id = p.indices[ip + i];
            if ((unsigned)id >= (unsigned)p.n_pages) {
                atomicOr(p.status, kBadPage);
                return -1;
            }
            return id;
        };
        auto chunk_of = [&](int ids, int i) -> const uint8_t* {
            const int id = __shfl_sync(0xffffffffu, ids, i);
            return id < 0 ? nullptr : p.chunks + ((size_t)id * p.H + kvh) * chunk_bytes(D);
        };
        const uint4 none = make_uint4(kZeroCodes, kZeroCodes, kZeroCodes, kZeroCodes);
        // keys: lane (position of eight, 16 bytes): positions 8 (x & 1) .., channels 64 (x >> 1) + 16 (lane / 8) ..; eight lanes fill a core matrix
        auto load_keys = [&](const uint8_t* chunk, int i) {
#pragma unroll
            for (int x = 0; x < kLoads; ++x)
                kr[i][x] = chunk == nullptr ? none : __ldg(reinterpret_cast<const uint4*>(chunk + (x >> 1) * 1024 + token_at(8 * (x & 1) + (lane & 7)) * 64 + (lane >> 3) * 16));
        };
        auto load_values = [&](const uint8_t* chunk, int i) {
#pragma unroll
            for (int x = 0; x < kLoads; ++x)
                vr[i][x] = chunk == nullptr ? none : __ldg(reinterpret_cast<const uint4*>(chunk + half_bytes(D)) + x * 32 + 4 * g + t);
        };
        int ids = page_of(0), ids_next = page_of(1);
#pragma unroll
        for (int i = 0; i < kPagesWarp; ++i) {
            const uint8_t* chunk = chunk_of(ids, i);
            load_keys(chunk, i);
            load_values(chunk, i);
        }
        const __half2 one = __half2half2(__ushort_as_half(0x3c00)), minus = __half2half2(__ushort_as_half(0xe480));      // 1, -1152
        for (int j = 0; j < n && ok; ++j) {
            if (j >= 2) ok = all(wait2(kKFree, j - 2));
            if (!ok) break;
            ids = ids_next;
            ids_next = page_of(j + 2);
            uint8_t* k_to = s_k + (j & 1) * k_bytes(D);
#pragma unroll
            for (int i = 0; i < kPagesWarp; ++i) {
#pragma unroll
                for (int x = 0; x < kLoads; ++x) {
                    const uint32_t w[4] = {kr[i][x].x, kr[i][x].y, kr[i][x].z, kr[i][x].w};
                    const int at = 16 * (first + i) + 8 * (x & 1) + (lane & 7);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t a = w[2 * half], c = w[2 * half + 1];
                        *reinterpret_cast<uint4*>(k_to + umma::offset_k(at, 8 * (x >> 1) + 2 * (lane >> 3) + half, D / 8)) =
                            make_uint4(codes_times(a, 0x4140, one, minus), codes_times(a, 0x4342, one, minus), codes_times(c, 0x4140, one, minus), codes_times(c, 0x4342, one, minus));
                    }
                }
                load_keys(chunk_of(ids, i), i);
            }
            umma::fence_operands();
            umma::bar_arrive(bar(kKFull + (j & 1)));
            ok = all(wait2(kKFull, j) && (j < 2 || wait2(kVFree, j - 2)));             // the first for the scales
            if (!ok) break;
            uint8_t* v_to = s_v + (j & 1) * k_bytes(D);
#pragma unroll
            for (int i = 0; i < kPagesWarp; ++i) {
                const __half2 s = s_times[j & (kScaleSlots - 1)][first + i], off = __hmul2(s, minus);
#pragma unroll
                for (int x = 0; x < kLoads; ++x) {
                    const uint32_t w[4] = {vr[i][x].x, vr[i][x].y, vr[i][x].z, vr[i][x].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        *reinterpret_cast<uint2*>(v_to + umma::offset_k(8 * (4 * x + k) + g, 2 * (first + i) + (t >> 1), kKeysTile / 8) + 8 * (t & 1)) =
                            make_uint2(codes_times(w[k], 0x4140, s, off), codes_times(w[k], 0x4342, s, off));
                }
                load_values(chunk_of(ids, i), i);
            }
            umma::fence_operands();
            umma::bar_arrive(bar(kVFull + (j & 1)));
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
        // ---- queries: a thread a row, fp16 with the row's power of two taken out ----
        uint8_t* q_to = s_q + tile * q_bytes(D);
        // a warp's 32 rows come by whole vectors and turn to a row a thread through where they will lie (a thread that asks for its own row's pieces: 32 rows in one load)
        constexpr int kPieces = D / 8;
        Eight<T> x[kPieces];
        uint32_t amax = 0;
        const long long mine = real ? (long long)head * p.q.head + (long long)tok * p.q.token : -1;
        const T* src = static_cast<const T*>(p.q.data) + b * p.q.seq + lane % kPieces * 8;
        uint8_t* turn = q_to + (warp & 3) * (q_bytes(D) / 4);
        auto at = [&](int r, int piece) { return reinterpret_cast<uint4*>(turn + r * (16 * kPieces) + ((piece ^ r) & (kPieces - 1)) * 16); };
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const long long from = __shfl_sync(0xffffffffu, mine, (32 / kPieces) * i + lane / kPieces);
            if (from >= 0) x[i].load(src + from);
            else x[i].zero();
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) *at((32 / kPieces) * i + lane / kPieces, lane % kPieces) = x[i].a;
        __syncwarp();
#pragma unroll
        for (int c = 0; c < kPieces; ++c) x[c].a = *at(lane, c);
        __syncwarp();
        int e2 = 0;
        if constexpr (std::is_same<T, bf16>::value) {
#pragma unroll
            for (int c = 0; c < D / 8; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(x[c].get(e)) & 0x7fffffffu);
            e2 = max((int)(amax >> 23) - 127 - 14, -126);
        }
        const float down = power_of_two(-e2);
        const float factor = power_of_two(e2) * p.scale;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
            uint32_t w[4];
            if constexpr (std::is_same<T, bf16>::value) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const __half2 v = __floats2half2_rn(x[c].get(2 * e) * down, x[c].get(2 * e + 1) * down);
                    w[e] = *reinterpret_cast<const uint32_t*>(&v);
                }
            } else {
                w[0] = x[c].a.x, w[1] = x[c].a.y, w[2] = x[c].a.z, w[3] = x[c].a.w;
            }
            *reinterpret_cast<uint4*>(q_to + umma::offset_k(row, c, D / 8)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        // for the scales. The wait for key tile j comes before what the next tile of its buffer depends on: the queries, later the weights of tile j - 1
        if (n > 0) ok = all(wait2(kKFull, 0));
        umma::fence_operands();
        umma::bar_arrive(bar(kQFull + tile));

        // ---- rows ----
        // O = sum 2^(score - m - r) value, l = sum 2^(score - m). m and r are whole numbers, so that the tile's t - r is exact beside a score - m
        float m = kNoRef, r = 0.f, l = 0.f;
        float lowest = -kFlat;                         // a tile's exponent less r, below which r is looked at again
        bool large = false;                            // some row's m is beyond kExact
        const int lane0 = 32 * (warp & 3);
        const int qpos = start + (real ? tok : last_tok);       // rows that are none see what the last token sees; nothing of theirs is kept
        const uint32_t tm = tm_s + tile * kKeysTile, tp = tm_p + tile * kPColumns, to = tm_o + tile * D;
        for (int j = 0; j < n && ok; ++j) {
            ok = all(wait1(kSFull + tile, j));
            if (!ok) break;
            umma::fence_after_sync();
            uint32_t s[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) umma::ld32_async(s[c], tm, lane0, 32 * c);
            float ks[kPagesTile];
            const float4* scales = reinterpret_cast<const float4*>(s_ks[j & (kScaleSlots - 1)]);
#pragma unroll
            for (int i = 0; i < kPagesTile / 4; ++i) {
                const float4 v = scales[i];
                ks[4 * i] = v.x * factor, ks[4 * i + 1] = v.y * factor, ks[4 * i + 2] = v.z * factor, ks[4 * i + 3] = v.w * factor;
            }
            umma::settle(s[0]);
            umma::settled(s[1]);
            umma::settled(s[2]);
            umma::settled(s[3]);
            if constexpr (kApart) {
                umma::fence_before_sync();
                umma::bar_arrive(bar(kSRead + tile));
            }
            const int k1 = qpos - (t0 + j) * kKeysTile;                  // the row's last key of the tile
            const bool cut = __any_sync(0xffffffffu, k1 < kKeysTile - 1);
            if (cut) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int x = 0; x < 32; ++x)
                        if (32 * c + (x & 16) + token_at(x & 15) > k1) s[c][x] = 0xff800000u;
            }
            float best = kNoRef;
#pragma unroll
            for (int i = 0; i < kPagesTile; ++i) {
                const uint32_t* v = &s[i >> 1][16 * (i & 1)];
                float a = largest3(v[0], v[1], v[2]), c = largest3(v[3], v[4], v[5]);
                a = largest3(__float_as_uint(a), v[6], v[7]), c = largest3(__float_as_uint(c), v[8], v[9]);
                a = largest3(__float_as_uint(a), v[10], v[11]), c = largest3(__float_as_uint(c), v[12], v[13]);
                best = fmaxf(best, largest3(__float_as_uint(a), __float_as_uint(c), __float_as_uint(fmaxf(__uint_as_float(v[14]), __uint_as_float(v[15])))) * ks[i]);
            }
            if constexpr (kApart) {                    // neither outputs nor weights are in use any more
                if (j > 0) ok = all(wait1(kPvDone + tile, j - 1));
                umma::fence_after_sync();
            }
            // one exponential a weight, 2^(score - m + t - r); the tile's sum of them, times 2^(r - t), is its part of l
            const float of_tile = s_tile[j & (kScaleSlots - 1)];
            float less = (of_tile - r) - m, back_to_l = ex2(r - of_tile);
            if (__builtin_expect(__any_sync(0xffffffffu, best - m > kReach - fmaxf(of_tile - r, 0.f) || of_tile - r > kFar || of_tile - r < lowest || large), 0)) {
                const float* ve = s_ve[j & (kScaleSlots - 1)];
                // where the exponents would move r far, only tokens with a code that is not zero count
                const bool paged = of_tile > 0.5f * kPaged, sparse = paged || __any_sync(0xffffffffu, of_tile - r > kLeap);
                float e = of_tile;
                uint32_t eight = 0;
                auto filled_of = [&](int c) {          // tokens 32 c .. as bits
                    uint32_t bits = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) bits |= __shfl_sync(0xffffffffu, eight, 4 * c + i) << 8 * i;
                    return bits;
                };
                if (__builtin_expect(sparse, 0)) {
                    if (!all(wait2(kVFull, j))) l = NAN;       // (the converting warps report it)
                    const uint8_t* from = s_v + (j & 1) * k_bytes(D) + (lane & 15) * umma::kLbo + (lane >> 4) * (D / 16) * (kKeysTile / 8) * umma::kLbo;
                    uint4 any = make_uint4(0, 0, 0, 0);
#pragma unroll 1
                    for (int i = 0; i < D / 2; ++i) {              // eight tokens of a channel
                        const uint4 w = *reinterpret_cast<const uint4*>(from + (i >> 3) * (kKeysTile / 8) * umma::kLbo + ((i + lane) & 7) * 16);
                        any.x |= w.x, any.y |= w.y, any.z |= w.z, any.w |= w.w;
                    }
                    const uint32_t words[4] = {any.x, any.y, any.z, any.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) eight |= (min(words[i] & 0x7fffu, 1u) | min(words[i] >> 16 & 0x7fffu, 1u) << 1) << 2 * i;
                    eight |= __shfl_xor_sync(0xffffffffu, eight, 16);
                    float most = kNoRef;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint32_t filled = filled_of(c);
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            float top = -INFINITY;
#pragma unroll
                            for (int x = 16 * half; x < 16 * half + 16; ++x) {
                                const uint32_t keep = (uint32_t)((int)(filled << (31 - x)) >> 31);
                                top = fmaxf(top, __uint_as_float((s[c][x] & keep) | (0xff800000u & ~keep)));
                            }
                            most = fmaxf(most, (__fmul_rn(top, ks[2 * c + half]) - best) + ve[2 * c + half]);      // -inf for a page that the row does not see
                        }
                    }
                    e = ceilf(most);
                }
                const bool raise = best - m > kReach - fmaxf(e - r, 0.f), sink = !raise && j > 0 && e > kNoRef && e - r < lowest && best > kNoRef;
                const float now = raise ? fmaxf(m, floorf(best) - kLift) : m, up = now - m, fit = floorf(best - now) + e - kLift;
                float r_now = raise ? fmaxf(fmaxf(r - up, fit), kLeast) : r;
                if (raise) lowest = -kFlat;
                if (__any_sync(0xffffffffu, sink)) {
                    // weights far down: r may come from tokens that turned out to add little. Not below where the outputs are
                    uint32_t top = 0;
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 16) {
                        uint32_t o[16];
                        umma::ld16(o, to, lane0, c0);
#pragma unroll
                        for (int x = 0; x < 16; ++x) top = max(top, o[x] & 0x7fffffffu);
                    }
                    const float there = top == 0 ? kNoRef : r + (float)((int)(top >> 23) - 127) - kLift;
                    if (sink) {
                        r_now = fminf(r, fmaxf(fmaxf(fit, there), kLeast));
                        if (there >= fit) lowest = -kFar;          // r is where the outputs are
                    }
                }
                if (__any_sync(0xffffffffu, raise || r_now != r)) {
                    // nothing is being added to these outputs: the scores were asked for behind the last value product
                    const float f = ex2((r - r_now) - up);
                    l *= ex2(-up);
                    m = now;
                    r = r_now;
                    if (j > 0) scale_outputs(to, lane0, D, f);
                    large = __any_sync(0xffffffffu, m != kNoRef && fabsf(m) > kExact);
                    less = (of_tile - r) - m;
                    back_to_l = ex2(r - of_tile);
                }
                if (__builtin_expect(sparse || large || __any_sync(0xffffffffu, fabsf(of_tile - r) > kFar), 0)) {
                    // sums here, and scores that have their page's exponent less r already. Products rounded as the maximum's was: what a fused one has more of a score
                    // beyond kExact may be many powers of two
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
#pragma unroll
                        for (int x = 0; x < 32; ++x) {
                            const float at = __uint_as_float(s[c][x]), w = __fmul_rn(at, ks[2 * c + (x >> 4)]) - m;
                            if (at != -INFINITY) l += ex2(w);
                            s[c][x] = __float_as_uint(w + (ve[2 * c + (x >> 4)] - r));
                        }
                    }
                    if (sparse) {                      // weights of what is zero are of no use, and may be beyond fp16
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const uint32_t filled = filled_of(c);
#pragma unroll
                            for (int x = 0; x < 32; ++x) {
                                const uint32_t keep = (uint32_t)((int)(filled << (31 - x)) >> 31);
                                s[c][x] = (s[c][x] & keep) | (0xff800000u & ~keep);
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kPagesTile; ++i) ks[i] = 1.f;
                    less = back_to_l = 0.f;
                }
            }
            Two sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
            // the masked form apart from the other: one loop for both spends two instructions a weight on masks that are not there
            auto weights = [&](auto masked) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t w16[16];
#pragma unroll
                    for (int x = 0; x < 32; x += 2) {
                        const float k = ks[2 * c + (x >> 4)];
                        Two w = fma2({__uint_as_float(s[c][x]), __uint_as_float(s[c][x + 1])}, {k, k}, {less, less});
                        w.x = ex2(w.x);
                        w.y = ex2(w.y);
                        if constexpr (decltype(masked)::value) {         // a scale that is no number does not reach a row that does not see its block
                            if (32 * c + (x & 16) + token_at(x & 15) > k1) w.x = 0.f;
                            if (32 * c + (x & 16) + token_at((x + 1) & 15) > k1) w.y = 0.f;
                        }
                        sum[(x >> 1) & 1] = add2(sum[(x >> 1) & 1], w);
                        const __half2 h = __floats2half2_rn(w.x, w.y);
                        w16[x / 2] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                    umma::st16_async(w16, tp, lane0, 16 * c);
                    if (c == 2) {                      // the first 96 keys' product begins (64: 157 us where this takes 154)
                        umma::stored();
                        umma::fence_before_sync();
                        umma::bar_arrive(bar(kPHalf + tile));
                    }
                }
            };
            if (cut) weights(std::true_type());
            else weights(std::false_type());
            l = fmaf((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y), back_to_l, l);
            umma::stored();
            if (j + 1 < n) ok = all(wait2(kKFull, j + 1));
            umma::fence_before_sync();
            umma::bar_arrive(bar(kPFull + tile));
        }
        if (ok && n > 0) ok = all(wait1(kPvDone + tile, n - 1));
        umma::fence_after_sync();
        if (!ok && lane == 0) atomicOr(p.status, kTimedOut);

        // ---- out ----
        const float inv = !ok ? NAN : l == 0.f ? 0.f : 1.f / l;
        const float back = r < -126.f ? ex2(r + 64.f) * 5.421010862427522e-20f : ex2(r);       // 2^r, 2^-64 of it apart where r is below fp32's exponents
        const int reciprocal = (65535 + p.G) / p.G;   // i / G is i * reciprocal >> 16 for i below 128
        auto target = [&](int r) -> T* {              // where row r of the CTA's 256 goes, or null
            const int in_tile = r & (kRowsTile - 1), in_tok = in_tile * reciprocal >> 16, r_tok = tok0 + (r / kRowsTile) * p.tile_tokens + in_tok;
            if (in_tile >= p.tile_tokens * p.G || r_tok >= p.tokens) return nullptr;
            return static_cast<T*>(p.out.data) + b * p.out.seq + (long long)(kvh * p.G + in_tile - in_tok * p.G) * p.out.head + (long long)r_tok * p.out.token;
        };
        const float by = inv * back;
        // pieces of 16 bytes, in an order of each row's own so that neither side meets a bank twice
        if constexpr (!kShared) {
            // a warp's 32 rows through its own part of the queries (all scores have been formed), so that whole vectors leave
            uint32_t o[D / 32][32];
            if (n > 0) {
#pragma unroll
                for (int c = 0; c < D / 32; ++c) umma::ld32_async(o[c], to, lane0, 32 * c);
                umma::settle(o[0]);
#pragma unroll
                for (int c = 1; c < D / 32; ++c) umma::settled(o[c]);
            }
            auto number = [&](int c) { return n > 0 ? __uint_as_float(o[c >> 5][c & 31]) * by : 0.f; };
            uint8_t* stage = s_q + tile * q_bytes(D) + (warp & 3) * (q_bytes(D) / 4);
            __syncwarp();
#pragma unroll
            for (int c = 0; c < kPieces; ++c)
                *reinterpret_cast<uint4*>(stage + lane * (kPieces * 16) + ((c ^ lane) & (kPieces - 1)) * 16) =
                    make_uint4(pack_as<T>(number(8 * c), number(8 * c + 1)), pack_as<T>(number(8 * c + 2), number(8 * c + 3)), pack_as<T>(number(8 * c + 4), number(8 * c + 5)),
                               pack_as<T>(number(8 * c + 6), number(8 * c + 7)));
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int r = (32 / kPieces) * i + lane / kPieces, piece = lane % kPieces;
                const uint4 w = *reinterpret_cast<const uint4*>(stage + r * (kPieces * 16) + ((piece ^ r) & (kPieces - 1)) * 16);
                T* dst = target(kRowsTile * tile + lane0 + r);
                if (dst != nullptr) *reinterpret_cast<uint4*>(dst + 8 * piece) = w;
            }
        } else {
            // ---- the shares of a row's keys, in order: each CTA of the cluster joins a part of the rows, from where all of them left theirs ----
            constexpr int kFours = D / 4;             // 16-byte pieces of a row of sums
            asm volatile("bar.sync 2, %0;" ::"n"(32 * kRowWarps) : "memory");       // keys and values have been read: the sums lie over them
            float4* mine_at = reinterpret_cast<float4*>(s_k) + (size_t)tid * kFours;
#pragma unroll
            for (int c0 = 0; c0 < D; c0 += 32) {
                uint32_t o[32];
                if (n > 0) umma::ld32(o, to, lane0, c0);
                auto number = [&](int x) { return n > 0 ? __uint_as_float(o[x]) * by : 0.f; };
#pragma unroll
                for (int x = 0; x < 32; x += 4) mine_at[(c0 + x) / 4 ^ (lane & (kFours - 1))] = make_float4(number(x), number(x + 1), number(x + 2), number(x + 3));
            }
            s_ml[tid] = make_float2(m, ok ? l : NAN);
            __syncwarp();
            cluster_sync();
            // what each share counts, then four numbers of a row at a time, eight such in flight. Rows that are none are left out
            const int rank = split % p.ctas, group = split / p.ctas, groups = p.n_splits / p.ctas;
            const int in_first = min(p.tile_tokens, last_tok + 1 - tok0) * p.G, in_all = (last_tok + 1 - tok0) * p.G;
            const int from = in_all * rank / p.ctas, rows = in_all * (rank + 1) / p.ctas - from;
            auto row_of = [&](int i) { return from + i < in_first ? from + i : kRowsTile + from + i - in_first; };
            const uint32_t at0 = umma::smem_addr(s_k), ml0 = umma::smem_addr(s_ml);
            float* factor_of = reinterpret_cast<float*>(s_q);         // [row][share]
            const int unit = blockIdx.x + blockIdx.y * gridDim.x;
            float* partial = p.partials + (size_t)(unit * groups + group) * partial_floats(D, kTiles * kRowsTile);
            if (tid < rows) {
                float2 ml[kMaxCluster];
                float best = kNoRef, sum = 0.f;
#pragma unroll
                for (int k = 0; k < kMaxCluster; ++k) {
                    ml[k] = k < p.ctas ? peer_f32x2(ml0 + 8 * row_of(tid), k) : make_float2(kNoRef, 0.f);
                    best = fmaxf(best, ml[k].x);
                }
#pragma unroll
                for (int k = 0; k < kMaxCluster; ++k) {
                    ml[k].y *= ex2(ml[k].x - best);
                    sum += ml[k].y;
                }
                const float part = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
                for (int k = 0; k < kMaxCluster; ++k)
                    if (k < p.ctas) factor_of[tid * kMaxCluster + k] = ml[k].y * part;
                if (groups > 1) reinterpret_cast<float2*>(partial + kTiles * kRowsTile * D)[from + tid] = make_float2(best, sum);
            }
            asm volatile("bar.sync 2, %0;" ::"n"(32 * kRowWarps) : "memory");
            constexpr int kAtOnce = 8, kRowsOnce = 32 * kRowWarps / kFours;
            const int piece = tid % kFours;
            auto store = [&](int i, float4 v) {
                T* dst = target(row_of(i));
                if (dst != nullptr) *reinterpret_cast<uint2*>(dst + 4 * piece) = make_uint2(pack_as<T>(v.x, v.y), pack_as<T>(v.z, v.w));
            };
            for (int r0 = tid / kFours; r0 < rows; r0 += kAtOnce * kRowsOnce) {
                float4 v[kAtOnce];
#pragma unroll
                for (int x = 0; x < kAtOnce; ++x) v[x] = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int k = 0; k < p.ctas; ++k) {
                    float4 y[kAtOnce];
#pragma unroll
                    for (int x = 0; x < kAtOnce; ++x) {
                        const int r = row_of(r0 + x * kRowsOnce);
                        y[x] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (r0 + x * kRowsOnce < rows) y[x] = peer_f32x4(at0 + 16 * (r * kFours + (piece ^ (r & (kFours - 1)))), k);
                    }
#pragma unroll
                    for (int x = 0; x < kAtOnce; ++x) {
                        const float w = factor_of[min(r0 + x * kRowsOnce, rows - 1) * kMaxCluster + k];
                        v[x].x = fmaf(y[x].x, w, v[x].x), v[x].y = fmaf(y[x].y, w, v[x].y), v[x].z = fmaf(y[x].z, w, v[x].z), v[x].w = fmaf(y[x].w, w, v[x].w);
                    }
                }
#pragma unroll
                for (int x = 0; x < kAtOnce; ++x) {
                    const int i = r0 + x * kRowsOnce;
                    if (i >= rows) continue;
                    if (groups == 1) store(i, v[x]);
                    else reinterpret_cast<float4*>(partial)[(from + i) * kFours + piece] = v[x];
                }
            }
            if (groups > 1) {
                // the clusters' sums: of the CTAs that have the same rows, the last one to come adds them up, in order
                asm volatile("bar.sync 2, %0;" ::"n"(32 * kRowWarps) : "memory");
                if (tid == 0) {
                    unsigned* counter = p.counters + unit * kMaxCluster + rank;
                    s_last = arrive(counter) == (unsigned)groups - 1;
                    if (s_last) *counter = 0;
                }
                asm volatile("bar.sync 2, %0;" ::"n"(32 * kRowWarps) : "memory");
                const float* first = p.partials + (size_t)unit * groups * partial_floats(D, kTiles * kRowsTile);
                for (int i = s_last ? tid / kFours : rows; i < rows; i += kRowsOnce) {
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    float best = kNoRef, sum = 0.f;
                    for (int k = 0; k < groups; ++k) {
                        const float* there = first + (size_t)k * partial_floats(D, kTiles * kRowsTile);
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(there + kTiles * kRowsTile * D) + from + i);
                        const float4 y = __ldcg(reinterpret_cast<const float4*>(there) + (from + i) * kFours + piece);
                        const float now = fmaxf(best, ml.x), keep = ex2(best - now), w = ml.y * ex2(ml.x - now);
                        best = now;
                        sum = fmaf(sum, keep, w);
                        v.x = fmaf(v.x, keep, y.x * w), v.y = fmaf(v.y, keep, y.y * w), v.z = fmaf(v.z, keep, y.z * w), v.w = fmaf(v.w, keep, y.w * w);
                    }
                    const float part = sum == 0.f ? 0.f : 1.f / sum;
                    store(i, make_float4(v.x * part, v.y * part, v.z * part, v.w * part));
                }
            }
        }
    }
    if constexpr (kShared) {
        __syncwarp();
        if (warp >= kRowWarps) cluster_sync();
        cluster_sync();                                // nobody leaves while its sums are read
    }
    if (warp >= kRowWarps && !ok && lane == 0) atomicOr(p.status, kTimedOut);
    umma::fence_before_sync();
    __syncthreads();
    if (warp == kMmaWarp) {
        umma::fence_after_sync();
        umma::tmem_free_n(tmem, 512);
    }
}

template <typename T, int D>
int launch(PromptParams p, int blocks, int most_splits, cudaStream_t st) {
    static std::atomic<unsigned long long> ready{0};             // a bit for each device
    static int rooms[64][kMaxCluster + 1];                       // clusters of so many CTAs that a device holds at once
    int dev = 0;
    LEANKV_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return LEANKV_ELIMIT;
    if (((ready.load(std::memory_order_acquire) >> dev) & 1ull) == 0) {
        LEANKV_CUDA_TRY(cudaFuncSetAttribute(prompt_kernel<T, D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes(D)));
        LEANKV_CUDA_TRY(cudaFuncSetAttribute(prompt_kernel<T, D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes(D)));
        for (int i = 2; i <= kMaxCluster; ++i) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(1, 1, i);
            cfg.blockDim = dim3(kThreads);
            cfg.dynamicSmemBytes = smem_bytes(D);
            cudaLaunchAttribute attr;
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = attr.val.clusterDim.y = 1, attr.val.clusterDim.z = i;
            cfg.attrs = &attr, cfg.numAttrs = 1;
            LEANKV_CUDA_TRY(cudaOccupancyMaxActiveClusters(&rooms[dev][i], prompt_kernel<T, D, true>, &cfg));
        }
        ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    // as many CTAs share a block's keys as leave the launch in one wave: a cluster, or several of eight (8 tokens behind 8000, 8 kv heads: one 39 us, two 28;
    // clusters of 16 43)
    const long long units = (long long)p.H * p.B * blocks;
    p.ctas = 1;
    p.first_blocks = (int)std::min((long long)blocks, std::max(1ll, sm_count() / ((long long)p.H * p.B)));
    for (int i = 2; i <= std::min(kMaxCluster, most_splits); ++i)
        if (units <= rooms[dev][i]) p.ctas = i;
    const long long groups = p.ctas < kMaxCluster ? 1 : std::max(1ll, std::min((long long)rooms[dev][kMaxCluster] / units, (long long)most_splits / kMaxCluster));
    p.n_splits = (int)(p.ctas * groups);
    const dim3 grid((unsigned)(p.H * p.B), (unsigned)blocks, (unsigned)p.n_splits);
    if (p.ctas == 1) LEANKV_CUDA_TRY(launch_early(prompt_kernel<T, D, false>, grid, dim3(kThreads), smem_bytes(D), st, p));
    else LEANKV_CUDA_TRY(launch_cluster_kernel_ex(true, dim3(1, 1, p.ctas), prompt_kernel<T, D, true>, grid, dim3(kThreads), smem_bytes(D), st, p));
    return LEANKV_OK;
}

}  // namespace
}  // namespace bytes
}  // namespace leankv

using namespace leankv;

extern "C" int leankv_byte_prompt_attn(const leankv_byte_attn_t* a, void* stream) {
    if (const int rc = bytes::check_attn(a, bytes::kWorkspaceBytes)) return rc;
    if (a->block_pages != nullptr || !(a->scale > 0.f)) return LEANKV_EINVAL;
    if (a->dtype == LEANKV_BYTES_F32) return LEANKV_EUNSUPPORTED;
    bytes::PromptParams p = {};
    p.chunks = static_cast<const uint8_t*>(a->pool.chunks);
    p.n_pages = a->pool.n_pages, p.H = a->pool.kv_heads, p.B = a->batch, p.G = a->q_heads / a->pool.kv_heads, p.tokens = a->tokens;
    p.tile_tokens = bytes::kRowsTile / p.G;
    p.q = a->q, p.out = a->out;
    p.scale = a->scale * bytes::kLog2e;
    p.indptr = a->kv_indptr, p.indices = a->kv_page_indices, p.last = a->kv_last_page_len;
    p.status = static_cast<int*>(a->workspace);
    p.counters = reinterpret_cast<unsigned*>(p.status + bytes::kStatusWords);
    p.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + bytes::kPartialsAt);
    const long long blocks = ((long long)p.tokens + bytes::kTiles * p.tile_tokens - 1) / (bytes::kTiles * p.tile_tokens);
    if (blocks > 65535 || (long long)p.H * p.B > 0x7fffffffll) return LEANKV_ELIMIT;
    // CTAs that share the keys have four key tiles each at least
    const int most_splits = (int)(std::min(((long long)a->max_pages_seq + bytes::kPagesTile - 1) / bytes::kPagesTile / 4, 64ll));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->pool.dim == 128) return a->dtype == LEANKV_BYTES_F16 ? bytes::launch<__half, 128>(p, (int)blocks, most_splits, st) : bytes::launch<bf16, 128>(p, (int)blocks, most_splits, st);
    return a->dtype == LEANKV_BYTES_F16 ? bytes::launch<__half, 64>(p, (int)blocks, most_splits, st) : bytes::launch<bf16, 64>(p, (int)blocks, most_splits, st);
}
