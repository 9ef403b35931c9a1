// Writing tokens into the 8-bit pages, and the stored numbers back.
//
// A warp takes the keys or the values of one page and kv head: 16 rows of dim numbers in registers, one maximum over the warp, the exponent from its
// bits, one rounding a number. Bound: the rows come once from memory and a chunk goes out once (2 + 1 bytes a number in 16-bit types).
// A page that holds tokens already (at most the first one of a call, and the only one of a decode step) is read, rounded once more
// if its scale grew, and written whole.

#include <algorithm>
#include <type_traits>

#include "byte_layout.cuh"
#include "tile_softmax.cuh"

namespace leankv {
namespace bytes {
namespace {

constexpr int kWarps = 4;

struct AppendParams {
    uint8_t* chunks;
    uint8_t* bounds;
    int H, n_pages, B, T, tiles;                  // tiles: pages that a sequence's new tokens can touch
    leankv_vectors_t k, v;
    const int32_t* indptr;
    const int32_t* indices;
    const int32_t* last;
};

// The codes of a word times 2^-shift, each rounded half to even.
__device__ __forceinline__ uint32_t coarser(uint32_t w, float f) {
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = (int)((w >> (8 * i)) & 0xffu) - 128;
        out |= (uint32_t)(__float2int_rn((float)c * f) + 128) << (8 * i);
    }
    return out;
}

// CTAs an SM. Seven leave the 16-bit types 72 registers at head size 128, for which 32 bytes of a thread are spilled (16 x 2011 tokens, bf16: 5, the compiler's own choice, 43.7 us, 6
// 41.0, 7 40.3)
template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32, sizeof(T) == 4 ? 4 : D == 128 ? 7 : 9) append_kernel(const AppendParams p) {
    using R = Rows<D>;
    __shared__ __align__(16) uint32_t s_words[kWarps][R::kWords];
    pdl_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * kWarps + warp;
    const int tile = (int)(unit % p.tiles), which = (int)(unit / p.tiles % 2);
    const long long pair = unit / p.tiles / 2;
    if (pair >= (long long)p.B * p.H) return;
    const int b = (int)(pair / p.H), h = (int)(pair % p.H);
    const int ip = p.indptr[b], pages = p.indptr[b + 1] - ip;
    const int end = (pages - 1) * kPage + p.last[b], start = end - p.T;       // the new tokens are the sequence's last ones
    if (pages <= 0 || start < 0) return;
    const int page = start / kPage + tile, first = page * kPage;
    if (page >= pages) return;
    const int id = p.indices[ip + page];
    if (id < 0 || id >= p.n_pages) return;

    uint8_t* chunk = p.chunks + ((size_t)id * p.H + h) * chunk_bytes(D);
    uint8_t* codes = chunk + which * half_bytes(D);
    float* scale = reinterpret_cast<float*>(chunk + 2 * half_bytes(D)) + which;
    const int c = R::channel(lane);
    const leankv_vectors_t from = which == 0 ? p.k : p.v;
    const T* x = static_cast<const T*>(from.data) + b * from.seq + h * from.head + 8 * c;

    Eight<T> row[R::kSets][4];
#pragma unroll
    for (int i = 0; i < R::kSets; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int pos = first + R::token(R::set(lane, i), j);
            if (pos >= start && pos < end) row[i][j].load(x + (long long)(pos - start) * from.token);
            else row[i][j].zero();
        }
    const bool opened = first < start;            // tokens of earlier calls are in the page
    uint32_t w[R::kSets][4][2];
    uint32_t old_scale = 0;
    if (opened) {
        old_scale = *reinterpret_cast<const uint32_t*>(scale);
        if (which == 0) R::read_keys(codes, lane, w);
        else R::read_values(codes, s_words[warp], lane, w);
    }
    // magnitudes as bits: a NaN is larger than infinity, infinity than all others
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < R::kSets; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = row[i][j].largest(amax);
    amax = __reduce_max_sync(0xffffffffu, Eight<T>::bits(amax));
    const bool bad = amax >= kTooLarge || (opened && (old_scale & 0x7fffffffu) > 0x7f800000u);
    int e = least_exponent<127>(amax);
    const int e_old = opened ? max((int)(old_scale >> 23) - 127, -126) : -126;
    e = max(e, e_old);
    // x 2^-e is exact, and adding 1.5 * 2^23 + 128 rounds it to a whole number, half to even: the sum's low byte is the stored code. (A conversion
    // to whole numbers has an eighth of the rate: 16 x 2011 tokens 55 us so, on conversions.) Slots without a token hold zeros
    const float to_codes = power_of_two(-e);
#pragma unroll
    for (int i = 0; i < R::kSets; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool old = opened && first + R::token(R::set(lane, i), j) < start;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t c[4];
#pragma unroll
                for (int k = 0; k < 4; k += 2) {
                    const Two v = fma2({row[i][j].get(4 * half + k), row[i][j].get(4 * half + k + 1)}, {to_codes, to_codes}, {12583040.f, 12583040.f});
                    c[k] = __float_as_uint(v.x), c[k + 1] = __float_as_uint(v.y);
                }
                const uint32_t q = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
                if (!old) w[i][j][half] = q;
                else if (e != e_old) w[i][j][half] = coarser(w[i][j][half], power_of_two(max(e_old - e, -126)));
                if (bad) w[i][j][half] = kZeroCodes;
            }
        }
    const uint32_t scale_bits = bad ? kNaN : __float_as_uint(power_of_two(e));
    if (lane == 0) *reinterpret_cast<uint32_t*>(scale) = scale_bits;
    if (which == 1) {
        R::write_values(codes, s_words[warp], lane, w);
        return;
    }
    R::write_keys(codes, lane, w);
    // largest and smallest code of each channel among the tokens that are there; codes are compared as unsigned bytes
    uint32_t top[2] = {0u, 0u}, low[2] = {0xffffffffu, 0xffffffffu};
#pragma unroll
    for (int i = 0; i < R::kSets; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (first + R::token(R::set(lane, i), j) >= end) continue;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                top[half] = __vmaxu4(top[half], w[i][j][half]);
                low[half] = __vminu4(low[half], w[i][j][half]);
            }
        }
#pragma unroll
    for (int o = R::kLanes; o < 32; o *= 2)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            top[half] = __vmaxu4(top[half], __shfl_xor_sync(0xffffffffu, top[half], o));
            low[half] = __vminu4(low[half], __shfl_xor_sync(0xffffffffu, low[half], o));
        }
    uint8_t* bounds = p.bounds + ((size_t)id * p.H + h) * bounds_bytes(D);
    if (lane < R::kLanes) {
        *reinterpret_cast<uint2*>(bounds + 8 * c) = make_uint2(top[0] ^ kZeroCodes, top[1] ^ kZeroCodes);
        *reinterpret_cast<uint2*>(bounds + D + 8 * c) = make_uint2(low[0] ^ kZeroCodes, low[1] ^ kZeroCodes);
    }
    if (lane == 0) *reinterpret_cast<uint32_t*>(bounds + 2 * D) = scale_bits;
}

struct UnpackParams {
    const uint8_t* chunks;
    int H, n_pages, B, T, tiles;
    void* k;
    void* v;
    const int32_t* indptr;
    const int32_t* indices;
    const int32_t* last;
};

// Two numbers as the type holds them, none beyond its range (an fp16 block of magnitudes around 65504 has codes for 65536).
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 v = __floats2half2_rn(fabsf(a) > 65504.f ? copysignf(65504.f, a) : a, fabsf(b) > 65504.f ? copysignf(65504.f, b) : b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, bf16) { return pack_bf16(a, b); }

template <typename T>
__device__ __forceinline__ void store8(T* to, const float (&v)[8]) {
    if constexpr (std::is_same<T, float>::value) {
        // a whole 32-byte sector of a lane at once (as two halves: 16 x 2011 tokens 69 us, so 54)
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
    } else {
        *reinterpret_cast<uint4*>(to) = make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) unpack_kernel(const UnpackParams p) {
    using R = Rows<D>;
    __shared__ __align__(16) uint32_t s_words[kWarps][R::kWords];
    pdl_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * kWarps + warp;
    const int tile = (int)(unit % p.tiles), which = (int)(unit / p.tiles % 2);
    const long long pair = unit / p.tiles / 2;
    if (pair >= (long long)p.B * p.H) return;
    const int b = (int)(pair / p.H), h = (int)(pair % p.H);
    const int at = p.indptr[b] + tile, pages = p.indptr[b + 1] - p.indptr[b];
    const int here = tile < pages - 1 ? kPage : tile == pages - 1 ? p.last[b] : 0;       // tokens in this page
    int id = here > 0 ? p.indices[at] : -1;
    if (id >= p.n_pages) id = -1;
    uint32_t w[R::kSets][4][2];
    float scale = 0.f;
    if (id >= 0) {
        const uint8_t* chunk = p.chunks + ((size_t)id * p.H + h) * chunk_bytes(D);
        scale = reinterpret_cast<const float*>(chunk + 2 * half_bytes(D))[which];
        if (which == 0) R::read_keys(chunk, lane, w);
        else R::read_values(chunk + half_bytes(D), s_words[warp], lane, w);
    }
    T* out = static_cast<T*>(which == 0 ? p.k : p.v) + (size_t)pair * p.T * D + 8 * R::channel(lane);
#pragma unroll
    for (int i = 0; i < R::kSets; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int tok = R::token(R::set(lane, i), j), pos = tile * kPage + tok;
            if (pos >= p.T) continue;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = id >= 0 && tok < here ? (float)((int)((w[i][j][e >> 2] >> (8 * (e & 3))) & 0xffu) - 128) * scale : 0.f;
            store8(out + (size_t)pos * D, v);
        }
}

template <typename F>
int by_type(int dtype, int dim, F&& f) {
    if (dim == 128) return dtype == LEANKV_BYTES_F16 ? f(__half(), std::integral_constant<int, 128>())
                         : dtype == LEANKV_BYTES_BF16 ? f(bf16(), std::integral_constant<int, 128>()) : f(0.f, std::integral_constant<int, 128>());
    return dtype == LEANKV_BYTES_F16 ? f(__half(), std::integral_constant<int, 64>())
         : dtype == LEANKV_BYTES_BF16 ? f(bf16(), std::integral_constant<int, 64>()) : f(0.f, std::integral_constant<int, 64>());
}

// CTAs of kWarps units each, or 0 where a launch does not hold so many.
long long grid_of(int B, int H, int tiles) {
    const long long units = (long long)B * H * 2 * tiles, n = (units + kWarps - 1) / kWarps;
    return n <= 0x7fffffffll ? n : 0;
}

}  // namespace
}  // namespace bytes
}  // namespace leankv

using namespace leankv;

extern "C" size_t leankv_byte_chunk_bytes(int dim) { return dim == 64 || dim == 128 ? bytes::chunk_bytes(dim) : 0; }
extern "C" size_t leankv_byte_bounds_bytes(int dim) { return dim == 64 || dim == 128 ? bytes::bounds_bytes(dim) : 0; }

extern "C" int leankv_byte_append(const leankv_byte_append_t* a, void* stream) {
    if (!a || !bytes::good_pool(&a->pool) || !bytes::good_type(a->dtype) || !a->k.data || !a->v.data || a->batch <= 0 || a->tokens <= 0 ||
        !a->kv_indptr || !a->kv_page_indices || !a->kv_last_page_len)
        return LEANKV_EINVAL;
    if (a->batch > LEANKV_BYTES_MAX_BATCH) return LEANKV_ELIMIT;
    const leankv_byte_pool_t& pool = a->pool;
    if (!bytes::aligned_pool(&pool) || !bytes::aligned_vectors(&a->k, a->dtype, a->batch, pool.kv_heads, a->tokens) ||
        !bytes::aligned_vectors(&a->v, a->dtype, a->batch, pool.kv_heads, a->tokens))
        return LEANKV_EALIGN;
    bytes::AppendParams p = {};
    p.chunks = static_cast<uint8_t*>(pool.chunks);
    p.bounds = static_cast<uint8_t*>(pool.bounds);
    p.H = pool.kv_heads, p.n_pages = pool.n_pages, p.B = a->batch, p.T = a->tokens;
    p.tiles = (int)(((long long)a->tokens + 2 * bytes::kPage - 2) / bytes::kPage);
    p.k = a->k, p.v = a->v;
    p.indptr = a->kv_indptr, p.indices = a->kv_page_indices, p.last = a->kv_last_page_len;
    const long long grid = bytes::grid_of(p.B, p.H, p.tiles);
    if (grid == 0) return LEANKV_ELIMIT;
    return bytes::by_type(a->dtype, pool.dim, [&](auto t, auto d) -> int {
        LEANKV_CUDA_TRY(launch_early(bytes::append_kernel<decltype(t), decltype(d)::value>, dim3((unsigned)grid), dim3(bytes::kWarps * 32), 0,
                                     static_cast<cudaStream_t>(stream), p));
        return LEANKV_OK;
    });
}

extern "C" int leankv_byte_unpack(const leankv_byte_pool_t* pool, int dtype, void* k_out, void* v_out, int B, int T, const int32_t* kv_indptr,
                                  const int32_t* kv_page_indices, const int32_t* kv_last_page_len, void* stream) {
    if (!bytes::good_pool(pool) || !bytes::good_type(dtype) || !k_out || !v_out || B <= 0 || T <= 0 || !kv_indptr || !kv_page_indices || !kv_last_page_len)
        return LEANKV_EINVAL;
    if (B > LEANKV_BYTES_MAX_BATCH) return LEANKV_ELIMIT;
    const uintptr_t loose = dtype == LEANKV_BYTES_F32 ? 31u : 15u;
    if (!bytes::aligned_pool(pool) || ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & loose) != 0) return LEANKV_EALIGN;
    bytes::UnpackParams p = {};
    p.chunks = static_cast<const uint8_t*>(pool->chunks);
    p.H = pool->kv_heads, p.n_pages = pool->n_pages, p.B = B, p.T = T;
    p.tiles = (int)(((long long)T + bytes::kPage - 1) / bytes::kPage);
    p.k = k_out, p.v = v_out;
    p.indptr = kv_indptr, p.indices = kv_page_indices, p.last = kv_last_page_len;
    const long long grid = bytes::grid_of(B, p.H, p.tiles);
    if (grid == 0) return LEANKV_ELIMIT;
    return bytes::by_type(dtype, pool->dim, [&](auto t, auto d) -> int {
        LEANKV_CUDA_TRY(launch_early(bytes::unpack_kernel<decltype(t), decltype(d)::value>, dim3((unsigned)grid), dim3(bytes::kWarps * 32), 0,
                                     static_cast<cudaStream_t>(stream), p));
        return LEANKV_OK;
    });
}
