// The 8-bit pages: where a code lies, and what the kernels that write and read them share.
//
// A chunk (one page, one kv head) is  keys | values | key scale, value scale, 8 bytes of padding.  Codes are stored as
// code + 128, so that a byte below the fp16 number 1024's high byte (0x64) is the number 1152 + code.
//   keys    [dim / 64][16 tokens][64 channels]: lane (g, t) of a warp reads channels 16 t .. 16 t + 15 of each 64 of tokens g and g + 8 with 16-byte
//           loads, rows 64 bytes apart: no bank is met twice. That is the A operand of mma.m16n8k16 with the channels of a step
//           taken as 4 s + {0, 1} and 4 s + {2, 3} of a lane's sixteen (any order of the channels will do, the query's is the same).
//   values  words of four tokens of a channel in the A operand's order: word i' of lane (g, t) in 512-byte part j holds channel
//           8 (4 j + i') + g, tokens 2t, 2t + 1, 2t + 8, 2t + 9.
// Both are read straight into registers; nothing is transposed or shuffled on the way to the tensor cores.
#pragma once

#include <type_traits>

#include "leankv_bytes.h"
#include "typed.cuh"

namespace leankv {
namespace bytes {

constexpr int kPage = 16;
constexpr uint32_t kZeroCodes = 0x80808080u;
constexpr uint32_t kNaN = 0x7fc00000u;
constexpr uint32_t kTooLarge = 0x7e800000u;          // 2^126

__host__ __device__ constexpr uint32_t half_bytes(int dim) { return kPage * dim; }            // keys or values of a chunk
__host__ __device__ constexpr uint32_t chunk_bytes(int dim) { return 2 * half_bytes(dim) + 16; }
__host__ __device__ constexpr uint32_t bounds_bytes(int dim) { return 2 * dim + 16; }

inline bool good_pool(const leankv_byte_pool_t* p) {
    return p && (p->dim == 64 || p->dim == 128) && p->kv_heads > 0 && p->n_pages > 0 && p->chunks && p->bounds;
}
inline bool aligned_pool(const leankv_byte_pool_t* p) { return aligned16(p->chunks) && aligned16(p->bounds); }
inline int type_size(int dtype) { return dtype == LEANKV_BYTES_F32 ? 4 : 2; }
inline bool good_type(int dtype) { return dtype >= LEANKV_BYTES_F16 && dtype <= LEANKV_BYTES_F32; }
// Strides that are used are whole 16-byte pieces.
inline bool aligned_vectors(const leankv_vectors_t* x, int dtype, int seqs, int heads, int tokens) {
    const long long piece = 16 / type_size(dtype);
    return aligned16(x->data) && (seqs <= 1 || x->seq % piece == 0) && (heads <= 1 || x->head % piece == 0) && (tokens <= 1 || x->token % piece == 0);
}

// What both attention entries ask of their arguments.
inline int check_attn(const leankv_byte_attn_t* a, size_t workspace_bytes) {
    if (!a || !good_pool(&a->pool) || !good_type(a->dtype) || !a->q.data || !a->out.data || a->batch <= 0 || a->tokens <= 0 || a->q_heads <= 0 ||
        a->q_heads % a->pool.kv_heads != 0 || !a->kv_indptr || !a->kv_page_indices || !a->kv_last_page_len || a->max_pages_seq < 0 || a->total_pages < 0 ||
        (a->block_pages != nullptr && (a->tokens != 1 || a->n_blocks <= 0)))
        return LEANKV_EINVAL;
    if (a->batch > LEANKV_BYTES_MAX_BATCH || a->q_heads / a->pool.kv_heads > LEANKV_BYTES_MAX_GROUP) return LEANKV_ELIMIT;
    if (!aligned_pool(&a->pool) || !aligned_vectors(&a->q, a->dtype, a->batch, a->q_heads, a->tokens) ||
        !aligned_vectors(&a->out, a->dtype, a->batch, a->q_heads, a->tokens) || !aligned16(a->workspace))
        return LEANKV_EALIGN;
    return a->workspace && a->workspace_bytes >= workspace_bytes ? LEANKV_OK : LEANKV_EWORKSPACE;
}

// The smallest e >= -126 with amax <= 127 * 2^e (most = 127) or 2047 * 2^e (most = 2047); amax as its bits, finite.
template <int kMost>
__device__ __forceinline__ int least_exponent(uint32_t amax_bits) {
    static_assert(kMost == 127 || kMost == 2047, "one less than a power of two");
    constexpr int kBits = kMost == 127 ? 7 : 11;
    // most = (2 - 2^(1 - bits)) * 2^(bits - 1): the border lies where the mantissa is all ones in its first bits - 1 places
    constexpr uint32_t kBorder = (0x7fffffu >> (24 - kBits)) << (24 - kBits);
    const int e = (int)(amax_bits >> 23) - 127 - (kBits - 1) + ((amax_bits & 0x7fffffu) > kBorder ? 1 : 0);
    return max(e, -126);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // -126 .. 127

// Four rows of four bytes, transposed.
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
    const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[0], w[1], 0x7362);
    const uint32_t c = __byte_perm(w[2], w[3], 0x5140), d = __byte_perm(w[2], w[3], 0x7362);
    w[0] = __byte_perm(a, c, 0x5410);
    w[1] = __byte_perm(a, c, 0x7632);
    w[2] = __byte_perm(b, d, 0x5410);
    w[3] = __byte_perm(b, d, 0x7632);
}

// How a warp shares a page's rows when it writes or unpacks them: a lane has channels 8 c .. 8 c + 7 of the tokens 2t, 2t + 1, 2t + 8, 2t + 9 for
// kSets values of t (four tokens are a word of the values' order).
template <int D>
struct Rows {
    static constexpr int kLanes = D / 8;                 // of a row
    static constexpr int kSets = D / 64;
    // values go through shared memory in words; parts of 128 words are padded so that lanes meet no bank twice
    static constexpr int kPad = D == 128 ? 8 : 16;
    static constexpr int kParts = D / 32;
    static constexpr int kWords = kParts * (128 + kPad);

    __device__ static int channel(int lane) { return lane % kLanes; }                               // c
    __device__ static int set(int lane, int i) { return lane / kLanes + i * (32 / kLanes); }        // t
    __device__ static int token(int t, int j) { return 2 * t + (j & 1) + 8 * (j >> 1); }            // of four
    __device__ static uint32_t key_offset(int tok, int c) { return (uint32_t)(c >> 3) * 1024u + (uint32_t)tok * 64u + (uint32_t)(c & 7) * 8u; }
    __device__ static int value_word(int c, int g, int t) { return (c >> 2) * (128 + kPad) + (g * 4 + t) * 4 + (c & 3); }

    // The values of a chunk as words in the lane's own order: w[i][j][half]: token j of set i, channels 8 c + 4 half .. + 3.
    __device__ static void read_values(const uint8_t* values, uint32_t* s, int lane, uint32_t (&w)[kSets][4][2]) {
#pragma unroll
        for (int j = 0; j < kParts; ++j)
            *reinterpret_cast<uint4*>(s + j * (128 + kPad) + lane * 4) = reinterpret_cast<const uint4*>(values)[j * 32 + lane];
        __syncwarp();
        const int c = channel(lane);
#pragma unroll
        for (int i = 0; i < kSets; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = s[value_word(c, 4 * half + e, set(lane, i))];
                transpose4(x);
#pragma unroll
                for (int j = 0; j < 4; ++j) w[i][j][half] = x[j];
            }
        __syncwarp();
    }
    __device__ static void write_values(uint8_t* values, uint32_t* s, int lane, const uint32_t (&w)[kSets][4][2]) {
        const int c = channel(lane);
#pragma unroll
        for (int i = 0; i < kSets; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t x[4] = {w[i][0][half], w[i][1][half], w[i][2][half], w[i][3][half]};
                transpose4(x);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[value_word(c, 4 * half + e, set(lane, i))] = x[e];
            }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < kParts; ++j)
            reinterpret_cast<uint4*>(values)[j * 32 + lane] = *reinterpret_cast<const uint4*>(s + j * (128 + kPad) + lane * 4);
    }
    __device__ static void read_keys(const uint8_t* keys, int lane, uint32_t (&w)[kSets][4][2]) {
#pragma unroll
        for (int i = 0; i < kSets; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint2 x = *reinterpret_cast<const uint2*>(keys + key_offset(token(set(lane, i), j), channel(lane)));
                w[i][j][0] = x.x;
                w[i][j][1] = x.y;
            }
    }
    __device__ static void write_keys(uint8_t* keys, int lane, const uint32_t (&w)[kSets][4][2]) {
#pragma unroll
        for (int i = 0; i < kSets; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<uint2*>(keys + key_offset(token(set(lane, i), j), channel(lane))) = make_uint2(w[i][j][0], w[i][j][1]);
    }
};

// Eight numbers as they lie in memory.
template <typename T> struct Eight {
    uint4 a;
    __device__ void load(const T* p) { a = __ldg(reinterpret_cast<const uint4*>(p)); }
    __device__ void zero() { a = make_uint4(0, 0, 0, 0); }
    // the largest magnitude so far, two numbers' bits side by side; `bits` makes it the bits of one fp32 number
    __device__ uint32_t largest(uint32_t m) const {
        m = __vmaxu2(m, a.x & 0x7fff7fffu);
        m = __vmaxu2(m, a.y & 0x7fff7fffu);
        m = __vmaxu2(m, a.z & 0x7fff7fffu);
        return __vmaxu2(m, a.w & 0x7fff7fffu);
    }
    __device__ static uint32_t bits(uint32_t m) {
        const uint32_t one = max(m & 0xffffu, m >> 16);
        if constexpr (std::is_same<T, bf16>::value) return one << 16;
        else return __float_as_uint(__half2float(__ushort_as_half((unsigned short)one)));
    }
    __device__ float get(int i) const {
        const uint32_t w = i < 2 ? a.x : i < 4 ? a.y : i < 6 ? a.z : a.w;
        if constexpr (sizeof(T) == 2 && std::is_same<T, bf16>::value) return __uint_as_float((i & 1) ? w & 0xffff0000u : w << 16);
        else return (i & 1) ? __high2float(*reinterpret_cast<const __half2*>(&w)) : __low2float(*reinterpret_cast<const __half2*>(&w));
    }
};
template <> struct Eight<float> {
    float4 a, b;
    __device__ void load(const float* p) {
        a = __ldg(reinterpret_cast<const float4*>(p));
        b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    }
    __device__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ uint32_t largest(uint32_t m) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(get(i)) & 0x7fffffffu);
        return m;
    }
    __device__ static uint32_t bits(uint32_t m) { return m; }
    __device__ float get(int i) const {
        const float4& v = i < 4 ? a : b;
        return (i & 3) == 0 ? v.x : (i & 3) == 1 ? v.y : (i & 3) == 2 ? v.z : v.w;
    }
};

// Two numbers in a 16-bit type.
template <typename T>
__device__ __forceinline__ uint32_t pack_as(float a, float b) {
    if constexpr (std::is_same<T, bf16>::value) {
        return pack_bf16(a, b);
    } else {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

}  // namespace bytes
}  // namespace leankv
