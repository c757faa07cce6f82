// paged_q4.cuh -- the 4-bit paged cache: how a block is laid out and how a group of 32 elements is quantised.
//
// A block ((page, layer, K or V, head): 64 tokens) holds the codes of all tokens, D / 2 bytes each, then their scales, one
// F16 per token and group of 32. Element e of a token has the value scale[e / 32] * (code[e] - 8). Eight elements 8 w ..
// 8 w + 7 are one 32-bit word, element e at bits 4 (e % 8); word w stands at place (w % 4) * (D / 32) + w / 4 of its token:
// lane t of four, which takes the words 4 G + t of every group G in a tensor-core fragment, then finds them side by side.
//
// The group's element of the largest magnitude, m (a negative one before a positive one), gets code 0: the scale is -m / 8,
// kept within +- 2720, rounded to BF16 and then to F16. With its 8 significant bits scale * (code - 8) and 24 * scale are
// exact in F16, so that the attention's products read the cache without a further rounding. The codes are
// floor(x * (1 / scale) + 8.5) in f32, every operation rounded, kept within 0 .. 15. A group with a NaN or an infinity has the
// scale NaN.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace gsvcu {
namespace {

template <int D>
struct Q4Block {
    static constexpr int ROW = D / 2, SCALES = D / 16;   // bytes of a token's codes and scales
    static constexpr int OFF_SCALES = PAGE * ROW;
    static constexpr int BYTES = PAGE * (ROW + SCALES);
};
// Byte of word w (elements 8 w ..) in its token's codes.
template <int D>
__device__ __forceinline__ int q4_place(int w) { return ((w & 3) * (D / 32) + (w >> 2)) * 4; }

// Order of elements by magnitude, a negative one before a positive one of the same.
__device__ __forceinline__ uint32_t q4_key(float x) {
    const uint32_t u = __float_as_uint(x);
    return (u << 1) | (u >> 31);
}
// Scale of a group whose largest key is `key`, and the factor of its codes.
__device__ __forceinline__ __half q4_scale(uint32_t key, float& inv) {
    const float m = __uint_as_float(key >> 1);
    float t = fminf(m * 0.125f, 2720.0f);
    if (!(key & 1u)) t = -t;
    if ((key >> 1) >= 0x7f800000u) t = __uint_as_float(0x7fffffffu);
    const __half d = __float2half_rn(__bfloat162float(__float2bfloat16_rn(t)));
    const float f = __half2float(d);
    inv = f != 0.0f ? __fdiv_rn(1.0f, f) : 0.0f;
    return d;
}
// Codes of 8 elements as a word. A number of 0 .. 15 added to 2^23, rounded down, ends in its floor; what the 2^23 leave in the
// word is taken off at the end. (The conversion instruction has a quarter of the rate.)
__device__ __forceinline__ uint32_t q4_word(const float* x, float inv) {
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float y = fminf(fmaxf(__fadd_rn(__fmul_rn(x[i], inv), 8.5f), 0.0f), 15.0f);   // (a NaN: 0)
        word += __float_as_uint(__fadd_rd(y, 8388608.0f)) << (4 * i);
    }
    return word - 0xfb000000u;   // 0x4b000000 (1 + 16 + ...), cut to 32 bits
}

// BF16 query rows whose largest element is below 1/4 enter F16 products times a power of two, which the factor of their scores
// is divided by: the largest comes to 2^14 .. 2^15, so that elements keep their 8 bits down to 2^-31 of it. As they are they
// would lose them below 2^-17 and vanish below 2^-25 (2^-23 of the largest in the rows that are left so, the rule).
// `row`: 8 elements of a row that this lane and its PIECES - 1 neighbours have; all lanes of the warp take part. False: none of
// the warp's rows is scaled; else `up` is this row's exponent, 0 .. 126.
template <int PIECES>
__device__ __forceinline__ bool small_queries(uint4 row, int& up) {
    constexpr uint32_t QUARTER = 0x3e80u;
    auto larger = [](uint32_t x, uint32_t y) {   // of each half
        uint32_t z;
        asm("max.u16x2 %0, %1, %2;" : "=r"(z) : "r"(x & 0x7fff7fffu), "r"(y & 0x7fff7fffu));
        return z;
    };
    const uint32_t two = larger(larger(row.x, row.y), larger(row.z, row.w));
    uint32_t m = max(two & 0xffffu, two >> 16);
    if (!__any_sync(0xffffffffu, m > 0 && m < QUARTER)) return false;
#pragma unroll
    for (int o = 1; o < PIECES; o *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    up = m == 0 || m >= QUARTER ? 0 : min(126, 141 - (int)(m >> 7));   // (bits from 7 on: the exponent, 127 for 2^0)
    return true;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }   // -126 .. 127

__device__ __forceinline__ uint32_t bits(__half2 h) { return *(const uint32_t*)&h; }
__device__ __forceinline__ __half2 half2_of(uint32_t u) { return *(const __half2*)&u; }
// (x & mask) | bits
template <uint32_t MASK, uint32_t BITS>
__device__ __forceinline__ uint32_t field(uint32_t x) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(y) : "r"(x), "n"(MASK), "n"(BITS));
    return y;
}
// scale * (code - 8) of the four codes in each half of x: v[i] = code i of the low half with d's low half, and of the high
// half (of a whole word: elements i and i + 4). A code moved to bits 6 .. 9 under the exponent of 16 is 16 + code, times d
// less 24 d.
__device__ __forceinline__ void q4_values(uint32_t x, __half2 d, __half2 m24d, uint32_t (&v)[4]) {
    v[0] = bits(__hfma2(half2_of(field<0x03c003c0u, 0x4c004c00u>(x << 6)), d, m24d));
    v[1] = bits(__hfma2(half2_of(field<0x03c003c0u, 0x4c004c00u>(x << 2)), d, m24d));
    v[2] = bits(__hfma2(half2_of(field<0x03c003c0u, 0x4c004c00u>(x >> 2)), d, m24d));
    v[3] = bits(__hfma2(half2_of(field<0x03c003c0u, 0x4c004c00u>(x >> 6)), d, m24d));
}

}  // namespace
}  // namespace gsvcu
