// ============================================================================
//  kv4.h -- the 4-bit paged cache.
//
//  A page of a layer holds, for each KV head, one block of 640 ng bytes, ng =
//  ceil(head_dim / 32) groups of 32 channels (the last may be half there):
//    K codes  uint32 [j 4][token 16][ng]   channels 32 g + 8 j + 2 n + h at bit 16 h + 4 n
//    V codes  uint32 [j 4][c 16][ng]       channels 32 g + 16 T + c of the tokens
//                                          4 j + 2 m + h at bit 16 h + 8 T + 4 m
//    K        fp16 [token 16][ng][scale, base]
//    V        fp16 [j 4][ng][scale, base][token 4 j ..]
//  so that lane 16 j + r of a wave finds its operands of the 16x16x32 matrix
//  instructions (row r, eight consecutive k from 8 j) in its own words: K of a page
//  with k over channels, V of two pages with k over tokens.  Two pages of 128
//  channels are four 16-byte loads a lane.
//
//  A code c stands for the fp16 number nearest to scale (16 + c) + base: 16 + c is
//  the bits 0x4C00 | c << 6, so a pair of values is a shift, an and-or and one
//  packed multiply-add, and a product over them is exact in the matrix unit.
//    scale = fp16((hi - lo) / 15), base = fp16(lo - 16 scale) over a group's 32
//  channels of one token, c = the nearest code, each step of it in fp32 as written.
//  Magnitudes past 2^14 are held as 2^14 (16 scale stays in fp16); a group that
//  holds a NaN or an infinity reads NaN; a group of one value is its base.
// ============================================================================
#pragma once
#include "internal.h"

namespace opure_kv4 {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

constexpr uint32_t GROUP = 32;                        // channels with one scale
constexpr uint32_t BLOCK = 640;                       // bytes a group of a page and KV head
constexpr float MOST = 16384.0f;                      // largest magnitude held

__host__ __device__ constexpr uint32_t groups(uint32_t hd) { return (hd + GROUP - 1u) / GROUP; }

// byte offsets in a block of ng groups
__host__ __device__ constexpr uint32_t v_codes(uint32_t ng) { return 256u * ng; }
__host__ __device__ constexpr uint32_t k_scales(uint32_t ng) { return 512u * ng; }
__host__ __device__ constexpr uint32_t v_scales(uint32_t ng) { return 576u * ng; }

__device__ __forceinline__ uint64_t block_at(uint32_t layer, uint32_t n_pages, uint32_t page, uint32_t n_kv, uint32_t head, uint32_t ng)
{
    return ((static_cast<uint64_t>(layer) * n_pages + page) * n_kv + head) * (BLOCK * ng);
}

__device__ __forceinline__ uint32_t half_bits(_Float16 v) { return __builtin_bit_cast(uint16_t, v); }

// A number that is rounded to fp32 before it is rounded to fp16: the compiler would
// make one instruction of a product and its conversion, which rounds once.
__device__ __forceinline__ _Float16 round_half(float v)
{
    asm volatile("" : "+v"(v));
    return static_cast<_Float16>(v);
}

// A group's scale and base from its smallest and largest value.
struct Scale {
    _Float16 s, b;
    bool bad;
    __device__ __forceinline__ Scale(float lo, float hi, bool nonfinite) : bad(nonfinite)
    {
        s = round_half(__fmul_rn(__fsub_rn(hi, lo), static_cast<float>(1.0 / 15.0)));
        b = round_half(__fsub_rn(lo, __fmul_rn(16.0f, static_cast<float>(s))));
    }
    // The group's values to their codes: rint((x - base) / scale - 16).  Where the quotient is 15.5 to 31.5 (past it both
    // ways clamp) a product with the scale's reciprocal is off from it by the two roundings, 2^-24 of it each, and those
    // of the two differences, 2^-20 each: under 2^-17 in all.  So it decides but for what lies nearer than 2^-16 to the
    // middle of two codes; there the quotient does (2,874 rows of 16 heads of 64: 12.4 us with quotients alone).
    template <int N>
    __device__ __forceinline__ void codes(float (&x)[N]) const
    {
        const float sf = static_cast<float>(s), bf = static_cast<float>(b), inv = __fdiv_rn(1.0f, sf);
        float c[N];
        bool near = false;
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            const float f = __fmaf_rn(__fsub_rn(x[i], bf), inv, -16.0f);
            c[i] = __builtin_rintf(f);
            near = near || __builtin_fabsf(__fsub_rn(f, c[i])) > 0.5f - 0x1p-16f;
        }
        if (__any(near))
#pragma unroll
            for (int i = 0; i < N; ++i) c[i] = __builtin_rintf(__fsub_rn(__fdiv_rn(__fsub_rn(x[i], bf), sf), 16.0f));
        const bool none = bad || s == static_cast<_Float16>(0);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = none ? 0.0f : fminf(fmaxf(c[i], 0.0f), 15.0f);
    }
    __device__ __forceinline__ uint32_t scale_bits() const { return bad ? 0x7E00u : half_bits(s); }
    __device__ __forceinline__ uint32_t base_bits() const { return bad ? 0x7E00u : half_bits(b); }
};

__device__ __forceinline__ half2_t pair(uint32_t w) { return __builtin_bit_cast(half2_t, w); }

// A mask and an exponent that the compiler does not know, a scalar and a vector
// register: with them a nibble is a shift and one and-or, with constants, of which an
// instruction has room for one, a shift, an and and an or.
struct Bits {
    uint32_t nibble = 0x03C003C0u, sixteen = 0x4C004C00u;
    __device__ __forceinline__ Bits()
    {
        asm volatile("" : "+s"(nibble));
        asm volatile("" : "+v"(sixteen));
    }
    // nibble N of both halves of a word as 16 + c
    template <int N>
    __device__ __forceinline__ half2_t codes(uint32_t w) const
    {
        const uint32_t at = N == 0 ? w << 6 : N == 1 ? w << 2 : N == 2 ? w >> 2 : w >> 6;
        return pair((at & nibble) | sixteen);
    }
};

__device__ __forceinline__ uint32_t values(half2_t c, half2_t s, half2_t b)
{
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(c, s, b));
}

// one value: channel d of K, or of V, of token u of a block
__device__ __forceinline__ float k_value(const uint8_t* block, uint32_t ng, uint32_t u, uint32_t d)
{
    const uint32_t w = reinterpret_cast<const uint32_t*>(block)[((d / 8u % 4u) * 16u + u) * ng + d / 32u];
    const uint32_t c = w >> (16u * (d & 1u) + 4u * (d / 2u % 4u)) & 15u;
    const _Float16* sb = reinterpret_cast<const _Float16*>(block + k_scales(ng)) + (u * ng + d / 32u) * 2u;
    return static_cast<float>(__builtin_fmaf16(static_cast<_Float16>(16u + c), sb[0], sb[1]));
}
__device__ __forceinline__ float v_value(const uint8_t* block, uint32_t ng, uint32_t u, uint32_t d)
{
    const uint32_t w = reinterpret_cast<const uint32_t*>(block + v_codes(ng))[((u / 4u) * 16u + d % 16u) * ng + d / 32u];
    const uint32_t c = w >> (16u * (u & 1u) + 8u * (d / 16u % 2u) + 4u * (u / 2u % 2u)) & 15u;
    const _Float16* sb = reinterpret_cast<const _Float16*>(block + v_scales(ng)) + ((u / 4u) * ng + d / 32u) * 8u + u % 4u;
    return static_cast<float>(__builtin_fmaf16(static_cast<_Float16>(16u + c), sb[0], sb[4]));
}

}  // namespace opure_kv4
