// cache.cuh -- the paged 8-bit key/value cache, as its kernels see it.
//
// A page holds 64 tokens of every key/value head: 64 x 64 codes per head
// (token-major, 4096 contiguous bytes) in e4m3, and one scale per head in
// e8m0 (code u means 2^(u - 127), 255 means NaN).  A stream's token i lies in
// slot i % 64 of page table[stream][i / 64].
//
// Scales are powers of two: dividing by one and moving codes from one scale
// to a larger one only changes exponents (subnormal codes aside), and a code
// times its scale is exact in bf16 as well as in fp32.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace ress {
namespace cache {

constexpr int PAGE = 64;
constexpr int BLOCK_BYTES = PAGE * HD;  // one head's codes in a page

// The pages of K or V: bytes, strides in bytes.
struct Pages {
    uint8_t *codes;
    uint8_t *scale;
    long long page_stride, head_stride;  // of codes
    long long scale_stride;              // of a page's scales; heads are contiguous
};

// The host-side checks of a cache that its calls share.
inline int check_cache(const ress_cache *c) {
    if (!c || !c->k_pages || !c->v_pages || !c->k_scale || !c->v_scale || !c->table || !c->lens) return RESS_E_ARG;
    if (c->n_pages <= 0 || c->heads <= 0 || c->streams <= 0 || c->table_width <= 0 || c->table_stride < 0)
        return RESS_E_ARG;
    if (((uintptr_t)c->k_pages | (uintptr_t)c->v_pages | (uintptr_t)c->page_stride | (uintptr_t)c->head_stride) & 15)
        return RESS_E_ARG;
    if (c->head_stride < BLOCK_BYTES || c->page_stride < BLOCK_BYTES || c->scale_stride < c->heads) return RESS_E_ARG;
    if (c->n_pages > (1 << 30) || c->heads > 65535 || c->streams > 65535 || c->table_width > (1 << 24))
        return RESS_E_SHAPE;
    return RESS_OK;
}

__device__ __forceinline__ float scale_value(int u) {
    return __uint_as_float(u == 255 ? 0x7FC00000u : (u == 0 ? 0x00400000u : (uint32_t)u << 23));
}
// 2^(127 - u) of a page's code, which append makes 247 at most; 0 for the NaN
// code, so that its page holds zeros
__device__ __forceinline__ float scale_inverse(int u) { return __uint_as_float(u == 255 ? 0u : (uint32_t)(254 - u) << 23); }

// The code of the smallest power of two that brings |x| <= amax to 448 or
// less, from the bits of amax (sign bit clear): 448 = 1.75 * 2^8, so the
// exponent field less 8, one more where the significand is above 1.75.
__device__ __forceinline__ int scale_code(uint32_t amax_bits) {
    if (amax_bits >= 0x7F800000u) return 255;  // infinity or NaN
    const int u = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return max(u, 0);
}

// Four values as e4m3 codes, rounded to nearest even.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}
// The top bits of the bytes of w that are NaN codes (0x7F, 0xFF).
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }
// Two codes as halves, exactly (e4m3 lies inside fp16).
__device__ __forceinline__ uint32_t e4m3_to_half2(uint16_t codes) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(codes));
    return r;
}

}  // namespace cache
}  // namespace ress
