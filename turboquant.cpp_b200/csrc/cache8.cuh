// What the kernels of the 8-bit cache share: where a row lies, its blocks' bytes, conversions of e4m3 codes.
//
// A cached element is an e4m3 code times 2^(b - 127).  The byte b belongs to 16 consecutive rows of one (page, plane, key/value head): a
// power of two, so that a block whose byte grows moves its codes' exponents (only what falls below e4m3's normal range loses bits a
// second time), and so that the kernels scale exactly wherever it is cheapest.
//   codes   [n_pages][2: keys, values][kv heads][page_size][head size] e4m3
//   scales  [n_pages][2][kv heads][page_size / 16] bytes
//   weights [n_pages][kv heads][page_size] float32 (caches that add up attention weights)
// Row t of sequence s lies at place held[s] + t - cu_seqlens[s]; place p in page table[s][p / page_size], row p % page_size.
#pragma once
#include <cuda_fp8.h>
#include <string.h>
#include "common.cuh"

#define C8_BLOCK 16
#define C8_MAX_HEAD_DIM 256
#define C8_NAN 0x7fu              // the code of what is not finite

// A cache as the kernels take it.
struct Cache8 {
    uint8_t* codes;
    uint8_t* scales;
    const int* table;
    int table_stride, page_size, n_pages, nkv, hd;
    int page_shift;                    // page_size = 2^page_shift, or -1 (a division a place was much of what the small kernels did)
    __device__ __forceinline__ int column(int place) const { return page_shift >= 0 ? place >> page_shift : place / page_size; }
    __device__ __forceinline__ int row(int place) const { return page_shift >= 0 ? place & (page_size - 1) : place % page_size; }
    __device__ __forceinline__ int page_of(int seq, int place) const {
        return TQ_CHECKED(table[(size_t)seq * table_stride + TQ_CHECKED(column(place), table_stride, TQ_IDX_TABLE_COLUMN)], n_pages, TQ_IDX_PAGE);
    }
    // first code of a (page, plane, head); offsets pass 32 bits in a large cache
    __device__ __forceinline__ size_t codes_at(int page, int plane, int g) const {
        return (((size_t)page * 2 + plane) * nkv + g) * (size_t)page_size * hd;
    }
    __device__ __forceinline__ size_t scales_at(int page, int plane, int g) const {
        return (((size_t)page * 2 + plane) * nkv + g) * (size_t)(page_size / C8_BLOCK);
    }
};

// 2^(b - 127), b from 1 to 254
__device__ __forceinline__ float c8_scale(uint32_t b) { return __uint_as_float(b << 23); }
// 2^(127 - b), b from 1 to 253 (the writer's largest byte is 247)
__device__ __forceinline__ float c8_inverse(uint32_t b) { return __uint_as_float((254u - b) << 23); }
// The byte of a block whose largest finite magnitude has these bits: the smallest b >= 1 with top <= 448 * 2^(b - 127); 448 = 1.75 * 2^8.
__device__ __forceinline__ uint32_t c8_byte(uint32_t top_bits) {
    const int b = (int)(top_bits >> 23) - 8 + ((top_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t)max(b, 1);
}
// The bits of |x| where x is finite, else 0.
__device__ __forceinline__ uint32_t c8_magnitude(float x) {
    const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}
// Two codes (lo in the low byte), rounded to nearest even; what is not finite becomes NaN (the conversion alone would make infinity 448).
__device__ __forceinline__ uint32_t c8_encode2(float lo, float hi) {
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
    uint32_t r = d;
    if (!(fabsf(lo) < INFINITY)) r = (r & 0xff00u) | C8_NAN;
    if (!(fabsf(hi) < INFINITY)) r = (r & 0x00ffu) | (C8_NAN << 8);
    return r;
}
// Two codes as float16 (exact: e4m3's values are float16 values)
__device__ __forceinline__ uint32_t c8_half2(uint32_t two) {
    uint32_t d;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"((uint16_t)two));
    return d;
}
// Four codes as two float16 pairs
__device__ __forceinline__ void c8_half4(uint32_t four, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(four));
}
// Four codes rounded again after a factor of 2^-shift (half2 `factor`, both halves; shift at most 24, where everything is 0): the
// product is exact in float16 down to 2^-24 and lies below half of e4m3's smallest step before it is not.
__device__ __forceinline__ uint32_t c8_shift4(uint32_t four, uint32_t factor) {
    uint32_t lo = c8_half2(four & 0xffffu), hi = c8_half2(four >> 16);
    asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(factor));
    asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(hi) : "r"(factor));
    uint16_t a, b;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(a) : "r"(lo));
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(b) : "r"(hi));
    return (uint32_t)a | ((uint32_t)b << 16);
}
// half2 with 2^-shift in both halves, shift 0 to 24 (from 15 on subnormal)
__device__ __forceinline__ uint32_t c8_shift_factor(int shift) {
    const uint32_t h = shift < 15 ? (uint32_t)(15 - shift) << 10 : shift <= 24 ? 1u << (24 - shift) : 0u;
    return h | (h << 16);
}
__device__ __forceinline__ uint4 c8_shift16(uint4 v, uint32_t factor) {
    return make_uint4(c8_shift4(v.x, factor), c8_shift4(v.y, factor), c8_shift4(v.z, factor), c8_shift4(v.w, factor));
}

// Entry points of calls that single steps make take one packed struct (addresses first, then whole numbers, then floats: no gaps but the padding at
// its end, which the caller sends too) and its length, which costs the caller a fifth of what two dozen arguments do; it is copied, since a
// Python bytes object need not be aligned for it.
#define C8_REQUIRE_CALL(what, C) TQ_REQUIRE(packed != nullptr && bytes == (int)sizeof(C), "%s: a call of %d bytes, not %d", what, bytes, (int)sizeof(C))
template <typename C> inline C c8_call(const void* packed) {
    C c;
    memcpy(&c, packed, sizeof(c));
    return c;
}

inline Cache8 c8_cache(const void* codes, const void* scales, const int* table, int table_stride, int page_size, int n_pages, int nkv, int hd) {
    int shift = 0;
    while ((1 << shift) < page_size) ++shift;
    return Cache8{(uint8_t*)codes, (uint8_t*)scales, table, table_stride, page_size, n_pages, nkv, hd, (1 << shift) == page_size ? shift : -1};
}

inline int c8_check(const char* what, const void* codes, const void* scales, int page_size, int n_pages, int nkv, int hd, int table_stride) {
    TQ_REQUIRE(hd % 16 == 0 && hd >= 16 && hd <= C8_MAX_HEAD_DIM, "%s: head size %d is not a multiple of 16 up to %d", what, hd, C8_MAX_HEAD_DIM);
    TQ_REQUIRE(page_size >= C8_BLOCK && page_size % C8_BLOCK == 0, "%s: page size %d is not a multiple of %d", what, page_size, C8_BLOCK);
    TQ_REQUIRE(n_pages >= 0 && nkv >= 1 && table_stride >= 1, "%s: %d pages, %d key/value heads, page tables %d wide", what, n_pages, nkv, table_stride);
    // (the attention kernels' offsets within a page are 32 bits wide)
    TQ_REQUIRE((long long)nkv * page_size < (1ll << 31) / hd, "%s: pages of %d rows of %d heads of %d have 2^31 codes a plane or more", what, page_size, nkv, hd);
    TQ_REQUIRE((uintptr_t)codes % 16 == 0, "%s: the codes must be 16-byte aligned", what);
    (void)scales;
    return 0;
}
