// The 8-bit cache's format and what its kernels share.
//
// A cached row (the key or the value of one token and kv head, hd features) is held as hd e4m3 codes c_i and one
// byte s: the values are c_i * 2^(s - 127).  With a = max |x_i| over the row's finite numbers, s - 127 is the
// smallest integer e for which a <= 448 * 2^e (448: e4m3's largest), held in [-100, 119]; c_i = e4m3(x_i * 2^-e),
// rounded to nearest even.  A power of two instead of a / 448: the codes float, so a row loses nothing by it but one
// binade of range below its largest number, while x * 2^-e and c * 2^e are exact, so that reading a row back rounds
// nothing (e4m3 times 2^e is a bfloat16 for every e allowed) and a scale is one byte.  e >= -100 keeps the smallest
// code's value a normal bfloat16, e <= 119 the largest code's finite.
//
// A row with a number that is not finite is held as codes of zero and the byte 255, and stands for NaNs; a query that
// sees such a key or value gives NaNs.  No code is ever a NaN, so that a product over a tile of keys leaves the
// queries alone that see none of the tile's bad rows (a weight of zero times NaN would not).
//
// The cache of a layer: codes [pages, 2, kv_heads, page_size, hd], scale bytes [pages, 2, kv_heads, page_size].
// Page numbers outside the cache are brought into it before a read (a table's entry of a page that was given back
// is -1), and nothing is written to them.
#pragma once

#include <cuda_fp8.h>
#include <string.h>

#include "common.cuh"

#define KV8_LEAST_BYTE 27     // 2^-100
#define KV8_MOST_BYTE 246     // 2^119

#define KV8_BAD_BYTE 255      // the row is NaNs; its codes are zeros, and kv8_scale gives infinity: 0 * inf = NaN

// The scale byte of a row whose largest number is `most` >= 0, infinity for a row that is not finite: with most = 1.m * 2^(E - 127), 448 * 2^e =
// 1.75 * 2^(e + 8) is the first not below it for e = E - 135, or one more where 1.m > 1.75.
__device__ __forceinline__ int kv8_scale_byte(float most) {
    if (!(most < INFINITY)) return KV8_BAD_BYTE;
    const uint32_t b = __float_as_uint(most);
    const int s = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(s, KV8_LEAST_BYTE), KV8_MOST_BYTE);
}
__device__ __forceinline__ float kv8_scale(int byte) { return __uint_as_float((uint32_t)byte << 23); }
__device__ __forceinline__ float kv8_inverse_scale(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }

// Four codes from four numbers (already times the inverse scale), the first in the lowest byte.
__device__ __forceinline__ uint32_t kv8_pack4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}
// The numbers that four codes stand for, without the row's scale.
__device__ __forceinline__ void kv8_unpack4(uint32_t w, float* v) {
    const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
    const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    v[0] = a.x;
    v[1] = a.y;
    v[2] = b.x;
    v[3] = b.y;
}

// Values as bfloat16 with their row's scale, which is exact for every scale: sign, exponent and mantissa of a code are moved to
// bfloat16's places, which reads as the code times 2^-120, subnormal codes included, and a product by 2^(120 + e) puts it
// right: by 2^min(120 + e, 127), in the low half of the factors, and by 2^max(e - 7, 0), in the high one.
__device__ __forceinline__ uint32_t kv8_value_factors(int e) {
    return ((uint32_t)(min(120 + e, 127) + 127) << 7) | ((uint32_t)(max(e - 7, 0) + 127) << 23);
}
__device__ __forceinline__ uint32_t kv8_mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// 16 codes of a row in their order
__device__ __forceinline__ void kv8_values16(const uint4& x, uint32_t f, uint32_t (&y)[8]) {
    const uint32_t in[4] = {x.x, x.y, x.z, x.w}, f1 = __byte_perm(f, f, 0x1010);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t lo = __byte_perm(in[k], 0u, 0x1404), hi = __byte_perm(in[k], 0u, 0x3424);      // a code above a zero byte
        y[2 * k] = kv8_mul_bf16x2((lo & 0x80008000u) | ((lo >> 4) & 0x07f007f0u), f1);
        y[2 * k + 1] = kv8_mul_bf16x2((hi & 0x80008000u) | ((hi >> 4) & 0x07f007f0u), f1);
    }
    if ((f >> 16) != 0x3f80u) {                           // a scale above 2^7
        const uint32_t f2 = __byte_perm(f, f, 0x3232);
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = kv8_mul_bf16x2(y[k], f2);
    }
}

// Division of a number in [0, 2^31) by a fixed page size d: with s = ceil(log2 d) and m = ceil(2^(31 + s) / d) < 2^32 + 1,
// m d - 2^(31 + s) < d <= 2^s, so that n m / 2^(31 + s) exceeds n / d by less than 2^-31 n / d < 1 / d and has its floor.
struct PageSplit {
    int size;
    uint32_t magic;
    int shift;
};
static inline PageSplit page_split(int size) {
    int s = 0;
    while ((1ll << s) < size) ++s;
    return PageSplit{size, (uint32_t)(((1ull << (31 + s)) + size - 1) / size), 31 + s};
}
__device__ __forceinline__ int page_of(const PageSplit& p, int key) {
    return (int)(((uint64_t)(uint32_t)key * p.magic) >> p.shift);
}
// The page that a request's table (a row of `width` entries) names for its page `logical`, brought into the cache.
__device__ __forceinline__ int page_id(const int* table, int logical, int width, int pages) {
    return (int)min((unsigned)table[min(logical, width - 1)], (unsigned)(pages - 1));
}

// The keys that the rows from position `first` to position `last` of one request can see, counted as v = 0 ..
// seen_count - 1: the kept first keys that lie before the window, then the window's keys up to `last`.
struct SeenKeys {
    int kept, lo, count;
};
__device__ __forceinline__ SeenKeys seen_keys(int first, int last, int window, int keep_first) {
    SeenKeys s;
    s.lo = window > 0 && first >= window ? first - window + 1 : 0;      // (`first` may be negative, the window 2^31 - 1)
    s.kept = min(keep_first, s.lo);
    s.count = max(0, last + 1 - s.lo + s.kept);
    return s;
}
__device__ __forceinline__ int key_of(const SeenKeys& s, int v) { return v < s.kept ? v : v - s.kept + s.lo; }
__device__ __forceinline__ bool sees(int pos, int key, int window, int keep_first) {
    return key <= pos && (window <= 0 || key > pos - window || key < keep_first);
}

// The entry points also take their arguments as one array of 64-bit numbers, a float as the bits of a double: a call
// through ctypes converts each argument by itself, 3.6 us for 21 of them against 0.7 for one packed string.
static inline float kv8_packed_float(long long bits) {
    double d;
    memcpy(&d, &bits, sizeof(d));
    return (float)d;
}
