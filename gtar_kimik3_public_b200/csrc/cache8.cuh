// The 8-bit cache: keys and values in pages as e4m3 numbers (four bits of exponent, three of mantissa, largest number 448) with one power
// of two a (position, kv head) beside them.
//
//   e = the smallest whole number with max |x| <= 448 * 2^e over the row's finite numbers, kept within -64 .. 119
//   x8 = round-to-nearest-even of x * 2^-e to e4m3 (numbers of less than 2^-6 have steps of 2^-9);  b = e + 127 is kept in a byte
//   x ~ x8 * 2^e
//
// A power of two, because x8 * 2^e is then exact in bfloat16 and in 32 bits, because b is the exponent field of the 32-bit number 2^e, and
// because a floating format gains nothing from a finer factor: the error is half a step, 2^-4 of the number, whatever the
// factor.  119 is the last power whose 448 * 2^e is a finite number; below 448 * 2^-64 a row's steps no longer shrink.  A number that is not
// finite is kept as e4m3's NaN (there is no infinity) and does not take part in the maximum.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

// One layer's pages, as the host hands them over (the same struct, field by field, in ops/functional.py).
struct GkPages8 {
    uint8_t *k, *v;          // [n_pages][n_kv][page_size][head_dim] e4m3
    uint8_t *k_exp, *v_exp;  // [n_pages][n_kv][page_size]
    const int* table;        // [n_slots][max_pages]
    int* error;              // where a kernel records a page, slot or length that cannot be
    long long n_pages;
    int n_slots, max_pages, n_kv, page_size, head_dim;
};

namespace cache8 {

constexpr int ERR_PLACE = 80;  // a slot, a page's number or a length outside the pools

constexpr int LOW = -64, HIGH = 119;

// The page that holds page `index` of the sequence in `slot`; -1, and a record of it, where there is no such page.
__device__ __forceinline__ int page_of(const GkPages8& p, int slot, int index) {
    int page = -1;
    if ((unsigned)slot < (unsigned)p.n_slots && (unsigned)index < (unsigned)p.max_pages) page = p.table[(size_t)slot * p.max_pages + index];
    if ((unsigned long long)(long long)page >= (unsigned long long)p.n_pages) {
        if (p.error) *p.error = ERR_PLACE;
        return -1;
    }
    return page;
}

// A sequence's length, none longer than its row of the table.
__device__ __forceinline__ int length_of(const GkPages8& p, int len) {
    const long long most = (long long)p.max_pages * p.page_size;
    if (len < 0 || len > most) {
        if (p.error) *p.error = ERR_PLACE;
        return len < 0 ? 0 : (int)most;
    }
    return len;
}

__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.f;  // NaN and infinities: nothing
}

// b of a row whose largest finite number is `top`: 448 is 1.75 * 2^8.
__device__ __forceinline__ int exponent_byte(float top) {
    const uint32_t bits = __float_as_uint(top);
    int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = e < LOW ? LOW : e > HIGH ? HIGH : e;
    return e + 127;
}

__device__ __forceinline__ float power_of(int b) { return __uint_as_float((uint32_t)b << 23); }          // 2^(b - 127), b = 63 .. 246
__device__ __forceinline__ float power_back(int b) { return __uint_as_float((uint32_t)(254 - b) << 23); }  // 2^(127 - b)

// Two numbers, scaled already, as e4m3: `lo` in the low byte.
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    // the conversion takes an infinity to 448; it is to be NaN like every number that is none
    lo = fabsf(lo) == INFINITY ? NAN : lo;
    hi = fabsf(hi) == INFINITY ? NAN : hi;
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Two e4m3 numbers as halves (exact).
__device__ __forceinline__ uint32_t halves2(uint16_t two) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(two));
    return r;
}
__device__ __forceinline__ float2 floats2(uint16_t two) {
    const uint32_t h = halves2(two);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// The host's part: what every entry asks of the pages.
inline int check(const GkPages8* p, const char* name) {
    GK_REQUIRE(p && p->k && p->v && p->k_exp && p->v_exp && p->table, "%s: pages are missing", name);
    GK_REQUIRE(p->n_pages > 0 && p->n_slots > 0 && p->max_pages > 0 && p->n_kv > 0 && p->page_size > 0 && p->page_size % 32 == 0,
               "%s: bad page geometry", name);
    GK_REQUIRE(p->head_dim > 0 && p->head_dim % 2 == 0 && p->head_dim <= 512, "%s: head_dim %d is not an even number up to 512", name, p->head_dim);
    GK_REQUIRE((((uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->k_exp | (uintptr_t)p->v_exp) & 15) == 0, "%s: pages must begin on 16-byte boundaries", name);
    return GK_OK;
}

}  // namespace cache8
