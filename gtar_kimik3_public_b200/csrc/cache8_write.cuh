// What is made of a row on its way into the 8-bit cache: RMSNorm and rotation, and its bytes.
#pragma once

#include "cache8.cuh"

namespace cache8 {

struct Norm8 {
    const void *wq, *wk;
    const float *cos_table, *sin_table;  // null: no rotation
    int table_positions, use_norm;
    float eps;
};

// A 64-bit number as 32 bits to be rounded on: what is cut off leaves its mark in the last bit, so that the second rounding is that of the number itself.
__device__ __forceinline__ float to_be_rounded(double x) {
    const float f = __double2float_rz(x);
    return (double)f == x || f != f ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

// RMSNorm and rotation of a row whose lanes hold N pairs each, pair i of a lane at `at(i)` of the halves; `lanes`: the row's, a power of two of them.
// Returns whether the position is one of the rotation's.
template <typename R, int N, typename TW, typename At>
__device__ __forceinline__ bool norm_rotate(R (&x)[N], R (&y)[N], const Norm8& a, const TW* w, int half, int pos, int lanes, unsigned mask, At at) {
    if (a.use_norm) {
        R ss = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) ss += x[i] * x[i] + y[i] * y[i];
        for (int o = 1; o < lanes; o <<= 1) ss += __shfl_xor_sync(mask, ss, o);
        const R inv = (R)1 / sqrt(ss / (R)(2 * half) + (R)a.eps);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (at(i) < half) {
                x[i] = (x[i] * inv) * (R)to_float(w[at(i)]);
                y[i] = (y[i] * inv) * (R)to_float(w[at(i) + half]);
            }
    }
    if (a.cos_table) {
        if ((unsigned)pos >= (unsigned)a.table_positions) return false;
        const float *cs = a.cos_table + (size_t)pos * half, *sn = a.sin_table + (size_t)pos * half;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (at(i) < half) {
                const R c = cs[at(i)], s = sn[at(i)], u = x[i], v = y[i];
                x[i] = u * c - v * s;
                y[i] = v * c + u * s;
            }
    }
    return true;
}

// ------------------------------------------------------------------ eight lanes a row of 64 or 128
template <int E, typename T>
__device__ __forceinline__ void load_run(const T* from, float (&v)[E]);
template <>
__device__ __forceinline__ void load_run<4, __nv_bfloat16>(const __nv_bfloat16* from, float (&v)[4]) {
    const uint2 raw = *reinterpret_cast<const uint2*>(from);
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.x)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.y));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}
template <>
__device__ __forceinline__ void load_run<8, __nv_bfloat16>(const __nv_bfloat16* from, float (&v)[8]) {
    const uint4 raw = *reinterpret_cast<const uint4*>(from);
    const __nv_bfloat162* pairs = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __bfloat1622float2(pairs[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}
template <>
__device__ __forceinline__ void load_run<4, float>(const float* from, float (&v)[4]) {
    const float4 f = *reinterpret_cast<const float4*>(from);
    v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
}
template <>
__device__ __forceinline__ void load_run<8, float>(const float* from, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
        const float4 f = *reinterpret_cast<const float4*>(from + i);
        v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
    }
}

template <>
__device__ __forceinline__ void load_run<2, __nv_bfloat16>(const __nv_bfloat16* from, float (&v)[2]) {
    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(from));
    v[0] = f.x, v[1] = f.y;
}
template <>
__device__ __forceinline__ void load_run<1, __nv_bfloat16>(const __nv_bfloat16* from, float (&v)[1]) { v[0] = __bfloat162float(*from); }
template <>
__device__ __forceinline__ void load_run<2, float>(const float* from, float (&v)[2]) {
    const float2 f = *reinterpret_cast<const float2*>(from);
    v[0] = f.x, v[1] = f.y;
}
template <>
__device__ __forceinline__ void load_run<1, float>(const float* from, float (&v)[1]) { v[0] = *from; }

// Two finite numbers, scaled already, as e4m3: `lo` in the low byte.
__device__ __forceinline__ uint32_t pack2_finite(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

template <int E>
__device__ __forceinline__ float sum_of_squares(const float (&x)[E], const float (&y)[E]) {  // a tree: seven roundings in a row with the lanes' three
    float s[E];
#pragma unroll
    for (int i = 0; i < E; ++i) s[i] = fmaf(x[i], x[i], y[i] * y[i]);
#pragma unroll
    for (int n = E / 2; n > 0; n >>= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) s[i] += s[i + n];
    return s[0];
}

// ------------------------------------------------------------------ a key as the formula in some 45 bits, rounded once
// A number as the sum of two 32-bit ones, the second at most half a step of the first: sums and products of two numbers are exact as such pairs (Dekker;
// Knuth).  64-bit arithmetic is a sixteenth as fast here.
struct Two8 {
    float h, l;
};
__device__ __forceinline__ Two8 sum_of(float a, float b) {
    const float s = __fadd_rn(a, b), t = __fsub_rn(s, a);
    return {s, __fadd_rn(__fsub_rn(a, __fsub_rn(s, t)), __fsub_rn(b, t))};
}
__device__ __forceinline__ Two8 product_of(float a, float b) {
    const float p = __fmul_rn(a, b);
    return {p, __fmaf_rn(a, b, -p)};
}
// The pair as 32 bits to be rounded on: what is cut off leaves its mark in the last bit.
__device__ __forceinline__ float to_be_rounded(float high, float low) {
    const float h = __fadd_rn(high, low), l = __fsub_rn(low, __fsub_rn(h, high));
    if (!(fabsf(h) < INFINITY) || l == 0.f) return fabsf(high) < INFINITY ? h : high;
    return __uint_as_float((__float_as_uint(h) - ((l < 0.f) != (h < 0.f) ? 1u : 0u)) | 1u);
}

constexpr float LARGEST = 3.402823466e38f;
// Squares whose sum is below SMALL_SQUARES end at 2^-149 with bits that count, where eps does not outweigh them; below LARGE_ROW no sum of squares leaves
// 32 bits.
constexpr float SMALL_EPS = 0x1p-60f, SMALL_SQUARES = 0x1p-52f, LARGE_ROW = 0x1p60f;

// A key, or a row of values as it is, by LANES lanes that have HD / 2 / LANES neighbouring numbers of each half: the numbers to be rounded; the byte of the
// row's power comes back.  By a whole warp rows of any size (FAR_ROW is added where squares had left 32 bits); by fewer lanes (where the registers that this
// takes cost the write more) only rows whose squares and rotation stay within 32 bits: the others are for `far_bytes`.
constexpr int FAR_ROW = 256;
// Two bytes of a far row: a zero has no sign, for the two ways of making it do not keep the same ones.
__device__ __forceinline__ uint32_t far_pair(uint32_t two) { return two & ~(__vcmpeq4(two & 0x7f7fu, 0u) & 0x8080u); }
template <int HD, int LANES, typename TW>
__device__ __forceinline__ int careful_row(const Norm8& a, const __nv_bfloat16* row, bool is_v, int pos, int sub, unsigned mask, float (&x)[2][HD / 2 / LANES]) {
    constexpr int E = HD / 2 / LANES, HALF = HD / 2;
    constexpr bool ANY = LANES == 32;
    bool far = false;
    float low[2][E];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        load_run<E>(row + h * HALF + sub * E, x[h]);
#pragma unroll
        for (int i = 0; i < E; ++i) low[h][i] = 0.f;
    }
    if (!is_v) {
        if (a.use_norm) {
            Two8 ss;
            float eps = a.eps;
            // (once, but for rows whose squares leave 32 bits: these a second time, the row times a power of two and eps times its square, which comes to
            // the same; the same code again, for a second sum of its own costs decode steps of 64 sequences 2%)
#pragma unroll 1
            for (;;) {
                ss = {0.f, 0.f};
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < E; ++i) {  // (the square of a bfloat16 number is exact)
                        const Two8 t = sum_of(ss.h, __fmul_rn(x[h][i], x[h][i]));
                        ss = {t.h, __fadd_rn(ss.l, t.l)};
                    }
#pragma unroll
                for (int o = 1; o < LANES; o <<= 1) {
                    const float oh = __shfl_xor_sync(mask, ss.h, o), ol = __shfl_xor_sync(mask, ss.l, o);
                    const Two8 t = sum_of(ss.h, oh);
                    ss = {t.h, __fadd_rn(t.l, __fadd_rn(ss.l, ol))};
                }
                if (!ANY || far || (ss.h < INFINITY && (eps >= SMALL_EPS || ss.h >= SMALL_SQUARES))) break;  // (the same for the lanes of the row)
                const float by = ss.h < INFINITY ? 0x1p70f : 0x1p-70f;
                far = true;
                eps = eps * by * by;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < E; ++i) x[h][i] *= by;
            }
            far = far && ss.h != 0.f;  // (a row of zeros is an ordinary one)
            const Two8 m = sum_of(ss.h * (1.f / HD), eps);  // (HD is a power of two)
            const float ml = fmaf(ss.l, 1.f / HD, m.l);
            float r = rsqrtf(m.h), dr = 0.f;
            if (m.h < INFINITY && m.h > 0.f) {  // 1 / sqrt(m) = r + dr: a step of Newton's
                const Two8 rr = product_of(r, r);
                const float e = __fsub_rn(__fmaf_rn(-rr.h, m.h, 1.f), __fmaf_rn(rr.l, m.h, __fmul_rn(rr.h, ml)));
                dr = 0.5f * r * e;
            }
            float w[2][E];
            load_run<E>((const TW*)a.wk + sub * E, w[0]);
            load_run<E>((const TW*)a.wk + HALF + sub * E, w[1]);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const Two8 p = product_of(x[h][i], w[h][i]), z = product_of(p.h, r);
                    x[h][i] = z.h;
                    low[h][i] = __fadd_rn(z.l, __fmaf_rn(p.h, dr, __fmul_rn(p.l, r)));
                }
        }
        if (a.cos_table && (unsigned)pos < (unsigned)a.table_positions) {
            float c[E], sn[E];
            load_run<E>(a.cos_table + (size_t)pos * HALF + sub * E, c);
            load_run<E>(a.sin_table + (size_t)pos * HALF + sub * E, sn);
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float u = x[0][i], v = x[1][i], ul = low[0][i], vl = low[1][i];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float s = h ? sn[i] : -sn[i];
                    const Two8 p = product_of(h ? v : u, c[i]), q = product_of(h ? u : v, s), t = sum_of(p.h, q.h);
                    x[h][i] = t.h;
                    low[h][i] = __fadd_rn(__fadd_rn(t.l, __fadd_rn(p.l, q.l)), __fmaf_rn(h ? vl : ul, c[i], __fmul_rn(h ? ul : vl, s)));
                    most = fmaxf(most, fabsf(t.h));
                }
            }
            if (ANY && !a.use_norm && __builtin_expect(most == INFINITY, 0)) {  // more than 32 bits hold: of finite numbers the largest that there is
                float u[E], v[E];
                load_run<E>(row + sub * E, u);
                load_run<E>(row + HALF + sub * E, v);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < E; ++i)
                        if (fabsf(x[h][i]) == INFINITY && fabsf(u[i]) < INFINITY && fabsf(v[i]) < INFINITY) {
                            x[h][i] = copysignf(LARGEST, x[h][i]);
                            low[h][i] = 0.f;
                        }
            }
        }
    }
    float top = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < E; ++i) {
            x[h][i] = to_be_rounded(x[h][i], low[h][i]);
            top = fmaxf(top, finite_abs(x[h][i]));
        }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) top = fmaxf(top, __shfl_xor_sync(mask, top, o));
    return exponent_byte(top) + (ANY && far ? FAR_ROW : 0);
}
// A key by eight lanes, as bytes: of any size, in 64 bits, a number after the other.
template <int HD, typename TW>
__device__ __noinline__ int far_bytes(const Norm8& a, const __nv_bfloat16* row, int pos, int sub, unsigned mask, uint32_t* four) {
    constexpr int E = HD / 16, HALF = HD / 2;
    const bool turns = a.cos_table && (unsigned)pos < (unsigned)a.table_positions;
    double inv = 1.0;
    if (a.use_norm) {
        double ss = 0.0;
#pragma unroll 1
        for (int i = 0; i < 2 * E; ++i) {
            const double x = __bfloat162float(row[(i < E ? i : HALF - E + i) + sub * E]);
            ss += x * x;
        }
        for (int o = 1; o < 8; o <<= 1) ss += __shfl_xor_sync(mask, ss, o);
        inv = 1.0 / sqrt(ss / HD + (double)a.eps);
    }
    float top = 0.f, back = 0.f;
    int b = 0;
#pragma unroll 1
    for (int i = 0; i < 4 * E; ++i) {  // twice through the lane's numbers: the maximum, the bytes
        const int h = i / E % 2, c = sub * E + i % E;
        if (i == 2 * E) {
            for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(mask, top, o));
            b = exponent_byte(top);
            back = power_back(b);
        }
        double u = __bfloat162float(row[c]), v = __bfloat162float(row[HALF + c]);
        if (a.use_norm) {
            u = (u * inv) * (double)to_float(((const TW*)a.wk)[c]);
            v = (v * inv) * (double)to_float(((const TW*)a.wk)[HALF + c]);
        }
        double x = h ? v : u;
        if (turns) {
            const double co = a.cos_table[(size_t)pos * HALF + c], si = a.sin_table[(size_t)pos * HALF + c];
            x = h ? v * co + u * si : u * co - v * si;
        }
        const float f = to_be_rounded(x);
        if (i < 2 * E) top = fmaxf(top, finite_abs(f));
        else reinterpret_cast<unsigned char*>(four)[i - 2 * E] = (unsigned char)far_pair(pack2(f * back, 0.f));
    }
    return b;
}
// The careful row by eight lanes, as bytes.
template <int HD, typename TW>
__device__ __noinline__ int careful_bytes(const Norm8& a, const __nv_bfloat16* row, bool is_v, bool far, int pos, int sub, unsigned mask, uint32_t* four) {
    constexpr int E = HD / 16;
    if (far) {  // it may be
        float most = 0.f, ss = 0.f;
        bool numbers = true;
#pragma unroll 1
        for (int i = 0; i < 2 * E; ++i) {
            const float v = fabsf(__bfloat162float(row[(i < E ? i : HD / 2 - E + i) + sub * E]));
            most = fmaxf(most, v);
            ss += v * v;
            numbers &= v < INFINITY;
        }
        for (int o = 1; o < 8; o <<= 1) {
            most = fmaxf(most, __shfl_xor_sync(mask, most, o));
            ss += __shfl_xor_sync(mask, ss, o);
        }
        if (!__all_sync(mask, numbers) || most >= LARGE_ROW || (most > 0.f && ss < SMALL_SQUARES && a.eps < SMALL_EPS))
            return far_bytes<HD, TW>(a, row, pos, sub, mask, four);
    }
    float x[2][E];
    const int b = careful_row<HD, 8, TW>(a, row, is_v, pos, sub, mask, x);
    const float back = power_back(b);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < E; i += 4)
            four[h * (E / 4) + i / 4] = pack2(x[h][i] * back, x[h][i + 1] * back) | pack2(x[h][i + 2] * back, x[h][i + 3] * back) << 16;
    return b;
}

// RMSNorm and rotation of a row in 32 bits.
template <int HD>
__device__ __forceinline__ void norm_rotate_32(const Norm8& a, float (&x)[HD / 16], float (&y)[HD / 16], const float (&w0)[HD / 16], const float (&w1)[HD / 16],
                                               const float (&c)[HD / 16], const float (&sn)[HD / 16], bool turns, unsigned mask) {
    constexpr int E = HD / 16;
    if (a.use_norm) {
        float ss = sum_of_squares(x, y);
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) ss += __shfl_xor_sync(mask, ss, o);
        const float inv = rsqrtf(fmaf(ss, 1.f / HD, a.eps));
#pragma unroll
        for (int i = 0; i < E; ++i) {
            x[i] = (x[i] * inv) * w0[i];
            y[i] = (y[i] * inv) * w1[i];
        }
    }
    if (turns) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float u = x[i], v = y[i];
            x[i] = u * c[i] - v * sn[i];
            y[i] = v * c[i] + u * sn[i];
        }
    }
}

// A lane's bytes of a key (normed and rotated in 32 bits, `row` what it was made of) or of a row of values; the byte of the row's power comes back.
template <int HD, typename TW>
__device__ __forceinline__ int make_bytes(const Norm8& a, const float (&x)[HD / 16], const float (&y)[HD / 16], bool turns, bool is_v, const __nv_bfloat16* row,
                                          int pos, int sub, unsigned mask, uint32_t (&four)[2][HD / 64]) {
    constexpr int E = HD / 16;
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) top = fmaxf(top, fmaxf(fabsf(x[i]), fabsf(y[i])));  // (passes over NaN)
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(mask, top, o));
    const int b = exponent_byte(top);
    const float back = power_back(b);
    // a row whose maximum is 0 or not to be trusted: it holds an infinity or NaN and is normed, its squares leave 32 bits (zeros come of it; or, with next
    // to no eps, lost bits), or its rotation does
    const bool far = !is_v && (top >= 0x1p127f || (a.use_norm && (top == 0.f || a.eps < SMALL_EPS)));  // (the same for the lanes of the row)
    bool care = far || top == INFINITY;
    if (is_v || !(a.use_norm || turns)) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < E; i += 4)
                four[h][i / 4] = pack2_finite((h ? y : x)[i] * back, (h ? y : x)[i + 1] * back) | pack2_finite((h ? y : x)[i + 2] * back, (h ? y : x)[i + 3] * back) << 16;
    } else {
        // How far a number x of a rotated pair (x, y) is from the formula, with r = 2^-24 for a rounding: 8 r of itself through the norm's factor (seven
        // roundings of the sum of squares and one of the mean, halved by the root; rsqrtf's two steps, 4 r), 3 r of what the rotation mixes, |u c| + |v s|
        // (the factor, the weight, the product), and r of itself through the last sum.  (|u c| + |v s|)^2 <= (u^2 + v^2) (c^2 + s^2) = x^2 + y^2, so that
        // this is 9 r |x| + 3 r (|x| + |y|), no more than 7.2e-7 of |x| + |y|; the test below rounds once more, 0.6e-7.  Where 1.25e-6 of |x| + |y| less
        // and as much more are not the same byte, or the maximum lies within 2^-18 of the next power's, the row is made over.
        care |= abs((int)(__float_as_uint(top) & 0x7fffffu) - 0x600000) < 32;
        const float slack = 1.25e-6f * back;
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            uint32_t less[2][2], more[2][2];
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const float t0 = slack * (fabsf(x[i + e]) + fabsf(y[i + e])), t1 = slack * (fabsf(x[i + e + 1]) + fabsf(y[i + e + 1]));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float u = (h ? y : x)[i + e], v = (h ? y : x)[i + e + 1];
                    less[h][e / 2] = pack2_finite(fmaf(u, back, -t0), fmaf(v, back, -t1));
                    more[h][e / 2] = pack2_finite(fmaf(u, back, t0), fmaf(v, back, t1));
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                four[h][i / 4] = less[h][0] | less[h][1] << 16;
                care |= four[h][i / 4] != (more[h][0] | more[h][1] << 16);
            }
        }
    }
    if (__any_sync(mask, care)) {
        uint32_t anew[2 * (E / 4)];
        const int power = careful_bytes<HD, TW>(a, row, is_v, far, pos, sub, mask, anew);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < E / 4; ++i) four[h][i] = anew[h * (E / 4) + i];
        return power;
    }
    return b;
}

}  // namespace cache8
