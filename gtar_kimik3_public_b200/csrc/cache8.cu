// Writing keys and values into the 8-bit cache, and reading them back (what is kept: cache8.cuh).
//
// The write does the attention input stage too, as the 16-bit cache's does: per-head RMSNorm of q and k (src/layers/rmsnorm.py:11-16),
// rotation (src/layers/rope.py:17-33), order of src/layers/attention.py:82-89.  All of it is 32-bit up to the one rounding of
// each result: q to its type, k and v to e4m3.

#include "cache8.cuh"

namespace {

using namespace cache8;

// ------------------------------------------------------------------ write
struct Write8 {
    const void *qkv, *wq, *wk;
    const float *cos_table, *sin_table;
    const int *tok_pos, *tok_seq, *slots;
    void* q_out;
    int n_tokens, n_q, n_seqs, table_positions, use_norm, write_kv;
    float eps;
};

// The byte that a k or v row's place begins at, or null.
__device__ __forceinline__ long long place_of(const GkPages8& p, const Write8& a, int t, int pos, int hk) {
    const int seq = a.tok_seq[t];
    if ((unsigned)seq >= (unsigned)a.n_seqs || pos < 0) {
        if (p.error) *p.error = ERR_PLACE;
        return -1;
    }
    const int page = page_of(p, a.slots[seq], pos / p.page_size);
    return page < 0 ? -1 : ((long long)page * p.n_kv + hk) * p.page_size + pos % p.page_size;
}

// A warp a (token, head): lane l has the pairs (i, i + head_dim / 2) of the rotation for i = l, l + 32, ...
template <typename T, typename TW>
__global__ void __launch_bounds__(128) write8_kernel(const GkPages8 p, const Write8 a) {
    constexpr int MAXP = 8;  // head_dim <= 512
    pdl_launch_dependents();
    pdl_wait();
    const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, n_heads = a.n_q + 2 * p.n_kv, d = p.head_dim, half = d >> 1;
    if (item >= (long long)a.n_tokens * n_heads) return;
    const int t = (int)(item / n_heads), head = (int)(item - (long long)t * n_heads);
    const bool is_q = head < a.n_q, is_k = !is_q && head < a.n_q + p.n_kv;
    if (!is_q && !a.write_kv) return;
    const int pos = a.tok_pos[t];
    const T* in = (const T*)a.qkv + ((size_t)t * n_heads + head) * d;
    float x[MAXP], y[MAXP];
#pragma unroll
    for (int i = 0; i < MAXP; ++i) {
        const int c = lane + 32 * i;
        x[i] = c < half ? to_float(in[c]) : 0.f;
        y[i] = c < half ? to_float(in[c + half]) : 0.f;
    }
    if (is_q || is_k) {
        if (a.use_norm) {
            const TW* w = (const TW*)(is_q ? a.wq : a.wk);
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < MAXP; ++i) ss += x[i] * x[i] + y[i] * y[i];
            const float inv = 1.0f / sqrtf(warp_sum(ss) / (float)d + a.eps);
#pragma unroll
            for (int i = 0; i < MAXP; ++i) {
                const int c = lane + 32 * i;
                if (c < half) {
                    x[i] = (x[i] * inv) * to_float(w[c]);
                    y[i] = (y[i] * inv) * to_float(w[c + half]);
                }
            }
        }
        if (a.cos_table) {
            if ((unsigned)pos >= (unsigned)a.table_positions) {
                if (p.error && lane == 0) *p.error = ERR_PLACE;
                return;
            }
#pragma unroll
            for (int i = 0; i < MAXP; ++i) {
                const int c = lane + 32 * i;
                if (c < half) {
                    const float cs = a.cos_table[(size_t)pos * half + c], sn = a.sin_table[(size_t)pos * half + c], u = x[i], v = y[i];
                    x[i] = u * cs - v * sn;
                    y[i] = v * cs + u * sn;
                }
            }
        }
    }
    if (is_q) {
        T* out = (T*)a.q_out + ((size_t)t * a.n_q + head) * d;
#pragma unroll
        for (int i = 0; i < MAXP; ++i) {
            const int c = lane + 32 * i;
            if (c < half) {
                out[c] = from_float<T>(x[i]);
                out[c + half] = from_float<T>(y[i]);
            }
        }
        return;
    }
    const long long place = place_of(p, a, t, pos, head - a.n_q - (is_k ? 0 : p.n_kv));
    if (place < 0) return;
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < MAXP; ++i) top = fmaxf(top, fmaxf(finite_abs(x[i]), finite_abs(y[i])));
    const int b = exponent_byte(warp_max(top));
    const float back = power_back(b);
    uint8_t* to = (is_k ? p.k : p.v) + place * d;
#pragma unroll
    for (int i = 0; i < MAXP; ++i) {
        const int c = lane + 32 * i;
        if (c < half) {
            const uint32_t two = pack2(x[i] * back, y[i] * back);
            to[c] = (uint8_t)two;
            to[c + half] = (uint8_t)(two >> 8);
        }
    }
    if (lane == 0) (is_k ? p.k_exp : p.v_exp)[place] = (uint8_t)b;
}

// The same for bfloat16 rows of 64 or 128: eight lanes a (token, head), which have HD / 16 neighbouring numbers of each half of the row in registers
// from the load to the store.  Everything a lane needs is asked for at once.
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

template <int HD, typename TW>
__global__ void __launch_bounds__(256) write8_wide_kernel(const GkPages8 p, const Write8 a) {
    constexpr int E = HD / 16, HALF = HD / 2;
    pdl_launch_dependents();
    pdl_wait();
    const int n_heads = a.n_q + 2 * p.n_kv, sub = threadIdx.x & 7;
    const long long item = (long long)blockIdx.x * 32 + (threadIdx.x >> 3);
    const bool valid = item < (long long)a.n_tokens * n_heads;  // every lane stays for the shuffles
    const int t = valid ? (int)(item / n_heads) : 0, head = valid ? (int)(item - (long long)t * n_heads) : 0;
    const bool is_q = head < a.n_q, is_k = !is_q && head < a.n_q + p.n_kv;
    const int pos = a.tok_pos[t];
    long long place = -1;
    if (valid && !is_q && a.write_kv) place = place_of(p, a, t, pos, head - a.n_q - (is_k ? 0 : p.n_kv));
    const __nv_bfloat16* in = (const __nv_bfloat16*)a.qkv + ((size_t)t * n_heads + head) * HD + sub * E;
    float x[E], y[E];
    load_run<E>(in, x);
    load_run<E>(in + HALF, y);
    bool good = true;
    const unsigned row_lanes = 0xffu << (threadIdx.x & 24);  // the lanes of this row go one way
    if (is_q || is_k) {
        if (a.use_norm) {
            const TW* w = (const TW*)(is_q ? a.wq : a.wk) + sub * E;
            float u[E], v[E], ss = 0.f;
            load_run<E>(w, u);
            load_run<E>(w + HALF, v);
#pragma unroll
            for (int i = 0; i < E; ++i) ss += x[i] * x[i] + y[i] * y[i];
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) ss += __shfl_xor_sync(row_lanes, ss, o);
            const float inv = 1.0f / sqrtf(ss / (float)HD + a.eps);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                x[i] = (x[i] * inv) * u[i];
                y[i] = (y[i] * inv) * v[i];
            }
        }
        if (a.cos_table) {
            good = (unsigned)pos < (unsigned)a.table_positions;
            if (good) {
                float c[E], sn[E];
                load_run<E>(a.cos_table + (size_t)pos * HALF + sub * E, c);
                load_run<E>(a.sin_table + (size_t)pos * HALF + sub * E, sn);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const float u = x[i], v = y[i];
                    x[i] = u * c[i] - v * sn[i];
                    y[i] = v * c[i] + u * sn[i];
                }
            } else if (valid && p.error) {
                *p.error = ERR_PLACE;
            }
        }
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) top = fmaxf(top, fmaxf(finite_abs(x[i]), finite_abs(y[i])));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!valid || !good) return;
    if (is_q) {
        __nv_bfloat16* out = (__nv_bfloat16*)a.q_out + ((size_t)t * a.n_q + head) * HD + sub * E;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t two[E / 2];
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                const __nv_bfloat162 pair = h ? __floats2bfloat162_rn(y[i], y[i + 1]) : __floats2bfloat162_rn(x[i], x[i + 1]);
                two[i / 2] = *reinterpret_cast<const uint32_t*>(&pair);
            }
            if constexpr (E == 8) *reinterpret_cast<uint4*>(out + h * HALF) = make_uint4(two[0], two[1], two[E / 2 - 2], two[E / 2 - 1]);
            else *reinterpret_cast<uint2*>(out + h * HALF) = make_uint2(two[0], two[1]);
        }
        return;
    }
    if (place < 0) return;
    const int b = exponent_byte(top);
    const float back = power_back(b);
    uint8_t* to = (is_k ? p.k : p.v) + place * HD + sub * E;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t four[E / 4];
#pragma unroll
        for (int i = 0; i < E; i += 4)
            four[i / 4] = h ? pack2(y[i] * back, y[i + 1] * back) | pack2(y[i + 2] * back, y[i + 3] * back) << 16
                            : pack2(x[i] * back, x[i + 1] * back) | pack2(x[i + 2] * back, x[i + 3] * back) << 16;
        if constexpr (E == 8) *reinterpret_cast<uint2*>(to + h * HALF) = make_uint2(four[0], four[E / 4 - 1]);
        else *reinterpret_cast<uint32_t*>(to + h * HALF) = four[0];
    }
    if (sub == 0) (is_k ? p.k_exp : p.v_exp)[place] = (uint8_t)b;
}

// ------------------------------------------------------------------ read back
// For attention over what was read: pages renumbered under a table, lengths and slots of their own, so that no number that cannot be reaches it; and
// a row of values that holds a NaN becomes zeros with a NaN key, which a token that does not see it cannot meet (0 * NaN).
struct Clean8 {
    int *table, *kv_len, *slots;  // [n_seqs][per], [n_seqs], [n_seqs]; null: read back under the pages' own numbers
    int per, own_numbers;         // pages a sequence; whether a page keeps its number or is seq * per + index
};

// N numbers of a row as bfloat16: e4m3 times a power of two, exact.
template <int N>
__device__ __forceinline__ void widen(const uint32_t* four, float f, uint32_t* out) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const float2 a = floats2((uint16_t)four[i]), b = floats2((uint16_t)(four[i] >> 16));
        const __nv_bfloat162 lo = __floats2bfloat162_rn(a.x * f, a.y * f), hi = __floats2bfloat162_rn(b.x * f, b.y * f);
        out[2 * i] = *reinterpret_cast<const uint32_t*>(&lo);
        out[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&hi);
    }
}

// Block (page of the sequence, sequence, kv head): the page's keys and values of the head as bfloat16; zeros behind the sequence's end.  HD / 16
// lanes a row, sixteen numbers each; HD = 0: any size, two numbers at a time.
template <int HD, bool CLEAN>
__global__ void __launch_bounds__(256) read8_kernel(const GkPages8 p, const int* __restrict__ kv_len, const int* __restrict__ slots, int last,
                                                    __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out, const Clean8 clean) {
    pdl_launch_dependents();
    pdl_wait();
    const int seq = blockIdx.y, index = blockIdx.x, hk = blockIdx.z, d = HD ? HD : p.head_dim;
    int len = length_of(p, kv_len[seq]);
    if (CLEAN && len > (long long)clean.per * p.page_size) {
        if (p.error) *p.error = ERR_PLACE;
        len = clean.per * p.page_size;
    }
    const bool seen = (long long)index * p.page_size < len && (last <= 0 || (index + 1) * (long long)p.page_size > (long long)len - last);
    const int page = seen ? page_of(p, slots[seq], index) : -1;
    int to_page = page;
    if (CLEAN) {
        to_page = clean.own_numbers ? max(page, 0) : seq * clean.per + index;
        if (hk == 0 && threadIdx.x == 0) {
            clean.table[seq * clean.per + index] = to_page;
            if (index == 0) {
                clean.kv_len[seq] = len;
                clean.slots[seq] = seq;
            }
        }
        if (!seen || (clean.own_numbers && page < 0)) return;
    } else if (page < 0) {
        return;
    }
    const int rows = page < 0 ? 0 : min(p.page_size, len - index * p.page_size);
    const size_t from = ((size_t)max(page, 0) * p.n_kv + hk) * p.page_size, to = ((size_t)to_page * p.n_kv + hk) * p.page_size;
    if constexpr (HD > 0) {
        constexpr int LANES = HD / 16;
        const int c = threadIdx.x % LANES * 16;
        for (int row = threadIdx.x / LANES; row < p.page_size; row += 256 / LANES) {
            uint32_t k[8] = {0, 0, 0, 0, 0, 0, 0, 0}, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (row < rows) {
                const uint4 x = *reinterpret_cast<const uint4*>(p.k + (from + row) * HD + c), y = *reinterpret_cast<const uint4*>(p.v + (from + row) * HD + c);
                const uint32_t ks[4] = {x.x, x.y, x.z, x.w}, vs[4] = {y.x, y.y, y.z, y.w};
                widen<16>(ks, power_of(p.k_exp[from + row]), k);
                widen<16>(vs, power_of(p.v_exp[from + row]), v);
                if (CLEAN) {
                    bool nan = false;
#pragma unroll
                    for (int i = 0; i < 4; ++i) nan |= __vcmpeq4(vs[i] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0;
                    const unsigned mine = ((1u << LANES) - 1) << ((threadIdx.x & 31) / LANES * LANES);
                    if (__ballot_sync(mine, nan) & mine) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = 0u, k[i] = 0x7fff7fffu;
                    }
                }
            }
            store32(k_out + (to + row) * HD + c, k);
            store32(v_out + (to + row) * HD + c, v);
        }
    } else {
        const int pairs = d >> 1;
        for (int i = threadIdx.x; i < p.page_size * pairs; i += 256) {
            const int row = i / pairs, c = (i - row * pairs) * 2;
            __nv_bfloat162 k = __floats2bfloat162_rn(0.f, 0.f), v = k;
            if (row < rows) {
                const float fk = power_of(p.k_exp[from + row]), fv = power_of(p.v_exp[from + row]);
                const float2 x = floats2(*reinterpret_cast<const uint16_t*>(p.k + (from + row) * d + c));
                const float2 y = floats2(*reinterpret_cast<const uint16_t*>(p.v + (from + row) * d + c));
                k = __floats2bfloat162_rn(x.x * fk, x.y * fk);
                v = __floats2bfloat162_rn(y.x * fv, y.y * fv);
            }
            *reinterpret_cast<__nv_bfloat162*>(k_out + (to + row) * d + c) = k;
            *reinterpret_cast<__nv_bfloat162*>(v_out + (to + row) * d + c) = v;
        }
    }
}

template <bool CLEAN>
int launch_read8(const GkPages8& p, const int* kv_len, const int* slots, int n_seqs, int most, int last, void* k_out, void* v_out, const Clean8& clean,
                 cudaStream_t stream) {
    const dim3 grid(most, n_seqs, p.n_kv);
    __nv_bfloat16 *k = (__nv_bfloat16*)k_out, *v = (__nv_bfloat16*)v_out;
    const bool wide = (((uintptr_t)k_out | (uintptr_t)v_out) & 31) == 0;  // 32-byte stores
    if (p.head_dim == 128 && wide) gk_launch(read8_kernel<128, CLEAN>, grid, dim3(256), 0, stream, p, kv_len, slots, last, k, v, clean);
    else if (p.head_dim == 64 && wide) gk_launch(read8_kernel<64, CLEAN>, grid, dim3(256), 0, stream, p, kv_len, slots, last, k, v, clean);
    else if constexpr (!CLEAN) gk_launch(read8_kernel<0, CLEAN>, grid, dim3(256), 0, stream, p, kv_len, slots, last, k, v, clean);
    else return gk_fail(GK_BAD_ARGUMENT, "read8: head_dim %d is not 64 or 128, or memory begins between 32 bytes", p.head_dim);
    GK_CHECK_LAUNCH("read8");
    return GK_OK;
}

}  // namespace

// `qkv` [n_tokens][(n_q + 2 n_kv) * head_dim] float32 or bfloat16; `q_out` [n_tokens][n_q][head_dim] of the same type.  Without
// `write_kv` the pages are left alone.
GK_EXPORT int gk_write8(const GkPages8* pages, const void* qkv, int dtype, const void* wq, const void* wk, int weight_dtype, int use_norm, float eps,
                        const float* cos_table, const float* sin_table, int table_positions, int max_position, const int* tok_pos,
                        const int* tok_seq, const int* slots, int n_seqs, void* q_out, int n_tokens, int n_q, int write_kv, void* stream) {
    const int status = cache8::check(pages, "write8");
    if (status != GK_OK) return status;
    GK_REQUIRE(GK_VALID_DTYPE(dtype) && GK_VALID_DTYPE(weight_dtype), "write8: bad dtype code");
    GK_REQUIRE(n_tokens >= 0 && n_q > 0 && n_seqs >= 0 && n_q % pages->n_kv == 0, "write8: bad sizes n_tokens=%d n_q=%d n_kv=%d", n_tokens, n_q, pages->n_kv);
    GK_REQUIRE(!use_norm || (wq && wk), "write8: norm weights missing");
    GK_REQUIRE((cos_table == nullptr) == (sin_table == nullptr), "write8: cos and sin tables go together");
    GK_REQUIRE(cos_table == nullptr || max_position < table_positions, "write8: position %d is beyond the rotary table (%d positions)", max_position,
               table_positions);
    if (n_tokens == 0) return GK_OK;
    GK_REQUIRE(qkv && q_out && tok_pos && tok_seq && slots, "write8: an array is missing");
    const Write8 a = {qkv, wq, wk, cos_table, sin_table, tok_pos, tok_seq, slots, q_out, n_tokens, n_q, n_seqs, table_positions, use_norm, write_kv, eps};
    const long long items = (long long)n_tokens * (n_q + 2 * pages->n_kv), blocks = (items + 3) / 4;
    GK_REQUIRE(blocks < 2147483647LL, "write8: too many tokens");
    if (dtype == GK_BF16 && (pages->head_dim == 64 || pages->head_dim == 128) && (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)wq | (uintptr_t)wk |
                                                                                  (uintptr_t)cos_table | (uintptr_t)sin_table) & 15) == 0) {
        GK_DISPATCH_DTYPE(weight_dtype, TW, {
            if (pages->head_dim == 64) gk_launch(write8_wide_kernel<64, TW>, dim3((unsigned)((items + 31) / 32)), dim3(256), 0, (cudaStream_t)stream, *pages, a);
            else gk_launch(write8_wide_kernel<128, TW>, dim3((unsigned)((items + 31) / 32)), dim3(256), 0, (cudaStream_t)stream, *pages, a);
        })
        GK_CHECK_LAUNCH("write8");
        return GK_OK;
    }
    GK_DISPATCH_DTYPE(dtype, T, {
        GK_DISPATCH_DTYPE(weight_dtype, TW, {
            gk_launch(write8_kernel<T, TW>, dim3((unsigned)blocks), dim3(128), 0, (cudaStream_t)stream, *pages, a);
        })
    })
    GK_CHECK_LAUNCH("write8");
    return GK_OK;
}

// The pages that hold each sequence's last `last` positions (0: all) as bfloat16 pages of the same numbers and geometry.
GK_EXPORT int gk_read8(const GkPages8* pages, const int* kv_len, const int* slots, int n_seqs, int max_kv_len, int last, void* k_out, void* v_out,
                       void* stream) {
    const int status = cache8::check(pages, "read8");
    if (status != GK_OK) return status;
    GK_REQUIRE(n_seqs >= 0 && n_seqs <= 65535 && max_kv_len >= 0 && last >= 0, "read8: bad sizes n_seqs=%d max_kv_len=%d last=%d", n_seqs, max_kv_len, last);
    if (n_seqs == 0 || max_kv_len == 0) return GK_OK;
    GK_REQUIRE(kv_len && slots && k_out && v_out, "read8: an array is missing");
    int most = (int)(((long long)max_kv_len + pages->page_size - 1) / pages->page_size);
    if (most > pages->max_pages) most = pages->max_pages;
    return launch_read8<false>(*pages, kv_len, slots, n_seqs, most, last, k_out, v_out, Clean8{}, (cudaStream_t)stream);
}

// The same for attention over what is read: `per` pages a sequence under numbers seq * per + index (`own_numbers`: their own), and `table`
// [n_seqs][per], `len_out` and `slots_out` [n_seqs] to go with them.  Heads of 64 or 128.
GK_EXPORT int gk_clean8(const GkPages8* pages, const int* kv_len, const int* slots, int n_seqs, int per, int own_numbers, int last, void* k_out, void* v_out,
                        int* table, int* len_out, int* slots_out, void* stream) {
    const int status = cache8::check(pages, "clean8");
    if (status != GK_OK) return status;
    GK_REQUIRE(n_seqs >= 0 && n_seqs <= 65535 && per > 0 && last >= 0 && (long long)n_seqs * per < 2147483647LL, "clean8: bad sizes n_seqs=%d per=%d last=%d",
               n_seqs, per, last);
    if (n_seqs == 0) return GK_OK;
    GK_REQUIRE(kv_len && slots && k_out && v_out && table && len_out && slots_out, "clean8: an array is missing");
    return launch_read8<true>(*pages, kv_len, slots, n_seqs, per, last, k_out, v_out, Clean8{table, len_out, slots_out, per, own_numbers}, (cudaStream_t)stream);
}
