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

// ------------------------------------------------------------------ read back
// Block (page of the sequence, sequence): the page's keys and values of every kv head as bfloat16 under the same page number; zeros behind the
// sequence's end.  Exact: e4m3 times a power of two.
__global__ void __launch_bounds__(256) read8_kernel(const GkPages8 p, const int* __restrict__ kv_len, const int* __restrict__ slots, int last,
                                                    __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out) {
    pdl_launch_dependents();
    pdl_wait();
    const int seq = blockIdx.y, index = blockIdx.x, d = p.head_dim;
    const int len = length_of(p, kv_len[seq]);
    if ((long long)index * p.page_size >= len) return;
    if (last > 0 && (index + 1) * (long long)p.page_size <= (long long)len - last) return;
    const int page = page_of(p, slots[seq], index);
    if (page < 0) return;
    const int rows = min(p.page_size, len - index * p.page_size), pairs = d >> 1;
    const size_t base = (size_t)page * p.n_kv * p.page_size;
    for (int i = threadIdx.x; i < p.n_kv * p.page_size * pairs; i += blockDim.x) {
        const int place = i / pairs, c = (i - place * pairs) * 2, row = place % p.page_size;
        __nv_bfloat162 k = __floats2bfloat162_rn(0.f, 0.f), v = k;
        if (row < rows) {
            const size_t at = (base + place) * d + c;
            const float fk = power_of(p.k_exp[base + place]), fv = power_of(p.v_exp[base + place]);
            const float2 x = floats2(*reinterpret_cast<const uint16_t*>(p.k + at)), y = floats2(*reinterpret_cast<const uint16_t*>(p.v + at));
            k = __floats2bfloat162_rn(x.x * fk, x.y * fk);
            v = __floats2bfloat162_rn(y.x * fv, y.y * fv);
        }
        const size_t to = (base + place) * d + c;
        *reinterpret_cast<__nv_bfloat162*>(k_out + to) = k;
        *reinterpret_cast<__nv_bfloat162*>(v_out + to) = v;
    }
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
    gk_launch(read8_kernel, dim3(most, n_seqs), dim3(256), 0, (cudaStream_t)stream, *pages, kv_len, slots, last, (__nv_bfloat16*)k_out,
              (__nv_bfloat16*)v_out);
    GK_CHECK_LAUNCH("read8");
    return GK_OK;
}
