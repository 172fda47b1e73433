// Causal grouped-query attention over the 8-bit cache (what is kept: cache8.cuh).
//
// For a token at position pos of its sequence, query head hq, kv head hk = hq / (n_q / n_kv), visible keys j <= pos (and j > pos - window
// where a window is set; src/layers/attention.py:116-119, src/ops/flash_attention_2.py:33-34):
//   s_j = scale * (q . k8_j) * 2^ek_j        o = sum_j exp(s_j - m) 2^ev_j v8_j / sum_j exp(s_j - m),   m = max_j s_j
// With `sink` one more term in the denominator: a key of score 0 without a value.  A token that sees no key gets zeros (one in front of position 0, of a
// sequence that brings more tokens than it has positions, is reported as well).  Keys that are not visible are not looked at, whatever their places hold.

#include "cache8.cuh"

namespace {

using namespace cache8;

struct Attend8 {
    const void* q;
    void* out;
    const int *cu_q, *kv_len, *slots;  // cu_q null: one token a sequence
    int n_tokens, n_seqs, n_q;
    float sl2;  // scale * log2(e)
    int window, sink;
};

// The sequence that token t belongs to, -1 behind the last one.
__device__ __forceinline__ int sequence_of(const int* cu_q, int n_seqs, int t) {
    if (t >= cu_q[n_seqs] || t < cu_q[0]) return -1;
    int lo = 0, hi = n_seqs;  // cu_q[lo] <= t < cu_q[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu_q[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Any even head size up to 512, any group, either type of q: a warp a (token, head), a key a lane for the scores and a column a lane
// for the values.
template <typename T>
__global__ void __launch_bounds__(128) attend8_rows_kernel(const GkPages8 p, const Attend8 a) {
    constexpr int MAX_ACC = 16;
    extern __shared__ float q_all[];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = p.head_dim;
    const long long item = (long long)blockIdx.x * 4 + warp;
    if (item >= (long long)a.n_tokens * a.n_q) return;
    const int t = (int)(item / a.n_q), hq = (int)(item - (long long)t * a.n_q), hk = hq / (a.n_q / p.n_kv);
    int seq = t, pos;
    if (a.cu_q) {
        seq = sequence_of(a.cu_q, a.n_seqs, t);
        if (seq < 0) return;
        pos = length_of(p, a.kv_len[seq]) - a.cu_q[seq + 1] + t;
        if (pos < 0 && p.error) *p.error = ERR_PLACE;  // more tokens than positions
    } else {
        pos = length_of(p, a.kv_len[seq]) - 1;
    }
    const int slot = a.slots[seq];
    float* q = q_all + warp * d;
    const T* row = (const T*)a.q + ((size_t)t * a.n_q + hq) * d;
    for (int c = lane; c < d; c += 32) q[c] = to_float(row[c]);
    __syncwarp();
    float m = -INFINITY, l = 0.f, acc[MAX_ACC];
#pragma unroll
    for (int i = 0; i < MAX_ACC; ++i) acc[i] = 0.f;
    const int lo = a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0;  // (the difference alone could leave 32 bits)
    for (int j0 = lo & ~31; j0 <= pos; j0 += 32) {  // a page is whole blocks of 32 keys
        const int page = page_of(p, slot, j0 / p.page_size), j = j0 + lane;
        if (page < 0) continue;  // its keys count as not visible
        const size_t place = ((size_t)page * p.n_kv + hk) * p.page_size + j0 % p.page_size;
        const bool visible = j >= lo && j <= pos;
        float s = -INFINITY, fv = 0.f;
        if (visible) {
            const uint16_t* k = reinterpret_cast<const uint16_t*>(p.k + (place + lane) * d);
            float dot = 0.f;
            for (int c = 0; c < d; c += 2) {
                const float2 x = floats2(k[c >> 1]);
                dot = fmaf(q[c], x.x, dot);
                dot = fmaf(q[c + 1], x.y, dot);
            }
            s = dot * a.sl2 * power_of(p.k_exp[place + lane]);
            fv = power_of(p.v_exp[place + lane]);
        }
        const float m_new = fmaxf(m, warp_max(s)), ref = m_new == -INFINITY ? 0.f : m_new;
        const float e = visible ? exp2f(s - ref) : 0.f, corr = m == ref ? 1.f : exp2f(m - ref);
        l = l * corr + warp_sum(e);
        m = m_new;
#pragma unroll
        for (int i = 0; i < MAX_ACC; ++i) acc[i] *= corr;
        for (int r = max(0, lo - j0); r <= min(31, pos - j0); ++r) {
            const float w = __shfl_sync(0xffffffffu, e, r), f = __shfl_sync(0xffffffffu, fv, r);
            const uint8_t* v = p.v + (place + r) * d;
#pragma unroll
            for (int i = 0; i < MAX_ACC; ++i) {
                const int c = lane + 32 * i;
                if (c < d) acc[i] = fmaf(w, floats2(v[c]).x * f, acc[i]);
            }
        }
    }
    if (a.sink) {
        const float top = fmaxf(m, 0.f), corr = m == -INFINITY ? 0.f : exp2f(m - top);
        l = l * corr + exp2f(-top);
#pragma unroll
        for (int i = 0; i < MAX_ACC; ++i) acc[i] *= corr;
    }
    T* out = (T*)a.out + ((size_t)t * a.n_q + hq) * d;
#pragma unroll
    for (int i = 0; i < MAX_ACC; ++i) {
        const int c = lane + 32 * i;
        if (c < d) out[c] = from_float<T>(l == 0.f ? 0.f : acc[i] / l);
    }
}

}  // namespace

// `q`, `out` [n_tokens][n_q][head_dim] float32 or bfloat16.  With `cu_q` [n_seqs + 1] sequence i owns the tokens cu_q[i] .. cu_q[i + 1] - 1, its
// last positions; without it one token a sequence.  kv_len counts a sequence's cached positions, the step's included.
GK_EXPORT int gk_attend8(const GkPages8* pages, const void* q, int dtype, void* out, const int* cu_q, const int* kv_len, const int* slots, int n_tokens,
                         int n_seqs, int n_q, float scale, int window, int sink, void* stream) {
    const int status = cache8::check(pages, "attend8");
    if (status != GK_OK) return status;
    GK_REQUIRE(GK_VALID_DTYPE(dtype), "attend8: bad dtype code");
    GK_REQUIRE(n_tokens >= 0 && n_seqs >= 0 && n_q > 0 && n_q % pages->n_kv == 0, "attend8: bad sizes n_tokens=%d n_seqs=%d heads %d/%d", n_tokens, n_seqs,
               n_q, pages->n_kv);
    GK_REQUIRE(cu_q || n_tokens == n_seqs, "attend8: without cu_q every sequence has one token");
    GK_REQUIRE(window >= 0, "attend8: window must be >= 0");
    if (n_tokens == 0 || n_seqs == 0) return GK_OK;
    GK_REQUIRE(q && out && kv_len && slots, "attend8: an array is missing");
    const Attend8 a = {q, out, cu_q, kv_len, slots, n_tokens, n_seqs, n_q, scale * 1.4426950408889634f, window, sink};
    const long long blocks = ((long long)n_tokens * n_q + 3) / 4;
    GK_REQUIRE(blocks < 2147483647LL, "attend8: too many tokens");
    GK_DISPATCH_DTYPE(dtype, T, {
        gk_launch(attend8_rows_kernel<T>, dim3((unsigned)blocks), dim3(128), (size_t)4 * pages->head_dim * sizeof(float), (cudaStream_t)stream, *pages, a);
    })
    GK_CHECK_LAUNCH("attend8");
    return GK_OK;
}
