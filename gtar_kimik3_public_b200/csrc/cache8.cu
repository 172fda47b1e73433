// Writing keys and values into the 8-bit cache, and reading them back (what is kept: cache8.cuh).
//
// The write does the attention input stage too, as the 16-bit cache's does: per-head RMSNorm of q and k (src/layers/rmsnorm.py:11-16),
// rotation (src/layers/rope.py:17-33), order of src/layers/attention.py:82-89.  Queries are 32-bit up to the one rounding to their type, values are only
// rounded.  Keys come out as the formula in 64 bits (or, in the wide kernels, some 45) rounded once: e4m3's steps are so coarse that a number 2^-22 beside the
// middle between two of them goes wrong by a sixteenth of itself, which 32 bits do to some three in a million.  The wide kernels make a key in 32
// bits and do it over where a number or its maximum lies next to a border, one row in some fifty (7,921 tokens of 32/8 heads of 128: 52 us; with
// every key in 64 bits 114), and in 64 bits where its squares leave 32.

#include "cache8_write.cuh"

namespace {

using namespace cache8;

// ------------------------------------------------------------------ write
struct Write8 : Norm8 {
    const void* qkv;
    const int *tok_pos, *tok_seq, *slots;
    void* q_out;
    int n_tokens, n_q, n_seqs, write_kv;
};

// A row's numbers as bytes and the byte of its power; pair i of a lane at `at(i)` of the halves.
template <int N, typename At>
__device__ __forceinline__ void store_bytes(const float (&x)[N], const float (&y)[N], uint8_t* to, uint8_t* to_exp, int half, int lanes, unsigned mask, bool first,
                                            At at) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, fmaxf(finite_abs(x[i]), finite_abs(y[i])));
    for (int o = 1; o < lanes; o <<= 1) top = fmaxf(top, __shfl_xor_sync(mask, top, o));
    const int b = exponent_byte(top);
    const float back = power_back(b);
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (at(i) < half) {
            const uint32_t two = pack2(x[i] * back, y[i] * back);
            to[at(i)] = (uint8_t)two;
            to[at(i) + half] = (uint8_t)(two >> 8);
        }
    if (first) *to_exp = (uint8_t)b;
}

// The place of a token's row of kv head 0, counted in rows (the next head's is a page further), or -1.
__device__ __forceinline__ long long place_of(const GkPages8& p, const Write8& a, int seq, int pos) {
    if ((unsigned)seq >= (unsigned)a.n_seqs || pos < 0) {
        if (p.error) *p.error = ERR_PLACE;
        return -1;
    }
    const int page = page_of(p, a.slots[seq], pos / p.page_size);
    return page < 0 ? -1 : (long long)page * p.n_kv * p.page_size + pos % p.page_size;
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
    const auto at = [&](int i) { return lane + 32 * i; };
    if (is_q) {
        if (!norm_rotate(x, y, a, (const TW*)a.wq, half, pos, 32, 0xffffffffu, at)) {
            if (p.error && lane == 0) *p.error = ERR_PLACE;
            return;
        }
        T* out = (T*)a.q_out + ((size_t)t * a.n_q + head) * d;
#pragma unroll
        for (int i = 0; i < MAXP; ++i)
            if (at(i) < half) {
                out[at(i)] = from_float<T>(x[i]);
                out[at(i) + half] = from_float<T>(y[i]);
            }
        return;
    }
    long long place = place_of(p, a, a.tok_seq[t], pos);
    if (place >= 0) place += (long long)(head - a.n_q - (is_k ? 0 : p.n_kv)) * p.page_size;
    if (is_k) {
        double u[MAXP], v[MAXP];
#pragma unroll
        for (int i = 0; i < MAXP; ++i) u[i] = x[i], v[i] = y[i];
        if (!norm_rotate(u, v, a, (const TW*)a.wk, half, pos, 32, 0xffffffffu, at)) {
            if (p.error && lane == 0) *p.error = ERR_PLACE;
            return;
        }
#pragma unroll
        for (int i = 0; i < MAXP; ++i) x[i] = to_be_rounded(u[i]), y[i] = to_be_rounded(v[i]);
    }
    if (place >= 0) store_bytes(x, y, (is_k ? p.k : p.v) + place * d, (is_k ? p.k_exp : p.v_exp) + place, half, 32, 0xffffffffu, lane == 0, at);
}

// bfloat16 rows of 64 or 128: eight lanes a row, which have HD / 16 neighbouring numbers of each half of it.  A task is 4 R rows of one token (its
// queries first, then keys and values), a warp's.  Few tokens: four rows, everything asked for at once (`write8_wide_kernel`).  Many: sixteen, by
// warps that stay and have the next task's rows and rotation under way in shared memory while they make this one's (`write8_stream_kernel`).  Bound by
// memory then; through registers the same work is bound by what may be under way in L1, of which the library's shared-memory split leaves 23 KB an SM.
// A row in a lane group's registers to where it belongs: a query, a key or a value.
template <int HD, typename TW>
__device__ __forceinline__ void finish_row(const GkPages8& p, const Write8& a, float (&x)[HD / 16], float (&y)[HD / 16], const float (&w0)[HD / 16],
                                           const float (&w1)[HD / 16], const float (&c)[HD / 16], const float (&sn)[HD / 16], bool turns, bool is_v,
                                           __nv_bfloat16* q_out, const __nv_bfloat16* in, int pos, long long place, int sub, unsigned mask) {
    constexpr int E = HD / 16, HALF = HD / 2;
    if (!is_v) norm_rotate_32<HD>(a, x, y, w0, w1, c, sn, turns, mask);
    if (q_out) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t two[E / 2];
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                const __nv_bfloat162 pair = h ? __floats2bfloat162_rn(y[i], y[i + 1]) : __floats2bfloat162_rn(x[i], x[i + 1]);
                two[i / 2] = *reinterpret_cast<const uint32_t*>(&pair);
            }
            if constexpr (E == 8) *reinterpret_cast<uint4*>(q_out + sub * E + h * HALF) = make_uint4(two[0], two[1], two[E / 2 - 2], two[E / 2 - 1]);
            else *reinterpret_cast<uint2*>(q_out + sub * E + h * HALF) = make_uint2(two[0], two[1]);
        }
        return;
    }
    uint32_t four[2][E / 4];
    const int b = make_bytes<HD, TW>(a, x, y, turns, is_v, in, pos, sub, mask, four);
    uint8_t* to = (is_v ? p.v : p.k) + place * HD + sub * E;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (E == 8) *reinterpret_cast<uint2*>(to + h * HALF) = make_uint2(four[h][0], four[h][E / 4 - 1]);
        else *reinterpret_cast<uint32_t*>(to + h * HALF) = four[h][0];
    }
    if (sub == 0) (is_v ? p.v_exp : p.k_exp)[place] = (uint8_t)b;
}

// A task: which token, which rows of it.
struct Task8 {
    int t, first, n_rows;  // rows first, first + 4, ... below n_rows of the queries, or of the keys and values
    bool queries;
    const __nv_bfloat16* in;
};
template <int HD, int R>
__device__ __forceinline__ Task8 task_of(const GkPages8& p, const Write8& a, unsigned task, int q_tasks, int tasks, int lane_row) {
    Task8 k;
    // keys and values of all tokens first, then queries: a warp that stays has one kind of row, and its weights, for long
    const unsigned kv_tasks = (unsigned)(tasks - q_tasks), kv_all = kv_tasks * (unsigned)a.n_tokens;
    k.queries = task >= kv_all;
    const unsigned of = k.queries ? task - kv_all : task, each = k.queries ? (unsigned)q_tasks : kv_tasks;
    k.t = (int)(of / each);
    k.first = (int)(of - (unsigned)k.t * each) * 4 * R + lane_row;
    k.n_rows = k.queries ? a.n_q : 2 * p.n_kv;
    k.in = (const __nv_bfloat16*)a.qkv + ((size_t)k.t * (a.n_q + 2 * p.n_kv) + (k.queries ? 0 : a.n_q)) * HD;
    return k;
}

template <int HD, typename TW>
__global__ void __launch_bounds__(128) write8_wide_kernel(const GkPages8 p, const Write8 a, int q_tasks, int tasks, unsigned n_tasks) {
    constexpr int E = HD / 16, HALF = HD / 2;
    pdl_launch_dependents();
    pdl_wait();
    const int sub = threadIdx.x & 7;
    const unsigned mask = 0xffu << (threadIdx.x & 24), task = blockIdx.x * 4 + (threadIdx.x >> 5);  // the lanes of a row go one way
    if (task >= n_tasks) return;
    const Task8 k = task_of<HD, 1>(p, a, task, q_tasks, tasks, (threadIdx.x & 31) >> 3);
    if (k.first >= k.n_rows) return;
    const int pos = a.tok_pos[k.t];
    const __nv_bfloat16* in = k.in + (size_t)k.first * HD;
    float x[E], y[E], w0[E], w1[E], c[E], sn[E];
    load_run<E>(in + sub * E, x);
    load_run<E>(in + HALF + sub * E, y);
    if (a.use_norm) {
        const TW* w = (const TW*)(k.queries ? a.wq : a.wk) + sub * E;
        load_run<E>(w, w0);
        load_run<E>(w + HALF, w1);
    }
    const bool is_v = !k.queries && k.first >= p.n_kv, turns = a.cos_table != nullptr && !is_v;
    if (turns) {
        if ((unsigned)pos >= (unsigned)a.table_positions) {
            if (p.error) *p.error = ERR_PLACE;
            return;
        }
        load_run<E>(a.cos_table + (size_t)pos * HALF + sub * E, c);
        load_run<E>(a.sin_table + (size_t)pos * HALF + sub * E, sn);
    }
    long long place = 0;
    if (!k.queries) {
        place = place_of(p, a, a.tok_seq[k.t], pos);
        if (place < 0) return;
        place += (long long)(is_v ? k.first - p.n_kv : k.first) * p.page_size;
    }
    finish_row<HD, TW>(p, a, x, y, w0, w1, c, sn, turns, is_v, k.queries ? (__nv_bfloat16*)a.q_out + ((size_t)k.t * a.n_q + k.first) * HD : nullptr, in, pos, place,
                       sub, mask);
}

constexpr int STREAM_R = 4;
template <int HD>
struct Stream8 {  // a warp's two places: sixteen rows and a row of the rotation, each piece where the lane that copies it reads it
    unsigned char rows[4][2][STREAM_R][2][32][HD / 8];
    float turn[4][2][2][32][HD / 16];
};
template <int BYTES>
__device__ __forceinline__ void copy_own(void* to, const void* from) {
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
    if constexpr (BYTES == 8) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(at), "l"(from) : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < BYTES; i += 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + i), "l"((const char*)from + i) : "memory");
    }
}

template <int HD, typename TW>
__global__ void __launch_bounds__(128, 4) write8_stream_kernel(const GkPages8 p, const Write8 a, int q_tasks, int tasks, unsigned n_tasks) {
    constexpr int E = HD / 16, HALF = HD / 2;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    Stream8<HD>& sm = *reinterpret_cast<Stream8<HD>*>(smem_raw);
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & 7, lane_row = lane >> 3;
    const unsigned mask = 0xffu << (lane & 24), stride = gridDim.x * 4;
    unsigned task = blockIdx.x * 4 + warp;
    if (task >= n_tasks) return;
    const unsigned kv_tasks = (unsigned)(tasks - q_tasks), kv_all = kv_tasks * (unsigned)a.n_tokens;
    const auto token = [&](unsigned k) { return k < kv_all ? k / kv_tasks : (k - kv_all) / (unsigned)q_tasks; };
    const auto position = [&](unsigned k) { return k < n_tasks ? a.tok_pos[token(k)] : 0; };
    // where a token's keys and values go takes three loads one behind another: each is asked for a task ahead of the next
    const auto sequence = [&](unsigned k) { return k < kv_all ? a.tok_seq[token(k)] : -1; };
    const auto slot_in = [&](int seq) { return (unsigned)seq < (unsigned)a.n_seqs ? a.slots[seq] : -1; };
    const auto page_in = [&](int slot, int pos) {
        const unsigned index = (unsigned)pos / (unsigned)p.page_size;
        return (unsigned)slot < (unsigned)p.n_slots && pos >= 0 && index < (unsigned)p.max_pages ? p.table[(size_t)slot * p.max_pages + index] : -1;
    };
    const auto ask = [&](unsigned which, int pos, int to) {
        if (which < n_tasks) {
            const Task8 k = task_of<HD, STREAM_R>(p, a, which, q_tasks, tasks, lane_row);
#pragma unroll
            for (int j = 0; j < STREAM_R; ++j) {
                const __nv_bfloat16* row = k.in + (size_t)min(k.first + 4 * j, k.n_rows - 1) * HD + sub * E;
                copy_own<HD / 8>(sm.rows[warp][to][j][0][lane], row);
                copy_own<HD / 8>(sm.rows[warp][to][j][1][lane], row + HALF);
            }
            if (a.cos_table && (unsigned)pos < (unsigned)a.table_positions) {
                copy_own<HD / 4>(sm.turn[warp][to][0][lane], a.cos_table + (size_t)pos * HALF + sub * E);
                copy_own<HD / 4>(sm.turn[warp][to][1][lane], a.sin_table + (size_t)pos * HALF + sub * E);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int pos = position(task), pos_next = position(task + stride), seq_2 = sequence(task + 2 * stride);
    int slot_next = slot_in(sequence(task + stride)), page = page_in(slot_in(sequence(task)), pos);
    ask(task, pos, 0);
    float w0[E], w1[E];
    bool weights_of_queries = false, weights = false;
    for (int in_hand = 0; task < n_tasks; task += stride, in_hand ^= 1) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");  // a lane reads only what it has copied itself
        ask(task + stride, pos_next, in_hand ^ 1);
        const int pos_here = pos, page_here = page;
        page = page_in(slot_next, pos_next);
        slot_next = slot_in(seq_2);
        seq_2 = sequence(task + 3 * stride);
        pos = pos_next;
        pos_next = position(task + 2 * stride);
        const Task8 k = task_of<HD, STREAM_R>(p, a, task, q_tasks, tasks, lane_row);
        const bool turns = a.cos_table != nullptr, known = !turns || (unsigned)pos_here < (unsigned)a.table_positions;
        const bool placed = k.queries || (unsigned long long)(long long)page_here < (unsigned long long)p.n_pages;
        if (!(known && placed) && p.error) *p.error = ERR_PLACE;
        if (!placed) continue;
        const long long place0 = k.queries ? 0 : (long long)page_here * p.n_kv * p.page_size + pos_here % p.page_size;
        float c[E], sn[E];
        if (a.use_norm && (!weights || weights_of_queries != k.queries)) {
            const TW* w = (const TW*)(k.queries ? a.wq : a.wk) + sub * E;
            load_run<E>(w, w0);
            load_run<E>(w + HALF, w1);
            weights = true;
            weights_of_queries = k.queries;
        }
        if (turns) {
            load_run<E>(sm.turn[warp][in_hand][0][lane], c);
            load_run<E>(sm.turn[warp][in_hand][1][lane], sn);
        }
#pragma unroll 1
        for (int j = 0; j < STREAM_R; ++j) {
            const int row = k.first + 4 * j;
            const bool is_v = !k.queries && row >= p.n_kv;
            if (row >= k.n_rows || (!is_v && !known)) continue;
            float x[E], y[E];
            load_run<E>(reinterpret_cast<const __nv_bfloat16*>(sm.rows[warp][in_hand][j][0][lane]), x);
            load_run<E>(reinterpret_cast<const __nv_bfloat16*>(sm.rows[warp][in_hand][j][1][lane]), y);
            finish_row<HD, TW>(p, a, x, y, w0, w1, c, sn, turns && !is_v, is_v, k.queries ? (__nv_bfloat16*)a.q_out + ((size_t)k.t * a.n_q + row) * HD : nullptr,
                               k.in + (size_t)row * HD, pos_here, place0 + (long long)(is_v ? row - p.n_kv : row) * p.page_size, sub, mask);
        }
    }
}

template <int HD, typename TW>
int launch_write8(const GkPages8& p, const Write8& a, cudaStream_t stream) {
    // Warps that stay have a ring to fill first.  us, four rows a warp / warps that stay: 16,384 rows of 128 7.4 / 9.7, 49,152 11.7 / 13.3, 65,536 15.6 / 14.8,
    // 196,608 40 / 31; 40,960 rows of 64 8.5 / 9.0, 81,920 13.1 / 14.4.
    const bool many = (long long)a.n_tokens * (a.n_q + 2 * p.n_kv) * HD >= 7 << 20;
    const int per = many ? 4 * STREAM_R : 4, q_tasks = (a.n_q + per - 1) / per, tasks = q_tasks + (a.write_kv ? (2 * p.n_kv + per - 1) / per : 0);
    const long long n_tasks = (long long)a.n_tokens * tasks, blocks = (n_tasks + 3) / 4;
    GK_REQUIRE(n_tasks + 148 * 4 * 4 * 3 < 4294967295LL, "write8: too many tokens");
    if (!many) {
        gk_launch(write8_wide_kernel<HD, TW>, dim3((unsigned)blocks), dim3(128), 0, stream, p, a, q_tasks, tasks, (unsigned)n_tasks);
        GK_CHECK_LAUNCH("write8");
        return GK_OK;
    }
    const int smem = (int)sizeof(Stream8<HD>);
    cudaError_t err = cudaFuncSetAttribute(write8_stream_kernel<HD, TW>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (err != cudaSuccess) return gk_fail(GK_CUDA_ERROR, "write8: %s", cudaGetErrorString(err));
    gk_launch(write8_stream_kernel<HD, TW>, dim3((unsigned)(blocks < 148 * 4 ? blocks : 148 * 4)), dim3(128), smem, stream, p, a, q_tasks, tasks, (unsigned)n_tasks);
    GK_CHECK_LAUNCH("write8");
    return GK_OK;
}

// ------------------------------------------------------------------ read back
// For attention over what was read: pages renumbered under a table, lengths, slots and starts of their own, so that no number that cannot be reaches it; and
// a row of values that holds a NaN becomes zeros with a NaN key, which a token that does not see it cannot meet (0 * NaN).
struct Clean8 {
    int *table, *kv_len, *slots, *cu_q;  // [n_seqs][per], [n_seqs], [n_seqs], [n_seqs + 1]
    const int* cu_q_in;
    int n_tokens, per, own_numbers;  // pages a sequence; whether a page keeps its number or is seq * per + index
    int max_q_len, window;           // what the attention is launched for: tokens a sequence at most, keys a token sees (0: all)
    __nv_bfloat16* out;              // [n_tokens][row]: its result; zeros here for tokens in front of their sequence's first position
    int row;
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
    const auto length_here = [&](int given) {
        int len = length_of(p, given);
        if (CLEAN && len > (long long)clean.per * p.page_size) {
            if (p.error) *p.error = ERR_PLACE;
            len = clean.per * p.page_size;
        }
        return len;
    };
    const int len = length_here(kv_len[seq]);
    if (CLEAN && seq == 0 && index == 0 && hk == 0 && threadIdx.x < 32) {  // starts within the queries, none before the one in front
        int before = 0;
        for (int base = 0; base <= (int)gridDim.y; base += 32) {
            const int i = base + threadIdx.x, given = i <= (int)gridDim.y ? clean.cu_q_in[i] : 0;
            int at = max(before, min(max(given, 0), clean.n_tokens));
#pragma unroll
            for (int w = 1; w < 32; w <<= 1) {
                const int other = __shfl_up_sync(0xffffffffu, at, w);
                if ((int)threadIdx.x >= w) at = max(at, other);
            }
            if (i <= (int)gridDim.y) {
                clean.cu_q[i] = at;
                if (at != given && p.error) *p.error = ERR_PLACE;
            }
            // A sequence with more tokens than the attention is launched for: the rest of them is left out.  With more tokens than positions: its first tokens would stand in front of position 0.  They see no key and get zeros here;
            // the prefill kernels pass over a tile of none but such.
            int first = __shfl_up_sync(0xffffffffu, at, 1), blind = 0;
            if (threadIdx.x == 0) first = before;
            if (i > 0 && i <= (int)gridDim.y) blind = max(0, at - first - length_here(kv_len[i - 1]));
            if ((blind > 0 || (i > 0 && at - first > clean.max_q_len)) && p.error) *p.error = ERR_PLACE;
            for (unsigned left = __ballot_sync(0xffffffffu, blind > 0); left; left &= left - 1) {
                const int who = __ffs(left) - 1;
                const size_t from = (size_t)__shfl_sync(0xffffffffu, first, who) * clean.row, n = (size_t)__shfl_sync(0xffffffffu, blind, who) * clean.row;
                for (size_t c = threadIdx.x; c < n; c += 32) clean.out[from + c] = __float2bfloat16_rn(0.f);
            }
            before = __shfl_sync(0xffffffffu, at, 31);
        }
    }
    long long back = last;  // how many of the sequence's last positions are wanted (0: all)
    if (CLEAN && clean.window > 0) {  // those that its first token sees, itself among them, and on; starts that are put in order make no sequence longer
        const int from = max(clean.cu_q_in[seq], 0), to = min(clean.cu_q_in[seq + 1], clean.n_tokens);
        back = max((long long)clean.window + max(0, to - from) - 1, 1LL);
    }
    const bool seen = (long long)index * p.page_size < len && (back <= 0 || (index + 1) * (long long)p.page_size > (long long)len - back);
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
    // Under its own number a page may be another, longer sequence's too: what lies behind this one's end is made as that one makes it, where there is
    // a power that the write makes.  (The prefill kernels set hidden keys' scores aside, and hidden values are finite.)
    const bool all = CLEAN && clean.own_numbers;
    const auto kept = [](int b) { return (unsigned)(b - 127 - LOW) <= (unsigned)(HIGH - LOW); };
    const size_t from = ((size_t)max(page, 0) * p.n_kv + hk) * p.page_size, to = ((size_t)to_page * p.n_kv + hk) * p.page_size;
    if constexpr (HD > 0) {
        constexpr int LANES = HD / 16;
        const int c = threadIdx.x % LANES * 16;
        for (int row = threadIdx.x / LANES; row < p.page_size; row += 256 / LANES) {
            uint32_t k[8] = {0, 0, 0, 0, 0, 0, 0, 0}, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (row < rows || (all && kept(p.k_exp[from + row]) && kept(p.v_exp[from + row]))) {
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
    const Write8 a = {{wq, wk, cos_table, sin_table, table_positions, use_norm, eps}, qkv, tok_pos, tok_seq, slots, q_out, n_tokens, n_q, n_seqs, write_kv};
    const long long items = (long long)n_tokens * (n_q + 2 * pages->n_kv), blocks = (items + 3) / 4;
    GK_REQUIRE(blocks < 2147483647LL, "write8: too many tokens");
    if (dtype == GK_BF16 && (pages->head_dim == 64 || pages->head_dim == 128) && (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)wq | (uintptr_t)wk |
                                                                                  (uintptr_t)cos_table | (uintptr_t)sin_table) & 15) == 0) {
        GK_DISPATCH_DTYPE(weight_dtype, TW, {
            return pages->head_dim == 64 ? launch_write8<64, TW>(*pages, a, (cudaStream_t)stream) : launch_write8<128, TW>(*pages, a, (cudaStream_t)stream);
        })
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
// [n_seqs][per], `len_out` and `slots_out` [n_seqs] and `cu_out` [n_seqs + 1] to go with them.  Heads of 64 or 128.  `window`: pages
// that no token sees are left out (0: none are).  `out` [n_tokens][n_q][head_dim], where the attention's result will be: a sequence's first tokens, where
// it brings more than it has positions, get zeros.  That is reported, and so are more tokens than `max_q_len`.
GK_EXPORT int gk_clean8(const GkPages8* pages, const int* cu_q, const int* kv_len, const int* slots, int n_tokens, int n_seqs, int n_q, int per,
                        int own_numbers, int max_q_len, int window, void* k_out, void* v_out, void* out, int* table, int* len_out, int* slots_out, int* cu_out,
                        void* stream) {
    const int status = cache8::check(pages, "clean8");
    if (status != GK_OK) return status;
    GK_REQUIRE(n_seqs >= 0 && n_seqs <= 65535 && n_q > 0 && per > 0 && max_q_len >= 0 && window >= 0 && (long long)n_seqs * per < 2147483647LL,
               "clean8: bad sizes n_seqs=%d n_q=%d per=%d max_q_len=%d window=%d", n_seqs, n_q, per, max_q_len, window);
    if (n_seqs == 0) return GK_OK;
    GK_REQUIRE(cu_q && kv_len && slots && k_out && v_out && out && table && len_out && slots_out && cu_out, "clean8: an array is missing");
    const Clean8 clean = {table, len_out, slots_out, cu_out, cu_q, n_tokens, per, own_numbers, max_q_len, window, (__nv_bfloat16*)out, n_q * pages->head_dim};
    return launch_read8<true>(*pages, kv_len, slots, n_seqs, per, 0, k_out, v_out, clean, (cudaStream_t)stream);
}
