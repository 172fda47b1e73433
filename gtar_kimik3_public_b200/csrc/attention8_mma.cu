// Attention of few rows over the 8-bit cache on the tensor cores: one new token per sequence, or a few (what is kept: cache8.cuh; formulas:
// attention8.cu).  bfloat16, heads of 64 or 128, pages of 64 positions.
//
// A row is a (token, query head of the kv head); up to 8 NT rows of a (sequence, kv head) are taken together, so that every key and value is
// read once for all of them.  Both products are turned over, so that the rows are the eight columns of m16n8k16:
//     S^T (16 keys x rows) = K8 Q^T          O^T (d x rows) += V8^T P^T
// with e4m3 numbers as halves (exact), the queries as halves under a power of two of their row's own (bfloat16 ones exact but for numbers of 2^-28 of the
// row's largest and less; those that the decode kernel has normed and rotated itself, in 32 bits, rounded by up to 2^-11 of each number, an eighth of what
// bfloat16 would cost them) and probabilities rounded to halves; sums are 32-bit.  A key's power of two multiplies its score, a value's goes into its
// probability.  So there are two running references a row:
//     l  = sum_j 2^(s_j - A)               A near the largest s_j           (s in powers of two)
//     o8 = sum_j 2^(s_j + ev_j - B) v8_j   B near the largest s_j + ev_j    out = o8 2^(B - A) / l
// A and B are moved only when a number would pass 2^14 or 2^15 (halves end at 65,504): after a sequence's first keys hardly ever, and then no lane
// has to ask the others for a maximum.  B is set 7 below the largest, so that probabilities keep all their bits down to 2^-21 of it.  Where a tile's
// values are more than 2^9 smaller than those that B goes by (a column in which the large ones have nothing would show what is lost), what the halves of
// probabilities above 2^-32 leave over is added by itself.  (To look for such tiles, none of which random keys and values have, costs 64 sequences of
// 1,024 to 8,192 tokens 0.4 of 101 us, one of 131,072 tokens 1.6 of 55, sixteen times four tokens 0.9 of 27.)
//
// The contraction over d may take d in any order that both operands share, and the keys of a product any order that P and V share: lane (g, t) =
// (lane / 4, lane % 4) reads sixteen bytes in one piece of the keys 4g .. 4g + 3, and of the values 8t .. 8t + 7 its own sixteen (or eight) columns,
// which the products then take byte by byte: no number but the probabilities is moved between lanes.  Every warp has a ring of its own in shared
// memory, 32 keys and values (8 KB) a place, filled with 16-byte asynchronous copies: there is no barrier of the block in the loop.
//
// Bound by memory, 129 bytes a key and as many a value, and next to that by the conversions to halves (two cycles of the integer pipe for two
// numbers, and two more to bring the upper two of a word down: 224 of some 300 such cycles for 16 keys).  Tried and taken back, 64 sequences of 1,024
// to 8,192 tokens with 32/8 heads (93 us for the bytes): loads straight into registers (163 us: what is under way has to fit into L1, of which the
// library's split leaves 23 KB an SM); scores by products of e4m3 numbers with the query as the sum of two of them (117 against 116: sm_100a makes
// halves of them under the hood); the scores of the next keys under the exponentials of these (116, no gain).

#include <atomic>

#include "cache8_write.cuh"

namespace {

using namespace cache8;

constexpr int WARPS = 4, THREADS = WARPS * 32, KEYS = 32, PAGE = 64, PER_PAGE = PAGE / KEYS;
constexpr float NONE = -3e38f;  // a reference before the first visible key

struct Rows8 {
    const __nv_bfloat16* q;
    __nv_bfloat16* out;
    const int *cu_q, *kv_len, *slots;  // cu_q null: one token a sequence
    int n_tokens, max_q_len, n_q, group, tiles, n_units;  // tiles: row tiles a sequence at most; a unit is a row tile of a sequence
    float sl2;                         // scale * log2(e)
    int window, sink;
    int n_splits;  // blocks of a cluster that share a (unit, kv head); 0: pieces of one size, about `pieces` of them
    int pieces;
    float *part_o, *part_abl;  // of pieces: [piece][row][D] and [piece][row][A, B, l]
};

// A step of one token a sequence that does its input stage too: `qkv` [n_seqs][(n_q + 2 n_kv) * D] is the packed projection; queries are normed and
// rotated here, and (`write_kv`) the new key and value put into the cache, by the warp that has the tile they lie in: it also puts their bytes into that
// tile's copy in shared memory, which is asked for without them.
struct Fused8 : Norm8 {
    const __nv_bfloat16* qkv;
    int weights_bf16, write_kv;
};

// A unit: which rows, which tokens, and the keys that some or all of them see.
struct Unit {
    int seq, row_first, n_rows, first_token, past, slot, pos_low, begin, end, all_begin, tile_0, n_tiles;
    bool sound;  // the sequence's length is one that the pages can hold
};
__device__ __forceinline__ Unit unit_of(const GkPages8& p, const Rows8& a, int unit, int most_rows) {
    Unit u;
    u.seq = a.cu_q ? unit / a.tiles : unit;
    u.row_first = a.cu_q ? (unit - u.seq * a.tiles) * most_rows : 0;
    // lengths, slots and the table are inputs of the step: they may be read while the kernel in front still runs
    const int given = a.kv_len[u.seq], len = length_of(p, given);
    u.sound = given == len;
    u.slot = a.slots[u.seq];
    u.first_token = a.cu_q ? a.cu_q[u.seq] : u.seq;
    int q_len = a.cu_q ? a.cu_q[u.seq + 1] - u.first_token : 1;
    if (a.cu_q) {  // tokens that there are none of, or more than the launch was made for: left out and recorded
        const int most = u.first_token < 0 ? 0 : min(a.n_tokens - u.first_token, a.max_q_len);
        if (q_len < 0 || q_len > most) {
            if (p.error) *p.error = ERR_PLACE;
            q_len = max(0, min(q_len, most));
        }
        if (q_len > len && p.error) *p.error = ERR_PLACE;  // the first of them stand in front of position 0: they see no key
    }
    u.n_rows = min(most_rows, q_len * a.group - u.row_first);
    u.past = len - q_len;
    u.pos_low = u.past + u.row_first / a.group;  // of the first row
    const int pos_high = u.past + (u.row_first + u.n_rows - 1) / a.group;
    // (compared first: a position in front of 0 less the largest window would leave 32 bits)
    u.begin = a.window > 0 && u.pos_low >= a.window ? u.pos_low - a.window + 1 : 0;
    u.end = max(u.begin, pos_high + 1);
    u.all_begin = a.window > 0 && pos_high >= a.window ? pos_high - a.window + 1 : 0;  // keys all_begin .. pos_low are seen by every row
    u.tile_0 = u.begin / KEYS;
    u.n_tiles = u.n_rows > 0 ? (u.end + KEYS - 1) / KEYS - u.tile_0 : 0;
    return u;
}

// Pieces: a (unit, kv head) of n tiles is cut into ceil(n / size) pieces, a block each; the pieces stand in one line, unit after unit, kv head after
// kv head.  The size is the step's tiles over the pieces that are wanted, so a step of any lengths makes at most `pieces` and one a pair.
__device__ __forceinline__ int piece_size(const GkPages8& p, const Rows8& a, int most_rows, int lane) {
    long long sum = 0;
    for (int base = 0; base < a.n_units; base += 32)
        sum += __reduce_add_sync(0xffffffffu, base + lane < a.n_units ? unit_of(p, a, base + lane, most_rows).n_tiles : 0);
    return (int)max((sum * p.n_kv + a.pieces - 1) / a.pieces, (long long)WARPS);
}
// The unit that holds the line's place `at` (n_units: none), or, with `of`, the unit `of`; `before`: the pieces in front of it.
__device__ __forceinline__ int unit_at(const GkPages8& p, const Rows8& a, int size, int at, int of, int most_rows, int lane, int& before) {
    int sum = 0;
    for (int base = 0; base < a.n_units; base += 32) {
        const int mine = base + lane < a.n_units ? (unit_of(p, a, base + lane, most_rows).n_tiles + size - 1) / size * p.n_kv : 0;
        int through = mine;
#pragma unroll
        for (int w = 1; w < 32; w <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, through, w);
            if (lane >= w) through += other;
        }
        const unsigned found = __ballot_sync(0xffffffffu, of >= 0 ? base + lane == of : sum + through > at);
        if (found) {
            const int who = __ffs(found) - 1;
            before = sum + __shfl_sync(0xffffffffu, through - mine, who);
            return base + who;
        }
        sum += __shfl_sync(0xffffffffu, through, 31);
    }
    before = sum;
    return a.n_units;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turned(uint32_t x) {  // an 8 x 8 matrix of halves, rows for columns
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t low_bf16(uint32_t four) {  // (exact)
    const float2 two = floats2((uint16_t)four);
    return pack_bf16(two.x, two.y);
}
__device__ __forceinline__ uint32_t low_halves(uint32_t four) { return halves2((uint16_t)four); }
__device__ __forceinline__ uint32_t high_halves(uint32_t four) { return halves2((uint16_t)(four >> 16)); }

// ------------------------------------------------------------------ 32 keys and values in shared memory
// [K 32 x D][V 32 x D][K's powers][V's powers]; 16-byte pieces change places with their neighbours so that the lanes that read together (keys 8m + i
// and 8m + 4 + i; values i, 8 + i, 16 + i and 24 + i) meet different banks.
template <int D>
struct Place {
    static constexpr int V = KEYS * D, KE = 2 * KEYS * D, VE = KE + KEYS, BYTES = VE + KEYS;
    __device__ static int key(int row, int byte) { return (row * D + byte) ^ ((row >> 2 & 1) << 6); }
    __device__ static int value(int row, int byte) { return V + ((row * D + byte) ^ ((row >> 3 & 3) << 5)); }
};

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

// Asks for the keys key0 .. key0 + 31, which begin at row0 of a page (-1: there is none).  Nothing of a place outside begin .. end - 1 is looked
// at: zeros come instead.
template <int D>
__device__ __forceinline__ void ask(uint32_t place, const GkPages8& p, int hk, int page, int row0, int key0, int begin, int end, int lane) {
    constexpr int PASSES = KEYS * D / 512, ROWS_A_PASS = 512 / D;
    const size_t from = (size_t)(unsigned)max(page, 0) * (unsigned)(p.n_kv * PAGE) + (unsigned)(hk * PAGE + row0);
    const uint8_t *k = p.k + from * D + lane * 16, *v = p.v + from * D + lane * 16;
    const int r = lane * 16 / D, byte = lane * 16 % D;
    if (page >= 0 && key0 >= begin && key0 + KEYS <= end) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            copy16(place + Place<D>::key(r + i * ROWS_A_PASS, byte), k + i * 512);
            copy16(place + Place<D>::value(r + i * ROWS_A_PASS, byte), v + i * 512);
        }
    } else {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int key = key0 + r + i * ROWS_A_PASS;
            const bool there = page >= 0 && key >= begin && key < end;
            copy16(place + Place<D>::key(r + i * ROWS_A_PASS, byte), there ? k + i * 512 : p.k, there);
            copy16(place + Place<D>::value(r + i * ROWS_A_PASS, byte), there ? v + i * 512 : p.v, there);
        }
    }
    // (the powers of hidden places come along: their scores are set aside before anything is made of them)
    if (lane < 4) copy16(place + Place<D>::KE + lane * 16, (lane < 2 ? p.k_exp : p.v_exp) + from + (lane & 1) * 16);
}

template <int W>
__device__ __forceinline__ void read_words(uint32_t (&r)[W], uint32_t from) {
    if constexpr (W == 4)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(from) : "memory");
    else
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(from) : "memory");
}
__device__ __forceinline__ uint32_t read_word(uint32_t from) {
    uint32_t r;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(from) : "memory");
    return r;
}

template <int D, int NT>
struct Smem8 {
    static constexpr int ROWS = 8 * NT, STRIDE = D + 4;
    union {
        unsigned char ring[WARPS][2][Place<D>::BYTES];
        float o[WARPS][ROWS * STRIDE];  // what a warp has of its rows, in the end
    };
    float abl[WARPS][ROWS][3];
    unsigned char fresh[2][D], fresh_power[2];  // bytes of the new key and value
    alignas(16) float from_o[ROWS * D + 8 * 4];  // from the other blocks of a cluster: [block][place] of four numbers
    float from_abl[8][ROWS][3];
};

// What the sums over visible keys make of a row: the factor of o8.  A row that sees nothing gets zeros.
__device__ __forceinline__ float factor_of(float A, float B, float sum, int sink) {
    if (sink) {
        const float top = fmaxf(A, 0.f);
        sum = sum * exp2_fast(A - top) + exp2_fast(-top);
        A = top;
    }
    return sum == 0.f ? 0.f : exp2_fast(B - A) / sum;
}
__device__ __forceinline__ __nv_bfloat16* out_row(const Rows8& a, const Unit& u, int hk, int r, int d) {
    const int row = u.row_first + r;
    return a.out + ((size_t)(u.first_token + row / a.group) * a.n_q + hk * a.group + row % a.group) * d;
}
__device__ __forceinline__ void store4(__nv_bfloat16* to, const float4& v, float f) {
    __nv_bfloat162 two[2] = {__floats2bfloat162_rn(v.x * f, v.y * f), __floats2bfloat162_rn(v.z * f, v.w * f)};
    *reinterpret_cast<uint2*>(to) = *reinterpret_cast<uint2*>(two);
}

// RMSNorm and rotation of a query whose columns 64 c + 16 t .. + 15 lane t of a quad holds.
template <int D>
__device__ __forceinline__ void norm_rotate_queries(const Fused8& f, float (&x)[D / 64][16], int pos, int t) {
    if (f.use_norm) {
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) ss += x[c][i] * x[c][i];
        ss += __shfl_xor_sync(0xffffffffu, ss, 1);
        ss += __shfl_xor_sync(0xffffffffu, ss, 2);
        const float inv = rsqrtf(fmaf(ss, 1.f / D, f.eps));
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int i = 0; i < 16; i += 8) {
                float w[8];
                if (f.weights_bf16) load_run<8>((const __nv_bfloat16*)f.wq + 64 * c + 16 * t + i, w);
                else load_run<8>((const float*)f.wq + 64 * c + 16 * t + i, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[c][i + e] = (x[c][i + e] * inv) * w[e];
            }
    }
    if (f.cos_table && (unsigned)pos < (unsigned)f.table_positions) {
        const size_t at = (size_t)pos * (D / 2) + (D == 128 ? 16 * t : 16 * (t & 1));
#pragma unroll
        for (int i = 0; i < 16; i += 8) {
            float c[8], s[8];
            load_run<8>(f.cos_table + at + i, c);
            load_run<8>(f.sin_table + at + i, s);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (D == 128) {
                    const float u = x[0][i + e], v = x[D / 64 - 1][i + e];
                    x[0][i + e] = u * c[e] - v * s[e];
                    x[D / 64 - 1][i + e] = v * c[e] + u * s[e];
                } else {  // the other half lies with lane t ^ 2
                    const float u = x[0][i + e], v = __shfl_xor_sync(0xffffffffu, u, 2);
                    x[0][i + e] = t < 2 ? u * c[e] - v * s[e] : u * c[e] + v * s[e];
                }
            }
        }
    }
}

// The new key and value of a sequence, a warp's work, D / 64 numbers of each half a lane.  Always the careful way: two numbers a lane take less long than
// code that is run for one key in fifty takes to be fetched (one kernel of 64 such keys: 3 us).
template <int D, typename TW>
__device__ __forceinline__ void new_rows(const GkPages8& p, const Rows8& a, const Fused8& f, const Unit& u, int hk, int lane, unsigned char (&bytes)[2][D],
                                         unsigned char (&powers)[2]) {
    constexpr int E = D / 64, HALF = D / 2;
    const int pos = u.past;
    const __nv_bfloat16* row = f.qkv + ((size_t)u.first_token * (a.n_q + 2 * p.n_kv) + a.n_q + hk) * D;
    const bool known = f.cos_table == nullptr || (unsigned)pos < (unsigned)f.table_positions;  // without a rotation the key stays out of the cache
    if (!known && p.error) *p.error = ERR_PLACE;
    float x[2][2][E];
    int b[2];
#pragma unroll
    for (int v = 0; v < 2; ++v) b[v] = careful_row<D, 32, TW>(f, row + (size_t)v * p.n_kv * D, v == 1, pos, lane, 0xffffffffu, x[v]);
    const bool far = b[0] >= FAR_ROW;
    if (far) b[0] -= FAR_ROW;
    const int page = page_of(p, u.slot, pos / PAGE);
    const size_t place = ((size_t)max(page, 0) * p.n_kv + hk) * PAGE + pos % PAGE;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const float back = power_back(b[v]);
        uint8_t* to = (v ? p.v : p.k) + place * D;
        const bool kept = page >= 0 && (v || known);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = h * HALF + lane * E;
            uint32_t two = pack2(x[v][h][0] * back, x[v][h][E - 1] * back);
            if (v == 0 && far) two = far_pair(two);
            if constexpr (E == 2) {
                *reinterpret_cast<uint16_t*>(&bytes[v][at]) = (uint16_t)two;
                if (kept) *reinterpret_cast<uint16_t*>(to + at) = (uint16_t)two;
            } else {
                bytes[v][at] = (unsigned char)two;
                if (kept) to[at] = (uint8_t)two;
            }
        }
        if (lane == 0) {
            powers[v] = (unsigned char)b[v];
            if (kept) (v ? p.v_exp : p.k_exp)[place] = (uint8_t)b[v];
        }
    }
    __syncwarp();
}

// A block's share of one (unit, kv head): the tiles tile_begin .. tile_end - 1.  `part` < 0: the whole of it or a cluster's split; else where its
// sums go.
template <int D, int NT, bool FUSED>
__device__ __forceinline__ void piece(const GkPages8& p, const Rows8& a, const Fused8& f, Smem8<D, NT>& sm, const Unit& u, int hk, int tile_begin, int tile_end, int split,
                                      int part) {
    constexpr int ROWS = 8 * NT, KS = D / 16, MT = D / 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n_rows = u.n_rows, row_first = u.row_first, first_token = u.first_token, past = u.past, begin = u.begin;
    const bool writes = FUSED && f.write_kv && u.sound;
    const int end = u.end - (writes ? 1 : 0);  // the new key's place is not read

    // the numbers of the pages of this warp's next 32 tiles, one a lane
    int at = tile_begin + warp;
    auto pages_from = [&](int tile) {
        const int mine = tile + lane * WARPS;
        return mine < tile_end ? page_of(p, u.slot, mine / PER_PAGE) : -1;
    };
    int ids = pages_from(at), used = 0;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(sm.ring[warp]);
    int asked = at, into = 0;  // the next tile to ask for, and its place
    auto ask_next = [&] {
        if (asked < tile_end) {
            const int page = __shfl_sync(0xffffffffu, ids, used);
            if (++used == 32) {
                ids = pages_from(asked + WARPS);
                used = 0;
            }
            ask<D>(ring + into, p, hk, page, (asked % PER_PAGE) * KEYS, asked * KEYS, begin, end, lane);
            asked += WARPS;
            into = Place<D>::BYTES - into;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // places before the step's tokens were written by earlier steps: they may be asked for while the kernel in front still runs
    const bool early = at < tile_end && (at + 1) * KEYS <= past;
    if (early) ask_next();
    pdl_wait();
    if (!early) ask_next();

    const int new_tile = writes ? past / KEYS : -1;
    const bool owns = writes && past >= 0 && new_tile >= tile_begin && new_tile < tile_end && (new_tile - tile_begin) % WARPS == warp;
    if (owns) {
        if (f.weights_bf16) new_rows<D, __nv_bfloat16>(p, a, f, u, hk, lane, sm.fresh, sm.fresh_power);
        else new_rows<D, float>(p, a, f, u, hk, lane, sm.fresh, sm.fresh_power);
    }

    // queries: lane (g, t) has of row g of each tile of eight the columns 64 c + 16 t .. + 15
    uint32_t qf[NT][KS][2];
    float factor[NT][2];  // of the rows 2t, 2t + 1: what a product of halves times a key's power makes a score in powers of two
    int last[NT][2];      // and the last key they see
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = n * 8 + g, row = row_first + r;
        float x[D / 64][16], top = 0.f;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
            uint4 raw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
            if (r < n_rows) {
                const __nv_bfloat16* q = FUSED ? f.qkv + ((size_t)first_token * (a.n_q + 2 * p.n_kv) + hk * a.group + row) * D
                                               : a.q + ((size_t)(first_token + row / a.group) * a.n_q + hk * a.group + row % a.group) * D;
                const uint4* src = reinterpret_cast<const uint4*>(q + 64 * c + 16 * t);
                raw[0] = src[0];
                raw[1] = src[1];
            }
            const __nv_bfloat162* pairs = reinterpret_cast<const __nv_bfloat162*>(raw);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 two = __bfloat1622float2(pairs[i]);
                x[c][2 * i] = two.x;
                x[c][2 * i + 1] = two.y;
            }
        }
        if (FUSED) norm_rotate_queries<D>(f, x, past, t);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(x[c][i]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = max((int)(__float_as_uint(top) >> 23) - 127 - 14, -110);  // the row's largest goes to 2^14 .. 2^15
        const float back = __uint_as_float((uint32_t)(127 - e) << 23), ahead = __uint_as_float((uint32_t)(127 + e) << 23) * a.sl2;
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                qf[n][4 * c + j][0] = pack_half(x[c][4 * j] * back, x[c][4 * j + 1] * back);
                qf[n][4 * c + j][1] = pack_half(x[c][4 * j + 2] * back, x[c][4 * j + 3] * back);
            }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            factor[n][h] = __shfl_sync(0xffffffffu, ahead, (2 * t + h) * 4);
            const int mine = n * 8 + 2 * t + h;
            last[n][h] = mine < n_rows ? past + (row_first + mine) / a.group : -1;
        }
    }

    float ref_a[NT][2], ref_b[NT][2], l[NT][2], o[NT][MT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int h = 0; h < 2; ++h) ref_a[n][h] = ref_b[n][h] = NONE, l[n][h] = 0.f;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][m][i] = 0.f;
    }

    using At = Place<D>;
    uint32_t k_at[4], v_at[8];  // this lane's pieces of a place: keys 4g + i, values 8t + i
#pragma unroll
    for (int i = 0; i < 4; ++i) k_at[i] = At::key(4 * g + i, 16 * t);
#pragma unroll
    for (int i = 0; i < 8; ++i) v_at[i] = At::value(8 * t + i, D / 8 * g);
    uint32_t place = ring;
    float gap = -INFINITY;  // the largest B - A - 2 of this lane's rows
#pragma unroll 1
    for (; at < tile_end; at += WARPS) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();  // the tile has come for every lane, and every lane is done with the place that is asked into next
        ask_next();
        const int key0 = at * KEYS;
        if (FUSED && owns && at == new_tile) {  // 4 D / 64 bytes a lane into the tile's copy
            const int row = past - key0, byte = (lane & 15) * (D / 16);
            unsigned char* key = sm.ring[warp][place == ring ? 0 : 1];
#pragma unroll
            for (int i = 0; i < D / 16; i += 4)
                *reinterpret_cast<uint32_t*>(key + (lane < 16 ? Place<D>::key(row, byte + i) : Place<D>::value(row, byte + i))) =
                    *reinterpret_cast<const uint32_t*>(&sm.fresh[lane >> 4][byte + i]);
            if ((lane & 15) == 0) key[(lane ? At::VE : At::KE) + row] = sm.fresh_power[lane >> 4];
            __syncwarp();
        }
        // scores of 32 keys x rows: s[h][n][0], [1] = key 4g + 2h, rows 2t, 2t + 1; [2], [3] = key 4g + 2h + 1
        float s[2][NT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < NT; ++n) s[h][n][0] = s[h][n][1] = s[h][n][2] = s[h][n][3] = 0.f;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
            uint32_t k[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) read_words(k[i], place + (k_at[i] ^ (uint32_t)(c * 64)));
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t a0 = low_halves(k[2 * h][j]), a1 = low_halves(k[2 * h + 1][j]), a2 = high_halves(k[2 * h][j]), a3 = high_halves(k[2 * h + 1][j]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma(s[h][n], a0, a1, a2, a3, qf[n][4 * c + j][0], qf[n][4 * c + j][1]);
                }
        }
        const uint32_t ke = read_word(place + At::KE + 4 * g), ve = read_word(place + At::VE + 4 * g);
        float kf[4], ev[4];  // of the keys 4g + i: 2^ek, and ev
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            kf[i] = power_of(ke >> (8 * i) & 0xff);
            ev[i] = __uint_as_float(__byte_perm(ve, 0x4b000000u, 0x7650 + i)) - (8388608.f + 127.f);  // the byte as the last of 2^23 + byte
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[h][n][i] = s[h][n][i] * factor[n][i & 1] * kf[2 * h + (i >> 1)];
        const bool edge = key0 < u.all_begin || key0 + KEYS - 1 > u.pos_low;  // the same for the warp: some rows do not see all of these keys
        uint32_t none = 0;  // keys whose values hold a NaN, at an edge
        if (edge) {
            if (a.cu_q) {
                // A value that is NaN would reach rows that do not see it, 0 * NaN: zeros stand for its row and the score is made NaN instead.
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    uint32_t v[D / 32];
                    read_words(v, place + v_at[i]);
                    bool nan = false;
#pragma unroll
                    for (int w = 0; w < D / 32; ++w) nan |= __vcmpeq4(v[w] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0;
                    none |= __reduce_or_sync(0xffffffffu, nan ? 1u << (8 * t + i) : 0u);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int mine = 4 * g + 2 * h + (i >> 1), key = key0 + mine, top = last[n][i & 1];
                        if (none >> mine & 1) s[h][n][i] = NAN;
                        if (key > top || (a.window > 0 && key <= top - a.window)) s[h][n][i] = -INFINITY;
                    }
#pragma unroll
            for (int i = 0; i < 4; ++i)  // (places that no row sees hold any power: theirs is not to look small)
                if (key0 + 4 * g + i >= u.end || key0 + 4 * g + i < begin) ev[i] = 4096.f;
        }
        bool beyond = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float ma = -INFINITY, mb = -INFINITY;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        ma = fmaxf(ma, s[h][n][i + 2 * j]);
                        mb = fmaxf(mb, s[h][n][i + 2 * j] + ev[2 * h + j]);
                    }
                beyond |= ma > ref_a[n][i] + 14.f || mb > ref_b[n][i] + 15.f;
            }
        const float least = fminf(fminf(ev[0], ev[1]), fminf(ev[2], ev[3]));  // below the gap: values that are small beside those that B goes by
        if (__any_sync(0xffffffffu, beyond || least < gap)) {
            if (__any_sync(0xffffffffu, beyond)) {
                gap = -INFINITY;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float ma = -INFINITY, mb = -INFINITY;
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                ma = fmaxf(ma, s[h][n][i + 2 * j]);
                                mb = fmaxf(mb, s[h][n][i + 2 * j] + ev[2 * h + j]);
                            }
#pragma unroll
                        for (int w = 4; w < 32; w <<= 1) {
                            ma = fmaxf(ma, __shfl_xor_sync(0xffffffffu, ma, w));
                            mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, w));
                        }
                        const float na = fmaxf(ref_a[n][i], ma), nb = fmaxf(ref_b[n][i], mb - 7.f);
                        const float fa = exp2_fast(ref_a[n][i] - na), fb = exp2_fast(ref_b[n][i] - nb);
                        l[n][i] *= fa;
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            o[n][m][i] *= fb;
                            o[n][m][2 + i] *= fb;
                        }
                        ref_a[n][i] = na;
                        ref_b[n][i] = nb;
                        if (na > NONE) gap = fmaxf(gap, nb - na - 2.f);
                    }
            }
            if (__builtin_expect(__any_sync(0xffffffffu, least < gap), 0)) {
                // What the halves of small probabilities leave over, as the sum of two bfloat16 numbers (which reach as far down as 32 bits do) times values
                // in bfloat16 (exact).  In a loop, for its code stands in the way of all the other tiles'.
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                    uint32_t high[NT][2], low[NT][2];
                    bool some = false;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float rest[2];
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const float score = h ? s[1][n][2 * j + i] : s[0][n][2 * j + i], x = exp2_fast(score + ((h ? ev[2 + j] : ev[j]) - ref_b[n][i]));
                                rest[i] = x < 0x1p-14f && score > ref_a[n][i] - 32.f ? x - __half2float(__float2half_rn(x)) : 0.f;
                                some |= rest[i] != 0.f;
                            }
                            const uint32_t two = pack_bf16(rest[0], rest[1]);
                            high[n][j] = turned(two);
                            low[n][j] = turned(pack_bf16(rest[0] - __uint_as_float(two << 16), rest[1] - __uint_as_float(two & 0xffff0000u)));
                        }
                    if (!__any_sync(0xffffffffu, some)) continue;
#pragma unroll
                    for (int w = 0; w < D / 32; ++w) {
                        uint32_t v[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int mine = 2 * h + (i & 1) * 4 + (i >> 1);
                            v[i] = read_word(place + (h ? v_at[2 + (i & 1) * 4 + (i >> 1)] : v_at[(i & 1) * 4 + (i >> 1)]) + 4 * w);
                            if (none >> (8 * t + mine) & 1) v[i] = 0u;
                        }
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t near = __byte_perm(v[0], v[1], e ? 0x7362 : 0x5140), far = __byte_perm(v[2], v[3], e ? 0x7362 : 0x5140);
                            const uint32_t a0 = low_bf16(near), a1 = low_bf16(near >> 16), a2 = low_bf16(far), a3 = low_bf16(far >> 16);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                mma_bf16(o[n][2 * w + e], a0, a1, a2, a3, high[n][0], high[n][1]);
                                mma_bf16(o[n][2 * w + e], a0, a1, a2, a3, low[n][0], low[n][1]);
                            }
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t pf[NT][2], v[4][D / 32];
#pragma unroll
            for (int i = 0; i < 4; ++i) read_words(v[i], place + v_at[2 * h + (i & 1) * 4 + (i >> 1)]);  // values 8t + 2h, + 4, + 1, + 5
            if (none) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (none >> (8 * t + 2 * h + (i & 1) * 4 + (i >> 1)) & 1)
#pragma unroll
                        for (int w = 0; w < D / 32; ++w) v[i][w] = 0u;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    l[n][i & 1] += exp2_fast(s[h][n][i] - ref_a[n][i & 1]);
                    w[i] = exp2_fast(s[h][n][i] + (ev[2 * h + (i >> 1)] - ref_b[n][i & 1]));
                }
                pf[n][0] = turned(pack_half(w[0], w[1]));
                pf[n][1] = turned(pack_half(w[2], w[3]));
            }
#pragma unroll
            for (int w = 0; w < D / 32; ++w) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {  // columns 4w + 2e (rows g of the product) and 4w + 2e + 1 (rows g + 8)
                    const uint32_t near = __byte_perm(v[0][w], v[1][w], e ? 0x7362 : 0x5140), far = __byte_perm(v[2][w], v[3][w], e ? 0x7362 : 0x5140);
                    const uint32_t a0 = low_halves(near), a1 = high_halves(near), a2 = low_halves(far), a3 = high_halves(far);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma(o[n][2 * w + e], a0, a1, a2, a3, pf[n][0], pf[n][1]);
                }
            }
        }
        place = place == ring ? ring + At::BYTES : ring;
    }

    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // nobody reads a ring any more
    // a warp's rows to shared memory: lane (g, t) has the columns D / 8 * g .. of the rows 2t, 2t + 1
    using S = Smem8<D, NT>;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float sum = l[n][h];
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
            const int r = n * 8 + 2 * t + h;
            if (r >= n_rows) continue;
            if (g == 0) {
                sm.abl[warp][r][0] = ref_a[n][h];
                sm.abl[warp][r][1] = ref_b[n][h];
                sm.abl[warp][r][2] = sum;
            }
            float* to = sm.o[warp] + r * S::STRIDE + (D / 8) * g;
#pragma unroll
            for (int m = 0; m < MT; m += 2)
                *reinterpret_cast<float4*>(to + 2 * m) = make_float4(o[n][m][h], o[n][m][2 + h], o[n][m + 1][h], o[n][m + 1][2 + h]);
        }
    __syncthreads();
    const bool cluster = a.n_splits > 1;
    if (cluster) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    // the block's four warps, four columns a thread
    const int quads = n_rows * (D / 4), room = cluster ? (quads + a.n_splits - 1) / a.n_splits : 0;
    for (int i = threadIdx.x; i < quads; i += THREADS) {
        const int r = i / (D / 4), c = (i - r * (D / 4)) * 4;
        float A = NONE, B = NONE;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) A = fmaxf(A, sm.abl[w][r][0]), B = fmaxf(B, sm.abl[w][r][1]);
        float sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float fb = exp2_fast(sm.abl[w][r][1] - B);
            const float4 v = *reinterpret_cast<const float4*>(sm.o[w] + r * S::STRIDE + c);
            sum += sm.abl[w][r][2] * exp2_fast(sm.abl[w][r][0] - A);
            acc.x += v.x * fb, acc.y += v.y * fb, acc.z += v.z * fb, acc.w += v.w * fb;
        }
        if (cluster) {  // to the block of the cluster that joins these columns; what the sums stand by to all of them
            const int owner = i % a.n_splits, place = i / a.n_splits;
            uint32_t remote, here = (uint32_t)__cvta_generic_to_shared(sm.from_o + (split * room + place) * 4);
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(here), "r"(owner));
            asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(remote), "f"(acc.x), "f"(acc.y), "f"(acc.z), "f"(acc.w) : "memory");
            if (c == 0) {
                here = (uint32_t)__cvta_generic_to_shared(&sm.from_abl[split][r][0]);
                for (int to = 0; to < a.n_splits; ++to) {
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(here), "r"(to));
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(A) : "memory");
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote + 4), "f"(B) : "memory");
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote + 8), "f"(sum) : "memory");
                }
            }
        } else if (part < 0) {
            store4(out_row(a, u, hk, r, D) + c, acc, factor_of(A, B, sum, a.sink));
        } else {
            const size_t to = (size_t)part * ROWS + r;
            *reinterpret_cast<float4*>(a.part_o + to * D + c) = acc;
            if (c == 0) {
                a.part_abl[to * 3] = A;
                a.part_abl[to * 3 + 1] = B;
                a.part_abl[to * 3 + 2] = sum;
            }
        }
    }
    if (!cluster) return;
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (int place = threadIdx.x; place * a.n_splits + split < quads; place += THREADS) {
        const int i = place * a.n_splits + split, r = i / (D / 4), c = (i - r * (D / 4)) * 4;
        float A = NONE, B = NONE, sum = 0.f;
        for (int w = 0; w < a.n_splits; ++w) A = fmaxf(A, sm.from_abl[w][r][0]), B = fmaxf(B, sm.from_abl[w][r][1]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < a.n_splits; ++w) {
            const float fb = exp2_fast(sm.from_abl[w][r][1] - B);
            const float4 v = *reinterpret_cast<const float4*>(sm.from_o + (w * room + place) * 4);
            sum += sm.from_abl[w][r][2] * exp2_fast(sm.from_abl[w][r][0] - A);
            acc.x += v.x * fb, acc.y += v.y * fb, acc.z += v.z * fb, acc.w += v.w * fb;
        }
        store4(out_row(a, u, hk, r, D) + c, acc, factor_of(A, B, sum, a.sink));
    }
}

template <int D, int NT, bool FUSED>
__global__ void __launch_bounds__(THREADS, NT == 1 ? 3 : 2) rows8_kernel(const GkPages8 p, const Rows8 a, const Fused8 f) {
    constexpr int ROWS = 8 * NT;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    Smem8<D, NT>& sm = *reinterpret_cast<Smem8<D, NT>*>(smem_raw);
    pdl_launch_dependents();
    if (a.n_splits > 0) {
        const Unit u = unit_of(p, a, blockIdx.z, ROWS);
        if (u.n_rows <= 0) {  // the same for a whole cluster
            pdl_wait();       // (who waits for this launch counts on its having waited)
            return;
        }
        if (a.n_splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // all are here before one stores into another's memory
        const int split = blockIdx.x, per = (u.n_tiles + a.n_splits - 1) / a.n_splits, tile_begin = u.tile_0 + split * per;
        piece<D, NT, FUSED>(p, a, f, sm, u, blockIdx.y, tile_begin, min(tile_begin + per, u.tile_0 + u.n_tiles), split, -1);
        return;
    }
    const int lane = threadIdx.x & 31, size = piece_size(p, a, ROWS, lane);
    int before;
    const int unit = unit_at(p, a, size, blockIdx.x, -1, ROWS, lane, before);
    if (unit == a.n_units) {
        pdl_wait();
        return;
    }
    const Unit u = unit_of(p, a, unit, ROWS);
    const int cuts = (u.n_tiles + size - 1) / size, hk = (blockIdx.x - before) / cuts, cut = blockIdx.x - before - hk * cuts;
    const int per = (u.n_tiles + cuts - 1) / cuts, tile_begin = u.tile_0 + cut * per;
    piece<D, NT, FUSED>(p, a, f, sm, u, hk, tile_begin, min(tile_begin + per, u.tile_0 + u.n_tiles), 0, cuts == 1 ? -1 : (int)blockIdx.x);
}

// The pieces of a pair joined: a block a (row, kv head, unit), its warps take every fourth piece each; pairs of one piece are done already.
template <int D, int NT>
__global__ void __launch_bounds__(THREADS) rows8_join_kernel(const GkPages8 p, const Rows8 a) {
    constexpr int ROWS = 8 * NT, C = D / 32;  // columns a lane
    __shared__ float sums[WARPS][D], total[WARPS];
    const int r = blockIdx.x, hk = blockIdx.y, unit = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch_dependents();
    const Unit u = unit_of(p, a, unit, ROWS);
    const int size = piece_size(p, a, ROWS, lane), cuts = (u.n_tiles + size - 1) / size;
    int before;
    unit_at(p, a, size, 0, unit, ROWS, lane, before);
    pdl_wait();
    if (cuts == 1 || r >= u.n_rows) return;
    const size_t base = (size_t)(before + hk * cuts) * ROWS + r;
    float A = NONE, B = NONE, sum = 0.f, acc[C];
    for (int s = lane; s < cuts; s += 32) {
        A = fmaxf(A, a.part_abl[(base + (size_t)s * ROWS) * 3]);
        B = fmaxf(B, a.part_abl[(base + (size_t)s * ROWS) * 3 + 1]);
    }
    A = warp_max(A), B = warp_max(B);
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] = 0.f;
#pragma unroll 8
    for (int s = warp; s < cuts; s += WARPS) {
        const size_t from = base + (size_t)s * ROWS;
        const float fa = exp2_fast(a.part_abl[from * 3] - A), fb = exp2_fast(a.part_abl[from * 3 + 1] - B);
        sum += a.part_abl[from * 3 + 2] * fa;
        const float* o = a.part_o + from * D + lane * C;
#pragma unroll
        for (int i = 0; i < C; ++i) acc[i] += o[i] * fb;
    }
#pragma unroll
    for (int i = 0; i < C; ++i) sums[warp][lane * C + i] = acc[i];
    if (lane == 0) total[warp] = sum;
    __syncthreads();
    if (warp) return;
    const float f = factor_of(A, B, (total[0] + total[1]) + (total[2] + total[3]), a.sink);
    __nv_bfloat16* out = out_row(a, u, hk, r, D) + lane * C;
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] = (sums[0][lane * C + i] + sums[1][lane * C + i]) + (sums[2][lane * C + i] + sums[3][lane * C + i]);
#pragma unroll
    for (int i = 0; i < C; i += 2) *reinterpret_cast<__nv_bfloat162*>(out + i) = __floats2bfloat162_rn(acc[i] * f, acc[i + 1] * f);
}

template <int D, int NT>
int places_of(int cluster) {
    const int smem = (int)sizeof(Smem8<D, NT>);
    cudaError_t err = cudaFuncSetAttribute(rows8_kernel<D, NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (err != cudaSuccess) return -(int)err;
    gk_prepare_kernel((const void*)rows8_kernel<D, NT, false>);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster * 1024, 1, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    err = cudaOccupancyMaxActiveClusters(&clusters, rows8_kernel<D, NT, false>, &cfg);
    return err == cudaSuccess ? clusters : -(int)err;
}

template <int D, int NT, bool FUSED>
int launch_rows8(const GkPages8& p, const Rows8& a, const Fused8& f, cudaStream_t stream) {
    const int smem = (int)sizeof(Smem8<D, NT>);
    static std::atomic<unsigned long long> configured{0};  // a bit a device (the attribute is the device's)
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err == cudaSuccess && (device > 63 || !(configured.load() >> device & 1))) {
        err = cudaFuncSetAttribute(rows8_kernel<D, NT, FUSED>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (err == cudaSuccess && device <= 63) configured.fetch_or(1ull << device);
    }
    if (err != cudaSuccess) return gk_fail(GK_CUDA_ERROR, "rows8: %s", cudaGetErrorString(err));
    if (a.n_splits > 0) {
        gk_launch_cluster(rows8_kernel<D, NT, FUSED>, dim3(a.n_splits, p.n_kv, a.n_units), dim3(THREADS), smem, stream, dim3(a.n_splits, 1, 1), p, a, f);
        GK_CHECK_LAUNCH("rows8");
        return GK_OK;
    }
    gk_launch(rows8_kernel<D, NT, FUSED>, dim3(a.pieces + a.n_units * p.n_kv), dim3(THREADS), smem, stream, p, a, f);
    GK_CHECK_LAUNCH("rows8");
    const int rows = (int)min(8LL * NT, (long long)a.group * (a.cu_q ? 8 * NT : 1));
    gk_launch_behind(rows8_join_kernel<D, NT>, dim3(rows, p.n_kv, a.n_units), dim3(THREADS), 0, stream, p, a);
    GK_CHECK_LAUNCH("rows8_join");
    return GK_OK;
}

}  // namespace

// How many clusters of `cluster` blocks of so many rows the device holds at once, or a negative CUDA error.
GK_EXPORT int gk_rows8_places(int head_dim, int rows, int cluster) {
    if ((head_dim != 64 && head_dim != 128) || (rows != 8 && rows != 16) || cluster < 1 || cluster > 8) return -1;
    if (head_dim == 64) return rows == 8 ? places_of<64, 1>(cluster) : places_of<64, 2>(cluster);
    return rows == 8 ? places_of<128, 1>(cluster) : places_of<128, 2>(cluster);
}

// Rows taken together: 8 or 16.  `splits` 1 .. 8: so many blocks, a cluster, share a (row tile, kv head); 0: the step's keys are cut into pieces of one
// size, about `pieces` of them, with (pieces + units * n_kv) * rows * (head_dim + 3) floats of scratch, units = sequences * row tiles a sequence.
// `q`, `out` [n_tokens][n_q][head_dim] bfloat16.  `max_q_len`: no sequence brings more tokens.
static int rows8_entry(const GkPages8* pages, const void* q, void* out, const int* cu_q, const int* kv_len, const int* slots, int n_tokens, int n_seqs, int n_q,
                       int max_q_len, int rows, int splits, int pieces, float* scratch, float scale, int window, int sink, const Fused8& f, void* stream) {
    const int status = cache8::check(pages, "rows8");
    if (status != GK_OK) return status;
    const GkPages8& p = *pages;
    GK_REQUIRE(n_seqs >= 0 && n_q > 0 && n_q % p.n_kv == 0 && max_q_len >= 1 && window >= 0, "rows8: bad sizes n_seqs=%d heads %d/%d max_q_len=%d window=%d",
               n_seqs, n_q, p.n_kv, max_q_len, window);
    GK_REQUIRE((p.head_dim == 64 || p.head_dim == 128) && p.page_size == PAGE, "rows8: head_dim %d is not 64 or 128, or page_size %d not %d", p.head_dim,
               p.page_size, PAGE);
    GK_REQUIRE(rows == 8 || rows == 16, "rows8: %d rows a tile", rows);
    GK_REQUIRE(splits >= 0 && splits <= 8 && (splits > 0 || (scratch && pieces > 0)), "rows8: %d splits, %d pieces", splits, pieces);
    if (n_seqs == 0) return GK_OK;
    GK_REQUIRE((q || f.qkv) && out && kv_len && slots, "rows8: an array is missing");
    GK_REQUIRE((((uintptr_t)q | (uintptr_t)f.qkv | (uintptr_t)out | (uintptr_t)scratch) & 15) == 0, "rows8: memory must begin on 16-byte boundaries");
    const long long group = n_q / p.n_kv, tiles = cu_q ? (max_q_len * group + rows - 1) / rows : 1, units = tiles * n_seqs;
    GK_REQUIRE(n_tokens >= 0 && (cu_q || (max_q_len == 1 && n_tokens == n_seqs && group <= rows)), "rows8: %lld heads a kv head do not fit %d rows", group, rows);
    GK_REQUIRE(units <= 65535 && p.n_kv <= 65535 && pieces + units * p.n_kv < 2147483647LL, "rows8: grid too large");
    const Rows8 a = {(const __nv_bfloat16*)q, (__nv_bfloat16*)out, cu_q, kv_len, slots, n_tokens, max_q_len, n_q, (int)group, (int)tiles, (int)units, scale * 1.4426950408889634f,
                     window, sink, splits, pieces, scratch, scratch ? scratch + (size_t)(pieces + units * p.n_kv) * rows * p.head_dim : nullptr};
    cudaStream_t s = (cudaStream_t)stream;
    if (f.qkv) {
        if (p.head_dim == 64) return rows == 8 ? launch_rows8<64, 1, true>(p, a, f, s) : launch_rows8<64, 2, true>(p, a, f, s);
        return rows == 8 ? launch_rows8<128, 1, true>(p, a, f, s) : launch_rows8<128, 2, true>(p, a, f, s);
    }
    if (p.head_dim == 64) return rows == 8 ? launch_rows8<64, 1, false>(p, a, f, s) : launch_rows8<64, 2, false>(p, a, f, s);
    return rows == 8 ? launch_rows8<128, 1, false>(p, a, f, s) : launch_rows8<128, 2, false>(p, a, f, s);
}

GK_EXPORT int gk_rows8(const GkPages8* pages, const void* q, void* out, const int* cu_q, const int* kv_len, const int* slots, int n_tokens, int n_seqs, int n_q,
                       int max_q_len, int rows, int splits, int pieces, float* scratch, float scale, int window, int sink, void* stream) {
    return rows8_entry(pages, q, out, cu_q, kv_len, slots, n_tokens, n_seqs, n_q, max_q_len, rows, splits, pieces, scratch, scale, window, sink, Fused8{}, stream);
}

// One token a sequence, from the packed projection `qkv` [n_seqs][(n_q + 2 n_kv) * head_dim] bfloat16: norm and rotation of queries and keys and the
// write of the new key and value (`write_kv`) happen inside.
GK_EXPORT int gk_rows8_fused(const GkPages8* pages, const void* qkv, const void* wq, const void* wk, int weight_dtype, int use_norm, float eps,
                             const float* cos_table, const float* sin_table, int table_positions, int max_position, int write_kv, void* out,
                             const int* kv_len, const int* slots, int n_seqs, int n_q, int rows, int splits, int pieces, float* scratch, float scale,
                             int window, void* stream) {
    GK_REQUIRE(qkv || n_seqs == 0, "rows8_fused: qkv is missing");
    GK_REQUIRE(GK_VALID_DTYPE(weight_dtype) && (!use_norm || (wq && wk)), "rows8_fused: norm weights missing or of a bad type");
    GK_REQUIRE((cos_table == nullptr) == (sin_table == nullptr), "rows8_fused: cos and sin tables go together");
    GK_REQUIRE(cos_table == nullptr || max_position < table_positions, "rows8_fused: position %d is beyond the rotary table (%d positions)", max_position,
               table_positions);
    GK_REQUIRE((((uintptr_t)wq | (uintptr_t)wk | (uintptr_t)cos_table | (uintptr_t)sin_table) & 15) == 0, "rows8_fused: weights and tables must begin on 16-byte boundaries");
    const Fused8 f = {{wq, wk, cos_table, sin_table, table_positions, use_norm, eps}, (const __nv_bfloat16*)qkv, weight_dtype == GK_BF16, write_kv};
    return rows8_entry(pages, nullptr, out, nullptr, kv_len, slots, n_seqs, n_seqs, n_q, 1, rows, splits, pieces, scratch, scale, window, 0, f, stream);
}
