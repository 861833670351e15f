// The paged key-value cache of a full-attention layer in serving (gfx950): new tokens' keys and values into the cache
// with the position rotation on the way (append), and one new token per sequence attending to its cache (attend).
//
// The cache is [pages, page, heads, dim] of bf16 or e4m3 with any strides of its first three dims, so both memory
// orders in use (token rows of all heads, or a page's rows of one head together) are the same code.  A page table
// int32 [sequences, columns] names the pages of a sequence: token t lies in row t % page of page table[s][t / page].
#include <type_traits>

#include "common.h"

namespace prism {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

struct Cache {
    char *k, *v;                                    // bf16 or e4m3
    int64_t k_page, k_tok, k_head;                  // strides in bytes
    int64_t v_page, v_tok, v_head;
    const float *k_scale, *v_scale;                 // e4m3: fp32 [heads]; null: 1
    const int32_t* table;
    int64_t table_ld;
    int seqs, cols;                                 // the table's rows and columns
    int pages, shift;                               // page = 1 << shift tokens
};

// ------------------------------------------------------------------------------------------------------------ append
// A thread takes 16 dims of one head as two pieces of 8 that a rotation in halves pairs: dims 8 j .. + 7 and R / 2 + 8
// j .. + 7 of the R rotated ones, the same split of the others.  Every piece is one 16-byte load, 16 bytes (8 of e4m3)
// stored; neighbouring lanes hold neighbouring pieces.  One workgroup row per token (blockIdx.x), the token's heads
// (queries, keys, values) over blockIdx.y.  Bound by memory: nothing is read or written twice; 8191 tokens of 24 + 2 x
// 4 heads of 256 into an e4m3 cache (254 MB) 50 us, 5.1 TB/s, what a large copy reaches (53 us without the non-temporal
// loads and cache stores; the queries are read again at once, so theirs are plain).
struct AppendArgs {
    const uint16_t *q, *k, *v;
    uint16_t* qo;
    int64_t ldq, hq_s, ldk, hk_s, ldv, hv_s, ldo, ho_s;       // row and head strides (elements)
    const float* rope;                                        // [rope_rows, R]: cosines, then sines
    int64_t ldr;
    const int32_t *pos, *seq, *n;
    int rope_rows, R, adjacent, HQ, HKV;
    Cache c;
};

__device__ __forceinline__ void load8(const uint16_t* p, float* f) {
    const v4u u = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(p));
#pragma unroll
    for (int j = 0; j < 4; j++) {
        f[2 * j] = __uint_as_float(u[j] << 16);
        f[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
    }
}

template <bool NT>
__device__ __forceinline__ void store8_bf16(void* p, const float* f) {
    v4u u;
#pragma unroll
    for (int j = 0; j < 4; j++) u[j] = f32_to_bf16(f[2 * j]) | (f32_to_bf16(f[2 * j + 1]) << 16);
    if (NT) __builtin_nontemporal_store(u, reinterpret_cast<v4u*>(p));
    else *reinterpret_cast<v4u*>(p) = u;
}

// x / scale clamped to the largest e4m3 value (NaN stays), rounded to nearest even.
__device__ __forceinline__ float e4m3_clamp(float x) { return x > 448.f ? 448.f : x < -448.f ? -448.f : x; }
__device__ __forceinline__ void store8_e4m3(void* p, const float* f, float scale) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const float a = e4m3_clamp(div_rn(f[4 * i], scale)), b = e4m3_clamp(div_rn(f[4 * i + 1], scale));
        const float c = e4m3_clamp(div_rn(f[4 * i + 2], scale)), d = e4m3_clamp(div_rn(f[4 * i + 3], scale));
        int u = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, u, true);
    }
    __builtin_nontemporal_store(v2u{w[0], w[1]}, reinterpret_cast<v2u*>(p));
}

template <int D, bool F8>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
    constexpr int PER = D / 16;                               // threads per head
    const int item = blockIdx.y * blockDim.x + threadIdx.x;
    const int head = item / PER, j = item % PER;
    const int64_t t = blockIdx.x;
    if (head >= a.HQ + 2 * a.HKV || t >= __ldg(a.n)) return;
    const bool is_q = head < a.HQ, is_v = head >= a.HQ + a.HKV;
    const int h = is_q ? head : is_v ? head - a.HQ - a.HKV : head - a.HQ;
    const uint16_t* src = is_q ? a.q + t * a.ldq + h * a.hq_s : is_v ? a.v + t * a.ldv + h * a.hv_s
                                                                    : a.k + t * a.ldk + h * a.hk_s;
    const bool rot = j < a.R / 16;
    const int o0 = rot ? 8 * j : a.R + 8 * (j - a.R / 16);
    const int o1 = o0 + (rot ? a.R / 2 : (D - a.R) / 2);
    float x[8], y[8];
    load8(src + o0, x);
    load8(src + o1, y);
    // a position without a place (negative, past the table or the rotations, a page that is none) skips the token
    const int p = __ldg(a.pos + t), s = a.seq ? __ldg(a.seq + t) : (int)t;
    if (p < 0 || s < 0 || s >= a.c.seqs || (p >> a.c.shift) >= a.c.cols || (a.R && p >= a.rope_rows)) return;
    const int page = __ldg(a.c.table + s * a.c.table_ld + (p >> a.c.shift));
    if (page < 0 || page >= a.c.pages) return;
    if (rot && !is_v) {
        const float* row = a.rope + p * a.ldr;
        const int half = a.R / 2;
        // products and sums round one by one, as the formula is written
        if (!a.adjacent) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float c = row[o0 + i], sn = row[half + o0 + i], u = x[i], w = y[i];
                x[i] = add_rn(mul_rn(u, c), -mul_rn(w, sn));
                y[i] = add_rn(mul_rn(w, c), mul_rn(u, sn));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float c = row[o0 / 2 + i], sn = row[half + o0 / 2 + i], u = x[2 * i], w = x[2 * i + 1];
                x[2 * i] = add_rn(mul_rn(u, c), -mul_rn(w, sn));
                x[2 * i + 1] = add_rn(mul_rn(w, c), mul_rn(u, sn));
                const float c1 = row[o1 / 2 + i], sn1 = row[half + o1 / 2 + i], u1 = y[2 * i], w1 = y[2 * i + 1];
                y[2 * i] = add_rn(mul_rn(u1, c1), -mul_rn(w1, sn1));
                y[2 * i + 1] = add_rn(mul_rn(w1, c1), mul_rn(u1, sn1));
            }
        }
    }
    if (is_q) {
        uint16_t* d = a.qo + t * a.ldo + h * a.ho_s;
        store8_bf16<false>(d + o0, x);
        store8_bf16<false>(d + o1, y);
        return;
    }
    const int64_t at = p & ((1 << a.c.shift) - 1);
    char* d = is_v ? a.c.v + page * a.c.v_page + at * a.c.v_tok + h * a.c.v_head
                   : a.c.k + page * a.c.k_page + at * a.c.k_tok + h * a.c.k_head;
    if (F8) {
        const float* sc = is_v ? a.c.v_scale : a.c.k_scale;
        const float scale = sc ? __ldg(sc + h) : 1.f;
        store8_e4m3(d + o0, x, scale);
        store8_e4m3(d + o1, y, scale);
    } else {
        store8_bf16<true>(d + 2 * o0, x);
        store8_bf16<true>(d + 2 * o1, y);
    }
}

// ------------------------------------------------------------------------------------------------------------ attend
// o[h] = sum_t softmax_t(scale q_h . k_t) v_t over a sequence's visible tokens, all query heads of one key head
// together (they read the same keys and values), in one pass with a running maximum and sum per query head.
//
// A wave takes blocks of 32 tokens: scores transposed, S^T = K Q^T (the keys as the MFMA's first operand,
// query heads its 16 columns), leave each lane the scores of ITS head (lane % 16) for tokens 4 g + r and 16 + 4 g + r
// (g = lane / 16, r < 4).  O^T = V^T P^T wants in each lane 8 tokens of its head as second operand, and the order of
// the 32 tokens along the product is free as long as both operands agree: taking them as the scores lie, P never
// leaves its lane, and neither do the maximum, the sum and the rescaling of O^T's columns (all of head lane % 16).
// V's operand needs 8 tokens of one dim per lane: a lane loads its 8 tokens' rows in pieces of D / 16 dims (16 lanes
// a whole row, contiguous) and turns the 8 x D/16 block with one v_perm per register.
// P is split into three bf16 parts, each what the last one left (the first two cut, the third rounded: within 2^-23 of the
// weight), so the weights carry fp32's bits and the output's one bf16 rounding is the only one that shows.  The further
// MFMAs are free beside the cache's bytes: with two parts, cut, the same times (98.7 and 98.7, 101.4 and 101.8, 126.8 and 126.7
// us for the three sizes below), and outputs that lean toward zero by 1e-5, what the weights lose and their sum does not.
//
// Work is split on the device, from the lengths (a captured launch serves every batch): a unit is what the four waves
// take in one round (128 tokens of a head, or 32 of four); laid one after the other, the sequences' units are dealt out
// `per` to a workgroup, so that `target` of them share all the work evenly, whatever the lengths.  A sequence within
// one workgroup gets its output at once; the others' parts are joined by a second kernel in a fixed order, so results
// do not depend on timing.
//
// Bound by the cache's bytes, read once: one sequence of 131071 tokens, 8 heads of 128 bf16 (537 MB), 98 us, 5.5 TB/s, 90
// of them this kernel (6.0 TB/s, more than a copy moves) and 7 the joining one; 40 of up to 20000, 4 heads of 256 e4m3
// (505 MB), 101 us, 5.0 TB/s; token rows of 8 heads of 64, 128 sequences of up to 4096 visible (613 MB), 125 us,
// 4.9 TB/s (runs of 512 bytes a token; the same heads' rows by the page take 120).  A short call (613 tokens) is launches
// and one chain of a unit's steps, 9 us.
struct AttendArgs {
    const uint16_t* q;
    uint16_t* out;
    int64_t ldq, hq_s, ldo, ho_s;
    const int32_t *lens, *n;
    float* part_o;                                            // [2 P, HQ, D]: two parts a workgroup
    float* part_ml;                                           // [2 P, HQ, 2]
    int2* plan;                                               // [T]: a sequence's first part and how many it has
    float scale;                                              // times log2 e
    int T, HQ, G, tiles, HT, window, target;
    Cache c;
};

constexpr int kWaves = 4;

template <int UNIT>
__device__ __forceinline__ int vis_units(const AttendArgs& a, int len, int* lo_out, int* len_out) {
    // (a column count times a page beyond 2^31 still bounds the length)
    const int64_t cap = (int64_t)a.c.cols << a.c.shift;
    len = max(0, (int)min((int64_t)len, cap));
    const int lo = a.window > 0 ? max(0, len - a.window) : 0;
    *lo_out = lo;
    *len_out = len;
    const int span = len - (lo & ~15);
    return span / UNIT + (span % UNIT != 0);
}

__device__ __forceinline__ long long wave_sum(long long v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    return v;
}

// Where workgroup p's units begin: unit u = p per of all sequences' one after the other (a sequence without tokens has
// one, for its zeros) lies in sequence b, `off` units from its start; `left` units to do.  The same in every lane; b <
// 0: none.
struct Plan {
    int b, off, left, per;
};
template <int UNIT>
__device__ __forceinline__ Plan make_plan(const AttendArgs& a, int p) {
    const int lane = threadIdx.x & 63;
    const int len0 = lane < a.T ? __ldg(a.lens + lane) : 0;   // (loads that need not wait for n)
    const int n = min(__ldg(a.n), a.T);
    int lo, len;
    const int units0 = lane < n ? max(1, vis_units<UNIT>(a, len0, &lo, &len)) : 0;
    long long total = __builtin_amdgcn_readfirstlane(units0);
    if (n > 1) {
        long long sum = units0;
        for (int b = lane + 64; b < n; b += 64) sum += max(1, vis_units<UNIT>(a, __ldg(a.lens + b), &lo, &len));
        total = wave_sum(sum);
    }
    Plan r;
    r.b = -1;
    r.per = max((int)((total * a.HT + a.target - 1) / a.target), 1);
    const long long u = (long long)p * r.per;
    if (u >= total) return r;
    r.left = (int)min((long long)r.per, total - u);
    if (n == 1) {
        r.b = 0, r.off = (int)u;
        return r;
    }
    long long base = 0;
    for (int b0 = 0; b0 < n; b0 += 64) {
        const int b = b0 + lane;
        const int units = b0 == 0 ? units0 : b < n ? max(1, vis_units<UNIT>(a, __ldg(a.lens + b), &lo, &len)) : 0;
        long long incl = units;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const long long up = __shfl_up(incl, o, kWave);
            if (lane >= o) incl += up;
        }
        const long long at = u - (base + incl - units);       // from the start of this lane's sequence
        const uint64_t m = __ballot(at >= 0 && at < units);
        if (m) {
            const int src = __builtin_ctzll(m);
            r.b = b0 + src;
            r.off = __shfl((int)at, src, kWave);
            break;
        }
        base += __shfl(incl, 63, kWave);
    }
    return r;
}

__device__ __forceinline__ v8bf as_bf(v4u x) { return __builtin_bit_cast(v8bf, x); }
__device__ __forceinline__ v4f mfma_bf16(v4u a, v4u b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(a), as_bf(b), c, 0, 0, 0);
}
// Two weights' upper parts as bf16, each cut to 8 bits strictly below the weight, and what is left of them.  What is left
// of a weight is then never 0: a part of 0 times an infinite value would be NaN, where the weight itself gives infinity.
__device__ __forceinline__ uint32_t below(float e0, float e1, float& r0, float& r1) {
    const uint32_t b0 = max(__float_as_uint(e0), 1u) - 1u, b1 = max(__float_as_uint(e1), 1u) - 1u;
    r0 = e0 - __uint_as_float(b0 & 0xffff0000u), r1 = e1 - __uint_as_float(b1 & 0xffff0000u);
    return __builtin_amdgcn_perm(b1, b0, 0x07060302u);
}
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

// Two e4m3 bytes (SEL: the upper two) as two bf16, exactly.
template <bool SEL>
__device__ __forceinline__ uint32_t e4m3x2_bf16(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, SEL));
}

// One 32-token block: its loads' sizes, and its values' registers.
template <int D, bool F8>
struct Block {
    static constexpr int RB = (F8 ? 1 : 2) * D;               // bytes of a token's row
    static constexpr int L = RB / 64;                         // loads of 1 KB for 16 tokens
    static constexpr int VB = RB / 16, VW = VB / 4;           // value bytes and words per token and lane
    // LDS bytes of a wave: the keys and values, at the end 16 columns of O
    static constexpr int STAGE = 4 * L * 1024 > 16 * (D + 4) * 4 ? 4 * L * 1024 : 16 * (D + 4) * 4;
    uint32_t v[2][4][VW];
};

// The lane's piece of its 8 tokens' values (4 g + r of each 16).
template <int D, bool F8>
__device__ __forceinline__ void read_v(Block<D, F8>& s, const char* vl) {
    using B = Block<D, F8>;
#pragma unroll
    for (int a = 0; a < 2; a++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const char* p = vl + (16 * a + r) * B::RB;
            if constexpr (B::VW == 1) {
                s.v[a][r][0] = *reinterpret_cast<const uint32_t*>(p);
            } else if constexpr (B::VW == 2) {
                const v2u x = *reinterpret_cast<const v2u*>(p);
                s.v[a][r][0] = x[0], s.v[a][r][1] = x[1];
            } else {
#pragma unroll
                for (int i = 0; i < B::VW / 4; i++) {         // dims 8 c .. and 128 + 8 c .. of 256 bf16
                    const v4u x = *reinterpret_cast<const v4u*>(p + 256 * i);
#pragma unroll
                    for (int w = 0; w < 4; w++) s.v[a][r][4 * i + w] = x[w];
                }
            }
        }
}

// The dim that fragment f of O^T holds in row m (piece m).
template <int D, bool F8>
__device__ __forceinline__ int dim_of(int f, int m) {
    if constexpr (D == 256 && !F8) return f < 8 ? 8 * m + f : 128 + 8 * m + f - 8;
    else return (D / 16) * m + f;
}

// Fragments 4 q .. 4 q + 3 of V's operand (4 dims of the lane's piece): 8 tokens each, as j = 4 a + r.
template <int D, bool F8>
__device__ __forceinline__ void turn_v(const Block<D, F8>& s, int q, v4u (&out)[4]) {
    if constexpr (!F8) {
#pragma unroll
        for (int f = 0; f < 4; f++) {
            const uint32_t sel = (f & 1) ? 0x07060302u : 0x05040100u;
#pragma unroll
            for (int w = 0; w < 4; w++)
                out[f][w] = __builtin_amdgcn_perm(s.v[w / 2][2 * (w % 2) + 1][2 * q + f / 2],
                                                  s.v[w / 2][2 * (w % 2)][2 * q + f / 2], sel);
        }
    } else {
#pragma unroll
        for (int a = 0; a < 2; a++) {
            const uint32_t r0 = s.v[a][0][q], r1 = s.v[a][1][q], r2 = s.v[a][2][q], r3 = s.v[a][3][q];
            const uint32_t x = __builtin_amdgcn_perm(r1, r0, 0x05010400u), y = __builtin_amdgcn_perm(r3, r2, 0x05010400u);
            const uint32_t z = __builtin_amdgcn_perm(r1, r0, 0x07030602u), w = __builtin_amdgcn_perm(r3, r2, 0x07030602u);
            const uint32_t d[4] = {__builtin_amdgcn_perm(y, x, 0x05040100u), __builtin_amdgcn_perm(y, x, 0x07060302u),
                                   __builtin_amdgcn_perm(w, z, 0x05040100u), __builtin_amdgcn_perm(w, z, 0x07060302u)};
#pragma unroll
            for (int f = 0; f < 4; f++) {
                out[f][2 * a] = e4m3x2_bf16<false>(d[f]);
                out[f][2 * a + 1] = e4m3x2_bf16<true>(d[f]);
            }
        }
    }
}

// SIDE: the four waves take four neighbouring heads of the same 32 tokens (unit: 32 tokens, no joining of waves)
// instead of four blocks of one head's: where a token's heads lie side by side in memory, a workgroup then reads 4 of
// them in one run.
template <int D, bool F8, bool SIDE>
__global__ __launch_bounds__(256, 2) void kv_attend_kernel(AttendArgs a) {
    using B = Block<D, F8>;
    constexpr int WT = SIDE ? 1 : kWaves, UNIT = 32 * WT, F = D / 16, QF = D / 32, L = B::L;
    extern __shared__ __align__(16) char lds[];               // per wave: keys, at the end 16 columns of O; then m and l
    // a part's heads, whose rows lie side by side in a cache of token rows, on one XCD (workgroup i runs on XCD i % 8)
    const int ht = blockIdx.x / 8 % a.HT, part = blockIdx.x / (8 * a.HT) * 8 + blockIdx.x % 8;
    const Plan pl = make_plan<UNIT>(a, part);
    if (pl.b < 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hk = SIDE ? 4 * ht + wave : ht / a.tiles, tile = SIDE ? 0 : ht % a.tiles;
    const int h0 = hk * a.G + 16 * tile, nh = min(16, a.G - 16 * tile);
    const int col = lane & 15, g = lane >> 4;
    int b = __builtin_amdgcn_readfirstlane(pl.b), off = __builtin_amdgcn_readfirstlane(pl.off);
    int left = __builtin_amdgcn_readfirstlane(pl.left);
    for (;;) {                                                // a sequence, or as much of it as is this workgroup's
        int lo, len;
        const int units = max(1, vis_units<UNIT>(a, __ldg(a.lens + b), &lo, &len)), seg = min(left, units - off);
        const int begin = (lo & ~15) + off * UNIT;
        const int end = seg == units - off ? len : begin + seg * UNIT;
        const bool whole = seg == units;

        v4u qf[QF];                                               // heads past the tile: zeros
#pragma unroll
        for (int i = 0; i < QF; i++) {
            const int d = F8 ? 64 * (i / 2) + 16 * g + 8 * (i % 2) : 32 * i + 8 * g;
            qf[i] = col < nh ? *reinterpret_cast<const v4u*>(a.q + b * a.ldq + (h0 + col) * a.hq_s + d) : v4u{0, 0, 0, 0};
        }
        const float sc = a.scale * (F8 && a.c.k_scale ? __ldg(a.c.k_scale + hk) : 1.f);

        v4f o[F];
#pragma unroll
        for (int f = 0; f < F; f++) o[f] = v4f{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;

        // the table through the scalar cache: a vector load would be waited for together with the values in flight
        // before it
        const auto* row = reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(
            reinterpret_cast<uintptr_t>(a.c.table + b * a.c.table_ld));
        const int last = len > 0 ? (len - 1) & ~15 : 0;           // the last 16 tokens that are there
        // Keys and values go to LDS by DMA, 1 KB a load.  Keys: 16 tokens x 64 bytes, four neighbouring lanes a token's
        // (the memory pipeline merges neighbouring lanes only), placed so that operand order reads without bank
        // conflicts; values: whole rows.  Every wait on them is written out: the compiler would wait for all of them at
        // each use.
        const uint32_t koff = (uint32_t)((lane >> 2) * a.c.k_tok) + 16 * ((lane & 3) ^ lds_turn(lane >> 4));
        const uint32_t voff = (uint32_t)(16 * lane / B::RB * a.c.v_tok) + 16 * lane % B::RB;
        const char* kb = a.c.k + hk * a.c.k_head;
        const char* vb = a.c.v + hk * a.c.v_head;
        char* stage = lds + wave * B::STAGE;
        const v4u* kl = reinterpret_cast<const v4u*>(stage) + 4 * col + (g ^ lds_turn(col >> 2));
        const char* vl = stage + 2 * L * 1024 + 4 * g * B::RB + (D == 256 && !F8 ? 16 : B::VB) * col;

        int64_t page[2];
        auto locate = [&](int t0) {
#pragma unroll
            for (int x = 0; x < 2; x++) page[x] = row[min(t0 + 16 * x, last) >> a.c.shift];  // 16 tokens never cross a page
        };
        auto clamp = [&] {
#pragma unroll
            for (int x = 0; x < 2; x++) page[x] = min(max((int)page[x], 0), a.c.pages - 1);
        };
        auto at = [&](int t0, int x) { return (int64_t)(min(t0 + 16 * x, last) & ((1 << a.c.shift) - 1)); };
        auto load_k = [&](int t0) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const char* p = kb + page[x] * a.c.k_page + at(t0, x) * a.c.k_tok + koff;
#pragma unroll
                for (int i = 0; i < L; i++) dma16(p + 64 * i, stage + (x * L + i) * 1024);
            }
        };
        auto load_v = [&](int t0) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const char* p = vb + page[x] * a.c.v_page + at(t0, x) * a.c.v_tok + voff;
#pragma unroll
                for (int i = 0; i < L; i++) dma16(p + i * (1024 / B::RB) * a.c.v_tok, stage + (2 * L + x * L + i) * 1024);
            }
        };
        B s;
        // One block of 32 tokens; with `more`, the next one's loads go out as this one's places in LDS become free.
        auto block = [&](int t0, auto more) {
            constexpr bool MORE = decltype(more)::value;
            vm_wait<2 * L>();  // the keys are there (the values' loads came after theirs)
            if (MORE) locate(t0 + UNIT);
            v4f st[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int i = 0; i < QF; i++) {
                    v4u kf;
                    if constexpr (F8) {
                        const v4u w = kl[(x * L + i / 2) * 64];
                        const uint32_t w0 = w[2 * (i % 2)], w1 = w[2 * (i % 2) + 1];
                        kf = v4u{e4m3x2_bf16<false>(w0), e4m3x2_bf16<true>(w0), e4m3x2_bf16<false>(w1),
                                 e4m3x2_bf16<true>(w1)};
                    } else {
                        kf = kl[(x * L + i) * 64];
                    }
                    st[x] = mfma_bf16(kf, qf[i], st[x]);
                }
            if (MORE) {
                clamp();
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // this block's keys are read
                load_k(t0 + UNIT);
            }
            vm_wait<MORE ? 2 * L : 0>();                          // the values are there
            read_v<D, F8>(s, vl);
            if (MORE) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // ... and read
                load_v(t0 + UNIT);
            }
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; j++) p[j] = mul_rn(st[j / 4][j % 4], sc);
            if (t0 < lo || (!MORE && t0 + 32 > len)) {
                // tokens outside get no weight, and their values, which may be anything (a page's unwritten rows), are
                // zeroed
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int t = t0 + 16 * (j / 4) + 4 * g + j % 4;
                    const bool in = t >= lo && t < len;
                    p[j] = in ? p[j] : -INFINITY;
#pragma unroll
                    for (int w = 0; w < B::VW; w++) s.v[j / 4][j % 4][w] = in ? s.v[j / 4][j % 4][w] : 0;
                }
            }
            float bm = p[0];
#pragma unroll
            for (int j = 1; j < 8; j++) bm = fmaxf(bm, p[j]);
            bm = fmaxf(bm, __shfl_xor(bm, 16, kWave));
            bm = fmaxf(bm, __shfl_xor(bm, 32, kWave));
            const float mn = fmaxf(m, bm), ref = mn == -INFINITY ? 0.f : mn;
            if (__any(mn > m)) {
                const float al = __builtin_amdgcn_exp2f(m - ref);
                l *= al;
#pragma unroll
                for (int f = 0; f < F; f++) o[f] *= al;
            }
            m = mn;
            uint32_t hi[4], mid[4], lo[4];
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float e0 = __builtin_amdgcn_exp2f(p[2 * w] - ref), e1 = __builtin_amdgcn_exp2f(p[2 * w + 1] - ref);
                l += e0 + e1;
                float r0, r1, s0, s1;
                hi[w] = below(e0, e1, r0, r1);
                mid[w] = below(r0, r1, s0, s1);
                lo[w] = __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{s0, s1}), v2bf));
            }
            const v4u ph = {hi[0], hi[1], hi[2], hi[3]}, pm = {mid[0], mid[1], mid[2], mid[3]},
                      pl = {lo[0], lo[1], lo[2], lo[3]};
#pragma unroll
            for (int q = 0; q < F / 4; q++) {
                v4u vf[4];
                turn_v<D, F8>(s, q, vf);
#pragma unroll
                for (int f = 0; f < 4; f++) {
                    o[4 * q + f] = mfma_bf16(vf[f], ph, o[4 * q + f]);
                    o[4 * q + f] = mfma_bf16(vf[f], pm, o[4 * q + f]);
                    o[4 * q + f] = mfma_bf16(vf[f], pl, o[4 * q + f]);
                }
            }
        };
        int t0 = begin + (SIDE ? 0 : 32 * wave);
        if (t0 < end) {
            locate(t0);
            clamp();
            load_k(t0);
            load_v(t0);
            for (; t0 + UNIT < end; t0 += UNIT) block(t0, std::true_type{});
            block(t0, std::false_type{});
        }

        // the four waves' columns, joined: each to the common maximum (SIDE: a wave's own)
        constexpr int LD = D + 4;
        float* lm = reinterpret_cast<float*>(lds + kWaves * B::STAGE);
        float* ll = lm + kWaves * 16;
        l += __shfl_xor(l, 16, kWave);
        l += __shfl_xor(l, 32, kWave);
        if (lane < 16) {
            lm[wave * 16 + lane] = m;
            ll[wave * 16 + lane] = l;
        }
        float* mine = reinterpret_cast<float*>(stage) + col * LD;
#pragma unroll
        for (int f = 0; f < F; f++)
#pragma unroll
            for (int r = 0; r < 4; r++) mine[dim_of<D, F8>(f, 4 * g + r)] = o[f][r];
        __syncthreads();
        // its first part's number and how many it has: the rest's units by `per`
        if (a.plan && off == 0 && ht == 0 && threadIdx.x == 0)
            a.plan[b] = int2{part, 1 + (units - seg + pl.per - 1) / pl.per};
        const float vs = F8 && a.c.v_scale ? __ldg(a.c.v_scale + hk) : 1.f;
        const int64_t slot = 2 * (int64_t)part + (off == 0);  // of a workgroup's parts one ends a sequence, one begins one
        const int w0 = SIDE ? wave : 0;
        for (int i = SIDE ? lane : threadIdx.x; i < nh * (D / 4); i += SIDE ? 64 : 256) {
            const int h = i / (D / 4), d = 4 * (i % (D / 4));
            float mm = lm[16 * w0 + h];
#pragma unroll
            for (int w = 1; w < WT; w++) mm = fmaxf(mm, lm[16 * w + h]);
            const float ref = mm == -INFINITY ? 0.f : mm;
            float sum = 0.f;
            v4f acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = w0; w < w0 + WT; w++) {
                const float e = __builtin_amdgcn_exp2f(lm[16 * w + h] - ref);
                sum += e * ll[16 * w + h];
                acc += e * *reinterpret_cast<const v4f*>(lds + w * B::STAGE + (h * LD + d) * 4);
            }
            if (whole) {
                // zeros without tokens; with tokens whose scores are all -inf 0 / 0, as the softmax is
                uint32_t u[4];
#pragma unroll
                for (int j = 0; j < 4; j++) u[j] = f32_to_bf16(len == 0 ? 0.f : div_rn(acc[j], sum) * vs);
                *reinterpret_cast<v2u*>(a.out + b * a.ldo + (h0 + h) * a.ho_s + d) =
                    v2u{u[0] | (u[1] << 16), u[2] | (u[3] << 16)};
            } else {
                const int64_t to = slot * a.HQ + h0 + h;
                *reinterpret_cast<v4f*>(a.part_o + to * D + d) = acc;
                if (d == 0) {
                    a.part_ml[2 * to] = mm;
                    a.part_ml[2 * to + 1] = sum;
                }
            }
        }
        left -= seg;
        if (left == 0) return;
        b++, off = 0;
        __syncthreads();                                          // the next sequence's loads overwrite what was joined
    }
}

// Joins the parts of sequence blockIdx.y's query heads hb blockIdx.x ..: groups of D / 4 threads, `share` of them (a
// power of two, as many as the parts need) to a head, each every share-th part in order, then the groups in order.
template <int D>
__global__ __launch_bounds__(256) void kv_join_kernel(AttendArgs a, int hb) {
    constexpr int TC = D / 4, NG = 256 / TC;
    __shared__ float lds[NG][D + 4];
    __shared__ float red[NG];
    const int b = blockIdx.y, n = __ldg(a.n);
    const int2 pl = a.plan[b];                                // (a row past n has none: not used)
    if (b >= n || pl.y < 2) return;
    const int c = threadIdx.x % TC, grp = threadIdx.x / TC;
    auto slot = [&](int i) { return 2 * (int64_t)(pl.x + i) + (i == 0); };
    int share = 2;
    while (share < NG && share < pl.y) share *= 2;
    share = min(share, NG);
    const int heads = NG / share, sub = grp % share;
    const int hend = min(a.HQ, (int)(blockIdx.x + 1) * hb);
    for (int h0 = blockIdx.x * hb; h0 < hend; h0 += heads) {
        const int h = h0 + grp / share;
        v4f acc = {0.f, 0.f, 0.f, 0.f};
        float sum = 0.f;
        if (h < hend) {
            float mm = -INFINITY;
            for (int i = c; i < pl.y; i += TC) mm = fmaxf(mm, a.part_ml[2 * (slot(i) * a.HQ + h)]);
#pragma unroll
            for (int o = TC / 2; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o, kWave));
            const float ref = mm == -INFINITY ? 0.f : mm;
            for (int i = sub; i < pl.y; i += share) {
                const int64_t at = slot(i) * a.HQ + h;
                const float e = __builtin_amdgcn_exp2f(a.part_ml[2 * at] - ref);
                sum += e * a.part_ml[2 * at + 1];
                acc += e * *reinterpret_cast<const v4f*>(a.part_o + at * D + 4 * c);
            }
        }
        *reinterpret_cast<v4f*>(&lds[grp][4 * c]) = acc;
        if (c == 0) red[grp] = sum;
        __syncthreads();
        if (h < hend && sub == 0) {
            for (int i = 1; i < share; i++) {
                acc += *reinterpret_cast<const v4f*>(&lds[grp + i][4 * c]);
                sum += red[grp + i];
            }
            const float vs = a.c.v_scale ? __ldg(a.c.v_scale + h / a.G) : 1.f;
            uint32_t u[4];
#pragma unroll
            for (int j = 0; j < 4; j++) u[j] = f32_to_bf16(div_rn(acc[j], sum) * vs);     // (two parts: there are tokens)
            *reinterpret_cast<v2u*>(a.out + b * a.ldo + h * a.ho_s + 4 * c) =
                v2u{u[0] | (u[1] << 16), u[2] | (u[3] << 16)};
        }
        __syncthreads();
    }
}

// LDS of a workgroup, and how many workgroups a launch's work is dealt out to: as many as are there at a time, two a CU
// where LDS holds them.  With 4 a CU (rows of 128 bytes leave LDS for them) 128 sequences of 100 - 4096 visible tokens,
// 8 heads of 64, took 138 us instead of 133.5, 64 of 8000 tokens, 8 heads of 128 e4m3, 205 instead of 199: every further
// part is more to join.  One a CU: 131071 tokens, 8 heads of 128 bf16, 98 us instead of 100, but 256 sequences of
// 20 - 300 tokens 50 instead of 41.
static int attend_lds(int64_t D, bool f8) {
    const int64_t stage = 4 * (f8 ? D : 2 * D) / 64 * 1024, o = 16 * (D + 4) * 4;
    return (int)(kWaves * (stage > o ? stage : o) + 2 * kWaves * 16 * 4);
}
static int attend_target(int64_t D, bool f8) {
    return 2 * attend_lds(D, f8) <= 160 * 1024 ? 512 : 256;
}

// Workgroups per head (or four side by side): all units at `per` each, no more than the target's share and no more than
// there are units.
static int64_t attend_parts(int64_t T, int64_t HT, int64_t cap, int64_t unit, int target) {
    const int64_t most = T * ((cap + unit - 1) / unit), split = target / HT + 1;
    return most < split ? most : split;
}

// Whether waves may take heads side by side: whole groups of four, a tile of query heads each, and enough sequences
// that the parts, now of four heads each, are few.  With and without, rows of 8 heads: 128 sequences of 100 - 4096
// visible tokens of 64 bf16 124 / 146 us, 64 of 8000 tokens of 128 364 / 391 (e4m3 199 / 234), 16 of 4000 of 64
// 34.7 / 37.6; but 8 of those 20.5 / 19.5, one of 32768 28 / 21, and 16 of 300 - 500 tokens of 128 e4m3 13.2 / 11.7.  The
// lengths are on the device, so the rule sees the rows of the batch and the room of the table: short sequences in a table
// with room for long ones take this form as well.
static bool attend_side(int64_t T, int64_t hq, int64_t heads, int64_t cap) {
    return heads % 4 == 0 && hq / heads <= 16 && T >= 16 && cap >= 1024;
}

// The cache's arguments, checked; strides from elements to bytes.
static_assert(sizeof(prism_kv_cache) == 19 * 8 && sizeof(prism_kv_append_args) == 41 * 8 &&
              sizeof(prism_kv_attend_args) == 32 * 8, "8-byte fields throughout");

static int make_cache(Cache& c, const prism_kv_cache& h) {
    if (!h.k || !h.v || !h.table || (h.e4m3 != 0 && h.e4m3 != 1)) return PRISM_ERR_ARG;
    if (!h.e4m3 && (h.k_scale || h.v_scale)) return PRISM_ERR_ARG;
    if (h.heads < 1 || h.heads > 65536 || (h.dim != 64 && h.dim != 128 && h.dim != 256)) return PRISM_ERR_SHAPE;
    if (h.page < 16 || h.page > 65536 || (h.page & (h.page - 1)) || h.pages < 1 || h.pages > INT32_MAX)
        return PRISM_ERR_SHAPE;
    if (h.seqs < 1 || h.seqs > INT32_MAX || h.cols < 1 || h.cols > (1 << 27) || h.table_ld < h.cols) return PRISM_ERR_SHAPE;
    const int64_t size = h.e4m3 ? 1 : 2, unit = 16 / size;
    if (h.k_page < 0 || h.k_tok < 0 || h.k_head < 0 || h.v_page < 0 || h.v_tok < 0 || h.v_head < 0) return PRISM_ERR_SHAPE;
    // a token's offset within 16 of them is a 32-bit number of bytes
    if (h.k_tok > (1 << 26) || h.v_tok > (1 << 26)) return PRISM_ERR_SHAPE;
    if (!PRISM_ALIGNED(h.k, 16) || !PRISM_ALIGNED(h.v, 16) || h.k_page % unit || h.k_tok % unit || h.k_head % unit ||
        h.v_page % unit || h.v_tok % unit || h.v_head % unit)
        return PRISM_ERR_ALIGN;
    int shift = 0;
    while ((1 << shift) < h.page) shift++;
    c = Cache{(char*)h.k, (char*)h.v, h.k_page * size, h.k_tok * size, h.k_head * size, h.v_page * size, h.v_tok * size,
              h.v_head * size, h.k_scale, h.v_scale, h.table, h.table_ld, (int)h.seqs, (int)h.cols, (int)h.pages, shift};
    return PRISM_OK;
}

}  // namespace prism

using namespace prism;

extern "C" int prism_kv_append(const prism_kv_append_args* args, void* stream) {
    if (!args) return PRISM_ERR_ARG;
    const prism_kv_append_args& h = *args;
    AppendArgs a{};
    const int rc = make_cache(a.c, h.cache);
    if (rc != PRISM_OK) return rc;
    const int64_t D = h.cache.dim, HKV = h.cache.heads;
    if (!h.k || !h.v || !h.pos || !h.n_rows || (h.hq > 0 && (!h.q || !h.q_out)) || (h.rot > 0 && !h.rope))
        return PRISM_ERR_ARG;
    if (h.adjacent != 0 && h.adjacent != 1) return PRISM_ERR_ARG;
    if (h.T < 0 || h.T > INT32_MAX || h.hq < 0 || h.hq > 65536 || h.rot < 0 || h.rot > D || h.rot % 16)
        return PRISM_ERR_SHAPE;
    if (h.rot > 0 && (h.ldr < h.rot || h.rope_rows < 1)) return PRISM_ERR_SHAPE;
    if (!PRISM_ALIGNED(h.k, 16) || !PRISM_ALIGNED(h.v, 16) || h.k_ld % 8 || h.k_hs % 8 || h.v_ld % 8 || h.v_hs % 8)
        return PRISM_ERR_ALIGN;
    if (h.hq > 0 && (!PRISM_ALIGNED(h.q, 16) || !PRISM_ALIGNED(h.q_out, 16) || h.q_ld % 8 || h.q_hs % 8 || h.o_ld % 8 ||
                     h.o_hs % 8))
        return PRISM_ERR_ALIGN;
    if (h.rot > 0 && (!PRISM_ALIGNED(h.rope, 16) || h.ldr % 4)) return PRISM_ERR_ALIGN;
    if (h.T == 0) return PRISM_OK;
    a.q = h.q, a.k = h.k, a.v = h.v, a.qo = h.q_out;
    a.ldq = h.q_ld, a.hq_s = h.q_hs, a.ldk = h.k_ld, a.hk_s = h.k_hs, a.ldv = h.v_ld, a.hv_s = h.v_hs;
    a.ldo = h.o_ld, a.ho_s = h.o_hs;
    a.rope = h.rope, a.ldr = h.ldr, a.pos = h.pos, a.seq = h.seq, a.n = h.n_rows;
    a.rope_rows = (int)(h.rope_rows < INT32_MAX ? h.rope_rows : INT32_MAX);
    a.R = (int)h.rot, a.adjacent = (int)h.adjacent, a.HQ = (int)h.hq, a.HKV = (int)HKV;
    // whole waves, as few idle lanes as the rows' pieces allow
    const int64_t items = (h.hq + 2 * HKV) * (D / 16), rows = (items + 255) / 256;
    const int tpb = (int)(((items + rows - 1) / rows + 63) / 64 * 64);
    const dim3 grid((unsigned)h.T, (unsigned)((items + tpb - 1) / tpb));
    const hipStream_t st = (hipStream_t)stream;
#define AP(DD) \
    do { \
        if (h.cache.e4m3) hipLaunchKernelGGL((kv_append_kernel<DD, true>), grid, dim3(tpb), 0, st, a); \
        else hipLaunchKernelGGL((kv_append_kernel<DD, false>), grid, dim3(tpb), 0, st, a); \
    } while (0)
    if (D == 64) AP(64); else if (D == 128) AP(128); else AP(256);
#undef AP
    PRISM_LAUNCH_CHECK();
    return PRISM_OK;
}

extern "C" int64_t prism_kv_attend_workspace_bytes(int64_t T, int64_t hq, int64_t heads, int64_t dim, int64_t cols,
                                                   int64_t page) {
    if (T < 1 || heads < 1 || hq < heads || hq % heads || dim < 1 || cols < 1 || page < 1) return 0;
    // the most of both ways that the strides may choose, and of both cache types (512 workgroups)
    const int64_t cap = cols * page, tiles = (hq / heads + 15) / 16;
    int64_t parts = cap <= 32 * kWaves ? 0 : attend_parts(T, heads * tiles, cap, 32 * kWaves, 512);
    if (attend_side(T, hq, heads, cap)) {
        const int64_t side = attend_parts(T, heads / 4, cap, 32, 512);
        if (side > parts) parts = side;
    }
    return parts ? 2 * parts * hq * (dim + 2) * 4 + T * 8 : 0;     // 0: one unit a sequence, nothing to join
}

extern "C" int prism_kv_attend(const prism_kv_attend_args* args, void* stream) {
    if (!args) return PRISM_ERR_ARG;
    const prism_kv_attend_args& h = *args;
    const int64_t T = h.cache.seqs, HQ = h.hq, HKV = h.cache.heads, D = h.cache.dim, cols = h.cache.cols;
    if (T < 0 || T > 65535) return PRISM_ERR_SHAPE;
    AttendArgs a{};
    prism_kv_cache hc = h.cache;
    hc.seqs = T > 0 ? T : 1;
    const int rc = make_cache(a.c, hc);
    if (rc != PRISM_OK) return rc;
    if (!h.q || !h.lens || !h.out || !h.n_rows) return PRISM_ERR_ARG;
    if (HQ < HKV || HQ % HKV || HQ > 65535 || h.window < 0 || cols * hc.page > INT32_MAX - 65536) return PRISM_ERR_SHAPE;
    if (!PRISM_ALIGNED(h.q, 16) || !PRISM_ALIGNED(h.out, 8) || h.q_ld % 8 || h.q_hs % 8 || h.o_ld % 4 || h.o_hs % 4)
        return PRISM_ERR_ALIGN;
    const int64_t need = prism_kv_attend_workspace_bytes(T, HQ, HKV, D, cols, hc.page);
    if (need > 0 && (!h.ws || h.ws_bytes < need)) return PRISM_ERR_ARG;
    if (need > 0 && !PRISM_ALIGNED(h.ws, 16)) return PRISM_ERR_ALIGN;
    if (T == 0) return PRISM_OK;
    const int64_t G = HQ / HKV, tiles = (G + 15) / 16, cap = cols * hc.page;
    const bool f8 = hc.e4m3 != 0;
    const bool side = hc.k_head < hc.k_tok && hc.v_head < hc.v_tok && attend_side(T, HQ, HKV, cap);
    const int64_t HT = side ? HKV / 4 : HKV * tiles, unit = side ? 32 : 32 * kWaves;
    a.target = attend_target(D, f8);
    const int64_t parts = attend_parts(T, HT, cap, unit, a.target), grid = (parts + 7) / 8 * 8 * HT;
    if (grid > INT32_MAX) return PRISM_ERR_SHAPE;
    a.q = h.q, a.out = h.out, a.ldq = h.q_ld, a.hq_s = h.q_hs, a.ldo = h.o_ld, a.ho_s = h.o_hs;
    a.lens = h.lens, a.n = h.n_rows;
    const bool joins = cap > unit;
    if (joins) {
        a.part_o = (float*)h.ws;
        a.part_ml = (float*)h.ws + 2 * parts * HQ * D;
        a.plan = (int2*)((float*)h.ws + 2 * parts * HQ * (D + 2));
    }
    a.scale = (float)h.scale * 1.44269504088896340736f;
    a.T = (int)T, a.HQ = (int)HQ, a.G = (int)G, a.tiles = (int)tiles, a.HT = (int)HT;
    a.window = (int)(h.window < INT32_MAX ? h.window : 0);
    const hipStream_t st = (hipStream_t)stream;
#define AT(DD, F8) \
    do { \
        static_assert(Block<DD, F8>::STAGE % 16 == 0, "LDS alignment"); \
        const int lds = attend_lds(DD, F8); \
        if (side) { \
            allow_lds(kv_attend_kernel<DD, F8, true>, lds); \
            hipLaunchKernelGGL((kv_attend_kernel<DD, F8, true>), dim3((unsigned)grid), dim3(256), lds, st, a); \
        } else { \
            allow_lds(kv_attend_kernel<DD, F8, false>, lds); \
            hipLaunchKernelGGL((kv_attend_kernel<DD, F8, false>), dim3((unsigned)grid), dim3(256), lds, st, a); \
        } \
    } while (0)
    if (D == 64) { if (f8) AT(64, true); else AT(64, false); }
    else if (D == 128) { if (f8) AT(128, true); else AT(128, false); }
    else { if (f8) AT(256, true); else AT(256, false); }
#undef AT
    PRISM_LAUNCH_CHECK();
    if (joins) {
        // a workgroup per head while there are few (long sequences have many parts), else one for a quarter as many as
        // it has groups: 128 sequences of 64 heads of 64 take 124 - 127 us in all, 130 with half as many, 137 with as
        // many (a chain of loads after the other), 131 with one
        const int hb = T * HQ <= 4096 ? 1 : (int)(256 / D);
        const dim3 jg((unsigned)((HQ + hb - 1) / hb), (unsigned)T);
        if (D == 64) hipLaunchKernelGGL(kv_join_kernel<64>, jg, dim3(256), 0, st, a, hb);
        else if (D == 128) hipLaunchKernelGGL(kv_join_kernel<128>, jg, dim3(256), 0, st, a, hb);
        else hipLaunchKernelGGL(kv_join_kernel<256>, jg, dim3(256), 0, st, a, hb);
        PRISM_LAUNCH_CHECK();
    }
    return PRISM_OK;
}
