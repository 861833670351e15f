// The paged key-value cache of a full-attention layer in serving (gfx950): new tokens' keys and values into the cache
// with the position rotation on the way (append), and one new token per sequence attending to its cache (attend).
//
// The cache is [pages, page, heads, dim] of bf16 or e4m3 with any strides of its first three dims, so both memory
// orders in use (token rows of all heads, or a page's rows of one head together) are the same code.  A page table
// int32 [sequences, columns] names the pages of a sequence: token t lies in row t % page of page table[s][t / page].
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
// A thread takes 16 dims of one head as two pieces of 8 that a rotation in halves pairs: dims 8 j .. + 7 and
// R / 2 + 8 j .. + 7 of the R rotated ones, the same split of the others.  Every piece is one 16-byte load, 16 bytes
// (8 of e4m3) stored; neighbouring lanes hold neighbouring pieces.  One workgroup row per token (blockIdx.x), the
// token's heads (queries, keys, values) over blockIdx.y.  Bound by memory: nothing is read or written twice.
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
    const v4u u = *reinterpret_cast<const v4u*>(p);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        f[2 * j] = __uint_as_float(u[j] << 16);
        f[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
    }
}

__device__ __forceinline__ void store8_bf16(void* p, const float* f) {
    v4u u;
#pragma unroll
    for (int j = 0; j < 4; j++) u[j] = f32_to_bf16(f[2 * j]) | (f32_to_bf16(f[2 * j + 1]) << 16);
    *reinterpret_cast<v4u*>(p) = u;
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
    *reinterpret_cast<v2u*>(p) = v2u{w[0], w[1]};
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
        store8_bf16(d + o0, x);
        store8_bf16(d + o1, y);
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
        store8_bf16(d + 2 * o0, x);
        store8_bf16(d + 2 * o1, y);
    }
}

// ------------------------------------------------------------------------------------------------------------ attend
// o[h] = sum_t softmax_t(scale q_h . k_t) v_t over a sequence's visible tokens, all query heads of one key head
// together (they read the same keys and values), in one pass with a running maximum and sum per query head.
//
// A wave takes blocks of 32 tokens with no LDS: scores transposed, S^T = K Q^T (the keys as the MFMA's first operand,
// query heads its 16 columns), leave each lane the scores of ITS head (lane % 16) for tokens 4 g + r and 16 + 4 g + r
// (g = lane / 16, r < 4).  O^T = V^T P^T wants in each lane 8 tokens of its head as second operand, and the order of
// the 32 tokens along the product is free as long as both operands agree: taking them as the scores lie, P never
// leaves its lane, and neither do the maximum, the sum and the rescaling of O^T's columns (all of head lane % 16).
// V's operand needs 8 tokens of one dim per lane: a lane loads its 8 tokens' rows in pieces of D / 16 dims (16 lanes
// a whole row, contiguous) and turns the 8 x D/16 block with one v_perm per register.
// P is split into two bf16 parts (truncated, then the rest), so the weights carry 16 bits and the output's one bf16
// rounding is the only one that shows; the second MFMA is free beside the cache's bytes.
//
// Work is split on the device, from the lengths (a captured launch serves every batch): a unit is what the four waves
// take in one round; `per` units to a workgroup bring the batch to about kTarget workgroups; a sequence gets
// max(1, ceil(units / per)) of them, shared evenly.  Sequences with one workgroup write their output; the others'
// parts are joined by a second kernel in a fixed order, so results do not depend on timing.
struct AttendArgs {
    const uint16_t* q;
    uint16_t* out;
    int64_t ldq, hq_s, ldo, ho_s;
    const int32_t *lens, *n;
    float* part_o;                                            // [P, HQ, D]
    float* part_ml;                                           // [P, HQ, 2]
    float scale;                                              // times log2 e
    int T, HQ, G, tiles, HT, window, target;
    Cache c;
};

constexpr int kWaves = 4;

struct Plan {
    int b, lo, len, begin, end, split, splits, first;         // first: index of the sequence's first part
};

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

// Work of part p (b < 0: none), or with p < 0 sequence `want`'s parts; the same in every lane.
template <int UNIT>
__device__ __forceinline__ Plan make_plan(const AttendArgs& a, int p, int want) {
    const int lane = threadIdx.x & 63;
    const int n = min(__ldg(a.n), a.T);
    int lo, len;
    long long sum = 0;
    for (int b = lane; b < n; b += 64) sum += vis_units<UNIT>(a, __ldg(a.lens + b), &lo, &len);
    const long long total = wave_sum(sum);
    const int per = max((int)((total * a.HT + a.target - 1) / a.target), 1);
    int base = 0;
    Plan r;
    r.b = -1;
    for (int b0 = 0; b0 < n; b0 += 64) {
        const int b = b0 + lane;
        int units = 0, nb = 0;
        lo = len = 0;
        if (b < n) {
            units = vis_units<UNIT>(a, __ldg(a.lens + b), &lo, &len);
            nb = max(1, (units + per - 1) / per);
        }
        int incl = nb;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int up = __shfl_up(incl, o, kWave);
            if (lane >= o) incl += up;
        }
        const int tot = __shfl(incl, 63, kWave);
        const int mine = base + incl - nb;                    // first part of this lane's sequence
        const bool hit = p < 0 ? b == want : nb > 0 && p >= mine && p < mine + nb;
        const uint64_t m = __ballot(hit);
        if (m) {
            const int src = __builtin_ctzll(m);
            const int u = __shfl(units, src, kWave), k = __shfl(nb, src, kWave);
            r.b = b0 + src;
            r.lo = __shfl(lo, src, kWave);
            r.len = __shfl(len, src, kWave);
            r.first = __shfl(mine, src, kWave);
            r.splits = k;
            r.split = p - r.first;
            const int each = u / k, more = u % k;             // the first `more` parts take one unit more
            const int ub = r.split * each + min(r.split, more);
            r.begin = (r.lo & ~15) + ub * UNIT;
            r.end = min(r.len, (int)min((int64_t)r.begin + (int64_t)(each + (r.split < more)) * UNIT, (int64_t)INT32_MAX));
            break;
        }
        base += tot;
    }
    return r;
}

template <typename V>
__device__ __forceinline__ V ld(const char* base, uint32_t off) {
    return *reinterpret_cast<const V*>(base + off);
}

__device__ __forceinline__ v8bf as_bf(v4u x) { return __builtin_bit_cast(v8bf, x); }
__device__ __forceinline__ v4f mfma_bf16(v4u a, v4u b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(a), as_bf(b), c, 0, 0, 0);
}
// Two e4m3 bytes (SEL: the upper two) as two bf16, exactly.
template <bool SEL>
__device__ __forceinline__ uint32_t e4m3x2_bf16(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, SEL));
}

// Registers of one 32-token block's keys and values, and the loads that fill them.
template <int D, bool F8>
struct Block {
    static constexpr int KL = F8 ? D / 64 : D / 32;           // 16-byte key loads per 16 tokens and lane
    static constexpr int VB = (F8 ? 1 : 2) * D / 16;          // value bytes per token and lane
    static constexpr int VW = VB / 4;                         // 4, 8 or 16 bytes a load (two of 16 for 32)
    v4u k[2][KL];
    uint32_t v[2][4][VW];
};

template <int D, bool F8>
__device__ __forceinline__ void load_k(Block<D, F8>& s, int a, const char* base, uint32_t off) {
#pragma unroll
    for (int i = 0; i < Block<D, F8>::KL; i++) s.k[a][i] = ld<v4u>(base, off + 64 * i);
}

template <int D, bool F8>
__device__ __forceinline__ void load_v(Block<D, F8>& s, int a, const char* base, uint32_t off, uint32_t step) {
    constexpr int VW = Block<D, F8>::VW;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        if constexpr (VW == 1) {
            s.v[a][r][0] = ld<uint32_t>(base, off + r * step);
        } else if constexpr (VW == 2) {
            const v2u x = ld<v2u>(base, off + r * step);
            s.v[a][r][0] = x[0], s.v[a][r][1] = x[1];
        } else {
#pragma unroll
            for (int i = 0; i < VW / 4; i++) {                // dims 8 c .. and 128 + 8 c .. of 256 bf16
                const v4u x = ld<v4u>(base, off + r * step + 256 * i);
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

template <int D, bool F8>
__global__ __launch_bounds__(256, 2) void kv_attend_kernel(AttendArgs a) {
    constexpr int UNIT = 32 * kWaves, F = D / 16, QF = D / 32;
    extern __shared__ float lds[];                            // [4][16][D + 4] O, then [4][16] m, [4][16] l
    const int ht = blockIdx.x % a.HT, part = blockIdx.x / a.HT;
    const Plan pl = make_plan<UNIT>(a, part, 0);
    if (pl.b < 0) return;
    const int hk = ht / a.tiles, tile = ht % a.tiles;
    const int h0 = hk * a.G + 16 * tile, nh = min(16, a.G - 16 * tile);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int b = __builtin_amdgcn_readfirstlane(pl.b), len = __builtin_amdgcn_readfirstlane(pl.len);
    const int lo = __builtin_amdgcn_readfirstlane(pl.lo), end = __builtin_amdgcn_readfirstlane(pl.end);
    const int begin = __builtin_amdgcn_readfirstlane(pl.begin);

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

    const int32_t* row = a.c.table + b * a.c.table_ld;
    const int last = len > 0 ? (len - 1) & ~15 : 0;           // the last 16 tokens that are there
    const uint32_t koff = (uint32_t)(col * a.c.k_tok) + 16 * g;
    const uint32_t voff = (uint32_t)(4 * g * a.c.v_tok) + (D == 256 && !F8 ? 16 : Block<D, F8>::VB) * col;
    const char* kb = a.c.k + hk * a.c.k_head;
    const char* vb = a.c.v + hk * a.c.v_head;

    for (int t0 = begin + 32 * wave; t0 < end; t0 += UNIT) {
        Block<D, F8> s;
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const int t = min(t0 + 16 * x, last);             // 16 tokens never cross a page
            const int64_t page = min(max(row[t >> a.c.shift], 0), a.c.pages - 1), at = t & ((1 << a.c.shift) - 1);
            load_k<D, F8>(s, x, kb + page * a.c.k_page + at * a.c.k_tok, koff);
            load_v<D, F8>(s, x, vb + page * a.c.v_page + at * a.c.v_tok, voff, (uint32_t)a.c.v_tok);
        }
        v4f st[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int i = 0; i < QF; i++) {
                v4u kf;
                if constexpr (F8) {
                    const uint32_t w0 = s.k[x][i / 2][2 * (i % 2)], w1 = s.k[x][i / 2][2 * (i % 2) + 1];
                    kf = v4u{e4m3x2_bf16<false>(w0), e4m3x2_bf16<true>(w0), e4m3x2_bf16<false>(w1),
                             e4m3x2_bf16<true>(w1)};
                } else {
                    kf = s.k[x][i];
                }
                st[x] = mfma_bf16(kf, qf[i], st[x]);
            }
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; j++) p[j] = mul_rn(st[j / 4][j % 4], sc);
        if (t0 < lo || t0 + 32 > len) {
            // tokens outside get no weight, and their values, which may be anything (a page's unwritten rows), are zeroed
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int t = t0 + 16 * (j / 4) + 4 * g + j % 4;
                const bool in = t >= lo && t < len;
                p[j] = in ? p[j] : -INFINITY;
#pragma unroll
                for (int w = 0; w < Block<D, F8>::VW; w++) s.v[j / 4][j % 4][w] = in ? s.v[j / 4][j % 4][w] : 0;
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
        uint32_t hi[4], lw[4];
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float e0 = __builtin_amdgcn_exp2f(p[2 * w] - ref), e1 = __builtin_amdgcn_exp2f(p[2 * w + 1] - ref);
            l += e0 + e1;
            // the upper part strictly below the weight, so that the rest of a weight is never 0 (0 times an infinite
            // value would be NaN, not infinite)
            const uint32_t b0 = max(__float_as_uint(e0), 1u) - 1u, b1 = max(__float_as_uint(e1), 1u) - 1u;
            hi[w] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
            const float r0 = e0 - __uint_as_float(b0 & 0xffff0000u), r1 = e1 - __uint_as_float(b1 & 0xffff0000u);
            lw[w] = __builtin_amdgcn_perm(__float_as_uint(r1), __float_as_uint(r0), 0x07060302u);
        }
        const v4u ph = {hi[0], hi[1], hi[2], hi[3]}, plo = {lw[0], lw[1], lw[2], lw[3]};
#pragma unroll
        for (int q = 0; q < F / 4; q++) {
            v4u vf[4];
            turn_v<D, F8>(s, q, vf);
#pragma unroll
            for (int f = 0; f < 4; f++) {
                o[4 * q + f] = mfma_bf16(vf[f], ph, o[4 * q + f]);
                o[4 * q + f] = mfma_bf16(vf[f], plo, o[4 * q + f]);
            }
        }
    }

    // the four waves' columns, joined: each to the common maximum
    constexpr int LD = D + 4;
    float* lm = lds + kWaves * 16 * LD;
    float* ll = lm + kWaves * 16;
    l += __shfl_xor(l, 16, kWave);
    l += __shfl_xor(l, 32, kWave);
    if (lane < 16) {
        lm[wave * 16 + lane] = m;
        ll[wave * 16 + lane] = l;
    }
    float* mine = lds + (wave * 16 + col) * LD;
#pragma unroll
    for (int f = 0; f < F; f++)
#pragma unroll
        for (int r = 0; r < 4; r++) mine[dim_of<D, F8>(f, 4 * g + r)] = o[f][r];
    __syncthreads();
    const float vs = F8 && a.c.v_scale ? __ldg(a.c.v_scale + hk) : 1.f;
    for (int i = threadIdx.x; i < nh * (D / 4); i += 256) {
        const int h = i / (D / 4), d = 4 * (i % (D / 4));
        float mm = lm[h];
#pragma unroll
        for (int w = 1; w < kWaves; w++) mm = fmaxf(mm, lm[16 * w + h]);
        const float ref = mm == -INFINITY ? 0.f : mm;
        float sum = 0.f;
        v4f acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const float e = __builtin_amdgcn_exp2f(lm[16 * w + h] - ref);
            sum += e * ll[16 * w + h];
            acc += e * *reinterpret_cast<const v4f*>(lds + (w * 16 + h) * LD + d);
        }
        if (pl.splits == 1) {
            uint32_t u[4];
#pragma unroll
            for (int j = 0; j < 4; j++) u[j] = f32_to_bf16(sum == 0.f ? 0.f : div_rn(acc[j], sum) * vs);
            *reinterpret_cast<v2u*>(a.out + b * a.ldo + (h0 + h) * a.ho_s + d) = v2u{u[0] | (u[1] << 16), u[2] | (u[3] << 16)};
        } else {
            const int64_t at = (int64_t)part * a.HQ + h0 + h;
            *reinterpret_cast<v4f*>(a.part_o + at * D + d) = acc;
            if (d == 0) {
                a.part_ml[2 * at] = mm;
                a.part_ml[2 * at + 1] = sum;
            }
        }
    }
}

// Joins the parts of sequence blockIdx.y, query head blockIdx.x: 256 threads as 1024 / D groups of D / 4, each group
// every 1024 / D-th part, then the groups in order.
template <int D>
__global__ __launch_bounds__(256) void kv_join_kernel(AttendArgs a) {
    constexpr int UNIT = 32 * kWaves, TC = D / 4, NG = 256 / TC;
    __shared__ float lds[NG][D + 4];
    __shared__ float red[NG];
    const int h = blockIdx.x, b = blockIdx.y;
    const Plan pl = make_plan<UNIT>(a, -1, b);
    if (pl.b < 0 || pl.splits < 2) return;
    const int64_t first = (int64_t)pl.first * a.HQ + h;
    float mm = -INFINITY;
    for (int i = threadIdx.x & 63; i < pl.splits; i += 64) mm = fmaxf(mm, a.part_ml[2 * (first + (int64_t)i * a.HQ)]);
    mm = wave_max(mm);
    const float ref = mm == -INFINITY ? 0.f : mm;
    const int c = threadIdx.x % TC, grp = threadIdx.x / TC;
    v4f acc = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
    for (int i = grp; i < pl.splits; i += NG) {
        const int64_t at = first + (int64_t)i * a.HQ;
        const float e = __builtin_amdgcn_exp2f(a.part_ml[2 * at] - ref);
        sum += e * a.part_ml[2 * at + 1];
        acc += e * *reinterpret_cast<const v4f*>(a.part_o + at * D + 4 * c);
    }
    *reinterpret_cast<v4f*>(&lds[grp][4 * c]) = acc;
    if (c == 0) red[grp] = sum;
    __syncthreads();
    if (grp) return;
    for (int i = 1; i < NG; i++) {
        acc += *reinterpret_cast<const v4f*>(&lds[i][4 * c]);
        sum += red[i];
    }
    const int hk = h / a.G;
    const float vs = a.c.v_scale ? __ldg(a.c.v_scale + hk) : 1.f;
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; j++) u[j] = f32_to_bf16(sum == 0.f ? 0.f : div_rn(acc[j], sum) * vs);
    *reinterpret_cast<v2u*>(a.out + b * a.ldo + h * a.ho_s + 4 * c) = v2u{u[0] | (u[1] << 16), u[2] | (u[3] << 16)};
}

// Workgroups that a launch's work is split into, at most (beside one for each further sequence and head).
constexpr int kTarget = 512;

static int64_t attend_parts(int64_t T, int64_t HT, int64_t cap) {
    const int64_t unit = 32 * kWaves, most = T * ((cap + unit - 1) / unit);
    const int64_t split = kTarget / HT + 1 + T;
    return most < split ? most : split;
}

// The cache's arguments, checked; strides in elements.
static int make_cache(Cache& c, void* k, int64_t k_page, int64_t k_tok, int64_t k_head, void* v, int64_t v_page,
                      int64_t v_tok, int64_t v_head, int e4m3, const float* k_scale, const float* v_scale,
                      const int32_t* table, int64_t table_ld, int64_t seqs, int64_t cols, int64_t pages, int64_t page,
                      int64_t HKV, int64_t D) {
    if (!k || !v || !table || (e4m3 != 0 && e4m3 != 1)) return PRISM_ERR_ARG;
    if (!e4m3 && (k_scale || v_scale)) return PRISM_ERR_ARG;
    if (HKV < 1 || HKV > 65536 || (D != 64 && D != 128 && D != 256)) return PRISM_ERR_SHAPE;
    if (page < 16 || page > 65536 || (page & (page - 1)) || pages < 1 || pages > INT32_MAX) return PRISM_ERR_SHAPE;
    if (seqs < 1 || seqs > INT32_MAX || cols < 1 || cols > (1 << 27) || table_ld < cols) return PRISM_ERR_SHAPE;
    const int64_t size = e4m3 ? 1 : 2, unit = 16 / size;
    if (k_page < 0 || k_tok < 0 || k_head < 0 || v_page < 0 || v_tok < 0 || v_head < 0) return PRISM_ERR_SHAPE;
    // a token's offset within 16 of them is a 32-bit number of bytes
    if (k_tok > (1 << 26) || v_tok > (1 << 26)) return PRISM_ERR_SHAPE;
    if (!PRISM_ALIGNED(k, 16) || !PRISM_ALIGNED(v, 16) || k_page % unit || k_tok % unit || k_head % unit ||
        v_page % unit || v_tok % unit || v_head % unit)
        return PRISM_ERR_ALIGN;
    int shift = 0;
    while ((1 << shift) < page) shift++;
    c = Cache{(char*)k, (char*)v, k_page * size, k_tok * size, k_head * size, v_page * size, v_tok * size,
              v_head * size, k_scale, v_scale, table, table_ld, (int)seqs, (int)cols, (int)pages, shift};
    return PRISM_OK;
}

}  // namespace prism

using namespace prism;

extern "C" int prism_kv_append(const uint16_t* q, int64_t ldq, int64_t hq_s, const uint16_t* k, int64_t ldk,
                               int64_t hk_s, const uint16_t* v, int64_t ldv, int64_t hv_s, uint16_t* q_out, int64_t ldo,
                               int64_t ho_s, const float* rope, int64_t ldr, int64_t rope_rows, int64_t rot,
                               int adjacent, const int32_t* pos, const int32_t* seq, void* k_cache, int64_t k_page,
                               int64_t k_tok, int64_t k_head, void* v_cache, int64_t v_page, int64_t v_tok,
                               int64_t v_head, int e4m3, const float* k_scale, const float* v_scale,
                               const int32_t* table, int64_t table_ld, int64_t seqs, int64_t cols, int64_t pages,
                               int64_t page, const int32_t* n_rows, int64_t T, int64_t HQ, int64_t HKV, int64_t D,
                               void* stream) {
    AppendArgs a{};
    const int rc = make_cache(a.c, k_cache, k_page, k_tok, k_head, v_cache, v_page, v_tok, v_head, e4m3, k_scale,
                              v_scale, table, table_ld, seqs, cols, pages, page, HKV, D);
    if (rc != PRISM_OK) return rc;
    if (!k || !v || !pos || !n_rows || (HQ > 0 && (!q || !q_out)) || (rot > 0 && !rope)) return PRISM_ERR_ARG;
    if (adjacent != 0 && adjacent != 1) return PRISM_ERR_ARG;
    if (T < 0 || T > INT32_MAX || HQ < 0 || HQ > 65536 || rot < 0 || rot > D || rot % 16) return PRISM_ERR_SHAPE;
    if (rot > 0 && (ldr < rot || rope_rows < 1)) return PRISM_ERR_SHAPE;
    if (!PRISM_ALIGNED(k, 16) || !PRISM_ALIGNED(v, 16) || ldk % 8 || hk_s % 8 || ldv % 8 || hv_s % 8)
        return PRISM_ERR_ALIGN;
    if (HQ > 0 && (!PRISM_ALIGNED(q, 16) || !PRISM_ALIGNED(q_out, 16) || ldq % 8 || hq_s % 8 || ldo % 8 || ho_s % 8))
        return PRISM_ERR_ALIGN;
    if (rot > 0 && (!PRISM_ALIGNED(rope, 16) || ldr % 4)) return PRISM_ERR_ALIGN;
    if (T == 0) return PRISM_OK;
    a.q = q, a.k = k, a.v = v, a.qo = q_out;
    a.ldq = ldq, a.hq_s = hq_s, a.ldk = ldk, a.hk_s = hk_s, a.ldv = ldv, a.hv_s = hv_s, a.ldo = ldo, a.ho_s = ho_s;
    a.rope = rope, a.ldr = ldr, a.pos = pos, a.seq = seq, a.n = n_rows;
    a.rope_rows = (int)(rope_rows < INT32_MAX ? rope_rows : INT32_MAX);
    a.R = (int)rot, a.adjacent = adjacent, a.HQ = (int)HQ, a.HKV = (int)HKV;
    // whole waves, as few idle lanes as the rows' pieces allow
    const int64_t items = (HQ + 2 * HKV) * (D / 16), rows = (items + 255) / 256;
    const int tpb = (int)(((items + rows - 1) / rows + 63) / 64 * 64);
    const dim3 grid((unsigned)T, (unsigned)((items + tpb - 1) / tpb));
    const hipStream_t st = (hipStream_t)stream;
#define AP(DD) \
    do { \
        if (e4m3) hipLaunchKernelGGL((kv_append_kernel<DD, true>), grid, dim3(tpb), 0, st, a); \
        else hipLaunchKernelGGL((kv_append_kernel<DD, false>), grid, dim3(tpb), 0, st, a); \
    } while (0)
    if (D == 64) AP(64); else if (D == 128) AP(128); else AP(256);
#undef AP
    PRISM_LAUNCH_CHECK();
    return PRISM_OK;
}

static int64_t attend_bytes(int64_t T, int64_t HQ, int64_t HKV, int64_t D, int64_t cap) {
    const int64_t G = HQ / HKV, HT = HKV * ((G + 15) / 16);
    return attend_parts(T, HT, cap) * HQ * (D + 2) * 4;
}

extern "C" int64_t prism_kv_attend_workspace_bytes(int64_t T, int64_t HQ, int64_t HKV, int64_t D, int64_t cols,
                                                   int64_t page) {
    if (T < 1 || HKV < 1 || HQ < HKV || HQ % HKV || D < 1 || cols < 1 || page < 1) return 0;
    if (cols * page <= 32 * kWaves) return 0;                // one unit: nothing to join
    return attend_bytes(T, HQ, HKV, D, cols * page);
}

extern "C" int prism_kv_attend(const uint16_t* q, int64_t ldq, int64_t hq_s, const void* k_cache, int64_t k_page,
                               int64_t k_tok, int64_t k_head, const void* v_cache, int64_t v_page, int64_t v_tok,
                               int64_t v_head, int e4m3, const float* k_scale, const float* v_scale,
                               const int32_t* table, int64_t table_ld, int64_t cols, int64_t pages, int64_t page,
                               const int32_t* lens, uint16_t* out, int64_t ldo, int64_t ho_s, const int32_t* n_rows,
                               int64_t T, int64_t HQ, int64_t HKV, int64_t D, float scale, int64_t window, void* ws,
                               int64_t ws_bytes, void* stream) {
    AttendArgs a{};
    if (T < 0 || T > 65535) return PRISM_ERR_SHAPE;
    const int rc = make_cache(a.c, const_cast<void*>(k_cache), k_page, k_tok, k_head, const_cast<void*>(v_cache), v_page,
                              v_tok, v_head, e4m3, k_scale, v_scale, table, table_ld, T > 0 ? T : 1, cols, pages, page,
                              HKV, D);
    if (rc != PRISM_OK) return rc;
    if (!q || !lens || !out || !n_rows) return PRISM_ERR_ARG;
    if (HQ < HKV || HQ % HKV || HQ > 65535 || window < 0 || cols * page > INT32_MAX - 65536) return PRISM_ERR_SHAPE;
    if (!PRISM_ALIGNED(q, 16) || !PRISM_ALIGNED(out, 8) || ldq % 8 || hq_s % 8 || ldo % 4 || ho_s % 4)
        return PRISM_ERR_ALIGN;
    const int64_t need = prism_kv_attend_workspace_bytes(T, HQ, HKV, D, cols, page);
    if (T > 0 && need > 0 && (!ws || ws_bytes < need)) return PRISM_ERR_ARG;
    if (need > 0 && !PRISM_ALIGNED(ws, 16)) return PRISM_ERR_ALIGN;
    if (T == 0) return PRISM_OK;
    const int64_t G = HQ / HKV, tiles = (G + 15) / 16, HT = HKV * tiles;
    const int64_t parts = attend_parts(T, HT, cols * page);
    if (parts * HT > INT32_MAX) return PRISM_ERR_SHAPE;
    a.q = q, a.out = out, a.ldq = ldq, a.hq_s = hq_s, a.ldo = ldo, a.ho_s = ho_s, a.lens = lens, a.n = n_rows;
    a.part_o = (float*)ws;
    a.part_ml = (float*)ws + parts * HQ * D;
    a.scale = scale * 1.44269504088896340736f;
    a.T = (int)T, a.HQ = (int)HQ, a.G = (int)G, a.tiles = (int)tiles, a.HT = (int)HT, a.target = kTarget;
    a.window = (int)(window < INT32_MAX ? window : 0);
    const hipStream_t st = (hipStream_t)stream;
    const size_t lds = (size_t)(kWaves * 16 * (D + 4) + 2 * kWaves * 16) * 4;
#define AT(DD, F8) \
    do { \
        allow_lds(kv_attend_kernel<DD, F8>, lds); \
        hipLaunchKernelGGL((kv_attend_kernel<DD, F8>), dim3((unsigned)(parts * HT)), dim3(256), lds, st, a); \
    } while (0)
    if (D == 64) { if (e4m3) AT(64, true); else AT(64, false); }
    else if (D == 128) { if (e4m3) AT(128, true); else AT(128, false); }
    else { if (e4m3) AT(256, true); else AT(256, false); }
#undef AT
    PRISM_LAUNCH_CHECK();
    if (need > 0) {
        const dim3 grid((unsigned)HQ, (unsigned)T);
        if (D == 64) hipLaunchKernelGGL(kv_join_kernel<64>, grid, dim3(256), 0, st, a);
        else if (D == 128) hipLaunchKernelGGL(kv_join_kernel<128>, grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL(kv_join_kernel<256>, grid, dim3(256), 0, st, a);
        PRISM_LAUNCH_CHECK();
    }
    return PRISM_OK;
}
