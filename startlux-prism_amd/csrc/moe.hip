// A mixture-of-experts layer for a few tokens on gfx950: the router's choice and the experts on e4m3 weights with block scales
// (fp8.hip's chunks), bf16 activations.
//
//   route     ids[t], w[t]: the top experts of a row of logits and their weights
//   experts   out[t] = sum_j w[t][j] down_e (silu(gate_e x_t) * (up_e x_t)),  e = ids[t][j]
//
// For a few tokens the experts' weights, read once, are the work: a chunk (16 rows x 128 inputs, 2 KB) is loaded straight
// into registers, several ahead, its codes become bf16 (exact) two at a time, and v_mfma_f32_16x16x32_bf16 multiplies them
// with up to 16 tokens' columns, four products per chunk chained from zero, then one fma by the block's scale into the fp32
// sum.  Which pairs (token, place) an expert has is found by every workgroup from the ids with ballots: no sorting launch.
//
// Three launches per 128 tokens.  moe_up_kernel leaves the hidden values h = silu(g) u of each pair in the workspace as two
// bf16 parts (h = hi + lo up to 2^-17 of it: the second product's operand; one part alone would add as much error as the bf16
// output's own rounding), moe_down_kernel each pair's outputs in fp32, moe_sum_kernel adds a token's in the order of its ids:
// no atomics, and what a token gets depends on the others only in the order of its fp32 sums, by T and the sizes (how K is split,
// and whether a hidden value's two parts are summed apart).
//
// The weights' bytes bound it: 64 tokens on 8 of 128 experts (H 2048, I 768; 594 MB) up 66, down 40, sum 4.6 us, 109 in all (5.5
// TB/s; memory read alone runs at 6.0); 11 tokens on 2 of 16 (5120, 1408; 265 MB) 29, 15 and 4.6, 45-51 in all; one token on 8 of 128
// (38 MB) 7.2, 4.7 and 2.9, 15.1 in all: three launches and their first loads.  Loads count by their number too: a ring's last round
// that asked past the end made these 115, 64 and 17.2.  Measured and dropped: the outputs of all experts summed by one workgroup per
// 16 outputs (64 tokens: down 160 us), or for one token a wave per pair (12 us against 5 + 2.5: each CU then goes to eight experts'
// pages); experts dealt out over the XCDs (no change, 11 tokens 75 against 62).
#include <math.h>

#include <type_traits>

#include "common.h"
#include "fp8.h"

namespace prism {

constexpr int kMoeTokens = 128;              // tokens per pass of the experts
constexpr int kMoeTop = 16;
constexpr int kWaves = 4;

// --------------------------------------------------------------------------------------------------------------- route
// An order-preserving integer of a number that may be chosen (greater than 0); 0 for NaN and -inf.
__device__ __forceinline__ uint32_t rank_of(float v) {
    const uint32_t u = __float_as_uint(v);
    if (v != v || u == 0xff800000u) return 0;
    const uint32_t z = u == 0x80000000u ? 0 : u;                              // -0 is 0
    return (z & 0x80000000u) ? ~z : z | 0x80000000u;
}
__device__ __forceinline__ uint64_t rank_of(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v), neg = 1ull << 63;
    if (v != v || u == 0xfff0000000000000ull) return 0;
    const uint64_t z = u == neg ? 0 : u;
    return (z & neg) ? ~z : z | neg;
}

struct RouteArgs {
    const void* x;
    int64_t x_ld;
    const float* bias;
    int32_t* ids;
    int64_t ids_ld;
    float* w;
    int64_t w_ld;
    const int32_t* n_rows;
    int T, E, top, renorm;
    float scale;
};

// The largest of the wave's values, by row shifts and broadcasts in the vector registers (a shuffle goes through the LDS unit:
// 18 of them per choice made the choices of 8 of 256 experts 18 of 20 us for 8191 tokens).
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#define PRISM_DPP_MAX(ctrl, rows) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xf, false))
    PRISM_DPP_MAX(0x111, 0xf);               // row_shr:1, 2, 4, 8: lane 15 of every 16 has their largest
    PRISM_DPP_MAX(0x112, 0xf);
    PRISM_DPP_MAX(0x114, 0xf);
    PRISM_DPP_MAX(0x118, 0xf);
    PRISM_DPP_MAX(0x142, 0xa);               // row_bcast:15 into rows 1 and 3, row_bcast:31 into rows 2 and 3
    PRISM_DPP_MAX(0x143, 0xc);
#undef PRISM_DPP_MAX
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// The number that a rank stands for.
__device__ __forceinline__ float of_rank(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }

// Whether no other fp32 number has x's sigmoid in 64 bits, so that logits order theirs beside x's: the next number's is at least
// (1 - p) 2^-24 |x| p away, 2^-49 p at 20 and 2^-45 p at +-2^-20, where exp (1 ulp), the sum and the division leave each within
// 2^-51 p; from -700 on exp(-x) does not overflow.
__device__ __forceinline__ bool sigmoids_apart(float x) { return x <= 20.f && x >= -700.f && fabsf(x) >= 0x1p-20f; }

// A wave per token, lane l holding experts l V .. l V + V - 1, so the lowest lane with the largest key, and in it the first, is
// the lowest number; top times the largest of all.
//
// Sigmoids are compared in 64 bits, but first in 32.  With a bias: p and p + bias in fp32 are within 2^-21 (1 + |p + bias|) of their
// values (expf's and three more roundings), so choices that lie further than 2^-19 (1 + |p + bias|) from the next are the same.
// Without one the logits are compared: they order the sigmoids unless a chosen one shares its 64-bit sigmoid with another logit
// (not sigmoids_apart).  Only where two sums are that close (one token in some thousand, and rows with equal ones) or a chosen
// logit is not apart, all 64-bit values are made and compared, their high halves first and the low ones between lanes that share
// them.  8191 tokens, 8 of 256: with a bias 12.7 us (13.7 all in 64 bits), without 8.4 (BIAS: 13.2 and 9.4 with one kernel for both),
// softmax 7.3.
template <int V, bool F32, bool SIG, bool BIAS>
__global__ __launch_bounds__(256) void moe_route_kernel(RouteArgs a) {
    kernel_args_now(a.x, a.x_ld, a.bias, a.ids, a.ids_ld, a.w, a.w_ld, a.n_rows, a.T, a.E, a.top, a.renorm, a.scale);
    const int t = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (t >= a.T) return;
    const int live = __ldg(a.n_rows);
    float x[V], bias[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int e = min(lane * V + i, a.E - 1);
        x[i] = F32 ? reinterpret_cast<const float*>(a.x)[t * a.x_ld + e]
                   : bf16_to_f32(reinterpret_cast<const uint16_t*>(a.x)[t * a.x_ld + e]);
        bias[i] = BIAS ? a.bias[e] : 0.f;
    }
    if (t >= live) return;
    uint32_t key[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        key[i] = rank_of(x[i]);
        if (BIAS && key[i]) key[i] = rank_of(add_rn(div_rn(1.f, add_rn(1.f, expf(-x[i]))), bias[i]));
        if (lane * V + i >= a.E) key[i] = 0;
    }
    int id = -1;                                                  // lane j: the j-th choice
    float lx = 0.f;                                               // and its logit
    bool sure = true;
    float last = 0.f;
    const int looks = a.top + (BIAS ? 1 : 0);            // (a bias: the next one too, which the last has to be clear of)
    for (int j = 0; j < looks; j++) {
        uint32_t best = key[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < V; i++)
            if (key[i] > best) best = key[i], at = i;
        const uint32_t most = wave_max_u32(best);
        if (most == 0) break;                                     // (none left)
        const int from = __builtin_ctzll(__ballot(best == most)), i0 = __builtin_amdgcn_readlane(at, from);
        float vx = x[0];
#pragma unroll
        for (int i = 0; i < V; i++) {
            if (i == i0) {
                vx = x[i];
                if (lane == from) key[i] = 0;
            }
        }
        vx = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(vx), from));
        if (SIG) {
            const float p = of_rank(most);
            if (BIAS ? j > 0 && !(last - p > 0x1p-19f * (1.f + fabsf(last))) : !sigmoids_apart(vx)) {
                sure = false;
                break;
            }
            last = p;
        }
        if (lane == j && j < a.top) id = from * V + i0, lx = vx;
    }
    if (SIG && !sure) {
        uint64_t wide[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            wide[i] = rank_of(x[i]) ? rank_of(1.0 / (1.0 + exp(-(double)x[i])) + (double)bias[i]) : 0;
            if (lane * V + i >= a.E) wide[i] = 0;
        }
        id = -1;
        for (int j = 0; j < a.top; j++) {
            uint64_t best = wide[0];
            int at = 0;
#pragma unroll
            for (int i = 1; i < V; i++)
                if (wide[i] > best) best = wide[i], at = i;
            const uint32_t hi = (uint32_t)(best >> 32), most = wave_max_u32(hi);
            if (most == 0) break;                                 // (a number's rank has a high half)
            uint64_t m = __ballot(hi == most);
            if (m & (m - 1)) {
                const uint32_t low = wave_max_u32(hi == most ? (uint32_t)best : 0u);
                m = __ballot(hi == most && (uint32_t)best == low);
            }
            const int from = __builtin_ctzll(m), i0 = __builtin_amdgcn_readlane(at, from);
            float vx = x[0];
#pragma unroll
            for (int i = 0; i < V; i++) {
                if (i == i0) {
                    vx = x[i];
                    if (lane == from) wide[i] = 0;
                }
            }
            vx = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(vx), from));
            if (lane == j) id = from * V + i0, lx = vx;
        }
    }
    float w = 0.f;
    if (SIG) {
        const double lp = 1.0 / (1.0 + exp(-(double)lx));
        double sum = 1.0;
        if (a.renorm) {
            sum = id >= 0 ? lp : 0.0;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);       // (top <= 16 lanes)
        }
        w = (float)(lp / sum * (double)a.scale);
    } else {
        const float m = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(lx)));       // the largest logit
        const float ex = id >= 0 ? expf(lx - m) : 0.f;
        float sum = 0.f;
        if (a.renorm) {
            sum = ex;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
        } else {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (lane * V + i < a.E) sum += expf(x[i] - m);
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
        }
        w = mul_rn(div_rn(ex, sum), a.scale);
    }
    if (lane < a.top) {
        a.ids[t * a.ids_ld + lane] = id;
        a.w[t * a.w_ld + lane] = id >= 0 ? w : 0.f;
    }
}

// ------------------------------------------------------------------------------------------------------------- experts
struct ExpertArgs {
    const uint16_t* x;
    int64_t x_ld;
    const int32_t* ids;
    int64_t ids_ld;
    const float* w;
    int64_t w_ld;
    const uint8_t *gate, *up, *down;
    const float *gate_s, *up_s, *down_s;
    uint16_t* h;                             // [pairs][2][128 KBI] bf16: the hidden values' parts
    float* y;                                // [pairs][H] fp32: the pairs' outputs
    void* out;
    int64_t o_ld;
    const int32_t* n_rows;
    int T, E, top, H, I, KBH, KBI;
    uint32_t div;                            // pair -> token: (pair div) >> 16 (pairs < 2048, top <= 16)
    int first, room;                         // the pass's tokens: room from first on
    int slots;                               // experts looked at per pass: all, or one per pair where those are fewer
    int vec;
};

// Every argument a kernel goes by in scalar registers at once: loaded where they are first used they come one memory round
// trip after another, which is most of a decode-size launch.
__device__ __forceinline__ void experts_now(const ExpertArgs& a) {
    kernel_args_now(a.x, a.x_ld, a.ids, a.ids_ld, a.w, a.w_ld, a.gate, a.up, a.down, a.gate_s, a.up_s, a.down_s, a.h, a.y, a.out,
                    a.n_rows);
    kernel_args_now(a.o_ld, a.T, a.E, a.top, a.H, a.I, a.KBH, a.KBI, a.div, a.first, a.room, a.slots, a.vec);
}

// The pass's live tokens (0 or less: none).  (A live count below zero is made zero first: less the pass's first token, the lowest
// ones would wrap to a full pass.)
__device__ __forceinline__ int pass_tokens(const ExpertArgs& a) {
    return __builtin_amdgcn_readfirstlane(min(max(min(a.T, __ldg(a.n_rows)), 0) - a.first, a.room));
}
__device__ __forceinline__ int token_of(const ExpertArgs& a, int pair) { return (int)((uint32_t)pair * a.div >> 16); }

// The expert of a pair of the pass; -1: none.
__device__ __forceinline__ int id_of(const ExpertArgs& a, int pair) {
    const int t = token_of(a, pair), e = a.ids[(a.first + t) * a.ids_ld + (pair - t * a.top)];
    return (uint32_t)e < (uint32_t)a.E ? e : -1;
}

// 16 e4m3 codes -> the bf16 fragments of their two 32-input products.
__device__ __forceinline__ void widen(v4i c, v8bf& lo, v8bf& hi) {
    v2bf t[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        t[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)c[i], 1.0f, false);
        t[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)c[i], 1.0f, true);
    }
    lo = __builtin_shufflevector(__builtin_shufflevector(t[0], t[1], 0, 1, 2, 3), __builtin_shufflevector(t[2], t[3], 0, 1, 2, 3),
                                 0, 1, 2, 3, 4, 5, 6, 7);
    hi = __builtin_shufflevector(__builtin_shufflevector(t[4], t[5], 0, 1, 2, 3), __builtin_shufflevector(t[6], t[7], 0, 1, 2, 3),
                                 0, 1, 2, 3, 4, 5, 6, 7);
}

__device__ __forceinline__ v4f bf_mfma(v8bf w, v4i x, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, __builtin_bit_cast(v8bf, x), c, 0, 0, 0);
}

__device__ __forceinline__ v4f scaled(v4f t, float s, v4f acc) {
    return v4f{__builtin_fmaf(t.x, s, acc.x), __builtin_fmaf(t.y, s, acc.y), __builtin_fmaf(t.z, s, acc.z),
               __builtin_fmaf(t.w, s, acc.w)};
}

constexpr uint32_t kOut = 0x80000000u;       // an offset past every buffer's range: reads as zeros

// This slot's expert e and its pairs, in order, in `list` (the workgroup's LDS: [pairs] entries, then [pairs] for the ids);
// the number of pairs, the same in every wave: 0 for an expert without any, for a pair without an expert (slots are pairs
// where those are fewer than the experts) and for one whose expert an earlier pair has.  Every wave writes the same list.
__device__ __forceinline__ int pairs_of(const ExpertArgs& a, int slot, int lane, uint16_t* list, int& e, int& tokens) {
    const bool by_pair = a.slots < a.E;
    e = slot;
    if (a.room * a.top <= 64) {
        // (the ids of rows that are not live are the caller's buffer as well: loaded beside the live count, not after it)
        int id = lane < a.room * a.top ? id_of(a, lane) : -1;
        tokens = pass_tokens(a);
        asm volatile("" ::"v"(id), "s"(tokens));
        if (lane >= tokens * a.top) id = -1;
        if (by_pair) e = __builtin_amdgcn_readlane(id, slot);
        if (e < 0) return 0;
        const uint64_t m = __ballot(id == e);
        if (m == 0 || (by_pair && __builtin_ctzll(m) != slot)) return 0;
        if (id == e) list[__popcll(m & ((1ull << lane) - 1))] = (uint16_t)lane;
        return __popcll(m);
    }
    tokens = pass_tokens(a);
    const int pairs = tokens * a.top;
    if (tokens <= 0 || (by_pair && slot >= pairs)) return 0;
    int16_t* ids = reinterpret_cast<int16_t*>(list) + a.room * a.top;
    for (int i = threadIdx.x; i < pairs; i += 64 * kWaves) ids[i] = (int16_t)id_of(a, i);
    __syncthreads();
    if (by_pair) e = __builtin_amdgcn_readfirstlane((int)ids[slot]);
    if (e < 0) return 0;
    int n = 0;
    for (int at = 0; at < pairs; at += 64) {
        const bool mine = at + lane < pairs && ids[at + lane] == e;
        const uint64_t m = __ballot(mine);
        if (by_pair && n == 0 && m && at + __builtin_ctzll(m) != slot) return 0;
        if (mine) list[n + __popcll(m & ((1ull << lane) - 1))] = (uint16_t)(at + lane);
        n += __popcll(m);
    }
    return n;
}

// A workgroup: 4 / KS times N 16-row tiles of the hidden values of one expert; KS waves split the inputs of a tile (wave part
// q: chunks q, q + KS, ...), each D chunks ahead.
template <int N, int KS, int D>
__global__ __launch_bounds__(64 * kWaves, 2) void moe_up_kernel(ExpertArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    experts_now(a);
    v4f* red = reinterpret_cast<v4f*>(lds);                                   // [waves][N][2][64] where K is split
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4, q = w % KS;
    uint16_t* list = reinterpret_cast<uint16_t*>(lds + (KS > 1 ? kWaves * N * 2048 : 0));
    int e, tokens;
    const int n = pairs_of(a, blockIdx.y, lane, list, e, tokens);
    if (n == 0) return;

    // (tiles past the last are the last once more, chunks past the last read as zeros: an offset past the range costs no traffic)
    const int tiles = a.I >> 4, t0 = (blockIdx.x * (kWaves / KS) + w / KS) * N, have = tiles - t0, tc = min(t0, tiles - 1);
    const uint32_t row = (uint32_t)a.KBH * 2048;                              // bytes of a 16-row tile
    const int64_t at = ((int64_t)e * tiles + tc) * row;
    const __amdgpu_buffer_rsrc_t gr = buf_rsrc(a.gate + at), ur = buf_rsrc(a.up + at);
    const int64_t sat = ((int64_t)e * ((a.I + 127) >> 7) + (tc >> 3)) * a.KBH;
    const __amdgpu_buffer_rsrc_t gsr = buf_rsrc(a.gate_s + sat), usr = buf_rsrc(a.up_s + sat);
    const __amdgpu_buffer_rsrc_t xr = buf_rsrc_n(a.x + a.first * a.x_ld, (uint32_t)((tokens - 1) * a.x_ld + a.H) * 2);
    struct Stage {
        v4i g[N][2], u[N][2], x[4];
        float gs, us;
    } st[D];
    for (int base = 0; base < n; base += 16) {
        const bool there = base + r < n;
        const int pair = there ? list[base + r] : 0;
        const uint32_t xo = there ? (uint32_t)(token_of(a, pair) * a.x_ld + 16 * g) * 2 : kOut;
        auto issue = [&](Stage& s, int b) {
            const uint32_t bc = min(b, a.KBH - 1), past = b < a.KBH ? 0u : kOut;
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    const uint32_t at = min(i, max(have, 1) - 1) * row + bc * 2048;
                    s.g[i][p] = buf_load16<kBufNT>(gr, (lane * 16 | past) + p * 1024, at);
                    s.u[i][p] = buf_load16<kBufNT>(ur, (lane * 16 | past) + p * 1024, at);
                }
            s.gs = __uint_as_float(buf_load4(gsr, past, bc * 4));
            s.us = __uint_as_float(buf_load4(usr, past, bc * 4));
#pragma unroll
            for (int p = 0; p < 2; p++) {
                const uint32_t o = b * 128 + p * 64 + 16 * g < a.H ? xo : kOut;
                s.x[2 * p] = buf_load16(xr, o + p * 128, bc * 256);
                s.x[2 * p + 1] = buf_load16(xr, o + p * 128 + 16, bc * 256);
            }
        };
        v4f ga[N], ua[N];
#pragma unroll
        for (int i = 0; i < N; i++) ga[i] = ua[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < D; d++) {
            issue(st[d], q + d * KS);
            __builtin_amdgcn_sched_barrier(0);
        }
        auto use = [&](const Stage& s) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                v4f tg = {0.f, 0.f, 0.f, 0.f}, tu = tg;
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    v8bf lo, hi;
                    widen(s.g[i][p], lo, hi);
                    tg = bf_mfma(hi, s.x[2 * p + 1], bf_mfma(lo, s.x[2 * p], tg));
                    widen(s.u[i][p], lo, hi);
                    tu = bf_mfma(hi, s.x[2 * p + 1], bf_mfma(lo, s.x[2 * p], tu));
                }
                ga[i] = scaled(tg, s.gs, ga[i]);
                ua[i] = scaled(tu, s.us, ua[i]);
            }
        };
        for (int b = q; b + D * KS < a.KBH; b += D * KS) {
#pragma unroll
            for (int d = 0; d < D; d++) {
                use(st[d]);
                issue(st[d], b + (d + D) * KS);
                // (else the uses of all stages gather in front and wait for all loads; the loads before the loop are kept in the
                // same order, as the wait in it has to serve both)
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int d = 0; d < D; d++) {                   // (the last round asks for nothing: loads past the end cost their issue)
            use(st[d]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (KS > 1) {
            if (base) __syncthreads();                                        // (the sums before are read)
#pragma unroll
            for (int i = 0; i < N; i++) {
                red[((w * N + i) * 2) * 64 + lane] = ga[i];
                red[((w * N + i) * 2 + 1) * 64 + lane] = ua[i];
            }
            __syncthreads();
        }
        // (of the KS waves of a tile, wave part i finishes tile i, i + KS, ...)
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (i % KS != q || i >= have || !there) continue;
            v4f gv = ga[i], uv = ua[i];
            if (KS > 1) {
                const int w0 = w - q;
#pragma unroll
                for (int j = 0; j < KS; j++) {
                    const v4f y = red[(((w0 + j) * N + i) * 2) * 64 + lane], z = red[(((w0 + j) * N + i) * 2 + 1) * 64 + lane];
                    if (j == 0) {
                        gv = y, uv = z;
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; k++) gv[k] = add_rn(gv[k], y[k]), uv[k] = add_rn(uv[k], z[k]);
                    }
                }
            }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float h = mul_rn(div_rn(gv[j], add_rn(1.f, expf(-gv[j]))), uv[j]);
                hi[j] = f32_to_bf16(h);
                const float rest = h - bf16_to_f32(hi[j]);
                lo[j] = (hi[j] & 0x7f80u) == 0x7f80u ? 0u : f32_to_bf16(rest);
            }
            uint16_t* o = a.h + (int64_t)pair * 2 * a.KBI * 128 + 16 * (t0 + i) + 4 * g;
            *reinterpret_cast<v2u*>(o) = v2u{hi[0] | hi[1] << 16, hi[2] | hi[3] << 16};
            *reinterpret_cast<v2u*>(o + a.KBI * 128) = v2u{lo[0] | lo[1] << 16, lo[2] | lo[3] << 16};
        }
    }
}

// The same for the outputs of one expert: N tiles share a chunk's hidden values, C pairs at a time.  C 8: the 16 columns are eight
// pairs' first parts and their second parts, half the loads and products of C 16, where they are two operands; an expert of
// more pairs reads its weights again for each C.
template <int N, int KS, int D, int C>
__global__ __launch_bounds__(64 * kWaves, 2) void moe_down_kernel(ExpertArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    experts_now(a);
    v4f* red = reinterpret_cast<v4f*>(lds);                                   // [waves][N][64] where K is split
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4, q = w % KS;
    uint16_t* list = reinterpret_cast<uint16_t*>(lds + (KS > 1 ? kWaves * N * 1024 : 0));
    int e, tokens;
    const int n = pairs_of(a, blockIdx.y, lane, list, e, tokens);
    if (n == 0) return;

    const int tiles = a.H >> 4, t0 = (blockIdx.x * (kWaves / KS) + w / KS) * N, have = tiles - t0, tc = min(t0, tiles - 1);
    const uint32_t row = (uint32_t)a.KBI * 2048, hrow = (uint32_t)a.KBI * 512;
    const __amdgpu_buffer_rsrc_t dr = buf_rsrc(a.down + ((int64_t)e * tiles + tc) * row);
    const __amdgpu_buffer_rsrc_t dsr = buf_rsrc(a.down_s + ((int64_t)e * ((a.H + 127) >> 7) + (tc >> 3)) * a.KBI);
    const __amdgpu_buffer_rsrc_t hr = buf_rsrc_n(a.h, (uint32_t)(tokens * a.top) * hrow);
    constexpr int P = C == 8 ? 1 : 2;                                         // operands of hidden values
    struct Stage {
        v4i d[N][2], h[P][4];
        float s;
    } st[D];
    for (int base = 0; base < n; base += C) {
        const int col = r % C;
        const bool there = base + col < n;
        const int pair = there ? list[base + col] : 0;
        const uint32_t ho = there ? (uint32_t)pair * hrow + 32 * g + (r / C) * (hrow / 2) : kOut;
        auto issue = [&](Stage& s, int b) {
            const uint32_t bc = min(b, a.KBI - 1), past = b < a.KBI ? 0u : kOut;
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int p = 0; p < 2; p++)
                    s.d[i][p] = buf_load16<kBufNT>(dr, (lane * 16 | past) + p * 1024, min(i, max(have, 1) - 1) * row + bc * 2048);
            s.s = __uint_as_float(buf_load4(dsr, past, bc * 4));
#pragma unroll
            for (int p = 0; p < 2; p++) {
                const uint32_t o = b * 128 + p * 64 + 16 * g < a.I ? ho : kOut;
#pragma unroll
                for (int k = 0; k < P; k++) {
                    s.h[k][2 * p] = buf_load16(hr, o + p * 128, bc * 256 + k * a.KBI * 256);
                    s.h[k][2 * p + 1] = buf_load16(hr, o + p * 128 + 16, bc * 256 + k * a.KBI * 256);
                }
            }
        };
        v4f y[N];
#pragma unroll
        for (int i = 0; i < N; i++) y[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < D; d++) {
            issue(st[d], q + d * KS);
            __builtin_amdgcn_sched_barrier(0);
        }
        auto use = [&](const Stage& s) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                v4f t = {0.f, 0.f, 0.f, 0.f}, l = t;
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    v8bf lo, hi;
                    widen(s.d[i][p], lo, hi);
                    t = bf_mfma(hi, s.h[0][2 * p + 1], bf_mfma(lo, s.h[0][2 * p], t));
                    if (P == 2) l = bf_mfma(hi, s.h[P - 1][2 * p + 1], bf_mfma(lo, s.h[P - 1][2 * p], l));
                }
                y[i] = scaled(t, s.s, y[i]);
                if (P == 2) y[i] = scaled(l, s.s, y[i]);
            }
        };
        for (int b = q; b + D * KS < a.KBI; b += D * KS) {
#pragma unroll
            for (int d = 0; d < D; d++) {
                use(st[d]);
                issue(st[d], b + (d + D) * KS);
                // (as in the up kernel)
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int d = 0; d < D; d++) {
            use(st[d]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (KS > 1) {
            if (base) __syncthreads();
#pragma unroll
            for (int i = 0; i < N; i++) red[(w * N + i) * 64 + lane] = y[i];
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (i % KS != q || i >= have) continue;
            v4f s = y[i];
            if (KS > 1) {
                const int w0 = w - q;
                s = red[(w0 * N + i) * 64 + lane];
#pragma unroll
                for (int j = 1; j < KS; j++) {
                    const v4f z = red[((w0 + j) * N + i) * 64 + lane];
#pragma unroll
                    for (int k = 0; k < 4; k++) s[k] = add_rn(s[k], z[k]);
                }
            }
            if (C == 8) {
#pragma unroll
                for (int k = 0; k < 4; k++) s[k] = add_rn(s[k], __shfl_xor(s[k], 8, kWave));
            }
            if (there && r < C) *reinterpret_cast<v4f*>(a.y + (int64_t)pair * a.H + 16 * (t0 + i) + 4 * g) = s;
        }
    }
}

template <int EPI>
__device__ __forceinline__ void store_out(const ExpertArgs& a, int t, int c, v4f y) {
    const int64_t o = (a.first + t) * a.o_ld + c;
    if (EPI == 0) {
        uint16_t* p = reinterpret_cast<uint16_t*>(a.out) + o;
        if (a.vec) {
            *reinterpret_cast<v2u*>(p) = v2u{f32_to_bf16(y.x) | f32_to_bf16(y.y) << 16, f32_to_bf16(y.z) | f32_to_bf16(y.w) << 16};
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) p[j] = (uint16_t)f32_to_bf16(y[j]);
        }
    } else {
        float* p = reinterpret_cast<float*>(a.out) + o;
#pragma unroll
        for (int j = 0; j < 4; j++) p[j] = add_rn(p[j], y[j]);
    }
}

// A token's pairs, weighted, in the order of its ids: a thread per four outputs.  All loads of four pairs go out at once (of
// pairs without an expert too: their places in the workspace hold anything).
template <int EPI>
__global__ __launch_bounds__(64) void moe_sum_kernel(ExpertArgs a) {
    experts_now(a);
    const int t = blockIdx.y, c = (blockIdx.x * 64 + threadIdx.x) * 4;
    if (c >= a.H) return;
    v4f y = {0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < a.top; j0 += 4) {
        int id[4];
        float pw[4];
        v4f v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int at = min(j0 + j, a.top - 1);
            id[j] = a.ids[(a.first + t) * a.ids_ld + at];
            pw[j] = a.w[(a.first + t) * a.w_ld + at];
            v[j] = *reinterpret_cast<const v4f*>(a.y + (int64_t)(t * a.top + at) * a.H + c);
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (j0 + j < a.top && (uint32_t)id[j] < (uint32_t)a.E) y = scaled(v[j], pw[j], y);
    }
    if (t < pass_tokens(a)) store_out<EPI>(a, t, c, y);
}

// The experts that as many random ids would reach.
inline double moe_reached(int64_t pairs, int64_t E) { return (double)E * (1.0 - pow(1.0 - 1.0 / (double)E, (double)pairs)); }

// How many of an expert's 16-row tiles a workgroup takes, of these numbers: the least time of the fullest CU, for as many experts as
// that many random ids would reach.  Its workgroups read at the CU's rate (tile_us a tile, about 23 GB/s), one alone at 5 / 8 of it,
// and each costs 0.8 us more.  Measured (us, all three launches; up with 4 / 2 / 1 tiles and down with 16 / 8 / 4, the other kernel at
// one form in each): 11 tokens on 2 of 16 experts, H 5120, I 1408: 59.0 / 53.4 / 50.1 and 59.1 / 55.8 / 53.3; 64 on 8 of 128, 2048, 768:
// 106 / 107 / 112 and 106 / 113 / 122; 2 on 3 of 8, 2752, 1824: 25.6 / 25.4 / 24.2 and 31.6 / 26.6 / 26.7; 5 on 8 of 40, 4560, 208:
// 31.6 / 32.0 / 26.8 and 32.5 / 32.1 / 35.3.
// Two stages in registers, so that three and more workgroups share a CU: with four (up) and three (down), two workgroups a CU, these
// were 54.6, 107, 28.3 and 37.6 and 63 tokens on 6 of 64 (640, 1760) 66 against 60.
inline int moe_form(int64_t pairs, int64_t E, int64_t tiles, double tile_us, const int* per, int forms) {
    const double reached = moe_reached(pairs, E);
    int best = 0;
    double least = 1e30;
    for (int i = 0; i < forms; i++) {
        const double rounds = ceil(reached * (double)((tiles + per[i] - 1) / per[i]) / 256.0);
        const double t = fmax(rounds, 1.6) * per[i] * tile_us + 0.8 * rounds;
        if (t < least) least = t, best = i;
    }
    return best;
}

}  // namespace prism

using namespace prism;

extern "C" int prism_moe_route(const prism_moe_route_args* args, void* stream) {
    if (!args) return PRISM_ERR_ARG;
    const prism_moe_route_args& h = *args;
    if (!h.x || !h.ids || !h.w || !h.n_rows || (h.f32 != 0 && h.f32 != 1) || (h.sigmoid != 0 && h.sigmoid != 1) ||
        (h.renorm != 0 && h.renorm != 1) || (h.bias && !h.sigmoid))
        return PRISM_ERR_ARG;
    if (h.T < 0 || h.T > INT32_MAX || h.E < 1 || h.E > 1024 || h.top < 1 || h.top > kMoeTop || h.top > h.E) return PRISM_ERR_SHAPE;
    if (h.x_ld < 0 || h.ids_ld < 0 || h.w_ld < 0 || (h.T > 1 && (h.ids_ld < h.top || h.w_ld < h.top)))
        return PRISM_ERR_SHAPE;
    if (!PRISM_ALIGNED(h.x, h.f32 ? 4 : 2) || !PRISM_ALIGNED(h.ids, 4) || !PRISM_ALIGNED(h.w, 4)) return PRISM_ERR_ALIGN;
    if (h.T == 0) return PRISM_OK;
    const RouteArgs a{h.x, h.x_ld, h.bias, h.ids, h.ids_ld, h.w, h.w_ld, h.n_rows, (int)h.T, (int)h.E, (int)h.top, (int)h.renorm,
                      (float)h.scale};
    const dim3 grid((unsigned)((h.T + 3) / 4));
    const hipStream_t st = (hipStream_t)stream;
#define RF(V, F) do { \
        if (h.bias) hipLaunchKernelGGL((moe_route_kernel<V, F, true, true>), grid, dim3(256), 0, st, a); \
        else if (h.sigmoid) hipLaunchKernelGGL((moe_route_kernel<V, F, true, false>), grid, dim3(256), 0, st, a); \
        else hipLaunchKernelGGL((moe_route_kernel<V, F, false, false>), grid, dim3(256), 0, st, a); \
    } while (0)
#define RT(V) do { if (h.f32) RF(V, true); else RF(V, false); } while (0)
    if (h.E <= 64) RT(1); else if (h.E <= 128) RT(2); else if (h.E <= 256) RT(4); else if (h.E <= 512) RT(8); else RT(16);
#undef RT
#undef RF
    PRISM_LAUNCH_CHECK();
    return PRISM_OK;
}

// The pairs' hidden values and outputs of a pass.
static int64_t moe_hidden_bytes(int64_t room, int64_t top, int64_t I) { return room * top * 2 * ((I + 127) / 128 * 128) * 2; }

extern "C" int64_t prism_moe_experts_workspace_bytes(int64_t T, int64_t top, int64_t H, int64_t I) {
    if (T < 1 || top < 1 || H < 1 || I < 1) return 0;
    const int64_t room = T < kMoeTokens ? T : kMoeTokens;
    return moe_hidden_bytes(room, top, I) + room * top * H * 4;
}

extern "C" int prism_moe_experts(const prism_moe_experts_args* args, void* stream) {
    if (!args) return PRISM_ERR_ARG;
    const prism_moe_experts_args& h = *args;
    if (!h.x || !h.ids || !h.w || !h.gate || !h.gate_s || !h.up || !h.up_s || !h.down || !h.down_s || !h.out || !h.n_rows ||
        (h.epi != 0 && h.epi != 1))
        return PRISM_ERR_ARG;
    if (h.T < 0 || h.T > INT32_MAX - kMoeTokens || h.E < 1 || h.E > 32767 || h.top < 1 || h.top > kMoeTop) return PRISM_ERR_SHAPE;
    if (h.H < 16 || h.I < 16 || h.H % 16 || h.I % 16 || h.H > kFp8MaxDim || h.I > kFp8MaxDim) return PRISM_ERR_SHAPE;
    if (h.x_ld < 0 || h.x_ld > kFp8MaxLd || h.ids_ld < 0 || h.w_ld < 0 || h.o_ld < 0) return PRISM_ERR_SHAPE;
    if (h.T > 1 && h.o_ld < h.H) return PRISM_ERR_SHAPE;
    const int64_t room = h.T < kMoeTokens ? h.T : kMoeTokens;
    // a pass's hidden values are reached by 31-bit offsets
    if ((int64_t)kMoeTokens * h.top * ((h.I + 127) / 128) * 512 > INT32_MAX) return PRISM_ERR_SHAPE;
    if (!PRISM_ALIGNED(h.x, 16) || h.x_ld % 8 || !PRISM_ALIGNED(h.gate, 16) || !PRISM_ALIGNED(h.up, 16) ||
        !PRISM_ALIGNED(h.down, 16) || !PRISM_ALIGNED(h.out, h.epi ? 4 : 2))
        return PRISM_ERR_ALIGN;
    if (h.T == 0) return PRISM_OK;
    const int64_t need = prism_moe_experts_workspace_bytes(h.T, h.top, h.H, h.I);
    if (!h.wsp || h.wsp_bytes < need) return PRISM_ERR_ARG;
    if (!PRISM_ALIGNED(h.wsp, 16)) return PRISM_ERR_ALIGN;
    ExpertArgs a{};
    a.x = h.x, a.x_ld = h.x_ld, a.ids = h.ids, a.ids_ld = h.ids_ld, a.w = h.w, a.w_ld = h.w_ld;
    a.gate = h.gate, a.up = h.up, a.down = h.down, a.gate_s = h.gate_s, a.up_s = h.up_s, a.down_s = h.down_s;
    a.h = (uint16_t*)h.wsp, a.y = (float*)((char*)h.wsp + moe_hidden_bytes(room, h.top, h.I));
    a.out = h.out, a.o_ld = h.o_ld, a.n_rows = h.n_rows;
    a.T = (int)h.T, a.E = (int)h.E, a.top = (int)h.top, a.H = (int)h.H, a.I = (int)h.I;
    a.KBH = (int)((h.H + 127) / 128), a.KBI = (int)((h.I + 127) / 128);
    a.div = 65536u / (uint32_t)h.top + 1;
    a.vec = h.o_ld % 4 == 0 && PRISM_ALIGNED(h.out, 8);
    const hipStream_t st = (hipStream_t)stream;
    const size_t ids_lds = (size_t)room * a.top * 4;             // the list and the ids
    const int up_per[] = {4, 2, 1}, down_per[] = {16, 8, 4};
    const int up = moe_form(room * a.top, a.E, a.I / 16, 0.178 * a.KBH, up_per, 3);
    const int down = moe_form(room * a.top, a.E, a.H / 16, 0.089 * a.KBI, down_per, 3);
    // eight pairs at a time in the down kernel where three or fewer are expected on an expert (2 tokens on 3 of 8, H 2752, I 1824 30.8
    // -> 28.5 us, one on 6 of 128, 1264, 336 15.0 -> 13.4; but 63 on 6 of 64, 640, 1760 69.8 -> 72.5, 64 on 8 of 128 109 -> 111)
    const bool eight = (double)(room * a.top) <= 3.0 * moe_reached(room * a.top, a.E);
    for (a.first = 0; a.first < a.T; a.first += kMoeTokens) {
        a.room = a.T - a.first < kMoeTokens ? a.T - a.first : kMoeTokens;      // (every row up to there is the caller's)
        a.slots = a.room * a.top < a.E ? a.room * a.top : a.E;
#define UP(N, KS, D) do { \
        const int per = kWaves / KS * N; \
        hipLaunchKernelGGL((moe_up_kernel<N, KS, D>), dim3((a.I / 16 + per - 1) / per, a.slots), dim3(64 * kWaves), \
                           ids_lds + (KS > 1 ? kWaves * N * 2048 : 0), st, a); \
    } while (0)
        // (down with 8 tiles: short sums are not split, 5 tokens on 8 of 40, I 208: 35.0 -> 32.1; from 7 blocks on they are, I 1760 67.5 ->
        // 65.2)
#define DOWN(N, KS, D, C) do { \
        const int per = kWaves / KS * N; \
        hipLaunchKernelGGL((moe_down_kernel<N, KS, D, C>), dim3((a.H / 16 + per - 1) / per, a.slots), dim3(64 * kWaves), \
                           ids_lds + (KS > 1 ? kWaves * N * 1024 : 0), st, a); \
    } while (0)
        if (up == 0) UP(2, 2, 2); else if (up == 1) UP(2, 4, 2); else UP(1, 4, 2);
        PRISM_LAUNCH_CHECK();
#define DOWNS(C) do { \
        if (down == 0) DOWN(4, 1, 2, C); else if (down == 2) DOWN(2, 2, 2, C); \
        else if (a.KBI <= 6) DOWN(2, 1, 2, C); else DOWN(4, 2, 2, C); \
    } while (0)
        if (eight) DOWNS(8); else DOWNS(16);
        PRISM_LAUNCH_CHECK();
#undef UP
#undef DOWN
#undef DOWNS
        const dim3 grid((a.H / 4 + 63) / 64, (unsigned)a.room);
        if (h.epi) hipLaunchKernelGGL((moe_sum_kernel<1>), grid, dim3(64), 0, st, a);
        else hipLaunchKernelGGL((moe_sum_kernel<0>), grid, dim3(64), 0, st, a);
        PRISM_LAUNCH_CHECK();
    }
    return PRISM_OK;
}
