// A mixture-of-experts layer for a few tokens on gfx950: the router's choice and the experts on e4m3 weights with block scales
// (fp8.hip's chunks), bf16 activations.
//
//   route     ids[t], w[t]: the top experts of a row of logits and their weights
//   experts   out[t] = sum_j w[t][j] down_e (silu(gate_e x_t) * (up_e x_t)),  e = ids[t][j]
//
// For a few tokens the experts' weights, read once, are the work: a chunk (16 rows x 128 inputs, 2 KB) is loaded straight
// into registers, its codes become bf16 (exact) two at a time, and v_mfma_f32_16x16x32_bf16 multiplies them with up to 16
// tokens' columns, four products per chunk chained from zero, then one fma by the block's scale into the fp32 sum.  Which
// pairs (token, place) an expert has is found by every wave from the ids with ballots: no sorting launch, and the order of
// all sums follows from the ids alone.
//
// Two launches.  moe_up_kernel: a workgroup per (expert, 16 hidden rows), its waves splitting the inputs; it leaves the hidden
// values h = silu(g) u of each pair in the workspace as two bf16 parts (h = hi + lo up to 2^-17 of it: the second product's
// operand; one part alone would add as much error as the bf16 output's own rounding).  moe_down_kernel: a workgroup per 16
// outputs of all tokens, its waves taking the experts in turn, each with its own sums of every token in LDS, which are added
// wave after wave at the end: no atomics, no third launch.
#include "common.h"
#include "fp8.h"

namespace prism {

constexpr int kMoeTokens = 128;              // tokens per pass of the experts (their sums lie in LDS)
constexpr int kMoeTop = 16;
constexpr int kUpWaves = 4, kDownWaves = 8;

// --------------------------------------------------------------------------------------------------------------- route
// An order-preserving integer of a number that may be chosen (greater than 0); 0 for NaN and -inf.
__device__ __forceinline__ uint64_t rank_of(float v) {
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

// A wave per token, lane l holding experts l, l + 64, ...; the best of all lanes, top times.
template <int V, bool F32, bool SIG>
__global__ __launch_bounds__(256) void moe_route_kernel(RouteArgs a) {
    const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (t >= min(a.T, __ldg(a.n_rows))) return;
    float x[V];
    double p[SIG ? V : 1];
    uint64_t key[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int e = lane + 64 * i;
        x[i] = __uint_as_float(0xff800000u);
        if (e < a.E)
            x[i] = F32 ? reinterpret_cast<const float*>(a.x)[t * a.x_ld + e]
                       : bf16_to_f32(reinterpret_cast<const uint16_t*>(a.x)[t * a.x_ld + e]);
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
        if (SIG) {
            const int e = lane + 64 * i;
            p[i] = 1.0 / (1.0 + exp(-(double)x[i]));
            key[i] = rank_of(x[i]) ? rank_of(p[i] + (a.bias && e < a.E ? (double)a.bias[e] : 0.0)) : 0;
        } else {
            key[i] = rank_of(x[i]);
        }
    }
    int id = -1;                                                  // lane j: the j-th choice
    float lx = 0.f;                                               // its logit, or
    double lp = 0.0;                                              // its sigmoid
    for (int j = 0; j < a.top; j++) {
        uint64_t best = 0;
        int at = 0;
#pragma unroll
        for (int i = 0; i < V; i++)
            if (key[i] > best) best = key[i], at = i;
        int e = lane + 64 * at;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t k2 = __shfl_xor((unsigned long long)best, o, kWave);
            const int e2 = __shfl_xor(e, o, kWave);
            if (k2 > best || (k2 == best && e2 < e)) best = k2, e = e2;
        }
        if (best == 0) break;                                     // (the same in every lane)
        float vx = 0.f;
        double vp = 0.0;
#pragma unroll
        for (int i = 0; i < V; i++)
            if (lane + 64 * i == e) {
                key[i] = 0, vx = x[i];
                if (SIG) vp = p[i];
            }
        vx = __shfl(vx, e & 63, kWave);
        if (SIG) vp = __shfl(vp, e & 63, kWave);
        if (lane == j) id = e, lx = vx, lp = vp;
    }
    float w = 0.f;
    if (SIG) {
        double sum = 1.0;
        if (a.renorm) {
            sum = id >= 0 ? lp : 0.0;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);       // (top <= 16 lanes)
        }
        w = (float)(lp / sum * (double)a.scale);
    } else {
        const float m = __shfl(lx, 0, kWave);                     // the largest logit
        const float ex = id >= 0 ? expf(lx - m) : 0.f;
        float sum = 0.f;
        if (a.renorm) {
            sum = ex;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
        } else {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (lane + 64 * i < a.E) sum += expf(x[i] - m);
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
    void* out;
    int64_t o_ld;
    const int32_t* n_rows;
    int T, E, top, H, I, KBH, KBI;
    uint32_t div;                            // pair -> token: (pair div) >> 16 (pairs < 2048, top <= 16)
    int slots;                               // experts looked at per pass: all, or one per pair where those are fewer
    int vec;
};

// The pass's tokens [first, first + tokens) and its pairs.
__device__ __forceinline__ int pass_pairs(const ExpertArgs& a, int first, int& tokens) {
    tokens = min(min(a.T, __ldg(a.n_rows)) - first, kMoeTokens);
    return tokens * a.top;
}
__device__ __forceinline__ int token_of(const ExpertArgs& a, int pair) { return (int)((uint32_t)pair * a.div >> 16); }

__device__ __forceinline__ int id_of(const ExpertArgs& a, int first, int pair, int pairs) {
    if (pair >= pairs) return -1;
    const int t = token_of(a, pair), e = a.ids[(first + t) * a.ids_ld + (pair - t * a.top)];
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

// A wave's expert of this slot and its pairs in `list`, in order; the number of pairs (0: none, or an earlier slot's).
// ids(i): the expert of pair i (-1: none).  by_pair: the slots are pairs, and a pair whose expert an earlier one has is none.
template <typename F>
__device__ __forceinline__ int pairs_of(F&& ids, int slot, bool by_pair, int pairs, int lane, uint16_t* list, int& e) {
    e = slot;
    if (by_pair) {
        e = __builtin_amdgcn_readfirstlane(ids(slot));
        if (e < 0) return 0;
    }
    int n = 0;
    for (int at = 0; at < pairs; at += 64) {
        const bool mine = at + lane < pairs && ids(at + lane) == e;
        const uint64_t m = __ballot(mine);
        if (by_pair && n == 0 && m && at + __builtin_ctzll(m) != slot) return 0;
        if (mine) list[n + __popcll(m & ((1ull << lane) - 1))] = (uint16_t)(at + lane);
        n += __popcll(m);
    }
    return n;
}

constexpr int kUpDepth = 4;
__global__ __launch_bounds__(64 * kUpWaves) void moe_up_kernel(ExpertArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    v4f* red = reinterpret_cast<v4f*>(lds);                                   // [waves][2][64]
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int first = blockIdx.z * kMoeTokens, tile = blockIdx.x, slot = blockIdx.y;
    int tokens;
    const int pairs = pass_pairs(a, first, tokens);
    const bool by_pair = a.slots < a.E;
    if (tokens <= 0 || (by_pair && slot >= pairs)) return;
    uint16_t* list = reinterpret_cast<uint16_t*>(lds + kUpWaves * 2048) + w * kMoeTokens * a.top;
    int e;
    const int n = pairs_of([&](int i) { return id_of(a, first, i, pairs); }, slot, by_pair, pairs, lane, list, e);
    if (n == 0) return;                                                       // (the same in all waves)

    const uint32_t row = (uint32_t)a.KBH * 2048;                              // bytes of a 16-row tile
    const int64_t at = ((int64_t)e * (a.I / 16) + tile) * row;
    const __amdgpu_buffer_rsrc_t gr = buf_rsrc_n(a.gate + at, row), ur = buf_rsrc_n(a.up + at, row);
    const int64_t sat = ((int64_t)e * ((a.I + 127) / 128) + tile / 8) * a.KBH;
    const float *gs = a.gate_s + sat, *us = a.up_s + sat;
    const __amdgpu_buffer_rsrc_t xr = buf_rsrc_n(a.x + first * a.x_ld, (uint32_t)((tokens - 1) * a.x_ld + a.H) * 2);
    struct Stage {
        v4i g[2], u[2], x[4];
    } st[kUpDepth];
    for (int base = 0; base < n; base += 16) {
        const bool there = base + r < n;
        const int pair = there ? list[base + r] : 0;
        const uint32_t xo = there ? (uint32_t)(token_of(a, pair) * a.x_ld + 16 * g) * 2 : kOut;
        auto issue = [&](Stage& s, int b) {
            const uint32_t past = b < a.KBH ? 0u : kOut;
#pragma unroll
            for (int p = 0; p < 2; p++) {
                s.g[p] = buf_load16<kBufNT>(gr, (b * 2048u + p * 1024 + lane * 16) | past, 0);
                s.u[p] = buf_load16<kBufNT>(ur, (b * 2048u + p * 1024 + lane * 16) | past, 0);
                const uint32_t o = (xo + b * 256u + p * 128) | past | (b * 128 + p * 64 + 16 * g < a.H ? 0u : kOut);
                s.x[2 * p] = buf_load16(xr, o, 0);
                s.x[2 * p + 1] = buf_load16(xr, o + 16, 0);
            }
        };
        v4f ga = {0.f, 0.f, 0.f, 0.f}, ua = ga;
#pragma unroll
        for (int d = 0; d < kUpDepth; d++) issue(st[d], w + d * kUpWaves);
        for (int b = w; b < a.KBH; b += kUpDepth * kUpWaves) {
#pragma unroll
            for (int d = 0; d < kUpDepth; d++) {
                const int kb = b + d * kUpWaves, kc = min(kb, a.KBH - 1);
                v4f tg = {0.f, 0.f, 0.f, 0.f}, tu = tg;
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    v8bf lo, hi;
                    widen(st[d].g[p], lo, hi);
                    tg = bf_mfma(hi, st[d].x[2 * p + 1], bf_mfma(lo, st[d].x[2 * p], tg));
                    widen(st[d].u[p], lo, hi);
                    tu = bf_mfma(hi, st[d].x[2 * p + 1], bf_mfma(lo, st[d].x[2 * p], tu));
                }
                ga = scaled(tg, gs[kc], ga);
                ua = scaled(tu, us[kc], ua);
                issue(st[d], kb + kUpDepth * kUpWaves);
            }
        }
        if (base) __syncthreads();                                            // (the sums before are read)
        red[(w * 2) * 64 + lane] = ga;
        red[(w * 2 + 1) * 64 + lane] = ua;
        __syncthreads();
        if (w == 0 && there) {
            for (int i = 1; i < kUpWaves; i++) {
                const v4f y = red[(i * 2) * 64 + lane], z = red[(i * 2 + 1) * 64 + lane];
#pragma unroll
                for (int j = 0; j < 4; j++) ga[j] = add_rn(ga[j], y[j]), ua[j] = add_rn(ua[j], z[j]);
            }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float h = mul_rn(div_rn(ga[j], add_rn(1.f, expf(-ga[j]))), ua[j]);
                hi[j] = f32_to_bf16(h);
                const float rest = h - bf16_to_f32(hi[j]);
                lo[j] = (hi[j] & 0x7f80u) == 0x7f80u ? 0u : f32_to_bf16(rest);
            }
            uint16_t* o = a.h + ((int64_t)first * a.top + pair) * 2 * a.KBI * 128 + 16 * tile + 4 * g;
            *reinterpret_cast<v2u*>(o) = v2u{hi[0] | hi[1] << 16, hi[2] | hi[3] << 16};
            *reinterpret_cast<v2u*>(o + a.KBI * 128) = v2u{lo[0] | lo[1] << 16, lo[2] | lo[3] << 16};
        }
    }
}

constexpr int kDownDepth = 4;
template <int EPI>
__global__ __launch_bounds__(64 * kDownWaves) void moe_down_kernel(ExpertArgs a, int parts) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int first = blockIdx.y * kMoeTokens, tile = blockIdx.x;
    int tokens;
    const int pairs = pass_pairs(a, first, tokens);
    if (tokens <= 0) return;
    const int room = min(a.T, kMoeTokens);                                    // as the host sized LDS
    v4f* sums = reinterpret_cast<v4f*>(lds) + w * room * 4;                   // [tokens][16 outputs], one per wave
    int16_t* ids = reinterpret_cast<int16_t*>(lds + kDownWaves * room * 64);
    uint16_t* list = reinterpret_cast<uint16_t*>(ids) + room * a.top * (1 + w);
    for (int i = threadIdx.x; i < pairs; i += 64 * kDownWaves) ids[i] = (int16_t)id_of(a, first, i, pairs);
    for (int i = lane; i < tokens * 4; i += 64) sums[i] = v4f{0.f, 0.f, 0.f, 0.f};
    __syncthreads();

    const bool by_pair = a.slots < a.E;
    const int units = min(a.slots, by_pair ? pairs : a.E) * parts;
    const uint32_t row = (uint32_t)a.KBI * 2048, hrow = (uint32_t)a.KBI * 512;
    const __amdgpu_buffer_rsrc_t hr = buf_rsrc_n(a.h + (int64_t)first * a.top * 2 * a.KBI * 128, (uint32_t)pairs * hrow);
    for (int u = w; u < units; u += kDownWaves) {
        int e;
        const int n = pairs_of([&](int i) { return (int)ids[i]; }, u / parts, by_pair, pairs, lane, list, e);
        if (n == 0) continue;
        const int part = u % parts, b0 = a.KBI * part / parts, b1 = a.KBI * (part + 1) / parts;
        const __amdgpu_buffer_rsrc_t dr = buf_rsrc_n(a.down + ((int64_t)e * (a.H / 16) + tile) * row, row);
        const float* ds = a.down_s + ((int64_t)e * ((a.H + 127) / 128) + tile / 8) * a.KBI;
        struct Stage {
            v4i d[2], h[2][4];
        } st[kDownDepth];
        for (int base = 0; base < n; base += 16) {
            const bool there = base + r < n;
            const int pair = there ? list[base + r] : 0;
            const uint32_t ho = there ? (uint32_t)pair * hrow + 32 * g : kOut;
            auto issue = [&](Stage& s, int b) {
                const uint32_t past = b < b1 ? 0u : kOut;
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    s.d[p] = buf_load16<kBufNT>(dr, (b * 2048u + p * 1024 + lane * 16) | past, 0);
                    const uint32_t o = (ho + b * 256u + p * 128) | past | (b * 128 + p * 64 + 16 * g < a.I ? 0u : kOut);
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        s.h[q][2 * p] = buf_load16(hr, o + q * a.KBI * 256u, 0);
                        s.h[q][2 * p + 1] = buf_load16(hr, o + q * a.KBI * 256u + 16, 0);
                    }
                }
            };
            v4f y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int d = 0; d < kDownDepth; d++) issue(st[d], b0 + d);
            for (int b = b0; b < b1; b += kDownDepth) {
#pragma unroll
                for (int d = 0; d < kDownDepth; d++) {
                    v4f t = {0.f, 0.f, 0.f, 0.f}, l = t;
#pragma unroll
                    for (int p = 0; p < 2; p++) {
                        v8bf lo, hi;
                        widen(st[d].d[p], lo, hi);
                        t = bf_mfma(hi, st[d].h[0][2 * p + 1], bf_mfma(lo, st[d].h[0][2 * p], t));
                        l = bf_mfma(hi, st[d].h[1][2 * p + 1], bf_mfma(lo, st[d].h[1][2 * p], l));
                    }
                    const float s = ds[min(b + d, a.KBI - 1)];
                    y = scaled(l, s, scaled(t, s, y));
                    issue(st[d], b + d + kDownDepth);
                }
            }
            // into this wave's sums; pairs of one token (an expert named twice) one after the other
            const int t = there ? token_of(a, pair) : -1;
            const float pw = there ? a.w[(first + t) * a.w_ld + (pair - t * a.top)] : 0.f;
            const int before = __shfl(t, lane - 1, kWave);
            const bool twice = __ballot(there && r > 0 && before == t) != 0;
            for (int j = 0; j < (twice ? a.top : 1); j++)
                if (there && (!twice || pair - t * a.top == j)) {
                    const v4f s = sums[t * 4 + g];
                    sums[t * 4 + g] = scaled(y, pw, s);
                }
        }
    }
    __syncthreads();
    const v4f* all = reinterpret_cast<const v4f*>(lds);
    for (int i = threadIdx.x; i < tokens * 4; i += 64 * kDownWaves) {
        v4f y = all[i];
        for (int j = 1; j < kDownWaves; j++) {
            const v4f z = all[j * room * 4 + i];
            y = v4f{add_rn(y.x, z.x), add_rn(y.y, z.y), add_rn(y.z, z.z), add_rn(y.w, z.w)};
        }
        const int64_t o = (first + i / 4) * a.o_ld + 16 * tile + 4 * (i & 3);
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
#define RT(V) do { \
        if (h.f32 && h.sigmoid) hipLaunchKernelGGL((moe_route_kernel<V, true, true>), grid, dim3(256), 0, st, a); \
        else if (h.f32) hipLaunchKernelGGL((moe_route_kernel<V, true, false>), grid, dim3(256), 0, st, a); \
        else if (h.sigmoid) hipLaunchKernelGGL((moe_route_kernel<V, false, true>), grid, dim3(256), 0, st, a); \
        else hipLaunchKernelGGL((moe_route_kernel<V, false, false>), grid, dim3(256), 0, st, a); \
    } while (0)
    if (h.E <= 64) RT(1); else if (h.E <= 128) RT(2); else if (h.E <= 256) RT(4); else if (h.E <= 512) RT(8); else RT(16);
#undef RT
    PRISM_LAUNCH_CHECK();
    return PRISM_OK;
}

extern "C" int64_t prism_moe_experts_workspace_bytes(int64_t T, int64_t top, int64_t I) {
    if (T < 1 || top < 1 || I < 1) return 0;
    return T * top * 2 * ((I + 127) / 128 * 128) * 2;
}

extern "C" int prism_moe_experts(const prism_moe_experts_args* args, void* stream) {
    if (!args) return PRISM_ERR_ARG;
    const prism_moe_experts_args& h = *args;
    if (!h.x || !h.ids || !h.w || !h.gate || !h.gate_s || !h.up || !h.up_s || !h.down || !h.down_s || !h.out || !h.n_rows ||
        (h.epi != 0 && h.epi != 1))
        return PRISM_ERR_ARG;
    if (h.T < 0 || h.T > 65535 * (int64_t)kMoeTokens || h.E < 1 || h.E > 32767 || h.top < 1 || h.top > kMoeTop) return PRISM_ERR_SHAPE;
    if (h.H < 16 || h.I < 16 || h.H % 16 || h.I % 16 || h.H > kFp8MaxDim || h.I > kFp8MaxDim) return PRISM_ERR_SHAPE;
    if (h.x_ld < 0 || h.x_ld > kFp8MaxLd || h.ids_ld < 0 || h.w_ld < 0 || h.o_ld < 0) return PRISM_ERR_SHAPE;
    if (h.T > 1 && h.o_ld < h.H) return PRISM_ERR_SHAPE;
    // a pass's hidden values are reached by 31-bit offsets
    if ((int64_t)kMoeTokens * h.top * ((h.I + 127) / 128) * 512 > INT32_MAX) return PRISM_ERR_SHAPE;
    if (!PRISM_ALIGNED(h.x, 16) || h.x_ld % 8 || !PRISM_ALIGNED(h.gate, 16) || !PRISM_ALIGNED(h.up, 16) ||
        !PRISM_ALIGNED(h.down, 16) || !PRISM_ALIGNED(h.out, h.epi ? 4 : 2))
        return PRISM_ERR_ALIGN;
    if (h.T == 0) return PRISM_OK;
    const int64_t need = prism_moe_experts_workspace_bytes(h.T, h.top, h.I);
    if (!h.wsp || h.wsp_bytes < need) return PRISM_ERR_ARG;
    if (!PRISM_ALIGNED(h.wsp, 16)) return PRISM_ERR_ALIGN;
    ExpertArgs a{};
    a.x = h.x, a.x_ld = h.x_ld, a.ids = h.ids, a.ids_ld = h.ids_ld, a.w = h.w, a.w_ld = h.w_ld;
    a.gate = h.gate, a.up = h.up, a.down = h.down, a.gate_s = h.gate_s, a.up_s = h.up_s, a.down_s = h.down_s;
    a.h = (uint16_t*)h.wsp, a.out = h.out, a.o_ld = h.o_ld, a.n_rows = h.n_rows;
    a.T = (int)h.T, a.E = (int)h.E, a.top = (int)h.top, a.H = (int)h.H, a.I = (int)h.I;
    a.KBH = (int)((h.H + 127) / 128), a.KBI = (int)((h.I + 127) / 128);
    a.div = 65536u / (uint32_t)h.top + 1;
    const int room = (int)(h.T < kMoeTokens ? h.T : kMoeTokens);
    a.slots = room * a.top < a.E ? room * a.top : a.E;
    a.vec = h.o_ld % 4 == 0 && PRISM_ALIGNED(h.out, 8);
    if (a.slots > 65535) return PRISM_ERR_SHAPE;
    const unsigned passes = (unsigned)((h.T + kMoeTokens - 1) / kMoeTokens);
    const hipStream_t st = (hipStream_t)stream;
    const size_t up_lds = (size_t)kUpWaves * (2048 + (size_t)kMoeTokens * a.top * 2);
    hipLaunchKernelGGL(moe_up_kernel, dim3(a.I / 16, a.slots, passes), dim3(64 * kUpWaves), up_lds, st, a);
    PRISM_LAUNCH_CHECK();
    const size_t down_lds = (size_t)kDownWaves * room * 64 + (size_t)room * a.top * 2 * (1 + kDownWaves);
    // few experts: their inputs are split, so that every wave has some
    int parts = (kDownWaves + a.slots - 1) / a.slots;
    if (parts > a.KBI) parts = a.KBI;
    if (h.epi) {
        allow_lds(moe_down_kernel<1>, down_lds);
        hipLaunchKernelGGL((moe_down_kernel<1>), dim3(a.H / 16, passes), dim3(64 * kDownWaves), down_lds, st, a, parts);
    } else {
        allow_lds(moe_down_kernel<0>, down_lds);
        hipLaunchKernelGGL((moe_down_kernel<0>), dim3(a.H / 16, passes), dim3(64 * kDownWaves), down_lds, st, a, parts);
    }
    PRISM_LAUNCH_CHECK();
    return PRISM_OK;
}
