// The gated delta rule of a linear-attention layer in serving (gfx950).  Per value head, with the state S fp32 [DK,
// DV], a = exp(g), key k and query q (normalised to length 1 in the kernel if asked, the query times a scale):
//   S <- a S;  u = beta (v - S^T k);  S <- S + k u^T;  o = S^T q.
// States, sums and factors are fp32, a chunk's gate sums fp64.
#include "common.h"

namespace prism {

struct DeltaArgs {
    const uint16_t *q, *k, *v;                                // bf16 [rows, heads, dim]
    int64_t ldq, hq_s, ldk, hk_s, ldv, hv_s;                  // row and head strides (elements)
    const float *g, *beta;                                    // [rows, HV]
    int64_t ldg, ldb;
    float* state;                                             // [slots, HV, DK, DV], slot stride lds_
    int64_t lds_;
    float* out;                                               // [rows, HV, DV]
    int64_t ldo, ho_s;
    const int32_t *cu, *slots, *n;                            // cu: prompts' first rows [seqs + 1]; n: live rows of a step
    int rows, seqs, nslots, HK, HV, norm;
    float scale, eps;
};

// Rows and state of sequence b; count 0 for nothing to do.  A step's row i is sequence i of one token.
__device__ __forceinline__ bool delta_seq(const DeltaArgs& a, int b, int& first, int& count, int& slot) {
    if (a.cu) {
        // rows stay inside the buffers whatever the offsets hold
        const int f = min(max(__ldg(a.cu + b), 0), a.rows), l = min(max(__ldg(a.cu + b + 1), 0), a.rows);
        first = f, count = max(l - f, 0);
    } else {
        first = b, count = b < __ldg(a.n);
    }
    slot = a.slots ? __ldg(a.slots + b) : b;
    return count > 0 && slot >= 0 && slot < a.nslots;
}

// What the lanes of a wave pass each other through LDS is in order at this point: the hardware keeps a wave's LDS operations
// in theirs, the fence keeps the compiler from moving them.
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ float wave_addf(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    return v;
}

// ------------------------------------------------------------------------------------------------------- recurrent form
// A workgroup holds NC columns of one head's state in registers from its only read to its only write: thread t the
// columns 4 (t % (NC / 4)) .. + 3 of the rows t / (NC / 4) + i RG.  Both sums over the rows, S^T k and S^T q, are taken
// of the decayed state at once (o = S^T q + (q . k) u), so a token costs one exchange between the waves.  Each wave
// holds its own copy of the token's key and query.  A step of many rows is bound by the state's bytes: 256 rows of 32
// heads of 128 x 128 (1.08 GB) 190 us, 5.7 TB/s; 40 rows of 48 heads (254 MB) 46 us, 5.5 TB/s (a copy in place of 1 GB:
// 5.9).  Several tokens of a sequence are bound by the exchange's chain, 1.5 us a token; loading the next token's
// inputs ahead did not show.
template <int DK, int DV, int NC>
__global__ __launch_bounds__(256) void delta_rec_kernel(DeltaArgs a) {
    constexpr int LC = NC / 4, RG = 256 / LC, RPT = DK / RG, E = DK / 64;
    __shared__ float kq[4][2][DK];
    __shared__ v4f red[2][4][2][LC];
    const int slices = DV / NC, slice = blockIdx.x % slices, head = blockIdx.x / slices % a.HV;
    const int b = blockIdx.x / slices / a.HV;
    int first, count, slot;
    if (!delta_seq(a, b, first, count, slot)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = threadIdx.x % LC, rg = threadIdx.x / LC;
    float* st = a.state + slot * a.lds_ + (int64_t)head * DK * DV + slice * NC + 4 * c;
    const int hk = head / (a.HV / a.HK);
    v4f s[RPT];
#pragma unroll
    for (int i = 0; i < RPT; i++)
        s[i] = __builtin_nontemporal_load(reinterpret_cast<const v4f*>(st + (rg + i * RG) * DV));
    for (int j = 0; j < count; j++) {
        const int64_t t = first + j;
        float kv[E], qv[E], kk = 0.f, qq = 0.f, qk = 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) {
            kv[e] = bf16_to_f32(a.k[t * a.ldk + hk * a.hk_s + e * 64 + lane]);
            qv[e] = bf16_to_f32(a.q[t * a.ldq + hk * a.hq_s + e * 64 + lane]);
        }
        const v2u vb = *reinterpret_cast<const v2u*>(a.v + t * a.ldv + head * a.hv_s + slice * NC + 4 * c);
        const float al = expf(a.g[t * a.ldg + head]), beta = a.beta[t * a.ldb + head];
#pragma unroll
        for (int e = 0; e < E; e++) {
            kk += kv[e] * kv[e];
            qq += qv[e] * qv[e];
            qk += kv[e] * qv[e];
        }
        const float rk = a.norm ? div_rn(1.f, sqrt_rn(wave_addf(kk) + a.eps)) : 1.f;
        const float rq = (a.norm ? div_rn(1.f, sqrt_rn(wave_addf(qq) + a.eps)) : 1.f) * a.scale;
        qk = wave_addf(qk) * rk * rq;
#pragma unroll
        for (int e = 0; e < E; e++) {
            kq[wave][0][e * 64 + lane] = kv[e] * rk;
            kq[wave][1][e * 64 + lane] = qv[e] * rq;
        }
        wave_lds_order();                                     // (the last token's readers are past its barrier)
        v4f w1 = {0.f, 0.f, 0.f, 0.f}, w2 = w1;
        float kr[RPT];
#pragma unroll
        for (int i = 0; i < RPT; i++) {
            kr[i] = kq[wave][0][rg + i * RG];
            const float qr = kq[wave][1][rg + i * RG];
            s[i] *= al;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                w1[x] = fmaf(kr[i], s[i][x], w1[x]);
                w2[x] = fmaf(qr, s[i][x], w2[x]);
            }
        }
#pragma unroll
        for (int o = LC; o < 64; o <<= 1)
#pragma unroll
            for (int x = 0; x < 4; x++) {
                w1[x] += __shfl_xor(w1[x], o, kWave);
                w2[x] += __shfl_xor(w2[x], o, kWave);
            }
        if (lane < LC) {
            red[j & 1][wave][0][lane] = w1;
            red[j & 1][wave][1][lane] = w2;
        }
        __syncthreads();                                      // (the other buffer's readers are past the last token's)
        w1 = red[j & 1][0][0][c];
        w2 = red[j & 1][0][1][c];
#pragma unroll
        for (int w = 1; w < 4; w++) {
            w1 += red[j & 1][w][0][c];
            w2 += red[j & 1][w][1][c];
        }
        v4f u;
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const uint32_t h = vb[x / 2];
            u[x] = beta * (__uint_as_float(x % 2 ? h & 0xffff0000u : h << 16) - w1[x]);
        }
#pragma unroll
        for (int i = 0; i < RPT; i++)
#pragma unroll
            for (int x = 0; x < 4; x++) s[i][x] = fmaf(kr[i], u[x], s[i][x]);
        if (rg == 0) {
            v4f o;
#pragma unroll
            for (int x = 0; x < 4; x++) o[x] = fmaf(qk, u[x], w2[x]);
            *reinterpret_cast<v4f*>(a.out + t * a.ldo + head * a.ho_s + slice * NC + 4 * c) = o;
        }
    }
#pragma unroll
    for (int i = 0; i < RPT; i++) __builtin_nontemporal_store(s[i], reinterpret_cast<v4f*>(st + (rg + i * RG) * DV));
}

// Columns per workgroup: 32 while that is what fills the card, the whole head (its 64 KB in one run) once there are
// heads enough.  At 48 heads of 128 x 128: 1 row 4.5 us with 32, 4.8 with 64, 5.4 with 128 columns; 8 rows 10.5, 9.4,
// 10.1; 16 rows 20.9, 20.7, 18.5; 256 rows of 32 heads 203, 203, 190 (214 without the non-temporal loads and stores).
template <int DK, int DV>
static int launch_rec(const DeltaArgs& a, hipStream_t st) {
    const int64_t heads = (int64_t)a.seqs * a.HV;
    if (heads * (DV / 32) > INT32_MAX) return PRISM_ERR_SHAPE;
#define RC(NC) \
    hipLaunchKernelGGL((delta_rec_kernel<DK, DV, NC>), dim3((unsigned)(heads * (DV / (NC)))), dim3(256), 0, st, a)
    if (heads >= 512) RC(DV);
    else if (heads >= 256) RC(64);
    else RC(32);
#undef RC
    return hipGetLastError() == hipSuccess ? (int)PRISM_OK : (int)PRISM_ERR_LAUNCH;
}

// ---------------------------------------------------------------------------------------------------------- chunked form
// Chunks of 64 tokens.  With G the running sum of g in the chunk, the chunk's updates solve a triangular system:
//   A_ij = beta_i e^(G_i - G_j) k_i . k_j (j < i),  X = (I + A)^-1,  U = X diag(beta) (V - diag(e^G) K S)
//   O = diag(e^G) Q S + P U,  P_ij = e^(G_i - G_j) q_i . k_j (j <= i);  S <- e^(G_63) S + K^T diag(e^(G_63 - G)) U
// Only S runs from chunk to chunk, so two kernels: delta_prep computes X diag(beta) and P of all chunks at once,
// delta_scan walks each sequence's chunks.  The normalisation is row scales (rk, rq), so K and Q stay the bf16 they
// are.
//
// The products run on the bf16 MFMA at fp32's precision and range: an fp32 operand is three bf16 that add up to it (S, R
// and U cut, 8 bits after 8; X and P each the rounding of what the last part left), three products against K or Q, which
// are bf16, six against another such triple (the three dropped ones are below 2^-23 of the terms).  Every value keeps its
// own exponent, so no value's size touches another's bits.  Pairs of fp16 under powers of two shared by a column need two
// and three products (8191 tokens, 16 key and 48 value heads of 128: 352 us instead of 381), but what a value keeps then
// depends on the largest of its column: a token's update was rounded by, or lost to, a large value that came after it.
//
// A token's outputs depend on its own and earlier tokens only, whatever finite values the later ones hold; what is not finite,
// an input or a product past fp32's range, reaches its whole chunk (zeros of a triangle times infinity).
//
// Everything that delta_scan multiplies from the left (K, Q, K^T, X diag(beta), P) lies in the workspace as MFMA
// fragments, 1 KB each in lane order.  Inside a product the order of the summed index is free: taking it as an
// accumulator's rows lie (lane group g: 4 g + r of one 16-row tile, then 4 g + r of the next), the accumulators of one
// product are the right operand of the next as they are, and a wave owns 16 columns of S for the whole sequence
// without exchanging anything.
constexpr int kC = 64;                                        // tokens per chunk
constexpr int kFrag = 1024;                                   // bytes of a fragment: 64 lanes of 8 bf16
constexpr int kTri = 6;       // fragments (i, s) of a lower triangle: 16-row tile i, 32 columns s <= i / 2
__host__ __device__ constexpr int tri(int i, int s) { return i < 2 ? i : 2 * i - 2 + s; }
// K, Q, K^T
__host__ __device__ constexpr int64_t rec_k(int DK) { return (int64_t)(4 * (DK / 32) * 2 + DK / 16 * 2) * kFrag; }
// X diag(beta), P, three parts each (two side by side, the third of all behind them); factors of K S, of Q S and of U; e^(G_63)
constexpr int64_t kRecV = 2 * 3 * kTri * kFrag + 4 * kC * 4;

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
__device__ __forceinline__ v4f mfma_bf16(v4u a, v4u b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma_f32(float a, float b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// LDS-DMA of 4 bytes a lane.
__device__ __forceinline__ void dma4(const void* g, void* lds) {
    __builtin_amdgcn_global_load_lds(g, (__attribute__((address_space(3))) void*)lds, 4, 0, 0);
}

// Eight fp32 (x then y) as three bf16 fragments, of which the first two round: h = RN(x), m = RN(x - h), l = x - h - m.  All
// differences are exact.  No inline assembly here: the compiler does not put the wait states between it and an MFMA that
// reads its result.
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
struct Split {
    v4u h, m, l;
};
__device__ __forceinline__ uint32_t bf16x2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{a, b}), v2bf));
}
__device__ __forceinline__ float low_half(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_half(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ Split split_rn(v4f x, v4f y) {
    Split r;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        float a = w < 2 ? x[2 * w] : y[2 * w - 4], b = w < 2 ? x[2 * w + 1] : y[2 * w - 3];
        r.h[w] = bf16x2(a, b);
        a -= low_half(r.h[w]), b -= high_half(r.h[w]);
        r.m[w] = bf16x2(a, b);
        r.l[w] = bf16x2(a - low_half(r.m[w]), b - high_half(r.m[w]));
    }
    return r;
}
// The same with parts cut to 8 bits, which is faster (8191 tokens 381 us, with rounded ones in the scan 396).
__device__ __forceinline__ uint32_t upper(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ float rest(float x) { return x - high_half(__float_as_uint(x)); }
__device__ __forceinline__ Split split_cut(v4f x, v4f y) {
    Split r;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const float a = w < 2 ? x[2 * w] : y[2 * w - 4], b = w < 2 ? x[2 * w + 1] : y[2 * w - 3];
        const float a1 = rest(a), b1 = rest(b);
        r.h[w] = upper(a, b);
        r.m[w] = upper(a1, b1);
        r.l[w] = upper(rest(a1), rest(b1));
    }
    return r;
}

// Chunk `id` of the workspace: sequence b's chunks start at id cu[b] / 64 + b, which leaves each sequence room for its
// ceil(length / 64) whatever the lengths.  False: no chunk has that number.
__device__ __forceinline__ bool find_chunk(const DeltaArgs& a, int id, int& first, int& count) {
    const int lane = threadIdx.x & 63;
    for (int b0 = 0; b0 < a.seqs; b0 += 64) {
        const int b = b0 + lane;
        int f = 0, n = 0;
        if (b < a.seqs) {
            f = min(max(__ldg(a.cu + b), 0), a.rows);
            n = max(min(max(__ldg(a.cu + b + 1), 0), a.rows) - f, 0);
        }
        const int at = id - (f / kC + b);
        const bool hit = at >= 0 && (int64_t)at * kC < n;
        const uint64_t m = __ballot(hit);
        if (m) {
            const int src = __builtin_ctzll(m), c = __shfl(at, src, kWave) * kC;
            first = __shfl(f, src, kWave) + c;
            count = min(__shfl(n, src, kWave) - c, kC);
            return true;
        }
    }
    return false;
}

// The records go past the caches (delta_scan reads them after all are written): 8191 tokens 379 us in all instead of
// 396 when that was measured.
__device__ __forceinline__ void put_frag(char* base, v4u v) {
    __builtin_nontemporal_store(v, reinterpret_cast<v4u*>(base + (threadIdx.x & 63) * 16));
}

// A workgroup per chunk (blockIdx.x) and value head (blockIdx.y), a wave per 16 of the chunk's rows (of X's columns
// where the system is solved).  Rows are loaded in their own order (a row per lane would take the memory pipeline four
// times as long) and become fragments through LDS.  The decays between tokens of different 16-row tiles are products of
// three that are at most 1, so that a diagonal tile's exponentials and a few are enough.  One chunk takes 9 us, the
// chain of its steps, and 8191 tokens of 16 key and 48 value heads of 128 take 92 us, the records' 333 MB for the most
// part.  With a third less of X and P (255 MB, 86 us) one wave for all four tiles took 13 and 100 us, each wave inverting
// its own diagonal block 9.4 and 109.
template <int DK>
__global__ __launch_bounds__(256, 4) void delta_prep_kernel(DeltaArgs a, char* wk, char* wv) {
    constexpr int KS = DK / 32, LD = kC + 4, LK = DK + 8, PR = DK / 8, NL = 16 * PR / 64;  // PR: 16-byte pieces of a row
    __shared__ __align__(16) uint16_t rows[2][kC * LK];       // K's and Q's rows; then A, then X, in place
    __shared__ double gsum[kC];
    __shared__ float rkv[kC], rqv[kC], bev[kC], upv[kC], dnv[kC];
    static_assert(sizeof(rows) >= kC * LD * 4, "A");
    float* x = reinterpret_cast<float*>(rows);
    int first, count;
    if (!find_chunk(a, blockIdx.x, first, count)) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int head = blockIdx.y, share = a.HV / a.HK, hk = head / share, part = head % share;
    const int own = 16 * w + col;                             // this lane's row where a fragment's rows are lanes
    char* rk = wk + ((int64_t)blockIdx.x * a.HK + hk) * rec_k(DK);
    char* rv = wv + ((int64_t)blockIdx.x * a.HV + head) * kRecV;

    v4u kr[NL], qr[NL];                                       // rows past the chunk are zeros
#pragma unroll
    for (int i = 0; i < NL; i++) {
        const int64_t t = first + min(16 * w + i * (64 / PR) + lane / PR, count - 1);
        kr[i] = *reinterpret_cast<const v4u*>(a.k + t * a.ldk + hk * a.hk_s + 8 * (lane % PR));
        qr[i] = *reinterpret_cast<const v4u*>(a.q + t * a.ldq + hk * a.hq_s + 8 * (lane % PR));
    }
    // the chunk's gates, one token per lane, the sums in 64 bits: the differences G_i - G_j are then as exact as the g.
    // Below -1e4 a decay is 0 either way, and sums stay finite (-inf minus -inf would not be a number)
    if (w == 0) {
        const bool in = lane < count;
        const int64_t t = first + min(lane, count - 1);
        const float be = a.beta[t * a.ldb + head];
        float gv = a.g[t * a.ldg + head];
        gv = !in ? 0.f : gv < -1e4f ? -1e4f : gv;
        double s = gv;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double up = __shfl_up(s, o, kWave);
            if (lane >= o) s += up;
        }
        gsum[lane] = s;
        bev[lane] = in ? be : 0.f;
        // from the last token before this one's tile, and to the last token of its tile
        const double before = __shfl(s, (lane & 48) - 1, kWave), last = __shfl(s, lane | 15, kWave);
        upv[lane] = expf((float)(s - (lane < 16 ? 0.0 : before)));
        dnv[lane] = expf((float)(last - s));
    }
#pragma unroll
    for (int i = 0; i < NL; i++) {
        const int row = 16 * w + i * (64 / PR) + lane / PR, at = row * LK + 8 * (lane % PR);
        *reinterpret_cast<v4u*>(rows[0] + at) = row < count ? kr[i] : v4u{0, 0, 0, 0};
        *reinterpret_cast<v4u*>(rows[1] + at) = row < count ? qr[i] : v4u{0, 0, 0, 0};
    }
    __syncthreads();
    // fragment s of tile i: its row col, dims 32 s + 8 g .. + 7
    auto get = [&](v4u (&f)[KS], const uint16_t* r, int i) {
#pragma unroll
        for (int s = 0; s < KS; s++) f[s] = *reinterpret_cast<const v4u*>(r + (16 * i + col) * LK + 32 * s + 8 * g);
    };
    // the tile's rows' normalising factors, if asked, from their lengths: the diagonal of K K^T or Q Q^T
    auto lengths = [&](const v4u (&f)[KS], float* unit, float scale) {
        v4f d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; s++) d = mfma_bf16(f[s], f[s], d);
        const float sq = col & 2 ? (col & 1 ? d[3] : d[2]) : (col & 1 ? d[1] : d[0]);
        // (rows past the chunk are zeros, whose length eps = 0 would divide by)
        if (g == col >> 2)
            unit[own] = own < count ? (a.norm ? div_rn(1.f, sqrt_rn(sq + a.eps)) : 1.f) * scale : 0.f;
    };
    v4u kf[KS], qf[KS];
    get(kf, rows[0], w);
    get(qf, rows[1], w);
    lengths(kf, rkv, 1.f);
    lengths(qf, rqv, a.scale);
    __syncthreads();
    // as delta_scan's left operand: fragment (w, s), dims 32 s + 4 g + j, then 32 s + 16 + 4 g + j
    auto copy = [&](char* to, const uint16_t* from) {
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const uint16_t* r = from + own * LK + 32 * s + 4 * g;
            const v2u lo = *reinterpret_cast<const v2u*>(r), hi = *reinterpret_cast<const v2u*>(r + 16);
            put_frag(to + (w * KS + s) * kFrag, v4u{lo[0], lo[1], hi[0], hi[1]});
        }
    };
    // this key head's fragments of K, K^T and Q are written by its first, second and last value head's workgroup
    if (part == 0) copy(rk, rows[0]);
    if (part == (share > 1 ? 1 : 0)) {
        // K^T: fragment (d, s), row 16 d + col, tokens 32 s + 4 g + j and 32 s + 16 + 4 g + j
        char* ft = rk + 8 * KS * kFrag;
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int e = 0; e < DK / 64; e++) {
                const int d = w * (DK / 64) + e;
                uint32_t u[8];
#pragma unroll
                for (int j = 0; j < 8; j++)
                    u[j] = rows[0][(32 * s + 16 * (j / 4) + 4 * g + j % 4) * LK + 16 * d + col];
                put_frag(ft + (2 * d + s) * kFrag,
                         v4u{u[0] | (u[1] << 16), u[2] | (u[3] << 16), u[4] | (u[5] << 16), u[6] | (u[7] << 16)});
            }
    }
    if (part == share - 1) copy(rk + 4 * KS * kFrag, rows[1]);

    // k_i . k_j and q_i . k_j, tiles j <= i = w, transposed: a lane holds row `own` for columns 4 g + r, which is a
    // fragment's order
    v4f pt[4], am[4];
    {
        const double gi = gsum[own];
        const float up = upv[own], ki = bev[own] * rkv[own], qi = rqv[own];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            pt[j] = am[j] = v4f{0.f, 0.f, 0.f, 0.f};
            if (j > w) continue;
            v4f kk = {0.f, 0.f, 0.f, 0.f}, qk = kk, f;
            v4u kj[KS];
            get(kj, rows[0], j);
#pragma unroll
            for (int s = 0; s < KS; s++) {
                kk = mfma_bf16(kj[s], kf[s], kk);
                qk = mfma_bf16(kj[s], qf[s], qk);
            }
            const int c0 = 16 * j + 4 * g;
            if (w == j) {
#pragma unroll
                for (int r = 0; r < 4; r++) f[r] = expf((float)(gi - gsum[c0 + r]));
            } else {
                const float mid = w == j + 1 ? up : up * expf((float)(gsum[16 * w - 1] - gsum[16 * j + 15]));
#pragma unroll
                for (int r = 0; r < 4; r++) f[r] = mid * dnv[c0 + r];
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                f[r] *= rkv[c0 + r];
                am[j][r] = c0 + r < own ? f[r] * ki * kk[r] : 0.f;
                pt[j][r] = c0 + r <= own ? f[r] * qi * qk[r] : 0.f;
            }
        }
    }
    __syncthreads();                                          // K's and Q's rows are read
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (j <= w) *reinterpret_cast<v4f*>(x + own * LD + 16 * j + 4 * g) = am[j];
    __syncthreads();

    // the four diagonal blocks of I + A inverted at once by forward substitution, a column per lane
    if (w == 0) {
        float* d = x + 16 * g * LD + 16 * g;
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float s = i == col ? 1.f : 0.f;
#pragma unroll
            for (int j4 = 0; j4 < (i + 3) / 4; j4++) {
                const v4f row = *reinterpret_cast<const v4f*>(d + i * LD + 4 * j4);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (4 * j4 + j < i) s = fmaf(-row[j], v[4 * j4 + j], s);
            }
            v[i] = s;
        }
        wave_lds_order();                                     // (the wave's reads come before its writes)
#pragma unroll
        for (int i = 0; i < 16; i++) d[i * LD + col] = v[i];
    }
    __syncthreads();
    // the blocks below, X_ij = -X_ii sum_k A_ik X_kj, column j = w: the X_kj are right operands as the accumulators
    // they come in, so nothing is stored before all are there
    {
        v4f y[4];                                             // [i - w]
#pragma unroll
        for (int r = 0; r < 4; r++) y[0][r] = x[(16 * w + 4 * g + r) * LD + own];
#pragma unroll
        for (int d = 1; d < 4; d++) {
            const int i = w + d;
            if (i > 3) continue;
            v4f s = {0.f, 0.f, 0.f, 0.f}, z = s;
#pragma unroll
            for (int k = 0; k < d; k++) {
                const v4f m = *reinterpret_cast<const v4f*>(x + (16 * i + col) * LD + 16 * (w + k) + 4 * g);
#pragma unroll
                for (int r = 0; r < 4; r++) s = mfma_f32(m[r], y[k][r], s);
            }
            const v4f xi = *reinterpret_cast<const v4f*>(x + (16 * i + col) * LD + 16 * i + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; r++) z = mfma_f32(xi[r], s[r], z);
            y[d] = -z;
        }
        __syncthreads();
#pragma unroll
        for (int d = 1; d < 4; d++)
            if (w + d < 4)
#pragma unroll
                for (int r = 0; r < 4; r++) x[(16 * (w + d) + 4 * g + r) * LD + own] = y[d][r];
    }
    __syncthreads();
    // X diag(beta) and P
    auto put_tri = [&](const v4f (&h)[4], char* to) {
#pragma unroll
        for (int s = 0; s < 2; s++) {
            if (s > w / 2) continue;
            const Split sp = split_rn(h[2 * s], h[2 * s + 1]);  // (zeros right of the diagonal)
            put_frag(to + 2 * tri(w, s) * kFrag, sp.h);
            put_frag(to + (2 * tri(w, s) + 1) * kFrag, sp.m);
            put_frag(to + (2 * kTri + tri(w, s)) * kFrag, sp.l);
        }
    };
    put_tri(pt, rv + 3 * kTri * kFrag);
    {
        v4f h[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            h[j] = v4f{0.f, 0.f, 0.f, 0.f};
            if (j <= w)
                h[j] = *reinterpret_cast<const v4f*>(x + own * LD + 16 * j + 4 * g) *
                       *reinterpret_cast<const v4f*>(bev + 16 * j + 4 * g);
        }
        put_tri(h, rv);
    }
    if (w == 0) {
        float* vec = reinterpret_cast<float*>(rv + 6 * kTri * kFrag);
        const double gl = gsum[lane], gc = gsum[kC - 1];
        const float e = expf((float)gl);
        vec[lane] = e * rkv[lane];
        vec[kC + lane] = e * rqv[lane];
        vec[2 * kC + lane] = expf((float)(gc - gl)) * rkv[lane];
        vec[3 * kC + lane] = expf((float)gc);
    }
}

// A workgroup walks the chunks of one sequence and value head for 32 columns of the state, twelve waves, three to a
// SIMD. Four waves to 16 columns: two hold the halves of S's rows and take what the next chunk waits for (K S, U, K^T
// U), two the chunk's output (Q S, P U); products split over the summed index: a wave multiplies its half of S's rows,
// or its half of U's tokens, and the halves' sums (fp32, always the same two added) meet in LDS.  The other four waves
// bring the fragments into LDS, each group while nobody reads it; the output waves touch the lines of the chunk after the
// next, so that those come from L2.  Two barriers per chunk:
//   state waves   K S, halves out        | halves in, R, X R out  | U in, S <- ..., S out
//   output waves  (P U of the last one)  | S in, Q S              | P U, halves out
//   loading waves                        | next K, P's thirds in  | all else of the next chunk in
// Bound by that chain where there are no more workgroups than CUs: 8191 tokens of one sequence, 16 key and 48 value heads of
// 128 (192 workgroups) take 284 us, 2.2 a chunk, and 208 with the state waves' work alone; LDS moves 390 KB a chunk (some 3100
// cycles).  158 KB of LDS leave one workgroup a CU: 1500 tokens in 5 prompts with 32 value heads are 640 workgroups, 40 us
// for 13 chunks a CU.
template <int DK>
struct ScanShared {
    v4u k[4 * (DK / 32)][64], q[4 * (DK / 32)][64], x[3 * kTri][64], pl[kTri][64];
    v4u kt[2][DK / 16 * 2][64], p[2][2 * kTri][64];           // a chunk's, the next one's beside them
    float vec[2][4 * kC];                                     // the factors likewise
    v4f sx[2][DK / 16][64], kx[2][4][64], ux[2][6][64], ox[2][4][64];
    uint32_t touched[64];
};

// What a wave of delta_scan walks along.
struct ScanAt {
    int first, count, nc, head, c0, w;                        // c0: the lane's column; w: which 16 of the workgroup's 32
    int64_t rks, rvs;                                         // bytes from a chunk's records to the next one's
};

// A product's fragments are read from LDS into registers.  The compiler spreads the reads over the phase; forced to its
// start, to have their latency behind what the right operand still takes, they come as bursts that hold the others up:
// 392 us for 8191 tokens instead of 372 (with operands of two parts).
// K or Q: 4 token tiles, the half's k
template <int DK, int HALF>
__device__ __forceinline__ void read_rows(v4u (&r)[DK / 64][4], const v4u (*f)[64]) {
#pragma unroll
    for (int k = 0; k < DK / 64; k++)
#pragma unroll
        for (int i = 0; i < 4; i++) r[k][i] = f[i * (DK / 32) + HALF * (DK / 64) + k][threadIdx.x & 63];
}
// X diag(beta) or P, the parts that lie side by side and the third ones: the columns of the half's tokens
template <int HALF>
__device__ __forceinline__ void read_tri(v4u (&r)[4][3], const v4u (*hm)[64], const v4u (*l)[64]) {
#pragma unroll
    for (int i = 2 * HALF; i < 4; i++) {
        r[i][0] = hm[2 * tri(i, HALF)][threadIdx.x & 63];
        r[i][1] = hm[2 * tri(i, HALF) + 1][threadIdx.x & 63];
        r[i][2] = l[tri(i, HALF)][threadIdx.x & 63];
    }
}
// acc += r s
__device__ __forceinline__ void mul_rows(v4f (&acc)[4], const v4u (&r)[4], const Split& s) {
#pragma unroll
    for (int i = 0; i < 4; i++) acc[i] = mfma_bf16(r[i], s.l, acc[i]);
#pragma unroll
    for (int i = 0; i < 4; i++) acc[i] = mfma_bf16(r[i], s.m, acc[i]);
#pragma unroll
    for (int i = 0; i < 4; i++) acc[i] = mfma_bf16(r[i], s.h, acc[i]);
}
// acc += r s, the small products first
template <int HALF>
__device__ __forceinline__ void mul_tri(v4f (&acc)[4], const v4u (&r)[4][3], const Split& s) {
#pragma unroll
    for (int p = 0; p < 6; p++) {
        const int e = p == 0 ? 2 : p == 1 || p == 3 ? 1 : 0;
        const v4u& y = p == 2 ? s.l : p == 1 || p == 4 ? s.m : s.h;
#pragma unroll
        for (int i = 2 * HALF; i < 4; i++) acc[i] = mfma_bf16(r[i][e], y, acc[i]);
    }
}

template <int DK, int DV, int HALF>
__device__ __forceinline__ void scan_state(const DeltaArgs& a, const ScanAt& at, int slot, ScanShared<DK>& x) {
    constexpr int KH = DK / 64, DH = DK / 32;
    const int lane = threadIdx.x & 63, g = lane >> 4, w = at.w;
    float* st = a.state + slot * a.lds_ + (int64_t)at.head * DK * DV + at.c0;
    v4f s[DH];
#pragma unroll
    for (int d = 0; d < DH; d++)
#pragma unroll
        for (int r = 0; r < 4; r++) s[d][r] = st[(16 * (HALF * DH + d) + 4 * g + r) * DV];
    uint32_t off[2][4];                                       // this half's tokens' values (bytes from the chunk's)
    uint16_t v[2][4];
    const char* vp = reinterpret_cast<const char*>(a.v + (int64_t)at.first * a.ldv + at.head * a.hv_s + at.c0);
    // rows past the chunk's end read its last row: their columns of X diag(beta) are zeros
    auto offsets = [&](int left) {
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                off[i][r] = 2u * (uint32_t)a.ldv * (uint32_t)min(32 * HALF + 16 * i + 4 * g + r, left - 1);
    };
    auto load_v = [&] {
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) v[i][r] = *reinterpret_cast<const uint16_t*>(vp + off[i][r]);
    };
    offsets(at.count);
    load_v();
#pragma unroll
    for (int d = 0; d < DH; d++) x.sx[w][HALF * DH + d][lane] = s[d];
    lds_barrier();
    for (int c = 0; c < at.nc; c++) {
        const float* vec = x.vec[c & 1];
        const int left = at.count - (c + 1) * kC;             // rows after this chunk
        v4f ks[4], u[4];
        v4u kr[KH][4], tr[4][3], tk[DH][2];
        read_rows<DK, HALF>(kr, x.k);
#pragma unroll
        for (int i = 0; i < 4; i++) ks[i] = u[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KH; k++) mul_rows(ks, kr[k], split_cut(s[2 * k], s[2 * k + 1]));
        // the other half's tokens' sums out, this half's in
        x.kx[w][2 - 2 * HALF][lane] = ks[2 - 2 * HALF];
        x.kx[w][3 - 2 * HALF][lane] = ks[3 - 2 * HALF];
        lds_barrier();
        v4f rr[2], ek[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            rr[i] = x.kx[w][2 * HALF + i][lane];
            ek[i] = *reinterpret_cast<const v4f*>(vec + 32 * HALF + 16 * i + 4 * g);
        }
        read_tri<HALF>(tr, x.x, x.x + 2 * kTri);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            rr[i] += ks[2 * HALF + i];
#pragma unroll
            for (int r = 0; r < 4; r++) rr[i][r] = fmaf(-ek[i][r], rr[i][r], bf16_to_f32(v[i][r]));
        }
        if (left > 0) {
            vp += 2 * kC * a.ldv;
            if (left < kC) offsets(left);
            load_v();
        }
        mul_tri<HALF>(u, tr, split_cut(rr[0], rr[1]));
#pragma unroll
        for (int i = 2 * HALF; i < 4; i++) x.ux[w][i + 2 * HALF][lane] = u[i];
        lds_barrier();
        v4f ux[4], ew[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (i >= 2 || HALF) ux[i] = x.ux[w][i < 2 || HALF ? i : i + 2][lane];
            ew[i] = *reinterpret_cast<const v4f*>(vec + 2 * kC + 16 * i + 4 * g);
        }
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int d = 0; d < DH; d++) tk[d][e] = x.kt[c & 1][2 * (HALF * DH + d) + e][lane];
        const float ec = vec[3 * kC];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (i >= 2 || HALF) u[i] += ux[i];                // (half 1 has no part of u[0], u[1]: zeros)
            u[i] *= ew[i];
        }
        v4f add[DH];
#pragma unroll
        for (int d = 0; d < DH; d++) add[d] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const Split us = split_cut(u[2 * e], u[2 * e + 1]);
#pragma unroll
            for (int d = 0; d < DH; d++) add[d] = mfma_bf16(tk[d][e], us.l, add[d]);
#pragma unroll
            for (int d = 0; d < DH; d++) add[d] = mfma_bf16(tk[d][e], us.m, add[d]);
#pragma unroll
            for (int d = 0; d < DH; d++) add[d] = mfma_bf16(tk[d][e], us.h, add[d]);
        }
#pragma unroll
        for (int d = 0; d < DH; d++)
#pragma unroll
            for (int r = 0; r < 4; r++) s[d][r] = fmaf(ec, s[d][r], add[d][r]);
#pragma unroll
        for (int d = 0; d < DH; d++) x.sx[w][HALF * DH + d][lane] = s[d];
    }
#pragma unroll
    for (int d = 0; d < DH; d++)
#pragma unroll
        for (int r = 0; r < 4; r++) st[(16 * (HALF * DH + d) + 4 * g + r) * DV] = s[d][r];
    lds_barrier();
}

// rec: the key head's (HALF 0) or the head's (1) records, whose lines these waves touch two chunks ahead; m of `per`:
// this workgroup among those that read them.
template <int DK, int HALF>
__device__ __forceinline__ void scan_out(const DeltaArgs& a, const ScanAt& at, const char* rec, int m, int per,
                                         ScanShared<DK>& x) {
    constexpr int KH = DK / 64, DH = DK / 32, LINES = (int)((HALF ? kRecV : rec_k(DK)) / 128);
    const int lane = threadIdx.x & 63, g = lane >> 4, w = at.w;
    const int64_t step = HALF ? at.rvs : at.rks;
    // (waited for once, at the end: nobody reads what they bring, but it has landed before the LDS is another workgroup's)
    auto touch = [&](const char* r) {
        for (int i = (2 * m + w) * 64 + lane; i < LINES; i += per * 128)
            dma4(r + i * 128, x.touched);
    };
    v4f mine[2];
    float* out = a.out + (int64_t)at.first * a.ldo + at.head * a.ho_s + at.c0;
    // the last chunk's sums of this half's tokens, joined, then stored (`left` rows of it are there)
    auto join = [&] {
#pragma unroll
        for (int i = 0; i < 2; i++) mine[i] += x.ox[w][2 * HALF + i][lane];
    };
    auto store = [&](int left) {
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int t = 32 * HALF + 16 * i + 4 * g + r;
                if (left >= kC || t < left) __builtin_nontemporal_store(mine[i][r], out + (int64_t)t * a.ldo);
            }
        out += kC * a.ldo;
    };
    lds_barrier();
    for (int c = 0; c < at.nc; c++) {
        const float* vec = x.vec[c & 1] + kC;
        lds_barrier();
        if (c) join();
        v4f o[4];
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = v4f{0.f, 0.f, 0.f, 0.f};
        v4f s[DH], eq[4];
        v4u qr[KH][4], tr[4][3];
#pragma unroll
        for (int d = 0; d < DH; d++) s[d] = x.sx[w][HALF * DH + d][lane];
        read_rows<DK, HALF>(qr, x.q);
#pragma unroll
        for (int i = 0; i < 4; i++) eq[i] = *reinterpret_cast<const v4f*>(vec + 16 * i + 4 * g);
#pragma unroll
        for (int k = 0; k < KH; k++) mul_rows(o, qr[k], split_cut(s[2 * k], s[2 * k + 1]));
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] *= eq[i];
        lds_barrier();
        if (c) store(kC);                                     // (here the state waves have more to do than these)
        if (c + 2 < at.nc) touch(rec + (c + 2) * step);
        v4f u0 = x.ux[w][2 * HALF][lane], u1 = x.ux[w][2 * HALF + 1][lane];
        read_tri<HALF>(tr, x.p[c & 1], x.pl);
        if (HALF) {
            u0 += x.ux[w][4][lane];
            u1 += x.ux[w][5][lane];
        }
        v4f pu[4];
#pragma unroll
        for (int i = 2 * HALF; i < 4; i++) pu[i] = v4f{0.f, 0.f, 0.f, 0.f};
        mul_tri<HALF>(pu, tr, split_cut(u0, u1));
#pragma unroll
        for (int i = 2 * HALF; i < 4; i++) o[i] += pu[i];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            x.ox[w][2 - 2 * HALF + i][lane] = o[2 - 2 * HALF + i];
            mine[i] = o[2 * HALF + i];
        }
    }
    vm_wait<0>();
    lds_barrier();
    join();
    store(at.count - (at.nc - 1) * kC);
}

// Wave `q` of the four: every fourth fragment.
template <int DK>
__device__ __forceinline__ void scan_load(const ScanAt& at, const char* rk, const char* rv, int q, ScanShared<DK>& x) {
    const int64_t rks = at.rks, rvs = at.rvs;
    constexpr int NK = 4 * (DK / 32), NT = DK / 16 * 2, NX = 3 * kTri;
    const int lane = threadIdx.x & 63;
    auto bring = [&](v4u (*to)[64], const char* from, int count) {
        for (int i = q; i < count; i += 4) dma16(from + i * kFrag + lane * 16, to[i]);
    };
    auto factors = [&](int c, const char* r) {
        if (q == 0) dma16(r + 2 * NX * kFrag + lane * 16, x.vec[c & 1]);
    };
    auto later = [&](int c, const char* k, const char* v) {   // what chunk c needs after its first barrier
        bring(x.q, k + NK * kFrag, NK);
        bring(x.x, v, NX);
        factors(c, v);
        bring(x.p[c & 1], v + NX * kFrag, 2 * kTri);
        bring(x.kt[c & 1], k + 2 * NK * kFrag, NT);
    };
    bring(x.k, rk, NK);
    later(0, rk, rv);
    vm_wait<0>();
    lds_barrier();
    for (int c = 0; c < at.nc; c++) {
        const bool more = c + 1 < at.nc;
        lds_barrier();
        bring(x.pl, rv + (NX + 2 * kTri) * kFrag, kTri);
        if (more) bring(x.k, rk + rks, NK);
        vm_wait<0>();
        lds_barrier();
        if (more) later(c + 1, rk + rks, rv + rvs);
        vm_wait<0>();
        rk += rks, rv += rvs;
    }
    lds_barrier();
}

template <int DK, int DV>
__global__ __launch_bounds__(768, 3) void delta_scan_kernel(DeltaArgs a, const char* wk, const char* wv, int keys) {
    constexpr int CT = DV / 32;
    extern __shared__ __align__(16) char shared[];
    ScanShared<DK>& x = *reinterpret_cast<ScanShared<DK>*>(shared);
    // the workgroups of one key head, which read the same K and Q, on one XCD (workgroup i runs on XCD i % 8)
    const int share = a.HV / a.HK, per = share * CT;
    const int grp = blockIdx.x / (8 * per), key = 8 * grp + blockIdx.x % 8, m = blockIdx.x / 8 % per;
    if (key >= keys) return;
    const int b = key / a.HK, hk = key % a.HK;
    ScanAt at;
    int slot;
    if (!delta_seq(a, b, at.first, at.count, slot)) return;
    at.head = hk * share + m / CT;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    at.w = wave & 1;
    at.c0 = 32 * (m % CT) + 16 * at.w + (lane & 15);
    at.nc = (at.count + kC - 1) / kC;
    const int64_t id = at.first / kC + b;
    const char* rk = wk + (id * a.HK + hk) * rec_k(DK);
    const char* rv = wv + (id * a.HV + at.head) * kRecV;
    at.rks = (int64_t)a.HK * rec_k(DK), at.rvs = (int64_t)a.HV * kRecV;
    switch (wave >> 1) {
        case 0: return scan_state<DK, DV, 0>(a, at, slot, x);
        case 1: return scan_state<DK, DV, 1>(a, at, slot, x);
        case 2: return scan_out<DK, 0>(a, at, rk, m, per, x);
        case 3: return scan_out<DK, 1>(a, at, rv, m % CT, CT, x);
        default: break;
    }
    scan_load<DK>(at, rk, rv, wave - 8, x);
}

static int64_t chunks(int64_t T, int64_t seqs) { return T / kC + seqs; }

template <int DK, int DV>
static int launch_chunks(const DeltaArgs& a, char* ws, hipStream_t st) {
    const int64_t nc = chunks(a.rows, a.seqs), keys = (int64_t)a.seqs * a.HK;
    const int64_t wgs = (keys + 7) / 8 * 8 * (a.HV / a.HK) * (DV / 32);
    if (nc > INT32_MAX || wgs > INT32_MAX) return PRISM_ERR_SHAPE;
    char* wv = ws + nc * a.HK * rec_k(DK);
    hipLaunchKernelGGL(delta_prep_kernel<DK>, dim3((unsigned)nc, (unsigned)a.HV), dim3(256), 0, st, a, ws, wv);
    PRISM_LAUNCH_CHECK();
    allow_lds(delta_scan_kernel<DK, DV>, sizeof(ScanShared<DK>));
    hipLaunchKernelGGL((delta_scan_kernel<DK, DV>), dim3((unsigned)wgs), dim3(768), sizeof(ScanShared<DK>), st, a, ws, wv,
                       (int)keys);
    PRISM_LAUNCH_CHECK();
    return PRISM_OK;
}

static int dispatch_rec(const DeltaArgs& a, int64_t DK, int64_t DV, hipStream_t st) {
    if (DK == 64) return DV == 64 ? launch_rec<64, 64>(a, st) : launch_rec<64, 128>(a, st);
    return DV == 64 ? launch_rec<128, 64>(a, st) : launch_rec<128, 128>(a, st);
}

static int dispatch_chunks(const DeltaArgs& a, int64_t DK, int64_t DV, char* ws, hipStream_t st) {
    if (DK == 64) return DV == 64 ? launch_chunks<64, 64>(a, ws, st) : launch_chunks<64, 128>(a, ws, st);
    return DV == 64 ? launch_chunks<128, 64>(a, ws, st) : launch_chunks<128, 128>(a, ws, st);
}

// A few rows go token by token: 1.5 us each for a sequence's at 48 heads, against 15.3 us for its first chunk (one
// sequence of 6 rows 12.3 us, 8 rows 15.4, 10 rows 18.5; 12 rows of 6 sequences 10.4 against 35).  The rule sees the rows
// in all, not the prompts' lengths, which are on the device: many short prompts go in chunks and take a chunk's records
// (2.6 MB at 16 and 48 heads of 128) and time each, 189 us for 40 prompts of 4 rows.
static bool by_token(int64_t T, int64_t seqs) { return T <= (seqs > 1 ? 12 : 8); }

static int64_t workspace_bytes(int64_t T, int64_t seqs, int64_t hk, int64_t hv, int64_t dk) {
    if (T < 1 || seqs < 1 || hk < 1 || hv < 1 || (dk != 64 && dk != 128) || by_token(T, seqs)) return 0;
    return chunks(T, seqs) * (hk * rec_k((int)dk) + hv * kRecV);
}

static_assert(sizeof(prism_delta_args) == 32 * 8, "8-byte fields throughout");

// A call's arguments, checked and launched; seqs sequences, in chunks where a prompt's rows are given and many enough.
static int run(const prism_delta_args& h, bool prompts, hipStream_t st) {
    const int64_t seqs = prompts ? h.seqs : h.T;
    if (!h.q || !h.k || !h.v || !h.g || !h.beta || !h.state || !h.out || !h.rows || (h.norm != 0 && h.norm != 1))
        return PRISM_ERR_ARG;
    if ((h.dk != 64 && h.dk != 128) || (h.dv != 64 && h.dv != 128)) return PRISM_ERR_SHAPE;
    if (h.hk < 1 || h.hv < h.hk || h.hv % h.hk || h.hv > 65535 || h.T < 0 || h.T > INT32_MAX || seqs < 0 ||
        seqs > INT32_MAX)
        return PRISM_ERR_SHAPE;
    if (h.nslots < 0 || h.nslots > INT32_MAX || h.slot_ld < h.hv * h.dk * h.dv) return PRISM_ERR_SHAPE;
    if (h.v_ld < 0 || h.v_ld > 1 << 24) return PRISM_ERR_SHAPE;   // a chunk's values within unsigned 32-bit offsets
    if (!PRISM_ALIGNED(h.q, 16) || !PRISM_ALIGNED(h.k, 16) || !PRISM_ALIGNED(h.v, 16) || !PRISM_ALIGNED(h.out, 16) ||
        !PRISM_ALIGNED(h.state, 16) || h.q_ld % 8 || h.q_hs % 8 || h.k_ld % 8 || h.k_hs % 8 || h.v_ld % 8 || h.v_hs % 8 ||
        h.o_ld % 4 || h.o_hs % 4 || h.slot_ld % 4)
        return PRISM_ERR_ALIGN;
    const int64_t need = prompts ? workspace_bytes(h.T, seqs, h.hk, h.hv, h.dk) : 0;
    if (need > 0 && (!h.ws || h.ws_bytes < need)) return PRISM_ERR_ARG;
    if (need > 0 && !PRISM_ALIGNED(h.ws, 16)) return PRISM_ERR_ALIGN;
    if (h.T == 0 || seqs == 0 || h.nslots == 0) return PRISM_OK;
    const DeltaArgs a{h.q, h.k, h.v, h.q_ld, h.q_hs, h.k_ld, h.k_hs, h.v_ld, h.v_hs, h.g, h.beta, h.g_ld, h.b_ld, h.state,
                      h.slot_ld, h.out, h.o_ld, h.o_hs, prompts ? h.rows : nullptr, h.slots, prompts ? nullptr : h.rows,
                      (int)h.T, (int)seqs, (int)h.nslots, (int)h.hk, (int)h.hv, (int)h.norm, (float)h.scale, (float)h.eps};
    return need > 0 ? dispatch_chunks(a, h.dk, h.dv, (char*)h.ws, st) : dispatch_rec(a, h.dk, h.dv, st);
}

}  // namespace prism

using namespace prism;

extern "C" int prism_delta_step(const prism_delta_args* args, void* stream) {
    return args ? run(*args, false, (hipStream_t)stream) : (int)PRISM_ERR_ARG;
}

extern "C" int prism_delta_prefill(const prism_delta_args* args, void* stream) {
    return args ? run(*args, true, (hipStream_t)stream) : (int)PRISM_ERR_ARG;
}

extern "C" int64_t prism_delta_prefill_workspace_bytes(int64_t T, int64_t seqs, int64_t hk, int64_t hv, int64_t dk,
                                                       int64_t dv) {
    return dv == 64 || dv == 128 ? workspace_bytes(T, seqs, hk, hv, dk) : 0;
}
