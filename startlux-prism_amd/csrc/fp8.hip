// 8-bit floating point projections with block scales for gfx950: the activation quantizer, the weight packer and the GEMM.
//
//   y[m][j] = sum_b as[m][b] ws[j / 128][b] (sum_i a[m][128 b + i] w[j][128 b + i])
//
// A block's inner sum is one v_mfma_scale_f32_16x16x128_f8f6f4 (unit scales) from a zero accumulator; its four values of a
// lane are then folded into the fp32 sums by one fma each with as ws.  A operand: the weights, lane 16 g + r row r, bytes
// 16 p .. of piece p = inputs 64 p + 16 g .. + 15; B operand: the activations likewise (any order of the inputs serves, so
// long as both share it); D, lane 16 g + r: activation row r, weight rows 4 g .. + 3.  So as is one value of a lane per 16
// rows, and ws one of the wave.
//
// Inside the MFMA the 8 products of a lane's 8 neighbouring bytes are aligned on the largest of them with 13 bits kept below
// it (measured: beside a product of 2^16 one of 2^3 counts, one of 2^2 does not), the groups are added in fp32.  So a
// product p is off by at most 2^-13 max of its group; on normal values with a shared scale the sum is 1.5e-5 off (2-norm),
// against the 1.7e-3 of the bf16 output.  v_mfma_f32_16x16x32_fp8_fp8 gives the same bits at half the rate.
#include <math.h>

#include "common.h"
#include "fp8.h"

namespace prism {

// ---------------------------------------------------------------------------------------------------------- quantizers
// e4m3 codes of two values already divided by their scale, nearest even; |v| <= 448 (1 + 2^-23) unless not finite.
// v_cvt_pk_fp8_f32 saturates to NaN only past 464; NaN stays NaN, an infinity becomes NaN.
__device__ __forceinline__ uint32_t e4m3_pk4(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

__device__ __forceinline__ float block_scale(float amax) { return div_rn(fmaxf(amax, kAmaxMin), kE4m3Max); }

// The codes of N values over their scale.  y = x RN(1 / s) is within 3 x 2^-24 of the IEEE quotient, so both round to one code
// unless a midpoint between codes lies within 4 of its last places: there, and below 2^-6 where the codes' spacing is fixed,
// the quotient itself is taken.  Bits equal the division's.
template <int N>
__device__ __forceinline__ void codes_of(const float* v, float s, uint32_t* codes) {
    const float r = div_rn(1.f, s);
    float y[N];
    bool near = false;
#pragma unroll
    for (int i = 0; i < N; i++) {
        y[i] = mul_rn(v[i], r);
        const uint32_t u = __float_as_uint(y[i]) & 0x7fffffffu;
        near |= (u & 0xfffffu) - 0x7fffcu <= 8u || u - 1u < 0x3c800000u - 1u;
    }
    if (__builtin_expect(near, 0)) {
#pragma unroll
        for (int i = 0; i < N; i++) y[i] = div_rn(v[i], s);
    }
#pragma unroll
    for (int i = 0; i < N / 4; i++) codes[i] = e4m3_pk4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
}

// 8 neighbouring lanes per (row, 128 inputs), 16 inputs each, U such units per thread a grid apart (the loads of all go out
// first).  VEC: 16-byte loads and stores (aligned rows, k % 16 == 0).  magic: 2^32 / KB, for a unit's row.
// Memory bounds it: 8191 x 17408 bf16 (428 MB) 91.5 us (4.7 TB/s; a copy runs at 5.07), 109 with 8 inputs a lane.
template <bool F32, bool VEC, int U>
__global__ __launch_bounds__(256) void fp8_quant_kernel(const void* __restrict__ x, int64_t x_ld, uint8_t* __restrict__ q,
                                                        int64_t q_ld, float* __restrict__ s, int64_t s_ld,
                                                        const int32_t* __restrict__ n_rows, int T, int k, int KB, uint32_t magic) {
    kernel_args_now(x, x_ld, q, q_ld, s, s_ld, n_rows, T, k, KB, magic);
    const uint32_t units = (uint32_t)max(min(T, __ldg(n_rows)), 0) * KB, step = gridDim.x * 32;
    const int sub = threadIdx.x & 7;
    for (uint32_t u0 = blockIdx.x * 32 + (threadIdx.x >> 3); u0 < units; u0 += step * U) {
        float v[U][16];
        uint32_t row[U], b[U];
#pragma unroll
        for (int j = 0; j < U; j++) {
            const uint32_t u = min(u0 + j * step, units - 1);                 // (the last once more, not stored)
            row[j] = __umulhi(u, magic);
            b[j] = u - row[j] * KB;
            if (b[j] >= (uint32_t)KB) row[j]++, b[j] -= KB;
            const int c = b[j] * 128 + sub * 16;
            if (VEC) {
                const int at = min(c, k - 16);                                // (past the last input: made zeros)
                if (F32) {
                    const v4f* p = reinterpret_cast<const v4f*>(reinterpret_cast<const float*>(x) + row[j] * x_ld + at);
#pragma unroll
                    for (int h = 0; h < 4; h++) {
                        const v4f f = __builtin_nontemporal_load(p + h);
#pragma unroll
                        for (int i = 0; i < 4; i++) v[j][4 * h + i] = f[i];
                    }
                } else {
                    const v4u* p = reinterpret_cast<const v4u*>(reinterpret_cast<const uint16_t*>(x) + row[j] * x_ld + at);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const v4u f = __builtin_nontemporal_load(p + h);
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            v[j][8 * h + 2 * i] = bf16_to_f32(f[i] & 0xffff), v[j][8 * h + 2 * i + 1] = __uint_as_float(f[i] & 0xffff0000u);
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; i++) v[j][i] = c < k ? v[j][i] : 0.f;
            } else {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int at = min(c + i, k - 1);
                    v[j][i] = F32 ? reinterpret_cast<const float*>(x)[row[j] * x_ld + at]
                                  : bf16_to_f32(reinterpret_cast<const uint16_t*>(x)[row[j] * x_ld + at]);
                    v[j][i] = c + i < k ? v[j][i] : 0.f;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < U; j++) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < 16; i++) m = fmaxf(m, fabsf(v[j][i]));
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, kWave));
            const float sc = block_scale(m);
            uint32_t o[4];
            codes_of<16>(v[j], sc, o);
            if (u0 + j * step >= units) continue;
            uint8_t* to = q + row[j] * q_ld + b[j] * 128 + sub * 16;
            if (VEC) {
                __builtin_nontemporal_store(v4u{o[0], o[1], o[2], o[3]}, reinterpret_cast<v4u*>(to));
            } else {
                *reinterpret_cast<v2u*>(to) = v2u{o[0], o[1]};
                *reinterpret_cast<v2u*>(to + 8) = v2u{o[2], o[3]};
            }
            if (sub == 0) s[row[j] * s_ld + b[j]] = sc;
        }
    }
}

// One workgroup per 128 x 128 block: thread t holds row t / 2's 64 inputs of half t % 2.
__global__ __launch_bounds__(256) void fp8_pack_kernel(const void* __restrict__ w, int f32, int64_t ld,
                                                       uint8_t* __restrict__ chunks, float* __restrict__ ws, int n, int k,
                                                       int KB) {
    __shared__ float red[4];
    const int b = blockIdx.x, nb = blockIdx.y, t = threadIdx.x, row = nb * 128 + t / 2, half = t & 1;
    float v[64], m = 0.f;
#pragma unroll
    for (int i = 0; i < 64; i++) {
        const int c = b * 128 + half * 64 + i;
        v[i] = 0.f;
        if (row < n && c < k)
            v[i] = f32 ? reinterpret_cast<const float*>(w)[row * ld + c]
                       : bf16_to_f32(reinterpret_cast<const uint16_t*>(w)[row * ld + c]);
        m = fmaxf(m, fabsf(v[i]));
    }
    m = wave_max(m);
    if ((t & 63) == 0) red[t >> 6] = m;
    __syncthreads();
    const float sc = block_scale(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    if (t == 0) ws[(int64_t)nb * KB + b] = sc;
    if (row >= (n + 15) / 16 * 16) return;
    uint8_t* c = chunks + ((int64_t)(row / 16) * KB + b) * 2048 + half * 1024 + (row & 15) * 16;
#pragma unroll
    for (int g = 0; g < 4; g++) {
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
            o[i] = e4m3_pk4(div_rn(v[16 * g + 4 * i], sc), div_rn(v[16 * g + 4 * i + 1], sc),
                            div_rn(v[16 * g + 4 * i + 2], sc), div_rn(v[16 * g + 4 * i + 3], sc));
        *reinterpret_cast<v4u*>(c + 256 * g) = v4u{o[0], o[1], o[2], o[3]};
    }
}

// ---------------------------------------------------------------------------------------------------------------- GEMM
__device__ __forceinline__ v8i join8(v4i lo, v4i hi) { return v8i{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w}; }

__device__ __forceinline__ v4f fp8_mfma(v8i w, v8i a) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
}

__device__ __forceinline__ v4f fold(v4f t, float s, v4f acc) {
    return v4f{__builtin_fmaf(t.x, s, acc.x), __builtin_fmaf(t.y, s, acc.y), __builtin_fmaf(t.z, s, acc.z),
               __builtin_fmaf(t.w, s, acc.w)};
}

struct Fp8Gemm {
    const uint8_t* a;
    int64_t a_ld;
    const float* as;
    int64_t as_ld;
    const uint8_t* w;
    const float* ws;
    void* out;
    int64_t o_ld;
    const int32_t* n_rows;
    float* part;             // split K: fp32 [splits][T][n rounded up to 4]
    const uint8_t* pa;       // panels: the activations as chunks [ceil(T / 16)][KB][2048] in the weights' order, or null,
    const float* ps;         // and their scales [KB][ps_ld]
    int ps_ld;
    int T, n, k, KB, NT;     // NT: 16-row weight tiles
    int vec;                 // the output's rows take whole stores of four values (2: of eight)
};

// Four outputs of row m, columns j .. j + 3 (those below n).
template <int EPI>
__device__ __forceinline__ void store4(const Fp8Gemm& g, int m, int j, v4f y) {
    if (EPI == 0) {
        uint16_t* o = reinterpret_cast<uint16_t*>(g.out) + m * g.o_ld + j;
        if (g.vec && j + 3 < g.n) {
            *reinterpret_cast<v2u*>(o) = v2u{f32_to_bf16(y.x) | f32_to_bf16(y.y) << 16, f32_to_bf16(y.z) | f32_to_bf16(y.w) << 16};
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (j + i < g.n) o[i] = (uint16_t)f32_to_bf16(y[i]);
        }
    } else {
        float* o = reinterpret_cast<float*>(g.out) + m * g.o_ld + j;
        if (g.vec && j + 3 < g.n) {
            v4f* p = reinterpret_cast<v4f*>(o);
            const v4f h = *p;
            *p = v4f{add_rn(h.x, y.x), add_rn(h.y, y.y), add_rn(h.z, y.z), add_rn(h.w, y.w)};
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (j + i < g.n) o[i] = add_rn(o[i], y[i]);
        }
    }
}

// Few rows (up to 16 MT): a workgroup owns N 16-row weight tiles, its W waves take the blocks of 128 inputs in turn (wave w block
// w, w + W, ...) straight from memory into registers, D blocks ahead, and add their sums through LDS, wave after wave.  Rows
// past T and blocks past the last read as zeros: their offsets lie past the buffers' range, which costs no traffic, and the loop
// has no branches.  Eight neighbouring lanes load an activation row's 128 bytes (a row per lane, as the MFMA wants it, takes
// the memory pipeline four times as long); the wave turns them in 2 KB of its own LDS per 16 rows: piece c of row r lies at
// slot c ^ (r % 8), so that the 16 rows of a fragment read lie on distinct banks.
// PA 1: up to 8 rows, one load a block instead of two.
// One launch, no join: for small weights and few rows.  What a load takes to issue counts as much as its bytes: 1 x 5120 x 5120 (320
// workgroups) took 10.1 us with the last round of a ring asking past the end and two loads of activations a block, 8.8 without
// the second, 7.4 with neither (8 waves; 4: 6.5-7.3, 3.6-4.1 TB/s; 1 x 13824 x 5120 13.3 and 12.8, 5.5 TB/s; 64 x 12544 x 1128 11.8
// and 9.0).  More stages than 5 or fewer: 7.6 (4), 7.7 (3), 8.1 (7).
constexpr int kStreamWaves = 4;
template <int MT, int N, int D, int PA, int EPI>
__global__ __launch_bounds__(64 * kStreamWaves) void fp8_stream_kernel(Fp8Gemm g) {
    constexpr int W = kStreamWaves;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    // (arguments loaded where they are first used come one memory round trip after another)
    kernel_args_now(g.a, g.a_ld, g.as, g.as_ld, g.w, g.ws, g.out, g.o_ld, g.n_rows, g.T, g.n, g.KB, g.NT, g.vec);
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, gr = lane >> 4;
    const int t0 = blockIdx.x * N, m0 = blockIdx.y * 16 * MT;
    const int n_rows = __builtin_amdgcn_readfirstlane(__ldg(g.n_rows));
    const int tiles = g.NT - t0, KB = g.KB;
    const uint32_t tile = (uint32_t)KB * 2048;
    const __amdgpu_buffer_rsrc_t wr = buf_rsrc(g.w + (int64_t)t0 * tile);
    const __amdgpu_buffer_rsrc_t br = buf_rsrc(g.ws + (int64_t)(t0 >> 3) * KB);    // (N tiles lie in one block of 128 rows)
    constexpr uint32_t kOut = 0x80000000u;
    struct Stage {
        v4i w[N][2], a[MT][PA];
        float s[MT], sw;
    } st[D];
    auto issue_w = [&](Stage& x, int b) {
        const uint32_t bc = min(b, KB - 1), past = b < KB ? 0u : kOut;                 // (wave-uniform)
        x.sw = __uint_as_float(buf_load4(br, past, bc * 4));
#pragma unroll
        for (int t = 0; t < N; t++)
#pragma unroll
            for (int p = 0; p < 2; p++) x.w[t][p] = buf_load16<kBufNT>(wr, (lane * 16 | past) + p * 1024, min(t, tiles - 1) * tile + bc * 2048);
    };
    // all T rows are read, those not live too: no load waits for the live count
    const int rows = min(g.T - m0, 16 * MT);
    const __amdgpu_buffer_rsrc_t ar = buf_rsrc_n(g.a + m0 * g.a_ld, (uint32_t)((rows - 1) * g.a_ld + KB * 128));
    const __amdgpu_buffer_rsrc_t sr = buf_rsrc_n(g.as + m0 * g.as_ld, (uint32_t)((rows - 1) * g.as_ld + KB) * 4);
    uint32_t aoff[MT][PA], soff[MT];
#pragma unroll
    for (int c = 0; c < MT; c++) {
#pragma unroll
        for (int p = 0; p < PA; p++) {
            const int m = 16 * c + 8 * p + (lane >> 3);
            aoff[c][p] = m < rows ? (uint32_t)(m * g.a_ld + 16 * (lane & 7)) : kOut;
        }
        soff[c] = 16 * c + r < rows ? (uint32_t)((16 * c + r) * g.as_ld) * 4 : kOut;
    }
    auto issue_a = [&](Stage& x, int b) {
        const uint32_t bc = min(b, KB - 1), past = b < KB ? 0u : kOut;
#pragma unroll
        for (int c = 0; c < MT; c++) {
#pragma unroll
            for (int p = 0; p < PA; p++) x.a[c][p] = buf_load16(ar, aoff[c][p] | past, bc * 128);
            x.s[c] = __uint_as_float(buf_load4(sr, soff[c] | past, bc * 4));
        }
    };
    uint8_t* turn = lds + w * MT * 2048;
    const int put = (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) * 16);
    const int get0 = r * 128 + ((gr ^ (r & 7)) * 16), get1 = r * 128 + (((4 + gr) ^ (r & 7)) * 16);
    v4f acc[N][MT];
#pragma unroll
    for (int t = 0; t < N; t++)
#pragma unroll
        for (int c = 0; c < MT; c++) acc[t][c] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < D; d++) {
        issue_w(st[d], w + d * W);
        issue_a(st[d], w + d * W);
        __builtin_amdgcn_sched_barrier(0);
    }
    const int live = min(g.T, n_rows) - m0;
    if (live <= 0) return;
    auto use = [&](const Stage& x) {
#pragma unroll
        for (int c = 0; c < MT; c++)
#pragma unroll
            for (int p = 0; p < PA; p++) *reinterpret_cast<v4i*>(turn + c * 2048 + p * 1024 + put) = x.a[c][p];
#pragma unroll
        for (int c = 0; c < MT; c++) {
            const v8i a = join8(*reinterpret_cast<const v4i*>(turn + c * 2048 + get0),
                                *reinterpret_cast<const v4i*>(turn + c * 2048 + get1));
            const float s = mul_rn(x.s[c], x.sw);
#pragma unroll
            for (int t = 0; t < N; t++) acc[t][c] = fold(fp8_mfma(join8(x.w[t][0], x.w[t][1]), a), s, acc[t][c]);
        }
    };
    for (int b = w; b + D * W < KB; b += D * W) {
#pragma unroll
        for (int d = 0; d < D; d++) {
            use(st[d]);
            issue_w(st[d], b + (d + D) * W);
            issue_a(st[d], b + (d + D) * W);
            // (else the uses of all stages gather in front and wait for all loads; the loads before the loop are kept in the same
            // order, as the wait in it has to serve both)
            __builtin_amdgcn_sched_barrier(0);
        }
    }
#pragma unroll
    for (int d = 0; d < D; d++) {                       // (the last round asks for nothing: loads past the end cost their issue)
        use(st[d]);
        __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();                                                                   // (the sums lie over the turns)
    v4f* red = reinterpret_cast<v4f*>(lds);
#pragma unroll
    for (int t = 0; t < N; t++)
#pragma unroll
        for (int c = 0; c < MT; c++) red[((t * MT + c) * W + w) * 64 + lane] = acc[t][c];
    __syncthreads();
    for (int i = w; i < N * MT; i += W) {
        v4f y = red[i * W * 64 + lane];
#pragma unroll
        for (int j = 1; j < W; j++) {
            const v4f z = red[(i * W + j) * 64 + lane];
            y = v4f{add_rn(y.x, z.x), add_rn(y.y, z.y), add_rn(y.z, z.z), add_rn(y.w, z.w)};
        }
        const int m = 16 * (i % MT) + r, j = (t0 + i / MT) * 16 + 4 * gr;
        if (m < live) store4<EPI>(g, m0 + m, j, y);
    }
}

// LDS-DMA by buffer offsets: each lane's 16 bytes from voff (VGPR) + soff (SGPR) to the wave's LDS base + lane x 16.
__device__ __forceinline__ void buf_dma16(__amdgpu_buffer_rsrc_t r, void* lds, uint32_t voff, uint32_t soff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, (int)voff, (int)soff, 0, 0);
}
__device__ __forceinline__ void copy4(const void* g, void* lds) {
    __builtin_amdgcn_global_load_lds(g, (__attribute__((address_space(3))) void*)lds, 4, 0, 0);
}

// Many rows: WM x WN waves of 16 AR activation rows by 16 BR weight rows; both operands by LDS-DMA, NS stages of 128 inputs.
// Weight chunks lie in LDS as in memory (a lane's fragments are contiguous); an activation row's 128 bytes lie as eight
// 16-byte pieces, piece c of row r at slot c ^ (r % 8), so that eight neighbouring lanes copy one row and the 16 rows of a
// fragment read lie on distinct banks.  Scales: those of the rows, then those of the weights' blocks of 128.
template <int WM, int WN, int AR, int BR>
struct Fp8Tile {
    static constexpr int W = WM * WN, TW = BR * WN, TA = AR * WM;
    static constexpr int AQ = TW * 2048, SC = (TA * 16 + 63) / 64, AS = AQ + TA * 2048, WS = AS + SC * 256, SINK = WS + 256;
    // every wave makes the same number of copies a stage, which the counted waits rely on: surplus ones go to the sink
    static constexpr int WD = (TW * 2 + W - 1) / W, AD = (TA * 2 + W - 1) / W, COPIES = WD + AD + 1;
    static constexpr int BYTES = SINK + 1024;
    static_assert(SC + 1 <= W, "a wave per 64 rows' scales and one for the weights'");
    static_assert(TW % 8 == 0 || 8 % TW == 0, "a workgroup's tiles and the blocks of 128 rows");
};

// A stage's first fragments are read before the previous stage's last products: one barrier a stage, right before those, says
// that the next stage has arrived and that this one has been read, so its place takes the copies of stage b + NS.  Within a
// stage each 16 rows' fragment is read one step ahead, and a step's results are folded under the next step's products.
// EPI 2: fp32 partial sums of this part of K to g.part.  PAN: the activations from panels.
//
// What bounds it: the copies into LDS.  At 8191 x 27648 x 5120 (256 x 256 tiles, 64 KB a stage from the L2s) the copies alone take
// 961 us from panels and 1081 from rows, the products alone 934, both 1113-1164 from card to card (1.99-2.08 PFLOP/s); at 333 x 5120 x 17408 the copies
// alone take all of the 45 us (605 MB from the L2s, 13 TB/s; 145 MB of it from memory).  Few rows run at the weights' rate (16 x 5120 x
// 17408: 15.9 us, 5.6 TB/s, and the join).  Measured and dropped: fragments read where they are used (1292), 128 x 256 tiles of 4
// waves (a third to twice slower: one wave a SIMD), 256 x 128 tiles (333 rows 63, 4096 x 5120 x 5120 149 against 142), six stages for
// few rows (23.0 against 21.6), the copies through registers (alone 720, but then the products wait for them: 1244 and more).
template <int WM, int WN, int AR, int BR, int NS, int EPI, bool PAN>
__global__ __launch_bounds__(64 * WM * WN, 2) void fp8_tile_kernel(Fp8Gemm g, int tiles_m, int tiles_n, int splits) {
    using S = Fp8Tile<WM, WN, AR, BR>;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    kernel_args_now(g.a, g.a_ld, g.as, g.as_ld, g.w, g.ws, g.n_rows, g.pa, g.ps, g.ps_ld, g.T, g.KB, g.NT, tiles_m, tiles_n, splits);
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, gr = lane >> 4;
    const int tiles = tiles_m * tiles_n, part = blockIdx.x / tiles;       // (a part's tiles together, as their order wants)
    int pm, pn;
    xcd_tile_coords(blockIdx.x - part * tiles, tiles_m, tiles_n, pm, pn);
    const int m0 = pm * 16 * S::TA, t0 = pn * S::TW, KB = g.KB;
    const int live = __builtin_amdgcn_readfirstlane(min(g.T, __ldg(g.n_rows)));
    if (m0 >= live) return;
    const int b0 = (int)((int64_t)KB * part / splits), nb = (int)((int64_t)KB * (part + 1) / splits) - b0;

    const __amdgpu_buffer_rsrc_t wr = buf_rsrc(g.w + ((int64_t)t0 * KB + b0) * 2048);
    const __amdgpu_buffer_rsrc_t ar = PAN ? buf_rsrc(g.pa + ((int64_t)(m0 / 16) * KB + b0) * 2048)
                                          : buf_rsrc_n(g.a + m0 * g.a_ld + b0 * 128,
                                                        (uint32_t)((min(live - m0, 16 * S::TA) - 1) * g.a_ld + nb * 128));
    uint32_t wsoff[S::WD], avoff[S::AD], asoff[S::AD];
    int wdst[S::WD], adst[S::AD];
#pragma unroll
    for (int i = 0; i < S::WD; i++) {
        const int c = w * S::WD + i;
        wsoff[i] = (uint32_t)(min(t0 + c / 2, g.NT - 1) - t0) * KB * 2048 + (c & 1) * 1024;
        wdst[i] = c < 2 * S::TW ? c * 1024 : S::SINK;
    }
#pragma unroll
    for (int i = 0; i < S::AD; i++) {
        const int c = w * S::AD + i, row = c * 8 + lane / 8;               // (rows past the live ones: zeros, past the range)
        avoff[i] = PAN ? lane * 16u : m0 + row < live ? (uint32_t)(row * g.a_ld) + (((lane & 7) ^ (row & 7)) * 16) : 0x80000000u;
        asoff[i] = PAN ? (uint32_t)(min(m0 / 16 + c / 2, (live - 1) / 16) - m0 / 16) * KB * 2048 + (c & 1) * 1024 : 0u;
        adst[i] = c < 2 * S::TA ? S::AQ + c * 1024 : S::SINK;
    }
    const float* ssrc = PAN ? g.ps + (int64_t)b0 * g.ps_ld + min(m0 + w * 64 + lane, live - 1)
                            : g.as + min(m0 + w * 64 + lane, live - 1) * g.as_ld + b0;
    const int sstep = PAN && w < S::SC ? g.ps_ld : 1;
    if (w >= S::SC) ssrc = g.ws + (int64_t)min((t0 >> 3) + lane, (g.NT - 1) >> 3) * KB + b0;
    const int sdst = w < S::SC ? S::AS + w * 256 : w == S::SC ? S::WS : S::SINK;
    auto issue = [&](int b) {
        uint8_t* l = lds + (b % NS) * S::BYTES;
#pragma unroll
        for (int i = 0; i < S::WD; i++) buf_dma16(wr, l + wdst[i], lane * 16, wsoff[i] + b * 2048);
#pragma unroll
        for (int i = 0; i < S::AD; i++) buf_dma16(ar, l + adst[i], avoff[i], asoff[i] + b * (PAN ? 2048 : 128));
        copy4(ssrc + (int64_t)b * sstep, l + sdst);
    };

    const int wn = w % WN, wm = w / WN;
    const int wat = BR * wn * 2048 + lane * 16, wsat = S::WS + (((t0 + BR * wn) >> 3) - (t0 >> 3)) * 4;
    const int row0 = 16 * AR * wm + r, aat = S::AQ + (PAN ? AR * wm * 2048 + lane * 16 : row0 * 128), sat = S::AS + row0 * 4;
    const int s0 = PAN ? 0 : (gr ^ (r & 7)) * 16, s1 = PAN ? 1024 : ((4 + gr) ^ (r & 7)) * 16;
    v8i wf[BR], af[2];
    float s[2], sw;
    v4f t[2][BR], acc[BR][AR];
    auto read_w = [&](const uint8_t* l, int a) {
        wf[a] = join8(*reinterpret_cast<const v4i*>(l + wat + a * 2048), *reinterpret_cast<const v4i*>(l + wat + a * 2048 + 1024));
    };
    auto read_a = [&](const uint8_t* l, int c) {
        const uint8_t* p = l + aat + c * 2048;
        af[c & 1] = join8(*reinterpret_cast<const v4i*>(p + s0), *reinterpret_cast<const v4i*>(p + s1));
        s[c & 1] = *reinterpret_cast<const float*>(l + sat + c * 64);
    };
    // step c of a stage but the last: its products, the next step's fragment, the previous step's fold
    auto step = [&](const uint8_t* l, int c, bool fold_before, float& before) {
        const float now = mul_rn(s[c & 1], sw);
        read_a(l, c + 1);
#pragma unroll
        for (int a = 0; a < BR; a++) t[c & 1][a] = fp8_mfma(wf[a], af[c & 1]);
        if (fold_before) {
#pragma unroll
            for (int a = 0; a < BR; a++) acc[a][(c + AR - 1) % AR] = fold(t[(c + 1) & 1][a], before, acc[a][(c + AR - 1) % AR]);
        }
        before = now;
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int a = 0; a < BR; a++)
#pragma unroll
        for (int c = 0; c < AR; c++) acc[a][c] = v4f{0.f, 0.f, 0.f, 0.f};
    static_assert(AR % 2 == 0, "a stage's last step and the next one's first use different registers");
#pragma unroll
    for (int i = 0; i < NS; i++)
        if (i < nb) issue(i);
    if (nb >= NS) vm_wait<(NS - 1) * S::COPIES>();
    else vm_wait<0>();
    lds_barrier();
#pragma unroll
    for (int a = 0; a < BR; a++) read_w(lds, a);
    read_a(lds, 0);
    sw = *reinterpret_cast<const float*>(lds + wsat);
    float before = 0.f;
#pragma unroll
    for (int c = 0; c < AR - 1; c++) step(lds, c, c > 0, before);
    for (int b = 1; b < nb; b++) {
        // stage b is there (in flight at most the stages after it that were requested) and stage b - 1 has been read
        if (b + NS - 1 <= nb) vm_wait<(NS - 2) * S::COPIES>();
        else vm_wait<0>();
        lds_barrier();
        if (b + NS - 1 < nb) issue(b + NS - 1);
        const uint8_t* l = lds + (b % NS) * S::BYTES;
        {
            const float now = mul_rn(s[(AR - 1) & 1], sw);
#pragma unroll
            for (int a = 0; a < BR; a++) {
                t[(AR - 1) & 1][a] = fp8_mfma(wf[a], af[(AR - 1) & 1]);
                read_w(l, a);
            }
            read_a(l, 0);
            sw = *reinterpret_cast<const float*>(l + wsat);
#pragma unroll
            for (int a = 0; a < BR; a++) acc[a][AR - 2] = fold(t[AR & 1][a], before, acc[a][AR - 2]);
            before = now;
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int c = 0; c < AR - 1; c++) step(l, c, true, before);
    }
    {
        const float now = mul_rn(s[(AR - 1) & 1], sw);
#pragma unroll
        for (int a = 0; a < BR; a++) t[(AR - 1) & 1][a] = fp8_mfma(wf[a], af[(AR - 1) & 1]);
#pragma unroll
        for (int a = 0; a < BR; a++) {
            acc[a][AR - 2] = fold(t[AR & 1][a], before, acc[a][AR - 2]);
            acc[a][AR - 1] = fold(t[(AR - 1) & 1][a], now, acc[a][AR - 1]);
        }
    }
    // bf16 rows of 64 outputs a wave, 128 bytes: turned in the wave's own part of the stages' LDS, so that eight neighbouring lanes
    // store one row (in the products' order a row gets 32 bytes at a time: 1595 x 24704 x 1152 76.9 -> 71.5 us, 8191 x
    // 27648 x 5120 1125 -> 1113)
    if constexpr (EPI == 0 && BR == 4) {
        const int j0 = 16 * (t0 + 4 * wn);
        if (g.vec == 2) lds_barrier();                                                 // (every wave has read its last fragments)
        if (g.vec == 2 && j0 + 64 <= g.n) {
            uint8_t* own = lds + w * AR * 2048;
            static_assert(S::W * AR * 2048 <= NS * S::BYTES, "the waves' outputs lie in the stages");
#pragma unroll
            for (int c = 0; c < AR; c++)
#pragma unroll
                for (int a = 0; a < 4; a++) {
                    const v4f y = acc[a][c];
                    *reinterpret_cast<v2u*>(own + (16 * c + r) * 128 + (((2 * a + (gr >> 1)) ^ (r & 7)) * 16) + (gr & 1) * 8) =
                        v2u{f32_to_bf16(y.x) | f32_to_bf16(y.y) << 16, f32_to_bf16(y.z) | f32_to_bf16(y.w) << 16};
                }
            const int sub = lane >> 3, piece = lane & 7;
#pragma unroll
            for (int i = 0; i < AR * 2; i++) {
                const int m = m0 + 16 * AR * wm + 8 * i + sub;
                if (m >= live) continue;
                *reinterpret_cast<v4u*>(reinterpret_cast<uint16_t*>(g.out) + m * g.o_ld + j0 + 8 * piece) =
                    *reinterpret_cast<const v4u*>(own + (8 * i + sub) * 128 + ((piece ^ sub) * 16));
            }
            return;
        }
    }
#pragma unroll
    for (int c = 0; c < AR; c++) {
        const int m = m0 + 16 * (AR * wm + c) + r;
        if (m >= live) continue;
#pragma unroll
        for (int a = 0; a < BR; a++) {
            const int j = 16 * (t0 + BR * wn + a) + 4 * gr;
            if (EPI == 2) {
                const int64_t n4 = (g.n + 3) & ~3;
                if (j < n4) *reinterpret_cast<v4f*>(g.part + ((int64_t)part * g.T + m) * n4 + j) = acc[a][c];
            } else if (j < g.n) {
                store4<EPI>(g, m, j, acc[a][c]);
            }
        }
    }
}

// Activation rows -> panels: a workgroup per chunk of 16 rows x 128 inputs, eight lanes a row's 128 bytes.  In rows a tile's
// copies are 128 bytes here and there, and its scales 4 bytes of a line each; in panels both are whole.  8191 x 5120: 21 us.
__global__ __launch_bounds__(128) void fp8_panel_kernel(Fp8Gemm g, uint8_t* __restrict__ pa, float* __restrict__ ps) {
    kernel_args_now(g.a, g.a_ld, g.as, g.as_ld, g.T, g.KB, g.ps_ld, pa, ps);
    const int b = blockIdx.x, row = threadIdx.x >> 3, c = threadIdx.x & 7, m = blockIdx.y * 16 + row;
    if (m >= g.T) return;                                      // (rows that are not live are copied too: no load before these)
    const v4i v = *reinterpret_cast<const v4i*>(g.a + m * g.a_ld + b * 128 + c * 16);
    *reinterpret_cast<v4i*>(pa + ((int64_t)blockIdx.y * g.KB + b) * 2048 + (c >> 2) * 1024 + ((c & 3) * 16 + row) * 16) = v;
    if (c == 0) ps[(int64_t)b * g.ps_ld + m] = g.as[m * g.as_ld + b];
}

// The parts of a split K added in their order: a thread per four outputs, the loads of four parts at once.
template <int EPI>
__global__ __launch_bounds__(64) void fp8_join_kernel(Fp8Gemm g, int splits) {
    kernel_args_now(g.part, g.out, g.o_ld, g.n_rows, g.T, g.n, g.vec, splits);
    const int n4 = (g.n + 3) & ~3, m = blockIdx.y, j = (blockIdx.x * 64 + threadIdx.x) * 4;
    const int n_rows = __ldg(g.n_rows);
    if (j >= n4) return;
    const float* p = g.part + (int64_t)m * n4 + j;
    v4f y = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < splits; i0 += 4) {
        v4f v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = *reinterpret_cast<const v4f*>(p + (int64_t)min(i0 + i, splits - 1) * g.T * n4);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (i0 + i >= splits) continue;
            if (i0 + i == 0) y = v[0];
            else y = v4f{add_rn(y.x, v[i].x), add_rn(y.y, v[i].y), add_rn(y.z, v[i].z), add_rn(y.w, v[i].w)};
        }
    }
    if (m < n_rows) store4<EPI>(g, m, j, y);
}

// Which kernel, into how many parts K is split, and whether the activations go to panels first: the least of the times in us that
// a model gives each (random codes, weights from memory; KB blocks of 128 inputs, NT 16-row weight tiles).  The model's constants come
// from the measurements named here, and at the chosen form it is within 15% of the time (1 x 5120 x 5120 7.9 and 7.1, 16 x 5120 x 17408
// 23.4 and 20.8, 48 x 13824 x 5120 21.1 and 21.7, 128 x 27648 x 5120 40.5 and 46.2, 1000 x 5120 x 5120 50.4 and 49, 4096 x 5120 x 5120 162
// and 155): forms nearer each other are told apart by the constants, not by a measurement of both.  Weights that the 256 MB
// memory-side cache holds take less than it says: three in turn 6.8, 18.8 and 17.0.
//   stream   2.6 + (workgroups on the fullest CU) a per block, and 0.5 per workgroup after the first; a = 0.06, 0.085, 0.1, 0.127, 0.16
//            for 8, 16, 32, 48, 64 rows: 8 x 13824 x 5120 14.0 (measured; the best tile form 17.3), 8 x 5120 x 17408 21.2 (20.0), 16 x
//            1024 x 5120 5.9 (7.7), 16 x 5120 x 5120 9.8 (10.5), 16 x 5120 x 17408 27.2 (20.7), 64 x 5120 x 5120 15.5 (13.9)
//   tiles    2.5 + (stages) x, or the weights at 5.2 TB/s, less with under 256 workgroups (16 x 5120 x 17408 in 5 and 6 parts, 200 and
//            240 workgroups: 19.2 and 18.7): 32 x 128 (rows x outputs) x = 0.65 with 256 workgroups, down to half of that with few (16 x
//            512 x 17408 in 1 and 8 parts 47.8 and 10.7), 64 x 128 0.7, both per round of 256 (48 x 13824 x 5120 in 2 and 3 parts, 216
//            and 324 workgroups: 21.7 and 27.5); 128 x 128 x = 0.95 up to 256, else 1.4 per round of 512 (a part of a round counts
//            0.4 more than its share, up to a round); 256 x 256 x = 2 per whole 256: 333 x 5120 x 17408 on 128 x 128 in 4 parts 59,
//            256 x 256 in 6 61; 1000 x 5120 x 5120 59 and (3 parts) 50; 2048 x 13824 x 5120 193 and 160; 4096 x 5120 x 5120 144 and
//            158; 128 x 27648 x 5120 48, on 64 x 128 56
//   parts    3 + 1.1e-6 per part and output: written, read and added by a second launch
//   panels   from 256 rows, past 45 us on 128 x 128 tiles (333 x 5120 x 17408 60 -> 55; 4096 x 5120 x 5120 144 -> 139, for which the model
//            takes 256 x 256, 155; but 128 x 5120 x 17408 34 -> 38), past 100 on 256 x 256 (8191 x 27648 x 5120 1161 -> 1142, the copy
//            included; 2048 x 5120 x 5120 79 -> 81)
struct Fp8Plan {
    int kind;            // 0 stream; tiles of rows x outputs: 1 32 x 128, 2 64 x 128, 3 128 x 128, 4 256 x 256
    int splits;
    int panels;
};

inline Fp8Plan fp8_plan(int64_t T, int64_t n, int64_t k) {
    const int64_t NT = (n + 15) / 16, KB = (k + 127) / 128;
    const double read = (double)(NT * KB) * 2048 / 5.2e6;
    Fp8Plan best{4, 1, 0};
    double least = 1e30;
    if (T <= 64) {
        const int mt = (int)((T + 15) / 16);
        const int64_t per = mt == 1 ? 1 : 2, wgs = (NT + per - 1) / per;
        const double a[] = {T <= 8 ? 0.06 : 0.085, 0.1, 0.127, 0.16}, fullest = (double)((wgs + 255) / 256);
        least = 2.6 + fullest * a[mt - 1] * (double)(per * KB) + 0.5 * (fullest - 1);
        best = {0, 1, 0};
    }
    const int64_t rows[] = {32, 64, 128, 256}, tiles[] = {8, 8, 8, 16};
    for (int kind = T <= 32 ? 1 : 2; kind <= 4; kind++) {
        const int64_t wgs = (T + rows[kind - 1] - 1) / rows[kind - 1] * ((NT + tiles[kind - 1] - 1) / tiles[kind - 1]);
        for (int s = 1; s <= 8 && (s == 1 || (KB / s >= 4 && T <= 65535)); s++) {          // (the join's grid)
            const double w = (double)(wgs * s), stages = (double)((KB + s - 1) / s);
            const double x = kind == 1 ? 0.65 * (w > 256 ? ceil(w / 256) : 0.5 + w / 512) : kind == 2 ? 0.7 * ceil(w / 256)
                           : kind == 3 ? (w <= 256 ? 0.95 : 1.4 * fmin(ceil(w / 512), w > 512 ? w / 512 + 0.4 : 1)) : 2.0 * ceil(w / 256);
            const double t = 2.5 + fmax(stages * x, read * (w < 256 ? 1.25 - w / 1024 : 1)) + (s > 1 ? 3 + 1.1e-6 * s * (double)T * (double)n : 0);
            if (t < least) least = t, best = {kind, s, T >= 256 && T <= 65535 * 16 && ((kind == 3 && t > 45) || (kind == 4 && t > 100))};
        }
    }
    return best;
}

}  // namespace prism

using namespace prism;

extern "C" int prism_fp8_pack(const void* w, int f32, int64_t ld, uint8_t* chunks, float* ws, int64_t n, int64_t k,
                              void* stream) {
    if (!w || !chunks || !ws || (f32 != 0 && f32 != 1)) return PRISM_ERR_ARG;
    if (n < 1 || k < 1 || n > kFp8MaxDim || k > kFp8MaxDim || ld < k) return PRISM_ERR_SHAPE;
    if (!PRISM_ALIGNED(chunks, 16)) return PRISM_ERR_ALIGN;
    const int KB = (int)((k + 127) / 128);
    hipLaunchKernelGGL(fp8_pack_kernel, dim3(KB, (unsigned)((n + 127) / 128)), dim3(256), 0, (hipStream_t)stream, w, f32, ld,
                       chunks, ws, (int)n, (int)k, KB);
    PRISM_LAUNCH_CHECK();
    return PRISM_OK;
}

extern "C" int prism_fp8_quant(const prism_fp8_quant_args* args, void* stream) {
    if (!args) return PRISM_ERR_ARG;
    const prism_fp8_quant_args& h = *args;
    if (!h.x || !h.q || !h.s || !h.n_rows || (h.f32 != 0 && h.f32 != 1)) return PRISM_ERR_ARG;
    const int64_t KB = (h.k + 127) / 128;
    if (h.T < 0 || h.T > INT32_MAX || h.k < 1 || h.k > kFp8MaxDim || h.x_ld < 0 || h.q_ld < 0 || h.s_ld < 0)
        return PRISM_ERR_SHAPE;
    if (h.T > 1 && (h.q_ld < 128 * KB || h.s_ld < KB)) return PRISM_ERR_SHAPE;
    if (h.T * KB > INT32_MAX) return PRISM_ERR_SHAPE;
    if (!PRISM_ALIGNED(h.q, 8) || h.q_ld % 8) return PRISM_ERR_ALIGN;
    if (h.T == 0) return PRISM_OK;
    const bool vec = h.k % 16 == 0 && PRISM_ALIGNED(h.x, 16) && h.x_ld % (h.f32 ? 4 : 8) == 0 && PRISM_ALIGNED(h.q, 16) && h.q_ld % 16 == 0;
    const int64_t groups = (h.T * KB + 31) / 32;
    const hipStream_t st = (hipStream_t)stream;
#define FQ(F, V, U) \
    hipLaunchKernelGGL((fp8_quant_kernel<F, V, U>), dim3((unsigned)((groups + U - 1) / U < 4096 ? (groups + U - 1) / U : 4096)), \
                       dim3(256), 0, st, h.x, h.x_ld, h.q, h.q_ld, h.s, h.s_ld, h.n_rows, (int)h.T, (int)h.k, (int)KB, (uint32_t)(0xffffffffu / KB))
    const bool many = groups >= 2048;
    if (h.f32) {
        if (!vec) FQ(true, false, 1); else if (many) FQ(true, true, 2); else FQ(true, true, 1);
    } else {
        if (!vec) FQ(false, false, 1); else if (many) FQ(false, true, 2); else FQ(false, true, 1);
    }
#undef FQ
    PRISM_LAUNCH_CHECK();
    return PRISM_OK;
}

static int64_t fp8_part_bytes(const Fp8Plan& p, int64_t T, int64_t n) { return ((int64_t)p.splits * T * ((n + 3) & ~3) * 4 + 15) & ~15; }
static int64_t fp8_panel_bytes(int64_t T, int64_t k) { return (T + 15) / 16 * ((k + 127) / 128) * 2048; }

extern "C" int64_t prism_fp8_gemm_workspace_bytes(int64_t T, int64_t n, int64_t k) {
    if (T < 1 || n < 1 || k < 1) return 0;
    const Fp8Plan p = fp8_plan(T, n, k);
    return (p.splits > 1 ? fp8_part_bytes(p, T, n) : 0) + (p.panels ? fp8_panel_bytes(T, k) + (k + 127) / 128 * ((T + 63) & ~63) * 4 : 0);
}

extern "C" int prism_fp8_gemm(const prism_fp8_gemm_args* args, void* stream) {
    if (!args) return PRISM_ERR_ARG;
    const prism_fp8_gemm_args& h = *args;
    if (!h.a || !h.as || !h.w || !h.ws || !h.out || !h.n_rows || (h.epi != 0 && h.epi != 1)) return PRISM_ERR_ARG;
    if (h.T < 0 || h.T > INT32_MAX / 512 || h.n < 1 || h.k < 1 || h.n > kFp8MaxDim || h.k > kFp8MaxDim) return PRISM_ERR_SHAPE;
    const int64_t KB = (h.k + 127) / 128;
    // (the few rows' operands are reached by 31-bit offsets)
    if (h.a_ld < 0 || h.as_ld < 0 || h.o_ld < 0 || h.a_ld > kFp8MaxLd || h.as_ld > kFp8MaxLd) return PRISM_ERR_SHAPE;
    if (h.T > 1 && h.o_ld < h.n) return PRISM_ERR_SHAPE;
    if (!PRISM_ALIGNED(h.a, 16) || !PRISM_ALIGNED(h.w, 16) || h.a_ld % 16 || !PRISM_ALIGNED(h.as, 4)) return PRISM_ERR_ALIGN;
    if (!PRISM_ALIGNED(h.out, h.epi ? 4 : 2)) return PRISM_ERR_ALIGN;
    if (h.T == 0) return PRISM_OK;
    const int64_t need = prism_fp8_gemm_workspace_bytes(h.T, h.n, h.k);
    if (need > 0 && (!h.wsp || h.wsp_bytes < need)) return PRISM_ERR_ARG;
    if (need > 0 && !PRISM_ALIGNED(h.wsp, 16)) return PRISM_ERR_ALIGN;
    Fp8Gemm g{h.a, h.a_ld, h.as, h.as_ld, h.w, h.ws, h.out, h.o_ld, h.n_rows, (float*)h.wsp, nullptr, nullptr, 0, (int)h.T, (int)h.n,
              (int)h.k, (int)KB, (int)((h.n + 15) / 16), 0};
    g.vec = h.o_ld % 4 == 0 && PRISM_ALIGNED(h.out, h.epi ? 16 : 8);
    if (!h.epi && h.o_ld % 8 == 0 && PRISM_ALIGNED(h.out, 16)) g.vec = 2;
    const Fp8Plan p = fp8_plan(h.T, h.n, h.k);
    const hipStream_t st = (hipStream_t)stream;
    if (p.panels) {
        uint8_t* pa = (uint8_t*)h.wsp + (p.splits > 1 ? fp8_part_bytes(p, h.T, h.n) : 0);
        float* ps = (float*)(pa + fp8_panel_bytes(h.T, h.k));
        g.ps_ld = (int)((h.T + 63) & ~63);
        hipLaunchKernelGGL(fp8_panel_kernel, dim3(g.KB, (unsigned)((h.T + 15) / 16)), dim3(128), 0, st, g, pa, ps);
        PRISM_LAUNCH_CHECK();
        g.pa = pa, g.ps = ps;
    }
#define EP(f) do { if (h.epi) f(1); else f(0); } while (0)
    if (p.kind == 0) {
#define ST(MT, N, D, PA, E) \
        hipLaunchKernelGGL((fp8_stream_kernel<MT, N, D, PA, E>), dim3((g.NT + N - 1) / N, (unsigned)((h.T + 16 * MT - 1) / (16 * MT))), \
                           dim3(64 * kStreamWaves), (size_t)MT * 2 * kStreamWaves * 1024, st, g)
#define S0(E) ST(1, 1, 5, 1, E)
#define S1(E) ST(1, 1, 5, 2, E)
#define S2(E) ST(2, 2, 2, 2, E)
#define S3(E) ST(3, 2, 2, 2, E)
#define S4(E) ST(4, 2, 2, 2, E)
        if (h.T <= 8) EP(S0); else if (h.T <= 16) EP(S1); else if (h.T <= 32) EP(S2); else if (h.T <= 48) EP(S3); else EP(S4);
#undef S0
#undef S1
#undef S2
#undef S3
#undef S4
#undef ST
    } else {
#define TL(WM, WN, AR, BR, NS, E, PAN) do { \
        using S = Fp8Tile<WM, WN, AR, BR>; \
        const int tm = (int)((h.T + 16 * S::TA - 1) / (16 * S::TA)), tn = (g.NT + S::TW - 1) / S::TW; \
        if ((int64_t)tm * tn * p.splits > INT32_MAX) return PRISM_ERR_SHAPE; \
        allow_lds(fp8_tile_kernel<WM, WN, AR, BR, NS, E, PAN>, (size_t)S::BYTES * NS); \
        hipLaunchKernelGGL((fp8_tile_kernel<WM, WN, AR, BR, NS, E, PAN>), dim3((unsigned)(tm * tn * p.splits)), dim3(64 * WM * WN), \
                           (size_t)S::BYTES * NS, st, g, tm, tn, p.splits); \
    } while (0)
#define TP(WM, WN, AR, BR, NS, E) do { if (g.pa) TL(WM, WN, AR, BR, NS, E, true); else TL(WM, WN, AR, BR, NS, E, false); } while (0)
#define ALL(E) do { \
        if (p.kind == 1) TL(1, 4, 2, 2, 3, E, false); else if (p.kind == 2) TL(1, 4, 4, 2, 3, E, false); \
        else if (p.kind == 3) TP(2, 2, 4, 4, 2, E); else TP(2, 4, 8, 4, 2, E); \
    } while (0)
        if (p.splits == 1) {
            EP(ALL);
        } else {
            ALL(2);
            PRISM_LAUNCH_CHECK();
            const dim3 grid((unsigned)((((g.n + 3) / 4) + 63) / 64), (unsigned)h.T);
            if (h.epi) hipLaunchKernelGGL((fp8_join_kernel<1>), grid, dim3(64), 0, st, g, p.splits);
            else hipLaunchKernelGGL((fp8_join_kernel<0>), grid, dim3(64), 0, st, g, p.splits);
        }
#undef ALL
#undef TP
#undef TL
    }
#undef EP
    PRISM_LAUNCH_CHECK();
    return PRISM_OK;
}
