// The gated delta rule of a linear-attention layer in serving (gfx950).  Per value head, with the state S fp32 [DK, DV],
// a = exp(g), key k and query q (normalised to length 1 in the kernel if asked, the query times a scale), all in fp32:
//   S <- a S;  u = beta (v - S^T k);  S <- S + k u^T;  o = S^T q.
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

__device__ __forceinline__ float wave_addf(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    return v;
}

// ------------------------------------------------------------------------------------------------------- recurrent form
// A workgroup holds NC columns of one head's state in registers from its only read to its only write: thread t the
// columns 4 (t % (NC / 4)) .. + 3 of the rows t / (NC / 4) + i RG.  Both sums over the rows, S^T k and S^T q, are taken
// of the decayed state at once (o = S^T q + (q . k) u), so a token costs one exchange between the waves.  Each wave
// holds its own copy of the token's key and query.  Bound by the state's bytes.
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
    for (int i = 0; i < RPT; i++) s[i] = *reinterpret_cast<const v4f*>(st + (rg + i * RG) * DV);
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
    for (int i = 0; i < RPT; i++) *reinterpret_cast<v4f*>(st + (rg + i * RG) * DV) = s[i];
}

template <int DK, int DV>
static int launch_rec(const DeltaArgs& a, hipStream_t st) {
    const int64_t heads = (int64_t)a.seqs * a.HV;
#define RC(NC) hipLaunchKernelGGL((delta_rec_kernel<DK, DV, NC>), dim3((unsigned)(heads * (DV / NC))), dim3(256), 0, st, a)
    if (heads * (DV / 32) <= INT32_MAX) RC(32); else return PRISM_ERR_SHAPE;
#undef RC
    return hipGetLastError() == hipSuccess ? (int)PRISM_OK : (int)PRISM_ERR_LAUNCH;
}

static int check(const DeltaArgs& a, int64_t rows, int64_t seqs, int64_t nslots, int64_t HK, int64_t HV, int64_t DK,
                 int64_t DV) {
    if (!a.q || !a.k || !a.v || !a.g || !a.beta || !a.state || !a.out || (a.norm != 0 && a.norm != 1)) return PRISM_ERR_ARG;
    if ((DK != 64 && DK != 128) || (DV != 64 && DV != 128)) return PRISM_ERR_SHAPE;
    if (HK < 1 || HV < HK || HV % HK || HV > 65536 || rows < 0 || rows > INT32_MAX || seqs < 0 || seqs > INT32_MAX)
        return PRISM_ERR_SHAPE;
    if (nslots < 0 || nslots > INT32_MAX || a.lds_ < HV * DK * DV) return PRISM_ERR_SHAPE;
    if (!PRISM_ALIGNED(a.q, 16) || !PRISM_ALIGNED(a.k, 16) || !PRISM_ALIGNED(a.v, 16) || !PRISM_ALIGNED(a.out, 16) ||
        !PRISM_ALIGNED(a.state, 16) || a.ldq % 8 || a.hq_s % 8 || a.ldk % 8 || a.hk_s % 8 || a.ldv % 8 || a.hv_s % 8 ||
        a.ldo % 4 || a.ho_s % 4 || a.lds_ % 4)
        return PRISM_ERR_ALIGN;
    return PRISM_OK;
}

static int dispatch_rec(const DeltaArgs& a, int64_t DK, int64_t DV, hipStream_t st) {
    if (DK == 64) return DV == 64 ? launch_rec<64, 64>(a, st) : launch_rec<64, 128>(a, st);
    return DV == 64 ? launch_rec<128, 64>(a, st) : launch_rec<128, 128>(a, st);
}

}  // namespace prism

using namespace prism;

extern "C" int prism_delta_step(const uint16_t* q, int64_t ldq, int64_t hq_s, const uint16_t* k, int64_t ldk,
                                int64_t hk_s, const uint16_t* v, int64_t ldv, int64_t hv_s, const float* g, int64_t ldg,
                                const float* beta, int64_t ldb, float* state, int64_t slot_stride, int64_t nslots,
                                const int32_t* slots, float* out, int64_t ldo, int64_t ho_s, const int32_t* n_rows,
                                int64_t T, int64_t HK, int64_t HV, int64_t DK, int64_t DV, int norm, float scale,
                                float eps, void* stream) {
    const DeltaArgs a{q, k, v, ldq, hq_s, ldk, hk_s, ldv, hv_s, g, beta, ldg, ldb, state, slot_stride, out, ldo, ho_s,
                      nullptr, slots, n_rows, (int)T, (int)T, (int)nslots, (int)HK, (int)HV, norm, scale, eps};
    const int rc = check(a, T, T, nslots, HK, HV, DK, DV);
    if (rc != PRISM_OK) return rc;
    if (!n_rows) return PRISM_ERR_ARG;
    if (T == 0 || nslots == 0) return PRISM_OK;
    return dispatch_rec(a, DK, DV, (hipStream_t)stream);
}

extern "C" int prism_delta_prefill(const uint16_t* q, int64_t ldq, int64_t hq_s, const uint16_t* k, int64_t ldk,
                                   int64_t hk_s, const uint16_t* v, int64_t ldv, int64_t hv_s, const float* g,
                                   int64_t ldg, const float* beta, int64_t ldb, float* state, int64_t slot_stride,
                                   int64_t nslots, const int32_t* slots, float* out, int64_t ldo, int64_t ho_s,
                                   const int32_t* cu, int64_t seqs, int64_t T, int64_t HK, int64_t HV, int64_t DK,
                                   int64_t DV, int norm, float scale, float eps, void* ws, int64_t ws_bytes,
                                   void* stream) {
    const DeltaArgs a{q, k, v, ldq, hq_s, ldk, hk_s, ldv, hv_s, g, beta, ldg, ldb, state, slot_stride, out, ldo, ho_s,
                      cu, slots, nullptr, (int)T, (int)seqs, (int)nslots, (int)HK, (int)HV, norm, scale, eps};
    const int rc = check(a, T, seqs, nslots, HK, HV, DK, DV);
    if (rc != PRISM_OK) return rc;
    if (!cu) return PRISM_ERR_ARG;
    if (T == 0 || seqs == 0 || nslots == 0) return PRISM_OK;
    return dispatch_rec(a, DK, DV, (hipStream_t)stream);
}

extern "C" int64_t prism_delta_prefill_workspace_bytes(int64_t T, int64_t seqs, int64_t HK, int64_t HV, int64_t DK,
                                                       int64_t DV) {
    return 0;
}
