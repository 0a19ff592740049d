// The gated delta rule on the fp32 states of the slots (sm_100a): what runs between lq_dequant and lq_quantize, and the decode of
// states that are kept in fp32.
//
// Per value head, with the state S [V][K] of the sequence's slot:
//     g_t = -exp(A_log) softplus(a_t + dt_bias),  beta_t = sigmoid(b_t)
//     q^_t = q_t scale / sqrt(|q_t|^2 + 1e-6),  k^_t = k_t / sqrt(|k_t|^2 + 1e-6)
//     S <- e^{g_t} S;   u_t = beta_t (v_t - S k^_t);   S <- S + u_t k^_t^T;   o_t = S q^_t
// States, gates, norms and sums are fp32 (in chunks: sums of gates fp64, factors of fp32 products two f16 pieces, 22 bits); outputs are rounded
// to bf16 once.
#include "lq_common.cuh"

namespace lq {

struct RuleParams {
    float* ssm;
    int64_t SS;
    const uint16_t* mixed;            // bf16 rows q | k | v
    int64_t mixed_stride;
    const uint16_t *a, *b;            // bf16 [T, HV]
    int64_t a_stride, b_stride;
    const float *A_log, *dt_bias;
    const int32_t* cu;                // first token of every sequence and the end of the last; NULL: sequence n is row n
    const int32_t* idx;
    const uint8_t* has_initial;       // NULL: every sequence continues its slot's state
    uint16_t* o;                      // bf16 [T, HV, V]
    int32_t NS, H, HV, N;
    int64_t T;
    float scale;
    int64_t shorter;                  // rule_recurrent_kernel takes the sequences with fewer tokens, rule_chunk_kernel the others
    float* work;                      // matrices of the segments, where sequences are split
    int32_t segs, pass;               // segments a sequence is split into (0: not), and which of the two passes over them this is
};

// log(1 + e^x) to fp32 precision for every x: 1 + e^x alone would cut e^x off at 2^-24, and a layer that starts with steps of a
// thousandth would decay wrongly by 6e-5 of its rate
__device__ __forceinline__ float softplus_full(float x) { return x <= SOFTPLUS_THRESHOLD ? log1pf(expf(x)) : x; }
// First token and length of sequence n, whatever the caller's offsets hold: never outside the T rows.
__device__ __forceinline__ void rule_span(const RuleParams& P, int n, int64_t& t0, int64_t& len) {
    if (!P.cu) { t0 = n; len = 1; return; }
    int64_t s = P.cu[n], e = P.cu[n + 1];
    s = s < 0 ? 0 : s > P.T ? P.T : s;
    e = e < s ? s : e > P.T ? P.T : e;
    t0 = s;
    len = e - s;
}

// ---- token by token -----------------------------------------------------------------------------------------------------
// A warp owns sixteen rows of one head's state, in registers from the first token to the last: eight lanes share a row (lane c of
// them the columns 4 c + 32 j .. + 3), four rows are worked on side by side.  q^ and k^ are computed by every warp for itself, so
// no warp waits for another.  Both products take the state before the update, S q = e^g (S_old q) + u (k^ . q^).  The gates of 32 tokens
// are computed at once, one token a lane.
// One token per sequence is a copy of the states: 256 rows of 32 heads 163 us, the measured copy rate.  From four tokens on the FMA pipe
// (60 % busy, 59 % of the cycles issue) and the latency of a token share the time; four warps a scheduler at 128 registers: 4 tokens of 128
// sequences of 32 heads 124 us, with three 137, with plain multiply-adds, a sum per row and three 158.  Carrying the decays in a scalar beside
// the state, which saves a fifth of the FMA instructions, was no faster.
constexpr int RW_ROWS = 16, RW_WARPS = 4, RW_CTAS = 4;
struct RuleToken {
    uint2 q[4], k[4];
    uint16_t v;                                             // of row 4 (lane & 3) + lane / 8
};
__device__ __forceinline__ RuleToken rule_load(const uint16_t* row, int qat, int kat, int vat) {
    RuleToken r;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        r.q[j] = __ldg(reinterpret_cast<const uint2*>(row + qat + 32 * j));
        r.k[j] = __ldg(reinterpret_cast<const uint2*>(row + kat + 32 * j));
    }
    r.v = __ldg(row + vat);
    return r;
}
__device__ __forceinline__ float2 rule_two(uint32_t w) { return make_float2(bf16lo(w), bf16hi(w)); }
__device__ __forceinline__ float2 rule_both(float x) { return make_float2(x, x); }
// Sums of eight values over the eight lanes that share a row; every exchange halves what a lane keeps, and lane l is left with value l.
__device__ __forceinline__ float oct_fold(const float (&v)[8], int lane) {
    float a[4], b[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = (lane & 4 ? v[4 + i] : v[i]) + __shfl_xor_sync(0xffffffffu, lane & 4 ? v[i] : v[4 + i], 4);
#pragma unroll
    for (int i = 0; i < 2; ++i) b[i] = (lane & 2 ? a[2 + i] : a[i]) + __shfl_xor_sync(0xffffffffu, lane & 2 ? a[i] : a[2 + i], 2);
    return (lane & 1 ? b[1] : b[0]) + __shfl_xor_sync(0xffffffffu, lane & 1 ? b[0] : b[1], 1);
}
__global__ void __launch_bounds__(32 * RW_WARPS, RW_CTAS) rule_recurrent_kernel(RuleParams P) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int PARTS = VD / (RW_ROWS * RW_WARPS);
    const int prog = blockIdx.x / PARTS, part = blockIdx.x % PARTS;
    const int n = prog / P.HV, hv = prog % P.HV, hk = hv / (P.HV / P.H);
    const int v0 = (part * RW_WARPS + warp) * RW_ROWS;
    int64_t t0, len;
    rule_span(P, n, t0, len);
    if (len == 0 || len >= P.shorter) return;
    const int slot = P.idx[n];
    const bool ours = slot > 0 && slot < P.NS;
    const int c = 4 * (lane & 7), r8 = lane >> 3;
    float4 s[4][4];                                         // [row v0 + 4 p + r8][columns c + 32 j ..]
    float* base = P.ssm + int64_t(ours ? slot : 0) * P.SS + int64_t(hv) * VD * KD + int64_t(v0 + r8) * KD + c;
    const bool keep = ours && (!P.has_initial || P.has_initial[n]);
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            s[p][j] = keep ? __ldcs(reinterpret_cast<const float4*>(base + 4 * p * KD + 32 * j)) : make_float4(0.f, 0.f, 0.f, 0.f);
    uint16_t* out = P.o + (t0 * P.HV + hv) * VD + v0 + r8 + 4 * (lane & 3);
    const int64_t ostep = int64_t(P.HV) * VD;
    if (!ours || !first_of_slot(P.idx, n, slot, lane)) {    // padding: zeros, and no state
        for (int t = 0; t < int(len); ++t, out += ostep)
            if (lane & 4) out[0] = 0;
        return;
    }
    const float ea = expf(P.A_log[hv]), dtb = P.dt_bias[hv];
    float alphas = 0.f, betas = 0.f;                        // of 32 tokens, one a lane
    const uint16_t* row = P.mixed + t0 * P.mixed_stride;
    const int qat = hk * KD + c, kat = (P.H + hk) * KD + c, vat = 2 * P.H * KD + hv * VD + v0 + 4 * (lane & 3) + r8, ntok = int(len);
    RuleToken x = rule_load(row, qat, kat, vat);
#pragma unroll 1
    for (int t = 0; t < ntok; ++t, out += ostep) {
        if ((t & 31) == 0) {
            const int64_t tl = t0 + (t + lane < ntok ? t + lane : t);
            alphas = expf(-ea * softplus_full(bf16_to_f(__ldg(P.a + tl * P.a_stride + hv)) + dtb));
            betas = sigmoidf_(bf16_to_f(__ldg(P.b + tl * P.b_stride + hv)));
        }
        const float alpha = __shfl_sync(0xffffffffu, alphas, t & 31), beta = __shfl_sync(0xffffffffu, betas, t & 31);
        float2 q[8], k[8], qq2, kk2, qk2;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            q[2 * j] = rule_two(x.q[j].x); q[2 * j + 1] = rule_two(x.q[j].y);
            k[2 * j] = rule_two(x.k[j].x); k[2 * j + 1] = rule_two(x.k[j].y);
        }
        const float vv = bf16_to_f(x.v);
        row += P.mixed_stride;
        if (t + 1 < ntok) x = rule_load(row, qat, kat, vat);
        qq2 = __fmul2_rn(q[0], q[0]);
        kk2 = __fmul2_rn(k[0], k[0]);
        qk2 = __fmul2_rn(q[0], k[0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) {
            qq2 = __ffma2_rn(q[i], q[i], qq2);
            kk2 = __ffma2_rn(k[i], k[i], kk2);
            qk2 = __ffma2_rn(q[i], k[i], qk2);
        }
        const float qq = oct_sum(qq2.x + qq2.y), kk = oct_sum(kk2.x + kk2.y);
        float qk = oct_sum(qk2.x + qk2.y);
        const float inq = rsqrtf(qq + 1e-6f) * P.scale, ink = rsqrtf(kk + 1e-6f);
        qk *= inq * ink;
        float part8[8];                                     // S k and S q of the four rows
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const float2* e = reinterpret_cast<const float2*>(&s[p][0]);
            float2 sk = __fmul2_rn(e[0], k[0]), sq = __fmul2_rn(e[0], q[0]);
#pragma unroll
            for (int i = 1; i < 8; ++i) {
                sk = __ffma2_rn(e[i], k[i], sk);
                sq = __ffma2_rn(e[i], q[i], sq);
            }
            part8[p] = sk.x + sk.y;
            part8[4 + p] = sq.x + sq.y;
        }
        const float sum = oct_fold(part8, lane);            // lanes 0 .. 3 of a row: S k of rows 0 .. 3; 4 .. 7: S q
        const float u = beta * (vv - alpha * (sum * ink)), uk = u * ink;
        const float uo = __shfl_xor_sync(0xffffffffu, u, 4);
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const float2 up = rule_both(__shfl_sync(0xffffffffu, uk, (lane & 24) | p));
            float2* e = reinterpret_cast<float2*>(&s[p][0]);
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = __ffma2_rn(up, k[i], __fmul2_rn(rule_both(alpha), e[i]));
        }
        if (lane & 4) out[0] = f_to_bf16(fmaf(alpha, sum * inq, uo * qk));
    }
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int j = 0; j < 4; ++j) __stcs(reinterpret_cast<float4*>(base + 4 * p * KD + 32 * j), s[p][j]);
}

}  // namespace lq
