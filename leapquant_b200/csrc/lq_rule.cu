// The gated delta rule on the fp32 states of the slots (sm_100a): what runs between lq_dequant and lq_quantize, and the decode of
// states that are kept in fp32.
//
// Per value head, with the state S [V][K] of the sequence's slot:
//     g_t = -exp(A_log) softplus(a_t + dt_bias),  beta_t = sigmoid(b_t)
//     q^_t = q_t scale / sqrt(|q_t|^2 + 1e-6),  k^_t = k_t / sqrt(|k_t|^2 + 1e-6)
//     S <- e^{g_t} S;   u_t = beta_t (v_t - S k^_t);   S <- S + u_t k^_t^T;   o_t = S q^_t
// States, gates, norms and sums are fp32 (sums of gates fp64); outputs are rounded to bf16 once.
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
};

// log(1 + e^x) to fp32 precision for every x: 1 + e^x alone would cut e^x off at 2^-24, and a layer that starts with steps of a
// thousandth would decay wrongly by 6e-5 of its rate
__device__ __forceinline__ float softplus_full(float x) { return x <= SOFTPLUS_THRESHOLD ? log1pf(expf(x)) : x; }
__device__ __forceinline__ float rule_log_decay(const RuleParams& P, int64_t t, int hv, float ea, float dtb) {
    return -ea * softplus_full(bf16_to_f(P.a[t * P.a_stride + hv]) + dtb);
}

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
// no warp waits for another.  Both products take the state before the update, S q = e^g (S_old q) + u (k^ . q^).
constexpr int RW_ROWS = 16, RW_WARPS = 4;
struct RuleToken {
    uint2 q[4], k[4];
    uint16_t v[4], a, b;
};
__device__ __forceinline__ RuleToken rule_load(const RuleParams& P, int64_t t, int hk, int hv, int v0, int lane) {
    RuleToken r;
    const uint16_t* row = P.mixed + t * P.mixed_stride;
    const int c = 4 * (lane & 7);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        r.q[j] = __ldg(reinterpret_cast<const uint2*>(row + hk * KD + c + 32 * j));
        r.k[j] = __ldg(reinterpret_cast<const uint2*>(row + (P.H + hk) * KD + c + 32 * j));
        r.v[j] = __ldg(row + 2 * P.H * KD + hv * VD + v0 + 4 * j + (lane >> 3));
    }
    r.a = __ldg(P.a + t * P.a_stride + hv);
    r.b = __ldg(P.b + t * P.b_stride + hv);
    return r;
}
__global__ void __launch_bounds__(32 * RW_WARPS) rule_recurrent_kernel(RuleParams P) {
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
    uint16_t* out = P.o + (t0 * P.HV + hv) * VD + v0 + r8;
    const int64_t ostep = int64_t(P.HV) * VD;
    if (!ours || !first_of_slot(P.idx, n, slot, lane)) {    // padding: zeros, and no state
        for (int64_t t = 0; t < len; ++t, out += ostep)
            if ((lane & 7) < 4) out[4 * (lane & 7)] = 0;
        return;
    }
    const float ea = expf(P.A_log[hv]), dtb = P.dt_bias[hv];
    RuleToken x = rule_load(P, t0, hk, hv, v0, lane);
    for (int64_t t = 0; t < len; ++t, out += ostep) {
        float q[16], k[16], qq = 0.f, kk = 0.f, qk = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t wq[2] = {x.q[j].x, x.q[j].y}, wk[2] = {x.k[j].x, x.k[j].y};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                q[4 * j + 2 * h] = bf16lo(wq[h]); q[4 * j + 2 * h + 1] = bf16hi(wq[h]);
                k[4 * j + 2 * h] = bf16lo(wk[h]); k[4 * j + 2 * h + 1] = bf16hi(wk[h]);
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            qq = fmaf(q[i], q[i], qq);
            kk = fmaf(k[i], k[i], kk);
            qk = fmaf(q[i], k[i], qk);
        }
        qq = oct_sum(qq);
        kk = oct_sum(kk);
        qk = oct_sum(qk);
        const float inq = rsqrtf(qq + 1e-6f) * P.scale, ink = rsqrtf(kk + 1e-6f);
        const float alpha = expf(-ea * softplus_full(bf16_to_f(x.a) + dtb)), beta = sigmoidf_(bf16_to_f(x.b));
        float vv[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) vv[p] = bf16_to_f(x.v[p]);
        if (t + 1 < len) x = rule_load(P, t0 + t + 1, hk, hv, v0, lane);
        qk *= inq * ink;
        float mine = 0.f;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            float sk = 0.f, sq = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float* e = &s[p][j].x;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sk = fmaf(e[i], k[4 * j + i], sk);
                    sq = fmaf(e[i], q[4 * j + i], sq);
                }
            }
            sk = oct_sum(sk) * ink;
            sq = oct_sum(sq) * inq;
            const float u = beta * (vv[p] - alpha * sk), uk = u * ink;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float* e = &s[p][j].x;
#pragma unroll
                for (int i = 0; i < 4; ++i) e[i] = fmaf(uk, k[4 * j + i], alpha * e[i]);
            }
            const float o = fmaf(alpha, sq, u * qk);
            if ((lane & 7) == p) mine = o;
        }
        if ((lane & 7) < 4) out[4 * (lane & 7)] = f_to_bf16(mine);
    }
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int j = 0; j < 4; ++j) __stcs(reinterpret_cast<float4*>(base + 4 * p * KD + 32 * j), s[p][j]);
}

}  // namespace lq
