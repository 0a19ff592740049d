// The gated delta rule in chunks of 64 tokens on the fifth-generation tensor cores (sm_100a).
//
// With G_t the sum of the log decays up to token t of a chunk and S_0 the state before it (lq_rule.cu has the rule token by token):
//     L_ts = beta_t e^{G_t - G_s} k^_t . k^_s (s < t)          T = (I + L)^-1
//     r_t  = beta_t (v_t - e^{G_t} S_0 k^_t)                    u = T r
//     o_t  = e^{G_t} S_0 q^_t + sum_{s <= t} e^{G_t - G_s} (q^_t . k^_s) u_s
//     S    = e^{G_C} S_0 + sum_t e^{G_C - G_t} u_t k^_t^T
//
// One CTA runs one (sequence, head) from its first chunk to its last.  All products with the state are taken transposed, so that the
// 128 rows of the tensor memory are the 128 value dimensions: a thread of the eight main warps owns half a row of the state (64
// columns, fp32 registers) or half the tokens of a row of r, u and o, and no row needs another one.
//     main warps   S -> f16 pieces in tensor memory (A operand); S k, S q; r -> pieces; u = T r; u -> pieces; o; S
//     prep warps   one chunk ahead: norms, f16 rows of k and q in shared memory (B operand), K K^T and Q K^T, decays, T and A
//
// Precision.  k and q are bf16 and become f16 without loss once a row is scaled by a power of two (what is lost lies 2^-25 below the
// row's norm); an fp32 operand is the sum of two f16 pieces, 22 bits.  f16 has few exponents, so every row of S, r and u carries
// a power of two of its own, from bounds that hold whatever the inputs: |k^| <= 1, 0 <= beta <= 1 and decays <= 1 make the rule a
// contraction, |r_t|, |u_t| / 2, |S| <= |S_0| + sum |v_t| =: B per row.  T is bounded by 1 for the same reason.  The products that
// only reach the bf16 outputs (S q, A u) take one piece, 2^-12.
#include "lq_tc.cuh"

namespace lq {

constexpr int RULE_SHORT = 8;                                // mean length from which lq_gdn_prefill works in chunks
constexpr int CT = 64;                                       // tokens of a chunk
// T and A lie within [-1, 1]; times 2^13 their small entries keep eleven bits down to 2^-27 as well
constexpr float MAT_UP = 8192.f, MAT_DOWN = 1.f / 8192.f;
constexpr int CK_MAIN = 256, CK_PREP = 128, CK_THREADS = CK_MAIN + CK_PREP;

// tensor memory: 512 columns.  D takes the place of X | XQ once both have been read, AU that of Y.
constexpr uint32_t TM_SHI = 0, TM_SLO = 64, TM_X = 128, TM_XQ = 192, TM_D = 128, TM_PHI = 256, TM_PLO = 288, TM_Y = 320, TM_AU = 320,
                   TM_UOP = 384, TM_G = 448;

// f16 operands, fp32 accumulator; B with the reduction contiguous (K-major) or, for S += u k^T, the 128 key columns (MN-major)
__host__ __device__ constexpr uint32_t ck_idesc(int n, bool b_mn) { return (1u << 4) | (b_mn ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | ((128u >> 4) << 24); }
// Descriptor of rows of 128 bytes in the 128-byte swizzle, eight rows (1 KB) after one another; `lbo`: bytes between blocks of 64
// elements of a MN-major operand (not used by a K-major one, which is advanced by hand).
__device__ __forceinline__ uint64_t ck_desc(uint32_t addr, uint32_t lbo) {
    return uint64_t((addr >> 4) & 0x3FFFu) | (uint64_t((lbo >> 4) & 0x3FFFu) << 16) | (uint64_t(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// byte offset of 16-byte chunk c (of 8) of a row in such a tile
__device__ __forceinline__ uint32_t ck_off(int row, int c) { return uint32_t(row) * 128u + (uint32_t(c ^ (row & 7)) << 4); }

struct ChunkScalars {                                        // of one chunk, by token
    float c1[CT];                                            // beta e^{G_t} kr_t: takes S k to what is subtracted from beta v
    float beta[CT];
    float c2[CT];                                            // e^{G_t} qr_t
    float c3[CT];                                            // e^{G_C - G_t} kr_t 2^-13 (u comes with the 2^13 of T)
    float decay;                                             // e^{G_C}
    int len;                                                 // tokens of the chunk, 1 .. 64
};
struct ChunkSmem {
    // start: 1 KB aligned.  tile: two blocks of 64 elements, each 64 rows of k and then 64 rows of q.
    unsigned char tile[2][32768];
    unsigned char thi[2][8192], tlo[2][8192], amat[2][8192];
    unsigned char raw[32768];                                // rows of k and q as they come: [128][128] bf16
    float L[CT][CT + 4];
    float tdiag[2][32][32], w[32][32];
    ChunkScalars sc[2];
    double G[CT];                                            // log2 of the decay from the chunk's start
    float kr[CT], qr[CT], ws[CT], gate_beta[CT];             // ws: kr_s times the decay from s to the end of its block of 16
    float2 part[2][CK_MAIN];
    uint64_t tile_full[2], ta_full[2], main_done[2], au_full[2], g_full, ks_full, qs_full, y_full, d_full, fin;
    uint32_t tm;
    int dead;
};

// Waits like warp_wait_bounded; once one wait of the CTA has run out, all later ones of every warp return at once, so that the CTA
// runs to its end (on rubbish) instead of waiting that long again and again.
__device__ __forceinline__ void ck_wait(ChunkSmem& s, uint64_t* bar, uint32_t parity) {
    for (uint32_t it = 0; it < WAIT_LIMIT; ++it) {
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return;
        if (it >= 64 && __any_sync(0xffffffffu, *reinterpret_cast<volatile int*>(&s.dead) != 0)) return;
    }
    s.dead = 1;
    atomicOr(&g_status, ST_CONSUMER_TIMEOUT);
}
__device__ __forceinline__ void cp_async16(void* dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }
// exponent e with b 2^e in [2^13, 2^14), within what fp32 scaling can carry
__device__ __forceinline__ int scale_exponent(float b) {
    const int e = 140 - int((__float_as_uint(b) >> 23) & 255u);
    return e < -100 ? -100 : e > 100 ? 100 : e;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// two fp32 values as an f16 head and an f16 remainder
__device__ __forceinline__ void split_h2(float2 x, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x.x, x.y);
    const float2 f = __half22float2(h);
    hi = h2_bits(h);
    lo = h2_bits(__floats2half2_rn(x.x - f.x, x.y - f.y));
}

// ---- prep warps -----------------------------------------------------------------------------------------------------------
// k and q rows of a chunk into the raw buffer (zeros behind the chunk's last token); every thread copies what it converts later
__device__ __forceinline__ void ck_fetch(ChunkSmem& s, const RuleParams& P, int hk, int64_t t0, int len, int pt) {
    const int lane = pt & 31, w = pt >> 5;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int r = 32 * w + 2 * i + (lane >> 4), t = r & 63, c = lane & 15;
        const bool in = t < len;
        const uint16_t* src = P.mixed + (in ? t0 + t : t0) * P.mixed_stride + ((r < 64 ? P.H : 0) + hk) * KD + 8 * c;
        cp_async16(s.raw + r * 256 + c * 16, src, in ? 16u : 0u);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}
__device__ __forceinline__ void ck_convert(ChunkSmem& s, int buf, int pt) {
    const int lane = pt & 31, w = pt >> 5;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
        const int r = 32 * w + 2 * i + (lane >> 4), c = lane & 15;
        const uint4 x = *reinterpret_cast<const uint4*>(s.raw + r * 256 + c * 16);
        const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
        float2 f[4], a2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[j] = bf16x2_to_f2(xw[j]);
            a2 = __ffma2_rn(f[j], f[j], a2);
        }
        float ss = a2.x + a2.y;
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        // the row times 2^-e has a norm in [1, 2); a sum of squares beyond fp32 makes the row zero, as 1 / sqrt(inf) does
        int e = (int((__float_as_uint(ss) >> 23) & 255u) - 127) >> 1;
        e = e < -60 ? -60 : e;
        const float m = ss <= 3.4e38f ? pow2f(-e) : 0.f;
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 y = __fmul2_rn(f[j], make_float2(m, m));
            h[j] = h2_bits(__floats2half2_rn(y.x, y.y));
        }
        *reinterpret_cast<uint4*>(s.tile[buf] + (c >> 3) * 16384 + ck_off(r, c & 7)) = make_uint4(h[0], h[1], h[2], h[3]);
        if (c == 0) (r < 64 ? s.kr : s.qr)[r & 63] = rsqrtf(ss + 1e-6f) * pow2f(e);
    }
}
// gates of the chunk, by one warp: lane l has the tokens 2 l and 2 l + 1
__device__ __forceinline__ void ck_gates(ChunkSmem& s, const RuleParams& P, int hv, int64_t t0, int len, float ea, float dtb, int lane) {
    double g[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int t = 2 * lane + i;
        float x = 0.f, beta = 0.f;
        if (t < len) {
            x = fmaxf(-ea * softplus_full(bf16_to_f(P.a[(t0 + t) * P.a_stride + hv]) + dtb) * 1.4426950408889634f, -1e30f);
            beta = sigmoidf_(bf16_to_f(P.b[(t0 + t) * P.b_stride + hv]));
        }
        g[i] = double(x);
        s.gate_beta[t] = beta;
    }
    double sum = g[0] + g[1];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const double o = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += o;
    }
    s.G[2 * lane] = sum - g[1];
    s.G[2 * lane + 1] = sum;
}
__device__ __forceinline__ float decay_between(double to, double from) { return exp2f(float(to - from)); }

// Gram rows -> L (fp32, k rows) and A (f16 operand, q rows).  The decay from s to t is taken in two steps over the end of s's block
// of 16 tokens, neither of which exceeds 1; inside the diagonal blocks it is taken in one.
__device__ __forceinline__ void ck_gram(ChunkSmem& s, int buf, uint32_t tm, int pt) {
    const int w = pt >> 5, t = pt & 63, tb = t >> 4;
    const bool isq = pt >= 64;
    const double Gt = s.G[t];
    const float rowf = isq ? s.qr[t] * MAT_UP : s.kr[t] * s.gate_beta[t];
    const uint32_t ta = tm + (uint32_t(32 * w) << 16) + TM_G;
#pragma unroll
    for (int hb = 0; hb < 2; ++hb) {
        uint32_t g[32];
        tmem_ld_32(ta + 32 * hb, g);
        float v[32];
#pragma unroll
        for (int b2 = 0; b2 < 2; ++b2) {
            const int b = 2 * hb + b2;
            if (b < tb) {
                const float f = rowf * decay_between(Gt, s.G[16 * b + 15]);
#pragma unroll
                for (int j = 0; j < 16; ++j) v[16 * b2 + j] = __uint_as_float(g[16 * b2 + j]) * (f * s.ws[16 * b + j]);
            } else if (b == tb) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int c = 16 * b + j;
                    const bool in = isq ? c <= t : c < t;
                    v[16 * b2 + j] = in ? __uint_as_float(g[16 * b2 + j]) * (rowf * s.kr[c] * decay_between(Gt, s.G[c])) : 0.f;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) v[16 * b2 + j] = 0.f;
            }
        }
        if (isq) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t h[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) h[j] = h2_bits(__floats2half2_rn(v[8 * c + 2 * j], v[8 * c + 2 * j + 1]));
                *reinterpret_cast<uint4*>(s.amat[buf] + ck_off(t, 4 * hb + c)) = make_uint4(h[0], h[1], h[2], h[3]);
            }
        } else {
#pragma unroll
            for (int c = 0; c < 8; ++c)
                *reinterpret_cast<float4*>(&s.L[t][32 * hb + 4 * c]) = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
        }
    }
}
__device__ __forceinline__ void ck_put_t(ChunkSmem& s, int buf, int t, int c, float x) {
    x *= MAT_UP;
    const __half h = __float2half_rn(x);
    const uint32_t off = ck_off(t, c >> 3) + 2 * (c & 7);
    *reinterpret_cast<__half*>(s.thi[buf] + off) = h;
    *reinterpret_cast<__half*>(s.tlo[buf] + off) = __float2half_rn(x - __half2float(h));
}
// T = (I + L)^-1 by 32 x 32 blocks: the two diagonal blocks by substitution (a lane has a column), then -T22 (L21 T11)
__device__ __forceinline__ void ck_invert(ChunkSmem& s, int buf, int pt) {
    const int w = pt >> 5, lane = pt & 31;
    if (w < 2) {
        const int o = 32 * w;
        float2 x[16];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            float2 acc = make_float2(0.f, 0.f);
            float last = 0.f;
#pragma unroll
            for (int m = 0; m + 4 <= ((i + 3) & ~3) && m < i; m += 4) {
                const float4 l = *reinterpret_cast<const float4*>(&s.L[o + i][o + m]);
                if (m + 2 <= i) acc = __ffma2_rn(make_float2(l.x, l.y), x[m / 2], acc);
                else last = fmaf(l.x, x[m / 2].x, last);
                if (m + 4 <= i) acc = __ffma2_rn(make_float2(l.z, l.w), x[m / 2 + 1], acc);
                else if (m + 3 <= i) last = fmaf(l.z, x[m / 2 + 1].x, last);
            }
            const float v = (lane == i ? 1.f : 0.f) - ((acc.x + acc.y) + last);
            if (i & 1) x[i / 2].y = v;
            else x[i / 2].x = v;
            s.tdiag[w][i][lane] = v;
            ck_put_t(s, buf, o + i, o + lane, v);
        }
    }
    named_bar(2, CK_PREP);
    {
        float2 x[16];
#pragma unroll
        for (int m = 0; m < 16; ++m) x[m] = make_float2(s.tdiag[0][2 * m][lane], s.tdiag[0][2 * m + 1][lane]);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            float2 acc = make_float2(0.f, 0.f);
#pragma unroll
            for (int m = 0; m < 8; ++m) {
                const float4 l = *reinterpret_cast<const float4*>(&s.L[32 + 8 * w + r][4 * m]);
                acc = __ffma2_rn(make_float2(l.x, l.y), x[2 * m], acc);
                acc = __ffma2_rn(make_float2(l.z, l.w), x[2 * m + 1], acc);
            }
            s.w[8 * w + r][lane] = acc.x + acc.y;
        }
    }
    named_bar(2, CK_PREP);
    {
        float2 x[16];
#pragma unroll
        for (int m = 0; m < 16; ++m) x[m] = make_float2(s.w[2 * m][lane], s.w[2 * m + 1][lane]);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            float2 acc = make_float2(0.f, 0.f);
#pragma unroll
            for (int m = 0; m < 8; ++m) {
                const float4 l = *reinterpret_cast<const float4*>(&s.tdiag[1][8 * w + r][4 * m]);
                acc = __ffma2_rn(make_float2(l.x, l.y), x[2 * m], acc);
                acc = __ffma2_rn(make_float2(l.z, l.w), x[2 * m + 1], acc);
            }
            ck_put_t(s, buf, 32 + 8 * w + r, lane, -(acc.x + acc.y));
        }
    }
}

__device__ __forceinline__ void ck_prep(ChunkSmem& s, const RuleParams& P, int hk, int hv, int64_t t0, int64_t len, int nchunk, uint32_t tm,
                                        int pt) {
    const int lane = pt & 31;
    const float ea = expf(P.A_log[hv]), dtb = P.dt_bias[hv];
    ck_fetch(s, P, hk, t0, int(len < CT ? len : CT), pt);
    for (int c = 0; c < nchunk; ++c) {
        const int buf = c & 1;
        const int64_t at = t0 + int64_t(c) * CT;
        const int64_t left = len - int64_t(c) * CT;
        const int n = int(left < CT ? left : CT);
        if (c >= 2) ck_wait(s, &s.main_done[buf], uint32_t((c >> 1) - 1) & 1u);
        ck_convert(s, buf, pt);
        if (pt >= 96) ck_gates(s, P, hv, at, n, ea, dtb, lane);
        fence_async_smem();
        tc_fence_before_sync();                              // (the Gram matrix of the chunk before has been read)
        named_bar(2, CK_PREP);
        if (pt == 0) {
            tc_fence_after_sync();
            const uint32_t ti = smem_u32(s.tile[buf]);
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                const uint64_t d = ck_desc(ti + (ks >> 2) * 16384 + (ks & 3) * 32, 16);
                umma_ss(tm + TM_G, d, d, ck_idesc(64, false), ks > 0);
            }
            umma_commit(&s.g_full);
        }
        if (c + 1 < nchunk) ck_fetch(s, P, hk, at + CT, int(left - CT < CT ? left - CT : CT), pt);
        if (pt < 64) {
            ChunkScalars& q = s.sc[buf];
            const double G = s.G[pt], Gc = s.G[CT - 1];
            const float e = exp2f(float(G)), kr = s.kr[pt], b = s.gate_beta[pt];
            q.c1[pt] = b * e * kr;
            q.beta[pt] = b;
            q.c2[pt] = e * s.qr[pt];
            q.c3[pt] = decay_between(Gc, G) * kr * MAT_DOWN;
            s.ws[pt] = decay_between(s.G[pt | 15], G) * kr;
            if (pt == 0) {
                q.decay = exp2f(float(Gc));
                q.len = n;
            }
        }
        named_bar(2, CK_PREP);
        if (pt == 0) mbar_arrive(&s.tile_full[buf]);
        __syncwarp();
        ck_wait(s, &s.g_full, uint32_t(c) & 1u);
        tc_fence_after_sync();
        ck_gram(s, buf, tm, pt);
        named_bar(2, CK_PREP);
        ck_invert(s, buf, pt);
        fence_async_smem();
        named_bar(2, CK_PREP);
        if (pt == 0) mbar_arrive(&s.ta_full[buf]);
        __syncwarp();
    }
    if (pt == 0) umma_commit(&s.fin);
}

// ---- main warps -----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void ck_main(ChunkSmem& s, const RuleParams& P, int hv, int64_t t0, int nchunk, float* Sg, bool keep, uint32_t tm, int tid) {
    const int lane = tid & 31, warp = tid >> 5, h = warp >> 2, v = 32 * (warp & 3) + lane;
    const uint32_t row = tm + (uint32_t(32 * (warp & 3)) << 16);
    float2 S[32];                                            // S[v][64 h ..]
    float* Srow = Sg + v * KD + 64 * h;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float4 x = keep ? *reinterpret_cast<const float4*>(Srow + 4 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
        S[2 * i] = make_float2(x.x, x.y);
        S[2 * i + 1] = make_float2(x.z, x.w);
    }
    const uint16_t* vrow = P.mixed + t0 * P.mixed_stride + 2 * P.H * KD + hv * VD + v;
    float back = 0.f, decay = 0.f;                           // 2^-eB and the decay of the chunk whose D is still to come
    for (int c = 0; c <= nchunk; ++c) {
        const int buf = c & 1;
        const uint32_t ph = uint32_t(c >> 1) & 1u;
        const ChunkScalars& q = s.sc[buf];
        int len = 0;
        uint32_t vv[16];
        float va = 0.f;
        if (c < nchunk) {
            ck_wait(s, &s.tile_full[buf], ph);
            len = q.len;
            const uint16_t* vp = vrow + (int64_t(c) * CT + 32 * h) * P.mixed_stride;
            uint32_t r[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = 32 * h + i < len ? uint32_t(__ldg(vp + i * P.mixed_stride)) : 0u;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                vv[i] = r[2 * i] | (r[2 * i + 1] << 16);
                va += fabsf(bf16lo(vv[i])) + fabsf(bf16hi(vv[i]));
            }
        }
        if (c > 0) {                                         // the state behind the chunk before
            ck_wait(s, &s.d_full, uint32_t(c - 1) & 1u);
            tc_fence_after_sync();
            const float2 d2 = make_float2(decay, decay), b2 = make_float2(back, back);
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                uint32_t r[32];
                tmem_ld_32(row + TM_D + 64 * h + 32 * p, r);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 d = make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
                    S[16 * p + i] = __ffma2_rn(d, b2, __fmul2_rn(S[16 * p + i], d2));
                }
            }
            if (c == nchunk) break;
            // every product of that chunk is through and its scalars have been read: its buffers are free
            if (c + 1 < nchunk && lane == 0) mbar_arrive(&s.main_done[buf ^ 1]);
            __syncwarp();
        }
        // the row's powers of two, from the whole row
        float2 n2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 32; ++i) n2 = __ffma2_rn(S[i], S[i], n2);
        s.part[buf][tid] = make_float2(n2.x + n2.y, va);
        tc_fence_before_sync();
        named_bar(1, CK_MAIN);
        const float2 mine = s.part[buf][tid], other = s.part[buf][tid ^ 128];
        const float norm = sqrtf(mine.x + other.x);
        const int eS = scale_exponent(norm), eB = scale_exponent(norm + (mine.y + other.y));
        {
            const float2 f = make_float2(pow2f(eS), pow2f(eS));
            uint32_t hi[32], lo[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) split_h2(__fmul2_rn(S[i], f), hi[i], lo[i]);
            tc_fence_after_sync();
            tmem_st_32(row + TM_SHI + 32 * h, hi);
            tmem_st_32(row + TM_SLO + 32 * h, lo);
            tmem_st_wait();
        }
        tc_fence_before_sync();
        named_bar(1, CK_MAIN);
        const uint32_t ti = smem_u32(s.tile[buf]);
        if (tid == 0) {                                      // S k^T, then S q^T
            tc_fence_after_sync();
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                const uint64_t d = ck_desc(ti + (ks >> 2) * 16384 + (ks & 3) * 32, 16);
                umma_f16_ts(tm + TM_X, tm + TM_SHI + 8 * ks, d, ck_idesc(64, false), ks > 0);
                umma_f16_ts(tm + TM_X, tm + TM_SLO + 8 * ks, d, ck_idesc(64, false), 1u);
            }
            umma_commit(&s.ks_full);
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
                umma_f16_ts(tm + TM_XQ, tm + TM_SHI + 8 * ks, ck_desc(ti + (ks >> 2) * 16384 + 8192 + (ks & 3) * 32, 16), ck_idesc(64, false), ks > 0);
            umma_commit(&s.qs_full);
        }
        __syncwarp();
        const float fB = pow2f(eB), fX = pow2f(eB - eS < -126 ? -126 : eB - eS);
        ck_wait(s, &s.ks_full, uint32_t(c) & 1u);
        tc_fence_after_sync();
        {                                                    // r = beta (v - e^G S k^), times 2^eB
            uint32_t x[32], hi[16], lo[16];
            tmem_ld_32(row + TM_X + 32 * h, x);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 c1 = *reinterpret_cast<const float2*>(&q.c1[32 * h + 2 * i]), be = *reinterpret_cast<const float2*>(&q.beta[32 * h + 2 * i]);
                const float2 xs = __fmul2_rn(make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), make_float2(-fX, -fX));
                const float2 bv = __fmul2_rn(__fmul2_rn(bf16x2_to_f2(vv[i]), make_float2(fB, fB)), be);
                split_h2(__ffma2_rn(c1, xs, bv), hi[i], lo[i]);
            }
            tmem_st_16(row + TM_PHI + 16 * h, hi);
            tmem_st_16(row + TM_PLO + 16 * h, lo);
            tmem_st_wait();
        }
        tc_fence_before_sync();
        named_bar(1, CK_MAIN);
        if (warp == 0) ck_wait(s, &s.ta_full[buf], ph);
        if (tid == 0) {                                      // u = T r
            tc_fence_after_sync();
            const uint32_t th = smem_u32(s.thi[buf]), tl = smem_u32(s.tlo[buf]);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                umma_f16_ts(tm + TM_Y, tm + TM_PHI + 8 * ks, ck_desc(th + ks * 32, 16), ck_idesc(64, false), ks > 0);
                umma_f16_ts(tm + TM_Y, tm + TM_PHI + 8 * ks, ck_desc(tl + ks * 32, 16), ck_idesc(64, false), 1u);
                umma_f16_ts(tm + TM_Y, tm + TM_PLO + 8 * ks, ck_desc(th + ks * 32, 16), ck_idesc(64, false), 1u);
            }
            umma_commit(&s.y_full);
        }
        __syncwarp();
        float2 o[16];                                        // e^G S q^, in outputs' units
        ck_wait(s, &s.qs_full, uint32_t(c) & 1u);
        tc_fence_after_sync();
        {
            uint32_t x[32];
            tmem_ld_32(row + TM_XQ + 32 * h, x);
            const float f = P.scale * pow2f(-eS);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                o[i] = __fmul2_rn(__fmul2_rn(make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), make_float2(f, f)),
                                  *reinterpret_cast<const float2*>(&q.c2[32 * h + 2 * i]));
        }
        ck_wait(s, &s.y_full, uint32_t(c) & 1u);
        tc_fence_after_sync();
        {                                                    // u for A u (one piece), u e^{G_C - G} kr for the state (two)
            uint32_t y[32], un[16], hi[16], lo[16];
            tmem_ld_32(row + TM_Y + 32 * h, y);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 u = make_float2(__uint_as_float(y[2 * i]), __uint_as_float(y[2 * i + 1]));
                un[i] = h2_bits(__floats2half2_rn(u.x * MAT_DOWN, u.y * MAT_DOWN));
                split_h2(__fmul2_rn(u, *reinterpret_cast<const float2*>(&q.c3[32 * h + 2 * i])), hi[i], lo[i]);
            }
            tmem_st_16(row + TM_UOP + 16 * h, un);
            tmem_st_16(row + TM_PHI + 16 * h, hi);
            tmem_st_16(row + TM_PLO + 16 * h, lo);
            tmem_st_wait();
        }
        tc_fence_before_sync();
        named_bar(1, CK_MAIN);
        if (tid == 0) {                                      // A u, then the chunk's part of the state
            tc_fence_after_sync();
            const uint32_t am = smem_u32(s.amat[buf]);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
                umma_f16_ts(tm + TM_AU, tm + TM_UOP + 8 * ks, ck_desc(am + ks * 32, 16), ck_idesc(64, false), ks > 0);
            umma_commit(&s.au_full[buf]);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                const uint64_t d = ck_desc(ti + ks * 2048, 16384);
                umma_f16_ts(tm + TM_D, tm + TM_PHI + 8 * ks, d, ck_idesc(128, true), ks > 0);
                umma_f16_ts(tm + TM_D, tm + TM_PLO + 8 * ks, d, ck_idesc(128, true), 1u);
            }
            umma_commit(&s.d_full);
        }
        __syncwarp();
        decay = q.decay;
        back = pow2f(-eB);
        ck_wait(s, &s.au_full[buf], ph);
        tc_fence_after_sync();
        {
            uint32_t x[32];
            tmem_ld_32(row + TM_AU + 32 * h, x);
            const float f = P.scale * back * MAT_DOWN;
            uint16_t* op = P.o + ((t0 + int64_t(c) * CT + 32 * h) * P.HV + hv) * VD + v;
            const int64_t step = int64_t(P.HV) * VD;
            const int m = len - 32 * h;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float y = fmaf(__uint_as_float(x[i]), f, (i & 1) ? o[i >> 1].y : o[i >> 1].x);
                if (i < m) op[i * step] = f_to_bf16(y);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
        *reinterpret_cast<float4*>(Srow + 4 * i) = make_float4(S[2 * i].x, S[2 * i].y, S[2 * i + 1].x, S[2 * i + 1].y);
    if (tid == 0) umma_commit(&s.fin);
}

__global__ void __launch_bounds__(CK_THREADS, 1) rule_chunk_kernel(RuleParams P) {
    extern __shared__ unsigned char dyn[];
    ChunkSmem& s = *reinterpret_cast<ChunkSmem*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_trigger();
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s.tile_full[i], 1);
            mbar_init(&s.ta_full[i], 1);
            mbar_init(&s.main_done[i], CK_MAIN / 32);
            mbar_init(&s.au_full[i], 1);
        }
        mbar_init(&s.g_full, 1);
        mbar_init(&s.ks_full, 1);
        mbar_init(&s.qs_full, 1);
        mbar_init(&s.y_full, 1);
        mbar_init(&s.d_full, 1);
        mbar_init(&s.fin, 2);
        s.dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    const int n = blockIdx.x / P.HV, hv = blockIdx.x % P.HV, hk = hv / (P.HV / P.H);
    int64_t t0, len;
    rule_span(P, n, t0, len);
    if (len == 0) return;
    const int slot = P.idx[n];
    if (slot <= 0 || slot >= P.NS || !first_of_slot(P.idx, n, slot, lane)) {       // padding: zeros, and no state
        for (int64_t i = tid; i < len * (VD / 8); i += CK_THREADS)
            *reinterpret_cast<uint4*>(P.o + ((t0 + i / (VD / 8)) * P.HV + hv) * VD + 8 * (i % (VD / 8))) = make_uint4(0u, 0u, 0u, 0u);
        return;
    }
    for (int i = tid; i < 2 * 8192 / 16; i += CK_THREADS) {                        // the upper right block of T stays zero
        reinterpret_cast<uint4*>(s.thi)[i] = make_uint4(0u, 0u, 0u, 0u);
        reinterpret_cast<uint4*>(s.tlo)[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    if (warp == 0) tmem_alloc(&s.tm, 512);
    fence_async_smem();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tm = s.tm;
    const int nchunk = int((len + CT - 1) / CT);
    if (tid >= CK_MAIN) ck_prep(s, P, hk, hv, t0, len, nchunk, tm, tid - CK_MAIN);
    else ck_main(s, P, hv, t0, nchunk, P.ssm + int64_t(slot) * P.SS + int64_t(hv) * VD * KD, !P.has_initial || P.has_initial[n], tm, tid);
    ck_wait(s, &s.fin, 0);                                   // no tensor-core instruction is left
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tm, 512);
}

static int rule_check(const lq_dims* d, const RuleParams& P) {
    if (d->K != KD || d->V != VD) return LQ_ERR_UNSUPPORTED;
    if (d->NS < 1 || d->HV < 1 || d->H < 1 || d->HV % d->H != 0 || d->SS < int64_t(d->HV) * d->V * d->K) return LQ_ERR_RANGE;
    if (d->SS & 3) return LQ_ERR_ALIGN;
    if (P.N < 0 || P.T < 0) return LQ_ERR_RANGE;
    if (P.N == 0 || P.T == 0) return LQ_OK;
    if (!P.ssm || !P.mixed || !P.a || !P.b || !P.A_log || !P.dt_bias || !P.idx || !P.o) return LQ_ERR_NULL;
    if (P.mixed_stride < 2 * int64_t(d->H) * KD + int64_t(d->HV) * VD || P.a_stride < d->HV || P.b_stride < d->HV) return LQ_ERR_RANGE;
    if ((P.mixed_stride & 7) || misaligned16({P.ssm, P.mixed, P.o})) return LQ_ERR_ALIGN;
    if (int64_t(P.N) * d->HV > (int64_t(1) << 29)) return LQ_ERR_RANGE;            // programs: the grid's first dimension
    return LQ_OK;
}
static int launch_recurrent(const RuleParams& P, cudaStream_t st) {
    const unsigned grid = unsigned(P.N) * unsigned(P.HV) * (VD / (RW_ROWS * RW_WARPS));
    const cudaError_t e = launch_dependent(rule_recurrent_kernel, grid, 32 * RW_WARPS, 0, st, P);
    if (e != cudaSuccess) { set_last_cuda_error(e); return LQ_ERR_LAUNCH; }
    return finish_launch();
}
static int launch_chunk(const RuleParams& P, cudaStream_t st) {
    constexpr size_t smem = sizeof(ChunkSmem) + 1024;
    static_assert(smem <= 227 * 1024, "the working set of a CTA");
    int rc = ensure_smem((const void*)rule_chunk_kernel, smem);
    if (rc) return rc;
    const cudaError_t e = launch_dependent(rule_chunk_kernel, unsigned(P.N) * unsigned(P.HV), CK_THREADS, smem, st, P);
    if (e != cudaSuccess) { set_last_cuda_error(e); return LQ_ERR_LAUNCH; }
    return finish_launch();
}

static RuleParams rule_params(const lq_dims* d, float* ssm, const void* mixed, int64_t mixed_stride, const void* a, int64_t a_stride,
                              const void* b, int64_t b_stride, const float* A_log, const float* dt_bias, const int32_t* cu,
                              const int32_t* idx, const uint8_t* has_initial, void* o, int32_t N, int64_t T, float scale) {
    RuleParams P;
    P.ssm = ssm; P.SS = d->SS; P.mixed = (const uint16_t*)mixed; P.mixed_stride = mixed_stride; P.a = (const uint16_t*)a;
    P.b = (const uint16_t*)b; P.a_stride = a_stride; P.b_stride = b_stride; P.A_log = A_log; P.dt_bias = dt_bias; P.cu = cu;
    P.idx = idx; P.has_initial = has_initial; P.o = (uint16_t*)o; P.NS = d->NS; P.H = d->H; P.HV = d->HV; P.N = N; P.T = T;
    P.scale = scale > 0.f ? scale : 1.0f / sqrtf(float(KD));
    return P;
}

}  // namespace lq

extern "C" int lq_gdn_prefill(const lq_dims* d, float* ssm, const void* mixed, int64_t mixed_stride, const void* a, int64_t a_stride,
                              const void* b, int64_t b_stride, const float* A_log, const float* dt_bias, const int32_t* cu,
                              const int32_t* idx, const uint8_t* has_initial, void* o, int32_t N, int64_t T, float scale,
                              void* stream) {
    using namespace lq;
    if (!d) return LQ_ERR_NULL;
    const RuleParams P = rule_params(d, ssm, mixed, mixed_stride, a, a_stride, b, b_stride, A_log, dt_bias, cu, idx, has_initial, o, N,
                                     T, scale);
    const int rc = rule_check(d, P);
    if (rc || N == 0 || T == 0) return rc;
    if (!cu) return LQ_ERR_NULL;
    const int impl = g_rule_impl.load(std::memory_order_relaxed);
    const bool tokens = impl == 1 || (impl == 0 && T < int64_t(RULE_SHORT) * N);
    return tokens ? launch_recurrent(P, static_cast<cudaStream_t>(stream)) : launch_chunk(P, static_cast<cudaStream_t>(stream));
}

extern "C" int lq_gdn_recurrent(const lq_dims* d, float* ssm, const void* mixed, int64_t mixed_stride, const void* a, int64_t a_stride,
                                const void* b, int64_t b_stride, const float* A_log, const float* dt_bias, const int32_t* idx, void* o,
                                int32_t N, float scale, void* stream) {
    using namespace lq;
    if (!d) return LQ_ERR_NULL;
    const RuleParams P = rule_params(d, ssm, mixed, mixed_stride, a, a_stride, b, b_stride, A_log, dt_bias, nullptr, idx, nullptr, o, N,
                                     N, scale);
    const int rc = rule_check(d, P);
    if (rc || N == 0) return rc;
    return launch_recurrent(P, static_cast<cudaStream_t>(stream));
}
