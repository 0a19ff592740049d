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
//     issue warp   their tensor-core instructions, the copies of v, the stores of the outputs
//     prep warps   two groups of four, a chunk each in turn, ahead of the main warps: norms, f16 rows of k and q in shared memory
//                  (B operand), K K^T and Q K^T, decays, T and A; rows of k and q by TMA
//
// What bounds it.  One sequence is a chain of chunks, and a chunk of one head is what one SM does at a time: 4.7 us, most of it the main
// chain, six hand-overs between registers, tensor memory and tensor cores; the two prep groups take about as long for a chunk, side by
// side with it.  Both are made of the same issue slots: 21 200 warp instructions a chunk, 0.51 an SM quarter's cycle.  FMA pipe 31 %, ALU 24 %,
// tensor pipe 27 % busy: a warp waits for tensor memory, barriers and its own results.  The loops are kept small, since an SM's
// instruction cache holds 32 KB (they are larger; when they were twice as long, fetching was the first stall), and what is seldom needed
// stands behind them.
//     one sequence of 8 192 tokens, 32 heads      600 us on 32 SMs, 447 split over 96
//     16 sequences of 4 096 tokens, 32 heads    1 269 us on all, 512 heads on 148 SMs
// On the way, one sequence of 8 192 tokens, not split: token by token 6 750 us; in chunks with one prep group 1 920; two groups, values and outputs
// through shared memory, instructions issued by a whole warp 810; the inverse on tensor cores, one scale per row 620; rows and outputs by
// TMA 570.  16 sequences of 4 096: loops instead of straight code and outputs accumulated in tensor memory 1 330 -> 1 170 us; roles and starts
// of the segments in the same kernel 1 207; outputs from two pieces 1 244 (1 263 with A u ahead of the state's products); the whole range of
// states and values, infinities and NaN 1 269.  Without gain: sixteen main warps with a quarter of a row each, two accumulators for S k,
// loops rolled up to 38 KB (spills: 684 us), hints to sleeping waits.
//
// Precision.  k and q are bf16 and become f16 without loss once a row is scaled by a power of two (what is lost lies 2^-25 below the
// row's norm); an fp32 operand is the sum of two f16 pieces, 22 bits.  f16 has few exponents, so every row of S, r and u carries
// a power of two of its own, from bounds that hold whatever the inputs: |k^| <= 1, 0 <= beta <= 1 and decays <= 1 make the rule a
// contraction, |r_t|, |u_t|, |S| <= |S_0| + sum |v_t| =: B per row, which is brought to 2^13 .. 2^15 for every chunk.  What a chunk
// makes of a row below 2^-38 of its B, as behind a decay of that much, is lost: the last bit of an f16.  T is bounded by 1 for the same
// reason.  The outputs get the same pieces as the state: with one piece each in S q and A u (11 bits) they lay 1.0e-3 of their norm from
// those of the plain form in 32 bits, with two 5e-5, as those of the token-by-token form do.
#include <cuda.h>
#include <stddef.h>

#include "lq_tc.cuh"

namespace lq {

// Sequences of fewer tokens are run token by token, longer ones in chunks.  A chunk costs a CTA 19 us however many tokens it has, the
// recurrence 8.6 us a token of 64 sequences of 32 heads and 0.45 us of one sequence, which leaves most of the device idle either way:
//     tokens                          24          28          32          40
//     64 sequences, 32 heads      212 : 279   248 : 280   282 : 282   352 : 281   us, token by token : in chunks
//      8 sequences, 32 heads       34 :  38    39 :  38    44 :  39    54 :  38
//      one sequence, 32 heads      13 :  19    14 :  19    16 :  19    20 :  19
constexpr int RULE_SHORT = 28;
// A batch of few heads whose sequences are long on average ends with its longest one, and SMs are idle by then: short sequences cost nothing
// in the chunked launch, but 0.45 us a token ahead of it.  Time with 8 against 28, lengths from 1 on evenly over their logarithm:
//     sequences x heads, per SM  0.6            1.3            2.0            2.6            2.9 .. 3.2     5.2 .. 5.4     8 .. 13        22
//     mean length 50 .. 130      0.87           0.92           0.73 .. 0.79   0.84           0.82 .. 0.91   0.97 .. 1.01   0.99 .. 1.12   1.06
//     mean length 150 .. 1 060   0.91 .. 0.97   0.81 .. 0.96   0.89 .. 0.97   0.91 .. 0.95   0.86 .. 0.99   0.93 .. 1.00   0.99 .. 1.06   1.02 .. 1.04
// It is used up to three heads an SM and from a mean of 256 tokens on: below that a batch may be drafts and single tokens, which the
// recurrence is for.  (8 heads and 32, 12 to 100 sequences.)
constexpr int RULE_SHORT_AMONG_LONG = 8;
constexpr int RANKED = 128;                                  // batches up to which CTAs take the longest sequences first
constexpr int CT = 64;                                       // tokens of a chunk
// T and A lie within [-1, 1]; times 2^13 their small entries keep eleven bits down to 2^-27 as well
constexpr float MAT_UP = 8192.f, MAT_DOWN = 1.f / 8192.f;
constexpr int MG = 2;                                        // threads that share a row of the state, each with
constexpr int SP = 64 / MG, TP = 32 / MG;                    // SP pairs of its columns and TP pairs of a chunk's tokens
constexpr int CK_MAIN = 128 * MG, CK_PREP = 128, CK_THREADS = CK_MAIN + 2 * CK_PREP + 32;
// Registers: 17 warps get 96 each (five of them share a quarter of the SM).  The main warps take over what the prep warps give up,
// 256 * 128 + 256 * 64 + 32 * 96 = 544 * 96; the launch looks that the kernel was built so, or they would wait for good.
constexpr int CK_REGS = 96, CK_MAIN_REGS = 128, CK_PREP_REGS = 64;
static_assert(MG == 2, "a thread exchanges its half of a row with one other");
static_assert(CK_MAIN * CK_MAIN_REGS + 2 * CK_PREP * CK_PREP_REGS + 32 * CK_REGS <= CK_THREADS * CK_REGS, "register split");

// Tensor memory, 512 columns.  D takes the place of X | XQ once both have been read.  The pieces of u for A u take that of S's heads once
// S q is through.  Two regions of 64 change roles with every chunk: one has S's remainders and, after S k, the outputs (e^G S q^ put there,
// A u added by the tensor cores), the other has u = T r -- and under the next chunk, whose remainders go there, the outputs stay.
constexpr uint32_t TM_SHI = 0, TM_UHI = 0, TM_ULO = 32, TM_X = 128, TM_XQ = 192, TM_D = 128, TM_PHI = 256, TM_PLO = 288;
__device__ __forceinline__ uint32_t tm_slo(int buf) { return buf ? 320u : 64u; }                    // and the outputs of the chunk
__device__ __forceinline__ uint32_t tm_gram(int buf) { return buf ? 384u : 448u; }                  // of the even and of the odd chunks

// f16 operands, fp32 accumulator; B with the reduction contiguous (K-major) or, for S += u k^T, the 128 key columns (MN-major)
__host__ __device__ constexpr uint32_t ck_idesc(int n, bool b_mn) { return (1u << 4) | (b_mn ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | ((128u >> 4) << 24); }
constexpr uint32_t CK_IDESC_BF16 = (1u << 7) | (1u << 10);    // both operands bf16
// Descriptor of rows of 128 bytes in the 128-byte swizzle, eight rows (1 KB) after one another; `lbo`: bytes between blocks of 64
// elements of a MN-major operand (not used by a K-major one, which is advanced by hand).
__device__ __forceinline__ uint64_t ck_desc(uint32_t addr, uint32_t lbo) {
    return uint64_t((addr >> 4) & 0x3FFFu) | (uint64_t((lbo >> 4) & 0x3FFFu) << 16) | (uint64_t(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Descriptor of an operand without swizzle, cores of eight rows by 16 bytes: the next eight rows follow, the next 16 bytes of a row are
// `kstep` bytes away.
__device__ __forceinline__ uint64_t ck_desc_cores(uint32_t addr, uint32_t kstep) {
    return uint64_t((addr >> 4) & 0x3FFFu) | (uint64_t(kstep >> 4) << 16) | (uint64_t(128 >> 4) << 32) | (1ull << 46);
}
// A [t][s] is kept in such cores, without the block of t < 32 <= s, which is zero: 16-byte chunk c (of 8) of row t
constexpr uint32_t AMAT_BYTES = 4096 + 2048;
__device__ __forceinline__ uint32_t ck_aoff(int t, int c) { return c < 4 ? c * 1024 + t * 16 : 4096 + (c - 4) * 512 + (t - 32) * 16; }
// byte offset of 16-byte chunk c (of 8) of a row in a swizzled tile
__device__ __forceinline__ uint32_t ck_off(int row, int c) { return uint32_t(row) * 128u + (uint32_t(c ^ (row & 7)) << 4); }

struct alignas(16) ChunkScalars {                                        // of one chunk, by token
    float c1[CT];                                            // -beta e^{G_t} kr_t: takes S k to what is added to beta v
    float beta[CT];
    float c2[CT];                                            // e^{G_t} qr_t 2^13, the scale of A u
    float c3[CT];                                            // e^{G_C - G_t} kr_t 2^-13 (u comes with the 2^13 of T)
    float decay;                                             // e^{G_C}
    int len;                                                 // tokens of the chunk, 1 .. 64; from bit 8 on ChunkOdd's `from`, bit 16: some bit of its q
};
struct alignas(16) PrepSmem {                                // of one prep group
    float L[3][32][36];                                      // blocks (0, 0), (1, 0), (1, 1); times 2^13, like all that becomes f16 on the way to T
    float tt[2][32][36];                                     // T^T of the two diagonal blocks of 32, times 2^13
    float2 G[CT];                                            // log2 of the decay from the chunk's start, head and remainder
    float gh[CT], gl[CT];                                    // the two apart and negated
    float kr[CT], qr[CT], ws[32], beta[CT];                  // 1 / |k|, 1 / |q|; ws: kr_s times the decay from s to token 31, for s < 32
    float down[2 * CT];                                      // powers of two that take the rows of k and q to f16
};
// Infinities and NaN.  A product with zero would carry them to tokens before their own, so they are taken out of a chunk's operands, and
// what depends on them becomes NaN at the end: a head's outputs and state from token `from` on (a key, a gate), the outputs of single
// tokens (q: bits by token), and a value dimension from its first such value on, which the main warps learn from the sums of |v|.
struct alignas(16) ChunkOdd {
    int from;                                                // CT: none
    uint32_t q[2];
};
constexpr int ODD_RING = 8;                                  // chunk c's: set up during chunk c - 4, last read when the outputs of c are written
struct alignas(16) ChunkSmem {
    // start: 1 KB aligned.  tile: two blocks of 64 elements, each 64 rows of k and then 64 rows of q.
    unsigned char tile[2][32768];
    unsigned char raw[32768];                                // the same as it comes, bf16
    unsigned char thi[8192], tlo[8192], v[16384];            // v: bf16, two blocks of 64 values by 64 rows
    unsigned char ahi[2][AMAT_BYTES], alo[2][AMAT_BYTES];
    uint16_t o[CT][VD];                                      // outputs on their way out
    PrepSmem prep[2];
    ChunkScalars sc[2];
    uint16_t vsum[8][VD];                                    // bf16 sums of |v| of a value dimension, over every eighth token each
    float part[2][CK_MAIN];
    ChunkOdd odd[ODD_RING];
    uint8_t vfrom[CK_MAIN];                                  // by main thread: first token of its value dimension that is not finite
    uint64_t raw_full[2], v_full[2], v_ready[2], tile_full[2], ta_full[2], main_done[2], au_full[2], g_full[2], ks_full, qs_full, y_full, d_full, s_ready, r_ready, u_ready, fin;
    uint32_t tm;
    int dead;                                                // a wait has run out
    int seq;                                                 // this CTA's sequence
    int len[RANKED];
};

static_assert(sizeof(ChunkScalars) % 16 == 0 && sizeof(PrepSmem) % 16 == 0 && offsetof(ChunkSmem, raw) % 1024 == 0 && offsetof(ChunkSmem, thi) % 1024 == 0 && offsetof(ChunkSmem, tlo) % 1024 == 0 &&
                  offsetof(ChunkSmem, ahi) % 16 == 0 && offsetof(ChunkSmem, alo) % 16 == 0 && offsetof(ChunkSmem, v) % 1024 == 0 && offsetof(ChunkSmem, o) % 128 == 0 &&
                  offsetof(ChunkSmem, prep) % 16 == 0 && offsetof(ChunkSmem, sc) % 16 == 0 && offsetof(ChunkSmem, vsum) % 16 == 0 &&
                  offsetof(PrepSmem, gh) % 16 == 0 && offsetof(PrepSmem, gl) % 16 == 0 && offsetof(PrepSmem, ws) % 16 == 0 && offsetof(ChunkSmem, raw_full) % 8 == 0,
              "vector accesses and swizzled tiles");

// Waits like warp_wait_bounded.  Once a wait of a warp has run out, its later ones test once and go on: the CTA runs to its end, on
// rubbish, and reports.
__device__ __forceinline__ void ck_wait(int& patience, uint64_t* bar, uint32_t parity) {
    int left = patience;
#pragma unroll 1
    while (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) {
        if (--left < 0) {
            patience = 0;
            break;
        }
    }
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }
// Exponent e with B 2^e in [2^13, 2^14), of b = B / 256 (a B beyond fp32's range is one as well: 2^128 of state and 64 values of 2^128).  At
// most 100: a row with a smaller bound, below 2^-87, is carried to 2^-125 at least, where fp32 ends.
constexpr int E_MIN = -122, E_MAX = 100;
__device__ __forceinline__ int scale_exponent(float b) {
    const int e = 132 - int((__float_as_uint(b) >> 23) & 255u);
    return e < E_MIN ? E_MIN : e > E_MAX ? E_MAX : e;
}
__device__ __forceinline__ uint32_t b2_bits(__nv_bfloat162 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ float2 f2_of(uint32_t a, uint32_t b) { return make_float2(__uint_as_float(a), __uint_as_float(b)); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
// two fp32 values as an f16 head and an f16 remainder: 22 bits.  (Two conversions there and one back, 6.5 cycles a pair; a head cut out
// with AND keeps the integer pipe busy for 9.)
__device__ __forceinline__ void split_h2(float2 x, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x.x, x.y);
    const float2 f = __half22float2(h), r = __fadd2_rn(x, make_float2(-f.x, -f.y));
    hi = h2_bits(h);
    lo = h2_bits(__floats2half2_rn(r.x, r.y));
}

// ---- prep warps -----------------------------------------------------------------------------------------------------------
// Group p prepares the chunks p, p + 2, ...: its latencies (a dozen dependent phases) are spread over two chunks of the main warps.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// decay from one token to a later one, of sums in two floats: their difference is good to 2^-24 of itself however large the sums are
__device__ __forceinline__ float decay_between(float2 to, float2 from) { return ex2((to.x - from.x) + (to.y - from.y)); }
__device__ __forceinline__ void prep_bar(int grp) { named_bar(2 + grp, CK_PREP); }

// k and q rows of a chunk, or its rows of v, as they come: boxes of 64 rows by 64 elements in the 128-byte swizzle.  Rows behind the
// chunk's last token belong to other sequences (or lie behind the tensor: zeros).
__device__ __forceinline__ void ck_fetch_kq(ChunkSmem& s, const CUtensorMap* rows, int xk, int xq, int t0, uint64_t* full) {
    mbar_arrive_expect_tx(full, 4 * 8192);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        tma_load_2d(s.raw + 16384 * b, rows, xk + 64 * b, t0, full);
        tma_load_2d(s.raw + 16384 * b + 8192, rows, xq + 64 * b, t0, full);
    }
}
__device__ __forceinline__ void ck_fetch_v(ChunkSmem& s, const CUtensorMap* rows, int xv, int t0, uint64_t* full) {
    mbar_arrive_expect_tx(full, 2 * 8192);
#pragma unroll
    for (int b = 0; b < 2; ++b) tma_load_2d(s.v + 8192 * b, rows, xv + 64 * b, t0, full);
}
// Sum of eight values over the sixteen lanes that share lane >> 4: every exchange halves what a lane keeps.  Lane l returns the total of
// value (l >> 1) & 7.
__device__ __forceinline__ float fold8(const float (&v)[8], int lane) {
    const bool u8 = lane & 8, u4 = lane & 4, u2 = lane & 2;
    float a[4], b[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = (u8 ? v[4 + i] : v[i]) + __shfl_xor_sync(0xffffffffu, u8 ? v[i] : v[4 + i], 8);
#pragma unroll
    for (int i = 0; i < 2; ++i) b[i] = (u4 ? a[2 + i] : a[i]) + __shfl_xor_sync(0xffffffffu, u4 ? a[i] : a[2 + i], 4);
    float s = (u2 ? b[1] : b[0]) + __shfl_xor_sync(0xffffffffu, u2 ? b[0] : b[1], 2);
    return s + __shfl_xor_sync(0xffffffffu, s, 1);
}
// whether one of two bf16 values is an infinity or NaN
__device__ __forceinline__ bool not_finite(uint32_t two) { return (two & 0x7f80u) == 0x7f80u || (two & 0x7f800000u) == 0x7f800000u; }
// Sums of |v| / 256 over the tokens g, g + 8, ... of a chunk (g: this half of a warp), for a bound: bf16 will do, rounded up by the reader.  A
// lane reads one 16-byte piece of the rows, the same eight values in all of them, since the swizzle goes by the row's number mod 8.
__device__ __forceinline__ void ck_vsum(unsigned char* v, uint16_t (&vsum)[8][VD], int w, int lane) {
    const int g = 2 * w + (lane >> 4), c = lane & 15;
    v += (c >> 3) * 8192 + g * 128 + (c & 7) * 16;
    const __nv_bfloat162 part = __floats2bfloat162_rn(1.f / 256, 1.f / 256);
    __nv_bfloat162 sum[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll 2
    for (int i = 0; i < 8; ++i) {
        const uint4 x = *reinterpret_cast<const uint4*>(v + 1024 * i);
        const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] = __hfma2(__habs2(*reinterpret_cast<const __nv_bfloat162*>(&xw[j])), part, sum[j]);
    }
    uint16_t* to = &vsum[g][64 * (c >> 3) + 8 * ((c & 7) ^ g)];
    *reinterpret_cast<uint4*>(to) = make_uint4(b2_bits(sum[0]), b2_bits(sum[1]), b2_bits(sum[2]), b2_bits(sum[3]));
    if (__builtin_expect(not_finite(b2_bits(__hadd2(__hadd2(sum[0], sum[1]), __hadd2(sum[2], sum[3])))), 0)) {
        // cleared; the place of a sum takes a NaN with the first such token in it
#pragma unroll 1
        for (int i = 63; i >= 0; --i) {
            uint16_t* x = reinterpret_cast<uint16_t*>(v + 1024 * (i >> 3)) + (i & 7);
            if (not_finite(*x)) {
                *x = 0;
                to[i & 7] = uint16_t(0x7fc0 | i >> 3);
            }
        }
        fence_async_smem();                                  // (the next copy of v goes to the same place)
    }
}
// rows behind the chunk's last token, which belong to other sequences, become zeros; pieces of 16 bytes, blocks of 64 rows
__device__ __forceinline__ void ck_clear(unsigned char* p, int blocks, int len, int pt, int threads) {
#pragma unroll 1
    for (int i = pt; i < blocks * 512; i += threads)
        if (((i >> 3) & 63) >= len) *reinterpret_cast<uint4*>(p + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
}
// Norms of the rows of k (warps 0 and 1) and q.  A lane takes the same 16 bytes of sixteen rows, whichever they are in the swizzle.
__device__ __forceinline__ void ck_norms(unsigned char* raw, float* rs, float* down, ChunkOdd& odd, int w, int lane) {
    const int c = lane & 15;
    raw += (c >> 3) * 16384 + (32 * w + (lane >> 4)) * 128 + (c & 7) * 16;
    rs += 32 * (w & 1);
    bool large = false;
#pragma unroll 1
    for (int p = 0; p < 2; ++p) {
        float ss[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint4 x = *reinterpret_cast<const uint4*>(raw + 2048 * p + 256 * i);
            const float2 f0 = bf16x2_to_f2(x.x), f1 = bf16x2_to_f2(x.y), f2 = bf16x2_to_f2(x.z), f3 = bf16x2_to_f2(x.w);
            const float2 a = __ffma2_rn(f1, f1, __fmul2_rn(f0, f0)), b = __ffma2_rn(f3, f3, __fmul2_rn(f2, f2)), c2 = __fadd2_rn(a, b);
            ss[i] = c2.x + c2.y;
        }
        const float sum = fold8(ss, lane);
        large |= !(sum <= 3.4e38f);
        // the row times 2^-e has a norm in [1, 2)
        int e = (int((__float_as_uint(sum) >> 23) & 255u) - 127) >> 1;
        e = e < -60 ? -60 : e;
        if (!(lane & 1)) {
            const int r = 16 * p + 2 * ((lane >> 1) & 7) + (lane >> 4);
            rs[r] = rsqrtf(sum + 1e-6f);
            down[32 * w + r] = pow2f(-e);
        }
    }
    // a sum of squares beyond fp32 makes the row zero, as 1 / sqrt(inf) does, and so does an infinity or NaN, which is noted
    if (__builtin_expect(__any_sync(0xffffffffu, large), 0)) {
        __syncwarp();                                        // (rs is another lane's)
#pragma unroll 1
        for (int i = 0; i < 16; ++i) {
            const int r = 2 * i + (lane >> 4);
            uint4* at = reinterpret_cast<uint4*>(raw + 256 * i);
            const unsigned bad = __ballot_sync(0xffffffffu, not_finite(at->x) || not_finite(at->y) || not_finite(at->z) || not_finite(at->w));
            const bool zero = !(rs[r] > 0.f);
            __syncwarp();
            if (zero) *at = make_uint4(0u, 0u, 0u, 0u);
            if (zero && c == 0) {
                rs[r] = 0.f;
                if (bad >> (lane & 16) & 0xffffu) {
                    if (w < 2) atomicMin(&odd.from, 32 * w + r);
                    else atomicOr(&odd.q[w & 1], 1u << r);
                }
            }
        }
    }
}
// rows of k and q as f16
__device__ __forceinline__ void ck_convert(const unsigned char* raw, unsigned char* tile, const float* down, int w, int lane) {
    const int c = lane & 15, at = (c >> 3) * 16384 + (32 * w + (lane >> 4)) * 128 + (c & 7) * 16;
    down += 32 * w + (lane >> 4);
#pragma unroll 1
    for (int p = 0; p < 4; ++p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 x = *reinterpret_cast<const uint4*>(raw + at + 1024 * p + 256 * i);
            const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
            const float m = down[8 * p + 2 * i];
            uint32_t h[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 y = __fmul2_rn(bf16x2_to_f2(xw[j]), both(m));
                h[j] = h2_bits(__floats2half2_rn(y.x, y.y));
            }
            *reinterpret_cast<uint4*>(tile + at + 1024 * p + 256 * i) = make_uint4(h[0], h[1], h[2], h[3]);
        }
    }
}
// log2(1 + e^x): with z = e^-|x| and r = z / (2 + z) <= 1/3, log(1 + z) = 2 (r + r^3/3 + r^5/5 + ...), the next term below 2^-24 of it
__device__ __forceinline__ float softplus_log2(float x) {
    const float z = ex2(-1.4426950408889634f * fabsf(x)), r = __fdividef(z, 2.0f + z), q = r * r;
    float p = 1.0f / 15.0f;
    p = fmaf(p, q, 1.0f / 13.0f);
    p = fmaf(p, q, 1.0f / 11.0f);
    p = fmaf(p, q, 1.0f / 9.0f);
    p = fmaf(p, q, 1.0f / 7.0f);
    p = fmaf(p, q, 1.0f / 5.0f);
    p = fmaf(p, q, 1.0f / 3.0f);
    p = fmaf(p, q, 1.0f);
    return fmaf(2.0f * 1.4426950408889634f * r, p, x > 0.f ? x * 1.4426950408889634f : 0.f);
}
// decays and beta of the chunk, by one warp: lane l has the tokens 2 l and 2 l + 1; sums in fp64
__device__ __forceinline__ void ck_gates(PrepSmem& s, ChunkOdd& odd, const uint16_t* a, int64_t a_step, const uint16_t* b, int64_t b_step, int len, float ea,
                                         float dtb, int lane) {
    double g[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int t = 2 * lane + i, u = t < len ? t : 0;
        const float x = -ea * softplus_log2(bf16_to_f(__ldg(a + u * a_step)) + dtb), y = bf16_to_f(__ldg(b + u * b_step));
        const float be = __fdividef(1.0f, 1.0f + ex2(-1.4426950408889634f * y));
        bool in = t < len;
        if (__builtin_expect(in && !(x <= 0.f && be >= 0.f), 0)) {
            atomicMin(&odd.from, t);
            in = false;
        }
        // a decay of 2^-300 leaves nothing in fp32; bounded, the differences stay finite
        g[i] = in ? double(x < -300.f ? -300.f : x) : 0.0;
        s.beta[t] = in ? be : 0.f;
    }
    double sum = g[0] + g[1];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const double o = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += o;
    }
    const double first = sum - g[1];
    const float h0 = float(first), h1 = float(sum);
    s.G[2 * lane] = make_float2(h0, float(first - double(h0)));
    s.G[2 * lane + 1] = make_float2(h1, float(sum - double(h1)));
}

// eight columns of a row of A or L to their places
__device__ __forceinline__ void ck_put8(PrepSmem& s, unsigned char* ahi, unsigned char* alo, bool isq, int t, int c8, const float2 (&y)[4]) {
    if (isq) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) split_h2(y[j], h[j], l[j]);
        *reinterpret_cast<uint4*>(ahi + ck_aoff(t, c8)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(alo + ck_aoff(t, c8)) = make_uint4(l[0], l[1], l[2], l[3]);
    } else {
        float* to = &s.L[(t >> 5) + (c8 >> 2)][t & 31][8 * (c8 & 3)];
        *reinterpret_cast<float4*>(to) = make_float4(y[0].x, y[0].y, y[1].x, y[1].y);
        *reinterpret_cast<float4*>(to + 4) = make_float4(y[2].x, y[2].y, y[3].x, y[3].y);
    }
}
// Gram rows -> L (fp32, k rows) and A (two f16 pieces, q rows); a thread has a row.  Inside a diagonal block of 32 tokens the decay is
// taken pair by pair; from the first block to the second in two steps over token 31, neither of which exceeds 1.
__device__ __forceinline__ void ck_gram(PrepSmem& s, unsigned char* ahi, unsigned char* alo, uint32_t gram, int w, int lane) {
    const bool isq = w >= 2;
    const int blk = w & 1, t = 32 * blk + lane;
    const float2 Gt = s.G[t];
    const float rowf = (isq ? s.qr[t] : s.kr[t] * s.beta[t]) * MAT_UP;
    gram += uint32_t(32 * w) << 16;
    if (blk == 1) {
        const float f = rowf * decay_between(Gt, s.G[31]);
#pragma unroll 1
        for (int c8 = 0; c8 < 4; ++c8) {
            uint32_t g[8];
            float2 y[4];
            tmem_ld_8(gram + 8 * c8, g);
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = __fmul2_rn(__fmul2_rn(f2_of(g[2 * j], g[2 * j + 1]), both(f)), *reinterpret_cast<const float2*>(&s.ws[8 * c8 + 2 * j]));
            ck_put8(s, ahi, alo, isq, t, c8, y);
        }
    }
    const int last = isq ? lane : lane - 1;                  // last column of the diagonal block that counts
#pragma unroll 1
    for (int c8 = 0; c8 < 4; ++c8) {
        uint32_t g[8];
        float2 y[4];
        tmem_ld_8(gram + 32 * blk + 8 * c8, g);
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
            const int c = 8 * c8 + 2 * j;
            const float4 fh = *reinterpret_cast<const float4*>(&s.gh[32 * blk + c]), fl = *reinterpret_cast<const float4*>(&s.gl[32 * blk + c]);
            const float2 d0 = __fadd2_rn(__fadd2_rn(both(Gt.x), make_float2(fh.x, fh.y)), __fadd2_rn(both(Gt.y), make_float2(fl.x, fl.y)));
            const float2 d1 = __fadd2_rn(__fadd2_rn(both(Gt.x), make_float2(fh.z, fh.w)), __fadd2_rn(both(Gt.y), make_float2(fl.z, fl.w)));
            const float4 kr = *reinterpret_cast<const float4*>(&s.kr[32 * blk + c]);
            const float2 z0 = __fmul2_rn(__fmul2_rn(f2_of(g[2 * j], g[2 * j + 1]), __fmul2_rn(both(rowf), make_float2(kr.x, kr.y))), make_float2(ex2(d0.x), ex2(d0.y)));
            const float2 z1 = __fmul2_rn(__fmul2_rn(f2_of(g[2 * j + 2], g[2 * j + 3]), __fmul2_rn(both(rowf), make_float2(kr.z, kr.w))), make_float2(ex2(d1.x), ex2(d1.y)));
            y[j] = make_float2(c <= last ? z0.x : 0.f, c < last ? z0.y : 0.f);
            y[j + 1] = make_float2(c + 2 <= last ? z1.x : 0.f, c + 2 < last ? z1.y : 0.f);
        }
        ck_put8(s, ahi, alo, isq, t, 4 * blk + c8, y);
    }
}
struct Pieces { uint32_t hi, lo; };
__device__ __forceinline__ Pieces pieces(float2 x) {
    Pieces p;
    split_h2(x, p.hi, p.lo);
    return p;
}
__device__ __forceinline__ void mma_pieces(float (&d)[4], const Pieces (&a)[4], const Pieces& b0, const Pieces& b1) {
    mma_h_16816(d, a[0].lo, a[1].lo, a[2].lo, a[3].lo, b0.hi, b1.hi);
    mma_h_16816(d, a[0].hi, a[1].hi, a[2].hi, a[3].hi, b0.lo, b1.lo);
    mma_h_16816(d, a[0].hi, a[1].hi, a[2].hi, a[3].hi, b0.hi, b1.hi);
}
__device__ __forceinline__ void put_t(unsigned char* thi, unsigned char* tlo, int t, int c, Pieces p) {
    const uint32_t off = ck_off(t, c >> 3) + 2 * (c & 7);
    *reinterpret_cast<uint32_t*>(thi + off) = p.hi;
    *reinterpret_cast<uint32_t*>(tlo + off) = p.lo;
}
// T = (I + L)^-1 in blocks: 16 x 16 by substitution (warp w has diagonal block w, a lane a column of T, which is a row of T^T), then twice
// the lower left block -T22 (L21 T11) of a square twice as large, on mma.sync.  The first product is taken transposed, (L21 T11)^T =
// T11^T L21^T: its accumulators are then the B operand of the second as they are.  Scales: L and T times 2^13, their product back to
// 2^10 (a sum of 32).  Loops rather than straight code: an SM's instruction cache holds 32 KB, and beyond that every instruction of the
// kernel costs 2.7 cycles.
__device__ __forceinline__ void ck_invert(PrepSmem& s, unsigned char* thi, unsigned char* tlo, uint64_t* t_free, uint32_t t_parity, int& patience,
                                          int grp, int w, int lane) {
    const int gid = lane >> 2, tig = lane & 3;
    {
        const int o = 16 * w, c = lane & 15;
        float* tt = &s.tt[w >> 1][(o & 16) + c][o & 16];     // this column of T
#pragma unroll
        for (int b = 0; b < 16; b += 4) {
            const float* l = &s.L[w & 2][(o & 16) + b][o & 16];
            float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int m = 0; m < b; m += 4) {
                const float4 x = *reinterpret_cast<const float4*>(tt + m);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float4 y = *reinterpret_cast<const float4*>(l + r * 36 + m);
                    a[r] = fmaf(y.x, x.x, fmaf(y.y, x.y, fmaf(y.z, x.z, fmaf(y.w, x.w, a[r]))));
                }
            }
            const float l10 = l[36 + b];
            const float2 l2 = *reinterpret_cast<const float2*>(l + 2 * 36 + b);
            const float4 l3 = *reinterpret_cast<const float4*>(l + 3 * 36 + b);
            float4 x;
            x.x = fmaf(a[0], -MAT_DOWN, c == b ? MAT_UP : 0.f);
            x.y = fmaf(fmaf(l10, x.x, a[1]), -MAT_DOWN, c == b + 1 ? MAT_UP : 0.f);
            x.z = fmaf(fmaf(l2.x, x.x, fmaf(l2.y, x.y, a[2])), -MAT_DOWN, c == b + 2 ? MAT_UP : 0.f);
            x.w = fmaf(fmaf(l3.x, x.x, fmaf(l3.y, x.y, fmaf(l3.z, x.z, a[3]))), -MAT_DOWN, c == b + 3 ? MAT_UP : 0.f);
            *reinterpret_cast<float4*>(tt + b) = x;          // (both halves of the warp: the same)
        }
        __syncwarp();
        if (t_free) ck_wait(patience, t_free, t_parity);     // the T of the chunk before has been used
        const float* d = &s.tt[w >> 1][(o & 16) + 2 * tig][(o & 16) + gid];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = 8 * (r & 1), n = 8 * (r >> 1);
            put_t(thi, tlo, o + gid + i, o + 2 * tig + n, pieces(make_float2(d[n * 36 + i], d[n * 36 + 36 + i])));
        }
    }
#pragma unroll 1
    for (int h = 16; h <= 32; h += 16) {
        prep_bar(grp);
        // of the square of 2 h at o: sixteen columns from n0 on, sixteen rows from i0 on (h = 16: two warps do the same)
        const int o = h == 16 ? 32 * (w >> 1) : 0, n0 = h == 16 ? 0 : 16 * (w & 1), i0 = h == 16 ? 0 : 16 * (w >> 1);
        float* t11 = &s.tt[h == 16 ? w >> 1 : 0][0][0];      // T^T of the two diagonal blocks, rows of 36
        const float* t22 = h == 16 ? t11 + 16 * 36 + 16 : &s.tt[1][0][0];
        const float* l21 = h == 16 ? &s.L[w & 2][16 + gid][2 * tig] : &s.L[1][gid][2 * tig];
        float d[2][4] = {};
#pragma unroll 1
        for (int k2 = 0; k2 <= i0; k2 += 16) {               // sixteen rows of L21 T11; T22 is lower triangular
            float X[2][4] = {};
            Pieces a[4], b[2][2];
#pragma unroll 1
            for (int ks = n0; ks < h; ks += 16) {            // so is T11
                const float* ta = t11 + (n0 + gid) * 36 + ks + 2 * tig;
#pragma unroll
                for (int r = 0; r < 4; ++r) a[r] = pieces(*reinterpret_cast<const float2*>(ta + (r & 1) * 8 * 36 + (r >> 1) * 8));
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float* l = l21 + (k2 + 8 * j) * 36 + ks;
                    mma_pieces(X[j], a, pieces(*reinterpret_cast<const float2*>(l)), pieces(*reinterpret_cast<const float2*>(l + 8)));
                }
            }
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int j = 0; j < 2; ++j) b[q][j] = pieces(__fmul2_rn(make_float2(X[j][2 * q], X[j][2 * q + 1]), both(0x1p-16f)));
            const float* tb = t22 + (k2 + 2 * tig) * 36 + i0 + gid;
#pragma unroll
            for (int r = 0; r < 4; ++r) a[r] = pieces(make_float2(tb[(r >> 1) * 8 * 36 + (r & 1) * 8], tb[(r >> 1) * 8 * 36 + 36 + (r & 1) * 8]));
#pragma unroll
            for (int q = 0; q < 2; ++q) mma_pieces(d[q], a, b[q][0], b[q][1]);
        }
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int i = i0 + gid + 8 * r, n = n0 + 8 * q + 2 * tig;
                const float2 y = __fmul2_rn(make_float2(d[q][2 * r], d[q][2 * r + 1]), both(-0x1p-10f));
                put_t(thi, tlo, o + h + i, o + n, pieces(y));
                if (h == 16) {
                    t11[n * 36 + 16 + i] = y.x;
                    t11[n * 36 + 36 + 16 + i] = y.y;
                }
            }
    }
}

// The values of chunk c are there: rows behind the chunk's end cleared (all of them: len = 0), and the sums for the bounds.
__device__ __forceinline__ void ck_values(ChunkSmem& s, int c, int64_t len, int grp, int w, int lane, int& patience) {
    const int buf = c & 1, pt = 32 * w + lane;
    const int64_t left = len - int64_t(c) * CT;
    ck_wait(patience, &s.v_full[buf], uint32_t(c >> 1) & 1u);
    if (left < CT) {
        ck_clear(s.v, 2, int(left), pt, CK_PREP);
        fence_async_smem();                                  // (the next copy of v goes to the same place)
        prep_bar(grp);
    }
    ck_vsum(s.v, s.vsum, w, lane);
    prep_bar(grp);
    if (pt == 0) mbar_arrive(&s.v_ready[buf]);
    __syncwarp();
}
__device__ __forceinline__ void ck_prep(ChunkSmem& s, const RuleParams& P, const CUtensorMap* rows, int hk, int hv, int64_t t0, int64_t len, int64_t vlen, int nchunk, uint32_t tm,
                                        int grp, int w, int lane, int& patience) {
    const uint32_t el = elect_one();
    const int pt = 32 * w + lane;
    PrepSmem& ps = s.prep[grp];
    ChunkScalars& q = s.sc[grp];
    const float ea = expf(P.A_log[hv]), dtb = P.dt_bias[hv];
    if (grp == 0 && w == 0 && el) ck_fetch_kq(s, rows, (P.H + hk) * KD, hk * KD, int(t0), &s.raw_full[0]);
    __syncwarp();
#pragma unroll 1
    for (int c = grp; c < nchunk; c += 2) {
        const uint32_t ph = uint32_t(c >> 1) & 1u, pc = uint32_t(c) & 1u;
        const int64_t at = t0 + int64_t(c) * CT, left = len - int64_t(c) * CT;
        const int n = int(left < CT ? left : CT);
        ChunkOdd& odd = s.odd[c & (ODD_RING - 1)];
        if (w == 3)
            ck_gates(ps, odd, P.a + at * P.a_stride + hv, P.a_stride, P.b + at * P.b_stride + hv, P.b_stride, n, ea, dtb, lane);
        ck_wait(patience, &s.raw_full[grp], ph);
        if (c != 1) ck_values(s, c == 0 ? 0 : c - 1, vlen, grp, w, lane, patience);     // of the chunk before: the other group has its hands full
        if (n < CT) {
            ck_clear(s.raw, 4, n, pt, CK_PREP);
            prep_bar(grp);
        }
        ck_norms(s.raw, w < 2 ? ps.kr : ps.qr, ps.down, odd, w, lane);
        fence_async_smem();
        prep_bar(grp);
        if (pt == 0) {
            ChunkOdd& later = s.odd[(c + 4) & (ODD_RING - 1)];
            later.from = CT;
            later.q[0] = later.q[1] = 0;
        }
        if (w == 0) {                                        // K K^T and Q K^T of the rows as they are
            tc_fence_after_sync();
            const uint64_t d0 = ck_desc(smem_u32(s.raw), 16);
#pragma unroll 4
            for (int ks = 0; ks < 8; ++ks) {
                const uint64_t d = d0 + uint64_t(((ks >> 2) * 16384 + (ks & 3) * 32) >> 4);
                umma_f16_ss(el, tm + tm_gram(grp), d, d, ck_idesc(64, false) | CK_IDESC_BF16, ks > 0);
            }
            umma_commit_if(el, &s.g_full[grp]);
            __syncwarp();
        }
        if (c >= 2) ck_wait(patience, &s.main_done[grp], ph ^ 1u);
        ck_convert(s.raw, s.tile[grp], ps.down, w, lane);
        ck_wait(patience, &s.g_full[grp], ph);               // (the rows as they are have been read, and the matrix is there)
        fence_async_smem();
        prep_bar(grp);
        if (w == 0 && el && c + 1 < nchunk) {                // the next chunk, for the other group, into the buffer that is free now
            ck_fetch_kq(s, rows, (P.H + hk) * KD, hk * KD, int(at) + CT, &s.raw_full[grp ^ 1]);
            if (c + 2 < nchunk)
#pragma unroll 1
                for (int b = 0; b < 4; ++b) tma_prefetch_2d(rows, ((b & 2 ? P.H : 0) + hk) * KD + 64 * (b & 1), int(at) + 2 * CT);
        }
        __syncwarp();
        if (w >= 2) {                                        // scalars for the main warps, which may then begin
            const int tk = pt - 64;
            const float2 G = ps.G[tk], Gc = ps.G[CT - 1];
            const float e = ex2(G.x + G.y), kr = __fdividef(ps.kr[tk], ps.down[tk]), b = ps.beta[tk];
            q.c1[tk] = -(b * e * kr);
            q.beta[tk] = b;
            q.c2[tk] = e * __fdividef(ps.qr[tk], ps.down[CT + tk]) * MAT_UP;
            q.c3[tk] = decay_between(Gc, G) * kr * MAT_DOWN;
            if (tk == 0) {
                q.decay = ex2(Gc.x + Gc.y);
                q.len = n | odd.from << 8 | ((odd.q[0] | odd.q[1]) != 0) << 16;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.tile_full[grp]);
        } else if (w == 1) {                                 // and for the Gram rows
            const float2 g0 = ps.G[lane], g1 = ps.G[lane + 32];
            ps.gh[lane] = -g0.x;
            ps.gl[lane] = -g0.y;
            ps.gh[lane + 32] = -g1.x;
            ps.gl[lane + 32] = -g1.y;
            ps.ws[lane] = decay_between(ps.G[31], g0) * ps.kr[lane];
        }
        prep_bar(grp);
        tc_fence_after_sync();
        ck_gram(ps, s.ahi[grp], s.alo[grp], tm + tm_gram(grp), w, lane);
        tc_fence_before_sync();                              // (the matrix has been read)
        prep_bar(grp);
        ck_invert(ps, s.thi, s.tlo, c > 0 ? &s.y_full : nullptr, pc ^ 1u, patience, grp, w, lane);
        fence_async_smem();
        prep_bar(grp);
        if (pt == 0) mbar_arrive(&s.ta_full[grp]);
        __syncwarp();
    }
    if (nchunk > 1 && (nchunk & 1) == grp) ck_values(s, nchunk - 1, vlen, grp, w, lane, patience);
    if (w == 0) umma_commit_if(el, &s.fin);
}

// ---- main warps -----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float sqrt_approx(float x) {
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two neighbouring tokens' values (2 i and 2 i + 1 of eight) of a value dimension, in the swizzle of their tile
__device__ __forceinline__ float2 v_two(const unsigned char* p, int vc, int i) {
    return make_float2(bf16_to_f(*reinterpret_cast<const uint16_t*>(p + 2 * i * 128 + ((vc ^ (2 * i)) << 4))),
                       bf16_to_f(*reinterpret_cast<const uint16_t*>(p + (2 * i + 1) * 128 + ((vc ^ (2 * i + 1)) << 4))));
}
// a warp has written its part of an operand in tensor memory
__device__ __forceinline__ void ck_ready(uint64_t* bar, int lane) {
    tmem_st_wait();
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
    __syncwarp();
}
// Chunk c's outputs are finished while S k of chunk c + 1 is under way, and leave for memory while T r of it is.
__device__ __forceinline__ void ck_main(ChunkSmem& s, const RuleParams& P, int hv, int64_t t0, int nchunk, const float* Sin, bool unit, float* Sout, bool outputs,
                                        uint32_t tm, int tid, int& patience) {
    const int lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), h = warp >> 2, v = 32 * (warp & 3) + lane;
    const uint32_t row = tm + (uint32_t(32 * (warp & 3)) << 16);
    float2 S[SP];                                            // S[v][2 SP h ..] times 2^e
    const int at = v * KD + 2 * SP * h;
#pragma unroll
    for (int i = 0; i < SP / 2; ++i) {
        float4 x = Sin ? *reinterpret_cast<const float4*>(Sin + at + 4 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
        if (unit) {
            const int d = v - 2 * SP * h - 4 * i;
            x = make_float4(d == 0 ? 1.f : 0.f, d == 1 ? 1.f : 0.f, d == 2 ? 1.f : 0.f, d == 3 ? 1.f : 0.f);
        }
        S[2 * i] = make_float2(x.x, x.y);
        S[2 * i + 1] = make_float2(x.z, x.w);
    }
    int e = Sin || unit ? 0 : E_MAX, plen = 0;
    float decay = 0.f, of = 0.f;                             // of the chunk before: its decay, and what its outputs are multiplied with
    const int vc = (v >> 3) & 7, voff = (v >> 6) * 8192 + 2 * TP * h * 128 + 2 * (v & 7);
#pragma unroll 1
    for (int c = 0; c <= nchunk; ++c) {
        const int buf = c & 1;
        const uint32_t ph = uint32_t(c >> 1) & 1u, slo = tm_slo(buf), tmy = tm_slo(buf ^ 1);
        const ChunkScalars& q = s.sc[buf];
        const unsigned char* vp = s.v + voff;
        float va = 0.f;
        if (c < nchunk) {
            ck_wait(patience, &s.tile_full[buf], ph);
            ck_wait(patience, &s.v_ready[buf], ph);
#pragma unroll
            for (int g = 0; g < 8; ++g) va += bf16_to_f(s.vsum[g][v]);
            va *= 1.125f;                                    // (sums in bf16: not below the true one, of |v| / 256)
            if (__builtin_expect(!(va < 3.4e38f), 0)) {      // some were not finite: when the first, and the sum of the others
                int from = CT;
                va = 0.f;
                const unsigned char* all = s.v + (v >> 6) * 8192 + 2 * (v & 7);
#pragma unroll 1
                for (int t = 0; t < CT; ++t) {
                    const uint32_t g = s.vsum[t & 7][v];
                    if ((g & 0x7f80u) == 0x7f80u && int(g & 7u) == t >> 3) from = min(from, t);
                    va += (1.f / 256) * fabsf(bf16_to_f(*reinterpret_cast<const uint16_t*>(all + t * 128 + ((vc ^ (t & 7)) << 4))));
                }
                s.vfrom[tid] = uint8_t(from);
            }
        }
        if (c > 0) {                                         // the state behind the chunk before
            ck_wait(patience, &s.d_full, uint32_t(c - 1) & 1u);
            tc_fence_after_sync();
#pragma unroll
            for (int p = 0; p < SP / 8; ++p) {
                uint32_t r[16];
                tmem_ld_16(row + TM_D + 2 * SP * h + 16 * p, r);
#pragma unroll
                for (int i = 0; i < 8; ++i) S[8 * p + i] = __ffma2_rn(S[8 * p + i], both(decay), f2_of(r[2 * i], r[2 * i + 1]));
            }
        }
        if (c < nchunk) {
            // the row's power of two: B = |S| + sum |v| becomes 2^13 or more
            const int pair = 4 + (warp & 3);                 // barrier of the warps that share these rows
#pragma unroll 1
            for (bool again = false;; again = true) {
                float2 n2[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) n2[i] = __fmul2_rn(S[i], S[i]);
#pragma unroll
                for (int i = 4; i < SP; ++i) n2[i & 3] = __ffma2_rn(S[i], S[i], n2[i & 3]);
                n2[0] = __fadd2_rn(__fadd2_rn(n2[0], n2[1]), __fadd2_rn(n2[2], n2[3]));
                const float mine = n2[0].x + n2[0].y;
                s.part[buf][tid] = mine;
                named_bar(pair, 32 * MG);
                const float sum2 = mine + s.part[buf][tid ^ 128];
                // (kept while the bound stays between 2^13 and 2^15)
                int de = scale_exponent(fmaf(sqrt_approx(sum2), pow2f(-e - 8), va)) - e;
                if (de == -1) de = 0;
                // Squares stand for their row while they are well inside fp32's range; at the largest exponent only those of zeros are not
                const bool beyond = !again && !(sum2 < 0x1p120f && (sum2 > 0x1p-100f || e == E_MAX));
                if (__all_sync(0xffffffffu, de == 0 && !beyond)) break;
                if (__any_sync(0xffffffffu, beyond)) {
                    // a state as the caller gives it, or one that decayed far within a chunk: first to a largest value in [1, 2).  (Both warps of
                    // the rows have seen the same sums.)
                    float big = 0.f;
#pragma unroll
                    for (int i = 0; i < SP; ++i) big = fmaxf(big, fmaxf(fabsf(S[i].x), fabsf(S[i].y)));
                    s.part[buf ^ 1][tid] = big;
                    named_bar(pair, 32 * MG);
                    big = fmaxf(big, s.part[buf ^ 1][tid ^ 128]);
                    de = 127 - int((__float_as_uint(big) >> 23) & 255u);
                    de = de < E_MIN - e ? E_MIN - e : de > E_MAX - e ? E_MAX - e : de;
                    de = de > 126 ? 126 : de;
                    if (big == 0.f) de = -e;
                    again = true;
                } else again = false;
                const float2 up = both(de < -126 ? 0.f : pow2f(de));
                e += de;
#pragma unroll
                for (int i = 0; i < SP; ++i) S[i] = __fmul2_rn(S[i], up);
                if (!again) break;
            }
        }
        if (c > 0) {
            ck_wait(patience, &s.au_full[buf ^ 1], uint32_t((c - 1) >> 1) & 1u);
            tc_fence_after_sync();
            // every product of that chunk is through, and its scalars have been read: its buffers are free
            if (c + 1 < nchunk && lane == 0) mbar_arrive(&s.main_done[buf ^ 1]);
            __syncwarp();
        }
        if (c < nchunk) {
#pragma unroll
            for (int p = 0; p < SP / 8; ++p) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    split_h2(S[8 * p + i], hi[i], lo[i]);
                }
                tmem_st_8(row + TM_SHI + SP * h + 8 * p, hi);
                tmem_st_8(row + slo + SP * h + 8 * p, lo);
            }
            ck_ready(&s.s_ready, lane);
        }
        if (c > 0) {                                         // outputs of the chunk before
#pragma unroll 2
            for (int p = 0; p < TP / 4; ++p) {
                uint32_t x[8];
                tmem_ld_8(row + tmy + 2 * TP * h + 8 * p, x);
                uint16_t* op = &s.o[2 * TP * h + 8 * p][v];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 y = __fmul2_rn(f2_of(x[2 * i], x[2 * i + 1]), both(of));
                    const uint32_t b = f2_to_bf16x2(y.x, y.y);
                    op[2 * i * VD] = uint16_t(b);
                    op[(2 * i + 1) * VD] = uint16_t(b >> 16);
                }
            }
            if (__builtin_expect(plen >> 8 != CT, 0)) {      // what depends on an infinity or NaN
                const uint32_t late = plen >> 8 & 255, bits = s.odd[(c - 1) & (ODD_RING - 1)].q[h];
#pragma unroll 1
                for (int i = 0; i < 2 * TP; ++i)
                    if (2 * TP * h + i >= late || (bits >> i & 1u)) s.o[2 * TP * h + i][v] = 0x7fff;
                plen &= 255;
            }
            fence_async_smem();
        }
        if (c == nchunk) {
            named_bar(1, CK_MAIN);
#pragma unroll 1
            for (int r = tid >> 4; r < (outputs ? plen & 255 : 0); r += CK_MAIN / 16)
                *reinterpret_cast<uint4*>(P.o + ((t0 + int64_t(c - 1) * CT + r) * P.HV + hv) * VD + 8 * (tid & 15)) =
                    *reinterpret_cast<const uint4*>(&s.o[r][8 * (tid & 15)]);
            break;
        }
        ck_wait(patience, &s.v_full[buf], ph);
        ck_wait(patience, &s.ks_full, uint32_t(c) & 1u);
        tc_fence_after_sync();
        {                                                    // r = beta (v - e^G S k^), times 2^e
            const float2 up = both(pow2f(e));
#pragma unroll 2
            for (int p = 0; p < TP / 4; ++p) {
                uint32_t x[8], hi[4], lo[4];
                tmem_ld_8(row + TM_X + 2 * TP * h + 8 * p, x);
                const float *c1 = &q.c1[2 * TP * h + 8 * p], *be = &q.beta[2 * TP * h + 8 * p];
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float4 cc = *reinterpret_cast<const float4*>(c1 + 2 * i), bb = *reinterpret_cast<const float4*>(be + 2 * i);
                    const float2 v0 = __fmul2_rn(v_two(vp + 1024 * p, vc, i), __fmul2_rn(up, make_float2(bb.x, bb.y)));
                    const float2 v1 = __fmul2_rn(v_two(vp + 1024 * p, vc, i + 1), __fmul2_rn(up, make_float2(bb.z, bb.w)));
                    split_h2(__ffma2_rn(make_float2(cc.x, cc.y), f2_of(x[2 * i], x[2 * i + 1]), v0), hi[i], lo[i]);
                    split_h2(__ffma2_rn(make_float2(cc.z, cc.w), f2_of(x[2 * i + 2], x[2 * i + 3]), v1), hi[i + 1], lo[i + 1]);
                }
                tmem_st_4(row + TM_PHI + TP * h + 4 * p, hi);
                tmem_st_4(row + TM_PLO + TP * h + 4 * p, lo);
            }
            ck_ready(&s.r_ready, lane);
        }
        ck_wait(patience, &s.qs_full, uint32_t(c) & 1u);
        tc_fence_after_sync();
#pragma unroll 2
        for (int p = 0; p < TP / 4; ++p) {                   // e^G S q^, for A u to be added to
            uint32_t x[8];
            tmem_ld_8(row + TM_XQ + 2 * TP * h + 8 * p, x);
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const float4 cc = *reinterpret_cast<const float4*>(&q.c2[2 * TP * h + 8 * p + 2 * i]);
                const float2 a = __fmul2_rn(f2_of(x[2 * i], x[2 * i + 1]), make_float2(cc.x, cc.y));
                const float2 b = __fmul2_rn(f2_of(x[2 * i + 2], x[2 * i + 3]), make_float2(cc.z, cc.w));
                x[2 * i] = __float_as_uint(a.x);
                x[2 * i + 1] = __float_as_uint(a.y);
                x[2 * i + 2] = __float_as_uint(b.x);
                x[2 * i + 3] = __float_as_uint(b.y);
            }
            tmem_st_8(row + slo + 2 * TP * h + 8 * p, x);
        }
        decay = q.decay;
        plen = q.len;
        if (__builtin_expect(s.vfrom[tid] != CT, 0)) {
            plen = min(int(s.vfrom[tid]), plen >> 8 & 255) << 8 | (plen & ~0xff00);
            s.vfrom[tid] = CT;
        }
        if ((plen >> 8 & 255) != CT) decay = __int_as_float(0x7fffffff);
        of = P.scale * pow2f(-e) * MAT_DOWN;
        ck_wait(patience, &s.y_full, uint32_t(c) & 1u);
        tc_fence_after_sync();
#pragma unroll 2
        for (int p = 0; p < TP / 4; ++p) {                   // the pieces of u for A u, and of u e^{G_C - G} kr for the state
            uint32_t y[8], uhi[4], ulo[4], hi[4], lo[4];
            tmem_ld_8(row + tmy + 2 * TP * h + 8 * p, y);
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const float4 cc = *reinterpret_cast<const float4*>(&q.c3[2 * TP * h + 8 * p + 2 * i]);
                const float2 u0 = f2_of(y[2 * i], y[2 * i + 1]), u1 = f2_of(y[2 * i + 2], y[2 * i + 3]);
                split_h2(__fmul2_rn(u0, both(MAT_DOWN)), uhi[i], ulo[i]);
                split_h2(__fmul2_rn(u1, both(MAT_DOWN)), uhi[i + 1], ulo[i + 1]);
                split_h2(__fmul2_rn(u0, make_float2(cc.x, cc.y)), hi[i], lo[i]);
                split_h2(__fmul2_rn(u1, make_float2(cc.z, cc.w)), hi[i + 1], lo[i + 1]);
            }
            tmem_st_4(row + TM_UHI + TP * h + 4 * p, uhi);
            tmem_st_4(row + TM_ULO + TP * h + 4 * p, ulo);
            tmem_st_4(row + TM_PHI + TP * h + 4 * p, hi);
            tmem_st_4(row + TM_PLO + TP * h + 4 * p, lo);
        }
        ck_ready(&s.u_ready, lane);
    }
    if (!Sout) return;
    const float2 down = both(pow2f(-e));
#pragma unroll
    for (int i = 0; i < SP / 2; ++i) {
        const float2 a = __fmul2_rn(S[2 * i], down), b = __fmul2_rn(S[2 * i + 1], down);
        *reinterpret_cast<float4*>(Sout + at + 4 * i) = make_float4(a.x, a.y, b.x, b.y);
    }
}

// The tensor-core instructions of the main chain, and the bulk stores of the outputs, by a warp of their own: whoever issues waits while
// the tensor cores are busy.
__device__ __forceinline__ void ck_issue(ChunkSmem& s, const CUtensorMap* rows, const CUtensorMap* outs, int xv, int hv, int t0, int nchunk, bool outputs, uint32_t tm,
                                         int& patience) {
    const uint32_t el = elect_one();
    if (el) ck_fetch_v(s, rows, xv, t0, &s.v_full[0]);
    __syncwarp();
#pragma unroll 1
    for (int c = 0; c < nchunk; ++c) {
        const int buf = c & 1;
        const uint32_t ph = uint32_t(c >> 1) & 1u, pc = uint32_t(c) & 1u, slo = tm + tm_slo(buf), tmy = tm + tm_slo(buf ^ 1);
        const uint64_t kq = ck_desc(smem_u32(s.tile[buf]), 16), kt = ck_desc(smem_u32(s.tile[buf]), 16384);
        ck_wait(patience, &s.tile_full[buf], ph);
        ck_wait(patience, &s.s_ready, pc);
        tc_fence_after_sync();
#pragma unroll 2
        for (int ks = 0; ks < 8; ++ks) {                     // S k^T
            const uint64_t d = kq + uint64_t(((ks >> 2) * 16384 + (ks & 3) * 32) >> 4);
            umma_f16_ts(el, tm + TM_X, tm + TM_SHI + 8 * ks, d, ck_idesc(64, false), ks > 0);
            umma_f16_ts(el, tm + TM_X, slo + 8 * ks, d, ck_idesc(64, false), 1u);
        }
        umma_commit_if(el, &s.ks_full);
#pragma unroll 2
        for (int ks = 0; ks < 8; ++ks) {                     // S q^T
            const uint64_t d = kq + uint64_t(((ks >> 2) * 16384 + 8192 + (ks & 3) * 32) >> 4);
            umma_f16_ts(el, tm + TM_XQ, tm + TM_SHI + 8 * ks, d, ck_idesc(64, false), ks > 0);
            umma_f16_ts(el, tm + TM_XQ, slo + 8 * ks, d, ck_idesc(64, false), 1u);
        }
        umma_commit_if(el, &s.qs_full);
        ck_wait(patience, &s.ta_full[buf], ph);
        ck_wait(patience, &s.r_ready, pc);
        tc_fence_after_sync();
        const uint64_t th = ck_desc(smem_u32(s.thi), 16), tl = ck_desc(smem_u32(s.tlo), 16);
#pragma unroll 2
        for (int ks = 0; ks < 4; ++ks) {                     // u = T r
            umma_f16_ts(el, tmy, tm + TM_PHI + 8 * ks, th + 2 * ks, ck_idesc(64, false), ks > 0);
            umma_f16_ts(el, tmy, tm + TM_PHI + 8 * ks, tl + 2 * ks, ck_idesc(64, false), 1u);
            umma_f16_ts(el, tmy, tm + TM_PLO + 8 * ks, th + 2 * ks, ck_idesc(64, false), 1u);
        }
        umma_commit_if(el, &s.y_full);
        if (el && c + 1 < nchunk) ck_fetch_v(s, rows, xv, t0 + (c + 1) * CT, &s.v_full[buf ^ 1]);        // (r is there: v has been read)
        if (el && c + 2 < nchunk) {                          // the buffer allows no earlier copy, but what it will copy can be in L2
            tma_prefetch_2d(rows, xv, t0 + (c + 2) * CT);
            tma_prefetch_2d(rows, xv + 64, t0 + (c + 2) * CT);
        }
        if (el && c > 0 && outputs) tma_store_2d(outs, s.o, hv * VD, t0 + (c - 1) * CT);      // outputs of the chunk before, a full one
        __syncwarp();
        ck_wait(patience, &s.u_ready, pc);
        tc_fence_after_sync();
#pragma unroll 2
        for (int ks = 0; ks < 4; ++ks) {                     // the chunk's part of the state, which the next one waits for
            umma_f16_ts(el, tm + TM_D, tm + TM_PHI + 8 * ks, kt + 128 * ks, ck_idesc(128, true), ks > 0);
            umma_f16_ts(el, tm + TM_D, tm + TM_PLO + 8 * ks, kt + 128 * ks, ck_idesc(128, true), 1u);
        }
        umma_commit_if(el, &s.d_full);
        const uint32_t ah = smem_u32(s.ahi[buf]), al = smem_u32(s.alo[buf]);
#pragma unroll 2
        for (int ks = 0; ks < 4; ++ks) {                     // A u; the values of tokens 32 .. reach the outputs of tokens 32 .. alone
            const uint32_t at = ks < 2 ? 2048u * ks : 4096u + 1024u * (ks - 2), step = ks < 2 ? 1024u : 512u, to = ks < 2 ? slo : slo + 32u;
            const uint32_t shape = ck_idesc(ks < 2 ? 64 : 32, false);
            umma_f16_ts(el, to, tm + TM_UHI + 8 * ks, ck_desc_cores(ah + at, step), shape, 1u);
            umma_f16_ts(el, to, tm + TM_UHI + 8 * ks, ck_desc_cores(al + at, step), shape, 1u);
            umma_f16_ts(el, to, tm + TM_ULO + 8 * ks, ck_desc_cores(ah + at, step), shape, 1u);
        }
        if (el) bulk_wait_read();                            // au_full says that the outputs' buffer is free, too
        __syncwarp();
        umma_commit_if(el, &s.au_full[buf]);
    }
    umma_commit_if(el, &s.fin);
    if (el) bulk_wait_all();
    __syncwarp();
}

// Sequence of rank r among those that are not left to the recurrence, the longest first (by their order in batches of more than RANKED, where
// ranking would take longer than it saves); -1 if there are not that many.
__device__ __forceinline__ int ck_sequence(ChunkSmem& s, const RuleParams& P, int r, int tid) {
    int64_t t0, len;
    if (tid == 0) s.seq = -1;
    if (P.N <= RANKED) {
        if (tid < P.N) {
            rule_span(P, tid, t0, len);
            s.len[tid] = int(len);
        }
        __syncthreads();
        if (tid < P.N && s.len[tid] >= P.shorter) {
            const int mine = s.len[tid];
            int rank = 0;
            for (int m = 0; m < P.N; ++m) rank += s.len[m] > mine || (s.len[m] == mine && m < tid);
            if (rank == r) s.seq = tid;
        }
    } else {                                                 // every warp counts in a part of its own, and the one that has the r-th looks for it
        const int lane = tid & 31, warp = tid >> 5, per = (P.N / (CK_THREADS / 32) + 32) & ~31, lo = warp * per, hi = P.N - lo < per ? P.N : lo + per;
        int count = 0;
#pragma unroll 4
        for (int m = lo + lane; m < hi; m += 32) {
            rule_span(P, m, t0, len);
            count += len >= P.shorter;
        }
        count = __reduce_add_sync(0xffffffffu, count);
        if (lane == 0) s.len[warp] = count;
        __syncthreads();
        for (int w = 0; w < warp; ++w) r -= s.len[w];
        if (r >= 0 && r < count) {
#pragma unroll 1
            for (int base = lo; r >= 0; base += 32) {
                bool in = false;
                if (base + lane < hi) {
                    rule_span(P, base + lane, t0, len);
                    in = len >= P.shorter;
                }
                const unsigned got = __ballot_sync(0xffffffffu, in);
                if (in && __popc(got & ((1u << lane) - 1)) == r) s.seq = base + lane;
                r -= __popc(got);
            }
        }
    }
    __syncthreads();
    return s.seq;
}

// Where there are fewer heads than SMs, a long sequence is split into segments.  The rule is linear in the state, S -> S M + B over a
// segment, and its M is the rule's own result from the unit matrix without values, its B that from zero:
//     pass 1   segment 0 as it is; of every other but the last, M and B
//     join     the state S_i that segment i starts from, S_{i+1} = S_i M_i + B_i
//     pass 2   the segments 1 .. from their states
// Every segment but the first and the last is run three times, but the chain is two segments long, with 30 us for two more launches and
// 2.5 us a join.  One sequence, whole -> in segments:
//     8 192 tokens  32 heads 600 -> 447 us (3 segments), 16 heads 262 (6), 8 heads 173 (10), 4 heads 140 (16)
//     2 048 tokens  32 heads 160 -> 148 us,              16 heads 108,     8 heads 84,       4 heads 81
struct Segments {
    float* work;                                             // of this sequence and head
    int64_t tokens;                                          // of a segment but the last: whole chunks
    int count;
    __device__ __forceinline__ float* start(int i) const { return work + int64_t(i - 1) * (VD * KD); }              // S_i; B_{i-1} until the join
    __device__ __forceinline__ float* map(int segs, int i) const { return work + int64_t(segs - 1 + i - 1) * (VD * KD); }     // M_i
};
__device__ __forceinline__ Segments rule_segments(const RuleParams& P, int n, int hv, int64_t len) {
    Segments g;
    g.work = P.work + (int64_t(n) * P.HV + hv) * (2 * P.segs - 3) * (VD * KD);
    const int64_t chunks = (len + CT - 1) / CT;
    g.tokens = (chunks + P.segs - 1) / P.segs * CT;
    g.count = int((len + g.tokens - 1) / g.tokens);
    return g;
}
// Four rows of a head's states, through all its segments.  Half of the threads of a column take half of the sum, so that a thread can have
// its part of M in flight at once: 64 KB of M from L2 and their latency is what a step takes.
constexpr int JOIN_ROWS = 4;
__global__ void __launch_bounds__(2 * KD) rule_join_kernel(RuleParams P) {
    __shared__ alignas(16) float rows[JOIN_ROWS][KD], part[JOIN_ROWS][KD];
    pdl_trigger();
    pdl_wait();
    constexpr int PARTS = VD / JOIN_ROWS, HALF = KD / 2;
    const int prog = blockIdx.x / PARTS, n = prog / P.HV, hv = prog % P.HV, k = threadIdx.x & (KD - 1), h = threadIdx.x / KD;
    int64_t t0, len;
    rule_span(P, n, t0, len);
    const int slot = P.idx[n];
    if (len < P.shorter || slot <= 0 || slot >= P.NS || !first_of_slot(P.idx, n, slot, k & 31)) return;
    const Segments g = rule_segments(P, n, hv, len);
    const int at = (blockIdx.x % PARTS) * JOIN_ROWS * KD + k;
    if (g.count > 2 && h == 0) {
#pragma unroll
        for (int r = 0; r < JOIN_ROWS; ++r) rows[r][k] = g.start(1)[at + r * KD];
    }
#pragma unroll 1
    for (int i = 1; i <= g.count - 2; ++i) {
        const float* m = g.map(P.segs, i) + h * HALF * KD + k;
        float* next = g.start(i + 1) + at;
        float x[HALF], acc[JOIN_ROWS];
#pragma unroll
        for (int j = 0; j < HALF; ++j) x[j] = m[j * KD];
#pragma unroll
        for (int r = 0; r < JOIN_ROWS; ++r) acc[r] = h ? 0.f : next[r * KD];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < HALF; j += 4)
#pragma unroll
            for (int r = 0; r < JOIN_ROWS; ++r) {
                const float4 s = *reinterpret_cast<const float4*>(&rows[r][h * HALF + j]);
                acc[r] = fmaf(s.w, x[j + 3], fmaf(s.z, x[j + 2], fmaf(s.y, x[j + 1], fmaf(s.x, x[j], acc[r]))));
            }
        if (h) {
#pragma unroll
            for (int r = 0; r < JOIN_ROWS; ++r) part[r][k] = acc[r];
        }
        __syncthreads();
        if (!h) {
#pragma unroll
            for (int r = 0; r < JOIN_ROWS; ++r) {
                acc[r] += part[r][k];
                rows[r][k] = acc[r];
                next[r * KD] = acc[r];
            }
        }
    }
}

__global__ void __launch_bounds__(CK_THREADS, 1) rule_chunk_kernel(RuleParams P, const __grid_constant__ CUtensorMap rows,
                                                                   const __grid_constant__ CUtensorMap outs) {
    extern __shared__ __align__(128) unsigned char rule_smem[];
    ChunkSmem& s = *reinterpret_cast<ChunkSmem*>(rule_smem + ((1024u - (smem_u32(rule_smem) & 1023u)) & 1023u));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_trigger();
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s.raw_full[i], 1);
            mbar_init(&s.v_full[i], 1);
            mbar_init(&s.v_ready[i], 1);
            mbar_init(&s.tile_full[i], 2);
            mbar_init(&s.ta_full[i], 1);
            mbar_init(&s.main_done[i], CK_MAIN / 32);
            mbar_init(&s.au_full[i], 1);
            mbar_init(&s.g_full[i], 1);
        }
        mbar_init(&s.ks_full, 1);
        mbar_init(&s.qs_full, 1);
        mbar_init(&s.y_full, 1);
        mbar_init(&s.d_full, 1);
        mbar_init(&s.s_ready, CK_MAIN / 32);
        mbar_init(&s.r_ready, CK_MAIN / 32);
        mbar_init(&s.u_ready, CK_MAIN / 32);
        mbar_init(&s.fin, 3);
        s.dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    int n, hv, role = 0;
    if (P.segs == 0) {
        n = ck_sequence(s, P, int(blockIdx.x) / P.HV, tid);
        hv = int(blockIdx.x) % P.HV;
        if (n < 0) return;
    } else {
        const int roles = P.pass == 1 ? 2 * P.segs - 3 : P.segs - 1, prog = int(blockIdx.x) / roles;
        role = int(blockIdx.x) % roles;
        n = prog / P.HV;
        hv = prog % P.HV;
    }
    const int hk = hv / (P.HV / P.H);
    int64_t t0, len;
    rule_span(P, n, t0, len);
    if (P.segs && len < P.shorter) return;
    const int slot = P.idx[n];
    if (slot <= 0 || slot >= P.NS || !first_of_slot(P.idx, n, slot, lane)) {       // padding: zeros, and no state
        if (P.pass == 2 || role > 0) return;
#pragma unroll 1
        for (int64_t i = tid; i < len * (VD / 8); i += CK_THREADS)
            *reinterpret_cast<uint4*>(P.o + ((t0 + i / (VD / 8)) * P.HV + hv) * VD + 8 * (i % (VD / 8))) = make_uint4(0u, 0u, 0u, 0u);
        return;
    }
    // what it starts from and where it leaves the state
    float* const state = P.ssm + int64_t(slot) * P.SS + int64_t(hv) * VD * KD;
    const float* from = !P.has_initial || P.has_initial[n] ? state : nullptr;
    float* to = state;
    bool unit = false, outputs = true;
    if (P.segs) {
        const Segments g = rule_segments(P, n, hv, len);
        int seg = 0;
        if (P.pass == 1) {
            if (role > 0) {
                seg = (role + 1) / 2;
                if (seg > g.count - 2) return;
                unit = !(role & 1);
                outputs = false;
                from = nullptr;
                to = unit ? g.map(P.segs, seg) : g.start(seg + 1);
            } else if (g.count > 1) to = g.start(1);
        } else {
            seg = role + 1;
            if (seg >= g.count) return;
            from = g.start(seg);
            if (seg < g.count - 1) to = nullptr;
        }
        t0 += seg * g.tokens;
        len = len - seg * g.tokens < g.tokens ? len - seg * g.tokens : g.tokens;
    }
#pragma unroll 1
    for (int i = tid; i < 2 * 8192 / 16; i += CK_THREADS) reinterpret_cast<uint4*>(s.thi)[i] = make_uint4(0u, 0u, 0u, 0u);   // the upper right
                                                                                    // blocks of T (head, remainder) stay zero
#pragma unroll 1
    for (int i = tid; i < 2 * 2 * 32 * 36; i += CK_THREADS) (&s.prep[i / (2 * 32 * 36)].tt[0][0][0])[i % (2 * 32 * 36)] = 0.f;
    if (tid < CK_MAIN) s.vfrom[tid] = CT;
    if (tid < ODD_RING) {
        s.odd[tid].from = CT;
        s.odd[tid].q[0] = s.odd[tid].q[1] = 0;
    }
    if (warp == 0) tmem_alloc(&s.tm, 512);
    fence_async_smem();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tm = s.tm;
    const int nchunk = int((len + CT - 1) / CT);
    const int uw = __shfl_sync(0xffffffffu, warp, 0);        // the warp's number, known to be the same in all lanes
    int patience = WAIT_LIMIT;
    if (uw == CK_THREADS / 32 - 1) {
        ck_issue(s, &rows, &outs, 2 * P.H * KD + hv * VD, hv, int(t0), nchunk, outputs, tm, patience);
    } else if (uw >= CK_MAIN / 32) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CK_PREP_REGS));
        ck_prep(s, P, &rows, hk, hv, t0, len, unit ? 0 : len, nchunk, tm, (uw - CK_MAIN / 32) >> 2, uw & 3, lane, patience);
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(CK_MAIN_REGS));
        ck_main(s, P, hv, t0, nchunk, from, unit, to, outputs, tm, tid, patience);
    }
    ck_wait(patience, &s.fin, 0);                            // no tensor-core instruction is left
    if (patience == 0) s.dead = 1;
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tm, 512);
    if (tid == 0 && s.dead) atomicOr(&g_status, ST_CONSUMER_TIMEOUT);
}

static int rule_check(const lq_dims* d, const RuleParams& P) {
    if (d->K != KD || d->V != VD) return LQ_ERR_UNSUPPORTED;
    if (d->NS < 1 || d->HV < 1 || d->H < 1 || d->HV % d->H != 0 || d->SS < int64_t(d->HV) * d->V * d->K) return LQ_ERR_RANGE;
    if (d->SS & 3) return LQ_ERR_ALIGN;
    if (P.N < 0 || P.T < 0 || P.T > 0x7fffffff) return LQ_ERR_RANGE;              // (offsets and coordinates of the tensor maps: 32 bits)
    if (P.N == 0 || P.T == 0) return LQ_OK;
    if (!P.ssm || !P.mixed || !P.a || !P.b || !P.A_log || !P.dt_bias || !P.idx || !P.o) return LQ_ERR_NULL;
    if (P.mixed_stride < 2 * int64_t(d->H) * KD + int64_t(d->HV) * VD || P.a_stride < d->HV || P.b_stride < d->HV) return LQ_ERR_RANGE;
    if ((P.mixed_stride & 7) || misaligned16({P.ssm, P.mixed, P.o})) return LQ_ERR_ALIGN;
    if (int64_t(P.N) * d->HV > (int64_t(1) << 29)) return LQ_ERR_RANGE;            // programs: the grid's first dimension
    const int64_t ow = int64_t(d->HV) * VD;                  // (the outputs of a head are written while another's rows are still read)
    if (rows_overlap(P.o, ow, ow, P.mixed, P.mixed_stride, 2 * int64_t(d->H) * KD + ow, P.T) ||
        rows_overlap(P.o, ow, ow, P.a, P.a_stride, d->HV, P.T) || rows_overlap(P.o, ow, ow, P.b, P.b_stride, d->HV, P.T))
        return LQ_ERR_RANGE;
    return LQ_OK;
}
static int launch_recurrent(const RuleParams& P, cudaStream_t st) {
    const unsigned grid = unsigned(P.N) * unsigned(P.HV) * (VD / (RW_ROWS * RW_WARPS));
    const cudaError_t e = launch_dependent(rule_recurrent_kernel, grid, 32 * RW_WARPS, 0, st, P);
    if (e != cudaSuccess) { set_last_cuda_error(e); return LQ_ERR_LAUNCH; }
    return finish_launch();
}
// Tensor map of a bf16 matrix [rows][cols] for boxes of 64 rows.
static int encode_rows(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t stride, uint32_t box, CUtensorMapSwizzle swizzle) {
    using Encode = decltype(&cuTensorMapEncodeTiled);
    static const Encode encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<Encode>(f);
    }();
    if (!encode) return LQ_ERR_LAUNCH;
    const cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)}, strides[1] = {cuuint64_t(stride) * 2};
    const cuuint32_t boxes[2] = {box, CT}, ones[2] = {1, 1};
    const CUresult e = encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return e == CUDA_SUCCESS ? LQ_OK : LQ_ERR_LAUNCH;
}
static int launch_chunk(const RuleParams& P, cudaStream_t st) {
    constexpr size_t smem = sizeof(ChunkSmem) + 1024;
    static_assert(smem <= 227 * 1024, "the working set of a CTA");
    CUtensorMap rows, outs;
    int rc = encode_rows(&rows, P.mixed, P.T, 2 * int64_t(P.H) * KD + int64_t(P.HV) * VD, P.mixed_stride, 64, CU_TENSOR_MAP_SWIZZLE_128B);
    if (!rc) rc = encode_rows(&outs, P.o, P.T, int64_t(P.HV) * VD, int64_t(P.HV) * VD, VD, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (!rc) rc = ensure_smem((const void*)rule_chunk_kernel, smem);
    static const int regs = [] {
        cudaFuncAttributes at;
        return cudaFuncGetAttributes(&at, rule_chunk_kernel) == cudaSuccess ? at.numRegs : 0;
    }();
    if (!rc && regs != CK_REGS) return LQ_ERR_LAUNCH;        // the register split of the warps would not add up
    if (rc) return rc;
    // no more than T / P.shorter sequences can be that long
    const int64_t most = P.T / P.shorter < P.N ? P.T / P.shorter : P.N;
    const unsigned heads = unsigned(P.segs ? P.N : most) * unsigned(P.HV);
    RuleParams Q = P;
    Q.pass = 1;
    cudaError_t e = launch_dependent(rule_chunk_kernel, heads * unsigned(P.segs ? 2 * P.segs - 3 : 1), CK_THREADS, smem, st, Q, rows, outs);
    if (e == cudaSuccess && P.segs) {
        e = launch_dependent(rule_join_kernel, heads * (VD / JOIN_ROWS), 2 * KD, 0, st, Q);
        Q.pass = 2;
        if (e == cudaSuccess) e = launch_dependent(rule_chunk_kernel, heads * unsigned(P.segs - 1), CK_THREADS, smem, st, Q, rows, outs);
    }
    if (e != cudaSuccess) { set_last_cuda_error(e); return LQ_ERR_LAUNCH; }
    return finish_launch();
}
// Segments that sequences are split into, 0 if that would not be faster: both passes have to fit the SMs at once, and a sequence of mean
// length has to save more by its shorter chain (4.7 us a chunk) than the launches and the joins cost.  (At the least 16 chunks in four segments
// of four.)
static int rule_segs(int64_t N, int64_t HV, int64_t T) {
    const int64_t chunks = T / N / CT, fit = (device_sm_count() / (N * HV) + 3) / 2;
    int64_t segs = fit < 16 ? fit : 16;
    if (segs > chunks / 4) segs = chunks / 4;
    return segs >= 3 && chunks * (segs - 2) >= 8 * segs ? int(segs) : 0;
}
static int64_t rule_work(int64_t N, int64_t HV, int segs) { return segs ? N * HV * (2 * segs - 3) * VD * KD * 4 : 0; }

static RuleParams rule_params(const lq_dims* d, float* ssm, const void* mixed, int64_t mixed_stride, const void* a, int64_t a_stride,
                              const void* b, int64_t b_stride, const float* A_log, const float* dt_bias, const int32_t* cu,
                              const int32_t* idx, const uint8_t* has_initial, void* o, int32_t N, int64_t T, float scale) {
    RuleParams P;
    P.ssm = ssm; P.SS = d->SS; P.mixed = (const uint16_t*)mixed; P.mixed_stride = mixed_stride; P.a = (const uint16_t*)a;
    P.b = (const uint16_t*)b; P.a_stride = a_stride; P.b_stride = b_stride; P.A_log = A_log; P.dt_bias = dt_bias; P.cu = cu;
    P.idx = idx; P.has_initial = has_initial; P.o = (uint16_t*)o; P.NS = d->NS; P.H = d->H; P.HV = d->HV; P.N = N; P.T = T;
    P.shorter = T + 1;
    P.work = nullptr;
    P.segs = 0;
    P.pass = 1;
    P.scale = scale > 0.f ? scale : 1.0f / sqrtf(float(KD));
    return P;
}

}  // namespace lq

extern "C" int lq_gdn_prefill_check(const lq_dims* d, const float* ssm, const void* mixed, int64_t mixed_stride, const void* a, int64_t a_stride,
                                    const void* b, int64_t b_stride, const float* A_log, const float* dt_bias, const int32_t* cu,
                                    const int32_t* idx, const void* o, int32_t N, int64_t T) {
    using namespace lq;
    if (!d) return LQ_ERR_NULL;
    if (N > 0 && T > 0 && !cu) return LQ_ERR_NULL;
    return rule_check(d, rule_params(d, const_cast<float*>(ssm), mixed, mixed_stride, a, a_stride, b, b_stride, A_log, dt_bias, cu, idx, nullptr,
                                     const_cast<void*>(o), N, T, 1.f));
}

extern "C" int lq_gdn_prefill(const lq_dims* d, float* ssm, const void* mixed, int64_t mixed_stride, const void* a, int64_t a_stride,
                              const void* b, int64_t b_stride, const float* A_log, const float* dt_bias, const int32_t* cu,
                              const int32_t* idx, const uint8_t* has_initial, void* o, int32_t N, int64_t T, float scale,
                              void* work, int64_t work_bytes, void* stream) {
    using namespace lq;
    const int rc = lq_gdn_prefill_check(d, ssm, mixed, mixed_stride, a, a_stride, b, b_stride, A_log, dt_bias, cu, idx, o, N, T);
    if (rc) return rc;
    if (misaligned16({work})) return LQ_ERR_ALIGN;
    if (N == 0 || T == 0) return LQ_OK;
    RuleParams P = rule_params(d, ssm, mixed, mixed_stride, a, a_stride, b, b_stride, A_log, dt_bias, cu, idx, has_initial, o, N,
                                     T, scale);
    // The lengths are on the device: a batch gets both kernels, and each of its sequences is run by one of them.
    const int impl = g_rule_impl.load(std::memory_order_relaxed);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    P.shorter = impl == 1 ? T + 1 : impl == 2 ? 1 : T / N >= 256 && int64_t(N) * d->HV <= 3 * device_sm_count() ? RULE_SHORT_AMONG_LONG : RULE_SHORT;
    if (T < P.shorter) return launch_recurrent(P, st);
    if (N == 1) P.shorter = 1;                               // one kernel for one sequence
    if (P.shorter > 1) {
        const int rc2 = launch_recurrent(P, st);
        if (rc2) return rc2;
    }
    const int segs = rule_segs(N, d->HV, T);
    if (work && segs && work_bytes >= rule_work(N, d->HV, segs)) {
        P.work = static_cast<float*>(work);
        P.segs = segs;
    }
    return launch_chunk(P, st);
}

extern "C" int64_t lq_prefill_work_bytes(int32_t N, int32_t HV, int64_t T) {
    using namespace lq;
    return N < 1 || HV < 1 || T < 1 ? 0 : rule_work(N, HV, rule_segs(N, HV, T));
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
