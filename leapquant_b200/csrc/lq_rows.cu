// Row operators around the gated delta rule (sm_100a): the causal conv1d of whole prompts in front of it, the gated RMS norm of its
// output behind it, and the residual + RMS norm between the blocks.  All of them read and write every element once.
#include "lq_common.cuh"

namespace lq {

__device__ __forceinline__ void unpack8(const uint4& w, float (&f)[8]) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = bf16lo(x[i]);
        f[2 * i + 1] = bf16hi(x[i]);
    }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(f2_to_bf16x2(f[0], f[1]), f2_to_bf16x2(f[2], f[3]), f2_to_bf16x2(f[4], f[5]), f2_to_bf16x2(f[6], f[7]));
}
// (not the read-only path: an output may be written over its input)
__device__ __forceinline__ uint4 ld_once(const void* p) { return __ldcs(reinterpret_cast<const uint4*>(p)); }
// x / (1 + e^-x) on the special function unit: relative errors of 2^-21 for |x| below 8 and 2^-24 |x| beyond, where bf16 keeps 2^-9.  (With
// expf and a true division these kernels are bound by their arithmetic: 32 768 rows of 8 192 channels 400 us, of 32 heads 188 us.)
__device__ __forceinline__ float silu(float x) { return __fdividef(x, 1.0f + __expf(-x)); }

// ---- causal conv1d over prompts -------------------------------------------------------------------------------------------
// A thread takes four channels of up to CP_TOKENS consecutive tokens of ONE sequence and keeps the three inputs before the current
// one in registers.  Piece j of sequence n is block cu[n] / CP_TOKENS + n + j of the grid: these ranges do not overlap, since a
// sequence of len tokens has at most len / CP_TOKENS + 1 whole steps of the first term, and a block finds its sequence by a search in
// cu.  The piece that holds a sequence's first token is the only reader of its conv state and writes the new one, from the last three
// inputs, when it has read the old one: no two blocks touch a slot.
// Memory bound, but not by far: two special functions per element alone take three quarters of the copy's time, so the kernel lives on warps
// that overlap (32 an SM at 64 registers).  32 768 rows of 8 192 channels: 214 us, 77 % of the measured copy rate (205 on one input again and
// again: what of it is still in L2); against those 205, eight channels a thread with half the warps 238, four rows a batch (the past inputs
// have to be moved around) 229, pieces of 48 tokens 201 but twice the latency.
constexpr int CP_TOKENS = 24, CP_BATCH = 6, CP_THREADS = 128;
struct ConvPromptParams {
    const uint16_t* x;
    int64_t x_stride;
    uint16_t* state;
    int64_t ss, sd, sp;                // strides of the state: slot, channel, tap
    const uint16_t *w, *bias;
    const int32_t *cu, *idx;
    const uint8_t* has_initial;
    uint16_t* out;
    int64_t out_stride;
    int32_t N, C, NS;
    int64_t T;
};
__device__ __forceinline__ int64_t cp_first(const ConvPromptParams& P, int n) {
    const int64_t s = P.cu[n];
    return s < 0 ? 0 : s > P.T ? P.T : s;
}
// the largest n with cu[n] / CP_TOKENS + n <= block, by a search of 32 places at a time (the whole warp calls)
__device__ __forceinline__ int cp_sequence(const ConvPromptParams& P, int64_t block, int lane) {
    int lo = 0, hi = P.N - 1;                                // the answer lies in [lo, hi]
    while (lo < hi) {
        const int step = (hi - lo + 32) / 32, n = lo + 1 + lane * step;
        const bool ok = n <= hi && cp_first(P, n) / CP_TOKENS + n <= block;
        const int got = __popc(__ballot_sync(0xffffffffu, ok));
        if (got == 0) hi = lo;
        else {
            lo = lo + 1 + (got - 1) * step;
            hi = min(hi, lo + step - 1);
        }
    }
    return lo;
}
__device__ __forceinline__ void unpack4(const uint2& w, float (&f)[4]) {
    f[0] = bf16lo(w.x);
    f[1] = bf16hi(w.x);
    f[2] = bf16lo(w.y);
    f[3] = bf16hi(w.y);
}
__device__ __forceinline__ uint2 pack4bf(const float (&f)[4]) { return make_uint2(f2_to_bf16x2(f[0], f[1]), f2_to_bf16x2(f[2], f[3])); }
__device__ __forceinline__ uint2 ldg2(const uint16_t* p) { return __ldcs(reinterpret_cast<const uint2*>(p)); }
__global__ void __launch_bounds__(CP_THREADS, 8) conv1d_prompt_kernel(ConvPromptParams P) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, n = cp_sequence(P, blockIdx.x, lane);
    const int64_t s0 = cp_first(P, n);
    int64_t len = P.cu[n + 1];
    len = (len > P.T ? P.T : len) - s0;
    const int64_t piece = int64_t(blockIdx.x) - (s0 / CP_TOKENS + n);
    const int64_t p0 = piece * CP_TOKENS;                    // first place of this piece in its sequence
    const int slot = P.idx[n];
    if (piece < 0 || p0 >= len || slot <= 0 || slot >= P.NS || !first_of_slot(P.idx, n, slot, lane)) return;
    const int c0 = 4 * (blockIdx.y * CP_THREADS + threadIdx.x);
    if (c0 >= P.C) return;
    float w[4][4], bias[4] = {0.f, 0.f, 0.f, 0.f}, h[3][4];
    {
        const uint4* wp = reinterpret_cast<const uint4*>(P.w + int64_t(c0) * 4);
#pragma unroll
        for (int i = 0; i < 2; ++i) {                        // the taps of channels c0 + 2 i and c0 + 2 i + 1
            float f[8];
            unpack8(__ldg(wp + i), f);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                w[t][2 * i] = f[t];
                w[t][2 * i + 1] = f[4 + t];
            }
        }
        if (P.bias) unpack4(__ldg(reinterpret_cast<const uint2*>(P.bias + c0)), bias);
    }
    const uint16_t* x = P.x + s0 * P.x_stride + c0;
    if (piece > 0) {
#pragma unroll
        for (int j = 0; j < 3; ++j) unpack4(__ldg(reinterpret_cast<const uint2*>(x + (p0 - 3 + j) * P.x_stride)), h[j]);
    } else {
        uint16_t* st = P.state + int64_t(slot) * P.ss + int64_t(c0) * P.sd;
        const bool keep = !P.has_initial || P.has_initial[n];
        const bool vec = P.sd == 1;
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            if (!keep) {
#pragma unroll
                for (int i = 0; i < 4; ++i) h[j][i] = 0.f;
            } else if (vec) {
                unpack4(*reinterpret_cast<const uint2*>(st + j * P.sp), h[j]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) h[j][i] = bf16_to_f(st[i * P.sd + j * P.sp]);
            }
        }
        // the inputs len - 3 .. len - 1, counted through the old state where the sequence is shorter than three
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            const int64_t p = len - 3 + j;
            uint2 nw;
            if (p >= 0) nw = __ldg(reinterpret_cast<const uint2*>(x + p * P.x_stride));
            else nw = p == -1 ? pack4bf(h[2]) : p == -2 ? pack4bf(h[1]) : pack4bf(h[0]);
            if (vec) {
                *reinterpret_cast<uint2*>(st + j * P.sp) = nw;
            } else {
                const uint32_t ww[2] = {nw.x, nw.y};
#pragma unroll
                for (int i = 0; i < 4; ++i) st[i * P.sd + j * P.sp] = uint16_t(ww[i >> 1] >> (16 * (i & 1)));
            }
        }
    }
    const int m = int(len - p0 < CP_TOKENS ? len - p0 : CP_TOKENS);
    x += p0 * P.x_stride;
    uint16_t* out = P.out + (s0 + p0) * P.out_stride + c0;
    auto row = [&](const uint2& in, uint16_t* to) {
        float f[4], y[4];
        unpack4(in, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            y[e] = silu(fmaf(w[3][e], f[e], fmaf(w[2][e], h[2][e], fmaf(w[1][e], h[1][e], fmaf(w[0][e], h[0][e], bias[e])))));
            h[0][e] = h[1][e];
            h[1][e] = h[2][e];
            h[2][e] = f[e];
        }
        *reinterpret_cast<uint2*>(to) = pack4bf(y);
    };
    int i0 = 0;
#pragma unroll 1
    for (; i0 + CP_BATCH <= m; i0 += CP_BATCH) {             // six rows a time: after every third the past inputs are back in their registers
        uint2 raw[CP_BATCH];
#pragma unroll
        for (int i = 0; i < CP_BATCH; ++i) raw[i] = ldg2(x + (i0 + i) * P.x_stride);
#pragma unroll
        for (int i = 0; i < CP_BATCH; ++i) row(raw[i], out + (i0 + i) * P.out_stride);
    }
#pragma unroll 1
    for (; i0 < m; ++i0) row(ldg2(x + i0 * P.x_stride), out + i0 * P.out_stride);
}

// ---- gated RMS norm of every head's output ----------------------------------------------------------------------------------
// y = o / sqrt(mean(o^2) + eps) * w * silu(z), rows of 128: sixteen lanes share a row.  Memory bound; a thread has the loads of four rows in
// flight.  32 768 x 32 rows: 146 us, 84 % of the measured copy rate; on one input again and again 131 (one row a thread 148, two 135, six 158).
constexpr int GN_ROWS = 4;                                   // rows of a thread, sixteen apart
__global__ void __launch_bounds__(256) gated_norm_kernel(const uint16_t* o, const uint16_t* z, int64_t z_stride, const uint16_t* w,
                                                         uint16_t* y, int64_t rows, int HV, float eps) {
    pdl_trigger();
    pdl_wait();
    const int64_t first = int64_t(blockIdx.x) * (16 * GN_ROWS) + (threadIdx.x >> 4);
    const int c = 8 * (threadIdx.x & 15);
    uint4 fo[GN_ROWS], fz[GN_ROWS];
#pragma unroll
    for (int r = 0; r < GN_ROWS; ++r) {
        const int64_t row = first + 16 * r;
        if (row < rows) {                                    // (half a warp at a time: the shuffles below stay inside the half)
            const int64_t t = row / HV;
            fo[r] = ld_once(o + row * VD + c);
            fz[r] = ld_once(z + t * z_stride + (row - t * HV) * VD + c);
        }
    }
    float ww[8];
    unpack8(__ldg(reinterpret_cast<const uint4*>(w + c)), ww);
    const unsigned half = 0xffffu << (threadIdx.x & 16);
#pragma unroll
    for (int r = 0; r < GN_ROWS; ++r) {
        const int64_t row = first + 16 * r;
        if (row >= rows) break;
        float f[8], g[8], s = 0.f;
        unpack8(fo[r], f);
        unpack8(fz[r], g);
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(f[i], f[i], s);
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) s += __shfl_xor_sync(half, s, d);
        const float inv = rsqrtf(s * (1.0f / VD) + eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = f[i] * inv * ww[i] * silu(g[i]);
        *reinterpret_cast<uint4*>(y + row * VD + c) = pack8(f);
    }
}

// ---- residual + RMS norm ----------------------------------------------------------------------------------------------------
// h = r + scale x;  r <- h;  y = h / sqrt(mean(h^2) + eps) * w.  One block per row, NV vectors of eight elements per thread; the
// norm is that of the fp32 sum, not of its rounding to bf16.  Memory bound: 16 384 rows of 4 096 in 84 us, 98 % of the measured copy rate.
template <int NV>
__global__ void __launch_bounds__(1024) add_norm_kernel(const uint16_t* x, int64_t x_stride, uint16_t* r, int64_t r_stride,
                                                        const uint16_t* w, uint16_t* y, int64_t y_stride, int D, float scale, float eps) {
    pdl_trigger();
    pdl_wait();
    __shared__ float part[32];
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    x += row * x_stride;
    r += row * r_stride;
    y += row * y_stride;
    uint4 xr[NV], rr[NV];
    float h[NV][8], s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = 8 * (threadIdx.x + i * blockDim.x);
        xr[i] = rr[i] = make_uint4(0u, 0u, 0u, 0u);
        if (c < D) {
            xr[i] = ld_once(x + c);
            rr[i] = *reinterpret_cast<const uint4*>(r + c);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = 8 * (threadIdx.x + i * blockDim.x);
        float f[8];
        unpack8(xr[i], f);
        unpack8(rr[i], h[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            h[i][e] = fmaf(scale, f[e], h[i][e]);
            s = fmaf(h[i][e], h[i][e], s);
        }
        if (c < D) *reinterpret_cast<uint4*>(r + c) = pack8(h[i]);
    }
    s = warp_sum(s);
    if (lane == 0) part[warp] = s;
    __syncthreads();
    s = warp_sum(lane < nw ? part[lane] : 0.f);
    const float inv = rsqrtf(s / float(D) + eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = 8 * (threadIdx.x + i * blockDim.x);
        if (c >= D) break;
        float ww[8];
        unpack8(__ldg(reinterpret_cast<const uint4*>(w + c)), ww);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[i][e] = h[i][e] * inv * ww[e];
        *reinterpret_cast<uint4*>(y + c) = pack8(h[i]);
    }
}

}  // namespace lq

extern "C" int lq_causal_conv1d_prompt(const lq_conv1d* conv, const int32_t* cu, const int32_t* idx, const uint8_t* has_initial, int32_t N,
                                       int64_t T, int32_t channels, int32_t NS, void* out, int64_t out_stride, void* stream) {
    using namespace lq;
    if (!conv) return LQ_ERR_NULL;
    if (N < 0 || T < 0 || channels < 8 || NS < 1) return LQ_ERR_RANGE;
    if (channels & 7) return LQ_ERR_UNSUPPORTED;
    if (N == 0 || T == 0) return LQ_OK;
    if (!conv->x || !conv->state || !conv->weight || !cu || !idx || !out) return LQ_ERR_NULL;
    if (conv->width != 4) return LQ_ERR_UNSUPPORTED;
    if (conv->x_stride < channels || out_stride < channels) return LQ_ERR_RANGE;
    if ((conv->x_stride & 7) || (out_stride & 7) || misaligned16({conv->x, conv->weight, conv->bias, out})) return LQ_ERR_ALIGN;
    if (reinterpret_cast<uintptr_t>(conv->state) & 7) return LQ_ERR_ALIGN;
    if (conv->stride_dim == 1 && ((conv->stride_tap & 3) || (conv->stride_slot & 3))) return LQ_ERR_ALIGN;
    if (rows_overlap(conv->x, conv->x_stride, channels, out, out_stride, channels, T)) return LQ_ERR_RANGE;
    const int64_t blocks = T / CP_TOKENS + N + 1;
    if (blocks > 0x7fffffff || (channels + 4 * CP_THREADS - 1) / (4 * CP_THREADS) > 65535) return LQ_ERR_RANGE;
    ConvPromptParams P;
    P.x = (const uint16_t*)conv->x; P.x_stride = conv->x_stride; P.state = (uint16_t*)conv->state; P.ss = conv->stride_slot;
    P.sd = conv->stride_dim; P.sp = conv->stride_tap; P.w = (const uint16_t*)conv->weight; P.bias = (const uint16_t*)conv->bias;
    P.cu = cu; P.idx = idx; P.has_initial = has_initial; P.out = (uint16_t*)out; P.out_stride = out_stride; P.N = N; P.C = channels;
    P.NS = NS; P.T = T;
    const dim3 grid(unsigned(blocks), unsigned((channels + 4 * CP_THREADS - 1) / (4 * CP_THREADS)));
    const cudaError_t e = launch_dependent(conv1d_prompt_kernel, grid, CP_THREADS, 0, static_cast<cudaStream_t>(stream), P);
    if (e != cudaSuccess) { set_last_cuda_error(e); return LQ_ERR_LAUNCH; }
    return finish_launch();
}

extern "C" int lq_gated_norm(const void* o, const void* z, int64_t z_stride, const void* weight, void* y, int64_t T, int32_t HV, int32_t V,
                             float eps, void* stream) {
    using namespace lq;
    if (V != VD) return LQ_ERR_UNSUPPORTED;
    if (T < 0 || HV < 1) return LQ_ERR_RANGE;
    if (T == 0) return LQ_OK;
    if (!o || !z || !weight || !y) return LQ_ERR_NULL;
    if (z_stride < int64_t(HV) * V) return LQ_ERR_RANGE;
    if ((z_stride & 7) || misaligned16({o, z, weight, y})) return LQ_ERR_ALIGN;
    const int64_t width = int64_t(HV) * V;
    if ((y != o && rows_overlap(y, width, width, o, width, width, T)) || rows_overlap(y, width, width, z, z_stride, width, T)) return LQ_ERR_RANGE;
    const int64_t rows = T * HV, blocks = (rows + 16 * GN_ROWS - 1) / (16 * GN_ROWS);
    if (blocks > 0x7fffffff) return LQ_ERR_RANGE;
    const cudaError_t e = launch_dependent(gated_norm_kernel, unsigned(blocks), 256, 0, static_cast<cudaStream_t>(stream),
                                           (const uint16_t*)o, (const uint16_t*)z, z_stride, (const uint16_t*)weight, (uint16_t*)y, rows,
                                           int(HV), eps);
    if (e != cudaSuccess) { set_last_cuda_error(e); return LQ_ERR_LAUNCH; }
    return finish_launch();
}

extern "C" int lq_add_norm(const void* x, int64_t x_stride, void* residual, int64_t r_stride, const void* weight, void* y, int64_t y_stride,
                           int64_t T, int32_t D, float scale, float eps, void* stream) {
    using namespace lq;
    if (D < 8 || (D & 7) || D > LQ_NORM_MAX_DIM) return LQ_ERR_UNSUPPORTED;
    if (T < 0 || T > 0x7fffffff) return LQ_ERR_RANGE;
    if (T == 0) return LQ_OK;
    if (!x || !residual || !weight || !y) return LQ_ERR_NULL;
    if (x_stride < D || r_stride < D || y_stride < D) return LQ_ERR_RANGE;
    if (((x_stride | r_stride | y_stride) & 7) || misaligned16({x, residual, weight, y})) return LQ_ERR_ALIGN;
    const auto apart = [&](const void* a, int64_t as, const void* b, int64_t bs) { return !rows_overlap(a, as, D, b, bs, D, T); };
    if (!apart(y, y_stride, residual, r_stride) || !(apart(y, y_stride, x, x_stride) || (y == x && y_stride == x_stride)) ||
        !(apart(x, x_stride, residual, r_stride) || (x == residual && x_stride == r_stride)))
        return LQ_ERR_RANGE;
    const int vecs = D / 8;
    const int nv = vecs > 1024 ? 2 : 1;
    const unsigned threads = unsigned(((vecs + nv - 1) / nv + 31) / 32 * 32);
    const cudaError_t e = launch_dependent(nv == 1 ? add_norm_kernel<1> : add_norm_kernel<2>, unsigned(T), threads, 0,
                                           static_cast<cudaStream_t>(stream), (const uint16_t*)x, x_stride, (uint16_t*)residual, r_stride,
                                           (const uint16_t*)weight, (uint16_t*)y, y_stride, int(D), scale, eps);
    if (e != cudaSuccess) { set_last_cuda_error(e); return LQ_ERR_LAUNCH; }
    return finish_launch();
}
