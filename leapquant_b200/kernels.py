"""Kernel factories of the 8-bit recurrent state, with the names and call signatures of the reference's
leapquant/kernels.py, backed by hand-written sm_100a CUDA behind a C ABI (include/leapquant_b200.h).

  make_gdn_step    GDN decode step            (reference leapquant/kernels.py:28,   launch signature :80-89)
  make_kda_step    KDA decode step            (reference leapquant/kernels.py:695,  launch signature :732-741)
  make_flush       end-of-window flush        (reference leapquant/kernels.py:1078, launch signature :1139-1148)
  make_dequant     8-bit -> fp32 in place     (reference leapquant/kernels.py:2042, launch signature :2053-2062)
  make_quantize    fp32 -> 8-bit in place     (reference leapquant/kernels.py:2127, launch signature :2136-2142)
  make_lowrank / lowrank_factor               (reference leapquant/kernels.py:2247, :2321)

The operators around them, which the reference leaves to the engine, have no counterpart there:

  make_gdn_prefill     gated delta rule of packed sequences on fp32 states     make_gdn_recurrent   one token per row of the same
  make_conv1d_prompt   causal conv1d + SiLU of packed prompts                  make_conv1d_update   one token per row of the same
  make_gated_norm      RMS norm of every head's output, times silu(gate)       make_add_norm        residual + RMS norm

Each factory returns a callable that takes the same tensors in the same order as the reference's compiled kernel.
The several aliasing views of the state tensor the reference passes (Sq, Sk, Sv, Skv, UQ, Sq16) all point into one
fp32 tensor; the callable takes the base address from the first of them and the slot stride SS from the factory.
The reference's tuning keywords (SMS, NSTAGE, NSTAGEQ, NCG, NNW, MAXIT, NMAX, NTP, RSG, PAD, MMT, BV, threads) are
accepted and ignored: scheduling is decided inside the library.  Shapes outside K = V = 128 raise NotImplementedError.
"""
import ctypes
import functools

import torch

from . import _lib

F32, BF16, I32, I8 = "float32", "bfloat16", "int32", "int8"
QMAX = 127.0
SOFTPLUS_THRESHOLD = 20.0
EPS = 1e-12
STEP_CFG = {(128, 128): (6, 3, 2), (64, 128): (10, 5, 5), (64, 64): (8, 4, 4)}


def _need_128(K, V, who):
    if (K, V) != (128, 128):
        raise NotImplementedError(f"{who}: (K, V) = ({K}, {V}); this build implements 128 x 128 heads only")


_launch = _lib.launch


def _work(work):
    """(pointer, bytes) of the optional mailbox scratch of the fused decode (an int32 tensor, zeroed once), or (None, 0)."""
    if work is None:
        return None, 0
    return _lib.ptr(work), work.nbytes


def decode_work_ints(rows, HV):
    """int32 elements of the `work` tensor of the fused decode (mailboxes of due heads: a fixed 16 KiB, whatever the call)."""
    return int(_lib.lib().lq_decode_work_bytes(int(rows), int(HV))) // 4


def make_gdn_step(NS, HV, H, K, V, L, SS, R=4, SMS=148, NSTAGE=None, NCG=None, NNW=None, scale=None, MAXIT=256):
    """Gated DeltaNet decode step on the 8-bit state.  Returns
    step(Sq, Sk, Sv, Skv, Kbuf, Ubuf, Wbuf, Pbuf, hcnt, mixed, a, b, A_log, dt_bias, UQ, idx, o)."""
    _need_128(K, V, "make_gdn_step")
    d = _lib.dims(NS, HV, H, K, V, L, R, SS)
    sc = float(K ** -0.5 if scale is None else scale)
    fn = _lib.lib().lq_gdn_step
    p = _lib.ptr

    def step(Sq, Sk, Sv, Skv, Kbuf, Ubuf, Wbuf, Pbuf, hcnt, mixed, a, b, A_log, dt_bias, UQ, idx, o):
        _launch(fn, "lq_gdn_step", Sq, d, p(Sq), p(Kbuf), p(Ubuf), p(Wbuf), p(Pbuf), p(hcnt), p(mixed), p(a), p(b),
                p(A_log), p(dt_bias), p(idx), p(o), int(mixed.shape[0]), sc)

    return step


def make_kda_step(NS, HV, H, K, V, L, SS, R=4, SMS=148, NSTAGE=6, NSTAGEQ=4, NCG=2, NNW=2, scale=128 ** -0.5, MAXIT=256,
                  GLB=0.0):
    """Kimi Delta Attention decode step (gate per key channel).  GLB != 0 selects the bounded gate.  Returns
    step(Sq, Sk, Sv, Skv, Kbuf, Ubuf, Wbuf, Pbuf, Gbuf, hcnt, mixed, a, b, A_log, dt_bias, UQ, idx, o)."""
    _need_128(K, V, "make_kda_step")
    d = _lib.dims(NS, HV, H, K, V, L, R, SS)
    sc, glb = float(scale), float(GLB)
    fn = _lib.lib().lq_kda_step
    p = _lib.ptr

    def step(Sq, Sk, Sv, Skv, Kbuf, Ubuf, Wbuf, Pbuf, Gbuf, hcnt, mixed, a, b, A_log, dt_bias, UQ, idx, o):
        _launch(fn, "lq_kda_step", Sq, d, p(Sq), p(Kbuf), p(Ubuf), p(Wbuf), p(Pbuf), p(Gbuf), p(hcnt), p(mixed), p(a),
                p(b), p(A_log), p(dt_bias), p(idx), p(o), int(mixed.shape[0]), sc, glb)

    return step


def make_decode(NS, HV, H, K, V, L, SS, R=4, ITERS=1, KDA=False, GLB=0.0, scale=None):
    """Step and flush in one launch (no counterpart factory in the reference, whose LeapQuantState.decode launches the two
    kernels one after the other, leapquant/state.py:99-116).  Returns, for GDN,
    decode(Sq, Kbuf, Ubuf, Wbuf, Pbuf, hcnt, mixed, a, b, A_log, dt_bias, Q0, idx, o) and for KDA the same with Gbuf
    after Pbuf; results equal those of the step followed by the flush."""
    _need_128(K, V, "make_decode")
    d = ctypes.pointer(_lib.dims(NS, HV, H, K, V, L, R, SS))
    sc = float(K ** -0.5 if scale is None else scale)
    iters, glb = int(ITERS), float(GLB)
    # One call per layer and token: at small batches its host side is what a decode step costs, so the tensors are tested and
    # their addresses taken in place, without a function call for each (one sequence, inputs sliced per token: 18.9 -> 11.8 us).
    if KDA:
        fn = _lib.lib().lq_kda_decode

        def decode(Sq, Kbuf, Ubuf, Wbuf, Pbuf, Gbuf, hcnt, mixed, a, b, A_log, dt_bias, Q0, idx, o, work=None):
            if not (Sq.is_cuda and Kbuf.is_cuda and Ubuf.is_cuda and Wbuf.is_cuda and Pbuf.is_cuda and Gbuf.is_cuda and hcnt.is_cuda
                    and mixed.is_cuda and a.is_cuda and b.is_cuda and A_log.is_cuda and dt_bias.is_cuda and Q0.is_cuda and idx.is_cuda
                    and o.is_cuda):
                _lib.not_cuda()
            wp, wn = (None, 0) if work is None else _work(work)
            _launch(fn, "lq_kda_decode", Sq, d, Sq.data_ptr(), Kbuf.data_ptr(), Ubuf.data_ptr(), Wbuf.data_ptr(), Pbuf.data_ptr(),
                    Gbuf.data_ptr(), hcnt.data_ptr(), mixed.data_ptr(), a.data_ptr(), b.data_ptr(), A_log.data_ptr(),
                    dt_bias.data_ptr(), idx.data_ptr(), o.data_ptr(), mixed.shape[0], sc, glb, Q0.data_ptr(), iters, wp, wn)
    else:
        fn = _lib.lib().lq_gdn_decode

        def decode(Sq, Kbuf, Ubuf, Wbuf, Pbuf, hcnt, mixed, a, b, A_log, dt_bias, Q0, idx, o, work=None):
            if not (Sq.is_cuda and Kbuf.is_cuda and Ubuf.is_cuda and Wbuf.is_cuda and Pbuf.is_cuda and hcnt.is_cuda and mixed.is_cuda
                    and a.is_cuda and b.is_cuda and A_log.is_cuda and dt_bias.is_cuda and Q0.is_cuda and idx.is_cuda and o.is_cuda):
                _lib.not_cuda()
            wp, wn = (None, 0) if work is None else _work(work)
            _launch(fn, "lq_gdn_decode", Sq, d, Sq.data_ptr(), Kbuf.data_ptr(), Ubuf.data_ptr(), Wbuf.data_ptr(), Pbuf.data_ptr(),
                    hcnt.data_ptr(), mixed.data_ptr(), a.data_ptr(), b.data_ptr(), A_log.data_ptr(), dt_bias.data_ptr(),
                    idx.data_ptr(), o.data_ptr(), mixed.shape[0], sc, Q0.data_ptr(), iters, wp, wn)

    return decode


def make_decode_conv(NS, HV, H, K, V, L, SS, R=4, ITERS=1, KDA=False, GLB=0.0, scale=None):
    """causal conv1d update + step + flush in one launch (no counterpart factory in the reference, whose plugin calls vLLM's
    causal_conv1d_update and then LeapQuantState.decode: leapquant/vllm/gdn.py:31-36, leapquant/vllm/glm.py:71-75).  Returns, for
    GDN, decode(Sq, Kbuf, Ubuf, Wbuf, Pbuf, hcnt, x, conv_state, conv_weight, conv_bias, a, b, A_log, dt_bias, Q0, idx, o) and
    for KDA the same with Gbuf after Pbuf.  x holds the raw q | k | v projections (bf16 [N, >= 2HK + HV V]); conv_state is the
    engine's conv cache viewed (slot, channel, width - 1) and is advanced in place; results equal make_conv1d_update followed by
    make_decode bit for bit."""
    _need_128(K, V, "make_decode_conv")
    d = _lib.dims(NS, HV, H, K, V, L, R, SS)
    sc = float(K ** -0.5 if scale is None else scale)
    iters, glb = int(ITERS), float(GLB)
    p = _lib.ptr
    if KDA:
        fn = _lib.lib().lq_kda_decode_conv

        def decode(Sq, Kbuf, Ubuf, Wbuf, Pbuf, Gbuf, hcnt, x, conv_state, conv_weight, conv_bias, a, b, A_log, dt_bias, Q0, idx, o,
                   work=None):
            cv = _lib.conv1d(x, conv_state, conv_weight, conv_bias)
            _launch(fn, "lq_kda_decode_conv", Sq, d, p(Sq), p(Kbuf), p(Ubuf), p(Wbuf), p(Pbuf), p(Gbuf), p(hcnt), cv, p(a), p(b),
                    p(A_log), p(dt_bias), p(idx), p(o), int(x.shape[0]), sc, glb, p(Q0), iters, *_work(work))
    else:
        fn = _lib.lib().lq_gdn_decode_conv

        def decode(Sq, Kbuf, Ubuf, Wbuf, Pbuf, hcnt, x, conv_state, conv_weight, conv_bias, a, b, A_log, dt_bias, Q0, idx, o, work=None):
            cv = _lib.conv1d(x, conv_state, conv_weight, conv_bias)
            _launch(fn, "lq_gdn_decode_conv", Sq, d, p(Sq), p(Kbuf), p(Ubuf), p(Wbuf), p(Pbuf), p(hcnt), cv, p(a), p(b),
                    p(A_log), p(dt_bias), p(idx), p(o), int(x.shape[0]), sc, p(Q0), iters, *_work(work))

    return decode


def make_conv1d_update(NS, channels):
    """The causal conv1d update alone, with the arithmetic of the fused kernels.  Returns
    update(x, conv_state, conv_weight, conv_bias, idx, out): out bf16 [N, channels] receives the activated rows, conv_state
    (slot, channel, width - 1) is advanced; rows with idx <= 0 are skipped.  Stands in for vLLM's causal_conv1d_update on
    single-token rows (call sites reference leapquant/vllm/gdn.py:32, leapquant/vllm/glm.py:72)."""
    fn = _lib.lib().lq_causal_conv1d_update
    p = _lib.ptr

    def update(x, conv_state, conv_weight, conv_bias, idx, out):
        cv = _lib.conv1d(x, conv_state, conv_weight, conv_bias)
        _launch(fn, "lq_causal_conv1d_update", x, cv, p(idx), int(x.shape[0]), int(channels), int(NS), p(out), out.stride(0))

    return update


def make_flush(NS, HV, K, V, L, SS, R=4, ITERS=1, SMS=148, NCG=3, MAXIT=128, PAD=8, KDA=False, MMT="bf16", PNMIN=1e-20,
               NMAX=0, NTP=0, RSG=None):
    """End-of-window flush of every head of the rows idx whose window is full.  Returns
    flush(Sq, Sk, Sv, Skv, Kbuf, Ubuf, Wbuf, Pbuf, Gbuf, hcnt, Sq16, UQ, Q0, idx)."""
    _need_128(K, V, "make_flush")
    d = _lib.dims(NS, HV, HV, K, V, L, R, SS)
    kda, iters = int(bool(KDA)), int(ITERS)
    fn = _lib.lib().lq_flush
    p = _lib.ptr

    def flush(Sq, Sk, Sv, Skv, Kbuf, Ubuf, Wbuf, Pbuf, Gbuf, hcnt, Sq16, UQ, Q0, idx):
        _launch(fn, "lq_flush", Sq, d, p(Sq), p(Kbuf), p(Ubuf), p(Wbuf), p(Pbuf), p(Gbuf) if kda else None, p(hcnt),
                p(Q0), p(idx), int(idx.shape[0]), kda, iters)

    return flush


def make_dequant(NS, HV, K, V, L, SS, BV=32, threads=128, kda=False, buf_dtype=F32, R=0):
    """fp32 S[slot] <- decay * deq(checkpoint) + live window entries, in place, for the listed slots.  Returns
    dequant(S0, Sq, Sk, Sv, Kbuf, Ubuf, Wbuf, Pbuf, Gbuf, hcnt, UQ, idx).  Window buffers must be bf16 (buf_dtype=BF16).
    kda=True rebuilds a KDA state (per-channel decay, Gbuf holding fp16 step factors) and leaves the window untouched."""
    _need_128(K, V, "make_dequant")
    if buf_dtype != BF16:
        raise NotImplementedError("make_dequant: the window buffers are bf16 in this build (buf_dtype=BF16)")
    if R not in (4, 8):
        raise NotImplementedError(f"make_dequant: R = {R}; supported 4 and 8")
    d = _lib.dims(NS, HV, HV, K, V, L, R, SS)
    kd = int(bool(kda))
    fn = _lib.lib().lq_dequant
    p = _lib.ptr

    def dequant(S0, Sq, Sk, Sv, Kbuf, Ubuf, Wbuf, Pbuf, Gbuf, hcnt, UQ, idx):
        _launch(fn, "lq_dequant", S0, d, p(S0), p(Kbuf), p(Ubuf), p(Wbuf), p(Pbuf), p(Gbuf) if kd else None, p(hcnt),
                p(idx), int(idx.shape[0]), kd)

    return dequant


def make_quantize(NS, HV, K, V, L, SS, R=4, ITERS=1, threads=128, kda=False):
    """8-bit checkpoint of the fp32 states in the listed slots, then window reset.  Returns
    quantize(S0, Sq, Sk, Sv, UQ, Wbuf, Pbuf, hcnt, Q0, idx[, Gbuf]).  kda=True (not in the reference's factory) resets a KDA
    window instead (Pbuf = 0, Gbuf = 1) and needs Gbuf as the last argument."""
    _need_128(K, V, "make_quantize")
    d = _lib.dims(NS, HV, HV, K, V, L, R, SS)
    kd, iters = int(bool(kda)), int(ITERS)
    fn = _lib.lib().lq_quantize
    p = _lib.ptr

    def quantize(S0, Sq, Sk, Sv, UQ, Wbuf, Pbuf, hcnt, Q0, idx, Gbuf=None):
        _launch(fn, "lq_quantize", S0, d, p(S0), p(Wbuf), p(Pbuf), p(Gbuf) if kd else None, p(hcnt), p(Q0), p(idx),
                int(idx.shape[0]), kd, iters)

    return quantize


def make_lowrank(K, V, R, ITERS, threads=128):
    """Rank-R subspace iteration with modified Gram-Schmidt.  Returns lowrank(S [N,K,V] f32, Q0 [V,R], U [N,K,R], Q [N,V,R])."""
    _need_128(K, V, "make_lowrank")
    fn = _lib.lib().lq_lowrank
    p = _lib.ptr
    iters = int(ITERS)

    def lowrank(S, Q0, U, Q):
        _launch(fn, "lq_lowrank", S, p(S), p(Q0), p(U), p(Q), int(S.shape[0]), K, V, R, iters)

    return lowrank


def _rule_operands(shape, strides, C, HV, V, S0, mixed, a, b, A_log, dt_bias, idx, o):
    """Checks the tensors that both forms of the gated delta rule take; returns the row strides of mixed, a and b."""
    T = mixed.shape[0]
    _lib.same_device(S0, mixed, a, b, A_log, dt_bias, idx, o)
    if S0.dtype is not torch.float32 or S0.shape != shape or S0.stride() != strides:
        raise _lib.LeapQuantError(f"gated delta rule, states: expected float32 {shape} with strides {strides}, got {S0.dtype} "
                                  f"{tuple(S0.shape)}, strides {S0.stride()}")
    _lib.whole(o, torch.bfloat16, (T, HV, V), "gated delta rule, outputs")
    _lib.whole(A_log, torch.float32, (HV,), "gated delta rule, A_log")
    _lib.whole(dt_bias, torch.float32, (HV,), "gated delta rule, dt_bias")
    return (_lib.rows(mixed, torch.bfloat16, (T, C), "gated delta rule, q | k | v rows"),
            _lib.rows(a, torch.bfloat16, (T, HV), "gated delta rule, a"), _lib.rows(b, torch.bfloat16, (T, HV), "gated delta rule, b"))


def _sequences(cu, idx, has_initial):
    """Checks the tensors that describe packed sequences; returns their number and the address of has_initial (or None)."""
    N = idx.shape[0]
    _lib.whole(idx, torch.int32, (N,), "packed sequences, slots")
    _lib.whole(cu, torch.int32, (N + 1,), "packed sequences, offsets")
    if has_initial is None:
        return N, None
    if has_initial.dtype not in (torch.bool, torch.uint8) or has_initial.shape != (N,) or not has_initial.is_contiguous():
        raise _lib.LeapQuantError(f"packed sequences, has_initial: expected contiguous bool ({N},), got {has_initial.dtype} "
                                  f"{tuple(has_initial.shape)}")
    return N, has_initial.data_ptr()


def make_gdn_prefill(NS, HV, H, K, V, SS, scale=None):
    """Gated delta rule of packed sequences on the fp32 states of their slots.  Returns
    prefill(S0, mixed, a, b, A_log, dt_bias, cu, idx, has_initial, o): S0 f32 [NS, HV, V, K] with slot stride SS, updated in place;
    mixed bf16 [T, 2HK + HV V] and a, b bf16 [T, HV] (row strides free); A_log, dt_bias f32 [HV]; cu i32 [N + 1], the first row of
    every sequence and the end of the last; idx i32 [N], their slots; has_initial bool [N] or None (all): False starts from a zero
    state; o bf16 [T, HV, V].  A sequence without tokens touches nothing; one with idx <= 0, idx >= NS or a slot that an earlier
    one names gets zeros in o and touches no state; rows of o that no sequence owns are left as they are.  The state after the last token
    is what remains: drafts that may be rejected need a copy of the state, or a call per token.  Long sequences of few
    heads are split over the SMs, for which the call takes scratch from torch's allocator (a few MB).
    prefill.check takes the same operands and only refuses what prefill would refuse."""
    _need_128(K, V, "make_gdn_prefill")
    shape, strides, C = (NS, HV, V, K), (SS, V * K, K, 1), 2 * H * K + HV * V
    d = ctypes.pointer(_lib.dims(NS, HV, H, K, V, 0, 0, SS))
    sc = float(K ** -0.5 if scale is None else scale)
    fn, fn_check, work_bytes = _lib.lib().lq_gdn_prefill, _lib.lib().lq_gdn_prefill_check, _lib.lib().lq_prefill_work_bytes

    def operands(S0, mixed, a, b, A_log, dt_bias, cu, idx, has_initial, o):
        ms, as_, bs = _rule_operands(shape, strides, C, HV, V, S0, mixed, a, b, A_log, dt_bias, idx, o)
        _lib.same_device(S0, cu, has_initial)
        N, hp = _sequences(cu, idx, has_initial)
        return ms, as_, bs, N, hp, mixed.shape[0]

    def check(S0, mixed, a, b, A_log, dt_bias, cu, idx, has_initial, o):
        ms, as_, bs, N, _, T = operands(S0, mixed, a, b, A_log, dt_bias, cu, idx, has_initial, o)
        _lib.check(fn_check(d, S0.data_ptr(), mixed.data_ptr(), ms, a.data_ptr(), as_, b.data_ptr(), bs, A_log.data_ptr(), dt_bias.data_ptr(),
                            cu.data_ptr(), idx.data_ptr(), o.data_ptr(), N, T), "lq_gdn_prefill")

    def prefill(S0, mixed, a, b, A_log, dt_bias, cu, idx, has_initial, o):
        ms, as_, bs, N, hp, T = operands(S0, mixed, a, b, A_log, dt_bias, cu, idx, has_initial, o)
        nw = work_bytes(N, HV, T) if T >= 768 and 0 < N * HV <= 256 else 0
        work = torch.empty(nw, dtype=torch.uint8, device=S0.device) if nw else None
        _launch(fn, "lq_gdn_prefill", S0, d, S0.data_ptr(), mixed.data_ptr(), ms, a.data_ptr(), as_, b.data_ptr(), bs, A_log.data_ptr(),
                dt_bias.data_ptr(), cu.data_ptr(), idx.data_ptr(), hp, o.data_ptr(), N, T, sc, work.data_ptr() if nw else None, nw)

    prefill.check = check
    return prefill


def make_gdn_recurrent(NS, HV, H, K, V, SS, scale=None):
    """Gated delta rule for one token per row on fp32 states.  Returns recurrent(S0, mixed, a, b, A_log, dt_bias, idx, o), the operands
    of make_gdn_prefill with T = N rows; rows with idx <= 0, idx >= NS or the slot of an earlier row write zeros and touch no state."""
    _need_128(K, V, "make_gdn_recurrent")
    shape, strides, C = (NS, HV, V, K), (SS, V * K, K, 1), 2 * H * K + HV * V
    d = ctypes.pointer(_lib.dims(NS, HV, H, K, V, 0, 0, SS))
    sc = float(K ** -0.5 if scale is None else scale)
    fn = _lib.lib().lq_gdn_recurrent

    def recurrent(S0, mixed, a, b, A_log, dt_bias, idx, o):
        ms, as_, bs = _rule_operands(shape, strides, C, HV, V, S0, mixed, a, b, A_log, dt_bias, idx, o)
        _lib.whole(idx, torch.int32, (mixed.shape[0],), "gated delta rule, slots")
        _launch(fn, "lq_gdn_recurrent", S0, d, S0.data_ptr(), mixed.data_ptr(), ms, a.data_ptr(), as_, b.data_ptr(), bs, A_log.data_ptr(),
                dt_bias.data_ptr(), idx.data_ptr(), o.data_ptr(), mixed.shape[0], sc)

    return recurrent


def make_conv1d_prompt(NS, channels):
    """Causal conv1d (width 4) + SiLU of packed prompts.  Returns prompt(x, conv_state, conv_weight, conv_bias, cu, idx, has_initial, out):
    x bf16 [T, >= channels], conv_state, conv_weight, conv_bias as for make_conv1d_update, cu, idx, has_initial as for
    make_gdn_prefill, out bf16 [T, channels] (not overlapping x).  conv_state receives the last three inputs of every sequence.
    The sums are fp32 and rounded once, without the update's rounding of every tap's product (so the same tokens one by one give other
    roundings).  Sequences without tokens, and those
    with idx <= 0, idx >= NS or the slot of an earlier one, are skipped (nothing read or written)."""
    fn = _lib.lib().lq_causal_conv1d_prompt

    def prompt(x, conv_state, conv_weight, conv_bias, cu, idx, has_initial, out):
        _lib.same_device(x, conv_state, conv_weight, conv_bias, cu, idx, has_initial, out)
        N, hp = _sequences(cu, idx, has_initial)
        if x.dim() != 2 or x.shape[1] < channels or tuple(conv_weight.shape) != (channels, 4) or conv_state.shape[:2] != (NS, channels) or (
                conv_bias is not None and tuple(conv_bias.shape) != (channels,)):
            raise _lib.LeapQuantError(f"conv1d prompt: x {tuple(x.shape)}, state {tuple(conv_state.shape)}, weight {tuple(conv_weight.shape)} "
                                      f"do not fit {NS} slots of {channels} channels")
        cv = _lib.conv1d(x, conv_state, conv_weight, conv_bias)
        if x.shape[0] == 1:
            cv.x_stride = -(-x.shape[1] // 8) * 8
        os_ = _lib.rows(out, torch.bfloat16, (x.shape[0], channels), "conv1d prompt, outputs")
        _launch(fn, "lq_causal_conv1d_prompt", x, cv, cu.data_ptr(), idx.data_ptr(), hp, N, x.shape[0], int(channels), int(NS),
                out.data_ptr(), os_)

    return prompt


def make_gated_norm(V, eps=1e-6):
    """Gated RMS norm of every head's output.  Returns norm(o, z, weight, y): y = o / sqrt(mean(o^2) + eps) * weight * silu(z) over the
    V values of a head; o, y bf16 [T, HV, V] (y may be o), z bf16 [T, HV * V] (row stride free), weight bf16 [V]."""
    if V != 128:
        raise NotImplementedError(f"make_gated_norm: V = {V}; this build implements heads of 128 only")
    eps = float(eps)
    fn = _lib.lib().lq_gated_norm

    def norm(o, z, weight, y):
        _lib.same_device(o, z, weight, y)
        if o.dim() != 3:
            raise _lib.LeapQuantError(f"gated norm: the outputs are [rows, heads, {V}], got {tuple(o.shape)}")
        T, HV = o.shape[:2]
        _lib.whole(o, torch.bfloat16, (T, HV, V), "gated norm, o")
        _lib.whole(y, torch.bfloat16, (T, HV, V), "gated norm, y")
        _lib.whole(weight, torch.bfloat16, (V,), "gated norm, weight")
        zs = _lib.rows(z, torch.bfloat16, (T, HV * V), "gated norm, z")
        _launch(fn, "lq_gated_norm", o, o.data_ptr(), z.data_ptr(), zs, weight.data_ptr(), y.data_ptr(), T, HV, V, eps)

    return norm


def make_add_norm(D, eps=1e-6, scale=1.0):
    """Residual stream and the norm that the next block reads.  Returns norm(x, residual, weight, y): residual <- residual + scale x;
    y = residual / sqrt(mean(residual^2) + eps) * weight, of the fp32 sum.  x, residual, y bf16 [T, D] (row strides free; y may be
    x, but overlaps neither otherwise), weight bf16 [D], which multiplies as it is: a layer that keeps w - 1 adds the 1 itself."""
    if D < 8 or D % 8 or D > 16384:
        raise NotImplementedError(f"make_add_norm: D = {D}; a multiple of 8 up to 16384 is supported")
    eps, scale = float(eps), float(scale)
    fn = _lib.lib().lq_add_norm

    def norm(x, residual, weight, y):
        _lib.same_device(x, residual, weight, y)
        T = x.shape[0]
        shape = (T, D)
        xs, rs = _lib.rows(x, torch.bfloat16, shape, "add norm, x"), _lib.rows(residual, torch.bfloat16, shape, "add norm, residual")
        ys = _lib.rows(y, torch.bfloat16, shape, "add norm, y")
        _lib.whole(weight, torch.bfloat16, (D,), "add norm, weight")
        _launch(fn, "lq_add_norm", x, x.data_ptr(), xs, residual.data_ptr(), rs, weight.data_ptr(), y.data_ptr(), ys, T, D, scale, eps)

    return norm


_mk_lowrank = functools.lru_cache(maxsize=None)(make_lowrank)
_Q0_LR = {}


def lowrank_factor(x, r, iters=3):
    """x: [..., K, V] fp32 CUDA -> U [..., K, r], Q [..., V, r] (one fused kernel)."""
    *lead, K, V = x.shape
    key = (str(x.device), V, r)
    if key not in _Q0_LR:
        _Q0_LR[key] = torch.randn(V, r, generator=torch.Generator().manual_seed(0)).to(x.device)
    xf = x.reshape(-1, K, V).contiguous().float()
    U = torch.empty(xf.shape[0], K, r, device=x.device, dtype=torch.float32)
    Q = torch.empty(xf.shape[0], V, r, device=x.device, dtype=torch.float32)
    _mk_lowrank(K, V, r, iters)(xf, _Q0_LR[key], U, Q)
    return U.reshape(*lead, K, r), Q.reshape(*lead, V, r)
