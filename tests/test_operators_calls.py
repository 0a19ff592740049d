"""Calls of the state object that its documentation allows and that depend on more than one call: parameters in bf16 that change between
calls, calls that are refused."""
import pytest
import torch

from test_operators import K, V, offsets, rule_inputs

gpu = pytest.mark.gpu


def test_fp32_copies_follow_their_parameter():
    """The copy is of the values that the tensor has now, whichever tensor had its address before."""
    from leapquant_b200.state import LeapQuantState
    st = LeapQuantState.__new__(LeapQuantState)              # (no device needed for this)
    st._f32 = {}
    p = torch.full((8,), 0.5, dtype=torch.bfloat16)
    assert torch.equal(st._p32(p), torch.full((8,), 0.5))
    p.data.fill_(-2.0)                                       # (as a weight reload does: the version counter stays)
    assert torch.equal(st._p32(p), torch.full((8,), -2.0))
    h = p.view(torch.float16)                                # another type at the same address
    assert torch.equal(st._p32(h), h.float())
    assert st._p32(p[:3]).shape == (3,)


def layer(seed, N=2, H=2, HV=4, T=70):
    from leapquant_b200.state import LeapQuantState
    ssm, mixed, a, b, A_log, dt_bias = rule_inputs(H, HV, T, N + 1, seed)
    st = LeapQuantState(ssm, H)
    return st, ssm, mixed, a, b, A_log.bfloat16(), dt_bias.bfloat16()


def calls(st, ssm, mixed, a, b, A_log, dt_bias, how):
    """One call of the state object on a copy of the states; returns outputs and the states' bits (a checkpoint's, read as fp32, can be NaN)."""
    idx = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    S, T = ssm.clone(), mixed.shape[0]
    if how == "prefill":
        o = torch.zeros(T, 4, V, dtype=torch.bfloat16, device="cuda")
        st.prefill(S, mixed, a, b, A_log, dt_bias, idx, offsets([T - 5, 5]).cuda(), o)
    elif how == "decode_dense":
        o = torch.zeros(2, 4, V, dtype=torch.bfloat16, device="cuda")
        st.decode_dense(S, mixed[:2], a[:2], b[:2], A_log, dt_bias, idx, o)
    else:
        o = torch.zeros(2, 4, V, dtype=torch.bfloat16, device="cuda")
        st.quantize(S, idx)
        st.decode(S, mixed[:2].contiguous(), a[:2].contiguous(), b[:2].contiguous(), A_log, dt_bias, idx, o)
    torch.cuda.synchronize()
    return o, S.view(torch.int32)


@gpu
@pytest.mark.parametrize("how", ["prefill", "decode_dense", "decode"])
def test_bf16_parameters_that_change(how):
    """A_log and dt_bias in bf16, updated in place between two calls, and others at the address of freed ones: the bits that the same
    values give in fp32."""
    st, ssm, mixed, a, b, A_log, dt_bias = layer(51)
    for step in range(3):
        got = calls(st, ssm, mixed, a, b, A_log, dt_bias, how)
        want = calls(st, ssm, mixed, a, b, A_log.float(), dt_bias.float(), how)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), step
        if step == 0:
            A_log.data.add_(1.0)
            dt_bias.data.mul_(0.5)
        else:
            at = A_log.data_ptr()
            del A_log
            A_log = torch.full((4,), -1.0, dtype=torch.bfloat16, device="cuda")
            assert A_log.data_ptr() == at, "the allocator hands the block out again"


@gpu
def test_bf16_parameters_in_graphs_and_on_streams():
    """A copy made under capture is filled by every replay, from what the parameter holds then; an eager call beside it has its own."""
    st, ssm, mixed, a, b, A_log, dt_bias = layer(52)
    idx = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    S, o = ssm.clone(), torch.zeros(2, 4, V, dtype=torch.bfloat16, device="cuda")
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        st.decode_dense(S, mixed[:2], a[:2], b[:2], A_log, dt_bias, idx, o)
    with torch.cuda.stream(torch.cuda.Stream()):             # before the first replay
        got = calls(st, ssm, mixed, a, b, A_log, dt_bias, "decode_dense")
    want = calls(st, ssm, mixed, a, b, A_log.float(), dt_bias.float(), "decode_dense")
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for _ in range(2):
        S.copy_(ssm)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[0]) and torch.equal(S.view(torch.int32), want[1])
        A_log.add_(1.0)
        want = calls(st, ssm, mixed, a, b, A_log.float(), dt_bias.float(), "decode_dense")


@gpu
def test_a_refused_prefill_conv_changes_nothing():
    """Whatever the rule refuses, the conv states have not been advanced; the corrected call then gives what it gives by itself."""
    from leapquant_b200 import _lib
    st, ssm, mixed, a, b, A_log, dt_bias = layer(53)
    A_log, dt_bias = A_log.float(), dt_bias.float()
    T, C = mixed.shape
    conv = torch.randn(3, 3, C, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    w = torch.randn(C, 4, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    idx, cu = torch.tensor([1, 2], dtype=torch.int32, device="cuda"), offsets([60, 10]).cuda()
    o = torch.zeros(T, 4, V, dtype=torch.bfloat16, device="cuda")
    good = dict(a=a, b=b, A_log=A_log, dt_bias=dt_bias, out=o, ssm=ssm, has_initial=None)
    buf = torch.zeros(T * 4 * V + 8, dtype=torch.bfloat16, device="cuda")
    over = torch.zeros(T * 4 * V + T * 8, dtype=torch.bfloat16, device="cuda")
    bad = [dict(a=a[:, :3]), dict(b=b.float()), dict(a=a[:T - 1]), dict(A_log=A_log[:3]), dict(dt_bias=dt_bias.double()[:2]), dict(out=o[:T - 1]),
           dict(out=o.float()), dict(ssm=ssm[:2]), dict(ssm=ssm.bfloat16()), dict(has_initial=torch.ones(3, dtype=torch.bool, device="cuda")), dict(out=o.cpu()),
           dict(out=buf[4:4 + T * 4 * V].view(T, 4, V)),                                 # outputs that start off 16 bytes
           dict(out=over[:T * 4 * V].view(T, 4, V), a=over[8:8 + T * 8].view(T, 8)[:, :4])]      # a inside the outputs
    x, before, states = mixed.contiguous(), conv.clone(), ssm.clone()

    def call(conv, ssm, a, b, A_log, dt_bias, out, has_initial):
        st.prefill_conv(ssm, x, conv.transpose(1, 2), w, None, a, b, A_log, dt_bias, idx, cu, out, has_initial)
        torch.cuda.synchronize()

    for kw in bad:
        with pytest.raises(_lib.LeapQuantError):
            call(conv, **{**good, **kw})
        assert torch.equal(conv, before) and torch.equal(ssm, states), list(kw)
    call(conv, **good)
    assert not torch.equal(conv[1:], before[1:]) and torch.equal(conv[0], before[0])
    act = torch.empty(T, C, dtype=torch.bfloat16, device="cuda")
    again, S, o2 = before.clone(), states.clone(), torch.zeros_like(o)
    st._kconv_prompt(x, again.transpose(1, 2), w, None, cu, idx, None, act)
    st.prefill(S, act, a, b, A_log, dt_bias, idx, cu, o2)
    assert torch.equal(again, conv) and torch.equal(S, ssm) and torch.equal(o2, o)


def test_the_check_of_a_prefill_answers_like_the_call():
    """lq_gdn_prefill_check on operands that lq_gdn_prefill refuses: the same codes, without a launch in either."""
    import ctypes
    from leapquant_b200 import _lib
    L, P = _lib.lib(), ctypes.c_void_p
    d = _lib.dims(8, 4, 2, 128, 128, 0, 0, 4 * 128 * 128)
    base = dict(ssm=P(1 << 40), mixed=P(1 << 41), ms=1024, a=P(1 << 42), as_=4, b=P(1 << 43), bs=4, A=P(256), dt=P(256), cu=P(256), idx=P(256), o=P(1 << 44), N=1, T=5)
    assert L.lq_gdn_prefill_check(d, *base.values()) == 0
    for kw, rc in ((dict(N=0), 0), (dict(T=0), 0), (dict(N=-1), -4), (dict(T=-1), -4), (dict(cu=None), -1), (dict(o=None), -1), (dict(ms=1028), -3), (dict(ms=1016), -4),
                   (dict(as_=3), -4), (dict(o=P((1 << 44) + 8)), -3), (dict(o=P((1 << 41) + 1024)), -4), (dict(o=P((1 << 42) + 16)), -4), (dict(ssm=P((1 << 40) + 4)), -3)):
        v = {**base, **kw}
        assert L.lq_gdn_prefill_check(d, *v.values()) == rc, kw
        N, T = v.pop("N"), v.pop("T")
        o = v.pop("o")
        assert L.lq_gdn_prefill(d, *v.values(), None, o, N, T, 0.0, None, 0, None) == rc, kw
    assert L.lq_gdn_prefill_check(None, *base.values()) == -1


@gpu
def test_a_layers_norms_and_residual():
    """Rule -> gated norm -> scaled residual norm of one prompt: every output of the last two and the residual stream, against 64 bits on
    the bf16 rows that each of them reads (the tolerances of the operators by themselves: half a bf16 step of 2^-8, and 2^-19 of the
    terms that cancel; one fp32 rounding of |h| < 16 for the stream)."""
    from leapquant_b200.kernels import make_add_norm, make_gated_norm
    st, ssm, mixed, a, b, A_log, dt_bias = layer(54)
    T, D = mixed.shape[0], 4 * V
    g = torch.Generator().manual_seed(4)
    z = torch.randn(T, D + 128, generator=g).bfloat16().cuda()[:, 128:]
    gw, nw = (1 + 0.1 * torch.randn(V, generator=g)).bfloat16().cuda(), (1 + 0.1 * torch.randn(D, generator=g)).bfloat16().cuda()
    res = torch.randn(T, D, generator=g).bfloat16().cuda()
    before = res.double()
    o = torch.zeros(T, 4, V, dtype=torch.bfloat16, device="cuda")
    y, out = torch.empty_like(o), torch.empty(T, D, dtype=torch.bfloat16, device="cuda")
    st.prefill(ssm, mixed, a, b, A_log.float(), dt_bias.float(), torch.tensor([1, 2], dtype=torch.int32, device="cuda"), offsets([60, 10]).cuda(), o)
    make_gated_norm(V)(o, z, gw, y)
    make_add_norm(D, scale=0.5)(y.view(T, D), res, nw, out)
    od, zd = o.double(), z.double().reshape(T, 4, V)
    y64 = od / torch.sqrt((od * od).mean(-1, keepdim=True) + 1e-6) * gw.double() * zd * torch.sigmoid(zd)
    assert float(((y.double() - y64).abs() - 2.0 ** -8 * y64.abs()).max()) <= 2.0 ** -19 * float(y64.abs().max())
    h = before + 0.5 * y.double().view(T, D)
    assert float(((res.double() - h).abs() - 2.0 ** -8 * h.abs()).max()) <= 2.0 ** -21
    out64 = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * nw.double()
    assert float(((out.double() - out64).abs() - 2.0 ** -8 * out64.abs()).max()) <= 2.0 ** -19 * float(out64.abs().max())


@gpu
def test_slots_and_offsets_in_other_layouts():
    """Slots, offsets and flags as columns of a scheduler's table and in 64 bits, as dequantize() and quantize() take slots: the same bits as
    from dense int32 tensors."""
    st, ssm, mixed, a, b, A_log, dt_bias = layer(55)
    A_log, dt_bias = A_log.float(), dt_bias.float()
    T, C = mixed.shape
    w = torch.randn(C, 4, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    idx, cu, hi = torch.tensor([2, 1], device="cuda"), offsets([60, 10]).cuda().long(), torch.tensor([True, False], device="cuda")
    table = lambda t: torch.stack([t, torch.zeros_like(t)], 1)[:, 0]
    got = []
    for i, c, h in ((idx.int(), cu.int(), hi), (idx, cu, hi), (table(idx.int()), table(cu.int()), table(hi)), (table(idx), table(cu), hi)):
        S, conv = ssm.clone(), torch.ones(3, 3, C, dtype=torch.bfloat16, device="cuda")
        o, o1, o2 = torch.zeros(T, 4, V, dtype=torch.bfloat16, device="cuda"), torch.zeros(T, 4, V, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 4, V, dtype=torch.bfloat16, device="cuda")
        st.prefill_conv(S, mixed, conv.transpose(1, 2), w, None, a, b, A_log, dt_bias, i, c, o, h)
        st.prefill(S, mixed, a, b, A_log, dt_bias, i, c, o1, h)
        st.decode_dense(S, mixed[:2], a[:2], b[:2], A_log, dt_bias, i, o2)
        got.append((S, conv, o, o1, o2))
    for other in got[1:]:
        assert all(torch.equal(x, y) for x, y in zip(other, got[0]))


@gpu
def test_calls_without_tokens_or_sequences():
    st, ssm, mixed, a, b, A_log, dt_bias = layer(56)
    A_log, dt_bias = A_log.float(), dt_bias.float()
    C = mixed.shape[1]
    w, conv, before = torch.ones(C, 4, dtype=torch.bfloat16, device="cuda"), torch.ones(3, 3, C, dtype=torch.bfloat16, device="cuda"), ssm.clone()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for T, cu, idx in ((0, i32(0, 0, 0), i32(1, 2)), (0, i32(0), i32()), (5, i32(0), i32()), (5, i32(3, 3), i32(1))):
        o = torch.full((T, 4, V), 7.0, dtype=torch.bfloat16, device="cuda")
        st.prefill(ssm, mixed[:T], a[:T], b[:T], A_log, dt_bias, idx, cu, o)
        st.prefill_conv(ssm, mixed[:T], conv.transpose(1, 2), w, None, a[:T], b[:T], A_log, dt_bias, idx, cu, o)
        assert bool((o == 7.0).all())
    st.decode_dense(ssm, mixed[:0], a[:0], b[:0], A_log, dt_bias, i32(), torch.empty(0, 4, V, dtype=torch.bfloat16, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(ssm, before) and bool((conv == 1).all())


@gpu
@pytest.mark.parametrize("how", ["fused", "step_flush", "conv", "conv_one_launch"])
def test_decode_takes_slots_in_any_layout(how):
    """A column of a table of slots names the slots in it, not the numbers that lie next to one another in memory."""
    st, ssm, mixed, a, b, A_log, dt_bias = layer(57, N=4)
    A_log, dt_bias = A_log.float(), dt_bias.float()
    C = mixed.shape[1]
    w = torch.randn(C, 4, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    idx = torch.tensor([3, 1], dtype=torch.int32, device="cuda")
    table = torch.stack([idx, torch.tensor([2, 4], dtype=torch.int32, device="cuda")], 1)[:, 0]
    every = torch.arange(1, 5, dtype=torch.int32, device="cuda")
    st.fused, st.conv_one_launch = how != "step_flush", how == "conv_one_launch"
    got = []
    for i in (idx, table):
        S, conv, o = ssm.clone(), torch.ones(5, 3, C, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 4, V, dtype=torch.bfloat16, device="cuda")
        st.quantize(S, every)
        x, ga, gb = mixed[:2].contiguous(), a[:2].contiguous(), b[:2].contiguous()
        if how.startswith("conv"):
            st.decode_conv(S, x, conv.transpose(1, 2), w, None, ga, gb, A_log, dt_bias, i, o)
        else:
            st.decode(S, x, ga, gb, A_log, dt_bias, i, o)
        got.append((o, conv, S.view(torch.int32), st.hcnt.clone()))
    assert all(torch.equal(x, y) for x, y in zip(*got))


@gpu
@pytest.mark.parametrize("kda", [False, True], ids=["gdn", "kda"])
@pytest.mark.parametrize("how", ["fused", "step_flush", "conv", "conv_one_launch"])
def test_decode_takes_rows_where_the_projections_left_them(how, kda):
    """q | k | v rows, a and b as slices of wider projections: the same bits as from dense tensors.  Outputs have to be dense."""
    from leapquant_b200.state import LeapQuantState
    H, HV, N = 2, 4, 3
    C, A = 2 * H * K + HV * V, HV * (K if kda else 1)
    ssm, mixed, _, _, A_log, dt_bias = rule_inputs(H, HV, N, N + 1, 58)
    dt_bias = dt_bias.repeat_interleave(K) if kda else dt_bias
    st = LeapQuantState(ssm, H, kda=kda)
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(N, C + 64 + A + HV + (-(A + HV)) % 8, generator=g).bfloat16().cuda()       # (rows start on 16 bytes)
    w = torch.randn(C, 4, generator=g).bfloat16().cuda()
    idx = torch.tensor([3, 1, 2], dtype=torch.int32, device="cuda")
    st.fused, st.conv_one_launch = how != "step_flush", how == "conv_one_launch"
    rows, a, b = wide[:, :C], wide[:, C + 64:C + 64 + A], wide[:, C + 64 + A:C + 64 + A + HV]
    got = []
    for x, ga, gb in ((rows.contiguous(), a.contiguous(), b.contiguous()), (rows, a, b)):
        S, conv, o = ssm.clone(), torch.ones(N + 1, 3, C, dtype=torch.bfloat16, device="cuda"), torch.zeros(N, HV, V, dtype=torch.bfloat16, device="cuda")
        st.quantize(S, torch.arange(1, N + 1, dtype=torch.int32, device="cuda"))
        if how.startswith("conv"):
            st.decode_conv(S, x, conv.transpose(1, 2), w, None, ga, gb, A_log, dt_bias, idx, o)
        else:
            st.decode(S, x, ga, gb, A_log, dt_bias, idx, o)
        got.append((o, conv, S.view(torch.int32), st.hcnt.clone()))
    assert all(torch.equal(x, y) for x, y in zip(*got))
    with pytest.raises(ValueError):
        st.decode(S, rows, a, b, A_log, dt_bias, idx, torch.zeros(N, HV, 2 * V, dtype=torch.bfloat16, device="cuda")[:, :, :V])
