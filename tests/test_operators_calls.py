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
