"""Infinities and NaN in the operands of the gated delta rule: they reach what the rule says that depends on them, nothing before their
token, no other row, and no other sequence -- in both forms.  What is finite in 64 bits is right to the tolerance of the ends of the
range (2^-15 of the terms, half a bf16 step), what is not is not finite here."""
import pytest
import torch

from test_operators import K, V, clean, impl, offsets, rule64, rule_inputs  # noqa: F401
from test_operators_precision import half_step

gpu = pytest.mark.gpu
H, HV = 2, 4
INF, NAN = float("inf"), float("nan")


def run(lens, inject, seed=71, slots=None, NS=None):
    from leapquant_b200.kernels import make_gdn_prefill
    n, T = len(lens), sum(lens)
    slots = slots or list(range(1, n + 1))
    NS = NS or n + 1
    ssm, mixed, a, b, A_log, dt_bias = rule_inputs(H, HV, T, NS, seed)
    inject(ssm, mixed, a, b, A_log, dt_bias)
    S64, o64 = ssm.double(), torch.zeros(T, HV, V, dtype=torch.float64, device="cuda")
    size, _ = rule64(S64, mixed, a, b, A_log, dt_bias, H, lens, slots, [False] * n, o64)
    o = torch.zeros(T, HV, V, dtype=torch.bfloat16, device="cuda")
    make_gdn_prefill(NS, HV, H, K, V, ssm.stride(0))(ssm, mixed, a, b, A_log, dt_bias, offsets(lens).cuda(), torch.tensor(slots, dtype=torch.int32).cuda(), None, o)
    fin = torch.isfinite(o64)
    assert torch.equal(torch.isfinite(o), fin), "outputs that are not finite"
    off = ((o.double() - o64).abs() - half_step(o64) - 2.0 ** -15 * size)[fin]
    assert float(off.max()) <= 0, float(off.max())
    fin = torch.isfinite(S64)
    assert torch.equal(torch.isfinite(ssm), fin), "states that are not finite"
    rows = fin.all(-1)
    norm = S64[rows].norm(dim=-1) + S64[rows].norm(dim=-1).mean()
    assert float(((ssm.double() - S64)[rows].norm(dim=-1) / norm).max()) <= 2.0 ** -15
    clean()


def put(what, value, t, lane=5):
    def inject(ssm, mixed, a, b, A_log, dt_bias):
        if what == "q":
            mixed[t, K + lane] = value                       # key head 1: value heads 2 and 3
        elif what == "k":
            mixed[t, H * K + K + lane] = value
        elif what == "v":
            mixed[t, 2 * H * K + 2 * V + lane] = value       # value head 2
        elif what in "ab":
            (a if what == "a" else b)[t, 1] = value          # value head 1
        elif what == "A_log":
            A_log[3] = value
        else:
            ssm[1, 2, lane, 77] = value
    return inject


@gpu
@pytest.mark.parametrize("t", [0, 37, 63, 64, 130, 149])
@pytest.mark.parametrize("what,value", [("q", NAN), ("q", INF), ("k", NAN), ("k", -INF), ("v", NAN), ("v", INF), ("a", NAN), ("b", NAN)])
def test_a_value_of_one_token(what, value, t, impl):
    run([150, 66], put(what, value, t))


@gpu
@pytest.mark.parametrize("what,value", [("a", INF), ("a", -INF), ("b", INF), ("b", -INF)])
def test_gates_at_infinity_are_ordinary(what, value, impl):
    """A decay of zero or one, a step of zero or one."""
    run([150, 66], put(what, value, 70))


@gpu
@pytest.mark.parametrize("what,value", [("state", NAN), ("state", INF), ("A_log", NAN)])
def test_a_state_or_a_parameter(what, value, impl):
    run([150, 66], put(what, value, 0))


@gpu
def test_several_at_once(impl):
    """Two sequences, several kinds in one chunk, value dimensions with different first tokens, a row of q that is not finite before the
    others, and a sequence of one whole chunk."""
    def inject(ssm, mixed, *rest):
        for what, value, t, lane in (("q", INF, 10, 3), ("q", NAN, 62, 0), ("v", NAN, 20, 9), ("v", INF, 12, 9), ("v", -INF, 41, 127), ("b", NAN, 50, 0), ("k", INF, 55, 1),
                                     ("v", NAN, 150, 0), ("q", NAN, 151, 0), ("a", NAN, 213, 0)):
            put(what, value, t, lane)(ssm, mixed, *rest)
    run([150, 64, 70], inject)


@gpu
@pytest.mark.parametrize("what,value,t", [("q", NAN, 700), ("k", INF, 700), ("v", NAN, 3), ("v", INF, 640), ("a", NAN, 1290), ("state", NAN, 0)])
def test_in_segments(what, value, t):
    from leapquant_b200 import _lib
    assert _lib.lib().lq_prefill_work_bytes(1, HV, 1300) > 0
    run([1300], put(what, value, t))


@gpu
@pytest.mark.parametrize("lens,slots", [([1, 63, 65, 40, 130, 30], [1, 0, 3, 2, 3, 4]), ([3, 2, 70, 0, 5], [2, 9, 1, 4, 1]), ([1300, 100], [1, 0])],
                         ids=["long", "short", "segments"])
@pytest.mark.parametrize("form", [0, 1, 2])
def test_rows_of_nobody(lens, slots, form):
    """NaN in the rows behind the last sequence and in those of padding entries and repeated slots, which the boxes of 64 rows run into:
    the same bits as with zeros there."""
    from leapquant_b200 import _lib
    from leapquant_b200.kernels import make_gdn_prefill
    T, NS = sum(lens) + 40, 6
    ssm, mixed, a, b, A_log, dt_bias = rule_inputs(H, HV, T, NS, 72)
    at, live, seen = offsets(lens).tolist(), torch.zeros(T, dtype=torch.bool), set()
    for n, s in enumerate(slots):
        live[at[n]:at[n + 1]] = 0 < s < NS and s not in seen
        seen.add(s)
    live = live.cuda()
    got = []
    _lib.set_option("rule_impl", form)
    try:
        for fill in (0.0, NAN):
            S, o = ssm.clone(), torch.full((T, HV, V), 7.0, dtype=torch.bfloat16, device="cuda")
            m, ga, gb = (torch.where(live[:, None], x, fill) for x in (mixed, a, b))
            make_gdn_prefill(NS, HV, H, K, V, S.stride(0))(S, m, ga, gb, A_log, dt_bias, offsets(lens).cuda(), torch.tensor(slots, dtype=torch.int32).cuda(), None, o)
            got.append((S, o))
    finally:
        _lib.set_option("rule_impl", 0)
    assert bool(torch.isfinite(got[0][1]).all()) and bool((got[1][1][sum(lens):] == 7.0).all())
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    clean()


@gpu
@pytest.mark.parametrize("lens", [[1300], [150, 66], [5, 3]], ids=["segments", "long", "short"])
@pytest.mark.parametrize("form", [0, 1, 2])
def test_fresh_sequences_on_slots_that_hold_anything(lens, form):
    """has_initial False: the slot's bits are not read, be they a checkpoint's or NaN; the conv's neither."""
    from leapquant_b200 import _lib
    from leapquant_b200.kernels import make_conv1d_prompt, make_gdn_prefill
    n, T = len(lens), sum(lens)
    ssm, mixed, a, b, A_log, dt_bias = rule_inputs(H, HV, T, n + 1, 73)
    C = mixed.shape[1]
    w = torch.randn(C, 4, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    cu, idx, fresh = offsets(lens).cuda(), torch.arange(1, n + 1, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.bool, device="cuda")
    got = []
    _lib.set_option("rule_impl", form)
    try:
        for fill in (0.0, NAN, INF):
            S, taps = torch.full_like(ssm, fill), torch.full((n + 1, 3, C), fill, dtype=torch.bfloat16, device="cuda")
            x, o = torch.empty(T, C, dtype=torch.bfloat16, device="cuda"), torch.empty(T, HV, V, dtype=torch.bfloat16, device="cuda")
            make_conv1d_prompt(n + 1, C)(mixed, taps.transpose(1, 2), w, None, cu, idx, fresh, x)
            make_gdn_prefill(n + 1, HV, H, K, V, S.stride(0))(S, x, a, b, A_log, dt_bias, cu, idx, fresh, o)
            got.append((x, o, S[1:], taps[1:]))
    finally:
        _lib.set_option("rule_impl", 0)
    assert all(bool(torch.isfinite(t).all()) for t in got[0])
    for other in got[1:]:
        assert all(torch.equal(x, y) for x, y in zip(other, got[0]))
    clean()
