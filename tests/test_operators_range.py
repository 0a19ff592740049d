"""The gated delta rule at the ends of its numbers' range: large and small states and values, rows of one head that lie far apart, states
that have all but decayed -- in both forms, which have to agree about what they carry.

Tolerance, row by row (a row of the state is one value dimension; no row reads another).  M_v = e^G |S_v| + sum e^(G_t - G_s) |u_s|
(rule64 carries scale M) bounds the terms that a row of the state is made of.  A token adds at most six factors (decays, norms, gates) that
are off by 2^-21 each, the operands' two f16 pieces 3 2^-24, sums of 64 to 128 products 2^-18: below 2^-17 of M, and the errors of
earlier tokens 2^-20 sqrt(T): for T <= 256 2^-16, together below 2^-15.  Outputs: the same times scale, and half a bf16 step.  In chunks the
smallest scaled row ends at 2^-125 and a product sums 128 of those: 2^-118; where a row has decayed far below the
bound B = |S| + sum |v| that a chunk starts with, the end of the f16 range is what counts, 2^-31 of B."""
import pytest
import torch

from test_operators import K, V, clean, impl, offsets, rule64, rule_inputs  # noqa: F401
from test_operators_precision import half_step

gpu = pytest.mark.gpu
H, HV = 2, 4


def check_rows(S, S64, o, o64, size, start, values, lens, slots, scale, T, rel=2.0 ** -15, B=None):
    """S, o against the 64-bit ones, every row of every sequence within its own bound."""
    t0 = 0
    for ln, slot in zip(lens, slots):
        M = size[t0:t0 + ln] / scale                         # [ln, HV, V]
        # B of any of the sequence's chunks: the state it starts from, and 64 values
        most = torch.maximum(M.amax(0), start[slot]) + 64 * values[t0:t0 + ln].amax(0) if B is None else B
        end = 2.0 ** -31 * most + 2.0 ** -118
        x, x64 = o[t0:t0 + ln].double(), o64[t0:t0 + ln]
        off = (x - x64).abs() - half_step(x64) - scale * (rel * M + end)
        assert float(off.max()) <= 0, ("outputs", slot, float(off.max()), float((off / (scale * M).clamp(min=1e-300)).max()))
        off = (S[slot].double() - S64[slot]).norm(dim=-1) - rel * M[-1] - end
        assert float(off.max()) <= 0, ("state", slot, float(off.max()), float((off / M[-1].clamp(min=1e-300)).max()))
        t0 += ln


def run(lens, change, seed, fresh=None, state=1.0, rel=2.0 ** -15, B=None):
    from leapquant_b200.kernels import make_gdn_prefill
    n, T = len(lens), sum(lens)
    slots = list(range(1, n + 1))
    ssm, mixed, a, b, A_log, dt_bias = rule_inputs(H, HV, T, n + 1, seed)
    ssm *= state
    change(ssm, mixed, a, b, A_log, dt_bias)
    start = ssm.double().norm(dim=-1)                        # of every slot's rows
    S64, o64 = ssm.double(), torch.zeros(T, HV, V, dtype=torch.float64, device="cuda")
    fresh = fresh or [False] * n
    size, _ = rule64(S64, mixed, a, b, A_log, dt_bias, H, lens, slots, fresh, o64)
    o = torch.zeros(T, HV, V, dtype=torch.bfloat16, device="cuda")
    hi = torch.tensor([not f for f in fresh], device="cuda")
    make_gdn_prefill(n + 1, HV, H, K, V, ssm.stride(0))(ssm, mixed, a, b, A_log, dt_bias, offsets(lens).cuda(), torch.tensor(slots, dtype=torch.int32).cuda(), hi, o)
    check_rows(ssm, S64, o, o64, size, start, mixed[:, 2 * H * K:].double().abs().view(T, HV, V), lens, slots, K ** -0.5, T, rel, B)
    clean()


def values(x):
    def change(ssm, mixed, a, b, A_log, dt_bias):
        mixed[:, 2 * H * K:] *= x
    return change


def nothing(*_):
    pass


def rows_apart(ssm, mixed, a, b, A_log, dt_bias):
    """Value dimensions from 2^-90 to 2^90, states and values alike."""
    f = torch.exp2(torch.linspace(-90, 90, V).round()).cuda()
    ssm *= f[:, None]
    mixed[:, 2 * H * K:] *= f.bfloat16().repeat(HV)


def states_apart(ssm, mixed, a, b, A_log, dt_bias):
    """States from 2^-60 to 2^100 under ordinary values."""
    ssm *= torch.exp2(torch.linspace(-60, 100, V).round()).cuda()[:, None]


def silent(steps, at=0):
    """No values, and `steps` tokens from `at` on that decay by 2^-7.2 each, the others by next to nothing."""
    def change(ssm, mixed, a, b, A_log, dt_bias):
        A_log.fill_(0.0)
        dt_bias.fill_(0.0)
        a.fill_(-20.0)
        a[at:at + steps] = 5.0
        mixed[:, 2 * H * K:] = 0
    return change


CASES = {"states_1e20": (nothing, 1e21), "states_1e30": (nothing, 1e31), "states_3e36": (nothing, 3e37), "states_1e-25": (nothing, 1e-24),
         "values_1e30": (values(1e30), 1.0), "values_1e36": (values(1e36), 1.0), "values_1e-20": (values(1e-20), 1e-20), "values_1e-28": (values(1e-28), 0.0),
         "both_1e36": (values(1e36), 1e37), "rows_apart": (rows_apart, 1.0), "states_apart": (states_apart, 1.0), "silent_2^-108": (silent(15), 1.0), "silent_2^-130": (silent(18, 70), 1.0),
         "silent_from_1e20": (silent(16), 1e21)}


@gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_ends_of_the_range(case, impl):
    change, state = CASES[case]
    run([150, 66], change, 61, fresh=[False, case.startswith("values")], state=state)


@gpu
@pytest.mark.parametrize("case", ["states_1e20", "values_1e36", "rows_apart", "states_apart", "values_1e-28"])
def test_ends_of_the_range_in_segments(case):
    """A sequence that is split: every segment starts anew, from zero, from the unit matrix and from the joined state.  1 400 tokens:
    2^-20 sqrt(T) is 2^-14.8, with the 2^-17 of a token and that of the join's sum below 2^-14."""
    from leapquant_b200 import _lib
    assert _lib.lib().lq_prefill_work_bytes(1, HV, 1400) > 0
    change, state = CASES[case]
    run([1400], change, 62, state=state, rel=2.0 ** -14)


@gpu
def test_a_row_that_shrank_keeps_its_bits(impl):
    """A row's power of two is chosen so that its bound B becomes 2^13 or more, also in the chunk after one that left an eighth of it.  The
    state starts at 1.001 2^m and loses 2^-2.95 in the first chunk and 2^-24 with the first token of the second; then 63 tokens write
    a little of it back along one key, all with the same rounding.  With the bound at 2^10 these add up to 50 2^-25 2^-10 = 2^-29.4 of B, with
    2^13 to 2^-32.4, against the 2^-31 of B that are promised: of the second chunk's B, 2^-2.95, since the first one, whose key meets zeros,
    writes nothing."""
    def change(ssm, mixed, a, b, A_log, dt_bias):
        A_log.fill_(0.0)
        dt_bias.fill_(0.0)
        a.fill_(-40.0)
        a[3] = 1.90625                                       # softplus: 2.0446 = 2.95 log 2
        a[64] = 16.625                                       # 23.98 log 2
        b.fill_(-4.84)                                       # beta = 2^-7
        mixed.zero_()
        for h in range(2 * H):                               # q and k
            mixed[:64, h * K + 5] = 1.0
            mixed[64:, h * K + 1] = 1.0
        ssm.zero_()
        ssm[1, :, :, 0] = 0.7
        ssm[1, :, :, 1] = 0.7 * (1 + torch.linspace(0, 0.4, V, device="cuda"))         # (their roundings differ)
        ssm *= 1.001 / ssm[1].norm(dim=-1).clamp(min=1e-30)[None, ..., None]
    run([128], change, 63, B=1.001 * 2.0 ** -2.949)
