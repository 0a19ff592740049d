"""What the gated delta rule's outputs promise: everything in fp32 or its equivalent, one rounding to bf16 on the way out -- whichever
form a sequence's length selects.

Tolerance.  An output may lie half a bf16 step from the 64-bit result, and the arithmetic's error beyond that (a value near the middle of
two steps may go to the other one).  Of size = scale M, M_v = e^G |S_v| + sum e^(G_t - G_s) |u_s| (rule64 carries it along), the terms of
an output add up to at most `size`.  An operand held in two f16 pieces is off by 2^-24 of itself (2^-12 for the head, 2^-12 of that for the
remainder) and the product of the two remainders that is left out is 2^-24 of the term: 3 2^-24.  A sum of 64 to 128 products in fp32,
taken in up to 24 steps of 2^-23: below 2^-18.  Six factors (decays, norms, scales) of at most 2^-21 each: below 2^-18.  Together below
2^-17 of size; the state that an output starts from may be off by the tokens' errors before it, 2^-20 sqrt(T) of itself, which
for T <= 256 is 2^-16.  So 2^-15 of size bounds both, and 2^-31 of B the end of the f16 range."""
import pytest
import torch

from test_operators import K, V, check_rule, clean, impl, rule_inputs, run_rule  # noqa: F401

gpu = pytest.mark.gpu


def half_step(x):
    """Half a step of bf16 at x: eight significant bits."""
    return torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -126))) - 8)


@gpu
@pytest.mark.parametrize("H,HV,lens", [(2, 4, [256]), (1, 3, [64, 30, 200, 65]), (16, 32, [130])], ids=["2-4", "1-3", "16-32"])
def test_outputs_are_rounded_once(H, HV, lens, impl):
    n = len(lens)
    S, S64, o, o64, (size, largest) = run_rule(H, HV, lens, list(range(1, n + 1)), n + 1, seed=40 + HV, fresh=[i % 2 == 1 for i in range(n)])
    T = sum(lens)
    off = (o.double() - o64).abs()[:T] - half_step(o64[:T]) - 2.0 ** -15 * size[:T] - 2.0 ** -31 * largest
    assert float(off.max()) <= 0, float(off.max())
    check_rule(S, S64, o, o64, (size, largest), max(lens))
    clean()


@gpu
def test_more_heads_than_sms():
    """Chunked heads in more than one wave (seven sequences of 32 heads, 224 CTAs for 148 SMs) at an ordinary layer's head counts,
    short sequences between them."""
    lens = [70, 3, 131, 64, 29, 100, 65, 90, 12]
    n = len(lens)
    S, S64, o, o64, (size, largest) = run_rule(16, 32, lens, list(range(n, 0, -1)), n + 1, seed=77, fresh=[i % 3 == 0 for i in range(n)])
    T = sum(lens)
    off = (o.double() - o64).abs()[:T] - half_step(o64[:T]) - 2.0 ** -15 * size[:T] - 2.0 ** -31 * largest
    assert float(off.max()) <= 0, float(off.max())
    check_rule(S, S64, o, o64, (size, largest), max(lens))
    assert bool((o[T:] == 7.0).all())
    clean()
