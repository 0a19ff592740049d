"""The operators around the decode step -- the gated delta rule on fp32 states, the conv1d of prompts, the gated norm and the
residual norm -- against plain implementations in 64 bits, and their refusals.

Tolerances.  A rounding to bf16 is off by at most 2^-8 of the value.
State (fp32): the rule is a contraction (|k^| <= 1, 0 <= beta <= 1, decay <= 1), so the errors of the tokens at most add up.  A
token's own error is that of sums of 128 fp32 products, about sqrt(128) 2^-24 < 2^-20 of the state's norm, and of random sign:
2^-20 sqrt(tokens) of the norm.
Outputs of the rule: 2^-8 of the value for the rounding to bf16, plus the arithmetic.  In o = e^G S_0 q^ + sum_s A_ts u_s the operands
S_0, A and u may be rounded to 11 bits, 2^-12 of each: an error of at most 2^-12 (e^G sum_k |S_vk q^_k| + 2 sum_s |A_ts u_s|), and since
|q^| <= scale and |A_ts| <= scale e^{G_t - G_s}, of at most 2^-11 scale M with M_v = e^{G_t} |S_v| + sum_s e^{G_t - G_s} |u_s|, which
rule64 carries along (M <- e^g M + |u|).  Where everything has decayed, what is left is the end of the f16 range: a row of S, r or u is
scaled by a power of two so that its bound B = |S_0| + sum |v_t| over the 64 tokens of a chunk becomes 2^13 or more, and the last bit of an
f16 is 2^-24 there; halved and summed over 64 tokens and two operands that is 2^-25 2^-13 64 2 = 2^-31 of B, times scale.
Norms and the conv1d: 2^-8 of the value, and 2^-19 of the terms that cancel (some ten fp32 operations of 2^-24, exp of 2^-22)."""
import ctypes
import math

import pytest
import torch

K = V = 128
CHUNK = 64
gpu = pytest.mark.gpu
HALF = 2.0 ** -8


def offsets(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32)


def rule64(S, mixed, a, b, A_log, dt_bias, H, lens, slots, fresh, out, scale=K ** -0.5):
    """The definition, token by token in 64 bits; S and out are changed in place.  Returns scale M of every output, and scale times a
    bound of B."""
    HV = A_log.shape[0]
    t = 0
    size = torch.zeros_like(out)
    seen = set()
    for n, (ln, slot) in enumerate(zip(lens, slots)):
        live = 0 < slot < S.shape[0] and slot not in seen
        seen.add(slot)
        if not live:
            out[t:t + ln] = 0
            t += ln
            continue
        if ln == 0:
            continue
        s = torch.zeros_like(S[slot]) if fresh[n] else S[slot].clone()
        M = s.norm(dim=-1)
        for _ in range(ln):
            x = mixed[t].double()
            q, k, v = x[:H * K].view(H, K), x[H * K:2 * H * K].view(H, K), x[2 * H * K:].view(HV, V)
            q = (q / torch.sqrt((q * q).sum(-1, keepdim=True) + 1e-6) * scale).repeat_interleave(HV // H, 0)
            k = (k / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-6)).repeat_interleave(HV // H, 0)
            z = a[t].double() + dt_bias.double()
            decay = torch.exp(-torch.exp(A_log.double()) * torch.log1p(torch.exp(z)))
            s = s * decay[:, None, None]
            u = torch.sigmoid(b[t].double())[:, None] * (v - torch.einsum("hvk,hk->hv", s, k))
            s = s + u[..., None] * k[:, None]
            out[t] = torch.einsum("hvk,hk->hv", s, q)
            M = M * decay[:, None] + u.abs()
            size[t] = scale * M
            t += 1
        S[slot] = s
    largest = float(size.max()) + scale * CHUNK * float(mixed[:, 2 * H * K:].double().abs().max())
    return size, largest


def rule_inputs(H, HV, rows, NS, seed, device="cuda", slot_pad=0, wide=0):
    """States, rows and gates of a layer; slot_pad: extra floats between slots, wide: extra elements between rows."""
    g = torch.Generator().manual_seed(seed)
    C = 2 * H * K + HV * V
    SS = HV * V * K + slot_pad
    ssm = torch.zeros(NS, SS).to(device)[:, :HV * V * K].view(NS, HV, V, K)
    ssm.copy_(0.1 * torch.randn(NS, HV, V, K, generator=g))
    mixed = torch.randn(rows, C + wide, generator=g).bfloat16().to(device)[:, wide:]
    ba = torch.randn(rows, 2 * HV, generator=g).bfloat16().to(device)
    A_log = torch.log(1 + 15 * torch.rand(HV, generator=g)).to(device)
    dt_bias = torch.log(torch.expm1(0.001 * 100 ** torch.rand(HV, generator=g))).to(device)
    return ssm, mixed, ba[:, HV:], ba[:, :HV], A_log, dt_bias


def check_rule(S, S64, o, o64, size, tokens, what=""):
    """size: what rule64 returned; tokens: the longest sequence."""
    S, o = S.double(), o.double()
    for h in range(S.shape[1]):
        n = float(S64[:, h].norm())
        assert float((S[:, h] - S64[:, h]).norm()) <= 2.0 ** -20 * math.sqrt(max(tokens, 1)) * n, (what, "state", h, float((S[:, h] - S64[:, h]).norm()) / n)
    size, largest = size
    off = (o - o64).abs() - HALF * o64.abs() - 2.0 ** -11 * size - 2.0 ** -31 * largest
    assert float(off.max()) <= 0, (what, "outputs", float(off.max()))


def run_rule(H, HV, lens, slots, NS, seed=0, fresh=None, tail=3, change=None, **kw):
    from leapquant_b200.kernels import make_gdn_prefill
    T = sum(lens) + tail
    ssm, mixed, a, b, A_log, dt_bias = rule_inputs(H, HV, T, NS, seed, **kw)
    if change is not None:
        change(mixed, a, b, A_log, dt_bias)
    fresh = fresh or [False] * len(lens)
    S64 = ssm.double().clone()
    o = torch.full((T, HV, V), 7.0, dtype=torch.bfloat16, device="cuda")
    o64 = o.double()
    size = rule64(S64, mixed, a, b, A_log, dt_bias, H, lens, slots, fresh, o64)
    hi = torch.tensor([not f for f in fresh], device="cuda") if any(fresh) else None
    make_gdn_prefill(NS, HV, H, K, V, ssm.stride(0))(ssm, mixed, a, b, A_log, dt_bias, offsets(lens).cuda(),
                                                    torch.tensor(slots, dtype=torch.int32).cuda(), hi, o)
    return ssm, S64, o, o64, size


@pytest.fixture(params=[1, 2], ids=["tokens", "chunks"])
def impl(request):
    """Both forms of lq_gdn_prefill, whatever the lengths."""
    from leapquant_b200 import _lib
    _lib.set_option("rule_impl", request.param)
    yield request.param
    _lib.set_option("rule_impl", 0)


def clean():
    from leapquant_b200 import _lib
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


# ---- the gated delta rule ----
@gpu
@pytest.mark.parametrize("lens", [[1], [5], [63], [64], [65], [200], [2, 1, 4, 3], [70, 1, 0, 128, 17, 64, 0, 33], [0, 129, 0]],
                         ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("H,HV", [(2, 4), (1, 3), (2, 2)])
def test_prefill_lengths_and_heads(lens, H, HV, impl):
    n = len(lens)
    slots = [n - i for i in range(n)]
    S, S64, o, o64, size = run_rule(H, HV, lens, slots, n + 2, seed=sum(lens) + HV, fresh=[i % 2 == 1 for i in range(n)])
    check_rule(S, S64, o, o64, size, max(lens))
    assert torch.equal(S[0].double(), S64[0]) and torch.equal(S[n + 1].double(), S64[n + 1]), "other slots"
    assert bool((o[sum(lens):] == 7.0).all()), "rows behind the last sequence"
    for i, ln in enumerate(lens):
        if ln == 0:
            assert torch.equal(S[slots[i]].double(), S64[slots[i]]), "a sequence without tokens"
    clean()


@gpu
@pytest.mark.parametrize("lens", [[90, 1, 66, 70, 5, 64], [2, 1, 3, 2, 1, 2]], ids=["long", "short"])
def test_prefill_padding_entries_and_repeated_slots(lens, impl):
    """idx <= 0, idx >= NS and the second entry of a slot: zeros in the outputs, no state touched."""
    slots = [3, 0, 99, 3, -1, 2]
    S, S64, o, o64, size = run_rule(2, 4, lens, slots, 5, seed=4)
    check_rule(S, S64, o, o64, size, max(lens))
    t = offsets(lens).tolist()
    for i in (1, 2, 3, 4):
        assert float(o[t[i]:t[i + 1]].float().abs().max()) == 0.0
    for slot in (0, 1, 4):
        assert torch.equal(S[slot].double(), S64[slot])
    clean()


@gpu
@pytest.mark.parametrize("kw", [dict(slot_pad=4096), dict(wide=64), dict(slot_pad=64, wide=8)], ids=["slots", "rows", "both"])
def test_prefill_strides(kw, impl):
    S, S64, o, o64, size = run_rule(2, 4, [100, 3, 64], [1, 2, 3], 4, seed=5, **kw)
    check_rule(S, S64, o, o64, size, 100)
    clean()


@gpu
@pytest.mark.parametrize("lens", [[18], [20], [1, 30, 5, 64, 19, 20, 21, 0, 100, 1], [(7 * i) % 45 for i in range(150)], [3] * 140 + [70],
                                  [27], [28], [64, 27, 28, 29, 0, 130], [2] * 300 + [28] + [1] * 500 + [65, 3, 30],
                                  [900, 7, 8, 9, 1, 20, 1100]],
                         ids=["18", "20", "mixed", "150", "141", "27", "28", "around28", "804", "among_long"])
def test_prefill_batches_of_short_and_long_sequences(lens):
    """What a caller gets by default: each sequence in the form that suits its length, in batches that are ranked by it and larger ones."""
    n = len(lens)
    slots = [(i * 7) % n + 1 if n % 7 else i + 1 for i in range(n)]
    S, S64, o, o64, size = run_rule(1, 2, lens, slots, n + 1, seed=n, fresh=[i % 3 == 0 for i in range(n)])
    check_rule(S, S64, o, o64, size, max(lens))
    assert bool((o[sum(lens):] == 7.0).all())
    clean()


def work_bytes(n, HV, T):
    from leapquant_b200 import _lib
    return _lib.lib().lq_prefill_work_bytes(n, HV, T)


def test_only_few_long_sequences_are_split():
    """Scratch is asked for where both passes fit 148 SMs and the chain is long enough; at least the states and maps of three segments."""
    assert work_bytes(1, 32, 8192) == 32 * 3 * 65536 and work_bytes(1, 8, 8192) == 8 * 17 * 65536
    for n, HV, T in ((1, 32, 512), (1, 64, 8192), (64, 32, 65536), (2, 32, 16384), (1, 1, 640), (0, 32, 8192), (1, 0, 8192), (1, 32, 0), (1 << 30, 1 << 30, 1 << 40)):
        assert work_bytes(n, HV, T) == 0, (n, HV, T)


@gpu
@pytest.mark.parametrize("H,HV,lens,slots", [(1, 2, [1300], [1]), (2, 4, [2500], [2]), (1, 1, [4096], [1]), (1, 2, [1281], [1]), (2, 2, [3600, 900, 12], [3, 1, 2]),
                                             (1, 2, [1400, 1400, 1500], [2, 0, 2]), (1, 1, [5, 0, 6000, 65], [1, 2, 3, 4]), (4, 32, [3000], [1])],
                         ids=lambda x: "-".join(map(str, x)) if isinstance(x, list) else None)
def test_prefill_split_over_segments(H, HV, lens, slots):
    """Few long sequences, which are run as segments and joined: odd lengths, short and empty ones beside them, padding, a repeated slot."""
    n = len(lens)
    assert work_bytes(n, HV, sum(lens) + 3) > 0
    for fresh in (None, [i % 2 == 0 for i in range(n)]):
        S, S64, o, o64, size = run_rule(H, HV, lens, slots, max(slots) + 2, seed=sum(lens) + HV, fresh=fresh)
        check_rule(S, S64, o, o64, size, max(lens))
        assert bool((o[sum(lens):] == 7.0).all())
        assert torch.equal(S[0].double(), S64[0])
    clean()


@gpu
@pytest.mark.parametrize("change", ["same_keys", "no_decay", "large_values", "small_values", "uneven_keys"])
def test_prefill_split_unusual_values(change):
    S, S64, o, o64, size = run_rule(2, 4, [1500], [1], 3, seed=6, change=globals()[change])
    check_rule(S, S64, o, o64, size, 1500, change)
    clean()


@gpu
def test_prefill_split_without_scratch_on_streams_and_in_graphs():
    """The same call twice, on a side stream, and captured and replayed beside another one: the same bits.  Without scratch the C entry
    runs a head on one SM: the same to fp32 roundings."""
    from leapquant_b200 import _lib
    from leapquant_b200.kernels import make_gdn_prefill
    H, HV, T = 2, 4, 1700
    ssm, mixed, a, b, A_log, dt_bias = rule_inputs(H, HV, T, 3, 21)
    f = make_gdn_prefill(3, HV, H, K, V, ssm.stride(0))
    cu, idx = offsets([T]).cuda(), torch.tensor([2], dtype=torch.int32, device="cuda")
    runs = []
    for how in ("plain", "again", "stream", "graph"):
        S, o = ssm.clone(), torch.zeros(T, HV, V, dtype=torch.bfloat16, device="cuda")
        call = lambda: f(S, mixed, a, b, A_log, dt_bias, cu, idx, None, o)
        torch.cuda.synchronize()
        if how == "stream":
            with torch.cuda.stream(torch.cuda.Stream()):
                call()
        elif how == "graph":
            g, S2, o2 = torch.cuda.CUDAGraph(), ssm.clone(), torch.zeros_like(o)
            with torch.cuda.graph(g):
                call()
                f(S2, mixed, a, b, A_log, dt_bias, cu, idx, None, o2)
            for s in (S, S2):
                s.copy_(ssm)
            g.replay()
            torch.cuda.synchronize()
            runs.append((S2, o2))
        else:
            call()
        torch.cuda.synchronize()
        runs.append((S, o))
    for S, o in runs[1:]:
        assert torch.equal(S, runs[0][0]) and torch.equal(o, runs[0][1])
    S, o = ssm.clone(), torch.zeros(T, HV, V, dtype=torch.bfloat16, device="cuda")
    _lib.launch(_lib.lib().lq_gdn_prefill, "lq_gdn_prefill", S, _lib.dims(3, HV, H, K, V, 0, 0, S.stride(0)), S.data_ptr(), mixed.data_ptr(), mixed.stride(0),
                a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), A_log.data_ptr(), dt_bias.data_ptr(), cu.data_ptr(), idx.data_ptr(), None, o.data_ptr(),
                1, T, K ** -0.5, None, 0)
    assert float((S - runs[0][0]).norm() / S.norm()) <= 2 * 2.0 ** -20 * math.sqrt(T)     # both within the bound of the 64-bit result
    clean()


@gpu
def test_prefills_side_by_side():
    """Calls on two streams at once, one that is split into segments and one that is not, on different slots of one state tensor, leave what
    they leave one after the other; and their other operators run between them."""
    from leapquant_b200.kernels import make_conv1d_prompt, make_gated_norm, make_gdn_prefill
    H, HV, lens = 2, 4, ([1500], [40, 7, 200, 3, 90])
    slots = ([6], [1, 2, 3, 4, 5])
    ssm, mixed, a, b, A_log, dt_bias = rule_inputs(H, HV, 1500, 7, 31)
    f, norm, conv = make_gdn_prefill(7, HV, H, K, V, ssm.stride(0)), make_gated_norm(V), make_conv1d_prompt(7, mixed.shape[1])
    cu, idx = [offsets(x).cuda() for x in lens], [torch.tensor(x, dtype=torch.int32, device="cuda") for x in slots]
    w = torch.randn(mixed.shape[1], 4, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    gw = torch.ones(V, dtype=torch.bfloat16, device="cuda")
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for together in (False, True, True, True):
        S, taps = ssm.clone(), torch.zeros(7, 3, mixed.shape[1], dtype=torch.bfloat16, device="cuda")
        outs = []
        torch.cuda.synchronize()
        for i in (0, 1):
            n = sum(lens[i])
            with torch.cuda.stream(streams[i]):
                x, o, y = torch.empty(n, mixed.shape[1], dtype=torch.bfloat16, device="cuda"), *(torch.empty(n, HV, V, dtype=torch.bfloat16, device="cuda") for _ in range(2))
                conv(mixed[:n], taps.transpose(1, 2), w, None, cu[i], idx[i], None, x)
                f(S, x, a[:n], b[:n], A_log, dt_bias, cu[i], idx[i], None, o)
                norm(o, mixed[:n, : HV * V], gw, y)
                outs += [o, y]
            if not together:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        got.append([S, taps] + outs)
    for other in got[1:]:
        assert all(torch.equal(x, y) for x, y in zip(other, got[0]))
    clean()


def same_keys(mixed, a, b, A_log, dt_bias):
    mixed[:, 256:512] = mixed[0, 256:512]                    # H = 2: every key the same, every step written in full
    b.fill_(8.0)
    a.fill_(-20.0)


def fast_decay(mixed, a, b, A_log, dt_bias):
    a[::3] = 30.0                                            # e^g of some tokens is zero, of the others near one
    a[1::3] = -9.0


def no_decay(mixed, a, b, A_log, dt_bias):
    a.fill_(-40.0)


def large_values(mixed, a, b, A_log, dt_bias):
    mixed[:, 512:] *= 1e6


def small_values(mixed, a, b, A_log, dt_bias):
    mixed[:, 512:] *= 1e-6


def large_keys(mixed, a, b, A_log, dt_bias):
    mixed[:, :512] *= 1e8


def small_keys(mixed, a, b, A_log, dt_bias):
    mixed[:, :512] *= 1e-4                                   # |k|^2 at the size of the 1e-6 that is added to it


def tiny_keys(mixed, a, b, A_log, dt_bias):
    mixed[:, :512] *= 1e-18


def zero_rows(mixed, a, b, A_log, dt_bias):
    mixed[5] = 0
    mixed[40:50, :512] = 0
    mixed[70:, 512:] = 0


def uneven_keys(mixed, a, b, A_log, dt_bias):
    mixed[:, 0:512:7] *= 2.0 ** -12                          # entries far below the others of their key


def decayed_and_silent(mixed, a, b, A_log, dt_bias):
    """Eleven tokens that leave 2^-79 of the state, and no values: what is left of it is all there is."""
    A_log.fill_(0.0)
    dt_bias.fill_(0.0)
    a.fill_(-20.0)
    a[:11] = 5.0
    a[150:161] = 5.0                                         # (the second sequence)
    mixed[:, 512:] = 0


@gpu
@pytest.mark.parametrize("change", [same_keys, fast_decay, decayed_and_silent, no_decay, large_values, small_values, large_keys, small_keys, tiny_keys,
                                    zero_rows, uneven_keys], ids=lambda f: f.__name__)
def test_prefill_unusual_values(change, impl):
    S, S64, o, o64, size = run_rule(2, 4, [150, 66], [1, 2], 3, seed=6, fresh=[False, True], change=change)
    check_rule(S, S64, o, o64, size, 150, change.__name__)
    clean()


@gpu
def test_prefill_in_pieces_equals_one_call(impl):
    """A prompt in three calls: what the pieces leave in the slot is what the next one takes up."""
    from leapquant_b200.kernels import make_gdn_prefill
    H, HV, T, cuts = 2, 4, 230, [0, 70, 71, 230]
    ssm, mixed, a, b, A_log, dt_bias = rule_inputs(H, HV, T, 3, 8)
    S64, o64 = ssm.double(), torch.zeros(T, HV, V, dtype=torch.float64, device="cuda")
    size = rule64(S64, mixed, a, b, A_log, dt_bias, H, [T], [2], [False], o64)
    f = make_gdn_prefill(3, HV, H, K, V, ssm.stride(0))
    o = torch.zeros(T, HV, V, dtype=torch.bfloat16, device="cuda")
    slot = torch.tensor([2], dtype=torch.int32, device="cuda")
    for lo, hi in zip(cuts, cuts[1:]):
        f(ssm, mixed[lo:hi], a[lo:hi], b[lo:hi], A_log, dt_bias, offsets([hi - lo]).cuda(), slot, None, o[lo:hi])
    check_rule(ssm, S64, o, o64, size, T)
    clean()


@gpu
def test_prefill_runs_do_not_differ_and_follow_their_stream(impl):
    """The same call twice gives the same bits; a call on a side stream, and one captured into a graph and replayed, too."""
    from leapquant_b200.kernels import make_gdn_prefill
    H, HV, lens = 4, 8, [300, 64, 5, 77]
    ssm, mixed, a, b, A_log, dt_bias = rule_inputs(H, HV, sum(lens), 5, 9)
    f = make_gdn_prefill(5, HV, H, K, V, ssm.stride(0))
    cu, idx = offsets(lens).cuda(), torch.tensor([4, 2, 1, 3], dtype=torch.int32, device="cuda")
    got = []
    for how in ("plain", "again", "stream", "graph"):
        S, o = ssm.clone(), torch.zeros(sum(lens), HV, V, dtype=torch.bfloat16, device="cuda")
        call = lambda: f(S, mixed, a, b, A_log, dt_bias, cu, idx, None, o)
        torch.cuda.synchronize()
        if how == "stream":
            with torch.cuda.stream(torch.cuda.Stream()):
                call()
        elif how == "graph":
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                call()
            S.copy_(ssm)
            g.replay()
        else:
            call()
        torch.cuda.synchronize()
        got.append((S, o))
    for S, o in got[1:]:
        assert torch.equal(S, got[0][0]) and torch.equal(o, got[0][1])
    clean()


@gpu
@pytest.mark.parametrize("N,H,HV", [(1, 2, 2), (7, 2, 4), (70, 1, 3)])
def test_recurrent(N, H, HV):
    """Several tokens one after the other, with padding rows, a repeated slot, and steps that leave rows out."""
    from leapquant_b200.kernels import make_gdn_recurrent
    NS, steps = N + 3, 4
    ssm, mixed, a, b, A_log, dt_bias = rule_inputs(H, HV, steps * N, NS, 11, slot_pad=64, wide=16)
    f = make_gdn_recurrent(NS, HV, H, K, V, ssm.stride(0))
    slots = [(5 * n) % N + 1 if N % 5 else n + 1 for n in range(N)]
    if N > 3:
        slots[1], slots[2], slots[3] = 0, -4, slots[0]
    S64 = ssm.double().clone()
    for t in range(steps):
        n = N if t != 1 else (N + 1) // 2
        at = slice(t * N, t * N + n)
        o = torch.full((n, HV, V), 7.0, dtype=torch.bfloat16, device="cuda")
        o64 = torch.zeros(n, HV, V, dtype=torch.float64, device="cuda")
        size = rule64(S64, mixed[at], a[at], b[at], A_log, dt_bias, H, [1] * n, slots[:n], [False] * n, o64)
        f(ssm, mixed[at], a[at], b[at], A_log, dt_bias, torch.tensor(slots[:n], dtype=torch.int32).cuda(), o)
        check_rule(ssm, S64, o, o64, size, t + 1)
    clean()


@gpu
def test_scale_is_the_factorys():
    from leapquant_b200.kernels import make_gdn_prefill, make_gdn_recurrent
    ssm, mixed, a, b, A_log, dt_bias = rule_inputs(1, 1, 70, 2, 12)
    for lens, make in (([70], make_gdn_prefill), ([1], make_gdn_recurrent)):
        S, S64, T = ssm.clone(), ssm.double(), sum(lens)
        o, o64 = torch.zeros(T, 1, V, dtype=torch.bfloat16, device="cuda"), torch.zeros(T, 1, V, dtype=torch.float64, device="cuda")
        size = rule64(S64, mixed, a, b, A_log, dt_bias, 1, lens, [1], [False], o64, scale=0.7)
        one = torch.ones(1, dtype=torch.int32, device="cuda")
        more = (offsets(lens).cuda(), one, None) if T > 1 else (one,)
        make(2, 1, 1, K, V, ssm.stride(0), scale=0.7)(S, mixed[:T], a[:T], b[:T], A_log, dt_bias, *more, o)
        check_rule(S, S64, o, o64, size, T)
    clean()


# ---- conv1d of prompts ----
def conv64(x, state, w, bias, lens, slots, fresh, out):
    """state [NS, C, 3] and out are changed in place."""
    t, seen = 0, set()
    for n, (ln, slot) in enumerate(zip(lens, slots)):
        live = 0 < slot < state.shape[0] and slot not in seen and ln > 0
        seen.add(slot)
        if live:
            past = state[slot].t() * (0.0 if fresh[n] else 1.0)
            full = torch.cat([past, x[t:t + ln]])                                       # [3 + ln, C]
            y = sum(w[:, j] * full[j:j + ln] for j in range(4)) + bias
            out[t:t + ln] = y * torch.sigmoid(y)
            state[slot] = full[ln:].t()
        t += ln


@gpu
@pytest.mark.parametrize("lens", [[1], [2], [3], [15, 16, 17, 1, 2], [0, 40, 0, 0, 100, 5, 0], [1] * 70, [33] * 40], ids=lambda x: f"{len(x)}x{max(x)}")
@pytest.mark.parametrize("channels", [8, 384, 1032])
@pytest.mark.parametrize("dim_first", [False, True], ids=["slot_tap_channel", "slot_channel_tap"])
def test_conv1d_prompt(lens, channels, dim_first):
    from leapquant_b200.kernels import make_conv1d_prompt
    g = torch.Generator().manual_seed(len(lens) + channels)
    n, T, NS = len(lens), sum(lens), len(lens) + 2
    slots = [n - i for i in range(n)]
    if n > 4:
        slots[1], slots[3] = 0, slots[0]
    fresh = [i % 3 == 0 for i in range(n)]
    x = torch.randn(T + 2, channels + 24, generator=g).bfloat16().cuda()
    store = torch.randn(*((NS, channels, 3) if dim_first else (NS, 3, channels)), generator=g).bfloat16().cuda()
    state = store if dim_first else store.transpose(1, 2)
    w, bias = (0.5 * torch.randn(channels, 4, generator=g)).bfloat16().cuda(), (0.1 * torch.randn(channels, generator=g)).bfloat16().cuda()
    for with_bias in (True, False):
        out = torch.full((T + 2, channels), 7.0, dtype=torch.bfloat16, device="cuda")
        st64, out64 = state.double().clone(), out.double()
        conv64(x[:T, 8:8 + channels].double(), st64, w.double(), bias.double() if with_bias else 0.0, lens, slots, fresh, out64)
        make_conv1d_prompt(NS, channels)(x[:, 8:8 + channels], state, w, bias if with_bias else None, offsets(lens).cuda(),
                                         torch.tensor(slots, dtype=torch.int32).cuda(), torch.tensor([not f for f in fresh]).cuda(), out)
        off = (out.double() - out64).abs() - HALF * out64.abs()
        assert float(off.max()) <= 2.0 ** -19 * 8, float(off.max())                     # terms of |w x| up to about 8
        assert torch.equal(state.double(), st64), "conv state"
    clean()


@gpu
def test_conv1d_prompt_in_pieces_equals_one_call():
    from leapquant_b200.kernels import make_conv1d_prompt
    g = torch.Generator().manual_seed(3)
    C, T, cuts = 256, 90, [0, 1, 3, 20, 90]
    x, w = torch.randn(T, C, generator=g).bfloat16().cuda(), torch.randn(C, 4, generator=g).bfloat16().cuda()
    store = torch.randn(2, 3, C, generator=g).bfloat16().cuda()
    s1, s2 = store.clone(), store.clone()
    o1, o2 = (torch.zeros(T, C, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    f, one = make_conv1d_prompt(2, C), torch.ones(1, dtype=torch.int32, device="cuda")
    f(x, s1.transpose(1, 2), w, None, offsets([T]).cuda(), one, None, o1)
    for lo, hi in zip(cuts, cuts[1:]):
        f(x[lo:hi], s2.transpose(1, 2), w, None, offsets([hi - lo]).cuda(), one, None, o2[lo:hi])
    assert torch.equal(o1, o2) and torch.equal(s1, s2)
    clean()


# ---- norms ----
@gpu
@pytest.mark.parametrize("T,HV", [(1, 1), (3, 5), (130, 32), (2049, 3)])
@pytest.mark.parametrize("size", [1.0, 1e-4, 1e4])
def test_gated_norm(T, HV, size):
    from leapquant_b200.kernels import make_gated_norm
    g = torch.Generator().manual_seed(T)
    o = (size * torch.randn(T, HV, V, generator=g)).bfloat16().cuda()
    o[0, 0] = 0
    z = (3 * torch.randn(T, HV * V + 256, generator=g)).bfloat16().cuda()[:, 256:]
    w = torch.randn(V, generator=g).bfloat16().cuda()
    f = make_gated_norm(V, eps=1e-5)
    y = torch.empty_like(o)
    f(o, z, w, y)
    od, zd = o.double(), z.double().reshape(T, HV, V)
    ref = od / torch.sqrt((od * od).mean(-1, keepdim=True) + 1e-5) * w.double() * zd * torch.sigmoid(zd)
    off = (y.double() - ref).abs() - HALF * ref.abs()
    assert float(off.max()) <= 2.0 ** -19 * float(ref.abs().max()), float(off.max())
    f(o, z, w, o)                                            # written over its input
    assert torch.equal(o, y)
    clean()


@gpu
@pytest.mark.parametrize("T", [1, 7, 300])
@pytest.mark.parametrize("D", [8, 128, 1000, 4096, 5120, 8200, 16384])
@pytest.mark.parametrize("scale", [1.0, -0.37])
def test_add_norm(T, D, scale):
    from leapquant_b200.kernels import make_add_norm
    g = torch.Generator().manual_seed(D + T)
    x = torch.randn(T, D + 8, generator=g).bfloat16().cuda()[:, 8:]
    r = torch.randn(T, D + 16, generator=g).bfloat16().cuda()[:, :D]
    w = torch.randn(D, generator=g).bfloat16().cuda()
    h = r.double() + scale * x.double()
    ref = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * w.double()
    f = make_add_norm(D, scale=scale)
    r2, x2, y = r.clone(), x.clone(), torch.empty(T, D, dtype=torch.bfloat16, device="cuda")
    f(x, r, w, y)
    assert float(((r.double() - h).abs() - HALF * h.abs()).max()) <= 2.0 ** -23 * 10     # one fp32 rounding of |h| < 10
    off = (y.double() - ref).abs() - HALF * ref.abs()
    assert float(off.max()) <= 2.0 ** -19 * float(ref.abs().max()), float(off.max())
    f(x2, r2, w, x2)                                         # written over the branch
    assert torch.equal(x2, y) and torch.equal(r2, r)
    clean()


# ---- a layer's operators together ----
@gpu
def test_layer_prompt_then_decode():
    """Raw projections -> conv1d -> rule -> gated norm -> residual norm, through the state object, against the same in 64 bits; then
    the checkpoint of the states, and tokens on it."""
    from leapquant_b200.kernels import make_add_norm, make_gated_norm
    from leapquant_b200.state import LeapQuantState
    H, HV, lens, slots, fresh = 2, 4, [130, 3, 66], [2, 3, 1], [True, False, True]
    T, C, D = sum(lens), 2 * H * K + HV * V, HV * V
    g = torch.Generator().manual_seed(13)
    ssm, _, a, b, A_log, dt_bias = rule_inputs(H, HV, T, 4, 13)
    proj = torch.randn(T, C + HV * V, generator=g).bfloat16().cuda()
    w, bias = (0.5 * torch.randn(C, 4, generator=g)).bfloat16().cuda(), (0.1 * torch.randn(C, generator=g)).bfloat16().cuda()
    conv = torch.randn(4, 3, C, generator=g).bfloat16().cuda()
    gw, nw = (1 + 0.1 * torch.randn(V, generator=g)).bfloat16().cuda(), (1 + 0.1 * torch.randn(D, generator=g)).bfloat16().cuda()
    res = torch.randn(T, D, generator=g).bfloat16().cuda()
    st = LeapQuantState(ssm, H)
    cu, idx, hi = offsets(lens).cuda(), torch.tensor(slots, dtype=torch.int32).cuda(), torch.tensor([not f for f in fresh]).cuda()
    # 64 bits, the bf16 roundings between the operators included (they are what the next one reads)
    S64, c64, act = ssm.double(), conv.double().transpose(1, 2).clone(), torch.zeros(T, C, dtype=torch.float64, device="cuda")
    conv64(proj[:, :C].double(), c64, w.double(), bias.double(), lens, slots, fresh, act)
    o64 = torch.zeros(T, HV, V, dtype=torch.float64, device="cuda")
    rule64(S64, act.bfloat16(), a, b, A_log, dt_bias, H, lens, slots, fresh, o64)
    o = torch.zeros(T, HV, V, dtype=torch.bfloat16, device="cuda")
    st.prefill_conv(ssm, proj[:, :C], conv.transpose(1, 2), w, bias, a, b, A_log, dt_bias, idx, cu, o, hi)
    # an activated row may round the other way where 64 bits and 32 lie on either side of a middle: 2^-8 of a few elements in 10^4,
    # which the rule spreads over the state: a hundredth of 2^-8
    assert float((ssm.double() - S64).norm() / S64.norm()) <= 2.0 ** -8 / 100
    assert float((o.double() - o64).norm() / o64.norm()) <= 2.0 ** -8
    assert torch.equal(conv.transpose(1, 2).double(), c64)
    y, out = torch.empty_like(o), torch.empty(T, D, dtype=torch.bfloat16, device="cuda")
    make_gated_norm(V)(o, proj[:, C:], gw, y)
    make_add_norm(D, scale=0.5)(y.view(T, D), res, nw, out)
    zd, od = proj[:, C:].double().reshape(T, HV, V), o.double()
    yd = od / torch.sqrt((od * od).mean(-1, keepdim=True) + 1e-6) * gw.double() * zd * torch.sigmoid(zd)
    assert float((y.double() - yd).norm() / yd.norm()) <= 2.0 ** -8
    assert bool(torch.isfinite(out).all())
    # the states become checkpoints, and a token on a checkpoint is near a token on the state it was made of (8 bits: 1 %)
    dense = ssm.clone()
    st.quantize(ssm, idx)
    xt = torch.randn(3, C, generator=g).bfloat16().cuda()
    at, bt = a[:3].contiguous(), b[:3].contiguous()
    o8, o32 = (torch.zeros(3, HV, V, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    st.decode(ssm, xt, at, bt, A_log, dt_bias, idx, o8)
    st.decode_dense(dense, xt, at, bt, A_log, dt_bias, idx, o32)
    assert float((o8.double() - o32.double()).norm() / o32.double().norm()) <= 2e-2
    clean()


@gpu
@pytest.mark.parametrize("state", ["fp32", "int8"])
def test_harness_on_own_operators(state):
    """The hybrid model with every operator of its GDN layers from this package: a prompt in one call leaves the states that its tokens
    leave one by one, and generation runs in a CUDA graph.  (Two paths through bf16 layers: they agree to the roundings of a few layers,
    2^-8 each, not to the bit.)"""
    from leapquant_b200.harness import HybridConfig, HybridTP, run_generation
    cfg = HybridConfig(hidden=256, layers=4, gdn_key_heads=2, gdn_value_heads=4, attn_q_heads=2, attn_kv_heads=1, mlp=512, vocab=512, window=16)
    B, T = 3, 75
    dev = torch.device("cuda", 0)
    tokens = torch.randint(0, cfg.vocab, (B, T), generator=torch.Generator().manual_seed(2)).cuda()
    whole = HybridTP(cfg, 0, 1, dev, "fp32", B, T + 2, operators="own")
    whole.prefill(tokens)
    single = HybridTP(cfg, 0, 1, dev, "fp32", B, T + 2, operators="own")
    for t in range(T):
        single.decode_step(tokens[:, t], torch.full((B,), t, dtype=torch.int64, device=dev))
    for l, (p, q) in enumerate(zip(whole.layers, single.layers)):
        if p["kind"] == "gdn":
            for name in ("ssm", "conv"):
                x, y = p[name][1:].double(), q[name][1:].double()
                assert float((x - y).norm() / y.norm()) <= (4 * l + 2) * 2.0 ** -8, (l, name)
            assert float(p["ssm"][0].abs().max()) == 0.0, "the null slot"
    got = run_generation(cfg, state, batch=B, prompt_len=40, new_tokens=20, operators="own")
    assert got["decode_mode"] == "cuda_graph", got["decode_mode"]
    assert all(0 <= i < cfg.vocab for i in got["last_tokens"])
    clean()


# ---- refusals ----
def test_argument_errors_are_codes():
    from leapquant_b200 import _lib
    L = _lib.lib()
    D = lambda **kw: _lib.dims(*[{**dict(NS=8, HV=4, H=2, K=128, V=128, L=0, R=0, SS=4 * 128 * 128), **kw}[n] for n in ("NS", "HV", "H", "K", "V", "L", "R", "SS")])
    one, mis = ctypes.c_void_p(256), ctypes.c_void_p(264)
    C = 2 * 2 * 128 + 4 * 128

    def prefill(d=None, ssm=one, mixed=one, ms=C, a=one, as_=4, b=one, bs=4, A=one, dt=one, cu=one, idx=one, o=one, N=1, T=1):
        return L.lq_gdn_prefill(d or D(), ssm, mixed, ms, a, as_, b, bs, A, dt, cu, idx, None, o, N, T, 0.0, None, 0, None)

    assert prefill(N=0) == 0 and prefill(T=0) == 0 and prefill(N=0, ssm=None) == 0
    assert prefill(N=-1) == -4 and prefill(T=-1) == -4 and prefill(N=1 << 30) == -4
    for k in ("ssm", "mixed", "a", "b", "A", "dt", "cu", "idx", "o"):
        assert prefill(**{k: None}) == -1, k
    assert prefill(d=D(K=64)) == -2 and prefill(d=D(V=64)) == -2 and prefill(d=D(H=3)) == -4 and prefill(d=D(SS=100)) == -4
    assert prefill(d=D(SS=4 * 128 * 128 + 2)) == -3 and prefill(ms=C + 4) == -3 and prefill(ms=C - 8) == -4
    assert prefill(as_=3) == -4 and prefill(bs=3) == -4
    for k in ("ssm", "mixed", "o"):
        assert prefill(**{k: mis}) == -3, k
    rec = lambda N=1, ssm=one, ms=C: L.lq_gdn_recurrent(D(), ssm, one, ms, one, 4, one, 4, one, one, one, one, N, 0.0, None)
    assert rec(N=0) == 0 and rec(N=-1) == -4 and rec(ssm=None) == -1 and rec(ssm=mis) == -3 and rec(ms=C + 1) == -3

    def conv(x=256, xs=64, state=256, sd=1, sp=64, ss=192, w=256, bias=None, width=4, cu=one, idx=one, out=one, os_=64, N=1, T=1, ch=64, NS=4):
        cv = _lib.LqConv1d(x, xs, state, ss, sd, sp, w, bias, width)
        return L.lq_causal_conv1d_prompt(cv, cu, idx, None, N, T, ch, NS, out, os_, None)

    assert conv(N=0) == 0 and conv(T=0) == 0 and conv(N=-1) == -4 and conv(ch=60) == -2 and conv(ch=0) == -4 and conv(width=3) == -2
    assert conv(x=None) == -1 and conv(state=None) == -1 and conv(w=None) == -1 and conv(cu=None) == -1 and conv(out=None) == -1
    assert conv(xs=56) == -4 and conv(os_=56) == -4 and conv(xs=68) == -3 and conv(os_=68) == -3 and conv(x=264) == -3
    assert conv(state=260) == -3 and conv(sp=66) == -3 and conv(ss=194) == -3 and conv(bias=264) == -3 and conv(NS=0) == -4

    gn = lambda o=one, z=one, zs=512, w=one, y=one, T=1, HV=4, V=128: L.lq_gated_norm(o, z, zs, w, y, T, HV, V, 1e-6, None)
    assert gn(T=0) == 0 and gn(T=-1) == -4 and gn(V=64) == -2 and gn(HV=0) == -4 and gn(zs=504) == -4 and gn(zs=516) == -3
    assert gn(o=None) == -1 and gn(y=None) == -1 and gn(o=mis) == -3 and gn(w=mis) == -3
    an = lambda x=one, xs=64, r=one, rs=64, w=one, y=one, ys=64, T=1, D=64: L.lq_add_norm(x, xs, r, rs, w, y, ys, T, D, 1.0, 1e-6, None)
    assert an(T=0) == 0 and an(T=-1) == -4 and an(D=60) == -2 and an(D=0) == -2 and an(D=16392, xs=16392) == -2
    assert an(x=None) == -1 and an(r=None) == -1 and an(xs=56) == -4 and an(ys=68) == -3 and an(r=mis) == -3


def test_overlapping_operands_are_refused():
    """Each call would launch if its operands were apart, and does not."""
    from leapquant_b200 import _lib
    L, P = _lib.lib(), ctypes.c_void_p
    at = lambda i: P((1 << 20) + 2 * i)                      # element i of a buffer that is never read
    far = P(1 << 40)
    d = _lib.dims(8, 4, 2, 128, 128, 0, 0, 4 * 128 * 128)
    C, W, T = 1024, 512, 100
    for k in (0, 512, C - 8, C * (T - 1)):                   # outputs within the rows, in the last row
        assert L.lq_gdn_prefill(d, far, at(0), C, far, 4, far, 4, far, far, far, far, None, at(k), 1, T, 0.0, None, 0, None) == -4, k
        assert L.lq_gdn_recurrent(d, far, at(0), C, far, 4, far, 4, far, far, far, at(k), T, 0.0, None) == -4, k
    assert L.lq_gdn_prefill(d, far, far, C, at(8), 4, far, 4, far, far, far, far, None, at(0), 1, T, 0.0, None, 0, None) == -4
    assert L.lq_gdn_prefill(d, far, far, C, far, 4, at(W * T - 8), 4, far, far, far, far, None, at(0), 1, T, 0.0, None, 0, None) == -4
    for xs, os_, k in ((64, 64, 0), (64, 64, 8), (64, 64, -64), (64, 128, 64 * (T - 1)), (256, 256, 56), (256, 256, 200), (256, 256, -256 - 56)):
        cv = _lib.LqConv1d(at(0), xs, far, 192, 1, 64, far, None, 4)
        assert L.lq_causal_conv1d_prompt(cv, far, far, None, 1, T, 64, 4, at(k), os_, None) == -4, (xs, os_, k)
    gn = lambda o, z, y, zs=W: L.lq_gated_norm(o, z, zs, far, y, T, 4, 128, 1e-6, None)
    assert gn(at(0), far, at(8)) == -4 and gn(at(0), far, at(-W)) == -4 and gn(far, at(0), at(0)) == -4 and gn(far, at(0), at(W), 2 * W) == -4
    an = lambda x, r, y, xs=64, rs=64, ys=64: L.lq_add_norm(x, xs, r, rs, P(1 << 41), y, ys, T, 64, 1.0, 1e-6, None)
    assert an(far, at(0), at(0)) == -4 and an(at(0), far, at(8)) == -4 and an(at(0), far, at(0), xs=128) == -4 and an(at(0), at(8), far) == -4
    assert an(far, at(0), at(64 * 99)) == -4 and an(at(0), at(40), far, xs=128, rs=128) == -4


def test_factories_refuse_shapes_and_host_tensors():
    from leapquant_b200 import _lib, kernels as KN
    with pytest.raises(NotImplementedError):
        KN.make_gdn_prefill(4, 4, 2, 64, 128, 4 * 128 * 128)
    with pytest.raises(NotImplementedError):
        KN.make_gdn_recurrent(4, 4, 2, 128, 64, 4 * 128 * 128)
    with pytest.raises(NotImplementedError):
        KN.make_gated_norm(64)
    for D in (4, 100, 20000):
        with pytest.raises(NotImplementedError):
            KN.make_add_norm(D)
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)
    S = torch.zeros(4, 4, 128, 128)
    for call in (lambda: KN.make_gdn_prefill(4, 4, 2, 128, 128, S.stride(0))(S, bf(3, 1024), bf(3, 4), bf(3, 4), torch.zeros(4), torch.zeros(4), i32(2), i32(1), None, bf(3, 4, 128)),
                 lambda: KN.make_gdn_recurrent(4, 4, 2, 128, 128, S.stride(0))(S, bf(3, 1024), bf(3, 4), bf(3, 4), torch.zeros(4), torch.zeros(4), i32(3), bf(3, 4, 128)),
                 lambda: KN.make_conv1d_prompt(4, 64)(bf(3, 64), bf(4, 64, 3), bf(64, 4), None, i32(2), i32(1), None, bf(3, 64)),
                 lambda: KN.make_gated_norm(128)(bf(3, 4, 128), bf(3, 512), bf(128), bf(3, 4, 128)),
                 lambda: KN.make_add_norm(64)(bf(3, 64), bf(3, 64), bf(64), bf(3, 64))):
        with pytest.raises(_lib.LeapQuantError):
            call()


def test_row_checks():
    from leapquant_b200 import _lib
    bf = torch.bfloat16
    t = torch.zeros(6, 80, dtype=bf)
    assert _lib.rows(t[:, 16:], bf, (6, 64), "t") == 80 and _lib.rows(t[:1, :64], bf, (1, 64), "t") == 64 and _lib.rows(t[:0], bf, (0, 80), "t") == 80
    for bad in (t.float(), t.t(), t[:, ::2], t[:, :40]):
        with pytest.raises(_lib.LeapQuantError):
            _lib.rows(bad, bf, (6, 80), "t")
    with pytest.raises(_lib.LeapQuantError):
        _lib.rows(torch.zeros(6, 160, dtype=bf)[:, ::2], bf, (6, 80), "t")
    with pytest.raises(_lib.LeapQuantError):
        _lib.whole(t[:, :40], bf, (6, 40), "t")


@gpu
def test_refusals_on_the_device():
    from leapquant_b200 import _lib, kernels as KN
    from leapquant_b200.state import LeapQuantState
    ssm, mixed, a, b, A_log, dt_bias = rule_inputs(2, 4, 6, 4, 1)
    o = torch.zeros(6, 4, V, dtype=torch.bfloat16, device="cuda")
    cu, idx = offsets([6]).cuda(), torch.ones(1, dtype=torch.int32, device="cuda")
    f = KN.make_gdn_prefill(4, 4, 2, K, V, ssm.stride(0))
    good = [ssm, mixed, a, b, A_log, dt_bias, cu, idx, None, o]
    f(*good)
    for i, bad in ((0, ssm.bfloat16()), (0, ssm[:3]), (1, mixed.float()), (1, mixed[:, :-128]), (1, mixed[:5]), (2, a[:, :3]), (2, a.float()),
                   (3, b[:5]), (4, A_log.double()), (5, dt_bias[:3]), (6, cu.long()), (6, offsets([3, 3]).cuda()), (7, idx.long()), (8, idx),
                   (8, torch.ones(2, dtype=torch.bool, device="cuda")), (9, o.float()), (9, o[:, :, ::2]), (9, o[:5]), (7, idx.cpu()), (9, o.cpu())):
        args = list(good)
        args[i] = bad
        with pytest.raises(_lib.LeapQuantError):
            f(*args)
    wide = torch.zeros(6, mixed.shape[1] + 4, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(_lib.LeapQuantError):                 # rows that do not start on 16 bytes
        f(ssm, wide[:, 4:], *good[2:])
    st = LeapQuantState(torch.zeros(4, 2, 128, 128, device="cuda"), 2, kda=True)
    with pytest.raises(NotImplementedError):
        st.prefill(*good[:6], idx, cu, o)
    with pytest.raises(NotImplementedError):
        st.decode_dense(*good[:6], idx, o)
    clean()
