"""What surrounds the decode step of a linear-attention layer, and how it is timed: the operators between the layer's projections.

  prefill   many tokens of packed sequences through the gated delta rule, on the fp32 states of their slots
  dense     one token per row of the same rule
  conv      the causal depthwise convolution (width 4, SiLU) of packed prompts, which produces the rows that `prefill` takes
  gated     RMS norm of every head's output, times its weight, times silu of the layer's gate projection
  add       residual stream plus the scaled output of a block, and the RMS norm that the next block reads

`run` computes an operator from elementary torch operations in 32 bits; with `own` it makes the framework's call instead.
"""
import math
import random

import torch

K = V = 128
TAPS = 4
EPS = 1e-6
own = False

BASE = {"kind": "prefill", "H": 16, "HV": 32, "N": 1, "lo": 1, "hi": 1, "lens_seed": 0, "pad": 0, "fresh": 0.0, "D": 4096, "scale": 1.0}


def _case(**kw):
    return {**BASE, **kw}


def listed():
    return [
        # a few tokens for each of many running sequences: drafted tokens that are verified
        _case(name="prefill_drafts", N=48, lo=2, hi=6, lens_seed=1),
        # one long new prompt: nothing to share the GPU with, the chain of its chunks decides
        _case(name="prefill_prompt_8k", lo=8192, hi=8192, fresh=1.0),
        # a scheduler's mixed batch on one of four tensor-parallel ranks: prompts and pieces of prompts of any length
        _case(name="prefill_ragged_shard", N=37, lo=1, hi=3000, lens_seed=2, H=4, HV=8, fresh=0.5),
        # a whole batch of prompts
        _case(name="prefill_64k", N=16, lo=4096, hi=4096, fresh=0.5),
        # one sequence, one token: all latency
        _case(name="dense_single", kind="dense", H=16, HV=16),
        # the decode batch on fp32 states, padded up as an engine does
        _case(name="dense_256", kind="dense", N=256, pad=11),
        # short prompts, one of them a single token
        _case(name="conv_short", kind="conv", N=3, lo=1, hi=40, lens_seed=3, fresh=0.5),
        # a batch of prompts
        _case(name="conv_32k", kind="conv", N=8, lo=4096, hi=4096, fresh=0.5),
        # a small decode batch, all latency
        _case(name="gated_8", kind="gated", N=8),
        # the output of the rule over a batch of prompts
        _case(name="gated_32k", kind="gated", N=32768),
        # an odd decode batch
        _case(name="add_7", kind="add", N=7),
        # the residual stream of a batch of prompts, branch scaled
        _case(name="add_16k", kind="add", N=16384, scale=0.5),
    ]


def draw(rng):
    """One more case of the same ranges."""
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["prefill", "prefill", "prefill", "dense", "conv", "gated", "add"])
    H, HV = rng.choice([(16, 32), (16, 32), (4, 8), (2, 8), (16, 16), (2, 2), (1, 3)])
    c = _case(kind=kind, H=H, HV=HV)
    if kind in ("prefill", "conv"):
        c["N"] = size(1, 64)
        c["hi"] = size(1, min(12000, 50000 // c["N"]))
        c["lo"] = size(1, c["hi"]) if rng.random() < 0.7 else c["hi"]
        c.update(lens_seed=rng.randrange(1000), fresh=rng.choice([0.0, 0.5, 1.0]), pad=rng.choice([0, 0, 3]))
    elif kind == "dense":
        c.update(N=size(1, 256), pad=rng.choice([0, 0, 5]))
    elif kind == "gated":
        c["N"] = size(1, 24000)
    else:
        c.update(N=size(1, 16000), D=rng.choice([4096, 4096, 2048, 1000, 5120, 520, 128]), scale=rng.choice([1.0, 1.0, 0.5, 0.22]))
    return c


def _lens(c):
    """Tokens of the case's sequences (the padding entries at the end have none)."""
    if c["kind"] == "dense":
        return [1] * c["N"]
    r = random.Random(c["lens_seed"])
    return [int(round(math.exp(r.uniform(math.log(c["lo"]), math.log(c["hi"]))))) for _ in range(c["N"])] + [0] * c["pad"]


# ---------------------------------------------------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c = {**BASE, **case}
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(1_000_003 * (seed % 100_000) + 29)

    def r(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    def u(*shape):
        return torch.rand(*shape, generator=gen, device=dev)

    def b(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.bfloat16)

    H, HV, kind = c["H"], c["HV"], c["kind"]
    s = {"case": c}
    if kind == "gated":
        # o comes out of the rule; z is the last part of the layer's q | k | v | z projection, and stays where it is
        s["o"] = (0.1 * b(c["N"], HV, V))
        C = 2 * H * K + HV * V
        s["z"] = b(c["N"], C + HV * V)[:, C:]
        s["weight"] = (1 + 0.1 * r(V)).to(torch.bfloat16)
        s["out"] = torch.empty(c["N"], HV, V, dtype=torch.bfloat16, device=dev)
        return s
    if kind == "add":
        s["x"], s["residual"] = b(c["N"], c["D"]), b(c["N"], c["D"])
        s["weight"] = (1 + 0.1 * r(c["D"])).to(torch.bfloat16)
        s["out"] = torch.empty(c["N"], c["D"], dtype=torch.bfloat16, device=dev)
        return s
    lens = _lens(c)
    N, T, C = len(lens), sum(lens), 2 * H * K + HV * V
    NS = c["N"] + 1
    s["longest"] = max(lens)
    slots = torch.randperm(NS - 1, generator=gen, device=dev)[:c["N"]].to(torch.int32) + 1
    s["idx"] = torch.cat([slots, torch.zeros(c["pad"], dtype=torch.int32, device=dev)])
    s["cu"] = torch.tensor([0] + lens, device=dev).cumsum(0).to(torch.int32)
    s["has_initial"] = u(N) >= c["fresh"] if kind != "dense" else None
    rows = T + (c["pad"] if kind == "dense" else 0)
    if kind == "conv":
        # the q | k | v part of the q | k | v | z projection, where the projection left it
        s["x"] = b(T, C + HV * V)[:, :C]
        s["conv_state"] = b(NS, TAPS - 1, C).transpose(1, 2)                             # (slot, channel, tap)
        s["weight"], s["bias"] = 0.5 * b(C, TAPS), 0.1 * b(C)
        s["out"] = torch.empty(T, C, dtype=torch.bfloat16, device=dev)
        return s
    s["mixed"] = b(rows, C)
    ba = b(rows, 2 * HV)
    s["b"], s["a"] = ba[:, :HV], ba[:, HV:]                                              # halves of one projection
    s["A_log"] = torch.log(1 + 15 * u(HV))                                               # as such layers are initialised
    s["dt_bias"] = torch.log(torch.expm1(0.001 * 100 ** u(HV)))
    s["ssm"] = 0.1 * r(NS, HV, V, K)
    s["out"] = torch.empty(rows, HV, V, dtype=torch.bfloat16, device=dev)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def _calls(s):
    """The handle of the case's operator, as a program keeps it."""
    if "call" not in s:
        from leapquant_b200 import kernels as KN
        c, ssm = s["case"], s.get("ssm")
        if c["kind"] == "prefill":
            s["call"] = KN.make_gdn_prefill(ssm.shape[0], c["HV"], c["H"], K, V, ssm.stride(0))
        elif c["kind"] == "dense":
            s["call"] = KN.make_gdn_recurrent(ssm.shape[0], c["HV"], c["H"], K, V, ssm.stride(0))
        elif c["kind"] == "conv":
            s["call"] = KN.make_conv1d_prompt(s["conv_state"].shape[0], s["x"].shape[1])
        elif c["kind"] == "gated":
            s["call"] = KN.make_gated_norm(V, eps=EPS)
        else:
            s["call"] = KN.make_add_norm(c["D"], eps=EPS, scale=c["scale"])
    return s["call"]


def run(s):
    kind = s["case"]["kind"]
    if own:
        f = _calls(s)
        if kind == "prefill":
            f(s["ssm"], s["mixed"], s["a"], s["b"], s["A_log"], s["dt_bias"], s["cu"], s["idx"], s["has_initial"], s["out"])
        elif kind == "dense":
            f(s["ssm"], s["mixed"], s["a"], s["b"], s["A_log"], s["dt_bias"], s["idx"], s["out"])
        elif kind == "conv":
            f(s["x"], s["conv_state"], s["weight"], s["bias"], s["cu"], s["idx"], s["has_initial"], s["out"])
        elif kind == "gated":
            f(s["o"], s["z"], s["weight"], s["out"])
        else:
            f(s["x"], s["residual"], s["weight"], s["out"])
    elif kind == "prefill":
        _prefill_plain(s)
    elif kind == "dense":
        _dense_plain(s)
    elif kind == "conv":
        _conv_plain(s)
    elif kind == "gated":
        x, z = s["o"].float(), s["z"].float().view(s["o"].shape)
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["weight"].float() * (z / (1 + torch.exp(-z)))
        s["out"].copy_(y)
    else:
        h = s["residual"].float() + s["case"]["scale"] * s["x"].float()
        s["residual"].copy_(h)
        s["out"].copy_(h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["weight"].float())
    if kind in ("prefill", "dense"):
        return {"o": s["out"], "state": s["ssm"]}
    if kind == "conv":
        return {"out": s["out"], "conv_state": s["conv_state"]}
    return {"out": s["out"], "residual": s["residual"]} if kind == "add" else {"out": s["out"]}


def _rows_plain(s, x, a, b):
    """q^, k^ [..., HV, K], v [..., HV, V] in 32 bits, log decay in 64 and beta in 32, of projected rows x [..., C]."""
    c = s["case"]
    H, HV = c["H"], c["HV"]
    q, k, v = x.float().split([H * K, H * K, HV * V], -1)
    q, k, v = q.unflatten(-1, (H, K)), k.unflatten(-1, (H, K)), v.unflatten(-1, (HV, V))
    q = q * (torch.rsqrt((q * q).sum(-1, keepdim=True) + 1e-6) * K ** -0.5)
    k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    q, k = q.repeat_interleave(HV // H, -2), k.repeat_interleave(HV // H, -2)
    g = -torch.exp(s["A_log"].double()) * torch.log1p(torch.exp(a.double() + s["dt_bias"].double()))
    return q, k, v, g, 1 / (1 + torch.exp(-b.float()))


def _dense_plain(s):
    rows = s["case"]["N"]
    q, k, v, g, beta = _rows_plain(s, s["mixed"][:rows], s["a"][:rows], s["b"][:rows])
    slot = s["idx"][:rows].long()
    S = s["ssm"][slot] * torch.exp(g).float()[..., None, None]
    new = beta[..., None] * (v - (S @ k[..., None])[..., 0])
    S = S + new[..., None] * k[..., None, :]
    s["ssm"][slot] = S
    s["out"][:rows] = (S @ q[..., None])[..., 0].to(torch.bfloat16)
    s["out"][rows:] = 0


def _prefill_plain(s):
    """Chunks of up to 64 tokens, all sequences side by side, the shorter ones filled up with tokens that change nothing."""
    N, longest = s["case"]["N"], s["longest"]
    C = min(64, longest)
    M = -(-longest // C)
    at = torch.arange(M * C, device="cuda")
    start, length = s["cu"][:N].long(), (s["cu"][1:N + 1] - s["cu"][:N]).long()
    live = at < length[:, None]
    token = torch.where(live, start[:, None] + at, 0)
    q, k, v, g, beta = _rows_plain(s, s["mixed"][token], s["a"][token], s["b"][token])
    q, k, v = (t.unflatten(1, (M, C)).permute(1, 0, 3, 2, 4) for t in (q, k, v))        # [M, N, HV, C, 128]
    g, beta = (torch.where(live[..., None], t, 0).unflatten(1, (M, C)).permute(1, 0, 3, 2) for t in (g, beta))
    G = g.cumsum(-1)                                                                    # [M, N, HV, C], 64 bits
    beta = beta[..., None]
    order = at[:C, None] - at[:C]
    decay = torch.where(order >= 0, torch.exp((G[..., :, None] - G[..., None, :]).clamp(max=0)), 0).float()
    L = torch.where(order > 0, beta * decay * (k @ k.mT), 0)
    T = torch.eye(C, device="cuda").expand(L.shape).contiguous()                        # (I + L)^-1, row by row
    for i in range(1, C):
        T[..., i, :i] = -(L[..., i:i + 1, :i] @ T[..., :i, :i])[..., 0, :]
    inner = decay * (q @ k.mT)
    e, left = torch.exp(G).float()[..., None], torch.exp(G[..., -1:] - G).float()[..., None]
    out = torch.empty_like(v)
    slot = s["idx"][:N].long()
    S = torch.where(s["has_initial"][:N, None, None, None], s["ssm"][slot], 0.0)
    for m in range(M):
        new = T[m] @ (beta[m] * (v[m] - e[m] * (k[m] @ S.mT)))
        out[m] = e[m] * (q[m] @ S.mT) + inner[m] @ new
        S = e[m][..., -1:, :] * S + (new * left[m]).mT @ k[m]
    s["ssm"][slot] = S
    s["out"][token[live]] = out.permute(1, 0, 3, 2, 4).flatten(1, 2)[live].to(torch.bfloat16)


def _conv_plain(s):
    N = s["case"]["N"]
    x, state = s["x"].float(), s["conv_state"]
    T, start = x.shape[0], s["cu"][:N].long()
    length = (s["cu"][1:N + 1] - s["cu"][:N]).long()
    slot = s["idx"][:N].long()
    past = torch.where(s["has_initial"][:N, None, None], state[slot].transpose(1, 2).float(), 0.0)      # [N, tap, C]
    seq = torch.repeat_interleave(torch.arange(N, device="cuda"), length, output_size=T)
    at = torch.arange(T, device="cuda") - start[seq]
    w = s["weight"].float()
    y = s["bias"].float() + w[:, 3] * x
    for j in range(3):
        p = at - 3 + j                                                                  # place of tap j in its sequence
        y = y + w[:, j] * torch.where((p >= 0)[:, None], x[(start[seq] + p).clamp(min=0)], past[seq, (3 + p).clamp(max=2)])
    s["out"].copy_(y / (1 + torch.exp(-y)))
    p = length[:, None] - 3 + torch.arange(3, device="cuda")                            # the last three inputs of each sequence
    last = torch.where((p >= 0)[..., None], x[(start[:, None] + p).clamp(min=0)], past.gather(1, (3 + p).clamp(0, 2)[..., None].expand_as(past)))
    state[slot] = last.transpose(1, 2).to(torch.bfloat16)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    c = {**BASE, **case}
    H, HV, N, kind = c["H"], c["HV"], c["N"], c["kind"]
    if kind == "gated":
        return {"bytes": 6 * N * HV * V, "flops": 12 * N * HV * V}
    if kind == "add":
        return {"bytes": 8 * N * c["D"], "flops": 8 * N * c["D"]}
    C, T = 2 * H * K + HV * V, sum(_lens(c))
    fresh = c["fresh"] if kind != "dense" else 0.0
    if kind == "conv":
        return {"bytes": 4 * T * C + 6 * N * C * (2 - fresh) + 10 * C, "flops": 12 * T * C}
    # q, k, v, gates and outputs of every token; a state read and written once; per token S k, the update and S q
    return {"bytes": T * (2 * C + 4 * HV + 2 * HV * V) + 4 * N * HV * K * V * (2 - fresh), "flops": 6 * K * V * HV * T}


# ---------------------------------------------------------------------------------------------------------------------
# the same from the definition, in 64 bits: one token after the other
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["kind"] == "gated":
        o, z = s["o"].double(), s["z"].double().reshape(s["o"].shape)
        return {"out": o / (o.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["weight"].double() * z * torch.sigmoid(z)}
    if c["kind"] == "add":
        h = s["residual"].double() + c["scale"] * s["x"].double()
        return {"out": h / (h.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["weight"].double(), "residual": h}
    N, idx = c["N"], s["idx"][:c["N"]].long()
    first = s["cu"][:N].long() if c["kind"] != "dense" else torch.arange(N, device="cuda")
    n = s["cu"][1:N + 1].long() - first
    keep = s["has_initial"][:N] if s["has_initial"] is not None else torch.ones(N, dtype=torch.bool, device="cuda")
    if c["kind"] == "conv":
        taps = s["conv_state"].double()
        hist = taps[idx] * keep[:, None, None]                                          # [N, C, 3]
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
        for t in range(s["longest"]):
            act = (n > t).nonzero()[:, 0]
            window = torch.cat([hist[act], s["x"][first[act] + t].double()[..., None]], -1)
            y = (window * s["weight"].double()).sum(-1) + s["bias"].double()
            out[first[act] + t] = y * torch.sigmoid(y)
            hist[act] = window[..., 1:]
        taps[idx] = hist
        return {"out": out, "conv_state": taps}
    H, HV = c["H"], c["HV"]
    state = s["ssm"].double()
    S = state[idx] * keep[:, None, None, None]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    A, dt = s["A_log"].double().exp(), s["dt_bias"].double()
    few = bool((n != s["longest"]).any())
    for t in range(s["longest"]):
        act = (n > t).nonzero()[:, 0] if few else slice(None)
        row = first[act] + t
        x = s["mixed"][row].double()
        q = x[:, :H * K].view(-1, H, 1, K).expand(-1, -1, HV // H, -1).reshape(-1, HV, K)
        k = x[:, H * K:2 * H * K].view(-1, H, 1, K).expand(-1, -1, HV // H, -1).reshape(-1, HV, K)
        v = x[:, 2 * H * K:].view(-1, HV, V)
        q = q / (q.pow(2).sum(-1, keepdim=True) + 1e-6).sqrt() / math.sqrt(K)
        k = k / (k.pow(2).sum(-1, keepdim=True) + 1e-6).sqrt()
        alpha = torch.exp(-A * torch.nn.functional.softplus(s["a"][row].double() + dt))
        P = S[act] * alpha[..., None, None] if few else S.mul_(alpha[..., None, None])
        delta = (v - torch.einsum("nhvk,nhk->nhv", P, k)) * torch.sigmoid(s["b"][row].double())[..., None]
        P = P.add_(delta[..., None] * k[..., None, :])
        out[row] = torch.einsum("nhvk,nhk->nhv", P, q)
        if few:
            S[act] = P
    state[idx] = S
    return {"o": out, "state": state}
