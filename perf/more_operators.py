"""The sparse MLP's operators, as measurable cases.

A decoder layer whose MLP is a set of experts runs, for each token,

  route    scores of the router's logits (softmax or sigmoid), a bias that
           balances the experts' load, groups of experts of which some stay, the
           top k, renormalised weights
  experts  each chosen expert's SwiGLU MLP, the sum of the k results by their
           weights, and what is added to it (the shared expert, the residual)
  linear   the shared expert's and other dense products with their epilogue:
           bias, activation (SwiGLU over gate|up rows among them), the sigmoid of
           a gate per row, residual

``run`` computes them in elementary torch operations, or, with ``own``, makes
the calls a user of ``multiplex_amd`` makes.

Hidden sizes are those of this repository's layers (2048, 4096; 12288 for the
MLP between) and odd ones; 256 experts of 512 with 8 a token is the largest set.
Activations and weights are bf16, routing weights float32, indices int32.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False


def listed():
    return [
        # a decode step of half a batch: softmax, eight of 256
        {"name": "route_decode", "kind": "route", "B": 64, "T": 1, "E": 256, "k": 8, "scoring": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "group_best": 1, "renormalize": True, "dtype": "bf16", "pad": False},
        # a long prompt: sigmoid scores, balanced by a bias, four of eight groups
        {"name": "route_prompt", "kind": "route", "B": 1, "T": 8192, "E": 256, "k": 8, "scoring": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "group_best": 2, "renormalize": True, "dtype": "f32", "pad": False},
        # prompts of different lengths in one padded step, an odd number of experts
        {"name": "route_ragged", "kind": "route", "B": 7, "T": 333, "E": 60, "k": 5, "scoring": "softmax", "bias": False,
         "groups": 3, "top_groups": 2, "group_best": 1, "renormalize": False, "dtype": "bf16", "pad": True},
        # one user's decode step: latency
        {"name": "experts_token", "kind": "experts", "N": 1, "layout": "2048x512/256:8", "base": True, "pad": False},
        # a decode step of a full batch: most experts have a row or two
        {"name": "experts_decode", "kind": "experts", "N": 64, "layout": "2048x512/256:8", "base": True, "pad": False},
        # the scheduler's prefill chunk
        {"name": "experts_chunk", "kind": "experts", "N": 512, "layout": "2048x512/256:8", "base": True, "pad": False},
        # a long prompt
        {"name": "experts_prompt", "kind": "experts", "N": 4096, "layout": "2048x512/256:8", "base": True, "pad": False},
        # few experts of odd sizes, some tokens padding
        {"name": "experts_odd", "kind": "experts", "N": 777, "layout": "1096x328/12:3", "base": False, "pad": True},
        # a shared expert's gate|up for one token: latency
        {"name": "linear_token", "kind": "linear", "M": 1, "K": 2048, "N": 512, "act": "swiglu", "bias": False,
         "gate": False, "residual": False},
        # a dense layer's down product and its residual, for a prefill chunk
        {"name": "linear_chunk", "kind": "linear", "M": 512, "K": 12288, "N": 4096, "act": "none", "bias": False,
         "gate": False, "residual": True},
        # a dense layer's gate|up for a long prompt
        {"name": "linear_prompt", "kind": "linear", "M": 4096, "K": 4096, "N": 12288, "act": "swiglu", "bias": False,
         "gate": False, "residual": False},
        # everything at once at odd sizes
        {"name": "linear_odd", "kind": "linear", "M": 333, "K": 1096, "N": 1001, "act": "gelu", "bias": True,
         "gate": True, "residual": True},
    ]


# hidden x inner / experts : experts a token
LAYOUTS = ("2048x512/256:8", "4096x1536/32:4", "2048x768/128:8", "1024x512/64:6", "1096x328/12:3", "1536x1000/8:2")
LARGEST = 6 * 4096 * 8 * 2048 * 512  # operations of experts_prompt


def _layout(case):
    """(hidden, inner, experts, experts a token)"""
    sizes, of = case["layout"].split("/")
    return (*map(int, sizes.split("x")), *map(int, of.split(":")))


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["route", "experts", "experts", "linear", "linear"])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        E = groups * _log(rng, 4, 512 // groups)
        top_groups = rng.randint(1, groups)
        B = _log(rng, 1, 64)
        return {"kind": kind, "B": B, "T": _log(rng, 1, 8192 // B), "E": E,
                "k": rng.randint(1, min(12, E // groups * top_groups)), "scoring": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.choice([False, True]), "groups": groups, "top_groups": top_groups,
                "group_best": rng.choice([1, 2]), "renormalize": rng.choice([False, True]),
                "dtype": rng.choice(["bf16", "f16", "f32"]), "pad": rng.choice([False, True])}
    if kind == "experts":
        layout = rng.choice(LAYOUTS)
        H, I, E, k = _layout({"layout": layout})
        return {"kind": kind, "N": _log(rng, 1, min(4096, LARGEST // (6 * k * H * I))), "layout": layout,
                "base": rng.choice([False, True]), "pad": rng.choice([False, False, True])}
    K, N = 8 * _log(rng, 8, 1536), _log(rng, 64, 12288)
    act = rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh", "swiglu", "swiglu"])
    return {"kind": kind, "M": _log(rng, 1, 4096), "K": K if K * N <= 4096 * 12288 else 8 * (4096 * 12288 // N // 8),
            "N": N, "act": act, "bias": rng.choice([False, True]), "gate": rng.choice([False, False, True]),
            "residual": rng.choice([False, True])}


# ------------------------------------------------------------------ inputs

class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed) * 6151 + 17)

    def n(self, *shape, dtype=torch.bfloat16, scale=1.0, mean=0.0):
        x = torch.randn(*shape, generator=self.g, device="cuda", dtype=torch.float32)
        return x.mul_(scale).add_(mean).to(dtype)

    def counts(self, B, hi):
        """B whole numbers of [0, hi] in random order, spread evenly."""
        u = torch.rand(B, generator=self.g, device="cuda", dtype=torch.float64)
        order = torch.randperm(B, generator=self.g, device="cuda")
        return ((order + u) / B * (hi + 1)).floor().clamp(0, hi).to(torch.int32)


DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _route_state(case, r):
    B, T, E = case["B"], case["T"], case["E"]
    # the router's columns of a product that holds the shared expert's gate too; experts differ in how liked they are
    wide = r.n(B, T, E + 1, dtype=torch.float32, scale=1.3) + r.n(E + 1, dtype=torch.float32, scale=0.5)
    s = {n: case[n] for n in ("k", "scoring", "groups", "top_groups", "group_best", "renormalize")}
    return {**s, "logits": wide.to(DTYPES[case["dtype"]])[..., :E],
            "bias": r.n(E, dtype=torch.float32, scale=0.05) if case["bias"] else None,
            "scale": 2.5 if case["scoring"] == "sigmoid" else 1.0, "n_new": r.counts(B, T) if case["pad"] else None}


def _experts_state(case, r):
    N = case["N"]
    H, I, E, k = _layout(case)
    liked = r.n(N, E, dtype=torch.float32) + r.n(E, dtype=torch.float32, scale=0.4)
    w, at = (liked - liked.amax(-1, keepdim=True)).exp().sort(-1, descending=True)
    w, at = w[:, :k] / w[:, :k].sum(-1, keepdim=True), at[:, :k].to(torch.int32)
    if case["pad"]:  # the last fifth of the tokens is padding
        at[N - N // 5:], w[N - N // 5:] = -1, 0.0
    return {"x": r.n(N, H), "gate_up": r.n(E, 2 * I, H, scale=H ** -0.5), "down": r.n(E, H, I, scale=I ** -0.5),
            "indices": at.contiguous(), "weights": w.contiguous(), "base": r.n(N, H) if case["base"] else None}


def _linear_state(case, r):
    M, K, N, act = case["M"], case["K"], case["N"], case["act"]
    rows = 2 * N if act == "swiglu" else N
    return {"x": r.n(M, K), "weight": r.n(rows, K, scale=K ** -0.5),
            "bias": r.n(rows, scale=0.3) if case["bias"] else None, "act": act,
            # the gate's logits: a column of a wider product
            "gate": r.n(M, 9)[:, 8] if case["gate"] else None, "residual": r.n(M, N) if case["residual"] else None}


def prepare(case, seed):
    r = _Rand(seed)
    make = {"route": _route_state, "experts": _experts_state, "linear": _linear_state}[case["kind"]]
    return {"kind": case["kind"], **make(case, r)}


# ---------------------------------------------------------- the plain forms

def _plain_route(s):
    """In 64 bits: an expert's score may lie next to another's."""
    x, k, G = s["logits"].double(), s["k"], s["groups"]
    B, T, E = x.shape
    if s["scoring"] == "softmax":
        p = (x - x.amax(-1, keepdim=True)).exp()
        p = p / p.sum(-1, keepdim=True)
    else:
        p = 1 / (1 + (-x).exp())
    c = p if s["bias"] is None else p + s["bias"].double()
    if s["top_groups"] < G:
        of = c.view(B, T, G, E // G)
        best = of.sort(-1, descending=True).values[..., : s["group_best"]].sum(-1)
        first = best.sort(dim=-1, descending=True, stable=True).indices[..., : s["top_groups"]]
        stays = torch.zeros_like(best, dtype=torch.bool).scatter_(-1, first, True)
        c = torch.where(stays[..., None], of, -math.inf).view(B, T, E)
    at = c.sort(dim=-1, descending=True, stable=True).indices[..., :k]
    w = p.gather(-1, at)
    if s["renormalize"]:
        w = w / w.sum(-1, keepdim=True)
    w = w * s["scale"]
    if s["n_new"] is not None:
        real = (torch.arange(T, device=x.device) < s["n_new"][:, None])[..., None]
        at, w = torch.where(real, at, -1), torch.where(real, w, 0.0)
    return at.to(torch.int32), w.float()


def _plain_experts(s):
    """The pairs (token, choice) sorted by expert, each expert's padded to whole
    blocks of rows, and one batched product over the blocks."""
    x, at = s["x"].float(), s["indices"].flatten().long()
    (N, H), (E, two, _), P = x.shape, s["gate_up"].shape, at.numel()
    R = 4
    while R < 256 and R * E < P:
        R *= 2
    n_blocks = P // R + min(E, P)
    at = torch.where(at < 0, E, at)  # padding goes behind the last expert
    e, order = at.sort(stable=True)
    counts = torch.zeros(E + 1, dtype=torch.long, device=x.device).scatter_add_(0, at, torch.ones_like(at))
    blocks = (counts + R - 1) // R
    ends = blocks.cumsum(0)
    rank = torch.arange(P, device=x.device) - (counts.cumsum(0) - counts)[e]
    place = torch.where(e < E, (ends - blocks)[e] * R + rank, n_blocks * R)
    of = torch.searchsorted(ends[:E].contiguous(), torch.arange(n_blocks, device=x.device), right=True).clamp(max=E - 1)
    rows = x.new_zeros(n_blocks * R + 1, H)
    rows[place] = x[order // s["indices"].shape[1]]
    h = torch.matmul(rows[:-1].view(n_blocks, R, H), s["gate_up"][of].float().transpose(1, 2).contiguous())
    g, u = h.split(two // 2, -1)
    a = g / (1 + (-g).exp()) * u
    y = torch.matmul(a, s["down"][of].float().transpose(1, 2).contiguous()).view(n_blocks * R, H)
    y = torch.cat([y, y.new_zeros(1, H)])
    back = torch.empty_like(place)
    back[order] = place
    out = (y[back].view(N, -1, H) * s["weights"][..., None]).sum(1)
    if s["base"] is not None:
        out = out + s["base"].float()
    return out.to(torch.bfloat16)


def _plain_linear(s):
    act = s["act"]
    y = torch.matmul(s["x"].float(), s["weight"].float().T)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if act == "swiglu":
        g, u = y.split(y.shape[1] // 2, -1)
        y = g / (1 + (-g).exp()) * u
    elif act == "silu":
        y = y / (1 + (-y).exp())
    elif act == "relu":
        y = y.clamp(min=0)
    elif act == "gelu":
        y = y * 0.5 * (1 + torch.erf(y * 0.5 ** 0.5))
    elif act == "gelu_tanh":
        y = y * 0.5 * (1 + torch.tanh((2 / math.pi) ** 0.5 * (y + 0.044715 * y * y * y)))
    if s["gate"] is not None:
        y = y / (1 + (-s["gate"].float()).exp())[:, None]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(torch.bfloat16)


def _own(s):
    import multiplex_amd as mx

    if s["kind"] == "route":
        return mx.route_experts(s["logits"], s["k"], scoring=s["scoring"], bias=s["bias"], groups=s["groups"],
                                top_groups=s["top_groups"], group_best=s["group_best"], renormalize=s["renormalize"],
                                scale=s["scale"], n_new=s["n_new"])
    if s["kind"] == "experts":
        return mx.expert_mlp(s["x"], s["gate_up"], s["down"], s["indices"], s["weights"], base=s["base"])
    return mx.linear_act(s["x"], s["weight"], bias=s["bias"], activation=None if s["act"] == "none" else s["act"],
                         row_gate=s["gate"], residual=s["residual"])


def run(s):
    if own:
        return _own(s)
    return {"route": _plain_route, "experts": _plain_experts, "linear": _plain_linear}[s["kind"]](s)


# -------------------------------------------------------------------- work

def work(case):
    if case["kind"] == "route":
        tokens = case["B"] * case["T"] / (2 if case["pad"] else 1)
        size = 4 if case["dtype"] == "f32" else 2
        out = case["B"] * case["T"] * case["k"] * 8
        return {"bytes": int(tokens * case["E"] * size + out + (4 * case["E"] if case["bias"] else 0)),
                "flops": int(tokens * case["E"] * 10)}
    if case["kind"] == "experts":
        H, I, E, k = _layout(case)
        N = case["N"]
        real = N - N // 5 if case["pad"] else N
        touched = E * (1 - (1 - k / E) ** real)  # of equally liked experts
        return {"bytes": int(touched * 6 * H * I + (real + N * (2 if case["base"] else 1)) * H * 2 + N * k * 8),
                "flops": 6 * real * k * H * I}
    M, K, N = case["M"], case["K"], case["N"]
    rows = 2 * N if case["act"] == "swiglu" else N
    return {"bytes": 2 * (M * K + rows * K + M * N * (2 if case["residual"] else 1) + (rows if case["bias"] else 0)
                          + (M if case["gate"] else 0)), "flops": 2 * M * K * rows}


# ------------------------------------------------------------------- exact

def _exact_route(case, s):
    """Token by token on the host: scores, then the largest one after the other."""
    B, T, E = s["logits"].shape
    k, G = case["k"], case["groups"]
    x = s["logits"].double().cpu().numpy().reshape(-1, E)
    if case["scoring"] == "softmax":
        z = np.exp(x - x.max(1, keepdims=True))
        score = z / z.sum(1, keepdims=True)
    else:
        score = 1.0 / (1.0 + np.exp(-x))
    order = score.copy()
    if s["bias"] is not None:
        order += s["bias"].double().cpu().numpy()
    rows = np.arange(len(x))
    width = E // G
    if case["top_groups"] < G:
        parts = np.sort(order.reshape(-1, G, width), -1)
        rest = parts[..., -case["group_best"]:].sum(-1)
        allowed = np.zeros((len(x), G), bool)
        for _ in range(case["top_groups"]):
            g = rest.argmax(1)
            allowed[rows, g] = True
            rest[rows, g] = -np.inf
        order[~np.repeat(allowed, width, 1)] = -np.inf
    indices = np.empty((len(x), k), np.int32)
    weights = np.empty((len(x), k))
    for j in range(k):
        best = order.argmax(1)  # the first of equals
        indices[:, j], weights[:, j] = best, score[rows, best]
        order[rows, best] = -np.inf
    if case["renormalize"]:
        weights /= weights.sum(1, keepdims=True)
    weights *= s["scale"]
    if s["n_new"] is not None:
        n_new = s["n_new"].cpu().numpy()
        for b in range(B):
            indices[b * T + n_new[b]: (b + 1) * T] = -1
            weights[b * T + n_new[b]: (b + 1) * T] = 0.0
    return torch.from_numpy(indices.reshape(B, T, k)), torch.from_numpy(weights.reshape(B, T, k))


def _exact_experts(s):
    N, H = s["x"].shape
    out = torch.zeros(N, H, dtype=torch.float64, device="cuda")
    if s["base"] is not None:
        out += s["base"].double()
    for e in range(s["gate_up"].shape[0]):
        token, choice = (s["indices"] == e).nonzero(as_tuple=True)
        if len(token):
            w13, w2 = s["gate_up"][e].double(), s["down"][e].double()
            both = s["x"][token].double() @ w13.T.contiguous()
            n = both.shape[1] // 2
            inner = both[:, :n] * torch.sigmoid(both[:, :n]) * both[:, n:]
            out.index_add_(0, token, inner @ w2.T.contiguous() * s["weights"][token, choice].double()[:, None])
    return out


def _exact_linear(s):
    F = torch.nn.functional
    y = s["x"].double() @ s["weight"].double().T.contiguous()
    if s["bias"] is not None:
        y += s["bias"].double()
    n = s["weight"].shape[0]
    y = {"none": lambda v: v, "relu": torch.relu, "silu": F.silu, "gelu": F.gelu,
         "gelu_tanh": lambda v: F.gelu(v, approximate="tanh"),
         "swiglu": lambda v: F.silu(v[:, : n // 2]) * v[:, n // 2:]}[s["act"]](y)
    if s["gate"] is not None:
        y = y * torch.sigmoid(s["gate"].double())[:, None]
    return y if s["residual"] is None else y + s["residual"].double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "route":
        return _exact_route(case, s)
    return _exact_experts(s) if case["kind"] == "experts" else _exact_linear(s)
