"""The sparse MLP's operators on the GPU against the float64 oracle
(``oracle/experts.py``): routing (indices exactly), dense products with an
epilogue, the experts' products, then the layers that run them together.

Tolerances are per element.  u = 2^-8 is the most that a rounding to bf16 is off,
relative to the value.  A product of bf16 values is exact in fp32, and a sum of K of
them formed in any order is off by at most K 2^-23 sum |x w| (2^-24 an addition,
twice that for a matrix unit that truncates), which ``_sums`` gives.

* linear_act: the sums' error through the activation (its slope is at most 1.13;
  for SwiGLU that of either factor times the other one), 2^-20 of its value for the
  exponentials and reciprocals (1 ulp each, and the argument's rounding), then u.
* expert_mlp: an inner value is off by u of itself and by its sums' error, which
  reach the result through |D|; each expert's result is off by up to 2^-12 of the
  largest of its four neighbouring columns (they wait as multiples of one power of
  two), and the output by u of itself.
* routing: one rounding to fp32, 2^-24, and as much again for the 64-bit part.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import multiplex_amd as mx
from oracle import experts as ox

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -8


def _np(t):
    return None if t is None else t.double().cpu().numpy()


def _r(g, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _sums(x, w):
    return x.shape[-1] * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T)


def _within(y, ref, tol):
    y = _np(y)
    assert y.shape == ref.shape
    fine = np.isfinite(ref)
    assert np.array_equal(fine, np.isfinite(y))
    assert np.array_equal(np.isnan(ref), np.isnan(y))
    over = np.abs(y - ref)[fine] - np.broadcast_to(tol, ref.shape)[fine]
    assert over.size == 0 or over.max() <= 0, f"off by {over.max():.3g} more than allowed"


def _check_linear(y, x, w, bias, act, gate, res):
    x, w, bias, gate, res = map(_np, (x, w, bias, gate, res))
    x2 = x.reshape(-1, x.shape[-1])
    ref = ox.linear_act(x, w, bias, act, gate, res)
    e = _sums(x2, w)
    s = x2 @ w.T
    if bias is not None:
        e = e + 2.0 ** -23 * (np.abs(s) + np.abs(bias))
        s = s + bias
    if act == "swiglu":
        n = w.shape[0] // 2
        g, up = s[:, :n], s[:, n:]
        value = ox.silu(g) * up
        e = 1.13 * e[:, :n] * (np.abs(up) + e[:, n:]) + np.abs(ox.silu(g)) * e[:, n:]
    else:
        value = ox.ACTIVATIONS[act](s)
        e = 1.13 * e + (2.0 ** -20 * np.abs(s) if act == "gelu" else 0)
    tol = e.reshape(ref.shape) + 2.0 ** -20 * np.abs(value).reshape(ref.shape) + U * np.abs(ref) + 1e-30
    _within(y, ref, tol)


# ------------------------------------------------------------- linear_act

SIZES = [(1, 1, 8), (1, 16, 64), (1, 512, 2048), (2, 33, 520), (3, 100, 1096), (4, 257, 72), (5, 7, 24), (16, 128, 64),
         (17, 130, 72), (31, 66, 1000), (64, 64, 128), (65, 129, 136), (130, 257, 200), (300, 520, 1096), (513, 260, 64)]
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh", "swiglu"]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear_act(M, N, K, act):
    g = _gen(M * 7 + N)
    rows = 2 * N if act == "swiglu" else N
    full = (M + N) % 2 == 0
    x, w = _r(g, M, K), _r(g, rows, K, scale=K ** -0.5)
    bias = _r(g, rows, dtype=[torch.bfloat16, torch.float32, torch.float16][M % 3]) if full else None
    gate = _r(g, M, dtype=[torch.float32, torch.bfloat16][M % 2]) if full or act is None else None
    res = _r(g, M, N) if full else None
    y = mx.linear_act(x, w, bias=bias, activation=act, row_gate=gate, residual=res)
    _check_linear(y, x, w, bias, act, gate, res)


@pytest.mark.parametrize("act", [None, "gelu", "swiglu"])
@pytest.mark.parametrize("M,N,K", [(600, 1000, 8200), (64, 1026, 8192), (130, 517, 12296)])
def test_linear_act_in_slices(M, N, K, act):
    """Sizes whose K is summed in slices, through a workspace that holds NaN."""
    need = mx.linear_act_workspace_bytes(M, N, K, act)
    if not need:
        pytest.skip("no slices at this size")
    g = _gen(K)
    rows = 2 * N if act == "swiglu" else N
    x, w = _r(g, M, K), _r(g, rows, K, scale=K ** -0.5)
    bias, gate, res = _r(g, rows), _r(g, M, dtype=torch.float32), _r(g, M, N)
    ws = torch.full((need + 16,), 0xff, dtype=torch.uint8, device=DEV)
    y = mx.linear_act(x, w, bias=bias, activation=act, row_gate=gate, residual=res, workspace=ws)
    _check_linear(y, x, w, bias, act, gate, res)
    assert (ws[need:] == 0xff).all()
    assert torch.equal(y, mx.linear_act(x, w, bias=bias, activation=act, row_gate=gate, residual=res, workspace=ws[:16]))
    _check_linear(mx.linear_act(x, w, activation=act), x, w, None, act, None, None)


@pytest.mark.parametrize("M", [1, 3, 40, 400])
@pytest.mark.parametrize("act", [None, "swiglu"])
def test_linear_act_strided(M, act):
    """Column slices: what lies beside them, NaN, is not read; out's neighbours stay."""
    g = _gen(M)
    K, N = 328, 96
    wide = torch.full((2, M, K + 16), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[..., 8:8 + K] = _r(g, 2, M, K)
    x = wide[..., 8:8 + K]
    w = _r(g, 2 * N if act else N, K, scale=K ** -0.5)
    gates = torch.full((2, M, 3), float("nan"), device=DEV)
    gates[..., 1] = _r(g, 2, M, dtype=torch.float32)
    res = torch.full((2, M, N + 5), float("nan"), dtype=torch.bfloat16, device=DEV)
    res[..., 3:3 + N] = _r(g, 2, M, N)
    out = torch.full((2, M, N + 7), 7.0, dtype=torch.bfloat16, device=DEV)
    y = mx.linear_act(x, w, activation=act, row_gate=gates[..., 1], residual=res[..., 3:3 + N], out=out[..., 2:2 + N])
    assert y.data_ptr() == out[..., 2:2 + N].data_ptr()
    _check_linear(y, x, w, None, act, gates[..., 1], res[..., 3:3 + N])
    assert (out[..., :2] == 7).all() and (out[..., 2 + N:] == 7).all()


@pytest.mark.parametrize("M", [2, 80])
def test_linear_act_odd_layouts(M):
    """Rows that are no multiple of 16 bytes apart, transposed x and residual, an offset weight: copied, not refused."""
    g = _gen(5)
    K, N = 40, 24
    x = _r(g, K, M).T
    w = _r(g, N * K + 1)[1:].view(N, K)
    res = _r(g, N, M).T
    _check_linear(mx.linear_act(x, w, residual=res), x, w, None, None, None, res)
    x = _r(g, M, K + 1)[:, 1:]
    _check_linear(mx.linear_act(x, w, residual=res), x, w, None, None, None, res)


@pytest.mark.parametrize("M", [1, 4, 70, 300])
def test_linear_act_over_its_residual(M):
    g = _gen(9)
    x, w, res = _r(g, M, 136), _r(g, 72, 136, scale=0.1), _r(g, M, 72)
    want = mx.linear_act(x, w, residual=res)
    assert mx.linear_act(x, w, residual=res, out=res) is res
    assert torch.equal(res, want)


@pytest.mark.parametrize("M", [3, 40, 300])
@pytest.mark.parametrize("K", [64, 200])
def test_linear_act_nonfinite_stays_in_its_row(M, K):
    g = _gen(K)
    x, w = _r(g, M, K), _r(g, 50, K)
    clean = mx.linear_act(x, w)
    bad = x.clone()
    bad[1, 3], bad[2, K - 1] = float("nan"), float("inf")
    y = mx.linear_act(bad, w)
    assert torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any()
    keep = [i for i in range(M) if i not in (1, 2)]
    assert torch.equal(y[keep], clean[keep])
    w[7, 5] = float("inf")
    y = mx.linear_act(x, w)
    cols = [i for i in range(50) if i != 7]
    assert torch.equal(y[:, cols], clean[:, cols]) and not torch.isfinite(y[:, 7]).any()


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh", "swiglu"])
def test_linear_act_extremes(act):
    """Activations far out, at zero, and of NaN."""
    v = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 4.0, -4.0, 90.0, -90.0, 3e4, -3e4, float("inf"), float("nan")])
    x = torch.zeros(len(v), 8, dtype=torch.bfloat16, device=DEV)
    x[:, 0] = v.to(DEV)
    w = torch.zeros(16 if act == "swiglu" else 8, 8, dtype=torch.bfloat16, device=DEV)
    w[0, 0] = 1
    if act == "swiglu":
        w[8, 1] = 1
        x[:, 1] = 2
    y = _np(mx.linear_act(x, w, activation=act))[:, 0]
    xv = _np(x)[:, 0]
    with np.errstate(all="ignore"):  # (an infinite gate's up is inf * 0 + 2: NaN)
        ref = ox.linear_act(_np(x), _np(w), None, act)[:, 0]
    assert np.array_equal(np.isnan(ref), np.isnan(y)) and np.array_equal(np.isinf(ref), np.isinf(y))
    fine = np.isfinite(ref)
    # a sigmoid below 2^-126, fp32's smallest normal number, comes out as 0 (1 / (1 + exp(90)) = 8e-40 does): off by
    # less than 2^-126 times what it multiplies, at most 2 x
    tiny = 2.0 ** -125 * np.abs(xv[fine]) + 1e-38
    tol = (U + 2.0 ** -20) * np.abs(ref[fine]) + 2.0 ** -20 * np.abs(xv[fine]) * (act == "gelu") + tiny
    assert (np.abs(y[fine] - ref[fine]) <= tol).all()


def test_linear_act_empty():
    w = _r(_gen(0), 16, 8)
    assert mx.linear_act(torch.empty(0, 8, dtype=torch.bfloat16, device=DEV), w).shape == (0, 16)
    assert mx.linear_act(torch.empty(3, 0, 8, dtype=torch.bfloat16, device=DEV), w, activation="swiglu").shape == (3, 0, 8)


# --------------------------------------------------------------- routing

def _check_route(got, logits, k, n_new=None, **kw):
    indices, weights = got
    E = logits.shape[-1]
    l = _np(logits).reshape(-1, E)
    bias = kw.pop("bias", None)
    ri, rw = ox.route(l, k, bias=None if bias is None else _np(bias), **kw)
    if n_new is not None:
        real = (np.arange(logits.shape[1]) < _np(n_new)[:, None]).reshape(-1)
        ri[~real], rw[~real] = -1, 0
    assert indices.dtype is torch.int32 and weights.dtype is torch.float32
    assert tuple(indices.shape) == tuple(logits.shape[:-1]) + (k,)
    assert np.array_equal(indices.cpu().numpy().reshape(-1, k), ri)
    _within(weights.reshape(-1, k), rw, 2.0 ** -23 * np.abs(np.where(np.isfinite(rw), rw, 0)) + 1e-45)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("N,E,k", [(1, 1, 1), (1, 256, 8), (3, 7, 7), (65, 64, 6), (130, 65, 4), (33, 257, 10),
                                   (5, 512, 16), (2, 1024, 64), (9, 100, 33), (700, 128, 8), (2100, 60, 4)])
def test_route(N, E, k, scoring, dtype):
    g = _gen(N + E)
    logits = _r(g, N, E, dtype=dtype, scale=1.5)
    kw = dict(scoring=scoring, renormalize=E % 2 == 0, scale=2.5 if N % 2 else 1.0)
    _check_route(mx.route_experts(logits, k, **kw), logits, k, **kw)
    bias = _r(g, E, dtype=torch.float32, scale=0.1)
    _check_route(mx.route_experts(logits, k, bias=bias, **kw), logits, k, bias=bias, **kw)


@pytest.mark.parametrize("N", [5, 1030])
@pytest.mark.parametrize("E,groups,top_groups,group_best,k", [(256, 8, 4, 2, 8), (64, 8, 1, 1, 8), (60, 3, 2, 2, 12),
                                                              (64, 64, 5, 2, 5), (1024, 16, 3, 1, 32), (12, 4, 4, 2, 3),
                                                              (130, 5, 2, 2, 20), (10, 2, 1, 2, 5)])
def test_route_groups(E, groups, top_groups, group_best, k, N):
    g = _gen(E)
    logits = _r(g, N, E, dtype=torch.float32)
    bias = _r(g, E, dtype=torch.float32, scale=0.1)
    for scoring in ("softmax", "sigmoid"):
        kw = dict(scoring=scoring, bias=bias, groups=groups, top_groups=top_groups, group_best=group_best)
        _check_route(mx.route_experts(logits, k, **kw), logits, k, **kw)


@pytest.mark.parametrize("E", [16, 256, 300])
@pytest.mark.parametrize("N", [6, 1200])
def test_route_ties_and_nonfinite(E, N):
    """Equal scores go to the lowest index; NaN is chosen last; a row of -inf has weights 0."""
    g = _gen(E)
    logits = torch.randint(-2, 3, (N, E), generator=g).float().to(DEV)  # few values: many ties
    k = 6
    for scoring in ("softmax", "sigmoid"):
        _check_route(mx.route_experts(logits, k, scoring=scoring), logits, k, scoring=scoring)
    logits[0] = 1.5
    logits[1] = float("-inf")
    logits[2, 3:] = float("-inf")
    logits[3, 2], logits[3, 5] = float("nan"), float("nan")
    logits[4] = float("nan")
    logits[5, 4] = float("inf")
    for scoring in ("softmax", "sigmoid"):
        for groups in (1, 2):
            kw = dict(scoring=scoring, groups=groups)
            _check_route(mx.route_experts(logits, k, **kw), logits, k, **kw)
    _check_route(mx.route_experts(logits[1:2], k, renormalize=False), logits[1:2], k, renormalize=False)


@pytest.mark.parametrize("B,T,E", [(1, 1, 8), (5, 3, 60), (7, 333, 60), (64, 17, 256)])
def test_route_padded(B, T, E):
    g = _gen(B)
    wide = torch.full((B, T, E + 3), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[..., 1:1 + E] = _r(g, B, T, E)
    logits = wide[..., 1:1 + E]
    n_new = torch.randint(-1, T + 2, (B,), generator=g).to(torch.int32).to(DEV)
    _check_route(mx.route_experts(logits, 4, n_new=n_new), logits, 4, n_new=n_new)


def test_route_layouts():
    g = _gen(2)
    t = _r(g, 12, 5, 4, dtype=torch.float32).permute(2, 1, 0)  # rows of stride
    _check_route(mx.route_experts(t, 3), t.contiguous(), 3)
    i, w = mx.route_experts(_r(g, 0, 8), 2)
    assert i.shape == (0, 2) and w.shape == (0, 2)
    i, w = mx.route_experts(_r(g, 9)[None, None], 2)
    assert i.shape == (1, 1, 2)


# --------------------------------------------------------------- experts

def _experts(g, N, H, I, E, k, base=False):
    x = _r(g, N, H)
    gate_up, down = _r(g, E, 2 * I, H, scale=H ** -0.5), _r(g, E, H, I, scale=I ** -0.5)
    indices = torch.rand(N, E, generator=g).argsort(-1)[:, :k].to(torch.int32).to(DEV).contiguous()
    weights = torch.rand(N, k, generator=g).to(DEV)
    return x, gate_up, down, indices, weights, _r(g, N, H) if base else None


def _check_experts(y, x, gate_up, down, indices, weights, base):
    x, gate_up, down, weights, base = map(_np, (x, gate_up, down, weights, base))
    indices = indices.cpu().numpy()
    E, H, I = down.shape
    ref = np.zeros_like(x) if base is None else base.copy()
    tol = np.full_like(ref, 1e-36) + 2.0 ** -23 * np.abs(ref)
    for e in np.unique(indices):
        if not 0 <= e < E:
            continue
        t, j = np.nonzero(indices == e)
        s, es = x[t] @ gate_up[e].T, _sums(x[t], gate_up[e])
        g, up = s[:, :I], s[:, I:]
        a = ox.silu(g) * up
        ea = 1.13 * es[:, :I] * (np.abs(up) + es[:, I:]) + np.abs(ox.silu(g)) * es[:, I:] + (U + 2.0 ** -20) * np.abs(a)
        r = a @ down[e].T
        er = ea @ np.abs(down[e]).T + _sums(np.abs(a) + ea, down[e])
        er += 2.0 ** -12 * np.repeat((np.abs(r) + er).reshape(len(t), -1, 4).max(-1), 4, -1)
        w = weights[t, j][:, None]
        np.add.at(ref, t, w * r)
        np.add.at(tol, t, np.abs(w) * er + 2.0 ** -22 * np.abs(w * r))
    _within(y, ref, tol + U * (np.abs(ref) + tol))


EXPERTS = [(1, 8, 8, 1, 1), (1, 64, 32, 4, 2), (1, 1096, 328, 12, 3), (2, 512, 200, 64, 8), (3, 72, 40, 5, 5), (7, 2048, 512, 16, 8),
           (33, 136, 72, 3, 2), (64, 256, 128, 16, 4), (130, 264, 136, 2, 2), (200, 264, 136, 4, 1), (500, 200, 264, 3, 3),
           (1500, 64, 32, 9, 3), (3000, 72, 24, 100, 3)]


@pytest.mark.parametrize("base", [False, True])
@pytest.mark.parametrize("N,H,I,E,k", EXPERTS)
def test_expert_mlp(N, H, I, E, k, base):
    args = _experts(_gen(N + H), N, H, I, E, k, base)
    y = mx.expert_mlp(*args[:5], base=args[5])
    _check_experts(y, *args)
    assert torch.equal(y, mx.expert_mlp(*args[:5], base=args[5]))  # whatever order the pairs came in


# rows of 128 and of 256 a tile; 157 MB of weights, which pass by the caches, in tiles of 64 and of 128
@pytest.mark.parametrize("N,H,I,E,k", [(2048, 72, 1000, 8, 2), (4096, 72, 1000, 8, 2), (200, 512, 200, 256, 6),
                                       (1400, 512, 200, 256, 6)])
def test_expert_mlp_other_tiles(N, H, I, E, k):
    args = _experts(_gen(N), N, H, I, E, k, True)
    args[3][N - 5:] = -1
    _check_experts(mx.expert_mlp(*args[:5], base=args[5]), *args)


@pytest.mark.parametrize("N", [1, 4, 50, 700])
def test_expert_mlp_choices(N):
    """Choices outside the experts add nothing, doubled ones add twice, tokens may have none."""
    g = _gen(N)
    x, gate_up, down, indices, weights, base = _experts(g, N, 136, 72, 6, 4, True)
    indices[:, 2] = indices[:, 0]
    indices[0, 1], indices[N // 2, 3], indices[N - 1] = -1, 6, torch.tensor([-1, 1 << 30, -(1 << 31), 99], device=DEV)
    weights[N - 1] = float("nan")  # of no expert: not used
    y = mx.expert_mlp(x, gate_up, down, indices, weights, base=base)
    _check_experts(y, x, gate_up, down, indices, torch.where(torch.isnan(weights), 0.0, weights), base)
    assert torch.equal(y[N - 1], base[N - 1])
    assert (mx.expert_mlp(x, gate_up, down, indices, weights)[N - 1] == 0).all()
    none = torch.full_like(indices, -1)
    assert torch.equal(mx.expert_mlp(x, gate_up, down, none, weights, base=base), base)


@pytest.mark.parametrize("N", [70, 900])
def test_expert_mlp_all_tokens_to_one(N):
    x, gate_up, down, indices, weights, _ = _experts(_gen(3), N, 264, 136, 40, 1)
    indices.fill_(37)
    _check_experts(mx.expert_mlp(x, gate_up, down, indices, weights), x, gate_up, down, indices, weights, None)


@pytest.mark.parametrize("N", [3, 30, 600])
def test_expert_mlp_nonfinite_stays_in_its_token(N):
    x, gate_up, down, indices, weights, _ = _experts(_gen(4), N, 136, 72, 4, 2)
    clean = mx.expert_mlp(x, gate_up, down, indices, weights)
    bad = x.clone()
    bad[1] = float("nan")
    y = mx.expert_mlp(bad, gate_up, down, indices, weights)
    keep = [i for i in range(N) if i != 1]
    assert torch.isnan(y[1]).all() and torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("N", [2, 60, 600])
def test_expert_mlp_nonfinite_weights_stay_in_their_column(N):
    """A column of inf or NaN beside others, which are as without."""
    x, gate_up, down, indices, weights, _ = _experts(_gen(5), N, 136, 72, 4, 2)
    clean = mx.expert_mlp(x, gate_up, down, indices, weights)
    bad = down.clone()
    bad[:, 9, 3], bad[:, 70, 0] = float("inf"), float("nan")
    y = mx.expert_mlp(x, gate_up, bad, indices, weights)
    assert not torch.isfinite(y[:, 9]).any() and torch.isnan(y[:, 70]).all()
    y[:, [9, 70]] = clean[:, [9, 70]]
    _check_experts(y, x, gate_up, down, indices, weights, None)


@pytest.mark.parametrize("scale", [1e-30, 1e-18, 1e18, 1e30])
@pytest.mark.parametrize("N", [3, 500])
def test_expert_mlp_far_magnitudes(N, scale):
    """Results near both ends of bf16's range."""
    x, gate_up, down, indices, weights, _ = _experts(_gen(6), N, 136, 72, 4, 2)
    down = (down.float() * scale).bfloat16()
    _check_experts(mx.expert_mlp(x, gate_up, down, indices, weights), x, gate_up, down, indices, weights, None)


@pytest.mark.parametrize("N", [2, 90])
def test_expert_mlp_layouts(N):
    """Strided rows, a workspace of one's own full of NaN, the output over the base."""
    g = _gen(8)
    x, gate_up, down, indices, weights, base = _experts(g, N, 136, 72, 6, 2, True)
    want = mx.expert_mlp(x, gate_up, down, indices, weights, base=base)
    wide = torch.full((N, 160), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 16:152] = x
    ws = torch.full((mx.expert_mlp_workspace_bytes(N, 136, 72, 6, 2) + 64,), 0xff, dtype=torch.uint8, device=DEV)
    out = torch.full((N, 144), 7.0, dtype=torch.bfloat16, device=DEV)
    got = mx.expert_mlp(wide[:, 16:152], gate_up, down, indices, weights, base=base, out=out[:, :136], workspace=ws)
    assert torch.equal(got, want) and (out[:, 136:] == 7).all()
    got = mx.expert_mlp(x.T.contiguous().T, gate_up, down, indices.T.contiguous().T, weights.T.contiguous().T,
                        base=base.T.contiguous().T)
    assert torch.equal(got, want)
    assert mx.expert_mlp(x, gate_up, down, indices, weights, base=base, out=base) is base
    assert torch.equal(base, want)


def test_expert_mlp_empty():
    x, gate_up, down, indices, weights, _ = _experts(_gen(1), 4, 16, 8, 2, 1)
    assert mx.expert_mlp(x[:0], gate_up, down, indices[:0], weights[:0]).shape == (0, 16)


# ------------------------------------------------------------- together

def _args(**kw):
    a = dict(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=128, intermediate_size=0,
             num_experts=24, num_experts_per_tok=4, moe_intermediate_size=72, shared_expert_intermediate_size=136)
    return mx.AttentionArgs(**{**a, **kw})


def _check_block(m, x, y, residual=None, n_new=None):
    """Each operator of the block on what the one before gave it."""
    a, H = m.args, m.args.hidden_size
    x2 = x.reshape(-1, H)
    both = mx.linear_act(x2, m.router)
    _check_linear(both, x2, m.router, None, None, None, None)
    kw = dict(scoring=a.scoring_func, groups=a.n_group, top_groups=a.topk_group, renormalize=a.norm_topk_prob,
              scale=a.routed_scaling_factor, bias=m.router_bias)
    indices, weights = mx.route_experts(both[:, : m.E], a.num_experts_per_tok, **kw)
    _check_route((indices, weights), both[:, : m.E], a.num_experts_per_tok, **kw)
    if n_new is not None:
        pad = (torch.arange(x.shape[1], device=DEV) >= n_new[:, None]).reshape(-1)
        indices[pad], weights[pad] = -1, 0
    base = None if residual is None else residual.reshape(-1, H)
    if m.shared_down_proj is not None:
        s = mx.linear_act(x2, m.shared_gate_up_proj, activation="swiglu")
        _check_linear(s, x2, m.shared_gate_up_proj, None, "swiglu", None, None)
        r = mx.linear_act(s, m.shared_down_proj, row_gate=both[:, m.E], residual=base)
        _check_linear(r, s, m.shared_down_proj, None, None, both[:, m.E], base)
        base = r
    _check_experts(y.reshape(-1, H), x2, m.gate_up_proj, m.down_proj, indices, weights, base)


@pytest.mark.parametrize("kw", [dict(), dict(shared_expert_intermediate_size=0, norm_topk_prob=False),
                                dict(scoring_func="sigmoid", n_group=4, topk_group=2, routed_scaling_factor=2.446, router_bias=True)])
@pytest.mark.parametrize("B,T", [(1, 1), (3, 2), (2, 70)])
def test_sparse_mlp(B, T, kw):
    torch.manual_seed(1)
    m = mx.SparseMLP(_args(**kw), DEV)
    if "n_group" in kw:
        m.router_bias.copy_(torch.randn(24, device=DEV) * 0.1)
    x, res = torch.randn(B, T, 256, device=DEV).bfloat16(), torch.randn(B, T, 256, device=DEV).bfloat16()
    kept = res.clone()
    _check_block(m, x, m(x))
    _check_block(m, x, m(x, residual=res), residual=res)
    assert torch.equal(res, kept)
    n_new = torch.arange(B, dtype=torch.int32, device=DEV) % (T + 1)
    _check_block(m, x, m(x, residual=res, n_new=n_new), residual=res, n_new=n_new)


def test_sparse_mlp_loads_separate_weights():
    g = _gen(6)
    H, E, I, S = 256, 24, 72, 136
    m = mx.SparseMLP(_args(), DEV)
    gate, wg, wu, wd = _r(g, E, H), _r(g, E, I, H), _r(g, E, I, H), _r(g, E, H, I)
    sg, su, sd, sgate = _r(g, S, H), _r(g, S, H), _r(g, H, S), _r(g, 1, H)
    m.load(gate, wg, wu, wd, sg, su, sd, sgate)
    assert torch.equal(m.router, torch.cat([gate, sgate])) and torch.equal(m.gate_up_proj[:, I:], wu)
    assert torch.equal(m.shared_gate_up_proj[:S], sg) and torch.equal(m.down_proj, wd)
    with pytest.raises(ValueError):
        m.load(gate, wg, wu, wd)


def test_sparse_mlp_in_a_graph():
    """Captured once, replayed on new inputs with eager work between."""
    torch.manual_seed(2)
    m = mx.SparseMLP(_args(), DEV)
    x = torch.randn(2, 9, 256, device=DEV).bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m(x)
    for i in range(4):
        x.copy_(torch.randn(2, 9, 256, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        want = m(x)
        assert torch.equal(got, want)


def test_expert_mlp_in_two_graphs():
    """Graphs with workspaces of their own, captured and replayed in turn, and with eager calls between."""
    args = _experts(_gen(12), 40, 264, 136, 12, 3, True)
    few = _experts(_gen(13), 2, 264, 136, 12, 3, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a in (args, few):
            mx.expert_mlp(*a[:5], base=a[5])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for a in (args, few):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(mx.expert_mlp(*a[:5], base=a[5]))
        graphs.append(g)
    for i in range(3):
        for a, g in zip((args, few), graphs):
            a[0].copy_(torch.randn(a[0].shape, device=DEV))
            a[3].copy_(torch.rand(a[0].shape[0], 12, device=DEV).argsort(-1)[:, :3])
            g.replay()
        torch.cuda.synchronize()
        for a, o in zip((args, few), outs):
            got = o.clone()
            assert torch.equal(got, mx.expert_mlp(*a[:5], base=a[5]))


def test_gradients_are_refused():
    """On the calls' short way too; without recording they run."""
    g = _gen(15)
    x, w = _r(g, 4, 136), _r(g, 24, 136)
    a = _experts(g, 4, 136, 72, 6, 2)
    logits = _r(g, 4, 16, dtype=torch.float32)
    calls = [lambda: mx.linear_act(x.requires_grad_(), w), lambda: mx.route_experts(logits.requires_grad_(), 2),
             lambda: mx.expert_mlp(*a[:4], a[4].requires_grad_())]
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            call()


def test_one_row_tensors():
    """x of one dimension, as a row."""
    g = _gen(14)
    x, w = _r(g, 136), _r(g, 24, 136)
    y = mx.linear_act(x, w)
    assert y.shape == (24,) and torch.equal(y, mx.linear_act(x[None], w)[0])
    i, wt = mx.route_experts(y, 2)
    assert i.shape == (2,) and torch.equal(i, mx.route_experts(y[None], 2)[0][0])
    a = _experts(g, 1, 136, 72, 6, 2)
    assert torch.equal(mx.expert_mlp(a[0][0], *a[1:3], a[3][0], a[4][0]), mx.expert_mlp(*a[:5])[0])


def test_calls_on_two_streams():
    args = _experts(_gen(11), 90, 264, 136, 12, 3, True)
    want = mx.expert_mlp(*args[:5], base=args[5])
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        s = streams[i % 2]
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(mx.expert_mlp(*args[:5], base=args[5]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("paged", [False, True])
def test_layers_with_a_sparse_mlp(paged):
    """A decoder layer's step against the parts it is made of, and a draft head's over it."""
    torch.manual_seed(4)
    a = _args()
    layer = mx.DecoderLayer(a, DEV)
    m = layer.mlp
    assert isinstance(m, mx.SparseMLP)
    x = torch.randn(2, 5, 256, device=DEV).bfloat16()

    def cache():
        return mx.PagedKVCache(mx.BlockPool(16, 2, 128, device=DEV), 2) if paged else mx.KVCache(2, 2, 128, 64, DEV)

    for n_new in [None, [5, 2]][: 1 + paged]:
        y = layer(x, cache(), n_new=n_new)
        h, mlp = layer.forward_parts(x, None, cache(), n_new)
        h2, z, counts = layer._attend(x, None, cache(), n_new)
        assert torch.equal(h, h2)
        gate = mx.linear_act(z, m.router)[..., m.E]
        s = mx.linear_act(z, m.shared_gate_up_proj, activation="swiglu")
        shared = mx.linear_act(s, m.shared_down_proj, row_gate=gate).float()
        # y = round(round(shared + h) + experts), mlp = round(round(shared) + experts)
        tol = 1.01 * U * ((shared + h.float()).abs() + y.float().abs() + shared.abs() + mlp.float().abs())
        off = (y.float() - (h.float() + mlp.float())).abs() - tol
        for b in range(2):
            n = 5 if n_new is None else n_new[b]
            assert off[b, :n].max() <= 0
    head = mx.MTPHead(a, 1, DEV)
    c = head.make_paged_cache(2, 16) if paged else head.make_cache(2, 64)
    out = head(x, x, c)
    assert out.shape == x.shape and torch.isfinite(out.float()).all()
