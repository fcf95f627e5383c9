"""The sparse MLP's operators on each of their kernels' paths: every tile that the sizes' rules
can choose, the planned experts where they are read in place, captured or overlapped, and
columns of one result that are far apart in size.

Tolerances as in ``test_gpu_experts``, from whose helpers they come; an expert's result
is rounded to 12 bits of significand on its way to the sum: off by at most 2^-12 of itself,
whatever lies beside it.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import multiplex_amd as mx
from oracle import experts as ox
from test_gpu_experts import DEV, U, _check_route, _experts, _gen, _np, _r, _sums, _within

pytestmark = pytest.mark.gpu


def _check_columns(y, x, gate_up, down, indices, weights, base):
    """Each column within what its own sums and roundings come to."""
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
        er += 2.0 ** -12 * (np.abs(r) + er)
        w = weights[t, j][:, None]
        np.add.at(ref, t, w * r)
        np.add.at(tol, t, np.abs(w) * er + 2.0 ** -22 * np.abs(w * r))
    _within(y, ref, tol + U * (np.abs(ref) + tol))


# few pairs; tiles of 64 rows, of 128 and of 256; 157 MB of weights, which pass by the caches, in tiles of 64 and of 128
PATHS = [(3, 136, 72, 4, 2), (600, 136, 72, 4, 2), (2048, 72, 1000, 8, 2), (4096, 72, 1000, 8, 2), (200, 512, 200, 256, 6),
         (1400, 512, 200, 256, 6)]


@pytest.mark.parametrize("base", [False, True])
@pytest.mark.parametrize("N,H,I,E,k", PATHS)
def test_expert_mlp_columns_far_apart(N, H, I, E, k, base):
    """Columns a thousand and a million times their neighbours, as hidden states have them."""
    x, gate_up, down, indices, weights, b = _experts(_gen(N), N, H, I, E, k, base)
    scale = torch.ones(H, device=DEV)
    scale[1::8], scale[6::16], scale[3::16] = 2.0 ** 10, 2.0 ** 20, 2.0 ** -10
    down = (down * scale[:, None]).bfloat16()
    y = mx.expert_mlp(x, gate_up, down, indices, weights, base=b)
    _check_columns(y, x, gate_up, down, indices, weights, b)


@pytest.mark.parametrize("N,H,I,E,k", PATHS[:3] + PATHS[4:5])
def test_expert_mlp_every_nan_stays_one(N, H, I, E, k):
    """NaNs of all sorts of bits among the weights: none becomes a number, and other columns are as without."""
    x, gate_up, down, indices, weights, _ = _experts(_gen(N), N, H, I, E, k)
    clean = mx.expert_mlp(x, gate_up, down, indices, weights)
    bits = torch.tensor([0x7fff, -1, 0x7f81, 0x7fc0, -0x7f, -0x40], dtype=torch.int16, device=DEV).view(torch.bfloat16)
    bad, cols = down.clone(), [0, 5, 18, 31, 44, H - 1]
    for c, v in zip(cols, bits):
        bad[:, c, I // 2] = v
    y = mx.expert_mlp(x, gate_up, bad, indices, weights)
    keep = [c for c in range(H) if c not in cols]
    assert torch.isnan(y[:, cols]).all() and torch.equal(y[:, keep], clean[:, keep])
    bad = x.clone()
    bad[1, :6] = bits
    y = mx.expert_mlp(bad, gate_up, down, indices, weights)
    assert torch.isnan(y[1]).all() and torch.equal(y[2:], clean[2:]) and torch.equal(y[0], clean[0])


@pytest.mark.parametrize("N,H,I,E,k", PATHS[:3])
def test_expert_mlp_in_place(N, H, I, E, k):
    """x, base and out the same rows."""
    x, gate_up, down, indices, weights, _ = _experts(_gen(N), N, H, I, E, k)
    want = mx.expert_mlp(x, gate_up, down, indices, weights, base=x)
    wide = torch.full((N, H + 16), 7.0, dtype=torch.bfloat16, device=DEV)
    rows = wide[:, 8:8 + H]
    rows.copy_(x)
    assert mx.expert_mlp(rows, gate_up, down, indices, weights, base=rows, out=rows) is rows
    assert torch.equal(rows, want) and (wide[:, :8] == 7).all() and (wide[:, 8 + H:] == 7).all()
    assert mx.expert_mlp(x, gate_up, down, indices, weights, base=x, out=x) is x
    assert torch.equal(x, want)


# --------------------------------------------------------------- routing

@pytest.mark.parametrize("times", [1, 200])  # of 20 tokens: 64 lanes a token, 32
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,top_groups,k", [(16, 4, 2, 4), (256, 8, 4, 8), (60, 3, 1, 20)])
def test_route_infinite_biases(E, groups, top_groups, k, scoring, times):
    """Experts that are always (+inf) or never (-inf) to be taken: as many groups stay as are asked for, one with
    both among its two best counting as -inf."""
    g = _gen(E)
    logits = _r(g, 20, E, dtype=torch.float32)
    width = E // groups
    for taken, never in (((0,), range(1, width)), ((1, width + 2), range(0, 0)), ((), range(E - width, E)),
                         ((), range(0, E)), ((E - 1,), range(0, E - 1))):
        bias = _r(g, E, dtype=torch.float32, scale=0.1)
        bias[list(never)] = float("-inf")
        bias[list(taken)] = float("inf")
        for group_best in (1, 2):
            kw = dict(scoring=scoring, bias=bias, groups=groups, top_groups=top_groups, group_best=group_best)
            indices, weights = mx.route_experts(logits.repeat(times, 1), k, **kw)
            _check_route((indices[:20], weights[:20]), logits, k, **kw)
            assert torch.equal(indices, indices[:20].repeat(times, 1))


# ------------------------------------------------- what follows an operator

def test_tangents_and_traces_are_refused():
    g = _gen(3)
    x, w, logits = _r(g, 8, 64), _r(g, 16, 64), _r(g, 8, 16, dtype=torch.float32)
    a = _experts(g, 8, 64, 32, 6, 2)
    calls = [(lambda t: mx.linear_act(t, w), x), (lambda t: mx.route_experts(t, 2)[1], logits),
             (lambda t: mx.expert_mlp(t, *a[1:5]), a[0])]
    for f, t in calls:
        want = f(t)
        with forward_ad.dual_level():
            assert torch.equal(f(t), want)
            with pytest.raises(ValueError, match="tangent"):
                f(forward_ad.make_dual(t, torch.ones_like(t)))
        for trace in (lambda: torch.jit.trace(f, (t,), check_trace=False), lambda: make_fx(f)(t)):
            with pytest.raises(ValueError, match="traced"):
                trace()
        assert torch.equal(f(t), want)


# ------------------------------------------------------------------ layers

def _layer_args(**kw):
    a = dict(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=128, intermediate_size=0,
             num_experts=24, num_experts_per_tok=4, moe_intermediate_size=72, shared_expert_intermediate_size=136)
    return mx.AttentionArgs(**{**a, **kw})


@pytest.mark.parametrize("experts", [24, 0])
def test_a_padded_step_uploads_its_counts_once(monkeypatch, experts):
    torch.manual_seed(5)
    layer = mx.DecoderLayer(_layer_args(num_experts=experts, intermediate_size=72), DEV)
    made, counts = [], mx.PagedKVCache.counts
    monkeypatch.setattr(mx.PagedKVCache, "counts", lambda self, n_new: made.append(counts(self, n_new)) or made[-1])
    x = torch.randn(2, 5, 256, device=DEV).bfloat16()
    cache = mx.PagedKVCache(mx.BlockPool(16, 2, 128, device=DEV), 2)
    layer(x, cache, n_new=[5, 2])
    assert len(made) == 1 and cache.lengths == [5, 2] and cache.pos0.tolist() == [5, 2]
    layer.forward_parts(x, None, cache, [0, 5])
    assert len(made) == 2 and cache.lengths == [5, 7] and cache.pos0.tolist() == [5, 7]
    for bad in ([1], [1, 6], [-1, 2]):
        with pytest.raises(ValueError):
            layer(x, cache, n_new=bad)
        assert cache.lengths == [5, 7] and cache.pos0.tolist() == [5, 7]
