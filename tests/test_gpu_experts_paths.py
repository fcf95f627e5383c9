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

import linear_sizes
import multiplex_amd as mx
from multiplex_amd import _lib
from oracle import experts as ox
from test_gpu_experts import (DEV, U, _check_block, _check_experts, _check_linear, _check_route, _experts, _gen, _np, _r,
                              _sums, _within)

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


# ------------------------------------------------------------- linear_act

@pytest.mark.parametrize("M,N,K,act,tile", linear_sizes.SIZES)
def test_linear_act_tiles(M, N, K, act, tile):
    """Bare and with the whole epilogue, into rows of their own and into columns of wider ones, through a workspace
    full of NaN; a row of NaN stays one."""
    g = _gen(M + N)
    rows = 2 * N if act == "swiglu" else N
    x, w = _r(g, M, K), _r(g, rows, K, scale=K ** -0.5)
    ws = torch.full((mx.linear_act_workspace_bytes(M, N, K, act) + 16,), 0xff, dtype=torch.uint8, device=DEV)
    wide = torch.full((M, N + 7), 7.0, dtype=torch.bfloat16, device=DEV)
    y = mx.linear_act(x, w, activation=act, workspace=ws)
    _check_linear(y, x, w, None, act, None, None)
    mx.linear_act(x, w, activation=act, out=wide[:, 3:3 + N])
    assert torch.equal(wide[:, 3:3 + N], y) and (wide[:, :3] == 7).all() and (wide[:, 3 + N:] == 7).all()
    x[1] = float("nan")
    bad = mx.linear_act(x, w, activation=act)
    assert torch.isnan(bad[1]).all() and torch.equal(bad[2:], y[2:]) and torch.equal(bad[0], y[0])
    x[1] = _r(g, K)

    act = act or [None, "relu", "silu", "gelu_tanh"][M % 4]
    bias, gate = _r(g, rows, dtype=[torch.bfloat16, torch.float32, torch.float16][N % 3]), _r(g, M, dtype=torch.float32)
    res = _r(g, M, N + 5)[:, 1:1 + N]
    y = mx.linear_act(x, w, bias=bias, activation=act, row_gate=gate, residual=res, workspace=ws)
    _check_linear(y, x, w, bias, act, gate, res)
    mx.linear_act(x, w, bias=bias, activation=act, row_gate=gate, residual=res, out=wide[:, 2:2 + N])
    assert torch.equal(wide[:, 2:2 + N], y) and (wide[:, :2] == 7).all() and (wide[:, 3 + N:] == 7).all()
    assert mx.linear_act(x, w, bias=bias, activation=act, row_gate=gate, residual=res, out=res) is res
    assert torch.equal(res, y)
    assert (ws[-16:] == 0xff).all()


# ------------------------------------------------------- planned experts

def _tile_rows(args):
    x, gate_up, down, indices = args[:4]
    return _lib.load().gdn_expert_mlp_tile_rows(x.shape[0], x.shape[1], down.shape[2], down.shape[0], indices.shape[1])


# (N, H, I, E, k), rows of a tile
PLANNED = [((600, 136, 72, 4, 2), 64), ((2048, 72, 1000, 8, 2), 128), ((4096, 72, 1000, 8, 2), 256)]


@pytest.mark.parametrize("scale", [1e-30, 1e-18, 1e18, 1e30])
@pytest.mark.parametrize("size,rows", PLANNED)
def test_planned_far_magnitudes(size, rows, scale):
    """Results near both ends of bf16's range."""
    args = list(_experts(_gen(6), *size))
    args[2] = (args[2].float() * scale).bfloat16()
    assert _tile_rows(args) == rows
    _check_columns(mx.expert_mlp(*args[:5]), *args)


@pytest.mark.parametrize("size,rows", PLANNED)
def test_planned_layouts(size, rows):
    """Strided rows, a workspace of one's own full of NaN, the output over the base."""
    x, gate_up, down, indices, weights, base = args = _experts(_gen(8), *size, True)
    assert _tile_rows(args) == rows
    N, H = x.shape
    want = mx.expert_mlp(x, gate_up, down, indices, weights, base=base)
    _check_columns(want, *args)
    wide = torch.full((N, H + 24), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 16:16 + H] = x
    need = mx.expert_mlp_workspace_bytes(N, H, down.shape[2], down.shape[0], indices.shape[1])
    ws = torch.full((need + 64,), 0xff, dtype=torch.uint8, device=DEV)
    out = torch.full((N, H + 8), 7.0, dtype=torch.bfloat16, device=DEV)
    got = mx.expert_mlp(wide[:, 16:16 + H], gate_up, down, indices, weights, base=base, out=out[:, :H], workspace=ws)
    assert torch.equal(got, want) and (out[:, H:] == 7).all() and (ws[need:] == 0xff).all()
    got = mx.expert_mlp(x.T.contiguous().T, gate_up, down, indices.T.contiguous().T, weights.T.contiguous().T,
                        base=base.T.contiguous().T, workspace=ws)  # (what the last call left in it)
    assert torch.equal(got, want)
    assert mx.expert_mlp(x, gate_up, down, indices, weights, base=base, out=base) is base
    assert torch.equal(base, want)


def test_planned_on_two_streams():
    args = _experts(_gen(11), 600, 264, 136, 12, 3, True)
    assert _tile_rows(args) > 0
    want = mx.expert_mlp(*args[:5], base=args[5])
    _check_experts(want, *args)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        s = streams[i % 2]
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(mx.expert_mlp(*args[:5], base=args[5]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_planned_in_two_graphs():
    """One planned in one launch and one in two, captured and replayed in turn, with eager calls between; their
    choices change from replay to replay."""
    sizes = [(600, 264, 136, 12, 3), (3000, 136, 72, 12, 3)]
    sets = [_experts(_gen(12 + i), *s, True) for i, s in enumerate(sizes)]
    assert all(_tile_rows(a) > 0 for a in sets)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a in sets:
            mx.expert_mlp(*a[:5], base=a[5])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for a in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(mx.expert_mlp(*a[:5], base=a[5]))
        graphs.append(g)
    for i in range(4):
        for a, g in zip(sets, graphs):
            a[0].copy_(torch.randn(a[0].shape, device=DEV))
            a[3].copy_(torch.rand(a[0].shape[0], 12, device=DEV).argsort(-1)[:, :3])
            if i == 2:
                a[3][10:] = 7  # all but a few of one expert
            g.replay()
        torch.cuda.synchronize()
        for a, o in zip(sets, outs):
            got = o.clone()
            assert torch.equal(got, mx.expert_mlp(*a[:5], base=a[5]))


# ------------------------------------------------------------ far offsets

def test_far_offsets_linear_act():
    """x, residual and out that pass 4 GiB: their last rows."""
    g = _gen(1)
    M, K, N, tail = 70000, 64, 32776, 40
    w = _r(g, N, K, scale=K ** -0.5)
    x = torch.empty(M, 32800, dtype=torch.bfloat16, device=DEV)[:, 8:8 + K]
    x.copy_(_r(g, M, K))
    res = torch.zeros(M, N, dtype=torch.bfloat16, device=DEV)
    res[-tail:] = _r(g, tail, N)
    y = mx.linear_act(x, w, residual=res)
    for rows in (slice(0, tail), slice(M // 2, M // 2 + tail), slice(M - tail, M)):
        _check_linear(y[rows], x[rows], w, None, None, None, res[rows])


def test_far_offsets_experts():
    """Results of pairs that wait in more than 4 GiB: the last tokens'."""
    g = _gen(2)
    N, H, I, E, k, tail = 300000, 1024, 16, 8, 8, 40
    gate_up, down = _r(g, E, 2 * I, H, scale=H ** -0.5), _r(g, E, H, I, scale=I ** -0.5)
    x = torch.randn(N, H, device=DEV).bfloat16()
    indices = torch.rand(N, E, device=DEV).argsort(-1).int()
    weights = torch.rand(N, k, device=DEV)
    y = mx.expert_mlp(x, gate_up, down, indices, weights)
    for rows in (slice(0, tail), slice(N // 2, N // 2 + tail), slice(N - tail, N)):
        _check_columns(y[rows], x[rows], gate_up, down, indices[rows], weights[rows], None)


def test_far_offsets_routing():
    """Logits that pass 4 GiB."""
    N, E, tail = 2200000, 1000, 20
    logits = torch.empty(N, 1024, dtype=torch.bfloat16, device=DEV)[:, 8:8 + E]
    logits.normal_()
    indices, weights = mx.route_experts(logits, 4)
    for rows in (slice(0, tail), slice(N // 2, N // 2 + tail), slice(N - tail, N)):
        _check_route((indices[rows], weights[rows]), logits[rows], 4)


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


@pytest.mark.parametrize("kw", [dict(), dict(shared_expert_intermediate_size=0, norm_topk_prob=False),
                                dict(scoring_func="sigmoid", n_group=4, topk_group=2, group_best=1,
                                     routed_scaling_factor=2.446, router_bias=True)])
def test_sparse_mlp_of_planned_pairs(kw):
    torch.manual_seed(1)
    B, T = 2, 200
    m = mx.SparseMLP(_layer_args(**{k: v for k, v in kw.items() if k != "group_best"}), DEV)
    if "n_group" in kw:
        m.router_bias.copy_(torch.randn(24, device=DEV) * 0.1)
    assert _lib.load().gdn_expert_mlp_tile_rows(B * T, 256, 72, 24, 4) > 0
    x, res = torch.randn(B, T, 256, device=DEV).bfloat16(), torch.randn(B, T, 256, device=DEV).bfloat16()
    _check_block(m, x, m(x))
    _check_block(m, x, m(x, residual=res), residual=res)
    n_new = torch.tensor([200, 3], dtype=torch.int32, device=DEV)
    _check_block(m, x, m(x, residual=res, n_new=n_new), residual=res, n_new=n_new)
    if "group_best" in kw:  # by their single best, the layer's own choice
        m.args.group_best = 1
        both = mx.linear_act(x, m.router)
        kw = dict(scoring="sigmoid", groups=4, top_groups=2, group_best=1, scale=2.446, bias=m.router_bias)
        indices, weights = mx.route_experts(both[..., :24], 4, **kw)
        _check_route((indices, weights), both[..., :24], 4, **kw)
        s = mx.linear_act(x, m.shared_gate_up_proj, activation="swiglu")
        base = mx.linear_act(s, m.shared_down_proj, row_gate=both[..., 24], residual=res)
        assert torch.equal(m(x, residual=res), mx.expert_mlp(x, m.gate_up_proj, m.down_proj, indices, weights, base=base))


def test_sparse_mlp_of_planned_pairs_in_a_graph():
    """Captured once, replayed on new inputs with eager work between."""
    torch.manual_seed(2)
    m = mx.SparseMLP(_layer_args(), DEV)
    x = torch.randn(2, 200, 256, device=DEV).bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m(x)
    for i in range(4):
        x.copy_(torch.randn(2, 200, 256, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        assert torch.equal(got, m(x))


def test_sparse_mlp_of_no_tokens():
    m = mx.SparseMLP(_layer_args(), DEV)
    for lead in ((0,), (0, 4), (3, 0)):
        x = torch.empty(*lead, 256, dtype=torch.bfloat16, device=DEV)
        assert m(x, residual=x).shape == x.shape
    x = torch.empty(0, 4, 256, dtype=torch.bfloat16, device=DEV)
    assert m(x, n_new=torch.empty(0, dtype=torch.int32, device=DEV)).shape == x.shape


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("T", [5, 150])
def test_draft_head_over_a_sparse_mlp(T, paged):
    """The head against its parts: the layer's MLP by the oracle, the final norm in float64."""
    torch.manual_seed(4)
    head = mx.MTPHead(_layer_args(), 1, DEV)
    layer = head.layers[0]
    for norm in (head.pre_fc_norm_embedding, head.pre_fc_norm_hidden, head.norm):
        norm.weight.data.copy_(1 + 0.2 * torch.randn(256, device=DEV))
    embed, hidden = (torch.randn(2, T, 256, device=DEV).bfloat16() for _ in range(2))

    def cache():
        return (head.make_paged_cache(2, 16) if paged else head.make_cache(2, 256))

    out = head(embed, hidden, cache())
    eh = torch.cat([head.pre_fc_norm_embedding(embed), head.pre_fc_norm_hidden(hidden)], -1)
    x = torch.nn.functional.linear(eh, head.fc)
    h, z, counts = layer._attend(x, None, cache()[0], None)
    assert counts is None
    m = layer.mlp(z)
    _check_block(layer.mlp, z, m)
    # s is rounded to bf16 (off by U of itself, and so by as much at most is its root mean square), then the result
    s = h.double() + m.double()
    y = s * torch.rsqrt((s * s).mean(-1, keepdim=True) + layer.input_layernorm.eps) * head.norm.weight.double()
    tol = 3.02 * U * y.abs() + 1e-6
    assert ((out.double() - y).abs() <= tol).all()
