"""What the sparse MLP's Python calls hand to the library, without a GPU: the calls' short
ways run on CPU tensors that claim a device, and the launch is a stand-in."""

from __future__ import annotations

import ctypes
import math
import random
import weakref

import linear_sizes
import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from multiplex_amd import _lib, attention, experts, linear
from oracle import experts as ox


class OnDevice(torch.Tensor):
    """A host tensor that the calls' short ways take for one of device 0."""

    def get_device(self):
        return 0


def _b(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnDevice)


def _i(*shape):
    return _b(*shape, dtype=torch.int32)


def _f(*shape):
    return _b(*shape, dtype=torch.float32)


@pytest.fixture
def made(monkeypatch):
    """(name, arguments) of the launches."""
    calls = []
    for mod in (experts, linear):
        monkeypatch.setattr(mod, "_stream", lambda dev: 0)
        monkeypatch.setattr(mod, "_require_device", lambda tensors, names: torch.device("cpu"))
    monkeypatch.setattr(_lib, "call", lambda dev, name, *args: calls.append((name, args)))
    return calls


def test_a_workspace_lives_until_its_launch(made, monkeypatch):
    """(Another thread may be given its memory otherwise: the library's call lets go of the interpreter.)"""
    x, w = _b(14, 12144), _b(494, 12144)
    assert linear.linear_act_workspace_bytes(14, 494, 12144) > 0
    made_here, alive = [], []
    empty = torch.empty

    def recorded(*args, **kw):
        t = empty(*args, **kw)
        made_here.append(weakref.ref(t))
        return t

    def launched(dev, name, *args):
        alive.extend(r() is not None and r().data_ptr() in args for r in made_here)

    monkeypatch.setattr(torch, "empty", recorded)
    monkeypatch.setattr(_lib, "call", launched)
    linear.linear_act(x, w)
    assert alive == [True]
    made_here.clear(), alive.clear()
    experts.expert_mlp(_b(4, 16), _b(3, 16, 16), _b(3, 16, 8), _i(4, 2), _f(4, 2))
    assert alive == [True]


def test_oracle_groups_of_infinite_biases():
    """A group whose two best are +inf and -inf has no sum: it counts as -inf."""
    inf = np.inf
    bias = np.array([inf, -inf, -inf, -inf, 0.5, 0, 0, 0, 0.4, 0, 0, 0, 0, 0, 0, 0])
    i, _ = ox.route(np.zeros((1, 16)), 4, scoring="sigmoid", bias=bias, groups=4, top_groups=2)
    assert i.tolist() == [[4, 8, 5, 6]]
    i, _ = ox.route(np.zeros((1, 16)), 4, scoring="sigmoid", bias=bias, groups=4, top_groups=2, group_best=1)
    assert i.tolist() == [[0, 4, 5, 6]]


# Each call as a function of one of its inputs.
CALLS = {
    "linear_act": (lambda x: linear.linear_act(x, _b(8, 16)), lambda: _b(4, 16)),
    "linear_act's weight": (lambda w: linear.linear_act(_b(4, 16), w), lambda: _b(8, 16)),
    "linear_act's row gate": (lambda r: linear.linear_act(_b(4, 16), _b(8, 16), row_gate=r), lambda: _f(4)),
    "route_experts": (lambda l: experts.route_experts(l, 2)[1], lambda: _f(4, 16)),
    "expert_mlp": (lambda x: experts.expert_mlp(x, _b(3, 16, 16), _b(3, 16, 8), _i(4, 2), _f(4, 2)), lambda: _b(4, 16)),
    "expert_mlp's weights": (lambda w: experts.expert_mlp(_b(4, 16), _b(3, 16, 16), _b(3, 16, 8), _i(4, 2), w),
                             lambda: _f(4, 2)),
}


@pytest.mark.parametrize("call", CALLS)
def test_a_tangent_is_refused(made, call):
    f, t = CALLS[call]
    with forward_ad.dual_level():
        f(t())  # none of its tensors has one
        assert len(made) == 1
        with pytest.raises(ValueError, match="tangent"):
            f(forward_ad.make_dual(t(), torch.ones_like(t())))
    assert len(made) == 1


@pytest.mark.parametrize("call", CALLS)
def test_a_trace_is_refused(made, call):
    """It would hold the result as a constant."""
    f, t = CALLS[call]
    plain = t().as_subclass(torch.Tensor)
    for trace in (lambda: torch.jit.trace(f, (plain,), check_trace=False), lambda: make_fx(f)(plain)):
        with pytest.raises(ValueError, match="traced"):
            trace()
    assert not made


def test_a_mode_that_only_looks_on_is_served(made):
    from torch.utils.flop_counter import FlopCounterMode

    with FlopCounterMode(display=False):
        for f, t in CALLS.values():
            f(t())
    assert len(made) == len(CALLS)


@pytest.mark.parametrize("N", [1, 300, 1 << 13])
def test_inner_rows_past_a_tiles_offsets_are_refused(N):
    """A tile's rows of inner values are found by 32-bit byte offsets: 256 of more than 2^22 values pass 2 GiB."""
    fake = 0x10000  # only ever compared, never read
    lib = _lib.load()

    def call(I):
        return lib.gdn_expert_mlp(fake, 8, fake, fake, fake, fake, None, 0, fake, 8, N, 8, I, 1, 1, fake + 8, 1 << 60, None)

    assert call((1 << 22) + 8) == _lib.ERR_UNSUPPORTED
    assert call(1 << 22) == _lib.ERR_INVALID  # as far as the workspace, which is misaligned


def _layer(**kw):
    a = dict(hidden_size=64, num_attention_heads=2, num_key_value_heads=1, head_dim=128, intermediate_size=32,
             num_experts=6, num_experts_per_tok=2, moe_intermediate_size=16, shared_expert_intermediate_size=24)
    return attention.AttentionArgs(**{**a, **kw})


@pytest.mark.parametrize("lead", [(5,), (4, 1), (1, 6), (2, 3), (2, 3, 4)])
def test_the_layers_calls_take_the_short_way(made, monkeypatch, lead):
    """(A row gate that is a column of a wider product, of any number of dimensions, among them.)"""
    for mod, name in ((linear, "_linear_act_general"), (experts, "_route_general"), (experts, "_expert_mlp_general")):
        monkeypatch.setattr(mod, name, lambda *a, name=name: pytest.fail(name))
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    m = experts.SparseMLP(_layer())
    m(_b(*lead, 64), residual=_b(*lead, 64))
    assert [n for n, _ in made] == ["gdn_linear_act", "gdn_route_experts", "gdn_linear_act", "gdn_linear_act", "gdn_expert_mlp"]
    gate, ld = made[3][1][6], made[3][1][8]
    assert gate - made[0][1][11] == 6 * 2 and ld == 7  # the seventh column of what the router's product wrote


def test_row_gates_of_other_layouts(made):
    """Evenly spaced ones are read in place (one value for all among them), others copied."""
    x, w = _b(2, 3, 16), _b(8, 16)
    for gate, ld in ((_f(2, 3), 1), (_f(2, 3, 5)[..., 2], 5), (_f(1).expand(2, 3), 0), (_f(3, 2).T, None),
                     (_f(2, 1).expand(2, 3), None), (_f(2, 4)[:, :3], None)):
        made.clear()
        linear.linear_act(x, w, row_gate=gate)
        (_, args), = made
        assert args[8] == (1 if ld is None else ld)
        assert (args[6] == gate.data_ptr()) == (ld is not None)


def test_the_layers_routing_is_its_arguments(made, monkeypatch):
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    for kw, want in ((dict(), (0, 1, 1, 2, 1, 1.0)),
                     (dict(scoring_func="sigmoid", n_group=3, topk_group=2, group_best=1, norm_topk_prob=False,
                           routed_scaling_factor=2.5), (1, 3, 2, 1, 0, 2.5))):
        made.clear()
        experts.SparseMLP(_layer(**kw))(_b(4, 64))
        (args,) = [a for n, a in made if n == "gdn_route_experts"]
        assert args[11:17] == want


@pytest.mark.parametrize("name,shape", [
    ("gate", (1, 64)), ("gate", (64,)), ("gate", (5, 64)), ("gate_proj", (1, 16, 64)), ("up_proj", (6, 16, 1)),
    ("up_proj", (6, 8, 64)), ("down_proj", (1, 64, 16)), ("down_proj", (64, 16)), ("shared_gate_proj", (23, 64)),
    ("shared_down_proj", (64, 1)), ("shared_expert_gate", (2, 64)), ("router_bias", (1,)),
])
def test_loading_other_shapes_is_refused(name, shape):
    """(A weight of one expert would be spread over all of them, halves of other sizes make a whole.)"""
    shapes = dict(gate=(6, 64), gate_proj=(6, 16, 64), up_proj=(6, 16, 64), down_proj=(6, 64, 16), shared_gate_proj=(24, 64),
                  shared_up_proj=(24, 64), shared_down_proj=(64, 24), shared_expert_gate=(1, 64), router_bias=(6,))
    m = experts.SparseMLP(_layer(router_bias=True))
    w = {n: torch.ones(s) for n, s in shapes.items()}
    before = {n: p.clone() for n, p in m.state_dict().items()}
    other = {"gate_proj": "up_proj", "up_proj": "gate_proj", "shared_gate_proj": "shared_up_proj"}.get(name)
    if shape == (1, 16, 64):  # both halves, as they would be given
        w[other] = torch.ones(shape)
    if shape in ((6, 8, 64), (23, 64)):  # the other half makes up for it
        w[other] = torch.ones(6, 24, 64) if len(shape) == 3 else torch.ones(25, 64)
    with pytest.raises(ValueError):
        m.load(**{**w, name: torch.ones(shape)})
    assert all(torch.equal(p, before[n]) for n, p in m.state_dict().items())


def test_loading_takes_the_shapes_that_it_names():
    m = experts.SparseMLP(_layer())
    w = [torch.randn(s).bfloat16() for s in ((6, 64), (6, 16, 64), (6, 16, 64), (6, 64, 16), (24, 64), (24, 64), (64, 24), (64,))]
    m.load(*w)
    assert torch.equal(m.router, torch.cat([w[0], w[7][None]])) and torch.equal(m.gate_up_proj[:, 16:], w[2])


def test_in_place_of_x_and_base(made):
    """out = base = x on the short way and on the long one alike; x alone, or other rows of it, are refused."""
    a = dict(gate_up=_b(3, 16, 16), down=_b(3, 16, 8), indices=_i(4, 2), weights=_f(4, 2))
    for x in (_b(4, 16), _b(4, 24)[:, :16], _b(4, 16).as_subclass(torch.Tensor)):
        assert experts.expert_mlp(x, **a, base=x, out=x) is x
        view = x[:]
        assert experts.expert_mlp(view, **a, base=x, out=x) is x
        with pytest.raises(ValueError, match="overlaps x"):
            experts.expert_mlp(x, **a, base=_b(4, 16), out=x)
    assert [n for n, _ in made] == ["gdn_expert_mlp"] * 6
    buf = _b(6, 24)
    with pytest.raises(ValueError, match="overlaps x"):
        experts.expert_mlp(buf[1:5, :16], **a, base=buf[:4, :16], out=buf[:4, :16])


# ------------------------------------------------------------------ the sizes' rules

def _linear_tile(M, N, K, act):
    tile = (ctypes.c_int32 * 3)()
    assert _lib.load().gdn_linear_act_tile(M, N, K, linear._ACTS[act], tile) == _lib.OK
    return tuple(tile)


@pytest.mark.parametrize("M,N,K,act,tile", linear_sizes.SIZES)
def test_linear_act_runs_the_tile(M, N, K, act, tile):
    """What the GPU tests run at these sizes is what they say (refit the sizes with the rule)."""
    assert _linear_tile(M, N, K, act) == tile
    need = linear.linear_act_workspace_bytes(M, N, K, act)
    pitch = (N + 3) // 4 * 4 * (2 if act == "swiglu" else 1)
    assert need == (4 * tile[2] * M * pitch if tile[2] > 1 else 0)


@pytest.mark.parametrize("act", [None, "gelu", "swiglu"])
@pytest.mark.parametrize("M,N,K", [(600, 1000, 8200), (64, 1026, 8192), (130, 517, 12296)])
def test_the_sliced_sizes_are_sliced(M, N, K, act):
    """Those of ``test_gpu_experts``, which passes over the ones that are not."""
    assert _linear_tile(M, N, K, act)[2] > 1 and linear.linear_act_workspace_bytes(M, N, K, act) > 0


def test_every_tile_is_run():
    """Each tile whole, and in every number of slices that the rule gives it, with and without SwiGLU."""
    run = {(act, tile) for *_, act, tile in linear_sizes.SIZES}
    rng = random.Random(1)
    for _ in range(20000):
        M, N, K = (int(math.exp(rng.uniform(math.log(a), math.log(b)))) for a, b in ((5, 6000), (8, 30000), (1, 1600)))
        for act in (None, "swiglu"):
            assert (act, _linear_tile(M, N, 8 * K, act)) in run
    for M in (1, 2, 3, 4):
        assert _linear_tile(M, 1000, 4096, None) == (0, 0, 0)


def test_the_tiles_calls_refuse_what_the_products_do():
    lib = _lib.load()
    tile = (ctypes.c_int32 * 3)()
    for args in ((-1, 8, 8, 0), (8, 0, 8, 0), (8, 8, 12, 0), (8, 8, 8, 6)):
        assert lib.gdn_linear_act_tile(*args, tile) == _lib.ERR_INVALID
    assert lib.gdn_linear_act_tile(8, 8, 8, 0, None) == _lib.ERR_INVALID
    assert lib.gdn_expert_mlp_tile_rows(8, 12, 8, 4, 2) == _lib.ERR_INVALID
    assert lib.gdn_expert_mlp_tile_rows(1, 64, 32, 4, 2) == 0
    assert lib.gdn_expert_mlp_tile_rows(4096, 2048, 512, 256, 8) in (64, 128, 256)
    # sizes that are refused for what they would span
    assert lib.gdn_expert_mlp_tile_rows(300, 8, (1 << 22) + 8, 1, 1) == _lib.ERR_UNSUPPORTED
    assert lib.gdn_expert_mlp_tile_rows(300, 1 << 16, 1 << 14, 1, 1) == _lib.ERR_UNSUPPORTED
    assert lib.gdn_linear_act_tile(300, 8, 1 << 23, 0, tile) == _lib.ERR_UNSUPPORTED
    assert lib.gdn_linear_act_tile(300, 1 << 24, 64, 5, tile) == _lib.ERR_UNSUPPORTED
