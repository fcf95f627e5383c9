"""The sparse MLP's operators without a GPU: the oracle against closed forms, the
refusals of the C entry points and of the Python calls, the launches' device."""

from __future__ import annotations

import contextlib

import numpy as np
import pytest
import torch

from multiplex_amd import _lib, attention, experts, linear
from oracle import experts as ox

FAKE = 0x10000  # only ever compared, never read


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


# ------------------------------------------------------------------ oracle

def test_oracle_linear_act_is_torchs():
    g = torch.Generator().manual_seed(1)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((5, 12), (6, 12), (6,)))
    F = torch.nn.functional
    y = F.linear(x, w, b)
    for name, f in ((None, lambda v: v), ("relu", F.relu), ("silu", F.silu), ("gelu", F.gelu),
                    ("gelu_tanh", lambda v: F.gelu(v, approximate="tanh")),
                    ("swiglu", lambda v: F.silu(v[:, :3]) * v[:, 3:])):
        got = ox.linear_act(x.numpy(), w.numpy(), b.numpy(), name)
        assert np.allclose(got, f(y).numpy(), rtol=1e-13, atol=1e-14), name
    gate, res = torch.randn(5, generator=g, dtype=torch.float64), torch.randn(5, 6, generator=g, dtype=torch.float64)
    got = ox.linear_act(x.numpy(), w.numpy(), row_gate=gate.numpy(), residual=res.numpy())
    assert np.allclose(got, (F.linear(x, w) * torch.sigmoid(gate)[:, None] + res).numpy(), rtol=1e-13, atol=1e-14)


def test_oracle_route_closed_forms():
    l = np.array([[0.0, 2.0, 1.0, 2.0]])
    i, w = ox.route(l, 3)
    assert i.tolist() == [[1, 3, 2]] and np.isclose(w.sum(), 1) and w[0, 0] == w[0, 1]
    i, w = ox.route(l, 2, scoring="sigmoid", renormalize=False, scale=2.0)
    assert np.allclose(w, 2 / (1 + np.exp(-2)))
    # a bias moves the choice, not the weight
    i, w = ox.route(l, 1, bias=np.array([5.0, 0, 0, 0]), renormalize=False)
    assert i.tolist() == [[0]] and np.isclose(w[0, 0], np.exp(0) / np.exp(l).sum())
    # the best single expert lies in the group that loses by its two best
    l = np.array([[3.0, -9.0, 2.0, 2.0]])
    assert ox.route(l, 1, scoring="sigmoid", groups=2, top_groups=1, group_best=2)[0].tolist() == [[2]]
    assert ox.route(l, 1, scoring="sigmoid", groups=2, top_groups=1, group_best=1)[0].tolist() == [[0]]
    i, w = ox.route(np.full((1, 4), -np.inf), 2)
    assert i.tolist() == [[0, 1]] and (w == 0).all()
    i, _ = ox.route(np.array([[np.nan, -5.0, np.nan]]), 3, scoring="sigmoid")
    assert i.tolist() == [[1, 0, 2]]


def test_oracle_experts_closed_forms():
    g = np.random.default_rng(0)
    x, gu, d = g.standard_normal((3, 4)), g.standard_normal((2, 6, 4)), g.standard_normal((2, 4, 3))

    def one(e, t):
        h = gu[e] @ x[t]
        return d[e] @ (h[:3] / (1 + np.exp(-h[:3])) * h[3:])

    y = ox.expert_mlp(x, gu, d, np.array([[0, 1], [1, 1], [-1, 2]]), np.array([[1.0, 2.0], [0.5, 0.5], [9.0, 9.0]]), x)
    assert np.allclose(y[0], x[0] + one(0, 0) + 2 * one(1, 0)) and np.allclose(y[1], x[1] + one(1, 1))
    assert np.array_equal(y[2], x[2])


# ---------------------------------------------------------- the C entry points

def _route(lib, **kw):
    a = dict(logits=FAKE, dt=0, ld=64, bias=None, n_new=None, indices=FAKE, weights=FAKE, B=2, T=3, E=64, k=4, sig=0,
             groups=1, top=1, best=2, re=1, scale=1.0)
    a.update(kw)
    return lib.gdn_route_experts(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(E=0), _lib.ERR_INVALID), (dict(E=1025, ld=1025), _lib.ERR_INVALID), (dict(k=0), _lib.ERR_INVALID),
    (dict(k=65, E=128, ld=128), _lib.ERR_INVALID), (dict(k=5, E=4), _lib.ERR_INVALID), (dict(B=-1), _lib.ERR_INVALID),
    (dict(T=-1), _lib.ERR_INVALID), (dict(groups=3), _lib.ERR_INVALID), (dict(groups=0), _lib.ERR_INVALID),
    (dict(groups=4, top=5), _lib.ERR_INVALID), (dict(groups=4, top=0), _lib.ERR_INVALID),
    (dict(groups=16, top=1, k=5), _lib.ERR_INVALID), (dict(best=3), _lib.ERR_INVALID), (dict(best=0), _lib.ERR_INVALID),
    (dict(E=128, ld=128, groups=128), _lib.ERR_INVALID), (dict(dt=3), _lib.ERR_INVALID), (dict(ld=63), _lib.ERR_INVALID),
    (dict(logits=None), _lib.ERR_INVALID), (dict(indices=None), _lib.ERR_INVALID), (dict(weights=None), _lib.ERR_INVALID),
    (dict(logits=FAKE + 2), _lib.ERR_INVALID), (dict(bias=FAKE + 1), _lib.ERR_INVALID),
    (dict(n_new=FAKE + 2), _lib.ERR_INVALID), (dict(B=1 << 20, T=1 << 20), _lib.ERR_UNSUPPORTED),
    (dict(B=0), _lib.OK), (dict(T=0, logits=None), _lib.OK),
])
def test_route_abi_refusals(lib, kw, status):
    assert _route(lib, **kw) == status


def _mlp(lib, **kw):
    a = dict(x=FAKE, ldx=64, gu=FAKE, d=FAKE, i=FAKE, w=FAKE, base=None, ldb=0, out=FAKE, ldo=64, N=4, H=64, I=32, E=8,
             k=2, ws=FAKE, bytes=1 << 30)
    a.update(kw)
    return lib.gdn_expert_mlp(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(H=60, ldx=64), _lib.ERR_INVALID), (dict(I=4), _lib.ERR_INVALID), (dict(E=0), _lib.ERR_INVALID),
    (dict(E=1025), _lib.ERR_INVALID), (dict(k=0), _lib.ERR_INVALID), (dict(k=65), _lib.ERR_INVALID),
    (dict(N=-1), _lib.ERR_INVALID), (dict(x=None), _lib.ERR_INVALID), (dict(gu=None), _lib.ERR_INVALID),
    (dict(d=None), _lib.ERR_INVALID), (dict(i=None), _lib.ERR_INVALID), (dict(w=None), _lib.ERR_INVALID),
    (dict(out=None), _lib.ERR_INVALID), (dict(ldx=56), _lib.ERR_INVALID), (dict(ldx=68), _lib.ERR_INVALID),
    (dict(ldo=68), _lib.ERR_INVALID), (dict(base=FAKE, ldb=8), _lib.ERR_INVALID), (dict(base=FAKE + 8, ldb=64), _lib.ERR_INVALID),
    (dict(x=FAKE + 8), _lib.ERR_INVALID), (dict(d=FAKE + 2), _lib.ERR_INVALID), (dict(i=FAKE + 2), _lib.ERR_INVALID),
    (dict(ws=None), _lib.ERR_INVALID), (dict(ws=FAKE + 8), _lib.ERR_INVALID), (dict(bytes=100), _lib.ERR_INVALID),
    (dict(N=1 << 25, bytes=1 << 60), _lib.ERR_UNSUPPORTED),  # x spans 4 GiB
    (dict(H=1 << 16, I=1 << 14, ldx=1 << 16, ldo=1 << 16, bytes=1 << 60), _lib.ERR_UNSUPPORTED),  # an expert does
    (dict(N=0, x=None), _lib.OK),
])
def test_expert_mlp_abi_refusals(lib, kw, status):
    assert _mlp(lib, **kw) == status


def test_expert_mlp_workspace(lib):
    f = lib.gdn_expert_mlp_workspace_bytes
    for N, H, I, E, k in ((1, 8, 8, 1, 1), (4, 64, 32, 8, 2), (4096, 2048, 512, 256, 8), (1000, 64, 32, 9, 5)):
        n = f(N, H, I, E, k)
        assert n >= N * k * (I + H) * 2
        assert _mlp(lib, N=N, H=H, I=I, E=E, k=k, ldx=H, ldo=H, bytes=n - 1) == _lib.ERR_INVALID
    assert f(4, 60, 32, 8, 2) == 0 and f(4, 64, 32, 8, 65) == 0 and f(-1, 64, 32, 8, 2) == 0


def _linear(lib, **kw):
    a = dict(x=FAKE, ldx=64, W=FAKE, bias=None, bdt=0, act=0, gate=None, gdt=0, ldg=0, res=None, ldr=0, out=FAKE, ldo=48,
             M=4, N=48, K=64, ws=None, bytes=0)
    a.update(kw)
    return lib.gdn_linear_act(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(K=60), _lib.ERR_INVALID), (dict(K=0), _lib.ERR_INVALID), (dict(N=0), _lib.ERR_INVALID),
    (dict(M=-1), _lib.ERR_INVALID), (dict(act=6), _lib.ERR_INVALID), (dict(act=-1), _lib.ERR_INVALID),
    (dict(x=None), _lib.ERR_INVALID), (dict(W=None), _lib.ERR_INVALID), (dict(out=None), _lib.ERR_INVALID),
    (dict(ldx=56), _lib.ERR_INVALID), (dict(ldx=68), _lib.ERR_INVALID), (dict(ldo=47), _lib.ERR_INVALID),
    (dict(res=FAKE, ldr=47), _lib.ERR_INVALID), (dict(gate=FAKE, ldg=-1), _lib.ERR_INVALID),
    (dict(bias=FAKE, bdt=5), _lib.ERR_INVALID), (dict(gate=FAKE, gdt=-1), _lib.ERR_INVALID),
    (dict(bias=FAKE + 2), _lib.ERR_INVALID), (dict(gate=FAKE + 1, gdt=1), _lib.ERR_INVALID),
    (dict(x=FAKE + 8), _lib.ERR_INVALID), (dict(W=FAKE + 8), _lib.ERR_INVALID), (dict(out=FAKE + 1), _lib.ERR_INVALID),
    (dict(M=1 << 31), _lib.ERR_INVALID), (dict(N=1 << 30, ldo=1 << 30), _lib.ERR_INVALID),
    (dict(act=5, N=1 << 24, K=64, ldo=1 << 24), _lib.ERR_UNSUPPORTED),  # gate and up more than 2 GiB apart
    (dict(K=1 << 23, ldx=1 << 23), _lib.ERR_UNSUPPORTED), (dict(ldx=1 << 23), _lib.ERR_UNSUPPORTED),
    (dict(M=512, N=4096, K=12288, ldx=12288, ldo=4096), _lib.ERR_INVALID),  # without its workspace
    (dict(M=512, N=4096, K=12288, ldx=12288, ldo=4096, ws=FAKE, bytes=1000), _lib.ERR_INVALID),
    (dict(M=512, N=4096, K=12288, ldx=12288, ldo=4096, ws=FAKE + 8, bytes=1 << 40), _lib.ERR_INVALID),
    (dict(M=0, x=None), _lib.OK),
])
def test_linear_act_abi_refusals(lib, kw, status):
    assert _linear(lib, **kw) == status


def test_linear_act_workspace(lib):
    """None for most sizes; where K is summed in slices, four bytes a sum and slice."""
    f = linear.linear_act_workspace_bytes
    assert f(1, 4096, 12288) == 0 and f(4096, 12288, 4096, "swiglu") == 0 and f(128, 4096, 2048) == 0
    assert f(512, 4096, 12288) % (512 * 4096 * 4) == 0 and f(512, 4096, 12288) >= 2 * 512 * 4096 * 4
    assert lib.gdn_linear_act_workspace_bytes(512, 4096, 12289, 0) == 0
    assert lib.gdn_linear_act_workspace_bytes(512, 4096, 12288, 9) == 0


# --------------------------------------------------------------- the Python calls

@pytest.fixture
def calls(monkeypatch):
    """The launches made by calls on CPU tensors, with the library's own checks of sizes left out."""
    made = []
    for mod in (experts, linear):
        monkeypatch.setattr(mod, "_require_device", lambda tensors, names: torch.device("cpu"))
        monkeypatch.setattr(mod, "_stream", lambda dev: 0)
    monkeypatch.setattr(_lib, "call", lambda dev, name, *args: made.append((name, args)))
    return made


def _b(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def _i(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.mark.parametrize("kw", [
    dict(x=torch.zeros(4, 16)), dict(weight=torch.zeros(8, 16)), dict(weight=_b(8, 24)), dict(weight=_b(2, 8, 16)),
    dict(activation="tanh"), dict(weight=_b(7, 16), activation="swiglu"), dict(x=_b(4, 12), weight=_b(8, 12)),
    dict(x=_b(4, 0), weight=_b(8, 0)), dict(weight=_b(0, 16)), dict(bias=_b(7)), dict(bias=_i(8)), dict(bias=_b(4), activation="swiglu"),
    dict(row_gate=_b(3)), dict(row_gate=_b(4, 1)), dict(row_gate=_i(4)), dict(residual=_b(4, 7)),
    dict(residual=torch.zeros(4, 8)), dict(out=_b(4, 7)), dict(out=torch.zeros(4, 8)), dict(out=_b(8, 4).T),
    dict(x=_b(4, 16).requires_grad_()), dict(bias=torch.zeros(8, requires_grad=True)),
])
def test_linear_act_refusals(calls, kw):
    with pytest.raises(ValueError):
        linear.linear_act(**{"x": _b(4, 16), "weight": _b(8, 16), **kw})
    assert not calls


def test_linear_act_out_must_lie_apart(calls):
    buf = _b(4, 64)
    x, w = buf[:, :16], _b(8, 16)
    with pytest.raises(ValueError):
        linear.linear_act(x, w, out=buf[:, 8:16])
    res = buf[:, 24:32]
    with pytest.raises(ValueError):  # one column on: another thread's
        linear.linear_act(_b(4, 16), w, residual=res, out=buf[:, 25:33])
    linear.linear_act(_b(4, 16), w, residual=res, out=res)
    assert [n for n, _ in calls] == ["gdn_linear_act"]


def test_gradients_may_be_switched_off(calls):
    with torch.no_grad():
        linear.linear_act(_b(4, 16).requires_grad_(), _b(8, 16))
    assert [n for n, _ in calls] == ["gdn_linear_act"]


@pytest.mark.parametrize("kw", [
    dict(logits=torch.zeros(())), dict(logits=_i(4, 16)), dict(scoring="max"), dict(bias=_b(16)), dict(bias=torch.zeros(15)),
    dict(n_new=_i(4)), dict(logits=torch.zeros(2, 3, 16), n_new=_i(3)),
    dict(logits=torch.zeros(2, 3, 16), n_new=torch.zeros(2, dtype=torch.int64)),
    dict(logits=torch.zeros(4, 16, requires_grad=True)),
])
def test_route_refusals(calls, kw):
    with pytest.raises(ValueError):
        experts.route_experts(**{"logits": torch.zeros(4, 16), "k": 2, **kw})
    assert not calls


@pytest.mark.parametrize("kw", [
    dict(x=torch.zeros(4, 16)), dict(gate_up=torch.zeros(3, 16, 16)), dict(down=torch.zeros(3, 16, 8)),
    dict(gate_up=_b(3, 15, 16)), dict(gate_up=_b(2, 16, 16)), dict(gate_up=_b(3, 16, 24)), dict(down=_b(3, 24, 8)),
    dict(down=_b(16, 8)), dict(gate_up=_b(3, 16, 32)[..., :16]), dict(down=_b(3, 8, 16).transpose(1, 2)),
    dict(indices=torch.zeros(4, 2, dtype=torch.int64)), dict(indices=_i(3, 2)), dict(indices=_i(8)),
    dict(weights=_b(4, 2)), dict(weights=torch.zeros(4, 3)), dict(base=_b(4, 8)), dict(base=torch.zeros(4, 16)),
    dict(out=_b(3, 16)), dict(out=torch.zeros(4, 16)), dict(workspace=torch.zeros(4, 1 << 12, dtype=torch.uint8)[:, ::2]),
    dict(weights=torch.zeros(4, 2, requires_grad=True)),
])
def test_expert_mlp_refusals(calls, kw):
    with pytest.raises(ValueError):
        experts.expert_mlp(**{"x": _b(4, 16), "gate_up": _b(3, 16, 16), "down": _b(3, 16, 8), "indices": _i(4, 2),
                              "weights": torch.zeros(4, 2), **kw})
    assert not calls


def test_expert_mlp_out_must_lie_apart(calls):
    a = dict(gate_up=_b(3, 16, 16), down=_b(3, 16, 8), indices=_i(4, 2), weights=torch.zeros(4, 2))
    x = _b(4, 16)
    for kw in (dict(x=x, out=x), dict(x=x, base=_b(5, 16)[:4], out=None)):
        if kw["out"] is None:
            buf = _b(5, 16)
            kw = dict(x=x, base=buf[:4], out=buf[1:])
        with pytest.raises(ValueError):
            experts.expert_mlp(**a, **kw)
    base = _b(4, 16)
    assert experts.expert_mlp(x, **a, base=base, out=base) is base
    assert [n for n, _ in calls] == ["gdn_expert_mlp"]


def test_expert_mlp_takes_a_workspace_that_fits(calls):
    a = dict(gate_up=_b(3, 16, 16), down=_b(3, 16, 8), indices=_i(4, 2), weights=torch.zeros(4, 2))
    need = experts.expert_mlp_workspace_bytes(4, 16, 8, 3, 2)
    fits, small = torch.zeros(need, dtype=torch.uint8), torch.zeros(need - 1, dtype=torch.uint8)
    experts.expert_mlp(_b(4, 16), **a, workspace=fits)
    experts.expert_mlp(_b(4, 16), **a, workspace=small)
    (_, one), (_, two) = calls
    assert one[-3] == fits.data_ptr() and one[-2] == need and two[-3] != small.data_ptr() and two[-2] >= need


def test_tensors_must_be_on_a_device():
    for f in (lambda: linear.linear_act(_b(4, 16), _b(8, 16)), lambda: experts.route_experts(torch.zeros(4, 16), 2),
              lambda: experts.expert_mlp(_b(4, 16), _b(3, 16, 16), _b(3, 16, 8), _i(4, 2), torch.zeros(4, 2))):
        with pytest.raises(ValueError):
            f()


def test_launches_enter_their_tensors_device(monkeypatch):
    inside, made = [], []

    @contextlib.contextmanager
    def enter(dev):
        inside.append(dev)
        yield
        inside.pop()

    class Library:
        def __getattr__(self, name):
            def f(*args):
                if name.endswith("_workspace_bytes"):
                    return 64
                assert inside, name
                made.append(name)
                return _lib.OK
            return f

    monkeypatch.setattr(_lib, "_current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", enter)
    monkeypatch.setattr(_lib, "_lib", Library())
    for mod in (experts, linear):
        monkeypatch.setattr(mod, "_stream", lambda dev: 0)
        monkeypatch.setattr(mod, "_require_device", lambda tensors, names: torch.device("cpu"))
    linear.linear_act(_b(4, 16), _b(8, 16))
    experts.route_experts(torch.zeros(4, 16), 2)
    experts.expert_mlp(_b(4, 16), _b(3, 16, 16), _b(3, 16, 8), _i(4, 2), torch.zeros(4, 2))
    assert made == ["gdn_linear_act", "gdn_route_experts", "gdn_expert_mlp"]


# ------------------------------------------------------------------- layers

def _args(**kw):
    a = dict(hidden_size=64, num_attention_heads=2, num_key_value_heads=1, head_dim=128, intermediate_size=32,
             num_experts=6, num_experts_per_tok=2, moe_intermediate_size=16, shared_expert_intermediate_size=24)
    return attention.AttentionArgs(**{**a, **kw})


def test_layers_take_a_sparse_mlp():
    assert isinstance(attention.DecoderLayer(_args()).mlp, experts.SparseMLP)
    assert isinstance(attention.DecoderLayer(_args(num_experts=0)).mlp, attention.MLP)
    m = experts.SparseMLP(_args())
    assert m.router.shape == (7, 64) and set(m.state_dict()) == {"router", "gate_up_proj", "down_proj",
                                                                 "shared_gate_up_proj", "shared_down_proj"}
    m = experts.SparseMLP(_args(router_bias=True))
    assert m.state_dict()["router_bias"].dtype is torch.float32
    other = experts.SparseMLP(_args(router_bias=True))
    other.load_state_dict(m.state_dict())
    with pytest.raises(ValueError):  # it comes with one
        m.load(*(torch.zeros(s) for s in ((6, 64), (6, 16, 64), (6, 16, 64), (6, 64, 16), (24, 64), (24, 64), (64, 24), (1, 64))))
    m = experts.SparseMLP(_args(shared_expert_intermediate_size=0))
    assert m.router.shape == (6, 64) and set(m.state_dict()) == {"router", "gate_up_proj", "down_proj"}


@pytest.mark.parametrize("kw", [dict(num_experts_per_tok=0), dict(num_experts_per_tok=7), dict(moe_intermediate_size=0),
                                dict(shared_expert_intermediate_size=-8)])
def test_sparse_mlp_refusals(kw):
    with pytest.raises(ValueError):
        experts.SparseMLP(_args(**kw))
