"""The paged attention cache without a GPU: the oracle's own invariants, the
argument checks of the calls and of the C ABI, frequencies, and the cache's
bookkeeping (its device calls replaced by the oracle on CPU tensors)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import multiplex_amd as mx
from multiplex_amd import _lib, paged, rotary
from oracle import paged as op

FAKE = 0x10000  # 64 KiB-aligned dummy address; only ever compared, never read
BF = torch.bfloat16


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


# ----------------------------------------------------------------- the ABI

def _tables(lib, **kw):
    a = dict(lengths=FAKE, n_new=None, table=FAKE, ld=4, held=FAKE, free=FAKE, n_free=FAKE, held_out=FAKE,
             n_free_out=FAKE, slots=FAKE, B=2, T=1, block=64, shared=0, n_blocks=9)
    a.update(kw)
    return lib.gdn_paged_tables(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(lengths=None), _lib.ERR_INVALID),
    (dict(table=None), _lib.ERR_INVALID),
    (dict(held=None), _lib.ERR_INVALID),
    (dict(free=None), _lib.ERR_INVALID),
    (dict(n_free=None), _lib.ERR_INVALID),
    (dict(held_out=None), _lib.ERR_INVALID),
    (dict(n_free_out=None), _lib.ERR_INVALID),
    (dict(slots=None), _lib.ERR_INVALID),
    (dict(B=-1), _lib.ERR_INVALID),
    (dict(T=-1), _lib.ERR_INVALID),
    (dict(block=48), _lib.ERR_INVALID),
    (dict(block=0), _lib.ERR_INVALID),
    (dict(block=1 << 21), _lib.ERR_INVALID),
    (dict(shared=5), _lib.ERR_INVALID),
    (dict(shared=-1), _lib.ERR_INVALID),
    (dict(B=4097), _lib.ERR_UNSUPPORTED),
    (dict(T=1 << 31), _lib.ERR_UNSUPPORTED),
    (dict(n_blocks=1 << 25), _lib.ERR_UNSUPPORTED),
    (dict(ld=1 << 30), _lib.ERR_UNSUPPORTED),
    (dict(B=0, n_free_out=2 * FAKE), _lib.ERR_INVALID),
    (dict(B=0), _lib.OK),
])
def test_tables_abi_refusals(lib, kw, status):
    assert _tables(lib, **kw) == status


def _rope(lib, **kw):
    a = dict(qg=FAKE, qg_ld=0, q_head=512, k=FAKE, v=FAKE, kv_ld=0, qw=FAKE, kw=FAKE, wdt=_lib.DTYPE_F32, eps=1e-6,
             pos0=FAKE, slots=FAKE, turns=FAKE, factor=1.0, il=0, q=FAKE, keys=FAKE, values=FAKE, B=2, T=3, Hq=16,
             Hkv=4, D=256, n_blocks=5, block=64, rot=64)
    a.update(kw)
    return lib.gdn_attn_rope(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    *[({n: None}, _lib.ERR_INVALID) for n in ("qg", "k", "v", "qw", "kw", "pos0", "turns", "q", "keys", "values")],
    (dict(D=64), _lib.ERR_UNSUPPORTED),
    (dict(q_head=255), _lib.ERR_INVALID),
    (dict(Hq=15), _lib.ERR_INVALID),
    (dict(rot=63), _lib.ERR_UNSUPPORTED),
    (dict(rot=258), _lib.ERR_UNSUPPORTED),
    (dict(rot=6, B=0), _lib.OK),
    (dict(rot=4, il=1, B=0), _lib.OK),
    (dict(slots=None), _lib.ERR_INVALID),           # dense: one block a row
    (dict(slots=None, n_blocks=2, block=2), _lib.ERR_INVALID),
    (dict(slots=None, n_blocks=0, B=0), _lib.OK),
    (dict(wdt=9), _lib.ERR_INVALID),
    (dict(eps=-1.0), _lib.ERR_INVALID),
    (dict(eps=float("nan")), _lib.ERR_INVALID),
    (dict(qg_ld=16 * 512 - 257), _lib.ERR_INVALID),
    (dict(kv_ld=1023), _lib.ERR_INVALID),
    (dict(block=0), _lib.ERR_INVALID),
    (dict(n_blocks=1 << 25), _lib.ERR_UNSUPPORTED),
    (dict(T=1 << 28), _lib.ERR_UNSUPPORTED),
    (dict(T=0), _lib.OK),
])
def test_rope_abi_refusals(lib, kw, status):
    assert _rope(lib, **kw) == status


def _attn(lib, **kw):
    a = dict(q=FAKE, qg=FAKE, qg_ld=0, keys=FAKE, values=FAKE, table=FAKE, ld=10, pos0=FAKE, n_new=None, out=FAKE,
             scale=0.1, B=2, T=3, Hq=16, Hkv=4, D=256, n_blocks=5, block=64, L=600, shared=2, n_prefix=1, n_own=2,
             prefix_rows=16, own_rows=128, ws=FAKE, ws_bytes=1 << 40)
    a.update(kw)
    return lib.gdn_paged_attn(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    *[({n: None}, _lib.ERR_INVALID) for n in ("q", "keys", "values", "table", "pos0", "out", "ws")],
    (dict(D=64), _lib.ERR_UNSUPPORTED),
    (dict(block=32), _lib.ERR_UNSUPPORTED),
    (dict(block=96), _lib.ERR_UNSUPPORTED),
    (dict(Hq=18), _lib.ERR_INVALID),
    (dict(n_blocks=0), _lib.ERR_INVALID),
    (dict(ld=0), _lib.ERR_INVALID),
    (dict(ld=1 << 26), _lib.ERR_INVALID),
    (dict(L=641), _lib.ERR_INVALID),
    (dict(L=130), _lib.ERR_INVALID),                # below the shared keys and the new ones
    (dict(shared=0), _lib.ERR_INVALID),             # prefix ranges without a prefix
    (dict(shared=-1), _lib.ERR_INVALID),
    (dict(n_own=0), _lib.ERR_INVALID),
    (dict(n_prefix=-1), _lib.ERR_INVALID),
    (dict(n_own=65536), _lib.ERR_INVALID),
    (dict(prefix_rows=64), _lib.ERR_INVALID),
    (dict(own_rows=0), _lib.ERR_INVALID),
    (dict(scale=0.0), _lib.ERR_INVALID),
    (dict(q=FAKE + 8), _lib.ERR_INVALID),
    (dict(keys=FAKE + 8), _lib.ERR_INVALID),
    (dict(qg=FAKE + 2), _lib.ERR_INVALID),
    (dict(qg_ld=16 * 512 + 2), _lib.ERR_INVALID),
    (dict(qg_ld=8), _lib.ERR_INVALID),
    (dict(ws_bytes=2 * 3 * 16 * 3 * 258 * 4 - 1), _lib.ERR_INVALID),
    (dict(B=1 << 16), _lib.ERR_UNSUPPORTED),
    (dict(T=700), _lib.ERR_INVALID),                # more than the tables hold
    (dict(B=0), _lib.OK),
    (dict(T=0), _lib.OK),
])
def test_attention_abi_refusals(lib, kw, status):
    assert _attn(lib, **kw) == status
    assert status == _lib.OK or _lib.last_error()


@pytest.mark.parametrize("T", [641, 700, 1 << 20])
def test_attention_pads_past_the_tables(lib, T):
    """With n_new, T is the width of the padding and bounds no keys; without, every token is one."""
    assert _attn(lib, T=T, n_new=FAKE, B=0) == _lib.OK
    assert _attn(lib, T=T, n_new=FAKE, q=None) == _lib.ERR_INVALID and "null pointer" in _lib.last_error()
    assert _attn(lib, T=T, B=0) == _lib.ERR_INVALID


@pytest.mark.parametrize("B,T,Hq,Hkv,D,n", [(2, 3, 16, 4, 256, 3), (7, 1, 12, 4, 128, 2), (64, 1, 16, 4, 256, 33)])
def test_attention_workspace_as_the_call_takes_it(lib, calls, monkeypatch, B, T, Hq, Hkv, D, n):
    """The Python call sizes the workspace by itself: exactly the library's."""
    made = []
    monkeypatch.setattr(_lib, "call", lambda dev, name, *args: made.append(args))
    mx.paged_attn(**_attn_args(q=_z(B, T, Hq, D, dtype=BF), keys=_z(5, Hkv, 64, D, dtype=BF),
                               values=_z(5, Hkv, 64, D, dtype=BF), table=_z(B, 4), pos0=_z(B)), n_split=(1, n - 1))
    assert made[0][-2] == lib.gdn_paged_attn_workspace_bytes(B, T, Hq, Hkv, D, n) and made[0][-3]


def test_attention_workspace(lib):
    f = lib.gdn_paged_attn_workspace_bytes
    assert f(2, 3, 16, 4, 256, 1) == 0
    assert f(2, 3, 16, 4, 256, 3) == 2 * 3 * 16 * 3 * 258 * 4
    assert f(0, 3, 16, 4, 256, 3) == 0 and f(2, 3, 15, 4, 256, 3) == 0


# ------------------------------------------------------- the Python checks

@pytest.fixture
def calls(monkeypatch):
    """The library calls made, on CPU tensors."""
    made = []
    for mod in (paged, rotary):
        monkeypatch.setattr(mod, "_require_device", lambda tensors, names: torch.device("cpu"))
        monkeypatch.setattr(mod, "_stream", lambda dev: 0)
    monkeypatch.setattr(paged, "_cu_count", lambda dev: 256)
    monkeypatch.setattr(_lib, "call", lambda dev, name, *args: made.append(name))
    return made


def _z(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype)


def _tables_args(**kw):
    a = dict(lengths=_z(3), T=2, table=_z(3, 5), held=_z(3), free=_z(9), n_free=_z(1), block=64)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(lengths=_z(3, 1)), dict(lengths=_z(3, dtype=torch.int64)), dict(T=-1), dict(table=_z(2, 5)),
    dict(table=_z(5, 3).t()), dict(table=_z(3)), dict(held=_z(4)), dict(held=_z(6)[::2]), dict(free=_z(3, 3)),
    dict(free=_z(9, dtype=torch.int64)), dict(n_free=_z(2)), dict(n_new=_z(2)), dict(held_out=_z(2)),
    dict(n_free_out=_z(0)), dict(slots=_z(3, 3)), dict(slots=_z(3, 2, dtype=torch.int64)),
])
def test_tables_refusals(calls, kw):
    with pytest.raises(ValueError):
        mx.paged_tables(**_tables_args(**kw))
    assert not calls
    mx.paged_tables(**_tables_args())
    assert calls == ["gdn_paged_tables"]


def _rope_args(**kw):
    a = dict(qg=_z(2, 3, 4 * 512, dtype=BF), k_new=_z(2, 3, 512, dtype=BF), v_new=_z(2, 3, 512, dtype=BF),
             q_norm_w=torch.ones(256), k_norm_w=torch.ones(256), eps=1e-6, pos0=_z(2),
             keys=_z(5, 2, 64, 256, dtype=BF), values=_z(5, 2, 64, 256, dtype=BF), rotary=mx.Rotary(64, 1e4),
             slots=_z(2, 3))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(qg=_z(2, 3, 4 * 512)), dict(keys=torch.zeros(5, 2, 64, 256)), dict(values=_z(5, 2, 64, 128, dtype=BF)),
    dict(keys=_z(5, 64, 2, 256, dtype=BF).transpose(1, 2)), dict(qg=_z(2, 3, 4 * 512 + 8, dtype=BF)),
    dict(qg=_z(2, 3, 3 * 512, dtype=BF)), dict(qg=_z(6, 4 * 512, dtype=BF)), dict(k_new=_z(2, 3, 256, dtype=BF)),
    dict(k_new=_z(2, 3, 520, dtype=BF)[..., :512]), dict(k_new=_z(3, 2, 512, dtype=BF).transpose(0, 1)),
    dict(k_new=_z(2, 4, 512, dtype=BF)[:, :3], v_new=_z(2, 4, 512, dtype=BF)[:, :3]),
    dict(pos0=_z(3)), dict(pos0=_z(2, dtype=torch.int64)), dict(slots=_z(2, 4)), dict(slots=_z(3, 2).t()),
    dict(slots=None), dict(q_norm_w=None), dict(q_norm_w=torch.ones(128)), dict(q_norm_w=torch.ones(256, dtype=BF)),
    dict(q_norm_w=torch.ones(256, dtype=torch.float64), k_norm_w=torch.ones(256, dtype=torch.float64)),
    dict(q_out=_z(2, 3, 4, 128, dtype=BF)), dict(q_out=_z(2, 3, 4, 256)),
])
def test_rope_refusals(calls, kw):
    with pytest.raises(ValueError):
        mx.attn_rope(**_rope_args(**kw))
    assert not calls
    mx.attn_rope(**_rope_args())
    mx.attn_rope(**_rope_args(qg=_z(2, 3, 4 * 256, dtype=BF), gated=False, q_norm_w=None, k_norm_w=None))
    assert calls == ["gdn_attn_rope"] * 2


def _attn_args(**kw):
    a = dict(q=_z(2, 3, 4, 256, dtype=BF), keys=_z(5, 2, 64, 256, dtype=BF), values=_z(5, 2, 64, 256, dtype=BF),
             table=_z(2, 4), pos0=_z(2), kv_len_max=200, shared=1)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(q=_z(2, 3, 4, 256)), dict(q=_z(2, 3, 1024, dtype=BF)), dict(q=_z(2, 3, 4, 128, dtype=BF)),
    dict(q=_z(2, 3, 5, 256, dtype=BF)), dict(keys=_z(5, 2, 128, 256, dtype=BF)), dict(table=_z(3, 4)),
    dict(table=_z(4)), dict(table=_z(2, 4, dtype=torch.int64)), dict(pos0=_z(2, 1)), dict(n_new=_z(3)),
    dict(kv_len_max=257), dict(kv_len_max=66), dict(shared=-1), dict(shared=4), dict(gate=_z(2, 3, 4 * 256, dtype=BF)),
    dict(gate=_z(2, 3, 4 * 512)), dict(out=_z(2, 3, 4, 128, dtype=BF)), dict(out=_z(2, 3, 4, 256)),
    dict(out=_z(2, 4, 3, 256, dtype=BF).transpose(1, 2)),
])
def test_attention_refusals(calls, kw):
    with pytest.raises(ValueError):
        mx.paged_attn(**_attn_args(**kw))
    assert not calls
    mx.paged_attn(**_attn_args())
    mx.paged_attn(**_attn_args(kv_len_max=64, n_new=_z(2)))
    assert calls == ["gdn_paged_attn"] * 2


def test_attention_workspace_must_be_whole(calls):
    with pytest.raises(ValueError, match="workspace"):
        mx.paged_attn(**_attn_args(workspace=_z(1 << 20)[::2]))
    assert not calls


def test_attention_tables_of_too_many_keys(lib):
    """Ranges are rounded up to steps and looked up a step of all lanes ahead, in 32 bits."""
    assert _attn(lib, ld=(1 << 24) + 1, L=1 << 30) == _lib.ERR_UNSUPPORTED
    assert _attn(lib, ld=(1 << 25) - 1, L=2**31 - 64) == _lib.ERR_UNSUPPORTED


def test_tensors_must_be_on_a_device():
    with pytest.raises(ValueError, match="ROCm"):
        mx.paged_tables(**_tables_args())
    with pytest.raises(ValueError, match="ROCm"):
        mx.attn_rope(**_rope_args())
    with pytest.raises(ValueError, match="ROCm"):
        mx.paged_attn(**_attn_args())


# ------------------------------------------------------------- frequencies

@pytest.mark.parametrize("scaling", [
    None, {"type": "default"}, {"rope_type": "linear", "factor": 3.0},
    {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768},
    {"type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096, "beta_fast": 16.0, "beta_slow": 2.0,
     "attention_factor": 1.25},
])
def test_frequencies(scaling):
    r = mx.Rotary(64, 1e6, scaling=scaling)
    oracle = None if scaling is None or scaling.get("type") == "default" else \
        {**scaling, "type": scaling.get("type") or scaling["rope_type"]}
    inv, factor = op.frequencies(64, 1e6, oracle)
    np.testing.assert_allclose(r.inv_freq, inv, rtol=1e-14)
    assert r.factor == pytest.approx(factor, rel=1e-15)
    assert r.plain == (oracle is None)
    # turns: the 64-bit fraction of a turn per position, rounded to half a step (2^-65 turns) from a
    # float64 frequency (2^-53 of it, a few such roundings)
    turns = r.turns.numpy().view(np.uint64).astype(np.float64) * 2.0**-64
    np.testing.assert_allclose(turns * 2 * math.pi, inv, rtol=1e-14, atol=2.0**-65 * 2 * math.pi)


def test_frequencies_given():
    inv = [0.5, 7.0, -1.0, 0.0]  # more than a turn per position, and backwards, are whole turns off
    r = mx.Rotary(8, 1e4, inv_freq=inv, interleaved=True)
    turns = r.turns.numpy().view(np.uint64).astype(np.float64) * 2.0**-64
    np.testing.assert_allclose(turns, np.array(inv) / (2 * math.pi) % 1.0, atol=1e-15)
    assert not r.plain and r.factor == 1.0 and not list(r.state_dict())


@pytest.mark.parametrize("made,move", [("meta", lambda m: m.to_empty(device="cpu")), ("cpu", lambda m: m.to(torch.bfloat16)),
                                       ("cpu", lambda m: m.to("meta").to_empty(device="cpu"))])
def test_frequencies_survive_a_move(made, move):
    """A layer made without memory and filled from a checkpoint has its frequencies, which no checkpoint holds."""
    args = mx.AttentionArgs(256, 2, 1, 128, 512, rope_scaling={"type": "linear", "factor": 2.0})
    want = mx.Attention(args).rotary.turns
    got = move(mx.Attention(args, made)).rotary.turns
    assert got.dtype is torch.int64 and got.device.type == "cpu" and torch.equal(got, want)


@pytest.mark.parametrize("kw", [
    dict(rot=7), dict(rot=-2), dict(base=0.0), dict(scaling={"type": "other", "factor": 2.0}),
    dict(scaling={"type": "linear", "factor": 0.0}), dict(scaling={"type": "linear", "factor": math.inf}),
    dict(inv_freq=[1.0]), dict(inv_freq=[1.0, math.nan, 1.0, 1.0]),
    dict(inv_freq=[1.0] * 4, scaling={"type": "linear", "factor": 2.0}),
    dict(scaling={"type": "yarn", "factor": 2.0, "original_max_position_embeddings": 0}),
])
def test_rotary_refusals(kw):
    with pytest.raises(ValueError):
        mx.Rotary(**{**dict(rot=8, base=1e4), **kw})


YARN40 = dict(type="yarn", factor=40.0, original_max_position_embeddings=4096)


@pytest.mark.parametrize("extra", [
    dict(mscale=1.0, mscale_all_dim=1.0), dict(mscale=0.707, mscale_all_dim=1.0), dict(mscale=1.0, mscale_all_dim=0.7),
    dict(mscale=1.0), dict(mscale=1.0, mscale_all_dim=0.0), dict(truncate=False), dict(truncate=True),
    dict(truncate=False, beta_fast=16.0, beta_slow=2.0, mscale=0.7, mscale_all_dim=0.9),
    dict(attention_factor=1.25, mscale=0.7, mscale_all_dim=0.9),
])
def test_yarn_keys_are_read(extra):
    """Every key that changes a yarn embedding, against the oracle and against transformers, whose frequencies are
    float32: 2^-24 per operation, a few of them."""
    utils = pytest.importorskip("transformers.modeling_rope_utils")
    from transformers import PretrainedConfig

    scaling, rot, base = {**YARN40, **extra}, 64, 1e4
    r = mx.Rotary(rot, base, scaling=scaling)
    inv, factor = op.frequencies(rot, base, scaling)
    np.testing.assert_allclose(r.inv_freq, inv, rtol=1e-13)
    assert r.factor == pytest.approx(factor, rel=1e-14)
    c = PretrainedConfig()
    c.rope_theta, c.head_dim, c.hidden_size, c.num_attention_heads = base, rot, 4 * rot, 4
    c.max_position_embeddings = 40 * 4096
    c.rope_parameters = c.rope_scaling = {**scaling, "rope_type": "yarn", "rope_theta": base}
    want, mag = utils.ROPE_INIT_FUNCTIONS["yarn"](c, torch.device("cpu"))
    np.testing.assert_allclose(r.inv_freq, want.double().numpy(), rtol=1e-6)
    assert r.factor == pytest.approx(mag, rel=1e-12)


@pytest.mark.parametrize("scaling", [
    dict(YARN40, short_factor=[1.0]), dict(YARN40, mscale=0.707), dict(YARN40, mscale_all_dim=1.0),
    dict(YARN40, mscale=0.0, mscale_all_dim=1.0), dict(YARN40, mscale=0.707, mscale_all_dim=0.0),
    dict(YARN40, mscale=math.nan, mscale_all_dim=1.0), dict(YARN40, attention_factor=math.inf),
    dict(YARN40, rope_theta=1e6), dict(type="default", rope_theta=1e6), dict(type="yarn", factor=4.0),
    dict(type="yarn", original_max_position_embeddings=4096), dict(type="linear"),
    dict(type="linear", factor=2.0, attention_factor=1.25), dict(type="linear", factor=2.0, high_freq_factor=4.0),
])
def test_scaling_keys_that_are_not_read_raise(scaling):
    with pytest.raises(ValueError):
        mx.Rotary(64, 1e4, scaling=scaling)


def test_scaling_of_a_whole_configuration():
    """Keys that say what the layer knows, or what text does not use, go with any kind."""
    said = dict(rope_theta=1e4, partial_rotary_factor=0.25, mrope_section=[11, 11, 10], mrope_interleaved=True,
                max_position_embeddings=163840, finetuned=True, beta_fast=None)
    assert mx.Rotary(64, 1e4, scaling={**YARN40, **said}).inv_freq == mx.Rotary(64, 1e4, scaling=YARN40).inv_freq
    assert mx.Rotary(64, 1e4, scaling={"rope_type": "default", **said}).plain
    args = dict(hidden_size=256, num_attention_heads=2, num_key_value_heads=1, head_dim=128, intermediate_size=512,
                rope_theta=1e4)
    mx.Attention(mx.AttentionArgs(**args, rope_scaling={**YARN40, **said}))
    with pytest.raises(ValueError, match="partial_rotary_factor"):
        mx.Attention(mx.AttentionArgs(**args, rope_scaling={**YARN40, "partial_rotary_factor": 1.0}))


def test_layers_take_scaled_frequencies():
    args = mx.AttentionArgs(256, 2, 1, 128, 512, rope_scaling={"type": "linear", "factor": 2.0}, rope_traditional=True)
    layer = mx.Attention(args)
    assert layer.rotary.interleaved and layer.rotary.rot == 32 and layer.rotary.inv_freq[0] == 0.5
    assert mx.Attention(mx.AttentionArgs(256, 2, 1, 128, 512)).rotary.plain


# ------------------------------------------------------------------ oracle

@pytest.mark.parametrize("seed", range(6))
def test_oracle_tables_own_every_block_once(seed):
    """Over random growth and rollback: held and free blocks are always all
    blocks once, and a token's slot stays where it was."""
    rng = np.random.default_rng(seed)
    B, block, width, n = 5, 4, 12, 40
    table, free, held, n_free = np.full((B, width), -1), np.arange(n), [0] * B, n
    lengths = np.zeros(B, int)
    for _ in range(30):
        lengths = np.maximum(lengths - rng.integers(0, 3, B) * rng.integers(0, 8, B), 0)
        T = int(rng.integers(1, 7))
        new = rng.integers(0, T + 1, B)
        before = table.copy()
        slots, held, n_free, table, free = op.tables(lengths, T, table, held, free, n_free, block, new)
        for b in range(B):
            keep = -(-int(lengths[b]) // block)
            np.testing.assert_array_equal(table[b, :keep], before[b, :keep])
        owned = [x for b in range(B) for x in table[b, : held[b]]] + list(free[:n_free])
        assert sorted(owned) == list(range(n))
        got = slots[slots >= 0]
        assert len(set(got.tolist())) == len(got)
        lengths = np.where((slots >= 0).any(1) | (new == 0), lengths + new, lengths)


# ------------------------------------------------------------------- cache

@pytest.fixture
def on_cpu(monkeypatch):
    """The cache's device calls, by the oracle on CPU tensors."""
    def tables(lengths, T, table, held, free, n_free, block, *, n_new=None, shared=0, held_out=None, n_free_out=None):
        s, h, f, t, fr = op.tables(lengths.numpy(), T, table.numpy(), held.numpy(), free.numpy(), n_free.item(), block,
                                   None if n_new is None else n_new.numpy(), shared)
        table.copy_(torch.from_numpy(t))
        free.copy_(torch.from_numpy(fr))
        held_out.copy_(torch.from_numpy(h))
        n_free_out.fill_(int(f))
        return torch.from_numpy(s).to(torch.int32), held_out, n_free_out

    monkeypatch.setattr(paged, "paged_tables", tables)
    monkeypatch.setattr(paged, "_pos_add", lambda pos, delta, lo: pos.add_(delta).clamp_(min=lo))


def _pool(n=40):
    return mx.BlockPool(n, 2, 128, 64)


def _write(cache, T, n_new=None, mark=0):
    """T new tokens a row whose keys are numbered by row and position; returns nothing."""
    new = [T] * cache.batch if n_new is None else n_new
    slots = cache.reserve(T, n_new)
    for b in range(cache.batch):
        for t in range(new[b]):
            s = int(slots[b, t])
            cache.pool.keys[s // 64, :, s % 64] = mark + cache.lengths[b] + t
            cache.pool.values[s // 64, :, s % 64] = -(mark + cache.lengths[b] + t)
    cache.advance(T, n_new)


def _check(cache, marks):
    """Every row's keys are those written, and the host's counts are the device's."""
    assert cache.lengths == cache.pos0.tolist() and cache._held == cache.held.tolist()
    assert cache.pool.free_blocks == int(cache.pool.n_free)
    k, v = cache.state
    assert k.shape[2] == cache.offset
    for b, mark in enumerate(marks):
        n = cache.lengths[b]
        want = (torch.arange(n) + torch.as_tensor(mark)).to(BF).expand(2, n)
        assert torch.equal(k[b, :, :n, 0], want) and torch.equal(v[b, :, :n, 5], -want)


def test_cache_grows_and_rolls_back(on_cpu):
    c = mx.PagedKVCache(_pool(), 3, capacity=64)
    _write(c, 70)
    _write(c, 9, [9, 0, 4])
    assert c.lengths == [79, 70, 74] and c.offset == c.size() == 79 and c.capacity >= 128
    _check(c, [0, 0, 0])
    assert c.trim(20) == 20 and c.lengths == [59, 50, 54]
    assert c.pool.free_blocks == 34
    _write(c, 1)                     # one block a row is enough again: three go back
    assert c.pool.free_blocks == 37
    _check(c, [0, 0, 0])
    assert c.trim(1000) == 60 and c.lengths == [0, 0, 0]
    _write(c, 300)                   # the tables widen
    _check(c, [0, 0, 0])
    c.release()
    assert c.batch == 0 and c.pool.free_blocks == 40 and sorted(c.pool.free.tolist()) == list(range(40))


def test_cache_full_pool_raises_and_stays(on_cpu):
    c = mx.PagedKVCache(_pool(5), 2, 64)
    _write(c, 100)
    with pytest.raises(RuntimeError, match="exhausted"):
        c.reserve(100)
    _check(c, [0, 0])
    _write(c, 20)
    _check(c, [0, 0])


def test_cache_filter_extract_merge(on_cpu):
    pool = _pool()
    a, b = mx.PagedKVCache(pool, 3), mx.PagedKVCache(pool, 1)
    _write(a, 100, [100, 7, 64])
    _write(b, 130, mark=3)
    a.filter([2, 0])
    assert a.lengths == [64, 100] and pool.free_blocks == 40 - 3 - 3
    _check(a, [0, 0])
    e = a.extract(1)
    _check(e, [0])
    _write(e, 5)
    _check(a, [0, 0])
    m = mx.PagedKVCache.merge([a, b])
    assert m.lengths == [64, 100, 130] and a.batch == b.batch == 0
    _check(m, [0, 0, 3])
    _write(m, 2)
    m.release()
    e.release()
    assert pool.free_blocks == 40 and sorted(pool.free.tolist()) == list(range(40))


@pytest.mark.parametrize("at", [0, 1])
@pytest.mark.parametrize("empty", ["left", "fork", "new"])
def test_rows_join_an_empty_batch(on_cpu, empty, at):
    """A batch whose rows have all left (or that never had any) takes rows of any prefix."""
    pool = _pool()
    prompt = mx.PagedKVCache(pool, 1)
    _write(prompt, 150)
    batch = mx.PagedKVCache(pool, 0) if empty == "new" else prompt.fork(2 if empty == "left" else 0)
    if empty == "left":
        batch.filter([])
    joins = prompt.fork(3)
    m = mx.PagedKVCache.merge([batch, joins] if at == 0 else [joins, batch])
    assert m.batch == 3 and m.shared == 2 and joins.batch == batch.batch == 0
    _write(m, 9)
    _check(m, [0] * 3)
    with pytest.raises(RuntimeError, match="fork"):
        prompt.release()
    m.release()
    empties = mx.PagedKVCache.merge([m, joins])
    assert empties.batch == empties.shared == 0
    prompt.release()
    assert pool.free_blocks == 40 and sorted(pool.free.tolist()) == list(range(40))


@pytest.mark.parametrize("keep", [[0, 0], [3], [-1]])
def test_cache_filter_refusals(on_cpu, keep):
    c = mx.PagedKVCache(_pool(), 3)
    with pytest.raises(ValueError):
        c.filter(keep)


def test_forks_share_the_prompt(on_cpu):
    pool = _pool()
    prompt = mx.PagedKVCache(pool, 1)
    _write(prompt, 150)
    f = prompt.fork(4)
    assert f.shared == 2 and f.lengths == [150] * 4 and pool.free_blocks == 40 - 3 - 4
    assert all(torch.equal(f.table[b, :2], prompt.table[0, :2]) for b in range(4))
    _check(f, [0] * 4)
    _write(f, 60, [60, 0, 1, 30])
    _write(prompt, 3)
    _check(f, [0] * 4)
    _check(prompt, [0])
    assert f.trim(1000) == 82 and f.lengths == [128] * 4   # the shared positions stay
    _write(f, 10)
    with pytest.raises(RuntimeError, match="fork"):
        prompt.release()
    assert prompt.trim(1000) == 25 and prompt.lengths == [128]
    g = prompt.fork(2)
    x = f.extract(3)
    assert x.shared == 2
    _check(x, [0])
    m = mx.PagedKVCache.merge([f, x, g])
    assert m.batch == 7 and m.shared == 2 and m.lengths == [138] * 5 + [128] * 2
    _check(m, [0] * 7)
    m.filter([6, 0])
    _check(m, [0, 0])
    m.release()
    prompt.release()
    assert pool.free_blocks == 40 and sorted(pool.free.tolist()) == list(range(40))


def test_forks_of_forks(on_cpu):
    pool = _pool()
    prompt = mx.PagedKVCache(pool, 1)
    _write(prompt, 64)
    f = prompt.fork(1)
    _write(f, 100)
    g = f.fork(3)
    assert (f.shared, g.shared) == (1, 2)
    _check(g, [0] * 3)
    assert f.trim(1000) == 36 and f.lengths == [128]
    for c in (g, f, prompt):
        c.release()
    assert pool.free_blocks == 40 and sorted(pool.free.tolist()) == list(range(40))


@pytest.mark.parametrize("step", ["index_copy_", "index_select", "fill_"])
@pytest.mark.parametrize("make", ["fork", "extract"])
def test_a_copy_that_fails_keeps_no_blocks(on_cpu, monkeypatch, make, step):
    """A fork or an extracted row that cannot be filled (out of memory, say): its blocks are free again, and the
    prompt is nobody's prefix."""
    pool = _pool()
    prompt = mx.PagedKVCache(pool, 1)
    _write(prompt, 150)
    rows = prompt.fork(2)
    _write(rows, 50)
    free = pool.free_blocks

    def fails(*args, **kw):
        raise MemoryError

    with monkeypatch.context() as m:
        m.setattr(torch.Tensor, step, fails)
        with pytest.raises(MemoryError) as kept:  # noqa: F841 (the failed cache lives on in its traceback)
            prompt.fork(3) if make == "fork" else rows.extract(1)
    assert pool.free_blocks == free == int(pool.n_free)
    _check(rows, [0, 0])
    rows.release()
    prompt.release()
    assert pool.free_blocks == 40 and sorted(pool.free.tolist()) == list(range(40))


def test_fork_of_a_short_prompt_shares_nothing(on_cpu):
    pool = _pool(3)
    prompt = mx.PagedKVCache(pool, 1)
    _write(prompt, 10)
    f = prompt.fork(2)
    assert f.shared == 0
    _check(f, [0, 0])
    with pytest.raises(RuntimeError, match="exhausted"):
        prompt.fork(1)
    assert pool.free_blocks == 0
    prompt.release()                  # nothing of it is shared
    _check(f, [0, 0])


def test_cache_state_is_replaced(on_cpu):
    pool = _pool()
    c = mx.PagedKVCache(pool, 2)
    _write(c, 70)
    k = torch.arange(90).to(BF).view(1, 1, 90, 1).expand(3, 2, 90, 128)
    c.state = k, -k
    assert c.batch == 3 and c.lengths == [90] * 3 and pool.free_blocks == 40 - 6
    _check(c, [0] * 3)
    with pytest.raises(ValueError):
        c.state = k[:, :1], -k[:, :1]
    with pytest.raises(RuntimeError, match="exhausted"):
        c.state = k.expand(3, 2, 90, 128).repeat(10, 1, 1, 1), -k.repeat(10, 1, 1, 1)
    _check(c, [0] * 3)


@pytest.mark.parametrize("rows,device,step", [(4097, "cpu", None), (2, "meta", None), (2, "cpu", "reserve"),
                                              (2, "cpu", "advance")])
def test_cache_state_that_cannot_be_replaced_stays(on_cpu, monkeypatch, rows, device, step):
    """More rows than a cache takes, tensors without values, or a step that fails half way: the contents are what
    they were (the pool has room for both), and no block is lost."""
    pool = _pool(5000)
    c = mx.PagedKVCache(pool, 2)
    _write(c, 70)

    def fails(*args, **kw):
        raise MemoryError

    k = torch.zeros(1, 2, 30, 128, dtype=BF, device=device).expand(rows, 2, 30, 128)
    with monkeypatch.context() as m:
        if step:
            m.setattr(mx.PagedKVCache, step, fails)
        with pytest.raises((ValueError, NotImplementedError, MemoryError)):
            c.state = k, k
    assert c.batch == 2 and pool.free_blocks == 5000 - 4
    _check(c, [0, 0])


def test_cache_state_is_replaced_where_only_its_own_blocks_are_left(on_cpu):
    pool = _pool(5)
    c = mx.PagedKVCache(pool, 2)
    _write(c, 100)
    k = torch.arange(60).to(BF).view(1, 1, 60, 1).expand(4, 2, 60, 128)
    c.state = k, -k
    assert c.batch == 4 and pool.free_blocks == 1
    _check(c, [0] * 4)


def test_cache_refusals(on_cpu):
    pool = _pool()
    with pytest.raises(ValueError):
        mx.BlockPool(0, 2, 128)
    with pytest.raises(ValueError):
        mx.BlockPool(4, 2, 128, block=96)
    with pytest.raises(ValueError):
        mx.PagedKVCache(pool, 4097)
    c = mx.PagedKVCache(pool, 2)
    for n_new in ([1], [1, -1], [1, 5]):
        with pytest.raises(ValueError):
            c.reserve(4, n_new)
    with pytest.raises(ValueError):
        c.fork(2)
    with pytest.raises(ValueError):
        c.extract(2)
    with pytest.raises(ValueError):
        mx.PagedKVCache.merge([c, c])
    with pytest.raises(ValueError):
        mx.PagedKVCache.merge([c, mx.PagedKVCache(_pool(), 1)])
    assert pool.free_blocks == 40


def test_ranges_are_within_the_keys():
    for cus in (64, 256):
        for B in (0, 1, 2, 7, 64, 300):
            for T in (0, 1, 3, 17, 200):
                for heads in ((16, 4, 256), (16, 2, 128), (8, 8, 128)):
                    for prefix in (0, 1, 64):
                        for own in (0, 1, 5, 150):
                            p, o, *rows = paged._ranges(cus, B, T, *heads, prefix, own)
                            assert o >= 1 and p <= prefix and set(rows) <= {16, 128}
                            assert o == 1 or 2 * o <= own + (0 if p else prefix)


def test_ranges_read_a_long_prefix_once():
    """Many rows of one token behind a long prefix share its pass; one row, or rows of whole tiles, do not."""
    assert paged._ranges(256, 64, 1, 16, 4, 256, 128, 8)[0] > 1
    assert paged._ranges(256, 32, 4, 16, 4, 256, 256, 11)[0] > 1
    assert paged._ranges(256, 1, 1, 16, 4, 256, 128, 8)[0] == 0
    assert paged._ranges(256, 4, 512, 16, 4, 256, 64, 10)[0] == 0
    assert paged._ranges(256, 1, 1, 16, 4, 256, 0, 500)[1] >= 32


def test_launches_enter_their_tensors_device(monkeypatch):
    """Another device than the current one: every launch is made with it current."""
    import contextlib

    inside, made = [], []

    @contextlib.contextmanager
    def enter(dev):
        inside.append(dev)
        yield
        inside.pop()

    class Library:
        def __getattr__(self, name):
            return lambda *args: made.append((name, len(inside))) or _lib.OK

    monkeypatch.setattr(_lib, "_current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", enter)
    monkeypatch.setattr(_lib, "_lib", Library())
    for mod in (paged, rotary):
        monkeypatch.setattr(mod, "_stream", lambda dev: 0)
        monkeypatch.setattr(mod, "_require_device", lambda tensors, names: torch.device("cpu"))
    monkeypatch.setattr(paged, "_cu_count", lambda dev: 256)
    mx.paged_tables(**_tables_args())
    mx.attn_rope(**_rope_args())
    mx.paged_attn(**_attn_args())
    assert made == [("gdn_paged_tables", 1), ("gdn_attn_rope", 1), ("gdn_paged_attn", 1)]


# ------------------------------------------------- what pins the oracle

@pytest.mark.parametrize("rot,base,scaling", [
    (64, 1e7, dict(type="yarn", factor=4.0, original_max_position_embeddings=32768)),
    (128, 1e6, dict(type="yarn", factor=40.0, original_max_position_embeddings=4096, beta_fast=16.0, beta_slow=2.0)),
])
def test_oracle_frequencies_are_transformers(rot, base, scaling):
    """float32 there: 2^-24 per operation, a few of them."""
    utils = pytest.importorskip("transformers.modeling_rope_utils")
    from transformers import PretrainedConfig

    c = PretrainedConfig()
    c.rope_theta, c.head_dim, c.hidden_size, c.num_attention_heads = base, rot, 4 * rot, 4
    c.max_position_embeddings = int(scaling["factor"] * scaling["original_max_position_embeddings"])
    c.rope_parameters = c.rope_scaling = {**scaling, "rope_type": scaling["type"], "rope_theta": base}
    inv, factor = utils.ROPE_INIT_FUNCTIONS["yarn"](c, torch.device("cpu"))
    ours, mag = op.frequencies(rot, base, scaling)
    np.testing.assert_allclose(inv.double().numpy(), ours, rtol=1e-6)
    assert mag == pytest.approx(factor, rel=1e-12)


def test_oracle_rotation_is_the_dense_oracles():
    from oracle import attention as oa

    rng = np.random.default_rng(1)
    x, w, pos = rng.standard_normal((5, 3, 128)), rng.standard_normal(128), np.arange(5) + 17
    inv, factor = op.frequencies(32, 1e4)
    want = oa.rope(oa.rms_norm(x, w, 1e-6)[None], pos[None], 32, 1e4)[0]
    np.testing.assert_allclose(op.norm_rotate(x, w, 1e-6, pos, inv, factor, False), want, atol=1e-12)
    # neighbouring pairs are one complex number each
    y = op.norm_rotate(x, None, 0.0, pos, inv, 1.5, True)
    z = (x[..., 0:32:2] + 1j * x[..., 1:32:2]) * np.exp(1j * pos[:, None, None] * inv) * 1.5
    np.testing.assert_allclose(y[..., 0:32:2] + 1j * y[..., 1:32:2], z, atol=1e-12)
    np.testing.assert_array_equal(y[..., 32:], x[..., 32:])


def test_oracle_attention_is_the_dense_softmax():
    rng = np.random.default_rng(2)
    B, T, Hq, Hkv, D, block = 2, 3, 4, 2, 8, 4
    pos0, n_new = [6, 0], [3, 2]
    keys, values = rng.standard_normal((2, 9, Hkv, block, D))
    table = np.array([[4, 7, 2], [8, 0, 1]])
    q, gate = rng.standard_normal((2, B, T, Hq, D))
    out = op.attend(q, keys, values, table, pos0, 0.3, n_new, gate)
    for b in range(B):
        k = torch.from_numpy(keys[table[b]]).transpose(0, 1).reshape(Hkv, -1, D).repeat_interleave(2, 0)
        v = torch.from_numpy(values[table[b]]).transpose(0, 1).reshape(Hkv, -1, D).repeat_interleave(2, 0)
        n = n_new[b]
        sees = torch.arange(k.shape[1]) <= pos0[b] + torch.arange(n)[:, None]
        s = (torch.from_numpy(q[b, :n]).transpose(0, 1) @ k.transpose(1, 2) * 0.3).masked_fill(~sees, -math.inf)
        want = (s.softmax(-1) @ v).transpose(0, 1) * torch.from_numpy(gate[b, :n]).sigmoid()
        np.testing.assert_allclose(out[b, :n], want.numpy(), atol=1e-12)
        assert not out[b, n:].any()
