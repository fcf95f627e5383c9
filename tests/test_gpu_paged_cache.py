"""The paged cache and the layers on it, on the GPU: a paged batch against the
same rows in a dense cache, forks of a prompt, the MTP head, a captured step,
and other streams.

LAYER_TOL = 1e-2: both paths round at the same points (the rotary prep is the
same kernel, bit for bit); what differs is the attention rows, each within
5e-3 of the exact ones in norm (their own and the softmax weights' rounding to
bf16, 2 u / sqrt(3) with 10% to spare, u = 2^-8), carried through o_proj and the
MLP: twice that.
"""

from __future__ import annotations

import pytest
import torch

import multiplex_amd as mx

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
LAYER_TOL = 1e-2
ARGS = dict(hidden_size=512, num_attention_heads=8, num_key_value_heads=2, head_dim=128, intermediate_size=1024)
# neighbouring pairs and a long-context scaling: the dense cache takes the same rotary prep then
ROPE = dict(rope_traditional=True, rope_scaling={"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096})


def _rel(a, b):
    a, b = a.double(), b.double()
    return ((a - b).norm(dim=-1) / b.norm(dim=-1)).max().item()


def _x(gen, B, T):
    return torch.randn(B, T, ARGS["hidden_size"], generator=gen).to(BF).to(DEV)


@pytest.mark.parametrize("head_dim", [128, 256])
def test_paged_layer_equals_dense_layer(head_dim):
    """Prefill, decode, verify, rollback, more prefill, with a rotary that both caches take."""
    torch.manual_seed(1)
    gen = torch.Generator().manual_seed(1)
    layer = mx.DecoderLayer(mx.AttentionArgs(**{**ARGS, "head_dim": head_dim}, **ROPE), DEV)
    B = 3
    dense = mx.KVCache(B, 2, head_dim, 256, DEV)
    pool = mx.BlockPool(40, 2, head_dim, 64, DEV)
    cache = mx.PagedKVCache(pool, B)
    for T, back in ((100, 0), (1, 0), (4, 3), (1, 0), (150, 10), (1, 0)):
        x = _x(gen, B, T)
        a, b = layer(x, dense), layer(x, cache)
        assert _rel(b, a) < LAYER_TOL, T
        dense.trim(back)
        assert cache.trim(back) == back
    assert cache.lengths == dense.lengths and cache.pos0.tolist() == cache.lengths
    for k, want in zip(cache.state, dense.state):
        assert torch.equal(k, want)
    assert cache.pool.free_blocks == int(pool.n_free) and cache.held.tolist() == cache._held


def test_plain_rotary_on_a_paged_cache():
    """Unscaled half pairs: the dense path rounds once more, before the rotation (k within two roundings)."""
    torch.manual_seed(2)
    gen = torch.Generator().manual_seed(2)
    layer = mx.Attention(mx.AttentionArgs(**ARGS), DEV)
    dense, cache = mx.KVCache(2, 2, 128, 256, DEV), mx.PagedKVCache(mx.BlockPool(20, 2, 128, 64, DEV), 2)
    x = _x(gen, 2, 90)
    a, b = layer(x, dense), layer(x, cache)
    # scores change by a rounding of q and of k (u / sqrt 3 each in norm): beside the attention's own error
    # on either side, the weights and so the rows move by as much again
    assert _rel(b, a) < 2 * LAYER_TOL
    (k, v), (kd, vd) = cache.state, dense.state
    assert torch.equal(v, vd)
    assert _rel(k, kd) < 8e-3  # 2 u


def test_ragged_rows_equal_rows_alone():
    torch.manual_seed(3)
    gen = torch.Generator().manual_seed(3)
    layer = mx.Attention(mx.AttentionArgs(**ARGS, **ROPE), DEV)
    pool = mx.BlockPool(60, 2, 128, 64, DEV)
    batch, alone = mx.PagedKVCache(pool, 4), [mx.PagedKVCache(pool, 1) for _ in range(4)]
    for T, n_new in ((130, [130, 7, 0, 64]), (5, [0, 5, 3, 1]), (1, [1, 1, 1, 1])):
        x = _x(gen, 4, T)
        for b, n in enumerate(n_new):
            x[b, n:] = float("nan")  # padding
        y = layer(x, batch, n_new=n_new)
        for b, n in enumerate(n_new):
            if n:
                assert _rel(y[b, :n], layer(x[b : b + 1, :n], alone[b])[0]) < LAYER_TOL
    assert batch.lengths == [131, 13, 4, 66] and batch.pos0.tolist() == batch.lengths
    m = mx.PagedKVCache.merge(alone)
    n = min(m.lengths)
    for a, b in zip(batch.state, m.state):
        assert torch.equal(a[:, :, :n], b[:, :, :n])
    with pytest.raises(ValueError, match="PagedKVCache"):
        layer(x, mx.KVCache(4, 2, 128, 256, DEV), n_new=[1] * 4)


def test_a_step_padded_past_a_fresh_caches_tables():
    """The tables list what the rows' real tokens need, however wide the call is padded."""
    torch.manual_seed(11)
    gen = torch.Generator().manual_seed(11)
    layer = mx.Attention(mx.AttentionArgs(**ARGS, **ROPE), DEV)
    pool = mx.BlockPool(20, 2, 128, 64, DEV)
    cache, alone = mx.PagedKVCache(pool, 2), [mx.PagedKVCache(pool, 1) for _ in range(2)]
    for T, n_new in ((300, [10, 5]), (512, [1, 0]), (700, [0, 200])):
        x = _x(gen, 2, T)
        y = layer(x, cache, n_new=n_new)
        for b, n in enumerate(n_new):
            if n:
                assert _rel(y[b, :n], layer(x[b : b + 1, :n], alone[b])[0]) < LAYER_TOL
    assert cache.lengths == cache.pos0.tolist() == [11, 205] and cache.capacity == 256


@pytest.mark.parametrize("rows", [1, 5, 40])
def test_forks_equal_whole_rows(rows):
    """A batch on a shared prompt against each row's prompt kept densely, through
    decode, a verify with rollback, and rows leaving."""
    torch.manual_seed(4)
    gen = torch.Generator().manual_seed(4)
    layer = mx.Attention(mx.AttentionArgs(**ARGS, **ROPE), DEV)
    pool = mx.BlockPool(20 + 6 * rows, 2, 128, 64, DEV)
    prompt = mx.PagedKVCache(pool, 1)
    x = _x(gen, 1, 333)
    layer(x, prompt)
    dense = mx.KVCache(rows, 2, 128, 512, DEV)
    layer(x.expand(rows, -1, -1).contiguous(), dense)
    fork = prompt.fork(rows)
    assert fork.shared == 5
    for T, back in ((1, 0), (4, 2), (1, 0), (70, 0), (1, 0)):
        x = _x(gen, fork.batch, T)
        assert _rel(layer(x, fork), layer(x, dense)) < LAYER_TOL, T
        fork.trim(back)
        dense.trim(back)
        if rows > 1 and T == 70:
            keep = list(range(0, rows, 2))[::-1]
            fork.filter(keep)
            dense.filter(keep)
    assert fork.lengths == dense.lengths
    for a, b in zip(fork.state, dense.state):
        assert torch.equal(a, b)
    fork.release()
    prompt.release()
    assert pool.free_blocks == int(pool.n_free) == pool.n_blocks
    assert sorted(pool.free.tolist()) == list(range(pool.n_blocks))


def test_mtp_head_on_paged_caches():
    torch.manual_seed(5)
    gen = torch.Generator().manual_seed(5)
    head = mx.MTPHead(mx.AttentionArgs(**ARGS, **ROPE), n_layers=2, device=DEV)
    dense, cache = head.make_cache(3), head.make_paged_cache(3, 30)
    for T, size in ((80, 80), (1, 81), (1, 82), (1, 80), (2, 82)):
        e, h = _x(gen, 3, T), _x(gen, 3, T)
        assert _rel(head(e, h, cache), head(e, h, dense)) < 2 * LAYER_TOL  # two layers
        head.trim_cache_to(cache, size)
        head.trim_cache_to(dense, size)
    assert cache[0].lengths == dense[0].lengths == [82] * 3


def _step(s, T):
    slots, _, _ = mx.paged_tables(s["pos0"], T, s["table"], s["held"], s["free"], s["n_free"], 64, shared=2,
                                  held_out=s["held"], n_free_out=s["n_free"])
    q = mx.attn_rope(s["qg"], s["k"], s["v"], s["w"], s["w"], 1e-6, s["pos0"], s["keys"], s["values"], s["rotary"],
                     slots=slots)
    o = mx.paged_attn(q, s["keys"], s["values"], s["table"], s["pos0"], 600, shared=2, gate=s["qg"])
    s["pos0"].add_(T)
    return o


def _step_state(seed, T):
    gen = torch.Generator().manual_seed(seed)
    B, Hq, Hkv, D, n = 6, 16, 4, 256, 60
    i32 = dict(dtype=torch.int32, device=DEV)
    wide = torch.randn(B, T, (2 * Hq + 2 * Hkv) * D, generator=gen).to(BF).to(DEV)
    qg, k, v = wide.split((2 * Hq * D, Hkv * D, Hkv * D), -1)
    table = torch.zeros(B, 10, **i32)
    table[:, :2] = torch.tensor([57, 3])
    free = torch.tensor([i for i in range(n) if i not in (3, 57)] + [0, 0], **i32)
    return dict(qg=qg, k=k, v=v, wide=wide, w=torch.ones(D, device=DEV), pos0=torch.full((B,), 128, **i32), table=table,
                held=torch.full((B,), 2, **i32), free=free, n_free=torch.full((1,), n - 2, **i32),
                keys=torch.randn(n, Hkv, 64, D, generator=gen).to(BF).to(DEV),
                values=torch.randn(n, Hkv, 64, D, generator=gen).to(BF).to(DEV),
                rotary=mx.Rotary(64, 1e7, device=DEV))


@pytest.mark.parametrize("T", [1, 3, 200])
def test_captured_step_replays(T):
    """Tables, append, attention and advance in one graph, replayed over growing
    rows with other work between, against the same steps run eagerly."""
    a, b = _step_state(6, T), _step_state(6, T)
    first = _step(a, T)  # a warm step outside the capture, on both
    assert torch.equal(first, _step(b, T))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(a, T)
    gen = torch.Generator().manual_seed(7)
    for i in range({1: 70, 3: 5, 200: 1}[T]):
        new = torch.randn(*a["wide"].shape, generator=gen).to(BF)
        a["wide"].copy_(new)
        b["wide"].copy_(new)
        graph.replay()
        want = _step(b, T)
        (a["wide"].float().sum() + want.float().sum()).item()
        assert torch.equal(out, want), i
    for n in ("table", "held", "free", "n_free", "pos0", "keys", "values"):
        assert torch.equal(a[n], b[n]), n


def test_other_stream():
    s, want = _step_state(8, 3), _step(_step_state(8, 3), 3)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = _step(s, 3)
    stream.synchronize()
    assert torch.equal(out, want)


def test_two_workspaces_on_two_streams():
    """Calls at once, each with a workspace of its own."""
    states = [_step_state(9, 1), _step_state(10, 1)]
    want = [_step(_step_state(9, 1), 1), _step(_step_state(10, 1), 1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    outs = []
    for st, s in zip(streams, states):
        with torch.cuda.stream(st):
            outs.append(_step(s, 1))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


@pytest.mark.parametrize("T", [1, 300])
def test_a_batch_of_no_rows(T):
    layer = mx.Attention(mx.AttentionArgs(**ARGS), DEV)
    cache = mx.PagedKVCache(mx.BlockPool(4, 2, 128, 64, DEV), 0)
    assert layer(torch.empty(0, T, 512, dtype=BF, device=DEV), cache).shape == (0, T, 512)
    assert cache.offset == 0 and cache.pool.free_blocks == 4


def test_counts_are_not_captured():
    cache = mx.PagedKVCache(mx.BlockPool(4, 2, 128, 64, DEV), 2)
    cache.reserve(2, [1, 2])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            cache.reserve(2, [1, 2])


@pytest.mark.parametrize("verb", ["reserve", "advance", "trim"])
def test_a_caches_steps_are_not_captured(verb):
    """The host's lengths and counts would not move with the replays."""
    c = mx.PagedKVCache(mx.BlockPool(8, 1, 128, 64, DEV), 2)
    c.reserve(70)
    c.advance(70)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capture"):
            getattr(c, verb)(3)
    assert c.lengths == [70, 70] and c._held == [2, 2] and c.pool.free_blocks == 4
    assert c.reserve(1).tolist() and c.held.tolist() == [2, 2] and c.pool.n_free.tolist() == [4]


def test_state_from_the_host():
    """Stored keys and values come back from host memory, as into a dense cache."""
    gen = torch.Generator().manual_seed(12)
    k, v = torch.randn(2, 3, 2, 90, 128, generator=gen)
    cache, dense = mx.PagedKVCache(mx.BlockPool(8, 2, 128, 64, DEV), 2), mx.KVCache(3, 2, 128, 256, DEV)
    cache.reserve(70)
    cache.advance(70)
    for c in (cache, dense):
        c.state = k, v
    assert cache.lengths == cache.pos0.tolist() == [90] * 3 and cache.pool.free_blocks == 2
    for a, b in zip(cache.state, dense.state):
        assert torch.equal(a, b)


def test_rows_past_the_batch_are_left_alone():
    """Buffers longer than the batch (views of a serving loop's largest): what lies behind stays."""
    i32 = dict(dtype=torch.int32, device=DEV)
    lengths, held, slots = torch.full((6,), 3, **i32), torch.full((6,), 9, **i32), torch.full((6, 2), 77, **i32)
    table = torch.full((6, 4), 55, **i32)
    held[:2] = 0
    free, n_free = torch.arange(8, **i32), torch.full((1,), 8, **i32)
    mx.paged_tables(lengths[:2], 2, table[:2], held[:2], free, n_free, 4, slots=slots[:2], held_out=held[:2],
                    n_free_out=n_free)
    assert held.tolist() == [2, 2, 9, 9, 9, 9] and (table[2:] == 55).all() and (slots[2:] == 77).all()
    assert table[:2].tolist() == [[7, 6, 55, 55], [5, 4, 55, 55]] and n_free.item() == 4
    assert slots[:2].tolist() == [[31, 24], [23, 16]]
