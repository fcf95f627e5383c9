"""The paged attention cache on the GPU against the float64 oracle
(``oracle/paged.py``): block tables (exactly), the rotary prep and attention
over tables, then the cache and the layers that use it.

Tolerances are relative norms per row.  u = 2^-8 is the unit roundoff of bf16:
one rounding's relative error per element lies in [-u, u], RMS at most
u / sqrt(3) = 2.3e-3 over a row (uniform over a half ulp, at the mantissa's low
end).

* ROPE_TOL = 4e-3: the only bf16 rounding is the output's, at most u = 3.9e-3 on
  every element and so on the row's norm; the fp32 arithmetic before it is below
  1e-6.
* ATT_TOL = 5e-3: the output's rounding and that of the softmax weights, which
  are rounded to bf16 for the product with V (their sum is not), add up to at
  most 2 u / sqrt(3) with 10% to spare.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import multiplex_amd as mx
from oracle import paged as op

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROPE_TOL = 4e-3
ATT_TOL = 5e-3


def _np(t):
    return t.double().cpu().numpy()


def _errs(y, ref):
    y, ref = np.asarray(y, np.float64), np.asarray(ref, np.float64)
    num = np.linalg.norm((y - ref).reshape(-1, y.shape[-1]), axis=-1)
    return num / np.maximum(np.linalg.norm(ref.reshape(-1, y.shape[-1]), axis=-1), 1e-30)


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ tables

def _tables_case(rng, B, T, block, shared, longest, ragged, spare, width=None):
    """Rows that hold what their lengths need (some a block more or less), tables of distinct blocks."""
    lengths = shared * block + rng.integers(0, longest + 1, B)
    held = -(-lengths // block)
    held = np.maximum(held + (rng.integers(0, 6, B) == 0) * rng.integers(0, 3, B), shared)
    lengths = np.where(rng.integers(0, 8, B) == 0, 0, lengths)  # rows that left
    n_new = rng.integers(-1, T + 2, B) if ragged else None
    width = int(max(held.max(), shared, 1)) + (T + block - 1) // block + 2 if width is None else width
    held = np.minimum(held, width)
    n = int(shared + (held - np.minimum(shared, held)).sum() + spare)
    order = rng.permutation(n)
    table = np.full((B, width), -7)
    table[:, :shared] = order[:shared]
    at = shared
    for b in range(B):
        k = held[b] - shared
        table[b, shared:held[b]] = order[at:at + k]
        at += k
    free = np.full(n, -9)
    free[:n - at] = order[at:]
    return lengths, n_new, table, held, free, n - at


@pytest.mark.parametrize("B,T,block,shared,longest,ragged,spare", [
    (1, 1, 64, 0, 0, False, 1),          # an empty row's first token
    (1, 1, 64, 0, 0, False, 0),          # ... and no block for it
    (3, 1, 64, 2, 200, False, 3),
    (5, 9, 128, 0, 700, True, 2),        # the list runs out
    (17, 70, 64, 3, 1000, True, 40),
    (256, 1, 64, 0, 4000, False, 300),
    (257, 3, 256, 1, 4000, True, 9),     # two rows a thread, the list runs out
    (1000, 9, 128, 16, 4000, True, 2000),
    (48, 512, 64, 32, 6000, True, 500),  # several workgroups
    (2, 4096, 64, 0, 100, False, 130),
    (4096, 1, 64, 0, 100, False, 2000),
    (7, 33, 1, 5, 40, True, 300),        # blocks of one position
    (4, 0, 64, 1, 300, False, 2),        # no tokens: blocks given back only
])
@pytest.mark.parametrize("in_place", [False, True])
def test_tables_match_oracle(B, T, block, shared, longest, ragged, spare, in_place):
    rng = np.random.default_rng(B * 1000 + T)
    lengths, n_new, table, held, free, n_free = _tables_case(rng, B, T, block, shared, longest, ragged, spare)
    ref = op.tables(lengths, T, table, held, free, n_free, block, n_new, shared)
    d = dict(lengths=_i32(lengths), table=_i32(table), held=_i32(held), free=_i32(free), n_free=_i32([n_free]))
    out = dict(held_out=d["held"], n_free_out=d["n_free"]) if in_place else {}
    for _ in range(1 if in_place else 2):  # without in-place counts the call can be repeated
        slots, h, f = mx.paged_tables(d["lengths"], T, d["table"], d["held"], d["free"], d["n_free"], block,
                                      n_new=None if n_new is None else _i32(n_new), shared=shared, **out)
        torch.cuda.synchronize()
        for got, want in zip((slots, h, f[0], d["table"], d["free"]), ref):
            np.testing.assert_array_equal(got.cpu().numpy(), want)
    if in_place:
        assert h is d["held"] and f is d["n_free"]


@pytest.mark.parametrize("B,T,block,shared,longest,ragged,spare", [
    (1024, 2, 64, 1, 700, True, 900),    # the last batch of one row a thread
    (1025, 3, 64, 2, 900, True, 2000),   # four rows a thread, the last thread's mostly past the batch
    (1027, 100, 64, 0, 300, False, 40),  # ... the list runs out, several workgroups
    (3001, 130, 128, 1, 500, True, 60),  # ... many workgroups, the list all but empty
    (4095, 5, 64, 3, 200, True, 4000),
    (4096, 1, 256, 2, 2000, True, 700),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_tables_of_many_ragged_rows(B, T, block, shared, longest, ragged, spare, in_place):
    """Over 1024 rows a thread of tables_kernel takes four: batches that end inside a thread's, ragged and shared."""
    rng = np.random.default_rng(B * 1000 + T)
    lengths, n_new, table, held, free, n_free = _tables_case(rng, B, T, block, shared, longest, ragged, spare)
    ref = op.tables(lengths, T, table, held, free, n_free, block, n_new, shared)
    d = dict(lengths=_i32(lengths), table=_i32(table), held=_i32(held), free=_i32(free), n_free=_i32([n_free]))
    out = dict(held_out=d["held"], n_free_out=d["n_free"]) if in_place else {}
    for _ in range(1 if in_place else 2):
        slots, h, f = mx.paged_tables(d["lengths"], T, d["table"], d["held"], d["free"], d["n_free"], block,
                                      n_new=None if n_new is None else _i32(n_new), shared=shared, **out)
        torch.cuda.synchronize()
        for got, want in zip((slots, h, f[0], d["table"], d["free"]), ref):
            np.testing.assert_array_equal(got.cpu().numpy(), want)


def test_tables_row_too_long_for_its_table():
    """A row that needs more blocks than its table is wide keeps what it holds
    and gets no slots; the others go on."""
    lengths, held, width = [100, 64 * 3, 10], [2, 3, 1], 3
    table = np.array([[4, 5, -1], [0, 1, 2], [3, -1, -1]])
    free = np.array([6, 7, 8, -1, -1, -1, -1, -1, -1])
    ref = op.tables(lengths, 30, table, held, free, 3, 64)
    d = _i32(table), _i32(free)
    slots, h, f = mx.paged_tables(_i32(lengths), 30, d[0], _i32(held), d[1], _i32([3]), 64)
    for got, want in zip((slots, h, f[0], *d), ref):
        np.testing.assert_array_equal(got.cpu().numpy(), want)
    assert (slots[1] == -1).all() and h.tolist() == [3, 3, 1]


# -------------------------------------------------------------------- rope

YARN = {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}


@pytest.mark.parametrize("B,T,Hq,Hkv,D,rot,interleaved,scaling,gated,wdt,far", [
    (3, 5, 16, 4, 256, 64, False, None, True, torch.float32, 100),
    (3, 5, 16, 4, 256, 64, False, YARN, True, torch.bfloat16, 2_000_000_000),
    (2, 7, 16, 4, 256, 256, True, YARN, False, torch.float16, 1_000_000),
    (1, 1, 4, 4, 128, 128, True, {"type": "linear", "factor": 2.5}, True, torch.float32, 70000),
    (4, 33, 12, 4, 128, 32, False, {"type": "linear", "factor": 8.0}, False, None, 70000),
    (1, 600, 16, 2, 256, 128, False, None, True, torch.float32, 10),    # three heads a wave
    (2, 500, 32, 8, 128, 64, True, None, True, torch.bfloat16, 5000),   # six heads a wave
    (2, 3, 5, 1, 256, 6, True, None, False, torch.float32, 300),        # a lane of two rotated, two plain dims
    (2, 3, 5, 1, 128, 0, False, None, True, torch.float32, 300),        # nothing rotated
    (3, 7, 6, 2, 256, 72, False, YARN, True, torch.float32, 300),       # pairs that end inside a lane's dims
    (3, 7, 7, 7, 128, 10, False, None, True, torch.bfloat16, 300),      # heads that end inside a group
    (2, 900, 7, 1, 128, 128, False, None, True, torch.float32, 300),    # ... several groups a wave
    (2, 900, 5, 1, 256, 100, True, None, False, torch.float16, 3000),
])
def test_rope_matches_oracle(B, T, Hq, Hkv, D, rot, interleaved, scaling, gated, wdt, far):
    """Against the oracle, with column slices at odd offsets, padded tokens, and slots in any order."""
    gen = torch.Generator().manual_seed(B * 100 + T)
    per, block = (2 * D if gated else D), 64
    wide = torch.randn(B, T, Hq * per + 2 * Hkv * D + 1, generator=gen).to(torch.bfloat16)
    cols = (1, 1 + Hq * per, 1 + Hq * per + Hkv * D, 1 + Hq * per + 2 * Hkv * D)
    n_blocks = B * T // block + 3
    slots = torch.randperm(n_blocks * block, generator=gen)[:B * T].view(B, T).to(torch.int32)
    n_new = torch.randint(0, T + 1, (B,), generator=gen) if B > 1 else torch.full((B,), T)
    slots[torch.arange(T) >= n_new[:, None]] = -1
    pos0 = torch.randint(0, far, (B,), generator=gen).to(torch.int32)
    w = [None, None] if wdt is None else [(torch.randn(D, generator=gen) * 0.2 + 1).to(wdt) for _ in range(2)]
    keys = torch.randn(n_blocks, Hkv, block, D, generator=gen).to(torch.bfloat16)
    values = torch.randn(n_blocks, Hkv, block, D, generator=gen).to(torch.bfloat16)
    dw, dk, dv = wide.to(DEV), keys.to(DEV), values.to(DEV)
    rotary = mx.Rotary(rot, 1e7, interleaved=interleaved, scaling=scaling, device=DEV)
    parts = [dw[..., a:b] for a, b in zip(cols, cols[1:])]
    q = mx.attn_rope(*parts, *(None if x is None else x.to(DEV) for x in w), 1e-6, pos0.to(DEV), dk, dv, rotary,
                     slots=slots.to(DEV), gated=gated)
    torch.cuda.synchronize()
    inv, factor = op.frequencies(rot, 1e7, scaling) if rot else (np.zeros(0), 1.0)
    rk, rv = _np(keys), _np(values)
    h = [None if x is None else _np(x) for x in w]
    for b in range(B):
        n = int(n_new[b])
        pos = int(pos0[b]) + np.arange(n)
        x = _np(wide[b, :n])
        ref = op.norm_rotate(x[:, cols[0]:cols[1]].reshape(n, Hq, per)[..., :D], h[0], 1e-6, pos, inv, factor, interleaved)
        assert _errs(_np(q[b, :n]), ref).max(initial=0) < ROPE_TOL
        assert not q[b, n:].any()
        s = slots[b, :n].numpy()
        rk[s // block, :, s % block] = op.norm_rotate(x[:, cols[1]:cols[2]].reshape(n, Hkv, D), h[1], 1e-6, pos, inv,
                                                      factor, interleaved)
        rv[s // block, :, s % block] = x[:, cols[2]:cols[3]].reshape(n, Hkv, D)
    assert _errs(_np(dk), rk).max() < ROPE_TOL
    np.testing.assert_array_equal(_np(dv), rv)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot,norm", [
    (256, 64, False), (256, 64, True), (128, 0, False), (256, 6, False), (256, 72, False), (256, 72, True),
    (128, 128, False), (128, 10, True),
])
def test_rope_keeps_infinities_where_they_are(D, rot, norm, interleaved):
    """inf and NaN in a live token: a dim that does not turn is its own alone (without a norm bit for bit), a pair
    that turns takes what the definition gives it, and with a norm an inf makes the other dims 0, a NaN all NaN.
    Finite values to a rounding, 2^-8 of the value; the angle's fp32 (below 1e-6) times |x| |w| < 20 beside it."""
    gen = torch.Generator().manual_seed(D + rot)
    B, T, Hq, Hkv = 2, 6, 4, 2
    q, k = (torch.randn(B, T, H, D, generator=gen).to(torch.bfloat16) for H in (Hq, Hkv))
    for x in (q, k):
        for t, (d, v) in enumerate([(D - 3, np.inf), (D - 4, np.nan), (rot, -np.inf), (rot + 1, np.nan), (2, np.inf)]):
            x[0, t, 0, d % D] = v
            x[1, t, -1, (d + 1) % D] = v
    v = torch.randn(B, T, Hkv * D, generator=gen).to(torch.bfloat16)
    w = torch.randn(D, generator=gen) * 0.2 + 1 if norm else None
    keys = torch.zeros(1, Hkv, 64, D, dtype=torch.bfloat16, device=DEV)
    values = torch.zeros_like(keys)
    rotary = mx.Rotary(rot, 1e4, interleaved=interleaved, device=DEV)
    dw = None if w is None else w.to(DEV)
    pos0, slots = [3, 50], np.arange(B * T).reshape(B, T)
    got = mx.attn_rope(q.view(B, T, -1).to(DEV), k.view(B, T, -1).to(DEV), v.to(DEV), dw, dw, 1e-6, _i32(pos0), keys,
                       values, rotary, slots=_i32(slots), gated=False)
    stored = keys[0].transpose(0, 1)[:B * T].reshape(B, T, Hkv, D)
    inv, factor = op.frequencies(rot, 1e4) if rot else (np.zeros(0), 1.0)
    for x, y in ((q, got), (k, stored)):
        for b in range(B):
            with np.errstate(invalid="ignore"):
                ref = op.norm_rotate(_np(x[b]), None if w is None else _np(w), 1e-6, pos0[b] + np.arange(T), inv, factor,
                                     interleaved)
            np.testing.assert_allclose(_np(y[b]), ref, rtol=2.0**-8, atol=2e-5)
            if not norm:
                np.testing.assert_array_equal(_np(y[b])[..., rot:], _np(x[b])[..., rot:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_into_a_dense_cache(interleaved):
    gen = torch.Generator().manual_seed(3)
    B, T, Hq, Hkv, D, rot, cap = 3, 5, 8, 2, 256, 64, 70
    x = torch.randn(B, T, (2 * Hq + 2 * Hkv) * D, generator=gen).to(torch.bfloat16)
    w = torch.randn(D, generator=gen) * 0.2 + 1
    pos0 = [0, 17, 90]  # the last is clamped so that its tokens fit
    kc = torch.zeros(B, Hkv, cap, D, dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)
    parts = x.to(DEV).split((2 * Hq * D, Hkv * D, Hkv * D), -1)
    rotary = mx.Rotary(rot, 1e7, interleaved=interleaved, scaling=YARN, device=DEV)
    q = mx.attn_rope(*parts, w.to(DEV), w.to(DEV), 1e-6, _i32(pos0), kc, vc, rotary)
    inv, factor = op.frequencies(rot, 1e7, YARN)
    for b, p0 in enumerate((0, 17, cap - T)):
        pos, xb = p0 + np.arange(T), _np(x[b])
        ref = op.norm_rotate(xb[:, :2 * Hq * D].reshape(T, Hq, 2 * D)[..., :D], _np(w), 1e-6, pos, inv, factor, interleaved)
        assert _errs(_np(q[b]), ref).max() < ROPE_TOL
        k = op.norm_rotate(xb[:, 2 * Hq * D:][:, :Hkv * D].reshape(T, Hkv, D), _np(w), 1e-6, pos, inv, factor, interleaved)
        assert _errs(_np(kc[b, :, p0:p0 + T]), k.transpose(1, 0, 2)).max() < ROPE_TOL
        np.testing.assert_array_equal(_np(vc[b, :, p0:p0 + T]), xb[:, (2 * Hq + Hkv) * D:].reshape(T, Hkv, D).transpose(1, 0, 2))
        rest = np.ones(cap, bool)
        rest[p0:p0 + T] = False
        assert not _np(kc[b])[:, rest].any() and not _np(vc[b])[:, rest].any()


# --------------------------------------------------------------- attention

def _attn_case(gen, B, T, heads, block, shared, tails, n_new, spare=2):
    """Pools whose unused places hold NaN, tables whose unused entries lie outside the pool."""
    Hq, Hkv, D = heads
    pos0 = [shared * block + t for t in tails]
    width = max(-(-(p + T) // block) for p in pos0) + 1
    need = [-(-(p + (T if n_new is None else n_new[b])) // block) for b, p in enumerate(pos0)]
    n = shared + sum(max(k - shared, 0) for k in need) + spare
    order = torch.randperm(n, generator=gen).tolist()
    table = np.full((B, width), -5)
    table[:, -1] = 2**30
    table[:, :shared] = order[:shared]
    at = shared
    keys = torch.full((n, Hkv, block, D), float("nan"))
    values = keys.clone()
    for b in range(B):
        for c in range(shared, need[b]):
            table[b, c] = order[at]
            at += 1
    for b in range(B):
        L = pos0[b] + (T if n_new is None else n_new[b])
        for c in range(need[b]):
            m = min(block, L - c * block)
            if c < shared and b:
                continue
            keys[table[b, c], :, :m] = torch.randn(Hkv, m, D, generator=gen)
            values[table[b, c], :, :m] = torch.randn(Hkv, m, D, generator=gen)
    q = torch.randn(B, T, Hq, D, generator=gen)
    gate = torch.randn(B, T, Hq, 2 * D, generator=gen)
    if n_new is not None:
        pad = torch.arange(T) >= torch.tensor(n_new)[:, None]
        q[pad], gate[pad] = float("nan"), float("nan")
    bf = torch.bfloat16
    return q.to(bf), gate.to(bf), keys.to(bf), values.to(bf), table, pos0


CASES = {
    # name: (B, T, (Hq, Hkv, D), block, shared blocks, own lengths before the call, n_new, n_split, gate)
    "one_token_of_one": (1, 1, (16, 4, 256), 64, 0, [0], None, None, True),
    "decode": (5, 1, (16, 4, 256), 64, 3, [0, 1, 63, 64, 300], None, None, True),
    "decode_ranges": (5, 1, (16, 4, 256), 64, 3, [0, 1, 63, 64, 300], None, (3, 4), True),
    "decode_apart": (5, 1, (16, 4, 256), 64, 3, [0, 1, 63, 64, 300], None, (0, 1), False),
    "decode_apart_ranges": (5, 1, (16, 4, 256), 64, 0, [0, 1, 63, 64, 300], None, (0, 5), True),
    "decode_d128": (6, 1, (16, 4, 128), 128, 2, [5, 1, 63, 64, 300, 127], None, (2, 2), True),
    "decode_g8": (3, 1, (16, 2, 256), 256, 1, [0, 255, 256], None, (4, 1), True),
    "decode_mha": (7, 1, (3, 3, 128), 64, 2, [9, 1, 0, 64, 30, 2, 3], None, (1, 1), False),
    "decode_many_rows": (40, 1, (16, 4, 256), 64, 5, [7 * b for b in range(40)], None, None, True),
    "verify": (4, 4, (16, 4, 256), 64, 2, [3, 100, 257, 0], None, None, True),
    "verify_padded": (5, 4, (16, 4, 256), 64, 2, [3, 100, 257, 0, 60], [4, 0, 1, 3, 2], (2, 2), True),
    "verify_padded_apart": (5, 4, (16, 4, 128), 64, 0, [3, 100, 257, 0, 60], [4, 0, 1, 3, 2], (0, 1), True),
    "odd_group": (9, 3, (12, 4, 128), 64, 7, [30 * b for b in range(9)], None, None, False),
    "chunk": (2, 70, (16, 4, 256), 64, 2, [0, 77], [70, 33], None, True),
    "chunk_ranges": (2, 70, (16, 4, 256), 128, 2, [0, 77], [70, 33], (0, 3), True),
    "chunk_prefix": (3, 40, (8, 4, 128), 64, 3, [0, 77, 5], [40, 33, 0], (2, 2), True),
    "long_chunk": (2, 150, (16, 4, 256), 64, 1, [0, 33], [150, 101], None, True),
    "long_chunk_d128": (1, 300, (16, 4, 128), 128, 0, [20], None, None, False),
    "long_chunk_ranges": (2, 130, (16, 4, 256), 64, 2, [0, 700], [130, 77], (0, 5), True),
    "prefix_200_rows": (50, 1, (16, 4, 256), 64, 9, [b for b in range(50)], None, (4, 1), True),
    "prefix_600_rows_d128": (75, 2, (16, 4, 128), 64, 4, [b for b in range(75)], [b % 3 for b in range(75)], (3, 2), True),
    "prefix_in_16s": (12, 1, (16, 4, 256), 64, 5, [13 * b for b in range(12)], None, (3, 1, 16, 16), True),
    "prefix_in_16s_of_3_heads": (9, 3, (12, 4, 128), 64, 7, [30 * b for b in range(9)], [b % 4 for b in range(9)], (4, 2, 16, 16), True),
    "own_in_16s": (3, 13, (16, 4, 256), 64, 1, [0, 60, 300], None, (0, 1, 128, 16), True),
    "own_in_16s_ranges": (3, 9, (16, 2, 128), 128, 1, [0, 60, 700], [9, 0, 5], (0, 4, 128, 16), True),
    "own_in_16s_of_3_heads": (2, 23, (6, 2, 256), 64, 0, [0, 133], [23, 7], (0, 2, 128, 16), False),
    "both_in_16s": (5, 8, (16, 4, 256), 64, 4, [0, 64, 200, 3, 127], [8, 1, 0, 7, 3], (2, 2, 16, 16), True),
    "own_in_128s_of_few": (4, 1, (16, 4, 256), 64, 2, [0, 5, 64, 200], None, (2, 1, 128, 128), True),
    "prefix_ends_in_range": (33, 1, (16, 4, 256), 64, 5, [b for b in range(33)], None, (3, 1), True),
}


@pytest.mark.parametrize("name", list(CASES))
def test_attention_matches_oracle(name):
    B, T, heads, block, shared, tails, n_new, n_split, gated = CASES[name]
    Hq, Hkv, D = heads
    q, gate, keys, values, table, pos0 = _attn_case(torch.Generator().manual_seed(11), B, T, heads, block, shared, tails, n_new)
    L = max(p + (T if n_new is None else n) for p, n in zip(pos0, n_new or [T] * B))
    out = mx.paged_attn(q.to(DEV), keys.to(DEV), values.to(DEV), _i32(table), _i32(pos0), L,
                        n_new=None if n_new is None else _i32(n_new), shared=shared,
                        gate=gate.flatten(2).to(DEV) if gated else None, n_split=n_split)
    torch.cuda.synchronize()
    ref = op.attend(_np(q), _np(keys), _np(values), table, pos0, D ** -0.5, n_new, _np(gate)[..., D:] if gated else None)
    for b in range(B):
        n = T if n_new is None else n_new[b]
        assert _errs(_np(out[b, :n]), ref[b, :n]).max(initial=0) < ATT_TOL, b
        assert not out[b, n:].any()


@pytest.mark.parametrize("T,n_split", [(1, (0, 1)), (1, (0, 3)), (1, (2, 1)), (40, (0, 1)), (40, (1, 2))])
def test_positions_below_the_shared_keys(T, n_split):
    """A position below the shared keys' end is read as that end, whether or not
    the shared keys are read apart."""
    heads, block, shared, tails = (16, 4, 256), 64, 2, [0, 5]
    q, _, keys, values, table, pos0 = _attn_case(torch.Generator().manual_seed(17), 2, T, heads, block, shared, tails, None)
    given = [pos0[0] - 30, pos0[1]]
    out = mx.paged_attn(q.to(DEV), keys.to(DEV), values.to(DEV), _i32(table), _i32(given), max(pos0) + T, shared=shared,
                        n_split=n_split)
    ref = op.attend(_np(q), _np(keys), _np(values), table, pos0, 256 ** -0.5)
    assert _errs(_np(out), ref).max() < ATT_TOL


@pytest.mark.parametrize("heads", [(16, 4, 256), (12, 4, 128)])
@pytest.mark.parametrize("shared,tails,n_new", [(0, [0, 3, 0, 58], [10, 5, 0, 70]), (2, [0, 60, 0, 64], [64, 4, 0, 0])])
def test_padding_past_the_tables(heads, shared, tails, n_new):
    """300 tokens a row of which few are real, over tables that list just what those need."""
    B, T, block = 4, 300, 64
    q, gate, keys, values, table, pos0 = _attn_case(torch.Generator().manual_seed(31), B, T, heads, block, shared, tails,
                                                    n_new)
    L = max(p + n for p, n in zip(pos0, n_new))
    table = np.ascontiguousarray(table[:, :-(-L // block)])
    assert T > table.shape[1] * block
    ref = op.attend(_np(q), _np(keys), _np(values), table, pos0, heads[2] ** -0.5, n_new, _np(gate)[..., heads[2]:])
    for split in (None, (0, 1), (0, 2, 16, 16), (0, 3, 128, 128), *([(2, 1, 16, 128), (1, 2, 128, 16)] if shared else [])):
        out = mx.paged_attn(q.to(DEV), keys.to(DEV), values.to(DEV), _i32(table), _i32(pos0), L, shared=shared,
                            n_new=_i32(n_new), gate=gate.flatten(2).to(DEV), n_split=split)
        torch.cuda.synchronize()
        for b, n in enumerate(n_new):
            assert _errs(_np(out[b, :n]), ref[b, :n]).max(initial=0) < ATT_TOL, (b, split)
            assert not out[b, n:].any()


def test_attention_inf_scores():
    """A row whose every score is -inf is NaN, one with a +inf score too, as the
    softmax of such scores is; their neighbours are untouched."""
    gen = torch.Generator().manual_seed(5)
    B, heads = 3, (4, 1, 256)
    q, _, keys, values, table, pos0 = _attn_case(gen, B, 1, heads, 64, 1, [5, 6, 7], None)
    q[:], keys[:] = q.abs() + 0.1, keys.abs() + 0.1
    q[0, 0, 1, 3] = -float("inf")
    q[1, 0, 2, 3] = float("inf")
    for split in ((0, 1), (1, 1)):
        out = mx.paged_attn(q.to(DEV), keys.to(DEV), values.to(DEV), _i32(table), _i32(pos0), max(pos0) + 1, shared=1,
                            n_split=split)
        ref = op.attend(_np(q), _np(keys), _np(values), table, pos0, 256 ** -0.5)
        bad = np.isnan(ref).any(-1)
        assert bad[0, 0].tolist() == [False, True, False, False] and bad[1, 0].tolist() == [False, False, True, False]
        got = _np(out)
        assert (np.isnan(got).all(-1) == bad).all()
        assert _errs(got[~bad], ref[~bad]).max() < ATT_TOL


def test_offsets_beyond_32_bits():
    """A pool of 4.6e9 elements: the rows' blocks are its last and first ones, and
    the result is that of a small pool, bit for bit."""
    gen = torch.Generator().manual_seed(9)
    B, T, heads, n = 3, 2, (16, 4, 256), 70000
    q, gate, keys, values, table, pos0 = _attn_case(gen, B, T, heads, 64, 1, [70, 0, 200], None)
    where = torch.tensor([0 if i == 0 else n - i for i in range(keys.shape[0])])
    big = [torch.empty(n, heads[1], 64, heads[2], dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    for pool, small in zip(big, (keys, values)):
        pool[where.to(DEV)] = small.to(DEV)
    inside = (table >= 0) & (table < len(where))
    far = np.where(inside, where.numpy()[np.where(inside, table, 0)], table)
    args = dict(shared=1, gate=gate.flatten(2).to(DEV))
    for split in ((0, 1), (2, 2)):
        want = mx.paged_attn(q.to(DEV), keys.to(DEV), values.to(DEV), _i32(table), _i32(pos0), 300, n_split=split, **args)
        got = mx.paged_attn(q.to(DEV), *big, _i32(far), _i32(pos0), 300, n_split=split, **args)
        assert torch.equal(got, want)
    # the rotary prep's writes
    x = torch.randn(2, 1, (2 * 16 + 2 * 4) * 256, generator=gen).to(torch.bfloat16).to(DEV)
    parts = x.split((2 * 16 * 256, 4 * 256, 4 * 256), -1)
    slots = torch.tensor([[n * 64 - 1], [5]], dtype=torch.int32, device=DEV)
    mx.attn_rope(*parts, None, None, 1e-6, _i32([0, 0]), *big, mx.Rotary(64, 1e4, device=DEV), slots=slots)
    assert torch.equal(big[1][n - 1, :, 63], parts[2][0, 0].view(4, 256))
    assert torch.equal(big[1][0, :, 5], parts[2][1, 0].view(4, 256))
    assert torch.equal(big[0][n - 1, :, 63], parts[1][0, 0].view(4, 256))  # position 0, no norm: k as it is


@pytest.mark.parametrize("seed", range(12))
def test_attention_of_any_shape(seed):
    """Random batches, heads, blocks, prefixes and padding, with the rule's key ranges and with others."""
    rng = np.random.default_rng(100 + seed)
    gen = torch.Generator().manual_seed(200 + seed)
    Hkv = int(rng.integers(1, 5))
    heads = (Hkv * int(rng.integers(1, 9)), Hkv, int(rng.choice([128, 256])))
    B, T = int(rng.integers(1, 20)), int(rng.choice([1, 1, 2, 5, 17, 40]))
    block, shared = int(rng.choice([64, 128, 256])), int(rng.integers(0, 6))
    tails = rng.integers(0, 400, B).tolist()
    n_new = rng.integers(0, T + 1, B).tolist() if rng.integers(0, 2) else None
    q, gate, keys, values, table, pos0 = _attn_case(gen, B, T, heads, block, shared, tails, n_new)
    L = max(p + (T if n_new is None else n) for p, n in zip(pos0, n_new or [T] * B))
    ref = op.attend(_np(q), _np(keys), _np(values), table, pos0, heads[2] ** -0.5, n_new, _np(gate)[..., heads[2]:])
    ranges = (int(rng.integers(0, 4)) if shared else 0, int(rng.integers(1, 5)))
    for split in (None, ranges, (*ranges, 16, 16), (*ranges, 128, 128)):
        out = mx.paged_attn(q.to(DEV), keys.to(DEV), values.to(DEV), _i32(table), _i32(pos0), L, shared=shared,
                            n_new=None if n_new is None else _i32(n_new), gate=gate.flatten(2).to(DEV), n_split=split)
        torch.cuda.synchronize()
        for b in range(B):
            n = T if n_new is None else n_new[b]
            assert _errs(_np(out[b, :n]), ref[b, :n]).max(initial=0) < ATT_TOL, (b, split)
            assert not out[b, n:].any()


def test_strided_inputs_and_given_outputs():
    """q as a strided view, the gate as a column slice, out and workspace given (one too small)."""
    gen = torch.Generator().manual_seed(21)
    B, T, heads = 3, 2, (16, 4, 256)
    q, gate, keys, values, table, pos0 = _attn_case(gen, B, T, heads, 64, 1, [70, 0, 200], None)
    args = (keys.to(DEV), values.to(DEV), _i32(table), _i32(pos0), 300)
    want = mx.paged_attn(q.to(DEV), *args, shared=1, gate=gate.flatten(2).to(DEV), n_split=(1, 2))
    wide = torch.zeros(B, T, 16 * 512 + 64, dtype=torch.bfloat16, device=DEV)
    wide[..., :16 * 512] = gate.flatten(2).to(DEV)
    strided = torch.zeros(B, T, 16, 512, dtype=torch.bfloat16, device=DEV)
    strided[..., :256] = q.to(DEV)
    out = torch.empty(B, T, 16, 256, dtype=torch.bfloat16, device=DEV)
    for nbytes in (8, 1 << 24):
        ws = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
        got = mx.paged_attn(strided[..., :256], *args, shared=1, gate=wide[..., :16 * 512], n_split=(1, 2), out=out,
                            workspace=ws)
        assert got is out and torch.equal(out, want)
