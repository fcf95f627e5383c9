"""The paged key/value cache's operators, as measurable cases.

A serving batch keeps the keys and values of an attention layer in blocks of a
pool ``[blocks, Hkv, block, D]``; a row's table lists its blocks, and requests
that continue one long prompt list the prompt's blocks in common.  A step runs

  tables   the rows' lengths and their new tokens -> blocks taken from (or given
           back to) the free list, the tables, one slot per new token
  rope     q/k RMSNorm, rotary positions (half or interleaved pairs, a part of
           the head or all of it, frequencies scaled for long contexts), q out,
           k and v into their slots
  attend   attention over the tables: the shared prefix once for all rows, each
           row's own keys, causal among its new tokens, times the output gate

``run`` computes them in elementary torch operations, or, with ``own``, makes
the calls a user of ``multiplex_amd`` makes.

The head layouts are the attention layers' of this repository (16 query and 4
key/value heads of 256) and neighbours of them.  Activations and the pools are
bf16; lengths, tables, slots and free lists are int32.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
BASE = 1.0e7
HEADS = {"16x4x256": (16, 4, 256), "12x4x128": (12, 4, 128), "16x2x256": (16, 2, 256), "32x8x128": (32, 8, 128)}


def listed():
    return [
        # a decode step of a full batch: one row in 64 starts a block
        {"name": "tables_decode", "kind": "tables", "B": 256, "T": 1, "block": 64, "len": 8192, "shared": 0},
        # the scheduler's prefill chunk for some of the rows, the others one token
        {"name": "tables_chunk", "kind": "tables", "B": 48, "T": 512, "block": 64, "len": 6000, "shared": 32},
        # a large batch after a verify: rollbacks give blocks back, some rows left
        {"name": "tables_verify", "kind": "tables", "B": 1000, "T": 9, "block": 128, "len": 4096, "shared": 16},
        # a decode step far into a context that the scaled frequencies reach
        {"name": "rope_decode", "kind": "rope", "B": 64, "T": 1, "heads": "16x4x256", "rot": 64, "interleaved": False,
         "scaling": "yarn", "gated": True, "block": 64, "len": 1000000},
        # one long prompt
        {"name": "rope_prompt", "kind": "rope", "B": 1, "T": 4096, "heads": "16x4x256", "rot": 64,
         "interleaved": False, "scaling": "none", "gated": True, "block": 64, "len": 0},
        # prompts of different lengths: interleaved pairs over the whole head, no output gate
        {"name": "rope_ragged", "kind": "rope", "B": 5, "T": 333, "heads": "12x4x128", "rot": 128,
         "interleaved": True, "scaling": "linear", "gated": False, "block": 128, "len": 70000},
        # a few users on one system prompt: latency
        {"name": "attend_decode_b4", "kind": "attend", "B": 4, "T": 1, "heads": "16x4x256", "shared": 2048,
         "tail": 150, "gated": True, "block": 64},
        # a full batch on a long document
        {"name": "attend_decode_b64", "kind": "attend", "B": 64, "T": 1, "heads": "16x4x256", "shared": 8192,
         "tail": 512, "gated": True, "block": 64},
        # a speculative round of four drafts for half a batch
        {"name": "attend_verify_b32", "kind": "attend", "B": 32, "T": 4, "heads": "16x4x256", "shared": 16384,
         "tail": 700, "gated": True, "block": 64},
        # prefill chunks of four rows behind the prefix
        {"name": "attend_chunk_b4", "kind": "attend", "B": 4, "T": 512, "heads": "16x4x256", "shared": 4096,
         "tail": 300, "gated": True, "block": 128},
        # an odd batch: three heads a group, prefix that ends inside two 64-key steps, no gate
        {"name": "attend_odd", "kind": "attend", "B": 17, "T": 3, "heads": "12x4x128", "shared": 1984,
         "tail": 333, "gated": False, "block": 64},
        # rows that share nothing
        {"name": "attend_apart", "kind": "attend", "B": 24, "T": 1, "heads": "32x8x128", "shared": 0, "tail": 4000,
         "gated": True, "block": 256},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tables", "rope", "attend", "attend"])
    block = rng.choice([64, 64, 128, 256])
    if kind == "tables":
        B = _log(rng, 1, 1000)
        return {"kind": kind, "B": B, "T": _log(rng, 1, min(4096, max(1, 24576 // B))), "block": block,
                "len": _log(rng, 64, 8192), "shared": rng.choice([0, _log(rng, 1, 40)])}
    heads = rng.choice(list(HEADS))
    D = HEADS[heads][2]
    if kind == "rope":
        B = _log(rng, 1, 128)
        return {"kind": kind, "B": B, "T": _log(rng, 1, max(1, 3500 // B)), "heads": heads,
                "rot": rng.choice([D // 4, D // 2, D]), "interleaved": rng.choice([False, True]),
                "scaling": rng.choice(["none", "linear", "yarn"]), "gated": rng.choice([False, True]), "block": block,
                "len": rng.choice([0, _log(rng, 100, 1000000)])}
    B = _log(rng, 1, 64)
    T = rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, 512)])
    T = max(1, min(T, 2048 // B))
    shared = rng.choice([0, 1, 1, 1]) * block * _log(rng, 1, max(1, min(16384, 2500000 // (B * T)) // block))
    return {"kind": kind, "B": B, "T": T, "heads": heads, "shared": shared, "tail": _log(rng, 1, max(64, 16384 // B)),
            "gated": rng.choice([False, True]), "block": block}


# ------------------------------------------------------------------ inputs

class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 29)

    def n(self, *shape, dtype=torch.bfloat16, scale=1.0, mean=0.0):
        x = torch.randn(*shape, generator=self.g, device="cuda", dtype=torch.float32)
        return (x * scale + mean).to(dtype)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device="cuda").to(torch.int32)

    def spread(self, B, hi):
        """B whole numbers of [1, hi] in random order, spread evenly: any seed's sum is about B (hi + 1) / 2."""
        u = torch.rand(B, generator=self.g, device="cuda", dtype=torch.float64)
        x = (self.perm(B).double() + u) / B * hi
        return (x.floor() + 1).clamp(1, hi).to(torch.int32)


def _blocks(n, block):
    return (n + block - 1) // block


def _tables_state(case, r):
    B, T, bs, shared = case["B"], case["T"], case["block"], case["shared"]
    lengths = shared * bs + r.spread(B, case["len"])
    if T == 1:
        n_new = None
    else:
        # a third of the rows run the whole step, the others less, down to none
        n_new = (r.spread(B, 3 * T) - 1).clamp(0, T)
    held = _blocks(lengths, bs)
    gone = r.spread(B, 16) == 1  # rows that left: they give their blocks back
    lengths = torch.where(gone, 0, lengths)
    if n_new is not None:
        n_new = torch.where(gone, 0, n_new)
        # a rollback of some drafts, which may leave the row with a block too many
        lengths = (lengths - r.spread(B, T)).clamp(min=0)
        lengths = torch.where(gone, lengths, lengths.clamp(min=shared * bs))
    most = shared + _blocks(case["len"] + T, bs)
    spare = B * _blocks(T, bs) + B
    n_blocks = shared + B * _blocks(case["len"], bs) + spare
    order = r.perm(n_blocks)
    cols = torch.arange(most, device="cuda")
    mine = (cols[None, :] >= shared) & (cols[None, :] < held[:, None])
    at = shared + (mine.flatten().cumsum(0).view(B, most) - 1)
    table = torch.where(mine, order[at.clamp(0, n_blocks - 1)], -1)
    table[:, :shared] = order[:shared]
    used = shared + int(mine.sum())
    free = torch.full((n_blocks,), -1, dtype=torch.int32, device="cuda")
    free[: n_blocks - used] = order[used:]
    n_free = torch.tensor([n_blocks - used], dtype=torch.int32, device="cuda")
    return {"lengths": lengths, "n_new": n_new, "T": T, "table": table.to(torch.int32), "held": held, "free": free,
            "n_free": n_free, "block": bs, "shared": shared}


SCALING = {"none": None, "linear": {"type": "linear", "factor": 4.0},
           "yarn": {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 262144}}


def _rope_state(case, r):
    Hq, Hkv, D = HEADS[case["heads"]]
    B, T, bs = case["B"], case["T"], case["block"]
    per_q = 2 * D if case["gated"] else D
    wide = r.n(B, T, Hq * per_q + 2 * Hkv * D)  # one projection's output: q (and its gate) | k | v
    qg, k, v = wide.split((Hq * per_q, Hkv * D, Hkv * D), -1)
    pos0 = r.spread(B, case["len"]) if case["len"] else torch.zeros(B, dtype=torch.int32, device="cuda")
    n_new = torch.full_like(pos0, T) if B == 1 or T == 1 else r.spread(B, T)
    # the new tokens' blocks lie anywhere in the pool
    per = _blocks(T, bs) + 1
    n_blocks = B * per + 3
    order = r.perm(n_blocks)[: B * per].view(B, per)
    t = torch.arange(T, device="cuda", dtype=torch.int32)
    at = pos0[:, None] % bs + t
    slots = order.gather(1, (at // bs).long()) * bs + at % bs
    slots = torch.where(t < n_new[:, None], slots, -1).to(torch.int32)
    s = {"qg": qg, "k": k, "v": v, "qw": r.n(D, dtype=torch.float32, scale=0.1, mean=1.0),
         "kw": r.n(D, dtype=torch.float32, scale=0.1, mean=1.0), "pos0": pos0, "slots": slots,
         "keys": r.n(n_blocks, Hkv, bs, D), "values": r.n(n_blocks, Hkv, bs, D), "gated": case["gated"],
         "rot": case["rot"], "interleaved": case["interleaved"], "scaling": case["scaling"], "heads": (Hq, Hkv, D)}
    if own:
        import multiplex_amd as mx

        s["rotary"] = mx.Rotary(case["rot"], BASE, interleaved=case["interleaved"], scaling=SCALING[case["scaling"]],
                                device="cuda")
    return s


def _attend_state(case, r):
    Hq, Hkv, D = HEADS[case["heads"]]
    B, T, bs = case["B"], case["T"], case["block"]
    prefix = case["shared"] // bs
    pos0 = case["shared"] + r.spread(B, case["tail"]) - 1
    n_new = None if B == 1 or T == 1 else r.spread(B, T)
    most = prefix + _blocks(case["tail"] + T, bs)
    per = most - prefix
    n_blocks = prefix + B * per + 5
    order = r.perm(n_blocks)
    table = torch.empty(B, most, dtype=torch.int32, device="cuda")
    table[:, :prefix] = order[:prefix]
    table[:, prefix:] = order[prefix:prefix + B * per].view(B, per)
    q = r.n(B, T, Hq, D)
    gate = r.n(B, T, 2 * Hq * D) if case["gated"] else None
    return {"q": q, "gate": gate, "keys": r.n(n_blocks, Hkv, bs, D), "values": r.n(n_blocks, Hkv, bs, D),
            "table": table, "pos0": pos0.to(torch.int32), "n_new": n_new, "shared": prefix,
            "kv_len_max": case["shared"] + case["tail"] - 1 + T, "heads": (Hq, Hkv, D), "T": T}


def prepare(case, seed):
    r = _Rand(seed)
    make = {"tables": _tables_state, "rope": _rope_state, "attend": _attend_state}[case["kind"]]
    return {"kind": case["kind"], **make(case, r)}


# ---------------------------------------------------------- the plain forms

def _plain_tables(s):
    """Every row's blocks for ``lengths + n_new`` positions (and the shared
    ones): rows with too many give the last back, in row order, onto the free
    list's end; rows with too few take from its end, in row order."""
    T, bs, table, held, free = s["T"], s["block"], s["table"], s["held"], s["free"]
    B, most = table.shape
    n_new = torch.full_like(held, T) if s["n_new"] is None else s["n_new"]
    need = torch.maximum(_blocks(s["lengths"] + n_new, bs), torch.full_like(held, s["shared"]))
    fits = need <= most
    need = torch.where(fits, need, held)
    cols = torch.arange(most, device=table.device, dtype=torch.int32)[None, :]
    back = (cols >= need[:, None]) & (cols < held[:, None])
    spill = torch.cat([free, free.new_zeros(1)])  # cells that nothing goes to write to the last entry
    at = torch.where(back, s["n_free"] + back.flatten().cumsum(0).view(B, most) - 1, free.numel())
    spill.scatter_(0, at.flatten(), table.flatten())
    top = s["n_free"] + back.sum()
    demand = (need - held).clamp(min=0)
    taken = demand.cumsum(0)
    ok = fits & ((taken <= top) | (demand == 0))
    demand = torch.where(ok, demand, 0)
    first = top - 1 - (demand.cumsum(0) - demand)
    new = (cols >= held[:, None]) & (cols < (held + demand)[:, None])
    at = (first[:, None] - (cols - held[:, None])).clamp(0, free.numel() - 1)
    table.copy_(torch.where(new, spill[at], table))
    free.copy_(spill[:-1])
    t = torch.arange(T, device=table.device, dtype=torch.int32)[None, :]
    pos = s["lengths"][:, None] + t
    page = table.gather(1, (pos // bs).clamp(max=most - 1).long())
    slots = torch.where(ok[:, None] & (t < n_new[:, None]), page * bs + pos % bs, -1)
    held_out = torch.where(ok, need, held)
    return slots.to(torch.int32), held_out.to(torch.int32), (top - demand.sum()).to(torch.int32), table, free


def _frequencies(rot, scaling):
    """Angle per position of each pair, in float64, and the factor of the rotated values."""
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    inv = BASE ** (-2.0 * i / rot)
    if scaling == "none":
        return inv, 1.0
    s = SCALING[scaling]["factor"]
    if scaling == "linear":
        return inv / s, 1.0
    # pairs that turn more than 32 times over the original context keep their frequency, those that turn less
    # than once are stretched by the factor, in between a ramp
    context = SCALING[scaling]["original_max_position_embeddings"]

    def pair(turns):
        return rot * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(BASE))

    lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot - 1)
    ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return inv / s * ramp + inv * (1 - ramp), 0.1 * math.log(s) + 1


def _plain_rope(s):
    Hq, Hkv, D = s["heads"]
    B, T = s["slots"].shape
    rot, half = s["rot"], s["rot"] // 2
    bs = s["keys"].shape[2]
    inv, factor = _frequencies(rot, s["scaling"])
    pos = s["pos0"][:, None] + torch.arange(T, device="cuda")
    ang = pos.double()[..., None] * inv
    cos, sin = (ang.cos() * factor).float()[:, :, None], (ang.sin() * factor).float()[:, :, None]

    def norm_rotate(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        if s["interleaved"]:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = x[..., :half], x[..., half:rot]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([y, x[..., rot:]], -1)

    valid = s["slots"] >= 0
    q = norm_rotate(s["qg"].reshape(B, T, Hq, -1)[..., :D], s["qw"]).to(torch.bfloat16)
    q = torch.where(valid[:, :, None, None], q, torch.zeros_like(q))
    k = norm_rotate(s["k"].reshape(B, T, Hkv, D), s["kw"]).to(torch.bfloat16)
    slot = s["slots"][valid].long()
    s["keys"][slot // bs, :, slot % bs] = k[valid]
    s["values"][slot // bs, :, slot % bs] = s["v"].reshape(B, T, Hkv, D)[valid]
    return q, s["keys"], s["values"]


def _plain_attend(s):
    Hq, Hkv, D = s["heads"]
    T, L = s["T"], s["kv_len_max"]
    B, bs, g = s["q"].shape[0], s["keys"].shape[2], Hq // Hkv
    n = _blocks(L, bs)

    def rows(pool):  # [B, Hkv, L, D] in 32 bits
        x = pool[s["table"][:, :n].long()]
        return x.transpose(1, 2).reshape(B, Hkv, n * bs, D)[:, :, :L].float()

    t = torch.arange(T, device="cuda")
    key = torch.arange(L, device="cuda")
    ends = s["pos0"].long() + (T if s["n_new"] is None else s["n_new"].long())
    k, v = rows(s["keys"]), rows(s["values"])
    v = torch.where((key < ends[:, None])[:, None, :, None], v, 0.0)
    q = s["q"].float().view(B, T, Hkv, g, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, g * T, D)
    sc = torch.matmul(q, k.transpose(2, 3)) * D ** -0.5
    sees = key <= (s["pos0"].long()[:, None] + t)[..., None]  # [B, T, L]
    sc = sc.view(B, Hkv, g, T, L).masked_fill(~sees[:, None, None], -math.inf)
    p = (sc - sc.amax(-1, keepdim=True)).exp()
    p = (p / p.sum(-1, keepdim=True)).view(B, Hkv, g * T, L)
    o = torch.matmul(p, v).view(B, Hkv, g, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D)
    if s["gate"] is not None:
        gate = s["gate"].view(B, T, Hq, 2 * D)[..., D:].float()
        o = o / (1 + (-gate).exp())
    if s["n_new"] is not None:
        o = torch.where((t < s["n_new"][:, None])[:, :, None, None], o, 0.0)
    return o.to(torch.bfloat16)


def _own(s):
    import multiplex_amd as mx

    if s["kind"] == "tables":
        slots, held, n_free = mx.paged_tables(s["lengths"], s["T"], s["table"], s["held"], s["free"], s["n_free"],
                                              s["block"], n_new=s["n_new"], shared=s["shared"])
        return slots, held, n_free, s["table"], s["free"]
    if s["kind"] == "rope":
        q = mx.attn_rope(s["qg"], s["k"], s["v"], s["qw"], s["kw"], EPS, s["pos0"], s["keys"], s["values"],
                         s["rotary"], slots=s["slots"], gated=s["gated"])
        return q, s["keys"], s["values"]
    return mx.paged_attn(s["q"], s["keys"], s["values"], s["table"], s["pos0"], s["kv_len_max"], n_new=s["n_new"],
                         shared=s["shared"], gate=s["gate"])


def run(s):
    if own:
        return _own(s)
    return {"tables": _plain_tables, "rope": _plain_rope, "attend": _plain_attend}[s["kind"]](s)


# -------------------------------------------------------------------- work

def work(case):
    B, T = case["B"], case["T"]
    if case["kind"] == "tables":
        # lengths, new tokens, held counts (in and out) and the free count; a slot per token and the table
        # entries that the step adds and its tokens read
        grown = B * _blocks((T + 1) // 2, case["block"])
        return {"bytes": 4 * (4 * B + 2 + B * T + 2 * grown), "flops": 0}
    Hq, Hkv, D = HEADS[case["heads"]]
    if case["kind"] == "rope":
        tokens = B * T if B == 1 or T == 1 else B * (T + 1) // 2
        vectors = tokens * (Hq + 2 * Hkv)
        return {"bytes": 2 * 2 * D * vectors + 4 * (B + B * T) + 8 * D,
                "flops": tokens * (Hq + Hkv) * (4 * D + 3 * case["rot"])}
    new = T if B == 1 or T == 1 else (T + 1) / 2
    tail = (case["tail"] - 1) / 2
    keys = case["shared"] + B * (tail + new)
    pairs = B * (new * (case["shared"] + tail) + new * (new + 1) / 2)
    io = B * new * Hq * D * (3 if case["gated"] else 2)
    return {"bytes": int(2 * (2 * keys * Hkv * D + io) + 4 * keys / case["block"]), "flops": int(4 * Hq * D * pairs)}


# ------------------------------------------------------------------- exact

def _exact_tables(s):
    """The same, one row after the other on the host."""
    bs, T, shared = s["block"], s["T"], s["shared"]
    lengths, held = s["lengths"].tolist(), s["held"].tolist()
    n_new = [T] * len(held) if s["n_new"] is None else s["n_new"].tolist()
    table, free, top = s["table"].tolist(), s["free"].tolist(), int(s["n_free"])
    need = [max(-(-(n + m) // bs), shared) for n, m in zip(lengths, n_new)]
    for row, have, want in zip(table, held, need):
        for c in range(want, have):
            free[top] = row[c]
            top += 1
    left, asked, slots, out = top, 0, [], []
    for b, row in enumerate(table):
        grow = need[b] - held[b]
        ok = need[b] <= len(row)
        if ok and grow > 0:
            asked += grow
            ok = asked <= top
            if ok:
                for c in range(held[b], need[b]):
                    left -= 1
                    row[c] = free[left]
        out.append(need[b] if ok else held[b])
        place = [lengths[b] + t for t in range(n_new[b])] if ok else []
        slots.append([row[p // bs] * bs + p % bs for p in place] + [-1] * (T - len(place)))

    def i32(x):
        return torch.tensor(x, dtype=torch.int32)

    return i32(slots), i32(out), i32([left]), i32(table), i32(free)


def _exact_rope(case, s):
    Hq, Hkv, D = s["heads"]
    rot, bs = s["rot"], s["keys"].shape[2]
    pairs = rot // 2
    freq = []
    for i in range(pairs):
        f = math.pow(BASE, -2.0 * i / rot)
        if case["scaling"] == "linear":
            f /= 4.0
        elif case["scaling"] == "yarn":
            def place(turns):
                return rot * math.log(262144 / (2 * math.pi * turns)) / (2 * math.log(BASE))

            lo, hi = max(int(math.floor(place(32))), 0), min(int(math.ceil(place(1))), rot - 1)
            keep = 1.0 - min(1.0, max(0.0, (i - lo) / (hi - lo if hi > lo else 0.001)))
            f = f * keep + f / 4.0 * (1.0 - keep)
        freq.append(f)
    mag = 0.1 * math.log(4.0) + 1.0 if case["scaling"] == "yarn" else 1.0
    freq = torch.tensor(freq, dtype=torch.float64, device="cuda")
    if s["interleaved"]:
        one = torch.arange(0, rot, 2, device="cuda")
        two = one + 1
    else:
        one = torch.arange(pairs, device="cuda")
        two = one + pairs
    q_out = torch.zeros(*s["slots"].shape, Hq, D, dtype=torch.float64, device="cuda")
    keys, values = s["keys"].double(), s["values"].double()
    step = s["qg"].shape[2] // Hq
    for b in range(q_out.shape[0]):
        n = int((s["slots"][b] >= 0).sum())
        angle = torch.outer(torch.arange(n, device="cuda", dtype=torch.float64) + float(s["pos0"][b]), freq)
        turn = torch.polar(torch.full_like(angle, mag), angle)[:, None]

        def through(x, w):
            x = x.double()
            x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / D + EPS) * w.double()
            z = torch.complex(x[..., one], x[..., two]) * turn
            y = x.clone()
            y[..., one], y[..., two] = z.real, z.imag
            return y

        q_out[b, :n] = through(s["qg"][b, :n].unflatten(-1, (Hq, step))[..., :D], s["qw"])
        slot = s["slots"][b, :n].long()
        page, off = slot.div(bs, rounding_mode="floor"), slot.remainder(bs)
        keys[page, :, off] = through(s["k"][b, :n].unflatten(-1, (Hkv, D)), s["kw"])
        values[page, :, off] = s["v"][b, :n].unflatten(-1, (Hkv, D)).double()
    return q_out, keys, values


def _exact_attend(s):
    Hq, Hkv, D = s["heads"]
    B, T, g, bs = s["q"].shape[0], s["T"], Hq // Hkv, s["keys"].shape[2]
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device="cuda")
    for b in range(B):
        start = int(s["pos0"][b])
        n = T if s["n_new"] is None else int(s["n_new"][b])
        L = start + n
        pages = s["table"][b, : -(-L // bs)].long()
        future = torch.ones(n, L, dtype=torch.bool, device="cuda").triu(start + 1)
        for h in range(Hkv):
            k = s["keys"][pages, h].reshape(-1, D)[:L].double()
            v = s["values"][pages, h].reshape(-1, D)[:L].double()
            for j in range(h * g, h * g + g):
                sc = (s["q"][b, :n, j].double() @ k.T.contiguous()) / math.sqrt(D)
                w = torch.softmax(sc.masked_fill(future, -math.inf), -1)
                out[b, :n, j] = w @ v
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].double().unflatten(-1, (Hq, 2 * D))[..., D:])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "tables":
        return _exact_tables(s)
    if case["kind"] == "rope":
        return _exact_rope(case, s)
    return _exact_attend(s)
