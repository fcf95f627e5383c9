"""The attention layers' KV cache in blocks, for batches that share a prefix.

multiplex serves many requests over one system prompt or document and keeps
their common prefix in its cache as blocks (``multiplex/kernel/prefixcache/``:
attention-KV block deltas, longest-prefix reuse).  With a dense cache per row,
every row holds and every decode step reads a copy of that prefix.  Here keys
and values live in one pool of blocks per layer, a row's table lists its
blocks, and rows that continue one prompt list the prompt's blocks in common:

  paged_tables   the rows' lengths and new tokens -> tables, slots, free list
                 (``gdn_paged_tables``; nothing is read back to the host)
  attn_rope      :mod:`multiplex_amd.rotary`: q/k norm, rotary positions, k and
                 v into their slots
  paged_attn     attention over the tables (``gdn_paged_attn``): the shared
                 blocks are read once for the whole batch
  BlockPool      one layer's blocks and their free list
  PagedKVCache   the rows of a batch over a pool; :class:`Attention`,
                 :class:`DecoderLayer` and :class:`MTPHead` take it wherever they
                 take a :class:`KVCache`
"""

from __future__ import annotations

import functools
import weakref
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib
from .attention import KVCache, _pos_add, _token_stride
from .gated_delta import _require_device, _stream

__all__ = ["paged_tables", "paged_attn", "BlockPool", "PagedKVCache"]


def _is_i32(t: torch.Tensor, shape: Tuple[int, ...], index: int) -> bool:
    return t.dtype is torch.int32 and t.shape == shape and t.get_device() == index and t.is_contiguous()


def _i32(t: torch.Tensor, shape: Tuple[int, ...], what: str) -> None:
    if t.dtype is not torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 {list(shape)} tensor (got {t.dtype} {list(t.shape)})")


def paged_tables(lengths: torch.Tensor, T: int, table: torch.Tensor, held: torch.Tensor, free: torch.Tensor,
                 n_free: torch.Tensor, block: int, *, n_new: Optional[torch.Tensor] = None, shared: int = 0,
                 held_out: Optional[torch.Tensor] = None, n_free_out: Optional[torch.Tensor] = None,
                 slots: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Blocks for the next T tokens of every row (``n_new[b]`` of them, padded
    to T, when given): returns ``(slots [B, T], held, n_free)``.

    lengths ``[B]`` (tokens a row holds), table ``[B, width]``, held ``[B]``
    (blocks its table lists), free ``[n_blocks]`` with the ``n_free`` ``[1]`` free
    blocks first, all int32.  A row needs ``ceil((lengths + new) / block)``
    blocks, its first ``shared`` ones always: what it holds beyond goes back onto
    the free list (so a rolled-back row, or one whose length is set to 0, gives
    its blocks back in the next call), what it lacks is taken from the list's
    end, rows in order.  From the first row that the list cannot serve whole on,
    rows that ask get nothing and their slots are -1, as are the slots of padding.

    ``table`` and ``free`` are written in place; the counts are returned in new
    tensors unless ``held_out=held``, ``n_free_out=n_free`` ask for them in place
    (without, the same call can be repeated).
    """
    dev = lengths.device
    index = lengths.get_device()
    T = int(T)
    # the whole check in a few operations; what is wrong is looked for only where something is
    if index < 0 or lengths.dim() != 1 or table.dim() != 2 or free.dim() != 1 or T < 0:
        _refuse_tables(lengths, T, table, held, free, n_free, n_new, held_out, n_free_out, slots)
    B, width, n_blocks = lengths.shape[0], table.shape[1], free.shape[0]
    row, one = (B,), (1,)
    if not (_is_i32(lengths, row, index) and _is_i32(table, (B, width), index) and _is_i32(held, row, index)
            and _is_i32(free, (n_blocks,), index) and _is_i32(n_free, one, index)
            and (n_new is None or _is_i32(n_new, row, index))
            and (held_out is None or held_out is held or _is_i32(held_out, row, index))
            and (n_free_out is None or n_free_out is n_free or _is_i32(n_free_out, one, index))
            and (slots is None or _is_i32(slots, (B, T), index))):
        _refuse_tables(lengths, T, table, held, free, n_free, n_new, held_out, n_free_out, slots)
    if held_out is None:
        held_out = torch.empty_like(held)
    if n_free_out is None:
        n_free_out = torch.empty_like(n_free) if B else n_free
    if slots is None:
        slots = lengths.new_empty((B, T))
    _lib.call(dev, "gdn_paged_tables", lengths.data_ptr(), None if n_new is None else n_new.data_ptr(),
              table.data_ptr(), width, held.data_ptr(), free.data_ptr(), n_free.data_ptr(), held_out.data_ptr(),
              n_free_out.data_ptr(), slots.data_ptr(), B, T, int(block), int(shared), n_blocks, _stream(dev))
    return slots, held_out, n_free_out


def _refuse_tables(lengths, T, table, held, free, n_free, n_new, held_out, n_free_out, slots) -> None:
    """Raises what is wrong with :func:`paged_tables`' arguments."""
    _require_device((lengths, table, held, free, n_free, n_new, held_out, n_free_out, slots),
                    ("lengths", "table", "held", "free", "n_free", "n_new", "held_out", "n_free_out", "slots"))
    if lengths.dim() != 1 or T < 0:
        raise ValueError("lengths must be a [B] tensor and T >= 0")
    if table.dim() != 2 or free.dim() != 1:
        raise ValueError("table must be [B, width] and free [n_blocks]")
    B = lengths.shape[0]
    for t, shape, what in ((lengths, (B,), "lengths"), (table, (B, table.shape[1]), "table"), (held, (B,), "held"),
                           (free, (free.shape[0],), "free"), (n_free, (1,), "n_free"), (n_new, (B,), "n_new"),
                           (held_out, (B,), "held_out"), (n_free_out, (1,), "n_free_out"), (slots, (B, T), "slots")):
        if t is not None:
            _i32(t, shape, what)


_cus = {}


def _cu_count(dev: torch.device) -> int:
    n = _cus.get(dev.index)
    if n is None:
        n = _cus[dev.index] = torch.cuda.get_device_properties(dev).multi_processor_count
    return n


# us that a workgroup takes, before its first and after its last keys and per step
# of them: 16 rows (128 keys a step), 128 rows (64 keys); us that the merge of the
# partial results takes, and per MB of them; how much of the time between a full
# row's and the average row's the workgroups take on average.  At head dims up to
# 128 and 256 (two workgroups a CU, and one).  Fitted to graph-replayed times of
# 7000 sizes (four head layouts of 3 to 8 query heads a group, 1 to 128 rows, 1 to
# 512 tokens, prefixes to 16384 and rows' own keys to 32768), 16 choices each; at
# 11500, with up to 40 choices measured, the rule's is 2.5 to 3.9% slower than the
# best of them on average, 8 to 11% at one in ten.
_US = ((5.2, 1.01, 7.2, 1.24, 4.1, 0.37, 0.25), (6.5, 1.23, 10.5, 1.52, 4.7, 0.28, 0.17))
_MB_US, _L2_MB_US = 5.5, 25.0  # MB a us from memory, and from the L2s
_PREFIX_RANGES = (0, 1, 2, 3, 4, 6, 8, 12, 16, 20, 24, 32, 48, 64)
_OWN_RANGES = (1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128, 256)


@functools.lru_cache(maxsize=4096)
def _ranges(cus: int, B: int, T: int, Hq: int, Hkv: int, D: int, prefix: int, own: int) -> Tuple[int, int, int, int]:
    """``(n_prefix, n_own, prefix_rows, own_rows)``: key ranges of the shared prefix
    (0: read with each row's own keys) and of a row's own keys, and the query rows
    of a workgroup over each; both lengths in steps of 64 keys.

    The prefix read once takes work from every row, but leaves partial results
    to merge; ranges make workgroups enough, each at a price.  So the choice is
    the least of the times that :data:`_US` gives, searched for once for a step's
    sizes: 15 to 550 us of the host's time, then 0.1.  (Decode of 64 rows of 16
    heads of 256 behind 8192 keys and up to 512 of their own, us: without a pass
    of the prefix 113, with it in 4 / 8 / 12 / 16 / 32 ranges 64 / 42 / 35.5 / 37 /
    47.5; 4 rows behind 2048: in 1 / 4 / 8 ranges of all keys 27 / 15 / 13.2, the
    prefix apart in 8 / 12 14.2 / 13.6.)

    Workgroups of 16 rows start and end sooner, but the keys are read once for
    every 16.  Where there are 17 to 512 rows, the better kind takes on average 0.89
    of the time of 128-row workgroups alone (6 x 4 drafts of 8 heads a group behind
    5952 keys 26.7 and, in 16s, 21.5 us; a row of 16 tokens over 2000 keys 17.3 and
    13.9; 32 rows of one token behind 8192 keys 28 and 32).
    """
    rows = T * (Hq // Hkv)
    few, few_step, many, many_step, merge, merge_mb, full = _US[D > 128]
    slots = cus * (1 if D > 128 else 2)
    read = 256e-6 * Hkv * D * (prefix + B * own / 2) / _MB_US  # the keys and values, rows half full

    def groups(n_rows, blocks, n, tile):
        """Workgroups of a kv-head, us that one takes, and MB that they read."""
        of = -(-blocks // n)
        n = -(-blocks // of) * -(-n_rows // tile)
        return n, few + few_step * -(-of // 2) if tile == 16 else many + many_step * of, 256e-6 * D * n * of

    def tiles(n_rows):
        return (16,) if n_rows <= 16 else (16, 128) if n_rows <= 512 else (128,)

    best, choice = None, (0, 1, 128, 128)
    for p, tp in [(0, 128)] + [(p, tp) for p in _PREFIX_RANGES[1:] for tp in tiles(B * rows)]:
        if p and (B == 1 or rows >= 256 or p > prefix):
            break
        own_p = max(own if p else own + prefix, 1)
        n_p, us_p, mb_p = groups(B * rows, prefix, p, tp) if p else (0, 0.0, 0.0)
        whole, rest = divmod(n_p * Hkv, slots)  # the prefix's workgroups go first, in rounds of all slots
        fill = 1.0 - own / (2 * own_p)
        for o, to in [(o, to) for o in _OWN_RANGES for to in tiles(rows)]:
            if o > 1 and 2 * o > own_p or p and o > 8:
                break
            n_o, us, mb = groups(rows, own_p, o, to)
            n_o *= max(B, 1) * Hkv
            mean = us * (full + (1.0 - full) * fill)
            free = slots - rest  # beside the prefix's last round
            rounds = us_p // mean if rest else 0.0
            if rest and n_o <= free * rounds:
                t = max(us_p, (-(-n_o // free) - 1) * mean + us)
            elif rest:
                left = -(-max(n_o - free * (rounds + 1), 0) // slots)
                t = max(us_p + (left * mean + us - mean if left else 0.0), rounds * mean + us)
            else:
                t = (-(-n_o // slots) - 1) * mean + us
            ends = many if 128 in (to, tp if p else 16) else few  # before the first and after the last keys
            t = max(whole * us_p + t, ends + read, ends + Hkv * (mb_p + B * mb * fill) / _L2_MB_US)
            if p + o > 1:
                t += merge + merge_mb * 4e-6 * B * T * Hq * D * (p + o)
            if best is None or t < best:
                best, choice = t, (p, o, tp, to)
    return choice


def paged_attn(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor, pos0: torch.Tensor,
               kv_len_max: int, *, n_new: Optional[torch.Tensor] = None, shared: int = 0,
               gate: Optional[torch.Tensor] = None, scale: Optional[float] = None,
               n_split: Optional[Tuple[int, ...]] = None, workspace: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal GQA attention of q ``[B, T, Hq, D]`` over the blocks that ``table``
    ``[B, width]`` lists (``gdn_paged_attn``), times sigmoid of the gate half of
    ``gate`` (``[B, T, Hq*2D]``, the q_proj output) when given.

    keys, values ``[n_blocks, Hkv, block, D]`` bf16 pools, block a power of two
    from 64 on; pos0 ``[B]`` int32: token t of row b sees keys 0 .. pos0[b] + t.
    ``n_new`` ``[B]`` int32: a row's tokens past it are padding, whose outputs are
    zeros; T may then exceed what the tables list.  ``kv_len_max`` bounds ``pos0[b] + n_new[b]`` (host value; keys beyond
    it are not read).  The first ``shared`` entries of every row's table have to
    be the same and full (``pos0[b] >= shared * block``): their keys are read
    once for the batch.  ``n_split`` sets the key ranges of the prefix (0: with
    each row's own keys) and of a row's own keys, and, where it has four entries,
    the query rows of a workgroup over each (16 or 128; otherwise 16 where no more
    are there); by default a rule does.
    ``workspace``: bytes for the partial results of several ranges (allocated
    when absent or too small); calls that overlap need one each.

    v of a call's own tokens is taken to be finite: a token's inf or NaN there
    reaches the earlier tokens of its row in the same call, as a weight of 0 times
    it does in any product.  What the pools hold past a row's tokens, in padding
    and in blocks of no row is never used.
    """
    dev = q.device
    index = q.get_device()
    kv_len_max, shared = int(kv_len_max), int(shared)
    if index < 0 or q.dim() != 4 or keys.dim() != 4 or table.dim() != 2:
        _refuse_attn(q, keys, values, table, pos0, kv_len_max, n_new, shared, gate, workspace, out)
    B, T, Hq, D = q.shape
    n_blocks, Hkv, block, Dk = keys.shape
    width = table.shape[1]
    bf16, row = torch.bfloat16, (B,)
    if not (q.dtype is bf16 and keys.dtype is bf16 and values.dtype is bf16 and keys.get_device() == index
            and values.get_device() == index and values.shape == keys.shape and keys.is_contiguous()
            and values.is_contiguous() and Dk == D and Hkv > 0 and Hq % Hkv == 0
            and _is_i32(table, (B, width), index) and _is_i32(pos0, row, index)
            and (n_new is None or _is_i32(n_new, row, index))
            and 0 <= shared * block <= kv_len_max - (T if n_new is None else 0) and kv_len_max <= width * block
            and (gate is None or (gate.dtype is bf16 and gate.shape == (B, T, Hq * 2 * D) and gate.get_device() == index))
            and (workspace is None or workspace.get_device() == index and workspace.is_contiguous())
            and (out is None or (out.dtype is bf16 and out.shape == q.shape and out.get_device() == index
                                 and out.is_contiguous()))):
        _refuse_attn(q, keys, values, table, pos0, kv_len_max, n_new, shared, gate, workspace, out)
    qg_ld = 0 if gate is None else _token_stride(gate, Hq * 2 * D, "gate")
    if not q.is_contiguous():
        q = q.contiguous()
    if out is None:
        out = torch.empty_like(q)
    prefix = shared * block
    if n_split is None:
        n_split = _ranges(_cu_count(dev), B, T, Hq, Hkv, D, prefix >> 6, (kv_len_max - prefix + 63) >> 6)
    if len(n_split) == 2:
        rows = T * (Hq // Hkv)
        n_split = (*n_split, 16 if B * rows <= 16 else 128, 16 if rows <= 16 else 128)
    n_prefix, n_own, prefix_rows, own_rows = n_split
    ws, ws_bytes = None, 0
    if n_prefix + n_own > 1:
        need = B * T * Hq * (n_prefix + n_own) * (D + 2)  # gdn_paged_attn_workspace_bytes, in floats
        if workspace is None or workspace.numel() * workspace.element_size() < 4 * need:
            workspace = torch.empty(need, dtype=torch.float32, device=dev)
        ws, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    _lib.call(dev, "gdn_paged_attn", q.data_ptr(), None if gate is None else gate.data_ptr(), qg_ld, keys.data_ptr(),
              values.data_ptr(), table.data_ptr(), width, pos0.data_ptr(), None if n_new is None else n_new.data_ptr(),
              out.data_ptr(), D ** -0.5 if scale is None else float(scale), B, T, Hq, Hkv, D, n_blocks, block,
              kv_len_max, shared, n_prefix, n_own, prefix_rows, own_rows, ws, ws_bytes, _stream(dev))
    return out


def _refuse_attn(q, keys, values, table, pos0, kv_len_max, n_new, shared, gate, workspace, out) -> None:
    """Raises what is wrong with :func:`paged_attn`'s arguments."""
    _require_device((q, keys, values, table, pos0, n_new, gate, workspace, out),
                    ("q", "keys", "values", "table", "pos0", "n_new", "gate", "workspace", "out"))
    for t, n in ((q, "q"), (keys, "keys"), (values, "values"), (gate, "gate"), (out, "out")):
        if t is not None and t.dtype is not torch.bfloat16:
            raise ValueError(f"{n} must be bfloat16 (got {t.dtype})")
    if q.dim() != 4:
        raise ValueError(f"q must be [B, T, Hq, D] (got {tuple(q.shape)})")
    B, T, Hq, D = q.shape
    if keys.dim() != 4 or values.shape != keys.shape or not keys.is_contiguous() or not values.is_contiguous():
        raise ValueError("keys and values must be contiguous [n_blocks, Hkv, block, D] tensors of one shape")
    _, Hkv, block, Dk = keys.shape
    if Dk != D or Hkv == 0 or Hq % Hkv != 0:
        raise ValueError(f"pools of {Hkv} heads of {Dk} do not match q's {Hq} heads of {D}")
    if table.dim() != 2:
        raise ValueError("table must be [B, width]")
    width = table.shape[1]
    _i32(table, (B, width), "table")
    _i32(pos0, (B,), "pos0")
    if n_new is not None:
        _i32(n_new, (B,), "n_new")
    if not 0 <= shared * block <= kv_len_max - (T if n_new is None else 0) or kv_len_max > width * block:
        raise ValueError(f"kv_len_max={kv_len_max} must lie in [shared * block + T, width * block = {width * block}]")
    if gate is not None and gate.shape != (B, T, Hq * 2 * D):
        raise ValueError(f"gate must be [{B}, {T}, {Hq * 2 * D}]")
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    if out is not None and (out.shape != q.shape or not out.is_contiguous()):
        raise ValueError(f"out must be a contiguous [{B}, {T}, {Hq}, {D}] tensor")


# ------------------------------------------------------------------ cache

class BlockPool:
    """``n_blocks`` blocks of one attention layer's keys and values, and the
    list of those no row holds (on the device; the host keeps its length)."""

    def __init__(self, n_blocks: int, n_kv_heads: int, head_dim: int, block: int = 64,
                 device: Optional[torch.device] = None):
        if n_blocks <= 0:
            raise ValueError("a pool needs at least one block")
        if block < 64 or block & (block - 1):
            raise ValueError(f"block must be a power of two from 64 on (got {block})")
        self.keys = torch.empty(n_blocks, n_kv_heads, block, head_dim, dtype=torch.bfloat16, device=device)
        self.values = torch.empty_like(self.keys)
        self.free = torch.arange(n_blocks - 1, -1, -1, dtype=torch.int32, device=device)  # lowest block first
        self.n_free = torch.full((1,), n_blocks, dtype=torch.int32, device=device)
        self.free_blocks = n_blocks

    @property
    def n_blocks(self) -> int:
        return self.keys.shape[0]

    @property
    def block(self) -> int:
        return self.keys.shape[2]

    @property
    def device(self) -> torch.device:
        return self.keys.device


class PagedKVCache:
    """A batch of rows over a :class:`BlockPool`, with :class:`KVCache`'s verbs.

    Row b's position p is row ``p % block`` of block ``table[b, p // block]``.
    Before a layer writes T tokens, :meth:`reserve` makes room for them (one
    launch, nothing read back) and returns their slots; :meth:`advance` and
    :meth:`trim` move the lengths, and blocks that a rollback left unused go
    back to the pool at the next :meth:`reserve`.  The host keeps the lengths
    and the number of free blocks, so a full pool raises before any launch, and
    a step of the cache cannot be captured into a graph (its calls can).

    :meth:`fork` starts a batch on a prompt: the rows' tables list the prompt's
    full blocks in common (``shared`` of them, read once for the batch by
    :func:`paged_attn`), the rest of it is copied.  The prompt's cache keeps its
    blocks while such a batch lives.  :meth:`release` gives a batch's blocks back
    (a cache that is dropped without it keeps them).  All caches of one pool are
    used on one stream.
    """

    def __init__(self, pool: BlockPool, batch: int, capacity: int = 256):
        if batch < 0 or batch > 4096:
            raise ValueError(f"batch must lie in [0, 4096] (got {batch})")
        self.pool = pool
        self.table = torch.zeros(batch, max(1, self._blocks(capacity)), dtype=torch.int32, device=pool.device)
        self.held = torch.zeros(batch, dtype=torch.int32, device=pool.device)
        self.pos0 = torch.zeros(batch, dtype=torch.int32, device=pool.device)
        self.lengths = [0] * batch
        self.shared = 0
        self._held = [0] * batch
        self._prefix: Optional[PagedKVCache] = None  # whose blocks the shared ones are
        self._forks: "weakref.WeakSet[PagedKVCache]" = weakref.WeakSet()

    def _blocks(self, tokens: int) -> int:
        return -(-int(tokens) // self.pool.block)

    @property
    def batch(self) -> int:
        return len(self.lengths)

    @property
    def capacity(self) -> int:
        return self.table.shape[1] * self.pool.block

    @property
    def offset(self) -> int:
        """The longest row's length."""
        return max(self.lengths, default=0)

    def size(self) -> int:
        return self.offset

    @property
    def floor(self) -> int:
        """Positions that stay: the shared ones, and those that forks share."""
        return max([self.shared] + [c.shared for c in self._forks if c.batch]) * self.pool.block

    def _counts(self, n_new) -> List[int]:
        counts = [int(n) for n in n_new]
        if len(counts) != self.batch or any(n < 0 for n in counts):
            raise ValueError(f"n_new must hold {self.batch} counts (got {counts})")
        return counts

    def _not_captured(self) -> None:
        if self.pool.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the host keeps a paged cache's lengths and block counts, which a graph's replays would "
                               "not move: capture paged_tables, attn_rope and paged_attn over tensors of their own")

    def _tables(self, lengths: torch.Tensor, host: Sequence[int], T: int, n_new: Optional[torch.Tensor],
                new: Sequence[int]) -> torch.Tensor:
        """One ``gdn_paged_tables`` in place, with the host's counts kept in step."""
        self._not_captured()
        need = [max(self._blocks(n + m), self.shared) for n, m in zip(host, new)]
        free = self.pool.free_blocks + sum(self._held) - sum(need)
        if free < 0:
            raise RuntimeError(f"block pool exhausted: {-free} blocks short for {sum(new)} new tokens")
        if max(need, default=0) > self.table.shape[1]:
            width = max(max(need), self.table.shape[1] + self._blocks(KVCache.step))
            table = torch.zeros(self.batch, width, dtype=torch.int32, device=self.pool.device)
            table[:, : self.table.shape[1]] = self.table
            self.table = table
        slots, _, _ = paged_tables(lengths, T, self.table, self.held, self.pool.free, self.pool.n_free,
                                   self.pool.block, n_new=n_new, shared=self.shared, held_out=self.held,
                                   n_free_out=self.pool.n_free)
        self._held = need
        self.pool.free_blocks = free
        return slots

    def reserve(self, T: int, n_new: Optional[Sequence[int]] = None,
                counts: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Room for T new tokens a row (``n_new[b]`` of them, padded to T);
        returns their slots ``[B, T]``.  ``counts`` is n_new on the device
        (:meth:`counts`), where the caller has it already."""
        T = int(T)
        if n_new is None:
            return self._tables(self.pos0, self.lengths, T, None, [T] * self.batch)
        new = self._counts(n_new)
        if max(new, default=0) > T:
            raise ValueError(f"n_new {new} must not exceed T={T}")
        return self._tables(self.pos0, self.lengths, T, self.counts(new) if counts is None else counts, new)

    def counts(self, n_new: Sequence[int]) -> torch.Tensor:
        """Per-row counts on the device (through pinned memory: no launch waits).
        A captured graph would copy them from memory that is gone at its replay."""
        if self.pool.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("per-row counts come from the host and cannot be captured into a graph")
        host = torch.tensor([int(n) for n in n_new], dtype=torch.int32)
        if self.pool.device.type != "cuda":
            return host
        return host.pin_memory().to(self.pool.device, non_blocking=True)

    def advance(self, T: int, n_new: Optional[Sequence[int]] = None, counts: Optional[torch.Tensor] = None) -> None:
        T = int(T)
        self._not_captured()
        if n_new is None:
            self.lengths = [n + T for n in self.lengths]
            _pos_add(self.pos0, T, -2**31)
        else:
            new = self._counts(n_new)
            self.lengths = [n + m for n, m in zip(self.lengths, new)]
            self.pos0.add_(self.counts(new) if counts is None else counts)

    def trim(self, n: int) -> int:
        """Drops the last ``n`` positions of every row (the drafter's rollback),
        at most down to the shared ones; returns how many the longest row lost."""
        self._not_captured()
        floor = self.floor
        n = max(0, min(int(n), self.offset - floor))
        # rows shorter than the floor (none of a fork's) keep what they hold
        if any(m < floor for m in self.lengths):
            raise RuntimeError("rows shorter than what forks share cannot be trimmed")
        self.lengths = [max(floor, m - n) for m in self.lengths]
        _pos_add(self.pos0, -n, floor)
        return n

    def filter(self, keep: Sequence[int]) -> None:
        """Keeps rows ``keep`` (a batch leave); the others' blocks go back to the pool."""
        keep = [int(i) for i in keep]
        if len(set(keep)) != len(keep) or any(not 0 <= i < self.batch for i in keep):
            raise ValueError(f"keep must name rows of [0, {self.batch}) once each (got {keep})")
        if any(c.batch for c in self._forks) and len(keep) < self.batch:
            raise RuntimeError("rows whose blocks a fork shares cannot leave before it")
        if len(keep) < self.batch:
            stay = [self.lengths[i] if i in set(keep) else 0 for i in range(self.batch)]
            self._tables(self.counts(stay), stay, 0, None, [0] * self.batch)
        idx = torch.as_tensor(keep, dtype=torch.long, device=self.pool.device)
        self.table = self.table.index_select(0, idx)
        self.held = self.held.index_select(0, idx)
        self.pos0 = self.pos0.index_select(0, idx)
        self.lengths = [self.lengths[i] for i in keep]
        self._held = [self._held[i] for i in keep]
        if not keep:
            self.shared, self._prefix = 0, None

    def release(self) -> None:
        """Gives every row's blocks back; the cache then has no rows."""
        self.filter([])

    def _like(self, batch: int) -> "PagedKVCache":
        """Rows over the same pool whose tables start with this cache's shared blocks."""
        c = PagedKVCache(self.pool, batch, self.capacity)
        if self.shared:
            c._share(self._prefix, self.table[:1], self.shared)
        return c

    def _share(self, prefix: "PagedKVCache", table: torch.Tensor, blocks: int) -> None:
        self.shared, self._prefix = blocks, prefix
        self.table[:, :blocks] = table[:, :blocks]
        self.held.fill_(blocks)
        self._held = [blocks] * self.batch
        prefix._forks.add(self)

    def _fill(self, n: int, table: torch.Tensor) -> None:
        """Every row's positions from the shared blocks on up to n, copied from the
        blocks of ``table`` ``[1, width]``.  Where that fails the cache has no rows
        and holds no blocks."""
        rows = self.batch
        try:
            self.pos0.fill_(n)
            self.lengths = [n] * rows
            self._tables(self.pos0, self.lengths, 0, None, [0] * rows)
            lo, hi = self.shared, self._blocks(n)
            if hi > lo:
                src = table[0, lo:hi].long()
                for pool in (self.pool.keys, self.pool.values):
                    blocks = pool.index_select(0, src)
                    for b in range(rows):
                        pool.index_copy_(0, self.table[b, lo:hi].long(), blocks)
        except BaseException:
            if sum(self._held) > self.shared * rows:
                self._tables(self.counts([0] * rows), [0] * rows, 0, None, [0] * rows)
            self.table, self.held, self.pos0 = self.table[:0], self.held[:0], self.pos0[:0]
            self.lengths, self._held, self.shared, self._prefix = [], [], 0, None
            raise

    def fork(self, n: int) -> "PagedKVCache":
        """n rows that continue this one-row cache's prompt, sharing its full blocks."""
        if self.batch != 1:
            raise ValueError(f"fork takes a cache of one row (got {self.batch})")
        c = PagedKVCache(self.pool, n, self.capacity)
        full = self.lengths[0] // self.pool.block
        if self._blocks(self.lengths[0]) > full and self.pool.free_blocks < n:
            raise RuntimeError(f"block pool exhausted: {n} rows need {n - self.pool.free_blocks} blocks more")
        if full:
            # blocks that this cache itself shares stay while it does
            c._share(self, self.table, full)
        c._fill(self.lengths[0], self.table)
        return c

    def extract(self, row: int) -> "PagedKVCache":
        """A one-row copy of row ``row`` (its shared blocks stay shared)."""
        row = int(row)
        if not 0 <= row < self.batch:
            raise ValueError(f"row {row} is not in [0, {self.batch})")
        if self._blocks(self.lengths[row]) - self.shared > self.pool.free_blocks:
            raise RuntimeError("block pool exhausted: no room for a row's copy")
        c = self._like(1)
        c._fill(self.lengths[row], self.table[row : row + 1])
        return c

    @classmethod
    def merge(cls, caches: Sequence["PagedKVCache"]) -> "PagedKVCache":
        """Rows of several caches of one pool as one batch (a batch join).  The
        rows move: the caches given have none afterwards.  One without rows joins
        any others of its pool."""
        first = next((c for c in caches if c.batch), caches[0])
        if len({id(c) for c in caches}) != len(caches):
            raise ValueError("a cache cannot be merged with itself")
        if any(c.pool is not first.pool or c.batch and (c.shared != first.shared or c._prefix is not first._prefix)
               for c in caches):
            raise ValueError("caches of different pools or prefixes cannot be merged")
        if any(f.batch for c in caches for f in c._forks):
            raise RuntimeError("rows whose blocks a fork shares cannot move")
        out = cls(first.pool, sum(c.batch for c in caches), max(c.capacity for c in caches))
        if first.batch and first.shared:
            out._share(first._prefix, first.table[:1], first.shared)
        r = 0
        for c in caches:
            out.table[r : r + c.batch, : c.table.shape[1]] = c.table
            r += c.batch
        out.held = torch.cat([c.held for c in caches])
        out.pos0 = torch.cat([c.pos0 for c in caches])
        out.lengths = [n for c in caches for n in c.lengths]
        out._held = [n for c in caches for n in c._held]
        for c in caches:
            c.table, c.held, c.pos0 = c.table[:0], c.held[:0], c.pos0[:0]
            c.lengths, c._held = [], []
            c.shared, c._prefix = 0, None
        return out

    @property
    def state(self):
        """Copies of keys and values up to the longest row, ``[B, Hkv, offset, D]``
        (past a shorter row's length its entries are unset)."""
        n = self._blocks(self.offset)
        pages = self.table[:, :n].long().clamp_(0, self.pool.n_blocks - 1)
        _, Hkv, bs, D = self.pool.keys.shape
        return tuple(p[pages].transpose(1, 2).reshape(self.batch, Hkv, n * bs, D)[..., : self.offset, :]
                     for p in (self.pool.keys, self.pool.values))

    @state.setter
    def state(self, kv) -> None:
        """Replaces the contents by ``[keys, values]`` ``[B, Hkv, L, D]``: every row
        then holds L positions of its own and shares none (a prefix-cache
        restore, as with :class:`KVCache`).  Where the pool has room for both, the
        old rows go last, and a step that fails leaves them."""
        keys, values = kv
        _, Hkv, bs, D = self.pool.keys.shape
        if keys.dim() != 4 or values.shape != keys.shape or (keys.shape[1], keys.shape[3]) != (Hkv, D):
            raise ValueError(f"state must be [keys, values] of one [B, {Hkv}, L, {D}] shape")
        B, _, L, _ = keys.shape
        own = sum(h - self.shared for h in self._held)
        if B * self._blocks(L) > self.pool.free_blocks + own:
            raise RuntimeError("block pool exhausted: no room for the state")
        if any(c.batch for c in self._forks):
            raise RuntimeError("rows whose blocks a fork shares cannot be replaced before it")
        fresh = PagedKVCache(self.pool, B, max(L, self.capacity))
        keys, values = keys.to(self.pool.keys), values.to(self.pool.values)
        beside = B * self._blocks(L) <= self.pool.free_blocks
        if not beside:
            self.release()
        try:
            slots = fresh.reserve(L).long()
            for pool, x in ((self.pool.keys, keys), (self.pool.values, values)):
                pool[slots // bs, :, slots % bs] = x.transpose(1, 2)
            fresh.advance(L)
        except BaseException:
            if any(fresh._held):
                fresh.release()
            raise
        if beside:
            self.release()
        self.table, self.held, self.pos0 = fresh.table, fresh.held, fresh.pos0
        self.lengths, self._held = fresh.lengths, fresh._held
