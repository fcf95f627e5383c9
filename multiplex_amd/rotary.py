"""Rotary positions from a table of frequencies, with the q/k norm and the cache
append of an attention layer in one launch (``gdn_attn_rope``).

:class:`Rotary` holds what a layer's rotary embedding needs: which pairs of a
head's dims turn together (``(i, i + rot/2)``, or ``(2i, 2i + 1)`` for mlx's
``traditional=True``), how many dims take part, and each pair's frequency,
scaled for contexts longer than the model's own where asked.  Frequencies are
kept as turns per position in 64-bit fixed point, so an angle is as exact at
position 1,000,000 as at 1 (a 32-bit product of position and frequency is off
by 0.06 rad there).
"""

from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

from . import _lib
from .gated_delta import _dtype_code, _require_device, _stream

__all__ = ["Rotary", "attn_rope"]


# what a rope_scaling dict may hold, by its kind; _SAID goes with every kind and changes nothing here (a base other
# than the layer's is refused; a token of text has one position in all sections of a head)
_SAID = ("type", "rope_type", "rope_theta", "partial_rotary_factor", "max_position_embeddings",
         "original_max_position_embeddings", "finetuned", "mrope_section", "mrope_interleaved")
_READ = {
    "linear": ("factor",),
    "yarn": ("factor", "beta_fast", "beta_slow", "attention_factor", "mscale", "mscale_all_dim", "truncate"),
}


def _kind(scaling: Optional[dict]) -> str:
    return (scaling.get("type") or scaling.get("rope_type") or "default") if scaling else "default"


def _number(scaling: dict, key: str, default: Optional[float] = None) -> float:
    x = scaling.get(key)
    x = default if x is None else x
    if x is None or not math.isfinite(x):
        raise ValueError(f"{_kind(scaling)} scaling needs a finite {key} (got {scaling.get(key)})")
    return float(x)


def _scaled(inv: Sequence[float], rot: int, base: float, scaling: Optional[dict]):
    """``(frequencies, factor)`` of a ``rope_scaling`` dict as model
    configurations hold it.  A key that would change them and is not read raises."""
    kind = _kind(scaling)
    if scaling and scaling.get("rope_theta") is not None and float(scaling["rope_theta"]) != base:
        raise ValueError(f"rope scaling says rope_theta={scaling['rope_theta']}, the layer base {base}")
    if kind == "default":
        return list(inv), 1.0
    if kind not in _READ:
        raise ValueError(f"rope scaling {kind!r} is not one of default, linear, yarn (give inv_freq instead)")
    unread = sorted(k for k, v in scaling.items() if v is not None and k not in _SAID and k not in _READ[kind])
    if unread:
        raise ValueError(f"{kind} scaling does not read {', '.join(unread)} (give inv_freq instead)")
    s = _number(scaling, "factor")
    if not s > 0:
        raise ValueError(f"rope scaling factor must be positive (got {s})")
    if kind == "linear":
        return [f / s for f in inv], 1.0
    # pairs that turn more than beta_fast times over the original context keep
    # their frequency, those below beta_slow turns are stretched by s, a ramp
    # over the pair index in between (its ends whole pairs, unless truncate is
    # false)
    context = _number(scaling, "original_max_position_embeddings")
    fast, slow = float(scaling.get("beta_fast") or 32.0), float(scaling.get("beta_slow") or 1.0)
    if not (context > 0 and base > 1 and fast > 0 and slow > 0):
        raise ValueError("yarn scaling needs base > 1 and a positive context and betas")

    def pair(turns):
        return rot * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(base))

    lo, hi = pair(fast), pair(slow)
    truncate = scaling.get("truncate")
    if truncate is None or truncate:
        lo, hi = math.floor(lo), math.ceil(hi)
    lo, hi = max(lo, 0), min(hi, rot - 1)
    span = hi - lo if hi != lo else 0.001
    ramp = [min(max((i - lo) / span, 0.0), 1.0) for i in range(rot // 2)]
    return [f / s * r + f * (1.0 - r) for f, r in zip(inv, ramp)], _yarn_factor(s, scaling)


def _yarn_factor(s: float, scaling: dict) -> float:
    """What the rotated dims grow by: ``attention_factor``, or 1 + ln(s) / 10, or
    with both mscales given the ratio of their 1 + mscale ln(s) / 10."""
    if scaling.get("attention_factor") is not None:
        return _number(scaling, "attention_factor")
    m, m_all = _number(scaling, "mscale", 1.0), _number(scaling, "mscale_all_dim", 0.0)

    def grown(m):
        return 0.1 * m * math.log(s) + 1.0 if s > 1 else 1.0

    if scaling.get("mscale") is not None and m != 0 and m_all != 0:
        return grown(m) / grown(m_all)
    if m != 1 or m_all != 0:  # read by some implementations, passed over by others
        raise ValueError("yarn scaling takes mscale and mscale_all_dim together (or give attention_factor)")
    return grown(1.0)


class Rotary(torch.nn.Module):
    """The rotary embedding of a head's first ``rot`` dims.

    ``inv_freq[i] = base ** (-2 i / rot)`` radians per position, scaled by
    ``scaling`` (``{"type": "linear", "factor": s}``, or ``"yarn"`` with
    ``factor``, ``original_max_position_embeddings`` and optionally
    ``beta_fast``, ``beta_slow``, ``truncate``, and ``attention_factor`` or
    ``mscale`` with ``mscale_all_dim``; a key that would change them and is not
    read raises), or given as ``inv_freq``.  ``interleaved`` pairs neighbouring
    dims.
    """

    def __init__(self, rot: int, base: float, *, interleaved: bool = False, scaling: Optional[dict] = None,
                 inv_freq: Optional[Sequence[float]] = None, device=None):
        super().__init__()
        if rot < 0 or rot % 2 != 0:
            raise ValueError(f"rot must be even (got {rot})")
        if not base > 0:
            raise ValueError(f"base must be positive (got {base})")
        self.rot, self.base, self.interleaved = int(rot), float(base), bool(interleaved)
        # what gdn_attn_qk computes: half pairs of unscaled frequencies
        self.plain = not interleaved and _kind(scaling) == "default" and inv_freq is None
        if inv_freq is None:
            inv = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
            self.inv_freq, self.factor = _scaled(inv, rot, float(base), scaling)
        else:
            if scaling:
                raise ValueError("give scaling or inv_freq, not both")
            self.inv_freq, self.factor = [float(f) for f in inv_freq], 1.0
            if len(self.inv_freq) != rot // 2 or not all(map(math.isfinite, self.inv_freq)):
                raise ValueError(f"inv_freq must hold {rot // 2} finite values")
        fixed = []
        for f in self.inv_freq:
            u = round(math.fmod(f / (2 * math.pi), 1.0) * 2.0**64) % 2**64
            fixed.append(u - 2**64 if u >= 2**63 else u)  # the same 64 bits as a signed number
        self._fixed = fixed
        self.register_buffer("turns", torch.tensor(fixed, dtype=torch.int64, device=device), persistent=False)

    def _apply(self, fn, recurse=True):
        """Moves the module; the frequencies are formed anew where they arrive, as
        a checkpoint for a layer made without memory does not hold them."""
        super()._apply(fn, recurse)
        dev = self.turns.device
        self.turns = torch.tensor(self._fixed, dtype=torch.int64, device=dev)
        return self


def _tokens(t: torch.Tensor, B: int, T: int, width: int, what: str) -> int:
    """Elements from one token to the next of a ``[B, T, width]`` view whose
    rows are contiguous (a column slice of a fused GEMM output)."""
    if t.shape != (B, T, width):
        raise ValueError(f"{what} must be a [{B}, {T}, {width}] view with contiguous rows (got {tuple(t.shape)})")
    row, token, dim = t.stride()
    if dim != 1 and width > 1:
        raise ValueError(f"{what} must be a [{B}, {T}, {width}] view with contiguous rows")
    ld = token if T > 1 else (row if B > 1 else width)
    if ld < width or (B > 1 and T > 1 and row != T * ld):
        raise ValueError(f"{what}: tokens must be one stride apart")
    return ld


def attn_rope(qg: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, q_norm_w: Optional[torch.Tensor],
              k_norm_w: Optional[torch.Tensor], eps: float, pos0: torch.Tensor, keys: torch.Tensor,
              values: torch.Tensor, rotary: Rotary, *, slots: Optional[torch.Tensor] = None, gated: bool = True,
              q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q/k RMSNorm, rotary positions and cache append (``gdn_attn_rope``).

    qg ``[B, T, Hq*2D]`` (per head: q, then the output gate; ``[B, T, Hq*D]``
    with ``gated=False``); k_new, v_new ``[B, T, Hkv*D]`` (each may be a column
    slice of one GEMM output); norm weights ``[D]`` or both None; pos0 ``[B]``
    int32 position of each row's first token.  With ``slots`` ``[B, T]``
    (:func:`multiplex_amd.paged_tables`) keys and values are block pools
    ``[n_blocks, Hkv, block, D]``, and a token of slot -1 is padding: its q is
    zeros, its k and v are not stored.  Without, they are a dense cache
    ``[B, Hkv, cap, D]``, appended to at pos0.  Returns q ``[B, T, Hq, D]``.

    The norm is not rounded before the rotation (:func:`attention.attn_qk`
    rounds there, as the reference does).
    """
    dev = qg.device
    index, turns = qg.get_device(), rotary._buffers["turns"]  # (a module's attribute is looked up three times as long)
    if index < 0 or qg.dim() != 3 or keys.dim() != 4:
        _refuse(qg, k_new, v_new, q_norm_w, k_norm_w, pos0, keys, values, turns, slots, gated, q_out)
    B, T, width = qg.shape
    n_blocks, Hkv, block, D = keys.shape
    q_head = 2 * D if gated else D
    Hq = width // q_head
    bf16, i32 = torch.bfloat16, torch.int32
    kv = (B, T, Hkv * D)
    if not (qg.dtype is bf16 and k_new.dtype is bf16 and v_new.dtype is bf16 and keys.dtype is bf16
            and values.dtype is bf16 and k_new.get_device() == v_new.get_device() == keys.get_device()
            == values.get_device() == pos0.get_device() == turns.get_device() == index
            and values.shape == keys.shape and keys.is_contiguous() and values.is_contiguous()
            and Hkv > 0 and Hq > 0 and width == Hq * q_head and Hq % Hkv == 0
            and k_new.shape == kv and v_new.shape == kv
            and pos0.dtype is i32 and pos0.shape == (B,) and pos0.is_contiguous()
            and (n_blocks == B and block >= T if slots is None else
                 slots.dtype is i32 and slots.shape == (B, T) and slots.get_device() == index and slots.is_contiguous())
            and (q_norm_w is None and k_norm_w is None or q_norm_w is not None and k_norm_w is not None
                 and q_norm_w.shape == k_norm_w.shape == (D,) and q_norm_w.dtype is k_norm_w.dtype
                 and q_norm_w.get_device() == k_norm_w.get_device() == index)
            and (q_out is None or q_out.dtype is bf16 and q_out.shape == (B, T, Hq, D) and q_out.get_device() == index
                 and q_out.is_contiguous())):
        _refuse(qg, k_new, v_new, q_norm_w, k_norm_w, pos0, keys, values, turns, slots, gated, q_out)
    qg_ld = _tokens(qg, B, T, width, "qg")
    kv_ld = _tokens(k_new, B, T, Hkv * D, "k_new")
    if _tokens(v_new, B, T, Hkv * D, "v_new") != kv_ld:
        raise ValueError("k_new and v_new must share one token stride")
    qn = kn = None
    wdt = 0
    if q_norm_w is not None:
        if not (q_norm_w.is_contiguous() and k_norm_w.is_contiguous()):
            q_norm_w, k_norm_w = q_norm_w.contiguous(), k_norm_w.contiguous()
        qn, kn, wdt = q_norm_w.data_ptr(), k_norm_w.data_ptr(), _dtype_code(q_norm_w, "q_norm_w")
    if q_out is None:
        q_out = qg.new_empty((B, T, Hq, D))
    _lib.call(dev, "gdn_attn_rope", qg.data_ptr(), qg_ld, q_head, k_new.data_ptr(), v_new.data_ptr(), kv_ld, qn, kn,
              wdt, float(eps), pos0.data_ptr(), None if slots is None else slots.data_ptr(), turns.data_ptr(),
              rotary.factor, int(rotary.interleaved), q_out.data_ptr(), keys.data_ptr(), values.data_ptr(), B, T, Hq,
              Hkv, D, n_blocks, block, rotary.rot, _stream(dev))
    return q_out


def _refuse(qg, k_new, v_new, q_norm_w, k_norm_w, pos0, keys, values, turns, slots, gated, q_out) -> None:
    """Raises what is wrong with :func:`attn_rope`'s arguments."""
    _require_device((qg, k_new, v_new, q_norm_w, k_norm_w, pos0, keys, values, slots, turns, q_out),
                    ("qg", "k_new", "v_new", "q_norm_w", "k_norm_w", "pos0", "keys", "values", "slots", "rotary", "q_out"))
    for t, n in ((qg, "qg"), (k_new, "k_new"), (v_new, "v_new"), (keys, "keys"), (values, "values"), (q_out, "q_out")):
        if t is not None and t.dtype is not torch.bfloat16:
            raise ValueError(f"{n} must be bfloat16 (got {t.dtype})")
    if keys.dim() != 4 or values.shape != keys.shape or not keys.is_contiguous() or not values.is_contiguous():
        raise ValueError("keys and values must be contiguous [n_blocks, Hkv, block, D] tensors of one shape")
    n_blocks, Hkv, block, D = keys.shape
    if qg.dim() != 3:
        raise ValueError(f"qg must be [B, T, Hq*{2 if gated else 1}D] (got {tuple(qg.shape)})")
    B, T, width = qg.shape
    q_head = 2 * D if gated else D
    Hq = width // q_head
    if Hq == 0 or width != Hq * q_head or Hkv == 0 or Hq % Hkv != 0:
        raise ValueError(f"qg's {width} columns are not heads of {q_head}, a multiple of {Hkv} of them")
    _tokens(k_new, B, T, Hkv * D, "k_new")
    _tokens(v_new, B, T, Hkv * D, "v_new")
    if pos0.dtype is not torch.int32 or tuple(pos0.shape) != (B,) or not pos0.is_contiguous():
        raise ValueError(f"pos0 must be a contiguous int32 [{B}] tensor")
    if slots is not None:
        if slots.dtype is not torch.int32 or tuple(slots.shape) != (B, T) or not slots.is_contiguous():
            raise ValueError(f"slots must be a contiguous int32 [{B}, {T}] tensor")
    elif n_blocks != B or block < T:
        raise ValueError(f"without slots keys must be a [B={B}, Hkv, cap >= {T}, D] cache (got {tuple(keys.shape)})")
    if (q_norm_w is None) != (k_norm_w is None):
        raise ValueError("give both norm weights or neither")
    if q_norm_w is not None and (tuple(q_norm_w.shape) != (D,) or tuple(k_norm_w.shape) != (D,)
                                 or q_norm_w.dtype != k_norm_w.dtype):
        raise ValueError(f"norm weights must be [{D}] tensors of one dtype")
    if q_out is not None and (tuple(q_out.shape) != (B, T, Hq, D) or not q_out.is_contiguous()):
        raise ValueError(f"q_out must be a contiguous [{B}, {T}, {Hq}, {D}] tensor")
