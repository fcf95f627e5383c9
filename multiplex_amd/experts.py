"""Sparse MLPs: a router's choice of experts, their products, and the layer.

The reference's trunks come with a dense MLP in every layer or with a sparse
one (mlx-lm's ``qwen3_5`` decoder layer takes either): many small SwiGLU
experts, of which a router takes a few per token, beside a shared expert that
every token runs.

  route_experts   scores, bias, groups, top-k, weights (``gdn_route_experts``)
  expert_mlp      the chosen experts' products and their weighted sum
                  (``gdn_expert_mlp``; nothing is read back to the host)
  SparseMLP       router, shared expert (:func:`multiplex_amd.linear_act`) and
                  experts; :class:`DecoderLayer` and :class:`MTPHead` take it for
                  ``AttentionArgs(num_experts=...)``
"""

from __future__ import annotations

import functools
from typing import Optional, Tuple

import torch

from . import _lib
from .gated_delta import _dtype_code, _ptr, _require_device, _stream
from .linear import _FLOATS, _even_rows, _forward_only, _out_rows, _watched, linear_act

__all__ = ["route_experts", "expert_mlp", "expert_mlp_workspace_bytes", "SparseMLP"]

_SCORING = {"softmax": 0, "sigmoid": 1}


def route_experts(logits: torch.Tensor, k: int, *, scoring: str = "softmax", bias: Optional[torch.Tensor] = None,
                  groups: int = 1, top_groups: int = 1, group_best: int = 2, renormalize: bool = True,
                  scale: float = 1.0, n_new: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(indices [..., k] int32, weights [..., k] fp32)`` of the k experts each token
    takes, from the router's ``logits [..., E]`` (bf16, fp16 or fp32; a column slice
    of a wider product is read in place).

    ``scoring``: "softmax" over the experts or "sigmoid" of each.  The choice goes
    by the score plus ``bias [E]`` (fp32), the weights are the scores alone.  With
    ``groups`` > 1, equal ranges of experts, only the ``top_groups`` ranges with the
    largest sums of their ``group_best`` (1 or 2) best can be chosen from (+inf and
    -inf, of biases, together count as -inf).
    ``renormalize`` divides the weights by their sum, ``scale`` multiplies them.

    The experts stand in the order of falling score, of equals the lowest index
    first; a NaN counts below every number, so the indices are always k different
    ones.  A token whose chosen scores are all 0 (its logits -inf) gets weights 0.
    ``n_new [B]`` int32, with logits ``[B, T, E]``: tokens past it are padding,
    with indices -1 and weights 0, which :func:`expert_mlp` passes over.
    Computed in 64 bits, so that scores that differ at all are told apart.
    """
    # a plain call's checks in a few operations; what is wrong, or laid out otherwise, is looked into below
    index, code, d = logits.get_device(), _FLOATS.get(logits.dtype), logits.dim()
    ld = _even_rows(logits) if d > 1 else None
    if (index < 0 or code is None or ld is None or k.__class__ is not int or k <= 0 or scoring not in _SCORING
            or _watched() or torch.is_grad_enabled() and (logits.requires_grad or bias is not None and bias.requires_grad)
            or n_new is not None and not (d == 3 and n_new.dtype is torch.int32 and n_new.get_device() == index
                                          and n_new.shape == logits.shape[:1] and n_new.is_contiguous())
            or bias is not None and not (bias.dtype is torch.float32 and bias.get_device() == index
                                         and bias.is_contiguous() and bias.shape == logits.shape[-1:])):
        return _route_general(logits, k, scoring, bias, groups, top_groups, group_best, renormalize, scale, n_new)
    dev, *lead = logits.device, *logits.shape
    E = lead[-1]
    lead[-1] = k
    indices = torch.empty(lead, dtype=torch.int32, device=dev)
    weights = torch.empty(lead, dtype=torch.float32, device=dev)
    T = lead[1] if n_new is not None else 1
    _lib.call(dev, "gdn_route_experts", logits.data_ptr(), code, ld, None if bias is None else bias.data_ptr(),
              None if n_new is None else n_new.data_ptr(), indices.data_ptr(), weights.data_ptr(),
              lead[0] if n_new is not None else indices.numel() // k, T, E, k, _SCORING[scoring], int(groups),
              int(top_groups), int(group_best), 1 if renormalize else 0, float(scale), _stream(dev))
    return indices, weights


def _route_general(logits, k, scoring, bias, groups, top_groups, group_best, renormalize, scale, n_new):
    """:func:`route_experts` of any layout; raises what is wrong with its arguments."""
    dev = _require_device((logits, bias, n_new), ("logits", "bias", "n_new"))
    if logits.dim() < 1:
        raise ValueError("logits must be [..., E]")
    if scoring not in _SCORING:
        raise ValueError(f"scoring must be one of {list(_SCORING)} (got {scoring!r})")
    dt = _dtype_code(logits, "logits")
    *lead, E = logits.shape
    k, groups, top_groups, group_best = int(k), int(groups), int(top_groups), int(group_best)
    _forward_only((logits, bias), ("logits", "bias"))
    if bias is not None and (bias.dtype is not torch.float32 or bias.shape != (E,)):
        raise ValueError(f"bias must be float32 [{E}] (got {bias.dtype} {list(bias.shape)})")
    B, T = logits.shape[:-1].numel(), 1
    if n_new is not None:
        if len(lead) != 2:
            raise ValueError("n_new needs logits of shape [B, T, E]")
        B, T = lead
        if n_new.dtype is not torch.int32 or n_new.shape != (B,):
            raise ValueError(f"n_new must be int32 [{B}] (got {n_new.dtype} {list(n_new.shape)})")
        n_new = n_new.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    ld = _even_rows(logits)
    if ld is None:
        logits, ld = logits.contiguous(), E
    indices = torch.empty((*lead, k), dtype=torch.int32, device=dev) if k > 0 else None
    weights = torch.empty((*lead, k), dtype=torch.float32, device=dev) if k > 0 else None
    _lib.call(dev, "gdn_route_experts", logits.data_ptr(), dt, ld, _ptr(bias), _ptr(n_new), _ptr(indices),
              _ptr(weights), B, T, E, k, _SCORING[scoring], groups, top_groups, group_best, int(bool(renormalize)),
              float(scale), _stream(dev))
    return indices, weights


@functools.lru_cache(maxsize=1024)
def expert_mlp_workspace_bytes(tokens: int, hidden: int, inner: int, experts: int, k: int) -> int:
    """Bytes that :func:`expert_mlp` needs as its workspace."""
    return int(_lib.load().gdn_expert_mlp_workspace_bytes(tokens, hidden, inner, experts, k))


def expert_mlp(x: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor, indices: torch.Tensor,
               weights: torch.Tensor, *, base: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``base + sum_j weights[..., j] * down_e(silu(gate_e(x)) * up_e(x))`` over each
    token's experts ``e = indices[..., j]`` (``gdn_expert_mlp``).

    x ``[..., H]``, gate_up ``[E, 2I, H]`` (per expert the gate's rows, then up's),
    down ``[E, H, I]``, base ``[..., H]`` bf16; H and I multiples of 8, the
    experts' weights and ``out``'s rows 16-byte aligned; indices ``[..., k]`` int32 and
    weights ``[..., k]`` fp32 as :func:`route_experts` returns them.  A choice outside ``[0, E)`` adds nothing, one that stands twice is
    added twice; a token without any is its base, or 0.  An expert's inner values
    are rounded to bf16, its result to 12 bits of significand or not at all (off by
    at most 2^-12 of itself), their fp32 sum once.

    ``workspace``: :func:`expert_mlp_workspace_bytes` bytes (allocated when absent
    or too small); calls that overlap need one each.  ``out`` may be the base
    itself (which may be x), and otherwise lies apart from all that is read (other
    columns of one buffer are refused too).  There is no backward.
    """
    index, bf16 = x.get_device(), torch.bfloat16
    E, H, I = down.shape if down.dim() == 3 else (0, 0, 0)
    lead, k = x.shape[:-1], indices.shape[-1] if indices.dim() else 0
    # a plain call's checks in a few operations; what is wrong, or laid out otherwise, is looked into below
    if not (index >= 0 and (out is None or out is base) and x.dtype is bf16 and gate_up.dtype is bf16 and down.dtype is bf16
            and indices.dtype is torch.int32 and weights.dtype is torch.float32 and gate_up.get_device() == index
            and down.get_device() == index and indices.get_device() == index and weights.get_device() == index
            and gate_up.shape == (E, 2 * I, H) and x.dim() > 0 and x.shape[-1] == H and indices.shape[:-1] == lead
            and weights.shape == indices.shape and x.is_contiguous() and gate_up.is_contiguous()
            and down.is_contiguous() and indices.is_contiguous() and weights.is_contiguous() and x.data_ptr() % 16 == 0
            and (base is None or base.dtype is bf16 and base.get_device() == index and base.shape == x.shape
                 and base.is_contiguous() and base.data_ptr() % 16 == 0)
            and (workspace is None or workspace.get_device() == index and workspace.is_contiguous()) and not _watched()
            and not (torch.is_grad_enabled() and (x.requires_grad or gate_up.requires_grad or down.requires_grad or
                                                  weights.requires_grad or base is not None and base.requires_grad))):
        return _expert_mlp_general(x, gate_up, down, indices, weights, base, out, workspace)
    dev = x.device
    return _expert_mlp_call(dev, x, H, gate_up, down, indices, weights, base, H,
                            torch.empty_like(x) if out is None else out, H, workspace,
                            x.numel() // H if H else 0, H, I, E, k)


def _expert_mlp_call(dev, x, ldx, gate_up, down, indices, weights, base, ldb, out, ldo, workspace, N, H, I, E, k):
    need = expert_mlp_workspace_bytes(N, H, I, E, k)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    _lib.call(dev, "gdn_expert_mlp", x.data_ptr(), ldx, gate_up.data_ptr(), down.data_ptr(), indices.data_ptr(),
              weights.data_ptr(), None if base is None else base.data_ptr(), ldb, out.data_ptr(), ldo, N, H, I, E, k,
              workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream(dev))
    return out


def _expert_mlp_general(x, gate_up, down, indices, weights, base, out, workspace):
    """:func:`expert_mlp` of any layout; raises what is wrong with its arguments."""
    dev = _require_device((x, gate_up, down, indices, weights, base, out, workspace),
                          ("x", "gate_up", "down", "indices", "weights", "base", "out", "workspace"))
    bf16 = torch.bfloat16
    if x.dtype is not bf16 or gate_up.dtype is not bf16 or down.dtype is not bf16:
        raise ValueError(f"x, gate_up and down must be bfloat16 (got {x.dtype}, {gate_up.dtype}, {down.dtype})")
    if x.dim() < 1 or down.dim() != 3 or gate_up.dim() != 3:
        raise ValueError("x must be [..., H], gate_up [E, 2I, H] and down [E, H, I]")
    H = x.shape[-1]
    E, _, I = down.shape
    if gate_up.shape != (E, 2 * I, H) or down.shape[1] != H or not gate_up.is_contiguous() or not down.is_contiguous():
        raise ValueError(f"gate_up must be a contiguous [E, 2I, {H}] and down a contiguous [E, {H}, I] of the same experts "
                         f"(got {list(gate_up.shape)}, {list(down.shape)})")
    lead = x.shape[:-1]
    k = indices.shape[-1] if indices.dim() else 0
    if indices.dtype is not torch.int32 or indices.shape != (*lead, k):
        raise ValueError(f"indices must be int32 {list(lead)} + [k] (got {indices.dtype} {list(indices.shape)})")
    if weights.dtype is not torch.float32 or weights.shape != indices.shape:
        raise ValueError(f"weights must be float32 {list(indices.shape)} (got {weights.dtype} {list(weights.shape)})")
    _forward_only((x, gate_up, down, weights, base), ("x", "gate_up", "down", "weights", "base"))
    N = lead.numel()
    ldx = _even_rows(x)
    if ldx is None or ldx % 8 or x.data_ptr() % 16:
        x, ldx = x.clone(memory_format=torch.contiguous_format), H
    indices, weights = indices.contiguous(), weights.contiguous()
    ldb = 0
    if base is not None:
        if base.dtype is not bf16 or base.shape != x.shape:
            raise ValueError(f"base must be bf16 {list(x.shape)} (got {base.dtype} {list(base.shape)})")
        ldb = _even_rows(base)
        if ldb is None or ldb % 8 or base.data_ptr() % 16:
            if out is not None:
                _out_rows(out, x.shape, None, (base,), ("base",))
            base, ldb = base.clone(memory_format=torch.contiguous_format), H
    if out is None:
        out, ldo = torch.empty(x.shape, dtype=bf16, device=dev), H
    else:
        # (x is read before anything is written, so it may be the rows of the base that out is)
        place = [(t.data_ptr(), _even_rows(t)) for t in (out, x, base) if t is not None]
        in_place = len(place) == 3 and place[0] == place[1] == place[2]
        _out_rows(out, x.shape, base, (None if in_place else x, gate_up, down, indices, weights, workspace),
                  ("x", "gate_up", "down", "indices", "weights", "workspace"))
        ldo = _even_rows(out)
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    return _expert_mlp_call(dev, x, ldx, gate_up, down, indices, weights, base, ldb, out, ldo, workspace, N, H, I, E, k)


def _weight(*shape, device, dtype) -> torch.nn.Parameter:
    w = torch.empty(*shape, device=device, dtype=dtype)
    torch.nn.init.normal_(w, 0.0, shape[-1] ** -0.5)
    return torch.nn.Parameter(w, requires_grad=False)


class SparseMLP(torch.nn.Module):
    """The sparse MLP of mlx-lm's ``qwen3_5`` layers: ``num_experts`` SwiGLU experts, of
    which the router takes ``num_experts_per_tok`` per token, and a shared one
    whose result is multiplied by the sigmoid of its own gate.

    The router's and the shared gate's rows are one weight (``router``: E rows,
    then the shared gate's), so both come from one product.  With
    ``args.router_bias`` the choice goes by the scores plus ``router_bias``.  The
    logits are rounded to bf16, as mlx-lm's router's are (its scores, as these, are
    formed in a wider type from there on).
    """

    def __init__(self, args, device=None, dtype=torch.bfloat16):
        super().__init__()
        H, E, I, S = (args.hidden_size, args.num_experts, args.moe_intermediate_size,
                      args.shared_expert_intermediate_size)
        if not 0 < args.num_experts_per_tok <= E:
            raise ValueError(f"num_experts_per_tok must lie in [1, num_experts = {E}] (got {args.num_experts_per_tok})")
        if I <= 0 or S < 0:
            raise ValueError("moe_intermediate_size must be positive and shared_expert_intermediate_size not negative")
        self.args = args
        self.E = E
        self.router = _weight(E + (1 if S else 0), H, device=device, dtype=dtype)
        self.router_bias = (torch.nn.Parameter(torch.zeros(E, device=device), requires_grad=False)
                            if args.router_bias else None)
        self.gate_up_proj = _weight(E, 2 * I, H, device=device, dtype=dtype)
        self.down_proj = _weight(E, H, I, device=device, dtype=dtype)
        self.shared_gate_up_proj = _weight(2 * S, H, device=device, dtype=dtype) if S else None
        self.shared_down_proj = _weight(H, S, device=device, dtype=dtype) if S else None

    @torch.no_grad()
    def load(self, gate, gate_proj, up_proj, down_proj, shared_gate_proj=None, shared_up_proj=None,
             shared_down_proj=None, shared_expert_gate=None, router_bias=None) -> None:
        """gate ``[E, H]``; the experts' gate_proj and up_proj ``[E, I, H]`` and down_proj
        ``[E, H, I]``; the shared expert's ``[S, H]``, ``[S, H]``, ``[H, S]`` and its gate's
        ``[1, H]``."""
        shared = (shared_gate_proj, shared_up_proj, shared_down_proj, shared_expert_gate)
        if any((t is None) != (self.shared_down_proj is None) for t in shared):
            raise ValueError("the shared expert's weights go with shared_expert_intermediate_size > 0, all of them")
        if (router_bias is None) != (self.router_bias is None):
            raise ValueError("a router bias goes with args.router_bias")
        E, H, I = self.down_proj.shape
        S = 0 if self.shared_down_proj is None else self.shared_down_proj.shape[1]
        for name, t, shape in (("gate", gate, (E, H)), ("gate_proj", gate_proj, (E, I, H)), ("up_proj", up_proj, (E, I, H)),
                               ("down_proj", down_proj, (E, H, I)), ("shared_gate_proj", shared_gate_proj, (S, H)),
                               ("shared_up_proj", shared_up_proj, (S, H)), ("shared_down_proj", shared_down_proj, (H, S)),
                               ("shared_expert_gate", None if shared_expert_gate is None else
                                shared_expert_gate.reshape(1, -1), (1, H)), ("router_bias", router_bias, (E,))):
            if t is not None and tuple(t.shape) != shape:
                raise ValueError(f"{name} must be {list(shape)} (got {list(t.shape)})")
        self.router.copy_(gate if shared_expert_gate is None else torch.cat([gate, shared_expert_gate.view(1, -1)]))
        self.gate_up_proj.copy_(torch.cat([gate_proj, up_proj], 1))
        self.down_proj.copy_(down_proj)
        if self.shared_down_proj is not None:
            self.shared_gate_up_proj.copy_(torch.cat([shared_gate_proj, shared_up_proj]))
            self.shared_down_proj.copy_(shared_down_proj)
        if router_bias is not None:
            self.router_bias.copy_(router_bias)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                n_new: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The MLP of x ``[..., H]``, plus ``residual`` where given.  With x ``[B, T, H]``,
        ``n_new`` ``[B]`` int32: the experts pass over the tokens past it."""
        a, bias = self.args, self.router_bias
        if bias is not None and bias.dtype is not torch.float32:  # the module was cast
            bias = bias.float()
        both = linear_act(x, self.router)
        indices, weights = route_experts(both[..., : self.E], a.num_experts_per_tok, scoring=a.scoring_func,
                                         bias=bias, groups=a.n_group, top_groups=a.topk_group,
                                         group_best=a.group_best, renormalize=a.norm_topk_prob,
                                         scale=a.routed_scaling_factor, n_new=n_new)
        base = residual
        if self.shared_down_proj is not None:
            s = linear_act(x, self.shared_gate_up_proj, activation="swiglu")
            base = linear_act(s, self.shared_down_proj, row_gate=both[..., self.E], residual=residual)
        return expert_mlp(x, self.gate_up_proj, self.down_proj, indices, weights, base=base,
                          out=None if base is residual else base)
