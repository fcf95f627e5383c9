"""Decode-shape projections of the GatedDeltaNet mixer (``gdn_linear_decode``).

At decode a mixer layer's GEMMs have few rows (one token per batch row)
and are bound by reading their weights: in_proj's 12352 x 2048 and
out_proj's 2048 x 4096 bf16 matrices at hidden 2048 (``dflash.py:348-350,
377-378``).  ``gdn_linear_decode`` streams each weight once, split over
64-column tiles and 512-wide K slices, for 1..64 rows, and can fold the
epilogue's gated RMSNorm (``norm(out, z)``) into out_proj's operand load,
so the norm's output is never written.

Graph-replayed against the separate norm kernel plus hipBLASLt at hidden
2048, the fused norm + out_proj takes 7.4-8.1 us against 12.6-13.4 us up to
16 rows, and loses beyond (11.4 against 10.9 us at 32 rows, 16.4 against
13.1 us at 64).  So the mixer uses ``gated_norm_linear_decode`` up to
``FUSED_NORM_MAX_ROWS`` rows; ``linear_decode`` (the same call without the
norm) is the unfused reference for tests.  Up to 16 rows and above 2048
columns it runs ``gdn_linear_rows16``'s kernel, which leaves the workspace it
is given alone.

:func:`linear` is the layers' plain projection: a few rows by
``gdn_linear_rows16``, the library beyond.  :func:`linear_act` is a projection
with its epilogue (bias, activation, row gate, residual) in the product's own kernels.

The sliced kernel sums its K slices through a workspace of fp32 partials and one
ticket per output tile; the tickets must start at zero and every call
leaves them zero, so one zero-initialised workspace serves every call of a
module on one stream (calls that overlap, on several streams, need one
each).
"""

from __future__ import annotations

import functools
import sys
from typing import Optional

import torch
import torch.autograd.forward_ad as forward_ad

from . import _lib
from .gated_delta import _dtype_code, _ptr, _require_device, _stream

__all__ = ["linear", "linear_act", "linear_act_workspace_bytes", "DECODE_MAX_ROWS", "FUSED_NORM_MAX_ROWS", "DecodeWorkspace", "linear_decode",
           "gated_norm_linear_decode", "linear_decode_workspace_bytes", "decode_shape_ok"]

DECODE_MAX_ROWS = 64
FUSED_NORM_MAX_ROWS = 16  # where the fused norm + projection beats the norm kernel plus the library GEMM
_K_SLICE = 512
_MAX_COLUMNS = 262144  # gdn_linear_rows16's limit


def linear_decode_workspace_bytes(M: int, N: int, K: int) -> int:
    return int(_lib.load().gdn_linear_decode_workspace_bytes(M, N, K))


def decode_shape_ok(M: int, N: int, K: int) -> bool:
    """Shapes ``gdn_linear_decode`` takes: 1..64 rows, K a multiple of 512, N of 8."""
    return 1 <= M <= DECODE_MAX_ROWS and K >= _K_SLICE and K % _K_SLICE == 0 and N % 8 == 0 and N > 0


class DecodeWorkspace:
    """A zero-initialised device buffer, grown (and zeroed again) on demand.

    Growing allocates, so a call under HIP graph capture must find the
    buffer already large enough: run the step once eagerly first.
    """

    def __init__(self):
        self.buf: Optional[torch.Tensor] = None

    def get(self, nbytes: int, device: torch.device) -> torch.Tensor:
        if self.buf is None or self.buf.device != device or self.buf.numel() < nbytes:
            self.buf = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        return self.buf


def _rows(t: torch.Tensor, width: int, what: str) -> int:
    """Row stride (elements) of a ``[M, width]`` matrix with contiguous,
    16-byte aligned rows (e.g. a column slice of a wider buffer)."""
    if t.dim() != 2 or t.shape[1] != width or t.stride(1) != 1:
        raise ValueError(f"{what} must be [M, {width}] with contiguous rows")
    ld = t.stride(0) if t.shape[0] > 1 else width
    if ld < width or ld % 8 != 0 or t.data_ptr() % 16 != 0:
        raise ValueError(f"{what}: rows must be 16-byte aligned and a multiple of 8 elements apart")
    return int(ld)


def _launch(x, gate, norm_weight, eps, head_dim, weight, out, workspace):
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise ValueError("gdn_linear_decode takes bf16 activations and weights")
    M, K = x.shape
    N = weight.shape[0]
    if weight.dim() != 2 or weight.shape[1] != K or not weight.is_contiguous():
        raise ValueError(f"weight must be a contiguous [N, {K}] matrix")
    if not decode_shape_ok(M, N, K):
        raise ValueError(f"gdn_linear_decode takes 1..{DECODE_MAX_ROWS} rows, K a multiple of 512 and N of 8 "
                         f"(got M={M}, N={N}, K={K})")
    dev = _require_device([x, gate, norm_weight, weight, out], ["x", "gate", "norm_weight", "weight", "out"])
    ldx = _rows(x, K, "x")
    ldg = _rows(gate, K, "gate") if gate is not None else 0
    if out is None:
        out = torch.empty(M, N, dtype=torch.bfloat16, device=dev)
    ldo = _rows(out, N, "out")
    need = linear_decode_workspace_bytes(M, N, K)
    ws = (workspace if workspace is not None else DecodeWorkspace()).get(need, dev)
    nw_dt = _dtype_code(norm_weight, "norm_weight") if norm_weight is not None else 0
    _lib.call(dev, "gdn_linear_decode", _ptr(x), ldx, _ptr(gate), ldg, _ptr(norm_weight), nw_dt, float(eps),
              int(head_dim), _ptr(weight), _ptr(out), ldo, M, N, K, _ptr(ws), ws.numel(), _stream(dev))
    return out


def linear(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """``x @ weight.T`` (``torch.nn.functional.linear`` without a bias).

    A few rows of bf16 (:func:`_rows16_shape` has the sizes) by
    ``gdn_linear_rows16``; the library elsewhere, and where differentiation,
    autocast, a function transform or a tensor subclass needs its operator.
    The call costs the host 6.7 us, the library's 17.6.
    """
    N, K = weight.shape
    rows = x.numel() // K if K else 0
    if (_rows16_shape(rows, N, K) and x.dtype is torch.bfloat16 and weight.dtype is torch.bfloat16
            and x.is_cuda and weight.is_cuda and x.shape[-1] == K and not _needs_operator(x, weight)
            and x.is_contiguous() and weight.is_contiguous() and x.get_device() == weight.get_device()):
        xp, wp = x.data_ptr(), weight.data_ptr()
        if (xp | wp) % 16 == 0:
            return _rows16(x, xp, wp, rows, N, K)
    return torch.nn.functional.linear(x, weight)


_transform_level = getattr(torch._C._functorch, "maybe_current_level", None)
_dispatch_modes = getattr(torch._C, "_len_torch_dispatch_stack", None)


def _needs_operator(x, weight) -> bool:
    """Whether something follows or replaces the operator on these operands: a
    recorded gradient, a forward-mode tangent (its tensors are plain ones that
    ask for no gradient), a function transform (vmap, jvp, grad), a dispatch
    mode or a trace, autocast, a tensor subclass."""
    if (type(x) is not torch.Tensor or type(weight) not in (torch.Tensor, torch.nn.Parameter)
            or torch.is_autocast_enabled() or (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad))):
        return True
    if _transform_level is None or _transform_level() is not None:
        return True
    if _dispatch_modes is None or _dispatch_modes() or torch.jit.is_tracing():
        return True
    # (outside a dual level, -1, no tensor has a tangent)
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(
        forward_ad.unpack_dual(t).tangent is not None for t in (x, weight))


def _rows16_shape(rows, N, K) -> bool:
    """The sizes :func:`linear` gives to ``gdn_linear_rows16`` (which refuses
    more than ``_MAX_COLUMNS`` columns).

    The lines follow graph-replayed times with the weights read from memory,
    as those of a model's layers are (each call another of 600 MB of them);
    behind them, after the slash, calls of one weight that stays in the
    last-level cache, where the library gains more.  us, against the library's:
      K to 4096, 16 rows:  4096 x 4096 9.9 / 9.3, 14.7 / 11.6 (4 rows 8.0 / 7.3, 14.7 / 11.3);
        10240 x 4096 18.4 / 16.8, 25.0 / 19.6; 12352 x 2048 12.2 / 11.5, 15.1 / 10.8 (8 rows 11.4 / 10.7,
        15.1 / 10.8); 6144 x 4096 13.6 / 12.9, 14.4 / 11.3.  Of 120 sizes from 512 to 4096 by 2056 to 24576
        it is the slower one at 13, by 10% at most (K = 2560 and 3584 at 4608 to 8192 columns, 16384 columns);
        with the weight in the cache at 75, by 57% at most (K = 2560 at 4608 to 6144 columns)
      K to 8192, 4 rows:   4096 x 8192 15.5 / 12.4, 15.5 / 13.0; 12288 x 8192 35.3 / 29.6, 39.5 / 31.4
      K to 12288, 2 rows:  4096 x 12288 18.4 / 16.2, 21.0 / 17.0; 16384 x 12288 69.9 / 69.1, 82.4 / 86.4
      K over 4096 at 4104 to 8192 columns, where the busiest CU has two 16-column tiles and most have
        fewer, is the library's: 5120 x 5120 at 4 rows 14.5 / 13.0, 14.0 / 11.5; 6144 x 8192 23.2 / 19.3,
        21.4 / 17.9 (and, with two on every CU, 8192 x 8192 32.0 / 20.3, 28.9 / 21.7; 8192 x 6144, 21% faster
        than the library from memory, goes there with them)
    """
    if K <= 4096:
        most = 16
    elif 4096 < N <= 8192:
        most = 0
    else:
        most = 4 if K <= 8192 else 2
    return 1 <= rows <= most and 512 <= K <= 12288 and K % _K_SLICE == 0 and 2048 < N <= _MAX_COLUMNS and N % 8 == 0


def _rows16(x, x_addr, w_addr, rows, N, K):
    dev = x.device
    out = torch.empty(*x.shape[:-1], N, dtype=torch.bfloat16, device=dev)
    _lib.call(dev, "gdn_linear_rows16", x_addr, K, w_addr, out.data_ptr(), N, rows, N, K, _stream(dev))
    return out


def linear_decode(x: torch.Tensor, weight: torch.Tensor, *, out: Optional[torch.Tensor] = None,
                  workspace: Optional[DecodeWorkspace] = None) -> torch.Tensor:
    """``x @ weight.T`` for ``x [M <= 64, K]`` (rows may be a column slice)."""
    return _launch(x, None, None, 0.0, 0, weight, out, workspace)


def gated_norm_linear_decode(y: torch.Tensor, z: torch.Tensor, norm_weight: Optional[torch.Tensor], eps: float,
                             head_dim: int, weight: torch.Tensor, *, out: Optional[torch.Tensor] = None,
                             workspace: Optional[DecodeWorkspace] = None) -> torch.Tensor:
    """``gated_rms_norm(y, z, norm_weight, eps) @ weight.T`` per head of
    ``head_dim`` (64 or 128) columns, with the norm computed inside the
    projection's operand load (gdn_gated_rmsnorm's rounding points).
    y, z ``[M, K]``."""
    if z.dtype != torch.bfloat16:
        raise ValueError("z must be bf16")
    if norm_weight is not None:
        if tuple(norm_weight.shape) != (head_dim,):
            raise ValueError(f"norm_weight must be [{head_dim}]")
        norm_weight = norm_weight.contiguous()
    return _launch(y, z, norm_weight, eps, head_dim, weight, out, workspace)


# -------------------------------------------------- products with an epilogue

_FLOATS = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_ACTS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4, "swiglu": 5}


def _even_rows(t: torch.Tensor) -> Optional[int]:
    """Elements from a row of ``[..., D]`` to the next where the rows are contiguous
    and evenly spaced (a column slice of a wider buffer), else None."""
    D = t.shape[-1]
    if t.is_contiguous():
        return D
    if t.dim() == 3:  # the usual column slice of [B, T, width]
        (_, T, _), (b, ld, one) = t.shape, t.stride()
        if one == 1 and T > 1 and b == T * ld and ld >= D:
            return ld
    if t.stride(-1) != 1 and D != 1:
        return None
    ld, rows = 0, 1
    for n, step in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if n == 1:
            continue
        if rows == 1:
            ld = step
        elif step != rows * ld:
            return None
        rows *= n
    return (D if rows == 1 else ld) if rows == 1 or ld >= D else None


_jit_tracing = getattr(torch._C, "_is_tracing", torch.jit.is_tracing)


def _watched() -> bool:
    """Whether something may follow the call that these calls do not serve
    (:func:`_forward_only` looks closer): a trace, a dispatch mode, a forward-mode level."""
    return bool(_jit_tracing() or getattr(forward_ad, "_current_level", 0) >= 0 or _dispatch_modes is None
                or _dispatch_modes())


def _spacing(t: torch.Tensor) -> Optional[int]:
    """Elements from a value of ``[...]`` to the next where they are evenly spaced (0: one
    value for all), else None."""
    if t.dim() == 1:
        return t.stride(0)
    if t.is_contiguous():
        return 1
    step, values = 1, 1
    for n, s in zip(reversed(t.shape), reversed(t.stride())):
        if n == 1:
            continue
        if values == 1:
            step = s
        elif s != values * step:
            return None
        values *= n
    return step


def _forward_only(tensors, names) -> None:
    """These calls have no backward and are no operators of torch's: a gradient or a
    tangent asked for is an error, not lost, and so is a trace, which would hold the
    result as a constant."""
    if torch.is_grad_enabled():
        for t, n in zip(tensors, names):
            if t is not None and t.requires_grad:
                raise ValueError(f"{n} requires a gradient, which this call does not form (use torch.no_grad())")
    proxies = sys.modules.get("torch.fx.experimental.proxy_tensor")  # (there is no such trace before it is imported)
    if torch.jit.is_tracing() or proxies is not None and proxies.get_proxy_mode() is not None:
        raise ValueError("this call cannot be traced: the trace would hold its result as a constant")
    if getattr(forward_ad, "_current_level", 0) >= 0:  # (outside a dual level, -1, no tensor has a tangent)
        for t, n in zip(tensors, names):
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{n} has a forward-mode tangent, which this call does not carry on")


def _apart(out: torch.Tensor, others, names) -> None:
    """``out`` must not overlap what other workgroups still read."""
    lo, hi = _extent(out)
    for t, n in zip(others, names):
        if t is not None and t.numel():
            a, b = _extent(t)
            if a < hi and lo < b:
                raise ValueError(f"out overlaps {n}")


def _extent(t: torch.Tensor):
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()) if n > 1)
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _out_rows(out: torch.Tensor, shape, added: Optional[torch.Tensor], reads, names) -> None:
    """``out`` is of ``shape``, apart from ``reads`` (and of ``added``, which may be
    the same rows, since each is read by the thread that writes it)."""
    if out.dtype is not torch.bfloat16 or out.shape != shape or _even_rows(out) is None:
        raise ValueError(f"out must be bf16 rows of shape {list(shape)}, evenly spaced (got {out.dtype} {list(out.shape)})")
    _apart(out, reads, names)
    if added is not None and not (added.data_ptr() == out.data_ptr() and added.stride() == out.stride()):
        _apart(out, (added,), ("what is added to it",))


def linear_act(x: torch.Tensor, weight: torch.Tensor, *, bias: Optional[torch.Tensor] = None,
               activation: Optional[str] = None, row_gate: Optional[torch.Tensor] = None,
               residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) * sigmoid(row_gate) + residual`` (``gdn_linear_act``), in
    one launch or, where K is summed in slices, two, rounded once.

    x ``[..., K]`` and weight ``[N, K]`` bf16, K a multiple of 8; ``activation`` is
    None, "relu", "silu", "gelu" (erf), "gelu_tanh" or "swiglu" (``silu(gate) * up``:
    weight's and bias's first half are the gate's rows, N is half of theirs).
    bias ``[rows of weight]``, row_gate ``[...]`` (one logit per row of x, such as
    a column of another product) in bf16, fp16 or fp32; residual ``[..., N]`` bf16.
    x and residual may be column slices of wider buffers.  ``out`` may be the
    residual itself, and otherwise lies apart from all that is read (other columns
    of one buffer are refused too).  ``workspace``: bytes for the sums of K's slices, which some
    sizes of five rows or more are formed in (:func:`linear_act_workspace_bytes`;
    allocated when absent or too small); calls that overlap need one each.  There is no backward.
    """
    # a plain call's checks in a few operations; what is wrong, or laid out otherwise, is looked into below
    index, bf16, act = x.get_device(), torch.bfloat16, _ACTS.get(activation)
    if (index >= 0 and act is not None and x.dtype is bf16 and weight.dtype is bf16 and weight.dim() == 2 and x.dim() > 0
            and out is None and workspace is None and weight.get_device() == index
            and x.is_contiguous() and weight.is_contiguous() and not _watched()
            and not (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                                  or bias is not None and bias.requires_grad
                                                  or row_gate is not None and row_gate.requires_grad
                                                  or residual is not None and residual.requires_grad))):
        rows, K = weight.shape
        N = rows // 2 if act == 5 else rows
        lead, xp, wp = x.shape[:-1], x.data_ptr(), weight.data_ptr()
        shape = lead + (N,)
        bias_dt = gate_dt = 0
        if bias is not None:
            bias_dt = _FLOATS.get(bias.dtype, -1) if (bias.shape == (rows,) and bias.get_device() == index
                                                      and bias.is_contiguous()) else -1
        ldg = 0
        if row_gate is not None:
            ldg = _spacing(row_gate)
            gate_dt = _FLOATS.get(row_gate.dtype, -1) if (row_gate.shape == lead and row_gate.get_device() == index
                                                          and ldg is not None) else -1
        if (x.shape[-1] == K and K > 0 and K % 8 == 0 and N > 0 and (act != 5 or rows % 2 == 0) and (xp | wp) % 16 == 0
                and bias_dt >= 0 and gate_dt >= 0
                and (residual is None or residual.dtype is bf16 and residual.get_device() == index
                     and residual.shape == shape and residual.is_contiguous())):
            dev, M = x.device, x.numel() // K
            out = x.new_empty(shape)
            need = linear_act_workspace_bytes(M, N, K, activation)
            # (bound until the call returns: its memory may be another thread's as soon as the tensor is gone)
            ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
            _lib.call(dev, "gdn_linear_act", xp, K, wp, None if bias is None else bias.data_ptr(), bias_dt, act,
                      None if row_gate is None else row_gate.data_ptr(), gate_dt, ldg,
                      None if residual is None else residual.data_ptr(), N, out.data_ptr(), N, M, N, K,
                      None if ws is None else ws.data_ptr(), need, _stream(dev))
            return out
    return _linear_act_general(x, weight, bias, activation, row_gate, residual, out, workspace)


@functools.lru_cache(maxsize=4096)
def linear_act_workspace_bytes(rows: int, N: int, K: int, activation: Optional[str] = None) -> int:
    """Bytes that :func:`linear_act` needs as its workspace (0 for most sizes)."""
    return int(_lib.load().gdn_linear_act_workspace_bytes(rows, N, K, _ACTS[activation]))


def _linear_act_general(x, weight, bias, activation, row_gate, residual, out, workspace):
    """:func:`linear_act` of any layout; raises what is wrong with its arguments."""
    dev = _require_device((x, weight, bias, row_gate, residual, out, workspace),
                          ("x", "weight", "bias", "row_gate", "residual", "out", "workspace"))
    if activation not in _ACTS:
        raise ValueError(f"activation must be one of {[a for a in _ACTS]} (got {activation!r})")
    if x.dtype is not torch.bfloat16 or weight.dtype is not torch.bfloat16:
        raise ValueError(f"x and weight must be bfloat16 (got {x.dtype}, {weight.dtype})")
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"weight must be [N, {x.shape[-1] if x.dim() else 'K'}] (got {list(weight.shape)})")
    rows, K = weight.shape
    act = _ACTS[activation]
    if act == 5 and rows % 2:
        raise ValueError("swiglu needs the gate's rows and as many of up's")
    _forward_only((x, weight, bias, row_gate, residual), ("x", "weight", "bias", "row_gate", "residual"))
    N = rows // 2 if act == 5 else rows
    lead = x.shape[:-1]
    shape = (*lead, N)
    M = lead.numel()
    if K % 8 or K == 0 or N == 0:
        raise ValueError(f"K must be a positive multiple of 8 and N positive (got K={K}, N={N})")
    ldx = _even_rows(x)
    if ldx is None or ldx % 8 or x.data_ptr() % 16:
        x, ldx = x.clone(memory_format=torch.contiguous_format), K
    if not weight.is_contiguous() or weight.data_ptr() % 16:
        weight = weight.clone(memory_format=torch.contiguous_format)
    bias_dt = gate_dt = ldg = ldr = 0
    if bias is not None:
        if bias.shape != (rows,):
            raise ValueError(f"bias must be [{rows}] (got {list(bias.shape)})")
        bias, bias_dt = bias.contiguous(), _dtype_code(bias, "bias")
    if row_gate is not None:
        if row_gate.shape != lead:
            raise ValueError(f"row_gate must be {list(lead)}, one value per row of x (got {list(row_gate.shape)})")
        gate_dt = _dtype_code(row_gate, "row_gate")
        ldg = _spacing(row_gate)
        if ldg is None:
            row_gate, ldg = row_gate.contiguous(), 1
    if residual is not None:
        if residual.dtype is not torch.bfloat16 or residual.shape != shape:
            raise ValueError(f"residual must be bf16 {list(shape)} (got {residual.dtype} {list(residual.shape)})")
        ldr = _even_rows(residual)
        if ldr is None:
            if out is not None:
                _apart(out, (residual,), ("residual",))
            residual, ldr = residual.contiguous(), N
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=dev)
        ldo = N
    else:
        _out_rows(out, shape, residual, (x, weight, bias, row_gate, workspace),
                  ("x", "weight", "bias", "row_gate", "workspace"))
        ldo = _even_rows(out)
    need = linear_act_workspace_bytes(M, N, K, activation)
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _lib.call(dev, "gdn_linear_act", x.data_ptr(), ldx, weight.data_ptr(), _ptr(bias), bias_dt, act, _ptr(row_gate),
              gate_dt, ldg, _ptr(residual), ldr, out.data_ptr(), ldo, M, N, K, _ptr(workspace),
              0 if workspace is None else workspace.numel() * workspace.element_size(), _stream(dev))
    return out
