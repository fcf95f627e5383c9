"""Float64 CPU restatement of the sparse MLP's operators: routing to experts, the
experts' products, and dense products with an epilogue.

TEST INFRASTRUCTURE ONLY.  Only ``tests/`` may import this module.  The product
package ``multiplex_amd`` never imports it.

What it restates: mlx-lm's sparse block of the ``qwen3_5`` layers (softmax over all
experts, top-k, renormalised weights, SwiGLU experts, a shared expert times the
sigmoid of its gate) and the routing forms of other sparse models (sigmoid scores, a
bias for the choice alone, groups of experts).  ``tests/test_experts.py`` pins it
against closed forms and a loop over single tokens.
"""

from __future__ import annotations

import math

import numpy as np

_erf = np.vectorize(math.erf, otypes=[np.float64])


def sigmoid(x):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-np.asarray(x, np.float64)))


def silu(x):
    return x * sigmoid(x)


ACTIVATIONS = {
    None: lambda y: y,
    "relu": lambda y: np.where(y < 0, 0.0, y),
    "silu": silu,
    "gelu": lambda y: 0.5 * y * (1.0 + _erf(y / math.sqrt(2.0))) if y.size else y,
    "gelu_tanh": lambda y: 0.5 * y * (1.0 + np.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))),
}


def linear_act(x, w, bias=None, activation=None, row_gate=None, residual=None):
    y = x @ w.T
    if bias is not None:
        y = y + bias
    if activation == "swiglu":
        n = y.shape[-1] // 2
        y = silu(y[..., :n]) * y[..., n:]
    else:
        y = ACTIVATIONS[activation](y)
    if row_gate is not None:
        y = y * sigmoid(row_gate)[..., None]
    return y if residual is None else y + residual


def route(logits, k, scoring="softmax", bias=None, groups=1, top_groups=1, group_best=2, renormalize=True, scale=1.0):
    """logits [N, E] -> indices [N, k], weights [N, k]."""
    N, E = logits.shape
    indices, weights = np.zeros((N, k), np.int64), np.zeros((N, k))
    for n in range(N):
        l = np.asarray(logits[n], np.float64)
        if scoring == "softmax":
            top = np.max(np.where(np.isnan(l), -np.inf, l))
            with np.errstate(invalid="ignore"):
                z = np.exp(l - (0.0 if top == -np.inf else top))
            s = z / (z.sum() if z.sum() != 0 else 1.0)
        else:
            s = sigmoid(l)
        c = s if bias is None else s + bias
        # NaN below every number: compared by (is a number, value), the lowest index first
        key = [(0, 0.0) if np.isnan(v) else (1, v) for v in c]
        allowed = range(E)
        if top_groups < groups:
            width = E // groups
            of = []
            for g in range(groups):
                best = sorted((v for v in c[g * width:(g + 1) * width] if not np.isnan(v)), reverse=True)
                best = (best + [-np.inf] * group_best)[: min(group_best, width)]
                of.append(-np.inf if np.inf in best and -np.inf in best else sum(best))  # (a sum that is none)
            first = sorted(range(groups), key=lambda g: (-of[g], g))[:top_groups]
            allowed = [e for e in range(E) if e // width in first]
        order = sorted(allowed, key=lambda e: (-key[e][0], -key[e][1], e))[:k]
        w = s[order]
        if renormalize:
            w = w / w.sum() if w.sum() != 0 else np.zeros(k)
        indices[n], weights[n] = order, w * scale
    return indices, weights


def expert_mlp(x, gate_up, down, indices, weights, base=None):
    """x [N, H]; a choice outside [0, E) adds nothing."""
    E, _, I = down.shape
    out = np.zeros_like(x) if base is None else np.array(base, np.float64)
    for t in range(x.shape[0]):
        for e, w in zip(indices[t], weights[t]):
            if 0 <= e < E:
                h = gate_up[e] @ x[t]
                out[t] += w * (down[e] @ (silu(h[:I]) * h[I:]))
    return out
