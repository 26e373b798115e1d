"""Text-side operators: what turns token ids into the context a DiT or UNet reads, and what training
such an encoder or prompt adapter needs. Four differentiable functions on hand-written sm_100a
kernels, and the modules built from them:

* :func:`embedding`: scaled token lookup; its gradient sums over tokens sorted by id;
* :func:`layer_norm`: forward and backward, with the reduction of the weight's gradient;
* :func:`linear`: ``act(x @ w.T + b) + residual`` in one tensor-core kernel;
* :func:`gated_linear`: ``act(x @ w_gate.T + b_gate) * (x @ w_up.T + b_up)`` in one kernel.

All take CUDA tensors with any leading dimensions and run on the current stream of the tensors'
device. The projections take bf16 and fp16, the norm and the embedding fp32 as well. Sums are fp32
(products, norm statistics, weight gradients) in a fixed order, so results repeat bit for bit;
outputs and gradients are rounded once to their type. Argument checks, allocation and the autograd
nodes are native (``_text_ext.so``). The gradients cannot be differentiated again, and there is no
forward-mode derivative: a dual tensor is refused. They are not traceable: ``torch.compile`` breaks the
graph at them, and function transforms (vmap, jvp) refuse them. Pre-activations are kept for the
backward pass in fp32: a 16-bit copy would round every gradient a second time. dz, the gradient before
the activation, is rounded to 16 bits for the two products that read it.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn

from . import _lib
from .kernels import act_code


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str | None = None,
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` for ``x`` [..., K], ``weight`` [N, K], ``bias`` [N] and
    ``residual`` [..., N]; ``activation`` is None, ``"relu"``, ``"silu"``, ``"gelu"`` (erf) or
    ``"gelu_tanh"``. One row up to many; all tensors bf16 or all fp16."""
    return _lib.text_ext().linear(x, weight, bias, act_code(activation), residual)


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: torch.Tensor | None = None,
                 b_up: torch.Tensor | None = None, *, activation: str | None = "silu") -> torch.Tensor:
    """``act(x @ w_gate.T + b_gate) * (x @ w_up.T + b_up)`` for ``x`` [..., K] and weights [N, K]: the
    first half of a gated feed-forward block (SwiGLU, GEGLU) without its two projections ever
    reaching memory. Types and activations as :func:`linear`."""
    return _lib.text_ext().gated_linear(x, w_gate, w_up, b_gate, b_up, act_code(activation))


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension; ``weight`` and ``bias``
    [D] in x's type or fp32. bf16, fp16 or fp32."""
    return _lib.text_ext().layer_norm(x, weight, bias, eps)


def embedding(ids: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0,
              padding_idx: int | None = None) -> torch.Tensor:
    """``scale * table[ids]`` for int64 or int32 ``ids`` of any shape and ``table`` [V, D]; the row of
    ``padding_idx`` gets no gradient. An id outside the table gives a zero row and sets the device
    error word, which ``diffucore_b200.device_error()`` returns as 3 (it waits for the device; call it
    where a step's results are read); it never reads outside the table."""
    return _lib.text_ext().embedding(ids, table, scale, padding_idx)


# ─── modules ────────────────────────────────────────────────────────────────────────────

class TokenEmbedding(nn.Module):
    """Token table with an output scale (``math.sqrt(dim)`` in models that scale their embeddings)."""

    def __init__(self, vocab: int, dim: int, scale: float = 1.0, padding_idx: int | None = None, device=None,
                 dtype=torch.bfloat16):
        super().__init__()
        self.scale, self.padding_idx = scale, padding_idx
        self.weight = nn.Parameter(torch.empty(vocab, dim, device=device, dtype=dtype))
        nn.init.normal_(self.weight, std=0.02)

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return embedding(ids, self.weight, scale=self.scale, padding_idx=self.padding_idx)


class LayerNorm(nn.Module):
    def __init__(self, dim: int, eps: float = 1e-5, bias: bool = True, device=None, dtype=torch.bfloat16):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(dim, device=device, dtype=dtype)) if bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, eps=self.eps)


class Linear(nn.Module):
    """``act(x @ weight.T + bias) + residual``; parameters named as ``nn.Linear``'s."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: str | None = None,
                 device=None, dtype=torch.bfloat16):
        super().__init__()
        self.activation = activation
        self.weight = nn.Parameter(torch.empty(out_features, in_features, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(out_features, device=device, dtype=dtype)) if bias else None
        nn.init.normal_(self.weight, std=1.0 / math.sqrt(in_features))

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        return linear(x, self.weight, self.bias, activation=self.activation, residual=residual)


class GatedFeedForward(nn.Module):
    """``down(act(gate(x)) * up(x)) + residual``: two launches forward."""

    def __init__(self, dim: int, hidden: int, activation: str = "silu", bias: bool = False, device=None,
                 dtype=torch.bfloat16):
        super().__init__()
        self.activation = activation
        kw = dict(bias=bias, device=device, dtype=dtype)
        self.gate = Linear(dim, hidden, **kw)
        self.up = Linear(dim, hidden, **kw)
        self.down = Linear(hidden, dim, **kw)

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        h = gated_linear(x, self.gate.weight, self.up.weight, self.gate.bias, self.up.bias, activation=self.activation)
        return self.down(h, residual)
