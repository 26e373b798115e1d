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
outputs and gradients are rounded once to their type. Pre-activations are kept for the backward pass
in fp32: a 16-bit copy would round every gradient a second time.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import kernels


def _flat(t: torch.Tensor | None, width: int) -> torch.Tensor | None:
    return t if t is None or t.dim() == 2 else t.reshape(math.prod(t.shape[:-1]), width)


def _wants_grad(*ts: torch.Tensor | None) -> bool:
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


def _check_width(what: str, x: torch.Tensor, width: int) -> None:
    if x.dim() < 1 or x.shape[-1] != width:
        raise ValueError(f"{what}: expected inputs of width {width}, got {tuple(x.shape)}")


# ─── linear ─────────────────────────────────────────────────────────────────────────────

class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2, w, b, res2, act):
        keep = act is not None and any(ctx.needs_input_grad[:3])
        x2, wk = kernels.matrix_operand(x2), kernels.matrix_operand(w)   # padded once for both passes
        y, z = kernels.linear(x2, wk, b, act, res2, keep_z=keep)
        ctx.act = act
        ctx.save_for_backward(x2, wk, z)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if dy.shape[0] == 0:
            dx = torch.zeros_like(x) if need_x else None
            dw = torch.zeros_like(w) if need_w else None
            db = w.new_zeros(w.shape[0]) if need_b else None
        elif need_x or need_w or need_b:
            dz, _, db, _ = kernels.act_grad(dy, z, None, ctx.act, bias_grad=need_b)
            if need_x or need_w:
                dz = kernels.matrix_operand(dz)
            if need_x:
                dx = kernels.linear_dx(dz, w)
            if need_w:
                dw, _ = kernels.linear_dw(dz, x)
        return dx, dw, db, dy if need_r else None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str | None = None,
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` for ``x`` [..., K], ``weight`` [N, K], ``bias`` [N] and
    ``residual`` [..., N]; ``activation`` is None, ``"relu"``, ``"silu"``, ``"gelu"`` (erf) or
    ``"gelu_tanh"``. One row up to many; all tensors bf16 or all fp16."""
    N, K = weight.shape
    _check_width("linear", x, K)
    if activation == "none":
        activation = None
    shape = (*x.shape[:-1], N)
    if residual is not None and residual.shape != shape:
        raise ValueError(f"linear: residual must have shape {shape}, got {tuple(residual.shape)}")
    x2, r2 = _flat(x, K), _flat(residual, N)
    if _wants_grad(x, weight, bias, residual):
        y = _Linear.apply(x2, weight, bias, r2, activation)
    else:
        y = kernels.linear(x2, weight, bias, activation, r2)[0]
    return y if x.dim() == 2 else y.view(shape)


# ─── gated linear ───────────────────────────────────────────────────────────────────────

class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2, wg, wu, bg, bu, act):
        x2, wgk, wuk = (kernels.matrix_operand(t) for t in (x2, wg, wu))
        h, zg, zu = kernels.gated_linear(x2, wgk, wuk, bg, bu, act, keep_z=True)
        ctx.act = act
        ctx.save_for_backward(x2, wgk, wuk, zg, zu)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, wg, wu, zg, zu = ctx.saved_tensors
        need_x, need_wg, need_wu, need_bg, need_bu = ctx.needs_input_grad[:5]
        if dh.shape[0] == 0:
            zero = [torch.zeros_like(t) if n else None for t, n in ((x, need_x), (wg, need_wg), (wu, need_wu))]
            return (*zero, *(wg.new_zeros(wg.shape[0]) if n else None for n in (need_bg, need_bu)), None)
        dg, du, dbg, dbu = kernels.act_grad(dh, zg, zu, ctx.act, bias_grad=need_bg or need_bu, bias_grad1=need_bu)
        dx = kernels.linear_dx(dg, wg, du, wu) if need_x else None
        dwg = dwu = None
        if need_wg and need_wu:
            dwg, dwu = kernels.linear_dw(dg, x, du)
        elif need_wg:
            dwg, _ = kernels.linear_dw(dg, x)
        elif need_wu:
            dwu, _ = kernels.linear_dw(du, x)
        return dx, dwg, dwu, dbg if need_bg else None, dbu, None


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: torch.Tensor | None = None,
                 b_up: torch.Tensor | None = None, *, activation: str | None = "silu") -> torch.Tensor:
    """``act(x @ w_gate.T + b_gate) * (x @ w_up.T + b_up)`` for ``x`` [..., K] and weights [N, K]: the
    first half of a gated feed-forward block (SwiGLU, GEGLU) without its two projections ever
    reaching memory. Types and activations as :func:`linear`."""
    N, K = w_gate.shape
    _check_width("gated_linear", x, K)
    if activation == "none":
        activation = None
    x2 = _flat(x, K)
    if _wants_grad(x, w_gate, w_up, b_gate, b_up):
        h = _GatedLinear.apply(x2, w_gate, w_up, b_gate, b_up, activation)
    else:
        h = kernels.gated_linear(x2, w_gate, w_up, b_gate, b_up, activation)[0]
    return h if x.dim() == 2 else h.view(*x.shape[:-1], N)


# ─── layer norm ─────────────────────────────────────────────────────────────────────────

class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2, w, b, eps):
        y, mean, rstd = kernels.layer_norm(x2, w, b, eps, keep_stats=True)
        ctx.kinds = (None if w is None else w.dtype, None if b is None else b.dtype)
        ctx.save_for_backward(x2, w, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, mean, rstd = ctx.saved_tensors
        _, need_w, need_b = ctx.needs_input_grad[:3]
        wk, bk = ctx.kinds
        if dy.shape[0] == 0:
            D = x.shape[1]
            return (torch.zeros_like(x), x.new_zeros(D, dtype=wk) if need_w else None,
                    x.new_zeros(D, dtype=bk) if need_b else None, None)
        # both sums in one type: fp32 when either vector is
        kind = torch.float32 if torch.float32 in (wk, bk) else x.dtype
        dx, dw, db = kernels.layer_norm_grad(dy, x, w, mean, rstd, need_w, need_b, kind)
        return dx, dw.to(wk) if need_w else None, db.to(bk) if need_b else None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension; ``weight`` and ``bias``
    [D] in x's type or fp32. bf16, fp16 or fp32."""
    _check_width("layer_norm", x, x.shape[-1] if x.dim() else 0)
    x2 = _flat(x, x.shape[-1])
    if _wants_grad(x, weight, bias):
        y = _LayerNorm.apply(x2, weight, bias, eps)
    else:
        y = kernels.layer_norm(x2, weight, bias, eps)[0]
    return y if x.dim() == 2 else y.view(x.shape)


# ─── embedding ──────────────────────────────────────────────────────────────────────────

class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, padding):
        ctx.save_for_backward(ids)
        ctx.args = (table.shape[0], scale, padding)
        return kernels.embedding(ids, table, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        ids, = ctx.saved_tensors
        return None, kernels.embedding_grad(dy, ids, *ctx.args), None, None


def embedding(ids: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0,
              padding_idx: int | None = None) -> torch.Tensor:
    """``scale * table[ids]`` for int64 or int32 ``ids`` of any shape and ``table`` [V, D]; the row of
    ``padding_idx`` gets no gradient. An id outside the table gives a zero row and sets the device
    error word (``_lib.device_error()`` returns 3); it never reads outside the table."""
    V, D = table.shape
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise ValueError(f"embedding: padding_idx {padding_idx} outside a table of {V} rows")
        padding_idx %= V
    flat = ids if ids.dim() == 1 else ids.reshape(-1)
    if _wants_grad(table):
        y = _Embedding.apply(flat, table, scale, -1 if padding_idx is None else padding_idx)
    else:
        y = kernels.embedding(flat, table, scale)
    return y if ids.dim() == 1 else y.view(*ids.shape, D)


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
