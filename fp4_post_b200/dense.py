"""The products of a model that stay in bf16, with what follows them in the same kernel and with gradients.

    linear                 act(x W^T + bias) * gate + residual: a projection that is not replaced by a Metis layer
    linear_cross_entropy   next-token loss of a head over the whole vocabulary, without its logits in memory
    token_logprobs         log-probabilities of given tokens under that head (and its entropy): what a policy-gradient step
                           takes of the policy and of its reference model

All three run on tcgen05 kernels of this library (csrc/dense_gemm.cu) and need CUDA tensors; nothing here computes on the CPU.
Operands are bfloat16, sums and softmax statistics fp32.  The inner size is a multiple of 8; rows may have any pitch that 16 bytes
divide (others are copied first).  A call runs on the current stream of its tensors' device and can be captured in a CUDA graph.
The reference leaves all of this to torch (nn.Linear, F.cross_entropy and TRL's selective log-softmax around src/grpo/grpo.py:199-215).
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import ops


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, gate, residual, activation):
        needs_x, needs_w, needs_b, needs_gate, _, _ = ctx.needs_input_grad
        keep_z = needs_gate or (activation is not None and (needs_x or needs_w or needs_b))
        out = ops.linear(x, weight, bias, activation=activation, gate=gate, residual=residual, return_preactivation=keep_z)
        y, z = out if keep_z else (out, None)
        ctx.activation = activation
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.save_for_backward(x if needs_w else None, weight if needs_x else None, gate if needs_x or needs_w or needs_b else None, z)
        ctx.x_shape, ctx.n = x.shape, weight.shape[0]
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, gate, z = ctx.saved_tensors
        needs_x, needs_w, needs_b, needs_gate, needs_residual, _ = ctx.needs_input_grad
        n, k = ctx.n, ctx.x_shape[-1]
        dy2 = dy.reshape(-1, n)
        rows = dy2.shape[0]
        dx = dw = db = dgate = None
        if rows == 0:
            dx = dy.new_zeros(ctx.x_shape) if needs_x else None
            dw = dy.new_zeros((n, k)) if needs_w else None
            db = dy.new_zeros(n, dtype=ctx.bias_dtype) if needs_b else None
            return dx, dw, db, dy if needs_gate else None, dy if needs_residual else None, None
        product = needs_x or needs_w
        gate2 = None if gate is None else gate.reshape(-1, n)
        # the gradient itself where nothing changes it and its rows can be read as they lie
        dz = dy2
        changed = product and (ctx.activation is not None or gate is not None or n % 8 != 0)
        if changed or needs_b or needs_gate:
            dz_new, dgate, db = ops.linear_pointwise(dy2, z, gate2, ctx.activation, want_dz=changed, want_dgate=needs_gate,
                                                     bias_dtype=ctx.bias_dtype if needs_b else None)
            dz = dz_new if changed else dz
        if needs_x:
            dx = ops.bf16_product(dz, weight).view(ctx.x_shape)
        if needs_w:
            dw = ops.bf16_product(dz, x.reshape(-1, k), a_mn_major=True)
        return dx, dw, db, None if dgate is None else dgate.view(dy.shape), dy if needs_residual else None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: Optional[str] = None,
           gate: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x @ weight.T + bias) * gate + residual, rounded to bf16 once.

    x [..., K], weight [N, K] (the layout of nn.Linear), bias [N] in bf16 or fp32; gate and residual are shaped like the output
    [..., N] (no broadcasting).  activation: None, "silu", "gelu" (erf form) or "gelu_tanh".  A SwiGLU block is
    linear(linear(h, w_gate, activation="silu", gate=linear(h, w_up)), w_down, residual=x).
    Differentiable once in all tensors; the backward pass keeps bf16(x @ weight.T + bias)."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, gate, residual)):
        return _Linear.apply(x, weight, bias, gate, residual, activation)
    return ops.linear(x, weight, bias, activation=activation, gate=gate, residual=residual)


class _HeadLoss(torch.autograd.Function):
    """form: "none" (a loss for each row), "sum", "mean", or "logprobs" (a log-probability for each row, and perhaps entropies)."""

    @staticmethod
    def forward(ctx, h, w, target, ignore_index, scale, form, entropy):
        ctx.set_materialize_grads(False)
        negate = form == "logprobs"
        nll, lse, ent = ops.head_loss(h, w, target, ignore_index=ignore_index, scale=scale, negate=negate, entropy=entropy)
        inv_count = None
        if form in ("sum", "mean"):
            nll, inv_count = ops.head_sum(nll, target, ignore_index=ignore_index, mean=form == "mean")
        ctx.save_for_backward(h, w, target, lse, inv_count)
        ctx.options = dict(ignore_index=ignore_index, scale=scale, negate=negate)
        if ent is not None:
            ctx.mark_non_differentiable(ent)
        return nll, ent

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _gent):
        if g is None:
            return None, None, None, None, None, None, None
        h, w, target, lse, inv_count = ctx.saved_tensors
        dh, dw = ops.head_backward(h, w, target, lse, g, inv_count=inv_count, want_dh=ctx.needs_input_grad[0],
                                   want_dw=ctx.needs_input_grad[1], **ctx.options)
        return dh, dw, None, None, None, None, None


def _head(hidden, weight, target, ignore_index, temperature, form, entropy):
    ops._need_cuda(hidden, "hidden")
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"shapes do not fit: hidden {tuple(hidden.shape)}, weight {tuple(weight.shape)}")
    if weight.shape[0] == 0 or weight.shape[1] == 0 or weight.shape[1] % 8 != 0:
        raise ValueError(f"weight {tuple(weight.shape)}: the inner size must be a positive multiple of 8")
    if target.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"targets must be int64 or int32, got {target.dtype}")
    if target.shape != hidden.shape[:-1]:
        raise ValueError(f"targets have shape {tuple(target.shape)}, hidden states {tuple(hidden.shape)}")
    temperature = float(temperature)
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"temperature must be positive and finite, not {temperature}")
    ops._same_device(hidden, weight=weight, target=target)
    for name, t in (("hidden", hidden), ("weight", weight)):
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    with ops._on_device(hidden.device):
        h, w = ops._operand_rows(hidden, "hidden"), ops._operand_rows(weight, "weight")
        t = target.reshape(-1).to(torch.int64).contiguous()
        if t.numel() == 0:
            # nothing to do, but the graph stays connected: the gradients are zeros
            rows = h.sum(dim=-1).float() * 0.0 + w.sum() * 0.0
            out = rows.sum() / (0.0 if form == "mean" else 1.0) if form in ("sum", "mean") else rows.view(target.shape)
            return out, rows.detach().view(target.shape)
        if torch.is_grad_enabled() and (h.requires_grad or w.requires_grad):
            out, ent = _HeadLoss.apply(h, w, t, int(ignore_index), 1.0 / temperature, form, entropy)
        else:
            negate = form == "logprobs"
            out, _, ent = ops.head_loss(h, w, t, ignore_index=int(ignore_index), scale=1.0 / temperature, negate=negate, entropy=entropy)
            if form in ("sum", "mean"):
                out = ops.head_sum(out, t, ignore_index=int(ignore_index), mean=form == "mean")[0]
    if out.dim() == 1:
        out = out.view(target.shape)
    return out, None if ent is None else ent.view(target.shape)


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean", temperature: float = 1.0) -> torch.Tensor:
    """F.cross_entropy(hidden @ weight.T / temperature, target, ignore_index=..., reduction=...) in fp32 without the logits.

    hidden [..., K] and weight [V, K] bf16, target [...] int64 or int32.  The logits are formed tile by tile in fp32 and folded
    into each row's maximum and sum; the backward pass forms them again, piece by piece of the vocabulary, and differentiates
    hidden and weight (once).  A target that is neither ignore_index nor in the vocabulary makes its loss NaN.  The mean over no
    row at all is NaN, as torch has it."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', not {reduction!r}")
    return _head(hidden, weight, target, ignore_index, temperature, reduction, False)[0]


def token_logprobs(hidden: torch.Tensor, weight: torch.Tensor, ids: torch.Tensor, *, temperature: float = 1.0, entropy: bool = False,
                   ignore_index: int = -100):
    """log softmax(hidden @ weight.T / temperature) at the given token ids, fp32, shaped like ids; 0 where ids is ignore_index.

    With entropy=True also the entropy of each row's distribution (ignored rows included), which carries no gradient."""
    out, ent = _head(hidden, weight, ids, ignore_index, temperature, "logprobs", entropy)
    return (out, ent) if entropy else out
