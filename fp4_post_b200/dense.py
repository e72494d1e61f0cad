"""The products of a model that stay in bf16, with what follows them in the same kernel and with gradients.

    linear                 act(x W^T + bias) * gate + residual: a projection that is not replaced by a Metis layer
    linear_cross_entropy   next-token loss of a head over the whole vocabulary, without its logits in memory
    token_logprobs         log-probabilities of given tokens under that head (and its entropy): what a policy-gradient step
                           takes of the policy and of its reference model

All three run on tcgen05 kernels of this library (csrc/dense_gemm.cu, csrc/dense_small.cu for few tokens) and need CUDA tensors;
nothing here computes on the CPU.  Operands are bfloat16, sums and softmax statistics fp32.  The inner size is a multiple of 8; rows may
have any pitch that 16 bytes divide (others are copied first).  A call runs on the current stream of its tensors' device and can be
captured in a CUDA graph (a backward pass too, while no eager graph of the same leaves is kept: see graphs.py).  The calls and their
gradients are native (csrc/dense_host.cpp); what is here is what they refuse, and the copies of tensors that the kernels cannot read as
they lie.  They are no operations of torch: forward-mode derivatives, function transforms, traces and tensor subclasses that dispatch by
themselves are refused.

Every wait of the kernels is bounded; one that runs out (0.4 s: a GPU that another process holds) ends the kernel and leaves its outputs
as they are.  status, an int32 tensor of one element on the same device that holds 0, receives a positive METIS_DEV_* code then, from the
call or from its backward pass: read it where a step's results are read.
The reference leaves all of this to torch (nn.Linear, F.cross_entropy and TRL's selective log-softmax around src/grpo/grpo.py:199-215).
"""
from __future__ import annotations

from typing import Optional

import torch

from . import cabi

_ACTIVATIONS = {None: cabi.ACT_NONE, "silu": cabi.ACT_SILU, "gelu": cabi.ACT_GELU, "gelu_tanh": cabi.ACT_GELU_TANH}
_FORMS = {"none": 0, "sum": 1, "mean": 2}
_LOGPROBS = 3


def _check(t, what: str, device: Optional[torch.device] = None, dtypes=(torch.bfloat16,)) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor, not {type(t).__name__}")
    if device is None and not t.is_cuda:
        raise RuntimeError(f"{what} must be a CUDA tensor: the bf16 products have no CPU fallback")
    if device is not None and t.device != device:
        raise ValueError(f"{what} is on {t.device}, not on {device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{what} must be {' or '.join(str(d).removeprefix('torch.') for d in dtypes)}, got {t.dtype}")


def _check_product(x, weight, what: str) -> None:
    _check(x, what)
    _check(weight, "weight", x.device)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"shapes do not fit: {what} {tuple(x.shape)}, weight {tuple(weight.shape)}")
    if weight.shape[0] == 0 or weight.shape[1] == 0 or weight.shape[1] % 8 != 0:
        raise ValueError(f"weight {tuple(weight.shape)}: the inner size must be a positive multiple of 8")


def _check_status(status, device: torch.device) -> None:
    if status is not None:
        _check(status, "status", device, (torch.int32,))
        if status.numel() != 1:
            raise ValueError(f"status must have one element, not {status.numel()}")


def _readable(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """t with contiguous elements on an address that 16 bytes divide."""
    if t is None:
        return None
    t = t.resolve_neg().contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: Optional[str] = None,
           gate: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x @ weight.T + bias) * gate + residual, rounded to bf16 once.

    x [..., K], weight [N, K] (the layout of nn.Linear), bias [N] in bf16 or fp32; gate and residual are shaped like the output
    [..., N] (no broadcasting).  activation: None, "silu", "gelu" (erf form) or "gelu_tanh".  A SwiGLU block is
    linear(linear(h, w_gate, activation="silu", gate=linear(h, w_up)), w_down, residual=x).
    Differentiable once in all tensors.  Besides their own rounding the gradients have those of what they are made of: the activation's slopes
    in fp16 (2^-11), act(..) in bf16 for the gate's, and above 128 rows dz, the output's gradient taken through the epilogue, in bf16 (up to
    128 rows in two bf16 numbers): 2.4e-3 of a gradient's norm in place of 1.7e-3."""
    try:
        code = _ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be None, 'silu', 'gelu' or 'gelu_tanh', not {activation!r}") from None
    host = cabi.dense_host()
    out = host.linear(x, weight, bias, gate, residual, code, status)
    if out is not None:
        return out
    _check_product(x, weight, "x")
    if bias is not None:
        _check(bias, "bias", x.device, (torch.bfloat16, torch.float32))
        if bias.shape != weight.shape[:1]:
            raise ValueError(f"bias has shape {tuple(bias.shape)}, not ({weight.shape[0]},)")
    shape = (*x.shape[:-1], weight.shape[0])
    for name, t in (("gate", gate), ("residual", residual)):
        if t is not None:
            _check(t, name, x.device)
            if tuple(t.shape) != shape:
                raise ValueError(f"{name} has shape {tuple(t.shape)}, not that of the output, {shape}")
    _check_status(status, x.device)
    out = host.linear(*(_readable(t) for t in (x, weight, bias, gate, residual)), code, status)
    if out is None:
        raise RuntimeError("linear cannot read these tensors")
    return out


def _head(hidden, weight, target, ignore_index, temperature, form, entropy, status):
    scale = 1.0 / temperature if temperature else 0.0
    if not 2.0 ** -149 <= scale <= 2.0 ** 127:             # (the kernels have it, and 1.44 times it, in 32 bits)
        raise ValueError(f"temperature must be positive and finite, and so must 1 / temperature in 32 bits, not {temperature}")
    host = cabi.dense_host()
    out = host.head(hidden, weight, target, ignore_index, scale, form, entropy, status)
    if out is not None:
        return out
    _check_product(hidden, weight, "hidden")
    _check(target, "target", hidden.device, (torch.int64, torch.int32))
    if target.shape != hidden.shape[:-1]:
        raise ValueError(f"targets have shape {tuple(target.shape)}, hidden states {tuple(hidden.shape)}")
    _check_status(status, hidden.device)
    if target.numel() == 0:
        # nothing to do, but the graph stays connected: the gradients are zeros
        rows = hidden.sum(dim=-1, dtype=torch.float32) + (weight[:1].float() * 0.0).sum()
        out = rows if form in (_FORMS["none"], _LOGPROBS) else rows.sum() / (0.0 if form == _FORMS["mean"] else 1.0)
        return out, rows.detach()
    out = host.head(_readable(hidden), _readable(weight), target.to(torch.int64).contiguous(), ignore_index, scale, form, entropy, status)
    if out is None:
        raise RuntimeError("the head's losses cannot read these tensors")
    return out


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean", temperature: float = 1.0, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """F.cross_entropy(hidden @ weight.T / temperature, target, ignore_index=..., reduction=...) in fp32 without the logits.

    hidden [..., K] and weight [V, K] bf16, target [...] int64 or int32.  The logits are formed tile by tile in fp32 and folded
    into each row's maximum and sum; the backward pass forms them again, piece by piece of the vocabulary, and differentiates
    hidden and weight (once).  The gradients are rounded to bf16; so is, above 128 rows, the logits' gradient that they are made of (up to 128 in
    two bf16 numbers): 1.9e-3 to 2.4e-3 of their norm in place of 1.7e-3.  A row whose target is ignore_index adds nothing, whatever it holds.  A target that is neither
    ignore_index nor in the vocabulary makes its loss NaN.  The mean over no row at all is NaN, as torch has it."""
    try:
        form = _FORMS[reduction]
    except (KeyError, TypeError):
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', not {reduction!r}") from None
    return _head(hidden, weight, target, ignore_index, temperature, form, False, status)[0]


def token_logprobs(hidden: torch.Tensor, weight: torch.Tensor, ids: torch.Tensor, *, temperature: float = 1.0, entropy: bool = False,
                   ignore_index: int = -100, status: Optional[torch.Tensor] = None):
    """log softmax(hidden @ weight.T / temperature) at the given token ids, fp32, shaped like ids; 0 where ids is ignore_index.

    Never positive, and as exact for a token that the model is sure of (1 - p of 1e-6) as for any.  Gradients as those of linear_cross_entropy.
    With entropy=True also the entropy of each row's distribution (0 likewise), which carries no gradient."""
    out = _head(hidden, weight, ids, ignore_index, temperature, _LOGPROBS, entropy, status)
    return out if entropy else out[0]
