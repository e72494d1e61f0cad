"""A Qwen2-style decoder in plain torch, the caller the Metis layers sit in during post-training.

The reference installs its layers into Hugging Face Qwen2 models (src/grpo/grpo.py:119-196:
`replace_linear_with_metis` swaps q/k/v/o/gate/up/down projections for BitLinear and lets q/k/v and
gate/up share one quantized activation).  This module is that model family restated with the same
sub-module names, so the same function installs the same layers, and nothing else: token embedding,
pre-norm blocks (RMSNorm -> GQA attention with rotary embeddings -> residual, RMSNorm -> SwiGLU ->
residual), final norm, untied bf16 lm_head.  Attention is torch's scaled_dot_product_attention.
It exists to measure the layer inside a whole training step (random weights, synthetic token ids); it
is not a model zoo.

With `fuse_norms=True` the two RMSNorms of a block hand their output to the projection group that
follows already quantized (RMSNorm.forward_quantized): one pass over the hidden state computes the
normalised tensor and its column mean, the next quantizes it for all projections of the group.

With `fuse_dense=True` what stays in bf16 runs on dense.py: the loss and `token_logprobs` take the head without its logits in
memory, and where o, gate and down are no Metis layers (target_modules of replace_linear_with_metis leaves them out) they have the
activation, the product with `up` and the residual in their own kernels.  q/k/v and up, which nothing follows, stay torch's.
A layer that has hooks is called like any module, and whatever has to see torch's operations gets them.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn.functional as Fn
from torch import nn
from torch.autograd import forward_ad

from fp4_post_b200 import dense, ops
from fp4_post_b200.Metis.Metis.bitlinear import forward_group
from fp4_post_b200.Metis.models.llama import RMSNorm


@dataclass
class DecoderConfig:
    hidden: int
    layers: int
    heads: int
    kv_heads: int
    head_dim: int
    ffn: int
    vocab: int
    rope_theta: float = 1e6
    eps: float = 1e-6
    qkv_bias: bool = True            # Qwen2: biases on q/k/v only

    def linear_flops_per_token(self, rank: int) -> int:
        """Algorithmic forward flops of the Metis projections per token: 2 N K + 2 r (K + N) each."""
        shapes = [(self.hidden, self.heads * self.head_dim), (self.hidden, self.kv_heads * self.head_dim),
                  (self.hidden, self.kv_heads * self.head_dim), (self.heads * self.head_dim, self.hidden),
                  (self.hidden, self.ffn), (self.hidden, self.ffn), (self.ffn, self.hidden)]
        return self.layers * sum(2 * n * k + 2 * rank * (k + n) for k, n in shapes)


QWEN2_1P5B = DecoderConfig(hidden=1536, layers=28, heads=12, kv_heads=2, head_dim=128, ffn=8960, vocab=151936)
QWEN2_7B = DecoderConfig(hidden=3584, layers=28, heads=28, kv_heads=4, head_dim=128, ffn=18944, vocab=152064)


def _rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x [B, H, T, D]; rotate-half convention."""
    x1, x2 = x[..., : x.shape[-1] // 2], x[..., x.shape[-1] // 2:]
    return x * cos + torch.cat((-x2, x1), dim=-1) * sin


def _plain(*tensors) -> bool:
    """Plain bf16 CUDA tensors of one device that only autograd follows: the library's own calls may take them.  Whatever has to see the
    torch operations gets them: forward-mode derivatives (which no_grad leaves on), vmap and the other function transforms, tensor subclasses,
    dispatch modes, tracing."""
    first = tensors[0]
    return (not torch.jit.is_tracing() and not torch.compiler.is_compiling()
            and torch._C._functorch.peek_interpreter_stack() is None and torch._C._len_torch_dispatch_stack() == 0
            and all(type(t) in (torch.Tensor, nn.Parameter) and t.is_cuda and t.dtype == torch.bfloat16 and t.device == first.device
                    and t.numel() > 0 and forward_ad.unpack_dual(t).tangent is None for t in tensors))


def _native(*tensors) -> bool:
    """Inference on such tensors: the elementwise pieces run as one launch each, with the same roundings."""
    return not torch.is_grad_enabled() and _plain(*tensors)


def _table_of(t: torch.Tensor, T: int, D: int) -> bool:
    """T rows of D elements, the same for every batch entry and head."""
    return t.dim() >= 2 and t.shape[-2:] == (T, D) and t.numel() == T * D


def _dense_weight(weight: torch.Tensor, *tensors) -> bool:
    """Whether dense.py takes this weight with these tensors: plain ones, an inner size that 8 divides."""
    return _plain(weight, *tensors) and weight.shape[1] % 8 == 0


def _bare(module: nn.Module, kind: type) -> bool:
    """Whether calling the module is no more than calling kind.forward: nothing derived, no hook of its own or of all modules, no forward put in
    its place."""
    g = nn.modules.module
    return (type(module) is kind and "forward" not in vars(module)
            and not any((module._forward_hooks, module._forward_pre_hooks, module._backward_hooks, module._backward_pre_hooks, g._global_forward_hooks,
                         g._global_forward_pre_hooks, g._global_backward_hooks, g._global_backward_pre_hooks)))


def _project(module: nn.Module, x: torch.Tensor, fuse: bool, *, activation=None, gate=None, residual=None):
    """activation(module(x)) * gate + residual, in one kernel where the module is a plain linear layer in bf16, its weight what its forward takes."""
    if fuse and _bare(module, nn.Linear) and _dense_weight(module.weight, x, *(t for t in (gate, residual, module.bias) if t is not None)):
        return dense.linear(x, module.weight, module.bias, activation=activation, gate=gate, residual=residual)
    y = module(x)
    if activation == "silu":
        y = Fn.silu(y)
    if gate is not None:
        y = y * gate
    return y if residual is None else residual + y


class Attention(nn.Module):
    def __init__(self, cfg: DecoderConfig, fuse_dense: bool = False):
        super().__init__()
        self.cfg = cfg
        self.fuse_dense = fuse_dense
        self.q_proj = nn.Linear(cfg.hidden, cfg.heads * cfg.head_dim, bias=cfg.qkv_bias)
        self.k_proj = nn.Linear(cfg.hidden, cfg.kv_heads * cfg.head_dim, bias=cfg.qkv_bias)
        self.v_proj = nn.Linear(cfg.hidden, cfg.kv_heads * cfg.head_dim, bias=cfg.qkv_bias)
        self.o_proj = nn.Linear(cfg.heads * cfg.head_dim, cfg.hidden, bias=False)

    def forward(self, h, cos, sin, residual=None):
        B, T, _ = h.shape
        c = self.cfg
        q, k, v = forward_group((self.q_proj, self.k_proj, self.v_proj), h)     # one shared activation, three branches
        q = q.view(B, T, c.heads, c.head_dim)
        k = k.view(B, T, c.kv_heads, c.head_dim)
        v = v.view(B, T, c.kv_heads, c.head_dim).transpose(1, 2)
        if c.head_dim % 8 == 0 and _table_of(cos, T, c.head_dim) and _table_of(sin, T, c.head_dim) and _native(q, k, cos, sin):
            q, k = (t.transpose(1, 2) for t in ops.rope_pair(q, k, cos, sin))
        else:
            q, k = _rope(q.transpose(1, 2), cos, sin), _rope(k.transpose(1, 2), cos, sin)
        a = Fn.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True)
        return _project(self.o_proj, a.transpose(1, 2).reshape(B, T, c.heads * c.head_dim), self.fuse_dense, residual=residual)


class MLP(nn.Module):
    def __init__(self, cfg: DecoderConfig, fuse_dense: bool = False):
        super().__init__()
        self.fuse_dense = fuse_dense
        self.gate_proj = nn.Linear(cfg.hidden, cfg.ffn, bias=False)
        self.up_proj = nn.Linear(cfg.hidden, cfg.ffn, bias=False)
        self.down_proj = nn.Linear(cfg.ffn, cfg.hidden, bias=False)

    def forward(self, h, residual=None):
        if self.fuse_dense and _bare(self.gate_proj, nn.Linear):
            act = _project(self.gate_proj, h, True, activation="silu", gate=self.up_proj(h))
        else:
            gate, up = forward_group((self.gate_proj, self.up_proj), h)
            if gate.shape == up.shape and gate.numel() % 8 == 0 and _native(gate, up):
                act = ops.silu_mul(gate, up)
            else:
                act = Fn.silu(gate) * up
        return _project(self.down_proj, act, self.fuse_dense, residual=residual)


class Block(nn.Module):
    def __init__(self, cfg: DecoderConfig, fuse_norms: bool, fuse_dense: bool = False):
        super().__init__()
        self.fuse_norms = fuse_norms
        self.fuse_dense = fuse_dense
        self.input_layernorm = RMSNorm(cfg.hidden, cfg.eps)
        self.self_attn = Attention(cfg, fuse_dense)
        self.post_attention_layernorm = RMSNorm(cfg.hidden, cfg.eps)
        self.mlp = MLP(cfg, fuse_dense)

    def _normed(self, norm, x, first_of_group):
        group = getattr(first_of_group, "activation_group", None)
        if self.fuse_norms and group is not None and x.is_cuda:
            return norm.forward_quantized(x, return_norm=True, activation_group=group)[1]
        return norm(x)

    def forward(self, x, cos, sin):
        # (the residual goes into a branch's last projection where nobody can see the branch by itself, or has put another module there)
        attn, mlp = self.self_attn, self.mlp
        h = self._normed(self.input_layernorm, x, attn.q_proj)
        x = attn(h, cos, sin, x) if self.fuse_dense and _bare(attn, Attention) else x + attn(h, cos, sin)
        h = self._normed(self.post_attention_layernorm, x, mlp.gate_proj)
        return mlp(h, x) if self.fuse_dense and _bare(mlp, MLP) else x + mlp(h)


class Decoder(nn.Module):
    def __init__(self, cfg: DecoderConfig, fuse_norms: bool = True, fuse_dense: bool = False):
        super().__init__()
        self.cfg = cfg
        self.fuse_dense = fuse_dense
        self.embed_tokens = nn.Embedding(cfg.vocab, cfg.hidden)
        self.layers = nn.ModuleList(Block(cfg, fuse_norms, fuse_dense) for _ in range(cfg.layers))
        self.norm = RMSNorm(cfg.hidden, cfg.eps)
        self.lm_head = nn.Linear(cfg.hidden, cfg.vocab, bias=False)      # stays bf16: not in the reference's target list

    def rotary(self, T: int, device, dtype):
        d = self.cfg.head_dim
        inv = 1.0 / (self.cfg.rope_theta ** (torch.arange(0, d, 2, device=device, dtype=torch.float32) / d))
        ang = torch.outer(torch.arange(T, device=device, dtype=torch.float32), inv)
        ang = torch.cat((ang, ang), dim=-1)
        return ang.cos().to(dtype)[None, None], ang.sin().to(dtype)[None, None]

    def hidden(self, ids: torch.Tensor) -> torch.Tensor:
        """What the head reads: the normalised hidden states [B, T, hidden]."""
        x = self.embed_tokens(ids)
        cos, sin = self.rotary(ids.shape[1], ids.device, x.dtype)
        for blk in self.layers:
            x = blk(x, cos, sin)
        return self.norm(x)

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return self.lm_head(self.hidden(ids))

    def _fused_head(self) -> bool:
        """Whether the head may be taken without its logits: they come from this class's forward, and from nothing put in its place."""
        return self.fuse_dense and type(self).forward is Decoder.forward and "forward" not in vars(self) and _bare(self.lm_head, nn.Linear)

    def loss(self, ids: torch.Tensor) -> torch.Tensor:
        """Next-token cross entropy on the given ids."""
        if self._fused_head():
            hidden = self.hidden(ids)
            if _dense_weight(self.lm_head.weight, hidden):
                target = Fn.pad(ids[:, 1:], (0, 1), value=-100)              # the last position of a row has no next token
                return dense.linear_cross_entropy(hidden, self.lm_head.weight, target)
            logits = self.lm_head(hidden)
        else:
            logits = self.forward(ids)
        return Fn.cross_entropy(logits[:, :-1].reshape(-1, logits.shape[-1]).float(), ids[:, 1:].reshape(-1))

    def token_logprobs(self, ids: torch.Tensor, temperature: float = 1.0, entropy: bool = False):
        """Log-probabilities of each row's tokens behind the first, fp32 [B, T - 1] (and the entropies of their distributions, without
        gradient): what a policy-gradient step takes of the policy and of its reference."""
        if self._fused_head():
            hidden = self.hidden(ids)
            if _dense_weight(self.lm_head.weight, hidden):
                target = Fn.pad(ids[:, 1:], (0, 1), value=-100)
                out = dense.token_logprobs(hidden, self.lm_head.weight, target, temperature=temperature, entropy=entropy)
                return (out[0][:, :-1], out[1][:, :-1]) if entropy else out[:, :-1]
            logits = self.lm_head(hidden)
        else:
            logits = self.forward(ids)
        logp = torch.log_softmax(logits[:, :-1].float() / temperature, dim=-1)
        picked = logp.gather(-1, ids[:, 1:, None])[..., 0]
        return (picked, -(logp.detach().exp() * logp.detach()).sum(dim=-1)) if entropy else picked
