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

With `fuse_rotary=True` queries and keys are turned by one kernel of rollout.py, forward and backward, with angles in fp32 in place of bf16 tables.
`Decoder.generate` is the rollout: prompts are prefilled once, their pages forked for a group of answers each, and a decode step appends to
the paged cache, attends over it and samples on kernels of that module, eagerly or as one CUDA graph.
"""
from __future__ import annotations

import operator
from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn.functional as Fn
from torch import nn
from torch.autograd import forward_ad

from fp4_post_b200 import dense, ops, rollout
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
    rope_scaling: Optional[dict] = None      # see rollout.rotary_frequencies
    rotary_dim: Optional[int] = None         # elements of a head that turn (all)
    rope_interleaved: bool = False           # pairs of neighbours in place of halves

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


def _rope_part(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """The same where pairs are neighbours, or a part of the head turns: the tables' width."""
    front, rest = x[..., :cos.shape[-1]], x[..., cos.shape[-1]:]
    if interleaved:
        turned = torch.stack((-front[..., 1::2], front[..., ::2]), dim=-1).flatten(-2)
        front = front * cos + turned * sin
    else:
        front = _rope(front, cos, sin)
    return torch.cat((front, rest), dim=-1)


def _plain(*tensors, dtypes=(torch.bfloat16,)) -> bool:
    """Plain CUDA tensors of one device and type (bf16) that only autograd follows: the library's own calls may take them.  Whatever has to see the
    torch operations gets them: forward-mode derivatives (which no_grad leaves on), vmap and the other function transforms, tensor subclasses,
    dispatch modes, tracing."""
    first = tensors[0]
    return (not torch.jit.is_tracing() and not torch.compiler.is_compiling()
            and torch._C._functorch.peek_interpreter_stack() is None and torch._C._len_torch_dispatch_stack() == 0
            and first.dtype in dtypes
            and all(type(t) in (torch.Tensor, nn.Parameter) and t.is_cuda and t.dtype == first.dtype and t.device == first.device
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


def _rotary_tables(cfg: DecoderConfig, T: int, device, dtype):
    """cos and sin [1, 1, T, rotary_dim] of the configuration."""
    d = cfg.head_dim if cfg.rotary_dim is None else cfg.rotary_dim
    if cfg.rope_scaling is None:
        inv, magnitude = 1.0 / (cfg.rope_theta ** (torch.arange(0, d, 2, device=device, dtype=torch.float32) / d)), 1.0
    else:
        scaled, magnitude = rollout.rotary_frequencies(d, cfg.rope_theta, cfg.rope_scaling)
        inv = torch.tensor(scaled, device=device, dtype=torch.float32)
    ang = torch.outer(torch.arange(T, device=device, dtype=torch.float32), inv)
    ang = ang.repeat_interleave(2, dim=-1) if cfg.rope_interleaved else torch.cat((ang, ang), dim=-1)
    cos, sin = ang.cos(), ang.sin()
    if magnitude != 1.0:
        cos, sin = cos * magnitude, sin * magnitude
    return cos.to(dtype)[None, None], sin.to(dtype)[None, None]


class _Cached:
    """What a block's attention does in generate(), in the place of its tables: a layer of the cache, with the tokens' slots and positions.  A prompt's
    tokens attend to one another (and are put into the cache), a new token to its sequence in the cache."""

    def __init__(self, cache, layer, rotary, slots, positions, prompt):
        self.cache, self.layer, self.rotary, self.slots, self.positions, self.prompt = cache, layer, rotary, slots, positions, prompt

    def __call__(self, q, k, v):
        """q [B, T, heads, head_dim], k and v [B, T, kv_heads, head_dim] -> [B, T, heads * head_dim]"""
        B, T, H, D = q.shape
        if self.prompt:
            q, k = self.rotary(q, k)
            self.cache.append(self.layer, None, k.flatten(0, 1), v.flatten(0, 1), self.slots, self.positions)
            a = Fn.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), is_causal=True, enable_gqa=True)
            return a.transpose(1, 2).reshape(B, T, H * D)
        q = self.cache.append(self.layer, q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), self.slots, rotary=self.rotary)
        return self.cache.attend(self.layer, q, self.slots).view(B, T, H * D)


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
        v = v.view(B, T, c.kv_heads, c.head_dim)
        if isinstance(cos, _Cached):
            return _project(self.o_proj, cos(q, k, v), self.fuse_dense, residual=residual)
        v = v.transpose(1, 2)
        if isinstance(cos, rollout.Rotary):
            if _plain(q, k, dtypes=(torch.bfloat16, torch.float32)):
                q, k = (t.transpose(1, 2) for t in cos(q, k, sin))
                a = Fn.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True)
                return _project(self.o_proj, a.transpose(1, 2).reshape(B, T, c.heads * c.head_dim), self.fuse_dense, residual=residual)
            cos, sin = _rotary_tables(c, T, h.device, q.dtype)
        if c.rope_interleaved or c.rotary_dim not in (None, c.head_dim):
            q, k = _rope_part(q.transpose(1, 2), cos, sin, c.rope_interleaved), _rope_part(k.transpose(1, 2), cos, sin, c.rope_interleaved)
        elif c.head_dim % 8 == 0 and _table_of(cos, T, c.head_dim) and _table_of(sin, T, c.head_dim) and _native(q, k, cos, sin):
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
    def __init__(self, cfg: DecoderConfig, fuse_norms: bool = True, fuse_dense: bool = False, fuse_rotary: bool = False):
        super().__init__()
        self.cfg = cfg
        self.fuse_dense = fuse_dense
        self.fuse_rotary = fuse_rotary
        self._rotaries = {}              # by device and configuration: the frequencies, no parameter of the model
        self.embed_tokens = nn.Embedding(cfg.vocab, cfg.hidden)
        self.layers = nn.ModuleList(Block(cfg, fuse_norms, fuse_dense) for _ in range(cfg.layers))
        self.norm = RMSNorm(cfg.hidden, cfg.eps)
        self.lm_head = nn.Linear(cfg.hidden, cfg.vocab, bias=False)      # stays bf16: not in the reference's target list

    def rotary(self, T: int, device, dtype):
        return _rotary_tables(self.cfg, T, device, dtype)

    def _rotary_of(self, device: torch.device) -> rollout.Rotary:
        """The configuration's rotary positions on a device, made once for what the configuration is.  (All are kept: a captured graph reads its own.)"""
        c = self.cfg
        key = device, c.head_dim, c.rope_theta, c.rotary_dim, c.rope_interleaved, repr(c.rope_scaling)
        r = self._rotaries.get(key)
        if r is None:
            r = self._rotaries[key] = rollout.Rotary(c.head_dim, theta=c.rope_theta, rotary_dim=c.rotary_dim, interleaved=c.rope_interleaved, scaling=c.rope_scaling, device=device)
        return r

    def hidden(self, ids: torch.Tensor) -> torch.Tensor:
        """What the head reads: the normalised hidden states [B, T, hidden]."""
        x = self.embed_tokens(ids)
        if self.fuse_rotary and self.cfg.head_dim % 8 == 0 and self.cfg.head_dim <= 256 and _plain(x, dtypes=(torch.bfloat16, torch.float32)):
            cos, sin = self._rotary_of(x.device), None
        else:
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

    @torch.no_grad()
    def generate(self, ids: torch.Tensor, lengths=None, *, max_new_tokens: int, answers: int = 1, temperature=1.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0,
                 eos: Optional[int] = None, generator: Optional[torch.Generator] = None, logprobs: bool = False, page_size: int = 16,
                 cache_dtype: torch.dtype = torch.bfloat16, cache_scales: Optional[torch.Tensor] = None, graphed: bool = False):
        """`answers` sampled continuations of each prompt: tokens [B * answers, n <= max_new_tokens] (and their log-probabilities under the model at
        that temperature, float32), the answers of a prompt behind one another.

        ids [B, T] on the GPU, prompts padded behind their `lengths` with anything (None: all T).  A prompt is prefilled once and its pages are shared by its answers;
        keys and values are kept in bfloat16 or (cache_dtype) float8_e4m3fn, there as x / cache_scales (float32 [layers, 2, kv_heads], see rollout.PagedCache; ones
        where None), which saturates at 448.  The pool has pages for max_new_tokens of every answer from the start.  eos ends an answer: what follows it is eos again, with
        log-probability 0, and takes no more pages.  temperature, top_k, top_p, min_p: see rollout.sample; generator draws its random numbers.  graphed: the
        decode step is captured after its first run and replayed (weights and what layers cache of them must not change meanwhile, shapes are fixed).
        The model is bfloat16; rotary positions are formed in fp32, as fuse_rotary has them in forward()."""
        c = self.cfg
        if ids.dim() != 2 or ids.shape[0] == 0 or ids.shape[1] == 0:
            raise ValueError(f"ids must be [prompts, tokens], not {tuple(ids.shape)}")
        if not ids.is_cuda:
            raise RuntimeError("generate() runs on a paged cache on the GPU: there is no CPU fallback")
        if max_new_tokens < 1 or answers < 1:
            raise ValueError("max_new_tokens and answers must be positive")
        if page_size <= 0 or page_size % 16:
            raise ValueError(f"page_size must be a multiple of 16, not {page_size}")
        B, T = ids.shape
        lengths = [T] * B if lengths is None else [operator.index(n) for n in lengths]
        if len(lengths) != B or min(lengths) < 1 or max(lengths) > T:
            raise ValueError(f"lengths must be {B} numbers from 1 to {T}")
        dev, rows = ids.device, B * answers
        # a prompt's pages, and of each answer those behind the whole ones that it shares
        whole = [n // page_size for n in lengths]
        pages = sum(-(-n // page_size) for n in lengths) + answers * sum(-(-(n + max_new_tokens) // page_size) - w for n, w in zip(lengths, whole))
        cache = rollout.PagedCache(c.layers, c.kv_heads, c.head_dim, pages=pages, sequences=B + rows, max_length=T + max_new_tokens, page_size=page_size,
                                   dtype=cache_dtype, scales=cache_scales, device=dev)
        rotary = self._rotary_of(dev)
        count = torch.tensor(lengths, dtype=torch.int64, device=dev)
        prompts, slots = torch.arange(B, device=dev), torch.arange(B, B + rows, device=dev)

        def run(x, place):
            for i, blk in enumerate(self.layers):
                x = blk(x, place(i), None)
            return x

        def pick(x, u):
            logits = self.lm_head(self.norm(x))
            if logits.dtype not in (torch.bfloat16, torch.float32):
                logits = logits.float()
            return rollout.sample(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, logprobs=True)

        # prompts: what is behind one belongs to no sequence, and is no token of the vocabulary perhaps (an embedding reads where it says)
        cache.reserve(prompts, count)
        at = torch.arange(T, device=dev).expand(B, T)
        inside = at < count[:, None]
        owner = torch.where(inside, prompts[:, None], -1).reshape(-1)
        x = run(self.embed_tokens(torch.where(inside, ids, 0)), lambda i: _Cached(cache, i, rotary, owner, at.reshape(-1), True))
        last = x[prompts, count - 1]
        cache.fork(prompts.repeat_interleave(answers), slots)
        cache.free(prompts)
        draws = torch.rand(max_new_tokens, rows, dtype=torch.float32, device=dev, generator=generator)
        tokens = torch.empty(max_new_tokens, rows, dtype=torch.int64, device=dev)
        logp = torch.empty(max_new_tokens, rows, dtype=torch.float32, device=dev)
        token, p = pick(last.repeat_interleave(answers, dim=0), draws[0])
        tokens[0], logp[0] = token, p
        live = slots.clone()
        u = draws[0].clone()

        def step():
            if eos is not None:
                live.masked_fill_(token == eos, -1)
            cache.reserve(live, 1)
            x = run(self.embed_tokens(token.clamp(min=0))[:, None], lambda i: _Cached(cache, i, rotary, live, None, False))
            new, p = pick(x[:, 0], u)
            if eos is not None:
                done = live < 0
                new, p = new.masked_fill(done, eos), p.masked_fill(done, 0.0)
            token.copy_(new)
            return p

        graph, n = None, 1
        while n < max_new_tokens:
            u.copy_(draws[n])
            if graph is not None:
                graph.replay()
            elif graphed and n == 2:
                # (the first step has run as it is: what a capture must not do for the first time is done)
                from fp4_post_b200.graphs import _capture_stream
                torch.cuda.synchronize(dev)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.device(dev), torch.cuda.graph(graph, stream=_capture_stream()):
                    p = step()
                graph.replay()
            else:
                p = step()
            tokens[n], logp[n] = token, p
            n += 1
            if eos is not None and n % 32 == 0 and bool(((token == eos) | (live < 0)).all()):
                break
        cache.check()
        if graph is not None:
            torch.cuda.synchronize(dev)
            graph.reset()
        tokens, logp = tokens[:n].t().contiguous(), logp[:n].t().contiguous()
        return (tokens, logp) if logprobs else tokens
