"""Decoder.generate, and the fused rotary positions in the decoder's forward and backward pass, on the GPU."""
import math

import pytest
import torch

import fp4_post_b200

fp4_post_b200.install_reference_aliases()

from fp4_post_b200 import ops  # noqa: E402
from fp4_post_b200.decoder import Decoder, DecoderConfig  # noqa: E402
from fp4_post_b200.graphs import GraphedStep  # noqa: E402
from grpo.grpo import MetisArgs, replace_linear_with_metis  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"
SMALL = DecoderConfig(hidden=256, layers=2, heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=1000)
ODD = DecoderConfig(hidden=160, layers=2, heads=6, kv_heads=1, head_dim=40, ffn=320, vocab=97, rope_theta=1e4, rotary_dim=20, rope_interleaved=True,
                    rope_scaling=dict(type="llama3", factor=8.0, original_max_position=64))


@pytest.fixture(scope="module", autouse=True)
def _lib(built_library):
    return built_library


def decoder(cfg, seed=0, dtype=torch.bfloat16, **kw):
    torch.manual_seed(seed)
    model = Decoder(cfg, fuse_norms=False, **kw).to(DEV).to(dtype)
    with torch.no_grad():
        model.lm_head.weight.mul_(4.0)                       # (answers that are not all alike)
    return model


def prompts(cfg, B, T, seed=1):
    return torch.randint(0, cfg.vocab, (B, T), device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))


@pytest.mark.parametrize("cfg", [SMALL, ODD])
def test_fused_rotary_positions_in_forward_and_backward(cfg):
    """In fp32 the two differ by the angles' rounding (tables form them in fp32, position times frequency: 24 positions, 2^-19 at most)."""
    plain, fused = decoder(cfg, dtype=torch.float32), decoder(cfg, dtype=torch.float32, fuse_rotary=True)
    ids = prompts(cfg, 2, 24)
    before = ops.launch_count()
    a, b = plain.loss(ids), fused.loss(ids)
    a.backward()
    b.backward()
    assert ops.launch_count() - before == 2 * cfg.layers     # one kernel for queries and keys, forward and backward
    torch.testing.assert_close(b, a, rtol=1e-4, atol=1e-4)
    for (n, p), q in zip(plain.named_parameters(), fused.parameters()):
        torch.testing.assert_close(q.grad, p.grad, rtol=2e-3, atol=2e-4 * float(p.grad.abs().max()), msg=n)


def test_a_training_step_with_fused_rotary_replays_from_a_graph():
    model = decoder(SMALL, fuse_rotary=True)
    ids = prompts(SMALL, 2, 32)

    def step():
        for p in model.parameters():
            p.grad = None
        loss = model.loss(ids)
        loss.backward()
        return loss
    eager = float(step())
    graphed = GraphedStep(step, warmup=1)
    assert abs(float(graphed()) - eager) < 1e-3
    g = model.layers[0].self_attn.q_proj.weight.grad
    assert torch.isfinite(g).all() and g.abs().sum() > 0
    graphed.release()


def teacher(model, ids, n, tokens, temperature):
    """Log-probabilities of the tokens behind ids[:n], from one forward pass over all of them."""
    full = torch.cat((ids[:n], tokens))[None]
    logits = model(full).float()[0, n - 1:-1]
    return logits, torch.log_softmax(logits / (temperature or 1.0), dim=-1).gather(1, tokens[:, None])[:, 0]


# The two ways round differently: attention's result, 2^-9 of it on the average, and what the products make of other shapes. Through 2 layers and a head of some
# 10 roundings each, on logits of a few units: 20^(1/2) 2^-9 of their size is 0.03, and the largest of some hundred such differences 3 to 4 times as much.
CLOSE = {torch.bfloat16: 0.12, torch.float8_e4m3fn: 0.6}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("cfg, kw", [(SMALL, dict(temperature=0.0)), (SMALL, dict(temperature=0.8, top_k=50, top_p=0.9, answers=3)), (ODD, dict(temperature=1.0, answers=2, page_size=32)),
                                     (SMALL, dict(temperature=1.0, answers=5, graphed=True))])
def test_generated_tokens_are_what_a_forward_pass_gives(cfg, kw, dtype):
    model = decoder(cfg, fuse_rotary=True)
    ids, lengths, n = prompts(cfg, 3, 40), [40, 1, 33], 25
    gen = torch.Generator(device=DEV).manual_seed(3)
    tokens, logp = model.generate(ids, lengths, max_new_tokens=n, logprobs=True, generator=gen, cache_dtype=dtype, **kw)
    answers = kw.get("answers", 1)
    assert tokens.shape == (3 * answers, n) and logp.shape == tokens.shape and tokens.dtype == torch.int64
    with torch.no_grad():
        for i, t in enumerate(tokens):
            logits, want = teacher(model, ids[i // answers], lengths[i // answers], t, kw["temperature"])
            heat = kw["temperature"] or 1.0
            assert float((logp[i] - want).abs().max()) <= CLOSE[dtype] / min(heat, 1.0), (i, (logp[i] - want).abs().max())
            if kw["temperature"] == 0.0:
                assert float((logits.max(dim=1).values - logits.gather(1, t[:, None])[:, 0]).max()) <= 2 * CLOSE[dtype]
            if kw.get("top_k"):
                rank = (logits > logits.gather(1, t[:, None]) + 2 * CLOSE[dtype]).sum(dim=1)
                assert int(rank.max()) < kw["top_k"]
    if answers > 1:
        assert len({tuple(t) for t in tokens.tolist()}) == 3 * answers


def test_the_graph_gives_what_the_steps_give():
    model = decoder(SMALL)
    ids = prompts(SMALL, 2, 20)
    run = lambda graphed: model.generate(ids, [20, 7], max_new_tokens=40, answers=4, temperature=0.9, top_p=0.95, logprobs=True, graphed=graphed,  # noqa: E731
                                         generator=torch.Generator(device=DEV).manual_seed(5))
    (a, pa), (b, pb), (c, pc) = run(False), run(True), run(True)
    assert torch.equal(a, b) and torch.equal(pa, pb) and torch.equal(b, c) and torch.equal(pb, pc)


@pytest.mark.parametrize("graphed", [False, True])
def test_an_answer_ends_at_its_end_token(graphed):
    model = decoder(SMALL)
    ids = prompts(SMALL, 2, 10)
    gen = lambda: torch.Generator(device=DEV).manual_seed(6)  # noqa: E731
    free, fp = model.generate(ids, max_new_tokens=70, answers=3, temperature=1.0, generator=gen(), logprobs=True)
    eos = int(free[1, 4])
    tokens, logp = model.generate(ids, max_new_tokens=70, answers=3, temperature=1.0, generator=gen(), eos=eos, logprobs=True, graphed=graphed)
    ended = 0
    for i in range(6):
        row = free[i].tolist()
        stop = row.index(eos) + 1 if eos in row else 70
        ended += stop < 70
        stop = min(stop, tokens.shape[1])
        # (rows that have ended leave the others' attention where it was, but for how its keys are split)
        same = (free[i, :stop] == tokens[i, :stop]).int().cumprod(0).sum()
        assert int(same) == stop or stop > 20, (i, int(same), stop)
        if int(same) == stop and stop < tokens.shape[1]:
            assert (tokens[i, stop:] == eos).all() and (logp[i, stop:] == 0).all()
    assert ended >= 1
    first = int(free[0, 0])
    only = model.generate(ids[:1], max_new_tokens=70, temperature=1.0, generator=gen(), eos=first)
    assert only.shape[1] <= 70


def test_generate_one_token_and_refusals():
    model = decoder(SMALL)
    ids = prompts(SMALL, 2, 10)
    assert model.generate(ids, max_new_tokens=1, answers=2).shape == (4, 1)
    assert model.generate(ids, max_new_tokens=2, graphed=True).shape == (2, 2)
    for kw in (dict(max_new_tokens=0), dict(max_new_tokens=1, answers=0), dict(max_new_tokens=1, lengths=[1]), dict(max_new_tokens=1, lengths=[0, 3]), dict(max_new_tokens=1, lengths=[3, 11]),
               dict(max_new_tokens=1, page_size=10), dict(max_new_tokens=1, page_size=0), dict(max_new_tokens=1, top_p=2.0), dict(max_new_tokens=1, temperature=-1.0)):
        with pytest.raises(ValueError):
            model.generate(ids, kw.pop("lengths", None), **kw)
    with pytest.raises(TypeError):
        decoder(SMALL, dtype=torch.float32).generate(ids, max_new_tokens=2)


@pytest.mark.parametrize("fuse_norms", [False, True])
def test_metis_layers_generate(fuse_norms):
    torch.manual_seed(0)
    model = Decoder(SMALL, fuse_norms=fuse_norms, fuse_rotary=True).to(DEV).to(torch.bfloat16)
    args = MetisArgs(forward_svd_rank=32, activation_lowrank_svd=32, backward_lowrank_svd=32, cache_quantized_weight=True)
    args.device = DEV
    replace_linear_with_metis(model, dtype=torch.bfloat16, metis_args=args, compute_dtype=torch.bfloat16)
    ids = prompts(SMALL, 2, 16)
    for graphed in (False, True):
        tokens, logp = model.generate(ids, max_new_tokens=12, answers=8, temperature=1.0, logprobs=True, graphed=graphed)
        assert tokens.shape == (16, 12) and int(tokens.min()) >= 0 and int(tokens.max()) < SMALL.vocab
        assert torch.isfinite(logp).all() and float(logp.max()) <= 0.0 and float(logp.mean()) > -3 * math.log(SMALL.vocab)
