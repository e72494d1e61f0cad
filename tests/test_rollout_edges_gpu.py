"""The rollout's calls (fp4_post_b200/rollout.py, Decoder.generate) where an answer is easily lost or spoilt: memory that has moved, calls that were refused, pages that are
absent, weights far below the largest, inference mode, configurations that change.  The plain sides are in 64 bits."""
import math

import pytest
import torch

import fp4_post_b200

fp4_post_b200.install_reference_aliases()

from fp4_post_b200 import rollout  # noqa: E402
from fp4_post_b200.decoder import Decoder, DecoderConfig  # noqa: E402

from test_rollout_gpu import check_attend, filled, gen, keys_values, new_cache, normal  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"
SMALL = DecoderConfig(hidden=256, layers=2, heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=1000)


@pytest.fixture(scope="module", autouse=True)
def _lib(built_library):
    return built_library


def decoder(cfg=SMALL, seed=0, dtype=torch.bfloat16, **kw):
    torch.manual_seed(seed)
    return Decoder(cfg, fuse_norms=False, **kw).to(DEV).to(dtype)


def prompts(B, T, cfg=SMALL, seed=1):
    return torch.randint(0, cfg.vocab, (B, T), device=DEV, generator=gen(seed))


# ---- memory that has moved --------------------------------------------------------------------------------------------

def test_a_cache_follows_its_tensors_memory():
    """Storage given back and taken again, or another tensor's put in its place, as a program does that has no use for the pool while it trains."""
    cache, twin = filled([40, 17], seed=40), filled([40, 17], seed=40)
    q, k, v = normal(2, 4, 64, seed=41), normal(2, 2, 64, seed=42), normal(2, 2, 64, seed=43)
    want = twin.attend(0, q)
    held = {n: getattr(cache, n).clone() for n in ("pool", "tables", "lengths", "refs")}
    decoys = []
    for name, copy in held.items():
        t = getattr(cache, name)
        size = t.untyped_storage().nbytes()
        t.untyped_storage().resize_(0)
        with pytest.raises(ValueError, match=name):
            cache.attend(0, q)
        with pytest.raises(ValueError, match=name):
            cache.reserve([0], 1)
        decoys.append(torch.full_like(copy, 3))              # (the allocator has the old memory at hand)
        t.untyped_storage().resize_(size)
        t.copy_(copy)
    assert torch.equal(cache.attend(0, q), want)
    for c in (cache, twin):
        c.append(0, None, k, v)
    assert torch.equal(cache.attend(0, q), twin.attend(0, q)) and all((d == 3).all() for d in decoys)
    old = cache.pool.clone()
    cache.pool.data = old
    cache.append(0, None, v, k)
    twin.append(0, None, v, k)
    assert torch.equal(cache.attend(0, q), twin.attend(0, q)) and cache.pool.data_ptr() == old.data_ptr()
    cache.check()


def test_a_cache_whose_tensors_have_become_others_is_refused():
    q = normal(2, 4, 64, seed=41)
    for name, other in (("pool", lambda t: t[:-1].clone()), ("pool", lambda t: t.float()), ("tables", lambda t: t[:, :-1].clone()), ("lengths", lambda t: t.long()), ("refs", lambda t: t.cpu()),
                        ("pool", lambda t: t.transpose(3, 4).contiguous().transpose(3, 4))):
        cache = filled([40, 17], seed=40)
        t = getattr(cache, name)
        t.data = other(t)
        for call in (lambda: cache.attend(0, q), lambda: cache.reserve([0], 1), lambda: cache.fork([0], [1]), lambda: cache.free(), lambda: cache.compact(),
                     lambda: cache.append(0, q, q[:, :2], q[:, :2])):
            with pytest.raises(ValueError, match=name):
                call()
    cache = filled([40, 17], seed=40, dtype=torch.float8_e4m3fn)
    cache.scales.untyped_storage().resize_(0)
    with pytest.raises(ValueError, match="scales"):
        cache.attend(0, q)


# ---- weights far below the largest ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("spread", [0.0, 0.5])
@pytest.mark.parametrize("n, low", [(65536, 26.0), (16384, 20.0), (3000, 12.0)])
def test_attend_keeps_what_lies_under_a_heavy_token(n, low, spread):
    """One token with nearly all of the weight and a value of zero, as a row's first one is in many models: the others' weights are 2^-low of its own, and the output is theirs
    alone.  All rows read the same pages, and there are as many of them as keep a row in one or two blocks.  8-bit pages: a weight goes into its product as fp16 of 2^11 times what it
    is to the largest at least: off by 2^-12 of itself, or where that is subnormal by 2^-25, 2^-36 of the largest."""
    rows, d = 512, 64
    pages = n // 16 + 1
    k, v = torch.zeros(n, d, device=DEV), 1.0 + 0.25 * torch.randn(n, d, device=DEV, generator=gen(50))
    k[:, 1:] = torch.randn(n, d - 1, device=DEV, generator=gen(51)) * spread
    k[0], v[0] = 0.0, 0.0
    k[0, 0] = 256.0
    pool = torch.zeros(pages, 1, 2, 1, 16, d, device=DEV)
    for i, t in enumerate((k, v)):
        pool[:, 0, i, 0] = torch.cat((t, torch.zeros(pages * 16 - n, d, device=DEV))).view(pages, 16, d)
    q = (torch.randn(rows, 1, d, device=DEV, generator=gen(52)) * 0.25).bfloat16()
    q[:, :, 0] = low * math.log(2.0) / 32.0
    slots = torch.zeros(rows, dtype=torch.int64, device=DEV)
    cache = rollout.PagedCache.of(pool.to(torch.float8_e4m3fn), torch.arange(pages, device=DEV, dtype=torch.int32)[None].contiguous(), torch.tensor([n], device=DEV, dtype=torch.int32),
                                  torch.ones(pages, device=DEV, dtype=torch.int32), scales=torch.ones(1, 2, 1, device=DEV))
    out, lse = cache.attend(0, q, slots, scale=0.125, return_lse=True)
    kv = keys_values(cache, 0, 0, n)[:, 0]
    x = q[:, 0].double() @ kv[0].t() * 0.125
    p = torch.softmax(x, dim=1)
    want, spread_v = p @ kv[1], p @ kv[1].abs()
    # (scores: fp32 sums of 64 products, queries to 2^-25 of their largest; see check_attend)
    e = 6 * 2.0 ** -22 * (q[:, 0].double().abs() @ kv[0].abs().t() * 0.125).amax(dim=1, keepdim=True) + 2.0 ** -20
    e = e + q[:, 0].double().abs().amax(dim=1, keepdim=True) * 2.0 ** -25 * kv[0].abs().sum(dim=1).max() * 0.125
    # A lane adds up to an eighth of a warp's fourth of a row's weights one after the other in fp32, each addition off by up to 2^-24 of the sum (behind the heavy one all that are below
    # 2^-24 of it leave it as it is); the tensor core 16 keys at a time, cut by 2^-22.
    summed = (n / 32 + 8) * 2.0 ** -24
    bound = 2.0 ** -8 * want.abs() + (2 * (e + 2.0 ** -12) + summed + (n / 64 + 8) * 2.0 ** -22) * spread_v + 2.0 ** -36 * p.amax(dim=1, keepdim=True) * kv[1].abs().sum(dim=0)
    off = (out[:, 0].double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())
    true_lse = torch.logsumexp(x, dim=1)
    assert ((lse[:, 0].double() - true_lse).abs() <= e[:, 0] + summed + 2.0 ** -22 * true_lse.abs() + 2.0 ** -20).all()


# ---- inference mode ---------------------------------------------------------------------------------------------------

def test_rotary_positions_made_in_inference_mode_train():
    with torch.inference_mode():
        r = rollout.Rotary(64)
        r(normal(3, 2, 64))
    x = normal(3, 2, 64).requires_grad_()
    (g,) = torch.autograd.grad(r(x).float().sum(), x)
    assert torch.equal(g, torch.autograd.grad(rollout.Rotary(64)(x).float().sum(), x)[0])


@pytest.mark.parametrize("graphed", [False, True])
def test_training_goes_on_behind_a_rollout_in_inference_mode(graphed):
    model, twin = decoder(fuse_rotary=True), decoder(fuse_rotary=True)
    ids = prompts(2, 24)
    with torch.inference_mode():
        tokens = model.generate(ids, max_new_tokens=5, answers=2, temperature=0.0, graphed=graphed)
    assert torch.equal(tokens, twin.generate(ids, max_new_tokens=5, answers=2, temperature=0.0))
    for m in (model, twin):
        m.loss(ids).backward()
    assert all(torch.equal(a.grad, b.grad) for a, b in zip(model.parameters(), twin.parameters()))


def test_a_cache_made_in_inference_mode_tells_its_reason_outside():
    with torch.inference_mode():
        cache = new_cache(pages=2)
    cache.reserve([0], 100)
    with pytest.raises(RuntimeError, match="not enough free pages"):
        cache.check()
    cache.check()
    with torch.inference_mode():
        cache.reserve([9], 1)
        with pytest.raises(RuntimeError, match="does not have"):
            cache.check()


# ---- configurations that change ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("change", [dict(rope_theta=1e4), dict(rope_scaling=dict(type="linear", factor=4.0)), dict(rotary_dim=32), dict(rope_interleaved=True)])
def test_fused_rotary_positions_follow_the_configuration(change):
    """As the tables do, which are made anew for each call."""
    import dataclasses
    model = decoder(dataclasses.replace(SMALL), fuse_rotary=True)
    ids = prompts(2, 40)
    model.generate(ids, max_new_tokens=2)
    for name, value in change.items():
        setattr(model.cfg, name, value)
    fresh = decoder(dataclasses.replace(SMALL, **change), fuse_rotary=True)
    with torch.no_grad():
        assert torch.equal(model(ids), fresh(ids))
    assert torch.equal(model.generate(ids, max_new_tokens=6, temperature=0.0), fresh.generate(ids, max_new_tokens=6, temperature=0.0))
    if "rope_scaling" in change:
        model.cfg.rope_scaling["factor"] = 8.0               # (changed in place)
        fresh = decoder(dataclasses.replace(SMALL, rope_scaling=dict(type="linear", factor=8.0)), fuse_rotary=True)
        with torch.no_grad():
            assert torch.equal(model(ids), fresh(ids))


# ---- the longest sequences ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_attend_at_the_longest_length(dtype):
    """2^31 - 16 tokens are what a table's 32-bit lengths end at; all pages but three are absent, so that no memory is asked for but the table's."""
    short = filled([43], seed=26, dtype=dtype)
    longest = 2 ** 31 - 16
    tables = torch.full((1, longest // 16), -1, dtype=torch.int32, device=DEV)
    for at, page in ((0, 0), (2 ** 26 + 5, 1), (longest // 16 - 1, 2)):
        tables[0, at] = short.tables[0, page]
    cache = rollout.PagedCache.of(short.pool, tables, torch.tensor([longest - 5], dtype=torch.int32, device=DEV), short.refs, scales=short.scales)
    q = normal(1, 4, 64, seed=27)
    out, lse = cache.attend(0, q, return_lse=True)
    check_attend(short, q, out, lse, [0])
