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
