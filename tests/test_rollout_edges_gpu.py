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


# ---- calls behind one that was refused --------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_tokens_that_no_reserve_made_room_for_are_not_written(dtype):
    """A group of answers that runs out of pages: what its sequences hold, shared pages among it, stays; behind pages that were freed the step is made again."""
    cache = new_cache(pages=6, sequences=7, dtype=dtype)
    bits = torch.uint8 if dtype == torch.float8_e4m3fn else torch.int16
    k, v = normal(32, 2, 64, seed=60), normal(32, 2, 64, seed=61)
    cache.reserve([0, 6], [32, 20])
    cache.append(0, None, k, v, [0] * 32, list(range(32)))
    cache.append(0, None, k[:20], v[:20], [6] * 20, list(range(20)))
    cache.fork([0] * 4, [1, 2, 3, 4])
    cache.check()
    live = torch.tensor([1, 2, -1, 3, 4, 6], device=DEV)
    before = [t.clone() for t in (cache.pool.view(bits), cache.tables, cache.lengths, cache.refs)]
    q, nk, nv = normal(6, 4, 64, seed=62), normal(6, 2, 64, seed=63), normal(6, 2, 64, seed=64)
    r = rollout.Rotary(64)
    for _ in range(2):                                       # four pages are asked for, two are there
        cache.reserve(live, 1)
        out = cache.append(0, q, nk, nv, live, rotary=r)
        assert all(torch.equal(a, b) for a, b in zip(before, (cache.pool.view(bits), cache.tables, cache.lengths, cache.refs)))
        assert torch.equal(out[[0, 5]], r(q[[0, 5]], None, torch.tensor([31, 19], device=DEV))) and (out[2] == 0).all()
        with pytest.raises(RuntimeError, match="not enough free pages"):
            cache.check()
        cache.append(0, q, nk, nv, live, rotary=r)           # (the reason has been read: there is still no room)
        assert torch.equal(cache.pool.view(bits), before[0])
    # explicit positions are the caller's own
    cache.append(0, None, v[:1], k[:1], [6], [3])
    assert not torch.equal(cache.pool.view(bits), before[0])
    cache.append(0, None, k[3:4], v[3:4], [6], [3])
    assert torch.equal(cache.pool.view(bits), before[0])
    cache.free([6])
    cache.reserve(live[:5], 1)
    cache.append(0, q[:5], nk[:5], nv[:5], live[:5], rotary=r)
    cache.check()
    plain_k = r(nk, None, torch.full((6,), 32, device=DEV))
    for i, s in ((0, 1), (1, 2), (3, 3), (4, 4)):
        got = keys_values(cache, 0, s, 33)
        want = torch.stack((plain_k[i], nv[i])).to(dtype).double() if dtype == torch.bfloat16 else torch.stack((r(nk[i:i + 1].float(), None, torch.tensor([32], device=DEV))[0], nv[i].float())).to(dtype).double()
        assert torch.equal(got[:, :, 32], want) and torch.equal(got[0, :, :32], k.to(dtype).double().transpose(0, 1))


def test_what_one_refused_call_asked_for_keeps_no_other_sequence_from_its_tokens():
    cache = new_cache(pages=4, sequences=5)
    k = normal(2, 2, 64, seed=65)
    cache.reserve([0, 1], 16)
    cache.reserve([0], 100)                                  # refused
    cache.fork([0], [1])                                     # refused
    cache.reserve([1, 2], 1)
    cache.append(0, None, k, k, [1, 2])
    cache.append(0, None, k, k, [0, 3])                      # (no room for 0, nothing in 3)
    assert torch.equal(keys_values(cache, 0, 1, 17)[0][:, 16], k[0].double()) and torch.equal(keys_values(cache, 0, 2, 1)[1][:, 0], k[1].double())
    assert (keys_values(cache, 0, 0, 16) == 0).all()
    with pytest.raises(RuntimeError, match="not enough"):
        cache.check()
    # a sequence that is emptied and begun again has nothing left of it
    cache.free([0])
    cache.reserve([0], 1)
    cache.append(0, None, k[:1], k[:1], [0])
    assert torch.equal(keys_values(cache, 0, 0, 1)[0][:, 0], k[0].double())
    # refused for a sequence given twice, a slot that is none, a sequence too long: all that were named are held back, and others are not
    for slots, counts in (([0, 1, 1], 1), ([0, 9], 1), ([0, 1], [1, 200]), ([0, 1], [1, -1])):
        cache.reserve(slots, counts)
        before = cache.pool.clone()
        cache.append(0, None, k[1:], k[1:], [0])
        assert torch.equal(cache.pool, before)
        cache.append(0, None, k[:1], k[:1], [2])
        assert not torch.equal(cache.pool, before)
        cache.append(0, None, k[1:], k[1:], [2])
        cache.reserve([0, 1], 0)                             # (a call that goes through, for no more room)
        cache.append(0, None, k[1:], k[1:], [0])
        assert not torch.equal(cache.pool, before)
        cache.append(0, None, k[:1], k[:1], [0])
        assert torch.equal(cache.pool, before)
        with pytest.raises(RuntimeError):
            cache.check()


def test_a_captured_step_that_ran_out_of_pages_goes_on_when_there_are_some():
    cache, twin = (new_cache(pages=5, sequences=4) for _ in range(2))
    slots = torch.tensor([0, 1], device=DEV)
    q, k = normal(2, 4, 64, seed=66), normal(2, 2, 64, seed=67)
    for c in (cache, twin):
        c.reserve([0, 1, 2], [15, 16, 32])

    def step(c):
        c.reserve(slots, 1)
        return c.attend(0, c.append(0, q, k, k, slots), slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
    for i in range(20):
        k.copy_(normal(2, 2, 64, seed=70 + i))
        if i == 6:
            before = cache.pool.clone(), cache.lengths.clone()
            cache.reserve([3], 16)                           # the last page
            cache.lengths[0] = twin.lengths[0] = 16
            graph.replay()
            assert torch.equal(cache.pool, before[0]) and int(cache.lengths[1]) == int(before[1][1])
            with pytest.raises(RuntimeError, match="not enough"):
                cache.check()
            cache.free([3, 2])
            twin.free([2])
        graph.replay()
        assert torch.equal(step(twin), out) and torch.equal(cache.lengths, twin.lengths)
    cache.check()


def test_without_a_word_for_each_sequence_nothing_goes_to_an_end_while_there_is_a_status():
    """The entry points as a program in C has them."""
    import ctypes as C
    from fp4_post_b200 import cabi
    L, cache, k = cabi.lib(), new_cache(pages=2, sequences=2), normal(2, 2, 64, seed=68)
    pool, status = cache.pool, torch.zeros(1, dtype=torch.int32, device=DEV)
    c = cabi.CacheArgs(pool=pool.data_ptr(), pages=2, layers=1, kv_heads=2, page_size=16, head_dim=64, dtype=cabi.DTYPE_BF16, tables=cache.tables.data_ptr(), sequences=2, width=cache.tables.shape[1],
                       lengths=cache.lengths.data_ptr(), refs=cache.refs.data_ptr(), status=status.data_ptr())
    stream = torch.cuda.current_stream().cuda_stream
    ws = torch.empty(L.metis_cache_workspace_bytes(C.byref(c), 2), dtype=torch.uint8, device=DEV)
    reserve = lambda n: L.metis_cache_reserve(C.byref(c), None, None, n, 0, 2, ws.data_ptr(), ws.numel(), stream)  # noqa: E731
    a = cabi.AppendArgs(tokens=2, layer=0, heads_q=0, k=k.data_ptr(), v=k.data_ptr(), k_token=128, k_head=64, v_token=128, v_head=64, stream=stream)
    assert reserve(16) == 0 and reserve(1) == 0 and L.metis_cache_append(C.byref(c), C.byref(a)) == 0
    assert int(status) == 16 and cache.lengths.tolist() == [16, 16] and (pool == 0).all()
    status.zero_()
    assert L.metis_cache_append(C.byref(c), C.byref(a)) == 0
    assert torch.equal(pool[:, 0, 0, :, 15], k) and int((pool != 0).any(dim=-1).sum()) == 8


# ---- pages that are absent ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("lengths", [[40, 33], [20000, 33], [700] * 300])
@pytest.mark.parametrize("heads, head_dim", [(4, 64), (40, 128)])
def test_a_row_whose_pages_are_all_absent_is_one_without_keys(lengths, dtype, heads, head_dim):
    """In one block, and split over several: zeros, and a logarithm of -inf.  Rows beside it stay."""
    cache = filled(lengths, head_dim=head_dim, dtype=dtype, seed=21)
    q = normal(len(lengths), heads, head_dim, seed=22)
    want, want_lse = cache.attend(0, q, return_lse=True)
    cache.tables[0] = torch.tensor([-1, cache.pool.shape[0], 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=DEV).repeat(cache.tables.shape[1])[:cache.tables.shape[1]]
    out, lse = cache.attend(0, q, return_lse=True)
    assert (out[0] == 0).all() and (lse[0] == -math.inf).all()
    assert torch.equal(out[1:], want[1:]) and torch.equal(lse[1:], want_lse[1:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_a_row_with_one_page_among_absent_ones_is_that_page(dtype):
    cache = filled([20000, 16, 33], seed=23, dtype=dtype)
    q = normal(3, 4, 64, seed=24)
    for at in (0, 700, 1249):
        cache.tables[0] = -1
        cache.tables[0, at] = cache.tables[1, 0]
        out, lse = cache.attend(0, q[[1, 1]], [0, 1], return_lse=True)
        check_attend(cache, q[1:2], out[1:], lse[1:], [1])
        check_attend(cache, q[1:2], out[:1], lse[:1], [1])


def test_a_free_that_names_a_sequence_that_is_none_does_nothing():
    cache = new_cache()
    cache.reserve([0, 2, 5], [20, 3, 100])
    before = [t.clone() for t in (cache.tables, cache.lengths, cache.refs)]
    for slots in ([0, 17], [6, 2], [0, 2, -1, 5, 1 << 40], [0] * 3000 + [6], torch.tensor([5, 2 ** 31 - 1], dtype=torch.int32, device=DEV)):
        cache.free(slots)
        assert all(torch.equal(a, b) for a, b in zip(before, (cache.tables, cache.lengths, cache.refs)))
        with pytest.raises(RuntimeError, match="does not have"):
            cache.check()
    cache.free([0, -1, 0, 5] * 2000)
    cache.check()
    assert cache.lengths.tolist() == [0, 0, 3, 0, 0, 0] and cache.free_pages() == 39


# ---- rotary positions' own precision --------------------------------------------------------------------------------------

@pytest.mark.parametrize("interleaved", [False, True])
def test_cosines_and_sines_are_as_exact_as_fp32_has_them(interleaved):
    """Of pairs (1, 0) the results are the cosine and the sine themselves.  The angle, less whole quarter turns, is phi in [-pi/4, pi/4]: cut off below 2^-34 of a turn and rounded to fp32,
    it is off by 2^-24 |phi| + 2^-31; sincospif by a step, 2^-23 of its result."""
    n = 16
    r = rollout.Rotary(n, theta=500.0, interleaved=interleaved)
    x = torch.zeros(40000, 1, n, device=DEV)
    first, second = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    x[..., first] = 1.0
    positions = torch.cat((torch.arange(30000, device=DEV), torch.randint(-2 ** 40, 2 ** 40, (10000,), device=DEV, generator=gen(80))))
    y = r(x, None, positions)[:, 0].double()
    turn = torch.tensor([[(p * b) % 2 ** 64 / 2 ** 64 for b in r.turns.tolist()] for p in positions.tolist()], dtype=torch.float64, device=DEV)
    c, s = torch.cos(2 * math.pi * turn), torch.sin(2 * math.pi * turn)
    phi = 2 * math.pi * (turn - torch.round(turn * 4) / 4).abs()
    off = 2.0 ** -24 * phi + 2.0 ** -31
    for got, value, other in ((y[:, first], c, s), (y[:, second], s, c)):
        bound = 2.0 ** -23 * value.abs() + off * (other.abs() + off) + 2.0 ** -50
        assert ((got - value).abs() <= bound).all(), float(((got - value).abs() / bound).max())


# ---- sampling on the borders between two tokens -------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [512, 3000])
def test_sample_takes_a_kept_token_at_every_border(vocab, dtype):
    """Random numbers on the borders between two tokens and a few steps of 64 bits beside them, half of the vocabulary masked: whatever the sums' roundings are, the token is one that is
    kept, and no farther from the border than the sums' own error."""
    for seed in range(12):
        x = (torch.rand(vocab, device=DEV, generator=gen(seed)) * -30).to(dtype)
        x[torch.rand(vocab, device=DEV, generator=gen(100 + seed)) < 0.5] = -math.inf
        x[(seed * 97) % vocab] = 0.0
        w = x.float().exp().double()
        sums = w.cumsum(0)
        u = (sums / sums[-1])[w > 0][:-1][:500]
        u = torch.cat([u + k * 2.0 ** -54 for k in range(-3, 4)] + [torch.tensor([1 - 2.0 ** -53], device=DEV, dtype=torch.float64)])
        u = u[(u >= 0) & (u < 1)].contiguous()
        for kw in (dict(), dict(top_p=1 - 2.0 ** -53), dict(top_k=vocab - 1)):
            token = rollout.sample(x.expand(u.numel(), vocab), u, **kw)
            assert int(token.min()) >= 0 and int(token.max()) < vocab and (w[token] > 0).all(), (seed, kw)
            mark, slack = u * sums[-1], float(sums[-1]) * 2.0 ** -44
            assert ((sums - w)[token] <= mark + slack).all() and (sums[token] >= mark - slack).all(), (seed, kw)


# ---- what calls take ------------------------------------------------------------------------------------------------------

def test_prompts_are_padded_with_anything():
    """Behind a prompt's length ids are not read: -100, or any other number that is no token, is as good as one."""
    model = decoder()
    ids = prompts(3, 20)
    lengths = [20, 1, 7]
    run = lambda x: model.generate(x, lengths, max_new_tokens=6, temperature=0.0, logprobs=True)  # noqa: E731
    want, want_p = run(torch.where(torch.arange(20, device=DEV) < torch.tensor(lengths, device=DEV)[:, None], ids, 0))
    behind = torch.arange(20, device=DEV)[None] >= torch.tensor(lengths, device=DEV)[:, None]
    for pad in (-100, -1, SMALL.vocab, 2 ** 40):
        got, got_p = run(ids.masked_fill(behind, pad))
        assert torch.equal(got, want) and torch.equal(got_p, want_p)


def test_slots_counts_and_positions_are_whole_numbers():
    cache = new_cache()
    cache.reserve([0], 20)
    k = normal(1, 2, 64)
    for call in (lambda: cache.reserve([0.5], 1), lambda: cache.reserve([1.0], 1), lambda: cache.reserve([0], [1.5]), lambda: cache.reserve([0], 1.5), lambda: cache.free([0.0]), lambda: cache.fork([0.2], [1]),
                 lambda: cache.fork([0], [1.7]), lambda: cache.append(0, None, k, k, [0.3]), lambda: cache.append(0, None, k, k, [0], [2.5]), lambda: cache.attend(0, k, [0.9]),
                 lambda: cache.reserve(["0"], 1), lambda: cache.reserve([None], 1)):
        with pytest.raises(TypeError):
            call()
    assert cache.lengths.tolist() == [20, 0, 0, 0, 0, 0]
    cache.reserve((i for i in (1, 2)), iter([3, 4]))
    cache.reserve(range(3, 5), [True, 2])
    assert cache.lengths.tolist() == [20, 3, 4, 1, 2, 0]
    with pytest.raises((ValueError, OverflowError, RuntimeError)):
        cache.reserve([2 ** 70], 1)
    cache.check()
    model, ids = decoder(), prompts(2, 8)
    for lengths in ([3, 2.5], torch.tensor([3.0, 2.0]), ["3", "2"]):
        with pytest.raises(TypeError):
            model.generate(ids, lengths, max_new_tokens=1)
    want = model.generate(ids, [3, 2], max_new_tokens=3, temperature=0.0)
    for lengths in (torch.tensor([3, 2]), torch.tensor([3, 2], device=DEV, dtype=torch.int32)):
        assert torch.equal(model.generate(ids, lengths, max_new_tokens=3, temperature=0.0), want)


def test_gradients_that_no_call_forms_are_refused_for_every_argument():
    x, u = normal(2, 50, dtype=torch.float32), torch.full((2,), 0.5, device=DEV)
    for kw in (dict(temperature=torch.ones(2, device=DEV)), dict(top_p=torch.full((2,), 0.5, device=DEV)), dict(min_p=torch.zeros(2, device=DEV))):
        (name, t), = kw.items()
        t.requires_grad_()
        with pytest.raises(RuntimeError, match=f"{name} requires a gradient"):
            rollout.sample(x, u, logprobs=True, **kw)
        with torch.no_grad():
            rollout.sample(x, u, logprobs=True, **kw)
    with pytest.raises(RuntimeError, match="u requires a gradient"):
        rollout.sample(x, u.clone().requires_grad_())
    q = normal(2, 4, 64)
    for name, dtype in (("pool", torch.bfloat16), ("scales", torch.float8_e4m3fn)):
        cache = filled([20, 5], seed=90, dtype=dtype)
        want = cache.attend(0, q)
        getattr(cache, name).requires_grad_()
        for call in (lambda: cache.attend(0, q), lambda: cache.append(0, q, q[:, :2], q[:, :2])):
            with pytest.raises(RuntimeError, match=f"{name} requires a gradient"):
                call()
        with torch.no_grad():
            assert torch.equal(cache.attend(0, q), want)


def test_frequencies_that_do_not_fit_are_refused():
    """Rotary's attributes are plain ones."""
    q, cache = normal(2, 4, 64), new_cache()
    cache.reserve(None, 3)
    for name, value in (("rotary_dim", 128), ("rotary_dim", 32), ("turns", lambda t: t[:-1]), ("turns", lambda t: t.float()), ("turns", lambda t: t.repeat_interleave(2)[::2]), ("turns", lambda t: t.cpu()),
                        ("rotary_dim", 0), ("rotary_dim", -64)):
        r = rollout.Rotary(64)
        setattr(r, name, value(r.turns) if callable(value) else value)
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            r(q)
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            cache.append(0, q, q[:, :2], q[:, :2], [0, 1], rotary=r)


def test_generate_takes_the_scales_of_an_8_bit_cache():
    """Keys of 2000 and more saturate at 448 unless they are scaled."""
    model = decoder()
    with torch.no_grad():
        for blk in model.layers:
            blk.self_attn.k_proj.bias.fill_(2000.0)
            blk.self_attn.v_proj.bias.fill_(1500.0)
    ids = prompts(2, 12)
    run = lambda **kw: model.generate(ids, max_new_tokens=10, temperature=0.0, logprobs=True, **kw)  # noqa: E731
    want, want_p = run()
    scales = torch.full((SMALL.layers, 2, SMALL.kv_heads), 16.0, device=DEV)
    got, got_p = run(cache_dtype=torch.float8_e4m3fn, cache_scales=scales)
    _, cut_p = run(cache_dtype=torch.float8_e4m3fn)
    assert float((got_p[:, 1:] - want_p[:, 1:]).abs().max()) < float((cut_p[:, 1:] - want_p[:, 1:]).abs().max())
    with pytest.raises(ValueError, match="scales"):
        run(cache_scales=scales)
    with pytest.raises(ValueError, match="scales"):
        run(cache_dtype=torch.float8_e4m3fn, cache_scales=scales[:1])


@pytest.mark.parametrize("share", [True, False])
def test_a_fork_of_absent_pages_has_them_absent(share):
    """Not pages of its own with what somebody else has left there."""
    cache = filled([40, 50, 0, 0, 0], seed=91)
    cache.pool[cache.refs == 0] = 100.0                      # (what a free page happens to hold)
    q = normal(5, 4, 64, seed=92)
    cache.tables[0, 2] = -1                                  # the part that a fork copies
    cache.tables[1, 0], cache.tables[1, 1] = cache.pool.shape[0] + 3, -7
    want, want_lse = cache.attend(0, q[[0, 1, 0, 1]], [0, 1, 0, 1], return_lse=True)
    refs, tables = cache.refs.clone(), cache.tables.clone()
    cache.fork([0, 1], [2, 4], share=share)
    cache.check()
    got, lse = cache.attend(0, q[[0, 1, 0, 1]], [0, 1, 2, 4], return_lse=True)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    assert int(cache.tables[2, 2]) == -1 and all(not 0 <= int(p) < cache.pool.shape[0] for p in cache.tables[4, :2])
    own = cache.tables[[2, 4], :4].flatten()
    own = own[(own >= 0) & (own < cache.pool.shape[0])].long()
    assert torch.equal(cache.refs, refs.index_add(0, own, torch.ones_like(own, dtype=torch.int32)))
    cache.free([2, 4])
    assert torch.equal(cache.refs, refs) and torch.equal(cache.tables, tables)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_generate_under_another_default_type(dtype):
    """Random numbers are fp32, whatever a program has set for its tensors."""
    model, ids = decoder(), prompts(2, 8)
    run = lambda: model.generate(ids, max_new_tokens=8, answers=2, top_p=0.9, generator=gen(5), logprobs=True)  # noqa: E731
    want, want_p = run()
    before = torch.get_default_dtype()
    try:
        torch.set_default_dtype(dtype)
        got, got_p = run()
    finally:
        torch.set_default_dtype(before)
    assert torch.equal(got, want) and torch.equal(got_p, want_p)


def test_a_scaling_that_is_not_known_is_named():
    import dataclasses
    model = decoder(dataclasses.replace(SMALL, rope_scaling=dict(type="linear", factor=2.0, long_factor=[1.0, 2.0])), fuse_rotary=True)
    for call in (lambda: model(prompts(1, 4)), lambda: model.generate(prompts(1, 4), max_new_tokens=1)):
        with pytest.raises(ValueError, match="long_factor"):
            call()
