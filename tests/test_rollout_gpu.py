"""Rotary positions, the paged cache with attention over it and sampling, against plain implementations in 64 bits."""
import math

import pytest
import torch

from fp4_post_b200 import cabi, ops, rollout

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}          # half a step, relative
LLAMA3 = dict(type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position=8192)
YARN = dict(type="yarn", factor=4.0, original_max_position=4096)


@pytest.fixture(scope="module", autouse=True)
def _lib(built_library):
    return built_library


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(*shape, seed=0, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, device=DEV, generator=gen(seed)) * scale).to(dtype)


# ---- rotary positions -------------------------------------------------------------------------------------------------

def turned(x, positions, *, theta=1e4, rotary_dim=None, interleaved=False, scaling=None, sign=1.0):
    """The definition in 64 bits, angles from whole numbers of Python (a position's fraction of a turn); and sqrt(a^2 + b^2) of each element's pair."""
    n = rotary_dim or x.shape[-1]
    freq, m = rollout.rotary_frequencies(n, theta, scaling)
    bits = [round(f / (2 * math.pi) * 2 ** 64) for f in freq]
    flat = positions.reshape(-1).tolist()
    turn = torch.tensor([[(p * b) % 2 ** 64 / 2 ** 64 for b in bits] for p in flat], dtype=torch.float64, device=DEV).reshape(*positions.shape, 1, n // 2)
    c, s = torch.cos(2 * math.pi * turn) * m, sign * torch.sin(2 * math.pi * turn) * m
    y = x.double().clone()
    size = torch.zeros_like(y)
    first, second = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    a, b = x[..., first].double(), x[..., second].double()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * m
    return y, size


def close_turned(got, x, positions, **kw):
    """Half a step of the type; the angle is off by 2^-24 of half a turn at most (its conversion to fp32) and cosine and sine by 2 steps: together below
    2^-21 of |a| + |b|."""
    want, size = turned(x, positions, **kw)
    off = (got.double() - want).abs()
    assert (off <= HALF[x.dtype] * want.abs() + 2.0 ** -21 * size).all(), float((off - HALF[x.dtype] * want.abs() - 2.0 ** -21 * size).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("head_dim, rotary_dim, heads, kv_heads, tokens", [
    (128, 128, 28, 4, 37), (64, 64, 4, 2, 1), (80, 44, 10, 5, 9), (16, 2, 1, 1, 3), (8, 8, 3, 1, 300), (256, 256, 2, 2, 5), (96, 32, 1, 1, 1000), (256, 250, 1, 1, 2), (128, 64, 40, 1, 2)])
def test_rotary(dtype, interleaved, head_dim, rotary_dim, heads, kv_heads, tokens):
    q, k = normal(2, tokens, heads, head_dim, seed=1, dtype=dtype), normal(2, tokens, kv_heads, head_dim, seed=2, dtype=dtype)
    positions = torch.randint(0, 100000, (2, tokens), device=DEV, generator=gen(3))
    r = rollout.Rotary(head_dim, theta=5e5, rotary_dim=rotary_dim, interleaved=interleaved)
    kw = dict(theta=5e5, rotary_dim=rotary_dim, interleaved=interleaved)
    a, b = r(q, k, positions)
    assert a.is_contiguous() and a.shape == q.shape and b.shape == k.shape and a.dtype == dtype
    close_turned(a, q, positions, **kw)
    close_turned(b, k, positions, **kw)
    assert torch.equal(r(q, None, positions.int()), a) and torch.equal(r(k, positions=positions), b)


@pytest.mark.parametrize("scaling", [None, dict(type="linear", factor=4.0), LLAMA3, YARN])
def test_rotary_scaled_for_long_contexts(scaling):
    x = normal(64, 2, 64, seed=4)
    positions = torch.randint(0, 1 << 20, (64,), device=DEV, generator=gen(5))
    close_turned(rollout.Rotary(64, scaling=scaling)(x, None, positions), x, positions, scaling=scaling)


def test_rotary_far_and_negative_positions():
    x = normal(8, 1, 128, seed=6, dtype=torch.float32)
    positions = torch.tensor([0, 1, -1, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31, 2 ** 40 + 3, -2 ** 45], device=DEV)
    close_turned(rollout.Rotary(128, theta=1e6)(x, None, positions), x, positions, theta=1e6)
    p32 = positions[:6].int()
    close_turned(rollout.Rotary(128, theta=1e6)(x[:6], None, p32), x[:6], p32, theta=1e6)


def test_rotary_default_and_broadcast_positions():
    x = normal(3, 11, 2, 32, seed=7)
    r = rollout.Rotary(32)
    t = torch.arange(11, device=DEV)
    want = r(x, None, t.expand(3, 11).contiguous())
    assert torch.equal(r(x), want) and torch.equal(r(x, None, t), want) and torch.equal(r(x, None, t[None]), want)
    one = torch.tensor([[4], [5], [6]], device=DEV)
    assert torch.equal(r(x, None, one), r(x, None, one.expand(3, 11).contiguous()))
    deep = x.reshape(3, 1, 11, 2, 32).expand(3, 2, 11, 2, 32)
    assert torch.equal(r(deep)[:, 1], want)
    assert torch.equal(r(x[0]), want[0]) and torch.equal(r(x[0, 5], None, t[5]), want[0, 5])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rotary_reads_tensors_of_any_strides(dtype):
    fused = normal(2, 6, 8 * 64 + 1, seed=8, dtype=dtype)
    positions = torch.arange(12, device=DEV).view(2, 6)
    r = rollout.Rotary(64)
    even = fused[..., :-1].unflatten(-1, (8, 64))
    for x in (even[..., :5, :], even[..., ::2, :], even.transpose(0, 1).contiguous().transpose(0, 1), even.transpose(1, 2).contiguous().transpose(1, 2),
              fused[..., 1:].unflatten(-1, (8, 64)), even[:, ::3], even[..., :1, :].expand(2, 6, 3, 64), even.transpose(2, 3).contiguous().transpose(2, 3), even.flip(2)):
        p = positions[:, ::3] if x.shape[1] == 2 else positions
        assert torch.equal(r(x, None, p), r(x.contiguous(), None, p.contiguous()))
    assert torch.equal(r(torch._neg_view(even), None, positions), r(-even, None, positions))


def test_rotary_without_tokens_or_heads():
    r = rollout.Rotary(64)
    assert r(torch.empty(2, 0, 3, 64, device=DEV)).shape == (2, 0, 3, 64)
    q, k = r(normal(5, 2, 64), torch.empty(5, 0, 64, device=DEV, dtype=torch.bfloat16))
    assert q.shape == (5, 2, 64) and k.shape == (5, 0, 64) and torch.equal(q, r(normal(5, 2, 64)))
    q, k = r(torch.empty(5, 0, 64, device=DEV, dtype=torch.bfloat16), normal(5, 2, 64))
    assert q.numel() == 0 and torch.equal(k, r(normal(5, 2, 64)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved, rotary_dim, scaling", [(False, 64, None), (True, 36, YARN)])
def test_rotary_gradients(dtype, interleaved, rotary_dim, scaling):
    q, k = normal(2, 9, 6, 64, seed=9, dtype=dtype).requires_grad_(), normal(2, 9, 2, 64, seed=10, dtype=dtype).requires_grad_()
    positions = torch.randint(0, 5000, (2, 9), device=DEV, generator=gen(11))
    kw = dict(rotary_dim=rotary_dim, interleaved=interleaved, scaling=scaling)
    r = rollout.Rotary(64, **kw)
    a, b = r(q, k, positions)
    da, db = normal(*a.shape, seed=12, dtype=dtype), normal(2, 2, 9, 64, seed=13, dtype=dtype).transpose(1, 2)      # (as attention gives it)
    dq, dk = torch.autograd.grad((a, b), (q, k), (da, db))
    close_turned(dq, da, positions, sign=-1.0, **kw)
    close_turned(dk, db, positions, sign=-1.0, **kw)
    # one of the two alone, and an expanded gradient
    a, b = r(q, k, positions)
    assert torch.equal(torch.autograd.grad(b, k, db)[0], dk)
    a, b = r(q, k.detach(), positions)
    assert torch.equal(torch.autograd.grad(a, q, da)[0], dq)
    (g,) = torch.autograd.grad(r(q, None, positions).sum(), q)
    close_turned(g, torch.ones_like(q), positions, sign=-1.0, **kw)


def test_rotary_gradients_against_differences():
    """The map is linear: in fp32 a difference over a step of 1 is its own rounding off the derivative."""
    r = rollout.Rotary(16, rotary_dim=12, interleaved=True, scaling=YARN)
    x, g = normal(5, 2, 16, seed=14, dtype=torch.float32).requires_grad_(), normal(5, 2, 16, seed=15, dtype=torch.float32)
    (dx,) = torch.autograd.grad(r(x), x, g)
    with torch.no_grad():
        base = (r(x).double() * g.double()).sum()
        for at in [(0, 0, 0), (1, 0, 5), (4, 1, 11), (3, 1, 12), (2, 0, 15)]:
            y = x.detach().clone()
            y[at] += 1.0
            assert abs(float((r(y).double() * g.double()).sum() - base) - float(dx[at])) < 1e-5


def test_rotary_is_differentiable_again():
    r = rollout.Rotary(16)
    x, g = normal(5, 2, 16, seed=16, dtype=torch.float32).requires_grad_(), normal(5, 2, 16, seed=17, dtype=torch.float32).requires_grad_()
    (dx,) = torch.autograd.grad(r(x), x, g, create_graph=True)
    w = normal(5, 2, 16, seed=18, dtype=torch.float32)
    (dg,) = torch.autograd.grad(dx, g, w)
    close_turned(dg, w, torch.arange(5, device=DEV))


def test_rotary_forward_and_backward_replay_from_a_graph():
    r = rollout.Rotary(64)
    x, g = normal(2, 8, 4, 64, seed=19), normal(2, 8, 4, 64, seed=20)
    positions = torch.arange(16, device=DEV).view(2, 8)

    def step():
        leaf = x.detach().requires_grad_()
        y = r(leaf, None, positions)
        return y.detach(), torch.autograd.grad(y, leaf, g)[0]
    from fp4_post_b200.graphs import GraphedStep
    graphed = GraphedStep(step, warmup=1)
    x.copy_(normal(2, 8, 4, 64, seed=21))
    positions.add_(1000)
    y, dx = graphed()
    torch.cuda.synchronize()
    close_turned(y, x, positions)
    close_turned(dx, g, positions, sign=-1.0)
    graphed.release()


def test_rotary_refuses():
    r = rollout.Rotary(64)
    q = normal(2, 3, 4, 64)
    for bad, error in [((q.half(),), TypeError), ((q, q.float()), TypeError), ((q, q[:1]), ValueError), ((q, None, torch.zeros(4, device=DEV, dtype=torch.long)), ValueError),
                       ((q, None, torch.zeros(2, 3, device=DEV)), TypeError), ((q, None, torch.zeros(2, 3, dtype=torch.long)), RuntimeError), ((q[..., :32],), ValueError),
                       ((q, q[..., :32]), ValueError), ((q, None, torch.zeros(1, 2, 3, device=DEV, dtype=torch.long)), ValueError), ((q[0, 0, 0],), ValueError), ((q.cpu(),), RuntimeError)]:
        with pytest.raises(error):
            r(*bad)
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        r(fwAD.make_dual(q, q))
    with pytest.raises(RuntimeError):
        torch.func.vmap(r)(q)


# ---- the cache --------------------------------------------------------------------------------------------------------

def new_cache(layers=1, kv_heads=2, head_dim=64, **kw):
    kw = dict(dict(pages=40, sequences=6, max_length=128, page_size=16), **kw)
    return rollout.PagedCache(layers, kv_heads, head_dim, **kw)


class Model:
    """The bookkeeping, in Python."""

    def __init__(self, pages, sequences, page, width):
        self.refs, self.tables, self.page, self.width = [0] * pages, [[] for _ in range(sequences)], page, width
        self.lengths = [0] * sequences

    def free_pages(self):
        return [p for p, r in enumerate(self.refs) if r == 0]

    def take(self, n):
        got = self.free_pages()[:n]
        for p in got:
            self.refs[p] = 1
        return got

    def reserve(self, slots, counts):
        live = [(s, c) for s, c in zip(slots, counts) if s >= 0]
        if len({s for s, _ in live}) < len(live) or any(s >= len(self.tables) or c < 0 or self.lengths[s] + c > self.width * self.page for s, c in live):
            return False
        need = [-(-(self.lengths[s] + c) // self.page) - len(self.tables[s]) for s, c in live]
        if sum(need) > len(self.free_pages()):
            return False
        for (s, c), n in zip(live, need):
            self.tables[s] += self.take(n)
            self.lengths[s] += c
        return True

    def fork(self, src, dst, share):
        """Moves (from, to, rows), or None."""
        live = [(s, d) for s, d in zip(src, dst) if s >= 0 and d >= 0]
        if len({d for _, d in live}) < len(live) or any(max(s, d) >= len(self.tables) or self.lengths[d] for s, d in live):
            return None
        full = [self.lengths[s] // self.page if share else 0 for s, _ in live]
        if sum(len(self.tables[s]) - f for (s, _), f in zip(live, full)) > len(self.free_pages()):
            return None
        moves, new = [], []
        for (s, d), f in zip(live, full):
            own = self.take(len(self.tables[s]) - f)
            for i, p in enumerate(own):
                moves.append((self.tables[s][f + i], p, min(self.page, self.lengths[s] - (f + i) * self.page)))
            for p in self.tables[s][:f]:
                self.refs[p] += 1
            new.append((d, self.tables[s][:f] + own, self.lengths[s]))
        for d, t, n in new:
            self.tables[d], self.lengths[d] = t, n
        return moves

    def free(self, slots):
        for s in slots:
            if 0 <= s < len(self.tables):
                for p in self.tables[s]:
                    self.refs[p] -= 1
                self.tables[s], self.lengths[s] = [], 0

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        holes, movers = [p for p in range(n) if self.refs[p] == 0], [p for p in range(n, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.tables = [[to.get(p, p) for p in t] for t in self.tables]
        return n, [(a, b, self.page) for a, b in to.items()]

    def same_as(self, cache):
        tables = torch.full((len(self.tables), self.width), -1, dtype=torch.int32)
        for i, t in enumerate(self.tables):
            tables[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
        assert torch.equal(cache.tables.cpu(), tables)
        assert cache.lengths.tolist() == self.lengths and cache.refs.tolist() == self.refs


@pytest.mark.parametrize("page, pages, sequences, dtype, seed", [(16, 40, 6, torch.bfloat16, 0), (48, 17, 9, torch.bfloat16, 1), (16, 9001, 40, torch.float8_e4m3fn, 2), (32, 300, 65, torch.bfloat16, 3)])
def test_bookkeeping_follows_a_plain_one(page, pages, sequences, dtype, seed):
    import random
    rng = random.Random(seed)
    head_dim = 24 if pages > 1000 else 40
    cache = rollout.PagedCache(3, 2, head_dim, pages=pages, sequences=sequences, max_length=page * 9, page_size=page, dtype=dtype)
    bits = torch.uint8 if dtype == torch.float8_e4m3fn else torch.int16
    cache.pool.view(bits).copy_(torch.randint(0, 100, cache.pool.shape, device=DEV, generator=gen(seed)))
    model, pool = Model(pages, sequences, page, cache.tables.shape[1]), cache.pool.view(bits).clone()
    refused = 0
    for step in range(120):
        op = rng.choice(["reserve", "reserve", "fork", "fork", "free", "compact"])
        pick = lambda n: [rng.randrange(-1, sequences + (rng.random() < 0.03)) for _ in range(n)]  # noqa: E731
        if op == "reserve":
            slots = rng.sample(range(sequences), rng.randint(1, sequences)) if rng.random() < 0.8 else pick(3)
            counts = [rng.choice([0, 1, 1, page - 1, page, rng.randint(0, 3 * page)]) for _ in slots]
            done = model.reserve(slots, counts)
            if rng.random() < 0.5:
                cache.reserve(slots, counts)
            else:
                cache.reserve(torch.tensor(slots, dtype=torch.int32, device=DEV), torch.tensor(counts, dtype=torch.int32, device=DEV))
        elif op == "fork":
            n = rng.randint(1, sequences)
            empty = [s for s in range(sequences) if not model.lengths[s]]
            src, dst = [rng.randrange(sequences) for _ in range(n)], pick(n)
            if empty and rng.random() < 0.8:
                dst = rng.sample(empty, min(n, len(empty)))
                src = src[:len(dst)]
            share = rng.random() < 0.7
            moves = model.fork(src, dst, share)
            done = moves is not None
            for a, b, rows in moves or []:
                pool[b, ..., :rows, :] = pool[a, ..., :rows, :]
            cache.fork(src, dst, share=share)
        elif op == "free":
            slots = pick(rng.randint(1, 4))
            model.free(slots)
            cache.free(slots)
            done = max(slots) < sequences
        else:
            n, moves = model.compact()
            for a, b, rows in moves:
                pool[b] = pool[a]
            assert int(cache.compact()) == n
            done = True
        model.same_as(cache)
        if done:
            cache.check()
        else:
            refused += 1
            with pytest.raises(RuntimeError, match="paged cache"):
                cache.check()
            cache.check()
        assert torch.equal(cache.pool.view(bits), pool), (step, op)
    assert refused > 3
    assert cache.free_pages() == len(model.free_pages())


def test_reasons_are_named_and_the_first_one_stays():
    cache = new_cache(pages=4)
    cache.reserve([0], 16 * 5)
    with pytest.raises(RuntimeError, match="not enough free pages"):
        cache.check()
    cache.reserve([6], 1)
    cache.reserve([0, 0], 1)
    with pytest.raises(RuntimeError, match="does not have"):
        cache.check()
    cache.reserve([0, 0], 1)
    with pytest.raises(RuntimeError, match="twice"):
        cache.check()
    for counts in (129, -1, 2 ** 62, 2 ** 63 - 1):
        cache.reserve([0], counts)
        with pytest.raises(RuntimeError, match="longer"):
            cache.check()
    cache.reserve(None, [1, 0, 0, 0, 0, 0])
    cache.fork([0], [0])
    with pytest.raises(RuntimeError, match="not empty"):
        cache.check()
    cache.fork([0, 0], [1, 1])
    with pytest.raises(RuntimeError, match="twice"):
        cache.check()
    cache.free([17])
    with pytest.raises(RuntimeError, match="does not have"):
        cache.check()
    assert cache.lengths.tolist() == [1, 0, 0, 0, 0, 0] and cache.free_pages() == 3
    cache.free()
    assert cache.free_pages() == 4


def test_empty_calls_do_nothing():
    cache = new_cache()
    none = torch.empty(0, dtype=torch.long, device=DEV)
    cache.reserve(none, 3)
    cache.fork(none, none)
    cache.free(none)
    assert int(cache.compact()) == 0
    cache.fork([0], [0])                                     # (an empty one is its own copy)
    cache.check()
    assert cache.append(0, normal(0, 4, 64), normal(0, 2, 64), normal(0, 2, 64)).shape == (0, 4, 64)
    assert cache.attend(0, normal(0, 4, 64)).shape == (0, 4, 64)


def test_caches_refuse():
    ok = dict(pages=4, sequences=2, max_length=32)
    for bad, error in [(dict(head_dim=20), ValueError), (dict(head_dim=264), ValueError), (dict(page_size=8), ValueError), (dict(page_size=0), ValueError),
                       (dict(dtype=torch.float32), TypeError), (dict(scales=torch.ones(1, 2, 2, device=DEV)), ValueError),
                       (dict(sequences=(1 << 17) + 1), ValueError)]:
        with pytest.raises(error):
            rollout.PagedCache(**{**dict(layers=1, kv_heads=2, head_dim=64), **ok, **bad})
    c = new_cache()
    for tensors, error in [((c.pool[0], c.tables, c.lengths, c.refs), ValueError), ((c.pool, c.tables.long(), c.lengths, c.refs), TypeError), ((c.pool, c.tables, c.lengths[:-1], c.refs), ValueError),
                           ((c.pool, c.tables, c.lengths, c.refs[1:]), ValueError), ((c.pool, c.tables.cpu(), c.lengths, c.refs), RuntimeError), ((c.pool.transpose(0, 1), c.tables, c.lengths, c.refs), ValueError),
                           ((c.pool, c.tables.t().contiguous().t(), c.lengths, c.refs), ValueError)]:
        with pytest.raises(error):
            rollout.PagedCache.of(*tensors)
    q, k = normal(6, 4, 64), normal(6, 2, 64)
    for call, error in [(lambda: c.append(1, q, k, k), ValueError), (lambda: c.append(-1, q, k, k), ValueError), (lambda: c.append(0, q, k[:, :1], k), ValueError),
                        (lambda: c.append(0, q[:5], k, k), ValueError), (lambda: c.append(0, q, k, k.float()), TypeError), (lambda: c.append(0, q, k, k, [0]), ValueError),
                        (lambda: c.append(0, q, k, k, None, torch.zeros(6, device=DEV)), TypeError), (lambda: c.append(0, q, k, k, rotary=rollout.Rotary(32)), ValueError),
                        (lambda: c.append(0, q.clone().requires_grad_(), k, k), RuntimeError), (lambda: c.attend(0, q[:, :3]), ValueError), (lambda: c.attend(0, q.requires_grad_()), RuntimeError),
                        (lambda: c.attend(0, k.cpu()), RuntimeError), (lambda: c.attend(0, k[..., :32]), ValueError), (lambda: c.attend(0, k, torch.zeros(6, dtype=torch.long)), RuntimeError)]:
        with pytest.raises(error):
            call()


# ---- append -----------------------------------------------------------------------------------------------------------

def stored(x, scale):
    """The 8-bit value nearest to x / scale (in fp32: the quotient that the format rounds is the fp32 one)."""
    return (x.float() / scale).clamp(-448, 448).to(torch.float8_e4m3fn)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("head_dim, rotary_dim, interleaved, heads, kv_heads", [(128, 128, False, 28, 4), (64, 64, True, 4, 4), (80, 20, False, 5, 1), (48, 10, True, 6, 2), (256, 256, False, 2, 1), (64, 0, False, 4, 2), (32, 32, False, 0, 2), (104, 104, True, 3, 1), (8, 8, False, 1, 1)])
def test_append(dtype, head_dim, rotary_dim, interleaved, heads, kv_heads):
    scales = 0.25 + torch.rand(2, 2, kv_heads, device=DEV, generator=gen(1)) if dtype == torch.float8_e4m3fn else None
    cache = rollout.PagedCache(2, kv_heads, head_dim, pages=30, sequences=5, max_length=100, page_size=16, dtype=dtype, scales=scales)
    cache.reserve([3, 0, 4], [37, 16, 1])
    bits = torch.uint8 if scales is not None else torch.int16
    cache.pool.view(bits).copy_(torch.randint(0, 100, cache.pool.shape, device=DEV, generator=gen(2)))
    before = cache.pool.clone()
    # all tokens of 3 and 0 in some order, one of 4, one of nobody, one of an empty sequence, ones behind and before a sequence, sequences that are none
    slots = [3] * 37 + [0] * 16 + [4, -1, 1, 0, 3, 0, 5, 1 << 40]
    positions = list(range(36, -1, -1)) + list(range(16)) + [0, 3, 0, 16, 37, -1, 2, 0]
    n = len(slots)
    qkv = normal(n, heads + 2 * kv_heads, head_dim, seed=3, scale=2.0)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    r = rollout.Rotary(head_dim, theta=1e6, rotary_dim=rotary_dim, interleaved=interleaved, scaling=LLAMA3) if rotary_dim else None
    out = cache.append(1, q if heads else None, k, v, slots, torch.tensor(positions, device=DEV, dtype=torch.int32), rotary=r)
    pos = torch.tensor(positions, device=DEV)
    # (its rotation is the tested one; appending keys and values is a matter of places and roundings)
    if heads:
        want = r(q, None, pos) if r else q.clone()
        want[[i for i, s in enumerate(slots) if not 0 <= s < 5]] = 0
        assert torch.equal(out, want)
    else:
        assert out is None
    turned_k = r(k.float(), None, pos) if r else k.float()
    want = before.clone()
    for i, (s, p) in enumerate(zip(slots, positions)):
        if not 0 <= s < 5 or not 0 <= p < int(cache.lengths[s]):
            continue
        page = int(cache.tables[s, p // 16])
        for j, x in enumerate((turned_k[i], v[i].float())):
            want.view(bits)[page, 1, j, :, p % 16] = (stored(x, scales[1, j][:, None]) if scales is not None else x.bfloat16()).view(bits)
    assert torch.equal(cache.pool.view(bits), want.view(bits))


@pytest.mark.parametrize("slots", [None, [4, 2, 0, 1, 3, 5]])
def test_append_to_the_end_of_each_sequence(slots):
    cache = new_cache()
    lengths = [1, 16, 17, 0, 33, 128]
    cache.reserve(None, lengths)
    k, v = normal(6, 2, 64, seed=1), normal(6, 2, 64, seed=2)
    r = rollout.Rotary(64)
    order = slots or list(range(6))
    q = cache.append(0, normal(6, 4, 64, seed=3), k, v, slots, rotary=r)
    last = torch.tensor([lengths[s] - 1 for s in order], device=DEV)
    assert torch.equal(q, r(normal(6, 4, 64, seed=3), None, last))
    turned_k = r(k, None, last)
    seen = torch.zeros_like(cache.pool)
    for i, s in enumerate(order):
        if lengths[s]:
            page, at = int(cache.tables[s, (lengths[s] - 1) // 16]), (lengths[s] - 1) % 16
            seen[page, 0, 0, :, at], seen[page, 0, 1, :, at] = turned_k[i], v[i]
    assert torch.equal(cache.pool, seen)


def test_append_rounds_what_8_bits_do_not_hold():
    cache = rollout.PagedCache(1, 1, 16, pages=2, sequences=2, max_length=16, dtype=torch.float8_e4m3fn, scales=torch.full((1, 2, 1), 0.5, device=DEV))
    cache.reserve([0], 1)
    x = torch.tensor([0.0, -0.0, 1.0, 224.0, 232.0, 240.0, 1e6, -1e6, math.inf, -math.inf, math.nan, 2.0 ** -10, 2.0 ** -11, 1.5 * 2.0 ** -10, 0.53125, 0.5625], device=DEV).bfloat16().view(1, 1, 16)
    cache.append(0, None, x, x, [0], [0])
    got = cache.pool[int(cache.tables[0, 0]), 0, :, 0, 0].float()
    assert torch.equal(got.nan_to_num(777.0), stored(x, 0.5).float().nan_to_num(777.0).view(1, 16).expand(2, 16))


def test_append_where_a_table_names_no_page_writes_nothing():
    cache = new_cache()
    cache.reserve([0], 40)
    cache.tables[0, 1], cache.tables[0, 2] = 40, -1
    k = normal(3, 2, 64)
    cache.append(0, None, k, k, [0, 0, 0], [5, 20, 35])
    assert int((cache.pool != 0).any(dim=-1).sum()) == 4 and torch.equal(cache.pool[0, 0, 0, :, 5], k[0])


# ---- attention ----------------------------------------------------------------------------------------------------------

def filled(lengths, *, kv_heads=2, head_dim=64, page=16, dtype=torch.bfloat16, layers=1, seed=0, garbage=True):
    """A cache of such sequences with its pages in random order; what belongs to nobody is NaN, infinite and huge."""
    import random
    rng = random.Random(seed)
    held = sum(-(-n // page) for n in lengths)
    pages, width = held + 5, -(-max(max(lengths), 1) // page) + 1
    order = rng.sample(range(pages), pages)
    e4m3 = dtype == torch.float8_e4m3fn
    pool = torch.empty(pages, layers, 2, kv_heads, page, head_dim, dtype=dtype, device=DEV)
    if garbage:
        pool.view(torch.uint8 if e4m3 else torch.int16).fill_(0x7f if e4m3 else 0x7fc1)        # NaN
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32)
    for i, n in enumerate(lengths):
        for j in range(-(-n // page)):
            p = tables[i, j] = order.pop()
            rows = min(page, n - j * page)
            pool[int(p), :, :, :, :rows] = normal(layers, 2, kv_heads, rows, head_dim, seed=seed * 1000 + i * 100 + j, scale=1.5).to(dtype)
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[tables[tables >= 0].long()] = 1
    scales = 0.5 + torch.rand(layers, 2, kv_heads, device=DEV, generator=gen(seed)) if e4m3 else None
    return rollout.PagedCache.of(pool, tables.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), refs.to(DEV), scales=scales)


def keys_values(cache, layer, slot, n):
    page = cache.page_size
    t = cache.tables[slot, :-(-n // page)].long()
    kv = cache.pool.view(torch.uint8 if cache.scales is not None else torch.bfloat16)[t, layer].view(cache.pool.dtype).double()
    if cache.scales is not None:
        kv = kv * cache.scales[layer].double()[None, :, :, None, None]
    return kv.permute(1, 2, 0, 3, 4).reshape(2, cache.kv_heads, -1, cache.head_dim)[:, :, :n]


def check_attend(cache, q, out, lse, slots, layer=0, scale=None):
    """fp32 sums of D products (each step of the tensor core may cut: (D / 16 + 2) 2^-22 of the sum of magnitudes covers them, the scale and its
    product), an exponential off by 2^-21, weights to 2^-12 (8-bit pools: fp16, with queries to 2^-25 of their row's largest) or 2^-15 (bf16 pools: the largest bf16
    below p leaves up to a step, 2^-7 p, which is rounded by half a step of its own, 2^-8 of it): a weight's relative error e enters numerator and
    denominator; one rounding of the result."""
    rows, heads, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    lengths = cache.lengths.tolist()
    group = heads // cache.kv_heads
    for i, s in enumerate(slots):
        n = lengths[s] if 0 <= s < len(lengths) else 0
        if n == 0:
            assert torch.equal(out[i], torch.zeros_like(out[i])) and (lse[i] == -math.inf).all()
            continue
        kv = keys_values(cache, layer, s, n).repeat_interleave(group, dim=1)
        x = torch.einsum("hd,hnd->hn", q[i].double(), kv[0]) * scale
        p = torch.softmax(x, dim=1)
        want = torch.einsum("hn,hnd->hd", p, kv[1])
        size = (torch.einsum("hd,hnd->hn", q[i].double().abs(), kv[0].abs()) * abs(scale)).amax(dim=1, keepdim=True)
        e = (d / 16 + 2) * 2.0 ** -22 * size + 2.0 ** -20
        if cache.scales is not None:
            e = e + q[i].double().abs().amax(dim=1, keepdim=True) * 2.0 ** -25 * kv[0].abs().sum(dim=2).amax(dim=1, keepdim=True) * abs(scale)
        weight = e + (2.0 ** -12 if cache.scales is not None else 2.0 ** -15)
        spread = torch.einsum("hn,hnd->hd", p, kv[1].abs())
        off = (out[i].double() - want).abs()
        bound = 2.0 ** -8 * want.abs() + 2 * weight * spread + 2.0 ** -24 * kv[1].abs().amax(dim=1)
        assert (off <= bound).all(), (i, s, n, float((off / bound).max()))
        true_lse = torch.logsumexp(x, dim=1)
        assert ((lse[i].double() - true_lse).abs() <= e[:, 0] + 2.0 ** -22 * true_lse.abs() + 2.0 ** -20).all(), (i, s, n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("heads, kv_heads, head_dim", [(28, 4, 128), (12, 2, 128), (2, 2, 64), (8, 1, 64), (9, 1, 64), (24, 2, 128), (33, 1, 128), (64, 1, 64), (80, 1, 128), (8, 1, 256), (40, 1, 256), (10, 5, 80), (6, 2, 16), (3, 1, 192), (5, 5, 32), (4, 2, 8), (6, 1, 72), (7, 1, 104), (2, 1, 248)])
def test_attend(dtype, heads, kv_heads, head_dim):
    lengths = [0, 1, 15, 16, 17, 31, 32, 63, 64, 65, 200, 0]
    cache = filled(lengths, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, seed=heads)
    q = normal(12, heads, head_dim, seed=5, scale=1.5)
    out, lse = cache.attend(0, q, return_lse=True)
    check_attend(cache, q, out, lse, range(12))
    assert torch.equal(cache.attend(0, q), out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("page", [16, 48, 64, 256])
def test_attend_pages_of_all_sizes_and_layers(dtype, page):
    cache = filled([500, 3, 0, 130, 257], page=page, layers=3, dtype=dtype, seed=page)
    q = normal(5, 6, 64, seed=6)
    for layer in range(3):
        out, lse = cache.attend(layer, q, return_lse=True)
        check_attend(cache, q, out, lse, range(5), layer=layer)


@pytest.mark.parametrize("lengths", [[1], [7], [5000], [30001], [0], [4096, 1], [1, 4097, 0, 0, 33], [700] * 33])
def test_attend_lengths_are_split_and_joined(lengths):
    cache = filled(lengths, head_dim=128, seed=len(lengths))
    q = normal(len(lengths), 14, 128, seed=7)
    out, lse = cache.attend(0, q, return_lse=True)
    check_attend(cache, q, out, lse, range(len(lengths)))


def test_attend_rows_of_any_sequences():
    cache = filled([40, 0, 300, 17], seed=8)
    slots = [2, -1, 0, 2, 4, 3, 1, 0, 1 << 33, 2]
    q = normal(10, 4, 64, seed=9)
    out, lse = cache.attend(0, q, slots, return_lse=True)
    check_attend(cache, q, out, lse, slots)
    narrow = [s if s < 1 << 31 else -7 for s in slots]
    assert torch.equal(cache.attend(0, q, torch.tensor(narrow, device=DEV, dtype=torch.int32)), out)
    # rows in strided tensors, and a batch shorter than the cache
    wide = normal(10, 7, 64, seed=10)
    assert torch.equal(cache.attend(0, wide[:, 2:6], slots), cache.attend(0, wide[:, 2:6].contiguous(), slots))
    assert torch.equal(cache.attend(0, q[:2]), cache.attend(0, q[:2], [0, 1]))
    odd = normal(10, 4, 65, seed=11)[..., 1:]
    assert torch.equal(cache.attend(0, odd, slots), cache.attend(0, odd.contiguous(), slots))


def test_attend_more_rows_than_a_launch_takes():
    lengths = [(i * 37) % 90 for i in range(2500)]
    cache = filled(lengths, kv_heads=1, head_dim=16, seed=12)
    q = normal(2500, 2, 16, seed=13)
    out, lse = cache.attend(0, q, return_lse=True)
    some = list(range(0, 2500, 83)) + [1023, 1024, 2047, 2048, 2499]
    for i in some:
        check_attend(cache, q[i:i + 1], out[i:i + 1], lse[i:i + 1], [i])
    back = torch.arange(2499, -1, -1, device=DEV)
    assert torch.allclose(cache.attend(0, q.flip(0), back).flip(0).float(), out.float(), rtol=2.0 ** -6, atol=1e-3)
    few = cache.attend(0, q[:1100])                          # (rows without slots past the first launch's)
    assert torch.allclose(few.float(), out[:1100].float(), rtol=2.0 ** -6, atol=1e-3)


def test_attend_scale_and_sharp_rows():
    cache = filled([200, 90], seed=14)
    q = normal(2, 4, 64, seed=15, scale=1.0)
    for scale in (1.0, 0.0, -0.5):
        out, lse = cache.attend(0, q, scale=scale, return_lse=True)
        check_attend(cache, q, out, lse, range(2), scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_attend_queries_of_all_magnitudes(dtype):
    """8-bit pools take queries in fp16: rows beyond its range are brought into it by powers of two."""
    cache = filled([50] * 6, seed=16, dtype=dtype)
    q = normal(6, 4, 64, seed=17)
    factors = torch.tensor([2.0 ** -60, 2.0 ** -30, 2.0 ** -14, 1.0, 2.0 ** 20, 2.0 ** 60], device=DEV)
    q = (q.float() * factors[:, None, None]).bfloat16()
    for i, f in enumerate(factors.tolist()):
        out, lse = cache.attend(0, q[i:i + 1], [i], scale=0.125 / f, return_lse=True)
        check_attend(cache, q[i:i + 1], out, lse, [i], scale=0.125 / f)


def test_attend_keys_that_are_infinite_or_not_numbers():
    cache = filled([100, 100, 100, 40], kv_heads=1, seed=18)
    page = lambda s, j: int(cache.tables[s, j])  # noqa: E731
    q = normal(4, 2, 64, seed=19).abs()
    k = cache.pool[:, 0, 0, 0]
    v = cache.pool[:, 0, 1, 0]
    k[page(0, 0)] = -math.inf                                # the first tile of a row weighs nothing
    v[page(1, 2), 3, 5] = math.inf
    k[page(2, 4), 1, 7] = math.nan
    k[page(3, 0)] = k[page(3, 1)] = -math.inf
    k[page(3, 2), :8] = -math.inf                            # a row whose keys all weigh nothing
    out, lse = cache.attend(0, q, return_lse=True)
    x = q[0].double() @ k[cache.tables[0, :7].long()].reshape(-1, 64)[16:100].double().t() / 8
    want = torch.softmax(x, dim=1) @ v[cache.tables[0, :7].long()].reshape(-1, 64)[16:100].double()
    assert torch.allclose(out[0].double(), want, rtol=2.0 ** -7, atol=1e-4) and torch.allclose(lse[0].double(), torch.logsumexp(x, 1), rtol=1e-5)
    assert (out[1][:, 5] == math.inf).all() and torch.isfinite(out[1][:, :5]).all() and torch.isfinite(out[1][:, 6:]).all() and torch.isfinite(lse[1]).all()
    assert torch.isnan(out[2]).all() and torch.isnan(lse[2]).all()
    assert torch.isnan(out[3]).all() and (lse[3] == -math.inf).all()           # as softmax of -inf alone


def test_attend_pages_that_are_none_are_absent():
    cache = filled([100, 64], seed=20)
    q = normal(2, 4, 64, seed=21)
    want = cache.attend(0, q, [1, 1])[0]
    tables = cache.tables.clone()
    cache.tables[0, :4] = tables[1, :4]
    cache.tables[0, 4], cache.tables[0, 5], cache.tables[0, 6] = -1, cache.pool.shape[0], 2 ** 31 - 1
    got, lse = cache.attend(0, q[[0, 0]], [0, 1], return_lse=True)
    assert torch.allclose(got[0].float(), got[1].float(), rtol=2.0 ** -6, atol=1e-3) and torch.allclose(lse[0], lse[1], rtol=1e-6, atol=1e-6)
    assert torch.equal(got[1], want)


def test_a_cache_whose_offsets_pass_32_bits():
    pages, shape = 1100, (4, 2, 8, 512, 128)                 # 4 Mi elements a page
    pool = torch.empty(pages, *shape, dtype=torch.bfloat16, device=DEV)
    assert pool.numel() > 2 ** 32
    tables = torch.tensor([[1099, 3, 1098], [1097, 1096, 1095]], dtype=torch.int32, device=DEV)
    cache = rollout.PagedCache.of(pool, tables, torch.tensor([1100, 700], dtype=torch.int32, device=DEV), torch.zeros(pages, dtype=torch.int32, device=DEV))
    for layer in (0, 3):
        k, v = normal(1800, 8, 128, seed=22), normal(1800, 8, 128, seed=23)
        slots, positions = [0] * 1100 + [1] * 700, list(range(1100)) + list(range(700))
        cache.append(layer, None, k, v, slots, positions)
        q = normal(2, 8, 128, seed=24)
        out, lse = cache.attend(layer, q, return_lse=True)
        check_attend(cache, q, out, lse, range(2), layer=layer)
        assert torch.equal(keys_values(cache, layer, 0, 1100)[1], v[:1100].double().transpose(0, 1))
    cache.refs[[1099, 3, 1098, 1097, 1096, 1095]] = 1
    want = pool[1099].clone()
    assert int(cache.compact()) == 6
    # (the last entry lies behind its sequence of two pages: it stays, its page is held and moves to the first hole)
    assert sorted(cache.tables.flatten().tolist()) == [1, 2, 3, 4, 5, 1095]
    assert torch.equal(pool[int(cache.tables[0, 0])], want)


def test_attend_gives_the_same_bits_again_and_on_other_streams():
    cache = filled([1000, 3, 77, 2000], seed=25, head_dim=128)
    q = normal(4, 14, 128, seed=26)
    first = cache.attend(0, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [cache.attend(0, q) for _ in range(5)]
    again = [cache.attend(0, q) for _ in range(5)]           # at the same time as the others
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, first) for o in outs + again)


def test_a_decode_step_replays_from_a_graph_as_its_sequences_grow():
    cache = new_cache(layers=2, pages=60, sequences=4)
    cache.reserve([0, 1, 3], [14, 1, 31])
    twin = new_cache(layers=2, pages=60, sequences=4)
    twin.reserve([0, 1, 3], [14, 1, 31])
    r = rollout.Rotary(64)
    q, k, v = normal(4, 6, 64, seed=27), normal(4, 2, 64, seed=28), normal(4, 2, 64, seed=29)
    slots = torch.tensor([3, 1, -1, 0], device=DEV)

    def step(c, q, k, v):
        c.reserve(slots, 1)
        return [c.attend(layer, c.append(layer, q * (layer + 1), k, v, slots, rotary=r), slots) for layer in range(2)]
    step(twin, q, k, v)
    twin.free()
    twin.reserve([0, 1, 3], [14, 1, 31])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(cache, q, k, v)
    for i in range(40):
        for t, s in ((q, 100), (k, 200), (v, 300)):
            t.copy_(normal(*t.shape, seed=s + i))
        graph.replay()
        want = step(twin, q, k, v)
        assert torch.equal(cache.tables, twin.tables) and torch.equal(cache.lengths, twin.lengths) and torch.equal(cache.refs, twin.refs)
        for layer in range(2):
            assert torch.equal(outs[layer], want[layer]), i
    cache.check()
    twin.check()


@pytest.mark.parametrize("length", [37, 32, 5])
def test_forked_sequences_grow_apart(length):
    """Two answers and their prompt each go on by tokens of their own: what they share stays, what they add is theirs."""
    cache = new_cache(pages=30, sequences=4)
    k, v = normal(length, 2, 64, seed=30), normal(length, 2, 64, seed=31)
    cache.reserve([0], length)
    cache.append(0, None, k, v, [0] * length, list(range(length)))
    cache.fork([0, 0], [2, 3])
    want = {s: ([k], [v]) for s in (0, 2, 3)}
    for step in range(20):
        slots = [2, 0, 3] if step % 3 else [3, 2]
        cache.reserve(slots, 1)
        nk, nv = normal(len(slots), 2, 64, seed=100 + step), normal(len(slots), 2, 64, seed=200 + step)
        cache.append(0, None, nk, nv, slots)
        for i, s in enumerate(slots):
            want[s][0].append(nk[i:i + 1])
            want[s][1].append(nv[i:i + 1])
    cache.check()
    for s, (ks, vs) in want.items():
        n = int(cache.lengths[s])
        assert n == sum(len(t) for t in ks)
        got = keys_values(cache, 0, s, n)
        assert torch.equal(got[0], torch.cat(ks).double().transpose(0, 1)) and torch.equal(got[1], torch.cat(vs).double().transpose(0, 1))
    cache.free([0])
    for s in (2, 3):
        assert torch.equal(keys_values(cache, 0, s, int(cache.lengths[s]))[0], torch.cat(want[s][0]).double().transpose(0, 1))
    before = {s: keys_values(cache, 0, s, int(cache.lengths[s])) for s in (2, 3)}
    cache.compact()
    for s in (2, 3):
        assert torch.equal(keys_values(cache, 0, s, int(cache.lengths[s])), before[s])


def test_graphs_of_several_caches_replay_in_turn():
    caches = [filled([900, 3, 40], seed=32, head_dim=128), filled([20, 1300, 0], seed=33, head_dim=128)]
    qs = [normal(3, 14, 128, seed=34), normal(3, 14, 128, seed=35)]
    x, u = normal(2, 9000, seed=36), torch.rand(2, device=DEV, generator=gen(37))
    graphs, outs = [], []
    for c, q in zip(caches, qs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((c.attend(0, q, return_lse=True), rollout.sample(x, u, top_p=0.8)))
        graphs.append(g)
    side = torch.cuda.Stream()
    for i in range(6):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    for c, q, ((out, lse), token) in zip(caches, qs, outs):
        want = c.attend(0, q, return_lse=True)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and torch.equal(token, rollout.sample(x, u, top_p=0.8))


def test_counts_are_whole_numbers_of_any_kind():
    import numpy as np
    cache = new_cache()
    cache.reserve([0], np.int64(3))
    cache.reserve(np.array([1, 2]), np.array([4, 5]))
    cache.check()
    assert cache.lengths.tolist() == [3, 4, 5, 0, 0, 0]


# ---- sampling -----------------------------------------------------------------------------------------------------------

def chosen(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row, by sorting; the weights in fp32, all else in 64 bits.  The token, the kept mask and the weights."""
    x = x.float()
    if torch.isnan(x).any():
        x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    top = x.max()
    if top == -math.inf:
        return -1, None, None
    heat = torch.tensor(temperature or 1.0, device=DEV, dtype=torch.float32)
    w = torch.where(x == top, torch.ones_like(x), ((x - top) * (1.0 / heat)).exp())
    order = torch.sort(x, descending=True, stable=True).indices
    ws = w[order].double()
    n = x.numel()
    k = 1 if temperature == 0 else min(top_k or n, n)
    kept = torch.arange(n, device=DEV) < k
    before = ws.cumsum(0) - ws
    total = ws[:k].sum()
    if top_p < 1.0:
        kept &= before < top_p * total
    kept &= ws >= torch.tensor(min_p, dtype=torch.float32).item()
    kept[0] = True
    mask = torch.zeros(n, dtype=torch.bool, device=DEV)
    mask[order[kept]] = True
    sums = torch.where(mask, w.double(), 0.0).cumsum(0)
    return int((sums <= u * sums[-1]).sum()), mask, w


def check_samples(logits, u, **kw):
    token, logp = rollout.sample(logits, u, logprobs=True, **kw)
    assert torch.equal(rollout.sample(logits, u, **kw), token) and token.dtype == torch.int64
    get = lambda v, i: v[i].item() if isinstance(v, torch.Tensor) else v  # noqa: E731
    for i in range(logits.shape[0]):
        row = {k: get(v, i) for k, v in kw.items()}
        want, mask, _ = chosen(logits[i], u[i].double().item(), **row)
        assert int(token[i]) == want, (i, int(token[i]), want, row)
        if want < 0:
            assert math.isnan(float(logp[i]))
            continue
        x = torch.nan_to_num(logits[i].double(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        if math.isinf(float(x.max())):
            exact = -math.log(int((x == math.inf).sum()))
        else:
            exact = float(torch.log_softmax(x / (row.get("temperature", 1.0) or 1.0), 0)[want])
        # weights are fp32 (2^-22 and, of an argument z rounded to fp32, |z| 2^-23: less than 2^-18 where a weight counts), 1 / temperature 2^-24 of z
        assert abs(float(logp[i]) - exact) <= 2.0 ** -18 + 2.0 ** -22 * abs(exact), (i, float(logp[i]), exact)
        # in 64 bits throughout: the token's share of the kept ones holds u, to what the weights' rounding moves
        if row.get("top_p", 1.0) == 1.0 and row.get("min_p", 0.0) == 0.0 and not math.isinf(float(x.max())):
            w = torch.where(mask, ((x - x.max()) / (row.get("temperature", 1.0) or 1.0)).exp(), 0.0)
            s = w.cumsum(0) / w.sum()
            low = float(s[want - 1]) if want else 0.0
            assert low - 2.0 ** -17 <= float(u[i]) <= float(s[want]) + 2.0 ** -17


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 97, 512, 513, 8192, 8193, 16385, 40000, 151936, 152064])
def test_sample(dtype, vocab):
    x = normal(6, vocab, seed=vocab, scale=3.0, dtype=dtype)
    u = torch.rand(6, device=DEV, generator=gen(vocab))
    for kw in (dict(), dict(temperature=0.7), dict(top_k=5), dict(top_k=300), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=0.0),
               dict(temperature=1.3, top_k=50, top_p=0.8, min_p=0.01), dict(top_k=vocab + 7, top_p=0.999), dict(temperature=0.1, top_p=0.5)):
        check_samples(x, u, **kw)


@pytest.mark.parametrize("vocab", [50, 3000, 152064])
def test_sample_equal_logits_go_by_index(vocab):
    x = torch.zeros(4, vocab, device=DEV)
    x[1] = torch.randint(0, 3, (vocab,), device=DEV, generator=gen(1)).float()
    x[2, ::2] = -0.0
    x[3] = -7.25
    u = torch.tensor([0.0, 0.3, 0.5, 0.999], device=DEV)
    for kw in (dict(), dict(top_k=7), dict(top_p=0.5), dict(top_k=20, top_p=0.25), dict(min_p=1.0), dict(temperature=0.0), dict(top_p=0.0), dict(top_k=1)):
        check_samples(x, u, **kw)
    assert rollout.sample(x, u, top_k=7)[[0, 3]].tolist() == [0, 6]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [300, 20000])
def test_sample_what_may_not_be_taken(dtype, vocab):
    x = normal(9, vocab, seed=2, scale=2.0, dtype=dtype)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 5:] = -math.inf
    x[3, ::3] = math.nan
    x[4, 17] = math.inf
    x[5, [3, 200, 280]] = math.inf
    x[6] = torch.finfo(dtype).min                            # a mask of the lowest value
    x[6, 100:110] = 1.0
    x[7] = -math.inf
    x[7, vocab - 1] = -1e30
    x[8, 1] = torch.finfo(dtype).max
    u = torch.rand(9, device=DEV, generator=gen(3))
    for kw in (dict(), dict(top_k=4), dict(top_p=0.7), dict(temperature=0.5, top_k=9, top_p=0.9, min_p=0.1), dict(temperature=0.0), dict(top_k=vocab - 2, top_p=0.99)):
        check_samples(x, u, **kw)
    token = rollout.sample(x, u)
    assert token[0] == -1 and token[1] == -1 and token[4] == 17 and token[7] == vocab - 1 and token[8] == 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sample_cuts_among_small_and_far_values(dtype):
    """Cuts among logits of tiny magnitude (subnormal ones too), far below the largest, and around huge ones."""
    n = 6000
    tiny = torch.ldexp(torch.randn(n, device=DEV, generator=gen(20)), torch.randint(-140, -6, (n,), device=DEV, generator=gen(21)))
    rows = [tiny, tiny - 0.0, torch.where(torch.arange(n, device=DEV) % 50 == 0, tiny + 3.0, tiny), -tiny.abs(), normal(n, seed=22, scale=300.0, dtype=torch.float32),
            normal(n, seed=23, scale=1e30, dtype=torch.float32), torch.where(torch.arange(n, device=DEV) == 77, 1000.0, tiny), normal(n, seed=24, scale=1e-30, dtype=torch.float32)]
    x = torch.stack(rows).to(dtype)
    x[1, ::2] = 0.0
    x[1, 1::4] = -0.0
    u = torch.rand(8, device=DEV, generator=gen(25))
    for kw in (dict(), dict(top_k=100), dict(top_p=0.5), dict(top_k=3000, top_p=0.4), dict(temperature=100.0, top_p=0.9), dict(temperature=1e3, top_k=40), dict(temperature=1e31, top_p=0.3), dict(temperature=0.01, top_k=70, top_p=0.99)):
        check_samples(x, u, **kw)


def test_sample_at_the_ends_of_u():
    x = normal(6, 1000, seed=4)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -53, 2.0 ** -60, 0.5, 0.25], device=DEV, dtype=torch.float64)
    check_samples(x, u)
    check_samples(x, u, top_p=0.6)
    bad = torch.tensor([1.0, -1e-9, math.nan, math.inf, 0.5, 2.0], device=DEV)
    assert rollout.sample(x, bad)[[0, 1, 2, 3, 5]].tolist() == [-1] * 5 and rollout.sample(x, bad)[4] >= 0


def test_sample_parameters_for_each_row():
    x = normal(8, 5000, seed=5, scale=2.5, dtype=torch.float32)
    u = torch.rand(8, device=DEV, generator=gen(6))
    kw = dict(temperature=torch.tensor([1.0, 0.0, 0.5, 2.0, 1.0, 0.25, 1e-3, 1e4], device=DEV), top_k=torch.tensor([0, 3, 1, 40, 5000, 6000, 2, 0], device=DEV, dtype=torch.int32),
              top_p=torch.tensor([1.0, 0.5, 0.5, 0.75, 0.125, 1.0, 0.5, 0.25], device=DEV), min_p=torch.tensor([0.0, 0.5, 0.0, 0.25, 0.0, 1.0, 0.0, 0.125], device=DEV))
    check_samples(x, u, **kw)
    for name, values in (("temperature", [-1.0, math.nan, math.inf, 1e-40]), ("top_p", [-0.5, math.nan]), ("min_p", [1.5, -0.5, math.nan])):
        for value in values:
            bad = kw[name].clone()
            bad[4] = value
            token, logp = rollout.sample(x, u, **{**kw, name: bad}, logprobs=True)
            assert token[4] == -1 and math.isnan(float(logp[4])) and torch.equal(torch.cat((token[:4], token[5:])), torch.cat((rollout.sample(x, u, **kw)[:4], rollout.sample(x, u, **kw)[5:])))


def test_sample_rows_of_any_stride_and_batch():
    x = normal(12, 3001, seed=7, dtype=torch.bfloat16)
    u = torch.rand(12, device=DEV, generator=gen(8))
    kw = dict(top_p=0.8, temperature=0.9)
    whole = rollout.sample(x, u, **kw)
    assert torch.equal(rollout.sample(x[::3], u[::3], **kw), whole[::3]) and torch.equal(rollout.sample(x[5:6], u[5:6], **kw), whole[5:6])
    wide = torch.empty(12, 3100, device=DEV, dtype=torch.bfloat16)
    wide[:, 7:3008] = x
    assert torch.equal(rollout.sample(wide[:, 7:3008], u, **kw), whole)
    assert torch.equal(rollout.sample(x.t().contiguous().t(), u, **kw), whole)
    assert torch.equal(rollout.sample(x[:1].expand(12, 3001), u, **kw), rollout.sample(x[:1].repeat(12, 1), u, **kw))
    assert rollout.sample(x[:0], u[:0]).shape == (0,)


def test_sample_frequencies_follow_the_distribution():
    """40000 draws: a count is off its mean by more than 6 standard deviations less than once in 10^8."""
    x = torch.tensor([0.0, 1.0, 2.0, 0.5, -1.0, 3.0, 3.0, -4.0], device=DEV)
    u = torch.rand(40000, device=DEV, generator=gen(9))
    token = rollout.sample(x.expand(40000, 8), u, temperature=1.5)
    p = torch.softmax(x.double() / 1.5, 0)
    count = torch.bincount(token, minlength=8).double()
    assert ((count - 40000 * p).abs() <= 6 * (40000 * p * (1 - p)).sqrt() + 1).all()


def test_sample_the_largest_vocabulary():
    for dtype in (torch.bfloat16, torch.float32):
        x = normal(2, 393216, seed=10, scale=2.0, dtype=dtype)
        check_samples(x, torch.tensor([0.3, 0.9], device=DEV), top_p=0.9)
    with pytest.raises(ValueError, match="393216"):
        rollout.sample(torch.zeros(1, 393217, device=DEV), torch.zeros(1, device=DEV))


def test_sample_replays_from_a_graph():
    x, u = normal(4, 20000, seed=11), torch.rand(4, device=DEV, generator=gen(12))
    rollout.sample(x, u, top_p=0.9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        token = rollout.sample(x, u, top_p=0.9)
    x.copy_(normal(4, 20000, seed=13))
    graph.replay()
    assert torch.equal(token, rollout.sample(x, u, top_p=0.9))


def test_sample_refuses():
    x, u = normal(2, 8), torch.zeros(2, device=DEV)
    for kw, error in [(dict(temperature=-1.0), ValueError), (dict(temperature=math.nan), ValueError), (dict(temperature=math.inf), ValueError), (dict(top_p=1.5), ValueError), (dict(top_p=-0.1), ValueError),
                      (dict(min_p=2.0), ValueError), (dict(top_k=-1), ValueError), (dict(top_k=2.5), ValueError), (dict(temperature="hot"), TypeError), (dict(temperature=torch.ones(3, device=DEV)), ValueError),
                      (dict(top_k=torch.ones(2, device=DEV)), TypeError), (dict(top_p=torch.ones(2)), RuntimeError)]:
        with pytest.raises(error):
            rollout.sample(x, u, **kw)
    for args, error in [((x[0], u), ValueError), ((x, u[:1]), ValueError), ((x.half(), u), TypeError), ((x, u.long()), TypeError), ((x, u.cpu()), RuntimeError), ((x[:, :0], u), ValueError),
                        ((x.float().requires_grad_(), u), RuntimeError)]:
        with pytest.raises(error):
            rollout.sample(*args)


def test_the_exponential_is_torch_s():
    """Tokens are compared with a plain form that takes its weights from torch: one vocabulary entry behind a border may differ if the two
    exponentials do.  Every 97th fp32 number from -104 to 0."""
    bits = torch.arange(0x80000000 - 2 ** 32, 0xC2D00000 - 2 ** 32, 97, device=DEV, dtype=torch.int64).to(torch.int32)
    z = bits.view(torch.float32)
    w = z.exp()
    # a row of two: the maximum 0 (weight 1) and z; -log of the sum of weights is the maximum's log-probability, to fp32
    pick = torch.randint(0, z.numel(), (4096,), device=DEV, generator=gen(14))
    x = torch.stack((torch.zeros(4096, device=DEV), z[pick]), dim=1)
    _, logp = rollout.sample(x, torch.zeros(4096, device=DEV), logprobs=True)
    assert torch.equal(logp, (-torch.log1p(w[pick].double())).float()) or ((logp.double() + torch.log1p(w[pick].double())).abs() <= 2.0 ** -24 * logp.double().abs() + 2.0 ** -53).all()


def test_lengths_that_no_call_has_left_are_refused():
    cache = new_cache()
    cache.reserve([0, 1], [20, 5])
    for length in (-1, -100, -2 ** 31, 129, 2 ** 31 - 1):
        cache.lengths[2] = length
        before = [t.clone() for t in (cache.tables, cache.lengths, cache.refs)]
        for call in (lambda: cache.reserve([1, 2], 3), lambda: cache.reserve([2], 128), lambda: cache.fork([0, 2], [3, 4]), lambda: cache.fork([2], [3], share=False)):
            call()
            assert all(torch.equal(a, b) for a, b in zip(before, (cache.tables, cache.lengths, cache.refs)))
            with pytest.raises(RuntimeError, match="longer"):
                cache.check()


def test_a_nucleus_of_more_than_all_is_out_of_range():
    x, u = normal(3, 500, seed=5), torch.full((3,), 0.5, device=DEV)
    token = rollout.sample(x, u, top_p=torch.tensor([1.0, 1.0 + 2.0 ** -20, 0.5], device=DEV))
    assert token[1] == -1 and token[0] == rollout.sample(x, u)[0] and token[2] == rollout.sample(x, u, top_p=0.5)[2]


def test_attend_scores_near_the_lowest_number_still_weigh():
    cache = filled([1, 3], kv_heads=1, seed=30)
    q = torch.zeros(2, 2, 64, device=DEV, dtype=torch.bfloat16)
    q[:, :, 0] = -(2.0 ** 64)
    for slot, n in ((0, 1), (1, 3)):
        cache.pool[int(cache.tables[slot, 0]), 0, 0, 0, :n] = 0.0
        cache.pool[int(cache.tables[slot, 0]), 0, 0, 0, :n, 0] = 1.3125 * 2.0 ** 63          # scores of -1.3125 2^127, -3.2e38 in powers of 2
    out = cache.attend(0, q, scale=1.0)
    for slot, n in ((0, 1), (1, 3)):
        v = keys_values(cache, 0, slot, n)[1, 0].double()
        assert torch.allclose(out[slot].double(), v.mean(dim=0).expand(2, 64), rtol=2.0 ** -8, atol=2.0 ** -14)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("heads, kv_heads, head_dim, lengths", [(70, 2, 64, [3000, 0, 17]), (48, 1, 256, [1, 5000]), (100, 1, 128, [40] * 70), (40, 1, 128, [0, 0]), (1024, 1, 16, [33, 700])])
def test_attend_groups_in_several_chunks(dtype, heads, kv_heads, head_dim, lengths):
    cache = filled(lengths, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, seed=heads)
    q = normal(len(lengths), heads, head_dim, seed=31)
    out, lse = cache.attend(0, q, return_lse=True)
    check_attend(cache, q, out, lse, range(len(lengths)))


def test_attend_refuses_groups_beyond_its_blocks():
    cache = filled([5], kv_heads=1, head_dim=16, seed=32)
    with pytest.raises(RuntimeError, match="1024 query heads"):
        cache.attend(0, normal(1, 1025, 16))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [2000, 40000, 152064])
def test_sample_a_bin_that_holds_nearly_all(dtype, vocab):
    """Distinct logits closer to one another than a first bin is wide, and a few far from them: more in the cut's bin than a block lists."""
    x = (normal(2, vocab, seed=vocab, scale=1e-3, dtype=torch.float32) + 3.0).to(dtype)
    x[0, 5:9] = 3.5
    x[1, 100:150] = -40.0
    u = torch.tensor([0.3, 0.9], device=DEV)
    for kw in (dict(top_p=0.5), dict(top_k=777), dict(top_k=1500, top_p=0.25), dict(temperature=0.05, top_p=0.9)):
        check_samples(x, u, **kw)
