"""The bf16 products with their epilogues and the head's losses (fp4_post_b200/dense.py) against plain torch in 64 bits.

Tolerances count roundings: a bf16 output is off by at most half a step, 2^-8 of its value; sums of K products in fp32 by at most
K 2^-23 of the sum of their magnitudes (each addition rounds or cuts at 2^-23 of what it adds up to); gradients that pass through a bf16
intermediate (dz, the logits' gradient, act(z) where the gate has a gradient) by 2^-8 for each, independent from element to element, so that the
2-norm of a product's error is that part of its norm."""
import math

import pytest
import torch

from fp4_post_b200 import dense

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -8


@pytest.fixture(scope="module", autouse=True)
def _lib(built_library):
    return built_library


def normal(*shape, scale=1.0, seed=0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def act64(name, z):
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    if name == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z


def rel(a, b):
    return float((a.double() - b).norm() / b.norm().clamp(min=1e-300))


def linear64(x, w, b, act, gate, residual):
    z = x @ w.t()
    if b is not None:
        z = z + b
    y = act64(act, z)
    if gate is not None:
        y = y * gate
    if residual is not None:
        y = y + residual
    return y


def check_linear(M, N, K, act=None, bias=None, gate=False, residual=False, grad=True, seed=0, prefix=()):
    prefix = prefix or (M,)
    x, w, dy = normal(*prefix, K, seed=seed), normal(N, K, scale=K ** -0.5, seed=seed + 1), normal(*prefix, N, seed=seed + 2)
    b = None if bias is None else normal(N, seed=seed + 3, dtype=bias)
    g = normal(*prefix, N, seed=seed + 4) if gate else None
    r = normal(*prefix, N, seed=seed + 5) if residual else None
    leaves = [t for t in (x, w, b, g, r) if t is not None]
    copies = [None if t is None else t.detach().double().requires_grad_(grad) for t in (x, w, b, g, r)]
    want = linear64(copies[0].reshape(-1, K), copies[1], copies[2], act, *(None if t is None else t.reshape(-1, N) for t in copies[3:]))
    if grad:
        for t in leaves:
            t.requires_grad_(True)
        y = dense.linear(x, w, b, activation=act, gate=g, residual=r)
        grads = torch.autograd.grad(y, leaves, dy)
    else:
        y = dense.linear(x, w, b, activation=act, gate=g, residual=r)
    assert y.shape == (*prefix, N) and y.dtype == torch.bfloat16
    with torch.no_grad():
        # the value's own rounding and the sum's error, through an activation of slope at most 1.13 and the gate
        slack = (K * 2.0 ** -23 * (copies[0].reshape(-1, K).abs() @ copies[1].abs().t()) + 2.0 ** -22 * (0 if b is None else copies[2].abs())) * 1.13
        # ... whose own functions are good to 2^-20 of their value
        slack = slack + 2.0 ** -20 * act64(act, (copies[0].reshape(-1, K) @ copies[1].t()) + (0 if b is None else copies[2])).abs()
        if gate:
            slack = slack * copies[3].reshape(-1, N).abs()
        tol = STEP * want.abs() + slack * (1 + STEP) + 1e-30
        assert ((y.double().reshape(-1, N) - want).abs() <= tol).all()
    if grad:
        exact = torch.autograd.grad(want, [t for t in copies if t is not None], dy.double().reshape(-1, N))
        for t, got, ref in zip(leaves, grads, exact):
            assert got.shape == t.shape and got.dtype == t.dtype
            # its own rounding, that of dz or act(z), and less than another of the slope's
            assert rel(got.reshape(ref.shape), ref) <= 3 * STEP, (tuple(t.shape), rel(got.reshape(ref.shape), ref))
        if residual:
            assert torch.equal(grads[-1], dy)


@pytest.mark.parametrize("act", [None, "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("gate,residual,bias", [(False, False, None), (True, True, torch.bfloat16), (False, True, torch.float32), (True, False, None)])
def test_linear_and_its_gradients(act, gate, residual, bias):
    check_linear(300, 520, 264, act, bias, gate, residual)


@pytest.mark.parametrize("M,N,K", [(1, 1, 8), (1, 33, 64), (2, 7, 16), (3, 8, 8), (17, 1003, 520), (64, 256, 64), (128, 130, 1000), (129, 129, 136), (255, 257, 72),
                                   (256, 256, 256), (257, 511, 24), (1021, 769, 40), (33, 2049, 3592), (700, 64, 2048)])
def test_linear_of_every_size(M, N, K):
    check_linear(M, N, K, "silu", torch.bfloat16, True, True, seed=M)
    check_linear(M, N, K, seed=N)


def test_linear_of_more_tiles_than_pairs():
    check_linear(2500, 2600, 192, "gelu", torch.float32, False, True)


def test_linear_keeps_leading_dimensions():
    check_linear(0, 136, 64, "silu", None, True, True, prefix=(2, 3, 5))
    x, w = normal(64), normal(24, 64, seed=1)
    assert torch.equal(dense.linear(x, w), dense.linear(x[None], w)[0])


def test_linear_reads_pitched_and_misaligned_rows():
    M, N, K = 150, 200, 128
    base, w, g = normal(M, 3 * K + 8), normal(N, 2 * K, seed=1), normal(M, 2 * N + 3, seed=2)
    for x in (base[:, K:2 * K], base[:, 3:3 + K], base[::2, :K].repeat(2, 1)[:M], base.t()[:K].t(), base[:1, :K].expand(M, K)):
        for weight in (w[:, :K], w[:, 5:5 + K], w.t()[:K].t()):
            for gate in (g[:, :N], g[:, 1:1 + N], g[:, ::2][:, :N]):
                got = dense.linear(x, weight, activation="silu", gate=gate, residual=gate)
                assert torch.equal(got, dense.linear(x.clone().contiguous(), weight.clone().contiguous(), activation="silu",
                                                     gate=gate.clone().contiguous(), residual=gate.clone().contiguous()))


def test_linear_of_no_rows():
    x, w, b, r = normal(0, 64), normal(24, 64, seed=1), normal(24, seed=2), normal(0, 24, seed=3)
    for t in (x, w, b, r):
        t.requires_grad_(True)
    y = dense.linear(x, w, b, activation="silu", residual=r)
    assert y.shape == (0, 24)
    gx, gw, gb, gr = torch.autograd.grad(y, (x, w, b, r), torch.empty_like(y))
    assert gx.shape == x.shape and gr.shape == r.shape and not gw.any() and not gb.any()


@pytest.mark.parametrize("M,N,K", [(1, 473, 344), (7, 33, 8), (24, 1001, 192), (64, 2000, 520), (65, 130, 64), (128, 515, 264), (129, 515, 264), (512, 1000, 192)])
def test_roundings_of_the_gradients(M, N, K):
    """Roundings of one type that fall independently add by squares.  Up to 128 rows dz goes as two bf16 numbers: dx and dW have their own
    rounding, with the slope's, an eighth of that (1.01; over as few as 56 elements the two may agree by a third, 1.05), and 2^-9 of it from the second
    number.  Above that dz is rounded: sqrt(2) and the slope's, 1.42.  The gate's gradient has act(z) in bf16 and its own, which fall anywhere
    where there are few.  (z in bf16 would take the erf form's dx to 1.6.)"""
    for act in ("silu", "gelu", "gelu_tanh"):
        x, w, dy, g = normal(M, K), normal(N, K, scale=K ** -0.5, seed=1), normal(M, N, seed=2), normal(M, N, seed=3)
        for gate in (None, g):
            leaves = [t.clone().requires_grad_(True) for t in (x, w) + ((gate,) if gate is not None else ())]
            y = dense.linear(*leaves[:2], activation=act, gate=leaves[2] if gate is not None else None)
            got = torch.autograd.grad(y, leaves, dy)
            copies = [t.detach().double().requires_grad_(True) for t in leaves]
            out = act64(act, copies[0] @ copies[1].t())
            exact = torch.autograd.grad(out * copies[2] if gate is not None else out, copies, dy.double())
            for i, (a, e) in enumerate(zip(got, exact)):
                off, least = (a.double() - e).norm(), (e.bfloat16().double() - e).norm()
                if i < 2 or M * N >= 10000:
                    assert off <= (1.1 if M <= 128 and i < 2 else 1.5) * least, (act, i, float(off / least))
                else:
                    assert ((a.double() - e).abs() <= 2.01 * STEP * e.abs() + 2.0 ** -18).all()          # (act(z) from z in fp32, of sums of K products)


@pytest.mark.parametrize("N", [776, 771])
@pytest.mark.parametrize("gate,residual", [(True, False), (True, True), (False, True), (False, False)])
def test_linear_of_many_rows_and_what_its_gradients_keep(N, gate, residual):
    # 2100 rows: the CTA pairs, whatever the shape; 771: rows that 16 bytes do not divide
    check_linear(2100, N, 136, "silu", torch.bfloat16, gate, residual, seed=N)
    check_linear(2100, N, 72, None, None, gate, residual, seed=N + 1)


def test_linear_of_many_rows_and_shifted_operands():
    M, N, K = 2100, 776, 72
    x, w, dy = normal(M, K), normal(N, K, scale=K ** -0.5, seed=1), normal(M, N, seed=2)
    g, r = (normal(M, N + 3, seed=s)[:, 1:1 + N] for s in (3, 4))
    def run(*extra):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, *extra)]
        y = dense.linear(*leaves[:2], activation="gelu", gate=leaves[2], residual=leaves[3])
        return (y, *torch.autograd.grad(y, leaves, dy))
    # the same sums by another epilogue: an element may fall on the other side of a rounding, one step, and few do
    assert all(rel(a.double(), b.double()) <= STEP for a, b in zip(run(g, r), run(g.contiguous(), r.contiguous())))


def test_linear_slopes_of_far_values():
    """Where the slope is small it keeps its relative accuracy: fp16 with 2^15 in front is normal down to 2^-29 (silu at z = -22)."""
    for M in (8, 512):
        z = torch.linspace(-20, -10, M, device="cuda", dtype=torch.float64).bfloat16()
        x = torch.zeros(M, 8, device="cuda", dtype=torch.bfloat16)
        x[:, 0] = z
        w = torch.zeros(264, 8, device="cuda", dtype=torch.bfloat16)
        w[:, 0] = 1
        x.requires_grad_(True)
        dy = torch.zeros(M, 264, device="cuda", dtype=torch.bfloat16)
        dy[:, 7] = 1
        got, = torch.autograd.grad(dense.linear(x, w, activation="silu"), x, dy)
        z = z.double()
        p = torch.sigmoid(z)
        want = p * (1 + z * (1 - p))
        # two roundings to bf16, one to fp16; 1 + z (1 - p) and the logistic function in fp32: a few parts in 2^20
        assert ((got[:, 0].double() - want) / want).abs().max() <= 2 * 2.0 ** -8 + 2.0 ** -11


def test_linear_gradients_of_some_inputs_only():
    M, N, K = 70, 72, 64
    x, w, b, g = normal(M, K), normal(N, K, seed=1), normal(N, seed=2), normal(M, N, seed=3)
    dy = normal(M, N, seed=4)
    every = [t.clone().requires_grad_(True) for t in (x, w, b, g)]
    want = torch.autograd.grad(dense.linear(*every[:3], activation="gelu", gate=every[3]), every, dy)
    for i in range(4):
        some = [t.clone().requires_grad_(i == j) for j, t in enumerate((x, w, b, g))]
        got, = torch.autograd.grad(dense.linear(*some[:3], activation="gelu", gate=some[3]), some[i], dy)
        assert torch.equal(got, want[i])
    # a gradient that is one value for all, as that of a sum
    y = dense.linear(*every[:3], activation="gelu", gate=every[3])
    got = torch.autograd.grad(y.sum(), every)
    want = torch.autograd.grad(dense.linear(*every[:3], activation="gelu", gate=every[3]), every, torch.ones_like(y))
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_linear_with_infinities_and_nan():
    x, w = normal(40, 64), normal(48, 64, seed=1).abs()
    x[3, 5] = float("inf")
    x[4, 5] = float("nan")
    for act in (None, "silu", "gelu", "gelu_tanh"):
        y = dense.linear(x, w, activation=act)
        assert torch.isinf(y[3]).all() and torch.isnan(y[4]).all() and torch.isfinite(y[5:]).all() and torch.isfinite(y[:3]).all()
    # far tails: nothing overflows into NaN
    far = torch.tensor([[-60000.0], [-300.0], [-90.0], [-20.0], [0.0], [20.0], [90.0], [60000.0]], device="cuda").bfloat16().expand(8, 8).contiguous()
    eye = torch.eye(8, device="cuda").bfloat16()
    for act in ("silu", "gelu", "gelu_tanh"):
        want = act64(act, far.double())
        got = dense.linear(far, eye, activation=act).double()
        assert torch.isfinite(got).all() and ((got - want).abs() <= STEP * want.abs() * 1.01 + 1e-30).all()


# ---- head -------------------------------------------------------------------------------------------------------

def head64(h, w, t, temperature, ignore_index=-100):
    logits = (h @ w.t()) / temperature
    logp = torch.log_softmax(logits, dim=1)
    live = t != ignore_index
    picked = logp.gather(1, torch.where(live, t, 0)[:, None])[:, 0]
    return torch.where(live, picked, 0.0), torch.where(live, -(logp.exp() * logp).sum(dim=1), 0.0), logits


def head_inputs(M, V, K, ignored=0.2, seed=0, size=2.0):
    h, w = normal(M, K, seed=seed), normal(V, K, scale=size * K ** -0.5, seed=seed + 1)
    g = torch.Generator(device="cuda").manual_seed(seed + 2)
    t = torch.randint(0, V, (M,), device="cuda", generator=g)
    t[torch.rand(M, device="cuda", generator=g) < ignored] = -100
    t[0] = V - 1
    return h, w, t


def check_head_gradients(got, exact, h64, w64, logits, g, t, temperature, tol):
    """Two roundings: the gradient's own and that of the logits' gradient G = g / T (p - [j = t]).  And p = exp(l - lse) is off by the
    error of its argument, at most 2 tol (1 + tol) p, before the one-hot is taken from it: where p is near 1 (a vocabulary of one token) G itself
    is nearly nothing and that error is what there is.  It reaches dh as (2 tol p |g| / T) |W| at most, dw as its transpose by |h|."""
    with torch.no_grad():
        p = torch.softmax(logits, dim=1) * (torch.where(t != -100, g.double(), 0.0).abs() / temperature).expand(logits.shape[0])[:, None]
        reach = ((p @ w64.abs()).norm(), (p.t() @ h64.abs()).norm())
        for a, e, r in zip(got, exact, reach):
            assert a.dtype == torch.bfloat16 and a.shape == e.shape
            assert float((a.double() - e).norm()) <= 2 * STEP * float(e.norm()) + 4 * tol * float(r)


def check_head(M, V, K, temperature=1.0, seed=0, ignored=0.2):
    h, w, t = head_inputs(M, V, K, ignored, seed)
    h64, w64 = h.double().requires_grad_(True), w.double().requires_grad_(True)
    logp, entropy, logits = head64(h64, w64, t, temperature)
    h.requires_grad_(True)
    w.requires_grad_(True)
    # the error of a logit, and what the sum over the vocabulary and its logarithm add
    with torch.no_grad():
        tol = (K * 2.0 ** -23 * (h64.abs() @ w64.abs().t()).max() / temperature + 2.0 ** -20 * (1 + logits.abs().max())).item()
    g = normal(M, seed=seed + 5, dtype=torch.float32)

    got, ent = dense.token_logprobs(h, w, t, temperature=temperature, entropy=True)
    assert got.dtype == torch.float32 and got.shape == t.shape and not ent.requires_grad
    assert (got.double() - logp).abs().max() <= 2 * tol
    assert (ent.double() - entropy).abs().max() <= (2 + 2 * math.log(V)) * tol
    assert not got[t == -100].any()
    for upstream, forms in ((g, "none"), (torch.tensor(0.7, device="cuda"), "sum"), (torch.tensor(0.7, device="cuda"), "mean")):
        loss = dense.linear_cross_entropy(h, w, t, reduction=forms, temperature=temperature)
        want = -logp if forms == "none" else -logp.sum() if forms == "sum" else -logp.sum() / (t != -100).sum()
        assert loss.shape == want.shape and loss.dtype == torch.float32
        assert (loss.double() - want).abs().max() <= 2 * tol * (M if forms == "sum" else 1) + 2.0 ** -23 * float(want.detach().abs().max())
        grads = torch.autograd.grad(loss, (h, w), upstream)
        exact = torch.autograd.grad(want, (h64, w64), upstream.double(), retain_graph=True)
        rows = upstream / (t != -100).sum() if forms == "mean" else upstream
        check_head_gradients(grads, exact, h64, w64, logits, rows, t, temperature, tol)
    back = torch.autograd.grad(got, (h, w), g)
    exact = torch.autograd.grad(logp, (h64, w64), g.double())
    check_head_gradients(back, exact, h64, w64, logits.detach(), g, t, temperature, tol)


@pytest.mark.parametrize("M,V,K", [(1, 97, 64), (2, 4931, 1472), (54, 3225, 104), (64, 513, 72), (128, 700, 136), (129, 700, 136), (300, 1000, 264)])
def test_roundings_of_the_heads_gradients(M, V, K):
    """Up to 128 rows the logits' gradient goes as two bf16 numbers: the gradients have their own rounding, with 2^-9 of it from the second
    number's.  Above that it goes as one: two roundings, which add by squares, sqrt(2)."""
    h, w, t = head_inputs(M, V, K)
    copies = [x.double().requires_grad_(True) for x in (h, w)]
    leaves = [x.requires_grad_(True) for x in (h, w)]
    g = normal(M, seed=7, dtype=torch.float32)
    logp, _, logits = head64(*copies, t, 0.7)
    for got, want, upstream in ((dense.token_logprobs(h, w, t, temperature=0.7), logp, g),
                                (dense.linear_cross_entropy(h, w, t, temperature=0.7), -logp.sum() / (t != -100).sum(), torch.tensor(0.7, device="cuda"))):
        grads = torch.autograd.grad(got, leaves, upstream)
        exact = torch.autograd.grad(want, copies, upstream.double(), retain_graph=True)
        for a, e in zip(grads, exact):
            off, least = (a.double() - e).norm(), (e.bfloat16().double() - e).norm()
            assert off <= (1.02 if M <= 128 else 1.5) * least, float(off / least)


def test_ignored_rows_take_nothing_of_their_gradient():
    h, w, t = head_inputs(70, 130, 64, 0.4)
    leaves = [x.requires_grad_(True) for x in (h, w)]
    g = normal(70, seed=9, dtype=torch.float32)
    bad = torch.where(t == -100, float("nan"), g)
    got = [torch.autograd.grad(dense.linear_cross_entropy(h, w, t, reduction="none"), leaves, x) for x in (g, bad)]
    assert all(torch.equal(a, b) for a, b in zip(*got)) and not got[0][0][t == -100].any()


@pytest.mark.parametrize("M,V,K", [(1, 2, 8), (1, 97, 64), (3, 1, 8), (24, 97, 64), (16, 4099, 256), (33, 256, 72), (128, 257, 64), (129, 1000, 128), (257, 513, 1000),
                                   (300, 5003, 96), (1021, 777, 40), (2, 30001, 64), (64, 6000, 3584)])
def test_losses_and_their_gradients(M, V, K):
    check_head(M, V, K, seed=M + V)
    check_head(M, V, K, temperature=0.6, ignored=0.0, seed=M)


def test_losses_over_many_tiles():
    check_head(700, 40003, 128)


def test_the_common_factor_of_a_mean_is_not_rounded():
    # 1 / 1021 is not a bf16 number: in the logits' gradient it would move every gradient by the same 2^-9 or so
    h, w, t = head_inputs(1021, 3001, 128, ignored=0.0, size=0.5)
    h.requires_grad_(True)
    w.requires_grad_(True)
    h64, w64 = h.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    logp, _, _ = head64(h64, w64, t, 1.0)
    for factor in (1.0, 1.0 / 3.0):
        dh, dw = torch.autograd.grad(dense.linear_cross_entropy(h, w, t), (h, w), torch.tensor(factor, device="cuda"))
        eh, ew = torch.autograd.grad(-logp.mean(), (h64, w64), torch.tensor(factor, device="cuda", dtype=torch.float64), retain_graph=True)
        for a, e in ((dh, eh), (dw, ew)):
            # The best factor between the two is 1, but for what independent roundings of 10^5 elements leave on average, and for one that is not
            # independent: the target's element of the logits' gradient is p - 1, and where p is less than half of bf16's step below 1 (2^-9, as
            # nearly everywhere here, p being about 1 / 3001) it is rounded to -1, too far from 0 by p.
            assert abs(float((a.double() * e).sum() / (e * e).sum()) - 1.0) <= STEP / 16 + float(logp.detach().exp().mean())


def test_gradients_over_several_pieces_of_the_vocabulary(monkeypatch):
    # 65536 rows take the vocabulary in pieces of 4096 columns: 9001 of them are three
    M, V, K = 65536, 9001, 16
    h, w, t = head_inputs(M, V, K)
    h.requires_grad_(True)
    w.requires_grad_(True)
    loss = dense.linear_cross_entropy(h, w, t, reduction="sum")
    got = torch.autograd.grad(loss, (h, w))
    h64, w64 = h.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    logp, _, _ = head64(h64, w64, t, 1.0)
    exact = torch.autograd.grad(-logp.sum(), (h64, w64))
    for a, e in zip(got, exact):
        assert rel(a, e) <= 2 * STEP


@pytest.mark.parametrize("ignored", [0.0, 0.4, 1.0])
def test_rows_that_are_brought_together(ignored):
    # a product of 10^12 operations: the rows that are not ignored are packed before it
    M, V, K = 4129, 131100, 1024
    h, w, t = head_inputs(M, V, K, ignored)
    if ignored == 1.0:
        t[:] = -100
    live = t != -100
    h[~live] = float("nan")
    h.requires_grad_(True)
    w.requires_grad_(True)
    logp, ent = dense.token_logprobs(h, w, t, entropy=True, temperature=1.5)
    g = normal(M, seed=9, dtype=torch.float32)
    dh, dw = torch.autograd.grad(logp, (h, w), g)
    assert not logp[~live].any() and not ent[~live].any() and not dh[~live].any()
    loss = dense.linear_cross_entropy(h, w, t)
    dh2, dw2 = torch.autograd.grad(loss, (h, w))
    if ignored == 1.0:
        assert not dw.any() and torch.isnan(loss) and not dh2.any() and not dw2.any()
        return
    h64, w64 = h[live].detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    want, want_ent, logits = head64(h64, w64, t[live], 1.5)
    with torch.no_grad():
        tol = (K * 2.0 ** -23 * (h64[:64].abs() @ w64.abs().t()).max() / 1.5 + 2.0 ** -20 * (1 + logits.abs().max())).item()
    assert (logp[live].double() - want).abs().max() <= 2 * tol
    assert (ent[live].double() - want_ent).abs().max() <= (2 + 2 * math.log(V)) * tol
    exact = torch.autograd.grad(want, (h64, w64), g[live].double())
    check_head_gradients((dh[live], dw), exact, h64, w64, logits.detach(), g[live], t[live], 1.5, tol)
    want = torch.nn.functional.cross_entropy(h64 @ w64.t(), t[live])
    assert abs(float(loss.detach()) - float(want.detach())) <= 2 * tol
    exact = torch.autograd.grad(want, (h64, w64))
    assert rel(dh2[live], exact[0]) <= 2 * STEP and rel(dw2, exact[1]) <= 2 * STEP


def test_launches_are_counted():
    from fp4_post_b200 import ops
    h, w, t = head_inputs(100, 500, 64)
    before = ops.launch_count()
    dense.token_logprobs(h, w, t)
    dense.linear(h, w)
    assert ops.launch_count() - before == 3


def test_rows_that_are_ignored():
    h, w, t = head_inputs(50, 300, 64)
    t[:] = -100
    h[7] = float("nan")                                   # a padded row may hold anything
    h.requires_grad_(True)
    w.requires_grad_(True)
    assert not dense.linear_cross_entropy(h, w, t, reduction="none").any()
    loss = dense.linear_cross_entropy(h, w, t, reduction="sum")
    assert loss == 0
    dh, = torch.autograd.grad(loss, h)
    assert not dh.any()
    assert torch.isnan(dense.linear_cross_entropy(h, w, t))
    t[3] = 5
    a = dense.linear_cross_entropy(h, w, t)
    b = dense.linear_cross_entropy(h, w, torch.where(t == -100, 299, t), ignore_index=299)
    assert torch.isfinite(a) and torch.equal(a, b)
    # int32 targets, leading dimensions
    c = dense.linear_cross_entropy(h.view(2, 25, 64), w, t.view(2, 25).int())
    assert torch.equal(a, c)


def test_targets_outside_the_vocabulary_give_nan_and_nothing_else():
    h, w, t = head_inputs(40, 300, 64, ignored=0.0)
    good = dense.linear_cross_entropy(h, w, t, reduction="none")
    for bad in (300, -1, 1 << 40, -(1 << 62)):
        u = t.clone()
        u[5] = bad
        hh = h.clone().requires_grad_(True)
        loss = dense.linear_cross_entropy(hh, w, u, reduction="none")
        assert torch.isnan(loss[5]) and torch.equal(loss[:5], good[:5]) and torch.equal(loss[6:], good[6:])
        dh, = torch.autograd.grad(loss, hh, torch.ones_like(loss))
        assert torch.isnan(dh[5]).all() and torch.isfinite(dh[:5]).all() and torch.isfinite(dh[6:]).all()


def test_extreme_logits():
    h, w, t = head_inputs(64, 1000, 64, ignored=0.0)
    big = (h.float() * 3000).bfloat16()                    # logits of thousands: one token takes it all
    logp, entropy, logits = head64(big.double(), w.double(), t, 1.0)
    got, ent = dense.token_logprobs(big, w, t, entropy=True)
    tol = 64 * 2.0 ** -23 * float((big.double().abs() @ w.double().abs().t()).max()) + 2.0 ** -20 * float(logits.abs().max())
    assert (got.double() - logp).abs().max() <= 2 * tol and torch.isfinite(ent).all() and (ent >= -1e-3).all()
    same = dense.token_logprobs(torch.zeros_like(h), w, t, entropy=True)       # all logits equal
    assert (same[0] + math.log(1000)).abs().max() <= 1e-5 and (same[1] - math.log(1000)).abs().max() <= 1e-5
    h[9, 3] = float("inf")
    got = dense.linear_cross_entropy(h, w, t, reduction="none")
    assert torch.isnan(got[9]) and torch.isfinite(got[:9]).all() and torch.isfinite(got[10:]).all()


def test_losses_of_no_rows():
    h, w, t = normal(0, 64), normal(100, 64, seed=1), torch.empty(0, dtype=torch.int64, device="cuda")
    h.requires_grad_(True)
    w.requires_grad_(True)
    assert dense.linear_cross_entropy(h, w, t, reduction="none").shape == (0,)
    loss = dense.linear_cross_entropy(h, w, t, reduction="sum")
    dh, dw = torch.autograd.grad(loss, (h, w))
    assert loss == 0 and dh.shape == h.shape and not dw.any()
    assert torch.isnan(dense.linear_cross_entropy(h, w, t))
    logp, ent = dense.token_logprobs(h, w, t, entropy=True)
    assert logp.shape == ent.shape == (0,)


# ---- refusals ---------------------------------------------------------------------------------------------------

def test_what_the_calls_refuse():
    x, w, t = normal(4, 64), normal(24, 64, seed=1), torch.zeros(4, dtype=torch.int64, device="cuda")
    y = normal(4, 24)
    cases = [(ValueError, lambda: dense.linear(x, w[:, :56])), (ValueError, lambda: dense.linear(x[:, :60].contiguous(), w[:, :60].contiguous())),
             (ValueError, lambda: dense.linear(x, w, y[0, :23])), (ValueError, lambda: dense.linear(x, w, gate=y[:1])), (ValueError, lambda: dense.linear(x, w, residual=y[0])),
             (TypeError, lambda: dense.linear(x.float(), w)), (TypeError, lambda: dense.linear(x, w.half())), (TypeError, lambda: dense.linear(x, w, y[0].half())),
             (TypeError, lambda: dense.linear(x, w, gate=y.float())), (ValueError, lambda: dense.linear(x, w, activation="tanh")),
             (ValueError, lambda: dense.linear(x, w, gate=y.cpu())), (ValueError, lambda: dense.linear(x, w[:0])),
             (ValueError, lambda: dense.linear_cross_entropy(x, w, t[:3])), (TypeError, lambda: dense.linear_cross_entropy(x, w, t.float())),
             (TypeError, lambda: dense.linear_cross_entropy(x.float(), w, t)), (TypeError, lambda: dense.linear_cross_entropy(x, w.float(), t)),
             (ValueError, lambda: dense.linear_cross_entropy(x, w, t, temperature=0.0)), (ValueError, lambda: dense.linear_cross_entropy(x, w, t, temperature=float("nan"))),
             (ValueError, lambda: dense.linear_cross_entropy(x, w.cpu(), t)), (ValueError, lambda: dense.token_logprobs(x, w, t.cpu())),
             (ValueError, lambda: dense.token_logprobs(x, w[:0], t)), (TypeError, lambda: dense.linear(x, None)), (TypeError, lambda: dense.linear(x, w, 3.0))]
    for i, (error, call) in enumerate(cases):
        with pytest.raises(error):
            call()
            raise AssertionError(f"case {i} was not refused")


# ---- how the calls are made -----------------------------------------------------------------------------------

def train_step(x, w, b, g, r, head, t, dy):
    """Everything together: a gated layer, a layer onto a residual, the loss, and all gradients."""
    h = dense.linear(x, w, b, activation="silu", gate=g)
    h = dense.linear(h, w, residual=r)
    loss = dense.linear_cross_entropy(h, head, t, temperature=0.9)
    logp, ent = dense.token_logprobs(h, head, t, entropy=True)
    grads = torch.autograd.grad((loss, logp), (x, w, b, g, r, head), (None, dy))
    return (loss.detach(), logp.detach(), ent, *grads)


def train_inputs(seed, M=300, K=256, V=1003):
    x, w, b = normal(M, K, seed=seed), normal(K, K, scale=K ** -0.5, seed=seed + 1), normal(K, seed=seed + 2)
    g, r, head = normal(M, K, seed=seed + 3), normal(M, K, seed=seed + 4), normal(V, K, scale=K ** -0.5, seed=seed + 5)
    t = torch.randint(0, V, (M,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    t[3::7] = -100
    return [v.requires_grad_(True) for v in (x, w, b, g, r, head)] + [t, normal(M, seed=seed + 6, dtype=torch.float32)]


def test_calls_together_and_again_give_the_same_bits():
    inputs = train_inputs(1)
    want = train_step(*inputs)
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(train_step(*inputs), want))
    # against torch in 64 bits: bf16 between the calls (h is rounded twice, and its gradients), so the norm of the whole goes by six roundings
    d = [v.detach().double().requires_grad_(True) for v in inputs[:6]]
    t, dy = inputs[6:]
    h = linear64(d[0], d[1], d[2], "silu", d[3], None)
    h = linear64(h, d[1], None, None, None, d[4])
    loss = torch.nn.functional.cross_entropy(h @ d[5].t() / 0.9, t)
    logp, ent, _ = head64(h, d[5], t, 1.0)
    exact = torch.autograd.grad((loss, logp), d, (None, dy.double()))
    assert rel(want[0], loss.detach()) <= 6 * STEP and rel(want[1], logp.detach()) <= 6 * STEP and rel(want[2], ent.detach()) <= 6 * STEP
    for a, e in zip(want[3:], exact):
        assert rel(a, e) <= 6 * STEP


def test_on_another_stream_and_from_several_threads():
    import threading
    inputs = train_inputs(2)
    want = train_step(*inputs)
    torch.cuda.synchronize()
    wrong = []

    def work():
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(st):
            for _ in range(10):
                got = train_step(*inputs)
                if not all(torch.equal(a, c) for a, c in zip(got, want)):
                    wrong.append(1)
    work()
    threads = [threading.Thread(target=work) for _ in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert not wrong


@pytest.mark.parametrize("M,V", [(300, 1003), (16, 5000), (2500, 300)])
def test_captured_in_graphs_that_are_replayed_in_turn(M, V):
    first, second = train_inputs(3, M=M, V=V), train_inputs(4, M=M, V=V)
    static = [train_inputs(5, M=M, V=V) for _ in range(2)]
    graphs, outs = [], []
    for s in static:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            train_step(*s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(train_step(*s))
        graphs.append(graph)
    for inputs in (first, second, first):
        want = train_step(*inputs)
        for s, graph in zip(static, graphs):
            with torch.no_grad():
                for a, c in zip(s, inputs):
                    a.copy_(c)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_backward_twice_and_a_graph_of_the_gradients():
    x, w = normal(40, 64).requires_grad_(True), normal(48, 64, seed=1).requires_grad_(True)
    y = dense.linear(x, w, activation="gelu")
    dy = normal(40, 48, seed=2)
    a = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    c = torch.autograd.grad(y, (x, w), dy)
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    t = torch.zeros(40, dtype=torch.int64, device="cuda")
    for out in (dense.linear(x, w, activation="gelu").float().sum(), dense.linear_cross_entropy(x, w, t)):
        gx, = torch.autograd.grad(out, x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            gx.float().sum().backward()
    # a saved tensor that was changed in between is noticed
    y = dense.linear(x, w)
    with torch.no_grad():
        w.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)


def test_offsets_beyond_32_bits():
    M, N, K = 70001, 32776, 8                                # 2.3 * 10^9 elements in y, gate and residual
    x, w = normal(M, K), normal(N, K, seed=1)
    g = normal(1, N, seed=2).expand(M, N).contiguous()
    y = dense.linear(x, w, activation="silu", gate=g, residual=g)
    rows = torch.tensor([0, 1, 35000, 65535, 65537, 69999, 70000], device="cuda")
    want = linear64(x[rows].double(), w.double(), None, "silu", g[rows].double(), g[rows].double())
    err = (y[rows].double() - want).abs()
    assert (err <= STEP * want.abs() + 2.0 ** -16 * (1 + g[rows].double().abs())).all()
    del y, g
    # (a vocabulary of 131080 rows and 20000 tokens: 2.6 * 10^9 logits)
    M, V, K = 20000, 131080, 8
    h, w, t = head_inputs(M, V, K)
    h.requires_grad_(True)
    loss = dense.linear_cross_entropy(h, w, t, reduction="sum")
    dh, = torch.autograd.grad(loss, h)
    rows = torch.arange(M - 300, M, device="cuda")
    h64 = h.detach()[rows].double().requires_grad_(True)
    logp, _, _ = head64(h64, w.double(), t[rows], 1.0)
    exact, = torch.autograd.grad(-logp.sum(), h64)
    assert rel(dh[rows], exact) <= 2 * STEP
    each = dense.token_logprobs(h, w, t)
    assert (each[rows].double() - logp).abs().max() <= 1e-4


def test_gradients_against_differences():
    """Central differences of the calls themselves, along random directions; steps that bf16 represents.  The loss is smooth, so that the difference over
    2 d is off by its third derivative (d^2 / 6 of it) and by the outputs' roundings over d."""
    M, N, K = 32, 40, 64
    x, w, t = normal(M, K), normal(N, K, scale=0.25, seed=1), torch.arange(M, device="cuda") % N
    x.requires_grad_(True)
    w.requires_grad_(True)
    gx, gw = torch.autograd.grad(dense.linear_cross_entropy(x, w, t, reduction="sum"), (x, w))
    for leaf, grad, other in ((x, gx, w), (w, gw, x)):
        direction = torch.randint(-1, 2, leaf.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).bfloat16()
        d = 2.0 ** -5
        moved = [(leaf.detach() + s * d * direction) for s in (1, -1)]
        real = [(m.double() - leaf.detach().double()) for m in moved]      # what bf16 made of the step
        f = [float(dense.linear_cross_entropy(*((m, other) if leaf is x else (other, m)), t, reduction="sum").double()) for m in moved]
        along = float((grad.double() * (real[0] - real[1])).sum())
        scale = float((grad.double().abs() * (real[0] - real[1]).abs()).sum())
        assert abs((f[0] - f[1]) - along) <= 0.02 * scale + 1e-3


# ---- the decoder ------------------------------------------------------------------------------------------------

@pytest.fixture()
def decoders():
    from fp4_post_b200.decoder import Decoder, DecoderConfig
    cfg = DecoderConfig(hidden=256, layers=2, heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=1003)
    torch.manual_seed(0)
    plain = Decoder(cfg, fuse_norms=False).cuda().bfloat16()
    fused = Decoder(cfg, fuse_norms=False, fuse_dense=True).cuda().bfloat16()
    fused.load_state_dict(plain.state_dict())
    return plain, fused, torch.randint(0, cfg.vocab, (3, 65), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))


def test_the_decoder_calls_them(decoders):
    from fp4_post_b200 import ops
    plain, fused, ids = decoders
    want, before = plain.loss(ids), ops.launch_count()
    loss = fused.loss(ids)
    # per block the o, gate and down projections, then the head: statistics, rows, mean
    assert ops.launch_count() - before == 2 * 3 + 3
    assert rel(loss.detach(), want.detach().double()) <= 2e-3
    want.backward()
    loss.backward()
    for (name, a), (_, c) in zip(fused.named_parameters(), plain.named_parameters()):
        # both sides round every tensor between their kernels to bf16, the plain one more of them (the logits among them)
        assert rel(a.grad, c.grad.double()) <= 0.05, name
    with torch.no_grad():
        logp, ent = fused.token_logprobs(ids, temperature=0.7, entropy=True)
        logp_p, ent_p = plain.token_logprobs(ids, temperature=0.7, entropy=True)
        # (the plain logits are rounded to bf16: 2^-8 of their size, at most 4 here, on either side of the difference)
        assert logp.shape == (3, 64) and (logp - logp_p).abs().max() <= 0.1 and (ent - ent_p).abs().max() <= 0.1
        assert torch.equal(logp, fused.token_logprobs(ids, temperature=0.7))
        assert rel(-fused.token_logprobs(ids).mean(), loss.detach().double()) <= 1e-6


def metis_decoder(fuse_dense, targets):
    import fp4_post_b200
    fp4_post_b200.install_reference_aliases()
    from fp4_post_b200.decoder import Decoder, DecoderConfig
    from grpo.grpo import MetisArgs, replace_linear_with_metis
    cfg = DecoderConfig(hidden=256, layers=2, heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=1003)
    torch.manual_seed(0)
    model = Decoder(cfg, fuse_dense=fuse_dense).cuda().bfloat16()
    args = MetisArgs(forward_svd_rank=32, activation_lowrank_svd=32, backward_lowrank_svd=32)
    args.device = "cuda"
    args.q_backward_input = args.q_backward_weight = args.q_backward_outputgrad = "nvfp4e2m1bnosr"
    replace_linear_with_metis(model, dtype=torch.bfloat16, metis_args=args, target_modules=targets, compute_dtype=torch.bfloat16)
    return model, torch.randint(0, cfg.vocab, (2, 64), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))


def test_the_decoder_with_metis_layers_and_fused_dense_steps_as_a_graph():
    from fp4_post_b200.graphs import GraphedStep
    model, ids = metis_decoder(True, None)
    params = list(model.parameters())

    def step():
        for p in params:
            p.grad = None
        loss = model.loss(ids)
        loss.backward()
        return loss
    want = float(step().detach())
    grads = [p.grad.clone() for p in params]
    runner = GraphedStep(step, warmup=1)
    loss = runner()
    torch.cuda.synchronize()
    assert float(loss.detach()) == want                     # round to nearest throughout: the same kernels, the same bits
    for p, g in zip(params, grads):
        assert torch.equal(p.grad, g)
    runner.release()


def test_the_decoder_with_some_projections_left_in_bf16():
    """o, gate and down stay plain layers beside Metis ones: fused, they are what they were but for the roundings between their kernels."""
    targets = ["q_proj", "k_proj", "v_proj", "up_proj"]
    (fused, ids), (plain, _) = metis_decoder(True, targets), metis_decoder(False, targets)
    plain.load_state_dict(fused.state_dict())
    a, c = fused.loss(ids), plain.loss(ids)
    assert rel(a.detach(), c.detach().double()) <= 5e-3
    a.backward()
    c.backward()
    for (name, p), (_, q) in zip(fused.named_parameters(), plain.named_parameters()):
        # (NVFP4 gradients: a rounding of an activation can move an element of a block by a step, an eighth of its size or more)
        assert torch.isfinite(p.grad).all() and (float(q.grad.double().norm()) < 1e-6 or rel(p.grad, q.grad.double()) <= 0.35), name
