"""The bf16 products and the head's losses (fp4_post_b200/dense.py) where an answer is easily lost: tokens that the model is sure of,
ignored rows that hold anything, derivatives and traces that the native calls cannot follow, waits that run out, saved tensors that come back
laid out otherwise.  The plain sides are torch in 64 bits.  A bf16 rounding is off by at most 2^-8 of the value (STEP)."""
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


# ---- tokens that the model is sure of -------------------------------------------------------------------------------

def sure_rows(M, V, K, temperature, seed=0):
    """Hidden states that lean on their token's row of the head so far that 1 - p of the target runs from 0.3 down to 1e-6, row by row."""
    w = normal(V, K, scale=K ** -0.5, seed=seed)
    t = torch.randperm(V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + 1))[:M]
    wt = w[t].double()
    direction = wt / (wt * wt).sum(dim=1, keepdim=True)                  # one unit of it is one unit of the target's logit
    want = 10.0 ** torch.linspace(math.log10(0.3), -6.0, M, device="cuda", dtype=torch.float64)
    # (the others' logits are some hundredths of it: their sum is about V)
    reach = temperature * (math.log(V) + torch.log((1 - want) / want))
    return (direction * reach[:, None]).bfloat16(), w, t


def exact_head(h, w, t, temperature):
    """log p of the target and 1 - p of it, without cancellation, and the logits, in 64 bits."""
    logits = h.double() @ w.double().t() / temperature
    others = logits.scatter(1, t[:, None], -math.inf)
    picked = logits.gather(1, t[:, None])[:, 0]
    odds = torch.logsumexp(others, dim=1) - picked                       # log((1 - p) / p)
    return -torch.nn.functional.softplus(odds), torch.sigmoid(odds), logits


def logit_error(h, w, logits, temperature, K):
    """What a logit is off by: sums of K products at 2^-23 of their magnitudes, its scaling and the logarithm's at 2^-23 each."""
    return K * 2.0 ** -23 * float((h.double().abs() @ w.double().abs().t()).max()) / temperature + 2.0 ** -21 * (1 + float(logits.abs().max()))


SURE = [(1, 97, 64), (9, 1003, 3584), (64, 1003, 256), (100, 1003, 3584), (200, 1003, 3584), (300, 2500, 512)]


@pytest.mark.parametrize("temperature", [1.0, 0.6, 1.7])
@pytest.mark.parametrize("M,V,K", SURE)
def test_log_probabilities_of_sure_tokens(M, V, K, temperature):
    """-log p = log(1 + (1 - p) / p) has the relative error of the odds, which is twice a logit's error, and of their sum, V additions of
    2^-24 at the most; it is never negative, so no log-probability is positive."""
    h, w, t = sure_rows(M, V, K, temperature)
    want, _, logits = exact_head(h, w, t, temperature)
    off = 2 * logit_error(h, w, logits, temperature, K) + V * 2.0 ** -24
    got, entropy = dense.token_logprobs(h, w, t, temperature=temperature, entropy=True)
    assert (got <= 0).all() and (entropy >= 0).all()
    assert ((got.double() - want).abs() <= 1.1 * off * want.abs()).all()
    loss = dense.linear_cross_entropy(h, w, t, temperature=temperature, reduction="none")
    assert torch.equal(loss, -got)
    # the entropy: (1 - p) / p times the others' distances, of which only the logits' differences are off
    logp = torch.log_softmax(logits, dim=1)
    exact = -(logp.exp() * logp).sum(dim=1)
    assert ((entropy.double() - exact).abs() <= 1.1 * (2 * off + 2.0 ** -20) * exact + 2.0 ** -22).all()


@pytest.mark.parametrize("M", [6, 70])
def test_a_target_of_infinite_logit_or_alone_in_its_vocabulary(M):
    h, w, t = normal(M, 64), normal(90, 64, seed=1), torch.arange(M, device="cuda")
    got = dense.token_logprobs(h, w[:1], torch.zeros_like(t), entropy=True)
    assert not got[0].any() and not got[1].any()                         # p = 1
    w[t[2]] = 0
    w[t[2], 0] = float("inf")
    h[:, 0] = h[:, 0].abs() + 1
    got = dense.token_logprobs(h, w, t)
    assert torch.isnan(got[2]) and torch.isnan(got).all()                # infinity less infinity, as a subtracted maximum has it
    w[t[2], 0] = -float("inf")
    got = dense.token_logprobs(h, w, t)
    assert got[2] == -float("inf") and torch.isfinite(got[:2]).all() and torch.isfinite(got[3:]).all()


@pytest.mark.parametrize("M", [6, 70])
def test_the_hottest_and_the_coldest_temperatures(M):
    h, w, t = normal(M, 64), normal(90, 64, seed=1), torch.arange(M, device="cuda")
    for temperature in (1e30, 1e38, 1e44):                  # all tokens alike
        got, entropy = dense.token_logprobs(h, w, t, temperature=temperature, entropy=True)
        assert (got + math.log(90)).abs().max() <= 1e-5 and (entropy - math.log(90)).abs().max() <= 1e-5
    best = (h.double() @ w.double().t()).argmax(dim=1)
    for temperature in (1e-4, 1e-20):                       # one takes it all (none is within 16 times 1e-4 of it, but for one row in a thousand)
        got = dense.token_logprobs(h, w, best, temperature=temperature)
        assert float((got > -1e-6).float().mean()) >= 0.98


def exact_logit_gradient(h, w, t, temperature):
    """softmax - one-hot over the temperature, the target's element without cancellation, in 64 bits."""
    logp, miss, logits = exact_head(h, w, t, temperature)
    return torch.softmax(logits, dim=1).scatter(1, t[:, None], -miss[:, None]) / temperature, miss, logits


def check_sure_gradients(got, G, h, w, M, off):
    """Every element of G has the relative error of its logits, and its rounding to bf16 (above 128 rows once, below in two numbers), the
    gradient its own: by elements, since a row of dh and of dw may be of any size."""
    g_off = off + (STEP if M > 128 else STEP * STEP)
    for a, want, reach in ((got[0], G @ w, G.abs() @ w.abs()), (got[1], G.t() @ h, G.abs().t() @ h.abs())):
        assert a.dtype == torch.bfloat16 and a.shape == want.shape
        assert ((a.double() - want).abs() <= STEP * want.abs() + 1.1 * g_off * reach).all()


@pytest.mark.parametrize("temperature", [1.0, 0.6])
@pytest.mark.parametrize("M,V,K", SURE)
def test_gradients_of_sure_tokens(M, V, K, temperature):
    """What a row adds is (1 - p) times a vector of its own size: each row weighed by 1 / (1 - p), all of them count alike in dw."""
    h, w, t = sure_rows(M, V, K, temperature)
    G, miss, logits = exact_logit_gradient(h, w, t, temperature)
    off = 2 * logit_error(h, w, logits, temperature, K) + V * 2.0 ** -24
    leaves = [h.requires_grad_(True), w.requires_grad_(True)]
    up = (1 / miss).float()
    h64, w64 = h.detach().double(), w.detach().double()
    for out, sign in ((dense.linear_cross_entropy(h, w, t, temperature=temperature, reduction="none"), 1.0), (dense.token_logprobs(h, w, t, temperature=temperature), -1.0)):
        with torch.no_grad():
            out.mul_(2)                                                  # the output is the caller's, to change as it likes
        check_sure_gradients(torch.autograd.grad(out, leaves, up), sign * up.double()[:, None] * G, h64, w64, M, off)
    loss = dense.linear_cross_entropy(h, w, t, temperature=temperature)
    check_sure_gradients(torch.autograd.grad(loss, leaves), G / M, h64, w64, M, off)


@pytest.mark.parametrize("M", [20, 300])
def test_the_c_call_without_kept_log_probabilities(M):
    """metis_head_backward forms the target's log-probability from lse: off by 2^-22 of the logits beside the kept one's error."""
    from fp4_post_b200 import cabi
    V, K = 777, 256
    L = cabi.lib()
    h, w, t = sure_rows(M, V, K, 1.0)
    t[1::5] = -100
    live = t != -100
    G, _, logits = exact_logit_gradient(h, w, t.clamp(min=0), 1.0)
    G[~live] = 0
    lse, nll, g = (torch.empty(M, device="cuda") for _ in range(3))
    g.fill_(1.0)
    ws = torch.empty(max(L.metis_head_loss_workspace_bytes(M, V, K, 0), L.metis_head_backward_workspace_bytes(M, V, K)), dtype=torch.uint8, device="cuda")
    a = cabi.HeadArgs(M=M, V=V, K=K, h=h.data_ptr(), ldh=K, w=w.data_ptr(), ldw=K, target=t.data_ptr(), ignore_index=-100, scale=1.0, lse=lse.data_ptr(),
                      workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=torch.cuda.current_stream().cuda_stream)
    assert L.metis_head_loss(a, nll.data_ptr(), None) == 0
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    assert L.metis_head_backward(a, g.data_ptr(), 1, None, dh.data_ptr(), K, dw.data_ptr(), K) == 0
    off = logit_error(h, w, logits, 1.0, K)
    h64, w64 = h.double(), w.double()
    one = torch.zeros_like(G).scatter(1, t.clamp(min=0)[:, None], 2.0 ** -21 * float(logits.abs().max())) * live[:, None]
    for got, want, reach, extra in ((dh, G @ w64, G.abs() @ w64.abs(), one @ w64.abs()), (dw, G.t() @ h64, G.abs().t() @ h64.abs(), one.t() @ h64.abs())):
        assert ((got.double() - want).abs() <= STEP * want.abs() + 1.1 * (2 * off + V * 2.0 ** -24 + STEP) * reach + extra).all()
    assert not dh[~live].any()


# ---- ignored rows --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("M,V,K", [(1, 97, 64), (20, 97, 64), (64, 300, 136), (100, 513, 64), (128, 300, 64), (129, 300, 64), (700, 1003, 128), (4129, 131100, 1024)])
def test_ignored_rows_may_hold_anything(M, V, K):
    """The same bits as with zeros there, on either side of every rule of size (the last is long enough for the rows to be packed)."""
    h, w = normal(M, K), normal(V, K, scale=K ** -0.5, seed=1)
    gen = torch.Generator(device="cuda").manual_seed(2)
    t = torch.randint(0, V, (M,), device="cuda", generator=gen)
    off = torch.rand(M, device="cuda", generator=gen) < 0.4
    off[0] = True
    t[off] = -100
    bad = h.clone()
    bad[off] = torch.tensor([float("nan"), float("inf"), -float("inf"), 3.3e38], device="cuda").bfloat16()[torch.arange(int(off.sum()) * K, device="cuda") % 4].view(-1, K)
    h[off] = 0
    g = normal(M, seed=9, dtype=torch.float32)
    w.requires_grad_(True)
    got = []
    for x in (h, bad):
        x.requires_grad_(True)
        loss = dense.linear_cross_entropy(x, w, t, reduction="sum")
        logp, ent = dense.token_logprobs(x, w, t, entropy=True)
        got.append((loss.detach(), logp.detach(), ent, *torch.autograd.grad(loss, (x, w)), *torch.autograd.grad(logp, (x, w), g), *torch.autograd.grad(dense.linear_cross_entropy(x, w, t), w)))
    for a, b in zip(*got):
        assert torch.equal(a, b) and torch.isfinite(a).all()


# ---- the decoder where torch has to see the operations ---------------------------------------------------------------

@pytest.fixture()
def decoders():
    from fp4_post_b200.decoder import Decoder, DecoderConfig
    cfg = DecoderConfig(hidden=256, layers=2, heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=1003)
    torch.manual_seed(0)
    plain = Decoder(cfg, fuse_norms=False).cuda().bfloat16()
    fused = Decoder(cfg, fuse_norms=False, fuse_dense=True).cuda().bfloat16()
    fused.load_state_dict(plain.state_dict())
    return plain, fused, torch.randint(0, cfg.vocab, (3, 65), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))


def mlp(model):
    return lambda h: model.layers[0].mlp(h)


@pytest.mark.parametrize("record", [False, True])
def test_forward_mode_derivatives_pass_through_the_fused_decoder(decoders, record):
    from torch.autograd import forward_ad
    plain, fused, ids = decoders
    h, dh = normal(3, 65, 256), normal(3, 65, 256, seed=1)
    got = []
    for model in (plain, fused):
        model.hidden = lambda ids: forward_ad.make_dual(h, dh)
        with forward_ad.dual_level(), torch.set_grad_enabled(record):
            outs = (model.layers[0].mlp(forward_ad.make_dual(h, dh)), model.loss(ids), model.token_logprobs(ids))
            got.append([t for out in outs for t in forward_ad.unpack_dual(out)])
    for a, b in zip(*got):
        assert a is not None and torch.equal(a, b)


def test_traces_and_transforms_of_the_fused_decoder_are_those_of_the_plain_one(decoders):
    from torch.fx.experimental.proxy_tensor import make_fx
    plain, fused, _ = decoders
    h, other = normal(3, 65, 256), normal(3, 65, 256, seed=1)
    with torch.no_grad():
        traced = torch.jit.trace(fused.layers[0].mlp, (h,), check_trace=False)
        as_graph = make_fx(mlp(fused))(h)
    want = plain.layers[0].mlp(other).detach()             # (with gradients on: silu and product are torch's, as those of a trace are)
    assert torch.equal(traced(other), want) and torch.equal(as_graph(other), want)
    assert torch.equal(torch.vmap(mlp(fused))(torch.stack((other, h))), torch.vmap(mlp(plain))(torch.stack((other, h))))
    grads = [torch.func.grad(lambda x: mlp(m)(x).float().sum())(other) for m in (plain, fused)]
    assert torch.equal(*grads)


def test_hooks_of_plain_layers_run_in_the_fused_decoder(decoders):
    plain, fused, ids = decoders
    ran = {}
    names = ["self_attn.o_proj", "mlp.gate_proj", "mlp.down_proj", "lm_head"]

    def layers(model):
        return [model.layers[0].get_submodule(n) if n != "lm_head" else model.lm_head for n in names]
    for model in (plain, fused):
        for name, m in zip(names, layers(model)):
            m.register_forward_hook(lambda m, args, out, key=(model, name): (ran.update({key: 1 + ran.get(key, 0)}), 1.25 * out)[1])
            m.register_full_backward_hook(lambda m, gi, go, key=(model, name, "backward"): ran.update({key: 1 + ran.get(key, 0)}))
    want, loss = plain.loss(ids), fused.loss(ids)
    want.backward()
    loss.backward()
    plain.token_logprobs(ids), fused.token_logprobs(ids)
    for name in names:
        assert ran[plain, name] == ran[fused, name] == 2 and ran[plain, name, "backward"] == ran[fused, name, "backward"] == 1
    # (the second block of the fused one runs on dense.py: roundings between its kernels, as in the decoder's own comparison)
    assert abs(float(loss.detach()) - float(want.detach())) <= 2e-3 * float(want.detach())


def test_a_weight_that_a_hook_makes_is_the_one_that_is_used(decoders):
    """weight_norm keeps the layer's type and puts its weight together in a hook in front of forward."""
    plain, fused, ids = decoders
    for model in (plain, fused):
        for m in (model.layers[0].mlp.gate_proj, model.layers[1].self_attn.o_proj, model.lm_head):
            torch.nn.utils.weight_norm(m)
            with torch.no_grad():
                m.weight_g.mul_(3)                          # (the weight of the last forward pass is stale now)
    with torch.no_grad():
        for model in (plain, fused):
            model.layers[0].mlp.down_proj.weight.zero_()    # (nothing on dense.py stays between the two that rounds apart)
            model.layers[1].mlp.down_proj.weight.zero_()
            model.layers[0].self_attn.o_proj.weight.zero_()
        assert torch.equal(plain.loss(ids), fused.loss(ids))
        assert torch.equal(plain.token_logprobs(ids), fused.token_logprobs(ids))
        for model in (plain, fused):
            model.layers[0].mlp.down_proj.weight.copy_(torch.eye(256, 512))
        h = normal(2, 5, 256)
        a, b = plain.layers[0].mlp(h), fused.layers[0].mlp(h)
        assert a.any() and torch.equal(a, b)                # one product by 1: no rounding of the down projection's


def test_function_transforms_are_refused():
    x, w, b, t = normal(3, 40, 64), normal(48, 64, seed=1), normal(3, 48, seed=2), torch.arange(40, device="cuda")
    calls = [(lambda v: dense.linear(v, w), x), (lambda v: dense.linear(x[0], w, v), b), (lambda v: dense.linear(x[0], w, residual=v), normal(3, 40, 48)),
             (lambda v: dense.linear(x[0], v), normal(3, 48, 64)), (lambda v: dense.token_logprobs(v, w, t), x), (lambda v: dense.token_logprobs(x[0], w, v), t.expand(3, 40).contiguous())]
    for call, batch in calls:
        with pytest.raises(RuntimeError):
            torch.vmap(call)(batch)
        if batch.is_floating_point():
            with pytest.raises(RuntimeError):
                torch.func.grad(lambda v: call(v).float().sum())(batch[0])
            with pytest.raises(RuntimeError):
                torch.func.jvp(call, (batch[0],), (batch[0],))


# ---- errors of the library ---------------------------------------------------------------------------------------------

def test_errors_of_the_library_are_raised_with_their_number():
    """In the call and, on a thread of autograd's, in its backward pass."""
    import ctypes as C
    from fp4_post_b200 import cabi
    L, host = cabi.lib(), cabi.dense_host()
    x, w, t = normal(40, 64).requires_grad_(True), normal(48, 64, seed=1).requires_grad_(True), torch.arange(40, device="cuda")
    calls = {"metis_linear": lambda: dense.linear(x, w), "metis_head_loss_keep": lambda: dense.linear_cross_entropy(x, w, t),
             "metis_linear_pointwise": lambda: torch.autograd.grad(dense.linear(x, w, activation="silu"), x, normal(40, 48)),
             "metis_bf16_product": lambda: torch.autograd.grad(dense.linear(x, w), x, normal(40, 48)),
             "metis_head_backward_kept": lambda: torch.autograd.grad(dense.linear_cross_entropy(x, w, t), x)}
    for name, call in calls.items():
        refuse = C.CFUNCTYPE(C.c_int32)(lambda: -7)
        assert host.bind(name, C.cast(refuse, C.c_void_p).value)
        try:
            with pytest.raises(RuntimeError, match=f"{name}: status -7"):
                call()
        finally:
            host.bind(name, C.cast(getattr(L, name), C.c_void_p).value)
        call()


# ---- the status word -------------------------------------------------------------------------------------------------

def calls_with(status, M):
    """Every call with a status word, and its backward pass."""
    x, w, y = normal(M, 64), normal(104, 64, scale=0.125, seed=1), normal(M, 104, seed=2)
    t = torch.arange(M, device="cuda") % 104
    for v in (x, w, y):
        v.requires_grad_(True)
    out = dense.linear(x, w, activation="silu", gate=y, status=status)
    torch.autograd.grad(out, (x, w, y), normal(M, 104, seed=3))
    torch.autograd.grad(dense.linear_cross_entropy(x, w, t, status=status), (x, w))
    logp, _ = dense.token_logprobs(x, w, t, entropy=True, status=status)
    torch.autograd.grad(logp.sum(), (x, w))
    with torch.no_grad():
        dense.linear(x, w, status=status)
        dense.linear(x[:, ::2].repeat(1, 2), w.t().contiguous().t(), status=status)      # (copied before it is read)
        dense.linear_cross_entropy(x, w, t.int(), status=status)


@pytest.fixture()
def entries():
    """Entry points bound to functions that note the status they are given and go on to the library."""
    import ctypes as C
    from fp4_post_b200 import cabi
    L, host, seen, keep = cabi.lib(), cabi.dense_host(), [], []

    def put(name, types, status):
        real = getattr(L, name)

        def noted(*args):
            seen.append((name, status(args)))
            return real(*args)
        keep.append(C.CFUNCTYPE(C.c_int32, *types)(noted))
        assert host.bind(name, C.cast(keep[-1], C.c_void_p).value)
    vp, i32, i64, of_args = C.c_void_p, C.c_int32, C.c_int64, lambda a: a[0].contents.status
    put("metis_linear", [C.POINTER(cabi.LinearArgs)], of_args)
    put("metis_bf16_product", [vp, i32, i64, vp, i64, i64, i64, i64, i32, vp, i64, vp, i64, vp, vp], lambda a: a[13])
    put("metis_head_loss_keep", [C.POINTER(cabi.HeadArgs), vp, vp, vp], of_args)
    put("metis_head_backward_kept", [C.POINTER(cabi.HeadArgs), vp, vp, i32, vp, vp, i64, vp, i64], of_args)
    yield seen
    for name in ("metis_linear", "metis_bf16_product", "metis_head_loss_keep", "metis_head_backward_kept"):
        host.bind(name, C.cast(getattr(L, name), C.c_void_p).value)


@pytest.mark.parametrize("M", [40, 300])
def test_every_launch_that_waits_has_the_callers_status_word(entries, M):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    calls_with(status, M)
    torch.cuda.synchronize()
    assert {at for _, at in entries} == {status.data_ptr()} and {n for n, _ in entries} == {"metis_linear", "metis_bf16_product", "metis_head_loss_keep", "metis_head_backward_kept"}
    assert status.item() == 0
    entries.clear()
    calls_with(None, M)
    assert entries and {at for _, at in entries} == {None}


def test_the_status_word_may_be_set_back_between_forward_and_backward():
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    x, w = normal(40, 64).requires_grad_(True), normal(48, 64, seed=1)
    out = dense.linear(x, w, activation="gelu", status=status)
    status.zero_()
    torch.autograd.grad(out, x, normal(40, 48, seed=2))
    assert status.item() == 0


def test_bad_status_words_are_refused():
    x, w, t = normal(4, 64), normal(24, 64, seed=1), torch.zeros(4, dtype=torch.int64, device="cuda")
    calls = [lambda s: dense.linear(x, w, status=s), lambda s: dense.linear_cross_entropy(x, w, t, status=s), lambda s: dense.token_logprobs(x, w, t, status=s),
             lambda s: dense.token_logprobs(x[:0], w, t[:0], status=s)]
    for call in calls:
        for bad, error in ((torch.zeros(1, dtype=torch.int32), ValueError), (torch.zeros(2, dtype=torch.int32, device="cuda"), ValueError),
                           (torch.zeros(0, dtype=torch.int32, device="cuda"), ValueError), (torch.zeros(1, dtype=torch.int64, device="cuda"), TypeError), (0, TypeError)):
            with pytest.raises(error):
                call(bad)


# ---- saved tensors ---------------------------------------------------------------------------------------------------

def otherwise(t):
    """The same values the other way round in memory."""
    if t.dim() == 0:
        return t.clone()
    if t.dim() == 1:
        return torch.stack((t, t), dim=1)[:, 0]
    return t.transpose(0, -1).contiguous().transpose(0, -1)


def misaligned(t):
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:]
    return flat.copy_(t.reshape(-1)).view(t.shape)


@pytest.mark.parametrize("M,N", [(40, 96), (40, 97), (300, 97), (1, 96)])
def test_saved_tensors_that_come_back_laid_out_otherwise(M, N):
    from torch.autograd.graph import save_on_cpu, saved_tensors_hooks
    K = 64
    x, w, b, g, r = normal(M, K), normal(N, K, scale=0.125, seed=1), normal(N, seed=2), normal(M, N, seed=3), normal(M, N, seed=4)
    t, dy, dl = torch.arange(M, device="cuda") % N, normal(M, N, seed=5), normal(M, seed=6, dtype=torch.float32)
    t[M // 2] = -100
    leaves = [v.requires_grad_(True) for v in (x, w, b, g, r)]

    def step():
        y = dense.linear(x, w, b, activation="gelu", gate=g, residual=r)
        z = dense.linear(x, w)
        return (*torch.autograd.grad(y, leaves, dy), *torch.autograd.grad(z, (x, w), dy), *torch.autograd.grad(dense.linear_cross_entropy(x, w, t), (x, w)),
                *torch.autograd.grad(dense.token_logprobs(x, w, t), (x, w), dl))
    want = step()
    for hooks in (saved_tensors_hooks(lambda v: v, otherwise), saved_tensors_hooks(lambda v: v, misaligned), saved_tensors_hooks(otherwise, lambda v: v), save_on_cpu(pin_memory=True)):
        with hooks:
            got = step()
        assert all(torch.equal(a, c) for a, c in zip(got, want))
    for spoil in (lambda v: v.cpu(), lambda v: v.float() if v.dtype != torch.float32 else v.double(), lambda v: v[:0]):
        with saved_tensors_hooks(lambda v: v, spoil), pytest.raises(RuntimeError, match="saved tensor"):
            torch.autograd.grad(dense.linear(x, w, activation="silu", gate=g), (x, w, g), dy)
        with saved_tensors_hooks(lambda v: v, spoil), pytest.raises(RuntimeError, match="saved tensor"):
            torch.autograd.grad(dense.token_logprobs(x, w, t), (x, w), dl)


def test_under_activation_checkpoints():
    from torch.utils.checkpoint import checkpoint
    x, w, u, head = normal(50, 64), normal(96, 64, scale=0.125, seed=1), normal(64, 96, scale=0.1, seed=2), normal(101, 64, scale=0.125, seed=3)
    t = torch.arange(50, device="cuda")
    leaves = [v.requires_grad_(True) for v in (x, w, u, head)]

    def run(x, w, u, head):
        h = dense.linear(dense.linear(x, w, activation="silu", gate=dense.linear(x, w)), u, residual=x)
        return dense.linear_cross_entropy(h, head, t)
    want = torch.autograd.grad(run(*leaves), leaves)
    for reentrant in (False, True):
        for v in leaves:
            v.grad = None
        checkpoint(run, *leaves, use_reentrant=reentrant).backward()
        assert all(torch.equal(v.grad, c) for v, c in zip(leaves, want))
