"""Refusals of the bf16 products, and the decoder's choice between them and torch's operations, that need no GPU."""
import ctypes as C

import pytest
import torch

from fp4_post_b200 import cabi, dense


@pytest.fixture(scope="module")
def L(built_library):
    return cabi.lib()


@pytest.fixture()
def p():
    buf = (C.c_uint8 * 4096)()
    yield C.addressof(buf) + (-C.addressof(buf)) % 256


def head_args(p, **changes):
    a = cabi.HeadArgs(M=4, V=40, K=16, h=p, ldh=16, w=p, ldw=16, target=p, ignore_index=-100, scale=1.0, lse=p, workspace=p, workspace_bytes=1 << 40)
    for k, v in changes.items():
        setattr(a, k, v)
    return a


def test_the_head_with_kept_log_probabilities_refuses_what_it_does_without(L, p):
    for changes, rc in ((dict(M=0), -2), (dict(K=20), -2), (dict(V=1 << 32), -7), (dict(h=None), -1), (dict(w=p + 2), -3), (dict(lse=None), -1),
                        (dict(negate=2), -1), (dict(workspace=None), -4), (dict(workspace_bytes=64), -4)):
        assert L.metis_head_loss_keep(head_args(p, **changes), p, None, p) == rc, changes
        assert L.metis_head_backward_kept(head_args(p, **changes), p, p, 0, None, p, 16, p, 16) == rc, changes
    assert L.metis_head_loss_keep(None, p, None, p) == -1 and L.metis_head_backward_kept(None, p, p, 0, None, p, 16, p, 16) == -1
    assert L.metis_head_loss_keep(head_args(p), None, None, p) == -1
    assert L.metis_head_backward_kept(head_args(p), p, None, 0, None, p, 16, p, 16) == -1
    assert L.metis_head_backward_kept(head_args(p), p, p, 1, p, p, 16, p, 16) == -1
    assert L.metis_head_backward_kept(head_args(p), p, p, 0, None, None, 16, None, 16) == -1


def test_temperatures_that_32_bits_cannot_divide_by_are_refused(L, p):
    x, w, t = torch.zeros(4, 16).bfloat16(), torch.zeros(24, 16).bfloat16(), torch.zeros(4, dtype=torch.int64)
    for temperature in (0.0, -1.0, float("inf"), float("nan"), 1e-39, 1e-300, 5e-324, 1e46, 1e300):
        with pytest.raises(ValueError, match="temperature"):
            dense.linear_cross_entropy(x, w, t, temperature=temperature)
        with pytest.raises(ValueError, match="temperature"):
            dense.token_logprobs(x, w, t, temperature=temperature)
    for scale in (0.0, -1.0, float("inf"), float("nan"), 3e38):
        assert L.metis_head_loss(head_args(p, scale=scale), p, None) == -1
        assert L.metis_head_backward(head_args(p, scale=scale), p, 0, None, p, 16, p, 16) == -1


def test_what_torch_would_not_see_is_refused(built_library):
    """Forward-mode derivatives and traces: the calls would return without a tangent, or as a constant of the trace."""
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w, b, y = torch.zeros(4, 16), torch.zeros(24, 16), torch.zeros(24), torch.zeros(4, 24)
    x, w, b, y = (t.bfloat16() for t in (x, w, b, y))
    t = torch.zeros(4, dtype=torch.int64)
    calls = [lambda x, w, b, y: dense.linear(x, w, b, gate=y, residual=y), lambda x, w, b, y: dense.linear_cross_entropy(x, w, t), lambda x, w, b, y: dense.token_logprobs(x, w, t)]
    for call in calls:
        for i in range(2):
            with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
                call(*(forward_ad.make_dual(v, torch.ones_like(v)) if j == i else v for j, v in enumerate((x, w, b, y))))
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, (x, w, b, y), check_trace=False)
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(call)(x, w, b, y)
    for kind in ("bias", "gate", "residual"):
        v = dict(bias=b, gate=y, residual=y)[kind]
        with forward_ad.dual_level(), torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            dense.linear(x, w, **{kind: forward_ad.make_dual(v, torch.ones_like(v))})

    class Logged(torch.Tensor):
        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    with pytest.raises(RuntimeError, match="subclass"):
        dense.linear(torch.Tensor._make_subclass(Logged, x), w)
    # outside of all that they are refused as before
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        dense.linear(x, w)


def test_launches_are_counted_without_the_library(monkeypatch, tmp_path):
    from fp4_post_b200 import ops
    monkeypatch.setattr(cabi, "_lib", None)
    monkeypatch.setattr(cabi, "LIB_PATH", tmp_path / "none.so")
    assert ops.launch_count() == sum(ops.LAUNCHES.values())


def test_the_native_modules_put_numbers_into_messages(tmp_path):
    """Beside torch: with a C++ runtime of its own such a module ends the process (hence one of its own here)."""
    import subprocess
    import sys
    from fp4_post_b200 import build
    source, target = tmp_path / "numbers.cpp", tmp_path / "numbers.so"
    source.write_text('#include <sstream>\n#include <string>\n'
                      'extern "C" const char* say(long n) { static std::string s; std::ostringstream o; o << "status " << n << " " << 1.5; s = o.str(); return s.c_str(); }\n')
    subprocess.run(build._host_command(source, target), check=True)
    code = f"import torch, ctypes; f = ctypes.CDLL({str(target)!r}).say; f.restype = ctypes.c_char_p; f.argtypes = [ctypes.c_long]; print(f(-7).decode())"
    assert subprocess.run([sys.executable, "-c", code], check=True, stdout=subprocess.PIPE, text=True).stdout.strip() == "status -7 1.5"


# ---- the decoder ---------------------------------------------------------------------------------------------------

def tiny(**options):
    from fp4_post_b200.decoder import Decoder, DecoderConfig
    torch.manual_seed(0)
    model = Decoder(DecoderConfig(hidden=64, layers=2, heads=4, kv_heads=2, head_dim=16, ffn=128, vocab=97), **options)
    return model, torch.randint(0, 97, (2, 12))


@pytest.mark.parametrize("fuse", [False, True])
def test_hooks_see_the_branches_of_a_block_without_the_residual(fuse):
    model, ids = tiny(fuse_dense=fuse)
    want = model(ids)
    block, seen = model.layers[0], {}
    handles = [m.register_forward_hook(lambda m, args, out, name=name: seen.update({name: (len(args), out)})) for name, m in (("attn", block.self_attn), ("mlp", block.mlp))]
    x = model.embed_tokens(ids)
    cos, sin = model.rotary(ids.shape[1], ids.device, x.dtype)
    out = block(x, cos, sin)
    for handle in handles:
        handle.remove()
    (n_attn, a), (n_mlp, b) = seen["attn"], seen["mlp"]
    assert n_attn == 3 and n_mlp == 1
    h = x + block.self_attn(block.input_layernorm(x), cos, sin)
    assert torch.equal(a, block.self_attn(block.input_layernorm(x), cos, sin)) and torch.equal(b, block.mlp(block.post_attention_layernorm(h)))
    assert torch.equal(out, x + a + b) and torch.equal(model(ids), want)
    seen.clear()
    with torch.nn.modules.module.register_module_forward_hook(lambda m, args, out: seen.update({id(m): out})):
        block(x, cos, sin)
    assert torch.equal(seen[id(block.self_attn)], a) and torch.equal(seen[id(block.mlp)], b)


@pytest.mark.parametrize("fuse", [False, True])
def test_modules_put_in_the_place_of_a_blocks_own(fuse):
    model, ids = tiny(fuse_dense=fuse)
    want, block = model(ids), model.layers[1]

    class Twice(torch.nn.Module):                           # what stood there, through the arguments that it takes
        def __init__(self, inner):
            super().__init__()
            self.inner = inner

        def __getattr__(self, name):
            return getattr(super().__getattr__("inner"), name) if name != "inner" else super().__getattr__(name)

        def forward(self, *args):
            assert len(args) in (1, 3)
            return self.inner(*args)
    block.self_attn, block.mlp = Twice(block.self_attn), Twice(block.mlp)
    assert torch.equal(model(ids), want)
    inner = model.layers[0].mlp.forward
    model.layers[0].mlp.forward = lambda h: inner(h)        # a forward of the instance's own
    assert torch.equal(model(ids), want)


@pytest.mark.parametrize("fuse", [False, True])
def test_the_loss_is_that_of_an_overridden_forward(fuse):
    from fp4_post_b200.decoder import Decoder

    class Cold(Decoder):
        def forward(self, ids):
            return super().forward(ids) * 0.5
    model, ids = tiny(fuse_dense=fuse)
    want = torch.nn.functional.cross_entropy(0.5 * model(ids)[:, :-1].reshape(-1, 97), ids[:, 1:].reshape(-1))
    plain = model.loss(ids)
    model.__class__ = Cold
    assert torch.equal(model.loss(ids), want) and not torch.equal(want, plain)
    torch.testing.assert_close(-model.token_logprobs(ids).mean(), want)
    model.__class__ = Decoder
    forward = model.forward
    model.forward = lambda ids: forward(ids) * 0.5
    assert torch.equal(model.loss(ids), want)
