"""Refusals of the bf16 products and the head's losses that need no GPU: the C entry points reject what they cannot run before they touch
the device, the Python calls reject it before they reach them."""
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


def linear_args(p, **changes):
    a = cabi.LinearArgs(M=4, N=24, K=16, x=p, ldx=16, w=p, ldw=16, y=p, ldy=24)
    for k, v in changes.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("changes,rc", [
    (dict(M=0), -2), (dict(N=0), -2), (dict(K=0), -2), (dict(K=-8), -2), (dict(K=12), -2), (dict(M=1 << 31), -7), (dict(N=1 << 33), -7),
    (dict(x=None), -1), (dict(w=None), -1), (dict(y=None), -1), (dict(ldx=8), -3), (dict(ldx=20), -3), (dict(ldw=12), -3), (dict(ldy=23), -1),
    (dict(activation=4), -1), (dict(activation=-1), -1)])
def test_linear_refuses(L, p, changes, rc):
    assert L.metis_linear(linear_args(p, **changes)) == rc and L.metis_last_error_string()


def test_linear_refuses_bad_parts_of_the_epilogue(L, p):
    assert L.metis_linear(None) == -1
    assert L.metis_linear(linear_args(p, x=p + 2)) == -3
    assert L.metis_linear(linear_args(p, w=p + 8)) == -3
    assert L.metis_linear(linear_args(p, bias=p, bias_dtype=7)) == -1
    assert L.metis_linear(linear_args(p, y=p + 1)) == -3 and L.metis_linear(linear_args(p, bias=p + 2, bias_dtype=1)) == -3
    for name, ld in (("gate", "ldgate"), ("residual", "ldr")):
        assert L.metis_linear(linear_args(p, **{name: p + 1, ld: 24})) == -3
        assert L.metis_linear(linear_args(p, **{name: p, ld: 23})) == -1
    for name, ld in (("act", "ldact"), ("slope", "ldslope")):                         # rows of 16-byte pieces
        for at, pitch in ((p + 2, 24), (p + 8, 24), (p, 16), (p, 28)):
            assert L.metis_linear(linear_args(p, activation=1, **{name: at, ld: pitch})) == -3
    assert L.metis_linear(linear_args(p, activation=0, slope=p, ldslope=24)) == -1    # nothing that has a slope


def test_pointwise_refuses(L, p):
    def call(**changes):
        a = cabi.LinearPointwiseArgs(M=4, N=24, dy=p, lddy=24, act=p, ldact=24, slope=p, ldslope=24, dz=p, lddz=24)
        for k, v in changes.items():
            setattr(a, k, v)
        return L.metis_linear_pointwise(a)
    assert L.metis_linear_pointwise(None) == -1
    assert call(M=0) == -2 and call(N=-1) == -2 and call(dy=None) == -1 and call(dz=None) == -1
    assert call(act=p + 2) == -3 and call(ldact=20) == -3 and call(slope=p + 8) == -3 and call(ldslope=16) == -3
    assert call(lddy=8) == -1 and call(lddz=8) == -1 and call(gate=p, ldgate=8) == -1 and call(dgate=p, lddg=2) == -1
    assert call(dbias=p, dbias_dtype=5) == -1 and call(half=4) == -1 and call(half=-8) == -1 and call(half=136) == -1 and call(M=9, half=8) == -1
    assert call(dz=p + 2) == -3 and call(lddz=28) == -3 and call(dy=p + 1) == -3          # dz is an operand of the products behind it
    assert call(dbias=p, dbias_dtype=0) == -4                                        # no workspace
    assert call(dbias=p, dbias_dtype=0, workspace=p, workspace_bytes=16) == -4
    assert call(dbias=p, dbias_dtype=0, workspace=p + 4, workspace_bytes=1 << 30) == -4
    assert call(act=None, dgate=p, lddg=24) == -1                                    # the gate's gradient needs act(z)


def test_product_refuses(L, p):
    call = lambda a=p, mn=0, lda=16, b=p, ldb=24, M=4, N=24, K=16, half=0, d=p, ldd=24: L.metis_bf16_product(a, mn, lda, b, ldb, M, N, K, half, d, ldd, None, 0, None, None)
    assert call(M=0) == -2 and call(K=0) == -2 and call(N=1 << 31) == -7
    assert call(a=None) == -1 and call(b=None) == -1 and call(d=None) == -1
    assert call(lda=8) == -3 and call(ldb=20) == -3 and call(ldd=12) == -3 and call(a=p + 4) == -3 and call(mn=1, lda=2) == -3
    assert call(N=23) == -2                                                           # rows of whole 16-byte pieces
    assert call(M=2100, K=100000, lda=100000) == -4 and L.metis_bf16_product_workspace_bytes(2100, 24, 100000, 0, 0) > 0   # split: no workspace
    for half in (-8, 4, 12, 136):                                                    # two parts: a multiple of 8 from the rows' number to 128
        assert call(half=half) == -1 and call(mn=1, half=half) == -1
    assert call(M=17, half=16) == -1 and call(mn=1, K=24, half=16) == -1
    assert call(mn=1, M=16, K=8, half=8) == -4 and L.metis_bf16_product_workspace_bytes(16, 24, 8, 1, 8) > 0        # the other operand's rows twice


def test_head_refuses(L, p):
    def args(**changes):
        a = cabi.HeadArgs(M=4, V=40, K=16, h=p, ldh=16, w=p, ldw=16, target=p, ignore_index=-100, scale=1.0, lse=p, workspace=p, workspace_bytes=1 << 40)
        for k, v in changes.items():
            setattr(a, k, v)
        return a
    bad = [(dict(M=0), -2), (dict(V=0), -2), (dict(K=20), -2), (dict(V=1 << 32), -7), (dict(h=None), -1), (dict(w=p + 2), -3), (dict(ldh=24 + 4), -3), (dict(ldw=8), -3),
           (dict(target=None), -1), (dict(lse=None), -1), (dict(negate=2), -1), (dict(workspace=None), -4), (dict(workspace=p + 8), -4), (dict(workspace_bytes=64), -4)]
    for changes, rc in bad:
        assert L.metis_head_loss(args(**changes), p, None) == rc, changes
        assert L.metis_head_backward(args(**changes), p, 0, None, p, 16, p, 16) == rc, changes
    assert L.metis_head_loss(None, p, None) == -1 and L.metis_head_backward(None, p, 0, None, p, 16, p, 16) == -1
    assert L.metis_head_loss(args(), None, None) == -1
    assert L.metis_head_backward(args(), None, 0, None, p, 16, p, 16) == -1
    assert L.metis_head_backward(args(), p, 2, None, p, 16, p, 16) == -1
    assert L.metis_head_backward(args(), p, 1, p, p, 16, p, 16) == -1                # a mean has one gradient for all rows
    assert L.metis_head_backward(args(), p, 0, None, None, 16, None, 16) == -1       # nothing asked for
    assert L.metis_head_backward(args(), p, 0, None, p, 8, p, 16) == -3 and L.metis_head_backward(args(), p, 0, None, p, 16, p + 2, 16) == -3
    assert L.metis_head_sum(None, p, -100, 4, 1, p, p, None) == -1 and L.metis_head_sum(p, p, -100, 0, 1, p, p, None) == -2
    assert L.metis_head_loss_workspace_bytes(0, 40, 16, 0) == 0 == L.metis_head_backward_workspace_bytes(4, 0, 16) == L.metis_linear_pointwise_workspace_bytes(0, 8)


def test_cpu_tensors_are_refused(built_library):
    x, w = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(24, 16, dtype=torch.bfloat16)
    t = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        dense.linear(x, w)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        dense.linear_cross_entropy(x, w, t)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        dense.token_logprobs(x, w, t)
    with pytest.raises(ValueError, match="reduction"):
        dense.linear_cross_entropy(x, w, t, reduction="average")
    with pytest.raises(ValueError, match="activation"):
        dense.linear(x, w, activation="relu6")


def test_the_decoder_with_fused_dense_layers_is_the_plain_one_on_the_cpu():
    from fp4_post_b200.decoder import Decoder, DecoderConfig
    cfg = DecoderConfig(hidden=64, layers=2, heads=4, kv_heads=2, head_dim=16, ffn=128, vocab=97)
    torch.manual_seed(0)
    plain = Decoder(cfg)
    fused = Decoder(cfg, fuse_dense=True)
    fused.load_state_dict(plain.state_dict())
    ids = torch.randint(0, cfg.vocab, (2, 12))
    assert torch.equal(plain(ids), fused(ids)) and torch.equal(plain.loss(ids), fused.loss(ids))
    logp, entropy = plain.token_logprobs(ids, temperature=0.8, entropy=True)
    assert logp.shape == entropy.shape == (2, 11)
    want = torch.log_softmax(plain(ids)[:, :-1] / 0.8, dim=-1)
    torch.testing.assert_close(logp, want.gather(-1, ids[:, 1:, None])[..., 0])
    torch.testing.assert_close(entropy, -(want.exp() * want).sum(-1))
    torch.testing.assert_close(-plain.token_logprobs(ids).mean(), plain.loss(ids))
