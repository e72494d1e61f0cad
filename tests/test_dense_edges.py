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
