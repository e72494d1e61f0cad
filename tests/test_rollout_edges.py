"""What rollout.py settles without a device, where it is easily got wrong."""
import ctypes as C
from decimal import Decimal, getcontext

import pytest
import torch

from fp4_post_b200 import cabi, rollout


def test_frequencies_are_plain_tensors_whatever_mode_they_are_made_in():
    with torch.inference_mode():
        made = rollout.Rotary(64, device="cpu")
    assert not made.turns.is_inference() and torch.equal(made.turns, rollout.Rotary(64, device="cpu").turns)


def test_a_cache_that_says_it_has_refused_sequences_has_them(built_library):
    buf = (C.c_uint8 * 4096)()
    p = C.addressof(buf) + (-C.addressof(buf)) % 256
    c = cabi.CacheArgs(pool=p, pages=4, layers=1, kv_heads=2, page_size=16, head_dim=64, dtype=cabi.DTYPE_BF16, tables=p, sequences=2, width=2, lengths=p, refs=p, status=p, flags=cabi.CACHE_HAS_REFUSED)
    assert cabi.lib().metis_cache_check(C.byref(c)) == -1
    for anything_else in (0, 1, -1, 0x52464452):
        c.flags = anything_else
        assert cabi.lib().metis_cache_check(C.byref(c)) == 0
    c.flags, c.refused = cabi.CACHE_HAS_REFUSED, p
    assert cabi.lib().metis_cache_check(C.byref(c)) == 0


@pytest.mark.parametrize("theta", [1e4, 5e5, 1e6, 1234.5])
@pytest.mark.parametrize("rotary_dim", [128, 44, 250])
def test_frequencies_are_within_2_to_the_minus_53_turns(theta, rotary_dim):
    """Against 50 digits.  theta^x is off by a step of 2^-52 or so, 2 pi and the quotient by half of one each, on at most 1 / (2 pi)."""
    getcontext().prec = 50
    log = Decimal(theta).ln()
    two_pi = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
    turns = rollout.Rotary(256, theta=theta, rotary_dim=rotary_dim, device="cpu").turns.tolist()
    assert len(turns) == rotary_dim // 2
    for i, t in enumerate(turns):
        exact = (log * -2 * i / rotary_dim).exp() / two_pi
        assert abs(Decimal(t % 2 ** 64) / 2 ** 64 - exact) <= Decimal(2) ** -53 * min(Decimal(1), 8 * exact) + Decimal(2) ** -65
