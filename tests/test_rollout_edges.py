"""What rollout.py settles without a device, where it is easily got wrong."""
import ctypes as C

import torch

from fp4_post_b200 import cabi, rollout


def test_frequencies_are_plain_tensors_whatever_mode_they_are_made_in():
    with torch.inference_mode():
        made = rollout.Rotary(64, device="cpu")
    assert not made.turns.is_inference() and torch.equal(made.turns, rollout.Rotary(64, device="cpu").turns)


def test_a_cache_that_says_it_has_refused_sequences_has_them(built_library):
    buf = (C.c_uint8 * 4096)()
    p = C.addressof(buf) + (-C.addressof(buf)) % 256
    c = cabi.CacheArgs(pool=p, pages=4, layers=1, kv_heads=2, page_size=16, head_dim=64, dtype=cabi.DTYPE_BF16, tables=p, sequences=2, width=2, lengths=p, refs=p, status=p, flags=1)
    assert cabi.lib().metis_cache_check(C.byref(c)) == -1
    c.refused = p
    assert cabi.lib().metis_cache_check(C.byref(c)) == 0
