"""What rollout.py settles without a device: rotary frequencies, and what its calls refuse."""
import ctypes as C
import math

import pytest
import torch

from fp4_post_b200 import cabi, rollout


@pytest.fixture(scope="module")
def L(built_library):
    return cabi.lib()


def test_frequencies_without_scaling():
    f, m = rollout.rotary_frequencies(8, 1e4)
    assert m == 1.0 and f == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-15)


def test_linear_scaling_divides_all_frequencies():
    plain, _ = rollout.rotary_frequencies(64, 5e5)
    f, m = rollout.rotary_frequencies(64, 5e5, dict(type="linear", factor=4.0))
    assert m == 1.0 and f == pytest.approx([x / 4 for x in plain], rel=1e-15)


def test_llama3_scaling_keeps_short_waves_and_divides_long_ones():
    plain, _ = rollout.rotary_frequencies(128, 5e5)
    f, m = rollout.rotary_frequencies(128, 5e5, dict(type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position=8192))
    assert m == 1.0
    for a, b in zip(plain, f):
        wave = 2 * math.pi / a
        if wave < 8192 / 4:
            assert b == pytest.approx(a, rel=1e-14)
        elif wave > 8192:
            assert b == pytest.approx(a / 8, rel=1e-14)
        else:
            assert a / 8 <= b <= a
    assert all(x > y for x, y in zip(f, f[1:]))


def test_yarn_scaling_interpolates_by_the_pair_and_sets_the_magnitude():
    plain, _ = rollout.rotary_frequencies(128, 1e4)
    f, m = rollout.rotary_frequencies(128, 1e4, dict(type="yarn", factor=4.0, original_max_position=4096))
    assert m == pytest.approx(0.1 * math.log(4) + 1)
    turns = [4096 * a / (2 * math.pi) for a in plain]
    for i, (a, b) in enumerate(zip(plain, f)):
        if turns[max(i - 1, 0)] > 32 and turns[min(i + 1, 63)] > 32:
            assert b == pytest.approx(a, rel=1e-14)
        if turns[max(i - 1, 0)] < 1:
            assert b == pytest.approx(a / 4, rel=1e-14)
    assert rollout.rotary_frequencies(128, 1e4, dict(type="yarn", factor=4.0, original_max_position=4096, attention_factor=1.5))[1] == 1.5


@pytest.mark.parametrize("rotary_dim, theta, scaling", [
    (7, 1e4, None), (0, 1e4, None), (8, 1.0, None), (8, math.inf, None), (8, 1e4, dict(type="ntk", factor=2.0)), (8, 1e4, dict(factor=2.0)),
    (8, 1e4, dict(type="linear")), (8, 1e4, dict(type="linear", factor=-1.0)), (8, 1e4, dict(type="linear", factor=2.0, beta_fast=1)),
    (8, 1e4, dict(type="llama3", factor=8.0)), (8, 1e4, dict(type="llama3", factor=8.0, low_freq_factor=4.0, high_freq_factor=4.0, original_max_position=8192)),
    (8, 1e4, dict(type="yarn", factor=4.0)),
])
def test_frequencies_refuse(rotary_dim, theta, scaling):
    with pytest.raises(ValueError):
        rollout.rotary_frequencies(rotary_dim, theta, scaling)


def test_turns_are_fractions_of_a_turn_in_64_bits():
    r = rollout.Rotary(16, theta=1e4, device="cpu")
    for i, t in enumerate(r.turns.tolist()):
        assert (t % 2 ** 64) / 2 ** 64 == pytest.approx(1e4 ** (-2 * i / 16) / (2 * math.pi), rel=1e-14)
    # positions far out: the whole-number product is the angle modulo a turn, where one in doubles has lost it
    p = 2 ** 40 + 12345
    angle = (p * r.turns[3].item()) % 2 ** 64 / 2 ** 64
    from decimal import Decimal, getcontext
    getcontext().prec = 60
    pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
    f = Decimal(1e4 ** (-6 / 16) / (2 * math.pi))
    assert abs(f - Decimal(1e4) ** (Decimal(-6) / 16) / (2 * pi)) < Decimal(2) ** -52
    assert abs(Decimal(angle) - (f * p) % 1) < Decimal(2) ** -23


@pytest.mark.parametrize("kw", [dict(head_dim=12), dict(head_dim=264), dict(head_dim=0), dict(head_dim=64, rotary_dim=66), dict(head_dim=64, rotary_dim=3)])
def test_rotary_refuses_sizes(kw):
    with pytest.raises(ValueError):
        rollout.Rotary(**kw, device="cpu")


def test_cpu_tensors_are_refused(built_library):
    r = rollout.Rotary(16, device="cpu")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        r(torch.zeros(2, 1, 16))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        rollout.sample(torch.zeros(2, 8), torch.zeros(2))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        rollout.PagedCache(1, 1, 16, pages=4, sequences=2, max_length=32, device="cpu")
    with pytest.raises(TypeError, match="logits must be a tensor"):
        rollout.sample([1.0], torch.zeros(1))
    with pytest.raises(TypeError, match="pool must be a tensor"):
        rollout.PagedCache.of(None, None, None, None)


def aligned(n=4096):
    buf = (C.c_uint8 * n)()
    p = C.addressof(buf)
    return buf, p + (-p) % 256


def cache_args(p, **kw):
    c = cabi.CacheArgs(pool=p, pages=4, layers=1, kv_heads=2, page_size=16, head_dim=64, dtype=cabi.DTYPE_BF16, tables=p, sequences=2, width=2, lengths=p, refs=p, status=p)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("kw, rc", [
    (dict(), 0), (dict(pool=None), -1), (dict(tables=None), -1), (dict(lengths=None), -1), (dict(refs=None), -1), (dict(status=None), -1), (dict(dtype=1), -1),
    (dict(dtype=cabi.DTYPE_E4M3), -1), (dict(pages=0), -2), (dict(pages=1 << 31), -2), (dict(layers=0), -2), (dict(kv_heads=0), -2), (dict(sequences=0), -2),
    (dict(sequences=(1 << 17) + 1), -2), (dict(width=0), -2), (dict(width=1 << 28), -7), (dict(page_size=8), -2), (dict(page_size=24), -2), (dict(head_dim=20), -2),
    (dict(head_dim=264), -2), (dict(head_dim=0), -2),
])
def test_caches_are_checked(L, kw, rc):
    buf, p = aligned()
    assert L.metis_cache_check(C.byref(cache_args(p, **kw))) == rc
    if "pool" not in kw:
        assert L.metis_cache_check(C.byref(cache_args(p, **{**kw, "pool": p + 8}))) == (rc or -3)


def test_a_scale_goes_with_8_bits_alone(L):
    buf, p = aligned()
    assert L.metis_cache_check(C.byref(cache_args(p, scales=p))) == -1
    assert L.metis_cache_check(C.byref(cache_args(p, scales=p, dtype=cabi.DTYPE_E4M3))) == 0
    assert L.metis_cache_check(None) == -1


def test_entry_points_reject_bad_arguments_without_a_device(L):
    buf, p = aligned()
    c = cache_args(p)
    ws = L.metis_cache_workspace_bytes(C.byref(c), 3)
    assert ws > 0 and L.metis_cache_workspace_bytes(None, 3) == 0
    reserve = lambda n=3, w=p, b=ws: L.metis_cache_reserve(C.byref(c), p, None, 1, 0, n, w, b, None)
    assert reserve(n=0) == -2 and reserve(w=None) == -1 and reserve(w=p + 4) == -1 and reserve(b=ws - 1) == -4
    assert L.metis_cache_fork(C.byref(c), None, p, 0, 3, 1, p, ws, None) == -1
    assert L.metis_cache_fork(C.byref(c), p, p, 0, 3, 1, p, ws - 1, None) == -4
    assert L.metis_cache_free(C.byref(c), p, 0, 0, None) == -2
    assert L.metis_cache_compact(C.byref(c), None, p, ws, None) == -1

    def rotary(**kw):
        a = cabi.RotaryArgs(tokens=2, inner=2, heads_q=1, heads_k=0, head_dim=16, rotary_dim=16, dtype=0, turns=p, magnitude=1.0, q=p, q_out=p)
        for k, v in kw.items():
            setattr(a, k, v)
        return L.metis_rotary(C.byref(a))
    assert rotary(q=None) == -1 and rotary(turns=None) == -1 and rotary(dtype=2) == -1 and rotary(heads_k=1) == -1
    assert rotary(tokens=0) == -2 and rotary(inner=0) == -2 and rotary(head_dim=20) == -2 and rotary(rotary_dim=18) == -2 and rotary(rotary_dim=7) == -2 and rotary(rotary_dim=0) == -2
    assert L.metis_rotary(None) == -1

    def append(**kw):
        a = cabi.AppendArgs(tokens=2, layer=0, heads_q=0, k=p, v=p, k_token=128, k_head=64, v_token=128, v_head=64)
        for k, v in kw.items():
            setattr(a, k, v)
        return L.metis_cache_append(C.byref(c), C.byref(a))
    assert append(k=None) == -1 and append(heads_q=2) == -1 and append(layer=1) == -2 and append(layer=-1) == -2 and append(tokens=0) == -2
    assert append(turns=p, rotary_dim=66) == -2 and append(k_token=4) == -3 and append(v=p + 8) == -3

    def attend(**kw):
        a = cabi.AttendArgs(rows=2, layer=0, heads_q=4, scale=1.0, q=p, q_row=256, q_head=64, out=p, workspace=p, workspace_bytes=16)
        for k, v in kw.items():
            setattr(a, k, v)
        return L.metis_cache_attend(C.byref(c), C.byref(a))
    assert attend(q=None) == -1 and attend(out=None) == -1 and attend(workspace=None) == -1 and attend(rows=0) == -2 and attend(heads_q=3) == -2 and attend(layer=1) == -2
    assert attend(q=p + 2) == -3 and attend(q_row=3) == -3

    def sample(**kw):
        a = cabi.SampleArgs(rows=1, vocab=8, logits=p, ld=8, dtype=0, u=p, temperature=1.0, top_p=1.0, token=p)
        for k, v in kw.items():
            setattr(a, k, v)
        return L.metis_sample(C.byref(a))
    assert sample(logits=None) == -1 and sample(u=None) == -1 and sample(token=None) == -1 and sample(dtype=2) == -1
    assert sample(rows=0) == -2 and sample(vocab=0) == -2 and sample(rows=2, ld=7) == -2 and sample(vocab=393217, ld=393217) == -7


def test_a_count_of_launches_needs_no_library():
    import subprocess
    import sys
    subprocess.run([sys.executable, "-c", "from fp4_post_b200 import cabi, ops\nassert ops.launch_count() == 0 and cabi._lib is None"], check=True, cwd=cabi.LIB_PATH.parents[2])
