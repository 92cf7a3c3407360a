"""Frequency plans of the rotary positions (host arithmetic, no GPU)."""

import math
from fractions import Fraction

import pytest

from qwen3_engine_from_scratch_b200.rope import RotaryPlan, rotary_frequencies


def test_unscaled_linear_and_ntk():
    f, gain = rotary_frequencies(8, base=10000.0)
    assert gain == 1.0 and f[0] == 1.0
    assert f == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-14)
    g, _ = rotary_frequencies(8, base=10000.0, scaling="linear", factor=4.0)
    assert g == pytest.approx([v / 4 for v in f], rel=1e-15)
    g, _ = rotary_frequencies(8, base=10000.0, scaling="ntk", factor=4.0)
    assert g[0] == 1.0 and g[-1] == pytest.approx(f[-1] / 4, rel=1e-12)


@pytest.mark.parametrize("scaling", ["bands", "yarn"])
def test_bands_and_yarn_ends(scaling):
    f, _ = rotary_frequencies(128, base=1e6)
    g, gain = rotary_frequencies(128, base=1e6, scaling=scaling, factor=4.0, original_len=32768)
    assert gain == (1.0 if scaling == "bands" else pytest.approx(0.1 * math.log(4.0) + 1))
    turns = [32768 * v / (2 * math.pi) for v in f]
    for a, b, n in zip(f, g, turns):
        assert a / 4 * (1 - 1e-12) <= b <= a
        if n > 40:                      # far above fast_turns: kept
            assert b == a
        if n < 0.8:                     # below slow_turns: squeezed
            assert b == pytest.approx(a / 4, rel=1e-12)
    ratio = [b / a for a, b in zip(f, g)]
    assert all(x >= y - 1e-15 for x, y in zip(ratio, ratio[1:]))
    assert rotary_frequencies(128, base=1e6, scaling=scaling, factor=1.0, original_len=32768)[0] == \
        pytest.approx(f, rel=1e-14)


def test_fixed_point_phase():
    """position * turns modulo 2^64 is the angle's fraction of a turn."""
    plan = RotaryPlan(64, base=10000.0, device="cpu")
    for i, t in enumerate(plan.turns.tolist()):
        want = Fraction(plan.freq[i]) / Fraction(2 * math.pi)
        for position in (1, 131072, 2 ** 31 - 1, -5):
            got = Fraction((position * t) % 2 ** 64, 2 ** 64)
            off = (position * want - got) % 1
            assert min(off, 1 - off) < abs(position) * Fraction(1, 2 ** 52)


def test_refusals():
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=1.0),
                dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, scaling="linear", factor=0.5),
                dict(rotary_dim=8, scaling="yarn", factor=2.0),
                dict(rotary_dim=2, scaling="ntk", factor=2.0),
                dict(rotary_dim=8, scaling="bands", factor=2.0, original_len=64, slow_turns=4.0,
                     fast_turns=1.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)
    with pytest.raises(ValueError):
        RotaryPlan(8, layout="thirds", device="cpu")


def test_c_entry_refusals(native_lib):
    """Argument checks of the C entries come before any launch."""
    lib = native_lib
    fake, odd = 16, 18
    norm = lambda **k: lib.b200_rms_norm(*{**dict(x=fake, xs=8, r=None, rs=0, w=fake, y=fake, ys=8, s=None,  # noqa: E731
                                                  h=None, hs=0, rows=1, hidden=8, eps=1e-6, dev=None,
                                                  st=None), **k}.values())
    assert norm(rows=0) == 0
    assert norm(rows=-1) == -1 and norm(hidden=0) == -1 and norm(x=None) == -1
    assert norm(r=fake) == -1 and norm(h=fake) == -1 and norm(w=None) == -1
    lin = lambda **k: lib.b200_linear(*{**dict(x=fake, xs=64, sx=None, w=fake, ws=64, sw=None, b=None, r=None,  # noqa: E731
                                               rs=0, o=fake, os=8, m=1, n=8, k=64, fp8=0, gated=0, act=0,
                                               dev=None, st=None), **k}.values())
    assert lin(m=0) == 0
    assert lin(m=-1) == -1 and lin(n=0) == -1 and lin(k=0) == -1 and lin(act=5) == -1 and lin(act=-1) == -1
    assert lin(fp8=1) == -1 and lin(sx=fake) == -1 and lin(os=7) == -1 and lin(xs=56) == -1
    assert lin(x=odd) == -3 and lin(ws=68) == -3 and lin(r=fake, rs=7) == -1
    rot = lambda **k: lib.b200_rotary(*{**dict(  # noqa: E731
        q=fake, a=8, b=8, c=8, k=None, d=0, e=0, f=0, qo=fake, g=8, h=8, i=8, ko=None, j=0, l=0, m=0, p=fake,
        pb=0, ps=1, p64=0, t=fake, gain=1.0, batch=1, seq=1, hq=1, hk=0, dim=8, r=8, inter=0, st=None), **k}.values())
    assert rot(seq=0) == 0 and rot(hq=0) == 0
    assert rot(r=7) == -1 and rot(r=10) == -1 and rot(batch=-1) == -1 and rot(p=None) == -1
    assert rot(q=None) == -1 and rot(hk=1) == -1
    assert lib.b200_rotary_tables(None, 0, 1, 0, fake, 1.0, fake, fake, 1, 1, 8, 0, None) == -1
    assert lib.b200_rotary_tables(fake, 0, 1, 0, fake, 1.0, None, fake, 1, 1, 8, 0, None) == -1


def test_c_entry_refusals_of_unaligned_rows(native_lib):
    lib = native_lib
    few = lambda **k: lib.b200_linear_unaligned(*{**dict(  # noqa: E731
        x=18, xs=65, sx=None, w=18, ws=65, sw=None, b=None, r=None, rs=0, o=16, os=8, m=1, n=8, k=65, fp8=0,
        gated=0, act=0, dev=None, st=None), **k}.values())
    assert few(m=0) == 0 and few(m=9) == -2 and few(k=0) == -1 and few(ws=64) == -1
    pack = lambda **k: lib.b200_pack_rows(*{**dict(src=17, ss=33, dst=32, ds=48, rows=2, n=33, st=None),  # noqa: E731
                                             **k}.values())
    assert pack(rows=0) == 0 and pack(rows=-1) == -1 and pack(n=0) == -1 and pack(ds=47) == -1
    assert pack(src=None) == -1 and pack(dst=40) == -3 and pack(ds=56) == -3


def test_c_entries_of_packed_words(native_lib):
    """One array of 64-bit words: the same refusals, and sizes past 31 bits are not cut."""
    import struct
    over, fake = 2**32 + 8, 16
    call = lambda name, form, words: getattr(native_lib, name)(struct.pack(form, *words))  # noqa: E731
    norm = [fake, 8, 0, 0, fake, fake, 8, 0, 0, 0, 1, 8, 1e-6, 0, 0]
    lin = [fake, 64, 0, fake, 64, 0, 0, 0, 0, fake, 8, 1, 8, 64, 0, 0, 0, 0, 0, 0]
    rot = [fake, 8, 8, 8, 0, 0, 0, 0, fake, 8, 8, 8, 0, 0, 0, 0, fake, 0, 1, 0, fake, 1.0, 1, 1, 1, 0, 8, 8, 0, 0]
    for name, form, words, changes in (
            ("b200_rms_norm_words", "12qd2q", norm,
             [(10, 0, 0), (10, -1, -1), (0, 0, -1), (2, fake, -1), (4, 0, -1), (11, over, -1), (11, -8, -1)]),
            ("b200_linear_words", "20q", lin,
             [(11, 0, 0), (11, -1, -1), (11, over, -1), (12, over, -1), (13, over, -1), (16, 5, -1), (14, 1, -1),
              (2, fake, -1), (10, 7, -1), (0, 18, -3), (4, 68, -3)]),
            ("b200_rotary_words", "21qd8q", rot,
             [(23, 0, 0), (24, 0, 0), (27, 7, -1), (22, -1, -1), (16, 0, -1), (25, 1, -1), (22, over, -1),
              (23, over, -1), (24, over, -1), (26, over, -1), (27, over, -1)])):
        assert getattr(native_lib, name)(None) == -1
        for place, value, status in changes:
            changed = list(words)
            changed[place] = value
            assert call(name, form, changed) == status, (name, place, value)
    lin[19], lin[11] = 1, 9
    assert call("b200_linear_words", "20q", lin) == -2
