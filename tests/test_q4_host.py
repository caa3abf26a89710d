"""Host-side rules of the rotary positions and the 4-bit cache: the angles, and
every refusal of the C entry points (NSRL_INVALID_SHAPE before any launch, so
no GPU is needed)."""
import ctypes as C
import math

import numpy as np
import pytest

import q4_plain as P


@pytest.fixture(scope="module")
def lib():
    from nsrl_b200 import build, cache, rotary
    build.build()
    cache._lib()
    L = rotary._lib()
    L.nsrl_last_error.restype = C.c_char_p
    return L


@pytest.mark.parametrize("rotary_dim", [2, 16, 64, 222])
def test_turns_are_the_rounded_frequencies(rotary_dim):
    """2^64 base^(-2i/n) / (2 pi), against doubles (relative error below 2^-48); the
    turn is a whole number of 2^-64, so its own rounding takes up to 2^-65."""
    from nsrl_b200.rotary import turns_per_position
    for i, t in enumerate(turns_per_position(rotary_dim, 500000)):
        f = 500000.0 ** (-2 * i / rotary_dim) / (2 * math.pi)
        assert abs(t / 2.0 ** 64 - f) <= f * 2.0 ** -48 + 2.0 ** -65


def test_scalings():
    from nsrl_b200.rotary import turns_per_position as turns
    n = 64
    plain = turns(n)
    assert all(abs(8 * a - b) <= 8 for a, b in zip(turns(n, scaling="linear", factor=8), plain))
    ntk = turns(n, scaling="ntk", factor=8)
    assert ntk[0] == plain[0] and abs(ntk[-1] * 8 / plain[-1] - 1) < 1e-12  # the fastest stays, the slowest by 8
    parts = turns(n, scaling="by_parts", factor=8, original_len=4096)
    for a, b in zip(parts, plain):
        over = 4096 * b / 2.0 ** 64
        if over >= 4:
            assert a == b
        elif over <= 1:
            assert abs(a * 8 - b) <= 8
        else:
            assert b / 8 < a < b


@pytest.mark.parametrize("bad", [dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=8, scaling="twice"),
                                 dict(rotary_dim=8, base=0), dict(rotary_dim=8, scaling="linear", factor=0),
                                 dict(rotary_dim=8, scaling="by_parts", factor=2)])
def test_bad_angles(bad):
    from nsrl_b200.rotary import turns_per_position
    with pytest.raises(ValueError):
        turns_per_position(**bad)


def test_the_integer_angle_is_the_angle():
    """cos and sin within 2^-27 (and half a Q30 step) of the real ones, near and far."""
    from nsrl_b200.rotary import turns_per_position
    for turn in turns_per_position(64):
        for p in (0, 1, -1, 7, 1000, 123457, 2 ** 31 - 1, -2 ** 31):
            c, s = P.cos_sin(p, turn)
            a = (p * turn % 2 ** 64) / 2.0 ** 64 * 2 * math.pi
            for got, want in ((c, math.cos(a)), (s, math.sin(a))):
                assert abs(got / 2.0 ** 30 - want) <= 2.0 ** -27 + 2.0 ** -30


def test_codes_stand_for_the_values():
    """|value - x| <= scale / 2, or below scale where the code was lowered at the top."""
    rng = np.random.default_rng(3)
    x = rng.integers(-32768, 32768, (200, 64)).astype(np.int16)
    x[0], x[1], x[2, :] = 32767, -32768, 5
    x[3] = np.where(np.arange(64) % 2, 32767, -32768)
    codes, words = P.quantise(x)
    v = P.dequantise(codes, words)
    scale = np.repeat(words.astype(np.int64) & 0xFFFF, 32, -1)
    err = np.abs(v - x)
    assert (v <= 32767).all() and (v >= -32768).all()
    low = v + scale > 32767
    assert (2 * err[~low] <= scale[~low]).all() and (err[low] < scale[low]).all()
    assert (v[0] == 32767).all() and (v[1] == -32768).all() and (v[2] == 5).all()


# ---------------------------------------------------------------- refusals ---
P16 = C.c_void_p(16)


def q4(**kw):
    from nsrl_b200.cache import Q4CacheC
    f = dict(k_codes=16, v_codes=16, k_scales=16, v_scales=16, scores=16, positions=16, batch=2, heads=4, head_dim=64,
             capacity=128)
    f.update(kw)
    return C.byref(Q4CacheC(**f))


BAD_CACHES = [dict(head_dim=32), dict(head_dim=0), dict(heads=0), dict(capacity=0), dict(capacity=100),
              dict(capacity=1 << 20), dict(k_codes=None), dict(v_scales=None), dict(k_codes=24), dict(scores=20),
              dict(batch=1 << 24)]


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_cache_refusals(lib, bad):
    c = q4(**bad)
    assert lib.nsrl_q4_cache_append(c, P16, P16, 256, 1, P16, None, None, P16, None) == 1
    assert lib.nsrl_q4_cache_read(c, None, 1, P16, P16, P16, None) == 1
    assert lib.nsrl_attention_decode_q4(P16, 256, c, P16, P16, None, 0, P16, None) == 1
    assert lib.nsrl_attention_decode_q4_workspace_size(c) == 0 and lib.nsrl_decode_block_q4_workspace_size(c) == 0
    assert lib.nsrl_q4_cache_evict(c, P16, P16, 8, 0, 0, P16, P16, P16, P16, 1 << 40, P16, None) == 1
    assert lib.nsrl_q4_cache_evict_workspace_size(c, 8) == 0
    assert b"invalid shape" in lib.nsrl_last_error()


def test_append_and_read_refusals(lib):
    good = q4()
    f = lib.nsrl_q4_cache_append
    assert f(good, P16, P16, 255, 1, P16, None, None, P16, None) == 1          # rows shorter than the heads
    assert f(good, P16, P16, 256, 129, P16, None, None, P16, None) == 1        # more tokens than slots
    assert f(good, None, P16, 256, 1, P16, None, None, P16, None) == 1
    assert f(good, P16, P16, 256, 1, None, None, None, P16, None) == 1
    assert f(good, P16, P16, 256, 1, P16, None, None, None, None) == 1
    assert f(good, P16, P16, 256, 0, P16, None, None, P16, None) == 0          # nothing to do
    assert f(q4(batch=0), None, None, 256, 1, None, None, None, None, None) == 0
    assert lib.nsrl_q4_cache_read(good, None, 129, P16, P16, P16, None) == 1
    assert lib.nsrl_q4_cache_read(good, None, 1, C.c_void_p(8), P16, P16, None) == 1
    assert lib.nsrl_q4_cache_read(good, None, 1, None, P16, P16, None) == 1


def test_attend_refusals(lib):
    f = lib.nsrl_attention_decode_q4
    assert f(P16, 255, q4(), P16, P16, None, 0, P16, None) == 1
    for i in (0, 3, 4, 7):
        args = [P16, 256, q4(), P16, P16, None, 0, P16, None]
        args[i] = None
        assert f(*args) == 1
    assert f(None, 256, q4(batch=0), None, None, None, 0, None, None) == 0
    big = q4(batch=4, capacity=65536)  # takes a workspace
    ws = lib.nsrl_attention_decode_q4_workspace_size(big)
    assert ws >= 4 * 16 * 65536
    for w, n in ((None, ws), (P16, ws), (C.c_void_p(256), ws - 1)):
        assert f(P16, 256, big, P16, P16, w, n, P16, None) == 1


def test_evict_refusals(lib):
    f = lib.nsrl_q4_cache_evict
    ws = lib.nsrl_q4_cache_evict_workspace_size(q4(), 32)
    assert ws > 0
    for keep in (0, 129):
        assert f(q4(), P16, P16, keep, 0, 0, P16, P16, P16, P16, 1 << 40, P16, None) == 1
    assert f(q4(), P16, P16, 32, 0, 0, P16, P16, P16, P16, ws - 1, P16, None) == 1
    assert f(q4(), P16, P16, 32, 0, 0, P16, P16, P16, None, ws, P16, None) == 1
    assert f(q4(), P16, P16, 32, 0, 0, P16, P16, P16, C.c_void_p(8), ws, P16, None) == 1
    assert f(q4(scores=None), P16, P16, 32, 0, 0, P16, P16, P16, P16, ws, P16, None) == 1
    assert f(q4(positions=None), P16, P16, 32, 0, 0, P16, P16, P16, P16, ws, P16, None) == 1
    assert f(q4(), P16, P16, 32, 1 << 31, 0, P16, P16, P16, P16, ws, P16, None) == 1
    assert f(q4(), None, P16, 32, 0, 0, P16, P16, P16, P16, ws, P16, None) == 1


def test_rotary_refusals(lib):
    from nsrl_b200.rotary import RotaryC
    f = lib.nsrl_rotary_rows

    def call(x=P16, rows=4, heads=2, hd=64, ldx=128, rot=RotaryC(16, 64, 0, 1 << 30), pos=P16, seq=0, y=C.c_void_p(32),
             ldy=128):
        return f(x, rows, heads, hd, ldx, None if rot is None else C.byref(rot), pos, seq, 0, y, ldy, None)

    for bad in (dict(rot=None), dict(rot=RotaryC(None, 64, 0, 1 << 30)), dict(rot=RotaryC(16, 63, 0, 1 << 30)),
                dict(rot=RotaryC(16, 0, 0, 1 << 30)), dict(rot=RotaryC(16, 66, 0, 1 << 30)),
                dict(rot=RotaryC(16, 64, 2, 1 << 30)), dict(rot=RotaryC(16, 64, 0, 0)), dict(heads=0), dict(hd=1),
                dict(hd=2000, ldx=4000, ldy=4000), dict(ldx=127), dict(ldy=127), dict(pos=None), dict(x=None),
                dict(y=None), dict(x=C.c_void_p(32), ldx=256), dict(rows=1 << 31)):
        assert call(**bad) == 1, bad
    assert call(rows=0) == 0


def test_decode_block_refusals(lib):
    from nsrl_b200.core import LinearParamsC as LP
    f = lib.nsrl_prenorm_attention_decode_block_q4
    lin = LP(16, None, 16, 256, 256)
    ws = lib.nsrl_decode_block_q4_workspace_size(q4())
    p256 = C.c_void_p(256)

    def call(x=P16, batch=2, d=256, heads=4, gamma=P16, lp=lin, cache=None, lens=P16, y=P16, w=p256, wb=ws, st=P16):
        return f(x, batch, d, heads, gamma, 1, *[C.byref(lp)] * 4, None, cache or q4(), lens, None, y, w, wb, st, None)

    for bad in (dict(batch=3), dict(heads=2), dict(lp=LP(16, None, 16, 256, 128)), dict(cache=q4(head_dim=16)),
                dict(x=None), dict(gamma=None), dict(lens=None), dict(y=None), dict(w=None), dict(w=P16), dict(wb=ws - 1),
                dict(st=None), dict(d=512)):
        assert call(**bad) == 1, bad
