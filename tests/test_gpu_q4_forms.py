"""Attention over the 4-bit cache in each of its forms: CTAs of 8 and of 16 warps
at every head dim, clusters of both, the largest shares of slots, the bound of
the 32-bit accumulators, masked slots next to live ones, and arrays past 2^32
bytes."""
import numpy as np
import pytest
import torch

from oracle import oracle as O

import q4_plain as P
from test_gpu_q4_cache import K, dev, filled, gaussian, host, i32  # noqa: F401

pytestmark = pytest.mark.gpu

# one CTA of 16 warps a row (more than 2,048 slots, fewer than 888 rows), unsorted and sorted by length
FORMS = [(150, 1, 256, 2064), (75, 2, 256, 4112), (600, 1, 256, 2064), (600, 1, 64, 2064), (150, 1, 64, 4112)]
# 8 warps up to 10,240 slots from 888 rows on, 16 past that
FORMS += [(222, 4, 256, 2064), (222, 4, 64, 2064), (888, 1, 64, 10240), (888, 1, 64, 10256), (888, 1, 256, 4096)]
# clusters of 2 CTAs of 16 warps, and of 4
FORMS += [(75, 1, 256, 8192), (80, 1, 64, 16384), (40, 1, 256, 16400), (37, 2, 16, 16400)]


def check_form(K, form, scored):
    """Context and scores of the longest row, the shortest and some between."""
    B, H, hd, cap = form
    g = torch.Generator(device="cuda").manual_seed(B + cap)
    draw = lambda lo, hi, shape, t: torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32).to(t)  # noqa: E731
    groups = max(1, hd // 32)
    codes = [draw(0, 256, (B, H, cap, hd // 2), torch.uint8) for _ in "kv"]
    ks = draw(1, 9, (B, H, cap, groups), torch.int32) | (draw(-60, 1, (B, H, cap, groups), torch.int32) << 16)
    vs = draw(1, 1000, (B, H, cap, groups), torch.int32) | (draw(-9000, 1, (B, H, cap, groups), torch.int32) << 16)
    old = draw(0, 1 << 20, (B, H, cap), torch.int32)
    cache = K.Q4Cache.of(*codes, ks, vs, old.clone() if scored else None)
    lens = np.random.default_rng(cap).integers(1, cap + 1, B)
    lens[B // 3], lens[B // 2] = cap, 1
    q = draw(-40, 41, (B, H * hd), torch.int16)
    ctx = cache.attend(q, i32(lens))
    for b in sorted({0, B // 3, B // 2, int(lens.argmax()), B - 1, 7}):
        one = slice(b, b + 1)
        k, v = (P.dequantise(host(c[one]), host(s[one])) for c, s in zip(codes, (ks, vs)))
        want, scores = P.attend(host(q[one]).reshape(1, H, hd), k, v, lens[one], host(old[one]))
        assert np.array_equal(host(ctx[one]), want)
        if scored:
            assert np.array_equal(host(cache.scores[one]), scores)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("scored", [True, False])
def test_forms_equal_the_oracle(K, form, scored):
    check_form(K, form, scored)


@pytest.mark.parametrize("hd,B,cap", [(64, 150, 32768), (256, 150, 32768), (64, 19, 262144), (256, 19, 262144)])
def test_largest_shares(K, hd, B, cap):
    """32,768 slots a CTA at 64 and 256 dims: one CTA a row, and eight."""
    check_form(K, (B, 1, hd, cap), True)


@pytest.mark.parametrize("hd", [16, 64, 256])
@pytest.mark.parametrize("code", [0xFF, 0xF0, 0x0F])
def test_the_accumulators_bound(K, hd, code):
    """32,768 equal logits in one CTA: p = 1 each, so p scale = 65535 is 255 in two byte planes of every slot, and
    the s32 sums reach 255 * 255 a slot, 255 * 255 * 8,192 a warp at 256 dims.  Dims of code 15 saturate upwards
    (a wrapped sum would not), dims of code 0 come out as the zero point."""
    B, cap = 150, 32768
    p = O.attention_row(np.zeros(hd, np.int16), np.zeros((cap, hd), np.int16), np.zeros((cap, hd), np.int16), hd, hd)[2]
    assert (np.asarray(p) == 1).all()
    cache = K.Q4Cache(B, 1, hd, cap)
    cache.k_scales.fill_(1)
    cache.v_codes.fill_(code)
    cache.v_scales.fill_(-1 & 0xFFFF | (-1234 << 16))
    ctx = host(cache.attend(torch.ones((B, hd), dtype=torch.int16, device="cuda"), i32([cap] * B)))
    for odd, nibble in ((0, code & 15), (1, code >> 4)):
        want = min(32767, (cap * (-1234 + 65535 * nibble) + (1 << 14)) >> 15)
        assert (ctx[:, odd::2] == want).all()
    assert (host(cache.scores) == 1).all()


# one launch, clusters, the split form; whole units of 32 slots and what is left over
@pytest.mark.parametrize("cap", [64, 8208, 262144])
@pytest.mark.parametrize("n", [16, 13, 64, 33])
def test_masked_slots_beside_live_ones_near_the_lowest(K, cap, n):
    """All logits are -2^31 (MASKED_LOGIT: no weight) but two that are 100 and 348 above it, so that -2^31 weighs
    something unless it is left out: -32768 * 32768 on 16 of 64 dims is -2^34, >> 3; 8 * 100 and 8 * 348 on another."""
    cache = K.Q4Cache(2, 1, 64, cap)
    cache.k_scales[..., 0] = 1 | (32767 << 16)  # first group: 32767 + 1
    cache.k_codes[..., :16] = 0x11
    cache.k_scales[..., 1] = 100                # second group: 100 times the code
    rng = np.random.default_rng(n)
    values = gaussian(rng, (2, n, 64), 4096)
    codes, words = P.quantise(values)
    cache.v_codes[:, 0, :n], cache.v_scales[:, 0, :n] = dev(codes), dev(words)
    values = P.dequantise(codes, words).astype(np.int16)
    live = [(3, 1), (n - 2, 3)]
    for slot, code in live:
        cache.k_codes[:, 0, slot, 16] = code    # dim 32
    cache.k_scales[:, 0, n - 2, 1] = 116        # 348 = 3 * 116
    q = torch.zeros((2, 64), dtype=torch.int16, device="cuda")
    q[:, :16] = -32768
    q[:, 32] = 8
    before = host(cache.scores).copy()
    got = cache.attend(q, i32([n, n]))
    # the same two slots with logits 0 and -248: weights go by differences
    query, keys = np.zeros(64, np.int16), np.zeros((2, 64), np.int16)
    query[0], keys[0, 0] = 8, -248
    for b in range(2):
        want = O.attention_row(query, keys, values[b, [3, n - 2]], 64, 64)
        assert np.array_equal(host(got)[b], want[0])
        scores = before[b, 0].copy()
        scores[[3, n - 2]] += np.asarray(want[2]).astype(np.int32)
        assert want[2][0] > 0 and np.array_equal(host(cache.scores)[b, 0], scores)


def test_arrays_past_32_bits(K):
    """Codes of 4.3 GB each: append, read, attention and eviction at the end of the last row."""
    B, hd, cap = 129, 256, 262144
    assert B * cap * hd // 2 > 1 << 32
    rng = np.random.default_rng(23)
    cache = K.Q4Cache(B, 1, hd, cap)
    k, v = gaussian(rng, (2 * B, hd), 300), gaussian(rng, (2 * B, hd), 4096)
    k[-2] = k[-1]  # the last row's query weighs its two tokens alike, and nothing else
    starts = [cap - 2] * B
    assert cache.append(dev(k), dev(v), i32(starts)) is True
    kq, vq = P.quantise(k.reshape(B, 1, 2, hd)), P.quantise(v.reshape(B, 1, 2, hd))
    kr, vr = cache.read(2, i32(starts))
    assert np.array_equal(host(kr), P.dequantise(*kq)) and np.array_equal(host(vr), P.dequantise(*vq))
    assert torch.equal(cache.k_codes[-1, 0, cap - 2:], dev(kq[0])[-1, 0])
    assert int(cache.k_codes[1:, :, :cap - 2].amax()) == 0 and int(cache.k_scales[-1, :, :cap - 2].amax()) == 0
    q = gaussian(rng, (B, hd), 32)
    q[-1] = k[-1] // 8
    lens = [2] * (B - 1) + [cap]
    ctx = host(cache.attend(dev(q), i32(lens)))
    full = [np.zeros((1, 1, cap, hd), np.int16) for _ in "kv"]
    for t, new in zip(full, (kq, vq)):
        t[0, 0, -2:] = P.dequantise(*new)[-1, 0]
    want, scores = P.attend(q[-1:].reshape(1, 1, hd), *full, [cap], np.zeros((1, 1, cap), np.int32))
    assert np.array_equal(ctx[-1:], want) and (ctx[:-1] == 0).all()
    assert np.array_equal(host(cache.scores[-1:]), scores) and scores[0, 0, -2:].min() > 16000
    cache.scores.zero_()
    lens = i32([cap] * B)
    assert cache.evict(lens, lens.clone(), 16, 0, 2) is True and host(lens).tolist() == [16] * B
    for got, new in ((cache.k_codes, kq[0]), (cache.v_codes, vq[0]), (cache.k_scales, kq[1]), (cache.v_scales, vq[1])):
        assert torch.equal(got[:, :, 14:16], dev(new)) and int(got[:, :, :14].abs().max() if got.dtype == torch.int32 else got[:, :, :14].max()) == 0
    assert host(cache.positions[-1, 0, :16]).tolist() == [0] * 14 + [cap - 2, cap - 1]
