"""The 4-bit KV cache on the GPU, bit for bit: append and read against the
plain quantisation, attention against the oracle's attention rows on the
dequantised values (and against the int16 decode), eviction against the plain
selection, and a decode loop of all of them."""
import numpy as np
import pytest
import torch

from oracle import oracle as O

import q4_plain as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from nsrl_b200 import build, cache
    build.build()
    return cache


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def host(t):
    return t.cpu().numpy()


def gaussian(rng, shape, sigma):
    return np.clip(np.rint(rng.normal(0, sigma, shape)), -32768, 32767).astype(np.int16)


def filled(K, rng, B, H, hd, cap, scored=True, sk=32, sv=4096):
    """A cache whose every slot holds a quantised random row -> (cache, k values, v values)."""
    kc, ks = P.quantise(gaussian(rng, (B, H, cap, hd), sk))
    vc, vs = P.quantise(gaussian(rng, (B, H, cap, hd), sv))
    scores = dev(rng.integers(0, 1000, (B, H, cap)).astype(np.int32)) if scored else None
    pos = dev(np.tile(np.arange(cap, dtype=np.int32), (B, H, 1))) if scored else None
    return K.Q4Cache.of(dev(kc), dev(vc), dev(ks), dev(vs), scores, pos), P.dequantise(kc, ks), P.dequantise(vc, vs)


# ----------------------------------------------------------- append, read ---
# (batch, heads, head_dim, capacity, tokens, ragged, row padding)
APPENDS = [(1, 1, 16, 16, 1, False, 0), (3, 2, 64, 48, 5, True, 0), (2, 5, 256, 32, 32, False, 8),
           (4, 3, 16, 112, 33, True, 3), (2, 8, 64, 64, 17, True, 1), (70, 4, 64, 16, 1, True, 256)]


@pytest.mark.parametrize("case", APPENDS)
def test_append_and_read(K, case):
    B, H, hd, cap, n, ragged, pad = case
    rng = np.random.default_rng(n + hd)
    cache, k0, v0 = filled(K, rng, B, H, hd, cap)
    before = [host(t).copy() for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales, cache.scores,
                                       cache.positions)]
    wide = [gaussian(rng, (B * n, H * hd + pad), s) for s in (32, 12000)]
    wide[0][0, :] = 32767  # a constant group, and one over the whole range
    wide[1][0, :] = np.where(np.arange(H * hd + pad) % 2, -32768, 32767)
    starts = rng.integers(0, cap - n + 1, B)
    counts = rng.integers(0, n + 1, B) if ragged else np.full(B, n)
    first = rng.integers(0, 10 ** 6, B)
    k, v = (dev(w)[:, pad:] for w in wide)  # unaligned where pad is odd
    assert cache.append(k, v, i32(starts), i32(counts) if ragged else None, i32(first)) is True
    expect = [b.copy() for b in before]
    for b in range(B):
        for x, c, s in ((wide[0], 0, 2), (wide[1], 1, 3)):
            rows = x[b * n:b * n + counts[b], pad:].reshape(-1, H, hd).transpose(1, 0, 2)
            codes, words = P.quantise(rows)
            expect[c][b, :, starts[b]:starts[b] + counts[b]] = codes
            expect[s][b, :, starts[b]:starts[b] + counts[b]] = words
        expect[4][b, :, starts[b]:starts[b] + counts[b]] = 0
        expect[5][b, :, starts[b]:starts[b] + counts[b]] = first[b] + np.arange(counts[b])
    for got, want in zip((cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales, cache.scores, cache.positions),
                         expect):
        assert np.array_equal(host(got), want)
    kr, vr = cache.read(n, i32(starts))
    for got, c, s in ((kr, 0, 2), (vr, 1, 3)):
        want = P.dequantise(expect[c], expect[s])
        want = np.stack([want[b, :, starts[b]:starts[b] + n] for b in range(B)])
        assert np.array_equal(host(got), want)
    assert np.array_equal(host(cache.read(cap)[0]), P.dequantise(expect[0], expect[2]))


def test_append_default_positions_and_unscored(K):
    rng = np.random.default_rng(1)
    cache = K.Q4Cache(2, 2, 64, 32)
    x = gaussian(rng, (2 * 3, 128), 4096)
    assert cache.append(dev(x), dev(x), i32([4, 29])) is True
    assert host(cache.positions)[0, 0, 4:7].tolist() == [4, 5, 6] and host(cache.positions)[1, 1, 29:].tolist() == [29, 30, 31]
    plain = K.Q4Cache(2, 2, 64, 32, scored=False)
    assert plain.append(dev(x), dev(x), i32([4, 29])) is True
    assert torch.equal(plain.k_codes, cache.k_codes)


@pytest.mark.parametrize("starts,counts", [([0, -1, 3], None), ([0, 15, 3], None), ([0, 3, 3], [2, 3, 2]),
                                           ([0, 3, 3], [2, -1, 2])])
def test_append_that_does_not_fit(K, starts, counts):
    """Sequence 1 does not fit: the call is rejected, that sequence is untouched, the others are written."""
    rng = np.random.default_rng(2)
    cache = K.Q4Cache(3, 1, 64, 16)
    x = gaussian(rng, (6, 64), 4096)
    st_before = host(cache.k_codes).copy()
    assert cache.append(dev(x), dev(x), i32(starts), None if counts is None else i32(counts)) is None
    assert np.array_equal(host(cache.k_codes)[1], st_before[1])
    assert np.array_equal(host(cache.k_codes)[2, 0, 3:5], P.quantise(x[4:6])[0])


def test_read_saturates_and_refuses(K):
    cache = K.Q4Cache(1, 1, 16, 16)
    cache.k_scales.fill_(5000 | (-32768 << 16))
    cache.k_codes.fill_(0xF0)
    k, _ = cache.read(1)
    assert host(k)[0, 0, 0].tolist() == [-32768, min(32767, -32768 + 15 * 5000)] * 8
    assert cache.read(4, i32([13])) is None and cache.read(4, i32([-1])) is None
    assert cache.read(17) is None


# --------------------------------------------------------------- attention ---
ATTENDS = [(1, 1, 64, 16, [1]), (2, 3, 64, 64, [31, 33]), (3, 2, 16, 48, [1, 17, 48]), (2, 2, 256, 160, [160, 129]),
           (1, 4, 64, 1024, [1000]), (4, 16, 64, 2048, [2048, 1, 2047, 1025]), (1, 1, 16, 4096, [4095]),
           (40, 8, 64, 272, None), (160, 1, 16, 80, None), (1, 2, 256, 2064, [2050]), (2, 1, 64, 8208, [8193, 64])]
# few rows and long enough for the split form: ragged rows of one chunk, of several, and that end with or just past one
ATTENDS += [(5, 2, 64, 32784, None), (8, 1, 64, 32768, [1, 2048, 2049, 4096, 4097, 32768, 31, 256]),
            (3, 2, 16, 36880, None), (2, 2, 256, 32784, [32783, 20481]), (1, 18, 16, 34000, [33999])]
# one below that, and as long of more rows than it takes
ATTENDS += [(2, 2, 64, 32752, None), (19, 1, 16, 32768, None), (10, 2, 64, 32784, None), (130, 2, 16, 4112, None),
            (150, 1, 64, 2064, None), (75, 2, 256, 592, None)]
# rows enough to be sorted by length, and more sequences than are
ATTENDS += [(75, 8, 16, 272, None), (300, 4, 64, 48, None), (120, 8, 16, 2064, None), (150, 4, 256, 32, None),
            (2, 300, 64, 80, [3, 80]), (4100, 1, 16, 16, None)]


@pytest.mark.parametrize("case", ATTENDS)
@pytest.mark.parametrize("scored", [True, False])
def test_attend_equals_the_oracle(K, case, scored):
    from nsrl_b200 import core
    B, H, hd, cap, lens = case
    rng = np.random.default_rng(cap + hd)
    lens = rng.integers(1, cap + 1, B) if lens is None else lens
    cache, kv, vv = filled(K, rng, B, H, hd, cap, scored)
    q = gaussian(rng, (B, H, hd), 32)
    old = host(cache.scores) if scored else None
    ctx, scores = P.attend(q, kv, vv, lens, old)
    qg = dev(q.reshape(B, H * hd))
    got = cache.attend(qg, i32(lens))
    assert np.array_equal(host(got), ctx)
    if scored:
        assert np.array_equal(host(cache.scores), scores)
    rows = lambda t: dev(t.transpose(0, 2, 1, 3).astype(np.int16).reshape(B, cap, H * hd))  # noqa: E731
    assert torch.equal(got, core.attention_decode(qg, rows(kv), rows(vv), i32(lens), H, hd))


@pytest.mark.parametrize("sk,sv", [(32, 4096), (300, 30000), (4096, 4096), (1, 1)])
def test_attend_flat_and_peaked_rows(K, sk, sv):
    rng = np.random.default_rng(sk)
    cache, kv, vv = filled(K, rng, 2, 2, 64, 512, True, sk, sv)
    q = gaussian(rng, (2, 2, 64), sk)
    ctx, scores = P.attend(q, kv, vv, [512, 333], host(cache.scores))
    assert np.array_equal(host(cache.attend(dev(q.reshape(2, 128)), i32([512, 333]))), ctx)
    assert np.array_equal(host(cache.scores), scores)


def test_attend_strided_queries_and_garbage_past_the_length(K):
    """q as columns of q | k | v rows (one of them unaligned); slots past the length hold anything."""
    rng = np.random.default_rng(4)
    cache, kv, vv = filled(K, rng, 3, 2, 64, 64)
    lens = [5, 40, 63]
    for b, n in enumerate(lens):
        cache.k_scales[b, :, n:] = -1
        cache.v_scales[b, :, n:] = 0x7FFFFFFF
        cache.v_codes[b, :, n:] = 255
    for first in (0, 3):
        qkv = gaussian(rng, (3, 400), 32)
        q = qkv[:, first:first + 128]
        ctx, scores = P.attend(q.reshape(3, 2, 64), kv, vv, lens, host(cache.scores))
        assert np.array_equal(host(cache.attend(dev(qkv)[:, first:first + 128], i32(lens))), ctx)
        assert np.array_equal(host(cache.scores), scores)


def test_attend_long_stream(K):
    """More slots than one CTA's share, and a share boundary inside; a weight on every slot."""
    rng = np.random.default_rng(5)
    cap = 100000
    cache, kv, vv = filled(K, rng, 1, 1, 64, cap, True, 8, 4096)
    q = gaussian(rng, (1, 1, 64), 8)
    for n in (cap, 50001):
        ctx, scores = P.attend(q, kv, vv, [n], host(cache.scores))
        assert np.array_equal(host(cache.attend(dev(q.reshape(1, 64)), i32([n]))), ctx)
        assert np.array_equal(host(cache.scores), scores)


def test_attend_long_streams_split(K):
    """Four streams of 100,000 slots: chunks of several CTAs, added up by the last to arrive."""
    rng = np.random.default_rng(16)
    cap = 100000
    cache, kv, vv = filled(K, rng, 1, 4, 64, cap, True, 8, 4096)
    q = gaussian(rng, (1, 4, 64), 8)
    for n in (cap, 65537, 3):
        ctx, scores = P.attend(q, kv, vv, [n], host(cache.scores))
        assert np.array_equal(host(cache.attend(dev(q.reshape(1, 256)), i32([n]))), ctx)
        assert np.array_equal(host(cache.scores), scores)


@pytest.mark.parametrize("B,cap", [(150, 32768), (19, 262144), (600, 32784)])
def test_attend_largest_shares(K, B, cap):
    """32,768 slots a CTA, the most logits that one keeps: one CTA a row, and eight;
    and rows sorted by length of two CTAs each."""
    g = torch.Generator(device="cuda").manual_seed(cap)
    draw = lambda lo, hi, shape, t: torch.randint(lo, hi, shape, generator=g, device="cuda").to(t)  # noqa: E731
    kc, vc = (draw(0, 256, (B, 1, cap, 8), torch.uint8) for _ in "kv")
    ks = draw(1, 9, (B, 1, cap, 1), torch.int32) | (draw(-60, 1, (B, 1, cap, 1), torch.int32) << 16)
    vs = draw(1, 1000, (B, 1, cap, 1), torch.int32) | (draw(-9000, 1, (B, 1, cap, 1), torch.int32) << 16)
    old = draw(0, 1 << 20, (B, 1, cap), torch.int32)
    cache = K.Q4Cache.of(kc, vc, ks, vs, old.clone())
    q = draw(-40, 41, (B, 16), torch.int16)
    lens = [cap - 7 * b for b in range(B)]
    ctx = cache.attend(q, i32(lens))
    k, v = cache.read(cap)
    for b in (0, 1, B - 1):
        one = slice(b, b + 1)
        want, scores = P.attend(host(q[one]).reshape(1, 1, 16), host(k[one]), host(v[one]), lens[one], host(old[one]))
        assert np.array_equal(host(ctx[one]), want)
        assert np.array_equal(host(cache.scores[one]), scores)


def test_attend_graphs_side_by_side(K):
    """Two captured calls on a cache without scores, each with its own workspace, replayed at once."""
    from nsrl_b200 import core
    rng = np.random.default_rng(17)
    B, H, cap = 1, 2, 40000
    cache, _, _ = filled(K, rng, B, H, 64, cap, False, 8, 4096)
    q = [dev(gaussian(rng, (B, H * 64), 8)) for _ in range(2)]
    lens = [i32([cap]), i32([33333])]
    want = [host(cache.attend(q[i], lens[i])) for i in range(2)]
    ctx = [torch.zeros((B, H * 64), dtype=torch.int16, device="cuda") for _ in range(2)]
    assert cache.attend_workspace_bytes() > 0
    ws = [torch.empty(cache.attend_workspace_bytes(), dtype=torch.uint8, device="cuda") for _ in range(2)]
    st = [core.Status() for _ in range(2)]
    streams, graphs = [torch.cuda.Stream() for _ in range(2)], [torch.cuda.CUDAGraph() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(2):
        with torch.cuda.graph(graphs[i], stream=streams[i]):
            assert cache.launch_attend(q[i], lens[i], ctx[i], st[i], ws[i]) == 0
    for _ in range(8):
        for c in ctx:
            c.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert np.array_equal(host(ctx[i]), want[i])
    with pytest.raises(core.NsrlError):
        cache.launch_attend(q[0], lens[0], ctx[0], st[0], ws[0].view(torch.int32))
    assert cache.launch_attend(q[0], lens[0], ctx[0], st[0], ws[0][:256]) != 0


def test_scores_saturate(K):
    rng = np.random.default_rng(6)
    cache, kv, vv = filled(K, rng, 1, 1, 64, 16)
    cache.scores.fill_(2 ** 31 - 2)
    q = gaussian(rng, (1, 64), 32)
    assert cache.attend(dev(q), i32([16])) is not None
    _, scores = P.attend(q.reshape(1, 1, 64), kv, vv, [16], np.full((1, 1, 16), 2 ** 31 - 2))
    assert np.array_equal(host(cache.scores), scores)


@pytest.mark.parametrize("cap", [16, 81920])  # one launch, and the split form
@pytest.mark.parametrize("lens", [[0, 5], [5, -1], [-3, 5]])
def test_attend_rejects_bad_lengths(K, lens, cap):
    cache = K.Q4Cache(2, 2, 64, cap)
    q = torch.ones((2, 128), dtype=torch.int16, device="cuda")
    assert cache.attend(q, i32([5, cap])) is not None
    assert cache.attend(q, i32([cap + 1 if n < 0 and n != -3 else n for n in lens])) is None


def test_attend_rejects_bad_lengths_among_many(K):
    cache = K.Q4Cache(150, 4, 64, 32)
    q = torch.ones((150, 256), dtype=torch.int16, device="cuda")
    good = [1 + i % 32 for i in range(150)]
    assert cache.attend_workspace_bytes() > 0 and cache.attend(q, i32(good)) is not None
    for bad in (0, -1, 33, 2 ** 31 - 1, -2 ** 31):
        assert cache.attend(q, i32(good[:77] + [bad] + good[78:])) is None
    assert cache.attend(q, i32(good)) is not None


@pytest.mark.parametrize("hd,cap", [(64, 16), (256, 16), (64, 262144), (256, 262144)])
def test_attend_rejects_logits_outside_i32(K, hd, cap):
    """q = k = 32767: (hd 2^30) >> log4(hd) is 2^33 (64 dims) and 2^34 (256)."""
    cache = K.Q4Cache(1, 1, hd, cap)
    x = torch.full((16, hd), 32767, dtype=torch.int16, device="cuda")
    assert cache.append(x, x, i32([0])) is True
    assert cache.attend(x[:1], i32([16])) is None


@pytest.mark.parametrize("cap", [16, 262144])
def test_masked_logits(K, cap):
    """A logit of exactly -2^31 is the reference's MASKED_LOGIT: no weight; all of them: a rejection.
    Values 32768 (zero 32767, scale 1, code 1) times q = -32768 on 16 of 64 dims: -2^34 >> 3."""
    cache = K.Q4Cache(2, 1, 64, cap)  # the larger takes the split form
    cache.k_scales.fill_(1 | (32767 << 16))
    cache.k_codes.fill_(0x11)
    cache.v_scales[..., :] = 1 | (100 << 16)
    q = torch.zeros((2, 64), dtype=torch.int16, device="cuda")
    q[:, :16] = -32768
    assert cache.attend(q, i32([16, 16])) is None
    cache.k_codes[:, 0, 3] = 0  # slot 3: 32767 -> -32768 * 32767 * 16 >> 3, above the others
    cache.v_scales[:, 0, 3] = 1 | (7000 << 16)
    got = cache.attend(q, i32([16, 16]))
    want = O.attention_row(np.zeros(64, np.int16), np.zeros((1, 64), np.int16), np.full((1, 64), 7000, np.int16), 64, 64)
    for b in range(2):
        assert np.array_equal(host(got)[b], want[0])
        assert host(cache.scores)[b, 0, :16].tolist() == [0] * 3 + [int(want[2][0])] + [0] * 12


# ---------------------------------------------------------------- eviction ---
# (batch, heads, head_dim, capacity, lens, keep, sinks, recent)
EVICTS = [(2, 2, 64, 64, [64, 40], 32, 4, 8), (1, 1, 64, 16, [16], 1, 0, 0), (3, 2, 16, 96, [96, 0, 33], 32, 0, 0),
          (2, 1, 256, 48, [48, 47], 47, 2, 5), (1, 3, 64, 48, [30], 48, 4, 4), (1, 2, 64, 3200, [3111], 1000, 4, 64),
          (2, 2, 16, 320, [320, 319], 100, 200, 300), (1, 1, 64, 40000, [39999], 15001, 1, 100),
          (1, 1, 16, 64, [64], 63, 0, 64)]


def check_evict(K, rng, case, scores, in_place=False):
    B, H, hd, cap, lens, keep, sinks, recent = case
    cache, _, _ = filled(K, rng, B, H, hd, cap)
    cache.scores.copy_(dev(scores.astype(np.int32)))
    pos = np.sort(rng.choice(4 * cap, (B, H, cap)).astype(np.int32), -1) if cap < 1000 else host(cache.positions)
    cache.positions.copy_(dev(pos))
    nxt = pos.max((1, 2)) + 1
    arrays = [host(t).copy() for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales)]
    s_out, p_out = np.full((B, H, cap), -7, np.int32), np.full((B, H, cap), -9, np.int32)
    if in_place:
        s_out, p_out = scores.astype(np.int32).copy(), pos.copy()
    for b in range(B):
        for h in range(H):
            n = min(lens[b], keep)
            s_out[b, h, :n], p_out[b, h, :n] = scores[b, h, :n], pos[b, h, :n]
            for src, dst in P.evict_moves(scores[b, h], pos[b, h], lens[b], int(nxt[b]), keep, sinks, recent):
                for a in arrays:
                    a[b, h, dst] = a[b, h, src]
                s_out[b, h, dst], p_out[b, h, dst] = scores[b, h, src], pos[b, h, src]
    from nsrl_b200 import core
    lg = i32(lens)
    if in_place:
        assert cache.evict(lg, i32(nxt), keep, sinks, recent) is True
        got_s, got_p, got_l = cache.scores, cache.positions, lg
    else:
        got_s, got_p, got_l = torch.full_like(cache.scores, -7), torch.full_like(cache.positions, -9), torch.zeros_like(lg)
        ws = torch.empty(cache.evict_workspace_bytes(keep), dtype=torch.uint8, device="cuda")
        st = core.Status()
        assert cache.launch_evict(lg, i32(nxt), keep, sinks, recent, got_s, got_p, got_l, ws, st) == 0
        assert st.fetch()[0] == 0
        assert host(lg).tolist() == lens and np.array_equal(host(cache.scores), scores)
    for got, want in zip((cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales, got_s, got_p), arrays + [s_out, p_out]):
        assert np.array_equal(host(got), want)
    assert host(got_l).tolist() == [min(n, keep) for n in lens]


@pytest.mark.parametrize("case", EVICTS)
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_equals_the_plain_selection(K, case, in_place):
    rng = np.random.default_rng(case[3])
    B, H, cap = case[0], case[1], case[3]
    scores = (rng.random((B, H, cap)) ** 6 * 1e7).astype(np.int64)
    check_evict(K, rng, case, scores, in_place)


@pytest.mark.parametrize("kind", ["equal", "zero", "few", "negative", "extreme"])
def test_evict_ties_and_signs(K, kind):
    rng = np.random.default_rng(11)
    case = (2, 2, 64, 208, [200, 77], 50, 3, 10)
    shape = (2, 2, 208)
    scores = {"equal": np.full(shape, 12345), "zero": np.zeros(shape), "few": rng.integers(0, 3, shape),
              "negative": rng.integers(-5, 5, shape), "extreme": rng.choice([0, 2 ** 31 - 1, -2 ** 31, 255, 256], shape)}[kind]
    check_evict(K, rng, case, scores.astype(np.int64))


def test_evict_bad_length_and_unscored(K):
    rng = np.random.default_rng(12)
    cache, _, _ = filled(K, rng, 3, 1, 64, 32)
    before = host(cache.k_codes).copy()
    lens = i32([33, 32, -1])
    assert cache.evict(lens, i32([32, 32, 32]), 8, 0, 0) is None
    after = host(cache.k_codes)
    assert np.array_equal(after[0], before[0]) and np.array_equal(after[2], before[2])
    assert not np.array_equal(after[1], before[1]) and host(lens).tolist() == [33, 8, -1]
    plain, _, _ = filled(K, rng, 1, 1, 64, 32, scored=False)
    assert plain.evict(i32([32]), i32([32]), 8) is None


# ----------------------------------------------------------------- together ---
def test_binding_refusals(K):
    from nsrl_b200 import core
    cache = K.Q4Cache(2, 2, 64, 32)
    st = core.Status()
    q = torch.zeros((2, 128), dtype=torch.int16, device="cuda")
    lens = i32([1, 1])
    for bad in (lambda: cache.attend(q.float(), lens), lambda: cache.attend(q.cpu(), lens),
                lambda: cache.attend(q, lens.long()), lambda: cache.attend(q, lens[:1]),
                lambda: cache.attend(q[:1], lens), lambda: cache.attend(q[:, :64], lens),
                lambda: cache.append(q[:1], q[:1], lens), lambda: cache.append(q, q[:, :64], lens),
                lambda: cache.launch_read(None, q, q, st),
                lambda: K.Q4Cache.of(cache.k_codes, cache.v_codes[:1], cache.k_scales, cache.v_scales),
                lambda: K.Q4Cache.of(cache.k_codes, cache.v_codes, cache.k_scales.long(), cache.v_scales)):
        with pytest.raises(core.NsrlError):
            bad()


def test_captured_step(K):
    """append + attend + evict captured once, replayed on new tokens: as the eager calls give."""
    from nsrl_b200 import core
    rng = np.random.default_rng(13)
    B, H, hd, cap, keep = 2, 2, 64, 48, 32
    made = [filled(K, np.random.default_rng(14), B, H, hd, cap)[0] for _ in range(2)]
    x = [dev(gaussian(rng, (B, 3 * H * hd), 300)) for _ in range(4)]
    rows = torch.empty_like(x[0])
    d = H * hd

    def step(cache, row, lens, nxt, ctx, ws, st):
        cache.launch_append(row[:, d:2 * d], row[:, 2 * d:], lens, None, nxt, st)
        lens += 1
        nxt += 1
        cache.launch_attend(row[:, :d], lens, ctx, st)
        cache.launch_evict(lens, nxt, keep, 2, 4, cache.scores, cache.positions, lens, ws, st)

    state = []
    for cache in made:
        state.append((cache, i32([31, 32]), i32([31, 32]), torch.zeros((B, d), dtype=torch.int16, device="cuda"),
                      torch.empty(cache.evict_workspace_bytes(keep), dtype=torch.uint8, device="cuda"), core.Status()))
    (c0, l0, n0, ctx0, ws0, st0), (c1, l1, n1, ctx1, ws1, st1) = state
    saved = [t.clone() for t in (c1.k_codes, c1.v_codes, c1.k_scales, c1.v_scales, c1.scores, c1.positions, l1, n1)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    rows.copy_(x[0])
    with torch.cuda.stream(s):
        step(c1, rows, l1, n1, ctx1, ws1, st1)  # warm-up on the capturing stream
    s.synchronize()
    for t, v in zip((c1.k_codes, c1.v_codes, c1.k_scales, c1.v_scales, c1.scores, c1.positions, l1, n1), saved):
        t.copy_(v)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step(c1, rows, l1, n1, ctx1, ws1, st1)
    for t in x:
        step(c0, t, l0, n0, ctx0, ws0, st0)
        rows.copy_(t)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(ctx0, ctx1)
    for a, b in zip((c0.k_codes, c0.v_codes, c0.k_scales, c0.v_scales, c0.scores, c0.positions, l0),
                    (c1.k_codes, c1.v_codes, c1.k_scales, c1.v_scales, c1.scores, c1.positions, l1)):
        assert torch.equal(a, b)
    assert st0.fetch()[0] == 0 and st1.fetch()[0] == 0


@pytest.mark.parametrize("d,H", [(128, 2), (256, 4), (64, 4), (256, 1)])
def test_decode_loop(K, d, H):
    """Streams of unlike lengths decoded through the block with rotary positions
    and a budget, against the oracle's norm, linears, attention rows and residual."""
    from nsrl_b200 import core, rotary, synth as Y
    B, cap, keep, recent, steps = 3, 32, 20, 4, 12
    hd = d // H
    w = {n: Y.i8_uniform(20 + i, (d, d)) for i, n in enumerate("qkvo")}
    shift = {n: Y.shift_for(d) + (7 if n in "qk" else 0) for n in "qkvo"}
    ol = [O.Linear(w[n], O.scales(1, shift[n], d)) for n in "qkvo"]
    gl = [core.Linear(torch.from_numpy(w[n]), core.make_scales(1, shift[n], d)) for n in "qkvo"]
    gamma = np.full(d, 30000, np.int16)
    plan = rotary.Rotary(hd, hd // 2, layout="interleaved")
    turns = [int(t) % (1 << 64) for t in plan.turns.cpu().tolist()]
    rng = np.random.default_rng(15)
    cache, kv, vv = filled(K, rng, B, H, hd, cap)
    lens, pos = np.array([3, 17, 20]), np.array([3, 40, 20])
    lg, pg = i32(lens), i32(pos)
    slot_pos = np.tile(np.arange(cap), (B, H, 1))
    scores = host(cache.scores).astype(np.int64)
    for step in range(steps):
        x = Y.q15_gaussian(100 + step, (B, d))
        n = O.rms_norm_rows(x, gamma, 1)
        q, k, v = (O.linear(n, l) for l in ol[:3])
        q, k = (P.rotate(t, H, hd, turns, "interleaved", pos) for t in (q, k))
        for t, vals in ((k, kv), (v, vv)):
            new = P.dequantise(*P.quantise(t.reshape(B, H, hd)))
            for b in range(B):
                vals[b, :, lens[b]] = new[b]
        for b in range(B):
            slot_pos[b, :, lens[b]] = pos[b]
            scores[b, :, lens[b]] = 0
        ctx, s = P.attend(q.reshape(B, H, hd), kv, vv, lens + 1, scores)
        scores = s.astype(np.int64)
        y, sat = O.residual_add(x, O.linear(ctx, ol[3]))
        got = K.prenorm_attention_decode_block_q4(dev(x), dev(gamma), 1, *gl, cache, lg, pg, plan)
        assert got is not None
        assert np.array_equal(host(got[0]), y.reshape(B, d)) and got[1] == sat, step
        lens, pos = lens + 1, pos + 1
        lg += 1
        pg += 1
        if step % 3 == 2:
            assert cache.evict(lg, pg, keep, 2, recent) is True
            for b in range(B):
                for h in range(H):
                    for src, dst in P.evict_moves(scores[b, h], slot_pos[b, h], lens[b], pos[b], keep, 2, recent):
                        for a in (kv, vv, scores, slot_pos):
                            a[b, h, dst] = a[b, h, src]
            lens = np.minimum(lens, keep)
            assert host(lg).tolist() == lens.tolist()
    for b in range(B):
        assert np.array_equal(host(cache.scores)[b, :, :lens[b]], scores[b, :, :lens[b]])
        assert np.array_equal(host(cache.positions)[b, :, :lens[b]], slot_pos[b, :, :lens[b]])


def test_decode_block_rejects_a_full_cache(K):
    from nsrl_b200 import core, synth as Y
    cache = K.Q4Cache(1, 2, 64, 16)
    lin = core.Linear(torch.from_numpy(Y.i8_uniform(1, (128, 128))), core.make_scales(1, 12, 128))
    x = dev(Y.q15_gaussian(3, (1, 128)))
    gamma = torch.full((128,), 30000, dtype=torch.int16, device="cuda")
    assert K.prenorm_attention_decode_block_q4(x, gamma, 1, lin, lin, lin, lin, cache, i32([15])) is not None
    assert K.prenorm_attention_decode_block_q4(x, gamma, 1, lin, lin, lin, lin, cache, i32([16])) is None


def test_decode_block_refuses_another_plan(K):
    from nsrl_b200 import core, rotary, synth as Y
    cache = K.Q4Cache(1, 2, 64, 16)
    lin = core.Linear(torch.from_numpy(Y.i8_uniform(1, (128, 128))), core.make_scales(1, 12, 128))
    x = dev(Y.q15_gaussian(3, (1, 128)))
    gamma = torch.full((128,), 30000, dtype=torch.int16, device="cuda")
    args = (x, gamma, 1, lin, lin, lin, lin, cache, i32([0]), None)
    with pytest.raises(core.NsrlError):
        K.prenorm_attention_decode_block_q4(*args, rotary.Rotary(16))
    assert K.prenorm_attention_decode_block_q4(*args, rotary.Rotary(64)) is not None
