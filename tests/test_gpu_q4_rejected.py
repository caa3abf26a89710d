"""What a rejected call over the 4-bit cache leaves behind: scores go on from
step to step, so a step that is mended and called again must count once."""
import numpy as np
import pytest
import torch

from test_gpu_q4_cache import K, dev, filled, gaussian, host, i32  # noqa: F401

pytestmark = pytest.mark.gpu


def twin(K, cache):
    """Another cache of the same contents."""
    return K.Q4Cache.of(*(t.clone() for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales, cache.scores,
                                              cache.positions)))


# (batch, heads, head_dim, capacity): one CTA a row, fewer and more sequences than its threads; clusters; rows sorted by
# length; more sequences than are sorted; the split form
FORMS = [(3, 2, 64, 64), (500, 1, 16, 16), (591, 1, 16, 2064), (2, 1, 64, 8208), (2, 2, 256, 2064), (150, 4, 64, 48),
         (75, 8, 256, 32), (4100, 1, 16, 16), (5000, 2, 64, 16), (2, 2, 64, 32784), (3, 1, 256, 32784)]


@pytest.mark.parametrize("form", FORMS)
def test_a_bad_length_leaves_every_score(K, form):
    B, H, hd, cap = form
    rng = np.random.default_rng(B + cap)
    cache, _, _ = filled(K, rng, B, H, hd, cap)
    other = twin(K, cache)
    q = dev(gaussian(rng, (B, H * hd), 32))
    lens = rng.integers(1, cap + 1, B)
    before = cache.scores.clone()
    for at, bad in ((0, 0), (B - 1, cap + 1), (B // 2, -1), (B - 1, 2 ** 31 - 1), (0, -2 ** 31)):
        wrong = lens.copy()
        wrong[at] = bad
        assert cache.attend(q, i32(wrong)) is None
        assert torch.equal(cache.scores, before)
    got, want = cache.attend(q, i32(lens)), other.attend(q, i32(lens))
    assert torch.equal(got, want) and torch.equal(cache.scores, other.scores)
    assert not torch.equal(cache.scores, before)


@pytest.mark.parametrize("form", [(3, 2, 64, 64), (150, 4, 64, 48), (2, 2, 64, 32784)])
def test_a_status_that_holds_a_rejection(K, form):
    """Launches that share a status word: after a rejection no score changes until it is reset."""
    from nsrl_b200 import core
    B, H, hd, cap = form
    rng = np.random.default_rng(B)
    cache, _, _ = filled(K, rng, B, H, hd, cap)
    other = twin(K, cache)
    q = dev(gaussian(rng, (B, H * hd), 32))
    good, bad = i32(np.full(B, cap)), i32([cap + 1] + [cap] * (B - 1))
    ctx, st, before = torch.zeros((B, H * hd), dtype=torch.int16, device="cuda"), core.Status(), cache.scores.clone()
    assert cache.launch_attend(q, bad, ctx, st) == 0 and cache.launch_attend(q, good, ctx, st) == 0
    assert st.fetch()[0] == core.NSRL_CORE_REJECTED and torch.equal(cache.scores, before)
    st.reset()
    assert cache.launch_attend(q, good, ctx, st) == 0 and st.fetch()[0] == 0
    assert torch.equal(ctx, other.attend(q, good)) and torch.equal(cache.scores, other.scores)


# (head_dim, capacity, length, the slot): one CTA a row, clusters (the slot in the last CTA's share), the split form
@pytest.mark.parametrize("hd,cap,n,slot", [(16, 64, 50, 3), (64, 64, 64, 63), (256, 64, 33, 0), (16, 8208, 8200, 8199),
                                           (64, 8208, 8208, 8207), (256, 2064, 2050, 2049), (64, 32784, 32784, 5),
                                           (256, 32784, 32784, 32783)])
def test_a_logit_outside_i32_leaves_its_row(K, hd, cap, n, slot):
    """One key of 32767s meets a query of 32767s: hd 2^30 >> log4(hd) is 2^32 and more.  The other keys are
    below 2^9, so their logits fit."""
    rng = np.random.default_rng(hd + cap)
    cache, _, _ = filled(K, rng, 2, 1, hd, cap)
    cache.k_codes[0, 0, slot] = 255
    cache.k_scales[0, 0, slot] = 1 | (32752 << 16)
    q = gaussian(rng, (2, hd), 32)
    q[0] = 32767
    before = cache.scores.clone()
    assert cache.attend(dev(q), i32([n, n])) is None
    assert torch.equal(cache.scores[0], before[0])


def linears(d):
    from nsrl_b200 import core, synth as Y
    return [core.Linear(torch.from_numpy(Y.i8_uniform(40 + i, (d, d))), core.make_scales(1, Y.shift_for(d) + up, d))
            for i, up in enumerate((7, 7, 0, 0))]


def test_decode_block_again_after_an_eviction(K):
    """A step with one full sequence is rejected; evicted and called again, it gives what it gives without the
    rejected call, the other sequences' scores among it."""
    from nsrl_b200 import rotary, synth as Y
    B, H, cap, keep, d = 3, 2, 48, 40, 128
    rng = np.random.default_rng(21)
    cache, _, _ = filled(K, rng, B, H, 64, cap)
    other = twin(K, cache)
    x, gamma = dev(Y.q15_gaussian(50, (B, d))), torch.full((d,), 30000, dtype=torch.int16, device="cuda")
    plan, ps, pos = rotary.Rotary(64), linears(d), i32([30, 100, 7])
    step = lambda c, lens: K.prenorm_attention_decode_block_q4(x, gamma, 1, *ps, c, lens, pos, plan)  # noqa: E731
    before, lens = cache.scores.clone(), i32([30, cap, 7])
    assert step(cache, lens) is None
    for b, n in ((0, 30), (1, cap), (2, 7)):
        assert torch.equal(cache.scores[b, :, :n], before[b, :, :n])
    results = []
    for c in (cache, other):
        lens = i32([30, cap, 7])
        assert c.evict(lens, pos, keep, 2, 4) is True and host(lens).tolist() == [30, keep, 7]
        results.append(step(c, lens))
        assert results[-1] is not None
    assert torch.equal(results[0][0], results[1][0]) and results[0][1] == results[1][1]
    for name in ("k_codes", "v_codes", "k_scales", "v_scales", "scores", "positions"):
        assert torch.equal(getattr(cache, name), getattr(other, name)), name
    assert not torch.equal(cache.scores[0, :, :30], before[0, :, :30])


def test_decode_block_rejected_by_its_norm(K):
    """A row of zeros with eps 0 has no inverse root: no sequence gains weight."""
    from nsrl_b200 import synth as Y
    B, H, cap, d = 3, 2, 48, 128
    cache, _, _ = filled(K, np.random.default_rng(22), B, H, 64, cap)
    x, gamma = dev(Y.q15_gaussian(51, (B, d))), torch.full((d,), 30000, dtype=torch.int16, device="cuda")
    x[1] = 0
    before = cache.scores.clone()
    assert K.prenorm_attention_decode_block_q4(x, gamma, 0, *linears(d), cache, i32([30, 31, 32])) is None
    for b, n in ((0, 30), (1, 31), (2, 32)):
        assert torch.equal(cache.scores[b, :, :n], before[b, :, :n])
