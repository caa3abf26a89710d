"""Rotary positions on the GPU: equal to the 64-bit plain form bit for bit,
within a rounding of the real rotation, and the backward pass against the
formula and against differences."""
import math

import numpy as np
import pytest
import torch

import q4_plain as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def R():
    from nsrl_b200 import build, rotary
    build.build()
    return rotary


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def turns_of(plan):
    return [int(t) % (1 << 64) for t in plan.turns.cpu().tolist()]


def rows_of(seed, rows, cols, lo=-32768, hi=32768):
    return np.random.default_rng(seed).integers(lo, hi, (rows, cols)).astype(np.int16)


# (rows, heads, head_dim, rotary_dim, row stride - heads * head_dim, layout): wide loads, odd strides, parts of a
# head, one row, more rows than a block, more pairs than the shared angles of a block hold
SHAPES = [(1, 1, 16, 16, 0, "half"), (5, 3, 64, 64, 64, "half"), (300, 8, 64, 32, 8, "interleaved"),
          (7, 2, 64, 64, 1, "interleaved"), (33, 1, 256, 96, 0, "half"), (4, 2, 10, 6, 3, "half"),
          (3, 1, 6, 2, 0, "interleaved"), (2, 1, 1024, 1024, 0, "half"), (700, 1, 16, 2, 0, "half"),
          (65, 40, 16, 16, 16, "interleaved"), (2, 300, 64, 48, 0, "half"), (12, 2, 64, 64, 8, "half")]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("backward", [False, True])
def test_equals_the_plain_form(R, shape, backward):
    rows, heads, hd, rot, pad, layout = shape
    cols = heads * hd
    plan = R.Rotary(hd, rot, 10000, layout)
    x = rows_of(rows + hd, rows, cols + pad)
    pos = np.random.default_rng(rows).integers(0, 200000, rows).astype(np.int32)
    ref = P.rotate(x[:, :cols], heads, hd, turns_of(plan), layout, pos, backward)
    xg = dev(x)
    got = plan.apply(xg, heads, dev(pos), backward=backward)
    assert np.array_equal(got.cpu().numpy(), ref)
    assert np.array_equal(xg.cpu().numpy(), x)
    plan.apply(xg, heads, dev(pos), backward=backward, out=xg)  # in place: columns past the heads stay
    assert np.array_equal(xg.cpu().numpy()[:, :cols], ref) and np.array_equal(xg.cpu().numpy()[:, cols:], x[:, cols:])


def test_unaligned_rows(R):
    plan = R.Rotary(64)
    x = rows_of(5, 9, 130)
    xg = dev(x)
    pos = np.arange(9, dtype=np.int32)
    got = plan.apply(xg[:, 1:], 2, dev(pos))
    assert np.array_equal(got.cpu().numpy(), P.rotate(x[:, 1:129], 2, 64, turns_of(plan), "half", pos))


def test_far_negative_and_default_positions(R):
    plan = R.Rotary(64, scaling="by_parts", factor=16, original_len=4096)
    x = rows_of(6, 8, 64)
    pos = np.array([0, -1, 2 ** 31 - 1, -2 ** 31, 1 << 30, 999999937, -123456789, 5], np.int32)
    got = plan.apply(dev(x), 1, dev(pos))
    assert np.array_equal(got.cpu().numpy(), P.rotate(x, 1, 64, turns_of(plan), "half", pos))
    got = plan.apply(dev(x), 1, seq_len=3)
    assert np.array_equal(got.cpu().numpy(), P.rotate(x, 1, 64, turns_of(plan), "half", np.arange(8) % 3))


@pytest.mark.parametrize("amplitude", [0.25, 1.2079441541679836, 1.9999999995])
def test_amplitude(R, amplitude):
    plan = R.Rotary(16, amplitude=amplitude)
    x = rows_of(7, 50, 16)
    pos = np.arange(50, dtype=np.int32) * 37
    ref = P.rotate(x, 1, 16, turns_of(plan), "half", pos, amplitude=plan.c().amplitude)
    assert np.array_equal(plan.apply(dev(x), 1, dev(pos)).cpu().numpy(), ref)


def real(x, heads, hd, turns, layout, pos, backward):
    y = x.reshape(-1, heads, hd).astype(np.float64).copy()
    for t, (i, j) in zip(turns, P.pair_dims(2 * len(turns), layout)):
        a = np.array([int(p) * t % 2 ** 64 / 2.0 ** 64 * 2 * math.pi for p in pos])[:, None]
        a = -a if backward else a
        u, v = y[:, :, i].copy(), y[:, :, j].copy()
        y[:, :, i], y[:, :, j] = u * np.cos(a) - v * np.sin(a), u * np.sin(a) + v * np.cos(a)
    return y.reshape(x.shape)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("backward", [False, True])
def test_within_a_rounding_of_the_rotation(R, layout, backward):
    """Half a step for the result's rounding, and |x0| + |x1| <= 2^15.6 times the
    2^-27 + 2^-30 that c and s may be off: below 2^-11."""
    plan = R.Rotary(64, 64, 10000, layout)
    x = rows_of(8, 200, 128, -23170, 23171)
    pos = np.random.default_rng(8).integers(0, 10 ** 9, 200).astype(np.int32)
    got = plan.apply(dev(x), 2, dev(pos), backward=backward).cpu().numpy()
    want = np.clip(real(x, 2, 64, turns_of(plan), layout, pos, backward), -32768, 32767)
    assert np.abs(got - want).max() <= 0.5 + 2.0 ** -11


def test_backward_against_differences(R):
    """<g, f(x + e) - f(x)> against <backward(g), e>: each of the two forward
    values is off by at most 0.5 + 2^-11, each backward value likewise, so the
    sums differ by at most sum |g| (1 + 2^-10) + sum |e| (0.5 + 2^-11)."""
    plan = R.Rotary(64, 48, 10000, "half")
    rng = np.random.default_rng(9)
    x, e, g = (rng.integers(-8000, 8000, (64, 192)).astype(np.int16) for _ in range(3))
    pos = dev(rng.integers(0, 5000, 64).astype(np.int32))
    f = lambda v: plan.apply(dev(v), 3, pos).cpu().numpy().astype(np.float64)  # noqa: E731
    back = plan.apply(dev(g), 3, pos, backward=True).cpu().numpy().astype(np.float64)
    diff = f((x + e).astype(np.int16)) - f(x)
    for row in range(64):
        lhs, rhs = (g[row] * diff[row]).sum(), (back[row] * e[row]).sum()
        bound = np.abs(g[row].astype(np.int64)).sum() * (1 + 2.0 ** -10) + np.abs(e[row].astype(np.int64)).sum() * (0.5 + 2.0 ** -11)
        assert abs(lhs - rhs) <= bound


def test_backward_undoes_forward(R):
    """The forward's rounding (at most 0.5 + 2^-11 on each of a pair) turns back into at
    most 0.708, the backward's adds 0.5 + 2^-11: 1.21, so whole numbers within 1."""
    plan = R.Rotary(256)
    x = rows_of(10, 40, 256, -20000, 20001)
    pos = dev(np.arange(40, dtype=np.int32) * 1001)
    there = plan.apply(dev(x), 1, pos)
    back = plan.apply(there, 1, pos, backward=True).cpu().numpy()
    assert np.abs(back.astype(int) - x).max() <= 1


def test_captured_and_on_another_stream(R):
    plan = R.Rotary(64)
    x = rows_of(11, 64, 256)
    xg, pos = dev(x), dev(np.arange(64, dtype=np.int32))
    out = torch.zeros((64, 256), dtype=torch.int16, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        plan.apply(xg, 4, pos, out=out)
    s.synchronize()
    ref = P.rotate(x, 4, 64, turns_of(plan), "half", np.arange(64))
    assert np.array_equal(out.cpu().numpy(), ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan.apply(xg, 4, pos, out=out)
    pos += 100
    g.replay()
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), P.rotate(x, 4, 64, turns_of(plan), "half", np.arange(64) + 100))


def test_refusals(R):
    from nsrl_b200 import core
    plan = R.Rotary(64)
    x = dev(rows_of(1, 4, 128))
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in (lambda: plan.apply(x.cpu(), 2, pos), lambda: plan.apply(x.float(), 2, pos),
                lambda: plan.apply(x, 3, pos), lambda: plan.apply(x.t(), 2, pos), lambda: plan.apply(x, 2, pos[:3]),
                lambda: plan.apply(x, 2, pos.long()), lambda: plan.apply(x, 2, pos, out=x[:2])):
        with pytest.raises(core.NsrlError):
            bad()
    assert plan.apply(x, 2) is None  # neither positions nor seq_len
    assert plan.apply(x[:0], 2, pos[:0]).shape == (0, 128)
    with pytest.raises(ValueError):
        R.Rotary(64, 63)
    with pytest.raises(ValueError):
        R.Rotary(64, amplitude=2.0)


def test_training_path(R):
    """q and k turn before the training attention, their gradients turn back after
    its backward: equal to the oracle's attention between plain rotations."""
    from nsrl_b200 import train as T
    from oracle import oracle as O
    B, S, d, H = 2, 24, 128, 2
    plan = R.Rotary(64, scaling="ntk", factor=4)
    rng = np.random.default_rng(12)
    qkv = (rng.normal(0, 1, (B * S, 3 * d)) * np.repeat([200, 200, 4000], d)).astype(np.int16)
    dC = rng.integers(-3000, 3000, (B * S, d)).astype(np.int16)
    pos = np.tile(np.arange(S), B)
    turned = qkv.copy()
    turned[:, :2 * d] = P.rotate(qkv[:, :2 * d], 2 * H, 64, turns_of(plan), "half", pos)
    q, k, v = (np.ascontiguousarray(turned[:, i * d:(i + 1) * d]) for i in range(3))
    probs = O.attention_probabilities(q, k, B, S, d, H)
    dq, dk, dv = O.attention_backward(q, k, v, probs, dC, B, S, d, H)[:3]
    want = P.rotate(np.concatenate([dq, dk], 1), 2 * H, 64, turns_of(plan), "half", pos, backward=True)
    g = dev(qkv)
    assert plan.apply(g, 2 * H, seq_len=S, out=g) is not None
    gq, gk, gv = (g[:, i * d:(i + 1) * d].contiguous() for i in range(3))
    ctx, Pg = T.attention_with_probabilities(gq, gk, gv, B, S, d, H)
    assert np.array_equal(Pg.cpu().numpy().reshape(probs.shape), probs)
    grads = T.attention_backward(gq, gk, gv, Pg, dev(dC), B, S, d, H)
    both = torch.cat(list(grads[:2]), 1)
    plan.apply(both, 2 * H, seq_len=S, backward=True, out=both)
    assert np.array_equal(both.cpu().numpy(), want) and np.array_equal(grads[2].cpu().numpy(), dv)


# (heads, head_dim, rotary_dim, row stride - heads * head_dim): wide loads, odd strides, part of a head
@pytest.mark.parametrize("shape", [(3, 64, 64, 8), (3, 64, 32, 0), (2, 64, 48, 5), (3, 10, 6, 1)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("amplitude", [0.7, 1.2079441541679836, 1.9999999995])
def test_amplitude_in_every_form(R, shape, layout, backward, amplitude):
    heads, hd, rot, pad = shape
    cols = heads * hd
    plan = R.Rotary(hd, rot, 10000, layout, amplitude=amplitude)
    x = rows_of(hd + pad, 70, cols + pad)
    pos = np.random.default_rng(pad).integers(-1000, 200000, 70).astype(np.int32)
    ref = P.rotate(x[:, :cols], heads, hd, turns_of(plan), layout, pos, backward, plan.c().amplitude)
    xg = dev(x)
    assert np.array_equal(plan.apply(xg, heads, dev(pos), backward=backward).cpu().numpy(), ref)
    plan.apply(xg, heads, dev(pos), backward=backward, out=xg)
    assert np.array_equal(xg.cpu().numpy()[:, :cols], ref) and np.array_equal(xg.cpu().numpy()[:, cols:], x[:, cols:])


@pytest.mark.parametrize("stride", [1100000008, 1100000003])
def test_rows_past_32_bits(R, stride):
    """Rows 2.2 GB apart, so the last begins past 2^31 elements and 2^32 bytes; in place, and out of it."""
    plan = R.Rotary(64)
    x = rows_of(13, 3, 128)
    pos = np.array([5, -7, 123456], np.int32)
    ref = P.rotate(x, 2, 64, turns_of(plan), "half", pos)
    far = torch.empty(2 * stride + 128, dtype=torch.int16, device="cuda").as_strided((3, 128), (stride, 1))
    assert 2 * stride > 1 << 31
    far.copy_(dev(x))
    assert np.array_equal(plan.apply(far, 2, dev(pos)).cpu().numpy(), ref)
    plan.apply(far, 2, dev(pos), out=far)
    assert np.array_equal(far.cpu().numpy(), ref)
