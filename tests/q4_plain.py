"""Plain 64-bit forms of the rotary positions and the 4-bit cache (numpy), for
the tests: written from the formulas in include/nsrl_b200.h."""
import math

import numpy as np

from oracle import oracle as O

CIRCLE = [(round(math.cos(2 * math.pi * i / 1024) * 2 ** 30), round(math.sin(2 * math.pi * i / 1024) * 2 ** 30))
          for i in range(1024)]


def cos_sin(position, turn, amplitude=1 << 30):
    """Q30 cos and sin of position * turn 2^-64 turns, in Python integers."""
    a = position * turn % (1 << 64)
    n = (a + (1 << 53)) >> 54
    d = a - (n << 54)
    C, S = CIRCLE[n % 1024]
    r = ((d >> 22) * 1686629713) >> 32
    h = ((r * r >> 32) + (1 << 14)) >> 15
    c = C - ((256 * C * h + S * r + (1 << 37)) >> 38)
    s = S - ((256 * S * h - C * r + (1 << 37)) >> 38)
    if amplitude != 1 << 30:
        c, s = (max(-(1 << 31) + 1, min((1 << 31) - 1, (v * amplitude + (1 << 29)) >> 30)) for v in (c, s))
    return c, s


def pair_dims(rotary_dim, layout):
    half = rotary_dim // 2
    return [(i, i + half) if layout == "half" else (2 * i, 2 * i + 1) for i in range(half)]


def rotate(x, heads, head_dim, turns, layout, positions, backward=False, amplitude=1 << 30):
    """x int16 [rows, heads * head_dim] -> the turned rows."""
    rows = x.shape[0]
    y = x.reshape(rows, heads, head_dim).astype(np.int64)
    out = y.copy()
    for turn, (i, j) in zip(turns, pair_dims(2 * len(turns), layout)):
        cs = np.array([cos_sin(int(p), turn, amplitude) for p in positions], np.int64)
        c, s = cs[:, :1], cs[:, 1:] * (-1 if backward else 1)
        out[:, :, i] = (y[:, :, i] * c - y[:, :, j] * s + (1 << 29)) >> 30
        out[:, :, j] = (y[:, :, i] * s + y[:, :, j] * c + (1 << 29)) >> 30
    return np.clip(out, -32768, 32767).astype(np.int16).reshape(rows, heads * head_dim)


def quantise(x):
    """int16 [..., head_dim] -> (codes uint8, scale words int32)."""
    x = x.astype(np.int64)
    hd = x.shape[-1]
    per = min(32, hd)
    g = x.reshape(x.shape[:-1] + (hd // per, per))
    zero = g.min(-1, keepdims=True)
    scale = np.maximum(1, -(-(g.max(-1, keepdims=True) - zero) // 15))
    code = (2 * (g - zero) + scale) // (2 * scale)
    code = code - (zero + scale * code > 32767)
    assert ((code >= 0) & (code <= 15)).all()
    code = code.reshape(x.shape)
    packed = (code[..., 0::2] | (code[..., 1::2] << 4)).astype(np.uint8)
    word = (scale | (zero << 16))[..., 0]
    return packed, word.astype(np.int32)


def dequantise(codes, words):
    codes = codes.astype(np.int64)
    v = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[:-1] + (-1,))
    per = v.shape[-1] // words.shape[-1]
    w = words.astype(np.int64)
    return v * np.repeat(w & 0xFFFF, per, -1) + np.repeat(w >> 16, per, -1)


def attend(q, kv, vv, lens, scores=None):
    """q [B, H, hd]; values kv, vv [B, H, cap, hd] that fit int16: the oracle's
    attention row of every (sequence, head) -> (ctx [B, H * hd], new scores)."""
    B, H, cap, hd = kv.shape
    ctx = np.zeros((B, H, hd), np.int16)
    new = None if scores is None else scores.astype(np.int64)
    for b in range(B):
        L = int(lens[b])
        for h in range(H):
            r = O.attention_row(q[b, h], kv[b, h, :L].astype(np.int16), vv[b, h, :L].astype(np.int16), hd, hd)
            assert r is not None
            ctx[b, h] = r[0]
            if new is not None:
                new[b, h, :L] += r[2].astype(np.int64)
    return ctx.reshape(B, H * hd), None if new is None else np.minimum(new, 2 ** 31 - 1).astype(np.int32)


def evict_moves(scores, positions, n, next_position, keep, sinks, recent):
    """[(from, to)] of one (sequence, head) of n slots."""
    if n <= keep:
        return []
    key = [1 << 31 if positions[i] < sinks or positions[i] >= next_position - recent else max(int(scores[i]), 0)
           for i in range(n)]
    kept = set(sorted(range(n), key=lambda i: (-key[i], i))[:keep])
    holes = [i for i in range(keep) if i not in kept]
    late = [i for i in range(keep, n) if i in kept]
    assert len(holes) == len(late)
    return list(zip(late, holes))
