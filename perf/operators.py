"""What is measured of the quantised KV cache and the rotary positions.

Four operators of this package, each as one pass over inputs that a serving or
training program has in hand:

  rotary  rotary positions on int16 query / key rows, and their gradient
  append  new keys and values into a 4-bit cache, and those rows read back
  attend  one query per sequence over the 4-bit cache, with the weights it
          gives each slot added to the slot's score
  evict   the slots with the least accumulated weight leave the cache, and the
          rows that stay are read back

`run` computes them with plain torch operations, or (`own`) with the calls that
a user makes.  Everything is integer arithmetic, so both give the same numbers.
"""
import decimal
import math

import numpy as np
import torch

own = False

GROUP = 32  # dims that share a scale and a zero point (the whole head below 32)


# ------------------------------------------------------------------ cases ---
def listed():
    return [
        # the q | k columns of the transformer block's Q|K|V rows (64 x 1,024 tokens, d_model 256)
        dict(name="rotary block forward", op="rotary", rows=65536, heads=8, head_dim=64, rotary_dim=64, stride=768,
             layout="half", backward=False, scaling="none", far=0),
        # a long-context model's gradient: part of the head, interleaved pairs, frequencies scaled by parts
        dict(name="rotary partial backward", op="rotary", rows=16351, heads=16, head_dim=64, rotary_dim=32,
             stride=1024, layout="interleaved", backward=True, scaling="by_parts", far=120000),
        # one decode step of 32 streams far into their contexts
        dict(name="rotary decode step", op="rotary", rows=32, heads=16, head_dim=64, rotary_dim=64, stride=1536,
             layout="half", backward=False, scaling="ntk", far=1000000),
        # prefill: eight prompts of up to 2,048 tokens, d_model 512
        dict(name="append prompts", op="append", batch=8, tokens=2048, heads=8, head_dim=64, capacity=2304,
             ragged=True),
        # one token for each of 256 streams
        dict(name="append decode step", op="append", batch=256, tokens=1, heads=8, head_dim=64, capacity=512,
             ragged=False),
        # one stream at the start of a conversation, d_model 256
        dict(name="attend one short stream", op="attend", batch=1, heads=4, head_dim=64, capacity=320, length=301,
             ragged=False, scored=True),
        # the small head dim of the 8-head profile, ragged
        dict(name="attend head_dim 16", op="attend", batch=64, heads=8, head_dim=16, capacity=1024, length=1021,
             ragged=True, scored=True),
        # the decode workload's prefix (8,192 tokens, d_model 512) at batch 32
        dict(name="attend batch 32", op="attend", batch=32, heads=8, head_dim=64, capacity=8320, length=8192,
             ragged=False, scored=True),
        # one long document
        dict(name="attend one long stream", op="attend", batch=1, heads=8, head_dim=64, capacity=131072,
             length=131071, ragged=False, scored=True),
        # the decode workload at its whole batch, streams of unlike lengths, no scores kept
        dict(name="attend batch 256", op="attend", batch=256, heads=8, head_dim=64, capacity=8320, length=8320,
             ragged=True, scored=False),
        # 256 streams past their budget by 64 tokens
        dict(name="evict step", op="evict", batch=256, heads=8, head_dim=64, capacity=2112, length=2112, keep=2048,
             sinks=4, recent=128, ragged=False),
        # 32 long prompts cut to their budget after prefill
        dict(name="evict after prefill", op="evict", batch=32, heads=8, head_dim=64, capacity=8192, length=8192,
             keep=2048, sinks=4, recent=256, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend", "evict"])
    head_dim = rng.choice([16, 64, 64, 256])
    if op == "rotary":
        heads = _log(rng, 1, 32)
        rows = _log(rng, 1, max(1, 33_000_000 // (heads * head_dim)))
        rotary_dim = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4, 2 * rng.randint(1, head_dim // 2)])
        return dict(op=op, rows=rows, heads=heads, head_dim=head_dim, rotary_dim=max(2, rotary_dim),
                    stride=heads * head_dim + rng.choice([0, 0, heads * head_dim, 8, rng.randint(1, 40)]),
                    layout=rng.choice(["half", "interleaved"]), backward=rng.random() < 0.4,
                    scaling=rng.choice(["none", "linear", "ntk", "by_parts"]), far=_log(rng, 1, 2000000))
    heads = _log(rng, 1, 16)
    if op == "append":
        tokens = rng.choice([1, _log(rng, 1, 2048)])
        batch = _log(rng, 1, max(1, min(256, 8_000_000 // (tokens * heads * head_dim))))
        return dict(op=op, batch=batch, tokens=tokens, heads=heads, head_dim=head_dim,
                    capacity=16 * ((tokens + rng.randint(0, 100) + 15) // 16), ragged=rng.random() < 0.5)
    length = _log(rng, 1, 131072 if op == "attend" else 32768)
    batch = _log(rng, 1, max(1, min(256, (400_000_000 if op == "attend" else 60_000_000) // (length * heads * head_dim))))
    case = dict(op=op, batch=batch, heads=heads, head_dim=head_dim, capacity=16 * ((length + rng.randint(0, 200) + 15) // 16),
                length=length, ragged=rng.random() < 0.5)
    if op == "attend":
        return dict(case, scored=rng.random() < 0.7)
    keep = max(1, int(length * rng.uniform(0.1, 1.1)))
    keep = min(keep, case["capacity"])
    return dict(case, keep=keep, sinks=rng.choice([0, 4]), recent=rng.randint(0, keep))


# ---------------------------------------------------------------- rotary ----
def rotary_turns(case):
    """Turns per position of each pair, in units of 2^-64 turn: base^(-2i/rotary_dim) / (2 pi), scaled."""
    with decimal.localcontext() as ctx:
        ctx.prec = 60
        D = decimal.Decimal
        pi = D("3.14159265358979323846264338327950288419716939937510582097494459")
        rot, factor, original = case["rotary_dim"], D(8), D(4096)
        base = D(10000)
        if case["scaling"] == "ntk" and rot > 2:
            base *= factor ** (D(rot) / D(rot - 2))
        out = []
        for i in range(rot // 2):
            turn = base ** (-D(2 * i) / D(rot)) / (2 * pi)
            if case["scaling"] == "linear":
                turn /= factor
            elif case["scaling"] == "by_parts":  # whole above 4 turns in the original context, divided below 1
                part = min(D(1), max(D(0), (original * turn - 1) / 3))
                turn *= part + (1 - part) / factor
            out.append(int((turn * D(1 << 64)).to_integral_value(decimal.ROUND_HALF_EVEN)))
    return [t - (1 << 64) if t >= 1 << 63 else t for t in out]


def circle():
    """cos and sin of i / 1024 turns in Q30."""
    a = np.arange(1024) * (2 * np.pi / 1024)
    return np.rint(np.cos(a) * 2.0 ** 30).astype(np.int64), np.rint(np.sin(a) * 2.0 ** 30).astype(np.int64)


def cos_sin(turns, positions, table):
    """Q30 cos and sin of positions x turns [rows, pairs]: the nearest of 1,024 points of the circle, turned by the
    remaining angle d (below 2^-11 turn) as 1 - d^2 / 2 and d."""
    t = positions[:, None] * turns[None, :]  # wraps at a whole turn
    near = ((t + (1 << 53)) >> 54)
    d = t - (near << 54)
    c0, s0 = table[0][near & 1023], table[1][near & 1023]
    r = ((d >> 22) * 1686629713) >> 32           # d in radians, Q38
    h = (((r * r) >> 32) + (1 << 14)) >> 15      # d^2 / 2, Q30
    c = c0 - ((c0 * h * 256 + s0 * r + (1 << 37)) >> 38)
    s = s0 - ((s0 * h * 256 - c0 * r + (1 << 37)) >> 38)
    return c, s


def rotate(x, c, s, heads, head_dim, layout, backward):
    """x [rows, heads * head_dim] int64; pairs (x0, x1) -> (x0 c - x1 s, x0 s + x1 c), rounded half up at 2^30, saturated."""
    rows, half = x.shape[0], c.shape[1]
    x = x.reshape(rows, heads, head_dim)
    if layout == "half":
        x0, x1 = x[:, :, :half], x[:, :, half:2 * half]
    else:
        x0, x1 = x[:, :, 0:2 * half:2], x[:, :, 1:2 * half:2]
    c, s = c[:, None, :], (-s if backward else s)[:, None, :]
    y0 = torch.clip((x0 * c - x1 * s + (1 << 29)) >> 30, -32768, 32767)
    y1 = torch.clip((x0 * s + x1 * c + (1 << 29)) >> 30, -32768, 32767)
    pairs = torch.concatenate([y0, y1], -1) if layout == "half" else torch.stack([y0, y1], -1).reshape(rows, heads, 2 * half)
    return torch.concatenate([pairs, x[:, :, 2 * half:]], -1).reshape(rows, heads * head_dim)


# ------------------------------------------------------------- the cache ----
def quantise(x):
    """int16 [..., head_dim] -> (codes uint8 [..., head_dim / 2], scales int32 [..., groups]).

    Per group: zero = min, scale = max(1, ceil((max - min) / 15)), code = round((x - zero) / scale), one less where
    zero + scale * code would pass 32767.  Byte i holds dim 2i in its low half; a scale word is scale | zero << 16."""
    x = x.int()
    g = x.unflatten(-1, (-1, min(GROUP, x.shape[-1])))
    zero = g.amin(-1, keepdim=True)
    scale = ((g.amax(-1, keepdim=True) - zero + 14) // 15).clamp(min=1)
    code = (2 * (g - zero) + scale) // (2 * scale)
    code = (code - (zero + scale * code > 32767).int()).flatten(-2)
    packed = (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8)
    return packed, (scale | (zero << 16)).squeeze(-1)


def dequantise(codes, scales, dtype):
    """The values that codes and scales stand for, zero + scale * code, [..., head_dim]."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(dtype)
    c = c.unflatten(-1, (scales.shape[-1], -1))
    return (c * (scales & 0xFFFF).to(dtype)[..., None] + (scales >> 16).to(dtype)[..., None]).flatten(-2)


def luts(device):
    """Q15 2^(-f / 256) for f < 256, and Q31 1 / m for 128 <= m < 256."""
    f = torch.arange(256, device=device, dtype=torch.float64)
    e = torch.floor(32768 * torch.exp2(-f / 256) + 0.5).long().clamp(max=32767)
    m = torch.arange(128, 256, device=device)
    return e, ((1 << 31) + m // 2) // m


def attend(q, codes_k, scales_k, codes_v, scales_v, lens, scores):
    """Base-2 softmax attention of one query per (sequence, head) over its first lens[b] slots."""
    B, H, cap = codes_k.shape[:3]
    hd = 2 * codes_k.shape[3]
    exp2, recip = luts(q.device)
    live = torch.arange(cap, device=q.device)[None, None, :] < lens[:, None, None]
    # the products stay below 2^53, so float64 holds them exactly
    dots = torch.matmul(dequantise(codes_k, scales_k, torch.float64), q.view(B, H, hd, 1).double()).squeeze(-1).long()
    logit = (dots >> (int(math.log2(hd)) // 2)).masked_fill(~live, -(1 << 40))
    mag = logit.amax(-1, keepdim=True) - logit
    w = torch.where(live & (mag < 15 * 256), exp2[mag & 255] >> (mag >> 8).clamp(max=15), 0)
    total = w.sum(-1, keepdim=True)
    shift = torch.frexp(total.double()).exponent.long() - 8  # brings the total's highest bit to bit 7
    top = torch.where(shift >= 0, total >> shift.clamp(min=0), total << (-shift).clamp(min=0))
    inv = torch.where(shift >= 0, recip[top - 128] >> shift.clamp(min=0), recip[top - 128] << (-shift).clamp(min=0))
    p = ((w * inv.clamp(max=(1 << 32) - 1) + (1 << 15)) >> 16).clamp(max=32767)
    acc = torch.matmul(p.double().unsqueeze(-2), dequantise(codes_v, scales_v, torch.float64)).long()
    ctx = ((acc + (1 << 14)) >> 15).clamp(-32768, 32767).to(torch.int16).reshape(B, H * hd)
    if scores is not None:
        scores.copy_((scores.long() + p).clamp(max=(1 << 31) - 1))
    return ctx


def evict(state):
    """Keeps `keep` slots of each (sequence, head): sinks and recent tokens first, then by score, then the lower slot.
    The kept rows at or past `keep` move into the free slots below it, both in ascending order."""
    c = state["case"]
    B, H, cap, keep = c["batch"], c["heads"], c["capacity"], c["keep"]
    slot = torch.arange(cap, device="cuda").expand(B, H, cap)
    lens, pos = state["lens"].long()[:, None, None], state["positions"].long()
    live = slot < lens
    safe = (pos < c["sinks"]) | (pos >= state["next"].long()[:, None, None] - c["recent"])
    key = torch.where(safe, 1 << 31, state["scores"].long().clamp(min=0))
    order = torch.where(live, key * (1 << 20) - slot, -(1 << 62)).argsort(-1, descending=True)
    rank = torch.empty_like(order).scatter_(-1, order, slot)
    kept = live & (rank < keep)
    # the i-th slot of (kept below keep, then holes below keep) takes the i-th of (kept below, kept at or past keep)
    holes = (slot < torch.minimum(lens, lens.new_tensor(keep))) & ~kept
    into = torch.where(kept & (slot < keep), slot, torch.where(holes, cap + slot, 3 * cap + slot)).argsort(-1)[..., :keep]
    source = torch.where(kept & (slot < keep), slot, torch.where(kept, cap + slot, 3 * cap + slot)).argsort(-1)[..., :keep]
    fits = torch.arange(keep, device="cuda") < lens
    row = lambda t: torch.gather(t, 2, source[..., None].expand(B, H, keep, t.shape[3])) if t.dim() == 4 else torch.gather(t, 2, source)  # noqa: E731

    def moved(t, out):  # rows that no sequence reaches stay as they were
        at = into if t.dim() == 3 else into[..., None].expand(B, H, keep, t.shape[3])
        ok = fits if t.dim() == 3 else fits[..., None]
        return out.scatter_(2, at, torch.where(ok, row(t), torch.gather(out, 2, at)))

    for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
        state[name] = moved(state[name], state[name].clone())
    moved(state["scores"], state["scores_out"])
    moved(state["positions"], state["positions_out"])
    state["lens_out"].copy_(state["lens"].clamp(max=keep))


def read(state, first, count):
    """Slots first[b] .. first[b] + count as int16 [batch, heads, count, head_dim]."""
    at = (first.long()[:, None, None] + torch.arange(count, device="cuda")).expand(-1, state["k_codes"].shape[1], -1)[..., None]
    out = []
    for codes, scales in (("k_codes", "k_scales"), ("v_codes", "v_scales")):
        c, s = state[codes], state[scales]
        c = torch.gather(c, 2, at.expand(-1, -1, -1, c.shape[3]))
        s = torch.gather(s, 2, at.expand(-1, -1, -1, s.shape[3]))
        out.append(dequantise(c, s, torch.int32).clamp(-32768, 32767).to(torch.int16))
    return out


# ------------------------------------------------------------ the passes ----
def gaussian(g, shape, sigma):
    return (torch.randn(shape, generator=g, device="cuda") * sigma).round_().clamp_(-32768, 32767).to(torch.int16)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case=case)

    def ints(lo, hi, shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)

    if case["op"] == "rotary":
        cols = case["heads"] * case["head_dim"]
        state["x"] = gaussian(g, (case["rows"], case["stride"]), 4096)[:, :cols]
        state["positions"] = ints(0, max(1, case["far"]), (1,)) + torch.arange(case["rows"], device="cuda", dtype=torch.int32) % 1024
        state["turns"] = torch.tensor(rotary_turns(case), dtype=torch.int64, device="cuda")
        state["table"] = [torch.from_numpy(t).cuda() for t in circle()]
        state["y"] = torch.empty((case["rows"], cols), dtype=torch.int16, device="cuda")
        if own:  # the plan that a program makes once per model
            from nsrl_b200 import rotary
            state["plan"] = rotary.Rotary(case["head_dim"], case["rotary_dim"], 10000, case["layout"], case["scaling"],
                                          factor=8, original_len=4096)
        return state
    B, H, hd, cap = case["batch"], case["heads"], case["head_dim"], case["capacity"]
    groups = max(1, hd // GROUP)
    if case["op"] == "append":
        n = case["tokens"]
        state["k"], state["v"] = gaussian(g, (B * n, H * hd), 32), gaussian(g, (B * n, H * hd), 4096)
        state["starts"] = ints(0, cap - n + 1, (B,))
        state["counts"] = ints(0, n + 1, (B,)) if case["ragged"] else torch.full((B,), n, dtype=torch.int32, device="cuda")
        state["k_codes"], state["v_codes"] = (torch.zeros((B, H, cap, hd // 2), dtype=torch.uint8, device="cuda") for _ in "kv")
        state["k_scales"], state["v_scales"] = (torch.zeros((B, H, cap, groups), dtype=torch.int32, device="cuda") for _ in "kv")
    else:
        state["k_codes"], state["k_scales"] = quantise(gaussian(g, (B, H, cap, hd), 32))
        state["v_codes"], state["v_scales"] = quantise(gaussian(g, (B, H, cap, hd), 4096))
        state["lens"] = ints(1, case["length"] + 1, (B,)) if case["ragged"] else torch.full((B,), case["length"], dtype=torch.int32, device="cuda")
    if case["op"] == "attend":
        state["q"] = gaussian(g, (B, H * hd), 32)
        state["scores"] = ints(0, 1 << 20, (B, H, cap)) if case["scored"] else None
        state["ctx"] = torch.empty((B, H * hd), dtype=torch.int16, device="cuda")
    elif case["op"] == "evict":
        # a few slots gather most of the weight, many hardly any
        state["scores"] = (torch.rand((B, H, cap), generator=g, device="cuda") ** 6 * 1e7).to(torch.int32)
        state["positions"] = torch.arange(cap, device="cuda", dtype=torch.int32).expand(B, H, cap).contiguous()
        state["next"] = state["lens"].clone()
        state["scores_out"], state["positions_out"] = torch.zeros_like(state["scores"]), torch.zeros_like(state["positions"])
        state["lens_out"] = torch.zeros_like(state["lens"])
        state["first"] = torch.zeros_like(state["lens"])
    if case["op"] != "attend":
        n = case["tokens"] if case["op"] == "append" else case["keep"]
        state["k_rows"], state["v_rows"] = (torch.empty((B, H, n, hd), dtype=torch.int16, device="cuda") for _ in "kv")
    if own:  # the cache's handle, the workspace and the status word that a program keeps
        from nsrl_b200 import cache, core
        state["cache"] = cache.Q4Cache.of(state["k_codes"], state["v_codes"], state["k_scales"], state["v_scales"],
                                          state.get("scores"), state.get("positions"))
        state["status"] = core.Status()
        if case["op"] == "evict":
            state["ws"] = torch.empty(state["cache"].evict_workspace_bytes(case["keep"]), dtype=torch.uint8, device="cuda")
    return state


def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        if op == "rotary":
            return state["plan"].apply(state["x"], case["heads"], state["positions"], backward=case["backward"], out=state["y"])
        cache, status = state["cache"], state["status"]
        if op == "append":
            cache.launch_append(state["k"], state["v"], state["starts"], state["counts"], None, status)
            cache.launch_read(state["starts"], state["k_rows"], state["v_rows"], status)
            return state["k_rows"], state["v_rows"]
        if op == "attend":
            cache.launch_attend(state["q"], state["lens"], state["ctx"], status)
            return state["ctx"], state["scores"]
        cache.launch_evict(state["lens"], state["next"], case["keep"], case["sinks"], case["recent"], state["scores_out"],
                           state["positions_out"], state["lens_out"], state["ws"], status)
        cache.launch_read(state["first"], state["k_rows"], state["v_rows"], status)
        return state["k_rows"], state["v_rows"], state["scores_out"], state["positions_out"], state["lens_out"]
    if op == "rotary":
        c, s = cos_sin(state["turns"], state["positions"].long(), state["table"])
        return rotate(state["x"].long(), c, s, case["heads"], case["head_dim"], case["layout"], case["backward"]).to(torch.int16)
    if op == "append":
        B, H, hd, n = case["batch"], case["heads"], case["head_dim"], case["tokens"]
        at = (state["starts"].long()[:, None, None] + torch.arange(n, device="cuda")).expand(B, H, n)[..., None]
        fits = (torch.arange(n, device="cuda") < state["counts"][:, None])[:, None, :, None]
        for x, codes, scales in (("k", "k_codes", "k_scales"), ("v", "v_codes", "v_scales")):
            new = quantise(state[x].view(B, n, H, hd).transpose(1, 2))
            for t, rows in zip((state[codes], state[scales]), new):
                i = at.expand(B, H, n, t.shape[3])
                t.scatter_(2, i, torch.where(fits, rows, torch.gather(t, 2, i)))
        return tuple(read(state, state["starts"], n))
    if op == "attend":
        ctx = attend(state["q"], state["k_codes"], state["k_scales"], state["v_codes"], state["v_scales"], state["lens"], state["scores"])
        return ctx, state["scores"]
    evict(state)
    k, v = read(state, torch.zeros_like(state["lens"]), case["keep"])
    return k, v, state["scores_out"], state["positions_out"], state["lens_out"]


def work(case):
    """Bytes of every input read once and every output written once; integer multiply-adds count as two operations."""
    if case["op"] == "rotary":
        n = case["rows"] * case["heads"] * case["head_dim"]
        return dict(bytes=4 * n + 4 * case["rows"], flops=3 * case["rows"] * case["heads"] * case["rotary_dim"])
    B, H, hd = case["batch"], case["heads"], case["head_dim"]
    row = 2 * (hd // 2 + 4 * max(1, hd // GROUP))  # a slot's codes and scales, key and value
    if case["op"] == "append":
        rows = B * case["tokens"] * H
        return dict(bytes=rows * (4 * hd + row + 4 * hd), flops=rows * 2 * hd * 6)
    length = case["length"] * (0.5 if case["ragged"] else 1)
    slots = B * H * length
    if case["op"] == "attend":
        return dict(bytes=slots * (row + (8 if case["scored"] else 0)) + 4 * B * H * hd, flops=slots * 4 * hd)
    # scores and positions of every slot; of the kept ones the rows that move, the new scores and positions, and the rows read back
    keep = min(case["keep"], length)
    moves = keep * max(0.0, 1 - keep / max(1.0, length))
    return dict(bytes=8 * slots + B * H * (moves * 2 * row + keep * (8 + row + 4 * hd)), flops=slots * 8)


# ------------------------------------------------------------- in 64 bits ---
def _np_dequantise(codes, scales):
    codes, scales = codes.cpu().numpy(), scales.cpu().numpy().astype(np.int64)
    values = np.empty(codes.shape[:-1] + (2 * codes.shape[-1],), np.int64)
    values[..., 0::2], values[..., 1::2] = codes & 15, codes >> 4
    per = values.shape[-1] // scales.shape[-1]
    return values * np.repeat(scales & 0xFFFF, per, -1) + np.repeat(scales >> 16, per, -1)


def _np_quantised(x):
    """What quantised int16 rows stand for, as int64."""
    x = x.astype(np.int64)
    out = np.empty_like(x)
    per = min(GROUP, x.shape[-1])
    for i in range(0, x.shape[-1], per):
        g = x[..., i:i + per]
        zero = g.min(-1, keepdims=True)
        scale = np.maximum(1, -((zero - g.max(-1, keepdims=True)) // 15))
        code = np.floor_divide(2 * (g - zero) + scale, 2 * scale)
        code = np.where(zero + scale * code > 32767, code - 1, code)
        out[..., i:i + per] = zero + scale * code
    return out


def _np_rotated(x, positions, case):
    """Pair by pair, with unsigned angles."""
    hd, half = case["head_dim"], case["rotary_dim"] // 2
    first = [i if case["layout"] == "half" else 2 * i for i in range(half)]
    apart = half if case["layout"] == "half" else 1
    c0, s0 = circle()
    x = x.reshape(x.shape[0], case["heads"], hd)
    out = x.astype(np.int64)
    for i, turn in enumerate(rotary_turns(case)):
        angle = positions.astype(np.int64).view(np.uint64) * np.uint64(turn % (1 << 64))
        point = ((angle + np.uint64(1 << 53)) >> np.uint64(54)) % np.uint64(1024)
        rest = (angle - (point << np.uint64(54))).view(np.int64) >> 22  # 2^-42 turn, either side of the point
        point = point.astype(np.int64)
        d = rest * 1686629713 >> 32
        dd = ((d * d >> 32) + 16384 >> 15) << 8
        c = (c0[point] - (c0[point] * dd + s0[point] * d + (1 << 37) >> 38))[:, None]
        s = (s0[point] - (s0[point] * dd - c0[point] * d + (1 << 37) >> 38))[:, None]
        s = -s if case["backward"] else s
        a, b = x[:, :, first[i]].astype(np.int64), x[:, :, first[i] + apart].astype(np.int64)
        out[:, :, first[i]] = a * c - b * s + 536870912 >> 30
        out[:, :, first[i] + apart] = a * s + b * c + 536870912 >> 30
    return np.clip(out, -32768, 32767).reshape(x.shape[0], -1)


def exact(case, seed):
    size = {"rotary": lambda: case["rows"] * case["heads"] * case["head_dim"] / 4,
            "append": lambda: case["batch"] * case["tokens"] * case["heads"] * case["head_dim"] / 2}.get(
        case["op"], lambda: case["batch"] * case["heads"] * case["capacity"] * case["head_dim"])()
    if size > 3e8:
        return None
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _np_rotated(s["x"].cpu().numpy(), s["positions"].cpu().numpy(), case)
    B, H, hd, cap = case["batch"], case["heads"], case["head_dim"], case["capacity"]
    if case["op"] == "append":
        n, counts = case["tokens"], s["counts"].cpu().numpy()
        live = (np.arange(n)[None, :] < counts[:, None])[:, None, :, None]
        return tuple(_np_quantised(s[x].cpu().numpy().reshape(B, n, H, hd)).transpose(0, 2, 1, 3) * live for x in "kv")
    lens = s["lens"].cpu().numpy()
    if case["op"] == "attend":
        exp2 = [min(32767, int(decimal.Decimal(32768) * decimal.Decimal(2) ** (-decimal.Decimal(f) / 256) + decimal.Decimal("0.5"))) for f in range(256)]
        exp2 = np.array(exp2, np.int64)
        q = s["q"].cpu().numpy().astype(np.int64).reshape(B, H, hd)
        ctx = np.zeros((B, H, hd), np.int64)
        scores = None if s["scores"] is None else s["scores"].cpu().numpy().astype(np.int64)
        for b in range(B):
            L = int(lens[b])
            K = _np_dequantise(s["k_codes"][b, :, :L], s["k_scales"][b, :, :L]).astype(np.float64)
            V = _np_dequantise(s["v_codes"][b, :, :L], s["v_scales"][b, :, :L]).astype(np.float64)
            for h in range(H):
                logit = (K[h] @ q[b, h].astype(np.float64)).astype(np.int64) >> (hd.bit_length() // 2)
                mag = logit.max() - logit
                w = np.where(mag < 15 * 256, exp2[mag & 255] >> np.minimum(mag >> 8, 15), 0)
                total = int(w.sum())
                shift = total.bit_length() - 8
                m = total >> shift if shift >= 0 else total << -shift
                inv = ((1 << 31) + m // 2) // m
                inv = min((1 << 32) - 1, inv >> shift if shift >= 0 else inv << -shift)
                p = np.minimum(32767, (w * inv + (1 << 15)) >> 16)
                ctx[b, h] = np.clip(((p.astype(np.float64) @ V[h]).astype(np.int64) + (1 << 14)) >> 15, -32768, 32767)
                if scores is not None:
                    scores[b, h, :L] = np.minimum((1 << 31) - 1, scores[b, h, :L] + p)
        return ctx.reshape(B, H * hd), scores
    keep, nxt = case["keep"], s["next"].cpu().numpy()
    k, v = _np_dequantise(s["k_codes"], s["k_scales"]), _np_dequantise(s["v_codes"], s["v_scales"])
    score, pos = s["scores"].cpu().numpy().astype(np.int64), s["positions"].cpu().numpy().astype(np.int64)
    score_out, pos_out = np.zeros_like(score), np.zeros_like(pos)
    for b in range(B):
        L = int(lens[b])
        for h in range(H):
            key = np.where((pos[b, h, :L] < case["sinks"]) | (pos[b, h, :L] >= nxt[b] - case["recent"]), 1 << 31, np.maximum(score[b, h, :L], 0))
            stays = np.sort(np.argsort(-key, kind="stable")[:keep])
            free = np.setdiff1d(np.arange(min(keep, L)), stays)
            late = stays[stays >= keep]
            k[b, h, free], v[b, h, free] = k[b, h, late], v[b, h, late]
            n = min(keep, L)
            score_out[b, h, :n], pos_out[b, h, :n] = score[b, h, :n], pos[b, h, :n]
            score_out[b, h, free], pos_out[b, h, free] = score[b, h, late], pos[b, h, late]
    return k[:, :, :keep], v[:, :, :keep], score_out, pos_out, np.minimum(lens, keep)
