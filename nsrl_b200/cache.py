"""The 4-bit KV cache: append, attention over it, eviction by accumulated
attention weight, and the decode block that uses them (include/nsrl_b200.h).

A slot of 64 dims takes 80 bytes (key and value) where the int16 cache takes
256.  The attention gives, on the values the codes stand for, exactly what
`core.attention_decode` gives on int16 ones.

`launch_*` methods enqueue on the current stream and return the C status code
without waiting (they may be captured into a graph; the device status tells
rejections later).  The methods without the prefix wait and return None when
the call was rejected, as the functions of `core` do.

Scores go on from step to step.  A call that is rejected for a length, or whose
status already holds a rejection, leaves all of them as they were, so a step
with a full sequence can be made again after an eviction; reset a status that
`launch_*` calls share after a rejection.

Calls on one cache run one after another: on one stream, or on several that the
caller orders.  Attention without scores only reads the cache, so it may run on
several streams at once, each call with a workspace of its own: `attend` takes
one for each call, `launch_attend` takes the cache's unless it is given another.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import core
from .rotary import Rotary, RotaryC

GROUP = 32  # dims that share a scale and a zero point (a whole head below 32)


class Q4CacheC(C.Structure):
    _fields_ = [("k_codes", C.c_void_p), ("v_codes", C.c_void_p), ("k_scales", C.c_void_p),
                ("v_scales", C.c_void_p), ("scores", C.c_void_p), ("positions", C.c_void_p),
                ("batch", C.c_size_t), ("heads", C.c_size_t), ("head_dim", C.c_size_t), ("capacity", C.c_size_t)]


def _lib():
    L = core.lib()
    if not getattr(L, "_q4_bound", False):
        vp, sz, lp, cp = C.c_void_p, C.c_size_t, C.POINTER(core.LinearParamsC), C.POINTER(Q4CacheC)
        L.nsrl_q4_cache_max_capacity.restype = sz
        L.nsrl_q4_cache_append.argtypes = [cp, vp, vp, sz, sz, vp, vp, vp, vp, vp]
        L.nsrl_q4_cache_read.argtypes = [cp, vp, sz, vp, vp, vp, vp]
        L.nsrl_attention_decode_q4_workspace_size.restype = sz
        L.nsrl_attention_decode_q4_workspace_size.argtypes = [cp]
        L.nsrl_attention_decode_q4.argtypes = [vp, sz, cp, vp, vp, vp, sz, vp, vp]
        L.nsrl_q4_cache_evict_workspace_size.restype = sz
        L.nsrl_q4_cache_evict_workspace_size.argtypes = [cp, sz]
        L.nsrl_q4_cache_evict.argtypes = [cp, vp, vp, sz, sz, sz, vp, vp, vp, vp, sz, vp, vp]
        L.nsrl_decode_block_q4_workspace_size.restype = sz
        L.nsrl_decode_block_q4_workspace_size.argtypes = [cp]
        L.nsrl_prenorm_attention_decode_block_q4.argtypes = [vp, sz, sz, sz, vp, C.c_uint64, lp, lp, lp, lp,
                                                             C.POINTER(RotaryC), cp, vp, vp, vp, vp, sz, vp, vp]
        L._q4_bound = True
    return L


class Q4Cache:
    """Codes and scales of `capacity` slots for every (sequence, head), empty at the start.

    scored: keep each slot's accumulated attention weight and position, which
    `evict` goes by."""

    def __init__(self, batch: int, heads: int, head_dim: int, capacity: int, scored: bool = True):
        dev = core._dev()
        groups = max(1, head_dim // GROUP)

        def zeros(shape, dtype):
            return torch.zeros((batch, heads, capacity) + shape, dtype=dtype, device=dev)

        self._take(zeros((head_dim // 2,), torch.uint8), zeros((head_dim // 2,), torch.uint8),
                   zeros((groups,), torch.int32), zeros((groups,), torch.int32),
                   zeros((), torch.int32) if scored else None, zeros((), torch.int32) if scored else None)

    @classmethod
    def of(cls, k_codes, v_codes, k_scales, v_scales, scores=None, positions=None) -> "Q4Cache":
        """A cache over the caller's tensors (layouts as in include/nsrl_b200.h, scales as int32 words)."""
        c = cls.__new__(cls)
        c._take(k_codes, v_codes, k_scales, v_scales, scores, positions)
        return c

    def _take(self, k_codes, v_codes, k_scales, v_scales, scores, positions):
        if k_codes.dim() != 4:
            raise core.NsrlError("k_codes must be [batch, heads, capacity, head_dim / 2]")
        B, H, cap, half = k_codes.shape
        self.batch, self.heads, self.capacity, self.head_dim = B, H, cap, 2 * half
        groups = max(1, self.head_dim // GROUP)
        self.k_codes, self.v_codes, self.k_scales, self.v_scales = k_codes, v_codes, k_scales, v_scales
        self.scores, self.positions = scores, positions
        dev = torch.cuda.current_device()
        ptr = [core._array(k_codes, torch.uint8, (B, H, cap, half), dev, "k_codes"),
               core._array(v_codes, torch.uint8, (B, H, cap, half), dev, "v_codes"),
               core._array(k_scales, torch.int32, (B, H, cap, groups), dev, "k_scales"),
               core._array(v_scales, torch.int32, (B, H, cap, groups), dev, "v_scales"),
               None if scores is None else core._array(scores, torch.int32, (B, H, cap), dev, "scores"),
               None if positions is None else core._array(positions, torch.int32, (B, H, cap), dev, "positions")]
        self.device, self._dev = k_codes.device, dev
        self._cols = H * self.head_dim
        self._c = Q4CacheC(*ptr, B, H, self.head_dim, cap)
        self._ref = C.byref(self._c)
        # the attention's workspace (4 bytes a slot and a little, none for a small cache) lives as long as the cache
        nbytes = _lib().nsrl_attention_decode_q4_workspace_size(self._ref)
        self._ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None
        self._ws_ptr, self._ws_bytes = (self._ws.data_ptr() if nbytes else None), nbytes

    def c(self) -> Q4CacheC:
        return self._c

    def _per_sequence(self, t: torch.Tensor, what: str) -> int:
        return core._array(t, torch.int32, (self.batch,), self._dev, what)

    def _here(self, t: torch.Tensor, what: str) -> int:
        """The address of a tensor that has its type and shape checked elsewhere, on the cache's device."""
        if t.get_device() != self._dev:
            raise core.NsrlError(f"{what} is on {t.device}, the cache on {self.device}")
        return t.data_ptr()

    def _stream(self) -> int:
        if torch.cuda.current_device() != self._dev:
            raise core.NsrlError(f"the cache is on {self.device}, not on the current device")
        return core._raw_stream(self._dev)

    # ---- enqueue only
    def launch_append(self, k, v, starts, counts, positions, status: core.Status) -> int:
        """k, v: int16 [batch * tokens, heads * head_dim] of one row stride; counts
        and positions may be None (nsrl_q4_cache_append)."""
        rows, cols = k.shape[0], self._cols
        if rows % max(1, self.batch) or k.shape[1] != cols or v.shape[1] != cols:
            raise core.NsrlError("k and v must be [batch * tokens, heads * head_dim]")
        stream = self._stream()
        (kp, ld), (vp, vld) = core._rows(k, rows, cols, self._dev, "k"), core._rows(v, rows, cols, self._dev, "v")
        if rows > 1 and vld != ld:
            raise core.NsrlError("k and v must have one row stride")
        return _lib().nsrl_q4_cache_append(self._ref, kp, vp, ld, rows // max(1, self.batch),
                                           self._per_sequence(starts, "starts"),
                                           None if counts is None else self._per_sequence(counts, "counts"),
                                           None if positions is None else self._per_sequence(positions, "positions"),
                                           self._here(status.buf, "the status"), stream)

    def launch_read(self, starts, k, v, status: core.Status) -> int:
        """k, v: int16 [batch, heads, tokens, head_dim], written (nsrl_q4_cache_read)."""
        if k.dim() != 4:
            raise core.NsrlError("k must be [batch, heads, tokens, head_dim]")
        stream, tokens = self._stream(), k.shape[2]
        shape = (self.batch, self.heads, tokens, self.head_dim)
        return _lib().nsrl_q4_cache_read(self._ref, None if starts is None else self._per_sequence(starts, "starts"),
                                         tokens, core._array(k, torch.int16, shape, self._dev, "k"),
                                         core._array(v, torch.int16, shape, self._dev, "v"),
                                         self._here(status.buf, "the status"), stream)

    def attend_workspace_bytes(self) -> int:
        return self._ws_bytes

    def launch_attend(self, q, lens, ctx, status: core.Status, ws=None) -> int:
        """q: int16 [batch, heads * head_dim] rows, ctx likewise and contiguous; ws:
        attend_workspace_bytes() of uint8, the cache's own by default
        (nsrl_attention_decode_q4)."""
        stream, cols = self._stream(), self._cols
        wp, wn = self._ws_ptr, self._ws_bytes
        if ws is not None:
            wp, wn = core._array(ws, torch.uint8, ws.shape, self._dev, "the workspace"), ws.numel()
        qp, ldq = core._rows(q, self.batch, cols, self._dev, "q")
        if q.shape[1] != cols:
            raise core.NsrlError("q must be [batch, heads * head_dim]")
        return _lib().nsrl_attention_decode_q4(qp, ldq, self._ref, self._per_sequence(lens, "lens"),
                                               core._array(ctx, torch.int16, (self.batch, cols), self._dev, "ctx"),
                                               wp, wn, self._here(status.buf, "the status"), stream)

    def evict_workspace_bytes(self, keep: int) -> int:
        return _lib().nsrl_q4_cache_evict_workspace_size(self._ref, keep)

    def launch_evict(self, lens, next_positions, keep, sinks, recent, scores_out, positions_out, lens_out, ws,
                     status: core.Status) -> int:
        """nsrl_q4_cache_evict; the outputs may be lens and the cache's own scores and positions."""
        stream, shape = self._stream(), (self.batch, self.heads, self.capacity)
        return _lib().nsrl_q4_cache_evict(
            self._ref, self._per_sequence(lens, "lens"), self._per_sequence(next_positions, "next_positions"), keep,
            sinks, recent, core._array(scores_out, torch.int32, shape, self._dev, "scores_out"),
            core._array(positions_out, torch.int32, shape, self._dev, "positions_out"),
            self._per_sequence(lens_out, "lens_out"), core._array(ws, torch.uint8, ws.shape, self._dev, "the workspace"),
            ws.numel(), self._here(status.buf, "the status"), stream)

    # ---- checked calls
    def append(self, k, v, starts, counts=None, positions=None) -> Optional[bool]:
        """Quantises the rows into the slots from starts[b]; True, or None when a sequence does not fit."""
        st = core.Status()
        h = core._run(lambda: self.launch_append(k, v, starts, counts, positions, st), st)
        return None if h is None else True

    def read(self, tokens: int, starts=None):
        """(k, v) int16 [batch, heads, tokens, head_dim] of the slots from starts[b] (0), or None."""
        k, v = (torch.empty((self.batch, self.heads, tokens, self.head_dim), dtype=torch.int16, device=self.device)
                for _ in range(2))
        st = core.Status()
        h = core._run(lambda: self.launch_read(starts, k, v, st), st)
        return None if h is None else (k, v)

    def attend(self, q, lens) -> Optional[torch.Tensor]:
        """The context rows [batch, heads * head_dim] of q over the first lens[b] slots, or None."""
        ctx = torch.empty((self.batch, self.heads * self.head_dim), dtype=torch.int16, device=self.device)
        ws = torch.empty(self._ws_bytes, dtype=torch.uint8, device=self.device) if self._ws_bytes else None
        st = core.Status()
        h = core._run(lambda: self.launch_attend(q, lens, ctx, st, ws), st)
        return None if h is None else ctx

    def evict(self, lens, next_positions, keep: int, sinks: int = 4, recent: int = 0) -> Optional[bool]:
        """Cuts every (sequence, head) to `keep` slots in place, lens included; True, or None."""
        nbytes = self.evict_workspace_bytes(keep)
        ws = torch.empty(max(256, nbytes), dtype=torch.uint8, device=self.device)
        if self.scores is None or self.positions is None:
            return None
        st = core.Status()
        h = core._run(lambda: self.launch_evict(lens, next_positions, keep, sinks, recent, self.scores,
                                                self.positions, lens, ws, st), st)
        return None if h is None else True


def prenorm_attention_decode_block_q4(x, rms_gamma, rms_eps, q, k, v, o, cache: Q4Cache, lens, positions=None,
                                      rotary: Optional[Rotary] = None):
    """One decode step of the prenorm attention block over a 4-bit cache
    (nsrl_prenorm_attention_decode_block_q4): x [B, d]; slot lens[b] of every
    head is written, then attended with the ones before it.  positions: of the
    new tokens (lens by default); returns (y, saturations) or None."""
    L = _lib()
    x, g = core._i16(x), core._i16(rms_gamma)
    B, d = x.shape
    if B != cache.batch or g.numel() != d:
        raise core.NsrlError("x must be [cache.batch, d] and rms_gamma [d]")
    if rotary is not None:
        if rotary.head_dim != cache.head_dim:
            raise core.NsrlError(f"the rotary plan is for head_dim {rotary.head_dim}, the cache has {cache.head_dim}")
        if rotary.turns.get_device() != cache._dev:
            raise core.NsrlError(f"the rotary plan is on {rotary.turns.device}, the cache on {cache.device}")
    stream = cache._stream()
    for name, lin in zip("qkvo", (q, k, v, o)):
        for t in (lin.weights, lin.scales) + (() if lin.bias is None else (lin.bias,)):
            cache._here(t, f"the {name} projection")
    xp, _ = core._rows(x, B, d, cache._dev, "x")
    gp = cache._here(g, "rms_gamma")
    lp = cache._per_sequence(lens, "lens")
    pp = None if positions is None else cache._per_sequence(positions, "positions")
    y = torch.empty_like(x)
    # of its own, so that blocks on two caches may run at once
    ws = torch.empty(max(256, L.nsrl_decode_block_q4_workspace_size(cache._ref)), dtype=torch.uint8, device=cache.device)
    st = core.Status()
    ps = [l.c() for l in (q, k, v, o)]
    h = core._run(lambda: L.nsrl_prenorm_attention_decode_block_q4(
        xp, B, d, cache.heads, gp, rms_eps, *[C.byref(p) for p in ps],
        None if rotary is None else C.byref(rotary.c()), cache._ref, lp, pp, y.data_ptr(), ws.data_ptr(), ws.numel(),
        st.buf.data_ptr(), stream), st)
    return None if h is None else (y, h.attention_saturations)
