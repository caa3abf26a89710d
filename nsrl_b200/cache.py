"""The 4-bit KV cache: append, attention over it, eviction by accumulated
attention weight, and the decode block that uses them (include/nsrl_b200.h).

A slot of 64 dims takes 80 bytes (key and value) where the int16 cache takes
256.  The attention gives, on the values the codes stand for, exactly what
`core.attention_decode` gives on int16 ones.

`launch_*` methods enqueue on the current stream and return the C status code
without waiting (they may be captured into a graph; the device status tells
rejections later).  The methods without the prefix wait and return None when
the call was rejected, as the functions of `core` do.
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
        L.nsrl_attention_decode_q4.argtypes = [vp, sz, cp, vp, vp, vp, vp]
        L.nsrl_q4_cache_evict_workspace_size.restype = sz
        L.nsrl_q4_cache_evict_workspace_size.argtypes = [cp, sz]
        L.nsrl_q4_cache_evict.argtypes = [cp, vp, vp, sz, sz, sz, vp, vp, vp, vp, sz, vp, vp]
        L.nsrl_decode_block_q4_workspace_size.restype = sz
        L.nsrl_decode_block_q4_workspace_size.argtypes = [sz, sz, sz]
        L.nsrl_prenorm_attention_decode_block_q4.argtypes = [vp, sz, sz, sz, vp, C.c_uint64, lp, lp, lp, lp,
                                                             C.POINTER(RotaryC), cp, vp, vp, vp, vp, sz, vp, vp]
        L._q4_bound = True
    return L


def _array(t: torch.Tensor, dtype, shape, what: str) -> int:
    """The address of a contiguous tensor on the current device, of this type and shape."""
    core._on_current_device(t, dtype, what)
    if tuple(t.shape) != shape or not t.is_contiguous():
        raise core.NsrlError(f"{what} must be contiguous and of shape {shape}")
    return t.data_ptr()


def _rows(t: torch.Tensor, rows: int, cols: int, what: str) -> tuple[int, int]:
    core._on_current_device(t, torch.int16, what)
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] != cols or (cols > 1 and t.stride(1) != 1):
        raise core.NsrlError(f"{what} must be [{rows}, {cols}] with contiguous columns")
    return t.data_ptr(), core._row_stride(t)


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
        self.device = k_codes.device
        ptr = [_array(k_codes, torch.uint8, (B, H, cap, half), "k_codes"),
               _array(v_codes, torch.uint8, (B, H, cap, half), "v_codes"),
               _array(k_scales, torch.int32, (B, H, cap, groups), "k_scales"),
               _array(v_scales, torch.int32, (B, H, cap, groups), "v_scales"),
               None if scores is None else _array(scores, torch.int32, (B, H, cap), "scores"),
               None if positions is None else _array(positions, torch.int32, (B, H, cap), "positions")]
        self._c = Q4CacheC(*ptr, B, H, self.head_dim, cap)
        self._ref = C.byref(self._c)

    def c(self) -> Q4CacheC:
        return self._c

    def _per_sequence(self, t: Optional[torch.Tensor], what: str) -> Optional[int]:
        return None if t is None else _array(t, torch.int32, (self.batch,), what)

    # ---- enqueue only
    def launch_append(self, k, v, starts, counts=None, positions=None, status: core.Status = None) -> int:
        """k, v: int16 [batch * tokens, heads * head_dim] of one row stride (nsrl_q4_cache_append)."""
        rows = k.shape[0]
        if rows % max(1, self.batch):
            raise core.NsrlError("k must hold the same number of rows for every sequence")
        cols = self.heads * self.head_dim
        kp, ld = _rows(k, rows, cols, "k")
        vp, ldv = _rows(v, rows, cols, "v")
        if rows > 1 and ld != ldv:
            raise core.NsrlError("k and v must have one row stride")
        self._here()
        return _lib().nsrl_q4_cache_append(self._ref, kp, vp, ld, rows // max(1, self.batch),
                                           self._per_sequence(starts, "starts"), self._per_sequence(counts, "counts"),
                                           self._per_sequence(positions, "positions"), status.buf.data_ptr(),
                                           core._stream())

    def launch_read(self, starts, k, v, status: core.Status) -> int:
        """k, v: int16 [batch, heads, tokens, head_dim], written (nsrl_q4_cache_read)."""
        if k.dim() != 4:
            raise core.NsrlError("k must be [batch, heads, tokens, head_dim]")
        shape = (self.batch, self.heads, k.shape[2], self.head_dim)
        kp, vp = _array(k, torch.int16, shape, "k"), _array(v, torch.int16, shape, "v")
        self._here()
        return _lib().nsrl_q4_cache_read(self._ref, self._per_sequence(starts, "starts"), k.shape[2], kp, vp,
                                         status.buf.data_ptr(), core._stream())

    def launch_attend(self, q, lens, ctx, status: core.Status) -> int:
        """q: int16 [batch, heads * head_dim] rows, ctx likewise and contiguous (nsrl_attention_decode_q4)."""
        cols = self.heads * self.head_dim
        qp, ldq = _rows(q, self.batch, cols, "q")
        cp = _array(ctx, torch.int16, (self.batch, cols), "ctx")
        self._here()
        return _lib().nsrl_attention_decode_q4(qp, ldq, self._ref, self._per_sequence(lens, "lens"), cp,
                                               status.buf.data_ptr(), core._stream())

    def evict_workspace_bytes(self, keep: int) -> int:
        return _lib().nsrl_q4_cache_evict_workspace_size(self._ref, keep)

    def launch_evict(self, lens, next_positions, keep, sinks, recent, scores_out, positions_out, lens_out, ws,
                     status: core.Status) -> int:
        """nsrl_q4_cache_evict; the outputs may be lens and the cache's own scores and positions."""
        shape = (self.batch, self.heads, self.capacity)
        core._on_current_device(ws, torch.uint8, "the workspace")
        self._here()
        return _lib().nsrl_q4_cache_evict(
            self._ref, self._per_sequence(lens, "lens"), self._per_sequence(next_positions, "next_positions"), keep,
            sinks, recent, _array(scores_out, torch.int32, shape, "scores_out"),
            _array(positions_out, torch.int32, shape, "positions_out"), self._per_sequence(lens_out, "lens_out"),
            ws.data_ptr(), ws.numel(), status.buf.data_ptr(), core._stream())

    def _here(self):
        if self.device.index != torch.cuda.current_device():
            raise core.NsrlError(f"the cache is on {self.device}, not on the current device")

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
        st = core.Status()
        h = core._run(lambda: self.launch_attend(q, lens, ctx, st), st)
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
    core._on_current_device(x, torch.int16, "x")
    cache._here()
    y = torch.empty_like(x)
    ws = core.workspace(L.nsrl_decode_block_q4_workspace_size(B, d, cache.heads))
    st = core.Status()
    ps = [l.c() for l in (q, k, v, o)]
    h = core._run(lambda: L.nsrl_prenorm_attention_decode_block_q4(
        x.data_ptr(), B, d, cache.heads, g.data_ptr(), rms_eps, *[C.byref(p) for p in ps],
        None if rotary is None else C.byref(rotary.c()), cache._ref, cache._per_sequence(lens, "lens"),
        cache._per_sequence(positions, "positions"), y.data_ptr(), ws.data_ptr(), ws.numel(), st.buf.data_ptr(),
        core._stream()), st)
    return None if h is None else (y, h.attention_saturations)
