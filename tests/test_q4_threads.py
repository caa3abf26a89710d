"""Attention calls on one cache from several threads: each works in a workspace of its own."""
import threading

import pytest
import torch


@pytest.fixture
def cache(monkeypatch):
    """A cache handle in host memory whose launches are recorded, not made."""
    from nsrl_b200 import cache as K, core

    class Status:
        buf = torch.zeros(8, dtype=torch.int64)

        def fetch(self):
            return core.NSRL_OK, core.DeviceStatusC()

    monkeypatch.setattr(core, "Status", Status)
    c = K.Q4Cache.__new__(K.Q4Cache)
    c.batch, c.heads, c.head_dim, c.capacity = 2, 2, 64, 40000
    c.device, c._cols = torch.device("cpu"), 128
    c._ws_bytes = 4096
    c._ws = torch.empty(c._ws_bytes, dtype=torch.uint8)
    c._ws_ptr = c._ws.data_ptr()
    return c


def test_checked_calls_do_not_share_a_workspace(cache, monkeypatch):
    from nsrl_b200 import cache as K, core
    both, seen = threading.Barrier(2, timeout=20), []

    def launch_attend(self, q, lens, ctx, status, ws=None):
        seen.append((self._ws_ptr if ws is None else ws.data_ptr(), self._ws_bytes if ws is None else ws.numel()))
        both.wait()  # the other call's workspace is in use too
        return core.NSRL_OK

    monkeypatch.setattr(K.Q4Cache, "launch_attend", launch_attend)
    q, lens = torch.zeros((2, 128), dtype=torch.int16), torch.ones(2, dtype=torch.int32)
    calls = [threading.Thread(target=lambda: cache.attend(q, lens)) for _ in range(2)]
    for t in calls:
        t.start()
    for t in calls:
        t.join()
    assert len(seen) == 2 and all(n >= cache._ws_bytes for _, n in seen)
    (a, n), (b, m) = sorted(seen)
    assert a + n <= b


def test_a_small_cache_needs_none(cache, monkeypatch):
    from nsrl_b200 import cache as K, core
    cache._ws, cache._ws_ptr, cache._ws_bytes = None, None, 0
    monkeypatch.setattr(K.Q4Cache, "launch_attend", lambda self, q, lens, ctx, status, ws=None: core.NSRL_OK if ws is None else 1)
    q, lens = torch.zeros((2, 128), dtype=torch.int16), torch.ones(2, dtype=torch.int32)
    assert cache.attend(q, lens).shape == (2, 128)


def test_decode_blocks_do_not_share_a_workspace(monkeypatch):
    """Two caches, two threads: the library's calls are recorded, not made."""
    from nsrl_b200 import cache as K, core
    both, seen = threading.Barrier(2, timeout=20), []

    class Lib:
        def nsrl_decode_block_q4_workspace_size(self, ref):
            return 4096

        def nsrl_prenorm_attention_decode_block_q4(self, *args):
            seen.append(args[-4:-2])
            both.wait()
            return core.NSRL_OK

    class Status:
        buf = torch.zeros(8, dtype=torch.int64)

        def fetch(self):
            return core.NSRL_OK, core.DeviceStatusC()

    class Params:
        weights, scales, bias = torch.zeros((128, 128), dtype=torch.int8), torch.zeros((128, 2), dtype=torch.int32), None

        def c(self):
            return core.LinearParamsC()

    monkeypatch.setattr(core, "Status", Status)
    monkeypatch.setattr(core, "_dev", lambda: torch.device("cpu"))
    monkeypatch.setattr(core, "_i16", lambda t: t)
    monkeypatch.setattr(core, "_rows", lambda t, rows, cols, dev, what: (t.data_ptr(), cols))
    monkeypatch.setattr(core, "_array", lambda t, dtype, shape, dev, what: t.data_ptr())
    monkeypatch.setattr(core, "_ws_cache", {})
    monkeypatch.setattr(K, "_lib", Lib)
    monkeypatch.setattr(K.Q4Cache, "_stream", lambda self: 0)
    x, g, lens = torch.zeros((2, 128), dtype=torch.int16), torch.zeros(128, dtype=torch.int16), torch.ones(2, dtype=torch.int32)

    def call():
        c = K.Q4Cache.__new__(K.Q4Cache)
        c.batch, c.heads, c.head_dim, c.device, c._dev = 2, 2, 64, torch.device("cpu"), -1
        c._c = K.Q4CacheC()
        c._ref = K.C.byref(c._c)
        K.prenorm_attention_decode_block_q4(x, g, 1, *[Params()] * 4, c, lens)

    calls = [threading.Thread(target=call) for _ in range(2)]
    for t in calls:
        t.start()
    for t in calls:
        t.join()
    assert len(seen) == 2
    (a, n), (b, m) = sorted(seen)
    assert n >= 4096 and m >= 4096 and a + n <= b
