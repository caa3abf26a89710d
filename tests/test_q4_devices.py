"""Calls over the 4-bit cache refuse parameters and status words that are not on
the cache's device (the kernels would read another memory's addresses).  On the
CPU: the library's calls are recorded, not made, and a cache on device 0 meets
tensors in host memory."""
import pytest
import torch


class There:
    """A tensor's stand-in on device 0."""

    def __init__(self, t):
        self.t, self.device, self.shape = t, "cuda:0", t.shape

    def get_device(self):
        return 0

    def data_ptr(self):
        return self.t.data_ptr()

    def numel(self):
        return self.t.numel()


class Status:
    def __init__(self, here=True):
        buf = torch.zeros(8, dtype=torch.int64)
        self.buf = There(buf) if here else buf

    def fetch(self):
        from nsrl_b200 import core
        return core.NSRL_OK, core.DeviceStatusC()


@pytest.fixture
def made(monkeypatch):
    """(cache, names of the library's calls)."""
    from nsrl_b200 import cache as K, core
    names = []

    class Lib:
        def __getattr__(self, name):
            def call(*args):
                names.append(name)
                return 4096 if name.endswith("size") else core.NSRL_OK
            return call

    monkeypatch.setattr(K, "_lib", Lib)
    monkeypatch.setattr(K.Q4Cache, "_stream", lambda self: 0)
    monkeypatch.setattr(core, "Status", Status)
    monkeypatch.setattr(core, "_i16", lambda t: t)
    monkeypatch.setattr(core, "_rows", lambda t, rows, cols, dev, what: (t.data_ptr(), cols))
    real = core._array
    monkeypatch.setattr(core, "_array", lambda t, dtype, shape, dev, what: real(t, dtype, shape, dev, what)
                        if what == "rms_gamma" else t.data_ptr())
    c = K.Q4Cache.__new__(K.Q4Cache)
    c.batch, c.heads, c.head_dim, c.capacity, c._cols = 2, 2, 64, 64, 128
    c.device, c._dev, c._ws_ptr, c._ws_bytes = torch.device("cpu"), 0, None, 0
    c._c = K.Q4CacheC()
    c._ref = K.C.byref(c._c)
    return c, names


def linear(**there):
    from nsrl_b200 import core

    class Params:
        weights, scales, bias = (There(torch.zeros((128, 128), dtype=torch.int8)),
                                 There(torch.zeros((128, 2), dtype=torch.int32)), None)

        def c(self):
            return core.LinearParamsC()

    p = Params()
    for name, t in there.items():
        setattr(p, name, t)
    return p


I16 = torch.zeros((2, 128), dtype=torch.int16)
I32 = torch.ones(2, dtype=torch.int32)


@pytest.mark.parametrize("which,bad", [(i, b) for i in range(4) for b in (
    dict(weights=torch.zeros((128, 128), dtype=torch.int8)), dict(scales=torch.zeros((128, 2), dtype=torch.int32)),
    dict(bias=torch.zeros(128, dtype=torch.int32)))])
def test_block_refuses_linears(made, which, bad):
    from nsrl_b200 import cache as K, core
    c, names = made
    ps = [linear() for _ in range(4)]
    ps[which] = linear(**bad)
    with pytest.raises(core.NsrlError):
        K.prenorm_attention_decode_block_q4(I16, gamma(), 1, *ps, c, I32)
    assert "nsrl_prenorm_attention_decode_block_q4" not in names


def gamma():
    """What _array takes for a contiguous int16 tensor on device 0."""
    class Gamma(torch.Tensor):
        def get_device(self):
            return 0
    return torch.zeros(128, dtype=torch.int16).as_subclass(Gamma)


def test_block_takes_what_is_there_and_refuses_the_gamma(made):
    from nsrl_b200 import cache as K, core
    c, names = made
    assert K.prenorm_attention_decode_block_q4(I16, gamma(), 1, *[linear() for _ in range(4)], c, I32) is not None
    assert "nsrl_prenorm_attention_decode_block_q4" in names
    names.clear()
    with pytest.raises(core.NsrlError):
        K.prenorm_attention_decode_block_q4(I16, torch.zeros(128, dtype=torch.int16), 1, *[linear() for _ in range(4)], c, I32)
    assert "nsrl_prenorm_attention_decode_block_q4" not in names


def test_launches_refuse_a_status_elsewhere(made):
    from nsrl_b200 import core
    c, names = made
    kv = torch.zeros((2, 2, 1, 64), dtype=torch.int16)
    ws = torch.zeros(256, dtype=torch.uint8)
    launches = [lambda st: c.launch_append(I16, I16, I32, None, None, st), lambda st: c.launch_read(None, kv, kv, st),
                lambda st: c.launch_attend(I16, I32, I16, st),
                lambda st: c.launch_evict(I32, I32, 8, 0, 0, I32, I32, I32, ws, st)]
    for launch in launches:
        names.clear()
        assert launch(Status()) == core.NSRL_OK and len(names) == 1
        with pytest.raises(core.NsrlError):
            launch(Status(here=False))
        assert len(names) == 1
