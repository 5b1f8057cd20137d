"""What the adapters' C entries refuse (CPU)."""

import ctypes

from ksdraft_amd import _lib

P = ctypes.c_void_p(256)  # never dereferenced


def forward(x=P, dtype=0, M=4, K=8, stride=8, a=P, n=2, r=4, N=16, index=P, per=1, base=P, base_stride=16, drop=0, stream_id=0, y=P, groups=None,
            size=0):
    return _lib.load().ksd_adapter_linear(x, dtype, M, K, stride, a, P, n, r, N, index, 1, per, P, base, base_stride, drop, 1, None,
                                          stream_id, y, None, groups, size, None)


def backward(dtype=0, M=4, N=16, stride=16, K=8, hidden=P, n=2, r=4, per=1, drop=0, work=P, size=1 << 50, da=P, groups=P,
             groups_size=1 << 50):
    return _lib.load().ksd_adapter_linear_backward(P, dtype, M, N, stride, P, K, 8, hidden, groups, groups_size, P, P, n, r, P, 1, per, P, None, 0, drop, 1,
                                                   None, 0, P, da, P, work, size, None)


def test_forward():
    assert forward(M=0) == 0
    assert forward(M=600000) == 1 and forward(M=600000, groups=P, size=64) == 1 and forward(M=600000, groups=ctypes.c_void_p(8), size=1 << 40) == 1
    for bad in (dict(M=-1), dict(K=0), dict(N=0), dict(r=0), dict(r=129), dict(n=0), dict(n=1 << 16), dict(per=0), dict(stride=7),
                dict(base_stride=15), dict(drop=65537), dict(drop=-1), dict(stream_id=-1), dict(x=None), dict(a=None), dict(index=None),
                dict(y=None), dict(M=1 << 31), dict(K=1 << 31), dict(N=1 << 31)):
        assert forward(**bad) == 1, bad
    assert forward(dtype=3) == 2


def test_backward():
    for bad in (dict(M=-1), dict(K=0), dict(N=0), dict(r=129), dict(n=0), dict(per=0), dict(stride=15), dict(hidden=None),
                dict(drop=70000), dict(work=None), dict(size=16), dict(work=ctypes.c_void_p(8)), dict(M=1 << 25), dict(da=None),
                dict(M=600000, groups=None), dict(M=600000, groups_size=64), dict(M=600000, groups=ctypes.c_void_p(8))):
        assert backward(**bad) == 1, bad
    assert backward(dtype=9) == 2
    need = ctypes.c_int64()
    f = _lib.load().ksd_adapter_linear_backward_workspace
    assert f(4, 8, 16, 4, 2, 1, 0, ctypes.byref(need)) == 0 and need.value > 0
    assert f(0, 8, 16, 4, 2, 1, 0, ctypes.byref(need)) == 0
    assert _lib.load().ksd_adapter_linear_workspace(0, 8, 16, 4, 2, 1, 0, ctypes.byref(need)) == 0 and need.value == 0
    assert f(4, 8, 16, 4, 2, 1, 7, ctypes.byref(need)) == 1 and f(4, 8, 16, 0, 2, 1, 0, ctypes.byref(need)) == 1
    assert f(4, 8, 16, 4, 2, 0, 0, ctypes.byref(need)) == 1 and f(4, 8, 16, 4, 2, 1, 0, None) == 1


def test_capture_guard(monkeypatch):
    """A captured call on a leaf of a living eager graph of another stream is refused."""
    import gc

    import pytest
    import torch
    dev = torch.device("cpu")
    at = dict(stream=1, capturing=False)
    monkeypatch.setattr(_lib, "stream_ptr", lambda d: at["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: at["capturing"])
    p, q = (torch.zeros(2, requires_grad=True) for _ in range(2))
    assert _lib.capture_guard(dev, torch.zeros(2), None, p * 2) is None  # no leaf that takes a gradient
    kept = _lib.capture_guard(dev, p, None)
    at["capturing"] = True
    assert _lib.capture_guard(dev, p) is None  # the same stream
    at["stream"] = 2
    assert _lib.capture_guard(dev, q) is None
    with pytest.raises(RuntimeError):
        _lib.capture_guard(dev, q, p)
    del kept
    gc.collect()
    assert _lib.capture_guard(dev, q, p) is None


def test_capture_guard_sees_through_a_cast(monkeypatch):
    """Adapters kept in fp32 and used in 16 bits: the leaf is the fp32 one."""
    import pytest
    import torch
    dev = torch.device("cpu")
    at = dict(stream=1, capturing=False)
    monkeypatch.setattr(_lib, "stream_ptr", lambda d: at["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: at["capturing"])
    seen = []

    class Guarded(torch.autograd.Function):
        @staticmethod
        def forward(ctx, t):
            ctx.guard = _lib.capture_guard(dev, t)
            seen.append(ctx.guard)
            return t * 2

        @staticmethod
        def backward(ctx, g):
            return g * 2

    p, q = (torch.zeros(2, requires_grad=True) for _ in range(2))
    y = Guarded.apply(p.to(torch.bfloat16))
    assert seen[0] is not None and seen[0].leaves == {id(p)}
    at.update(stream=2, capturing=True)
    Guarded.apply(q.to(torch.bfloat16))
    with pytest.raises(RuntimeError):
        Guarded.apply(p.to(torch.float16))
    del y
    seen.clear()
    Guarded.apply(p.to(torch.float16))
