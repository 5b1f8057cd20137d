"""The captured calls' look at the living graphs, while another thread's forward adds one (CPU)."""

import threading
import weakref

import torch

from ksdraft_amd import _lib


def test_another_thread_adds(monkeypatch):
    dev, leaves, kept, capturing = torch.device("cpu"), [torch.zeros(2, requires_grad=True) for _ in range(6)], [], {}

    def add():
        kept.append(_lib.capture_guard(dev, leaves[5]))

    class Watched(weakref.WeakSet):
        def __iter__(self):
            for n, item in enumerate(super().__iter__()):
                if n == 1:
                    t = threading.Thread(target=add)
                    t.start()
                    t.join(0.3)  # it has added, or waits for this look to end
                    threads.append(t)
                yield item
    threads = []
    monkeypatch.setattr(_lib, "_eager_graphs", Watched())
    monkeypatch.setattr(_lib, "stream_ptr", lambda d: threading.get_ident())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing.get(threading.get_ident(), False))
    for p in leaves[:4]:
        kept.append(_lib.capture_guard(dev, p))
    capturing[threading.get_ident()] = True
    assert _lib.capture_guard(dev, leaves[4]) is None
    assert len(threads) == 1
    threads[0].join(20)
    assert len(kept) == 5 and len(_lib._eager_graphs) == 5
