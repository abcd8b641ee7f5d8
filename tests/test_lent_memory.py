"""Views of memory that the library owns, and what may be closed while they live: the Python twin over a device
without a GPU, whose closing entries are written down.  Memory goes after its last view, and what it hangs on after it."""
import itertools
import threading

import numpy as np
import pytest

from rstr import hip
from test_pool_ops_refusals import fake_lib, pool, pytestmark  # noqa: F401


class Recorder:
    """The device without a GPU, with the closing entries written down; its decoder is one address."""

    def __init__(self, real):
        self._real, self.closed, self._logits = real, [], np.zeros((2, 512), np.float32)

    def __getattr__(self, name):
        f = getattr(self._real, name)
        if not name.endswith("_close"):
            return f

        def close(h):
            rc = f(h)
            if rc == 0:
                self.closed.append(name[5:-6])
            return rc

        return close

    def rstr_decoder_open(self, model, pool, batch, pps, maxpos, split, out):
        out._obj.value = 1
        return 0

    rstr_prefill_open = rstr_decoder_open

    def rstr_decode_logits_device(self, h, out):
        out._obj.value = self._logits.ctypes.data
        return 0

    def rstr_decoder_close(self, h):
        self.closed.append("decoder")
        return 0


@pytest.fixture
def rec(fake_lib, monkeypatch):  # noqa: F811
    r = Recorder(fake_lib)
    monkeypatch.setattr(hip, "_lib", r)
    return r


def opened(s):
    p = pool(s)
    b = hip.BlockBounds(p)
    return p.model, p, b, hip.Decoder(p.model, p, 2, 2, 32)


def views_of(p, b, d):
    return dict(keys=p.pages_device(0, 0), values=p.pages_device(1, 1), bounds=b.device(1), logits=d.logits_device())


def test_closed_without_views(rec):
    """Without views memory goes with its handle, and a model's with what is over it."""
    with hip.Session(0) as s:
        m, p, b, d = opened(s)
        views_of(p, b, d)
        for x, name in ((d, "decoder"), (b, "bounds"), (p, "pool"), (m, "model")):
            x.close()
            x.close()
            assert rec.closed[-1] == name and not x.h
        assert s.children == []
    assert rec.closed == ["decoder", "bounds", "pool", "model", "session"]


@pytest.mark.parametrize("held", ["keys", "values", "bounds", "logits"])
def test_session_closed_under_a_view(rec, held):
    """What the view shows stays, and what that hangs on; all else goes with the session."""
    s = hip.Session(0)
    _, p, b, d = opened(s)
    view = views_of(p, b, d)[held]
    s.close()
    hangs = dict(keys=["pool"], values=["pool"], bounds=["bounds", "pool"], logits=["decoder", "pool"])[held] + ["model", "session"]
    assert sorted(rec.closed) == sorted({"decoder", "bounds", "pool", "model", "session"} - set(hangs))
    n = len(rec.closed)
    view.data_ptr(), view.__cuda_array_interface__
    del view
    assert rec.closed[n:] == hangs
    s.close()
    assert len(rec.closed) == 5


def test_every_order(rec):
    """Handles and views, ended in any order: each piece of memory goes once, after all views of it and all that hangs on it."""
    what = ["m", "p", "b", "d", "keys", "bounds", "logits"]
    orders = list(itertools.permutations(what))
    np.random.default_rng(3).shuffle(orders)
    for order in orders[:300]:
        rec.closed.clear()
        s = hip.Session(0)
        m, p, b, d = opened(s)
        views = views_of(p, b, d)
        del views["values"]
        live, refused = dict(m=m, p=p, b=b, d=d, **views), []
        del m, p, b, d, views
        for x in order:
            y = live.pop(x)
            if x in "mpbd":
                try:
                    y.close()
                except hip.RstrError as e:
                    assert x == "p" and "b" in live and e.code == -4
                    refused.append(y)
            del y
            ended = set(order[:order.index(x) + 1]) - ({"p"} if refused else set())
            assert ("decoder" in rec.closed) == ({"d", "logits"} <= ended)
            assert ("bounds" in rec.closed) == ({"b", "bounds"} <= ended)
            assert ("pool" in rec.closed) == ({"p", "keys", "b", "bounds", "d", "logits"} <= ended)
            assert ("model" in rec.closed) == ({"m", "p", "keys", "b", "bounds", "d", "logits"} <= ended)
        s.close()
        assert sorted(rec.closed) == ["bounds", "decoder", "model", "pool", "session"] and rec.closed[-1] == "session"


def test_ended_handles(rec):
    """A closed handle takes no calls while views keep its memory, and a pool stays open for plans and bounds under views too."""
    with hip.Session(0) as s:
        m, p, b, d = opened(s)
        sel, plan = hip.BlockSelect(b, 4, 2, 5, 7), hip.PagedAttention(p, 4, 2, 5)
        views = views_of(p, b, d)
        with pytest.raises(hip.RstrError, match="open selections") as e:
            b.close()
        assert e.value.code == -4
        sel.close()
        b.close()
        with pytest.raises(hip.RstrError, match="open attention plans"):
            p.close()
        plan.close()
        p.close()
        assert rec.closed == ["select", "pool_attn"] and views["bounds"].shape == (4, 2, 2, 128)
        for call in (lambda: b.device(0), lambda: p.pages_device(0, 0), lambda: hip.BlockBounds(p), lambda: hip.PagedAttention(p, 4, 2, 5)):
            with pytest.raises(hip.RstrError):
                call()
        views.clear()
        assert rec.closed == ["select", "pool_attn", "bounds"]  # (the decoder is open)
    assert rec.closed == ["select", "pool_attn", "bounds", "decoder", "pool", "model", "session"]


def test_views_that_die_on_other_threads(rec):
    s = hip.Session(0)
    _, p, b, d = opened(s)
    views = [[f() for f in (lambda: p.pages_device(0, 0), lambda: b.device(0)) for _ in range(200)] for _ in range(8)]
    s.close()
    threads = [threading.Thread(target=v.clear) for v in views]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert rec.closed == ["decoder", "bounds", "pool", "model", "session"]


def test_memory_of_a_capture(rec, monkeypatch):
    """Nothing is freed while the stream is captured (freeing waits for the device), but with what leaves next."""
    import torch
    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    s = hip.Session(0)
    _, p, b, d = opened(s)
    view = p.pages_device(0, 0)
    for x in (d, b, p):
        x.close()
    assert rec.closed == ["decoder", "bounds"]
    capturing[0] = True
    del view
    assert rec.closed == ["decoder", "bounds"]
    capturing[0] = False
    s.close()
    assert rec.closed == ["decoder", "bounds", "pool", "model", "session"]
