"""The C handles behind decoders and plans against their engine's, in every order that Python may close or
collect them: each is closed once, and before the engine that it uses.  On a stand-in for the library, since
what goes wrong otherwise is a read of freed memory."""
import gc

import numpy as np
import pytest


class FakeLibrary:
    """Opens handles 1, 2, ... and keeps a log of what is closed; every other call succeeds."""

    def __init__(self):
        self.log, self.kind, self.next = [], {}, 1

    def __getattr__(self, name):
        if name.endswith("_close") or name == "eii_close":
            return lambda h: self.log.append((name, h.value))

        def call(*args):
            if "open" in name:
                args[-1]._obj.value = self.next
                self.kind[self.next] = name
                self.next += 1
            return 0
        return call


@pytest.fixture
def fake(monkeypatch):
    import _eii
    f = FakeLibrary()
    monkeypatch.setattr(_eii, "_lib", f)
    gc.collect()
    yield f
    gc.collect()


OPEN = {
    "eii_decoder_close": lambda m, e: m.Decoder(e, 1, 8),
    "eii_paged_decoder_close": lambda m, e: m.PagedDecoder(e, 16, 16, 4),
    "eii_linear_plan_close": lambda m, e: m.LinearPlan(e, np.zeros((16, 32), np.int8), np.ones(16), np.ones(16), 16, 0, 0, 16),
}


@pytest.mark.parametrize("close", OPEN)
def test_engine_closed_first(fake, close):
    """engine.close(), then the object is collected: nothing is closed on a freed engine."""
    import _eii
    e = _eii.Engine("model", 0)
    d = OPEN[close](_eii, e)
    e.close()
    assert fake.log == [(close, 2), ("eii_close", 1)]
    assert not d.h
    d.close()
    del d
    gc.collect()
    e.close()
    assert fake.log == [(close, 2), ("eii_close", 1)]


@pytest.mark.parametrize("close", OPEN)
def test_object_in_a_cycle_outlives_the_engine(fake, close):
    """An object kept alive by a reference cycle (an exception's traceback holds its frame) is collected after the
    engine has been closed, when a later allocation runs the collector."""
    import _eii
    e = _eii.Engine("model", 0)

    def failing():
        d = OPEN[close](_eii, e)
        try:
            raise ValueError(d)
        except ValueError as error:
            kept = error  # error -> traceback -> this frame -> kept -> error
        return kept is not None
    gc.disable()
    try:
        assert failing()
        e.close()
        gc.collect()
    finally:
        gc.enable()
    assert fake.log == [(close, 2), ("eii_close", 1)]


@pytest.mark.parametrize("close", OPEN)
def test_engine_and_object_collected_at_once(fake, close):
    """Both in one cycle: the collector runs their finalisers in an order of its own."""
    import _eii
    for first in (0, 1):
        fake.log.clear()
        e = _eii.Engine("model", 0)
        d = OPEN[close](_eii, e)
        e.peer = d
        both = [e, d] if first else [d, e]
        both.append(both)
        handles = [d.h.value, e.h.value]
        del e, d, both
        gc.collect()
        assert [h for _, h in fake.log] == handles and fake.log[0][0] == close


def test_closed_in_order(fake):
    """The object first, as include/eii.h asks a C caller: the engine has nothing left to close."""
    import _eii
    e = _eii.Engine("model", 0)
    d = [OPEN[k](_eii, e) for k in OPEN]
    d[1].close()
    assert fake.log == [("eii_paged_decoder_close", 3)] and not d[1].h
    d[0].close()
    d[0].close()
    e.close()
    assert [h for _, h in fake.log] == [3, 2, 4, 1]


def test_failed_open_leaves_nothing_to_close(fake, monkeypatch):
    import _eii
    e = _eii.Engine("model", 0)
    monkeypatch.setattr(FakeLibrary, "eii_decoder_open", lambda *a: _eii.EII_ERR_ARG, raising=False)
    monkeypatch.setattr(FakeLibrary, "eii_last_error", lambda *a: b"refused", raising=False)
    with pytest.raises(_eii.EiiError, match="refused"):
        _eii.Decoder(e, 1, 8)
    gc.collect()
    e.close()
    assert fake.log == [("eii_close", 1)]
