"""A call of the attention block's operators that its C entry point refuses raises
that status's exception and is made once only: a second call could succeed after an
error that an earlier launch had left, and would run the work again. (No GPU here.)"""

import pytest

from breccia_b200 import _lib, kvcache


@pytest.fixture
def entry(monkeypatch):
    calls = []
    e = kvcache._Entry("brc_kv_write")
    statuses = []

    def fn(*args):
        calls.append(args)
        return statuses.pop(0)

    e.fn = fn
    monkeypatch.setattr(kvcache, "_current_device", lambda: 0)
    monkeypatch.setattr(kvcache, "_current_stream", lambda index: 7 + index)
    return e, calls, statuses


def test_ok(entry):
    e, calls, statuses = entry
    statuses += [_lib.BRC_OK]
    assert e(0, 1, 2) is None and calls == [(1, 2, 7)]


@pytest.mark.parametrize("status,error", [
    (_lib.BRC_ERR_SHAPE, ValueError), (_lib.BRC_ERR_RANGE, ValueError), (_lib.BRC_ERR_ALIGN, ValueError),
    (_lib.BRC_ERR_DTYPE, TypeError), (_lib.BRC_ERR_NULL, _lib.BrecciaB200Error),
    (_lib.BRC_ERR_UNSUPPORTED, _lib.BrecciaB200Error), (_lib.BRC_ERR_CUDA, _lib.BrecciaB200Error)])
def test_refusal(entry, status, error):
    e, calls, statuses = entry
    statuses += [status, _lib.BRC_OK]  # a second call would pass
    with pytest.raises(error, match="brc_kv_write"):
        e(0, 1, 2)
    assert calls == [(1, 2, 7)]
