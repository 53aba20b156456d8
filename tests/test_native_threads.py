"""First calls of an entry point from several threads at once, on the CPU: each gets all of the
library's functions, and so does every later call."""

from __future__ import annotations

import threading
import time

import pytest

from linattn_amd import _native as N


@pytest.mark.parametrize("cls,names", [
    (N.LaRotaryArgs, ("la_rotary",)),
    (N.LaPagedAttnArgs, ("la_paged_attention_workspace", "la_paged_attention")),
])
def test_first_calls_meet(monkeypatch, cls, names):
    lib = N.load()

    def slow():  # (as the opening of a library: other threads run meanwhile)
        time.sleep(0.05)
        return lib

    monkeypatch.setattr(N, "load", slow)
    _, functions = N.by_bytes(cls, *names)
    start, got = threading.Barrier(4), [None] * 4

    def call(i):
        start.wait()
        time.sleep(0.02 * i)  # (some while another has begun)
        got[i] = list(functions())

    threads = [threading.Thread(target=call, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for fns in (*got, functions()):
        assert [fn.__name__ for fn in fns] == list(names)
        for fn in fns:
            plain = getattr(lib, fn.__name__)
            assert fn.restype is plain.restype and len(fn.argtypes) == len(plain.argtypes)
