"""Failures of the calls without a handle (relative position bias, norm) stay with the thread that made them, without a GPU."""
import ctypes
import threading

import pytest

from spion_amd import _lib
from spion_amd import norm as rn
from spion_amd import relative_bias as rb


@pytest.fixture(autouse=True)
def nothing_pending(monkeypatch):
    monkeypatch.setenv("SPION_QUIET", "1")
    _lib.core().spion_clear_error()
    yield
    _lib.core().spion_clear_error()


def _refused(name):
    """One call that is refused before any GPU work."""
    bias = name.startswith("spion_bias")
    lib = (rb if bias else rn)._lib_typed()
    call = rb._Call() if bias else rn._Call()
    if name.endswith("workspace"):
        return getattr(lib, name)(ctypes.addressof(call), *((0,) if bias else ())) == -1
    return getattr(lib, name)(ctypes.addressof(call), None) != 0


CALLS = ["spion_bias_workspace", "spion_bias_attention_forward", "spion_bias_attention_backward", "spion_rms_norm_workspace",
         "spion_rms_norm_forward", "spion_rms_norm_backward"]


def _elsewhere(work):
    found = []
    t = threading.Thread(target=lambda: found.append(work()))
    t.start()
    t.join()
    return found[0]


@pytest.mark.parametrize("name", CALLS)
def test_another_thread_neither_finds_nor_clears_a_failure(name):
    lib = _lib.core()
    assert _refused(name)
    assert _elsewhere(lambda: (lib.spion_error_pending(), lib.spion_last_error(), lib.spion_take_call_error())) == (0, b"", b"")
    _elsewhere(lib.spion_clear_error)
    assert lib.spion_error_pending() == 1 and lib.spion_last_error().startswith(name.encode())
    with pytest.raises(_lib.SpionLibraryError, match=name):
        _lib.check_call(False, "call")
    assert lib.spion_error_pending() == 0


@pytest.mark.parametrize("name", CALLS)
def test_a_failure_leaves_the_process_wide_slot_alone(name):
    lib = _lib.core()
    lib.spion_set_stream(None, None)  # of a handle that is none: any thread finds it
    assert _elsewhere(lib.spion_last_error).startswith(b"spion_set_stream")
    assert _refused(name) and lib.spion_last_error().startswith(name.encode())
    with pytest.raises(_lib.SpionLibraryError, match=name):
        _lib.check_call(False, "call")
    _lib.check_call(True, "call")  # a call that succeeded is not asked what else is pending
    assert lib.spion_last_error().startswith(b"spion_set_stream")
    assert _refused(name)
    lib.spion_set_stream(None, None)
    assert lib.spion_last_error().startswith(b"spion_set_stream")  # the later one
    lib.spion_clear_error()
    assert lib.spion_error_pending() == 0 and lib.spion_last_error() == b""


def test_threads_that_fail_and_clear_at_once():
    lib = _lib.core()
    stop = threading.Event()

    def clear():
        while not stop.is_set():
            lib.spion_clear_error()

    others = [threading.Thread(target=clear) for _ in range(2)]
    for t in others:
        t.start()
    try:
        for i in range(3000):
            name = CALLS[i % len(CALLS)]
            assert _refused(name) and lib.spion_take_call_error().startswith(name.encode()), i
    finally:
        stop.set()
        for t in others:
            t.join()


def test_a_failure_without_a_message_raises():
    with pytest.raises(_lib.SpionLibraryError, match="call failed"):
        _lib.check_call(False, "call")
