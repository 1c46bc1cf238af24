"""The bindings of the paged cache and the verification, on the host."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

NAMES = ["sq_paged_append", "sq_paged_attention", "sq_paged_read", "sq_verify_drafts", "sq_paged_status"]


@pytest.mark.parametrize("name", NAMES)
def test_calls_give_up_the_interpreter_lock(name):
    """They can wait for the GPU; other threads go on meanwhile."""
    from sqb200 import paged
    assert not paged._fn(name)._flags_ & C._FUNCFLAG_PYTHONAPI
