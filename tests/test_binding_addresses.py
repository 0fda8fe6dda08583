"""What the binding takes for an address, and that plain numbers, which callers with arenas of their own pass for every
argument, take no detour through an exception."""
import ctypes
import sys

import numpy as np
import pytest

from decisive_amd import rocm


class Number(int):
    pass


def raised(x):
    """The exceptions that pass through the lookup of x's address."""
    seen = []

    def trace(frame, event, arg):
        if event == "exception":
            seen.append(arg[0])
        return trace

    before = sys.gettrace()
    sys.settrace(trace)
    try:
        rocm._addr(x)
    finally:
        sys.settrace(before)
    return seen


@pytest.mark.parametrize("x", [None, 0, 1 << 47, (1 << 64) - 1])
def test_numbers_are_their_own_address(x):
    assert rocm._addr(x) == x
    assert raised(x) == []


def test_tensors_arrays_and_other_numbers():
    import torch
    t, a = torch.zeros(5), np.zeros(5)
    assert rocm._addr(t[2:]) == t.data_ptr() + 8
    assert raised(t) == []
    assert rocm._addr(a[1:]) == a.ctypes.data + 8
    assert rocm._addr(Number(77)) == 77 and rocm._addr(True) == 1


@pytest.mark.parametrize("x", [1.5, "address", [1], ctypes.c_float(1)])
def test_what_has_no_address_is_refused(x):
    with pytest.raises(TypeError):
        rocm._addr(x)
