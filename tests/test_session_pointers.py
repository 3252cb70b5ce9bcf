"""Session.run_ptrs checks the pointer lists against the plan before the library is called (host only)."""
import ctypes

import pytest

from emx_onnx_cgen_b200.runtime import Session


def session(n_in, n_out):
    s = Session.__new__(Session)
    s.handle = None
    s._ins, s._outs = (ctypes.c_void_p * n_in)(), (ctypes.c_void_p * n_out)()
    s.calls = []
    s._run = lambda handle, ins, outs, *rest: s.calls.append((list(ins), list(outs))) or 0
    return s


def test_a_list_for_another_plan_is_refused():
    """One input too few or too many would put every later pointer on the wrong tensor."""
    s = session(3, 2)
    for ins, outs in (([1, 2], [7, 8]), ([1, 2, 3, 4], [7, 8]), ([], [7, 8]), ([1, 2, 3], [7])):
        with pytest.raises(ValueError, match="pointers"):
            s.run_ptrs(ins, outs)
    assert not s.calls
    s.run_ptrs([1, 2, 3], (7, 8))
    s.run_ptrs((4, 5, 6), [9, 10])
    assert s.calls == [([1, 2, 3], [7, 8]), ([4, 5, 6], [9, 10])]


def test_a_plan_without_inputs():
    s = session(0, 1)
    s.run_ptrs([], [5])
    with pytest.raises(ValueError, match="pointers"):
        s.run_ptrs([1], [5])
    assert s.calls == [([], [5])]
