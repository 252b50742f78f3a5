"""What recording costs: arithmetic on arrays of the arithmetic types pays nothing for storage types and scales."""
import sys

import charmnumeric_b200 as cnp
from charmnumeric_b200 import frontend as F


def calls(fn):
    """Calls of the front end's functions (comprehensions aside) that `fn` makes."""
    n = 0

    def count(frame, event, _):
        nonlocal n
        code = frame.f_code
        n += event == "call" and code.co_filename == F.__file__ and not code.co_name.startswith("<")
    sys.setprofile(count)
    try:
        fn()
    finally:
        sys.setprofile(None)
    return n


def test_a_stencil_sweep_records_in_as_few_calls_as_without_storage_types():
    u = cnp.zeros((64, 64))

    def sweep():
        u[1:-1, 1:-1] = 0.25 * (u[:-2, 1:-1] + u[2:, 1:-1] + u[1:-1, :-2] + u[1:-1, 2:])
    sweep()
    assert calls(sweep) <= 104
