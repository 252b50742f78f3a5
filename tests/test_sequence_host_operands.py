"""CPU tests of host data given to the sequence model operators."""
import numpy as np
import pytest

import charmnumeric_b200 as cnp
from tests.helpers import run_oracle


def z(*shape, dtype="float32"):
    return cnp.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("call", [
    lambda: cnp.causal_conv(z(2, 3, 4), z(4, 2), lengths=[2 ** 32 + 1, 2]),
    lambda: cnp.causal_conv(z(2, 3, 4), z(4, 2), lengths=[1.5, 2.0]),
    lambda: cnp.selective_scan(z(2, 3, 4), z(2, 3, 4), z(4, 2), z(2, 3, 2), z(2, 3, 2), lengths=[float("nan"), 1.0]),
    lambda: cnp.random.sample(z(2, 4), z(2), top_k=[2 ** 31, 1]),
    lambda: cnp.random.sample(z(2, 4), z(2), top_k=np.array([0.5, 1.0])),
    lambda: cnp.dequantize([[300, 1]], np.ones((1, 1), "float32")),
])
def test_numbers_that_an_integer_operand_cannot_hold_are_refused(call):
    with pytest.raises(ValueError):
        call()


def test_whole_numbers_of_other_types_are_taken():
    x = np.arange(12.0).reshape(2, 3, 2)
    got = run_oracle(lambda: {k + str(i): v for i, n in enumerate(([1, 3], np.array([1, 3], np.uint8), [1.0, 3.0], (True, 3)))
                              for k, v in zip("ys", cnp.causal_conv(cnp.asarray(x), np.ones((2, 2)), lengths=n))})
    for i in range(1, 4):
        np.testing.assert_array_equal(got[f"y{i}"], got["y0"])
        np.testing.assert_array_equal(got[f"s{i}"], got["s0"])
