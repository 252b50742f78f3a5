"""CPU tests of the scales of 8-bit codes: how many columns each stands for goes with them."""
import numpy as np
import pytest

import charmnumeric_b200 as cnp
from tests.helpers import run_oracle

# groups of 30 of 100 columns make as many scales as groups of 25
X = np.random.default_rng(7).standard_normal((5, 100)).astype("float32")


def values(change, codes=lambda q: q):
    got = run_oracle(lambda: (lambda q, s: {"q": q, "s": s, "v": cnp.dequantize(codes(q), change(s), dtype="float32")})(
        *cnp.rms_norm(cnp.asarray(X), bits=8, group=30)))
    return got["v"], got["q"] * np.repeat(got["s"], 30, -1)[:, :100]


def assigned(s):
    out = cnp.zeros(s.shape, dtype="float32")
    out[...] = s
    return out


@pytest.mark.parametrize("change", [lambda s: s, lambda s: s.copy(), lambda s: s[:], lambda s: cnp.array(s), assigned,
                                    lambda s: s.astype("float64"), lambda s: cnp.abs(s)])
def test_scales_keep_their_group(change):
    v, want = values(change)
    np.testing.assert_array_equal(v, want)


def test_rows_and_multiples_of_scales():
    v, want = values(lambda s: s[1:3], lambda q: q[1:3])
    np.testing.assert_array_equal(v, want[1:3])
    v, want = values(lambda s: s * 2.0)
    np.testing.assert_array_equal(v, 2 * want)
    v, want = values(lambda s: s + s.copy())
    np.testing.assert_array_equal(v, 2 * want)


@pytest.mark.parametrize("change", ["host", "number", "part", "sum"])
def test_scales_that_were_assigned_to_ask_for_the_group(change):
    q, s = cnp.rms_norm(cnp.asarray(X), bits=8, group=30)
    _, other = cnp.rms_norm(cnp.asarray(X), bits=8, group=25)
    if change == "host":
        s[...] = np.ones((5, 4), "float32")
    elif change == "number":
        s[...] = 1
    elif change == "part":
        s[1:2] = other[1:2]
    else:
        s = s + other
    with pytest.raises(ValueError):
        cnp.dequantize(q, s)
    cnp.dequantize(q, s, group=25)


def test_scales_put_together_from_rows():
    def parts(s):
        out = cnp.zeros(s.shape, dtype="float32")
        out[:2] = s[:2]
        out[2:] = s[2:]
        return out
    v, want = values(parts)
    np.testing.assert_array_equal(v, want)
    v, want = values(lambda s: (s.__setitem__(slice(0, 1), np.zeros((1, 4), "float32")), s)[1])
    np.testing.assert_array_equal(v, want)
    assert (v[0] == 0).all()


def test_scales_assigned_over_others():
    def over(s):
        _, other = cnp.rms_norm(cnp.asarray(X), bits=8, group=25)
        other[...] = s
        return other
    v, want = values(over)
    np.testing.assert_array_equal(v, want)


def test_scales_from_elsewhere_divide_evenly():
    q, s = np.arange(-8, 8, dtype="int8").reshape(2, 8), np.array([[1, 2], [3, 4]], "float32")
    got = run_oracle(lambda: {"v": cnp.dequantize(cnp.asarray(q), cnp.asarray(s))})
    np.testing.assert_array_equal(got["v"], q * np.repeat(s, 4, -1))
    with pytest.raises(ValueError):
        cnp.dequantize(np.zeros((2, 7), "int8"), s)
