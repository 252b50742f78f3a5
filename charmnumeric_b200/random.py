"""Seeded random arrays.  The reference's ``random.randn`` returns a zero array
(charmnumeric/random.py:4-5); ``uniform`` here is generated on the device from a
counter-based generator so the values do not depend on the number of GPUs; ``sample`` draws tokens
from such numbers."""
from .frontend import uniform, zeros  # noqa: F401
from .sequence import sample  # noqa: F401


def randn(*shape, dtype="float64"):
    """As in the reference: a zero array of the given shape."""
    return zeros(shape, dtype=dtype)
