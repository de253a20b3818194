"""CPU checks of the host side around the window attention and 8-bit cache
calls: helpers of the package, split counts, the build of the binding."""
import math

from grout_b200 import attn


def test_default_scale():
    """The softmax scale that the attention calls use where none is given."""
    assert attn.default_scale() == 1.0 / math.sqrt(128)
    assert attn.default_scale(64) == 0.125
