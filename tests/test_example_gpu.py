"""The example of the token mixers between the projections runs, and decoding leaves what one pass over all tokens does.

Both ways compute the same values with other orders of fp32 sums (errors of 1e-6 and below); where such a difference
changes an int8 activation's code, a quantized row moves by one step of 127 in one of its 512 - 1024 inputs, of the order
1e-4 of the output.  2e-2 is far above a few of them and far below what a wrong token, position or state leaves (order 1)."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "startlux-prism_amd", "examples",
                    "hybrid_decode.py")


@pytest.mark.parametrize("lens,steps", [((37, 5, 70), 6), ((1,), 3), ((130, 64, 1, 16), 2)])
def test_decoding_agrees_with_one_pass(dev, lens, steps):
    spec = importlib.util.spec_from_file_location("hybrid_decode", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.main(lens, steps, dev) < 2e-2
