"""The example that runs prompt attention, the 4-bit cache and its decode
together: against the same steps over 16-bit pages the outputs differ by no more
than 4-bit rounding explains.

Bound: a group's values are off by at most half a step, 1/30 of its range; for
normal rows a range is about 5 sigma, so the rounding has rms 5 / 15 / sqrt(12) =
0.1 sigma in keys and values.  Values: 0.1 of the output, whose own size shrinks
with averaging in the same way.  Keys: scores of unit variance are off by 0.1 rms,
weights by 10%, again 0.1 of the output.  Together 0.14; asserted below 0.25.
"""

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "prompt_then_int4_decode.py")


def test_prompt_append_decode_and_second_chunk():
    spec = importlib.util.spec_from_file_location("prompt_then_int4_decode", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    decode, chunk, (small, large) = example.run()
    for a, b in (decode, chunk):
        assert a.shape == b.shape and a.isfinite().all()
        assert (a.float() - b.float()).norm() <= 0.25 * b.float().norm()
    assert small * 512 == large * 144          # bytes per token and head at 128 dims
