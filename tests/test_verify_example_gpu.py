"""The example that runs the verification operators together, at a small size.

Tolerances.  K rows: the plain run's rows differ from the cache's by the cache's
step (int8: half of 1/127 of the row's maximum; e4m3: 2^-4 of an element at
most; fp16: its rounding) and by what fp16 roundings of two layers' hidden
states add, a few 2^-10 of the maximum: 2^-7 is allowed for those.  Logits: unit
variance by construction; the hidden state's fp16 roundings (about 10 of 2^-11,
of elements a few units in size) reach a logit as a sum of 512 random signs, so
some 0.01; 0.06 is allowed.
"""

import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache,step", [("int8", 0.5 / 127), ("float8_e4m3fn", 2.0**-4), ("float16", 2.0**-11)])
def test_drafts_are_verified_as_plain_decoding_would(cache, step):
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import verify_drafts

    taken, shortfall, row = verify_drafts.main(cache, new_tokens=24)
    assert taken > 1.5
    assert shortfall <= 0.06
    assert row <= step + 2.0**-7
