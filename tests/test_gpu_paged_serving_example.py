"""The paged-serving example end to end: prompts, chunks beside decoding, and
captured decode steps give what one call over the whole text gives, up to the
cache's quantisation."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu
pytest.importorskip("torch")
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


# bf16 pages hold what the whole-text call reads (two roundings of the output
# apart); int8 rounds k and v to 1/254 of a row's largest value (about 3 times
# its rms: 0.7 % of the rms on average, 1.2 % with the shift of the weights),
# e4m3 to 2^-4 of each value at most (2.6 % rms)
@pytest.mark.parametrize("cache,bound", [("bf16", 0.008), ("int8", 0.03), ("fp8", 0.08)])
def test_paged_serving_example(cache, bound):
    import paged_serving

    assert paged_serving.main(steps=6, cache=cache, chunk=60) <= bound
