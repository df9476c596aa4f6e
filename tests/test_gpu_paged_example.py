"""examples/paged_decode.py: append, decode and evict together with the MoE
layer in a serving loop.  With all tokens kept the attention is dense attention
in bf16 (keys, values and output rounded to 8 bits: 3 x 2^-8 of the largest
value); with a budget no cache passes it."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "burn-extended_b200", "examples"))


def test_all_tokens_kept_is_dense_attention():
    import paged_decode
    far, sizes = paged_decode.serve(steps=24)
    assert far <= 3 * 2.0 ** -8, far
    assert sizes[-1] == [64, 31, 144, 25]


def test_a_budget_holds():
    import paged_decode
    _, sizes = paged_decode.serve(steps=40, budget=32)
    for step, now in enumerate(sizes):
        assert now == [min(32, n + step + 1) if n < 32 else 32 for n in (40, 7, 120, 1)]
