"""The attention block's calls together with the matmuls: a decoder layer whose answers share a prompt."""
from __future__ import annotations

import os
import sys

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import shared_prompt  # noqa: E402


@pytest.mark.parametrize("answers,prompt,steps", [(3, 70, 4), (1, 33, 2), (20, 300, 18)])
def test_shared_and_separate_prompts_agree(cuda, answers, prompt, steps):
    """Both runs append the same keys and values and differ in the order of the attention's fp32 sums, some
    1e-6 of a row. The projections behind it quantize their rows to 8 bits: a value next to a
    rounding boundary may fall on its other side, a step of 1 / 127 of a block's largest value on a
    few of a row's 1,536 or 8,960 terms: at most 1e-3 of a row, were one value in 60 to flip."""
    assert shared_prompt.run(answers, prompt, steps) < 1e-3
