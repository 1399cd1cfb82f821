"""The numbers a scored text ends up with, and how the command writes them."""
from __future__ import annotations

import json
import math

import pytest

from quanta_b200.__main__ import _numbers
from quanta_b200.engine.score import TextScores


def test_perplexity():
    assert TextScores([-1.0, -3.0]).perplexity == pytest.approx(math.exp(2.0))
    assert math.isnan(TextScores().perplexity)
    assert TextScores([-1000.0, -900.0]).perplexity == math.inf      # a mean whose exponential is no float
    assert TextScores([-1.0, -math.inf]).perplexity == math.inf


def test_lines_are_json():
    line = {"tokens": 1, "perplexity": math.nan, "logprobs": [-math.inf, -0.5], "top_ids": [[3, 4]], "top_logprobs": [[math.inf, -1.0]]}
    assert json.loads(json.dumps(_numbers(line), allow_nan=False)) == {
        "tokens": 1, "perplexity": None, "logprobs": [None, -0.5], "top_ids": [[3, 4]], "top_logprobs": [[None, -1.0]]}
