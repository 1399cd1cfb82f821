"""Status words: what a kernel records takes three of them, so fewer are refused before anything is launched."""
from __future__ import annotations

import pytest
import torch

from quanta_b200 import kernels

E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("words", [0, 1, 2])
def test_too_few_status_words(words):
    status = torch.zeros(8, dtype=torch.int32)[3: 3 + words]
    x, w = torch.zeros(5, 256).to(E4M3), torch.zeros(300, 256).to(E4M3)
    with pytest.raises(ValueError, match="status"):
        kernels.linear_fp8(x, torch.zeros(2, 5), w, torch.zeros(3, 2), torch.zeros(5, 300), status)
    with pytest.raises(ValueError, match="status"):
        kernels.token_logprobs(torch.zeros(4, 100), torch.zeros(4, dtype=torch.int32), torch.zeros(4), None, status=status)
