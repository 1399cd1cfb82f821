"""Rows that fill the 48 KB of shared memory that a kernel has unasked, but for what its own variables take: it has to ask for more."""
from __future__ import annotations

import pytest
import torch

from tests.test_gedelorn_mechanisms_gpu import test_norm_in_parts_and_gate as _norm_in_parts
from tests.test_tirizen_gpu import test_streams_between_two_sublayers_in_one_launch as _streams

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S,width,K", [(1, 11968, 1), (2, 11969, 1), (3, 12000, 2), (2, 12256, 1), (1, 12288, 1)])
def test_norm_over_several_streams(S, width, K):
    _streams(S, width, K)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,E,parts", [(2, 6128, 1), (4, 3071, 1), (3, 4086, 1), (24, 1023, 2), (2, 6144, 1), (3, 4097, 1)])
def test_norm_behind_a_recurrence(H, E, parts, dtype):
    _norm_in_parts(H, E, parts, dtype)
