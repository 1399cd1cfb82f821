"""Norms into 8-bit rows of more than 8,192 numbers, which have a kernel of their own: selected rows, rows that are not there, no addend, several
slots, the widest rows, and the refusal of wider ones."""
from __future__ import annotations

import pytest
import torch

from quanta_b200 import kernels
from tests.test_fp8_gpu import DEV, _empty_rows, _gen, _randn, test_norm as _norm_within

E4M3 = torch.float8_e4m3fn


def test_wider_rows_are_refused():
    H = kernels.FP8_NORM_MAX_WIDTH + 1
    h, q, s = torch.zeros(2, H), torch.zeros(2, H).to(E4M3), torch.zeros(-(-H // 128), 2)
    with pytest.raises(ValueError, match=str(kernels.FP8_NORM_MAX_WIDTH)):
        kernels.add_rmsnorm_fp8(h, None, torch.ones(H), 1e-5, q, s)


@pytest.mark.gpu
@pytest.mark.parametrize("gain", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,H,S", [(3, 8200, 3), (2, 8193, 8), (5, 12345, 2), (2, 51200, 1), (1, 51199, 2)])
def test_slots_and_the_widest(n, H, S, dtype, gain):
    _norm_within(n, H, S, dtype, gain)


@pytest.mark.gpu
@pytest.mark.parametrize("H", [8193, 8200, 20000])
def test_selected_rows_and_no_addend(H):
    g = _gen(H)
    h, w = _randn(g, 6, H), 1 + 0.1 * _randn(g, H)
    d, dg = _randn(g, 6, H), _randn(g, H)
    rows = torch.tensor([5, 0, 0, 3], dtype=torch.int32, device=DEV)
    for gain in (None, dg):
        full, full_s = _empty_rows(6, H)
        h2 = h.clone()
        kernels.add_rmsnorm_fp8(h2, d, w, 1e-5, full, full_s, delta_gain=gain, delta_eps=1e-6)
        q, s = _empty_rows(4, H)
        before = h.clone()
        kernels.add_rmsnorm_fp8(h, d, w, 1e-5, q, s, rows=rows, store_h=False, delta_gain=gain, delta_eps=1e-6)
        assert torch.equal(h, before) and torch.equal(q.float(), full.float()[rows.long()]) and torch.equal(s, full_s[:, rows.long()])
        q2, s2 = _empty_rows(6, H)
        kernels.add_rmsnorm_fp8(h2, None, w, 1e-5, q2, s2)      # the sum is in h2
        assert torch.equal(q2.float(), full.float()) and torch.equal(s2, full_s)
        q3, s3 = _empty_rows(4, H)
        h3 = h.clone()
        kernels.add_rmsnorm_fp8(h3, d, w, 1e-5, q3, s3, rows=torch.tensor([-1, 2, 6, 1 << 30], dtype=torch.int32, device=DEV), store_h=False, delta_gain=gain,
                                delta_eps=1e-6)
        bad = [0, 2, 3]
        assert torch.equal(h3, h) and torch.all(torch.isnan(q3.float()[bad])) and torch.all(torch.isnan(s3[:, bad]))
        assert torch.equal(q3.float()[1], full.float()[2]) and torch.equal(s3[:, 1], full_s[:, 2])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", [12032, 12033, 12224, 12225, 12256, 12288, 12289])
def test_rows_that_fill_what_shared_memory_a_kernel_has_unasked(H, dtype):
    """48 KB, of which the kernel's own variables take some: a row that leaves no room for them has to ask for more."""
    _norm_within(3, H, 1, dtype, False)
