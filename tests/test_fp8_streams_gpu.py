"""Products of e4m3 matrices cut along k, on several streams at once, at sizes of which shared memory lets more blocks onto an SM than tensor
memory does: the blocks of a cluster then wait for tensor memory while others of it are done (see test_tensor_memory_order for why that ends)."""
from __future__ import annotations

import pytest
import torch

from tests.test_fp8_gpu import _operands, _product_within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("early", [False, True])
@pytest.mark.parametrize("T,K,N", [(64, 1024, 4096), (64, 1040, 2500), (40, 1536, 4700), (24, 1408, 4736), (64, 1280, 2400)])
def test_products_in_four_parts_on_four_streams(T, K, N, early):
    from quanta_b200 import kernels
    rounds, kinds = 24, 4
    ops = [_operands(T, K, N, seed) for seed in range(kinds)]
    want = [torch.empty(T, N, device=DEV) for _ in ops]
    status = kernels.new_status(DEV)
    for o, w in zip(ops, want):
        kernels.linear_fp8(*o, w, status)
        _product_within(w, *o)
    streams = [torch.cuda.Stream() for _ in ops]
    outs = [[torch.full((T, N), float("nan"), device=DEV) for _ in range(rounds)] for _ in ops]
    torch.cuda.synchronize()
    for i in range(rounds):
        for stream, o, out in zip(streams, ops, outs):
            with torch.cuda.stream(stream):
                kernels.linear_fp8(*o, out[i], status, early=early)
    torch.cuda.synchronize()
    assert int(status[0]) == 0
    assert all(torch.equal(got, w) for out, w in zip(outs, want) for got in out)

