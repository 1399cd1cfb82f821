"""Tensor memory and the barriers of a cluster.  The wait for tensor memory has no bound.  A block that holds some while it waits at its cluster's
barrier for a block that has none yet can therefore wait for good: that block may ask on an SM whose columns are held by blocks of its own cluster,
or by those of another, which wait for theirs in the same way.  So blocks that ask for tensor memory one by one give it back before they wait for the
others of their cluster; only the blocks of a pair, which get theirs together, hold it across their barriers."""
from __future__ import annotations

import re

import pytest

from quanta_b200.csrc import build
from tests.test_launch_order import _functions

BARRIER = re.compile(r"cluster_sync_all\(\)|barrier\.cluster")


def _kernels():
    for path in sorted(build.SRC_DIR.glob("*.cu")):
        for name, _, body in _functions(path.read_text()):
            if "tcgen05.alloc.cta_group::1" in body:
                yield pytest.param(body, id=f"{path.stem}-{name}")


@pytest.mark.parametrize("body", list(_kernels()))
def test_tensor_memory_is_given_back_before_the_clusters_barriers(body):
    body = re.sub(r"if \(PAIR\) cluster_sync_all\(\);", "", body)
    taken, given = body.index("tcgen05.alloc.cta_group::1"), body.index("tcgen05.dealloc.cta_group::1")
    assert taken < given and not BARRIER.search(body, taken, given)
    # nobody reads an accumulator that is gone
    assert "__syncthreads();" in body[taken: given] and "tcgen05.ld" not in body[given:] and "tmem_ld" not in body[given:]


def test_the_kernels_are_found():
    assert len(list(_kernels())) >= 4


def test_a_block_that_gave_up_gives_its_products_time():
    """Nobody waits for the accumulators of a block that gave up, so it lets the products on their way end before the columns are another's."""
    bodies = [b for n, _, b in _functions((build.SRC_DIR / "linear_fp8.cu").read_text()) if "tcgen05.dealloc" in b]
    assert len(bodies) == 2
    for body in bodies:
        given = body.index("tcgen05.dealloc")
        assert re.search(r"\*abort_flag\) l8_give_time\(\);", body[body.rindex("__syncthreads();", 0, given): given])
