"""Lengths beyond what a table row has places for, up to the largest 32-bit value: every call takes the row as full."""
import pytest
import torch

from paged_util import ints, offsets
from test_gpu_paged_decode import decode, filled, queries
from test_gpu_paged_prefill import prefill

pytestmark = pytest.mark.gpu

BEYOND = [0, 1, 15, 4000, 2 ** 30, 2 ** 31 - 1 - 6 * 16 - 15, 2 ** 31 - 1 - 6 * 16]      # added to the row's 96 places: up to 2^31 - 1


def cache(rows=3):
    """Rows of six places; row 0 has a page in each, row 1 in the first three, row 2 in the first."""
    c = filled([90, 40, 10], heads=2, dim=64, ps=16, seed=1, stale_nan=False)
    from runtherder_b200.kv_cache import PagedKVCache
    slabs = {n: getattr(c, n) for n in PagedKVCache.SLABS}
    slabs["page_table"] = c.page_table[:, :6].contiguous()
    c = PagedKVCache.from_tensors(**slabs)
    assert c.page_table.ge(0).sum(1).tolist() == [6, 3, 1]
    for r in range(3):
        for p in c.page_table[r].tolist():
            if p >= 0:
                c.ref_counts[p] = 1
    return c


@pytest.mark.parametrize("beyond", BEYOND)
def test_page_operations(beyond):
    c = cache()
    c.lens.copy_(ints([96 + beyond, 40, 10]))
    cu = offsets([20, 0, 4])
    table, refs, k_before = c.page_table.clone(), c.ref_counts.clone(), c.k.clone()
    c.reserve(cu, 3)
    assert torch.equal(c.page_table, table) and torch.equal(c.ref_counts, refs)
    assert c.status.tolist() == [-(-(96 + beyond + 20) // 16) - 6, 0]
    k = queries(24, 2, 64, 5)
    c.append(0, k, k, cu, 24, 3)
    changed = (c.k != k_before).any(-1).any(-2).nonzero().tolist()
    assert all(p == int(table[2, 0]) for _, p, *_ in changed)
    c.advance(cu, 3)
    assert c.lens.tolist() == [96 + beyond, 40, 14]
    c.fork(ints([0]), ints([1]), 1)                            # the child holds the places that there are
    assert c.page_table[1].tolist() == table[0].tolist()
    assert c.lens.tolist() == [96 + beyond, 96, 14]
    assert all(c.ref_counts[p] == 2 for p in table[0].tolist())


@pytest.mark.parametrize("beyond", BEYOND)
@pytest.mark.parametrize("splits", [1, 2])
def test_attention(beyond, splits):
    """The same bits as for a length that is just the row's places."""
    c = cache()
    q, cu = queries(90, 8, 64, 6), offsets([70, 15, 5])
    c.lens.copy_(ints([96, 25, 5]))
    want, one = prefill(c, q, cu, 8, 0.1, splits), decode(c, q[:3], 8, 0.1)
    c.lens.copy_(ints([96 + beyond, 25, 5]))
    assert torch.equal(prefill(c, q, cu, 8, 0.1, splits), want)
    assert torch.equal(decode(c, q[:3], 8, 0.1), one)
