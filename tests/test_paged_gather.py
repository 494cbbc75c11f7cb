"""PagedKVCache.gather on host tensors: a row's keys in order, none of another row's, and its ends."""
import pytest
import torch

from paged_util import e4m3_table
from runtherder_b200._lib import RhError
from runtherder_b200.kv_cache import PagedKVCache


def cache():
    g = torch.Generator().manual_seed(2)
    c = PagedKVCache(2, 7, 16, 3, 64, 4, 3, device="cpu")
    for t in (c.k, c.v):
        t.copy_(torch.randint(0, 127, t.shape, dtype=torch.uint8, generator=g))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.rand(t.shape, generator=g))
    c.page_table.copy_(torch.tensor([[3, 6, 0], [1, -1, 5], [2, 9, -1], [-1, -1, -1]], dtype=torch.int32))
    return c


@pytest.mark.parametrize("layer", [0, 1])
@pytest.mark.parametrize("row", [0, 1, 2, 3])
@pytest.mark.parametrize("count", [0, 1, 16, 17, 40, 48])
def test_keys_in_order_and_nothing_of_other_rows(layer, row, count):
    c, values = cache(), e4m3_table().float()
    for got, codes, scale in zip(c.gather(layer, row, count), (c.k, c.v), (c.k_scale, c.v_scale)):
        assert got.shape == (3, count, 64) and got.dtype == torch.float32
        for j in range(count):
            page = int(c.page_table[row, j // 16])
            want = values[codes[layer, page, :, j % 16].long()] * scale[layer, page, :, j % 16, None] if 0 <= page < 7 else torch.zeros(3, 64)
            assert torch.equal(got[:, j], want), (j, page)


def test_refusals():
    c = cache()
    for bad in ((2, 0, 1), (-1, 0, 1), (0, 4, 1), (0, -1, 1), (0, 0, 49), (0, 0, -1)):
        with pytest.raises(RhError):
            c.gather(*bad)
