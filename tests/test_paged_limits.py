"""Cache descriptions at the edge of what 32-bit index arithmetic of the page operations holds.  Every call is refused before anything is
launched; nothing is dereferenced."""
import pytest
import torch

from runtherder_b200._lib import RhError
from runtherder_b200.kv_cache import PagedKVCache
from test_paged_refusals import A, DIM, INVALID, append, decode, pages, prefill, refused, slabs


@pytest.mark.parametrize("rows", [(1 << 24) + 1, 1 << 27, 1 << 28, 715827883, (1 << 30) - 1])
def test_more_rows_than_the_page_operations_can_number(rows):
    """advance numbers 32 threads per row (2^27 rows and more wrapped around), fork's scratch three ints (715827883 and more did)."""
    c = pages(num_rows=rows, pages_per_row=1)
    refused(DIM, *append(c))
    refused(DIM, "rh_kv_pages_reserve", c, None, A, 1, None)
    refused(DIM, "rh_kv_pages_release", c, None, 1, -1, None)
    refused(DIM, "rh_kv_pages_advance", c, None, A, rows, None)
    refused(DIM, "rh_kv_pages_fork", c, A, A, rows, None)
    refused(DIM, "rh_kv_pages_compact", c, None)
    refused(DIM, *decode(c))
    refused(DIM, *prefill(c))


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf"), 3e38])
def test_softmax_scales_that_are_no_numbers(scale):
    """The prefill would take a NaN for the smallest scale there is, and weigh all keys alike."""
    c = pages()
    refused(INVALID, "rh_flash_decode_paged_bf16", A, A, 512, c, 0, None, 2, 4, scale, A, None, None, None)
    refused(INVALID, "rh_flash_prefill_packed_bf16", A, A, 512, c, 0, None, A, 4, 2, 4, scale, A, 2, None)


def test_the_class_refuses_them_too():
    n = (1 << 24) + 1
    with pytest.raises(RhError):
        PagedKVCache.from_tensors(**slabs(page_table=torch.empty(n, 1, dtype=torch.int32), lens=torch.empty(n, dtype=torch.int32)))
