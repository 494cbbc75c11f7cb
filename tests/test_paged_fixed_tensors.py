"""A cache's tensors are those whose addresses its calls hand to the kernels: they are written into, not replaced."""
import pytest
import torch

from runtherder_b200._lib import RhError
from runtherder_b200.kv_cache import PagedKVCache


@pytest.mark.parametrize("name", PagedKVCache.SLABS + ("scratch",))
def test_tensors_of_a_cache_are_not_replaced(name):
    c = PagedKVCache(1, 4, 16, 2, 64, 3, 2, device="cpu")
    before = getattr(c, name)
    with pytest.raises(RhError):
        setattr(c, name, torch.zeros_like(before))
    assert getattr(c, name) is before
    if name != "scratch":
        assert getattr(c._struct, name) == before.data_ptr()
    before.fill_(1)
    c.note = 1                     # other attributes are the caller's
