"""Lengths at and behind the end of a table row, all of whose pages hold numbers: what is attended ends with the row."""
import math

import pytest
import torch

from paged_util import check_attention, ints, offsets, row_contents
from test_gpu_paged_decode import BLOCKS, decode, filled, queries
from test_gpu_paged_prefill import HOLD, prefill

pytestmark = pytest.mark.gpu


def full(rows, per, ps, heads, dim, seed):
    """Rows whose every place has a page of numbers of its own."""
    c = filled([per * ps - 1] * rows, heads=heads, dim=dim, ps=ps, seed=seed, stale_nan=False)
    from runtherder_b200.kv_cache import PagedKVCache
    return PagedKVCache.from_tensors(**{**{n: getattr(c, n) for n in PagedKVCache.SLABS}, "page_table": c.page_table[:, :per].contiguous()})


@pytest.mark.parametrize("dim,ps,hq,hkv", [(128, 16, 12, 4), (64, 64, 8, 1)])
@pytest.mark.parametrize("batch", [2, 30])
def test_decode_ends_with_the_table_row(batch, dim, ps, hq, hkv):
    per, scale = 512 // ps + 1, 1.0 / math.sqrt(dim)
    c = full(batch, per, ps, hkv, dim, seed=batch)
    room = per * ps
    lens = [[room - 2, room - 1, room, room + 1, room + 1000, 2 ** 30 - 1, 2 ** 31 - 1][i % 7] for i in range(batch)]
    c.lens.copy_(ints(lens))
    c.page_table[:, : 512 // ps] = c.page_table[0, : 512 // ps].clone()      # the first 512 keys are everybody's
    q = queries(batch, hq, dim, ps)
    for shared in (0, 512, room + 256, 2 ** 31 - 1):
        shared_keys = min(shared, room) // 256 * 256
        assert shared_keys <= 512
        out = decode(c, q, hq, scale, (c.page_table[0].clone(), ints([shared])) if shared else None)
        for i in range(batch):
            n = min(lens[i] + 1, room)
            k, v = row_contents(c, 0, i, n)
            assert bool(torch.isfinite(k).all()) and bool(torch.isfinite(v).all())
            check_attention(out[i: i + 1], q[i: i + 1], k, v, n, scale, (i, shared), **BLOCKS)


@pytest.mark.parametrize("dim,ps,hq,hkv", [(128, 16, 12, 4), (64, 64, 8, 1)])
@pytest.mark.parametrize("splits", [1, 3])
def test_prefill_ends_with_the_table_row(splits, dim, ps, hq, hkv):
    per, scale, new = 384 // ps, 0.11, [40, 3, 70, 1]
    c = full(4, per, ps, hkv, dim, seed=splits)
    room = per * ps
    held = [room - 40, room - 1, room - 30, room + 500]         # the last places; beyond them tokens see what the row holds
    c.lens.copy_(ints(held))
    q = queries(sum(new), hq, dim, 3)
    out = prefill(c, q, offsets(new), hq, scale, splits)
    at = 0
    for i, (n, h) in enumerate(zip(new, held)):
        k, v = row_contents(c, 0, i, room)
        assert bool(torch.isfinite(k).all()) and bool(torch.isfinite(v).all())
        for t in range(n):
            seen = min(h + t + 1, room)
            check_attention(out[at + t: at + t + 1], q[at + t: at + t + 1], k[:, :seen], v[:, :seen], seen, scale, (i, t), **HOLD)
        at += n
