"""Entries that see no key are zero whatever their q holds: a fixed-size batch's padding is seldom initialised."""
import math

import pytest
import torch

from paged_util import check_attention, ints, offsets, row_contents
from test_gpu_paged_decode import BLOCKS, decode, filled, queries
from test_gpu_paged_prefill import prefill

pytestmark = pytest.mark.gpu

BAD = [float("nan"), float("inf"), float("-inf")]


def spoil(q, i):
    """Row i in full, then single values of it."""
    q[i] = BAD[i % 3]
    q[i, 1:] = 0.5
    q[i, 1, 3] = BAD[(i + 1) % 3]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("shared", [0, 256, 1024])
@pytest.mark.parametrize("batch", [3, 5, 40, 130])            # 6, 10 query rows per kv head: mma.sync; 80, 260: tcgen05, one and two row blocks
def test_decode(batch, shared, dim):
    hq, hkv, ps = 4, 2, 16
    idle, unknown = [1], [2]
    lens = [shared + (7 * i) % 50 for i in range(batch)]
    for i in idle:
        lens[i] = -1
    c = filled(lens, shared=shared, heads=hkv, dim=dim, ps=ps, seed=batch)
    rows = list(range(batch))
    for i, r in zip(unknown, (batch + 9,)):
        rows[i] = r
    q = queries(batch, hq, dim, shared)
    for i in idle + unknown:
        spoil(q, i)
    scale = 1.0 / math.sqrt(dim)
    table = (c.page_table[0].clone(), ints([shared])) if shared else None
    hold = BLOCKS if batch * hq // hkv >= 17 else {}

    def holds(q, bad_head=None):
        """Every entry is what its own q gives, whatever the others' are; NaN where the entry itself is active and holds one."""
        out = decode(c, q, hq, scale, table, rows=rows)
        for i in range(batch):
            if i in idle + unknown:
                assert not out[i].any(), (i, out[i].isnan().sum().item())
                continue
            k, v = row_contents(c, 0, i, lens[i] + 1)
            own, mine = out[i: i + 1], q[i: i + 1]
            if i == 0 and bad_head is not None:
                assert own[0, bad_head].isnan().all()
                own, mine = own.clone(), mine.clone()
                own[0, bad_head], mine[0, bad_head] = own[0, bad_head ^ 1], mine[0, bad_head ^ 1]
            check_attention(own, mine, k, v, lens[i] + 1, scale, i, **hold)

    holds(q)
    q[0, 2, 5] = float("nan")
    holds(q, 2)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("splits", [1, 3])
def test_prefill(splits, dim):
    """Idle and unknown rows, and a row none of whose pages exist."""
    hq, hkv, ps = 4, 2, 16
    c = filled([40, -1, 99, 500], heads=hkv, dim=dim, ps=ps, seed=1)
    c.lens.copy_(ints([30, -1, 80, 450]))
    c.page_table[2] = -1
    new, rows = [11, 4, 20, 51, 3], [0, 1, 2, 3, 77]
    q = queries(sum(new), hq, dim, 2)
    at = [sum(new[:i]) for i in range(5)]
    for i in (1, 2, 4):
        for t in range(new[i]):
            spoil(q, at[i] + t)
    hold = dict(extra=2.0 * 2.0 ** -11, small_step=2.0 ** -25, q_step=2.0 ** -16)
    spot = at[3] + 7

    def holds(q, bad_head=None):
        out = prefill(c, q, offsets(new), hq, 0.1, splits, rows=rows)
        q = q.clone()
        if bad_head is not None:
            assert out[spot, bad_head].isnan().all()
            out[spot, bad_head], q[spot, bad_head] = out[spot, bad_head ^ 1], q[spot, bad_head ^ 1]
        for i, r in enumerate(rows):
            part = slice(at[i], at[i] + new[i])
            if i in (1, 2, 4):
                assert not out[part].any(), i
            else:
                held = int(c.lens[r])
                k, v = row_contents(c, 0, r, held + new[i])
                check_attention(out[part], q[part], k, v, held + 1, 0.1, i, **hold)

    holds(q)
    for bad in BAD:
        again = q.clone()
        again[spot, 2, 9] = bad
        holds(again, 2)
