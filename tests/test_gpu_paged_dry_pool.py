"""A pool that runs dry in the middle of a step and recovers.  Every row's tokens are kept in a plain list beside the cache:
a token counts for its row exactly when the cache had a page for it, and what the row holds afterwards has to be that list."""
import math

import pytest
import torch

from paged_util import check_attention, ints, offsets, row_contents
from test_gpu_paged_cache import reference_append

pytestmark = pytest.mark.gpu

HEADS, DIM, PS = 2, 64, 16


class Session:
    """A cache, and the tokens that each row was given and had a page for."""

    def __init__(self, pages, rows, per):
        from runtherder_b200.kv_cache import PagedKVCache
        self.c = PagedKVCache(1, pages, PS, HEADS, DIM, rows, per)
        self.c.k.fill_(0x7f)                           # places that no token was stored to must never be read
        self.c.v.fill_(0xff)
        self.kept = [[] for _ in range(rows)]
        self.gen = torch.Generator(device="cuda").manual_seed(pages)
        self.c.start(rows)

    def step(self, rows, new, stored):
        """reserve, append, advance as documented; `stored` of each row's new tokens have a page."""
        k = torch.randn(sum(new), HEADS, DIM, device="cuda", generator=self.gen).to(torch.bfloat16)
        cu, on, n = offsets(new), ints(rows), len(rows)
        self.c.reserve(cu, n, on)
        self.c.append(0, k, k, cu, sum(new), n, on)
        self.c.advance(cu, n, on)
        at = 0
        for r, count, kept in zip(rows, new, stored):
            self.kept[r] += list(k[at: at + kept])
            at += count
        self.holds()

    def release(self, row, new_len=-1):
        self.c.release(1, ints([row])) if new_len else self.c.start(1, ints([row]))
        self.kept[row] = []

    def holds(self):
        """lens and contents are the kept tokens, and the next token attends exactly them (and itself, where it was stored)."""
        lens = self.c.lens.tolist()
        for r, kept in enumerate(self.kept):
            if lens[r] < 0:
                assert not kept
                continue
            assert lens[r] == len(kept), (r, lens[r], len(kept))
            if kept:
                codes, scales = reference_append(torch.stack(kept), HEADS, DIM)
                want = codes.view(torch.float8_e4m3fn).double() * scales.double().unsqueeze(-1)
                for got in row_contents(self.c, 0, r, len(kept)):
                    assert torch.equal(got, want.permute(1, 0, 2)), r


def test_a_row_gets_the_page_it_missed_once_one_is_free():
    s = Session(pages=3, rows=2, per=4)
    s.step([0, 1], [16, 32], [16, 32])
    assert s.c.status.tolist() == [0, 0]
    for missed in (1, 2, 3):                            # the pool is dry: each step says so, and the row stays where it is
        s.step([0], [1], [0])
        assert s.c.status.tolist() == [missed, 0]
    s.release(1)
    for _ in range(20):                                 # the row goes on where it stopped, over the next page's border too
        s.step([0], [1], [1])
    assert s.c.status.tolist() == [3, 0] and len(s.kept[0]) == 36
    from runtherder_b200 import kernels as K
    q = torch.randn(1, 4, DIM, device="cuda", generator=s.gen).to(torch.bfloat16)
    s.c.lens[0] = 35                                    # the last token that was stored attends all 36
    out = torch.empty(1, 4, DIM, dtype=torch.bfloat16, device="cuda")
    part = torch.empty(K.flash_decode_paged_scratch_floats(1, 4, HEADS, DIM), device="cuda")
    K.flash_decode_paged_bf16(out, q, s.c, 0, 1, 4, 1.0 / math.sqrt(DIM), part)
    k, v = row_contents(s.c, 0, 0, 36)
    check_attention(out, q, k, v, 36, 1.0 / math.sqrt(DIM))


def test_a_step_that_fits_in_part():
    """Tokens up to the first place without a page are kept, the others are given again by the caller."""
    s = Session(pages=4, rows=3, per=8)
    s.step([0, 1], [14, 16], [14, 16])                  # three pages are left ... of which row 2 takes one
    s.step([2], [3], [3])
    s.step([0, 1], [40, 5], [18, 0])                    # row 0: two places of its page, the last free page, then nothing
    assert s.c.status.tolist() == [2 + 1, 0] and s.c.lens.tolist() == [32, 16, 3]
    s.release(2)
    s.step([1, 0], [5, 1], [5, 0])                      # the page goes to the first of the batch
    assert s.c.lens.tolist() == [32, 21, -1]
    s.release(1)
    s.step([0], [32], [32])
    assert s.c.lens.tolist() == [64, -1, -1] and s.c.status.tolist() == [2 + 1 + 1, 0]


def test_a_row_that_outgrows_its_table_stays_full():
    s = Session(pages=9, rows=1, per=2)
    s.step([0], [30], [30])
    s.step([0], [1000], [2])
    s.step([0], [1], [0])
    assert s.c.lens.tolist() == [32]
    assert s.c.status[0].item() == (-(-1030 // PS) - 2) + 1
    s.release(0, 0)
    s.step([0], [17], [17])


def test_many_rows_and_long_entries():
    """More columns than a warp has lanes, and more rows than a CTA's warps: every row stops at its own first missing place."""
    rows, per = 40, 70
    s = Session(pages=rows * 40, rows=rows, per=per)
    s.step(list(range(rows)), [1 + 7 * r for r in range(rows)], [1 + 7 * r for r in range(rows)])
    new, stored = [], []
    free = rows * 40 - sum(-(-(1 + 7 * r) // PS) for r in range(rows))
    for r in range(rows):                               # pages are handed out in the order of the batch
        held, more = 1 + 7 * r, (1000 if r % 3 else 600) - 7 * r
        lack = -(-(held + more) // PS) - -(-held // PS)
        got = min(lack, free)
        free -= got
        new.append(more)
        stored.append(min(more, (-(-held // PS) + got) * PS - held))
    assert free == 0 and any(0 < a < b for a, b in zip(stored, new))
    s.step(list(range(rows)), new, stored)


def test_a_place_that_reserve_does_not_fill_is_counted():
    """A row whose partly filled page was taken out of its table, or whose table names a page outside the pool: such a place is not
    filled (what lay there is gone, or never was), the row stays, and every reserve says so."""
    s = Session(pages=8, rows=3, per=4)
    s.step([0, 1, 2], [20, 16, 5], [20, 16, 5])
    s.c.page_table[0, 1] = -1
    s.c.page_table[1, 1] = 8
    cu = offsets([1, 1, 1])
    for n in (1, 2):
        s.c.reserve(cu, 3)
        s.c.append(0, *[torch.ones(3, HEADS, DIM, device="cuda", dtype=torch.bfloat16)] * 2, cu, 3, 3)
        s.c.advance(cu, 3)
        assert s.c.lens.tolist() == [20, 16, 5 + n] and s.c.status.tolist() == [2 * n, 0]
