"""Offsets that name more tokens than the call has (a batch cut short): the tokens that the call has are computed, nothing else is
touched.  The entries are those of the offsets, cut at num_tokens."""
import math

import pytest
import torch

from paged_util import check_attention, offsets, row_contents
from test_gpu_paged_prefill import HOLD, batch, prefill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,held,total", [
    ([100, 300, 5000], [0, 0, 0], 400), ([20, 3000, 70, 9], [5, 100, 0, 3], 60), ([33] * 40, [7] * 40, 500), ([4000], [0], 1), ([64, 64], [0, 2000], 64),
])
@pytest.mark.parametrize("splits", [1, 4])
def test_prefill_of_a_batch_cut_short(new, held, total, splits):
    hq, hkv, dim, ps = 8, 2, 128, 32
    c, q, cu = batch(new, held, hq, hkv, dim, ps, seed=total)
    scale = 1.0 / math.sqrt(dim)
    out = prefill(c, q[:total], cu, hq, scale, splits, total=total)
    at = 0
    for i, (n, h) in enumerate(zip(new, held)):
        n_here = max(0, min(n, total - at))
        if n_here:
            k, v = row_contents(c, 0, i, h + n_here)
            check_attention(out[at: at + n_here], q[at: at + n_here], k, v, h + 1, scale, (i, n_here), **HOLD)
        at += n


def test_offsets_that_do_not_start_at_zero():
    """Tokens in front of the first entry are nobody's, as those behind the last are."""
    hq, hkv, dim = 8, 2, 64
    new, held = [50, 7], [3, 90]
    c, _, cu = batch(new, held, hq, hkv, dim, 16, seed=3)
    q = batch([70], [0], hq, hkv, dim, 16, seed=4)[1]
    cu = cu + 6
    for splits in (1, 3):
        out = prefill(c, q, cu, hq, 0.1, splits, total=70, num_seqs=2)
        assert (out[:6] == 7.0).all() and (out[63:] == 7.0).all()
        for i, at in ((0, 6), (1, 56)):
            k, v = row_contents(c, 0, i, held[i] + new[i])
            check_attention(out[at: at + new[i]], q[at: at + new[i]], k, v, held[i] + 1, 0.1, i, **HOLD)
