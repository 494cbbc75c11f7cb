"""Keys whose weights are tiny beside one large one, and whose sum is not: they count in the numerator as they do in the
denominator.  The large key's V is zero, so what the others add is the whole output."""
import math

import pytest
import torch

from paged_util import check_attention, ints, offsets, row_contents
from test_gpu_paged_decode import decode
from test_gpu_paged_prefill import prefill

pytestmark = pytest.mark.gpu

# A weight enters the second product as f16, in units where the row's largest is 2^7 at least: half a step of its subnormals, 2^-25, is
# 2^-32 of the largest.  V is rounded twice (the scale, then the product), 2^-11 each; q in two E4M3 parts, 2^-16.
HOLD = dict(extra=2.0 * 2.0 ** -11, small_step=2.0 ** -32, q_step=2.0 ** -16)


def one_large_key(keys, dim, heads, where, below, rows=1, shared=0):
    """A cache whose rows hold `keys` keys: the one at `where` scores `below` (log2) more than all the others."""
    from runtherder_b200.kv_cache import PagedKVCache
    ps = 64
    per = -(-keys // ps)
    c = PagedKVCache(1, per, ps, heads, dim, rows, per)
    c.page_table.copy_(torch.arange(per, dtype=torch.int32, device="cuda").expand(rows, per))
    c.k.zero_()
    c.k_scale.fill_(1.0)
    one, half = 0x38, 0x30                             # E4M3 of 1 and of 0.5
    c.k[0, where // ps, :, where % ps] = one
    c.v.fill_(half)
    c.v[..., 1::2] = half | 0x80
    c.v[0, where // ps, :, where % ps] = 0
    c.v_scale.fill_(0.25)
    c.lens.fill_(keys - 1)
    q = torch.ones(rows, 4 * heads, dim, dtype=torch.bfloat16, device="cuda")
    return c, q, below * math.log(2.0) / dim


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("keys,where,below", [(8192, 0, 26.0), (8192, 8191, 25.0), (20000, 300, 27.5), (130, 64, 24.25)])
@pytest.mark.parametrize("splits", [1, 3])
def test_prefill(keys, where, below, splits, dim):
    c, q, scale = one_large_key(keys, dim, 2, where, below)
    c.lens.fill_(keys - 1)
    out = prefill(c, q, offsets([1]), 8, scale, splits)
    k, v = row_contents(c, 0, 0, keys)
    check_attention(out, q, k, v, keys, scale, **HOLD)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [1, 3, 20, 70])
def test_decode_with_and_without_a_shared_prefix(rows, dim):
    keys = 8192
    for where in (0, keys - 1):
        c, q, scale = one_large_key(keys, dim, 2, where, 26.0, rows=rows)
        k, v = row_contents(c, 0, 0, keys)
        for shared in (0, 4096, keys):
            out = decode(c, q, 8, scale, (c.page_table[0].clone(), ints([shared])) if shared else None)
            for i in range(rows):
                check_attention(out[i: i + 1], q[i: i + 1], k, v, keys, scale, (where, shared, i), **HOLD)


def test_a_tile_cannot_be_lost_beside_tiles_of_other_v_scales():
    """Tiles whose V scale is above a half carry it in the exponent, beside tiles whose scale is in the operand.  Tile t is the only
    one with values in dimension t, so a tile that is lost is a dimension that is zero."""
    for dim, tiles in ((128, 120), (64, 60)):
        from runtherder_b200.kv_cache import PagedKVCache
        ps = 64
        c = PagedKVCache(1, tiles, ps, 2, dim, 1, tiles)
        c.page_table.copy_(torch.arange(tiles, dtype=torch.int32, device="cuda").view(1, -1))
        g = torch.Generator(device="cuda").manual_seed(dim)
        c.k.copy_(torch.randn(c.k.shape, device="cuda", generator=g).to(torch.float8_e4m3fn).view(torch.uint8))
        c.k_scale.fill_(0.5)
        c.v.zero_()
        for t in range(tiles):
            c.v[0, t, :, :, t] = 0x38
            c.v_scale[0, t] = 2.0 ** (t % 9 - 4) if t % 2 else 2.0 ** -10
        n = tiles * ps
        c.lens.fill_(n - 3)
        q = torch.randn(3, 8, dim, device="cuda", generator=g).to(torch.bfloat16)
        out = prefill(c, q, offsets([3]), 8, 1.0 / math.sqrt(dim)) if dim else None
        k, v = row_contents(c, 0, 0, n)
        # Relative to each dimension's own value: a tile's 64 weights (f16, 2^-11 each) in units of a maximum that lies at most
        # 2^(4 + 8) above theirs by the V scales and some 2^6 by the scores, so at 2^-11 of 2^7 or more: subnormals' half step
        # 2^-25 is 2^-21 of them.  Scores: 2^-16 of |q| sum |k| scale = 4 * 128 * 0.4 / 11, four times over.
        want = torch.stack([torch.softmax((q[i].double().view(2, 4, 1, dim) * k[:, None, : n - 2 + i]).sum(-1) / math.sqrt(dim), -1) @ v[:, : n - 2 + i]
                            for i in range(3)]).view(3, 8, dim)
        got = out.double()
        used = want[..., :tiles]
        assert (used > 0).all()
        assert ((got[..., :tiles] - used).abs() <= used * (2.0 ** -8 + 4 * 2.0 ** -11 + 4 * 2.0 ** -16 * 20 + 2.0 ** -13)).all()
        assert not got[..., tiles:].any()
