"""rh_flash_decode_paged_bf16 against attention in 64 bits over what the pages hold (paged_util.check_attention derives the
tolerance): head layouts, page sizes, lengths from one key on, shared prefixes and rows that do not take part."""
import math
import random

import pytest
import torch

from paged_util import check_attention, ints, offsets, row_contents

pytestmark = pytest.mark.gpu


def filled(lens, shared=0, heads=2, dim=128, ps=16, rows=None, seed=0, k_mul=1.0, v_spread=0.0, layers=1, stale_nan=True, own_shared_pages=False):
    """A cache whose row i holds lens[i] tokens and has a place for one more (-1: idle); the first `shared` keys of all rows
    lie in the same pages.  Every place that is no key of a row holds NaN codes and NaN scales."""
    from runtherder_b200.kv_cache import PagedKVCache
    R = len(lens) if rows is None else rows
    per = max(1, max(-(-(n + 1) // ps) for n in lens)) + 1
    g = torch.Generator(device="cuda").manual_seed(seed)
    sp = shared // ps
    counts = [0 if n < 0 else -(-(n + 1) // ps) for n in lens]
    total = sp + sum(max(0, n - sp) for n in counts) + 2
    c = PagedKVCache(layers, total, ps, heads, dim, R, per)
    order = torch.randperm(total, generator=g, device="cuda").tolist()
    at = sp
    table = [[-1] * per for _ in range(R)]
    for i, n in enumerate(counts):
        table[i][:n] = order[:sp][:n] + order[at: at + max(0, n - sp)]
        at += max(0, n - sp)
    c.page_table.copy_(ints(table))
    c.lens.copy_(ints([(lens[i] if i < len(lens) else -1) for i in range(R)]))
    for codes, scales, spread in ((c.k, c.k_scale, 0.0), (c.v, c.v_scale, v_spread)):
        x = torch.randn(*codes.shape, device="cuda", generator=g) * (k_mul if codes is c.k else 1.0)
        if spread:
            x *= torch.exp(torch.randn(*codes.shape[:-1], 1, device="cuda", generator=g) * spread)
        s = x.abs().amax(-1) / 448.0
        codes.copy_((x / s.unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8))
        scales.copy_(s)
    if stale_nan:
        key = torch.zeros(total, ps, dtype=torch.bool, device="cuda")
        for i, n in enumerate(lens):
            for j in range(counts[i]):
                key[table[i][j], : min(ps, n + 1 - j * ps)] = True
        c.k.masked_fill_(~key[None, :, None, :, None], 0x7f)
        c.v.masked_fill_(~key[None, :, None, :, None], 0xff)
        c.k_scale.masked_fill_(~key[None, :, None], float("nan"))
        c.v_scale.masked_fill_(~key[None, :, None], float("inf"))
    return c


def queries(n, heads, dim, seed, mul=1.0):
    g = torch.Generator(device="cuda").manual_seed(1000 + seed)
    return (torch.randn(n, heads, dim, device="cuda", generator=g) * mul).to(torch.bfloat16)


def decode(c, q, num_q, scale, shared=None, rows=None, layer=0, out=None, partial=None):
    from runtherder_b200 import kernels as K
    n = q.shape[0]
    out = torch.full((n, num_q, c.head_dim), float("nan"), dtype=torch.bfloat16, device="cuda") if out is None else out
    need = K.flash_decode_paged_scratch_floats(n, num_q, c.num_kv_heads, c.head_dim)
    partial = torch.full((need,), float("nan"), device="cuda") if partial is None else partial
    table, length = (None, None) if shared is None else shared
    K.flash_decode_paged_bf16(out, q, c, layer, n, num_q, scale, partial, table, length, None if rows is None else ints(rows))
    return out


BLOCKS = dict(extra=2.0 * 2.0 ** -11, small_step=2.0 ** -25, q_step=2.0 ** -16)     # the tcgen05 form of the prefix rounds the V operand (code x f16 of the scale) to f16


def check(c, out, q, scale, lens, rows=None, layer=0, what="", **hold):
    worst = 0.0
    for i in range(q.shape[0]):
        row = i if rows is None else rows[i]
        n = lens[row] if 0 <= row < len(lens) else -1
        if n < 0:
            assert not out[i].any(), (what, i)
            continue
        k, v = row_contents(c, layer, row, n + 1)
        worst = max(worst, check_attention(out[i: i + 1], q[i: i + 1], k, v, n + 1, scale, (what, i, n), **hold))
    return worst


CASES = [
    # lens (-1: idle), q heads, kv heads, dim, page size
    ([0], 8, 2, 128, 16), ([15], 4, 4, 128, 16), ([16], 3, 1, 64, 16), ([1000], 24, 8, 128, 16), ([8195], 24, 8, 128, 64),
    ([0, 1, 14, 15, 16, 17, 31, 32, 33], 6, 2, 128, 32), ([5, -1, 700, 63, -1, 64], 32, 8, 128, 64), ([333, 20, 1], 40, 8, 64, 16),
    ([77, 500], 16, 1, 64, 128), ([300, 0, 9], 28, 4, 128, 256), ([40] * 70, 2, 2, 64, 16), ([2100, 3, 3, 3], 9, 1, 128, 16),
    ([-1, -1], 4, 2, 128, 16), ([3] * 300, 8, 8, 128, 16),
]


@pytest.mark.parametrize("lens,hq,hkv,dim,ps", CASES)
@pytest.mark.parametrize("flavour", ["plain", "peaked", "spread"])
def test_own_keys(lens, hq, hkv, dim, ps, flavour):
    kw, mul = {"plain": ({}, 1.0), "peaked": ({}, 6.0), "spread": (dict(v_spread=2.0), 3.0)}[flavour]
    c = filled(lens, heads=hkv, dim=dim, ps=ps, seed=len(lens) + dim, **kw)
    q = queries(len(lens), hq, dim, ps, mul)
    scale = 1.0 / math.sqrt(dim)
    check(c, decode(c, q, hq, scale), q, scale, lens, what=flavour)


SHARED = [
    # shared keys, own keys behind them per sequence (-1 own: the row holds nothing at all), q heads, kv heads, dim, page size
    (256, [0, 1, 2, 40], 8, 2, 128, 16), (512, [0, 16, 17], 24, 8, 128, 64), (300, [5, 0, 100, 1], 6, 2, 64, 16),
    (1024, [3, -1, 90, 0, -1], 16, 2, 128, 128), (2048, [1] * 33, 4, 4, 64, 32), (768, [10, 700], 40, 8, 128, 256),
    (255, [4, 9], 4, 1, 128, 16), (4096, [100] * 12, 32, 8, 128, 16), (512, [20] * 130, 8, 8, 128, 16),
    (1536, [30, -1] + [9] * 80, 24, 8, 128, 16), (2816, [2] * 100, 8, 1, 64, 32), (1024, [1] * 17, 16, 4, 128, 64), (768, [0] * 300, 4, 1, 128, 128),
]


@pytest.mark.parametrize("shared,own,hq,hkv,dim,ps", SHARED)
@pytest.mark.parametrize("mul", [1.0, 5.0])
def test_shared_prefix(shared, own, hq, hkv, dim, ps, mul):
    """The prefix lies in whole pages; shared_len may name more than is cut down to a multiple of 256, or nothing."""
    pages = shared // ps * ps
    lens = [-1 if o < 0 else pages + o for o in own]
    c = filled(lens, shared=pages, heads=hkv, dim=dim, ps=ps, seed=shared)
    q = queries(len(own), hq, dim, shared, mul)
    scale = 1.0 / math.sqrt(dim)
    table = c.page_table[next(i for i, n in enumerate(lens) if n >= 0)].clone()
    out = decode(c, q, hq, scale, (table, ints([pages])))
    hold = BLOCKS if len(own) * hq // hkv >= 17 else {}      # (the tcgen05 form takes prefixes from 17 query rows on)
    check(c, out, q, scale, lens, what="shared", **hold)
    plain = decode(c, q, hq, scale)
    check(c, plain, q, scale, lens, what="own")
    none = decode(c, q, hq, scale, (table, ints([0])))
    assert torch.equal(none, plain)
    assert torch.equal(out, decode(c, q, hq, scale, (table, ints([pages]))))     # the same call twice: the same bits


@pytest.mark.parametrize("batch,hq,hkv", [(6, 8, 2), (70, 8, 2), (40, 8, 2)])
def test_rows_shorter_than_the_prefix_and_nan_keys(batch, hq, hkv):
    """A row that holds fewer keys than are shared attends those it holds, whatever the others are: NaN codes among the keys it
    does not see must not reach it, and must reach the rows that do see them."""
    dim, ps, shared = 128, 16, 512
    lens = [shared + 7] * batch
    c = filled(lens, shared=shared, heads=hkv, dim=dim, ps=ps, seed=3)
    bad = int(c.page_table[0, 300 // ps])
    c.v[0, bad, 0, 300 % ps, 5] = 0x7f
    short = {1: 299, 2: 0, 4: -1, batch - 1: 100}
    for r, n in short.items():
        lens[r] = n
        c.lens[r] = n
    q = queries(batch, hq, dim, 5)
    scale = 1.0 / math.sqrt(dim)
    out = decode(c, q, hq, scale, (c.page_table[0].clone(), ints([shared])))
    clean = filled([shared + 7] * batch, shared=shared, heads=hkv, dim=dim, ps=ps, seed=3)
    group = hq // hkv
    hold = BLOCKS if batch * group >= 17 else {}
    for i in range(batch):
        if lens[i] < 0:
            assert not out[i].any()
        elif i in short:
            k, v = row_contents(clean, 0, i, lens[i] + 1)
            check_attention(out[i: i + 1], q[i: i + 1], k, v, lens[i] + 1, scale, ("short", i), **hold)
        else:
            k, v = row_contents(clean, 0, i, lens[i] + 1)
            assert torch.isnan(out[i, :group, 5]).all(), i            # the poisoned dimension of the heads that see the key
            check_attention(out[i: i + 1, group:], q[i: i + 1, group:], k[1:], v[1:], lens[i] + 1, scale, ("rest", i), **hold)


def test_rows_layers_strides_and_pages_that_are_not_there():
    dim, ps, hq, hkv = 128, 16, 12, 4
    lens = [100, 33, -1, 257]
    c = filled(lens, heads=hkv, dim=dim, ps=ps, seed=8, layers=3)
    rows = [3, 1, 2, 9, -1, 0, 3]                       # an idle row, rows that do not exist, one row twice
    wide = queries(len(rows), hq + 2 * hkv, dim, 1).view(len(rows), -1)
    q = wide[:, : hq * dim]
    scale = 0.1
    out = decode(c, q, hq, scale, rows=rows, layer=2)
    check(c, out, q.reshape(len(rows), hq, dim), scale, lens, rows=rows, layer=2)
    # keys of a page that is missing or no page of the pool are left out
    c.page_table[3, 2], c.page_table[3, 5] = -1, c.num_pages
    out = decode(c, q, hq, scale, rows=[3] * len(rows), layer=1)
    keep = [j for j in range(258) if j // ps not in (2, 5)]
    c.page_table[3, 2], c.page_table[3, 5] = 0, 0
    k, v = row_contents(c, 1, 3, 258)
    for i in range(len(rows)):
        check_attention(out[i: i + 1], q[i: i + 1].reshape(1, hq, dim), k[:, keep], v[:, keep], len(keep), scale, "missing pages")
    # a length behind the table row ends with the row
    c.lens[1] = c.pages_per_row * ps + 1000
    c.page_table[1] = c.page_table[3].clone()
    c.page_table[1, 2], c.page_table[1, 5] = 7, 7
    n = c.pages_per_row * ps
    c.page_table[1, -(-258 // ps):] = 7
    out = decode(c, q[:1], hq, scale, rows=[1], layer=0)
    k, v = row_contents(c, 0, 1, n)
    finite = torch.isfinite(k).all() and torch.isfinite(v).all()
    if bool(finite):
        check_attention(out, q[:1].reshape(1, hq, dim), k, v, n, scale, "full table")


def test_extreme_scales_and_queries():
    """Zero K and V rows (scale 0), V magnitudes 1e-6 and 1e4 side by side, queries of 1e30, 1e-30 and zero."""
    dim, ps, hq, hkv = 128, 16, 8, 2
    lens = [200, 45]
    c = filled(lens, heads=hkv, dim=dim, ps=ps, seed=12, stale_nan=False)
    p = c.page_table[0].tolist()
    c.k_scale[0, p[1], :, 3:6] = 0
    c.v_scale[0, p[2], :, 1:9] = 0
    c.v_scale[0, p[3]] *= 1e4
    c.v_scale[0, p[4]] *= 1e-6
    q = queries(2, hq, dim, 4)
    q[0, 0] = 0
    q[1, 5] *= 1e-30
    scale = 1.0 / math.sqrt(dim)
    check(c, decode(c, q, hq, scale), q, scale, lens)
    big = q.clone()
    big[0, 2] *= 1e28                                   # with a softmax scale that brings the scores back to order one
    out = decode(c, big, hq, scale * 1e-28)
    flat = check(c, out, big, scale * 1e-28, lens)
    assert flat <= 1.0


@pytest.mark.parametrize("shared", [0, 256])
@pytest.mark.parametrize("scale,mul", [(0.0, 1e-25), (1e-30, 1e-20), (-1e-3, 1e-36)])
def test_scores_that_vanish(shared, scale, mul):
    lens = [shared + n for n in (0, 5, 40, 17, 3)]
    c = filled(lens, shared=shared, heads=2, dim=128, ps=16, seed=14)
    q = (queries(5, 8, 128, 3).float() * mul).to(torch.bfloat16)
    for i in (2, 4):                                         # shorter than what is shared: the prefix masks keys too
        lens[i] = 9
        c.lens[i] = 9
    out = decode(c, q, 8, scale, (c.page_table[0].clone(), ints([shared])) if shared else None)
    check(c, out, q, scale, lens, **BLOCKS)


def test_long_cache_beyond_32_bit_offsets():
    """Codes of a page behind 4 GB of the pool."""
    from runtherder_b200.kv_cache import PagedKVCache
    dim, ps, hkv = 128, 256, 8
    pages = (1 << 32) // (hkv * ps * dim) + 9            # a slab of more than 2^32 bytes
    c = PagedKVCache(1, pages, ps, hkv, dim, 2, 3)
    small = filled([300, 700], heads=hkv, dim=dim, ps=ps, seed=2, stale_nan=False)
    c.lens.copy_(small.lens)
    for r in range(2):
        for j in range(3):
            src = int(small.page_table[r, j])
            if src >= 0:
                dst = pages - 1 - 3 * r - j
                c.page_table[r, j] = dst
                c.k[0, dst], c.v[0, dst], c.k_scale[0, dst], c.v_scale[0, dst] = small.k[0, src], small.v[0, src], small.k_scale[0, src], small.v_scale[0, src]
    q = queries(2, 16, dim, 1)
    assert torch.equal(decode(c, q, 16, 0.1), decode(small, q, 16, 0.1))
    # and append and copy reach them as well
    k = queries(1, hkv, dim, 9)
    c.append(0, k, k, offsets([1]), 1, 1, ints([1]))
    small.append(0, k, k, offsets([1]), 1, 1, ints([1]))
    assert torch.equal(c.k[0, pages - 1 - 3 - 2, :, 700 - 512], small.k[0, int(small.page_table[1, 2]), :, 700 - 512])
    c.copy(ints([pages - 1]), ints([0]), 1)
    assert torch.equal(c.k[0, 0], c.k[0, pages - 1]) and torch.equal(c.v_scale[0, 0], c.v_scale[0, pages - 1])


@pytest.mark.parametrize("shared", [0, 512])
def test_captured_and_replayed_with_changing_lengths(shared):
    """Two graphs with scratch of their own on two streams; lengths and the shared length change between replays."""
    from runtherder_b200 import kernels as K
    K.init(0)
    dim, ps, hq, hkv = 128, 16, 16, 4
    lens = [shared + 60, shared + 61, shared + 200]
    c = filled(lens, shared=shared, heads=hkv, dim=dim, ps=ps, seed=6, stale_nan=False)
    table, length = c.page_table[0].clone(), ints([shared])
    scale = 0.09
    runs = []
    for i in range(2):
        q = queries(3, hq, dim, 20 + i)
        out = torch.zeros(3, hq, dim, dtype=torch.bfloat16, device="cuda")
        partial = torch.empty(K.flash_decode_paged_scratch_floats(3, hq, hkv, dim), device="cuda")
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            decode(c, q, hq, scale, (table, length), out=out, partial=partial)
        runs.append((q, out, stream, graph, partial))    # a graph's scratch lives as long as the graph
    for step in range(4):
        now = [max(0, n - 17 * step) for n in lens]
        c.lens.copy_(ints(now))
        length.fill_(shared if step != 2 else 0)
        torch.cuda.synchronize()
        for q, out, stream, graph, _ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for q, out, *_ in runs:
            check(c, out, q, scale, now, what=step)


def test_refusals():
    from runtherder_b200 import kernels as K
    from runtherder_b200._lib import RhError
    c = filled([20, 3], heads=2, dim=128)
    q = queries(2, 8, 128, 0)
    out = torch.empty(2, 8, 128, dtype=torch.bfloat16, device="cuda")
    part = torch.empty(K.flash_decode_paged_scratch_floats(2, 8, 2, 128), device="cuda")
    ok = dict(out=out, q=q, layer=0, num_seqs=2, num_q_heads=8, scale=0.1, partial=part)
    K.flash_decode_paged_bf16(cache=c, **ok)
    for bad in (dict(out=out[:1]), dict(out=out.float()), dict(q=q.float()), dict(q=q[:, :4]), dict(q=q.transpose(1, 2)), dict(layer=1), dict(layer=-1), dict(num_seqs=0),
                dict(num_seqs=3), dict(num_q_heads=7), dict(partial=part[:-1]), dict(partial=part.double()), dict(shared_len=ints([0])),
                dict(shared_pages=c.page_table), dict(shared_pages=c.page_table[0, 1:].contiguous(), shared_len=ints([0])), dict(q=q.cpu()), dict(rows=torch.zeros(2, dtype=torch.int32)), dict(shared_pages=c.page_table, shared_len=torch.zeros(1, dtype=torch.int64, device="cuda")),
                dict(rows=ints([0])), dict(partial=torch.empty(part.numel() + 1, device="cuda")[1:])):
        with pytest.raises(RhError):
            K.flash_decode_paged_bf16(cache=c, **{**ok, **bad})
