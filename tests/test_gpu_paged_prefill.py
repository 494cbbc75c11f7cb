"""rh_flash_prefill_packed_bf16 against attention in 64 bits over what the pages hold (paged_util.check_attention derives the
tolerance; here the V operand is rounded to f16 once more, 2^-11 of each term, as is the scale it is multiplied with, and q is
the sum of two E4M3 parts, off by at most 2^-16 of the row's largest value)."""
import math

import pytest
import torch

from paged_util import check_attention, ints, offsets, row_contents
from test_gpu_paged_decode import filled, queries

pytestmark = pytest.mark.gpu

HOLD = dict(extra=2.0 * 2.0 ** -11, small_step=2.0 ** -25, q_step=2.0 ** -16)      # the V operand: f16 of (code x f16 of the scale)


def prefill(c, q, cu, num_q, scale, splits=1, rows=None, layer=0, out=None, total=None, num_seqs=None):
    from runtherder_b200 import kernels as K
    total = q.shape[0] if total is None else total
    n = (cu.numel() - 1) if num_seqs is None else num_seqs
    out = torch.full((total, num_q, c.head_dim), 7.0, dtype=torch.bfloat16, device="cuda") if out is None else out
    part = torch.full((K.flash_prefill_packed_scratch_floats(total, num_q, c.head_dim, splits),), float("nan"), device="cuda")
    K.flash_prefill_packed_bf16(out, q, c, layer, cu, total, n, num_q, scale, part, splits, None if rows is None else ints(rows))
    return out


def check(c, out, q, new, held, scale, rows=None, layer=0, what="", mixed=False):
    at, worst = 0, 0.0
    for i, (n, h) in enumerate(zip(new, held)):
        row = i if rows is None else rows[i]
        if n and h >= 0:
            k, v = row_contents(c, layer, row, h + n)
            worst = max(worst, check_attention(out[at: at + n], q[at: at + n], k, v, h + 1, scale, (what, i, n, h), mixed=mixed, **HOLD))
        elif n:
            assert not out[at: at + n].any(), (what, i)
        at += n
    assert (out[at:] == 7.0).all(), "padding was written"
    return worst


def batch(new, held, hq, hkv, dim, ps, seed=0, mul=1.0, pad=0, layers=1, **kw):
    """A cache that holds the keys of every entry's history and new tokens, with lens set to the history."""
    c = filled([(h + n - 1 if h >= 0 else -1) for n, h in zip(new, held)], heads=hkv, dim=dim, ps=ps, seed=seed, layers=layers, **kw)
    c.lens.copy_(ints(held))
    return c, queries(sum(new) + pad, hq, dim, seed, mul), offsets(new)


CASES = [
    # new tokens, history, q heads, kv heads, dim, page size
    ([1], [0], 8, 2, 128, 16), ([1], [63], 4, 4, 64, 16), ([64], [0], 4, 1, 128, 32), ([65, 1, 63], [0, 64, 1], 6, 2, 128, 16),
    ([5, 0, 33, 129, 200], [0, 0, 0, 0, 0], 24, 8, 128, 16), ([300, 7], [0, 700], 32, 8, 64, 64), ([40, 41], [1000, 3], 28, 4, 128, 128),
    ([17] * 40, [5] * 40, 8, 8, 64, 16), ([130, 0, 2], [20, 5, 0], 40, 8, 128, 256), ([600], [0], 2, 2, 128, 64), ([257], [511], 9, 1, 64, 32),
    ([3, 50, 4], [-1, 10, 100], 16, 4, 128, 16), ([128, 128, 127], [0, 1, 62], 7, 7, 128, 16),
]


@pytest.mark.parametrize("new,held,hq,hkv,dim,ps", CASES)
@pytest.mark.parametrize("flavour", ["plain", "peaked", "spread"])
def test_packed_batches(new, held, hq, hkv, dim, ps, flavour):
    """`spread` has V scales of widely different size: some tiles carry them in the exponent."""
    kw, mul = {"plain": ({}, 1.0), "peaked": ({}, 6.0), "spread": (dict(v_spread=4.0), 3.0)}[flavour]
    c, q, cu = batch(new, held, hq, hkv, dim, ps, seed=sum(new) + dim, mul=mul, pad=3, **kw)
    scale = 1.0 / math.sqrt(dim)
    check(c, prefill(c, q, cu, hq, scale), q, new, held, scale, what=flavour, mixed=flavour == "spread")


@pytest.mark.parametrize("new,held,hq,hkv,dim,ps,splits", [
    ([1], [5000], 8, 2, 128, 16, 8), ([40, 3], [1500, 0], 32, 8, 64, 32, 3), ([130, 5, 0, 64], [64, 2000, 3, 700], 6, 2, 128, 64, 5), ([2], [1], 4, 4, 128, 16, 64),
    ([300], [900], 32, 8, 128, 16, 2),
])
def test_keys_dealt_to_several_ranges(new, held, hq, hkv, dim, ps, splits):
    c, q, cu = batch(new, held, hq, hkv, dim, ps, seed=splits, pad=2, mul=2.0)
    scale = 1.0 / math.sqrt(dim)
    out = prefill(c, q, cu, hq, scale, splits)
    check(c, out, q, new, held, scale, what=splits)
    assert torch.equal(out, prefill(c, q, cu, hq, scale, splits))
    check(c, prefill(c, q, cu, hq, scale), q, new, held, scale, what="one range")


def test_rows_layers_strides_and_missing_pages():
    dim, ps, hq, hkv = 128, 16, 12, 4
    c, q0, _ = batch([60, 90, 1], [10, 0, 100], hq, hkv, dim, ps, seed=4, layers=2)
    rows, new = [2, 0, 99, 1], [1, 60, 5, 90]
    wide = queries(sum(new), hq + 8, dim, 2).view(sum(new), -1)
    q = wide[:, 8 * dim:]
    out = prefill(c, q, offsets(new), hq, 0.1, rows=rows, layer=1)
    flat = q.reshape(-1, hq, dim)
    for at, n, row, h in ((0, 1, 2, 100), (1, 60, 0, 10), (66, 90, 1, 0)):
        k, v = row_contents(c, 1, row, h + n)
        check_attention(out[at: at + n], flat[at: at + n], k, v, h + 1, 0.1, (row,), **HOLD)
    assert not out[61:66].any()                                  # an unknown row
    # a page that is missing and one that is none of the pool: their keys are left out
    c.page_table[2, 1], c.page_table[2, 4] = -1, c.num_pages + 5
    out = prefill(c, q, offsets([1]), hq, 0.1, rows=[2], total=1)
    c.page_table[2, 1], c.page_table[2, 4] = 0, 0
    keep = [j for j in range(101) if j // ps not in (1, 4)]
    k, v = row_contents(c, 0, 2, 101)
    check_attention(out[:1], flat[:1], k[:, keep], v[:, keep], len(keep), 0.1, "missing", **HOLD)


@pytest.mark.parametrize("dim", [64, 128])
def test_nan_keys_reach_the_tokens_that_see_them_and_no_others(dim):
    """A NaN code in V, in K, a NaN V scale and an infinite one, each in the middle of a prompt."""
    hq, hkv, n = 8, 2, 200
    scale = 1.0 / math.sqrt(dim)
    clean, q, cu = batch([n], [0], hq, hkv, dim, 16, seed=5)
    for place, how in ((130, "v"), (150, "k"), (70, "v_scale"), (199, "inf"), (0, "v")):
        c, q, cu = batch([n], [0], hq, hkv, dim, 16, seed=5)
        page, slot = int(c.page_table[0, place // 16]), place % 16
        if how in ("v", "k"):
            (c.v if how == "v" else c.k)[0, page, 0, slot, 3] = 0x7f
        else:
            c.v_scale[0, page, 0, slot] = float("nan") if how == "v_scale" else float("inf")
        out = prefill(c, q, cu, hq, scale)
        k, v = row_contents(clean, 0, 0, n)
        group = hq // hkv
        if place:
            check_attention(out[:place], q[:place], k[:, :place], v[:, :place], 1, scale, how, **HOLD)
        check_attention(out[:, group:], q[:, group:], k[1:], v[1:], 1, scale, (how, "other head"), **HOLD)
        assert torch.isnan(out[place:, :group, 3]).all(), (how, place)


def test_extreme_scales_and_queries():
    hq, hkv, dim, n = 8, 2, 128, 300
    c, q, cu = batch([n], [0], hq, hkv, dim, 16, seed=6, stale_nan=False)
    p = c.page_table[0].tolist()
    c.k_scale[0, p[1], :, 3:6] = 0
    c.v_scale[0, p[2], :, 1:9] = 0
    c.v_scale[0, p[3]] *= 1e6
    c.v_scale[0, p[5]] *= 1e-9
    c.v_scale[0, p[9]] *= 1e-4
    scale = 1.0 / math.sqrt(dim)
    check(c, prefill(c, q, cu, hq, scale), q, [n], [0], scale, mixed=True)
    q[4] = 0
    q[200, 5] *= 1e-30
    check(c, prefill(c, q, cu, hq, scale), q, [n], [0], scale, mixed=True)
    q *= 1e28
    check(c, prefill(c, q, cu, hq, scale * 1e-28), q, [n], [0], scale * 1e-28, mixed=True)
    q[7, 2, 5], q[9, 1, 0] = float("inf"), float("nan")
    out = prefill(c, q, cu, hq, scale * 1e-28)
    assert torch.isnan(out[7, 2]).all() and torch.isnan(out[9, 1]).all()
    q[7, 2, 5], q[9, 1, 0] = 0, 0
    out[7, 2], out[9, 1] = prefill(c, q, cu, hq, scale * 1e-28)[7, 2], prefill(c, q, cu, hq, scale * 1e-28)[9, 1]
    check(c, out, q, [n], [0], scale * 1e-28, mixed=True)


@pytest.mark.parametrize("scale", [0.0, -0.1])
def test_softmax_scale_of_zero_and_below(scale):
    c, q, cu = batch([70, 5], [0, 40], 8, 2, 128, 16, seed=11)
    check(c, prefill(c, q, cu, 8, scale), q, [70, 5], [0, 40], scale)


@pytest.mark.parametrize("scale,mul", [(0.0, 1e-25), (1e-30, 1e-20), (-1e-37, 1e-30), (1e-3, 1e-36)])
def test_scores_that_vanish(scale, mul):
    """Softmax scale times the queries' size below what fp32 holds: every visible key counts the same, masked ones not at all."""
    c, q, cu = batch([70, 5], [0, 40], 8, 2, 128, 16, seed=12)
    q = (q.float() * mul).to(torch.bfloat16)
    check(c, prefill(c, q, cu, 8, scale), q, [70, 5], [0, 40], scale)


def test_queries_of_widely_different_size_in_a_row():
    """Elements far below a row's largest one: what the two parts of q lose must stay within 2^-16 of it."""
    hq, hkv, dim = 8, 2, 128
    c, q, cu = batch([150], [30], hq, hkv, dim, 32, seed=13)
    q *= torch.exp2(-torch.randint(0, 22, q.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).float()).to(torch.bfloat16)
    for mul in (1.0, 200.0):
        check(c, prefill(c, q * mul, cu, hq, 0.1), q * mul, [150], [30], 0.1)


def test_long_prompt_sampled_tokens_and_repeatability():
    """8192 tokens in one of three sequences: sampled tokens against 64 bits, the same bits twice."""
    hq, hkv, dim, ps = 32, 8, 128, 64
    new, held = [100, 8000, 92], [0, 0, 4000]
    c, q, cu = batch(new, held, hq, hkv, dim, ps, seed=7)
    scale = 1.0 / math.sqrt(dim)
    out = prefill(c, q, cu, hq, scale)
    assert torch.equal(out, prefill(c, q, cu, hq, scale))
    k, v = row_contents(c, 0, 1, 8000)
    for i in (0, 1, 63, 64, 4001, 7935, 7999):
        t = 100 + i
        check_attention(out[t: t + 1], q[t: t + 1], k[:, : i + 1], v[:, : i + 1], i + 1, scale, i, **HOLD)
    k, v = row_contents(c, 0, 2, 4092)
    check_attention(out[8100:], q[8100:], k, v, 4001, scale, "behind", **HOLD)


def test_pages_beyond_32_bit_offsets():
    """Append, copy and packed prefill on pages that start more than 2^32 bytes into a layer's codes, in the second layer."""
    from runtherder_b200 import kernels as K
    from runtherder_b200.kv_cache import PagedKVCache
    heads, hq, ps, dim, n = 8, 32, 256, 128, 300
    pages = (1 << 32) // (heads * ps * dim) + 40
    c = PagedKVCache(2, pages, ps, heads, dim, 1, 2)
    mine = [pages - 1, pages - 7]
    c.page_table.copy_(ints([mine]))
    c.lens.fill_(0)
    for p in mine:
        c.ref_counts[p] = 1
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn(n, heads, dim, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    cu, q = offsets([n]), queries(n, hq, dim, 3)
    c.append(1, k, v, cu, n, 1)
    kk, vv = row_contents(c, 1, 0, n)
    for got, x in ((kk, k), (vv, v)):           # half a step of E4M3 is 2^-4 of the value, and 2^-10 / 448 of the row's largest below its normal range
        x = x.double().transpose(0, 1)
        assert ((got - x).abs() <= 2.0 ** -4 * 1.001 * x.abs() + x.abs().amax(-1, keepdim=True) * 2.0 ** -10 / 448).all()
    assert not c.k[0, mine[0]].any() and not c.k[1, 0].any()
    check(c, prefill(c, q, cu, hq, 0.09, layer=1), q, [n], [0], 0.09, layer=1)
    K.kv_pages_copy(c, ints(mine), ints([3, 1]), 2)
    for slab in (c.k, c.v, c.k_scale, c.v_scale):
        assert torch.equal(slab[:, 3], slab[:, mine[0]]) and torch.equal(slab[:, 1], slab[:, mine[1]])


def test_captured_and_replayed_with_other_lengths():
    from runtherder_b200 import kernels as K
    K.init(0)
    hq, hkv, dim, ps = 16, 4, 128, 16
    c, q, _ = batch([90, 60, 50], [30, 0, 200], hq, hkv, dim, ps, seed=9, stale_nan=False)
    cu = offsets([90, 60, 50])
    runs = []
    for splits in (1, 3):
        out = torch.full((200, hq, dim), 7.0, dtype=torch.bfloat16, device="cuda")
        part = torch.empty(K.flash_prefill_packed_scratch_floats(200, hq, dim, splits), device="cuda")
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            K.flash_prefill_packed_bf16(out, q, c, 0, cu, 200, 3, hq, 0.1, part, splits)
        runs.append((out, part, graph, stream))
    for new, held in (([90, 60, 50], [30, 0, 200]), ([0, 10, 1], [3, 40, 17]), ([100, 0, 0], [20, 1, 1]), ([1, 1, 1], [119, 59, 249])):
        cu.copy_(offsets(new))
        c.lens.copy_(ints(held))
        for out, _, graph, stream in runs:
            out.fill_(7.0)
        torch.cuda.synchronize()
        for out, _, graph, stream in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for out, *_ in runs:
            check(c, out, q, new, held, 0.1)
    assert K.device_error() == 0


def test_refusals():
    from runtherder_b200 import kernels as K
    from runtherder_b200._lib import RhError
    c, q, cu = batch([5, 3], [0, 0], 8, 2, 128, 16)
    out = torch.empty(8, 8, 128, dtype=torch.bfloat16, device="cuda")
    part = torch.empty(K.flash_prefill_packed_scratch_floats(8, 8, 128, 2), device="cuda")
    ok = dict(out=out, q=q, layer=0, cu_seqlens=cu, num_tokens=8, num_seqs=2, num_q_heads=8, scale=0.1, partial=part, num_splits=2)
    K.flash_prefill_packed_bf16(cache=c, **ok)
    for bad in (dict(out=out[:7]), dict(out=out.half()), dict(q=q.float()), dict(q=q[:7]), dict(layer=1), dict(num_seqs=0), dict(num_seqs=3),
                dict(num_tokens=0), dict(num_tokens=9), dict(num_q_heads=7), dict(partial=None), dict(partial=part[:-1]), dict(num_splits=0),
                dict(num_splits=65), dict(cu_seqlens=cu.long()), dict(cu_seqlens=cu[:2]), dict(rows=ints([1]))):
        with pytest.raises(RhError):
            K.flash_prefill_packed_bf16(cache=c, **{**ok, **bad})
