"""The paged operators together, as a server uses them: a system prompt is prefilled once and forked, the requests' own
prompts follow as one ragged batch, decoding steps recorded into a graph share the prompt's keys, requests end, the pool is
compacted, and decoding goes on.  Attention is held against 64 bits over what the pages hold at each step, and what the
pages hold against every sequence's own list of keys and values at the end."""
import math

import pytest
import torch

from paged_util import Model, check_attention, e4m3_table, ints, offsets, row_contents
from test_gpu_paged_cache import reference_append
from test_gpu_paged_decode import BLOCKS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests,prompt,ps,heads,dim", [(3, 300, 16, 2, 128), (25, 523, 64, 2, 128), (9, 40, 32, 3, 64)])
def test_a_serving_session(requests, prompt, ps, heads, dim):
    from runtherder_b200 import kernels as K
    from runtherder_b200.kv_cache import PagedKVCache
    K.init(0)
    layers, hq, steps = 2, 4 * heads, 12
    per = -(-(prompt + 64) // ps)
    pages = per + (requests + 1) * (-(-64 // ps) + 2)
    cache, model = PagedKVCache(layers, pages, ps, heads, dim, requests + 1, per), Model(pages, ps, requests + 1, per)
    g = torch.Generator(device="cuda").manual_seed(7)
    scale = 1.0 / math.sqrt(dim)
    inv_freq = (10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float32) / dim)).contiguous()
    said = [[([], []) for _ in range(layers)] for _ in range(requests + 1)]      # per row and layer: the keys (codes, scales) and values

    def fresh(n):
        return [torch.randn(layers, n, h, dim, device="cuda", generator=g).to(torch.bfloat16) for h in (hq, heads, heads)]

    def remember(layer, rows, new, k, v):
        at = 0
        for r, n in zip(rows, new):
            for kept, x in zip(said[r][layer], (k, v)):
                if n:
                    kept.append(reference_append(x[at: at + n], heads, dim))
            at += n

    def prefill(rows, new):
        q, k, v = fresh(sum(new))
        cu, on = offsets(new), ints(rows)
        held = cache.lens[on.long()].tolist()
        positions = torch.cat([torch.arange(h, h + n) for h, n in zip(held, new)]).to(torch.int32).cuda()
        cache.reserve(cu, len(rows), on)
        model.reserve(rows, new)
        splits = K.flash_prefill_packed_splits(sum(new), len(rows), max(h + n for h, n in zip(held, new)), hq, heads, dim)
        scratch = torch.empty(max(1, K.flash_prefill_packed_scratch_floats(sum(new), hq, dim, splits)), device="cuda")
        for layer in range(layers):
            K.rope_bf16(q[layer], k[layer], positions, inv_freq, sum(new), hq, heads, dim)
            cache.append(layer, k[layer], v[layer], cu, sum(new), len(rows), on)
            out = torch.empty_like(q[layer])
            K.flash_prefill_packed_bf16(out, q[layer], cache, layer, cu, sum(new), len(rows), hq, scale, scratch, splits, on)
            remember(layer, rows, new, k[layer], v[layer])
            at = 0
            for r, n, h in zip(rows, new, held):
                if n:
                    kk, vv = row_contents(cache, layer, r, h + n)
                    check_attention(out[at: at + n], q[layer, at: at + n], kk, vv, h + 1, scale, ("prefill", layer, r), **BLOCKS)
                at += n
        cache.advance(cu, len(rows), on)
        model.advance(rows, new)
        model.check(cache)

    cache.start(1, ints([0]))
    model.release([0], 0)
    prefill([0], [prompt])
    children = list(range(1, requests + 1))
    cache.fork(ints([0] * requests), ints(children), requests)
    model.fork([0] * requests, children)
    for r in children:
        said[r] = [tuple(list(x) for x in layer) for layer in said[0]]
    model.check(cache)
    prefill(children, [(7 * r) % 30 for r in children])          # (the first request of thirty has nothing to add)

    # ---- decoding steps, recorded once ----
    q, k, v = (torch.empty(layers, requests, h, dim, dtype=torch.bfloat16, device="cuda") for h in (hq, heads, heads))
    out = torch.empty_like(q)
    on, one_each = ints(children), offsets([1] * requests)
    positions = torch.empty(requests, dtype=torch.int32, device="cuda")
    shared_len = ints([prompt // ps * ps])
    scratch = torch.empty(K.flash_decode_paged_scratch_floats(requests, hq, heads, dim), device="cuda")
    shared_pages = cache.page_table[0]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        torch.index_select(cache.lens, 0, on.long(), out=positions)
        cache.reserve(one_each, requests, on)
        for layer in range(layers):
            K.rope_bf16(q[layer], k[layer], positions, inv_freq, requests, hq, heads, dim)
            cache.append(layer, k[layer], v[layer], one_each, requests, requests, on)
            K.flash_decode_paged_bf16(out[layer], q[layer], cache, layer, requests, hq, scale, scratch, shared_pages, shared_len, on)
        cache.advance(one_each, requests, on)

    def decode(live, what):
        for into, x in zip((q, k, v), fresh(requests)):
            into.copy_(x)
        held = list(model.lens)
        graph.replay()
        model.reserve(children, [1] * requests)
        for layer in range(layers):
            for i, r in enumerate(children):
                if r not in live:
                    assert not out[layer, i].any(), (what, "an idle row's output", r)
                    continue
                remember(layer, [r], [1], k[layer, i: i + 1], v[layer, i: i + 1])
                kk, vv = row_contents(cache, layer, r, held[r] + 1)
                check_attention(out[layer, i: i + 1], q[layer, i: i + 1], kk, vv, held[r] + 1, scale, (what, layer, r), **BLOCKS)
        model.advance(children, [1] * requests)
        model.check(cache)

    live = set(children)
    for step in range(steps):
        if step == steps // 2:       # every third request ends, and the pages that are left move together
            gone = children[::3]
            cache.release(len(gone), ints(gone))
            model.release(gone)
            live -= set(gone)
            cache.compact()
            model.compact()
            model.check(cache)
        decode(live, step)
    assert model.short == 0 and model.refused == 0

    values = e4m3_table().cuda()
    for r in [0] + sorted(live):
        for layer in range(layers):
            for kept, got in zip(said[r][layer], row_contents(cache, layer, r, model.lens[r], values)):
                codes, scales = (torch.cat([x[i] for x in kept]) for i in range(2))
                want = values[codes.view(torch.uint8).long()] * scales.double().unsqueeze(-1)
                assert torch.equal(want.permute(1, 0, 2), got), (r, layer)
