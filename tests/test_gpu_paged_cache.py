"""The paged FP8 cache on the GPU: bookkeeping against a host model (whole numbers: equal), page contents bit for bit, the
append against the library's own one-sequence cache writer (bit-identical codes and scales: the same arithmetic)."""
import random

import pytest
import torch

from paged_util import Model, ints, offsets

pytestmark = pytest.mark.gpu


def make(layers=2, pages=24, ps=16, heads=2, dim=64, rows=6, per=5, seed=0):
    from runtherder_b200.kv_cache import PagedKVCache
    c = PagedKVCache(layers, pages, ps, heads, dim, rows, per)
    g = torch.Generator(device="cuda").manual_seed(seed)
    for t in (c.k, c.v):                       # stale contents everywhere, NaN codes among them
        t.copy_(torch.randint(0, 256, t.shape, dtype=torch.uint8, device="cuda", generator=g))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.rand(t.shape, device="cuda", generator=g))
        t.view(-1)[::97] = float("nan")
    return c, Model(pages, ps, rows, per)


def bits(cache):
    return [t.clone().view(torch.int32) if t.dtype == torch.float32 else t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]


def same(cache, want):
    for got, w in zip(bits(cache), want):
        assert torch.equal(got, w)


def apply_moves(want, moves):
    before = [t.clone() for t in want]
    for src, dst, fill in moves:
        for t, b in zip(want, before):
            t[:, dst, :, :fill] = b[:, src, :, :fill]


@pytest.mark.parametrize("seed", range(6))
def test_bookkeeping_follows_the_host_model(seed):
    """Random start / reserve / advance / fork / release / compact steps, with rows out of range, rows named twice, a pool that
    runs dry and sequences that outgrow their table row."""
    rng = random.Random(seed)
    ps = rng.choice([16, 32, 64])
    c, m = make(pages=rng.choice([12, 40, 5000]), ps=ps, rows=rng.choice([3, 8, 70]), per=rng.choice([2, 5]), seed=seed, heads=1, layers=1)
    R = c.num_rows
    for step in range(40):
        op = rng.choice(["start", "grow", "grow", "grow", "fork", "fork", "release", "compact"])
        n = rng.randint(1, min(R, 6))
        rows = rng.sample(range(R), n)
        if rng.random() < 0.2:
            rows[rng.randrange(n)] = rng.choice([-1, R, rows[0]])
        want = bits(c)
        if op == "start":
            c.start(n, ints(rows))
            m.release(rows, 0)
        elif op == "release":
            c.release(n, ints(rows))
            m.release(rows, -1)
        elif op == "grow":
            new = [rng.choice([0, 1, rng.randint(1, 2 * ps)]) for _ in rows]
            c.reserve(offsets(new), n, ints(rows))
            m.reserve(rows, new)
            m.check(c)
            unique = sorted(set(r for r in rows if 0 <= r < R))     # a step names a row once
            held = [new[rows.index(r)] for r in unique]
            cap = [h if m.lens[r] < 0 or m.lens[r] + h <= sum(p >= 0 for p in m.table[r]) * ps else 0 for r, h in zip(unique, held)]
            if unique:
                c.advance(offsets(cap), len(unique), ints(unique))
                m.advance(unique, cap)
        elif op == "fork":
            parents = [rng.randrange(R) for _ in rows]
            if rng.random() < 0.2:
                parents[0] = rng.choice([-2, R])
            c.fork(ints(parents), ints(rows), n)
            apply_moves(want, m.fork(parents, rows))
        else:
            c.compact()
            apply_moves(want, [(s, d, ps) for s, d in m.compact()])
        m.check(c)
        same(c, want)


@pytest.mark.parametrize("ps,heads,dim,layers,n", [(16, 1, 64, 1, 1), (16, 8, 128, 3, 5), (64, 3, 128, 2, 7), (256, 2, 64, 1, 2), (128, 5, 64, 2, 11)])
def test_copy_pages(ps, heads, dim, layers, n):
    c, _ = make(layers=layers, pages=2 * n + 3, ps=ps, heads=heads, dim=dim)
    order = torch.randperm(2 * n + 3, generator=torch.Generator().manual_seed(n)).tolist()
    src, dst = order[:n], order[n: 2 * n]
    if n > 2:
        src[1] = src[0]                        # one page copied twice
        dst[2] = 2 * n + 3                     # no page of the pool: skipped
    want = bits(c)
    apply_moves(want, [(s, d, ps) for s, d in zip(src, dst) if d < 2 * n + 3])
    c.copy(ints(src), ints(dst), n)
    same(c, want)
    assert c.status.tolist() == [0, 1 if n > 2 else 0]


@pytest.mark.parametrize("pages,used", [(20000, 4000), (8192, 8192), (8193, 1), (16385, 9000), (3, 0)])
def test_compact_pools_of_many_pages(pages, used):
    rows, per = 100, 100
    c, m = make(layers=1, pages=pages, ps=16, rows=rows, per=per, heads=1, dim=64)
    rng = random.Random(pages)
    for i, p in enumerate(rng.sample(range(pages), used)):
        m.table[i % rows][i // rows] = p
        m.refs[p] = 1
    for i in range(min(used, 50)):                        # a second row lists some of them
        p = m.table[i % rows][i // rows]
        m.table[(i + 1) % rows][per - 1] = p
        m.refs[p] = 2
    c.page_table.copy_(ints(m.table))
    c.ref_counts.copy_(ints(m.refs))
    want = bits(c)
    c.compact()
    apply_moves(want, [(s, d, 16) for s, d in m.compact()])
    m.check(c)
    same(c, want)


def test_fork_of_a_long_row_and_many_children():
    """More children than a warp has lanes, page lists longer than a warp is wide, and parents that are children themselves."""
    c, m = make(pages=900, ps=16, rows=80, per=70, heads=2, dim=64, layers=2)
    new = [70 * 16 - 3, 33 * 16, 5]
    c.start(3, ints([0, 1, 2]))
    m.release([0, 1, 2], 0)
    c.reserve(offsets(new), 3)
    m.reserve([0, 1, 2], new)
    c.advance(offsets(new), 3)
    m.advance([0, 1, 2], new)
    rng = random.Random(3)
    for _ in range(3):
        parents = [rng.randrange(3 if _ == 0 else 80) for _i in range(77)]
        children = rng.sample(range(3, 80), 77) if _ == 0 else rng.sample(range(80), 77)
        want = bits(c)
        c.fork(ints(parents), ints(children), 77)
        apply_moves(want, m.fork(parents, children))
        m.check(c)
        same(c, want)


def reference_append(k, heads, dim):
    """Codes and scales of [tokens, heads, dim] through the one-sequence cache writer."""
    from runtherder_b200 import kernels as K
    n = k.shape[0] * heads
    q = torch.empty(n, dim, dtype=torch.uint8, device="cuda")
    s = torch.empty(n, dtype=torch.float32, device="cuda")
    K.quantize_kv_fp8(q, s, k.contiguous(), torch.zeros(1, dtype=torch.int32, device="cuda"), 1, n, dim)
    return q.view(-1, heads, dim), s.view(-1, heads)


@pytest.mark.parametrize("heads,dim,ps,new,strided", [
    (2, 64, 16, [1], False), (8, 128, 16, [1] * 40, False), (3, 128, 64, [7, 0, 65, 1, 130, 0], True), (1, 64, 32, [33, 31, 0], True),
    (5, 64, 128, [300], False), (16, 128, 16, [17, 16, 15], True),
])
def test_append_is_the_cache_writer_at_the_rows_places(heads, dim, ps, new, strided):
    from runtherder_b200.kv_cache import PagedKVCache
    rng = random.Random(len(new) * dim)
    n, R = len(new), len(new) + 2
    held = [rng.choice([0, ps - 1, ps, rng.randint(0, 3 * ps)]) for _ in new]
    per = max(-(-(h + x) // ps) for h, x in zip(held, new)) + 1
    c, _ = make(layers=2, pages=R * per, ps=ps, heads=heads, dim=dim, rows=R, per=per)
    rows = rng.sample(range(R), n)
    idle = [r for r in range(R) if r not in rows]
    c.page_table.copy_(torch.randperm(R * per, device="cuda").to(torch.int32).view(R, per))
    for r, h in zip(rows, held):
        c.lens[r] = h
    pad = 3                                     # tokens behind the last sequence are nobody's
    total = sum(new) + pad
    g = torch.Generator(device="cuda").manual_seed(dim)
    wide = torch.randn(total, (4 + 2 * heads) * dim, device="cuda", generator=g).to(torch.bfloat16)
    k, v = wide[:, 4 * dim: (4 + heads) * dim], wide[:, (4 + heads) * dim:]
    k[0] = 0                                    # a zero row: scale 0, codes 0
    v[-1 - pad, 0] = float("inf")
    if not strided:
        k, v = k.contiguous().view(total, heads, dim), v.contiguous().view(total, heads, dim)
    want = bits(c)
    c.append(1, k, v, offsets(new), total, n, ints(rows))
    at = 0
    for i, r in enumerate(rows):
        for name, x in ((0, k), (1, v)):
            codes, scales = reference_append(x[at: at + new[i]].reshape(-1, heads, dim), heads, dim) if new[i] else (None, None)
            for j in range(new[i]):
                pos = held[i] + j
                page = int(c.page_table[r, pos // ps])
                want[name][1, page, :, pos % ps] = codes[j]
                want[2 + name][1, page, :, pos % ps] = scales[j].view(torch.int32)
        at += new[i]
    same(c, want)
    # idle rows, rows and pages out of range, and positions behind the table row: nothing is stored
    c.lens[rows[0]] = -1
    c.page_table[idle[0]] = torch.tensor([-1, c.num_pages, -7][: per] + [-1] * (per - 3), dtype=torch.int32, device="cuda")[:per]
    c.lens[idle[0]] = 0
    c.lens[idle[1]] = per * ps
    for bad in (rows[0], idle[0], idle[1], -1, R, 1 << 30):
        c.append(1, k, v, offsets([min(total, ps)]), min(total, ps), 1, ints([bad]))
    same(c, want)


@pytest.mark.parametrize("n", [3, 70])
def test_a_row_named_twice_counts_once(n):
    """reserve, append and advance take the first of the entries that name a row; the others' tokens go nowhere."""
    c, m = make(layers=1, pages=200, ps=16, rows=80, per=4, heads=2, dim=64)
    c.start(80)
    m.release(range(80), 0)
    rows = list(range(n - 1))
    rows.insert(n // 2 + 1, rows[0])                     # the second one lies in front of others' tokens
    new = [3 + i % 20 for i in range(n)]
    k = torch.randn(sum(new), 2, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(torch.bfloat16)
    cu, on = offsets(new), ints(rows)
    first = [(r, x) for i, (r, x) in enumerate(zip(rows, new)) if r not in rows[:i]]
    codes, scales = reference_append(k, 2, 64)
    for _ in range(2):
        c.reserve(cu, n, on)
        m.reserve(rows, new)
        m.check(c)
        c.append(0, k, k, cu, sum(new), n, on)
        for i, r in enumerate(rows):
            if r in rows[:i]:
                continue
            at = sum(new[:i])
            pos = torch.arange(m.lens[r], m.lens[r] + new[i])
            page = torch.tensor([m.table[r][x] for x in (pos // 16).tolist()])
            for got, want in ((c.k, codes), (c.v, codes), (c.k_scale, scales), (c.v_scale, scales)):
                assert torch.equal(got[0, page.cuda(), :, (pos % 16).cuda()], want[at: at + new[i]]), (i, r)
        c.advance(cu, n, on)
        m.advance([r for r, _ in first], [x for _, x in first])
        m.check(c)


def test_empty_and_full_batches_and_identity_rows():
    c, m = make(pages=30, rows=4, per=6, heads=1)
    c.start(4)
    m.release(range(4), 0)
    c.reserve(offsets([0, 0, 0, 0]), 4)
    m.check(c)
    c.reserve(offsets([16, 17, 0, 96]), 4)
    m.reserve(range(4), [16, 17, 0, 96])
    m.check(c)
    c.reserve(offsets([16, 17, 0, 97]), 4)       # again: nothing is lacking, and the last row's table is too short
    m.reserve(range(4), [16, 17, 0, 97])
    m.check(c)
    c.compact()
    m.compact()
    m.check(c)


def test_step_recorded_into_a_graph_and_another_stream():
    """reserve, append, advance and fork captured once and replayed: pages are handed out by what the device holds then."""
    from runtherder_b200 import kernels as K
    K.init(0)
    c, m = make(pages=64, ps=16, rows=4, per=8, heads=2, dim=128)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(40, 2, 128, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    cu, new = offsets([9, 11]), [9, 11]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    parents, children = ints([0, 1]), ints([2, 3])
    c.start(2)
    m.release([0, 1], 0)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        c.reserve(cu, 2)
        for layer in range(2):
            c.append(layer, k, v, cu, 20, 2)
        c.advance(cu, 2)
        c.fork(parents, children, 2)
    codes, scales = reference_append(k[:20], 2, 128)
    for step in range(5):
        graph.replay()
        m.reserve([0, 1], new)
        m.advance([0, 1], new)
        m.fork([0, 1], [2, 3])
        torch.cuda.synchronize()
        m.check(c)
        for row, at, n in ((0, 0, 9), (1, 9, 11), (2, 0, 9), (3, 9, 11)):
            for layer in range(2):
                for i in range(n):
                    pos = (step * n) + i
                    page = m.table[row][pos // 16]
                    assert torch.equal(c.k[layer, page, :, pos % 16], codes[at + i])
                    assert torch.equal(c.k_scale[layer, page, :, pos % 16], scales[at + i])


def test_calls_on_the_wrong_device_or_type_are_refused():
    from runtherder_b200._lib import RhError
    c, _ = make()
    k = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    cu = offsets([4])
    for bad in (dict(k=k.float()), dict(k=k.cpu()), dict(k=k[:2]), dict(k=k.transpose(0, 1)), dict(k=torch.zeros(4, 64, 2, dtype=torch.bfloat16, device="cuda").transpose(1, 2)),
                dict(cu=cu.long()), dict(cu=cu[:1]), dict(cu=cu.cpu()), dict(rows=torch.zeros(1, device="cuda"))):
        a = dict(k=k, cu=cu, rows=None)
        a.update(bad)
        with pytest.raises(RhError):
            c.append(0, a["k"], k, a["cu"], 4, 1, a["rows"])
    c.device_index = 1
    with pytest.raises(RhError):
        c.compact()
