"""The paged-cache operators in their plain form and as the framework's calls, with the cases they are measured on.

A cache in pages holds the keys and values of a batch of sequences as E4M3 codes with one fp32 scale per token and head:
codes [layers, pages, kv heads, page size, head dim], scales [layers, pages, kv heads, page size].  A row of the page
table lists a sequence's pages (-1: none) and `lens` the tokens it holds (-1: an idle row).  Four operators work on it:

  append   quantises the new keys and values of a packed batch into its rows' pages
  pages    copies listed pages, forks sequences, compacts the pool
  prefill  causal attention of a packed batch's new tokens over what their rows hold and over themselves
  decode   attention of one new token per row; the rows may share a prefix, which is computed once for all of them
"""
import math
import random

import torch

own = False


# ---------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of 32 sequences puts one token each into its row: launch latency
        {"name": "append 32 tokens", "op": "append", "seqs": 32, "tokens": 32, "history": 1000, "kv_heads": 8, "head_dim": 128, "page": 16},
        # the K/V of a packed batch of prompts
        {"name": "append 8192 tokens", "op": "append", "seqs": 9, "tokens": 8192, "history": 0, "kv_heads": 8, "head_dim": 128, "page": 64},
        # a handful of pages moved, all layers: the smallest call
        {"name": "copy 4 pages", "op": "copy", "pages": 4, "pool": 64, "layers": 28, "kv_heads": 8, "head_dim": 128, "page": 16},
        # a beam step: every beam becomes a child of another one
        {"name": "fork 8 beams", "op": "fork", "parents": 4, "children": 8, "length": 1203, "layers": 28, "kv_heads": 8, "head_dim": 128, "page": 16},
        # one prompt sampled 64 times, large pages
        {"name": "fork 64 samples", "op": "fork", "parents": 1, "children": 64, "length": 2039, "layers": 28, "kv_heads": 8, "head_dim": 128, "page": 64},
        # a fragmented pool packed to its front
        {"name": "compact 1500 pages", "op": "compact", "pool": 1500, "rows": 40, "layers": 12, "kv_heads": 8, "head_dim": 128, "page": 16},
        # five short prompts, one of them a single token
        {"name": "prefill 511 tokens", "op": "prefill", "seqs": 5, "tokens": 511, "history": 0, "q_heads": 24, "kv_heads": 8, "head_dim": 128, "page": 16},
        # a full prefill batch of ragged prompts
        {"name": "prefill 8192 tokens", "op": "prefill", "seqs": 6, "tokens": 8192, "history": 0, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64},
        # chunks behind long histories, heads of 64
        {"name": "prefill behind 12000", "op": "prefill", "seqs": 3, "tokens": 700, "history": 12000, "q_heads": 32, "kv_heads": 8, "head_dim": 64, "page": 32},
        # one sequence alone: the latency of a decode step
        {"name": "decode 1 x 8196", "op": "decode", "seqs": 1, "shared": 0, "own": 8196, "q_heads": 24, "kv_heads": 8, "head_dim": 128, "page": 16},
        # a small batch behind a common prompt
        {"name": "decode 12 x (8192 + 600)", "op": "decode", "seqs": 12, "shared": 8192, "own": 600, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16},
        # a large batch behind a long common prompt
        {"name": "decode 128 x (32768 + 900)", "op": "decode", "seqs": 128, "shared": 32768, "own": 900, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: sizes even over the logarithm of their range, cut down where it would cost more than the largest listed one."""
    case = _drawn(rng)
    size = {"append": "tokens", "copy": "pages", "fork": "children", "compact": "pool", "prefill": "tokens", "decode": "shared"}[case["op"]]
    while _cost(case) > 1.0 and case[size] > 1:
        case[size] = case[size] * 2 // 3
        if case["op"] in ("append", "prefill"):
            case["seqs"] = min(case["seqs"], case[size])
    return case


def _cost(case):
    """Of a pass, as a share of the largest listed one: its memory traffic, its products, and the scores that the plain form holds."""
    w = work(case)
    cost = max(w["bytes"] / 4.2e8, w["flops"] / 1.45e11)
    if case["op"] == "prefill":
        new, held = _new_tokens(case), _held(case)
        cost = max(cost, case["seqs"] * case["q_heads"] * max(new) * max(h + n for h, n in zip(held, new)) / 2.5e9)
    return cost


def _drawn(rng):
    op = rng.choice(["append", "copy", "fork", "compact", "prefill", "prefill", "decode", "decode"])
    page = rng.choice([16, 32, 64, 128])
    dim = rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    pool = {"kv_heads": kv, "head_dim": dim, "page": page}
    if op == "append":
        seqs = _spread(rng, 1, 64)
        return {"op": op, "seqs": seqs, "tokens": max(seqs, _spread(rng, 1, 8192)), "history": rng.choice([0, _spread(rng, 1, 2000)]), **pool}
    if op == "copy":
        n = _spread(rng, 1, 96)
        return {"op": op, "pages": n, "pool": 2 * n + rng.randint(1, 40), "layers": rng.randint(1, 28), **pool, "page": min(page, 64)}
    if op == "fork":
        return {"op": op, "parents": rng.randint(1, 8), "children": _spread(rng, 1, 48), "length": _spread(rng, 1, 2500), "layers": rng.randint(1, 20), **pool, "page": min(page, 64)}
    if op == "compact":
        return {"op": op, "pool": _spread(rng, 40, 1200), "rows": rng.randint(1, 60), "layers": rng.randint(1, 10), **pool, "page": min(page, 32)}
    heads = {"q_heads": kv * group, **pool}
    if op == "prefill":
        seqs = _spread(rng, 1, 24)
        tokens = max(seqs, _spread(rng, 1, 6000))
        history = rng.choice([0, 0, _spread(rng, 1, 10000)]) if tokens < 1500 else 0
        return {"op": op, "seqs": seqs, "tokens": tokens, "history": history, **heads}
    seqs = _spread(rng, 1, 128)
    return {"op": op, "seqs": seqs, "shared": rng.choice([0, _spread(rng, 64, 32768)]), "own": _spread(rng, 1, 900 if seqs > 8 else 12000), **heads}


def _rng(case, what):
    return random.Random("%s %s" % (what, sorted((k, v) for k, v in case.items() if k != "name")))


def _new_tokens(case):
    """New tokens of each sequence of a packed batch: ragged, at least one each, the given total."""
    n, total = case["seqs"], case["tokens"]
    rng = _rng(case, "tokens")
    w = [math.exp(rng.uniform(0.0, 3.5)) for _ in range(n)]
    got = [1 + int((total - n) * x / sum(w)) for x in w]
    got[rng.randrange(n)] += total - sum(got)
    return got


def _held(case):
    """Tokens that each sequence of the batch holds before the call."""
    rng = _rng(case, "held")
    if case["op"] == "decode":   # the own part: from a tenth of `own` to all of it; the new token is counted in
        return [case["shared"] + max(1, int(case["own"] * rng.uniform(0.1, 1.0))) - 1 if i else case["shared"] + case["own"] - 1 for i in range(case["seqs"])]
    return [int(case["history"] * rng.uniform(0.3, 1.0)) if i else case["history"] for i in range(case["seqs"])]


def _pages_for(tokens, page):
    return -(-tokens // page)


# ---------------------------------------------------------------------------------------------- inputs

def _gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def _pool(case, layers, pages, gen):
    """A pool as quantising keys and values that are normally distributed leaves it: a row's largest code is 448."""
    kv, dim, ps = case["kv_heads"], case["head_dim"], case["page"]
    out = []
    for _ in range(2):
        codes = torch.empty(layers, pages, kv, ps, dim, dtype=torch.uint8, device="cuda")
        scale = torch.empty(layers, pages, kv, ps, dtype=torch.float32, device="cuda")
        for i in range(layers):
            x = torch.randn(pages, kv, ps, dim, generator=gen, device="cuda")
            s = x.abs().amax(-1) / 448.0
            codes[i] = (x / s.unsqueeze(-1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
            scale[i] = s
        out += [codes, scale]
    return {"k": out[0], "k_scale": out[1], "v": out[2], "v_scale": out[3]}


def _tables(rows, width, pages):
    return {"page_table": torch.full((rows, width), -1, dtype=torch.int32, device="cuda"), "lens": torch.full((rows,), -1, dtype=torch.int32, device="cuda"),
            "ref_counts": torch.zeros(pages, dtype=torch.int32, device="cuda"), "status": torch.zeros(2, dtype=torch.int32, device="cuda")}


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _batch_cache(case, new, held, gen):
    """The pool and tables of a packed batch whose rows hold `held` tokens and have room for `new` more."""
    ps, shared = case["page"], case.get("shared", 0) // case["page"]
    need = [_pages_for(h + n, ps) for h, n in zip(held, new)]
    total = shared + sum(n - shared for n in need) + 3
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)   # pages of a pool in use lie anywhere
    t = _tables(case["seqs"], max(need) + 2, total)
    rows, cols, at = [], [], shared
    source = []
    for r, n in enumerate(need):
        rows += [r] * n
        cols += range(n)
        source += list(range(shared)) + list(range(at, at + n - shared))
        at += n - shared
    t["page_table"][_ints(rows).long(), _ints(cols).long()] = order[_ints(source).long()]
    t["ref_counts"].index_add_(0, order[_ints(source).long()].long(), torch.ones(len(source), dtype=torch.int32, device="cuda"))
    t["lens"].copy_(_ints(held))
    return {**_pool(case, 1, total, gen), **t}


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda").to(torch.bfloat16)


def prepare(case, seed):
    gen = _gen(seed)
    op, dim = case["op"], case["head_dim"]
    st = {"case": case}
    if op in ("append", "prefill"):
        new, held = _new_tokens(case), _held(case)
        st.update(_batch_cache(case, new, held, gen))
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        st["cu_seqlens"] = _ints(cu)
        if op == "append":
            st["new_k"], st["new_v"] = (_randn(gen, cu[-1], case["kv_heads"], dim) for _ in range(2))
        else:
            st["q"] = _randn(gen, cu[-1], case["q_heads"], dim)
            st["out"] = torch.empty_like(st["q"])
            # what the plain form needs to know of the lengths on the host
            st["longest"], st["keys"] = max(new), max(h + n for h, n in zip(held, new))
    elif op == "decode":
        held = _held(case)
        st.update(_batch_cache(case, [1] * case["seqs"], held, gen))
        st["q"] = _randn(gen, case["seqs"], case["q_heads"], dim)
        st["out"] = torch.empty_like(st["q"])
        st["shared_len"] = _ints([case["shared"] // case["page"] * case["page"]])
        st["keys"] = max(held) + 1
    elif op == "copy":
        st.update(_pool(case, case["layers"], case["pool"], gen), **_tables(1, 1, case["pool"]))
        pick = torch.randperm(case["pool"], generator=gen, device="cuda")[: 2 * case["pages"]].to(torch.int32)
        st["src"], st["dst"] = pick[: case["pages"]].contiguous(), pick[case["pages"]:].contiguous()
    elif op == "fork":
        ps, kids = case["page"], case["children"]
        per = _pages_for(case["length"], ps)
        total = case["parents"] * per + 2 * kids + 5
        st.update(_pool(case, case["layers"], total, gen), **_tables(case["parents"] + kids, per + 2, total))
        order = torch.randperm(total, generator=gen, device="cuda")[: case["parents"] * per].to(torch.int32)
        st["page_table"][: case["parents"], :per] = order.view(case["parents"], per)
        st["ref_counts"][order.long()] = 1
        st["lens"][: case["parents"]] = case["length"]
        st["parents"] = torch.randint(case["parents"], (kids,), generator=gen, device="cuda", dtype=torch.int32)
        st["children"] = torch.arange(case["parents"], case["parents"] + kids, dtype=torch.int32, device="cuda")
    else:   # compact: about 60 % of the pool is live, spread over rows of equal length
        live = max(1, int(0.6 * case["pool"]) // case["rows"])
        live, rows = (live, case["rows"]) if live * case["rows"] <= case["pool"] else (1, case["pool"])
        st.update(_pool(case, case["layers"], case["pool"], gen), **_tables(rows, live + 1, case["pool"]))
        order = torch.randperm(case["pool"], generator=gen, device="cuda")[: live * rows].to(torch.int32)
        st["page_table"][:, :live] = order.view(rows, live)
        st["ref_counts"][order.long()] = 1
        st["lens"][:] = live * case["page"]
        st["table_before"], st["refs_before"] = st["page_table"].clone(), st["ref_counts"].clone()
    if own:   # the handle that a program keeps for its cache, and the scratch of the attention calls
        from runtherder_b200 import kernels as K
        from runtherder_b200.kv_cache import PagedKVCache
        st["cache"] = PagedKVCache.from_tensors(**{n: st[n] for n in ("k", "v", "k_scale", "v_scale", "page_table", "lens", "ref_counts", "status")})
        if op == "prefill":
            # a program that builds the batch knows its lengths, and picks the split of the keys by them
            st["splits"] = K.flash_prefill_packed_splits(st["q"].shape[0], case["seqs"], st["keys"], case["q_heads"], case["kv_heads"], dim)
            st["partial"] = torch.empty(K.flash_prefill_packed_scratch_floats(st["q"].shape[0], case["q_heads"], dim, st["splits"]), device="cuda")
        if op == "decode":
            st["partial"] = torch.empty(K.flash_decode_paged_scratch_floats(case["seqs"], case["q_heads"], case["kv_heads"], dim), device="cuda")
    return st


# ---------------------------------------------------------------------------------------------- one pass

def _f8(st):
    """The pool as the values that its codes stand for, with their scales."""
    return st["k"].view(torch.float8_e4m3fn), st["k_scale"], st["v"].view(torch.float8_e4m3fn), st["v_scale"]


def run(st):
    op = st["case"]["op"]
    return _run_own[op](st) if own else _run_plain[op](st)


def _append(st):
    cu = st["cu_seqlens"].long()
    ps, total = st["case"]["page"], st["new_k"].shape[0]
    t = torch.arange(total, device="cuda")
    row = torch.searchsorted(cu, t, right=True) - 1
    pos = st["lens"].long()[row] + t - cu[row]
    page, slot = st["page_table"].long()[row, pos // ps], pos % ps
    for name in ("k", "v"):
        x = st["new_" + name].float()
        amax = x.abs().amax(-1)
        inv = torch.where(amax > 0, 448.0 / amax, torch.zeros_like(amax))
        code = (x * inv.unsqueeze(-1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
        st[name][0][page, :, slot] = code
        st[name + "_scale"][0][page, :, slot] = amax / 448.0
    return _f8(st)


def _append_own(st):
    from runtherder_b200 import kernels as K
    K.kv_append_paged_fp8(st["cache"], 0, st["new_k"], st["new_v"], st["cu_seqlens"], st["new_k"].shape[0], st["case"]["seqs"])
    return _f8(st)


_SLABS = ("k", "v", "k_scale", "v_scale")


def _copy(st):
    src, dst = st["src"].long(), st["dst"].long()
    for n in _SLABS:
        st[n][:, dst] = st[n][:, src]
    return _f8(st)


def _copy_own(st):
    from runtherder_b200 import kernels as K
    K.kv_pages_copy(st["cache"], st["src"], st["dst"], st["case"]["pages"])
    return _f8(st)


def _lowest_free(refs, count):
    """The `count` lowest pages without a reference."""
    return torch.argsort((refs > 0).to(torch.int8), stable=True)[:count]


def _fork(st):
    """children[i] becomes a copy of parents[i]: whole pages are shared, the filled part of the last one is copied."""
    ps, table, refs = st["case"]["page"], st["page_table"], st["ref_counts"]
    parents, children = st["parents"].long(), st["children"].long()
    old, new = table[children].clone(), table[parents].clone()
    lens = st["lens"][parents]
    full, tail = (lens // ps).long(), (lens % ps).long()
    cols = torch.arange(table.shape[1], device="cuda")
    new = torch.where(cols < full.unsqueeze(1), new, torch.full_like(new, -1))
    open_rows = tail > 0
    fresh = _lowest_free(refs, parents.shape[0])[torch.cumsum(open_rows.long(), 0) - 1]     # in the order of the children
    fresh = torch.where(open_rows, fresh, torch.zeros_like(fresh))
    at = full.clamp(max=table.shape[1] - 1).unsqueeze(1)
    new.scatter_(1, at, torch.where(open_rows, fresh, new.gather(1, at).squeeze(1).long()).to(torch.int32).unsqueeze(1))
    count = torch.zeros(refs.shape[0] + 1, dtype=torch.int32, device="cuda")                # the last bin takes the -1 of unused places
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    count.index_add_(0, torch.where(new >= 0, new.long(), refs.shape[0]).flatten(), one.expand(new.numel()))
    count.index_add_(0, torch.where(old >= 0, old.long(), refs.shape[0]).flatten(), -one.expand(old.numel()))
    # the copied rows of a page: those below the fill of its sequence; where nothing is open the page is copied onto itself
    source = torch.where(open_rows, table[parents].gather(1, at).squeeze(1).long(), fresh)
    keep = torch.arange(ps, device="cuda") < tail.unsqueeze(1)
    for n in _SLABS:
        pool = st[n]
        mask = keep[None, :, None, :, None] if pool.dim() == 5 else keep[None, :, None, :]
        put = torch.where(mask, pool[:, source], pool[:, fresh])
        if_open = open_rows.view(1, -1, *([1] * (pool.dim() - 2)))
        pool[:, fresh] = torch.where(if_open, put, pool[:, fresh])
    refs.add_(count[:-1])
    table[children] = new
    st["lens"][children] = lens
    return (*_f8(st), table, refs, st["lens"])


def _fork_own(st):
    from runtherder_b200 import kernels as K
    K.kv_pages_fork(st["cache"], st["parents"], st["children"], st["case"]["children"])
    return (*_f8(st), st["page_table"], st["ref_counts"], st["lens"])


def _restore(st):
    """The tables before the pool was compacted: a pass compacts the same fragmented pool again."""
    st["page_table"].copy_(st["table_before"])
    st["ref_counts"].copy_(st["refs_before"])


def _compact(st):
    """The k-th used page at or above the number of used pages moves to the k-th unused page below it."""
    _restore(st)
    refs, table = st["ref_counts"], st["page_table"]
    used = refs > 0
    live = used.sum()
    ids = torch.arange(refs.shape[0], device="cuda")
    moves, holes = used & (ids >= live), ~used & (ids < live)
    dst_of_rank = torch.argsort((~holes).to(torch.int8), stable=True)
    src_of_rank = torch.argsort((~moves).to(torch.int8), stable=True)
    to = torch.where(moves, dst_of_rank[(torch.cumsum(moves.long(), 0) - 1).clamp(min=0)], ids)
    n_moves = moves.sum()
    # rank k moves src_of_rank[k] -> dst_of_rank[k] for k < n_moves; the rest of the ranks copy a page onto itself
    rank = ids[: (refs.shape[0] + 1) // 2]
    act = rank < n_moves
    src, dst = torch.where(act, src_of_rank[rank], src_of_rank[0]), torch.where(act, dst_of_rank[rank], src_of_rank[0])
    for n in _SLABS:
        st[n][:, dst] = st[n][:, src]
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), table))
    refs.copy_(torch.where(ids < live, torch.where(holes, refs[src_of_rank[(torch.cumsum(holes.long(), 0) - 1).clamp(min=0)]], refs), torch.zeros_like(refs)))
    return (*_f8(st), table, refs)


def _compact_own(st):
    from runtherder_b200 import kernels as K
    _restore(st)
    K.kv_pages_compact(st["cache"])
    return (*_f8(st), st["page_table"], st["ref_counts"])


def _gathered(st, pages):
    """Keys and values of page lists [..., n] as fp32 [..., kv heads, n * page, head dim]."""
    out = []
    for n in ("k", "v"):
        x = st[n][0][pages].view(torch.float8_e4m3fn).float() * st[n + "_scale"][0][pages].unsqueeze(-1)
        x = x.movedim(-4, -3)
        out.append(x.reshape(*x.shape[:-3], -1, x.shape[-1]))
    return out


def _softmax_parts(s, mask):
    """exp(s - max) where the mask holds, the maximum and the sum, of scores s (overwritten)."""
    s.masked_fill_(~mask, -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    e = s.sub_(m).exp_()
    return e, m, e.sum(-1, keepdim=True)


def _prefill(st):
    case, cu, q = st["case"], st["cu_seqlens"].long(), st["q"]
    hq, kv, dim, n, keys = case["q_heads"], case["kv_heads"], case["head_dim"], st["longest"], st["keys"]
    i = torch.arange(n, device="cuda")
    new = cu[1:] - cu[:-1]
    at = (cu[:-1].unsqueeze(1) + i).clamp(max=q.shape[0] - 1)                             # [B, n]
    live = i < new.unsqueeze(1)
    qs = q[at].float().view(-1, n, kv, hq // kv, dim).permute(0, 2, 3, 1, 4)              # [B, kv, group, n, D]
    pages = st["page_table"][:, : _pages_for(keys, case["page"])].long().clamp(min=0)
    k, v = _gathered(st, pages)                                                           # [B, kv, keys, D]
    s = torch.matmul(qs.reshape(qs.shape[0], kv, -1, dim), k.transpose(-1, -2)).view(*qs.shape[:4], -1).mul_(1.0 / math.sqrt(dim))
    j = torch.arange(s.shape[-1], device="cuda")
    mask = (j <= (st["lens"].long().unsqueeze(1) + i).unsqueeze(-1)) & live.unsqueeze(-1)  # [B, n, keys]
    e, _, total = _softmax_parts(s, mask[:, None, None])
    v = torch.where((j < (st["lens"].long() + new).unsqueeze(1))[:, None, :, None], v, torch.zeros_like(v))
    o = torch.matmul(e.view(e.shape[0], kv, -1, e.shape[-1]), v).view(qs.shape) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(-1, n, hq, dim)
    return o[live].to(torch.bfloat16)


def _prefill_own(st):
    from runtherder_b200 import kernels as K
    case = st["case"]
    K.flash_prefill_packed_bf16(st["out"], st["q"], st["cache"], 0, st["cu_seqlens"], st["q"].shape[0], case["seqs"], case["q_heads"],
                                1.0 / math.sqrt(case["head_dim"]), st["partial"], st["splits"])
    return st["out"]


def _decode(st):
    case = st["case"]
    b, hq, kv, dim, ps = case["seqs"], case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    shared = case["shared"] // ps
    q = st["q"].float().view(b, kv, hq // kv, dim)
    k0, v0 = _gathered(st, st["page_table"][0, :shared].long())                           # [kv, shared keys, D]
    k1, v1 = _gathered(st, st["page_table"][:, shared: _pages_for(st["keys"], ps)].long().clamp(min=0))   # [B, kv, own keys, D]
    s0 = torch.matmul(q.transpose(0, 1).reshape(kv, b * hq // kv, dim), k0.transpose(-1, -2)).view(kv, b, hq // kv, shared * ps).transpose(0, 1)
    s1 = torch.matmul(q, k1.transpose(-1, -2))
    j = torch.arange(s0.shape[-1] + s1.shape[-1], device="cuda")
    mask = j <= st["lens"].long().unsqueeze(1)
    e, _, total = _softmax_parts(torch.cat([s0, s1], -1).mul_(1.0 / math.sqrt(dim)), mask[:, None, None])
    v1 = torch.where(mask[:, None, shared * ps:, None], v1, torch.zeros_like(v1))
    o = torch.matmul(e[..., : shared * ps].transpose(0, 1).reshape(kv, b * hq // kv, shared * ps), v0).view(kv, b, hq // kv, dim).transpose(0, 1)
    o = (o + torch.matmul(e[..., shared * ps:], v1)) / total.clamp(min=1e-30)
    return o.reshape(b, hq, dim).to(torch.bfloat16)


def _decode_own(st):
    from runtherder_b200 import kernels as K
    case = st["case"]
    K.flash_decode_paged_bf16(st["out"], st["q"], st["cache"], 0, case["seqs"], case["q_heads"], 1.0 / math.sqrt(case["head_dim"]), st["partial"],
                              st["page_table"], st["shared_len"])
    return st["out"]


_run_plain = {"append": _append, "copy": _copy, "fork": _fork, "compact": _compact, "prefill": _prefill, "decode": _decode}
_run_own = {"append": _append_own, "copy": _copy_own, "fork": _fork_own, "compact": _compact_own, "prefill": _prefill_own, "decode": _decode_own}


# ---------------------------------------------------------------------------------------------- the work that a pass cannot do without

def work(case):
    op, kv, dim, ps = case["op"], case["kv_heads"], case["head_dim"], case["page"]
    row = kv * (dim + 4)                           # one token's codes and scales, keys or values, one layer
    if op == "append":
        return {"bytes": 2 * case["tokens"] * (kv * dim * 2 + row) + 4 * (2 * case["seqs"] + 1), "flops": 4 * case["tokens"] * kv * dim}
    if op == "copy":
        return {"bytes": 2 * 2 * case["layers"] * case["pages"] * ps * row, "flops": 0}
    if op == "fork":
        tail, full = case["length"] % ps, case["length"] // ps
        return {"bytes": 2 * 2 * case["layers"] * case["children"] * tail * row + 4 * case["children"] * (4 * full + 6), "flops": 0}
    if op == "compact":
        live = max(1, int(0.6 * case["pool"]) // case["rows"])
        used = live * case["rows"] if live * case["rows"] <= case["pool"] else case["pool"]
        moved = used * (case["pool"] - used) / case["pool"]      # of the used pages, those above their number
        return {"bytes": 2 * 2 * case["layers"] * moved * ps * row + 8 * (case["pool"] + used), "flops": 0}
    hq = case["q_heads"]
    if op == "prefill":
        pairs, keys = 0, 0
        for n, h in zip(_new_tokens(case), _held(case)):
            pairs += n * h + n * (n + 1) // 2
            keys += h + n
        return {"bytes": 4 * case["tokens"] * hq * dim + 2 * keys * row, "flops": 4 * dim * hq * pairs}
    shared = case["shared"] // ps * ps
    own_keys = sum(h + 1 - shared for h in _held(case))
    return {"bytes": 4 * case["seqs"] * hq * dim + 2 * (shared + own_keys) * row, "flops": 4 * dim * hq * (shared * case["seqs"] + own_keys)}


# ---------------------------------------------------------------------------------------------- the definition in 64 bits

def _e4m3_values():
    """The 256 values of E4M3 by its definition: sign, four bits of exponent with bias 7, three of mantissa; 0x7f and 0xff are no numbers."""
    out = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out.append(math.nan if (c & 127) == 127 else -x if c & 128 else x)
    return torch.tensor(out, dtype=torch.float64, device="cuda")


def _keys_of(st, name, row, count, values):
    """Keys or values 0..count-1 of a table row, [kv heads, count, D] in 64 bits."""
    ps = st["case"]["page"]
    pages = st["page_table"][row, : _pages_for(count, ps)].long()
    x = values[st[name][0, pages].long()] * st[name + "_scale"][0, pages].double().unsqueeze(-1)
    return x.permute(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[3])[:, :count]


def _attend(q, k, v, first, scale):
    """Tokens q [n, heads, D] over keys k [kv, keys, D]: token i sees the first `first` + i keys."""
    n, hq, dim = q.shape
    out = torch.empty(n, hq, dim, dtype=torch.float64, device="cuda")
    j = torch.arange(k.shape[1], device="cuda")
    for h in range(hq):
        kk, vv = k[h * k.shape[0] // hq], v[h * k.shape[0] // hq]
        for a in range(0, n, 2048):
            z = q[a: a + 2048, h].double() @ kk.T * scale
            z[j.unsqueeze(0) >= first + torch.arange(a, a + z.shape[0], device="cuda").unsqueeze(1)] = -math.inf
            out[a: a + 2048, h] = torch.softmax(z, -1) @ vv
    return out


def exact(case, seed):
    global own
    keep, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = keep
    op, values = case["op"], _e4m3_values()
    if op in ("copy", "fork", "compact"):
        return None                                  # nothing is computed: values move, and counts are whole numbers
    if op == "append":
        cu, held, table, ps = st["cu_seqlens"].tolist(), st["lens"].tolist(), st["page_table"].tolist(), case["page"]
        page, slot = [], []
        for r in range(case["seqs"]):
            for p in range(held[r], held[r] + cu[r + 1] - cu[r]):
                page.append(table[r][p // ps])
                slot.append(p % ps)
        page, slot = torch.tensor(page, device="cuda"), torch.tensor(slot, device="cuda")
        positive = values[:127]
        result = []
        for name in ("k", "v"):
            code = values[st[name][0].long()]
            scale = st[name + "_scale"][0].double()
            x = st["new_" + name].double()
            s = x.abs().amax(-1) / 448.0
            y = (x.abs() / s.unsqueeze(-1)).clamp(max=448.0)
            up = torch.searchsorted(positive, y.contiguous()).clamp(max=126)
            low = (up - 1).clamp(min=0)
            nearer = (positive[up] - y < y - positive[low]) | ((positive[up] - y == y - positive[low]) & (up % 2 == 0))
            code[page, :, slot] = torch.where(nearer, positive[up], positive[low]) * torch.sign(x)
            scale[page, :, slot] = s
            result += [code.unsqueeze(0), scale.unsqueeze(0)]
        return tuple(result)
    scale = 1.0 / math.sqrt(case["head_dim"])
    if op == "prefill":
        cu, held = st["cu_seqlens"].tolist(), st["lens"].tolist()
        parts = []
        for r in range(case["seqs"]):
            n = cu[r + 1] - cu[r]
            k, v = (_keys_of(st, x, r, held[r] + n, values) for x in ("k", "v"))
            parts.append(_attend(st["q"][cu[r]: cu[r + 1]], k, v, held[r] + 1, scale))
        return torch.cat(parts)
    if sum(h + 1 for h in _held(case)) * case["kv_heads"] > 64_000_000:
        return None
    parts = []
    for r, h in enumerate(st["lens"].tolist()):
        k, v = (_keys_of(st, x, r, h + 1, values) for x in ("k", "v"))
        parts.append(_attend(st["q"][r: r + 1], k, v, h + 1, scale))
    return torch.cat(parts)
