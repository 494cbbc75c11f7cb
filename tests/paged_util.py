"""A plain host model of the paged cache (page lists, counts, contents) and 64-bit attention over it, for the tests."""
from __future__ import annotations

import math

import numpy as np
import torch


def e4m3_table() -> torch.Tensor:
    """The 256 values of E4M3, from its definition."""
    out = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out.append(math.nan if (c & 127) == 127 else -x if c & 128 else x)
    return torch.tensor(out, dtype=torch.float64)


class Model:
    """The bookkeeping of a paged cache on the host: lowest free pages first, in the order of the call."""

    def __init__(self, num_pages, page_size, num_rows, pages_per_row):
        self.ps, self.per = page_size, pages_per_row
        self.refs = [0] * num_pages
        self.table = [[-1] * pages_per_row for _ in range(num_rows)]
        self.lens = [-1] * num_rows
        self.short = self.refused = 0

    def free_pages(self):
        return [i for i, r in enumerate(self.refs) if r == 0]

    def release(self, rows, new_len=-1):
        for r in rows:
            if not 0 <= r < len(self.table):
                self.refused += 1
                continue
            for p in self.table[r]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[r] = [-1] * self.per
            self.lens[r] = new_len

    def reserve(self, rows, new):
        seen, asked = set(), []
        for r, n in zip(rows, new):
            if not 0 <= r < len(self.table) or r in seen:
                self.refused += 1
                continue
            seen.add(r)
            if self.lens[r] < 0 or n <= 0:
                continue
            need = -(-(self.lens[r] + n) // self.ps)
            self.short += max(0, need - self.per)
            asked += [(r, j) for j in range(-(-self.lens[r] // self.ps), min(need, self.per)) if self.table[r][j] < 0]
        free = self.free_pages()
        for (r, j), p in zip(asked, free):
            self.table[r][j] = p
            self.refs[p] = 1
        self.short += max(0, len(asked) - len(free))

    def advance(self, rows, new):
        for r, n in zip(rows, new):
            if 0 <= r < len(self.table) and self.lens[r] >= 0:
                self.lens[r] += n

    def fork(self, parents, children):
        """Returns the copies (source page, destination page, keys) that the fork makes."""
        seen, todo, moves = set(), [], []
        for p, c in zip(parents, children):
            ok = 0 <= p < len(self.table) and 0 <= c < len(self.table)
            if ok and c not in seen:
                seen.add(c)
                if p != c:
                    n = self.lens[p]
                    full = max(n, 0) // self.ps
                    tail = self.table[p][full] if n > 0 and n % self.ps and full < self.per else -1
                    todo.append([c, n, self.table[p][:full], tail])
            else:
                if ok or (0 <= c < len(self.table) and not 0 <= p < len(self.table)):
                    if 0 <= c < len(self.table):
                        seen.add(c)
                self.refused += 1
        for t in todo:
            for p in t[2]:
                self.refs[p] += 1
        free = self.free_pages()
        fresh = {}
        for t in todo:
            if t[3] >= 0:
                if free:
                    p = free.pop(0)
                    self.refs[p] = 1
                    fresh[t[0]] = p
                    moves.append((t[3], p, t[1] % self.ps))
                else:
                    self.short += 1
        for c, n, pages, tail in todo:
            for p in self.table[c]:
                if p >= 0:
                    self.refs[p] -= 1
            row = pages + ([fresh[c]] if c in fresh else [])
            self.table[c] = row + [-1] * (self.per - len(row))
            self.lens[c] = n if n <= 0 or n % self.ps == 0 or c in fresh else len(pages) * self.ps
        return moves

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        src = [i for i, r in enumerate(self.refs) if r > 0 and i >= used]
        dst = [i for i, r in enumerate(self.refs) if r == 0 and i < used]
        to = dict(zip(src, dst))
        for s, d in to.items():
            self.refs[d], self.refs[s] = self.refs[s], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return list(to.items())

    def check(self, cache):
        assert cache.page_table.tolist() == self.table
        assert cache.ref_counts.tolist() == self.refs
        assert cache.lens.tolist() == self.lens
        assert cache.status.tolist() == [self.short, self.refused]


def offsets(new):
    return torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def row_contents(cache, layer, row, count, values=None):
    """Keys and values 0..count-1 of a row in 64 bits [kv heads, count, D], by the definition of the codes."""
    values = e4m3_table().to(cache.k.device) if values is None else values
    pages = cache.page_table[row, : -(-count // cache.page_size)].long()
    out = []
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = values[codes[layer, pages].view(torch.uint8).long()] * scale[layer, pages].double().unsqueeze(-1)
        out.append(x.permute(1, 0, 2, 3).reshape(cache.num_kv_heads, -1, cache.head_dim)[:, :count])
    return out


def attend(q, k, v, first, scale):
    """Tokens q [n, heads, D] over k, v [kv heads, keys, D] in 64 bits: token i sees the first `first` + i keys; a token
    that sees none is zero."""
    n, hq, dim = q.shape
    kk = k.repeat_interleave(hq // k.shape[0], 0)
    vv = v.repeat_interleave(hq // v.shape[0], 0)
    z = torch.einsum("nhd,hkd->hnk", q.double(), kk) * scale
    seen = torch.arange(kk.shape[1], device=q.device)[None] < (first + torch.arange(n, device=q.device))[:, None]
    z = z.masked_fill(~seen[None], -math.inf)
    m = z.amax(-1, keepdim=True) if kk.shape[1] else torch.zeros(hq, n, 1, dtype=torch.float64, device=q.device)
    e = torch.exp(z - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    e = torch.where(seen[None], e, torch.zeros_like(e))
    total = e.sum(-1, keepdim=True)
    vs = torch.where(seen.any(0)[None, :, None], vv, torch.zeros_like(vv))
    o = torch.einsum("hnk,hkd->hnd", e, vs) / torch.where(total > 0, total, torch.ones_like(total))
    return o.permute(1, 0, 2)


def check_attention(out, q, k, v, first, scale, what="", extra=0.0, small_step=2.0 ** -34, mixed=False, q_step=0.0):
    """Holds tokens `out` [n, heads, D] (bf16) against attend() in 64 bits, within what the arithmetic allows, derived:

      the store            a bf16 rounding                                                    2^-8 |o|
      the weights          one f16 rounding each, on A = sum_j p_j |v_j|                      2^-11 A
      the scores           fp32 sums of exact products: 2^-18 of B = max_j sum_d |q_d k_jd|, and the log2-domain score's own
                           roundings, three of 2^-23 of its size and the V scale's (at most 40); numerator and
                           denominator both carry them                                       2 (2^-18 scale B + 2^-21 (|x| + 40)) A
      small weights        f16 loses what is below 2^-24 in units where the largest is 2^10   n 2^-34 max |v|   (`small_step`: 2^-25
                           where the largest weight may be 1: half a step of 2^-24)
      `extra`              of A, for forms that round once more
      `q_step`             of max |q| sum_d |k_jd|, for a form that rounds q: joins the scores' error
      `mixed`              keys whose V scale rides in the exponent beside keys whose scale is folded into V, times 2^8: the
                           latter's weights are taken relative to a maximum that is up to 2^(lg vs + 8) higher, |v| <= 224:
                           n 2^-25 2^7 max_i p_i max |v_i|
    """
    n, hq, dim = q.shape
    want = attend(q, k, v, first, scale)
    kk, vv = k.repeat_interleave(hq // k.shape[0], 0), v.repeat_interleave(hq // v.shape[0], 0)
    seen = (torch.arange(kk.shape[1], device=q.device)[None] < (first + torch.arange(n, device=q.device))[:, None])[None]
    fk, fv = torch.nan_to_num(kk), torch.nan_to_num(vv)
    z = torch.einsum("nhd,hkd->hnk", q.double(), fk) * scale
    big = torch.where(seen, torch.einsum("nhd,hkd->hnk", q.double().abs(), fk.abs()), torch.zeros_like(z)).amax(-1, keepdim=True) * scale
    top = torch.where(seen, z.abs(), torch.zeros_like(z)).amax(-1, keepdim=True) / math.log(2.0)
    zz = z.masked_fill(~seen, -math.inf)
    m = zz.amax(-1, keepdim=True)
    p = torch.exp(zz - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    a = torch.einsum("hnk,hkd->hnd", p, fv.abs())
    sums = torch.where(seen, fk.abs().sum(-1)[:, None], torch.zeros_like(z)).amax(-1, keepdim=True)
    rounded = q_step * abs(scale) * q.double().abs().amax(-1).t().unsqueeze(-1) * sums
    delta = 2.0 * (2.0 ** -18 * big + rounded + 2.0 ** -21 * (top + 40.0))
    small = kk.shape[1] * small_step * fv.abs().amax((-2, -1), keepdim=True)
    if mixed:
        small = small + kk.shape[1] * 2.0 ** -18 * (p * fv.abs().amax(-1)[:, None]).amax(-1, keepdim=True)
    tol = (2.0 ** -8 * want.abs() + ((2.0 ** -11 + delta + extra) * a + small).permute(1, 0, 2)) + 1e-30
    got = out.double()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), finite), (what, "finite where the exact value is not, or the other way round")
    err = torch.where(finite, (got - want).abs(), torch.zeros_like(tol))
    worst = float((err / tol).nan_to_num().max()) if err.numel() else 0.0
    assert worst <= 1.0, (what, worst)
    return worst
