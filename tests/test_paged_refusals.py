"""Argument checks of the paged-cache entry points.  Every call here must be refused before anything is launched, so
the tests need no GPU: addresses are made up and never touched."""
import ctypes as C

import pytest
import torch

from runtherder_b200 import _lib
from runtherder_b200._lib import KVPages, RhError
from runtherder_b200.kv_cache import PagedKVCache

OK, INVALID, DIM, MISALIGNED = 0, 1, 2, 3
A = 0x10000     # a 16-byte aligned address that nothing dereferences


def pages(**change):
    d = dict(k=A, v=A, k_scale=A, v_scale=A, page_table=A, lens=A, ref_counts=A, status=A, scratch=A, num_layers=2, num_pages=10,
             page_size=16, num_kv_heads=2, head_dim=128, num_rows=4, pages_per_row=3)
    d.update(change)
    return C.byref(KVPages(**d))


def refused(want, fn, *args):
    status = getattr(_lib.lib, fn)(*args)
    assert status == want, (status, _lib.lib.rh_last_error_string())
    assert fn.encode() in _lib.lib.rh_last_error_string()


def append(cache, layer=0, k=A, v=A, ks=256, vs=256, rows=None, cu=A, tokens=4, seqs=2):
    return ("rh_kv_append_paged_fp8", cache, layer, k, v, ks, vs, rows, cu, tokens, seqs, None)


@pytest.mark.parametrize("change,want", [
    (dict(k=None), INVALID), (dict(v_scale=None), INVALID), (dict(page_table=None), INVALID), (dict(lens=None), INVALID),
    (dict(ref_counts=None), INVALID), (dict(status=None), INVALID), (dict(scratch=None), INVALID), (dict(num_layers=0), INVALID),
    (dict(num_pages=0), INVALID), (dict(num_rows=-1), INVALID), (dict(pages_per_row=0), INVALID), (dict(num_kv_heads=0), INVALID),
    (dict(page_size=8), DIM), (dict(page_size=24), DIM), (dict(page_size=512), DIM), (dict(page_size=0), DIM), (dict(head_dim=96), DIM),
    (dict(head_dim=256), DIM), (dict(num_pages=1 << 25), DIM), (dict(num_rows=1 << 20, pages_per_row=1 << 12), DIM),
    (dict(num_pages=1 << 23, num_kv_heads=8, page_size=64), DIM), (dict(k=A + 8), MISALIGNED), (dict(v_scale=A + 4), MISALIGNED),
])
def test_bad_cache_descriptions(change, want):
    c = pages(**change)
    refused(want, *append(c))
    refused(want, "rh_kv_pages_reserve", c, None, A, 1, None)
    refused(want, "rh_kv_pages_release", c, None, 1, -1, None)
    refused(want, "rh_kv_pages_advance", c, None, A, 1, None)
    refused(want, "rh_kv_pages_fork", c, A, A, 1, None)
    refused(want, "rh_kv_pages_copy", c, A, A, 1, None)
    refused(want, "rh_kv_pages_compact", c, None)


def test_bad_call_arguments():
    c = pages()
    for bad in (dict(layer=-1), dict(layer=2), dict(k=None), dict(v=None), dict(cu=None), dict(tokens=0), dict(seqs=0), dict(seqs=5),
                dict(ks=255), dict(vs=128)):
        refused(INVALID, *append(c, **bad))
    for bad in (dict(k=A + 2), dict(v=A + 8), dict(ks=260), dict(vs=257)):
        refused(MISALIGNED, *append(c, **bad))
    refused(INVALID, *append(None))
    refused(INVALID, "rh_kv_pages_compact", None, None)
    refused(INVALID, "rh_kv_pages_reserve", c, None, None, 1, None)
    refused(INVALID, "rh_kv_pages_reserve", c, None, A, 5, None)
    refused(INVALID, "rh_kv_pages_advance", c, None, A, 0, None)
    refused(INVALID, "rh_kv_pages_release", c, None, 5, -1, None)
    refused(INVALID, "rh_kv_pages_release", c, None, 1, 3, None)
    refused(INVALID, "rh_kv_pages_fork", c, None, A, 1, None)
    refused(INVALID, "rh_kv_pages_fork", c, A, A, 5, None)
    refused(INVALID, "rh_kv_pages_copy", c, A, None, 1, None)
    refused(INVALID, "rh_kv_pages_copy", c, A, A, 11, None)


def decode(cache, out=A, q=A, stride=512, layer=0, rows=None, seqs=2, heads=4, partial=A, shared=None, length=None):
    return ("rh_flash_decode_paged_bf16", out, q, stride, cache, layer, rows, seqs, heads, 0.1, partial, shared, length, None)


def prefill(cache, out=A, q=A, stride=512, layer=0, rows=None, cu=A, tokens=4, seqs=2, heads=4, partial=A, splits=2):
    return ("rh_flash_prefill_packed_bf16", out, q, stride, cache, layer, rows, cu, tokens, seqs, heads, 0.1, partial, splits, None)


def test_bad_attention_arguments():
    c = pages()
    for call in (decode, prefill):
        refused(INVALID, *call(None))
        refused(DIM, *call(pages(head_dim=96)))
        refused(INVALID, *call(pages(lens=None)))
        for bad in (dict(out=None), dict(q=None), dict(partial=None), dict(layer=-1), dict(layer=2), dict(seqs=0), dict(seqs=5), dict(heads=0),
                    dict(heads=3), dict(stride=511)):
            refused(INVALID, *call(c, **bad))
        for bad in (dict(q=A + 8), dict(stride=516), dict(partial=A + 8), dict(out=A + 2)):
            refused(MISALIGNED, *call(c, **bad))
        refused(DIM, *call(c, heads=1026, stride=1026 * 128))
    refused(INVALID, *decode(c, shared=A))
    refused(INVALID, *decode(c, length=A))
    refused(INVALID, *decode(c, rows=A, seqs=4097))
    refused(DIM, *decode(pages(page_size=256, num_pages=1 << 20, num_rows=1 << 8, pages_per_row=1 << 20), rows=A, seqs=256))
    refused(MISALIGNED, *decode(c, out=A + 4))
    refused(MISALIGNED, *prefill(c, out=A + 8))
    for bad in (dict(cu=None), dict(tokens=0), dict(splits=0), dict(splits=65)):
        refused(INVALID, *prefill(c, **bad))


def test_attention_scratch_sizes():
    splits, floats = _lib.lib.rh_flash_prefill_packed_splits, _lib.lib.rh_flash_prefill_packed_scratch_floats
    assert floats(100, 8, 128, 1) == 0 and floats(100, 8, 128, 0) == 0 and floats(0, 8, 128, 4) == 0
    assert floats(100, 8, 128, 4) >= 4 * 100 * 8 * 130
    assert floats(1 << 20, 64, 128, 16) > 1 << 32      # counted in 64 bits
    assert splits(0, 1, 1, 8, 8, 128) == 1 and splits(4, 1, 100, 3, 2, 128) == 1


def test_scratch_sizes():
    f = _lib.lib.rh_kv_pages_scratch_ints
    assert f(0, 1, 1) == 0 and f(1, 0, 1) == 0 and f(1, 1, 0) == 0
    assert f(4, 10, 3) >= 3 * 4 + 2 * 10 + 1 + 3 * 10 + 4 * 3
    assert f(1 << 14, 1 << 20, 1 << 14) > 1 << 28      # counted in 64 bits


def slabs(**change):
    L, N, H, ps, D, rows, per = 1, 4, 2, 16, 64, 3, 2
    d = dict(k=torch.zeros(L, N, H, ps, D, dtype=torch.uint8), v=torch.zeros(L, N, H, ps, D, dtype=torch.uint8), k_scale=torch.zeros(L, N, H, ps),
             v_scale=torch.zeros(L, N, H, ps), page_table=torch.zeros(rows, per, dtype=torch.int32), lens=torch.zeros(rows, dtype=torch.int32),
             ref_counts=torch.zeros(N, dtype=torch.int32), status=torch.zeros(2, dtype=torch.int32))
    d.update(change)
    return d


def test_python_class_checks_its_tensors():
    c = PagedKVCache.from_tensors(**slabs())
    assert (c.num_layers, c.num_pages, c.num_kv_heads, c.page_size, c.head_dim, c.num_rows, c.pages_per_row) == (1, 4, 2, 16, 64, 3, 2)
    for bad in (dict(k=torch.zeros(4, 2, 16, 64, dtype=torch.uint8)), dict(v=torch.zeros(1, 4, 2, 16, 32, dtype=torch.uint8)),
                dict(v=torch.zeros(1, 4, 2, 16, 64, dtype=torch.int8)), dict(k_scale=torch.zeros(1, 4, 16, 2)), dict(lens=torch.zeros(4, dtype=torch.int32)),
                dict(lens=torch.zeros(3, dtype=torch.int64)), dict(ref_counts=torch.zeros(5, dtype=torch.int32)), dict(status=torch.zeros(1, dtype=torch.int32)),
                dict(page_table=torch.zeros(2, 3, dtype=torch.int32).t()), dict(v=torch.zeros(1, 4, 2, 64, 16, dtype=torch.uint8).transpose(3, 4))):
        with pytest.raises(RhError):
            PagedKVCache.from_tensors(**slabs(**bad))
    with pytest.raises(RhError):
        PagedKVCache.from_tensors(**{k: v for k, v in slabs().items() if k != "status"})
    for bad in (dict(page_size=24), dict(page_size=8), dict(head_dim=96), dict(num_pages=0), dict(num_rows=0)):
        d = dict(num_layers=1, num_pages=4, page_size=16, num_kv_heads=2, head_dim=64, num_rows=3, pages_per_row=2, device="cpu")
        d.update(bad)
        with pytest.raises(RhError):
            PagedKVCache(**d)


def test_a_cache_in_host_memory_is_refused():
    from runtherder_b200 import kernels as K
    c = PagedKVCache.from_tensors(**slabs())
    k, cu = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: c.start(1), lambda: c.compact(), lambda: c.append(0, k, k, cu, 4, 3), lambda: c.reserve(cu, 3), lambda: c.fork(cu, cu, 2),
                 lambda: K.flash_prefill_packed_bf16(k, k, c, 0, cu, 4, 3, 2, 0.1), lambda: K.flash_decode_paged_bf16(k, k, c, 0, 3, 2, 0.1, k)):
        with pytest.raises(RhError):
            call()
