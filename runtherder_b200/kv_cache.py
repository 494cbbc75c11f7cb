"""FP8 E4M3 KV caches with per-(token, kv_head) scales: `KVCache`, one sequence, and `PagedKVCache`, a batch of them.

`KVCache` has the slab layout and append rule of runtherder's engine::KVCache
(include/runtherder/engine/kv_cache.h:18-22, 62-89).

K and V slabs are [num_layers, max_seq_len, num_kv_heads, head_dim] E4M3 bytes; the scale slabs
[num_layers, max_seq_len, num_kv_heads] fp32.  The write position is a device-resident int32 so a
captured CUDA graph picks up a new position on every replay; like the reference, the device does
not check it against max_seq_len — `append` callers own that bound (`check_bound` helps).
"""
from __future__ import annotations

import ctypes

import torch

from . import kernels as K
from ._lib import KVPages, RhError, lib


class KVCache:
    def __init__(self, num_layers: int, max_seq_len: int, num_kv_heads: int, head_dim: int, device="cuda"):
        for name, v in (("num_layers", num_layers), ("max_seq_len", max_seq_len), ("num_kv_heads", num_kv_heads),
                        ("head_dim", head_dim)):
            if v < 1:
                raise RhError("KVCache", 1, f"KVCache {name} must be >= 1")
        self.num_layers, self.max_seq_len = num_layers, max_seq_len
        self.num_kv_heads, self.head_dim = num_kv_heads, head_dim
        shape = (num_layers, max_seq_len, num_kv_heads, head_dim)
        self.k = torch.zeros(shape, dtype=torch.uint8, device=device)
        self.v = torch.zeros(shape, dtype=torch.uint8, device=device)
        self.k_scale = torch.zeros(shape[:3], dtype=torch.float32, device=device)
        self.v_scale = torch.zeros(shape[:3], dtype=torch.float32, device=device)

    def _layer(self, layer: int):
        if not 0 <= layer < self.num_layers:
            raise RhError("KVCache", 1, "KVCache layer out of range")
        return self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer]

    def check_bound(self, start_pos: int, n_new: int) -> None:
        """The host-side bound the reference checks in LlamaModel::stage (llama.cu:263-264)."""
        if start_pos < 0 or start_pos + n_new > self.max_seq_len:
            raise RhError("KVCache", 1, f"positions {start_pos}..{start_pos + n_new} exceed max_seq_len "
                                        f"{self.max_seq_len}")

    def append(self, layer: int, k, v, n_new: int, at_pos, stream=None) -> None:
        """Quantise n_new bf16 keys and values into `layer` at row *at_pos (kv_cache.h:62-78):
        two quantize_kv_fp8 calls, exactly as the reference issues them."""
        if n_new < 1:
            raise RhError("KVCache", 1, "KVCache append n_new must be >= 1")
        if at_pos is None:
            raise RhError("KVCache", 1, "KVCache append at_pos must not be null")
        kc, vc, ks, vs = self._layer(layer)
        rows = n_new * self.num_kv_heads
        K.quantize_kv_fp8(kc, ks, k, at_pos, self.num_kv_heads, rows, self.head_dim, stream)
        K.quantize_kv_fp8(vc, vs, v, at_pos, self.num_kv_heads, rows, self.head_dim, stream)

    def rope_append(self, layer: int, q, k, v, positions, inv_freq, n_new: int, at_pos, num_q_heads: int,
                    q_norm=None, k_norm=None, eps: float = 1e-6, k_out=None, stream=None) -> None:
        """Fused path: [QK-norm +] RoPE on q (in place) and k, then the append of rotated k and of v."""
        kc, vc, ks, vs = self._layer(layer)
        K.rope_kv_fp8(q, k_out, k, v, q_norm, k_norm, eps, positions, inv_freq, kc, ks, vc, vs, at_pos, n_new,
                      num_q_heads, self.num_kv_heads, self.head_dim, stream)

    def view(self, layer: int):
        """(k, v, k_scale, v_scale) of one layer — what attention kernels consume (kv_cache.h:80-89)."""
        return self._layer(layer)


class PagedKVCache:
    """A pool of pages shared by `num_rows` sequences, for batched prefill and decode.

    k, v are [layers, pages, kv heads, page size, head dim] E4M3 bytes, the scales [layers, pages, kv heads, page size].
    page_table [rows, pages_per_row] lists a sequence's pages (-1: none), lens [rows] the tokens it holds (-1: idle row),
    ref_counts [pages] the rows that list a page.  All of it is device-resident and changed by kernels only, so a step

        cache.reserve(cu_seqlens, n); per layer: cache.append(...), attention; cache.advance(cu_seqlens, n)

    can be recorded into a CUDA graph.  A batch is named by `cu_seqlens` (offsets of its packed tokens) and `rows` (None:
    entry i is row i).  Calls on one cache from several streams must be ordered by the caller."""

    SLABS = ("k", "v", "k_scale", "v_scale", "page_table", "lens", "ref_counts", "status")

    def __init__(self, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, num_rows: int,
                 pages_per_row: int, device="cuda"):
        for name, v in (("num_layers", num_layers), ("num_pages", num_pages), ("page_size", page_size),
                        ("num_kv_heads", num_kv_heads), ("head_dim", head_dim), ("num_rows", num_rows),
                        ("pages_per_row", pages_per_row)):
            if v < 1:
                raise RhError("PagedKVCache", 1, f"PagedKVCache {name} must be >= 1")
        shape = (num_layers, num_pages, num_kv_heads, page_size, head_dim)
        i32 = dict(dtype=torch.int32, device=device)
        self._adopt(k=torch.zeros(shape, dtype=torch.uint8, device=device), v=torch.zeros(shape, dtype=torch.uint8, device=device),
                    k_scale=torch.zeros(shape[:4], dtype=torch.float32, device=device),
                    v_scale=torch.zeros(shape[:4], dtype=torch.float32, device=device),
                    page_table=torch.full((num_rows, pages_per_row), -1, **i32), lens=torch.full((num_rows,), -1, **i32),
                    ref_counts=torch.zeros(num_pages, **i32), status=torch.zeros(2, **i32))

    @classmethod
    def from_tensors(cls, **slabs) -> "PagedKVCache":
        """A cache over tensors that the caller owns, named and laid out as in the class's description."""
        self = cls.__new__(cls)
        self._adopt(**slabs)
        return self

    def __setattr__(self, name, value) -> None:
        if name in self.SLABS + ("scratch",) and "_struct" in self.__dict__:     # the kernels have the addresses of those it was made of
            raise RhError("PagedKVCache", 1, f"{name} of a cache cannot be replaced: copy into it, or make a cache by from_tensors")
        super().__setattr__(name, value)

    def _adopt(self, **slabs) -> None:
        if set(slabs) != set(self.SLABS):
            raise RhError("PagedKVCache", 1, f"PagedKVCache is made of {', '.join(self.SLABS)}")
        k = slabs["k"]
        if k.dim() != 5 or slabs["page_table"].dim() != 2:
            raise RhError("PagedKVCache", 1, "k must be [layers, pages, kv heads, page size, head dim], page_table [rows, pages_per_row]")
        L, N, H, ps, D = k.shape
        rows, per_row = slabs["page_table"].shape
        want = {"k": ((L, N, H, ps, D), torch.uint8), "v": ((L, N, H, ps, D), torch.uint8),
                "k_scale": ((L, N, H, ps), torch.float32), "v_scale": ((L, N, H, ps), torch.float32),
                "page_table": ((rows, per_row), torch.int32), "lens": ((rows,), torch.int32),
                "ref_counts": ((N,), torch.int32), "status": ((2,), torch.int32)}
        for name, (shape, dtype) in want.items():
            t = slabs[name]
            if tuple(t.shape) != tuple(shape) or not t.is_contiguous() or t.device != k.device or \
                    (t.dtype != dtype and not (dtype == torch.uint8 and t.dtype == torch.float8_e4m3fn)):
                raise RhError("PagedKVCache", 1, f"{name} must be contiguous {tuple(shape)} {dtype} on {k.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
            setattr(self, name, t)
        if ps & (ps - 1) or not 16 <= ps <= 256:
            raise RhError("PagedKVCache", 2, "page_size must be a power of two in 16..256")
        if D not in (64, 128):
            raise RhError("PagedKVCache", 2, "head_dim must be 64 or 128")
        if rows > 1 << 24:
            raise RhError("PagedKVCache", 2, "at most 2^24 rows")
        self.num_layers, self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = L, N, H, ps, D
        self.num_rows, self.pages_per_row = rows, per_row
        self.device_index = k.device.index if k.is_cuda else -1
        self.scratch = torch.empty(int(lib.rh_kv_pages_scratch_ints(rows, N, per_row)), dtype=torch.int32, device=k.device)
        self._struct = KVPages(*(getattr(self, n).data_ptr() for n in self.SLABS), self.scratch.data_ptr(), L, N, ps, H, D, rows, per_row)
        self.desc = ctypes.byref(self._struct)

    # ---- bookkeeping

    def start(self, num_rows: int, rows=None, stream=None) -> None:
        """The rows become new, empty sequences (what they held is released)."""
        K.kv_pages_release(self, num_rows, rows, 0, stream)

    def release(self, num_rows: int, rows=None, stream=None) -> None:
        """The rows become idle; their pages are free once no other row lists them."""
        K.kv_pages_release(self, num_rows, rows, -1, stream)

    def reserve(self, cu_seqlens, num_seqs: int, rows=None, stream=None) -> None:
        K.kv_pages_reserve(self, cu_seqlens, num_seqs, rows, stream)

    def advance(self, cu_seqlens, num_seqs: int, rows=None, stream=None) -> None:
        K.kv_pages_advance(self, cu_seqlens, num_seqs, rows, stream)

    def fork(self, parents, children, count: int, stream=None) -> None:
        K.kv_pages_fork(self, parents, children, count, stream)

    def copy(self, src, dst, count: int, stream=None) -> None:
        K.kv_pages_copy(self, src, dst, count, stream)

    def compact(self, stream=None) -> None:
        K.kv_pages_compact(self, stream)

    # ---- contents

    def append(self, layer: int, k, v, cu_seqlens, num_tokens: int, num_seqs: int, rows=None, stream=None) -> None:
        """Quantises the packed batch's new keys and values into `layer` behind what its rows hold."""
        K.kv_append_paged_fp8(self, layer, k, v, cu_seqlens, num_tokens, num_seqs, rows, stream)

    def gather(self, layer: int, row: int, count: int):
        """Keys and values 0..count-1 of a row as fp32 [kv heads, count, head dim], for tests and inspection; zeros where the row
        has no page."""
        if not (0 <= layer < self.num_layers and 0 <= row < self.num_rows and 0 <= count <= self.pages_per_row * self.page_size):
            raise RhError("PagedKVCache", 1, f"gather of layer {layer}, row {row}, {count} keys: out of range")
        pages = self.page_table[row, : -(-count // self.page_size)].long()
        there = (pages >= 0) & (pages < self.num_pages)
        pages = torch.where(there, pages, torch.zeros_like(pages))
        out = []
        for codes, scale in ((self.k, self.k_scale), (self.v, self.v_scale)):
            x = K.dequantize_kv_fp8(codes[layer, pages].contiguous(), scale[layer, pages])
            x = torch.where(there[:, None, None, None], x, torch.zeros_like(x))
            out.append(x.transpose(0, 1).reshape(self.num_kv_heads, pages.numel() * self.page_size, self.head_dim)[:, :count])
        return tuple(out)
