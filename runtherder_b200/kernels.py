"""Python mirror of runtherder's kernel API (namespace runtherder::kernels).

Function names, argument order and argument meaning follow the reference headers
include/runtherder/kernels/{rmsnorm,quantization,rope,activation,embedding}.cuh; the
fused entry points at the bottom are additions.  Tensors are torch CUDA tensors (or raw
device addresses as int); every call only enqueues work on `stream` (default: torch's
current stream) and raises RhError where the reference would print and exit.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from ._lib import RhError, call

TensorOrPtr = Union[torch.Tensor, int, None]

__all__ = [
    "RhError", "rmsnorm_bf16_forward", "rmsnorm_add_bf16_forward", "quantize_per_token_int8",
    "dequantize_w8a8", "quantize_kv_fp8", "dequantize_kv_fp8", "swiglu_bf16_forward", "rope_bf16",
    "embedding_lookup_bf16_forward", "qkv_bias_add_bf16_forward", "stage_positions", "decode_advance",
    "flash_split_scratch_floats", "flash_decode_split_bf16", "flash_prefill_bf16", "tune", "bias_rope_kv_fp8", "rmsnorm_add_quant_int8", "swiglu_quant_int8", "rope_kv_fp8",
    "rmsnorm_add_last_row", "init", "kv_append_paged_fp8", "kv_pages_reserve", "kv_pages_release", "kv_pages_advance",
    "kv_pages_fork", "kv_pages_copy", "kv_pages_compact", "flash_decode_paged_bf16", "flash_decode_paged_scratch_floats",
    "flash_prefill_packed_bf16", "flash_prefill_packed_splits", "flash_prefill_packed_scratch_floats",
]


def _ptr(t: TensorOrPtr, dtype: Optional[torch.dtype] = None, numel: Optional[int] = None, name: str = "tensor"):
    """Device address of `t`, after the host-side checks a C++ caller gets from the type system."""
    if t is None:
        return None
    if isinstance(t, int):
        return t
    if not t.is_cuda:
        raise RhError(name, 1, f"{name} must be a CUDA tensor")
    if not t.is_contiguous():
        raise RhError(name, 1, f"{name} must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise RhError(name, 1, f"{name} must have dtype {dtype}, got {t.dtype}")
    if numel is not None and t.numel() < numel:
        raise RhError(name, 1, f"{name} holds {t.numel()} elements, {numel} needed")
    return t.data_ptr()


def _stream(stream) -> Optional[int]:
    if stream is None:     # the current stream's handle without the Stream object around it: a launch is a few microseconds
        return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice()) or None
    if isinstance(stream, torch.cuda.Stream):
        return stream.cuda_stream or None
    return int(stream) or None


_BF, _I8, _I32, _F32, _U8 = torch.bfloat16, torch.int8, torch.int32, torch.float32, torch.uint8
_FP8 = (torch.uint8, torch.float8_e4m3fn)


def _fp8_ptr(t, numel, name):
    if isinstance(t, torch.Tensor) and t.dtype not in _FP8:
        raise RhError(name, 1, f"{name} must be uint8 or float8_e4m3fn, got {t.dtype}")
    return _ptr(t, None, numel, name)


def tune(key: str, value: int) -> None:
    """Set a process-wide tuning knob of the library (`rh_tune`); value <= 0 restores the default."""
    call("rh_tune", key.encode(), int(value))


def rmsnorm_bf16_forward(y, x, g, num_tokens: int, hidden_dim: int, eps: float, stream=None) -> None:
    """y = (x / rms(x)) * g; y may alias x.  (rmsnorm.cuh:15-22)"""
    n = num_tokens * hidden_dim
    call("rh_rmsnorm_bf16", _ptr(y, _BF, n, "y"), _ptr(x, _BF, n, "x"), _ptr(g, _BF, hidden_dim, "g"),
         num_tokens, hidden_dim, eps, _stream(stream))


def rmsnorm_add_bf16_forward(y, h_out, x, residual, g, num_tokens: int, hidden_dim: int, eps: float,
                             stream=None) -> None:
    """h_out = x + residual, y = rmsnorm(h_out) * g; h_out may alias residual.  (rmsnorm.cuh:36-45)"""
    n = num_tokens * hidden_dim
    call("rh_rmsnorm_add_bf16", _ptr(y, _BF, n, "y"), _ptr(h_out, _BF, n, "h_out"), _ptr(x, _BF, n, "x"),
         _ptr(residual, _BF, n, "residual"), _ptr(g, _BF, hidden_dim, "g"), num_tokens, hidden_dim, eps,
         _stream(stream))


def rmsnorm_add_last_row(y_last, x, residual, g, num_tokens: int, hidden_dim: int, eps: float, stream=None) -> None:
    """y_last[hidden_dim] = row num_tokens-1 of rmsnorm(x + residual) * g: the final norm when only the last
    token feeds lm_head (llama3.cu:254-263 normalises every row and slices)."""
    n = num_tokens * hidden_dim
    call("rh_rmsnorm_add_last_row_bf16", _ptr(y_last, _BF, hidden_dim, "y_last"), _ptr(x, _BF, n, "x"),
         _ptr(residual, _BF, n, "residual"), _ptr(g, _BF, hidden_dim, "g"), num_tokens, hidden_dim, eps, _stream(stream))


def device_error() -> int:
    """rh_device_error: the sticky per-device word a bounded wait records into when it gives up
    ((source line << 8) | 1; 0 = no kernel has given up so far).  Synchronises the device."""
    import ctypes
    word = ctypes.c_int(-1)
    call("rh_device_error", ctypes.byref(word))
    return int(word.value)


def init(device: int = 0) -> None:
    """rh_init: makes every kernel of the library resident and set up on `device`, so that even the first
    call of an entry point may be recorded into a CUDA graph."""
    call("rh_init", int(device))


def quantize_per_token_int8(q, x_scale, x, num_tokens: int, dim: int, stream=None) -> None:
    """q = round(x / x_scale), x_scale = row amax / 127.  (quantization.cuh:17-22)"""
    n = num_tokens * dim
    call("rh_quantize_per_token_int8", _ptr(q, _I8, n, "q"), _ptr(x_scale, _F32, num_tokens, "x_scale"),
         _ptr(x, _BF, n, "x"), num_tokens, dim, _stream(stream))


def dequantize_w8a8(y, acc, x_scale, w_scale, m: int, n: int, stream=None) -> None:
    """y = acc * x_scale[row] * w_scale[col].  (quantization.cuh:31-37)"""
    call("rh_dequantize_w8a8", _ptr(y, _BF, m * n, "y"), _ptr(acc, _I32, m * n, "acc"),
         _ptr(x_scale, _F32, m, "x_scale"), _ptr(w_scale, _BF, n, "w_scale"), m, n, _stream(stream))


def quantize_kv_fp8(q, scale, x, at_pos, rows_per_pos: int, num_rows: int, head_dim: int, stream=None) -> None:
    """E4M3 rows with scale = amax/448, written from row at_pos*rows_per_pos on; at_pos is a
    device-resident int32.  (quantization.cuh:50-57)"""
    call("rh_quantize_kv_fp8", _fp8_ptr(q, None, "q"), _ptr(scale, _F32, None, "scale"),
         _ptr(x, _BF, num_rows * head_dim, "x"), _ptr(at_pos, _I32, 1, "at_pos"), rows_per_pos, num_rows,
         head_dim, _stream(stream))


def dequantize_kv_fp8(q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """float(q) * scale, the read side of the KV cache (quantization.cuh:63-66).  q: [..., D] E4M3
    bytes, scale: [...] fp32.  Convenience for tests and cache consumers written in torch."""
    return q.view(torch.float8_e4m3fn).to(torch.float32) * scale.unsqueeze(-1)


def swiglu_bf16_forward(y, gate, up, n: int, stream=None) -> None:
    """y[i] = silu(gate[i]) * up[i]; y may alias gate or up.  (activation.cuh:16-21)"""
    call("rh_swiglu_bf16", _ptr(y, _BF, n, "y"), _ptr(gate, _BF, n, "gate"), _ptr(up, _BF, n, "up"), n,
         _stream(stream))


def rope_bf16(q, k, positions, inv_freq, seq_len: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
              stream=None) -> None:
    """In-place RoPE on q [T,Hq,D] and k [T,Hkv,D]; token t rotates by positions[t].  (rope.cuh:16-25)"""
    call("rh_rope_bf16", _ptr(q, _BF, seq_len * num_q_heads * head_dim, "q"),
         _ptr(k, _BF, seq_len * num_kv_heads * head_dim, "k"), _ptr(positions, _I32, seq_len, "positions"),
         _ptr(inv_freq, _F32, head_dim // 2, "inv_freq"), seq_len, num_q_heads, num_kv_heads, head_dim,
         _stream(stream))


def embedding_lookup_bf16_forward(out, embedding_table, token_ids, num_tokens: int, hidden_dim: int,
                                  stream=None) -> None:
    """out[i] = embedding_table[token_ids[i]].  (embedding.cuh:14-20)"""
    call("rh_embedding_lookup_bf16", _ptr(out, _BF, num_tokens * hidden_dim, "out"),
         _ptr(embedding_table, _BF, hidden_dim, "embedding_table"), _ptr(token_ids, _I32, num_tokens, "token_ids"),
         num_tokens, hidden_dim, _stream(stream))


def qkv_bias_add_bf16_forward(q, k, v, q_bias, k_bias, v_bias, n: int, q_dim: int, kv_dim: int, stream=None) -> None:
    """q[r] += q_bias, k[r] += k_bias, v[r] += v_bias for every row, in place.  (bias.cuh:20-30)"""
    call("rh_qkv_bias_add_bf16", _ptr(q, _BF, n * q_dim, "q"), _ptr(k, _BF, n * kv_dim, "k"), _ptr(v, _BF, n * kv_dim, "v"),
         _ptr(q_bias, _BF, q_dim, "q_bias"), _ptr(k_bias, _BF, kv_dim, "k_bias"), _ptr(v_bias, _BF, kv_dim, "v_bias"),
         n, q_dim, kv_dim, _stream(stream))


def stage_positions(positions, decode_pos, start_pos: int, n: int, stream=None) -> None:
    """positions[:n] = start_pos + arange(n), decode_pos[0] = start_pos, on the device (llama.cu:266-274)."""
    call("rh_stage_positions", _ptr(positions, _I32, n, "positions"), _ptr(decode_pos, _I32, 1, "decode_pos"), start_pos, n,
         _stream(stream))


def decode_advance(token_slot, position, decode_pos, next_token, step: int = 1, stream=None) -> None:
    """token_slot[0] = next_token[0]; position[0] += step; decode_pos[0] += step — graph-capturable step update."""
    call("rh_decode_advance", _ptr(token_slot, _I32, 1, "token_slot"), _ptr(position, _I32, 1, "position"),
         _ptr(decode_pos, _I32, 1, "decode_pos"), _ptr(next_token, _I32, 1, "next_token"), step, _stream(stream))


def flash_split_scratch_floats(num_q_heads: int, head_dim: int, max_splits: int) -> int:
    """Floats of scratch a split decode needs (flash_decode.cuh:11-25)."""
    from ._lib import lib
    return int(lib.rh_flash_split_scratch_floats(num_q_heads, head_dim, max_splits))


def flash_decode_split_bf16(out, q, k, v, k_scale, v_scale, partial, num_splits: int, cache_len, num_q_heads: int,
                            num_kv_heads: int, head_dim: int, scale: float, stream=None) -> None:
    """One query token attends keys 0..*cache_len of the FP8 cache; cache_len is a device-resident int32,
    partial caller-owned fp32 scratch of flash_split_scratch_floats(...) floats.  (flash_decode.cuh:27-62)"""
    need = flash_split_scratch_floats(num_q_heads, head_dim, num_splits)
    call("rh_flash_decode_split_bf16", _ptr(out, _BF, num_q_heads * head_dim, "out"),
         _ptr(q, _BF, num_q_heads * head_dim, "q"), _fp8_ptr(k, None, "k"), _fp8_ptr(v, None, "v"),
         _ptr(k_scale, _F32, None, "k_scale"), _ptr(v_scale, _F32, None, "v_scale"),
         _ptr(partial, _F32, need, "partial"), num_splits, _ptr(cache_len, _I32, 1, "cache_len"), num_q_heads,
         num_kv_heads, head_dim, float(scale), _stream(stream))


def flash_prefill_bf16(out, q, k, v, k_scale, v_scale, n_new: int, cache_len, num_q_heads: int, num_kv_heads: int,
                       head_dim: int, scale: float, stream=None) -> None:
    """n_new query tokens attend causally over the FP8 cache (token t sees keys 0..*cache_len + t); cache_len is
    a device-resident int32.  head_dim 128.  (flash_prefill.cuh:27-40)"""
    call("rh_flash_prefill_bf16", _ptr(out, _BF, n_new * num_q_heads * head_dim, "out"),
         _ptr(q, _BF, n_new * num_q_heads * head_dim, "q"), _fp8_ptr(k, None, "k"), _fp8_ptr(v, None, "v"),
         _ptr(k_scale, _F32, None, "k_scale"), _ptr(v_scale, _F32, None, "v_scale"), n_new,
         _ptr(cache_len, _I32, 1, "cache_len"), num_q_heads, num_kv_heads, head_dim, float(scale), _stream(stream))


# ---- fused entry points ---------------------------------------------------------------------

def rmsnorm_add_quant_int8(q, x_scale, h_out, y, x, residual, g, num_tokens: int, hidden_dim: int, eps: float,
                           stream=None) -> None:
    """[residual add +] RMSNorm + per-token INT8 in one pass; equals rmsnorm(_add)_bf16_forward followed
    by quantize_per_token_int8 of the stored result.  residual=None: plain norm; y=None: no bf16 store."""
    n = num_tokens * hidden_dim
    call("rh_rmsnorm_add_quant_int8", _ptr(q, _I8, n, "q"), _ptr(x_scale, _F32, num_tokens, "x_scale"),
         _ptr(h_out, _BF, n, "h_out"), _ptr(y, _BF, n, "y"), _ptr(x, _BF, n, "x"),
         _ptr(residual, _BF, n, "residual"), _ptr(g, _BF, hidden_dim, "g"), num_tokens, hidden_dim, eps,
         _stream(stream))


def swiglu_quant_int8(q, x_scale, y, gate, up, num_tokens: int, inter_dim: int, stream=None) -> None:
    """SwiGLU + per-token INT8 of the bf16-rounded product; y=None skips the bf16 store."""
    n = num_tokens * inter_dim
    call("rh_swiglu_quant_int8", _ptr(q, _I8, n, "q"), _ptr(x_scale, _F32, num_tokens, "x_scale"),
         _ptr(y, _BF, n, "y"), _ptr(gate, _BF, n, "gate"), _ptr(up, _BF, n, "up"), num_tokens, inter_dim,
         _stream(stream))


def rope_kv_fp8(q, k_out, k_in, v_in, q_norm, k_norm, eps: float, positions, inv_freq, k_cache, k_scale,
                v_cache, v_scale, at_pos, seq_len: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                stream=None) -> None:
    """[per-head RMSNorm of q,k +] RoPE + FP8 KV-cache append of rotated k and of v at slot *at_pos."""
    nq, nk = seq_len * num_q_heads * head_dim, seq_len * num_kv_heads * head_dim
    call("rh_rope_kv_fp8", _ptr(q, _BF, nq, "q"), _ptr(k_out, _BF, nk, "k_out"), _ptr(k_in, _BF, nk, "k_in"),
         _ptr(v_in, _BF, nk, "v_in"), _ptr(q_norm, _BF, head_dim, "q_norm"), _ptr(k_norm, _BF, head_dim, "k_norm"),
         eps, _ptr(positions, _I32, seq_len, "positions"), _ptr(inv_freq, _F32, head_dim // 2, "inv_freq"),
         _fp8_ptr(k_cache, None, "k_cache"), _ptr(k_scale, _F32, None, "k_scale"),
         _fp8_ptr(v_cache, None, "v_cache"), _ptr(v_scale, _F32, None, "v_scale"), _ptr(at_pos, _I32, 1, "at_pos"),
         seq_len, num_q_heads, num_kv_heads, head_dim, _stream(stream))


def bias_rope_kv_fp8(q, k_out, k_in, v_in, q_bias, k_bias, v_bias, positions, inv_freq, k_cache, k_scale, v_cache,
                     v_scale, at_pos, seq_len: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                     stream=None) -> None:
    """Qwen2: projection biases + RoPE + FP8 KV-cache append in one launch; equals qkv_bias_add_bf16_forward
    followed by rope_kv_fp8 (v_in is left unmodified)."""
    nq, nk = seq_len * num_q_heads * head_dim, seq_len * num_kv_heads * head_dim
    call("rh_bias_rope_kv_fp8", _ptr(q, _BF, nq, "q"), _ptr(k_out, _BF, nk, "k_out"), _ptr(k_in, _BF, nk, "k_in"),
         _ptr(v_in, _BF, nk, "v_in"), _ptr(q_bias, _BF, num_q_heads * head_dim, "q_bias"),
         _ptr(k_bias, _BF, num_kv_heads * head_dim, "k_bias"), _ptr(v_bias, _BF, num_kv_heads * head_dim, "v_bias"),
         _ptr(positions, _I32, seq_len, "positions"), _ptr(inv_freq, _F32, head_dim // 2, "inv_freq"),
         _fp8_ptr(k_cache, None, "k_cache"), _ptr(k_scale, _F32, None, "k_scale"),
         _fp8_ptr(v_cache, None, "v_cache"), _ptr(v_scale, _F32, None, "v_scale"), _ptr(at_pos, _I32, 1, "at_pos"),
         seq_len, num_q_heads, num_kv_heads, head_dim, _stream(stream))


# ---- a batch of sequences in a paged cache (runtherder_b200.kv_cache.PagedKVCache) -----------------

def _cptr(cache, t, dtype, numel: Optional[int], name: str):
    """_ptr for an argument of a call on `cache`: it must lie on the cache's device."""
    if t is not None and not isinstance(t, int) and t.get_device() != cache.device_index:
        raise RhError(name, 1, f"{name} must be on cuda:{cache.device_index}, where the cache is, got {t.device}")
    return _ptr(t, dtype, numel, name)


def _token_rows(cache, t, num_tokens: int, heads: int, head_dim: int, name: str):
    """Address and token stride of [num_tokens, heads, head_dim] bf16 whose tokens may lie apart (a slice of a
    fused projection); within a token the values are contiguous."""
    if isinstance(t, int):
        return t, heads * head_dim
    if t.get_device() != cache.device_index:
        raise RhError(name, 1, f"{name} must be on cuda:{cache.device_index}, where the cache is, got {t.device}")
    if t.dtype != _BF:
        raise RhError(name, 1, f"{name} must have dtype {_BF}, got {t.dtype}")
    width = heads * head_dim
    if t.is_contiguous():
        if t.numel() < num_tokens * width:
            raise RhError(name, 1, f"{name} holds {t.numel()} elements, {num_tokens * width} needed")
        if num_tokens > 1 and t.dim() == 3 and t.shape[0] >= num_tokens and t.shape[2] == head_dim and t.shape[1] != heads:
            raise RhError(name, 1, f"{name} has {t.shape[1]} heads per token, {heads} expected: pass the slice of them")
        return t.data_ptr(), width
    inside = (head_dim, 1) if t.dim() == 3 else (1,)
    if t.dim() not in (2, 3) or t.shape[0] < num_tokens or t.stride()[1:] != inside or t.shape[1:].numel() != width or \
            (t.dim() == 3 and t.shape[2] != head_dim):
        raise RhError(name, 1, f"{name} must be [tokens, heads, head_dim] with contiguous tokens, got {tuple(t.shape)} with strides {t.stride()}")
    return t.data_ptr(), t.stride(0)


def _on_device(cache, fn: str) -> None:
    if cache.device_index < 0:
        raise RhError(fn, 1, "the cache is not on a CUDA device")
    if cache.device_index != torch._C._cuda_getDevice():
        raise RhError(fn, 1, f"the cache is on device {cache.device_index}, the current device is {torch.cuda.current_device()}")


def _paged_call(cache, stream, fn: str, *args) -> None:
    """An entry point whose first argument is a paged cache, on the cache's device."""
    _on_device(cache, fn)
    call(fn, cache.desc, *args, _stream(stream))


def kv_append_paged_fp8(cache, layer: int, k, v, cu_seqlens, num_tokens: int, num_seqs: int, rows=None, stream=None) -> None:
    """Quantises the packed batch's new keys and values [num_tokens, Hkv, D] into its rows' pages, at positions lens[row]
    and on.  Tokens at or behind cu_seqlens[num_seqs] are padding."""
    kp, ks = _token_rows(cache, k, num_tokens, cache.num_kv_heads, cache.head_dim, "k")
    vp, vs = _token_rows(cache, v, num_tokens, cache.num_kv_heads, cache.head_dim, "v")
    _paged_call(cache, stream, "rh_kv_append_paged_fp8", layer, kp, vp, ks, vs, _cptr(cache, rows, _I32, num_seqs, "rows"),
                _cptr(cache, cu_seqlens, _I32, num_seqs + 1, "cu_seqlens"), num_tokens, num_seqs)


def kv_pages_reserve(cache, cu_seqlens, num_seqs: int, rows=None, stream=None) -> None:
    """Gives the batch's active rows the pages that their new tokens need: the lowest free ones, in the order of the batch."""
    _paged_call(cache, stream, "rh_kv_pages_reserve", _cptr(cache, rows, _I32, num_seqs, "rows"), _cptr(cache, cu_seqlens, _I32, num_seqs + 1, "cu_seqlens"),
                num_seqs)


def kv_pages_release(cache, num_rows: int, rows=None, new_len: int = -1, stream=None) -> None:
    """Drops the rows' pages; new_len 0 starts an empty sequence, -1 leaves the row idle."""
    _paged_call(cache, stream, "rh_kv_pages_release", _cptr(cache, rows, _I32, num_rows, "rows"), num_rows, new_len)


def kv_pages_advance(cache, cu_seqlens, num_seqs: int, rows=None, stream=None) -> None:
    """lens[row] += the batch's new tokens, at the end of a step; a row stops at its first place without a page."""
    _paged_call(cache, stream, "rh_kv_pages_advance", _cptr(cache, rows, _I32, num_seqs, "rows"), _cptr(cache, cu_seqlens, _I32, num_seqs + 1, "cu_seqlens"),
                num_seqs)


def kv_pages_fork(cache, parents, children, count: int, stream=None) -> None:
    """Row children[i] becomes a copy of row parents[i]: whole pages are shared, the filled part of the last one is copied."""
    _paged_call(cache, stream, "rh_kv_pages_fork", _cptr(cache, parents, _I32, count, "parents"), _cptr(cache, children, _I32, count, "children"), count)


def kv_pages_copy(cache, src, dst, count: int, stream=None) -> None:
    """Page dst[i] := page src[i] in every layer; the tables are left alone."""
    _paged_call(cache, stream, "rh_kv_pages_copy", _cptr(cache, src, _I32, count, "src"), _cptr(cache, dst, _I32, count, "dst"), count)


def kv_pages_compact(cache, stream=None) -> None:
    """Packs the used pages to the front of the pool; the page table and the reference counts follow."""
    _paged_call(cache, stream, "rh_kv_pages_compact")


def flash_decode_paged_scratch_floats(num_seqs: int, num_q_heads: int, num_kv_heads: int, head_dim: int) -> int:
    """Floats of scratch that flash_decode_paged_bf16 needs on the current device."""
    from ._lib import lib
    return int(lib.rh_flash_decode_paged_scratch_floats(num_seqs, num_q_heads, num_kv_heads, head_dim))


def flash_decode_paged_bf16(out, q, cache, layer: int, num_seqs: int, num_q_heads: int, scale: float, partial, shared_pages=None,
                            shared_len=None, rows=None, stream=None) -> None:
    """One new token per entry attends keys 0..lens[row] of its row.  shared_pages / shared_len: the first *shared_len keys of
    every entry lie in these pages (a page-table row: pages_per_row entries) and are read once for all of them."""
    fn, D = "rh_flash_decode_paged_bf16", cache.head_dim
    _on_device(cache, fn)
    qp, qs = _token_rows(cache, q, num_seqs, num_q_heads, D, "q")
    need = flash_decode_paged_scratch_floats(num_seqs, num_q_heads, cache.num_kv_heads, D)
    call(fn, _cptr(cache, out, _BF, num_seqs * num_q_heads * D, "out"), qp, qs, cache.desc, layer, _cptr(cache, rows, _I32, num_seqs, "rows"), num_seqs,
         num_q_heads, float(scale), _cptr(cache, partial, _F32, need, "partial"), _cptr(cache, shared_pages, _I32, cache.pages_per_row, "shared_pages"),
         _cptr(cache, shared_len, _I32, 1, "shared_len"), _stream(stream))


def flash_prefill_packed_splits(num_tokens: int, num_seqs: int, max_keys: int, num_q_heads: int, num_kv_heads: int, head_dim: int) -> int:
    """Into how many key ranges flash_prefill_packed_bf16 had best deal the keys of this batch (max_keys: its longest row with
    the new tokens): more than one where few new tokens stand behind long histories."""
    from ._lib import lib
    return int(lib.rh_flash_prefill_packed_splits(num_tokens, num_seqs, max_keys, num_q_heads, num_kv_heads, head_dim))


def flash_prefill_packed_scratch_floats(num_tokens: int, num_q_heads: int, head_dim: int, num_splits: int) -> int:
    """Floats of scratch that flash_prefill_packed_bf16 needs for this many key ranges (0 for one)."""
    from ._lib import lib
    return int(lib.rh_flash_prefill_packed_scratch_floats(num_tokens, num_q_heads, head_dim, num_splits))


def flash_prefill_packed_bf16(out, q, cache, layer: int, cu_seqlens, num_tokens: int, num_seqs: int, num_q_heads: int, scale: float,
                              partial=None, num_splits: int = 1, rows=None, stream=None) -> None:
    """A packed batch's new tokens attend causally: token i of an entry sees keys 0..lens[row] + i of its row."""
    fn, D = "rh_flash_prefill_packed_bf16", cache.head_dim
    _on_device(cache, fn)
    qp, qs = _token_rows(cache, q, num_tokens, num_q_heads, D, "q")
    need = flash_prefill_packed_scratch_floats(num_tokens, num_q_heads, D, num_splits)
    call(fn, _cptr(cache, out, _BF, num_tokens * num_q_heads * D, "out"), qp, qs, cache.desc, layer, _cptr(cache, rows, _I32, num_seqs, "rows"),
         _cptr(cache, cu_seqlens, _I32, num_seqs + 1, "cu_seqlens"), num_tokens, num_seqs, num_q_heads, float(scale),
         _cptr(cache, partial, _F32, need, "partial") if num_splits > 1 else None, num_splits, _stream(stream))
