"""The paged KV cache in 8 bits: quantised as it is written, read back, attended.

A cache of ``quantized_cache`` holds codes ``[blocks, kv_heads, 16, head_dim]`` (int8 or
OCP e4m3, ``torch.float8_e4m3fn``) for K and for V and one fp32 scale per token's
row of a head, ``[blocks, kv_heads, 2, 16]`` (K's scales, then V's): half a bf16 cache's
bytes.  A code stands for ``code * scale``:

  e4m3  scale ``2^e``, the least with ``amax / 2^e <= 448``; relative error up to
        2^-4 of each value (2^-10 of the scale near zero); the largest values of the rows'
        type stay finite
  int8  scale ``amax / 127``; error up to ``amax / 254``

The ops keep the manner of ``ops`` (``RuntimeError`` for bad arguments, the current torch
stream unless one is given, no fallback) and launch the kernels of
csrc/quant_cache.hip and csrc/quant_decode.hip, ordinary calls by way of csrc/bind.cpp.  ``PagedKVCache(kv_dtype=...)`` is
the cache manager over them.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from .ops import _WDTYPES as _DTYPES
from .ops import _check_cuda, _check_ints, _fail, _oob_ptr, _ptr
from .prompt import _empty

__all__ = ["QuantizedCache", "quantized_cache", "reshape_and_cache_quantized",
           "gather_quantized_kv", "quantized_decode_attention", "decode_workspace"]

PAGE = 16
CODES = {torch.float8_e4m3fn: 0, torch.int8: 1}


class QuantizedCache(NamedTuple):
    """One layer's cache: the three tensors that the ops take, views of ``storage``
    (uint8 ``[blocks, block bytes]``), in which a block is one contiguous piece."""

    key_cache: torch.Tensor
    value_cache: torch.Tensor
    scales: torch.Tensor
    storage: torch.Tensor


def quantized_cache(num_blocks: int, num_kv_heads: int, head_dim: int,
                    kv_dtype: torch.dtype = torch.float8_e4m3fn,
                    device: str | torch.device = "cuda") -> QuantizedCache:
    """A zeroed cache of ``num_blocks`` blocks of 16 tokens: per block K's codes, V's
    codes and the scales."""
    if kv_dtype not in CODES:
        _fail(f"kv_dtype must be torch.float8_e4m3fn or torch.int8, got {kv_dtype}")
    if num_blocks <= 0 or num_kv_heads <= 0 or head_dim not in (64, 128, 256):
        _fail(f"need blocks, KV heads and head_dim 64, 128 or 256, got {num_blocks}, "
              f"{num_kv_heads}, {head_dim}")
    codes = num_kv_heads * PAGE * head_dim
    storage = torch.zeros((num_blocks, 2 * codes + num_kv_heads * 2 * PAGE * 4),
                          dtype=torch.uint8, device=device)
    shape = (num_blocks, num_kv_heads, PAGE, head_dim)
    k, v = (storage[:, i * codes:(i + 1) * codes].view(kv_dtype).unflatten(1, shape[1:])
            for i in range(2))
    scales = storage[:, 2 * codes:].view(torch.float32).unflatten(1, (num_kv_heads, 2, PAGE))
    return QuantizedCache(k, v, scales, storage)


def _check_quantized(key_cache: torch.Tensor, value_cache: torch.Tensor, scales: torch.Tensor):
    """Shapes, types and strides of a cache's tensors; returns (blocks, heads, dim, code,
    block stride of the codes, block stride of the scales)."""
    shape, st, ss, dt = key_cache.shape, key_cache.stride(), scales.stride(), key_cache.dtype
    code = CODES.get(dt)
    if code is None or value_cache.dtype is not dt:
        _fail("key_cache and value_cache must both be float8_e4m3fn or int8, got "
              f"{dt} and {value_cache.dtype}")
    if len(shape) != 4 or shape[2] != PAGE:
        _fail(f"key_cache must be [num_blocks, num_kv_heads, 16, head_dim], got {tuple(shape)}")
    nb, h, _, d = shape
    if value_cache.shape != shape or value_cache.stride() != st:
        _fail("key_cache and value_cache must have the same shape and strides")
    if scales.dtype is not torch.float32 or scales.shape != (nb, h, 2, PAGE):
        _fail(f"scales must be float32 [{nb}, {h}, 2, 16], got {scales.dtype} "
              f"{tuple(scales.shape)}")
    if st[1:] != (PAGE * d, d, 1) and (st[3] != 1 or st[2] != d or h > 1):
        _fail(f"key_cache: a block must be contiguous (strides {st})")
    if ss[1:] != (2 * PAGE, PAGE, 1) and (ss[3] != 1 or ss[2] != PAGE or h > 1):
        _fail(f"scales: a block must be contiguous (strides {ss})")
    if nb > 1:
        return nb, h, d, code, st[0], ss[0]
    # (of a single block any stride is valid)
    return nb, h, d, code, max(st[0], h * PAGE * d), max(ss[0], h * 2 * PAGE)


def _check_tokens(name: str, t: torch.Tensor, heads: int, dim: int) -> int:
    """``[tokens, heads, dim]`` bf16 or fp16 with a token's heads contiguous; returns the
    elements between tokens."""
    sh, st = t.shape, t.stride()
    if len(sh) != 3 or sh[1] != heads or sh[2] != dim:
        _fail(f"{name} must be [tokens, {heads}, {dim}], got {tuple(sh)}")
    if t.dtype not in _DTYPES:
        _fail(f"{name} must be bfloat16 or float16, got {t.dtype}")
    if st[2] != 1 or (st[1] != dim and heads > 1):
        _fail(f"{name}: heads of a token must be contiguous (strides {st})")
    return st[0] if sh[0] > 1 else heads * dim


def _stream(index: int, stream: Optional[torch.cuda.Stream]) -> int:
    return stream.cuda_stream if stream is not None else _lib.current_stream_of(index)


def _check_device(*ts: Optional[torch.Tensor]) -> int:
    """The GPU that all of them are on."""
    index = ts[0].get_device()
    for t in ts:
        if t is not None and (t.get_device() != index or index < 0):
            _check_cuda(*ts)                    # (says which)
    return index


def _status(name: str, st: int) -> None:
    if st:
        _lib.check(name, st)


def reshape_and_cache_quantized(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor,
                                value_cache: torch.Tensor, scales: torch.Tensor,
                                slot_mapping: torch.Tensor, *,
                                oob_count: Optional[torch.Tensor] = None,
                                stream: Optional[torch.cuda.Stream] = None) -> None:
    """Quantise key[i]/value[i] into cache slot ``slot_mapping[i]`` (in place).

    ``reshape_and_cache_flash`` for a quantised cache: key/value ``[num_tokens,
    num_kv_heads, head_dim]`` bf16 or fp16 (slices of a fused tensor will do), int64
    slot_mapping whose length is the token count, a negative slot is padding.  The
    slots of a call must be distinct.  A row that holds an infinity or a NaN reads back
    as NaN."""
    st = (_lib._bind or _lib.binding()).write(key, value, key_cache, value_cache, scales,
                                              slot_mapping, oob_count, stream)
    if st is not None:
        return _status("kvc_reshape_and_cache_quantized", st)
    index = _check_device(key_cache, value_cache, scales, key, value, slot_mapping, oob_count)
    nb, h, d, code, cs, ss = _check_quantized(key_cache, value_cache, scales)
    if slot_mapping.dtype is not torch.int64 or slot_mapping.dim() != 1 \
            or not slot_mapping.is_contiguous():
        _fail("slot_mapping must be a contiguous 1-D int64 tensor")
    n = slot_mapping.numel()
    ks, vs = _check_tokens("key", key, h, d), _check_tokens("value", value, h, d)
    if key.dtype is not value.dtype:
        _fail(f"key is {key.dtype}, value {value.dtype}")
    if key.shape[0] < n or value.shape[0] < n:
        _fail(f"key and value have {key.shape[0]} and {value.shape[0]} rows but slot_mapping "
              f"has {n}")
    _lib.call_on(index, "kvc_reshape_and_cache_quantized", key.data_ptr(),
                 value.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
                 scales.data_ptr(), slot_mapping.data_ptr(), n, h, d, PAGE, nb,
                 _DTYPES[key.dtype], code, ks, vs, cs, ss, _oob_ptr(oob_count),
                 _stream(index, stream))


def gather_quantized_kv(key_cache: torch.Tensor, value_cache: torch.Tensor, scales: torch.Tensor,
                        block_table: torch.Tensor, cu_seq_lens: torch.Tensor, max_seq_len: int,
                        out_key: Optional[torch.Tensor] = None,
                        out_value: Optional[torch.Tensor] = None,
                        seq_starts: Optional[torch.Tensor] = None, *,
                        dtype: torch.dtype = torch.bfloat16,
                        oob_count: Optional[torch.Tensor] = None,
                        stream: Optional[torch.cuda.Stream] = None):
    """Each sequence's cached K and V as contiguous rows of ``dtype`` (that of the outputs,
    if they are given).

    ``gather_kv`` for a quantised cache: row ``cu_seq_lens[b] + i`` of the outputs receives
    token ``seq_starts[b] + i`` of sequence ``b`` (block-table row ``b``); ``max_seq_len``
    (host int) must bound every length.  Values are ``code * scale`` in fp32, rounded
    once (e4m3 values in bf16 are exact).  Returns ``(out_key, out_value)``, each
    ``[total_tokens, num_kv_heads, head_dim]``; give both to avoid reading the total back
    from the device."""
    st = (_lib._bind or _lib.binding()).read(key_cache, value_cache, scales, block_table,
                                             cu_seq_lens, max_seq_len, out_key, out_value,
                                             seq_starts, oob_count, stream)
    if st is not None:
        _status("kvc_gather_quantized_kv", st)
        return out_key, out_value
    index = _check_device(key_cache, value_cache, scales, block_table, cu_seq_lens, seq_starts,
                          out_key, out_value, oob_count)
    nb, h, d, code, cs, ss = _check_quantized(key_cache, value_cache, scales)
    if block_table.dtype is not torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1:
        _fail("block_table must be a 2-D int32 tensor with contiguous rows")
    batch = cu_seq_lens.numel() - 1
    _check_ints("cu_seq_lens", cu_seq_lens, 1, index)
    if batch > block_table.shape[0]:
        _fail("cu_seq_lens must have batch+1 entries with batch <= block_table rows")
    if seq_starts is not None:
        _check_ints("seq_starts", seq_starts, batch, index)
    if not 0 <= max_seq_len < 1 << 31:
        _fail(f"max_seq_len must be in 0..2^31-1, got {max_seq_len}")
    if out_key is None or out_value is None:
        given = out_key if out_key is not None else out_value
        dt = dtype if given is None else given.dtype
        total = int(cu_seq_lens[-1].item()) if batch > 0 else 0
        dev = key_cache.device
        if out_key is None:
            out_key = _empty((total, h, d), dt, dev, stream)
        if out_value is None:
            out_value = _empty((total, h, d), dt, dev, stream)
    os = _check_tokens("out_key", out_key, h, d)
    ov = _check_tokens("out_value", out_value, h, d)
    if out_key.dtype is not out_value.dtype:
        _fail(f"out_key is {out_key.dtype}, out_value {out_value.dtype}")
    rows = min(out_key.shape[0], out_value.shape[0])
    if rows > 1 and os != ov:
        _fail("out_key and out_value must share the token stride")
    if rows == 0:
        return out_key, out_value
    _lib.call_on(index, "kvc_gather_quantized_kv", key_cache.data_ptr(), value_cache.data_ptr(),
                 scales.data_ptr(), block_table.data_ptr(), block_table.stride(0),
                 block_table.shape[1], cu_seq_lens.data_ptr(), _ptr(seq_starts), batch,
                 int(max_seq_len), h, d, PAGE, nb, _DTYPES[out_key.dtype], code, cs, ss,
                 out_key.data_ptr(), out_value.data_ptr(), max(os, ov), rows,
                 _oob_ptr(oob_count), _stream(index, stream))
    return out_key, out_value


def decode_workspace(batch: int, num_qo_heads: int, num_kv_heads: int, head_dim: int,
                     device: str | torch.device = "cuda") -> torch.Tensor:
    """Device memory for ``quantized_decode_attention``, for batches of up to ``batch``
    requests: of one call at a time (calls on several streams, and graphs that may run
    side by side, need one each); nothing is kept in it between calls."""
    need = _lib.load().kvc_quantized_decode_workspace_bytes(batch, num_qo_heads, num_kv_heads,
                                                            head_dim)
    return torch.empty(max(int(need), 16), dtype=torch.uint8, device=device)


def quantized_decode_attention(q: torch.Tensor, key_cache: torch.Tensor,
                               value_cache: torch.Tensor, scales: torch.Tensor,
                               indptr: torch.Tensor, indices: torch.Tensor,
                               last_page_len: torch.Tensor, *,
                               sm_scale: Optional[float] = None,
                               out: Optional[torch.Tensor] = None,
                               lse: Optional[torch.Tensor] = None, return_lse: bool = False,
                               workspace: Optional[torch.Tensor] = None,
                               stream: Optional[torch.cuda.Stream] = None):
    """Attention of one new token per request over its cached tokens.

    ``q [B, num_qo_heads, head_dim]`` bf16 or fp16, at most 16 query heads per KV head;
    ``indptr [B + 1]``, ``indices`` and ``last_page_len [B]`` are the requests' pages, as the
    bf16 decode's, int32 on the device (read by the kernel: no plan, and a captured launch
    serves other lengths and pages).  Returns ``out`` (as ``q``) or ``(out, lse)``, ``lse``
    float32 ``[B, num_qo_heads]``, the natural-log log-sum-exp of the scaled logits (-inf, and
    ``out`` 0, for a request without tokens).  ``workspace``: from ``decode_workspace``;
    made for the call if not given."""
    got = (_lib._bind or _lib.binding()).decode(q, key_cache, value_cache, scales, indptr, indices,
                                                last_page_len, sm_scale, out, lse, return_lse,
                                                workspace, stream)
    if got is not None:
        if got.__class__ is int:
            _status("kvc_quantized_decode", got)
        return got
    index = _check_device(key_cache, value_cache, scales, q, indptr, indices, last_page_len, out,
                          lse, workspace)
    nb, hkv, d, code, cs, ss = _check_quantized(key_cache, value_cache, scales)
    if q.dim() != 3:
        _fail(f"q must be [requests, num_qo_heads, head_dim], got {tuple(q.shape)}")
    batch, hq = q.shape[:2]
    qs = _check_tokens("q", q, hq, d)
    if hq == 0 or hq % hkv:
        _fail(f"num_qo_heads ({hq}) must be a multiple of num_kv_heads ({hkv})")
    _check_ints("indptr", indptr, batch + 1, index)
    _check_ints("indices", indices, 0, index)
    _check_ints("last_page_len", last_page_len, batch, index)
    if out is None:
        out = q.new_empty((batch, hq, d)) if stream is None else \
            _empty((batch, hq, d), q.dtype, q.device, stream)
        os = hq * d
    else:
        os = _check_tokens("out", out, hq, d)
        if out.dtype is not q.dtype or out.shape[0] < batch:
            _fail(f"out must be {q.dtype} [{batch}, {hq}, {d}], got {out.dtype} "
                  f"{tuple(out.shape)}")
    if lse is None:
        if return_lse:
            lse = q.new_empty((batch, hq), dtype=torch.float32) if stream is None else \
                _empty((batch, hq), torch.float32, q.device, stream)
    elif lse.dtype is not torch.float32 or not lse.is_contiguous() or lse.numel() < batch * hq:
        _fail("lse must be contiguous float32 [requests, num_qo_heads]")
    if workspace is None:
        if stream is None:
            workspace = decode_workspace(batch, hq, hkv, d, q.device)
        else:
            with torch.cuda.stream(stream):     # the memory of the stream that uses it
                workspace = decode_workspace(batch, hq, hkv, d, q.device)
    elif not workspace.is_contiguous():
        _fail("workspace must be contiguous (decode_workspace makes it)")
    _lib.call_on(index, "kvc_quantized_decode", q.data_ptr(), qs, key_cache.data_ptr(),
                 value_cache.data_ptr(), scales.data_ptr(), cs, ss, nb, indptr.data_ptr(),
                 indices.data_ptr(), indices.numel(), last_page_len.data_ptr(), batch, hq, hkv, d,
                 PAGE, _DTYPES[q.dtype], code,
                 float(sm_scale) if sm_scale is not None else d ** -0.5, workspace.data_ptr(),
                 workspace.numel() * workspace.element_size(), out.data_ptr(), os, _ptr(lse),
                 _stream(index, stream))
    return (out, lse) if return_lse else out
