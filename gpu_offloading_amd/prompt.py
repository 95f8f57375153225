"""Attention of whole prompts over their own contiguous K/V.

``BatchPromptAttentionWrapper`` covers the attention that the reference engine
runs for new prompts outside the paged cache (src/MoE/moe_engine.py:2081,
3776): packed sequences, causal or full, grouped heads, bf16 or fp16, head_dim
64, 128 or 256.  It has the ``plan`` / ``run`` form of the paged wrappers:
``plan`` reads the host index pointers, cuts every prompt's queries into tiles
and stages the work list with one small H2D copy; ``run`` launches the kernel of
csrc/prompt.hip once per layer.
"""
from __future__ import annotations

import math
from typing import Optional, Union

import numpy as np
import torch

from . import _lib
from .ops import _WDTYPES as _DTYPES
from .prefill import _fail, _host_int32

__all__ = ["BatchPromptAttentionWrapper"]

_DTYPE_NAMES = {"bfloat16": torch.bfloat16, "bf16": torch.bfloat16,
                "float16": torch.float16, "fp16": torch.float16, "half": torch.float16}


def _dtype(dt: Union[str, torch.dtype]) -> torch.dtype:
    got = _DTYPE_NAMES.get(dt, dt) if isinstance(dt, str) else dt
    if got not in _DTYPES:
        _fail(f"only bfloat16 and float16 are supported, got {dt}")
    return got


def _scale(sm_scale: Optional[float], head_dim: int) -> float:
    s = float(sm_scale) if sm_scale is not None else 1.0 / math.sqrt(head_dim)
    if not (math.isfinite(s) and s > 0.0):
        _fail(f"sm_scale must be positive and finite, got {s}")
    return s


def stage_plan(name: str, sched, args: tuple, capacity: int, device: torch.device) -> torch.Tensor:
    """The host plan function ``name(*args, sched, image, capacity)``, run again
    with the capacity it asks for where ``capacity`` int32 are too few, and its
    image's device copy.  (The guess comes from index pointers that the function
    is the first to check: 16 MiB at most.)"""
    lib = _lib.load()
    capacity = min(capacity, 1 << 22)
    while True:
        image = torch.empty(max(capacity, 8), dtype=torch.int32, pin_memory=True)
        st = getattr(lib, name)(*args, sched, image.data_ptr(), image.numel())
        if st == _lib.KVC_ERR_WORKSPACE and sched.plan_ints > image.numel():
            capacity = int(sched.plan_ints)
            continue
        _lib.check(name, st)
        return image[:max(int(sched.plan_ints), 8)].to(device, non_blocking=True)


class PlannedRuns:
    """A wrapper whose runs read device memory that its plan staged.  A run on
    another stream than the plan's is ordered after the plan's copies, and their
    memory is kept for it; under graph capture the order is the caller's, and
    the graph may be replayed until the next plan."""

    def __init__(self, float_workspace_buffer: torch.Tensor):
        if not float_workspace_buffer.is_cuda:
            _fail("float_workspace_buffer must be a GPU tensor")
        self._device = float_workspace_buffer.device
        self._index = self._device.index
        self._sched = None
        self._staged: tuple = ()
        self._plan_ptr = 0
        self._plan_stream: Optional[int] = None
        self._plan_event: Optional[torch.cuda.Event] = None
        self._ordered: set = set()
        self._dtype = torch.bfloat16
        self._sm_scale = 0.0

    def _set_staged(self, *tensors: torch.Tensor) -> None:
        self._staged = tensors
        self._plan_ptr = tensors[0].data_ptr()
        self._plan_stream = _lib.current_stream_handle(self._device)
        self._plan_event = torch.cuda.Event()
        self._plan_event.record(torch.cuda.current_stream(self._device))
        self._ordered = set()

    def _run_stream(self, stream: Optional[torch.cuda.Stream]) -> int:
        sh = stream.cuda_stream if stream is not None else _lib.current_stream_handle(self._device)
        if sh == self._plan_stream:
            return sh
        if sh not in self._ordered \
                and not torch.cuda.is_current_stream_capturing():
            st = stream if stream is not None else torch.cuda.current_stream(self._device)
            st.wait_event(self._plan_event)
            for t in self._staged:
                t.record_stream(st)
            self._ordered.add(sh)
        return sh


class BatchPromptAttentionWrapper(PlannedRuns):
    """Self-attention of packed prompts.  ``float_workspace_buffer`` only fixes
    the device (interface parity with the paged wrappers)."""

    def plan(self, qo_indptr: torch.Tensor, kv_indptr: Optional[torch.Tensor] = None, *,
             num_qo_heads: int, num_kv_heads: int, head_dim: int, causal: bool = True,
             sm_scale: Optional[float] = None,
             q_data_type: Union[str, torch.dtype] = torch.bfloat16) -> None:
        """Stage the work list for ``run``.  Sequence b's queries are rows
        ``qo_indptr[b]:qo_indptr[b+1]``, its keys rows
        ``kv_indptr[b]:kv_indptr[b+1]`` (default: the same rows); with
        ``causal`` query i sees keys ``j <= i + kv_len - q_len``.  The index
        pointers are int32 and may live on the host or the device (the
        schedule is computed from host copies)."""
        dt = _dtype(q_data_type)
        scale = _scale(sm_scale, head_dim)
        batch = qo_indptr.numel() - 1
        if batch < 0:
            _fail("qo_indptr must have at least one entry")
        qo = _host_int32(qo_indptr, batch + 1, "qo_indptr")
        if kv_indptr is None:
            kv = qo
        elif kv_indptr.numel() != batch + 1:
            _fail("qo_indptr and kv_indptr must have the same length")
        else:
            kv = _host_int32(kv_indptr, batch + 1, "kv_indptr")
        sched = _lib.KvcPromptSchedule()
        group = max(1, num_qo_heads // max(1, num_kv_heads))
        tokens = int(max(0, int(qo[-1]) - int(qo[0])))
        guess = 16384 + 8 * max(1, num_kv_heads) * (tokens * group // 256 + batch)
        plan = stage_plan("kvc_prompt_plan", sched,
                          (qo.ctypes.data, kv.ctypes.data, batch, num_qo_heads, num_kv_heads,
                           head_dim, 1 if causal else 0), guess, self._device)
        self._set_staged(plan)
        self._sched, self._dtype, self._sm_scale = sched, dt, scale

    @property
    def schedule(self) -> Optional[_lib.KvcPromptSchedule]:
        return self._sched

    def run(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
            out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
            return_lse: bool = False, stream: Optional[torch.cuda.Stream] = None):
        """Attention of ``q [tokens, num_qo_heads, head_dim]`` over ``k``/``v
        [tokens, num_kv_heads, head_dim]`` (rows past the planned ones are left
        alone; slices of one fused tensor will do).  Returns ``out`` or ``(out,
        lse)``, ``lse`` float32 ``[tokens, num_qo_heads]``, natural log, -inf for
        a query that sees no key."""
        s = self._sched
        if s is None:
            _fail("run() called before plan()")
        hq, hkv, d = s.num_qo_heads, s.num_kv_heads, s.head_dim
        dt, dev = self._dtype, self._index
        total = s.total_q
        qs = check_rows("q", q, total, hq, d, dt, dev)
        ks = check_rows("k", k, s.total_kv, hkv, d, dt, dev)
        vs = check_rows("v", v, s.total_kv, hkv, d, dt, dev)
        if out is None:
            out = _empty((total, hq, d), dt, self._device, stream)
            os = hq * d
        else:
            os = check_rows("out", out, total, hq, d, dt, dev)
        if lse is None:
            if return_lse:
                lse = _empty((total, hq), torch.float32, self._device, stream)
        elif (lse.dtype != torch.float32 or not lse.is_contiguous()
              or lse.numel() < total * hq or lse.device != self._device):
            _fail("lse must be contiguous float32 [tokens, num_qo_heads] on the wrapper's device")
        nbytes, ws = s.workspace_bytes, None
        if nbytes:
            ws = _empty(nbytes, torch.uint8, self._device, stream)
        _lib.call_on(dev, "kvc_prompt_run", s, self._plan_ptr,
                     None if ws is None else ws.data_ptr(), nbytes, q.data_ptr(), qs,
                     k.data_ptr(), ks, v.data_ptr(), vs, _DTYPES[dt], self._sm_scale, out.data_ptr(), os,
                     None if lse is None else lse.data_ptr(), self._run_stream(stream))
        return (out, lse) if return_lse else out


def _empty(shape, dtype, device, stream: Optional[torch.cuda.Stream]) -> torch.Tensor:
    """An output from the memory of the stream that writes it."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def check_rows(name: str, t: torch.Tensor, rows: int, heads: int, dim: int, dtype: torch.dtype,
               device: int) -> int:
    """Checks ``[rows or more, heads, dim]`` of ``dtype`` on GPU ``device`` with
    the heads of a token contiguous; returns the elements between tokens."""
    sh, st = t.shape, t.stride()
    if len(sh) != 3 or sh[0] < rows or sh[1] != heads or sh[2] != dim:
        _fail(f"{name} must be [{rows}, {heads}, {dim}], got {tuple(sh)}")
    if t.dtype is not dtype or st[2] != 1 or (st[1] != dim and heads > 1):
        _fail(f"{name} must be {dtype} with the heads of a token contiguous")
    if t.get_device() != device:
        _fail(f"{name} on {t.device}, the wrapper's device is cuda:{device}")
    return st[0] if sh[0] > 1 else heads * dim     # of a single token: any valid stride
