"""Attention weight per cached token, from which a cache evicts single tokens.

``BatchAttentionWeightsWrapper`` is the chunk form (several query tokens per
request: prompts, the last tokens of prompts, continuation chunks);
``ops.decode_attention_weights`` is the form of a decode step and
``ops.evict_kv`` evicts by the scores that either accumulates.
``kv_cache.PagedKVCache`` carries the state through an engine's steps
(``track_attention``).  Kernels: csrc/weights.hip, csrc/evict.hip.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _lib
from .ops import _ptr, check_scores
from .prefill import _fail, _host_int32
from .prompt import _DTYPES, PlannedRuns, _dtype, _empty, _scale, check_rows, stage_plan

__all__ = ["BatchAttentionWeightsWrapper"]


class BatchAttentionWeightsWrapper(PlannedRuns):
    """Attention weights of multi-token queries over a paged cache ("NHD").
    ``float_workspace_buffer`` only fixes the device."""

    def plan(self, qo_indptr: torch.Tensor, paged_kv_indptr: torch.Tensor,
             paged_kv_indices: torch.Tensor, paged_kv_last_page_len: torch.Tensor,
             num_qo_heads: int, num_kv_heads: int, head_dim: int, page_size: int, *,
             causal: bool = True, sm_scale: Optional[float] = None,
             q_data_type: Union[str, torch.dtype] = torch.bfloat16,
             new_tokens: Optional[torch.Tensor] = None) -> None:
        """Stage the work list for ``run``, in the paged prefill wrapper's terms:
        request b's queries are the last ``qo_indptr[b+1] - qo_indptr[b]`` tokens
        of its cached ones.  ``new_tokens`` (int32 per request, default: the
        query tokens) of its last tokens get their first score; a prompt whose
        last tokens vote for all of it passes its whole length."""
        dt = _dtype(q_data_type)
        scale = _scale(sm_scale, head_dim)
        batch = qo_indptr.numel() - 1
        if batch < 0:
            _fail("qo_indptr must have at least one entry")
        if paged_kv_indptr.numel() != batch + 1:
            _fail("qo_indptr and paged_kv_indptr must have the same length")
        qo = _host_int32(qo_indptr, batch + 1, "qo_indptr")
        kv = _host_int32(paged_kv_indptr, batch + 1, "paged_kv_indptr")
        lpl = _host_int32(paged_kv_last_page_len, batch, "paged_kv_last_page_len")
        new = None if new_tokens is None else _host_int32(new_tokens, batch, "new_tokens")
        idx = paged_kv_indices
        if idx.dtype != torch.int32:
            _fail("paged_kv_indices must be int32")
        total = int(kv[-1])
        if idx.numel() < total:
            _fail(f"paged_kv_indices has {idx.numel()} entries, paged_kv_indptr[-1] = {total}")
        idx = idx.reshape(-1)[:total]
        if not idx.is_cuda:
            idx = idx.contiguous().pin_memory().to(self._device, non_blocking=True)
        elif idx.device != self._device:
            _fail("paged_kv_indices on a different device than the workspace")
        sched = _lib.KvcWeightsSchedule()
        guess = 24576 + 22 * max(1, num_kv_heads) * (total // 16 + 2 * batch)
        plan = stage_plan("kvc_weights_plan", sched,
                          (qo.ctypes.data, kv.ctypes.data, lpl.ctypes.data,
                           None if new is None else new.ctypes.data, batch, num_qo_heads,
                           num_kv_heads, head_dim, page_size, 1 if causal else 0),
                          guess, self._device)
        self._set_staged(plan, idx.contiguous())
        self._sched, self._dtype, self._sm_scale = sched, dt, scale

    @property
    def schedule(self) -> Optional[_lib.KvcWeightsSchedule]:
        return self._sched

    def run(self, q: torch.Tensor, lse: torch.Tensor, k_cache: torch.Tensor,
            scores: torch.Tensor, positions: Optional[torch.Tensor] = None,
            position_offsets: Optional[torch.Tensor] = None,
            seq_ids: Optional[torch.Tensor] = None, *,
            stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """Accumulate into ``scores`` (float32 ``[blocks, heads, 16]``) the
        weights that ``q [tokens, num_qo_heads, head_dim]`` gives, with ``lse
        [tokens, num_qo_heads]`` as the attention of these queries returned
        it.  ``positions`` (int32, as ``scores``) gets the new tokens' slots +
        ``position_offsets[seq_ids[b]]`` (``seq_ids`` defaults to b).  Returns
        ``scores``."""
        s = self._sched
        if s is None:
            _fail("run() called before plan()")
        dev = self._index
        qs = check_rows("q", q, s.total_q, s.num_qo_heads, s.head_dim, self._dtype, dev)
        cs = check_scores(dev, q.dtype, lse, s.total_q, s.num_qo_heads, k_cache, s.num_kv_heads,
                          s.head_dim, scores, positions, position_offsets, seq_ids, s.batch)
        if s.num_units == 0:
            return scores
        sh = self._run_stream(stream)
        indices, nbytes, ws = self._staged[1], s.workspace_bytes, None
        if nbytes:
            ws = _empty(nbytes, torch.uint8, self._device, stream)
        _lib.call_on(dev, "kvc_batch_attention_weights_run", s, self._plan_ptr,
                     None if ws is None else ws.data_ptr(), nbytes, q.data_ptr(), qs,
                     lse.data_ptr(), k_cache.data_ptr(), cs[0], cs[1], k_cache.shape[0],
                     indices.data_ptr(), indices.numel(), _DTYPES[self._dtype], self._sm_scale,
                     scores.data_ptr(), _ptr(positions), _ptr(position_offsets),
                     0 if position_offsets is None else position_offsets.numel(), _ptr(seq_ids), sh)
        return scores
