"""CPU tests of a quantised PagedKVCache's own steps around its ops: which streams it orders and
in what order it works.  (The ops themselves are stand-ins here: nothing is launched.)"""
import types

import pytest
import torch

from gpu_offloading_amd import _lib, quantized
from gpu_offloading_amd.kv_cache import PagedKVCache


def cpu_cache(**kw):
    return PagedKVCache(1, 2, 128, max_seqs=4, max_seq_len=64, num_qo_heads=4, kv_page_budget=8,
                        device="cpu", kv_dtype=torch.float8_e4m3fn, **kw)


def test_prefill_takes_part_in_the_order_of_streams(monkeypatch):
    """prefill on any stream is entered among the step's users before its reads are launched, as
    decode is, so that the next step's appends come after them."""
    c = cpu_cache()
    done = []
    c._decode_wrapper = object()
    c._step_stream_for_call = lambda: done.append("step")
    c._chunk_wrapper = types.SimpleNamespace(
        _plan_stream=1, _run_stream=lambda s: done.append("plan") or 1,
        run=lambda *a, **kw: done.append("attention"))
    c._quant_chunks = (None, None, 3, 3)
    monkeypatch.setattr(quantized, "gather_quantized_kv", lambda *a: done.append("read"))
    c.prefill(0, torch.zeros(3, 4, 128, dtype=torch.bfloat16))
    assert sorted(done[:2]) == ["plan", "step"] and done[2:] == ["read", "attention"]


class Stream:
    """A stream that notes which others it waits for."""

    def __init__(self, handle):
        self.cuda_stream, self.waits = handle, []

    def wait_stream(self, other):
        self.waits.append(other.cuda_stream)


@pytest.mark.parametrize("step_handle", [None, 1, 2])
def test_the_next_plan_waits_for_a_prefill_on_another_stream(monkeypatch, step_handle):
    """Chunks planned on stream 1 and attended to on stream 2: every later plan on stream 1 comes
    after the read, whatever decode step was set up before, and on which stream."""
    c = cpu_cache()
    main, side = Stream(1), Stream(2)
    now = [main]
    monkeypatch.setattr(_lib, "current_stream_handle", lambda device: now[0].cuda_stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: now[0])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda h, device=None: Stream(h))
    monkeypatch.setattr(quantized, "gather_quantized_kv", lambda *a: None)
    c._decode_wrapper, c._step_handle = object(), step_handle
    c._chunk_wrapper = types.SimpleNamespace(
        _plan_stream=1, _run_stream=lambda s: now[0].cuda_stream, run=lambda *a, **kw: None)
    c._quant_chunks = (None, None, 3, 3)
    q = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
    now[0] = side
    c.prefill(0, q)
    assert side.waits == ([1] if step_handle == 1 else [])
    now[0] = main
    plans = []
    c._plan_quant_chunks = lambda *a: plans.append(list(main.waits))
    c.plan_prefill([0], [0])
    assert plans == [[2]]              # another chunk plan, ...
    assert c._claim_step_buffer() == 1 and main.waits == [2, 2]     # ... and a step of any kind
    assert c._step_users == {} and c._step_handle == 1
    c.prefill(0, q)                    # on the plan's own stream: nothing to wait for
    c.plan_prefill([0], [0])
    assert main.waits == [2, 2]
