"""GPU tests of a quantised PagedKVCache's steps where they meet: reads on one stream and the next
step's writes on another."""
import pytest
import torch

import quant_ref as ref
from gpu_offloading_amd.kv_cache import PagedKVCache
from test_gpu_quantized_cache import Model, rows

pytestmark = pytest.mark.gpu

HOLD = 40_000_000            # cycles that the side stream waits (some 20 ms)


@pytest.mark.parametrize("setup", ["step", "chunk"])
@pytest.mark.parametrize("codec", ref.CODECS)
def test_pages_are_read_before_they_are_handed_out_again(gpu, codec, setup):
    """A chunk's attention held up on a side stream; meanwhile its sequence is freed and another
    one's tokens go into the same pages."""
    n, hkv, group, d = 300, 2, 4, 128
    pages = (n + 15) // 16
    c = PagedKVCache(1, hkv, d, max_seqs=3, max_seq_len=320, num_qo_heads=hkv * group,
                     kv_page_budget=pages, device=gpu, kv_dtype=codec, workspace_bytes=1 << 22)
    m = Model(c)
    k, v, k2, v2 = (rows((n, hkv, d), i, torch.bfloat16) for i in range(4))
    q = rows((n, hkv * group, d), 5, torch.bfloat16).to(gpu)
    moved = [t.to(gpu) for t in (k, v, k2, v2)]

    def plan(s):
        c.ensure_pages(s, pages)
        return c.prepare_step(continuation_seq_ids=[s], continuation_lens=[n]) \
            if setup == "step" else c.prepare_prefill_chunk([s], [n])

    slots = plan(0)
    held = c.block_table[0, :pages].tolist()
    c.append(0, *moved[:2], slots)
    m.append(0, 0, k, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(HOLD)
        out, lse = c.prefill(0, q, return_lse=True)
    c.free_seq(0)
    slots = plan(1)
    assert sorted(c.block_table[1, :pages].tolist()) == sorted(held)
    c.append(0, *moved[2:], slots)
    torch.cuda.synchronize()
    m.check_chunk(out, lse, q, 0, 0)
    m.append(1, 0, k2, v2)
    out, lse = c.prefill(0, q, return_lse=True)
    m.check_chunk(out, lse, q, 1, 0)


def test_a_refused_chunk_plan_leaves_the_mixed_step_undone(gpu, monkeypatch):
    """Lengths on both sides, the decode plan and the chunks planned before stay as they were
    where a mixed step's chunks cannot be planned; the step made again then is right."""
    c = PagedKVCache(1, 2, 128, max_seqs=3, max_seq_len=320, num_qo_heads=8, kv_page_budget=40,
                     device=gpu, kv_dtype=ref.INT8, workspace_bytes=1 << 22)
    m = Model(c)

    def new(n, seed):
        k, v = (rows((n, 2, 128), seed + i, torch.bfloat16) for i in range(2))
        return k, v, rows((n, 8, 128), seed + 2, torch.bfloat16).to(gpu)

    for s, n in ((0, 40), (1, 50)):
        c.ensure_pages(s, 6)
        k, v, q = new(n, s * 10)
        c.append(0, k.to(gpu), v.to(gpu), c.prepare_prefill_chunk([s], [n]))
        m.append(s, 0, k, v)
    c.plan_decode([0, 1])
    qd = new(2, 50)[2]
    want = c.decode(0, qd), c.prefill(0, q)

    def refuse(*args):
        raise RuntimeError("no plan")

    with monkeypatch.context() as p:
        p.setattr("gpu_offloading_amd.prompt.stage_plan", refuse)
        c.ensure_pages(2, 1)
        with pytest.raises(RuntimeError, match="no plan"):
            c.prepare_step([0], [2], [9], [1], [30])
    assert c._seq_lens_cpu.tolist() == c.seq_lens.tolist() == [40, 50, 0]
    assert torch.equal(c.decode(0, qd), want[0]) and torch.equal(c.prefill(0, q), want[1])
    slots = c.prepare_step([0], [2], [9], [1], [30])
    assert c._seq_lens_cpu.tolist() == c.seq_lens.tolist() == [41, 80, 9]
    k, v, q = new(40, 70)
    c.append(0, k.to(gpu), v.to(gpu), slots)
    for s, (a, b) in enumerate(((0, 1), (10, 40), (1, 10))):
        m.append(s, 0, k[a:b], v[a:b])
    m.check_decode(*c.decode(0, q[:1], return_lse=True), q[:1], [0], 0)
    m.check_chunk(*c.prefill(0, q[10:], return_lse=True), q[10:], 1, 0)
