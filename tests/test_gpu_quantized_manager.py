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
