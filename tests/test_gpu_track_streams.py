"""GPU tests of attention tracking across streams: weights calls held up on a side
stream while the host plans, evicts and frees ahead on another one.  Scores, positions
and K/V equal those of the same calls on one stream."""
import pytest
import torch

from gpu_offloading_amd.kv_cache import PagedKVCache

pytestmark = pytest.mark.gpu

HKV, HQ, D = 8, 32, 128
HOLD = 40_000_000            # cycles that the side stream waits (some 20 ms)


def _r(gpu, *shape, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(torch.bfloat16).to(gpu)


class Run:
    """A cache of three prompts, two of them evicted once, and the stream on which its
    layer calls run (None: the current one)."""

    def __init__(self, gpu, side):
        self.gpu, self.side, self.seed, self.kept = gpu, side, 10, []
        c = self.c = PagedKVCache(1, HKV, D, max_seqs=4, max_seq_len=400, num_qo_heads=HQ,
                                  kv_page_budget=60, device=gpu)
        c.track_attention()
        lens = [70, 130, 33]
        for s, n in enumerate(lens):
            c.ensure_pages(s, (n + 15) // 16)
        slots = c.prepare_step(prefill_seq_ids=[0, 1, 2], prefill_lens=lens)
        c.plan_prompt(lens)
        c.plan_chunk_weights([0, 1, 2], lens)
        k, v, q = (_r(gpu, sum(lens), h, D, seed=i) for h, i in ((HKV, 1), (HKV, 2), (HQ, 3)))
        c.append(0, k, v, slots)
        _, lse = c.prompt(q, k, v, return_lse=True)
        c.chunk_weights(0, q, lse)
        c.evict([0, 1], [50, 64], [5, 9])
        torch.cuda.synchronize()

    def rows(self, n):
        self.seed += 3
        got = [_r(self.gpu, n, h, D, seed=self.seed + i) for i, h in enumerate((HKV, HKV, HQ))]
        self.kept += got             # the side stream reads them late
        return got

    def held(self, call):
        """call(), on the side stream behind a wait."""
        if self.side is None:
            return call()
        self.side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(self.side):
            torch.cuda._sleep(HOLD)
            return call()

    def state(self):
        torch.cuda.synchronize()
        c = self.c
        got = []
        for s in range(4):
            n = int(c._seq_lens_cpu[s])
            pages = c.block_table[s, :(n + 15) // 16].long()
            got.append([x[pages].transpose(1, 2).flatten(0, 1)[:n] if x.dim() == 3 else
                        x[pages].flatten(0, 1)[:n]
                        for x in (c.scores[0], c.positions[0], c.k_cache[0], c.v_cache[0])])
        return got


def _same(gpu, story):
    out = []
    for side in (None, torch.cuda.Stream()):
        run = Run(gpu, side)
        story(run)
        out.append(run.state())
    for a, b in zip(*out):
        for x, y in zip(a, b):
            assert torch.equal(x, y)
    assert any(x[0].numel() for x in out[0])


def _fused_step(run, seqs):
    c = run.c
    for s in seqs:
        c.ensure_pages(s, int(c._seq_lens_cpu[s]) // 16 + 1)
    k, v, q = run.rows(len(seqs))
    run.kept.append(c.prepare_decode_step(seqs))

    def layer():
        _, lse = c.append_and_decode(0, k, v, q, return_lse=True)
        c.decode_weights(0, q, lse)
    run.held(layer)


def _planned_step(run, seqs):
    c = run.c
    for s in seqs:
        c.ensure_pages(s, int(c._seq_lens_cpu[s]) // 16 + 1)
    k, v, q = run.rows(len(seqs))
    slots = c.slot_mapping(seqs, [1] * len(seqs))
    c.append(0, k, v, slots)
    c.advance(seqs, 1)
    c.plan_decode(seqs)

    def layer():
        _, lse = c.decode(0, q, return_lse=True)
        c.decode_weights(0, q, lse)
    run.held(layer)


def test_plans_behind_held_up_weights(gpu):
    """The next plan_decode neither frees nor rewrites what the last one's calls read."""
    def story(run):
        _planned_step(run, [0, 1, 2])
        _planned_step(run, [1])
        _planned_step(run, [2, 0])
    _same(gpu, story)


def test_eviction_behind_held_up_weights(gpu):
    def story(run):
        _fused_step(run, [1, 0, 2])
        run.c.evict([0, 1, 2], [40, 60, 20], [3, 3, 3])
        _fused_step(run, [2, 1])
        _planned_step(run, [0])
        run.c.evict([0, 1], 32, 1)
    _same(gpu, story)


def test_freed_and_mixed_behind_held_up_weights(gpu):
    """A sequence is freed and another takes its place; a mixed step with a chunk."""
    def story(run):
        c = run.c
        _fused_step(run, [0, 1, 2])
        if run.side is not None:     # (who gives pages away waits for their readers)
            torch.cuda.current_stream().wait_stream(run.side)
        c.free_seq(1)
        c.ensure_pages(1, 3)
        c.ensure_pages(0, 8)
        slots = c.prepare_step(decode_seq_ids=[2], prefill_seq_ids=[1], prefill_lens=[40],
                               continuation_seq_ids=[0], continuation_lens=[30])
        c.plan_prompt([40])
        c.plan_chunk_weights([1, 0], [40, 30])
        k, v, q = run.rows(71)

        def layer():
            c.append(0, k, v, slots)
            _, l0 = c.decode(0, q[:1], return_lse=True)
            c.decode_weights(0, q[:1], l0)
            _, l1 = c.prompt(q[1:41], k[1:41], v[1:41], return_lse=True)
            _, l2 = c.prefill(0, q[41:], return_lse=True)
            c.chunk_weights(0, q[1:], torch.cat([l1, l2]))
        run.held(layer)
        run.kept.append(slots)
        c.evict([0, 1], [30, 30], 4)
        _fused_step(run, [1, 2, 0])
    _same(gpu, story)


def test_the_upload_reaches_other_streams(gpu):
    """Counts uploaded on one stream, read by a step set up and run on another."""
    run = Run(gpu, None)
    c, other = run.c, torch.cuda.Stream()
    want = [c.next_position(s) for s in (0, 1, 2)]
    with torch.cuda.stream(other):
        torch.cuda._sleep(HOLD)
        c._evicted_dirty = True
        c._upload_evicted()
    assert c._evicted_at[0] == other.cuda_stream
    _fused_step(run, [0, 1, 2])
    torch.cuda.synchronize()
    for s in range(3):
        n = int(c._seq_lens_cpu[s])
        page = int(c.block_table[s, (n - 1) // 16])
        assert (c.positions[0][page, :, (n - 1) % 16] == want[s]).all()


def test_counts_are_zero_before_the_first_plan(gpu):
    """A plan made before track_attention: its weights calls read no stale memory."""
    junk = [torch.full((4,), 12345, dtype=torch.int32, device=gpu) for _ in range(64)]
    del junk
    c = PagedKVCache(1, HKV, D, max_seqs=4, max_seq_len=400, num_qo_heads=HQ, kv_page_budget=60,
                     device=gpu)
    c.track_attention()
    assert not c._evicted_dev.any()
