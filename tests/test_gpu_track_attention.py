"""GPU test of attention tracking and eviction through PagedKVCache, as an engine
would use them: new prompts (their own attention, append, weights), a mixed step
with a continuation chunk, decode steps, eviction, further steps, a swap of an
evicted sequence.  A model of the cache on the host in 64 bits holds, per layer,
sequence and KV head, which token sits in which slot and its score; the scores'
tolerance is what their fp32 sums and the attention's log-sum-exp (bf16
exponentials only enter the outputs) allow."""
import random

import numpy as np
import pytest
import torch

import attention_ref as ref
from gpu_offloading_amd.kv_cache import PagedKVCache
from gpu_offloading_amd.offload import SwapPreemption

pytestmark = pytest.mark.gpu

HKV, HQ, D, LAYERS = 2, 8, 128, 2
SCALE = D ** -0.5


class Model:
    """Tokens of each (sequence, layer, head): slot -> [position, K row, V row, score]."""

    def __init__(self, cache):
        self.cache, self.tok, self.seen = cache, {}, {}

    def append(self, s, k, v):
        """k, v [layers, tokens, HKV, D]"""
        p0 = self.seen.get(s, 0)
        for layer in range(LAYERS):
            for h in range(HKV):
                t = self.tok.setdefault((s, layer, h), [])
                t += [[p0 + i, k[layer, i, h].cpu().double(), v[layer, i, h].cpu().double(), 0.0]
                      for i in range(k.shape[1])]
        self.seen[s] = p0 + k.shape[1]

    def attend(self, s, layer, q, votes=None):
        """Attention of the last len(q) tokens' queries: adds the weights of the last
        ``votes`` rows to the scores and returns (out, lse, tolerances)."""
        m = len(q)
        got = []
        for h in range(HKV):
            t = self.tok[s, layer, h]
            k, v = (torch.stack([x[i] for x in t])[:, None] for i in (1, 2))
            g = slice(h * HQ // HKV, (h + 1) * HQ // HKV)
            o, l, ot, lt = ref.attention(q[:, g], k, v, len(t) - m, True, SCALE)
            r = m if votes is None else min(votes, m)
            w, _ = ref.weights(q[m - r:, g], l[m - r:], k, len(t) - r, True, SCALE)
            for x, y in zip(t, w[0].tolist()):
                x[3] += y
            got.append((o, l, ot, lt))
        return [torch.cat([x[i] for x in got], 1) for i in range(4)]

    def evict(self, s, keep, recent):
        for layer in range(LAYERS):
            for h in range(HKV):
                t = self.tok[s, layer, h]
                # by the device's scores: a tie within rounding may fall either way
                score = self.scores(s, layer, h)
                dst, src = ref.evict(score, [x[0] for x in t], len(t), keep, recent, self.seen[s])
                for a, b in zip(dst, src):
                    t[a] = t[b]
                del t[keep:]

    def scores(self, s, layer, h):
        c = self.cache
        n = len(self.tok[s, layer, h])
        pages = c.block_table[s, :(n + 15) // 16].cpu().long()
        return c.scores[layer].cpu()[pages, h].flatten()[:n].tolist()

    def check(self, steps):
        c = self.cache
        for (s, layer, h), t in self.tok.items():
            n = len(t)
            assert int(c.seq_lens[s]) == n == int(c._seq_lens_cpu[s])
            assert c.next_position(s) == self.seen[s]
            pages = c.block_table[s, :(n + 15) // 16].cpu().long()
            assert (c.block_table[s, (n + 15) // 16:] == -1).all() or c.seq_pages(s) * 16 >= n
            rows = [x[pages, :, h].flatten(0, 1)[:n] for x in (c.k_cache[layer].cpu(),
                                                               c.v_cache[layer].cpu())]
            for i, x in ((1, rows[0]), (2, rows[1])):
                assert torch.equal(x.double(), torch.stack([y[i] for y in t]))
            place = c.positions[layer].cpu()[pages, h].flatten()[:n]
            assert place.tolist() == [x[0] for x in t]
            got = torch.tensor(self.scores(s, layer, h)).double()
            want = torch.tensor([x[3] for x in t]).double()
            # each term is off by at most 2^-11 relative: scores of |q||k| / sqrt(D) < 40 at
            # 128 fp32 additions (2^-17 each at most), the log-sum-exp alike
            assert ((got - want).abs() <= 2.0 ** -10 * want + 1e-6).all(), (s, layer, h)


def _r(gpu, *shape, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(torch.bfloat16).to(gpu)


def _close(got, want, tol, what):
    ref.assert_within(got, want, tol, what)


def test_prompts_chunks_decodes_and_evictions(gpu):
    rng = random.Random(1)
    order = list(range(80))
    rng.shuffle(order)
    c = PagedKVCache(LAYERS, HKV, D, max_seqs=6, max_seq_len=80 * 16, num_qo_heads=HQ,
                     kv_page_budget=80, free_page_order=order, device=gpu)
    c.track_attention()
    m = Model(c)
    seed = [100]

    def r(*shape):
        seed[0] += 1
        return _r(gpu, *shape, seed=seed[0])

    def decode(seqs):
        for s in seqs:
            c.ensure_pages(s, int(c._seq_lens_cpu[s]) // 16 + 1)
        c.prepare_decode_step(seqs)
        k, v, q = r(LAYERS, len(seqs), HKV, D), r(LAYERS, len(seqs), HKV, D), r(LAYERS, len(seqs), HQ, D)
        for i, s in enumerate(seqs):
            m.append(s, k[:, i:i + 1], v[:, i:i + 1])
        for layer in range(LAYERS):
            out, lse = c.append_and_decode(layer, k[layer], v[layer], q[layer], return_lse=True)
            c.decode_weights(layer, q[layer], lse)
            for i, s in enumerate(seqs):
                o, l, ot, lt = m.attend(s, layer, q[layer, i:i + 1])
                _close(out[i:i + 1], o, 2 * ot + 2.0 ** -9, "decode")   # (its kernel's own bar)

    # Two new prompts; in the first only the last 20 tokens vote.
    lens = [150, 60]
    for s, n in zip((4, 1), lens):
        c.ensure_pages(s, (n + 15) // 16)
    slots = c.prepare_step(prefill_seq_ids=[4, 1], prefill_lens=lens)
    c.plan_prompt(lens)
    c.plan_chunk_weights([4, 1], [20, 60], lens)
    k, v, q = r(LAYERS, 210, HKV, D), r(LAYERS, 210, HKV, D), r(LAYERS, 210, HQ, D)
    m.append(4, k[:, :150], v[:, :150])
    m.append(1, k[:, 150:], v[:, 150:])
    for layer in range(LAYERS):
        c.append(layer, k[layer], v[layer], slots)
        out, lse = c.prompt(q[layer], k[layer], v[layer], return_lse=True)
        c.chunk_weights(layer, q[layer, 130:], lse[130:])
        for s, rows, votes in ((4, slice(0, 150), 20), (1, slice(150, 210), None)):
            o, l, ot, lt = m.attend(s, layer, q[layer, rows], votes)
            _close(out[rows], o, ot, "prompt")
            _close(lse[rows], l, lt, "prompt lse")
    m.check(1)
    decode([1, 4])
    decode([4])
    m.check(3)

    free = c.pages_free
    m.evict(4, 64, 10)
    c.evict([4, 1], [64, 100], [10, 0])      # sequence 1 has 61 tokens: left alone
    assert c.pages_free == free + (152 + 15) // 16 - 4 and c.seq_pages(4) == 4
    assert c.next_position(4) == 152 and c.next_position(1) == 61
    with pytest.raises(RuntimeError):
        c.decode(0, q[0, :2])                # the plan is gone
    m.check(3)

    # A mixed step: sequence 1 decodes, the evicted one gets a chunk of 40 tokens.
    c.ensure_pages(4, 7)
    slots = c.prepare_step(decode_seq_ids=[1], continuation_seq_ids=[4], continuation_lens=[40])
    c.plan_chunk_weights([4], [40])
    k, v, q = r(LAYERS, 41, HKV, D), r(LAYERS, 41, HKV, D), r(LAYERS, 41, HQ, D)
    m.append(1, k[:, :1], v[:, :1])
    m.append(4, k[:, 1:], v[:, 1:])
    for layer in range(LAYERS):
        c.append(layer, k[layer], v[layer], slots)
        _, lse = c.decode(layer, q[layer, :1], return_lse=True)
        c.decode_weights(layer, q[layer, :1], lse)
        m.attend(1, layer, q[layer, :1])
        _, lse = c.prefill(layer, q[layer, 1:], return_lse=True)
        c.chunk_weights(layer, q[layer, 1:], lse)
        m.attend(4, layer, q[layer, 1:])
    m.check(5)
    decode([4, 1])
    m.evict(4, 33, 33)
    m.evict(1, 20, 0)
    c.evict([1, 4], [20, 33], [0, 33])
    m.check(6)

    # The evicted sequence is preempted and resumes in another slot with its state.
    pre = SwapPreemption(c)
    pre.preempt(4, key="x")
    n = c.pages_free
    c.ensure_pages(0, n)       # other tokens in its old pages
    for layer in range(LAYERS):
        c.scores[layer][c.block_table[0, :n].long()] = -1.0
    c.free_seq(0)
    pre.resume("x", 3)
    c.synchronize_swaps()
    for layer in range(LAYERS):
        for h in range(HKV):
            m.tok[3, layer, h] = m.tok.pop((4, layer, h))
    m.seen[3] = m.seen.pop(4)
    m.check(6)
    decode([1, 3])
    m.check(7)
    c.free_seq(3)
    assert c.next_position(3) == 0
    c.reset()
    assert c.next_position(1) == 0 and not any(t.any() for t in c.scores + c.positions)


def test_decode_weights_replayed_from_a_graph(gpu):
    """The layer calls of a step, the weights among them, captured once and replayed
    in later steps: scores equal those of eager steps on an equal cache."""
    def make():
        c = PagedKVCache(1, 8, D, max_seqs=2, max_seq_len=200, num_qo_heads=32, kv_page_budget=30,
                         device=gpu)
        c.track_attention()
        for s, n in ((0, 40), (1, 100)):
            c.ensure_pages(s, 12)
        slots = c.prepare_step(prefill_seq_ids=[0, 1], prefill_lens=[40, 100])
        c.plan_prompt([40, 100])
        c.plan_chunk_weights([0, 1], [40, 100])
        k, v, q = (_r(gpu, 140, h, D, seed=s) for h, s in ((8, 1), (8, 2), (32, 3)))
        c.append(0, k, v, slots)
        _, lse = c.prompt(q, k, v, return_lse=True)
        c.chunk_weights(0, q, lse)
        return c

    a, b = make(), make()
    k, v, q = (torch.zeros(2, h, D, dtype=torch.bfloat16, device=gpu) for h in (8, 8, 32))
    key, graph = None, None
    for step in range(5):
        for t, h, s in ((k, 8, 1), (v, 8, 2), (q, 32, 3)):
            t.copy_(_r(gpu, 2, h, D, seed=50 + 10 * step + s))
        a.prepare_decode_step([0, 1])
        _, lse = a.append_and_decode(0, k, v, q, return_lse=True)
        a.decode_weights(0, q, lse)
        b.prepare_decode_step([0, 1])
        if b.decode_graph_key() != key:
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                _, lse_b = b.append_and_decode(0, k, v, q, return_lse=True)
                b.decode_weights(0, q, lse_b)
            key = b.decode_graph_key()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a.scores[0], b.scores[0]) and torch.equal(a.positions[0], b.positions[0])
        assert torch.equal(a.k_cache[0], b.k_cache[0])


def test_refusals(gpu):
    c = PagedKVCache(1, 8, D, max_seqs=2, max_seq_len=64, num_qo_heads=8, kv_page_budget=8,
                     device=gpu)
    q, lse = _r(gpu, 1, 8, D, seed=1), torch.zeros(1, 8, device=gpu)
    for call in (lambda: c.evict([0], 4), lambda: c.decode_weights(0, q, lse),
                 lambda: c.plan_chunk_weights([0], [1]), lambda: c.chunk_weights(0, q, lse),
                 lambda: c.prompt(q, q, q)):
        with pytest.raises(RuntimeError):
            call()
    c.ensure_pages(0, 1)
    c.advance([0], 1)
    with pytest.raises(RuntimeError):
        c.track_attention()
    c.free_seq(0)
    c.track_attention()
    c.track_attention()
    c.ensure_pages(0, 4)
    c.advance([0], 50)
    for bad in (dict(keep=4, recent=5), dict(keep=-1), dict(keep=4, recent=-1), dict(keep=[1, 2])):
        with pytest.raises(ValueError):
            c.evict([0], **bad)
    for bad in ([0, 0], [2], [-1]):
        with pytest.raises(ValueError):
            c.evict(bad, 4)
    for ids, n, new in (([0], [51], None), ([0], [-1], None), ([0], [1, 1], None),
                        ([0], [1], [51]), ([0, 0], [1, 1], None)):
        with pytest.raises(ValueError):
            c.plan_chunk_weights(ids, n, new)
    with pytest.raises(RuntimeError):
        c.decode_weights(0, q, lse)
    with pytest.raises(ValueError):
        c.plan_prompt([4, -1])
    c.plan_prompt([2])
    with pytest.raises(RuntimeError):
        c.prompt(q, q, q)             # one row for two tokens
