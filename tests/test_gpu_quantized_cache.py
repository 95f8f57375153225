"""GPU tests of a quantised PagedKVCache as an engine uses it: new prompts, a mixed step with a
continuation chunk, decode steps (eager, captured, with groups that the bf16 decode does not
take), gather, swap, snapshot.  A model on the host keeps each token's quantised rows; outputs
are held to 64-bit attention over them within derived bounds."""
import math

import numpy as np
import pytest
import torch

import attention_ref
import quant_ref as ref
from gpu_offloading_amd.kv_cache import PagedKVCache
from gpu_offloading_amd.offload import SwapPreemption

pytestmark = pytest.mark.gpu

LAYERS = 2


def rows(shape, seed, dtype, std=0.5):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


class Model:
    """The values that a quantised cache stands for, per sequence and layer."""

    def __init__(self, cache):
        self.c, self.held = cache, {}

    def append(self, s, layer, k, v):
        new = []
        for x in (k, v):
            codes, scale = ref.encode(x, self.c.kv_dtype)
            new.append((ref.values(codes, self.c.kv_dtype), scale))
        old = self.held.get((s, layer))
        self.held[s, layer] = new if old is None else \
            [tuple(np.concatenate(t) for t in zip(a, b)) for a, b in zip(old, new)]

    def values(self, s, layer, i):
        x, scale = self.held[s, layer][i]
        return (torch.from_numpy(x).float() * torch.from_numpy(scale)[..., None]).to(self.c.dtype)

    def check_decode(self, out, lse, q, seqs, layer):
        hkv, d = self.c.num_kv_heads, self.c.head_dim
        group = self.c.num_heads // hkv
        for b, s in enumerate(seqs):
            for h in range(hkv):
                g = slice(h * group, (h + 1) * group)
                (k, ks), (v, vs) = ((torch.from_numpy(x[:, h]), torch.from_numpy(y[:, h]))
                                    for x, y in self.held[s, layer])
                o, l, ot, lt = ref.attention(q[b, g].cpu(), k, ks, v, vs, d ** -0.5, self.c.dtype)
                assert ((out[b, g].cpu().double() - o).abs() <= ot).all(), (s, h, layer)
                assert ((lse[b, g].cpu().double() - l).abs() <= lt).all(), (s, h, layer)

    def check_chunk(self, out, lse, q, s, layer):
        """A chunk's queries see the cache's values as the read-back rounds them."""
        k, v = self.values(s, layer, 0), self.values(s, layer, 1)
        o, l, ot, lt = attention_ref.attention(q.cpu(), k, v, len(k) - len(q), True,
                                               self.c.head_dim ** -0.5)
        assert ((out.cpu().double() - o).abs() <= ot).all()
        assert ((lse.cpu().double() - l).abs() <= lt).all()


def make(gpu, codec, dtype=torch.bfloat16, hkv=2, group=4, d=128, pages=120, max_seqs=6):
    order = np.random.default_rng(3).permutation(pages).tolist()
    return PagedKVCache(LAYERS, hkv, d, max_seqs=max_seqs, max_seq_len=640,
                        num_qo_heads=hkv * group, kv_page_budget=pages, free_page_order=order,
                        device=gpu, dtype=dtype, kv_dtype=codec, workspace_bytes=1 << 24,
                        staging_bytes=1 << 22)


def grow(c, s, n):
    c.ensure_pages(s, (n + 15) // 16)


def decode_step(c, m, seqs, seed, fused):
    for s in seqs:
        grow(c, s, int(c._seq_lens_cpu[s]) + 1)
    slots = c.prepare_decode_step(seqs)
    for layer in range(LAYERS):
        k, v = (rows((len(seqs), c.num_kv_heads, c.head_dim), seed * 10 + layer * 2 + i, c.dtype)
                for i in range(2))
        q = rows((len(seqs), c.num_heads, c.head_dim), seed * 10 + 7, c.dtype).to(c.device)
        for b, s in enumerate(seqs):
            m.append(s, layer, k[b:b + 1], v[b:b + 1])
        if fused:
            out, lse = c.append_and_decode(layer, k.to(c.device), v.to(c.device), q, return_lse=True)
        else:
            c.append(layer, k.to(c.device), v.to(c.device), slots)
            out, lse = c.decode(layer, q, return_lse=True)
        m.check_decode(out, lse, q, seqs, layer)


@pytest.mark.parametrize("codec", ref.CODECS)
@pytest.mark.parametrize("dtype,group,d", [(torch.bfloat16, 4, 128), (torch.float16, 3, 64),
                                           (torch.bfloat16, 5, 256)])
def test_engine_flow(gpu, codec, dtype, group, d):
    c = make(gpu, codec, dtype, group=group, d=d)
    m = Model(c)
    hkv, hq = c.num_kv_heads, c.num_heads
    # two new prompts
    lens = [37, 200]
    for s, n in enumerate(lens):
        grow(c, s, n)
    slots = c.prepare_step(prefill_seq_ids=[0, 1], prefill_lens=lens)
    c.plan_prompt(lens)
    for layer in range(LAYERS):
        k, v = (rows((sum(lens), hkv, d), 100 + layer * 2 + i, dtype) for i in range(2))
        q = rows((sum(lens), hq, d), 110, dtype).to(gpu)
        c.append(layer, k.to(gpu), v.to(gpu), slots)
        c.prompt(q, k.to(gpu), v.to(gpu))
        for s, (a, b) in enumerate(((0, 37), (37, 237))):
            m.append(s, layer, k[a:b], v[a:b])
    # decode steps, one of them fused
    decode_step(c, m, [1, 0], 1, True)
    decode_step(c, m, [0, 1], 2, False)
    # a mixed step: sequence 0 decodes, 2 is a new prompt, 1 continues with a chunk
    for s, n in ((0, 40), (1, 202 + 50), (2, 20)):
        grow(c, s, n)
    slots = c.prepare_step([0], [2], [20], [1], [50])
    for layer in range(LAYERS):
        k, v = (rows((71, hkv, d), 200 + layer * 2 + i, dtype) for i in range(2))
        q = rows((71, hq, d), 210, dtype).to(gpu)
        c.append(layer, k.to(gpu), v.to(gpu), slots)
        for s, (a, b) in ((0, (0, 1)), (2, (1, 21)), (1, (21, 71))):
            m.append(s, layer, k[a:b], v[a:b])
        out, lse = c.decode(layer, q[:1], return_lse=True)
        m.check_decode(out, lse, q[:1], [0], layer)
        out, lse = c.prefill(layer, q[21:], return_lse=True)
        m.check_chunk(out, lse, q[21:], 1, layer)
    # a chunk step of its own, two sequences
    grow(c, 0, 40 + 30)
    grow(c, 2, 20 + 1)
    slots = c.prepare_prefill_chunk([2, 0], [1, 30])
    for layer in range(LAYERS):
        k, v = (rows((31, hkv, d), 300 + layer * 2 + i, dtype) for i in range(2))
        q = rows((31, hq, d), 310, dtype).to(gpu)
        c.append(layer, k.to(gpu), v.to(gpu), slots)
        m.append(2, layer, k[:1], v[:1])
        m.append(0, layer, k[1:], v[1:])
        out, lse = c.prefill(layer, q, return_lse=True)
        m.check_chunk(out[:1], lse[:1], q[:1], 2, layer)
        m.check_chunk(out[1:], lse[1:], q[1:], 0, layer)
    # read back, and plan_decode over what is cached
    gk, gv = c.gather(1, [2, 0, 1])
    assert gk.dtype is dtype
    assert torch.equal(gk.cpu(), torch.cat([m.values(s, 1, 0) for s in (2, 0, 1)]))
    assert torch.equal(gv.cpu(), torch.cat([m.values(s, 1, 1) for s in (2, 0, 1)]))
    c.plan_decode([1, 2])
    q = rows((2, hq, d), 400, dtype).to(gpu)
    out, lse = c.decode(0, q, return_lse=True)
    m.check_decode(out, lse, q, [1, 2], 0)
    # a snapshot, other contents, and back
    snap = c.kv_snapshot()
    c.fill_kv_random(0.3, torch.Generator(device=gpu).manual_seed(1))
    gk, _ = c.gather(0, [1])
    assert not torch.equal(gk.cpu(), m.values(1, 0, 0)) and 0.2 < gk.float().std() < 0.4
    c.kv_restore(snap)
    assert torch.equal(c.decode(0, q), out)


def test_swap_moves_codes_and_scales(gpu):
    """Sequences swapped out and restored into other pages, as preemption does it; the host
    image is half a bf16 cache's and a little."""
    c = make(gpu, ref.E4M3, hkv=8, group=4)
    m = Model(c)
    pre = SwapPreemption(c, host_budget_bytes=LAYERS * 13 * c.page_bytes)
    lens = [200, 77]
    for s, n in enumerate(lens):
        grow(c, s, n)
    slots = c.prepare_step(prefill_seq_ids=[0, 1], prefill_lens=lens)
    for layer in range(LAYERS):
        k, v = (rows((277, 8, 128), layer * 2 + i, torch.bfloat16) for i in range(2))
        c.append(layer, k.to(gpu), v.to(gpu), slots)
        m.append(0, layer, k[:200], v[:200])
        m.append(1, layer, k[200:], v[200:])
    decode_step(c, m, [0, 1], 1, True)
    assert pre.can_preempt(0)
    handle = pre.preempt(0, "r0")
    assert handle.num_bytes == LAYERS * 13 * c.page_bytes == LAYERS * 13 * (2 * 16 * 8 * 128 + 1024)
    assert not pre.can_preempt(1)
    grow(c, 3, 230)                       # takes pages, some of them the victim's
    c.append(0, rows((230, 8, 128), 9, torch.bfloat16).to(gpu),
             rows((230, 8, 128), 9, torch.bfloat16).to(gpu), c.slot_mapping([3], [230]))
    c.swap_in(handle, seq_ids=[2])
    for layer in range(LAYERS):
        m.held[2, layer] = m.held.pop((0, layer))
    for layer in range(LAYERS):
        gk, gv = c.gather(layer, [2, 1])
        assert torch.equal(gk.cpu(), torch.cat([m.values(s, layer, 0) for s in (2, 1)]))
        assert torch.equal(gv.cpu(), torch.cat([m.values(s, layer, 1) for s in (2, 1)]))
    decode_step(c, m, [1, 2], 2, False)


def test_decode_steps_replayed_from_one_graph(gpu):
    """A step's launches captured once and replayed after later prepare_decode_step calls, as
    long as decode_graph_key stays the same; every replay equals the eager step bit for bit."""
    c = make(gpu, ref.INT8, max_seqs=3)
    n0 = [5, 90, 250]
    slots = None
    for s, n in enumerate(n0):
        grow(c, s, 400)
    slots = c.prepare_step(prefill_seq_ids=[0, 1, 2], prefill_lens=n0)
    for layer in range(LAYERS):
        c.append(layer, rows((345, 2, 128), layer, torch.bfloat16).to(gpu),
                 rows((345, 2, 128), layer + 5, torch.bfloat16).to(gpu), slots)
    k, v = (torch.empty(3, 2, 128, dtype=torch.bfloat16, device=gpu) for _ in "kv")
    q = torch.empty(3, 8, 128, dtype=torch.bfloat16, device=gpu)
    outs = [torch.empty_like(q) for _ in range(LAYERS)]
    assert c.decode_graph_key() == ()

    def layers():
        for layer in range(LAYERS):
            c.append_and_decode(layer, k, v, q, out=outs[layer])

    graph = key = None
    for step in range(40):
        for i, t in enumerate((k, v, q)):
            t.copy_(rows(tuple(t.shape), step * 3 + i, torch.bfloat16))
        c.prepare_decode_step([2, 0, 1])
        if key != c.decode_graph_key():
            assert graph is None          # (nothing outgrows its buffer here)
            layers()                      # warm, outside the capture
            torch.cuda.synchronize()
            graph, key = torch.cuda.CUDAGraph(), c.decode_graph_key()
            with torch.cuda.graph(graph):
                layers()
        for t in outs:
            t.fill_(math.nan)
        graph.replay()
        got = [t.clone() for t in outs]
        for t in outs:
            t.fill_(math.nan)
        layers()
        assert all(torch.equal(a, b) for a, b in zip(got, outs)), step
        assert got[0].isfinite().all()


def test_streams(gpu):
    """Decode and prefill on another stream than their plan's are ordered after it."""
    c = make(gpu, ref.E4M3)
    m = Model(c)
    grow(c, 0, 300)
    slots = c.prepare_prefill_chunk([0], [299])
    k, v = (rows((299, 2, 128), i, torch.bfloat16) for i in range(2))
    q = rows((299, 8, 128), 5, torch.bfloat16).to(gpu)
    c.append(0, k.to(gpu), v.to(gpu), slots)
    m.append(0, 0, k, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = c.prefill(0, q, return_lse=True)
    side.synchronize()
    m.check_chunk(out, lse, q, 0, 0)
    c.prepare_decode_step([0])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        k1, v1 = (rows((1, 2, 128), 7 + i, torch.bfloat16) for i in range(2))
        out, lse = c.append_and_decode(0, k1.to(gpu), v1.to(gpu), q[:1], return_lse=True)
    m.append(0, 0, k1, v1)
    side.synchronize()
    m.check_decode(out, lse, q[:1], [0], 0)


def test_refusals(gpu):
    for kw in (dict(codec=torch.float8_e5m2), dict(codec=ref.INT8, dtype=torch.float32),
               dict(codec=ref.INT8, d=96), dict(codec=ref.E4M3, group=17)):
        with pytest.raises(ValueError, match="quantised"):
            make(gpu, **kw)
    c = make(gpu, ref.E4M3)
    with pytest.raises(RuntimeError, match="track"):
        c.track_attention()
    q = torch.zeros(1, 8, 128, dtype=torch.bfloat16, device=gpu)
    with pytest.raises(RuntimeError, match="planned"):
        c.decode(0, q)
    with pytest.raises(RuntimeError, match="plan_prefill"):
        c.prefill(0, q)
    with pytest.raises(RuntimeError, match="prepare_decode_step"):
        c.append_and_decode(0, q[:, :2], q[:, :2], q)
    grow(c, 0, 20)
    c.prepare_decode_step([0])
    for bad in (q.half(), q[:, :4], q[0], q[:0]):
        with pytest.raises(RuntimeError, match="q must be"):
            c.decode(0, bad)
    with pytest.raises(RuntimeError, match="key"):
        c.append(0, q, q, torch.zeros(1, dtype=torch.int64, device=gpu))
    cpu = PagedKVCache(1, 2, 128, max_seqs=2, max_seq_len=64, kv_page_budget=4, device="cpu",
                       kv_dtype=ref.E4M3)
    cpu.ensure_pages(0, 2)
    assert cpu.seq_pages(0) == 2 and cpu.page_bytes == 2 * 16 * 2 * 128 + 256
    with pytest.raises(RuntimeError, match="GPU"):
        cpu.decode(0, q)
