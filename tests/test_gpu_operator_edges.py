"""GPU tests of the prompt attention, the attention weights and the eviction in
calls that their own files do not make: work shared out in many small pieces,
other streams and plans, graphs beside each other, places past 2^32 bytes, short
position offsets, bounds of nothing, and refused arguments.  References and
tolerances as there."""
import pytest
import torch

import attention_ref as ref
from gpu_offloading_amd import ops
from gpu_offloading_amd.eviction import BatchAttentionWeightsWrapper
from gpu_offloading_amd.prompt import BatchPromptAttentionWrapper
from test_gpu_eviction import Pool, _check_weights, _chunk, _evict, _lse, _randn

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _ints(gpu, x):
    return torch.tensor(x, dtype=torch.int32, device=gpu)


def _prompt(gpu):
    return BatchPromptAttentionWrapper(torch.empty(16, dtype=torch.uint8, device=gpu))


@pytest.mark.parametrize("short", [150, 420])
@pytest.mark.parametrize("d,group", [(64, 4), (128, 4), (128, 3), (256, 2)])
def test_workgroups_with_several_pieces(gpu, d, group, short):
    """A long prompt among many short ones: its key tiles are cut, and with enough of
    them a workgroup walks pieces of several requests."""
    lens = [1900] + [40 + 37 * (i % 7) for i in range(short)]
    pool, q, lse, w = _chunk(gpu, lens, [1900] + [min(n, 33) for n in lens[1:]], 2, group, d, BF,
                             seed=d + group)
    assert w.schedule.num_parts > 0
    assert short == 150 or w.schedule.num_units > w.schedule.num_workgroups
    got = []
    for _ in range(2):
        s = torch.zeros_like(pool.scores)
        got.append(w.run(q, lse, pool.kc, s))
    assert torch.equal(*got)


def test_chunk_weights_on_another_stream_and_after_another_plan(gpu):
    pool, q, lse, w = _chunk(gpu, [900, 70], [900, 9], 1, 8, 128, BF, seed=3)
    assert w.schedule.num_parts > 0                        # a workspace is used
    want = w.run(q, lse, pool.kc, torch.zeros_like(pool.scores))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        inside = w.run(q, lse, pool.kc, torch.zeros_like(pool.scores))
    zero = torch.zeros_like(pool.scores)
    s.wait_stream(torch.cuda.current_stream())
    named = w.run(q, lse, pool.kc, zero, stream=s)
    w.plan(torch.tensor([0, 5, 9], dtype=torch.int32), pool.indptr.cpu(), pool.indices,
           pool.lpl.cpu(), 8, 1, 128, 16)
    before = pool.scores.clone(), pool.positions.clone()
    w.run(q, lse, pool.kc, pool.scores, pool.positions)
    torch.cuda.synchronize()
    assert torch.equal(inside, want) and torch.equal(named, want)
    _check_weights(pool, before, q, lse, [5, 4], [5, 4], True, [0, 0], 128 ** -0.5)


def test_two_captured_runs_replayed_in_turn(gpu):
    """Two graphs of one plan, each with partial sums of its own, eager runs between."""
    pool, q, lse, w = _chunk(gpu, [800], [800], 1, 8, 64, HF, seed=5)
    assert w.schedule.num_parts > 0
    qs = [_randn(gpu, *q.shape, seed=i, dtype=HF) for i in (1, 2)]
    outs = [torch.zeros_like(pool.scores) for _ in qs]
    graphs = []
    for x, o in zip(qs, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            w.run(x, lse, pool.kc, o)
    for turn in range(3):
        for i in (0, 1):
            qs[i].copy_(_randn(gpu, *q.shape, seed=10 * turn + i, dtype=HF))
        for g in graphs:
            g.replay()
        for x, o in zip(qs, outs):
            assert torch.equal(o, w.run(x, lse, pool.kc, torch.zeros_like(pool.scores)))


def test_decode_weights_on_another_stream_and_short_offsets(gpu):
    """A sequence without an entry in position_offsets counts as never evicted."""
    lens = [30, 1, 77]
    pool = Pool(gpu, lens, 2, 128, BF, seed=4)
    q, lse = _randn(gpu, 3, 4, 128, seed=1, dtype=BF), _lse(gpu, 3, 4, 2)
    before = pool.scores.clone(), pool.positions.clone()
    s = torch.cuda.Stream()
    args = _ints(gpu, [5, 6]), _ints(gpu, [1, 2, -1])
    s.wait_stream(torch.cuda.current_stream())
    ops.decode_attention_weights(q, lse, pool.kc, pool.indptr, pool.indices, pool.lpl, pool.scores,
                                 pool.positions, args[0], seq_ids=args[1], stream=s)
    torch.cuda.synchronize()
    _check_weights(pool, before, q, lse, [1] * 3, [1] * 3, True, [6, 0, 0], 128 ** -0.5)
    pool.scores.copy_(before[0])
    pool.positions.copy_(before[1])
    w = BatchAttentionWeightsWrapper(torch.empty(16, dtype=torch.uint8, device=gpu))
    w.plan(torch.tensor([0, 1, 2, 3], dtype=torch.int32), pool.indptr.cpu(), pool.indices,
           pool.lpl.cpu(), 4, 2, 128, 16)
    w.run(q, lse, pool.kc, pool.scores, pool.positions, *args)
    _check_weights(pool, before, q, lse, [1] * 3, [1] * 3, True, [6, 0, 0], 128 ** -0.5)


def test_evict_to_nothing_and_on_another_stream(gpu):
    lens = [40, 17, 0, 5]
    pool = Pool(gpu, lens, 2, 64, BF, seed=6)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    assert _evict(gpu, pool, [0, 1, 0, 5], [0, 1, 0, 5], False, None, stream=s) > 0
    ops.evict_kv(pool.kc, pool.vc, pool.scores, pool.table[:0], *(_ints(gpu, []) for _ in range(3)), 0)


def test_nothing_to_do(gpu):
    """Empty batches, and requests without tokens, leave everything as it is."""
    pool = Pool(gpu, [0, 20, 0], 1, 64, BF, seed=8)
    scores = pool.scores.clone()
    q, lse = _randn(gpu, 4, 2, 64, seed=1, dtype=BF), _lse(gpu, 4, 2, 2)
    ops.decode_attention_weights(q[:0], lse[:0], pool.kc, pool.indptr[:1], pool.indices,
                                 pool.lpl[:0], pool.scores)
    ops.decode_attention_weights(q[:2], lse[:2], pool.kc, _ints(gpu, [0, 0, 0]), pool.indices,
                                 _ints(gpu, [0, 0]), pool.scores)
    w = BatchAttentionWeightsWrapper(torch.empty(16, dtype=torch.uint8, device=gpu))
    for qo, kv, lpl in (([0], [0], []), ([0, 0, 0, 0], [0, 0, 2, 2], [0, 4, 0])):
        w.plan(*(torch.tensor(x, dtype=torch.int32) for x in (qo, kv)), pool.indices,
               torch.tensor(lpl, dtype=torch.int32), 2, 1, 64, 16)
        w.run(q, lse, pool.kc, pool.scores)
    assert torch.equal(pool.scores, scores)
    p = _prompt(gpu)
    for ip in ([0], [0, 0, 0]):
        p.plan(torch.tensor(ip, dtype=torch.int32), num_qo_heads=2, num_kv_heads=1, head_dim=64)
        out, l = p.run(q[:0], q[:0, :1], q[:0, :1], return_lse=True)
        assert out.shape == (0, 2, 64) and l.shape == (0, 2)


@pytest.fixture(scope="module")
def big(gpu):
    """A layer past 4 GiB; scores and positions as large as it needs."""
    pages = 72_000
    kv = torch.empty(pages, 2, 16, 8, 128, dtype=BF, device=gpu)
    assert kv.numel() * 2 > 1 << 32
    yield kv
    del kv
    torch.cuda.empty_cache()


def test_a_cache_past_4_gib(gpu, big):
    """Pages at both ends of the layer through both forms and the eviction, beside
    the same tokens in a small one."""
    small = Pool(gpu, [300, 90], 8, 128, BF, seed=11)
    n, pages = small.kc.shape[0], big.shape[0]
    place = torch.tensor([0, pages - 1] + list(range(66_000, 66_000 + n - 2)), device=gpu)
    big[place, 0], big[place, 1] = small.kc, small.vc
    scores = torch.zeros(pages, 8, 16, device=gpu)
    positions = torch.zeros(pages, 8, 16, dtype=torch.int32, device=gpu)
    scores[place], positions[place] = small.scores, small.positions
    indices = place[small.indices.long()].int()
    table = torch.where(small.table >= 0, place[small.table.clamp(min=0).long()].int(), small.table)
    q, lse = _randn(gpu, 340, 32, 128, seed=1, dtype=BF), _lse(gpu, 340, 32, 2)
    w = BatchAttentionWeightsWrapper(torch.empty(16, dtype=torch.uint8, device=gpu))
    for kc, vc, sc, ps, idx, tab in ((small.kc, small.vc, small.scores, small.positions,
                                      small.indices, small.table),
                                     (big[:, 0], big[:, 1], scores, positions, indices, table)):
        w.plan(torch.tensor([0, 300, 340], dtype=torch.int32), small.indptr.cpu(), idx,
               small.lpl.cpu(), 32, 8, 128, 16, new_tokens=torch.tensor([300, 90],
                                                                        dtype=torch.int32))
        w.run(q, lse, kc, sc, ps)
        ops.decode_attention_weights(q[:2], lse[:2], kc, small.indptr, idx, small.lpl, sc, ps)
        ops.evict_kv(kc, vc, sc, tab, _ints(gpu, [300, 90]), _ints(gpu, [128, 40]),
                     _ints(gpu, [16, 8]), 300, ps)
    torch.cuda.synchronize()
    assert torch.equal(scores[place], small.scores)
    assert torch.equal(positions[place], small.positions)
    assert torch.equal(big[place, 0], small.kc) and torch.equal(big[place, 1], small.vc)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompt_tokens_4_mib_apart(gpu, d):
    """K, V, Q and the output past 2^32 bytes from their first token."""
    lens, step = [700, 450], 1 << 21
    n = sum(lens)
    print("prompt far", d, flush=True)

    def far(heads, seed):
        x = torch.empty(n * step, dtype=BF, device=gpu).as_strided((n, heads, d), (step, d, 1))
        x.copy_(_randn(gpu, n, heads, d, seed=seed, dtype=BF))
        return x
    q, k, v, out = far(2, 1), far(1, 2), far(1, 3), far(2, 4)
    w = _prompt(gpu)
    w.plan(torch.tensor(ref.cumulative(lens), dtype=torch.int32), num_qo_heads=2, num_kv_heads=1,
           head_dim=d)
    _, lse = w.run(q, k, v, out=out, return_lse=True)
    want, wl = w.run(*(x.contiguous() for x in (q, k, v)), return_lse=True)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, wl)


def test_refused_arguments(gpu):
    pool = Pool(gpu, [40], 2, 128, BF, seed=1)
    q, lse = _randn(gpu, 1, 4, 128, seed=1, dtype=BF), _lse(gpu, 1, 4, 2)

    def decode(**kw):
        a = dict(q=q, lse=lse, key_cache=pool.kc, indptr=pool.indptr, indices=pool.indices,
                 last_page_len=pool.lpl, scores=pool.scores, positions=pool.positions)
        ops.decode_attention_weights(**{**a, **kw})
    w = BatchAttentionWeightsWrapper(torch.empty(16, dtype=torch.uint8, device=gpu))
    with pytest.raises(RuntimeError, match="before plan"):
        w.run(q, lse, pool.kc, pool.scores)
    w.plan(torch.tensor([0, 1], dtype=torch.int32), pool.indptr.cpu(), pool.indices,
           pool.lpl.cpu(), 4, 2, 128, 16)

    def chunk(**kw):
        a = dict(q=q, lse=lse, k_cache=pool.kc, scores=pool.scores, positions=pool.positions)
        kw = {{"key_cache": "k_cache"}.get(k, k): v for k, v in kw.items()}
        w.run(**{**a, **kw})
    wide = torch.zeros(1, 4, 256, dtype=BF, device=gpu)
    for call in (decode, chunk):
        for bad in (dict(q=q.half()), dict(q=q.float()), dict(q=wide[:, :, ::2]), dict(q=q.cpu()),
                    dict(lse=lse.half()), dict(lse=lse[:, :2]), dict(lse=lse[:0]),
                    dict(key_cache=pool.kc[:, :8]), dict(key_cache=pool.kc.half()),
                    dict(scores=pool.scores[:-1]), dict(scores=pool.scores.double()),
                    dict(scores=pool.scores.cpu()), dict(positions=pool.scores),
                    dict(position_offsets=_ints(gpu, [])), dict(seq_ids=_ints(gpu, [])),
                    dict(seq_ids=torch.zeros(1, dtype=torch.int64, device=gpu))):
            with pytest.raises(RuntimeError):
                call(**bad)
    with pytest.raises(RuntimeError):
        decode(indptr=pool.indptr.long())
    with pytest.raises(RuntimeError):
        decode(indptr=pool.indptr[:1])
    with pytest.raises(RuntimeError):
        decode(sm_scale=float("nan"))
    one = [_ints(gpu, [x]) for x in (40, 16, 4)]

    def evict(**kw):
        a = dict(key_cache=pool.kc, value_cache=pool.vc, scores=pool.scores, block_table=pool.table,
                 seq_lens=one[0], keep=one[1], recent=one[2], max_seq_len=40)
        ops.evict_kv(**{**a, **kw})
    for bad in (dict(value_cache=pool.vc.half()), dict(value_cache=pool.vc[:-1]),
                dict(scores=pool.scores[:, :1]), dict(positions=pool.scores),
                dict(block_table=pool.table.long()), dict(block_table=pool.table[:0]),
                dict(block_table=pool.table.t()), dict(keep=one[1].long()),
                dict(recent=_ints(gpu, [])), dict(seq_ids=_ints(gpu, [])), dict(max_seq_len=-1),
                dict(workspace=torch.empty(8, dtype=torch.uint8, device=gpu))):
        with pytest.raises(RuntimeError):
            evict(**bad)
    p = _prompt(gpu)
    k = _randn(gpu, 5, 2, 128, seed=2, dtype=BF)
    q5 = _randn(gpu, 5, 4, 128, seed=3, dtype=BF)
    with pytest.raises(RuntimeError, match="before plan"):
        p.run(q5, k, k)
    ip = torch.tensor([0, 5], dtype=torch.int32)
    for kw in (dict(num_qo_heads=5, num_kv_heads=2, head_dim=128),
               dict(num_qo_heads=4, num_kv_heads=2, head_dim=96),
               dict(num_qo_heads=258, num_kv_heads=2, head_dim=64),
               dict(num_qo_heads=4, num_kv_heads=2, head_dim=128, q_data_type=torch.float32)):
        with pytest.raises(RuntimeError):
            p.plan(ip, **kw)
    p.plan(ip, num_qo_heads=4, num_kv_heads=2, head_dim=128)
    for bad in ((q5[:4], k, k), (q5, k[:4], k), (q5, k, k[:4]), (q5.half(), k, k), (q5, k.half(), k),
                (q5[:, :2], k, k), (q5, k.cpu(), k), (q5.cpu(), k, k)):
        with pytest.raises(RuntimeError):
            p.run(*bad)
    with pytest.raises(RuntimeError):
        p.run(q5, k, k, out=torch.empty_like(q5[:4]))
    with pytest.raises(RuntimeError):
        p.run(q5, k, k, lse=torch.empty(5, 4, device=gpu, dtype=BF))
