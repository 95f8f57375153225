"""GPU tests of the prompt attention (csrc/prompt.hip) against attention in 64
bits: element types, head dims and groups, lengths from nothing to several key
tiles, strided inputs, rows that see no key, inf and NaN where a query does not
look, streams and graphs.  The tolerances are the error bounds of
attention_ref.attention."""
import math

import pytest
import torch

import attention_ref as ref
from gpu_offloading_amd.prompt import BatchPromptAttentionWrapper

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _wrapper(gpu):
    return BatchPromptAttentionWrapper(torch.empty(16, dtype=torch.uint8, device=gpu))


def _randn(gpu, *shape, seed, dtype, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(gpu)


def _check(out, lse, q, k, v, qlens, kvlens, causal, scale):
    qa, ka = ref.cumulative(qlens), ref.cumulative(kvlens)
    for b, (m, n) in enumerate(zip(qlens, kvlens)):
        qs, ks = slice(qa[b], qa[b + 1]), slice(ka[b], ka[b + 1])
        o, l, otol, ltol = ref.attention(q[qs], k[ks], v[ks], n - m, causal, scale)
        ref.assert_within(out[qs], o, otol, f"sequence {b} ({m}, {n}) out")
        ref.assert_within(lse[qs], l, ltol, f"sequence {b} ({m}, {n}) lse")


def _run(gpu, qlens, kvlens, hkv, group, d, dtype, causal, seed, std=1.0):
    print("prompt", qlens, kvlens, hkv, group, d, dtype, causal, flush=True)
    q = _randn(gpu, sum(qlens) + 3, hkv * group, d, seed=seed, dtype=dtype, std=std)
    k = _randn(gpu, sum(kvlens) + 1, hkv, d, seed=seed + 1, dtype=dtype)
    v = _randn(gpu, sum(kvlens) + 1, hkv, d, seed=seed + 2, dtype=dtype)
    w = _wrapper(gpu)
    w.plan(torch.tensor(ref.cumulative(qlens), dtype=torch.int32),
           torch.tensor(ref.cumulative(kvlens), dtype=torch.int32), num_qo_heads=hkv * group,
           num_kv_heads=hkv, head_dim=d, causal=causal, q_data_type=dtype)
    out = torch.full_like(q, 7.0)
    lse = torch.full((q.shape[0], hkv * group), 7.0, device=gpu)
    w.run(q, k, v, out=out, lse=lse)
    torch.cuda.synchronize()
    # rows behind the last sequence stay as they were
    assert (out[sum(qlens):] == 7).all() and (lse[sum(qlens):] == 7).all()
    _check(out, lse, q, k, v, qlens, kvlens, causal, d ** -0.5)
    return q, k, v, out, lse, w


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("causal", [True, False])
def test_dims_and_types(gpu, d, dtype, causal):
    lens = [1, 63, 64, 65, 0, 2, 130, 17]
    _run(gpu, lens, lens, 2, 4, d, dtype, causal, seed=d)


@pytest.mark.parametrize("hkv,group", [(1, 1), (3, 2), (1, 3), (2, 5), (1, 8), (1, 12), (1, 32),
                                       (1, 100), (1, 128), (5, 1)])
def test_groups(gpu, hkv, group):
    lens = [5, 40, 1, 77]
    _run(gpu, lens, lens, hkv, group, 128 if group < 9 else 64, BF, True, seed=group)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_long_enough_for_interior_tiles(gpu, d):
    lens = [513, 700, 257]
    _run(gpu, lens, lens, 1, 2, d, BF, True, seed=3, std=3.0)


def test_queries_and_keys_of_other_lengths(gpu):
    """More keys than queries (the last queries of a longer history), fewer
    (the first queries see nothing and give 0 and -inf), none at all."""
    q, k, v, out, lse, _ = _run(gpu, [5, 9, 3, 0, 70], [100, 4, 0, 8, 65], 2, 3, 64, BF, True, 11)
    assert (out[5:10] == 0).all() and (lse[5:10] == -math.inf).all()
    assert (out[14:17] == 0).all() and (lse[14:17] == -math.inf).all()
    _run(gpu, [5, 9, 3, 0, 70], [100, 4, 0, 8, 65], 2, 3, 128, BF, False, 12)


def test_slices_of_a_fused_projection(gpu):
    hq, hkv, d, lens = 8, 2, 128, [100, 33]
    qkv = _randn(gpu, 133, hq + 2 * hkv, d, seed=4, dtype=BF)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    w = _wrapper(gpu)
    w.plan(torch.tensor([0, 100, 133], dtype=torch.int32, device=gpu), num_qo_heads=hq,
           num_kv_heads=hkv, head_dim=d)
    wide = torch.full((133, hq + 2, d), 3.0, dtype=BF, device=gpu)
    out, lse = w.run(q, k, v, out=wide[:, 1:-1], return_lse=True)
    _check(out, lse, q, k, v, lens, lens, True, d ** -0.5)
    assert (wide[:, 0] == 3).all() and (wide[:, -1] == 3).all()
    again = w.run(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(again, out)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_a_query_does_not_feel_what_it_does_not_see(gpu, d, bad, dtype):
    """A key and a value that are not finite, at token 70 of 150 (inside a
    boundary tile of the queries around it) and in the last token: queries before
    it are as without it; queries from it on see it."""
    n, hq, hkv = 150, 4, 2
    q = _randn(gpu, n, hq, d, seed=1, dtype=dtype)
    k = _randn(gpu, n, hkv, d, seed=2, dtype=dtype)
    v = _randn(gpu, n, hkv, d, seed=3, dtype=dtype)
    w = _wrapper(gpu)
    w.plan(torch.tensor([0, n], dtype=torch.int32), num_qo_heads=hq, num_kv_heads=hkv, head_dim=d,
           q_data_type=dtype)
    clean, clean_lse = w.run(q, k, v, return_lse=True)
    v2 = v.clone()
    v2[70, 0, 5] = bad
    v2[149, 1, d - 1] = bad
    out, lse = w.run(q, k, v2, return_lse=True)
    want = clean.clone()
    want[70:, :2, 5] = bad            # KV head 0 serves query heads 0 and 1
    want[149:, 2:, d - 1] = bad
    assert torch.equal(torch.nan_to_num(out.float(), 1e9, 2e9, -2e9),
                       torch.nan_to_num(want.float(), 1e9, 2e9, -2e9))
    assert torch.equal(lse, clean_lse)
    k2 = k.clone()
    k2[70] = bad
    out = w.run(q, k2, v)
    assert torch.equal(out[:70], clean[:70])


def test_not_finite_in_a_tile_that_all_rows_see(gpu):
    """Values that are not finite in an interior tile reach every query behind it."""
    n = 300
    q, k, v = (_randn(gpu, n, 1, 64, seed=s, dtype=BF) for s in (1, 2, 3))
    v[3, 0, 7] = math.inf
    w = _wrapper(gpu)
    w.plan(torch.tensor([0, n], dtype=torch.int32), num_qo_heads=1, num_kv_heads=1, head_dim=64)
    out = w.run(q, k, v)
    assert torch.isfinite(out[:3]).all() and (out[3:, 0, 7] == math.inf).all()
    assert torch.isfinite(out[:, 0, :7]).all() and torch.isfinite(out[:, 0, 8:]).all()


def test_scores_of_any_finite_size(gpu):
    """Rows whose scores are all far below or above 0, up to the type's largest
    values: the softmax only depends on their differences."""
    n, d = 40, 128
    q = torch.zeros(n, 1, d, dtype=BF, device=gpu)
    k = torch.zeros(n, 1, d, dtype=BF, device=gpu)
    v = _randn(gpu, n, 1, d, seed=3, dtype=BF)
    q[:, :, 0] = 2.0 ** 60
    k[:, 0, 0] = -2.0 ** 60
    k[7, 0, 0] = -2.0 ** 59       # every query that sees key 7 attends to it alone
    w = _wrapper(gpu)
    w.plan(torch.tensor([0, n], dtype=torch.int32), num_qo_heads=1, num_kv_heads=1, head_dim=d)
    out, lse = w.run(q, k, v, return_lse=True)
    assert torch.equal(out[7:], v[7].expand(n - 7, 1, d))
    mean = v[:7].double().cumsum(0) / torch.arange(1, 8, device=gpu)[:, None, None]
    # p = 1 exactly, so: fp32 sums, one rounding of the result
    assert ((out[:7].double() - mean).abs() <= mean.abs() * 2.0 ** -8 + 2.0 ** -20).all()
    assert torch.isfinite(lse).all() and (lse < -2.0 ** 115).all()


def test_another_stream_and_one_plan_for_many_runs(gpu):
    lens = [200, 31]
    q, k, v, out, lse, w = _run(gpu, lens, lens, 2, 2, 128, BF, True, seed=21)
    q2 = _randn(gpu, *q.shape, seed=99, dtype=BF)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = w.run(q2, k, v)
    explicit = w.run(q, k, v, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(explicit, out[:231])
    assert torch.equal(got, w.run(q2, k, v))


def test_captured_and_replayed(gpu):
    lens = [90, 160]
    q, k, v, out, lse, w = _run(gpu, lens, lens, 1, 4, 64, HF, True, seed=31)
    gout, glse = torch.empty_like(out), torch.empty_like(lse)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w.run(q, k, v, out=gout, lse=glse)
    for seed in (1, 2, 3):
        q.copy_(_randn(gpu, *q.shape, seed=seed, dtype=HF))
        g.replay()
        want, wl = w.run(q, k, v, return_lse=True)
        torch.cuda.synchronize()
        assert torch.equal(gout[:250], want) and torch.equal(glse[:250], wl)


def test_many_sequences_and_a_longer_one(gpu):
    """More units than workgroups, one sequence of 2500 tokens among short ones."""
    g = torch.Generator().manual_seed(8)
    lens = torch.randint(0, 60, (80,), generator=g).tolist() + [2500]
    q = _randn(gpu, sum(lens), 8, 64, seed=5, dtype=BF)
    k = _randn(gpu, sum(lens), 4, 64, seed=6, dtype=BF)
    v = _randn(gpu, sum(lens), 4, 64, seed=7, dtype=BF)
    w = _wrapper(gpu)
    w.plan(torch.tensor(ref.cumulative(lens), dtype=torch.int32), num_qo_heads=8, num_kv_heads=4,
           head_dim=64)
    out, lse = w.run(q, k, v, return_lse=True)
    _check(out, lse, q, k, v, lens[:80], lens[:80], True, 0.125)
    at = sum(lens[:80])
    for i in (0, 1, 63, 64, 1000, 2499):
        o, l, otol, ltol = ref.attention(q[at + i:at + i + 1], k[at:at + i + 1], v[at:at + i + 1],
                                         i, True, 0.125)
        ref.assert_within(out[at + i:at + i + 1], o, otol, f"row {i}")
        ref.assert_within(lse[at + i:at + i + 1], l, ltol, f"row {i} lse")


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("qlens,kvlens,causal", [
    ([2100], [2100], True), ([700, 1], [1900, 1], False), ([1700], [1300], True),
    ([2900], [2400], True)])
def test_keys_of_few_units_in_pieces(gpu, d, dtype, qlens, kvlens, causal):
    """Few query tiles over many keys: pieces of them joined, in the same order every
    time; queries that see no key, or none of a piece, among them."""
    q, k, v, out, lse, w = _run(gpu, qlens, kvlens, 1, 3, d, dtype, causal, seed=d)
    assert w.schedule.num_parts > 0 or (d == 64 and kvlens == [1300])
    again, l2 = w.run(q, k, v, return_lse=True)
    assert torch.equal(again, out[:sum(qlens)]) and torch.equal(l2, lse[:sum(qlens)])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_pieces_of_keys_that_are_not_finite(gpu, d, bad):
    """In a late key's K or V they reach the queries that see it and no other."""
    n, at = 2200, 1500
    q = _randn(gpu, n, 2, d, seed=1, dtype=BF)
    k, v = (_randn(gpu, n, 1, d, seed=i, dtype=BF) for i in (2, 3))
    w = _wrapper(gpu)
    w.plan(torch.tensor([0, n], dtype=torch.int32), num_qo_heads=2, num_kv_heads=1, head_dim=d)
    assert w.schedule.num_parts > 0
    want, wl = w.run(q, k, v, return_lse=True)
    v[at, 0, 5] = bad
    got, gl = w.run(q, k, v, return_lse=True)
    assert torch.equal(got[:at], want[:at]) and torch.equal(gl, wl)
    assert not torch.isfinite(got[at:, :, 5]).any()
    rest = [i for i in range(d) if i != 5]
    assert torch.equal(got[:, :, rest], want[:, :, rest])
    k[at, 0, 5] = math.nan
    got, gl = w.run(q, k, v, return_lse=True)
    assert torch.equal(got[:at], want[:at]) and torch.equal(gl[:at], wl[:at])
    assert torch.isnan(got[at:]).all() and torch.isnan(gl[at:]).all()


def test_pieces_captured_and_replayed(gpu):
    q, k, v, out, lse, w = _run(gpu, [1500], [1500], 1, 4, 128, BF, True, seed=5)
    assert w.schedule.num_parts > 0
    outs = [torch.empty_like(out) for _ in range(2)]
    graphs = []
    for o in outs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            w.run(q, k, v, out=o)
    for seed in (1, 2, 3):
        q.copy_(_randn(gpu, *q.shape, seed=seed, dtype=BF))
        for g in graphs:
            g.replay()
        want = w.run(q, k, v)
        torch.cuda.synchronize()
        assert all(torch.equal(o[:1500], want) for o in outs)
