"""GPU tests of the attention weights' chunk form where its rows are cut into pieces at
large groups, with NaN in the tokens in front of and behind the queries and their
log-sum-exp: a row read past its unit's tokens would show (tests/test_weights_rows.py
proves the addresses on the CPU first).  Reference and tolerances as in
test_gpu_eviction.py."""
import math

import pytest
import torch

import attention_ref as ref
from gpu_offloading_amd.eviction import BatchAttentionWeightsWrapper
from test_gpu_eviction import Pool, _check_weights, _lse, _randn

pytestmark = pytest.mark.gpu


def _spaced(gpu, x):
    """x between two tokens of NaN."""
    wide = torch.full((x.shape[0] + 4, *x.shape[1:]), math.nan, dtype=x.dtype, device=gpu)
    wide[2:-2] = x
    return wide[2:-2]


@pytest.mark.parametrize("group,d,qlens,causal", [
    *((g, d, [129], True) for g in (32, 64, 96, 128) for d in (64, 128, 256)),
    (64, 128, [777], True), (64, 256, [300, 250], False), (96, 64, [777], True),
    (48, 64, [40, 129], True), (128, 64, [333], False)])
def test_pieces_of_large_groups(gpu, group, d, qlens, causal):
    print("weights pieces", group, d, qlens, causal, flush=True)
    lens = [n + 9 * i for i, n in enumerate(qlens)]
    pool = Pool(gpu, lens, 1, d, torch.bfloat16, seed=group)
    q = _spaced(gpu, _randn(gpu, sum(qlens), group, d, seed=1, dtype=torch.bfloat16))
    lse = _spaced(gpu, _lse(gpu, sum(qlens), group, 2))
    w = BatchAttentionWeightsWrapper(torch.empty(16, dtype=torch.uint8, device=gpu))
    w.plan(torch.tensor(ref.cumulative(qlens), dtype=torch.int32), pool.indptr.cpu(), pool.indices,
           pool.lpl.cpu(), group, 1, d, 16, causal=causal)
    assert w.schedule.num_parts > 0
    before = pool.scores.clone(), pool.positions.clone()
    w.run(q, lse, pool.kc, pool.scores, pool.positions)
    torch.cuda.synchronize()
    _check_weights(pool, before, q, lse, qlens, qlens, causal, [0] * len(lens), d ** -0.5)
