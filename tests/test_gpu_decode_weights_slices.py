"""GPU test of the decode step's attention weights for a part of a batch: index pointers
that do not begin at 0."""
import pytest
import torch

from gpu_offloading_amd import ops
from test_gpu_eviction import Pool, _check_weights, _lse, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first,last", [(1, 5), (2, 3), (4, 5), (3, 5)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_requests_behind_the_first(gpu, first, last, d):
    """Pages in front of the requests' belong to none and stay as they were."""
    lens = [200, 17, 0, 64, 300]
    print("decode weights slice", first, last, d, flush=True)
    pool = Pool(gpu, lens, 2, d, torch.bfloat16, seed=d)
    q, lse = _randn(gpu, 5, 4, d, seed=1, dtype=torch.bfloat16), _lse(gpu, 5, 4, 2)
    before = pool.scores.clone(), pool.positions.clone()
    ops.decode_attention_weights(q[first:last], lse[first:last], pool.kc,
                                 pool.indptr[first:last + 1].clone(), pool.indices,
                                 pool.lpl[first:last].clone(), pool.scores, pool.positions)
    torch.cuda.synchronize()
    one = [int(first <= b < last and n > 0) for b, n in enumerate(lens)]
    rows = [b for b in range(5) if one[b]]
    _check_weights(pool, before, q[rows], lse[rows], one, one, True, [0] * 5, d ** -0.5)
