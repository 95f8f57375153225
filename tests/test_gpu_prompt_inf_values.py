"""GPU tests of the prompt attention on infinities in values that a query sees: inf where
the value's weight is above 0, NaN where the weight vanishes (0 times inf), on the causal
edge as in the tiles that all rows see, whole units and pieces alike."""
import math

import pytest
import torch

from gpu_offloading_amd.prompt import BatchPromptAttentionWrapper

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,at", [(90, 70), (400, 70), (400, 399), (2200, 1500)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
def test_weights_that_vanish_and_that_do_not(gpu, d, dtype, n, at, bad):
    """Token `at` has a score 300 below the others' for one query head and the same for
    the other: the weight of the first vanishes in every row with another key."""
    print("inf values", d, dtype, n, at, bad, flush=True)
    q = torch.zeros(n, 2, d, dtype=dtype)
    k = torch.zeros(n, 1, d, dtype=dtype)
    q[:, 0, 1] = d ** 0.5 if d != 128 else 11.3125
    k[at, 0, 1] = -300.0
    g = torch.Generator().manual_seed(n)
    v = torch.randn(n, 1, d, generator=g).to(dtype)
    w = BatchPromptAttentionWrapper(torch.empty(16, dtype=torch.uint8, device=gpu))
    w.plan(torch.tensor([0, n], dtype=torch.int32), num_qo_heads=2, num_kv_heads=1, head_dim=d,
           q_data_type=dtype)
    q, k, v = q.to(gpu), k.to(gpu), v.to(gpu)
    clean = w.run(q, k, v)
    v[at, 0, 5] = bad
    out = w.run(q, k, v)
    torch.cuda.synchronize()
    want = clean.clone()
    want[at:, 0, 5] = math.nan
    want[at:, 1, 5] = bad
    assert torch.equal(torch.nan_to_num(out.float(), 1e9, 2e9, -2e9),
                       torch.nan_to_num(want.float(), 1e9, 2e9, -2e9))
