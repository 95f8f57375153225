"""GPU tests of the prompt attention on scores far beyond 2^24 that are no powers of
two, where the product of a score with the scale rounds: as in 32 bits, equal scores
have equal weights and the largest takes all.  Every query's scores differ by nothing
or by more than their own rounding can hide."""
import math

import pytest
import torch

import attention_ref as ref
from gpu_offloading_amd.prompt import BatchPromptAttentionWrapper

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _attend(gpu, q, k, v, scale, dtype):
    w = BatchPromptAttentionWrapper(torch.empty(16, dtype=torch.uint8, device=gpu))
    n, hq, d = q.shape
    w.plan(torch.tensor([0, n], dtype=torch.int32), num_qo_heads=hq, num_kv_heads=k.shape[1],
           head_dim=d, sm_scale=scale, q_data_type=dtype)
    return (*w.run(q, k, v, return_lse=True), w)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype,size,scale", [
    (BF, 1.3e5, None), (BF, 3.7e6, 0.31), (BF, 1.9e12, None), (BF, 7.3e17, 0.011),
    (HF, 1.1e4, 0.7), (HF, 2.3e4, 1.7), (HF, 4.4e4, None)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("n", [37, 300, 1500])
def test_equal_scores_share_and_the_largest_takes_all(gpu, d, dtype, size, scale, sign, n):
    """Keys of four sizes, in runs of 29 tokens, so that the maximum grows on the way
    (sign 1) or is the first run's (sign -1)."""
    print("large scores", d, dtype, size, scale, sign, n, flush=True)
    q = torch.zeros(n, 1, d, dtype=dtype)
    k = torch.zeros(n, 1, d, dtype=dtype)
    q[:, 0, 3] = sign * size * (1 + torch.arange(n) % 5 / 11)
    level = torch.arange(n) // 29 % 4
    k[:, 0, 3] = size * torch.tensor([0.37, 0.53, 0.71, 0.93])[level]
    v = torch.randn(n, 1, d, generator=torch.Generator().manual_seed(n)).to(dtype)
    out, lse, w = _attend(gpu, q.to(gpu), k.to(gpu), v.to(gpu), scale, dtype)
    assert (w.schedule.num_parts > 0) == (n == 1500 and d > 64)
    out, lse = out.cpu().double(), lse.cpu().double()
    sc = d ** -0.5 if scale is None else scale
    s = q[:, 0, 3].double()[:, None] * k[:, 0, 3].double() * sc
    s = s.masked_fill(torch.arange(n) > torch.arange(n)[:, None], -math.inf)
    top = s.max(1, keepdim=True).values
    p = (s == top).double()
    # the others are further off than 2^10 and than what two roundings of a score move
    gap = (top - s.masked_fill(p.bool(), -math.inf)).min(1).values
    assert (gap > 1024 + top[:, 0].abs() * 2.0 ** -20).all()
    count = p.sum(1, keepdim=True)
    want = (p / count) @ v[:, 0].double()
    # p is 1 exactly: fp32 sums, the division, the result's rounding
    tol = (want.abs() * ref.half_step(dtype) * 1.01
           + (p / count) @ v[:, 0].double().abs() * (count + 4) * 2.0 ** -24 + 2.0 ** -25)
    ref.assert_within(out[:, 0], want, tol, "out")
    # the scale in base 2, the scaled score, the constant and the result: a step each
    wl = (top + count.log())[:, 0]
    ref.assert_within(lse[:, 0], wl, 8 * 2.0 ** -24 * (wl.abs() + 1), "lse")
