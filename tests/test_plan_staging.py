"""CPU test of the pinned memory that the planning wrappers ask for: bounded whatever
the index pointers hold, as these are only checked by the plan function itself."""
import pytest
import torch

from gpu_offloading_amd.prompt import BatchPromptAttentionWrapper


@pytest.mark.parametrize("ends,heads", [([0, 2 ** 31 - 1], 128), ([0, 5, 2 ** 31 - 1], 8),
                                        ([0, 2 ** 20], 128)])
def test_a_plan_stages_little_before_its_size_is_known(monkeypatch, ends, heads):
    sizes = []

    def empty(n, dtype, pin_memory):
        sizes.append(n)
        if len(sizes) == 2:
            raise MemoryError            # the second one is what the plan asked for
        assert n <= 1 << 22 and pin_memory
        return torch.zeros(n, dtype=dtype)
    monkeypatch.setattr(torch, "empty", empty)
    w = object.__new__(BatchPromptAttentionWrapper)
    w._device = torch.device("cpu")
    with pytest.raises((RuntimeError, MemoryError)):
        w.plan(torch.tensor(ends, dtype=torch.int32), num_qo_heads=heads, num_kv_heads=1,
               head_dim=64)
    assert (len(sizes) == 2) == (ends[-1] == 2 ** 20)    # refused, but for the last
