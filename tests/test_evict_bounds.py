"""CPU test: bounds on the sequence lengths that a 32-bit integer does not hold are
refused, not cut to their lower bits."""
import pytest

from gpu_offloading_amd import ops


@pytest.mark.parametrize("bound", [2 ** 31, 2 ** 32, 2 ** 32 + 5, -1, -2 ** 40])
def test_max_seq_len_beyond_32_bits(bound):
    with pytest.raises(RuntimeError, match="max_seq_len"):
        ops.evict_workspace_bytes(2, 3, bound)


def test_max_seq_len_within():
    assert ops.evict_workspace_bytes(2, 3, 0) == 0
    assert ops.evict_workspace_bytes(2, 3, 100) == 2 * 3 * (1 + 2 * 50) * 4
    assert ops.evict_workspace_bytes(1, 1, 2 ** 31 - 1) > 2 ** 32
