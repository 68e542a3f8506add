"""Host side of the matching operators at the edges of what the documentation allows, without a GPU."""
import pytest
import torch

from custereomatching_amd import matching

CPU = torch.device("cpu")


@pytest.mark.parametrize("name", ["key_lengths", "query_offset"])
def test_positions_of_64_bits_keep_their_order(name):
    """Beyond 32 bits they become the nearest 32-bit number, not their low half."""
    top, low = (1 << 31) - 1, -(1 << 31)
    far = [1 << 31, (1 << 32) + 5, (1 << 40) + 5, (1 << 63) - 1, top, 7, 0, -1, low, low - 1, -(1 << 32), -(1 << 63)]
    got = matching._index_tensor(torch.tensor(far), name, len(far), CPU)
    assert got.dtype == torch.int32 and got.tolist() == [top] * 5 + [7, 0, -1] + [low] * 4


def test_tangents_are_refused():
    import torch.autograd.forward_ad as fw

    x = torch.ones(3)
    matching._no_tangent(x, x)
    with fw.dual_level():
        matching._no_tangent(x)
        with pytest.raises(RuntimeError, match="forward-mode"):
            matching._no_tangent(x, fw.make_dual(x, x))
