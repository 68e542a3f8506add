"""Host side of the matching operators at the edges of what the documentation allows, without a GPU."""
import ctypes

import pytest
import torch

from custereomatching_amd import _lib, matching
from tests.test_matching_host import err, geo

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


def test_strides_that_the_kernels_do_not_take_are_copied():
    """Key and value positions from 2^24 elements apart; query positions and heads only where a backward reads them."""
    far = torch.zeros((3, 1 << 24), dtype=torch.float16)[:, :8].reshape(3, 8).as_strided((1, 3, 1, 8), (0, 1 << 24, 0, 1))
    far[0, 1] = 3.0
    got = matching._rows16(far, matching._NEAR_POSITIONS)
    assert got.stride(1) == 8 and torch.equal(got, far)
    assert matching._rows16(far) is far and matching._rows16(far[:, :1], matching._NEAR_POSITIONS).data_ptr() == far.data_ptr()
    heads = torch.zeros((1, 2, 1 << 18, 64), dtype=torch.float16).transpose(1, 2)[:, :5]  # [B, L, heads, C] of [B, heads, L, C]
    assert heads.stride(2) == 1 << 24
    assert matching._rows16(heads, matching._NEAR_POSITIONS) is heads
    assert matching._rows16(heads, matching._NEAR_HEADS).is_contiguous()


def test_far_strides_at_the_c_entry():
    for op, kw, ok in [(0, dict(q_stride=[0, 1 << 24, 1 << 24]), True), (1, dict(q_stride=[0, 1 << 24, 8]), False),
                       (1, dict(q_stride=[0, 8, 1 << 24], group=2), False), (1, dict(q_stride=[0, 8, 1 << 24]), True),
                       (0, dict(k_stride=[0, 1 << 24, 8]), False), (0, dict(v_stride=[0, 1 << 24, 8]), False),
                       (0, dict(k_stride=[1 << 40, 8, 1 << 30]), True), (2, dict(q_stride=[0, 1 << 24, 0]), True),
                       (3, dict(q_stride=[0, 1 << 24, 0]), False), (3, dict(k_stride=[0, 1 << 24, 0]), False),
                       (1, dict(kv_heads=1 << 18, query_len=1, batch=1), False), (0, dict(kv_heads=1 << 18, query_len=1, batch=1), True)]:
        g = geo(op, **kw)
        n = _lib.lib.custma_match_workspace_bytes(ctypes.byref(g), op)
        assert (n > 0) == ok, (op, kw)
        assert ok or "2^24" in err()


def test_sizes_whose_product_leaves_64_bits():
    """Refused, whatever the product wraps to: 2^29 * 2^29 * 2^6 rows are 2^64."""
    top = 1 << 29
    for op, kw in [(0, dict(batch=top, query_len=top, kv_heads=64, key_len=1)), (0, dict(batch=top, key_len=top, kv_heads=64, query_len=1)),
                   (0, dict(batch=top, query_len=1 << 24, kv_heads=1 << 20, key_len=1)), (2, dict(batch=top, query_len=top)),
                   (3, dict(batch=top, key_len=top)), (2, dict(batch=1 << 28, query_len=1, key_len=top, channels=16384))]:
        g = geo(op, **kw)
        assert _lib.lib.custma_match_workspace_bytes(ctypes.byref(g), op) == 0, (op, kw)
        assert "2^46" in err()


def test_image_sizes_whose_product_leaves_64_bits():
    fake = 1 << 20
    for H, W in ((1 << 36, 1 << 36), (1 << 62, 1 << 62), (1 << 40, 1 << 32), (1, 1 << 40)):
        assert _lib.lib.custma_descriptors(fake, 0, H, W, 3, 1, fake, None, None) < 0 and "workgroups" in err()
        assert _lib.lib.custma_descriptors_backward(fake, 0, H, W, 3, 1, fake, fake, None, fake, None) < 0 and "workgroups" in err()
