"""The matching operators' host side, without a GPU: the C ABI refuses before it touches the device, workspaces cover
what the plans carve, and the Python shim's argument checks."""
import ctypes

import pytest
import torch

import custereomatching_amd as cm
from custereomatching_amd import _lib, matching

FAKE = 1 << 20  # a 256-byte aligned address that is never dereferenced


def geo(op=_lib.MATCH_ATTENTION, **kw):
    g = _lib.MatchGeo()
    entropy = op >= _lib.MATCH_ENTROPY
    d = dict(dtype=_lib.F16, out_f32=0, batch=2, query_len=10, key_len=20, kv_heads=1, group=1, channels=64,
             value_channels=0 if entropy else 64, left=-1, right=-1, sinks=0, scale=1.0)
    d.update(kw)
    for n, v in d.items():
        if n.endswith("stride"):
            getattr(g, n)[:] = v
        else:
            setattr(g, n, v)
    return g


def err():
    return _lib.lib.custma_last_error().decode()


BAD = [
    (dict(dtype=_lib.F32), "dtype"), (dict(dtype=7), "dtype"), (dict(batch=-1), "sizes"), (dict(query_len=-1), "sizes"),
    (dict(key_len=1 << 30), "sizes"), (dict(kv_heads=0), "kv_heads"), (dict(group=0), "kv_heads"),
    (dict(query_len=1 << 29, group=4), "group"), (dict(channels=0), "channels"), (dict(channels=20), "channels"),
    (dict(channels=264), "channels"), (dict(value_channels=0), "value_channels"), (dict(value_channels=12), "value_channels"),
    (dict(value_channels=300), "value_channels"), (dict(left=-2), "left"), (dict(right=-5), "left"), (dict(sinks=-1), "sinks"),
    (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(q_stride=[8, 8, 4]), "strides"), (dict(k_stride=[8, -8, 8]), "strides"), (dict(v_stride=[1, 8, 8]), "strides"),
]


@pytest.mark.parametrize("kw,word", BAD)
def test_attention_refuses_geometry(kw, word):
    g = geo(**kw)
    for op in (_lib.MATCH_ATTENTION, _lib.MATCH_ATTENTION_BACKWARD):
        assert _lib.lib.custma_match_workspace_bytes(ctypes.byref(g), op) == 0
        assert word in err()
    rc = _lib.lib.custma_match_attention(ctypes.byref(g), FAKE, FAKE, FAKE, FAKE, None, None, FAKE, 1 << 40, None)
    assert rc == _lib.E_ARG and word in err()
    rc = _lib.lib.custma_match_attention_backward(ctypes.byref(g), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE,
                                                  None, FAKE, 1 << 40, None)
    assert rc == _lib.E_ARG and word in err()


@pytest.mark.parametrize("kw,rc,word", [(dict(kv_heads=2), _lib.E_ARG, "heads"), (dict(sinks=1), _lib.E_ARG, "sinks"),
                                        (dict(offset=FAKE), _lib.E_ARG, "offsets"), (dict(value_channels=8), _lib.E_ARG, "value"),
                                        (dict(channels=16392), _lib.E_ARG, "channels"),
                                        (dict(channels=512, left=3), _lib.E_UNSUPPORTED, "window")])
def test_entropy_refuses_geometry(kw, rc, word):
    g = geo(_lib.MATCH_ENTROPY, **kw)
    assert _lib.lib.custma_match_workspace_bytes(ctypes.byref(g), _lib.MATCH_ENTROPY) == 0
    assert word in err()
    assert _lib.lib.custma_match_entropy(ctypes.byref(g), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40, None) == rc
    assert _lib.lib.custma_match_entropy_backward(ctypes.byref(g), FAKE, FAKE, FAKE, FAKE, None, None, FAKE, FAKE, None,
                                                  FAKE, 1 << 40, None) == rc


def test_null_alignment_and_workspace():
    L, g = _lib.lib, geo()
    n = L.custma_match_workspace_bytes(ctypes.byref(g), _lib.MATCH_ATTENTION)
    assert n > 0
    call = lambda q=FAKE, k=FAKE, v=FAKE, o=FAKE, ws=FAKE, b=n: L.custma_match_attention(  # noqa: E731
        ctypes.byref(g), q, k, v, o, None, None, ws, b, None)
    assert call(q=None) == _lib.E_NULL and call(k=None) == _lib.E_NULL and call(o=None) == _lib.E_NULL
    assert call(ws=None) == _lib.E_NULL
    assert call(b=n - 1) == _lib.E_WORKSPACE
    assert call(q=FAKE + 2) == _lib.E_ARG and "aligned" in err()
    assert call(ws=FAKE + 16) == _lib.E_ARG and "aligned" in err()
    assert L.custma_match_attention(None, FAKE, FAKE, FAKE, FAKE, None, None, FAKE, n, None) == _lib.E_NULL
    # the 16-bit output's rounding error is required by the backward
    m = L.custma_match_workspace_bytes(ctypes.byref(g), _lib.MATCH_ATTENTION_BACKWARD)
    assert L.custma_match_attention_backward(ctypes.byref(g), FAKE, FAKE, FAKE, FAKE, None, FAKE, FAKE, FAKE, FAKE, FAKE, None,
                                             FAKE, m, None) == _lib.E_NULL
    # and a power of two beside the gradients belongs to a 32-bit output
    assert L.custma_match_attention_backward(ctypes.byref(g), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE,
                                             FAKE, m, None) == _lib.E_ARG and "unit" in err()
    e = geo(_lib.MATCH_ENTROPY)
    b = L.custma_match_workspace_bytes(ctypes.byref(e), _lib.MATCH_ENTROPY)
    assert L.custma_match_entropy(ctypes.byref(e), FAKE, FAKE, None, FAKE, FAKE, FAKE, FAKE, b, None) == _lib.E_NULL
    assert L.custma_match_entropy(ctypes.byref(e), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, b - 1, None) == _lib.E_WORKSPACE
    assert L.custma_match_workspace_bytes(ctypes.byref(e), 9) == 0 and "operation" in err()


@pytest.mark.parametrize("kw", [dict(query_len=0), dict(key_len=0), dict(query_len=0, key_len=0), dict(batch=0)])
def test_workspace_of_nothing(kw):
    for op in range(4):
        g = geo(op, **kw)
        if op < 2:
            g.left, g.sinks = 3, 5
        assert _lib.lib.custma_match_workspace_bytes(ctypes.byref(g), op) > 0
        if op >= 2:
            g.channels = 512
            assert _lib.lib.custma_match_workspace_bytes(ctypes.byref(g), op) > 0


def test_too_many_rows_for_a_launch():
    g = geo(batch=1 << 20, query_len=1 << 10, key_len=64)
    assert _lib.lib.custma_match_attention(ctypes.byref(g), FAKE, FAKE, FAKE, FAKE, None, None, FAKE, 1 << 50, None) == _lib.E_UNSUPPORTED
    assert "workgroups" in err()


def test_nothing_to_do_needs_no_pointers():
    g = geo(batch=0)
    assert _lib.lib.custma_match_attention(ctypes.byref(g), None, None, None, None, None, None, None, 0, None) == 0
    g = geo()
    assert _lib.lib.custma_match_attention_backward(ctypes.byref(g), None, None, None, None, None, None, None, None, None, None,
                                                    None, None, 0, None) == 0


@pytest.mark.parametrize("args,word", [((0, 4, 4, 17, 1), "kernel_size"), ((0, 4, 4, 0, 1), "kernel_size"), ((2, 4, 4, 3, 1), "image dtype"),
                                       ((0, 4, 4, 3, 0), "descriptor dtype"), ((0, -1, 4, 3, 1), "size"),
                                       ((0, 1 << 21, 1 << 20, 3, 1), "workgroups")])
def test_descriptors_refuse(args, word):
    d, H, W, k, o = args
    assert _lib.lib.custma_descriptors(FAKE, d, H, W, k, o, FAKE, None, None) < 0 and word in err()
    assert _lib.lib.custma_descriptors_backward(FAKE, d, H, W, k, o, FAKE, FAKE, None, FAKE, None) < 0 and word in err()


def test_descriptors_null_and_empty():
    L = _lib.lib
    assert L.custma_descriptors(None, 0, 0, 5, 3, 1, None, None, None) == 0
    assert L.custma_descriptors(None, 0, 5, 5, 3, 1, FAKE, None, None) == _lib.E_NULL
    assert L.custma_descriptors(FAKE, 0, 5, 5, 3, 1, FAKE + 8, None, None) == _lib.E_ARG
    assert L.custma_descriptors_backward(FAKE, 0, 5, 5, 3, 1, FAKE, None, None, FAKE, None) == _lib.E_NULL


# ---- the Python shim ----

def test_shim_refuses_cpu_tensors():
    q = torch.zeros(1, 2, 1, 8, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="query must be a CUDA tensor"):
        cm.match_attention(q, q, q)
    with pytest.raises(RuntimeError, match="query must be a CUDA tensor"):
        cm.match_cross_entropy(q[0, :, 0], q[0, :, 0], torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="image must be a CUDA tensor"):
        cm.zncc_descriptors(torch.zeros(4, 4), 3)
    with pytest.raises(RuntimeError, match="camera must be a CUDA tensor"):
        cm.stereo_soft_disparity(torch.zeros(4, 4), torch.zeros(4, 4), 0, 3)
    with pytest.raises(RuntimeError, match="camera must be a CUDA tensor"):
        cm.stereo_match_loss(torch.zeros(4, 4), torch.zeros(4, 4), torch.zeros(4, 4, dtype=torch.int64), 0, 3)
    with pytest.raises(TypeError, match="query must be a torch.Tensor"):
        cm.match_attention([1], q, q)


def test_shim_bounds():
    assert matching._bounds((None, None)) == (-1, -1) and matching._bounds((0, 5)) == (0, 5)
    assert matching._bounds((1 << 60, None)) == (1 << 40, -1)
    for bad, kind in (((1,), ValueError), (3, ValueError), ((-1, 0), ValueError), ((1.5, 0), TypeError), ((True, 0), TypeError)):
        with pytest.raises(kind):
            matching._bounds(bad)


def test_shim_index_tensors():
    f = lambda x: matching._index_tensor(x, "key_lengths", 3, torch.device("cpu"))  # noqa: E731
    assert f(None) is None and f(7).tolist() == [7, 7, 7] and f(0).tolist() == [0, 0, 0]
    assert matching._index_tensor(0, "query_offset", 3, torch.device("cpu")) is None
    assert f(torch.tensor([1, 2, 3])).dtype == torch.int32
    assert f(torch.arange(6, dtype=torch.int32)[::2]).is_contiguous()
    for bad, kind in ((torch.zeros(3), TypeError), (torch.zeros(2, dtype=torch.int32), ValueError), (1.0, TypeError),
                      (True, TypeError), (1 << 31, ValueError)):
        with pytest.raises(kind):
            f(bad)


def test_shim_rows_keep_views_that_the_kernels_can_read():
    fused = torch.arange(2 * 5 * 48, dtype=torch.float32).to(torch.bfloat16).reshape(2, 5, 48)
    view = fused[..., 16:32].unflatten(-1, (2, 8))
    assert matching._rows16(view) is view
    assert matching._rows16(fused.transpose(0, 1)) is not None and matching._rows16(fused.transpose(0, 1)).stride(-1) == 1
    for x in (fused[..., 1:17], fused[..., ::2], fused.reshape(2, 48, 5).transpose(1, 2)[..., :40]):
        y = matching._rows16(x)
        assert y.is_contiguous() and torch.equal(x, y)
    odd = matching._rows16(fused[..., :13])
    assert odd.shape[-1] == 16 and torch.equal(odd[..., :13], fused[..., :13]) and not odd[..., 13:].any()
