"""Row matching on vectors per pixel: softmax read-out (attention) and softmax cross entropy between the
positions of two rows, differentiable and without the score volume.

The cost volume scores every camera pixel of a row against the projector pixels of that row, and
``stereo_disparity_soft`` reduces it without storing it, but has no gradient.  These operators are the
differentiable reductions, on any vectors: learned features, or the ZNCC descriptors below.

* :func:`zncc_descriptors` -- the centred, unit-norm patch of each pixel as a vector; the dot product of a
  camera and a projector descriptor is their ZNCC.
* :func:`match_attention` -- ``softmax(scale * q . k) v`` along the row, with a window of visible columns and
  a few first columns that stay visible in front of it (``sinks``); heads that share keys, sequences of
  different lengths, and a position of the first query make the same operator the windowed attention of a
  sequence model, prompt and single token.
* :func:`match_cross_entropy` -- ``log sum_j exp(scale * x . w_j) - scale * x . w_target`` over the candidate
  columns, or over one large shared class matrix.
* :func:`stereo_soft_disparity`, :func:`stereo_match_loss` -- both on a camera / projector pair.

Scores are products of 16-bit vectors summed in 32 bits; softmax statistics, sums and losses are 32-bit.
Results do not depend on the run: there are no atomics.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple, Union

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .stereo_matching_wrapper import _LAYOUTS, _check_pair, _dtype_code, _stream_ptr, _workspace

_VECTOR_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_NONE = -1  # no bound
Window = Tuple[Optional[int], Optional[int]]


def _check_vectors(x: torch.Tensor, name: str, dims) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not x.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if x.dim() not in dims:
        raise RuntimeError(f"{name} must have {' or '.join(str(d) for d in dims)} dimensions, got shape {tuple(x.shape)}")
    if x.dtype not in _VECTOR_DTYPES:
        raise RuntimeError(f"{name} must be float16 or bfloat16, got {x.dtype}")


def _check_same(x: torch.Tensor, name: str, like: torch.Tensor, like_name: str) -> None:
    if x.dtype != like.dtype:
        raise RuntimeError(f"{name} dtype {x.dtype} != {like_name} dtype {like.dtype}")
    if x.device != like.device:
        raise RuntimeError(f"{like_name} and {name} must be on the same device")


def _bounds(window: Window) -> Tuple[int, int]:
    try:
        left, right = window
    except (TypeError, ValueError):
        raise ValueError(f"window must be (left, right), each an int or None, got {window!r}") from None
    out = []
    for name, v in (("left", left), ("right", right)):
        if v is None:
            out.append(_NONE)
            continue
        if isinstance(v, bool) or not isinstance(v, int):
            raise TypeError(f"window {name} must be an int or None, got {v!r}")
        if v < 0:
            raise ValueError(f"window {name} must be >= 0, got {v}")
        out.append(min(v, 1 << 40))
    return out[0], out[1]


# dimensions of [B, L, heads, C] along which a kernel addresses the rows of a tile in 32 bits from its first one
_NEAR_POSITIONS, _NEAR_HEADS = (1,), (1, 2)
_MAX_STRIDE = 1 << 24  # kMaxStride in csrc/match_api.hip


def _rows16(x: torch.Tensor, near: Tuple[int, ...] = ()) -> torch.Tensor:
    """Channels padded with zeros to a multiple of 8, rows 16-byte aligned: what the kernels load; and rows less than 2^24
    elements apart along the dimensions ``near``.  A view of a larger tensor (a slice of a fused projection, a cache)
    passes as it is; anything else is copied once."""
    if x.shape[-1] % 8:
        return F.pad(x, (0, -x.shape[-1] % 8))
    sizes, strides = x.shape[:-1], x.stride()[:-1]
    if (x.stride(-1) == 1 or x.shape[-1] == 1) and all(n <= 1 or s % 8 == 0 for n, s in zip(sizes, strides)) \
            and x.data_ptr() % 16 == 0 and all(sizes[n] <= 1 or strides[n] < _MAX_STRIDE for n in near):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _strides(x: torch.Tensor):
    """(batch, position, head) strides of [B, L, heads, C] (or [B, L, C]); a size of 1 has any stride."""
    return [s if n > 1 else 0 for n, s in zip(x.shape[:-1], x.stride()[:-1])]


def _finite(scale, name: str = "scale") -> float:
    scale = float(scale)
    if not math.isfinite(scale) or abs(scale) > 3e38:  # it becomes a 32-bit number
        raise ValueError(f"{name} must be finite, got {scale}")
    return scale


def _index_tensor(x, name: str, batch: int, device: torch.device) -> Optional[torch.Tensor]:
    """[batch] int32 on the device."""
    if x is None:
        return None
    if isinstance(x, int) and not isinstance(x, bool):
        if not -(1 << 31) <= x < 1 << 31:
            raise ValueError(f"{name} must fit in 32 bits, got {x}")
        return None if x == 0 and name == "query_offset" else torch.full((batch,), x, dtype=torch.int32, device=device)
    if not isinstance(x, torch.Tensor) or x.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be None, an int, or an int32 / int64 tensor [{batch}]")
    if tuple(x.shape) != (batch,):
        raise ValueError(f"{name} must have shape {(batch,)}, got {tuple(x.shape)}")
    if x.device != device:
        raise RuntimeError(f"{name} must be on {device}")
    if x.dtype == torch.int64:  # the kernels clamp what 32 bits hold
        x = x.clamp(-(1 << 31), (1 << 31) - 1)
    return x.to(torch.int32).contiguous()


_Strides = ctypes.c_int64 * 3


def _geo(q, k, v, sizes, scale, bounds, sinks=0, out_f32=False, offset=None, length=None) -> _lib.MatchGeo:
    """sizes = (B, Lq, Lk, key heads, group, C, Cv); q, k, v the strides (batch, position, head) of each."""
    B, Lq, Lk, Hkv, G, C, Cv = sizes
    return _lib.MatchGeo(_VECTOR_DTYPES[q.dtype], out_f32, B, Lq, Lk, Hkv, G, C, Cv, _Strides(*_strides(q)),
                         _Strides(*_strides(k)), _Strides(*(_strides(v) if v is not None else ())), bounds[0], bounds[1],
                         sinks, _ptr(offset), _ptr(length), scale)


class _on:
    """``with torch.cuda.device`` only where the device is not the current one already."""

    def __init__(self, dev):
        self.guard = None if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _ptr(x: Optional[torch.Tensor]):
    return None if x is None or x.numel() == 0 else x.data_ptr()


def _no_tangent(*inputs: torch.Tensor) -> None:
    """The kernels read a dual tensor's values and would drop its tangent without a word."""
    if any(forward_ad.unpack_dual(x).tangent is not None for x in inputs):
        raise RuntimeError("the matching operators have no forward-mode derivatives; differentiate them in reverse mode")


def _trains(*inputs: torch.Tensor) -> bool:
    return torch.is_grad_enabled() and any(x.requires_grad for x in inputs)


def _attention_sizes(q, k, v):
    B, Lq, Hq, C = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    return B, Lq, Lk, Hkv, Hq // Hkv, C, v.shape[3]


def _attention_forward(q, k, v, offset, length, bounds, sinks, scale, out_dtype, train, want_lse):
    """(out, low, lse); low and lse are None where nobody asks."""
    sizes = _attention_sizes(q, k, v)
    wide = out_dtype == torch.float32
    dev = q.device
    lead = q.shape[:3]
    out = torch.empty((*lead, sizes[6]), dtype=out_dtype, device=dev)
    lse = torch.empty(lead, dtype=torch.float32, device=dev) if train or want_lse else None
    # the backward subtracts grad . out from grad . v: where the output is 16-bit it gets the rounding error too
    low = torch.empty_like(out) if train and not wide else None
    if out.numel():
        g = _geo(q, k, v, sizes, scale, bounds, sinks, wide, offset, length)
        with _on(dev):
            ws = _workspace(_lib.match_workspace_bytes(g, _lib.MATCH_ATTENTION, "match_attention"), dev)
            _lib.check(_lib.lib.custma_match_attention(ctypes.byref(g), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(low),
                                                       _ptr(lse), ws.data_ptr(), ws.numel(), _stream_ptr(dev)),
                       "match_attention")
    return out, low, lse


def _attention_backward(saved, args, grad, want, unit=None):
    """Gradients of q, k, v where wanted.  ``unit``: one device float for the power of two that the gradients are still to
    be multiplied by (see _PairAttention)."""
    q, k, v, out, low, lse, offset, length = saved
    bounds, sinks, scale = args
    sizes = _attention_sizes(q, k, v)
    dev = q.device
    grad = grad.contiguous()
    if grad.data_ptr() % 16:
        grad = grad.clone()
    grads = [torch.empty(x.shape, dtype=x.dtype, device=dev) if w else None for x, w in zip((q, k, v), want)]
    if sizes[0]:
        g = _geo(q, k, v, sizes, scale, bounds, sinks, out.dtype == torch.float32, offset, length)
        with _on(dev):
            ws = _workspace(_lib.match_workspace_bytes(g, _lib.MATCH_ATTENTION_BACKWARD, "match_attention"), dev)
            _lib.check(_lib.lib.custma_match_attention_backward(
                ctypes.byref(g), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(low), _ptr(lse), _ptr(grad),
                _ptr(grads[0]), _ptr(grads[1]), _ptr(grads[2]), _ptr(unit), ws.data_ptr(), ws.numel(), _stream_ptr(dev)),
                "match_attention_backward")
    return grads


class _MatchAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offset, length, bounds, sinks, scale, out_dtype):
        out, low, lse = _attention_forward(q, k, v, offset, length, bounds, sinks, scale, out_dtype, True, True)
        ctx.save_for_backward(q, k, v, out, low, lse, offset, length)
        ctx.args = (bounds, sinks, scale)
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, _):
        if grad is None:
            return (None,) * 9
        return (*_attention_backward(ctx.saved_tensors, ctx.args, grad, ctx.needs_input_grad), *(None,) * 6)


def match_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, *, window: Window = (None, None),
                    sinks: int = 0, scale: Optional[float] = None,
                    query_offset: Union[None, int, torch.Tensor] = None,
                    key_lengths: Union[None, int, torch.Tensor] = None,
                    out_dtype: Optional[torch.dtype] = None, return_lse: bool = False):
    """``out[b, i, h] = sum_j softmax_j(scale * q_i . k_j) v_j`` over the keys that query i sees.

    ``query`` [B, Lq, heads, C], ``key`` [B, Lk, key_heads, C], ``value`` [B, Lk, key_heads, Cv], all float16
    or all bfloat16; ``heads`` is a multiple of ``key_heads`` and head h reads key head
    ``h // (heads // key_heads)``.  [B, L, C] tensors (rows of an image pair) are one head.  C and Cv up to 256.

    Query i is at position ``p = query_offset[b] + i``.  It sees key j iff ``j < key_lengths[b]``,
    ``j <= p + right`` and (``j >= p - left`` or ``j < sinks``), with ``window = (left, right)`` and None for no
    bound.  ``(0, D)`` is the window layout of the cost volume, ``(n - 1, 0)`` a causal window of n.  A query that
    sees nothing has output 0 and no gradient.  ``query_offset`` (default 0) and ``key_lengths`` (default Lk) are
    an int of 32 bits or an integer tensor [B] on the device; a length outside [0, Lk] counts as the nearer end, an
    offset outside +-2^30 likewise.  Keys and values behind a length are never read.

    ``scale`` defaults to ``C ** -0.5``.  ``out_dtype``: the inputs' type (default) or float32, for values that
    need more than 16 bits, such as coordinates.  ``return_lse`` adds ``log sum_j exp(scale * q_i . k_j)``
    [B, Lq, heads] in float32 (-inf where nothing is seen), which has no gradient.

    Any strides; rows that are not 16-byte aligned, or 2^24 elements and more apart, are copied first.  Gradients go to all three inputs.  In float16 an
    output gradient far below 1 leaves the type's range inside, as its products do: scale the loss, or take a float32
    output, whose gradient is scaled here, by one power of two for the whole tensor: what is 2^-24 of the largest is lost.

    Probabilities (and in the backward their products with the gradient) enter the 16-bit products rounded once, for values
    of up to 32 channels and a float32 output in two parts: a wide 16-bit output is off by up to one and a half times its
    own rounding."""
    rows = isinstance(query, torch.Tensor) and query.dim() == 3
    dims = (3,) if rows else (3, 4) if not isinstance(query, torch.Tensor) else (4,)
    _check_vectors(query, "query", (3, 4))
    _check_vectors(key, "key", dims)
    _check_vectors(value, "value", dims)
    _check_same(key, "key", query, "query")
    _check_same(value, "value", query, "query")
    _no_tangent(query, key, value)
    if rows:
        query, key, value = query.unsqueeze(2), key.unsqueeze(2), value.unsqueeze(2)
    B, Lq, Hq, C = query.shape
    Lk, Hkv = key.shape[1], key.shape[2]
    if key.shape[0] != B or key.shape[3] != C:
        raise RuntimeError(f"key shape {tuple(key.shape)} does not fit query shape {tuple(query.shape)}")
    if tuple(value.shape[:3]) != tuple(key.shape[:3]):
        raise RuntimeError(f"value shape {tuple(value.shape)} does not fit key shape {tuple(key.shape)}")
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"query heads ({Hq}) must be a multiple of key heads ({Hkv})")
    Cv = value.shape[3]
    if not 1 <= C <= 256 or not 1 <= Cv <= 256:
        raise ValueError(f"match_attention needs 1 to 256 channels, got {C} and {Cv}")
    bounds = _bounds(window)
    if isinstance(sinks, bool) or not isinstance(sinks, int):
        raise TypeError("sinks must be an int")
    if sinks < 0:
        raise ValueError(f"sinks must be >= 0, got {sinks}")
    if out_dtype is None:
        out_dtype = query.dtype
    if out_dtype not in (query.dtype, torch.float32):
        raise ValueError(f"out_dtype must be {query.dtype} or torch.float32, got {out_dtype}")
    scale = C ** -0.5 if scale is None else _finite(scale)
    offset = _index_tensor(query_offset, "query_offset", B, query.device)
    length = _index_tensor(key_lengths, "key_lengths", B, query.device)
    near = () if not _trains(query, key, value) else _NEAR_HEADS if Hq > Hkv else _NEAR_POSITIONS  # the backward's
    q, k, v = _rows16(query, near), _rows16(key, _NEAR_POSITIONS), _rows16(value, _NEAR_POSITIONS)
    args = (q, k, v, offset, length, bounds, min(sinks, 1 << 30), scale, out_dtype)
    if _trains(q, k, v):
        out, lse = _MatchAttention.apply(*args)
    else:
        out, _, lse = _attention_forward(*args, False, return_lse)
    out = out[..., :Cv] if out.shape[-1] != Cv else out
    if rows:
        out = out.squeeze(2)
    if not return_lse:
        return out
    return out, lse.squeeze(2) if rows else lse


def _entropy_forward(x, w, target, bounds, scale, reduction):
    """(value, lse, total): the loss as reduced, the rows' log-sum-exp, and where reduced [sum, 1 / counted, mean]."""
    B, N, C = x.shape
    V = w.shape[1]
    dev = x.device
    loss = torch.empty((B, N), dtype=torch.float32, device=dev)
    lse = torch.empty((B, N), dtype=torch.float32, device=dev)
    total = None if reduction == "none" else torch.empty(3, dtype=torch.float32, device=dev)
    if B == 0 or N == 0 or V == 0:
        loss.zero_()
        if total is not None:
            total.zero_()
    else:
        g = _geo(x, w, None, (B, N, V, 1, 1, C, 0), scale, bounds)
        with _on(dev):
            ws = _workspace(_lib.match_workspace_bytes(g, _lib.MATCH_ENTROPY, "match_cross_entropy"), dev)
            _lib.check(_lib.lib.custma_match_entropy(ctypes.byref(g), _ptr(x), _ptr(w), _ptr(target), _ptr(loss), _ptr(lse),
                                                     _ptr(total), ws.data_ptr(), ws.numel(), _stream_ptr(dev)),
                       "match_cross_entropy")
    return (loss if total is None else total[2 if reduction == "mean" else 0]), lse, total


def _entropy_backward(saved, args, grad, inv, want, unit=None):
    """Gradients of x and w where wanted; inv: 1 / counted of a mean, unit as in _attention_backward."""
    x, w, target, lse = saved
    bounds, scale, reduction = args
    B, N, C = x.shape
    V = w.shape[1]
    dev = x.device
    gx, gw = [torch.empty(t.shape, dtype=t.dtype, device=dev) if n else None for t, n in zip((x, w), want)]
    if B == 0 or N == 0 or V == 0:
        return gx.zero_() if gx is not None else None, gw.zero_() if gw is not None else None
    g = _geo(x, w, None, (B, N, V, 1, 1, C, 0), scale, bounds)
    weight = factor = None
    if reduction == "none":
        weight = grad.contiguous()
    else:
        factor = grad * inv if reduction == "mean" else grad.contiguous()
    with _on(dev):
        ws = _workspace(_lib.match_workspace_bytes(g, _lib.MATCH_ENTROPY_BACKWARD, "match_cross_entropy"), dev)
        _lib.check(_lib.lib.custma_match_entropy_backward(
            ctypes.byref(g), _ptr(x), _ptr(w), _ptr(target), _ptr(lse), _ptr(weight), _ptr(factor), _ptr(gx),
            _ptr(gw), _ptr(unit), ws.data_ptr(), ws.numel(), _stream_ptr(dev)), "match_cross_entropy_backward")
    return gx, gw


class _MatchEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, target, bounds, scale, reduction):
        value, lse, total = _entropy_forward(x, w, target, bounds, scale, reduction)
        ctx.save_for_backward(x, w, target, lse)
        # beside the value in `total`, which is detached from it: a caller may edit the loss in place
        ctx.inv = total[1] if reduction == "mean" else None
        ctx.args = (bounds, scale, reduction)
        return value.detach() if total is not None else value

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return (*_entropy_backward(ctx.saved_tensors, ctx.args, grad, ctx.inv, ctx.needs_input_grad), *(None,) * 4)


def match_cross_entropy(query: torch.Tensor, classes: torch.Tensor, target: torch.Tensor, *, scale: float = 1.0,
                        window: Window = (None, None), reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of each query over its candidate classes, without the scores:
    ``loss_i = log sum_j exp(scale * x_i . w_j) - scale * x_i . w_{target_i}``.

    ``query`` [N, C] or [B, N, C]; ``classes`` [V, C], shared by all queries, or [B, V, C] (the projector
    row of each camera row); both float16 or both bfloat16.  ``target`` int64 or int32 of the query's leading
    shape.  ``window = (left, right)``: query i of a row sees classes ``i - left .. i + right`` (None: no bound;
    ``(0, D)`` is the window layout of the cost volume).

    A target that is not one of its query's visible classes (-1, -100, out of the window, V and above) marks a
    query without ground truth: it does not count, its loss and gradients are 0.  ``reduction``: "mean" over
    the queries that count (0 if none does), "sum", or "none" (the query's leading shape); float32.

    C up to 16384, up to 256 with a window; a window needs one class matrix per row.  Gradients go to ``query``
    and ``classes`` in their type; in float16 use "sum" or a scaled loss, a mean over many rows underflows."""
    _check_vectors(query, "query", (2, 3))
    _check_vectors(classes, "classes", (2, 3))
    _check_same(classes, "classes", query, "query")
    _no_tangent(query, classes)
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    bounds, scale = _bounds(window), _finite(scale)
    lead, C = tuple(query.shape[:-1]), query.shape[-1]
    if classes.shape[-1] != C:
        raise RuntimeError(f"classes shape {tuple(classes.shape)} does not fit query shape {tuple(query.shape)}")
    windowed = bounds != (_NONE, _NONE)
    limit = 256 if windowed else 16384
    if not 1 <= C <= limit:
        raise ValueError(f"match_cross_entropy needs 1 to {limit} channels{' with a window' if windowed else ''}, got {C}")
    if not isinstance(target, torch.Tensor) or target.dtype not in (torch.int32, torch.int64):
        raise TypeError("target must be an int32 or int64 tensor")
    if tuple(target.shape) != lead:
        raise RuntimeError(f"target shape {tuple(target.shape)} != query's leading shape {lead}")
    if target.device != query.device:
        raise RuntimeError("query and target must be on the same device")
    if classes.dim() == 3:
        if query.dim() != 3 or classes.shape[0] != query.shape[0]:
            raise RuntimeError(f"classes shape {tuple(classes.shape)} does not fit query shape {tuple(query.shape)}")
        x, w = query, classes
    else:
        if query.dim() == 3 and windowed:
            raise ValueError("a window needs one class matrix per row: classes [B, V, C]")
        x, w = query.reshape(1, -1, C), classes.unsqueeze(0)
    t = target.to(torch.int64).reshape(x.shape[:2]).contiguous()
    x, w = _rows16(x, _NEAR_POSITIONS if _trains(x, w) else ()), _rows16(w, _NEAR_POSITIONS)
    if _trains(x, w):
        loss = _MatchEntropy.apply(x, w, t, bounds, scale, reduction)
    else:
        loss = _entropy_forward(x, w, t, bounds, scale, reduction)[0]
    return loss.reshape(lead) if reduction == "none" else loss


def _check_kernel_size(k: int) -> None:
    if not 1 <= k <= 16:
        raise ValueError(f"descriptors need kernel_size in [1, 16], got {k}")


def _descriptors_forward(image, k, dtype, train):
    H, W = image.shape
    out = torch.empty((H, W, -(-k * k // 8) * 8), dtype=dtype, device=image.device)
    stats = torch.empty((H, W, 2), dtype=torch.float32, device=image.device) if train else None
    if out.numel():
        with _on(image.device):
            _lib.check(_lib.lib.custma_descriptors(image.data_ptr(), _dtype_code(image), H, W, k, _VECTOR_DTYPES[dtype],
                                                   out.data_ptr(), _ptr(stats), _stream_ptr(image.device)),
                       "zncc_descriptors")
    return out, stats


def _descriptors_backward(image, stats, k, grad, unit=None):
    H, W = image.shape
    grad = grad.contiguous()
    if grad.data_ptr() % 16:
        grad = grad.clone()
    out = torch.empty_like(image)
    if out.numel():
        with _on(image.device):
            _lib.check(_lib.lib.custma_descriptors_backward(
                image.data_ptr(), _dtype_code(image), H, W, k, _VECTOR_DTYPES[grad.dtype], _ptr(stats), grad.data_ptr(),
                _ptr(unit), out.data_ptr(), _stream_ptr(image.device)), "zncc_descriptors_backward")
    return out


class _Descriptors(torch.autograd.Function):
    @staticmethod
    def forward(ctx, image, k, dtype):
        out, stats = _descriptors_forward(image, k, dtype, True)
        ctx.save_for_backward(image, stats)
        ctx.k = k
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        image, stats = ctx.saved_tensors
        return _descriptors_backward(image, stats, ctx.k, grad), None, None


def zncc_descriptors(image: torch.Tensor, kernel_size: int, dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """[H, W] image (float32 or float16) -> [H, W, C] unit vectors in ``dtype`` (float16 or bfloat16): the
    zero-padded ``kernel_size`` x ``kernel_size`` patch around each pixel, minus its mean, over
    ``sqrt(sum of squares + 1e-8)``, in row-major tap order; C is ``kernel_size ** 2`` rounded up to a multiple
    of 8, the rest zeros.  kernel_size 1 to 16, taps as in the cost volume; the epsilon has its value, but stands under
    each vector's norm instead of under the product of two.  Any range of values; a pixel that is not finite reaches the
    patches that hold it.  Differentiable."""
    if not isinstance(image, torch.Tensor):
        raise TypeError("image must be a torch.Tensor")
    if not image.is_cuda:
        raise RuntimeError("image must be a CUDA tensor")
    if image.dim() != 2:
        raise RuntimeError(f"image must be a 2-D [H, W] tensor, got shape {tuple(image.shape)}")
    if not image.is_contiguous():
        raise RuntimeError("image must be contiguous")
    _dtype_code(image)
    if not isinstance(kernel_size, int) or isinstance(kernel_size, bool):
        raise TypeError("kernel_size must be an int")
    _check_kernel_size(kernel_size)
    if dtype not in _VECTOR_DTYPES:
        raise RuntimeError(f"unsupported descriptor dtype {dtype} (float16 or bfloat16)")
    _no_tangent(image)
    if _trains(image):
        return _Descriptors.apply(image, kernel_size, dtype)
    return _descriptors_forward(image, kernel_size, dtype, False)[0]


def _pair(camera, projector, D, kernel_size, layout):
    _check_pair(camera, projector, kernel_size)
    _check_kernel_size(kernel_size)
    _no_tangent(camera, projector)
    if layout not in _LAYOUTS:
        raise ValueError(f"layout must be one of {sorted(_LAYOUTS)}, got {layout!r}")
    W = camera.shape[1]
    if layout == "full":
        return W, (None, None)
    D = int(D)
    if not 0 <= D < W:
        raise ValueError(f"window layout needs 0 <= D < W, got D={D} W={W}")
    return W - D, (0, D)


def _pair_backward(ctx, images, stats, grads, unit):
    """The images' gradients from those of their descriptors; columns behind the last query have none."""
    out = []
    for image, st, g in zip(images, stats, grads):
        if g is not None and g.shape[1] < image.shape[1]:
            g = F.pad(g, (0, 0, 0, image.shape[1] - g.shape[1]))
        out.append(None if g is None else _descriptors_backward(image, st, ctx.k, g, unit))
    return out


# The pair operators are one node each, descriptors and all: the gradient of a mean over pixels would leave float16's
# range, so the descriptors' gradients travel near 1 and their power of two (unit) beside them, until the images' 32-bit
# gradients take it up.  It belongs to one backward pass and to no other.

class _PairAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, camera, projector, value, k, WO, window, beta, train):
        (cam, cs), (proj, ps) = (_descriptors_forward(x, k, torch.float16, train) for x in (camera, projector))
        qkv = cam[:, :WO].unsqueeze(2), proj.unsqueeze(2), value
        out, _, lse = _attention_forward(*qkv, None, None, window, 0, beta, torch.float32, train, False)
        if train:
            ctx.save_for_backward(camera, projector, cs, ps, *qkv, out, lse)
            ctx.k, ctx.args = k, (window, 0, beta)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        camera, projector, cs, ps, q, k, v, out, lse = ctx.saved_tensors
        want = ctx.needs_input_grad
        unit = torch.empty(1, dtype=torch.float32, device=q.device)
        dq, dk, _ = _attention_backward((q, k, v, out, None, lse, None, None), ctx.args, grad, (want[0], want[1], False), unit)
        grads = [x.squeeze(2) if x is not None else None for x in (dq, dk)]
        return (*_pair_backward(ctx, (camera, projector), (cs, ps), grads, unit), *(None,) * 6)


class _PairEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, camera, projector, target, k, WO, window, beta, reduction, train):
        (cam, cs), (proj, ps) = (_descriptors_forward(x, k, torch.float16, train) for x in (camera, projector))
        value, lse, total = _entropy_forward(cam[:, :WO], proj, target, window, beta, reduction)
        if train:
            ctx.save_for_backward(camera, projector, cs, ps, cam[:, :WO], proj, target, lse)
            ctx.inv = total[1] if reduction == "mean" else None
            ctx.k, ctx.args = k, (window, beta, reduction)
        return value.detach() if total is not None else value

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        camera, projector, cs, ps, *saved = ctx.saved_tensors
        unit = torch.empty(1, dtype=torch.float32, device=camera.device)
        grads = _entropy_backward(saved, ctx.args, grad, ctx.inv, ctx.needs_input_grad, unit)
        return (*_pair_backward(ctx, (camera, projector), (cs, ps), grads, unit), *(None,) * 7)


def stereo_soft_disparity(camera: torch.Tensor, projector: torch.Tensor, D: int, kernel_size: int,
                          layout: str = "full", beta: float = 50.0) -> torch.Tensor:
    """The soft-argmax of :func:`stereo_disparity_soft` with gradients to both images, still without the volume:
    [H, WO] float32 ``sum_s s * softmax(beta * cost)_s`` over the layout's last axis (examples/verify.py:31-39).
    Costs are products of float16 :func:`zncc_descriptors`, so they are within about 1e-3 of the volume's and
    a flat patch scores 0; kernel_size 1 to 16.  The gradients pass through float16 vectors in one unit: pixels whose
    output gradient is 2^-24 of the largest get none."""
    WO, window = _pair(camera, projector, D, kernel_size, layout)
    if not beta > 0:
        raise ValueError(f"beta must be > 0, got {beta}")
    H, W = camera.shape
    if W >= 1 << 22:
        raise ValueError(f"stereo_soft_disparity needs W < 2^22, got {W}")
    j = torch.arange(W, device=camera.device)
    value = torch.stack([(j >> 11).half(), (j & 2047).half(), *[torch.zeros(W, device=j.device).half()] * 6], -1)[:, None]
    # float16 holds 0 .. 2047 exactly: the column in two parts
    parts = _PairAttention.apply(camera.contiguous(), projector.contiguous(), value.expand(H, W, 1, 8), kernel_size, WO,
                                 _bounds(window), _finite(beta, "beta"), _trains(camera, projector))
    column = parts[:, :, 0, 0] * 2048.0 + parts[:, :, 0, 1]
    if layout == "window":
        column = column - torch.arange(WO, device=j.device, dtype=torch.float32)
    return column


def stereo_match_loss(camera: torch.Tensor, projector: torch.Tensor, target: torch.Tensor, D: int, kernel_size: int,
                      layout: str = "full", beta: float = 50.0, reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of ``softmax(beta * cost)`` over the candidates of each pixel, with gradients to both images and
    without the volume.  ``target`` [H, WO] integer: the true index on the layout's last axis as
    :func:`stereo_disparity` returns it (full: the projector column; window: the offset s, column w + s); any
    other value marks a pixel without ground truth, which does not count.  ``reduction`` as in
    :func:`match_cross_entropy`.  Costs as in :func:`stereo_soft_disparity`."""
    WO, window = _pair(camera, projector, D, kernel_size, layout)
    if not beta > 0:
        raise ValueError(f"beta must be > 0, got {beta}")
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    H, W = camera.shape
    if not isinstance(target, torch.Tensor) or target.dtype not in (torch.int32, torch.int64):
        raise TypeError("target must be an int32 or int64 tensor")
    if tuple(target.shape) != (H, WO):
        raise RuntimeError(f"target shape {tuple(target.shape)} != {(H, WO)}")
    if target.device != camera.device:
        raise RuntimeError("camera and target must be on the same device")
    if layout == "window":
        column = target.to(torch.int64) + torch.arange(WO, device=target.device)
        target = torch.where((target >= 0) & (target <= int(D)), column, -1)
    return _PairEntropy.apply(camera.contiguous(), projector.contiguous(), target.to(torch.int64).contiguous(), kernel_size,
                              WO, _bounds(window), _finite(beta, "beta"), reduction, _trains(camera, projector))
