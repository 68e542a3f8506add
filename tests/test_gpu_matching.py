"""The matching operators on the GPU against 64-bit references, at the sizes and masks where they can go wrong.
Tolerances: tests/matching_ref.py derives one per element from the roundings that a right kernel makes."""
import pytest
import torch

import custereomatching_amd as cm
from tests import matching_ref as R

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rand(g, *shape, dtype=F16, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _attention_case(gpu, B, Lq, Lk, Hq, Hkv, C, Cv, window=(None, None), sinks=0, offset=None, length=None, dtype=F16,
                    out_dtype=None, train=True, scale=None, seed=0):
    g = _gen(seed)
    q, k, v = (_rand(g, B, n, h, c, dtype=dtype) for n, h, c in ((Lq, Hq, C), (Lk, Hkv, C), (Lk, Hkv, Cv)))
    out_dtype = out_dtype or dtype
    scale = C ** -0.5 if scale is None else scale
    go = _rand(g, B, Lq, Hq, Cv, dtype=out_dtype) if train else None
    off = [0] * B if offset is None else offset
    n = [Lk] * B if length is None else length
    see = R.visible(Lq, Lk, window, sinks, off, [min(max(x, 0), Lk) for x in n], gpu)
    want = R.attention(q, k, v, see, scale, out_dtype, go)
    if train:
        q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    out, lse = cm.match_attention(q, k, v, window=window, sinks=sinks, scale=scale,
                                  query_offset=None if offset is None else torch.tensor(offset, device=gpu, dtype=torch.int32),
                                  key_lengths=None if length is None else torch.tensor(length, device=gpu, dtype=torch.int32),
                                  out_dtype=out_dtype, return_lse=True)
    assert out.dtype == out_dtype and lse.dtype == F32
    R.check(out, want["out"], "out")
    R.check(lse, want["lse"], "lse")
    if train:
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), go)
        R.check(dq, want["dq"], "dq")
        R.check(dk, want["dk"], "dk")
        R.check(dv, want["dv"], "dv")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("C,Cv", [(8, 8), (32, 32), (64, 64), (128, 128), (256, 256), (128, 8), (88, 32), (232, 16),
                                  (64, 128), (200, 72), (1, 1), (49, 5), (33, 130)])
def test_attention_channels(gpu, dtype, C, Cv):
    _attention_case(gpu, 2, 70, 133, 1, 1, C, Cv, dtype=dtype)


@pytest.mark.parametrize("Lq,Lk", [(1, 1), (1, 2), (2, 1), (31, 33), (32, 64), (33, 65), (127, 129), (128, 128), (129, 200),
                                   (300, 517), (1, 5000), (5, 3000)])
def test_attention_lengths(gpu, Lq, Lk):
    _attention_case(gpu, 1, Lq, Lk, 2, 1, 64, 64, dtype=BF16, seed=Lq)
    _attention_case(gpu, 1, Lq, Lk, 2, 2, 128, 32, dtype=F16, seed=Lk)


@pytest.mark.parametrize("window,sinks", [((0, 0), 0), ((0, 40), 0), ((0, 300), 2), ((5, 0), 0), ((5, 0), 1), ((63, 0), 4),
                                          ((64, 0), 70), ((100, 0), 200), ((None, 0), 0), ((20, None), 3), ((None, 7), 5),
                                          ((17, 9), 130), ((1000, 1000), 3)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_windows(gpu, window, sinks, dtype):
    _attention_case(gpu, 2, 259, 259, 2, 1, 64, 64, window, sinks, dtype=dtype)


@pytest.mark.parametrize("C", [32, 128, 256])
def test_attention_windows_wide_vectors(gpu, C):
    _attention_case(gpu, 1, 200, 230, 4, 2, C, C, (37, 0), 3, dtype=BF16)
    _attention_case(gpu, 1, 150, 230, 1, 1, C, 8, (0, 64), 1, dtype=F16, out_dtype=F32)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 1), (4, 2), (5, 5), (12, 3), (40, 1)])
def test_attention_shared_heads(gpu, Hq, Hkv):
    _attention_case(gpu, 2, 65, 90, Hq, Hkv, 64, 64, (30, 0), 2, dtype=BF16)


def test_attention_ragged(gpu):
    """Lengths of 0, 1 and beyond the buffer; positions before and behind the keys."""
    _attention_case(gpu, 6, 50, 100, 2, 1, 64, 64, (15, 0), 3, offset=[0, 50, 0, -20, 500, 40],
                    length=[100, 100, 0, 30, 100, 1000], dtype=BF16)
    _attention_case(gpu, 4, 1, 1000, 8, 2, 128, 128, (None, 0), 0, offset=[999, 0, 400, 7], length=[1000, 1, 401, 0],
                    dtype=BF16, train=False)
    _attention_case(gpu, 3, 4, 777, 4, 4, 256, 256, (100, 0), 5, offset=[773, 100, 0], length=[777, 104, 1], dtype=F16)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("go_scale", [1.0, 1e-7])
def test_attention_float32_output(gpu, dtype, go_scale):
    """The output keeps 32-bit accuracy, and small output gradients do not vanish on their way through 16 bits."""
    g = _gen(3)
    q, k, v = _rand(g, 3, 40, 1, 64, dtype=dtype), _rand(g, 3, 90, 1, 64, dtype=dtype), _rand(g, 3, 90, 1, 8, dtype=dtype)
    go = _rand(g, 3, 40, 1, 8, dtype=F32, scale=go_scale)
    see = R.visible(40, 90, (0, 50), 0, [0] * 3, [90] * 3, gpu)
    want = R.attention(q, k, v, see, 2.0, F32, go)
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    out = cm.match_attention(q, k, v, window=(0, 50), scale=2.0, out_dtype=F32)
    R.check(out, want["out"], "out")
    for got, n in zip(torch.autograd.grad(out, (q, k, v), go), ("dq", "dk", "dv")):
        R.check(got, want[n], n)


def test_attention_gradient_against_differences(gpu):
    """<gradient, d> against (f(x + h d) - f(x - h d)) / 2h of the 64-bit formula: the kernel's gradient is off by its
    bound against |d|, the difference by the third derivative (h = 1e-4: far below)."""
    g = _gen(11)
    q, k, v = (_rand(g, 1, n, 2, 64, dtype=BF16) for n in (40, 60, 60))
    go = _rand(g, 1, 40, 2, 64, dtype=BF16)
    see = R.visible(40, 60, (20, 0), 2, [0], [60], gpu)

    def f(q, k, v):
        s = torch.einsum("blhc,bmhc->bhlm", q, k) * 0.125
        P = torch.softmax(torch.where(see[:, None], s, -1e300), -1)
        return (torch.einsum("bhlm,bmhc->blhc", P, v) * go.double()).sum()

    want = R.attention(q, k, v, see, 0.125, BF16, go)
    x = [t.requires_grad_(True) for t in (q, k, v)]
    out = cm.match_attention(*x, window=(20, 0), sinks=2, scale=0.125)
    grads = torch.autograd.grad(out, x, go)
    for n, (t, gr) in enumerate(zip(x, grads)):
        d = torch.randn(t.shape, generator=g, device=gpu, dtype=torch.float64)
        lo, hi = ([y.detach().double() + (s * 1e-4 * d if m == n else 0.0) for m, y in enumerate(x)] for s in (-1, 1))
        slope = float((f(*hi) - f(*lo)) / 2e-4)
        bound = float((want[("dq", "dk", "dv")[n]][1] * d.abs()).sum())
        assert abs(float((gr.double() * d).sum()) - slope) <= bound + 1e-4 * abs(slope)


def test_attention_only_the_gradients_asked_for(gpu):
    g = _gen(5)
    q, k, v = (_rand(g, 2, n, 1, 64) for n in (30, 200, 200))
    go = _rand(g, 2, 30, 1, 64)
    full = [x.clone().requires_grad_(True) for x in (q, k, v)]
    ref = torch.autograd.grad(cm.match_attention(*full, window=(3, 50), sinks=1), full, go)
    for n in range(3):
        xs = [x.clone().requires_grad_(m == n) for m, x in enumerate((q, k, v))]
        got, = torch.autograd.grad(cm.match_attention(*xs, window=(3, 50), sinks=1), [xs[n]], go)
        assert torch.equal(got, ref[n])


def test_attention_empty(gpu):
    for B, Lq, Lk in ((0, 5, 5), (2, 0, 5), (2, 5, 0), (0, 0, 0)):
        q, k, v = (torch.ones(B, n, 2, 64, device=gpu, dtype=F16, requires_grad=True) for n in (Lq, Lk, Lk))
        out, lse = cm.match_attention(q, k, v, sinks=1, window=(1, 1), return_lse=True)
        assert out.shape == (B, Lq, 2, 64) and not out.any()
        assert (lse == float("-inf")).all()
        for x, gx in zip((q, k, v), torch.autograd.grad(out, (q, k, v), torch.ones_like(out))):
            assert gx.shape == x.shape and not gx.any()


def test_attention_rows_without_heads(gpu):
    g = _gen(2)
    q, k, v = _rand(g, 3, 20, 40), _rand(g, 3, 50, 40), _rand(g, 3, 50, 8)
    out = cm.match_attention(q, k, v, window=(0, 30), scale=1.0)
    ref = cm.match_attention(q.unsqueeze(2), k.unsqueeze(2), v.unsqueeze(2), window=(0, 30), scale=1.0)
    assert out.shape == (3, 20, 8) and torch.equal(out, ref.squeeze(2))


def test_attention_strides(gpu):
    """Slices of one projection, transposed heads, expanded (broadcast) keys, rows at odd addresses: same results as
    contiguous copies, and the gradients arrive in the views' places."""
    g = _gen(7)
    fused = _rand(g, 2, 77, (4 + 2 + 2) * 64, dtype=BF16).requires_grad_(True)
    go = _rand(g, 2, 77, 4, 64, dtype=BF16)

    def split(x):
        a, b, c = x.split([256, 128, 128], -1)
        return a.unflatten(-1, (4, 64)), b.unflatten(-1, (2, 64)), c.unflatten(-1, (2, 64))

    out = cm.match_attention(*split(fused), window=(9, 0), sinks=1)
    ref_in = [x.detach().contiguous().requires_grad_(True) for x in split(fused)]
    ref = cm.match_attention(*ref_in, window=(9, 0), sinks=1)
    assert torch.equal(out, ref)
    gf, = torch.autograd.grad(out, fused, go)
    for a, b in zip(split(gf), torch.autograd.grad(ref, ref_in, go)):
        assert torch.equal(a, b)
    # [B, heads, L, C] storage
    t = [x.detach().transpose(1, 2).contiguous().transpose(1, 2) for x in ref_in]
    assert torch.equal(cm.match_attention(*t, window=(9, 0), sinks=1), ref)
    # one key row for the whole batch: its gradient is the batch's sum
    k1 = ref_in[1][:1].detach().clone().requires_grad_(True)
    o1 = cm.match_attention(ref_in[0].detach(), k1.expand(2, -1, -1, -1), ref_in[2].detach())
    g1, = torch.autograd.grad(o1, k1, go)
    k2 = k1.detach().repeat(2, 1, 1, 1).requires_grad_(True)
    g2, = torch.autograd.grad(cm.match_attention(ref_in[0].detach(), k2, ref_in[2].detach()), k2, go)
    assert torch.equal(g1, g2.sum(0, keepdim=True))
    # an address that is not a multiple of 16 bytes
    flat = torch.empty(ref_in[0].numel() + 1, device=gpu, dtype=BF16)
    flat[1:] = ref_in[0].detach().flatten()
    odd = flat[1:].view_as(ref_in[0])
    assert odd.data_ptr() % 16 and torch.equal(cm.match_attention(odd, *ref_in[1:], window=(9, 0), sinks=1), ref)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attention_garbage_behind_the_length(gpu, bad):
    """Keys and values behind a sequence are never read, whatever they hold; their gradients are zeros."""
    g = _gen(9)
    q, k, v = (_rand(g, 2, n, 2, 64, dtype=BF16) for n in (40, 100, 100))
    go = _rand(g, 2, 40, 2, 64, dtype=BF16)
    length = torch.tensor([60, 1], device=gpu, dtype=torch.int32)
    res = []
    for fill in (0.0, bad):
        kk, vv = k.clone(), v.clone()
        for b, n in enumerate((60, 1)):
            kk[b, n:] = fill
            vv[b, n:] = fill
        x = [t.clone().requires_grad_(True) for t in (q, kk, vv)]
        out = cm.match_attention(*x, key_lengths=length, window=(50, 0), sinks=2)
        res.append([out, *torch.autograd.grad(out, x, go)])
    for a, b in zip(*res):
        assert torch.equal(a, b)
    assert not res[1][2][0, 60:].any() and not res[1][3][1, 1:].any()


@pytest.mark.parametrize("scale", [-0.3, 0.0, 5.0])
def test_attention_scales(gpu, scale):
    _attention_case(gpu, 2, 70, 133, 2, 1, 64, 64, (40, 0), 2, dtype=BF16, scale=scale)
    _attention_case(gpu, 2, 70, 133, 1, 1, 128, 8, (0, 40), 0, dtype=F16, out_dtype=F32, scale=scale)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("where", ["key", "value", "both"])
@pytest.mark.parametrize("C,Cv,out_dtype", [(64, 64, None), (128, 8, F32), (256, 256, None)])
def test_attention_values_that_are_not_finite(gpu, bad, where, C, Cv, out_dtype):
    """A key that holds inf or NaN touches the queries that see it and no other, forward and backward, though it shares
    their tiles: the others' outputs and gradients are what they are without it."""
    g = _gen(31)
    L, at = 150, 70
    q, k, v = (_rand(g, 1, L, 2, C, dtype=BF16), _rand(g, 1, L, 1, C, dtype=BF16), _rand(g, 1, L, 1, Cv, dtype=BF16))
    sees = R.visible(L, L, (20, 0), 0, [0], [L], gpu)[0, :, at]  # queries 70 .. 90
    go = _rand(g, 1, L, 2, Cv, dtype=out_dtype or BF16)
    go[:, sees] = 0.0  # no gradient through the touched queries' outputs (their rows' own are not looked at)
    res = []
    for poison in (False, True):
        kk, vv = k.clone(), v.clone()
        if poison and where != "value":
            kk[0, at, 0, 3] = bad
        if poison and where != "key":
            vv[0, at, 0, 1] = bad
        x = [t.clone().requires_grad_(True) for t in (q, kk, vv)]
        out = cm.match_attention(*x, window=(20, 0), out_dtype=out_dtype)
        res.append([out.detach(), *torch.autograd.grad(out, x, go)])
    clean, dirty = res
    assert torch.isfinite(clean[0]).all()
    assert torch.equal(clean[0][:, ~sees], dirty[0][:, ~sees])
    assert torch.equal(clean[1][:, ~sees], dirty[1][:, ~sees])
    if where != "key":
        assert not torch.isfinite(dirty[0][:, sees, :, 1]).any()
    if where == "value":  # only its own channel: the others' sums do not touch it
        keep = [c for c in range(Cv) if c != 1]
        assert torch.equal(clean[0][..., keep], dirty[0][..., keep])
    # keys that no touched query sees
    far = torch.ones(L, dtype=torch.bool, device=gpu)
    far[at - 20:at + 21] = False
    for n in (2, 3):
        assert torch.equal(clean[n][:, far], dirty[n][:, far])


def test_attention_queries_that_are_not_finite(gpu):
    """A query of NaN spoils its own output and the gradients of the keys that it sees."""
    g = _gen(37)
    L, at = 200, 100
    q, k, v = (_rand(g, 1, L, 1, 64, dtype=BF16) for _ in range(3))
    go = _rand(g, 1, L, 1, 64, dtype=BF16)
    res = []
    for poison in (False, True):
        qq = q.clone()
        if poison:
            qq[0, at] = float("nan")
        x = [t.clone().requires_grad_(True) for t in (qq, k, v)]
        out = cm.match_attention(*x, window=(20, 0))
        res.append([out.detach(), *torch.autograd.grad(out, x, go)])
    keep = torch.arange(L, device=gpu) != at
    far = (torch.arange(L, device=gpu) < at - 20) | (torch.arange(L, device=gpu) > at)
    for n, rows in ((0, keep), (1, keep), (2, far), (3, far)):
        assert torch.equal(res[0][n][:, rows], res[1][n][:, rows]), n
    assert not torch.isfinite(res[1][0][0, at]).any()


def test_attention_step_equals_prompt(gpu):
    """Generation one token at a time against a cache gives what the prompt form gives, within both bounds."""
    g = _gen(13)
    L, B = 150, 2
    q, k, v = (_rand(g, B, L, h, 64, dtype=BF16) for h in (6, 2, 2))
    see = R.visible(L, L, (40, 0), 4, [0] * B, [L] * B, gpu)
    want = R.attention(q, k, v, see, 0.125, BF16)["out"]
    cache_k, cache_v = (torch.full((B, 256, 2, 64), float("nan"), device=gpu, dtype=BF16) for _ in range(2))
    for t in range(L):
        cache_k[:, t], cache_v[:, t] = k[:, t], v[:, t]
        pos = torch.full((B,), t, device=gpu, dtype=torch.int32)
        out = cm.match_attention(q[:, t:t + 1], cache_k, cache_v, window=(40, 0), sinks=4, scale=0.125,
                                 query_offset=pos, key_lengths=pos + 1)
        R.check(out, (want[0][:, t:t + 1], want[1][:, t:t + 1]), f"token {t}")


def test_attention_offsets_past_32_bits(gpu):
    """A cache of more than 2^31 elements: the last keys, behind a window."""
    Lk, C = 9_000_000, 256
    assert Lk * C > 2 ** 31
    g = _gen(17)
    k = torch.zeros((1, Lk, 1, C), device=gpu, dtype=F16)
    v = torch.zeros((1, Lk, 1, C), device=gpu, dtype=F16)
    k[:, -300:], v[:, -300:] = _rand(g, 1, 300, 1, C), _rand(g, 1, 300, 1, C)
    q = _rand(g, 1, 2, 2, C)
    out = cm.match_attention(q, k, v, window=(200, 0), query_offset=Lk - 2)
    see = R.visible(2, 300, (200, 0), 0, [298], [300], gpu)
    R.check(out, R.attention(q, k[:, -300:], v[:, -300:], see, C ** -0.5, F16)["out"], "out")


def test_attention_is_deterministic(gpu):
    g = _gen(19)
    x = [_rand(g, 2, n, h, 128, dtype=BF16).requires_grad_(True) for n, h in ((500, 4), (700, 2), (700, 2))]
    go = _rand(g, 2, 500, 4, 128, dtype=BF16)
    runs = []
    for _ in range(3):
        out = cm.match_attention(*x, window=(300, 5), sinks=3)
        runs.append([out, *torch.autograd.grad(out, x, go)])
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


# ---- cross entropy ----

def _entropy_case(gpu, B, N, V, C, window=(None, None), dtype=F16, shared=False, seed=0, reduction="sum", scale=None):
    g = _gen(seed)
    scale = (4.0 / C ** 0.5) if scale is None else scale
    x = _rand(g, B, N, C, dtype=dtype)
    w = _rand(g, 1 if shared else B, V, C, dtype=dtype)
    target = torch.randint(-1, V + 1, (B, N), generator=g, device=gpu)
    see = R.visible(N, V, window, 0, [0], [V], gpu)
    weight = torch.ones(B, N, device=gpu)
    if reduction == "none":
        weight = torch.randn((B, N), generator=g, device=gpu)
    wide = w.expand(B, V, C) if shared else w
    want = R.entropy(x, wide, target, see, scale, weight)
    count = int(want["counts"].sum())
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    arg = w[0] if shared else w
    loss = cm.match_cross_entropy(x, arg, target, scale=scale, window=window, reduction=reduction)
    value, bound = want["loss"]
    if reduction == "none":
        R.check(loss, want["loss"], "loss")
        dx, dw = torch.autograd.grad(loss, (x, w), weight)
        f = 1.0
    else:
        f = 1.0 if reduction == "sum" else 1.0 / max(1, count)
        R.check(loss, (value.sum() * f, bound.sum() * f + abs(float(value.sum() * f)) * 2.0 ** -22), "loss")
        dx, dw = torch.autograd.grad(loss, (x, w), torch.tensor(1.0, device=gpu))
    tiny = R.TINY[dtype]
    scaled = lambda p: (p[0] * f, p[1] * f * (1 + 2.0 ** -20) + tiny)  # noqa: E731
    R.check(dx, scaled(want["dx"]), "dx")
    want_dw = want["dw"]
    if shared and B > 1:
        flat = R.entropy(x.detach().reshape(1, B * N, C), w.detach(), target.reshape(1, -1), see.new_ones((1, 1, V)), scale,
                         weight.reshape(1, -1))
        want_dw = flat["dw"]
    R.check(dw, scaled(want_dw), "dw")
    return count


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("C", [8, 32, 64, 128, 256, 49, 121, 232, 1])
def test_entropy_channels(gpu, dtype, C):
    _entropy_case(gpu, 2, 70, 150, C, dtype=dtype)


@pytest.mark.parametrize("window", [(0, 0), (0, 40), (0, 200), (7, None), (30, 3), (None, 0), (500, 500)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_entropy_windows(gpu, window, dtype):
    _entropy_case(gpu, 3, 200, 261, 64, window, dtype=dtype)
    _entropy_case(gpu, 2, 130, 130, 128, window, dtype=dtype, reduction="none")


@pytest.mark.parametrize("N,V", [(1, 1), (1, 3000), (33, 1), (129, 127), (500, 2000), (2, 50000)])
def test_entropy_sizes(gpu, N, V):
    _entropy_case(gpu, 1, N, V, 64, dtype=BF16, shared=True, seed=N)
    _entropy_case(gpu, 1, N, V, 264, dtype=BF16, shared=True, seed=N)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("N,V,C", [(1, 1000, 512), (255, 257, 264), (256, 256, 320), (300, 1500, 1000), (700, 5003, 768),
                                   (40, 20011, 2048), (257, 300, 4104)])
def test_entropy_wide_vectors(gpu, dtype, N, V, C):
    _entropy_case(gpu, 1, N, V, C, dtype=dtype, shared=True)


@pytest.mark.parametrize("C", [64, 512])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("shared", [False, True])
def test_entropy_reductions(gpu, C, reduction, shared):
    assert _entropy_case(gpu, 3, 90, 333, C, dtype=BF16, shared=shared, reduction=reduction) > 100


def test_entropy_pieces(gpu):
    """Enough rows that the classes are taken in several pieces (128 MiB of 16-bit scores a piece)."""
    _entropy_case(gpu, 1, 20000, 4000, 264, dtype=BF16, shared=True, reduction="mean")


def test_entropy_nothing_counts(gpu):
    for C in (64, 512):
        x = torch.ones(1, 50, C, device=gpu, dtype=BF16, requires_grad=True)
        w = torch.ones(1, 70, C, device=gpu, dtype=BF16, requires_grad=True)
        for reduction in ("mean", "sum", "none"):
            for t in (-1, -100, 70, 2 ** 40):
                loss = cm.match_cross_entropy(x, w, torch.full((1, 50), t, device=gpu), reduction=reduction)
                assert not loss.any()
                dx, dw = torch.autograd.grad(loss.sum(), (x, w))
                assert not dx.any() and not dw.any()
    # a target that exists but lies outside its query's window
    x, w = x[..., :64].detach().requires_grad_(True), w[..., :64].detach().requires_grad_(True)
    loss = cm.match_cross_entropy(x, w, torch.full((1, 50), 60, device=gpu), window=(0, 5))
    assert float(loss) == 0.0 and not torch.autograd.grad(loss, w)[0].any()


def test_entropy_empty(gpu):
    for C in (64, 512):
        for N, V in ((0, 5), (5, 0), (0, 0)):
            x = torch.ones(N, C, device=gpu, dtype=F16, requires_grad=True)
            w = torch.ones(V, C, device=gpu, dtype=F16, requires_grad=True)
            loss = cm.match_cross_entropy(x, w, torch.zeros(N, device=gpu, dtype=torch.int64))
            assert float(loss) == 0.0
            dx, dw = torch.autograd.grad(loss, (x, w))
            assert not dx.any() and not dw.any() and dw.shape == (V, C)


@pytest.mark.parametrize("C", [64, 512])
def test_entropy_confident_and_ignored_rows(gpu, C):
    """Scores of thousands (probabilities of exactly 0 and 1), and NaN in a row that does not count."""
    g = _gen(23)
    x, w = _rand(g, 1, 130, C, dtype=BF16, scale=30.0), _rand(g, 1, 400, C, dtype=BF16, scale=30.0)
    t = torch.randint(0, 400, (1, 130), generator=g, device=gpu)
    t[:, ::3] = -1
    x[:, 0] = float("nan")
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    loss = cm.match_cross_entropy(x, w, t, reduction="none")
    ref = R.entropy(x[:, 1:].detach(), w.detach(), t[:, 1:], torch.ones(1, 129, 400, dtype=torch.bool, device=gpu), 1.0,
                    torch.ones(1, 129, device=gpu))
    R.check(loss[:, 1:], ref["loss"], "loss")
    assert float(loss[0, 0]) == 0.0
    dx, dw = torch.autograd.grad(loss.sum(), (x, w))
    R.check(dx[:, 1:], ref["dx"], "dx")
    assert not dx[:, 0].any()


# ---- descriptors ----

@pytest.mark.parametrize("k", [1, 2, 3, 5, 8, 9, 11, 15, 16])
@pytest.mark.parametrize("image_dtype,dtype", [(F32, F16), (F32, BF16), (F16, F16), (F16, BF16)])
def test_descriptors(gpu, k, image_dtype, dtype):
    g = _gen(k)
    for H, W in ((1, 1), (3, 65), (40, 130), (70, 64)):
        img = torch.rand((H, W), generator=g, device=gpu).to(image_dtype)
        if H > 20:
            img[4:30, 10:50] = 0.5  # flat: unit vectors of nothing
        go = _rand(g, H, W, -(-k * k // 8) * 8, dtype=dtype)
        want = R.descriptors(img, k, dtype, go)
        img.requires_grad_(True)
        d = cm.zncc_descriptors(img, k, dtype)
        assert d.dtype == dtype
        R.check(d, want["d"], f"d {H}x{W}")
        gi, = torch.autograd.grad(d, img, go)
        assert gi.dtype == image_dtype
        R.check(gi, want["dI"], f"dI {H}x{W}")


def test_descriptors_many_bands(gpu):
    """Several strips and bands of the backward, each image row from one owner."""
    g = _gen(29)
    img = torch.rand((300, 500), generator=g, device=gpu)
    go = _rand(g, 300, 500, 128)
    want = R.descriptors(img, 11, F16, go)["dI"]
    img.requires_grad_(True)
    R.check(torch.autograd.grad(cm.zncc_descriptors(img, 11), img, go)[0], want, "dI")


def test_descriptors_score_like_the_volume(gpu):
    from tests.golden.inputs import make_pair

    c, p = (torch.from_numpy(x).to(gpu) for x in make_pair(24, 96, 20, seed=4))
    vol = cm.stereo_matching(c, p, 0, 9)
    dc, dp = cm.zncc_descriptors(c, 9).float(), cm.zncc_descriptors(p, 9).float()
    # two vectors rounded to fp16: off by at most 2 (2^-11 + 2^-22) of sum |c p| <= 1; epsilon is placed differently
    assert float((torch.bmm(dc, dp.transpose(1, 2).contiguous()) - vol).abs().max()) <= 2 * 2.0 ** -11 + 2e-5
