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


@pytest.mark.parametrize("window", [(1 << 40, 1 << 40), ((1 << 31) - 1, (1 << 31) - 1), (1 << 30, (1 << 30) - 1)])
def test_attention_bounds_and_positions_at_their_ends(gpu, window):
    """Windows and positions of 2^30 and more: what each query sees is the rule's, in Python integers."""
    for off in (-(1 << 30), -(1 << 30) + 7, (1 << 30) - 7, 1 << 30, 0):
        _attention_case(gpu, 1, 40, 50, 2, 1, 32, 32, window, 3, offset=[off], dtype=BF16)


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
    assert float(loss.detach()) == 0.0 and not torch.autograd.grad(loss, w)[0].any()


def test_entropy_empty(gpu):
    for C in (64, 512):
        for N, V in ((0, 5), (5, 0), (0, 0)):
            x = torch.ones(N, C, device=gpu, dtype=F16, requires_grad=True)
            w = torch.ones(V, C, device=gpu, dtype=F16, requires_grad=True)
            loss = cm.match_cross_entropy(x, w, torch.zeros(N, device=gpu, dtype=torch.int64))
            assert float(loss.detach()) == 0.0
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


def test_descriptors_gradient_against_differences(gpu):
    """As for the attention: the 64-bit formula's difference along a direction, and the gradient's bound against it."""
    g = _gen(31)
    img = torch.rand((20, 70), generator=g, device=gpu)
    go = _rand(g, 20, 70, 56)

    def f(x):
        x = torch.nn.functional.pad(x, (3, 3, 3, 3)).unfold(0, 7, 1).unfold(1, 7, 1).reshape(20, 70, 49)
        c = x - x.mean(-1, keepdim=True)
        return (c * (c.square().sum(-1, keepdim=True) + 1e-8).rsqrt() * go[..., :49].double()).sum()

    bound = R.descriptors(img, 7, F16, go)["dI"][1]
    d = torch.randn((20, 70), generator=g, device=gpu, dtype=torch.float64)
    x = img.double()
    slope = float((f(x + 1e-5 * d) - f(x - 1e-5 * d)) / 2e-5)
    img.requires_grad_(True)
    got, = torch.autograd.grad(cm.zncc_descriptors(img, 7), img, go)
    # differences: h^2 / 6 of a third derivative of a few times (|d| / norm)^3 |go|, norms above 0.5 here: below 1e-5
    assert abs(float((got.double() * d).sum()) - slope) <= float((bound * d.abs()).sum()) + 1e-5 * (1 + abs(slope))


def test_entropy_gradient_against_differences(gpu):
    g = _gen(32)
    x, w = _rand(g, 2, 30, 64, dtype=BF16), _rand(g, 2, 50, 64, dtype=BF16)
    target = torch.randint(0, 50, (2, 30), generator=g, device=gpu)
    see = R.visible(30, 50, (4, 30), 0, [0], [50], gpu)
    ref = R.entropy(x, w, target, see, 0.2, torch.ones((2, 30), device=gpu))

    def f(x, w):
        s = torch.where(see, torch.bmm(x, w.transpose(1, 2).contiguous()) * 0.2, -1e300)
        loss = torch.logsumexp(s, -1) - s.gather(-1, target[..., None])[..., 0]
        return torch.where(ref["counts"], loss, 0.0).sum()

    xs = [x.requires_grad_(True), w.requires_grad_(True)]
    grads = torch.autograd.grad(cm.match_cross_entropy(*xs, target, scale=0.2, window=(4, 30), reduction="sum"), xs)
    for n, (t, gr) in enumerate(zip(xs, grads)):
        d = torch.randn(t.shape, generator=g, device=gpu, dtype=torch.float64)
        lo, hi = ([y.detach().double() + (s * 1e-4 * d if m == n else 0.0) for m, y in enumerate(xs)] for s in (-1, 1))
        slope = float((f(*hi) - f(*lo)) / 2e-4)
        bound = float((ref[("dx", "dw")[n]][1] * d.abs()).sum())
        assert abs(float((gr.double() * d).sum()) - slope) <= bound + 1e-4 * abs(slope)


# ---- the operators together, on image pairs ----

def _pair(gpu, H, W, seed):
    from tests.golden.inputs import make_pair

    return [torch.from_numpy(x).to(gpu) for x in make_pair(H, W, 20, seed=seed)]


def _through_descriptors(img, k, dd):
    """The image gradient, with bound, of descriptor gradients dd = (value, bound): the descriptors' Jacobian is
    s (I - 1/K - d d^T), so an error e of dd gives at most s (e + mean e + (e . |d|) |d|) on each tap."""
    K = k * k
    value, bound = dd
    ref = R.descriptors(img, k, F16, value)
    o = k // 2
    pad = torch.nn.functional.pad(img.double(), (o, k - 1 - o, o, k - 1 - o))
    H, W = img.shape
    x = pad.unfold(0, k, 1).unfold(1, k, 1).reshape(H, W, K)
    c = x - x.mean(-1, keepdim=True)
    s = (c.square().sum(-1, keepdim=True) + 1e-8).rsqrt()
    d, e = (c * s).abs(), bound[..., :K]
    term = s * (e + e.mean(-1, keepdim=True) + (e * d).sum(-1, keepdim=True) * d)
    acc = torch.zeros_like(pad)
    for t in range(K):
        acc[t // k:t // k + H, t % k:t % k + W] += term[..., t]
    return ref["dI"][0], ref["dI"][1] + 1.001 * acc[o:o + H, o:o + W]


def _wide(x, W):
    """Rows behind WO have no gradient."""
    return tuple(torch.nn.functional.pad(t, (0, 0, 0, W - t.shape[1])) for t in x)


@pytest.mark.parametrize("layout", ["full", "window"])
@pytest.mark.parametrize("size", [1.0, 1e-9])
def test_soft_disparity(gpu, layout, size):
    """Against the 64-bit formulas on the float16 descriptors, and gradients that keep their accuracy at any size."""
    H, W, D, k, beta = 17, 90, 30, 7, 20.0
    cam, proj = _pair(gpu, H, W, 6)
    WO, window = (W, (None, None)) if layout == "full" else (W - D, (0, D))
    g = torch.randn((H, WO), generator=_gen(33), device=gpu) * size
    dc, dp = cm.zncc_descriptors(cam, k), cm.zncc_descriptors(proj, k)
    j = torch.arange(W, device=gpu)
    v = torch.zeros((H, W, 1, 8), device=gpu, dtype=F16)
    v[..., 1] = j[None, :, None].half()  # below 2048: the first part is 0
    go = torch.zeros((H, WO, 1, 8), device=gpu)
    go[:, :, 0, 0], go[:, :, 0, 1] = 2048 * g, g
    unit = 2.0 ** torch.frexp(go.abs().max()).exponent.double()
    see = R.visible(WO, W, window, 0, [0] * H, [W] * H, gpu)
    ref = R.attention(dc[:, :WO, None], dp[:, :, None], v, see, beta, F32, (go / unit).float())
    cam.requires_grad_(True)
    proj.requires_grad_(True)
    got = cm.stereo_soft_disparity(cam, proj, D, k, layout=layout, beta=beta)
    assert got.shape == (H, WO) and got.dtype == F32
    value, bound = (x[:, :, 0] for x in ref["out"])
    first = torch.arange(WO, device=gpu, dtype=torch.float64) if layout == "window" else 0.0
    R.check(got, (value[..., 1] - first, 2048 * bound[..., 0] + bound[..., 1] + 2.0 ** -22 * W), "soft")
    gc, gp = torch.autograd.grad(got, (cam, proj), g)
    for img, got, name in ((cam, gc, "dq"), (proj, gp, "dk")):
        value, bound = _through_descriptors(img.detach(), k, _wide([x[:, :, 0] for x in ref[name]], W))
        R.check(got, (value * unit, bound * unit), name)


@pytest.mark.parametrize("layout", ["full", "window"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_match_loss(gpu, layout, reduction):
    H, W, D, k, beta = 17, 90, 30, 7, 20.0
    cam, proj = _pair(gpu, H, W, 7)
    WO, window = (W, (None, None)) if layout == "full" else (W - D, (0, D))
    rng = _gen(34)
    target = torch.randint(-3, W + 3 if layout == "full" else D + 4, (H, WO), generator=rng, device=gpu)
    size = torch.rand((H, WO) if reduction == "none" else (), generator=rng, device=gpu) * 1e-8
    dc, dp = cm.zncc_descriptors(cam, k), cm.zncc_descriptors(proj, k)
    valid = (target >= 0) & (target <= (W - 1 if layout == "full" else D))
    column = torch.where(valid, target + (torch.arange(WO, device=gpu) if layout == "window" else 0), -1)
    see = R.visible(WO, W, window, 0, [0], [W], gpu)
    if reduction == "none":  # the largest weight in [1, 2)
        unit = 2.0 ** (torch.frexp(size.max()).exponent.double() - 1)
        weight = (size / unit).float()
    else:
        unit = size.double() / (valid.sum() if reduction == "mean" else 1)
        weight = torch.ones((H, WO), device=gpu)
    ref = R.entropy(dc[:, :WO], dp, column, see, beta, weight)
    assert bool((ref["counts"] == valid).all())
    cam.requires_grad_(True)
    proj.requires_grad_(True)
    loss = cm.stereo_match_loss(cam, proj, target, D, k, layout=layout, beta=beta, reduction=reduction)
    value, bound = ref["loss"]
    if reduction == "none":
        R.check(loss, (value, bound), "loss")
    else:
        n = valid.sum() if reduction == "mean" else 1
        R.check(loss, (value.sum() / n, (bound.sum() + 2.0 ** -22 * value.abs().sum()) / n), "loss")
    gc, gp = torch.autograd.grad(loss, (cam, proj), size)
    for img, got, name in ((cam, gc, "dx"), (proj, gp, "dw")):
        value, bound = _through_descriptors(img.detach(), k, _wide(ref[name], W))
        R.check(got, (value * unit, (bound + 2.0 ** -21 * value.abs()) * unit), name)  # the unit's own 32-bit roundings


@pytest.mark.parametrize("layout", ["full", "window"])
def test_pair_operators_beside_the_volume(gpu, layout):
    """Costs of float16 descriptors are within delta of the volume's, so the softmax's weights are within
    exp(+-2 beta delta) and the disparity and the loss within what that allows."""
    H, W, D, k, beta = 24, 96, 20, 9, 50.0
    cam, proj = _pair(gpu, H, W, 4)
    delta = 2 * 2.0 ** -11 + 4e-5  # as in test_descriptors_score_like_the_volume, and the scores' 32-bit sums
    index = cm.stereo_disparity(cam, proj, D, k, layout=layout)[0]
    cost = cm.stereo_matching(cam, proj, D, k, layout).double()
    P = torch.softmax(beta * cost, -1)
    s = torch.arange(cost.shape[-1], device=gpu, dtype=torch.float64)
    mean = (P * s).sum(-1)
    spread = (P * (s - mean[..., None]).abs()).sum(-1)
    grow = torch.tensor(2 * beta * delta).expm1().item()
    got = cm.stereo_soft_disparity(cam, proj, D, k, layout=layout, beta=beta)
    assert bool(((got.double() - mean).abs() <= grow * spread + 1e-4).all())
    loss = cm.stereo_match_loss(cam, proj, index, D, k, layout=layout, beta=beta, reduction="none")
    want = -torch.log(P).gather(-1, index[..., None])[..., 0]
    assert bool(((loss.double() - want).abs() <= 2 * beta * delta + 1e-5).all())


@pytest.mark.parametrize("image_dtype", [F32, F16])
def test_pair_operators_in_one_step(gpu, image_dtype):
    """A training step on both: the gradient of the sum is the sum of the gradients; a second backward gives the same."""
    cam, proj = (x.to(image_dtype).requires_grad_(True) for x in _pair(gpu, 20, 100, 8))
    index, _ = cm.stereo_disparity(cam.detach(), proj.detach(), 25, 9, layout="window")[:2]

    def parts():
        a = cm.stereo_match_loss(cam, proj, index, 25, 9, layout="window")
        b = (cm.stereo_soft_disparity(cam, proj, 25, 9, layout="window") - index).abs().mean()
        return a, b

    a, b = parts()
    ga, gb = (torch.autograd.grad(x, (cam, proj), retain_graph=True) for x in (a, b))
    both = torch.autograd.grad(a + b, (cam, proj), retain_graph=True)
    again = torch.autograd.grad(a + b, (cam, proj))
    for x, y, z, w in zip(ga, gb, both, again):
        assert torch.equal(x + y, z) and torch.equal(z, w) and bool(z.any())
    only, = torch.autograd.grad(parts()[0], [proj])
    assert torch.equal(only, ga[1])


def test_pair_operators_empty_and_flat(gpu):
    e = torch.zeros((0, 40), device=gpu, requires_grad=True)
    soft = cm.stereo_soft_disparity(e, e, 8, 5, layout="window")
    assert soft.shape == (0, 32)
    loss = cm.stereo_match_loss(e, e, torch.zeros((0, 32), dtype=torch.int64, device=gpu), 8, 5, layout="window")
    assert float(loss.detach()) == 0.0 and torch.autograd.grad(loss + soft.sum(), e)[0].shape == (0, 40)
    f = torch.full((6, 40), 0.25, device=gpu, requires_grad=True)  # the borders of a flat image still see zeros outside
    soft = cm.stereo_soft_disparity(f, f, 8, 1, layout="window")
    assert bool(((soft - 4.0).abs() < 1e-4).all())  # one tap: nothing to tell columns apart
    assert not torch.autograd.grad(soft.sum(), f)[0].any()


# ---- streams and graphs ----

def _calls(gpu):
    """name -> (inputs, function of the inputs, output gradient or None): one call of each operator and kind."""
    g = _gen(41)
    q, k, v = (_rand(g, 2, 70, h, 64, dtype=BF16) for h in (4, 2, 2))
    rows = [_rand(g, 3, n, 128) for n in (60, 90)]
    value = _rand(g, 3, 90, 8)
    target = torch.randint(-1, 90, (3, 60), generator=g, device=gpu)
    wide = [_rand(g, 100, 512, dtype=BF16), _rand(g, 700, 512, dtype=BF16)]
    wide_t = torch.randint(-1, 700, (100,), generator=g, device=gpu)
    step = [_rand(g, 2, n, h, 128, dtype=BF16) for n, h in ((1, 8), (1500, 2), (1500, 2))]
    at, n = torch.tensor([1499, 30], device=gpu), torch.tensor([1500, 31], device=gpu)
    images = _pair(gpu, 20, 80, 9)
    index = torch.randint(-1, 21, (20, 60), generator=g, device=gpu)
    return {
        "attention": ((q, k, v), lambda q, k, v: cm.match_attention(q, k, v, window=(40, 0), sinks=2)),
        "rows": ((*rows, value), lambda q, k, v: cm.match_attention(q, k, v, window=(0, 30), scale=0.3, out_dtype=F32)),
        "step": (tuple(step), lambda q, k, v: cm.match_attention(q, k, v, window=(None, 0), query_offset=at, key_lengths=n)),
        "entropy": (tuple(rows), lambda x, w: cm.match_cross_entropy(x, w, target, scale=0.1, window=(0, 30))),
        "entropy_none": (tuple(rows), lambda x, w: cm.match_cross_entropy(x, w, target, scale=0.1, reduction="none")),
        "entropy_wide": (tuple(wide), lambda x, w: cm.match_cross_entropy(x, w, wide_t, scale=0.05)),
        "descriptors": ((images[0],), lambda x: cm.zncc_descriptors(x, 9)),
        "disparity": (tuple(images), lambda c, p: cm.stereo_soft_disparity(c, p, 20, 9, layout="window")),
        "loss": (tuple(images), lambda c, p: cm.stereo_match_loss(c, p, index, 20, 9, layout="window")),
    }


def _run(fn, inputs, go):
    leaves = [x.detach().requires_grad_(True) for x in inputs]  # new leaves: no older graph holds them
    out = fn(*leaves)
    return (out.detach(), *torch.autograd.grad(out, leaves, go))


CALLS = ["attention", "rows", "step", "entropy", "entropy_none", "entropy_wide", "descriptors", "disparity", "loss"]


def _case(gpu, name):
    inputs, fn = _calls(gpu)[name]
    out = fn(*inputs)
    return inputs, fn, torch.randn(out.shape, generator=_gen(42), device=gpu).to(out.dtype)


@pytest.mark.parametrize("name", CALLS)
def test_on_a_side_stream(gpu, name):
    inputs, fn, go = _case(gpu, name)
    want = _run(fn, inputs, go)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    results = []
    for s in (side, other, side):  # two streams at work at once, each call with its own workspace
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            results.append(_run(fn, inputs, go))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.current_stream().wait_stream(other)
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", CALLS)
def test_captured_and_replayed(gpu, name):
    """Forward and backward in two graphs, replayed in turn on new inputs with eager work between."""
    inputs, fn, go = _case(gpu, name)
    graphs = []
    for _ in range(2):
        held = [x.clone() for x in inputs]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            _run(fn, held, go)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = _run(fn, held, go)
        graphs.append((graph, held, outs))
    for turn in range(3):
        fresh = [[(x * (1.0 - 0.1 * turn - 0.03 * n)).to(x.dtype) for x in inputs] for n in range(2)]
        for (graph, held, _), new in zip(graphs, fresh):
            for h, x in zip(held, new):
                h.copy_(x)
            graph.replay()
        eager = [_run(fn, new, go) for new in fresh]
        torch.cuda.synchronize()
        for (_, _, outs), want in zip(graphs, eager):
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), (name, turn)


def test_same_tensor_everywhere(gpu):
    """Query, key and value one tensor: the gradient is the sum of the three."""
    x = _rand(_gen(43), 2, 80, 2, 64, dtype=BF16).requires_grad_(True)
    go = _rand(_gen(44), 2, 80, 2, 64, dtype=BF16)
    got, = torch.autograd.grad(cm.match_attention(x, x, x, window=(20, 0)), x, go)
    three = [x.detach().clone().requires_grad_(True) for _ in range(3)]
    a, b, c = torch.autograd.grad(cm.match_attention(*three, window=(20, 0)), three, go)
    # the engine adds three bfloat16 gradients in an order of its own: two roundings
    want = a.double() + b.double() + c.double()
    assert bool(((got.double() - want).abs() <= 2 * 2.0 ** -8 * (a.abs() + b.abs() + c.abs()).double()).all())


def test_loss_may_be_edited_in_place(gpu):
    x, w = (_rand(_gen(45), 40, 64).requires_grad_(True) for _ in range(2))
    target = torch.arange(40, device=gpu)
    for reduction in ("mean", "sum", "none"):
        ref = torch.autograd.grad(cm.match_cross_entropy(x, w, target, reduction=reduction).sum() * 2, x)[0]
        loss = cm.match_cross_entropy(x, w, target, reduction=reduction)
        loss.mul_(2)
        assert torch.equal(torch.autograd.grad(loss.sum(), x)[0], ref)


def test_from_two_threads(gpu):
    """Calls from two host threads at once, each on a stream of its own."""
    import threading

    cases = {n: _case(gpu, n) for n in ("attention", "entropy_wide", "loss")}
    want = {n: _run(fn, inputs, go) for n, (inputs, fn, go) in cases.items()}
    torch.cuda.synchronize()
    got, errors = [{}, {}], []

    def work(n):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for name, (inputs, fn, go) in cases.items():
                    got[n][name] = _run(fn, inputs, go)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for g in got:
        assert all(torch.equal(a, b) for n in cases for a, b in zip(g[n], want[n]))


@pytest.mark.parametrize("kind", [int, torch.int32, torch.int64])
def test_positions_and_lengths_of_any_kind(gpu, kind):
    """An int, or a tensor of either width; a padded batch's keys behind the length get zero gradients."""
    g = _gen(46)
    q, k, v = (_rand(g, 2, n, 2, 64, dtype=BF16).requires_grad_(True) for n in (12, 200, 200))
    go = _rand(g, 2, 12, 2, 64, dtype=BF16)
    off, n = (80, 93) if kind is int else (torch.full((2,), x, dtype=kind, device=gpu) for x in (80, 93))
    out = cm.match_attention(q, k, v, window=(30, 0), sinks=2, query_offset=off, key_lengths=n)
    ref = cm.match_attention(q, k[:, :93], v[:, :93], window=(30, 0), sinks=2, query_offset=80)
    assert torch.equal(out, ref)
    for a, b in zip(torch.autograd.grad(out, (q, k, v), go), torch.autograd.grad(ref, (q, k, v), go)):
        assert torch.equal(a, b)
    dk = torch.autograd.grad(cm.match_attention(q, k, v, window=(30, 0), query_offset=off, key_lengths=n), k, go)[0]
    assert not dk[:, 93:].any() and not dk[:, :50].any() and bool(dk[:, 50:92].any())


# ---- refusals ----

def test_refusals(gpu):
    z = lambda *s, dtype=F16: torch.zeros(s, dtype=dtype, device=gpu)  # noqa: E731
    q, k, v = z(2, 5, 4, 16), z(2, 9, 2, 16), z(2, 9, 2, 8)
    for args, kw, exc in [
        ((q.float(), k, v), {}, RuntimeError), ((q, k.bfloat16(), v), {}, RuntimeError), ((q, k.cpu(), v), {}, RuntimeError),
        ((q[0, 0], k, v), {}, RuntimeError), ((q[0], k, v), {}, RuntimeError), ((q, k[:1], v), {}, RuntimeError),
        ((q, k[..., :8], v), {}, RuntimeError), ((q, k, v[:, :8]), {}, RuntimeError), ((q[:, :, :3], k, v), {}, ValueError),
        ((q, k[:, :, :0], v[:, :, :0]), {}, ValueError), ((z(1, 1, 1, 257), z(1, 1, 1, 257), v), {}, RuntimeError),
        ((z(1, 1, 1, 257), z(1, 1, 1, 257), z(1, 1, 1, 8)), {}, ValueError), ((z(1, 1, 1, 0), z(1, 1, 1, 0), z(1, 1, 1, 8)), {}, ValueError),
        ((q, k, v), dict(window=(1,)), ValueError), ((q, k, v), dict(window=(-1, 0)), ValueError),
        ((q, k, v), dict(window=(1.5, 0)), TypeError), ((q, k, v), dict(sinks=-1), ValueError), ((q, k, v), dict(sinks=1.0), TypeError),
        ((q, k, v), dict(scale=float("nan")), ValueError), ((q, k, v), dict(scale=1e39), ValueError),
        ((q, k, v), dict(out_dtype=BF16), ValueError), ((q, k, v), dict(out_dtype=torch.float64), ValueError),
        ((q, k, v), dict(query_offset=[0, 0]), TypeError), ((q, k, v), dict(query_offset=torch.zeros(2, device=gpu)), TypeError),
        ((q, k, v), dict(key_lengths=torch.zeros(3, dtype=torch.int32, device=gpu)), ValueError),
        ((q, k, v), dict(key_lengths=torch.zeros(2, dtype=torch.int32)), RuntimeError), ((q, k, v), dict(key_lengths=1 << 31), ValueError),
    ]:
        with pytest.raises(exc):
            cm.match_attention(*args, **kw)
    x, w, t = z(3, 7, 16), z(3, 9, 16), torch.zeros((3, 7), dtype=torch.int64, device=gpu)
    for args, kw, exc in [
        ((x.float(), w, t), {}, RuntimeError), ((x, w.bfloat16(), t), {}, RuntimeError), ((x, w[:2], t), {}, RuntimeError),
        ((x, w[..., :8], t), {}, RuntimeError), ((x, w, t.float()), {}, TypeError), ((x, w, t[:2]), {}, RuntimeError),
        ((x, w, t.cpu()), {}, RuntimeError), ((x, w, t), dict(reduction="max"), ValueError), ((x, w, t), dict(window=(0, -1)), ValueError),
        ((x, w[0], t), dict(window=(0, 3)), ValueError), ((x[0], w, t[0]), {}, RuntimeError),
        ((z(1, 4, 264), z(1, 4, 264), t[:1, :4]), dict(window=(0, 2)), ValueError), ((z(4, 16392), z(4, 16392), t[0, :4]), {}, ValueError),
    ]:
        with pytest.raises(exc):
            cm.match_cross_entropy(*args, **kw)
    img = torch.zeros((6, 20), device=gpu)
    for args, exc in [((img.cpu(), 3), RuntimeError), ((img[0], 3), RuntimeError), ((img.t(), 3), RuntimeError),
                      ((img, 17), ValueError), ((img, 0), ValueError), ((img, 3.0), TypeError), ((img, 3, F32), RuntimeError),
                      ((img.double(), 3), RuntimeError), (([1.0], 3), TypeError)]:
        with pytest.raises(exc):
            cm.zncc_descriptors(*args)
    t = torch.zeros((6, 20), dtype=torch.int64, device=gpu)
    with pytest.raises(ValueError):
        cm.stereo_soft_disparity(img, img, 20, 3, layout="window")
    with pytest.raises(ValueError):
        cm.stereo_soft_disparity(img, img, 4, 3, beta=0.0)
    with pytest.raises(ValueError):
        cm.stereo_match_loss(img, img, t, 4, 3, layout="rows")
    with pytest.raises(RuntimeError):
        cm.stereo_match_loss(img, img, t, 4, 3, layout="window")
    with pytest.raises(TypeError):
        cm.stereo_match_loss(img, img, t.float(), 4, 3)
    with pytest.raises(ValueError):
        cm.stereo_match_loss(img, img, t, 4, 3, reduction="max")
