"""The matching operators on the GPU: values that are not finite outside of what they may reach, and calls at the edges of
what the documentation allows.  References and tolerances as in test_gpu_matching.py."""
import pytest
import torch

import custereomatching_amd as cm
from tests import matching_ref as R

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rand(g, *shape, dtype=F16, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


# ---- cross entropy: rows that do not count ----

@pytest.mark.parametrize("C", [64, 256, 264, 512])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("dtype,reduction", [(BF16, "mean"), (F16, "sum"), (BF16, "none")])
def test_entropy_gradients_beside_ignored_rows(gpu, C, bad, dtype, reduction):
    """Rows without a target, or of weight 0, hold inf or NaN: both gradients are what they are without these rows."""
    g = _gen(51)
    N, V, scale = 330, 600, 4.0 / C ** 0.5
    x, w = _rand(g, 1, N, C, dtype=dtype), _rand(g, 1, V, C, dtype=dtype)
    t = torch.randint(0, V, (1, N), generator=g, device=gpu)
    weight = torch.rand((1, N), generator=g, device=gpu) + 0.5 if reduction == "none" else torch.ones((1, N), device=gpu)
    t[:, ::5] = -100
    if reduction == "none":
        weight[:, 3::7] = 0.0
    keep = (t[0] >= 0) & (weight[0] != 0)
    x[:, ~keep] = bad
    see = torch.ones((1, 1, V), dtype=torch.bool, device=gpu)
    want = R.entropy(x[:, keep], w, t[:, keep], see, scale, weight[:, keep])
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    loss = cm.match_cross_entropy(x, w, t, scale=scale, reduction=reduction)
    dx, dw = torch.autograd.grad(loss, (x, w), weight if reduction == "none" else torch.tensor(1.0, device=gpu))
    f = 1.0 / int(keep.sum()) if reduction == "mean" else 1.0
    scaled = lambda p: (p[0] * f, p[1] * f * (1 + 2.0 ** -20) + R.TINY[dtype])  # noqa: E731
    R.check(dw, scaled(want["dw"]), "dw")
    R.check(dx[:, keep], scaled(want["dx"]), "dx")
    assert not dx[:, ~keep].any()


@pytest.mark.parametrize("C", [64, 512])
@pytest.mark.parametrize("bad", [NAN, INF])
def test_entropy_ignored_rows_beside_a_class_that_is_not_finite(gpu, C, bad):
    """A class of NaN spoils every row that counts; a row that does not has no gradient all the same."""
    g = _gen(52)
    x, w = _rand(g, 100, C, dtype=BF16), _rand(g, 300, C, dtype=BF16)
    w[7, 3] = bad
    t = torch.randint(0, 300, (100,), generator=g, device=gpu)
    t[::3] = -1
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    loss = cm.match_cross_entropy(x, w, t, scale=0.1, reduction="none")
    assert not loss[t < 0].any()
    dx, = torch.autograd.grad(loss.sum(), x)
    assert not dx[t < 0].any() and not torch.isfinite(dx[t >= 0]).all(-1).any()


# ---- attention: lengths and positions ----

def test_lengths_and_positions_beyond_32_bits(gpu):
    """The nearer end: all keys, or none; positions behind or in front of everything."""
    g = _gen(53)
    far = [(1 << 63) - 1, 1 << 32, (1 << 32) + 5, 1 << 31, -(1 << 32) + 9, -(1 << 63)]
    B = len(far)
    q, k, v = (_rand(g, B, n, 2, 64, dtype=BF16) for n in (12, 50, 50))
    length = torch.tensor(far, device=gpu)
    out = cm.match_attention(q, k, v, key_lengths=length)
    assert torch.equal(out[:4], cm.match_attention(q, k, v)[:4]) and not out[4:].any()
    near = torch.tensor([1 << 30 if x > 0 else -(1 << 30) for x in far], device=gpu)
    for window in ((None, 0), (1 << 30, 0), (0, 1 << 30)):
        a, b = (cm.match_attention(q, k, v, window=window, query_offset=p) for p in (length, near))
        assert torch.equal(a, b)
    assert bool(cm.match_attention(q, k, v, window=(None, 0), query_offset=length)[:4].any())


# ---- descriptors ----

def _reach(H, W, k, y, x, device):
    """[H, W]: pixels whose patch holds pixel (y, x)."""
    r = k // 2
    rows, cols = torch.arange(H, device=device)[:, None], torch.arange(W, device=device)
    return (rows >= y - (k - 1 - r)) & (rows <= y + r) & (cols >= x - (k - 1 - r)) & (cols <= x + r)


@pytest.mark.parametrize("k", [1, 2, 3, 8, 15, 16])
@pytest.mark.parametrize("bad", [NAN, INF, -INF, 1e30, 3e38, 1e7])
def test_descriptors_beside_a_pixel_far_out(gpu, k, bad):
    """A pixel that is not finite, or far larger than the rest, touches the patches that hold it and no other, bit for bit."""
    g = _gen(54)
    for H, W in ((70, 100), (300, 200)):
        img = torch.rand((H, W), generator=g, device=gpu)
        clean = cm.zncc_descriptors(img, k)
        for y, x in ((0, 0), (3, 63), (H // 2, 64), (H - 1, W - 1)):
            dirty_img = img.clone()
            dirty_img[y, x] = bad
            dirty, reach = cm.zncc_descriptors(dirty_img, k), _reach(H, W, k, y, x, gpu)
            assert torch.equal(clean[~reach], dirty[~reach]), (H, W, y, x)
            if not abs(bad) < INF:
                assert not torch.isfinite(dirty[reach][:, :k * k]).any()
            else:
                R.check(dirty, R.descriptors(dirty_img, k, F16)["d"], f"d {H}x{W} {y},{x}")


def _grads(img, k, go):
    img = img.detach().requires_grad_(True)
    return torch.autograd.grad(cm.zncc_descriptors(img, k), img, go)[0]


@pytest.mark.parametrize("k", [1, 2, 3, 8, 15, 16])
@pytest.mark.parametrize("bad", [NAN, INF, 60000.0])
@pytest.mark.parametrize("where", ["gradient", "image"])
def test_descriptors_gradient_beside_a_value_far_out(gpu, k, bad, where):
    """A descriptor's gradient reaches the pixels of its patch, a pixel those of every patch that holds it; the others'
    gradients are the same bit for bit."""
    g = _gen(55)
    for H, W in ((70, 100), (300, 200)):
        img = torch.rand((H, W), generator=g, device=gpu)
        go = _rand(g, H, W, -(-k * k // 8) * 8, scale=0.01)
        clean = _grads(img, k, go)
        for y, x in ((0, 0), (3, 63), (H // 2, 64), (H - 1, W - 1)):
            img2, go2 = img.clone(), go.clone()
            if where == "image":
                img2[y, x] = bad
                holds = _reach(H, W, k, y, x, gpu).nonzero()  # patches that hold the pixel
                (y0, x0), (y1, x1) = holds[0].tolist(), holds[-1].tolist()
            else:
                go2[y, x, k * k // 2] = bad
                (y0, x0), (y1, x1) = (y, x), (y, x)
            r = k // 2
            reach = torch.zeros((H, W), dtype=torch.bool, device=gpu)
            reach[max(0, y0 - r):y1 + k - r, max(0, x0 - r):x1 + k - r] = True
            dirty = _grads(img2, k, go2)
            assert torch.equal(clean[~reach], dirty[~reach]), (H, W, y, x)
            if abs(bad) < INF:
                R.check(dirty, R.descriptors(img2, k, F16, go2)["dI"], f"dI {H}x{W} {y},{x}")
            elif k > 1:  # one tap: nothing but zeros
                assert not torch.isfinite(dirty[reach]).any()


def _descriptors_about_the_centre(image, k, dtype, g):
    """matching_ref.descriptors with the taps taken relative to the centre pixel first, which is exact in 64 bits here: the
    mean of a flat patch of 1e18 is off by 100 in 64 bits, its norm then by ten powers of ten."""
    H, W = image.shape
    o, K = k // 2, k * k
    u = 2.0 ** -24
    img = image.double().requires_grad_(True)
    pad = torch.nn.functional.pad(img, (o, k - 1 - o, o, k - 1 - o))
    x = pad.unfold(0, k, 1).unfold(1, k, 1).reshape(H, W, K)
    x = x - x[..., o * k + o, None]
    c = x - x.mean(-1, keepdim=True)
    s = (c.square().sum(-1, keepdim=True) + 1e-8).rsqrt()
    d = c * s
    g64 = g[..., :K].double()
    dI, = torch.autograd.grad(d, img, g64)
    with torch.no_grad():
        ec = (K + 2) * u * x.abs().amax(-1, keepdim=True)
        ed = s * ec + d.abs() * ((K + 8) * u + s * ec)
        a = (g64.abs() * d.abs()).sum(-1, keepdim=True)
        rs = (K + 16) * u + (s * ec) * (1 + d.abs().sum(-1, keepdim=True))
        term = s * (g64.abs() + g64.abs().mean(-1, keepdim=True) + a * d.abs())
        err = term * (3 * rs + (K + 16 + 2 * K) * u) + s * a * s * ec
        acc = torch.zeros_like(pad)
        for t in range(K):
            acc[t // k:t // k + H, t % k:t % k + W] += err[..., t]
    pads = (0, -K % 8)
    return (tuple(torch.nn.functional.pad(z, pads) for z in R._finish(d.detach(), ed.detach(), dtype)),
            R._finish(dI, acc[o:o + H, o:o + W], image.dtype))


@pytest.mark.parametrize("k", [2, 7, 15])
@pytest.mark.parametrize("level,texture", [(200.3, 1e-3), (1000.3, 0.02), (40000.37, 0.1), (3e6, 20.0), (1e-4, 1e-6), (1e18, 1e13), (1e25, 1e24)])
def test_descriptors_of_any_range(gpu, k, level, texture):
    """Weak texture on a high level, and a flat part: the norm does not cancel, and does not leave float32's range."""
    g = _gen(56)
    img = level + texture * torch.rand((40, 130), generator=g, device=gpu)
    img[4:30, 10:50] = level
    go = _rand(g, 40, 130, -(-k * k // 8) * 8)
    d, dI = _descriptors_about_the_centre(img, k, F16, go)
    R.check(cm.zncc_descriptors(img, k), d, "d")
    R.check(_grads(img, k, go), dI, "dI")


# ---- the pair operators ----

def _image_pair(gpu, H, W, seed):
    from tests.golden.inputs import make_pair

    return [torch.from_numpy(x).to(gpu).requires_grad_(True) for x in make_pair(H, W, 20, seed=seed)]


def _nodes(fn):
    seen, todo = [], [fn]
    while todo:
        n = todo.pop()
        if n is not None and n not in seen:
            seen.append(n)
            todo += [m for m, _ in n.next_functions]
    return seen


@pytest.mark.parametrize("op", ["disparity", "loss", "loss_none"])
def test_backward_passes_of_one_graph_interleaved(gpu, op):
    """A second backward pass of the same graph, with gradients 2^30 times smaller, runs in front of every node of the
    first: both are what they are alone."""
    cam, proj = _image_pair(gpu, 20, 100, 8)
    if op == "disparity":
        out = cm.stereo_soft_disparity(cam, proj, 25, 9, layout="window")
    else:
        index = cm.stereo_disparity(cam.detach(), proj.detach(), 25, 9, layout="window")[0]
        out = cm.stereo_match_loss(cam, proj, index, 25, 9, layout="window", reduction="none" if "none" in op else "mean")
    go = torch.rand(out.shape, generator=_gen(57), device=gpu)
    want = torch.autograd.grad(out, (cam, proj), go, retain_graph=True)
    small = torch.autograd.grad(out, (cam, proj), go * 2.0 ** -30, retain_graph=True)
    busy, inner, handles = [False], [], []

    def hook(grads):
        if not busy[0]:
            busy[0] = True
            inner.append(torch.autograd.grad(out, (cam, proj), go * 2.0 ** -30, retain_graph=True))
            busy[0] = False

    for node in _nodes(out.grad_fn):
        if "AccumulateGrad" not in node.name():
            handles.append(node.register_prehook(hook))
    got = torch.autograd.grad(out, (cam, proj), go, retain_graph=True)
    for h in handles:
        h.remove()
    assert inner
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for one in inner:
        assert all(torch.equal(a, b) for a, b in zip(one, small))


def test_backward_passes_of_one_graph_from_two_threads(gpu):
    import threading

    cam, proj = _image_pair(gpu, 40, 200, 8)
    out = cm.stereo_soft_disparity(cam, proj, 25, 9, layout="window")
    gos = [torch.ones_like(out) * 2.0 ** -e for e in (0, 20, 40)]
    want = [torch.autograd.grad(out, (cam, proj), g, retain_graph=True) for g in gos]
    torch.cuda.synchronize()
    got, errors = [[] for _ in gos], []

    def work(n):
        try:
            for _ in range(20):
                got[n].append(torch.autograd.grad(out, (cam, proj), gos[n], retain_graph=True))
            torch.cuda.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(len(gos))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for mine, ref in zip(got, want):
        assert len(mine) == 20 and all(torch.equal(a, b) for one in mine for a, b in zip(one, ref))


# ---- forward-mode derivatives ----

@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(gpu, grad):
    """There are no forward-mode formulas: a dual tensor raises, also where nothing asks for a gradient."""
    import torch.autograd.forward_ad as fw

    g = _gen(58)
    q, k, v = (_rand(g, 1, 9, 2, 16).requires_grad_(grad) for _ in range(3))
    x, w, t = _rand(g, 9, 16).requires_grad_(grad), _rand(g, 20, 16).requires_grad_(grad), torch.zeros(9, device=gpu, dtype=torch.int64)
    img = torch.rand((8, 30), generator=g, device=gpu).requires_grad_(grad)
    with fw.dual_level():
        d = lambda y: fw.make_dual(y, torch.ones_like(y))  # noqa: E731
        for call in (lambda: cm.match_attention(d(q), k, v), lambda: cm.match_attention(q, d(k), v),
                     lambda: cm.match_attention(q, k, d(v)), lambda: cm.match_cross_entropy(d(x), w, t),
                     lambda: cm.match_cross_entropy(x, d(w), t), lambda: cm.zncc_descriptors(d(img), 3),
                     lambda: cm.stereo_soft_disparity(d(img), img, 5, 3), lambda: cm.stereo_soft_disparity(img, d(img), 5, 3),
                     lambda: cm.stereo_match_loss(img, d(img), torch.zeros((8, 30), device=gpu, dtype=torch.int64), 5, 3)):
            with pytest.raises(RuntimeError):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError):
                call()
        assert cm.match_attention(q, k, v).shape == q.shape  # no tangent: as always
    x0 = img.detach()
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda y: cm.zncc_descriptors(y, 3), (x0,), (x0,))


# ---- strides of 2^24 elements and more ----

@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("which", ["query positions", "query heads", "key positions", "value positions", "all"])
def test_attention_far_strides(gpu, which, train):
    """[B, heads, L, C] storage of a long sequence, positions that lie 2^24 elements apart: as contiguous copies."""
    g = _gen(59)
    big = (1 << 24) + 8

    def spread(x, dim):  # the same values with a stride of `big` along dim
        shape = list(x.shape)
        n = shape[dim]
        store = torch.empty(n * big, device=gpu, dtype=x.dtype)
        strides, s = [0] * 4, 1
        for i in (3, 2, 1, 0):
            if i != dim:
                strides[i] = s
                s *= shape[i]
        strides[dim] = big
        view = store.as_strided(shape, strides)
        view.copy_(x)
        return view

    q, k, v = _rand(g, 1, 5, 4, 64, dtype=BF16), _rand(g, 1, 6, 2, 64, dtype=BF16), _rand(g, 1, 6, 2, 64, dtype=BF16)
    go = _rand(g, 1, 5, 4, 64, dtype=BF16)
    far = [q, k, v]
    for n, (name, dim) in enumerate((("query positions", 1), ("key positions", 1), ("value positions", 1))):
        if which in (name, "all"):
            far[n] = spread(far[n], dim)
    if which == "query heads":
        far[0] = spread(q, 2)
    ref_in, far = ([x.detach().requires_grad_(train) for x in xs] for xs in ([q, k, v], far))
    ref, got = (cm.match_attention(*xs, window=(3, 0), sinks=1) for xs in (ref_in, far))
    assert torch.equal(got, ref)
    if train:
        for a, b in zip(torch.autograd.grad(got, far, go), torch.autograd.grad(ref, ref_in, go)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("C", [64, 512])
def test_entropy_far_strides(gpu, C):
    g = _gen(60)
    big = (1 << 24) + 8
    x, w = _rand(g, 4, C, dtype=BF16), _rand(g, 6, C, dtype=BF16)
    t = torch.tensor([0, 5, -1, 3], device=gpu)
    res = []
    for far in (False, True):
        xs = []
        for y in (x, w):
            z = y.clone()
            if far:
                z = torch.empty(len(y) * big, device=gpu, dtype=BF16).as_strided(y.shape, (big, 1))
                z.copy_(y)
            xs.append(z.detach().requires_grad_(True))
        loss = cm.match_cross_entropy(*xs, t, scale=0.1)
        res.append([loss.detach(), *torch.autograd.grad(loss, xs)])
    for a, b in zip(*res):
        assert torch.equal(a, b)


# ---- sizes at their ends ----

@pytest.mark.parametrize("C", [64, 512])
def test_entropy_without_classes_at_the_c_entry(gpu, C):
    import ctypes

    from custereomatching_amd import _lib, matching

    x, w = torch.ones((1, 50, C), device=gpu, dtype=F16), torch.ones((1, 0, C), device=gpu, dtype=F16)
    t = torch.zeros((1, 50), device=gpu, dtype=torch.int64)
    loss, lse, total = (torch.full(s, 7.0, device=gpu) for s in ((50,), (50,), (3,)))
    g = matching._geo(x, w, None, (1, 50, 0, 1, 1, C, 0), 1.0, (-1, -1))
    n = _lib.lib.custma_match_workspace_bytes(ctypes.byref(g), _lib.MATCH_ENTROPY)
    ws = torch.empty(n, dtype=torch.uint8, device=gpu)
    rc = _lib.lib.custma_match_entropy(ctypes.byref(g), x.data_ptr(), None, t.data_ptr(), loss.data_ptr(), lse.data_ptr(),
                                       total.data_ptr(), ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, _lib.lib.custma_last_error()
    assert not loss.any() and bool((lse == -INF).all()) and total.tolist() == [0.0, 1.0, 0.0]


def test_entropy_of_more_rows_than_a_launch_has_threads_for(gpu):
    """70 million rows (one query, repeated): 64 threads a row would be more than 2^32."""
    N, C = 70_000_003, 264
    g = _gen(61)
    x, w = _rand(g, 1, C), _rand(g, 3, C)
    t = torch.arange(N, device=gpu) % 4  # 3: no such class
    got = cm.match_cross_entropy(x.expand(N, C), w, t, scale=0.1, reduction="none")
    few = cm.match_cross_entropy(x.expand(4, C), w, t[:4], scale=0.1, reduction="none")
    assert float(few[3]) == 0.0 and bool((few[:3] > 0).all())
    for n in range(4):
        assert bool((got[n::4] == few[n]).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_gradients_near_the_largest_float32(gpu, dtype):
    """Output gradients of 2^127 and more: a power of two beyond float32's range must not turn up beside them."""
    g = _gen(62)
    q, k = _rand(g, 1, 3, 1, 64, dtype=dtype), torch.zeros((1, 4, 1, 64), device=gpu, dtype=dtype)
    v = torch.full((1, 4, 1, 8), 0.125, device=gpu, dtype=dtype)
    go = torch.zeros((1, 3, 1, 8), device=gpu)
    go[0, 0, 0, 0], go[0, 1, 0, 1], go[0, 2, 0, 2] = 1.5 * 2.0 ** 127, 2.0 ** 127, 2.0 ** 126
    xs = [x.requires_grad_(True) for x in (q, k, v)]
    out = cm.match_attention(*xs, window=(0, 0), out_dtype=F32)  # key i alone is seen by query i: P = 1, dS = 0
    dq, dk, dv = torch.autograd.grad(out, xs, go)
    assert not dq.any() and not dk.any()
    assert torch.equal(dv[0, :3], go[0].to(dtype)) and not dv[0, 3].any()


# ---- output gradients that are not finite ----

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_attention_small_gradients_beside_one_that_is_not_finite(gpu, dtype, bad):
    """float32 output gradients of 1e-9: the power of two that carries them is theirs, whatever another row holds."""
    g = _gen(63)
    # large keys and values: the queries' gradients are some 1e-3, in float16's range
    q, k, v = (_rand(g, 1, n, 1, 64, dtype=dtype, scale=s) for n, s in ((60, 1e-3), (90, 1e3), (90, 1e3)))
    go = _rand(g, 1, 60, 1, 64, dtype=F32, scale=1e-9)
    res = []
    for poison in (False, True):
        go2 = go.clone()
        if poison:
            go2[0, 7, 0, 3] = bad
        xs = [x.clone().requires_grad_(True) for x in (q, k, v)]
        res.append(torch.autograd.grad(cm.match_attention(*xs, window=(0, 5), scale=0.1, out_dtype=F32), xs, go2))
    rows, keys = torch.arange(60, device=gpu) != 7, (torch.arange(90, device=gpu) < 7) | (torch.arange(90, device=gpu) > 12)
    assert bool(res[0][0].any())
    for n, keep in ((0, rows), (1, keys), (2, keys)):
        assert torch.equal(res[0][n][:, keep], res[1][n][:, keep]), n


@pytest.mark.parametrize("C", [64, 512])
@pytest.mark.parametrize("bad", [NAN, INF])
def test_entropy_small_weights_beside_one_that_is_not_finite(gpu, C, bad):
    g = _gen(64)
    x, w = _rand(g, 90, C, scale=100.0), _rand(g, 50, C)
    t = torch.randint(0, 50, (90,), generator=g, device=gpu)
    weight = torch.rand((90,), generator=g, device=gpu) * 1e-7
    res = []
    for poison in (False, True):
        wt = weight.clone()
        if poison:
            wt[7] = bad
        xs = [y.clone().requires_grad_(True) for y in (x, w)]
        res.append(torch.autograd.grad(cm.match_cross_entropy(*xs, t, scale=50.0, reduction="none"), xs, wt))
    keep = torch.arange(90, device=gpu) != 7
    assert bool(res[0][0].any()) and torch.equal(res[0][0][keep], res[1][0][keep])


@pytest.mark.parametrize("bad", [NAN, INF])
@pytest.mark.parametrize("op", ["disparity", "loss"])
def test_pair_gradients_beside_one_that_is_not_finite(gpu, op, bad):
    """One pixel's gradient spoils what its patch and its candidates' patches hold, in its row's reach; not the image."""
    cam, proj = _image_pair(gpu, 40, 100, 8)
    if op == "disparity":
        out = cm.stereo_soft_disparity(cam, proj, 25, 5, layout="window")
    else:
        index = cm.stereo_disparity(cam.detach(), proj.detach(), 25, 5, layout="window")[0]
        out = cm.stereo_match_loss(cam, proj, index, 25, 5, layout="window", reduction="none")
    go = torch.rand(out.shape, generator=_gen(65), device=gpu) * 1e-9
    clean = torch.autograd.grad(out, (cam, proj), go, retain_graph=True)
    go[20, 30] = bad
    dirty = torch.autograd.grad(out, (cam, proj), go)
    far = (torch.arange(40, device=gpu) < 18) | (torch.arange(40, device=gpu) > 22)
    for a, b in zip(clean, dirty):
        assert bool(a.any()) and torch.equal(a[far], b[far])


@pytest.mark.parametrize("C,Cv,out_dtype", [(64, 64, None), (128, 8, F32), (256, 256, None), (128, 128, F32)])
@pytest.mark.parametrize("Lq", [20, 200])
def test_attention_rows_do_not_depend_on_their_neighbours(gpu, C, Cv, out_dtype, Lq):
    """A query's output, log-sum-exp and gradient are the same bit for bit whatever the other queries of its tile hold."""
    g = _gen(66)
    q, k, v = (_rand(g, 1, n, 1, c, dtype=BF16) for n, c in ((Lq, C), (700, C), (700, Cv)))
    go = _rand(g, 1, Lq, 1, Cv, dtype=out_dtype or BF16)
    other = q * 8.0
    keep = torch.arange(Lq, device=gpu) % 7 == 3
    other[:, keep] = q[:, keep]
    res = []
    for x in (q, other):
        x = x.detach().requires_grad_(True)
        out, lse = cm.match_attention(x, k, v, window=(None, 650), scale=C ** -0.5 * 8, out_dtype=out_dtype, return_lse=True)
        res.append([out.detach(), lse.detach(), torch.autograd.grad(out, x, go)[0]])
    for a, b in zip(*res):
        assert torch.equal(a[:, keep], b[:, keep])


@pytest.mark.parametrize("H,W,D", [(3, 0, 0), (0, 0, 0), (1, 1, 0), (2, 2, 1), (5, 70, 69)])
@pytest.mark.parametrize("layout", ["full", "window"])
def test_pair_operators_at_the_smallest_sizes(gpu, H, W, D, layout):
    if layout == "window" and W == 0:
        pytest.skip("a window needs a column")
    WO = W if layout == "full" else W - D
    cam, proj = (torch.rand((H, W), generator=_gen(67 + n), device=gpu).requires_grad_(True) for n in range(2))
    soft = cm.stereo_soft_disparity(cam, proj, D, 16, layout=layout)
    loss = cm.stereo_match_loss(cam, proj, torch.zeros((H, WO), dtype=torch.int64, device=gpu), D, 16, layout=layout)
    assert soft.shape == (H, WO) and bool(torch.isfinite(soft).all()) and bool(torch.isfinite(loss))
    for out in (soft.sum(), loss):
        for x, gx in zip((cam, proj), torch.autograd.grad(out, (cam, proj), retain_graph=True)):
            assert gx.shape == x.shape and bool(torch.isfinite(gx).all())
    if W == 1:  # one candidate: log-sum-exp less its own score, each within matching_ref's bound for scores of up to 50
        assert abs(float(loss.detach())) <= 2 * 50 * (256 + 4) * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -21 * 100 + 1e-6
