"""The matching operators in 64 bits, from their formulas, with bounds on what a right kernel may be off by.

Bounds.  u = eps / 2 of the vectors' type is the largest relative error of one rounding to it; ``tiny`` the
absolute one where fp16 is subnormal (2^-25).  Products of two 16-bit values are exact in 32 bits; a sum of n of them
is off by at most n 2^-24 sum |a b|, in any order.  So
  scores        es = |scale| (C + 4) 2^-24 sum |q k|,  P = exp(s - lse) is off by the factor E = 2 max es + 2^-20
                (the exponent's, the hardware exp2's and the sum's own roundings: a few 2^-23 each);
  P for P V     rounded once: u P + tiny (split in two parts for a 32-bit output, and for up to 32 value channels with
                gradients: u^2 P + tiny);
  out           (u + E) sum P |v| + tiny sum |v| + rounding of the result;
  D = go . out  out as above but not its last rounding, which the backward gets back to u^2;
  dS = P (go . v - D)   E |dS| + P ((Cv + 8) 2^-24 sum |go v| + sum |go| (out's error)), then rounded: u |dS| + tiny
                (in two parts for up to 32 value channels and for the cross entropy up to 256: u^2 |dS| + tiny; P of dv
                likewise);
  a 32-bit go is itself rounded: P u sum |go| (|v| + |out|), and u |go| in dv;
  dq, dk, dv    those against |k|, |q|, |go|, and the result's own rounding.
"""
import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}


def visible(Lq, Lk, window, sinks, offset, length, device):
    """[B, Lq, Lk]; offset, length: lists of ints."""
    j = torch.arange(Lk, device=device)
    out = []
    for off, n in zip(offset, length):
        p = off + torch.arange(Lq, device=device)[:, None]
        see = (j < n).expand(Lq, Lk)
        left, right = window
        if right is not None:
            see = see & (j <= p + right)
        if left is not None:
            see = see & ((j >= p - left) | (j < sinks))
        out.append(see)
    return torch.stack(out) if out else torch.zeros((0, Lq, Lk), dtype=torch.bool, device=device)


def _finish(value, bound, dtype):
    u = U[dtype]
    return value, (bound + u * (value.abs() + bound) + TINY[dtype]) * 1.001 + 1e-30


def attention(q, k, v, see, scale, out_dtype, go=None):
    """{name: (value, bound)} for out, lse and, with go, dq, dk, dv.  [B, L, heads, C] tensors, any type."""
    t = q.dtype
    u, tiny = U[t], TINY[t]
    B, Lq, Hq, C = q.shape
    Hkv = k.shape[2]
    G = Hq // Hkv
    q64, k64, v64 = (x.double().permute(0, 2, 1, 3) for x in (q, k, v))
    k64, v64 = k64.repeat_interleave(G, 1), v64.repeat_interleave(G, 1)
    kt, vt = k64.transpose(-1, -2).contiguous(), v64.transpose(-1, -2).contiguous()
    s = q64 @ kt * scale
    es = abs(scale) * (C + 4) * 2.0 ** -24 * (q64.abs() @ kt.abs())
    m = see[:, None]
    s = torch.where(m, s, float("-inf"))
    any_ = m.any(-1, keepdim=True)
    lse = torch.logsumexp(torch.where(any_, s, 0.0), -1, keepdim=True)
    P = torch.where(m, torch.exp(s - lse), 0.0)
    E = 2 * torch.where(m, es, 0.0).amax(-1, keepdim=True) + 2.0 ** -20 if P.shape[-1] else torch.zeros_like(lse)
    A, seen = P @ v64.abs(), m.double() @ v64.abs()
    out = P @ v64
    ud = u * u if v.shape[3] <= 32 else u
    up = u * u if out_dtype == torch.float32 else u if go is None else ud
    eo = (up + E) * A + tiny * seen
    back = lambda x: x.permute(0, 2, 1, 3)  # noqa: E731
    lse_ref = torch.where(any_, lse, float("-inf"))[..., 0].transpose(1, 2)
    res = {"out": _finish(back(out), back(eo), out_dtype),
           "lse": (lse_ref, (E[..., 0] + 2.0 ** -22 * lse[..., 0].abs()).transpose(1, 2) + 1e-6)}
    if go is None:
        return res
    g64 = go.double().permute(0, 2, 1, 3)
    ug = u if go.dtype == torch.float32 else 0.0
    if ug:  # kept relative to the largest value: below it fp16 becomes subnormal
        tiny_g = tiny * 2 * float(g64.abs().max()) if g64.numel() else 0.0
    else:
        tiny_g = 0.0
    eg = ug * g64.abs() + tiny_g
    dp = g64 @ vt
    D = (g64 * out).sum(-1, keepdim=True)
    dS = P * (dp - D)
    eD = (g64.abs() * (eo + u * u * out.abs())).sum(-1, keepdim=True)
    edp = (v.shape[3] + 8) * 2.0 ** -24 * (g64.abs() @ vt.abs()) + eg @ vt.abs() + (eg * out.abs()).sum(-1, keepdim=True)
    edS = E * dS.abs() + P * (edp + eD)
    top = 2 * float(g64.abs().max()) if ug and g64.numel() else 1.0  # dS is rounded after the scaling of a 32-bit go
    edS = edS + ud * (dS.abs() + edS) + torch.where(m, tiny * top, 0.0)
    dq, edq = scale * (dS @ k64), abs(scale) * (edS @ k64.abs()) + 2.0 ** -18 * abs(scale) * (dS.abs() @ k64.abs())
    T = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    dk, edk = scale * (T(dS) @ q64), abs(scale) * (T(edS) @ q64.abs()) + 2.0 ** -18 * abs(scale) * (T(dS.abs()) @ q64.abs())
    eP = (ud + E) * P + torch.where(m, tiny, 0.0)
    dv = T(P) @ g64
    edv = T(eP) @ g64.abs() + T(P) @ eg + 2.0 ** -18 * (T(P) @ g64.abs())

    def heads(x):  # sum over the group
        b, h, L, c = x.shape
        return x.reshape(b, Hkv, G, L, c).sum(2).permute(0, 2, 1, 3)

    res["dq"] = _finish(back(dq), back(edq), t)
    res["dk"] = _finish(heads(dk), heads(edk), t)
    res["dv"] = _finish(heads(dv), heads(edv), t)
    return res


def entropy(x, w, target, see, scale, weight):
    """[B, N, C], [B, V, C], [B, N], visible [1 or B, N, V]; weight [B, N] multiplies the rows' losses (32-bit).
    {name: (value, bound)} for loss (rows), dx, dw (of sum weight * loss); and who counts."""
    t = x.dtype
    u, tiny = U[t], TINY[t]
    C, V = x.shape[-1], w.shape[1]
    x64, w64 = x.double(), w.double()
    wt = w64.transpose(1, 2).contiguous()
    s = x64 @ wt * scale
    es = abs(scale) * (C + 4) * 2.0 ** -24 * (x64.abs() @ wt.abs())
    see = see.expand(s.shape)
    hot = (torch.arange(V, device=x.device) == target[..., None]) & see
    counts = hot.any(-1)
    s = torch.where(see, s, float("-inf"))
    any_ = see.any(-1, keepdim=True)
    lse = torch.logsumexp(torch.where(any_, s, 0.0), -1, keepdim=True)
    P = torch.where(see, torch.exp(s - lse), 0.0)
    E = 2 * torch.where(see, es, 0.0).amax(-1, keepdim=True) + 2.0 ** -20
    st = torch.where(hot, s, 0.0).sum(-1)
    loss = torch.where(counts, lse[..., 0] - st, 0.0)
    el = torch.where(counts, E[..., 0] + 2.0 ** -21 * (lse[..., 0].abs() + st.abs()) + 1e-6, 1e-30)
    wgt = torch.where(counts, weight.double(), 0.0)[..., None]
    top = wgt.abs().amax() if wgt.numel() else wgt.new_zeros(())
    dz = wgt * (P - hot.double())
    edz = E * (wgt * P).abs()
    ud = u * u if C <= 256 else u
    edz = edz + ud * (dz.abs() + edz) + torch.where(see & counts[..., None], tiny * 2.0 ** -14, 0.0) * top
    edz = edz + 2.0 ** -22 * dz.abs()  # the weight's own division by the largest one
    T = lambda a: a.transpose(1, 2).contiguous()  # noqa: E731
    dx, edx = scale * (dz @ w64), abs(scale) * (edz @ w64.abs() + 2.0 ** -18 * (dz.abs() @ w64.abs()))
    dw, edw = scale * (T(dz) @ x64), abs(scale) * (T(edz) @ x64.abs() + 2.0 ** -18 * (T(dz.abs()) @ x64.abs()))
    return {"loss": (loss, el), "dx": _finish(dx, edx, t), "dw": _finish(dw, edw, t), "counts": counts}


def descriptors(image, k, dtype, g=None):
    """d and, with g, the image gradient, by autograd in 64 bits, with bounds."""
    H, W = image.shape
    o, K = k // 2, k * k
    img = image.double().requires_grad_(True)
    pad = torch.nn.functional.pad(img, (o, k - 1 - o, o, k - 1 - o))
    x = pad.unfold(0, k, 1).unfold(1, k, 1).reshape(H, W, K)
    c = x - x.mean(-1, keepdim=True)
    s = (c.square().sum(-1, keepdim=True) + 1e-8).rsqrt()
    d = c * s
    # taps are taken relative to the centre pixel: |x - mid| <= R, summed in 32 bits
    R = (x - x[..., (k // 2) * k + k // 2, None]).abs().amax(-1, keepdim=True)
    ec = (K + 2) * 2.0 ** -24 * R  # the mean's error, and so each centred tap's
    ed = s * ec + d.abs() * ((K + 8) * 2.0 ** -24 + s * ec)
    pads = (0, -K % 8)
    res = {"d": tuple(torch.nn.functional.pad(z, pads) for z in _finish(d.detach(), ed.detach(), dtype))}
    if g is None:
        return res
    g64 = g[..., :K].double()
    dI, = torch.autograd.grad(d, img, g64)
    with torch.no_grad():
        # terms s g, s b, s^2 a (I - m): relative errors of s (its sum of squares), a and the sums
        a = (g64.abs() * d.abs()).sum(-1, keepdim=True)
        rs = (K + 16) * 2.0 ** -24 + (s * ec) * (1 + d.abs().sum(-1, keepdim=True))
        term = s * (g64.abs() + g64.abs().mean(-1, keepdim=True) + a * d.abs())
        err = term * (3 * rs + (K + 16) * 2.0 ** -24) + s * a * s * ec
        acc = torch.zeros_like(pad)
        for t in range(K):
            acc[t // k:t // k + H, t % k:t % k + W] += err[..., t]
        total = torch.zeros_like(pad)
        for t in range(K):
            total[t // k:t // k + H, t % k:t % k + W] += term[..., t]
        bound = acc[o:o + H, o:o + W] + 2 * K * 2.0 ** -24 * total[o:o + H, o:o + W]
    res["dI"] = _finish(dI, bound, image.dtype)
    return res


def check(got, want, name):
    value, bound = want
    top = torch.finfo(got.dtype).max
    got = got.double()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    same = got == value  # infinities
    # beyond the type's largest value (fp16: 65504) the rounding is to infinity, of the value's sign
    same = same | (torch.isinf(got) & (got.sign() == value.sign()) & (value.abs() + bound >= top))
    off = torch.where(same, 0.0, (got - value).abs())
    bad = ~(off <= bound)
    if bool(bad.any()):
        at = int(torch.where(bad, off / bound, -1.0).flatten().argmax())
        raise AssertionError(f"{name}: {int(bad.sum())} of {got.numel()} out of bound, worst at flat index {at}: got "
                             f"{float(got.flatten()[at])}, want {float(value.flatten()[at])} +- {float(bound.flatten()[at])}")
