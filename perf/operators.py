"""Timed cases of the matching operators: descriptors of image patches, attention along rows, and softmax cross
entropy over candidate columns.

``run`` computes a case either in its plain form (elementary torch operations in 32 bits, scores held in memory a
slice at a time) or, where ``own`` is true, through the package's public operators.  ``exact`` gives the same
outputs in 64 bits from the definitions.

Visibility, shared by attention and cross entropy: query i sits at position p = offset + i, and key j is visible to
it iff j < length, j <= p + right, and j >= p - left or j < sinks (a bound of -1 in a case: none on that side).
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_EPS = 1e-8


def listed():
    return [
        # the descriptors of one structured-light capture at the size of the example driver, with the image gradient
        {"name": "descriptors_330x422_k15", "op": "descriptors", "H": 330, "W": 422, "k": 15, "image": "fp32",
         "dtype": "fp16"},
        # the same for a 2048 x 2048 capture with 11 x 11 patches, the size of the volume benchmarks
        {"name": "descriptors_2048_k11", "op": "descriptors", "H": 2048, "W": 2048, "k": 11, "image": "fp32",
         "dtype": "fp16"},
        # one new position against caches of different fill, everything visible: generation, latency and cache bandwidth
        {"name": "attention_step_cache_32k", "op": "attention", "B": 8, "Lq": 1, "Lk": 32768, "Hq": 16, "Hkv": 4,
         "C": 128, "Cv": 128, "left": -1, "right": 0, "sinks": 0, "ragged": True, "dtype": "bf16", "train": False,
         "fp32_out": False, "value_grad": False},
        # one new position of one sequence, a window and sinks in a long cache: the smallest call
        {"name": "attention_step_window", "op": "attention", "B": 1, "Lq": 1, "Lk": 100001, "Hq": 16, "Hkv": 4,
         "C": 128, "Cv": 128, "left": 1023, "right": 0, "sinks": 4, "ragged": True, "dtype": "bf16", "train": False,
         "fp32_out": False, "value_grad": False},
        # a prompt read in one call, queries, keys and values as slices of one projection
        {"name": "attention_prompt_8k", "op": "attention", "B": 1, "Lq": 8192, "Lk": 8192, "Hq": 16, "Hkv": 4,
         "C": 128, "Cv": 128, "left": 1023, "right": 0, "sinks": 4, "ragged": False, "dtype": "bf16", "train": False,
         "fp32_out": False, "value_grad": False},
        # a training step on sequences of different lengths in one padded batch, odd sizes
        {"name": "attention_train_ragged", "op": "attention", "B": 5, "Lq": 2047, "Lk": 2047, "Hq": 8, "Hkv": 2,
         "C": 64, "Cv": 64, "left": 511, "right": 0, "sinks": 3, "ragged": True, "dtype": "bf16", "train": True,
         "fp32_out": False, "value_grad": True},
        # differentiable soft disparity: 11 x 11 descriptors of a 2048 x 2048 pair, columns w .. w + 256 as candidates,
        # the column's coordinate as value
        {"name": "attention_rows_2048_window", "op": "attention", "B": 2048, "Lq": 1792, "Lk": 2048, "Hq": 1,
         "Hkv": 1, "C": 128, "Cv": 8, "left": 0, "right": 256, "sinks": 0, "ragged": False, "dtype": "fp16",
         "train": True, "fp32_out": True, "value_grad": False},
        # warping 32 learned channels along whole rows by 9 x 9 descriptors, all projector columns, a 1024 x 1024 pair
        {"name": "attention_rows_1024_full", "op": "attention", "B": 1024, "Lq": 1024, "Lk": 1024, "Hq": 1, "Hkv": 1,
         "C": 88, "Cv": 32, "left": -1, "right": -1, "sinks": 0, "ragged": False, "dtype": "fp16", "train": True,
         "fp32_out": False, "value_grad": True},
        # matching loss of the example driver's capture: 15 x 15 descriptors, 200 disparities
        {"name": "entropy_rows_330x422", "op": "entropy", "B": 330, "N": 222, "V": 422, "C": 232, "shared": False,
         "left": 0, "right": 200, "dtype": "fp16", "train": True, "ignored": 0.1},
        # matching loss of a 2048 x 2048 pair, 11 x 11 descriptors, 256 disparities
        {"name": "entropy_rows_2048", "op": "entropy", "B": 2048, "N": 1792, "V": 2048, "C": 128, "shared": False,
         "left": 0, "right": 256, "dtype": "fp16", "train": True, "ignored": 0.1},
        # training over one large shared vocabulary, wide vectors, odd counts
        {"name": "entropy_vocabulary_train", "op": "entropy", "B": 1, "N": 4093, "V": 50021, "C": 1024,
         "shared": True, "left": -1, "right": -1, "dtype": "bf16", "train": True, "ignored": 0.05},
        # the loss alone of a short held-out text over a larger vocabulary
        {"name": "entropy_vocabulary_loss", "op": "entropy", "B": 1, "N": 333, "V": 128000, "C": 512,
         "shared": True, "left": -1, "right": -1, "dtype": "bf16", "train": False, "ignored": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["descriptors", "attention", "attention", "attention", "entropy", "entropy"])
    if op == "descriptors":
        return {"op": op, "H": _log(rng, 1, 2048), "W": _log(rng, 16, 2048), "k": rng.randint(3, 15),
                "image": rng.choice(["fp32", "fp16"]), "dtype": rng.choice(["fp16", "bf16"])}
    dtype = rng.choice(["fp16", "bf16"])
    if op == "attention":
        kind = rng.choice(["step", "sequence", "rows"])
        if kind == "rows":
            W = _log(rng, 64, 2048)
            full = rng.random() < 0.4
            D = W // rng.randint(3, 12)
            return {"op": op, "B": _log(rng, 16, 1024), "Lq": W if full else W - D, "Lk": W, "Hq": 1, "Hkv": 1,
                    "C": rng.choice([16, 32, 49, 56, 88, 128, 176, 232]), "Cv": rng.choice([2, 8, 16, 32]),
                    "left": -1 if full else 0, "right": -1 if full else D, "sinks": 0 if full else rng.randint(0, 2),
                    "ragged": False, "dtype": dtype, "train": rng.random() < 0.7, "fp32_out": rng.random() < 0.5,
                    "value_grad": rng.random() < 0.5}
        C = rng.choice([32, 64, 80, 96, 128, 192, 256])
        kv = rng.randint(1, 4)
        windowed = rng.random() < 0.6
        if kind == "step":
            L = _log(rng, 1, 60000)
            return {"op": op, "B": _log(rng, 1, 16), "Lq": rng.choice([1, 1, 1, 2, 5]), "Lk": max(L, 5),
                    "Hq": kv * rng.choice([1, 2, 4, 5, 8]), "Hkv": kv, "C": C, "Cv": C,
                    "left": _log(rng, 1, 4096) if windowed else -1, "right": 0,
                    "sinks": rng.randint(0, 8) if windowed else 0, "ragged": True, "dtype": dtype, "train": False,
                    "fp32_out": rng.random() < 0.2, "value_grad": False}
        L = _log(rng, 1, 4096)
        return {"op": op, "B": rng.randint(1, 4), "Lq": L, "Lk": L, "Hq": kv * rng.choice([1, 2, 3, 4]), "Hkv": kv,
                "C": C, "Cv": C, "left": _log(rng, 1, 2048) if windowed else -1, "right": 0,
                "sinks": rng.randint(0, 8) if windowed else 0, "ragged": rng.random() < 0.5, "dtype": dtype,
                "train": rng.random() < 0.6, "fp32_out": False, "value_grad": True}
    if rng.random() < 0.5:
        W = _log(rng, 64, 2048)
        full = rng.random() < 0.4
        D = W // rng.randint(3, 12)
        return {"op": op, "B": _log(rng, 16, 1024), "N": W if full else W - D, "V": W,
                "C": rng.choice([16, 32, 49, 56, 88, 128, 176, 232]), "shared": False, "left": -1 if full else 0,
                "right": -1 if full else D, "dtype": dtype, "train": rng.random() < 0.7, "ignored": 0.1}
    return {"op": op, "B": 1, "N": _log(rng, 1, 4096), "V": _log(rng, 1000, 50000),
            "C": rng.choice([64, 100, 128, 256, 384, 512, 768, 1000, 1024]), "shared": True, "left": -1, "right": -1,
            "dtype": dtype, "train": rng.random() < 0.6, "ignored": 0.05}


def _bound(v):
    return None if v < 0 else v


def _lengths(case, seed):
    """(offsets, lengths) of each batch entry, host integers: a cache or a padded batch filled to different lengths."""
    rng = np.random.default_rng(seed)
    B, Lq, Lk = case["B"], case["Lq"], case["Lk"]
    if not case["ragged"]:
        return np.zeros(B, np.int64), np.full(B, Lk, np.int64)
    low = max(Lq if Lq < Lk else 1, Lk // 2)
    lengths = rng.integers(low, Lk + 1, size=B)
    lengths[0] = Lk
    offsets = lengths - Lq if Lq < Lk else np.zeros(B, np.int64)
    return offsets, lengths


def _rand(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _unit(x):
    return x / x.norm(dim=-1, keepdim=True)


def _rows(gen, B, N, V, C, left, right, dtype):
    """Unit vectors of a row of candidates and of queries that are noisy copies of a candidate in reach, and that
    candidate's index. Neighbouring candidates resemble each other as overlapping patches do (cosine 10/11), and a
    query's cosine with its own candidate is about a half, so a softmax at beta = 50 spreads over a few columns."""
    i = torch.arange(N, device="cuda")
    lo = torch.zeros_like(i) if left is None else (i - left).clamp(min=0)
    hi = torch.full_like(i, V - 1) if right is None else (i + right).clamp(max=V - 1)
    u = torch.rand((B, N), generator=gen, device="cuda")
    target = torch.minimum(lo + (u * (hi - lo + 1)).long(), hi)
    keys = torch.empty((B, V, C), device="cuda", dtype=dtype)
    query = torch.empty((B, N, C), device="cuda", dtype=dtype)
    for b in range(0, B, 256):
        n = min(256, B - b)
        r = _rand(gen, n, V + 10, C)
        near = r[:, :V].clone()
        for t in range(1, 11):
            near += r[:, t:t + V]
        near = _unit(near)
        keys[b:b + n] = near.to(dtype)
        near = torch.take_along_dim(near, target[b:b + n, :, None], 1)
        query[b:b + n] = _unit(near + (3.0 / C) ** 0.5 * _rand(gen, n, N, C)).to(dtype)
    return query, keys, target


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "descriptors":
        H, W, k = case["H"], case["W"], case["k"]
        # a speckle pattern under slowly varying light, in [0, 1], with a patch-sized flat spot
        speckle = torch.rand((H, W), generator=gen, device="cuda")
        light = 0.6 + 0.4 * torch.sin(torch.arange(W, device="cuda") * 0.01 + torch.arange(H, device="cuda")[:, None] * 0.02)
        image = (speckle * light).clamp(0, 1)
        if H > 4 * k and W > 4 * k:
            image[k:3 * k, k:3 * k] = 0.5
        s["image"] = image.to(_DTYPES[case["image"]])
        C8 = -(-k * k // 8) * 8
        s["grad"] = _rand(gen, H, W, C8).to(_DTYPES[case["dtype"]])
    elif case["op"] == "attention":
        B, Lq, Lk, Hq, Hkv, C, Cv = (case[n] for n in ("B", "Lq", "Lk", "Hq", "Hkv", "C", "Cv"))
        dtype = _DTYPES[case["dtype"]]
        s["out_dtype"] = torch.float32 if case["fp32_out"] else dtype
        if Hq == 1 and Hkv == 1:
            q, k, _ = _rows(gen, B, Lq, Lk, C, _bound(case["left"]), _bound(case["right"]), dtype)
            s["query"], s["key"] = q.unsqueeze(2), k.unsqueeze(2)
            if Cv < 16:  # coordinates of the column, in units that 16 bits hold exactly
                j = torch.arange(Lk, device="cuda")
                v = torch.stack([(j >> (c % 2 * 5)) & 31 for c in range(Cv)], -1).float()
                v = v.expand(B, Lk, Cv)
            else:
                v = _rand(gen, B, Lk, Cv)
            s["value"] = v.to(dtype).reshape(B, Lk, 1, Cv)
            s["scale"] = 50.0
        else:
            if Lq == Lk and C == Cv:  # slices of one projection
                fused = _rand(gen, B, Lq, (Hq + 2 * Hkv) * C).to(dtype)
                q, k, v = fused.split([Hq * C, Hkv * C, Hkv * C], -1)
            else:
                q, k, v = (_rand(gen, B, n, h).to(dtype) for n, h in ((Lq, Hq * C), (Lk, Hkv * C), (Lk, Hkv * Cv)))
            s["query"], s["key"] = q.unflatten(-1, (Hq, C)), k.unflatten(-1, (Hkv, C))
            s["value"] = v.unflatten(-1, (Hkv, Cv))
            s["scale"] = C ** -0.5
        offsets, lengths = _lengths(case, seed)
        if case["ragged"]:
            s["offsets"] = torch.from_numpy(offsets).to("cuda", torch.int32)
            s["lengths"] = torch.from_numpy(lengths).to("cuda", torch.int32)
        else:
            s["offsets"] = s["lengths"] = None
        if case["train"]:
            s["grad"] = _rand(gen, B, Lq, Hq, Cv).to(s["out_dtype"])
    else:
        B, N, V, C = (case[n] for n in ("B", "N", "V", "C"))
        dtype = _DTYPES[case["dtype"]]
        if case["shared"]:
            s["query"] = _rand(gen, N, C).to(dtype)
            s["classes"] = (_rand(gen, V, C) * C ** -0.5).to(dtype)
            s["target"] = torch.randint(0, V, (N,), generator=gen, device="cuda")
            # a mean in bf16; fp16 gradients of a mean over thousands of rows would be subnormal
            s["scale"], s["reduction"] = 1.0, "mean" if dtype == torch.bfloat16 else "sum"
        else:
            s["query"], s["classes"], s["target"] = _rows(gen, B, N, V, C, _bound(case["left"]),
                                                          _bound(case["right"]), dtype)
            s["scale"], s["reduction"] = 50.0, "sum"  # a sum: gradients of a mean over pixels leave fp16's range
        drop = torch.rand(s["target"].shape, generator=gen, device="cuda") < case["ignored"]
        s["target"] = torch.where(drop, -1, s["target"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        leaves = {"descriptors": ("image",), "entropy": ("query", "classes"),
                  "attention": ("query", "key", "value") if case.get("value_grad") else ("query", "key")}[case["op"]]
        s["leaves"] = []
        if case.get("train", True):
            for n in leaves:
                s[n] = s[n].detach().requires_grad_(True)
                s["leaves"].append(s[n])
    return s


# ---- the framework's operators ----

def _run_own(s):
    import custereomatching_amd as cm

    case = s["case"]
    if case["op"] == "descriptors":
        d = cm.zncc_descriptors(s["image"], case["k"], dtype=_DTYPES[case["dtype"]])
        return [d.detach(), *torch.autograd.grad(d, s["leaves"], s["grad"])]
    window = (_bound(case["left"]), _bound(case["right"]))
    if case["op"] == "attention":
        out = cm.match_attention(s["query"], s["key"], s["value"], window=window, sinks=case["sinks"],
                                 scale=s["scale"], query_offset=s["offsets"], key_lengths=s["lengths"],
                                 out_dtype=s["out_dtype"])
        if not case["train"]:
            return [out]
        return [out.detach(), *torch.autograd.grad(out, s["leaves"], s["grad"])]
    loss = cm.match_cross_entropy(s["query"], s["classes"], s["target"], scale=s["scale"], window=window,
                                  reduction=s["reduction"])
    if not case["train"]:
        return [loss]
    return [loss.detach(), *torch.autograd.grad(loss, s["leaves"])]


# ---- the plain forms ----

def _plain_descriptors(s):
    case = s["case"]
    k, I = case["k"], s["image"].float()
    H, W = I.shape
    o, K = k // 2, k * k
    pad = torch.zeros((H + k - 1, W + k - 1), device=I.device)
    pad[o:o + H, o:o + W] = I
    x = torch.stack([pad[i:i + H, j:j + W] for i in range(k) for j in range(k)], -1)
    x = x - x.sum(-1, keepdim=True) / K
    n = torch.sqrt((x * x).sum(-1, keepdim=True) + _EPS)
    x = x / n
    g = s["grad"][..., :K].float()
    a = (g * x).sum(-1, keepdim=True)
    dx = (g - g.sum(-1, keepdim=True) / K - a * x) / n
    dpad = torch.zeros_like(pad)
    for t in range(K):
        dpad[t // k:t // k + H, t % k:t % k + W] += dx[..., t]
    d = torch.zeros((H, W, -(-K // 8) * 8), device=I.device)
    d[..., :K] = x
    return [d.to(s["grad"].dtype), dpad[o:o + H, o:o + W].to(s["image"].dtype)]


def _visible(Lq, Lk, left, right, sinks, offsets, lengths, device):
    """[B or 1, Lq, Lk] truth values."""
    j = torch.arange(Lk, device=device)
    p = torch.arange(Lq, device=device)[None, :, None]
    if offsets is not None:
        p = p + offsets.long()[:, None, None]
    see = torch.ones((1, 1, Lk), dtype=torch.bool, device=device)
    if lengths is not None:
        see = see & (j < lengths.long()[:, None, None])
    if right >= 0:
        see = see & (j <= p + right)
    if left >= 0:
        see = see & ((j >= p - left) | (j < sinks))
    return see.expand(see.shape[0], Lq, Lk)


def _plain_attention(s):
    case = s["case"]
    B, Lq, Lk, Hq, Hkv, C, Cv = (case[n] for n in ("B", "Lq", "Lk", "Hq", "Hkv", "C", "Cv"))
    G, scale, train = Hq // Hkv, s["scale"], case["train"]
    dtype, dev = s["query"].dtype, s["query"].device
    out = torch.empty((B, Lq, Hq, Cv), device=dev, dtype=s["out_dtype"])
    dq = torch.empty((B, Lq, Hq, C), device=dev, dtype=dtype) if train else None
    dk = torch.empty((B, Lk, Hkv, C), device=dev, dtype=dtype) if train else None
    dv = torch.empty((B, Lk, Hkv, Cv), device=dev, dtype=dtype) if train and case["value_grad"] else None
    step = max(1, min(B, int(1.5e9 // (Hq * Lq * Lk))))

    def heads(x, h, g):  # [b, L, h*g, c] -> [b, h, g*L, c]
        b, L, _, c = x.shape
        return x.float().reshape(b, L, h, g, c).permute(0, 2, 3, 1, 4).reshape(b, h, g * L, c)

    def back(x, L, g):  # [b, h, g*L, c] -> [b, L, h*g, c]
        b, h, _, c = x.shape
        return x.reshape(b, h, g, L, c).permute(0, 3, 1, 2, 4).reshape(b, L, h * g, c)

    for b in range(0, B, step):
        e = min(B, b + step)
        see = _visible(Lq, Lk, case["left"], case["right"], case["sinks"],
                       None if s["offsets"] is None else s["offsets"][b:e],
                       None if s["lengths"] is None else s["lengths"][b:e], dev)
        see = see[:, None, None].expand(see.shape[0], 1, G, Lq, Lk).reshape(see.shape[0], 1, G * Lq, Lk)
        q, k, v = heads(s["query"][b:e], Hkv, G), heads(s["key"][b:e], Hkv, 1), heads(s["value"][b:e], Hkv, 1)
        z = torch.matmul(q, k.transpose(-1, -2)) * scale
        z = torch.where(see, z, float("-inf"))
        m = z.amax(-1, keepdim=True)
        m = torch.where(m > float("-inf"), m, 0.0)
        P = torch.exp(z - m)
        total = P.sum(-1, keepdim=True)
        P = P / torch.where(total > 0, total, 1.0)
        o = torch.matmul(P, v)
        out[b:e] = back(o, Lq, G).to(out.dtype)
        if train:
            do = heads(s["grad"][b:e], Hkv, G)
            dp = torch.matmul(do, v.transpose(-1, -2))
            ds = P * (dp - (P * dp).sum(-1, keepdim=True)) * scale
            dq[b:e] = back(torch.matmul(ds, k), Lq, G).to(dtype)
            dk[b:e] = back(torch.matmul(ds.transpose(-1, -2).contiguous(), q), Lk, 1).to(dtype)
            if dv is not None:
                dv[b:e] = back(torch.matmul(P.transpose(-1, -2).contiguous(), do), Lk, 1).to(dtype)
    return [t for t in (out, dq, dk, dv) if t is not None]


def _plain_entropy(s):
    case = s["case"]
    B, N, V = case["B"], case["N"], case["V"]
    X, Wt, T = s["query"].reshape(B, N, -1), s["classes"].reshape(B, V, -1), s["target"].reshape(B, N)
    scale, train, dev = s["scale"], case["train"], X.device
    see = _visible(N, V, case["left"], case["right"], 0, None, None, dev)
    step = max(1, min(B, int(1.0e9 // (N * V))))
    valid = (T >= 0) & (T < V)
    safe = torch.where(valid, T, 0)
    valid = valid & see[0][torch.arange(N, device=dev)[None], safe]
    count = valid.sum()
    weight = valid.float() if s["reduction"] == "sum" else valid.float() / count.clamp(min=1)
    total = torch.zeros((), device=dev, dtype=torch.float64)
    dx = torch.empty_like(X) if train else None
    dw = torch.empty_like(Wt) if train else None
    for b in range(0, B, step):
        e = min(B, b + step)
        x, w = X[b:e].float(), Wt[b:e].float()
        z = torch.matmul(x, w.transpose(-1, -2)) * scale
        z = torch.where(see, z, float("-inf"))
        m = z.amax(-1, keepdim=True)
        P = torch.exp(z - m)
        sums = P.sum(-1, keepdim=True)
        picked = torch.take_along_dim(z, safe[b:e, :, None], 2)
        row = (torch.log(sums) + m - picked)[..., 0]
        total += torch.where(valid[b:e], row, 0.0).double().mul(weight[b:e]).sum()
        if train:
            hot = torch.arange(V, device=dev) == safe[b:e, :, None]
            dz = (P / sums - hot.float()) * (weight[b:e, :, None] * scale)
            dx[b:e] = torch.matmul(dz, w).to(X.dtype)
            dw[b:e] = torch.matmul(dz.transpose(-1, -2).contiguous(), x).to(X.dtype)
    loss = total.float()
    if not train:
        return [loss]
    return [loss, dx.reshape(s["query"].shape), dw.reshape(s["classes"].shape)]


_PLAIN = {"descriptors": _plain_descriptors, "attention": _plain_attention, "entropy": _plain_entropy}


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- the definitions in 64 bits, differentiated by autograd ----

def _exact_descriptors(s):
    case = s["case"]
    k, H, W = case["k"], case["H"], case["W"]
    o = k // 2
    image = s["image"].double().requires_grad_(True)
    padded = torch.nn.functional.pad(image, (o, k - 1 - o, o, k - 1 - o))
    d = padded.unfold(0, k, 1).unfold(1, k, 1).reshape(H, W, k * k)
    d = d - d.mean(-1, keepdim=True)
    d = d * (d.square().sum(-1, keepdim=True) + _EPS).rsqrt()
    g, = torch.autograd.grad(d, image, s["grad"][..., :k * k].double())
    return [torch.nn.functional.pad(d.detach(), (0, -(k * k) % 8)), g]


def _exact_attention(s):
    case = s["case"]
    G, parts = case["Hq"] // case["Hkv"], []
    step = max(1, min(case["B"], int(4e8 // (case["Hq"] * case["Lq"] * case["Lk"]))))
    for b in range(0, case["B"], step):
        part = slice(b, b + step)
        q, k, v = (s[n][part].double().requires_grad_(case["train"]) for n in ("query", "key", "value"))
        see = _visible(case["Lq"], case["Lk"], case["left"], case["right"], case["sinks"],
                       None if s["offsets"] is None else s["offsets"][part],
                       None if s["lengths"] is None else s["lengths"][part], q.device)
        outs = []
        for h in range(case["Hq"]):
            kh, vh = k[:, :, h // G], v[:, :, h // G]
            z = (q[:, :, h] @ kh.transpose(1, 2).contiguous()) * s["scale"]
            z = z.masked_fill(~see, float("-inf"))
            none = ~see.any(-1, keepdim=True)
            P = torch.softmax(z.masked_fill(none, 0.0), -1).masked_fill(none, 0.0)
            outs.append(P @ vh)
        out = torch.stack(outs, 2)
        grads = []
        if case["train"]:
            leaves = (q, k, v) if case["value_grad"] else (q, k)
            grads = torch.autograd.grad(out, leaves, s["grad"][part].double())
        parts.append([out.detach(), *grads])
        del out, outs, z, P
    return [torch.cat(t) for t in zip(*parts)]


def _exact_entropy(s):
    case = s["case"]
    B, N, V = case["B"], case["N"], case["V"]
    see = _visible(N, V, case["left"], case["right"], 0, None, None, "cuda")
    X, Wt, T = s["query"].reshape(B, N, -1), s["classes"].reshape(B, V, -1), s["target"].reshape(B, N)
    counted = ((T >= 0) & (T < V)).sum()
    loss, dx, dw = torch.zeros((), dtype=torch.float64, device="cuda"), [], []
    step = max(1, min(B, int(4e8 // (N * V))))
    for b in range(0, B, step):
        x = X[b:b + step].double().requires_grad_(case["train"])
        w = Wt[b:b + step].double().requires_grad_(case["train"])
        t = T[b:b + step]
        z = ((x @ w.transpose(1, 2).contiguous()) * s["scale"]).masked_fill(~see, float("-inf"))
        row = torch.logsumexp(z, -1) - z.gather(2, t.clamp(min=0)[..., None])[..., 0]
        part = row[t >= 0].sum()
        if s["reduction"] == "mean":
            part = part / counted.clamp(min=1)
        loss = loss + part.detach()
        if case["train"]:
            gx, gw = torch.autograd.grad(part, (x, w))
            dx.append(gx)
            dw.append(gw)
        del z, row, part
    if not case["train"]:
        return [loss]
    return [loss, torch.cat(dx).reshape(s["query"].shape), torch.cat(dw).reshape(s["classes"].shape)]


def exact(case, seed):
    pairs = {"descriptors": lambda c: c["H"] * c["W"] * c["k"] ** 2,
             "attention": lambda c: c["B"] * c["Hq"] * c["Lq"] * c["Lk"] * (c["C"] + c["Cv"]) * (3 if c["train"] else 1),
             "entropy": lambda c: c["B"] * c["N"] * c["V"] * c["C"] * (3 if c["train"] else 1)}[case["op"]](case)
    if pairs > 2e13:  # beyond about 20 seconds
        return None
    s = _inputs(case, seed)
    return {"descriptors": _exact_descriptors, "attention": _exact_attention, "entropy": _exact_entropy}[case["op"]](s)


def _visible_pairs(Lq, Lk, left, right, sinks, offsets, lengths):
    total = 0
    for off, n in zip(offsets, lengths):
        p = off + np.arange(Lq, dtype=np.int64)
        hi = np.minimum(n, p + right + 1) if right >= 0 else np.full(Lq, n, np.int64)
        hi = np.maximum(hi, 0)
        lo = np.clip(p - left, 0, hi) if left >= 0 else np.zeros(Lq, np.int64)
        first = np.minimum(np.minimum(sinks, lo), hi) if left >= 0 else 0
        total += int((hi - lo).sum() + np.sum(first))
    return total


def work(case):
    size = {"fp32": 4, "fp16": 2, "bf16": 2}
    if case["op"] == "descriptors":
        pixels, K = case["H"] * case["W"], case["k"] ** 2
        image, row = size[case["image"]], -(-K // 8) * 8 * size[case["dtype"]]
        return {"bytes": pixels * (2 * image + 2 * row), "flops": pixels * K * 10}
    if case["op"] == "attention":
        B, Lq, Lk, Hq, Hkv, C, Cv = (case[n] for n in ("B", "Lq", "Lk", "Hq", "Hkv", "C", "Cv"))
        offsets, lengths = _lengths(case, 0)
        if case["ragged"]:
            pairs = _visible_pairs(Lq, Lk, case["left"], case["right"], case["sinks"], offsets, lengths)
        else:
            pairs = B * _visible_pairs(Lq, Lk, case["left"], case["right"], case["sinks"], offsets[:1], lengths[:1])
        # keys that any query of an entry can see are the ones that have to be read
        keys = 0
        for off, n in zip(offsets, lengths):
            hi = min(n, off + Lq + case["right"]) if case["right"] >= 0 else n
            lo = max(0, off - case["left"]) if case["left"] >= 0 else 0
            keys += max(0, hi - lo) + min(case["sinks"], lo, max(hi, 0))
        q, o = B * Lq * Hq * C * 2, B * Lq * Hq * Cv * (4 if case["fp32_out"] else 2)
        read = int(keys) * Hkv * (C + Cv) * 2
        flops = 2 * pairs * Hq * (C + Cv)
        total = q + o + read
        if case["train"]:
            flops += 2 * pairs * Hq * (2 * C + (2 if case["value_grad"] else 1) * Cv)
            total += o + q + B * Lk * Hkv * (C + (Cv if case["value_grad"] else 0)) * 2
        return {"bytes": total, "flops": flops}
    B, N, V, C = (case[n] for n in ("B", "N", "V", "C"))
    pairs = B * _visible_pairs(N, V, case["left"], case["right"], 0, [0], [V])
    rows = B * (N + V) * C * 2
    return {"bytes": rows * (2 if case["train"] else 1) + B * N * 8 + 4, "flops": 2 * pairs * C * (3 if case["train"] else 1)}
