"""Performance cases of the operators around a block of any width: what a program that trains or serves such blocks calls.

Three kinds of pass, each over a range of sizes, types and layouts:

  residual_norm  the seam between two branches: the branch's output normalised, gated, scaled and added to the residual,
                 and the sum normalised for the next branch; forward, or forward and every gradient
  int8           a 1x1 product in 8-bit integers: every token quantised by its largest channel, weights held as 8-bit integers
                 with a scale for each output channel
  clip           the norm of all gradients together, and the gradients scaled to a largest norm

`own` chooses between the plain form (torch operations in 32 bits, or 64 where a rounding decides) and the package's operators.
`listed()` holds the named cases, `draw(rng)` more of the same ranges.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5


# ------------------------------------------------------------------ cases
def _seam(name, layout, norm, B, C, H, W, dtype, post, gate, scale, train):
    """layout "first": tensors (B,C,H,W); "last": (B,H*W,C).  gate: "none", "full" (a value for each element) or "image" (one
    for each image and channel); a gate passes through a sigmoid."""
    return {"name": name, "kind": "residual_norm", "layout": layout, "norm": norm, "B": B, "C": C, "H": H, "W": W, "dtype": dtype,
            "post": post, "gate": gate, "scale": scale, "train": train}


def _int8(name, layout, B, H, W, K, N, dtype, bias):
    return {"name": name, "kind": "int8", "layout": layout, "B": B, "H": H, "W": W, "K": K, "N": N, "dtype": dtype, "bias": bias}


def _clip(name, tensors, smallest, largest, dtype, ratio):
    """`tensors` gradients of `smallest` to `largest` elements; `ratio`: the allowed norm over the norm there is."""
    return {"name": name, "kind": "clip", "tensors": tensors, "smallest": smallest, "largest": largest, "dtype": dtype,
            "ratio": ratio}


def listed():
    return [
        # The smallest call: one small tile or feature map at the seam of two branches. Latency.
        _seam("seam_small", "first", "layer", 1, 64, 24, 20, "fp32", False, "none", True, False),
        # The denoiser's block at the benchmark's batch and resolution, with a norm on either side of the seam.
        _seam("seam_dncnn", "first", "layer", 8, 64, 256, 256, "fp32", True, "none", True, False),
        # A wider super-resolution block on bf16 tensors of an odd size, gated for each image and channel.
        _seam("seam_odd_gated_bf16", "first", "layer", 2, 96, 111, 167, "bf16", True, "image", True, False),
        # The denoiser's training patches: forward and all gradients.
        _seam("seam_train_patches", "first", "layer", 8, 64, 64, 64, "fp32", True, "none", True, True),
        # Wide channels_last tokens with a gate for each element, in training.
        _seam("seam_train_tokens_bf16", "last", "rms", 4, 1024, 31, 33, "bf16", True, "full", True, True),
        # The smallest product: the 64 -> 128 layer of a block on one small feature map. Latency.
        _int8("int8_small", "first", 1, 24, 20, 64, 128, "fp32", True),
        # The same layer at the denoiser's batch and resolution: the largest in memory.
        _int8("int8_dncnn", "first", 8, 256, 256, 64, 128, "fp32", True),
        # The block's 128 -> 64 layer on a whole photograph of odd size, bf16 tensors.
        _int8("int8_photo_bf16", "first", 1, 321, 481, 128, 64, "bf16", True),
        # A wide linear layer over many tokens: the largest in operations.
        _int8("int8_tokens_wide_bf16", "last", 8, 32, 32, 4096, 4096, "bf16", False),
        # The deblurring network's gradients (102 tensors, 308 k elements): launches.
        _clip("clip_usrnet", 102, 64, 14000, "fp32", 0.5),
        # The denoiser's gradients in bf16, clipped into 32-bit master gradients (284 tensors, 0.8 M elements).
        _clip("clip_dncnn_master", 284, 64, 10000, "bf16", 0.25),
        # A large model's gradients, tensors of odd sizes.
        _clip("clip_large", 48, 60001, 6000001, "fp32", 0.5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choice(["residual_norm", "residual_norm", "int8", "int8", "clip"])
    if kind == "clip":
        small = _log_int(rng, 1, 100000)
        case = _clip("", _log_int(rng, 1, 600), small, _log_int(rng, small, 6000000), rng.choice(["fp32", "bf16"]),
                     rng.choice([0.1, 0.5, 0.9, 2.0]))
        return case if sum(_sizes(case)) <= 64000000 else None
    H = _log_int(rng, 1, 300)
    case = {"layout": rng.choice(["first", "last"]), "B": _log_int(rng, 1, 8), "H": H,
            "W": min(300, max(1, int(H * rng.uniform(0.6, 1.7)))), "dtype": rng.choice(["fp32", "bf16"])}
    tokens = case["B"] * case["H"] * case["W"]
    if kind == "int8":
        case.update(kind=kind, K=_log_int(rng, 16, 4096), N=_log_int(rng, 16, 4096), bias=rng.random() < 0.5)
        if tokens * (case["K"] + case["N"]) > 64000000 or tokens * case["K"] * case["N"] > 8192 * 4096 * 2048:
            return None
        return case
    case.update(kind=kind, C=_log_int(rng, 8, 1024 if case["layout"] == "first" else 4096),
                norm=rng.choice(["layer", "rms"]), post=rng.random() < 0.6, gate=rng.choice(["none", "full", "image"]),
                scale=rng.random() < 0.6, train=rng.random() < 0.5)
    return case if tokens * case["C"] <= (8000000 if case["train"] else 32000000) else None


def draw(rng):
    while True:
        case = _draw_once(rng)
        if case is not None:
            case.pop("name", None)
            return case


def _sizes(case):
    """Elements of each gradient: spread over the logarithm, in an order that mixes them."""
    n, lo, hi = case["tensors"], case["smallest"], case["largest"]
    at = [((37 * i) % n) / max(1, n - 1) for i in range(n)]
    return [max(1, int(lo * (hi / lo) ** u)) for u in at]


# ------------------------------------------------------------------ what a program has in hand
def _normal(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def _shape(case, C):
    B, H, W = case["B"], case["H"], case["W"]
    return (B, C, H, W) if case["layout"] == "first" else (B, H * W, C)


def _per_channel(case, v):
    return v.view(1, -1, 1, 1) if case["layout"] == "first" else v


def _channel_dim(case):
    return 1 if case["layout"] == "first" else -1


def _tokens_first(case, x):
    """(B,C,H,W) or (B,T,C) as (B,T,C)."""
    return x.flatten(2).transpose(1, 2) if case["layout"] == "first" else x


def _features(case, C, g):
    """Activations: channels of their own level and spread, some tokens far larger than others."""
    x = _normal(g, *_shape(case, C))
    x *= _per_channel(case, 0.25 + torch.rand(C, device="cuda", generator=g))
    x += _per_channel(case, 0.5 * _normal(g, C))
    size = torch.exp(_normal(g, *_shape(case, 1)))
    return (x * size).to(DTYPES[case["dtype"]])


def _prepare_seam(case, g):
    C, dtype, train = case["C"], DTYPES[case["dtype"]], case["train"]
    s = {"case": case, "x": _features(case, C, g), "branch": _features(case, C, g)}
    s["pre_weight"], s["pre_bias"] = 1 + 0.2 * _normal(g, C), 0.1 * _normal(g, C)
    if case["post"]:
        s["post_weight"], s["post_bias"] = 1 + 0.2 * _normal(g, C), 0.1 * _normal(g, C)
    if case["norm"] == "rms":
        s["pre_bias"] = s["post_bias"] = None
    if case["scale"]:
        s["scale"] = 0.3 * _normal(g, C)
    if case["gate"] == "full":
        s["gate"] = _normal(g, *_shape(case, C)).to(dtype)
    elif case["gate"] == "image":
        s["gate"] = _normal(g, *((case["B"], C, 1, 1) if case["layout"] == "first" else (case["B"], 1, C))).to(dtype)
    names = ("x", "branch", "scale", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias")
    s["names"] = [n for n in names if s.get(n) is not None]
    if train:
        for n in s["names"]:
            s[n].requires_grad_(True)
        # gradients of a mean loss
        s["dy"] = (_normal(g, *s["x"].shape) / 64).to(dtype)
        s["dz"] = (_normal(g, *s["x"].shape) / 64).to(dtype)
    return s


def _prepare_int8(case, g):
    K, N = case["K"], case["N"]
    s = {"case": case, "x": _features(case, K, g)}
    weight = _normal(g, N, K) * (0.5 + torch.rand(N, 1, device="cuda", generator=g)) / math.sqrt(K)
    s["weight_scale"] = weight.abs().amax(1) / 127
    # rows begin at multiples of 16 bytes, as programs hold such matrices
    rows = torch.zeros(N, (K + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    s["weight_q"] = rows[:, :K]
    s["weight_q"].copy_(torch.round(weight / s["weight_scale"][:, None]).clamp(-127, 127))
    s["bias"] = 0.1 * _normal(g, N) if case["bias"] else None
    return s


def _prepare_clip(case, g):
    sizes, dtype = _sizes(case), DTYPES[case["dtype"]]
    flat = _normal(g, sum(sizes))
    parts = list(flat.split(sizes))
    level = torch.exp(1.5 * _normal(g, len(sizes)) - 6).tolist()
    grads = [(p * v).to(dtype) for p, v in zip(parts, level)]
    norm = math.sqrt(sum(float(x.double().square().sum()) for x in grads))
    master = torch.empty(sum(sizes), device="cuda")
    return {"case": case, "grads": grads, "max_norm": case["ratio"] * norm, "master": master, "out": list(master.split(sizes))}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"residual_norm": _prepare_seam, "int8": _prepare_int8, "clip": _prepare_clip}[case["kind"]](case, g)


# ------------------------------------------------------------------ one pass
def _norm_plain(v, weight, bias, case):
    d = _channel_dim(case)
    if case["norm"] == "layer":
        v = v - v.mean(d, keepdim=True)
    v = v / torch.sqrt(v.square().mean(d, keepdim=True) + EPS) * _per_channel(case, weight)
    return v if bias is None else v + _per_channel(case, bias)


def _residual_norm_plain(s, case):
    dtype = DTYPES[case["dtype"]]
    t = s["branch"].float()
    if case["post"]:
        t = _norm_plain(t, s["post_weight"], s["post_bias"], case)
    if case["gate"] != "none":
        t = t / (1 + torch.exp(-s["gate"].float()))
    if case["scale"]:
        t = t * _per_channel(case, s["scale"])
    y = s["x"].float() + t
    return y.to(dtype), _norm_plain(y, s["pre_weight"], s["pre_bias"], case).to(dtype)


def _residual_norm_own(s, case):
    from conversenet_b200 import functional as CF
    return CF.residual_norm(s["x"], s["branch"], scale=s.get("scale"), gate=s.get("gate"), post_weight=s.get("post_weight"),
                            post_bias=s.get("post_bias"), pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], eps=EPS,
                            norm=case["norm"], gate_act="sigmoid" if case["gate"] != "none" else None,
                            data_format="channels_" + case["layout"])


def _run_seam(s):
    case = s["case"]
    call = _residual_norm_own if own else _residual_norm_plain
    if not case["train"]:
        with torch.no_grad():
            y, z = call(s, case)
        return {"y": y, "z": z}
    y, z = call(s, case)
    grads = torch.autograd.grad((y, z), [s[n] for n in s["names"]], (s["dy"], s["dz"]))
    return {"y": y.detach(), "z": z.detach(), **{"d" + n: v for n, v in zip(s["names"], grads)}}


def _run_int8(s):
    case = s["case"]
    if own:
        from conversenet_b200 import functional as CF
        return CF.pointwise_int8(s["x"], s["weight_q"], s["weight_scale"], s["bias"], data_format="channels_" + case["layout"])
    # which integer a value is rounded to is decided in 64 bits; the product is in 32
    x = _tokens_first(case, s["x"]).double()
    top = x.abs().amax(2, keepdim=True)
    q = torch.round(x * 127 / torch.where(top == 0, 1.0, top)).float()
    out = (q @ s["weight_q"].float().t()) * (top / 127).float() * s["weight_scale"]
    if s["bias"] is not None:
        out = out + s["bias"]
    out = out.to(DTYPES[case["dtype"]])
    return out.transpose(1, 2).reshape(_shape(case, case["N"])).contiguous() if case["layout"] == "first" else out


def _run_clip(s):
    if own:
        from conversenet_b200 import functional as CF
        _, norm = CF.clip_by_global_norm(s["grads"], s["max_norm"], out=s["out"])
        return {"master": s["master"], "norm": norm}
    norm = torch.stack(torch._foreach_norm(s["grads"], 2, dtype=torch.float32)).square().sum().sqrt()
    coefficient = (s["max_norm"] / (norm + 1e-6)).clamp(max=1)
    grads = s["grads"] if s["case"]["dtype"] == "fp32" else [g.float() for g in s["grads"]]
    torch._foreach_copy_(s["out"], torch._foreach_mul(grads, coefficient))
    return {"master": s["master"], "norm": norm}


def run(state):
    return {"residual_norm": _run_seam, "int8": _run_int8, "clip": _run_clip}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ from the definitions, in 64 bits
def _exact_normed(v, layer):
    """(normalised rows, 1 / their spread) over the last axis."""
    v = v - v.mean(-1, keepdim=True) if layer else v
    r = (v.pow(2).sum(-1, keepdim=True) / v.shape[-1] + EPS).rsqrt()
    return v * r, r


def _exact_normed_back(d, h, r, layer):
    """Gradient of _exact_normed: `d` with what lies along h (and along a constant) taken out."""
    out = d - h * (d * h).mean(-1, keepdim=True)
    return r * (out - d.mean(-1, keepdim=True) if layer else out)


def _exact_seam(case, seed):
    s = prepare(case, seed)
    rows = {n: _tokens_first(case, s[n].detach()).double() for n in ("x", "branch", "gate", "dy", "dz") if s.get(n) is not None}
    vec = {n: s[n].detach().double() for n in s["names"] if n not in rows}
    layer, first, C = case["norm"] == "layer", case["layout"] == "first", case["C"]
    one = torch.ones(C, dtype=torch.float64, device="cuda")
    a, gain = vec.get("scale", one), torch.sigmoid(rows["gate"]) if "gate" in rows else one.view(1, 1, C)
    p = rows["branch"]
    if case["post"]:
        h, r = _exact_normed(p, layer)
        p = h * vec["post_weight"] + vec.get("post_bias", 0 * one)
    y = rows["x"] + a * gain * p
    k, q = _exact_normed(y, layer)
    z = k * vec["pre_weight"] + vec.get("pre_bias", 0 * one)

    def back(v):
        return v.transpose(1, 2).reshape(_shape(case, C)) if first else v

    out = {"y": back(y), "z": back(z)}
    if not case["train"]:
        return out
    d = rows["dy"] + _exact_normed_back(rows["dz"] * vec["pre_weight"], k, q, layer)
    got = {"x": back(d), "scale": (d * gain * p).sum((0, 1)), "pre_weight": (rows["dz"] * k).sum((0, 1)),
           "pre_bias": rows["dz"].sum((0, 1))}
    if "gate" in rows:
        dg = d * a * p * gain * (1 - gain)
        if case["gate"] == "image":
            got["gate"] = dg.sum(1).view(s["gate"].shape)
        else:
            got["gate"] = back(dg)
    dp = d * a * gain
    if case["post"]:
        got["post_weight"], got["post_bias"] = (dp * h).sum((0, 1)), dp.sum((0, 1))
        dp = _exact_normed_back(dp * vec["post_weight"], h, r, layer)
    got["branch"] = back(dp)
    return {**out, **{"d" + n: got[n] for n in s["names"]}}


def _exact_int8(case, seed):
    s = prepare(case, seed)
    x = _tokens_first(case, s["x"]).double()
    top = x.abs().amax(-1, keepdim=True).clamp(min=1e-300)
    # the nearest integer, an even one where two are as near: twice the distance is compared without a division
    low = torch.floor(127 * x / top)
    above = 254 * x - (2 * low + 1) * top
    q = low + ((above > 0) | ((above == 0) & (low % 2 != 0))).double()
    out = torch.matmul(q * (top / 127), s["weight_q"].double().t() * s["weight_scale"].double())
    if s["bias"] is not None:
        out = out + s["bias"].double()
    return out.transpose(1, 2).reshape(_shape(case, case["N"])) if case["layout"] == "first" else out


def _exact_clip(case, seed):
    s = prepare(case, seed)
    every = torch.cat([g.double() for g in s["grads"]])
    norm = torch.linalg.vector_norm(every)
    return {"master": every * min(1.0, s["max_norm"] / (float(norm) + 1e-6)), "norm": norm}


def exact(case, seed):
    return {"residual_norm": _exact_seam, "int8": _exact_int8, "clip": _exact_clip}[case["kind"]](case, seed)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "clip":
        n = sum(_sizes(case))
        return {"bytes": (e + 4) * n, "flops": 3 * n}
    tokens = case["B"] * case["H"] * case["W"]
    if case["kind"] == "int8":
        K, N = case["K"], case["N"]
        return {"bytes": tokens * e * (K + N) + N * K + 4 * N * (2 if case["bias"] else 1), "flops": 2 * tokens * K * N}
    C = case["C"]
    n, vectors = tokens * C, C * (1 + case["post"]) * (2 if case["norm"] == "layer" else 1) + C * case["scale"]
    full, image = case["gate"] == "full", case["B"] * C * (case["gate"] == "image")
    if not case["train"]:
        return {"bytes": e * (n * (4 + full) + image) + 4 * vectors, "flops": 20 * n}
    # x, branch, dy, dz (and gate) in; y, z, dx, dbranch (and dgate) out
    return {"bytes": e * (n * (8 + 2 * full) + 2 * image) + 8 * vectors, "flops": 60 * n}
