"""functional.residual_norm against its formula in 64 bits, forward and gradients, and what it refuses.

Tolerances.  An output value is the end of a chain of at most 24 fp32 roundings (2^-24 each) of values that are not above four
times the largest of its token (the data's channels have means and spreads of the same order): 96 . 2^-24 of the token's largest
output; a bf16 output is rounded once more, 2^-8 of itself.  A norm's gradient is r (v - mean(v) - h mean(v h)), which may cancel
(with one channel altogether): what is rounded there is r v and products of it with |h| <= sqrt(C) that average out, so the
tolerance is 96 . 2^-24 of the token's largest r v, carried on to the branch and the gate by their factors.  A parameter's gradient is a sum over tokens: its terms carry those
96 . 2^-24, fewer than 64 additions in a row add 64 . 2^-24 of the sum of magnitudes."""
import ctypes

import pytest
import torch

from conversenet_b200 import functional as CF

NAMES = ("x", "branch", "scale", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias")
EPS = 1e-5


def _case(layout, C, B, H, W, dtype, norm, post, gate, scale, pre=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    first = layout == "first"
    shape = (B, C, H, W) if first else (B, H * W, C)

    def per_channel(v):
        return v.view(1, C, 1, 1) if first else v

    def features():
        x = torch.randn(shape, device="cuda", generator=g) * per_channel(0.5 + torch.rand(C, device="cuda", generator=g))
        return (x + per_channel(0.5 * torch.randn(C, device="cuda", generator=g))).to(dtype)

    t = {"x": features(), "branch": features()}
    if scale:
        t["scale"] = 0.5 + torch.rand(C, device="cuda", generator=g)
    if gate == "full":
        t["gate"] = torch.randn(shape, device="cuda", generator=g).to(dtype)
    if gate == "image":
        t["gate"] = torch.randn((B, C, 1, 1) if first else (B, 1, C), device="cuda", generator=g).to(dtype)
    for name in (["post"] if post else []) + (["pre"] if pre else []):
        t[name + "_weight"] = 0.5 + torch.rand(C, device="cuda", generator=g)
        if norm == "layer":
            t[name + "_bias"] = 0.5 * torch.randn(C, device="cuda", generator=g)
    t["dy"] = torch.randn(shape, device="cuda", generator=g).to(dtype)
    t["dz"] = torch.randn(shape, device="cuda", generator=g).to(dtype)
    return t


def _formula(t, layout, norm, act):
    """(y, z or None) from tensors of any type."""
    first = layout == "first"
    d = 1 if first else -1

    def ch(v):
        return v.reshape(1, -1, 1, 1) if first else v.reshape(-1)

    def n(v, name):
        if norm == "layer":
            v = v - v.mean(d, keepdim=True)
        v = v / torch.sqrt((v * v).mean(d, keepdim=True) + EPS) * ch(t[name + "_weight"])
        return v + ch(t[name + "_bias"]) if name + "_bias" in t else v

    p = n(t["branch"], "post") if "post_weight" in t else t["branch"]
    if "gate" in t:
        p = p * (torch.sigmoid(t["gate"]) if act else t["gate"])
    if "scale" in t:
        p = p * ch(t["scale"])
    y = t["x"] + p
    return y, n(y, "pre") if "pre_weight" in t else None


def _call(t, layout, norm, act):
    return CF.residual_norm(t["x"], t["branch"], t.get("scale"), t.get("gate"), t.get("post_weight"), t.get("post_bias"),
                            t.get("pre_weight"), t.get("pre_bias"), EPS, norm, "sigmoid" if act else None, "channels_" + layout)


def _before_cancelling(t, layout, norm, act):
    """For each token the largest of the values that the gradients of x, branch and a gate of each element are formed from."""
    d = 1 if layout == "first" else -1
    t = {n: v.detach() for n, v in t.items()}

    def ch(v):
        return v.reshape(1, -1, 1, 1) if layout == "first" else v.reshape(-1)

    def r(v):
        v = v - v.mean(d, keepdim=True) if norm == "layer" else v
        return 1 / torch.sqrt((v * v).mean(d, keepdim=True) + EPS)

    y, _ = _formula(t, layout, norm, act)
    x = (t["dy"].abs() + r(y) * (t["dz"] * ch(t["pre_weight"])).abs()).amax(d, keepdim=True)
    a = ch(t["scale"]).abs() if "scale" in t else torch.ones_like(y)
    s = (torch.sigmoid(t["gate"]) if act else t["gate"]) if "gate" in t else torch.ones_like(y)
    w = ch(t["post_weight"]).abs() if "post_weight" in t else torch.ones_like(y)
    branch = x * (a * s.abs() * w).amax(d, keepdim=True) * (r(t["branch"]) if "post_weight" in t else 1)
    p = (y - t["x"]) / s if "gate" in t else y
    return {"x": x, "branch": branch, "gate": x * p.abs().amax(d, keepdim=True)}


def _close(got, ref, channel_dim, what, top=None):
    ref = ref.detach()
    top = ref.abs().amax(channel_dim, keepdim=True) if top is None else top
    tol = 96 * 2.0 ** -24 * top + (2.0 ** -8 * ref.abs() if got.dtype == torch.bfloat16 else 0)
    over = (got.detach().double() - ref).abs() - tol
    assert float(over.max()) <= 0, (what, float(over.max()), float(top.max()))


CASES = [
    # layout, C, B, H, W, dtype, norm, post, gate, scale
    ("first", 64, 2, 24, 20, "fp32", "layer", True, "none", True),
    ("first", 64, 1, 128, 96, "fp32", "layer", True, "none", True),         # four pixels a thread, vectors
    ("first", 64, 1, 111, 167, "bf16", "rms", True, "full", True),          # odd rows
    ("first", 64, 1, 111, 167, "fp32", "layer", True, "full", False),
    ("first", 96, 2, 75, 87, "bf16", "layer", True, "image", True),
    ("first", 96, 1, 128, 128, "bf16", "layer", False, "full", True),
    ("first", 200, 2, 13, 17, "fp32", "rms", True, "image", False),
    ("first", 128, 1, 111, 97, "bf16", "layer", True, "none", True),
    ("first", 120, 1, 100, 100, "fp32", "layer", True, "full", True),
    ("first", 200, 1, 111, 97, "bf16", "layer", True, "image", True),       # sixteen channels a thread
    ("first", 256, 1, 100, 98, "fp32", "rms", True, "full", True),
    ("first", 300, 2, 9, 11, "bf16", "layer", True, "full", True),          # wide: values are read again
    ("first", 1030, 1, 5, 7, "fp32", "layer", True, "image", True),
    ("first", 1, 2, 5, 7, "fp32", "rms", True, "none", True),
    ("first", 7, 3, 1, 1, "fp32", "layer", True, "none", True),             # one pixel an image
    ("first", 9, 70, 3, 1, "fp32", "layer", False, "image", False),         # more images than rows of threads
    ("last", 64, 2, 24, 20, "fp32", "layer", True, "none", True),
    ("last", 3, 2, 5, 7, "bf16", "rms", True, "full", True),
    ("last", 257, 3, 31, 3, "fp32", "layer", True, "image", True),
    ("last", 1024, 2, 31, 3, "bf16", "rms", True, "full", True),
    ("last", 2500, 1, 7, 5, "fp32", "layer", True, "full", True),
    ("last", 4100, 1, 3, 5, "bf16", "layer", True, "none", True),
    ("last", 16384, 1, 3, 1, "fp32", "rms", True, "image", True),
    ("last", 40, 1, 1, 1, "fp32", "layer", False, "none", False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_against_the_formula(case):
    layout, C, B, H, W, dtype, norm, post, gate, scale = case
    dtype = {"fp32": torch.float32, "bf16": torch.bfloat16}[dtype]
    act = gate != "none"
    t = _case(layout, C, B, H, W, dtype, norm, post, gate, scale)
    names = [n for n in NAMES if n in t]
    for n in names:
        t[n].requires_grad_(True)
    d = {n: t[n].detach().double().requires_grad_(n in names) for n in t}
    y64, z64 = _formula(d, layout, norm, act)
    ref = dict(zip(names, torch.autograd.grad((y64, z64), [d[n] for n in names], (d["dy"], d["dz"]), retain_graph=True)))
    with torch.no_grad():
        y0, z0 = _call(t, layout, norm, act)
    y, z = _call(t, layout, norm, act)
    assert torch.equal(y, y0) and torch.equal(z, z0) and y.dtype == dtype
    dim = 1 if layout == "first" else -1
    _close(y, y64, dim, "y")
    _close(z, z64, dim, "z")
    got = dict(zip(names, torch.autograd.grad((y, z), [t[n] for n in names], (t["dy"], t["dz"]), retain_graph=True)))
    again = torch.autograd.grad((y, z), [t[n] for n in names], (t["dy"], t["dz"]))
    tops = _before_cancelling(d, layout, norm, act)
    # the sums of magnitudes behind each parameter's gradient: the gradient with respect to it at every token, on its own
    for n, a in zip(names, again):
        assert torch.equal(got[n], a), n                   # the same bits at every call
        assert got[n].dtype == t[n].dtype and got[n].shape == t[n].shape
        if n in ("x", "branch") or (n == "gate" and gate == "full"):
            _close(got[n], ref[n], dim, n, tops[n])
            continue
        shape = y.shape
        if n == "gate":
            wide = d[n].detach().expand(shape).clone().requires_grad_(True)
        else:
            v = d[n].detach()
            wide = (v.reshape(1, -1, 1, 1) if layout == "first" else v).expand(shape).clone().requires_grad_(True)
        e = {k: (wide if k == n else v.detach()) for k, v in d.items()}
        yw, zw = _wide_formula(e, n, layout, norm, act)
        terms = torch.autograd.grad((yw * e["dy"]).sum() + (zw * e["dz"]).sum(), wide)[0].abs()
        if n == "gate":
            total = terms.sum((2, 3) if layout == "first" else 1).reshape(ref[n].shape)
        else:
            total = terms.sum((0, 2, 3) if layout == "first" else (0, 1))
        tol = 160 * 2.0 ** -24 * total + (2.0 ** -8 * ref[n].abs() if got[n].dtype == torch.bfloat16 else 0)
        # (what a token's gradient loses is measured by its largest, which the terms of other channels may have)
        tol = tol + 96 * 2.0 ** -24 * total.max()
        over = (got[n].double() - ref[n]).abs() - tol
        assert float(over.max()) <= 0, (n, float(over.max()))


def _wide_formula(t, name, layout, norm, act):
    """The formula with parameter `name` given for every element."""
    first = layout == "first"
    d = 1 if first else -1

    def ch(v, n):
        return v if n == name else v.reshape(1, -1, 1, 1) if first else v.reshape(-1)

    def n(v, part):
        if norm == "layer":
            v = v - v.mean(d, keepdim=True)
        v = v / torch.sqrt((v * v).mean(d, keepdim=True) + EPS) * ch(t[part + "_weight"], part + "_weight")
        return v + ch(t[part + "_bias"], part + "_bias") if part + "_bias" in t else v

    p = n(t["branch"], "post") if "post_weight" in t else t["branch"]
    if "gate" in t:
        p = p * (torch.sigmoid(t["gate"]) if act else t["gate"])
    if "scale" in t:
        p = p * ch(t["scale"], "scale")
    y = t["x"] + p
    return y, n(y, "pre")


@pytest.mark.gpu
@pytest.mark.parametrize("layout,gate", [("first", "full"), ("first", "image"), ("last", "full"), ("last", "none")])
def test_gradients_against_differences(layout, gate):
    """Central differences of the kernel's own forward.  L is linear in y and z; along a direction of step h the error is of the order
    of h^2 (h = 2^-6, values of order 1: below 1e-3 of the derivative's scale) plus 2^-24 sqrt(n) |L terms| / h."""
    t = _case(layout, 24, 2, 6, 5, torch.float32, "layer", True, gate, True, seed=3)
    names = [n for n in NAMES if n in t]
    for n in names:
        t[n].requires_grad_(True)

    def loss(tt):
        y, z = _call(tt, layout, "layer", gate != "none")
        return (y.double() * t["dy"].double() + z.double() * t["dz"].double()).sum()

    got = dict(zip(names, torch.autograd.grad(loss(t), [t[n] for n in names])))
    g = torch.Generator(device="cuda").manual_seed(11)
    h = 2.0 ** -6
    for n in names:
        v = torch.randn(t[n].shape, device="cuda", generator=g)
        v = v / v.norm()
        with torch.no_grad():
            a = loss({**t, n: t[n] + h * v})
            b = loss({**t, n: t[n] - h * v})
        want = float((got[n].double() * v.double()).sum())
        scale = float(got[n].double().norm()) + 1e-3
        assert abs(float(a - b) / (2 * h) - want) <= 5e-3 * scale, n


@pytest.mark.gpu
def test_parts():
    """Each tensor absent, one gradient alone, strides, empty batches."""
    t = _case("first", 20, 2, 6, 7, torch.float32, "layer", False, "none", False, pre=False)
    y = _call(t, "first", "layer", False)
    assert torch.equal(y, t["x"] + t["branch"])
    t = _case("first", 20, 2, 6, 7, torch.float32, "layer", True, "full", True)
    y, z = _call(t, "first", "layer", True)
    # strided tensors and an odd start in memory
    wide = torch.zeros(2, 41, 6, 7, device="cuda")
    wide[:, 1::2] = t["x"]
    s = dict(t, x=wide[:, 1::2], branch=t["branch"].to(memory_format=torch.channels_last))
    for a, b in zip(_call(s, "first", "layer", True), (y, z)):
        assert torch.equal(a, b)
    base = torch.empty(t["x"].numel() + 1, device="cuda")
    base[1:] = t["x"].flatten()
    for a, b in zip(_call(dict(t, x=base[1:].view_as(t["x"])), "first", "layer", True), (y, z)):
        assert torch.equal(a, b)
    # channels_last tensors that begin at odd places: the scalar kernels
    for dtype in (torch.float32, torch.bfloat16):
        u = _case("last", 64, 2, 6, 7, dtype, "layer", True, "full", True)
        base = torch.empty(u["x"].numel() + 1, device="cuda", dtype=dtype)
        base[1:] = u["x"].flatten()
        for a, b in zip(_call(dict(u, x=base[1:].view_as(u["x"])), "last", "layer", True), _call(u, "last", "layer", True)):
            assert float((a.double() - b.double()).abs().max()) <= (2.0 ** -6 if dtype == torch.bfloat16 else 1e-5)
    # z alone, y alone, one leaf alone
    for n in ("x", "gate", "post_bias", "scale", "pre_weight"):
        leaf = t[n].clone().requires_grad_(True)
        y, z = _call(dict(t, **{n: leaf}), "first", "layer", True)
        d = {k: v.double() for k, v in t.items()}
        dl = d[n].clone().requires_grad_(True)
        y64, z64 = _formula(dict(d, **{n: dl}), "first", "layer", True)
        for out, ref, go in ((z, z64, "dz"), (y, y64, "dy")):
            if n == "pre_weight" and go == "dy":
                continue
            a, = torch.autograd.grad(out, leaf, t[go], retain_graph=True)
            b, = torch.autograd.grad(ref, dl, d[go], retain_graph=True)
            assert float((a.double() - b).norm() / b.norm()) <= 1e-5, (n, go)
    e = _case("first", 20, 2, 6, 7, torch.float32, "layer", True, "image", True)
    e = {n: (v[:0] if n in ("x", "branch", "gate", "dy", "dz") else v).requires_grad_(True) for n, v in e.items()}
    y, z = _call(e, "first", "layer", True)
    assert y.shape == z.shape == (0, 20, 6, 7)
    g = torch.autograd.grad((y, z), [e["x"], e["scale"], e["pre_weight"]], (torch.zeros_like(y), torch.zeros_like(z)))
    assert g[0].shape == (0, 20, 6, 7) and not g[1].any() and not g[2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("C", [24, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_tensors_that_begin_anywhere(C, dtype):
    """Rows of an odd length in tensors that begin between 16-byte boundaries, also at the very first byte of their memory."""
    for offset in (0, 1, 3):
        t = _case("first", C, 2, 37, 11, dtype, "layer", True, "full", True, seed=offset)
        for n in ("x", "branch", "gate", "dy", "dz"):
            base = torch.zeros(t[n].numel() + offset, device="cuda", dtype=dtype)
            base[offset:] = t[n].flatten()
            t[n + "_moved"] = base[offset:].view_as(t[n])
        plain = {n: t[n].clone().requires_grad_(True) for n in NAMES if n in t}
        moved = {n: t.get(n + "_moved", t[n]).detach().requires_grad_(True) for n in NAMES if n in t}
        a = torch.autograd.grad(_call(plain, "first", "layer", True), list(plain.values()), (t["dy"], t["dz"]))
        b = torch.autograd.grad(_call(moved, "first", "layer", True), list(moved.values()), (t["dy_moved"], t["dz_moved"]))
        for n, p, q in zip(plain, a, b):
            assert torch.equal(p, q), (n, offset)


@pytest.mark.gpu
def test_values_that_are_no_numbers_stay_in_their_tokens():
    t = _case("first", 64, 1, 128, 80, torch.float32, "layer", True, "full", True)
    y0, z0 = _call(t, "first", "layer", True)
    for bad in (float("inf"), float("nan")):
        x = t["x"].clone()
        x[0, 5, 3, 7] = bad
        y, z = _call(dict(t, x=x), "first", "layer", True)
        keep = torch.ones(128, 80, dtype=torch.bool, device="cuda")
        keep[3, 7] = False
        assert torch.equal(y[..., keep], y0[..., keep]) and torch.equal(z[..., keep], z0[..., keep])
        assert bool(torch.isnan(z[0, :, 3, 7]).all()) and not bool(torch.isfinite(y[0, 5, 3, 7]))


@pytest.mark.gpu
def test_streams_graphs_and_saved_tensors():
    t = _case("first", 96, 2, 40, 31, torch.bfloat16, "layer", True, "image", True)
    y0, z0 = _call(t, "first", "layer", True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y1, z1 = _call(t, "first", "layer", True)
    side.synchronize()
    assert torch.equal(y0, y1) and torch.equal(z0, z1)
    static = dict(t, x=t["x"].clone())
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        ya, za = _call(static, "first", "layer", True)
    with torch.cuda.graph(g2):
        yb, zb = _call(static, "first", "layer", True)
    static["x"].copy_(2 * t["x"])
    g2.replay()
    g1.replay()
    torch.cuda.synchronize()
    y2, z2 = _call(dict(t, x=2 * t["x"]), "first", "layer", True)
    for a, b in ((ya, y2), (za, z2), (yb, y2), (zb, z2)):
        assert torch.equal(a, b)
    # a change in place between forward and backward is noticed; what the backward reads is released by it
    x = t["x"].clone().requires_grad_(True)
    branch = t["branch"].clone()
    y, z = _call(dict(t, x=x, branch=branch), "first", "layer", True)
    branch.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad((y, z), x, (t["dy"], t["dz"]))
    y, z = _call(dict(t, x=x), "first", "layer", True)
    torch.autograd.grad((y, z), x, (t["dy"], t["dz"]))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad((y, z), x, (t["dy"], t["dz"]))
    # one differentiation
    y, z = _call(dict(t, x=x), "first", "layer", True)
    g, = torch.autograd.grad((y, z), x, (t["dy"], t["dz"]), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated once"):
        g.sum().backward()


@pytest.mark.gpu
def test_many_images_the_widest_and_other_ranks():
    t = _case("first", 8, 70000, 2, 1, torch.float32, "layer", True, "image", True)          # more images than a grid's second axis
    names = [n for n in NAMES if n in t]
    for n in names:
        t[n].requires_grad_(True)
    y, z = _call(t, "first", "layer", True)
    d = {n: v.detach().double().requires_grad_(n in names) for n, v in t.items()}
    y64, z64 = _formula(d, "first", "layer", True)
    _close(y, y64, 1, "y")
    _close(z, z64, 1, "z")
    got = torch.autograd.grad((y, z), [t["gate"], t["scale"], t["pre_weight"]], (t["dy"], t["dz"]))
    ref = torch.autograd.grad((y64, z64), [d["gate"], d["scale"], d["pre_weight"]], (d["dy"], d["dz"]))
    for a, b in zip(got, ref):
        assert float((a.double() - b).norm() / b.norm()) <= 1e-5
    t = _case("first", 16384, 1, 3, 5, torch.bfloat16, "rms", True, "full", True)
    y, z = _call(t, "first", "rms", True)
    y64, z64 = _formula({n: v.double() for n, v in t.items()}, "first", "rms", True)
    _close(y, y64, 1, "y")
    _close(z, z64, 1, "z")
    # (T,C), and tokens of three dimensions with a gate for each image
    t = _case("last", 48, 3, 4, 6, torch.float32, "layer", True, "image", True)
    y, z = _call(t, "last", "layer", True)
    u = dict(t, x=t["x"].view(3, 4, 6, 48), branch=t["branch"].view(3, 4, 6, 48), gate=t["gate"].view(3, 1, 1, 48))
    for a, b in zip(_call(u, "last", "layer", True), (y, z)):
        assert torch.equal(a.view_as(b), b)
    flat = {n: v for n, v in t.items() if n != "gate"}
    y, z = _call(flat, "last", "layer", False)
    u = dict(flat, x=t["x"].reshape(-1, 48), branch=t["branch"].reshape(-1, 48))
    for a, b in zip(_call(u, "last", "layer", False), (y, z)):
        assert torch.equal(a.view_as(b), b)


@pytest.mark.gpu
def test_a_captured_step():
    """Forward and gradients captured into a graph and replayed on other inputs."""
    t = _case("first", 64, 2, 30, 31, torch.float32, "layer", True, "image", True)
    names = [n for n in NAMES if n in t]
    static = {n: v.clone() for n, v in t.items()}
    for n in names:
        static[n].requires_grad_(True)

    def step():
        y, z = _call(static, "first", "layer", True)
        return (y, z) + torch.autograd.grad((y, z), [static[n] for n in names], (static["dy"], static["dz"]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    other = _case("first", 64, 2, 30, 31, torch.float32, "layer", True, "image", True, seed=9)
    with torch.no_grad():
        for n, v in other.items():
            static[n].copy_(v)
    graph.replay()
    torch.cuda.synchronize()
    captured = [c.detach().clone() for c in captured]
    for a, b in zip(captured, step()):
        assert torch.equal(a, b.detach())


@pytest.mark.gpu
def test_saved_tensor_hooks_checkpointing_and_threads():
    """What the backward reads passes through saved-tensor hooks; a checkpoint runs the forward again; calls from several threads on
    streams of their own."""
    import threading
    from torch.utils.checkpoint import checkpoint
    t = _case("first", 40, 2, 24, 28, torch.float32, "layer", True, "full", True)
    names = [n for n in NAMES if n in t]
    leaves = [t[n].requires_grad_(True) for n in names]
    ref = torch.autograd.grad(_call(t, "first", "layer", True), leaves, (t["dy"], t["dz"]))
    moved = []

    def pack(v):
        moved.append(v.shape)
        return v.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda v: v.cuda()):
        out = _call(t, "first", "layer", True)
    for a, b in zip(torch.autograd.grad(out, leaves, (t["dy"], t["dz"])), ref):
        assert torch.equal(a, b)
    assert len(moved) == len(names) + 1                        # the tensors, and the means and spreads
    out = checkpoint(lambda x, b: _call(dict(t, x=x, branch=b), "first", "layer", True), t["x"], t["branch"], use_reentrant=False)
    for a, b in zip(torch.autograd.grad(out, leaves, (t["dy"], t["dz"])), ref):
        assert torch.equal(a, b)
    wrong = []

    def work(k):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(stream):
            for _ in range(20):
                with torch.no_grad():
                    mine = {n: v.detach().clone() for n, v in t.items()}
                ls = [mine[n].requires_grad_(True) for n in names]
                got = torch.autograd.grad(_call(mine, "first", "layer", True), ls, (mine["dy"], mine["dz"]))
                stream.synchronize()
                wrong.extend(n for n, a, b in zip(names, got, ref) if not torch.equal(a, b))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """2^31 elements and more in a tensor: the last tokens against the formula."""
    HW = (1 << 27) + 64
    x = torch.zeros(1, 16, 1, HW, dtype=torch.bfloat16, device="cuda")
    branch = torch.zeros_like(x)
    t = _case("first", 16, 1, 1, 512, torch.bfloat16, "layer", True, "none", True)
    x[..., -512:], branch[..., -512:] = t["x"], t["branch"]
    big = dict(t, x=x, branch=branch)
    y, z = _call(big, "first", "layer", False)
    y0, z0 = _call(t, "first", "layer", False)
    d = {n: v.double() for n, v in t.items()}
    for a, b, r in zip((y, z), (y0, z0), _formula(d, "first", "layer", False)):
        _close(a[..., -512:], r, 1, "end")
        _close(b, r, 1, "alone")
    assert bool(torch.isfinite(z[..., :512]).all())


@pytest.mark.gpu
def test_refusals():
    t = _case("first", 8, 1, 4, 4, torch.float32, "layer", True, "none", True)
    x, b, w = t["x"], t["branch"], t["pre_weight"]
    bad = [
        (RuntimeError, dict(x=x[0])),                                                # rank
        (RuntimeError, dict(branch=b[:, :4])),                                       # shape
        (RuntimeError, dict(branch=b.bfloat16())),                                   # type
        (RuntimeError, dict(x=x.half(), branch=b.half())),
        (RuntimeError, dict(scale=w[:4])),
        (RuntimeError, dict(pre_weight=None, pre_bias=w)),                           # a bias without its weight
        (RuntimeError, dict(gate=torch.ones(1, 8, 4, 1, device="cuda"))),
        (RuntimeError, dict(gate=torch.ones(1, 8, 4, 4, device="cuda", dtype=torch.bfloat16))),
        (RuntimeError, dict(scale=torch.ones(8, dtype=torch.int32, device="cuda"))),
        (RuntimeError, dict(scale=torch.ones(8))),                                   # on the CPU
        (RuntimeError, dict(eps=-1.0)),
        (RuntimeError, dict(eps=float("nan"))),
        (ValueError, dict(norm="batch")),
        (ValueError, dict(gate_act="relu")),
        (ValueError, dict(data_format="NCHW")),
        (RuntimeError, dict(x=torch.zeros(2, 20000, device="cuda"), branch=torch.zeros(2, 20000, device="cuda"),
                            pre_weight=None, data_format="channels_last")),
    ]
    for err, change in bad:
        args = dict(x=x, branch=b, pre_weight=w)
        args.update(change)
        with pytest.raises(err):
            CF.residual_norm(**args)
    wide = torch.zeros(1, 5000, 2, 2, device="cuda", requires_grad=True)
    y = CF.residual_norm(wide, wide, post_weight=torch.ones(5000, device="cuda"))
    with pytest.raises(RuntimeError, match="fixed maximum"):
        torch.autograd.grad(y.sum(), wide)


def test_refusals_without_a_device():
    x = torch.zeros(1, 4, 2, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        CF.residual_norm(x, x)
    with pytest.raises(ValueError):
        CF.residual_norm(x, x, norm="group")


def test_c_abi_refusals():
    from conversenet_b200 import _cabi

    class Args(ctypes.Structure):
        _fields_ = ([(n, ctypes.c_void_p) for n in ("x", "branch", "gate", "y", "z", "scale", "post_w", "post_b", "pre_w", "pre_b",
                                                    "stats", "dy", "dz", "dx", "dbranch", "dgate", "dscale", "dpost_w", "dpost_b",
                                                    "dpre_w", "dpre_b")] +
                    [("B", ctypes.c_longlong), ("HW", ctypes.c_longlong)] +
                    [(n, ctypes.c_int) for n in ("C", "channels_last", "rms", "gate_kind", "gate_act", "io_dtype")] +
                    [("eps", ctypes.c_float), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
                     ("stream", ctypes.c_void_p)])

    lib = _cabi.load()
    one = 16                                   # never dereferenced: validation fails first

    def fwd(**change):
        a = Args(x=one, branch=one, y=one, B=1, HW=4, C=8, eps=1e-5)
        for k, v in change.items():
            setattr(a, k, v)
        return lib.cvb_residual_norm_fwd(ctypes.byref(a))

    def bwd(**change):
        a = Args(x=one, branch=one, dy=one, dx=one, B=1, HW=4, C=8, eps=1e-5)
        for k, v in change.items():
            setattr(a, k, v)
        return lib.cvb_residual_norm_bwd(ctypes.byref(a))

    assert lib.cvb_residual_norm_fwd(None) == lib.cvb_residual_norm_bwd(None) == -1
    for change in (dict(x=None), dict(branch=None), dict(y=None), dict(B=0), dict(HW=0), dict(C=0), dict(io_dtype=5),
                   dict(gate_kind=3), dict(gate_kind=1), dict(gate=one), dict(post_b=one), dict(pre_b=one), dict(pre_w=one),
                   dict(eps=-1.0), dict(eps=float("nan"))):
        assert fwd(**change) == -1, change
    assert fwd(C=16385) == -7
    for change in (dict(dy=None), dict(dx=None), dict(dz=one), dict(post_w=one), dict(branch=None, dbranch=one), dict(dz=one, pre_w=one)):
        assert bwd(**change) == -1, change
    assert bwd(dscale=one, dx=None) == -4                      # sums without a workspace
    assert bwd(C=5000) == -7
    assert lib.cvb_residual_norm_workspace_bytes(64, 8, 0) >= 16 * 64
    assert lib.cvb_residual_norm_workspace_bytes(0, 8, 0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("gate_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(3, 40, 1, 1), (3, 1, 40), (5, 40), (2, 1, 1, 40)], ids=str)
def test_a_gate_for_each_image_of_one_pixel(shape, dtype, gate_dtype):
    """Its shape is that of x; its type is its own, as at every other size."""
    first = shape[1] == 40 and len(shape) == 4
    layout, C = "first" if first else "last", 40
    g = torch.Generator(device="cuda").manual_seed(2)
    t = {n: torch.randn(shape, device="cuda", generator=g).to(dtype) for n in ("x", "branch", "dy", "dz")}
    t["gate"] = torch.randn(shape, device="cuda", generator=g).to(gate_dtype)
    for n in ("scale", "post_weight", "post_bias", "pre_weight", "pre_bias"):
        t[n] = 0.5 + torch.rand(C, device="cuda", generator=g)
    d = {n: v.double() for n, v in t.items()}
    for n in NAMES:
        t[n].requires_grad_(True)
        d[n].requires_grad_(True)
    out = _call(t, layout, "layer", True)
    ref = _formula(d, layout, "layer", True)
    dim = 1 if first else -1
    for a, b in zip(out, ref):
        _close(a, b, dim, "outputs")
    got = torch.autograd.grad(out, [t[n] for n in NAMES], (t["dy"], t["dz"]))
    want = torch.autograd.grad(ref, [d[n] for n in NAMES], (d["dy"], d["dz"]))
    tops = _before_cancelling(d, layout, "layer", True)
    with torch.no_grad():
        # A vector's gradient is a sum of at most five terms, each off by 96 . 2^-24 of the largest value it is formed from (dz; or the
        # gradient of y, at most the branch's scale and gate times the token's top) times what is normalised (|h| <= sqrt(C)) or p.
        top = tops["x"].max() * (d["scale"].max() * 1.0)
        p = ((d["post_weight"].max() * C ** 0.5) + d["post_bias"].max())
        sizes = {"pre_bias": d["dz"].abs().max(), "pre_weight": d["dz"].abs().max() * C ** 0.5, "post_bias": top,
                 "post_weight": top * C ** 0.5, "scale": tops["x"].max() * p}
    for n, a, b in zip(NAMES, got, want):
        assert a.dtype == t[n].dtype and a.shape == t[n].shape
        if n in tops:
            over = (a.double() - b).abs() - 96 * 2.0 ** -24 * tops[n] - (torch.finfo(a.dtype).eps / 2 + 2.0 ** -24) * b.abs() - \
                (2.0 ** -25 if a.dtype == torch.float16 else 0)                # (half of fp16's smallest number)
        else:
            over = (a.double() - b).abs() - 160 * 2.0 ** -24 * 5 * sizes[n]
        assert float(over.max()) <= 0, (n, float(over.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("C,HW", [(24, 96), (24, 9600), (80, 9600), (120, 9600), (24, 9599)])
def test_c_abi_stats_that_begin_anywhere(C, HW, dtype):
    """Means and spreads kept at any float of a caller's buffer, read by the gradients there, and nothing written beside them."""
    from conversenet_b200 import _cabi
    lib = _cabi.load()
    t = _case("first", C, 1, HW, 1, dtype, "layer", True, "none", True)
    vec = dict(scale="scale", post_w="post_weight", post_b="post_bias", pre_w="pre_weight", pre_b="pre_bias")
    got = []
    for offset in (0, 1, 2, 3):
        room = torch.full((4 * HW + 8,), 7.0, device="cuda")
        o = {n: torch.empty_like(t["x"]) for n in ("y", "z", "dx", "dbranch")}
        a = _arguments(x=t["x"], branch=t["branch"], dy=t["dy"], dz=t["dz"], **{k: t[n] for k, n in vec.items()}, **o)
        a.B, a.HW, a.C, a.eps, a.io_dtype = 1, HW, C, EPS, int(dtype == torch.bfloat16)
        a.stats, a.stream = room[4 + offset:].data_ptr(), torch.cuda.current_stream().cuda_stream
        assert lib.cvb_residual_norm_fwd(ctypes.byref(a)) == 0
        assert lib.cvb_residual_norm_bwd(ctypes.byref(a)) == 0
        assert bool((room[:4 + offset] == 7).all()) and bool((room[4 + offset + 4 * HW:] == 7).all())
        got.append([room[4 + offset:4 + offset + 4 * HW].clone(), *o.values()])
    for other in got[1:]:
        for a, b in zip(got[0], other):
            # other pixels a thread, the same channels and order of sums: fp32 roundings at most, and a neighbour in the tensors' type
            a, b = a.double(), b.double()
            eps = torch.finfo(dtype).eps
            assert bool(((a - b).abs() <= eps * a.abs() + 1e-5 * a.abs().max()).all())


def _arguments(**tensors):
    class Args(ctypes.Structure):
        _fields_ = ([(n, ctypes.c_void_p) for n in ("x", "branch", "gate", "y", "z", "scale", "post_w", "post_b", "pre_w", "pre_b",
                                                    "stats", "dy", "dz", "dx", "dbranch", "dgate", "dscale", "dpost_w", "dpost_b",
                                                    "dpre_w", "dpre_b")] +
                    [("B", ctypes.c_longlong), ("HW", ctypes.c_longlong)] +
                    [(n, ctypes.c_int) for n in ("C", "channels_last", "rms", "gate_kind", "gate_act", "io_dtype")] +
                    [("eps", ctypes.c_float), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
                     ("stream", ctypes.c_void_p)])

    return Args(**{n: v.data_ptr() for n, v in tensors.items()})


def test_c_abi_addresses():
    from conversenet_b200 import _cabi

    lib = _cabi.load()
    one = 16                                   # never dereferenced: validation fails first

    def fwd(**change):
        a = _arguments()
        for k, v in dict(dict(x=one, branch=one, y=one, B=1, HW=4, C=8, eps=1e-5), **change).items():
            setattr(a, k, v)
        return lib.cvb_residual_norm_fwd(ctypes.byref(a))

    def bwd(**change):
        a = _arguments()
        for k, v in dict(dict(x=one, branch=one, dy=one, dx=one, B=1, HW=4, C=8, eps=1e-5), **change).items():
            setattr(a, k, v)
        return lib.cvb_residual_norm_bwd(ctypes.byref(a))

    # addresses between elements
    for name in ("x", "branch", "y"):
        assert fwd(**{name: 18}) == -1 and fwd(**{name: 17, "io_dtype": 1}) == -1, name
    for name in ("scale", "stats", "post_w"):
        assert fwd(**{name: 18}) == -1, name
    assert fwd(gate=18, gate_kind=1) == -1 and fwd(gate=18, gate_kind=2, io_dtype=1) == -1
    assert fwd(post_w=one, post_b=18) == -1 and fwd(pre_w=18, z=one) == -1 and fwd(pre_w=one, z=18) == -1
    for name in ("dy", "dx", "dbranch"):
        assert bwd(**{name: 18}) == -1, name
    assert bwd(dscale=18, workspace=one, workspace_bytes=1 << 30) == -1
    assert bwd(dscale=one, workspace=18, workspace_bytes=1 << 30) == -4
    assert bwd(gate=one, gate_kind=1, dgate=18) == -1 and bwd(gate=one, gate_kind=2, dgate=18, io_dtype=1) == -1


@pytest.mark.gpu
def test_forward_mode_is_refused():
    """There is no tangent of the outputs: a call that would lose one says so."""
    import torch.autograd.forward_ad as fwd
    t = {n: v for n, v in _case("first", 8, 1, 4, 4, torch.float32, "layer", True, "full", True).items() if n in NAMES}
    y0, z0 = _call(t, "first", "layer", True)
    for leaf in (False, True):
        with fwd.dual_level():
            for n in t:
                v = t[n].clone().requires_grad_(leaf)
                with pytest.raises(RuntimeError, match="forward-mode"):
                    _call(dict(t, **{n: fwd.make_dual(v, torch.ones_like(v))}), "first", "layer", True)
            y, z = _call(t, "first", "layer", True)
            assert torch.equal(y, y0) and torch.equal(z, z0)


@pytest.mark.gpu
@pytest.mark.parametrize("layout,C", [("first", 8), ("first", 300), ("last", 8), ("last", 7)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["full", "image"])
def test_the_sigmoid_and_its_slope(layout, C, dtype, kind):
    """From one end of the gate's range to the other.  u = 2^-24: e = exp(-g) is off by 2^-22 (ex2.approx) and two products' roundings, 6 u;
    s = 1 / (1 + e) by that, a sum and an approximate quotient (2 units, 2^-22): 11 u; the smaller of s and 1 - s by one product more,
    12 u; the slope is its product with one minus it: 14 u.  All is multiplied by 1 and added to 0.  A gate of an image is done with expf (2
    units) and a division, which is less.  For a gate of each element in bf16 the exponent's argument is rounded too, |g| 2^-23 of e:
    2^-17 at 2^6."""
    first, T = layout == "first", 512 if kind == "full" else 1
    B = 512 // T
    g = torch.linspace(-64, 64, 512 * C, dtype=torch.float64, device="cuda")
    g = g[torch.randperm(512 * C, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")].view(512, C)
    g[0, 0], g[1, 0], g[2, 0], g[3, 0] = float("inf"), -float("inf"), torch.finfo(dtype).max, torch.finfo(dtype).min

    def lay(v):
        v = v.view(B, T, C)
        return v.permute(0, 2, 1).reshape(B, C, T, 1).contiguous() if first else v

    gate = lay(g.to(dtype)).requires_grad_(True)
    x, branch = torch.zeros(gate.shape, dtype=dtype, device="cuda"), torch.ones(gate.shape, dtype=dtype, device="cuda")
    if kind == "image":          # two pixels, so that it is one
        x, branch = (v.repeat(1, 1, 2, 1) if first else v.repeat(1, 2, 1) for v in (x, branch))
    branch.requires_grad_(True)
    y = CF.residual_norm(x, branch, gate=gate, gate_act="sigmoid", data_format="channels_" + layout)
    slope, through = torch.autograd.grad(y, (gate, branch), torch.ones_like(y))
    exact = gate.detach().double()
    e = torch.exp(-exact.abs())
    small, large = e / (1 + e), 1 / (1 + e)
    s, ds = torch.where(exact > 0, large, small).expand_as(y), small * large * (y.numel() // gate.numel())
    last = torch.finfo(dtype).eps / 2
    exactly = dtype == torch.float32 or kind == "image"
    for got, want, tol in ((y.detach().double(), s, 11 * 2.0 ** -24 if exactly else 2.0 ** -16),
                           (through.double(), s, 13 * 2.0 ** -24 if exactly else 2.0 ** -16),
                           (slope.double(), ds, 14 * 2.0 ** -24 if exactly else 2.0 ** -15)):
        over = (got - want).abs() - (tol + last) * want - 2.0 ** -126           # (numbers that fp32 flushes or loses digits of)
        assert float(over.max()) <= 0, float((over / want.clamp(min=2.0 ** -126)).max())


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["first", "last"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate", ["none", "full", "image"])
def test_a_token_of_one_channel_has_no_spread(layout, dtype, gate):
    """Its mean is itself: z is the bias, and nothing comes back through the norm.  The gradients' kernel forms y again, in every gate's
    way to the last bit, or its difference from the mean would be 300 times larger than a rounding."""
    t = _case(layout, 1, 2, 61, 47, dtype, "layer", False, gate, True)
    names = [n for n in NAMES if n in t]
    for n in names:
        t[n].requires_grad_(True)
    y, z = _call(t, layout, "layer", gate != "none")
    got = dict(zip(names, torch.autograd.grad((y, z), [t[n] for n in names], (t["dy"], t["dz"]))))
    assert torch.equal(z, t["pre_bias"].detach().to(dtype).expand_as(z))
    assert torch.equal(got["x"], t["dy"]) and float(got["pre_weight"]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    ("first", 64, 1, 128, 96, "fp32", "layer", True, "full", True),
    ("first", 300, 2, 9, 11, "fp32", "layer", True, "full", True),
    ("first", 96, 2, 15, 17, "bf16", "rms", False, "image", True),
    ("first", 1030, 1, 5, 7, "bf16", "layer", True, "image", False),
    ("last", 64, 2, 24, 20, "bf16", "layer", True, "full", True),
    ("last", 257, 3, 31, 3, "fp32", "layer", False, "full", False),
    ("last", 1024, 2, 31, 3, "fp32", "rms", True, "image", True),
], ids=lambda c: "-".join(map(str, c)))
def test_a_gate_that_is_taken_as_it_is(case):
    """gate_act None: against the formula, forward and gradients."""
    layout, C, B, H, W, dtype, norm, post, gate, scale = case
    t = _case(layout, C, B, H, W, {"fp32": torch.float32, "bf16": torch.bfloat16}[dtype], norm, post, gate, scale, seed=4)
    names = [n for n in NAMES if n in t]
    d = {n: v.double() for n, v in t.items()}
    for n in names:
        t[n].requires_grad_(True)
        d[n].requires_grad_(True)
    out, ref = _call(t, layout, norm, False), _formula(d, layout, norm, False)
    dim = 1 if layout == "first" else -1
    for a, b in zip(out, ref):
        _close(a, b, dim, "outputs")
    tops = _before_cancelling(d, layout, norm, False)
    got = torch.autograd.grad(out, [t[n] for n in names], (t["dy"], t["dz"]))
    want = torch.autograd.grad(ref, [d[n] for n in names], (d["dy"], d["dz"]))
    for n, a, b in zip(names, got, want):
        if n in ("x", "branch") or (n == "gate" and gate == "full"):
            _close(a, b, dim, n, tops[n])
        else:
            # sums over tokens of terms of both signs: 1e-5 of the norm, as the parts above are held to, and the type's rounding
            assert float((a.double() - b).norm()) <= (1e-5 + torch.finfo(a.dtype).eps / 2) * float(b.norm()), n
