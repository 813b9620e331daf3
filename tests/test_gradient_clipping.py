"""functional.grad_norm, clip_by_global_norm and clip_grad_norm_ against their formula in 64 bits.

The norm is rounded once to fp32 after sums that are exact to 8 . 2^-24 (eight squares in a row are added in fp32) and half of that in
the root: 5 . 2^-24.  A scaled value is the product of a value and a factor of that error, rounded: 7 . 2^-24, and 2^-8 in bf16."""
import ctypes
import math

import pytest
import torch

from conversenet_b200 import functional as CF

SIZES = [(1,), (3, 5), (64, 128, 1, 1), (8192,), (8193,), (100003,), (7, 0), (1, 128, 7, 7), (40, 40, 3, 3), (16384,)]


def _grads(dtype, seed, level=1.0, sizes=SIZES):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(level * (i + 1) * torch.randn(s, device="cuda", generator=g)).to(dtype[i % len(dtype)]) for i, s in enumerate(sizes)]


def _norm(grads, kind=2.0):
    every = torch.cat([g.double().flatten() for g in grads])
    return float(torch.linalg.vector_norm(every, kind))


def _check(out, grads, norm, max_norm):
    c = min(1.0, max_norm / (norm + 1e-6))
    for o, g in zip(out, grads):
        ref = g.double() * c
        tol = (7 * 2.0 ** -24 + (2.0 ** -8 if o.dtype == torch.bfloat16 else 0)) * ref.abs() + 2.0 ** -149
        assert o.shape == g.shape and bool(((o.double() - ref).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [(torch.float32,), (torch.bfloat16,), (torch.float32, torch.bfloat16)],
                         ids=["fp32", "bf16", "mixed"])
@pytest.mark.parametrize("kind", [2.0, 1.0, float("inf")])
@pytest.mark.parametrize("ratio", [0.0, 0.3, 0.999, 2.0])
def test_against_the_formula(dtype, kind, ratio):
    grads = _grads(dtype, 1)
    norm = _norm(grads, kind)
    out, got = CF.clip_by_global_norm(grads, ratio * norm, kind)
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(float(got) - norm) <= 5 * 2.0 ** -24 * norm
    _check(out, grads, norm, ratio * norm)
    assert float(CF.grad_norm(grads, kind)) == float(got)
    # into one buffer at odd places, in 32 bits
    flat = torch.full((sum(g.numel() for g in grads) + 3,), 5.0, device="cuda")
    parts = [p.view(g.shape) for p, g in zip(flat[1:-2].split([g.numel() for g in grads]), grads)]
    keep = [g.clone() for g in grads]
    same, got2 = CF.clip_by_global_norm(grads, ratio * norm, kind, out=parts)
    assert same is parts and float(got2) == float(got)
    _check(parts, grads, norm, ratio * norm)
    assert float(flat[0]) == 5 and bool((flat[-2:] == 5).all()) and all(torch.equal(a, b) for a, b in zip(keep, grads))
    # in place, as torch's own does it
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads] + [torch.nn.Parameter(torch.zeros(3, device="cuda"))]
    for p, g in zip(params, grads):
        p.grad = g.clone()
    version = params[0].grad._version
    got3 = CF.clip_grad_norm_(iter(params), ratio * norm, kind)
    assert float(got3) == float(got) and params[0].grad._version > version
    _check([p.grad for p in params[:-1]], grads, norm, ratio * norm)


@pytest.mark.gpu
def test_as_torch_does_it():
    grads = _grads((torch.float32,), 4)
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g.clone()
    want = torch.nn.utils.clip_grad_norm_(params, 3.0)
    theirs = [p.grad.clone() for p in params]
    for p, g in zip(params, grads):
        p.grad = g.clone()
    got = CF.clip_grad_norm_(params, 3.0)
    assert abs(float(got) - float(want)) <= 1e-5 * float(want)
    for p, t in zip(params, theirs):
        assert torch.allclose(p.grad, t, rtol=1e-5, atol=0)
    one = torch.nn.Parameter(torch.zeros(5, device="cuda"))
    one.grad = torch.ones(5, device="cuda")
    assert float(CF.clip_grad_norm_(one, 1.0)) == pytest.approx(math.sqrt(5))
    assert float(CF.clip_grad_norm_([torch.nn.Parameter(torch.zeros(5, device="cuda"))], 1.0)) == 0.0
    assert float(CF.grad_norm([])) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("level", [1e-44, 1e-30, 1e-20, 1e-13, 1e15, 1e25, 3e36])
def test_squares_beyond_fp32(level):
    grads = _grads((torch.float32,), 2, level)
    norm = _norm(grads)
    got = float(CF.grad_norm(grads))
    assert abs(got - norm) <= 5 * 2.0 ** -24 * norm + 2.0 ** -149 if norm < 3.4e38 else got == float("inf")
    if norm < 3.4e38 and level > 1e-30:
        out, _ = CF.clip_by_global_norm(grads, 0.5 * norm)
        _check(out, grads, norm, 0.5 * norm)
    mixed = grads + [torch.zeros(5000, device="cuda"), torch.full((9,), level, device="cuda")]
    assert float(CF.grad_norm(mixed)) >= got


@pytest.mark.gpu
def test_values_that_are_no_numbers():
    for kind in (2.0, 1.0, float("inf")):
        for at in (0, 8191, 8192, 100000):
            grads = _grads((torch.float32,), 3)
            grads[5][at] = float("inf")
            out, norm = CF.clip_by_global_norm(grads, 1.0, kind)
            assert float(norm) == float("inf") and not out[2].any() and math.isnan(float(out[5][at]))
            grads[4][5] = float("nan")
            out, norm = CF.clip_by_global_norm(grads, 1.0, kind)
            assert math.isnan(float(norm)) and bool(torch.isnan(out[2]).all())
    p = torch.nn.Parameter(torch.zeros(4, device="cuda"))
    p.grad = torch.tensor([1.0, float("nan"), 2.0, 3.0], device="cuda")
    with pytest.raises(RuntimeError, match="not finite"):
        CF.clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
    assert float(p.grad[0]) == 1.0


@pytest.mark.gpu
def test_many_tensors_layouts_and_offsets():
    g = torch.Generator(device="cuda").manual_seed(0)
    many = [torch.randn(1 + (37 * i) % 300, device="cuda", generator=g) for i in range(2500)]          # more than a launch takes
    norm = _norm(many)
    out, got = CF.clip_by_global_norm(many, 0.25 * norm)
    assert abs(float(got) - norm) <= 5 * 2.0 ** -24 * norm
    _check(out, many, norm, 0.25 * norm)
    # dense tensors of another order keep it; others are read through a copy
    a = torch.randn(4, 6, 5, 7, device="cuda", generator=g).to(memory_format=torch.channels_last)
    b = torch.randn(9, 40, device="cuda", generator=g)[:, ::3]
    c = torch.randn(1, 8, device="cuda", generator=g).expand(5, 8)
    out, got = CF.clip_by_global_norm([a, b, c], 1.0)
    norm = _norm([a, b, c])
    _check(out, [a, b, c], norm, 1.0)
    assert out[0].stride() == a.stride() and out[1].is_contiguous()
    into = [torch.empty(4, 6, 5, 7, device="cuda"), torch.empty(9, 14, device="cuda"), torch.empty(5, 8, device="cuda")]
    CF.clip_by_global_norm([a, b, c], 1.0, out=into)
    _check(into, [a, b, c], norm, 1.0)
    base = torch.randn(50001, device="cuda", generator=g)
    for first in range(1, 4):                       # vectors that begin between 16-byte boundaries, in and out
        v = base[first:]
        n = _norm([v])
        out, got = CF.clip_by_global_norm([v], 0.5 * n, out=[torch.empty(v.numel() + first, device="cuda")[first:]])
        _check(out, [v], n, 0.5 * n)
    h = base.bfloat16()
    for first in range(0, 9):
        v = h[first:]
        n = _norm([v])
        out, got = CF.clip_by_global_norm([v], 0.5 * n)
        _check(out, [v], n, 0.5 * n)


@pytest.mark.gpu
def test_streams_and_graphs():
    grads = _grads((torch.float32, torch.bfloat16), 6)
    out, norm = CF.clip_by_global_norm(grads, 2.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out2, norm2 = CF.clip_by_global_norm(grads, 2.0)
    side.synchronize()
    assert float(norm) == float(norm2) and all(torch.equal(a, b) for a, b in zip(out, out2))
    static = [g.clone() for g in grads]
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        a, na = CF.clip_by_global_norm(static, 2.0)
    with torch.cuda.graph(g2):
        b, nb = CF.clip_by_global_norm(static, 0.5)
    for s, g in zip(static, grads):
        s.copy_(4 * g)
    g2.replay()
    g1.replay()
    torch.cuda.synchronize()
    for o, n, m in ((a, na, 2.0), (b, nb, 0.5)):
        ref, rn = CF.clip_by_global_norm([4 * g for g in grads], m)
        assert float(n) == float(rn) and all(torch.equal(x, y) for x, y in zip(o, ref))


@pytest.mark.gpu
def test_elements_past_32_bits():
    n = (1 << 31) + 12345
    x = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    x[-5:] = 2.0
    x[0] = 4.0
    out, norm = CF.clip_by_global_norm([x], 3.0, out=[x])
    assert float(norm) == 6.0
    assert float(x[0]) == pytest.approx(2.0, rel=1e-2) and bool((x[-5:] == x[-1]).all()) and float(x[-1]) == pytest.approx(1.0, rel=1e-2)


@pytest.mark.gpu
def test_refusals():
    x, y = torch.ones(100, device="cuda"), torch.ones(100, device="cuda")
    for tensors, out in [([x, x], True), ([x, x[:50]], True),                          # the same memory twice
                         ([x, y], [y, x]), ([x[:50]], [x[25:75]]), ([x, y], [x, x]),   # written before it is read
                         ([x], [x.view(torch.bfloat16)[:100]]),
                         ([x], [y[:50]]), ([x], [y, y]), ([x[::2]], True), ([x], [y.half()]), ([x.double()], None), ([x.half()], None),
                         ([x, torch.ones(3)], None), ([x], [torch.ones(100)]), ([x.expand(4, 100)], True),
                         ([torch.eye(4, device="cuda").to_sparse()], None)]:
        with pytest.raises(RuntimeError):
            CF.clip_by_global_norm(tensors, 1.0, out=out)
    assert bool((x == 1).all()) and bool((y == 1).all())
    for bad in (-1.0, float("nan")):
        with pytest.raises(RuntimeError):
            CF.clip_by_global_norm([x], bad)
    with pytest.raises(ValueError):
        CF.grad_norm([x], 3.0)
    assert float(CF.grad_norm([x, x])) == pytest.approx(math.sqrt(200))                # read twice is fine


def test_refusals_without_a_device():
    with pytest.raises(RuntimeError, match="CUDA"):
        CF.grad_norm([torch.ones(3)])
    with pytest.raises(ValueError):
        CF.clip_by_global_norm([torch.ones(3)], 1.0, norm_type=0.5)


def test_c_abi_refusals():
    from conversenet_b200 import _cabi

    class Span(ctypes.Structure):
        _fields_ = [("in_", ctypes.c_void_p), ("out", ctypes.c_void_p), ("n", ctypes.c_longlong), ("in_type", ctypes.c_int),
                    ("out_type", ctypes.c_int)]

    lib = _cabi.load()
    p = ctypes.c_void_p(16)                                # never dereferenced: validation fails first
    ws = lib.cvb_clip_workspace_bytes(1)
    assert lib.cvb_clip_workspace_bytes(5000) > ws > 0

    def call(span=None, count=1, kind=2, max_norm=1.0, scale=1, norm=p, work=p, size=ws):
        s = (Span * 1)(span or Span(16, 16, 4, 0, 0))
        return lib.cvb_clip_by_norm(s, count, kind, max_norm, scale, norm, work, size, None)

    assert call(Span(None, 16, 4, 0, 0)) == -1
    assert call(Span(16, None, 4, 0, 0)) == -1
    assert call(Span(18, 16, 4, 0, 0)) == -1               # between elements
    assert call(Span(16, 17, 4, 0, 1)) == -1
    assert call(Span(16, 16, 4, 0, 1)) == -1               # in place needs one type
    assert call(Span(16, 16, -1, 0, 0)) == -1
    assert call(Span(16, 16, 1 << 45, 0, 0)) == -7
    assert call(Span(16, 16, 4, 3, 0)) == -1
    assert call(kind=3) == call(count=-1) == call(norm=None) == call(max_norm=-1.0) == call(max_norm=float("nan")) == -1
    assert call(work=None) == call(size=ws - 1) == -4


def test_c_abi_addresses():
    from conversenet_b200 import _cabi
    lib = _cabi.load()
    p, size = ctypes.c_void_p(16), lib.cvb_clip_workspace_bytes(0)        # never dereferenced: validation fails first

    def call(norm=p, work=p):
        return lib.cvb_clip_by_norm(None, 0, 2, 1.0, 0, norm, work, size, None)

    assert call(work=ctypes.c_void_p(20)) == -4                # sums of 64 bits
    assert call(norm=ctypes.c_void_p(18)) == -1


@pytest.mark.gpu
def test_tensors_with_a_history():
    """No result has one: where one would be recorded the call is refused; `clip_grad_norm_` records none, as torch's own does not."""
    import torch.autograd.forward_ad as fwd
    p = torch.nn.Parameter(torch.randn(50, device="cuda"))
    x = torch.randn(50, device="cuda")
    loss = (p ** 3).sum()
    grad, = torch.autograd.grad(loss, p, create_graph=True)
    assert grad.requires_grad
    for call in (lambda: CF.grad_norm([x, grad]), lambda: CF.grad_norm([p]), lambda: CF.clip_by_global_norm([grad], 1.0),
                 lambda: CF.clip_by_global_norm([x], 1.0, out=[p]), lambda: CF.clip_by_global_norm([x], 1.0, out=[p * 1])):
        with pytest.raises(RuntimeError, match="no_grad"):
            call()
    with torch.no_grad():
        assert float(CF.grad_norm([grad])) == pytest.approx(float(grad.norm()), rel=1e-5)
        out, _ = CF.clip_by_global_norm([grad], 1.0)
        CF.clip_by_global_norm([x], 1.0, out=[p])
    assert not out[0].requires_grad and float(p.norm()) == pytest.approx(1.0, rel=1e-5)
    p.grad = grad
    before = float(grad.norm())
    assert float(CF.clip_grad_norm_([p], 0.5 * before, error_if_nonfinite=True)) == pytest.approx(before, rel=1e-5)
    assert float(p.grad.norm()) == pytest.approx(0.5 * before, rel=1e-5)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: CF.grad_norm([dual]), lambda: CF.clip_by_global_norm([dual], 1.0)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


@pytest.mark.gpu
def test_outputs_from_any_iterable():
    x = [torch.randn(9, device="cuda"), torch.randn(5, device="cuda")]
    into = [torch.empty_like(t) for t in x]
    out, norm = CF.clip_by_global_norm(iter(x), 0.5, out=iter(into))
    assert [a is b for a, b in zip(out, into)] == [True, True]
    _check(into, x, float(norm), 0.5)
    with pytest.raises(RuntimeError):
        CF.clip_by_global_norm([], 0.5, out=into)
    assert CF.clip_by_global_norm([], 0.5, out=[])[0] == []
    with pytest.raises(TypeError):
        CF.clip_by_global_norm(x, 0.5, out=False)
