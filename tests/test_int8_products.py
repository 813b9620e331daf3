"""functional.quantize_tokens, quantize_weight, int8_product and pointwise_int8 against their definitions in 64 bits.

The integers have to be equal, borders between two of them included.  A product's sum is exact in 32 bits; of what follows, the
conversion of the sum, the scale, two products and an addition round, each by 2^-24 at most: 5 . 2^-24 of the product's magnitude and
2^-24 of the result's, plus 2^-8 of the result in bf16."""
import ctypes

import pytest
import torch

from conversenet_b200 import Int8Pointwise
from conversenet_b200 import functional as CF

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _integers(x):
    """The nearest integers to 127 x / max |x| over the last dimension, an even one where two are as near."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    low = torch.floor(127 * x / torch.where(top == 0, 1.0, top))
    above = 254 * x - (2 * low + 1) * top
    return low + ((above > 0) | ((above == 0) & (low % 2 != 0))).double(), top / 127


def _rows(x, first):
    return x.permute(0, 2, 3, 1) if first else x


def _features(shape, first, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, device="cuda", generator=g)
    token = list(shape)
    token[1 if first else -1] = 1
    return (x * torch.exp(2 * torch.randn(token, device="cuda", generator=g))).to(dtype)


def _check_product(out, q, scale, weight_q, weight_scale, bias, first):
    ref = (q @ weight_q.double().t()) * scale * weight_scale.double()
    size = ref.abs()
    if bias is not None:
        ref = ref + bias.double()
    tol = 5 * 2.0 ** -24 * size + 2.0 ** -24 * ref.abs() + (2.0 ** -8 * ref.abs() if out.dtype == torch.bfloat16 else 0)
    over = (_rows(out, first).double() - ref).abs() - tol
    assert float(over.max()) <= 0, float(over.max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("K", [1, 3, 16, 17, 64, 100, 128, 250, 512, 600, 5000])
def test_integers_are_the_nearest(K, dtype):
    dtype = DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(K)
    T = 2000 if K <= 600 else 240
    plain = torch.randn(T, K, device="cuda", generator=g) * torch.exp(8 * torch.randn(T, 1, device="cuda", generator=g))
    halves = torch.randint(-126, 126, (T, K), device="cuda", generator=g) + 0.5           # largest 127: every value a border
    halves[:, 0] = 127
    top = torch.randint(1 << 23, 1 << 24, (T, 1), device="cuda", generator=g).double()
    odd = 2 * torch.randint(-127, 127, (T, K), device="cuda", generator=g).double() + 1
    near = (odd * top / 254).float()                                                      # borders as near as fp32 comes
    near[:, 0] = top[:, 0].float()
    beside = torch.nextafter(near, torch.randn(T, K, device="cuda", generator=g) * 1e9)
    beside[:, 0] = top[:, 0].float()
    for name, x in (("plain", plain), ("halves", halves), ("near", near), ("beside", beside), ("tiny", plain * 1e-35),
                    ("subnormal", plain * 1e-40), ("half of the largest", torch.round(plain.sign()) * (0.5 + 0.5 * (plain > 0)))):
        x = x.to(dtype).contiguous()
        ref, scale = _integers(x)
        q, s = CF.quantize_tokens(x, "channels_last")
        assert q.dtype == torch.int8 and q.shape == x.shape and s.shape == (T,)
        assert torch.equal(q.double(), ref), name
        # a quotient rounded once; of subnormal numbers by half of 2^-149
        assert bool(((s.double() - scale[:, 0]).abs() <= 2.0 ** -24 * scale[:, 0] + 2.0 ** -150).all()), name
        W = 40
        planes = x.t().reshape(1, K, T // W, W).contiguous()
        q2, s2 = CF.quantize_tokens(planes)
        assert torch.equal(q2.reshape(T, K), q) and torch.equal(s2.reshape(T), s), name
        if K <= 600:
            # the same integers on the way to a product: with unit weights they come out times the scale
            unit = torch.eye(K, dtype=torch.int8, device="cuda")
            out = CF.pointwise_int8(planes.float() if dtype == torch.float32 else planes, unit, torch.ones(K, device="cuda"))
            want = (ref * s.double()[:, None]).to(dtype)
            assert torch.equal(out.reshape(K, T).t(), want if dtype == torch.float32 else (q.float() * s[:, None]).to(dtype)) or \
                name in ("tiny", "subnormal"), name


PRODUCTS = [
    # layout, B, H, W, K, N, dtype, bias
    ("first", 1, 24, 20, 64, 128, "fp32", True),
    ("first", 2, 33, 31, 64, 128, "bf16", True),
    ("first", 3, 5, 7, 1, 1, "fp32", False),
    ("first", 1, 16, 16, 33, 10, "fp32", True),
    ("first", 2, 61, 47, 128, 64, "bf16", False),
    ("first", 1, 20, 20, 127, 300, "fp32", True),          # more output channels than a pass
    ("first", 1, 200, 201, 96, 160, "fp32", True),         # two groups a block
    ("first", 2, 9, 11, 129, 70, "fp32", True),            # beyond the kernel that quantises on the way
    ("first", 1, 40, 40, 300, 520, "bf16", True),
    ("first", 1, 2, 3, 64, 700, "fp32", True),
    ("first", 5, 1, 1, 64, 64, "fp32", True),
    ("last", 1, 1, 1, 64, 64, "fp32", True),
    ("last", 1, 24, 20, 64, 128, "fp32", False),
    ("last", 3, 43, 1, 100, 77, "bf16", True),
    ("last", 2, 31, 17, 1000, 333, "fp32", True),
    ("last", 1, 130, 1, 4096, 257, "bf16", False),
    ("last", 40, 64, 1, 256, 1024, "fp32", True),          # every tile width
    ("last", 1, 300, 200, 48, 64, "fp32", True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", PRODUCTS, ids=lambda c: "-".join(map(str, c)))
def test_against_the_definition(case):
    layout, B, H, W, K, N, dtype, with_bias = case
    first, dtype = layout == "first", DTYPES[dtype]
    x = _features((B, K, H, W) if first else (B, H * W, K), first, dtype, K + N)
    g = torch.Generator(device="cuda").manual_seed(N)
    weight = torch.randn(N, K, device="cuda", generator=g)
    bias = torch.randn(N, device="cuda", generator=g) if with_bias else None
    wq, ws = CF.quantize_weight(weight.view(N, K, 1, 1) if first else weight)
    ref, wscale = _integers(weight)
    assert torch.equal(wq.double(), ref) and wq.shape == (N, K) and wq.stride(0) % 16 == 0
    q, scale = _integers(_rows(x, first))
    out = CF.pointwise_int8(x, wq, ws, bias, "channels_" + layout)
    assert out.dtype == dtype and out.is_contiguous()
    assert out.shape == ((B, N, H, W) if first else (B, H * W, N))
    _check_product(out, q, scale, wq, ws, bias, first)
    assert torch.equal(out, CF.pointwise_int8(x, wq, ws, bias, "channels_" + layout))
    # the two parts by themselves; weights and tokens in rows that begin anywhere
    qt, st = CF.quantize_tokens(x, "channels_" + layout)
    two = CF.int8_product(qt, st, wq, ws, bias, dtype, "channels_" + layout)
    _check_product(two, q, scale, wq, ws, bias, first)
    copies = CF.int8_product(qt.contiguous(), st, wq.contiguous(), ws, bias, dtype, "channels_" + layout)
    assert torch.equal(two, copies)
    from conversenet_b200 import _cabi
    assert _cabi.load().cvb_last_device_status(1) == 0


@pytest.mark.gpu
def test_extremes():
    """The largest sums, rows of zeros, tokens with infinities and NaN, long tokens, magnitudes at the ends of fp32."""
    K = 131072
    q = torch.full((3, K), 127, dtype=torch.int8, device="cuda")
    q[1] = -127
    q[2, ::2] = -127
    w = torch.full((2, K), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    one = torch.ones(3, device="cuda")
    out = CF.int8_product(q, one, w, torch.ones(2, device="cuda"))
    want = (q.double() @ w.double().t())
    assert float((out.double() - want).abs().max()) <= 2.0 ** -24 * 2.0 ** 31
    for K, first in ((64, True), (300, True), (64, False), (5000, False)):
        shape = (1, K, 10, 20) if first else (200, K)
        x = _features(shape, first, torch.float32, 1)
        rows = _rows(x, first).reshape(200, K) if not first else None
        N = 48
        wq, ws = CF.quantize_weight(torch.randn(N, K, device="cuda"))
        bias = torch.randn(N, device="cuda")
        fmt = "channels_first" if first else "channels_last"
        plain = CF.pointwise_int8(x, wq, ws, bias, fmt)
        view = (lambda t: t.reshape(t.shape[1], 200).t()) if first else (lambda t: t)
        x2 = x.clone()
        view(x2)[3] = 0
        view(x2)[5, K // 2] = float("inf")
        view(x2)[7, 0] = float("-inf")
        view(x2)[11, K - 1] = float("nan")
        view(x2)[13] *= 1e-37 / view(x2)[13].abs().max()
        view(x2)[17] *= 3e38 / view(x2)[17].abs().max()
        y = view(CF.pointwise_int8(x2, wq, ws, bias, fmt))
        p = view(plain)
        same = [i for i in range(200) if i not in (3, 5, 7, 11, 13, 17)]
        assert torch.equal(y[same], p[same])
        assert torch.equal(y[3], bias)
        for i in (5, 7, 11):
            assert bool(torch.isnan(y[i]).all())
        qq, ss = CF.quantize_tokens(x2, fmt)
        qq, ss = qq.reshape(200, K), ss.reshape(200)
        for i in (5, 7, 11):
            assert bool(torch.isnan(ss[i])) and not qq[i].any()
        assert not qq[3].any() and float(ss[3]) == 0
        ref, scale = _integers(view(x2)[[13, 17]])
        assert torch.equal(qq[[13, 17]].double(), ref)
        want = (ref @ wq.double().t()) * scale * ws.double() + bias.double()
        # (beyond the largest fp32 number, 2^128 - 2^103 once rounded, an infinity)
        fits, over = want.abs() < 2.0 ** 127.999, want.abs() > 2.0 ** 128
        got = y[[13, 17]].double()
        assert float(((got - want).abs() - 2.0 ** -20 * want.abs())[fits].max()) <= 0
        assert torch.equal(got[over], want[over].sign() * float("inf"))
    # nothing to do
    wq, ws = CF.quantize_weight(torch.randn(8, 16, device="cuda"))
    assert CF.pointwise_int8(torch.zeros(0, 16, 3, 3, device="cuda"), wq, ws).shape == (0, 8, 3, 3)
    assert CF.pointwise_int8(torch.zeros(0, 16, device="cuda"), wq, ws, data_format="channels_last").shape == (0, 8)


@pytest.mark.gpu
def test_many_small_images_and_other_ranks():
    """Images of one pixel, which are tokens side by side, and of a few; tokens with more dimensions."""
    wq, ws = CF.quantize_weight(torch.randn(40, 64, device="cuda"))
    x = _features((30000, 64, 1, 1), True, torch.float32, 2)
    y = CF.pointwise_int8(x, wq, ws)
    assert torch.equal(y.flatten(1), CF.pointwise_int8(x.flatten(1), wq, ws, data_format="channels_last"))
    q, s = CF.quantize_tokens(x)
    assert q.shape == (30000, 1, 1, 64) and torch.equal(CF.int8_product(q, s, wq, ws, data_format="channels_first"), y)
    x = _features((3000, 64, 1, 2), True, torch.bfloat16, 3)
    q, scale = _integers(_rows(x, True))
    _check_product(CF.pointwise_int8(x, wq, ws), q, scale, wq, ws, None, True)
    x = _features((2, 3, 5, 7, 64), False, torch.float32, 4)
    y = CF.pointwise_int8(x, wq, ws, data_format="channels_last")
    assert y.shape == (2, 3, 5, 7, 40) and torch.equal(y.view(-1, 40), CF.pointwise_int8(x.view(-1, 64), wq, ws, data_format="channels_last"))


@pytest.mark.gpu
def test_module_streams_and_graphs():
    torch.manual_seed(0)
    conv = torch.nn.Conv2d(70, 33, 1).cuda()
    lin = torch.nn.Linear(70, 33, bias=False).cuda()
    mc, ml = Int8Pointwise(conv), Int8Pointwise(lin)
    x = _features((2, 70, 19, 23), True, torch.float32, 5)
    with torch.no_grad():
        y = mc(x)
        # half a step for each weight and each input value, an input of a token's largest size
        ref = torch.nn.functional.conv2d(x.double(), conv.weight.double(), conv.bias.double())
        top = x.abs().amax(1, keepdim=True).double()
        wtop = conv.weight.abs().amax(1).double().view(1, -1, 1, 1)
        steps = (x.abs().double().sum(1, keepdim=True) * wtop + top * conv.weight.abs().double().sum(1).view(1, -1, 1, 1)) / 254
        bound = steps + 70 * top * wtop / 254 ** 2
        assert float(((y.double() - ref).abs() - 1.0001 * bound - 1e-5).max()) <= 0
        t = x.permute(0, 2, 3, 1).contiguous()
        assert torch.equal(ml(t), CF.pointwise_int8(t, *CF.quantize_weight(lin.weight), None, "channels_last"))
        # copies and state dicts
        import copy
        other = copy.deepcopy(mc)
        other.load_state_dict(Int8Pointwise(torch.nn.Conv2d(70, 33, 1).cuda()).state_dict())
        other.load_state_dict(mc.state_dict())
        assert torch.equal(other(x), y)
        # another stream; two captured graphs replayed in the other order
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            z = mc(x)
        side.synchronize()
        assert torch.equal(y, z)
        sx, st = x.clone(), t.clone()
        ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(ga):
            a = mc(sx)
        with torch.cuda.graph(gb):
            b = ml(st)
        sx.copy_(-3 * x)
        st.copy_(-3 * t)
        gb.replay()
        ga.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, mc(-3 * x)) and torch.equal(b, ml(-3 * t))
        # strided inputs
        assert torch.equal(mc(x.to(memory_format=torch.channels_last)), y)
        wide = torch.zeros(2, 70, 19, 46, device="cuda")
        wide[..., ::2] = x
        assert torch.equal(mc(wide[..., ::2]), y)
        base = torch.zeros(x.numel() + 1, device="cuda")
        base[1:] = x.flatten()
        assert torch.equal(mc(base[1:].view_as(x)), y)
        base[1:] = t.flatten()
        assert torch.equal(ml(base[1:].view_as(t)), ml(t))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Outputs of 2^31 elements and more, their last tokens against a call of those tokens alone."""
    K, N = 16, 64
    HW = (1 << 25) + 130
    g = torch.Generator(device="cuda").manual_seed(0)
    wq, ws = CF.quantize_weight(torch.randn(N, K, device="cuda", generator=g))
    tail = torch.randn(1, K, 1, 300, device="cuda", generator=g).bfloat16()
    x = torch.zeros(1, K, 1, HW, dtype=torch.bfloat16, device="cuda")
    x[..., -300:] = tail
    y = CF.pointwise_int8(x, wq, ws)
    assert torch.equal(y[..., -300:], CF.pointwise_int8(tail, wq, ws)) and not y[..., :5000].any()
    t = x.view(K, HW).t().contiguous()
    del x, y
    y = CF.pointwise_int8(t, wq, ws, data_format="channels_last")
    assert torch.equal(y[-300:], CF.pointwise_int8(t[-300:].clone(), wq, ws, data_format="channels_last")) and not y[:5000].any()


@pytest.mark.gpu
def test_refusals():
    x = torch.randn(1, 16, 4, 4, device="cuda")
    wq, ws = CF.quantize_weight(torch.randn(8, 16, device="cuda"))
    for args in [(x[0], wq, ws), (x.half(), wq, ws), (x, wq[:, :8], ws), (x, wq.float(), ws), (x, wq, ws[:4]), (x, wq, ws, ws[:4]),
                 (x, wq.cpu(), ws), (x, wq, ws.cpu()), (x, wq, ws.int()), (x, wq[0], ws)]:
        with pytest.raises(RuntimeError):
            CF.pointwise_int8(*args)
    with pytest.raises(ValueError):
        CF.pointwise_int8(x, wq, ws, data_format="NHWC")
    with pytest.raises(RuntimeError, match="inference"):
        CF.pointwise_int8(x.clone().requires_grad_(True), wq, ws)
    with pytest.raises(RuntimeError, match="inference"):
        CF.quantize_tokens(x.clone().requires_grad_(True))
    with torch.no_grad():
        CF.pointwise_int8(x.clone().requires_grad_(True), wq, ws)
    q, s = CF.quantize_tokens(x)
    for args in [(q.int(), s, wq, ws), (q, s[:, :2], wq, ws), (q, s, wq[:, :4], ws)]:
        with pytest.raises(RuntimeError):
            CF.int8_product(*args)
    with pytest.raises(RuntimeError):
        CF.int8_product(q, s, wq, ws, dtype=torch.float16)
    with pytest.raises(RuntimeError):
        CF.int8_product(q[0], s[0], wq, ws, data_format="channels_first")
    with pytest.raises(RuntimeError, match="131072"):
        CF.quantize_tokens(torch.zeros(1, 131073, device="cuda"), "channels_last")


def test_refusals_without_a_device():
    with pytest.raises(RuntimeError, match="CUDA"):
        CF.pointwise_int8(torch.zeros(1, 4, 2, 2), torch.zeros(4, 4, dtype=torch.int8), torch.ones(4))
    with pytest.raises(TypeError):
        Int8Pointwise(torch.nn.GELU())
    for conv in (torch.nn.Conv2d(4, 4, 3), torch.nn.Conv2d(4, 4, 1, stride=2), torch.nn.Conv2d(4, 4, 1, groups=2),
                 torch.nn.Conv2d(4, 4, 1, padding=1)):
        with pytest.raises(ValueError):
            Int8Pointwise(conv)


def test_c_abi_refusals():
    from conversenet_b200 import _cabi
    lib = _cabi.load()
    p = ctypes.c_void_p(16)                                # never dereferenced: validation fails first
    odd = ctypes.c_void_p(24)
    assert lib.cvb_quantize_tokens(None, p, p, 1, 4, 8, 16, 0, 0, None) == -1
    assert lib.cvb_quantize_tokens(p, odd, p, 1, 4, 8, 16, 0, 0, None) == -1
    assert lib.cvb_quantize_tokens(p, p, p, 1, 4, 8, 8, 0, 0, None) == -1          # rows between 16-byte boundaries
    assert lib.cvb_quantize_tokens(p, p, p, 1, 4, 17, 16, 0, 0, None) == -1
    assert lib.cvb_quantize_tokens(p, p, p, 0, 4, 8, 16, 0, 0, None) == -1
    assert lib.cvb_quantize_tokens(p, p, p, 1, 4, 8, 16, 0, 4, None) == -1
    assert lib.cvb_quantize_tokens(p, p, p, 1, 4, 131073, 131088, 0, 0, None) == -7
    assert lib.cvb_quantize_tokens(p, p, p, 1 << 20, 1 << 20, 8, 16, 0, 0, None) == -7
    f = lib.cvb_int8_product
    assert f(p, 16, p, p, 16, p, None, None, 1, 4, 8, 4, 0, 0, None) == -1
    assert f(p, 16, p, odd, 16, p, None, p, 1, 4, 8, 4, 0, 0, None) == -1
    assert f(p, 16, p, p, 8, p, None, p, 1, 4, 8, 4, 0, 0, None) == -1
    assert f(p, 16, p, p, 16, p, None, p, 1, 4, 8, 0, 0, 0, None) == -1
    need = lib.cvb_pointwise_int8_workspace_bytes(1, 100, 300, 8, 1, 0)
    assert need >= 100 * 304 + 400
    assert lib.cvb_pointwise_int8_workspace_bytes(1, 100, 64, 8, 0, 0) == 0          # quantised on the way
    assert lib.cvb_pointwise_int8(p, p, 304, p, None, p, 1, 100, 300, 8, 1, 0, None, 0, None) == -4
    assert lib.cvb_pointwise_int8(p, p, 304, p, None, p, 1, 100, 300, 8, 1, 0, p, need - 1, None) == -4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("K", [3, 64, 128, 250, 600, 5000])
@pytest.mark.parametrize("power", [95, 96, 97, 103, 104])
def test_integers_of_large_tokens_are_the_nearest(K, dtype, power):
    """Borders between two integers in tokens up to the largest finite number: the constructions of the test above times a power of
    two, which is exact (the largest magnitudes are 2^23 to 2^24 times it)."""
    dtype = DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(K + power)
    T = 2000 if K <= 600 else 240
    up = 2.0 ** power
    top = torch.randint(1 << 23, 1 << 24, (T, 1), device="cuda", generator=g).float()
    top[0] = (1 << 24) - 1
    odd = 2 * torch.randint(-127, 127, (T, K), device="cuda", generator=g).double() + 1
    near = (odd * top.double() / 254).float()
    beside = torch.nextafter(near, torch.randn(T, K, device="cuda", generator=g) * 1e9)
    halves = 131072.0 * (torch.randint(-126, 126, (T, K), device="cuda", generator=g) + 0.5)
    half = torch.where(torch.rand(T, K, device="cuda", generator=g) < 0.5, 0.5 * top, -0.5 * top)
    near[:, 0] = beside[:, 0] = half[:, 0] = top[:, 0]
    halves[:, 0] = 127 * 131072.0
    for name, x in (("near", near), ("beside", beside), ("halves", halves), ("half of the largest", half)):
        if dtype == torch.bfloat16:          # (rounded first: the largest would become an infinity)
            x = x.clamp(-16711680.0, 16711680.0).to(dtype).float()
        x = (x * up).to(dtype)
        assert bool(torch.isfinite(x).all())
        ref, scale = _integers(x)
        q, s = CF.quantize_tokens(x, "channels_last")
        assert torch.equal(q.double(), ref), name
        assert bool(((s.double() - scale[:, 0]).abs() <= 2.0 ** -24 * scale[:, 0]).all()), name
        planes = x.t().reshape(1, K, T // 40, 40).contiguous()
        q2, s2 = CF.quantize_tokens(planes)
        assert torch.equal(q2.reshape(T, K), q) and torch.equal(s2.reshape(T), s), name
        if K <= 128:
            # on the way to a product: unit weights of 2^-8, so that no result is beyond fp32
            out = CF.pointwise_int8(planes, torch.eye(K, dtype=torch.int8, device="cuda"), torch.full((K,), 2.0 ** -8, device="cuda"))
            want = ((q.float() * 2.0 ** -8) * s[:, None]).to(dtype)
            assert torch.equal(out.reshape(K, T).t(), want), name


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["first", "last"])
def test_the_largest_sum_of_all(layout):
    """131072 products of -128 and -128 are 2^31, one more than a signed 32-bit integer holds; every one of these sums is an fp32
    number."""
    K = 131072
    q = torch.full((1, 1, 3, K), -128, dtype=torch.int8, device="cuda")
    q[0, 0, 1] = 127
    q[0, 0, 2, K // 2:] = 0
    w = torch.full((300, K), -128, dtype=torch.int8, device="cuda")
    w[1::3] = 127
    w[2::3, :] = 0
    out = CF.int8_product(q, torch.ones(1, 1, 3, device="cuda"), w, torch.ones(300, device="cuda"), data_format="channels_" + layout)
    want = torch.tensor([[-128.0 * -128, -128 * 127, 0], [127 * -128, 127 * 127, 0], [-64 * -128, -64 * 127, 0]],
                        dtype=torch.float64, device="cuda").repeat(1, 100) * K
    assert float(want.max()) == 2.0 ** 31 and torch.equal(want.float().double(), want)
    assert torch.equal(out.permute(0, 2, 3, 1).reshape(3, 300).double() if layout == "first" else out.reshape(3, 300).double(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [17, 128, 140])
@pytest.mark.parametrize("HW", [2, 5, 31, 33, 95, 127, 129, 300])
def test_planes_that_end_inside_a_warp(HW, K):
    """The last pixels of each image leave some of a warp's lanes without one, in several groups of output channels."""
    B, N = 3, 305
    g = torch.Generator(device="cuda").manual_seed(HW + K)
    x = torch.randn(B, K, 1, HW, device="cuda", generator=g)
    wq, ws = CF.quantize_weight(torch.randn(N, K, device="cuda", generator=g))
    q, scale = _integers(_rows(x, True))
    _check_product(CF.pointwise_int8(x, wq, ws), q, scale, wq, ws, None, True)
    qt, st = CF.quantize_tokens(x)
    for fmt in ("channels_first", "channels_last"):
        _check_product(CF.int8_product(qt, st, wq, ws, data_format=fmt), q, scale, wq, ws, None, fmt == "channels_first")


def test_c_abi_addresses():
    from conversenet_b200 import _cabi
    lib = _cabi.load()
    p = ctypes.c_void_p(16)                                # never dereferenced: validation fails first
    f = lib.cvb_int8_product
    # addresses between elements
    assert lib.cvb_quantize_tokens(ctypes.c_void_p(18), p, p, 1, 4, 8, 16, 0, 0, None) == -1
    assert lib.cvb_quantize_tokens(ctypes.c_void_p(17), p, p, 1, 4, 8, 16, 0, 1, None) == -1
    between = ctypes.c_void_p(18)
    assert lib.cvb_quantize_tokens(p, p, between, 1, 4, 8, 16, 0, 0, None) == -1
    assert f(p, 16, between, p, 16, p, None, p, 1, 4, 8, 4, 0, 0, None) == -1
    assert f(p, 16, p, p, 16, between, None, p, 1, 4, 8, 4, 0, 0, None) == -1
    assert f(p, 16, p, p, 16, p, between, p, 1, 4, 8, 4, 0, 0, None) == -1
    assert f(p, 16, p, p, 16, p, None, between, 1, 4, 8, 4, 0, 0, None) == -1
    for change in (0, 3, 4, 5):
        args = [p, p, 64, p, p, p]
        args[change] = between
        assert lib.cvb_pointwise_int8(*args, 1, 100, 64, 8, 0, 0, None, 0, None) == -1, change


@pytest.mark.gpu
def test_a_module_of_another_type_keeps_its_scales():
    """Casting the module leaves scales and biases in 32 bits: rounded to bf16 every output would be 2^-9 off."""
    torch.manual_seed(1)
    conv = torch.nn.Conv2d(64, 48, 1).cuda()
    x = _features((1, 64, 9, 10), True, torch.float32, 6)
    m = Int8Pointwise(conv)
    y = m(x)
    state = m.state_dict()
    for cast in (torch.nn.Module.bfloat16, torch.nn.Module.half, torch.nn.Module.double, lambda n: n.cpu().to("cuda", torch.bfloat16)):
        n = cast(torch.nn.Sequential(Int8Pointwise(conv)))
        assert n[0].weight_scale.dtype == n[0].bias.dtype == torch.float32 and n[0].weight_scale.is_cuda
        assert torch.equal(n(x), y)
        n[0].load_state_dict(state)
        assert torch.equal(n(x), y)
    assert Int8Pointwise(torch.nn.Linear(64, 8, bias=False).cuda()).bfloat16().bias is None


@pytest.mark.gpu
def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd
    x = torch.randn(1, 16, 4, 4, device="cuda")
    wq, ws = CF.quantize_weight(torch.randn(8, 16, device="cuda"))
    bias = torch.randn(8, device="cuda")
    q, s = CF.quantize_tokens(x)
    with fwd.dual_level():
        dual = [fwd.make_dual(v, torch.ones_like(v)) for v in (x, ws, bias, s)]
        for call in (lambda: CF.pointwise_int8(dual[0], wq, ws, bias), lambda: CF.pointwise_int8(x, wq, dual[1], bias),
                     lambda: CF.pointwise_int8(x, wq, ws, dual[2]), lambda: CF.quantize_tokens(dual[0]),
                     lambda: CF.int8_product(q, dual[3], wq, ws), lambda: CF.int8_product(q, s, wq, dual[1]),
                     lambda: CF.int8_product(q, s, wq, ws, dual[2])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
