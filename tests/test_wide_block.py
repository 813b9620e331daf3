"""A block of 96 channels, which the fused 64-channel kernels do not take, built from the operators: trained with a clipped step, and
served in 8-bit integers, against the same block of plain tensor operations around the same Converse2D layers."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from conversenet_b200 import Converse2D, Int8Pointwise, LayerNorm, ResidualNorm
from conversenet_b200 import functional as CF

C = 96


class Block(nn.Module):
    """x + a1 N(conv1(N(x))), then y + a2 N(conv2(N(y))): `ConverseBlockAlphaVariant` with a norm behind each branch and a gate."""

    def __init__(self):
        super().__init__()
        self.first = LayerNorm(C, eps=1e-5, data_format="channels_first")
        self.up = nn.ModuleList([nn.Conv2d(C, 2 * C, 1), nn.Conv2d(C, 2 * C, 1)])
        self.down = nn.ModuleList([nn.Conv2d(2 * C, C, 1), nn.Conv2d(2 * C, C, 1)])
        self.converse = Converse2D(2 * C, 2 * C, 3, padding=2)
        self.seams = nn.ModuleList([ResidualNorm(C, gate_act="sigmoid"), ResidualNorm(C, pre=False, gate_act="sigmoid")])

    def branch(self, i, z):
        t = F.gelu(self.up[i](z))
        if i == 0:
            t = F.gelu(self.converse(t))
        return self.down[i](t)

    def forward(self, x, gate):
        b = self.branch(0, self.first(x))
        y, z = self.seams[0](x, b, gate)
        return self.seams[1](y, self.branch(1, z), gate)

    def plain(self, x, gate):
        def norm(v, w, b):
            v = v - v.mean(1, keepdim=True)
            return v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-5) * w.view(1, -1, 1, 1) + b.view(1, -1, 1, 1)

        z = self.first(x)
        for i, s in enumerate(self.seams):
            x = x + s.scale * torch.sigmoid(gate) * norm(self.branch(i, z), s.post_weight, s.post_bias)
            if i == 0:
                z = norm(x, s.pre_weight, s.pre_bias)
        return x


@pytest.fixture
def block():
    before = torch.backends.cudnn.allow_tf32, torch.backends.cuda.matmul.allow_tf32
    torch.backends.cudnn.allow_tf32 = torch.backends.cuda.matmul.allow_tf32 = False
    torch.manual_seed(0)
    m = Block().cuda()
    with torch.no_grad():
        for s in m.seams:
            s.scale.copy_(0.5 + torch.rand_like(s.scale))
            s.post_weight.add_(0.2 * torch.randn_like(s.post_weight))
    yield m
    torch.backends.cudnn.allow_tf32, torch.backends.cuda.matmul.allow_tf32 = before


@pytest.mark.gpu
def test_a_training_step(block):
    x = torch.randn(2, C, 33, 28, device="cuda")
    gate = torch.randn(2, C, 1, 1, device="cuda", requires_grad=True)
    go = torch.randn_like(x)
    params = list(block.parameters())
    ref = torch.autograd.grad(block.plain(x, gate), params + [gate], go)
    out = block(x, gate)
    out.backward(go)
    # the two differ by the order of fp32 sums, which a block passes on a few times: 1e-4 of each gradient's norm at most, as the
    # 64-channel block's gradients are held to
    for p, r in zip(params + [gate], ref):
        assert float((p.grad - r).norm()) <= 1e-4 * float(r.norm()) + 1e-6, tuple(p.shape)
    total = torch.sqrt(sum(r.double().square().sum() for r in ref[:-1]))
    grads = [p.grad.clone() for p in params]
    norm = CF.clip_grad_norm_(params, 0.1)
    assert abs(float(norm) - float(total)) <= 1e-4 * float(total)
    for p, g in zip(params, grads):
        assert torch.allclose(p.grad, g * (0.1 / (float(norm) + 1e-6)), rtol=1e-5, atol=0)
    assert float(CF.grad_norm([p.grad for p in params])) == pytest.approx(0.1, rel=1e-4)


@pytest.mark.gpu
def test_serving_in_integers(block):
    block.eval()
    x = torch.randn(2, C, 33, 28, device="cuda")
    gate = torch.randn(2, C, 1, 1, device="cuda")
    with torch.no_grad():
        full = block(x, gate)
        for layers in (block.up, block.down):
            for i, c in enumerate(layers):
                layers[i] = Int8Pointwise(c)
        out = block(x, gate)

        class Plain(nn.Module):
            def __init__(self, q):
                super().__init__()
                self.q = q

            def forward(self, v):
                v = v.permute(0, 2, 3, 1).double()
                top = v.abs().amax(-1, keepdim=True)
                t = torch.round(127 * v / top) * (top / 127)
                w = self.q.weight_rows[:, :self.q.in_channels].double() * self.q.weight_scale.double()[:, None]
                return (t @ w.t() + self.q.bias.double()).permute(0, 3, 1, 2).float().contiguous()

        graph = torch.cuda.CUDAGraph()
        static = x.clone()
        with torch.cuda.graph(graph):
            served = block(static, gate)
        static.zero_()
        static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(served, out)
        for layers in (block.up, block.down):
            for i, c in enumerate(layers):
                layers[i] = Plain(c)
        want = block.plain(x, gate)
        # A value next to a border may take the other integer after sums in another order, which moves a token by a step of 1/127 of its
        # largest value in one channel of 96: rare, so the norms agree far below that
        assert float((out - want).norm() / want.norm()) <= 1e-3
        # eight bits: every operand of four layers is off by at most half of 1/127 of its largest
        assert float((out - full).norm() / full.norm()) <= 0.05


@pytest.mark.gpu
@pytest.mark.parametrize("which", [("conv1", 1), ("conv1", 5), ("conv2", 1), ("conv2", 3), None], ids=str)
@pytest.mark.parametrize("alphas", [False, True])
def test_integer_layers_in_the_64_channel_block(which, alphas):
    """The framework's own blocks with one or all of their 1x1 layers replaced: every layer is called, as in a block of another width."""
    from conversenet_b200 import ConverseBlock, ConverseBlockAlphaVariant
    torch.manual_seed(0)
    m = (ConverseBlockAlphaVariant if alphas else ConverseBlock)(64, 64, 3, padding=2).cuda().eval()
    if alphas:
        with torch.no_grad():
            m.alpha1.normal_(), m.alpha2.normal_()
    x = torch.randn(2, 64, 24, 20, device="cuda")
    with torch.no_grad():
        full = m(x)
    for name, i in [which] if which else [("conv1", 1), ("conv1", 5), ("conv2", 1), ("conv2", 3)]:
        getattr(m, name)[i] = Int8Pointwise(getattr(m, name)[i])

    def layers(v):
        a1, a2 = (m.alpha1, m.alpha2) if alphas else (1, 1)
        v = a1 * m._branch1(v) + v
        return a2 * m.conv2(v) + v

    from conversenet_b200.util_converse import _exact_fp32
    with torch.no_grad(), _exact_fp32():
        want = layers(x)
    with torch.no_grad():
        out = m(x)
        # eight bits: every operand of four layers is off by at most half of 1/127 of its largest
        assert torch.equal(out, want) and 0 < float((out - full).norm() / full.norm()) <= 0.05
    with pytest.raises(RuntimeError, match="inference"):
        m(x)
    for p in m.parameters():
        p.requires_grad_(False)
    assert torch.equal(m(x), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [None, torch.bfloat16])
def test_integer_layers_in_the_denoiser(dtype):
    from conversenet_b200 import ConverseBlock
    from conversenet_b200.models import ConverseDnCNN
    torch.manual_seed(0)
    net = ConverseDnCNN().cuda().eval()
    net.activation_dtype = dtype
    x = torch.rand(1, 1, 24, 28, device="cuda")
    with torch.no_grad():
        for m in net.modules():
            if isinstance(m, ConverseBlock):
                for seq in (m.conv1, m.conv2):
                    for i, layer in enumerate(seq):
                        if isinstance(layer, nn.Conv2d):
                            seq[i] = Int8Pointwise(layer)
        out = net(x)
        assert out.shape == x.shape and bool(torch.isfinite(out).all())
        assert torch.equal(out, net(x))


def test_which_layers_the_block_kernels_read():
    from conversenet_b200 import ConverseBlock

    class Shared(nn.Module):                       # a layer of someone's own around a convolution's weights
        def __init__(self, conv):
            super().__init__()
            self.weight, self.bias, self.out_channels = conv.weight, conv.bias, conv.out_channels

    m = ConverseBlock(64, 64)

    def plain():
        return m._plain_layers(m.conv1._modules, m.conv2._modules)

    assert plain()
    m.conv1[5] = Shared(m.conv1[5])
    assert plain()
    for seq, i in ((m.conv1, 1), (m.conv2, 3)):
        kept, seq[i] = seq[i], nn.Identity()
        assert not plain()
        seq[i] = kept
