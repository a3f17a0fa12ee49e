"""KAN layers and networks that use the operators around a layer: 8-bit input checkpoints, norms, gated residual
connections, all of them together in a training step."""
import pytest
import torch

import torchsplinekan_b200 as sk
from block_util import restored

pytestmark = pytest.mark.gpu


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def seeded(make, seed=0):
    torch.manual_seed(seed)
    net = make()
    with torch.no_grad():                    # parameters that start as ones and zeros get values of their own
        for name, p in net.named_parameters():
            if p.dim() == 1:
                p.add_(0.2 * torch.randn_like(p))
    return net


# ---- the layer's checkpoint ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,i,o,dtype", [(1, 7, 5, torch.float32), (37, 300, 20, torch.float32), (2048, 256, 128, torch.float32),
                                            (600, 33, 17, torch.float64)])
@pytest.mark.parametrize("form", ["int8", "e4m3"])
def test_layer_checkpoint(rows, i, o, dtype, form):
    """Same output bits; gradients bit for bit those of the plain layer at the restored input."""
    layer = seeded(lambda: sk.KANLinear(i, o, activation_checkpoint=form)).cuda().to(dtype)
    plain = seeded(lambda: sk.KANLinear(i, o)).cuda().to(dtype)
    plain.load_state_dict(layer.state_dict())
    x = (torch.rand(rows, i, device="cuda", dtype=dtype, generator=torch.Generator("cuda").manual_seed(1)) * 2.2 - 1.1)
    dy = torch.randn(rows, o, device="cuda", dtype=dtype)
    xc = x.clone().requires_grad_()
    y = layer(xc)
    assert torch.equal(y, plain(x))
    xr = sk.unpack_activation(*sk.pack_activation(x, form), dtype)
    # what is restored is codes * scales; the product is rounded to the layer's type
    assert rel(xr, restored(x, form)) <= 2.0 ** -23
    xr.requires_grad_()
    got = torch.autograd.grad(y, [xc, *layer.parameters()], dy)
    want = torch.autograd.grad(plain(xr), [xr, *plain.parameters()], dy)
    for g, w in zip(got, want):
        assert torch.equal(g, w)
    with torch.no_grad():
        assert torch.equal(layer(x), y)
    assert layer.make_like().activation_checkpoint == form


def test_layer_checkpoint_refuses_second_derivatives_and_the_regulariser_keeps_its_input():
    layer = sk.KANLinear(16, 8, activation_checkpoint="int8").cuda()
    plain = sk.KANLinear(16, 8).cuda()
    plain.load_state_dict(layer.state_dict())
    x = torch.rand(50, 16, device="cuda").requires_grad_()
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(layer(x).sum(), x, create_graph=True)
    grads = []
    for net in (layer, plain):
        y, reg = net.forward_with_regularization(x, 0.1, 0.1)
        grads.append(torch.autograd.grad(y.square().sum() + reg, [x, *net.parameters()]))
    for g, w in zip(*grads):
        assert torch.equal(g, w)
    layer.double()
    xd = x.detach().double().cpu().requires_grad_()
    layer.cpu()
    (g,) = torch.autograd.grad(layer(xd).sum(), xd, create_graph=True)       # the dense backend has no checkpoint
    assert g.requires_grad


def test_layer_checkpoint_saves_its_memory():
    """Between forward and backward a 1024-wide stack holds a quarter of its inputs."""
    x = torch.rand(8192, 1024, device="cuda") * 2 - 1
    held = {}
    for form in (None, "int8"):
        net = sk.KAN([1024] * 4, activation_checkpoint=form).cuda()
        with torch.no_grad():
            net(x)                                                    # workspaces
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        y = net(x)
        torch.cuda.synchronize()
        held[form] = torch.cuda.memory_allocated() - base
        del y, net
    n = 8192 * 1024
    # the outputs of the first two layers are kept (the first input is the caller's), and the result is
    assert held[None] >= 3 * 4 * n
    assert held["int8"] <= 4 * n + 3 * (n + n // 32) + (1 << 20)


def test_layer_checkpoint_and_gradient_sink():
    layer = seeded(lambda: sk.KANLinear(64, 300, activation_checkpoint="int8", backend="cuda")).cuda()
    plain = seeded(lambda: sk.KANLinear(64, 300, activation_checkpoint="int8", backend="cuda")).cuda()
    plain.load_state_dict(layer.state_dict())
    x = torch.rand(30000, 64, device="cuda") * 2 - 1
    bucket = sk.GradientBucket([layer], direct=True)
    try:
        bucket.zero_grad()
        layer(x).square().sum().backward()
        bucket.finish()
        plain(x).square().sum().backward()
        for (n, p), q in zip(layer.named_parameters(), plain.parameters()):
            assert rel(p.grad, q.grad) < 1e-6, n
    finally:
        bucket.remove()


def test_network_of_blocks_and_gradient_buckets():
    """Buckets over a whole network: the layers' gradients from their sinks, those of norms and connections from autograd."""
    make = lambda: seeded(lambda: sk.KAN([64, 128, 128, 128], norm="layer", residual=True, gate="silu", activation_checkpoint="int8",
                                         backend="cuda")).cuda()
    net, plain = make(), make()
    plain.load_state_dict(net.state_dict())
    x = torch.randn(30000, 64, device="cuda")
    bucket = sk.GradientBucket(net, direct=True)
    try:
        assert len(bucket.buckets) == len(net.parameter_modules()) == 8 and len(bucket._sinks) == 3
        for _ in range(2):
            bucket.zero_grad()
            net(x).square().mean().backward()
            bucket.finish()
        plain(x).square().mean().backward()
        held = {b.data_ptr(): b.data_ptr() + 4 * b.numel() for b in bucket.buckets}
        for (n, p), q in zip(net.named_parameters(), plain.parameters()):
            assert rel(p.grad, q.grad) < 1e-6, n
            assert any(lo <= p.grad.data_ptr() < hi for lo, hi in held.items()), n
    finally:
        bucket.remove()


# ---- networks of blocks --------------------------------------------------------------------------------------------------
CONFIGS = [dict(norm="rms"), dict(norm="layer", residual=True), dict(norm="rms", residual=True, gate="silu", scale_init=0.3),
           dict(residual=True), dict(norm="layer", residual=True, gate="sigmoid")]


@pytest.mark.parametrize("config", CONFIGS)
@pytest.mark.parametrize("widths", [[12, 24, 24, 24, 5], [130, 130, 130]])
def test_network_matches_its_dense_form(config, widths):
    """Forward, regulariser and all gradients against the float64 network on the CPU, which runs the dense formulas.  Each
    of the layers' kernels is good to 1e-5 of its largest result; the values pass through four of them, and their
    gradients through four more."""
    net = seeded(lambda: sk.KAN(widths, **config)).cuda()
    ref = seeded(lambda: sk.KAN(widths, **config)).double()
    ref.load_state_dict({k: v.double().cpu() for k, v in net.state_dict().items()})
    x = torch.randn(60, widths[0], device="cuda")
    y, reg = net.forward_with_regularization(x, 0.3, 0.1)
    yr, regr = ref.forward_with_regularization(x.double().cpu(), 0.3, 0.1)
    assert rel(net(x), ref(x.double().cpu()).cuda()) < 4e-5 and rel(y, yr.cuda()) < 4e-5 and abs(float(reg) / float(regr) - 1) < 1e-4
    got = torch.autograd.grad(net(x).square().sum(), list(net.parameters()))
    want = torch.autograd.grad(ref(x.double().cpu()).square().sum(), list(ref.parameters()))
    for (n, _), g, w in zip(net.named_parameters(), got, want):
        assert rel(g, w.cuda()) < 8e-5, n
    assert net.widths == widths


@pytest.mark.parametrize("form", ["int8", "e4m3"])
def test_network_with_checkpoints(form):
    """One training step of everything together.  The output does not depend on the checkpoints; a restored tensor is off
    by about 0.8 % (int8, groups whose largest value is 3.5 times their rms: step / sqrt(12)) or 2.6 % (e4m3: half a step
    of 2^-3, uniform) of its rms, and each of the 3 blocks restores four of them."""
    make = lambda f: seeded(lambda: sk.KAN([96, 200, 200, 200, 200, 10], norm="rms", residual=True, gate="silu", scale_init=0.5,
                                           activation_checkpoint=f)).cuda()
    net, plain = make(form), make(None)
    plain.load_state_dict(net.state_dict())
    x = torch.randn(700, 96, device="cuda")
    y = net(x)
    assert torch.equal(y, plain(x))
    got = torch.autograd.grad(y.square().sum(), list(net.parameters()))
    want = torch.autograd.grad(plain(x).square().sum(), list(plain.parameters()))
    bound = (0.008 if form == "int8" else 0.026) * 12 ** 0.5 * 2
    for (n, _), g, w in zip(net.named_parameters(), got, want):
        assert rel(g, w) < bound, n
    for n, p in zip(got, want):
        assert bool(torch.isfinite(n).all())


def test_half_precision_stream():
    """A bfloat16 stream through a residual stack: the layers compute in float32, the stream stays bfloat16."""
    net = seeded(lambda: sk.KAN([64, 64, 64], norm="rms", residual=True, gate="silu", activation_checkpoint="int8")).cuda()
    x = torch.randn(30, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = net(x)
    assert y.dtype == torch.bfloat16
    y.float().square().sum().backward()
    assert x.grad.dtype == torch.bfloat16 and bool(torch.isfinite(x.grad.float()).all())
    assert rel(y, net(x.detach().float())) < 2.0 ** -7             # one rounding per block, two blocks


def test_network_in_a_captured_step():
    net = seeded(lambda: sk.KAN([64, 128, 128, 128, 8], norm="rms", residual=True, gate="silu", activation_checkpoint="int8")).cuda()
    x = torch.randn(512, 64, device="cuda")

    def step():
        for p in net.parameters():
            p.grad = None
        loss = net(x).square().mean()
        loss.backward()
        return loss
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(); step()
    torch.cuda.current_stream().wait_stream(side)
    for p in net.parameters():
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()
    captured = [p.grad for p in net.parameters()]
    for seed in (3, 4):
        x.copy_(torch.randn(512, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)))
        graph.replay()
        got = [float(loss)] + [g.clone() for g in captured]
        want = [float(step())] + [p.grad.clone() for p in net.parameters()]
        assert got[0] == pytest.approx(want[0], rel=1e-6)
        for g, w in zip(got[1:], want[1:]):
            assert rel(g, w) < 1e-6


def test_export_extend_and_update_keep_the_blocks():
    net = seeded(lambda: sk.KAN([20, 40, 40, 3], norm="layer", residual=True, gate="sigmoid")).cuda()
    x = torch.randn(400, 20, device="cuda")
    frozen = net.export_inference()
    assert not any(p.requires_grad for p in frozen.parameters()) and rel(frozen(x), net(x)) < 1e-5
    assert rel(frozen(x[:1]), net(x[:1])) < 1e-5
    net.update_grid(x)
    finer = net.extend_grid(9, x)
    assert finer.widths == net.widths == [20, 40, 40, 3] and finer.layers[0].grid_size == 9
    assert rel(finer(x), net(x)) < 0.05          # a refit of the splines on the samples, not the same function
    with pytest.raises(ValueError, match="chains"):
        net.prune(x)
