"""CPU-side checks of the operators around a layer: dense formulas, refusals, argument checks of the C ABI."""
import ctypes

import pytest
import torch

import torchsplinekan_b200 as sk
from torchsplinekan_b200 import _native


def test_dense_formulas_and_their_derivatives():
    torch.manual_seed(0)
    t = lambda *s: torch.randn(*s, dtype=torch.float64, requires_grad=True)
    x, y, gate, w, b, s = t(2, 3, 5), t(2, 3, 5), t(2, 1, 5), t(5), t(5), t(5)
    for kind in ("rms", "layer"):
        f = lambda x, w, b: sk.block_norm(x, w, b, kind=kind)
        assert torch.autograd.gradcheck(f, (x, w, b)) and torch.autograd.gradgradcheck(f, (x, w, b))
        f = lambda x, y, g, s, w, b: sk.gated_residual(x, y, gate=g, gate_activation="silu", scale=s, post_norm=kind,
                                                       post_weight=w, next_norm="layer", next_bias=b)
        assert torch.autograd.gradcheck(f, (x, y, gate, s, w, b))
    assert torch.allclose(sk.block_norm(x, w, b, kind="layer", eps=1e-5), torch.nn.functional.layer_norm(x, (5,), w, b, 1e-5))
    out = sk.gated_residual(x.bfloat16(), y.float(), scale=s.float())
    assert out.dtype == torch.bfloat16 and torch.equal(out, (x.bfloat16().float() + y.float() * s.float()).bfloat16())
    packed = sk.gated_residual(x, torch.cat([y, y], -1), gate="packed", gate_activation="sigmoid")
    assert torch.allclose(packed, x + y * torch.sigmoid(y))


def test_refusals():
    x, y, w = torch.zeros(2, 3, 8), torch.zeros(2, 3, 8), torch.ones(8)
    for call, words in (
            (lambda: sk.block_norm(x, kind="batch"), "kind"),
            (lambda: sk.block_norm(x, kind=None), "kind"),
            (lambda: sk.block_norm(x, checkpoint="int4"), "checkpoint"),
            (lambda: sk.gated_residual(x, y, gate="both"), "packed"),
            (lambda: sk.gated_residual(x, y, gate=y, gate_activation="relu"), "gate_activation"),
            (lambda: sk.gated_residual(x, y, post_norm="batch"), "post_norm"),
            (lambda: sk.gated_residual(x, y, next_norm=["rms"]), "next_norm"),
            (lambda: sk.pack_activation(x, "int4"), "format"),
            (lambda: sk.pack_activation(x, None), "format")):
        with pytest.raises(ValueError, match=words):
            call()
    for call, words in (
            (lambda: sk.block_norm(x.long()), "float32, float64"),
            (lambda: sk.block_norm(torch.zeros(())), "at least one column"),
            (lambda: sk.block_norm(torch.zeros(3, 0)), "at least one column"),
            (lambda: sk.block_norm(x, torch.ones(7)), "weight must have shape"),
            (lambda: sk.block_norm(x, w.double()), "weight must be"),
            (lambda: sk.block_norm(x.half(), w.half()), "weight must be"),
            (lambda: sk.block_norm(x, eps=0.0), "eps"),
            (lambda: sk.block_norm(x, eps=float("nan")), "eps"),
            (lambda: sk.block_norm(x, eps=1e-45), "eps"),
            (lambda: sk.block_norm(x, checkpoint="int8"), "CUDA"),
            (lambda: sk.gated_residual(x, y[:, :2]), "y must have shape"),
            (lambda: sk.gated_residual(x, y.double()), "y must be"),
            (lambda: sk.gated_residual(x, y, gate="packed"), "side by side"),
            (lambda: sk.gated_residual(x, y, gate_activation="silu"), "needs a gate"),
            (lambda: sk.gated_residual(x, y, gate=y[:1]), "trailing row dimensions"),
            (lambda: sk.gated_residual(x, y, gate=y[..., :1]), "trailing row dimensions"),
            (lambda: sk.gated_residual(x, y, gate=y[0]), "trailing row dimensions"),
            (lambda: sk.gated_residual(x, y, post_weight=w), "post_norm"),
            (lambda: sk.gated_residual(x, y, next_bias=w), "next_norm"),
            (lambda: sk.gated_residual(x, y, checkpoint="e4m3"), "CUDA"),
            (lambda: sk.pack_activation(x), "CUDA"),
            (lambda: sk.unpack_activation(x.to(torch.int8), torch.zeros(2, 3, 1)), "CUDA"),
            (lambda: sk.unpack_activation(x.to(torch.int8), torch.zeros(2, 3, 2)), "scales must have shape"),
            (lambda: sk.unpack_activation(x.to(torch.int8), torch.zeros(2, 3, 1), torch.int32), "dtype")):
        with pytest.raises(RuntimeError, match=words):
            call()


def test_argument_structure_matches_the_header():
    """Field names and order of the ctypes structure are those of the C one, and so is its size (every field is an int, a
    double, an int64 or a pointer)."""
    import os
    import re
    from conftest import ROOT
    text = open(os.path.join(ROOT, "include", "kan_b200.h")).read()
    body = re.search(r"typedef struct kanb200_block_args \{(.*?)\} kanb200_block_args;", text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = []
    for decl in body.split(";"):
        names = re.sub(r"\b(const|void|int64_t|int|double)\b|\*", " ", decl)
        fields += [n.strip() for n in names.split(",") if n.strip()]
    assert fields == [n for n, _ in _native.BlockArgs._fields_]
    assert ctypes.sizeof(_native.BlockArgs) == 6 * 4 + 8 * (len(fields) - 6)


def test_c_abi_refuses_before_any_launch():
    lib, p = _native.lib(), 4096                   # never dereferenced: every call below is refused

    def args(**kw):
        base = dict(dtype=_native.F32, next_norm=_native.NORM_RMS, eps=1e-6, rows=4, width=8, x=p, x_stride=8, h=p)
        return _native.BlockArgs(**{**base, **kw})

    def refused(words, backward=False, **kw):
        a = args(**kw)
        rc = lib.kanb200_block_backward(ctypes.byref(a), None, 0, None) if backward else \
            lib.kanb200_block_forward(ctypes.byref(a), None)
        assert rc == _native.EINVAL and words in _native.last_error(), (rc, _native.last_error())

    refused("stream", dtype=9)
    refused("sizes", width=0)
    refused("sizes", rows=-1)
    refused("too large", rows=1 << 60)
    refused("eps", eps=0.0)
    refused("eps", eps=1e-40)
    refused("norm", next_norm=5)
    refused("activation", gate_act=7)
    refused("checkpoint", checkpoint=3)
    refused("negative", x_stride=-8)
    refused("x must", x=None)
    refused("h must", h=None)
    refused("out must", y=p, y_stride=8)
    refused("norm is needed", next_norm=0)
    refused("need y", scale=p)
    refused("its norm", y=p, out=p, post_weight=p)
    refused("multiple", y=p, out=p, gate=p, gate_rows=3)
    refused("per row", y=p, out=p, gate=p, gate_rows=2, gate_codes=p, gate_scales=p, checkpoint=1)
    refused("together", x_codes=p, checkpoint=1)
    refused("format", x_codes=p, x_scales=p)
    refused("aligned", next_stats=p + 4)
    refused("dout or dh", backward=True)
    refused("statistics", backward=True, dh=p)
    refused("need dh", backward=True, dout=p, has_branch=1, y=p, dnext_weight=p)
    refused("did not have", backward=True, dh=p, next_stats=p, dy=p, dy_stride=8)
    refused("codes must be given", backward=True, dout=p, has_branch=1)
    refused("post norm", backward=True, dout=p, has_branch=1, y=p, dpost_weight=p)
    refused("overlap", backward=True, dout=p, has_branch=1, y=p, dy=p, dy_stride=4)
    assert lib.kanb200_block_forward(None, None) == _native.EINVAL
    assert lib.kanb200_block_forward(ctypes.byref(args(rows=0)), None) == 0
    # a backward that needs scratch and gets none
    a = args(dh=p, dh_stride=8, next_stats=p, dx=p, dnext_weight=p, rows=400)
    need = lib.kanb200_block_backward_workspace_bytes(ctypes.byref(a))
    assert need > 0 and lib.kanb200_block_backward(ctypes.byref(a), None, 0, None) == _native.EWORKSPACE
    pk = lambda dtype=0, form=1, x=p, stride=8, rows=4, width=8: lib.kanb200_pack_activation(dtype, form, x, stride, p, p, rows,
                                                                                             width, None)
    assert pk(dtype=5) == pk(form=0) == pk(x=None) == pk(stride=-1) == pk(rows=-1) == pk(width=0) == _native.EINVAL
    assert pk(rows=0) == 0
    assert lib.kanb200_unpack_activation(0, 3, p, p, p, 4, 8, None) == _native.EINVAL


def test_networks_of_blocks_on_the_dense_backend():
    torch.manual_seed(1)
    net = sk.KAN([6, 8, 8, 2], norm="rms", residual=True, gate="silu", activation_checkpoint="int8").double()
    assert net.widths == [6, 8, 8, 2] and net.layers[1].out_features == 16
    x = torch.randn(5, 6, dtype=torch.float64, requires_grad=True)
    h = sk.block_norm(x, net.norms[0].weight)
    h = net.layers[0](h)
    y = net.layers[1](sk.block_norm(h, net.norms[1].weight))
    c = net.connections["1"]
    z = h + c.scale * torch.nn.functional.silu(y[:, 8:]) * sk.block_norm(y[:, :8].contiguous(), c.post_weight)
    want = net.layers[2](sk.block_norm(z, net.norms[2].weight))
    assert torch.allclose(net(x), want, atol=1e-12)
    assert torch.autograd.gradcheck(lambda t: net(t), (x,))
    frozen = net.export_inference()
    assert torch.allclose(frozen(x), net(x), atol=1e-10) and not any(p.requires_grad for p in frozen.parameters())
    y, reg = net.forward_with_regularization(x)
    assert torch.allclose(y, net(x)) and torch.allclose(reg, net.regularization_loss(x=x))
    plain = sk.KAN([6, 8, 2])
    assert sorted(k for k, _ in plain.named_parameters()) == sorted(k for k, _ in sk.KAN.from_layers(list(plain.layers)).named_parameters())
    state = plain.__getstate__()
    state.pop("norms"), state.pop("connections")
    old = sk.KAN.__new__(sk.KAN)
    old.__setstate__(state)                                   # pickled before the blocks existed
    assert torch.equal(old(x.detach().float()), plain(x.detach().float()))
    for bad, words in ((dict(norm="batch"), "norm"), (dict(gate="silu"), "residual"), (dict(gate="relu", residual=True), "gate"),
                       (dict(residual=True), "equal widths"), (dict(activation_checkpoint="int4"), "activation_checkpoint")):
        with pytest.raises(ValueError, match=words):
            sk.KAN([6, 8, 2], **bad)
    with pytest.raises(ValueError, match="share eps"):
        sk.GatedResidual(8)(torch.zeros(2, 8), torch.zeros(2, 8), sk.BlockNorm(8, eps=1e-3))
    with pytest.raises(ValueError, match="chains"):
        sk.KAN([4, 4, 4], residual=True).prune(torch.zeros(3, 4))


PARAMETERS = ("scale", "post_weight", "post_bias", "next_weight", "next_bias")


def block_call(width, dtype, backward, rows=700, **kw):
    """Arguments of a connection with everything, all pointers aligned (nothing here is launched)."""
    p = 1 << 20
    a = dict(dtype=dtype, post_norm=_native.NORM_LAYER, next_norm=_native.NORM_LAYER, eps=1e-6, rows=rows, width=width, x=p,
             x_stride=width, y=p, y_stride=width, gate=p, gate_stride=width, gate_rows=1, post_stats=p, next_stats=p,
             **{n: p for n in PARAMETERS})
    if backward:
        a.update(has_branch=1, dout=p, dout_stride=width, dh=p, dh_stride=width, dx=p, dy=p, dy_stride=width, dgate=p,
                 dgate_stride=width, **{"d" + n: p for n in PARAMETERS})
    else:
        a.update(out=p, h=p)
    return _native.BlockArgs(**{**a, **kw})


@pytest.mark.parametrize("dtype", [_native.F32, _native.F64, _native.F16, _native.BF16])
@pytest.mark.parametrize("width", [64, 1024, 8192])
@pytest.mark.parametrize("backward", [0, 1])
def test_parameters_of_any_alignment_are_not_read_16_bytes_at_a_time(dtype, width, backward):
    lib, element, p = _native.lib(), 8 if dtype == _native.F64 else 4, 1 << 20
    at_once = lambda **kw: lib.kanb200_block_columns_at_once(ctypes.byref(block_call(width, dtype, backward, **kw)), backward)
    assert at_once() == 4
    for name in PARAMETERS:
        assert at_once(**{name: p + element}) == 1, name
    assert at_once(rows=-1) == _native.EINVAL
    # parameters of a norm alone
    alone = dict(y=None, gate=None, scale=None, post_norm=0, post_weight=None, post_bias=None)
    if backward:
        alone.update(has_branch=0, dy=None, dgate=None, dscale=None, dpost_weight=None, dpost_bias=None)
    assert at_once(**alone) == 4 and at_once(**alone, next_weight=p + element) == 1


@pytest.mark.parametrize("dtype", [_native.F32, _native.F64, _native.F16, _native.BF16])
def test_column_sums_of_any_alignment_leave_through_a_slab(dtype):
    """A handful of rows runs in one block that stores the parameters' gradients itself, 16 bytes at a time; a result that
    such stores cannot reach goes through scratch and the kernel that adds slabs element by element."""
    lib, element, p = _native.lib(), 8 if dtype == _native.F64 else 4, 1 << 20
    need = lambda **kw: lib.kanb200_block_backward_workspace_bytes(ctypes.byref(block_call(1024, dtype, 1, rows=3, **kw)))
    assert need() == 0
    for name in PARAMETERS:
        assert need(**{"d" + name: p + element}) >= 1024 * element, name


def test_scratch_that_16_byte_stores_cannot_reach_is_refused():
    lib = _native.lib()
    a = block_call(1024, _native.F32, 1)
    need = lib.kanb200_block_backward_workspace_bytes(ctypes.byref(a))
    assert need > 0
    for off in (4, 8):
        assert lib.kanb200_block_backward(ctypes.byref(a), (1 << 20) + off, need, None) == _native.EINVAL
        assert "workspace" in _native.last_error()


@pytest.mark.parametrize("config", [dict(norm="rms"), dict(residual=True), dict(norm="layer", residual=True, gate="silu")])
def test_node_scores_of_networks_of_blocks_are_refused(config):
    """Walking the layers as a plain chain would score them on inputs that they never see."""
    from torchsplinekan_b200.pruning import node_scores
    with pytest.raises(ValueError, match="node_scores works on plain chains"):
        node_scores(sk.KAN([4, 4, 4], **config), torch.zeros(3, 4))
    incoming, outgoing = node_scores(sk.KAN([4, 4, 4]), torch.zeros(3, 4))
    assert len(incoming) == len(outgoing) == 1


def test_tensors_without_memory_are_refused_by_name():
    """Fake CUDA tensors need no device: the refusal comes before anything touches one."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, w = torch.empty(4, 8, device="cuda"), torch.ones(8, device="cuda", requires_grad=True)
        codes, scales = torch.empty(4, 8, dtype=torch.int8, device="cuda"), torch.empty(4, 1, device="cuda")
        for name, call in (("block_norm", lambda: sk.block_norm(x, w)),
                           ("gated_residual", lambda: sk.gated_residual(x, x, scale=w, next_norm="rms")),
                           ("pack_activation", lambda: sk.pack_activation(x)),
                           ("unpack_activation", lambda: sk.unpack_activation(codes, scales))):
            with pytest.raises(RuntimeError, match=name + ": fake tensors"):
                call()
        assert sk.block_norm(torch.empty(4, 8)).shape == (4, 8)          # the dense formulas trace
