"""The norm in front of a layer, the gated residual connection behind it and 8-bit checkpoints, against plain float64
forms with tolerances that count roundings (block_util)."""
import itertools

import pytest
import torch

import torchsplinekan_b200 as sk
from block_util import (DTYPES, ROUNDOFF, activation, assert_close, branch_type, norm, norm_backward, pack, restored)

pytestmark = pytest.mark.gpu

EPS = 1e-6
# one token to many rows; widths below, at and beyond a warp's 128 columns, every tile of the kernels, and beyond them
SIZES = [(1, 1), (1, 1024), (3, 5), (2, 31), (9, 64), (70, 127), (5, 128), (4, 129), (700, 16), (33, 260), (20, 1000), (6, 1001),
         (3, 2048), (2, 4099), (3, 8192), (2, 16384), (2, 20004), (1, 33001)]


def randn(*shape, dtype=torch.float64, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", dtype=torch.float64, generator=g).to(dtype)


def stream(rows, width, dtype, seed=1):
    """Rows of different sizes, an offset and a few loud columns."""
    x = randn(*(rows if isinstance(rows, tuple) else (rows,)), width, seed=seed)
    x = x * torch.where(torch.arange(width, device="cuda") % 37 == 3, 8.0, 1.0) + 0.3
    return x.to(dtype)


def d64(t):
    return None if t is None else t.detach().double()


# ---- norm ------------------------------------------------------------------------------------------------------------
def check_norm(x, w, b, kind, form, dh, rows_extra=0):
    """Forward and all gradients of one call."""
    dtype = x.dtype
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    h = sk.block_norm(*leaves, kind=kind, eps=EPS, checkpoint=form)
    assert h.dtype == branch_type(dtype) and h.is_contiguous()
    width = x.shape[-1]
    value, _, _, _ = norm(d64(x), d64(w), d64(b), kind, EPS)
    assert_close(h, value, dtype, width, what="h")
    with torch.no_grad():
        assert torch.equal(sk.block_norm(x, w, b, kind=kind, eps=EPS), h)          # no gradient wanted: same bits
    grads = torch.autograd.grad(h, [t for t in leaves if t is not None], dh)
    _, (vhat, vmag), r, rmag = norm(d64(x), None, None, kind, EPS, at=restored(x, form))
    want = norm_backward(vhat, vmag, r, rmag, d64(w), d64(dh), d64(dh).abs(), kind)
    for name, got, ref in zip([n for n, t in zip(("dx", "dw", "db"), leaves) if t is not None], grads,
                              [v for v, t in zip(want, leaves) if t is not None]):
        # a column sum adds up to all rows in a chain on top
        extra = rows_extra if name == "dx" else x.numel() // width
        assert_close(got, ref, dtype, width, extra, what=name)


@pytest.mark.parametrize("rows,width", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_sizes(rows, width, dtype):
    bt = branch_type(dtype)
    for kind, form in (("rms", None), ("layer", "int8")):
        check_norm(stream(rows, width, dtype), 1 + randn(width, dtype=bt, seed=2) * 0.2,
                   randn(width, dtype=bt, seed=3) if kind == "layer" else None, kind, form,
                   randn(rows, width, dtype=bt, seed=4))


@pytest.mark.parametrize("kind,has_w,has_b,form", list(itertools.product(["rms", "layer"], [True, False], [True, False],
                                                                         [None, "int8", "e4m3"])))
def test_norm_options(kind, has_w, has_b, form):
    for dtype in (torch.float32, torch.bfloat16):
        check_norm(stream((3, 4), 300, dtype), randn(300, dtype=torch.float32, seed=2) if has_w else None,
                   randn(300, dtype=torch.float32, seed=3) if has_b else None, kind, form,
                   randn(3, 4, 300, dtype=torch.float32, seed=4))


# ---- gated residual --------------------------------------------------------------------------------------------------
def gated_oracle(c, out, dout, dh):
    """(value, magnitude) of every output of one call; ``out``: what the kernel stored (its norm is taken of that)."""
    x, y, gate, scale, pw, pb, nw, nb = (d64(c[k]) for k in ("x", "y", "gate", "scale", "pw", "pb", "nw", "nb"))
    width = x.shape[-1]
    if c["packed"]:
        y, gate = y[..., :width], y[..., width:]
    one = torch.ones_like(x)
    form = c["form"]

    def branch(y_at, gate_at):
        if c["post"]:
            (z, zmag), (yhat, ymag), r, rmag = norm(y, pw, pb, c["post"], EPS, at=y_at)
        else:
            (z, zmag), (yhat, ymag), r, rmag = (y_at, y_at.abs()), (y_at, y_at.abs()), one, one
        a, amag, da, damag = activation(gate_at, c["act"]) if gate is not None else (one, one, one, one)
        return z, zmag, yhat, ymag, r, rmag, a, amag, da, damag

    s = scale if scale is not None else torch.ones(width, dtype=torch.float64, device="cuda")
    z, zmag, *_, a, amag, _, _ = branch(y, gate)
    res = {"out": (x + s * a * z, x.abs() + s.abs() * amag * zmag)}
    stored = d64(out)
    g, gmag = (d64(dout), d64(dout).abs()) if dout is not None else (torch.zeros_like(x), torch.zeros_like(x))
    if c["next"]:
        res["h"], (_, _), _, _ = norm(stored, nw, nb, c["next"], EPS)
        if dh is not None:
            _, (ohat, omag), r, rmag = norm(stored, None, None, c["next"], EPS, at=restored(out, form))
            (dv, dvmag), res["dnw"], res["dnb"] = norm_backward(ohat, omag, r, rmag, nw, d64(dh), d64(dh).abs(), c["next"])
            g, gmag = g + dv, gmag + dvmag
    res["dx"] = (g, gmag)
    keep = lambda t, full: restored(t, form).reshape(full.shape) if form else full
    per_row = gate is not None and gate.shape == x.shape
    y32 = c["y"][..., :width] if c["packed"] else c["y"]
    g32 = c["y"][..., width:] if c["packed"] else c["gate"]
    z, zmag, yhat, ymag, r, rmag, a, amag, da, damag = branch(keep(y32, y), keep(g32, gate) if per_row else gate)
    rows = lambda t: t.reshape(-1, width).sum(0)
    res["dscale"] = (rows(g * a * z), rows(gmag * amag * zmag))
    if gate is not None:
        dgate, dgmag = g * s * da * z, gmag * s.abs() * damag * zmag
        if gate.dim() == 1:
            res["dgate"] = (rows(dgate), rows(dgmag))
        else:
            res["dgate"] = (dgate.sum_to_size(gate.shape), dgmag.sum_to_size(gate.shape))
    dz, dzmag = g * s * a, gmag * s.abs() * amag
    if c["post"]:
        res["dy"], res["dpw"], res["dpb"] = norm_backward(yhat, ymag, r, rmag, pw, dz, dzmag, c["post"])
    else:
        res["dy"] = (dz, dzmag)
    if c["packed"]:
        res["dy"] = tuple(torch.cat([p, q], -1) for p, q in zip(res["dy"], res.pop("dgate")))
    return res


def make_gated(lead, width, dtype, gate="row", act="silu", scale=True, post="rms", next="rms", form=None, bias=True, seed=10):
    lead = lead if isinstance(lead, tuple) else (lead,)
    bt = branch_type(dtype)
    shared = {"sequence": lead[:1] + (1,) * (len(lead) - 1) + (width,), "all": (width,), "row": lead + (width,)}
    c = dict(packed=gate == "packed", act=act if gate else None, post=post, next=next, form=form,
             x=stream(lead, width, dtype, seed),
             y=randn(*lead, 2 * width if gate == "packed" else width, dtype=bt, seed=seed + 1),
             gate=randn(*shared[gate], dtype=bt, seed=seed + 2) if gate in shared else None,
             scale=randn(width, dtype=bt, seed=seed + 3) if scale else None,
             pw=1 + randn(width, dtype=bt, seed=seed + 4) if post else None,
             pb=randn(width, dtype=bt, seed=seed + 5) if post == "layer" and bias else None,
             nw=1 + randn(width, dtype=bt, seed=seed + 6) if next else None,
             nb=randn(width, dtype=bt, seed=seed + 7) if next == "layer" and bias else None)
    return c


LEAVES = (("x", "dx"), ("y", "dy"), ("gate", "dgate"), ("scale", "dscale"), ("pw", "dpw"), ("pb", "dpb"), ("nw", "dnw"),
          ("nb", "dnb"))


def call_gated(c):
    return sk.gated_residual(c["x"], c["y"], gate="packed" if c["packed"] else c["gate"], gate_activation=c["act"],
                             scale=c["scale"], post_norm=c["post"], post_weight=c["pw"], post_bias=c["pb"],
                             next_norm=c["next"], next_weight=c["nw"], next_bias=c["nb"], eps=EPS, checkpoint=c["form"])


def check_gated(c, use_out=True, use_h=True, only=None):
    dtype, shape = c["x"].dtype, c["x"].shape
    width = shape[-1]
    names = [n for n, _ in LEAVES if c[n] is not None and (only is None or n in only)]
    live = dict(c)
    for n in names:
        live[n] = c[n].detach().requires_grad_()
    got = call_gated(live)
    outs = got if isinstance(got, tuple) else (got,)
    with torch.no_grad():
        again = call_gated(c)
    for p, q in zip(outs, again if isinstance(again, tuple) else (again,)):
        assert torch.equal(p, q)
    dout = randn(*shape, seed=31).to(dtype) if use_out else None
    dh = randn(*shape, dtype=branch_type(dtype), seed=32) if c["next"] and use_h else None
    pairs = [(o, d) for o, d in zip(outs, (dout, dh)) if d is not None]
    grads = torch.autograd.grad([o for o, _ in pairs], [live[n] for n in names], [d for _, d in pairs], allow_unused=True)
    want = gated_oracle(c, outs[0], dout, dh)
    assert_close(outs[0], want["out"], dtype, width, what="out")
    if c["next"]:
        assert_close(outs[1], want["h"], dtype, width, what="h")
    total = c["x"].numel() // width
    for n, g in zip(names, grads):
        key = dict(LEAVES)[n]
        if n in ("nw", "nb") and dh is None:
            assert g is None
            continue
        summed = n not in ("x", "y") and not (n == "gate" and c["gate"].shape == shape)
        # the gradient of a row's stream carries the roundings of two norms
        assert_close(g, want[key], dtype, width, (total if summed else 0) + 64, what=key)
    return outs, dict(zip(names, grads))


@pytest.mark.parametrize("rows,width", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_sizes(rows, width, dtype):
    check_gated(make_gated(rows, width, dtype))
    check_gated(make_gated(rows, width, dtype, gate="packed", act="sigmoid", post="layer", next="layer", form="int8"))


@pytest.mark.parametrize("gate,post,next,form", list(itertools.product(["row", "sequence", "all", "packed", None],
                                                                       [None, "rms", "layer"], [None, "rms", "layer"],
                                                                       [None, "e4m3"])))
def test_gated_options(gate, post, next, form):
    act = {"row": "sigmoid", "sequence": None, "all": "silu", "packed": "silu", None: None}[gate]
    for dtype, scale in ((torch.float32, True), (torch.bfloat16, False)):
        check_gated(make_gated((3, 5), 132, dtype, gate, act, scale, post, next, form))


@pytest.mark.parametrize("rows,width,dtype", [(9, 5, torch.float32), (3, 40, torch.float64), (5, 270, torch.float32),
                                              (5, 592, torch.bfloat16), (3, 2060, torch.float32), (2, 8195, torch.float32)])
@pytest.mark.parametrize("absent", [("scale", "pw", "pb", "nw", "nb"), ("scale", "pw"), ("scale",), ("pw",), ("pb", "nb"), ("nw",)])
def test_absent_parameters(rows, width, dtype, absent):
    """Widths that leave threads without a column, and the parameters whose place a constant takes."""
    for post, next, gate in itertools.product(["rms", "layer"], ["rms", "layer"], ["row", None, "all"]):
        c = make_gated(rows, width, dtype, gate, post=post, next=next)
        c.update((name, None) for name in absent)
        check_gated(c)


@pytest.mark.parametrize("lead,width,gate", [((1, 1), 64, "sequence"), ((1, 2000), 40, "sequence"), ((7, 311), 96, "sequence"),
                                             ((1500, 2), 33, "sequence"), ((2, 3, 70), 260, "sequence"), ((2500,), 24, "all"),
                                             ((2, 900), 1030, "all"), ((3, 1), 48, "sequence"), ((400, 5), 1, "sequence"),
                                             ((2, 3), 33001, "sequence"), ((2, 45), 9000, "sequence"), ((3, 200), 2052, "all")])
def test_shared_gate_gradients(lead, width, gate):
    for act in (None, "silu"):
        check_gated(make_gated(lead, width, torch.float32, gate, act, form="int8"))


@pytest.mark.parametrize("rows,width,dtype", [(3001, 64, torch.float32), (5000, 200, torch.float64), (4097, 1024, torch.bfloat16),
                                              (2999, 777, torch.float32), (1300, 2052, torch.float32)])
def test_many_rows(rows, width, dtype):
    bt = branch_type(dtype)
    check_norm(stream(rows, width, dtype), randn(width, dtype=bt, seed=2), randn(width, dtype=bt, seed=3), "layer", None,
               randn(rows, width, dtype=bt, seed=4))
    check_gated(make_gated(rows, width, dtype))


@pytest.mark.parametrize("rows,width", [(60000, 24), (40000, 60), (20000, 132), (5000, 1030), (1200, 4100)])
@pytest.mark.parametrize("form", ["int8", "e4m3"])
def test_many_rows_without_a_sum_over_the_row(rows, width, form):
    """Scales and statistics that one lane brings for all, row after row, where nothing else keeps the lanes together: no
    post norm behind its codes, or one whose input needs no gradient.  Gradients per row, so a scale of another row shows."""
    for gate in ("row", "packed"):
        check_gated(make_gated(rows, width, torch.float32, gate, post=None, next=None, form=form))
    check_gated(make_gated(rows, width, torch.bfloat16, "row", post="layer", next=None, form=form), only=("x", "gate", "scale"))
    check_gated(make_gated(rows, width, torch.float32, "row", post="rms", next="rms", form=form), only=("gate",))


@pytest.mark.parametrize("rows,width", [(1, 8), (7, 64), (4097, 20), (5000, 333), (3001, 1024), (1001, 5000), (37, 33001)])
def test_sums_over_rows_hold_every_row_once(rows, width):
    """Sums of small whole numbers have no rounding, in whatever order they are formed: a row that is left out or counted twice
    shows, however many there are."""
    whole = lambda *shape, seed: torch.randint(-8, 9, shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).float()
    x, y, dout = whole(rows, width, seed=1), whole(rows, width, seed=2), whole(rows, width, seed=3)
    scale, gate = whole(width, seed=4).requires_grad_(), whole(width, seed=5).requires_grad_()
    for g, factor in ((None, 1.0), (gate, gate.detach())):
        out = sk.gated_residual(x, y, gate=g, scale=scale)
        got = torch.autograd.grad(out, [scale] if g is None else [scale, gate], dout)
        assert torch.equal(got[0], (dout.double() * y.double()).sum(0).float() * factor)
        if g is not None:
            assert torch.equal(got[1], (dout.double() * y.double()).sum(0).float() * scale.detach())
    b = torch.zeros(width, device="cuda", requires_grad=True)
    (got,) = torch.autograd.grad(sk.block_norm(x, None, b, kind="layer"), b, dout)
    assert torch.equal(got, dout.sum(0))
    out = sk.gated_residual(x, y, post_norm="rms", post_bias=b)
    (got,) = torch.autograd.grad(out, b, dout)
    assert torch.equal(got, dout.sum(0))
    for batch in (d for d in (3, 7, 11) if rows % d == 0):
        per = whole(batch, 1, width, seed=6).requires_grad_()
        view = lambda t: t.view(batch, -1, width)
        (got,) = torch.autograd.grad(sk.gated_residual(view(x), view(y), gate=per), per, view(dout))
        assert torch.equal(got, view(dout * y).sum(1, keepdim=True))


def test_only_one_result_used():
    c = make_gated(40, 200, torch.float32)
    check_gated(c, use_h=False)
    check_gated(c, use_out=False)
    c["form"] = "int8"
    check_gated(c, use_h=False)
    check_gated(c, use_out=False)


@pytest.mark.parametrize("only", [("x",), ("y",), ("gate",), ("scale",), ("pw",), ("nb",), ("y", "nw"), ("x", "pb")])
def test_some_gradients_only(only):
    check_gated(make_gated(30, 140, torch.float32, post="layer", next="layer"), only=only)
    check_gated(make_gated((4, 30), 140, torch.float32, "sequence", post="layer", next="layer"), only=only)


def test_same_bits_on_every_run():
    c = make_gated((6, 700), 516, torch.float32, "sequence")
    first = check_gated(c)
    second = check_gated(c)
    for p, q in zip(first[0], second[0]):
        assert torch.equal(p, q)
    for n in first[1]:
        assert torch.equal(first[1][n], second[1][n]), n


# ---- layouts -----------------------------------------------------------------------------------------------------------
def strided(t, how):
    """The same values with other strides or another alignment."""
    if how == "rows":                             # rows further apart than their width, start off by one element
        wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 7, dtype=t.dtype, device=t.device)
        wide[..., 1:1 + t.shape[-1]] = t
        return wide[..., 1:1 + t.shape[-1]]
    if how == "columns":                          # columns apart
        return t.transpose(0, -1).contiguous().transpose(0, -1)
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)      # dense but not aligned
    flat[1:] = t.reshape(-1)
    return flat[1:].view(t.shape)


@pytest.mark.parametrize("how", ["rows", "columns", "shifted"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(how, dtype):
    for width in (64, 256, 1001):
        x = stream(12, width, dtype)
        w, dh = randn(width, dtype=torch.float32, seed=2), randn(12, width, dtype=torch.float32, seed=4)
        check_norm(strided(x, how), w, None, "rms", None, strided(dh, how))
        check_norm(strided(x, how), w, None, "layer", "int8", strided(dh, how))
        c = make_gated((3, 4), width, dtype, "row")
        for n in ("x", "y", "gate"):
            c[n] = strided(c[n], how)
        check_gated(c)
        c = make_gated((3, 4), width, dtype, "packed", form="e4m3")
        c["y"] = strided(c["y"], how)
        check_gated(c)
        codes, scales = sk.pack_activation(strided(x, how))
        want = sk.pack_activation(x)
        assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [64, 1024, 8192])
def test_parameters_that_are_views_into_a_flat_buffer(width, dtype):
    """Every parameter one element behind a 16-byte boundary, each alone and all of them, forward and backward."""
    bt = branch_type(dtype)
    w, b, dh = randn(width, dtype=bt, seed=2), randn(width, dtype=bt, seed=3), randn(9, width, dtype=bt, seed=4)
    for shifted in (("w",), ("b",), ("w", "b")):
        check_norm(stream(9, width, dtype), strided(w, "shifted") if "w" in shifted else w,
                   strided(b, "shifted") if "b" in shifted else b, "layer", "int8" if width == 64 else None, dh)
    names = ("scale", "pw", "pb", "nw", "nb")
    for gate, shifted in (("row", names), ("sequence", names), *((None, (n,)) for n in names)):
        c = make_gated((3, 4), width, dtype, gate, None if gate is None else "silu", post="layer", next="layer")
        for n in shifted:
            c[n] = strided(c[n], "shifted")
            assert c[n].is_contiguous() and c[n].data_ptr() % 16 != 0
        check_gated(c)


def test_column_sums_at_any_address():
    """The C entry point with parameter gradients that 16-byte stores cannot reach, from one block and from many."""
    import ctypes
    from torchsplinekan_b200 import _native
    for rows, width in ((3, 64), (900, 64), (3, 1024), (700, 1024)):
        x, w = stream(rows, width, torch.float32), randn(width, dtype=torch.float32, seed=2)
        dh = randn(rows, width, dtype=torch.float32, seed=4)
        leaves = [w.clone().requires_grad_(), torch.zeros(width, device="cuda", requires_grad=True)]
        want = torch.autograd.grad(sk.block_norm(x, *leaves, kind="layer", eps=EPS), leaves, dh)
        h, stats = torch.empty_like(x), torch.empty(rows, 2, device="cuda")
        flat = torch.full((2, width + 2), float("nan"), device="cuda")
        a = _native.BlockArgs(dtype=_native.F32, next_norm=_native.NORM_LAYER, eps=EPS, rows=rows, width=width,
                              x=x.data_ptr(), x_stride=width, next_weight=w.data_ptr(), next_stats=stats.data_ptr(),
                              h=h.data_ptr(), dh=dh.data_ptr(), dh_stride=width, dnext_weight=flat.data_ptr() + 4,
                              dnext_bias=flat.data_ptr() + 4 * (width + 3))
        lib, st = _native.lib(), torch.cuda.current_stream().cuda_stream
        assert lib.kanb200_block_forward(ctypes.byref(a), st) == 0
        need = lib.kanb200_block_backward_workspace_bytes(ctypes.byref(a))
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        assert need > 0 and lib.kanb200_block_backward(ctypes.byref(a), ws.data_ptr(), need, st) == 0
        for row, v in zip(flat, want):
            assert torch.equal(row[1:-1], v) and bool(torch.isnan(row[[0, -1]]).all())


def test_views_that_negate_lazily():
    """The imaginary part of a conjugate negates when it is read; its memory holds the other sign."""
    z = torch.complex(randn(40, 1, dtype=torch.float32), randn(40, 1, dtype=torch.float32, seed=1))
    lazy, w = z.conj().imag, torch.full((1,), 2.0, device="cuda")
    assert lazy.is_neg()
    plain = lazy.clone()
    minus = lambda t: torch._neg_view(-t)
    x, v = randn(9, 64, dtype=torch.float32, seed=2), randn(64, dtype=torch.float32, seed=3)
    for got, want in ((sk.block_norm(lazy, w), sk.block_norm(plain, w)),
                      (sk.gated_residual(lazy, lazy), 2 * plain), (sk.block_norm(minus(x), minus(v)), sk.block_norm(x, v)),
                      (sk.gated_residual(x, minus(x), scale=minus(v)), sk.gated_residual(x, x, scale=v)),
                      (sk.unpack_activation(*sk.pack_activation(lazy)), sk.unpack_activation(*sk.pack_activation(plain)))):
        assert torch.equal(got, want)
    grads = []
    for f in (minus, lambda t: t):
        leaf, wl = x.clone().requires_grad_(), v.clone().requires_grad_()
        grads.append(torch.autograd.grad(sk.gated_residual(f(leaf), f(leaf), scale=f(wl), post_norm="rms", next_norm="layer"),
                                         [leaf, wl], (f(x), f(x))))
    for p, q in zip(*grads):
        assert torch.equal(p, q)


def test_broadcast_rows_and_gradients():
    """Rows of stride 0 in the inputs and in the incoming gradients."""
    one = randn(1, 96, dtype=torch.float32).expand(50, 96)
    w = randn(96, dtype=torch.float32, seed=2)
    check_norm(one, w, None, "rms", None, one)
    x = stream(50, 96, torch.float32).requires_grad_()
    sk.block_norm(x, w).sum().backward()          # the gradient of a sum has stride 0 everywhere
    (want,) = torch.autograd.grad(sk.block_norm(x, w), x, torch.ones(50, 96, device="cuda"))
    assert torch.equal(x.grad, want)
    # one tensor in several places: its gradients add up
    t = stream(20, 64, torch.float32).requires_grad_()
    out = sk.gated_residual(t, t, gate=t, gate_activation="silu", scale=None, post_norm="rms")
    (got,) = torch.autograd.grad(out.square().sum(), t)
    q = t.detach().double().requires_grad_()
    ref = q + torch.nn.functional.silu(q) * q * (q.square().mean(-1, keepdim=True) + EPS).rsqrt()
    (want,) = torch.autograd.grad(ref.square().sum(), q)
    assert float((got.double() - want).abs().max()) <= 400 * ROUNDOFF[torch.float32] * float(want.abs().max())


def test_offsets_beyond_32_bits():
    """A half-precision stream of more than 2^31 elements: the last rows are read and written at their own place."""
    rows, width = (1 << 21) + 9, 1024
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    tail = stream(9, width, torch.bfloat16)
    x[-9:] = tail
    codes, scales = sk.pack_activation(x)
    want = sk.pack_activation(tail)
    assert torch.equal(codes[-9:], want[0]) and torch.equal(scales[-9:], want[1])
    back = sk.unpack_activation(codes, scales, torch.bfloat16)
    assert torch.equal(back[-9:], sk.unpack_activation(*want, torch.bfloat16))
    del codes, back
    w = randn(width, dtype=torch.float32, seed=2).requires_grad_()
    x.requires_grad_()
    h = sk.block_norm(x, w)
    with torch.no_grad():
        assert torch.equal(h[-9:], sk.block_norm(tail, w))
    dh = torch.zeros(1, 1, device="cuda").expand(rows, width).contiguous()
    dh[-9:] = randn(9, width, dtype=torch.float32, seed=3)
    dx, dw = torch.autograd.grad(h, [x, w], dh)
    t = tail.clone().requires_grad_()
    wdx, wdw = torch.autograd.grad(sk.block_norm(t, w), [t, w], dh[-9:])
    assert torch.equal(dx[-9:], wdx)
    with torch.no_grad():
        xhat = sk.block_norm(tail)
        assert bool(((dw - wdw).abs() <= 32 * ROUNDOFF[torch.float32] * (dh[-9:].abs() * xhat.abs()).sum(0)).all())


# ---- values at the edge ------------------------------------------------------------------------------------------------
def test_rows_of_zeros_and_constants():
    """A zero row has r = eps^-1/2 and gives zeros; a constant row gives zeros under the mean-subtracting norm."""
    x = torch.zeros(3, 200, device="cuda")
    x[1] = 5.0
    assert torch.equal(sk.block_norm(x)[0], torch.zeros(200, device="cuda"))
    h = sk.block_norm(x, kind="layer")
    assert float(h.abs().max()) <= 5.0 * 2 ** -24 * 8 / EPS ** 0.5
    for kind in ("rms", "layer"):
        check_norm(torch.zeros(4, 130, device="cuda"), randn(130, dtype=torch.float32), None, kind, "int8",
                   randn(4, 130, dtype=torch.float32, seed=5))


def test_squares_that_overflow():
    """r = 0 for a row whose squares overflow: finite elements become 0, forward and backward."""
    for width in (24, 500, 40000):
        x = torch.full((3, width), 1e30, device="cuda")
        x[1] = randn(width, dtype=torch.float32)
        x[2, ::2] = -1e30
        for kind in ("rms", "layer"):
            t = x.clone().requires_grad_()
            h = sk.block_norm(t, kind=kind)
            (dx,) = torch.autograd.grad(h, t, torch.ones_like(h))
            assert bool((h[2] == 0).all()) and bool((dx[2] == 0).all()) and bool(torch.isfinite(h).all()) and bool(torch.isfinite(dx).all())
            if kind == "rms":
                assert bool((h[0] == 0).all())
            assert float(h[1].abs().max()) > 0.5


def test_sums_that_overflow():
    """Beyond that the mean itself overflows: NaN from the mean-subtracting norm, still 0 from RMS, and only in that row."""
    for width in (24, 512, 40000):
        x = torch.full((3, width), 3e38, device="cuda")
        x[1] = randn(width, dtype=torch.float32)
        assert bool((sk.block_norm(x)[[0, 2]] == 0).all())
        h = sk.block_norm(x, kind="layer")
        assert h.isnan().all(1).tolist() == [True, False, True] and bool(torch.isfinite(h[1]).all())
        assert bool(sk.block_norm(x.cpu(), kind="layer")[0].isnan().all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_bad_row_stays_alone(bad):
    """NaN and infinities make their own row NaN, in both directions, and no other."""
    c = make_gated(40, 300, torch.float32)
    c["y"][7, 299] = bad
    live = dict(c)
    for n in ("x", "y", "gate"):
        live[n] = c[n].clone().requires_grad_()
    out, h = call_gated(live)
    dx, dy, dg = torch.autograd.grad([out, h], [live["x"], live["y"], live["gate"]], [torch.ones_like(out), torch.ones_like(h)])
    for t in (h, dx, dy, dg):
        rows = torch.isfinite(t).all(1)
        assert not bool(rows[7]) and int(rows.sum()) == 39


def test_saturated_gates():
    """Gates far into both ends of the activation: finite values and gradients."""
    c = make_gated(6, 64, torch.float32, gate="row", act="sigmoid")
    c["gate"] = torch.linspace(-200, 200, 6 * 64, device="cuda").view(6, 64)
    check_gated(c)
    c["act"] = "silu"
    check_gated(c)


@pytest.mark.parametrize("width", [8, 1000, 4096, 40000])
def test_gates_are_accurate_far_from_zero(width):
    """The activation alone (a branch of ones next to a stream of zeros leaves its value as it is), over all gates whose
    sigmoid is a normal number.  Roundings, in units of 2^-24: 2^t 4 and 1 / a 2 (the instructions' bounds), the sum in front of
    it 1, the remainder of t's rounding 1; SiLU's product 1 more."""
    rows = 1 << 17 if width <= 8 else 64
    g = torch.linspace(-87.3, 40.0, rows * width, device="cuda", dtype=torch.float64).float().view(rows, width)
    x, y = torch.zeros(rows, width, device="cuda"), torch.ones(rows, width, device="cuda")
    s = torch.sigmoid(g.double())
    worst = {}
    for act, want, units in (("sigmoid", s, 8), ("silu", g.double() * s, 9)):
        got = sk.gated_residual(x, y, gate=g, gate_activation=act).double()
        worst[act] = float(((got - want).abs() / want.abs().clamp_min(1e-300)).max()) * 2 ** 24
        assert worst[act] <= units, worst
    # derivatives: of the magnitudes s and |g| s (1 - s), where 1 - s carries the error of s
    for act, want, mag in (("sigmoid", s * (1 - s), s), ("silu", s * (1 + g.double() * (1 - s)), s * (1 + g.double().abs()))):
        leaf = g.clone().requires_grad_()
        (got,) = torch.autograd.grad(sk.gated_residual(x, y, gate=leaf, gate_activation=act), leaf, torch.ones_like(x))
        assert float(((got.double() - want).abs() / mag).max()) * 2 ** 24 <= 24
    ends = torch.tensor([-float("inf"), -1e30, -200.0, 200.0, 1e30, float("inf"), float("nan"), 0.0], device="cuda")
    at = torch.zeros(rows, width, device="cuda")
    at[:, :8] = ends
    got = sk.gated_residual(x, y, gate=at, gate_activation="sigmoid")[0, :8]
    assert got.isnan().tolist() == [False] * 6 + [True, False] and got[[0, 1, 2, 3, 4, 5, 7]].tolist() == [0, 0, 0, 1, 1, 1, 0.5]


# ---- checkpoints -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,width", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", ["int8", "e4m3"])
def test_pack_bits(rows, width, dtype, form):
    """Codes and scales are the definition's, bit for bit, and so is what comes back."""
    x = stream(rows, width, dtype)
    x[0, 0] = 0.0
    codes, scales = sk.pack_activation(x, form)
    assert codes.dtype == (torch.int8 if form == "int8" else torch.float8_e4m3fn) and codes.shape == x.shape
    q, s = pack(x, form)
    assert torch.equal(scales, s)
    assert torch.equal(codes.to(q.dtype), q)
    back = sk.unpack_activation(codes, scales, dtype)
    want = (q * s.repeat_interleave(128, -1)[:, :width]).to(dtype)
    assert back.dtype == dtype and torch.equal(back, want)
    # half a code step for int8; half a step of e4m3 (2^-4 of the value, 2^-10 scale steps below its normal range)
    step = s.double().repeat_interleave(128, -1)[:, :width]
    off = (restored(x, form) - x.double()).abs()
    tol = step * 0.5 if form == "int8" else torch.maximum(x.double().abs() * 2.0 ** -4, step * 2.0 ** -10)
    # the three roundings before the code (1 / top, scale, 1 / scale, product) move it by up to 4 u of its value
    assert bool((off <= tol + 4 * ROUNDOFF[branch_type(dtype)] * x.double().abs() + 1e-300).all())


def test_pack_extreme_groups():
    tiny = torch.finfo(torch.float32).tiny
    x = torch.zeros(6, 300, device="cuda")
    x[1, :128] = tiny / 8                          # subnormal group: its scale is the smallest normal
    x[2, 130] = float("nan")
    x[3, 10] = float("inf")
    x[4] = 3.0e38
    x[5, 299] = -1.0
    for form in ("int8", "e4m3"):
        codes, scales = sk.pack_activation(x, form)
        q, s = pack(x, form)
        assert torch.equal(codes.to(torch.float32), q) and torch.equal(torch.nan_to_num(scales, 7.0), torch.nan_to_num(s, 7.0))
        back = sk.unpack_activation(codes, scales)
        assert bool((back[0] == 0).all()) and bool(torch.isnan(back[2, 128:256]).all()) and bool(torch.isfinite(back[2, :128]).all())
        assert bool(torch.isnan(back[3, :128]).all()) and bool(torch.isfinite(back[3, 128:]).all())
        assert bool((back[4] / 3.0e38 - 1).abs().max() < 1e-6) and float(back[5, 299]) == pytest.approx(-1.0, abs=1e-6)
        assert float(back[1].abs().max()) <= tiny / 8 + tiny / 2


def test_checkpoint_holds_an_eighth_of_float64_a_quarter_of_float32():
    """What a training step keeps: codes and scales instead of the input, nothing else of its size."""
    x = stream(4096, 1024, torch.float32)
    base = torch.cuda.memory_allocated()
    kept = {}
    one = torch.ones((), device="cuda", requires_grad=True)
    for form in (None, "int8"):
        h2 = sk.block_norm(x * one, checkpoint=form) * 1.0          # the norm's input lives in its node alone
        torch.cuda.synchronize()
        kept[form] = torch.cuda.memory_allocated() - base - h2.numel() * 4
        del h2
    n = x.numel()
    assert kept[None] >= 4 * n and kept["int8"] <= n * (1 + 4 / 128) + 4096 * 8 + 8192


# ---- refusals ----------------------------------------------------------------------------------------------------------
def test_refusals_on_the_device():
    x, y = torch.zeros(4, 8, device="cuda"), torch.zeros(4, 8, device="cuda")
    for call, words in ((lambda: sk.block_norm(x.int()), "float32, float64"),
                        (lambda: sk.block_norm(x, torch.zeros(8)), "device"),
                        (lambda: sk.gated_residual(x, y.cpu()), "device"),
                        (lambda: sk.pack_activation(x.cpu()), "CUDA"),
                        (lambda: sk.unpack_activation(x, x), "int8 or float8"),
                        (lambda: sk.unpack_activation(x.to(torch.int8), torch.zeros(4, 2, device="cuda")), "shape"),
                        (lambda: sk.unpack_activation(x.to(torch.int8), torch.zeros(4, 1, device="cuda"), torch.float64), "scales")):
        with pytest.raises(RuntimeError, match=words):
            call()
    t = x.clone().requires_grad_()
    h = sk.block_norm(t, checkpoint="int8")
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(h.sum(), t, create_graph=True)
    out = sk.gated_residual(t, y, checkpoint="int8")
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(out.sum(), t, create_graph=True)


def test_function_transforms_are_refused():
    x = torch.ones(3, 4, 8, device="cuda")
    for call in (lambda: torch.vmap(lambda t: sk.block_norm(t))(x), lambda: torch.func.grad(lambda t: sk.block_norm(t).sum())(x),
                 lambda: torch.vmap(lambda t: sk.gated_residual(t, t))(x), lambda: torch.vmap(lambda t: sk.pack_activation(t))(x)):
        with pytest.raises(RuntimeError, match="torch.func"):
            call()
    got = sk.block_norm(torch.nn.Parameter(x), torch.nn.Parameter(torch.ones(8, device="cuda")))
    assert got.requires_grad and torch.allclose(got, x)


def test_graph_is_used_once_and_inputs_stay():
    """A second backward without retain_graph, and an input changed in between, are errors; forward mode is refused."""
    x = stream(5, 64, torch.float32).requires_grad_()
    w = torch.ones(64, device="cuda", requires_grad=True)
    for call in (lambda t: sk.block_norm(t, w), lambda t: sk.block_norm(t, w, checkpoint="int8"),
                 lambda t: sk.gated_residual(t, t * 1.0, scale=w, post_norm="rms")):
        out = call(x).sum()
        out.backward(retain_graph=True)
        out.backward()
        with pytest.raises(RuntimeError, match="second time"):
            out.backward()
    t = x.detach() * 1.0
    t.requires_grad_()
    out = sk.block_norm(t, w)
    with torch.no_grad():
        t.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))
        for call in (lambda: sk.block_norm(dual), lambda: sk.gated_residual(x, dual)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_no_rows():
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.zeros(0, 64, dtype=dtype, device="cuda", requires_grad=True)
        w = torch.ones(64, device="cuda", requires_grad=True)
        y = torch.zeros(0, 64, device="cuda", requires_grad=True)
        out, h = sk.gated_residual(x, y, gate=y, gate_activation="silu", scale=w, post_norm="rms", next_norm="layer",
                                   next_weight=w, checkpoint="int8")
        h2 = sk.block_norm(x, w, checkpoint="e4m3")
        assert out.shape == h.shape == h2.shape == (0, 64) and out.dtype == dtype and h.dtype == torch.float32
        (g,) = torch.autograd.grad(out.float().sum() + h.sum() + h2.sum(), w)
        assert torch.equal(g, torch.zeros(64, device="cuda"))
    codes, scales = sk.pack_activation(torch.zeros(0, 200, device="cuda"))
    assert codes.shape == (0, 200) and scales.shape == (0, 2) and sk.unpack_activation(codes, scales).shape == (0, 200)


# ---- higher derivatives, streams, graphs ---------------------------------------------------------------------------------
def test_second_derivatives():
    w, b = randn(6, seed=2).requires_grad_(), randn(6, seed=3).requires_grad_()
    x, y = randn(3, 6, seed=4).requires_grad_(), randn(3, 12, seed=5).requires_grad_()
    s, pw, nw = (randn(6, seed=k).requires_grad_() for k in (6, 7, 8))
    for kind in ("rms", "layer"):
        f = lambda x, w, b: sk.block_norm(x, w, b, kind=kind)
        assert torch.autograd.gradcheck(f, (x, w, b)) and torch.autograd.gradgradcheck(f, (x, w, b))
        f = lambda x, y, s, pw, nw, b: sk.gated_residual(x, y, gate="packed", gate_activation="silu", scale=s, post_norm=kind,
                                                         post_weight=pw, next_norm=kind, next_weight=nw, next_bias=b)
        assert torch.autograd.gradcheck(f, (x, y, s, pw, nw, b)) and torch.autograd.gradgradcheck(f, (x, y, s, pw, nw, b))
    gate = randn(1, 6, seed=9).requires_grad_()
    y1 = randn(3, 6, seed=5).requires_grad_()
    f = lambda x, y, g: sk.gated_residual(x, y, gate=g, gate_activation="sigmoid")
    assert torch.autograd.gradcheck(f, (x, y1, gate)) and torch.autograd.gradgradcheck(f, (x, y1, gate))


def test_another_stream():
    c = make_gated(500, 512, torch.float32)
    want = check_gated(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = check_gated(c)
    torch.cuda.current_stream().wait_stream(side)
    for n in want[1]:
        assert torch.equal(want[1][n], got[1][n])


def test_two_captured_graphs_replayed_together():
    """Forward and backward captured twice, replayed on two streams at once: no shared scratch."""
    cases = [make_gated((4, 600), 384, torch.float32, "sequence", seed=s) for s in (10, 50)]
    want = [check_gated(c)[1] for c in cases]
    graphs, grads = [], []
    for c in cases:
        live = {k: v.detach().requires_grad_() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
        names = [n for n, _ in LEAVES if c[n] is not None]
        dout, dh = randn(*c["x"].shape, seed=31).float(), randn(*c["x"].shape, seed=32).float()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(call_gated(live), [live[n] for n in names], (dout, dh))
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(call_gated(live), [live[n] for n in names], (dout, dh))
        graphs.append(graph)
        grads.append((dict(zip(names, got)), live, dout, dh))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for w, (g, *_) in zip(want, grads):
        for n in w:
            assert torch.equal(w[n], g[n]), n


def test_gradients_against_differences():
    """The float32 kernels' gradients against differences of the float64 kernels' values."""
    c = make_gated((2, 3), 20, torch.float64, "sequence")
    dout, dh = randn(2, 3, 20, seed=31), randn(2, 3, 20, seed=32)
    live = {k: v.detach().float().requires_grad_() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    names = [n for n, _ in LEAVES if c[n] is not None]
    grads = torch.autograd.grad(call_gated(live), [live[n] for n in names], (dout.float(), dh.float()))

    def loss(cc):
        out, h = call_gated(cc)
        return float((out * dout).sum() + (h * dh).sum())

    for n, g in zip(names, grads):
        direction = randn(*c[n].shape, seed=77)
        step = 1e-6
        hi, lo = ({**c, n: c[n] + s * step * direction} for s in (1, -1))
        slope = (loss(hi) - loss(lo)) / (2 * step)
        got = float((g.double() * direction).sum())
        # float32 gradients of a few hundred terms; the difference's own error is about 1e-16 / step of the loss
        scale = float((g.double().abs() * direction.abs()).sum())
        assert abs(got - slope) <= 400 * ROUNDOFF[torch.float32] * scale + 1e-7 * abs(loss(c)) + 1e-6 * scale, n
