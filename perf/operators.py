"""Cases of the operators around a KAN layer: the norm in front of it, the gated residual connection behind it, and the
8-bit checkpoints that a training step keeps of their inputs.

``own = False`` computes every operator with elementary torch operations; ``own = True`` calls this package."""
import math

import torch

own = False

GROUP = 128                          # columns of a row that share one scale of a checkpoint
EPS = 1e-6
DTYPES = {"float32": torch.float32, "float64": torch.float64, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _norm(name, rows, width, dtype="float32", kind="rms", checkpoint="none", train=True):
    return dict(name=name, op="norm", rows=rows, width=width, dtype=dtype, kind=kind, checkpoint=checkpoint, train=train)


def _gated(name, rows, width, dtype="float32", gate="row", act="silu", seq=1, post="rms", after="rms",
           checkpoint="none", train=True):
    return dict(name=name, op="gated", rows=rows, width=width, dtype=dtype, gate=gate, act=act, seq=seq, post=post,
                after=after, checkpoint=checkpoint, train=train)


def _checkpoint(name, rows, width, dtype="float32", form="int8"):
    return dict(name=name, op="checkpoint", rows=rows, width=width, dtype=dtype, form=form)


def listed():
    return [
        # one row in front of a 1024 -> 1024 layer: an exported network answering a single request
        _norm("norm one row", 1, 1024, train=False),
        # the training batch of the 1024 -> 1024 benchmark layer
        _norm("norm train 64k x 1024", 65536, 1024),
        # half-precision stream of an odd width, mean-subtracting norm with its bias, input kept in 8 bits
        _norm("norm train bf16 odd int8", 9001, 1001, "bfloat16", "layer", "int8"),
        # a wide stream whose norm inputs are kept as 8-bit floats
        _norm("norm train wide e4m3", 8192, 4096, "float32", "rms", "e4m3"),
        # four rows through the connection behind a layer that returns value and gate side by side
        _gated("gated four rows packed", 4, 1024, gate="packed", train=False),
        # a long prompt whose gate comes from a conditioning vector per sequence; the next block's norm is fused
        _gated("gated prompt per sequence", 8192, 4096, gate="sequence", act="none", seq=2048, post="none", after="layer",
               train=False),
        # training step of a block with everything: a gate per row, both norms, all gradients
        _gated("gated train rows", 16384, 1024),
        # ragged training batch: nine sequences of 457 rows, odd width, conditioning gate, no norm behind
        _gated("gated train odd sequences", 9 * 457, 777, gate="sequence", act="sigmoid", seq=457, post="layer", after="none"),
        # the float64 configuration with 131072 rows of width 64: residual scale alone, both norms
        _gated("gated train f64 narrow", 131072, 64, "float64", gate="none", act="none"),
        # half-precision stream, value and gate side by side, both kept in 8 bits for the backward
        _gated("gated train bf16 int8", 16384, 2048, "bfloat16", gate="packed", after="none", checkpoint="int8"),
        # the input of the 1024 -> 1024 benchmark layer, packed in the forward and restored in the backward
        _checkpoint("checkpoint 64k x 1024", 65536, 1024),
        # an odd half-precision activation as 8-bit floats
        _checkpoint("checkpoint odd e4m3", 5003, 333, "bfloat16", "e4m3"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "gated", "gated", "gated", "checkpoint"])
    width = _log(rng, 8, 8192)
    if rng.random() < 0.5:
        width = max(8, width // 32 * 32)
    rows = _log(rng, 1, max(1, min(131072, (1 << 24) // width)))
    if op == "checkpoint":
        case = _checkpoint("", rows, width, rng.choice(["float32", "float32", "bfloat16", "float16"]),
                           rng.choice(["int8", "e4m3"]))
    elif op == "norm":
        case = _norm("", rows, width, rng.choice(["float32", "float32", "bfloat16", "float16", "float64"]),
                     rng.choice(["rms", "layer"]), rng.choice(["none", "none", "int8", "e4m3"]), rng.random() < 0.7)
        if case["dtype"] == "float64" or not case["train"]:
            case["checkpoint"] = "none"
    else:
        dtype = rng.choice(["float32", "float32", "float32", "bfloat16", "float64"])
        after = "none" if dtype == "bfloat16" else rng.choice(["rms", "rms", "layer", "none"])
        gate = rng.choice(["none", "row", "sequence", "packed"])
        seq = 1
        if gate == "sequence":
            seq = _log(rng, 1, rows)
            rows = max(1, rows // seq) * seq
        train = rng.random() < 0.7
        keep = "none" if not train or after != "none" or dtype == "float64" else rng.choice(["none", "int8", "e4m3"])
        case = _gated("", rows, width, dtype, gate, "none" if gate == "none" else rng.choice(["none", "sigmoid", "silu"]), seq,
                      rng.choice(["none", "rms", "layer"]), after, keep, train)
    del case["name"]
    return case


def _branch(dtype):
    """The type of the layers' side: they compute in 32 bits next to a half-precision stream."""
    return torch.float64 if dtype == torch.float64 else torch.float32


def work(case):
    n = case["rows"] * case["width"]
    S = torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    B = 8 if case["dtype"] == "float64" else 4
    if case["op"] == "checkpoint":
        scales = 4 * case["rows"] * -(-case["width"] // GROUP)
        return {"bytes": 2 * n * S + 2 * (n + scales), "flops": 5 * n}
    if case["op"] == "norm":
        return {"bytes": n * (S + B) * (2 if case["train"] else 1), "flops": n * (16 if case["train"] else 5)}
    per_row = case["gate"] in ("row", "packed")
    gates = 0 if case["gate"] == "none" else n if per_row else n // case["seq"]
    after = case["after"] != "none"
    size = n * (2 * S + B + (B if after else 0)) + gates * B                       # x, y, gate -> out, h
    if case["train"]:
        size += n * (S + B + (S + B if after else 0)) + gates * B                  # dout, dh -> dx, dy, dgate
    return {"bytes": size, "flops": n * (50 if case["train"] else 16)}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, width, dtype = case["rows"], case["width"], DTYPES[case["dtype"]]
    branch = _branch(dtype)
    shape = (rows, width) if case.get("gate") != "sequence" else (rows // case["seq"], case["seq"], width)

    def randn(*size, like=branch):
        return torch.randn(*size, device="cuda", generator=g, dtype=torch.float64 if like == torch.float64 else torch.float32).to(like)

    def stream():
        # a residual stream: unit rows with a few columns that run an order of magnitude larger
        loud = 1 + 9 * (torch.rand(width, device="cuda", generator=g) < 0.01)
        return (randn(*shape) * loud.to(branch)).to(dtype)

    if case["op"] == "checkpoint":
        return {"case": case, "x": stream()}
    leaf = (lambda t: t.requires_grad_()) if case["train"] else (lambda t: t)
    s = {"case": case, "x": leaf(stream())}
    if case["op"] == "norm":
        s["weight"] = leaf(1 + 0.1 * randn(width))
        s["bias"] = leaf(0.1 * randn(width)) if case["kind"] == "layer" else None
        if case["train"]:
            s["dh"] = randn(*shape)
        return s
    s["y"] = leaf(randn(*shape[:-1], 2 * width) if case["gate"] == "packed" else randn(*shape))
    s["gate"] = {"none": lambda: None, "packed": lambda: None, "row": lambda: leaf(randn(*shape)),
                 "sequence": lambda: leaf(randn(shape[0], 1, width))}[case["gate"]]()
    s["scale"] = leaf(0.5 + 0.1 * randn(width))
    for side, kind in (("post", case["post"]), ("next", case["after"])):
        s[side + "_weight"] = leaf(1 + 0.1 * randn(width)) if kind != "none" else None
        s[side + "_bias"] = leaf(0.1 * randn(width)) if kind == "layer" else None
    if case["train"]:
        s["dout"] = randn(*shape).to(dtype)
        s["dh"] = randn(*shape) if case["after"] != "none" else None
    return s


GATED_LEAVES = ("x", "y", "gate", "scale", "post_weight", "post_bias", "next_weight", "next_bias")


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return {"norm": _own_norm, "gated": _own_gated, "checkpoint": _own_checkpoint}[case["op"]](state, case)
    with torch.no_grad():
        return {"norm": _plain_norm, "gated": _plain_gated, "checkpoint": _plain_checkpoint}[case["op"]](state, case)


def _or_none(name):
    return None if name == "none" else name


def _own_norm(s, case):
    import torchsplinekan_b200 as kan
    if not case["train"]:
        return {"h": kan.block_norm(s["x"], s["weight"], s["bias"], kind=case["kind"], eps=EPS)}
    h = kan.block_norm(s["x"], s["weight"], s["bias"], kind=case["kind"], eps=EPS, checkpoint=_or_none(case["checkpoint"]))
    names = [n for n in ("x", "weight", "bias") if s[n] is not None]
    grads = torch.autograd.grad(h, [s[n] for n in names], s["dh"])
    return {"h": h.detach(), **{"d" + n: v for n, v in zip(names, grads)}}


def _own_gated(s, case):
    import torchsplinekan_b200 as kan
    gate = "packed" if case["gate"] == "packed" else s["gate"]
    got = kan.gated_residual(s["x"], s["y"], gate=gate, gate_activation=_or_none(case["act"]), scale=s["scale"],
                             post_norm=_or_none(case["post"]), post_weight=s["post_weight"], post_bias=s["post_bias"],
                             next_norm=_or_none(case["after"]), next_weight=s["next_weight"], next_bias=s["next_bias"],
                             eps=EPS, checkpoint=_or_none(case["checkpoint"]))
    outs = got if isinstance(got, tuple) else (got,)
    result = dict(zip(("out", "h"), (t.detach() for t in outs)))
    if case["train"]:
        names = [n for n in GATED_LEAVES if s[n] is not None]
        grads = torch.autograd.grad(outs, [s[n] for n in names], (s["dout"], s["dh"])[:len(outs)])
        result.update({"d" + n: v for n, v in zip(names, grads)})
    return result


def _own_checkpoint(s, case):
    import torchsplinekan_b200 as kan
    codes, scales = kan.pack_activation(s["x"], case["form"])
    return {"scales": scales, "restored": kan.unpack_activation(codes, scales, s["x"].dtype)}


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _packed(x, form):
    """(values after the round trip, scales) of a checkpoint of ``x`` in 32 bits."""
    rows, width = x.shape
    groups = -(-width // GROUP)
    xg = x.new_zeros(rows, groups * GROUP)
    xg[:, :width] = x
    xg = xg.view(rows, groups, GROUP)
    top = 127.0 if form == "int8" else 448.0
    scales = (xg.abs().amax(-1) * (1.0 / top)).clamp_min(torch.finfo(x.dtype).tiny)
    q = xg * scales.reciprocal()[..., None]
    q = q.round().clamp(-top, top) if form == "int8" else q.to(torch.float8_e4m3fn).to(x.dtype)
    return (q * scales[..., None]).view(rows, -1)[:, :width], scales


def _plain_checkpoint(s, case):
    values, scales = _packed(s["x"].to(torch.float32), case["form"])
    return {"scales": scales, "restored": values.to(s["x"].dtype)}


def _stats(v, kind):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    return mean, ((v - mean).square().mean(-1, keepdim=True) + EPS).rsqrt()


def _norm_gradient(vhat, rstd, kind, weight, d):
    """Gradient of a norm's input, and of its weight and bias, from the gradient ``d`` of its output."""
    v = d * weight
    inner = v - vhat * (v * vhat).mean(-1, keepdim=True)
    if kind == "layer":
        inner = inner - v.mean(-1, keepdim=True)
    return rstd * inner, _over_rows(d * vhat), _over_rows(d)


def _over_rows(t):
    return t.reshape(-1, t.shape[-1]).sum(0)


def _kept(v, form):
    return v if form == "none" else _packed(v.reshape(-1, v.shape[-1]), form)[0].view(v.shape)


def _plain_norm(s, case):
    x = s["x"].to(_branch(s["x"].dtype))
    mean, rstd = _stats(x, case["kind"])
    h = (x - mean) * rstd * s["weight"]
    if s["bias"] is not None:
        h = h + s["bias"]
    if not case["train"]:
        return {"h": h}
    xhat = (_kept(x, case["checkpoint"]) - mean) * rstd
    dx, dweight, dbias = _norm_gradient(xhat, rstd, case["kind"], s["weight"], s["dh"])
    result = {"h": h, "dx": dx.to(s["x"].dtype), "dweight": dweight}
    if s["bias"] is not None:
        result["dbias"] = dbias
    return result


def _activation(gate, act):
    """Value and derivative of the gate's activation."""
    if act == "none":
        return gate, torch.ones_like(gate)
    sig = 1 / (1 + torch.exp(-gate))
    if act == "sigmoid":
        return sig, sig * (1 - sig)
    return gate * sig, sig * (1 + gate * (1 - sig))


def _plain_gated(s, case):
    x = s["x"].to(_branch(s["x"].dtype))
    width, scale = case["width"], s["scale"]
    y, gate = s["y"], s["gate"]
    if case["gate"] == "packed":
        y, gate = y[..., :width], y[..., width:]
    a = _activation(gate, case["act"])[0] if gate is not None else torch.ones_like(scale)
    pmean, prstd = _stats(y, case["post"]) if case["post"] != "none" else (None, None)

    def post(v):
        if case["post"] == "none":
            return v, v
        vhat = (v - pmean) * prstd
        z = vhat * s["post_weight"]
        return vhat, z if s["post_bias"] is None else z + s["post_bias"]

    out = x + scale * a * post(y)[1]
    result = {"out": out.to(s["x"].dtype)}
    if case["after"] != "none":
        nmean, nrstd = _stats(out, case["after"])
        nhat = (out - nmean) * nrstd
        h = nhat * s["next_weight"]
        result["h"] = h if s["next_bias"] is None else h + s["next_bias"]
    if not case["train"]:
        return result

    grads = {}
    g = s["dout"].to(x.dtype)
    if case["after"] != "none":
        dnext, grads["next_weight"], grads["next_bias"] = _norm_gradient(nhat, nrstd, case["after"], s["next_weight"], s["dh"])
        g = g + dnext
    grads["x"] = g.to(s["x"].dtype)
    per_row = case["gate"] in ("row", "packed")
    y_, gate_ = _kept(y, case["checkpoint"]), _kept(gate, case["checkpoint"]) if per_row else gate
    yhat, z = post(y_)
    if gate is not None:
        a, da = _activation(gate_, case["act"])
        dgate = g * scale * da * z
        grads["gate"] = dgate.sum(1, keepdim=True) if case["gate"] == "sequence" else dgate
    grads["scale"] = _over_rows(g * a * z)
    dz = g * scale * a
    if case["post"] == "none":
        grads["y"] = dz
    else:
        grads["y"], grads["post_weight"], grads["post_bias"] = _norm_gradient(yhat, prstd, case["post"], s["post_weight"], dz)
    if case["gate"] == "packed":
        grads["y"] = torch.cat([grads["y"], grads["gate"]], -1)
    result.update({"d" + n: grads[n] for n in GATED_LEAVES if s[n] is not None})
    return result


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _standardised(v, kind, at=None):
    """``(at - mean) / sqrt(var + eps)`` with the moments of ``v``, and the factor of the moments."""
    m = v.mean(-1, keepdim=True) if kind == "layer" else 0.0
    sd = torch.sqrt((v - m).pow(2).mean(-1, keepdim=True) + EPS)
    return ((v if at is None else at) - m) / sd, sd


def _through(d, vhat, sd, kind):
    """The Jacobian of the standardisation, transposed, applied to ``d``."""
    n = vhat.shape[-1]
    along = torch.einsum("...i,...i->...", d, vhat)[..., None] / n
    flat = d.sum(-1, keepdim=True) / n if kind == "layer" else 0.0
    return (d - flat - along * vhat) / sd


def _roundtrip(v, form):
    """The checkpoint's values: what is held are its codes and its 32-bit scales, so these are formed as stored."""
    if form == "none":
        return v
    flat = v.reshape(-1, v.shape[-1])
    parts = []
    for lo in range(0, flat.shape[1], GROUP):
        part = flat[:, lo:lo + GROUP].float()
        top = 127 if form == "int8" else 448
        one = (part.abs().max(1, keepdim=True).values * (1.0 / top)).clamp_min(torch.finfo(torch.float32).tiny)
        q = part * one.reciprocal()
        q = torch.round(q).clamp(-top, top) if form == "int8" else q.to(torch.float8_e4m3fn)
        parts.append(q.double() * one.double())
    return torch.cat(parts, 1).view(v.shape)


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    x = d["x"]
    rows_of = lambda t: t.reshape(-1, t.shape[-1]).sum(0)
    if case["op"] == "checkpoint":
        flat = torch.nn.functional.pad(x, (0, -x.shape[1] % GROUP)).view(x.shape[0], -1, GROUP)
        top = 127 if case["form"] == "int8" else 448
        return {"scales": (flat.abs().amax(-1) / top).clamp_min(torch.finfo(torch.float32).tiny),
                "restored": _roundtrip(x, case["form"])}
    if case["op"] == "norm":
        xhat, sd = _standardised(x, case["kind"])
        h = xhat * d["weight"] + d.get("bias", 0.0)
        if not case["train"]:
            return {"h": h}
        kept = _standardised(x, case["kind"], _roundtrip(x, case["checkpoint"]))[0]
        result = {"h": h, "dx": _through(d["dh"] * d["weight"], kept, sd, case["kind"]), "dweight": rows_of(d["dh"] * kept)}
        if "bias" in d:
            result["dbias"] = rows_of(d["dh"])
        return result

    width, packed = case["width"], case["gate"] == "packed"
    y = d["y"][..., :width] if packed else d["y"]
    gate = d["y"][..., width:] if packed else d.get("gate")

    def branch(y_, gate_):
        """out - x, and the factors of its gradients, with the post norm's moments always those of ``y``."""
        yhat, sd = _standardised(y, case["post"], y_) if case["post"] != "none" else (y_, 1.0)
        z = yhat * d.get("post_weight", 1.0) + d.get("post_bias", 0.0)
        if gate_ is None:
            return d["scale"] * z, z, yhat, sd, 1.0, None
        sig = torch.sigmoid(gate_)
        a, da = {"none": (gate_, torch.ones_like(gate_)), "sigmoid": (sig, sig - sig * sig),
                 "silu": (gate_ * sig, sig + gate_ * (sig - sig * sig))}[case["act"]]
        return d["scale"] * a * z, z, yhat, sd, a, da

    out = x + branch(y, gate)[0]
    result = {"out": out}
    if case["after"] != "none":
        nhat, nsd = _standardised(out, case["after"])
        result["h"] = nhat * d["next_weight"] + d.get("next_bias", 0.0)
    if not case["train"]:
        return result
    g = d["dout"]
    grads = {}
    if case["after"] != "none":
        g = g + _through(d["dh"] * d["next_weight"], nhat, nsd, case["after"])
        grads["next_weight"], grads["next_bias"] = rows_of(d["dh"] * nhat), rows_of(d["dh"])
    kept_gate = _roundtrip(gate, case["checkpoint"]) if case["gate"] in ("row", "packed") else gate
    _, z, yhat, sd, a, da = branch(_roundtrip(y, case["checkpoint"]), kept_gate)
    dz = g * d["scale"] * a
    grads["x"], grads["scale"] = g, rows_of(g * a * z)
    grads["post_weight"], grads["post_bias"] = rows_of(dz * yhat), rows_of(dz)
    grads["y"] = _through(dz * d["post_weight"], yhat, sd, case["post"]) if case["post"] != "none" else dz
    if gate is not None:
        dgate = g * d["scale"] * da * z
        grads["gate"] = dgate.sum(1, keepdim=True) if case["gate"] == "sequence" else dgate
        if packed:
            grads["y"] = torch.cat([grads["y"], grads["gate"]], -1)
    result.update({"d" + n: grads[n] for n in GATED_LEAVES if s[n] is not None})
    return result
