"""Plain float64 forms of the operators around a layer, each value with the magnitude its rounding errors scale with
(imported by the tests, not collected).

A result in floating point with unit roundoff u is off by at most (number of roundings) * u times the sum of the
magnitudes of the terms it is formed from.  Every function here returns ``(value, magnitude)`` pairs where ``magnitude``
is that sum, formed with the absolute values of the terms.
"""
import torch

GROUP = 128
ROUNDOFF = {torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53}
DTYPES = [torch.float32, torch.float64, torch.bfloat16, torch.float16]


def branch_type(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def roundings(width):
    """Bound on the roundings behind one element: a sum over the row adds at most ceil(width / 128) + 16 terms in a
    chain (a thread's share, then lanes and warps), twice (mean and variance, or the two sums of a backward), and the
    element itself takes fewer than 40 operations, exp included (2 ulp)."""
    return 2 * (-(-width // 128) + 16) + 48


def assert_close(got, want, dtype, width, extra=0, what=""):
    """``got`` against ``(value, magnitude)``: rounding errors of the arithmetic, then half a step of the result's type
    where that is a narrower one."""
    value, magnitude = want
    u = ROUNDOFF[branch_type(dtype)]
    # What underflows is off by up to the smallest normal number (a gate of -100 has a sigmoid of 4e-44, which float32
    # arithmetic makes 0: exp(100) is beyond its range); the factors behind it are below 2^20 in these tests (r is at most
    # eps^-1/2 = 1000, weights and gradients below 2^5).
    tol = (roundings(width) + extra) * u * magnitude.to(value.device) + torch.finfo(branch_type(dtype)).tiny * 2.0 ** 20
    if got.dtype in (torch.bfloat16, torch.float16):
        tol = tol + torch.finfo(got.dtype).eps / 2 * (value.abs() + tol) + torch.finfo(got.dtype).smallest_normal
    off = (got.double() - value).abs()
    bad = off > tol
    assert got.shape == value.shape, (what, got.shape, value.shape)
    assert not bool(bad.any()) and bool(torch.isfinite(got.double()).all()), (
        what, float((off / (tol)).max()), int(bad.sum()))


def moments(v, kind, eps):
    m = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    return m, ((v - m).square().mean(-1, keepdim=True) + eps).rsqrt()


def norm(v, w, b, kind, eps, at=None):
    """(value, magnitude) of the norm's result and of the normalised row; ``at``: what stands for ``v`` in the numerator
    (the moments are always those of ``v``)."""
    m, r = moments(v, kind, eps)
    at = v if at is None else at
    vhat, mag = (at - m) * r, (at.abs() + m.abs()) * r
    # the relative error of r is that of the variance: the cancellation v - m enters through its magnitude
    blow = ((v.abs() + m.abs()).square().mean(-1, keepdim=True) + eps) * r.square()
    mag = mag * blow
    z, zmag = vhat, mag
    if w is not None:
        z, zmag = z * w, zmag * w.abs()
    if b is not None:
        z, zmag = z + b, zmag + b.abs()
    return (z, zmag), (vhat, mag), r * 1.0, r * blow


def norm_backward(vhat, vmag, r, rmag, w, d, dmag, kind):
    """(value, magnitude) of the gradients of input, weight and bias for the output gradient ``d``."""
    w = torch.ones_like(vhat[..., :1, :].reshape(-1, vhat.shape[-1])[0]) if w is None else w
    u, umag = d * w, dmag * w.abs()
    dv = u - vhat * (u * vhat).mean(-1, keepdim=True)
    mag = umag + vmag * (umag * vmag).mean(-1, keepdim=True)
    if kind == "layer":
        dv, mag = dv - u.mean(-1, keepdim=True), mag + umag.mean(-1, keepdim=True)
    rows = lambda t: t.reshape(-1, t.shape[-1]).sum(0)
    return (r * dv, rmag * mag), (rows(d * vhat), rows(dmag * vmag)), (rows(d), rows(dmag))


def activation(g, act):
    """value, its magnitude, derivative, its magnitude"""
    if act is None:
        return g, g.abs(), torch.ones_like(g), torch.ones_like(g)
    s = torch.sigmoid(g)
    smag = s * (1 + g.abs())                      # an error of u |g| in the exponent's argument
    if act == "sigmoid":
        return s, smag, s * (1 - s), smag
    return g * s, g.abs() * smag, s * (1 + g * (1 - s)), smag * (1 + g.abs())


def pack(x, form):
    """(codes as values, scales) by the definition, in the branch's type: bit for bit what the kernel stores."""
    x = x.to(branch_type(x.dtype))
    flat = x.reshape(-1, x.shape[-1])
    top = 127.0 if form == "int8" else 448.0
    codes, scales = [], []
    for lo in range(0, flat.shape[1], GROUP):
        part = flat[:, lo:lo + GROUP]
        s = (part.abs().amax(1, keepdim=True) * (1.0 / top)).clamp_min(torch.finfo(x.dtype).tiny)
        q = part * s.reciprocal()
        if form == "int8":
            q = q.round().clamp(-top, top)
        else:
            q = q.clamp(-top, top).to(torch.float8_e4m3fn).to(x.dtype)
        codes.append(torch.where(torch.isfinite(s), q, torch.zeros_like(q)))
        scales.append(s)
    return torch.cat(codes, 1).view(x.shape), torch.cat(scales, 1).view(x.shape[:-1] + (-1,))


def restored(x, form):
    """float64 values of the checkpoint of ``x`` (``x`` itself without one)."""
    if form is None:
        return x.double()
    q, s = pack(x, form)
    full = s.double().repeat_interleave(GROUP, -1)[..., :x.shape[-1]]
    return q.double() * full
