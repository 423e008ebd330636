"""Plain 64-bit forms of the group norm and of gradient clipping, and what rounding allows a float32 kernel to be off: shared by the
tests of both.  u = 2^-24 is half a step of float32 relative to the value; an output type adds half a step of its own."""
import torch

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# below its smallest normal number a type's steps stop shrinking: half of the last one
FLOOR = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def norm64(x, groups, weight, bias, eps, act, residual, dy=None):
    """{name: (value, largest allowed error)} of y and, with dy, of all gradients; float64, from the definition.

    The kernel forms x - mean (1 rounding), times rstd * gamma in forward or rstd and then gamma in backward (2 roundings of the
    constants, 1-2 of the fused multiply-adds), adds beta and the residual (2 roundings): z is off by at most
    8u (|xhat gamma| + |lo gamma| + |beta| + |res|), lo = what rounding the mean to 32 bits left, in units of the deviation.
    SiLU: e^-z by exp2 of a rounded product is off by (1.5 |z| + 2) u relative, the reciprocal and the products by 5u more."""
    n, c = x.shape[0], x.shape[-1]
    cg = c // groups
    xd = x.double().reshape(n, -1, groups, cg)
    m = xd.shape[1] * cg
    mean = xd.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt((xd - mean).square().mean((1, 3), keepdim=True) + eps)
    full = lambda t: t.expand(n, xd.shape[1], groups, cg).reshape(n, -1, c)       # noqa: E731
    xhat = ((xd - mean) * rstd).reshape(n, -1, c)
    lo = full((mean.abs() * U) * rstd)
    rstd, mean = full(rstd), full(mean)
    w = torch.ones(c, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    b = torch.zeros(c, dtype=torch.float64, device=x.device) if bias is None else bias.double()
    res = torch.zeros_like(xhat) if residual is None else residual.double().reshape(n, -1, c)
    z = xhat * w + b + res
    dz_err = 8 * U * ((xhat * w).abs() + (lo * w).abs() + b.abs() + res.abs())       # of z
    if act == "none":
        y, ey = z, dz_err
    elif act == "relu":
        y, ey = torch.relu(z), dz_err
    else:
        sig = torch.sigmoid(z)
        y = z * sig
        ey = 1.1 * dz_err + ((1.5 * z.abs() + 7) * (1 - sig) + 3) * U * y.abs()
    shape, dt = x.shape, x.dtype
    out = lambda v, e, t: (v, e + HALF_STEP[t] * (v.abs() + e) + FLOOR[t])           # noqa: E731
    r = {"y": out(y.reshape(shape), ey.reshape(shape), dt)}
    if dy is None:
        return r
    g = dy.double().reshape(n, -1, c)
    if act == "relu":
        d, ed = (z > 0).double(), torch.zeros_like(z)
    elif act == "silu":
        d = sig * (1 + z * (1 - sig))
        # |silu''| <= 1/2; sig is off by (1.5|z| + 7)(1 - sig) u relative, 1 - sig by as much absolute
        es = ((1.5 * z.abs() + 7) * (1 - sig) + 2) * U * sig
        ed = 0.5 * dz_err + es * (1 + 2 * z.abs()) + 4 * U * (sig * (1 + z.abs()))
    else:
        d, ed = torch.ones_like(z), torch.zeros_like(z)
    dz, edz = g * d, g.abs() * ed + (U * (g * d).abs() if act == "silu" else 0)
    exh = 4 * U * (xhat.abs() + lo)
    if residual is not None:
        r["dresidual"] = out(dz.reshape(shape), edz.reshape(shape), dt)
    r["dbias"] = out(dz.sum((0, 1)), edz.sum((0, 1)), torch.float32)
    r["dweight"] = out((dz * xhat).sum((0, 1)), (edz * xhat.abs() + dz.abs() * exh).sum((0, 1)), torch.float32)
    gz, egz = dz * w, edz * w.abs() + U * (dz * w).abs()
    gmean = lambda t: full(t.reshape(n, -1, groups, cg).mean((1, 3), keepdim=True))   # noqa: E731
    c1, c2 = gmean(gz), gmean(gz * xhat)
    ec1 = gmean(egz) + U * c1.abs()
    ec2 = gmean(egz * xhat.abs() + gz.abs() * exh) + U * c2.abs()
    inner = gz - c1 - xhat * c2
    ei = egz + ec1 + xhat.abs() * ec2 + c2.abs() * exh + 3 * U * (gz.abs() + c1.abs() + (xhat * c2).abs())
    r["dx"] = out((inner * rstd).reshape(shape), (rstd * (ei + 2 * U * inner.abs())).reshape(shape), dt)
    return r


def within(got, want, what):
    value, allowed = want
    assert got.shape == value.shape, (what, got.shape, value.shape)
    off = (got.double() - value).abs()
    bad = ~(off <= allowed)
    if bool(bad.any()):
        i = int((off / allowed.clamp_min(1e-300)).argmax())
        raise AssertionError("%s: %d of %d values are off; the worst is %.9g, exact %.9g, allowed +-%.3g" % (
            what, int(bad.sum()), bad.numel(), float(got.reshape(-1)[i]), float(value.reshape(-1)[i]), float(allowed.reshape(-1)[i])))
