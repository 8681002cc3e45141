"""Plain implementations in float64 of the operators around the mixer, with an
elementwise bound on what a result of a given type may differ from them.

The bounds follow from the arithmetic, not from measurement. u = 2^-24 is half
an ulp of fp32, R = 2^-8 of bf16 (the unit of a rounding to the tensors' type;
R = u for fp32). A product of K terms summed in fp32 is off by at most
2(K + 4)u times the sum of the terms' magnitudes (the factor 2 allows for
truncation in place of rounding inside the matrix unit). An activation is
evaluated in fp32 to 2^-20 (1 + |z|) of its magnitude (exp and the reciprocal
of the hardware are good to an ulp; an argument's rounding moves exp by
|z| u), and passes on an error of its argument times its largest slope (1.13
for SiLU and GELU); its derivative's own slope is at most 0.8.
"""

import math

import torch

U = 2.0 ** -24
F = torch.float64


def unit(dtype):
    return 2.0 ** -8 if dtype == torch.bfloat16 else U


def act(z, kind):
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "gelu":
        return z * 0.5 * torch.erfc(-z / math.sqrt(2.0))
    return z


def slope(z, kind):
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s + z * s * (1 - s)
    if kind == "relu":
        return (z > 0).to(F)
    if kind == "gelu":
        return 0.5 * torch.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-z * z / 2) / math.sqrt(
            2 * math.pi)
    return torch.ones_like(z)


def product(a, b, ea=None, eb=None):
    """(a b, bound) for fp32 sums, given bounds on a's and b's entries."""
    k = a.shape[1]
    mag = a.abs() @ b.abs()
    err = 2 * (k + 4) * U * mag
    if ea is not None:
        err = err + ea @ b.abs()
    if eb is not None:
        err = err + a.abs() @ eb
    if ea is not None and eb is not None:
        err = err + ea @ eb
    return a @ b, err


def act_err(z, ez, kind):
    a = act(z, kind)
    if kind == "identity":
        return a, ez
    return a, 1.13 * ez + 2.0 ** -20 * (1 + z.abs()) * (a.abs() + ez)


def slope_err(z, ez, kind):
    s = slope(z, kind)
    if kind == "identity":
        return s, torch.zeros_like(z)
    if kind == "relu":  # a jump at zero
        return s, (z.abs() <= ez).to(F)
    return s, 0.8 * ez + 2.0 ** -20 * (1 + z.abs()) * (s.abs() + 1)


def rounded(v, e, dtype):
    """The bound after a rounding to `dtype`; the smallest bf16 and fp32 steps
    near zero are below 1e-38."""
    return e + unit(dtype) * (v.abs() + e) + 1e-37


def linear(x, w, b, kind, res, dtype):
    z, ez = product(x, w)
    if b is not None:
        z = z + b
        ez = ez + 2 * U * (z.abs() + b.abs())
    a, ea = act_err(z, ez, kind)
    out = a if res is None else a + res
    return (z, ez), (out, rounded(out, ea + U * out.abs(), dtype))


def linear_bwd(dy, x, w, z, ez, kind, dtype):
    """Gradients, the pre-activation kept in `dtype`."""
    if kind == "identity":
        dz, edz = dy, torch.zeros_like(dy)
    else:
        s, es = slope_err(z, rounded(z, ez, dtype), kind)
        dz = dy * s
        edz = rounded(dz, dy.abs() * es + 2 * U * dz.abs(), dtype)
    dx, edx = product(dz, w.t().contiguous(), edz)
    dw, edw = product(x.t().contiguous(), dz, None, edz)
    n = dy.shape[0]
    db, edb = dz.sum(0), edz.sum(0) + 2 * (n + 4) * U * dz.abs().sum(0)
    if kind != "identity" and dtype == torch.bfloat16:
        pass  # the bias' sum takes d_z before its rounding: inside the same bound
    return {"d_x": (dx, rounded(dx, edx, dtype)), "d_weight": (dw, rounded(dw, edw, dtype)),
            "d_bias": (db, rounded(db, edb, dtype))}


def ffn(x, wg, wu, wd, kind, res, dtype):
    (g, eg), (u, eu) = product(x, wg), product(x, wu)
    a, ea = act_err(g, eg, kind)
    h = a * u
    eh = rounded(h, ea * u.abs() + a.abs() * eu + ea * eu + 2 * U * h.abs(), dtype)
    o, eo = product(h, wd, eh)
    out = o if res is None else o + res
    return {"out": (out, rounded(out, eo + U * out.abs(), dtype)),
            "gate": (g, rounded(g, eg, dtype)), "up": (u, rounded(u, eu, dtype))}


def ffn_bwd(dy, x, wg, wu, wd, kind, dtype):
    (g, eg), (u, eu) = product(x, wg), product(x, wu)
    eg, eu = rounded(g, eg, dtype), rounded(u, eu, dtype)  # as they are kept
    dh, edh = product(dy, wd.t().contiguous())
    a, ea = act_err(g, eg, kind)
    s, es = slope_err(g, eg, kind)

    def mul(p, ep, q, eq):
        return p * q, ep * q.abs() + p.abs() * eq + ep * eq + 2 * U * (p * q).abs()

    dhu, edhu = mul(dh, edh, u, eu)
    dg, edg = mul(dhu, edhu, s, es)
    du, edu = mul(dh, edh, a, ea)
    h, eh = mul(a, ea, u, eu)
    edg, edu, eh = rounded(dg, edg, dtype), rounded(du, edu, dtype), rounded(h, eh, dtype)
    dx1, e1 = product(dg, wg.t().contiguous(), edg)
    dx2, e2 = product(du, wu.t().contiguous(), edu)
    dx = dx1 + dx2
    out = {"d_x": (dx, rounded(dx, e1 + e2 + U * dx.abs(), dtype))}
    xt = x.t().contiguous()
    for name, (v, e) in {"d_w_gate": product(xt, dg, None, edg),
                         "d_w_up": product(xt, du, None, edu),
                         "d_w_down": product(h.t().contiguous(), dy, eh.t().contiguous())}.items():
        out[name] = (v, rounded(v, e, dtype))
    return out


def norm(x, res, w, eps, dtype):
    """sum, out, and the unrounded out with its bound."""
    s = x if res is None else x + res
    n = s.shape[1]
    es = U * s.abs()
    inv = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + eps)
    y = s * inv * w
    # The mean of squares is off by (n + 6)u of itself (its terms are positive),
    # so inv by half of that and its own rounding.
    ey = (2 * (n + 6) * U + 8 * U) * y.abs()
    return (s, rounded(s, es, dtype)), (y, rounded(y, ey, dtype)), (y, ey)


def norm_bwd(s, w, dy, ds, eps, dtype, wdtype):
    n, rows = s.shape[1], s.shape[0]
    inv = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + eps)
    unit_s = s * inv
    k = 2 * (n + 6) * U + 12 * U
    dot = (dy * w * unit_s).abs().mean(1, keepdim=True)
    dx = inv * (dy * w - unit_s * (dy * w * unit_s).mean(1, keepdim=True))
    edx = k * inv * ((dy * w).abs() + 3 * unit_s.abs() * dot)
    if ds is not None:
        dx = dx + ds
        edx = edx + U * dx.abs()
    dw = (dy * unit_s).sum(0)
    edw = (k + 2 * (rows + 4) * U) * (dy * unit_s).abs().sum(0)
    return {"d_x": (dx, rounded(dx, edx, dtype)), "d_weight": (dw, rounded(dw, edw, wdtype))}


def check(got, ref, what):
    value, bound = ref
    assert tuple(got.shape) == tuple(value.shape), f"{what}: {got.shape} {value.shape}"
    if got.numel() == 0:
        return
    d = (got.to(F) - value).abs()
    bad = ~(d <= bound)
    if bad.any():
        i = int((d / bound).nan_to_num(math.inf).argmax())
        raise AssertionError(
            f"{what}: {int(bad.sum())} of {got.numel()} outside the bound; at {i}: "
            f"{got.flatten()[i].item()} for {value.flatten()[i].item()}, "
            f"bound {bound.flatten()[i].item()}")
