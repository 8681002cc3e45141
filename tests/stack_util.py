"""Plain implementations in float64 of block_norm, embedding and attention, with
elementwise bounds as in layer_util.

Attention's bounds. A score c q·k is a product of D terms, in fp32; an exponential
passes on its argument's error as a relative one and adds 2^-20 (1 + |s|) of its own
(the argument's rounding included). A weight for the matrix unit is rounded to the
tensors' type, so a sum of weights times values is off by that unit of its terms'
magnitudes; the sum of the weights is not rounded. Gradients follow from the same
products (layer_util.product) with the errors of their factors.
"""

import math

import torch

from layer_util import F, U, product, rounded, unit


def rms(z, eps):
    return 1 / torch.sqrt((z * z).mean(1, keepdim=True) + eps)


def block_norm(x, r, pre, post, gate, scale, eps, dtype):
    """sum and out, each with its bound; gate broadcasts to x."""
    n = x.shape[1]
    k = 2 * (n + 6) * U + 8 * U
    u = x if post is None else x * rms(x, eps) * post
    eu = torch.zeros_like(u) if post is None else k * u.abs()
    g = torch.ones_like(x[:, :1]) if gate is None else gate
    s = scale * r + g * u
    es = g.abs() * eu + 4 * U * ((scale * r).abs() + (g * u).abs())
    inv = rms(s, eps)
    y = s * inv * pre
    moved = (s.abs() * es).sum(1, keepdim=True) / ((s * s).sum(1, keepdim=True) + n * eps)
    ey = (inv * pre).abs() * es + y.abs() * (moved + k)
    return (s, rounded(s, es, dtype)), (y, rounded(y, ey, dtype))


def block_norm_bwd(x, s, pre, post, gate, scale, dy, de, eps, dtype, wdtype, kind):
    rows, n = x.shape
    k = 2 * (n + 6) * U + 12 * U
    g = torch.ones_like(x[:, :1]) if gate is None else gate
    inv = rms(s, eps)
    w, d = s * inv, dy * pre
    ds = inv * (d - w * (d * w).mean(1, keepdim=True))
    eds = k * inv * (d.abs() + 3 * w.abs() * (d * w).abs().mean(1, keepdim=True))
    ds, eds = ds + de, eds + 2 * U * (ds + de).abs()
    inv_x = rms(x, eps) if post is not None else torch.ones_like(inv)
    p = post if post is not None else torch.ones_like(x[0])
    nx = x * inv_x
    kx = k if post is not None else 0.0
    u, eu = nx * p, (kx + 2 * U) * (nx * p).abs()
    dg = ds * u
    edg = eds * u.abs() + ds.abs() * eu + eds * eu + 2 * U * dg.abs()
    e = ds * g * p
    ee = eds * (g * p).abs() + 3 * U * e.abs()
    if post is None:
        dx, edx = e, ee
    else:
        dx = inv_x * (e - nx * (e * nx).mean(1, keepdim=True))
        edx = (inv_x * (ee + nx.abs() * (ee * nx.abs()).mean(1, keepdim=True))
               + 2 * k * inv_x * (e.abs() + 3 * nx.abs() * (e * nx).abs().mean(1, keepdim=True)))
    out = {"d_x": (dx, rounded(dx, edx, dtype)),
           "d_residual": (scale * ds, rounded(scale * ds, abs(scale) * eds + U * (scale * ds).abs(),
                                              dtype))}
    col = 2 * (rows + 4) * U

    def column(v, ev, to):
        t = v.sum(0)
        return t, rounded(t, ev.sum(0) + col * v.abs().sum(0), to)

    out["d_pre_weight"] = column(dy * w, k * (dy * w).abs(), wdtype)
    if post is not None:
        v = ds * g * nx
        out["d_post_weight"] = column(v, eds * (g * nx).abs() + k * v.abs(), wdtype)
    if kind == "channel":
        out["d_gate"] = column(dg, edg, wdtype)
    elif kind == "token":
        t = dg.sum(1, keepdim=True)
        out["d_gate"] = (t, rounded(t, edg.sum(1, keepdim=True) + 2 * (n + 4) * U
                                    * dg.abs().sum(1, keepdim=True), dtype))
    elif kind == "full":
        out["d_gate"] = (dg, rounded(dg, edg, dtype))
    return out


def embedding(ids, table, scale, dtype):
    there = (ids >= 0) & (ids < table.shape[0])
    v = torch.where(there[:, None], table[ids.clamp(0, table.shape[0] - 1)] * scale,
                    torch.zeros_like(table[:1]))
    return v, rounded(v, U * v.abs(), dtype)


def embedding_bwd(ids, d_out, vocab, scale, dtype):
    there = (ids >= 0) & (ids < vocab)
    at = ids[there]
    zeros = torch.zeros(vocab, d_out.shape[1], dtype=F, device=d_out.device)
    v = zeros.index_add(0, at, d_out[there]) * scale
    mag = zeros.index_add(0, at, d_out[there].abs()) * abs(scale)
    count = torch.bincount(at, minlength=vocab)[:, None].to(F)
    return v, rounded(v, 2 * (count + 4) * U * mag, dtype)


def head(q, k, v, scale, causal, dtype):
    """One head of one sequence: n queries over m keys, the last query at the last key.
    out, lse, P and what P's entries and scores are off by."""
    n, m, d = q.shape[0], k.shape[0], q.shape[1]
    s, es = product(q, k.t().contiguous())
    s, es = s * scale, es * scale + 2 * U * (s * scale).abs()
    seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
    if causal:
        seen = seen.tril(m - n)
    rel = torch.where(seen, es + 2.0 ** -20 * (1 + s.abs()), torch.zeros_like(s))
    top = rel.amax(1, keepdim=True) if m else rel.new_zeros(n, 1)
    masked = s.masked_fill(~seen, -math.inf)
    some = seen.any(1, keepdim=True)
    lse = torch.logsumexp(masked, 1, keepdim=True) if m else q.new_full((n, 1), -math.inf)
    p = torch.where(some & seen, torch.exp(masked - torch.where(some, lse, torch.zeros_like(lse))),
                    torch.zeros_like(s))
    # exp's argument is taken against the maximum: its rounding goes with |s − max|.
    r = unit(dtype) if dtype == torch.bfloat16 else 0.0
    out = p @ v
    eo = (r + 3 * top + 4 * (m + 8) * U) * (p @ v.abs())
    elses = top + 2 * (m + 8) * U + 4 * U * torch.where(some, lse.abs(), torch.zeros_like(lse))
    return {"out": out, "eo": rounded(out, eo, dtype), "lse": lse, "elses": elses, "p": p,
            "rel": rel, "scores": s}


def head_bwd(q, k, v, do, scale, f, dtype):
    p, out = f["p"], f["out"]
    n, m, d = q.shape[0], k.shape[0], q.shape[1]
    # The forward's lse enters P, its out (rounded) enters delta.
    ep = p * (f["rel"] + f["elses"] + 2.0 ** -20 * (1 + f["lse"].abs().nan_to_num(posinf=0.0)))
    dp, edp = product(do, v.t().contiguous())
    delta = (do * out).sum(1, keepdim=True)
    edelta = ((do.abs() * f["eo"]).sum(1, keepdim=True)
              + 2 * (d + 4) * U * (do * out).abs().sum(1, keepdim=True))
    ds = p * (dp - delta)
    eds = (ep * (dp - delta).abs() + (p + ep) * (edp + edelta) + 4 * U * p * (dp.abs() + delta.abs()))
    pr, dsr = rounded(p, ep, dtype), rounded(ds, eds, dtype)
    dv, edv = product(p.t().contiguous(), do, pr.t().contiguous())
    dq, edq = product(ds, k, dsr)
    dk, edk = product(ds.t().contiguous(), q, dsr.t().contiguous())
    return {"d_q": (dq * scale, edq * scale), "d_k": (dk * scale, edk * scale), "d_v": (dv, edv)}


def attention(q, k, v, spans, scale, causal, dtype, do=None):
    """q [rows, heads, dim] and so on in float64; spans: (first query row, queries, first
    key row, keys) of every sequence. Values with bounds of out, lse and the gradients."""
    heads, kv = q.shape[1], k.shape[1]
    scale = q.shape[2] ** -0.5 if scale is None else scale
    zero = torch.zeros_like
    got = {"out": (zero(q), zero(q)), "lse": (zero(q[..., 0]) - math.inf, zero(q[..., 0]))}
    if do is not None:
        got.update({"d_q": (zero(q), zero(q)), "d_k": (zero(k), zero(k)),
                    "d_v": (zero(v), zero(v))})
    for q0, n, k0, m in spans:
        for h in range(heads if n else 0):
            g = h // (heads // kv)
            rows, keys = slice(q0, q0 + n), slice(k0, k0 + m)
            args = (q[rows, h].contiguous(), k[keys, g].contiguous(), v[keys, g].contiguous())
            f = head(*args, scale, causal, dtype)
            got["out"][0][rows, h], got["out"][1][rows, h] = f["out"], f["eo"]
            got["lse"][0][rows, h] = f["lse"][:, 0]
            got["lse"][1][rows, h] = f["elses"][:, 0]
            if do is None:
                continue
            b = head_bwd(*args, do[rows, h].contiguous(), scale, f, dtype)
            got["d_q"][0][rows, h], got["d_q"][1][rows, h] = b["d_q"]
            for name in ("d_k", "d_v"):
                got[name][0][keys, g] += b[name][0]
                got[name][1][keys, g] += b[name][1]
    for name in ("d_q", "d_k", "d_v"):
        if name in got:
            value, bound = got[name]
            # A group's heads and the rows are one fp32 sum.
            got[name] = (value, rounded(value, 2 * bound, dtype))
    return got
