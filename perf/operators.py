"""The operators around a delta-rule mixer in a decoder layer: the cases whose
speed is watched, one pass of each, and their values in 64 bits.

A case is a dict; `op` names the operator and `mode` how it is used.

  norm         residual addition and root-mean-square norm.
               "fwd": add_rms_norm; "8bit": the same with its output in 8 bits
               and one scale a row (add_rms_norm_8bit); "train": the forward
               and its gradients (add_rms_norm_backward)
  linear       act(x W + bias) + residual. "fwd": linear; "train": the forward
               and its gradients (linear_forward, linear_backward)
  linear_8bit  the same product from operands held in 8 bits with one scale a
               row (linear_8bit)
  ffn          (act(x Wg) * (x Wu)) Wd + residual. "fwd": gated_ffn; "train":
               the forward and its gradients (gated_ffn_forward,
               gated_ffn_backward)

Sizes: `rows` tokens; `dim` is the model width (a linear's input), `out` a
linear's output, `hidden` the feed-forward width.
"""

import importlib
import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-5
F8 = torch.float8_e4m3fn
F8_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _norm(name, mode, rows, dim, dtype="bf16", residual=True):
    case = {"op": "norm", "mode": mode, "rows": rows, "dim": dim, "dtype": dtype,
            "residual": residual}
    return {"name": name, **case} if name else case


def _linear(name, mode, rows, dim, out, dtype="bf16", act="identity", bias=False, residual=False):
    case = {"op": "linear", "mode": mode, "rows": rows, "dim": dim, "out": out, "dtype": dtype,
            "act": act, "bias": bias, "residual": residual}
    return {"name": name, **case} if name else case


def _linear_8bit(name, rows, dim, out, dtype="bf16", act="identity", bias=False, residual=False):
    case = {"op": "linear_8bit", "mode": "fwd", "rows": rows, "dim": dim, "out": out,
            "dtype": dtype, "act": act, "bias": bias, "residual": residual}
    return {"name": name, **case} if name else case


def _ffn(name, mode, rows, dim, hidden, dtype="bf16", act="silu", residual=True):
    case = {"op": "ffn", "mode": mode, "rows": rows, "dim": dim, "hidden": hidden, "dtype": dtype,
            "act": act, "residual": residual}
    return {"name": name, **case} if name else case


def listed():
    # The model width is 16 heads of 128 keys; a Gated DeltaNet layer's input
    # projection has 2048 + 2048 + 4096 + 16 + 4096 columns (q, k, v, beta and
    # the output gate), its output projection 16 heads of 256 values as input.
    return [
        # One decoded token for each of a large batch, handed to an 8-bit product.
        _norm("norm_8bit_256", "8bit", 256, 2048),
        # Training over a batch of long sequences: all traffic.
        _norm("norm_train_32768", "train", 32768, 2048),
        # The input projection over a prompt of two sequences.
        _linear("in_proj_8192", "fwd", 8192, 2048, 12304),
        # The output projection onto the residual stream, in training.
        _linear("out_proj_train_16384", "train", 16384, 4096, 2048, residual=True),
        # The input projection of one decoded token: the weight's traffic.
        _linear("in_proj_1", "fwd", 1, 2048, 12304),
        # A small float32 layer in training, of no round size, with everything on.
        _linear("linear_f32_train_500", "train", 500, 256, 1039, "f32", "silu", True, True),
        # The output projection over a prompt from 8-bit operands.
        _linear_8bit("out_proj_8bit_4096", 4096, 4096, 2048, residual=True),
        # The input projection of one decoded token for each of a large batch.
        _linear_8bit("in_proj_8bit_256", 256, 2048, 12304),
        # The feed-forward block of one decoded token.
        _ffn("ffn_1", "fwd", 1, 2048, 5632),
        # The same for a large batch of them.
        _ffn("ffn_256", "fwd", 256, 2048, 5632),
        # Training over a batch of long sequences: the largest.
        _ffn("ffn_train_16384", "train", 16384, 2048, 5632),
        # Training in float32 at a small width, ragged (8/3 of 256 is no round number).
        _ffn("ffn_f32_train_1000", "train", 1000, 256, 683, "f32"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """A width: most are multiples of 64 or 16, as models have them, the rest of any size."""
    n, r = _log(rng, low, high), rng.random()
    return n if r < 0.3 else max(16, n // 16 * 16) if r < 0.5 else max(64, n // 64 * 64)


def draw(rng):
    op = rng.choice(["norm", "linear", "linear_8bit", "ffn"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    rows = _log(rng, 1, 32768)
    if op == "norm":
        dim = _width(rng, 64, 8192)
        rows = min(rows, (32768 * 2048) // (dim * (2 if dtype == "f32" else 1)))
        return _norm(None, rng.choice(["fwd", "8bit", "train"]), rows, dim, dtype,
                     rng.random() < 0.7)
    # The largest listed training pass has 3.4e12 operations; in float32 they
    # take about twenty times as long.
    most = 1.5e11 if dtype == "f32" and op != "linear_8bit" else 2e12
    dim = _width(rng, 64, 4096)
    if op == "ffn":
        mode, hidden = rng.choice(["fwd", "train"]), _width(rng, 128, 8192)
        rows = max(1, min(rows, int(most / (18.0 * dim * hidden))))
        return _ffn(None, mode, rows, dim, hidden, dtype, rng.choice(["silu", "silu", "gelu", "relu"]),
                    rng.random() < 0.7)
    out = _width(rng, 64, 12304)
    rows = max(1, min(rows, int(most / (6.0 * dim * out))))
    act = rng.choice(["identity", "identity", "silu", "relu", "gelu"])
    bias, residual = rng.random() < 0.4, rng.random() < 0.4
    if op == "linear_8bit":
        return _linear_8bit(None, rows, dim, out, dtype, act, bias, residual)
    return _linear(None, rng.choice(["fwd", "train"]), rows, dim, out, dtype, act, bias, residual)


def _codes(x):
    """Rows in 8 bits with a scale each, in storage whose rows are padded with
    zeros to 16 bytes: what a program keeps of its weights."""
    scale = x.abs().amax(1).clamp_min(1e-12) / F8_MAX
    rows, dim = x.shape
    store = torch.zeros(rows, (dim + 15) // 16 * 16, dtype=torch.uint8, device=x.device).view(F8)
    store[:, :dim].copy_((x / scale[:, None]).to(F8))
    return store[:, :dim], scale


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    op, rows, dim, dtype = case["op"], case["rows"], case["dim"], DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0, as_dtype=dtype):
        return (torch.randn(*shape, generator=gen, device=DEVICE) * scale + mean).to(as_dtype)

    s = dict(case)
    train = case["mode"] == "train"
    if op == "norm":
        s["x"] = normal(rows, dim)
        s["residual"] = normal(rows, dim, scale=2.0) if case["residual"] else None
        s["weight"] = normal(dim, scale=0.1, mean=1.0)
        if train:
            s["d_out"], s["d_sum"] = normal(rows, dim), normal(rows, dim)
    elif op == "linear_8bit":
        out = case["out"]
        s["x"], s["x_scale"] = _codes(normal(rows, dim, as_dtype=torch.float32))
        s["weight"], s["weight_scale"] = _codes(
            normal(out, dim, scale=dim ** -0.5, as_dtype=torch.float32))
        s["bias"] = normal(out, scale=0.1) if case["bias"] else None
        s["residual"] = normal(rows, out) if case["residual"] else None
    elif op == "linear":
        out = case["out"]
        s["x"] = normal(rows, dim)
        s["weight"] = normal(dim, out, scale=dim ** -0.5)
        s["bias"] = normal(out, scale=0.1) if case["bias"] else None
        s["residual"] = normal(rows, out) if case["residual"] else None
        if train:
            s["d_out"] = normal(rows, out)
    else:
        hidden = case["hidden"]
        s["x"] = normal(rows, dim)
        s["w_gate"] = normal(dim, hidden, scale=dim ** -0.5)
        s["w_up"] = normal(dim, hidden, scale=dim ** -0.5)
        s["w_down"] = normal(hidden, dim, scale=hidden ** -0.5)
        s["residual"] = normal(rows, dim) if case["residual"] else None
        if train:
            s["d_out"] = normal(rows, dim)
    return s


# -- the framework's operators ---------------------------------------------------

def _run_own(s):
    dn = importlib.import_module("burn-deltanet_amd")
    op, train = s["op"], s["mode"] == "train"
    if op == "norm":
        if s["mode"] == "8bit":
            rows8, total = dn.add_rms_norm_8bit(s["x"], s["residual"], s["weight"], EPS)
            return {"codes": rows8.codes, "scale": rows8.scale, **_some(sum=total, on=s["residual"])}
        out, total = dn.add_rms_norm(s["x"], s["residual"], s["weight"], EPS)
        got = {"out": out, **_some(sum=total, on=s["residual"])}
        if train:
            got["d_x"], got["d_weight"] = dn.add_rms_norm_backward(s["d_out"], s["d_sum"], total,
                                                                   s["weight"], EPS)
        return got
    act = dn.Activation[s["act"].upper()]
    if op == "linear_8bit":
        return {"out": dn.linear_8bit(dn.Rows8(s["x"], s["x_scale"]),
                                      dn.Rows8(s["weight"], s["weight_scale"]), s["bias"], act,
                                      s["residual"], DTYPES[s["dtype"]])}
    if op == "linear":
        if not train:
            return {"out": dn.linear(s["x"], s["weight"], s["bias"], act, s["residual"])}
        out, preact = dn.linear_forward(s["x"], s["weight"], s["bias"], act, s["residual"])
        g = dn.linear_backward(s["d_out"], s["x"], s["weight"], preact, act,
                               bias=s["bias"] is not None)
        return {"out": out, "d_x": g.d_x, "d_weight": g.d_weight,
                **_some(d_bias=g.d_bias, on=s["bias"])}
    if not train:
        return {"out": dn.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["w_down"], act,
                                    s["residual"])}
    out, gate, up = dn.gated_ffn_forward(s["x"], s["w_gate"], s["w_up"], s["w_down"], act,
                                         s["residual"])
    g = dn.gated_ffn_backward(s["d_out"], s["x"], s["w_gate"], s["w_up"], s["w_down"], gate, up,
                              act)
    return {"out": out, "d_x": g.d_x, "d_w_gate": g.d_w_gate, "d_w_up": g.d_w_up,
            "d_w_down": g.d_w_down}


def _some(on, **values):
    """The outputs that there are only where an optional input is."""
    return {} if on is None else values


# -- the plain forms ---------------------------------------------------------------

def _act(z, kind):
    if kind == "silu":
        return z / (1.0 + torch.exp(-z))
    if kind == "relu":
        return torch.clamp_min(z, 0.0)
    if kind == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_grad(z, kind):
    if kind == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        return p * (1.0 + z * (1.0 - p))
    if kind == "relu":
        return (z > 0).float()
    if kind == "gelu":
        return (0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
                + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi)))
    return torch.ones_like(z)


def _float(t):
    return None if t is None else t.float()


def _plain_norm(s):
    dtype = s["x"].dtype
    x, weight = s["x"].float(), s["weight"].float()
    total = x if s["residual"] is None else x + s["residual"].float()
    inv = torch.rsqrt((total * total).mean(1, keepdim=True) + EPS)
    unit = total * inv
    out = unit * weight
    got = {} if s["residual"] is None else {"sum": total.to(dtype)}
    if s["mode"] == "8bit":
        scale = out.abs().amax(1) * (1.0 / F8_MAX)
        codes = torch.where(scale[:, None] > 0, out / scale[:, None], out)
        return {"codes": codes.to(F8), "scale": scale, **got}
    got["out"] = out.to(dtype)
    if s["mode"] == "train":
        d_out = s["d_out"].float()
        d_unit = d_out * weight
        d_x = inv * (d_unit - unit * (d_unit * unit).mean(1, keepdim=True)) + s["d_sum"].float()
        got["d_x"], got["d_weight"] = d_x.to(dtype), (d_out * unit).sum(0).to(s["weight"].dtype)
    return got


def _plain_linear(s):
    dtype = DTYPES[s["dtype"]]
    if s["op"] == "linear_8bit":
        x, weight = s["x"].float(), s["weight"].float().t()
        z = (x @ weight) * s["x_scale"][:, None] * s["weight_scale"]
    else:
        x, weight = s["x"].float(), s["weight"].float()
        z = x @ weight
    if s["bias"] is not None:
        z = z + s["bias"].float()
    out = _act(z, s["act"])
    if s["residual"] is not None:
        out = out + s["residual"].float()
    got = {"out": out.to(dtype)}
    if s["mode"] == "train":
        d_z = s["d_out"].float()
        if s["act"] != "identity":
            d_z = d_z * _act_grad(z, s["act"])
        got["d_x"], got["d_weight"] = (d_z @ weight.t()).to(dtype), (x.t() @ d_z).to(dtype)
        if s["bias"] is not None:
            got["d_bias"] = d_z.sum(0).to(dtype)
    return got


def _plain_ffn(s):
    dtype = s["x"].dtype
    x, w_gate, w_up, w_down = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    gate, up = x @ w_gate, x @ w_up
    active = _act(gate, s["act"])
    h = active * up
    out = h @ w_down
    if s["residual"] is not None:
        out = out + s["residual"].float()
    got = {"out": out.to(dtype)}
    if s["mode"] == "train":
        d_out = s["d_out"].float()
        d_h = d_out @ w_down.t()
        d_gate, d_up = d_h * up * _act_grad(gate, s["act"]), d_h * active
        got["d_x"] = (d_gate @ w_gate.t() + d_up @ w_up.t()).to(dtype)
        got["d_w_gate"] = (x.t() @ d_gate).to(dtype)
        got["d_w_up"] = (x.t() @ d_up).to(dtype)
        got["d_w_down"] = (h.t() @ d_out).to(dtype)
    return got


def run(state):
    if own:
        return _run_own(state)
    return {"norm": _plain_norm, "ffn": _plain_ffn}.get(state["op"], _plain_linear)(state)


# -- values in 64 bits ---------------------------------------------------------------

def _exact_act(z, kind):
    f = torch.nn.functional
    return {"silu": f.silu, "relu": f.relu, "gelu": f.gelu}.get(kind, lambda t: t)(z)


def exact(case, seed):
    """The definitions in float64, the gradients by torch's differentiation of them."""
    s = prepare(case, seed)
    train = s["mode"] == "train"

    def leaf(key):
        return None if s.get(key) is None else s[key].double().requires_grad_(train)

    if s["op"] == "norm":
        x, residual, weight = leaf("x"), leaf("residual"), leaf("weight")
        total = x if residual is None else x + residual
        out = total / (total.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * weight
        got = {"sum": total.detach()} if residual is not None else {}
        if s["mode"] == "8bit":
            scale = out.abs().amax(-1) / F8_MAX
            return {"codes": out / scale.unsqueeze(-1), "scale": scale, **got}
        got["out"] = out.detach()
        if train:
            d = torch.autograd.grad((out, total) if residual is not None else (out,), (x, weight),
                                    (s["d_out"].double(), s["d_sum"].double())
                                    if residual is not None else (s["d_out"].double(),))
            # Without a residual the sum is the input, whose own cotangent is added.
            got["d_x"] = d[0] if residual is not None else d[0] + s["d_sum"].double()
            got["d_weight"] = d[1]
        return got
    if s["op"] == "ffn":
        leaves = [leaf(k) for k in ("x", "w_gate", "w_up", "w_down")]
        x, w_gate, w_up, w_down = leaves
        out = torch.mm(_exact_act(torch.mm(x, w_gate), s["act"]) * torch.mm(x, w_up), w_down)
        names = ("d_x", "d_w_gate", "d_w_up", "d_w_down")
    else:
        x, weight, bias = leaf("x"), leaf("weight"), leaf("bias")
        if s["op"] == "linear_8bit":
            z = torch.mm(x * s["x_scale"].double().unsqueeze(1),
                         (weight * s["weight_scale"].double().unsqueeze(1)).t())
        else:
            z = torch.mm(x, weight)
        out = _exact_act(z if bias is None else z + bias, s["act"])
        leaves = [x, weight] + ([] if bias is None else [bias])
        names = ("d_x", "d_weight", "d_bias")
    got = {"out": (out if s["residual"] is None else out + s["residual"].double()).detach()}
    if train:
        got.update(zip(names, torch.autograd.grad(out, leaves, s["d_out"].double())))
    return got


def work(case):
    op, rows, dim, train = case["op"], case["rows"], case["dim"], case["mode"] == "train"
    size = 4 if case["dtype"] == "f32" else 2
    if op == "norm":
        n = rows * dim
        streams = 2 + 2 * case["residual"]  # x, out; residual, sum
        if case["mode"] == "8bit":
            return {"bytes": n * ((streams - 1) * size + 1) + 4 * rows + dim * size, "flops": 6 * n}
        if train:  # d_out, d_sum, d_x
            return {"bytes": n * (streams + 3) * size + 2 * dim * size, "flops": 16 * n}
        return {"bytes": n * streams * size + dim * size, "flops": 6 * n}
    if op == "ffn":
        hidden = case["hidden"]
        weights = 3 * dim * hidden
        streams = 2 + case["residual"] + 2 * train  # x, out, residual; d_out, d_x
        return {"bytes": (rows * dim * streams + weights * (2 if train else 1)) * size,
                "flops": rows * weights * (6.0 if train else 2.0)}
    out = case["out"]
    in_size = 1 if op == "linear_8bit" else size
    count = rows * dim * in_size + dim * out * in_size
    count += (rows * out * (1 + case["residual"]) + out * case["bias"]) * size
    if op == "linear_8bit":
        count += 4 * (rows + out)
    if train:  # d_out; d_x, d_weight, d_bias
        count += (rows * out + rows * dim + dim * out + out * case["bias"]) * size
    return {"bytes": count, "flops": rows * dim * out * (6.0 if train else 2.0)}
