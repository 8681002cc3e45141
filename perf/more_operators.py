"""The operators of a decoder stack between its token ids and its logits, beside
the delta-rule mixer and the operators around it: the cases whose speed is
watched, one pass of each, and their values in 64 bits.

A case is a dict; `op` names the operator and `mode` how it is used.

  block_norm   a block's output joins the residual stream: norm after the block,
               its gate, the scaled residual, norm before the next block.
               "fwd": block_norm; "train": the forward and its gradients
  embedding    rows of a table by token id, scaled. "fwd": embedding; "train":
               the forward and the table's gradient
  attention    softmax attention with grouped heads. "prompt": whole packed
               sequences, causal; "train": the same and its gradients; "cache":
               the last `new` tokens of every sequence over its cached keys

Sizes: `rows` or `tokens` rows of the batch; `dim` a row's width, of a head for
attention; `sequences` of different lengths that add up to `tokens`, with
`padding` rows behind them.
"""

import importlib
import math
import random

import torch

own = False

DEVICE = "cuda"
EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _block_norm(name, mode, rows, dim, dtype="bf16", gate="channel", post=True, scale=1.0):
    case = {"op": "block_norm", "mode": mode, "rows": rows, "dim": dim, "dtype": dtype,
            "gate": gate, "post": post, "scale": scale}
    return {"name": name, **case} if name else case


def _embedding(name, mode, tokens, vocab, dim, dtype="bf16", scale=1.0):
    case = {"op": "embedding", "mode": mode, "tokens": tokens, "vocab": vocab, "dim": dim,
            "dtype": dtype, "scale": scale}
    return {"name": name, **case} if name else case


def _attention(name, mode, tokens, sequences, heads, kv_heads, dim, dtype="bf16", padding=0):
    case = {"op": "attention", "mode": mode, "tokens": tokens, "sequences": sequences,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "padding": padding}
    return {"name": name, **case} if name else case


def _cache(name, sequences, new, cached, heads, kv_heads, dim, dtype="bf16"):
    case = {"op": "attention", "mode": "cache", "sequences": sequences, "new": new,
            "cached": cached, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype}
    return {"name": name, **case} if name else case


def listed():
    # The model width is 16 heads of 128, as the delta-rule layers have it; an
    # attention layer between them shares each key head among four query heads.
    return [
        # The joint of one decoded token: latency.
        _block_norm("block_norm_1", "fwd", 1, 2048),
        # Training over a batch of long sequences: all traffic.
        _block_norm("block_norm_train_32768", "train", 32768, 2048),
        # A small float32 stack in training, of no round size, a gate value a token and channel.
        _block_norm("block_norm_f32_train_777", "train", 777, 1039, "f32", "full", True, 0.5),
        # One decoded token for each of a large batch.
        _embedding("embedding_256", "fwd", 256, 50000, 2048),
        # Training: the gradient writes the whole table.
        _embedding("embedding_train_16384", "train", 16384, 50000, 2048, "bf16", 45.0),
        # The same in float32 at a small, ragged size.
        _embedding("embedding_f32_train_3001", "train", 3001, 1009, 200, "f32"),
        # Prompts of several requests, packed, in a batch rounded up.
        _attention("attention_prompt_16384", "prompt", 16300, 6, 16, 4, 128, padding=84),
        # A training batch of a few documents.
        _attention("attention_train_8192", "train", 8192, 4, 16, 4, 128),
        # One long document: the largest.
        _attention("attention_train_long_16384", "train", 16384, 1, 16, 4, 128),
        # One decoded token for each of 64 requests.
        _cache("attention_cache_64", 64, 1, 8192, 16, 4, 128),
        # One decoded token of one long request.
        _cache("attention_cache_1_long", 1, 1, 65536, 16, 4, 128),
        # A small float32 stack in training: odd lengths, a narrow head.
        _attention("attention_f32_train_1000", "train", 1000, 3, 6, 2, 40, "f32", padding=5),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """A width: most are multiples of 64 or 16, as models have them, the rest of any size."""
    n, r = _log(rng, low, high), rng.random()
    return n if r < 0.3 else max(16, n // 16 * 16) if r < 0.5 else max(64, n // 64 * 64)


def draw(rng):
    op = rng.choice(["block_norm", "embedding", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if op == "block_norm":
        dim = _width(rng, 64, 8192)
        rows = min(_log(rng, 1, 32768), (32768 * 2048) // (dim * (2 if dtype == "f32" else 1)))
        return _block_norm(None, rng.choice(["fwd", "train"]), rows, dim, dtype,
                           rng.choice(["none", "channel", "token", "full"]), rng.random() < 0.7,
                           rng.choice([1.0, round(rng.uniform(0.2, 1.5), 3)]))
    if op == "embedding":
        dim, vocab = _width(rng, 64, 4096), _log(rng, 300, 100000)
        vocab = min(vocab, 50000 * 2048 // dim)
        tokens = min(_log(rng, 1, 65536), 16384 * 4096 // dim)
        return _embedding(None, rng.choice(["fwd", "train"]), tokens, vocab, dim, dtype,
                          rng.choice([1.0, round(dim ** 0.5, 3)]))
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8])
    group = min(group, max(1, 16 // kv_heads))
    dim = rng.choice([64, 128, 128, 256, 96, 40, 72, 33])
    if rng.random() < 0.35:
        sequences = _log(rng, 1, 128)
        # The cache of every sequence, 2^31 bytes at most.
        most = (1 << 28) // (sequences * kv_heads * dim)
        return _cache(None, sequences, rng.choice([1, 1, 1, 2, 5, 33]),
                      max(40, min(_log(rng, 64, 65536), most)), kv_heads * group, kv_heads, dim,
                      dtype)
    mode = rng.choice(["prompt", "train"])
    tokens = _log(rng, 1, 16384)
    # The largest listed pass has 16 heads of 128; in float32 it would take ten times as long.
    if dtype == "f32":
        tokens = min(tokens, 4000)
    if dim > 128:
        tokens = min(tokens, 11000)
    return _attention(None, mode, tokens, min(tokens, _log(rng, 1, 32)), kv_heads * group, kv_heads,
                      dim, dtype, rng.choice([0, 0, 17]))


def _lengths(case):
    """How long the sequences are: a few long ones and many short ones, an empty
    one where there are many. With a cache, how many keys each has."""
    n = case["sequences"]
    if case["mode"] == "cache":
        rng = random.Random(1000003 * n + case["cached"])
        low = max(case["new"], case["cached"] // 4)
        return [case["cached"] if i == 0 else rng.randint(low, case["cached"]) for i in range(n)]
    rng = random.Random(1000003 * n + case["tokens"])
    shares = [rng.expovariate(1.0) + 0.05 for _ in range(n)]
    if n > 8:
        shares[n // 2] = 0.0
    total, at, cuts = sum(shares), 0.0, [0]
    for s in shares[:-1]:
        at += s
        cuts.append(int(case["tokens"] * at / total))
    cuts.append(case["tokens"])
    return [b - a for a, b in zip(cuts, cuts[1:])]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    op, dim, dtype = case["op"], case["dim"], DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0):
        return (torch.randn(*shape, generator=gen, device=DEVICE) * scale + mean).to(dtype)

    s = dict(case)
    train = case["mode"] == "train"
    if op == "block_norm":
        rows = case["rows"]
        s["x"], s["residual"] = normal(rows, dim, scale=1.5), normal(rows, dim, scale=2.0)
        s["pre_weight"] = normal(dim, scale=0.1, mean=1.0)
        s["post_weight"] = normal(dim, scale=0.1, mean=1.0) if case["post"] else None
        shape = {"none": None, "channel": (dim,), "token": (rows, 1), "full": (rows, dim)}
        shape = shape[case["gate"]]
        s["gate_value"] = None if shape is None else normal(*shape, scale=0.2, mean=0.7)
        if train:
            s["d_out"], s["d_sum"] = normal(rows, dim), normal(rows, dim)
    elif op == "embedding":
        tokens, vocab = case["tokens"], case["vocab"]
        # Ids as text has them, few of them often; every 50th or so is padding (-1).
        u = torch.rand(tokens, generator=gen, device=DEVICE)
        ids = (torch.exp(u * math.log(vocab)) - 1.0).long().clamp_(0, vocab - 1)
        pad = torch.rand(tokens, generator=gen, device=DEVICE) < 0.02
        s["ids"] = torch.where(pad, torch.full_like(ids, -1), ids)
        s["table"] = normal(vocab, dim)
        if train:
            s["d_out"] = normal(tokens, dim)
    else:
        heads, kv = case["heads"], case["kv_heads"]
        s["lengths"] = lengths = _lengths(case)
        if case["mode"] == "cache":
            n, new, cached = case["sequences"], case["new"], case["cached"]
            s["q"] = normal(n * new, heads, dim)
            s["k"], s["v"] = normal(n * cached, kv, dim), normal(n * cached, kv, dim)
            ints = torch.arange(n + 1, device=DEVICE, dtype=torch.int32)
            s["offsets"] = ints * new
            s["starts"] = ints[:-1] * cached
            s["counts"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
        else:
            rows = case["tokens"] + case["padding"]
            s["q"] = normal(rows, heads, dim)
            s["k"], s["v"] = normal(rows, kv, dim), normal(rows, kv, dim)
            ends = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
            s["offsets"] = torch.tensor(ends, dtype=torch.int32, device=DEVICE)
            if train:
                s["d_out"] = normal(rows, heads, dim)
    return s


# -- the framework's operators ---------------------------------------------------

def _run_own(s):
    dn = importlib.import_module("burn-deltanet_amd")
    op, train = s["op"], s["mode"] == "train"
    if op == "block_norm":
        out, total = dn.block_norm(s["x"], s["residual"], s["pre_weight"], s["post_weight"],
                                   s["gate_value"], s["scale"], EPS)
        got = {"out": out, "sum": total}
        if train:
            g = dn.block_norm_backward(s["d_out"], s["d_sum"], s["x"], total, s["pre_weight"],
                                       s["post_weight"], s["gate_value"], s["scale"], EPS)
            got.update(d_x=g.d_x, d_residual=g.d_residual, d_pre_weight=g.d_pre_weight,
                       **_some(on=s["post_weight"], d_post_weight=g.d_post_weight),
                       **_some(on=s["gate_value"], d_gate=g.d_gate))
        return got
    if op == "embedding":
        got = {"out": dn.embedding(s["ids"], s["table"], s["scale"])}
        if train:
            got["d_table"] = dn.embedding_backward(s["d_out"], s["ids"], s["vocab"], s["scale"])
        return got
    if s["mode"] == "cache":
        return {"out": dn.attention(s["q"], s["k"], s["v"], s["offsets"],
                                    dn.KeySpans(s["starts"], s["counts"]))}
    if not train:
        return {"out": dn.attention(s["q"], s["k"], s["v"], s["offsets"])}
    out, lse = dn.attention_forward(s["q"], s["k"], s["v"], s["offsets"])
    g = dn.attention_backward(s["d_out"], s["q"], s["k"], s["v"], out, lse, s["offsets"])
    return {"out": out, "d_q": g.d_q, "d_k": g.d_k, "d_v": g.d_v}


def _some(on, **values):
    """The outputs that there are only where an optional input is."""
    return {} if on is None else values


# -- the plain forms ---------------------------------------------------------------

def _float(t):
    return None if t is None else t.float()


def _plain_block_norm(s):
    dtype = s["x"].dtype
    x, residual, pre = s["x"].float(), s["residual"].float(), s["pre_weight"].float()
    post, gate = _float(s["post_weight"]), _float(s["gate_value"])
    u = x
    if post is not None:
        inv_x = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
        unit_x = x * inv_x
        u = unit_x * post
    total = s["scale"] * residual + (u if gate is None else gate * u)
    inv = torch.rsqrt((total * total).mean(1, keepdim=True) + EPS)
    unit = total * inv
    got = {"out": (unit * pre).to(dtype), "sum": total.to(dtype)}
    if s["mode"] != "train":
        return got
    d_out = s["d_out"].float()
    d_unit = d_out * pre
    d_total = inv * (d_unit - unit * (d_unit * unit).mean(1, keepdim=True)) + s["d_sum"].float()
    got["d_pre_weight"] = (d_out * unit).sum(0).to(dtype)
    got["d_residual"] = (s["scale"] * d_total).to(dtype)
    d_u = d_total
    if gate is not None:
        d_gate = d_total * u
        if gate.dim() == 1:
            d_gate = d_gate.sum(0)
        elif gate.shape[1] == 1 and u.shape[1] != 1:
            d_gate = d_gate.sum(1, keepdim=True)
        got["d_gate"] = d_gate.to(dtype)
        d_u = d_total * gate
    if post is not None:
        got["d_post_weight"] = (d_u * unit_x).sum(0).to(dtype)
        d_n = d_u * post
        d_u = inv_x * (d_n - unit_x * (d_n * unit_x).mean(1, keepdim=True))
    got["d_x"] = d_u.to(dtype)
    return got


def _plain_embedding(s):
    dtype, ids, vocab = s["table"].dtype, s["ids"], s["vocab"]
    there = (ids >= 0) & (ids < vocab)
    rows = s["table"][torch.where(there, ids, torch.zeros_like(ids))].float() * s["scale"]
    got = {"out": torch.where(there[:, None], rows, torch.zeros_like(rows)).to(dtype)}
    if s["mode"] == "train":
        # One row more takes what is padding.
        table = torch.zeros(vocab + 1, s["dim"], device=ids.device)
        table.index_add_(0, torch.where(there, ids, torch.full_like(ids, vocab)),
                         s["d_out"].float() * s["scale"])
        got["d_table"] = table[:vocab].to(dtype)
    return got


def _spans(s):
    """Of every sequence: its first query row, how many, its first key row, how many."""
    if s["mode"] == "cache":
        return [(i * s["new"], s["new"], i * s["cached"], m) for i, m in enumerate(s["lengths"])]
    at, spans = 0, []
    for n in s["lengths"]:
        spans.append((at, n, at, n))
        at += n
    return spans


def _plain_attention(s):
    q, k, v = s["q"], s["k"], s["v"]
    heads, kv, dim, train = s["heads"], s["kv_heads"], s["dim"], s["mode"] == "train"
    group, scale = heads // kv, 1.0 / math.sqrt(dim)
    new = lambda t: torch.zeros(t.shape, dtype=torch.float32, device=t.device)
    out = new(q)
    if train:
        d_q, d_k, d_v = new(q), new(k), new(v)
    for q0, n, k0, m in _spans(s):
        if n == 0 or m == 0:
            continue
        ks = k[k0:k0 + m].float().transpose(0, 1).contiguous()
        vs = v[k0:k0 + m].float().transpose(0, 1).contiguous()
        kt, vt = ks.transpose(1, 2).contiguous(), vs.transpose(1, 2).contiguous()
        # Query rows at a time, so that the scores stay within 2^29 values.
        step = max(1, (1 << 29) // (heads * m))
        for a in range(0, n, step):
            b = min(n, a + step)
            rows = slice(q0 + a, q0 + b)

            def grouped(t):  # [kv, group * rows, dim]
                return (t[rows].float().reshape(b - a, kv, group, dim).permute(1, 2, 0, 3)
                        .reshape(kv, group * (b - a), dim))

            def back(t):
                return t.reshape(kv, group, b - a, dim).permute(2, 0, 1, 3).reshape(b - a, heads, dim)

            qs = grouped(q)
            scores = torch.matmul(qs, kt) * scale
            last = torch.arange(a, b, device=q.device) + (m - n)
            hidden = torch.arange(m, device=q.device)[None, :] > last[:, None]
            scores = scores.view(kv, group, b - a, m).masked_fill(hidden, -math.inf)
            p = torch.exp(scores - scores.amax(-1, keepdim=True))
            p = (p / p.sum(-1, keepdim=True)).view(kv, group * (b - a), m)
            o = torch.matmul(p, vs)
            out[rows] = back(o)
            if train:
                do = grouped(s["d_out"])
                d_v[k0:k0 + m] += torch.matmul(p.transpose(1, 2), do).transpose(0, 1)
                ds = torch.matmul(do, vt)
                ds = p * (ds - (do * o).sum(-1, keepdim=True)) * scale
                d_q[rows] = back(torch.matmul(ds, ks))
                d_k[k0:k0 + m] += torch.matmul(ds.transpose(1, 2), qs).transpose(0, 1)
    got = {"out": out.to(q.dtype)}
    if train:
        got.update(d_q=d_q.to(q.dtype), d_k=d_k.to(q.dtype), d_v=d_v.to(q.dtype))
    return got


def run(state):
    if own:
        return _run_own(state)
    return {"block_norm": _plain_block_norm, "embedding": _plain_embedding,
            "attention": _plain_attention}[state["op"]](state)


# -- values in 64 bits ---------------------------------------------------------------

def _exact_block_norm(s):
    train = s["mode"] == "train"
    names = [n for n in ("x", "residual", "pre_weight", "post_weight", "gate_value")
             if s[n] is not None]
    t = {n: s[n].double().requires_grad_(train) for n in names}
    norm = lambda z, w: z / (z.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w
    u = norm(t["x"], t["post_weight"]) if "post_weight" in t else t["x"]
    total = t["residual"] * s["scale"] + u * t.get("gate_value", 1.0)
    out = norm(total, t["pre_weight"])
    got = {"out": out.detach(), "sum": total.detach()}
    if train:
        d = torch.autograd.grad((out, total), [t[n] for n in names],
                                (s["d_out"].double(), s["d_sum"].double()))
        got.update({("d_gate" if n == "gate_value" else "d_" + n): g for n, g in zip(names, d)})
    return got


def _exact_embedding(s):
    ids, vocab, scale = s["ids"], s["vocab"], s["scale"]
    there = ((ids >= 0) & (ids < vocab)).double().unsqueeze(1)
    out = s["table"].double().index_select(0, ids.clamp(0, vocab - 1)) * there * scale
    got = {"out": out}
    if s["mode"] == "train":
        at = ids.clamp(0, vocab - 1).unsqueeze(1).expand(-1, s["dim"])
        got["d_table"] = torch.zeros(vocab, s["dim"], dtype=torch.float64, device=ids.device
                                     ).scatter_add_(0, at, s["d_out"].double() * there * scale)
    return got


def _exact_attention(s):
    heads, dim, train = s["heads"], s["dim"], s["mode"] == "train"
    group = heads // s["kv_heads"]
    zeros = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=t.device)
    got = {"out": zeros(s["q"])}
    if train:
        got.update(d_q=zeros(s["q"]), d_k=zeros(s["k"]), d_v=zeros(s["v"]))
    for q0, n, k0, m in _spans(s):
        for h in range(heads if m else 0):
            ks = s["k"][k0:k0 + m, h // group].double()
            vs = s["v"][k0:k0 + m, h // group].double()
            for a in range(0, n, 4096):
                rows = slice(q0 + a, q0 + min(n, a + 4096))
                qs = s["q"][rows, h].double()
                leaves = [x.detach().requires_grad_(train) for x in (qs, ks, vs)]
                logits = torch.mm(leaves[0], leaves[1].t()) / dim ** 0.5
                seen = torch.ones_like(logits, dtype=torch.bool).tril(m - n + a)
                o = torch.mm(logits.masked_fill(~seen, -math.inf).softmax(-1), leaves[2])
                got["out"][rows, h] = o.detach()
                if train:
                    d = torch.autograd.grad(o, leaves, s["d_out"][rows, h].double())
                    got["d_q"][rows, h] = d[0]
                    got["d_k"][k0:k0 + m, h // group] += d[1]
                    got["d_v"][k0:k0 + m, h // group] += d[2]
    return got


def exact(case, seed):
    """The definitions in float64, the gradients by torch's differentiation of them."""
    s = prepare(case, seed)
    return {"block_norm": _exact_block_norm, "embedding": _exact_embedding,
            "attention": _exact_attention}[s["op"]](s)


def work(case):
    op, dim, train = case["op"], case["dim"], case["mode"] == "train"
    size = 4 if case["dtype"] == "f32" else 2
    if op == "block_norm":
        n = case["rows"] * dim
        gate = {"none": 0, "channel": dim, "token": case["rows"], "full": n}[case["gate"]]
        vectors = dim * (1 + case["post"]) + gate
        # x, residual, out, sum; with the gradients d_out, d_sum, d_x, d_residual too.
        return {"bytes": (n * (8 if train else 4) + vectors * (2 if train else 1)) * size,
                "flops": n * (36 if train else 10)}
    if op == "embedding":
        n = case["tokens"] * dim
        # The gathered rows, out and the ids; d_out and the table's gradient.
        count = 2 * n * size + 8 * case["tokens"]
        if train:
            count += (n + case["vocab"] * dim) * size
        return {"bytes": count, "flops": n * (2 if train else 1)}
    heads, kv = case["heads"], case["kv_heads"]
    lengths = _lengths(case)
    if case["mode"] == "cache":
        new = case["new"]
        pairs = sum(m * new - new * (new - 1) // 2 for m in lengths)
        rows, keys = case["sequences"] * new, sum(lengths)
    else:
        pairs = sum(n * (n + 1) // 2 for n in lengths)
        rows = keys = case["tokens"]
    q_size, k_size = rows * heads * dim * size, keys * kv * dim * size
    return {"bytes": (2 * q_size + 2 * k_size) if not train else (4 * q_size + 4 * k_size),
            "flops": pairs * heads * dim * (14 if train else 4)}
