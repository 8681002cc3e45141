"""The operators of a stack as they are used together: the hybrid decoder's tokens one at
a time against its prompt and its gradients against float64; captured graphs; streams."""

import importlib.util
import sys

import pytest
import torch

from conftest import ROOT, load_package

dn = load_package()
pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("hybrid_decoder",
                                                  ROOT / "examples" / "hybrid_decoder.py")
    mod = importlib.util.module_from_spec(spec)
    sys.modules["hybrid_decoder"] = mod
    spec.loader.exec_module(mod)
    return mod


def test_example_runs(example):
    """bf16: some ten roundings of 2^-9 on the way, each of which the next norms and
    products pass on: a few per cent at most between the two orders of summation."""
    off, losses = example.main()
    assert off < 0.06
    assert all(torch.isfinite(torch.tensor(losses)))


def plain_logits(d, weights, tokens):
    """The decoder's formulas in float64 on `weights` (in Decoder.weights' order)."""
    it = iter(weights)
    table, head, first = next(it), next(it), next(it)
    norm = lambda z, w: z / (z.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * w
    stream = table[tokens] * d.scale
    h = norm(stream, first)
    n, hd = d.nheads, d.head_dim
    for kind, layer in zip(d.mixers, d.layers):
        w = {name: next(it) for name in layer}
        kv = d.kv_heads if kind == "attention" else n
        p = h @ w["qkv"]
        q = p[..., :n * hd].unflatten(-1, (n, hd))
        k = p[..., n * hd:(n + kv) * hd].unflatten(-1, (kv, hd))
        v = p[..., (n + kv) * hd:(n + 2 * kv) * hd].unflatten(-1, (kv, hd))
        B, S = tokens.shape
        if kind == "attention":
            k, v = (t.repeat_interleave(n // kv, 2) for t in (k, v))
            s = torch.einsum("bihd,bjhd->bhij", q, k) * hd ** -0.5
            s = s.masked_fill(torch.ones(S, S, device=s.device).triu(1).bool(), -float("inf"))
            mixed = torch.einsum("bhij,bjhd->bihd", s.softmax(-1), v)
        else:
            q, k = (torch.nn.functional.normalize(t, dim=-1) for t in (q, k))
            beta = torch.sigmoid(p[..., (n + 2 * kv) * hd:])[..., None]
            state, rows = torch.zeros(B, n, hd, hd, dtype=p.dtype, device=p.device), []
            for t in range(S):
                seen = torch.einsum("bhkv,bhk->bhv", state, k[:, t])
                state = state + torch.einsum("bhk,bhv->bhkv", k[:, t],
                                             beta[:, t] * (v[:, t] - seen))
                rows.append(torch.einsum("bhkv,bhk->bhv", state, q[:, t]) * hd ** -0.5)
            mixed = torch.stack(rows, 1)
        y = mixed.flatten(-2) @ w["out"]
        stream = d.residual_scale * stream + w["mix_gate"] * norm(y, w["mix_post"])
        h = norm(stream, w["mix_pre"])
        y = (torch.nn.functional.silu(h @ w["w_gate"]) * (h @ w["w_up"])) @ w["w_down"]
        stream = d.residual_scale * stream + w["ffn_gate"] * norm(y, w["ffn_post"])
        h = norm(stream, w["ffn_pre"])
    return h @ head


def test_gradients_of_the_decoder(example):
    """fp32: sums of some hundred terms, through four blocks: 1e-4 of a gradient's norm is
    about 2^11 times the rounding unit."""
    d = example.Decoder(97, 64, 4, 2, 32, 100, ("attention", "delta", "attention"), F32)
    gen = torch.Generator("cuda").manual_seed(2)
    tokens = torch.randint(0, 97, (2, 41), generator=gen, device="cuda")
    weights = d.weights()
    for w in weights:
        w.requires_grad_(True)
    loss = example.loss_of(d, tokens)
    grads = torch.autograd.grad(loss, weights)
    wide = [w.detach().double().requires_grad_(True) for w in weights]
    logits = plain_logits(d, wide, tokens[:, :-1])
    want_loss = torch.nn.functional.cross_entropy(logits.flatten(0, 1), tokens[:, 1:].flatten())
    assert abs(loss.item() - want_loss.item()) < 1e-5
    for got, want in zip(grads, torch.autograd.grad(want_loss, wide)):
        assert ((got.double() - want).norm() / want.norm()).item() < 1e-4


# -- graphs and streams ----------------------------------------------------------------


def operands(seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    made = lambda *shape: torch.randn(shape, generator=gen, device="cuda").to(BF)
    ids = torch.randint(-1, 70, (300,), generator=gen, device="cuda")
    off = torch.tensor([0, 120, 300], dtype=torch.int32, device="cuda")
    return {"ids": ids, "table": made(70, 256), "d": made(300, 256), "x": made(300, 256),
            "r": made(300, 256), "w": made(256), "p": made(256), "g": made(256),
            "q": made(300, 4, 64), "k": made(300, 2, 64), "v": made(300, 2, 64),
            "do": made(300, 4, 64), "off": off, "q1": made(1, 4, 64),
            "off1": torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
            "long_k": made(20000, 2, 64), "long_v": made(20000, 2, 64),
            "at": torch.tensor([7], dtype=torch.int32, device="cuda"),
            "count": torch.tensor([19000], dtype=torch.int32, device="cuda")}


def everything(t):
    """Every operator and its gradients; the cached keys are split among workgroups."""
    out, lse = dn.attention_forward(t["q"], t["k"], t["v"], t["off"])
    h, total = dn.block_norm(t["x"], t["r"], t["w"], t["p"], t["g"], 0.5)
    return [dn.embedding(t["ids"], t["table"], 2.0),
            dn.embedding_backward(t["d"], t["ids"], 70, 2.0), h, total,
            *dn.block_norm_backward(t["d"], t["r"], t["x"], total, t["w"], t["p"], t["g"], 0.5),
            out, lse,
            *dn.attention_backward(t["do"], t["q"], t["k"], t["v"], out, lse, t["off"]),
            dn.attention(t["q1"], t["long_k"], t["long_v"], t["off1"],
                         dn.KeySpans(t["at"], t["count"]))]


def equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b)) and len(a) == len(b)


def test_captured_and_replayed():
    """Two graphs over the same kind of work, replayed in turn on new inputs, with eager
    work and synchronisation between."""
    inputs, graphs = [operands(1), operands(2)], []
    stream = torch.cuda.Stream()
    for t in inputs:
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            everything(t)
        torch.cuda.current_stream().wait_stream(stream)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = everything(t)
        graphs.append((g, got))
    for seed in (3, 4, 5):
        want = []
        for i, t in enumerate(inputs):
            for name, value in operands(10 * seed + i).items():
                t[name].copy_(value)
            want.append([x.clone() for x in everything(t)])
        torch.cuda.synchronize()
        for g, got in graphs:
            for x in got:
                x.fill_(7)
            g.replay()
        everything(inputs[0])
        torch.cuda.synchronize()
        for (_, got), w in zip(graphs, want):
            assert equal(got, w)


def test_on_two_streams_at_once():
    inputs = [operands(21), operands(22)]
    want = [everything(t) for t in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for s, t in zip(streams, inputs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(everything(t))
        torch.cuda.synchronize()
        assert equal(got[0], want[0]) and equal(got[1], want[1])
