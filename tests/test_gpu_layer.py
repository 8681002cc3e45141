"""The operators around the mixer against float64, over sizes, strides, types
and values where their kernels can go wrong. Bounds are derived in layer_util."""

import math

import pytest
import torch

import layer_util as R
from conftest import load_package
from gpu_util import DEV, announce

pytestmark = pytest.mark.gpu
dn = load_package()
BF, F32 = torch.bfloat16, torch.float32
TYPES = {"bf16": BF, "f32": F32}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def inside(t, before=3, after=5):
    """The matrix `t` as a view inside a larger one that is NaN elsewhere: rows
    farther apart than they are wide, an odd element's offset, guards above and
    below."""
    rows, cols = t.shape
    big = torch.full((rows + 2, cols + before + after), math.nan, dtype=t.dtype, device=t.device)
    view = big[1:rows + 1, before:before + cols]
    view.copy_(t)
    return view


def d(t):
    return None if t is None else t.to(torch.float64)


# -- norm ------------------------------------------------------------------------

NORM_SHAPES = [(1, 1), (1, 64), (3, 7), (2, 513), (5, 2048), (257, 256), (4, 2049), (3, 4100),
               (2, 8192), (2, 8200), (2, 20001), (2100, 1000), (2049, 2048), (2049, 300)]


@pytest.mark.parametrize("rows,dim", NORM_SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("residual", [False, True])
def test_add_rms_norm(rows, dim, dtype, residual):
    announce(f"add_rms_norm {rows}x{dim} {dtype} residual={residual}")
    g, T = gen(rows * 7 + dim), TYPES[dtype]
    x, w = normal(g, rows, dim, dtype=T), normal(g, dim, dtype=T)
    r = normal(g, rows, dim, dtype=T, scale=3.0) if residual else None
    out, total = dn.add_rms_norm(x, r, w, 1e-5)
    s_ref, y_ref, (y, ey) = R.norm(d(x), d(r), d(w), 1e-5, T)
    R.check(out, y_ref, "out")
    if residual:
        R.check(total, s_ref, "sum")
    else:
        assert total is x
    rows8, total8 = dn.add_rms_norm_8bit(x, r, w, 1e-5)
    assert torch.equal(total8, total)
    top = y.abs().amax(1)
    scale = top / 448
    R.check(rows8.scale, (scale, 4 * R.U * scale + ey.amax(1) / 448 + 1e-37), "scale")
    # Half a step of e4m3: 2^-4 of a normal code, 2^-10 below 2^-6.
    back = rows8.codes.to(torch.float64) * scale[:, None]
    step = torch.maximum(y.abs() / 16, scale[:, None] * 2.0 ** -10)
    R.check(back, (y, 1.01 * step + 2 * ey), "codes")
    pad = (dim + 15) // 16 * 16
    store = rows8.codes.as_strided((rows, pad), (pad, 1))
    assert not store.view(torch.uint8)[:, dim:].any()


@pytest.mark.parametrize("rows,dim", NORM_SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("with_sum", [False, True])
def test_add_rms_norm_backward(rows, dim, dtype, with_sum):
    announce(f"add_rms_norm_backward {rows}x{dim} {dtype} d_sum={with_sum}")
    g, T = gen(rows * 11 + dim), TYPES[dtype]
    s, w, dy = normal(g, rows, dim, dtype=T), normal(g, dim, dtype=T), normal(g, rows, dim, dtype=T)
    ds = normal(g, rows, dim, dtype=T) if with_sum else None
    d_x, d_w = dn.add_rms_norm_backward(dy, ds, s, w, 1e-5)
    ref = R.norm_bwd(d(s), d(w), d(dy), d(ds), 1e-5, T, T)
    R.check(d_x, ref["d_x"], "d_x")
    R.check(d_w, ref["d_weight"], "d_weight")


def test_add_rms_norm_float_weight_views_and_special_rows():
    announce("add_rms_norm: fp32 weight, strided views, zero and non-finite rows")
    g = gen(5)
    x, r, w = normal(g, 9, 260, dtype=BF), normal(g, 9, 260, dtype=BF), normal(g, 260)
    x[2], r[2] = 0, 0
    x[4, 7], r[5, 200] = math.inf, math.nan
    for xx, rr in ((x, r), (inside(x), inside(r))):
        out, total = dn.add_rms_norm(xx, rr, w, 1e-5)
        s_ref, y_ref, _ = R.norm(d(x), d(r), d(w), 1e-5, BF)
        ok = [0, 1, 2, 3, 6, 7, 8]
        R.check(out[ok], (y_ref[0][ok], y_ref[1][ok]), "out")
        R.check(total[ok], (s_ref[0][ok], s_ref[1][ok]), "sum")
        assert not out[2].any()
        # An infinite value: its own product is inf·0, the others are 0.
        assert torch.isnan(out[4, 7]) and not out[4, :7].any()
        assert torch.isnan(out[5]).all()
        q, _ = dn.add_rms_norm_8bit(xx, rr, w, 1e-5)
        assert float(q.scale[2]) == 0.0 and not q.codes[2].float().any()
        assert torch.isnan(q.scale[4]) and torch.isnan(q.scale[5])
        assert torch.isfinite(q.codes[ok].float()).all()


def test_add_rms_norm_eps_and_scale_extremes():
    announce("add_rms_norm: tiny and large rows")
    g = gen(6)
    x = normal(g, 4, 128, dtype=F32) * torch.tensor([1e-18, 1e-4, 1.0, 1e15], device=DEV)[:, None]
    w = torch.ones(128, device=DEV)
    out, _ = dn.add_rms_norm(x, None, w, 1e-6)
    R.check(out, R.norm(d(x), None, d(w), 1e-6, F32)[1], "out")


# -- linear ------------------------------------------------------------------------

# rows, in, out: few rows, tile edges, ragged contractions, odd widths.
LINEAR_SHAPES = [
    (1, 1, 1), (1, 64, 128), (1, 2048, 520), (2, 100, 1039), (3, 7, 5), (7, 256, 256),
    (15, 72, 136), (16, 520, 64), (17, 64, 300), (32, 33, 65), (33, 1024, 24), (48, 512, 1000),
    (63, 640, 128), (64, 96, 2000), (65, 128, 128), (100, 250, 683), (129, 200, 264),
    (256, 256, 256), (257, 72, 520), (300, 1000, 136), (513, 136, 1033), (1000, 683, 250),
    (520, 4096, 64), (2, 5000, 40), (96, 8192, 48),
]
ACTS = ["identity", "silu", "relu", "gelu"]


@pytest.mark.parametrize("rows,k,n", LINEAR_SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_linear(rows, k, n, dtype):
    T = TYPES[dtype]
    for i, kind in enumerate(ACTS):
        bias, residual, views = i in (1, 3), i in (2, 3), i in (0, 2)
        announce(f"linear {rows}x{k}x{n} {dtype} {kind} bias={bias} residual={residual} views={views}")
        g = gen(rows + k * 3 + n * 5 + i)
        x, w = normal(g, rows, k, dtype=T), normal(g, k, n, dtype=T, scale=k ** -0.5)
        b = normal(g, n, dtype=T) if bias else None
        r = normal(g, rows, n, dtype=T) if residual else None
        xs, ws, rs = (inside(x), inside(w), None if r is None else inside(r)) if views else (x, w, r)
        A = dn.Activation[kind.upper()]
        (z, ez), out_ref = R.linear(d(x), d(w), d(b), kind, d(r), T)
        out, preact = dn.linear_forward(xs, ws, b, A, rs)
        R.check(out, out_ref, "out")
        assert torch.equal(dn.linear(xs, ws, b, A, rs), out)
        if kind == "identity":
            assert preact is None
        else:
            R.check(preact, (z, R.rounded(z, ez, T)), "preact")


@pytest.mark.parametrize("rows", [2, 70])
@pytest.mark.parametrize("kind", ACTS)
def test_activations_keep_nan(rows, kind):
    announce(f"linear {rows}x64x72 {kind}: NaN in a row")
    g = gen(rows)
    x, w = normal(g, rows, 64), normal(g, 64, 72)
    x[1, 3] = math.nan
    out, preact = dn.linear_forward(x, w, None, dn.Activation[kind.upper()])
    assert torch.isnan(out[1]).all() and not torch.isnan(out[0]).any()
    if preact is not None:
        dx = dn.linear_backward(torch.ones_like(out), x, w, preact,
                                dn.Activation[kind.upper()]).d_x
        assert not torch.isnan(dx[0]).any()


@pytest.mark.parametrize("rows,k,n", LINEAR_SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_linear_backward(rows, k, n, dtype):
    T = TYPES[dtype]
    for i, kind in enumerate(ACTS):
        views = i % 2 == 0
        announce(f"linear_backward {rows}x{k}x{n} {dtype} {kind} views={views}")
        g = gen(rows + k * 7 + n * 5 + i)
        x, w = normal(g, rows, k, dtype=T), normal(g, k, n, dtype=T, scale=k ** -0.5)
        dy = normal(g, rows, n, dtype=T)
        A = dn.Activation[kind.upper()]
        (z, ez), _ = R.linear(d(x), d(w), None, kind, None, T)
        _, preact = dn.linear_forward(x, w, None, A)
        xs, ws, ds = (inside(x), inside(w), inside(dy)) if views else (x, w, dy)
        grads = dn.linear_backward(ds, xs, ws, preact, A, bias=True)
        ref = R.linear_bwd(d(dy), d(x), d(w), z, ez, kind, T)
        for name in ("d_x", "d_weight", "d_bias"):
            R.check(getattr(grads, name), ref[name], name)
        only = dn.linear_backward(ds, xs, ws, preact, A, need_x=False)
        assert only.d_x is None and only.d_bias is None
        assert torch.equal(only.d_weight, grads.d_weight)


@pytest.mark.parametrize("rows,k,n", [(5, 40, 70), (16, 2048, 264), (70, 72, 300), (200, 136, 1033),
                                      (300, 264, 520)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_linear_keeps_non_finite_values_in_their_rows_and_columns(rows, k, n, dtype):
    announce(f"linear {rows}x{k}x{n} {dtype}: inf and NaN")
    g, T = gen(9), TYPES[dtype]
    x, w = normal(g, rows, k, dtype=T), normal(g, k, n, dtype=T)
    clean = dn.linear(x, w)
    x[rows - 1, k - 1] = math.inf  # the last row, the last term: next to every edge
    w[k - 1, n - 1] = math.nan
    x[0, 0] = math.nan
    out = dn.linear(x, w)
    assert torch.equal(out[1:rows - 1, :n - 1], clean[1:rows - 1, :n - 1])
    assert torch.isnan(out[0]).all() and torch.isnan(out[:, n - 1]).all()
    assert torch.isinf(out[rows - 1, :n - 1]).all()
    dy = normal(g, rows, n, dtype=T)
    dy[rows - 1, 0] = math.inf
    w[k - 1, n - 1] = 1.0
    x[0, 0], x[rows - 1, k - 1] = 1.0, 1.0
    gr = dn.linear_backward(dy, x, w)
    assert torch.isfinite(gr.d_x[:rows - 1]).all()
    assert torch.isfinite(gr.d_weight[:, 1:]).all()


def test_linear_takes_leading_axes_empty_rows_and_expanded_inputs():
    announce("linear: leading axes, no rows, expanded input")
    g = gen(3)
    x, w = normal(g, 2, 5, 64, dtype=BF), normal(g, 64, 72, dtype=BF)
    out = dn.linear(x, w)
    assert out.shape == (2, 5, 72)
    assert torch.equal(out.reshape(10, 72), dn.linear(x.reshape(10, 64), w))
    assert dn.linear(x[:, :0], w).shape == (2, 0, 72)
    gr = dn.linear_backward(out[:, :0], x[:, :0], w, bias=True)
    assert not gr.d_weight.any() and not gr.d_bias.any() and gr.d_x.shape == (2, 0, 64)
    row = normal(g, 1, 64, dtype=BF)
    assert torch.equal(dn.linear(row.expand(70, 64), w), dn.linear(row.repeat(70, 1), w))
    assert torch.equal(dn.linear(x[0], w.t().contiguous().t()), out[0])  # columns adjacent


# -- 8-bit linear --------------------------------------------------------------------


@pytest.mark.parametrize("rows,k,n", [(1, 1, 1), (1, 2048, 520), (3, 40, 7), (16, 250, 130),
                                      (17, 128, 128), (64, 683, 300), (100, 136, 1033),
                                      (257, 2048, 264), (300, 64, 513), (2, 5000, 40)])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_linear_8bit(rows, k, n, out):
    T = TYPES[out]
    for i, kind in enumerate(ACTS):
        announce(f"linear_8bit {rows}x{k}x{n} {out} {kind}")
        g = gen(rows + k * 3 + n * 5 + i)
        xq = dn.quantize_rows(normal(g, rows, k))
        wq = dn.quantize_rows(normal(g, n, k, scale=k ** -0.5))
        b = normal(g, n, dtype=T) if i % 2 else None
        r = normal(g, rows, n, dtype=T) if i >= 2 else None
        x = d(xq.codes) * d(xq.scale)[:, None]
        w = (d(wq.codes) * d(wq.scale)[:, None]).t().contiguous()
        _, ref = R.linear(x, w, d(b), kind, d(r), T)
        got = dn.linear_8bit(xq, wq, b, dn.Activation[kind.upper()], r, T)
        R.check(got, ref, "out")


def test_norm_into_linear_8bit():
    announce("add_rms_norm_8bit into linear_8bit")
    g = gen(12)
    x, res, w = normal(g, 70, 250, dtype=BF), normal(g, 70, 250, dtype=BF), normal(g, 250, dtype=BF)
    wq = dn.quantize_rows(normal(g, 90, 250, scale=250 ** -0.5))
    q, _ = dn.add_rms_norm_8bit(x, res, w)
    out = dn.linear_8bit(q, wq)
    ref = R.linear(d(q.codes) * d(q.scale)[:, None],
                   (d(wq.codes) * d(wq.scale)[:, None]).t().contiguous(), None, "identity", None, BF)
    R.check(out, ref[1], "out")


# -- gated feed-forward ----------------------------------------------------------------

FFN_SHAPES = [(1, 64, 128), (1, 2048, 520), (3, 7, 5), (16, 72, 136), (17, 250, 683), (33, 64, 64),
              (64, 520, 1000), (65, 128, 128), (100, 136, 300), (256, 256, 512), (300, 250, 683),
              (513, 136, 264), (2, 40, 5000)]


@pytest.mark.parametrize("rows,dim,hidden", FFN_SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["silu", "gelu", "relu", "identity"])
def test_gated_ffn(rows, dim, hidden, dtype, kind):
    views = kind in ("gelu", "relu")
    announce(f"gated_ffn {rows}x{dim}x{hidden} {dtype} {kind} views={views}")
    g, T = gen(rows + dim * 3 + hidden), TYPES[dtype]
    x = normal(g, rows, dim, dtype=T)
    wg, wu = (normal(g, dim, hidden, dtype=T, scale=dim ** -0.5) for _ in range(2))
    wd = normal(g, hidden, dim, dtype=T, scale=hidden ** -0.5)
    res = normal(g, rows, dim, dtype=T) if kind != "identity" else None
    dy = normal(g, rows, dim, dtype=T)
    A = dn.Activation[kind.upper()]
    if views:
        both = torch.cat([wg, wu], 1)  # the halves of one matrix
        a = (inside(x), both[:, :hidden], both[:, hidden:], inside(wd))
    else:
        a = (x, wg, wu, wd)
    out, gate, up = dn.gated_ffn_forward(*a, A, res)
    ref = R.ffn(d(x), d(wg), d(wu), d(wd), kind, d(res), T)
    R.check(out, ref["out"], "out")
    R.check(gate, ref["gate"], "gate")
    R.check(up, ref["up"], "up")
    assert torch.equal(dn.gated_ffn(*a, A, res), out)
    grads = dn.gated_ffn_backward(inside(dy) if views else dy, *a, gate, up, A)
    ref = R.ffn_bwd(d(dy), d(x), d(wg), d(wu), d(wd), kind, T)
    for name, r in ref.items():
        R.check(getattr(grads, name), r, name)


def test_gated_ffn_without_rows():
    announce("gated_ffn: no rows")
    g = gen(1)
    wg, wu, wd = normal(g, 64, 72), normal(g, 64, 72), normal(g, 72, 64)
    x = torch.empty(0, 64, device=DEV)
    out, gate, up = dn.gated_ffn_forward(x, wg, wu, wd)
    assert out.shape == (0, 64) and gate.shape == (0, 72)
    gr = dn.gated_ffn_backward(x, x, wg, wu, wd, gate, up)
    assert not gr.d_w_gate.any() and not gr.d_w_up.any() and not gr.d_w_down.any()


# -- gradients against differences, autograd --------------------------------------------


def test_gradients_agree_with_differences():
    """Central differences of the fp32 operators along random directions. The
    loss is a sum of about 1e3 terms of order one, known to 1e-4; over a step of
    1e-2 that is 1e-2 of a derivative of order 30, and the third derivative adds
    1e-4 of it."""
    announce("gradients against differences")
    g = gen(77)
    rows, dim, hidden = 24, 40, 56
    x, res = normal(g, rows, dim), normal(g, rows, dim)
    gamma = normal(g, dim) * 0.1 + 1.0
    w = [normal(g, dim, hidden, scale=dim ** -0.5), normal(g, dim, hidden, scale=dim ** -0.5),
         normal(g, hidden, dim, scale=hidden ** -0.5), normal(g, dim, dim, scale=dim ** -0.5),
         normal(g, dim)]
    leaves = [x, res, gamma] + w
    c = normal(g, rows, dim)

    def loss(ls):
        out, total = dn.add_rms_norm(ls[0], ls[1], ls[2])
        y = dn.gated_ffn(out, ls[3], ls[4], ls[5], dn.Activation.SILU, total)
        return dn.linear(y, ls[6], ls[7], dn.Activation.GELU, total)

    ls = [t.clone().requires_grad_(True) for t in leaves]
    grads = torch.autograd.grad(loss(ls), ls, c)
    for i in range(len(leaves)):
        v = normal(g, *leaves[i].shape)
        v = v / v.norm()
        step = 1e-2
        plus, minus = list(leaves), list(leaves)
        plus[i], minus[i] = leaves[i] + step * v, leaves[i] - step * v
        with torch.no_grad():
            diff = (((loss(plus) - loss(minus)).double() * c.double()).sum() / (2 * step)).item()
        want = (grads[i].double() * v.double()).sum().item()
        assert abs(diff - want) <= 2e-2 * max(1.0, abs(want)), (i, diff, want)


def test_autograd_matches_the_explicit_halves():
    announce("autograd of the layer's operators")
    g = gen(8)
    x = normal(g, 3, 11, 64, dtype=BF).requires_grad_(True)
    res = normal(g, 3, 11, 64, dtype=BF).requires_grad_(True)
    gamma = normal(g, 64, dtype=BF).requires_grad_(True)
    out, total = dn.add_rms_norm(x, res, gamma)
    d_out, d_sum = normal(g, 3, 11, 64, dtype=BF), normal(g, 3, 11, 64, dtype=BF)
    got = torch.autograd.grad((out, total), (x, res, gamma), (d_out, d_sum))
    d_x, d_w = dn.add_rms_norm_backward(d_out, d_sum, total.detach(), gamma.detach())
    assert torch.equal(got[0], d_x) and torch.equal(got[1], d_x) and torch.equal(got[2], d_w)
    # Only one of the outputs used, and no residual.
    out, total = dn.add_rms_norm(x, None, gamma)
    gx, = torch.autograd.grad(out, x, d_out)
    want, _ = dn.add_rms_norm_backward(d_out, None, x.detach(), gamma.detach())
    assert torch.equal(gx, want)
    w = normal(g, 64, 40, dtype=BF).requires_grad_(True)
    b = normal(g, 40, dtype=BF).requires_grad_(True)
    y = dn.linear(x, w, b, dn.Activation.SILU)
    dy = normal(g, 3, 11, 40, dtype=BF)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), dy)
    _, pre = dn.linear_forward(x.detach(), w.detach(), b.detach(), dn.Activation.SILU)
    want = dn.linear_backward(dy, x.detach(), w.detach(), pre, dn.Activation.SILU, bias=True)
    assert torch.equal(gx, want.d_x) and torch.equal(gw, want.d_weight) and torch.equal(gb, want.d_bias)


# -- streams, graphs, repeatability ---------------------------------------------------------


def test_other_streams_graphs_and_repeats():
    announce("layer operators on another stream, in a graph, repeated")
    g = gen(21)
    x, res, gamma = normal(g, 40, 256, dtype=BF), normal(g, 40, 256, dtype=BF), normal(g, 256, dtype=BF)
    wg, wu = normal(g, 256, 704, dtype=BF, scale=0.06), normal(g, 256, 704, dtype=BF, scale=0.06)
    wd = normal(g, 704, 256, dtype=BF, scale=0.04)

    def layer():
        out, total = dn.add_rms_norm(x, res, gamma)
        y, gate, up = dn.gated_ffn_forward(out, wg, wu, wd, residual=total)
        gr = dn.gated_ffn_backward(y, out, wg, wu, wd, gate, up)
        d_x, d_w = dn.add_rms_norm_backward(gr.d_x, y, total, gamma)
        lb = dn.linear_backward(d_x, x, wg[:, :256].contiguous(), bias=True)
        return [y, gr.d_w_gate, gr.d_w_down, d_x, d_w, lb.d_x, lb.d_weight, lb.d_bias]

    want = [t.clone() for t in layer()]
    torch.cuda.synchronize()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(layer(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer()
    for _ in range(4):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(layer(), want))
