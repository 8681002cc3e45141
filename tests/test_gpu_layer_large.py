"""The operators around the mixer at sizes that the large products' kernel
serves: whole rounds of tiles, tiles whose contraction is dealt out to several
workgroups, ragged last steps and edges, each layout and epilogue; and the
example that runs the operators together."""

import importlib.util
import math

import pytest
import torch

import layer_util as R
from conftest import ROOT
from test_gpu_layer import BF, DEV, d, dn, gen, inside, normal
from gpu_util import announce

pytestmark = pytest.mark.gpu


def view(t):
    """Inside a larger matrix that is NaN elsewhere, rows at 16-byte steps."""
    return inside(t, 8, 8)


@pytest.mark.parametrize("rows,k,n", [(4096, 4104, 4096), (4104, 8200, 4104), (2568, 16392, 1800)])
def test_linear_large(rows, k, n):
    announce(f"linear {rows}x{k}x{n}")
    g = gen(rows + k)
    x, w = normal(g, rows, k, dtype=BF), normal(g, k, n, dtype=BF, scale=k ** -0.5)
    b, r = normal(g, n, dtype=BF), normal(g, rows, n, dtype=BF)
    A = dn.Activation.GELU
    (z, ez), ref = R.linear(d(x), d(w), d(b), "gelu", d(r), BF)
    out, preact = dn.linear_forward(view(x), view(w), b, A, view(r))
    R.check(out, ref, "out")
    R.check(preact, (z, R.rounded(z, ez, BF)), "preact")
    dy = normal(g, rows, n, dtype=BF)
    got = dn.linear_backward(view(dy), view(x), view(w), preact, A, bias=True)
    want = R.linear_bwd(d(dy), d(x), d(w), z, ez, "gelu", BF)
    for name in ("d_x", "d_weight", "d_bias"):
        R.check(getattr(got, name), want[name], name)
    again = dn.linear_backward(dy, x, w, preact, A, bias=True)
    assert torch.equal(again.d_x, got.d_x) and torch.equal(again.d_weight, got.d_weight)


@pytest.mark.parametrize("rows,k,n", [(4104, 8200, 4104)])
def test_linear_8bit_large(rows, k, n):
    announce(f"linear_8bit {rows}x{k}x{n}")
    g = gen(rows)
    xq = dn.quantize_rows(normal(g, rows, k))
    wq = dn.quantize_rows(normal(g, n, k, scale=k ** -0.5))
    b = normal(g, n, dtype=BF)
    x = d(xq.codes) * d(xq.scale)[:, None]
    w = (d(wq.codes) * d(wq.scale)[:, None]).t().contiguous()
    _, ref = R.linear(x, w, d(b), "silu", None, BF)
    R.check(dn.linear_8bit(xq, wq, b, dn.Activation.SILU), ref, "out")


@pytest.mark.parametrize("rows,k,n", [(1, 5632, 2048), (16, 8200, 264), (7, 16424, 8), (2, 4096, 4096)])
def test_linear_few_rows_of_a_long_contraction(rows, k, n):
    announce(f"linear {rows}x{k}x{n}")
    g = gen(rows + k)
    x, w = normal(g, rows, k, dtype=BF), normal(g, k, n, dtype=BF, scale=k ** -0.5)
    b, r = normal(g, n, dtype=BF), normal(g, rows, n, dtype=BF)
    (z, ez), ref = R.linear(d(x), d(w), d(b), "silu", d(r), BF)
    out, preact = dn.linear_forward(view(x), view(w), b, dn.Activation.SILU, view(r))
    R.check(out, ref, "out")
    R.check(preact, (z, R.rounded(z, ez, BF)), "preact")
    assert torch.equal(dn.linear(x, w, b, dn.Activation.SILU, r), out)


def test_gated_ffn_large():
    rows, dim, hidden = 4104, 8200, 4104
    announce(f"gated_ffn {rows}x{dim}x{hidden}")
    g = gen(4)
    x = normal(g, rows, dim, dtype=BF)
    wg, wu = (normal(g, dim, hidden, dtype=BF, scale=dim ** -0.5) for _ in range(2))
    wd = normal(g, hidden, dim, dtype=BF, scale=hidden ** -0.5)
    res, dy = normal(g, rows, dim, dtype=BF), normal(g, rows, dim, dtype=BF)
    both = torch.cat([wg, wu], 1)
    a = (view(x), both[:, :hidden], both[:, hidden:], view(wd))
    out, gate, up = dn.gated_ffn_forward(*a, residual=view(res))
    ref = R.ffn(d(x), d(wg), d(wu), d(wd), "silu", d(res), BF)
    for name, got in (("out", out), ("gate", gate), ("up", up)):
        R.check(got, ref[name], name)
    del ref
    grads = dn.gated_ffn_backward(view(dy), *a, gate, up)
    for name, r in R.ffn_bwd(d(dy), d(x), d(wg), d(wu), d(wd), "silu", BF).items():
        R.check(getattr(grads, name), r, name)


def test_large_products_keep_non_finite_values_in_their_rows_and_columns():
    rows, k, n = 4104, 4104, 4360
    announce(f"linear {rows}x{k}x{n}: inf and NaN")
    g = gen(2)
    x, w = normal(g, rows, k, dtype=BF), normal(g, k, n, dtype=BF)
    clean = dn.linear(x, w)
    x[rows - 1, k - 1], x[0, 0] = math.inf, math.nan
    w[k - 1, n - 1] = math.nan
    out = dn.linear(x, w)
    assert torch.equal(out[1:rows - 1, :n - 1], clean[1:rows - 1, :n - 1])
    assert torch.isnan(out[0]).all() and torch.isnan(out[:, n - 1]).all()
    assert torch.isinf(out[rows - 1, :n - 1]).all()


def test_example_runs_the_operators_together():
    """A token's rounding differs from the prompt's in every bf16 step (2^-8 of
    each of about a dozen tensors between x and y): 5 % in the norm is beyond
    what they can add up to, and far below what a wrong state, window or
    projection gives. The loss falls along its gradient."""
    announce("examples/gated_deltanet_layer.py")
    spec = importlib.util.spec_from_file_location("layer_example",
                                                  ROOT / "examples" / "gated_deltanet_layer.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    worst, losses = mod.main()
    assert worst["bf16"] < 0.05 and worst["8-bit"] < 0.05
    assert all(b < a for a, b in zip(losses, losses[1:]))
