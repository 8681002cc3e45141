"""What the header and the descriptions of the operators around the mixer
promise beside their formulas: outputs that lie on inputs, 8-bit rows in the
storage of wider ones, the shapes and orders of differentiation, sizes up to
the stated limits. References and bounds as in layer_util."""

import ctypes
import math

import pytest
import torch

import layer_util as R
from test_gpu_layer import BF, DEV, F32, TYPES, d, dn, gen, inside, normal
from gpu_util import announce

pytestmark = pytest.mark.gpu
abi = dn.abi
F8 = torch.float8_e4m3fn


def entry(name, struct, **fields):
    """One call of a C entry with the library's own workspace; tensors are given
    by their address and, as <name>_stride, the distance of their rows."""
    a = struct()
    for k, v in fields.items():
        if isinstance(v, torch.Tensor):
            setattr(a, k, v.data_ptr())
            if hasattr(a, k + "_stride"):
                setattr(a, k + "_stride", v.stride(0))
        elif v is not None:
            setattr(a, k, v)
    abi.check(getattr(abi.lib(), name)(ctypes.byref(a), torch.cuda.current_stream().cuda_stream))


# -- outputs on inputs -----------------------------------------------------------


@pytest.mark.parametrize("rows,dim", [(3, 300), (2100, 1000), (5, 2049), (3, 8192), (70, 8200),
                                      (2, 20001)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("on", ["d_out", "d_sum"])
def test_norm_gradient_on_its_inputs(rows, dim, dtype, on):
    announce(f"dn_add_rms_norm_bwd {rows}x{dim} {dtype}: d_x on {on}")
    g, T = gen(rows + dim), TYPES[dtype]
    s, w = normal(g, rows, dim, dtype=T), normal(g, dim, dtype=T)
    t = {"d_out": normal(g, rows, dim, dtype=T), "d_sum": normal(g, rows, dim, dtype=T)}
    ref = R.norm_bwd(d(s), d(w), d(t["d_out"]), d(t["d_sum"]), 1e-5, T, T)
    d_w = torch.empty_like(w)
    entry("dn_add_rms_norm_bwd", abi.AddRmsNormBwdArgs, rows=rows, dim=dim, eps=1e-5,
          dtype=abi.dtype_tag(T), weight_dtype=abi.dtype_tag(T), sum=s, weight=w, d_x=t[on],
          d_weight=d_w, **t)
    R.check(t[on], ref["d_x"], "d_x")
    R.check(d_w, ref["d_weight"], "d_weight")


@pytest.mark.parametrize("rows,dim", [(3, 300), (2100, 1000), (5, 2049), (3, 8192), (4, 8200)])
@pytest.mark.parametrize("out", ["bf16", "f32", "f8"])
@pytest.mark.parametrize("on", ["x", "residual"])
def test_norm_sum_on_its_inputs(rows, dim, out, on):
    announce(f"dn_add_rms_norm {rows}x{dim} into {out}: sum on {on}")
    T = F32 if out == "f32" else BF
    g = gen(rows + dim)
    t = {"x": normal(g, rows, dim, dtype=T), "residual": normal(g, rows, dim, dtype=T)}
    w = normal(g, dim, dtype=T)
    s_ref, y_ref, _ = R.norm(d(t["x"]), d(t["residual"]), d(w), 1e-5, T)
    if out == "f8":
        rows8, _ = dn.add_rms_norm_8bit(t["x"], t["residual"], w)
    pad = (dim + 15) // 16 * 16
    y = torch.empty((rows, pad), dtype=F8 if out == "f8" else T, device=DEV)
    scale = torch.empty(rows, device=DEV)
    entry("dn_add_rms_norm", abi.AddRmsNormArgs, rows=rows, dim=dim, eps=1e-5,
          dtype=abi.dtype_tag(T), weight_dtype=abi.dtype_tag(T),
          out_dtype=abi.DN_F8 if out == "f8" else abi.dtype_tag(T), weight=w, out=y, scale=scale,
          sum=t[on], **t)
    R.check(t[on], s_ref, "sum")
    if out == "f8":
        assert torch.equal(y[:, :dim].view(torch.uint8), rows8.codes.view(torch.uint8))
        assert torch.equal(scale, rows8.scale)
    else:
        R.check(y[:, :dim], y_ref, "out")


# One shape for each kernel and for each way to split its contraction.
@pytest.mark.parametrize("rows,k,n", [(1, 5632, 2048), (3, 72, 136), (40, 100, 70), (70, 72, 300),
                                      (256, 2048, 264), (1000, 683, 250), (2568, 16392, 1800)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_linear_on_its_residual(rows, k, n, dtype):
    announce(f"dn_linear {rows}x{k}x{n} {dtype}: out on the residual")
    g, T = gen(rows + k + n), TYPES[dtype]
    x, w = normal(g, rows, k, dtype=T), normal(g, k, n, dtype=T, scale=k ** -0.5)
    r = normal(g, rows, n, dtype=T)
    want = dn.linear(x, w, None, dn.Activation.SILU, r)
    tag = abi.dtype_tag(T)
    entry("dn_linear", abi.LinearArgs, rows=rows, in_dim=k, out_dim=n, dtype=tag, out_dtype=tag,
          activation=abi.DN_ACT_SILU, x=x, weight=w, residual=r, out=r)
    assert torch.equal(r, want)


@pytest.mark.parametrize("rows,dim,hidden", [(1, 264, 520), (33, 64, 64), (300, 250, 683)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gated_ffn_on_its_residual(rows, dim, hidden, dtype):
    announce(f"dn_gated_ffn {rows}x{dim}x{hidden} {dtype}: out on the residual")
    g, T = gen(rows + dim + hidden), TYPES[dtype]
    x, r = normal(g, rows, dim, dtype=T), normal(g, rows, dim, dtype=T)
    wg, wu = (normal(g, dim, hidden, dtype=T, scale=dim ** -0.5) for _ in range(2))
    wd = normal(g, hidden, dim, dtype=T, scale=hidden ** -0.5)
    want = dn.gated_ffn(x, wg, wu, wd, residual=r)
    entry("dn_gated_ffn", abi.GatedFfnArgs, rows=rows, dim=dim, hidden=hidden,
          dtype=abi.dtype_tag(T), activation=abi.DN_ACT_SILU, x=x, w_gate=wg, w_up=wu,
          w_in_stride=hidden, w_down=wd, residual=r, out=r)
    assert torch.equal(r, want)


# -- 8-bit rows in wider storage ----------------------------------------------------


def compact(r, cols):
    """The columns `cols` of 8-bit rows in storage of their own."""
    part = r.codes[:, cols]
    n, k = part.shape
    store = torch.zeros((n, (k + 15) // 16 * 16), dtype=F8, device=DEV)
    store[:, :k].copy_(part)
    return dn.Rows8(store[:, :k], r.scale)


EIGHT_BIT_SHAPES = [(1, 1000, 264), (16, 250, 130), (40, 100, 70), (70, 40, 72), (257, 683, 264),
                    (300, 100, 1033), (1, 100, 3), (4104, 4100, 4104)]


@pytest.mark.parametrize("rows,k,n", EIGHT_BIT_SHAPES)
def test_linear_8bit_takes_codes_that_are_not_adjacent(rows, k, n):
    announce(f"linear_8bit {rows}x{k}x{n}: every other column of wider codes")
    g = gen(rows + k)
    xq, wq = dn.quantize_rows(normal(g, rows, 2 * k)), dn.quantize_rows(normal(g, n, 2 * k))
    other = slice(None, None, 2)
    want = dn.linear_8bit(compact(xq, other), compact(wq, other))
    assert torch.equal(dn.linear_8bit(dn.Rows8(xq.codes[:, other], xq.scale),
                                      dn.Rows8(wq.codes[:, other], wq.scale)), want)


@pytest.mark.parametrize("rows,k,n", EIGHT_BIT_SHAPES)
def test_linear_8bit_takes_a_part_of_wider_codes(rows, k, n):
    """What stands beside the part, numbers or NaN, is not multiplied."""
    announce(f"linear_8bit {rows}x{k}x{n}: columns 16 on of wider codes")
    g = gen(rows + k + 1)
    xq, wq = (dn.quantize_rows(normal(g, m, k + 40)) for m in (rows, n))
    part = slice(16, 16 + k)
    want = dn.linear_8bit(compact(xq, part), compact(wq, part))
    for beside in (None, math.nan):
        if beside is not None:
            xq.codes[:, 16 + k:] = beside
            wq.codes[:, 16 + k:] = beside
        got = dn.linear_8bit(dn.Rows8(xq.codes[:, part], xq.scale),
                             dn.Rows8(wq.codes[:, part], wq.scale))
        assert torch.equal(got, want)


def test_linear_8bit_refuses_rows_whose_storage_ends_early():
    announce("linear_8bit: storage that ends inside the last word")
    g = gen(3)
    store = dn.quantize_rows(normal(g, 4, 48)).codes.flatten()
    short = torch.empty(3 * 48 + 40, dtype=torch.uint8, device=DEV).view(F8)
    short.copy_(store[:short.numel()])
    codes = short.as_strided((4, 40), (48, 1))
    w = dn.quantize_rows(normal(g, 72, 40))
    with pytest.raises(dn.DeltaError, match="16-byte") as e:
        dn.linear_8bit(dn.Rows8(codes, torch.ones(4, device=DEV)), w)
    assert e.value.code == -9


@pytest.mark.parametrize("stride", [0, 3, 40, 41, 48])
def test_norm_8bit_of_one_row_needs_no_stride(stride):
    announce(f"dn_add_rms_norm into 8 bits, one row, out_stride {stride}")
    g = gen(4)
    x, w = normal(g, 1, 40), normal(g, 40)
    want, _ = dn.add_rms_norm_8bit(x, None, w)
    y, scale = torch.full((48,), 1.0, device=DEV).to(F8), torch.empty(1, device=DEV)
    entry("dn_add_rms_norm", abi.AddRmsNormArgs, rows=1, dim=40, eps=1e-5, out_dtype=abi.DN_F8,
          x=x, weight=w, out=y.data_ptr(), out_stride=stride, scale=scale)
    assert torch.equal(y[:40].view(torch.uint8), want.codes[0].view(torch.uint8))
    got = y[40:].float()
    filled = max(0, stride - 40)
    assert not got[:filled].any() and (got[filled:] == 1.0).all()


@pytest.mark.parametrize("dim", [7, 250, 2049, 8201])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_norm_8bit_pads_non_finite_rows_with_zeros_too(dim, bad):
    announce(f"add_rms_norm_8bit 3x{dim}: {bad} in a row")
    x = normal(gen(dim), 3, dim)
    x[1, dim - 1] = bad
    codes = dn.add_rms_norm_8bit(x, None, torch.ones(dim, device=DEV))[0].codes
    pad = (dim + 15) // 16 * 16
    assert not codes.as_strided((3, pad), (pad, 1)).view(torch.uint8)[:, dim:].any()


def test_norm_8bit_of_the_smallest_values_is_finite():
    """A row whose scale is the smallest number of fp32, and stands for 1.4 of it."""
    announce("add_rms_norm_8bit: rows of denormal values")
    tiny = 2.0 ** -149
    w = (torch.arange(0, 628, device=DEV, dtype=torch.float64) * tiny).float()
    q, _ = dn.add_rms_norm_8bit(torch.ones(2, 628, device=DEV), None, w)
    assert (q.scale.double() == tiny).all()
    codes = q.codes.float()
    assert torch.isfinite(codes).all()
    assert (codes[:, 448:] == 448).all() and (codes[:, :16].cpu() == torch.arange(16.)).all()


# -- differentiation ---------------------------------------------------------------


def operators(g, T=F32, lead=(2, 3), res=(2, 3)):
    """(name, operator, its inputs): each differentiable operator as a function of
    all its inputs."""
    x = normal(g, *lead, 24, dtype=T)
    r24, r40 = normal(g, *res, 24, dtype=T), normal(g, *res, 40, dtype=T)
    w, b = normal(g, 24, 40, dtype=T, scale=0.2), normal(g, 40, dtype=T)
    wg, wu = normal(g, 24, 56, dtype=T, scale=0.2), normal(g, 24, 56, dtype=T, scale=0.2)
    wd = normal(g, 56, 24, dtype=T, scale=0.2)
    return [
        ("add_rms_norm", lambda x, r, w: dn.add_rms_norm(x, r, w)[0], (x, r24, normal(g, 24, dtype=T))),
        ("linear", lambda x, w, b, r: dn.linear(x, w, b, dn.Activation.SILU, r), (x, w, b, r40)),
        ("gated_ffn", lambda x, g, u, d, r: dn.gated_ffn(x, g, u, d, residual=r),
         (x, wg, wu, wd, r24)),
    ]


@pytest.mark.parametrize("which", range(3), ids=["add_rms_norm", "linear", "gated_ffn"])
@pytest.mark.parametrize("cotangent", ["of the output", "constant"])
def test_second_derivatives_are_refused(which, cotangent):
    """A penalty on the gradient would otherwise lose its part without a word."""
    name, fn, leaves = operators(gen(31))[which]
    announce(f"{name}: gradient of a gradient, cotangent {cotangent}")
    leaves = [t.requires_grad_(True) for t in leaves]
    out = fn(*leaves)
    loss = out.sum() if cotangent == "constant" else out.square().sum()
    plain = torch.autograd.grad(loss, leaves, retain_graph=True)
    graphed = torch.autograd.grad(loss, leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, graphed))
    with pytest.raises(dn.DeltaError, match="second derivative") as e:
        (loss + graphed[0].square().sum()).backward()
    assert e.value.code == -9


@pytest.mark.parametrize("cotangent", ["of the output", "constant"])
def test_second_derivatives_of_the_delta_rule_are_refused(cotangent):
    announce(f"DeltaInput.run: gradient of a gradient, cotangent {cotangent}")
    g = gen(32)
    q, k, v = (normal(g, 1, 64, 2, 64, scale=0.1).requires_grad_(True) for _ in range(3))
    gates = torch.rand(1, 64, 2, 1, generator=g, device=DEV)
    y, _ = dn.DeltaInput(q, k, v, gates, gates, None, torch.zeros(1, 2, 64, 64, device=DEV)).run()
    loss = y.sum() if cotangent == "constant" else y.square().sum()
    plain = torch.autograd.grad(loss, (q, k, v), retain_graph=True)
    graphed = torch.autograd.grad(loss, (q, k, v), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, graphed))
    with pytest.raises(dn.DeltaError, match="second derivative") as e:
        (loss + graphed[0].square().sum()).backward()
    assert e.value.code == -9


@pytest.mark.parametrize("which", range(3), ids=["add_rms_norm", "linear", "gated_ffn"])
@pytest.mark.parametrize("grad_mode", [False, True])
def test_tangents_are_refused(which, grad_mode):
    name, fn, leaves = operators(gen(33))[which]
    announce(f"{name}: forward-mode differentiation, grad mode {grad_mode}")
    ad = torch.autograd.forward_ad
    with ad.dual_level(), torch.set_grad_enabled(grad_mode):
        want = fn(*leaves)  # no tangents: as ever
        for i in range(len(leaves)):
            dual = list(leaves)
            dual[i] = ad.make_dual(leaves[i], torch.ones_like(leaves[i]))
            with pytest.raises(NotImplementedError, match="jvp"):
                fn(*dual)
    assert torch.equal(fn(*leaves), want)


@pytest.mark.parametrize("which", range(3), ids=["add_rms_norm", "linear", "gated_ffn"])
def test_gradient_of_a_residual_has_its_shape(which):
    name, fn, leaves = operators(gen(34), lead=(2, 3), res=(6,))[which]
    announce(f"{name}: x [2, 3, dim], residual [6, dim]")
    at = 1 if name == "add_rms_norm" else -1
    leaves = [t.requires_grad_(True) for t in leaves]
    out = fn(*leaves)
    assert out.shape[:2] == (2, 3)
    c = normal(gen(35), *out.shape)
    got = torch.autograd.grad(out, leaves, c)
    same = list(leaves)
    same[at] = leaves[at].detach().reshape(2, 3, -1).requires_grad_(True)
    want = torch.autograd.grad(fn(*same), same, c)
    for a, b, leaf in zip(got, want, leaves):
        assert a.shape == leaf.shape and torch.equal(a, b.reshape(a.shape))


def test_only_the_sum_of_a_norm_used_with_a_residual_of_another_shape():
    announce("add_rms_norm: only the sum's gradient, residual [6, dim]")
    g = gen(36)
    x, r = normal(g, 2, 3, 24).requires_grad_(True), normal(g, 6, 24).requires_grad_(True)
    c = normal(g, 2, 3, 24)
    gx, gr = torch.autograd.grad(dn.add_rms_norm(x, r, normal(g, 24))[1], (x, r), c)
    assert torch.equal(gx, c) and torch.equal(gr, c.reshape(6, 24))


def test_autograd_of_the_products_matches_the_explicit_halves():
    announce("autograd of gated_ffn and of linear's residual")
    g = gen(37)
    A = dn.Activation
    (_, _, (x, w, b, r40)), (_, _, (_, wg, wu, wd, r24)) = operators(g, BF)[1:]
    for act in (A.SILU, A.GELU):
        leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd, r24)]
        y = dn.gated_ffn(*leaves[:4], act, leaves[4])
        dy = normal(g, *y.shape, dtype=BF)
        got = torch.autograd.grad(y, leaves, dy)
        out, gate, up = dn.gated_ffn_forward(x, wg, wu, wd, act, r24)
        assert torch.equal(out, y)
        want = dn.gated_ffn_backward(dy, x, wg, wu, wd, gate, up, act)
        for a, b_ in zip(got, (*want, dy)):
            assert torch.equal(a, b_)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r40)]
    y = dn.linear(*leaves[:3], A.RELU, leaves[3])
    dy = normal(g, *y.shape, dtype=BF)
    got = torch.autograd.grad(y, leaves, dy)
    out, pre = dn.linear_forward(x, w, b, A.RELU, r40)
    assert torch.equal(out, y)
    want = dn.linear_backward(dy, x, w, pre, A.RELU, bias=True)
    for a, b_ in zip(got, (*want, dy)):
        assert torch.equal(a, b_)


# -- GELU's tail ---------------------------------------------------------------------


def gelu_points():
    z = torch.cat([torch.linspace(-12, 6, 1801, device=DEV), torch.linspace(-1, 1, 401, device=DEV)])
    return z.float().reshape(-1, 1)


@pytest.mark.parametrize("rows", [40, 2202])
def test_gelu_keeps_its_tail(rows):
    """One term with a weight of one: the argument z is exact. Its scaling by a
    rounded 1/sqrt(2) is off by 2u, which moves the normal distribution function
    by at most 2(z^2 + 1)u of itself; erfc is good to 16 ulps (the most that
    OpenCL allows it), 32u, and a few products follow: (2 z^2 + 40)u."""
    announce(f"linear {rows}x1x4 fp32 gelu: its tail")
    z = gelu_points()
    z = z[:: max(1, z.shape[0] // rows)][:rows].contiguous()
    got = dn.linear(z, torch.ones(1, 4, device=DEV), None, dn.Activation.GELU)
    z = z.expand(-1, 4)
    want = R.act(d(z), "gelu")
    R.check(got, (want, (2 * d(z) ** 2 + 40) * R.U * want.abs() + 1e-37), "gelu")


def test_slope_of_gelu_keeps_its_tail():
    """Its two terms, each as above (the exponential's argument is off by 2u of
    z^2/2, and it is good to 2 ulps), add up with their errors."""
    announce("linear_backward fp32 gelu: its tail")
    z, one = gelu_points(), torch.ones(1, 1, device=DEV)
    got = dn.linear_backward(torch.ones_like(z), z, one, z, dn.Activation.GELU,
                             need_weight=False).d_x
    zz = d(z)
    cdf = 0.5 * torch.erfc(-zz / math.sqrt(2.0))
    rest = zz * torch.exp(-zz * zz / 2) / math.sqrt(2 * math.pi)
    bound = (2 * zz ** 2 + 40) * R.U * (cdf + rest.abs()) + 1e-37
    R.check(got, (cdf + rest, bound), "slope")


# -- sizes ----------------------------------------------------------------------------


@pytest.mark.parametrize("eight_bit", [False, True])
def test_norm_of_more_rows_than_a_launch_has_threads_for(eight_bit):
    rows = (1 << 26) + 5
    announce(f"add_rms_norm {rows}x1, 8-bit {eight_bit}")
    x, w = normal(gen(40), rows, 1, dtype=BF), torch.full((1,), 1.5, dtype=BF, device=DEV)
    if eight_bit:
        (codes, scale), _ = dn.add_rms_norm_8bit(x, None, w)
        top = 1.5 * (x.float() / (x.float().square() + 1e-5).sqrt()).abs()[:, 0]
        assert ((scale * 448 - top).abs() <= 1e-5 * top).all()
        sign = torch.where(x[:, 0] < 0, -448.0, 448.0)
        assert ((codes[:, 0].float() == sign) | (scale == 0)).all()
    else:
        out, _ = dn.add_rms_norm(x, None, w)
        for part in (slice(0, 1000), slice((1 << 26) - 1000, rows)):
            R.check(out[part], R.norm(d(x[part]), None, d(w), 1e-5, BF)[1], "out")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_linear_of_more_rows_than_a_launch_has_threads_for(dtype):
    rows, T = (1 << 30) + 77, TYPES[dtype]
    announce(f"linear {rows}x1x1 {dtype}")
    x = torch.empty(rows, 1, dtype=T, device=DEV)
    x[:, 0] = torch.arange(rows, device=DEV, dtype=torch.int32).remainder_(251).to(T)
    w = torch.full((1, 1), 3.0, dtype=T, device=DEV)
    out = dn.linear(x, w)
    assert torch.equal(out, x * w)
