"""The operators around the delta-rule mixer in a decoder layer: the norm with
the residual's addition, the linear projection, the same from 8-bit operands,
and the gated feed-forward block, each with its gradients.

The reference's blocks end at their projections; these are what a layer built
on them needs next. `add_rms_norm`, `linear` and `gated_ffn` take part in
torch's autograd where an input requires a gradient, of first order: second
derivatives and forward-mode tangents are refused. The `*_forward` and
`*_backward` functions are the two halves for programs that run their own
backward pass. Weights lie as Burn's Linear holds them, [in, out], applied as
x @ weight. Every computation is a call into libdeltanet_core.so, but for
quantize_rows, which lays weights out once.
"""

from __future__ import annotations

import ctypes
from enum import IntEnum
from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import abi
from .abi import DeltaError
from .autograd import first_order


class Activation(IntEnum):
    """GELU is the exact form, z·Φ(z)."""
    IDENTITY = abi.DN_ACT_IDENTITY
    SILU = abi.DN_ACT_SILU
    RELU = abi.DN_ACT_RELU
    GELU = abi.DN_ACT_GELU


class Rows8(NamedTuple):
    """A matrix held in 8 bits: e4m3 `codes` [rows, dim] with one `scale` a row;
    row i stands for codes[i] * scale[i]. The codes are a view of storage whose
    rows start at multiples of 16 bytes and are whole multiples of 16 long, or a
    part of wider ones: what stands past `dim` is not used."""

    codes: Tensor
    scale: Tensor


class LinearGrads(NamedTuple):
    d_x: Optional[Tensor]
    d_weight: Optional[Tensor]
    d_bias: Optional[Tensor]


class GatedFfnGrads(NamedTuple):
    d_x: Optional[Tensor]
    d_w_gate: Optional[Tensor]
    d_w_up: Optional[Tensor]
    d_w_down: Optional[Tensor]


F8 = torch.float8_e4m3fn


# The current device's index, without torch.cuda.current_device()'s check that
# CUDA is initialised: it is asked only about tensors that live there.
_device = torch._C._cuda_getDevice


def _gpu(t: Tensor, what: str) -> None:
    if not t.is_cuda:
        raise DeltaError(-6, f"{what}: tensors must live on the GPU (no CPU fallback)")
    if t.get_device() != _device():
        raise DeltaError(-6, f"{what}: lives on another GPU than the current one")


def _rows(t: Tensor, what: str) -> Tensor:
    """`t` as [rows, dim] with contiguous rows that do not overlap: a view where
    its strides allow one, else a copy."""
    _gpu(t, what)
    if t.dim() != 2:
        if t.dim() == 0:
            raise DeltaError(-2, f"{what}: expected [..., dim], got a scalar")
        t = t.reshape(-1, t.shape[-1]) if t.numel() else t.new_empty(
            (t.shape[:-1].numel(), t.shape[-1]))
    if t.is_contiguous():
        return t
    n, d = t.shape
    s0, s1 = t.stride()
    return t if (s1 == 1 or d == 1) and (n <= 1 or s0 >= d) else t.contiguous()


def _like(t: Optional[Tensor], x: Tensor, shape, what: str) -> Optional[Tensor]:
    """An input of x's dtype whose last axis and count match `shape` (rows, dim)."""
    if t is None:
        return None
    if t.dtype != x.dtype:
        raise DeltaError(-7, f"{what}: expected {x.dtype}, got {t.dtype}")
    if t.dim() == 0 or t.shape[-1] != shape[1] or t.numel() != shape[0] * shape[1]:
        raise DeltaError(-2, f"{what}: expected {list(shape)}, got {list(t.shape)}")
    return _rows(t, what)


def _weight(w: Tensor, shape, dtype, what: str) -> Tensor:
    if w.dtype != dtype:
        raise DeltaError(-7, f"{what}: expected {dtype}, got {w.dtype}")
    if tuple(w.shape) != shape:
        raise DeltaError(-2, f"{what}: expected {list(shape)}, got {list(w.shape)}")
    return _rows(w, what)


def _vector(v: Optional[Tensor], n: int, dtype, what: str) -> Optional[Tensor]:
    if v is None:
        return None
    _gpu(v, what)
    if dtype is not None and v.dtype != dtype:
        raise DeltaError(-7, f"{what}: expected {dtype}, got {v.dtype}")
    if tuple(v.shape) != (n,):
        raise DeltaError(-2, f"{what}: expected [{n}], got {list(v.shape)}")
    return v if v.is_contiguous() else v.contiguous()


def _x_shape(x: Tensor) -> Tuple[int, int]:
    if x.dim() == 2:
        return x.shape
    if x.dim() == 0:
        raise DeltaError(-2, "x: expected [..., dim], got a scalar")
    return x.shape[:-1].numel(), x.shape[-1]


def _grows(*ts) -> bool:
    """Whether a derivative is wanted: one of the backward pass, or (it is
    refused there, as the function has none) a tangent of the forward one."""
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    if forward_ad._current_level >= 0:
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                return True
    return False


def _shaped(grad: Optional[Tensor], shape) -> Optional[Tensor]:
    """A residual's gradient: its leading axes may be others than the output's."""
    return None if grad is None or shape is None else grad.reshape(shape)


def _p(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()


_ENTRIES = {}


def _call(fn, args, sized, device) -> None:
    """The call on torch's current stream, with a workspace from torch's
    stream-ordered allocator where one is needed."""
    entry = _ENTRIES.get(fn)
    if entry is None:
        L = abi.lib()
        entry = _ENTRIES[fn] = (getattr(L, fn), getattr(L, fn + "_workspace_bytes", None))
    ref = ctypes.byref(args)
    ws = None
    if sized:
        n = entry[1](ref)
        if n:
            ws = torch.empty(n, dtype=torch.uint8, device=device)
            args.workspace, args.workspace_bytes = ws.data_ptr(), n
    rc = entry[0](ref, torch._C._cuda_getCurrentRawStream(_device()))
    if rc:
        abi.check(rc)


# -- norm ----------------------------------------------------------------------


def _norm(x, residual, weight, eps, f8):
    rows, dim = _x_shape(x)
    tag = abi.dtype_tag(x.dtype)
    x2 = _rows(x, "x")
    r2 = _like(residual, x, (rows, dim), "residual")
    w = _vector(weight, dim, None, "weight")
    a = abi.AddRmsNormArgs()
    a.rows, a.dim, a.eps = rows, dim, float(eps)
    a.dtype, a.weight_dtype, a.out_dtype = tag, abi.dtype_tag(w.dtype), abi.DN_F8 if f8 else tag
    a.x, a.x_stride, a.weight = x2.data_ptr(), x2.stride(0), w.data_ptr()
    total = x
    if r2 is not None:
        total = torch.empty_like(x, memory_format=torch.contiguous_format)
        a.residual, a.residual_stride = r2.data_ptr(), r2.stride(0)
        a.sum, a.sum_stride = total.data_ptr(), dim
    scale = None
    if f8:
        out = torch.empty((rows, (dim + 15) // 16 * 16), dtype=F8, device=x.device)
        scale = torch.empty(rows, dtype=torch.float32, device=x.device)
        a.out, a.out_stride, a.scale = out.data_ptr(), out.stride(0), scale.data_ptr()
        if out.shape[1] != dim:
            out = out[:, :dim]
    else:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        a.out, a.out_stride = out.data_ptr(), dim
    _call("dn_add_rms_norm", a, False, x.device)
    return out, scale, total


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        out, _, total = _norm(x, residual, weight, eps, False)
        ctx.eps, ctx.residual_shape = eps, None if residual is None else residual.shape
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(total, weight)
        return out, (total if residual is not None else total.view_as(total))

    @staticmethod
    @first_order
    def backward(ctx, d_out, d_sum):
        total, weight = ctx.saved_tensors
        if d_out is None:
            return d_sum, _shaped(d_sum, ctx.residual_shape), None, None
        d_x, d_w = add_rms_norm_backward(d_out, d_sum, total, weight, ctx.eps,
                                         need_weight=ctx.needs_input_grad[2])
        return d_x, _shaped(d_x, ctx.residual_shape), d_w, None


def add_rms_norm(x: Tensor, residual: Optional[Tensor], weight: Tensor,
                 eps: float = 1e-5) -> Tuple[Tensor, Tensor]:
    """sum = x + residual; out = sum / sqrt(mean(sum²) + eps) * weight over the
    last axis, from the unrounded sum. Returns (out, sum); without a residual
    the sum is x itself. The gradient is taken at the sum as it is returned."""
    if _grows(x, residual, weight):
        return _AddRmsNorm.apply(x, residual, weight, eps)
    out, _, total = _norm(x, residual, weight, eps, False)
    return out, total


def add_rms_norm_8bit(x: Tensor, residual: Optional[Tensor], weight: Tensor,
                      eps: float = 1e-5) -> Tuple[Rows8, Tensor]:
    """add_rms_norm with its output in 8 bits, as linear_8bit reads it: per row
    scale = max|out| / 448, codes = out / scale in e4m3. No gradient."""
    out, scale, total = _norm(x, residual, weight, eps, True)
    return Rows8(out, scale), total


def add_rms_norm_backward(d_out: Tensor, d_sum: Optional[Tensor], total: Tensor, weight: Tensor,
                          eps: float = 1e-5, need_weight: bool = True
                          ) -> Tuple[Tensor, Optional[Tensor]]:
    """The gradients of add_rms_norm at its `sum`: (d_x, d_weight); d_residual
    is d_x."""
    rows, dim = _x_shape(total)
    s2 = _rows(total, "sum")
    do = _like(d_out, total, (rows, dim), "d_out")
    ds = _like(d_sum, total, (rows, dim), "d_sum")
    w = _vector(weight, dim, None, "weight")
    d_x = torch.empty(total.shape, dtype=total.dtype, device=total.device)
    d_w = torch.empty_like(w) if need_weight else None
    a = abi.AddRmsNormBwdArgs()
    a.rows, a.dim, a.eps = rows, dim, float(eps)
    a.dtype, a.weight_dtype = abi.dtype_tag(total.dtype), abi.dtype_tag(w.dtype)
    a.sum, a.sum_stride, a.weight = s2.data_ptr(), s2.stride(0), w.data_ptr()
    a.d_out, a.d_out_stride = do.data_ptr(), do.stride(0)
    if ds is not None:
        a.d_sum, a.d_sum_stride = ds.data_ptr(), ds.stride(0)
    a.d_x, a.d_x_stride, a.d_weight = d_x.data_ptr(), dim, _p(d_w)
    _call("dn_add_rms_norm_bwd", a, need_weight, total.device)
    return d_x, d_w


# -- linear --------------------------------------------------------------------


def _linear(x, weight, bias, activation, residual, keep):
    rows, k = _x_shape(x)
    if weight.dim() != 2 or weight.shape[0] != k:
        raise DeltaError(-2, f"weight: expected [{k}, out], got {list(weight.shape)}")
    n = weight.shape[1]
    tag = abi.dtype_tag(x.dtype)
    x2 = _rows(x, "x")
    w = _weight(weight, (k, n), x.dtype, "weight")
    b = _vector(bias, n, x.dtype, "bias")
    r = _like(residual, x, (rows, n), "residual")
    out = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=x.device)
    a = abi.LinearArgs()
    a.rows, a.in_dim, a.out_dim = rows, k, n
    a.dtype = a.out_dtype = tag
    a.activation = int(activation)
    a.x, a.x_stride, a.weight, a.weight_stride = x2.data_ptr(), x2.stride(0), w.data_ptr(), w.stride(0)
    a.out, a.out_stride = out.data_ptr(), n
    if b is not None:
        a.bias = b.data_ptr()
    if r is not None:
        a.residual, a.residual_stride = r.data_ptr(), r.stride(0)
    preact = None
    if keep and activation != Activation.IDENTITY:
        preact = torch.empty((rows, n), dtype=x.dtype, device=x.device)
        a.preact, a.preact_stride = preact.data_ptr(), n
    _call("dn_linear", a, True, x.device)
    return out, preact


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        out, preact = _linear(x, weight, bias, activation, residual, True)
        ctx.activation = activation
        ctx.residual_shape = None if residual is None else residual.shape
        ctx.save_for_backward(x, weight, preact)
        return out

    @staticmethod
    @first_order
    def backward(ctx, d_out):
        x, weight, preact = ctx.saved_tensors
        need = ctx.needs_input_grad
        g = linear_backward(d_out, x, weight, preact, ctx.activation, bias=need[2], need_x=need[0],
                            need_weight=need[1])
        return (g.d_x, g.d_weight, g.d_bias,
                _shaped(d_out, ctx.residual_shape) if need[3] else None, None)


def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None,
           activation: Activation = Activation.IDENTITY,
           residual: Optional[Tensor] = None) -> Tensor:
    """act(x @ weight + bias) + residual, weight [in, out]. An operand whose last
    axis is not contiguous, such as the transposed view of a weight [out, in], is
    copied in every call: a program lays such a weight out once."""
    if _grows(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, residual, activation)
    return _linear(x, weight, bias, activation, residual, False)[0]


def linear_forward(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None,
                   activation: Activation = Activation.IDENTITY,
                   residual: Optional[Tensor] = None) -> Tuple[Tensor, Optional[Tensor]]:
    """linear and what its backward needs beside its inputs: the activation's
    argument, or None where the activation is the identity."""
    return _linear(x, weight, bias, activation, residual, True)


def linear_backward(d_out: Tensor, x: Tensor, weight: Tensor, preact: Optional[Tensor] = None,
                    activation: Activation = Activation.IDENTITY, bias: bool = False,
                    need_x: bool = True, need_weight: bool = True) -> LinearGrads:
    """The gradients of linear (that of its residual is d_out)."""
    rows, k = _x_shape(x)
    if weight.dim() != 2 or weight.shape[0] != k:
        raise DeltaError(-2, f"weight: expected [{k}, out], got {list(weight.shape)}")
    n = weight.shape[1]
    tag = abi.dtype_tag(x.dtype)
    x2 = _rows(x, "x")
    w = _weight(weight, (k, n), x.dtype, "weight")
    do = _like(d_out, x, (rows, n), "d_out")
    a = abi.LinearBwdArgs()
    a.rows, a.in_dim, a.out_dim, a.dtype, a.activation = rows, k, n, tag, int(activation)
    a.x, a.x_stride, a.weight, a.weight_stride = x2.data_ptr(), x2.stride(0), w.data_ptr(), w.stride(0)
    a.d_out, a.d_out_stride = do.data_ptr(), do.stride(0)
    if activation != Activation.IDENTITY:
        if preact is None:
            raise DeltaError(-6, "preact: linear_forward's is needed for this activation")
        pre = _like(preact, x, (rows, n), "preact")
        a.preact, a.preact_stride = pre.data_ptr(), pre.stride(0)
    dev = x.device
    d_x = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
    d_w = torch.empty((k, n), dtype=x.dtype, device=dev) if need_weight else None
    d_b = torch.empty(n, dtype=x.dtype, device=dev) if bias else None
    a.d_x, a.d_x_stride, a.d_weight, a.d_bias = _p(d_x), k, _p(d_w), _p(d_b)
    _call("dn_linear_bwd", a, True, dev)
    return LinearGrads(d_x, d_w, d_b)


def quantize_rows(t: Tensor) -> Rows8:
    """A matrix [rows, dim] as linear_8bit reads it, for weights (their
    transpose: rows are the outputs) that are laid out once."""
    if t.dim() != 2:
        raise DeltaError(-2, f"quantize_rows: expected [rows, dim], got {list(t.shape)}")
    t = t.float()
    scale = t.abs().amax(1) / 448.0
    # A denormal scale may stand for less than a 448th of its row's largest value.
    codes = torch.where(scale[:, None] > 0, t / scale[:, None], t).clamp(-448.0, 448.0)
    return Rows8(_padded(codes.to(F8)), scale)


def _padded(codes: Tensor) -> Tensor:
    """A copy in storage whose rows are padded with zeros to a multiple of 16."""
    rows, dim = codes.shape
    store = torch.zeros((rows, (dim + 15) // 16 * 16), dtype=F8, device=codes.device)
    store[:, :dim].copy_(codes)
    return store[:, :dim]


def _codes(r: Rows8, what: str) -> Tensor:
    c = r.codes
    if c.dtype != F8:
        raise DeltaError(-7, f"{what}: expected {F8} codes, got {c.dtype}")
    if c.dim() != 2:
        raise DeltaError(-2, f"{what}: expected [rows, dim] codes, got {list(c.shape)}")
    _gpu(c, what)
    rows, dim = c.shape
    if c.stride(1) != 1 and dim > 1:
        return _padded(c)
    # A row's last word is read whole, the last row's too.
    if dim % 16 and rows and (c.storage_offset() + (rows - 1) * c.stride(0) + (dim + 15) // 16 * 16
                              > c.untyped_storage().nbytes()):
        raise DeltaError(-9, f"{what}: 8-bit rows must be stored up to the next 16-byte boundary")
    return c


def linear_8bit(x: Rows8, weight: Rows8, bias: Optional[Tensor] = None,
                activation: Activation = Activation.IDENTITY, residual: Optional[Tensor] = None,
                out_dtype=torch.bfloat16) -> Tensor:
    """act(x @ weightᵀ + bias) + residual from operands in 8 bits: x [rows, in]
    and weight [out, in], as add_rms_norm_8bit and quantize_rows make them, or
    columns of such from a multiple of 16 on (other views are copied in every
    call). bias, residual and the output are of `out_dtype`. No gradient."""
    c, w = _codes(x, "x"), _codes(weight, "weight")
    rows, k = c.shape
    n = w.shape[0]
    if w.shape[1] != k:
        raise DeltaError(-2, f"weight: expected [out, {k}], got {list(w.shape)}")
    xs = _vector(x.scale, rows, torch.float32, "x.scale")
    wscale = _vector(weight.scale, n, torch.float32, "weight.scale")
    out = torch.empty((rows, n), dtype=out_dtype, device=c.device)
    b = _vector(bias, n, out_dtype, "bias")
    r = _like(residual, out, (rows, n), "residual")
    a = abi.LinearArgs()
    a.rows, a.in_dim, a.out_dim = rows, k, n
    a.dtype, a.out_dtype, a.activation = abi.DN_F8, abi.dtype_tag(out_dtype), int(activation)
    a.x, a.x_stride, a.weight, a.weight_stride = c.data_ptr(), c.stride(0), w.data_ptr(), w.stride(0)
    a.x_scale, a.weight_scale = xs.data_ptr(), wscale.data_ptr()
    a.out, a.out_stride = out.data_ptr(), n
    if b is not None:
        a.bias = b.data_ptr()
    if r is not None:
        a.residual, a.residual_stride = r.data_ptr(), r.stride(0)
    _call("dn_linear", a, True, c.device)
    return out


# -- gated feed-forward ----------------------------------------------------------


def _ffn_weights(w_gate, w_up, w_down, dim, dtype):
    if w_gate.dim() != 2:
        raise DeltaError(-2, f"w_gate: expected [{dim}, hidden], got {list(w_gate.shape)}")
    hidden = w_gate.shape[1]
    g = _weight(w_gate, (dim, hidden), dtype, "w_gate")
    u = _weight(w_up, (dim, hidden), dtype, "w_up")
    d = _weight(w_down, (hidden, dim), dtype, "w_down")
    if dim > 1 and g.stride(0) != u.stride(0):
        g, u = g.contiguous(), u.contiguous()
    return hidden, g, u, d


def _ffn(x, w_gate, w_up, w_down, activation, residual, keep):
    rows, dim = _x_shape(x)
    tag = abi.dtype_tag(x.dtype)
    x2 = _rows(x, "x")
    hidden, g, u, d = _ffn_weights(w_gate, w_up, w_down, dim, x.dtype)
    r = _like(residual, x, (rows, dim), "residual")
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    a = abi.GatedFfnArgs()
    a.rows, a.dim, a.hidden, a.dtype, a.activation = rows, dim, hidden, tag, int(activation)
    a.x, a.x_stride = x2.data_ptr(), x2.stride(0)
    a.w_gate, a.w_up, a.w_in_stride = g.data_ptr(), u.data_ptr(), g.stride(0)
    a.w_down, a.w_down_stride = d.data_ptr(), d.stride(0)
    a.out, a.out_stride = out.data_ptr(), dim
    if r is not None:
        a.residual, a.residual_stride = r.data_ptr(), r.stride(0)
    gate = up = None
    if keep:
        kept = torch.empty((2, rows, hidden), dtype=x.dtype, device=x.device)
        gate, up = kept[0], kept[1]
        a.gate, a.up, a.kept_stride = gate.data_ptr(), up.data_ptr(), hidden
    _call("dn_gated_ffn", a, True, x.device)
    return out, gate, up


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, residual, activation):
        out, gate, up = _ffn(x, w_gate, w_up, w_down, activation, residual, True)
        ctx.activation = activation
        ctx.residual_shape = None if residual is None else residual.shape
        ctx.save_for_backward(x, w_gate, w_up, w_down, gate, up)
        return out

    @staticmethod
    @first_order
    def backward(ctx, d_out):
        x, w_gate, w_up, w_down, gate, up = ctx.saved_tensors
        need = ctx.needs_input_grad
        g = gated_ffn_backward(d_out, x, w_gate, w_up, w_down, gate, up, ctx.activation,
                               need_x=need[0], need_in=need[1] or need[2], need_down=need[3])
        return (g.d_x, g.d_w_gate if need[1] else None, g.d_w_up if need[2] else None, g.d_w_down,
                _shaped(d_out, ctx.residual_shape) if need[4] else None, None)


def gated_ffn(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor,
              activation: Activation = Activation.SILU,
              residual: Optional[Tensor] = None) -> Tensor:
    """(act(x @ w_gate) * (x @ w_up)) @ w_down + residual; w_gate and w_up
    [dim, hidden] (they may be the halves of one matrix), w_down [hidden, dim]."""
    if _grows(x, w_gate, w_up, w_down, residual):
        return _GatedFfn.apply(x, w_gate, w_up, w_down, residual, activation)
    return _ffn(x, w_gate, w_up, w_down, activation, residual, False)[0]


def gated_ffn_forward(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor,
                      activation: Activation = Activation.SILU,
                      residual: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """gated_ffn and what its backward needs beside its inputs: (out, x @ w_gate,
    x @ w_up)."""
    return _ffn(x, w_gate, w_up, w_down, activation, residual, True)


def gated_ffn_backward(d_out: Tensor, x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor,
                       gate: Tensor, up: Tensor, activation: Activation = Activation.SILU,
                       need_x: bool = True, need_in: bool = True,
                       need_down: bool = True) -> GatedFfnGrads:
    """The gradients of gated_ffn (that of its residual is d_out)."""
    rows, dim = _x_shape(x)
    tag = abi.dtype_tag(x.dtype)
    x2 = _rows(x, "x")
    hidden, wg, wu, wd = _ffn_weights(w_gate, w_up, w_down, dim, x.dtype)
    do = _like(d_out, x, (rows, dim), "d_out")
    kg, ku = _like(gate, x, (rows, hidden), "gate"), _like(up, x, (rows, hidden), "up")
    if rows > 1 and kg.stride(0) != ku.stride(0):
        kg, ku = kg.contiguous(), ku.contiguous()
    a = abi.GatedFfnBwdArgs()
    a.rows, a.dim, a.hidden, a.dtype, a.activation = rows, dim, hidden, tag, int(activation)
    a.x, a.x_stride = x2.data_ptr(), x2.stride(0)
    a.w_gate, a.w_up, a.w_in_stride = wg.data_ptr(), wu.data_ptr(), wg.stride(0)
    a.w_down, a.w_down_stride = wd.data_ptr(), wd.stride(0)
    a.d_out, a.d_out_stride = do.data_ptr(), do.stride(0)
    a.gate, a.up, a.kept_stride = kg.data_ptr(), ku.data_ptr(), kg.stride(0)
    new = lambda shape, need: (torch.empty(shape, dtype=x.dtype, device=x.device)
                               if need else None)
    d_x = new(x.shape, need_x)
    d_g, d_u = new((dim, hidden), need_in), new((dim, hidden), need_in)
    d_d = new((hidden, dim), need_down)
    a.d_x, a.d_x_stride = _p(d_x), dim
    a.d_w_gate, a.d_w_up, a.d_w_down = _p(d_g), _p(d_u), _p(d_d)
    _call("dn_gated_ffn_bwd", a, True, x.device)
    return GatedFfnGrads(d_x, d_g, d_u, d_d)
