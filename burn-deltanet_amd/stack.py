"""What makes layers a stack: the embedding of token ids, and the joint between a
block and the residual stream (norm after the block, gate, scaled residual, norm
before the next one), each with its gradients.

`embedding` and `block_norm` take part in torch's autograd where an input
requires a gradient, of first order, as the operators of `layer` do; the
`*_backward` functions are for programs that run their own backward pass. Every
computation is a call into libdeltanet_core.so.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor

from . import abi
from .abi import DeltaError
from .autograd import first_order
from .layer import _call, _gpu, _grows, _like, _p, _rows, _shaped, _vector, _x_shape


class BlockNormGrads(NamedTuple):
    d_x: Optional[Tensor]
    d_residual: Optional[Tensor]
    d_pre_weight: Optional[Tensor]
    d_post_weight: Optional[Tensor]
    d_gate: Optional[Tensor]


# -- block_norm ------------------------------------------------------------------


def _gate(gate: Optional[Tensor], x: Tensor, rows: int, dim: int, weight_dtype, what: str):
    """The gate's kind and the tensor that the kernel reads: [dim] in the weights'
    type, one value a row ([..., 1]) or x's shape in x's type. Where dim is 1 a
    gate [..., 1] is x's shape; where x is [dim] one of the weights' type is a channel's."""
    if gate is None:
        return abi.DN_GATE_NONE, None
    if gate.dim() == 1 and (x.dim() != 1 or (gate.shape[0] == dim and gate.dtype == weight_dtype)):
        return abi.DN_GATE_CHANNEL, _vector(gate, dim, weight_dtype, what)
    if gate.dim() and gate.shape[-1] == 1 and dim != 1 and gate.numel() == rows:
        return abi.DN_GATE_TOKEN, _like(gate, x, (rows, 1), what)
    if gate.dim() and gate.shape[-1] == dim and gate.numel() == rows * dim:
        return abi.DN_GATE_FULL, _like(gate, x, (rows, dim), what)
    raise DeltaError(-2, f"{what}: expected [{dim}], [{rows}, 1] or [{rows}, {dim}], "
                         f"got {list(gate.shape)}")


def _block_norm(x, residual, pre_weight, post_weight, gate, residual_scale, eps):
    rows, dim = _x_shape(x)
    tag = abi.dtype_tag(x.dtype)
    x2 = _rows(x, "x")
    r2 = _like(residual, x, (rows, dim), "residual")
    pre = _vector(pre_weight, dim, None, "pre_weight")
    post = _vector(post_weight, dim, pre.dtype, "post_weight")
    kind, g = _gate(gate, x, rows, dim, pre.dtype, "gate")
    out, total = x.new_empty(x.shape), x.new_empty(x.shape)
    a = abi.BlockNormArgs(
        rows, dim, x2.stride(0), r2.stride(0), 0 if g is None else g.stride(0), dim, dim, eps,
        residual_scale, tag, abi.dtype_tag(pre.dtype), kind, x2.data_ptr(), r2.data_ptr(),
        pre.data_ptr(), _p(post), _p(g), total.data_ptr(), out.data_ptr())
    _call("dn_block_norm", a, False, x.device)
    return out, total


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, pre_weight, post_weight, gate, residual_scale, eps):
        out, total = _block_norm(x, residual, pre_weight, post_weight, gate, residual_scale, eps)
        ctx.residual_scale, ctx.eps, ctx.residual_shape = residual_scale, eps, residual.shape
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, total, pre_weight, post_weight, gate)
        return out, total

    @staticmethod
    @first_order
    def backward(ctx, d_out, d_sum):
        x, total, pre_weight, post_weight, gate = ctx.saved_tensors
        need = ctx.needs_input_grad
        if d_out is None and d_sum is None:
            return (None,) * 7
        g = block_norm_backward(d_out, d_sum, x, total, pre_weight, post_weight, gate,
                                ctx.residual_scale, ctx.eps, need_x=need[0], need_residual=need[1],
                                need_weights=need[2] or need[3], need_gate=need[4])
        return (g.d_x, _shaped(g.d_residual, ctx.residual_shape),
                g.d_pre_weight if need[2] else None, g.d_post_weight if need[3] else None,
                g.d_gate, None, None)


def block_norm(x: Tensor, residual: Tensor, pre_weight: Tensor,
               post_weight: Optional[Tensor] = None, gate: Optional[Tensor] = None,
               residual_scale: float = 1.0, eps: float = 1e-5) -> Tuple[Tensor, Tensor]:
    """A block's output x joins the residual stream:

        u = x / sqrt(mean(x²) + eps) * post_weight    (u = x without post_weight)
        sum = residual_scale * residual + gate * u
        out = sum / sqrt(mean(sum²) + eps) * pre_weight

    over the last axis, from the unrounded sum. Returns (out, sum): the next block's
    input and the stream after this one. gate: one value a channel [dim], a token
    [..., 1] or an element (x's shape). post_weight and a channel's gate are of
    pre_weight's type, the other gates of x's. The gradient is taken at the sum as
    it is returned."""
    if _grows(x, residual, pre_weight, post_weight, gate):
        return _BlockNorm.apply(x, residual, pre_weight, post_weight, gate, residual_scale, eps)
    return _block_norm(x, residual, pre_weight, post_weight, gate, residual_scale, eps)


def block_norm_backward(d_out: Optional[Tensor], d_sum: Optional[Tensor], x: Tensor, total: Tensor,
                        pre_weight: Tensor, post_weight: Optional[Tensor] = None,
                        gate: Optional[Tensor] = None, residual_scale: float = 1.0,
                        eps: float = 1e-5, need_x: bool = True, need_residual: bool = True,
                        need_weights: bool = True, need_gate: bool = True) -> BlockNormGrads:
    """The gradients of block_norm at its `sum`; d_out or d_sum may be None (zeros)."""
    rows, dim = _x_shape(x)
    tag = abi.dtype_tag(x.dtype)
    x2 = _rows(x, "x")
    s2 = _like(total, x, (rows, dim), "sum")
    do = _like(d_out, x, (rows, dim), "d_out")
    ds = _like(d_sum, x, (rows, dim), "d_sum")
    pre = _vector(pre_weight, dim, None, "pre_weight")
    post = _vector(post_weight, dim, pre.dtype, "post_weight")
    kind, g = _gate(gate, x, rows, dim, pre.dtype, "gate")
    dev = x.device
    a = abi.BlockNormBwdArgs()
    a.rows, a.dim, a.eps, a.residual_scale = rows, dim, float(eps), float(residual_scale)
    a.dtype, a.weight_dtype, a.gate_kind = tag, abi.dtype_tag(pre.dtype), kind
    a.x, a.x_stride, a.sum, a.sum_stride = x2.data_ptr(), x2.stride(0), s2.data_ptr(), s2.stride(0)
    a.pre_weight, a.post_weight = pre.data_ptr(), _p(post)
    if g is not None:
        a.gate, a.gate_stride = g.data_ptr(), g.stride(0)
    if do is not None:
        a.d_out, a.d_out_stride = do.data_ptr(), do.stride(0)
    if ds is not None:
        a.d_sum, a.d_sum_stride = ds.data_ptr(), ds.stride(0)
    d_x = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
    d_r = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_residual else None
    d_pre = torch.empty_like(pre) if need_weights else None
    d_post = torch.empty_like(post) if need_weights and post is not None else None
    d_g = (torch.empty(gate.shape, dtype=gate.dtype, device=dev)
           if need_gate and gate is not None else None)
    a.d_x, a.d_x_stride, a.d_residual, a.d_residual_stride = _p(d_x), dim, _p(d_r), dim
    a.d_pre_weight, a.d_post_weight, a.d_gate = _p(d_pre), _p(d_post), _p(d_g)
    a.d_gate_stride = dim if kind == abi.DN_GATE_FULL else 1
    _call("dn_block_norm_bwd", a, True, dev)
    return BlockNormGrads(d_x, d_r, d_pre, d_post, d_g)


# -- embedding ---------------------------------------------------------------------


def _ids(tokens: Tensor) -> Tensor:
    if tokens.dtype not in (torch.int64, torch.int32):
        raise DeltaError(-7, f"tokens: expected int64 or int32, got {tokens.dtype}")
    _gpu(tokens, "tokens")
    return tokens if tokens.is_contiguous() else tokens.contiguous()


def _embedding(tokens, table, scale):
    if table.dim() != 2:
        raise DeltaError(-2, f"table: expected [vocab, dim], got {list(table.shape)}")
    ids, (vocab, dim) = _ids(tokens), table.shape
    tag = abi.dtype_tag(table.dtype)
    t = _rows(table, "table")
    out = table.new_empty(tokens.shape + (dim,))
    a = abi.EmbeddingArgs(ids.numel(), vocab, dim, t.stride(0), dim, scale, tag,
                          int(ids.dtype == torch.int64), ids.data_ptr(), t.data_ptr(),
                          out.data_ptr())
    _call("dn_embedding", a, False, table.device)
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, table, scale):
        ctx.vocab, ctx.scale = table.shape[0], scale
        ctx.save_for_backward(tokens)
        return _embedding(tokens, table, scale)

    @staticmethod
    @first_order
    def backward(ctx, d_out):
        tokens, = ctx.saved_tensors
        return None, embedding_backward(d_out, tokens, ctx.vocab, ctx.scale), None


def embedding(tokens: Tensor, table: Tensor, scale: float = 1.0) -> Tensor:
    """scale * table[tokens]: [..., dim] from ids [...] (int64 or int32) and a table
    [vocab, dim]. An id outside [0, vocab), as padding has, gives a row of zeros and
    takes no part in the gradient."""
    if _grows(table):
        return _Embedding.apply(tokens, table, scale)
    return _embedding(tokens, table, scale)


def embedding_backward(d_out: Tensor, tokens: Tensor, vocab: int, scale: float = 1.0) -> Tensor:
    """The table's gradient [vocab, dim], of d_out's type: row v is scale times the sum
    of d_out over the tokens with id v, summed in fp32 in a fixed order (not the tokens'):
    two calls on one device agree to the bit."""
    ids = _ids(tokens)
    if d_out.dim() == 0 or d_out.shape[:-1] != tokens.shape:
        raise DeltaError(-2, f"d_out: expected {list(tokens.shape)} and a last axis, "
                             f"got {list(d_out.shape)}")
    dim = d_out.shape[-1]
    tag = abi.dtype_tag(d_out.dtype)
    d = _rows(d_out if d_out.dim() > 1 else d_out.unsqueeze(0), "d_out")
    d_table = torch.empty((vocab, dim), dtype=d_out.dtype, device=d_out.device)
    a = abi.EmbeddingBwdArgs()
    a.tokens, a.vocab, a.dim, a.scale = ids.numel(), vocab, dim, float(scale)
    a.dtype, a.wide_ids = tag, int(ids.dtype == torch.int64)
    a.ids, a.d_out, a.d_out_stride = ids.data_ptr(), d.data_ptr(), d.stride(0)
    a.d_table, a.d_table_stride = d_table.data_ptr(), dim
    _call("dn_embedding_bwd", a, True, d_out.device)
    return d_table
