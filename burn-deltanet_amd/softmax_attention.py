"""Softmax attention with grouped heads, for the attention layers that a stack has
between its delta-rule layers: over whole packed sequences, with its gradients, and
over cached keys for the tokens that follow.

`attention` takes part in torch's autograd where an input requires a gradient, of
first order, as the operators of `layer` do; `attention_forward` and
`attention_backward` are the two halves for programs that run their own backward
pass. Every computation is a call into libdeltanet_core.so.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor

from . import abi
from .abi import DeltaError, nan_scale
from .autograd import first_order
from .layer import _call, _gpu, _grows, _p


LEAST_GRADIENT_SCALE = 2.0 ** -96  # dn_attention_bwd's (deltanet_core.h)


class KeySpans(NamedTuple):
    """The rows of k and v that each sequence's queries attend to: lengths[s] rows from
    starts[s] on (int32, [sequences]). Spans may overlap, as where sequences share
    their first keys."""

    starts: Tensor
    lengths: Tensor


class AttentionGrads(NamedTuple):
    d_q: Optional[Tensor]
    d_k: Optional[Tensor]
    d_v: Optional[Tensor]


def _heads(t: Tensor, what: str) -> Tensor:
    """`t` as [rows, heads, dim] with a row's heads side by side: a view where its
    strides allow one, else a copy."""
    _gpu(t, what)
    if t.dim() < 3:
        raise DeltaError(-2, f"{what}: expected [..., heads, dim], got {list(t.shape)}")
    if t.dim() > 3:
        t = t.reshape((t.shape[:-2].numel(),) + t.shape[-2:])
    n, h, d = t.shape
    s0, s1, s2 = t.stride()
    return t if (s2 == 1 or d <= 1) and (s1 == d or h <= 1) and (n <= 1 or s0 >= h * d) \
        else t.contiguous()


def _ints(t: Tensor, n: int, what: str) -> Tensor:
    _gpu(t, what)
    if t.dtype not in (torch.int32, torch.int64):
        raise DeltaError(-7, f"{what}: expected int32 or int64, got {t.dtype}")
    if tuple(t.shape) != (n,):
        raise DeltaError(-2, f"{what}: expected [{n}], got {list(t.shape)}")
    if t.dtype == torch.int64:
        t = t.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def _check(q, k, v, offsets, spans):
    """The operands as rows, and how many sequences they hold. `spans`: whether the keys
    are others than the queries' rows."""
    for t, what in ((k, "k"), (v, "v")):
        if t.dtype != q.dtype:
            raise DeltaError(-7, f"{what}: expected {q.dtype}, got {t.dtype}")
    abi.dtype_tag(q.dtype)
    q3, k3, v3 = _heads(q, "q"), _heads(k, "k"), _heads(v, "v")
    if k3.shape != v3.shape or k3.shape[2] != q3.shape[2]:
        raise DeltaError(-2, f"k, v: expected [..., heads, {q3.shape[2]}] of one shape, "
                             f"got {list(k.shape)} and {list(v.shape)}")
    if not spans and (k3.shape[0] != q3.shape[0]
                      or (offsets is None and k.shape[:-2] != q.shape[:-2])):
        raise DeltaError(-2, f"k, v: expected the queries' rows {list(q.shape[:-2])} without key "
                             f"spans, got {list(k.shape[:-2])}")
    if offsets is None:
        if q.dim() != 4:
            raise DeltaError(-2, "q: expected [batch, sequence, heads, dim] without offsets")
        return q3, k3, v3, None, q.shape[0]
    if offsets.dim() != 1 or offsets.shape[0] < 1:
        raise DeltaError(-2, f"offsets: expected [sequences + 1], got {list(offsets.shape)}")
    n = offsets.shape[0] - 1
    return q3, k3, v3, _ints(offsets, n + 1, "offsets"), n


def _attention(q, k, v, offsets, keys, scale, causal, keep):
    q3, k3, v3, off, n = _check(q, k, v, offsets, keys is not None)
    a = abi.AttentionArgs()
    if keys is not None:
        starts = _ints(keys.starts, n, "keys.starts")
        lengths = _ints(keys.lengths, n, "keys.lengths")
        a.key_starts, a.key_lengths = starts.data_ptr(), lengths.data_ptr()
    a.tokens, a.nheads, a.head_dim = q3.shape
    a.key_rows, a.kv_heads, a.sequences = k3.shape[0], k3.shape[1], n
    a.scale, a.causal, a.dtype = nan_scale(scale), int(bool(causal)), abi.dtype_tag(q.dtype)
    a.q, a.q_stride, a.k, a.k_stride = q3.data_ptr(), q3.stride(0), k3.data_ptr(), k3.stride(0)
    a.v, a.v_stride, a.offsets = v3.data_ptr(), v3.stride(0), _p(off)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    a.out, a.out_stride = out.data_ptr(), q3.shape[1] * q3.shape[2]
    lse = None
    if keep:
        lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device)
        a.lse = lse.data_ptr()
    _call("dn_attention", a, True, q.device)
    return out, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, scale, causal):
        out, lse = _attention(q, k, v, offsets, None, scale, causal, True)
        ctx.scale, ctx.causal = scale, causal
        ctx.save_for_backward(q, k, v, offsets, out, lse)
        return out

    @staticmethod
    @first_order
    def backward(ctx, d_out):
        q, k, v, offsets, out, lse = ctx.saved_tensors
        need = ctx.needs_input_grad
        g = attention_backward(d_out, q, k, v, out, lse, offsets, ctx.scale, ctx.causal,
                               need_q=need[0], need_k=need[1], need_v=need[2])
        return g.d_q, g.d_k, g.d_v, None, None, None


def attention(q: Tensor, k: Tensor, v: Tensor, offsets: Optional[Tensor] = None,
              keys: Optional[KeySpans] = None, scale: Optional[float] = None,
              causal: bool = True) -> Tensor:
    """softmax(scale q kᵀ) v for every head; q [tokens, heads, dim], k and v
    [rows, kv_heads, dim], head h reads key head h // (heads / kv_heads), dim up to 256.

    offsets (int32, [sequences + 1], from 0 on) says where the packed sequences start;
    without it the operands are [batch, sequence, heads, dim]. Without `keys` a
    sequence's keys are its own rows; with it the queries are the last tokens over
    longer spans of a cache (no gradient). Causal: the i-th of n queries over m keys
    sees keys 0 … i + m − n. scale: 1/sqrt(dim) unless given; gradients need 2⁻⁹⁶ or
    more. A row that sees no key, or none with a score above −inf, and every row behind
    the last sequence, is zeros; keys that a row does not see have no influence on it,
    whatever they hold. The numbers in offsets and spans stay on the GPU and are not
    checked: beyond the tensors' ends they are cut off."""
    if _grows(q, k, v):
        if keys is not None:
            raise DeltaError(-9, "attention over key spans has no gradient")
        if scale is not None and 0 < scale < LEAST_GRADIENT_SCALE:
            raise DeltaError(-9, "attention's gradients need a scale of at least 2^-96")
        return _Attention.apply(q, k, v, offsets, scale, causal)
    return _attention(q, k, v, offsets, keys, scale, causal, False)[0]


def attention_forward(q: Tensor, k: Tensor, v: Tensor, offsets: Optional[Tensor] = None,
                      keys: Optional[KeySpans] = None, scale: Optional[float] = None,
                      causal: bool = True) -> Tuple[Tensor, Tensor]:
    """attention and, in fp32, the natural log of every row's sum of exp(scale q kᵀ)
    (−inf where it sees no key): [..., heads], what its backward needs beside its inputs."""
    return _attention(q, k, v, offsets, keys, scale, causal, True)


def attention_backward(d_out: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor,
                       offsets: Optional[Tensor] = None, scale: Optional[float] = None,
                       causal: bool = True, need_q: bool = True, need_k: bool = True,
                       need_v: bool = True) -> AttentionGrads:
    """The gradients of attention without key spans."""
    q3, k3, v3, off, n = _check(q, k, v, offsets, False)
    for t, what in ((d_out, "d_out"), (out, "out")):
        if t.dtype != q.dtype:
            raise DeltaError(-7, f"{what}: expected {q.dtype}, got {t.dtype}")
        if t.shape != q.shape:
            raise DeltaError(-2, f"{what}: expected {list(q.shape)}, got {list(t.shape)}")
    if lse.dtype != torch.float32:
        raise DeltaError(-7, f"lse: expected {torch.float32}, got {lse.dtype}")
    if lse.shape != q.shape[:-1]:
        raise DeltaError(-2, f"lse: expected {list(q.shape[:-1])}, got {list(lse.shape)}")
    _gpu(lse, "lse")
    lse = lse.contiguous()
    o3, d3 = _heads(out, "out"), _heads(d_out, "d_out")
    new = lambda t, need: (torch.empty(t.shape, dtype=t.dtype, device=t.device)
                           if need else None)
    d_q, d_k, d_v = new(q, need_q), new(k, need_k), new(v, need_v)
    a = abi.AttentionBwdArgs()
    a.tokens, a.nheads, a.head_dim = q3.shape
    a.kv_heads, a.sequences = k3.shape[1], n
    a.scale, a.causal, a.dtype = nan_scale(scale), int(bool(causal)), abi.dtype_tag(q.dtype)
    a.q, a.q_stride, a.k, a.k_stride = q3.data_ptr(), q3.stride(0), k3.data_ptr(), k3.stride(0)
    a.v, a.v_stride, a.offsets = v3.data_ptr(), v3.stride(0), _p(off)
    a.out, a.out_stride, a.d_out, a.d_out_stride = (o3.data_ptr(), o3.stride(0), d3.data_ptr(),
                                                    d3.stride(0))
    a.lse, a.d_q, a.d_k, a.d_v = lse.data_ptr(), _p(d_q), _p(d_k), _p(d_v)
    a.d_q_stride = q3.shape[1] * q3.shape[2]
    a.d_k_stride = a.d_v_stride = k3.shape[1] * k3.shape[2]
    _call("dn_attention_bwd", a, True, q.device)
    return AttentionGrads(d_q, d_k, d_v)
