"""Refusals of the operators around the mixer: the C entries' checks of their
arguments, before anything touches the device, and the Python mirrors'."""

import ctypes

import pytest
import torch

from conftest import load_package
from test_abi import fake_pointers

dn = load_package()
abi = dn.abi
FAKE = 0x1000  # never dereferenced: every case fails its checks first

NORM = (abi.AddRmsNormArgs, "dn_add_rms_norm",
        dict(rows=4, dim=8, x_stride=8, residual_stride=8, sum_stride=8, out_stride=8, eps=1e-5),
        ["x", "weight", "out", "scale"])
NORM_BWD = (abi.AddRmsNormBwdArgs, "dn_add_rms_norm_bwd",
            dict(rows=4, dim=8, sum_stride=8, d_out_stride=8, d_sum_stride=8, d_x_stride=8,
                 eps=1e-5), ["sum", "weight", "d_out", "d_x", "d_weight"])
LINEAR = (abi.LinearArgs, "dn_linear",
          dict(rows=4, in_dim=8, out_dim=6, x_stride=8, weight_stride=6, residual_stride=6,
               out_stride=6, preact_stride=6), ["x", "weight", "out"])
LINEAR_BWD = (abi.LinearBwdArgs, "dn_linear_bwd",
              dict(rows=4, in_dim=8, out_dim=6, x_stride=8, weight_stride=6, d_out_stride=6,
                   preact_stride=6, d_x_stride=8), ["d_out", "x", "weight", "d_x", "d_weight"])
FFN = (abi.GatedFfnArgs, "dn_gated_ffn",
       dict(rows=4, dim=8, hidden=6, x_stride=8, w_in_stride=6, w_down_stride=8,
            residual_stride=8, out_stride=8, kept_stride=6),
       ["x", "w_gate", "w_up", "w_down", "out"])
FFN_BWD = (abi.GatedFfnBwdArgs, "dn_gated_ffn_bwd",
           dict(rows=4, dim=8, hidden=6, x_stride=8, w_in_stride=6, w_down_stride=8,
                d_out_stride=8, kept_stride=6, d_x_stride=8),
           ["d_out", "x", "w_gate", "w_up", "w_down", "gate", "up", "d_x", "d_w_gate", "d_w_up",
            "d_w_down"])
BIG = 1 << 25


@pytest.mark.parametrize("entry,over,code,msg", [
    (NORM, dict(rows=-1), -2, "rows must not be negative"),
    (NORM, dict(dim=0), -2, "width"),
    (NORM, dict(dim=BIG), -2, "tensor too large"),
    (NORM, dict(rows=1 << 31), -2, "tensor too large"),
    (NORM, dict(dtype=2), -7, "dtype"),
    (NORM, dict(weight_dtype=5), -7, "dtype"),
    (NORM, dict(out_dtype=1), -7, "out_dtype"),
    (NORM, dict(eps=-1.0), -2, "eps"),
    (NORM, dict(eps=float("nan")), -2, "eps"),
    (NORM, dict(x=None), -6, "x is NULL"),
    (NORM, dict(weight=None), -6, "weight is NULL"),
    (NORM, dict(x_stride=7), -2, "cannot be 7 apart"),
    (NORM, dict(residual=FAKE, residual_stride=0), -2, "residual"),
    (NORM, dict(out_dtype=2, scale=None), -6, "scales"),
    (NORM_BWD, dict(d_x=None), -6, "d_x is NULL"),
    (NORM_BWD, dict(d_out_stride=4), -2, "d_out"),
    (NORM_BWD, dict(workspace=FAKE, workspace_bytes=1), -8, "workspace too small"),
    (NORM_BWD, dict(workspace=FAKE + 4, workspace_bytes=1 << 20), -8, "16-byte"),
    (LINEAR, dict(out_dim=0), -2, "width"),
    (LINEAR, dict(in_dim=1 << 23, out_dim=1 << 23, x_stride=1 << 23, weight_stride=1 << 23,
                  out_stride=1 << 23), -2, "tensor too large"),
    (LINEAR, dict(dtype=3), -7, "dtype"),
    (LINEAR, dict(dtype=1), -7, "out_dtype must be the operands' dtype"),
    (LINEAR, dict(activation=3), -2, "activation"),
    (LINEAR, dict(activation=-1), -2, "activation"),
    (LINEAR, dict(weight=None), -6, "weight is NULL"),
    (LINEAR, dict(weight_stride=5), -2, "weight"),
    (LINEAR, dict(preact=FAKE, preact_stride=2), -2, "preact"),
    (LINEAR, dict(dtype=2, weight_stride=8), -6, "scales"),
    (LINEAR, dict(dtype=2, x_scale=FAKE, weight_scale=FAKE, weight_stride=8), -9, "16-byte"),
    (LINEAR, dict(dtype=2, x_scale=FAKE, weight_scale=FAKE, x_stride=16, weight_stride=16,
                  x=FAKE + 8), -9, "16-byte"),
    (LINEAR_BWD, dict(activation=1), -6, "preact is NULL"),
    (LINEAR_BWD, dict(dtype=2), -7, "dtype"),
    (LINEAR_BWD, dict(x=None), -6, "x is NULL"),
    (FFN, dict(hidden=0), -2, "width"),
    (FFN, dict(w_up=None), -6, "w_up is NULL"),
    (FFN, dict(gate=FAKE), -6, "kept together"),
    (FFN, dict(w_in_stride=4), -2, "w_gate"),
    (FFN, dict(activation=7), -2, "activation"),
    (FFN_BWD, dict(up=None), -6, "up is NULL"),
    (FFN_BWD, dict(d_w_up=None), -6, "formed together"),
    (FFN_BWD, dict(d_x_stride=3), -2, "d_x"),
])
@fake_pointers
def test_c_entries_refuse(entry, over, code, msg):
    struct, name, sizes, pointers = entry
    a = struct()
    for k, v in sizes.items():
        setattr(a, k, v)
    for k in pointers:
        setattr(a, k, FAKE)
    for k, v in over.items():
        setattr(a, k, v)
    L = abi.lib()
    assert getattr(L, name)(ctypes.byref(a), None) == code
    assert msg in L.dn_last_error().decode()
    if hasattr(L, name + "_workspace_bytes") and code != -8:
        assert getattr(L, name + "_workspace_bytes")(ctypes.byref(a)) == 0


def test_null_arguments():
    L = abi.lib()
    for name in ("dn_add_rms_norm", "dn_add_rms_norm_bwd", "dn_linear", "dn_linear_bwd",
                 "dn_gated_ffn", "dn_gated_ffn_bwd"):
        assert getattr(L, name)(None, None) == -6


def test_nothing_to_do():
    """No rows: the forwards and a gradient of the rows alone return at once."""
    for struct, name, sizes, _ in (NORM, LINEAR, FFN):
        a = struct()
        for k, v in sizes.items():
            setattr(a, k, v)
        a.rows = 0
        a.weight = a.w_gate = a.w_up = a.w_down = FAKE
        assert getattr(abi.lib(), name)(ctypes.byref(a), None) == 0


X = torch.zeros(4, 8)


@pytest.mark.parametrize("call,code,msg", [
    (lambda: dn.linear(X, torch.zeros(8, 6)), -6, "must live on the GPU"),
    (lambda: dn.linear(X, torch.zeros(7, 6)), -2, "weight"),
    (lambda: dn.linear(torch.zeros(()), torch.zeros(7, 6)), -2, "scalar"),
    (lambda: dn.linear(X.double(), torch.zeros(8, 6).double()), -7, "float64"),
    (lambda: dn.add_rms_norm(X, None, torch.zeros(8)), -6, "must live on the GPU"),
    (lambda: dn.add_rms_norm(X.half(), None, torch.zeros(8)), -7, "float16"),
    (lambda: dn.gated_ffn(X, torch.zeros(8), torch.zeros(8, 6), torch.zeros(6, 8)), -6,
     "must live on the GPU"),
    (lambda: dn.linear_8bit(dn.Rows8(X, torch.zeros(4)), dn.Rows8(X, torch.zeros(4))), -7,
     "codes"),
    (lambda: dn.quantize_rows(torch.zeros(3)), -2, "rows, dim"),
])
def test_python_refuses_before_the_library(call, code, msg):
    with pytest.raises(dn.DeltaError, match=msg) as e:
        call()
    assert e.value.code == code


@pytest.mark.gpu
@pytest.mark.parametrize("call,code,msg", [
    (lambda x: dn.linear(x, torch.zeros(8, 6, device="cuda").bfloat16()), -7, "weight"),
    (lambda x: dn.linear(x, torch.zeros(8, 6, device="cuda"), torch.zeros(5, device="cuda")), -2,
     "bias"),
    (lambda x: dn.linear(x, torch.zeros(8, 6, device="cuda"), residual=x), -2, "residual"),
    (lambda x: dn.linear(x, torch.zeros(8, 6, device="cuda"),
                         residual=torch.zeros(6, device="cuda")), -2, "residual"),
    (lambda x: dn.linear_backward(torch.zeros(4, 6, device="cuda"), x,
                                  torch.zeros(8, 6, device="cuda"),
                                  activation=dn.Activation.SILU), -6, "preact"),
    (lambda x: dn.add_rms_norm(x, x[:2], torch.zeros(8, device="cuda")), -2, "residual"),
    (lambda x: dn.add_rms_norm(x, None, torch.zeros(7, device="cuda")), -2, "weight"),
    (lambda x: dn.gated_ffn(x, torch.zeros(8, 6, device="cuda"), torch.zeros(8, 5, device="cuda"),
                            torch.zeros(6, 8, device="cuda")), -2, "w_up"),
    (lambda x: dn.linear_8bit(dn.quantize_rows(x), dn.quantize_rows(x[:, :4])), -2, "weight"),
    (lambda x: dn.linear_8bit(
        dn.Rows8(torch.zeros(4, 8, device="cuda").to(torch.float8_e4m3fn),
                 torch.ones(4, device="cuda")), dn.quantize_rows(x)), -9, "16-byte"),
])
def test_python_refuses_on_the_gpu(call, code, msg):
    with pytest.raises(dn.DeltaError, match=msg) as e:
        call(torch.zeros(4, 8, device="cuda"))
    assert e.value.code == code
