"""Refusals of block_norm, embedding and attention: the C entries' checks of their
arguments, before anything touches the device, and the Python mirrors'."""

import ctypes

import pytest
import torch

from conftest import load_package
from test_abi import fake_pointers

dn = load_package()
abi = dn.abi
FAKE = 0x1000  # never dereferenced: every case fails its checks first

NORM = (abi.BlockNormArgs, "dn_block_norm",
        dict(rows=4, dim=8, x_stride=8, residual_stride=8, gate_stride=8, sum_stride=8,
             out_stride=8, eps=1e-5, residual_scale=1.0),
        ["x", "residual", "pre_weight", "post_weight", "sum", "out"])
NORM_BWD = (abi.BlockNormBwdArgs, "dn_block_norm_bwd",
            dict(rows=4, dim=8, x_stride=8, sum_stride=8, gate_stride=8, d_out_stride=8,
                 d_sum_stride=8, d_x_stride=8, d_residual_stride=8, d_gate_stride=8, eps=1e-5,
                 residual_scale=1.0),
            ["x", "sum", "pre_weight", "post_weight", "d_out", "d_sum", "d_x", "d_residual",
             "d_pre_weight", "d_post_weight"])
EMB = (abi.EmbeddingArgs, "dn_embedding",
       dict(tokens=4, vocab=10, dim=8, table_stride=8, out_stride=8, scale=1.0),
       ["ids", "table", "out"])
EMB_BWD = (abi.EmbeddingBwdArgs, "dn_embedding_bwd",
           dict(tokens=4, vocab=10, dim=8, d_out_stride=8, d_table_stride=8, scale=1.0),
           ["ids", "d_out", "d_table"])
ATT = (abi.AttentionArgs, "dn_attention",
       dict(tokens=4, key_rows=4, sequences=1, nheads=4, kv_heads=2, head_dim=8, q_stride=32,
            k_stride=16, v_stride=16, out_stride=32, scale=float("nan"), causal=1),
       ["q", "k", "v", "offsets", "out"])
ATT_BWD = (abi.AttentionBwdArgs, "dn_attention_bwd",
           dict(tokens=4, sequences=1, nheads=4, kv_heads=2, head_dim=8, q_stride=32, k_stride=16,
                v_stride=16, out_stride=32, d_out_stride=32, d_q_stride=32, d_k_stride=16,
                d_v_stride=16, scale=float("nan"), causal=1),
           ["q", "k", "v", "offsets", "out", "lse", "d_out", "d_q", "d_k", "d_v"])
INF = float("inf")


@pytest.mark.parametrize("entry,over,code,msg", [
    (NORM, dict(rows=-1), -2, "rows must not be negative"),
    (NORM, dict(dim=0), -2, "width"),
    (NORM, dict(dim=1 << 25), -2, "tensor too large"),
    (NORM, dict(dtype=2), -7, "dtype"),
    (NORM, dict(weight_dtype=3), -7, "dtype"),
    (NORM, dict(eps=-1.0), -2, "eps"),
    (NORM, dict(residual_scale=INF), -2, "residual_scale"),
    (NORM, dict(residual=None), -6, "residual is NULL"),
    (NORM, dict(pre_weight=None), -6, "pre_weight is NULL"),
    (NORM, dict(sum=None), -6, "sum is NULL"),
    (NORM, dict(out_stride=7), -2, "cannot be 7 apart"),
    (NORM, dict(gate_kind=4), -2, "gate_kind"),
    (NORM, dict(gate_kind=1), -6, "gate is NULL"),
    (NORM, dict(gate_kind=2, gate=FAKE, gate_stride=0), -2, "gate"),
    (NORM, dict(gate_kind=3, gate=FAKE, gate_stride=5), -2, "gate"),
    (NORM_BWD, dict(x=None), -6, "x is NULL"),
    (NORM_BWD, dict(d_gate=FAKE), -2, "without a gate"),
    (NORM_BWD, dict(post_weight=None), -6, "without post_weight"),
    (NORM_BWD, dict(gate_kind=3, gate=FAKE, d_gate=FAKE, d_gate_stride=3), -2, "d_gate"),
    (NORM_BWD, dict(d_residual_stride=1), -2, "d_residual"),
    (NORM_BWD, dict(workspace=FAKE, workspace_bytes=1), -8, "workspace too small"),
    (NORM_BWD, dict(workspace=FAKE + 8, workspace_bytes=1 << 20), -8, "16-byte"),
    (EMB, dict(tokens=-1), -2, "tokens"),
    (EMB, dict(tokens=(1 << 28) + 1), -2, "tensor too large"),
    (EMB, dict(vocab=0), -2, "width"),
    (EMB, dict(vocab=(1 << 24) + 1), -2, "tensor too large"),
    (EMB, dict(dim=(1 << 23) + 1, table_stride=1 << 24, out_stride=1 << 24), -2,
     "tensor too large"),
    (EMB, dict(scale=INF), -2, "scale"),
    (EMB, dict(ids=None), -6, "ids is NULL"),
    (EMB, dict(table_stride=4), -2, "table"),
    (EMB, dict(dtype=2), -7, "dtype"),
    (EMB_BWD, dict(d_table=None), -6, "d_table is NULL"),
    (EMB_BWD, dict(d_out_stride=1), -2, "d_out"),
    (EMB_BWD, dict(workspace=FAKE, workspace_bytes=16), -8, "workspace too small"),
    (ATT, dict(tokens=-1), -2, "negative"),
    (ATT, dict(nheads=3), -2, "multiple"),
    (ATT, dict(kv_heads=0), -2, "multiple"),
    (ATT, dict(head_dim=0), -2, "head_dim"),
    (ATT, dict(head_dim=257), -9, "head_dim"),
    (ATT, dict(tokens=1 << 30), -2, "tensor too large"),
    (ATT, dict(tokens=1 << 26, nheads=4, kv_heads=4), -2, "tensor too large"),
    (ATT, dict(sequences=1 << 29), -2, "tensor too large"),
    (ATT, dict(scale=0.0), -2, "scale"),
    (ATT, dict(scale=-1.0), -2, "scale"),
    (ATT, dict(scale=INF), -2, "scale"),
    (ATT, dict(scale=1e-60), -2, "scale"),
    (ATT, dict(dtype=2), -7, "dtype"),
    (ATT, dict(offsets=None, sequences=3), -2, "equal lengths"),
    (ATT, dict(offsets=None, sequences=0), -2, "equal lengths"),
    (ATT, dict(key_rows=5), -2, "queries' rows"),
    (ATT, dict(key_starts=FAKE), -6, "go together"),
    (ATT, dict(key_starts=FAKE, key_lengths=FAKE, key_rows=-1), -2, "key_rows"),
    (ATT, dict(q_stride=31), -2, "q"),
    (ATT, dict(v=None), -6, "v is NULL"),
    (ATT_BWD, dict(lse=None), -6, "lse is NULL"),
    (ATT_BWD, dict(d_k_stride=15), -2, "d_k"),
    (ATT_BWD, dict(head_dim=300, q_stride=4800, k_stride=4800, v_stride=4800, out_stride=4800,
                   d_out_stride=4800), -9, "head_dim"),
    (ATT_BWD, dict(workspace=FAKE, workspace_bytes=8), -8, "workspace too small"),
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
    for name in ("dn_block_norm", "dn_block_norm_bwd", "dn_embedding", "dn_embedding_bwd",
                 "dn_attention", "dn_attention_bwd"):
        assert getattr(L, name)(None, None) == -6


def test_nothing_to_do():
    """No rows: the forwards, and the gradients of rows alone, return at once."""
    L = abi.lib()
    for struct, name, sizes, pointers in (NORM, EMB, ATT, ATT_BWD):
        a = struct()
        for k, v in sizes.items():
            setattr(a, k, v)
        for k in pointers:
            setattr(a, k, FAKE)
        setattr(a, "rows" if name.startswith("dn_block") else "tokens", 0)
        if name == "dn_attention":
            a.key_rows = 0
        assert getattr(L, name)(ctypes.byref(a), None) == 0


def test_python_needs_the_gpu():
    x, w = torch.zeros(2, 8), torch.ones(8)
    q = torch.zeros(4, 2, 8)
    off = torch.tensor([0, 4], dtype=torch.int32)
    for call in (lambda: dn.block_norm(x, x, w), lambda: dn.embedding(torch.tensor([1]), x),
                 lambda: dn.embedding_backward(x, torch.tensor([1, 0]), 3),
                 lambda: dn.attention(q, q, q, off),
                 lambda: dn.attention_backward(q, q, q, q, q, q[..., 0], off)):
        with pytest.raises(dn.DeltaError) as e:
            call()
        assert e.value.code == -6


def on(*shape, dtype=torch.float32):
    return torch.ones(shape, dtype=dtype, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("call,code,msg", [
    (lambda: dn.block_norm(on(2, 8), on(2, 7), on(8)), -2, "residual"),
    (lambda: dn.block_norm(on(2, 8), on(2, 8, dtype=torch.bfloat16), on(8)), -7, "residual"),
    (lambda: dn.block_norm(on(2, 8), on(2, 8), on(7)), -2, "pre_weight"),
    (lambda: dn.block_norm(on(2, 8), on(2, 8), on(8), on(8, dtype=torch.bfloat16)), -7,
     "post_weight"),
    (lambda: dn.block_norm(on(2, 8), on(2, 8), on(8), None, on(3, 1)), -2, "gate"),
    (lambda: dn.block_norm(on(2, 8), on(2, 8), on(8), None, on(2, 1, dtype=torch.bfloat16)), -7,
     "gate"),
    (lambda: dn.block_norm(on(2, 8), on(2, 8), on(8), None, on()), -2, "gate"),
    (lambda: dn.block_norm(on(2, 8).half(), on(2, 8).half(), on(8)), -7, "dtype"),
    (lambda: dn.block_norm_backward(on(3, 8), None, on(2, 8), on(2, 8), on(8)), -2, "d_out"),
    (lambda: dn.embedding(on(2), on(4, 8)), -7, "tokens"),
    (lambda: dn.embedding(on(2, dtype=torch.long), on(8)), -2, "table"),
    (lambda: dn.embedding(torch.ones(2, dtype=torch.long), on(4, 8)), -6, "GPU"),
    (lambda: dn.embedding_backward(on(3, 8), on(2, dtype=torch.long), 4), -2, "d_out"),
    (lambda: dn.embedding_backward(on(2, 8), on(2, dtype=torch.long), 0), -2, "width"),
    (lambda: dn.attention(on(4, 2, 8), on(4, 2, 8), on(4, 2, 8)), -2, "without offsets"),
    (lambda: dn.attention(on(4, 3, 8), on(4, 2, 8), on(4, 2, 8), on(2, dtype=torch.int32)), -2,
     "multiple"),
    (lambda: dn.attention(on(4, 2, 8), on(4, 2, 7), on(4, 2, 7), on(2, dtype=torch.int32)), -2,
     "k, v"),
    (lambda: dn.attention(on(4, 2, 8), on(5, 2, 8), on(5, 2, 8), on(2, dtype=torch.int32)), -2,
     "without key"),
    (lambda: dn.attention(on(4, 2, 300), on(4, 2, 300), on(4, 2, 300), on(2, dtype=torch.int32)),
     -9, "head_dim"),
    (lambda: dn.attention(on(4, 2, 8), on(4, 2, 8).bfloat16(), on(4, 2, 8),
                          on(2, dtype=torch.int32)), -7, "k"),
    (lambda: dn.attention(on(4, 2, 8), on(4, 2, 8), on(4, 2, 8), on(2)), -7, "offsets"),
    (lambda: dn.attention(on(4, 2, 8), on(4, 2, 8), on(4, 2, 8), on(2, dtype=torch.int32),
                          dn.KeySpans(on(2, dtype=torch.int32), on(1, dtype=torch.int32))), -2,
     "keys.starts"),
    (lambda: dn.attention(on(4, 2, 8), on(4, 2, 8), on(4, 2, 8), on(2, dtype=torch.int32), None,
                          0.0), -2, "scale"),
    (lambda: dn.attention(on(2, 4, 2, 8), on(2, 3, 2, 8), on(2, 3, 2, 8)), -2, "k, v"),
    (lambda: dn.attention_backward(on(4, 2, 8), on(4, 2, 8), on(4, 2, 8), on(4, 2, 8),
                                   on(4, 2, 8), on(4, 1), on(2, dtype=torch.int32)), -2, "lse"),
])
def test_python_refuses_on_the_gpu(call, code, msg):
    with pytest.raises(dn.DeltaError) as e:
        call()
    assert e.value.code == code and msg in str(e.value)
