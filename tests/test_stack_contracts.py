"""What attention, block_norm and embedding promise at the edges of what they accept:
refusals, values that are not finite, sizes where a kernel's other form takes over."""

import ctypes

import pytest
import torch

import stack_util as su
from conftest import load_package
from layer_util import F, U, check
from test_abi import fake_pointers
from test_gpu_attention import check_all, made, packed, wide
from test_stack_checks import ATT, ATT_BWD, FAKE

dn = load_package()
abi = dn.abi
gpu = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def filled(entry, **over):
    struct, _, sizes, pointers = entry
    a = struct()
    for k, v in {**sizes, **dict.fromkeys(pointers, FAKE), **over}.items():
        setattr(a, k, v)
    return a


def refusal(entry, **over):
    """The entry's code and message; nothing touches the device."""
    L = abi.lib()
    rc = getattr(L, entry[1])(ctypes.byref(filled(entry, **over)), None)
    return rc, L.dn_last_error().decode()


def ints(*xs):
    return torch.tensor(xs, dtype=torch.int32, device="cuda")


# -- attention: the scale ------------------------------------------------------------


@fake_pointers
def test_scales_that_leave_fp32_are_refused():
    """Gradients start their scores at the log-sum over the scale, and all exponents are
    taken of scale log2(e): both have to be fp32 numbers."""
    for scale in (2.0 ** -97, 2e-38, 1e-40):
        rc, message = refusal(ATT_BWD, scale=scale)
        assert rc == -9 and "2^-96" in message
        assert abi.lib().dn_attention_bwd_workspace_bytes(
            ctypes.byref(filled(ATT_BWD, scale=scale))) == 0
    for entry in (ATT, ATT_BWD):
        rc, message = refusal(entry, scale=2.5e38)
        assert rc == -2 and "scale" in message
    # Within the limits the next check is reached.
    small = dict(workspace=FAKE, workspace_bytes=8)
    for scale in (2.0 ** -96, 2.3e38):
        assert refusal(ATT_BWD, scale=scale, **small)[0] == -8


@gpu
def test_gradients_of_a_small_scale_are_refused_in_time():
    """Before the forward, not in the backward pass."""
    q = torch.ones(4, 1, 8, device="cuda", requires_grad=True)
    with pytest.raises(dn.DeltaError, match="2\\^-96") as e:
        dn.attention(q, q, q, ints(0, 4), None, 2.0 ** -97)
    assert e.value.code == -9
    assert dn.attention(q.detach(), q.detach(), q.detach(), ints(0, 4), None, 2.0 ** -97).all()


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_gradients_at_the_smallest_scale(dtype):
    """All weights are alike: d_v is a mean of d_out. Sums that start at the log-sum (6.9)
    and take 64 products are off by 2 (64 + 4) u 6.9 = 940 u, for which the bound's term
    for the weights' own sum, 2 (1000 + 8) u, has room."""
    check_all(*packed([1000], 0, 1, 1, 64, dtype), scale=2.0 ** -96, causal=False)


# -- attention: values that are not finite -------------------------------------------


@gpu
@pytest.mark.parametrize("rows", [31, 32, 33, 63, 64, 65, 191])
@pytest.mark.parametrize("heads,kv,dim,dtype", [
    (1, 1, 64, BF), (1, 1, 64, F32), (2, 1, 128, BF), (3, 1, 40, F32), (1, 1, 256, F32),
    (1, 1, 256, BF), (2, 2, 128, F32)])
def test_a_key_without_weight(rows, heads, kv, dim, dtype):
    """A key whose scores are all -inf has a weight of zero: its d_k and d_v are zeros,
    however many rows a tile lacks, and the other keys' are those of a batch whose rows
    skip it."""
    q, k, v, off, spans, do = packed([rows], 0, heads, kv, dim, dtype, seed=3)
    q[:, :, 5] = (q[:, :, 5].abs() + 0.125).to(dtype)
    at = 20
    k[at, 0, 5] = -INF
    for causal in (True, False):
        out, lse = dn.attention_forward(q, k, v, off, None, None, causal)
        assert out.isfinite().all() and lse.isfinite().all()
        g = dn.attention_backward(do, q, k, v, out, lse, off, None, causal)
        assert not g.d_k[at, 0].any() and not g.d_v[at, 0].any()
        assert g.d_k.isfinite().all() and g.d_v.isfinite().all()
        far = k.clone()  # a finite key as far away: the same weights of zero
        far[at, 0] = 0
        far[at, 0, 5] = -2e4
        out2, lse2 = dn.attention_forward(q, far, v, off, None, None, causal)
        want = dn.attention_backward(do, q, far, v, out2, lse2, off, None, causal)
        assert torch.equal(out, out2) and torch.equal(lse, lse2)
        assert torch.equal(g.d_k, want.d_k) and torch.equal(g.d_v, want.d_v)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_row_without_a_finite_score(dtype, dim):
    """The first row sees the first key alone, with a score of -inf: zeros, a log-sum of
    -inf, and no part in any gradient; the others are as if it were not there."""
    q, k, v, off, spans, do = packed([70], 0, 1, 1, dim, dtype, seed=4)
    q[:, :, 5] = (q[:, :, 5].abs() + 0.125).to(dtype)
    k[0, 0, 5] = -INF
    out, lse = dn.attention_forward(q, k, v, off)
    assert not out[0].any() and lse[0] == -INF and lse[1:].isfinite().all()
    g = dn.attention_backward(do, q, k, v, out, lse, off)
    rest = [i for i in range(dim) if i != 5]  # 0 (-inf) there
    assert not g.d_q[0, 0, rest].any() and not g.d_k[0].any() and not g.d_v[0].any()
    one = [t[1:].clone() for t in (q, k, v)]
    ref = su.attention(*wide(*one), [(0, 69, 0, 69)], None, True, dtype, do[1:].to(F))
    check(out[1:], ref["out"], "out")
    check(g.d_q[1:, 0][:, rest], tuple(t[:, 0][:, rest] for t in ref["d_q"]), "d_q")
    check(g.d_k[1:], ref["d_k"], "d_k")
    check(g.d_v[1:], ref["d_v"], "d_v")


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [7, 64, 100, 300])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_an_infinite_value_that_a_row_sees(dtype, rows, dim):
    """Weights are above zero: the sum is that infinity, in the tile where a row's keys
    start as in later ones, and as the gradient of v the same; both infinities make NaN."""
    q, k, v, off, spans, do = packed([rows], 0, 2, 1, dim, dtype, seed=5)
    v[3, 0, 7], v[5, 0, 6], v[2, 0, 9], v[rows // 2 + 2, 0, 9] = INF, -INF, INF, -INF
    for causal in (True, False):
        out, lse = dn.attention_forward(q, k, v, off, None, None, causal)
        first = lambda at: at if causal else 0
        assert (out[first(3):, :, 7] == INF).all() and (out[first(5):, :, 6] == -INF).all()
        both = first(rows // 2 + 2)
        assert out[both:, :, 9].isnan().all() and (out[first(2):both, :, 9] == INF).all()
        for at, col in ((3, 7), (5, 6), (2, 9)):
            assert out[:first(at), :, col].isfinite().all()
        rest = [i for i in range(dim) if i not in (6, 7, 9)]
        tame = v.clone()
        tame[:, 0, [6, 7, 9]] = 0
        want, _ = dn.attention_forward(q, k, tame, off, None, None, causal)
        assert torch.equal(out[..., rest], want[..., rest])
    q, k, v, off, spans, do = packed([rows], 0, 2, 1, dim, dtype, seed=5)
    out, lse = dn.attention_forward(q, k, v, off)
    last = rows - 2
    do[last, 1, 4] = -INF
    g = dn.attention_backward(do, q, k, v, out, lse, off)
    assert (g.d_v[:last + 1, 0, 4] == -INF).all() and g.d_v[last + 1, 0, 4].isfinite()


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_an_infinite_value_at_the_largest_score(dtype):
    """The key outweighs all before it by more than fp32 holds."""
    q, k, v, off, spans, do = packed([70], 0, 1, 1, 64, dtype, seed=5)
    q[:, 0, 0] = 8
    k[:, 0, 0] = 0
    k[66, 0, 0], v[66, 0, 3] = 400, INF  # a score of 400: 2^577 times the others' weights
    out = dn.attention(q, k, v, off)
    assert (out[66:, 0, 3] == INF).all() and out[:66].isfinite().all()
    assert out[66:, 0, [i for i in range(64) if i != 3]].isfinite().all()


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_query_that_sees_an_infinite_key(dtype, dim):
    """dS is 0 there, and 0 inf is NaN, in tiles that a row sees whole as in the others."""
    q, k, v, off, spans, do = packed([200], 0, 2, 1, dim, dtype, seed=6)
    q[:, :, 5] = (q[:, :, 5].abs() + 0.125).to(dtype)
    k[20, 0, 5] = -INF
    out, lse = dn.attention_forward(q, k, v, off)
    g = dn.attention_backward(do, q, k, v, out, lse, off)
    assert g.d_q[20:, :, 5].isnan().all() and g.d_q[:20].isfinite().all()
    assert g.d_q[..., [i for i in range(dim) if i != 5]].isfinite().all()


# -- attention: shapes ---------------------------------------------------------------


@gpu
def test_both_halves_refuse_keys_of_another_batch():
    """As many rows as q, but in other sequences."""
    on = lambda *shape: torch.ones(shape, device="cuda")
    q, k = on(2, 6, 2, 8), on(3, 4, 2, 8)
    for call in (lambda: dn.attention(q, k, k), lambda: dn.attention_forward(q, k, k),
                 lambda: dn.attention_backward(q, q, k, k, q, on(2, 6, 2))):
        with pytest.raises(dn.DeltaError, match="without key spans") as e:
            call()
        assert e.value.code == -2
    # With offsets only the rows count, as in the forward.
    off = ints(0, 6, 12)
    out, lse = dn.attention_forward(q, k, k, off)
    assert dn.attention_backward(q, q, k, k, out, lse, off).d_k.shape == k.shape


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_padding_without_requests(dtype):
    """Rows of padding over a cache, and no request: zeros, whatever the cache holds."""
    gen = torch.Generator("cuda").manual_seed(7)
    q, cache = made(gen, (9, 4, 64), dtype), made(gen, (50, 2, 64), dtype)
    cache[:] = NAN
    none = dn.KeySpans(ints(), ints())
    out, lse = dn.attention_forward(q, cache, cache, ints(0), none)
    assert out.shape == q.shape and not out.any() and (lse == -INF).all()
    out = dn.attention(q[:0], cache, cache, ints(0), none)
    assert out.shape == (0, 4, 64)
    with pytest.raises(dn.DeltaError, match="multiple"):  # empty calls are checked too
        dn.attention(q[:0, :3], cache, cache, ints(0), none)


@fake_pointers
def test_key_rows_without_sequences():
    assert refusal(ATT, tokens=0, sequences=0, key_rows=9)[0] == 0
    assert refusal(ATT, tokens=0, sequences=1, key_rows=9)[0] == -2


# -- embedding -----------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("tokens,vocab,wide_ids", [(64, 2, True), (5000, 3, False),
                                                   (20000, 1, True), (33333, 700, True),
                                                   (40000, 140000, False)])
def test_every_token_counts_once(tokens, vocab, wide_ids):
    """Whole numbers below 2^24 in the sums: fp32 holds them exactly, so that a token that
    is lost or taken twice shows."""
    gen = torch.Generator("cuda").manual_seed(8)
    ids = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    ids[::3] = vocab - 1  # many lanes of a step share an id
    d = torch.randint(-9, 10, (tokens, 24), generator=gen, device="cuda")
    d[:, 0] = 1
    want = torch.zeros(vocab, 24, dtype=torch.long, device="cuda").index_add(0, ids, d)
    got = dn.embedding_backward(d.float(), ids if wide_ids else ids.int(), vocab)
    assert torch.equal(got.long(), want) and torch.equal(got, got.round())


@gpu
@pytest.mark.parametrize("tokens", [9, 16, 8 * 64, 8 * 65, 8 * 66 + 3, 8 * 129, 4096, 4097,
                                    32 * 193 + 1, 32 * 4161])
def test_ids_of_many_parts(tokens):
    """One id between two others, of up to thousands of the sums that are joined: as many
    as are looked for at a time, one more, one less, and at a second level."""
    gen = torch.Generator("cuda").manual_seed(9)
    d = torch.randint(-9, 10, (tokens, 5), generator=gen, device="cuda")
    for before, behind in ((0, 0), (1, 1), (33, 40), (tokens // 2, 1), (tokens - 9, 0)):
        ids = torch.ones(tokens, dtype=torch.long, device="cuda")
        ids[:before] = 0
        ids[tokens - behind:] = 2
        want = torch.zeros(3, 5, dtype=torch.long, device="cuda").index_add(0, ids, d)
        got = dn.embedding_backward(d.float(), ids, 3)
        assert torch.equal(got.long(), want) and torch.equal(got, got.round())


@gpu
def test_many_tokens_of_few_values_leave_few_parts():
    """Sums of 32 tokens, however little there is to do: a join of four times the parts
    took up to 2.4 times as long."""
    a = filled((abi.EmbeddingBwdArgs, "dn_embedding_bwd",
                dict(tokens=65536, vocab=300, dim=64, d_out_stride=64, d_table_stride=64,
                     scale=1.0), ["ids", "d_out", "d_table"]))
    n = abi.lib().dn_embedding_bwd_workspace_bytes(ctypes.byref(a))
    assert n <= 2 * 65536 * 4 + 65536 // 32 * 2 * 64 * 4 + 4096
