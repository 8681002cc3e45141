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


# -- attention: forms that sizes choose ----------------------------------------------


@gpu
def test_gradients_at_large_scores(monkeypatch):
    """Scores up to a few hundred. The gradients of the keys start their sums at the
    log-sum over the scale: its magnitude is one more term of the product's, 2 (D + 4) u
    of it beside the log-sum's own bound."""
    head = su.head

    def started(q, *rest):
        f = head(q, *rest)
        f["elses"] = f["elses"] + 2 * (q.shape[1] + 4) * U * f["lse"].abs()
        return f

    monkeypatch.setattr(su, "head", started)
    for dtype in (BF, F32):
        for dim in (64, 128, 256):
            q, k, v, off, spans, do = packed([200, 140], 0, 2, 1, dim, dtype)
            k = (k.float() * torch.linspace(0.1, 12, 340, device="cuda")[:, None, None]).to(dtype)
            check_all(q, k, v, off, spans, do, scale=1.0)


def cus():
    return torch.cuda.get_device_properties(0).multi_processor_count


def crowd(kv, per_tile, dtype, dim, group=2, seed=10):
    """Enough short sequences for the gradients of keys and values to be formed together:
    two workgroups a CU, of `per_tile` keys each."""
    n = 2 * cus() // kv + 1
    lengths = [(37 * i) % 90 + 1 for i in range(n - 2)] + [0, 3 * per_tile + 7]
    t = packed(lengths, 5, group * kv, kv, dim, dtype, seed)
    assert (t[0].shape[0] // per_tile + n + 1) * kv >= 2 * cus()
    return t


@gpu
@pytest.mark.parametrize("kv,dim,dtype,group,causal", [
    (16, 64, BF, 2, True), (16, 40, BF, 1, False), (16, 40, F32, 3, True),
    (16, 128, F32, 1, True), (16, 128, F32, 2, False), (16, 33, BF, 1, True)])
def test_d_k_and_d_v_together(kv, dim, dtype, group, causal):
    q, k, v, off, spans, do = crowd(kv, 128 if dtype == BF else 64, dtype, dim, group)
    check_all(q, k, v, off, spans, do, causal=causal)


@gpu
@pytest.mark.parametrize("dim,dtype", [(64, BF), (128, F32)])
@pytest.mark.parametrize("what", [NAN, INF])
def test_later_keys_of_rows_that_are_not_finite(dim, dtype, what):
    """d_k and d_v formed together: a row reaches no later key, and no other sequence."""
    q, k, v, off, spans, do = crowd(16, 128 if dtype == BF else 64, dtype, dim)
    out, lse = dn.attention_forward(q, k, v, off)
    g = dn.attention_backward(do, q, k, v, out, lse, off)
    first, n = spans[-1][:2]
    at = first + n // 2
    do[at, 1, 3], do[at, 5, 2] = what, what
    q[at, 1, 4], q[at, 7, 2] = what, what
    g2 = dn.attention_backward(do, q, k, v, out, lse, off)
    same = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
    same[first:at + 1] = False
    for name in ("d_k", "d_v"):
        a, b = getattr(g, name), getattr(g2, name)
        assert torch.equal(a[same], b[same])
        assert torch.equal(a[:, 4:], b[:, 4:])  # other key heads
    assert not g2.d_v[first:at + 1, 0, 3].isfinite().any()
    assert not g2.d_k[first:at + 1, 3].isfinite().all(-1).any()


@gpu
@pytest.mark.parametrize("dim,dtype,many", [(64, BF, True), (64, BF, False), (128, BF, False),
                                            (40, F32, True), (128, F32, True), (256, F32, False),
                                            (256, BF, False)])
def test_one_gradient_at_a_time(dim, dtype, many):
    q, k, v, off, spans, do = (crowd(16, 128 if dtype == BF else 64, dtype, dim, 1) if many
                               else packed([150, 1, 0, 77], 3, 4, 2, dim, dtype))
    out, lse = dn.attention_forward(q, k, v, off)
    ref = su.attention(*wide(q, k, v), spans, None, True, dtype, do.to(F))
    for names in (["d_q"], ["d_k"], ["d_v"], ["d_q", "d_v"], ["d_k", "d_v"]):
        need = {f"need_{n}": f"d_{n}" in names for n in "qkv"}
        g = dn.attention_backward(do, q, k, v, out, lse, off, **need)
        for name in ("d_q", "d_k", "d_v"):
            if name in names:
                check(getattr(g, name), ref[name], name)
            else:
                assert getattr(g, name) is None


@gpu
@pytest.mark.parametrize("heads,kv,dtype", [(256, 1, BF), (60, 3, BF), (100, 1, F32)])
def test_large_groups(heads, kv, dtype):
    """More heads of a group than rows of a tile, and numbers that share no factor with it."""
    check_all(*packed([70, 1, 3], 2, heads, kv, 64, dtype))


@gpu
@pytest.mark.parametrize("heads,kv,dim,dtype,new", [
    (4, 1, 128, BF, 3), (2, 2, 64, F32, 5), (6, 2, 40, BF, 1), (8, 1, 256, BF, 2),
    (3, 1, 128, F32, 70), (4, 4, 33, BF, 2)])
def test_split_keys(heads, kv, dim, dtype, new):
    """Keys that are split among workgroups: several new tokens, spans of very different
    lengths that end inside a tile, parts without a key, and values that are not finite
    where no row looks and where all do."""
    gen = torch.Generator("cuda").manual_seed(11)
    rows = 6000
    k, v = made(gen, (rows, kv, dim), dtype), made(gen, (rows, kv, dim), dtype)
    spans = [(0, 4999), (4900, 300), (5500, new - 1)]
    used = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for a, n in spans:
        used[a:a + n] = True
    k[~used], v[~used] = NAN, INF
    n = len(spans)
    assert 2 * cus() // (n * kv) >= 2 and rows // n // 256 >= 2  # more than one part
    q = made(gen, (n * new, heads, dim), dtype)
    keys = dn.KeySpans(ints(*(a for a, _ in spans)), ints(*(m for _, m in spans)))
    offsets = ints(*(i * new for i in range(n + 1)))
    where = [(i * new, new, a, m) for i, (a, m) in enumerate(spans)]
    for causal in (True, False):
        out, lse = dn.attention_forward(q, k, v, offsets, keys, None, causal)
        ref = su.attention(*wide(q, k, v), where, None, causal, dtype)
        check(out, ref["out"], "out")
        seen = ref["lse"][0] > -INF
        assert torch.equal(lse > -INF, seen)
        check(lse[seen], (ref["lse"][0][seen], ref["lse"][1][seen]), "lse")
        hot = v.clone()
        hot[2500, 0, 5] = INF  # seen by the first request's rows alone
        got = dn.attention(q, k, hot, offsets, keys, None, causal)
        group = heads // kv
        assert (got[:new, :group, 5] == INF).all()
        got[:new, :group, 5] = out[:new, :group, 5]
        assert torch.equal(got, out)


# -- block_norm ----------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("dim", [96, 1024, 4096, 9000])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("over", ["x", "residual"])
def test_sum_over_an_input(dim, dtype, over):
    """`sum` may lie on x or on the residual."""
    gen = torch.Generator("cuda").manual_seed(12)
    x, r = made(gen, (37, dim), dtype), made(gen, (37, dim), dtype)
    pre, post, gate = (made(gen, (dim,), dtype) for _ in range(3))
    want, total = dn.block_norm(x, r, pre, post, gate, 0.5)
    out, to = torch.empty_like(x), x if over == "x" else r
    a = abi.BlockNormArgs(37, dim, dim, dim, dim, dim, dim, 1e-5, 0.5, abi.dtype_tag(dtype),
                          abi.dtype_tag(dtype), abi.DN_GATE_CHANNEL, x.data_ptr(), r.data_ptr(),
                          pre.data_ptr(), post.data_ptr(), gate.data_ptr(), to.data_ptr(),
                          out.data_ptr())
    assert abi.lib().dn_block_norm(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(to, total) and torch.equal(out, want)


@gpu
@pytest.mark.parametrize("dtype,wdtype", [(BF, F32), (F32, BF), (F32, F32)])
def test_gates_of_a_lone_row(dtype, wdtype):
    """x [dim]: every kind of gate, as for x [1, dim]."""
    gen = torch.Generator("cuda").manual_seed(14)
    x, r, dy, full = (made(gen, (40,), dtype) for _ in range(4))
    pre, channel = made(gen, (40,), wdtype), made(gen, (40,), wdtype)
    token = made(gen, (1,), dtype)
    for gate, shape in ((None, None), (channel, (40,)), (full, (1, 40)), (token, (1, 1))):
        if gate is full and dtype == wdtype:
            continue  # the same as a channel's
        alone = gate if gate is None else gate.clone()
        same = None if gate is None else gate.reshape(shape)
        out, total = dn.block_norm(x, r, pre, None, alone)
        want, ref = dn.block_norm(x[None], r[None], pre, None, same)
        assert out.shape == (40,) and torch.equal(out, want[0]) and torch.equal(total, ref[0])
        g = dn.block_norm_backward(dy, None, x, total, pre, None, alone)
        h = dn.block_norm_backward(dy[None], None, x[None], ref, pre, None, same)
        assert torch.equal(g.d_x, h.d_x[0]) and torch.equal(g.d_pre_weight, h.d_pre_weight)
        if gate is not None:
            assert g.d_gate.shape == gate.shape and g.d_gate.dtype == gate.dtype
            assert torch.equal(g.d_gate, h.d_gate.reshape(gate.shape))


# -- differentiation -----------------------------------------------------------------


def operators():
    gen = torch.Generator("cuda").manual_seed(13)
    t = lambda *shape: made(gen, shape, F32)
    off, tokens = ints(0, 7, 12), torch.arange(12, device="cuda") % 5
    return {
        "attention": (lambda q, k, v: dn.attention(q, k, v, off),
                      (t(12, 4, 16), t(12, 2, 16), t(12, 2, 16))),
        "block_norm": (lambda *a: dn.block_norm(*a)[0],
                       (t(12, 24), t(12, 24), t(24), t(24), t(12, 1))),
        "embedding": (lambda table: dn.embedding(tokens, table), (t(5, 24),))}


@gpu
@pytest.mark.parametrize("name", ["attention", "block_norm", "embedding"])
@pytest.mark.parametrize("grad_mode", [False, True])
def test_tangents_are_refused(name, grad_mode):
    fn, leaves = operators()[name]
    ad = torch.autograd.forward_ad
    with ad.dual_level(), torch.set_grad_enabled(grad_mode):
        want = fn(*leaves)  # no tangents: as ever
        for i in range(len(leaves)):
            dual = list(leaves)
            dual[i] = ad.make_dual(leaves[i], torch.ones_like(leaves[i]))
            with pytest.raises(NotImplementedError, match="jvp"):
                fn(*dual)
    assert torch.equal(fn(*leaves), want)


@gpu
@pytest.mark.parametrize("name", ["attention", "block_norm", "embedding"])
def test_gradients_of_one_leaf_at_a_time(name):
    """Other leaves' gradients are not asked for: the same numbers."""
    fn, leaves = operators()[name]
    every = [t.clone().requires_grad_(True) for t in leaves]
    out = fn(*every)
    c = torch.randn_like(out)
    want = torch.autograd.grad(out, every, c)
    for i, leaf in enumerate(leaves):
        one = list(leaves)
        one[i] = leaf.clone().requires_grad_(True)
        got, = torch.autograd.grad(fn(*one), one[i], c)
        assert torch.equal(got, want[i])
