"""attention on the GPU against float64, within bounds derived from the arithmetic
(stack_util)."""

import pytest
import torch

import stack_util as su
from conftest import load_package
from layer_util import F, check

dn = load_package()
pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def made(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def packed(lengths, padding, heads, kv, dim, dtype, seed=1):
    gen = torch.Generator("cuda").manual_seed(seed)
    rows = sum(lengths) + padding
    ends = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    spans = [(a, b - a, a, b - a) for a, b in zip(ends, ends[1:])]
    q, k, v = (made(gen, (rows, h, dim), dtype) for h in (heads, kv, kv))
    return q, k, v, torch.tensor(ends, dtype=torch.int32, device="cuda"), spans, \
        made(gen, (rows, heads, dim), dtype)


def wide(*ts):
    return [t.to(F) for t in ts]


def check_all(q, k, v, offsets, spans, do, scale=None, causal=True, flat=lambda t: t):
    out, lse = dn.attention_forward(q, k, v, offsets, None, scale, causal)
    ref = su.attention(*wide(flat(q), flat(k), flat(v)), spans, scale, causal, q.dtype,
                       flat(do).to(F))
    check(flat(out), ref["out"], "out")
    seen = ref["lse"][0] > -float("inf")
    l = lse.reshape(ref["lse"][0].shape)
    assert torch.equal(l > -float("inf"), seen)
    check(l[seen], (ref["lse"][0][seen], ref["lse"][1][seen]), "lse")
    assert torch.equal(out, dn.attention(q, k, v, offsets, None, scale, causal))
    g = dn.attention_backward(do, q, k, v, out, lse, offsets, scale, causal)
    for name in ("d_q", "d_k", "d_v"):
        check(flat(getattr(g, name)), ref[name], name)
    again = dn.attention_backward(do, q, k, v, out, lse, offsets, scale, causal)
    assert all(torch.equal(a, b) for a, b in zip(g, again))  # the same bits


LENGTHS = [[1], [2], [64], [65], [130], [1, 1, 1], [3, 0, 200, 1, 64, 0], [127, 128, 129, 0]]


@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("heads,kv,dim,dtype", [
    (4, 1, 128, BF), (2, 2, 64, BF), (6, 2, 40, F32), (3, 1, 33, BF), (2, 1, 256, BF),
    (1, 1, 72, F32), (8, 1, 128, F32), (2, 2, 200, F32)])
def test_packed(lengths, heads, kv, dim, dtype):
    check_all(*packed(lengths, 0, heads, kv, dim, dtype))


@pytest.mark.parametrize("heads,kv,dim,dtype", [(4, 2, 128, BF), (3, 3, 64, F32), (7, 1, 96, BF)])
def test_without_mask(heads, kv, dim, dtype):
    check_all(*packed([100, 1, 37, 0, 190], 9, heads, kv, dim, dtype), causal=False)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_long_enough_to_split(dtype):
    """Few tiles of rows over many keys: the keys are split, and joined in order."""
    check_all(*packed([1100], 0, 2, 1, 64, dtype))
    check_all(*packed([600, 700], 5, 2, 2, 128, dtype), causal=False)


def test_many_sequences():
    """More sequences than a wave has lanes, empty ones among them."""
    lengths = [(7 * i) % 5 for i in range(333)]
    check_all(*packed(lengths, 3, 2, 1, 64, BF))


@pytest.mark.parametrize("heads,kv,dim,dtype", [(4, 1, 128, BF), (2, 2, 40, F32)])
def test_batch(heads, kv, dim, dtype):
    """[batch, sequence, heads, dim] without offsets, and a scale of the caller's."""
    q, k, v, _, spans, do = packed([70, 70, 70], 0, heads, kv, dim, dtype)
    shape = lambda t: t.view(3, 70, *t.shape[1:])
    check_all(shape(q), shape(k), shape(v), None, spans, shape(do), 0.2, True,
              lambda t: t.reshape(210, *t.shape[2:]))


@pytest.mark.parametrize("dim,dtype", [(64, BF), (128, BF), (40, F32)])
def test_views_of_a_projection(dim, dtype):
    """q, k and v as columns of one projection, at an odd offset; int64 offsets."""
    gen = torch.Generator("cuda").manual_seed(4)
    heads, kv, rows = 4, 2, 150
    wide_t = made(gen, (rows, (heads + 2 * kv) * dim + 7), dtype)
    cut = lambda a, n: wide_t[:, 3 + a * dim:3 + (a + n) * dim].unflatten(1, (n, dim))
    q, k, v = cut(0, heads), cut(heads, kv), cut(heads + kv, kv)
    offsets = torch.tensor([0, 33, 150], device="cuda")
    check_all(q, k, v, offsets, [(0, 33, 0, 33), (33, 117, 33, 117)],
              made(gen, (rows, heads, dim), dtype))
    # Heads that are not side by side are laid out.
    t = made(gen, (heads, rows, dim), dtype).transpose(0, 1)
    assert torch.equal(dn.attention(t, k, v, offsets), dn.attention(t.contiguous(), k, v, offsets))


def test_large_scores():
    """Scores up to a few hundred: weights of one, differences far below them, and a
    maximum that grows along the keys."""
    for dtype in (BF, F32):
        q, k, v, off, spans, do = packed([200, 140], 0, 2, 1, 64, dtype)
        k = (k.float() * torch.linspace(0.1, 12, 340, device="cuda")[:, None, None]).to(dtype)
        out, lse = dn.attention_forward(q, k, v, off, None, 1.0)
        ref = su.attention(*wide(q, k, v), spans, 1.0, True, dtype)
        check(out, ref["out"], "out")
        check(lse, ref["lse"], "lse")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_what_a_row_does_not_see(dtype, what, dim):
    """Values of later tokens, of other sequences and behind the last one, whatever they
    are, leave a row's results as they were: forward, and in the gradients the other
    way round."""
    q, k, v, off, spans, do = packed([70, 75], 8, 4, 2, dim, dtype)
    out, lse = dn.attention_forward(q, k, v, off)
    g = dn.attention_backward(do, q, k, v, out, lse, off)
    at = 70 + 40
    for t in (k, v):
        t[at, 0, 5] = what
        t[145:] = what
    q[145:], do2 = what, do.clone()
    do2[145:] = what
    out2, lse2 = dn.attention_forward(q, k, v, off)
    same = torch.ones(153, dtype=torch.bool, device="cuda")
    same[at:145] = False
    assert torch.equal(out[same], out2[same]) and torch.equal(lse[same], lse2[same])
    assert torch.equal(out[:, 2:], out2[:, 2:])  # the other key head's
    assert not out2[at:145, :2, 5].isfinite().any()
    g2 = dn.attention_backward(do2, q, k, v, out2, lse2, off)
    assert torch.equal(g.d_q[same], g2.d_q[same])
    assert torch.equal(g.d_k[:70], g2.d_k[:70]) and torch.equal(g.d_v[:70], g2.d_v[:70])
    assert torch.equal(g.d_q[:, 2:], g2.d_q[:, 2:]) and torch.equal(g.d_k[:, 1], g2.d_k[:, 1])
    assert not any(t[145:].any() for t in (out2, g2.d_q, g2.d_k, g2.d_v))
    # Backward: a token's cotangent and query do not reach later keys.
    q, k, v, off, spans, do = packed([70, 75], 8, 4, 2, dim, dtype)
    do[at, 1, 3] = what
    g3 = dn.attention_backward(do, q, k, v, out, lse, off)
    later = slice(at + 1, 153)
    assert torch.equal(g.d_k[later], g3.d_k[later]) and torch.equal(g.d_v[later], g3.d_v[later])
    assert not g3.d_v[70:at + 1, 0, 3].isfinite().any()
    assert torch.equal(g.d_v[:70], g3.d_v[:70])


@pytest.mark.parametrize("heads,kv,dim,dtype,new", [
    (4, 1, 128, BF, 1), (16, 4, 128, BF, 1), (2, 2, 64, F32, 1), (6, 2, 40, BF, 3),
    (8, 1, 256, BF, 2), (7, 7, 33, F32, 5), (3, 1, 128, BF, 70)])
def test_cached_keys(heads, kv, dim, dtype, new):
    """New tokens over spans of a cache: no keys at all, fewer than there are queries, spans
    that overlap, and a cache whose other rows hold anything."""
    gen = torch.Generator("cuda").manual_seed(6)
    rows = 3000
    k, v = made(gen, (rows, kv, dim), dtype), made(gen, (rows, kv, dim), dtype)
    spans = [(0, 900), (100, 64), (1000, 0), (1000, 1), (1001, new + 2), (100, 1700), (2900, 100)]
    used = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for a, n in spans:
        used[a:a + n] = True
    k[~used], v[~used] = float("nan"), float("inf")
    n = len(spans)
    q = made(gen, (n * new, heads, dim), dtype)
    ints = lambda xs: torch.tensor(xs, dtype=torch.int32, device="cuda")
    keys = dn.KeySpans(ints([a for a, _ in spans]), ints([m for _, m in spans]))
    offsets = ints([i * new for i in range(n + 1)])
    where = [(i * new, new, a, m) for i, (a, m) in enumerate(spans)]
    for causal in (True, False):
        out, lse = dn.attention_forward(q, k, v, offsets, keys, None, causal)
        ref = su.attention(*wide(q, k, v), where, None, causal, dtype)
        check(out, ref["out"], "out")
        seen = ref["lse"][0] > -float("inf")
        assert torch.equal(lse > -float("inf"), seen)
        check(lse[seen], (ref["lse"][0][seen], ref["lse"][1][seen]), "lse")
    # The same from a batch of single tokens, [batch, new, heads, dim].
    assert torch.equal(dn.attention(q.view(n, new, heads, dim), k, v, None, keys).flatten(0, 1),
                       dn.attention(q, k, v, offsets, keys))


def test_spans_beyond_the_tensors():
    """Offsets and spans that leave the tensors are cut off at their ends."""
    gen = torch.Generator("cuda").manual_seed(7)
    ints = lambda xs: torch.tensor(xs, dtype=torch.int32, device="cuda")
    q, k, v = (made(gen, (40, 2, 64), BF) for _ in range(3))
    big = 2 ** 31 - 1
    out = dn.attention(q, k, v, ints([0, 10, big]))
    assert torch.equal(out, dn.attention(q, k, v, ints([0, 10, 40])))
    keys = dn.KeySpans(ints([5, -7]), ints([big, 12]))
    good = dn.KeySpans(ints([5, 0]), ints([35, 12]))
    off = ints([0, 3, 6])
    assert torch.equal(dn.attention(q[:6], k, v, off, keys), dn.attention(q[:6], k, v, off, good))
    for bad in ([3, 50, -4], [0, 30, 10], [-big, big, -big], [0, -1, -1]):
        out = dn.attention(q, k, v, ints(bad))  # anything, but inside
        assert out.shape == q.shape


def test_a_cache_past_32_bits():
    """Rows whose first value is more than 2^32 bytes, and 2^31 values, from the start."""
    rows, heads, kv, dim = 9_000_000, 4, 2, 128
    gen = torch.Generator("cuda").manual_seed(13)
    k = torch.empty(rows, kv, dim, dtype=BF, device="cuda")
    v = torch.empty(rows, kv, dim, dtype=BF, device="cuda")
    k[-700:], v[-700:] = made(gen, (700, kv, dim), BF), made(gen, (700, kv, dim), BF)
    q = made(gen, (3, heads, dim), BF)
    ints = lambda xs: torch.tensor(xs, dtype=torch.int32, device="cuda")
    off, counts = ints([0, 1, 3]), ints([650, 300])
    got = dn.attention(q, k, v, off, dn.KeySpans(ints([rows - 700, rows - 300]), counts))
    want = dn.attention(q, k[-700:].clone(), v[-700:].clone(), off,
                        dn.KeySpans(ints([0, 400]), counts))
    # The split of the keys goes by the cache's size: the same sums in another order.
    ref = su.attention(*wide(q, k[-700:], v[-700:]), [(0, 1, 0, 650), (1, 2, 400, 300)], None,
                       True, BF)
    check(got, ref["out"], "out")
    check(want, ref["out"], "out of the short cache")


def test_no_requests():
    """A batch without requests over a cache."""
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    k = torch.ones(50, 2, 64, dtype=BF, device="cuda")
    out = dn.attention(torch.empty(0, 1, 4, 64, dtype=BF, device="cuda"), k, k, None,
                       dn.KeySpans(none, none))
    assert out.shape == (0, 1, 4, 64)


def test_nothing_there():
    empty = torch.empty(0, 4, 64, dtype=BF, device="cuda")
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    out, lse = dn.attention_forward(empty, empty, empty, off)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    g = dn.attention_backward(out, empty, empty, empty, out, lse, off)
    assert g.d_q.shape == (0, 4, 64)
    # Rows, but no sequence holds them.
    q = torch.ones(9, 4, 64, dtype=BF, device="cuda")
    out, lse = dn.attention_forward(q, q, q, off)
    assert not out.any() and (lse == -float("inf")).all()
    g = dn.attention_backward(q, q, q, q, out, lse, off)
    assert not g.d_q.any() and not g.d_k.any() and not g.d_v.any()


def test_autograd():
    q, k, v, off, _, do = packed([50, 30], 4, 4, 2, 64, F32)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(dn.attention(*leaves, off), leaves, do)
    out, lse = dn.attention_forward(q, k, v, off)
    want = dn.attention_backward(do, q, k, v, out, lse, off)
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    # Broadcast keys: one key head expanded to two.
    one = k[:, :1].clone().requires_grad_(True)
    got, = torch.autograd.grad(dn.attention(q, one.expand(-1, 2, -1), v, off), one, do)
    out, lse = dn.attention_forward(q, k[:, :1].expand(-1, 2, -1), v, off)
    want = dn.attention_backward(do, q, k[:, :1].expand(-1, 2, -1), v, out, lse, off)
    assert torch.allclose(got, want.d_k.sum(1, keepdim=True), rtol=1e-6, atol=1e-6)
    g, = torch.autograd.grad(dn.attention(*leaves, off), leaves[0], do, create_graph=True)
    with pytest.raises(dn.DeltaError, match="second derivative"):
        g.sum().backward()
    with pytest.raises(dn.DeltaError, match="no gradient"):
        dn.attention(*leaves, off, dn.KeySpans(off[:2], off[1:]))


def test_gradient_against_differences():
    """Central differences of the float64 formula along a random direction."""
    q, k, v, off, spans, do = packed([21, 40], 0, 4, 2, 16, F32, seed=11)
    out, lse = dn.attention_forward(q, k, v, off)
    g = dn.attention_backward(do, q, k, v, out, lse, off)
    gen = torch.Generator("cuda").manual_seed(12)
    args = wide(q, k, v)
    steps = [torch.randn(a.shape, generator=gen, device="cuda", dtype=F) for a in args]

    def loss(h):
        moved = [a + h * d for a, d in zip(args, steps)]
        return (su.attention(*moved, spans, None, True, F32)["out"][0] * do.to(F)).sum().item()

    h = 1e-5  # truncation ~ h² = 1e-10, rounding ~ 1e-16 / h = 1e-11 of the loss
    want = (loss(h) - loss(-h)) / (2 * h)
    got = sum((a.to(F) * d).sum().item() for a, d in zip(g, steps))
    size = sum((a.to(F) * d).abs().sum().item() for a, d in zip(g, steps))
    assert abs(got - want) <= 1e-5 * size
