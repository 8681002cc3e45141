"""block_norm and embedding on the GPU against float64, within bounds derived from
the arithmetic (stack_util, layer_util)."""

import pytest
import torch

import stack_util as su
from conftest import load_package
from layer_util import F, check

dn = load_package()
pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def made(gen, shape, dtype, scale=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale + mean).to(dtype)


def joint(rows, dim, dtype, wdtype, kind, post, seed=1):
    gen = torch.Generator("cuda").manual_seed(seed)
    x, r = made(gen, (rows, dim), dtype), made(gen, (rows, dim), dtype, 2.0)
    pre = made(gen, (dim,), wdtype, 0.2, 1.0)
    pw = made(gen, (dim,), wdtype, 0.2, 1.0) if post else None
    gate = {"none": None, "channel": made(gen, (dim,), wdtype, 0.5),
            "token": made(gen, (rows, 1), dtype, 0.5),
            "full": made(gen, (rows, dim), dtype, 0.5)}[kind]
    return x, r, pre, pw, gate, made(gen, (rows, dim), dtype), made(gen, (rows, dim), dtype)


def wide(t):
    return None if t is None else t.to(F)


def check_joint(x, r, pre, post, gate, dy, de, kind, scale=0.75, eps=1e-5, what=""):
    out, total = dn.block_norm(x, r, pre, post, gate, scale, eps)
    ref_s, ref_y = su.block_norm(*map(wide, (x, r, pre, post, gate)), scale, eps, x.dtype)
    check(total, ref_s, what + " sum")
    check(out, ref_y, what + " out")
    got = dn.block_norm_backward(dy, de, x, total, pre, post, gate, scale, eps)
    zero = torch.zeros_like(x)
    ref = su.block_norm_bwd(*map(wide, (x, total, pre, post, gate)), scale,
                            wide(zero if dy is None else dy), wide(zero if de is None else de),
                            eps, x.dtype, pre.dtype, kind)
    for name, value in ref.items():
        check(getattr(got, name), value, what + " " + name)


@pytest.mark.parametrize("kind", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("rows,dim,dtype,wdtype", [
    (1, 2048, BF, BF), (5, 7, F32, F32), (70, 200, BF, F32), (33, 512, F32, BF),
    (9, 513, BF, BF), (130, 1039, F32, F32), (1500, 64, BF, BF), (300, 2048, BF, F32),
    (17, 4096, F32, F32), (11, 4104, BF, BF), (6, 8192, F32, F32), (70, 8200, BF, BF),
    (3, 10001, F32, BF)])
def test_block_norm(rows, dim, dtype, wdtype, kind, post):
    check_joint(*joint(rows, dim, dtype, wdtype, kind, post), kind)


@pytest.mark.parametrize("rows", [1100, 5000])
def test_block_norm_many_rows(rows):
    """More rows than workgroups of the backward: every one walks several."""
    check_joint(*joint(rows, 640, BF, BF, "channel", True), "channel")
    check_joint(*joint(4 * rows, 96, F32, F32, "token", True), "token")


@pytest.mark.parametrize("dim", [256, 1024, 9000])
def test_block_norm_absent_cotangents(dim):
    x, r, pre, post, gate, dy, de = joint(40, dim, BF, BF, "channel", True)
    check_joint(x, r, pre, post, gate, dy, None, "channel")
    check_joint(x, r, pre, post, gate, None, de, "channel")


@pytest.mark.parametrize("dim", [96, 520, 8232])
def test_block_norm_of_views(dim):
    """Columns of wider tensors (at odd offsets), and a leading axis of another shape."""
    gen = torch.Generator("cuda").manual_seed(3)
    for dtype in (BF, F32):
        ts = [made(gen, (24, dim + 5), dtype)[:, 3:3 + dim] for _ in range(5)]
        x, r, gate, dy, de = ts
        pre, post = made(gen, (dim,), dtype, 0.2, 1.0), made(gen, (dim,), dtype, 0.2, 1.0)
        check_joint(x, r, pre, post, gate, dy, de, "full")
    out, total = dn.block_norm(x.reshape(2, 12, dim), r, pre, post, gate)
    flat, ft = dn.block_norm(x, r, pre, post, gate)
    assert out.shape == (2, 12, dim)
    assert torch.equal(out.flatten(0, 1), flat) and torch.equal(total.flatten(0, 1), ft)


@pytest.mark.parametrize("dim", [64, 2048, 9000])
def test_block_norm_of_zero_rows(dim):
    """A row of zeros is normalised by eps; large values do not overflow where their
    squares fit fp32."""
    x, r, pre, post, gate, dy, de = joint(4, dim, F32, F32, "channel", True)
    x[0], r[1] = 0, 0
    x[2] *= 1e15
    check_joint(x, r, pre, post, gate, dy, de, "channel")


def test_block_norm_keeps_rows_apart():
    """A row that is not finite leaves the others as they were."""
    for dim in (300, 2048, 9000):
        x, r, pre, post, gate, dy, de = joint(12, dim, BF, BF, "token", True)
        out, total = dn.block_norm(x, r, pre, post, gate)
        y = x.clone()
        y[5, 7] = float("nan")
        out2, total2 = dn.block_norm(y, r, pre, post, gate)
        rest = [i for i in range(12) if i != 5]
        assert torch.equal(out[rest], out2[rest]) and torch.equal(total[rest], total2[rest])
        assert out2[5].isnan().all()


@pytest.mark.parametrize("kind", ["none", "channel", "token", "full"])
def test_block_norm_no_rows(kind):
    x, r, pre, post, gate, dy, de = joint(0, 64, BF, BF, kind, True)
    out, total = dn.block_norm(x, r, pre, post, gate)
    assert out.shape == total.shape == (0, 64)
    g = dn.block_norm_backward(dy, de, x, total, pre, post, gate)
    assert not g.d_pre_weight.any() and not g.d_post_weight.any() and g.d_x.shape == (0, 64)
    if kind == "channel":
        assert not g.d_gate.any()


def test_block_norm_without_anything_is_add_rms_norm():
    """No norm after the block, no gate, a scale of one: the sums are the same numbers."""
    x, r, pre, _, _, _, _ = joint(64, 1024, BF, BF, "none", False)
    out, total = dn.block_norm(x, r, pre)
    out2, total2 = dn.add_rms_norm(x, r, pre)
    assert torch.equal(total, total2)
    assert (out.float() - out2.float()).abs().max() <= 2.0 ** -7 * out2.float().abs().max()


def test_block_norm_autograd():
    """The Function against the explicit halves; broadcast residual shapes; first order."""
    x, r, pre, post, gate, dy, de = joint(24, 192, F32, F32, "channel", True)
    leaves = [t.clone().requires_grad_(True) for t in (x.view(2, 12, 192), r, pre, post, gate)]
    out, total = dn.block_norm(*leaves[:3], leaves[3], leaves[4], 0.5, 1e-6)
    grads = torch.autograd.grad((out, total), leaves,
                                (dy.view(2, 12, 192), de.view(2, 12, 192)))
    want = dn.block_norm_backward(dy, de, x, total.detach().view(24, 192), pre, post, gate, 0.5,
                                  1e-6)
    for got, ref, leaf in zip(grads, want, leaves):
        assert got.shape == leaf.shape
        assert torch.equal(got.reshape(ref.shape), ref)
    # One output alone.
    out, total = dn.block_norm(*leaves[:3], leaves[3], leaves[4], 0.5, 1e-6)
    only, = torch.autograd.grad(total, leaves[0], de.view(2, 12, 192))
    ref = dn.block_norm_backward(None, de, x, total.detach().view(24, 192), pre, post, gate, 0.5,
                                 1e-6)
    assert torch.equal(only.view(24, 192), ref.d_x)
    out, _ = dn.block_norm(*leaves[:3], leaves[3], leaves[4], 0.5, 1e-6)
    g, = torch.autograd.grad(out.sum(), leaves[0], create_graph=True)
    with pytest.raises(dn.DeltaError, match="second derivative"):
        g.sum().backward()


@pytest.mark.parametrize("kind", ["channel", "token", "full"])
def test_block_norm_gradient_against_differences(kind):
    """Central differences of the float64 formula along a random direction: d_x, d_gate
    and the weights' gradients together."""
    x, r, pre, post, gate, dy, de = joint(6, 48, F32, F32, kind, True, seed=8)
    out, total = dn.block_norm(x, r, pre, post, gate, 0.6)
    g = dn.block_norm_backward(dy, de, x, total, pre, post, gate, 0.6)
    gen = torch.Generator("cuda").manual_seed(9)
    args = [wide(t) for t in (x, r, pre, post, gate)]
    steps = [torch.randn(a.shape, generator=gen, device="cuda", dtype=F) for a in args]

    def loss(h):
        (s, _), (y, _) = su.block_norm(*[a + h * d for a, d in zip(args, steps)], 0.6, 1e-5, F32)
        return ((y * wide(dy)).sum() + (s * wide(de)).sum()).item()

    h = 1e-5  # truncation ~ h² = 1e-10, rounding ~ 1e-16 / h = 1e-11 of the loss
    want = (loss(h) - loss(-h)) / (2 * h)
    got = sum((wide(a) * d).sum().item() for a, d in zip(g, steps))
    size = sum((wide(a) * d).abs().sum().item() for a, d in zip(g, steps))
    assert abs(got - want) <= 1e-5 * size


# -- embedding -----------------------------------------------------------------------


def looked_up(tokens, vocab, dim, dtype, wide_ids, skew, seed=5):
    gen = torch.Generator("cuda").manual_seed(seed)
    u = torch.rand(tokens, generator=gen, device="cuda")
    ids = (u * vocab).long() if skew == "even" else ((vocab + 1.0) ** u - 1).long()
    ids.clamp_(0, vocab - 1)
    if skew == "one":
        ids.fill_(vocab // 2)
    elif tokens > 4:  # outside: padding, far above, the largest and the smallest numbers
        big = 2 ** 62 if wide_ids else 2 ** 31 - 1
        ids[torch.tensor([0, 2, tokens // 2, tokens - 1], device="cuda")] = torch.tensor(
            [-1, vocab, big, -big], device="cuda")
    return (ids if wide_ids else ids.int(), made(gen, (vocab, dim), dtype),
            made(gen, (tokens, dim), dtype))


@pytest.mark.parametrize("tokens,vocab,dim,dtype,wide_ids,skew", [
    (1, 1, 1, BF, True, "one"), (1, 300, 2048, BF, False, "even"), (31, 5, 7, F32, True, "log"),
    (32, 40, 64, BF, True, "one"), (33, 40, 64, F32, False, "one"), (64, 257, 8, BF, True, "log"),
    (100, 1009, 200, F32, True, "log"), (700, 3, 33, BF, False, "even"),
    (1024, 600, 1039, BF, True, "log"), (1025, 131073, 16, F32, True, "even"),
    (5000, 50000, 128, BF, True, "log"), (3001, 1009, 2056, F32, False, "log"),
    (2048, 7, 4100, BF, True, "log"), (4097, 20, 72, F32, True, "one"),
    (17001, 300, 2048, BF, True, "log"), (70000, 1000, 520, F32, True, "log")])
def test_embedding(tokens, vocab, dim, dtype, wide_ids, skew):
    ids, table, d = looked_up(tokens, vocab, dim, dtype, wide_ids, skew)
    scale = 1.0 if dim == 64 else 2.5
    out = dn.embedding(ids, table, scale)
    check(out, su.embedding(ids.long(), table.to(F), scale, dtype), "out")
    g = dn.embedding_backward(d, ids, vocab, scale)
    check(g, su.embedding_bwd(ids.long(), d.to(F), vocab, scale, dtype), "d_table")
    assert torch.equal(g, dn.embedding_backward(d, ids, vocab, scale))  # the same bits


def test_embedding_of_views():
    ids, table, d = looked_up(96, 50, 24, BF, True, "log")
    store = torch.zeros(50, 31, dtype=BF, device="cuda")
    store[:, 5:29] = table
    assert torch.equal(dn.embedding(ids, store[:, 5:29]), dn.embedding(ids, table))
    assert torch.equal(dn.embedding(ids.view(8, 12).t(), table),
                       dn.embedding(ids, table).view(8, 12, 24).transpose(0, 1))
    flat = dn.embedding_backward(d, ids, 50)
    wide_d = torch.zeros(96, 40, dtype=BF, device="cuda")
    wide_d[:, 9:33] = d
    assert torch.equal(dn.embedding_backward(wide_d[:, 9:33], ids, 50), flat)
    assert torch.equal(dn.embedding_backward(d.view(8, 12, 24), ids.view(8, 12), 50), flat)
    one = dn.embedding(ids[3], table)  # a lone id
    assert one.shape == (24,)
    assert torch.equal(dn.embedding_backward(d[3], ids[3], 50).sum(0), d[3])


def test_embedding_no_tokens():
    _, table, d = looked_up(8, 50, 24, BF, True, "log")
    none = torch.empty(0, dtype=torch.long, device="cuda")
    assert dn.embedding(none, table).shape == (0, 24)
    assert not dn.embedding_backward(d[:0], none, 50).any()
    outside = torch.full((8,), -1, device="cuda")
    assert not dn.embedding(outside, table).any()
    assert not dn.embedding_backward(d, outside, 50).any()


def test_embedding_keeps_ids_apart():
    """A gradient row that is not finite reaches its own id's row only; so does padding's."""
    ids, table, d = looked_up(4000, 90, 64, F32, True, "log")
    before = dn.embedding_backward(d, ids, 90)
    d[0] = float("nan")  # padding (-1)
    d[7] = float("inf")
    after = dn.embedding_backward(d, ids, 90)
    rest = torch.arange(90, device="cuda") != ids[7]
    assert torch.equal(before[rest], after[rest]) and after[ids[7]].isinf().all()


def test_embedding_autograd():
    ids, table, d = looked_up(200, 60, 40, F32, True, "log")
    leaf = table.clone().requires_grad_(True)
    out = dn.embedding(ids, leaf, 1.5)
    g, = torch.autograd.grad(out, leaf, d)
    assert torch.equal(g, dn.embedding_backward(d, ids, 60, 1.5))
    g, = torch.autograd.grad(dn.embedding(ids, leaf), leaf, d, create_graph=True)
    with pytest.raises(dn.DeltaError, match="second derivative"):
        g.sum().backward()
