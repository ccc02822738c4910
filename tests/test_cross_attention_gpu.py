"""``torchode_amd.cross_attention`` against its definition in float64: types, lengths from nothing to many tiles, head dimensions of every
alignment, shared heads, masks that leave nothing, strides, gradients; HIP graphs, ``vmap`` and ``torch.compile``."""
import math

import pytest
import torch

import torchode_amd as to
from tests import field_oracle

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# batch, queries, keys, heads, heads of keys, head_dim
SHAPES = [
    (1, 1, 1, 1, 1, 1),
    (2, 1, 1, 4, 2, 16),
    (3, 1, 50, 4, 4, 16),
    (2, 1, 1000, 8, 2, 64),
    (1, 1, 5001, 8, 1, 128),
    (2, 5, 33, 6, 3, 20),
    (2, 7, 31, 2, 2, 33),
    (1, 32, 32, 1, 1, 32),
    (2, 33, 65, 4, 4, 40),
    (2, 100, 96, 3, 1, 64),
    (1, 200, 129, 2, 2, 80),
    (2, 128, 300, 4, 2, 128),
    (1, 513, 70, 2, 1, 96),
    (1, 130, 600, 9, 9, 8),
    (40, 3, 17, 2, 1, 5),
    (2, 1, 2, 48, 1, 64),  # one token, more rows than a tile
    (1, 2000, 40, 1, 1, 64),  # many rows for few keys
    (1, 65, 40, 2, 1, 256),
    (2, 1, 700, 4, 4, 200),
    (2, 5, 900, 6, 2, 80),  # 15 rows for a head of keys
    (1, 9, 3000, 2, 1, 48),
    (2, 300, 500, 2, 2, 256),
    (9, 60, 90, 3, 1, 32),  # more samples than dies, a number of heads that is no power of two
]
ids = lambda s: "-".join(map(str, s))


def made(shape, dtype, *, lengths=None, holes=0.0, seed=0):
    B, Lq, Lk, H, Hkv, D = shape
    g = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=g, dtype=torch.float64).to(dtype).cuda()
    t = dict(q=randn(B, Lq, H, D) * 1.5, k=randn(B, Lk, Hkv, D), v=randn(B, Lk, Hkv, D))
    rest = {}
    if lengths == "ragged":
        n = torch.randint(0, Lk + 1, (B,), generator=g)
        n[0] = 0
        n[-1] = Lk if B > 1 else n[-1]
        rest["lengths"] = n.to(torch.int32 if seed % 2 else torch.int64).cuda()
    if holes:
        rest["mask"] = (torch.rand((B, Lk), generator=g) >= holes).cuda()
    return t, rest, randn(B, Lq, H, D)


def check(t, rest, grad, dtype, *, scale=None, gradients=True):
    leaves = {k: v.detach().requires_grad_(gradients) for k, v in t.items()}
    out = to.cross_attention(**leaves, **rest, scale=scale)
    assert out.dtype == dtype and out.shape == t["q"].shape and out.is_contiguous()
    want = field_oracle.cross_attention(dtype, *(t[k].double() for k in "qkv"), rest.get("lengths"), rest.get("mask"), scale, grad.double() if gradients else None)
    _close(out.detach(), want["out"], "out", dtype)
    if gradients:
        for name, got in zip("qkv", torch.autograd.grad(out, list(leaves.values()), grad)):
            assert got.dtype == dtype
            _close(got, want[name], f"gradient of {name}", dtype)
    assert torch.equal(to.cross_attention(**t, **rest, scale=scale), out.detach())
    return out.detach()


def _close(got, want, what, dtype):
    value, size, narrow = want
    field_oracle.assert_close(got, value, size, what, narrow, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=ids)
def test_values_and_gradients(shape, dtype):
    if dtype == "f32" and shape[5] > 128:
        pytest.skip("float32 heads have up to 128 values")
    check(*made(shape, DTYPES[dtype], seed=SHAPES.index(shape)), DTYPES[dtype])


@pytest.mark.parametrize("holes", [0.0, 0.3, 1.0])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(4, 1, 77, 4, 2, 32), (5, 40, 130, 2, 2, 64), (3, 150, 64, 4, 1, 24), (6, 2, 700, 2, 1, 128)], ids=ids)
def test_masks(shape, dtype, holes):
    t, rest, grad = made(shape, DTYPES[dtype], lengths="ragged", holes=holes, seed=shape[2])
    out = check(t, rest, grad, DTYPES[dtype])
    assert not out[0].any()
    if holes == 1.0:
        assert not out.any()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(3, 1, 90, 4, 2, 32), (3, 70, 90, 2, 2, 64), (3, 40, 20, 2, 1, 16)], ids=ids)
def test_what_lies_behind_a_mask_reaches_nothing(shape, dtype, value):
    t, rest, grad = made(shape, DTYPES[dtype], lengths="ragged", holes=0.4, seed=3)

    def run(t):
        t = {k: v.detach().clone().requires_grad_() for k, v in t.items()}
        out = to.cross_attention(**t, **rest)
        return [out.detach(), *torch.autograd.grad(out, list(t.values()), grad)]

    clean = run(t)
    allowed = rest["mask"] & (torch.arange(shape[2], device="cuda")[None] < rest["lengths"][:, None])
    spoiled = {k: v if k == "q" else torch.where(allowed[:, :, None, None], v, value) for k, v in t.items()}
    for a, b in zip(clean, run(spoiled)):
        assert torch.equal(a, b)
    for g in clean[2:]:
        assert not g[~allowed].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [1, 5, 40, 300])
def test_a_single_key_has_no_gradient_of_its_score(dtype, queries):
    """Its weight is 1 whatever the score, so q and k get zeros, and not what rounding leaves of a difference of equal numbers."""
    for keys, lengths in ((1, None), (200, [1, 0, 1])):
        t, _, grad = made((3, queries, keys, 4, 2, 32), DTYPES[dtype], seed=20)
        rest = {} if lengths is None else dict(lengths=torch.tensor(lengths).cuda())
        leaves = {k: v.requires_grad_() for k, v in t.items()}
        dq, dk, dv = torch.autograd.grad(to.cross_attention(**leaves, **rest), list(leaves.values()), grad)
        assert not dq.any() and not dk.any() and dv[0, 0].all()


def test_samples_stay_apart():
    t, rest, grad = made((3, 40, 50, 2, 2, 32), torch.float32, seed=4)
    clean = to.cross_attention(**t)
    t["k"][1, 7, 0, 3] = math.nan
    out = to.cross_attention(**t)
    assert torch.equal(out[[0, 2]], clean[[0, 2]]) and torch.equal(out[1, :, 1], clean[1, :, 1]) and out[1, :, 0].isnan().all()


@pytest.mark.parametrize("lengths", [[-5, 3, 1000], [-(2**31), 2**31 - 1, 0], [1, 2, 9]])
def test_lengths_outside_the_keys(lengths):
    t, _, grad = made((3, 4, 9, 2, 1, 16), torch.float32, seed=5)
    n = torch.tensor(lengths, dtype=torch.int64).cuda()
    check(t, dict(lengths=n.clamp(0, 9)), grad, torch.float32)
    want = to.cross_attention(**t, lengths=n.clamp(0, 9))
    assert torch.equal(to.cross_attention(**t, lengths=n), want) and torch.equal(to.cross_attention(**t, lengths=n.int()), want)
    if n.max() > 1000:
        assert torch.equal(to.cross_attention(**t, lengths=n * 2**20), want)


@pytest.mark.parametrize("scale", [0.0, -0.4, 2.5, 1e-3])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales(dtype, scale):
    t, rest, grad = made((2, 40, 70, 2, 1, 32), DTYPES[dtype], lengths="ragged", seed=6)
    check(t, rest, grad, DTYPES[dtype], scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(dtype):
    """Weights of one for the largest score: the running maximum moves, and all else underflows."""
    t, rest, grad = made((2, 50, 400, 2, 2, 64), DTYPES[dtype], seed=7)
    t["q"] *= 30
    check(t, rest, grad, DTYPES[dtype])
    order = (t["q"][:, :1, :1].double() * t["k"].double()).sum(3)[:, :, 0].argsort(dim=1)  # rising scores for the first row
    for k in ("k", "v"):
        t[k] = torch.stack([t[k][b, order[b]] for b in range(2)])
    check(t, rest, grad, DTYPES[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    dtype = DTYPES[dtype]
    g = torch.Generator().manual_seed(8)
    randn = lambda *s: torch.randn(s, generator=g).to(dtype).cuda()
    B, Lq, Lk, H, D = 2, 45, 70, 3, 24
    grad = randn(B, Lq, H, D)
    kv = randn(B, Lk, 2, H, D)  # one projection of both
    variants = [
        dict(q=randn(B, H, Lq, D).transpose(1, 2), k=kv[:, :, 0], v=kv[:, :, 1]),
        dict(q=randn(B, Lq, H * D + 3)[..., 3:].unflatten(2, (H, D)), k=randn(Lk, B, H, D).transpose(0, 1), v=randn(B, Lk, D, H).transpose(2, 3)),
        dict(q=randn(1, Lq, H, D).expand(B, Lq, H, D), k=randn(B, Lk, 1, D).expand(B, Lk, H, D), v=randn(1, 1, H, D).expand(B, Lk, H, D)),
        dict(q=randn(B, 2 * Lq, H, D)[:, ::2], k=randn(B, Lk, H, 2 * D)[..., ::2], v=randn(B, Lk, 2 * H, D)[:, :, 1::2]),
    ]
    for t in variants:
        check(t, {}, grad, dtype)
        same = {k: v.contiguous() for k, v in t.items()}
        assert torch.equal(to.cross_attention(**t), to.cross_attention(**same))
    # a cotangent in another order
    leaves = {k: v.clone().requires_grad_() for k, v in variants[0].items()}
    out = to.cross_attention(**leaves)
    a = torch.autograd.grad(out, list(leaves.values()), grad, retain_graph=True)
    b = torch.autograd.grad(out, list(leaves.values()), grad.transpose(1, 2).contiguous().transpose(1, 2))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    mask = torch.rand((B, 2 * Lk), generator=g).cuda() < 0.5
    t = variants[0]
    assert torch.equal(to.cross_attention(**t, mask=mask[:, ::2]), to.cross_attention(**t, mask=mask[:, ::2].contiguous()))
    assert torch.equal(to.cross_attention(**t, mask=mask[:1, :Lk].expand(B, Lk)), to.cross_attention(**t, mask=mask[:1, :Lk].repeat(B, 1)))
    assert torch.equal(to.cross_attention(**t, mask=mask[:, :Lk]), to.cross_attention(**t, mask=mask[:, :Lk].contiguous()))


@pytest.mark.parametrize("shape", [(0, 3, 4, 2, 1, 8), (2, 0, 4, 2, 1, 8), (2, 3, 0, 2, 1, 8), (2, 0, 0, 2, 2, 8)], ids=ids)
def test_empty(shape):
    t, rest, grad = made(shape, torch.float32)
    leaves = {k: v.requires_grad_() for k, v in t.items()}
    out = to.cross_attention(**leaves)
    assert out.shape == t["q"].shape and not out.any()
    for k, g in zip("qkv", torch.autograd.grad(out, list(leaves.values()), grad)):
        assert g.shape == t[k].shape and not g.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2, 40, 50, 2, 1, 16), (2, 1, 300, 4, 2, 64), (1, 300, 20, 2, 2, 128)], ids=ids)
def test_some_gradients_only(shape, dtype):
    t, rest, grad = made(shape, DTYPES[dtype], seed=9)
    full = {k: v.clone().requires_grad_() for k, v in t.items()}
    want = dict(zip("qkv", torch.autograd.grad(to.cross_attention(**full), list(full.values()), grad)))
    for name in "qkv":
        one = {k: v.clone().requires_grad_(k == name) for k, v in t.items()}
        assert torch.equal(torch.autograd.grad(to.cross_attention(**one), one[name], grad)[0], want[name])


def test_gradients_against_differences():
    t, rest, _ = made((1, 3, 5, 2, 1, 4), torch.float32, seed=10)
    grad = torch.randn(1, 3, 2, 4, generator=torch.Generator().manual_seed(1)).cuda()
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    gradients = torch.autograd.grad(to.cross_attention(**leaves), list(leaves.values()), grad)
    for name, g in zip("qkv", gradients):
        for i in range(t[name].numel()):
            # central differences in float32: the step's truncation (h^2) and the values' rounding (2^-24 / h) are below 1e-3
            h, values = 1e-2, []
            for sign in (1, -1):
                moved = {k: v.clone() for k, v in t.items()}
                moved[name].view(-1)[i] += sign * h
                values.append((to.cross_attention(**moved).double() * grad).sum())
            assert abs((values[0] - values[1]) / (2 * h) - g.flatten()[i]) < 2e-3


def test_same_bits_every_time():
    t, rest, grad = made((3, 200, 1500, 8, 2, 64), torch.bfloat16, lengths="ragged", holes=0.1, seed=11)
    leaves = {k: v.requires_grad_() for k, v in t.items()}

    def run():
        out = to.cross_attention(**leaves, **rest)
        return [out.detach(), *torch.autograd.grad(out, list(leaves.values()), grad)]

    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_two_streams_at_once():
    t, rest, _ = made((2, 1, 20000, 8, 2, 64), torch.bfloat16, seed=12)
    u, more, _ = made((2, 300, 900, 8, 2, 64), torch.bfloat16, seed=13)
    want = [to.cross_attention(**t), to.cross_attention(**u)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            a = to.cross_attention(**t)
        b = to.cross_attention(**u)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])


@pytest.mark.parametrize("shape", [(2, 1, 6000, 4, 2, 64), (2, 150, 200, 4, 2, 64), (1, 3000, 20, 2, 2, 32)], ids=ids)
def test_captured_forward_and_backward(shape):
    t, rest, grad = made(shape, torch.float32, lengths="ragged", seed=15)
    static = {k: v.clone().requires_grad_() for k, v in t.items()}

    def run(t):
        out = to.cross_attention(**t, **rest)
        return [out, *torch.autograd.grad(out, list(t.values()), grad)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(static)
    for i in range(4):
        with torch.no_grad():
            for k in t:
                static[k].copy_(t[k] * (1 + 0.25 * i))
            rest["lengths"].add_(i).clamp_(0, shape[2])
        graph.replay()
        want = run({k: v.detach().clone().requires_grad_() for k, v in static.items()})
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_mapped_over_samples():
    t, rest, grad = made((5, 9, 40, 4, 2, 16), torch.float32, lengths="ragged", holes=0.2, seed=16)

    def f(q, k, v, n, m):
        return to.cross_attention(q[None], k[None], v[None], lengths=n[None], mask=m[None])[0]

    out = torch.func.vmap(f)(*t.values(), rest["lengths"], rest["mask"])
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    whole = to.cross_attention(**leaves, **rest)
    assert torch.equal(out, whole)

    def pulled(q, k, v, n, m, g):
        return torch.func.vjp(lambda *x: f(*x, n, m), q, k, v)[1](g)

    got = torch.func.vmap(pulled)(*t.values(), rest["lengths"], rest["mask"], grad)
    assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(whole, list(leaves.values()), grad)))
    # a context that all mapped samples share: a gradient of its own for each of them
    got = torch.func.vmap(lambda q, g: torch.func.vjp(lambda k: to.cross_attention(q[None], k[None], t["v"][:1])[0], t["k"][0])[1](g)[0])(t["q"], grad)
    shared = t["k"][:1].repeat(5, 1, 1, 1).requires_grad_()
    (want,) = torch.autograd.grad(to.cross_attention(t["q"], shared, t["v"][:1].expand(5, -1, -1, -1)), shared, grad)
    assert torch.equal(got, want)


def test_not_differentiable_twice():
    t, _, _ = made((1, 2, 3, 1, 1, 4), torch.float32)
    q = t["q"].requires_grad_()
    (g,) = torch.autograd.grad(to.cross_attention(**t).square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(g.sum(), q)


def test_compiled():
    t, rest, grad = made((2, 20, 30, 4, 2, 16), torch.float32, lengths="ragged", seed=17)
    f = lambda q, k, v, n: to.cross_attention(2 * q, k, v, lengths=n) + 1
    eager = [v.clone().requires_grad_() for v in t.values()]
    out = f(*eager, rest["lengths"])
    want = torch.autograd.grad(out, eager, grad)
    leaves = [v.clone().requires_grad_() for v in t.values()]
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(*leaves, rest["lengths"])
    assert torch.equal(got, out)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, leaves, grad), want))


# every form of the two backward kernels: up to 32 rows a head of keys and more, up to 32 keys and more, keys and rows in one piece and in several
@pytest.mark.parametrize("exponent", [-17, -13, -7, 6, 12])
@pytest.mark.parametrize(
    "shape", [(2, 1, 2, 1, 1, 128), (2, 1, 60, 4, 2, 16), (2, 12, 3000, 2, 1, 16), (2, 40, 20, 2, 2, 64), (1, 600, 20, 2, 2, 32), (1, 1100, 300, 2, 1, 64), (1, 100, 2500, 2, 2, 128), (2, 70, 90, 2, 1, 256)], ids=ids
)
def test_float16_gradients_of_cotangents_of_any_size(shape, exponent):
    """Gradients are linear in the cotangent: what is allowed at cotangents of 2^e is what is allowed at 1, times 2^e, and the steps of the
    results' own type."""
    B, Lq, Lk, H, Hkv, D = shape
    t, rest, grad = made(shape, torch.float16, seed=30)
    # many keys: weights near 1 / Lk, and gradients of q that float16 can hold all the same
    scale = 1.0 if Lk > 1000 else None
    if scale:
        t["q"] = t["q"] / (2 * math.sqrt(D))
    size = 2.0**exponent
    grad = (grad.float() * size).half()
    leaves = {k: v.requires_grad_() for k, v in t.items()}
    got = torch.autograd.grad(to.cross_attention(**leaves, scale=scale), list(leaves.values()), grad)
    want = field_oracle.cross_attention(torch.float16, *(v.detach().double() for v in t.values()), None, None, scale, grad.double() / size)
    for name, g in zip("qkv", got):
        value, tolerance, narrow = (size * x for x in want[name])
        fits = value.abs() < 65000
        assert not g.isnan().any() and not (g.isinf() & fits).any()
        field_oracle.assert_close(torch.where(fits, g, 0), torch.where(fits, value, 0), tolerance, f"gradient of {name}", narrow, torch.float16)


def test_float16_gradients_of_large_cotangents():
    """Score gradients beyond 65 504 whose sums are not."""
    g = torch.Generator().manual_seed(31)
    randn = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)
    t = dict(q=randn(4, 1, 1, 128) * 0.1, k=randn(4, 2, 1, 128) * 0.5, v=randn(4, 2, 1, 128))
    t = {k: v.half().cuda().requires_grad_() for k, v in t.items()}
    grad = (randn(4, 1, 1, 128) * 6000 + 6000 * t["v"][:, :1].detach().cpu().double()).half().cuda()
    got = torch.autograd.grad(to.cross_attention(**t), list(t.values()), grad)
    want = field_oracle.cross_attention(torch.float16, *(v.detach().double() for v in t.values()), None, None, None, grad.double())
    assert all(want[name][0].abs().max() < 65504 for name in "qk")
    q, k, v = (t[name].detach().cpu().double() for name in "qkv")
    p = torch.softmax(q[:, 0] @ k[:, :, 0].mT / math.sqrt(128), dim=2)
    dp = grad.cpu().double()[:, 0] @ v[:, :, 0].mT
    assert (p * (dp - (p * dp).sum(2, keepdim=True))).abs().max() > 65504
    for name, x in zip("qk", got):
        _close(x, want[name], f"gradient of {name}", torch.float16)


@pytest.mark.parametrize("where", ["q", "k"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2, 1, 50, 2, 2, 32), (2, 1, 5000, 2, 2, 64), (2, 20, 300, 2, 1, 64), (2, 300, 40, 1, 1, 64), (2, 300, 700, 2, 1, 64), (300, 40, 100, 2, 2, 16)], ids=ids)
def test_a_row_of_nan_reaches_all_that_it_looks_at(shape, dtype, where):
    """The weights of a row whose scores hold a NaN are NaN, and so are the gradients of all values it looks at."""
    B, Lq, Lk, H, Hkv, D = shape
    t, _, grad = made(shape, DTYPES[dtype], seed=32)
    t[where][1, 0, 0, 3] = math.nan
    lengths = torch.full((B,), Lk - 1, device="cuda")
    leaves = {k: v.requires_grad_() for k, v in t.items()}
    out = to.cross_attention(**leaves, lengths=lengths)
    dq, dk, dv = torch.autograd.grad(out, list(leaves.values()), grad)
    assert out[1, 0, 0].isnan().all() and out[0].isfinite().all()
    assert dq[1, 0, 0].isnan().all() and dk[1, : Lk - 1, 0].isnan().all() and dv[1, : Lk - 1, 0].isnan().all()
    assert not dk[1, Lk - 1].any() and not dv[1, Lk - 1].any() and dk[0].isfinite().all() and dv[0].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(4, 1, 3, 2, 2, 16), (4, 5, 700, 4, 2, 32), (4, 40, 20, 2, 2, 64), (4, 300, 1030, 2, 1, 64)], ids=ids)
def test_a_single_key_that_a_mask_leaves_has_no_gradient_of_its_score(shape, dtype):
    """As one of a single length: by the mask alone, and by both."""
    B, Lq, Lk, H, Hkv, D = shape
    t, _, grad = made(shape, DTYPES[dtype], seed=33)
    mask = torch.zeros((B, Lk), dtype=torch.bool, device="cuda")
    mask[0, 0] = mask[1, Lk - 1] = mask[2, Lk // 2] = mask[3, Lk // 2] = mask[3, Lk - 1] = True
    for rest, zero in ((dict(mask=mask), [0, 1, 2]), (dict(mask=mask, lengths=torch.tensor([Lk, Lk, Lk, Lk - 1], device="cuda")), [0, 1, 2, 3])):
        leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
        out = to.cross_attention(**leaves, **rest)
        dq, dk, dv = torch.autograd.grad(out, list(leaves.values()), grad)
        assert not dq[zero].any() and not dk[zero].any() and not dv[~mask].any()
        assert all(dv[b][mask[b]].any() for b in (0, 1, 2, 3)) and (len(zero) == 4 or (dq[3].any() and dk[3].any()))
        want = field_oracle.cross_attention(DTYPES[dtype], *(t[k].double() for k in "qkv"), rest.get("lengths"), mask, None, grad.double())
        for name, got in zip(("out", *"qkv"), (out.detach(), dq, dk, dv)):
            _close(got, want[name], name, DTYPES[dtype])


@pytest.mark.parametrize("batch,training", [(2**26 + 41, False), (2**24 + 41, True)])
def test_more_workgroups_than_a_grid_has_in_a_row(batch, training):
    """2^32 threads and more: as the same samples a part at a time."""
    g = torch.Generator("cuda").manual_seed(34)
    t = {k: torch.randn((batch, 2 if k != "q" else 1, 1, 4), generator=g, dtype=torch.float16, device="cuda").requires_grad_(training) for k in "qkv"}
    grad = torch.randn((batch, 1, 1, 4), generator=g, dtype=torch.float16, device="cuda")

    def run(t, grad):
        out = to.cross_attention(**t)
        return [out.detach(), *(torch.autograd.grad(out, list(t.values()), grad) if training else [])]

    whole, step = run(t, grad), 2**23
    for first in range(0, batch, step):
        part = run({k: v.detach()[first : first + step].requires_grad_(training) for k, v in t.items()}, grad[first : first + step])
        assert all(torch.equal(a[first : first + step], b) for a, b in zip(whole, part))


# Sizes that take each form of many samples: float32 with 512 groups of 128 rows and more (four wavefronts on tiles that they share, and up to 128 keys in
# LDS), single tokens with more of them than share keys between wavefronts, and every number of 32 keys that stays in LDS.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(
    "shape",
    [
        (256, 40, 70, 2, 2, 32),
        (256, 140, 100, 2, 2, 64),
        (513, 33, 128, 1, 1, 64),
        (256, 20, 70, 4, 2, 32),
        (256, 40, 129, 2, 2, 32),
        (256, 50, 300, 2, 2, 64),
        (130, 70, 129, 4, 4, 80),
        (128, 130, 300, 4, 4, 128),
        (70, 200, 300, 9, 9, 20),
        (2, 300, 60, 2, 1, 128),
        (2, 300, 70, 2, 1, 128),
        (2, 300, 128, 2, 2, 32),
        (2, 300, 120, 2, 1, 128),
        (513, 40, 90, 1, 1, 64),
        (2, 200, 500, 2, 2, 96),
        (8200, 1, 200, 1, 1, 32),
        (2100, 2, 40, 4, 4, 16),
        (1100, 3, 33, 8, 8, 8),
        (300, 7, 700, 2, 2, 40),
        (3, 40, 20, 2, 1, 200),
    ],
    ids=ids,
)
def test_forms_of_many_samples(shape, dtype):
    if dtype == "f32" and shape[5] > 128:
        pytest.skip("float32 heads have up to 128 values")
    check(*made(shape, DTYPES[dtype], lengths="ragged", holes=0.2, seed=sum(shape)), DTYPES[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
def test_forms_of_many_samples_without_a_mask(dtype):
    """(and without lengths: tiles of which every key may be looked at take a shorter way)"""
    check(*made((256, 140, 320, 2, 2, 64), DTYPES[dtype], seed=35), DTYPES[dtype])


def test_tangents_are_refused():
    t, _, grad = made((2, 3, 5, 2, 1, 8), torch.float32)
    q = t["q"].requires_grad_()
    out = to.cross_attention(**t)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out, q, torch.autograd.forward_ad.make_dual(grad, grad))

    def derivative(v):
        return torch.func.jvp(lambda v: to.cross_attention(v, t["k"], t["v"]), (v,), (torch.ones_like(v),))

    for f in (derivative, torch.compile(derivative, backend="eager")):
        with pytest.raises(NotImplementedError, match="jvp|forward-mode"):
            f(q.detach())


@pytest.mark.parametrize("how", ["trace", "make_fx", "make_fx of gradients", "make_fx of vjp", "make_fx of vmap", "make_fx of a backward pass", "make_fx, symbolic"])
def test_recorded_programs(how):
    """What records a program sees the operation: its replay computes from new inputs what a call does."""
    from torch.fx.experimental.proxy_tensor import make_fx

    (first, dy), (other, _) = ((list(t.values()), dy) for t, _, dy in (made((3, 5, 7, 4, 2, 16), torch.bfloat16, seed=s) for s in (36, 37)))
    lengths = torch.tensor([7, 0, 4], device="cuda")

    def call(q, k, v):
        return to.cross_attention(q, k, v, lengths=None if how in ("make_fx of vmap", "make_fx, symbolic") else lengths)

    def gradients(*values):
        leaves = [v.detach().requires_grad_() for v in values]
        return torch.autograd.grad(call(*leaves), leaves, dy)

    def pulled(*values):
        return torch.func.vjp(call, *values)[1](dy)

    def mapped(*values):
        return torch.func.vmap(lambda *one: call(*(v[None] for v in one))[0])(*values)

    f = {"make_fx of gradients": gradients, "make_fx of vjp": pulled, "make_fx of vmap": mapped}.get(how, call)
    if how == "make_fx of a backward pass":  # (of a graph that was there before)
        leaves = [v.clone().requires_grad_() for v in first]
        y = call(*leaves)
        program = make_fx(lambda g: torch.autograd.grad(y, leaves, g, retain_graph=True))(dy)
        for got, want in zip(program(2 * dy), torch.autograd.grad(y, leaves, 2 * dy)):
            assert torch.equal(got, want)
        return
    with torch.no_grad() if how == "trace" else torch.enable_grad():
        program = torch.jit.trace(f, tuple(first)) if how == "trace" else make_fx(f, tracing_mode="symbolic" if "symbolic" in how else "real")(*first)
    held = torch.empty(1 << 20, device="cuda").fill_(7)  # (memory that a program without its kernels would find)
    del held
    for values in (first, other):
        got, want = program(*values), f(*values)
        for a, b in zip(*((x,) if torch.is_tensor(x) else x for x in (got, want))):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_batched_cotangents(dtype):
    """As one after the other: autograd.grad with is_grads_batched, a Jacobian, and vmap around autograd.grad."""
    t, _, _ = made((2, 3, 5, 4, 2, 4), DTYPES[dtype], seed=38)
    lengths = torch.tensor([5, 3], device="cuda")
    leaves = [v.requires_grad_() for v in t.values()]
    call = lambda q, k, v: to.cross_attention(q, k, v, lengths=lengths)
    out = call(*leaves)
    grad = torch.randn((6, *out.shape), generator=torch.Generator().manual_seed(1)).to(DTYPES[dtype]).cuda()
    want = [torch.stack(g) for g in zip(*(torch.autograd.grad(out, leaves, g, retain_graph=True) for g in grad))]
    got = torch.autograd.grad(out, leaves, grad, is_grads_batched=True, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    (got,) = torch.autograd.grad(out, leaves[1], grad, is_grads_batched=True, retain_graph=True)
    assert torch.equal(got, want[1])
    for dim in range(5):
        got = torch.func.vmap(lambda g: torch.autograd.grad(out, leaves, g, retain_graph=True), in_dims=dim)(grad.movedim(0, dim))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    rows = torch.autograd.functional.jacobian(call, tuple(v.detach() for v in leaves), vectorize=True)
    one = torch.autograd.functional.jacobian(call, tuple(v.detach() for v in leaves))
    assert all(torch.equal(a, b) for a, b in zip(rows, one))


@pytest.mark.parametrize("which", ["q", "k", "v", "grad"])
@pytest.mark.parametrize("head_dim", [1, 8])
def test_views_that_are_flagged_negative(which, head_dim):
    """The imaginary part of a conjugate: its memory holds the values of the other sign."""
    t, _, grad = made((2, 3, 5, 2, 1, head_dim), torch.float32, seed=39)
    t["grad"] = grad
    flagged = {**t, which: torch.complex(torch.zeros_like(t[which]), -t[which]).conj().imag}
    assert flagged[which].is_neg() and torch.equal(flagged[which], t[which])

    def run(q, k, v, grad):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out = to.cross_attention(*leaves)
        return [out.detach(), *torch.autograd.grad(out, leaves, grad)]

    assert all(torch.equal(a, b) for a, b in zip(run(**flagged), run(**t)))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", [(418, 112, 4, 8, 8, 16), (60, 400, 300, 4, 4, 64), (700, 8, 50, 4, 4, 64), (2, 1, 20000, 16, 4, 64), (16, 500, 900, 4, 2, 128)], ids=ids)
def test_an_output_and_what_rounding_takes_off_it(shape, dtype):
    """Their sum is what was there ahead of the rounding, also where that lay in the middle between two steps of the type."""
    from torchode_amd import _lib

    dtype = DTYPES[dtype]
    t, _, _ = made(shape, dtype, seed=40)
    out, low, _ = _lib.load_host().cross_attention_forward(t["q"], t["k"], t["v"], None, None, None)
    want, size, narrow = field_oracle.cross_attention(dtype, *(t[k].double() for k in "qkv"), None, None, None)["out"]
    error = (out.double() + low.double() - want).abs()
    # (the remainder's own rounding: half a step of half a step, and of float16's smallest numbers)
    tolerance = field_oracle.ROUNDINGS * 2.0**-24 * size + narrow + (torch.finfo(dtype).eps / 2) ** 2 * want.abs() + (2.0**-25 if dtype == torch.float16 else 0)
    assert (error <= tolerance).all(), ((error / tolerance).max(), int((error > tolerance).sum()))
