"""``torchode_amd.group_norm`` against its definition in float64: types, grids and channels of every alignment, activations,
modulation, gradients; inside solves, HIP graphs, ``vmap`` and ``torch.compile``."""
import pytest
import torch

import torchode_amd as to
from tests import field_oracle

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f64": torch.float64, "bf16": torch.bfloat16, "f16": torch.float16}
KINDS = [None, "silu", "gelu", "tanh", "relu"]
# batch, grid, channels, groups
SHAPES = [
    (3, (), 6, 3),
    (1, (1,), 4, 4),  # groups of a single value: nothing but the bias is left
    (5, (3,), 1, 1),
    (2, (7, 5), 2, 1),
    (3, (5, 7), 30, 5),
    (4, (8, 8), 32, 8),
    (2, (64, 64), 16, 4),
    (1, (131, 129), 40, 8),
    (2, (9, 11), 640, 32),
    (3, (2, 3, 4, 5), 24, 3),
    (1, (20011,), 6, 2),
    (2, (50,), 1501, 1),  # an odd row, wider than a workgroup
    (2, (33,), 2056, 8),
    (33000, (2,), 4, 2),  # more samples than one dimension of a grid takes
    (300, (16,), 8, 8),
    (1, (700, 90), 64, 1),
]


def made(shape, dtype, *, params, modulated, per_sample=False, seed=0, offset=1.0):
    B, grid, C, _ = shape
    g = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)
    x = offset * randn(C) + randn(B, *grid, C) * (0.5 + randn(C).abs())
    affine = (B, C) if per_sample else (C,)
    t = dict(x=x.to(dtype), weight=(1 + 0.3 * randn(*affine)).to(params), bias=(0.3 * randn(*affine)).to(params))
    if modulated:
        t.update(scale=(0.4 * randn(B, C)).to(params), shift=(0.4 * randn(B, C)).to(params))
    return {k: v.cuda() for k, v in t.items()}, randn(B, *grid, C).to(dtype).cuda()


def check(shape, dtype, kind, t, dy, *, eps=1e-5, gradients=True, narrow=0.0):
    G = shape[3]
    leaves = {k: v.detach().requires_grad_(gradients) for k, v in t.items()}
    rest = {k: v for k, v in leaves.items() if k != "x"}
    y = to.group_norm(leaves["x"], G, rest.get("weight"), rest.get("bias"), scale=rest.get("scale"), shift=rest.get("shift"), activation=kind, eps=eps)
    assert y.dtype == dtype and y.shape == t["x"].shape
    names = ("weight", "bias", "scale", "shift")
    want = field_oracle.group_norm(dtype, t["x"].double(), G, *(t[k].double() if k in t else None for k in names), kind, eps, dy.double() if gradients else None)
    field_oracle.assert_close(y.detach(), *want["y"], "y", dtype=dtype)
    if gradients:
        for name, got in zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)):
            assert got.dtype == t[name].dtype
            field_oracle.assert_close(got, *want[name], f"gradient of {name}", dtype=dtype)
    with torch.no_grad():  # the same kernels without a graph
        again = to.group_norm(t["x"], G, t.get("weight"), t.get("bias"), scale=t.get("scale"), shift=t.get("shift"), activation=kind, eps=eps)
    assert torch.equal(again, y.detach()) or (again.isnan() == y.isnan()).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, (s[0], *s[1], s[2]))) + f"g{s[3]}")
def test_values_and_gradients(shape, dtype):
    i = SHAPES.index(shape)
    t, dy = made(shape, DTYPES[dtype], params=DTYPES[dtype], modulated=i % 2 == 0, seed=i)
    check(shape, DTYPES[dtype], KINDS[i % 5], t, dy)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_activations(dtype, kind):
    shape = (3, (13, 6), 24, 4)
    t, dy = made(shape, DTYPES[dtype], params=DTYPES[dtype], modulated=True, seed=5)
    t["weight"] *= 6  # (far into both tails)
    check(shape, DTYPES[dtype], kind, t, dy)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_parameters_in_float32(dtype):
    shape = (5, (11, 12), 40, 10)
    t, dy = made(shape, DTYPES[dtype], params=torch.float32, modulated=True, seed=6)
    check(shape, DTYPES[dtype], "silu", t, dy)
    t["scale"], t["shift"] = t["scale"].to(DTYPES[dtype]), t["shift"].to(DTYPES[dtype])
    check(shape, DTYPES[dtype], "silu", t, dy)


@pytest.mark.parametrize("left_out", [("weight",), ("bias", "scale"), ("weight", "bias", "scale", "shift"), ("shift",)])
def test_parameters_left_out(left_out):
    shape = (3, (10,), 12, 2)
    t, dy = made(shape, torch.float32, params=torch.float32, modulated=True, seed=7)
    check(shape, torch.float32, "gelu", {k: v for k, v in t.items() if k not in left_out}, dy)


@pytest.mark.parametrize("modulated", [False, True])
def test_weights_of_each_sample(modulated):
    shape = (4, (6, 5), 20, 4)
    t, dy = made(shape, torch.float32, params=torch.float32, modulated=modulated, per_sample=True, seed=8)
    check(shape, torch.float32, "silu", t, dy)


def test_some_gradients_only():
    t, dy = made((3, (10,), 12, 2), torch.float32, params=torch.float32, modulated=True, seed=9)
    full = {k: v.clone().requires_grad_() for k, v in t.items()}
    y = to.group_norm(full["x"], 2, full["weight"], full["bias"], scale=full["scale"], shift=full["shift"], activation="silu")
    want = dict(zip(full, torch.autograd.grad(y, list(full.values()), dy)))
    for name in full:
        one = {k: v.clone().requires_grad_(k == name) for k, v in t.items()}
        y = to.group_norm(one["x"], 2, one["weight"], one["bias"], scale=one["scale"], shift=one["shift"], activation="silu")
        assert torch.equal(torch.autograd.grad(y, one[name], dy)[0], want[name])


@pytest.mark.parametrize("dtype", ["f32", "f64", "bf16"])
def test_means_far_from_zero(dtype):
    shape = (2, (40, 40), 24, 3)
    t, dy = made(shape, DTYPES[dtype], params=DTYPES[dtype], modulated=False, seed=10, offset=300.0)
    check(shape, DTYPES[dtype], "silu", t, dy)


def test_a_first_value_far_from_the_others():
    shape = (2, (500,), 8, 2)
    t, dy = made(shape, torch.float32, params=torch.float32, modulated=False, seed=11)
    t["x"][:, 0] = 1e4
    check(shape, torch.float32, None, t, dy)


def test_groups_without_spread():
    x = torch.full((2, 30, 8), 3.25, device="cuda", requires_grad=True)
    y = to.group_norm(x, 2, torch.full((8,), 2.0, device="cuda"), torch.full((8,), 0.5, device="cuda"))
    assert torch.equal(y, torch.full_like(x, 0.5))
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert dx.abs().max() < 1e-3  # (2 / sqrt(1e-5) times the rounding error of a mean of ones)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_samples_and_groups_stay_apart(value):
    t, dy = made((4, (9, 9), 16, 4), torch.float32, params=torch.float32, modulated=True, seed=12)

    def run(x):
        x = x.clone().requires_grad_()
        y = to.group_norm(x, 4, t["weight"], t["bias"], scale=t["scale"], shift=t["shift"], activation="tanh")
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    clean = run(t["x"])
    spoiled = t["x"].clone()
    spoiled[2, 4, 4, 5] = value
    for a, b in zip(clean, run(spoiled)):
        assert b[2, :, :, 4:8].isnan().any()
        b[2, :, :, 4:8] = a[2, :, :, 4:8]
        assert torch.equal(a, b)


def test_layouts():
    g = torch.Generator().manual_seed(13)
    base = torch.randn((3, 20, 6, 5), generator=g).cuda()
    w = torch.randn((32,), generator=g).cuda()[::2]
    for x in (base.permute(0, 2, 3, 1)[..., :16], torch.randn((3, 6, 5, 33), generator=g).cuda()[..., 1:17], base[:, :16].reshape(3, 16, 30).transpose(1, 2)):
        assert torch.equal(to.group_norm(x, 4, w, activation="silu"), to.group_norm(x.contiguous(), 4, w.contiguous(), activation="silu"))
    flat = torch.randn((1 + 3 * 30 * 16,), generator=g).cuda()  # an address that is no multiple of 16 bytes
    x = flat[1:].view(3, 30, 16)
    assert torch.equal(to.group_norm(x, 4), to.group_norm(x.clone(), 4))


@pytest.mark.parametrize("shape", [(0, 5, 4), (3, 0, 4)])
def test_empty(shape):
    t = dict(x=torch.zeros(shape, device="cuda"), weight=torch.ones(4, device="cuda"), bias=torch.ones(4, device="cuda"), scale=torch.ones(shape[0], 4, device="cuda"))
    t = {k: v.requires_grad_() for k, v in t.items()}
    y = to.group_norm(t["x"], 2, t["weight"], t["bias"], scale=t["scale"])
    assert y.shape == shape
    for k, g in zip(t, torch.autograd.grad(y, list(t.values()), torch.zeros_like(y))):
        assert g.shape == t[k].shape and not g.any()


def test_gradients_against_differences():
    t, _ = made((2, (3, 2), 6, 2), torch.float64, params=torch.float64, modulated=True, seed=14)
    for kind in ("silu", "gelu", "tanh"):
        f = lambda x, w, b, s, h: to.group_norm(x, 2, w, b, scale=s, shift=h, activation=kind)
        assert torch.autograd.gradcheck(f, [v.requires_grad_() for v in t.values()])


def test_same_bits_every_time():
    t, dy = made((6, (37, 41), 48, 6), torch.bfloat16, params=torch.float32, modulated=True, seed=15)
    t = {k: v.requires_grad_() for k, v in t.items()}

    def run():
        y = to.group_norm(t["x"], 6, t["weight"], t["bias"], scale=t["scale"], shift=t["shift"], activation="silu")
        return [y.detach(), *torch.autograd.grad(y, list(t.values()), dy)]

    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_another_stream():
    t, _ = made((8, (64, 64), 32, 4), torch.float32, params=torch.float32, modulated=False, seed=16)
    want = to.group_norm(t["x"], 4, t["weight"], t["bias"], activation="silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = to.group_norm(t["x"] + 0, 4, t["weight"], t["bias"], activation="silu")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_captured_forward_and_backward():
    t, dy = made((4, (30, 31), 24, 4), torch.float32, params=torch.float32, modulated=True, seed=17)
    static = {k: v.clone().requires_grad_() for k, v in t.items()}

    def run(t):
        y = to.group_norm(t["x"], 4, t["weight"], t["bias"], scale=t["scale"], shift=t["shift"], activation="silu")
        return [y, *torch.autograd.grad(y, list(t.values()), dy)]

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
        graph.replay()
        want = run({k: v.detach().clone().requires_grad_() for k, v in static.items()})
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_mapped_over_samples():
    """vmap of values and of gradients: the same as one call with all samples, weights and their gradients of each sample included."""
    t, dy = made((5, (6, 7), 12, 3), torch.float32, params=torch.float32, modulated=True, seed=18)

    def f(w, b, x, s, h):
        return to.group_norm(x[None], 3, w, b, scale=s[None], shift=h[None], activation="silu")[0]

    y = torch.func.vmap(f, in_dims=(None, None, 0, 0, 0))(t["weight"], t["bias"], t["x"], t["scale"], t["shift"])
    assert torch.equal(y, to.group_norm(t["x"], 3, t["weight"], t["bias"], scale=t["scale"], shift=t["shift"], activation="silu"))

    def pulled(x, s, h, g):
        value, pull = torch.func.vjp(f, t["weight"], t["bias"], x, s, h)
        return value, pull(g)

    value, gradients = torch.func.vmap(pulled)(t["x"], t["scale"], t["shift"], dy)
    assert torch.equal(value, y)
    leaves = {k: (v[None].repeat(5, 1) if k in ("weight", "bias") else v).clone().requires_grad_() for k, v in t.items()}
    out = to.group_norm(leaves["x"], 3, leaves["weight"], leaves["bias"], scale=leaves["scale"], shift=leaves["shift"], activation="silu")
    want = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), dy)))
    for name, got in zip(("weight", "bias", "x", "scale", "shift"), gradients):
        assert torch.equal(got, want[name]), name


def test_not_differentiable_twice():
    x = torch.randn(2, 5, 4, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(to.group_norm(x, 2).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(g.sum(), x)


def test_compiled():
    t, dy = made((4, (10,), 16, 4), torch.float32, params=torch.float32, modulated=True, seed=19)

    def f(x, w, b, s, h):
        return to.group_norm(2 * x, 4, w, b, scale=s, shift=h, activation="silu") + 1

    names = ("x", "weight", "bias", "scale", "shift")
    eager = [t[k].clone().requires_grad_() for k in names]
    y = f(*eager)
    want = torch.autograd.grad(y, eager, dy)
    leaves = [t[k].clone().requires_grad_() for k in names]
    out = torch.compile(f, backend="aot_eager", fullgraph=True)(*leaves)
    assert torch.equal(out, y)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, dy), want))


def test_more_workgroups_than_a_grid_has_in_a_row():
    """2^32 threads and more: as the same samples a part at a time."""
    batch, step, g = 2**26 + 41, 2**23, torch.Generator("cuda").manual_seed(20)
    x, dy = (torch.randn((batch, 4), generator=g, dtype=torch.float16, device="cuda") for _ in range(2))
    scale = torch.randn((batch, 4), generator=g, dtype=torch.float16, device="cuda")

    def run(x, scale, dy):
        leaves = [x.detach().requires_grad_(), scale.detach().requires_grad_()]
        y = to.group_norm(leaves[0], 2, scale=leaves[1], activation="silu")
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    whole = run(x, scale, dy)
    for first in range(0, batch, step):
        part = run(x[first : first + step], scale[first : first + step], dy[first : first + step])
        assert all(torch.equal(a[first : first + step], b) for a, b in zip(whole, part))


@pytest.mark.parametrize("dtype,channels", [("bf16", 2048), ("f16", 2048), ("f32", 1024), ("f64", 512)])
def test_as_many_groups_as_channels(dtype, channels):
    """All channels of a row in one workgroup, each a group of its own."""
    shape = (1030, (5,), channels, channels)
    t, dy = made(shape, DTYPES[dtype], params=DTYPES[dtype], modulated=True, seed=21)
    check(shape, DTYPES[dtype], "silu", t, dy)


@pytest.mark.parametrize("value", [30000.0, 3000.0, -0.0123, 57.0])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize(
    "shape", [(3, (30,), 16, 2), (2, (45, 53), 120, 12), (200, (45, 53), 40, 4), (2, (131, 129), 24, 3), (3, (37,), 30, 5), (150, (157,), 102, 3), (2, (33,), 1501, 1)], ids=lambda s: "x".join(map(str, (s[0], *s[1], s[2])))
)
def test_16_bit_groups_without_spread(shape, dtype, value):
    """Nothing but the bias is left of values that are all the same, and no gradient of the weight."""
    B, grid, C, G = shape
    x = torch.full((B, *grid, C), value, dtype=DTYPES[dtype], device="cuda", requires_grad=True)
    weight = torch.linspace(-2, 2, C, device="cuda", requires_grad=True)
    bias = torch.linspace(0, 1, C, device="cuda").to(DTYPES[dtype]).float()
    y = to.group_norm(x, G, weight, bias)
    assert torch.equal(y, bias.to(DTYPES[dtype]).expand_as(x))
    (dw,) = torch.autograd.grad(y, weight, torch.randn_like(y))
    assert not dw.any()
    with torch.no_grad():
        assert torch.equal(to.group_norm(x, G, weight, bias), y)


def activated(kind, z, grad=None):
    """act(z), and grad * act'(z), by way of the shift of samples whose weight is zero: z reaches the activation as it is."""
    shift = z.detach()[:, None].requires_grad_()
    x = torch.arange(4.0, device="cuda", dtype=z.dtype)[None, :, None].expand(z.shape[0], 4, 1)
    y = to.group_norm(x, 1, torch.zeros(1, dtype=z.dtype, device="cuda"), shift=shift, activation=kind)
    if grad is None:
        return y[:, 0, 0].detach()
    cotangent = torch.zeros_like(y)
    cotangent[:, 0, 0] = grad
    return y[:, 0, 0].detach(), torch.autograd.grad(y, shift, cotangent)[0][:, 0]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_gelu_over_its_range(dtype):
    """To the rounding of the result and, in float32, of the steps before it, in units of 2^-24 of the value.  The power's argument z^2 / (2 ln 2) is
    rounded three times (the square, the constant, their product), each of which is z^2 / 2 units of the power: 3 / 2 z^2.  The reciprocal t is off by a
    unit in the last place, which is 2, and the ratio of tail and density changes 3.2 times as fast as t at |z| = 1 and less beyond: 6.4; the power itself
    2, the last of the polynomial's products and sums 3, three products 3: below 16."""
    dtype = DTYPES[dtype]
    z = torch.cat([torch.linspace(-13, 13, 400_001, dtype=torch.float64), torch.linspace(-1.01, 1.01, 200_001, dtype=torch.float64)]).to(dtype).cuda()
    y, slope = activated("gelu", z, torch.ones_like(z))
    want, derivative = field_oracle.activation("gelu", z.double())
    steps = torch.finfo(dtype).eps / 2 + (2.0**-24 * (16 + 1.5 * z.double() ** 2) if dtype == torch.float32 else 2.0**-16)
    least = 2.0**-25 if dtype == torch.float16 else 2.0**-126
    d = (y.double() - want).abs() - (steps * want.abs() + least)
    assert (d <= 0).all(), (z[d.argmax()], y[d.argmax()], want[d.argmax()])
    # (the derivative is a sum of two: both are rounded)
    terms = (want / z.double()).nan_to_num(0.5).abs() + (z.double() * torch.exp(-0.5 * z.double() ** 2) * 0.3989422804014327).abs()
    d = (slope.double() - derivative).abs() - (steps * (terms + derivative.abs()) + least)
    assert (d <= 0).all(), (z[d.argmax()], slope[d.argmax()], derivative[d.argmax()])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_activations_of_very_large_values(dtype, kind):
    """Up to the largest numbers, and of infinity where the limit is one."""
    dtype = DTYPES[dtype]
    most = torch.finfo(dtype).max
    sizes = [v for v in (20.0, 87.0, 88.5, 90.0, 104.0, 130.0, 700.0, 1000.0, 6e4, 1e20, 1e30, 2.3e38, 2.4e38, 3.3e38, 1e300) if v < most] + [most]
    z = torch.tensor(sizes + [-v for v in sizes], dtype=torch.float64).to(dtype).cuda()
    y, slope = activated(kind, z, torch.ones_like(z))
    want, derivative = field_oracle.activation(kind, z.double())
    # (values that underflow count as zero; 128 units and one for each unit of |z|, of which the power's argument has as many as it is large)
    tolerance = torch.finfo(dtype).eps * (129 + z.double().abs().clamp(max=1000))
    for got, value in ((y, want), (slope, derivative)):
        d = (got.double() - value).abs()
        assert ((d <= tolerance * value.abs() + 1e-36 + (2.0**-24 if dtype == torch.float16 else 0)) | (got.double() == value)).all(), (z[d.argmax()], got, value)
    infinite = torch.tensor([float("inf")], dtype=dtype, device="cuda")
    assert activated(kind, infinite).item() == (1.0 if kind == "tanh" else float("inf"))
    assert activated(kind, -infinite).item() in {None: {-float("inf")}, "tanh": {-1.0}, "relu": {0.0}}.get(kind, set()) or kind in ("silu", "gelu")
    assert activated(kind, torch.full_like(infinite, float("nan"))).isnan().all()


# Parts of a sample that take 16 and 32 vectors a thread, with rows of whole vectors and of several positions: 128 workgroups or more of 64 KiB and more.
@pytest.mark.parametrize(
    "dtype,shape",
    [
        ("f32", (130, (64, 60), 8, 2)),
        ("f32", (130, (64, 64), 16, 4)),
        ("f32", (130, (72, 64), 16, 4)),
        ("f32", (130, (4501,), 6, 2)),
        ("f64", (130, (64, 60), 4, 2)),
        ("f64", (130, (90, 70), 4, 2)),
        ("f64", (130, (4501,), 3, 1)),
        ("bf16", (130, (60, 50), 16, 2)),
        ("bf16", (130, (90, 70), 16, 2)),
        ("bf16", (64, (40, 40), 320, 32)),
        ("f16", (130, (90, 70), 16, 2)),
        ("f16", (130, (60, 50), 16, 2)),
        ("f16", (130, (4501,), 12, 3)),
        ("bf16", (130, (4501,), 12, 3)),
    ],
    ids=lambda v: v if isinstance(v, str) else "x".join(map(str, (v[0], *v[1], v[2]))),
)
@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_parts_of_many_vectors(dtype, shape, kind):
    t, dy = made(shape, DTYPES[dtype], params=DTYPES[dtype], modulated=True, seed=22)
    check(shape, DTYPES[dtype], kind, t, dy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, (s[0], *s[1], s[2]))) + f"g{s[3]}")
def test_values_without_a_graph(shape, dtype):
    """No statistics are asked for there: to the last bit what a call with them gives, and that by its definition."""
    i = SHAPES.index(shape)
    t, _ = made(shape, DTYPES[dtype], params=DTYPES[dtype], modulated=i % 2 == 0, seed=i)
    kind, names = KINDS[i % 5], ("weight", "bias", "scale", "shift")
    call = lambda x: to.group_norm(x, shape[3], t["weight"], t["bias"], scale=t.get("scale"), shift=t.get("shift"), activation=kind)
    with torch.no_grad():
        y = call(t["x"])
    graph = call(t["x"].clone().requires_grad_())
    assert graph.requires_grad and not y.requires_grad and torch.equal(y, graph)
    want = field_oracle.group_norm(DTYPES[dtype], t["x"].double(), shape[3], *(t[k].double() if k in t else None for k in names), kind, 1e-5)
    field_oracle.assert_close(y, *want["y"], "y", dtype=DTYPES[dtype])


@pytest.mark.parametrize("positions", [180, 400, 900, 2000])
@pytest.mark.parametrize("wrapped", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_parts_of_few_vectors(dtype, wrapped, positions):
    """One to eight vectors a thread: two or three of them in a row of one or two positions."""
    vector = 128 // torch.finfo(DTYPES[dtype]).bits
    shape = (9, (positions + 1,), vector * 3 // 2 if wrapped else 2 * vector, 3 if wrapped else 2)
    t, dy = made(shape, DTYPES[dtype], params=DTYPES[dtype], modulated=True, seed=positions)
    check(shape, DTYPES[dtype], KINDS[positions % 5], t, dy)


def test_tangents_are_refused():
    x = torch.randn(2, 5, 4, device="cuda", requires_grad=True)
    y = to.group_norm(x, 2)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, x, dual)

    def derivative(v):
        return torch.func.jvp(lambda v: to.group_norm(v, 2), (v,), (torch.ones_like(v),))

    for f in (derivative, torch.compile(derivative, backend="eager")):
        with pytest.raises(NotImplementedError, match="jvp|forward-mode"):
            f(x.detach())


@pytest.mark.parametrize("how", ["trace", "make_fx", "make_fx of gradients", "make_fx of vjp", "make_fx of vmap", "make_fx of a backward pass", "make_fx, symbolic"])
def test_recorded_programs(how):
    """What records a program sees the operation: its replay computes from new inputs what a call does."""
    from torch.fx.experimental.proxy_tensor import make_fx

    shape = (3, (10,), 12, 2)
    (first, dy), (other, _) = ((list(t.values()), dy) for t, dy in (made(shape, torch.float32, params=torch.float32, modulated=True, seed=s) for s in (23, 24)))

    def call(x, weight, bias, scale, shift):
        return to.group_norm(x, 2, weight, bias, scale=scale, shift=shift, activation="silu")

    def gradients(*values):
        leaves = [v.detach().requires_grad_() for v in values]
        return torch.autograd.grad(call(*leaves), leaves, dy)

    def pulled(*values):
        return torch.func.vjp(call, *values)[1](dy)

    def mapped(*values):
        x, _, _, scale, shift = values
        return torch.func.vmap(lambda x, s, h: call(x[None], None, None, s[None], h[None])[0])(x, scale, shift)

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


@pytest.mark.parametrize("kind", [None, "silu"])
def test_batched_cotangents(kind):
    """As one after the other: autograd.grad with is_grads_batched, a Jacobian, and vmap around autograd.grad."""
    shape = (2, (3,), 8, 2)
    t, _ = made(shape, torch.float32, params=torch.float32, modulated=True, seed=25)
    leaves = [v.requires_grad_() for v in t.values()]
    call = lambda x, w, b, s, h: to.group_norm(x, 2, w, b, scale=s, shift=h, activation=kind)
    y = call(*leaves)
    dy = torch.randn((5, *y.shape), generator=torch.Generator().manual_seed(1)).cuda()
    want = [torch.stack(g) for g in zip(*(torch.autograd.grad(y, leaves, g, retain_graph=True) for g in dy))]
    got = torch.autograd.grad(y, leaves, dy, is_grads_batched=True, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    (got,) = torch.autograd.grad(y, leaves[3], dy, is_grads_batched=True, retain_graph=True)
    assert torch.equal(got, want[3])
    for dim in range(3):  # (whichever axis is the mapped one)
        got = torch.func.vmap(lambda g: torch.autograd.grad(y, leaves, g, retain_graph=True), in_dims=dim)(dy.movedim(0, dim))
        for name, a, b in zip(t, got, want):
            # (gradients of shared weights are added up over the samples of one cotangent in another order: two of them, so that it is the same)
            assert torch.equal(a, b), name
    rows = torch.autograd.functional.jacobian(call, tuple(v.detach() for v in leaves), vectorize=True)
    one = torch.autograd.functional.jacobian(call, tuple(v.detach() for v in leaves))
    assert all(torch.equal(a, b) for a, b in zip(rows, one))


@pytest.mark.parametrize("dim", [0, 1, 2, 3])
def test_mapped_along_any_axis(dim):
    t, dy = made((5, (6, 7), 12, 3), torch.float32, params=torch.float32, modulated=False, seed=26)
    f = lambda x, w, b: to.group_norm(x[None], 3, w, b, activation="silu")[0]
    pulled = lambda x, g: torch.func.vjp(f, x, t["weight"], t["bias"])[1](g)
    want = torch.func.vmap(pulled)(t["x"], dy)
    for x_dim, g_dim in ((dim, dim), (0, dim), (dim, 0)):
        got = torch.func.vmap(pulled, in_dims=(x_dim, g_dim))(t["x"].movedim(0, x_dim), dy.movedim(0, g_dim))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # one sample for all cotangents, whose own axes are the grid's
    x = t["x"][0]
    pull = torch.func.vjp(f, x, t["weight"], t["bias"])[1]
    got = torch.func.vmap(pull, in_dims=dim)(dy.movedim(0, dim))
    for a, b in zip(got, zip(*(pull(g) for g in dy))):
        assert torch.equal(a, torch.stack(b))


@pytest.mark.parametrize("which", ["x", "weight", "bias", "scale", "shift", "dy"])
def test_views_that_are_flagged_negative(which):
    """The imaginary part of a conjugate: its memory holds the values of the other sign."""
    t, dy = made((3, (5,), 1, 1), torch.float32, params=torch.float32, modulated=True, seed=27)
    t["dy"] = dy
    flagged = {**t, which: torch.complex(torch.zeros_like(t[which]), -t[which]).conj().imag}
    assert flagged[which].is_neg() and torch.equal(flagged[which], t[which])

    def run(x, weight, bias, scale, shift, dy):
        leaves = [v.detach().requires_grad_() for v in (x, weight, bias, scale, shift)]
        y = to.group_norm(leaves[0], 1, leaves[1], leaves[2], scale=leaves[3], shift=leaves[4], activation="silu")
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    assert all(torch.equal(a, b) for a, b in zip(run(**flagged), run(**t)))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_float32_gradients_of_the_parameters_of_16_bit_data(dtype, kind):
    """One position a sample: a gradient of the shift is a single product, and float32."""
    shape = (2000, (1,), 64, 2)
    t, dy = made(shape, DTYPES[dtype], params=torch.float32, modulated=True, seed=28)
    check(shape, DTYPES[dtype], kind, t, dy)
