"""Refusals of the operators for right-hand sides of one's own: without a GPU."""
import pytest
import torch

import torchode_amd as to

Z = torch.zeros


@pytest.mark.parametrize(
    "x,groups,kwargs,message",
    [
        (Z(4), 1, {}, r"\[batch, \.\.\., channels\]"),
        (Z(2, 3, 4), 3, {}, "cannot be divided"),
        (Z(2, 3, 4), 0, {}, "cannot be divided"),
        (Z(2, 3, 4), -2, {}, "cannot be divided"),
        (Z(2, 3, 0), 1, {}, "cannot be divided"),
        (Z(2, 3, 4), 2, dict(weight=Z(3)), "weight must be"),
        (Z(2, 3, 4), 2, dict(weight=Z(3, 4)), "weight must be"),
        (Z(2, 3, 4), 2, dict(weight=Z(4), bias=Z(2, 4)), "the same shape"),
        (Z(2, 3, 4), 2, dict(scale=Z(4)), "scale must be"),
        (Z(2, 3, 4), 2, dict(shift=Z(2, 5)), "shift must be"),
        (Z(2, 3, 4), 2, dict(weight=Z(4).double()), "x's type"),
        (Z(2, 3, 4).double(), 2, dict(weight=Z(4)), "x's type"),
        (Z(2, 3, 4).bfloat16(), 2, dict(weight=Z(4).half()), "x's type"),
        (Z(2, 3, 4).bfloat16(), 2, dict(weight=Z(4).bfloat16(), bias=Z(4)), "the same type"),
        (Z(2, 3, 4), 2, dict(activation="swish"), "activation"),
        (Z(2, 3, 4), 2, dict(weight=Z(4, device="meta")), "is on meta"),
    ],
)
def test_group_norm_refuses(x, groups, kwargs, message):
    with pytest.raises(ValueError, match=message):
        to.group_norm(x, groups, **kwargs)


def test_group_norm_refuses_other_types_and_devices():
    with pytest.raises(NotImplementedError, match="float32"):
        to.group_norm(Z(2, 3, 4, dtype=torch.long), 2)
    with pytest.raises(RuntimeError, match="AMD GPU"):
        to.group_norm(Z(2, 3, 4), 2)
    with pytest.raises(RuntimeError, match="AMD GPU"):
        to.group_norm(Z(2, 3, 4, requires_grad=True), 2, activation="silu")
    with pytest.raises(TypeError, match="must be a tensor"):
        to.group_norm([1.0], 1)


Q, K = Z(2, 3, 4, 8), Z(2, 5, 2, 8)


@pytest.mark.parametrize(
    "q,k,v,kwargs,message",
    [
        (Q[0], K, K, {}, r"\[batch, queries, heads, head_dim\]"),
        (Q, K, K[:, 1:], {}, "k and v must both"),
        (Q, K[0], K[0], {}, "k and v must both"),
        (Q, K[:1], K[:1], {}, "differ in batch or head_dim"),
        (Q, K[..., 1:], K[..., 1:], {}, "differ in batch or head_dim"),
        (Q[:, :, :3], K, K, {}, "evenly"),
        (Q, K[:, :, :0], K[:, :, :0], {}, "evenly"),
        (Q, K.half(), K.half(), {}, "the same type"),
        (Z(1, 1, 1, 129), Z(1, 1, 1, 129), Z(1, 1, 1, 129), {}, "1 to 128"),
        (Z(1, 1, 1, 257).half(), Z(1, 1, 1, 257).half(), Z(1, 1, 1, 257).half(), {}, "1 to 256"),
        (Z(1, 1, 1, 0), Z(1, 1, 1, 0), Z(1, 1, 1, 0), {}, "1 to 128"),
        (Q, K, K, dict(lengths=Z(2)), "lengths must be"),
        (Q, K, K, dict(lengths=Z(3, dtype=torch.int32)), "lengths must be"),
        (Q, K, K, dict(mask=Z(2, 5)), "mask must be"),
        (Q, K, K, dict(mask=Z(2, 4, dtype=torch.bool)), "mask must be"),
        (Q, K, K, dict(scale=float("inf")), "scale must be finite"),
        (Q, K, K, dict(lengths=Z(2, dtype=torch.int32, device="meta")), "is on meta"),
    ],
)
def test_cross_attention_refuses(q, k, v, kwargs, message):
    with pytest.raises(ValueError, match=message):
        to.cross_attention(q, k, v, **kwargs)


def test_cross_attention_refuses_other_types_and_devices():
    with pytest.raises(NotImplementedError, match="float32, bfloat16 and float16"):
        to.cross_attention(Q.double(), K.double(), K.double())
    with pytest.raises(RuntimeError, match="AMD GPU"):
        to.cross_attention(Q, K, K)
    with pytest.raises(RuntimeError, match="AMD GPU"):
        to.cross_attention(Q.clone().requires_grad_(), K, K)


def test_c_entries_report_what_they_do_not_take():
    import ctypes as C

    from torchode_amd import _lib

    lib = _lib.load()
    for name in ("tode_group_norm", "tode_group_norm_backward", "tode_cross_attention", "tode_cross_attention_backward"):
        assert getattr(lib, name)(None, None) == _lib.E_INVALID and b"null" in lib.tode_last_error()
    zeros = C.create_string_buffer(4096)  # sizes of zero: no group, no head
    for name in ("tode_group_norm", "tode_cross_attention"):
        assert getattr(lib, name + "_workspace_bytes")(zeros, 0) == _lib.E_INVALID and b"bad sizes" in lib.tode_last_error()
        assert getattr(lib, name)(zeros, None) == _lib.E_INVALID


def attention_args(**fields):
    """struct tode_cross_attention_args of one sample of two queries and three keys, float32, without a tensor."""
    import ctypes as C

    class Args(C.Structure):
        _fields_ = [(n, C.c_int32) for n in ("dtype", "heads", "kv_heads", "head_dim")] + [(n, C.c_int64) for n in ("batch", "queries", "keys")] + [("scale", C.c_double)]
        _fields_ += [(n, C.c_void_p) for n in "qkv"] + [(n, C.c_int64 * 3) for n in ("q_strides", "k_strides", "v_strides", "grad_strides")]
        _fields_ += [("lengths", C.c_void_p), ("mask", C.c_void_p), ("mask_stride", C.c_int64), ("lengths_are_64", C.c_int32), ("reserved", C.c_int32)]
        _fields_ += [(n, C.c_void_p) for n in ("out", "out_low", "lse", "grad_out", "dq", "dk", "dv", "workspace")] + [("workspace_bytes", C.c_int64)]

    a = Args(dtype=0, heads=1, kv_heads=1, head_dim=8, batch=1, queries=2, keys=3, scale=1.0)
    for name, value in fields.items():
        setattr(a, name, type(getattr(a, name))(*value) if isinstance(value, tuple) else value)
    return a


@pytest.mark.parametrize("name", ["q_strides", "k_strides", "v_strides", "grad_strides"])
def test_c_entry_of_cross_attention_refuses_negative_strides(name):
    import ctypes as C

    from torchode_amd import _lib

    lib = _lib.load()
    assert lib.tode_cross_attention_workspace_bytes(C.byref(attention_args(k_strides=(24, 8, 8))), 0) == 0
    for strides in ((-1, 8, 8), (24, -8, 8), (24, 8, -(2**40))):
        args = attention_args(**{name: strides})
        assert lib.tode_cross_attention_workspace_bytes(C.byref(args), 1) == _lib.E_INVALID and b"negative" in lib.tode_last_error()
        assert lib.tode_cross_attention_backward(C.byref(args), None) == _lib.E_INVALID and b"negative" in lib.tode_last_error()
        if name != "grad_strides":  # (not read by the forward pass)
            assert lib.tode_cross_attention_workspace_bytes(C.byref(args), 0) == _lib.E_INVALID
            assert lib.tode_cross_attention(C.byref(args), None) == _lib.E_INVALID and b"negative" in lib.tode_last_error()
    assert lib.tode_cross_attention(C.byref(attention_args(mask_stride=-3)), None) == _lib.E_INVALID and b"negative" in lib.tode_last_error()


# The operators and their differentiable arguments, small and on the CPU: what is refused there is refused ahead of the device.
CALLS = {
    "group_norm": (dict(x=Z(2, 3, 4), weight=Z(4), bias=Z(4), scale=Z(2, 4), shift=Z(2, 4)), lambda t: to.group_norm(t["x"], 2, t["weight"], t["bias"], scale=t["scale"], shift=t["shift"])),
    "cross_attention": (dict(q=Q, k=K, v=K.clone()), lambda t: to.cross_attention(**t)),
}


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("name,argument", [(n, a) for n, (tensors, _) in CALLS.items() for a in tensors])
def test_tangents_are_refused(name, argument, requires_grad):
    tensors, call = CALLS[name]
    t = {k: v.clone().requires_grad_(requires_grad) for k, v in tensors.items()}
    with torch.autograd.forward_ad.dual_level():
        t[argument] = torch.autograd.forward_ad.make_dual(t[argument], torch.ones_like(t[argument]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(t)


@pytest.mark.parametrize("name", CALLS)
def test_recorded_programs_hold_the_operation(name):
    """Whatever records a program or looks on sees an operation of the dispatcher, and not the allocation of its result."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    import torchode_amd.ops  # noqa: F401 (registers them)

    tensors, call = CALLS[name]
    operation = getattr(torch.ops.torchode_amd, name)
    with FakeTensorMode():
        t = {k: torch.empty(v.shape, device="cuda:0") for k, v in tensors.items()}
        first = next(iter(t.values()))
        out = call(t)
        assert out.shape == first.shape and out.device == first.device

        def program(*values):
            return call(dict(zip(t, values)))

        graph = make_fx(program)(*t.values()).graph
        assert [n.target for n in graph.nodes if n.op == "call_function"][0] == operation.default, graph
