"""Operators for a right-hand side of one's own: what a neural field computes between its linear layers.

``group_norm`` normalises a field on grids (channels last), modulates it by the time and applies the activation;
``cross_attention`` lets the state of every sample look at what an encoder has said about it.  Both are functions of
tensors on the GPU, a few hand-written kernels each (``csrc/tode_norm.hip``, ``csrc/tode_attention.hip``), with gradients:
an ``f`` that calls them goes wherever an ``f`` of torch operations goes -- ``AutoDiffAdjoint`` with and without gradients, HIP
graphs of its iterations (``graph_iterations``), both backsolve adjoints (``BacksolveAdjoint`` calls ``f`` one sample at a time under
``vmap``: shape the state with ``y.reshape(-1, ...)`` there), ``torch.compile`` of ``f``, ``torch.jit.trace`` and ``make_fx``.  Samples stay
independent of each other, as the solver takes them to be.

Neither is differentiable twice or in forward mode: both are refused, as are ``torch.func.grad`` and ``vjp`` inside of a program that is being
compiled (by PyTorch, which has no such transforms of operators).  The reference leaves ``f`` to the user (terms.py:13-19).
"""
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib

# A call inside torch.func.vmap, vjp, ... hands out tensors in wrappers: those go through the autograd.Functions below, others through
# nodes of the extension (csrc/tode_host.cpp).
_transformed = torch._C._are_functorch_transforms_active


def _ops():
    """The operators that the dispatcher knows, for programs that something records."""
    from . import ops

    return ops


def _without_tangents(name, *tensors):
    """In a program that is being compiled (elsewhere the extension looks): PyTorch lets operators without a forward-mode derivative drop tangents."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative")


def group_norm(
    x: torch.Tensor,
    n_groups: int,
    weight: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    *,
    scale: Optional[torch.Tensor] = None,
    shift: Optional[torch.Tensor] = None,
    activation: Optional[str] = None,
    eps: float = 1e-5,
) -> torch.Tensor:
    """``act((n * weight + bias) * (1 + scale) + shift)`` with ``n`` the values of ``x`` ``[B, ..., C]`` less the mean of their
    sample's group and divided by ``sqrt(variance + eps)``: groups of ``C / n_groups`` neighbouring channels, mean and (biased) variance over
    all axes between the first and the last.

    ``weight`` and ``bias`` are ``[C]``, or ``[B, C]`` for one of each sample; ``scale`` and ``shift`` ``[B, C]``: the modulation by
    each sample's own time (or by anything else known of the sample).  Any of the four may be left out.  ``activation``: ``None``, ``"silu"``,
    ``"gelu"`` (with the error function), ``"tanh"`` or ``"relu"`` (of derivative 0 at 0).  Types: float32, float64, bfloat16, float16;
    with the latter two, ``weight`` and ``bias``, and ``scale`` and ``shift``, may be float32.  Statistics, sums and everything up
    to the result's rounding are float32 (float64 for float64).  ``x`` is read in place if it is contiguous, from a copy otherwise."""
    if activation not in _lib.ACTIVATIONS:
        raise ValueError(f"group_norm: activation must be one of {list(_lib.ACTIVATIONS)}, got {activation!r}")
    act = _lib.ACTIVATIONS[activation]
    if torch.compiler.is_compiling():
        _without_tangents("group_norm", x, weight, bias, scale, shift)
        return _ops().group_norm(x, n_groups, weight, bias, scale, shift, act, eps)
    if _transformed():
        return _GroupNorm.apply(x, weight, bias, scale, shift, n_groups, act, eps)[0]
    y = _lib.load_host().group_norm(x, n_groups, weight, bias, scale, shift, act, eps)
    return _ops().group_norm(x, n_groups, weight, bias, scale, shift, act, eps) if y is None else y


def _first(t, dim, size):
    """The mapped axis of a tensor in front; a tensor without one is repeated along it."""
    if t is None:
        return None
    return t.expand(size, *t.shape) if dim is None else t.movedim(dim, 0)


def _fold_norm(size, dims, x, weight, bias, scale, shift, per_sample):
    """The arguments of a mapped group norm as those of one with ``size`` times as many samples."""
    x_dim, w_dim, b_dim, scale_dim, shift_dim = dims
    x = _first(x, x_dim, size)
    samples = x.shape[1]
    per_sample = per_sample or any(t is not None and (d is not None or t.ndim == 2) for t, d in ((weight, w_dim), (bias, b_dim)))
    fold = lambda t: t.reshape(size * samples, *t.shape[2:])

    def affine(t, dim):
        if t is None or not per_sample:
            return t
        t = _first(t, dim, size)
        return fold(t[:, None].expand(size, samples, t.shape[-1]) if t.ndim == 2 else t)

    modulation = [None if t is None else fold(_first(t, d, size)) for t, d in ((scale, scale_dim), (shift, shift_dim))]
    return samples, fold(x), affine(weight, w_dim), affine(bias, b_dim), *modulation


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(x, weight, bias, scale, shift, n_groups, act, eps):
        if _lib.load_host().watched(x):
            return _ops().group_norm_forward(x, n_groups, weight, bias, scale, shift, act, eps)
        return _lib.load_host().group_norm_forward(x, n_groups, weight, bias, scale, shift, act, eps)

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, weight, bias, scale, shift, ctx.n_groups, ctx.act, _ = inputs
        _, mean, rstd = output
        ctx.mark_non_differentiable(mean, rstd)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, scale, shift, mean, rstd)

    @staticmethod
    def backward(ctx, dy, _mean, _rstd):
        if dy is None:
            return (None,) * 8
        x, weight, bias, scale, shift, mean, rstd = ctx.saved_tensors
        want = sum(1 << i for i in range(5) if ctx.needs_input_grad[i])
        gradients = _GroupNormBackward.apply(dy, x, mean, rstd, weight, bias, scale, shift, ctx.n_groups, ctx.act, want)
        return (*gradients, None, None, None)

    @staticmethod
    def vmap(info, in_dims, x, weight, bias, scale, shift, n_groups, act, eps):
        samples, *folded = _fold_norm(info.batch_size, in_dims[:5], x, weight, bias, scale, shift, False)
        out = _GroupNorm.apply(*folded, n_groups, act, eps)
        return tuple(t.reshape(info.batch_size, samples, *t.shape[1:]) for t in out), (0, 0, 0)


class _GroupNormBackward(torch.autograd.Function):
    @staticmethod
    def forward(dy, x, mean, rstd, weight, bias, scale, shift, n_groups, act, want):
        if _lib.load_host().watched(x):
            return _ops().group_norm_backward(dy, x, mean, rstd, n_groups, weight, bias, scale, shift, act, want)
        return _lib.load_host().group_norm_backward(dy, x, mean, rstd, n_groups, weight, bias, scale, shift, act, want)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *_):
        raise NotImplementedError("group_norm is not differentiable twice")

    @staticmethod
    def vmap(info, in_dims, dy, x, mean, rstd, weight, bias, scale, shift, n_groups, act, want):
        size = info.batch_size
        dy_dim, x_dim, mean_dim, rstd_dim, *dims = in_dims[:8]
        # (every mapped sample has its own gradient of a weight, also of one that they share)
        samples, x, *params = _fold_norm(size, (x_dim, *dims), x, weight, bias, scale, shift, True)
        dy, mean, rstd = _fold(size, (dy_dim, mean_dim, rstd_dim), dy, mean, rstd)
        out = list(_GroupNormBackward.apply(dy, x, mean, rstd, *params, n_groups, act, want))
        out = [None if g is None else g.reshape(size, samples, *g.shape[1:]) for g in out]
        for i, (t, d) in enumerate(((weight, dims[0]), (bias, dims[1]))):
            if out[1 + i] is not None and t.ndim == (1 if d is None else 2):
                out[1 + i] = out[1 + i].sum(1)
        return tuple(out), tuple(None if g is None else 0 for g in out)


def cross_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    lengths: Optional[torch.Tensor] = None,
    mask: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """``softmax(scale * q @ k.T) @ v`` of every sample and head: ``q`` ``[B, queries, heads, D]`` are the tokens of the state (a
    state that is one vector is a single one), ``k`` and ``v`` ``[B, keys, kv_heads, D]`` what an encoder has made of the sample's context.
    Head ``h`` of ``q`` looks at head ``h // (heads // kv_heads)`` of ``k`` and ``v``.

    ``lengths`` (``[B]``, int32 or int64): sample ``b`` looks at its first ``lengths[b]`` positions (none if negative, all if more than there are);
    ``mask`` (``[B, keys]``, bool): and only at those with ``True``.  What lies at the other positions -- infinities and NaN
    included -- reaches no result, and gets gradients of zero.  A sample without any position to look at gets zeros.
    ``scale``: ``1 / sqrt(D)`` unless given.

    Types: float32 (``D`` up to 128), bfloat16, float16 (up to 256).  Scores, softmax and sums are float32; with the latter two
    the softmax's weights (and in the backward pass the scores' gradients) are rounded to the data's type ahead of the product with ``v``
    (``q``, ``k``), float16 ones in a range of their own; the weights of up to eight rows (queries times the heads that share a head of
    keys) are not.  Tensors are read in place, whatever the strides of their first three axes; the values of a head have to lie
    side by side, a tensor where they do not is copied."""
    if torch.compiler.is_compiling():
        _without_tangents("cross_attention", q, k, v)
        return _ops().cross_attention(q, k, v, lengths, mask, scale)
    if _transformed():
        return _CrossAttention.apply(q, k, v, lengths, mask, scale)[0]
    out = _lib.load_host().cross_attention(q, k, v, lengths, mask, scale)
    return _ops().cross_attention(q, k, v, lengths, mask, scale) if out is None else out


def _fold(size, dims, *tensors):
    """Mapped tensors with the mapped axis and the one of samples as one."""
    fronted = (_first(t, d, size) for t, d in zip(tensors, dims))
    return [None if t is None else t.reshape(size * t.shape[1], *t.shape[2:]) for t in fronted]


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(q, k, v, lengths, mask, scale):
        if _lib.load_host().watched(q):
            return _ops().cross_attention_forward(q, k, v, lengths, mask, scale)
        return _lib.load_host().cross_attention_forward(q, k, v, lengths, mask, scale)

    @staticmethod
    def setup_context(ctx, inputs, output):
        q, k, v, lengths, mask, ctx.scale = inputs
        ctx.mark_non_differentiable(*output[1:])
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, *output, lengths, mask)

    @staticmethod
    def backward(ctx, grad, _low, _lse):
        if grad is None:
            return (None,) * 6
        q, k, v, out, low, lse, lengths, mask = ctx.saved_tensors
        want_q, want_k, want_v = ctx.needs_input_grad[:3]
        dq, dk, dv = _CrossAttentionBackward.apply(grad, q, k, v, out, low, lse, lengths, mask, ctx.scale, want_q, want_k or want_v)
        return dq, dk, dv, None, None, None

    @staticmethod
    def vmap(info, in_dims, q, k, v, lengths, mask, scale):
        out = _CrossAttention.apply(*_fold(info.batch_size, in_dims, q, k, v, lengths, mask), scale)
        return tuple(t.reshape(info.batch_size, t.shape[0] // info.batch_size, *t.shape[1:]) for t in out), (0, 0, 0)


class _CrossAttentionBackward(torch.autograd.Function):
    @staticmethod
    def forward(grad, q, k, v, out, low, lse, lengths, mask, scale, want_q, want_kv):
        if _lib.load_host().watched(q):
            return _ops().cross_attention_backward(grad, q, k, v, out, low, lse, lengths, mask, scale, want_q, want_kv)
        return _lib.load_host().cross_attention_backward(grad, q, k, v, out, low, lse, lengths, mask, scale, want_q, want_kv)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *_):
        raise NotImplementedError("cross_attention is not differentiable twice")

    @staticmethod
    def vmap(info, in_dims, grad, q, k, v, out, low, lse, lengths, mask, scale, want_q, want_kv):
        folded = _fold(info.batch_size, in_dims, grad, q, k, v, out, low, lse, lengths, mask)
        gradients = _CrossAttentionBackward.apply(*folded, scale, want_q, want_kv)
        gradients = tuple(None if g is None else g.reshape(info.batch_size, g.shape[0] // info.batch_size, *g.shape[1:]) for g in gradients)
        return gradients, tuple(None if g is None else 0 for g in gradients)
