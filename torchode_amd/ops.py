"""``torch.ops.torchode_amd``: the whole-solve entry point of the C ABI as PyTorch operators.

The library's own eager path calls the C ABI through an extension of its own (``csrc/tode_host.cpp``) or ``ctypes``
(``_lib.py``): fewer microseconds per call than the dispatcher.  The operators here are the same entry points for programs that PyTorch
captures: ``torch.compile(solver.solve)`` with a built-in term records the whole solve as one node,
``torchode_amd::solve_builtin``, instead of breaking the graph at a foreign function call.  The
operators are registered by ``libtorchode_amd_ops.so`` (``csrc/tode_torch_ops.cpp``, built by
``torchode_amd.build`` next to ``libtorchode_amd.so``), for the GPU only: there is no CPU
implementation, and a call with CPU tensors fails in the dispatcher.  Shapes and dtypes of the
results for tracing come from the functions registered below.

Reference: the loop these replace is ``AutoDiffAdjoint.solve`` (adjoints.py:42-311); the reference's
own route to a compiled solve is ``torch.compile`` of that loop (docs/jit.ipynb).
"""
import os
import threading
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib, build

_lock = threading.Lock()
_loaded = False


def load() -> None:
    """Loads the operator library (after the library it calls into) and registers the tracing rules."""
    if not _loaded:  # (read without the lock: a tracer that runs through here sees one global and no lock)
        _load_once()


@torch.compiler.disable
def _load_once() -> None:
    global _loaded
    with _lock:
        if _loaded:
            return
        _lib.load()
        if not os.path.exists(build.OPS_LIB):
            build.link_ops_library()
        torch.ops.load_library(build.OPS_LIB)

        @torch.library.register_fake("torchode_amd::solve_builtin")
        def _(y0, t_start, t_end, t_eval, dt0, params, shared_params, method, term, term_scalars, controller_kind, control, max_steps, allow_one_kernel):
            B, F = y0.shape
            E = 1 if t_eval is None else max(t_eval.shape[1], 1)
            stat = lambda: y0.new_empty((B,), dtype=torch.long)
            return y0.new_empty((B, E, F)), stat(), stat(), stat(), stat(), torch.empty((), dtype=torch.long, device="cpu")

        @torch.library.register_fake("torchode_amd::mlp_pack_weights")
        def _(raw, matrix_inputs, n_features=64):
            return raw.new_empty((_lib.MLP_PACKED_SIZE["bfloat16" if matrix_inputs == _lib.MLP_INPUTS["bfloat16"] else "float32"],))

        _loaded = True


def solve_builtin(
    y0: torch.Tensor,
    t_start: torch.Tensor,
    t_end: torch.Tensor,
    t_eval: Optional[torch.Tensor],
    dt0: Optional[torch.Tensor],
    params: Optional[torch.Tensor],
    shared_params: Optional[torch.Tensor],
    method: int,
    term: int,
    term_scalars: Sequence[float],
    controller_kind: int,
    control: Sequence[float],
    max_steps: Optional[int] = None,
    allow_one_kernel: bool = True,
):
    """``(ys, n_steps, n_accepted, n_initialized, status, iterations)`` of one whole solve with a built-in term
    (``tode_solve_builtin_auto``).  ``iterations`` is an int64 scalar on the CPU: the loop iterations, from which
    ``stats["n_f_evals"]`` follows."""
    load()
    return torch.ops.torchode_amd.solve_builtin(
        y0, t_start, t_end, t_eval, dt0, params, shared_params, method, term, list(term_scalars), controller_kind, list(control),
        -1 if max_steps is None else int(max_steps), allow_one_kernel,
    )  # fmt: skip


def mlp_pack_weights(raw: torch.Tensor, matrix_inputs: int, n_features: int = 64) -> torch.Tensor:
    load()
    return torch.ops.torchode_amd.mlp_pack_weights(raw, matrix_inputs, n_features)


def group_norm_forward(x, n_groups, weight, bias, scale, shift, activation, eps):
    """The result of ``torchode_amd.group_norm``, its means and the reciprocals of its deviations, as one operation of a program that is being recorded."""
    return torch.ops.torchode_amd.group_norm(x, n_groups, weight, bias, scale, shift, activation, eps)


def group_norm(x, n_groups, weight, bias, scale, shift, activation, eps):
    return group_norm_forward(x, n_groups, weight, bias, scale, shift, activation, eps)[0]


def _where_wanted(gradients, wanted):
    """A list of the wanted gradients, with None for the others."""
    left = iter(gradients)
    return tuple(next(left) if w else None for w in wanted)


def group_norm_backward(dy, x, mean, rstd, n_groups, weight, bias, scale, shift, activation, want):
    wanted = [want >> i & 1 and t is not None for i, t in enumerate((x, weight, bias, scale, shift))]
    want = sum(1 << i for i in range(5) if wanted[i])
    return _where_wanted(torch.ops.torchode_amd.group_norm_backward(dy, x, mean, rstd, n_groups, weight, bias, scale, shift, activation, want), wanted)


def cross_attention_forward(q, k, v, lengths, mask, scale):
    """``torchode_amd.cross_attention`` likewise, with what rounding took off the result and its rows' log-sums."""
    return torch.ops.torchode_amd.cross_attention(q, k, v, lengths, mask, scale)


def cross_attention(q, k, v, lengths, mask, scale):
    return cross_attention_forward(q, k, v, lengths, mask, scale)[0]


def cross_attention_backward(grad, q, k, v, out, low, lse, lengths, mask, scale, want_q, want_kv):
    return _where_wanted(torch.ops.torchode_amd.cross_attention_backward(grad, q, k, v, out, low, lse, lengths, mask, scale, want_q, want_kv), (want_q, want_kv, want_kv))


# The operators of a right-hand side (field_ops.py) are registered here, over the same native calls that the eager functions make.
_Three = Tuple[torch.Tensor, torch.Tensor, torch.Tensor]
_Opt = Optional[torch.Tensor]


@torch.library.custom_op("torchode_amd::group_norm", mutates_args=(), device_types="cuda")
def _group_norm(x: torch.Tensor, n_groups: int, weight: _Opt, bias: _Opt, scale: _Opt, shift: _Opt, activation: int, eps: float) -> _Three:
    return _lib.load_host().group_norm_forward(x, n_groups, weight, bias, scale, shift, activation, eps)


@_group_norm.register_fake
def _(x, n_groups, weight, bias, scale, shift, activation, eps):
    statistics = lambda: x.new_empty((x.shape[0], n_groups), dtype=torch.float64 if x.dtype == torch.float64 else torch.float32)
    return x.new_empty(x.shape), statistics(), statistics()


@torch.library.custom_op("torchode_amd::group_norm_backward", mutates_args=(), device_types="cuda")
def _group_norm_backward(
    dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, n_groups: int, weight: _Opt, bias: _Opt, scale: _Opt, shift: _Opt, activation: int, want: int
) -> List[torch.Tensor]:
    """The gradients that bit i of ``want`` asks for, in the order x, weight, bias, scale, shift."""
    return [g for g in _lib.load_host().group_norm_backward(dy, x, mean, rstd, n_groups, weight, bias, scale, shift, activation, want) if g is not None]


@_group_norm_backward.register_fake
def _(dy, x, mean, rstd, n_groups, weight, bias, scale, shift, activation, want):
    return [t.new_empty(t.shape) for i, t in enumerate((x, weight, bias, scale, shift)) if want >> i & 1]


def _group_norm_context(ctx, inputs, output):
    x, ctx.n_groups, weight, bias, scale, shift, ctx.activation, _ = inputs
    ctx.mark_non_differentiable(*output[1:])
    ctx.save_for_backward(x, weight, bias, scale, shift, *output[1:])


def _group_norm_gradients(ctx, dy, _mean, _rstd):
    x, weight, bias, scale, shift, mean, rstd = ctx.saved_tensors
    want = sum(1 << i for i, j in enumerate((0, 2, 3, 4, 5)) if ctx.needs_input_grad[j])
    dx, *rest = group_norm_backward(dy, x, mean, rstd, ctx.n_groups, weight, bias, scale, shift, ctx.activation, want)
    return dx, None, *rest, None, None


_group_norm.register_autograd(_group_norm_gradients, setup_context=_group_norm_context)


@torch.library.custom_op("torchode_amd::cross_attention", mutates_args=(), device_types="cuda")
def _cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: _Opt, mask: _Opt, scale: Optional[float]) -> _Three:
    return _lib.load_host().cross_attention_forward(q, k, v, lengths, mask, scale)


@_cross_attention.register_fake
def _(q, k, v, lengths, mask, scale):
    return q.new_empty(q.shape), q.new_empty((*q.shape[:3], 0 if q.dtype == torch.float32 else q.shape[3])), q.new_empty(q.shape[:3], dtype=torch.float32)


@torch.library.custom_op("torchode_amd::cross_attention_backward", mutates_args=(), device_types="cuda")
def _cross_attention_backward(
    grad: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, low: torch.Tensor, lse: torch.Tensor, lengths: _Opt, mask: _Opt,
    scale: Optional[float], want_q: bool, want_kv: bool,
) -> List[torch.Tensor]:  # fmt: skip
    """The gradient of q, those of k and v, as far as wanted."""
    return [g for g in _lib.load_host().cross_attention_backward(grad, q, k, v, out, low, lse, lengths, mask, scale, want_q, want_kv) if g is not None]


@_cross_attention_backward.register_fake
def _(grad, q, k, v, out, low, lse, lengths, mask, scale, want_q, want_kv):
    return [t.new_empty(t.shape) for t, wanted in ((q, want_q), (k, want_kv), (v, want_kv)) if wanted]


def _cross_attention_context(ctx, inputs, output):
    q, k, v, lengths, mask, ctx.scale = inputs
    ctx.mark_non_differentiable(*output[1:])
    ctx.save_for_backward(q, k, v, *output, lengths, mask)


def _cross_attention_gradients(ctx, grad, _low, _lse):
    want_q, want_k, want_v = ctx.needs_input_grad[:3]
    *saved, lengths, mask = ctx.saved_tensors
    return *cross_attention_backward(grad, *saved, lengths, mask, ctx.scale, want_q, want_k or want_v), None, None, None


_cross_attention.register_autograd(_cross_attention_gradients, setup_context=_cross_attention_context)
