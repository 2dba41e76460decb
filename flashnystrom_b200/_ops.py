"""torch.library registration of the forward and backward as custom operators, so that
torch.compile / torch.export trace through `flash_nystrom_attention` without a graph break (the
reference lists this as future work, README.md:387; its autograd.Function behind pybind breaks the
graph).

    torch.ops.flashnystrom_b200.nystrom_fwd(q, k, v, num_landmarks, newton_iter, kappa_star)
        -> (out, q_landmarks, k_landmarks, k2_inv, step2, lse1, lse2, lse3, ns_iterates, k2, bmat)
    torch.ops.flashnystrom_b200.nystrom_bwd(d_out, q, k, v, <the ten saved tensors>, ...)
        -> (dq, dk, dv)

    torch.ops.flashnystrom_b200.decay_fwd(q, k, v, log_decay, scale, initial_state, seq_lens, want_state=True, bounded=False)
        -> (out, final_state, states at the cuts)
    torch.ops.flashnystrom_b200.decay_bwd(..., want_initial=True) -> (dq, dk, dv, d_initial_state)
    torch.ops.flashnystrom_b200.decay_step(q, k, v, state, log_decay, scale, slots) -> out, with state written
    torch.ops.flashnystrom_b200.norm_fwd(x, weight, bias, eps, num_groups, keep=True) -> (y, mean, rstd)
    torch.ops.flashnystrom_b200.norm_bwd(..., want_x=True, want_weight=True, want_bias=True) -> (dx, d_weight, d_bias)

All have fake (meta) implementations, and the forward ones have their autograd formulas registered, so the
operators work under FakeTensorMode, AOT autograd and opcheck.  Eager calls go through the C++ module
(csrc/native.cpp) and, where that hands them back, through the autograd functions of flash_nystrom.py (less dispatcher
overhead per call); `flash_nystrom_attention` switches to the operators while a compiler is tracing."""
from typing import Optional, Tuple

import torch

from . import _C

_LIB = "flashnystrom_b200"


@torch.library.custom_op(f"{_LIB}::nystrom_fwd", mutates_args=(), device_types="cuda")
def nystrom_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, num_landmarks: int, newton_iter: int,
                kappa_star: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                                            torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                                            torch.Tensor]:
    r = _C.forward(q.contiguous(), k.contiguous(), v.contiguous(), num_landmarks, newton_iter, kappa_star, False, True)
    # r = [out, q, k, qt, kt, k2inv, step2, lse1, lse2, lse3, iterates, k2, bmat]; q and k are the
    # caller's own tensors and an operator must not return its inputs
    return (r[0], r[3], r[4], r[5], r[6], r[7], r[8], r[9], r[10], r[11], r[12])


@nystrom_fwd.register_fake
def _(q, k, v, num_landmarks, newton_iter, kappa_star):
    B, H, N, D = q.shape
    m, J = num_landmarks, newton_iter
    f32 = dict(dtype=torch.float32, device=q.device)
    return (torch.empty_like(q, memory_format=torch.contiguous_format),
            torch.empty(B, H, m, D, **f32), torch.empty(B, H, m, D, **f32), torch.empty(B, H, m, m, **f32),
            torch.empty(B, H, m, D, **f32), torch.empty(B, H, N, **f32), torch.empty(B, H, m, **f32),
            torch.empty(B, H, m, **f32), torch.empty(B, H, J + 1, m, m, **f32), torch.empty(B, H, m, m, **f32),
            torch.empty(B, H, m, D, **f32))


@torch.library.custom_op(f"{_LIB}::nystrom_bwd", mutates_args=(), device_types="cuda")
def nystrom_bwd(d_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                q_landmarks: torch.Tensor, k_landmarks: torch.Tensor, k2_inv: torch.Tensor, step2: torch.Tensor,
                lse1: torch.Tensor, lse2: torch.Tensor, lse3: torch.Tensor, ns_iterates: torch.Tensor,
                k2: torch.Tensor, bmat: torch.Tensor, num_landmarks: int, newton_iter: int,
                kappa_star: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    dq, dk, dv = _C.backward(d_out.contiguous(), q.contiguous(), k.contiguous(), q_landmarks, k_landmarks, k2_inv, step2,
                             lse1, lse2, lse3, ns_iterates, k2, bmat, v.contiguous(), out, num_landmarks, newton_iter,
                             True, kappa_star)
    return dq, dk, dv


@nystrom_bwd.register_fake
def _(d_out, q, k, v, out, q_landmarks, k_landmarks, k2_inv, step2, lse1, lse2, lse3, ns_iterates, k2, bmat,
      num_landmarks, newton_iter, kappa_star):
    c = torch.contiguous_format
    return (torch.empty_like(q, memory_format=c), torch.empty_like(k, memory_format=c),
            torch.empty_like(v, memory_format=c))


def _setup_context(ctx, inputs, output):
    q, k, v, m, J, kappa = inputs
    ctx.save_for_backward(q, k, v, *output)
    ctx.m, ctx.J, ctx.kappa = m, J, kappa


def _backward(ctx, d_out, *unused_saved_grads):
    q, k, v, out, qt, kt, k2inv, step2, lse1, lse2, lse3, iters, k2, bmat = ctx.saved_tensors
    dq, dk, dv = nystrom_bwd(d_out, q, k, v, out, qt, kt, k2inv, step2, lse1, lse2, lse3, iters, k2, bmat,
                             ctx.m, ctx.J, ctx.kappa)
    return dq, dk, dv, None, None, None


nystrom_fwd.register_autograd(_backward, setup_context=_setup_context)


def attention_via_ops(q, k, v, num_landmarks, newton_iter, kappa_star):
    """The attention output through the registered operators (differentiable, traceable)."""
    return nystrom_fwd(q, k, v, int(num_landmarks), int(newton_iter), float(kappa_star))[0]


# ---- causal attention with a decay ------------------------------------------------------------------------
# Tensors are taken and given back in the order of memory that they have, as by eager calls; what is not wanted has no elements.
def _rows_like(t):
    """Uninitialised, in the order that t's heads and rows have in memory (t itself where it can be read in place, its contiguous copy otherwise)."""
    B, H, N, D = t.shape
    in_place = t.size(3) == 1 or t.stride(3) == 1
    for i in range(3):
        in_place = in_place and (t.size(i) == 1 or t.stride(i) > 0)
    if in_place and t.stride(1) < t.stride(2):
        return t.new_empty_strided((B, H, N, D), (N * H * D, D, H * D, 1))
    return t.new_empty((B, H, N, D))


def _segment_bound(B, H, N, D, dtype, sms):
    """Floats that the states at the cuts take at most, for sizes that need not be numbers yet: a slice has no more segments than units of 64 (float32) or 128
    rows, all slices together no more than two rounds of CTAs, or one each."""
    unit, slots = (64, 2 * sms if D <= 64 else sms) if dtype == torch.float32 else (128, sms)
    units = (N + unit - 1) // unit
    return D * D * torch.sym_min(B * H * units, torch.sym_max(B * H, 2 * slots))


def _bound_of(q):
    return _segment_bound(*q.shape, q.dtype, torch.cuda.get_device_properties(q.device).multi_processor_count)


def _segment_floats(q):
    from . import _lib
    import ctypes as C
    shape = _lib.DecayShape(q.shape[0], q.shape[1], q.shape[2], q.shape[3], _C._DTYPES[q.dtype], 1.0, _C._flags & _lib.FNB_FLAG_FORCE_GENERIC)
    with _C._on_device(q.device):
        return _lib.load().fnb_decay_segment_floats(C.byref(shape))


@torch.library.custom_op(f"{_LIB}::decay_fwd", mutates_args=(), device_types="cuda")
def decay_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, scale: float,
              initial_state: Optional[torch.Tensor], seq_lens: Optional[torch.Tensor], want_state: bool = True,
              bounded: bool = False) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """bounded: the states at the cuts in room by _segment_bound, whose size holds for symbols, in place of what this very length takes."""
    return _C.native().decay_forward(q, k, v, log_decay, scale, initial_state, seq_lens, want_state, int(_bound_of(q)) if bounded else -1, _C._status(q.device))


@decay_fwd.register_fake
def _(q, k, v, log_decay, scale, initial_state, seq_lens, want_state=True, bounded=False):
    B, H, N, D = q.shape
    f32 = dict(dtype=torch.float32, device=q.device)
    return (_rows_like(q), torch.empty((B, H, D, D) if want_state else (0,), **f32), torch.empty(_bound_of(q) if bounded else _segment_floats(q), **f32))


@torch.library.custom_op(f"{_LIB}::decay_bwd", mutates_args=(), device_types="cuda")
def decay_bwd(d_out: torch.Tensor, d_state: Optional[torch.Tensor], q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, scale: float,
              initial_state: Optional[torch.Tensor], seq_lens: Optional[torch.Tensor], segments: torch.Tensor,
              want_initial: bool = True) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return _C.native().decay_backward(d_out, d_state, q, k, v, log_decay, scale, initial_state, seq_lens, segments, want_initial, _C._status(q.device))


@decay_bwd.register_fake
def _(d_out, d_state, q, k, v, log_decay, scale, initial_state, seq_lens, segments, want_initial=True):
    B, H, N, D = q.shape
    return _rows_like(q), _rows_like(k), _rows_like(v), torch.empty((B, H, D, D) if want_initial else (0,), dtype=torch.float32, device=q.device)


def _decay_context(ctx, inputs, output):
    q, k, v, log_decay, scale, initial_state, seq_lens, want_state, _ = inputs
    ctx.save_for_backward(q, k, v, log_decay, initial_state, seq_lens, output[2])
    ctx.scale, ctx.want_state = scale, want_state
    ctx.set_materialize_grads(False)


def _decay_backward(ctx, d_out, d_state, _unused):
    q, k, v, log_decay, initial_state, seq_lens, segments = ctx.saved_tensors
    if not ctx.want_state:
        d_state = None
    if d_out is None and d_state is None:
        return (None,) * 9
    want_initial = initial_state is not None and ctx.needs_input_grad[5]
    dq, dk, dv, ds = decay_bwd(torch.zeros_like(q) if d_out is None else d_out, d_state, q, k, v, log_decay, ctx.scale, initial_state, seq_lens, segments,
                               want_initial)
    return dq, dk, dv, None, None, ds if want_initial else None, None, None, None


decay_fwd.register_autograd(_decay_backward, setup_context=_decay_context)


def decay_attention_via_ops(q, k, v, log_decay, scale, initial_state, seq_lens, want_state):
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("log_decay is a constant here: it has no gradient")
    out, state, _ = decay_fwd(q, k, v, log_decay, scale, initial_state, seq_lens, want_state, torch.compiler.is_compiling())
    return out, state


@torch.library.custom_op(f"{_LIB}::decay_step", mutates_args=("state",), device_types="cuda")
def decay_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, state: torch.Tensor, log_decay: torch.Tensor, scale: float,
               slots: Optional[torch.Tensor]) -> torch.Tensor:
    return _C.native().decay_step(q, k, v, state, log_decay, scale, slots)


@decay_step.register_fake
def _(q, k, v, state, log_decay, scale, slots):
    return torch.empty_like(q, memory_format=torch.contiguous_format)


# ---- layer norm -------------------------------------------------------------------------------------------
@torch.library.custom_op(f"{_LIB}::norm_fwd", mutates_args=(), device_types="cuda")
def norm_fwd(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float, num_groups: int,
             keep: bool = True) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """keep: the statistics too, which the backward reads."""
    return _C.native().norm_forward(x, weight, bias, eps, num_groups, keep)


@norm_fwd.register_fake
def _(x, weight, bias, eps, num_groups, keep=True):
    runs = x.numel() // x.shape[-1] * num_groups if keep else 0
    f32 = dict(dtype=torch.float32, device=x.device)
    return torch.empty_like(x, memory_format=torch.contiguous_format), torch.empty(runs, **f32), torch.empty(runs, **f32)


@torch.library.custom_op(f"{_LIB}::norm_bwd", mutates_args=(), device_types="cuda")
def norm_bwd(d_y: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor, rstd: torch.Tensor, eps: float, num_groups: int,
             param_f32: bool, want_x: bool = True, want_weight: bool = True, want_bias: bool = True) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _C.native().norm_backward(d_y, x, weight, mean, rstd, eps, num_groups, param_f32, want_x, want_weight, want_bias)


@norm_bwd.register_fake
def _(d_y, x, weight, mean, rstd, eps, num_groups, param_f32, want_x=True, want_weight=True, want_bias=True):
    p = dict(dtype=torch.float32 if param_f32 else x.dtype, device=x.device)
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if want_x else x.new_empty(0)
    return dx, torch.empty(x.shape[-1] if want_weight else 0, **p), torch.empty(x.shape[-1] if want_bias else 0, **p)


def _norm_context(ctx, inputs, output):
    x, weight, bias, eps, num_groups, _ = inputs
    ctx.save_for_backward(x, weight, output[1], output[2])
    ctx.eps, ctx.num_groups, ctx.has_bias = eps, num_groups, bias is not None
    param = weight if weight is not None else bias
    ctx.param_f32 = param is None or param.dtype == torch.float32


def _norm_backward(ctx, d_y, _mean, _rstd):
    x, weight, mean, rstd = ctx.saved_tensors
    want = ctx.needs_input_grad[0], weight is not None and ctx.needs_input_grad[1], ctx.has_bias and ctx.needs_input_grad[2]
    grads = norm_bwd(d_y, x, weight, mean, rstd, ctx.eps, ctx.num_groups, ctx.param_f32, *want)
    return (*(g if w else None for g, w in zip(grads, want)), None, None, None)


norm_fwd.register_autograd(_norm_backward, setup_context=_norm_context)


def layer_norm_via_ops(x, weight, bias, eps, num_groups):
    return norm_fwd(x, weight, bias, eps, num_groups, torch.is_grad_enabled())[0]
